"""How callers reach the operators of the paged key-value cache: from several threads, under torch's tracers, with a
workspace of their own, with parameters, and with what is out of range.  Formulas and tolerances are
``tests/test_paged_kv.py``'s."""
import importlib.util
import math
import threading

import pytest
import torch

from tests.conftest import ROOT
from tests.test_paged_kv import LENGTHS, N, TYPES, attention, batch, check_attention, close, generator, kl, rope_tables, step_inputs

gpu = pytest.mark.gpu
P = kl.paged_kv
WORKSPACE = 5                                                        # its place in PAGED_ATTENTION_ARGS


def attend(case, **kw):
    q, cache, table, lengths = case
    return kl.paged_attention(q, cache.k_cache, cache.v_cache, table, lengths, cache.k_scales, cache.v_scales, **kw)


# ---- scratch -------------------------------------------------------------------------
@gpu
def test_calls_under_way_have_scratch_of_their_own(monkeypatch):
    """A call from another thread can come between the two launches of a split one: it must not have its scratch."""
    cases = [batch(generator(i), torch.bfloat16, False, 4, 2, 128, 16, [3000, 50], poison=False) for i in (30, 31)]
    refs = [attend(c) for c in cases]
    real, seen = P._call, []

    def call(index, fn, *args):
        seen.append(N.PAGED_ATTENTION_ARGS.unpack(args[0])[WORKSPACE])
        if len(seen) == 1:                                           # as another thread would, before this call launches
            inner.append(attend(cases[1]))
        real(index, fn, *args)

    inner = []
    monkeypatch.setattr(P, "_call", call)
    outer = attend(cases[0])
    assert seen[0] != seen[1]
    assert torch.equal(outer, refs[0]) and torch.equal(inner[0], refs[1])


@gpu
def test_threads_on_one_stream():
    """Rows at other places of outputs of other sizes, from threads that share the default stream, linears between them."""
    w = kl.quantize_int8_rowwise(torch.randn(512, 512, generator=generator(2), device="cuda"))
    x = torch.randn(4, 512, generator=generator(3), device="cuda").bfloat16()
    cases = [batch(generator(40 + i), torch.bfloat16, False, 4, 2, 128, 16, lengths, poison=False)
             for i, lengths in enumerate(([4000], [70, 3000, 900], [2500] * 5, [5, 5000]))]
    refs = [attend(c) for c in cases]
    torch.cuda.synchronize()
    outs, failed, start = [[] for _ in cases], [], threading.Barrier(len(cases))

    def work(i):
        try:
            start.wait()
            for _ in range(60):
                outs[i].append(attend(cases[i]))
                kl.quant_linear(x, w)
        except Exception as e:                                       # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for out, ref in zip(outs, refs):
        assert len(out) == 60 and all(torch.equal(o, ref) for o in out)


def test_scratch_of_one_call():
    """None for rows that are not split, and never more than what serves any call of these heads."""
    bytes_for = N.lib().kl_paged_attention_call_bytes
    for heads, kv_heads, dim in ((4, 2, 128), (8, 8, 64), (16, 2, 128), (32, 2, 128), (40, 1, 64), (12, 1, 256)):
        for form in (N.KL_KV_SAME, N.KL_KV_INT8):
            assert bytes_for(1, heads, kv_heads, dim, form, 0, 16) == bytes_for(3, heads, kv_heads, dim, form, 16, 16) == 0
            assert bytes_for(2000, heads, kv_heads, dim, form, 1000, 1) == 0
            most = kl.paged_attention_workspace_bytes(1, heads, kv_heads, dim)
            sizes = [bytes_for(b, heads, kv_heads, dim, form, columns, 16) for b in (1, 3) for columns in (100, 5000)]
            assert all(0 < n <= most for n in sizes) and max(sizes) > sizes[0]
    assert bytes_for(0, 4, 2, 128, N.KL_KV_SAME, 100, 16) == 0


# ---- weights of f16 caches --------------------------------------------------------------
@gpu
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 128), (8, 8, 64), (16, 2, 128), (8, 1, 64), (32, 2, 128), (16, 1, 64), (12, 1, 256)])
@pytest.mark.parametrize("low,high", [(-28.0, -16.0), (-20.62, -20.62), (-25.5, -25.5)])
def test_small_weights_of_f16_caches(heads, kv_heads, dim, low, high):
    """One key in eight has nearly all the weight and values of zero; the output is that of the others, 2^low to 2^high of it."""
    g = generator(dim + heads)
    q, cache, table, lengths = batch(g, torch.float16, False, heads, kv_heads, dim, 16, [4097, 300, 16385, 17], poison=False)
    q.zero_()
    q[..., 0] = 1.0
    k = low + (high - low) * torch.rand(cache.k_cache.shape[:3], generator=g, device="cuda")
    heavy = torch.rand(k.shape, generator=g, device="cuda") < 0.125
    cache.k_cache[..., 0] = torch.where(heavy, 0.0, k)
    cache.v_cache.copy_(500 + 1000 * torch.rand(cache.v_cache.shape, generator=g, device="cuda"))
    cache.v_cache[heavy] = 0.0
    check_attention(q, cache, table, lengths, scale=math.log(2.0))


@gpu
def test_int8_values_of_very_different_size_for_f16_queries():
    """A value scale of 3e7 on a key that weighs nothing."""
    q, cache, table, lengths = batch(generator(22), torch.float16, True, 4, 2, 128, 16, [400, 90], poison=False)
    cache.v_scales.fill_(0.01)
    cache.v_scales[table[0, 3].long(), :, 5] = 3e7
    cache.k_scales.fill_(0.02)
    q = q.abs()
    cache.k_cache.copy_(cache.k_cache.abs())
    cache.k_cache[table[0, 3].long(), :, 5] = -127
    check_attention(q * 2, cache, table, lengths)


# ---- tracers -----------------------------------------------------------------------------
def fake_step():
    """Shapes of a step, for a fake mode."""
    q, k = (torch.empty(5, h, 128, dtype=torch.bfloat16, device="cuda") for h in (4, 2))
    cache = torch.empty(3, 2, 16, 128, dtype=torch.bfloat16, device="cuda")
    at, cos = torch.empty(5, dtype=torch.int64, device="cuda"), torch.empty(9, 64, device="cuda")
    return q, k, cache, at, cos, torch.empty(5, 3, dtype=torch.int32, device="cuda"), torch.empty(5, dtype=torch.int32, device="cuda")


def all_three(q, k, cache, at, cos, table, lengths):
    turned = kl.qk_norm_rope_write(q, k, k, None, None, cos, cos, at, at, cache, cache)
    return kl.paged_attention(turned, cache, cache, table, lengths), *kl.read_kv(cache, cache, at)


def test_functions_give_shapes_under_a_fake_mode():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        args = fake_step()
        out, k, v = all_three(*args)
    assert out.shape == (5, 4, 128) and k.shape == v.shape == (5, 2, 128) and out.dtype == torch.bfloat16
    out, k, v = all_three(*args)                                     # fake tensors after their mode
    assert out.shape == (5, 4, 128) and k.shape == v.shape == (5, 2, 128)


@pytest.mark.parametrize("mode", ["real", "symbolic"])
def test_functions_are_operators_in_a_traced_graph(mode):
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.fx.experimental.symbolic_shapes import ShapeEnv
    if mode == "real":                                               # traced as they are: tensors that are fake before
        with FakeTensorMode():
            graph = make_fx(all_three)(*fake_step())
    else:
        with FakeTensorMode(shape_env=ShapeEnv()):
            args = fake_step()
        graph = make_fx(all_three, tracing_mode="symbolic")(*args)
    names = [str(n.target) for n in graph.graph.nodes]
    for name in ("qk_norm_rope_write", "paged_attention", "read_kv"):
        assert sum(name in n for n in names) == 1


@gpu
@pytest.mark.parametrize("tracer", ["make_fx", "jit", "functionalize"])
def test_traced_calls_follow_their_inputs(tracer):
    from torch.fx.experimental.proxy_tensor import make_fx
    cases = [batch(generator(50 + i), torch.bfloat16, True, 4, 2, 128, 16, [700, 40, 9], poison=False) for i in range(2)]
    cos, sin = rope_tables(None, 128, 1000)

    def step(q, k, c, d, cs, ds, table, lengths, positions, slots):
        if tracer != "functionalize":                                # which takes no operator that writes to its arguments
            q = kl.qk_norm_rope_write(q, k, k * 2, None, None, cos, sin, positions, slots, c, d, cs, ds)
        out, lse = kl.paged_attention(q, c, d, table, lengths, cs, ds, return_lse=True)
        k, v = kl.read_kv(c, d, slots, cs, ds)
        return out, lse, k, v

    inputs = []
    for i, (q, cache, table, lengths) in enumerate(cases):
        k = torch.randn(3, 2, 128, generator=generator(60 + i), device="cuda").bfloat16()
        at = lengths.long() - 1
        inputs.append((q, k, *cache, table, lengths, at, kl.kv_slots(table, torch.arange(3, device="cuda"), at, 16)))

    def copies(args):
        return [t.clone() for t in args]

    refs = [step(*copies(args)) for args in inputs]
    if tracer == "functionalize":
        traced = make_fx(torch.func.functionalize(step))(*copies(inputs[0]))
    elif tracer == "make_fx":
        traced = make_fx(step)(*copies(inputs[0]))
    else:
        traced = torch.jit.trace(step, tuple(copies(inputs[0])), check_trace=False)
    for args, ref in zip(inputs, refs):
        got = traced(*copies(args))
        assert all(torch.equal(a, b) for a, b in zip(got, ref))


def test_a_traced_call_keeps_its_workspace():
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    with FakeTensorMode():
        q, _, cache, _, _, table, lengths = fake_step()
        space = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
        graph = make_fx(lambda q, space: kl.paged_attention(q, cache, cache, table, lengths, workspace=space))(q, space)
    call, = (n for n in graph.graph.nodes if "paged_attention" in str(n.target))
    given = [n for n in graph.graph.nodes if n.op == "placeholder"]
    assert given[1] in call.all_input_nodes


@gpu
def test_a_compiled_call_uses_its_workspace(monkeypatch):
    case = batch(generator(33), torch.bfloat16, False, 4, 2, 128, 16, [3000, 50], poison=False)
    space = torch.zeros(kl.paged_attention_workspace_bytes(2, 4, 2, 128), dtype=torch.uint8, device="cuda")
    ref, real, seen = attend(case), P._call, []

    def call(index, fn, *args):
        seen.append(N.PAGED_ATTENTION_ARGS.unpack(args[0])[WORKSPACE])
        real(index, fn, *args)

    compiled = torch.compile(lambda space: attend(case, workspace=space), backend="aot_eager", fullgraph=True)
    monkeypatch.setattr(P, "_call", call)
    assert torch.equal(compiled(space), ref) and seen == [space.data_ptr()]
    with pytest.raises(Exception, match="workspace"):
        compiled(space[:64])


# ---- positions and arguments ----------------------------------------------------------------
def test_kv_slots_of_positions_outside_the_table():
    """A position before the sequence or past its pages has no slot: negative, so not cached."""
    table = torch.tensor([[4, 2], [0, 9]], dtype=torch.int32)
    for kind in (torch.int32, torch.int64):
        rows, positions = torch.tensor([0, 0, 1, 1, 0, 1]), torch.tensor([-1, 17, -16, 32, 2 ** 30, 31], dtype=kind)
        slots = kl.kv_slots(table, rows, positions, 16)
        assert slots.dtype == torch.int64 and slots[[1, 5]].tolist() == [33, 9 * 16 + 15]
        assert (slots[[0, 2, 3, 4]] < 0).all()
    unused = torch.tensor([[7, -1]], dtype=torch.int32)              # a column that is not used yet
    assert (kl.kv_slots(unused, torch.zeros(16, dtype=torch.int64), torch.arange(16, 32), 16) < 0).all()
    none = torch.zeros(2, 0, dtype=torch.int32)
    assert (kl.kv_slots(none, torch.tensor([0, 1]), torch.tensor([0, 5]), 16) < 0).all()
    assert kl.kv_slots(none, torch.tensor([], dtype=torch.int64), torch.tensor([], dtype=torch.int64), 16).shape == (0,)


@gpu
def test_tensors_that_require_grad_are_refused():
    g = generator(70)
    q, k, v, qw, kw = step_inputs(g, torch.bfloat16, 3, 4, 2, 128, True, "fused")
    cos, sin = rope_tables(g, 128, 64)
    at = torch.arange(3, device="cuda")
    cache = kl.new_kv_cache(2, 16, 2, 128, torch.int8)
    table, lengths = torch.zeros(3, 1, dtype=torch.int32, device="cuda"), torch.ones(3, dtype=torch.int32, device="cuda")
    write = [q, k, v, qw, kw, cos, sin, at, at, *cache]
    attending = [q, cache.k_cache, cache.v_cache, table, lengths, cache.k_scales, cache.v_scales]
    reading = [cache.k_cache, cache.v_cache, at, cache.k_scales, cache.v_scales]
    for fn, args in ((kl.qk_norm_rope_write, write), (kl.paged_attention, attending), (kl.read_kv, reading)):
        for i, t in enumerate(args):
            if t.is_floating_point():
                learnt = list(args)
                learnt[i] = torch.nn.Parameter(t.clone()) if t is qw else t.clone().requires_grad_()
                with pytest.raises(ValueError, match="inference"):
                    fn(*learnt)
                with torch.no_grad():
                    fn(*learnt)
        fn(*args)


@gpu
def test_numbers_that_f32_does_not_hold_are_refused():
    q, cache, table, lengths = batch(generator(71), torch.bfloat16, False, 4, 2, 128, 16, [40], poison=False)
    for scale in (1e39, -1e300, 3.39e38):
        with pytest.raises(ValueError, match="scale"):
            attend((q, cache, table, lengths), scale=scale)
    qq, k, v, qw, kw = step_inputs(generator(72), torch.bfloat16, 1, 4, 2, 128, True, "fused")
    cos, sin = rope_tables(None, 128, 8)
    at = torch.zeros(1, dtype=torch.int64, device="cuda")
    for epsilon in (1e39, 1e-60, 3.39e38):
        with pytest.raises(ValueError, match="epsilon"):
            kl.qk_norm_rope_write(qq, k, v, qw, kw, cos, sin, at, at, *cache, epsilon=epsilon)


def other_torch(monkeypatch, *names):
    """``paged_kv`` as it loads where torch lacks ``names`` of ``torch._C``."""
    for name in names:
        monkeypatch.delattr(torch._C, name, raising=False)
    spec = importlib.util.spec_from_file_location(f"{kl.__name__}.paged_kv_other", ROOT / kl.__name__ / "paged_kv.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


HIDDEN = ("_cuda_getCurrentRawStream", "_cuda_getDevice", "_dynamo", "_len_torch_dispatch_stack", "_is_tracing", "_functorch")


@gpu
@pytest.mark.parametrize("name", HIDDEN)
def test_functions_without_torchs_private_names(monkeypatch, name):
    case = batch(generator(73), torch.bfloat16, False, 4, 2, 128, 16, [900, 5], poison=False)
    q, cache, table, lengths = case
    ref = attend(case)
    with monkeypatch.context() as m:
        module = other_torch(m, name)
    out = module.paged_attention(q, cache.k_cache, cache.v_cache, table, lengths)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = module.paged_attention(q, cache.k_cache, cache.v_cache, table, lengths)
    side.synchronize()
    assert torch.equal(out, ref) and torch.equal(again, ref)


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_a_value_that_is_not_finite_stays_in_its_element(dtype):
    case = batch(generator(74), TYPES[dtype], False, 4, 2, 128, 16, [700, 90], poison=False)
    q, cache, table, lengths = case
    before = attend(case)
    for value in (torch.inf, -torch.inf, torch.nan):
        cache.v_cache[table[0, 2].long(), 1, 5, 7] = value
        after = attend(case)
        hit = torch.zeros_like(before, dtype=torch.bool)
        hit[0, 2:, 7] = True
        assert not torch.isfinite(after[hit]).any() and torch.equal(after[~hit], before[~hit])


# ---- rows that are not split ---------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype,quantized", [("bf16", False), ("f16", False), ("bf16", True), ("f16", True)])
@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 2, 128), (32, 2, 128), (40, 1, 128), (16, 1, 64), (17, 1, 64), (12, 1, 256), (24, 2, 256)])
def test_whole_rows_of_many_heads(dtype, quantized, heads, kv_heads, dim):
    """Short rows and rows that are many are not split, with 8 and 16 heads per block and several blocks per row too."""
    short = [n for n in LENGTHS if n <= 200]
    check_attention(*batch(generator(heads + dim), TYPES[dtype], quantized, heads, kv_heads, dim, 16, short))
    many = [(i * 41) % 500 if i % 7 else 0 for i in range(900 // kv_heads)] + [500]
    check_attention(*batch(generator(heads), TYPES[dtype], quantized, heads, kv_heads, dim, 16, many))
