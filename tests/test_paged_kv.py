"""The paged key-value cache: ``qk_norm_rope_write``, ``read_kv`` and
``paged_attention`` against their formulas in 64 bits.

Tolerances, derived from the arithmetic:

* ``U`` is the unit roundoff of the 16-bit type (8 and 11 significant bits): every 16-bit result is rounded once (``U * |ref|``).
* Norm and rotation are f32: three products and sums on values that are at most the row's largest magnitude, and a mean
  of up to 256 squares: within ``2^-20`` of that magnitude.
* Attention: scores are f32 dot products of ``head_dim`` terms, so a score is off by at most ``2^-21`` of the sum of its terms'
  magnitudes (``reach``), and so is the log of its weight; weights carry 16 bits or more into the products with the values
  (``2^-16``).  The result is off by that share of ``sum_j p_j |v_j|``.
"""
import numpy as np
import pytest
import torch

from tests.conftest import load_kl

kl = load_kl()
N = kl._native
gpu = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SMALL = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}     # half the step of the subnormals


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def close(actual, ref, dtype, extra):
    """Within one rounding to ``dtype`` of ``ref`` give or take ``extra`` (a tensor or a number)."""
    off = (actual.double() - ref).abs()
    allowed = U[dtype] * ref.abs() + SMALL[dtype] + 1.01 * extra
    assert off.shape == ref.shape and not torch.isnan(actual).any()
    worst = (off - allowed).max().item() if off.numel() else 0.0
    assert worst <= 0, f"over tolerance by {worst:.3g}"


def make_cache(g, dtype, quantized, pages, kv_heads, page, dim, order="heads"):
    """Random contents; ``order`` "tokens" lays the pages out [page, token, head, element]."""
    shape = (pages, page, kv_heads, dim) if order == "tokens" else (pages, kv_heads, page, dim)
    if quantized:
        k, v = (torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8) for _ in range(2))
        s = [torch.rand(shape[:3], generator=g, device="cuda") * 0.02 + 0.002 for _ in range(2)]
    else:
        k, v = (torch.randn(shape, generator=g, device="cuda").to(dtype) for _ in range(2))
        s = [None, None]
    if order == "tokens":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
        s = [None if t is None else t.transpose(1, 2) for t in s]
    return kl.KVCache(k, v, *s)


def dense(cache, row, length, what):
    """Keys (0) or values (1) of one sequence in 64 bits: [kv_heads, length, dim]."""
    page = cache.k_cache.shape[2]
    ids = row[:-(-length // page)].long()
    x = cache[what][ids].double()
    if cache[2 + what] is not None:
        x = x * cache[2 + what][ids].double()[..., None]
    return x.permute(1, 0, 2, 3).flatten(1, 2)[:, :length]


def attention(q, cache, table, lengths, scale=None):
    """out, lse, and what both may be off by, in 64 bits."""
    group, dim = q.shape[1] // cache.k_cache.shape[1], q.shape[2]
    scale = dim ** -0.5 if scale is None else scale
    out, lse = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.full(q.shape[:2], -torch.inf, dtype=torch.float64, device=q.device)
    spread, reach = torch.zeros_like(out), torch.zeros_like(lse)
    for b, n in enumerate(lengths.tolist()):
        if n <= 0:
            continue
        k, v = (dense(cache, table[b], n, i).repeat_interleave(group, 0) for i in (0, 1))
        s = torch.einsum("hd,hld->hl", q[b].double(), k) * scale
        p = torch.softmax(s, -1)
        out[b], lse[b] = torch.einsum("hl,hld->hd", p, v), torch.logsumexp(s, -1)
        spread[b] = torch.einsum("hl,hld->hd", p, v.abs())
        reach[b] = (torch.einsum("hd,hld->hl", q[b].double().abs(), k.abs()) * abs(scale)).max(-1).values
    share = 2.0 ** -16 + 2.0 ** -21 * reach
    return out, lse, spread * share[..., None], 2.0 ** -20 * (1 + lse.abs().clamp(max=1e9)) + 2.0 ** -21 * reach


def batch(g, dtype, quantized, heads, kv_heads, dim, page, lengths, order="heads", spare=2, poison=True):
    """q, cache, page table and lengths of a batch whose unused slots hold what must not be used."""
    counts = [-(-max(n, 0) // page) for n in lengths]
    pages = sum(counts) + spare
    cache = make_cache(g, dtype, quantized, pages, kv_heads, page, dim, order)
    ids = torch.randperm(pages, generator=g, device="cuda").int()
    columns = max(counts + [1])
    table = torch.full((len(lengths), columns + 3), -7, dtype=torch.int32, device="cuda")[:, :columns]
    used = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
    at = 0
    for b, (n, c) in enumerate(zip(lengths, counts)):
        table[b, :c] = ids[at:at + c]
        for i in range(c):
            used[table[b, i], :max(0, min(page, n - i * page))] = True
        at += c
    if poison:
        for t in ([cache.k_scales, cache.v_scales] if quantized else [cache.k_cache, cache.v_cache]):
            where = ~used[:, None, :].expand(pages, kv_heads, page)
            t[where] = torch.nan
    q = torch.randn(len(lengths), heads, dim, generator=g, device="cuda").to(dtype)
    return q, cache, table, torch.tensor(lengths, dtype=torch.int32, device="cuda")


def check_attention(q, cache, table, lengths, scale=None):
    out, lse = kl.paged_attention(q, cache.k_cache, cache.v_cache, table, lengths, cache.k_scales, cache.v_scales, scale=scale,
                                  return_lse=True)
    ref, ref_lse, extra, extra_lse = attention(q, cache, table, lengths, scale)
    close(out, ref, q.dtype, extra)
    empty = torch.isinf(ref_lse)
    assert torch.equal(empty, torch.isinf(lse)) and (lse[empty] < 0).all()
    assert ((lse.double() - ref_lse).abs()[~empty] <= extra_lse[~empty]).all()
    assert (out[empty] == 0).all()
    assert N.device_status(0) == N.KL_OK
    return out


LENGTHS = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 200, 511, 1000, 4097]


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 8, 128), (8, 8, 64), (6, 2, 128), (4, 1, 256), (32, 2, 128), (17, 1, 64), (40, 1, 128), (12, 1, 256)])
def test_attention_over_ragged_lengths(dtype, quantized, heads, kv_heads, dim):
    check_attention(*batch(generator(heads + dim), TYPES[dtype], quantized, heads, kv_heads, dim, 16, LENGTHS))


@gpu
@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 32, 100, 128, 5000])
def test_attention_over_page_sizes(quantized, page):
    check_attention(*batch(generator(page), torch.bfloat16, quantized, 4, 2, 128, page, [5, 0, 16, 129, 1025, 77]))


@gpu
@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("lengths", [[1], [37], [64], [65], [20000], [0], [0, 0, 0], [3000] * 3, [1] * 700, [0, 16000] + [5] * 300, [5, 300] * 300 + [3000]])
def test_attention_of_few_and_many_sequences(quantized, lengths):
    check_attention(*batch(generator(len(lengths)), torch.bfloat16, quantized, 6, 2, 128, 16, lengths))


@gpu
@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("longest", [250, 990])
def test_attention_of_many_rows(quantized, longest):
    """More rows than two waves of CTAs, of very different lengths, some empty."""
    lengths = [(i * i * 37) % (longest + 1) if i % 9 else 0 for i in range(130)] + [longest]
    check_attention(*batch(generator(longest), torch.bfloat16, quantized, 16, 8, 64, 16, lengths))


@gpu
@pytest.mark.parametrize("quantized", [False, True])
def test_attention_strides(quantized):
    """A cache laid out by token, queries inside a fused row, a table inside a wider one."""
    g = generator(3)
    q, cache, table, lengths = batch(g, torch.bfloat16, quantized, 16, 8, 128, 16, [300, 17, 0, 1200], order="tokens")
    fused = torch.randn(4, 32 * 128, generator=g, device="cuda").bfloat16()
    check_attention(fused[:, :2048].view(4, 16, 128), cache, table, lengths)
    check_attention(fused.view(4, 32, 128)[:, 1::2], cache, table, lengths)
    odd = torch.randn(4, 16 * 128 + 1, generator=g, device="cuda").bfloat16()[:, 1:].view(4, 16, 128)
    assert odd.data_ptr() % 16
    check_attention(odd, cache, table, lengths)


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("quantized", [False, True])
def test_attention_of_peaked_scores(dtype, quantized):
    """Large scores whose maximum moves along the row, and weights that underflow."""
    q, cache, table, lengths = batch(generator(9), TYPES[dtype], quantized, 4, 2, 128, 16, [700, 70, 3], poison=False)
    check_attention(q * 16, cache, table, lengths)
    check_attention(q, cache, table, lengths, scale=-3.0)
    check_attention(q, cache, table, lengths, scale=0.0)


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_attention_int8_scales_of_very_different_size(dtype):
    """Values whose scales differ by many powers of two: large ones with no weight, small ones with all of it."""
    g = generator(21)
    q, cache, table, lengths = batch(g, TYPES[dtype], True, 4, 2, 128, 16, [400, 90], poison=False)
    cache.v_scales.mul_(torch.exp2(torch.randint(-24, 3, cache.v_scales.shape, generator=g, device="cuda").float()))
    check_attention(q * 4, cache, table, lengths)
    cache.v_scales.fill_(0.01)
    cache.v_scales[table[0, 3].long(), :, 5] = 3e7           # its key is made to weigh nothing
    cache.k_cache[table[0, 3].long(), :, 5] = 0
    cache.k_scales[:] = 0.02
    q = q.abs()
    cache.k_cache[:] = cache.k_cache.abs()
    cache.k_cache[table[0, 3].long(), :, 5] = -127
    if dtype == "bf16":
        check_attention(q * 2, cache, table, lengths)


@gpu
def test_attention_of_infinite_and_nan_inputs():
    """A key of -inf scores has weight 0; a NaN in a used key reaches its own sequence and heads only."""
    q, cache, table, lengths = batch(generator(4), torch.bfloat16, False, 4, 2, 64, 16, [100, 100, 40], poison=False)
    args = (cache.k_cache, cache.v_cache, table, lengths)
    before = kl.paged_attention(q, *args)
    cache.k_cache[table[1, 2].long(), 1, 3, 7] = torch.nan
    after = kl.paged_attention(q, *args)
    assert torch.isnan(after[1, 2:]).all() and torch.equal(after[1, :2], before[1, :2])
    assert torch.equal(after[0], before[0]) and torch.equal(after[2], before[2])
    cache.k_cache[table[1, 2].long(), 1, 3, 7] = 0.0
    q[1, 2:] = q[1, 2:].abs()
    cache.k_cache[table[1, 0].long(), 1, 0] = -torch.inf
    out, lse = kl.paged_attention(q, *args, return_lse=True)
    cache.k_cache[table[1, 0].long(), 1, 0] = 0
    k, v = dense(cache, table[1], 100, 0), dense(cache, table[1], 100, 1)
    s = torch.einsum("hd,hld->hl", q[1, 2:].double(), k[1:].repeat(2, 1, 1)) * 64 ** -0.5
    s[:, 0] = -torch.inf
    ref = torch.softmax(s, -1) @ v[1]
    close(out[1, 2:], ref, torch.bfloat16, torch.softmax(s, -1) @ v[1].abs() * 2.0 ** -14)


@gpu
def test_attention_is_deterministic_and_joins_by_lse():
    q, cache, table, lengths = batch(generator(6), torch.bfloat16, False, 16, 8, 128, 16, [9000, 40, 2500], poison=False)
    args = (cache.k_cache, cache.v_cache)
    out, lse = kl.paged_attention(q, *args, table, lengths, return_lse=True)
    for _ in range(5):
        again = kl.paged_attention(q, *args, table, lengths, return_lse=True)
        assert torch.equal(again[0], out) and torch.equal(again[1], lse)
    cut = torch.tensor([64 * 16, 0, 16], dtype=torch.int32, device="cuda")
    rest = torch.stack([torch.nn.functional.pad(table[b, c // 16:], (0, c // 16)) for b, c in enumerate(cut.tolist())]).contiguous()
    o1, l1 = kl.paged_attention(q, *args, table, cut, return_lse=True)
    o2, l2 = kl.paged_attention(q, *args, rest, lengths - cut, return_lse=True)
    w1, w2 = torch.exp(l1.double() - lse)[..., None], torch.exp(l2.double() - lse)[..., None]
    close(out, o1.double() * w1 + o2.double() * w2, torch.bfloat16, 2.0 ** -8 * (o1.double().abs() * w1 + o2.double().abs() * w2)
          + 2.0 ** -13)


@gpu
def test_attention_on_another_stream_and_in_a_graph():
    q, cache, table, lengths = batch(generator(8), torch.bfloat16, True, 16, 8, 128, 16, [5000, 33], poison=False)
    args = (q, cache.k_cache, cache.v_cache, table, lengths, cache.k_scales, cache.v_scales)
    ref = kl.paged_attention(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [kl.paged_attention(*args) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(o, ref) for o in outs)
    space = torch.zeros(max(16, kl.paged_attention_workspace_bytes(2, 16, 8, 128)), dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kl.paged_attention(*args, workspace=space)
    for n in ((5000, 33), (1, 2), (0, 48)):
        lengths.copy_(torch.tensor(n, dtype=torch.int32))
        graph.replay()
        assert torch.equal(out, kl.paged_attention(*args))


@gpu
def test_captured_behind_copies_and_memsets():
    """In a graph every launch waits for what comes before it, copies and memsets too, and for the operators among each other."""
    q, cache, table, lengths = batch(generator(18), torch.bfloat16, False, 4, 2, 128, 16, [2000, 33], poison=False)
    k, v = (torch.randn(2, 2, 128, generator=generator(19), device="cuda").bfloat16() for _ in range(2))
    cos, sin = rope_tables(None, 128, cache.k_cache.shape[0] * 16)
    lens, slots, new = torch.zeros_like(lengths), torch.zeros(2, dtype=torch.int64, device="cuda"), torch.zeros_like(v)
    space = torch.zeros(kl.paged_attention_workspace_bytes(2, 4, 2, 128), dtype=torch.uint8, device="cuda")
    wanted = kl.kv_slots(table, torch.arange(2, device="cuda"), lengths.long() - 1, 16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        slots.copy_(wanted)
        new.zero_()
        lens.copy_(lengths)
        turned = kl.qk_norm_rope_write(q, k, new, None, None, cos, sin, slots, slots, *cache)
        first = kl.paged_attention(turned, cache.k_cache, cache.v_cache, table, lens, workspace=space)
        new.copy_(v)
        turned = kl.qk_norm_rope_write(q, k, new, None, None, cos, sin, slots, slots, *cache)
        second = kl.paged_attention(turned, cache.k_cache, cache.v_cache, table, lens, workspace=space)
        got = kl.read_kv(cache.k_cache, cache.v_cache, slots)[1]
    for _ in range(20):
        lens.zero_()
        slots.fill_(1)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, v)
        ref = kl.qk_norm_rope_write(q, k, torch.zeros_like(v), None, None, cos, sin, slots, slots, *cache)
        assert torch.equal(first, kl.paged_attention(ref, cache.k_cache, cache.v_cache, table, lengths))
        kl.qk_norm_rope_write(q, k, v, None, None, cos, sin, slots, slots, *cache)
        assert torch.equal(second, kl.paged_attention(ref, cache.k_cache, cache.v_cache, table, lengths))


@gpu
def test_attention_out_of_range_table_is_recorded_not_read():
    q, cache, table, lengths = batch(generator(5), torch.bfloat16, False, 4, 2, 128, 16, [40, 40, 40], poison=False)
    ref = kl.paged_attention(q, cache.k_cache, cache.v_cache, table, lengths)
    assert N.device_status(0, reset=True) == N.KL_OK
    bad = table.clone()
    bad[1, 1] = cache.k_cache.shape[0]
    bad[1, 2] = -1
    out = kl.paged_attention(q, cache.k_cache, cache.v_cache, bad, lengths)
    assert N.device_status(0, reset=True) == N.KL_ERR_INVALID
    assert torch.equal(out[0], ref[0]) and torch.equal(out[2], ref[2])
    only = kl.paged_attention(q, cache.k_cache, cache.v_cache, table, torch.tensor([40, 16, 40], dtype=torch.int32, device="cuda"))
    close(out[1], only[1].double(), torch.bfloat16, 2.0 ** -7)
    long = torch.tensor([40, 49, 40], dtype=torch.int32, device="cuda")
    cut = torch.tensor([40, 48, 40], dtype=torch.int32, device="cuda")
    over = kl.paged_attention(q, cache.k_cache, cache.v_cache, table, long)
    assert N.device_status(0, reset=True) == N.KL_ERR_INVALID
    assert torch.equal(over, kl.paged_attention(q, cache.k_cache, cache.v_cache, table, cut))
    assert N.device_status(0, reset=True) == N.KL_OK


@gpu
@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("page", [16, 24])
def test_attention_bad_pages_of_a_long_row_are_absent(quantized, page):
    """Pages out of range here and there: as if the sequence consisted of the other pages."""
    q, cache, table, _ = batch(generator(page), torch.bfloat16, quantized, 4, 2, 128, page, [page * 90, page * 7], poison=False)
    lengths = torch.tensor([page * 90, page * 7], dtype=torch.int32, device="cuda")
    gone = [3, 20, 21, 22, 23, 24, 25, 26, 27, 28, 50, 89]
    bad = table.clone()
    bad[0, gone] = torch.tensor([-1, 2 ** 30, cache.k_cache.shape[0]] * 4, dtype=torch.int32, device="cuda")
    out = kl.paged_attention(q, cache.k_cache, cache.v_cache, bad, lengths, cache.k_scales, cache.v_scales)
    assert N.device_status(0, reset=True) == N.KL_ERR_INVALID
    kept = [i for i in range(90) if i not in gone]
    short = table[:, :len(kept)].clone()
    short[0] = table[0, kept]
    ref, _, extra, _ = attention(q, cache, short, torch.tensor([page * len(kept), page * 7], dtype=torch.int32, device="cuda"))
    close(out, ref, torch.bfloat16, extra)


# ---- write and read -----------------------------------------------------------------
def rope_tables(g, dim, positions=5000):
    turn = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * 1e6 ** (
        -torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim)
    return turn.cos().float(), turn.sin().float()


def norm_rope(x, weight, cos, sin, eps=1e-6):
    y = x.double()
    if weight is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    c, s = cos.double()[:, None], sin.double()[:, None]
    a, b = y.chunk(2, -1)
    return torch.cat((a * c - b * s, b * c + a * s), -1)


def step_inputs(g, dtype, tokens, heads, kv_heads, dim, norm, layout):
    n = (heads + 2 * kv_heads) * dim
    if layout == "fused":
        rows = torch.randn(tokens, n, generator=g, device="cuda").to(dtype)
    elif layout == "odd":                                            # rows that are not 16-byte aligned
        rows = torch.randn(tokens, n + 3, generator=g, device="cuda").to(dtype)[:, 1:n + 1]
    else:
        rows = None
    if rows is None:                                                 # separate tensors, heads before tokens
        q, k, v = (torch.randn(h, tokens, dim, generator=g, device="cuda").to(dtype).transpose(0, 1) for h in (heads, kv_heads, kv_heads))
    else:
        q, k, v = (t.unflatten(1, (-1, dim)) for t in rows.split([heads * dim, kv_heads * dim, kv_heads * dim], 1))
    w = [(1 + 0.3 * torch.randn(dim, generator=g, device="cuda")).to(dtype) for _ in range(2)] if norm else [None, None]
    return q, k, v, *w


def check_write(seed, dtype, quantized, tokens, heads, kv_heads, dim, page, norm=True, layout="fused", order="heads"):
    g = generator(seed)
    q, k, v, qw, kw = step_inputs(g, dtype, tokens, heads, kv_heads, dim, norm, layout)
    cache = make_cache(g, dtype, quantized, tokens // page + 3, kv_heads, page, dim, order)
    slots = torch.randperm(cache.k_cache.shape[0] * page, generator=g, device="cuda")[:tokens]
    skip = torch.rand(tokens, generator=g, device="cuda") < 0.2
    slots = torch.where(skip, -1 - slots, slots)
    cos, sin = rope_tables(g, dim)
    positions = torch.randint(0, 5000, (tokens,), generator=g, device="cuda")
    old = [None if t is None else t.clone() for t in cache]
    out = kl.qk_norm_rope_write(q, k, v, qw, kw, cos, sin, positions, slots, *cache)
    assert N.device_status(0) == N.KL_OK
    ref_q, ref_k = (norm_rope(x, w, cos[positions], sin[positions]) for x, w in ((q, qw), (k, kw)))
    close(out, ref_q, dtype, 2.0 ** -20 * ref_q.abs().amax(-1, keepdim=True))
    kept = ~skip
    where, off = slots[kept] // page, slots[kept] % page
    extra = 2.0 ** -20 * ref_k.abs().amax(-1, keepdim=True)[kept]
    if quantized:
        scale = cache.k_scales[where, :, off].double()
        want = ref_k[kept].abs().amax(-1) / 127
        assert ((scale - want).abs() <= 2.0 ** -19 * want).all()
        off_by = (cache.k_cache[where, :, off].double() * scale[..., None] - ref_k[kept]).abs()
        assert (off_by <= scale[..., None] * 0.5 + 256 * extra).all()
        x = v[kept].float()                                          # untouched by norm and rotation: equal to the last bit
        s = x.abs().amax(-1) / torch.tensor(127.0, device="cuda")
        s = torch.where(s == 0, 1.0, s)
        assert torch.equal(cache.v_scales[where, :, off], s)
        assert torch.equal(cache.v_cache[where, :, off], torch.round(x / s[..., None]).clamp(-127, 127).to(torch.int8))
    else:
        close(cache.k_cache[where, :, off], ref_k[kept], dtype, extra)
        assert torch.equal(cache.v_cache[where, :, off], v[kept])
    untouched = torch.ones(cache.k_cache.shape[0], page, dtype=torch.bool, device="cuda")
    untouched[where, off] = False
    for now, then in zip(cache, old):
        if now is not None:
            assert torch.equal(now.transpose(1, 2)[untouched], then.transpose(1, 2)[untouched])
    got_k, got_v = kl.read_kv(cache.k_cache, cache.v_cache, slots, cache.k_scales, cache.v_scales, dtype=dtype)
    for got, codes, scales in ((got_k, cache.k_cache, cache.k_scales), (got_v, cache.v_cache, cache.v_scales)):
        x = codes[where, :, off]
        if quantized:
            x = (x.float() * scales[where, :, off, None]).to(dtype)
        assert torch.equal(got[kept], x) and (got[skip] == 0).all()


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 8, 128), (8, 8, 64), (5, 1, 128), (4, 2, 256)])
@pytest.mark.parametrize("tokens", [1, 3, 130])
def test_write_and_read(dtype, quantized, heads, kv_heads, dim, tokens):
    check_write(tokens + dim, TYPES[dtype], quantized, tokens, heads, kv_heads, dim, 16)


@gpu
@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("layout,order,page,norm", [("odd", "heads", 16, True), ("separate", "tokens", 1, True), ("fused", "tokens", 24, False),
                                                   ("odd", "tokens", 7, False)])
def test_write_and_read_layouts(quantized, layout, order, page, norm):
    for dim in (64, 128, 256):
        check_write(dim + page, torch.bfloat16, quantized, 77, 6, 3, dim, page, norm, layout, order)


@gpu
def test_write_of_zero_and_tiny_and_unbounded_rows():
    """All-zero rows get scale 1 and zeros; a NaN or an infinity makes its own row NaN and no other."""
    g = generator(1)
    q, k, v, _, _ = step_inputs(g, torch.bfloat16, 6, 2, 2, 64, False, "fused")
    k[0] = 0
    v[0] = 0
    v[1] = 1e-40
    v[2, 0, 5] = torch.nan
    v[3, 1, 6] = torch.inf
    k[4, 1, 0] = -torch.inf
    v[5] = 3e38
    cos, sin = torch.ones(8, 32, device="cuda"), torch.zeros(8, 32, device="cuda")
    cache = kl.new_kv_cache(2, 16, 2, 64, torch.int8)
    slots = torch.arange(6, device="cuda")
    kl.qk_norm_rope_write(q, k, v, None, None, cos, sin, slots, slots, *cache)
    rk, rv = kl.read_kv(cache.k_cache, cache.v_cache, slots, cache.k_scales, cache.v_scales)
    assert (rk[0] == 0).all() and (rv[0] == 0).all() and (cache.v_scales[0, :, 0] == 1).all()
    assert torch.isnan(rv[2, 0]).all() and torch.isnan(rv[3, 1]).all() and torch.isnan(rk[4, 1]).all()
    for clean in (rv[2, 1], rv[3, 0], rk[4, 0], rv[1], rv[5], rk[5]):
        assert torch.isfinite(clean).all()
    assert torch.equal(rv[5], v[5])


@gpu
def test_write_and_read_out_of_range_is_recorded_not_done():
    g = generator(2)
    q, k, v, qw, kw = step_inputs(g, torch.bfloat16, 4, 4, 2, 128, True, "fused")
    cos, sin = rope_tables(g, 128, 64)
    cache = kl.new_kv_cache(2, 16, 2, 128)
    at = torch.arange(4, device="cuda")
    assert N.device_status(0, reset=True) == N.KL_OK
    kl.qk_norm_rope_write(q, k, v, qw, kw, cos, sin, at, torch.tensor([0, 1, 32, 2 ** 40], device="cuda"), *cache)
    assert N.device_status(0, reset=True) == N.KL_ERR_INVALID
    assert (cache.v_cache[0, :, 2:] == 0).all() and (cache.v_cache[1] == 0).all() and torch.equal(cache.v_cache[0, :, 1], v[1])
    kl.qk_norm_rope_write(q, k, v, qw, kw, cos, sin, torch.tensor([0, 64, -1, 63], device="cuda"), at, *cache)
    assert N.device_status(0, reset=True) == N.KL_ERR_INVALID
    rk, rv = kl.read_kv(cache.k_cache, cache.v_cache, torch.tensor([0, 32, -5, 1], device="cuda"))
    assert N.device_status(0, reset=True) == N.KL_ERR_INVALID
    assert torch.equal(rv[0], v[0]) and torch.equal(rv[3], v[1]) and (rv[1:3] == 0).all() and (rk[1:3] == 0).all()


@gpu
@pytest.mark.parametrize("quantized", [False, True])
def test_offsets_past_32_bits(quantized):
    """A cache of more than 2^31 elements (2^32 bytes), written, read and attended to at its far end."""
    dtype = torch.int8 if quantized else torch.bfloat16
    pages, page, kv_heads, dim = 8200, 256, 8, 128
    k, v = (torch.empty(pages, kv_heads, page, dim, dtype=dtype, device="cuda") for _ in range(2))
    assert k.numel() > 2 ** 31
    scales = [torch.ones(pages, kv_heads, page, device="cuda") for _ in range(2)] if quantized else [None, None]
    cache = kl.KVCache(k, v, *scales)
    g = generator(12)
    n = 300
    q, kk, vv, qw, kw = step_inputs(g, torch.bfloat16, n, 16, 8, 128, True, "fused")
    cos, sin = rope_tables(g, 128, 512)
    table = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32, device="cuda")
    at = torch.arange(n, device="cuda")
    slots = kl.kv_slots(table, torch.zeros_like(at), at, page)
    out = kl.qk_norm_rope_write(q, kk, vv, qw, kw, cos, sin, at, slots, *cache)
    ref = norm_rope(kk, kw, cos[at], sin[at])
    rk, rv = kl.read_kv(cache.k_cache, cache.v_cache, slots, *scales)
    step = ref.abs().amax(-1, keepdim=True) / 127 if quantized else 0.0
    close(rk, ref, torch.bfloat16, 0.51 * step + 2.0 ** -8 * step + 1e-5)
    check_attention(out[-1:], cache, table, torch.tensor([n], dtype=torch.int32, device="cuda"))


@gpu
def test_empty_calls():
    cache = kl.new_kv_cache(2, 16, 2, 64)
    z = torch.zeros(0, device="cuda", dtype=torch.int64)
    q, k = (torch.empty(0, h, 64, device="cuda", dtype=torch.bfloat16) for h in (4, 2))
    cos = torch.zeros(4, 32, device="cuda")
    assert kl.qk_norm_rope_write(q, k, k, None, None, cos, cos, z, z, *cache).shape == (0, 4, 64)
    assert kl.read_kv(cache.k_cache, cache.v_cache, z)[0].shape == (0, 2, 64)
    out = kl.paged_attention(q, cache.k_cache, cache.v_cache, torch.zeros(0, 3, dtype=torch.int32, device="cuda"), z.int())
    assert out.shape == (0, 4, 64)
    none = kl.paged_attention(torch.ones(2, 4, 64, device="cuda", dtype=torch.bfloat16), cache.k_cache, cache.v_cache,
                              torch.zeros(2, 0, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"))
    assert (none == 0).all()


# ---- refusals --------------------------------------------------------------------------
@gpu
def test_argument_errors():
    dev = "cuda"
    cache = kl.new_kv_cache(4, 16, 2, 128)
    eight = kl.new_kv_cache(4, 16, 2, 128, torch.int8)
    q = torch.zeros(3, 4, 128, device=dev, dtype=torch.bfloat16)
    k = torch.zeros(3, 2, 128, device=dev, dtype=torch.bfloat16)
    table, lengths = torch.zeros(3, 4, dtype=torch.int32, device=dev), torch.ones(3, dtype=torch.int32, device=dev)
    cos, at, w = torch.ones(8, 64, device=dev), torch.arange(3, device=dev), torch.ones(128, device=dev, dtype=torch.bfloat16)

    def refused(match, fn, *args, **kw):
        with pytest.raises(ValueError, match=match):
            fn(*args, **kw)

    attend, write, read = kl.paged_attention, kl.qk_norm_rope_write, kl.read_kv
    refused("batch, heads", attend, q[0], *cache[:2], table, lengths)
    refused("FP16/BF16", attend, q.float(), *cache[:2], table, lengths)
    refused("CUDA", attend, q.cpu(), *cache[:2], table, lengths)
    refused("contiguous head", attend, q.transpose(1, 2).contiguous().transpose(1, 2), *cache[:2], table, lengths)
    refused("multiple", attend, q[:, :3], *cache[:2], table, lengths)
    refused("head_dim", attend, q[..., :64], *cache[:2], table, lengths)
    refused("page_table", attend, q, *cache[:2], table.long(), lengths)
    refused("page_table", attend, q, *cache[:2], table[:2], lengths)
    refused("contiguous rows", attend, q, *cache[:2], table[:, ::2], lengths)
    refused("lengths", attend, q, *cache[:2], table, lengths.long())
    refused("lengths", attend, q, *cache[:2], table, lengths[:2])
    refused("finite", attend, q, *cache[:2], table, lengths, scale=float("nan"))
    refused("needs k_scales", attend, q, *eight[:2], table, lengths)
    refused("only an int8", attend, q, *cache[:2], table, lengths, k_scales=eight.k_scales)
    refused("activations", attend, q.half(), *cache[:2], table, lengths)
    refused("scales must be", attend, q, *eight[:2], table, lengths, k_scales=eight.k_scales[:2], v_scales=eight.v_scales)
    refused("FP32", attend, q, *eight[:2], table, lengths, k_scales=eight.k_scales.half(), v_scales=eight.v_scales)
    refused("page_size, head_dim", attend, q, cache.k_cache, cache.v_cache[:2], table, lengths)
    refused("equal strides", attend, q, cache.k_cache, cache.v_cache.transpose(1, 2).contiguous().transpose(1, 2), table, lengths)
    refused("workspace", attend, q, *cache[:2], table, lengths, workspace=torch.zeros(16, dtype=torch.uint8))
    refused("inference", attend, q.clone().requires_grad_(), *cache[:2], table, lengths)
    refused("head_dim must be", kl.new_kv_cache, 2, 16, 2, 96)
    refused("holds", kl.new_kv_cache, 2, 16, 2, 128, torch.float32)
    refused("positive", kl.new_kv_cache, 0, 16, 2, 128)

    good = (q, k, k, w, w, cos, cos, at, at)
    for i, bad, match in ((0, q[:2], "tokens"), (0, q.float(), "dtype"), (1, k.half(), "dtype"), (2, k[:, :1], "tokens"),
                          (3, None, "together"), (3, w[:64], "q_weight"), (4, w.float(), "k_weight"), (5, cos[:, :32], "cos and sin"),
                          (6, cos.double(), "FP32"), (7, at.int(), "positions"), (8, at[:2], "slots"), (8, at.cpu(), "slots"),
                          (0, q.clone().requires_grad_(), "inference")):
        args = list(good)
        args[i] = bad
        refused(match, write, *args, *cache)
    refused("epsilon", write, *good, *cache, epsilon=0.0)
    refused("match the cache", write, q, k[:, :1], k[:, :1], w, w, cos, cos, at, at, *cache)
    refused("slots", read, *cache[:2], at.int())
    refused("FP16/BF16", read, *cache[:2], at, dtype=torch.float32)
    refused("activations", read, *cache[:2], at, dtype=torch.float16)
    # 16-byte alignment of the cache's rows is checked by the library
    odd = torch.zeros(4 * 2 * 16 * 128 + 8, device=dev, dtype=torch.bfloat16)[1:1 + 4 * 2 * 16 * 128].view(4, 2, 16, 128)
    with pytest.raises(N.NativeError, match="16-byte"):
        attend(q, odd, odd, table, lengths)


def test_c_abi_rejects_bad_arguments_without_a_gpu():
    lib = N.lib()
    fake = 256

    def cache(k=fake, v=fake, ks=0, vs=0, strides=(4096, 2048, 128), fmt=N.KL_KV_SAME, pages=2, page=16, heads=2, dim=128):
        return N.KV_CACHE.pack(k, v, ks, vs, *strides, 32, 16, 1, fmt, pages, page, heads, dim)

    def attend(c=None, q=fake, dtype=N.KL_DT_BF16, batch=1, heads=4, columns=2, lengths=fake, scale=1.0, out=fake, table=fake):
        args = N.PAGED_ATTENTION_ARGS.pack(q or 0, table or 0, lengths or 0, out or 0, 0, 0, 0, 512, 128, 2, c or cache(), dtype, batch,
                                           heads, columns, scale)
        return lib.kl_paged_attention(args, None)

    bad = N.KL_ERR_INVALID
    assert lib.kl_read_kv(None, N.KL_DT_BF16, fake, 1, fake, fake, None) == bad
    assert lib.kl_paged_attention(None, None) == bad and lib.kl_qk_norm_rope_write(None, None) == bad
    for c in (cache(k=0), cache(k=8), cache(strides=(4096, 2048, 132)), cache(fmt=2), cache(fmt=N.KL_KV_INT8), cache(pages=0),
              cache(page=0), cache(heads=0), cache(dim=96)):
        assert attend(c) == bad and lib.kl_read_kv(c, N.KL_DT_BF16, fake, 1, fake, fake, None) == bad
    assert b"head_dim" in lib.kl_last_error()
    assert attend(dtype=N.KL_DT_F32) == bad and attend(heads=3) == bad and attend(batch=-1) == bad and attend(columns=-1) == bad
    assert attend(scale=float("inf")) == bad and attend(scale=float("nan")) == bad
    assert attend(q=None) == bad and attend(out=None) == bad and attend(lengths=None) == bad and attend(table=None) == bad
    assert attend(out=fake + 4) == bad and attend(columns=1 << 28) == bad
    assert attend(batch=0) == N.KL_OK

    def write(c=None, tokens=1, heads=4, qw=fake, kw=fake, rows=8, eps=1e-6, q=fake, slots=fake, dtype=N.KL_DT_BF16):
        args = N.KV_WRITE_ARGS.pack(q or 0, fake, fake, qw or 0, kw or 0, fake, fake, fake, slots or 0, fake, 512, 128, 256, 128, 256, 128,
                                    c or cache(), dtype, tokens, heads, rows, eps)
        return lib.kl_qk_norm_rope_write(args, None)

    assert write(tokens=-1) == bad and write(heads=0) == bad and write(kw=None) == bad and write(rows=0) == bad
    assert write(eps=0.0) == bad and write(eps=float("nan")) == bad and write(q=None) == bad and write(slots=None) == bad
    assert write(tokens=1 << 30) == bad and write(dtype=N.KL_DT_F32) == bad and write(cache(dim=32)) == bad
    assert write(tokens=0) == N.KL_OK
    assert lib.kl_read_kv(cache(), N.KL_DT_BF16, fake, -1, fake, fake, None) == bad
    assert lib.kl_read_kv(cache(), N.KL_DT_BF16, None, 1, fake, fake, None) == bad
    assert lib.kl_read_kv(cache(), N.KL_DT_BF16, fake, 1, fake + 8, fake, None) == bad
    assert lib.kl_read_kv(cache(), N.KL_DT_BF16, fake, 0, fake, fake, None) == N.KL_OK
    assert lib.kl_paged_attention_workspace_bytes(0, 4, 2, 128) == 0


def test_kv_slots():
    table = torch.tensor([[4, 2], [0, 9]], dtype=torch.int32)
    rows, positions = torch.tensor([0, 0, 1]), torch.tensor([3, 17, 16])
    assert kl.kv_slots(table, rows, positions, 16).tolist() == [67, 33, 144]


# ---- as operators of torch, and together ------------------------------------------------
def test_registered_operators_and_fake_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    schema = torch.ops.kl_b200.qk_norm_rope_write.default._schema
    assert [a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write] == [
        "k_cache", "v_cache", "k_scales", "v_scales"]
    with FakeTensorMode():
        q, k = (torch.empty(5, h, 128, dtype=torch.bfloat16, device="cuda") for h in (4, 2))
        cache = torch.empty(3, 2, 16, 128, dtype=torch.bfloat16, device="cuda")
        at, cos = torch.empty(5, dtype=torch.int64, device="cuda"), torch.empty(9, 64, device="cuda")
        out = torch.ops.kl_b200.qk_norm_rope_write(q, k, k, None, None, cos, cos, at, at, cache, cache)
        assert out.shape == q.shape and out.dtype == torch.bfloat16
        o, lse = torch.ops.kl_b200.paged_attention(q, cache, cache, torch.empty(5, 3, dtype=torch.int32, device="cuda"), at.int())
        assert o.shape == q.shape and lse.shape == (5, 4) and lse.dtype == torch.float32
        a, b = torch.ops.kl_b200.read_kv(cache.to(torch.int8), cache.to(torch.int8), at, dtype=torch.float16)
        assert a.shape == b.shape == (5, 2, 128) and a.dtype == torch.float16


@gpu
def test_compiled_calls_equal_eager_ones():
    q, cache, table, lengths = batch(generator(14), torch.bfloat16, True, 4, 2, 64, 16, [100, 7], poison=False)
    k = torch.randn(2, 2, 64, device="cuda").bfloat16()
    cos, sin = rope_tables(None, 64, 200)
    positions = lengths.long() - 1
    slots = kl.kv_slots(table, torch.arange(2, device="cuda"), positions, 16)

    def step(q, k, v, c, d, cs, ds):
        q = kl.qk_norm_rope_write(q, k, v, None, None, cos, sin, positions, slots, c, d, cs, ds)
        out, lse = kl.paged_attention(q, c, d, table, lengths, cs, ds, return_lse=True)
        return out * 2, lse, *kl.read_kv(c, d, slots, cs, ds)

    mine, other = ([t.clone() for t in cache] for _ in range(2))
    eager = step(q, k, k, *mine)
    compiled = torch.compile(step, backend="aot_eager", fullgraph=True)(q, k, k, *other)
    assert all(torch.equal(a, b) for a, b in zip(eager, compiled))
    assert all(torch.equal(a, b) for a, b in zip(mine, other))


@gpu
@pytest.mark.parametrize("int8_cache", [False, True])
def test_example_decodes_like_the_uncached_sequence(int8_cache):
    import importlib.util
    from tests.conftest import ROOT
    spec = importlib.util.spec_from_file_location("paged_decode", ROOT / "examples" / "paged_decode.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    error, _ = example.main(batch=3, prompt=77, steps=5, int8_cache=int8_cache)
    # bf16 attention outputs differ by up to two roundings (2^-7); int8 keys and values by a step's half of their largest element,
    # 1/254 of about three times their root mean square, averaged over the sequence
    assert error < (2.0 ** -7 + 3 / 254 if int8_cache else 2.0 ** -7)
