"""The operators between the quantized QKV projection and the output projection of a decoder layer, as cases to be timed.

* ``write``: per-head RMSNorm of queries and keys, rotary positions and the write of keys and values into a paged
  cache, in one pass (``qk_norm_rope_write``).  An int8 cache is read back in the same pass (``read_kv``), so that its
  outputs are the values that its codes stand for.
* ``read``: the cached keys and values of given slots, dequantised (``read_kv``).
* ``attend``: attention of one new token per sequence over the paged cache (``paged_attention``).

``own`` chooses between the plain torch forms below and the package's kernels; both take what ``prepare`` returns.
A cache is ``[pages, kv_heads, page_size, head_dim]`` in the activations' type, or int8 with one f32 scale per token and
head (``[pages, kv_heads, page_size]``); a slot is ``page * page_size + offset``.
"""
import importlib
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
EPSILON = 1e-6
MAX_POSITION = 40960
MOST_TOKENS = 64 * 8192          # cached tokens of the largest attention case
MOST_WRITTEN = 16384             # tokens of the largest write
MOST_READ = 65536                # tokens of the largest read


def _attend(name, dtype, cache, heads, kv_heads, dim, page, batch, shortest, longest, lse=False):
    return {"name": name, "op": "attend", "dtype": dtype, "cache": cache, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "page": page, "batch": batch, "shortest": shortest, "longest": longest, "lse": lse}


def _write(name, dtype, cache, heads, kv_heads, dim, page, requests, tokens, start, norm=True):
    return {"name": name, "op": "write", "dtype": dtype, "cache": cache, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "page": page, "requests": requests, "tokens": tokens, "start": start, "norm": norm}


def _read(name, dtype, cache, kv_heads, dim, page, requests, tokens):
    return {"name": name, "op": "read", "dtype": dtype, "cache": cache, "kv_heads": kv_heads, "dim": dim, "page": page,
            "requests": requests, "tokens": tokens}


def listed():
    return [
        # one chat request a few words in: the latency of a call
        _attend("attend-first-words", "bf16", "same", 16, 8, 128, 16, 1, 37, 37),
        # one request with a long document: the whole GPU works on one sequence
        _attend("attend-long-document", "bf16", "same", 16, 8, 128, 16, 1, 32768, 32768, lse=True),
        # a busy server: requests of every age, some slots of the batch idle
        _attend("attend-ragged-batch", "bf16", "same", 24, 8, 128, 64, 32, 0, 4099),
        # the same server with its cache in 8 bits and the memory that this frees used for more and longer requests
        _attend("attend-int8-full-server", "bf16", "int8", 16, 8, 128, 16, 64, 1021, 8192),
        # many short requests in f16, small heads without sharing, pages of an odd size
        _attend("attend-many-short-f16", "f16", "same", 8, 8, 64, 24, 192, 1, 301),
        # many query heads on few cached ones, 8-bit cache
        _attend("attend-int8-shared-heads", "f16", "int8", 32, 2, 128, 32, 7, 500, 16001),
        # one new token of one request
        _write("write-one-token", "bf16", "same", 16, 8, 128, 16, 1, 1, 777),
        # one new token of each request of a batch, 8-bit cache, read back
        _write("write-int8-batch", "bf16", "int8", 24, 8, 128, 16, 48, 1, 2047),
        # prompts of several requests
        _write("write-prompts", "bf16", "same", 16, 8, 128, 16, 8, 1531, 0),
        # a prompt without norms in f16 into an 8-bit cache, read back
        _write("write-int8-prompt-f16", "f16", "int8", 32, 8, 64, 64, 1, 8192, 0, norm=False),
        # a long cached prefix as a prompt's attention wants it
        _read("read-int8-prefix", "bf16", "int8", 8, 128, 16, 1, 65536),
        # short prefixes of a few requests
        _read("read-short-prefixes", "bf16", "same", 8, 128, 32, 3, 211),
    ]


def _between(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _without_name(case):
    return {key: value for key, value in case.items() if key != "name"}


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "f16"])
    cache = rng.choice(["same", "int8"])
    heads, kv_heads, dim = rng.choice([(16, 8, 128), (24, 8, 128), (32, 8, 64), (8, 8, 64), (32, 2, 128), (10, 5, 128), (16, 4, 64)])
    page = rng.choice([16, 16, 32, 64, 24, 8])
    op = rng.choice(["attend", "attend", "attend", "write", "write", "read"])
    if op == "attend":
        longest = _between(rng, 1, 32768)
        most = MOST_TOKENS // (2 if cache == "int8" else 4)
        batch = _between(rng, 1, max(1, min(256, most // longest)))
        shortest = rng.choice([0, 1, longest // 3, longest]) if batch > 1 else longest
        return _without_name(_attend("", dtype, cache, heads, kv_heads, dim, page, batch, shortest, longest, lse=rng.random() < 0.3))
    if op == "write":
        requests = _between(rng, 1, 128)
        tokens = 1 if rng.random() < 0.4 else _between(rng, 1, MOST_WRITTEN // requests)
        start = rng.choice([0, rng.randrange(0, 20000)])
        return _without_name(_write("", dtype, cache, heads, kv_heads, dim, page, requests, tokens, start, norm=rng.random() < 0.7))
    requests = _between(rng, 1, 32)
    return _without_name(_read("", dtype, cache, kv_heads, dim, page, requests, _between(rng, 1, MOST_READ // requests)))


def _lengths(case):
    """The cached lengths of a batch: evenly spread from the shortest to the longest."""
    n, a, b = case["batch"], case["shortest"], case["longest"]
    return [b] if n == 1 else [a + (b - a) * i // (n - 1) for i in range(n)]


def _pages(count, page):
    return -(-count // page)


def _new_cache(case, pages, g, device):
    """A cache in which earlier requests have left their keys and values: (k, v, k_scales, v_scales)."""
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    if case["cache"] == "int8":
        k, v = (torch.randint(-127, 128, shape, generator=g, device=device, dtype=torch.int8) for _ in range(2))
        ks, vs = (torch.rand(shape[:3], generator=g, device=device) * 0.02 + 0.005 for _ in range(2))
        return k, v, ks, vs
    k, v = (torch.randn(shape, generator=g, device=device, dtype=torch.bfloat16).to(TYPES[case["dtype"]]) for _ in range(2))
    return k, v, None, None


def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device).manual_seed(seed)
    dtype, page, dim, kv_heads = TYPES[case["dtype"]], case["page"], case["dim"], case["kv_heads"]
    state = {"case": case}
    if case["op"] == "attend":
        lengths = _lengths(case)
        columns = max(1, _pages(max(lengths), page))
        counts = [_pages(n, page) for n in lengths]
        pages = sum(counts) + 3
        ids = torch.randperm(pages, generator=g, device=device).to(torch.int32)[:sum(counts)]
        order = torch.randperm(len(lengths), generator=g, device=device)
        count = torch.tensor(counts, device=device)[order]
        table = torch.zeros(len(lengths), columns, dtype=torch.int32, device=device)
        table[torch.arange(columns, device=device)[None, :] < count[:, None]] = ids
        state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=device)[order]
        state["page_table"] = table
        state["q"] = (torch.randn(len(lengths), case["heads"], dim, generator=g, device=device) * 1.5).to(dtype)
        state["k_cache"], state["v_cache"], state["k_scales"], state["v_scales"] = _new_cache(case, pages, g, device)
        return state
    requests, tokens = case["requests"], case["tokens"]
    start = case.get("start", 0)
    first = start // page                                   # pages before the first written token belong to others
    columns = _pages(start + tokens, page) - first
    pages = requests * columns + 2
    table = torch.randperm(pages, generator=g, device=device)[:requests * columns].view(requests, columns)
    at = torch.arange(start, start + tokens, device=device)
    state["slots"] = (table[:, at // page - first] * page + at % page).reshape(-1)
    state["k_cache"], state["v_cache"], state["k_scales"], state["v_scales"] = _new_cache(case, pages, g, device)
    if case["op"] == "read":
        return state
    n, heads = requests * tokens, case["heads"]
    fused = torch.randn(n, (heads + 2 * kv_heads) * dim, generator=g, device=device).to(dtype)
    q, k, v = fused.split([heads * dim, kv_heads * dim, kv_heads * dim], dim=1)
    state["q"], state["k"], state["v"] = q.view(n, heads, dim), k.view(n, kv_heads, dim), v.view(n, kv_heads, dim)
    state["q_weight"] = state["k_weight"] = None
    if case["norm"]:
        state["q_weight"], state["k_weight"] = ((1 + 0.2 * torch.randn(dim, generator=g, device=device)).to(dtype) for _ in range(2))
    turn = torch.arange(MAX_POSITION, device=device, dtype=torch.float64)[:, None] * 1e6 ** (
        -torch.arange(0, dim, 2, device=device, dtype=torch.float64) / dim)
    state["cos"], state["sin"] = turn.cos().float(), turn.sin().float()
    state["positions"] = at.repeat(requests)
    return state


# ---- plain forms ------------------------------------------------------------------
def _norm_rope(x, weight, cos, sin):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPSILON) * weight.float()
    a, b = x.chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _codes(x):
    scale = x.abs().amax(-1) / 127
    scale = torch.where(scale == 0, 1.0, scale)
    return torch.round(x / scale[..., None]).clamp(-127, 127).to(torch.int8), scale


def _plain_read(state):
    page, dtype = state["k_cache"].shape[2], TYPES[state["case"]["dtype"]]
    where, off = state["slots"] // page, state["slots"] % page
    k, v = state["k_cache"][where, :, off], state["v_cache"][where, :, off]
    if state["k_scales"] is not None:
        k = k.float() * state["k_scales"][where, :, off, None]
        v = v.float() * state["v_scales"][where, :, off, None]
    return k.to(dtype), v.to(dtype)


def _plain_write(state):
    cos, sin = state["cos"][state["positions"]][:, None], state["sin"][state["positions"]][:, None]
    q = _norm_rope(state["q"], state["q_weight"], cos, sin).to(state["q"].dtype)
    k, v = _norm_rope(state["k"], state["k_weight"], cos, sin), state["v"].float()
    page = state["k_cache"].shape[2]
    where, off = state["slots"] // page, state["slots"] % page
    if state["k_scales"] is None:
        state["k_cache"][where, :, off] = k.to(state["k_cache"].dtype)
        state["v_cache"][where, :, off] = v.to(state["v_cache"].dtype)
        return q
    state["k_cache"][where, :, off], state["k_scales"][where, :, off] = _codes(k)
    state["v_cache"][where, :, off], state["v_scales"][where, :, off] = _codes(v)
    return q


def _plain_attend(state):
    q, table, lengths = state["q"], state["page_table"].long(), state["lengths"]
    k, v = state["k_cache"][table].float(), state["v_cache"][table].float()          # [batch, columns, kv_heads, page, dim]
    if state["k_scales"] is not None:
        k, v = k * state["k_scales"][table][..., None], v * state["v_scales"][table][..., None]
    batch, columns, kv_heads, page, dim = k.shape
    k = k.transpose(1, 2).reshape(batch, kv_heads, columns * page, dim)
    v = v.transpose(1, 2).reshape(batch, kv_heads, columns * page, dim)
    scores = q.float().view(batch, kv_heads, -1, dim) @ k.transpose(2, 3) * dim ** -0.5
    there = (torch.arange(columns * page, device=q.device) < lengths[:, None])[:, None, None]
    scores = torch.where(there, scores, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    weights = torch.exp(scores - top)
    total = weights.sum(-1, keepdim=True)
    out = weights @ torch.where(there.transpose(2, 3), v, 0.0) / torch.where(total == 0, 1.0, total)
    lse = (top + torch.log(total)).reshape(batch, -1)
    return out.reshape(q.shape).to(q.dtype), lse


# ---- one pass -----------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        kl = importlib.import_module("gpu-kernel-lab_b200")
        cache = state["k_cache"], state["v_cache"]
        scales = {"k_scales": state["k_scales"], "v_scales": state["v_scales"]}
        if case["op"] == "attend":
            out = kl.paged_attention(state["q"], *cache, state["page_table"], state["lengths"], **scales,
                                     return_lse=case["lse"])
            return list(out) if case["lse"] else [out]
        if case["op"] == "read":
            return list(kl.read_kv(*cache, state["slots"], **scales, dtype=TYPES[case["dtype"]]))
        q = kl.qk_norm_rope_write(state["q"], state["k"], state["v"], state["q_weight"], state["k_weight"], state["cos"],
                                  state["sin"], state["positions"], state["slots"], *cache, **scales, epsilon=EPSILON)
        if case["cache"] == "int8":
            return [q, *kl.read_kv(*cache, state["slots"], **scales, dtype=TYPES[case["dtype"]]),
                    state["k_scales"], state["v_scales"]]
        return [q, *cache]
    if case["op"] == "attend":
        out, lse = _plain_attend(state)
        return [out, lse] if case["lse"] else [out]
    if case["op"] == "read":
        return list(_plain_read(state))
    q = _plain_write(state)
    if case["cache"] == "int8":
        return [q, *_plain_read(state), state["k_scales"], state["v_scales"]]
    return [q, state["k_cache"], state["v_cache"]]


def work(case):
    dim, kv_heads = case["dim"], case["kv_heads"]
    entry = dim + 4 if case["cache"] == "int8" else 2 * dim                # bytes of one cached key or value
    if case["op"] == "attend":
        tokens, batch, heads = sum(_lengths(case)), case["batch"], case["heads"]
        columns = sum(_pages(n, case["page"]) for n in _lengths(case))
        return {"bytes": tokens * kv_heads * 2 * entry + batch * (heads * dim * 4 + 4) + columns * 4 + (batch * heads * 4 if case["lse"] else 0),
                "flops": tokens * heads * dim * 4}
    n = case["requests"] * case["tokens"]
    read_back = n * 8 + n * kv_heads * 2 * (entry + 2 * dim)
    if case["op"] == "read":
        return {"bytes": read_back, "flops": n * kv_heads * 2 * dim if case["cache"] == "int8" else 0}
    heads = case["heads"]
    moved = n * ((heads + 2 * kv_heads) * dim * 2 + heads * dim * 2 + 2 * kv_heads * entry + 16) + case["tokens"] * dim * 4
    return {"bytes": moved + (read_back if case["cache"] == "int8" else 0), "flops": n * (heads + kv_heads) * dim * (7 if case["norm"] else 3)}


# ---- the definitions in 64 bits --------------------------------------------------------
def _exact_heads(x, weight, angle_cos, angle_sin):
    y = x.double()
    if weight is not None:
        y = y / ((y * y).sum(-1, keepdim=True) / y.shape[-1] + EPSILON).sqrt() * weight.double()
    half = y.shape[-1] // 2
    turned = torch.empty_like(y)
    turned[..., :half] = y[..., :half] * angle_cos - y[..., half:] * angle_sin
    turned[..., half:] = y[..., half:] * angle_cos + y[..., :half] * angle_sin
    return turned


def exact(case, seed):
    state = prepare(case, seed)
    page = case["page"]
    if case["op"] == "attend":
        group, outs, lses = case["heads"] // case["kv_heads"], [], []
        for q, row, length in zip(state["q"].double(), state["page_table"].long(), state["lengths"].tolist()):
            if length == 0:
                outs.append(torch.zeros_like(q))
                lses.append(torch.full_like(q[:, 0], -math.inf))
                continue
            ids = row[:_pages(length, page)]
            k, v = state["k_cache"][ids].double(), state["v_cache"][ids].double()
            if state["k_scales"] is not None:
                k *= state["k_scales"][ids].double()[..., None]
                v *= state["v_scales"][ids].double()[..., None]
            k, v = (t.permute(1, 0, 2, 3).flatten(1, 2)[:, :length].repeat_interleave(group, 0) for t in (k, v))
            scores = torch.einsum("hd,hld->hl", q, k) / math.sqrt(case["dim"])
            outs.append(torch.einsum("hl,hld->hd", torch.softmax(scores, -1), v))
            lses.append(torch.logsumexp(scores, -1))
        return [torch.stack(outs), torch.stack(lses)] if case["lse"] else [torch.stack(outs)]
    slots = state["slots"]
    if case["op"] == "write":
        cos, sin = (state[t].double()[state["positions"]].unsqueeze(1) for t in ("cos", "sin"))
        q = _exact_heads(state["q"], state["q_weight"], cos, sin)
        new = _exact_heads(state["k"], state["k_weight"], cos, sin), state["v"].double()
        if case["cache"] != "int8":
            caches = []
            for cache, value in zip((state["k_cache"], state["v_cache"]), new):
                cache = cache.double().transpose(1, 2).reshape(-1, case["kv_heads"], case["dim"])
                cache[slots] = value
                caches.append(cache.view(-1, page, case["kv_heads"], case["dim"]).transpose(1, 2))
            return [q, *caches]
        values, scales = [], []
        for name, value in zip(("k_scales", "v_scales"), new):
            step = value.abs().max(-1).values / 127
            step[step == 0] = 1
            values.append((value / step.unsqueeze(-1)).round() * step.unsqueeze(-1))
            table = state[name].double().transpose(1, 2).reshape(-1, case["kv_heads"])
            table[slots] = step
            scales.append(table.view(-1, page, case["kv_heads"]).transpose(1, 2))
        return [q, *values, *scales]
    found = []
    for cache, scales in ((state["k_cache"], state["k_scales"]), (state["v_cache"], state["v_scales"])):
        value = cache.double().transpose(1, 2).flatten(0, 1)[slots]
        if scales is not None:
            value = value * scales.double().transpose(1, 2).flatten(0, 1)[slots].unsqueeze(-1)
        found.append(value)
    return found
