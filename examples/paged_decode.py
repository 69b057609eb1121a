"""A decoder layer's attention block on the quantized linears and the paged key-value cache.

    python examples/paged_decode.py [--int8-cache] [--batch 4] [--prompt 200] [--steps 32]

``PagedAttentionBlock`` is QKV projection (one fused int8 linear), per-head norms, rotary positions and cache write (one
launch), attention and output projection.  Prompts are written and read back for a plain causal attention; then each
step writes one token per sequence and attends over its pages.  The script checks the last step against the whole
sequences computed at once without a cache, and times the decode step as a CUDA graph.
"""
from __future__ import annotations

import argparse
import importlib
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
kl = importlib.import_module("gpu-kernel-lab_b200")


def rope_tables(head_dim, positions, base=1e6, device="cuda"):
    turn = torch.arange(positions, device=device, dtype=torch.float64)[:, None] * base ** (
        -torch.arange(0, head_dim, 2, device=device, dtype=torch.float64) / head_dim)
    return turn.cos().float(), turn.sin().float()


def causal_attention(q, k, v):
    """Plain attention of one sequence: q [tokens, heads, dim], k and v [tokens, kv_heads, dim]."""
    group = q.shape[1] // k.shape[1]
    k, v = (t.repeat_interleave(group, 1) for t in (k, v))
    scores = torch.einsum("qhd,khd->hqk", q.float(), k.float()) * q.shape[2] ** -0.5
    scores.masked_fill_(torch.ones(scores.shape[1:], dtype=torch.bool, device=q.device).triu(1), -torch.inf)
    return torch.einsum("hqk,khd->qhd", scores.softmax(-1), v.float()).to(q.dtype)


class PagedAttentionBlock:
    """``heads`` and ``kv_heads`` of ``head_dim`` on a hidden size; random weights, int8 projections."""

    def __init__(self, hidden, heads, kv_heads, head_dim, pages, page_size=16, int8_cache=False, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.heads, self.kv_heads, self.dim, self.page_size = heads, kv_heads, head_dim, page_size
        rows = (heads + 2 * kv_heads) * head_dim
        self.w_qkv = kl.quantize_int8_rowwise(torch.randn(rows, hidden, generator=g, device="cuda") * hidden ** -0.5)
        self.w_o = kl.quantize_int8_rowwise(torch.randn(hidden, heads * head_dim, generator=g, device="cuda") * hidden ** -0.5)
        self.q_norm, self.k_norm = ((1 + 0.1 * torch.randn(head_dim, generator=g, device="cuda")).bfloat16() for _ in range(2))
        self.cos, self.sin = rope_tables(head_dim, pages * page_size)
        self.cache = kl.new_kv_cache(pages, page_size, kv_heads, head_dim, torch.int8 if int8_cache else torch.bfloat16)

    def project(self, x):
        qkv = kl.quant_linear(x, self.w_qkv).unflatten(1, (-1, self.dim))
        return qkv.split([self.heads, self.kv_heads, self.kv_heads], 1)

    def write(self, x, positions, slots):
        return kl.qk_norm_rope_write(*self.project(x), self.q_norm, self.k_norm, self.cos, self.sin, positions, slots, *self.cache)

    def prefill(self, x, page_row):
        """One prompt ``x`` [tokens, hidden] into the pages ``page_row``."""
        positions = torch.arange(len(x), device="cuda")
        slots = kl.kv_slots(page_row[None], torch.zeros_like(positions), positions, self.page_size)
        q = self.write(x, positions, slots)
        k, v = kl.read_kv(self.cache.k_cache, self.cache.v_cache, slots, self.cache.k_scales, self.cache.v_scales)
        return kl.quant_linear(causal_attention(q, k, v).flatten(1), self.w_o)

    def decode(self, x, page_table, lengths):
        """One token ``x`` [batch, hidden] of each sequence, whose cache then holds ``lengths`` tokens."""
        positions = lengths.long() - 1
        slots = kl.kv_slots(page_table, torch.arange(len(x), device="cuda"), positions, self.page_size)
        q = self.write(x, positions, slots)
        out = kl.paged_attention(q, self.cache.k_cache, self.cache.v_cache, page_table, lengths, self.cache.k_scales, self.cache.v_scales)
        return kl.quant_linear(out.flatten(1), self.w_o)


@torch.inference_mode()
def main(batch=4, prompt=200, steps=32, int8_cache=False, hidden=1024, heads=16, kv_heads=8, head_dim=128):
    columns = -(-(prompt + steps) // 16)
    block = PagedAttentionBlock(hidden, heads, kv_heads, head_dim, batch * columns, int8_cache=int8_cache)
    page_table = torch.randperm(batch * columns, device="cuda").int().view(batch, columns)
    x = torch.randn(batch, prompt + steps, hidden, device="cuda").bfloat16()
    for b in range(batch):
        block.prefill(x[b, :prompt], page_table[b])
    for t in range(prompt, prompt + steps):
        lengths = torch.full((batch,), t + 1, dtype=torch.int32, device="cuda")
        y = block.decode(x[:, t], page_table, lengths)

    # the same from the whole sequences, without a cache
    worst = 0.0
    for b in range(batch):
        q, k, v = block.project(x[b])
        scratch = kl.new_kv_cache(columns, 16, kv_heads, head_dim)
        at = torch.arange(len(x[b]), device="cuda")
        q = kl.qk_norm_rope_write(q, k, v, block.q_norm, block.k_norm, block.cos, block.sin, at, at, *scratch)
        k, v = kl.read_kv(*scratch[:2], at)
        ref = kl.quant_linear(causal_attention(q, k, v)[-1:].flatten(1), block.w_o)
        worst = max(worst, ((y[b].float() - ref[0].float()).norm() / ref.float().norm()).item())

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        block.decode(x[:, -1], page_table, lengths)
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    graph.replay()
    start.record()
    for _ in range(100):
        graph.replay()
    end.record()
    torch.cuda.synchronize()
    return worst, start.elapsed_time(end) * 10


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--int8-cache", action="store_true")
    for name, default in (("batch", 4), ("prompt", 200), ("steps", 32)):
        ap.add_argument("--" + name, type=int, default=default)
    error, step_us = main(**vars(ap.parse_args()))
    print(f"last step against the uncached sequences: relative difference {error:.2g}; decode step {step_us:.1f} us")
