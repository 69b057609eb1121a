"""The paged key-value cache of a decoder layer: write, read back, attend.

These are the steps between the quantized QKV projection and ``o_proj``:

* ``qk_norm_rope_write``: RMSNorm of every query and key head, rotary positions
  and the cache write, one launch for any number of tokens (the reference's
  ``learning/08_decode/fused_qkv_cache.py:7-54``, on pages);
* ``paged_attention``: attention of one new token per sequence over its pages
  (``serving/paged_attention.py:11-101``);
* ``read_kv``: cached keys and values of given slots, dequantised, for a
  prompt's attention over a cached prefix (``serving/paged_gather.py:8-28``).

A cache is ``k_cache`` and ``v_cache``, ``[pages, kv_heads, page_size,
head_dim]`` with contiguous heads' elements and otherwise any (equal) strides:
a cache laid out ``[pages, page_size, kv_heads, head_dim]`` is passed as
``cache.transpose(1, 2)``.  It holds the activations' type (bf16 or f16), or int8
codes with one f32 scale per token and head in ``k_scales`` and ``v_scales``
``[pages, kv_heads, page_size]``.  ``new_kv_cache`` allocates one; ``kv_slots``
turns positions into slots (``page * page_size + offset``).

Arguments are checked on the host (``ValueError``).  What only the device sees
(a position, slot or page id out of range, a length beyond the page table) never leads to an
access outside the buffers and is recorded for ``_native.device_status``; a
negative slot is not cached and a negative length is an empty sequence.

The functions are for inference: tensors that require grad are refused, as
``qwen_rmsnorm`` refuses them.  Called eagerly they launch directly; under
``torch.compile``, ``torch.export``, ``make_fx``, ``torch.jit.trace``, a fake or other dispatch mode, a
``torch.func`` transform or with tensors of a subclass they are the operators
``torch.ops.kl_b200.*`` of the same names.
"""
from __future__ import annotations

import functools
from typing import NamedTuple, Optional

import torch

from . import _native as N

HEAD_DIMS = (64, 128, 256)
# A call of one token is as long as its host side, so three calls take torch's shorter ways: the current stream
# as an integer (torch.cuda.current_stream() takes 2 us), the current device, and an allocation on it (0.9 us, 1.5 to 2.5 by
# empty_like, new_empty or torch.empty). A torch without one of their names takes the longer way.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_empty_here = getattr(getattr(getattr(torch._C, "_dynamo", None), "guards", None), "_empty_strided_cuda", None)
_is_compiling, _is_grad_enabled = torch.compiler.is_compiling, torch.is_grad_enabled
# Who may be looking at a call: dispatch modes (make_fx, fake tensors), jit.trace, torch.func. A torch that lacks one of these
# names takes every call through the operators.
_modes = getattr(torch._C, "_len_torch_dispatch_stack", None)
_tracing = getattr(torch._C, "_is_tracing", None)
_transform = getattr(getattr(torch._C, "_functorch", None), "peek_interpreter_stack", None)
_BLIND = None in (_modes, _tracing, _transform)
_PLAIN = (torch.Tensor, torch.nn.Parameter)
_I8, _I32, _I64, _F32 = torch.int8, torch.int32, torch.int64, torch.float32
_F32_LEAST, _F32_MOST = 2.0 ** -149, 3.0e38             # what an epsilon is at least; the library's bound of both numbers
_CODES = {torch.bfloat16: N.KL_DT_BF16, torch.float16: N.KL_DT_F16}


class KVCache(NamedTuple):
    """``k_cache`` and ``v_cache``, and their scales where they are int8."""
    k_cache: torch.Tensor
    v_cache: torch.Tensor
    k_scales: Optional[torch.Tensor] = None
    v_scales: Optional[torch.Tensor] = None


def new_kv_cache(pages, page_size, kv_heads, head_dim, dtype=torch.bfloat16, device="cuda") -> KVCache:
    """An empty cache; ``dtype`` is bf16, f16 or ``torch.int8``."""
    if dtype not in (*_CODES, torch.int8):
        raise ValueError('a cache holds bf16, f16 or int8')
    if head_dim not in HEAD_DIMS:
        raise ValueError('head_dim must be 64, 128 or 256')
    if min(pages, page_size, kv_heads) < 1:
        raise ValueError('pages, page_size and kv_heads must be positive')
    k, v = (torch.zeros(pages, kv_heads, page_size, head_dim, dtype=dtype, device=device) for _ in range(2))
    if dtype != torch.int8:
        return KVCache(k, v)
    return KVCache(k, v, *(torch.ones(pages, kv_heads, page_size, device=device) for _ in range(2)))


def kv_slots(page_table, rows, positions, page_size):
    """Slots (int64) of ``positions`` of the sequences ``rows`` of ``page_table``.

    A position that the table has no column for has slot -1, which is not cached: one before the sequence, as ``lengths - 1`` of an
    empty one is, or past its pages.
    """
    columns = page_table.shape[1]
    if columns == 0:
        return torch.full_like(positions + rows, -1, dtype=torch.int64)
    positions = positions.long()
    column = positions // page_size
    there = column.clamp(0, columns - 1)
    slots = torch.add(positions % page_size, page_table[rows, there], alpha=page_size)
    return torch.where(column == there, slots, -1)


def _refuse_grad(*tensors):
    if _is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError('inference only; use torch.inference_mode()')


def _traced(x, cache):
    """Whether a call is to go through the dispatcher: its outputs are allocated past it otherwise, and unknown to who traces it."""
    return (_is_compiling() or _BLIND or _modes() > 0 or _tracing() or _transform() is not None
            or type(x) not in _PLAIN or type(cache) not in _PLAIN)


def _pack_cache(k_cache, v_cache, k_scales, v_scales, dtype, index):
    """Checks of the cache that the three operators share, and its ``kl_kv_cache``; ``index`` is the CUDA device."""
    shape = k_cache.shape
    strides = k_cache.stride()
    held = k_cache.dtype
    if len(shape) != 4 or v_cache.shape != shape:
        raise ValueError('k_cache and v_cache must be [pages, kv_heads, page_size, head_dim]')
    if v_cache.stride() != strides or strides[3] != 1:
        raise ValueError('k_cache and v_cache must have equal strides and contiguous head elements')
    if index < 0 or k_cache.get_device() != index or v_cache.get_device() != index:
        raise ValueError('the cache must be on the same CUDA device as the other tensors')
    pages, kv_heads, page_size, head_dim = shape
    if head_dim not in HEAD_DIMS:
        raise ValueError('head_dim must be 64, 128 or 256')
    if v_cache.dtype is not held:
        raise ValueError('k_cache and v_cache must have one dtype')
    if held is _I8:
        if k_scales is None or v_scales is None:
            raise ValueError('an int8 cache needs k_scales and v_scales')
        scale_strides = k_scales.stride()
        if k_scales.shape != shape[:3] or v_scales.shape != shape[:3] or v_scales.stride() != scale_strides:
            raise ValueError('scales must be [pages, kv_heads, page_size] with equal strides')
        if (k_scales.dtype is not _F32 or v_scales.dtype is not _F32 or k_scales.get_device() != index
                or v_scales.get_device() != index):
            raise ValueError('scales must be FP32 on the cache\'s device')
        return N.KV_CACHE.pack(k_cache.data_ptr(), v_cache.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(), strides[0],
                               strides[1], strides[2], *scale_strides, N.KL_KV_INT8, pages, page_size, kv_heads, head_dim)
    if k_scales is not None or v_scales is not None:
        raise ValueError('only an int8 cache has scales')
    if held is not dtype:
        raise ValueError('the cache must be int8 or of the activations\' dtype')
    return N.KV_CACHE.pack(k_cache.data_ptr(), v_cache.data_ptr(), 0, 0, strides[0], strides[1], strides[2], 0, 0, 0, N.KL_KV_SAME,
                           pages, page_size, kv_heads, head_dim)


def _check_vector(t, name, dtype, count, index):
    if t.dtype is not dtype or t.shape != (count,) or t.get_device() != index or not t.is_contiguous():
        raise ValueError(f'{name} must be a contiguous {dtype} vector of {count} on the cache\'s device')


def _empty(like, shape, strides, dtype, index):
    """An uninitialised tensor on CUDA device ``index``, that of ``like``; ``strides`` are a contiguous tensor's."""
    if _empty_here is not None and index == _current_device():
        return _empty_here(shape, strides, dtype)
    return like.new_empty(shape, dtype=dtype)


def _call(index, fn, *args):
    """``fn(*args, stream)`` with CUDA device ``index`` current."""
    if index == _current_device():
        status = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, _raw_stream(index))
    if status:
        N.check(status)


@functools.lru_cache(maxsize=256)
def paged_attention_workspace_bytes(batch, heads, kv_heads, head_dim) -> int:
    """Bytes of scratch that ``paged_attention`` needs, for a ``workspace`` of the caller's own."""
    return N.lib().kl_paged_attention_workspace_bytes(batch, heads, kv_heads, head_dim)


@functools.lru_cache(maxsize=1024)
def _call_bytes(batch, heads, kv_heads, head_dim, quantized, columns, page_size) -> int:
    """Of that scratch, what one call needs: nothing where its rows are not split."""
    return N.lib().kl_paged_attention_call_bytes(batch, heads, kv_heads, head_dim, N.KL_KV_INT8 if quantized else N.KL_KV_SAME, columns,
                                                 page_size)


def qk_norm_rope_write(q, k, v, q_weight, k_weight, cos, sin, positions, slots, k_cache, v_cache, k_scales=None, v_scales=None,
                       epsilon=1e-6):
    """Normalise and rotate queries and keys, write keys and values to ``slots``; returns the queries.

    * ``q`` ``[tokens, heads, head_dim]``, ``k`` and ``v`` ``[tokens, kv_heads, head_dim]``, bf16 or f16: any strides with
      contiguous head elements, so views of a fused projection's output are taken as they are;
    * ``q_weight``, ``k_weight`` ``[head_dim]``, or both None for a model without these norms;
    * ``cos``, ``sin`` f32 ``[max_positions, head_dim / 2]``: element ``d`` rotates with ``d + head_dim / 2``;
    * ``positions``, ``slots`` int64 ``[tokens]``; slots are distinct, a negative one is not cached.

    The arithmetic is f32 up to one rounding at the store (an int8 cache quantises the f32 value).
    """
    _refuse_grad(q, k, v, q_weight, k_weight, cos, sin, k_cache, v_cache, k_scales, v_scales)
    call = torch.ops.kl_b200.qk_norm_rope_write if _traced(q, k_cache) else write_cuda
    return call(q, k, v, q_weight, k_weight, cos, sin, positions, slots, k_cache, v_cache, k_scales, v_scales, epsilon)


def write_cuda(q, k, v, q_weight, k_weight, cos, sin, positions, slots, k_cache, v_cache, k_scales=None, v_scales=None, epsilon=1e-6):
    """``qk_norm_rope_write`` on CUDA tensors."""
    shape, kv_shape = q.shape, k.shape
    if len(shape) != 3 or len(kv_shape) != 3 or v.shape != kv_shape or shape[0] != kv_shape[0] or shape[2] != kv_shape[2]:
        raise ValueError('q must be [tokens, heads, head_dim], k and v [tokens, kv_heads, head_dim]')
    tokens, heads, dim = shape
    dtype, index = q.dtype, q.get_device()
    if dtype not in _CODES or k.dtype is not dtype or v.dtype is not dtype:
        raise ValueError('q, k and v must have matching FP16/BF16 dtype')
    if index < 0 or k.get_device() != index or v.get_device() != index:
        raise ValueError('q, k, v and the cache must be on the same CUDA device')
    sq, sk, sv = q.stride(), k.stride(), v.stride()
    if tokens and (sq[2] != 1 or sk[2] != 1 or sv[2] != 1):
        raise ValueError('q, k and v must have contiguous head elements')
    cache = _pack_cache(k_cache, v_cache, k_scales, v_scales, dtype, index)
    if kv_shape[1] != k_cache.shape[1] or dim != k_cache.shape[3]:
        raise ValueError('k and v must match the cache\'s heads and head_dim')
    q_weight_at = k_weight_at = 0
    if q_weight is not None and k_weight is not None:
        _check_vector(q_weight, 'q_weight', dtype, dim, index)
        _check_vector(k_weight, 'k_weight', dtype, dim, index)
        if not _F32_LEAST <= epsilon < _F32_MOST:
            raise ValueError('epsilon must be finite and positive in FP32')
        q_weight_at, k_weight_at = q_weight.data_ptr(), k_weight.data_ptr()
    elif q_weight is not None or k_weight is not None:
        raise ValueError('q_weight and k_weight must be given together')
    table = cos.shape
    if len(table) != 2 or table[0] == 0 or 2 * table[1] != dim or sin.shape != table:
        raise ValueError('cos and sin must be [max_positions, head_dim / 2]')
    if (cos.dtype is not _F32 or sin.dtype is not _F32 or cos.get_device() != index or sin.get_device() != index
            or not cos.is_contiguous() or not sin.is_contiguous()):
        raise ValueError('cos and sin must be contiguous FP32 on the cache\'s device')
    _check_vector(positions, 'positions', _I64, tokens, index)
    _check_vector(slots, 'slots', _I64, tokens, index)
    out = _empty(q, (tokens, heads, dim), (heads * dim, dim, 1), dtype, index)
    if tokens:
        args = N.KV_WRITE_ARGS.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), q_weight_at, k_weight_at, cos.data_ptr(),
                                    sin.data_ptr(), positions.data_ptr(), slots.data_ptr(), out.data_ptr(), sq[0], sq[1], sk[0],
                                    sk[1], sv[0], sv[1], cache, _CODES[dtype], tokens, heads, table[0], epsilon)
        _call(index, N.lib().kl_qk_norm_rope_write, args)
    return out


def read_kv(k_cache, v_cache, slots, k_scales=None, v_scales=None, dtype=None):
    """Keys and values ``[tokens, kv_heads, head_dim]`` of ``slots`` (int64), zeros for a negative slot.

    ``dtype`` (bf16 or f16) is that of the result of an int8 cache, bf16 if not given; a 16-bit cache returns its own.
    """
    _refuse_grad(k_cache, v_cache, k_scales, v_scales)
    call = torch.ops.kl_b200.read_kv if _traced(slots, k_cache) else read_cuda
    return call(k_cache, v_cache, slots, k_scales, v_scales, dtype)


def read_cuda(k_cache, v_cache, slots, k_scales=None, v_scales=None, dtype=None):
    """``read_kv`` on CUDA tensors."""
    if dtype is None:
        dtype = torch.bfloat16 if k_cache.dtype is _I8 else k_cache.dtype
    if dtype not in _CODES:
        raise ValueError('keys and values are read as FP16/BF16')
    index = slots.get_device()
    cache = _pack_cache(k_cache, v_cache, k_scales, v_scales, dtype, index)
    tokens = slots.numel()
    _check_vector(slots, 'slots', _I64, tokens, index)
    _, kv_heads, _, dim = k_cache.shape
    shape, strides = (tokens, kv_heads, dim), (kv_heads * dim, dim, 1)
    k, v = _empty(k_cache, shape, strides, dtype, index), _empty(k_cache, shape, strides, dtype, index)
    if tokens:
        _call(index, N.lib().kl_read_kv, cache, _CODES[dtype], slots.data_ptr(), tokens, k.data_ptr(), v.data_ptr())
    return k, v


def paged_attention(q, k_cache, v_cache, page_table, lengths, k_scales=None, v_scales=None, scale=None, return_lse=False,
                    workspace=None):
    """Attention of one new token per sequence: ``softmax(scale * q K^T) V`` over each sequence's cached tokens.

    * ``q`` ``[batch, heads, head_dim]``, bf16 or f16, contiguous head elements; ``heads`` a multiple of the cache's;
    * ``page_table`` int32 ``[batch, columns]``: page ``i`` of a sequence holds its tokens ``i * page_size ...``; entries
      past its length are not read;
    * ``lengths`` int32 ``[batch]``, the new token (written before) included; a sequence of length 0 gives zeros; a used value
      that is not finite makes its element infinite or NaN;
    * ``scale`` is ``head_dim ** -0.5`` if not given.

    Returns the output, or ``(output, lse)`` with ``return_lse``: f32 ``[batch, heads]``, the log of the sum of the
    exponentials (``-inf`` for a length of 0), by which parts of a sequence can be joined.  ``workspace`` (uint8, of
    ``paged_attention_workspace_bytes``) takes the place of scratch allocated for the call; calls that share one must not
    overlap, on the device or, from several threads, on the host.
    """
    _refuse_grad(q, k_cache, v_cache, k_scales, v_scales)
    if _traced(q, k_cache):
        both = torch.ops.kl_b200.paged_attention(q, k_cache, v_cache, page_table, lengths, k_scales, v_scales, scale, workspace)
        return both if return_lse else both[0]
    return attention_cuda(q, k_cache, v_cache, page_table, lengths, k_scales, v_scales, scale, workspace, return_lse)


def attention_cuda(q, k_cache, v_cache, page_table, lengths, k_scales=None, v_scales=None, scale=None, workspace=None,
                   return_lse=True):
    """``paged_attention`` on CUDA tensors."""
    shape = q.shape
    if len(shape) != 3:
        raise ValueError('q must be [batch, heads, head_dim]')
    batch, heads, dim = shape
    dtype, index = q.dtype, q.get_device()
    if dtype not in _CODES:
        raise ValueError('q must be FP16/BF16')
    if index < 0:
        raise ValueError('q and the cache must be on the same CUDA device')
    strides = q.stride()
    if batch and strides[2] != 1:
        raise ValueError('q must have contiguous head elements')
    cache = _pack_cache(k_cache, v_cache, k_scales, v_scales, dtype, index)
    kv_heads = k_cache.shape[1]
    if dim != k_cache.shape[3] or heads == 0 or heads % kv_heads:
        raise ValueError('q must match the cache\'s head_dim and have a multiple of its heads')
    table = page_table.shape
    if len(table) != 2 or table[0] != batch or page_table.dtype is not _I32 or page_table.get_device() != index:
        raise ValueError('page_table must be int32 [batch, columns] on the cache\'s device')
    table_stride, step = page_table.stride()
    if step != 1 and table[1] > 1:
        raise ValueError('page_table must have contiguous rows')
    _check_vector(lengths, 'lengths', _I32, batch, index)
    if scale is None:
        scale = dim ** -0.5
    elif not -_F32_MOST < scale < _F32_MOST:
        raise ValueError('scale must be finite in FP32')
    out = _empty(q, (batch, heads, dim), (heads * dim, dim, 1), dtype, index)
    lse = _empty(q, (batch, heads), (heads, 1), _F32, index) if return_lse else None
    if batch:
        if workspace is None:                            # not N.workspace: another thread's call may come between this one's two launches
            need = _call_bytes(batch, heads, kv_heads, dim, k_cache.dtype is _I8, table[1], k_cache.shape[2])
            workspace = _empty(q, (need,), (1,), torch.uint8, index) if need else None
        elif workspace.get_device() != index or not workspace.is_contiguous():
            raise ValueError('workspace must be contiguous, on the cache\'s device')
        args = N.PAGED_ATTENTION_ARGS.pack(
            q.data_ptr(), page_table.data_ptr(), lengths.data_ptr(), out.data_ptr(), 0 if lse is None else lse.data_ptr(),
            0 if workspace is None else workspace.data_ptr(), 0 if workspace is None else workspace.nbytes, strides[0], strides[1],
            table_stride, cache, _CODES[dtype], batch, heads, table[1], scale)
        _call(index, N.lib().kl_paged_attention, args)
    return (out, lse) if return_lse else out
