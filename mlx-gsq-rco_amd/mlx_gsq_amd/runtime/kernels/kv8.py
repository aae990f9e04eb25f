"""The 8-bit K/V cache of the gated attention layers, on libgsq.so (include/gsq.h: gsq_kv8_write,
gsq_kv8_read, gsq_attn_kv8).

Caches are uint8 (B, kv_heads, max_len, head_dim) with float32 scales (B, kv_heads, max_len), for K and
for V: a row x is held as ``scale = max|x| / 127`` and ``u = 128 + round(x / scale)``. The reference keeps
a 16-bit cache (mlx-lm's, behind mlx_gsq/models/qwen35.py:114-152); this one takes half its bytes.
``pos`` is a device tensor of one int64, or one for each row of the batch: the position of the
first new token. ``parents`` (int32 on the device, (S,) or (B, S), S <= 64) makes the new tokens a tree of
drafted ones: token t follows token ``parents[t] < t``, or the cached tokens (-1), sits at cache
position ``pos + t`` and is rotated at ``pos`` + its depth. Rows whose tokens do not all lie inside the
cache, or whose parents are not such, get NaN outputs and keep their cache. Tensors on one GPU, fp16 or
bf16 activations, head_dim 64, 128 or 256; calls run on the current stream and may be captured. They carry
no derivative, and refuse tensors that autograd follows.
"""
from __future__ import annotations

from functools import lru_cache

import torch

from ... import _lib
from .model_ops import MAX_TREE, no_derivative

HEAD_DIMS = (64, 128, 256)


_16_BIT = (torch.float16, torch.bfloat16)


def _one_gpu(t, *others):
    """The device of the tensors (None among them for what is not given)."""
    index = t.get_device()
    if index < 0:
        raise ValueError("tensors must be on one GPU device")
    for o in others:
        if o is not None and o.get_device() != index:
            raise ValueError("tensors must be on one GPU device")
    return t.device


def _caches(k_cache, v_cache, k_scale, v_scale):
    """Shape of the caches after checking them."""
    shape = k_cache.shape
    if len(shape) != 4 or v_cache.shape != shape:
        raise ValueError("k_cache and v_cache must be (B, kv_heads, max_len, head_dim) of one shape")
    if k_cache.dtype is not torch.uint8 or v_cache.dtype is not torch.uint8:
        raise TypeError("8-bit caches are uint8")
    rows = shape[:3]
    if (k_scale.shape != rows or v_scale.shape != rows or k_scale.dtype is not torch.float32
            or v_scale.dtype is not torch.float32):
        raise ValueError("scales must be float32 (B, kv_heads, max_len)")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous() and k_scale.is_contiguous() and v_scale.is_contiguous()):
        raise ValueError("caches and scales must be contiguous")
    return shape


def _row_stride(t, B, S, n, dtype):
    """Elements between the (B, S) rows of n values of t."""
    if t.dtype is not dtype:
        raise ValueError("activations must share one dtype")
    if tuple(t.shape) != (B, S, n):
        raise ValueError(f"attention tensor shapes do not match the head configuration: {tuple(t.shape)}, not {(B, S, n)}")
    row, token, inner = t.stride()
    if inner != 1 and n > 1:
        raise ValueError("rows must have unit inner stride")
    if S < 2:  # the stride between tokens means nothing
        return row
    if B > 1 and row != S * token:
        raise ValueError("(B, S) rows must lie at one stride")
    return token


def _where(pos, parents, B, S):
    """(positions, trees) of a call after checking the tensors."""
    n = pos.numel()
    if pos.dtype is not torch.int64 or (n != 1 and n != B) or not pos.is_contiguous():
        raise ValueError("pos must be one int64, or one for each batch row")
    if parents is None:
        return n, 0
    if parents.dtype is not torch.int32 or tuple(parents.shape) not in ((S,), (B, S)) or not parents.is_contiguous():
        raise ValueError("parents must be contiguous int32 (S,) or (B, S)")
    if S > MAX_TREE:
        raise ValueError(f"a tree holds at most {MAX_TREE} tokens, not {S}")
    return n, parents.shape[0] if parents.dim() == 2 else 1


def _dtype_code(t):
    if t.dtype not in _16_BIT:
        raise TypeError(f"unsupported dtype {t.dtype}")
    return _lib.DTYPE_CODES[t.dtype]


def kv8_write(qg, k, v, q_norm_w, k_norm_w, inv_freq, k_cache, v_cache, k_scale, v_scale, pos, *, heads: int,
              kv_heads: int, head_dim: int, rotary_dim: int, eps: float, parents=None):
    """S new tokens of B rows: qg (B, S, heads * 2 head_dim) with [q | gate] per head, k and v (B, S,
    kv_heads * head_dim), unit inner stride and the (B, S) rows at one stride each. q and k are
    RMS-normalized per head (``q_norm_w``, ``k_norm_w``, eps) and rotated on their first rotary_dim dims
    (rotate-half, inv_freq (rotary_dim / 2,) float64); k and v go into the caches, quantised from their
    unrounded values. Returns the queries (B, S, heads * head_dim) for ``attn_kv8``."""
    no_derivative(qg, k, v, q_norm_w, k_norm_w, inv_freq, k_scale, v_scale)
    dev = _one_gpu(qg, k, v, q_norm_w, k_norm_w, inv_freq, k_cache, v_cache, k_scale, v_scale, pos, parents)
    dtype, code = qg.dtype, _dtype_code(qg)
    B, S = qg.shape[:2]
    shape = _caches(k_cache, v_cache, k_scale, v_scale)
    n_pos, n_trees = _where(pos, parents, B, S)
    if shape[0] != B or shape[1] != kv_heads or shape[3] != head_dim or inv_freq.numel() != rotary_dim // 2:
        raise ValueError("attention tensor shapes do not match the head configuration")
    if inv_freq.dtype is not torch.float64 or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be contiguous float64")
    for t in (q_norm_w, k_norm_w):
        if t.dtype is not dtype or t.numel() != head_dim or not t.is_contiguous():
            raise ValueError("norm weights must be contiguous, head_dim values in the activation dtype")
    q = qg.new_empty((B, S, heads * head_dim))
    _lib.launch("gsq_kv8_write", dev, (
        qg.data_ptr(), _row_stride(qg, B, S, heads * 2 * head_dim, dtype), k.data_ptr(),
        _row_stride(k, B, S, kv_heads * head_dim, dtype), v.data_ptr(), _row_stride(v, B, S, kv_heads * head_dim, dtype),
        q_norm_w.data_ptr(), k_norm_w.data_ptr(), inv_freq.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
        k_scale.data_ptr(), v_scale.data_ptr(), pos.data_ptr(), n_pos, None if parents is None else parents.data_ptr(),
        n_trees, q.data_ptr(), B, S, heads, kv_heads, head_dim, rotary_dim, shape[2], eps, code), "kv8_write")
    return q


def kv8_read(k_cache, v_cache, k_scale, v_scale, *, dtype, start: int = 0, length=None):
    """The values that positions ``start .. start + length - 1`` (default: to the end) of both caches stand
    for, rounded to ``dtype`` (float32, float16 or bfloat16): (k, v), each (B, kv_heads, length, head_dim)."""
    no_derivative(k_scale, v_scale)
    dev = _one_gpu(k_cache, v_cache, k_scale, v_scale)
    B, G, L, hd = _caches(k_cache, v_cache, k_scale, v_scale)
    if dtype not in _lib.DTYPE_CODES:
        raise TypeError(f"unsupported dtype {dtype}")
    n = L - start if length is None else length
    if start < 0 or n < 0 or start + n > L:
        raise ValueError(f"positions {start} .. + {n} of a cache of {L}")
    k = torch.empty((B, G, n, hd), dtype=dtype, device=dev)
    v = torch.empty_like(k)
    _lib.launch("gsq_kv8_read", dev, (
        k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), k.data_ptr(), v.data_ptr(), B * G, L,
        start, n, hd, _lib.DTYPE_CODES[dtype]), "kv8_read")
    return k, v


_cus: dict = {}


def _device_cus(dev) -> int:
    n = _cus.get(dev.index)
    if n is None:
        n = _cus[dev.index] = torch.cuda.get_device_properties(dev).multi_processor_count
    return n


@lru_cache(4096)
def _splits(*sizes) -> int:
    return _lib.lib().gsq_attn_kv8_splits(*sizes)


def attn_kv8(q, qg, k_cache, v_cache, k_scale, v_scale, pos, *, heads: int, kv_heads: int, head_dim: int, parents=None,
             splits=None):
    """Gated grouped-query attention of the S tokens that ``kv8_write`` has written: q its queries (B, S,
    heads * head_dim), qg the [q | gate] rows it read. Token t attends to positions 0 .. pos + t; in a
    tree to those before ``pos``, its ancestors and itself. ``splits``: workgroups that share the positions
    of one tile of rows (default: as many as fill the device). Returns (B, S, heads * head_dim)."""
    no_derivative(q, qg, k_scale, v_scale)
    dev = _one_gpu(q, qg, k_cache, v_cache, k_scale, v_scale, pos, parents)
    dtype, code = q.dtype, _dtype_code(q)
    B, S = q.shape[:2]
    shape = _caches(k_cache, v_cache, k_scale, v_scale)
    n_pos, n_trees = _where(pos, parents, B, S)
    L = shape[2]
    if shape[0] != B or shape[1] != kv_heads or shape[3] != head_dim:
        raise ValueError("attention tensor shapes do not match the head configuration")
    q_stride, qg_stride = _row_stride(q, B, S, heads * head_dim, dtype), _row_stride(qg, B, S, heads * 2 * head_dim, dtype)
    out = q.new_empty((B, S, heads * head_dim))
    if splits is None:
        splits = _splits(B, S, heads, kv_heads, head_dim, L, _device_cus(dev))
    work = None
    if splits > 1:
        work = torch.empty(B * heads * S * splits * (head_dim + 2), dtype=torch.float32, device=dev)
    _lib.launch("gsq_attn_kv8", dev, (
        q.data_ptr(), q_stride, qg.data_ptr(), qg_stride, k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(),
        v_scale.data_ptr(), pos.data_ptr(), n_pos, None if parents is None else parents.data_ptr(), n_trees, out.data_ptr(),
        heads * head_dim, None if work is None else work.data_ptr(), splits, B, S, heads, kv_heads, head_dim, L, code),
        "attn_kv8")
    return out
