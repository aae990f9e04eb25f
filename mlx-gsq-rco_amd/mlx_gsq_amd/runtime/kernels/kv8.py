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
bf16 activations, head_dim 64, 128 or 256; calls run on the current stream and may be captured.
"""
from __future__ import annotations

import torch

from ... import _lib
from .model_ops import MAX_TREE, _on_gpu

HEAD_DIMS = (64, 128, 256)


def _caches(k_cache, v_cache, k_scale, v_scale):
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape:
        raise ValueError("k_cache and v_cache must be (B, kv_heads, max_len, head_dim) of one shape")
    if k_cache.dtype != torch.uint8 or v_cache.dtype != torch.uint8:
        raise TypeError("8-bit caches are uint8")
    if any(s.dtype != torch.float32 or s.shape != k_cache.shape[:3] for s in (k_scale, v_scale)):
        raise ValueError("scales must be float32 (B, kv_heads, max_len)")
    if not all(t.is_contiguous() for t in (k_cache, v_cache, k_scale, v_scale)):
        raise ValueError("caches and scales must be contiguous")


def _rows(what, B, S, *ts):
    """Row strides of (B, S, n) tensors of 16-bit rows."""
    dtype = ts[0].dtype
    if dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"unsupported dtype {dtype}")
    out = []
    for t in ts:
        if (t.dim() != 3 or tuple(t.shape[:2]) != (B, S) or t.stride(2) != 1 or t.dtype != dtype
                or (B > 1 and S > 1 and t.stride(0) != S * t.stride(1))):
            raise ValueError(f"{what} must be (B, S, n) of one dtype, unit inner stride, rows at one stride")
        # a single token's row stride is that of the batch
        out.append(t.stride(0) if S == 1 else t.stride(1))
    return out


def _where(pos, parents, B, S):
    """(positions, trees) of a call after checking the tensors."""
    if pos.dtype != torch.int64 or pos.numel() not in (1, B) or not pos.is_contiguous():
        raise ValueError("pos must be one int64, or one for each batch row")
    if parents is None:
        return pos.numel(), 0
    if parents.dtype != torch.int32 or tuple(parents.shape) not in ((S,), (B, S)) or not parents.is_contiguous():
        raise ValueError("parents must be contiguous int32 (S,) or (B, S)")
    if S > MAX_TREE:
        raise ValueError(f"a tree holds at most {MAX_TREE} tokens, not {S}")
    return pos.numel(), parents.shape[0] if parents.dim() == 2 else 1


def kv8_write(qg, k, v, q_norm_w, k_norm_w, inv_freq, k_cache, v_cache, k_scale, v_scale, pos, *, heads: int,
              kv_heads: int, head_dim: int, rotary_dim: int, eps: float, parents=None):
    """S new tokens of B rows: qg (B, S, heads * 2 head_dim) with [q | gate] per head, k and v (B, S,
    kv_heads * head_dim), unit inner stride and the (B, S) rows at one stride each. q and k are
    RMS-normalized per head (``q_norm_w``, ``k_norm_w``, eps) and rotated on their first rotary_dim dims
    (rotate-half, inv_freq (rotary_dim / 2,) float64); k and v go into the caches, quantised from their
    unrounded values. Returns the queries (B, S, heads * head_dim) for ``attn_kv8``."""
    ts = (qg, k, v, q_norm_w, k_norm_w, inv_freq, k_cache, v_cache, k_scale, v_scale, pos)
    dev = _on_gpu(*ts, *(() if parents is None else (parents,)))
    _caches(k_cache, v_cache, k_scale, v_scale)
    B, S = qg.shape[:2]
    strides = _rows("qg, k and v", B, S, qg, k, v)
    n_pos, n_trees = _where(pos, parents, B, S)
    if (qg.shape[2] != heads * 2 * head_dim or k.shape[2] != kv_heads * head_dim or v.shape[2] != kv_heads * head_dim
            or q_norm_w.numel() != head_dim or k_norm_w.numel() != head_dim or inv_freq.numel() != rotary_dim // 2
            or tuple(k_cache.shape[:2]) != (B, kv_heads) or k_cache.shape[3] != head_dim):
        raise ValueError("attention tensor shapes do not match the head configuration")
    if inv_freq.dtype != torch.float64 or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be contiguous float64")
    for t in (q_norm_w, k_norm_w):
        if t.dtype != qg.dtype or not t.is_contiguous():
            raise ValueError("norm weights must be contiguous in the activation dtype")
    q = torch.empty(B, S, heads * head_dim, dtype=qg.dtype, device=dev)
    _lib.launch("gsq_kv8_write", dev, (
        qg.data_ptr(), strides[0], k.data_ptr(), strides[1], v.data_ptr(), strides[2], q_norm_w.data_ptr(),
        k_norm_w.data_ptr(), inv_freq.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(),
        v_scale.data_ptr(), pos.data_ptr(), n_pos, None if parents is None else parents.data_ptr(), n_trees, q.data_ptr(), B,
        S, heads, kv_heads, head_dim, rotary_dim, k_cache.shape[2], float(eps), _lib.DTYPE_CODES[qg.dtype]), "kv8_write")
    return q


def kv8_read(k_cache, v_cache, k_scale, v_scale, *, dtype, start: int = 0, length=None):
    """The values that positions ``start .. start + length - 1`` (default: to the end) of both caches stand
    for, rounded to ``dtype`` (float32, float16 or bfloat16): (k, v), each (B, kv_heads, length, head_dim)."""
    dev = _on_gpu(k_cache, v_cache, k_scale, v_scale)
    _caches(k_cache, v_cache, k_scale, v_scale)
    if dtype not in _lib.DTYPE_CODES:
        raise TypeError(f"unsupported dtype {dtype}")
    B, G, L, hd = k_cache.shape
    n = L - start if length is None else length
    if start < 0 or n < 0 or start + n > L:
        raise ValueError(f"positions {start} .. + {n} of a cache of {L}")
    k = torch.empty(B, G, n, hd, dtype=dtype, device=dev)
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


def attn_kv8(q, qg, k_cache, v_cache, k_scale, v_scale, pos, *, heads: int, kv_heads: int, head_dim: int, parents=None,
             splits=None):
    """Gated grouped-query attention of the S tokens that ``kv8_write`` has written: q its queries (B, S,
    heads * head_dim), qg the [q | gate] rows it read. Token t attends to positions 0 .. pos + t; in a
    tree to those before ``pos``, its ancestors and itself. ``splits``: workgroups that share the positions
    of one tile of rows (default: as many as fill the device). Returns (B, S, heads * head_dim)."""
    dev = _on_gpu(q, qg, k_cache, v_cache, k_scale, v_scale, pos, *(() if parents is None else (parents,)))
    _caches(k_cache, v_cache, k_scale, v_scale)
    B, S = q.shape[:2]
    strides = _rows("q and qg", B, S, q, qg)
    n_pos, n_trees = _where(pos, parents, B, S)
    L = k_cache.shape[2]
    if (q.shape[2] != heads * head_dim or qg.shape[2] != heads * 2 * head_dim
            or tuple(k_cache.shape[:2]) != (B, kv_heads) or k_cache.shape[3] != head_dim):
        raise ValueError("attention tensor shapes do not match the head configuration")
    out = torch.empty(B, S, heads * head_dim, dtype=q.dtype, device=dev)
    if splits is None:
        splits = _lib.lib().gsq_attn_kv8_splits(B, S, heads, kv_heads, head_dim, L, _device_cus(dev))
    work = None
    if splits > 1:
        work = torch.empty(B * heads * S * splits * (head_dim + 2), dtype=torch.float32, device=dev)
    _lib.launch("gsq_attn_kv8", dev, (
        q.data_ptr(), strides[0], qg.data_ptr(), strides[1], k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(),
        v_scale.data_ptr(), pos.data_ptr(), n_pos, None if parents is None else parents.data_ptr(), n_trees, out.data_ptr(),
        heads * head_dim, None if work is None else work.data_ptr(), int(splits), B, S, heads, kv_heads, head_dim, L,
        _lib.DTYPE_CODES[q.dtype]), "attn_kv8")
    return out
