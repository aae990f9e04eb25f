"""Steps that serve many requests at once, over paged caches, on libgsq.so (include/gsq.h: gsq_page_plan,
gsq_page_advance, gsq_page_release, gsq_paged_write, gsq_attn_paged, gsq_gdn_packed).

The new tokens of a step's sequences (prompts, pieces of prompts, single tokens) are packed behind one another into N
rows. K and V lie in pages (n_pages, kv_heads, page_size, head_dim), page_size 16, 32, 64, 128 or 256; the block table
(requests, max_pages) int32 names each request's pages. The reference serves one sequence over one cache (mlx-lm's, behind
mlx_gsq/models/qwen35.py:114-152).

``page_plan`` lays a step out on the device, and everything else follows that plan: calls run on the current stream, wait
for nothing and may be captured; a replay follows what the plan's tensors then hold. Rows of a sequence that is
not served, or whose numbers do not fit, get NaN outputs and leave caches and states alone; rows behind the last sequence
get zeros. Tensors on one GPU, fp16 or bf16 activations. The calls carry no derivative, and refuse tensors that
autograd follows.
"""
from __future__ import annotations

from functools import lru_cache
from typing import NamedTuple

import torch

from ... import _lib
from .kv8 import _device_cus, _dtype_code, _one_gpu
from .model_ops import no_derivative

PAGE_SIZES = (16, 32, 64, 128, 256)
MAX_SEQUENCES = 1024


class PagePlan(NamedTuple):
    """A step of B sequences and N packed rows: sequence b's tokens are rows ``cu[b] .. cu[b + 1] - 1``, it belongs to request
    ``rows[b]`` (-1: not served) and has ``lens[b]`` positions, its new ones among them; ``pos`` and ``slots`` (page * page_size +
    row in the page) of each row, -1 where there is none."""
    cu: torch.Tensor     # (B + 1,) int32
    rows: torch.Tensor   # (B,) int32
    lens: torch.Tensor   # (B,) int32
    pos: torch.Tensor    # (N,) int64
    slots: torch.Tensor  # (N,) int64


def _int32(shape, *ts):
    for t in ts:
        if t.dtype is not torch.int32 or (shape is not None and tuple(t.shape) != shape) or not t.is_contiguous():
            raise ValueError("lengths, requests, counts, free pages and the block table must be contiguous int32 of fitting shapes")


def _table(table, lengths, held):
    if table.dim() != 2:
        raise ValueError("the block table must be (requests, max_pages)")
    _int32(None, table)
    _int32((table.shape[0],), lengths, held)


def page_plan(requests, new_tokens, lengths, held, table, free, n_free, *, tokens: int, page_size: int) -> PagePlan:
    """The layout of a step in which request ``requests[b]`` brings ``new_tokens[b]`` tokens behind its ``lengths[r]`` cached
    ones, over ``tokens`` rows. Pages that it needs beyond the ``held[r]`` it has are taken from the end of ``free``
    ((n_pages,), the first ``n_free[0]`` of them free), sequence by sequence; ``table``, ``held`` and ``n_free`` are updated.
    A sequence is not served if its request is out of range or named before, if it does not fit its table row or the
    rows, or if the pages run out before it. Lengths stay (``page_advance``): the same call again gives the same step,
    before ``gdn_packed`` has advanced a recurrent state for it."""
    dev = _one_gpu(requests, new_tokens, lengths, held, table, free, n_free)
    B = requests.shape[0] if requests.dim() == 1 else -1
    _int32((B,), requests, new_tokens)
    _table(table, lengths, held)
    _int32((free.numel(),), free)
    _int32((1,), n_free)
    R, W = table.shape
    cu = torch.empty(B + 1, dtype=torch.int32, device=dev)
    two = torch.empty((2, B), dtype=torch.int32, device=dev)
    at = torch.empty((2, tokens), dtype=torch.int64, device=dev)
    rows, lens = two.unbind(0)
    pos, slots = at.unbind(0)
    _lib.launch("gsq_page_plan", dev, (
        requests.data_ptr(), new_tokens.data_ptr(), lengths.data_ptr(), held.data_ptr(), table.data_ptr(), free.data_ptr(),
        n_free.data_ptr(), B, R, W, free.numel(), tokens, page_size, cu.data_ptr(), rows.data_ptr(), lens.data_ptr(),
        pos.data_ptr(), slots.data_ptr()), "page_plan")
    return PagePlan(cu, rows, lens, pos, slots)


def page_advance(plan: PagePlan, lengths):
    """``lengths`` of the requests served become the plan's: the step's tokens are cached."""
    dev = _one_gpu(plan.rows, plan.lens, lengths)
    _int32(plan.rows.shape, plan.rows, plan.lens)
    _int32((lengths.numel(),), lengths)
    _lib.launch("gsq_page_advance", dev, (plan.rows.data_ptr(), plan.lens.data_ptr(), lengths.data_ptr(), plan.rows.numel(),
                                          lengths.numel()), "page_advance")


def page_release(requests, lengths, held, table, free, n_free):
    """The pages of ``requests`` back to ``free``, in the opposite order of ``page_plan``'s taking; their lengths, pages held and
    table entries are cleared. Requests out of range, or named before, are passed over."""
    dev = _one_gpu(requests, lengths, held, table, free, n_free)
    _int32((requests.numel(),), requests)
    _table(table, lengths, held)
    _int32((free.numel(),), free)
    _int32((1,), n_free)
    R, W = table.shape
    _lib.launch("gsq_page_release", dev, (requests.data_ptr(), lengths.data_ptr(), held.data_ptr(), table.data_ptr(),
                                          free.data_ptr(), n_free.data_ptr(), requests.numel(), R, W, free.numel()),
                "page_release")


def _pages(k_pages, v_pages, dtype):
    shape = k_pages.shape
    if len(shape) != 4 or v_pages.shape != shape:
        raise ValueError("k_pages and v_pages must be (n_pages, kv_heads, page_size, head_dim) of one shape")
    if k_pages.dtype is not dtype or v_pages.dtype is not dtype or not (k_pages.is_contiguous() and v_pages.is_contiguous()):
        raise ValueError("pages must be contiguous in the activation dtype")
    return shape


def _head_rows(t, N, heads, hd, dtype):
    """(token stride, head stride) of t (N, heads, hd)."""
    if t.dtype is not dtype or tuple(t.shape) != (N, heads, hd):
        raise ValueError(f"activations must share one dtype and the head layout: {tuple(t.shape)}, not {(N, heads, hd)}")
    token, head, inner = t.stride()
    if inner != 1:
        raise ValueError("rows must have unit inner stride")
    return token, head


def paged_write(q, k, v, q_norm_w, k_norm_w, inv_freq, k_pages, v_pages, pos, slots, *, eps: float):
    """New tokens into their slots: q (N, heads, head_dim), k and v (N, kv_heads, head_dim) with unit inner stride and any
    others; q and k are RMS-normalized per head (weights of head_dim values, ``eps``) and rotated at ``pos`` (int64, (N,)) on
    their first 2 len(inv_freq) dims (rotate-half, float64 frequencies), k and v written to row ``slots`` (int64, (N,), each
    one once; -1: nowhere) of the pages. Returns the queries (N, heads, head_dim), zeros for tokens without a slot."""
    no_derivative(q, k, v, q_norm_w, k_norm_w, inv_freq, k_pages, v_pages)
    dev = _one_gpu(q, k, v, q_norm_w, k_norm_w, inv_freq, k_pages, v_pages, pos, slots)
    dtype, code = q.dtype, _dtype_code(q)
    n_pages, G, P, hd = _pages(k_pages, v_pages, dtype)
    if q.dim() != 3:
        raise ValueError("q must be (tokens, heads, head_dim)")
    N, H = q.shape[:2]
    strides = (_head_rows(q, N, H, hd, dtype), _head_rows(k, N, G, hd, dtype), _head_rows(v, N, G, hd, dtype))
    if inv_freq.dtype is not torch.float64 or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be contiguous float64")
    for t in (q_norm_w, k_norm_w):
        if t.dtype is not dtype or t.numel() != hd or not t.is_contiguous():
            raise ValueError("norm weights must be contiguous, head_dim values in the activation dtype")
    for t in (pos, slots):
        if t.dtype is not torch.int64 or tuple(t.shape) != (N,) or not t.is_contiguous():
            raise ValueError("pos and slots must be contiguous int64, one for each token")
    out = q.new_empty((N, H, hd))
    _lib.launch("gsq_paged_write", dev, (
        q.data_ptr(), *strides[0], k.data_ptr(), *strides[1], v.data_ptr(), *strides[2], q_norm_w.data_ptr(), k_norm_w.data_ptr(),
        inv_freq.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), pos.data_ptr(), slots.data_ptr(), out.data_ptr(), N, H, G,
        hd, 2 * inv_freq.numel(), n_pages, P, eps, code), "paged_write")
    return out


@lru_cache(4096)
def _attn_work(*sizes) -> int:
    return _lib.lib().gsq_attn_paged_work(*sizes)


@lru_cache(4096)
def _gdn_work(*sizes) -> int:
    return _lib.lib().gsq_gdn_packed_work(*sizes)


def _sequences(plan):
    """Sequences of a plan after checking what attention and recurrence read of it."""
    B = plan.rows.numel()
    if tuple(plan.cu.shape) != (B + 1,):
        raise ValueError("a plan's cu must be (B + 1,), its rows and lens (B,)")
    _int32((B,), plan.rows, plan.lens)
    _int32((B + 1,), plan.cu)
    return B


def attn_paged(q, k_pages, v_pages, table, plan: PagePlan, *, gate=None, max_new=None):
    """Grouped-query attention of a step's packed tokens over their requests' pages, which hold the new tokens too
    (``paged_write``): q its queries (N, heads, head_dim), contiguous; a token sees its request's positions up to its own.
    ``gate`` (N, heads, head_dim, unit inner stride): outputs times its sigmoid. ``max_new``: most new tokens of a
    sequence, where the caller knows it (it chooses kernels; longer ones are served too). Returns (N, heads, head_dim)."""
    no_derivative(q, k_pages, v_pages) if gate is None else no_derivative(q, k_pages, v_pages, gate)
    dev = _one_gpu(q, k_pages, v_pages, table, plan.cu, plan.rows, plan.lens, gate)
    dtype, code = q.dtype, _dtype_code(q)
    n_pages, G, P, hd = _pages(k_pages, v_pages, dtype)
    if q.dim() != 3 or q.shape[2] != hd or not q.is_contiguous():
        raise ValueError("q must be contiguous (tokens, heads, head_dim)")
    N, H = q.shape[:2]
    B = _sequences(plan)
    if table.dim() != 2:
        raise ValueError("the block table must be (requests, max_pages)")
    _int32(None, table)
    R, W = table.shape
    g_token, g_head = (0, 0) if gate is None else _head_rows(gate, N, H, hd, dtype)
    out = torch.empty_like(q)
    most, cus = N if max_new is None else max_new, _device_cus(dev)
    size = _attn_work(N, B, H, G, hd, W, P, most, cus)
    work = torch.empty(size, dtype=torch.float32, device=dev) if size > 0 else None
    _lib.launch("gsq_attn_paged", dev, (
        q.data_ptr(), None if gate is None else gate.data_ptr(), g_token, g_head, k_pages.data_ptr(), v_pages.data_ptr(),
        table.data_ptr(), plan.cu.data_ptr(), plan.rows.data_ptr(), plan.lens.data_ptr(), out.data_ptr(),
        None if work is None else work.data_ptr(), N, B, R, W, H, G, hd, n_pages, P, most, cus, code), "attn_paged")
    return out


def gdn_packed(qkv, z, ab, conv_state, conv_w, ssm_a, dt_bias, rec_state, norm_w, plan: PagePlan, *, key_heads: int,
               value_heads: int, head_k_dim: int, head_v_dim: int, eps: float, max_new=None):
    """``gdn_seq`` over a step's packed sequences: qkv (N, conv_dim), z (N, Hv*dv) and ab (N, 2 Hv) with unit inner stride;
    request r has the states conv_state[r] (K-1, conv_dim) and rec_state[r] (Hv, dk, dv, float32), advanced in place. A
    sequence that begins its request (as many positions as new tokens) begins from zeros, whatever its states hold. No two
    sequences may name one request. head_k_dim 32, 64 or 128, head_v_dim 64, 128 or 256; ``max_new`` as for
    ``attn_paged``. Returns (N, Hv*dv)."""
    no_derivative(qkv, z, ab, conv_state, conv_w, ssm_a, dt_bias, rec_state, norm_w)
    dev = _one_gpu(qkv, z, ab, conv_state, conv_w, ssm_a, dt_bias, rec_state, norm_w, plan.cu, plan.rows, plan.lens)
    dtype, code = qkv.dtype, _dtype_code(qkv)
    B = _sequences(plan)
    conv_dim = 2 * key_heads * head_k_dim + value_heads * head_v_dim
    if qkv.dim() != 2:
        raise ValueError("qkv must be (tokens, conv_dim)")
    N, R, K = qkv.shape[0], rec_state.shape[0], conv_w.shape[-1]
    for t, n in ((qkv, conv_dim), (z, value_heads * head_v_dim), (ab, 2 * value_heads)):
        if t.dtype is not dtype or tuple(t.shape) != (N, n) or t.stride(1) != 1:
            raise ValueError("qkv, z and ab must be (tokens, n) of one dtype and the head configuration, unit inner stride")
    for t in (conv_state, conv_w, norm_w):
        if t.dtype is not dtype or not t.is_contiguous():
            raise ValueError("conv_state, conv_w and norm_w must be contiguous in the activation dtype")
    for t in (ssm_a, dt_bias, rec_state):
        if t.dtype is not torch.float32 or not t.is_contiguous():
            raise ValueError("ssm_a, dt_bias and rec_state must be contiguous float32")
    if (tuple(conv_state.shape) != (R, K - 1, conv_dim) or conv_w.numel() != conv_dim * K
            or tuple(rec_state.shape) != (R, value_heads, head_k_dim, head_v_dim) or norm_w.numel() != head_v_dim
            or ssm_a.numel() != value_heads or dt_bias.numel() != value_heads):
        raise ValueError("GatedDeltaNet tensor shapes do not match the head configuration")
    out = qkv.new_empty((N, value_heads * head_v_dim))
    most = N if max_new is None else max_new
    size = _gdn_work(N, B, key_heads, value_heads, head_k_dim, head_v_dim, K, most)
    work = torch.empty(max(size, 1), dtype=torch.float32, device=dev)
    _lib.launch("gsq_gdn_packed", dev, (
        qkv.data_ptr(), qkv.stride(0), z.data_ptr(), z.stride(0), ab.data_ptr(), ab.stride(0), conv_state.data_ptr(),
        conv_w.data_ptr(), ssm_a.data_ptr(), dt_bias.data_ptr(), rec_state.data_ptr(), norm_w.data_ptr(), plan.cu.data_ptr(),
        plan.rows.data_ptr(), plan.lens.data_ptr(), out.data_ptr(), out.stride(0), work.data_ptr(), N, B, R, key_heads,
        value_heads, head_k_dim, head_v_dim, K, eps, most, code), "gdn_packed")
    return out
