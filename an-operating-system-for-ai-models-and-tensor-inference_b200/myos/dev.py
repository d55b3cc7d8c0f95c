"""Operators on tensors already in device memory: one serving step over a
paged KV cache (the device-pointer section of include/myos_cuda.h).

  paged_tables         block tables, slot maps and positions from request lengths
  qk_norm_rope_store   per-head norm and rotation of q and k, K/V into the pages
  paged_attention      attention of one new token per sequence over the pages
  logit_controls       penalties, biases, grammar masks, and the greedy id

Tensors are torch CUDA tensors, all on one device; the work runs there, on
``stream`` (a torch.cuda.Stream or a raw handle; default: torch's current
stream of that device), without a synchronization, and writes into the tensors
that it is given. As with any kernel launched outside torch's allocator, a
tensor last used on another stream needs the caller's own ordering. The last
dimension of every tensor is contiguous; rows may be strided. A refused call
raises MyosError with the C call's status and has no effect.
"""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import torch

from . import _lib
from ._lib import ERR_ARG, ERR_SHAPE, MyosError

WORK_BYTES = _lib.PAGED_WORK_BYTES
_KV = {torch.float32: _lib.KV_F32, torch.bfloat16: _lib.KV_BF16}
_W32 = (torch.int32, torch.uint32)


def _refuse(code, msg):
    raise MyosError(code, msg)


class _Call:
    """Pointers of one call's tensors, all on the first one's device."""
    __slots__ = ("dev",)

    def __init__(self, first):
        if not isinstance(first, torch.Tensor) or not first.is_cuda:
            _refuse(ERR_ARG, "tensors live on a CUDA device")
        self.dev = first.get_device()

    def ptr(self, t, what, dtypes, ndim=1):
        """The address of t (0 for None)."""
        if t is None:
            return None
        if not isinstance(t, torch.Tensor) or t.get_device() != self.dev:
            _refuse(ERR_ARG, f"{what}: not a tensor on cuda:{self.dev}")
        if t.dtype is not dtypes and not (type(dtypes) is tuple and t.dtype in dtypes):
            _refuse(ERR_ARG, f"{what}: dtype {t.dtype}")
        if t.dim() != ndim:
            _refuse(ERR_SHAPE, f"{what}: {ndim} dimensions wanted, got {t.dim()}")
        if t.stride(-1) != 1 and t.size(-1) > 1:
            _refuse(ERR_ARG, f"{what}: the last dimension is not contiguous")
        return t.data_ptr()

    def vec(self, t, what, dtypes, n):
        """The address of a 1-D tensor of n values (None stays None)."""
        p = self.ptr(t, what, dtypes)
        if t is not None and t.size(0) != n:
            _refuse(ERR_SHAPE, f"{what}: {n} values wanted, got {t.size(0)}")
        return p

    def run(self, what, fn, *args, stream=None):
        if stream is None:
            stream = torch.cuda.current_stream(self.dev)
        stream = getattr(stream, "cuda_stream", stream)
        if self.dev == torch.cuda.current_device():
            st = fn(*args, stream)
        else:
            with torch.cuda.device(self.dev):
                st = fn(*args, stream)
        if st != 0:
            _refuse(st, what)


def _row_stride(t):
    """Elements from one row of t to the next; a single row has none of its own."""
    if t.size(0) > 1:
        return t.stride(0)
    n = 1
    for s in t.shape[1:]:
        n *= s
    return max(t.stride(0), n)


def _packed(t, what):
    """[rows, heads, d] with the heads of a row next to each other."""
    if t.size(1) > 1 and t.stride(1) != t.size(2):
        _refuse(ERR_ARG, f"{what}: the heads of a row are not contiguous")


class PagedKV:
    """One layer's paged cache: k and v as [num_pages, num_kv_heads, page_size,
    head_dim] views, f32 or bf16, with the same strides (a cache kept as
    [num_pages, page_size, num_kv_heads, head_dim] is passed as
    ``t.permute(0, 2, 1, 3)``). Holds the tensors, copies nothing."""

    def __init__(self, k, v):
        c = _Call(k)
        kp, vp = c.ptr(k, "k", (torch.float32, torch.bfloat16), 4), c.ptr(v, "v", k.dtype, 4)
        pages, heads, slots, d = k.shape
        sp, sh, ss, _ = k.stride()
        if v.shape != k.shape or v.stride() != k.stride():
            _refuse(ERR_SHAPE, "k and v differ in shape or strides")
        if max(pages, heads, slots, d) > 0x7fffffff:
            _refuse(ERR_SHAPE, "cache dimensions")
        # a dimension of one element has no stride of its own
        n = max(d, ss if slots > 1 else 0, sh if heads > 1 else 0)
        self.k, self.v, self.dev = k, v, c.dev
        self.num_kv_heads, self.head_dim = heads, d
        self.c = _lib.PagedKV(kp, vp, sp if pages > 1 else n, sh if heads > 1 else n,
                              ss if slots > 1 else n, pages, slots, heads, d, _KV[k.dtype], 0)
        self.ref = C.byref(self.c)


def rope_table(num_pos: int, rot_dim: int, theta: float):
    """(cos, sin) numpy arrays [num_pos, rot_dim / 2], as the engine's own
    table (tensor_core rope.rs:186-194)."""
    L = _lib.load()
    cs = np.empty((num_pos, rot_dim // 2), np.float32)
    sn = np.empty((num_pos, rot_dim // 2), np.float32)
    st = L.myos_rope_table(cs.ctypes.data_as(_lib._f32p), sn.ctypes.data_as(_lib._f32p), num_pos,
                           rot_dim, theta)
    if st != 0:
        _refuse(st, "rope_table")
    return cs, sn


def paged_tables(block_table, ctx_lens, new_lens, free_pages, num_free, page_size: int,
                 num_pages: int, slots, positions, row_seq, kv_lens, seq_starts, result,
                 stream=None):
    """Gives each request the pages for its new tokens (from the end of
    free_pages[:num_free]) and maps the step's packed rows to cache slots:
    myos_dev_paged_tables. block_table [nseq, max_blocks] is updated in place;
    slots (int64), positions, row_seq [max_rows], kv_lens [nseq], seq_starts
    [nseq + 1] and result [2] (pages left, requests refused) are written. All
    integers but slots are int32."""
    c, i32 = _Call(block_table), torch.int32
    table = c.ptr(block_table, "block_table", i32, 2)
    nseq, blocks = block_table.shape
    rows = slots.size(0)
    c.run("paged_tables", _lib.load().myos_dev_paged_tables, table, _row_stride(block_table), blocks,
          c.vec(ctx_lens, "ctx_lens", i32, nseq), c.vec(new_lens, "new_lens", i32, nseq), nseq,
          c.ptr(free_pages, "free_pages", i32), free_pages.size(0),
          c.vec(num_free, "num_free", i32, 1), page_size, num_pages,
          c.ptr(slots, "slots", torch.int64), c.vec(positions, "positions", i32, rows),
          c.vec(row_seq, "row_seq", i32, rows), rows, c.vec(kv_lens, "kv_lens", i32, nseq),
          c.vec(seq_starts, "seq_starts", i32, nseq + 1), c.vec(result, "result", i32, 2),
          stream=stream)


def qk_norm_rope_store(q_out, qkv, kv: PagedKV, positions, slots, cos=None, sin=None,
                       q_gamma=None, k_gamma=None, eps: float = 1e-6, stream=None):
    """q_out [rows, num_q_heads, d] = the q heads of qkv [rows, (num_q_heads +
    2 num_kv_heads) d], per-head RMSNorm (bf16 q_gamma; None: none) and rotated
    by cos/sin [num_pos, rot_dim / 2] at positions [rows]; k likewise with
    k_gamma, then k and v into the cache at slots [rows] (int64, negative: not
    stored): myos_dev_qk_norm_rope_store. q_out may be a view of qkv's own q
    part."""
    c, f32 = _Call(qkv), torch.float32
    rows, width = qkv.size(0), qkv.size(-1)
    qp, ip = c.ptr(q_out, "q_out", f32, 3), c.ptr(qkv, "qkv", f32, 2)
    hq, d = q_out.size(1), kv.head_dim
    if kv.dev != c.dev:
        _refuse(ERR_ARG, f"kv: not on cuda:{c.dev}")
    if q_out.size(0) != rows or q_out.size(2) != d or width != (hq + 2 * kv.num_kv_heads) * d:
        _refuse(ERR_SHAPE, "q_out, qkv and the cache disagree")
    _packed(q_out, "q_out")
    half = npos = 0
    if cos is not None or sin is not None:
        if cos is None or sin is None or cos.shape != sin.shape:
            _refuse(ERR_SHAPE, "cos and sin come together, of one shape")
        npos, half = cos.shape
        if not cos.is_contiguous() or not sin.is_contiguous():
            _refuse(ERR_ARG, "cos and sin are contiguous")
    c.run("qk_norm_rope_store", _lib.load().myos_dev_qk_norm_rope_store, qp, _row_stride(q_out), ip,
          _row_stride(qkv), rows, hq, kv.ref, c.vec(q_gamma, "q_gamma", torch.bfloat16, d),
          c.vec(k_gamma, "k_gamma", torch.bfloat16, d), eps, c.ptr(cos, "cos", f32, 2),
          c.ptr(sin, "sin", f32, 2), npos, 2 * half,
          c.vec(positions, "positions", torch.int32, rows),
          c.vec(slots, "slots", torch.int64, rows), stream=stream)


def paged_attention(out, q, kv: PagedKV, block_table, kv_lens, work, scale=None, window: int = 0,
                    lse=None, stream=None):
    """out [nseq, num_q_heads, d] = attention of q (same shape) over the last
    ``window`` (0: all) of each sequence's kv_lens keys; lse [nseq, num_q_heads]
    (optional) their log-sum-exp. scale defaults to 1 / sqrt(d). work: at least
    WORK_BYTES of uint8, zeroed once before its first use, not shared by calls
    that may run at the same time: myos_dev_paged_attn."""
    c, f32 = _Call(q), torch.float32
    qp, op = c.ptr(q, "q", f32, 3), c.ptr(out, "out", f32, 3)
    nseq, hq, d = q.shape
    if kv.dev != c.dev:
        _refuse(ERR_ARG, f"kv: not on cuda:{c.dev}")
    if out.shape != q.shape or d != kv.head_dim:
        _refuse(ERR_SHAPE, "out, q and the cache disagree")
    _packed(q, "q")
    _packed(out, "out")
    lp = c.ptr(lse, "lse", f32, 2)
    if lse is not None and (lse.shape != (nseq, hq) or not lse.is_contiguous()):
        _refuse(ERR_SHAPE, "lse: [nseq, num_q_heads], contiguous")
    table = c.ptr(block_table, "block_table", torch.int32, 2)
    if block_table.size(0) != nseq:
        _refuse(ERR_SHAPE, "block_table: one row per sequence")
    c.run("paged_attention", _lib.load().myos_dev_paged_attn, op, _row_stride(out), lp, qp,
          _row_stride(q), nseq, hq, kv.ref, table, _row_stride(block_table), block_table.size(1),
          c.vec(kv_lens, "kv_lens", torch.int32, nseq),
          1.0 / math.sqrt(d) if scale is None else scale, window,
          c.ptr(work, "work", torch.uint8), work.size(0), stream=stream)


def logit_controls(out, logits, history=None, prompt_lens=None, hist_lens=None, repetition=None,
                   frequency=None, presence=None, bias_starts=None, bias_ids=None, bias_vals=None,
                   mask=None, mask_rows=None, ids=None, stream=None):
    """out [rows, vocab] = logits under each row's penalties (history [rows,
    width] int32, the first prompt_lens of its hist_lens tokens the prompt),
    biases (entries bias_starts[r] .. bias_starts[r + 1] of bias_ids /
    bias_vals) and grammar mask (32 tokens a word, set: allowed; row r uses mask
    mask_rows[r], negative: none); ids [rows] (int32 or uint32) the greedy ids
    of the result: myos_dev_logit_controls. out may be logits (in place) or
    None (only ids)."""
    c, f32, i32 = _Call(logits), torch.float32, torch.int32
    lp, op = c.ptr(logits, "logits", f32, 2), c.ptr(out, "out", f32, 2)
    rows, vocab = logits.shape
    if out is not None and out.shape != logits.shape:
        _refuse(ERR_SHAPE, "out and logits differ in shape")
    hp, mp = c.ptr(history, "history", i32, 2), c.ptr(mask, "mask", _W32, 2)
    if history is not None and history.size(0) != rows:
        _refuse(ERR_SHAPE, "history: one row per row of logits")
    nb = 0
    if bias_starts is not None:
        if bias_ids is None or bias_vals is None or bias_ids.shape != bias_vals.shape:
            _refuse(ERR_SHAPE, "bias_ids and bias_vals come together, of one shape")
        nb = bias_ids.size(0)
    if mask is not None and mask.size(1) * 32 < vocab:
        _refuse(ERR_SHAPE, "mask: fewer bits than the vocabulary")
    a = _lib.LogitControls(
        hp, 0 if history is None else _row_stride(history), 0 if history is None else history.size(1),
        c.vec(prompt_lens, "prompt_lens", i32, rows), c.vec(hist_lens, "hist_lens", i32, rows),
        c.vec(repetition, "repetition", f32, rows), c.vec(frequency, "frequency", f32, rows),
        c.vec(presence, "presence", f32, rows), c.vec(bias_starts, "bias_starts", i32, rows + 1),
        c.ptr(bias_ids, "bias_ids", i32), c.ptr(bias_vals, "bias_vals", f32), nb,
        mp, 0 if mask is None else _row_stride(mask), 0 if mask is None else mask.size(0),
        c.vec(mask_rows, "mask_rows", i32, rows))
    c.run("logit_controls", _lib.load().myos_dev_logit_controls, op,
          0 if out is None else _row_stride(out), lp, _row_stride(logits), rows, vocab, C.byref(a),
          c.vec(ids, "ids", _W32, rows), stream=stream)
