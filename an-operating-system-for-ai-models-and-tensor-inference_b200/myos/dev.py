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

import numpy as np
import torch

from . import _lib
from ._lib import ERR_ARG, ERR_SHAPE, MyosError

WORK_BYTES = _lib.PAGED_WORK_BYTES
_KV = {torch.float32: _lib.KV_F32, torch.bfloat16: _lib.KV_BF16}
_F32, _I32, _W32 = (torch.float32,), (torch.int32,), (torch.int32, torch.uint32)
_I64, _BF16, _U8 = (torch.int64,), (torch.bfloat16,), (torch.uint8,)

# A serving step makes these calls once per layer and token, each a few
# microseconds of device time, so the checks below ask a tensor the fewest
# questions that settle them; _refusal finds the reason after one failed.


def _refuse(code, msg):
    raise MyosError(code, msg)


def _refusal(t, what, dtypes, dev, shape):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        _refuse(ERR_ARG, f"{what}: not a CUDA tensor")
    if t.get_device() != dev:
        _refuse(ERR_ARG, f"{what}: on cuda:{t.get_device()}, not cuda:{dev}")
    if t.dtype not in dtypes:
        _refuse(ERR_ARG, f"{what}: dtype {t.dtype}")
    if tuple(t.shape) != tuple(shape):
        _refuse(ERR_SHAPE, f"{what}: {list(shape)} wanted, got {list(t.shape)}")
    _refuse(ERR_ARG, f"{what}: strides {t.stride()}")


def _device(t, what):
    """The ordinal of a CUDA tensor's device."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        _refuse(ERR_ARG, f"{what}: not a CUDA tensor")
    return t.get_device()


def _vec(t, what, dtypes, dev, n):
    """The address of n contiguous values; None stays None."""
    if t is None:
        return None
    try:
        if t.dtype in dtypes and t.get_device() == dev and t.numel() == n and t.is_contiguous():
            return t.data_ptr()
    except AttributeError:
        pass
    _refusal(t, what, dtypes, dev, (n,))


def _rows(t, what, dtypes, dev, shape):
    """(address, elements from row to row) of a tensor of this shape whose rows
    are contiguous; a single row has no stride of its own."""
    try:
        if t.dtype in dtypes and t.get_device() == dev and t.shape == shape:
            if t.is_contiguous():
                n = t.numel()
                return t.data_ptr(), n // shape[0] if n else 0
            st = t.stride()
            if len(shape) == 2:
                row = shape[1]
                ok = st[1] == 1 or row == 1
            else:
                row = shape[1] * shape[2]
                ok = (st[2] == 1 or shape[2] == 1) and (st[1] == shape[2] or shape[1] == 1)
            if ok:
                return t.data_ptr(), st[0] if shape[0] > 1 else row
    except AttributeError:
        pass
    _refusal(t, what, dtypes, dev, shape)


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream",
                      lambda d: torch.cuda.current_stream(d).cuda_stream)


_fns = {}


def _fn(name):
    f = _fns.get(name)
    if f is None:
        f = _fns[name] = getattr(_lib.load(), name)
    return f


def _run(what, dev, stream, fn, *args):
    stream = _raw_stream(dev) if stream is None else getattr(stream, "cuda_stream", stream)
    if dev == torch.cuda.current_device():
        st = fn(*args, stream)
    else:
        with torch.cuda.device(dev):
            st = fn(*args, stream)
    if st != 0:
        _refuse(st, what)


class PagedKV:
    """One layer's paged cache: k and v as [num_pages, num_kv_heads, page_size,
    head_dim] views, f32 or bf16, with the same strides (a cache kept as
    [num_pages, page_size, num_kv_heads, head_dim] is passed as
    ``t.permute(0, 2, 1, 3)``). Holds the tensors, copies nothing."""

    __slots__ = ("k", "v", "dev", "num_kv_heads", "head_dim", "c", "ref")

    def __init__(self, k, v):
        dev = _device(k, "k")
        kind, shape, st = _KV.get(k.dtype), k.shape, k.stride()
        if kind is None:
            _refuse(ERR_ARG, f"k: dtype {k.dtype}")
        if len(shape) != 4 or max(shape) > 0x7fffffff:
            _refuse(ERR_SHAPE, f"k: [pages, heads, slots, dim] wanted, got {list(shape)}")
        pages, heads, slots, d = shape
        sp, sh, ss, sd = st
        if (getattr(v, "shape", None) != shape or v.dtype is not k.dtype or v.get_device() != dev
                or v.stride() != st):
            _refuse(ERR_ARG, "k and v differ in shape, strides, dtype or device")
        if sd != 1 and d > 1:
            _refuse(ERR_ARG, "the last dimension is not contiguous")
        if 1 in shape:  # a dimension of one element has no stride of its own
            n = max(d, ss if slots > 1 else 0, sh if heads > 1 else 0)
            sp, sh, ss = (x if m > 1 else n for x, m in ((sp, pages), (sh, heads), (ss, slots)))
        self.k, self.v, self.dev = k, v, dev
        self.num_kv_heads, self.head_dim = heads, d
        self.c = _lib.PagedKV(k.data_ptr(), v.data_ptr(), sp, sh, ss, pages, slots, heads, d, kind, 0)
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
    dev = _device(block_table, "block_table")
    table, stride = _rows(block_table, "block_table", _I32, dev, block_table.shape)
    nseq, blocks = block_table.shape
    rows, cap = slots.numel(), free_pages.numel()
    _run("paged_tables", dev, stream, _fn("myos_dev_paged_tables"), table, stride, blocks,
         _vec(ctx_lens, "ctx_lens", _I32, dev, nseq), _vec(new_lens, "new_lens", _I32, dev, nseq),
         nseq, _vec(free_pages, "free_pages", _I32, dev, cap), cap,
         _vec(num_free, "num_free", _I32, dev, 1), page_size, num_pages,
         _vec(slots, "slots", _I64, dev, rows), _vec(positions, "positions", _I32, dev, rows),
         _vec(row_seq, "row_seq", _I32, dev, rows), rows, _vec(kv_lens, "kv_lens", _I32, dev, nseq),
         _vec(seq_starts, "seq_starts", _I32, dev, nseq + 1), _vec(result, "result", _I32, dev, 2))


def qk_norm_rope_store(q_out, qkv, kv: PagedKV, positions, slots, cos=None, sin=None,
                       q_gamma=None, k_gamma=None, eps: float = 1e-6, stream=None):
    """q_out [rows, num_q_heads, d] = the q heads of qkv [rows, (num_q_heads +
    2 num_kv_heads) d], per-head RMSNorm (bf16 q_gamma; None: none) and rotated
    by cos/sin [num_pos, rot_dim / 2] at positions [rows]; k likewise with
    k_gamma, then k and v into the cache at slots [rows] (int64, negative: not
    stored): myos_dev_qk_norm_rope_store. q_out may be a view of qkv's own q
    part."""
    dev = _device(qkv, "qkv")
    if kv.dev != dev:
        _refuse(ERR_ARG, f"kv: on cuda:{kv.dev}, not cuda:{dev}")
    rows, hq, d = q_out.shape
    qp, qs = _rows(q_out, "q_out", _F32, dev, (rows, hq, kv.head_dim))
    ip, istride = _rows(qkv, "qkv", _F32, dev, (rows, (hq + 2 * kv.num_kv_heads) * d))
    npos = rot = 0
    cp = sp = None
    if cos is not None or sin is not None:
        npos, half = (cos if cos is not None else sin).shape
        rot = 2 * half
        cp, cstride = _rows(cos, "cos", _F32, dev, (npos, half))
        sp, sstride = _rows(sin, "sin", _F32, dev, (npos, half))
        if npos > 1 and not cstride == sstride == half:
            _refuse(ERR_ARG, "cos and sin are contiguous")
    _run("qk_norm_rope_store", dev, stream, _fn("myos_dev_qk_norm_rope_store"), qp, qs, ip, istride,
         rows, hq, kv.ref, _vec(q_gamma, "q_gamma", _BF16, dev, d),
         _vec(k_gamma, "k_gamma", _BF16, dev, d), eps, cp, sp, npos, rot,
         _vec(positions, "positions", _I32, dev, rows), _vec(slots, "slots", _I64, dev, rows))


def paged_attention(out, q, kv: PagedKV, block_table, kv_lens, work, scale=None, window: int = 0,
                    lse=None, stream=None):
    """out [nseq, num_q_heads, d] = attention of q (same shape) over the last
    ``window`` (0: all) of each sequence's kv_lens keys; lse [nseq, num_q_heads]
    (optional) their log-sum-exp. scale defaults to 1 / sqrt(d). work: at least
    WORK_BYTES of uint8, zeroed once before its first use, not shared by calls
    that may run at the same time: myos_dev_paged_attn."""
    dev = _device(q, "q")
    if kv.dev != dev:
        _refuse(ERR_ARG, f"kv: on cuda:{kv.dev}, not cuda:{dev}")
    nseq, hq, d = shape = q.shape
    if d != kv.head_dim:
        _refuse(ERR_SHAPE, f"q: head_dim {d}, the cache's is {kv.head_dim}")
    qp, qs = _rows(q, "q", _F32, dev, shape)
    op, ostride = _rows(out, "out", _F32, dev, shape)
    lp = None
    if lse is not None:
        lp, lstride = _rows(lse, "lse", _F32, dev, (nseq, hq))
        if nseq > 1 and lstride != hq:
            _refuse(ERR_ARG, "lse is contiguous")
    blocks = block_table.shape[-1]
    tp, ts = _rows(block_table, "block_table", _I32, dev, (nseq, blocks))
    bytes_ = work.numel()
    _run("paged_attention", dev, stream, _fn("myos_dev_paged_attn"), op, ostride, lp, qp, qs, nseq,
         hq, kv.ref, tp, ts, blocks, _vec(kv_lens, "kv_lens", _I32, dev, nseq),
         d ** -0.5 if scale is None else scale, window, _vec(work, "work", _U8, dev, bytes_), bytes_)


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
    dev = _device(logits, "logits")
    rows, vocab = shape = logits.shape
    lp, ls = _rows(logits, "logits", _F32, dev, shape)
    op = ostride = hp = hs = width = mp = ms = masks = nb = 0
    if out is not None:
        op, ostride = _rows(out, "out", _F32, dev, shape)
    if history is not None:
        width = history.shape[-1]
        hp, hs = _rows(history, "history", _I32, dev, (rows, width))
    if bias_starts is not None:
        if bias_ids is None or bias_vals is None:
            _refuse(ERR_ARG, "bias_starts, bias_ids and bias_vals come together")
        nb = bias_ids.numel()
    if mask is not None:
        masks, words = mask.shape
        mp, ms = _rows(mask, "mask", _W32, dev, (masks, words))
        if words * 32 < vocab:
            _refuse(ERR_SHAPE, "mask: fewer bits than the vocabulary")
    a = _lib.LogitControls(
        hp, hs, width, _vec(prompt_lens, "prompt_lens", _I32, dev, rows),
        _vec(hist_lens, "hist_lens", _I32, dev, rows),
        _vec(repetition, "repetition", _F32, dev, rows),
        _vec(frequency, "frequency", _F32, dev, rows), _vec(presence, "presence", _F32, dev, rows),
        _vec(bias_starts, "bias_starts", _I32, dev, rows + 1),
        _vec(bias_ids, "bias_ids", _I32, dev, nb) if nb else None,
        _vec(bias_vals, "bias_vals", _F32, dev, nb) if nb else None, nb,
        mp, ms, masks, _vec(mask_rows, "mask_rows", _I32, dev, rows))
    if not nb:
        a.bias_starts = None
    _run("logit_controls", dev, stream, _fn("myos_dev_logit_controls"), op, ostride, lp, ls, rows,
         vocab, C.byref(a), _vec(ids, "ids", _W32, dev, rows))
