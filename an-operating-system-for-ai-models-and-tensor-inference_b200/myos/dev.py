"""Operators on tensors already in device memory: one serving step over a
paged KV cache (the device-pointer section of include/myos_cuda.h).

  PagedKV              one layer's paged cache, a view of its K and V tensors
  paged_tables         block tables, slot maps and positions from request lengths
  qk_norm_rope_store   per-head norm and rotation of q and k, K/V into the pages
  paged_attention      attention of one new token per sequence over the pages
  logit_controls       penalties, biases, grammar masks, and the greedy id
  rope_table           cos and sin of the rotary angles (host arrays)

Tensors are torch CUDA tensors, all on one device; the work runs there, on
``stream`` (a torch.cuda.Stream or a raw handle; default: torch's current
stream of that device), without a synchronization, and writes into the tensors
that it is given. As with any kernel launched outside torch's allocator, a
tensor last used on another stream needs the caller's own ordering. The last
dimension of every tensor is contiguous; rows may be strided. A refused call
raises MyosError with the C call's status and has no effect.

The checks and calls are native (lib/_myos_dev.so, built by ``build.py``
against the installed torch); there is no fallback.
"""
from __future__ import annotations

import importlib.machinery
import importlib.util
import os

import numpy as np
import torch  # noqa: F401  (its libraries, which the extension links)

from . import _lib
from ._lib import MyosError

WORK_BYTES = _lib.PAGED_WORK_BYTES


def _native():
    path = os.path.join(_lib.LIB_DIR, "_myos_dev.so")
    if not os.path.exists(path):
        raise RuntimeError(f"{path} is missing: build it with python build.py (torch installed)")
    _lib.load()
    loader = importlib.machinery.ExtensionFileLoader("_myos_dev", path)
    module = importlib.util.module_from_spec(importlib.util.spec_from_loader("_myos_dev", loader))
    loader.exec_module(module)
    return module


_m = _native()
PagedKV = _m.PagedKV
paged_tables = _m.paged_tables
qk_norm_rope_store = _m.qk_norm_rope_store
paged_attention = _m.paged_attention
logit_controls = _m.logit_controls


def rope_table(num_pos: int, rot_dim: int, theta: float):
    """(cos, sin) numpy arrays [num_pos, rot_dim / 2], as the engine's own
    table (tensor_core rope.rs:186-194)."""
    cs = np.empty((num_pos, rot_dim // 2), np.float32)
    sn = np.empty((num_pos, rot_dim // 2), np.float32)
    st = _lib.load().myos_rope_table(cs.ctypes.data_as(_lib._f32p), sn.ctypes.data_as(_lib._f32p),
                                     num_pos, rot_dim, theta)
    if st != 0:
        raise MyosError(st, "rope_table")
    return cs, sn
