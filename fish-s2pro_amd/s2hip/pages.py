"""A KV cache in pages, keys and values in 4 bits, on device memory over the s2hip
C ABI (include/s2hip.h, s2hip_pages_*): head norms, rotation and cache write of new
tokens, attention over the requests' pages, and the pages' management (fork, cut,
free, grow, reorder; compaction of a pool).

Arrays are device pointers (integers, e.g. torch tensors' data_ptr()) on the
handle's device; activations are float32, tables, lengths and counts int32.  Calls
launch on the given stream (0: the default stream) and return at once; the caller
keeps the arrays alive and orders calls on one handle on the device.  Failures
raise ``S2HipError``.  There is no CPU fallback.  torch's HIP runtime: as KvOps.
"""

from __future__ import annotations

import ctypes
import sys

import numpy as np

from . import _lib
from .engine import S2HipError

ERR_LENS = 1
ERR_POSITION = 2
ERR_RANGE = 4
ERR_PAGE = 8
ERR_FULL = 16
ERR_REFS = 32

MAX_ROPE_DIMS = 1 << 16

SCALINGS = {"none": 0, "linear": 1, "stretch": 2, "parts": 3}


def rope_frequencies(dims: int, base: float = 1.0e6, scaling: str = "none", factor: float = 1.0, context: float = 8192,
                     low: float = 1.0, high: float = 32.0):
    """(angles per position of dims / 2 pairs, gain) for PagedKv (s2hip_rope_frequencies);
    needs no device.  scaling: "none", "linear", "stretch" or "parts"."""
    L = _lib.load()
    if scaling not in SCALINGS:
        raise S2HipError(f"rope: scaling {scaling!r} is not one of {', '.join(SCALINGS)}")
    if not 2 <= dims <= MAX_ROPE_DIMS or dims % 2:  # (a C caller's dims are 32 bits without a sign)
        raise S2HipError(f"rope: dims {dims} is not an even number of 2..{MAX_ROPE_DIMS}")
    freq, gain = np.zeros(dims // 2), ctypes.c_double()
    err = ctypes.create_string_buffer(_lib.ERR_CAP)
    if not L.s2hip_rope_frequencies(dims, base, SCALINGS[scaling], factor, context, low, high, freq.ctypes.data,
                                    ctypes.byref(gain), err, _lib.ERR_CAP):
        raise S2HipError(err.value.decode())
    return freq, gain.value


class PagedKv:
    def __init__(self, heads: int, kv_heads: int, head_dim: int, page_tokens: int, pages: int, table_pages: int,
                 max_requests: int = 16, max_tokens: int = 4096, rope_dims: int = 0, rope_half: bool = False,
                 rope_base: float = 1.0e6, rope_gain: float = 0.0, rope_freq=None, eps: float = 1.0e-6,
                 scale: float = 0.0, device: int = 0):
        """pages: of a layer's pool; table_pages: entries of a request's row of the
        table; max_requests, max_tokens: the most rows, and requests * n_tokens, of one
        call.  rope_freq, rope_gain: from rope_frequencies, in place of rope_base (then
        rope_dims is twice their number).  scale 0: 1 / sqrt(head_dim)."""
        L = _lib.load()
        runtimes = _lib.hip_runtimes()
        if "torch" in sys.modules and len(runtimes) > 1:
            raise S2HipError("two HIP runtimes in this process (" + ", ".join(runtimes) + "): import torch before the first s2hip handle")
        freq = None
        if rope_freq is not None:
            freq = np.ascontiguousarray(rope_freq, dtype=np.float64).reshape(-1)
            if rope_dims not in (0, 2 * freq.size) or freq.size == 0:
                raise S2HipError(f"rope_dims {rope_dims} is not twice the {freq.size} frequencies")
            rope_dims = 2 * freq.size
        cfg = _lib.PagesConfig(device, heads, kv_heads, head_dim, page_tokens, pages, table_pages, max_requests, max_tokens, rope_dims,
                               int(rope_half), rope_base, rope_gain, None if freq is None else freq.ctypes.data, eps, scale)
        self._err = ctypes.create_string_buffer(_lib.ERR_CAP)
        h = L.s2hip_pages_open(ctypes.byref(cfg), self._err, _lib.ERR_CAP)
        if not h:
            raise S2HipError(self._err.value.decode())
        self._h, self._L = h, L

    def close(self):
        """The work on the handle has to be done (its streams synchronised)."""
        if getattr(self, "_h", None):
            self._L.s2hip_pages_close(self._h)
            self._h = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _check(self, ok):
        if not ok:
            raise S2HipError(self._err.value.decode())

    @property
    def page_bytes(self) -> int:
        """Bytes of a page of one layer."""
        return self._L.s2hip_pages_bytes(self._h)

    @staticmethod
    def view(pool: int, table: int, lens: int, requests: int, new_lens: int = 0):
        """A layer's pool and the requests' rows (s2hip_pages_view), for the calls below."""
        return _lib.PagesView(pool, table, lens, new_lens, requests)

    def errors(self, stream: int = 0) -> int:
        """ERR_* bits that calls have set on the device since the last errors(); waits for the stream."""
        bits = ctypes.c_uint32(0)
        self._check(self._L.s2hip_pages_errors(self._h, stream, ctypes.byref(bits), self._err, _lib.ERR_CAP))
        return bits.value

    def append(self, view, qkv: int, n_tokens: int, positions: int, q_out: int, q_norm: int = 0, k_norm: int = 0,
               k_held: int = 0, v_held: int = 0, stream: int = 0):
        """QK-norm, rotation and cache write of the new tokens (s2hip_pages_append)."""
        self._check(self._L.s2hip_pages_append(self._h, view, qkv, n_tokens, positions, q_norm, k_norm, q_out, k_held,
                                               v_held, stream, self._err, _lib.ERR_CAP))

    def attend(self, view, q: int, n_tokens: int, out: int, stream: int = 0):
        """Attention of the new tokens over the requests' pages (s2hip_pages_attend)."""
        self._check(self._L.s2hip_pages_attend(self._h, view, q, n_tokens, out, stream, self._err, _lib.ERR_CAP))

    def update(self, view, refs: int, refs_out: int, table_out: int, lens_out: int, source: int = 0, keep: int = 0,
               add: int = 0, layers: int = 1, layer_stride: int = 0, stream: int = 0):
        """The rows made anew: forked, reordered, cut, freed, grown (s2hip_pages_update)."""
        self._check(self._L.s2hip_pages_update(self._h, view, layers, layer_stride, source, keep, add, refs, refs_out,
                                               table_out, lens_out, stream, self._err, _lib.ERR_CAP))

    def compact(self, view, refs: int, refs_out: int, table_out: int, used_out: int, moved_to: int = 0, layers: int = 1,
                layer_stride: int = 0, stream: int = 0):
        """The pages in use moved to the front of the pools (s2hip_pages_compact)."""
        self._check(self._L.s2hip_pages_compact(self._h, view, layers, layer_stride, refs, refs_out, table_out, used_out,
                                                moved_to, stream, self._err, _lib.ERR_CAP))
