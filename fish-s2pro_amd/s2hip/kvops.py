"""KV-cache operators on device memory over the s2hip C ABI (include/s2hip.h,
s2hip_kv_*): head norms, rotation and cache write of new tokens, attention of
a batch whose requests share a long prefix, the same with every key's weight
accumulated, and eviction by those weights.

Arrays are device pointers (integers, e.g. torch tensors' data_ptr()) on the
handle's device; activations are float32, caches float32 or float16.  Calls
launch on the given stream (e.g. torch.cuda.current_stream().cuda_stream; 0:
the default stream) and return at once; the caller keeps the arrays alive and
orders calls on one handle on the device.  Failures raise ``S2HipError``.
There is no CPU fallback.

torch brings a HIP runtime of its own, which s2hip shares if torch was imported
before s2hip's library was loaded (the first handle does that); pointers and
streams of torch's are no good to the other runtime otherwise, and KvOps refuses.
"""

from __future__ import annotations

import ctypes
import sys

from . import _lib
from .engine import S2HipError

ERR_LENS = 1
ERR_POSITION = 2
ERR_F16_RANGE = 4


class KvOps:
    def __init__(self, heads: int, kv_heads: int, head_dim: int, max_requests: int = 16, max_tokens: int = 4096,
                 kv_f16: bool = False, rope_base: float = 1.0e6, eps: float = 1.0e-6, scale: float = 0.0,
                 device: int = 0):
        """max_requests, max_tokens: the most requests, and requests * n_tokens,
        of one call.  scale 0: 1 / sqrt(head_dim)."""
        L = _lib.load()
        runtimes = _lib.hip_runtimes()
        if "torch" in sys.modules and len(runtimes) > 1:
            raise S2HipError("two HIP runtimes in this process (" + ", ".join(runtimes) + "): import torch before the first s2hip handle")
        cfg = _lib.KvConfig(device, heads, kv_heads, head_dim, int(kv_f16), max_requests, max_tokens, rope_base, eps,
                            scale)
        self._err = ctypes.create_string_buffer(_lib.ERR_CAP)
        h = L.s2hip_kv_open(ctypes.byref(cfg), self._err, _lib.ERR_CAP)
        if not h:
            raise S2HipError(self._err.value.decode())
        self._h, self._L = h, L

    def close(self):
        """The work on the handle has to be done (its streams synchronised)."""
        if getattr(self, "_h", None):
            self._L.s2hip_kv_close(self._h)
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

    @staticmethod
    def view(k: int, v: int, lens: int, requests: int, capacity: int, new_lens: int = 0, prefix_k: int = 0,
             prefix_v: int = 0, prefix_len: int = 0, prefix_capacity: int = 0, request_stride: int = 0,
             head_stride: int = 0, slot_stride: int = 0, prefix_head_stride: int = 0, prefix_slot_stride: int = 0):
        """Where the caches of a layer are (s2hip_kv_view), for the calls below;
        strides in elements, 0 for the dense layout."""
        return _lib.KvView(k, v, lens, new_lens, prefix_k, prefix_v, request_stride, head_stride, slot_stride,
                           prefix_head_stride, prefix_slot_stride, requests, capacity, prefix_len, prefix_capacity)

    def errors(self, stream: int = 0) -> int:
        """ERR_* bits that calls have set on the device since the last errors(); waits for the stream."""
        bits = ctypes.c_uint32(0)
        self._check(self._L.s2hip_kv_errors(self._h, stream, ctypes.byref(bits), self._err, _lib.ERR_CAP))
        return bits.value

    def append(self, view, qkv: int, n_tokens: int, positions: int, q_out: int, q_norm: int = 0, k_norm: int = 0,
               scores: int = 0, slot_positions: int = 0, stream: int = 0):
        """QK-norm, rotation and cache write of the new tokens (s2hip_kv_append)."""
        self._check(self._L.s2hip_kv_append(self._h, view, qkv, n_tokens, positions, q_norm, k_norm, q_out, scores,
                                            slot_positions, stream, self._err, _lib.ERR_CAP))

    def attend(self, view, q: int, n_tokens: int, out: int, stream: int = 0):
        """Attention over the shared prefix and the own caches (s2hip_kv_attend)."""
        self._check(self._L.s2hip_kv_attend(self._h, view, q, n_tokens, out, stream, self._err, _lib.ERR_CAP))

    def attend_weigh(self, view, q: int, n_tokens: int, out: int, weights_out: int, weights_in: int = 0,
                     prefix_weights_out: int = 0, prefix_weights_in: int = 0, stream: int = 0):
        """attend, with every key's weight added to weights_in (s2hip_kv_attend_weigh)."""
        self._check(self._L.s2hip_kv_attend_weigh(self._h, view, q, n_tokens, out, weights_in, weights_out,
                                                  prefix_weights_in, prefix_weights_out, stream, self._err,
                                                  _lib.ERR_CAP))

    def evict(self, view, keep: int, recent: int, sinks: int, scores: int, positions: int, scores_out: int,
              positions_out: int, lens_out: int, layers: int = 1, layer_stride: int = 0, stream: int = 0):
        """Caches cut down to `keep` slots by score (s2hip_kv_evict)."""
        self._check(self._L.s2hip_kv_evict(self._h, view, layers, layer_stride, keep, recent, sinks, scores, positions,
                                           scores_out, positions_out, lens_out, stream, self._err, _lib.ERR_CAP))
