"""Position rotation of queries and keys, with a norm of each head before it
(C ABI section 7 of include/magpie_tts_rt_b200.h).

``Rotation`` holds what a layer's rotation needs: which dims are turned together
and how far per position, and the weights of the heads' norms, if it has any.
``Rotation.rotate`` turns rows of queries and keys; ``PagedCache.append`` does the
same on the way into a cache.

    y = x / sqrt(mean(x^2) + eps) * weight              over a head, where a weight is given
    (y_a, y_b) -> (y_a cos t - y_b sin t, y_b cos t + y_a sin t),   t = position * frequency_i

for a = i, b = i + rotary_dim / 2 (``interleaved``: a = 2 i, b = 2 i + 1); dims from
rotary_dim on are not turned.  Angles are taken in 64 bits, sums of squares and
the rest in 32, results are rounded once.  No gradient is recorded.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from magpie_tts_rt_b200 import _lib as L
from magpie_tts_rt_b200 import paged_cache as _cache
from magpie_tts_rt_b200.paged_cache import _DTYPES, HEAD_DIMS, MAX_ROWS, _check, _raw_stream, _rows_of, _share, _written_rows

MAX_HEADS = 1 << 16


class Rotation:
    def __init__(self, head_dim: int, rotary_dim: Optional[int] = None, base: float = 10000.0, interleaved: bool = False,
                 frequencies: Optional[torch.Tensor] = None, q_norm: Optional[torch.Tensor] = None,
                 k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6, device="cuda"):
        """rotary_dim (a multiple of 16, all of head_dim if not given) dims of a
        head are turned, pair i by base^(-2 i / rotary_dim) radians a position, or
        by frequencies [rotary_dim / 2] (any real type).  q_norm, k_norm [head_dim]:
        weights of the norms.  All of it is copied, which is waited for: later changes of
        the tensors do not reach the rotation, and any stream may use it.  A rotation may
        be dropped while calls that use it are still queued, but must outlive CUDA graphs
        captured with it (a graph reads frequencies and weights when it is replayed)."""
        _check(head_dim in HEAD_DIMS, f"head_dim must be one of {HEAD_DIMS}")
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        _check(16 <= rotary_dim <= head_dim and rotary_dim % 16 == 0, "rotary_dim must be a multiple of 16, at most head_dim")
        _check(0 <= eps <= torch.finfo(torch.float32).max, "eps must not be negative, and held by single precision")
        if frequencies is None:
            _check(base > 0 and math.isfinite(base), "base must be positive")
            radians = [base ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)]
            frequencies = torch.tensor(radians, dtype=torch.float64)
        else:
            _check(tuple(frequencies.shape) == (rotary_dim // 2,) and not frequencies.is_complex(),
                   "frequencies must be [rotary_dim / 2]")
        self.head_dim, self.rotary_dim, self.interleaved, self.eps = head_dim, rotary_dim, bool(interleaved), float(eps)
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self._index = self.device.index if self.device.type == "cuda" else -1
        self.turns = (frequencies.detach().double() / (2 * math.pi)).to(self.device)
        self.q_norm, self.k_norm = (self._weight(w, n) for w, n in ((q_norm, "q_norm"), (k_norm, "k_norm")))
        if self.device.type == "cuda":  # any stream may be the first to use them
            torch.cuda.current_stream(self.device).synchronize()
        self._raw = _raw_stream(self.device)
        self._streams = set()
        self._c = {}
        for dtype, code in _DTYPES.items():
            c = L.Rotation(head_dim, rotary_dim, int(self.interleaved), code, self.turns.data_ptr())
            c.q_weight, c.k_weight = (None if w is None else w.data_ptr() for w in (self.q_norm, self.k_norm))
            c.eps = self.eps
            self._c[dtype] = (c, ctypes.byref(c))

    def _weight(self, w: Optional[torch.Tensor], name: str) -> Optional[torch.Tensor]:
        if w is None:
            return None
        _check(tuple(w.shape) == (self.head_dim,) and w.dtype.is_floating_point, f"{name} must be [head_dim]")
        return w.detach().to(device=self.device, dtype=torch.float32, copy=True)

    def _on_stream(self, handle: int, stream) -> None:
        """Calls on this stream read the rotation's tensors: their memory is not
        reused before those calls are done."""
        if handle not in self._streams:
            if stream is None:
                stream = torch.cuda.current_stream(self.device)
            for t in (self.turns, self.q_norm, self.k_norm):
                if t is not None:
                    t.record_stream(stream)
            self._streams.add(handle)

    def rotate(self, q: Optional[torch.Tensor], k: Optional[torch.Tensor], positions: torch.Tensor,
               q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None, stream=None):
        """(q, k) normed and turned: q [rows, q_heads, head_dim], k [rows, kv_heads,
        head_dim] bf16 or f16 (either may be None), rows of any stride with
        contiguous heads, positions [rows] int32.  q_out and k_out may be q and k;
        otherwise they must not overlap what the call reads, nor each other."""
        first = k if q is None else q
        if first is None or first.dim() != 3:
            raise ValueError("a rotation needs queries or keys, [rows, heads, head_dim]")
        index, dtype, rows = self._index, first.dtype, first.shape[0]
        if dtype not in _DTYPES or rows > MAX_ROWS:
            raise ValueError(f"q and k must be bfloat16 or float16, of at most {MAX_ROWS} rows")
        if positions.dtype is not torch.int32 or positions.shape != (rows,) or positions.get_device() != index or \
                not positions.is_contiguous():
            raise ValueError(f"positions must be a contiguous int32 vector of {rows} on the rotation's device")
        if stream is None:
            handle = self._raw(index)
        elif stream.device.index == index:
            handle = stream.cuda_stream
        else:
            raise ValueError("the stream belongs to another device than the rotation")
        given = q_out is not None and k_out is not None
        q_heads, q_at, q_row, q_to, q_to_row, q_out = self._side(q, q_out, "q", rows, dtype, stream)
        k_heads, k_at, k_row, k_to, k_to_row, k_out = self._side(k, k_out, "k", rows, dtype, stream)
        if given and _share(q_to // 2, k_to // 2, q_heads * self.head_dim, k_heads * self.head_dim, rows, (q_to_row, k_to_row)):
            raise ValueError("q_out and k_out share memory")
        args = L.RotateRows(rows, q_heads, k_heads, 0, q_at, k_at, None, q_to, k_to, q_row, k_row, 0, q_to_row, k_to_row,
                            positions.data_ptr())
        if handle not in self._streams:
            self._on_stream(handle, stream)
        call = L.lib.mtt_b200_launch_rotate_heads
        if _cache._current_device() == index:
            rc = call(self._c[dtype][1], ctypes.byref(args), handle)
        else:
            with torch.cuda.device(index):
                rc = call(self._c[dtype][1], ctypes.byref(args), handle)
        if rc != L.STATUS_OK:
            raise RuntimeError(f"mtt_b200_launch_rotate_heads failed with status {rc}")
        return q_out, k_out

    def _side(self, x, out, name, rows, dtype, stream):
        """(heads, address, row stride, out's address and row stride, out) of queries or keys."""
        if x is None:
            _check(out is None, f"{name}_out without {name}")
            return 0, None, 0, None, 0, None
        shape = x.shape
        if len(shape) != 3 or shape[0] != rows or shape[2] != self.head_dim or shape[1] > MAX_HEADS:
            raise ValueError("q and k must be [rows, heads, head_dim]")
        stride = _rows_of(x, shape, x.stride(), name, dtype, self._index)
        if out is None:
            if stream is None:
                out = x.new_empty(shape)
            else:
                with torch.cuda.stream(stream):
                    out = x.new_empty(shape)
            return shape[1], x.data_ptr(), stride, out.data_ptr(), shape[1] * shape[2], out
        _check(out.shape == shape, f"{name}_out must have {name}'s shape")
        return shape[1], x.data_ptr(), stride, out.data_ptr(), _written_rows(out, shape, name + "_out", dtype, self._index), out
