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
from magpie_tts_rt_b200.paged_cache import _DTYPES, HEAD_DIMS, MAX_ROWS, _check, _raw_stream, _rows_of

MAX_HEADS = 1 << 16


class Rotation:
    def __init__(self, head_dim: int, rotary_dim: Optional[int] = None, base: float = 10000.0, interleaved: bool = False,
                 frequencies: Optional[torch.Tensor] = None, q_norm: Optional[torch.Tensor] = None,
                 k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6, device="cuda"):
        """rotary_dim (a multiple of 16, all of head_dim if not given) dims of a
        head are turned, pair i by base^(-2 i / rotary_dim) radians a position, or
        by frequencies [rotary_dim / 2] (any real type).  q_norm, k_norm [head_dim]:
        weights of the norms.  All of it is copied: later changes of the tensors do
        not reach the rotation."""
        _check(head_dim in HEAD_DIMS, f"head_dim must be one of {HEAD_DIMS}")
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        _check(16 <= rotary_dim <= head_dim and rotary_dim % 16 == 0, "rotary_dim must be a multiple of 16, at most head_dim")
        _check(eps >= 0 and math.isfinite(eps), "eps must not be negative")
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
        otherwise they must not overlap what the call reads."""
        _check(q is not None or k is not None, "a rotation needs queries or keys")
        first = q if q is not None else k
        dtype, index = first.dtype, first.get_device()
        _check(dtype in _DTYPES, "q and k must be bfloat16 or float16")
        _check(index == self._index, "q and k must be on the rotation's device")
        _check(first.dim() == 3, "q and k must be [rows, heads, head_dim]")
        rows = first.shape[0]
        _check(rows <= MAX_ROWS, f"at most {MAX_ROWS} rows")
        if positions.dtype is not torch.int32 or positions.shape != (rows,) or positions.get_device() != index or \
                not positions.is_contiguous():
            raise ValueError(f"positions must be a contiguous int32 vector of {rows} on the rotation's device")
        args = L.RotateRows()
        args.rows, args.positions = rows, positions.data_ptr()
        if stream is None:
            handle, ctx = self._raw(index), None
        else:
            _check(stream.device.index == index, "the stream belongs to another device than the rotation")
            handle, ctx = stream.cuda_stream, torch.cuda.stream(stream)
        outs = []
        for name, x, out in (("q", q, q_out), ("k", k, k_out)):
            if x is None:
                _check(out is None, f"{name}_out without {name}")
                outs.append(None)
                continue
            _check(x.dim() == 3 and x.shape[0] == rows and x.shape[2] == self.head_dim and x.shape[1] <= MAX_HEADS,
                   "q and k must be [rows, heads, head_dim]")
            stride = _rows_of(x, x.shape, x.stride(), name, dtype, index)
            if out is None:
                if ctx is None:
                    out = torch.empty(x.shape, dtype=dtype, device=self.device)
                else:
                    with ctx:
                        out = torch.empty(x.shape, dtype=dtype, device=self.device)
            else:
                _check(out.shape == x.shape, f"{name}_out must have {name}'s shape")
            out_stride = _rows_of(out, x.shape, out.stride(), name + "_out", dtype, index)
            if name == "q":
                args.q_heads, args.q, args.q_row_stride = x.shape[1], x.data_ptr(), stride
                args.q_out, args.q_out_row_stride = out.data_ptr(), out_stride
            else:
                args.kv_heads, args.k, args.k_row_stride = x.shape[1], x.data_ptr(), stride
                args.k_out, args.k_out_row_stride = out.data_ptr(), out_stride
            outs.append(out)
        self._on_stream(handle, stream)
        call = L.lib.mtt_b200_launch_rotate_heads
        if _cache._current_device() == index:
            rc = call(self._c[dtype][1], ctypes.byref(args), handle)
        else:
            with torch.cuda.device(index):
                rc = call(self._c[dtype][1], ctypes.byref(args), handle)
        if rc != L.STATUS_OK:
            raise RuntimeError(f"mtt_b200_launch_rotate_heads failed with status {rc}")
        return tuple(outs)
