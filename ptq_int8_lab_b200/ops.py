# -*- coding: utf-8 -*-
"""Token operators on torch CUDA tensors (C ABI: the token operators of include/ptq8.h).

The engine's arithmetic for a language model's layers: int8 activations with one scale per
token, int8 or packed int4 weights with one scale per output channel, exact int32 sums.

  ``quantize_rows``   codes and scale of each token, optionally gathered (dispatch to experts)
  ``linear``          product with one weight matrix, optional bias and SwiGLU
  ``linear_grouped``  the same with rows grouped by expert, each with its own weights

Calls enqueue on the current torch stream (or the one given) and return; nothing
synchronises or allocates except outputs that the caller does not pass.  What is refused
raises ``Ptq8Error``; tensors on the CPU are refused too.
"""
from __future__ import annotations

import ctypes
import struct
from typing import Optional, Tuple

import torch

from .engine import Ptq8Error, lib

EPI_NONE = 0
EPI_SWIGLU = 1   # weights hold gate channels, then up channels: y = silu(gate) * up

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_ROWS = struct.Struct("QqqQqQqQii")           # ptq8_rows_args
_LINEAR = struct.Struct("QqQQqqQQQqQqiiiiii")  # ptq8_linear_args

try:
    _raw_stream = torch._C._cuda_getCurrentRawStream
except AttributeError:   # a torch without CUDA
    def _raw_stream(device: int) -> int:
        return torch.cuda.current_stream(device).cuda_stream


def _matrix(name: str, t: torch.Tensor, dtypes, device: int) -> Tuple[int, int, int]:
    """(rows, columns, row pitch) of a 2-D tensor with consecutive columns."""
    if t.dtype not in dtypes:
        raise Ptq8Error(f"{name}: dtype {t.dtype}")
    if t.get_device() != device:
        raise Ptq8Error(f"{name}: on {t.device}, not on cuda:{device}")
    if t.dim() != 2:
        raise Ptq8Error(f"{name}: shape {tuple(t.shape)}, two dimensions are wanted")
    rows, cols = t.shape
    pitch, step = t.stride()
    if step != 1 and cols > 1:
        raise Ptq8Error(f"{name}: columns {step} elements apart, not consecutive")
    return rows, cols, (pitch if rows > 1 else max(cols, 1))


def _vector(name: str, t: torch.Tensor, dtype, shape, device: int) -> int:
    if t.dtype != dtype or t.shape != shape:
        raise Ptq8Error(f"{name}: {t.dtype} {tuple(t.shape)}, {dtype} {tuple(shape)} is wanted")
    if t.get_device() != device:
        raise Ptq8Error(f"{name}: on {t.device}, not on cuda:{device}")
    if not t.is_contiguous():
        raise Ptq8Error(f"{name}: not contiguous")
    return t.data_ptr()


_F32, _I32, _I8, _BYTES = torch.float32, torch.int32, (torch.int8,), (torch.uint8, torch.int8)


class Int8Ops:
    """Handle of the token operators; one per device per host thread."""

    def __init__(self, device: int = 0):
        self._h = None
        err = ctypes.create_string_buffer(1024)
        self._lib = lib()
        self._h = self._lib.ptq8_ops_create(device, err, len(err))
        if not self._h:
            raise Ptq8Error(err.value.decode(errors="replace"), 3)
        self.device = device
        self._rows_args = ctypes.create_string_buffer(_ROWS.size)
        self._linear_args = ctypes.create_string_buffer(_LINEAR.size)

    def _check(self, rc: int):
        if rc:
            raise Ptq8Error(self._lib.ptq8_ops_last_error(self._h).decode(errors="replace"), rc)

    def _stream(self, stream, given: bool) -> int:
        if stream is None:
            return _raw_stream(self.device)
        if not given:
            raise Ptq8Error("with stream, out is wanted too: a tensor made here would belong to the current stream")
        return int(getattr(stream, "cuda_stream", stream))

    def quantize_rows(self, x: torch.Tensor, rows: Optional[torch.Tensor] = None, out=None,
                      stream=None) -> Tuple[torch.Tensor, torch.Tensor]:
        """(codes int8 [R, width], scale f32 [R]) of x [T, width] (f32 / f16 / bf16):
        scale = max(max|x| / 127, 1e-8), codes = round_half_away(x / scale).

        rows (int32 [R]): output row r is token rows[r]; an index outside [0, T) gives codes 0
        and scale 0.  Codes made here have rows that start at multiples of 16 bytes."""
        n, width, ldx = _matrix("x", x, _TYPES, self.device)
        at, r = 0, n
        if rows is not None:
            r = rows.numel()
            at = _vector("rows", rows, _I32, (r,), self.device)
        if out is None:
            stream = self._stream(stream, False)
            codes = torch.empty((r, (width + 15) // 16 * 16), dtype=torch.int8, device=x.device)[:, :width]
            scale = torch.empty(r, dtype=_F32, device=x.device)
        else:
            stream = self._stream(stream, True)
            codes, scale = out
        cr, cw, ldc = _matrix("codes", codes, _I8, self.device)
        if cr != r or cw != width:
            raise Ptq8Error(f"codes: shape {(cr, cw)}, {(r, width)} is wanted")
        if r == 0:
            return codes, scale
        _ROWS.pack_into(self._rows_args, 0, x.data_ptr(), ldx, n, at, r, codes.data_ptr(), ldc,
                        _vector("scale", scale, _F32, (r,), self.device), width, _TYPES[x.dtype])
        self._check(self._lib.ptq8_quantize_rows(self._h, self._rows_args, stream))
        return codes, scale

    def _product(self, call, x, x_scale, offsets, w, w_scale, bias, bits, act, dtype, out, stream):
        d = self.device
        rows, k, ldx = _matrix("x", x, _I8, d)
        if bits != 8 and bits != 4:
            raise Ptq8Error(f"bits {bits}: 8 or 4")
        if act != EPI_NONE and act != EPI_SWIGLU:
            raise Ptq8Error(f"act {act}: EPI_NONE or EPI_SWIGLU")
        if offsets is None:
            channels, wide, ldw = _matrix("w", w, _I8 if bits == 8 else _BYTES, d)
            groups = gstride = at = 0
            shape = (channels,)
        else:
            if w.dim() != 3:
                raise Ptq8Error(f"w: shape {tuple(w.shape)}, [groups, channels, in] is wanted")
            groups = w.shape[0]
            if groups == 0:
                raise Ptq8Error("w: no groups")
            gstride = w.stride(0)
            channels, wide, ldw = _matrix("w", w[0], _I8 if bits == 8 else _BYTES, d)
            if groups == 1:
                gstride = ldw * channels
            shape = (groups, channels)
            at = _vector("offsets", offsets, _I32, (groups + 1,), d)
        if wide != (k if bits == 8 else (k + 1) // 2):
            raise Ptq8Error(f"w: rows of {wide} bytes for {k} input features at {bits} bits")
        n = channels
        if act == EPI_SWIGLU:
            if channels % 2:
                raise Ptq8Error(f"w: {channels} channels do not split into gate and up")
            n = channels // 2
        if out is None:
            stream = self._stream(stream, False)
            if dtype not in _TYPES:
                raise Ptq8Error(f"dtype {dtype}: f32, f16 or bf16")
            out = torch.empty((rows, n), dtype=dtype, device=x.device)
        else:
            stream = self._stream(stream, True)
        yr, yc, ldy = _matrix("out", out, _TYPES, d)
        if yr != rows or yc != n:
            raise Ptq8Error(f"out: shape {(yr, yc)}, {(rows, n)} is wanted")
        _LINEAR.pack_into(self._linear_args, 0, x.data_ptr(), ldx, _vector("x_scale", x_scale, _F32, (rows,), d),
                          w.data_ptr(), ldw, gstride, _vector("w_scale", w_scale, _F32, shape, d),
                          0 if bias is None else _vector("bias", bias, _F32, shape, d), out.data_ptr(), ldy, at, rows,
                          k, n, groups, bits, act, _TYPES[out.dtype])
        self._check(call(self._h, self._linear_args, stream))
        return out

    def linear(self, x: torch.Tensor, x_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
               bias: Optional[torch.Tensor] = None, bits: int = 8, act: int = EPI_NONE,
               dtype: torch.dtype = torch.bfloat16, out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
        """y [T, out] of codes x [T, in] (scale x_scale [T]) and weight codes w [channels, in] (bits 8) or
        [channels, (in + 1) // 2] (bits 4: code k in the low half of byte k // 2 for even k), scale w_scale
        [channels].  act EPI_SWIGLU: channels = 2 * out, gate then up.  dtype: of y where out is not given."""
        return self._product(self._lib.ptq8_linear, x, x_scale, None, w, w_scale, bias, bits, act, dtype, out, stream)

    def linear_grouped(self, x: torch.Tensor, x_scale: torch.Tensor, offsets: torch.Tensor, w: torch.Tensor,
                       w_scale: torch.Tensor, bias: Optional[torch.Tensor] = None, bits: int = 8,
                       act: int = EPI_NONE, dtype: torch.dtype = torch.bfloat16,
                       out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
        """linear() with rows offsets[g] .. offsets[g + 1] - 1 (int32 [groups + 1], on the device) meeting
        w[g] [channels, in], w_scale[g] and bias[g].  Rows of no group are not written."""
        if offsets is None:
            raise Ptq8Error("offsets: None")
        return self._product(self._lib.ptq8_linear_grouped, x, x_scale, offsets, w, w_scale, bias, bits, act, dtype,
                             out, stream)

    def check_device_error(self, stream=None):
        """Wait for the stream; raise Ptq8Error (status PTQ8_ERR_TIMEOUT) if a bounded device wait ran out."""
        self._check(self._lib.ptq8_ops_check_device_error(self._h, self._stream(stream, True)))

    def set_wait_test(self, wait_limit_cycles: int = 0, stall_first_load: bool = False):
        """Failure-detection test hook (see ptq8_ops_set_wait_test)."""
        self._check(self._lib.ptq8_ops_set_wait_test(self._h, int(wait_limit_cycles), 1 if stall_first_load else 0))

    def __del__(self):
        h, self._h = getattr(self, "_h", None), None
        if h:
            self._lib.ptq8_ops_destroy(h)
