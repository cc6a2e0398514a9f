# -*- coding: utf-8 -*-
"""Token operators on torch CUDA tensors (C ABI: the token operators of include/ptq8.h).

The engine's arithmetic for a language model's layers: int8 activations with one scale per
token, int8 or packed int4 weights with one scale per output channel, exact int32 sums.

  ``quantize_rows``   codes and scale of each token, optionally gathered (dispatch to experts)
  ``linear``          product with one weight matrix, optional bias and SwiGLU
  ``linear_grouped``  the same with rows grouped by expert, each with its own weights

Calls enqueue on the current torch stream (or the one given) and return; nothing
synchronises or allocates except outputs that the caller does not pass.  What is refused
raises ``Ptq8Error``; tensors on the CPU are refused too.  There are no gradients: outputs
never require one, also where an input does.
"""
from __future__ import annotations

import ctypes
import struct
from typing import NamedTuple, Optional, Tuple

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


# Calls check their tensors with inline conditions; where one fails, these say what is wrong (or return:
# a single column has no pitch to be consecutive).

def _check_matrix(name: str, t: torch.Tensor, dtypes, dims: int, device: int):
    if t.dim() != dims:
        raise Ptq8Error(f"{name}: shape {tuple(t.shape)}, {'two dimensions are' if dims == 2 else '[groups, channels, in] is'} wanted")
    if t.dtype not in dtypes:
        raise Ptq8Error(f"{name}: dtype {t.dtype}")
    if t.get_device() != device:
        raise Ptq8Error(f"{name}: on {t.device}, not on cuda:{device}")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise Ptq8Error(f"{name}: columns {t.stride(-1)} elements apart, not consecutive")


def _check_vector(name: str, t: torch.Tensor, dtype, values: int, device: int):
    if t.dtype != dtype or t.numel() != values:
        raise Ptq8Error(f"{name}: {t.dtype} {tuple(t.shape)}, {values} values of {dtype} are wanted")
    if t.get_device() != device:
        raise Ptq8Error(f"{name}: on {t.device}, not on cuda:{device}")
    if not t.is_contiguous():
        raise Ptq8Error(f"{name}: not contiguous")


_F32, _I32, _INT8 = torch.float32, torch.int32, torch.int8
_CODES = {8: (torch.int8,), 4: (torch.uint8, torch.int8)}


KERNEL_ANY, KERNEL_FEW, KERNEL_TILES = 0, 1, 2


class LinearChoice(NamedTuple):
    """What a product runs on (ptq8_linear_choice); the fields after kernel are those of KERNEL_TILES."""
    kernel: int
    variant: int
    ctas: int
    tokens: int
    w_bits: int
    epilogue: int
    split: int
    stages: int
    turns: int
    operand_tiles: int
    smem_bytes: int


def linear_variants() -> int:
    return lib().ptq8_linear_variants()


def linear_choice(rows: int, in_features: int, out_features: int, bits: int = 8, act: int = EPI_NONE, groups: int = 0,
                  variant: Optional[int] = None, split: int = 1, sms: int = 148, pitch: int = 16) -> Optional[LinearChoice]:
    """What linear() (groups 0) or linear_grouped() runs on, for rows laid at multiples of `pitch` bytes; or, with `variant`,
    that variant's launch (None: it cannot serve the call).  Needs no device."""
    wide = (in_features + 1) // 2 if bits == 4 else in_features
    ldx, ldw = (-(-v // pitch) * pitch for v in (in_features, wide))
    channels = out_features * (2 if act == EPI_SWIGLU else 1)
    at = 1 << 12   # an address that no one reads
    args = _LINEAR.pack(at, ldx, at, at, ldw, ldw * channels, at, 0, at, out_features, at if groups else 0, rows, in_features,
                        out_features, groups, bits, act, 2)
    out = (ctypes.c_int * len(LinearChoice._fields))()
    if variant is None:
        rc = lib().ptq8_linear_choose(sms, args, 1 if groups else 0, out)
    else:
        rc = lib().ptq8_linear_choose_as(sms, args, 1 if groups else 0, variant, split, out)
    if rc and variant is None:
        raise Ptq8Error("linear_choice: not a product", rc)
    return None if rc else LinearChoice(*out)


class Int8Ops:
    """Handle of the token operators; one per device per host thread.  close() (or a with block) ends it with a last check
    for device waits that ran out."""

    def __init__(self, device: int = 0):
        self._h = None
        err = ctypes.create_string_buffer(1024)
        self._lib = lib()
        self._linear, self._grouped = self._lib.ptq8_linear, self._lib.ptq8_linear_grouped
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
        d = self.device
        x_type = _TYPES.get(x.dtype)
        if x.dim() != 2:
            _check_matrix("x", x, _TYPES, 2, d)
        n, width = x.shape
        ldx, step = x.stride()
        if x_type is None or x.get_device() != d or step != 1:
            _check_matrix("x", x, _TYPES, 2, d)
        at, r = 0, n
        if rows is not None:
            r = rows.numel()
            if rows.dtype is not _I32 or not rows.is_contiguous() or rows.get_device() != d:
                _check_vector("rows", rows, _I32, r, d)
            at = rows.data_ptr()
        stream = self._stream(stream, out is not None)
        if out is None:
            codes = torch.empty((r, (width + 15) // 16 * 16), dtype=_INT8, device=x.device)[:, :width]
            scale = torch.empty(r, dtype=_F32, device=x.device)
        else:
            codes, scale = out
            if codes.dim() != 2:
                _check_matrix("codes", codes, (_INT8,), 2, d)
            c_rows, c_cols = codes.shape
            if c_rows != r or c_cols != width:
                raise Ptq8Error(f"codes: shape {tuple(codes.shape)}, {(r, width)} is wanted")
            if scale.dtype is not _F32 or scale.numel() != r or not scale.is_contiguous() or scale.get_device() != d:
                _check_vector("scale", scale, _F32, r, d)
        ldc, step = codes.stride()
        if codes.dtype is not _INT8 or codes.get_device() != d or step != 1:
            _check_matrix("codes", codes, (_INT8,), 2, d)
        if r:
            _ROWS.pack_into(self._rows_args, 0, x.data_ptr(), ldx, n, at, r, codes.data_ptr(), ldc,
                            scale.data_ptr(), width, x_type)
            rc = self._lib.ptq8_quantize_rows(self._h, self._rows_args, stream)
            if rc:
                self._check(rc)
        return codes, scale

    def _product(self, call, x, x_scale, offsets, w, w_scale, bias, bits, act, dtype, out, stream):
        d = self.device
        codes = _CODES.get(bits)
        if codes is None:
            raise Ptq8Error(f"bits {bits}: 8 or 4")
        if act != EPI_NONE and act != EPI_SWIGLU:
            raise Ptq8Error(f"act {act}: EPI_NONE or EPI_SWIGLU")
        if x.dim() != 2:
            _check_matrix("x", x, (_INT8,), 2, d)
        rows, k = x.shape
        ldx, step = x.stride()
        if x.dtype is not _INT8 or x.get_device() != d or step != 1:
            _check_matrix("x", x, (_INT8,), 2, d)
        groups = gstride = at = 0
        dims = 2 if offsets is None else 3
        if w.dim() != dims:
            _check_matrix("w", w, codes, dims, d)
        if offsets is None:
            channels, wide = w.shape
            ldw, step = w.stride()
        else:
            groups, channels, wide = w.shape
            gstride, ldw, step = w.stride()
            if groups == 0:
                raise Ptq8Error("w: no groups")
            if offsets.dtype is not _I32 or offsets.numel() != groups + 1 or not offsets.is_contiguous() or offsets.get_device() != d:
                _check_vector("offsets", offsets, _I32, groups + 1, d)
            at = offsets.data_ptr()
        if w.dtype not in codes or w.get_device() != d or step != 1:
            _check_matrix("w", w, codes, dims, d)
        if wide != (k if bits == 8 else (k + 1) // 2):
            raise Ptq8Error(f"w: rows of {wide} bytes for {k} input features at {bits} bits")
        if x_scale.dtype is not _F32 or x_scale.numel() != rows or not x_scale.is_contiguous() or x_scale.get_device() != d:
            _check_vector("x_scale", x_scale, _F32, rows, d)
        values = groups * channels if groups else channels
        if w_scale.dtype is not _F32 or w_scale.numel() != values or not w_scale.is_contiguous() or w_scale.get_device() != d:
            _check_vector("w_scale", w_scale, _F32, values, d)
        b = 0
        if bias is not None:
            if bias.dtype is not _F32 or bias.numel() != values or not bias.is_contiguous() or bias.get_device() != d:
                _check_vector("bias", bias, _F32, values, d)
            b = bias.data_ptr()
        n = channels
        if act == EPI_SWIGLU:
            if channels % 2:
                raise Ptq8Error(f"w: {channels} channels do not split into gate and up")
            n = channels // 2
        stream = self._stream(stream, out is not None)
        if out is None:
            if dtype not in _TYPES:
                raise Ptq8Error(f"dtype {dtype}: f32, f16 or bf16")
            out = torch.empty((rows, n), dtype=dtype, device=x.device)
        elif out.dim() != 2:
            _check_matrix("out", out, _TYPES, 2, d)
        y_type = _TYPES.get(out.dtype)
        y_rows, y_cols = out.shape
        ldy, step = out.stride()
        if y_type is None or step != 1 or out.get_device() != d:
            _check_matrix("out", out, _TYPES, 2, d)
        if y_rows != rows or y_cols != n:
            raise Ptq8Error(f"out: shape {tuple(out.shape)}, {(rows, n)} is wanted")
        _LINEAR.pack_into(self._linear_args, 0, x.data_ptr(), ldx, x_scale.data_ptr(), w.data_ptr(), ldw, gstride,
                          w_scale.data_ptr(), b, out.data_ptr(), ldy, at, rows, k, n, groups, bits, act,
                          y_type)
        rc = call(self._h, self._linear_args, stream)
        if rc:
            self._check(rc)
        return out

    def linear(self, x: torch.Tensor, x_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
               bias: Optional[torch.Tensor] = None, bits: int = 8, act: int = EPI_NONE,
               dtype: torch.dtype = torch.bfloat16, out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
        """y [T, out] of codes x [T, in] (scale x_scale [T]) and weight codes w [channels, in] (bits 8) or
        [channels, (in + 1) // 2] (bits 4: code k in the low half of byte k // 2 for even k), scale w_scale
        [channels].  act EPI_SWIGLU: channels = 2 * out, gate then up.  dtype: of y where out is not given."""
        return self._product(self._linear, x, x_scale, None, w, w_scale, bias, bits, act, dtype, out, stream)

    def linear_grouped(self, x: torch.Tensor, x_scale: torch.Tensor, offsets: torch.Tensor, w: torch.Tensor,
                       w_scale: torch.Tensor, bias: Optional[torch.Tensor] = None, bits: int = 8,
                       act: int = EPI_NONE, dtype: torch.dtype = torch.bfloat16,
                       out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
        """linear() with rows offsets[g] .. offsets[g + 1] - 1 (int32 [groups + 1], on the device) meeting
        w[g] [channels, in], w_scale[g] and bias[g].  Rows of no group are not written."""
        if offsets is None:
            raise Ptq8Error("offsets: None")
        return self._product(self._grouped, x, x_scale, offsets, w, w_scale, bias, bits, act, dtype,
                             out, stream)

    def check_device_error(self, stream=None):
        """Wait for the stream; raise Ptq8Error (status PTQ8_ERR_TIMEOUT) if a bounded device wait ran out."""
        self._check(self._lib.ptq8_ops_check_device_error(self._h, self._stream(stream, True)))

    def set_wait_test(self, wait_limit_cycles: int = 0, stall_first_load: bool = False):
        """Failure-detection test hook (see ptq8_ops_set_wait_test)."""
        self._check(self._lib.ptq8_ops_set_wait_test(self._h, int(wait_limit_cycles), 1 if stall_first_load else 0))

    def set_choice_test(self, variant: int = -1, split: int = 1):
        """Test hook: products run as one tile variant (see ptq8_ops_set_choice_test)."""
        self._check(self._lib.ptq8_ops_set_choice_test(self._h, int(variant), int(split)))

    def _destroy(self):
        h, self._h = getattr(self, "_h", None), None
        if h:
            self._lib.ptq8_ops_destroy(h)

    def close(self, stream=None):
        """check_device_error(), then give the handle up.  (Without it nothing is waited for: calls in flight finish, but
        a device wait of theirs that runs out is not reported.)"""
        try:
            if self._h:
                self.check_device_error(stream)
        finally:
            self._destroy()

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        self._destroy()
