# -*- coding: utf-8 -*-
"""Token operators on torch CUDA tensors (C ABI: the token operators of include/ptq8.h).

The engine's arithmetic for a language model's layers: int8 activations with one scale per
token, int8 or packed int4 weights with one scale per output channel, exact int32 sums.

  ``quantize_rows``   codes and scale of each token, optionally gathered (dispatch to experts)
  ``linear``          product with one weight matrix, optional bias and SwiGLU
  ``linear_grouped``  the same with rows grouped by expert, each with its own weights

And generation with 4 bits, activations kept as floats:

  ``linear_w4``       product with 4-bit weights that have a scale per group of input features
  ``cache_write``     keys and values of new tokens into a paged cache of 4-bit codes (``Cache4``, ``new_cache``)
  ``cache_read``      the floats that stand there
  ``cache_attention`` attention over it, causal, from one new token per sequence to pieces of prompts

Calls enqueue on the current torch stream (or the one given) and return; nothing
synchronises or allocates except outputs that the caller does not pass.  What is refused
raises ``Ptq8Error``; tensors on the CPU are refused too.  There are no gradients: outputs
never require one, also where an input does.
"""
from __future__ import annotations

import ctypes
import importlib.util
import struct
from functools import cached_property
from typing import NamedTuple, Optional, Tuple

import torch

from .engine import Ptq8Error, lib

EPI_NONE = 0
EPI_SWIGLU = 1   # weights hold gate channels, then up channels: y = silu(gate) * up

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_ROWS = struct.Struct("QqqQqQqQii")           # ptq8_rows_args
_LINEAR = struct.Struct("QqQQqqQQQqQqiiiiii")  # ptq8_linear_args
_W4 = struct.Struct("QqQqQqQQqqiiiiiiii")      # ptq8_linear_w4_args
_CACHE = "QQQQqqqqqqqqQqQQqiiiiii"             # ptq8_cache
_CACHE_ROWS = struct.Struct(_CACHE + "QQqqqqqii")       # ptq8_cache_rows_args
_ATTENTION = struct.Struct(_CACHE + "QQqqqqqQqfiii")    # ptq8_cache_attention_args

try:
    _raw_stream = torch._C._cuda_getCurrentRawStream
except AttributeError:   # a torch without CUDA
    def _raw_stream(device: int) -> int:
        return torch.cuda.current_stream(device).cuda_stream


_host = None


def _host_module():
    """ptq8_host: the calls of linear_w4 and the cache operators without the interpreter's share (built beside libptq8.so against the
    installed torch).  Loaded at their first call; the operators that do without it never look for it."""
    global _host
    if _host is None:
        from .build import HOST
        if not HOST.exists():
            raise Ptq8Error(f"{HOST} not found: build it with `python -m ptq_int8_lab_b200.build`")
        spec = importlib.util.spec_from_file_location("ptq8_host", HOST)
        try:
            module = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(module)
        except ImportError as e:
            raise Ptq8Error(f"{HOST} does not fit this Python or torch ({e}): build it with `python -m ptq_int8_lab_b200.build`") from e
        L = lib()
        module.entries(*(ctypes.cast(f, ctypes.c_void_p).value for f in
                         (L.ptq8_cache_write, L.ptq8_cache_read, L.ptq8_cache_attention, L.ptq8_cache_attention_workspace, L.ptq8_linear_w4)))
        _host = module
    return _host


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


_F32, _I32, _INT8, _U8, _BF16 = torch.float32, torch.int32, torch.int8, torch.uint8, torch.bfloat16
_WORKSPACE = struct.Struct("Qq")
_WORKSPACE_AT = struct.calcsize("@" + _CACHE + "QQqqqqq")   # its place in ptq8_cache_attention_args
_CODES = {8: (torch.int8,), 4: (torch.uint8, torch.int8)}


class Cache4(NamedTuple):
    """Keys and values of one layer in 4 bits: pages of `page` tokens, for each head of a page its rows one after another.

    Codes are two per byte, the even one low; scales are (step, least) pairs: code c stands for least + step * c."""
    k: torch.Tensor         # uint8 [pages, kv_heads, page, head_dim // 2]
    k_scale: torch.Tensor   # bf16 [pages, kv_heads, page, 2]
    v: torch.Tensor
    v_scale: torch.Tensor


def new_cache(pages: int, kv_heads: int, head_dim: int, page: int = 64, device: int = 0) -> Cache4:
    """An empty Cache4: zeros stand for zeros."""
    def part(n, dtype):
        return torch.zeros((pages, kv_heads, page, n), dtype=dtype, device=f"cuda:{device}")
    return Cache4(part(head_dim // 2, torch.uint8), part(2, torch.bfloat16), part(head_dim // 2, torch.uint8), part(2, torch.bfloat16))


def _check_part(name: str, t: torch.Tensor, dtype, shape, device: int):
    if t.dtype != dtype or tuple(t.shape) != shape:
        raise Ptq8Error(f"cache.{name}: {t.dtype} {tuple(t.shape)}, {dtype} {shape} is wanted")
    if t.get_device() != device:
        raise Ptq8Error(f"cache.{name}: on {t.device}, not on cuda:{device}")
    if t.stride(3) != 1 or t.stride(2) != shape[3]:
        raise Ptq8Error(f"cache.{name}: a head's rows of a page are not consecutive")


def _check_rows(name: str, t: torch.Tensor, dtypes, shape, device: int):
    if t.dtype not in dtypes:
        raise Ptq8Error(f"{name}: dtype {t.dtype}")
    if t.dim() != 3 or tuple(t.shape) != shape:
        raise Ptq8Error(f"{name}: shape {tuple(t.shape)}, {shape} is wanted")
    if t.get_device() != device:
        raise Ptq8Error(f"{name}: on {t.device}, not on cuda:{device}")
    if t.stride(2) != 1:
        raise Ptq8Error(f"{name}: columns {t.stride(2)} elements apart, not consecutive")


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
        self._w4_args = ctypes.create_string_buffer(_W4.size)
        self._cache_args = ctypes.create_string_buffer(_CACHE_ROWS.size)
        self._attention_args = ctypes.create_string_buffer(_ATTENTION.size)
        self._linear_w4, self._cache_write, self._cache_read = self._lib.ptq8_linear_w4, self._lib.ptq8_cache_write, self._lib.ptq8_cache_read
        self._cache_attention = self._lib.ptq8_cache_attention
        self._workspaces = {}   # bytes, by the sizes of a call

    @cached_property
    def _host_rows(self):
        return _host_module().cache_rows

    @cached_property
    def _host_attention(self):
        return _host_module().cache_attention

    @cached_property
    def _host_w4(self):
        return _host_module().linear_w4

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

    def linear_w4(self, x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, group: int, bias: Optional[torch.Tensor] = None,
                  act: int = EPI_NONE, dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
        """y [T, out] of float activations x [T, in] (f32 / f16 / bf16) and 4-bit weight codes w [channels, (in + 1) // 2] (code k in the
        low half of byte k // 2 for even k) with a scale per `group` consecutive input features: w_scale [channels,
        ceil(in / group)] (f32 / f16 / bf16).  act EPI_SWIGLU: channels = 2 * out, gate then up.  dtype: of y where out is not given
        (None: x's).  For generation: one to some tens of tokens."""
        d = self.device
        if out is not None and stream is None:
            rc = self._host_w4(self._h, d, x, w, w_scale, group, bias, act, out, _raw_stream(d))
            if rc == 0:
                return out
            if rc > 0:
                self._check(rc)
        # (out of the ordinary: one look after another, and what is wrong is said)
        if act != EPI_NONE and act != EPI_SWIGLU:
            raise Ptq8Error(f"act {act}: EPI_NONE or EPI_SWIGLU")
        if not 0 < group <= 0x7FFFFFFF:
            raise Ptq8Error(f"group {group}")
        x_type, s_type = _TYPES.get(x.dtype), _TYPES.get(w_scale.dtype)
        if x_type is None or x.dim() != 2 or x.get_device() != d:
            _check_matrix("x", x, _TYPES, 2, d)
        if w.dtype not in _CODES[4] or w.dim() != 2 or w.get_device() != d:
            _check_matrix("w", w, _CODES[4], 2, d)
        if s_type is None or w_scale.dim() != 2 or w_scale.get_device() != d:
            _check_matrix("w_scale", w_scale, _TYPES, 2, d)
        rows, k = x.shape
        channels, wide = w.shape
        ldx, x_step = x.stride()
        ldw, w_step = w.stride()
        lds, s_step = w_scale.stride()
        if x_step != 1 or w_step != 1 or s_step != 1:
            for name, t, dtypes in (("x", x, _TYPES), ("w", w, _CODES[4]), ("w_scale", w_scale, _TYPES)):
                _check_matrix(name, t, dtypes, 2, d)
        if wide != (k + 1) // 2:
            raise Ptq8Error(f"w: rows of {wide} bytes for {k} input features at 4 bits")
        if w_scale.shape != (channels, -(-k // group)):
            raise Ptq8Error(f"w_scale: shape {tuple(w_scale.shape)}, {(channels, -(-k // group))} is wanted")
        b = 0
        if bias is not None:
            if bias.dtype is not _F32 or bias.numel() != channels or not bias.is_contiguous() or bias.get_device() != d:
                _check_vector("bias", bias, _F32, channels, d)
            b = bias.data_ptr()
        n = channels
        if act == EPI_SWIGLU:
            if channels % 2:
                raise Ptq8Error(f"w: {channels} channels do not split into gate and up")
            n = channels // 2
        stream = self._stream(stream, out is not None)
        if out is None:
            dtype = dtype or x.dtype
            if dtype not in _TYPES:
                raise Ptq8Error(f"dtype {dtype}: f32, f16 or bf16")
            out = torch.empty((rows, n), dtype=dtype, device=x.device)
        elif out.dim() != 2:
            _check_matrix("out", out, _TYPES, 2, d)
        y_type = _TYPES.get(out.dtype)
        ldy, step = out.stride()
        if y_type is None or step != 1 or out.get_device() != d:
            _check_matrix("out", out, _TYPES, 2, d)
        if out.shape != (rows, n):
            raise Ptq8Error(f"out: shape {tuple(out.shape)}, {(rows, n)} is wanted")
        _W4.pack_into(self._w4_args, 0, x.data_ptr(), ldx, w.data_ptr(), ldw, w_scale.data_ptr(), lds, b, out.data_ptr(), ldy, rows, k, n,
                      group, act, x_type, s_type, y_type, 0)
        rc = self._linear_w4(self._h, self._w4_args, stream)
        if rc:
            self._check(rc)
        return out

    def _cache(self, cache, table, lengths, starts, tokens):
        """The fields of ptq8_cache.  tokens: the new tokens."""
        k, ks, v, vs = cache
        d = self.device
        shape = k.shape
        if len(shape) != 4:
            raise Ptq8Error(f"cache.k: shape {tuple(shape)}, [pages, kv_heads, page, head_dim // 2] is wanted")
        pages, heads, page, half = shape
        pairs = (pages, heads, page, 2)
        k_at, v_at, ks_at, vs_at = k.stride(), v.stride(), ks.stride(), vs.stride()
        # one look at all that is wanted of the four; where it fails, _check_part says what is wrong
        if not (k.dtype is _U8 and v.dtype is _U8 and ks.dtype is _BF16 and vs.dtype is _BF16 and v.shape == shape and ks.shape == pairs
                and vs.shape == pairs and k_at[2:] == (half, 1) and v_at[2:] == (half, 1) and ks_at[2:] == (2, 1) and vs_at[2:] == (2, 1)
                and k.get_device() == d and v.get_device() == d and ks.get_device() == d and vs.get_device() == d):
            for name, t, dtype, want in (("k", k, _U8, tuple(shape)), ("v", v, _U8, tuple(shape)), ("k_scale", ks, _BF16, pairs), ("v_scale", vs, _BF16, pairs)):
                _check_part(name, t, dtype, want, d)
        shape = table.shape
        if len(shape) != 2:
            _check_matrix("table", table, (_I32,), 2, d)
        seqs, wide = shape
        pitch, step = table.stride()
        if table.dtype is not _I32 or step != 1 or table.get_device() != d:
            _check_matrix("table", table, (_I32,), 2, d)
        if lengths.dtype is not _I32 or lengths.numel() != seqs or not lengths.is_contiguous() or lengths.get_device() != d:
            _check_vector("lengths", lengths, _I32, seqs, d)
        at = 0
        if starts is not None:
            if starts.dtype is not _I32 or starts.numel() != seqs + 1 or not starts.is_contiguous() or starts.get_device() != d:
                _check_vector("starts", starts, _I32, seqs + 1, d)
            at = starts.data_ptr()
        elif tokens != seqs:
            raise Ptq8Error(f"{tokens} tokens without starts, but {seqs} sequences")
        return (k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), k_at[0], k_at[1], v_at[0], v_at[1], 2 * ks_at[0], 2 * ks_at[1],
                2 * vs_at[0], 2 * vs_at[1], table.data_ptr(), pitch, lengths.data_ptr(), at, pages, wide, page, heads, 2 * half, seqs, 0)

    def _cache_rows(self, call, cache, k, v, table, lengths, starts, stream):
        shape = k.shape
        if len(shape) != 3:
            raise Ptq8Error(f"k: shape {tuple(shape)}, [tokens, kv_heads, head_dim] is wanted")
        tokens = shape[0]
        fields = self._cache(cache, table, lengths, starts, tokens)
        d, dtype = self.device, k.dtype
        kind, want = _TYPES.get(dtype), (tokens, fields[19], fields[20])
        if kind is None or shape != want or k.get_device() != d:
            _check_rows("k", k, _TYPES, want, d)
        if v.dtype is not dtype or v.shape != want or v.get_device() != d:
            _check_rows("v", v, (dtype,), want, d)
        k_token, k_head, k_step = k.stride()
        v_token, v_head, v_step = v.stride()
        if k_step != 1 or v_step != 1:
            _check_rows("k", k, (dtype,), want, d)
            _check_rows("v", v, (dtype,), want, d)
        _CACHE_ROWS.pack_into(self._cache_args, 0, *fields, k.data_ptr(), v.data_ptr(), k_token, k_head, v_token, v_head, tokens, kind, 0)
        rc = call(self._h, self._cache_args, stream)
        if rc:
            self._check(rc)

    def cache_write(self, cache: Cache4, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor,
                    starts: Optional[torch.Tensor] = None, stream=None) -> None:
        """Keys and values k, v [T, kv_heads, head_dim] (f32 / f16 / bf16) of new tokens into the cache, in 4 bits.

        table int32 [sequences, n]: the pages of each sequence; lengths int32 [sequences]: its positions, the new tokens (its
        last ones) among them; starts int32 [sequences + 1]: sequence b's new tokens are starts[b] .. starts[b + 1] - 1, without
        it token b alone.  Positions without a page are skipped.  A page that is written belongs to one sequence."""
        if stream is None:
            rc = self._host_rows(True, self._h, self.device, cache, k, v, table, lengths, starts, _raw_stream(self.device))
            if rc == 0:
                return
            if rc > 0:
                self._check(rc)
        self._cache_rows(self._cache_write, cache, k, v, table, lengths, starts, self._stream(stream, True))

    def cache_read(self, cache: Cache4, table: torch.Tensor, lengths: torch.Tensor, starts: Optional[torch.Tensor] = None,
                   tokens: Optional[int] = None, dtype: torch.dtype = torch.bfloat16, out=None, stream=None) -> Tuple[torch.Tensor, torch.Tensor]:
        """(k, v) [T, kv_heads, head_dim] that the cache holds at the positions where cache_write with the same arguments
        writes; zeros where a position has no page.  With starts and without out, tokens is T.  Rows of no sequence are not
        written."""
        if out is not None and stream is None:
            k, v = out
            rc = self._host_rows(False, self._h, self.device, cache, k, v, table, lengths, starts, _raw_stream(self.device))
            if rc == 0:
                return k, v
            if rc > 0:
                self._check(rc)
        stream = self._stream(stream, out is not None)
        if out is None:
            if dtype not in _TYPES:
                raise Ptq8Error(f"dtype {dtype}: f32, f16 or bf16")
            if tokens is None:
                if starts is not None:
                    raise Ptq8Error("tokens: None; with starts and without out it tells how many there are")
                tokens = table.shape[0]
            shape = (tokens, cache[0].shape[1], 2 * cache[0].shape[3])
            out = tuple(torch.empty(shape, dtype=dtype, device=f"cuda:{self.device}") for _ in range(2))
        k, v = out
        self._cache_rows(self._cache_read, cache, k, v, table, lengths, starts, stream)
        return k, v

    def cache_attention(self, q: torch.Tensor, cache: Cache4, table: torch.Tensor, lengths: torch.Tensor,
                        starts: Optional[torch.Tensor] = None, scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                        workspace: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
        """softmax(scale * q k^T) v of queries q [T, heads, head_dim] (f16 / bf16) over the cache, causal: a token sees the positions
        of its sequence up to its own.  table, lengths, starts as in cache_write (which comes first: the new tokens attend to
        themselves too).  heads is a multiple of the cache's kv_heads; scale: head_dim ** -0.5 where not given.  A token that sees
        nothing gets zeros; tokens of no sequence are not written.

        workspace: uint8, cache_attention_workspace() bytes; one is made where it is not given, which with stream it has to be."""
        if stream is not None and (out is None or workspace is None):
            raise Ptq8Error("with stream, out and workspace are wanted too: tensors made here would belong to the current stream")
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        if stream is None and workspace is None:
            rc = self._host_attention(self._h, self.device, q, cache, table, lengths, starts, scale, out, _raw_stream(self.device))
            if rc == 0:
                return out
            if rc > 0:
                self._check(rc)
        stream = self._stream(stream, True)
        need = self._attention(q, cache, table, lengths, starts, scale, out)
        if workspace is None:
            at, size = 0, 0
            if need:
                workspace = torch.empty(need, dtype=_U8, device=q.device)
                at, size = workspace.data_ptr(), need
        else:
            if workspace.dtype is not _U8 or not workspace.is_contiguous() or workspace.get_device() != self.device:
                raise Ptq8Error(f"workspace: {workspace.dtype} on {workspace.device}, consecutive uint8 on cuda:{self.device} is wanted")
            at, size = workspace.data_ptr(), workspace.numel()
        args = self._attention_args
        _WORKSPACE.pack_into(args, _WORKSPACE_AT, at, size)
        rc = self._cache_attention(self._h, args, stream)
        if rc:
            self._check(rc)
        return out

    def _attention(self, q, cache, table, lengths, starts, scale, out) -> int:
        """Fills the argument struct, all but its workspace; the bytes that that needs."""
        shape = q.shape
        if len(shape) != 3:
            raise Ptq8Error(f"q: shape {tuple(shape)}, [tokens, heads, head_dim] is wanted")
        d = self.device
        tokens, heads, dim = shape
        fields = self._cache(cache, table, lengths, starts, tokens)
        dtype = q.dtype
        kind = _TYPES.get(dtype)
        if not kind or dim != fields[20] or q.get_device() != d:
            _check_rows("q", q, (torch.float16, _BF16), (tokens, heads, fields[20]), d)
        if out.dtype is not dtype or out.shape != shape or out.get_device() != d:
            _check_rows("out", out, (dtype,), tuple(shape), d)
        q_token, q_head, q_step = q.stride()
        o_token, o_head, o_step = out.stride()
        if q_step != 1 or o_step != 1:
            _check_rows("q", q, (dtype,), tuple(shape), d)
            _check_rows("out", out, (dtype,), tuple(shape), d)
        args = self._attention_args
        _ATTENTION.pack_into(args, 0, *fields, q.data_ptr(), out.data_ptr(), q_token, q_head, o_token, o_head, tokens, 0, 0,
                             dim ** -0.5 if scale is None else scale, heads, kind, 0)
        # a function of these numbers alone, asked for once
        key = (tokens, heads, fields[19], dim, fields[21], starts is None)
        need = self._workspaces.get(key)
        if need is None:
            need = self._lib.ptq8_cache_attention_workspace(self._h, args)
            if need < 0:
                self._check(1)
            if len(self._workspaces) >= 4096:
                self._workspaces.clear()
            self._workspaces[key] = need
        return need

    def cache_attention_workspace(self, q: torch.Tensor, cache: Cache4, table: torch.Tensor, lengths: torch.Tensor,
                                  starts: Optional[torch.Tensor] = None) -> int:
        """Bytes of workspace that cache_attention() needs for tensors of these shapes.  A workspace serves one call at a time."""
        return self._attention(q, cache, table, lengths, starts, None, q)

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
