# -*- coding: utf-8 -*-
"""Quantized SwiGLU MLPs on the token operators: one weight pair for every token, or experts.

    python -m ptq_int8_lab_b200.mlp [--tokens 16] [--hidden 1024] [--width 2048] [--experts 8] [--top 2] [--bits 8]

builds a dense MLP and one with experts from random weights, runs both on random hidden
states and prints how far they are from the same MLPs in float.

Weights are quantized on the host with the engine's own quantizer (one scale per output
channel, int8 or int4) and laid out once; activations are quantized per token on the way.
A dense layer is four launches, one with experts the same four between its routing and the
weighted sum of its rows.  No gradient passes through them.
"""
from __future__ import annotations

import argparse
from typing import Optional, Tuple

import numpy as np
import torch

from . import engine as E
from .ops import EPI_SWIGLU, Int8Ops
from .package import pack_w4


def lay_weights(w, bits: int = 8, device: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
    """(codes, scale) on the device of float weights [..., channels, in]: int8 codes [..., channels, in] or int4
    codes two per byte [..., channels, (in + 1) // 2], rows at multiples of 16 bytes; scale f32 [..., channels]."""
    if bits not in (4, 8):
        raise E.Ptq8Error(f"bits {bits}: 8 or 4")
    w = np.asarray(w, dtype=np.float32)
    if w.ndim < 2:
        raise E.Ptq8Error(f"weights of shape {w.shape}: [..., channels, in] is wanted")
    codes, scale = E.quantize_weight(w.reshape(-1, w.shape[-1]), bits)
    rows = pack_w4(codes) if bits == 4 else codes
    pitch = (rows.shape[1] + 15) // 16 * 16
    laid = torch.zeros((rows.shape[0], pitch), dtype=torch.uint8 if bits == 4 else torch.int8, device=f"cuda:{device}")
    laid[:, :rows.shape[1]] = torch.from_numpy(np.ascontiguousarray(rows)).to(laid.device)
    laid = laid.view(*w.shape[:-1], pitch)[..., :rows.shape[1]]
    return laid, torch.from_numpy(scale).view(*w.shape[:-1]).to(laid.device)


class Int8MLP:
    """y = (silu(x Wg^T) * (x Wu^T)) Wd^T with int8 activations per token.

    gate_up [2 * width, hidden] (gate rows, then up rows), down [hidden, width], float."""

    def __init__(self, gate_up, down, bits: int = 8, device: int = 0, ops: Optional[Int8Ops] = None):
        self.ops = ops or Int8Ops(device)
        self.bits = bits
        self.gate_up = lay_weights(gate_up, bits, self.ops.device)
        self.down = lay_weights(down, bits, self.ops.device)

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        o = self.ops
        codes, scale = o.quantize_rows(x)
        h = o.linear(codes, scale, *self.gate_up, bits=self.bits, act=EPI_SWIGLU, dtype=x.dtype)
        codes, scale = o.quantize_rows(h)
        return o.linear(codes, scale, *self.down, bits=self.bits, dtype=x.dtype)


class Int8Experts:
    """The same with `experts` weight pairs: a token's `top` best experts by its router logits, weighted by
    the softmax over them.  router [experts, hidden], gate_up [experts, 2 * width, hidden], down [experts, hidden,
    width], float.  Nothing waits for the host: the experts' row counts stay on the device."""

    def __init__(self, router, gate_up, down, top: int, bits: int = 8, device: int = 0, ops: Optional[Int8Ops] = None):
        self.ops = ops or Int8Ops(device)
        self.bits, self.top = bits, top
        self.router = torch.as_tensor(np.asarray(router, dtype=np.float32), device=f"cuda:{self.ops.device}")
        if not 1 <= top <= self.router.shape[0]:
            raise E.Ptq8Error(f"top {top} of {self.router.shape[0]} experts")
        self.gate_up = lay_weights(gate_up, bits, self.ops.device)
        self.down = lay_weights(down, bits, self.ops.device)
        self.first = torch.arange(self.router.shape[0] + 1, dtype=torch.int64, device=self.router.device)

    def route(self, x: torch.Tensor):
        """(weights [T, top], rows: the token of each row in expert order, offsets, where: the row of each choice)."""
        best, ids = torch.topk(x.float() @ self.router.t(), self.top, dim=1)
        ids = ids.reshape(-1)
        sorted_ids, order = torch.sort(ids, stable=True)
        offsets = torch.searchsorted(sorted_ids, self.first).to(torch.int32)
        where = torch.empty_like(order)
        where[order] = torch.arange(order.numel(), device=order.device)
        rows = torch.div(order, self.top, rounding_mode="floor").to(torch.int32)
        return torch.softmax(best, dim=1), rows, offsets, where

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        o = self.ops
        weight, rows, offsets, where = self.route(x)
        codes, scale = o.quantize_rows(x, rows=rows)
        h = o.linear_grouped(codes, scale, offsets, *self.gate_up, bits=self.bits, act=EPI_SWIGLU, dtype=x.dtype)
        codes, scale = o.quantize_rows(h)
        y = o.linear_grouped(codes, scale, offsets, *self.down, bits=self.bits, dtype=torch.float32)
        y = y[where].view(x.shape[0], self.top, y.shape[1])
        return (y * weight[..., None]).sum(dim=1).to(x.dtype)


def _float_mlp(x, gate_up, down):
    g, u = (x @ gate_up.t()).chunk(2, dim=1)
    return (torch.nn.functional.silu(g) * u) @ down.t()


def main(argv=None) -> Tuple[float, float]:
    """Runs both; returns the relative differences from float (dense, experts)."""
    ap = argparse.ArgumentParser(description="Dense and expert MLPs with int8 activations, against float.")
    for name, value in (("tokens", 16), ("hidden", 1024), ("width", 2048), ("experts", 8), ("top", 2), ("bits", 8), ("seed", 0)):
        ap.add_argument("--" + name, type=int, default=value)
    a = ap.parse_args(argv)
    rng = np.random.default_rng(a.seed)
    w1 = (rng.normal(0, 1, (a.experts, 2 * a.width, a.hidden)) / np.sqrt(a.hidden)).astype(np.float32)
    w2 = (rng.normal(0, 1, (a.experts, a.hidden, a.width)) / np.sqrt(a.width)).astype(np.float32)
    router = (rng.normal(0, 1, (a.experts, a.hidden)) / np.sqrt(a.hidden)).astype(np.float32)
    x = torch.from_numpy(rng.normal(0, 1, (a.tokens, a.hidden)).astype(np.float32)).cuda()
    ops = Int8Ops(0)
    got = Int8MLP(w1[0], w2[0], a.bits, ops=ops)(x)
    f1, f2 = torch.from_numpy(w1).cuda(), torch.from_numpy(w2).cuda()
    want = _float_mlp(x, f1[0], f2[0])
    dense = float((got - want).norm() / want.norm())
    print(f"dense: {a.tokens} tokens, {a.hidden} -> 2 x {a.width} -> {a.hidden}, W{a.bits}A8: "
          f"relative difference from float {dense:.4f}")
    moe = Int8Experts(router, w1, w2, a.top, a.bits, ops=ops)
    got = moe(x)
    p, ids = torch.topk(x @ moe.router.t(), a.top, dim=1)
    p = torch.softmax(p, dim=1)
    want = torch.stack([sum(p[t, j] * _float_mlp(x[t:t + 1], f1[e], f2[e])[0] for j, e in enumerate(ids[t].tolist()))
                        for t in range(a.tokens)])
    ops.check_device_error()
    experts = float((got - want).norm() / want.norm())
    print(f"experts: top {a.top} of {a.experts}: relative difference from float {experts:.4f}")
    return dense, experts


if __name__ == "__main__":
    main()
