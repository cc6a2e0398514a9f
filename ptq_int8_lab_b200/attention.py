# -*- coding: utf-8 -*-
"""Attention of a language model's layer in 4 bits: projections with grouped 4-bit weights, keys and values in a 4-bit cache.

    python -m ptq_int8_lab_b200.attention [--sequences 4] [--prompt 200] [--steps 8] [--hidden 1024] [--heads 16]
                                          [--kv-heads 4] [--group 64]

writes random prompts into a layer's cache in one call, generates tokens of random hidden states one at
a time, and prints how far the layer's outputs are from the same layer in float.

A step of one token per sequence is five launches: projection, cache, attention and the joining of its parts, projection.
Lengths and tables stay on the device, so that a captured graph of a step serves every step.
"""
from __future__ import annotations

import argparse
from typing import Callable, Optional, Tuple

import numpy as np
import torch

from .engine import Ptq8Error
from .mlp import lay_groups
from .ops import Int8Ops, new_cache


class Int4Attention:
    """y = softmax(q k^T / sqrt(d)) v Wo^T, (q, k, v) = x Wqkv^T, causal, over the sequences' cached keys and values.

    qkv [(heads + 2 * kv_heads) * head_dim, hidden] (queries, keys, values; a head's rows together), out [hidden, heads *
    head_dim], float.  pages: of the layer's cache, of `page` tokens each."""

    def __init__(self, qkv, out, heads: int, kv_heads: int, pages: int, page: int = 64, group: int = 128, device: int = 0,
                 ops: Optional[Int8Ops] = None):
        self.ops = ops or Int8Ops(device)
        self.heads, self.kv_heads, self.group = heads, kv_heads, group
        qkv = np.asarray(qkv, dtype=np.float32)
        if heads <= 0 or kv_heads <= 0 or qkv.shape[0] % (heads + 2 * kv_heads):
            raise Ptq8Error(f"qkv of {qkv.shape[0]} rows for {heads} heads and 2 x {kv_heads} of keys and values")
        self.head_dim = qkv.shape[0] // (heads + 2 * kv_heads)
        self.qkv = lay_groups(qkv, group, self.ops.device)
        self.out = lay_groups(out, group, self.ops.device)
        self.cache = new_cache(pages, kv_heads, self.head_dim, page, self.ops.device)

    def __call__(self, x: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, starts: Optional[torch.Tensor] = None,
                 rotate: Optional[Callable[[torch.Tensor, torch.Tensor], Tuple[torch.Tensor, torch.Tensor]]] = None) -> torch.Tensor:
        """x [T, hidden] (f16 / bf16): the new tokens of all sequences; table, lengths, starts as Int8Ops.cache_write has them
        (lengths with the new tokens).  rotate: what a model does to queries and keys before they meet, (q, k) -> (q, k)."""
        o, h, kv = self.ops, self.heads, self.kv_heads
        both = o.linear_w4(x, *self.qkv, self.group).view(x.shape[0], h + 2 * kv, self.head_dim)
        q, k, v = both[:, :h], both[:, h:h + kv], both[:, h + kv:]
        if rotate is not None:
            q, k = rotate(q, k)
        o.cache_write(self.cache, k, v, table, lengths, starts)
        y = o.cache_attention(q, self.cache, table, lengths, starts)
        return o.linear_w4(y.view(x.shape[0], h * self.head_dim), *self.out, self.group)


def _float_layer(x, qkv, out, heads, kv_heads, new):
    """The same for one sequence in float: outputs of its last `new` positions."""
    n, d = x.shape[0], qkv.shape[0] // (heads + 2 * kv_heads)
    both = (x @ qkv.t()).view(n, heads + 2 * kv_heads, d)
    q, k, v = both[-new:, :heads], both[:, heads:heads + kv_heads], both[:, heads + kv_heads:]
    k, v = (t.repeat_interleave(heads // kv_heads, dim=1) for t in (k, v))
    z = torch.einsum("ihd,jhd->hij", q, k) * d ** -0.5
    seen = torch.arange(n, device=x.device)[None] <= torch.arange(n - new, n, device=x.device)[:, None]
    p = torch.softmax(z.masked_fill(~seen, float("-inf")), dim=-1)
    return torch.einsum("hij,jhd->ihd", p, v).reshape(new, heads * d) @ out.t()


def main(argv=None) -> Tuple[float, float]:
    """Runs prompts and steps; returns the relative differences from float (prompts, steps)."""
    ap = argparse.ArgumentParser(description="An attention layer with 4-bit weights and a 4-bit cache, against float.")
    for name, value in (("sequences", 4), ("prompt", 200), ("steps", 8), ("hidden", 1024), ("heads", 16), ("kv-heads", 4), ("head-dim", 64),
                        ("group", 64), ("page", 64), ("seed", 0)):
        ap.add_argument("--" + name, type=int, default=value)
    a = ap.parse_args(argv)
    rng = np.random.default_rng(a.seed)
    qkv = (rng.normal(0, 1, ((a.heads + 2 * a.kv_heads) * a.head_dim, a.hidden)) / np.sqrt(a.hidden)).astype(np.float32)
    out = (rng.normal(0, 1, (a.hidden, a.heads * a.head_dim)) / np.sqrt(a.heads * a.head_dim)).astype(np.float32)
    prompts = [max(1, a.prompt * (i + 1) // a.sequences) for i in range(a.sequences)]   # of differing lengths
    each = -(-(a.prompt + a.steps) // a.page)
    layer = Int4Attention(qkv, out, a.heads, a.kv_heads, a.sequences * each, a.page, a.group)
    table = torch.from_numpy(rng.permutation(a.sequences * each).astype(np.int32)).view(a.sequences, each).cuda()
    states = [torch.from_numpy(rng.normal(0, 1, (n + a.steps, a.hidden)).astype(np.float32)).cuda().to(torch.bfloat16) for n in prompts]
    lengths = torch.tensor(prompts, dtype=torch.int32, device="cuda")
    starts = torch.tensor(np.concatenate(([0], np.cumsum(prompts))), dtype=torch.int32, device="cuda")
    got = [layer(torch.cat([s[:n] for s, n in zip(states, prompts)]), table, lengths, starts)]
    for i in range(a.steps):
        lengths += 1
        got.append(layer(torch.stack([s[n + i] for s, n in zip(states, prompts)]), table, lengths))
    layer.ops.check_device_error()
    w1, w2 = torch.from_numpy(qkv).cuda(), torch.from_numpy(out).cuda()
    want = [_float_layer(s.float(), w1, w2, a.heads, a.kv_heads, s.shape[0]) for s in states]
    ends = np.cumsum(prompts)
    far = lambda g, w: float((g.float() - w).norm() / w.norm())   # noqa: E731
    prompt = far(got[0], torch.cat([w[:n] for w, n in zip(want, prompts)]))
    steps = far(torch.stack(got[1:]), torch.stack([torch.stack([w[n + i] for w, n in zip(want, prompts)]) for i in range(a.steps)])) if a.steps else 0.0
    print(f"attention, {a.heads} heads of {a.head_dim} over {a.kv_heads}, 4-bit weights (groups of {a.group}) and cache: {int(ends[-1])} prompt tokens, "
          f"relative difference from float {prompt:.4f}; {a.steps} steps of {a.sequences} sequences {steps:.4f}")
    return prompt, steps


if __name__ == "__main__":
    main()
