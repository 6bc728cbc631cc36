"""The K/V cache in 4 or 8 bits in 64-bit torch on the CPU (test infrastructure only).

Restates the form that include/q35.h gives: groups of 64 values as ``low + step
* code`` and causal attention over the values. No reference counterpart; pinned
by hand-made groups and brute force over all codes (tests/test_kvq.py).
"""

from __future__ import annotations

import torch

BF16 = torch.bfloat16


def groups(dim: int, values: bool) -> torch.Tensor:
    """The dims of every group, [dim / 64, 64]."""
    d = torch.arange(dim)
    g = (d % (dim // 16)) // 4 if values else d // 64
    return torch.stack([d[g == i] for i in range(dim // 64)])


def quantise(x: torch.Tensor, bits: int, values: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes uint8 [..., tokens, dim] and params bf16 [..., dim / 64, tokens, 2]."""
    x = x.double()
    top = 2**bits - 1
    codes = torch.zeros(x.shape, dtype=torch.uint8)
    params = []
    for dims in groups(x.shape[-1], values):
        y = x[..., dims]
        finite = torch.isfinite(y).all(-1)
        y = torch.where(finite[..., None], y, 0.0)
        low, high = y.amin(-1), y.amax(-1)
        step = ((high - low).float().double() / top).float()
        # a range past the fp32 maximum: in halves
        half = ((high / 2 - low / 2).float().double() / (top / 2)).float()
        step = torch.where(torch.isfinite((high - low).float()), step, half).to(BF16)
        s = step.double()[..., None]
        r = torch.where(s > 0, (y - low[..., None]) / torch.where(s > 0, s, 1.0), 0.0)
        codes[..., dims] = r.round().clamp(0, top).to(torch.uint8)  # ties to even
        nan = torch.full_like(step, float("nan"))
        params.append(torch.stack((torch.where(finite, step, nan), torch.where(finite, low.to(BF16), nan)), -1))
    return codes, torch.stack(params, -3)


def pack(codes: torch.Tensor, bits: int) -> torch.Tensor:
    return codes if bits == 8 else codes[..., 0::2] | (codes[..., 1::2] << 4)


def unpack(packed: torch.Tensor, bits: int) -> torch.Tensor:
    return packed if bits == 8 else torch.stack((packed & 15, packed >> 4), -1).flatten(-2)


def dequantise(codes: torch.Tensor, params: torch.Tensor, values: bool) -> torch.Tensor:
    """``low + step * code`` in 64 bits, [..., tokens, dim]."""
    out = torch.empty(codes.shape, dtype=torch.float64)
    for g, dims in enumerate(groups(codes.shape[-1], values)):
        p = params[..., g, :, :].double()
        out[..., dims] = p[..., 1:] + p[..., :1] * codes[..., dims].double()
    return out


def attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, starts, scale: float) -> torch.Tensor:
    """Causal GQA: ``q [B, QH, L, D]``, ``k, v [B, KVH, C, D]``; row i of
    sequence b sees the keys 0 .. starts[b] + i. ``[B, L, QH * D]``, 64 bits;
    a row that sees no key is zero, and keys that no row sees are not touched."""
    batch, heads, length, dim = q.shape
    kv_heads, capacity = k.shape[1:3]
    out = torch.zeros(batch, length, heads, dim, dtype=torch.float64)
    for b in range(batch):
        for h in range(heads):
            kv = h * kv_heads // heads
            for i in range(length):
                n = min(max(int(starts[b]) + i + 1, 0), capacity)
                if n:
                    s = (k[b, kv, :n].double() @ q[b, h, i].double()) * scale
                    out[b, i, h] = torch.softmax(s, 0) @ v[b, kv, :n].double()
    return out.flatten(2)
