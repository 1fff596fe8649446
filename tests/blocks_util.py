"""Plain 64-bit implementations of the 8-bit block cache and of rotary positions, on the CPU."""

import torch

TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def encode(x: torch.Tensor, dtype):
    """Whole blocks (..., block, D) -> codes and float32 scales, in the float32 steps that the storage is defined by."""
    x = x.float()
    top = x.abs().amax(dim=(-2, -1))
    largest = torch.full_like(top, TOP[dtype])             # (a number over a tensor would be the number times a rounded reciprocal)
    inv = torch.where(top > 0, largest / top, torch.zeros_like(top)).clamp(max=torch.finfo(torch.float32).max)
    y = x * inv[..., None, None]
    return (y.round() if dtype is torch.int8 else y).to(dtype), top / largest


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """Codes (B, H, T, D) and scales (B, H, T / block) as float64 rows."""
    n = codes.shape[2] // max(scales.shape[2], 1)
    return codes.to(torch.float32).double() * scales.double().repeat_interleave(n, dim=2)[..., None]


def attention(q, k, v, scale, window=None, sinks=0):
    """Causal attention of the last tokens, all float64 on the CPU: q (B, Hq, Tq, D) over k, v (B, H, T, D)."""
    q, k, v = q.double(), k.double(), v.double()
    b, hq, t, d = q.shape
    h, total = k.shape[1], k.shape[2]
    k, v = k.repeat_interleave(hq // h, dim=1), v.repeat_interleave(hq // h, dim=1)
    pos, j = torch.arange(total - t, total)[:, None], torch.arange(total)[None, :]
    seen = j <= pos
    if window:
        seen &= (pos - j < window) | (j < sinks)
    s = (q @ k.transpose(-1, -2) * scale).masked_fill(~seen, float("-inf"))
    w = torch.softmax(s, dim=-1)
    return w @ v


def rotary(x, freqs, positions, interleaved, factor):
    """x (B, H, L, D) in float64; positions (L,) or (B, L)."""
    x = x.double()
    r = 2 * freqs.numel()
    pos = positions.double()
    ang = pos[..., None] * freqs.double().cpu()
    ang = ang[None, None] if ang.dim() == 2 else ang[:, None]
    cos, sin = ang.cos() * factor, ang.sin() * factor
    out = x.clone()
    if interleaved:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        out[..., 0:r:2], out[..., 1:r:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        out[..., :r // 2], out[..., r // 2:r] = a * cos - b * sin, b * cos + a * sin
    return out
