"""The turn of keys and queries by their positions in FP64, and how far FP32 arithmetic may be from it."""

import math

import torch

import kv_oracle


def turned(x, positions, inv_freq, interleaved):
    """(rows, bound) of x [rows, heads, D] (BF16, CPU): each value's turn, and how far FP32 may be off it.

    The bound. The angle in turns is a product of three FP64 numbers (2 roundings: 2^-52 of itself), its part of a turn rounded to FP32
    (at most 2^-26 turns: 2^-23.3 as an angle); cos and sin are within 4 units of their last place (2^-22 of 1); a turned value
    is two products and a sum, three roundings of at most 2^-24 (|a| + |b|). Together under (|a| + |b|) (2^-21 + 2^-49 turns)."""
    pairs = inv_freq.numel()
    angle = positions.double()[:, None, None] * inv_freq.double()
    x = x.double()
    first = x[..., :2 * pairs]
    a, b = (first[..., 0::2], first[..., 1::2]) if interleaved else first.chunk(2, -1)
    y = (a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin())
    off = (a.abs() + b.abs()) * (2.0**-21 + angle.abs() / (2 * math.pi) * 2.0**-49)
    join = (lambda u, v: torch.stack((u, v), -1).flatten(-2)) if interleaved else (lambda u, v: torch.cat((u, v), -1))
    rest = x[..., 2 * pairs:]
    return torch.cat((join(*y), rest), -1), torch.cat((join(off, off), torch.zeros_like(rest)), -1)


def check_held(codes, scales, want, off, fmt):
    """Rows that the cache holds, against FP64 rows that may be `off` before their rounding: half a step of the format."""
    if fmt == "bf16":
        allowed = off + 2.0**-8 * (want.abs() + off) + 2.0**-134
        got = codes.double()
    else:
        top = kv_oracle.TOP[fmt]
        most, most_off = want.abs().amax(-1), off.amax(-1)
        scale = most / top
        assert ((scales.double() - scale).abs() <= most_off / top + scale * 2.0**-22).all()
        got = kv_oracle.values(codes, scales)
        # a scale that is off moves every value of the row by no more than the largest; the scaled value's own roundings: 2^-21
        step = 0.5 * scale[..., None] if fmt == "int8" else torch.maximum(2.0**-4 * want.abs(), 2.0**-10 * scale[..., None])
        allowed = step * (1 + 2.0**-18) + 2 * most_off[..., None] + want.abs() * 2.0**-20
    far = (got - want).abs() / allowed.clamp(min=1e-300)
    print(f"  of what the roundings allow: {far.max():.3f}", flush=True)
    assert far.max() <= 1
