"""What the rotating append refuses, on the CPU: every refusal comes before any launch, with a reason."""

import ctypes

import pytest
import torch

import w4a16
from test_kv_refusals import A, CONFIG, batch, cache


def append(c=None, b=None, k=A * 256, v=A * 320, ks=(128, 64), vs=(128, 64), q=A * 384, qs=(256, 64), heads=4, out=A * 448, os=(256, 64),
           freq=A * 600, rotary=32, interleaved=0, positions=A * 610):
    c, b = c or cache(), b or batch()
    return w4a16.lib.w4a16_kv_append_rope_bf16(ctypes.byref(c), ctypes.byref(b), k, *ks, v, *vs, q, *qs, heads, out, *os, freq, rotary,
                                               interleaved, positions, None)


@pytest.mark.parametrize("args,why", [
    (dict(c=cache(head_dim=96)), "head_dim"), (dict(b=batch(rows=-1)), "extents"),
    (dict(k=None), "null"), (dict(v=None), "null"), (dict(freq=None), "null"), (dict(q=None), "q_heads"), (dict(out=None), "q_heads"),
    (dict(heads=0), "q_heads"), (dict(heads=-1), "q_heads"), (dict(heads=65536), "q_heads"), (dict(rotary=0), "rotary_dim"),
    (dict(rotary=12), "rotary_dim"), (dict(rotary=72), "rotary_dim"), (dict(rotary=-8), "rotary_dim"),
    (dict(k=A * 256 + 8), "aligned"), (dict(q=A * 384 + 2), "aligned"), (dict(out=A * 448 + 8), "aligned"),
    (dict(freq=A * 600 + 2), "aligned"), (dict(positions=A * 610 + 1), "aligned"),
    (dict(ks=(130, 64)), "strides"), (dict(vs=(128, -64)), "strides"), (dict(qs=(4, 64)), "strides"), (dict(os=(256, 1 << 62)), "strides"),
    (dict(os=(256, 32)), "each other"), (dict(os=(0, 64)), "each other"),
    (dict(k=A + 64), "overlap"), (dict(q=A), "overlap"), (dict(out=A * 64), "overlap"), (dict(freq=A + 16), "overlap"),
    (dict(positions=A * 64), "overlap"), (dict(out=A * 384 + 128), "overlap"), (dict(out=A * 256), "overlap"), (dict(out=A * 320 - 256), "overlap"),
    (dict(freq=A * 448), "overlap"), (dict(positions=A * 448 + 64), "overlap"), (dict(c=cache(v=A + 1024)), "overlap"),
    (dict(c=cache(format=1, k_scale=A * 448, v_scale=A * 3)), "overlap"),
    # in place with other strides
    (dict(out=A * 384, os=(320, 64)), "overlap"),
])
def test_calls(args, why):
    assert append(**args) == CONFIG
    assert why in w4a16.last_error()


def test_nothing_to_do():
    for b in (batch(rows=0), batch(seqs=0)):
        assert append(b=b) == 0
        assert append(b=b, q=None, heads=0, out=None) == 0


def test_binding():
    for make in (lambda: w4a16.Rope(torch.ones(8)), lambda: w4a16.Rope(None), lambda: w4a16.Rope.of(12), lambda: w4a16.Rope.of(0)):
        with pytest.raises(w4a16.W4A16Error):
            make()
