"""A cache whose buffers share memory takes no write: refused on the CPU, before any launch."""

import pytest

import w4a16
from test_kv_refusals import A, CONFIG, cache, write

CODES, SCALES = 4 * 2 * 16 * 64, 4 * 2 * 16 * 4  # bytes of one buffer of test_kv_refusals.cache() in 8 bits


@pytest.mark.parametrize("fields", [
    dict(k_scale=A * 2, v_scale=A * 2), dict(k_scale=A * 2, v_scale=A * 2 + SCALES - 16), dict(k_scale=A + CODES - 16, v_scale=A * 3),
    dict(k_scale=A * 3, v_scale=A * 64), dict(k_scale=A * 64 + 32, v_scale=A * 3), dict(k_scale=A * 3, v_scale=A + 64),
])
def test_write(fields):
    assert write(c=cache(format=1, **fields)) == CONFIG
    assert "overlap" in w4a16.last_error()
