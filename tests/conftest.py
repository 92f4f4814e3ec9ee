"""Shared test setup: import paths, the ``gpu`` marker, and the parity metrics."""

import os
import sys

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "haskell-infer-demo_amd")
for p in (ROOT, PKG):
    if p not in sys.path:
        sys.path.insert(0, p)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs an MI355X (runs the HIP library on cuda:0)")


# Tests that hold a wrong value: what it is, and where the right one is tested.
HOLD_WRONG_VALUES = {
    "test_paged_attention.py::test_rows_that_see_nothing":
        "places the rows of a sequence whose kv_lens pass its table by the table's end (kv_lens 40 of 32 places: 29 to 31 for "
        "three rows) where the interface, the write and the read have them at kv_lens (37 to 39): "
        "test_lengths_past_the_table.py has the right places, and everything else that this test looks at",
}


def pytest_collection_modifyitems(items):
    for item in items:
        for name, why in HOLD_WRONG_VALUES.items():
            if f"{item.path.name}::{getattr(item, 'originalname', item.name)}" == name:
                item.add_marker(pytest.mark.xfail(reason=why, strict=True))


@pytest.fixture(scope="session")
def cuda():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no GPU visible")
    return torch.device("cuda", 0)


@pytest.fixture(autouse=True)
def _no_split_wait_timeouts(request):
    """After every GPU test: no bounded split-K wait gave up on an unwritten partial."""
    yield
    if request.node.get_closest_marker("gpu") is None:
        return
    import torch

    if not torch.cuda.is_available():
        return
    import w4a16

    w4a16.split_wait_status()


def bf16_f32(bits):
    return (np.asarray(bits, dtype=np.uint16).astype(np.uint32) << 16).view(np.float32)


def parity_metrics(got_bits, ref, ref_is_bits=True, floor_div=64.0):
    """Compare BF16 outputs with the oracle.

    rel_l2: ||got - ref|| / ||ref|| over the whole output.
    max_ulp: max |got - ref| in BF16 ULPs of max(|ref|, rms(ref)/floor_div) (default 64). Near
    zero an element's own ULP is far below the FP32 accumulation error of any FP32-accumulated
    kernel (the reference's included), so the ULP there is taken at that floor.
    """
    got = bf16_f32(got_bits).astype(np.float64)
    r = bf16_f32(ref).astype(np.float64) if ref_is_bits else np.asarray(ref, np.float64)
    diff = np.abs(got - r)
    rel_l2 = float(np.linalg.norm(diff) / max(np.linalg.norm(r), 1e-30))
    rms = float(np.sqrt(np.mean(r * r))) if r.size else 0.0
    mag = np.maximum(np.abs(r), rms / floor_div)
    ulp = np.exp2(np.floor(np.log2(np.maximum(mag, 1e-38))) - 7)
    ulps = diff / ulp
    # the same difference in ULPs of each element's own value, without the floor: how many
    # near-zero elements the floor admits beyond the north star's "<= 2 BF16 ULP"
    own = diff / np.exp2(np.floor(np.log2(np.maximum(np.abs(r), 1e-38))) - 7)
    return {"rel_l2": rel_l2, "max_ulp": float(ulps.max()) if ulps.size else 0.0,
            "n_over_1ulp": int((ulps > 1.0).sum()), "n": int(r.size),
            "n_over_2ulp_own": int((own > 2.0).sum()),
            "max_ulp_own": float(own.max()) if own.size else 0.0}


def assert_parity(got_bits, ref, what, rel_l2=1e-3, max_ulp=2.0, ref_is_bits=True,
                  floor_div=64.0):
    m = parity_metrics(got_bits, ref, ref_is_bits, floor_div)
    print(f"{what}: rel_l2={m['rel_l2']:.3g} max_ulp={m['max_ulp']:.3g} "
          f">1ulp={m['n_over_1ulp']}/{m['n']} own>2ulp={m['n_over_2ulp_own']} "
          f"(max own {m['max_ulp_own']:.3g})", flush=True)
    assert m["rel_l2"] <= rel_l2, (what, m)
    assert m["max_ulp"] <= max_ulp, (what, m)
    # Elements past 2 ULPs of their own value (all near zero, admitted by the floor above):
    # over the whole GPU suite 0.009% of the elements. A kernel-stage check may hold at most
    # 0.1% of its elements (and a handful), an end-to-end check (floor rms/16) 1%, so the floor
    # cannot hide a systematic error.
    own_cap = m["n"] // (1000 if floor_div >= 64.0 else 100)
    assert m["n_over_2ulp_own"] <= max(8, own_cap), (what, m)
    return m
