"""rotary_frequencies with rope_scaling dicts as published model configurations
have them, against the formulas written out here."""
from __future__ import annotations

import math

import pytest

import sparse_decode as sdp


def freq(*a, **kw):
    inv, mult = sdp.rotary_frequencies(*a, **kw, device="cpu")
    return inv.tolist(), mult


def yarn(rot, base, factor, old, fast=32.0, slow=1.0, truncate=True):
    """Pair i keeps its frequency below the pair that makes `fast` turns over the old context, is divided by factor
    above the one that makes `slow`, and is a linear blend between; the two bounds are whole numbers if truncate."""
    lo, hi = (rot * math.log(old / (t * 2 * math.pi)) / (2 * math.log(base)) for t in (fast, slow))
    if truncate:
        lo, hi = math.floor(lo), math.ceil(hi)
    lo, hi = max(lo, 0), min(hi, rot - 1)
    out = []
    for i in range(rot // 2):
        x, r = base ** (-2 * i / rot), min(max((i - lo) / (hi - lo), 0.0), 1.0)
        out.append(x * (1 - r) + x / factor * r)
    return out


@pytest.mark.parametrize("more,truncate", [({}, True), ({"truncate": True}, True), ({"truncate": False}, False)])
def test_yarn_bounds_are_whole_pairs_unless_told_otherwise(more, truncate):
    """A configuration with truncate: false blends from 8.09 to 17.40, not from 8 to 18."""
    s = {"rope_type": "yarn", "factor": 32.0, "beta_fast": 32.0, "beta_slow": 1.0,
         "original_max_position_embeddings": 4096, **more}
    got, mult = freq(64, 150000.0, s)
    assert got == pytest.approx(yarn(64, 150000.0, 32.0, 4096, truncate=truncate), rel=1e-6)
    assert mult == pytest.approx(0.1 * math.log(32) + 1)
