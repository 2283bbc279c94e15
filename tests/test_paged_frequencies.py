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


LONG, SHORT = [1.0 + 0.5 * i for i in range(48)], [1.0 + 0.01 * i for i in range(48)]
PUBLISHED = {"type": "longrope", "long_factor": LONG, "short_factor": SHORT}  # the lengths stand outside the dict


def longrope(each):
    return [10000.0 ** (-2 * i / 96) / f for i, f in enumerate(each)]


def test_longrope_takes_the_lengths_that_stand_outside_the_dict():
    got, mult = freq(96, 10000.0, PUBLISHED, max_position_embeddings=131072, original_max_position_embeddings=4096)
    assert got == pytest.approx(longrope(LONG), rel=1e-6)
    assert mult == pytest.approx(math.sqrt(1 + math.log(32) / math.log(4096))) == pytest.approx(1.19, abs=1e-2)
    got, mult = freq(96, 10000.0, PUBLISHED, max_position_embeddings=4096, original_max_position_embeddings=4096)
    assert got == pytest.approx(longrope(SHORT), rel=1e-6) and mult == 1.0
    # what the dict says itself comes first
    s = {**PUBLISHED, "factor": 8.0, "original_max_position_embeddings": 16384}
    got, mult = freq(96, 10000.0, s, max_position_embeddings=131072, original_max_position_embeddings=4096)
    assert got == pytest.approx(longrope(LONG), rel=1e-6)
    assert mult == pytest.approx(math.sqrt(1 + math.log(8) / math.log(16384)))


@pytest.mark.parametrize("more", [{}, {"max_position_embeddings": 131072}, {"original_max_position_embeddings": 4096}])
def test_longrope_without_its_lengths_is_refused(more):
    with pytest.raises(ValueError):
        freq(96, 10000.0, PUBLISHED, **more)


@pytest.mark.parametrize("missing", ["long_factor", "short_factor"])
def test_longrope_without_its_factors_is_refused(missing):
    s = {k: v for k, v in PUBLISHED.items() if k != missing}
    with pytest.raises(ValueError):
        freq(96, 10000.0, s, max_position_embeddings=131072 if missing == "long_factor" else 4096,
             original_max_position_embeddings=4096)


def test_longrope_without_an_original_length_to_scale_by_is_refused():
    with pytest.raises(ValueError):
        freq(96, 10000.0, {**PUBLISHED, "factor": 32.0})
    got, mult = freq(96, 10000.0, {**PUBLISHED, "factor": 32.0, "attention_factor": 1.25})  # needs none
    assert got == pytest.approx(longrope(LONG), rel=1e-6) and mult == 1.25
