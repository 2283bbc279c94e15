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


COMPLETE = {
    "linear": {"rope_type": "linear", "factor": 4.0},
    "llama3": {"rope_type": "llama3", "factor": 8.0, "original_max_position_embeddings": 8192},
    "yarn": {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768},
}


@pytest.mark.parametrize("kind,key", [(k, key) for k, s in COMPLETE.items() for key in s if key != "rope_type"])
def test_a_missing_key_is_refused_and_not_guessed(kind, key):
    s = COMPLETE[kind]
    freq(64, 10000.0, s)
    for without in ({k: v for k, v in s.items() if k != key}, {**s, key: None}):
        with pytest.raises(ValueError, match=key):
            freq(64, 10000.0, without)


@pytest.mark.parametrize("kind", ["llama3", "yarn"])
def test_the_original_length_may_stand_outside_the_dict(kind):
    s = dict(COMPLETE[kind])
    old = s.pop("original_max_position_embeddings")
    assert freq(64, 10000.0, s, original_max_position_embeddings=old) == freq(64, 10000.0, COMPLETE[kind])
    # and the dict's own comes first
    assert freq(64, 10000.0, COMPLETE[kind], original_max_position_embeddings=77) == freq(64, 10000.0, COMPLETE[kind])


@pytest.mark.parametrize("s", [
    {**COMPLETE["yarn"], "long_mscale": 1.2}, {**COMPLETE["linear"], "beta_fast": 32.0},
    {**COMPLETE["llama3"], "attention_factor": 1.1}, {"rope_type": "default", "factor": 4.0},
    {"type": "default", "mrope_section": [16, 24, 24]}, {**COMPLETE["yarn"], "mscale": 0.7},
    {**COMPLETE["yarn"], "mscale_all_dim": 0.7}, {**COMPLETE["linear"], "rope_theta": 5e5},
    {**COMPLETE["llama3"], "low_freq_factor": 4.0}])
def test_what_is_not_honoured_is_refused(s):
    """Keys that would change the angles and that the kind's formula does not have; half of a pair; another base."""
    with pytest.raises(ValueError):
        freq(64, 10000.0, s)


def test_keys_that_change_nothing_pass():
    for kind, s in COMPLETE.items():
        more = {**s, "type": kind, "rope_theta": 10000, "partial_rotary_factor": 0.5, "attention_factor": None}
        assert freq(64, 10000.0, more) == freq(64, 10000.0, s)
    assert freq(64, 10000.0, {**COMPLETE["yarn"], "finetuned": True}) == freq(64, 10000.0, COMPLETE["yarn"])
    assert freq(64, 10000.0, {**COMPLETE["yarn"], "truncate": None}) == freq(64, 10000.0, COMPLETE["yarn"])
    assert freq(64, 10000.0, {**COMPLETE["yarn"], "mscale": 1.0, "mscale_all_dim": 1.0})[1] == 1.0
    assert freq(64, 10000.0, {}) == freq(64, 10000.0)


def test_lengths_in_the_dict_of_a_kind_without_them_pass():
    """A context's lengths do not change the angles of these kinds; longrope reads them in the dict as well."""
    lengths = {"original_max_position_embeddings": 4096, "max_position_embeddings": 131072}
    for s in (COMPLETE["linear"], {"rope_type": "default"}):
        assert freq(64, 10000.0, {**s, **lengths}) == freq(64, 10000.0, s)
    assert freq(64, 10000.0, {**COMPLETE["yarn"], "max_position_embeddings": 131072}) == freq(64, 10000.0, COMPLETE["yarn"])
    assert freq(96, 10000.0, {**PUBLISHED, **lengths}) == freq(96, 10000.0, PUBLISHED, **lengths)
