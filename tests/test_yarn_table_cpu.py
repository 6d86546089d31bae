"""YaRN tables against the formula written out pair by pair in 64 bits: each key of the scaling dictionary, how many
positions the table covers, and what is refused.

Tolerance: the table is the fp32 rounding (2^-24 of itself) of values of at most the amplitude whose angles, up to
positions x 1 radian in 64 bits, are off by 2^-52 of themselves in a few operations: under 2^-30 here."""
import math

import pytest
import torch

from adallm_b200.rotary_embedding import RotaryEmbedding, build_cos_sin_cache, get_rope

BASE, TRAINED, FACTOR = 1e4, 512, 8.0
YARN = {"rope_type": "yarn", "factor": FACTOR, "original_max_position_embeddings": TRAINED}


def formula(width, rows, amplitude, fast=32.0, slow=1.0, truncate=True):
    half = width // 2
    low, high = (half * math.log(TRAINED / (n * 2 * math.pi)) / math.log(BASE) for n in (fast, slow))
    if truncate:
        low, high = math.floor(low), math.ceil(high)
    low, high = max(low, 0), min(high, width - 1)
    cos, sin = [], []
    pos = torch.arange(rows, dtype=torch.float64)
    for i in range(half):
        ramp = min(max((i - low) / (high - low), 0.0), 1.0)
        f = BASE ** (-2 * i / width)
        angle = pos * (f * (1 - ramp) + f / FACTOR * ramp)
        cos.append(angle.cos() * amplitude)
        sin.append(angle.sin() * amplitude)
    return torch.stack(cos + sin, 1)


def near(table, want, amplitude):
    assert table.shape == (want.shape[0], 1, want.shape[1]) and table.dtype == torch.float32
    assert ((table[:, 0].double() - want).abs() <= 2.0 ** -24 * want.abs() + 2.0 ** -30 * amplitude).all()


def scale(m):
    return 0.1 * m * math.log(FACTOR) + 1


@pytest.mark.parametrize("keys,amplitude,ramp", [
    ({}, scale(1), {}), ({"mscale": 1.0, "mscale_all_dim": 1.0}, 1.0, {}),
    ({"mscale": 0.707, "mscale_all_dim": 1.0}, scale(0.707) / scale(1), {}),
    ({"attention_factor": 1.25}, 1.25, {}), ({"attention_factor": 0.5, "mscale": 1.0, "mscale_all_dim": 1.0}, 0.5, {}),
    ({"truncate": False}, scale(1), dict(truncate=False)), ({"truncate": True}, scale(1), {}),
    ({"beta_fast": 16.0, "beta_slow": 2}, scale(1), dict(fast=16.0, slow=2.0)),
    ({"beta_fast": None, "attention_factor": None, "mscale": None, "truncate": None, "rope_theta": BASE}, scale(1), {}),
    ({"partial_rotary_factor": 0.5}, scale(1), {})])
@pytest.mark.parametrize("width", [64, 128])
def test_every_key(keys, amplitude, ramp, width):
    rows = int(FACTOR) * TRAINED
    near(build_cos_sin_cache(width, rows, BASE, {**YARN, **keys}), formula(width, rows, amplitude, **ramp), amplitude)


def test_tables_cover_the_scaled_length():
    """A model's max_position may be the trained length or lie between; positions behind the table would be clamped."""
    want = formula(64, 5000, scale(1))
    for asked, rows in ((TRAINED, 4096), (1000, 4096), (4096, 4096), (5000, 5000)):
        near(build_cos_sin_cache(64, asked, BASE, YARN), want[:rows], scale(1))
    assert RotaryEmbedding(128, 64, 640, BASE, YARN).cos_sin_cache.shape == (4096, 1, 64)
    assert get_rope(128, 128, 640, BASE, YARN).cos_sin_cache.shape == (4096, 1, 128)
    odd = {**YARN, "factor": 1.5, "original_max_position_embeddings": 333}
    assert build_cos_sin_cache(64, 16, BASE, odd).shape[0] == 500
    assert build_cos_sin_cache(64, 16, BASE, {"rope_type": "linear", "factor": 4.0}).shape[0] == 16
    # without the original length max_position is the scaled one
    near(build_cos_sin_cache(64, 4096, BASE, {"type": "yarn", "factor": FACTOR}), want[:4096], scale(1))
    assert all(build_cos_sin_cache(64, n, BASE, {"type": "yarn", "factor": f}).shape[0] == n for n in (1000, 4097)
               for f in (1.1, 3.0, 7.7))


@pytest.mark.parametrize("keys", [
    {"mscale": 1.0}, {"mscale_all_dim": 1.0}, {"mscale": 0.0, "mscale_all_dim": 1.0}, {"mscale": 1.0, "mscale_all_dim": -1.0},
    {"attention_factor": 0.0}, {"attention_factor": math.nan}, {"extrapolation_factor": 1.0}, {"short_factor": [1.0]},
    {"factor": None}, {"factor": 0.0}, {"factor": math.inf}, {"original_max_position_embeddings": 0}, {"beta_fast": 1.0, "beta_slow": 2.0}, {"beta_slow": 0.0}, {"rope_theta": 5e5}])
def test_refusals(keys):
    with pytest.raises(ValueError):
        build_cos_sin_cache(128, 4096, BASE, {**YARN, **keys})
