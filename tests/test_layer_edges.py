"""Corners of the layer's operators, on the CPU (no kernel runs)."""
import math

import pytest
import torch

import prism_amd


@pytest.mark.parametrize("dim,factor,length", [(128, 8.0, 65536), (128, 8.0, 131072), (8, 8.0, 8192), (64, 4.0, 8192),
                                               (128, 16.0, 4096), (32, 2.0, 1 << 20)])
def test_yarn_ramp_past_the_last_pair(dim, factor, length):
    """The ramp ends where a pair would turn beta_slow times, past the head's last
    pair too: pairs that turn more often than that are not divided in full."""
    fast, slow, base = 32.0, 1.0, 10000.0
    f, _ = prism_amd.rotary_frequencies(dim, base=base, scaling="yarn", factor=factor, original_length=length, device="cpu")
    where = lambda n: dim * math.log(length / (n * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
    low, high = max(math.floor(where(fast)), 0), min(math.ceil(where(slow)), dim - 1)
    for i in range(dim // 2):
        plain = base ** (-2 * i / dim)
        share = min(max((i - low) / (high - low), 0.0), 1.0)
        want = plain * (1 - share) + plain / factor * share
        # powers, one division, two products and a sum in float64: 8 half steps
        assert abs(float(f[i]) - want) <= 8 * 2.0 ** -53 * want, i
        turns = length * plain / (2 * math.pi)
        if turns >= fast:
            assert share == 0.0
        if turns > slow * base ** (2 / dim):  # (more than one whole pair away from the ramp's end)
            assert share < 1.0 and float(f[i]) > plain / factor


@pytest.mark.parametrize("betas", [(1.0, 32.0), (4.0, 4.0), (32.0, 0.0), (32.0, -1.0), (math.nan, 1.0), (32.0, math.nan),
                                   (math.inf, 1.0)])
def test_yarn_refuses_ends_out_of_order(betas):
    fast, slow = betas
    with pytest.raises(ValueError, match="beta_fast"):
        prism_amd.rotary_frequencies(64, scaling="yarn", factor=4.0, original_length=8192, beta_fast=fast, beta_slow=slow,
                                     device="cpu")
