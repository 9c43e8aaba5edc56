"""rope_frequencies against YaRN as published (Peng et al. 2023), written out index by index in 64 bits: the ramp runs
between the (real) indices whose frequencies turn `fast` and `slow` times within original_len, the lower rounded down and
at least 0, the upper rounded up and at most rotary_dim - 1.  The table is the 64-bit value rounded to f32: half a step."""
import math

import numpy as np
import pytest

HALF_STEP = 2.0 ** -24


def published(dim, theta, factor, original_len, fast=32.0, slow=1.0):
    def index(turns):
        return dim * math.log(original_len / (turns * 2 * math.pi)) / (2 * math.log(theta))

    low, high = max(math.floor(index(fast)), 0), min(math.ceil(index(slow)), dim - 1)
    out = []
    for i in range(dim // 2):
        f = theta ** (-2.0 * i / dim)
        ramp = min(max((i - low) / (high - low if high != low else 1e-3), 0.0), 1.0)
        out.append(f / factor * ramp + f * (1 - ramp))
    return np.array(out)


@pytest.mark.parametrize("dim,theta,factor,original_len", [
    (128, 1e4, 16.0, 4096), (64, 1e7, 4.0, 32768), (128, 1e6, 8.0, 32768),
    # the slowest frequency turns more than once within original_len: the ramp ends past the table
    (128, 1e4, 4.0, 65536), (128, 1e4, 4.0, 131072), (128, 1e4, 8.0, 131072), (16, 1e4, 4.0, 32768), (32, 1e4, 2.0, 1 << 20)])
def test_yarn_table(dim, theta, factor, original_len):
    from exl3_b200.attention import rope_frequencies

    got, attention_factor = rope_frequencies(dim, theta, factor, original_len)
    want = published(dim, theta, factor, original_len)
    # 16 u for the 64-bit powers and products on both sides, far below half a step of f32
    assert np.all(np.abs(got.astype(np.float64) - want) <= (HALF_STEP + 16 * 2.0 ** -53) * want)
    assert attention_factor == pytest.approx(0.1 * math.log(factor) + 1, rel=1e-15)


def test_yarn_divides_in_full_only_what_turns_less_than_slow():
    """theta 1e4 behind 131072 positions: the last of 64 frequencies turns 2.4 times and lies on the ramp."""
    from exl3_b200.attention import rope_frequencies

    plain = rope_frequencies(128, 1e4)[0].astype(np.float64)
    got = rope_frequencies(128, 1e4, 4.0, 131072)[0].astype(np.float64)
    assert np.all(131072 * plain / (2 * math.pi) > 1)
    assert np.all(got > plain / 4 * 1.01)
