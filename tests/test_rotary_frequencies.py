"""Rotary frequencies of scaled contexts: every key of a ``rope_scaling``
dictionary is used or refused.

The expected values are the published formulas, worked out here element by
element.  Tolerance 1e-12 relative: a dozen binary64 roundings of 2^-53 each,
and of the powers and logarithms that they enter, stay below 1e-14."""
from __future__ import annotations

import math

import pytest
import torch

from nanopointllm_amd import attention as A

YARN = {"rope_type": "yarn", "factor": 40.0, "original_max_position_embeddings": 4096}
LLAMA3 = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 8192}


def frequencies(scaling, d=128, base=10000.0):
    return A.rotary_frequencies(d, base=base, scaling=scaling, device="cpu")


# ------------------------------------------------------------ the amplitude
@pytest.mark.parametrize("m, m_all, want", [
    (1.0, 1.0, 1.0),
    # (0.1 m ln 40 + 1) / (0.1 m_all ln 40 + 1), ln 40 = 3.6888794541139363
    (1.0, 0.707, 1.36888794541139363 / 1.2608037774058553),
    (0.707, 1.0, 1.2608037774058553 / 1.36888794541139363),
    (2.0, 0.5, 1.7377758908227873 / 1.1844439727056968),
])
def test_yarn_amplitude_of_two_scales(m, m_all, want):
    plain = frequencies(YARN)
    assert math.isclose(plain.attention_factor, 1.36888794541139363, rel_tol=1e-12)
    got = frequencies({**YARN, "mscale": m, "mscale_all_dim": m_all})
    assert math.isclose(got.attention_factor, want, rel_tol=1e-12)
    assert torch.equal(got.inv_freq, plain.inv_freq)


def test_yarn_amplitude_given_or_left_out():
    scales = {"mscale": 1.0, "mscale_all_dim": 0.5}
    # A given amplitude is the amplitude; None is a key left out.
    assert frequencies({**YARN, **scales, "attention_factor": 1.3}).attention_factor == 1.3
    for key in ("attention_factor", "mscale", "mscale_all_dim", "beta_fast", "beta_slow",
                "truncate"):
        got = frequencies({**YARN, key: None})
        assert got.attention_factor == frequencies(YARN).attention_factor
        assert torch.equal(got.inv_freq, frequencies(YARN).inv_freq)
    # Both scales are of the factor: a factor of one has none.
    assert frequencies({**YARN, **scales, "factor": 1.0}).attention_factor == 1.0


# ------------------------------------------------------- the blend's borders
@pytest.mark.parametrize("truncate", [True, False])
@pytest.mark.parametrize("fast, slow, d, base", [(32.0, 1.0, 128, 10000.0), (20.0, 2.0, 64, 1e6),
                                                 (32.0, 1.0, 80, 500000.0)])
def test_yarn_borders_whole_or_as_they_are(fast, slow, d, base, truncate):
    got = frequencies({**YARN, "beta_fast": fast, "beta_slow": slow, "truncate": truncate}, d, base)

    def border(turns):
        return d * math.log(4096 / (2 * math.pi * turns)) / (2 * math.log(base))

    low, high = border(fast), border(slow)
    if truncate:
        low, high = math.floor(low), math.ceil(high)
    low, high = max(low, 0), min(high, d - 1)
    for i, f in enumerate(got.inv_freq.tolist()):
        plain = base ** (-2 * i / d)
        slowed = min(max((i - low) / (high - low), 0.0), 1.0)
        assert math.isclose(f, plain * ((1 - slowed) + slowed / 40.0), rel_tol=1e-12), i


# ------------------------------------------------------------------ refusals
def without(scaling, key):
    return {k: v for k, v in scaling.items() if k != key}


@pytest.mark.parametrize("scaling, message", [
    # keys that the kind does not use
    ({**YARN, "low_freq_factor": 1.0}, "low_freq_factor"),
    ({**YARN, "finetuned": True}, "finetuned"),
    ({**LLAMA3, "mscale": 1.0}, "mscale"),
    ({"type": "linear", "factor": 2.0, "original_max_position_embeddings": 64}, "original_max"),
    ({"type": "ntk", "factor": 2.0, "alpha": 3.0}, "alpha"),
    ({"rope_type": "default", "mrope_section": [16, 24, 24]}, "mrope_section"),
    ({"factor": 4.0}, "factor"),
    ({"rope_type": "default", "factor": 4.0}, "factor"),
    # keys that it needs
    (without(YARN, "original_max_position_embeddings"), "original_max_position_embeddings"),
    (without(YARN, "factor"), "factor"),
    (without(LLAMA3, "original_max_position_embeddings"), "original_max_position_embeddings"),
    (without(LLAMA3, "low_freq_factor"), "low_freq_factor"),
    (without(LLAMA3, "high_freq_factor"), "high_freq_factor"),
    ({"type": "linear"}, "factor"),
    ({"type": "linear", "factor": None}, "factor"),
    # one of a pair, and two that differ
    ({**YARN, "mscale": 1.0}, "mscale_all_dim"),
    ({**YARN, "mscale_all_dim": 1.0}, "mscale"),
    ({**YARN, "type": "linear"}, "rope_type"),
    ({**YARN, "rope_theta": 500000.0}, "rope_theta"),
    # values outside the formulas
    ({**YARN, "mscale": 0.0, "mscale_all_dim": 1.0}, "mscale"),
    ({**YARN, "mscale": 1.0, "mscale_all_dim": -1.0}, "mscale"),
    ({**YARN, "original_max_position_embeddings": 0}, "original_max_position_embeddings"),
    ({**YARN, "beta_fast": 0.0}, "beta"),
    ({**YARN, "beta_fast": 1.0, "beta_slow": 2.0}, "beta"),
    ({**YARN, "truncate": "no"}, "truncate"),
    ({**YARN, "attention_factor": math.nan}, "attention_factor"),
    ({**YARN, "factor": math.inf}, "factor"),
    ({**YARN, "factor": "forty"}, "factor"),
    ({**LLAMA3, "original_max_position_embeddings": -1}, "original_max_position_embeddings"),
])
def test_refused_dictionaries(scaling, message):
    with pytest.raises(ValueError, match=message):
        frequencies(scaling)


def test_bases():
    assert torch.equal(frequencies({**YARN, "rope_theta": 10000}).inv_freq,
                       frequencies(YARN).inv_freq)
    with pytest.raises(ValueError, match="base"):
        frequencies(YARN, base=1.0)      # no logarithm to place the borders by
    for base in (math.inf, math.nan, -1.0):
        with pytest.raises(ValueError, match="base"):
            frequencies(None, base=base)
    assert frequencies({"rope_type": "default"}).attention_factor == 1.0
    assert frequencies({"rope_type": "default", "factor": 1.0}).attention_factor == 1.0
