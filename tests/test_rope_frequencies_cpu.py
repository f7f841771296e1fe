"""Frequencies of rotary embeddings that YaRN scales in the form that models' files mean, against values worked out by hand."""
import math

import pytest
import torch

from zllm_b200 import ffi
from zllm_b200.backend import rope_frequencies


def pairs(rotary, base, factor, context, **kwargs):
    return rope_frequencies(rotary, base, ffi.ROPE_SCALE_YARN_PAIRS, factor=factor, original_context=context, **kwargs)



# 128 values, base 1e6, 4 times 32768 positions: pair i turns 32768 / (2 pi) 1e6^(-i / 64) times. 32 turns lie at 64 ln(162.975) / ln(1e6) = 64 x 5.09359 / 13.81551 = 23.596, one at
# 64 ln(5215.19) / 13.81551 = 64 x 8.55933 / 13.81551 = 39.651: a ramp of 17 pairs from 23 to 40.
# 64 values, base 1e4, 16 times 4096: 32 ln(20.3718) / ln(1e4) = 32 x 3.01415 / 9.21034 = 10.472 and 32 ln(651.899) / 9.21034 = 32 x 6.47989 / 9.21034 = 22.514: 13 pairs from 10 to 23.
@pytest.mark.parametrize("rotary,base,factor,context,low,high", [(128, 1e6, 4.0, 32768, 23, 40), (64, 1e4, 16.0, 4096, 10, 23)])
def test_the_ramp_is_linear_in_the_pairs_number(rotary, base, factor, context, low, high):
    got, by = pairs(rotary, base, factor, context)
    half = rotary // 2
    for i in range(half):
        divided = min(max(i - low, 0), high - low) / (high - low)  # how much of the pair is divided
        want = base ** (-i / half) * (1 - divided + divided / factor)
        assert abs(float(got[i]) - want) <= 2.0 ** -23 * want, i  # both sides round once from f64
    assert by == pytest.approx(0.1 * math.log(factor) + 1, rel=2.0 ** -23)


def test_single_frequencies_by_hand():
    got, _ = pairs(128, 1e6, 4.0, 32768)
    plain, _ = rope_frequencies(128, 1e6)
    assert torch.equal(got[:24], plain[:24]) and torch.equal(got[40:], plain[40:] / 4)
    # pair 32 has 1e6^(-1/2) = 1e-3 and is 9 of 17 on the way: 1e-3 (8 + 9 / 4) / 17 = 1e-3 x 10.25 / 17
    assert float(got[32]) == pytest.approx(1e-3 * 10.25 / 17, rel=2.0 ** -23)
    # pair 24 has 1e6^(-24/64) = 10^(-2.25), 1 of 17 on the way: 10^(-2.25) x 16.25 / 17
    assert float(got[24]) == pytest.approx(10 ** -2.25 * 16.25 / 17, rel=2.0 ** -23)
    # pair 39, 16 of 17: 10^(-3.65625) x (1 + 4) / 17
    assert float(got[39]) == pytest.approx(10 ** -3.65625 * 5 / 17, rel=2.0 ** -23)


def test_where_the_two_forms_agree_and_where_they_do_not():
    in_pairs, by = pairs(128, 1e6, 4.0, 32768)
    in_turns, by_too = rope_frequencies(128, 1e6, ffi.ROPE_SCALE_YARN, factor=4.0, original_context=32768)
    assert by == by_too and torch.equal(in_pairs[:23], in_turns[:23]) and torch.equal(in_pairs[40:], in_turns[40:])
    assert ((in_pairs / in_turns - 1).abs() > 0.01).sum() == 16


def test_borders_outside_of_the_pairs():
    plain, _ = rope_frequencies(16, 1e4)
    # every pair turns more often than 32 times: 8 ln(1e12 / (64 pi)) / ln(1e4) = 19.4, past the last number of 15
    assert torch.equal(pairs(16, 1e4, 8.0, 1e12)[0], plain)
    # none turns once: both borders are pair 0, which is kept, as the ramp begins behind it
    got = pairs(16, 1e4, 8.0, 5.0)[0]
    assert torch.equal(got[1:], plain[1:] / 8) and torch.equal(got[:1], plain[:1])
    factors = [1.0, 2.0, 4.0, 8.0, 1.0, 1.0, 1.0, 0.5]
    scaled = pairs(16, 1e4, 8.0, 4096, pair_factors=factors)[0]
    assert torch.allclose(scaled, pairs(16, 1e4, 8.0, 4096)[0] / torch.tensor(factors), rtol=2.0 ** -22, atol=0)


@pytest.mark.parametrize("kwargs", [dict(base=1.0), dict(base=0.5), dict(beta_slow=0.0), dict(beta_slow=-1.0), dict(beta_slow=32.0), dict(context=0.0), dict(factor=0.0), dict(factor=math.inf), dict(context=math.nan)])
def test_parameters_without_a_ramp_are_refused(kwargs):
    a = {**dict(rotary=64, base=1e4, factor=4.0, context=4096.0), **kwargs}
    with pytest.raises(ffi.ZqFailure) as e:
        pairs(a.pop("rotary"), a.pop("base"), a.pop("factor"), a.pop("context"), **a)
    assert e.value.code == 4
