"""How far the logarithm of a row's sum of exponentials is off: rows of one to three entries, whose errors do not average
out, with a score that cancels it, so that what is written is the error itself."""
import numpy as np
import pytest
import torch as T

from pages_util import beam

pytestmark = pytest.mark.gpu

BELOW = (0.0, 0.37, 1.7)                               # the entries, below the largest one
ROWS = 1 << 16


def error(qa, dtype, vocab, low, high):
    """the largest error of the logarithm, with the largest entry at 2^16 places from low to high"""
    top = T.linspace(low, high, ROWS).to(dtype).float()
    x = (top[:, None] - T.tensor(BELOW[:vocab])).to(dtype)
    d = x.double() - x.double().max(1, keepdim=True)[0]
    lse = T.log(T.exp(d).sum(1))
    score = lse.float()
    out = beam(qa, x.cuda(), score.tolist(), None, 1, ROWS)[2][:, 0].astype(np.float64)
    # a number of 2^-22 is written with 2^-46
    return float(np.abs(out - (score.double() - lse).numpy()).max())


RANGES = pytest.mark.parametrize("low,high", [(-30.0, 30.0), (-1.0, 1.0), (29.0, 31.0), (-200.0, -30.0), (-1e-3, 1e-3)])
VOCAB = pytest.mark.parametrize("vocab", [1, 2, 3])
TYPES = pytest.mark.parametrize("dtype", [T.float32, T.bfloat16], ids=["f32", "bf16"])


@TYPES
@VOCAB
@RANGES
def test_error_of_the_logarithm(qa, gpu, dtype, vocab, low, high):
    """an exponential: 2^-23 (v_exp_f32's 1 ulp) and ln 2 2^-25 (its argument up to 1/2, rounded twice); one of the share's
    reference the same; two are added in fp32: 2^-24.  Less than 3 x 2^-23 of the sum."""
    assert error(qa, dtype, vocab, low, high) <= 3 * 2.0 ** -23


@pytest.mark.parametrize("top", [40.0, -40.0, 300.0, 1e4])
def test_shares_are_joined_exactly(qa, gpu, top):
    """two entries far apart in the row: each is its share's reference, its sum 1, so that what joins them is all there is;
    in 64 bits that is off by some 2^-50, and by what is written of a number below 2^-20 with 24 bits"""
    rows, vocab = 96, 40000
    below = T.linspace(0.0, 6.0, rows)
    x = T.full((rows, vocab), -np.inf)
    x[:, 0], x[:, vocab - 1] = top, top - below
    d = x[:, vocab - 1].double() - top
    lse = T.log1p(T.exp(d))
    score = lse.float()
    out = beam(qa, x.cuda(), score.tolist(), None, 1, rows)[2][:, 0].astype(np.float64)
    assert float(np.abs(out - (score.double() - lse).numpy()).max()) <= 2.0 ** -44


@TYPES
@VOCAB
@RANGES
def test_error_of_the_sum(qa, gpu, dtype, vocab, low, high):
    """an exponential: 2^-23 and ln 2 2^-25, as above; two are added in fp32: 2^-24.  Less than 2^-22 of the sum."""
    assert error(qa, dtype, vocab, low, high) <= 1.25 * 2.0 ** -23 + (vocab > 1) * 2.0 ** -24
