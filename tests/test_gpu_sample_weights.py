"""How far the weights of a draw are off: the border between one entry and a thousand equal ones, summed as they are or listed
as the class that top-p's cut is in, found to the last bit of the random number."""
import math

import numpy as np
import pytest
import torch as T

from test_gpu_sample import draw

pytestmark = pytest.mark.gpu

N, STEPS = 1000, 64


@pytest.mark.parametrize("mode", ["summed", "listed"])
def test_border(qa, gpu, mode):
    """a weight is off by v_exp_f32's 1 ulp (2^-23) and what its argument of up to 1/2 is rounded by (ln 2 2^-25), all of the
    equal ones by the same; the border 1 / (1 + N w), near 1/2, by a quarter of that, and by one step of u"""
    a = (T.arange(192).float() * 0.00137 + math.log(N) - 0.13)
    border = 1.0 / (1.0 + N * np.exp(-a.double().numpy()))
    x = T.zeros(len(a), N + 1)
    x[:, 1:] = -a[:, None]
    step = 2.0 ** -25                                      # u below 1/2; above it two steps are one number
    u = (np.rint(border / step)[:, None] + np.arange(-STEPS // 2, STEPS // 2)) * step
    rows = x.repeat_interleave(STEPS, 0)
    n = rows.shape[0]
    got = np.array(draw(qa, rows, p=[1 - 2.0 ** -24] * n if mode == "listed" else None,
                        u=u.ravel().tolist())).reshape(u.shape)
    first = got == 0
    assert first[:, 0].all() and not first[:, -1].any() and (np.diff(first.astype(int), axis=1) <= 0).all()
    found = np.array([r[f][-1] for r, f in zip(u.astype(np.float32).astype(np.float64), first)])
    off = np.abs(found - border)
    assert off.max() <= 0.25 * (2.0 ** -23 + 2.0 ** -25) + 2.0 ** -24
