"""yb_sample where its fixed-point weights could go wrong: neighbours of the
largest logit at small temperatures, and tokens of very small weight."""
import math

import numpy as np
import pytest
import torch

from lm_util import sample_ref
from test_gpu_lm_sample import run

pytestmark = pytest.mark.gpu

OFF = {"none": {}, "min_p": dict(min_p=[0.05] * 6), "top_p": dict(top_p=[0.9] * 6), "top_k": dict(top_k=[40] * 6),
       "off": dict(top_k=[0] * 6, top_p=[1.0] * 6, min_p=[0.0] * 6)}


def steps_below(x, n):
    x = np.float32(x)
    for _ in range(n):
        x = np.nextafter(x, np.float32(-np.inf))
    return x


def check(x, u, t, **kw):
    """Tokens equal to those of the 64-bit form, in which tokens below 2^-45 of the largest weight, which yb_lm.h says
    are never chosen, are left out (together they weigh less than V 2^-45 < 2^-32); log-probabilities within 2^-22."""
    token, lp = run(torch.from_numpy(x).cuda(), u, temperature=[t] * len(x), **kw)
    for b in range(len(x)):
        row = x[b].astype(np.float64)
        row[(row.max() - row) / t > 45.0 * np.log(2.0)] = -np.inf
        want, wlp = sample_ref(row, float(u[b]), temperature=t, **{k: v[b] for k, v in kw.items()})
        assert token[b] == want, (t, b, token[b], want)
        assert abs(lp[b] - wlp) <= 2.0 ** -22 * max(1.0, abs(wlp)), (t, b, lp[b], wlp)


@pytest.mark.parametrize("top", [12.3, 0.7, -7.1, 29.0, 3e12, -1e-3])
@pytest.mark.parametrize("filters", list(OFF))
def test_neighbours_of_the_largest_logit(top, filters):
    """One to three 32-bit steps below the maximum, at temperatures for which a step is a fraction of an octave and
    ones for which it is 10^10 octaves: those tokens weigh what the formula says, mostly nothing."""
    V, B = 4000, 6
    x = np.full((B, V), top, np.float32) - np.abs(np.float32(top)) * np.linspace(0.1, 1.0, V, dtype=np.float32)
    for b in range(B):
        at = [(7 + 613 * b) % V, (900 + 131 * b) % V, (2500 + 77 * b) % V, (3999 - 5 * b) % V]
        order = [(0, 1, 2, 3), (3, 2, 1, 0), (1, 0, 1, 1), (1, 1, 0, 2), (2, 1, 1, 0), (0, 3, 1, 1)][b]
        for i, n in zip(at, order):
            x[b, i] = steps_below(top, n)
    u = np.array([0.0, 0.1, 0.35, 0.6, 0.9, 0.999], np.float32)
    step = float(np.float32(top) - steps_below(top, 1))
    # In octaves a step: 2^-2 up to 2^35, where fp64 meets its own steps, and some tiny temperatures as they are.
    for t in [step * 2.0 ** -e for e in range(-2, 36)] + [1e-6, 1e-8, 1e-9, 1e-10, 1e-12, 1e-14, 1e-16]:
        t = float(np.float32(t))
        if not t > 0.0:
            continue
        check(x, u, t, **OFF[filters])


def test_every_row_gets_a_token():
    """Rows on which nothing but the maximum weighs anything: its token, with log-probability 0."""
    V = 9000
    for t in (1e-9, 2e-9, 1e-10, 1e-12):
        x = np.full((3, V), -3.0, np.float32)
        x[:, 100:8000:3] = steps_below(12.3, 1)
        x[0, 0] = x[1, 4500] = x[2, V - 1] = np.float32(12.3)
        token, lp = run(torch.from_numpy(x).cuda(), [0.0, 0.5, 0.9999], temperature=[t] * 3)
        assert token.tolist() == [0, 4500, V - 1] and lp.tolist() == [0.0, 0.0, 0.0], t


@pytest.mark.parametrize("octaves", [20, 30, 36, 42, 44])
@pytest.mark.parametrize("V", [300, 3000, 50001])
def test_log_probability_of_light_tokens(V, octaves):
    """A peak at the last index and tokens of weight 2^-octaves before it: u = 0 takes the first of those.  Its
    log-probability is that of its logit, not of its weight in whole units of 2^-44.

    Bound: the result's rounding, half a step of 2^-24 |lp|; the whole weight, summed in units of 2^-44, is off by at
    most V 2^-45 < 2^-27 of the peak's; 2^-22 max(1, |lp|) covers both."""
    x = np.full((6, V), -(octaves + 0.37) * math.log(2.0), np.float32)  # no whole number of 2^-44
    x -= np.linspace(0.0, 0.2, V, dtype=np.float32)
    x[:, -1] = 0.0
    for kw in ({}, dict(top_k=[V - 1, 2, 7, 40, 250, 290]), dict(min_p=[2.0 ** -46] * 6)):
        token, lp = run(torch.from_numpy(x).cuda(), [0.0] * 6, **kw)
        for b in range(6):
            want, wlp = sample_ref(x[b], 0.0, **{k: v[b] for k, v in kw.items()})
            assert want == 0 and token[b] == 0
            assert abs(lp[b] - wlp) <= 2.0 ** -22 * max(1.0, abs(wlp)), (lp[b], wlp)
