"""yb_attn_run where single parts of its arithmetic could go wrong: caps far from
the scores, scores of -infinity under a cap."""
import math

import pytest
import torch

from lm_util import half_step, half_subnormal

pytestmark = pytest.mark.gpu

T = {"f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24


def capped_case(Sq, Sk, D, dt, scale, cap, gain, causal, seed=0):
    """(out, o, bound): attention of one head under a cap against its 64-bit form.

    As lm_util.attention_ref, but with the capped score in 32 bits as what it is: 16 u |s| for the tanh (polynomial
    and its coefficients 8 u; exponential form from 3/8 of the cap on: its argument 3 u, ex2 2^-22.5 and the
    reciprocal 2 u, which the slope of the tanh brings to under 15 u of its value), 4 u |s| as there."""
    import yb_ops

    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = T[dt]
    q = (torch.randn(1, Sq, 1, D, generator=g, device="cuda") * gain).to(dtype)
    k = torch.randn(1, Sk, 1, D, generator=g, device="cuda").to(dtype)
    v = torch.randn(1, Sk, 1, D, generator=g, device="cuda").to(dtype)
    att = yb_ops.Attention(1, 1, D, dtype, scale=scale, cap=cap, causal=causal)
    out = att(q, k, v)[0, :, 0].double()
    att.check()
    qd, kd, vd = (x[0, :, 0].double() for x in (q, k, v))
    scale, cap = (float(torch.tensor(x, dtype=torch.float32)) for x in (scale, cap))
    see = torch.ones(Sq, Sk, dtype=torch.bool, device="cuda")
    if causal:
        see = torch.arange(Sk, device="cuda")[None] <= torch.arange(Sq, device="cuda")[:, None] + Sk - Sq
    s = cap * torch.tanh(qd @ kd.T * scale / cap)
    mag = (qd.abs() @ kd.abs().T * scale).where(see, torch.zeros((), dtype=torch.float64, device="cuda"))
    smax = s.abs().where(see, torch.zeros((), dtype=torch.float64, device="cuda")).amax(-1)
    p = torch.softmax(s.masked_fill(~see, -math.inf), -1)
    o = p @ vd
    e = (D + 4) * U * mag.amax(-1) + 20 * U * smax
    a = half_step(dtype)
    bound = (a + 4 * e + 2.0 ** -20 + 2 * Sk * U)[:, None] * (p @ vd.abs()) + a * o.abs() + half_subnormal(dtype)
    return out, o, bound


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("scale,cap", [(0.125, 200.0), (0.125, 1000.0), (0.125, 1e4), (0.125, 1e6), (0.125, 1e30), (1.0, 1000.0),
                                       (1.0, 5e4), (0.01, 0.3), (0.125, 3e-5), (1.0, 5e-39)])
def test_caps_of_any_size(scale, cap, causal, dt):
    """Caps far above every score change next to nothing, those far below flatten every score."""
    for gain in (0.0, 0.4, 1.5, 8.0):
        for Sq, Sk, D in ((150, 300, 64), (3, 900, 40)):
            out, o, bound = capped_case(Sq, Sk, D, dt, scale, cap, gain, causal)
            over = (out - o).abs() - bound
            assert float(over.max()) <= 0, (gain, Sq, float(((out - o).abs() / bound).max()))


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("scale,cap,dot", [(32.0, 1e5, 32), (1.0, 4000.0, 96), (1.0, 1000.0, 32), (0.125, 500.0, 96),
                                           (0.125, 1e6, 8), (32.0, 1e5, 960)])
def test_equal_scores_weigh_equally(scale, cap, dot, dt):
    """Two keys of the same, exactly formed score, one among keys far below the cap, the other in a half block with
    one near the cap (seen by a neighbouring row): whichever form of the tanh each takes, their weights agree.

    Values 1 and -1: |o| <= half the relative difference of the weights, which is twice the error of a score,
    2 x 16 u s, and their roundings to the operands' type, a half step each; the result's own is of second order."""
    import yb_ops

    D, Sk = 8, 256
    dtype = T[dt]
    q = torch.zeros(1, 2, 1, D, device="cuda")
    q[0, 0, 0, 0] = 1.0
    q[0, 1, 0, 1] = 64.0
    k = torch.zeros(1, Sk, 1, D, device="cuda")
    v = torch.zeros(1, Sk, 1, D, device="cuda")
    far = 1.0
    while far * 64.0 * scale < 2.0 * cap and far < 2.0 ** 14:
        far *= 2.0
    k[0, 40, 0, 1] = far  # row 1 alone: about the cap
    k[0, 20, 0, 0] = k[0, 200, 0, 0] = dot
    # All other keys score -1024 for row 0, which weighs nothing beside the two.
    k[0, :, 0, 2] = -1.0
    k[0, 20, 0, 2] = k[0, 200, 0, 2] = 0.0
    q[0, 0, 0, 2] = 64.0 if scale * dot < 1000 else 1.0
    low = 1000.0 / scale / float(q[0, 0, 0, 2])
    k[0, :, 0, 2] *= min(2.0 ** math.ceil(math.log2(max(low, 1.0))), 2.0 ** 14)
    v[0, 20, 0, :] = 1.0
    v[0, 200, 0, :] = -1.0
    out = yb_ops.Attention(1, 1, D, dtype, scale=scale, cap=cap)(q.to(dtype), k.to(dtype), v.to(dtype))
    s = cap * math.tanh(dot * scale / cap)
    other = cap * math.tanh(-1000.0 / cap)
    assert s - other > 30 * math.log(2.0)  # the rest weighs nothing
    assert float(out[0, 0].double().abs().max()) <= (2 * 16 * U * s + 2 * half_step(dtype)) / 2 * (1 + 2.0 ** -7)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("slopes", [False, True])
@pytest.mark.parametrize("Sk", [3, 64, 200, 1500])
def test_scores_of_minus_infinity_under_a_cap(Sk, slopes, dt):
    """tanh(-infinity) = -1: such keys weigh e^(-cap) beside a score of 0, and all alike where there are no others."""
    import yb_ops

    dtype = T[dt]
    D, cap = 16, 2.0
    g = torch.Generator(device="cuda").manual_seed(Sk)
    v = torch.randn(1, Sk, 1, D, generator=g, device="cuda").to(dtype)
    q = torch.zeros(1, 2, 1, D, device="cuda", dtype=dtype)
    q[..., 0] = 1.0
    sl = torch.tensor([0.01], device="cuda") if slopes else None
    for finite in ([], [0], [Sk - 1], [Sk // 2]):
        k = torch.zeros(1, Sk, 1, D, device="cuda", dtype=dtype)
        k[..., 0] = -math.inf
        for j in finite:
            k[0, j, 0, 0] = 0.0
        att = yb_ops.Attention(1, 1, D, dtype, cap=cap)
        out = att(q, k, v, slopes=sl)
        att.check()
        s = torch.full((2, Sk), -cap, dtype=torch.float64, device="cuda")
        for j in finite:
            s[:, j] = 0.0
        if slopes:
            row = torch.arange(2, device="cuda")[:, None] + Sk - 2
            s -= 0.01 * (row - torch.arange(Sk, device="cuda")).abs().double()
        p = torch.softmax(s, -1)
        want = p @ v[0, :, 0].double()
        a = half_step(dtype)
        e = 20 * U * (cap + 0.01 * Sk)
        bound = (a + 4 * e + 2.0 ** -20 + 2 * Sk * U) * (p @ v[0, :, 0].double().abs()) + a * want.abs() + half_subnormal(dtype)
        assert float(((out[0, :, 0].double() - want).abs() - bound).max()) <= 0, finite
