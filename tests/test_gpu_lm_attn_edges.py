"""yb_attn_run where single parts of its arithmetic could go wrong: caps far from
the scores, scores of -infinity under a cap, and rows that are computed again
because of a value that is not finite."""
import math

import pytest
import torch

from lm_util import attention_ref, check_attention, half_step, half_subnormal

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


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("cap,slopes", [(0.0, False), (20.0, False), (0.0, True), (20.0, True)])
def test_rows_computed_again(cap, slopes, causal, dt):
    """A NaN in one dimension of some values: rows that see it have it there, their other dimensions as ever."""
    import yb_ops

    dtype = T[dt]
    for n, (B, Sq, Sk, Hq, Hkv, D) in enumerate([(1, 200, 200, 4, 2, 64), (2, 3, 700, 8, 2, 128), (3, 1, 33, 2, 1, 8),
                                                  (1, 130, 1500, 3, 1, 72), (160, 2, 300, 1, 1, 40)]):
        g = torch.Generator(device="cuda").manual_seed(n)
        q, k, v, out = (torch.randn(B, s, h, D, generator=g, device="cuda").to(dtype)
                        for s, h in ((Sq, Hq), (Sk, Hkv), (Sk, Hkv), (Sq, Hq)))
        v[:, Sk // 2, :, 5] = math.nan
        v[:, 1, :, 0] = math.nan
        kw = {"slopes": torch.tensor([2.0 ** -(h + 3) for h in range(Hq)], device="cuda") if slopes else None}
        if n == 1:
            kw["k_len"] = torch.tensor([700, 351], dtype=torch.int32, device="cuda")
        if n == 3 and causal:
            kw["prefix"] = torch.tensor([800], dtype=torch.int32, device="cuda")
        before = out.clone()
        att = yb_ops.Attention(Hq, Hkv, D, dtype, cap=cap, causal=causal)
        att(q, k, v, out=out, **kw)
        att.check()
        check_attention(out, before, attention_ref(q, k, v, att.scale, cap, causal, dt=dtype, **kw))
        assert bool(out.isnan().any())


def test_rows_computed_again_over_many_keys():
    """160 sequences of 300,000 keys (one tensor for all) and 128 rows, a NaN seen by every row: two tiles to a CTA, whose
    other roles wait while the first one's rows are computed again (32 rows of a warp, once 0.23 us a key: 2.2 s, where
    a wait gives up after 2)."""
    import yb_ops

    B, Sq, Sk, D = 160, 128, 300000, 8
    g = torch.Generator(device="cuda").manual_seed(0)
    q = torch.randn(B, Sq, 1, D, generator=g, device="cuda").bfloat16()
    k = torch.randn(1, Sk, 1, D, generator=g, device="cuda").bfloat16().expand(B, -1, -1, -1)
    v = torch.ones(1, Sk, 1, D, device="cuda").bfloat16()
    v[:, 0, :, 5] = math.nan
    att = yb_ops.Attention(1, 1, D, torch.bfloat16)
    out = att(q, k, v.expand(B, -1, -1, -1))
    att.check()
    nan = torch.isnan(out)
    assert bool(nan[..., 5].all()) and int(nan.sum()) == B * Sq
    # Values of 1 average to 1; sums of Sk positive terms in 32 bits on either side.
    rest = torch.cat((out[..., :5], out[..., 6:]), -1).double()
    assert float((rest - 1).abs().max()) <= 2 * Sk * U + half_step(torch.bfloat16)


@pytest.mark.parametrize("Sq,Sk", [(1, 2), (1, 100), (200, 300), (1, 5000), (3, 20000)])
def test_values_near_the_end_of_the_range(Sq, Sk):
    """Averages of bf16 values of 3e38 are such values, though their sum is past 32 bits."""
    import yb_ops

    g = torch.Generator(device="cuda").manual_seed(Sk)
    q = torch.randn(1, Sq, 2, 64, generator=g, device="cuda").bfloat16()
    k = torch.randn(1, Sk, 1, 64, generator=g, device="cuda").bfloat16()
    v = torch.full((1, Sk, 1, 64), 3e38, device="cuda").bfloat16()
    v[..., 1] *= -1
    v[..., 2] = 1.0
    v[..., 3] = torch.randn(1, Sk, 1, generator=g, device="cuda").bfloat16() * 1e37
    att = yb_ops.Attention(2, 1, 64, torch.bfloat16)
    out = torch.zeros_like(q)
    att(q, k, v, out=out)
    att.check()
    check_attention(out, out, attention_ref(q, k, v, att.scale))


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("near_end", [False, True])
@pytest.mark.parametrize("lead", [9, 20, 33, 34, 35, 40, 50, 60, 61, 62, 66, 66.5, 67, 80])
def test_pieces_of_very_different_references(lead, near_end, dt):
    """Keys of score 0 but for two, a unit apart, far above and in pieces of different CTAs: either may outgrow its
    piece's reference by any amount, or be it, and both count.  With a value near the end of the range beside them the
    piece is computed again, from other references."""
    import yb_ops

    dtype = T[dt]
    Sk, D = 20000, 8
    q = torch.zeros(1, 1, 1, D, device="cuda").to(dtype)
    q[..., 0] = 1.0
    for a, b in ((300, 15000), (15000, 300), (19999, 70), (130, 19900), (10000, 5000), (64, 19840)):
        k = torch.zeros(1, Sk, 1, D, device="cuda").to(dtype)
        v = torch.zeros(1, Sk, 1, D, device="cuda").to(dtype)
        k[0, a, 0, 0], k[0, b, 0, 0] = lead, lead + 1
        v[0, a], v[0, b] = 1.0, -1.0
        if near_end and dt == "bf16":
            v[0, a, 0, 7] = v[0, (a + 1) % Sk, 0, 7] = 3e38
        out = torch.zeros_like(q)
        att = yb_ops.Attention(1, 1, D, dtype, scale=1.0)
        att(q, k, v, out=out)
        att.check()
        check_attention(out, out, attention_ref(q, k, v, 1.0))


def test_an_object_that_dies_within_a_capture():
    """Its handle is not freed there (that synchronizes, which a capture does not survive)."""
    import yb_ops

    g = torch.Generator(device="cuda").manual_seed(0)
    q, k, v = (torch.randn(1, n, 2, 64, generator=g, device="cuda").bfloat16() for n in (1, 300, 300))
    att, other = (yb_ops.Attention(2, 2, 64, torch.bfloat16) for _ in range(2))
    want = att(q, k, v)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = att(q, k, v)
        del other
    graph.replay()
    att.check()
    assert torch.equal(out, want)
