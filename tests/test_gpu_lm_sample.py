"""yb_sample against its 64-bit form: tokens equal, log-probabilities within
2^-22 (the 32-bit rounding of the result, at most 2^-24 of |lp| < 4; larger ones
in proportion) plus 2^-40 for the fixed-point weights."""
import numpy as np
import pytest
import torch

from lm_util import sample_ref

pytestmark = pytest.mark.gpu

T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def run(logits, u, **kw):
    import yb_ops

    dev = {k: torch.tensor(v, dtype=torch.int32 if k == "top_k" else torch.float32).cuda() for k, v in kw.items()}
    token, lp = yb_ops.sample(logits, torch.tensor(u, dtype=torch.float32).cuda(), **dev)
    torch.cuda.synchronize()
    return token.cpu().numpy(), lp.cpu().numpy()


def check(logits, u, **kw):
    token, lp = run(logits, u, **kw)
    x = logits.double().cpu().numpy()
    f = {k: (np.asarray(v) if k == "top_k" else np.asarray(v, np.float32)) for k, v in kw.items()}
    for b in range(x.shape[0]):
        want, wlp = sample_ref(x[b], float(np.float32(u[b])), **{k: v[b] for k, v in f.items()})
        assert token[b] == want, (b, token[b], want)
        if np.isinf(wlp):
            assert lp[b] == wlp
        else:
            assert abs(lp[b] - wlp) <= 2.0 ** -22 * max(1.0, abs(wlp)) + 2.0 ** -40, (b, lp[b], wlp)


def logits_of(B, V, dt, seed, gain=2.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, V, generator=g) * gain
    x[:, torch.randint(0, V, (3,), generator=g)] += 6.0
    return x.to(T[dt]).cuda()


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V", [1, 2, 31, 1000, 4097, 50001, 131071, 262144])
def test_plain_and_filtered(V, dt):
    B = 9
    x = logits_of(B, V, dt, V)
    rng = np.random.default_rng(V)
    u = rng.random(B).astype(np.float32)
    check(x, u)
    check(x, u, temperature=[0.7] * B)
    check(x, u, temperature=[0.0, 1e-30, 0.3, 1.0, 1.7, 20.0, 1e30, float("inf"), -1.0])
    check(x, u, top_k=[0, 1, 2, 5, 50, 700, 3000, -3, 10 ** 9])
    check(x, u, top_p=[1.0, 0.99, 0.9, 0.5, 0.1, 1e-3, 0.0, -1.0, 2.0])
    check(x, u, min_p=[0.0, 1e-6, 0.01, 0.05, 0.3, 0.99, 1.0, 7.0, -1.0])
    check(x, u, temperature=[1.3] * B, top_k=[0, 40, 1000, 3, 40, 40, 600, 0, 9], top_p=[0.9] * 4 + [1.0, 0.3, 0.8] * 1 + [0.7, 0.95],
          min_p=[0.0, 0.02, 0.0, 0.0, 0.1, 0.0, 0.001, 0.05, 0.0])


@pytest.mark.parametrize("V", [700, 5000, 100003])
def test_ties(V):
    """Whole logits: every value is shared by many tokens, so each border falls among equals."""
    B = 12
    g = torch.Generator().manual_seed(5)
    x = torch.randint(-4, 5, (B, V), generator=g).float().cuda()
    u = np.linspace(0, 0.999, B).astype(np.float32)
    check(x, u, top_k=[1, 2, 3, 10, 77, 300, 511, 512, 513, V - 1, V, V + 1])
    check(x, u, top_p=list(np.linspace(0.05, 0.97, B)))
    check(x, u, top_k=[V // 2] * B, top_p=[0.6] * B)
    check(torch.zeros_like(x), u, top_k=[V // 3] * B)
    check(torch.zeros_like(x), u, top_p=[0.5] * B)
    check(torch.full_like(x, -3.4028234e38), u, top_p=[0.25] * B)  # all at the type's lowest value
    z = x.clone()
    z[:, ::2] = -0.0
    z[:, 1::2] = 0.0
    check(z, u, top_k=[7] * B)  # the two zeros are equal


def test_masked_and_odd_values():
    V, inf, nan = 2000, float("inf"), float("nan")
    x = logits_of(8, V, "f32", 3)
    x[0] = -inf
    x[1] = nan
    x[2, :-1] = -inf  # one token left, the last
    x[3, ::2] = nan
    x[4, 5] = inf
    x[4, 1200] = inf
    x[5, ::3] = -3.4028234e38
    x[6] = -inf
    x[6, 17] = -3.4028234e38
    x[7, 100:] = -inf
    u = np.array([0.3, 0.3, 0.9, 0.7, 0.6, 0.99, 0.5, 0.999], np.float32)
    for kw in ({}, dict(top_k=[20] * 8), dict(top_p=[0.9] * 8), dict(min_p=[0.1] * 8), dict(temperature=[0.0] * 8)):
        check(x, u, **kw)
    token, lp = run(x, u)
    assert token[0] == -1 and token[1] == -1 and lp[0] == -inf and token[2] == V - 1 and token[6] == 17


def test_random_numbers_at_the_ends():
    x = logits_of(6, 3000, "f32", 9)
    u = np.array([0.0, -0.5, 1.0, 2.0, float("nan"), np.nextafter(np.float32(1), np.float32(0))], np.float32)
    check(x, u)
    check(x, u, top_k=[9] * 6)


def test_strides_and_alignment():
    big = logits_of(10, 5003, "bf16", 4)
    u = np.random.default_rng(1).random(5).astype(np.float32)
    check(big[::2, 1:4999], u, top_p=[0.9] * 5)
    check(big[:5, 3:], u, top_k=[30] * 5)
    check(big[:1].expand(5, -1), u)  # one row for all


def test_many_rows():
    B, V = 700, 1500
    x = logits_of(B, V, "f16", 6)
    u = np.random.default_rng(2).random(B).astype(np.float32)
    check(x, u, temperature=[0.9] * B, top_k=[60] * B, top_p=[0.92] * B)


def test_output_buffers_streams_and_replay():
    """A captured call follows its inputs; the capture and an eager call on another stream agree."""
    import yb_ops

    V, B = 40000, 3
    x = logits_of(B, V, "f32", 12)
    u = torch.rand(B, device="cuda")
    k = torch.full((B,), 50, dtype=torch.int32, device="cuda")
    yb_ops.sample(x, u, top_k=k)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        token, lp = yb_ops.sample(x, u, top_k=k)
    side = torch.cuda.Stream()
    for seed in range(4):
        x.copy_(logits_of(B, V, "f32", 100 + seed))
        u.uniform_()
        k.fill_(1 + 20 * seed)
        g.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            t2, lp2 = yb_ops.sample(x, u, top_k=k)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert torch.equal(token, t2) and torch.equal(lp, lp2)


def test_binding_refusals():
    import yb_ops
    import yolo_b200 as yb

    x, u = torch.zeros(2, 10, device="cuda"), torch.zeros(2, device="cuda")
    for bad in (lambda: yb_ops.sample(x.cpu(), u), lambda: yb_ops.sample(x.int(), u), lambda: yb_ops.sample(x[0], u),
                lambda: yb_ops.sample(x.t(), u), lambda: yb_ops.sample(x, u[:1]), lambda: yb_ops.sample(x, u.double()),
                lambda: yb_ops.sample(x, None), lambda: yb_ops.sample(x, u, top_k=u),
                lambda: yb_ops.sample(x, u, token=torch.zeros(2, dtype=torch.int64, device="cuda"))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(yb.YBError):
        yb_ops.sample(torch.zeros(1, 262145, device="cuda"), u[:1])
    t, _ = yb_ops.sample(x[:0], u[:0])
    assert t.shape == (0,)
