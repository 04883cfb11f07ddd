"""64-bit forms of the text-decoder operators (include/yb_lm.h), with the error
bounds their tests hold the kernels to."""
import math

import numpy as np
import torch


def half_step(dt) -> float:
    return torch.finfo(dt).eps / 2


def half_subnormal(dt) -> float:
    """The rounding error of values below the type's smallest normal number."""
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2


def attention_ref(q, k, v, scale, cap=0.0, causal=False, q_len=None, k_len=None, prefix=None, key_range=None,
                  slopes=None, dt=None):
    """(o, bound, used) in float64: o [B, Sq, Hq, D], zeros where nothing is visible; bound, the error allowed per
    element; used [B, Sq], the rows in use.

    With p the exact weights (sum 1), s the scores, a the type's half step, and 32-bit arithmetic of unit u = 2^-24:
      score error  e = (D + 4) u scale sum|q||k|      products and sums of the dot
                     + 4 u |s|max                     scaling, log2(e), the difference to the maximum, bias
                     + cap 2^-20                      tanh (documented here as the allowance of the capped score)
      each weight is off by the factor 1 + 2e (its own error and the maximum's) + 2^-21 (exp2, 2 ulp, both in the
      weight and the sum), and is rounded to the operand type (a);
      sums of n positive terms in 32 bits: n u (weights and values);
      |o - exact| <= (a + 4 e + 2^-20 + 2 n u) sum p|v| + a |o|.
    """
    dt = dt or q.dtype
    B, Sq, Hq, D = q.shape
    Sk, Hkv = k.shape[1], k.shape[2]
    dev = q.device
    G = Hq // Hkv
    qd = q.double().permute(0, 2, 1, 3)
    kd = k.double().permute(0, 2, 1, 3).repeat_interleave(G, 1)
    vd = v.double().permute(0, 2, 1, 3).repeat_interleave(G, 1)
    ql = q_len.long().clamp(0, Sq) if q_len is not None else torch.full((B,), Sq, device=dev)
    kl = k_len.long().clamp(0, Sk) if k_len is not None else torch.full((B,), Sk, device=dev)
    i, j = torch.arange(Sq, device=dev), torch.arange(Sk, device=dev)
    pos = (kl - ql)[:, None] + i[None]
    see = (j[None, None] < kl[:, None, None]).expand(B, Sq, Sk)
    if causal:
        c = j[None, None] <= pos[..., None]
        if prefix is not None:
            c = c | (j[None, None] < prefix.long()[:, None, None])
        see = see & c
    if key_range is not None:
        r = key_range.long()
        see = see & (j >= r[..., 0:1]) & (j < r[..., 1:2])
    see = see[:, None]
    u = 2.0 ** -24
    s = qd @ kd.transpose(2, 3) * scale
    mag = qd.abs() @ kd.abs().transpose(2, 3) * scale
    if cap:
        s = cap * torch.tanh(s / cap)
    if slopes is not None:
        s = s - slopes.double()[None, :, None, None] * (pos[..., None] - j).abs().double()[:, None]
    neg = torch.full((), -math.inf, dtype=torch.float64, device=dev)
    s = torch.where(see, s, neg)
    m = s.amax(-1, keepdim=True) if Sk else torch.full((B, Hq, Sq, 1), -math.inf, dtype=torch.float64, device=dev)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    p = torch.where(see, p, 0.0)
    p = p / torch.where(p.sum(-1, keepdim=True) == 0.0, 1.0, p.sum(-1, keepdim=True))
    # Masked keys take no part, whatever they hold: their value rows count as zero for the rows that do not see them.
    clean = torch.where(torch.isfinite(vd), vd, 0.0)
    o = p @ clean
    bad = (see & ~torch.isfinite(vd).all(-1)[:, :, None]).any(-1)  # rows that see a non-finite value
    if bool(bad.any()):
        for b, h, r in bad.nonzero().tolist():
            at = see[b, 0, r].nonzero()[:, 0]
            o[b, h, r] = (p[b, h, r, at, None] * vd[b, h, at]).sum(0)
    seen = torch.where(see, mag, 0.0)
    smax = torch.where(see, s.abs(), 0.0)
    zero = torch.zeros((B, Hq, Sq), dtype=torch.float64, device=dev)
    e = (D + 4) * u * (seen.amax(-1) if Sk else zero) + 4 * u * (smax.amax(-1) if Sk else zero) + cap * 2.0 ** -20
    a = half_step(dt)
    bound = (a + 4 * e + 2.0 ** -20 + 2 * Sk * u)[..., None] * (p @ clean.abs()) + a * o.abs() + half_subnormal(dt)
    used = i[None] < ql[:, None]
    return o.permute(0, 2, 1, 3), bound.permute(0, 2, 1, 3), used


def check_attention(out, before, ref):
    """out against attention_ref's result; rows out of use must equal `before` bit for bit."""
    o, bound, used = ref
    assert torch.equal(out[~used], before[~used])
    got, want, tol = out[used].double(), o[used], bound[used]
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    ok = ~torch.isnan(want)
    over = ((got - want).abs() - tol)[ok]
    assert over.numel() == 0 or float(over.max()) <= 1e-30, \
        f"over the bound by {float(over.max()):.3g}, worst ratio {float(((got - want).abs() / tol.clamp_min(1e-300))[ok].max()):.3g}"


def rotate_ref(x, weight, pos, inv_freq, eps, weight_add, interleaved):
    """(y, bound) in float64 for x [..., S, H, D] at positions pos [..., S].

    In 32 bits of unit u = 2^-24: sum of D squares, division, root and reciprocal (D + 6) u / 2 + 3 u relative, weight
    and two products 3 u: under (D / 2 + 10) u of |y|; cos and sin to 4 u (their own 2 ulp, the reduced angle's
    rounding put back to second order), three operations a rotated element: 8 u (|y0| + |y1|); then the type's half
    step of the result."""
    D, R = x.shape[-1], 2 * inv_freq.shape[0]
    xd = x.double()
    w = (torch.ones(D, dtype=torch.float64, device=x.device) if weight is None else weight.double()) + weight_add
    y = xd / torch.sqrt((xd * xd).mean(-1, keepdim=True) + eps) * w
    ang = (pos.double()[..., None] * inv_freq)[..., None, :]
    c, s = torch.cos(ang), torch.sin(ang)
    i = torch.arange(R // 2, device=x.device)
    l, r = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
    out, mag = y.clone(), y.abs().clone()
    out[..., l] = y[..., l] * c - y[..., r] * s
    out[..., r] = y[..., r] * c + y[..., l] * s
    mag[..., l] = mag[..., r] = y[..., l].abs() + y[..., r].abs()
    u = 2.0 ** -24
    return out, (D / 2 + 18) * u * mag + half_step(x.dtype) * (1 + 2.0 ** -10) * out.abs() + half_subnormal(x.dtype)


def sample_ref(logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    """(token, logprob) of one row of float64 logits."""
    x = np.asarray(logits, np.float64).copy()
    big = float(np.finfo(np.float32).max)
    x[np.isposinf(x)] = big
    live = np.flatnonzero(x > -np.inf)  # NaN compares false
    if live.size == 0:
        return -1, -math.inf
    t = 1.0 if temperature is None else float(temperature)
    best = int(live[np.argmax(x[live])])
    if not t > 0.0:
        return best, 0.0
    w = np.exp((x[live] - x[best]) / t)
    order = np.argsort(-x[live], kind="stable")
    n = order.size if top_k is None or top_k <= 0 else min(int(top_k), order.size)
    p = 1.0 if top_p is None or not top_p < 1.0 else float(top_p)
    if p < 1.0:
        mass = np.cumsum(w[order[:n]])
        n = 1 + int(np.sum(mass[:-1] < p * mass[-1]))
    kept = np.zeros(live.size, bool)
    kept[order[:n]] = True
    if min_p is not None and min_p > 0.0:
        kept &= w >= min(float(min_p), 1.0)
    at = np.flatnonzero(kept)
    mass = np.cumsum(w[at])
    u = min(max(float(u), 0.0), 1.0) if not math.isnan(u) else 0.0
    k = min(int(np.searchsorted(mass, u * mass[-1], side="right")), at.size - 1)
    if u >= 1.0:
        k = at.size - 1
    return int(live[at[k]]), math.log(w[at[k]] / mass[-1]) if w[at[k]] > 0 else -math.inf
