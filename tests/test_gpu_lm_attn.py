"""yb_attn_run against its 64-bit form (bounds in lm_util.attention_ref)."""
import pytest
import torch

from lm_util import attention_ref, check_attention

pytestmark = pytest.mark.gpu

T = {"f16": torch.float16, "bf16": torch.bfloat16}


def tensors(B, Sq, Sk, Hq, Hkv, D, dt, seed=0, gain=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def n(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    dtype = T[dt]
    return ((n(B, Sq, Hq, D) * gain).to(dtype), n(B, Sk, Hkv, D).to(dtype), n(B, Sk, Hkv, D).to(dtype),
            n(B, Sq, Hq, D).to(dtype))


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def run_case(B, Sq, Sk, Hq, Hkv, D, dt="bf16", cap=0.0, causal=False, scale=None, seed=0, gain=1.5, edit=None, **kw):
    import yb_ops

    q, k, v, out = tensors(B, Sq, Sk, Hq, Hkv, D, dt, seed, gain)
    if edit:
        edit(q, k, v)
    if kw.pop("slopes", False):
        kw["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / Hq) for h in range(Hq)], device="cuda")
    before = out.clone()
    att = yb_ops.Attention(Hq, Hkv, D, T[dt], scale=scale, cap=cap, causal=causal)
    att(q, k, v, out=out, **kw)
    att.check()
    ref = attention_ref(q, k, v, att.scale, cap, causal, dt=T[dt], **kw)
    check_attention(out, before, ref)
    return out


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("D", [8, 40, 64, 72, 80, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_head_dims(D, causal, dt):
    run_case(2, 150, 150, 4, 2, D, dt, causal=causal, seed=D)


@pytest.mark.parametrize("Sq,Sk", [(1, 1), (1, 2), (1, 127), (1, 128), (1, 129), (1, 1000), (2, 2), (5, 130), (127, 127),
                                   (128, 128), (129, 129), (255, 257), (256, 512), (300, 64), (513, 640), (1, 9000),
                                   (7, 5000), (90, 3500)])
@pytest.mark.parametrize("causal", [False, True])
def test_lengths(Sq, Sk, causal):
    run_case(2, Sq, Sk, 4, 2, 64, causal=causal, seed=Sq + Sk)


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (3, 3), (7, 1), (8, 1), (14, 2), (12, 4), (40, 2), (128, 1), (130, 1),
                                    (100, 1)])
@pytest.mark.parametrize("Sq,Sk", [(1, 333), (70, 200)])
def test_head_groups(Hq, Hkv, Sq, Sk):
    run_case(2, Sq, Sk, Hq, Hkv, 64, "f16", causal=True, seed=Hq)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("cap", [1.0, 20.0, 50.0])
@pytest.mark.parametrize("gain", [0.5, 1.5, 12.0])
def test_cap(cap, gain, dt):
    run_case(1, 200, 300, 4, 1, 64, dt, cap=cap, gain=gain)
    run_case(2, 1, 700, 4, 1, 128, dt, cap=cap, gain=gain, causal=True)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_slopes(cap, causal, dt):
    run_case(1, 260, 260, 6, 3, 80, dt, cap=cap, causal=causal, slopes=True)
    run_case(2, 3, 900, 6, 3, 64, dt, cap=cap, causal=causal, slopes=True)


def test_ragged():
    for Sq, Sk, ql, kl in [(1, 600, [1, 1, 1, 0, 1], [600, 1, 128, 77, 0]), (300, 400, [300, 1, 0, 129, 300], [400, 1, 50, 300, 10]),
                           (40, 3000, [40, 1, 39, 40, 7], [3000, 129, 2500, 1, 40]), (4, 100, [9, -3, 4, 4, 2], [200, 50, -7, 3, 100])]:
        for causal in (False, True):
            run_case(5, Sq, Sk, 4, 2, 64, causal=causal, q_len=i32(ql), k_len=i32(kl))


def test_tiles_without_keys_between_others():
    """Many short sequences, every second one without a key: a CTA goes through tiles with and without work."""
    B = 400
    kl = [(b * 37) % 500 + 1 if b % 2 else 0 for b in range(B)]
    ql = [3 if b % 5 else 0 for b in range(B)]
    for causal in (False, True):
        run_case(B, 3, 512, 8, 4, 64, causal=causal, q_len=i32(ql), k_len=i32(kl))
        run_case(60, 3, 3000, 8, 4, 64, causal=causal, k_len=i32([6 * k for k in kl[:60]]))


@pytest.mark.parametrize("Sk", [500, 3000])
def test_runs_of_tiles_without_keys(Sk):
    """Runs of sequences without a key, of every length, between ones that have some: the roles of a CTA pass the empty
    ones at their own pace and must still meet at the others (att.check reports a wait that ran out)."""
    import yb_ops

    B = 600
    kl = [0] * B
    at = 0
    for run in range(1, 30):
        at += run % 7 + 1
        if at < B:
            kl[at] = (run * 911) % Sk + 1
    for at in range(200, B, 3):
        kl[at] = (at * 37) % Sk + 1
    q, k, v, out = tensors(B, 1, Sk, 16, 8, 64, "bf16")
    att = yb_ops.Attention(16, 8, 64, torch.bfloat16, causal=True)
    want = None
    for _ in range(30):
        got = att(q, k, v, k_len=i32(kl))
        want = got if want is None else want
        assert torch.equal(got, want)
    att.check()
    run_case(B, 1, Sk, 4, 2, 64, causal=True, k_len=i32(kl))


def test_prefix():
    for Sq, Sk in [(300, 300), (100, 700), (1, 400)]:
        run_case(4, Sq, Sk, 4, 2, 64, causal=True, prefix=i32([0, 1, 200, 10 ** 6]))
        run_case(4, Sq, Sk, 4, 2, 64, causal=True, prefix=i32([-5, 130, 64, 128]), k_len=i32([Sk, Sk // 2, 100, 5]),
                 cap=30.0)


def ranges(B, S, cuts):
    r = torch.zeros(B, S, 2, dtype=torch.int32)
    edges = [0] + cuts + [S]
    for a, e in zip(edges[:-1], edges[1:]):
        r[:, a:e, 0], r[:, a:e, 1] = a, e
    return r.cuda()


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("slopes", [False, True])
def test_documents(causal, slopes):
    run_case(1, 700, 700, 4, 2, 64, causal=causal, slopes=slopes, key_range=ranges(1, 700, [1, 2, 130, 131, 500, 699]))
    run_case(2, 300, 300, 2, 2, 128, "f16", causal=causal, slopes=slopes, key_range=ranges(2, 300, [128, 256]),
             k_len=i32([300, 200]), q_len=i32([300, 200]))


def test_rows_that_see_nothing():
    r = ranges(1, 300, [100])
    r[:, 50:60] = 0  # empty
    r[:, 60, 0], r[:, 60, 1] = 7, 3  # end before begin
    r[:, 61, 0], r[:, 61, 1] = 290, 10 ** 9  # past the end
    r[:, 62, 0], r[:, 62, 1] = -(10 ** 9), 4
    r[:, 63, 0], r[:, 63, 1] = 2 ** 31 - 1, 2 ** 31 - 1
    r[:, 64, 0], r[:, 64, 1] = -(2 ** 31), -(2 ** 31)
    out = run_case(1, 300, 300, 4, 2, 64, causal=False, key_range=r)
    assert not bool(out[:, 50:61].any()) and not bool(out[:, 63:65].any())
    run_case(1, 300, 300, 4, 2, 64, causal=True, key_range=r)
    # More rows than keys: the first rows lie before every key.
    out = run_case(1, 300, 40, 4, 2, 64, causal=True)
    assert not bool(out[:, :260].any())
    out = run_case(2, 5, 0, 4, 2, 64)
    assert not bool(out.any())


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), "low"])
@pytest.mark.parametrize("Sq", [1, 200])
def test_unused_keys_may_hold_anything(bad, Sq):
    """Keys past k_len, and those of other documents, must not reach a row."""
    def edit(q, k, v):
        x = torch.finfo(k.dtype).min if bad == "low" else bad
        for t in (k, v):
            t[0, 150:] = x
            t[1, 300:] = x

    run_case(2, Sq, 512, 4, 2, 64, causal=False, k_len=i32([150, 300]), edit=edit)
    run_case(2, Sq, 512, 4, 2, 128, "f16", causal=True, k_len=i32([150, 300]), q_len=i32([min(Sq, 150), Sq]), edit=edit,
             cap=30.0, slopes=True)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_masked_documents_may_hold_anything(bad):
    def edit(q, k, v):
        k[:, 40:60] = bad
        v[:, 40:60, :, 3:9] = bad
        v[:, 255:258] = bad

    r = ranges(1, 300, [40, 60, 255, 258])
    for causal in (False, True):
        import yb_ops

        q, k, v, out = tensors(1, 300, 300, 4, 2, 64, "bf16")
        edit(q, k, v)
        att = yb_ops.Attention(4, 2, 64, torch.bfloat16, causal=causal)
        att(q, k, v, out=out, key_range=r)
        att.check()
        # The rows that see none of it equal those of clean inputs.
        q2, k2, v2, _ = tensors(1, 300, 300, 4, 2, 64, "bf16")
        ref = attention_ref(q2, k2, v2, att.scale, causal=causal, key_range=r)
        free = torch.ones(300, dtype=torch.bool, device="cuda")
        free[40:60] = False
        free[255:258] = False
        o, bound, _ = ref
        assert bool(torch.isfinite(out[0, free].float()).all())
        assert float(((out.double() - o).abs() - bound)[0, free].max()) <= 0
        assert bool((~torch.isfinite(out[0, 255:258].float())).all())


def test_causal_rows_before_a_bad_key():
    """Rows before a NaN value do not see it; those from it on do."""
    import yb_ops

    for Sq, Sk, at in [(300, 300, 140), (300, 300, 0), (3, 900, 898)]:
        q, k, v, out = tensors(1, Sq, Sk, 4, 2, 64, "bf16")
        v[0, at, :, 5] = float("nan")
        att = yb_ops.Attention(4, 2, 64, torch.bfloat16, causal=True)
        att(q, k, v, out=out)
        att.check()
        nan = torch.isnan(out[0, :, :, 5].float())
        row = torch.arange(Sq, device="cuda") + Sk - Sq
        assert torch.equal(nan, (row >= at)[:, None].expand_as(nan))
        other = out[0].clone()
        other[..., 5] = 0
        assert bool(torch.isfinite(other.float()).all())


def test_nan_scores_reach_their_rows_only():
    import yb_ops

    q, k, v, out = tensors(1, 200, 200, 4, 2, 64, "bf16")
    q[0, 17, 2, 0] = float("nan")
    q[0, 130, :, 0] = float("inf")
    att = yb_ops.Attention(4, 2, 64, torch.bfloat16)
    att(q, k, v, out=out)
    att.check()
    nan = torch.isnan(out[0].float()).any(-1)
    want = torch.zeros_like(nan)
    want[17, 2] = True
    want[130] = True
    assert torch.equal(nan, want)


def test_layouts():
    """Caches with heads before rows, slices of a packed projection, one cache for all sequences."""
    import yb_ops

    B, Sq, Sk, Hq, Hkv, D = 3, 130, 200, 6, 2, 64
    q, k, v, out = tensors(B, Sq, Sk, Hq, Hkv, D, "bf16")
    att = yb_ops.Attention(Hq, Hkv, D, torch.bfloat16, causal=True)
    want = att(q, k, v)
    kh = k.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    vh = v.permute(1, 0, 2, 3).contiguous().permute(1, 0, 2, 3)
    qh = q.permute(2, 1, 0, 3).contiguous().permute(2, 1, 0, 3)
    oh = torch.zeros(Hq, B, Sq, D, dtype=q.dtype, device="cuda").permute(1, 2, 0, 3)
    assert torch.equal(att(qh, kh, vh, out=oh), want)
    pack = torch.randn(B, Sk, (Hq + 2 * Hkv) * D + 16, device="cuda").bfloat16()
    qp = pack[:, :Sq, 8: 8 + Hq * D].unflatten(-1, (Hq, D))
    kp = pack[..., 8 + Hq * D: 8 + (Hq + Hkv) * D].unflatten(-1, (Hkv, D))
    vp = pack[..., 8 + (Hq + Hkv) * D: 8 + (Hq + 2 * Hkv) * D].unflatten(-1, (Hkv, D))
    assert torch.equal(att(qp, kp, vp), att(qp.contiguous(), kp.contiguous(), vp.contiguous()))
    one = att(q, k[:1].expand(B, -1, -1, -1), v[:1].expand(B, -1, -1, -1))
    assert torch.equal(one, att(q, k[:1].repeat(B, 1, 1, 1), v[:1].repeat(B, 1, 1, 1)))
    wide = torch.randn(B, Sk, Hkv, 2 * D, device="cuda").bfloat16()  # rows wider than the head
    assert torch.equal(att(q, wide[..., :D], wide[..., D:]), att(q, wide[..., :D].contiguous(), wide[..., D:].contiguous()))
    att.check()


def test_offsets_past_32_bits():
    import yb_ops

    Sk, H, D, stride = 36000, 2, 64, 65536
    big = torch.empty(Sk * stride, dtype=torch.bfloat16, device="cuda")
    kv = big.view(Sk, stride)[:, : 2 * H * D].view(1, Sk, 2 * H, D)
    k, v = kv[:, :, :H], kv[:, :, H:]
    assert (Sk - 1) * k.stride(1) > 2 ** 31
    k.normal_()
    v.normal_()
    q = torch.randn(1, 2, 4, D, device="cuda").bfloat16()
    att = yb_ops.Attention(4, H, D, torch.bfloat16, causal=True)
    got = att(q, k, v)
    att.check()
    check_attention(got, got, attention_ref(q, k, v, att.scale, causal=True))


def test_same_result_every_time():
    import yb_ops

    for Sq, Sk in [(1, 20000), (300, 600)]:
        q, k, v, _ = tensors(2, Sq, Sk, 8, 2, 128, "bf16")
        att = yb_ops.Attention(8, 2, 128, torch.bfloat16, causal=True)
        want = att(q, k, v)
        for _ in range(5):
            assert torch.equal(att(q, k, v), want)


def test_two_streams_and_two_captures():
    """Calls in flight at once, and two captured graphs replayed at once, do not share scratch."""
    import yb_ops

    att = yb_ops.Attention(8, 2, 64, torch.bfloat16, causal=True)
    sets = [tensors(2, 1, 12000, 8, 2, 64, "bf16", seed=s)[:3] for s in range(2)]
    klen = [i32([12000, 5000]), i32([11, 9000])]
    want = [att(*s, k_len=n).clone() for s, n in zip(sets, klen)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s, n in zip(sets, klen):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(att(*s, k_len=n))
        graphs.append(g)
    for _ in range(20):
        eager = []
        for st, g, s, n in zip(streams, graphs, sets, klen):
            with torch.cuda.stream(st):
                g.replay()
                eager.append(att(*s, k_len=n))
        torch.cuda.synchronize()
        for o, e, w in zip(outs, eager, want):
            assert torch.equal(o, w) and torch.equal(e, w)
    # A replay follows the lengths on the device.
    klen[0].copy_(i32([100, 12000]))
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], att(*sets[0], k_len=klen[0]))
    att.check()


@pytest.mark.parametrize("Sq,Sk", [(1, 300), (2, 9000), (700, 700)])
def test_a_wait_that_runs_out_is_reported(Sq, Sk):
    """The next run after yb_attn_debug_withhold loads nothing: its waits give up after 1 ms, the handle reports it
    once, and later runs are as before."""
    import yb_ops
    import yolo_b200 as yb

    q, k, v, _ = tensors(4, Sq, Sk, 16, 8, 64, "bf16")
    att = yb_ops.Attention(16, 8, 64, torch.bfloat16, causal=True)
    want = att(q, k, v)
    att.check()
    yb.check(yb.lib().yb_attn_debug_withhold(att._h), "yb_attn_debug_withhold")
    att(q, k, v)
    with pytest.raises(yb.YBError):
        att.check()
    att.check()
    assert torch.equal(att(q, k, v), want)
    att.check()


def test_refusals():
    import yb_ops
    import yolo_b200 as yb

    q, k, v, out = tensors(2, 3, 9, 4, 2, 64, "bf16")
    att = yb_ops.Attention(4, 2, 64, torch.bfloat16)
    n = i32([1, 1])
    for bad in (lambda: att(q.cpu(), k, v), lambda: att(q.half(), k, v), lambda: att(q[..., :32], k, v),
                lambda: att(q, k[:1], v), lambda: att(q, k, v[:, :5]), lambda: att(q, k, v, out=out[:, :2]),
                lambda: att(q, k, v, q_len=n[:1]), lambda: att(q, k, v, k_len=n.long()),
                lambda: att(q, k, v, slopes=n), lambda: att(q[0], k, v),
                lambda: att(q, k, v, out=out[:1].expand(2, -1, -1, -1)),
                lambda: att(q, k, v, key_range=torch.zeros(2, 9, 2, dtype=torch.int32, device="cuda")),
                lambda: yb_ops.Attention(4, 2, 64, torch.float32), lambda: yb_ops.Attention(4, 3, 64, torch.float16),
                lambda: yb_ops.Attention(4, 2, 60, torch.float16), lambda: yb_ops.Attention(4, 2, 256, torch.float16),
                lambda: yb_ops.Attention(4, 2, 64, torch.float16, device="cpu")):
        with pytest.raises(ValueError):
            bad()
    odd = torch.zeros(2, 3, 4, 68, device="cuda").bfloat16()[..., :64]
    for bad in (lambda: att(odd, k, v), lambda: att(q, k, v, prefix=n), lambda: att(q, k, v, out=q),
                lambda: att(q, k[:, :1].expand(-1, 9, -1, -1), v),
                lambda: yb_ops.Attention(4, 2, 64, torch.bfloat16, cap=-1.0)(q, k, v),
                lambda: yb_ops.Attention(4, 2, 64, torch.bfloat16, scale=0.0)(q, k, v)):
        with pytest.raises(yb.YBError):
            bad()
    assert att(q[:0], k[:0], v[:0]).shape == (0, 3, 4, 64)
    assert att(q[:, :0], k, v).shape == (2, 0, 4, 64)


def test_decode_step_of_the_operators_together():
    """Prompt, then token after token, captured once and replayed: norm and rotation into the cache, attention over
    it, a projection, sampling.  Each step's hidden row equals attention over the whole text at once."""
    import yb_ops

    torch.manual_seed(0)
    B, P, N, Hq, Hkv, D, V = 3, 37, 6, 8, 2, 64, 5000
    att = yb_ops.Attention(Hq, Hkv, D, torch.bfloat16, causal=True, cap=50.0)
    inv = 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D)
    qw, kw = 1 + 0.2 * torch.randn(D, device="cuda"), 1 + 0.2 * torch.randn(D, device="cuda")
    table = torch.randn(V, (Hq + 2 * Hkv) * D, device="cuda").bfloat16()
    head = (torch.randn(Hq * D, V, device="cuda") * 0.3).bfloat16()
    plen = i32([P, 20, 1])
    kc = torch.full((B, P + N, Hkv, D), float("nan"), dtype=torch.bfloat16, device="cuda")
    vc = kc.clone()

    def split(x):
        x = x.unflatten(-1, (Hq + 2 * Hkv, D))
        return x[..., :Hq, :], x[..., Hq: Hq + Hkv, :], x[..., Hq + Hkv:, :]

    tokens = torch.randint(0, V, (B, P), device="cuda")
    q, k, v = split(table[tokens])
    qr, _ = yb_ops.qk_norm_rope(q, k, qw, kw, inv, k_out=kc, v=v, v_out=vc, start=i32([0] * B), length=plen)
    o = att(qr, kc, vc, q_len=plen, k_len=plen)
    first = o[torch.arange(B), (plen - 1).long()]
    u = torch.rand(N + 1, B, device="cuda")
    temp = torch.full((B,), 0.9, device="cuda")
    top_p = torch.full((B,), 0.9, device="cuda")
    tok, _ = yb_ops.sample(first.flatten(1) @ head, u[0], temperature=temp, top_p=top_p)
    state = {"tok": tok.clone(), "start": plen.clone(), "len": plen + 1, "u": u[0].clone()}

    def step():
        q, k, v = split(table[state["tok"].long()][:, None])
        qr, _ = yb_ops.qk_norm_rope(q, k, qw, kw, inv, k_out=kc, v=v, v_out=vc, start=state["start"])
        o = att(qr, kc, vc, k_len=state["len"])
        logits = o.flatten(1) @ head
        t, lp = yb_ops.sample(logits, state["u"], temperature=temp, top_p=top_p)
        return o, logits, t, lp

    step()  # loads what a first call loads; writes the rows that the first replay writes again
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o, logits, t, lp = step()
    text = [tokens[b, : int(plen[b])].tolist() + [int(tok[b])] for b in range(B)]
    for n in range(N):
        state["u"].copy_(u[n + 1])
        g.replay()
        torch.cuda.synchronize()
        # The whole text at once.
        for b in range(B):
            ids = torch.tensor(text[b], device="cuda")[None]
            qa, ka, va = split(table[ids])
            qa, ka = yb_ops.qk_norm_rope(qa, ka, qw, kw, inv)
            assert torch.equal(ka[0], kc[b, : ids.shape[1]])
            ref = attention_ref(qa[:, -1:], ka, va.contiguous(), att.scale, 50.0, True)
            check_attention(o[b: b + 1], o[b: b + 1], ref)
        again, _ = yb_ops.sample(logits, state["u"], temperature=temp, top_p=top_p)
        assert torch.equal(again, t) and bool((t >= 0).all()) and bool((lp <= 0).all())
        for b in range(B):
            text[b].append(int(t[b]))
        state["tok"].copy_(t)
        state["start"].add_(1)
        state["len"].add_(1)
    att.check()
