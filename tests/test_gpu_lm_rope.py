"""yb_qk_norm_rope against its 64-bit form (bounds in lm_util.rotate_ref)."""
import pytest
import torch

from lm_util import rotate_ref

pytestmark = pytest.mark.gpu

T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def freqs(R, base=10000.0):
    return base ** (-torch.arange(0, R, 2, dtype=torch.float64, device="cuda") / max(R, 1))


def close(got, want, bound):
    over = (got.double() - want).abs() - bound
    assert over.numel() == 0 or float(over.max()) <= 0, float(over.max())


def run_case(B, S, rows, Hq, Hkv, D, R, dt, interleaved=False, ragged=False, start=None, positions=None, packed=True,
             with_v=True, weights=True, weight_add=0.0, eps=1e-6, seed=0, offset=0):
    import yb_ops

    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = T[dt]
    width = (Hq + 2 * Hkv) * D + offset
    qkv = (torch.randn(B, S, width, generator=g, device="cuda") * 2).to(dtype)[..., offset:]
    q = qkv[..., : Hq * D].unflatten(-1, (Hq, D))
    k = qkv[..., Hq * D: (Hq + Hkv) * D].unflatten(-1, (Hkv, D))
    v = qkv[..., (Hq + Hkv) * D:].unflatten(-1, (Hkv, D))
    if not packed:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    qw = 1 + 0.3 * torch.randn(D, generator=g, device="cuda") if weights else None
    kw = 1 + 0.3 * torch.randn(D, generator=g, device="cuda") if weights else None
    inv = freqs(R)
    kc = torch.randn(B, rows, Hkv, D, generator=g, device="cuda").to(dtype)
    vc = torch.randn(B, rows, Hkv, D, generator=g, device="cuda").to(dtype)
    qo = torch.randn(B, S, Hq, D, generator=g, device="cuda").to(dtype)
    length = torch.tensor([(S * (b + 2)) // (B + 1) if b else S for b in range(B)], dtype=torch.int32).cuda() if ragged else None
    st = torch.tensor(start, dtype=torch.int32).cuda() if start is not None else None
    pos = torch.tensor(positions, dtype=torch.int32).cuda() if positions is not None else None
    want_q, want_k, want_v = qo.double(), kc.double(), vc.double()
    bq, bk = torch.zeros_like(want_q), torch.zeros_like(want_k)
    for b in range(B):
        n = int(length[b]) if ragged else S
        a = start[b] if start is not None else 0
        p = pos[b, :n] if pos is not None else a + torch.arange(n, device="cuda")
        want_q[b, :n], bq[b, :n] = rotate_ref(q[b, :n], qw, p, inv, eps, weight_add, interleaved)
        yk, e = rotate_ref(k[b, :n], kw, p, inv, eps, weight_add, interleaved)
        for t in range(n):
            if 0 <= a + t < rows:
                want_k[b, a + t], bk[b, a + t] = yk[t], e[t]
                if with_v:
                    want_v[b, a + t] = v[b, t].double()
    yb_ops.qk_norm_rope(q, k, qw, kw, inv, q_out=qo, k_out=kc, v=v if with_v else None, v_out=vc if with_v else None,
                        start=st, length=length, positions=pos, eps=eps, weight_add=weight_add,
                        interleaved=interleaved)
    torch.cuda.synchronize()
    close(qo, want_q, bq)
    close(kc, want_k, bk)
    assert torch.equal(vc.double(), want_v)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,R", [(2, 2), (6, 4), (64, 64), (80, 80), (96, 64), (128, 128), (128, 32), (200, 0),
                                 (256, 256), (258 - 4, 254), (250, 100)])
def test_head_sizes(D, R, interleaved, dt):
    run_case(2, 5, 9, 4, 2, D, R, dt, interleaved, start=[3, 0], seed=D)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_batches(dt):
    run_case(1, 1, 1, 1, 1, 64, 64, dt)
    run_case(16, 1, 33, 32, 8, 128, 128, dt, start=[2 * b for b in range(16)])
    run_case(3, 1700, 1700, 5, 1, 64, 64, dt, ragged=True)
    run_case(2, 31, 40, 7, 7, 96, 96, dt, ragged=True, packed=False, start=[9, 1])
    run_case(2, 12, 12, 3, 3, 64, 64, dt, with_v=False, weights=False)
    run_case(2, 12, 12, 3, 3, 64, 64, dt, weight_add=1.0, eps=0.01)


def test_far_positions():
    S = 6
    pos = [[0, 1, 1000003, 2 ** 31 - 1, -5, -(2 ** 31)], [7, 7, 123456789, 10 ** 6, 10 ** 9, 2]]
    run_case(2, S, S, 2, 2, 128, 128, "f32", positions=pos)
    run_case(2, S, S, 2, 2, 128, 64, "bf16", True, positions=pos)


def test_rows_outside_the_cache_are_not_written():
    run_case(3, 8, 10, 2, 2, 64, 64, "bf16", start=[-3, 6, 2 ** 31 - 4])


def test_unaligned_rows():
    for off in (1, 3):
        run_case(2, 4, 6, 3, 1, 64, 64, "bf16", start=[1, 2], offset=off)
        run_case(2, 4, 6, 3, 1, 64, 64, "f32", True, offset=off)


def test_in_place_and_other_layouts():
    import yb_ops

    B, S, Hq, Hkv, D = 2, 9, 4, 2, 64
    inv = freqs(D)
    q = torch.randn(B, S, Hq, D, device="cuda").bfloat16()
    k = torch.randn(B, S, Hkv, D, device="cuda").bfloat16()
    q0, k0 = yb_ops.qk_norm_rope(q, k, None, None, inv)
    # Heads before rows.
    kc = torch.zeros(B, Hkv, 20, D, device="cuda").bfloat16().permute(0, 2, 1, 3)
    q1, _ = yb_ops.qk_norm_rope(q.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3), k, None, None, inv, k_out=kc)
    assert torch.equal(q0, q1) and torch.equal(kc[:, :S], k0) and not bool(kc[:, S:].any())
    yb_ops.qk_norm_rope(q, k, None, None, inv, q_out=q, k_out=k)
    assert torch.equal(q, q0) and torch.equal(k, k0)


def test_offsets_past_32_bits():
    """A cache whose last rows lie more than 2^31 elements behind its first."""
    import yb_ops

    B, S, H, D, rows, stride = 1, 3, 2, 64, 40000, 65536
    big = torch.empty(rows * stride, dtype=torch.bfloat16, device="cuda")
    cache = big.view(rows, stride)[:, : H * D].view(1, rows, H, D)
    assert (rows - 1) * cache.stride(1) > 2 ** 31
    k = torch.randn(B, S, H, D, device="cuda").bfloat16()
    start = torch.tensor([rows - S], dtype=torch.int32, device="cuda")
    _, k0 = yb_ops.qk_norm_rope(k, k, None, None, freqs(D), positions=torch.arange(rows - S, rows, device="cuda", dtype=torch.int32)[None])
    yb_ops.qk_norm_rope(k, k, None, None, freqs(D), k_out=cache, start=start)
    assert torch.equal(cache[:, rows - S:], k0)


def test_binding_refusals():
    import yb_ops
    import yolo_b200 as yb

    q = torch.zeros(2, 3, 4, 64, device="cuda").bfloat16()
    k = torch.zeros(2, 3, 2, 64, device="cuda").bfloat16()
    inv, w = freqs(64), torch.ones(64, device="cuda")
    i32 = torch.zeros(2, dtype=torch.int32, device="cuda")
    f = yb_ops.qk_norm_rope
    for bad in (lambda: f(q.cpu(), k, w, w, inv), lambda: f(q, k.half(), w, w, inv), lambda: f(q, k[:1], w, w, inv),
                lambda: f(q, k, w.half(), w, inv), lambda: f(q, k, w, w, inv.float()), lambda: f(q, k, w, w, inv, v=k),
                lambda: f(q, k, w, w, inv, start=i32), lambda: f(q, k, w, w, inv, length=i32.long()),
                lambda: f(q.transpose(2, 3), k, w, w, inv), lambda: f(q.double(), k.double(), w, w, inv),
                lambda: f(q, k, w, w, inv, k_out=k[:, :1].expand(-1, 3, -1, -1)),
                lambda: f(q, k, w, w, inv, positions=i32)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(yb.YBError):
        f(q, k, w, w, freqs(66))
    with pytest.raises(yb.YBError):
        f(q, k, w, w, inv, k_out=k, start=i32)
