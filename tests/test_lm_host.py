"""What the text-decoder operators (include/yb_lm.h) refuse, on the CPU: every
refusal is decided on the host before any device work, so the calls here pass
pointers that nothing reads."""
import ctypes as C
import struct

import pytest

ATTN = ["q", "k", "v", "o", "q_len", "k_len", "prefix", "key_range", "slopes"]
GOOD_ATTN = dict(q=4096, k=8192, v=12288, o=16384, q_len=0, k_len=0, prefix=0, key_range=0, slopes=0,
                 q_stride=(1024, 512, 64), k_stride=(1024, 128, 64), v_stride=(1024, 128, 64),
                 o_stride=(1024, 512, 64), dtype=2, B=2, Sq=2, Sk=8, Hq=8, Hkv=2, D=64, causal=0, scale=0.125, cap=0.0)


def attn_args(**kw):
    a = dict(GOOD_ATTN)
    a.update(kw)
    return struct.pack("@9P12q8i2f", *[a[n] for n in ATTN], *a["q_stride"], *a["k_stride"], *a["v_stride"],
                       *a["o_stride"], a["dtype"], a["B"], a["Sq"], a["Sk"], a["Hq"], a["Hkv"], a["D"], a["causal"],
                       a["scale"], a["cap"])


BAD_ATTN = [
    dict(B=-1), dict(Sq=-1), dict(Sk=-1), dict(Hq=0), dict(Hkv=0), dict(Hkv=3), dict(D=0), dict(D=4), dict(D=60),
    dict(D=136), dict(dtype=0), dict(dtype=3), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
    dict(scale=float("inf")), dict(scale=3e38), dict(cap=1e-44), dict(cap=3e38), dict(scale=1e-30, cap=1e20),
    dict(cap=-1.0), dict(cap=float("nan")), dict(causal=2), dict(prefix=64),
    dict(o=4096), dict(o=8192), dict(q=4104), dict(o=16386), dict(q_stride=(1024, 516, 64)),
    dict(q_stride=(1024, 0, 64)), dict(k_stride=(1024, 128, 0)), dict(k_stride=(1024, -128, 64)),
    dict(o_stride=(0, 512, 64)), dict(v_stride=(1028, 128, 64)), dict(key_range=4100), dict(Sk=(1 << 30) + 1),
    dict(B=1 << 20, Sq=1 << 20),
]


@pytest.mark.parametrize("kw", BAD_ATTN, ids=str)
def test_attention_refusals(kw):
    import yolo_b200 as yb

    L = yb.lib()
    assert L.yb_attn_run(None, attn_args(**kw), None, 0, None) == yb.ERROR_INVALID_DIMS
    assert "attn" in yb.last_error()


@pytest.mark.parametrize("name", ["q", "k", "v", "o"])
def test_attention_null_operands(name):
    import yolo_b200 as yb

    assert yb.lib().yb_attn_run(None, attn_args(**{name: 0}), None, 0, None) == yb.ERROR_NULL_POINTER


def test_attention_needs_a_handle():
    import yolo_b200 as yb

    L = yb.lib()
    n = C.c_size_t(7)
    for kw in (dict(), dict(B=0), dict(Sq=0), dict(k_stride=(0, 128, 64)), dict(Hkv=1, k_stride=(1024, 128, 3))):
        assert L.yb_attn_run(None, attn_args(**kw), None, 0, None) == yb.ERROR_NULL_POINTER
    assert L.yb_attn_run(None, None, None, 0, None) == yb.ERROR_NULL_POINTER
    assert L.yb_attn_workspace(None, attn_args(), C.byref(n)) == yb.ERROR_NULL_POINTER
    assert L.yb_attn_workspace(None, attn_args(D=12), C.byref(n)) == yb.ERROR_INVALID_DIMS and n.value == 0
    assert L.yb_attn_check(None) == yb.ERROR_NULL_POINTER
    assert L.yb_attn_destroy(None) == yb.ERROR_NULL_POINTER
    assert L.yb_attn_debug_withhold(None) == yb.ERROR_NULL_POINTER
    assert L.yb_attn_create(0, None) == yb.ERROR_NULL_POINTER


QK = ["q", "k", "v", "q_out", "k_out", "v_out", "q_weight", "k_weight", "inv_freq", "start", "length", "positions"]
GOOD_QK = dict(q=4096, k=8192, v=0, q_out=16384, k_out=20480, v_out=0, q_weight=64, k_weight=64, inv_freq=64, start=0,
               length=0, positions=0, strides=[(1024, 512, 64)] * 6, dtype=2, B=2, S=2, rows=8, Hq=8, Hkv=2, D=64,
               R=64, interleaved=0, eps=1e-6, add=0.0)


def qk_args(**kw):
    a = dict(GOOD_QK)
    a.update(kw)
    return struct.pack("@12P18q9i2f0q", *[a[n] for n in QK], *[x for s in a["strides"] for x in s], a["dtype"], a["B"],
                       a["S"], a["rows"], a["Hq"], a["Hkv"], a["D"], a["R"], a["interleaved"], a["eps"], a["add"])


BAD_QK = [
    dict(B=-1), dict(S=-1), dict(Hq=-1), dict(Hkv=-1), dict(rows=-1), dict(D=0), dict(D=63), dict(D=258), dict(R=-2),
    dict(R=66), dict(R=31), dict(dtype=-1), dict(dtype=3), dict(interleaved=2), dict(eps=-1.0),
    dict(eps=float("nan")), dict(add=float("inf")), dict(strides=[(1024, 512, -64)] * 6), dict(Hq=65537),
    dict(B=1 << 16, S=1 << 16), dict(k_out=8192, start=64),
    dict(q_out=4096, strides=[(1024, 512, 64)] * 3 + [(2048, 1024, 64)] * 3),
    dict(v=24576, v_out=24576, start=64),
]


@pytest.mark.parametrize("kw", BAD_QK, ids=str)
def test_qk_norm_rope_refusals(kw):
    import yolo_b200 as yb

    assert yb.lib().yb_qk_norm_rope(qk_args(**kw), None) == yb.ERROR_INVALID_DIMS
    assert "qk_norm_rope" in yb.last_error()


@pytest.mark.parametrize("kw", [dict(q=0), dict(k=0), dict(q_out=0), dict(k_out=0), dict(inv_freq=0), dict(v=64),
                                dict(v_out=64)], ids=str)
def test_qk_norm_rope_null(kw):
    import yolo_b200 as yb

    assert yb.lib().yb_qk_norm_rope(qk_args(**kw), None) == yb.ERROR_NULL_POINTER
    assert yb.lib().yb_qk_norm_rope(None, None) == yb.ERROR_NULL_POINTER


def test_qk_norm_rope_nothing_to_do():
    import yolo_b200 as yb

    for kw in (dict(B=0), dict(S=0), dict(Hq=0, Hkv=0)):
        assert yb.lib().yb_qk_norm_rope(qk_args(q=0, k=0, **kw), None) == yb.SUCCESS


GOOD_SAMPLE = dict(logits=4096, u=4096, temperature=0, top_k=0, top_p=0, min_p=0, token=4096, logprob=0, stride=100,
                   dtype=0, B=2, V=100)


def sample_args(**kw):
    a = dict(GOOD_SAMPLE)
    a.update(kw)
    return struct.pack("@8Pq3i0q", a["logits"], a["u"], a["temperature"], a["top_k"], a["top_p"], a["min_p"],
                       a["token"], a["logprob"], a["stride"], a["dtype"], a["B"], a["V"])


@pytest.mark.parametrize("kw", [dict(B=-1), dict(V=0), dict(V=262145), dict(stride=-1), dict(dtype=3), dict(dtype=-1),
                                dict(B=(1 << 27) + 1)], ids=str)
def test_sample_refusals(kw):
    import yolo_b200 as yb

    assert yb.lib().yb_sample(sample_args(**kw), None) == yb.ERROR_INVALID_DIMS
    assert "sample" in yb.last_error()


def test_sample_null_and_empty():
    import yolo_b200 as yb

    L = yb.lib()
    for name in ("logits", "u", "token"):
        assert L.yb_sample(sample_args(**{name: 0}), None) == yb.ERROR_NULL_POINTER
    assert L.yb_sample(None, None) == yb.ERROR_NULL_POINTER
    assert L.yb_sample(sample_args(B=0, logits=0, u=0, token=0), None) == yb.SUCCESS


def test_argument_structures_match_the_binding():
    import yb_ops

    assert yb_ops._ATTN.size == len(attn_args()) and yb_ops._QK.size == len(qk_args())
    assert yb_ops._SAMPLE.size == len(sample_args())
