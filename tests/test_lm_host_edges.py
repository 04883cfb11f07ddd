"""Refusals of the text-decoder operators that a plain check of each argument misses (on the CPU: all are decided before
any device work)."""
import pytest

from test_lm_host import attn_args, qk_args, sample_args


@pytest.mark.parametrize("kw", [dict(B=(1 << 31) - 1, Sq=1 << 30, Hq=8, Hkv=8), dict(B=1 << 30, Sq=1 << 30, Hq=16, Hkv=1),
                                dict(B=1 << 30, Sq=1 << 30, Hq=1 << 30, Hkv=1), dict(B=1 << 16, Sq=1 << 15, Hq=1, Hkv=1)],
                         ids=str)
def test_attention_sizes_whose_product_passes_64_bits(kw):
    import yolo_b200 as yb

    assert yb.lib().yb_attn_run(None, attn_args(**kw), None, 0, None) == yb.ERROR_INVALID_DIMS
    assert "attn" in yb.last_error()


@pytest.mark.parametrize("kw", [dict(q_len=4098), dict(k_len=4097), dict(slopes=4098), dict(prefix=4098, causal=1),
                                dict(key_range=4100)], ids=str)
def test_attention_pointers_off_their_boundary(kw):
    import yolo_b200 as yb

    assert yb.lib().yb_attn_run(None, attn_args(**kw), None, 0, None) == yb.ERROR_INVALID_DIMS
    assert "aligned" in yb.last_error()


@pytest.mark.parametrize("kw", [dict(q=4097), dict(k=8193), dict(q_out=16385), dict(k_out=20481), dict(v=24577, v_out=28672),
                                dict(v=24576, v_out=28673), dict(dtype=0, q=4098), dict(dtype=0, k_out=20482),
                                dict(q_weight=66), dict(k_weight=65), dict(inv_freq=68), dict(start=66), dict(length=65),
                                dict(positions=66)], ids=str)
def test_qk_norm_rope_pointers_off_their_boundary(kw):
    import yolo_b200 as yb

    assert yb.lib().yb_qk_norm_rope(qk_args(**kw), None) == yb.ERROR_INVALID_DIMS
    assert "aligned" in yb.last_error()


@pytest.mark.parametrize("kw", [dict(logits=4098), dict(logits=4097, dtype=2), dict(u=4098), dict(temperature=4097),
                                dict(top_k=4098), dict(top_p=4098), dict(min_p=4098), dict(token=4098),
                                dict(logprob=4097)], ids=str)
def test_sample_pointers_off_their_boundary(kw):
    import yolo_b200 as yb

    assert yb.lib().yb_sample(sample_args(**kw), None) == yb.ERROR_INVALID_DIMS
    assert "aligned" in yb.last_error()
