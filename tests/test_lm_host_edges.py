"""Refusals of the text-decoder operators that a plain check of each argument misses (on the CPU: all are decided before
any device work)."""
import pytest

from test_lm_host import attn_args


@pytest.mark.parametrize("kw", [dict(B=(1 << 31) - 1, Sq=1 << 30, Hq=8, Hkv=8), dict(B=1 << 30, Sq=1 << 30, Hq=16, Hkv=1),
                                dict(B=1 << 30, Sq=1 << 30, Hq=1 << 30, Hkv=1), dict(B=1 << 16, Sq=1 << 15, Hq=1, Hkv=1)],
                         ids=str)
def test_attention_sizes_whose_product_passes_64_bits(kw):
    import yolo_b200 as yb

    assert yb.lib().yb_attn_run(None, attn_args(**kw), None, 0, None) == yb.ERROR_INVALID_DIMS
    assert "attn" in yb.last_error()
