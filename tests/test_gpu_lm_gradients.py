"""The operators of yb_ops have no gradients: tensors that ask for one are refused, not taken silently."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def leaf(*shape, dtype=torch.bfloat16):
    return torch.randn(*shape, device="cuda").to(dtype).requires_grad_()


def test_tensors_that_require_gradients_are_refused():
    import yb_ops

    q, k = leaf(2, 3, 4, 64), leaf(2, 3, 2, 64)
    w = leaf(64, dtype=torch.float32)
    inv = torch.ones(32, dtype=torch.float64, device="cuda")
    x, u = leaf(2, 100, dtype=torch.float32), torch.rand(2, device="cuda")
    att = yb_ops.Attention(4, 2, 64, torch.bfloat16)
    d = torch.Tensor.detach
    calls = [lambda: att(q, d(k), d(k)), lambda: att(d(q), k, d(k)), lambda: att(d(q), d(k), k * 2),
             lambda: att(d(q), d(k), d(k), slopes=leaf(4, dtype=torch.float32)),
             lambda: yb_ops.qk_norm_rope(q, d(k), None, None, inv), lambda: yb_ops.qk_norm_rope(d(q), k, None, None, inv),
             lambda: yb_ops.qk_norm_rope(d(q), d(k), w, None, inv), lambda: yb_ops.sample(x, u)]
    for call in calls:
        with pytest.raises(ValueError, match="no gradients"):
            call()
        with torch.no_grad():
            call()
    att.check()
