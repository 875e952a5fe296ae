"""A second backward pass through an operator that is differentiable once is refused in that operator's name."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def leaf(*shape):
    return torch.randn(*shape, device="cuda", dtype=torch.bfloat16).requires_grad_(True)


def calls():
    from csn_b200 import ops
    w = leaf(64)
    yield "gated_scan", lambda x: ops.gated_scan(x, x.detach())[0], leaf(2, 8, 64)
    yield "silu_gated_linear", lambda x: ops.silu_gated_linear(x, leaf(32, 64), leaf(32, 64)), leaf(8, 64)
    yield "dropout_add", lambda x: ops.dropout_add(x, None, 0.5, torch.randint(1 << 62, (2,), device="cuda")), leaf(8, 64)
    yield "linear_attention", lambda x: ops.linear_attention(x, x.detach(), x.detach(), torch.zeros(2, device="cuda"))[0], leaf(1, 8, 2, 16)
    yield "layer_norm", lambda x: ops.layer_norm(x, w, w.detach()), leaf(8, 64)


def test_the_operator_is_named():
    for name, call, x in calls():
        (g,) = torch.autograd.grad(call(x).float().square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match=f"^{name} is differentiable once"):
            g.float().sum().backward()
