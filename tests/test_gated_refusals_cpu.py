"""What the gated block's operators refuse before they look at a device."""
import pytest
import torch
from torch.autograd import forward_ad

from csn_b200 import ops

csn = torch.ops.csn


def t(*shape, d=torch.bfloat16):
    return torch.zeros(*shape, dtype=d)


def calls():
    """Each operator on the tensors of a dict: name -> (call, {argument: tensor})."""
    f, h, w, rng = t(2, 4, 8), t(2, 8, d=torch.float32), t(6, 8), torch.zeros(2, dtype=torch.int64)
    scan = {"f": f, "x": f.clone(), "h0": h, "gate": f.clone()}
    step = {"f": f[0].clone(), "x": f[0].clone(), "h": t(4, 8, d=torch.float32), "gate": f[0].clone()}
    ffn = {"x": f, "w_gate": w, "w_up": w.clone()}
    drop = {"x": f, "residual": f.clone()}
    return {
        "gated_scan": (lambda f, x, h0, gate: ops.gated_scan(f, x, h0=h0, gate=gate), scan),
        "gated_step": (lambda f, x, h, gate: ops.gated_step(f, x, h, gate=gate), step),
        "silu_gated_linear": (lambda x, w_gate, w_up: ops.silu_gated_linear(x, w_gate, w_up), ffn),
        "dropout_add": (lambda x, residual: ops.dropout_add(x, residual, 0.1, rng), drop),
        "csn::gated_scan_fwd": (lambda f, x, h0, gate: csn.gated_scan_fwd(f, x, h0, gate, None), scan),
        "csn::gated_step": (lambda f, x, h, gate: csn.gated_step(f, x, h, gate), step),
        "csn::silu_gated_linear_fwd": (lambda x, w_gate, w_up: csn.silu_gated_linear_fwd(x, w_gate, w_up), ffn),
        "csn::dropout_add": (lambda x, residual: csn.dropout_add(x, residual, 6554, rng), drop),
    }


@pytest.mark.parametrize("name,argument", [(n, a) for n, (_, args) in calls().items() for a in args])
def test_forward_mode_is_refused(name, argument):
    """An input that carries a tangent is refused: the result would have none, without a word."""
    call, args = calls()[name]
    with forward_ad.dual_level():
        args = {**args, argument: forward_ad.make_dual(args[argument], torch.ones_like(args[argument]))}
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(**args)
