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


# ------------------------------------------------- the registered backward operators
F32 = torch.float32


def scan_args(packed):
    """(f, x, gate, cu, marks, dy, dh_last) that fit: 3 sequences of 70 steps, or 3 in 210 rows."""
    lead, cu = ((210,), torch.tensor([0, 70, 140, 210], dtype=torch.int32)) if packed else ((3, 70), None)
    marks = csn.gated_scan_fwd(t(*lead, 8).to("meta"), t(*lead, 8).to("meta"), None, None, None if cu is None else cu.to("meta"))[2]
    return {"f": t(*lead, 8), "x": t(*lead, 8), "gate": t(*lead, 8), "cu_seqlens": cu, "marks": t(marks.numel(), d=F32),
            "dy": t(*lead, 8), "dh_last": t(3, 8, d=F32)}


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("name,bad", [
    ("marks", lambda v: v[:-1].clone()), ("marks", lambda v: v.bfloat16()), ("marks", lambda v: v.double()),
    ("marks", lambda v: v.view(2, -1)), ("marks", lambda v: torch.zeros(2 * v.numel())[::2]), ("marks", lambda v: torch.zeros(v.numel() + 1)[1:]),
    ("dy", lambda v: v[:-1]), ("dy", lambda v: v[..., :-1]), ("dy", lambda v: v.float()), ("dy", lambda v: v.half()),
    ("dy", lambda v: v.view(1, *v.shape)), ("dy", lambda v: v[..., 0]),
    ("dh_last", lambda v: v[:-1]), ("dh_last", lambda v: v[:, :-1]), ("dh_last", lambda v: v.int()), ("dh_last", lambda v: v.view(-1)),
    ("f", lambda v: v.float()), ("f", lambda v: v[:-1]), ("x", lambda v: v[..., :-1]), ("gate", lambda v: v[:-1]),
    ("gate", lambda v: v.half()), ("f", lambda v: v.view(-1)),
])
def test_scan_backward_refuses(packed, name, bad):
    args = scan_args(packed)
    with pytest.raises(ValueError):
        csn.gated_scan_bwd(*{**args, name: bad(args[name])}.values())


@pytest.mark.parametrize("bad", [lambda c: c.long(), lambda c: c[:1], lambda c: c[:-1], lambda c: c.view(2, 2), lambda c: None])
def test_scan_backward_refuses_borders(bad):
    args = scan_args(True)
    with pytest.raises(ValueError):
        csn.gated_scan_bwd(*{**args, "cu_seqlens": bad(args["cu_seqlens"])}.values())


@pytest.mark.parametrize("name,bad", [
    ("dy", lambda v: v[:-1]), ("dy", lambda v: v[..., :-1]), ("dy", lambda v: v.float()), ("dy", lambda v: v.half()),
    ("dy", lambda v: v.view(-1, v.shape[-1])), ("dy", lambda v: v[0, 0, 0]), ("x", lambda v: v[..., :-1]), ("x", lambda v: v.half()),
    ("x", lambda v: v[:, :-1]), ("w_gate", lambda v: v[:-1]), ("w_up", lambda v: v[:, :-1]), ("w_up", lambda v: v.float()),
    ("w_gate", lambda v: v.view(-1)),
])
def test_feed_forward_backward_refuses(name, bad):
    args = {"x": t(2, 5, 8), "w_gate": t(6, 8), "w_up": t(6, 8), "dy": t(2, 5, 6)}
    with pytest.raises(ValueError):
        csn.silu_gated_linear_bwd(*{**args, name: bad(args[name])}.values())


@pytest.mark.parametrize("packed", [False, True])
def test_backward_operators_want_cuda_tensors(packed):
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        csn.gated_scan_bwd(*scan_args(packed).values())
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        csn.silu_gated_linear_bwd(t(2, 5, 8), t(6, 8), t(6, 8), t(2, 5, 6))


def test_forward_mode_is_refused_by_backward_operators():
    scan = {**scan_args(False), "cu_seqlens": None}
    ffn = {"x": t(2, 5, 8), "w_gate": t(6, 8), "w_up": t(6, 8), "dy": t(2, 5, 6)}
    for call, args in ((csn.gated_scan_bwd, scan), (csn.silu_gated_linear_bwd, ffn)):
        for k, v in args.items():
            if v is None:
                continue
            with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
                call(*{**args, k: forward_ad.make_dual(v, torch.ones_like(v))}.values())
