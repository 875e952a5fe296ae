"""What the gated block's operators promise and refuse on the GPU, beyond their numbers."""
import pytest
import torch
from torch.autograd import forward_ad

import test_gated_refusals_cpu as refusals

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from csn_b200 import ops
    return ops


def rand(shape, seed, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype).cuda()


# dropout_add, whose (seed, offset) are the CPU's in that list, stands in the next test
@pytest.mark.parametrize("name", [n for n in refusals.calls() if not n.endswith("dropout_add")])
def test_forward_mode_is_refused(name):
    """On tensors that the kernels take."""
    call, args = refusals.calls()[name]
    args = {k: v.cuda() for k, v in args.items()}
    with forward_ad.dual_level():
        for k, v in args.items():
            dual = forward_ad.make_dual(v, torch.ones_like(v))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(**{**args, k: dual})


def test_tangents_of_gradients_are_refused(ops):
    f, h = rand((2, 70, 8), 1), rand((2, 8), 2, torch.float32)
    w, rng = rand((6, 8), 3), torch.tensor([1, 2], device="cuda")
    outs = (lambda x: ops.gated_scan(x, x)[0], lambda x: ops.gated_scan(x, x, h0=h)[1],
            lambda x: ops.silu_gated_linear(x, w, w), lambda x: ops.dropout_add(x, None, 0.5, rng),
            lambda x: ops.dropout_add(f, x, 0.5, rng))
    for out in outs:
        x = f.detach().requires_grad_(True)
        y = out(x)
        with forward_ad.dual_level():
            dy = forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y))
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(y, x, dy)
    x = f.detach()
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: ops.dropout_add(dual, None, 0.5, rng), lambda: ops.dropout_add(x, dual, 0.5, rng)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


def test_registered_backward_operators(ops):
    """They are the backward passes that autograd runs, and refuse what does not fit."""
    csn = torch.ops.csn
    f, x, gate, dy = (rand((3, 70, 24), i) for i in range(4))
    h0, dh = rand((3, 24), 5, torch.float32), rand((3, 24), 6)
    leaves = [t.detach().requires_grad_(True) for t in (f, x, h0, gate)]
    y, h = ops.gated_scan(*leaves[:3], gate=leaves[3])
    want = torch.autograd.grad((y, h), leaves, (dy, dh.float()))
    marks = csn.gated_scan_fwd(f, x, h0, gate, None)[2]
    got = csn.gated_scan_bwd(f, x, gate, None, marks, dy, dh)  # a state's gradient of any floating type
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    a, wg, wu, dz = rand((2, 50, 24), 7), rand((40, 24), 8), rand((40, 24), 9), rand((2, 50, 40), 10)
    leaves = [t.detach().requires_grad_(True) for t in (a, wg, wu)]
    want = torch.autograd.grad(ops.silu_gated_linear(*leaves), leaves, dz)
    for p, q in zip(want, csn.silu_gated_linear_bwd(a, wg, wu, dz)):
        assert p.shape == q.shape and torch.equal(p, q)
    for bad in (lambda: csn.gated_scan_bwd(f, x, gate, None, marks[:-4].clone(), dy, dh), lambda: csn.gated_scan_bwd(f, x, gate, None, marks, dy[:2], dh),
                lambda: csn.gated_scan_bwd(f, x, gate, None, marks, dy.float(), dh), lambda: csn.silu_gated_linear_bwd(a, wg, wu, dz[:, :-1]),
                lambda: csn.silu_gated_linear_bwd(a, wg, wu, dz.half())):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: csn.gated_scan_bwd(f, x, gate, None, marks, dy, dh.cpu()), lambda: csn.gated_scan_bwd(f, x, gate, None, marks.cpu(), dy, dh),
                lambda: csn.silu_gated_linear_bwd(a, wg, wu, dz.cpu())):
        with pytest.raises(RuntimeError, match="CUDA tensors"):
            bad()
