"""The gated recurrent block: its operators together as they are used, trained, packed, captured and
advanced token by token, against the block written out in 64 bits.

A float32 pass through the block sums products over at most 3 d + f + d numbers one after the other
(projections) between norms and gates of slope <= 2: with 2^-23 an addition this is far below 1e-4 of
the result's norm.  In bfloat16 every tensor between two operators is rounded (2^-9 on average, 2^-8
at most, eleven tensors deep): 5e-2."""
import math

import numpy as np
import pytest
import torch

import gated_oracle as orc

pytestmark = pytest.mark.gpu
BOUND = {torch.float32: 1e-4, torch.bfloat16: 5e-2}


def build(d, f, p, dtype, seed=0):
    from csn_b200.modules import GatedRecurrentBlock
    torch.manual_seed(seed)
    return GatedRecurrentBlock(d, d_inner=d, d_ffn=f, dropout=p).cuda().to(dtype)


def written_out(blk, x, h0, borders):
    """The block in float64 with torch's elementary operations and autograd: (out, states, parameters).
    Masks are drawn from where the generator stands."""
    P = {k: v.detach().double().requires_grad_(True) for k, v in blk.named_parameters()}
    norm = lambda v, n: ((v - v.mean(-1, keepdim=True)) / (v.var(-1, unbiased=False, keepdim=True) + 1e-5).sqrt()  # noqa: E731
                         * P[n + ".weight"] + P[n + ".bias"])

    def dropped(v, drop):
        if not drop.training or drop.p == 0:
            return v
        seed, offset = drop.numbers(v.device).tolist()
        cut = round(drop.p * 65536)
        keep = orc.philox_halves(v.numel(), seed, offset) >= cut
        return v * torch.tensor(keep, device=v.device).reshape(v.shape) * (65536 / (65536 - cut))

    rows = norm(x, "ln_1") @ P["mixer.in_proj.weight"].t() + P["mixer.in_proj.bias"]
    f, v, gate = rows.split(blk.mixer.d_inner, -1)
    hs, last = [], []
    for s, (b, e) in enumerate(borders):
        h = h0[s]
        for t in range(b, e):
            a = torch.sigmoid(f[t])
            h = a * h + (1 - a) * v[t]
            hs.append(h)
        last.append(h)
    y = torch.stack(hs) * gate * torch.sigmoid(gate)
    x = x + dropped(y @ P["mixer.out_proj.weight"].t() + P["mixer.out_proj.bias"], blk.drop_1)
    z = norm(x, "ln_2")
    g = z @ P["ffn.w_gate.weight"].t()
    u = g * torch.sigmoid(g) * (z @ P["ffn.w_up.weight"].t())
    return x + dropped(u @ P["ffn.w_down.weight"].t(), blk.drop_2), torch.stack(last), P


def far(got, want):
    return float((got.detach().double() - want.detach()).norm() / want.detach().norm())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("p", [0.0, 0.2])
@pytest.mark.parametrize("packed", [False, True])
def test_training_pass(dtype, p, packed):
    d, f = 32, 72
    blk = build(d, f, p, dtype)
    g = torch.Generator().manual_seed(3)
    if packed:
        borders, shape = [(0, 5), (5, 5), (5, 80), (80, 97)], (97, d)
        cu = torch.tensor([0, 5, 5, 80, 97], dtype=torch.int32, device="cuda")
    else:
        borders, shape, cu = [(0, 40), (40, 80)], (2, 40, d), None
    x = torch.randn(*shape, generator=g).to(dtype).cuda().requires_grad_(True)
    h0 = torch.randn(len(borders), d, generator=g).cuda().requires_grad_(True)
    dout, dh = torch.randn(*shape, generator=g).cuda(), torch.randn(len(borders), d, generator=g).cuda()
    state = torch.cuda.get_rng_state()
    out, h = blk(x, h0, cu)
    torch.cuda.set_rng_state(state)
    ((out.float() * dout).sum() + (h * dh).sum()).backward()
    x64, h64 = x.detach().double().reshape(-1, d).requires_grad_(True), h0.detach().double().requires_grad_(True)
    want, wh, P = written_out(blk, x64, h64, borders)
    ((want * dout.double().reshape(-1, d)).sum() + (wh * dh.double()).sum()).backward()
    assert far(out.reshape(-1, d), want.detach()) < BOUND[dtype] and far(h.detach(), wh.detach()) < BOUND[dtype]
    assert far(x.grad.reshape(-1, d), x64.grad) < BOUND[dtype] and far(h0.grad, h64.grad) < BOUND[dtype]
    for k, v in blk.named_parameters():
        assert v.grad is not None and v.grad.dtype == dtype
        assert far(v.grad, P[k].grad) < BOUND[dtype], k


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_token_by_token_is_the_whole_sequence(dtype):
    B, T, d = 3, 20, 32
    blk = build(d, 64, 0.3, dtype).eval()
    x = torch.randn(B, T, d, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    with torch.no_grad():
        whole, last = blk(x)
        h = blk.init_state(B)
        steps = torch.stack([blk.step(x[:, t], h) for t in range(T)], 1)
    assert far(steps, whole.double()) < BOUND[dtype] and far(h, last.double()) < BOUND[dtype]


def test_prompt_and_then_tokens():
    """The states that a prompt leaves are the ones that generation goes on from."""
    B, T, d = 2, 30, 32
    blk = build(d, 64, 0.0, torch.float32).eval()
    x = torch.randn(B, T, d, generator=torch.Generator().manual_seed(2)).cuda()
    with torch.no_grad():
        whole, last = blk(x)
        _, h = blk(x[:, :20])
        for t in range(20, T):
            out = blk.step(x[:, t], h)
    assert far(out, whole[:, -1].double()) < 1e-4 and far(h, last.double()) < 1e-4


def test_captured_training_step_draws_new_masks():
    from csn_b200 import graphs
    B, T, d = 2, 24, 32
    blk = build(d, 64, 0.25, torch.float32)
    x, y = (torch.randn(B, T, d, generator=torch.Generator().manual_seed(i)).cuda() for i in (4, 5))
    loss = lambda out: ((out[0] - y) ** 2).mean()  # noqa: E731
    step = graphs.TrainStepGraph(blk, None, [x], loss_fn=loss)
    state = torch.cuda.get_rng_state()
    outs, grads = [], []
    for _ in range(3):
        outs.append(step(x)[0].clone())
        grads.append([v.grad.clone() for v in blk.parameters()])
    assert not torch.equal(outs[0], outs[1]) and not torch.equal(outs[1], outs[2])
    del step
    torch.cuda.set_rng_state(state)
    for out, gr in zip(outs, grads):
        blk.zero_grad(set_to_none=True)
        o, _ = blk(x)
        ((o - y) ** 2).mean().backward()
        assert far(out, o.detach().double()) < 1e-5
        for a, v in zip(gr, blk.parameters()):
            assert far(a, v.grad.double()) < 1e-4


@pytest.mark.parametrize("reentrant", [False, True])
def test_checkpointed_pass_keeps_its_masks(reentrant):
    """A forward pass that is run again in the backward pass has the same masks: the same bits throughout."""
    from torch.utils.checkpoint import checkpoint
    blk = build(32, 72, 0.25, torch.bfloat16)
    x = torch.randn(2, 40, 32, generator=torch.Generator().manual_seed(8)).bfloat16().cuda().requires_grad_(True)
    leaves = [x, *blk.parameters()]
    state = torch.cuda.get_rng_state()
    got = []
    for run in (lambda: blk(x), lambda: checkpoint(blk, x, use_reentrant=reentrant)):
        torch.cuda.set_rng_state(state)
        for v in leaves:
            v.grad = None
        out, h = run()
        (out.float().square().sum() + h.sum()).backward()
        got.append([out.detach(), *(v.grad for v in leaves)])
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_copied_layers_draw_their_own_masks():
    import copy
    from csn_b200.modules import DropoutAdd
    a = DropoutAdd(0.5)
    x = torch.ones(4096, device="cuda")
    assert not torch.equal(a(x), copy.deepcopy(a)(x))


def test_generation_under_inference_mode():
    blk = build(32, 72, 0.0, torch.bfloat16).eval()
    x = torch.randn(3, 32, generator=torch.Generator().manual_seed(9)).bfloat16().cuda()
    outs = []
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            h = blk.init_state(3)
            outs.append((blk.step(x, h), h))
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])


def test_registered_operators_and_their_gradients():
    import csn_b200.ops as ops
    csn = torch.ops.csn
    g = torch.Generator().manual_seed(7)
    f, x, gate = (torch.randn(2, 80, 32, generator=g).cuda().requires_grad_(True) for _ in range(3))
    h0 = torch.randn(2, 32, generator=g).cuda().requires_grad_(True)
    w1, w2 = (torch.randn(48, 32, generator=g).bfloat16().cuda().requires_grad_(True) for _ in range(2))
    rng = torch.tensor([3, 9], device="cuda")

    def registered():
        y, h, _ = csn.gated_scan_fwd(f, x, h0, gate, None)
        z = csn.dropout_add(y, x, 6554, rng)
        return csn.silu_gated_linear_fwd(z.bfloat16(), w1, w2).float().sum() + h.sum()

    def direct():
        y, h = ops.gated_scan(f, x, h0=h0, gate=gate)
        z = ops.dropout_add(y, x, 6554 / 65536, rng)
        return ops.silu_gated_linear(z.bfloat16(), w1, w2).float().sum() + h.sum()

    leaves = (f, x, gate, h0, w1, w2)
    one, two = registered(), direct()
    assert torch.equal(one, two)
    for a, b in zip(torch.autograd.grad(one, leaves), torch.autograd.grad(two, leaves)):
        assert torch.equal(a, b)
    h = torch.zeros(2, 32, device="cuda")
    h2 = h.clone()
    with torch.no_grad():
        assert torch.equal(csn.gated_step(f[:, 0], x[:, 0], h, gate[:, 0]), ops.gated_step(f[:, 0], x[:, 0], h2, gate=gate[:, 0]))
    assert torch.equal(h, h2)


def test_empty_batches_and_single_tokens():
    blk = build(32, 64, 0.1, torch.bfloat16)
    for shape in ((0, 5, 32), (2, 0, 32), (1, 1, 32)):
        x = torch.zeros(*shape, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        out, h = blk(x)
        assert out.shape == x.shape and h.shape == (shape[0], 32)
        if math.prod(shape):
            out.sum().backward()
            assert np.isfinite(x.grad.float().cpu().numpy()).all()
