"""Linear attention, its gradients and its step on the GPU against 64-bit forms, at the sizes and layouts where they can go wrong."""
import numpy as np
import pytest
import torch

import linear_attention_oracle as orc

pytestmark = pytest.mark.gpu
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
ALL = list(TYPES)


@pytest.fixture(scope="module")
def ops():
    from csn_b200 import ops
    return ops


def make(shape, kind, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(TYPES[kind]).cuda()


def decays(H, kind="mixed"):
    if kind == "none":
        return torch.zeros(H, device="cuda")
    g = -torch.exp2(-torch.linspace(0.0, 9.0, H)) * 2.0  # e^-2 a step to 1 / 256
    if kind == "shut" and H > 1:
        g[1] = -torch.inf
    return g.cuda()


def fused(lead, H, Hk, Dk, Dv, kind, seed, scale=1.0):
    """q, k, v as slices of one projection's rows."""
    cuts = [H * Dk, Hk * Dk, Hk * Dv]
    a, b, c = make((*lead, sum(cuts)), kind, seed, scale).split(cuts, -1)
    return a.unflatten(-1, (H, Dk)), b.unflatten(-1, (Hk, Dk)), c.unflatten(-1, (Hk, Dv))


def bounds(name, size, n, kind, sizes):
    """What a result may be off before its last rounding (see the oracle): the step-by-step bound, and for 16-bit tensors what
    the tensor-core path rounds once more."""
    K, top = sizes
    b = orc.steps(n, K) * orc.U * size
    if kind == "float32":
        return b
    if name in ("s", "ds0"):
        return b + (2.0 ** -22 * n * top if kind == "float16" else 0.0)
    b = b + 1.01 * orc.HALF_STEP[TYPES[kind]] * size
    return b + (2.0 ** -24 * 256 * top if kind == "float16" else 0.0)


def check(ops, q, k, v, g, s0, cu, kind, grads=True, scale=None, do=None, ds=None, wants=None):
    H, Dk, Dv = q.shape[-2], q.shape[-1], v.shape[-1]
    if cu is None:
        B, T = q.shape[:2]
        borders = [(b * T, (b + 1) * T) for b in range(B)]
    else:
        n = cu.tolist()
        borders = list(zip(n[:-1], n[1:]))
    longest = max([b - a for a, b in borders] + [1])
    leaves = {n: t for n, t in (("q", q), ("k", k), ("v", v), ("s0", s0)) if t is not None}
    if grads:
        leaves = {n: t.detach().requires_grad_(True) for n, t in leaves.items()}
    o, s = ops.linear_attention(leaves["q"], leaves["k"], leaves["v"], g, s0=leaves.get("s0"), cu_seqlens=cu, scale=scale)
    assert o.dtype == q.dtype and o.shape == (*q.shape[:-1], Dv)
    assert s.dtype == torch.float32 and s.shape == (len(borders), H, Dk, Dv)
    flat = lambda t: None if t is None else t.detach().double().cpu().flatten(0, -3)  # noqa: E731
    zero = torch.zeros(len(borders), H, Dk, Dv, dtype=torch.float64)
    wide = lambda t: zero if t is None else t.detach().double().cpu()  # noqa: E731
    rows = torch.zeros(*q.shape[:-1], Dv) if do is None else do
    want = orc.attention(flat(q), flat(k), flat(v), g.cpu(), wide(s0), borders, Dk ** -0.5 if scale is None else scale,
                         flat(rows) if grads else None, wide(ds) if grads else None)
    got = {"o": o, "s": s}
    if grads:
        outs, given = zip(*[(a, b) for a, b in ((o, do), (s, ds)) if b is not None])
        names = wants or list(leaves)
        for n, t in zip(names, torch.autograd.grad(outs, [leaves[n] for n in names], given)):
            got["d" + n] = t
            assert t.dtype == leaves[n].dtype and t.shape == leaves[n].shape
    for n, t in got.items():
        value, size = want[n]
        top = float(size.max()) if size.numel() else 0.0
        state = n in ("s", "ds0")
        allowed = bounds(n, size, longest, kind, (max(Dk, Dv), top))
        share = orc.used(t.detach().double().cpu().reshape(value.shape), value, allowed, torch.float32 if state else TYPES[kind])
        assert share <= 1.0, f"{n}: {share:.2f} of the allowed error"


def dense(ops, kind, B, T, H, Hk, Dk, Dv, decay="mixed", grads=True, s0=True, scale=None):
    q, k, v = fused((B, T), H, Hk, Dk, Dv, kind, 1)
    states = lambda seed: make((B, H, Dk, Dv), "float32", seed, 3.0)  # noqa: E731
    check(ops, q, k, v, decays(H, decay), states(2) if s0 else None, None, kind, grads, scale, make((B, T, H, Dv), kind, 3), states(4))


@pytest.mark.parametrize("kind", ALL)
@pytest.mark.parametrize("B,T,H,Hk,Dk,Dv", [(1, 1, 1, 1, 1, 1), (2, 1, 2, 2, 64, 64), (1, 2, 3, 1, 16, 8), (2, 15, 2, 1, 40, 24),
                                            (1, 16, 1, 1, 128, 128), (2, 37, 4, 2, 64, 64), (1, 127, 2, 2, 64, 128),
                                            (1, 128, 2, 1, 128, 64), (2, 129, 3, 3, 72, 104), (1, 255, 2, 2, 32, 32),
                                            (1, 257, 1, 1, 120, 8), (3, 300, 2, 1, 33, 50), (1, 200, 2, 2, 7, 128)])
def test_dense(ops, kind, B, T, H, Hk, Dk, Dv):
    dense(ops, kind, B, T, H, Hk, Dk, Dv)


@pytest.mark.parametrize("kind", ALL)
@pytest.mark.parametrize("decay", ["none", "shut"])
def test_decays_of_one_and_zero(ops, kind, decay):
    dense(ops, kind, 2, 140, 2, 2, 64, 64, decay)
    dense(ops, kind, 1, 20, 3, 1, 24, 56, decay, s0=False)


@pytest.mark.parametrize("kind", ALL)
@pytest.mark.parametrize("T,Dk,Dv", [(1000, 64, 64), (1537, 32, 48), (700, 128, 128), (2048, 16, 16)])
def test_long(ops, kind, T, Dk, Dv):
    """Few heads and many steps: sequences are cut into segments."""
    dense(ops, kind, 1, T, 2, 1, Dk, Dv)


@pytest.mark.parametrize("kind", ALL)
@pytest.mark.parametrize("lengths,behind", [([5], 0), ([0, 3, 0, 0, 70, 1], 4), ([64, 64, 1, 127, 0], 0), ([0, 0], 6), ([1] * 40, 1),
                                            ([300, 2, 513], 70), ([128, 256, 129], 3)])
def test_packed(ops, kind, lengths, behind):
    cu = torch.tensor(np.cumsum([0] + lengths), dtype=torch.int32, device="cuda")
    L, S = sum(lengths) + behind, len(lengths)
    for H, Hk, Dk, Dv in ((2, 2, 64, 64), (4, 2, 40, 72)):
        q, k, v = fused((L,), H, Hk, Dk, Dv, kind, 1)
        s = lambda seed: make((S, H, Dk, Dv), "float32", seed)  # noqa: E731
        check(ops, q, k, v, decays(H), s(2), cu, kind, True, None, make((L, H, Dv), kind, 3), s(4))


@pytest.mark.parametrize("kind", ALL)
def test_rows_of_no_sequence(ops, kind):
    """What stands in them does not matter, and they come out as 0."""
    cu = torch.tensor([3, 9, 9, 150], dtype=torch.int32, device="cuda")
    L, H, D = 170, 2, 64
    q, k, v = fused((L,), H, 1, D, D, kind, 1)
    do, s0 = make((L, H, D), kind, 3), make((3, H, D, D), "float32", 2)
    clean = [t[3:150].clone().requires_grad_(True) for t in (q, k, v)]
    o1, s1 = ops.linear_attention(*clean, decays(H), s0=s0, cu_seqlens=cu - 3)
    want = torch.autograd.grad(o1, clean, do[3:150])
    for t in (q, k, v, do):
        t[:3], t[150:] = float("nan"), float("inf")
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    o, s = ops.linear_attention(*leaves, decays(H), s0=s0, cu_seqlens=cu)
    got = torch.autograd.grad(o, leaves, do)
    for a, b in zip((o, *got), (o1, *want)):
        assert (a[:3] == 0).all() and (a[150:] == 0).all() and torch.equal(a[3:150], b)
    assert torch.equal(s, s1) and torch.equal(s[1], s0[1])


@pytest.mark.parametrize("kind", ALL)
def test_empty(ops, kind):
    g = decays(2)
    s0 = make((3, 2, 8, 16), "float32", 1)
    q, k, v = (make((3, 0, 2, d), kind, 1).requires_grad_(True) for d in (8, 8, 16))
    o, s = ops.linear_attention(q, k, v, g, s0=s0.requires_grad_(True))
    assert o.shape == (3, 0, 2, 16) and torch.equal(s, s0)
    ds = make((3, 2, 8, 16), "float32", 2)
    assert torch.equal(torch.autograd.grad(s, s0, ds)[0], ds)
    z = torch.zeros(0, 5, 2, 8, device="cuda", dtype=TYPES[kind])
    o, s = ops.linear_attention(z, z, z, g)
    assert o.shape == (0, 5, 2, 8) and s.shape == (0, 2, 8, 8)


@pytest.mark.parametrize("kind", ALL)
def test_gradients_one_by_one_and_of_one_result(ops, kind):
    q, k, v = fused((2, 150), 4, 2, 64, 32, kind, 1)
    s0, do, ds = make((2, 4, 64, 32), "float32", 2), make((2, 150, 4, 32), kind, 3), make((2, 4, 64, 32), "float32", 4)
    for wants in (["q"], ["k"], ["v"], ["s0"], ["k", "s0"]):
        check(ops, q, k, v, decays(4), s0, None, kind, True, None, do, ds, wants)
    check(ops, q, k, v, decays(4), s0, None, kind, True, None, do, None)
    check(ops, q, k, v, decays(4), s0, None, kind, True, None, None, ds)
    check(ops, q, k, v, decays(4), None, None, kind, True, 0.3, do, ds)


@pytest.mark.parametrize("kind", ["bfloat16", "float32"])
def test_layouts(ops, kind):
    """Heads before steps, steps in another order, a broadcast head, unaligned rows: the same numbers."""
    B, T, H, D = 2, 140, 2, 64
    q, k, v = (make((B, T, H, D), kind, i) for i in (1, 2, 3))
    g = decays(H)
    want = ops.linear_attention(q, k, v, g)
    turned = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    for a, b in zip(ops.linear_attention(*turned, g), want):
        assert torch.equal(a, b)
    check(ops, *(t.flip(1) for t in (q, k, v)), g, None, None, kind, False)
    check(ops, q, k[:, :, :1].expand(B, T, H, D), v, g, None, None, kind, False)
    off = [torch.empty(B * T * H * D + 1, device="cuda", dtype=t.dtype)[1:].view(B, T, H, D).copy_(t) for t in (q, k, v)]
    check(ops, *off, g, make((B, H, D, D), "float32", 5), None, kind, True, None, make((B, T, H, D), kind, 4))
    wide = [torch.zeros(B, T, H, 2 * D, device="cuda", dtype=t.dtype)[..., ::2].copy_(t) for t in (q, k, v)]
    check(ops, *wide, g, None, None, kind, False)


def test_gradient_against_differences(ops):
    q, k, v = fused((1, 40), 2, 1, 12, 20, "float32", 1)
    s0, g = make((1, 2, 12, 20), "float32", 2), decays(2)
    do, ds = make((1, 40, 2, 20), "float32", 3), make((1, 2, 12, 20), "float32", 4)
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v, s0)]

    def value(ts):
        o, s = ops.linear_attention(*ts[:3], g, s0=ts[3])
        return (o.double() * do).sum() + (s.double() * ds).sum()

    grads = torch.autograd.grad(value(leaves), leaves)
    for i, t in enumerate(leaves):
        way = make(t.shape, "float32", 10 + i)
        # each input enters its sums once: the difference of two calls has no second-order term
        ends = [value([u.detach() + (e * way if j == i else 0.0) for j, u in enumerate(leaves)]) for e in (0.5, -0.5)]
        want, got = float(ends[0] - ends[1]), float((grads[i].double() * way).sum())
        # both sides are sums of some thousand float32 results, each off by a few hundred units of its size at most
        assert abs(want - got) <= 1e-4 * float(abs(ends[0]) + abs(ends[1]) + (grads[i] * way).abs().sum())


# ------------------------------------------------------------------------- step
@pytest.mark.parametrize("kind", ALL)
@pytest.mark.parametrize("B,H,Hk,Dk,Dv", [(1, 1, 1, 1, 1), (2, 4, 2, 64, 64), (3, 3, 1, 128, 128), (2, 2, 2, 33, 50), (5, 2, 2, 8, 128),
                                          (1, 4, 1, 128, 4), (2, 2, 1, 100, 7), (70, 16, 16, 32, 32)])
def test_step_is_a_sequence_of_one(ops, kind, B, H, Hk, Dk, Dv):
    g = decays(H, "shut")
    s = make((B, H, Dk, Dv), "float32", 2)
    for t in range(3):
        q, k, v = fused((B,), H, Hk, Dk, Dv, kind, 10 + t)
        want = orc.attention(*(u.double().cpu() for u in (q, k, v)), g.cpu(), s.double().cpu(), [(b, b + 1) for b in range(B)], Dk ** -0.5)
        before = s.data_ptr()
        o = ops.linear_attention_step(q, k, v, g, s)
        assert s.data_ptr() == before and o.dtype == q.dtype
        for got, (value, size), typ in ((o, want["o"], TYPES[kind]), (s, want["s"], torch.float32)):
            assert orc.used(got, value, orc.steps(1, Dk) * orc.U * size, typ) <= 1.0


def test_steps_are_the_sequence(ops):
    """A prompt, then single tokens going on from its state, as generation runs them."""
    B, T, H, D = 2, 150, 2, 64
    q, k, v = fused((B, T + 4), H, 1, D, D, "float32", 1)
    g = decays(H)
    want, last = ops.linear_attention(q, k, v, g)
    o, s = ops.linear_attention(q[:, :T], k[:, :T], v[:, :T], g)
    outs = [ops.linear_attention_step(q[:, t], k[:, t], v[:, t], g, s) for t in range(T, T + 4)]
    got = torch.cat([o, torch.stack(outs, 1)], 1)
    for a, b in ((got, want), (s, last)):
        assert (a - b).abs().max() <= orc.steps(T + 4, D) * orc.U * 10 * b.abs().max()
