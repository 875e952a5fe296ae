"""The gated recurrent block's operators on the GPU against 64-bit forms, at the sizes and layouts
where they can go wrong; tolerances are the oracle's rounding bounds."""
import numpy as np
import pytest
import torch

import gated_oracle as orc

pytestmark = pytest.mark.gpu
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


@pytest.fixture(scope="module")
def ops():
    from csn_b200 import ops
    return ops


def to64(t):
    return t.detach().double().cpu().numpy()


def make(shape, kind, seed, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale + shift).to(TYPES[kind]).cuda()


def check(got, want, kind, what):
    used = orc.within(to64(got), want[0], want[1], kind)
    assert used <= 1.0, f"{what}: {used:.2f} of the allowed error"


# ------------------------------------------------------------------------ the scan
def scan_case(ops, f, x, h0, gate, cu, kind, grads=True, dy=None, dh=None):
    dense = cu is None
    C = f.shape[-1]
    if dense:
        B, T = f.shape[:2]
        borders = [(b * T, (b + 1) * T) for b in range(B)]
    else:
        n = cu.tolist()
        borders = list(zip(n[:-1], n[1:]))
    leaves = {k: v for k, v in (("f", f), ("x", x), ("h0", h0), ("gate", gate)) if v is not None}
    if grads:
        leaves = {k: v.detach().requires_grad_(True) for k, v in leaves.items()}
    y, h = ops.gated_scan(leaves["f"], leaves["x"], h0=leaves.get("h0"), gate=leaves.get("gate"), cu_seqlens=cu)
    assert y.shape == f.shape and y.dtype == f.dtype and h.dtype == torch.float32
    flat = lambda t: None if t is None else to64(t).reshape(-1, C)  # noqa: E731
    S = len(borders)
    want = orc.gated_scan(flat(f), flat(x), flat(h0) if h0 is not None else np.zeros((S, C)), flat(gate), borders,
                          flat(dy) if grads else None, flat(dh) if grads else None)
    check(y.reshape(-1, C), want["y"], kind, "y")
    check(h, want["h"], "float32", "h")
    if not grads:
        return
    outs, given = zip(*[(o, d) for o, d in ((y, dy), (h, dh)) if d is not None])
    got = dict(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), given)))
    for name, key in (("f", "df"), ("x", "dx"), ("gate", "dgate"), ("h0", "dh0")):
        if name in got:
            assert got[name].dtype == leaves[name].dtype and got[name].shape == leaves[name].shape
            check(got[name].reshape(-1, C), want[key], "float32" if name == "h0" else kind, key)


def bias(C):
    return torch.linspace(0, 7, C).cuda()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("B,T,C,gated", [(1, 1, 1, True), (2, 1, 64, False), (3, 7, 33, True), (1, 8, 65, False),
                                         (2, 63, 66, True), (2, 64, 130, True), (1, 65, 64, False), (2, 129, 31, True),
                                         (1, 700, 64, True), (5, 200, 96, False)])
def test_scan_dense(ops, kind, B, T, C, gated):
    f = (make((B, T, C), kind, 1).float() + bias(C)).to(TYPES[kind])
    x, gate = make((B, T, C), kind, 2), make((B, T, C), kind, 3, scale=2.0) if gated else None
    h0, dy, dh = make((B, C), "float32", 4), make((B, T, C), kind, 5), make((B, C), "float32", 6)
    scan_case(ops, f, x, h0, gate, None, kind, dy=dy, dh=dh)


@pytest.mark.parametrize("kind", ["bfloat16", "float32"])
@pytest.mark.parametrize("T", [1, 2, 8, 9, 16, 17, 31, 32, 33])
def test_scan_of_many_short_sequences(ops, kind, T):
    """Several sequences to a CTA, and fewer of them than the last CTA has room for."""
    for B, C in ((13, 66), (1, 33), (64, 64)):
        f = (make((B, T, C), kind, 1).float() + bias(C)).to(TYPES[kind])
        scan_case(ops, f, make((B, T, C), kind, 2), make((B, C), "float32", 4), make((B, T, C), kind, 3), None, kind,
                  dy=make((B, T, C), kind, 5), dh=make((B, C), "float32", 6))


@pytest.mark.parametrize("B,T,C", [(1, 5000, 64), (1, 1027, 40), (2, 2048, 128), (1, 4097, 6)])
def test_scan_long(ops, B, T, C):
    for kind in ("bfloat16", "float32"):
        f = (make((B, T, C), kind, 1).float() + bias(C)).to(TYPES[kind])
        x, gate = make((B, T, C), kind, 2), make((B, T, C), kind, 3)
        h0, dy, dh = make((B, C), "float32", 4), make((B, T, C), kind, 5), make((B, C), "float32", 6)
        scan_case(ops, f, x, h0, gate, None, kind, dy=dy, dh=dh)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("lengths,behind", [([5], 0), ([0, 3, 0, 0, 70, 1], 4), ([64, 64, 1, 127, 0], 0),
                                            ([0, 0], 6), ([1] * 40, 1), ([300, 2, 513], 70)])
def test_scan_packed(ops, kind, lengths, behind):
    cu = torch.tensor(np.cumsum([0] + lengths), dtype=torch.int32, device="cuda")
    L, S = sum(lengths) + behind, len(lengths)
    for C in (64, 35):
        f = (make((L, C), kind, 1).float() + bias(C)).to(TYPES[kind])
        x, gate = make((L, C), kind, 2), make((L, C), kind, 3)
        scan_case(ops, f, x, make((S, C), "float32", 4), gate, cu, kind, dy=make((L, C), kind, 5),
                  dh=make((S, C), "float32", 6))


def test_scan_first_rows_of_no_sequence(ops):
    cu = torch.tensor([3, 9, 9, 80], dtype=torch.int32, device="cuda")
    L, C = 90, 32
    f, x, gate = (make((L, C), "bfloat16", i) for i in (1, 2, 3))
    # what stands in rows of no sequence does not matter
    for t in (f, x, gate):
        t[:3], t[80:] = float("nan"), float("inf")
    dy = make((L, C), "bfloat16", 5)
    fl, xl, gl = (t.detach().requires_grad_(True) for t in (f, x, gate))
    y, h = ops.gated_scan(fl, xl, gate=gl, cu_seqlens=cu)
    got = torch.autograd.grad(y, (fl, xl, gl), dy)
    for t in (y, *got):
        assert torch.equal(t[:3], torch.zeros_like(t[:3])) and torch.equal(t[80:], torch.zeros_like(t[80:]))
        assert torch.isfinite(t).all()
    inner = [t[3:80] for t in (f, x, gate, dy)]
    want = orc.gated_scan(*(to64(t) for t in inner[:2]), np.zeros((3, C)), to64(inner[2]), [(0, 6), (6, 6), (6, 77)],
                          to64(inner[3]))
    check(y[3:80], want["y"], "bfloat16", "y")
    check(got[0][3:80], want["df"], "bfloat16", "df")


@pytest.mark.parametrize("kind", ["bfloat16", "float32"])
def test_scan_strided_rows(ops, kind):
    B, T, C = 3, 150, 64
    rows = make((B, T + 2, 3 * C + 1), kind, 1)
    f, x, gate = (rows[:, 1:T + 1, i * C + o:(i + 1) * C + o] for i, o in ((0, 0), (1, 1), (2, 0)))
    dy = make((T, B, C), kind, 5).transpose(0, 1)
    scan_case(ops, f, x, make((B, C), "float32", 4), gate, None, kind, dy=dy, dh=make((B, C), "float32", 6))
    # one row of x for every step of a sequence, a gate in another order of axes, a broadcast gradient
    x1 = make((B, 1, C), kind, 7).expand(B, T, C)
    gate1 = make((B, C, T), kind, 8).transpose(1, 2)
    scan_case(ops, f, x1, None, gate1, None, kind, dy=make((1, 1, 1), kind, 9).expand(B, T, C))


def test_scan_gradient_of_broadcast_inputs(ops):
    B, T, C = 2, 70, 32
    f0 = make((1, 1, C), "float32", 1).requires_grad_(True)
    x0 = make((1, T, C), "float32", 2).requires_grad_(True)
    dy = make((B, T, C), "float32", 3)
    y, _ = ops.gated_scan(f0.expand(B, T, C), x0.expand(B, T, C))
    df, dx = torch.autograd.grad(y, (f0, x0), dy)
    full = [t.detach().expand(B, T, C).contiguous().requires_grad_(True) for t in (f0, x0)]
    wide = torch.autograd.grad(ops.gated_scan(*full)[0], full, dy)
    torch.testing.assert_close(df, wide[0].sum((0, 1), keepdim=True), rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(dx, wide[1].sum(0, keepdim=True), rtol=1e-5, atol=1e-6)


def test_scan_only_the_last_state_or_some_gradients(ops):
    B, T, C = 2, 90, 48
    f, x = make((B, T, C), "float32", 1), make((B, T, C), "float32", 2)
    scan_case(ops, f, x, None, None, None, "float32", dh=make((B, C), "float32", 3))
    fl = f.detach().requires_grad_(True)
    y, h = ops.gated_scan(fl, x)
    (df,) = torch.autograd.grad(y.sum() + h.sum(), fl)
    want = orc.gated_scan(to64(f).reshape(-1, C), to64(x).reshape(-1, C), np.zeros((B, C)), None,
                          [(0, T), (T, 2 * T)], np.ones((B * T, C)), np.ones((B, C)))
    check(df.reshape(-1, C), want["df"], "float32", "df")


def test_scan_of_no_steps(ops):
    h0 = make((3, 32), "float32", 1).requires_grad_(True)
    f = torch.empty(3, 0, 32, device="cuda")
    y, h = ops.gated_scan(f, f, h0=h0)
    assert y.shape == (3, 0, 32) and torch.equal(h, h0)
    (d,) = torch.autograd.grad(h, h0, torch.ones_like(h))
    assert torch.equal(d, torch.ones_like(d))
    y, h = ops.gated_scan(f[:0], f[:0])
    assert y.shape == (0, 0, 32) and h.shape == (0, 32)


def test_scan_saturated_gates(ops):
    """Forget logits at both ends: the state passes on unchanged, or is the input."""
    T, C = 100, 64
    x = make((1, T, C), "float32", 2)
    h0 = make((1, C), "float32", 3)
    for f, want in ((float("inf"), h0[:, None].expand(1, T, C)), (float("-inf"), x), (200.0, h0[:, None].expand(1, T, C)),
                    (-200.0, x)):
        y, h = ops.gated_scan(torch.full_like(x, f), x, h0=h0)
        assert torch.equal(y, want) and torch.equal(h, want[:, -1])


def test_scan_gradient_against_differences(ops):
    """Central differences of the 64-bit form: the formulas themselves."""
    T, C = 9, 4
    f, x, gate = (to64(make((T, C), "float32", i)) for i in (1, 2, 3))
    h0, dy, dh = to64(make((1, C), "float32", 4)), to64(make((T, C), "float32", 5)), to64(make((1, C), "float32", 6))

    def loss(f, x, h0, gate):
        o = orc.gated_scan(f, x, h0, gate, [(0, T)])
        return (o["y"][0] * dy).sum() + (o["h"][0] * dh).sum()

    want = orc.gated_scan(f, x, h0, gate, [(0, T)], dy, dh)
    args = [f, x, h0, gate]
    for k, name in enumerate(("df", "dx", "dh0", "dgate")):
        num = np.zeros_like(args[k])
        for i in np.ndindex(num.shape):
            for s in (1, -1):
                v = [a.copy() for a in args]
                v[k][i] += s * 1e-5
                num[i] += s * loss(*v) / 2e-5
        assert np.abs(num - want[name][0]).max() < 1e-8
    t = [torch.tensor(v, device="cuda", dtype=torch.float32) for v in (f, x, h0, gate, dy, dh)]
    scan_case(ops, t[0][None], t[1][None], t[2], t[3][None], None, "float32", dy=t[4][None], dh=t[5])


# ------------------------------------------------------------------------ the step
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("B,C,gated", [(1, 1, True), (3, 33, False), (8, 512, True), (5, 130, True), (257, 66, False)])
def test_step_is_the_scan(ops, kind, B, C, gated):
    T = 5
    rows = make((T, B, 3 * C), kind, 1)
    f, x, gate = rows[..., :C], rows[..., C:2 * C], rows[..., 2 * C:] if gated else None
    h0 = make((B, C), "float32", 4)
    h = h0.clone()
    ys = torch.stack([ops.gated_step(f[t], x[t], h, gate=None if gate is None else gate[t]) for t in range(T)])
    flat = lambda t: None if t is None else to64(t.transpose(0, 1)).reshape(-1, C)  # noqa: E731
    want = orc.gated_scan(flat(f), flat(x), to64(h0), flat(gate), [(b * T, (b + 1) * T) for b in range(B)])
    check(ys.transpose(0, 1).reshape(-1, C), want["y"], kind, "y")
    check(h, want["h"], "float32", "h")


# --------------------------------------------------------- gated feed-forward product
def ffn_case(ops, x, wg, wu, kind, dy=None):
    leaves = [t.detach().requires_grad_(dy is not None) for t in (x, wg, wu)]
    y = ops.silu_gated_linear(*leaves)
    want = orc.silu_gated_linear(*(to64(t).reshape(-1, t.shape[-1]) for t in (x, wg, wu)), kind,
                                 None if dy is None else to64(dy).reshape(-1, wg.shape[0]))
    assert y.shape == (*x.shape[:-1], wg.shape[0]) and y.dtype == x.dtype
    check(y.reshape(-1, wg.shape[0]), want["y"], kind, "y")
    if dy is not None:
        for got, leaf, name in zip(torch.autograd.grad(y, leaves, dy), leaves, ("dx", "dwg", "dwu")):
            assert got.shape == leaf.shape and got.dtype == leaf.dtype
            check(got.reshape(-1, leaf.shape[-1]), want[name], kind, name)


@pytest.mark.parametrize("kind", ["bfloat16", "float16"])
@pytest.mark.parametrize("R,C,F", [(1, 8, 8), (1, 64, 256), (3, 1, 1), (2, 7, 5), (5, 72, 40), (17, 129, 65),
                                   (64, 64, 64), (65, 136, 72), (128, 128, 256), (130, 200, 264), (300, 96, 130),
                                   (257, 65, 511), (1000, 48, 96), (129, 520, 1032)])
def test_ffn(ops, kind, R, C, F):
    x = make((R, C), kind, 1)
    wg, wu = make((F, C), kind, 2, scale=C ** -0.5), make((F, C), kind, 3, scale=C ** -0.5)
    ffn_case(ops, x, wg, wu, kind, make((R, F), kind, 4))


@pytest.mark.parametrize("R", [1, 8, 9, 16, 33, 64, 65, 100])
def test_ffn_of_few_rows(ops, R):
    C, F = 520, 1160
    ffn_case(ops, make((R, C), "bfloat16", 1), make((F, C), "bfloat16", 2, scale=C ** -0.5),
             make((F, C), "bfloat16", 3, scale=C ** -0.5), "bfloat16")


@pytest.mark.parametrize("C,F", [(2112, 64), (2240, 100), (2624, 576), (1088, 64), (512, 1000), (4160, 40), (9, 3)])
def test_ffn_of_few_rows_over_every_split(ops, C, F):
    """Cuts of the channels among the CTAs of a cluster that do not come out even."""
    for R in (2, 40):
        ffn_case(ops, make((R, C), "bfloat16", 1), make((F, C), "bfloat16", 2, scale=C ** -0.5),
                 make((F, C), "bfloat16", 3, scale=C ** -0.5), "bfloat16")


@pytest.mark.parametrize("kind", ["bfloat16", "float16"])
@pytest.mark.parametrize("R,C,F", [(70, 1536, 136), (130, 1541, 75), (300, 1600, 64), (65, 2048, 33)])
def test_ffn_wide_layers_keep_their_products(ops, kind, R, C, F):
    """From some width on the backward pass takes both products from the forward pass."""
    x = make((R, C), kind, 1)
    wg, wu = make((F, C), kind, 2, scale=C ** -0.5), make((F, C), kind, 3, scale=C ** -0.5)
    ffn_case(ops, x, wg, wu, kind, make((R, F), kind, 4))
    ffn_case(ops, x, wg, wu, kind, make((R, F + 1), kind, 4)[:, 1:])


def test_ffn_many_rows_narrow_weights(ops):
    R, C, F = 5000, 64, 128
    ffn_case(ops, make((R, C), "bfloat16", 1), make((F, C), "bfloat16", 2, scale=0.1),
             make((F, C), "bfloat16", 3, scale=0.1), "bfloat16", make((R, F), "bfloat16", 4, scale=0.01))


def test_ffn_strided_and_shaped(ops):
    kind, C, F = "bfloat16", 64, 96
    base = make((6, 7, 2 * C + 3), kind, 1)
    w = make((2 * F, C + 8), kind, 2, scale=0.1)
    wg, wu = w[:F, 8:], w[F:, :C]
    ffn_case(ops, base[..., 1:C + 1], wg, wu, kind, make((6, 7, F), kind, 4))
    ffn_case(ops, base[:, 2, :C], wg, wu, kind, make((1, 1), kind, 4).expand(6, F))
    ffn_case(ops, make((C,), kind, 5), wg, wu, kind, make((F,), kind, 6))
    ffn_case(ops, make((C, 9), kind, 5).t(), make((C, F), kind, 6, scale=0.1).t(), wu, kind, make((9, F), kind, 7))
    # one row of weights for every hidden unit
    ffn_case(ops, base[0, :, :C], make((1, C), kind, 8).expand(F, C), wu, kind, make((7, F), kind, 9))


def test_ffn_same_weights_twice(ops):
    """The gradient of a weight used on both sides is the sum of both."""
    x, w = make((70, 64), "bfloat16", 1), make((72, 64), "bfloat16", 2, scale=0.1).requires_grad_(True)
    dy = make((70, 72), "bfloat16", 3)
    (got,) = torch.autograd.grad(ops.silu_gated_linear(x, w, w), w, dy)
    want = orc.silu_gated_linear(to64(x), to64(w), to64(w), "bfloat16", to64(dy))
    value = want["dwg"][0] + want["dwu"][0]
    bound = sum(want[k][1] + orc.rounding(np.abs(want[k][0]) + want[k][1], "bfloat16") for k in ("dwg", "dwu"))
    assert orc.within(to64(got), value, bound, "bfloat16") <= 1.0


def test_ffn_of_nothing(ops):
    z = lambda *s: torch.zeros(*s, device="cuda", dtype=torch.bfloat16, requires_grad=True)  # noqa: E731
    for R, C, F in ((0, 16, 8), (4, 0, 8), (4, 16, 0)):
        x, wg, wu = z(R, C), z(F, C), z(F, C)
        y = ops.silu_gated_linear(x, wg, wu)
        assert y.shape == (R, F) and not y.any()
        for g, t in zip(torch.autograd.grad(y, (x, wg, wu), torch.ones_like(y)), (x, wg, wu)):
            assert g.shape == t.shape and not g.any()


def test_ffn_small_float16_gradients(ops):
    """Gradients near float16's smallest number keep the precision that the type gives the result."""
    R, C, F = 512, 64, 64
    x, wg, wu = make((R, C), "float16", 1), make((F, C), "float16", 2, 0.2), make((F, C), "float16", 3, 0.2)
    ffn_case(ops, x, wg, wu, "float16", make((R, F), "float16", 4, scale=2e-6))


# ------------------------------------------------------------------------- dropout
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n,p", [(1, 0.5), (7, 0.3), (8, 0.5), (1000, 0.1), (4099, 0.7), (33, 0.0), (33, 1.0)])
def test_dropout(ops, kind, n, p):
    seed, offset = (12345 << 31) + 77, (1 << 40) + 5
    rng = torch.tensor([seed, offset], device="cuda")
    x, res, dy = (make((n,), kind, i) for i in (1, 2, 3))
    keep = orc.philox_halves(n, seed, offset) >= round(p * 65536)
    factor = keep * (65536.0 / max(1, 65536 - round(p * 65536)))
    xl, rl = x.detach().requires_grad_(True), res.detach().requires_grad_(True)
    y = ops.dropout_add(xl, rl, p, rng)
    dx, dres = torch.autograd.grad(y, (xl, rl), dy)
    scaled = to64(x) * factor
    check(y, (to64(res) + scaled, 2 * orc.U * np.abs(scaled) + orc.U * (np.abs(to64(res)) + np.abs(scaled))), kind, "y")
    check(dx, (to64(dy) * factor, 2 * orc.U * np.abs(to64(dy) * factor)), kind, "dx")
    assert torch.equal(dres, dy)
    alone = ops.dropout_add(x, None, p, rng)
    check(alone, (scaled, 2 * orc.U * np.abs(scaled)), kind, "alone")
    assert torch.equal(alone == 0, torch.tensor(~keep, device="cuda") | (x == 0))


def test_dropout_known_block(ops):
    """The published test value of Philox4x32-10 for an all-zero counter and key."""
    halves = orc.philox_halves(8, 0, 0)
    words = [int(halves[2 * i]) | int(halves[2 * i + 1]) << 16 for i in range(4)]
    assert words == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]


def test_dropout_rate_and_independence(ops):
    n, p = 1 << 20, 0.1
    one = torch.ones(n, device="cuda")
    masks = [ops.dropout_add(one, None, p, torch.tensor(r, device="cuda")) != 0 for r in ([1, 0], [1, 1], [2, 0])]
    for m in masks:  # six standard deviations of a binomial count
        assert abs(m.float().mean().item() - 0.9) < 6 * (0.09 / n) ** 0.5
    for i, j in ((0, 1), (0, 2), (1, 2)):
        assert abs((masks[i] & masks[j]).float().mean().item() - 0.81) < 6 * (0.81 * 0.19 / n) ** 0.5
    assert torch.equal(masks[0], ops.dropout_add(one, None, p, torch.tensor([1, 0], device="cuda")) != 0)


def test_dropout_dropped_infinities(ops):
    x = torch.full((4096,), float("inf"), device="cuda")
    res = make((4096,), "float32", 1)
    y = ops.dropout_add(x, res, 0.5, torch.tensor([3, 4], device="cuda"))
    kept = torch.isinf(y)
    assert 0 < int(kept.sum()) < 4096 and torch.equal(y[~kept], res[~kept])


def test_dropout_strided_and_broadcast(ops):
    rng = torch.tensor([5, 6], device="cuda")
    x = make((6, 40), "bfloat16", 1).t()
    res = make((1, 6), "bfloat16", 2).requires_grad_(True)
    y = ops.dropout_add(x, res.expand(40, 6), 0.25, rng)
    assert torch.equal(y, ops.dropout_add(x.contiguous(), res.expand(40, 6).contiguous(), 0.25, rng))
    (d,) = torch.autograd.grad(y, res, torch.ones_like(y))
    assert d.shape == (1, 6) and torch.equal(d, torch.full_like(d, 40.0))
    odd = make((81,), "bfloat16", 3)[1:]
    assert torch.equal(ops.dropout_add(odd, None, 0.25, rng), ops.dropout_add(odd.clone(), None, 0.25, rng))


def test_dropout_changed_numbers_are_noticed(ops):
    rng = torch.tensor([5, 6], device="cuda")
    x = make((64,), "float32", 1).requires_grad_(True)
    y = ops.dropout_add(x, None, 0.5, rng)
    rng += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


# -------------------------------------------------- streams, graphs, refusals, errors
def test_other_stream_and_captured_replay(ops):
    B, T, C, F = 2, 300, 64, 128
    f, x, gate = (make((B, T, C), "bfloat16", i) for i in (1, 2, 3))
    wg, wu = make((F, C), "bfloat16", 4, scale=0.1), make((F, C), "bfloat16", 5, scale=0.1)
    h, rng = make((B, C), "float32", 6), torch.tensor([7, 8], device="cuda")

    def run():
        leaves = [t.detach().requires_grad_(True) for t in (f, x, gate, wg, wu)]
        y, last = ops.gated_scan(*leaves[:2], gate=leaves[2])
        z = ops.silu_gated_linear(ops.dropout_add(y, leaves[1], 0.1, rng), leaves[3], leaves[4])
        step = h.clone()
        ys = ops.gated_step(f[:, 0], x[:, 0], step)
        grads = torch.autograd.grad((z, last), leaves, (torch.ones_like(z), torch.ones_like(last)))
        return [y, last, z, ys, step, *grads]

    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(want, other):
        assert torch.equal(a, b)
    del want, other
    graphs, outs = [], []
    for _ in range(2):  # two graphs of the same calls, replayed one after the other and mixed
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run())
        graphs.append(g)
    for t, s in ((f, 11), (x, 12), (gate, 13), (wg, 14), (wu, 15)):
        t.copy_(make(t.shape, "bfloat16", s, scale=0.3))
    rng.add_(1)
    for g in (graphs[0], graphs[1], graphs[0]):
        g.replay()
    torch.cuda.synchronize()
    want = run()
    for out in outs:
        for a, b in zip(want, out):
            assert torch.equal(a, b)


def test_calls_of_two_streams_at_once(ops):
    f, x, gate = (make((3, 900, 96), "bfloat16", i) for i in (1, 2, 3))
    a, wg, wu = make((700, 200), "bfloat16", 4), make((300, 200), "bfloat16", 5, 0.1), make((300, 200), "bfloat16", 6, 0.1)
    dy, da = make((3, 900, 96), "bfloat16", 7), make((700, 300), "bfloat16", 8)

    def run():
        leaves = [t.detach().requires_grad_(True) for t in (f, x, gate, a, wg, wu)]
        y, h = ops.gated_scan(*leaves[:2], gate=leaves[2])
        z = ops.silu_gated_linear(*leaves[3:])
        few = ops.silu_gated_linear(a[:20], wg, wu)
        return [y, h, z, few, *torch.autograd.grad((y, z), leaves, (dy, da))]

    want = run()
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(run())
    torch.cuda.synchronize()
    for out in got:
        for a_, b_ in zip(want, out):
            assert torch.equal(a_, b_)


def test_some_gradients_only(ops):
    """What is not asked for does not change what is."""
    R, C, F = 90, 72, 80
    x, wg, wu, dy = make((R, C), "bfloat16", 1), make((F, C), "bfloat16", 2, 0.1), make((F, C), "bfloat16", 3, 0.1), make((R, F), "bfloat16", 4)
    every = [t.detach().requires_grad_(True) for t in (x, wg, wu)]
    want = torch.autograd.grad(ops.silu_gated_linear(*every), every, dy)
    for keep in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1), (0, 1, 1)):
        args = [t.detach().requires_grad_(bool(k)) for t, k in zip((x, wg, wu), keep)]
        got = torch.autograd.grad(ops.silu_gated_linear(*args), [t for t, k in zip(args, keep) if k], dy)
        for g, w in zip(got, [w for w, k in zip(want, keep) if k]):
            assert torch.equal(g, w)
    rng = torch.tensor([1, 2], device="cuda")
    res = x.detach().requires_grad_(True)
    (d,) = torch.autograd.grad(ops.dropout_add(x, res, 0.5, rng), res, x)
    assert torch.equal(d, x)
    (d,) = torch.autograd.grad(ops.dropout_add(res, x, 0.5, rng), res, x)
    assert torch.equal(d, ops.dropout_add(x, None, 0.5, rng))
    T = 70
    f, v = make((2, T, C), "float16", 5), make((2, T, C), "float16", 6)
    h0 = make((2, C), "float16", 7).requires_grad_(True)
    y, h = ops.gated_scan(f, v, h0=h0)
    (d,) = torch.autograd.grad(h, h0, torch.ones_like(h))
    assert d.dtype == torch.float16
    want = orc.gated_scan(to64(f).reshape(-1, C), to64(v).reshape(-1, C), to64(h0), None, [(0, T), (T, 2 * T)], None, np.ones((2, C)))
    check(d, want["dh0"], "float16", "dh0")


def test_offsets_past_32_bits(ops):
    """Rows far apart, and a tensor of more than 2^31 elements."""
    T, C, far = 70, 64, 1 << 25
    big = torch.empty(T * far, device="cuda", dtype=torch.bfloat16).view(T, far)
    big[:, :3 * C] = make((T, 3 * C), "bfloat16", 1)
    f, x, gate = (big[:, i * C:(i + 1) * C] for i in range(3))
    scan_case(ops, f[None], x[None], None, gate[None], None, "bfloat16", dy=make((1, T, C), "bfloat16", 5))
    cu = torch.tensor([0, 33, T], dtype=torch.int32, device="cuda")
    scan_case(ops, f, x, None, gate, cu, "bfloat16", dy=make((T, C), "bfloat16", 5))
    w = make((2 * 72, C), "bfloat16", 6, scale=0.1)
    ffn_case(ops, x, w[:72], w[72:], "bfloat16", make((T, 72), "bfloat16", 7))
    ffn_case(ops, x[:40], w[:72], w[72:], "bfloat16")
    h = torch.zeros(T, C, device="cuda")
    assert torch.equal(ops.gated_step(f, x, h), ops.gated_step(f.contiguous(), x.contiguous(), torch.zeros_like(h)))
    del big, f, x, gate
    n = (1 << 31) + 29
    one = torch.ones(n, device="cuda", dtype=torch.bfloat16)
    y = ops.dropout_add(one, None, 0.5, torch.tensor([11, 12], device="cuda"))
    first = (1 << 31) - 64  # a multiple of 8: block 2^28 - 8 on
    halves = orc.philox_halves(64 + 29, 11, 12, first // 8)
    assert torch.equal(y[first:].float().cpu(), torch.tensor(np.where(halves >= 32768, 2.0, 0.0), dtype=torch.float32))


def test_same_inputs_same_bits(ops):
    f, x, dy = (make((2, 1500, 64), "bfloat16", i) for i in (1, 2, 3))
    xw, wg, wu, dw = (make(s, "bfloat16", 4, scale=0.2) for s in ((3000, 64), (128, 64), (128, 64), (3000, 128)))

    def run():
        leaves = [t.detach().requires_grad_(True) for t in (f, x, xw, wg, wu)]
        y, h = ops.gated_scan(*leaves[:2])
        z = ops.silu_gated_linear(*leaves[2:])
        return [y, h, z, *torch.autograd.grad((y, z), leaves, (dy, dw))]

    first = run()
    for _ in range(3):
        for a, b in zip(first, run()):
            assert torch.equal(a, b)


def test_refusals(ops):
    t = lambda *s, d=torch.bfloat16: torch.zeros(*s, device="cuda", dtype=d)  # noqa: E731
    f = t(2, 4, 8)
    for bad in (lambda: ops.gated_scan(f, t(2, 4, 9)), lambda: ops.gated_scan(f, t(2, 4, 8, d=torch.float16)),
                lambda: ops.gated_scan(f.double(), f.double()), lambda: ops.gated_scan(f[0], f[0]),
                lambda: ops.gated_scan(f, f, h0=t(3, 8)), lambda: ops.gated_scan(f, f, gate=t(2, 4, 4)),
                lambda: ops.gated_scan(f[0], f[0], cu_seqlens=torch.tensor([0, 4], device="cuda")),
                lambda: ops.gated_scan(f[0], f[0], cu_seqlens=torch.zeros(1, dtype=torch.int32, device="cuda")),
                lambda: ops.gated_scan(f, f, cu_seqlens=torch.zeros(2, dtype=torch.int32, device="cuda")),
                lambda: ops.gated_step(f[0], f[0], t(4, 8)), lambda: ops.gated_step(f[0], f[0], t(3, 8, d=torch.float32)),
                lambda: ops.gated_step(f[0].clone().requires_grad_(True), f[0], t(4, 8, d=torch.float32)),
                lambda: ops.silu_gated_linear(t(4, 8), t(6, 9), t(6, 9)),
                lambda: ops.silu_gated_linear(t(4, 8), t(6, 8), t(7, 8)),
                lambda: ops.silu_gated_linear(*(t(*s, d=torch.float32) for s in ((4, 8), (6, 8), (6, 8)))),
                lambda: ops.dropout_add(f, t(2, 4, 1), 0.1, torch.zeros(2, dtype=torch.int64, device="cuda")),
                lambda: ops.dropout_add(f, f, 1.5, torch.zeros(2, dtype=torch.int64, device="cuda")),
                lambda: ops.dropout_add(f, f, float("nan"), torch.zeros(2, dtype=torch.int64, device="cuda")),
                lambda: ops.dropout_add(f, f, 0.1, torch.zeros(3, dtype=torch.int64, device="cuda")),
                lambda: ops.dropout_add(f, f, 0.1, torch.zeros(2, device="cuda"))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        ops.gated_scan(f.cpu(), f)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        ops.dropout_add(f, f, 0.1, torch.zeros(2, dtype=torch.int64))
    g = f.clone().requires_grad_(True)
    (d,) = torch.autograd.grad(ops.gated_scan(g, f)[0].sum(), g, create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()
