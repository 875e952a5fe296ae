"""The gated block's operators over the whole range of what enters them, against 64-bit forms whose bounds are relative
to what an output is made of: forget gates that close, float16 gradients of mixed sizes and products near the type's end."""
import numpy as np
import pytest
import torch

import gated_oracle as orc

pytestmark = pytest.mark.gpu
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
U = orc.U


@pytest.fixture(scope="module")
def ops():
    from csn_b200 import ops
    return ops


def to64(t):
    return t.detach().double().cpu().numpy()


def rand(shape, kind, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(TYPES[kind]).cuda()


def check(got, want, kind, what):
    used = orc.within(to64(got), want[0], want[1], kind)
    assert used <= 1.0, f"{what}: {used:.2f} of the allowed error"


# ------------------------------------------------------------------------ the scan
# With e = exp(f), off by (4 + 2 |f|) U of itself (two steps of the fast exponential, and its rounded argument):
# q = 1 / (1 + e) is off by that share of e q = a, by the sum's rounding (1 U) and the reciprocal's (4 U); for f < 0
# a = e q is off by (4 + 2 |f|) U (its share of e, the smaller one of q included twice at most: 2 (4 + 2 |f|)), 5 U and its own
# rounding, so by less than (16 + 4 |f|) U of itself; for f >= 0 a = 1 - q by q's error and one rounding of a number
# in [1/2, 1], U.  The states are sums of terms, each a product along its way; `size` is the sum of the terms' sizes.  A
# step multiplies a term by a (its error, and 1 U for the product) and rounds a sum (1 U of its size); composing steps first
# and applying the maps after that rounds as many products and sums along any way, and one product and one sum more for
# each of the up to three levels (steps of a warp, warps of a pass, chunks), so 4 U a step and 16 U at the end
# cover any order.  A product of decays that falls below 2^-126 loses bits: SMALL of what it multiplies.
SMALL = 2.0 ** -120


def closed_scan(f, x, h0, gate, borders, dy, dh):
    L, C = f.shape
    a, q = orc.sigmoid(f), orc.sigmoid(-f)
    rel = (16 + 4 * np.abs(f)) * U
    a_off = np.where(f < 0, rel * a, rel * q + U)
    q_off = rel * np.minimum(a, q) + 6 * U * q
    w = orc.sigmoid(gate) if gate is not None else None
    silu = gate * w if gate is not None else np.ones_like(f)
    fast = (16 + 2 * np.abs(gate)) * U if gate is not None else 0.0
    silu_off = fast * np.abs(silu)

    def run(order, start, add, add_off):
        """s_t = a_t s_{t-1} + add_t along `order`: (before, its error, its size) at each row, and those at the end."""
        s, off, size = start.copy(), np.zeros(C), np.abs(start)
        for t in order:
            yield t, s, off + (16 * U + SMALL) * size, size
            off = a[t] * off + (a_off[t] + 4 * U * a[t]) * size + add_off[t] + 4 * U * np.abs(add[t])
            s, size = a[t] * s + add[t], a[t] * size + np.abs(add[t])
        yield None, s, off + (16 * U + SMALL) * size, size

    zero = lambda: np.zeros((L, C))  # noqa: E731
    before, before_off, h, h_off = zero(), zero(), zero(), zero()
    last, last_off = np.zeros_like(h0), np.zeros_like(h0)
    for s, (b, e) in enumerate(borders):
        seen = list(run(range(b, e), h0[s], q * x, q_off * np.abs(x) + U * np.abs(q * x)))
        for (t, v, off, _), (_, v1, off1, _) in zip(seen, seen[1:]):
            before[t], before_off[t], h[t], h_off[t] = v, off, v1, off1
        last[s], last_off[s] = seen[-1][1:3]
    out = {"y": (h * silu, h_off * np.abs(silu) + np.abs(h) * silu_off + 2 * U * np.abs(h * silu)), "h": (last, last_off)}
    # lam_t = e_t + mu_t with mu_{t-1} = a_t lam_t: the same recurrence with a_t (e_t + mu_t)
    e_t = dy * silu
    e_off = np.abs(dy) * silu_off + 2 * U * np.abs(e_t)
    lam, lam_off = zero(), zero()
    dh0, dh0_off = np.zeros_like(h0), np.zeros_like(h0)
    for s, (b, e) in enumerate(borders):
        add = a * e_t
        add_off = a_off * np.abs(e_t) + a * e_off + U * np.abs(add)
        for t, mu, off, size in run(range(e - 1, b - 1, -1), dh[s], add, add_off):
            if t is None:
                dh0[s], dh0_off[s] = mu, off
            else:
                lam[t], lam_off[t] = e_t[t] + mu, e_off[t] + off + U * (np.abs(e_t[t]) + size)
    D = before - x
    D_off = before_off + U * np.abs(D)
    df = lam * D * a * q
    out["dx"] = (lam * q, q * lam_off + (q_off + 2 * U * q) * np.abs(lam))
    out["df"] = (df, a * q * (np.abs(lam) * D_off + np.abs(D) * lam_off + lam_off * D_off)
                 + (a_off * q + a * q_off) * np.abs(lam * D) + 6 * U * np.abs(df))
    out["dh0"] = (dh0, dh0_off)
    if gate is not None:
        slope = w * (1 + gate * (1 - w))
        slope_off = w * (fast * np.abs(gate) + 2 * fast * (1 + np.abs(gate) * (1 - w)))
        out["dgate"] = (dy * h * slope, np.abs(dy) * (h_off * np.abs(slope) + np.abs(h) * slope_off + 3 * U * np.abs(h * slope)))
    return out


def closing(T, C, kind, seed):
    """Forget logits from -30 to 30 in every row, and channels that stay at one of them."""
    g = torch.Generator().manual_seed(seed)
    f = torch.rand(T, C, generator=g) * 60 - 30
    for i, v in enumerate((-8.0, -12.0, -15.0, -18.0, -25.0, 12.0)):
        if i < C:
            f[:, i] = v
    return f.to(TYPES[kind]).cuda()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("S,T,C,gated", [(3, 1, 8, False), (2, 5, 33, True), (2, 70, 40, True), (1, 130, 31, False), (1, 700, 24, True)])
def test_scan_of_gates_that_close(ops, kind, S, T, C, gated):
    """The decay of a closed gate keeps its own precision, and with it what is left of a large state and the gradients
    of the logits and of the first state: one row, warps that share a CTA, several passes, chunks."""
    f = closing(S * T, C, kind, 1)
    x, dy = rand((S * T, C), kind, 2), rand((S * T, C), kind, 3)
    gate = rand((S * T, C), kind, 4) if gated else None
    h0, dh = rand((S, C), "float32", 5, scale=1e4), rand((S, C), "float32", 6)
    want = closed_scan(*(to64(t) for t in (f, x, h0)), None if gate is None else to64(gate), [(s * T, s * T + T) for s in range(S)],
                       to64(dy), to64(dh))
    args = {"f": f, "x": x, "gate": gate}
    for packed in (False, True):
        leaves = {k: (t if packed else t.view(S, T, C)).detach().requires_grad_(True) for k, t in args.items() if t is not None}
        leaves["h0"] = h0.detach().requires_grad_(True)
        cu = torch.arange(0, S * T + 1, T, device="cuda", dtype=torch.int32) if packed else None
        y, h = ops.gated_scan(leaves["f"], leaves["x"], h0=leaves["h0"], gate=leaves.get("gate"), cu_seqlens=cu)
        grads = dict(zip(leaves, torch.autograd.grad((y, h), list(leaves.values()), (dy.view(y.shape), dh))))
        check(y.reshape(-1, C), want["y"], kind, "y")
        check(h, want["h"], "float32", "h")
        for name, key in (("f", "df"), ("x", "dx"), ("gate", "dgate"), ("h0", "dh0")):
            if name in grads:
                check(grads[name].reshape(-1, C), want[key], "float32" if name == "h0" else kind, key)


@pytest.mark.parametrize("kind", list(TYPES))
def test_step_of_gates_that_close(ops, kind):
    """What a closed gate leaves of a state far larger than its input."""
    B, C = 5, 48
    f, x, gate = closing(B, C, kind, 1), rand((B, C), kind, 2, scale=1e-3), rand((B, C), kind, 3)
    h = rand((B, C), "float32", 4, scale=1e4)
    want = closed_scan(*(to64(t) for t in (f, x, h)), to64(gate), [(b, b + 1) for b in range(B)], np.zeros((B, C)), np.zeros((B, C)))
    y = ops.gated_step(f, x, h, gate=gate)
    check(y, want["y"], kind, "y")
    check(h, want["h"], "float32", "h")


# ------------------------------------------------------- the gated product in float16
# dg and du are float16 numbers under one scale that brings the largest finite |dy| to 2^10 or above, or where dg or du would not
# fit then, the largest of these to 2^14 or above: they keep 2^-11 of themselves, or half of float16's smallest
# step, 2^-25, over the scale.  With e = exp(-|g|), off by (4 + 2 |g|) U, 1 / (1 + e) is off by that share of e, a
# sum and a reciprocal (5 U), and sigmoid of a negative number by a share of itself.
def scaled_ffn(x, wg, wu, dy):
    C, F, R = x.shape[1], wg.shape[0], x.shape[0]
    sums = lambda k: (k + 16) * 2 * U  # noqa: E731
    g, u = x @ wg.T, x @ wu.T
    g_off, u_off = sums(C) * (np.abs(x) @ np.abs(wg).T), sums(C) * (np.abs(x) @ np.abs(wu).T)
    w = orc.sigmoid(g)
    w_rel = (4 + 2 * np.abs(g)) * U * orc.sigmoid(-g) + 8 * U
    silu, slope = g * w, w * (1 + g * (1 - w))
    # |silu'| <= 1.1, |silu''| <= 0.5, |g w (1 - w)| <= 0.3, and 1 - w is off by w's error and a rounding
    silu_off = 1.1 * g_off + (w_rel + U) * np.abs(silu)
    slope_off = 0.5 * g_off + w_rel * np.abs(slope) + w * (np.abs(g) * (w_rel * w + U) + 3 * U * (1 + np.abs(g) * (1 - w)))
    dg, du = dy * u * slope, dy * silu
    dg_off = np.abs(dy) * (u_off * (np.abs(slope) + slope_off) + np.abs(u) * slope_off) + 4 * U * np.abs(dg)
    du_off = np.abs(dy) * silu_off + 2 * U * np.abs(du)
    top, peak = np.abs(dy).max(), max(np.abs(dg).max(), np.abs(du).max())
    floor = 2.0 ** -25 * max(top / 2 ** 10, peak / 2 ** 14)
    dg_off, du_off = (o + orc.HALF_STEP["float16"] * np.abs(v) + floor for o, v in ((dg_off, dg), (du_off, du)))
    aw, au, ax = np.abs(wg), np.abs(wu), np.abs(x)
    return {"dx": (dg @ wg + du @ wu, dg_off @ aw + du_off @ au + sums(2 * F) * (np.abs(dg) @ aw + np.abs(du) @ au)),
            "dwg": (dg.T @ x, dg_off.T @ ax + sums(R) * (np.abs(dg).T @ ax)),
            "dwu": (du.T @ x, du_off.T @ ax + sums(R) * (np.abs(du).T @ ax))}


def ffn_grads(ops, x, wg, wu, dy):
    leaves = [t.detach().requires_grad_(True) for t in (x, wg, wu)]
    return dict(zip(("dx", "dwg", "dwu"), torch.autograd.grad(ops.silu_gated_linear(*leaves), leaves, dy)))


# forming the products again, and keeping them (C >= 1536); rows whose tiles are whole or cut, whole pieces or odd
@pytest.mark.parametrize("R,C,F", [(200, 64, 64), (130, 72, 35), (150, 1536, 40), (70, 1541, 33)])
@pytest.mark.parametrize("largest", [1e3, 1.0, 1e-3])
def test_ffn_float16_gradients_of_mixed_sizes(ops, R, C, F, largest):
    """A row of gradients keeps its precision beside one that is 10^7 times as large."""
    x, wg, wu = rand((R, C), "float16", 1), rand((F, C), "float16", 2, C ** -0.5), rand((F, C), "float16", 3, C ** -0.5)
    size = (10.0 ** (-7 * torch.arange(R) / (R - 1))).cuda()[:, None] * largest
    dy = (rand((R, F), "float32", 4).sign() * size).half()
    want = scaled_ffn(*(to64(t) for t in (x, wg, wu, dy)))
    for name, got in ffn_grads(ops, x, wg, wu, dy).items():
        check(got, want[name], "float16", name)
    # a gradient that overflowed spoils its own row of dx alone
    dy[3, 5] = float("inf")
    dx = ffn_grads(ops, x, wg, wu, dy)["dx"]
    rest = [r for r in range(R) if r != 3]
    assert not torch.isfinite(dx[3]).all()
    some = scaled_ffn(to64(x)[rest], to64(wg), to64(wu), to64(dy)[rest])["dx"]
    check(dx[rest], some, "float16", "dx beside an infinity")


@pytest.mark.parametrize("R,C,F", [(200, 64, 64), (130, 72, 35), (150, 1536, 40), (70, 1541, 33)])
@pytest.mark.parametrize("large", ["gate", "up"])
def test_ffn_float16_gradients_of_large_products(ops, R, C, F, large):
    """Products near 10^5, with gradients that are small enough for the result."""
    s = C ** -0.5
    x = rand((R, C), "float16", 1, 64.0)
    wg = rand((F, C), "float16", 2, 1024 * s if large == "gate" else s / 64)
    wu = rand((F, C), "float16", 3, s / 2 ** 18 if large == "gate" else 1024 * s)
    dy = rand((R, F), "float16", 4, 1e-4)
    want = scaled_ffn(*(to64(t) for t in (x, wg, wu, dy)))
    for name, got in ffn_grads(ops, x, wg, wu, dy).items():
        assert torch.isfinite(got).all(), name
        check(got, want[name], "float16", name)


@pytest.mark.parametrize("R,C,F", [(200, 64, 72), (100, 1536, 40)])
def test_ffn_float16_gradients_in_a_captured_pass(ops, R, C, F):
    """A replayed pass forms dg and du again, or not, as its inputs of that replay ask for; and on several streams at once."""
    ordinary = [rand(s, "float16", i, v) for i, (s, v) in enumerate((((R, C), 1.0), ((F, C), C ** -0.5), ((F, C), C ** -0.5), ((R, F), 1.0)))]
    large = [ordinary[0] * 64, ordinary[1] * 1024, ordinary[2] / 2 ** 12, ordinary[3] * 1e-4]
    at = [t.clone() for t in ordinary]
    run = lambda: [v for _, v in sorted(ffn_grads(ops, *at).items())]  # noqa: E731
    want = {}
    for name, given in (("ordinary", ordinary), ("large", large)):
        for a, b in zip(at, given):
            a.copy_(b)
        want[name] = [t.clone() for t in run()]
        assert all(torch.isfinite(t).all() for t in want[name])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for name, given in (("large", large), ("ordinary", ordinary), ("large", large), ("large", large)):
        for a, b in zip(at, given):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want[name]):
            assert torch.equal(a, b)
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(run())
    torch.cuda.synchronize()
    for outs in got:
        for a, b in zip(outs, want["large"]):
            assert torch.equal(a, b)
