"""The linear-attention operators together, as they are used: modules, captured steps, streams, and the calls that their documentation allows."""
import pytest
import torch

import linear_attention_oracle as orc

pytestmark = pytest.mark.gpu
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


@pytest.fixture(scope="module")
def ops():
    from csn_b200 import ops
    return ops


def make(shape, kind, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(TYPES[kind]).cuda()


def decays(H):
    return (-torch.exp2(-torch.linspace(0.0, 9.0, H)) * 2.0).cuda()


def block(kind, **kw):
    from csn_b200.modules import LinearAttentionBlock
    torch.manual_seed(0)
    return LinearAttentionBlock(128, 4, **kw).cuda().to(TYPES[kind])


@pytest.mark.parametrize("kind", list(TYPES))
def test_block_trains_and_generates(kind):
    """Gradients reach every parameter; a sequence, its two halves, a packed one and its tokens one by one agree."""
    blk = block(kind, num_kv_heads=2)
    x = make((2, 150, 128), kind, 1).requires_grad_(True)
    out, s = blk(x)
    (out.float().square().mean() + s.square().mean()).backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() and p.grad.abs().sum() > 0 for p in [x, *blk.parameters()])
    blk.eval()
    with torch.no_grad():
        whole, last = blk(x)
        first, mid = blk(x[:, :70])
        rest, end = blk(x[:, 70:], mid)
        cu = torch.tensor([0, 150, 300], dtype=torch.int32, device="cuda")
        packed, ends = blk(x.flatten(0, 1), cu_seqlens=cu)
        state = mid.clone()
        steps = torch.stack([blk.step(x[:, t], state) for t in range(70, 80)], 1)
        shorter = blk(x[:, 70:80], mid)[1]
    # every value passes a dozen roundings to the layer's type on its way, each half a step of values of a few units
    near = lambda a, b, n=16: (a.float() - b.float()).abs().max() <= n * orc.HALF_STEP[TYPES[kind]] * (1 + b.float().abs().max()) + 2e-5  # noqa: E731
    assert near(torch.cat([first, rest], 1), whole) and near(end, last) and near(packed.view_as(whole), whole) and near(ends, last)
    assert near(steps, whole[:, 70:80]) and near(state, shorter)


@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
def test_captured_training_step(kind):
    """The block's forward and backward pass as one CUDA graph gives what it gives eagerly, on every replay."""
    from csn_b200.graphs import TrainStepGraph

    class Model(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.blocks = torch.nn.ModuleList([block(kind, num_kv_heads=2) for _ in range(2)])

        def forward(self, x):
            for b in self.blocks:
                x, s = b(x)
            return x, x.float().square().mean() + s.square().mean()

    model = Model()
    xs = [make((1, 700, 128), kind, i) for i in (1, 2)]  # long enough for segments
    want = []
    for x in xs:
        model.zero_grad(set_to_none=True)
        out, loss = model(x)
        loss.backward()
        want.append((out.detach().clone(), [p.grad.clone() for p in model.parameters()]))
        del out, loss
    model.zero_grad(set_to_none=True)
    step = TrainStepGraph(model, None, [xs[0]])
    for i in (0, 1, 0):
        out = step(xs[i])[0]
        assert torch.equal(out, want[i][0])
        for p, g in zip(model.parameters(), want[i][1]):
            assert torch.equal(p.grad, g)


def test_two_graphs_and_eager_calls_share_nothing(ops):
    """Workspaces of captured calls are their own: replays in any order, with eager calls between, on two streams."""
    g = decays(2)
    ins = [[make((1, 1500, 2, 64), "bfloat16", 10 * j + i) for i in range(3)] for j in range(2)]
    want = [ops.linear_attention(*i, g) for i in ins]
    graphs, outs = [], []
    for i in ins:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.linear_attention(*i, g))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        again = ops.linear_attention(*ins[0], g)
        torch.cuda.synchronize()
        for got, w in ((outs[0], want[0]), (outs[1], want[1]), (again, want[0])):
            assert torch.equal(got[0], w[0]) and torch.equal(got[1], w[1])


def test_other_streams(ops):
    """Calls on three streams at a time give what they give alone."""
    g = decays(4)
    ins = [[make((2, 600, 4, 64), "float16", 10 * j + i) for i in range(3)] for j in range(3)]
    do = make((2, 600, 4, 64), "float16", 99)

    def run(i):
        leaves = [t.detach().requires_grad_(True) for t in i]
        o, _ = ops.linear_attention(*leaves, g)
        return [o.detach(), *torch.autograd.grad(o, leaves, do)]

    want = [run(i) for i in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ins]
    got = [[] for _ in ins]
    for _ in range(3):
        for j, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[j] = run(ins[j])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for w, r in zip(want, got) for a, b in zip(w, r))


@pytest.mark.parametrize("kind", list(TYPES))
def test_the_same_bits_again(ops, kind):
    q, k, v, do = (make((2, 900, 4, 40), kind, i) for i in range(4))
    runs = []
    for _ in range(2):
        leaves = [t.detach().requires_grad_(True) for t in (q, k[:, :, :2], v[:, :, :2])]
        o, s = ops.linear_attention(*leaves, decays(4))
        runs.append([o, s, *torch.autograd.grad((o, s), leaves, (do, torch.ones_like(s)))])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


@pytest.mark.parametrize("kind", list(TYPES))
def test_infinities_stay_in_their_sequences_heads_and_blocks(ops, kind):
    B, T, H, D = 2, 400, 2, 64
    q, k, v = (make((B, T, H, D), kind, i) for i in range(3))
    g = decays(H)
    want, last = ops.linear_attention(q, k, v, g)
    k2, v2 = k.clone(), v.clone()
    k2[1, 300, 1, 3], v2[1, 301, 1, 5] = float("inf"), float("nan")
    o, s = ops.linear_attention(q, k2, v2, g)
    first = 256 if kind != "float32" else 300  # 16 bits: the block's other outputs, too
    assert torch.equal(o[0], want[0]) and torch.equal(o[1, :, 0], want[1, :, 0]) and torch.equal(o[1, :first], want[1, :first])
    assert torch.equal(s[0], last[0]) and torch.equal(s[1, 0], last[1, 0])
    assert not torch.isfinite(o[1, 301:, 1, 5]).any() and torch.isfinite(s[1, 1, 4, 6])


def test_float16_keeps_its_range(ops):
    """Products far above 65504 and far below 2^-14, whose results fit."""
    B, T, H, D = 1, 200, 2, 64
    g = decays(H)
    q, k, v = (make((B, T, H, D), "float16", i) for i in range(3))
    for a, b, c in ((100.0, 100.0, 2.0 ** -10), (2.0 ** -9, 2.0 ** -9, 2.0 ** 9), (2.0 ** -12, 400.0, 16.0)):
        x, y, z = (q * a).half(), (k * b).half(), (v * c).half()
        o, s = ops.linear_attention(x, y, z, g, scale=1.0 / 64)
        want = orc.attention(*(t.double().cpu().flatten(0, 1) for t in (x, y, z)), g.cpu(), torch.zeros(1, H, D, D, dtype=torch.float64), [(0, T)], 1.0 / 64)
        # one more rounding than the oracle's step-by-step bound, relative to the largest of a row
        for got, (value, size), typ, more in ((o, want["o"], torch.float16, 1.01 * 2.0 ** -11 + 2.0 ** -16), (s, want["s"], torch.float32, 2.0 ** -22 * T)):
            bound = orc.steps(T, D) * orc.U * size + more * size.max()
            assert orc.used(got.reshape(value.shape), value, bound, typ) <= 1.0


def test_long_offsets(ops):
    """Rows whose places lie past 2^31 elements, and a single long row of heads."""
    H, D = 2, 64
    pitch = 1 << 23  # elements from row to row
    T = 300
    room = torch.empty(T * pitch + 3 * H * D, device="cuda", dtype=torch.bfloat16)
    rows = room[:T * pitch].view(T, pitch)[:, :3 * H * D].unflatten(-1, (3, H, D))
    small = make((T, 3, H, D), "bfloat16", 1)
    rows.copy_(small)
    g = decays(H)
    got = ops.linear_attention(*(rows[None, :, i] for i in range(3)), g)
    want = ops.linear_attention(*(small[None, :, i].contiguous() for i in range(3)), g)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("borders", [[-5, 60, 30, 400], [0, 500, 100, 100], [200, 150, 100, 50], [1 << 30, -(1 << 30), 7, 9]])
def test_any_borders_stay_inside(ops, kind, borders):
    """Borders outside the rows, or falling ones, are cut to what is there: every access stays inside, and what a sequence with good
    borders of its own gives is finite."""
    cu = torch.tensor(borders, dtype=torch.int32, device="cuda")
    L, S = 300, len(borders) - 1
    q, k, v = (make((L, 2, 64), kind, i).requires_grad_(True) for i in range(3))
    o, s = ops.linear_attention(q, k, v, decays(2), s0=make((S, 2, 64, 64), "float32", 4), cu_seqlens=cu)
    torch.autograd.grad((o, s), (q, k, v), (torch.ones_like(o), torch.ones_like(s)))
    torch.cuda.synchronize()
    good = [(a, b) for a, b in zip(borders[:-1], borders[1:]) if 0 <= a < b <= L]
    for a, b in good[:1]:
        assert torch.isfinite(o[a:b]).all()


def test_no_rows(ops):
    """Packed sequences without a row: the states pass through, and so do their gradients."""
    for kind in TYPES:
        q = torch.zeros(0, 2, 16, device="cuda", dtype=TYPES[kind])
        s0 = make((3, 2, 16, 16), "float32", 1).requires_grad_(True)
        o, s = ops.linear_attention(q, q, q, decays(2), s0=s0, cu_seqlens=torch.zeros(4, dtype=torch.int32, device="cuda"))
        ds = make((3, 2, 16, 16), "float32", 2)
        assert o.shape == (0, 2, 16) and torch.equal(s, s0) and torch.equal(torch.autograd.grad(s, s0, ds)[0], ds)


def test_registered_operators(ops):
    csn = torch.ops.csn
    q, k, v = (make((2, 140, 2, 32), "bfloat16", i).requires_grad_(True) for i in range(3))
    s0 = make((2, 2, 32, 32), "float32", 4).requires_grad_(True)
    g, do, ds = decays(2), make((2, 140, 2, 32), "bfloat16", 5), make((2, 2, 32, 32), "float32", 6)
    a = ops.linear_attention(q, k, v, g, s0=s0)
    b = csn.linear_attention_fwd(q, k, v, g, s0, None, None)
    for x, y in zip((*a, *torch.autograd.grad(a, (q, k, v, s0), (do, ds))), (*b, *torch.autograd.grad(b, (q, k, v, s0), (do, ds)))):
        assert torch.equal(x, y)
    s1, s2 = s0.detach().clone(), s0.detach().clone()
    with torch.no_grad():
        one = ops.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, s1)
        two = csn.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, s2, None)
    assert torch.equal(one, two) and torch.equal(s1, s2)


def test_second_derivatives_are_refused(ops):
    q, k, v = (make((1, 20, 1, 16), "float32", i).requires_grad_(True) for i in range(3))
    o, _ = ops.linear_attention(q, k, v, decays(1))
    (dq,) = torch.autograd.grad(o.sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        dq.sum().backward()
    x = make((4, 64), "bfloat16", 1).requires_grad_(True)
    w, b = torch.ones(64, device="cuda", dtype=torch.bfloat16), torch.zeros(64, device="cuda", dtype=torch.bfloat16)
    (dx,) = torch.autograd.grad(ops.layer_norm(x, w, b).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        dx.sum().backward()


def test_step_changes_only_its_state(ops):
    """The state's version rises, a state with a gradient is refused, and a step in a graph advances it at every replay."""
    q, k, v = (make((2, 2, 32), "bfloat16", i) for i in range(3))
    g, s = decays(2), torch.zeros(2, 2, 32, 32, device="cuda")
    version = s._version
    ops.linear_attention_step(q, k, v, g, s)
    assert s._version > version
    with pytest.raises(ValueError):
        ops.linear_attention_step(q, k, v, g, s.clone().requires_grad_(True))
    eager = s.clone()
    graph = torch.cuda.CUDAGraph()
    kept = s.clone()
    with torch.cuda.graph(graph):
        o = ops.linear_attention_step(q, k, v, g, s)
    s.copy_(kept)
    for _ in range(3):
        graph.replay()
        want = ops.linear_attention_step(q, k, v, g, eager)
        assert torch.equal(s, eager) and torch.equal(o, want)


def test_gated_block_in_16_bits_norms_its_own_type(ops):
    """GatedRecurrentBlock's norms of bfloat16 rows, of a width that float32 rows may not have, too."""
    from csn_b200.modules import GatedRecurrentBlock
    torch.manual_seed(0)
    blk = GatedRecurrentBlock(1032, d_inner=64, d_ffn=64).cuda().bfloat16()
    x = make((2, 40, 1032), "bfloat16", 1).requires_grad_(True)
    out, _ = blk(x)
    out.float().square().mean().backward()
    assert torch.isfinite(out).all() and all(torch.isfinite(p.grad).all() for p in [x, *blk.parameters()])
