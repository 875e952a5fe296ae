"""Layer norm of 16-bit rows against its 64-bit form, at the widths, strides and values where it can go wrong."""
import pytest
import torch

import linear_attention_oracle as orc

pytestmark = pytest.mark.gpu
TYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16}


@pytest.fixture(scope="module")
def ops():
    from csn_b200 import ops
    return ops


def make(shape, typ, seed, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale + shift).to(typ).cuda()


def check(ops, x, w, b, dy, eps=1e-5, wants="xwb"):
    leaves = {n: t.detach().requires_grad_(n in wants) for n, t in (("x", x), ("w", w), ("b", b))}
    y = ops.layer_norm(leaves["x"], leaves["w"], leaves["b"], eps)
    assert y.dtype == x.dtype and y.shape == x.shape
    flat = lambda t: t.detach().double().reshape(-1, x.shape[-1])  # noqa: E731
    want = orc.layer_norm(flat(x), w.double(), b.double(), eps, flat(dy))
    got = {"y": y}
    names = [n for n in "xwb" if n in wants]
    for n, t in zip(names, torch.autograd.grad(y, [leaves[n] for n in names], dy)):
        assert t.dtype == leaves[n].dtype and t.shape == leaves[n].shape
        got["d" + n] = t
    for n, t in got.items():
        value, bound = want[n]
        share = orc.used(t.reshape(value.shape), value, bound, t.dtype)
        assert share <= 1.0, f"{n}: {share:.2f} of the allowed error"


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("C", [1, 2, 7, 8, 64, 96, 128, 136, 250, 256, 771, 1024, 1032, 2048, 2050, 4096, 5000, 8192, 8200, 16384, 20001, 40000])
def test_widths(ops, kind, wide, C):
    typ = TYPES[kind]
    for R in (1, 3, 37):
        x = make((R, C), typ, C + R, 2.0, 0.5)
        w, b = (make((C,), torch.float32 if wide else typ, C + i, 0.3, s) for i, s in ((1, 1.0), (2, 0.0)))
        check(ops, x, w, b, make((R, C), typ, C + 3))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("R,C", [(5000, 128), (4099, 771), (20001, 16), (3001, 2048), (700, 8192), (65, 16392)])
def test_many_rows(ops, kind, R, C):
    typ = TYPES[kind]
    check(ops, make((R, C), typ, 1, 2.0, 0.5), make((C,), torch.float32, 2, 0.3, 1.0), make((C,), torch.float32, 3), make((R, C), typ, 4))


@pytest.mark.parametrize("kind", list(TYPES))
def test_layouts(ops, kind):
    typ = TYPES[kind]
    w, b = make((96,), typ, 1, 0.3, 1.0), make((96,), typ, 2)
    whole = make((6, 5, 200), typ, 3)
    dy = make((6, 5, 96), typ, 4)
    for x in (whole[..., 8:104], whole[..., 3:99], whole[..., :192:2], whole[..., :96].transpose(0, 1).contiguous().transpose(0, 1)):
        check(ops, x, w, b, dy)
    check(ops, whole[0, 0, :96], w, b, dy[0, 0])
    check(ops, whole[..., :96], w, b, dy[:1, :1].expand(6, 5, 96))  # a broadcast gradient
    check(ops, whole[..., :96], w[:1].expand(96), b, dy)
    off = torch.empty(96 * 30 + 1, device="cuda", dtype=typ)[1:].view(30, 96).copy_(whole[..., :96].reshape(30, 96))
    check(ops, off, w, b, dy.reshape(30, 96))


@pytest.mark.parametrize("wants", ["x", "w", "b", "xw", "wb"])
def test_gradients_one_by_one(ops, wants):
    typ = torch.bfloat16
    check(ops, make((50, 136), typ, 1), make((136,), typ, 2), make((136,), typ, 3), make((50, 136), typ, 4), wants=wants)


@pytest.mark.parametrize("C", [128, 771, 8192])
def test_values(ops, C):
    """Rows far from 0, of one value, and with a NaN or an infinity, which stay in their rows."""
    x = make((8, C), torch.float16, 1, 0.5, 200.0)
    x[2] = 3.0
    w, b, dy = make((C,), torch.float16, 2, 0.3, 1.0), make((C,), torch.float16, 3), make((8, C), torch.float16, 4)
    check(ops, x, w, b, dy, eps=1e-3)
    want = ops.layer_norm(x, w, b)
    assert torch.equal(want[2], b)
    x[4, C // 2], x[6, 0] = float("nan"), float("inf")
    y = ops.layer_norm(x, w, b)
    assert y[4].isnan().all() and y[6].isnan().all()
    keep = [0, 1, 2, 3, 5, 7]
    assert torch.equal(y[keep], want[keep])


def test_empty(ops):
    x = torch.zeros(0, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    w, b = (torch.ones(64, device="cuda", dtype=torch.bfloat16, requires_grad=True) for _ in range(2))
    y = ops.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.zeros_like(y))
    assert y.shape == dx.shape == (0, 64) and (dw == 0).all() and (db == 0).all()


def test_the_same_bits_again(ops):
    x, w, b, dy = make((3001, 512), torch.bfloat16, 1), make((512,), torch.float32, 2), make((512,), torch.float32, 3), make((3001, 512), torch.bfloat16, 4)
    runs = []
    for _ in range(2):
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        runs.append(torch.autograd.grad(ops.layer_norm(*leaves), leaves, dy))
    assert all(torch.equal(p, q) for p, q in zip(*runs))
