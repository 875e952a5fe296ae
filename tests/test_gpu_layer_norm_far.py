"""Layer norm of 16-bit rows far from 0 with little or no variance: what is left of a row is its distance from the mean, and
that has to be formed before anything is rounded.

Rows of one value: the distance is 0, so y is the bias and the weight's gradient is 0, to the bit.  In rows of 2000 and as many
of 1999 and 2001, whose sums float32 holds exactly, the places of 2000 are 0 in the same way."""
import pytest
import torch

from test_gpu_layer_norm_rows import TYPES, make, ops  # noqa: F401

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
WIDTHS = [8, 64, 100, 136, 250, 256, 771, 1024, 2048, 2050, 4096, 5000, 8192, 10000, 16384, 20000, 40001]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("C", WIDTHS)
def test_rows_of_one_value(ops, kind, wide, C):  # noqa: F811
    typ = TYPES[kind]
    weights = torch.float32 if wide else typ
    values = torch.tensor([100.0, -1000.0, 5000.0, 60000.0, 0.1, 1.0, 2047.0], device="cuda").to(typ)
    x = values[:, None].expand(-1, C).contiguous().requires_grad_(True)
    w, b = make((C,), weights, 1, 0.3, 1.0).requires_grad_(True), make((C,), weights, 2)
    y = ops.layer_norm(x, w, b)
    assert torch.equal(y, b.to(typ).expand_as(y))
    dy = make((len(values), C), typ, 3)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert (dw == 0).all()
    g = dy.double() * w.detach().double()
    r, mean = 1e-5 ** -0.5, g.mean(1, keepdim=True)
    # r (g - mean g): the sum's C additions, the product, the root and the last steps, then the rounding to 16 bits
    bound = r * U * (8 * g.abs() + (C + 8) * g.abs().mean(1, keepdim=True))
    want = r * (g - mean)
    assert ((dx.double() - want).abs() <= bound + torch.finfo(typ).eps / 2 * (want.abs() + bound)).all()


@pytest.mark.parametrize("kind,middle,step", [("float16", 2000.0, 1.0), ("float16", 1000.0, 0.5), ("bfloat16", 200.0, 1.0)])
@pytest.mark.parametrize("C", [64, 250, 771, 1024, 2048, 5000, 8192])
def test_places_of_the_mean(ops, kind, middle, step, C):  # noqa: F811
    typ = TYPES[kind]
    R = 12
    x = torch.full((R, C), middle)
    order = torch.randperm(C // 4 * 2, generator=torch.Generator().manual_seed(C)) + C // 4
    x[:, order[::2]] += step
    x[:, order[1::2]] -= step
    same = (x == middle).all(0).cuda()
    x = x.to(typ).cuda()
    w, b = make((C,), torch.float32, 1, 0.3, 1.0).requires_grad_(True), torch.zeros(C, device="cuda")
    y = ops.layer_norm(x, w, b)
    assert (y[:, same] == 0).all() and (y[:, ~same] != 0).all()
    dy = make((R, C), typ, 3)
    dw, = torch.autograd.grad(y, w, dy)
    # elsewhere the mean is exact and h takes what the squares' sum leaves of its deviation, and the sum over rows its R additions
    d = x.double() - middle
    h = d / (d.square().mean(1, keepdim=True) + 1e-5).sqrt()
    allowed = (C + 16 + R) * U * (dy.double() * h).abs().sum(0)
    assert (dw[same] == 0).all() and ((dw.double() - (dy.double() * h).sum(0)).abs() <= allowed).all()


@pytest.mark.parametrize("C", [96, 771, 2048, 8200, 20001])
def test_distance_from_the_mean(ops, C):  # noqa: F811
    """float16 rows around 2000.  The mean is a float32 number: off by half a step, U |mean|, and by what its second sum leaves,
    (C + 4) U of the mean distance.  The distance takes its own rounding, and the product and the root, whose relative error
    is half the variance's, what the squares' sum adds."""
    x = make((64, C), torch.float16, 1, 0.57, 2000.0)
    w, b, dy = torch.ones(C, device="cuda", requires_grad=True), torch.zeros(C, device="cuda"), make((64, C), torch.float16, 3)
    y = ops.layer_norm(x, w, b)
    d = x.double() - x.double().mean(1, keepdim=True)
    var = (d * d).mean(1, keepdim=True) + 1e-5
    first = (C + 2) * U * x.double().abs().mean(1, keepdim=True)  # of the first mean, which the second sum corrects
    de = U * 2001 + (C + 4) * U * (d.abs().mean(1, keepdim=True) + first) + U * d.abs()
    rel = (C + 16) * U + 2 * (first / var.sqrt()) ** 2 * (C + 16) * U + (U * 2001) ** 2 / var
    want = d * var.rsqrt()
    bound = 1.01 * (de * var.rsqrt() + want.abs() * (rel + 4 * U))
    assert ((y.double() - want).abs() <= bound + 2.0 ** -11 * (want.abs() + bound)).all()
    dw, = torch.autograd.grad(y, w, dy)
    allowed = (dy.double().abs() * bound).sum(0) + 70 * U * (dy.double() * want).abs().sum(0)
    assert ((dw.double() - (dy.double() * want).sum(0)).abs() <= allowed * 1.01).all()


@pytest.mark.parametrize("C", [64, 771, 2048, 8200, 20001])
def test_squares_past_the_range(ops, C):  # noqa: F811
    """bfloat16 rows whose squares float32 does not hold: the deviation is infinite and y the bias; a NaN stays one."""
    x = torch.ones(4, C, device="cuda", dtype=torch.bfloat16)
    x[:3, ::2] = -1.0
    x[:3] *= 1e30
    x[1, 0], x[3, 1] = float("nan"), float("nan")
    w, b = make((C,), torch.bfloat16, 1, 0.3, 1.0), make((C,), torch.bfloat16, 2)
    y = ops.layer_norm(x, w, b)
    assert torch.equal(y[0], b) and torch.equal(y[2], b) and y[1].isnan().all() and y[3].isnan().all()


@pytest.mark.parametrize("C", [64, 771, 20000])
def test_backward_without_rows_or_weight(C):
    """A caller of the C ABI that has no rows need not have a weight: the sums over rows are 0."""
    import ctypes
    from csn_b200 import _lib
    null = ctypes.c_void_p(0)
    nbytes = _lib.load().csn_layer_norm_rows_bwd_workspace_bytes(0, C)
    work = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    for code, typ in ((1, torch.bfloat16), (0, torch.float32)):
        for which in ((0, 1), (0,), (1,)):
            sums = [torch.full((C + 8,), 7.0, device="cuda", dtype=typ) for _ in range(2)]
            out = [ctypes.c_void_p(t.data_ptr()) if i in which else null for i, t in enumerate(sums)]
            _lib.call("csn_layer_norm_rows_bwd", null, C, null, C, null, null, null, null, *out, 0, C, 1, code, ctypes.c_void_p(work.data_ptr()),
                      nbytes, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
            for i, t in enumerate(sums):
                assert (t[:C] == (0.0 if i in which else 7.0)).all() and (t[C:] == 7.0).all()
