"""Packed batches whose sequences are cut into segments in the backward pass too: the first pass that runs back in time, the states
joined from the last segment on, sequences that begin inside a block, end inside a segment, or lie between cut ones."""
import numpy as np
import pytest
import torch

from test_gpu_linear_attention import ALL, check, decays, fused, make, ops  # noqa: F401

pytestmark = pytest.mark.gpu
CODE = {"float32": 0, "bfloat16": 1, "float16": 2}


def assert_cut(lengths, L, H, Dk, Dv, kind):
    """Told from the workspace, which holds a state for each unit, both ways: segments of half the longest sequence at most."""
    from csn_b200 import _lib
    nbytes = _lib.load().csn_linear_attention_workspace_bytes(len(lengths), L, H, H, Dk, Dv, 1, CODE[kind], 0, 1)
    assert nbytes >= 2 * 4 * H * Dk * Dv * (L // (max(lengths) // 2) + len(lengths))


@pytest.mark.parametrize("kind", ALL)
@pytest.mark.parametrize("H,Hk,Dk,Dv", [(2, 2, 64, 64), (2, 1, 128, 128), (4, 2, 40, 72), (3, 1, 72, 104)])
@pytest.mark.parametrize("lengths,behind", [([2100], 0), ([33, 0, 1290, 1, 777, 129], 6), ([255, 1024, 3, 1025, 1], 1)])
def test_gradients(ops, kind, H, Hk, Dk, Dv, lengths, behind):  # noqa: F811
    L, S = sum(lengths) + behind, len(lengths)
    assert_cut(lengths, L, H, Dk, Dv, kind)
    cu = torch.tensor(np.cumsum([0] + lengths), dtype=torch.int32, device="cuda")
    q, k, v = fused((L,), H, Hk, Dk, Dv, kind, 1)
    s = lambda seed: make((S, H, Dk, Dv), "float32", seed)  # noqa: E731
    check(ops, q, k, v, decays(H), s(2), cu, kind, True, None, make((L, H, Dv), kind, 3), s(4))


@pytest.mark.parametrize("kind", ALL)
def test_gradients_one_by_one(ops, kind):  # noqa: F811
    """Each gradient alone takes the first passes and joins that it needs: the same bits as together."""
    lengths, (H, Hk, Dk, Dv) = [40, 1500, 600], (2, 1, 64, 32)
    L = sum(lengths)
    assert_cut(lengths, L, H, Dk, Dv, kind)
    cu = torch.tensor(np.cumsum([0] + lengths), dtype=torch.int32, device="cuda")
    leaves = [t.detach().requires_grad_(True) for t in (*fused((L,), H, Hk, Dk, Dv, kind, 1), make((3, H, Dk, Dv), "float32", 2))]
    do, ds = make((L, H, Dv), kind, 3), make((3, H, Dk, Dv), "float32", 4)

    def grads(which):
        out = ops.linear_attention(*leaves[:3], decays(H), s0=leaves[3], cu_seqlens=cu)
        return torch.autograd.grad(out, [leaves[i] for i in which], (do, ds))

    whole = grads(range(4))
    for which in ((0,), (1,), (2,), (3,), (0, 2), (1, 3)):
        assert all(torch.equal(g, whole[i]) for i, g in zip(which, grads(which)))


@pytest.mark.parametrize("kind", ALL)
def test_neighbours_and_rows_behind_do_not_matter(ops, kind):  # noqa: F811
    """A cut sequence between others whose rows are NaN, and NaN behind the last: its results are those that it has alone."""
    H, D, (a, b), L = 2, 64, (300, 1813), 2200
    q, k, v = fused((L,), H, 1, D, D, kind, 1)
    do, s0, ds = make((L, H, D), kind, 3), make((3, H, D, D), "float32", 2), make((3, H, D, D), "float32", 4)
    cu = torch.tensor([0, a, b, L - 3], dtype=torch.int32, device="cuda")

    def run():
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v, s0)]
        o, s = ops.linear_attention(*leaves[:3], decays(H), s0=leaves[3], cu_seqlens=cu)
        return [o.detach(), s.detach(), *torch.autograd.grad((o, s), leaves, (do, ds))]

    want = run()
    for t in (q, k, v, do):
        t[:a], t[b:] = float("nan"), float("nan")
    got = run()
    for i, (x, y) in enumerate(zip(got, want)):
        rows = slice(1, 2) if i in (1, 5) else slice(a, b)
        assert torch.equal(x[rows], y[rows]) and torch.isfinite(x[rows]).all()
        if i not in (1, 5):
            assert (x[L - 3:] == 0).all()
