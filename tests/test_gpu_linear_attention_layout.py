"""Partial gradients of shared heads at the places in the workspace where their rows do not fall on 32 bytes by themselves."""
import ctypes

import pytest
import torch

import linear_attention_oracle as orc
from test_gpu_linear_attention import TYPES, check, decays, fused, make, ops  # noqa: F401

pytestmark = pytest.mark.gpu
HALF = ["bfloat16", "float16"]
# rows * H * Dk = 4 mod 8, so that the partial gradients of v end 16 bytes past a multiple of 32 unless room is left
SIZES = [(3, 3, 12, 8), (37, 2, 10, 64), (150, 2, 9, 64), (5, 3, 36, 104)]


@pytest.mark.parametrize("kind", HALF)
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("T,H,Dk,Dv", SIZES)
def test_gradients_of_shared_heads(ops, kind, packed, T, H, Dk, Dv):  # noqa: F811
    lead = (T,) if packed else (1, T)
    cu = torch.tensor([0, T // 3, T], dtype=torch.int32, device="cuda") if packed else None
    S = 2 if packed else 1
    q, k, v = fused(lead, H, 1, Dk, Dv, kind, 1)
    check(ops, q, k, v, decays(H), make((S, H, Dk, Dv), "float32", 2), cu, kind, True, None, make((*lead, H, Dv), kind, 3),
          make((S, H, Dk, Dv), "float32", 4))


@pytest.mark.parametrize("kind", HALF)
@pytest.mark.parametrize("T,H,Dk,Dv", [(37, 2, 16, 64), (150, 3, 24, 40)])
def test_workspace_on_16_bytes(ops, kind, T, H, Dk, Dv):  # noqa: F811
    """A caller of the C ABI may hand over a workspace that lies on 16 bytes and not on 32: the same bits."""
    from csn_b200 import _lib
    q, k, v = (make((1, T, n, d), kind, i) for i, n, d in ((1, H, Dk), (2, 1, Dk), (3, 1, Dv)))
    do, g, code = make((1, T, H, Dv), kind, 4), decays(H), {"bfloat16": 1, "float16": 2}[kind]
    strides = (ctypes.c_int64 * 12)(*(n for t in (q, k, v, do) for n in t.stride()[:3]))
    nbytes = _lib.load().csn_linear_attention_workspace_bytes(1, T, H, 1, Dk, Dv, 0, code, 0, 1)
    ptr = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    results = []
    for off in (0, 16):
        room = torch.full((nbytes + 64,), 0x55, dtype=torch.uint8, device="cuda")
        work = room[off:off + nbytes]
        out = [torch.empty_like(t) for t in (q, k, v)]
        _lib.call("csn_linear_attention_bwd", ptr(q), ptr(k), ptr(v), ptr(do), strides, ptr(g), None, None, None, *(ptr(t) for t in out),
                  None, 1, T, H, 1, Dk, Dv, Dk ** -0.5, code, ptr(work), nbytes, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
        torch.cuda.synchronize()
        assert (room[:off] == 0x55).all() and (room[off + nbytes:] == 0x55).all()
        results.append(out)
    assert all(torch.equal(a, b) for a, b in zip(*results))
    zero = torch.zeros(1, H, Dk, Dv, dtype=torch.float64)
    flat = lambda t: t.double().cpu().flatten(0, 1)  # noqa: E731
    want = orc.attention(flat(q), flat(k), flat(v), g.cpu(), zero, [(0, T)], Dk ** -0.5, flat(do), zero)
    for n, t in zip(("dq", "dk", "dv"), results[1]):
        value, size = want[n]
        bound = orc.steps(T, max(Dk, Dv)) * orc.U * size + 1.01 * orc.HALF_STEP[TYPES[kind]] * size
        if kind == "float16":
            bound = bound + 2.0 ** -24 * 256 * float(size.max())
        assert orc.used(t.cpu().reshape(value.shape), value, bound, TYPES[kind]) <= 1.0
