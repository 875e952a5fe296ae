"""Borders of packed sequences that reach outside the rows, or fall: what the scan reads and writes stays inside its buffers,
and borders outside mean the nearest row."""
import ctypes
import random

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
GUARD = 256  # bytes on either side of a buffer
MARK = 0xA5


class Guarded:
    """A buffer between two strips of bytes that nothing may change."""

    def __init__(self, size):
        self.size = size
        self.all = torch.full((GUARD + (size + 255) // 256 * 256 + GUARD,), MARK, dtype=torch.uint8, device="cuda")

    @property
    def ptr(self):
        return ctypes.c_void_p(self.all.data_ptr() + GUARD)

    def put(self, t):
        raw = t.contiguous().view(-1).view(torch.uint8)
        assert raw.numel() == self.size
        self.all[GUARD:GUARD + self.size] = raw
        return self

    def get(self, dtype):
        return self.all[GUARD:GUARD + self.size].clone().view(dtype)

    def intact(self):
        return bool((self.all[:GUARD] == MARK).all()) and bool((self.all[GUARD + self.size:] == MARK).all())


def scan(lib, f, x, gate, cu, h0, dy, dh):
    """Both passes of a packed batch over guarded buffers: (outputs by name, whether every guard stands)."""
    L, C = f.shape
    S, code = cu.numel() - 1, 2 if f.dtype == torch.float16 else 1
    n, s = L * C * 2, S * C * 4
    inputs = {k: Guarded(v.numel() * v.element_size()).put(v) for k, v in
              dict(f=f, x=x, gate=gate, cu=cu, h0=h0, dy=dy, dh=dh).items()}
    out = {k: Guarded(v) for k, v in dict(y=n, h=s, marks=4 * lib.csn_gated_scan_marks(S, L, C, 1), df=n, dx=n, dgate=n, dh0=s).items()}
    strides = (ctypes.c_int64 * 8)(0, C, 0, C, 0, C, 0, C)
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    i, o = (lambda k: inputs[k].ptr), (lambda k: out[k].ptr)
    room = [lib.csn_gated_scan_workspace_bytes(S, L, C, 1, code, b) for b in (0, 1)]
    work = [Guarded(r) for r in room]
    assert lib.csn_gated_scan_fwd(i("f"), i("x"), i("gate"), strides, i("h0"), i("cu"), o("y"), o("h"), o("marks"), S, L, C, code,
                                  work[0].ptr, room[0], stream) == 0
    assert lib.csn_gated_scan_bwd(i("f"), i("x"), i("gate"), i("dy"), strides, i("cu"), o("marks"), i("dh"), o("df"), o("dx"),
                                  o("dgate"), o("dh0"), S, L, C, code, work[1].ptr, room[1], stream) == 0
    torch.cuda.synchronize()
    stand = all(b.intact() for b in (*inputs.values(), *out.values(), *work))
    return {k: b.get(torch.float32 if k in ("h", "dh0") else f.dtype) for k, b in out.items() if k != "marks"}, stand


@pytest.mark.parametrize("seed", range(24))
def test_any_borders(seed):
    from csn_b200 import _lib
    lib = _lib.load()
    rng = random.Random(seed)
    S, L, C = rng.choice([1, 2, 7, 40]), rng.randint(1, 3000), rng.choice([8, 64, 66, 35])
    kind = rng.choice([torch.bfloat16, torch.float16])
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s, d=kind: torch.randn(*s, generator=g).to(d).cuda()  # noqa: E731
    f, x, gate, dy = (rand(L, C) for _ in range(4))
    h0, dh = rand(S, C, d=torch.float32), rand(S, C, d=torch.float32)
    far = rng.choice([50, 1 << 30])
    cu = [rng.randint(-far, L + far) for _ in range(S + 1)]
    rising = torch.tensor(sorted(cu), dtype=torch.int32, device="cuda")
    got, stand = scan(lib, f, x, gate, rising, h0, dy, dh)
    assert stand
    want, _ = scan(lib, f, x, gate, rising.clamp(0, L), h0, dy, dh)
    for k in want:
        assert torch.equal(got[k], want[k]), k
    # rows of no sequence are 0, and no element that should be written is left as it was
    inside = np.zeros(L, bool)
    lo, hi = (int(v) for v in rising.clamp(0, L)[[0, -1]])
    inside[lo:hi] = True
    for k in ("y", "df", "dx", "dgate"):
        rows = got[k].view(L, C)
        assert not rows[torch.tensor(~inside, device="cuda")].any() and torch.isfinite(rows).all(), k
    # falling borders mean nothing, and do no harm
    _, stand = scan(lib, f, x, gate, torch.tensor(cu, dtype=torch.int32, device="cuda"), h0, dy, dh)
    assert stand
