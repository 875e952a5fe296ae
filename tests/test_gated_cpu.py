"""The gated recurrent block's entry points without a GPU: sizes of their buffers, and what the C ABI
refuses before it touches a device."""
import ctypes

import pytest

NULL = ctypes.c_void_p(0)


@pytest.fixture(scope="module")
def lib():
    from csn_b200 import _build, _lib
    _build.build()
    return _lib.load()


def strides(*v):
    return (ctypes.c_int64 * 8)(*v)


def fake(offset=0):
    """A pointer that is looked at, never followed."""
    return ctypes.c_void_p(4096 + offset)


def refused(lib, rc, code, text):
    assert rc == code and text in lib.csn_last_error().decode()


@pytest.mark.parametrize("packed,S,T", [(0, 1, 1), (0, 3, 64), (0, 5, 129), (1, 4, 1000), (1, 100, 7)])
def test_marks_hold_every_pass_of_every_sequence(lib, packed, S, T):
    """Sequence s keeps its states from row0 // 64 + s on: rooms do not overlap and end inside."""
    import random
    rng = random.Random(S * T)
    C = 3
    have = lib.csn_gated_scan_marks(S, T, C, packed)
    assert have % C == 0
    for _ in range(50):
        if packed:
            cu = sorted(rng.randint(0, T) for _ in range(S + 1))
        else:
            cu = [s * T for s in range(S + 1)]
        end = 0
        for s in range(S):
            first = cu[s] // 64 + s
            assert first >= end
            end = first + -(-(cu[s + 1] - cu[s]) // 64)
            assert end * C <= have


@pytest.mark.parametrize("seed", range(6))
def test_any_borders_stay_inside(lib, seed):
    """The scan's arithmetic for a packed batch (which sequence and chunk a unit works on, its marks and its
    neighbours' maps), written out: every row, mark and map is inside its buffer for rising borders and,
    though the results mean nothing then, for any others."""
    import random
    rng = random.Random(seed)
    for _ in range(60):
        S, T, C = rng.randint(1, 40), rng.randint(1, 3000), rng.choice([8, 64, 771])
        cu = [rng.randint(-50, T + 50) for _ in range(S + 1)]
        rising = rng.random() < 0.5
        if rising:
            cu = sorted(min(max(v, 0), T) for v in cu)
        need = lib.csn_gated_scan_workspace_bytes(S, T, C, 1, 1, 0) // (C * 8)
        units = need if need else S
        # the chunk that this size has: units = T // chunk + S
        for chunk in ([c for c in range(256, T + 64, 64) if T // c + S == units][:1] if need else [-(-T // 64) * 64]):
            cut = [min(max(v, 0), T) for v in cu]
            base = [cut[i] // chunk + i for i in range(S)]
            done = [0] * T
            for u in range(T // chunk + S):
                s = max((i for i in range(S) if base[i] <= u), default=-1) if rising else rng.choice(
                    [i for i in range(S) if base[i] <= u] or [-1])
                if s < 0:
                    continue
                row0, length = cut[s], max(cut[s + 1], cut[s]) - cut[s]
                k = u - base[s]
                assert k >= 0
                first, past = min(k * chunk, length), min(k * chunk + chunk, length)
                if k > 0 and first >= length:
                    continue
                assert 0 <= row0 + first <= row0 + past <= T
                for t in range(first, past):
                    done[row0 + t] += 1
                if past > first:
                    assert row0 // 64 + s + (past - 1) // 64 < lib.csn_gated_scan_marks(S, T, C, 1) // C
                    assert 0 <= u - k and u + (length - 1) // chunk - k < T // chunk + S
            if rising:
                assert all(n == (cut[0] <= t < cut[-1]) for t, n in enumerate(done))


def test_marks_of_nothing(lib):
    assert lib.csn_gated_scan_marks(0, 5, 8, 0) == 0 and lib.csn_gated_scan_marks(5, 5, 0, 0) == 0


def test_scan_refuses(lib):
    p, st = fake(), strides()

    def fwd(f=p, x=p, g=NULL, s=st, h0=NULL, cu=NULL, y=p, S=2, T=4, C=8, dtype=1):
        return lib.csn_gated_scan_fwd(f, x, g, s, h0, cu, y, NULL, NULL, S, T, C, dtype, NULL, 0, NULL)

    refused(lib, fwd(S=-1), 1, "S, T, C >= 0")
    refused(lib, fwd(T=-1), 1, "S, T, C >= 0")
    refused(lib, fwd(dtype=3), 2, "dtype")
    refused(lib, fwd(S=2 ** 31, C=64), 1, "tiles")
    refused(lib, fwd(f=NULL), 1, "required")
    refused(lib, fwd(y=NULL), 1, "required")
    refused(lib, fwd(s=None), 1, "required")
    refused(lib, fwd(x=fake(1)), 1, "aligned")
    refused(lib, fwd(h0=fake(8)), 1, "aligned")
    refused(lib, fwd(y=fake(2)), 1, "aligned")
    assert fwd(S=0) == 0 and fwd(C=0) == 0

    def bwd(marks=p, dy=p, df=p, dh0=NULL, T=4):
        return lib.csn_gated_scan_bwd(p, p, NULL, dy, st, NULL, marks, NULL, df, p, NULL, dh0, 2, T, 8, 1, NULL, 0, NULL)

    refused(lib, bwd(marks=NULL), 1, "required")
    refused(lib, bwd(dy=NULL), 1, "required")
    refused(lib, bwd(df=NULL), 1, "required")
    refused(lib, bwd(marks=fake(4)), 1, "aligned")
    refused(lib, bwd(dy=fake(1)), 1, "aligned")
    refused(lib, bwd(df=fake(2)), 1, "aligned")
    refused(lib, bwd(dh0=fake(4)), 1, "aligned")


def test_long_scans_need_their_workspace(lib):
    p, st = fake(), strides()
    need = lib.csn_gated_scan_workspace_bytes(1, 65536, 64, 0, 1, 0)
    assert need > 0 and need % (64 * 8) == 0
    rc = lib.csn_gated_scan_fwd(p, p, NULL, st, NULL, NULL, p, NULL, NULL, 1, 65536, 64, 1, p, need - 1, NULL)
    refused(lib, rc, 1, "workspace")
    assert lib.csn_gated_scan_workspace_bytes(256, 4096, 4096, 0, 1, 0) == 0
    # a packed batch has room for the chunks of every sequence, whatever their lengths
    for S, T, C in ((1, 5000, 64), (37, 20011, 771), (400, 900, 64), (3, 1 << 20, 128)):
        for backward in (0, 1):
            units = lib.csn_gated_scan_workspace_bytes(S, T, C, 1, 1, backward) // (C * 8)
            assert units == 0 or units >= S + 1
    assert lib.csn_gated_scan_workspace_bytes(1, 65536, 64, 0, 9, 0) == 0


def test_step_refuses(lib):
    p, st = fake(), strides()
    step = lambda f=p, h=p, y=p, B=2, C=8, dtype=1: lib.csn_gated_step(f, p, NULL, st, h, y, B, C, dtype, NULL)  # noqa: E731
    refused(lib, step(B=-1), 1, "negative")
    refused(lib, step(dtype=-1), 2, "dtype")
    refused(lib, step(h=NULL), 1, "missing")
    refused(lib, step(h=fake(4)), 1, "misaligned")
    refused(lib, step(f=fake(1)), 1, "misaligned")
    # a state that shares memory with what the step reads beside it (the first row, the last) or with its result
    refused(lib, step(f=fake(1 << 20), h=p, y=fake(2 << 20)), 1, "shares memory")
    refused(lib, lib.csn_gated_step(fake(1 << 20), p, NULL, (ctypes.c_int64 * 3)(64, 8, 0), fake((1 << 20) + 128), fake(2 << 20),
                                    2, 8, 1, NULL), 1, "shares memory")
    refused(lib, step(f=fake(1 << 20), h=fake(2 << 20), y=fake(2 << 20)), 1, "shares memory")
    assert step(B=0) == 0


def test_ffn_refuses(lib):
    p = fake()

    def fwd(x=p, y=p, R=4, C=8, F=8, ldx=8, dtype=1, ws=NULL, nb=0, pre=NULL):
        return lib.csn_silu_gated_linear_fwd(x, ldx, p, C, p, C, y, pre, R, C, F, dtype, ws, nb, NULL)

    refused(lib, fwd(R=-1), 1, "R, C, F")
    refused(lib, fwd(F=2 ** 22), 1, "R, C, F")
    refused(lib, fwd(dtype=0), 2, "dtype")
    refused(lib, fwd(x=NULL), 1, "required")
    refused(lib, fwd(x=fake(1)), 1, "aligned")
    refused(lib, fwd(y=fake(2)), 1, "misaligned")
    refused(lib, fwd(pre=fake(8)), 1, "misaligned")
    for odd in (dict(x=fake(8)), dict(ldx=12), dict(ldx=0), dict(C=9, ldx=16), dict(R=2, ldx=-8)):
        refused(lib, fwd(**odd), 1, "workspace")  # a copy is needed, and there is no room for it
    assert fwd(R=0) == 0 and fwd(F=0) == 0

    def bwd(dy=p, dx=p, R=4, C=8, F=8, ws=p, nb=1 << 30):
        return lib.csn_silu_gated_linear_bwd(p, C, p, C, p, C, dy, F, NULL, dx, p, p, R, C, F, 1, ws, nb, NULL)

    refused(lib, bwd(dy=NULL), 1, "missing")
    refused(lib, bwd(dx=fake(2)), 1, "misaligned")
    refused(lib, bwd(ws=NULL, nb=0), 1, "workspace")
    refused(lib, bwd(nb=8), 1, "workspace")
    refused(lib, bwd(C=-2), 1, "R, C, F")


def test_ffn_copies_and_their_room(lib):
    copies = lambda x=fake(), ldx=64, ldg=64, ldu=64, R=5, C=64, F=7: lib.csn_silu_gated_linear_copies(  # noqa: E731
        x, ldx, fake(), ldg, fake(), ldu, R, C, F)
    assert copies() == 0 and copies(ldx=72) == 0 and copies(ldx=68) == 1 and copies(x=fake(2)) == 1
    assert copies(ldg=65) == 2 and copies(ldu=0) == 4 and copies(C=63, ldx=63, ldg=63, ldu=63) == 7
    assert copies(R=1, ldx=0) == 0  # the stride of one row says nothing
    room = lib.csn_silu_gated_linear_workspace_bytes
    assert room(5, 64, 7, 0, 0) == 0
    assert room(5, 63, 7, 7, 0) >= (5 + 7 + 7) * 128
    assert room(5, 63, 7, 7, 1) >= room(5, 63, 7, 7, 0) + 2 * 5 * 16
    assert room(0, 64, 7, 7, 1) == 0


def test_dropout_refuses(lib):
    p = fake()
    drop = lambda x=p, rng=p, n=8, cut=100, dtype=0: lib.csn_dropout_add(x, NULL, rng, p, n, cut, dtype, NULL)  # noqa: E731
    refused(lib, drop(n=-1), 1, "n >= 0")
    refused(lib, drop(cut=65537), 1, "cut")
    refused(lib, drop(cut=-1), 1, "cut")
    refused(lib, drop(dtype=7), 2, "dtype")
    refused(lib, drop(x=fake(4)), 1, "misaligned")
    refused(lib, drop(rng=NULL), 1, "missing")
    assert drop(n=0) == 0


@pytest.mark.parametrize("name", ["gated_scan_fwd", "gated_scan_bwd", "gated_step", "silu_gated_linear_fwd",
                                  "silu_gated_linear_bwd", "dropout_add"])
def test_operator_is_registered(name):
    import torch
    import csn_b200.ops  # noqa: F401
    assert getattr(torch.ops.csn, name).default._schema.name == f"csn::{name}"


def test_fake_shapes_on_meta(lib):
    import torch
    import csn_b200.ops  # noqa: F401
    csn = torch.ops.csn
    m = lambda *s, d=torch.bfloat16: torch.empty(*s, device="meta", dtype=d)  # noqa: E731
    for f, cu, S in ((m(3, 70, 8), None, 3), (m(300, 8), m(6, d=torch.int32), 5)):
        y, h, marks = csn.gated_scan_fwd(f, f, None, f, cu)
        assert y.shape == f.shape and y.dtype == f.dtype and h.shape == (S, 8) and h.dtype == torch.float32
        rows = f.shape[0] if cu is not None else f.shape[1]
        assert marks.numel() == lib.csn_gated_scan_marks(S, rows, 8, int(cu is not None))
        df, dx, dh0, dgate = csn.gated_scan_bwd(f, f, None, cu, marks, f, h)
        assert df.shape == dx.shape == f.shape and dh0.shape == (S, 8) and dgate.numel() == 0
    x, w = m(2, 5, 16), m(24, 16)
    assert csn.silu_gated_linear_fwd(x, w, w).shape == (2, 5, 24)
    assert [tuple(t.shape) for t in csn.silu_gated_linear_bwd(x, w, w, m(2, 5, 24))] == [(2, 5, 16), (24, 16), (24, 16)]
    assert csn.dropout_add(x, None, 100, m(2, d=torch.int64)).shape == x.shape
    assert csn.gated_step(m(4, 8), m(4, 8), m(4, 8, d=torch.float32), None).shape == (4, 8)


def test_operators_want_cuda_tensors():
    import torch
    from csn_b200 import modules, ops
    t = torch.zeros(2, 3, 8)
    for call in (lambda: ops.gated_scan(t, t), lambda: ops.gated_step(t[0], t[0], t[0].clone()),
                 lambda: ops.silu_gated_linear(t.bfloat16(), t[0].bfloat16(), t[0].bfloat16()),
                 lambda: ops.dropout_add(t, None, 0.5, torch.zeros(2, dtype=torch.int64))):
        with pytest.raises(RuntimeError, match="CUDA tensors"):
            call()
    with pytest.raises(ValueError):
        modules.DropoutAdd(1.5)


def test_feed_forward_shares_the_gglu_parameters():
    from csn_b200.modules import GatedFeedForward
    from python.clifford_model import GeometricGatedLinearUnit
    a, b = GatedFeedForward(16, 24), GeometricGatedLinearUnit(16, 24)
    assert {k: v.shape for k, v in a.state_dict().items()} == {k: v.shape for k, v in b.state_dict().items()}


def test_dropout_seed_follows_the_generator():
    import torch
    from csn_b200.modules import DropoutAdd
    torch.manual_seed(5)
    drop = DropoutAdd(0.1)
    a, b = drop.numbers("cpu"), drop.numbers("cpu")
    assert a.dtype == torch.int64 and a.shape == (2,) and a[0] != b[0] and a[1] != b[1]
    torch.manual_seed(5)
    assert torch.equal(a, drop.numbers("cpu")) and torch.equal(b, DropoutAdd(0.1).numbers("cpu"))
    assert not drop.state_dict()  # nothing that copies of a layer, or the ranks of a job, would share
