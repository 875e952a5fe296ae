"""What the linear-attention block's operators refuse before they look at a device, their shapes under tracing, and the modules' bookkeeping."""
import ctypes

import pytest
import torch
from torch.autograd import forward_ad

from csn_b200 import ops
from csn_b200.modules import LinearAttention, LinearAttentionBlock

csn = torch.ops.csn
BF, F32 = torch.bfloat16, torch.float32


def t(*shape, d=BF):
    return torch.zeros(*shape, dtype=d)


def dense(B=2, T=5, H=4, Hk=2, Dk=16, Dv=24):
    return {"q": t(B, T, H, Dk), "k": t(B, T, Hk, Dk), "v": t(B, T, Hk, Dv), "log_decay": t(H, d=F32), "s0": t(B, H, Dk, Dv, d=F32)}


def packed(**kw):
    args = {n: v[0] if n in "qkv" else v for n, v in dense(B=3, **kw).items()}
    return {**args, "cu_seqlens": torch.tensor([0, 2, 2, 5], dtype=torch.int32)}


def step():
    return {"q": t(2, 4, 16), "k": t(2, 2, 16), "v": t(2, 2, 24), "log_decay": t(4, d=F32), "s": t(2, 4, 16, 24, d=F32)}


BAD = [("q", lambda v: v.float()), ("k", lambda v: v.half()), ("v", lambda v: v.float()), ("q", lambda v: v[..., :-1]), ("q", lambda v: v.int()),
       ("k", lambda v: v[..., :-1]), ("k", lambda v: v[..., :1, :]), ("v", lambda v: v[..., :1, :]), ("q", lambda v: v[..., :3, :]),
       ("k", lambda v: v[:-1]), ("v", lambda v: v[:-1]), ("q", lambda v: v[0]), ("log_decay", lambda v: v[:-1]),
       ("log_decay", lambda v: v.double()), ("log_decay", lambda v: v.bfloat16()), ("log_decay", lambda v: torch.zeros(8)[::2]),
       ("log_decay", lambda v: v.view(2, 2)), ("q", lambda v: v[..., :0, :])]


@pytest.mark.parametrize("form", [dense, packed, step])
@pytest.mark.parametrize("name,bad", BAD)
def test_shapes_and_types_are_refused(form, name, bad):
    args = form()
    if bad(args[name]).shape == args[name].shape and bad(args[name]).dtype == args[name].dtype and bad(args[name]).is_contiguous():
        pytest.skip("fits")
    call = ops.linear_attention_step if form is step else ops.linear_attention
    with pytest.raises(ValueError):
        call(**{**args, name: bad(args[name])})


@pytest.mark.parametrize("bad", [lambda v: v[:-1], lambda v: v[:, :-1], lambda v: v.int(), lambda v: v.transpose(2, 3), lambda v: v[0]])
def test_states_are_refused(bad):
    with pytest.raises(ValueError):
        ops.linear_attention(**{**dense(), "s0": bad(dense()["s0"])})
    with pytest.raises(ValueError):
        ops.linear_attention_step(**{**step(), "s": bad(step()["s"])})


def test_step_wants_its_state_as_it_is():
    for bad in (t(2, 4, 16, 24), t(4, 2, 16, 24, d=F32).transpose(0, 1), t(2 * 4 * 16 * 24 + 1, d=F32)[1:].view(2, 4, 16, 24)):
        with pytest.raises((ValueError, RuntimeError)):
            ops.linear_attention_step(**{**step(), "s": bad})


@pytest.mark.parametrize("bad", [lambda c: c.long(), lambda c: c[:1], lambda c: c.view(2, 2), lambda c: c[:-1]])
def test_borders_are_refused(bad):
    with pytest.raises(ValueError):
        ops.linear_attention(**{**packed(), "cu_seqlens": bad(packed()["cu_seqlens"])})


@pytest.mark.parametrize("Dk,Dv", [(129, 16), (16, 129), (256, 256)])
def test_wide_heads_are_refused(Dk, Dv):
    with pytest.raises(ValueError, match="1 to 128"):
        ops.linear_attention(**dense(Dk=Dk, Dv=Dv))


def test_trained_decays_are_refused():
    args = dense()
    with pytest.raises(ValueError, match="log_decay"):
        ops.linear_attention(**{**args, "log_decay": args["log_decay"].requires_grad_()})


def test_cpu_tensors_are_refused():
    for call in (lambda: ops.linear_attention(**dense()), lambda: ops.linear_attention(**packed()), lambda: ops.linear_attention_step(**step()),
                 lambda: ops.layer_norm(t(3, 8), t(8), t(8))):
        with pytest.raises(RuntimeError, match="CUDA tensors"):
            call()


@pytest.mark.parametrize("name", ["q", "k", "v", "s0"])
def test_forward_mode_is_refused(name):
    args = dense()
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        ops.linear_attention(**{**args, name: forward_ad.make_dual(args[name], torch.ones_like(args[name]))})


@pytest.mark.parametrize("x,w,b", [(t(3, 8), t(7), t(8)), (t(3, 8), t(8), t(1)), (t(3, 8), t(8, 1), t(8)), (t(3, 0), t(0), t(0)),
                                   (t(3, 8), t(8).int(), t(8)), (t(3, 8), None, t(8)), (t(3, 8), t(8), None), (torch.tensor(0.0, dtype=BF), t(1), t(1))])
def test_layer_norm_refuses(x, w, b):
    with pytest.raises(ValueError):
        ops.layer_norm(x, w, b)


def test_shapes_under_tracing():
    m = lambda args: {n: None if v is None else v.to("meta") for n, v in args.items()}  # noqa: E731
    a = m(dense())
    o, s = csn.linear_attention_fwd(a["q"], a["k"], a["v"], a["log_decay"], a["s0"], None, None)
    assert o.shape == (2, 5, 4, 24) and o.dtype == BF and s.shape == (2, 4, 16, 24) and s.dtype == F32
    grads = csn.linear_attention_bwd(a["q"], a["k"], a["v"], a["log_decay"], a["s0"], None, o, s, 0.5)
    assert [g.shape for g in grads] == [a[n].shape for n in ("q", "k", "v", "s0")]
    a = m(packed())
    o, s = csn.linear_attention_fwd(a["q"], a["k"], a["v"], a["log_decay"], None, a["cu_seqlens"], None)
    assert o.shape == (5, 4, 24) and s.shape == (3, 4, 16, 24)


@pytest.mark.parametrize("name,bad", [("do", lambda v: v[:-1]), ("do", lambda v: v[..., :-1]), ("do", lambda v: v.float()), ("ds_last", lambda v: v[:-1]),
                                      ("ds_last", lambda v: v.int()), ("q", lambda v: v[:-1]), ("s0", lambda v: v[:-1])])
def test_registered_backward_refuses(name, bad):
    args = {**dense(), "cu_seqlens": None, "do": t(2, 5, 4, 24), "ds_last": t(2, 4, 16, 24, d=F32), "scale": 0.5}
    with pytest.raises(ValueError):
        csn.linear_attention_bwd(*{**args, name: bad(args[name])}.values())


# ------------------------------------------------------------------------ the C ABI
@pytest.fixture(scope="module")
def lib():
    from csn_b200 import _build, _lib
    _build.build()
    return _lib.load()


null = ctypes.c_void_p(0)


def test_c_entries_refuse(lib):
    def fwd(S=1, T=4, H=2, Hk=1, Dk=8, Dv=8, dtype=1):
        return lib.csn_linear_attention_fwd(null, null, null, None, null, null, null, null, null, S, T, H, Hk, Dk, Dv, 1.0, dtype, null, 0, null)

    assert fwd() == 1 and b"missing" in lib.csn_last_error()
    assert fwd(S=-1) == 1 and b"negative" in lib.csn_last_error()
    assert fwd(H=3, Hk=2) == 1 and b"divide" in lib.csn_last_error()
    assert fwd(Dk=129) == 2 and fwd(Dv=0) == 2 and fwd(dtype=3) == 2
    assert fwd(S=0) == 0  # an empty problem is a no-op
    assert lib.csn_linear_attention_step(null, null, null, None, null, null, null, 2, 2, 1, 8, 8, 1.0, 0, null) == 1
    assert lib.csn_linear_attention_bwd(*[null] * 4, None, *[null] * 8, 1, 4, 2, 1, 8, 8, 1.0, 0, null, 0, null) == 1
    assert lib.csn_layer_norm_rows_fwd(null, 8, null, null, null, null, null, 2, 8, 1e-5, 1, 1, null) == 1
    assert lib.csn_layer_norm_rows_fwd(null, 8, null, null, null, null, null, 2, 8, 1e-5, 0, 0, null) == 2  # float32 rows are csn_layer_norm_fwd's
    assert lib.csn_layer_norm_rows_fwd(null, 8, null, null, null, null, null, 2, 8, 1e-5, 1, 2, null) == 2
    assert lib.csn_layer_norm_rows_fwd(null, 8, null, null, null, null, null, 0, 8, 1e-5, 1, 1, null) == 0
    assert lib.csn_layer_norm_rows_bwd(null, 8, null, 8, null, null, null, null, null, null, 2, 8, 1, 1, null, 0, null) == 1


def test_step_refuses_shared_memory(lib):
    """Found by the addresses alone: nothing is launched."""
    s = (ctypes.c_float * (2 * 2 * 8 * 8 + 64))()
    base = (ctypes.addressof(s) + 15) // 16 * 16
    st = (ctypes.c_int64 * 6)(16, 8, 16, 8, 16, 8)
    far, n = base + (1 << 30), 2 * 2 * 8 * 8 * 4

    def call(q=far, k=far + 4096, v=far + 8192, o=far + 12288, decay=far + 16384):
        return lib.csn_linear_attention_step(*(ctypes.c_void_p(p) for p in (q, k, v)), st, ctypes.c_void_p(decay), ctypes.c_void_p(base),
                                             ctypes.c_void_p(o), 2, 2, 2, 8, 8, 1.0, 0, null)

    for bad in ({"q": base}, {"k": base + n - 16}, {"v": base - 64}, {"o": base + 16}, {"decay": base + 32}):
        assert call(**bad) == 1 and b"shares memory" in lib.csn_last_error()


def test_workspace_is_a_function_of_the_sizes(lib):
    w = lib.csn_linear_attention_workspace_bytes
    assert w(8, 4096, 16, 16, 128, 128, 0, 1, 0, 0) == 0  # enough heads: nothing is cut
    assert w(1, 65536, 8, 8, 128, 128, 0, 1, 0, 0) > 0 and w(1, 65536, 8, 8, 128, 128, 0, 1, 0, 1) > 0
    assert w(2, 64, 4, 2, 16, 16, 0, 1, 0, 1) >= 2 * 64 * 4 * 32 * 4  # gradients of shared heads, before they are added up
    assert w(2, 64, 4, 2, 15, 16, 0, 1, 1, 0) >= 2 * 64 * 4 * 16 * 2  # a copy of q in rows of 16
    assert w(2, 64, 4, 2, 15, 16, 0, 0, 15, 0) == 0  # float32 operands are read where they lie
    assert w(-1, 4, 1, 1, 8, 8, 0, 1, 0, 0) == 0


def test_which_operands_are_copied(lib):
    def copies(strides, q=64, do=None, dtype=1, S=2, T=8, packed=0):
        p = [ctypes.c_void_p(a) for a in (q, 64, 64)] + [ctypes.c_void_p(do) if do else null]
        return lib.csn_linear_attention_copies(*p, (ctypes.c_int64 * 12)(*strides), S, T, 4, 2, 16, 16, packed, dtype)

    fits = [512, 64, 16] + [256, 32, 16] * 2 + [512, 64, 16]
    assert copies(fits) == 0 and copies(fits, do=64) == 0
    assert copies(fits, q=66) == 1 and copies(fits, do=72) == 8
    assert copies([512, 64, 12] + fits[3:]) == 1 and copies(fits[:3] + [256, 32, 0] + fits[6:]) == 2 and copies(fits[:6] + [250, 32, 16] + fits[9:]) == 4
    assert copies(fits[:6] + [250, 32, 16] + fits[9:], packed=1) == 0  # packed rows have no sequence stride
    assert copies([1] * 12, dtype=0) == 0 and copies([1] * 12, T=0) == 0


# -------------------------------------------------------------------------- modules
def test_modules_keep_their_decays():
    m = LinearAttention(64, 4, num_kv_heads=2)
    decay = m.log_decay.clone()
    m.bfloat16()
    assert m.log_decay.dtype == F32 and torch.equal(m.log_decay, decay) and m.in_proj.weight.dtype == BF
    assert "log_decay" not in m.state_dict() and m.init_state(3).shape == (3, 4, 16, 16)
    b = LinearAttentionBlock(64, 4).half()
    assert b.mixer.log_decay.dtype == F32
    assert LinearAttention(64, 4).to(torch.float16).to("meta").log_decay.device.type == "meta"


def test_layer_norm_module_off_the_gpu():
    """What went to the library's layer norm on the CPU still does."""
    from csn_b200.modules import LayerNorm
    m = LayerNorm(6).bfloat16()
    x = torch.randn(3, 6).bfloat16()
    assert torch.equal(m(x), torch.nn.functional.layer_norm(x, (6,), m.weight, m.bias, m.eps))


@pytest.mark.parametrize("kw", [{"num_heads": 4, "num_kv_heads": 3}, {"num_heads": 0}, {"num_heads": 1, "head_dim": 129}, {"num_heads": 4, "num_kv_heads": 0}])
def test_modules_refuse(kw):
    with pytest.raises((ValueError, ZeroDivisionError)):
        LinearAttention(64, **kw)


# ------------------------------------------------------- the 64-bit forms that the kernels are held against
def differences(value, leaves, grads):
    """Central differences along one direction for each input, against the inner product of its gradient."""
    for i, x in enumerate(leaves):
        way, e = torch.randn(x.shape, dtype=torch.float64, generator=torch.Generator().manual_seed(i)), 1e-5
        ends = [value(*[u + s * e * way if j == i else u for j, u in enumerate(leaves)]) for s in (1.0, -1.0)]
        want, got = (ends[0] - ends[1]) / (2 * e), (grads[i] * way).sum()
        # the third-order term is e^2 of values of a few units, the rounding of the ends 1e-16 / e of theirs
        assert abs(want - got) <= 1e-7 * (1.0 + abs(want) + ends[0].abs())


def test_oracles_gradients_are_differences():
    import linear_attention_oracle as orc
    r = lambda *s: torch.randn(*s, dtype=torch.float64, generator=torch.Generator().manual_seed(sum(s)))  # noqa: E731
    L, H, Hk, Dk, Dv, borders = 11, 4, 2, 5, 3, [(0, 4), (4, 4), (4, 10)]
    g, do, ds = -r(H).abs(), r(L, H, Dv), r(3, H, Dk, Dv)
    ins = [r(L, H, Dk), r(L, Hk, Dk), r(L, Hk, Dv), r(3, H, Dk, Dv)]

    def attention(q, k, v, s0):
        out = orc.attention(q, k, v, g, s0, borders, 0.3)
        return (out["o"][0] * do).sum() + (out["s"][0] * ds).sum()

    got = orc.attention(*ins[:3], g, ins[3], borders, 0.3, do, ds)
    differences(attention, ins, [got[n][0] for n in ("dq", "dk", "dv", "ds0")])
    dy, ins = r(6, 9), [r(6, 9) + 2.0, r(9), r(1, 9)[0]]
    got = orc.layer_norm(*ins, 1e-3, dy)
    differences(lambda x, w, b: (orc.layer_norm(x, w, b, 1e-3)["y"][0] * dy).sum(), ins, [got[n][0] for n in ("dx", "dw", "db")])
