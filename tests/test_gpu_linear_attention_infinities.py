"""How far an infinity or a NaN in one row reaches: the results that depend on it, and in 16 bits the rest of its block of 128 steps,
in that head and sequence.  Everything else keeps its bits, gradients too."""
import pytest
import torch

from test_gpu_linear_attention import ALL, decays, make, ops  # noqa: F401

pytestmark = pytest.mark.gpu
AT = 300  # of blocks 0, 128, 256, 384
# {input: {result: the steps that depend on it}}: `own` the step itself, `on` it and later ones, `back` it and earlier ones
DEPENDS = {"q": {"o": "own", "dk": "back", "dv": "back"}, "k": {"o": "on", "dq": "on", "dv": "own"}, "v": {"o": "on", "dq": "on", "dk": "own"},
           "do": {"dq": "own", "dk": "back", "dv": "back"}}


@pytest.mark.parametrize("kind", ALL)
@pytest.mark.parametrize("name", list(DEPENDS))
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_reach(ops, kind, name, bad):  # noqa: F811
    B, T, H, D = 2, 500, 2, 64
    ins = {n: make((B, T, H, D), kind, i) for i, n in enumerate(("q", "k", "v", "do"))}
    ins["ds"] = make((B, H, D, D), "float32", 5)

    def run(ins):
        leaves = [ins[n].detach().requires_grad_(True) for n in "qkv"]
        s0 = make((B, H, D, D), "float32", 6).requires_grad_(True)
        o, s = ops.linear_attention(*leaves, decays(H), s0=s0)
        grads = torch.autograd.grad((o, s), [*leaves, s0], (ins["do"], ins["ds"]))
        return dict(zip(("o", "s", "dq", "dk", "dv", "ds0"), (o.detach(), s.detach(), *grads)))

    want = run(ins)
    ins[name] = ins[name].clone()
    ins[name][1, AT, 1, 7] = bad
    got = run(ins)
    for n in want:
        assert torch.equal(got[n][0], want[n][0]), n  # the other sequence
    for n in ("o", "dq", "dk", "dv"):
        assert torch.equal(got[n][1, :, 0], want[n][1, :, 0]), n  # the other head
        a, b = got[n][1, :, 1], want[n][1, :, 1]
        reach = DEPENDS[name].get(n)
        first, past = {None: (0, 0), "own": (AT, AT + 1), "on": (AT, T), "back": (0, AT + 1)}[reach]
        if kind != "float32" and reach in ("on", "back"):
            first, past = first // 128 * 128, min(-(-past // 128) * 128, T)
        keep = torch.ones(T, dtype=torch.bool, device="cuda")
        keep[first:past] = False
        assert torch.equal(a[keep], b[keep]), n
        if reach:
            assert not torch.isfinite(a[AT]).all()
    assert torch.equal(got["s"][1, 0], want["s"][1, 0]) and torch.equal(got["ds0"][1, 0], want["ds0"][1, 0])
    if name in "kv":
        assert torch.equal(got["ds0"], want["ds0"]) and not torch.isfinite(got["s"][1, 1]).all()
    else:
        assert torch.equal(got["s"], want["s"]) and not torch.isfinite(got["ds0"][1, 1]).all()
