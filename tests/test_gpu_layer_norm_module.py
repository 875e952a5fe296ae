"""modules.LayerNorm of 16-bit features whose width is no kernel's in float32: what the library's layer norm does, to the bit, with
the derivatives and types that only it has."""
import pytest
import torch
import torch.nn.functional as F
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("typ", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("C", [6, 1032, 2048])
def test_other_widths(C, typ):
    from csn_b200.modules import LayerNorm
    torch.manual_seed(0)
    m = LayerNorm(C).cuda().to(typ)
    x = torch.randn(4, C, device="cuda").to(typ).requires_grad_(True)
    plain = lambda u: F.layer_norm(u, (C,), m.weight, m.bias, m.eps)  # noqa: E731
    assert torch.equal(m(x), plain(x))
    with torch.autocast("cuda"):
        assert m(x).dtype == plain(x).dtype == torch.float32
    t = torch.randn_like(x)
    with forward_ad.dual_level():
        got, want = (forward_ad.unpack_dual(f(forward_ad.make_dual(x.detach(), t))).tangent for f in (m, plain))
        assert torch.equal(got, want)

    def second(f):
        (g,) = torch.autograd.grad(f(x).square().sum(), x, create_graph=True)
        return torch.autograd.grad(g.square().sum(), x)[0]

    assert torch.equal(second(m), second(plain))
    assert torch.equal(torch.func.vmap(m)(x), torch.func.vmap(plain)(x))


def test_blocks_under_autocast():
    """A block in bfloat16 under autocast gives and trains in its own type, at a width that is no kernel's in float32."""
    from csn_b200.modules import GatedRecurrentBlock, LinearAttentionBlock
    torch.manual_seed(0)
    for blk in (GatedRecurrentBlock(1032, d_inner=64, d_ffn=64), LinearAttentionBlock(1032, 4, head_dim=30, d_ffn=64)):
        blk = blk.cuda().bfloat16()
        x = torch.randn(2, 20, 1032, device="cuda", dtype=torch.bfloat16)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            out, _ = blk(x)
        out.float().square().mean().backward()
        assert out.dtype == torch.bfloat16 and all(torch.isfinite(p.grad).all() for p in blk.parameters())
