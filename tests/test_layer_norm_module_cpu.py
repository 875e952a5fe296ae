"""Where the modules' layer norms go: traced with CUDA tensors that have no memory, which only the library's layer norm can be."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from csn_b200 import ops
from csn_b200.modules import BlockLayerNorm, GatedRecurrentBlock, LayerNorm, LinearAttention, LinearAttentionBlock

BF = torch.bfloat16


def run(module, C, typ):
    with FakeTensorMode(allow_non_fake_inputs=True):
        x = torch.empty(3, C, dtype=typ, device="cuda")
        w, b = (torch.empty(C, dtype=typ, device="cuda") for _ in range(2))
        m = module(C, device="meta")
        m.weight, m.bias = torch.nn.Parameter(w), torch.nn.Parameter(b)
        return m(x)


@pytest.mark.parametrize("typ", [BF, torch.float16, torch.float32])
@pytest.mark.parametrize("C", [6, 1032, 2048, 8192])
def test_layer_norm_of_other_widths_is_the_librarys(C, typ):
    y = run(LayerNorm, C, typ)
    assert y.shape == (3, C) and y.dtype == typ


@pytest.mark.parametrize("module,C,typ,kernel", [(LayerNorm, 2048, BF, False), (LayerNorm, 6, BF, False), (LayerNorm, 64, BF, True),
                                                 (LayerNorm, 64, torch.float32, True), (BlockLayerNorm, 2048, BF, True),
                                                 (BlockLayerNorm, 6, torch.float16, True), (BlockLayerNorm, 2048, torch.float32, False)])
def test_who_goes_to_the_kernels(monkeypatch, module, C, typ, kernel):
    calls = []
    monkeypatch.setattr(ops, "layer_norm", lambda x, *a: calls.append(a) or x)
    run(module, C, typ)
    assert bool(calls) == kernel


def test_blocks_have_the_wider_norm():
    for m, names in ((GatedRecurrentBlock(64), ("ln_1", "ln_2")), (LinearAttentionBlock(64, 4), ("ln_1", "ln_2")), (LinearAttention(64, 4), ("norm",))):
        for n in names:
            norm = getattr(m, n)
            assert isinstance(norm, BlockLayerNorm) and isinstance(norm, LayerNorm) and list(norm.state_dict()) == ["weight", "bias"]
