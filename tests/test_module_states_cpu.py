"""What the recurrent blocks' modules keep in float32, however they are made and moved."""
import pytest
import torch

from csn_b200.modules import GatedRecurrence, GatedRecurrentBlock, LinearAttention, LinearAttentionBlock


@pytest.fixture(params=[torch.bfloat16, torch.float16, torch.float64])
def default(request):
    before = torch.get_default_dtype()
    torch.set_default_dtype(request.param)
    yield request.param
    torch.set_default_dtype(before)


def test_decays_do_not_follow_the_default_type(default):
    want = [-(2.0 ** -(5.0 + 7.0 * i / 3)) for i in range(4)]
    for m in (LinearAttention(64, 4), LinearAttentionBlock(64, 4).mixer):
        assert m.in_proj.weight.dtype == default and m.log_decay.dtype == torch.float32
        # 1 - x has x to half a step of numbers below 1, and log1p(-x) is x and x^2 / 2
        assert all(abs(g - w) <= 0.6 * w * w + 2.0 ** -22 * abs(w) for g, w in zip(m.log_decay.tolist(), want))


def test_states_do_not_follow_the_default_type(default):
    for m in (LinearAttention(64, 4), LinearAttentionBlock(64, 4), GatedRecurrence(64), GatedRecurrentBlock(64)):
        assert m.init_state(3).dtype == torch.float32
