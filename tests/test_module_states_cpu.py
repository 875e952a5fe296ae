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


def same_after(m, decay):
    assert m.log_decay.dtype == torch.float32 and torch.equal(m.log_decay.cpu(), decay) and "log_decay" not in m.state_dict()


def test_decays_of_a_module_made_without_memory():
    """Made on the meta device, given memory and then its weights: a state_dict does not hold the decays, so the module has to."""
    plain = LinearAttentionBlock(64, 4)
    decay = plain.mixer.log_decay.clone()
    for move in (lambda m: m.to_empty(device="cpu"), lambda m: m.bfloat16().to_empty(device="cpu"),
                 lambda m: m.to_empty(device="meta").half().to_empty(device="cpu")):
        with torch.device("meta"):
            m = LinearAttentionBlock(64, 4)
        assert m.mixer.log_decay.is_meta
        m = move(m)
        m.load_state_dict(plain.state_dict())
        same_after(m.mixer, decay)


def test_decays_outlive_to_empty_and_moves():
    """Decays that a user has put in place, too."""
    m = LinearAttention(64, 4)
    mine = torch.tensor([-0.5, -0.25, -0.125, -torch.inf])
    m.log_decay.copy_(mine)
    for move in (lambda: m.to_empty(device="cpu"), m.bfloat16, m.double, m.float, m.half, m.share_memory, lambda: m.to("cpu", torch.bfloat16)):
        assert move() is m
        same_after(m, mine)


def test_a_block_inside_a_larger_module():
    with torch.device("meta"):
        m = torch.nn.Sequential(LinearAttentionBlock(64, 4), torch.nn.Linear(64, 8))
    m = m.to_empty(device="cpu").bfloat16()
    same_after(m[0].mixer, LinearAttention(64, 4).log_decay)
