"""CPU: the policy with a memory cast and moved."""
import copy

import pytest
import torch

from tum_adlr_deep_reinforcement_learning_amd.rollout import RetentionActorCritic


@pytest.mark.parametrize("cast", [lambda p: p.bfloat16(), lambda p: p.half(), lambda p: p.to("cpu", torch.bfloat16),
                                  lambda p: torch.nn.Sequential(p).bfloat16()[0]])
def test_decays_stay_float32(cast):
    p = RetentionActorCritic(14, 3)
    decay = p.log_decay.clone()
    q = cast(p)
    assert q is p and p.embed.weight.dtype in (torch.bfloat16, torch.float16)
    assert torch.equal(p.log_decay, decay) and p.new_memory(2).dtype == torch.float32
    assert "log_decay" in p.state_dict() and not any(n == "log_decay" for n, _ in p.named_parameters())
    assert torch.equal(copy.deepcopy(p).log_decay, decay)
    assert p.float().embed.weight.dtype == torch.float32 and torch.equal(p.log_decay, decay)
    assert RetentionActorCritic(14, 3).double().log_decay.dtype == torch.float64  # (for a restatement in 64 bits)
    assert RetentionActorCritic(14, 3).to("meta").log_decay.is_meta
