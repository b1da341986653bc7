"""What the optimizer refuses before it needs a device."""
import pytest
import torch

from warpconvnet_b200.optim import AdamW, moment_slots


@pytest.mark.parametrize("kw", [{"lr": -1.0}, {"betas": (1.0, 0.9)}, {"betas": (0.9, -0.1)}, {"eps": -1e-8}, {"weight_decay": -0.1}, {"state_bits": 16},
                                {"lr": torch.ones(2)}])
def test_arguments(kw):
    with pytest.raises(ValueError):
        AdamW([torch.nn.Parameter(torch.zeros(3))], **kw)


def test_groups_have_moments_of_one_kind():
    opt = AdamW([torch.nn.Parameter(torch.zeros(3))], state_bits=8)
    with pytest.raises(ValueError):
        opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(3))], "state_bits": 32})
    assert len(opt.param_groups) == 1


def test_parameters_on_the_host_are_refused():
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.zeros(3)
    with pytest.raises(ValueError):
        AdamW([p]).step()


def test_slots_are_whole_blocks():
    assert moment_slots([1, 256, 257, 0, 5]) == ([0, 256, 512, 1024, 1024], 1280)
