"""A state that is refused half way: the optimizer goes on as if nothing had been asked."""
import copy

import pytest
import torch

from warpconvnet_b200.optim import AdamW

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("what", ["size", "names", "missing group"])
def test_training_goes_on_after_a_refused_state(bits, what):
    runs = []
    for refuse in (False, True):
        params = [torch.nn.Parameter(torch.linspace(-1, 1, n, device=DEV)) for n in (300, 700)]
        opt = AdamW(params, lr=1e-2, state_bits=bits)
        for i in range(4):
            for p in params:
                p.grad = torch.full_like(p, 0.1 * (i + 1))
            opt.step()
            if refuse and i == 1:
                saved = copy.deepcopy(opt.state_dict())
                saved["param_groups"][0]["lr"] = 5.0
                if what == "size":
                    saved["state"][1]["exp_avg_sq"] = saved["state"][1]["exp_avg_sq"].new_zeros(1)
                elif what == "names":
                    saved["state"][1]["more"] = torch.zeros(1)
                else:
                    saved["param_groups"] = []
                with pytest.raises(ValueError):
                    opt.load_state_dict(saved)
        runs.append([*params, *(t for p in params for t in opt.state[p].values())])
    assert all(torch.equal(a, b) for a, b in zip(*runs)) and int(opt.state[params[0]]["step"]) == 4
