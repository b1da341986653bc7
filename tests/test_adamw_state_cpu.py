"""States that the optimizer refuses, and what is left of its own then."""
import copy

import pytest
import torch

from warpconvnet_b200.optim import AdamW


def parameters():
    return [torch.nn.Parameter(torch.arange(3.0)), torch.nn.Parameter(torch.ones(2, 2))]


def stepped(cls=torch.optim.AdamW, **kw):
    """The state of an optimizer of torch's after a step."""
    params = parameters()
    for p in params:
        p.grad = torch.ones_like(p)
    opt = cls(params, lr=0.5, **kw)
    opt.step()
    return opt.state_dict()


def wrong_size():
    saved = copy.deepcopy(stepped())
    saved["state"][1]["exp_avg"] = torch.zeros(5)
    return saved


def wrong_group():
    saved = copy.deepcopy(stepped())
    saved["param_groups"][0]["params"] = [0]
    del saved["state"][1]
    return saved


def two_groups():
    saved = copy.deepcopy(stepped())
    saved["param_groups"].append({**saved["param_groups"][0], "params": []})
    return saved


@pytest.mark.parametrize("saved", [lambda: stepped(amsgrad=True), wrong_size, wrong_group, two_groups, stepped],
                         ids=["amsgrad", "wrong_size", "wrong_group", "two_groups", "parameters_on_the_host"])
def test_a_refused_state_leaves_everything_as_it_was(saved):
    params = parameters()
    opt = AdamW(params, lr=0.1, betas=(0.5, 0.6))
    kept = {p: {"exp_avg": torch.full_like(p, 7.0)} for p in params}   # (stands for what a step leaves: that needs a device)
    arenas = {p: object() for p in params}
    opt.state.update(kept)
    opt._arena_of.update(arenas)
    before = {k: v for k, v in opt.param_groups[0].items() if k != "params"}
    with pytest.raises(ValueError):
        opt.load_state_dict(saved())
    assert {k: v for k, v in opt.param_groups[0].items() if k != "params"} == before
    assert opt.param_groups[0]["params"] == params and opt._arena_of == arenas
    assert all(opt.state[p] is kept[p] for p in params)


@pytest.mark.parametrize("saved", [lambda: stepped(maximize=True), lambda: stepped(torch.optim.Adam, weight_decay=0.1),
                                   lambda: torch.optim.AdamW(parameters(), maximize=True).state_dict(), lambda: torch.optim.AdamW(parameters(), amsgrad=True).state_dict()],
                         ids=["maximize", "adam", "maximize_before_a_step", "amsgrad_before_a_step"])
def test_states_of_another_rule_are_refused(saved):
    """What would be loaded and then not followed."""
    opt = AdamW(parameters(), lr=0.1)
    with pytest.raises(ValueError, match="maximize|amsgrad|decoupled"):
        opt.load_state_dict(saved())
    assert opt.param_groups[0]["lr"] == 0.1 and "maximize" not in opt.param_groups[0]


def test_groups_of_another_rule_are_refused():
    p, q = parameters()
    for kw in ({"maximize": True}, {"amsgrad": True}, {"decoupled_weight_decay": False}):
        with pytest.raises(ValueError, match="maximize|amsgrad|decoupled"):
            AdamW([{"params": [p], **kw}])
        opt = AdamW([p])
        with pytest.raises(ValueError, match="maximize|amsgrad|decoupled"):
            opt.add_param_group({"params": [q], **kw})
        assert len(opt.param_groups) == 1
    AdamW([{"params": [p], "maximize": False, "amsgrad": False, "fused": True, "decoupled_weight_decay": True}])
    AdamW(parameters()).load_state_dict(torch.optim.AdamW(parameters(), lr=0.5).state_dict())


def test_a_scalers_numbers_go_to_the_device_of_each_parameter(monkeypatch):
    """A GradScaler leaves its scale and its flag on one device; parameters may be on several."""
    seen = []
    monkeypatch.setattr("warpconvnet_b200.optim.adamw.adamw_step",
                        lambda params, grads, *a, grad_scale, found_inf, **kw: seen.append((params[0].device, grad_scale.device, found_inf.device)))
    params = [torch.nn.Parameter(torch.zeros(3)), torch.nn.Parameter(torch.zeros(3, device="meta"))]
    for p in params:
        p.grad = torch.zeros_like(p)
    opt = AdamW(params)
    opt.grad_scale, opt.found_inf = torch.ones(1), torch.zeros(1)
    opt.step()
    assert len(seen) == 2 and all(p == scale == found for p, scale, found in seen)
