"""optim.AdamW's bookkeeping around its device tables, on the CPU: what captured launches read stays allocated, and addresses that did
not reach a table are sent again.  Tables are stand-ins here; the launches themselves are tested in test_gpu_adamw.py."""
import copy

import numpy as np
import torch

from erfnet_pytorch_amd import optim


def _with_plan(captured):
    """An optimizer of one parameter that has taken 3 steps by a table of its own."""
    p = torch.nn.Parameter(torch.ones(6))
    opt = optim.AdamW([p], lr=1e-2)
    opt.state[p].update(step=torch.zeros(()), exp_avg=torch.zeros(6), exp_avg_sq=torch.zeros(6))
    plan = optim._Plan(p.device, 0)
    plan.params, plan.first_chunk, plan.steps, plan.captured = [p], np.array([0]), torch.tensor([3], dtype=torch.int32), captured
    opt._plans = [[plan]]
    opt._lr = [[1e-2, {p.device: torch.full((1,), 1e-2, dtype=torch.float64)}]]
    opt._copies, opt._copies_captured = {0: (torch.zeros(6), p)}, captured
    return opt, p, plan


def test_loading_keeps_what_captured_launches_read():
    opt, p, plan = _with_plan(True)
    lr, copies, old = opt._lr[0][1][p.device], opt._copies, opt.state[p]["exp_avg"]
    saved = copy.deepcopy(opt.state_dict())
    assert float(saved["state"][0]["step"]) == 3
    saved["state"][0]["exp_avg"].fill_(2.0)
    opt.load_state_dict(saved)
    assert any(k is plan for k in opt._kept) and opt._plans is None
    assert opt._lr[0][1][p.device] is lr and (opt._copies is copies or any(k is copies for k in opt._kept))
    assert torch.equal(opt.state[p]["exp_avg"], torch.full((6,), 2.0)) and opt.state[p]["exp_avg"] is not old
    assert float(opt.state[p]["step"]) == 3


def test_loading_drops_tables_that_no_captured_launch_reads():
    opt, p, plan = _with_plan(False)
    opt.load_state_dict(copy.deepcopy(opt.state_dict()))
    assert opt._kept == [] and opt._plans is None


def test_copies_start_without_tables():
    opt, p, plan = _with_plan(True)
    other = copy.deepcopy(opt)
    q, = other.param_groups[0]["params"]
    assert other._plans is None and other._kept == [] and other._lr == [] and other._copies == {} and opt._plans == [[plan]]
    assert float(other.state[q]["step"]) == 3
