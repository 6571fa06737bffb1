"""optim.AdamW's bookkeeping around its device tables, on the CPU: what captured launches read stays allocated, and addresses that did
not reach a table are sent again.  Tables are stand-ins here; the launches themselves are tested in test_gpu_adamw.py."""
import copy

import numpy as np
import pytest
import torch

from erfnet_pytorch_amd import optim


def _with_plan(captured):
    """An optimizer of one parameter that has taken 3 steps by a table of its own."""
    p = torch.nn.Parameter(torch.ones(6))
    opt = optim.AdamW([p], lr=1e-2)
    opt.state[p].update(step=torch.zeros(()), exp_avg=torch.zeros(6), exp_avg_sq=torch.zeros(6))
    plan = optim._Plan(0, p.device, 0)
    plan.params, plan.first_chunk, plan.steps, plan.captured = [p], np.array([0]), torch.tensor([3], dtype=torch.int32), captured
    plan.counts = [0.0]
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


def test_a_look_that_refuses_a_gradient_notes_none():
    a, b = (torch.nn.Parameter(torch.zeros(3)) for _ in range(2))
    a.grad, b.grad = torch.zeros(3), torch.zeros(3)
    w = optim._host.ParamWatch()
    w.bind([[a, b]])
    assert [w.look([[a, b]]) for _ in range(2)] == [1, 0]
    old, a.grad = (a.grad, b.grad), torch.zeros(3)
    b.grad = torch.sparse_coo_tensor(torch.tensor([[0]]), torch.tensor([1.0]), (3,))
    with pytest.raises(ValueError, match="gradient"):
        w.look([[a, b]])
    b.grad = old[1]
    assert [w.look([[a, b]]) for _ in range(2)] == [1, 0]               # a's is noted now


class _Recorder:
    """The launches of an optimizer, in place of the device: (addresses sent to a table, step launched), in order."""

    def __init__(self, monkeypatch, opt):
        self.sent, self.steps, self.fail_step = [], [], None
        recorder = self

        class Watch:
            def __init__(self):
                self.w = optim._host.ParamWatch()

            def __getattr__(self, name):
                return getattr(self.w, name)

            def set_grads(self, table, which, copies, stream):
                recorder.sent.append(table)
        opt._watch = Watch()

        def call(name, table, chunks, steps, n, lr, *rest):
            assert name == "erf_adamw_step"
            if recorder.fail_step == len(recorder.steps):
                recorder.fail_step = None
                raise RuntimeError("refused")
            recorder.steps.append(table)
        monkeypatch.setattr(optim, "call", call)
        monkeypatch.setattr(optim.ops, "require_gpu", lambda *a: None)
        monkeypatch.setattr(optim.ops, "_stream", lambda: 0)
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
        monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: None, raising=False)                # a CPU device has index None


def _two_groups(monkeypatch):
    a, b = (torch.nn.Parameter(torch.ones(5)) for _ in range(2))
    opt = optim.AdamW([{"params": [a]}, {"params": [b]}])
    a.grad, b.grad = torch.zeros(5), torch.zeros(5)
    return opt, a, b, _Recorder(monkeypatch, opt)


def test_a_refused_launch_leaves_the_later_tables_to_be_filled(monkeypatch):
    opt, a, b, rec = _two_groups(monkeypatch)
    rec.fail_step = 0
    with pytest.raises(RuntimeError, match="refused"):
        opt.step()
    tables = [plans[0].table.data_ptr() for plans in opt._plans]
    assert rec.steps == [] and tables[1] not in rec.sent
    opt.step()
    assert rec.steps == tables and tables[1] in rec.sent
    rec.sent.clear()
    opt.step()
    assert rec.sent == [] and rec.steps == 2 * tables                   # nothing moved
    a.grad = torch.zeros(5)
    rec.fail_step = len(rec.steps)
    with pytest.raises(RuntimeError, match="refused"):
        opt.step()
    opt.step()
    assert tables[0] in rec.sent and tables[1] in rec.sent


def test_a_learning_rate_that_is_refused_leaves_the_tables_to_be_filled(monkeypatch):
    opt, a, b, rec = _two_groups(monkeypatch)
    opt.step()
    rec.sent.clear()
    a.grad = torch.zeros(5)
    opt.param_groups[1]["lr"] = "fast"
    with pytest.raises(ValueError):
        opt.step()
    opt.param_groups[1]["lr"] = 1e-3
    opt.step()
    assert set(rec.sent) == {plans[0].table.data_ptr() for plans in opt._plans}


@pytest.mark.parametrize("key,value", [("betas", (0.9, 1.0)), ("eps", -1.0), ("eps", float("nan")), ("weight_decay", "much")])
def test_settings_that_are_refused_update_no_group(monkeypatch, key, value):
    opt, a, b, rec = _two_groups(monkeypatch)
    good, opt.param_groups[1][key] = opt.param_groups[1][key], value
    for _ in range(2):
        with pytest.raises(ValueError):
            opt.step()
    assert rec.steps == [] and a._version == 0
    opt.param_groups[1][key] = good
    opt.step()
    tables = [plans[0].table.data_ptr() for plans in opt._plans]
    assert rec.steps == tables and set(rec.sent) == set(tables) and a._version == 1


def test_places_for_copies_that_could_not_be_made_are_made_by_the_next_step(monkeypatch):
    p = torch.nn.Parameter(torch.ones(4, 5))
    opt = optim.AdamW([p])
    p.grad = torch.zeros(4, 5)
    rec = _Recorder(monkeypatch, opt)
    opt.step()
    p.grad = torch.zeros(5, 4).t()
    with monkeypatch.context() as m:
        def full(*a, **k):
            raise torch.OutOfMemoryError("full")
        m.setattr(torch, "empty_like", full)
        with pytest.raises(torch.OutOfMemoryError):
            opt.step()
    opt.step()
    plan, = opt._plans[0]
    assert len(opt._copies) == 1 and plan.copies == [opt._copies[0][0].data_ptr()] and rec.sent[-1] == plan.table.data_ptr()


# ------------------------------------------------------------------------------------------------ gradients that come and go
def test_the_watch_tells_gradients_that_come_and_go():
    ps = [torch.nn.Parameter(torch.zeros(3)) for _ in range(4)]
    ps[0].grad, ps[1].grad = torch.zeros(3), torch.zeros(3)
    w = optim._host.ParamWatch()
    w.bind([ps[:2], ps[2:]], [2])                                       # the third is in the tables without a gradient
    assert w.present() == [True, True, False] and [w.look([ps]) for _ in range(2)] == [1, 0]
    old, ps[1].grad = ps[1].grad, None
    assert [w.look([ps]) for _ in range(2)] == [1, 0] and w.present() == [True, False, False]
    before = [p._version for p in ps]
    w.bump()
    assert [p._version - b for p, b in zip(ps, before)] == [1, 0, 0, 0]
    ps[1].grad, ps[2].grad = old, torch.zeros(3)
    assert [w.look([ps]) for _ in range(2)] == [1, 0] and w.present() == [True, True, True]
    ps[2].grad = torch.zeros(6)[::2]
    assert w.look([ps]) == 1 and w.copied() == [2]
    ps[2].grad = None
    assert [w.look([ps]) for _ in range(2)] == [1, 0] and w.copied() == []
    ps[3].grad = torch.zeros(3)
    assert w.look([ps]) == 2


def _three(monkeypatch):
    ps = [torch.nn.Parameter(torch.ones(n)) for n in (5, 9000, 7)]
    opt = optim.AdamW(ps)
    ps[0].grad, ps[1].grad = (torch.zeros_like(p) for p in ps[:2])
    rec = _Recorder(monkeypatch, opt)
    opt.step()
    return opt, ps, rec, opt._plans[0][0]


def test_gradients_that_come_and_go_leave_the_tables_in_place(monkeypatch):
    opt, ps, rec, plan = _three(monkeypatch)
    for gone in ([1], [0, 1], [0], []):
        for i in (0, 1):
            ps[i].grad = None if i in gone else torch.zeros_like(ps[i])
        n = len(rec.steps)
        opt.step()
        assert opt._plans == [[plan]] and len(rec.steps) - n == (len(gone) < 2)


def test_a_first_gradient_beside_a_captured_table_gets_a_table_of_its_own(monkeypatch):
    opt, ps, rec, plan = _three(monkeypatch)
    plan.captured = True
    plan.steps += torch.tensor([1, 4, 4, 4], dtype=torch.int32)         # what launches would count
    ps[0].grad = None
    ps[2].grad = torch.zeros_like(ps[2])
    opt.step()
    assert len(opt._plans[0]) == 2 and opt._plans[0][0] is plan and opt._plans[0][1].params == [ps[2]] and opt._kept == []
    assert plan.steps.tolist() == [1, 4, 4, 4] and rec.steps[-2:] == [q.table.data_ptr() for q in opt._plans[0]]
    assert [float(opt.state_dict()["state"][i]["step"]) for i in range(3)] == [1, 4, 0]
    opt.refresh()                                                       # nothing was replaced: the captured table is taken up again
    opt.step()
    assert plan in opt._plans[0] and plan.steps.tolist() == [1, 4, 4, 4]
    ps[1].data = ps[1].data.clone()                                     # elsewhere now: the captured launch has the old place
    ps[1].grad = torch.zeros_like(ps[1])
    opt.step()
    assert not any(q is plan for q in opt._plans[0]) and any(q is plan for q in opt._kept)
    assert sorted(id(p) for q in opt._plans[0] for p in q.params) == sorted(map(id, ps))


def test_a_first_gradient_without_captured_tables_makes_one_table_of_all(monkeypatch):
    opt, ps, rec, plan = _three(monkeypatch)
    plan.steps += 3
    ps[0].grad = None
    ps[2].grad = torch.zeros_like(ps[2])
    opt.step()
    q, = opt._plans[0]
    assert q.params == ps and q.steps.tolist() == [3, 3, 3, 3, 0] and opt._kept == []


def test_parameters_that_share_memory_take_steps_in_turn(monkeypatch):
    """As long as only one of them has a gradient."""
    t = torch.ones(10)
    a, b = torch.nn.Parameter(t[:6]), torch.nn.Parameter(t[4:])
    opt = optim.AdamW([a, b])
    rec = _Recorder(monkeypatch, opt)
    for p, q in ((a, b), (b, a), (a, b)):
        p.grad, q.grad = torch.zeros(6), None
        opt.step()
        assert [r.params for r in opt._plans[0]] == [[p]]
    b.grad = torch.zeros(6)
    with pytest.raises(ValueError, match="share memory"):
        opt.step()


# ------------------------------------------------------------------------------------------------ state changed by hand
def test_counts_changed_by_hand_are_taken_over(monkeypatch):
    opt, ps, rec, plan = _three(monkeypatch)
    plan.steps += 4
    assert [float(opt.state_dict()["state"][i]["step"]) for i in (0, 1)] == [4, 4]
    opt.state[ps[0]]["step"] = torch.tensor(10.0)
    opt.refresh()
    opt.step()
    q, = opt._plans[0]
    assert q.steps.tolist() == [10, 4, 4, 4]
    opt.state[ps[1]]["step"] = opt.state[ps[1]]["step"].clone()         # moved about, not changed
    q.steps += 1
    assert [float(opt.state_dict()["state"][i]["step"]) for i in (0, 1)] == [11, 5]
    opt.state[ps[1]]["step"].fill_(2.0)
    opt.refresh()
    assert [float(opt.state_dict()["state"][i]["step"]) for i in (0, 1)] == [11, 2]


@pytest.mark.parametrize("captured", [False, True])
def test_state_taken_away_starts_anew(monkeypatch, captured):
    opt, ps, rec, plan = _three(monkeypatch)
    plan.steps += 4
    plan.captured = captured
    del opt.state[ps[0]]
    opt.state[ps[1]] = {}
    opt.refresh()
    opt.step()
    q, = opt._plans[0]
    assert q is not plan and q.steps.tolist() == [0, 0, 0, 0] and opt._kept == ([plan] if captured else [])
    assert set(opt.state[ps[0]]) == {"step", "exp_avg", "exp_avg_sq"}


def test_an_error_between_tables_and_gradients_keeps_captured_tables(monkeypatch):
    opt, ps, rec, plan = _three(monkeypatch)
    plan.captured = True
    opt.refresh()
    looks = opt._watch.w.look

    def look(groups):
        opt._watch.look = looks
        raise KeyboardInterrupt
    opt._watch.look = look
    with pytest.raises(KeyboardInterrupt):
        opt.step()
    assert opt._plans is None and any(k is plan for k in opt._kept)
    opt.step()
    assert opt._plans == [[plan]] and opt._kept == []
