"""AdamW(state_bits=8): the optimizer's state as a program meets it between steps."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _optimizer(sizes=(5000, 100, 70000), **kw):
    from mpnn_amd.optim import AdamW

    ps = [torch.nn.Parameter(torch.ones(n, device="cuda")) for n in sizes]
    return AdamW(ps, state_bits=8, **kw), ps


def _step(opt, ps, skip=()):
    for i, p in enumerate(ps):
        p.grad = None if i in skip else torch.full_like(p, 0.1 * (i + 1))
    opt.step()


def _counts(opt, ps):
    return [float(opt.state[p]["step"]) for p in ps]


def test_a_parameter_is_restarted_alone():
    """Writing a parameter's `step` in place is that parameter's affair: its next step is its first again."""
    opt, ps = _optimizer()
    for _ in range(3):
        _step(opt, ps)
    other, qs = _optimizer()
    other.load_state_dict(opt.state_dict())
    with torch.no_grad():
        for p, q in zip(ps, qs):
            q.copy_(p)
    opt.state[ps[0]]["step"].zero_()
    other.state[qs[0]]["step"] = torch.tensor(0.0)      # the same by a tensor of its own
    assert _counts(opt, ps) == [0.0, 3.0, 3.0] == _counts(other, qs)
    for o, xs in ((opt, ps), (other, qs)):
        _step(o, xs)
        assert _counts(o, xs) == [1.0, 4.0, 4.0]
    assert all(torch.equal(p, q) for p, q in zip(ps, qs))
    opt.state[ps[1]]["step"].fill_(10)
    opt.state[ps[2]]["step"] += 5
    _step(opt, ps, skip=(0,))
    assert _counts(opt, ps) == [1.0, 11.0, 10.0]


def test_counts_of_groups_and_of_parameters_that_come_and_go():
    opt, ps = _optimizer()
    _step(opt, ps, skip=(1,))
    new = [torch.nn.Parameter(torch.ones(n, device="cuda")) for n in (4100, 7)]
    opt.add_param_group({"params": new, "lr": 1e-2})
    ps = ps + new
    _step(opt, ps, skip=(0, 4))
    _step(opt, ps)
    assert _counts(opt, ps) == [2.0, 2.0, 3.0, 2.0, 1.0]
    opt.state[ps[2]].clear()                            # a parameter that starts anew
    _step(opt, ps)
    assert _counts(opt, ps) == [3.0, 3.0, 1.0, 3.0, 2.0]
    saved = opt.state_dict()
    assert all(st["step"].numel() == 1 and st["step"].untyped_storage().nbytes() == 4 for st in saved["state"].values())
    _step(opt, ps)
    assert [float(saved["state"][i]["step"]) for i in range(5)] == [3.0, 3.0, 1.0, 3.0, 2.0], "a checkpoint does not go on counting"


def test_a_count_that_two_parameters_share_by_the_callers_hand():
    opt, ps = _optimizer()
    _step(opt, ps)
    opt.state[ps[1]]["step"] = opt.state[ps[2]]["step"]
    _step(opt, ps)
    _step(opt, ps)
    assert _counts(opt, ps) == [3.0, 3.0, 3.0]
