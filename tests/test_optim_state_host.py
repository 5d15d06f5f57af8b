"""The 8-bit optimizer's checkpoints without a GPU."""
import pytest
import torch


@pytest.mark.parametrize("source", ["torch", "ours"])
def test_a_loaded_count_is_a_copy(source):
    """Stepping the optimizer that a state came from does not move the one that loaded it."""
    from mpnn_amd.optim import AdamW

    new = lambda: [torch.nn.Parameter(torch.ones(5000)), torch.nn.Parameter(torch.ones(10))]   # noqa: E731
    ps = new()
    ref = torch.optim.AdamW(ps)
    for p in ps:
        p.grad = torch.ones_like(p)
    ref.step()
    if source == "ours":                       # the class with 32-bit moments counts as torch does, in place
        first = AdamW(new())
        first.load_state_dict(ref.state_dict())
        steps = [st["step"] for st in first.state.values()]
        opt = AdamW(new(), state_bits=8)
        opt.load_state_dict(first.state_dict())
    else:
        steps = [st["step"] for st in ref.state.values()]
        opt = AdamW(new(), state_bits=8)
        opt.load_state_dict(ref.state_dict())
    for s in steps:
        s += 2
    assert [float(st["step"]) for st in opt.state.values()] == [1.0, 1.0]
    assert [st["exp_avg"].dtype for st in opt.state.values()] == [torch.float8_e4m3fn, torch.float32]
    list(opt.state.values())[0]["step"].zero_()
    assert [float(st["step"]) for st in opt.state.values()] == [0.0, 1.0] and float(steps[0]) == 3.0
