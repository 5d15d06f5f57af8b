"""adamw_step over lists of tensors: what it refuses, and the ways in which long or scattered lists are split."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_tensors_that_share_memory_are_refused():
    from mpnn_amd.optim import adamw_step

    def lists():
        z = lambda n, t=torch.float32: torch.zeros(n, device="cuda").to(t)   # noqa: E731
        e = torch.float8_e4m3fn
        return dict(params=[z(256), z(256)], grads=[z(256), z(256)], exp_avgs=[z(256, e), z(256, e)],
                    exp_avg_sqs=[z(256, e), z(256, e)], exp_avg_scales=[z(4), z(4)], exp_avg_sq_scales=[z(4), z(4)])

    names = list(lists())
    adamw_step(step=1, **lists())
    same = lists()
    same["grads"][1] = same["grads"][0]            # two parameters may have the same gradient
    adamw_step(step=1, **same)
    for name in names:
        if name != "grads":
            bad = lists()
            bad[name][1] = bad[name][0]
            with pytest.raises(ValueError, match="share memory"):
                adamw_step(step=1, **bad)
    for a, b in (("exp_avgs", "exp_avg_sqs"), ("exp_avg_scales", "exp_avg_sq_scales")):
        bad = lists()
        bad[b][1] = bad[a][0]
        with pytest.raises(ValueError, match="share memory"):
            adamw_step(step=1, **bad)
    bad = lists()
    bad["grads"][0] = bad["params"][1]
    with pytest.raises(ValueError, match="gradient shares memory"):
        adamw_step(step=1, **bad)
    bad = lists()                                  # codes in a gradient's bytes, scales in a parameter's
    bad["exp_avgs"][1] = bad["grads"][1].view(torch.float8_e4m3fn)[512:768]
    with pytest.raises(ValueError, match="gradient shares memory"):
        adamw_step(step=1, **bad)
    bad = lists()
    bad["exp_avg_scales"][0] = bad["params"][0][252:]
    with pytest.raises(ValueError, match="share memory"):
        adamw_step(step=1, **bad)
    wide = lists()
    wide.update(exp_avgs=[torch.zeros(256, device="cuda")] * 2, exp_avg_sqs=[torch.zeros(256, device="cuda") for _ in range(2)],
                exp_avg_scales=[None, None], exp_avg_sq_scales=[None, None])
    with pytest.raises(ValueError, match="share memory"):
        adamw_step(step=1, **wide)
