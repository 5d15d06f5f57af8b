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


# ---- the ways a list is split ----------------------------------------------------------------------------------
# A launch of the step takes 16 or 120 tensors, one of the norm 16 or 320 that lie within 8 GB, else 128.  Values are compared as
# tests/test_gpu_optim_mixed.py says: codes, scales and 32-bit moments exactly, parameters to the roundings of their update.
def _sizes(n, seed):
    g = torch.Generator().manual_seed(seed)
    return [int(x) for x in torch.randint(1, 400, (n,), generator=g)]


@pytest.mark.parametrize("n", [15, 16, 17, 119, 120, 121, 240, 241, 319, 320, 321, 640, 641, 700])
def test_numbers_of_tensors_around_those_of_a_launch(n):
    from test_gpu_optim_mixed import Tensors, _check_step, _grads

    sizes = _sizes(n, n)
    sizes[n // 2] = 70001                          # one that has several chunks of the norm
    t = Tensors(sizes, n, lambda k: k % 3 > 0)
    for k in (1, 2):
        _check_step(t, _grads(sizes, 100 * n + k), k, seed=n, max_norm=0.3)


@pytest.mark.parametrize("max_norm", [0.0, 0.4])
def test_codes_at_any_byte(max_norm):
    """8-bit moments cut from one buffer: a table holds codes of one residue modulo four, the rounding follows the place in the list."""
    from test_gpu_optim_mixed import Tensors, _check_step, _grads

    sizes = _sizes(40, 3)
    t = Tensors(sizes, 3, lambda k: k % 4 > 0)
    buf, at = torch.zeros(2 * sum(sizes) + 400, device="cuda").to(torch.float8_e4m3fn), 0
    for i, k in enumerate(sizes):
        if t.a[i] is None:
            continue
        for x in (t.m, t.v):
            at += (0, 1, 0, 3, 2, 0, 0, 1)[i % 8]
            x[i] = buf[at:at + k]
            at += k
    for k in (1, 2, 3):
        _check_step(t, _grads(sizes, 60 + k), k, seed=11, max_norm=max_norm)
    assert int((buf.float() != 0).sum()) == sum(int((x.float() != 0).sum()) for x in t.m + t.v if x.dtype == buf.dtype)


@pytest.mark.parametrize("n", [9, 130, 300])
@pytest.mark.parametrize("far", ["grads", "all"])
def test_tensors_more_than_8_gb_apart(n, far):
    """Distances in units of four bytes that 32 bits do not hold: the norm goes by pointers, the step opens another table."""
    from test_gpu_optim_mixed import Tensors, _check_step, _grads

    sizes = _sizes(n, n + 1)
    sizes[1] = 40001
    buf = torch.empty((1 << 31) + (1 << 24), device="cuda")
    end, ends = buf.numel(), {0: 0, 1: buf.numel()}

    def cut(k, i):
        """Places at the buffer's two ends in turn, towards its middle."""
        k += -k % 4
        if i % 2:
            ends[1] -= k
            return ends[1]
        ends[0] += k
        return ends[0] - k

    t = Tensors(sizes, 5, lambda k: k % 3 > 0)
    if far == "all":
        for i, k in enumerate(sizes):
            at = cut(k, i)
            t.p[i] = buf[at:at + k].copy_(t.p[i])
            if t.a[i] is None:
                at = cut(k, i + 1)
                t.m[i] = buf[at:at + k].zero_()
    places = [cut(k, i) for i, k in enumerate(sizes)]
    for k in (1, 2):
        grads = [buf[a:a + s].copy_(g) for a, s, g in zip(places, sizes, _grads(sizes, 200 + k))]
        assert max(g.data_ptr() for g in grads) - min(g.data_ptr() for g in grads) > 1 << 33 and ends[0] < ends[1] <= end
        _check_step(t, grads, k, seed=7, max_norm=0.3)
