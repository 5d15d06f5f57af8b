"""AdamW with 8-bit and 32-bit moments (mpnn_adamw_mixed) against its definition in 64 bits (oracle/adamw_oracle.py).

Bounds.  Codes, scales and 32-bit moments are exact: both sides compute the same fp64 operations on the same inputs (clipping
differs in the order of an fp64 sum, 1e-16 relative, against borders between codes that lie 2^-19 apart).
The update is fp32 with one rounding (2^-24 relative) an operation: of p: the factor 1 - lr wd, its product, the difference: 3
in |p|; of the move: m, v (halved by the root), root (its last place twice: the device's square root may be one off), the
factor 1 / sqrt(1 - b2^t), its product, eps, the sum, the quotient, the factor lr / (1 - b1^t), its product, the difference:
at most 12.  |error| <= 2^-24 (3 |p| + 12 |move|)."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
HYPER = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2)


class Tensors:
    """Lists on the device and their copies as float64 arrays."""

    def __init__(self, sizes, seed, wide=lambda n: n >= 64, shift=0):
        g = torch.Generator().manual_seed(seed)
        self.p, self.m, self.v, self.a, self.b = [], [], [], [], []
        for n in sizes:
            self.p.append((torch.randn(n + shift, generator=g) * 0.3).cuda()[shift:])
            if wide(n):
                self.m.append(torch.zeros(n + shift, device="cuda").to(torch.float8_e4m3fn)[shift:])
                self.v.append(torch.zeros(n + shift, device="cuda").to(torch.float8_e4m3fn)[shift:])
                self.a.append(torch.ones(-(-n // 64), device="cuda"))
                self.b.append(torch.ones(-(-n // 64), device="cuda"))
            else:
                self.m.append(torch.zeros(n + shift, device="cuda")[shift:])
                self.v.append(torch.zeros(n + shift, device="cuda")[shift:])
                self.a.append(None)
                self.b.append(None)

    def lists(self):
        return [[None if t is None else t.cpu().float().double().numpy() for t in x] for x in (self.p, self.m, self.v, self.a, self.b)]


def _grads(sizes, seed, shift=0):
    g = torch.Generator().manual_seed(seed)
    out = []
    for n in sizes:
        x = torch.randn(n + shift, generator=g) * 10.0 ** float(torch.randint(-4, 1, (1,), generator=g))
        x = x * torch.exp(2 * torch.randn(n + shift, generator=g)) * (torch.rand(n + shift, generator=g) > 0.1)
        out.append(x.cuda()[shift:])
    return out


def _check_step(t, grads, k, seed=0, max_norm=0.0, hyper=HYPER):
    from mpnn_amd.optim import adamw_step
    from oracle import adamw_oracle as orc

    before = t.lists()
    g64 = [g.cpu().double().numpy() for g in grads]
    want = orc.step(before[0], g64, before[1], before[2], before[3], before[4], k, hyper["lr"], hyper["betas"], hyper["eps"],
                    hyper["weight_decay"], seed, max_norm)
    ss = adamw_step(t.p, grads, t.m, t.v, t.a, t.b, step=k, seed=seed, max_grad_norm=max_norm, **hyper)
    if max_norm > 0:
        total = sum(float((g * g).sum()) for g in g64)
        same = (math.isnan(total) and math.isnan(float(ss))) or float(ss) == total
        assert same or abs(float(ss) - total) <= 2.0**-23 * total
    else:
        assert ss is None
    p, m, v, a, b = t.lists()
    for i, (q, wm, wv, wa, wb, move) in enumerate(want):
        np.testing.assert_array_equal(m[i], wm, err_msg=f"m of tensor {i} ({len(q)})")
        np.testing.assert_array_equal(v[i], wv, err_msg=f"v of tensor {i} ({len(q)})")
        if wa is not None:
            np.testing.assert_array_equal(a[i], wa)
            np.testing.assert_array_equal(b[i], wb)
        fin = np.isfinite(q)
        np.testing.assert_array_equal(np.isnan(q), np.isnan(p[i]))
        err = np.abs(p[i] - q)[fin]
        bound = 2.0**-24 * (3 * np.abs(before[0][i]) + 12 * np.abs(move))[fin] + 1e-45
        assert (err <= bound).all(), (i, float((err / bound).max()))


ODD = [1, 2, 3, 63, 64, 65, 127, 128, 500, 1023, 1024, 1025, 2047, 2048, 2049, 4096, 6151, 30011]


@pytest.mark.parametrize("max_norm", [0.0, 0.7, 1e9])
@pytest.mark.parametrize("shift", [0, 1, 2])
@pytest.mark.parametrize("wide", ["large", "all", "none"])
def test_steps(max_norm, shift, wide):
    t = Tensors(ODD, 1, {"large": lambda n: n >= 1000, "all": lambda n: True, "none": lambda n: False}[wide], shift)
    for k in range(1, 5):
        _check_step(t, _grads(ODD, 10 + k, shift), k, seed=3, max_norm=max_norm)


def test_many_tensors():
    """More tensors than one launch takes (60 of the step, 128 of the norm)."""
    sizes = [int(4000 ** (i / 299)) for i in range(300)]
    t = Tensors(sizes, 2, lambda n: n % 3 > 0)
    for k in (1, 2):
        _check_step(t, _grads(sizes, 20 + k), k, seed=9, max_norm=0.5)


def test_large_tensor_and_hyper_parameters():
    t = Tensors([5_000_003], 3)
    g = _grads([5_000_003], 30)
    _check_step(t, g, 1, seed=0xFFFFFFFF)
    _check_step(t, g, 2, seed=-1, max_norm=0.1, hyper=dict(lr=0.5, betas=(0.0, 0.0), eps=1e-3, weight_decay=0.0))
    _check_step(t, g, 70000, seed=5, hyper=dict(lr=0.0, betas=(0.95, 0.99), eps=0.0, weight_decay=0.1))


def test_zero_and_extreme_gradients():
    n = 640
    for value in (0.0, 1e-45, 1e-38, 1e-22, 1e-10, 1.0, 1e10, 1.5e19, 3e38):
        t = Tensors([n, 64], 4, lambda n: True)
        for k in (1, 2):
            g = _grads([n, 64], 40 + k)
            g[0][:] = value
            g[0][::7] = -value
            g[0][64:128] = 0
            g[0][200:] *= 1e-6
            _check_step(t, g, k)
    assert bool((t.v[0][64:128].float() == 0).all()) and bool((t.m[0][64:128].float() == 0).all())


@pytest.mark.parametrize("poison", [math.nan, math.inf, -math.inf])
def test_not_finite(poison):
    """A block that holds a NaN or an infinity reads back as NaN; the other blocks are what they are."""
    t = Tensors([300, 100], 5, lambda n: n == 300)
    g = _grads([300, 100], 50)
    g[0][70] = poison
    g[1][3] = poison
    _check_step(t, g, 1)
    assert torch.isnan(t.a[0]).tolist() == [False, True, False, False, False]
    _check_step(t, _grads([300, 100], 51), 2)
    assert torch.isnan(t.p[0]).nonzero().flatten().tolist() == list(range(64, 128))
    t = Tensors([300, 100], 5, lambda n: n == 300)
    g = _grads([300, 100], 50)
    g[0][70] = poison
    _check_step(t, g, 1, max_norm=0.5)     # the norm is NaN or infinite: every gradient becomes NaN, or 0 (NaN where infinite)


def test_rounding_is_unbiased():
    """The mean of the stored moments over many seeds is the exact moment: a code step is at most 1/8 of a moment of normal
    size, a rounding's standard deviation at most half of it, so the mean of 4096 lies within 6 / 64 of that half step."""
    from mpnn_amd.optim import adamw_step, unpack_moment

    n, seeds = 256, 4096
    g = torch.Generator().manual_seed(6)
    m0 = 0.1 * torch.randn(n, generator=g).cuda()
    sums = [torch.zeros(n, device="cuda", dtype=torch.float64) for _ in range(2)]
    for seed in range(seeds):
        m, v = (torch.zeros(n, device="cuda").to(torch.float8_e4m3fn) for _ in range(2))
        a, b = torch.ones(4, device="cuda"), torch.ones(4, device="cuda")
        adamw_step([torch.zeros(n, device="cuda")], [m0], [m], [v], [a], [b], step=1, seed=seed)
        sums[0] += unpack_moment(m, a)
        sums[1] += unpack_moment(v, b)
    for total, exact, scale in zip(sums, (0.1 * m0.double(), 0.001 * m0.double() ** 2), (a, b)):
        each = scale.double().repeat_interleave(64)
        step = torch.maximum(exact.abs() / 8, each * 2.0**-9)
        off = (total / seeds - exact).abs()
        ok = off <= 6 / 64 * step / 2 + 2.0**-17 * step
        ok |= (exact > 0) & (exact < each * 2.0**-9)      # held at the lowest code
        assert bool(ok.all()), float((off / step).max())


def test_optimizer_equals_the_function_and_spans_groups():
    from mpnn_amd.optim import AdamW, adamw_step, unpack_moment

    shapes = [(128, 384), (128,), (21, 128), (4096,), (64, 65)]
    make = lambda s: [torch.randn(*x, generator=torch.Generator().manual_seed(s + i)).cuda() for i, x in enumerate(shapes)]   # noqa: E731
    ps = [torch.nn.Parameter(x) for x in make(0)]
    opt = AdamW([{"params": ps[:2], "lr": 3e-3}, {"params": ps[2:], "weight_decay": 0.0}], lr=1e-3, max_grad_norm=0.3,
                state_bits=8, seed=17)
    t = Tensors([x.numel() for x in ps], 0, lambda n: n >= 4096)
    for q, p in zip(t.p, ps):
        q.copy_(p.detach().view(-1))
    for k in (1, 2, 3):
        gs = make(100 * k)
        for p, g in zip(ps, gs):
            p.grad = g
        versions = [p._version for p in ps]
        opt.step()
        assert all(p._version > v for p, v in zip(ps, versions))
        total = math.sqrt(sum(float((g.double() ** 2).sum()) for g in gs))
        assert abs(float(opt.last_grad_sumsq) - total**2) <= 1e-6 * total**2
    st = opt.state[ps[0]]
    assert st["exp_avg"].dtype == torch.float8_e4m3fn and st["exp_avg"].shape == ps[0].shape
    assert st["exp_avg_scale"].numel() == 768 and opt.state[ps[1]]["exp_avg"].dtype == torch.float32
    assert "exp_avg_scale" not in opt.state[ps[2]] and float(st["step"]) == 3.0
    # one group, no clipping: the class is the function
    ps = [torch.nn.Parameter(x) for x in make(0)]
    opt = AdamW(ps, lr=2e-3, weight_decay=0.1, state_bits=8, seed=4)
    for k in (1, 2):
        gs = make(100 * k)
        for p, g in zip(ps, gs):
            p.grad = g
        opt.step()
        adamw_step(t.p, [g.view(-1) for g in gs], t.m, t.v, t.a, t.b, step=k, lr=2e-3, weight_decay=0.1, seed=4)
    for p, q, m, a in zip(ps, t.p, t.m, t.a):
        assert torch.equal(p.detach().view(-1), q)
        if a is not None:
            assert torch.equal(unpack_moment(opt.state[p]["exp_avg"].view(-1), opt.state[p]["exp_avg_scale"]), unpack_moment(m, a))


def test_checkpoints_of_either_width(tmp_path):
    from mpnn_amd.optim import AdamW, unpack_moment

    def run(opt, ps, ks):
        for k in ks:
            for i, p in enumerate(ps):
                p.grad = torch.randn(p.shape, generator=torch.Generator().manual_seed(10 * k + i)).cuda()
            opt.step()

    new = lambda: [torch.nn.Parameter(torch.full((70, 80), 0.5).cuda()), torch.nn.Parameter(torch.ones(80).cuda())]   # noqa: E731
    a = new()
    opt_a = AdamW(a, state_bits=8, seed=3)
    run(opt_a, a, (1, 2))
    path = tmp_path / "opt.pt"
    torch.save({"opt": opt_a.state_dict(), "p": [p.detach() for p in a]}, path)
    ckpt = torch.load(path, weights_only=True)
    b = new()
    for p, q in zip(b, ckpt["p"]):
        p.data.copy_(q)
    opt_b = AdamW(b, state_bits=8, seed=3)
    opt_b.load_state_dict(ckpt["opt"])
    assert opt_b.state[b[0]]["exp_avg"].dtype == torch.float8_e4m3fn
    run(opt_a, a, (3,))
    run(opt_b, b, (3,))
    assert all(torch.equal(p, q) for p, q in zip(a, b)), "a resumed run is the same run"
    wide = AdamW(new(), state_bits=32)
    wide.load_state_dict(ckpt["opt"])          # 8 -> 32: the stored values
    st = list(wide.state.values())[0]
    s8 = ckpt["opt"]["state"][0]
    assert set(st) == {"step", "exp_avg", "exp_avg_sq"} and st["exp_avg"].dtype == torch.float32
    assert torch.equal(st["exp_avg"], unpack_moment(s8["exp_avg"], s8["exp_avg_scale"]).cuda())
    run(wide, wide.param_groups[0]["params"], (3,))
    ps = new()
    ref = torch.optim.AdamW(ps)
    run(ref, ps, (1, 2))
    back = AdamW(new(), state_bits=8)
    back.load_state_dict(ref.state_dict())     # 32 -> 8: to nearest, half a step of a 3-bit mantissa or of the lowest code
    st, want = list(back.state.values())[0], list(ref.state.values())[0]
    for name in ("exp_avg", "exp_avg_sq"):
        got = unpack_moment(st[name], st[name + "_scale"])
        low = st[name + "_scale"].repeat_interleave(64)[:5600].view(70, 80) * 2.0**-9
        assert bool(((got - want[name]).abs() <= torch.maximum(want[name].abs() * 2.0**-4, low)).all())
    assert bool((unpack_moment(st["exp_avg_sq"], st["exp_avg_sq_scale"]) > 0).all())
    run(back, back.param_groups[0]["params"], (3,))


def test_step_counts_of_parameters_that_join_later():
    """Each parameter has its own bias correction; one without a gradient keeps its count; counts survive a checkpoint."""
    from mpnn_amd.optim import AdamW

    def run(opt, ps, skip):
        for i, p in enumerate(ps):
            p.grad = None if i in skip else torch.full_like(p, 0.1 * (i + 1))
        opt.step()

    new = lambda: [torch.nn.Parameter(torch.ones(n).cuda()) for n in (5000, 100, 70000)]   # noqa: E731
    ps = new()
    opt = AdamW(ps, state_bits=8)
    for skip in ((), (1,), (0, 1), ()):
        run(opt, ps, skip)
    assert [float(opt.state[p]["step"]) for p in ps] == [3.0, 2.0, 4.0]
    ref = [torch.nn.Parameter(torch.ones_like(p)) for p in ps]
    opt_ref = torch.optim.AdamW(ref)
    for skip in ((), (1,), (0, 1), ()):
        run(opt_ref, ref, skip)
    # constant gradients: every moment of a tensor is the same number, a code times a power of two is 2^-4 off at most, v's
    # root 2^-5; four steps of 1e-3 each move p by that much of 4e-3
    for p, q in zip(ps, ref):
        assert float((p - q).detach().abs().max()) <= 4e-3 * 2 * (2.0**-3 + 2.0**-4)
    other = new()
    again = AdamW(other, state_bits=8)
    again.load_state_dict(opt.state_dict())
    for p, q in zip(other, ps):
        p.data.copy_(q)
    for o, xs in ((opt, ps), (again, other)):
        run(o, xs, (2,))
    assert [float(again.state[p]["step"]) for p in other] == [4.0, 3.0, 4.0]
    assert all(torch.equal(p, q) for p, q in zip(ps, other))


def test_function_in_a_graph_and_on_another_stream():
    """A captured step is the step (its number, hence its rounding, is the captured one); two graphs share nothing."""
    from mpnn_amd.optim import adamw_step

    sizes = [5000, 70, 64 * 300]
    runs = []
    for captured in (False, True):
        sets = [Tensors(sizes, 20 + k, lambda n: n > 100) for k in range(2)]
        grads = [[torch.empty(n, device="cuda") for n in sizes] for _ in range(2)]
        steps = [lambda t=t, g=g, k=k: adamw_step(t.p, g, t.m, t.v, t.a, t.b, step=3 + k, seed=k, max_grad_norm=0.5)
                 for k, (t, g) in enumerate(zip(sets, grads))]
        if captured:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            scratch = Tensors(sizes, 99, lambda n: n > 100)
            with torch.cuda.stream(side):          # warm-up on tensors of its own, on another stream
                adamw_step(scratch.p, grads[0], scratch.m, scratch.v, scratch.a, scratch.b, step=1, max_grad_norm=0.5)
            torch.cuda.current_stream().wait_stream(side)
            graphs, norms = [], []
            for f in steps:
                graphs.append(torch.cuda.CUDAGraph())
                with torch.cuda.graph(graphs[-1]):
                    norms.append(f())
        seen = []
        for k in range(4):
            for i in (0, 1):
                for dst, src in zip(grads[i], _grads(sizes, 60 + 2 * k + i)):
                    dst.copy_(src)
                if captured:
                    graphs[i].replay()
                    seen.append(float(norms[i]))
                else:
                    seen.append(float(steps[i]()))
        runs.append((seen, [x for t in sets for x in t.lists()]))
    assert runs[0][0] == runs[1][0]
    for x, y in zip(runs[0][1], runs[1][1]):
        for u, v in zip(x, y):
            assert u is v is None or np.array_equal(u, v)


def test_elements_beyond_32_bits_of_offset():
    """2^31 + 192 elements: addresses pass 2^33 bytes, element numbers 2^31."""
    from mpnn_amd.optim import adamw_step
    from oracle import adamw_oracle as orc

    n = 2**31 + 192
    p, g = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    m, v = (torch.zeros(n, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn) for _ in range(2))
    a, b = torch.ones(n // 64, device="cuda"), torch.ones(n // 64, device="cuda")
    ends = (slice(0, 128), slice(n - 256, n))
    for s in ends:
        g[s] = _grads([s.stop - s.start], 70)[0]
    adamw_step([p], [g], [m], [v], [a], [b], step=1, seed=5, weight_decay=0.0)
    key = int(orc.random_bits([0], int(orc.random_bits([1], 5)[0]))[0])
    for s in ends:
        r = orc.random_bits(np.arange(s.start, s.stop, dtype=np.uint64), key)
        x = g[s].cpu().double().numpy()
        for got, scale, want, u, pos in ((m, a, (1.0 - 0.9) * x, r & np.uint32(0xFFFF), False),
                                         (v, b, (1.0 - 0.999) * (x * x), r >> np.uint32(16), True)):
            codes, sc = orc.store(want, u / 65536.0, pos)
            np.testing.assert_array_equal(got[s].cpu().float().double().numpy(), codes)
            np.testing.assert_array_equal(scale[s.start // 64:s.stop // 64].cpu().double().numpy(), sc)
        assert bool(((p[s] != 0) == (g[s] != 0)).all())
    assert int((p != 0).sum()) == sum(int((g[s] != 0).sum()) for s in ends), "nothing else moved"


def test_refusals():
    from mpnn_amd.optim import AdamW, adamw_step

    z = lambda n, t=torch.float32: torch.zeros(n, device="cuda").to(t)   # noqa: E731
    e = torch.float8_e4m3fn
    good = dict(params=[z(100)], grads=[z(100)], exp_avgs=[z(100, e)], exp_avg_sqs=[z(100, e)], exp_avg_scales=[z(2)],
                exp_avg_sq_scales=[z(2)])
    adamw_step(step=1, **good)
    bad = [dict(grads=[z(99)]), dict(exp_avgs=[z(100)]), dict(exp_avg_sqs=[z(100)]), dict(exp_avg_scales=[None]),
           dict(exp_avg_scales=[z(1)]), dict(exp_avg_sq_scales=[z(2).half()]), dict(grads=[]), dict(exp_avgs=[z(200, e)[::2]])]
    for change in bad:
        with pytest.raises(ValueError):
            adamw_step(step=1, **{**good, **change})
    for change in (dict(params=[z(100).half()]), dict(grads=[z(200)[::2]]), dict(exp_avgs=[z(100, e).cpu()])):
        with pytest.raises(RuntimeError):
            adamw_step(step=1, **{**good, **change})
    with pytest.raises(ValueError):
        adamw_step(step=0, **good)
    twice = {n: x * 2 for n, x in good.items()}
    with pytest.raises(ValueError, match="share memory"):
        adamw_step(step=1, **twice)
    long = z(150)
    lapping = {**{n: x + [y.clone() for y in x] for n, x in good.items()}, "params": [long[:100], long[50:]]}
    with pytest.raises(ValueError, match="share memory"):
        adamw_step(step=1, **lapping)
    assert adamw_step([], [], [], [], [], [], step=1) is None
    p = torch.nn.Parameter(z(5000))
    p.grad = torch.ones_like(p)
    opt = AdamW([p], state_bits=8)
    opt.step()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    assert float(opt.state[p]["step"]) == 1.0
    p.grad = torch.ones(5000, device="cuda")[None][:, ::1].expand(2, 5000)[0].clone()
    opt.state[p]["exp_avg_scale"] = z(3)
    with pytest.raises(ValueError):
        opt.step()
    assert float(opt.state[p]["step"]) == 1.0, "a refused step does not count"


def test_training_step_with_8_bit_moments():
    import mpnn_amd
    from mpnn_amd import training
    from mpnn_amd.synthetic import synthetic_batch

    torch.manual_seed(0)
    results = []
    for _ in range(2):
        torch.manual_seed(1)
        model = mpnn_amd.ProteinMPNN(k_neighbors=16, augment_eps=0.0, dropout=0.0).train().cuda()
        opt, sched = training.make_optimizer(model, lr=1e-3, total_steps=200, max_grad_norm=1.0, state_bits=8)
        b = synthetic_batch(B=1, L=40, seed=3, device="cuda")
        batch = (b["X"], b["S"], b["mask"], b["chain_M"], b["residue_idx"], b["chain_encoding_all"])
        for _ in range(3):
            training.train_step(model, opt, batch, scheduler=sched, fix_order=b["fix_order"], max_grad_norm=1.0)
        with torch.no_grad():                      # the inference path sees the updated weights
            lp = model.eval()(*batch, fix_order=b["fix_order"])
        assert torch.isfinite(lp).all() and float(opt.last_grad_sumsq) > 0
        results.append([p.detach().clone() for p in model.parameters()])
    assert all(torch.equal(p, q) for p, q in zip(*results)), "the same seed gives the same run"
    held = sum(t.numel() * t.element_size() for st in opt.state.values() for n, t in st.items() if n != "step")
    assert held < 0.3 * 8 * sum(p.numel() for p in model.parameters())
