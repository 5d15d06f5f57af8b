"""beam_select and beam_reorder against their definitions in 64 bits (oracle/beam_oracle.py).

Bounds.  Whole numbers are equal: the inputs are random, so two candidates that are no ties lie further apart than the
kernel's fp64 errors (1e-11 against gaps of 1e-7 and more), and ties are made on purpose where the definition settles them.
Scores are an fp64 sum rounded once to fp32: half a step, 2^-24 relative, plus the kernel's exponentials (1.1e-12 relative
in the sum, so 1.1e-12 absolute in its logarithm); 2^-23 relative + 1e-10 holds both."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
NEG = -math.inf


def _case(B, W, V, dtype, seed, bias="none", forced=0.0, dead=True):
    g = torch.Generator().manual_seed(seed)
    logits = (2.5 * torch.randn(B, W, V, generator=g)).to(dtype)
    scores = -torch.cumsum(torch.rand(B, W, generator=g), 1)
    if dead and B > 1:
        scores[B - 1, 1:] = NEG
    add = None
    if bias != "none":
        shape = {"shared": (V,), "group": (B, 1, V), "beam": (W, V), "each": (B, W, V)}[bias]
        add = 0.3 * torch.randn(shape, generator=g)
        add = add.masked_fill(torch.rand(shape, generator=g) < 0.3, NEG)
    f = None
    if forced:
        f = torch.where(torch.rand(B, W, generator=g) < forced, torch.randint(0, V, (B, W), generator=g), torch.tensor(-1))
    return logits, scores, add, f


def _check(got, want):
    s, p, t = (x.cpu() for x in got)
    ws, wp, wt = want
    assert torch.equal(p, wp) and torch.equal(t, wt)
    fin = torch.isfinite(ws)
    assert torch.equal(torch.isnan(s), torch.isnan(ws)) and torch.equal(s == NEG, ws == NEG)
    err = (s[fin].double() - ws[fin]).abs()
    assert bool((err <= 2.0**-23 * ws[fin].abs() + 1e-10).all()), float(err.max())


def _run(logits, scores, bias=None, forced=None, n_out=None):
    import mpnn_amd
    from oracle import beam_oracle as orc

    dev = lambda t: None if t is None else t.cuda()   # noqa: E731
    got = mpnn_amd.beam_select(dev(logits), dev(scores), dev(bias), dev(forced), n_out)
    _check(got, orc.select(logits, scores, bias, forced, n_out))
    return got


SIZES = [(1, 1, 1), (1, 4, 21), (300, 2, 5), (2, 200, 21), (2, 128, 32), (1, 17, 480), (2, 4, 2040), (1, 3, 2700), (3, 1, 21), (64, 16, 21), (2, 64, 21), (2, 64, 32), (2, 33, 21), (5, 3, 64), (2, 7, 300),
         (4, 2, 1000), (2, 5, 1200), (3, 4, 2047), (1, 8, 2048), (2, 3, 5003), (1, 2, 40001), (1, 65, 21), (1, 256, 5)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,W,V", SIZES)
def test_select(B, W, V, dtype):
    _run(*_case(B, W, V, dtype, seed=V + W))


@pytest.mark.parametrize("B,W,V,n", [(3, 17, 174, 17), (2, 9, 468, 18), (2, 6, 882, 6), (3, 64, 250, 64), (2, 256, 60, 256),
                                     (3, 2, 700, 2), (2, 1, 1024, 9), (3, 40, 600, 40), (2, 70, 900, 64), (2, 100, 130, 100),
                                     (2, 64, 20000, 64), (1, 64, 131072, 64), (2, 200, 3000, 200), (2, 3, 40000, 256),
                                     (40, 20, 17000, 20)])
@pytest.mark.parametrize("values", ["fp32", "bf16", "coarse"])
def test_select_ways_of_splitting(B, W, V, n, values):
    """Sizes on each side of the rules that split a call; the last group is at a search's first step (one beam alive)."""
    import mpnn_amd
    from oracle import beam_oracle as orc

    g = torch.Generator().manual_seed(W + V)
    logits = 2.5 * torch.randn(B, W, V, generator=g)
    logits = logits.bfloat16() if values == "bf16" else (4 * logits).round() / 4 if values == "coarse" else logits
    scores = -torch.cumsum(torch.rand(B, W, generator=g), 1)
    scores[B - 1, 1:] = NEG
    got = mpnn_amd.beam_select(logits.cuda(), scores.cuda(), n_out=n)
    _check(got, orc.select_large(logits, scores, n))


@pytest.mark.parametrize("bias", ["shared", "group", "beam", "each"])
@pytest.mark.parametrize("B,W,V", [(4, 4, 21), (2, 16, 21), (3, 5, 700), (2, 3, 9001)])
def test_select_bias_and_forced(B, W, V, bias):
    _run(*_case(B, W, V, torch.float32, 5, bias, 0.3))
    _run(*_case(B, W, V, torch.bfloat16, 6, bias, 0.3))


@pytest.mark.parametrize("n_out", [1, 2, 9, 63, 64, 65, 130, 256])
@pytest.mark.parametrize("B,W,V", [(2, 4, 21), (1, 3, 1500), (2, 2, 9001)])
def test_select_numbers_kept(B, W, V, n_out):
    _run(*_case(B, W, V, torch.float32, 7, "each", 0.2), n_out=n_out)
    _run(*_case(B, W, V, torch.bfloat16, 8), n_out=n_out)


@pytest.mark.parametrize("W,V", [(3, 21), (4, 32), (2, 1300), (2, 5000), (2, 600), (1, 1000), (60, 400), (9, 900)])
def test_select_ties(W, V):
    """Constant logits: every token of a beam ties, and with equal scores the beams do too."""
    for scores in (torch.zeros(2, W), -torch.arange(2.0 * W).view(2, W) / 8):
        for n in (W, 40):
            _run(torch.full((2, W, V), 1.25), scores, n_out=n)
            _run(torch.full((2, W, V), 1.25, dtype=torch.bfloat16), scores, n_out=n)
    coarse = torch.randint(0, 3, (2, W, V), generator=torch.Generator().manual_seed(1)).float()   # few values, -0 and +0
    coarse = torch.where(coarse == 1, torch.tensor(-0.0), coarse - (coarse == 0).float() * 0)
    _run(coarse, torch.zeros(2, W), n_out=11)


@pytest.mark.parametrize("W,V", [(4, 21), (3, 3001)])
def test_select_rows_without_candidates(W, V):
    logits, scores, _, _ = _case(3, W, V, torch.float32, 9, dead=False)
    bias = torch.zeros(3, W, V)
    bias[0] = NEG                       # nothing left in a whole group
    bias[1, 0] = NEG                    # ... in one beam
    bias[2, 1, 5:] = NEG                # ... a few tokens of one beam
    logits[1, 0, 3] = math.nan          # NaN and infinities where the mask lies
    logits[1, 0, 4] = math.inf
    logits[2, 1, 7] = math.nan
    _run(logits, scores, bias)
    low = logits.nan_to_num(0, 0, 0)
    low[2] = torch.finfo(torch.float32).min            # the type's lowest value is a value
    _run(low, scores)
    low = low.clone()
    low[0, :, 2:] = NEG                                # -inf as logits
    low[1, 1] = NEG
    _run(low, scores, n_out=2 * W)
    _run(low.half(), torch.full((3, W), NEG))


@pytest.mark.parametrize("W,V", [(4, 21), (3, 3001)])
def test_select_not_finite(W, V):
    logits, scores, _, _ = _case(4, W, V, torch.float32, 10, dead=False)
    logits[0, 1, 2] = math.nan
    logits[1, 0, V - 1] = math.inf
    logits[1, 2, 0] = math.nan
    scores[2, 1] = math.nan
    scores[3, 0] = math.inf
    _run(logits, scores)
    _run(logits, scores, forced=torch.tensor([[1] * W, [-1] * W, [2] * W, [-1] * W]))


def test_select_nan_alone_in_its_part_of_the_row():
    """A long row is read in parts: one that holds a NaN and nothing else that counts breaks its beam all the same."""
    for V, where in ((2 * 2048 + 1, slice(4096, None)), (3 * 2048, slice(2048, 4096)), (3001, slice(0, 3001))):
        logits, scores, _, _ = _case(3, 2, V, torch.float32, 13, dead=False)
        logits[1, 1, where] = math.nan
        bias = torch.zeros(3, 2, V)
        bias[1, 1, where] = NEG
        bias[1, 1, where.start] = 0.0
        _run(logits, scores)
        _run(logits, scores, bias)
        _run(logits.bfloat16(), scores)


@pytest.mark.parametrize("W,V", [(4, 21), (2, 64), (1, 5000), (3, 9001), (2, 300)])
@pytest.mark.parametrize("n_out", [1, 3, 70, 255, 256])
def test_select_unequal_logits_of_equal_scores(W, V, n_out):
    """Scores that fp64 cannot tell apart tie, whatever their logits: the lowest tokens are kept."""
    g = torch.Generator().manual_seed(14)
    tiny = 1e-25 * torch.randn(2, W, V, generator=g)          # every score is score - log V
    _run(tiny, torch.zeros(2, W), n_out=n_out)
    _run(tiny.bfloat16(), -torch.rand(2, W, generator=g), n_out=n_out)
    few = torch.where(torch.rand(2, W, V, generator=g) < 0.02, tiny, -10.0 - torch.rand(2, W, V, generator=g))
    _run(few, torch.zeros(2, W), n_out=n_out)                 # a few such tokens above all others
    _run(few, torch.zeros(2, W), torch.where(torch.rand(V, generator=g) < 0.5, torch.tensor(NEG), torch.tensor(0.0)), n_out=n_out)
    _run(few, torch.zeros(2, W), forced=torch.tensor([[0] + [-1] * (W - 1)] * 2), n_out=n_out)
    # scores of 2^40: fp64's step there is 2^-12, so neighbouring logits share one.  Whole quarters with a distance of 2^-14:
    # all rounding of x - lse (1e-11 at most) stays on its side unless lse lies within that of an odd 2^-13
    logits = torch.randint(-20, 20, (2, W, V), generator=g) / 4 + torch.randint(0, 3, (2, W, V), generator=g) * 2.0**-14
    _run(logits, torch.full((2, W), -2.0**40), n_out=n_out)


@pytest.mark.parametrize("W,V", [(4, 21), (5, 47), (33, 21), (2, 600), (3, 4999), (5, 20011)])
def test_select_beams_of_equal_logits_tie(W, V):
    """Equal beams tie to the last bit, wherever their rows begin in memory: the lowest of them is kept for each token."""
    import mpnn_amd
    from oracle import beam_oracle as orc

    g = torch.Generator().manual_seed(15)
    for dtype in (torch.float32, torch.bfloat16):
        row = (3 * torch.randn(2, 1, V, generator=g)).to(dtype)
        apart = torch.cat([row] * W, 1)                                            # rows one after the other
        padded = torch.cat([torch.zeros(2, W, 3, dtype=dtype), apart], 2)[:, :, 3:]
        want = orc.select(apart, torch.zeros(2, W), None, None, 2 * W)
        assert torch.equal(want[1][0], torch.arange(W).repeat(2))
        for logits in (apart.cuda(), padded.cuda(), row.cuda().expand(2, W, V)):
            _check(mpnn_amd.beam_select(logits, torch.zeros(2, W, device="cuda"), n_out=2 * W), want)


def test_select_large_magnitudes():
    logits, scores, _, _ = _case(2, 4, 21, torch.float32, 11)
    _run(logits * 1e30, scores)
    _run(logits * 1e4, scores * 1e5)
    _run(logits[..., :1].expand(2, 4, 2500) * 1e-30, scores)


def test_select_strides():
    import mpnn_amd
    from oracle import beam_oracle as orc

    g = torch.Generator().manual_seed(12)
    for V in (21, 4099):
        base = torch.randn(6, 3, V + 3, generator=g)                          # beams outermost, rows at odd offsets
        view = base.transpose(0, 1)[:, :, 1:V + 1]
        scores = torch.randn(6, 3, generator=g).t()
        got = mpnn_amd.beam_select(base.cuda().transpose(0, 1)[:, :, 1:V + 1], scores.cuda())
        _check(got, orc.select(view, scores))
        half = base.half()
        got = mpnn_amd.beam_select(half.cuda().transpose(0, 1)[:, :, 1:V + 1], scores.cuda())
        _check(got, orc.select(half.transpose(0, 1)[:, :, 1:V + 1], scores))
        cols = torch.randn(3, V, 6, generator=g)                              # tokens not adjacent
        got = mpnn_amd.beam_select(cols.cuda().transpose(1, 2), scores.cuda())
        _check(got, orc.select(cols.transpose(1, 2), scores))
        rep = torch.randn(1, 1, V, generator=g).expand(3, 6, V)               # one row for all beams
        got = mpnn_amd.beam_select(rep.cuda(), scores.cuda(), bias=rep.cuda()[0, 0])
        _check(got, orc.select(rep, scores, bias=rep[0, 0]))


def test_offsets_beyond_32_bits():
    """Rows that lie 2^31 elements and more apart: logits of a selection, states of more than 4 GiB."""
    import mpnn_amd
    from oracle import beam_oracle as orc

    V, far = 2100, 2**31 + 5
    buf = torch.zeros(far + V, device="cuda", dtype=torch.float16)
    rows = buf.as_strided((1, 2, V), (2 * far, far, 1))
    small = torch.randn(1, 2, V, generator=torch.Generator().manual_seed(2)).half()
    rows.copy_(small)
    scores = torch.tensor([[-0.5, -0.25]])
    _check(mpnn_amd.beam_select(rows, scores.cuda(), n_out=7), orc.select(small, scores, n_out=7))
    _check(mpnn_amd.beam_select(rows[..., :30], scores.cuda(), n_out=7), orc.select(small[..., :30], scores, n_out=7))
    del buf, rows
    n = 2**31 + 64
    state = torch.zeros(1, 3, n, device="cuda", dtype=torch.uint8)
    ends = torch.randint(1, 255, (1, 3, 96), generator=torch.Generator().manual_seed(3)).to(torch.uint8)
    state[..., :32] = ends[..., :32].cuda()
    state[..., -64:] = ends[..., 32:].cuda()
    parent = torch.tensor([[2, 0, 0]])
    mpnn_amd.beam_reorder(state, parent.cuda())
    want = orc.reorder(ends, parent)
    assert torch.equal(state[..., :32].cpu(), want[..., :32]) and torch.equal(state[..., -64:].cpu(), want[..., 32:])
    state = state.view(1, 3, -1, 64)                       # positions of 64 bytes, the last ones alone move back
    rank = torch.arange(state.shape[2], device="cuda", dtype=torch.int32).flip(0)[None]
    mpnn_amd.beam_reorder(state, torch.tensor([[1, 2, 1]]).cuda(), length=1, rank=rank)
    last = orc.reorder(want[..., 32:], torch.tensor([[1, 2, 1]]))
    assert torch.equal(state[:, :, -1].cpu(), last) and torch.equal(state[:, :, 0, :32].cpu(), want[..., :32])


def test_inference_tensors_and_grad_mode():
    import mpnn_amd
    from oracle import beam_oracle as orc

    logits, scores, bias, forced = _case(2, 3, 40, torch.float32, 14, "each", 0.2)
    with torch.inference_mode():
        dev = [x.cuda() for x in (logits, scores, bias, forced)]
        out = mpnn_amd.beam_select(*dev)
        state = torch.arange(2 * 3 * 4.0).view(2, 3, 4)
        gpu = state.cuda()
        mpnn_amd.beam_reorder(gpu, out[1])
    want = orc.select(logits, scores, bias, forced)
    _check(out, want)
    assert torch.equal(gpu.cpu(), orc.reorder(state, want[1]))
    leaf = logits.cuda().requires_grad_()
    out = mpnn_amd.beam_select(leaf * 1.0, scores.cuda(), bias.cuda(), forced.cuda())
    assert not out[0].requires_grad
    _check(out, want)


def test_select_refusals():
    import mpnn_amd

    z = lambda *s: torch.zeros(s, device="cuda")   # noqa: E731
    ok = dict(logits=z(2, 3, 5), scores=z(2, 3))
    mpnn_amd.beam_select(**ok)
    for bad in (dict(logits=z(2, 5)), dict(logits=z(2, 3, 5).double()), dict(logits=z(2, 3, 0)), dict(logits=z(2, 0, 5), scores=z(2, 0)),
                dict(scores=z(3, 2)), dict(scores=z(2, 3).double()), dict(bias=z(4)), dict(bias=z(5).half()), dict(bias=z(1)[0]),
                dict(forced=z(2, 3)), dict(n_out=0), dict(n_out=257), dict(logits=z(1, 257, 2), scores=z(1, 257))):
        with pytest.raises(ValueError, match="beam_select"):
            mpnn_amd.beam_select(**{**ok, **bad})
    for bad in (dict(bias=torch.zeros(5)), dict(forced=torch.zeros(2, 3, dtype=torch.int64)), dict(scores=torch.zeros(2, 3)),
                dict(bias=z(3, 2, 5)), dict(forced=z(4).long())):
        with pytest.raises(RuntimeError):
            mpnn_amd.beam_select(**{**ok, **bad})
    with pytest.raises(TypeError):
        mpnn_amd.beam_select([1], z(2, 3))
    parent = torch.zeros(2, 3, device="cuda", dtype=torch.int64)
    for bad in (dict(states=z(3, 2, 4)), dict(states=z(2)), dict(parent=parent[0]), dict(parent=z(2, 3)), dict(rank=parent),
                dict(length=3, states=z(2, 3)), dict(length=3, states=[z(2, 3, 4), z(2, 3, 5)]), dict(length=parent[0]),
                dict(length=3, rank=parent), dict(length=3, rank=z(2, 4))):
        with pytest.raises(ValueError, match="beam_reorder"):
            mpnn_amd.beam_reorder(**{**dict(states=z(2, 3, 4), parent=parent), **bad})
    with pytest.raises(TypeError):
        mpnn_amd.beam_reorder(7, parent)
    with pytest.raises(TypeError):
        mpnn_amd.beam_reorder(z(2, 3, 4), parent, length="x")


def test_select_empty_batch_and_repeat():
    import mpnn_amd

    s, p, t = mpnn_amd.beam_select(torch.zeros(0, 4, 21, device="cuda"), torch.zeros(0, 4, device="cuda"))
    assert s.shape == p.shape == t.shape == (0, 4)
    logits, scores, bias, forced = _case(2, 5, 20011, torch.bfloat16, 13, "each", 0.1)
    a = mpnn_amd.beam_select(logits.cuda(), scores.cuda(), bias.cuda(), forced.cuda())
    for _ in range(3):
        b = mpnn_amd.beam_select(logits.cuda(), scores.cuda(), bias.cuda(), forced.cuda())
        assert all(torch.equal(x, y) for x, y in zip(a, b))


# ---- states -----------------------------------------------------------------------------------------------------
def _parent(B, W, seed):
    g = torch.Generator().manual_seed(seed)
    p = torch.randint(0, W, (B, W), generator=g)
    p[0] = torch.arange(W).flip(0)      # a permutation without a fixed row
    return p


STATES = {
    "rows": lambda B, W, g: torch.randn(B, W, 40, generator=g),
    "scalar": lambda B, W, g: torch.randint(0, 99, (B, W), generator=g),
    "bytes": lambda B, W, g: torch.randint(0, 255, (B, W, 13), generator=g).to(torch.uint8),
    "flags": lambda B, W, g: torch.rand(B, W, 5, 7, generator=g) < 0.5,
    "half": lambda B, W, g: torch.randn(B, W, 3, 5, generator=g).half(),
    "odd": lambda B, W, g: torch.randn(B, W, 7, 33, generator=g)[:, :, :, 1:30],
    "beams_first": lambda B, W, g: torch.randn(W, B, 11, 8, generator=g).transpose(0, 1),
    "prefix": lambda B, W, g: torch.randn(B, W, 3, 20, 16, generator=g).bfloat16()[:, :, :, :13],
    "column": lambda B, W, g: torch.randn(B, W, 9, 6, generator=g)[..., 2],
    "nan": lambda B, W, g: torch.full((B, W, 4), math.nan),
    "long": lambda B, W, g: torch.randn(B, W, 3001, generator=g).double(),
}


@pytest.mark.parametrize("B,W", [(1, 1), (1, 2), (3, 4), (2, 9), (2, 64), (1, 65), (1, 129), (1, 256)])
def test_reorder(B, W):
    import mpnn_amd
    from oracle import beam_oracle as orc

    g = torch.Generator().manual_seed(B * 1000 + W)
    parent = _parent(B, W, W)
    cpu = [f(B, W, g) for f in STATES.values()]
    gpu = [torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device="cuda").copy_(x) for x in cpu]
    out = mpnn_amd.beam_reorder(gpu, parent.cuda())
    assert out is gpu
    for name, x, y in zip(STATES, cpu, gpu):
        want = orc.reorder(x, parent)
        assert torch.equal(y.cpu().contiguous().view(torch.uint8), want.contiguous().view(torch.uint8)), name
    one = mpnn_amd.beam_reorder(gpu[0], parent.to(torch.int32).cuda())
    assert one is gpu[0] and torch.equal(one.cpu(), orc.reorder(orc.reorder(cpu[0], parent), parent))


@pytest.mark.parametrize("W", [1, 3, 16, 70])
@pytest.mark.parametrize("how", ["int", "zero", "all", "ragged"])
@pytest.mark.parametrize("ranked", [False, True])
def test_reorder_length(W, how, ranked):
    import mpnn_amd
    from oracle import beam_oracle as orc

    B, L = 3, 19
    g = torch.Generator().manual_seed(W)
    parent = _parent(B, W, W + 1)
    length = {"int": 7, "zero": 0, "all": 19, "ragged": torch.tensor([0, 19, 5])}[how]
    rank = torch.argsort(torch.rand(B, L, generator=g), 1) if ranked else None
    cpu = [torch.randn(W, B, L, 256, generator=g).transpose(0, 1)[..., 128:], torch.randint(0, 21, (B, W, L), generator=g),
           torch.randn(B, W, L, 21, generator=g), torch.randn(B, W, L, 3, 4, generator=g).half()]
    gpu = [torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device="cuda").copy_(x) for x in cpu]
    mpnn_amd.beam_reorder(gpu, parent.cuda(), length.cuda() if how == "ragged" else length, None if rank is None else rank.cuda())
    for x, y in zip(cpu, gpu):
        assert torch.equal(y.cpu(), orc.reorder(x, parent, length, rank))


def test_reorder_leaves_the_rest_alone():
    """Bytes between and behind the rows of a view, and rows whose parent is none, stay as they were."""
    import mpnn_amd
    from oracle import beam_oracle as orc

    g = torch.Generator().manual_seed(3)
    buf = torch.randn(2, 5, 6, 40, generator=g)
    parent = torch.tensor([[4, -1, 5, 0, 0], [1, 2, 3, 4, 99]])
    dev = buf.cuda()
    mpnn_amd.beam_reorder(dev[:, :, 1:4, 3:21], parent.cuda())
    want = buf.clone()
    want[:, :, 1:4, 3:21] = orc.reorder(buf[:, :, 1:4, 3:21], parent)
    assert torch.equal(dev.cpu(), want)


def test_reorder_interleaved_states_and_overlaps():
    import mpnn_amd
    from oracle import beam_oracle as orc

    g = torch.Generator().manual_seed(4)
    buf = torch.randn(2, 3, 10, 16, generator=g)
    parent = _parent(2, 3, 5)
    dev = buf.cuda()
    v0 = dev._version
    mpnn_amd.beam_reorder([dev[..., :8], dev[..., 8:]], parent.cuda(), length=4)       # rows of one between the other's
    assert torch.equal(dev.cpu(), orc.reorder(buf, parent, 4)) and dev._version > v0
    for pair in ([dev, dev], [dev[..., :9], dev[..., 8:]], [dev[:, :, :5], dev[:, :, 4:]], [dev, dev.view(2, 3, 160)]):
        with pytest.raises(ValueError, match="share memory"):
            mpnn_amd.beam_reorder(pair, parent.cuda())
    with pytest.raises(ValueError, match="share memory"):
        mpnn_amd.beam_reorder(torch.zeros(2, 1, 4, device="cuda").expand(2, 3, 4), parent.cuda())
    with pytest.raises(ValueError, match="contiguous"):
        mpnn_amd.beam_reorder(torch.zeros(2, 3, 4, 6, 8, device="cuda")[:, :, :3, :5, :7], parent.cuda())
    p = torch.nn.Parameter(torch.zeros(2, 3, 4, device="cuda"))
    with pytest.raises(RuntimeError, match="gradients"):
        mpnn_amd.beam_reorder(p, parent.cuda())


def test_reorder_of_the_parents_themselves():
    """A history of parents is a state like any other, also the one that says who moves where, or when."""
    import mpnn_amd
    from oracle import beam_oracle as orc

    g = torch.Generator().manual_seed(8)
    history = torch.randint(0, 5, (3, 5, 7), generator=g)
    dev = history.cuda()
    mpnn_amd.beam_reorder(dev, dev[:, :, 2])
    assert torch.equal(dev.cpu(), orc.reorder(history, history[:, :, 2]))
    parent = torch.randint(0, 40, (2, 40), generator=g)
    dev = parent.cuda()
    mpnn_amd.beam_reorder([dev, dev.clone()], dev)
    assert torch.equal(dev.cpu(), orc.reorder(parent, parent))
    table = torch.randint(0, 9, (2, 2, 9), generator=g, dtype=torch.int32)
    dev = table.cuda()
    mpnn_amd.beam_reorder(dev, torch.tensor([[1, 0], [1, 1]]).cuda(), length=4, rank=dev[:, 0])
    assert torch.equal(dev.cpu(), orc.reorder(table, torch.tensor([[1, 0], [1, 1]]), 4, table[:, 0]))


def test_reorder_many_states():
    import mpnn_amd
    from oracle import beam_oracle as orc

    g = torch.Generator().manual_seed(6)
    parent = _parent(3, 4, 7)
    cpu = [torch.randn(3, 4, 5 + i, generator=g).to(torch.float32 if i % 2 else torch.float16) for i in range(41)]
    gpu = [x.cuda() for x in cpu]
    mpnn_amd.beam_reorder(gpu, parent.cuda())
    for x, y in zip(cpu, gpu):
        assert torch.equal(y.cpu(), orc.reorder(x, parent))
    assert mpnn_amd.beam_reorder([], parent.cuda()) == []
    empty = torch.zeros(3, 4, 0, device="cuda")
    assert mpnn_amd.beam_reorder(empty, parent.cuda()) is empty


# ---- both, as a search uses them --------------------------------------------------------------------------------
def _toy_search(select, reorder, tables, W, steps, device):
    """A first-order model with a state per beam: the search's own bookkeeping is what is tested."""
    V = tables.shape[-1]
    B = tables.shape[0]
    state = torch.zeros(B, W, steps, device=device, dtype=torch.int64)       # the letters so far
    run = torch.zeros(B, W, 5, device=device)                                # a running state of the model
    scores = torch.full((B, W), NEG, device=device)
    scores[:, 0] = 0.0
    group = torch.arange(B, device=device)[:, None]
    for t in range(steps):
        last = state[:, :, t - 1] if t else torch.zeros(B, W, dtype=torch.int64, device=device)
        logits = tables[group, last] + run.sum(-1, keepdim=True) * torch.arange(V, device=device) / V
        scores, parent, token = select(logits, scores)
        scores = scores.float()
        state, run = reorder(state, parent), reorder(run, parent)
        state[:, :, t] = token
        run[:, :, t % 5] = token.float() * 0.25
    return scores, state


@pytest.mark.parametrize("W,V,steps", [(1, 21, 6), (4, 21, 9), (30, 21, 4), (3, 2500, 4)])
def test_search_loop(W, V, steps):
    import mpnn_amd
    from oracle import beam_oracle as orc

    tables = torch.randn(3, V, V, generator=torch.Generator().manual_seed(V + W))
    a = _toy_search(mpnn_amd.beam_select, mpnn_amd.beam_reorder, tables.cuda(), W, steps, "cuda")
    b = _toy_search(orc.select, orc.reorder, tables, W, steps, "cpu")
    assert torch.equal(a[1].cpu(), b[1])
    # The model's own logits differ between the devices: `x * v / V` is two roundings on the CPU and, as a product with the
    # rounded reciprocal, three on the GPU, so at most 5 * 2^-24 relative apart (adding the table's entry rounds once more on
    # each side: 7), and |x| <= 5 * (V - 1) / 4.  A log-softmax passes twice that on (the logit's and the sum's), each step.
    atol = steps * 2 * 7 * 2.0**-24 * (1.25 * V + 5)
    assert torch.allclose(a[0].cpu(), b[0], rtol=steps * 2.0**-22, atol=atol)


@pytest.mark.parametrize("V", [21, 6007])
def test_search_step_in_a_graph_and_on_another_stream(V):
    import mpnn_amd

    cases = [_case(3, 4, V, torch.float32, s, "shared", 0.1) for s in range(4)]
    logits, scores, bias, forced = (x.cuda() for x in cases[0])
    state = torch.randn(3, 4, 50, device="cuda")
    first = state.clone()

    def step():
        out = mpnn_amd.beam_select(logits, scores, bias, forced)
        mpnn_amd.beam_reorder(state, out[1])
        return out

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        eager = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for c in cases + cases[:2]:
        for dst, src in zip((logits, scores, bias, forced), c):
            dst.copy_(src)
        state.copy_(first)
        graph.replay()
        torch.cuda.synchronize()
        got, moved = [x.clone() for x in out], state.clone()
        state.copy_(first)
        eager = step()
        assert all(torch.equal(x, y) for x, y in zip(got, eager)) and torch.equal(moved, state)
