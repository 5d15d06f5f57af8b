"""ProteinMPNN.beam_search: the sequences, their log-probs and their scores against teacher-forced forwards (HIP and CPU
oracle) and against a search that computes every step with whole forwards and selects with the 64-bit oracle."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

CASES = {
    "k48_vc": (dict(k_neighbors=48, use_virtual_center=True), dict(B=2, L=96, seed=3, lengths=[96, 70], n_chains=2,
                                                                   design_fraction=0.7), 5),
    "k30_cutoff": (dict(k_neighbors=30, edge_cutoff=14.0), dict(B=1, L=65, seed=8, n_chains=1, design_fraction=1.0), 32),
    "k16_short": (dict(k_neighbors=16), dict(B=3, L=40, seed=5, lengths=[40, 31, 12], n_chains=2, design_fraction=0.5), 2),
    "k64": (dict(k_neighbors=64), dict(B=2, L=70, seed=13, lengths=[70, 65], n_chains=2, design_fraction=0.8), 3),
    "one_layer": (dict(k_neighbors=8, num_decoder_layers=1, num_encoder_layers=1), dict(B=1, L=9, seed=1, design_fraction=1.0), 64),
    "one_residue": (dict(k_neighbors=4), dict(B=2, L=1, seed=2, design_fraction=1.0), 30),
}


def build(kw):
    import mpnn_amd
    from mpnn_amd.synthetic import fill_parameters_

    model = mpnn_amd.ProteinMPNN(augment_eps=0.0, dropout=0.0, **kw).eval()
    fill_parameters_(model, seed=0)
    return model.to("cuda")


def inputs(bkw):
    from mpnn_amd.synthetic import synthetic_batch

    b = {k: v.to("cuda") for k, v in synthetic_batch(**bkw).items()}
    return b, (b["X"], b["mask"], b["chain_M"], b["residue_idx"], b["chain_encoding_all"])


def score_bound(L, score):
    """A score is rounded to fp32 at each of L steps (2^-24 |score|); its terms are log-probs, the kernels' fp32 logits on both
    sides: 1e-5 apart, as the forward and the sampler are held to."""
    return L * (2.0**-24 * abs(score) + 1e-5)


@pytest.mark.parametrize("name", list(CASES))
def test_matches_teacher_forced_forward(name):
    kw, bkw, W = CASES[name]
    model = build(kw)
    b, args = inputs(bkw)
    out = model.beam_search(*args, S_true=b["S"], beam_width=W, seed=11)
    S, lp, scores, order = out["S"], out["log_probs"], out["scores"], out["order"]
    B, L = b["S"].shape
    assert S.shape == (W, B, L) and scores.shape == (W, B) and order.shape == (B, L)
    fixed = (b["chain_M"] * b["mask"]) == 0
    with torch.no_grad():
        for w in range(W):
            assert int(S[w].min()) >= 0 and int(S[w].max()) < 21
            assert torch.equal(S[w][fixed], b["S"][fixed])
            ref = model(b["X"], S[w], b["mask"], b["chain_M"], b["residue_idx"], b["chain_encoding_all"], fix_order=order)
            assert float((ref - lp[w]).abs().max()) <= 1e-5
            mine = (ref.gather(-1, S[w].unsqueeze(-1)).squeeze(-1).double() * (~fixed)).sum(-1)
            for i in range(B):
                if float(scores[w, i]) > -math.inf:
                    assert abs(float(mine[i]) - float(scores[w, i])) <= score_bound(L, float(mine[i])), (w, i)
    # best first, every living hypothesis another sequence, as many as there can be
    for i in range(B):
        live = [w for w in range(W) if float(scores[w, i]) > -math.inf]
        designed = int((~fixed[i]).sum())
        assert len(live) == min(W, 21 ** min(designed, 4)) and live == list(range(len(live)))
        assert len({tuple(S[w, i].tolist()) for w in live}) == len(live)
        assert bool((scores[:-1, i] >= scores[1:, i]).all())


def _search_by_forwards(model, b, order, W, bias=None):
    """Every step: one whole forward per hypothesis, its log-probs at the step's residue, the 64-bit oracle's choice."""
    from oracle import beam_oracle as orc

    B, L = b["S"].shape
    S = torch.zeros(B, W, L, dtype=torch.int64)
    scores = torch.full((B, W), -math.inf)
    scores[:, 0] = 0.0
    fixed = ((b["chain_M"] * b["mask"]) == 0).cpu()
    group = torch.arange(B)
    for t in range(L):
        i = order[:, t].cpu()
        logits = torch.empty(B, W, 21)
        with torch.no_grad():
            for w in range(W):
                lp = model(b["X"], S[:, w].cuda(), b["mask"], b["chain_M"], b["residue_idx"], b["chain_encoding_all"], fix_order=order)
                logits[:, w] = lp.cpu()[group, i]
        forced = torch.where(fixed[group, i], b["S"].cpu()[group, i], torch.tensor(-1))
        best, parent, token = orc.select(logits, scores, bias, forced)
        scores = best.float()
        S = orc.reorder(S, parent)
        S[group.view(B, 1), torch.arange(W), i.view(B, 1)] = token
    return S.transpose(0, 1), scores.t()


@pytest.mark.parametrize("name,W", [("k16_short", 3), ("k48_vc", 2), ("one_layer", 25), ("k64", 1)])
@pytest.mark.parametrize("biased", [False, True])
def test_matches_a_search_by_whole_forwards(name, W, biased):
    kw, bkw, _ = CASES[name]
    if name in ("k48_vc", "k64"):
        bkw = dict(B=2, L=52, seed=9, lengths=[52, 50], n_chains=1, design_fraction=0.8)
    model = build(kw)
    b, args = inputs(bkw)
    bias = None
    if biased:
        bias = 0.5 * torch.randn(21, generator=torch.Generator().manual_seed(1))
        bias[[4, 20]] = -math.inf
    out = model.beam_search(*args, S_true=b["S"], beam_width=W, fix_order=b["fix_order"], logit_bias=bias)
    assert torch.equal(out["order"], b["fix_order"])
    S, scores = _search_by_forwards(model, b, b["fix_order"], W, bias)
    live = scores > -math.inf
    assert torch.equal(out["S"].cpu()[live], S[live])
    got = out["scores"].cpu()
    assert torch.equal(got == -math.inf, ~live)
    bound = scores[live].abs() * 2.0**-23 * S.shape[-1] + 1e-5 * S.shape[-1]
    assert bool(((got - scores)[live].abs() <= bound).all())


def test_oracle_log_probs():
    """The reference's teacher-forced forward on the CPU returns the log-probs of every hypothesis."""
    from conftest import oracle_cfg
    from oracle import mpnn_oracle as orc

    kw, bkw, W = CASES["k48_vc"]
    model = build(kw)
    b, args = inputs(bkw)
    out = model.beam_search(*args, S_true=b["S"], beam_width=W, seed=2)
    sd = {k: v.detach().cpu() for k, v in model.state_dict().items()}
    c = {k: v.cpu() for k, v in b.items()}
    with torch.no_grad():
        for w in (0, W - 1):
            ref = orc.forward(sd, oracle_cfg(kw), c["X"], out["S"][w].cpu(), c["mask"], c["chain_M"], c["residue_idx"],
                              c["chain_encoding_all"], fix_order=out["order"].cpu(), formulation="edge")
            err = (out["log_probs"][w].cpu().double() - ref.double()).abs()
            assert bool((err <= 1e-5 + 1e-4 * ref.double().abs()).all()), float(err.max())


def test_greedy_and_reproducible_and_wider_is_no_other_problem():
    kw, bkw, _ = CASES["k30_cutoff"]
    model = build(kw)
    b, args = inputs(bkw)
    one = model.beam_search(*args, beam_width=1, seed=5)
    assert torch.equal(one["S"][0], one["log_probs"][0].argmax(-1)), "one beam takes the best letter everywhere"
    again = model.beam_search(*args, beam_width=1, seed=5)
    assert all(torch.equal(one[k], again[k]) for k in one)
    assert not torch.equal(model.beam_search(*args, beam_width=1, seed=6)["order"], one["order"])
    wide = [model.beam_search(*args, beam_width=8, fix_order=one["order"]) for _ in range(2)]
    assert all(torch.equal(wide[0][k], wide[1][k]) for k in wide[0]), "the same call gives the same bits"


def test_few_letters_and_dead_hypotheses():
    """Two letters left and three residues: eight sequences, the other places of twenty are dead."""
    model = build(dict(k_neighbors=4))
    b, args = inputs(dict(B=2, L=3, seed=4, design_fraction=1.0))
    bias = torch.full((21,), -math.inf)
    bias[[3, 7]] = 0.0
    out = model.beam_search(*args, beam_width=20, logit_bias=bias)
    for i in range(2):
        assert [bool(s > -math.inf) for s in out["scores"][:, i].tolist()] == [True] * 8 + [False] * 12
        assert len({tuple(s) for s in out["S"][:8, i].tolist()}) == 8
        assert set(out["S"][:8, i].flatten().tolist()) == {3, 7}
        total = torch.logsumexp(out["scores"][:8, i].double(), 0)
        assert abs(float(total)) <= 3 * 8 * 2.0**-22, "all sequences' probabilities add up to one"


def test_nothing_designed_and_f16_and_refusals():
    model = build(dict(k_neighbors=16))
    b, args = inputs(dict(B=2, L=30, seed=4, design_fraction=1.0))
    none = (args[0], args[1], torch.zeros_like(args[2])) + args[3:]
    out = model.beam_search(*none, S_true=b["S"], beam_width=3)
    assert torch.equal(out["S"][0], b["S"]) and out["scores"][0].tolist() == [0.0, 0.0]
    full = model.beam_search(*args, beam_width=4, seed=1)
    half = model.set_precision("f16").beam_search(*args, beam_width=4, seed=1)
    model.set_precision("fp32")
    with torch.no_grad():
        ref = model(b["X"], half["S"][0], b["mask"], b["chain_M"], b["residue_idx"], b["chain_encoding_all"], fix_order=half["order"])
    assert float((ref - half["log_probs"][0]).abs().max()) <= 5e-2      # the mode's stated tolerance
    assert not torch.equal(full["log_probs"], half["log_probs"])
    for kw in (dict(beam_width=0), dict(beam_width=65), dict(fix_order=torch.zeros(2, 30, dtype=torch.int64, device="cuda")),
               dict(fix_order=full["order"][:1]), dict(logit_bias=torch.zeros(3))):
        with pytest.raises(ValueError):
            model.beam_search(*args, **kw)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        model.beam_search(*(t.cpu() for t in args))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = model.beam_search(*args, beam_width=4, seed=1)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(full[k], other[k]) for k in full)


def test_inputs_elsewhere_or_of_another_size_are_refused():
    """Before anything is launched: the kernels take bare addresses."""
    model = build(dict(k_neighbors=16))
    b, args = inputs(dict(B=2, L=30, seed=4, design_fraction=1.0))
    given = dict(X=args[0], mask=args[1], residue_idx=args[3], chain_encoding_all=args[4])
    rest = dict(chain_M=args[2], S_true=b["S"], fix_order=model.beam_search(*args, beam_width=1)["order"], beam_width=2)
    for name in given:
        for bad, error in ((given[name].cpu(), RuntimeError), (given[name][:, :29], ValueError), (given[name][:1], ValueError)):
            with pytest.raises(error):
                model.beam_search(**{**given, name: bad}, **rest)
    for name in ("chain_M", "S_true", "fix_order"):
        with pytest.raises((RuntimeError, ValueError)):
            model.beam_search(**given, **{**rest, name: rest[name].cpu()})
        with pytest.raises((RuntimeError, ValueError)):
            model.beam_search(**given, **{**rest, name: rest[name][:, :29]})
    for noise in (torch.zeros(2, 29, 4, 3, device="cuda"), torch.zeros(2, 30, 4, 3)):
        from mpnn_amd import engine
        with pytest.raises(ValueError):
            engine.beam_search(model, *args, beam_width=2, backbone_noise=noise)
    assert model.beam_search(**given, **rest)["S"].shape == (2, 2, 30)
