"""Cases that time the framework's beam-search and optimizer operators, beside a plain form of each.

Three operators:

  select   beam search's choice of the next hypotheses (`mpnn_amd.beam_select`): the log-softmax of every beam's logits,
           added to the beams' scores, and the best of all beams x tokens, with the beam and the token of each
  reorder  the beams' decoder states follow their hypotheses (`mpnn_amd.beam_reorder`): row j of every group becomes what
           row parent[j] held, in place, over several tensors at once
  adamw    one AdamW step over many tensors (`mpnn_amd.optim.adamw_step`), the moments of the large ones held in 8 bits
           with a scale for each 64 elements and rounded stochastically, those of the small ones in 32 bits

`own` chooses between the plain form (elementary torch operations) and the framework's calls.
"""
import math

import numpy as np
import torch

own = False

NEG = float("-inf")
BLOCK = 64


# ---------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one protein, four beams, the model's 21 letters: what a single design call pays at every residue
        dict(name="select_one_structure", op="select", B=1, W=4, V=21, n=4, dtype="float32", bias="none", forced=0.0),
        # a batch of 64 proteins with 16 beams, one letter excluded, a tenth of the structures at a fixed residue
        dict(name="select_structures", op="select", B=64, W=16, V=21, n=16, dtype="float32", bias="shared", forced=0.1),
        # a sub-word vocabulary of odd size, half precision, 2 W candidates kept
        dict(name="select_words", op="select", B=8, W=5, V=32003, n=10, dtype="bfloat16", bias="none", forced=0.0),
        # the largest: a batch of 32 with 8 beams over 2^17 tokens and a mask of its own for every beam
        dict(name="select_largest", op="select", B=32, W=8, V=131072, n=8, dtype="float32", bias="each", forced=0.05),
        # one protein of 100 residues, 37 of them decoded: three decoder layers' rows, the letters and their log-probs
        dict(name="reorder_one_structure", op="reorder", kind="design", B=1, W=8, L=100, t=37),
        # a batch of 16 proteins of 512 residues, 16 beams, half decoded
        dict(name="reorder_structures", op="reorder", kind="design", B=16, W=16, L=512, t=257),
        # keys and values of two layers in half precision, the decoded prefix of a longer buffer
        dict(name="reorder_cache", op="reorder", kind="cache", B=8, W=4, heads=8, T=4096, t=4001, D=128, layers=2,
             dtype="bfloat16"),
        # the parameters of the default model with the gradient norm clipped: 41 tensors in 8 bits, 77 in 32
        dict(name="adamw_model", op="adamw", kind="model", step=100, clip=1.0),
        # many tensors of odd sizes, no clipping, an early step
        dict(name="adamw_ragged", op="adamw", kind="ragged", tensors=300, largest=60000, sizes=1, step=2, clip=0.0),
        # the largest: 100 million parameters in 30 tensors
        dict(name="adamw_largest", op="adamw", kind="even", tensors=30, largest=3400001, sizes=2, step=1000, clip=0.5),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.499)))))))


def draw(rng):
    op = rng.choice(["select", "reorder", "adamw"])
    if op == "select":
        V = _log_uniform(rng, 2, 131072)
        W = _log_uniform(rng, 1, 64)
        B = _log_uniform(rng, 1, max(1, min(256, 33000000 // (V * W))))
        return dict(op=op, B=B, W=W, V=V, n=min(W * rng.choice([1, 1, 2]), 64),
                    dtype=rng.choice(["float32", "float32", "bfloat16", "float16"]),
                    bias=rng.choice(["none", "shared", "group", "each"]), forced=rng.choice([0.0, 0.1]))
    if op == "reorder" and rng.random() < 0.5:
        L = _log_uniform(rng, 1, 1024)
        W = _log_uniform(rng, 1, 48)
        B = _log_uniform(rng, 1, max(1, min(64, 131072 // (L * W))))
        return dict(op=op, kind="design", B=B, W=W, L=L, t=rng.randint(0, L))
    if op == "reorder":
        D = rng.choice([32, 64, 80, 128])
        dtype = rng.choice(["bfloat16", "float16", "float32"])
        heads = rng.randint(1, 16)
        W = _log_uniform(rng, 2, 32)
        T = _log_uniform(rng, 1, 8192)
        B = _log_uniform(rng, 1, max(1, min(32, (134000000 if dtype != "float32" else 67000000) // (T * W * heads * D))))
        return dict(op=op, kind="cache", B=B, W=W, heads=heads, T=T, t=rng.randint(1, T), D=D, layers=rng.randint(1, 2),
                    dtype=dtype)
    largest = _log_uniform(rng, 100, 2000000)
    return dict(op=op, kind=rng.choice(["ragged", "even"]), tensors=_log_uniform(rng, 1, max(1, min(400, 50000000 // largest))),
                largest=largest, sizes=rng.randint(0, 10**6), step=rng.choice([1, 2, 10, 1000]),
                clip=rng.choice([0.0, 0.5, 1.0]))


# ---------------------------------------------------------------------------------------------------------------
# what a program has in hand
# ---------------------------------------------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _parents(B, W, g):
    """Parents as a selection leaves them: the better beams of a group have more of the next hypotheses."""
    return (W * torch.rand(B, W, device="cuda", generator=g) ** 1.5).long().clamp_(max=W - 1)


def _model_sizes():
    """Parameter sizes of the default model: hidden size 128, three encoder and three decoder layers, 21 letters."""
    H = 128
    sizes = [16 * 66, 16, H * 416, H, H, H * H, H, 21 * H, 21 * H, 21]
    for extra, norms, gates in ((3 * H, 3, 2), (4 * H, 2, 1)):
        layer = [H] * (2 * norms) + [H * extra, H, H * H, H, H * H, H] * gates + [4 * H * H, 4 * H, 4 * H * H, H]
        sizes += layer * 3
    return sizes


def _sizes(case):
    if case["kind"] == "model":
        return _model_sizes()
    n, top = case["tensors"], case["largest"]
    if case["kind"] == "even":
        return [max(1, top - 37 * i) for i in range(n)]
    u = np.random.RandomState(case["sizes"]).rand(n)
    return [max(1, int(top ** x)) for x in u[:-1]] + [top]


def _flat(sizes):
    """Element offsets of tensors that start at multiples of 64 elements of one buffer, and the buffer's size."""
    starts, at = [], 0
    for n in sizes:
        starts.append(at)
        at += -(-n // BLOCK) * BLOCK
    return starts, at


def _prepare_adamw(case, seed):
    g = _generator(seed)
    sizes = _sizes(case)
    wide = [n for n in sizes if n >= 4096]      # moments in 8 bits
    small = [n for n in sizes if n < 4096]      # moments in 32 bits
    s = dict(op="adamw", step=case["step"], clip=case["clip"], seed=seed & 0xFFFFFFFF)
    for tag, ns in (("8", wide), ("32", small)):
        starts, total = _flat(ns)
        real = torch.zeros(total, device="cuda")
        for a, n in zip(starts, ns):
            real[a:a + n] = 1.0
        p = torch.randn(total, device="cuda", generator=g) * 0.05 * real
        # gradients differ in size from tensor to tensor and inside one; some are exactly zero (letters that do not occur)
        size = torch.exp(2.0 * torch.randn(-(-total // BLOCK), device="cuda", generator=g)).repeat_interleave(BLOCK)[:total]
        grad = torch.randn(total, device="cuda", generator=g) * 1e-3 * size * real
        grad = grad * (torch.rand(total, device="cuda", generator=g) > 0.02)
        m = 0.3 * grad + 3e-4 * size * torch.randn(total, device="cuda", generator=g) * real
        v = (1e-3 * size) ** 2 * torch.exp(torch.randn(total, device="cuda", generator=g)) * real
        if case["step"] == 1:
            m, v = torch.zeros_like(m), torch.zeros_like(v)
        s["p" + tag], s["g" + tag] = p, grad
        cut = [slice(a, a + n) for a, n in zip(starts, ns)]
        s["cut" + tag] = cut
        if tag == "32":
            s["m32"], s["v32"] = m, v
        else:
            for name, x in (("m", m), ("v", v)):
                top = x.view(-1, BLOCK).abs().amax(1)
                scale = torch.where(top > 0, torch.exp2(torch.floor(torch.log2(top.clamp(min=1e-30))) - 7), torch.ones_like(top))
                codes = (x.view(-1, BLOCK) / scale[:, None]).to(torch.float8_e4m3fn)
                s[name + "8"], s[name + "8_scale"] = codes.view(-1), scale
            # the plain form works on whole blocks: the tensor a block belongs to, and where in it the block starts
            of = [torch.full((-(-n // BLOCK),), i, dtype=torch.int64) for i, n in enumerate(ns)]
            at = [torch.arange(0, n, BLOCK, dtype=torch.int64) for n in ns]
            s["block_tensor"] = torch.cat(of).cuda() if of else torch.zeros(0, dtype=torch.int64, device="cuda")
            s["block_start"] = torch.cat(at).cuda() if at else torch.zeros(0, dtype=torch.int64, device="cuda")
    # the lists of a training loop: parameters, gradients and the optimizer's state, one tensor each
    blocks = [slice(c.start // BLOCK, -(-c.stop // BLOCK)) for c in s["cut8"]]
    s["params"] = [s["p8"][c] for c in s["cut8"]] + [s["p32"][c] for c in s["cut32"]]
    s["grads"] = [s["g8"][c] for c in s["cut8"]] + [s["g32"][c] for c in s["cut32"]]
    s["exp_avgs"] = [s["m8"][c] for c in s["cut8"]] + [s["m32"][c] for c in s["cut32"]]
    s["exp_avg_sqs"] = [s["v8"][c] for c in s["cut8"]] + [s["v32"][c] for c in s["cut32"]]
    s["exp_avg_scales"] = [s["m8_scale"][b] for b in blocks] + [None] * len(small)
    s["exp_avg_sq_scales"] = [s["v8_scale"][b] for b in blocks] + [None] * len(small)
    return s


def prepare(case, seed):
    if case["op"] == "adamw":
        return _prepare_adamw(case, seed)
    g = _generator(seed)
    B, W = case["B"], case["W"]
    if case["op"] == "select":
        V = case["V"]
        logits = (2.5 * torch.randn(B, W, V, device="cuda", generator=g)).to(getattr(torch, case["dtype"]))
        scores = -torch.cumsum(torch.rand(B, W, device="cuda", generator=g), 1)
        scores[B // 2, 1:] = NEG                                    # a group at its first step: one beam is alive
        shape = {"none": None, "shared": (1, 1, V), "group": (B, 1, V), "each": (B, W, V)}[case["bias"]]
        bias = None
        if shape:                                                   # a fifth of the tokens is excluded
            bias = 0.1 * torch.randn(shape, device="cuda", generator=g)
            bias = bias.masked_fill_(torch.rand(shape, device="cuda", generator=g) < 0.2, NEG)
        forced = None
        if case["forced"]:                                          # groups at a fixed residue, finished hypotheses
            forced = torch.randint(0, V, (B, W), device="cuda", generator=g)
            forced = torch.where(torch.rand(B, W, device="cuda", generator=g) < case["forced"], forced, -torch.ones_like(forced))
        return dict(op="select", logits=logits, scores=scores, bias=bias, forced=forced, n=case["n"])
    parent = _parents(B, W, g)
    if case["kind"] == "design":
        L, H = case["L"], 128
        rows = [torch.randn(W, B, L, 2 * H, device="cuda", generator=g) for _ in range(3)]
        states = [x.transpose(0, 1)[..., H:] for x in rows]
        states.append(torch.randint(0, 21, (W, B, L), device="cuda", generator=g).transpose(0, 1))
        states.append(torch.randn(W, B, L, 21, device="cuda", generator=g).transpose(0, 1))
        rank = torch.argsort(torch.rand(B, L, device="cuda", generator=g), 1).to(torch.int32)
        return dict(op="reorder", states=states, parent=parent, length=case["t"], rank=rank)
    shape = (B, W, case["heads"], case["T"], case["D"])
    dtype = getattr(torch, case["dtype"])
    states = [torch.randn(shape, device="cuda", generator=g, dtype=dtype)[:, :, :, :case["t"]] for _ in range(2 * case["layers"])]
    return dict(op="reorder", states=states, parent=parent, length=None, rank=None)


# ---------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------
def _plain_select(s):
    """In 64 bits: the choice is a comparison, and candidates of different beams lie next to each other."""
    logits, scores, bias, forced, n = s["logits"], s["scores"].double(), s["bias"], s["forced"], s["n"]
    B, W, V = logits.shape
    x = logits.double()
    if bias is not None:
        x = torch.where(bias == NEG, torch.full_like(x, NEG), x + bias.double())
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == NEG, torch.zeros_like(top), top)
    lse = top + torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    c = torch.where(x == NEG, x, scores[..., None] + (x - lse))
    if forced is not None:
        place = torch.arange(V, device=x.device) == forced[..., None]
        c = torch.where(forced[..., None] < 0, c, torch.where(place, scores[..., None], torch.full_like(c, NEG)))
    value, at = torch.sort(c.view(B, W * V), dim=1, descending=True, stable=True)
    value, at = value[:, :n], at[:, :n]
    stay = (torch.arange(n, device=x.device) % W)[None].expand(B, n)    # a slot without a candidate keeps its beam
    none = torch.zeros_like(stay) if forced is None else forced.clamp(min=0).gather(1, stay)
    dead = value == NEG
    return value.float(), torch.where(dead, stay, at // V), torch.where(dead, none, at % V)


def _plain_reorder(s):
    parent, length, rank = s["parent"], s["length"], s["rank"]
    group = torch.arange(parent.shape[0], device=parent.device)[:, None]
    for x in s["states"]:
        moved = x[group, parent]
        if length is not None:
            live = (rank < length).view(rank.shape[0], 1, rank.shape[1], *([1] * (x.dim() - 3)))
            moved = torch.where(live, moved, x)
        x.copy_(moved)
    return s["states"]


LR, B1, B2, EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 1e-2


def _hash(x, key):
    """32 random bits for each number x < 2^32 (multiplication, then murmur3's published finalizer)."""
    low = 0xFFFFFFFF
    h = ((x * 0x9E3779B1) & low) ^ key
    h = ((h ^ (h >> 16)) * 0x85EBCA6B) & low
    h = ((h ^ (h >> 13)) * 0xC2B2AE35) & low
    return h ^ (h >> 16)


def _to_codes(x, r16, keep):
    """x in blocks of 64 as e4m3 codes and powers of two: a block's largest magnitude lies in [128, 256) scales, and each
    element goes up to the next code with the probability r16 / 65536 says.  keep: what is above zero stays above it."""
    top = x.abs().amax(1)
    power = torch.frexp(top)[1] - 1
    scale = torch.where(top > 0, torch.exp2((power - 7).clamp(min=-126).double()), torch.ones_like(top))
    scale = torch.where(torch.isfinite(top) & (power < 128), scale, torch.full_like(top, float("nan")))
    y = x.abs() / scale[:, None]
    step = torch.exp2(((torch.frexp(y)[1] - 1).clamp(min=-6) - 3).double())
    q = torch.floor(y / step + r16.double() * 2.0**-16) * step
    if keep:
        q = torch.where((q == 0) & (y > 0), torch.full_like(q, 2.0**-9), q)
    q = torch.where(q == 0, q, torch.copysign(q, x))
    return q.float().to(torch.float8_e4m3fn).view(-1), scale.float()


def _plain_adamw(s):
    """Moments in 64 bits up to their rounding (a value next to a border between two codes), the update in 32."""
    k = s["step"]
    coef = 1.0
    if s["clip"] > 0:
        sumsq = s["g8"].double().square().sum() + s["g32"].double().square().sum()
        coef = (s["clip"] / (sumsq.sqrt() + 1e-6)).clamp(max=1.0)

    def moments(g, m, v):
        g = g.double() * coef
        return B1 * m + (1.0 - B1) * g, B2 * v + (1.0 - B2) * (g * g)

    def update(p, m, v):
        rate, root = LR / (1.0 - B1**k), math.sqrt(1.0 - B2**k)
        m, v = m.float(), v.float()
        p.copy_(p * (1.0 - LR * DECAY) - rate * (m / (v.sqrt() / root + EPS)))

    m, v = moments(s["g32"], s["m32"].double(), s["v32"].double())
    update(s["p32"], m, v)
    s["m32"].copy_(m)
    s["v32"].copy_(v)

    decode = lambda c, scale: c.float().view(-1, BLOCK).double() * scale.double()[:, None]   # noqa: E731
    m, v = moments(s["g8"].view(-1, BLOCK), decode(s["m8"], s["m8_scale"]), decode(s["v8"], s["v8_scale"]))
    update(s["p8"].view(-1, BLOCK), m, v)
    key = _hash(s["block_tensor"], _hash(torch.full_like(s["block_tensor"], k), s["seed"]))
    r = _hash(s["block_start"][:, None] + torch.arange(BLOCK, device=m.device), key[:, None])
    if m.shape[0]:
        for name, x, bits in (("m8", m, r & 0xFFFF), ("v8", v, r >> 16)):
            codes, scale = _to_codes(x, bits, name == "v8")
            s[name].copy_(codes)
            s[name + "_scale"].copy_(scale)
    return [s[n] for n in ("p8", "m8", "m8_scale", "v8", "v8_scale", "p32", "m32", "v32")]


def run(s):
    if s["op"] == "select":
        if own:
            import mpnn_amd
            return mpnn_amd.beam_select(s["logits"], s["scores"], bias=s["bias"], forced=s["forced"], n_out=s["n"])
        return _plain_select(s)
    if s["op"] == "reorder":
        if own:
            import mpnn_amd
            return mpnn_amd.beam_reorder(s["states"], s["parent"], length=s["length"], rank=s["rank"])
        return _plain_reorder(s)
    if own:
        from mpnn_amd.optim import adamw_step
        adamw_step(s["params"], s["grads"], s["exp_avgs"], s["exp_avg_sqs"], s["exp_avg_scales"], s["exp_avg_sq_scales"],
                   step=s["step"], lr=LR, betas=(B1, B2), eps=EPS, weight_decay=DECAY, seed=s["seed"],
                   max_grad_norm=s["clip"])
        return [s[n] for n in ("p8", "m8", "m8_scale", "v8", "v8_scale", "p32", "m32", "v32")]
    return _plain_adamw(s)


# ---------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "select":
        B, W, V = case["B"], case["W"], case["V"]
        item = 4 if case["dtype"] == "float32" else 2
        bias = {"none": 0, "shared": V, "group": B * V, "each": B * W * V}[case["bias"]]
        forced = 8 * B * W if case["forced"] else 0
        return {"bytes": B * W * V * item + 4 * bias + forced + 4 * B * W + 20 * B * case["n"], "flops": 20.0 * B * W * V}
    if case["op"] == "reorder":
        B, W = case["B"], case["W"]
        if case["kind"] == "design":
            return {"bytes": 2 * B * W * case["t"] * (3 * 512 + 8 + 84) + 8 * B * W + 4 * B * case["L"] + 1, "flops": 0}
        item = 4 if case["dtype"] == "float32" else 2
        return {"bytes": 2 * 2 * case["layers"] * B * W * case["heads"] * case["t"] * case["D"] * item + 8 * B * W, "flops": 0}
    sizes = _sizes(case)
    wide, small = sum(n for n in sizes if n >= 4096), sum(n for n in sizes if n < 4096)
    again = 4 * (wide + small) if case["clip"] else 0    # the norm needs every gradient before the first is used
    return {"bytes": wide * (12 + 4 + 16.0 / BLOCK) + small * 28 + again, "flops": 30.0 * (wide + small)}


# ---------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits, written apart from the plain forms
# ---------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "select":
        B, W, V = s["logits"].shape
        out = torch.full((B, case["n"]), NEG, dtype=torch.float64)
        bias = None if s["bias"] is None else s["bias"].expand(B, W, V)
        for b in range(B):
            x = s["logits"][b].to(torch.float64)
            if bias is not None:
                x = x + bias[b].to(torch.float64)
            p = (torch.log_softmax(x, 1).nan_to_num(nan=NEG) + s["scores"][b].double()[:, None])
            if s["forced"] is not None:
                for w in (s["forced"][b] >= 0).nonzero().flatten().tolist():
                    p[w] = NEG
                    p[w, s["forced"][b, w]] = s["scores"][b, w].double()
            best = torch.topk(p.flatten(), min(case["n"], W * V)).values
            out[b, :best.numel()] = best.cpu()
        return out, None, None
    if case["op"] == "reorder":
        parent = s["parent"].tolist()
        out = []
        for x in s["states"]:
            if not x.is_floating_point():
                out.append(None)
                continue
            y = x.double()
            for b, row in enumerate(parent):
                if s["length"] is None:
                    y[b] = x[b].double().index_select(0, s["parent"][b])
                else:
                    live = (s["rank"][b] < s["length"]).nonzero().flatten()
                    for j, q in enumerate(row):
                        y[b, j].index_copy_(0, live, x[b, q].index_select(0, live).double())
            out.append(y)
        return out
    return _exact_adamw(case, s)


def _exact_adamw(case, s):
    grid = [0.0] + [2.0**-9 * i for i in range(1, 8)] + [2.0**e * (1 + f / 8.0) for e in range(-6, 9) for f in range(8)]
    grid = torch.tensor(grid, dtype=torch.float64, device="cuda")
    k = case["step"]
    norm = math.sqrt(float(sum((g.double() ** 2).sum() for g in s["grads"])))
    coef = min(1.0, case["clip"] / (norm + 1e-6)) if case["clip"] else 1.0

    def random_bits(i, key):
        h = (i.astype(np.uint32) * np.uint32(0x9E3779B1)) ^ np.uint32(key)
        h = (h ^ (h >> np.uint32(16))) * np.uint32(0x85EBCA6B)
        h = (h ^ (h >> np.uint32(13))) * np.uint32(0xC2B2AE35)
        return h ^ (h >> np.uint32(16))

    def rounded(x, u, keep):
        n = x.numel()
        pad = torch.nn.functional.pad(x, (0, -n % BLOCK)).view(-1, BLOCK)
        top = pad.abs().max(1).values
        scale = torch.tensor([2.0 ** max(math.frexp(t)[1] - 8, -126) if t else 1.0 for t in top.tolist()], dtype=torch.float64,
                             device="cuda")
        y = (pad.abs() / scale[:, None]).flatten()[:n]
        lower = torch.searchsorted(grid, y, right=True) - 1
        share = (y - grid[lower]) / (grid[lower + 1] - grid[lower])
        code = lower + (share + u >= 1.0).long()
        if keep:
            code = torch.where((code == 0) & (y > 0), torch.ones_like(code), code)
        return torch.sign(x) * grid[code], scale

    out = {n: torch.zeros_like(s[n], dtype=torch.float64) for n in ("p8", "m8", "m8_scale", "v8", "v8_scale", "p32", "m32", "v32")}
    key = int(random_bits(np.array([k]), s["seed"])[0])
    for i, g in enumerate(s["grads"]):
        wide = s["exp_avg_scales"][i] is not None
        n = g.numel()
        m, v = s["exp_avgs"][i].float().double(), s["exp_avg_sqs"][i].float().double()
        if wide:
            m = m * s["exp_avg_scales"][i].double().repeat_interleave(BLOCK)[:n]
            v = v * s["exp_avg_sq_scales"][i].double().repeat_interleave(BLOCK)[:n]
        g = g.double() * coef
        m, v = m + (1 - B1) * (g - m), v + (1 - B2) * (g * g - v)
        p = s["params"][i].double()
        p = p - LR * DECAY * p - LR * (m / (1 - B1**k)) / (torch.sqrt(v / (1 - B2**k)) + EPS)
        tag = "8" if wide else "32"
        cut = s["cut" + tag][i if wide else i - len(s["cut8"])]
        out["p" + tag][cut] = p
        if not wide:
            out["m32"][cut], out["v32"][cut] = m, v
            continue
        r = torch.from_numpy(random_bits(np.arange(n, dtype=np.uint32), random_bits(np.array([i]), key)[0]).astype(np.int64)).cuda()
        blocks = slice(cut.start // BLOCK, -(-cut.stop // BLOCK))
        out["m8"][cut], out["m8_scale"][blocks] = rounded(m, (r % 65536).double() / 65536, False)
        out["v8"][cut], out["v8_scale"][blocks] = rounded(v, (r // 65536).double() / 65536, True)
    return [out[n] for n in ("p8", "m8", "m8_scale", "v8", "v8_scale", "p32", "m32", "v32")]
