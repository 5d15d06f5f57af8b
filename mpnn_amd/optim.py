"""AdamW and gradient-norm clipping of the reference's training loop on the HIP library.

`AdamW` is `torch.optim.AdamW(lr, betas, eps, weight_decay)` as the reference constructs it (train.py:217; no amsgrad,
not maximize): same update, same `state_dict` layout (`step`, `exp_avg`, `exp_avg_sq` per parameter), so the
`optimizer_state_dict` of a reference checkpoint (train.py:548-568) loads.  One launch covers 48 parameter tensors
(`mpnn_adamw_step`); with `max_grad_norm` the clip of train.py:389-390 is folded into the same pass (the norm is
reduced on the device by `mpnn_grad_sumsq`, nothing synchronises with the host).  `clip_grad_norm_` is the stand-alone
form with torch's signature.  Parameters and gradients must be fp32 tensors on a ROCm device (no CPU fallback).

`AdamW(state_bits=8)` keeps the moments of large tensors in 8 bits (no counterpart in the reference): 2.1 bytes an element
instead of 8, and 16.25 bytes of traffic a step instead of 28.  A moment is an e4m3 code (`exp_avg`, `exp_avg_sq`:
torch.float8_e4m3fn, the parameter's shape) times a power of two for each 64 consecutive elements (`exp_avg_scale`,
`exp_avg_sq_scale`), rounded stochastically and reproducibly; `unpack_moment` / `pack_moment` convert, and checkpoints of
either width load into either optimizer.  `adamw_step` is the functional form over lists of tensors.
"""
from __future__ import annotations

import ctypes

import torch

from ._lib import call, host_call, ptr, stream_ptr


def _tables(tensors):
    n = len(tensors)
    return (ctypes.c_void_p * n)(*[t.data_ptr() for t in tensors])


def _check(tensors, what):
    for t in tensors:
        if not t.is_cuda or t.dtype != torch.float32 or not t.is_contiguous():
            raise RuntimeError(f"mpnn_amd.optim: {what} must be contiguous fp32 tensors on a ROCm device "
                               "(the HIP path has no CPU fallback)")


def grad_sumsq(grads):
    """Device scalar: sum of squares over all gradient elements (ceil(n / 48) + 1 launches; per-workgroup partials are
    added in a fixed tree, so the value - and the clip coefficient derived from it - is the same on every run)."""
    _check(grads, "gradients")
    dev = grads[0].device
    out = torch.empty(1, device=dev, dtype=torch.float32)
    sizes = [g.numel() for g in grads]
    numel = (ctypes.c_int * len(grads))(*sizes)
    need = sum(((max(sizes[k:k + 48]) + 2047) // 2048) * len(sizes[k:k + 48]) for k in range(0, len(sizes), 48))
    ws = torch.empty(need, device=dev, dtype=torch.float32)
    call("mpnn_grad_sumsq", len(grads), _tables(grads), numel, ptr(out), ptr(ws), need, stream_ptr())
    return out


def clip_grad_norm_(parameters, max_norm):
    """torch.nn.utils.clip_grad_norm_(parameters, max_norm) with the L2 norm: scales every `.grad` in place by
    min(1, max_norm / (total_norm + 1e-6)) and returns total_norm (a device tensor; no host synchronisation)."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [p.grad for p in parameters if p.grad is not None and p.grad.numel()]
    if not grads:
        return torch.zeros(())
    with torch.cuda.device(grads[0].device):
        ss = grad_sumsq(grads)
        numel = (ctypes.c_int * len(grads))(*[g.numel() for g in grads])
        call("mpnn_grad_scale", len(grads), _tables(grads), numel, ptr(ss), float(max_norm), stream_ptr())
    return ss.sqrt().reshape(())


BLOCK = 64      # elements of an 8-bit moment that share a scale


def pack_moment(x, positive=False):
    """fp32 tensor -> (e4m3 codes of its shape, scales [ceil(numel / 64)]): the stored form of an 8-bit moment, rounded to
    nearest (conversion of checkpoints; the step itself rounds stochastically).  positive: values above 0 do not become 0
    (second moments)."""
    n = x.numel()
    y = torch.nn.functional.pad(x.detach().to(torch.float32).reshape(-1), (0, -n % BLOCK)).view(-1, BLOCK)
    top = y.abs().amax(1) if n else y.new_zeros(0)
    e = (torch.frexp(top)[1] - 8).clamp(min=-126)
    scale = torch.where(top > 0, torch.exp2(e.double()).float(), torch.ones_like(top))
    scale = torch.where(torch.isfinite(top), scale, torch.full_like(top, float("nan")))
    q = y.double() / scale.double()[:, None]
    if positive:
        q = torch.where((q > 0) & (q < 2.0**-9), torch.full_like(q, 2.0**-9), q)
    q = q.nan_to_num(0.0, 0.0, 0.0)
    return q.float().to(torch.float8_e4m3fn).view(-1)[:n].view(x.shape), scale


def unpack_moment(codes, scale):
    """The fp32 values of an 8-bit moment."""
    n = codes.numel()
    return (codes.to(torch.float32).reshape(-1) * scale.repeat_interleave(BLOCK)[:n]).view(codes.shape)


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, exp_avg_scales, exp_avg_sq_scales, *, step, lr=1e-3,
               betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, seed=0, max_grad_norm=0.0):
    """One AdamW step over lists of tensors, in place.  params, grads: contiguous fp32.  Tensors whose scales are None keep
    fp32 moments; the others hold float8_e4m3fn codes and fp32 scales (see the module's docstring; zeros and ones to begin
    with).  step: 1 for the first.  seed, step, the place in the list and the element decide the rounding of 8-bit moments.
    max_grad_norm > 0 clips by the norm over all gradients.  Returns the squared norm (a device scalar) then, else None.
    No two tensors may share memory, but for gradients among themselves.  A replayed HIP graph of this call repeats its step and
    its hyper-parameters."""
    return host_call("mpnn_adamw_mixed", "adamw", params, grads, exp_avgs, exp_avg_sqs, exp_avg_scales, exp_avg_sq_scales, step,
                     lr, betas[0], betas[1], eps, weight_decay, int(seed) & 0xFFFFFFFF, 0, max_grad_norm, None)


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW on the HIP library.  state_bits=8: moments of tensors with at least `min_8bit_numel` elements are
    held in 8 bits (the others in 32), rounded by `seed`; the step then counts from each parameter's own state, on the host,
    so it cannot be captured into a HIP graph."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, max_grad_norm=0.0, state_bits=32,
                 min_8bit_numel=4096, seed=0):
        if state_bits not in (8, 32):
            raise ValueError("mpnn_amd.optim.AdamW: state_bits is 8 or 32")
        if lr < 0 or eps < 0 or not 0 <= betas[0] < 1 or not 0 <= betas[1] < 1 or weight_decay < 0:
            raise ValueError("mpnn_amd.optim.AdamW: invalid hyper-parameter")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, amsgrad=False,
                                      maximize=False, foreach=None, capturable=False, differentiable=False,
                                      fused=None, decoupled_weight_decay=True))
        self.max_grad_norm = float(max_grad_norm)
        self.state_bits, self.min_8bit_numel, self.seed = state_bits, int(min_8bit_numel), int(seed)
        self._counts, self._steps, self._at = None, [], {}  # 8-bit moments: see _gather_counts
        self.last_grad_sumsq = None  # device scalar of the last step (its square root is the unclipped gradient norm)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        live = [[p for p in g["params"] if p.grad is not None and p.numel()] for g in self.param_groups]
        every = [p for ps in live for p in ps]
        if not every:
            return loss
        if self.state_bits == 8:
            self._step_mixed(live, every)
            return loss
        _check(every, "parameters")
        _check([p.grad for p in every], "gradients")
        with torch.cuda.device(every[0].device):
            ss = None
            if self.max_grad_norm > 0.0:  # the clip norm spans every group, as clip_grad_norm_(model.parameters()) does
                ss = self.last_grad_sumsq = grad_sumsq([p.grad for p in every])
            for group, ps in zip(self.param_groups, live):
                if not ps:
                    continue
                steps = set()
                for p in ps:
                    st = self.state[p]
                    if not st:
                        st["step"] = torch.tensor(0.0)
                        st["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                        st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                    st["step"] += 1
                    steps.add(int(st["step"]))
                # parameters that joined later have their own bias correction: one call per distinct step count
                for k in sorted(steps):
                    sel = [p for p in ps if int(self.state[p]["step"]) == k]
                    m = [self.state[p]["exp_avg"] for p in sel]
                    v = [self.state[p]["exp_avg_sq"] for p in sel]
                    _check(m + v, "optimizer state")
                    numel = (ctypes.c_int * len(sel))(*[p.numel() for p in sel])
                    lr = group["lr"]
                    call("mpnn_adamw_step", len(sel), _tables(sel), _tables([p.grad for p in sel]), _tables(m), _tables(v),
                         numel, float(lr), float(group["betas"][0]), float(group["betas"][1]), float(group["eps"]),
                         float(group["weight_decay"]), k, ptr(ss), self.max_grad_norm, stream_ptr())
            # the kernels write the parameters behind autograd's back: bump the version counters, which key the
            # inference kernels' packed-weight cache (engine.PackedWeights) and guard saved tensors
            try:
                torch.autograd.graph.increment_version(every)
            except (AttributeError, TypeError):
                for p in every:
                    torch.autograd.graph.increment_version(p) if hasattr(torch.autograd.graph, "increment_version") else None
        return loss

    def _new_state(self, p):
        st = {"step": torch.tensor(0.0)}
        if p.numel() < self.min_8bit_numel:
            st["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
            st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
            return st
        for name in ("exp_avg", "exp_avg_sq"):
            st[name] = torch.zeros(p.shape, device=p.device, dtype=torch.float8_e4m3fn)
            st[name + "_scale"] = torch.ones(-(-p.numel() // BLOCK), device=p.device, dtype=torch.float32)
        return st

    def _step_mixed(self, live, every):
        if every[0].is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("mpnn_amd.optim.AdamW(state_bits=8): a step counts on the host and cannot be captured into a HIP "
                               "graph")
        parts, self.last_grad_sumsq = None, None
        grads = [[p.grad for p in ps] for ps in live]
        if self.max_grad_norm > 0.0:
            parts = host_call("mpnn_grad_sumsq_parts", "grad_sumsq_parts", [g for gs in grads for g in gs])
        states = [[self.state[p] for p in ps] for ps in live]
        places = lambda: [[self._at.get(id(st.get("step"))) for st in sts] for sts in states]   # noqa: E731
        at_of = places()
        if any(None in at for at in at_of):
            for ps, sts in zip(live, states):
                for p, st in zip(ps, sts):
                    if not st:
                        st.update(self._new_state(p))
            self._gather_counts()
            at_of = places()
        counts, first = self._counts.tolist(), 0
        for group, *own, at in zip(self.param_groups, live, grads, states, at_of):
            taken = [counts[i] for i in at]
            for k in sorted(set(taken)):
                sel = (*own, at)
                if taken.count(k) < len(taken):
                    sel = [[x for x, c in zip(xs, taken) if c == k] for xs in sel]
                ps, gs, sts, places_k = sel
                lists = [[st.get(n) for st in sts] for n in ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")]
                ss = host_call("mpnn_adamw_mixed", "adamw", ps, gs, *lists, int(k) + 1, group["lr"], group["betas"][0],
                               group["betas"][1], group["eps"], group["weight_decay"], self.seed & 0xFFFFFFFF, first,
                               self.max_grad_norm, parts)
                self.last_grad_sumsq = ss if ss is not None else self.last_grad_sumsq
                first += len(ps)
                i = places_k[0]
                if places_k == list(range(i, i + len(ps))):
                    self._counts[i:i + len(ps)] += 1
                else:
                    self._counts[places_k] += 1

    def _gather_counts(self):
        """Make every parameter's `step` an element of one tensor: an operation counts for all (adding to each of 118 tensors
        costs more than the kernels), and a program that writes one of them restarts that parameter alone.  Done whenever a
        state holds a `step` that is not such an element (a new parameter, a loaded state, one that a program put there)."""
        states = [st for st in self.state.values() if "step" in st]
        self._counts = torch.tensor([float(st["step"]) for st in states], dtype=torch.float32, device="cpu")
        self._steps = [self._counts[i] for i in range(len(states))]   # kept: their ids are the keys of _at
        self._at = {id(s): i for i, s in enumerate(self._steps)}
        for st, s in zip(states, self._steps):
            st["step"] = s

    def state_dict(self):
        """As torch's; with 8-bit moments every parameter gets a `step` tensor of its own (an optimizer that adds to them in
        place may load it)."""
        sd = super().state_dict()
        if self.state_bits == 8:
            sd["state"] = {k: {**st, "step": st["step"].clone()} for k, st in sd["state"].items()}
        return sd

    def load_state_dict(self, state_dict):
        """Checkpoints of 8-bit and of 32-bit moments (this optimizer's, torch's) load into an optimizer of either width.  With
        8-bit moments the state is copied: codes, scales and counts of two optimizers may not get out of step."""
        super().load_state_dict(state_dict)
        for p, st in self.state.items():
            if "exp_avg" not in st:
                continue
            wide = self.state_bits == 8 and p.numel() >= self.min_8bit_numel
            for name in ("exp_avg", "exp_avg_sq"):
                scale = st.pop(name + "_scale", None)
                if scale is None:
                    if wide:
                        st[name], st[name + "_scale"] = pack_moment(st[name], name == "exp_avg_sq")
                    elif self.state_bits == 8:
                        st[name] = st[name].clone()
                elif wide:   # torch has cast the codes to the parameter's type, without loss
                    st[name], st[name + "_scale"] = st[name].to(torch.float8_e4m3fn), scale.clone()
                else:
                    st[name] = unpack_moment(st[name], scale)
        if self.state_bits == 8:
            self._gather_counts()   # torch hands on the source's own `step` tensors, which their owner may add to in place
