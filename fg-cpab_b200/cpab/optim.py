"""AdamW over all tensors of a network, one kernel launch for those of one type
and state kind (256 at most), its states in 32 or 8 bits.

    m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2
    p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)

in float32 whatever the parameters' type.  8-bit states are e4m3 codes of m
and of sqrt(v) with one float32 scale per 256 elements, rounded
stochastically (their averages move by less than a code's spacing per step,
so rounding to nearest would stop them).  No counterpart in the reference.
"""
import torch

from . import _ext, _native

SCALE_BLOCK = 256  # elements of an 8-bit state that share a scale


def adamw_(params, grads, exp_avgs, exp_avg_sqs, steps, *, lr, betas=(0.9, 0.999), eps=1e-8,
           weight_decay=0.01, scales=None, seed=0, workspace=None):
    """One AdamW step over lists of CUDA tensors, in place.  params and grads
    float32, float16 or bfloat16; steps: one float32 element each (its own), the
    steps taken so far, counted up by the call.  A parameter's states are both
    float32, or both float8_e4m3fn codes (exp_avg_sqs then holds those of the
    second moment's square root) with scales[i] float32 [ceil(numel / 256), 2]
    (columns: first moment, root).  lr: a number, or one float32 on the params'
    device (a schedule inside a captured graph).  seed chooses the random bits of the
    8-bit rounding.  workspace: one int32, 0 (a program that steps often
    keeps one; calls that overlap on the GPU need one each)."""
    _step([(params, grads, exp_avgs, exp_avg_sqs, scales, steps, lr, betas, eps, weight_decay)],
          seed, workspace)


def _step(groups, seed, workspace):
    """One call over groups of (params, grads, exp_avgs, exp_avg_sqs, scales
    or None, steps, lr, betas, eps, weight_decay)."""
    p, g, m, v, sc, st, counts, hyper, lrs = [], [], [], [], [], [], [], [], []
    any_scales = any(q[4] is not None for q in groups)
    for params, grads, ms, vs, scales, steps, lr, betas, eps, wd in groups:
        n = len(params)
        if not (len(grads) == len(ms) == len(vs) == len(steps) == n) or \
                (scales is not None and len(scales) != n):
            raise ValueError("adamw: lists of different lengths")
        p += params
        g += grads
        m += ms
        v += vs
        st += steps
        if any_scales:
            sc += scales if scales is not None else [None] * n
        counts.append(n)
        on_device = torch.is_tensor(lr)
        if on_device and (not lr.is_cuda or lr.dtype != torch.float32 or lr.numel() != 1):
            raise ValueError("lr must be a number or one float32 element on the device")
        if on_device and n and lr.device != params[0].device:
            raise ValueError("lr is on %s, the parameters on %s" % (lr.device, params[0].device))
        lrs.append(lr if on_device else None)
        hyper += [0.0 if on_device else float(lr), float(betas[0]), float(betas[1]), float(eps), float(wd)]
    if not p:
        return
    if workspace is None:
        workspace = torch.zeros(1, device=p[0].device, dtype=torch.int32)
    elif workspace.dtype != torch.int32 or workspace.device != p[0].device or workspace.numel() < 1:
        raise ValueError("workspace must be one int32 on the parameters' device")
    ext = _ext.module()
    if ext is None:
        _native.adamw(p, g, m, v, sc, st, counts, hyper, lrs, int(seed), workspace)
    else:
        _ext.call(ext.adamw, p, g, m, v, sc, st, counts, hyper, lrs, int(seed) & 0xFFFFFFFF, workspace)


def _capturing():
    return torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing()


class AdamW(torch.optim.Optimizer):
    """lr, betas, eps and weight_decay of torch.optim.AdamW's constructor (not
    amsgrad, maximize nor the choices of its implementations), its state names
    (step, exp_avg, exp_avg_sq) and state dicts, with the step of adamw_; step()
    can be captured in a CUDA graph (counts and, if given as a tensor, lr live on
    the device) once the parameters have states, that is after one step.

    state_bits=8 keeps the states of parameters of at least min_8bit_size
    elements as e4m3 codes (state names exp_avg, root_avg_sq, scales): 2.03
    instead of 8 bytes per parameter.  seed: of their stochastic rounding (an
    option of the groups, so that state_dict keeps it and a resumed run rounds as
    it would have)."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, *,
                 state_bits=32, min_8bit_size=4096, seed=0):
        if not torch.is_tensor(lr) and not lr >= 0:
            raise ValueError("lr must not be negative, got %r" % (lr,))
        if not all(0.0 <= b < 1.0 for b in betas):
            raise ValueError("betas must be in [0, 1), got %r" % (betas,))
        if not eps >= 0 or not weight_decay >= 0:
            raise ValueError("eps and weight_decay must not be negative")
        if state_bits not in (8, 32):
            raise ValueError("state_bits must be 8 or 32, got %r" % (state_bits,))
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay,
                                      state_bits=state_bits, min_8bit_size=min_8bit_size,
                                      seed=int(seed)))
        self._workspace = {}

    def __setstate__(self, state):
        # (of copies and pickles, which hold the options, groups and states only)
        super().__setstate__(state)
        self.__dict__.setdefault("_workspace", {})
        for options in (self.defaults, *self.param_groups):
            options.setdefault("seed", 0)

    @property
    def seed(self):
        """The first group's; setting it sets every group's."""
        return self.param_groups[0]["seed"]

    @seed.setter
    def seed(self, value):
        for group in self.param_groups:
            group["seed"] = int(value)

    def _state(self, p, group):
        state = self.state[p]
        if not state:
            if _capturing():
                raise RuntimeError("AdamW: a parameter without a state in a captured step: every replay "
                                   "would begin anew; take one step, or load states, before the capture")
            state["step"] = torch.zeros((), device=p.device, dtype=torch.float32)
            eight = group["state_bits"] == 8 and p.numel() >= group["min_8bit_size"]
            kind = torch.float8_e4m3fn if eight else torch.float32
            state["exp_avg"] = torch.zeros_like(p, dtype=kind, memory_format=torch.preserve_format)
            state["root_avg_sq" if eight else "exp_avg_sq"] = torch.zeros_like(
                p, dtype=kind, memory_format=torch.preserve_format)
            if eight:
                blocks = (p.numel() + SCALE_BLOCK - 1) // SCALE_BLOCK
                state["scales"] = torch.zeros(blocks, 2, device=p.device, dtype=torch.float32)
        return state

    @torch.no_grad()
    def step(self, closure=None):
        """One step over every parameter that has a gradient."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        calls = {}  # by device and seed
        for group in self.param_groups:
            lists = {}
            for p in group["params"]:
                g = p.grad
                if g is None:
                    continue
                if g.is_sparse:
                    raise RuntimeError("AdamW does not take sparse gradients")
                s = self.state[p]
                if not s:
                    s = self._state(p, group)
                to = lists.get(p.device)
                if to is None:
                    to = lists[p.device] = ([], [], [], [], [], [])
                scales = s.get("scales")
                to[0].append(p)
                to[1].append(g)
                to[2].append(s["exp_avg"])
                to[3].append(s["exp_avg_sq"] if scales is None else s["root_avg_sq"])
                to[4].append(scales)
                to[5].append(s["step"])
            for device, to in lists.items():
                scales = to[4] if any(t is not None for t in to[4]) else None
                lr = group["lr"]
                if torch.is_tensor(lr) and lr.is_cuda and lr.device != device:
                    lr = lr.to(device, non_blocking=True)
                calls.setdefault((device, group["seed"]), []).append(
                    (*to[:4], scales, to[5], lr, group["betas"], group["eps"], group["weight_decay"]))
        for (device, seed), groups in calls.items():
            workspace = self._workspace.get(device)
            if workspace is None:
                workspace = torch.zeros(1, device=device, dtype=torch.int32)
                if not _capturing():  # (there it is 0 in replays only)
                    self._workspace[device] = workspace
            _step(groups, seed, workspace)
        return loss

    def load_state_dict(self, state_dict):
        """As torch's, which casts states to their parameter's type: the
        states' own types are put back (float32 for 16-bit moments of torch's
        AdamW).  Options that a saved group lacks stay as they are; amsgrad and
        maximize, which this step does not have, are refused."""
        groups = state_dict["param_groups"]
        for option in ("amsgrad", "maximize"):
            if any(saved.get(option) for saved in groups):
                raise ValueError("AdamW has no %s, which the state dict asks for" % option)
        if len(groups) == len(self.param_groups):
            groups = [{**{k: own[k] for k in self.defaults if k in own}, **saved}
                      for own, saved in zip(self.param_groups, groups)]
        super().load_state_dict({**state_dict, "param_groups": groups})
        params = [p for g in self.param_groups for p in g["params"]]
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        for i, p in zip(ids, params):
            saved = state_dict["state"].get(i)
            if saved:
                for k, v in saved.items():
                    if torch.is_tensor(v):
                        kind = v.dtype if v.dtype == torch.float8_e4m3fn else torch.float32
                        self.state[p][k] = v.detach().to(p.device, kind, copy=True)
