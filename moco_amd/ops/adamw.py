"""AdamW over many tensors, with the moments in 32 or in 8 bits, and the
gradient norm over many tensors.

Beside FusedSGD and MultiTensorEMA (multi_tensor.py), and like them a few
launches for the whole list (ops/hip/adamw.hip), with a plain-PyTorch path on
CPU.  The reference trains with SGD only (main_moco.py:205-208); AdamW is what
encoders with token norms are trained with.

One step, for weight p with gradient g::

    g    = grad * min(1, max_norm / (total_norm + 1e-6))      (if clipped)
    m    = beta1 * m + (1 - beta1) * g
    v    = beta2 * v + (1 - beta2) * g * g
    p    = p * (1 - lr * weight_decay)
           - lr / (1 - beta1^step) * m / (sqrt(v) / sqrt(1 - beta2^step) + eps)

Everything is computed in 32 bits; a 16-bit weight is rounded to nearest once,
at the end, so an update below half a step of a bf16 weight (2^-9 of it) is
lost, as it is with torch.optim.AdamW.

8-bit moments.  Every 256 consecutive elements (in memory order) share two
scales.  m is an e4m3 code (rounded to nearest) times scales[:, 0].  v is kept
as its root, an unsigned code with 4 exponent and 4 fraction bits times
scales[:, 1]: the root has half the octaves of v, so the codes' 19 octaves
reach 2^-38 of a block's largest v.  The root is rounded stochastically, by a
hash of (seed, step, number in the list, element): with beta2 = 0.999 one step
moves it by some 0.05%, codes are 3 to 6% apart, and rounding to nearest would
hold it still.  A v above zero keeps a code above zero.  A gradient that is
not finite reaches the scale, so all 256 elements of its block.

On the GPU torch.jit.trace and make_fx of these functions, and fake tensors,
are errors.
"""

import math
from typing import List, Optional, Sequence, Tuple

import torch

from . import ext, use_hip

BLOCK = 256
_TOP_M, _TOP_R, _TINY = 448.0, 1.9375, 1e-30
_FLOATS = (torch.float32, torch.bfloat16, torch.float16)

Tensors = Sequence[torch.Tensor]


# ---------------------------------------------------------------------------
# layout
# ---------------------------------------------------------------------------

def _is_dense(t: torch.Tensor) -> bool:
    """Non-overlapping and without gaps, in any order of the dimensions."""
    if t.numel() == 0:
        return True
    want = 1
    for stride, size in sorted((st, sz) for st, sz in
                               zip(t.stride(), t.shape) if sz != 1):
        if stride != want:
            return False
        want *= size
    return True


def _same_layout(a: torch.Tensor, b: torch.Tensor) -> bool:
    return a.shape == b.shape and (a.stride() == b.stride() or all(
        sz <= 1 or x == y for sz, x, y in
        zip(a.shape, a.stride(), b.stride())))


def _flat(t: torch.Tensor) -> torch.Tensor:
    """A dense tensor's elements in memory order."""
    return t.as_strided((t.numel(),), (1,))


def _check_overlap(tensors) -> None:
    """tensors: (tensor, written) pairs of one call."""
    spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(),
                    w) for t, w in tensors if t.numel())
    wrote = read = 0
    for begin, end, w in spans:
        if begin < wrote or (w and begin < read):
            raise ValueError("the tensors of one call must not share memory")
        if w:
            wrote = max(wrote, end)
        else:
            read = max(read, end)


def _check_step(step, lr, betas, eps, weight_decay, max_norm, total_norm):
    if int(step) != step or step < 1:
        raise ValueError(f"step counts from 1, got {step}")
    if not lr >= 0.0 or not eps >= 0.0 or not weight_decay >= 0.0:
        raise ValueError("lr, eps and weight_decay must not be negative, got "
                         f"{lr}, {eps}, {weight_decay}")
    if len(betas) != 2 or not all(0.0 <= b < 1.0 for b in betas):
        raise ValueError(f"betas must be two numbers in [0, 1), got {betas}")
    if max_norm is None:
        if total_norm is not None:
            raise ValueError("total_norm is used with max_norm only")
    elif not max_norm >= 0.0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")


def _check_scales(s: torch.Tensor, like: torch.Tensor, i: int) -> None:
    rows = -(-like.numel() // BLOCK)
    if s.device != like.device or s.dtype != torch.float32 or \
            not s.is_contiguous() or s.shape != (rows, 2):
        raise ValueError(f"scales {i} must be contiguous float32 "
                         f"[{rows}, 2]")


def _check_lists(params, grads, ms, vs, scales, total_norm):
    n = len(params)
    if any(len(x) != n for x in (grads, ms, vs)) or \
            (scales is not None and len(scales) != n):
        raise ValueError("the lists of tensors differ in length")
    m_type, v_type = (torch.float32,) * 2 if scales is None else \
        (torch.float8_e4m3fn, torch.uint8)
    spans = []
    for i, (p, g, m, v) in enumerate(zip(params, grads, ms, vs)):
        if p.dtype not in _FLOATS:
            raise TypeError("params must be float32, bfloat16 or float16, "
                            f"got {p.dtype}")
        if g.dtype != p.dtype:
            raise TypeError(f"gradient {i} is {g.dtype}, its parameter "
                            f"{p.dtype}")
        if g.layout != torch.strided:
            raise ValueError("sparse gradients are not supported")
        if m.dtype != m_type or v.dtype != v_type:
            raise TypeError(f"the moments must be {m_type} and {v_type}")
        if any(t.device != params[0].device for t in (p, g, m, v)):
            raise ValueError("all tensors must be on one device")
        if not _is_dense(p) or not all(_same_layout(p, t) for t in (g, m, v)):
            raise ValueError(f"parameter {i}, its gradient and its moments "
                             "must be dense and laid out alike")
        spans += [(p, True), (g, False), (m, True), (v, True)]
        if scales is not None:
            _check_scales(scales[i], p, i)
            spans.append((scales[i], True))
    if params and total_norm is not None:
        if total_norm.numel() != 1 or total_norm.dtype != torch.float32 \
                or total_norm.device != params[0].device:
            raise ValueError("total_norm must be one float32 on the tensors' "
                             "device")
        spans.append((total_norm, False))
    _check_overlap(spans)


# ---------------------------------------------------------------------------
# 8-bit codes (plain; the kernels do the same per block)
# ---------------------------------------------------------------------------

def _blocks(flat: torch.Tensor) -> torch.Tensor:
    pad = -flat.numel() % BLOCK
    return torch.nn.functional.pad(flat, (0, pad)).view(-1, BLOCK)


def _decode_root(code: torch.Tensor) -> torch.Tensor:
    return (code.to(torch.int32) << 19).view(torch.float32) * 2.0 ** 112


def _dither(n: int, key: int, device) -> torch.Tensor:
    """19 random bits for each of n elements (the kernels' hash)."""
    mask = 0xFFFFFFFF
    x = (torch.arange(n, dtype=torch.int64, device=device) + key) & mask
    x = (x * 0x9E3779B9) & mask
    x = x ^ (x >> 15)
    x = (x * 0xBB67AE85) & mask
    x = x ^ (x >> 16)
    return (x >> 13).to(torch.int32)


def _encode(m: torch.Tensor, r: torch.Tensor, key: Optional[int]):
    """Codes and scales of flat 32-bit m and r = sqrt(v); r is rounded to
    nearest where key is None."""
    n = m.numel()
    m, r = _blocks(m), _blocks(r)
    sm = m.abs().amax(1, keepdim=True).clamp_min(_TINY) * (1 / _TOP_M)
    sr = r.amax(1, keepdim=True).clamp_min(_TINY) * (1 / _TOP_R)
    # an infinity in a block makes all of it a NaN
    sm, sr = (t.masked_fill(t == math.inf, math.nan) for t in (sm, sr))
    mc = (m * sm.reciprocal()).clamp(-_TOP_M, _TOP_M).to(torch.float8_e4m3fn)
    q = r * sr.reciprocal()
    dither = 1 << 18 if key is None else \
        _dither(q.numel(), key, q.device).view_as(q)
    rc = (((q * 2.0 ** -112).view(torch.int32) + dither) >> 19).clamp(0, 255)
    rc = torch.where(q > 0, rc.clamp_min(1), torch.zeros_like(rc))
    return (mc.view(-1)[:n], rc.to(torch.uint8).view(-1)[:n],
            torch.cat([sm, sr], 1))


def _decode(m: torch.Tensor, v: torch.Tensor, scales: torch.Tensor):
    """Flat 32-bit (m, sqrt(v)) of dense codes, in memory order."""
    s = scales.repeat_interleave(BLOCK, 0)[:m.numel()]
    return _flat(m).float() * s[:, 0], _decode_root(_flat(v)) * s[:, 1]


# ---------------------------------------------------------------------------
# functional forms
# ---------------------------------------------------------------------------

def grad_norm(grads: Tensors) -> torch.Tensor:
    """2-norm over all elements of all tensors, as a float32 scalar on their
    device (no host sync).  Squares and sums are taken in 64 bits.

    grads: float32, bfloat16 or float16 tensors on one device, of any shapes,
    strides and mix of types.
    """
    grads = list(grads)
    if not grads:
        raise ValueError("grad_norm needs at least one tensor")
    if use_hip(*grads[:1]):
        return ext().grad_norm(grads, False)
    for g in grads:
        if g.layout != torch.strided:
            raise ValueError("sparse gradients are not supported")
        if g.dtype not in _FLOATS:
            raise TypeError("gradients must be float32, bfloat16 or float16, "
                            f"got {g.dtype}")
        if g.device != grads[0].device:
            raise ValueError("gradients must be on one device")
    with torch.no_grad():
        return torch.stack([g.double().square().sum() for g in grads]
                           ).sum().sqrt().float()


def _plain_step(params, grads, ms, vs, scales, step, lr, betas, eps,
                weight_decay, max_norm, total_norm, seed):
    coef = None
    if max_norm is not None:
        if total_norm is None:
            total_norm = grad_norm(grads)
        coef = (torch.full_like(total_norm, max_norm)
                / (total_norm + 1e-6)).clamp(max=1.0).reshape(())
    b1, b2 = betas
    inv_root = 1.0 / math.sqrt(1.0 - b2 ** step)
    step_size = lr / (1.0 - b1 ** step)
    key = seed * 0x6A09E667 + step * 0xA54FF53A
    for i, (p, g, m8, v8) in enumerate(zip(params, grads, ms, vs)):
        if p.numel() == 0:
            continue
        gf = _flat(g).float()
        if coef is not None:
            gf = gf * coef
        if scales is None:
            m, v = _flat(m8), _flat(v8)
        else:
            m, r = _decode(m8, v8, scales[i])
            v = r * r
        m = m * b1 + gf * (1.0 - b1)
        v = v * b2 + (gf * gf) * (1.0 - b2)
        r = v.sqrt()
        q = m / (r * inv_root + eps)
        _flat(p).copy_(_flat(p).float() * (1.0 - lr * weight_decay)
                       - q * step_size)
        if scales is not None:
            m, v, s = _encode(m, r, (key + i * 0x3C6EF372) & 0xFFFFFFFF)
            scales[i].copy_(s)
        _flat(m8).copy_(m)
        _flat(v8).copy_(v)
    return total_norm


def _adamw(params, grads, ms, vs, scales, step, lr, betas, eps, weight_decay,
           max_norm, total_norm, seed):
    _check_step(step, lr, betas, eps, weight_decay, max_norm, total_norm)
    params, grads = list(params), list(grads)
    if use_hip(*params[:1]):
        return ext().adamw_step(
            params, grads, ms, vs, scales, int(step), lr, betas[0], betas[1],
            eps, weight_decay, max_norm, total_norm, seed & 0xFFFFFFFF)
    _check_lists(params, grads, ms, vs, scales, total_norm)
    if not params:
        return total_norm
    # as the GPU's entry point takes them: a numpy or torch scalar would round
    # what is computed of it to its own type
    lr, eps, weight_decay = float(lr), float(eps), float(weight_decay)
    betas = tuple(float(b) for b in betas)
    max_norm = None if max_norm is None else float(max_norm)
    with torch.no_grad():
        return _plain_step(params, grads, ms, vs, scales, int(step), lr, betas,
                           eps, weight_decay, max_norm, total_norm, int(seed))


def adamw_(params: Tensors, grads: Tensors, exp_avgs: Tensors,
           exp_avg_sqs: Tensors, *, step: int, lr: float,
           betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
           weight_decay: float = 0.01, max_norm: Optional[float] = None,
           total_norm: Optional[torch.Tensor] = None
           ) -> Optional[torch.Tensor]:
    """One AdamW step in place, over lists of tensors.

    params, grads: float32, bfloat16 or float16, a gradient of its
        parameter's type; exp_avgs, exp_avg_sqs: float32.  The four of one
        parameter are dense and laid out alike (in any memory format), all on
        one device, and what is written shares no memory (a gradient may be
        given for several parameters).
    step: counts from 1.
    max_norm: scales the gradients (where they are used, not in memory) by
        min(1, max_norm / (norm + 1e-6)).  norm is `total_norm`, a float32
        scalar on the device such as grad_norm gives, or that of `grads`.

    Returns the norm that the clip went by (None without one).  In a captured
    graph step, lr and the other numbers are those of the capture.
    """
    return _adamw(params, grads, exp_avgs, exp_avg_sqs, None, step, lr, betas,
                  eps, weight_decay, max_norm, total_norm, 0)


def adamw8bit_(params: Tensors, grads: Tensors, exp_avgs: Tensors,
               exp_avg_sqs: Tensors, scales: Tensors, *, step: int, lr: float,
               betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 0.01, max_norm: Optional[float] = None,
               total_norm: Optional[torch.Tensor] = None, seed: int = 0
               ) -> Optional[torch.Tensor]:
    """adamw_ with the moments in 8 bits.

    exp_avgs: float8_e4m3fn codes, exp_avg_sqs: uint8 codes, laid out as
        their parameter; scales: contiguous float32 [ceil(numel / 256), 2].
        All zeros is the state before the first step.
    seed: of the stochastic rounding of sqrt(v); the step is hashed with it.
    """
    return _adamw(params, grads, exp_avgs, exp_avg_sqs, scales, step, lr,
                  betas, eps, weight_decay, max_norm, total_norm, seed)


def adamw8bit_values(exp_avgs: Tensors, exp_avg_sqs: Tensors, scales: Tensors,
                     dtype: torch.dtype = torch.float32
                     ) -> Tuple[List[torch.Tensor], List[torch.Tensor]]:
    """(m, v) that adamw8bit_'s codes stand for, laid out as they are."""
    if dtype not in _FLOATS:
        raise TypeError(f"values are float32, bfloat16 or float16, not "
                        f"{dtype}")
    exp_avgs = list(exp_avgs)
    if use_hip(*exp_avgs[:1]):
        ms, vs = ext().adamw8bit_values(exp_avgs, exp_avg_sqs, scales, dtype)
        return ms, vs
    if len(exp_avg_sqs) != len(exp_avgs) or len(scales) != len(exp_avgs):
        raise ValueError("the lists of tensors differ in length")
    for i, (m, v, sc) in enumerate(zip(exp_avgs, exp_avg_sqs, scales)):
        if m.dtype != torch.float8_e4m3fn or v.dtype != torch.uint8:
            raise TypeError("the codes must be float8_e4m3fn and uint8")
        if m.device != exp_avgs[0].device or v.device != m.device:
            raise ValueError("all tensors must be on one device")
        if not _is_dense(m) or not _same_layout(m, v):
            raise ValueError(f"codes {i} must be dense and laid out alike")
        _check_scales(sc, m, i)
    ms, vs = [], []
    for m, v, s in zip(exp_avgs, exp_avg_sqs, scales):
        with torch.no_grad():
            mf, r = _decode(m, v, s)
            for out, flat in ((ms, mf), (vs, r * r)):
                t = torch.empty_like(m, dtype=dtype)
                _flat(t).copy_(flat)
                out.append(t)
    return ms, vs


# ---------------------------------------------------------------------------
# optimizer
# ---------------------------------------------------------------------------

def _check_saved(i: int, p: torch.Tensor, saved: dict) -> None:
    """A parameter's saved state: moments of its shape, in 32 or 16 bits, or
    codes with their scales."""
    step = saved["step"]
    if step is None or int(step) != step or step < 0:
        raise ValueError(f"step of parameter {i} is {step}")
    m, v = saved["exp_avg"], saved["exp_avg_sq"]
    for t in (m, v):
        if not isinstance(t, torch.Tensor) or t.layout != torch.strided or \
                t.shape != p.shape:
            raise ValueError(f"the moments of parameter {i} must be tensors "
                             f"{tuple(p.shape)}")
    scales = saved.get("scales")
    if scales is None:
        if m.dtype not in _FLOATS or v.dtype not in _FLOATS:
            raise ValueError(f"the moments of parameter {i} are {m.dtype} and "
                             f"{v.dtype}, without scales")
        return
    if m.dtype != torch.float8_e4m3fn or v.dtype != torch.uint8:
        raise ValueError(f"the codes of parameter {i} are {m.dtype} and "
                         f"{v.dtype}")
    if not _is_dense(m) or not _same_layout(m, v):
        raise ValueError(f"the codes of parameter {i} must be dense and laid "
                         "out alike")
    if not isinstance(scales, torch.Tensor):
        raise ValueError(f"the scales of parameter {i} are not a tensor")
    _check_scales(scales, m, i)


class FusedAdamW(torch.optim.Optimizer):
    """AdamW (torch.optim.AdamW's step) as a few fused HIP launches.

    state_bits: 32 (float32 moments) or 8 (adamw8bit_'s); may be set per
        parameter group, e.g. 32 for a group of norm weights and biases.
    max_grad_norm: clips by the norm over the gradients of all groups; the
        gradients themselves are left as they are.  The norm of the last step
        is kept in `last_grad_norm`, a float32 scalar on the device.
    seed: of the 8-bit moments' stochastic rounding.

    All parameters lie on one device.  step() reads lr and the step count on
    the host, so it is not captured into a graph: run it after each replay,
    as MoCoStepper does.  state_dict() holds neither max_grad_norm nor seed,
    which a resumed run gives again; copies and pickles of the optimizer do.
    """

    def __init__(self, params, lr: float = 1e-3,
                 betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 0.01, state_bits: int = 32,
                 max_grad_norm: Optional[float] = None, seed: int = 0):
        _check_step(1, lr, betas, eps, weight_decay, max_grad_norm, None)
        self.max_grad_norm = max_grad_norm
        self.seed = int(seed)
        self.last_grad_norm: Optional[torch.Tensor] = None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps,
                                      weight_decay=weight_decay,
                                      state_bits=state_bits))

    # the base class copies and pickles groups and state alone
    def __getstate__(self):
        return {**super().__getstate__(), "max_grad_norm": self.max_grad_norm,
                "seed": self.seed, "last_grad_norm": self.last_grad_norm}

    def __setstate__(self, state):
        super().__setstate__(state)
        # (a pickle of the base's part alone)
        for name, value in (("max_grad_norm", None), ("seed", 0),
                            ("last_grad_norm", None)):
            self.__dict__.setdefault(name, value)

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        bits = self.param_groups[-1]["state_bits"]
        if bits not in (8, 32):
            del self.param_groups[-1]
            raise ValueError(f"state_bits must be 8 or 32, got {bits}")

    def _init_state(self, p, bits):
        state = self.state[p]
        if not _is_dense(p):
            raise ValueError("FusedAdamW needs dense parameters, got strides "
                             f"{p.stride()} for shape {tuple(p.shape)}")

        def zeros(dtype):
            return torch.zeros_like(p, dtype=dtype,
                                    memory_format=torch.preserve_format)
        state["step"] = 0
        state["exp_avg"] = zeros(torch.float8_e4m3fn if bits == 8
                                 else torch.float32)
        state["exp_avg_sq"] = zeros(torch.uint8 if bits == 8
                                    else torch.float32)
        if bits == 8:
            state["scales"] = torch.zeros(-(-p.numel() // BLOCK), 2,
                                          dtype=torch.float32, device=p.device)
        return state

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if torch.cuda.is_available() and \
                torch.cuda.is_current_stream_capturing():
            raise RuntimeError("FusedAdamW.step() counts its steps on the "
                               "host and cannot be captured into a graph")
        # lists of equal step count, per group and kind of state
        buckets, every_grad, last = {}, [], None
        for gi, group in enumerate(self.param_groups):
            for p in group["params"]:
                g = p.grad
                if g is None:
                    continue
                if g.is_sparse:
                    raise ValueError("sparse gradients are not supported")
                state = self.state[p] or self._init_state(
                    p, group["state_bits"])
                if g.stride() != p.stride() and not _same_layout(p, g):
                    g = torch.empty_like(p).copy_(g)
                scales = state.get("scales")
                key = (gi, state["step"], scales is not None)
                if key != last:
                    last = key
                    ps, gs, ms, vs, ss = buckets.setdefault(
                        key, ([], [], [], [], []))
                ps.append(p)
                gs.append(g)
                ms.append(state["exp_avg"])
                vs.append(state["exp_avg_sq"])
                ss.append(scales)
                every_grad.append(g)
        norm = None
        if self.max_grad_norm is not None and every_grad:
            # (on the GPU: read through the caches, for the step's sake)
            norm = self.last_grad_norm = \
                ext().grad_norm(every_grad, True) \
                if use_hip(every_grad[0]) else grad_norm(every_grad)
        for n, ((gi, count, eight), lists) in enumerate(buckets.items()):
            group = self.param_groups[gi]
            # each bucket's list counts from 0: a hash of its own
            _adamw(*lists[:4], lists[4] if eight else None, count + 1,
                   group["lr"], group["betas"], group["eps"],
                   group["weight_decay"], self.max_grad_norm, norm,
                   self.seed + n)
            for p in lists[0]:
                self.state[p]["step"] = count + 1
        return loss

    def load_state_dict(self, state_dict):
        """Also takes the state of torch.optim.AdamW.  The moments keep their
        own types (the base class casts them to the parameter's, and a group
        may so go on with 32-bit moments that were saved, whatever its
        state_bits) and follow their parameter's memory format.  A state that
        does not fit is refused before anything is loaded."""
        for group in state_dict["param_groups"]:
            if group.get("amsgrad") or group.get("maximize"):
                raise ValueError("amsgrad and maximize are not supported")
            if not group.get("decoupled_weight_decay", True) and \
                    group["weight_decay"]:
                raise ValueError("the state's weight decay is Adam's, a part "
                                 "of the gradient: not supported")
        if any(not {"step", "exp_avg", "exp_avg_sq"} <= s.keys()
               for s in state_dict["state"].values() if s):
            raise ValueError("not the state of an AdamW: no step and moments")
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        states = [(i, p, state_dict["state"].get(i))
                  for i, p in zip(ids, params)]
        for i, p, saved in states:
            if saved:
                _check_saved(i, p, saved)
        bits = [group["state_bits"] for group in self.param_groups]
        super().load_state_dict(state_dict)
        for group, own_bits in zip(self.param_groups, bits):
            group.setdefault("state_bits", own_bits)
        for _, p, saved in states:
            if not saved:
                continue
            state = self.state[p]
            state["step"] = int(saved["step"])
            m, v = (saved[k].to(p.device) for k in ("exp_avg", "exp_avg_sq"))
            scales = saved.get("scales")
            if scales is not None:
                scales = scales.to(p.device, copy=True)
                if not _same_layout(m, p):
                    # the blocks of another memory order: read back, laid out
                    # anew and rounded once more
                    (m,), (v,) = adamw8bit_values([m], [v], [scales])
                    m, r = (torch.empty_like(p, dtype=torch.float32).copy_(t)
                            for t in (m, v.sqrt()))
                    codes = _encode(_flat(m), _flat(r), None)
                    m, v, scales = (
                        *(torch.empty_like(p, dtype=c.dtype) for c in
                          codes[:2]), codes[2])
                    _flat(m).copy_(codes[0])
                    _flat(v).copy_(codes[1])
                state["scales"] = scales

            def own(t):
                if t.dtype in _FLOATS:
                    t = t.float()
                return torch.empty_like(p, dtype=t.dtype).copy_(t)
            state["exp_avg"], state["exp_avg_sq"] = own(m), own(v)
