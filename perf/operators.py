"""What is timed of the training-step operators, and their plain forms.

- ``adamw``      ops.adamw_: AdamW over many tensors, 32-bit moments,
                 optionally with the gradient-norm clip in the same call
- ``adamw8``     ops.adamw8bit_: the same step with 8-bit moments, and
                 ops.adamw8bit_values, which reads them back
- ``grad_norm``  ops.grad_norm: the 2-norm over all gradients
- ``norm``       ops.norm_residual: the norms after and before a residual
                 block with its gate and residual scale, forward alone or
                 forward and backward

``own`` false runs elementary torch operations, ``own`` true the framework.
"""

import math
import random

import torch

own = False

BLOCK = 256           # elements that share a pair of scales (adamw8)
TOP_M, TOP_R = 448.0, 1.9375     # largest value of a code, per moment
TINY = 1e-30          # least block maximum that a scale stands for
EPS = 1e-8
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16,
          "fp16": torch.float16}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def _optim(name, op, layout, dtype, elements=0, tensors=0, clip=False):
    c = {"op": op, "layout": layout, "dtype": dtype, "elements": elements,
         "tensors": tensors, "clip": clip}
    return {"name": name, **c} if name else c


def _norm_case(name, rows, width, stream, branch, kind, gate, act, scale,
               train):
    c = {"op": "norm", "rows": rows, "width": width, "stream": stream,
         "branch": branch, "kind": kind, "gate": gate, "act": act,
         "scale": scale, "train": train}
    return {"name": name, **c} if name else c


def listed():
    return [
        # the projection head alone (4 tensors): fine-tuning it, where the
        # launch and the host cost most
        _optim("adamw_head", "adamw", "head", "fp32"),
        # the pretraining model, ResNet-50 with its head, clipped
        _optim("adamw_resnet50", "adamw", "resnet50", "fp32", clip=True),
        # bf16 weights of a stack of wide transformer-like blocks
        _optim("adamw_wide_bf16", "adamw", "blocks", "bf16"),
        # the pretraining model with the moments in 8 bits
        _optim("adamw8_resnet50", "adamw8", "resnet50", "fp32"),
        # bf16 weights, 8-bit moments, clipped: the memory-bound end
        _optim("adamw8_wide_bf16", "adamw8", "blocks", "bf16", clip=True),
        # odd lengths, from one element on: biases, gains, odd vocabularies
        _optim("adamw8_ragged", "adamw8", "ragged", "fp32", 3_000_001, 40),
        # gradient monitoring of the pretraining model
        _optim("grad_norm_resnet50", "grad_norm", "resnet50", "fp32"),
        # odd bf16 gradients, long sums
        _optim("grad_norm_ragged_bf16", "grad_norm", "ragged", "bf16",
               150_000_001, 60),
        # one token on its way through a block at serving
        _norm_case("norm_token", 1, 2048, "bf16", "bf16", "rms", "none",
                   "none", "none", False),
        # a contrastive batch of 256 rows in fp32 at the encoder's width
        _norm_case("norm_batch", 256, 2048, "fp32", "fp32", "layer", "none",
                   "none", "vector", True),
        # many tokens, gated by a full projection
        _norm_case("norm_tokens", 16384, 4096, "bf16", "bf16", "rms", "full",
                   "silu", "vector", True),
        # odd sizes, fp32 stream under bf16 blocks, one gate per token
        _norm_case("norm_odd", 5003, 1001, "fp32", "bf16", "layer", "row",
                   "sigmoid", "vector", True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["adamw", "adamw8", "grad_norm", "norm", "norm"])
    if op == "norm":
        width = _log(rng, 48, 8192)
        if rng.random() < 0.5:  # usual widths come in multiples of 64
            width = max(64, width // 64 * 64)
        rows = _log(rng, 1, max(2, 40_000_000 // width))
        stream, branch = rng.choice(
            [("fp32", "fp32"), ("bf16", "bf16"), ("fp16", "fp16"),
             ("fp32", "bf16"), ("fp32", "fp16")])
        gate = rng.choice(["none", "full", "row"])
        act = "none" if gate == "none" else rng.choice(
            ["none", "sigmoid", "silu"])
        return _norm_case(None, rows, width, stream, branch,
                          rng.choice(["rms", "layer"]), gate, act,
                          rng.choice(["none", "vector"]),
                          rng.random() < 0.7)
    elements = _log(rng, 2_000, 100_000_000)
    tensors = _log(rng, 1, min(200, max(2, elements // 500)))
    return _optim(None, op, "ragged", rng.choice(["fp32", "bf16", "fp16"]),
                  elements, tensors,
                  clip=op != "grad_norm" and rng.random() < 0.5)


def _resnet50():
    """Shapes of the ResNet-50 query encoder with its 2-layer head."""
    s = [(64, 3, 7, 7), (64,), (64,)]
    cin = 64
    for mid, blocks in ((64, 3), (128, 4), (256, 6), (512, 3)):
        for b in range(blocks):
            s += [(mid, cin, 1, 1), (mid,), (mid,),
                  (mid, mid, 3, 3), (mid,), (mid,),
                  (4 * mid, mid, 1, 1), (4 * mid,), (4 * mid,)]
            if b == 0:
                s += [(4 * mid, cin, 1, 1), (4 * mid,), (4 * mid,)]
            cin = 4 * mid
    return s + [(2048, 2048), (2048,), (128, 2048), (128,)]


def _shapes(case):
    lay = case["layout"]
    if lay == "head":
        return [(2048, 2048), (2048,), (128, 2048), (128,)]
    if lay == "resnet50":
        return _resnet50()
    if lay == "blocks":
        w = 2048
        return [(3 * w, w), (w, w), (4 * w, w), (w, 4 * w), (w,), (w,)] * 4
    # ragged: `tensors` lengths of one element up, `elements` in all
    rng = random.Random(case["elements"] * 1009 + case["tensors"])
    n = case["tensors"]
    w = [math.exp(rng.uniform(0, 7)) for _ in range(n)]
    room, k = case["elements"] - n, case["elements"] / sum(w)
    out = []
    for x in w[:-1]:
        take = max(0, min(room, int(x * k) - 1))
        room -= take
        out.append((1 + take,))
    return out + [(1 + room,)]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _mix(x):
    """32-bit hash of int64 values, whose low half counts."""
    mask = 0xFFFFFFFF
    x = (x * 0x9E3779B9) & mask
    x = x ^ (x >> 15)
    x = (x * 0xBB67AE85) & mask
    x = x ^ (x >> 16)
    return x


def _encode_root(q, dither):
    """Codes of q in [0, 1.9375]: 4 exponent and 4 fraction bits, rounded
    up where the 19 bits that are dropped and `dither` carry; 1 at least
    for what is above zero."""
    bits = (q * 2.0 ** -112).view(torch.int32)
    code = torch.clamp((bits + dither) >> 19, max=255)
    return torch.maximum(code, (q > 0).to(code.dtype)).to(torch.uint8)


def _decode_root(code):
    return (code.to(torch.int32) << 19).view(torch.float32) * 2.0 ** 112


def _prepare_optim(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    shapes, dtype = _shapes(case), DTYPES[case["dtype"]]
    # all tensors lie in one buffer per kind (as buckets of a distributed
    # run do), each from a whole block on
    sizes = [math.prod(s) for s in shapes]
    starts, total = [], 0
    for n in sizes:
        starts.append(total)
        total += -(-n // BLOCK) * BLOCK
    dev = "cuda"
    used = torch.zeros(total, dtype=torch.bool, device=dev)
    size = torch.full((total // BLOCK,), 1e-3, device=dev)
    pick = random.Random(seed)
    for n, at in zip(sizes, starts):
        used[at:at + n] = True
        # tensors differ in the size of their gradients by decades
        size[at // BLOCK:(at + n + BLOCK - 1) // BLOCK] = \
            10 ** pick.uniform(-5, -2)
    size = size.repeat_interleave(BLOCK)

    def rand():
        return torch.randn(total, device=dev, generator=gen) * used

    def views(flat):
        out = []
        for s, n, at in zip(shapes, sizes, starts):
            t = flat[at:at + n]
            if len(s) == 4:  # the framework keeps filters channels_last
                t = t.view(s[0], s[2], s[3], s[1]).permute(0, 3, 1, 2)
            else:
                t = t.view(s)
            out.append(t)
        return out

    st = {"case": case, "flat_g": (rand() * size).to(dtype), "step": 100,
          "seed": seed & 0xFFFF, "lr": 1e-3, "betas": (0.9, 0.999),
          "weight_decay": 0.1, "max_norm": 0.5 if case["clip"] else None}
    st["grads"] = views(st["flat_g"])
    if case["op"] == "grad_norm":
        return st
    st["flat_p"] = (rand() * 0.02).to(dtype)
    st["params"] = views(st["flat_p"])
    m = rand() * size * 0.3
    root = (rand() * size).abs() * 0.7 + size * 0.3 * used
    if case["op"] == "adamw":
        st["flat_m"], st["flat_v"] = m, root * root
    else:
        sm = torch.clamp_min(m.view(-1, BLOCK).abs().amax(1), TINY) / TOP_M
        sr = torch.clamp_min(root.view(-1, BLOCK).amax(1), TINY) / TOP_R
        st["flat_m"] = (m.view(-1, BLOCK) / sm[:, None]).clamp(
            -TOP_M, TOP_M).to(torch.float8_e4m3fn).view(-1)
        st["flat_v"] = _encode_root(root.view(-1, BLOCK) / sr[:, None],
                                    1 << 18).view(-1)
        st["flat_scales"] = torch.stack([sm, sr], 1).contiguous()
        st["scales"] = [st["flat_scales"][at // BLOCK:-(-(at + n) // BLOCK)]
                        for n, at in zip(sizes, starts)]
        # what each block's first element counts from in the rounding hash
        st["base"] = torch.tensor(
            [0x3C6EF372 * t + b * BLOCK for t, n in enumerate(sizes)
             for b in range(-(-n // BLOCK))], device=dev) & 0xFFFFFFFF
    st["exp_avgs"] = views(st["flat_m"])
    st["exp_avg_sqs"] = views(st["flat_v"])
    return st


def _prepare_norm(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    n, c, dev = case["rows"], case["width"], "cuda"
    tx, th = DTYPES[case["stream"]], DTYPES[case["branch"]]
    train = case["train"]

    def rand(*shape, scale=1.0, shift=0.0, dtype=torch.float32):
        t = torch.randn(*shape, device=dev, generator=gen)
        return (t * scale + shift).to(dtype)

    st = {"case": case, "x": rand(n, c, scale=1.5, shift=0.1, dtype=tx),
          "branch": rand(n, c, scale=0.8, shift=-0.05, dtype=th),
          "gate": None, "scale": None}
    if case["gate"] != "none":
        st["gate"] = rand(n, c if case["gate"] == "full" else 1, dtype=th)
    if case["scale"] == "vector":
        st["scale"] = rand(c, scale=0.05, shift=0.3)
    kind = torch.nn.RMSNorm if case["kind"] == "rms" else torch.nn.LayerNorm
    for k in ("post", "pre"):
        mod = kind(c, eps=1e-6, device=dev)
        with torch.no_grad():
            mod.weight.copy_(rand(c, scale=0.1, shift=1.0))
            if case["kind"] == "layer":
                mod.bias.copy_(rand(c, scale=0.1))
        st[k] = mod.requires_grad_(train)
    if train:
        st["d_r"] = rand(n, c, dtype=tx)
        st["d_y"] = rand(n, c, dtype=th)
        st["leaves"] = [t.requires_grad_() for t in
                        (st["x"], st["branch"], st["gate"], st["scale"],
                         *st["post"].parameters(), *st["pre"].parameters())
                        if t is not None]
    return st


def prepare(case, seed):
    if case["op"] == "norm":
        return _prepare_norm(case, seed)
    return _prepare_optim(case, seed)


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------

def _plain_grad_norm(flat):
    # a sum over up to 1e8 squares: in 64 bits, rounded at the end
    return flat.double().square().sum().sqrt().float()


def _plain_adamw(st):
    b1, b2 = st["betas"]
    lr, step, eight = st["lr"], st["step"], st["case"]["op"] == "adamw8"
    g = st["flat_g"].float()
    norm = None
    if st["max_norm"] is not None:
        norm = _plain_grad_norm(st["flat_g"])
        g = g * torch.clamp(torch.full_like(norm, st["max_norm"])
                            / (norm + 1e-6), max=1.0)
    if eight:
        s_m, s_r = st["flat_scales"][:, :1], st["flat_scales"][:, 1:]
        m = (st["flat_m"].float().view(-1, BLOCK) * s_m).view(-1)
        r = (_decode_root(st["flat_v"]).view(-1, BLOCK) * s_r).view(-1)
        v = r * r
    else:
        m, v = st["flat_m"], st["flat_v"]
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    r = v.sqrt()
    q = m / (r * (1 / math.sqrt(1 - b2 ** step)) + EPS)
    p = st["flat_p"].float() * (1 - lr * st["weight_decay"]) \
        - q * (lr / (1 - b1 ** step))
    st["flat_p"].copy_(p)
    if not eight:
        st["flat_m"].copy_(m)
        st["flat_v"].copy_(v)
        return norm, st["flat_p"], st["flat_m"], st["flat_v"]
    m, r = m.view(-1, BLOCK), r.view(-1, BLOCK)
    s_m = torch.clamp_min(m.abs().amax(1, keepdim=True), TINY) * (1 / TOP_M)
    s_r = torch.clamp_min(r.amax(1, keepdim=True), TINY) * (1 / TOP_R)
    st["flat_scales"].copy_(torch.cat([s_m, s_r], 1))
    st["flat_m"].copy_((m * s_m.reciprocal()).clamp(-TOP_M, TOP_M)
                       .to(torch.float8_e4m3fn).view(-1))
    key = st["seed"] * 0x6A09E667 + step * 0xA54FF53A
    at = st["base"][:, None] + torch.arange(BLOCK, device=m.device) + key
    dither = (_mix(at) >> 13).to(torch.int32)
    st["flat_v"].copy_(_encode_root(r * s_r.reciprocal(), dither).view(-1))
    m = st["flat_m"].float().view(-1, BLOCK) * s_m
    r = _decode_root(st["flat_v"]).view(-1, BLOCK) * s_r
    # read back in bf16: a code's 4 or 5 digits, times its scale
    return (norm, st["flat_p"], m.view(-1).bfloat16(),
            (r * r).view(-1).bfloat16())


def _plain_norm(x, mod):
    if isinstance(mod, torch.nn.LayerNorm):
        x = x - x.mean(-1, keepdim=True)
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + mod.eps)
    y = y * mod.weight
    return y if getattr(mod, "bias", None) is None else y + mod.bias


def _plain_norm_residual(st):
    add = _plain_norm(st["branch"].float(), st["post"])
    if st["gate"] is not None:
        g = st["gate"].float()
        act = st["case"]["act"]
        s = g if act == "none" else 1 / (1 + torch.exp(-g))
        add = add * (g * s if act == "silu" else s)
    if st["scale"] is not None:
        add = add * st["scale"]
    r = st["x"].float() + add
    y = _plain_norm(r, st["pre"])
    return r.to(st["x"].dtype), y.to(st["branch"].dtype)


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        from moco_amd import ops
    if op == "norm":
        if own:
            r, y = ops.norm_residual(
                state["x"], state["branch"], post=state["post"],
                pre=state["pre"], gate=state["gate"],
                gate_act=None if case["act"] == "none" else case["act"],
                scale=state["scale"])
        else:
            r, y = _plain_norm_residual(state)
        if not case["train"]:
            return r, y
        return r, y, torch.autograd.grad((r, y), state["leaves"],
                                         (state["d_r"], state["d_y"]))
    if op == "grad_norm":
        return ops.grad_norm(state["grads"]) if own \
            else _plain_grad_norm(state["flat_g"])
    if not own:
        return _plain_adamw(state)
    kw = dict(step=state["step"], lr=state["lr"], betas=state["betas"],
              eps=EPS, weight_decay=state["weight_decay"],
              max_norm=state["max_norm"])
    if op == "adamw":
        norm = ops.adamw_(state["params"], state["grads"],
                          state["exp_avgs"], state["exp_avg_sqs"], **kw)
        return norm, state["flat_p"], state["flat_m"], state["flat_v"]
    norm = ops.adamw8bit_(state["params"], state["grads"],
                          state["exp_avgs"], state["exp_avg_sqs"],
                          state["scales"], seed=state["seed"], **kw)
    (m,), (v,) = ops.adamw8bit_values(
        [state["flat_m"]], [state["flat_v"]], [state["flat_scales"]],
        dtype=torch.bfloat16)
    return norm, state["flat_p"], m, v


# ---------------------------------------------------------------------------
# work
# ---------------------------------------------------------------------------

def work(case):
    size = {"fp32": 4, "bf16": 2, "fp16": 2}
    if case["op"] == "norm":
        n, c = case["rows"], case["width"]
        sx, sh = size[case["stream"]], size[case["branch"]]
        gate = {"none": 0, "row": n, "full": n * c}[case["gate"]] * sh
        vecs = (2 if case["kind"] == "rms" else 4) + \
            (case["scale"] == "vector")
        data = n * c * (2 * sx + 2 * sh) + gate + 4 * c * vecs
        flops = 14 * n * c
        if case["train"]:  # dr, dy in; dx, dh, dgate, d(vectors) out
            data += n * c * (2 * sx + 2 * sh) + gate + 4 * c * vecs
            flops += 40 * n * c
        return {"bytes": data, "flops": flops}
    n = sum(math.prod(s) for s in _shapes(case))
    t = size[case["dtype"]]
    if case["op"] == "grad_norm":
        return {"bytes": n * t + 4, "flops": 2 * n}
    flops = (15 + 3 * case["clip"]) * n
    if case["op"] == "adamw":
        return {"bytes": n * (3 * t + 16), "flops": flops}
    # codes and scales in and out, and the moments read back in bf16
    return {"bytes": n * (3 * t + 4 + 4) + n // BLOCK * 16,
            "flops": flops + 30 * n}


# ---------------------------------------------------------------------------
# from the definitions, in 64 bits
# ---------------------------------------------------------------------------

def _exact_root_value(code):
    e, f = torch.div(code.long(), 16, rounding_mode="floor"), code.long() % 16
    low = f.double() / 16 * 2.0 ** -14
    high = (1 + f.double() / 16) * torch.pow(2.0, (e - 15).double())
    return torch.where(e == 0, low, high)


def _exact_optim(case, seed):
    st = _prepare_optim(case, seed)
    g = st["flat_g"].double()
    norm = torch.linalg.vector_norm(g)
    if case["op"] == "grad_norm":
        return norm
    (b1, b2), t = st["betas"], st["step"]
    if st["max_norm"] is None:
        norm = None
    else:
        g = g * min(1.0, st["max_norm"] / (float(norm) + 1e-6))
    eight = case["op"] == "adamw8"
    m, v = st["flat_m"].double(), st["flat_v"]
    if eight:
        s = st["flat_scales"].double().repeat_interleave(BLOCK, 0)
        m, v = m * s[:, 0], (_exact_root_value(v) * s[:, 1]) ** 2
        del s
    else:
        v = v.double()
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g ** 2
    p = st["flat_p"].double()
    p = p - st["lr"] * (st["weight_decay"] * p + (m / (1 - b1 ** t)) / (
        (v / (1 - b2 ** t)) ** 0.5 + EPS))
    if not eight:
        return norm, p, m, v
    del g
    # m: to the nearest of sign * (8 + f) * 2^(e - 10), e in -5..
    s_m = (m.view(-1, BLOCK).abs().max(1, keepdim=True).values).clamp(
        min=TINY) / TOP_M
    q = m.view(-1, BLOCK) / s_m
    step = torch.pow(2.0, torch.floor(torch.log2(
        q.abs().clamp(min=2.0 ** -6))) - 3)
    m = (torch.round(q / step) * step * s_m).view(-1)
    del q, step
    # sqrt(v): up with the probability of what is cut off
    r = v.sqrt().view(-1, BLOCK)
    s_r = r.max(1, keepdim=True).values.clamp(min=TINY) / TOP_R
    r = r / s_r
    e = torch.floor(torch.log2(r.clamp(min=2.0 ** -14)))
    place = (e + 14) * 16 + r / torch.pow(2.0, e) * 16
    at = st["base"][:, None] + torch.arange(BLOCK, device=r.device) + (
        st["seed"] * 0x6A09E667 + t * 0xA54FF53A)
    code = torch.floor(place + (_mix(at) >> 13).double() / 2 ** 19)
    del at, place, e
    code = torch.where(r > 0, code.clamp(1, 255), torch.zeros_like(code))
    v = ((_exact_root_value(code) * s_r) ** 2).view(-1)
    return norm, p, m, v


def _exact_norm(case, seed):
    st = _prepare_norm(case, seed)
    d = {k: v.detach().double() for k, v in st.items()
         if isinstance(v, torch.Tensor)}
    layer, act = case["kind"] == "layer", case["act"]
    w = {k: [p.detach().double() for p in st[k].parameters()]
         for k in ("post", "pre")}

    def normed(t):
        t = t - t.mean(1, keepdim=True) if layer else t
        inv = ((t * t).mean(1, keepdim=True) + 1e-6) ** -0.5
        return t * inv, inv

    def back(dt, hat, inv):
        out = dt - hat * (dt * hat).mean(1, keepdim=True)
        return inv * (out - dt.mean(1, keepdim=True) if layer else out)

    h_hat, h_inv = normed(d["branch"])
    out = h_hat * w["post"][0] + (w["post"][1] if layer else 0)
    one = torch.ones(1, 1, dtype=torch.float64, device=out.device)
    gate = d.get("gate", one)
    sig = torch.sigmoid(gate)
    a = one if case["gate"] == "none" else \
        {"none": gate, "sigmoid": sig, "silu": gate * sig}[act]
    scale = d.get("scale", one[0])
    r = d["x"] + scale * a * out
    r_hat, r_inv = normed(r)
    y = r_hat * w["pre"][0] + (w["pre"][1] if layer else 0)
    if not case["train"]:
        return r, y
    dr = d["d_r"] + back(d["d_y"] * w["pre"][0], r_hat, r_inv)
    dn = dr * scale * a
    grads = [dr, back(dn * w["post"][0], h_hat, h_inv)]
    if case["gate"] != "none":
        slope = {"none": torch.ones_like(gate), "sigmoid": sig * (1 - sig),
                 "silu": sig * (1 + gate * (1 - sig))}[act]
        da = dr * scale * out
        if case["gate"] == "row":
            da = da.sum(1, keepdim=True)
        grads.append(da * slope)
    if case["scale"] != "none":
        grads.append((dr * a * out).sum(0))
    for dt, hat in ((dn, h_hat), (d["d_y"], r_hat)):
        grads.append((dt * hat).sum(0))
        if layer:
            grads.append(dt.sum(0))
    return r, y, tuple(grads)


def exact(case, seed):
    return _exact_norm(case, seed) if case["op"] == "norm" \
        else _exact_optim(case, seed)
