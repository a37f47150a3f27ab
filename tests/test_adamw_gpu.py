"""AdamW, its 8-bit moments and the gradient norm on the GPU, against the
definitions in 64 bits."""

import numpy as np
import pytest
import torch

from adamw_oracle import (HALF, LEAST, check_codes, decode, dither, mem,
                          root_value, step64)

pytestmark = pytest.mark.gpu

# one element; around a block of 256, a vector of 8 and a chunk of 4096; more
# tensors than a launch takes
SHAPES = [(1,), (7,), (255,), (256,), (257,), (4095,), (4096,), (4097,),
          (3, 5, 7), (0,), (64, 3, 7, 7), (1000, 33), (300_001,)]
MANY = [(n % 61 + 1,) for n in range(150)]


def make(shapes, dtype, eight, seed=0, offset=0):
    """Weights and their state, every tensor `offset` elements behind an
    aligned address."""
    gen = torch.Generator().manual_seed(seed)

    def place(t):
        flat = torch.zeros(t.numel() + offset, dtype=t.dtype, device="cuda")
        out = flat[offset:].view(t.shape)
        out.copy_(t)
        return out

    ps = [place(torch.randn(s, generator=gen).mul(0.1).to(dtype))
          for s in shapes]
    ms = [place(torch.zeros(s).to(torch.float8_e4m3fn if eight
                                  else torch.float32)) for s in shapes]
    vs = [place(torch.zeros(s, dtype=torch.uint8 if eight
                            else torch.float32)) for s in shapes]
    if not eight:
        return ps, ms, vs
    return ps, ms, vs, [torch.zeros(-(-p.numel() // 256), 2, device="cuda")
                        for p in ps]


def grads_for(ps, seed, place=lambda g: g):
    gen = torch.Generator().manual_seed(seed)
    out = []
    for i, p in enumerate(ps):
        g = torch.randn(p.shape, generator=gen) * 10.0 ** -(i % 4)
        out.append(place(g.to(p.dtype).cuda()))
    return out


def check_step(state, gs, call, step, coef, kw, dtype, eight, seed):
    before = [mem(p) for p in state[0]]
    if eight:
        mv = [decode(*x) for x in zip(*state[1:])]
        mv = [(m, r * r) for m, r in mv]
    else:
        mv = [(mem(m), mem(v)) for m, v in zip(*state[1:])]
    call()
    torch.cuda.synchronize()
    for i, p in enumerate(state[0]):
        p2, m2, v2, dp, dm, dv = step64(
            before[i], mem(gs[i]), *mv[i], step, kw["lr"], kw["betas"],
            kw["eps"], kw["weight_decay"], coef)
        assert (abs(mem(p) - p2) <= dp + HALF[dtype] * (abs(p2) + dp)
                + LEAST[dtype]).all(), i
        if eight:
            check_codes(m2, np.sqrt(v2), dm, state[1][i], state[2][i],
                        state[3][i], i, step, seed)
        else:
            assert (abs(mem(state[1][i]) - m2) <= dm).all(), i
            assert (abs(mem(state[2][i]) - v2) <= dv).all(), i


KW = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)


@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("shapes,offset,max_norm",
                         [(SHAPES, 0, None), (SHAPES, 1, 0.05),
                          (MANY, 0, 1e6), (SHAPES, 3, None)])
def test_steps_against_64_bits(dtype, eight, shapes, offset, max_norm):
    from moco_amd.ops import adamw8bit_, adamw_
    state = make(shapes, dtype, eight, offset=offset)
    for step in range(1, 4):
        gs = grads_for(state[0], step)
        norm = np.sqrt(sum((mem(g) ** 2).sum() for g in gs))
        coef = 1.0 if max_norm is None else min(1, max_norm / (norm + 1e-6))
        out = []

        def call():
            args = (state[0], gs, *state[1:])
            out.append(adamw8bit_(*args, step=step, seed=9,
                                  max_norm=max_norm, **KW) if eight
                       else adamw_(*args, step=step, max_norm=max_norm,
                                   **KW))
        check_step(state, gs, call, step, coef, KW, dtype, eight, 9)
        if max_norm is None:
            assert out[0] is None
        else:
            assert out[0].is_cuda and out[0].shape == ()
            # two roundings: the root, and to 32 bits
            assert abs(float(out[0]) - norm) <= 2 * 2.0 ** -24 * norm


@pytest.mark.parametrize("eight", [False, True])
def test_mixed_types_and_memory_formats_in_one_call(eight):
    from moco_amd.ops import adamw8bit_, adamw_
    shapes = [(16, 8, 3, 3), (300,), (24, 8, 1, 1), (5000,), (77,)]
    types = [torch.float32, torch.bfloat16, torch.float32, torch.float16,
             torch.bfloat16]
    st = [make([s], d, eight, seed=i) for i, (s, d) in
          enumerate(zip(shapes, types))]
    state = [[x[k][0] for x in st] for k in range(len(st[0]))]
    for k in range(3):  # filters in channels_last
        for i in (0, 2):
            state[k][i] = state[k][i].contiguous(
                memory_format=torch.channels_last)
    gs = [torch.empty_like(p).copy_(g) for p, g in
          zip(state[0], grads_for(state[0], 1))]
    before = [[mem(t) for t in x] for x in state[:1]][0]
    (adamw8bit_ if eight else adamw_)(
        state[0], gs, *state[1:], step=1, **KW,
        **({"seed": 2} if eight else {}))
    for i, p in enumerate(state[0]):
        zero = np.zeros(p.numel())
        p2, m2, v2, dp, dm, dv = step64(before[i], mem(gs[i]), zero, zero, 1,
                                        KW["lr"], KW["betas"], KW["eps"],
                                        KW["weight_decay"], 1.0)
        assert (abs(mem(p) - p2) <= dp + HALF[types[i]] * (abs(p2) + dp)
                + LEAST[types[i]]).all()
        if eight:
            check_codes(m2, np.sqrt(v2), dm, state[1][i], state[2][i],
                        state[3][i], i, 1, 2)


def test_values_of_all_codes_gpu():
    from moco_amd.ops import adamw8bit_values
    code = torch.arange(256, dtype=torch.uint8, device="cuda")
    for reps, off in ((1, 0), (37, 0), (5, 3)):
        c = code.repeat(reps + 1)[off:off + 256 * reps + 5]
        n = c.numel()
        s = torch.rand(-(-n // 256), 2, device="cuda") + 0.5
        rows = s.repeat_interleave(256, 0)[:n].cpu()
        for dtype in HALF:
            (m,), (v,) = adamw8bit_values([c.view(torch.float8_e4m3fn)], [c],
                                          [s], dtype=dtype)
            want = (c.cpu().view(torch.float8_e4m3fn).float()
                    * rows[:, 0]).to(dtype)
            assert torch.equal(m.cpu().nan_to_num(7e3),
                               want.nan_to_num(7e3))
            r = torch.from_numpy(root_value(c.cpu().numpy().astype(np.int64))
                                 ).float() * rows[:, 1]
            assert torch.equal(v.cpu(), (r * r).to(dtype))


def test_rounding_to_e4m3_matches_torch():
    """All signs and magnitudes, subnormals and ties among them: one step
    from empty moments with beta1 = 0 stores the gradient itself."""
    from moco_amd.ops import adamw8bit_
    base = torch.arange(-448.0, 448.25, 0.25)
    fine = torch.arange(-64, 65) * 2.0 ** -11
    g = torch.cat([base, fine])
    n = g.numel()
    pad = -n % 255
    rows = torch.cat([g, torch.zeros(pad)]).view(-1, 255)
    g = torch.cat([torch.full((rows.shape[0], 1), 448.0), rows], 1).view(-1)
    st = make([(g.numel(),)], torch.float32, True)
    adamw8bit_(st[0], [g.cuda()], *st[1:], step=1, lr=0.0,
               betas=(0.0, 0.9), weight_decay=0.0)
    # 448 * (1 / 448) is one half step from 1: the scale is 1 to 2^-24
    sm = st[3][0][:, 0].repeat_interleave(256).cpu()
    want = (g * sm.reciprocal()).clamp(-448, 448).to(torch.float8_e4m3fn)
    assert torch.equal(st[1][0].cpu().float(), want.float())


def test_codes_are_those_of_32_bit_arithmetic():
    """Bit for bit over three steps: numpy's float32 operations are each
    rounded correctly, and so are the kernel's up to the codes (the quotient
    after them is not, and is not looked at)."""
    from moco_amd.ops import adamw8bit_
    f = np.float32
    n, b1, b2 = 100_003, 0.9, 0.999
    rows = -(-n // 256)
    st = make([(n,)], torch.float32, True)
    m, r = np.zeros(rows * 256, f), np.zeros(rows * 256, f)
    for step in range(1, 4):
        gs = grads_for(st[0], step)
        adamw8bit_(st[0], gs, *st[1:], step=step, seed=4, lr=1e-3,
                   betas=(b1, b2))
        g = np.zeros(rows * 256, f)
        g[:n] = gs[0].cpu().numpy()
        m = m * f(b1) + g * f(1 - b1)
        r = np.sqrt((r * r) * f(b2) + (g * g) * f(1 - b2))
        m, r = m.reshape(-1, 256), r.reshape(-1, 256)
        sm = np.maximum(abs(m).max(1, keepdims=True), f(1e-30)) * f(1 / 448)
        sr = np.maximum(r.max(1, keepdims=True), f(1e-30)) * f(1 / 1.9375)
        assert np.array_equal(st[3][0].cpu().numpy(), np.hstack([sm, sr]))
        mc = torch.from_numpy(np.clip(m * (f(1) / sm), f(-448), f(448))).to(
            torch.float8_e4m3fn)
        bits = (r * (f(1) / sr) * f(2.0 ** -112)).view(np.int32)
        up = (dither(rows * 256, 0, step, 4) * 2 ** 19).astype(np.int32)
        rc = np.minimum((bits + up.reshape(-1, 256)) >> 19, 255)
        rc = np.where(r > 0, np.maximum(rc, 1), 0)
        assert torch.equal(st[1][0].cpu().float(), mc.float().view(-1)[:n])
        assert np.array_equal(st[2][0].cpu().numpy(), rc.reshape(-1)[:n])
        m = (mc.float().numpy() * sm).reshape(-1)
        r = ((rc.astype(np.int32) << 19).view(f) * f(2.0 ** 112)
             * sr).reshape(-1)


@pytest.mark.parametrize("dtype", list(HALF))
def test_grad_norm_gpu(dtype):
    from moco_amd.ops import grad_norm
    # one launch up to 32 chunks of 4096, two and more behind
    for shapes in (SHAPES, MANY, [(0,)], [(5_000_003,)], [(1,)], [(4096,)],
                   [(4097,), (0,), (3,)], [(131072,)], [(131073,)],
                   [(5,)] * 32, [(5,)] * 33, [(4096,)] * 31 + [(4095,)]):
        gs = grads_for([torch.empty(s, dtype=dtype) for s in shapes], 3)
        want = np.sqrt(sum((mem(g) ** 2).sum() for g in gs))
        got = grad_norm(gs)
        assert got.is_cuda and got.dtype == torch.float32
        assert abs(float(got) - want) <= 2 * 2.0 ** -24 * want
        assert torch.equal(got, grad_norm(gs))
    x = torch.randn(100, 64, device="cuda").to(dtype)
    views = [x[:, ::3], x[3, 1:], x[:1].expand(9, 64), x.t()]
    want = np.sqrt(sum((v.double().cpu().numpy() ** 2).sum() for v in views))
    assert abs(float(grad_norm(views)) - want) <= 2 * 2.0 ** -24 * want
    for bad in (float("nan"), float("inf")):
        x[5, 5] = bad
        assert str(float(grad_norm([x]))) == str(bad)


def test_nonfinite_gradients_gpu():
    from moco_amd.ops import adamw8bit_, adamw8bit_values, adamw_
    for eight in (False, True):
        for bad in (float("nan"), float("inf")):
            st = make([(5000,), (300,)], torch.float32, eight)
            gs = grads_for(st[0], 0)
            gs[0][300] = bad
            (adamw8bit_ if eight else adamw_)(st[0], gs, *st[1:], step=1,
                                              lr=0.1)
            wrong = ~torch.isfinite(st[0][0])
            assert wrong.sum() == 1 and wrong[300]
            assert torch.isfinite(st[0][1]).all()
            if eight:
                ms, vs = adamw8bit_values(*st[1:])
                for t in (ms[0], vs[0]):
                    assert torch.isnan(t).sum() == 256
                    assert torch.isnan(t[256:512]).all()
            st = make([(5000,), (300,)], torch.float32, eight)
            norm = (adamw8bit_ if eight else adamw_)(
                st[0], gs, *st[1:], step=1, lr=0.1, max_norm=1.0)
            assert not torch.isfinite(norm)
            if bad != bad:
                assert torch.isnan(st[0][1]).all()


def test_total_norm_on_another_stream_and_repeatability():
    """The same call gives the same bits, on any stream."""
    from moco_amd.ops import adamw8bit_, grad_norm
    ends = []
    for use in (False, True):
        st = make(SHAPES, torch.float32, True)
        s = torch.cuda.Stream() if use else torch.cuda.current_stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for step in range(1, 4):
                gs = grads_for(st[0], step)
                norm = grad_norm(gs)
                out = adamw8bit_(st[0], gs, *st[1:], step=step, max_norm=0.5,
                                 total_norm=norm, **KW)
                assert out is norm or torch.equal(out, norm)
        s.synchronize()
        ends.append([t.cpu() for x in st for t in x])
    for a, b in zip(*ends):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("eight", [False, True])
def test_captured_call_replays(eight):
    """A functional call in a graph, replayed with eager work between."""
    from moco_amd.ops import adamw8bit_, adamw_, grad_norm
    call = adamw8bit_ if eight else adamw_
    a, b = (make(MANY, torch.float32, eight) for _ in range(2))
    gs = grads_for(a[0], 1)
    kw = dict(step=5, max_norm=0.5, **KW)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        captured = call(a[0], gs, *a[1:], **kw)
    for k in range(4):
        for x, y in zip(gs, grads_for(a[0], 10 + k)):
            x.copy_(y)
        g.replay()
        want = call(b[0], gs, *b[1:], **kw)
        assert torch.equal(captured, want)
        assert torch.equal(want, grad_norm(gs))
        torch.cuda.synchronize()
        for x, y in zip(a, b):
            for t, u in zip(x, y):
                assert torch.equal(t.view(torch.uint8), u.view(torch.uint8))


def test_refusals_gpu():
    """Nothing is launched: the weights stay as they are."""
    from moco_amd.ops import adamw8bit_, adamw_, grad_norm
    for eight in (False, True):
        call = adamw8bit_ if eight else adamw_

        def attempt(exc, edit):
            st = make([(4, 6), (300,)], torch.float32, eight)
            st = [list(st[0]), grads_for(st[0], 0), *map(list, st[1:])]
            edit(st)
            was = [t.clone() for t in st[0]]
            with pytest.raises(exc):
                call(*st, step=1, lr=0.1)
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(was, st[0]))

        def put(k, i, f):
            return lambda st: st[k].__setitem__(i, f(st[k][i]))
        attempt(ValueError, lambda st: st[1].pop())
        attempt(ValueError, put(1, 0, lambda t: t.view(6, 4)))
        attempt(ValueError, put(1, 0, lambda t: t.t().contiguous().t()))
        attempt(ValueError, put(1, 0, lambda t: t.to_sparse()))
        attempt(ValueError, put(1, 0, lambda t: t.cpu()))
        attempt(ValueError, put(0, 1, lambda t: t.cpu()))
        attempt(TypeError, put(1, 1, lambda t: t.bfloat16()))
        attempt(TypeError, put(2, 0, lambda t: t.float().double()))
        attempt(ValueError, lambda st: [x.append(x[0]) for x in st])
        attempt(ValueError, lambda st: st[1].__setitem__(1, st[0][1]))
        if eight:
            attempt(ValueError, put(4, 1, lambda t: t[:1]))
            attempt(ValueError, put(4, 1, lambda t: t.double()))
    with pytest.raises(ValueError):
        grad_norm([torch.zeros(3, device="cuda"), torch.zeros(3)])
    with pytest.raises(TypeError):
        grad_norm([torch.zeros(3, device="cuda", dtype=torch.float64)])


def test_writes_are_counted_and_empty_views_allowed():
    from moco_amd.ops import adamw8bit_, adamw_
    for eight in (False, True):
        st = make([(300,), (0,)], torch.float32, eight)
        st[0][1] = st[0][0][7:7]
        gs = grads_for(st[0], 0)
        was = [st[0][0]._version, gs[0]._version] + [
            x[0]._version for x in st[1:]]
        (adamw8bit_ if eight else adamw_)(st[0], gs, *st[1:], step=1, lr=0.1)
        now = [st[0][0]._version, gs[0]._version] + [
            x[0]._version for x in st[1:]]
        assert [a > b for a, b in zip(now, was)] == \
            [True, False] + [True] * (len(st) - 1)
        with pytest.raises(TypeError):
            (adamw8bit_ if eight else adamw_)([st[0][0]], [3], *st[1:],
                                              step=1, lr=0.1)


@pytest.mark.parametrize("bits", [8, 32])
def test_optimizer_gpu(bits):
    """A model in channels_last with bf16 and fp32 weights; the CPU's plain
    path runs beside it."""
    import copy

    from moco_amd.ops import FusedAdamW
    torch.manual_seed(0)
    m = torch.nn.Sequential(torch.nn.Conv2d(3, 16, 3), torch.nn.BatchNorm2d(
        16), torch.nn.Flatten(), torch.nn.Linear(16, 5).bfloat16())
    c = copy.deepcopy(m)
    m = m.cuda().to(memory_format=torch.channels_last)
    c = c.to(memory_format=torch.channels_last)
    kw = dict(lr=1e-2, state_bits=bits, max_grad_norm=0.1, seed=1)
    om, oc = FusedAdamW(m.parameters(), **kw), FusedAdamW(c.parameters(), **kw)
    for s in range(3):
        gen = torch.Generator().manual_seed(s)
        for p, q in zip(m.parameters(), c.parameters()):
            q.grad = torch.randn(q.shape, generator=gen).to(q.dtype)
            p.grad = q.grad.cuda()  # contiguous: laid out by the optimizer
        om.step()
        oc.step()
        assert torch.allclose(om.last_grad_norm.cpu(), oc.last_grad_norm,
                              rtol=2.0 ** -22)
    for p, q in zip(m.parameters(), c.parameters()):
        # three steps of lr; square roots may differ by an ulp, and a code
        # near its border may round the other way: a bf16 weight by a step
        tol = 2.0 ** -7 if q.dtype == torch.bfloat16 else 1e-5
        assert torch.allclose(p.float().cpu(), q.float(), rtol=tol,
                              atol=1e-5 if bits == 32 else 2e-3)
    g = torch.cuda.CUDAGraph()
    x = torch.zeros(1, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        x.add_(1)
        with pytest.raises(RuntimeError):
            om.step()
