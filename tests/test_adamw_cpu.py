"""AdamW, its 8-bit moments and the gradient norm: the plain path, refusals
and the optimizer's bookkeeping (all on CPU)."""

import copy

import numpy as np
import pytest
import torch

from adamw_oracle import (HALF, LEAST, check_codes, decode, mem, root_value,
                          step64)
from moco_amd.ops import (FusedAdamW, adamw8bit_, adamw8bit_values, adamw_,
                          grad_norm)
from moco_amd.ops.adamw import _dither


def make(shapes, dtype=torch.float32, eight=False, seed=0, device="cpu"):
    """Weights, gradients and empty moments."""
    gen = torch.Generator().manual_seed(seed)
    ps, gs = ([torch.randn(s, generator=gen).mul(k).to(dtype).to(device)
               for s in shapes] for k in (0.1, 0.01))
    ms = [torch.zeros_like(p, dtype=torch.float8_e4m3fn if eight
                           else torch.float32) for p in ps]
    vs = [torch.zeros_like(p, dtype=torch.uint8 if eight
                           else torch.float32) for p in ps]
    if not eight:
        return ps, gs, ms, vs
    return ps, gs, ms, vs, [torch.zeros(-(-p.numel() // 256), 2,
                                        device=device) for p in ps]


SHAPES = [(1,), (255,), (256,), (257,), (3, 5, 7), (0,), (1000, 9)]


@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("max_norm", [None, 0.05, 1e6])
def test_steps_against_64_bits(dtype, eight, max_norm):
    state = make(SHAPES, dtype, eight)
    kw = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
    gen = torch.Generator().manual_seed(5)
    for step in range(1, 4):
        gs = [torch.randn(p.shape, generator=gen).mul(0.01).to(dtype)
              for p in state[0]]
        state = (state[0], gs, *state[2:])
        before = [mem(p) for p in state[0]]
        if eight:
            mv = [decode(m, v, s) for m, v, s in zip(*state[2:])]
            mv = [(m, r * r) for m, r in mv]
        else:
            mv = [(mem(m), mem(v)) for m, v in zip(state[2], state[3])]
        norm = np.sqrt(sum((mem(g) ** 2).sum() for g in gs))
        coef = 1.0 if max_norm is None else min(1, max_norm / (norm + 1e-6))
        if eight:
            got = adamw8bit_(*state, step=step, seed=3, max_norm=max_norm,
                             **kw)
        else:
            got = adamw_(*state, step=step, max_norm=max_norm, **kw)
        if max_norm is None:
            assert got is None
        else:
            assert abs(float(got) - norm) <= 2 * 2.0 ** -24 * norm
        for i, p in enumerate(state[0]):
            p2, m2, v2, dp, dm, dv = step64(
                before[i], mem(gs[i]), *mv[i], step, kw["lr"], kw["betas"],
                kw["eps"], kw["weight_decay"], coef)
            assert (abs(mem(p) - p2) <= dp + HALF[dtype] * (abs(p2) + dp)
                    + LEAST[dtype]).all()
            if eight:
                check_codes(m2, np.sqrt(v2), dm, state[2][i], state[3][i],
                            state[4][i], i, step, 3)
            else:
                assert (abs(mem(state[2][i]) - m2) <= dm).all()
                assert (abs(mem(state[3][i]) - v2) <= dv).all()


def test_matches_torch_adamw_over_steps():
    """The same trajectory as torch.optim.AdamW: each step may differ by the
    roundings of one step (64-bit tests above), 1e-6 of lr-sized updates
    and of the weights over ten steps."""
    ps = make(SHAPES)[0]
    a = [torch.nn.Parameter(p.clone()) for p in ps]
    b = [torch.nn.Parameter(p.clone()) for p in ps]
    oa = FusedAdamW(a, lr=1e-2, weight_decay=0.1)
    ob = torch.optim.AdamW(b, lr=1e-2, weight_decay=0.1)
    gen = torch.Generator().manual_seed(1)
    for _ in range(10):
        for x, y in zip(a, b):
            x.grad = torch.randn(x.shape, generator=gen)
            y.grad = x.grad.clone()
        oa.step()
        ob.step()
    for x, y in zip(a, b):
        assert torch.allclose(x, y, rtol=1e-5, atol=1e-6)


def test_channels_last_and_odd_strides_keep_their_places():
    p = torch.randn(8, 4, 3, 3)
    g = torch.randn(8, 4, 3, 3)
    plain = [p.clone(), g.clone(), torch.zeros_like(p), torch.zeros_like(p)]
    cl = [t.clone(memory_format=torch.channels_last) for t in plain]
    for state in (plain, cl):
        adamw_(*[[t] for t in state], step=1, lr=0.1)
    assert cl[0].is_contiguous(memory_format=torch.channels_last)
    assert torch.equal(plain[0], cl[0])
    # strides of dimensions of one element say nothing
    w = torch.randn(8, 4, 1, 1)
    v = w.clone(memory_format=torch.channels_last)
    adamw_([w], [v], [torch.zeros(8, 4, 1, 1)], [torch.zeros(8, 4, 1, 1)],
           step=1, lr=0.1)


def test_grad_norm_mixes_types_and_counts_expanded_elements():
    ts = [torch.randn(1000), torch.randn(7, 3).bfloat16(),
          torch.randn(5).half(), torch.zeros(0),
          torch.tensor([2.0]).expand(9), torch.randn(6, 8)[:, ::3]]
    want = np.sqrt(sum((t.double().numpy() ** 2).sum() for t in ts))
    got = grad_norm(ts)
    assert got.dtype == torch.float32 and got.shape == ()
    assert abs(float(got) - want) <= 2.0 ** -24 * want
    assert float(grad_norm([torch.zeros(0)])) == 0.0
    big = [torch.full((100,), 1e30)]  # squares leave fp32's range
    assert abs(float(grad_norm(big)) / 1e31 - 1) < 1e-6


def test_nonfinite_gradients():
    """A NaN reaches the weight it belongs to, and with 8-bit moments its
    block's scale; under a clip it reaches all."""
    for eight, value in ((False, "nan"), (True, "nan"), (True, "inf")):
        state = make([(600,)], eight=eight)
        state[1][0][300] = float(value)
        (adamw8bit_ if eight else adamw_)(*state, step=1, lr=0.1)
        bad = torch.isnan(state[0][0])
        assert bad.sum() == 1 and bad[300]
        if eight:
            (m,), (v,) = adamw8bit_values(*[[t[0]] for t in state[2:]])
            for t in (m, v):
                assert torch.isnan(t).sum() == 256
                assert torch.isnan(t[256:512]).all()
        state = make([(600,), (3,)], eight=eight)
        state[1][0][300] = float("nan")
        norm = (adamw8bit_ if eight else adamw_)(*state, step=1, lr=0.1,
                                                 max_norm=1.0)
        assert torch.isnan(norm) and torch.isnan(state[0][1]).all()


def test_zero_gradients_leave_only_decay():
    for eight in (False, True):
        state = make([(600,)], eight=eight)
        state[1][0].zero_()
        was = state[0][0].clone()
        (adamw8bit_ if eight else adamw_)(*state, step=1, lr=0.1,
                                          weight_decay=0.5)
        assert torch.equal(state[0][0], was * (1 - 0.1 * 0.5))
        if eight:
            (m,), (v,) = adamw8bit_values(*[[t[0]] for t in state[2:]])
            assert not m.any() and not v.any()


def test_values_of_all_codes():
    """Every code, in each supported type of value."""
    m = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn)
    v = torch.arange(256, dtype=torch.uint8)
    s = torch.tensor([[0.5, 0.25]])
    (mv,), (vv,) = adamw8bit_values([m], [v], [s])
    want = m.float() * 0.5
    assert torch.equal(mv.nan_to_num(7e7), want.nan_to_num(7e7))
    r = root_value(np.arange(256)) * 0.25
    assert np.array_equal(vv.double().numpy(), r * r)
    assert root_value(np.arange(256)).max() == 1.9375
    for dtype in HALF:
        got = adamw8bit_values([m], [v], [s], dtype=dtype)[1][0]
        assert torch.equal(got, vv.to(dtype))


def test_dither_is_uniform_and_free_of_the_last_step():
    """Mean and spread of 2^16 values: their errors are 1/sqrt(12 n) and
    about 1/sqrt(5 n) of the variance 1/12; five of those are allowed.  Two
    steps are uncorrelated to 5/sqrt(n)."""
    n = 1 << 16
    a, b = (_dither(n, (s * 0xA54FF53A) & 0xFFFFFFFF, "cpu").double() / 2 ** 19
            for s in (7, 8))
    assert abs(a.mean() - 0.5) < 5 / np.sqrt(12 * n)
    assert abs(a.var() * 12 - 1) < 5 * np.sqrt(0.8 / n)
    assert abs(np.corrcoef(a.numpy(), b.numpy())[0, 1]) < 5 / np.sqrt(n)
    assert abs(np.corrcoef(a[1:].numpy(), a[:-1].numpy())[0, 1]) \
        < 5 / np.sqrt(n)


def test_stochastic_rounding_keeps_the_second_moment_moving():
    """Without gradients sqrt(v) must decay with beta2, although one step
    moves it by far less than a code.  Each rounding adds at most 2^-4 of
    the value, with a mean of zero; 200 of them over 1020 elements average
    to a spread of 2^-4 * sqrt(200 / 1020) / 2 = 0.014 at most.  Rounding to
    nearest would stay at 1.  Each block's first element keeps its scale."""
    n, k, b2 = 1024, 200, 0.999
    ps, gs, ms, vs, ss = make([(n,)], eight=True)
    gs[0].fill_(1.0)
    gs[0][::256] = 4.0
    kw = dict(lr=0.0, weight_decay=0.0, betas=(0.9, b2))
    adamw8bit_(ps, gs, ms, vs, ss, step=1, **kw)
    keep = torch.ones(n, dtype=torch.bool)
    keep[::256] = False
    v0 = adamw8bit_values(ms, vs, ss)[1][0][keep].double().sqrt().mean()
    gs[0][keep] = 0.0
    for t in range(2, 2 + k):
        adamw8bit_(ps, gs, ms, vs, ss, step=t, **kw)
    v1 = adamw8bit_values(ms, vs, ss)[1][0][keep].double().sqrt().mean()
    assert abs(float(v1 / v0) - b2 ** (k / 2)) < 0.05
    assert float(v1 / v0) < 0.95


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------

def refused(exc, eight=False, edit=lambda s: None, **kw):
    state = make([(4, 6), (300,)], eight=eight)
    state = tuple(list(x) for x in state)
    edit(state)
    kw = {"step": 1, "lr": 0.1, **kw}
    was = [t.clone() for t in state[0]]
    with pytest.raises(exc):
        (adamw8bit_ if eight else adamw_)(*state, **kw)
    assert all(torch.equal(a, b) for a, b in zip(was, state[0]))


def put(k, i, make_it):
    def edit(state):
        state[k][i] = make_it(state[k][i])
    return edit


@pytest.mark.parametrize("kw", [
    dict(step=0), dict(step=1.5), dict(lr=-1.0), dict(lr=float("nan")),
    dict(eps=-1e-9), dict(weight_decay=-0.1), dict(betas=(1.0, 0.9)),
    dict(betas=(0.9,)), dict(max_norm=-1.0), dict(max_norm=float("nan")),
    dict(total_norm=torch.tensor(1.0)),
    dict(max_norm=1.0, total_norm=torch.ones(2)),
    dict(max_norm=1.0, total_norm=torch.tensor(1.0, dtype=torch.float64)),
])
def test_bad_numbers_are_refused(kw):
    refused(ValueError, **kw)
    refused(ValueError, eight=True, **kw)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("exc,edit", [
    (ValueError, lambda s: s[1].pop()),
    (ValueError, lambda s: s[3].pop()),
    (ValueError, put(1, 0, lambda t: t.view(6, 4))),
    (ValueError, put(1, 0, lambda t: t.t().contiguous().t())),
    (ValueError, put(1, 1, lambda t: t[:299])),
    (ValueError, put(2, 0, lambda t: t.view(24))),
    (TypeError, put(1, 1, lambda t: t.bfloat16())),
    (TypeError, put(2, 0, lambda t: t.float().double())),
    (TypeError, put(3, 0, lambda t: t.to(torch.int16))),
    (ValueError, put(1, 0, lambda t: t.to_sparse())),
    (ValueError, put(1, 0, lambda t: t.to("meta"))),
    # the same weight twice; a moment that is another's; a gradient that is
    # a weight
    (ValueError, lambda s: [x.append(x[0]) for x in s]),
    (ValueError, lambda s: [x.append(x[1].clone()) for x in s[:2]] + [
        x.append(x[1]) for x in s[2:]]),
    (ValueError, lambda s: s[1].__setitem__(1, s[0][1])),
])
def test_bad_lists_are_refused(eight, exc, edit):
    refused(exc, eight=eight, edit=edit)


def test_bad_types_gaps_and_scales_are_refused():
    with pytest.raises(TypeError):
        adamw_(*[[torch.zeros(4, dtype=torch.float64)]] * 2,
               [torch.zeros(4)], [torch.zeros(4)], step=1, lr=0.1)
    gap = [torch.zeros(8)[::2] for _ in range(4)]
    with pytest.raises(ValueError):
        adamw_(*[[t] for t in gap], step=1, lr=0.1)
    for bad in (torch.zeros(1, 2), torch.zeros(2, 2).double(),
                torch.zeros(2, 3), torch.zeros(2, 4)[:, ::2]):
        refused(ValueError, eight=True, edit=put(4, 1, lambda t: bad))
        m, v = torch.zeros(300).to(torch.float8_e4m3fn), \
            torch.zeros(300, dtype=torch.uint8)
        with pytest.raises(ValueError):
            adamw8bit_values([m], [v], [bad])
    with pytest.raises(TypeError):
        adamw8bit_values([v], [v], [torch.zeros(2, 2)])
    with pytest.raises(TypeError):
        adamw8bit_values([m], [v], [torch.zeros(2, 2)], dtype=torch.float64)
    with pytest.raises(ValueError):
        adamw8bit_values([m], [v, v], [torch.zeros(2, 2)])
    with pytest.raises(ValueError):
        grad_norm([])
    with pytest.raises(TypeError):
        grad_norm([torch.zeros(3, dtype=torch.int32)])


def test_one_gradient_for_two_weights_is_allowed():
    ps, gs, ms, vs = make([(300,), (300,)])
    adamw_(ps, [gs[0], gs[0]], ms, vs, step=1, lr=0.1)
    assert torch.equal(ms[0], ms[1])


def test_writes_are_counted():
    """A graph that saved a weight notices that it has changed."""
    for eight in (False, True):
        state = make([(300,)], eight=eight)
        was = [x[0]._version for x in state]
        (adamw8bit_ if eight else adamw_)(*state, step=1, lr=0.1)
        assert [x[0]._version > w for x, w in zip(state, was)] == \
            [True, False] + [True] * (len(state) - 2)


def test_empty_view_inside_another_tensor():
    ps, gs, ms, vs = make([(300,), (0,)])
    ps[1] = ps[0][7:7]
    adamw_(ps, gs, ms, vs, step=1, lr=0.1)


def test_empty_lists():
    assert adamw_([], [], [], [], step=1, lr=0.1) is None
    assert adamw8bit_([], [], [], [], [], step=1, lr=0.1) is None
    assert adamw8bit_values([], [], []) == ([], [])


# ---------------------------------------------------------------------------
# optimizer
# ---------------------------------------------------------------------------

def params(seed=0, dtype=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter(torch.randn(s, generator=gen).to(dtype))
            for s in ((8, 4, 3, 3), (300,), (5, 7))]


def give_grads(ps, seed):
    gen = torch.Generator().manual_seed(seed)
    for p in ps:
        p.grad = torch.randn(p.shape, generator=gen).to(p.dtype)


def test_optimizer_clips_over_all_groups_and_keeps_gradients():
    a, b = params(), params()
    oa = FusedAdamW([{"params": a[:1], "lr": 0.02}, {"params": a[1:]}],
                    lr=0.01, max_grad_norm=0.5)
    ob = torch.optim.AdamW([{"params": b[:1], "lr": 0.02},
                            {"params": b[1:]}], lr=0.01)
    for s in range(3):
        give_grads(a, s)
        give_grads(b, s)
        kept = [p.grad.clone() for p in a]
        oa.step()
        norm = torch.nn.utils.clip_grad_norm_(b, 0.5)
        ob.step()
        assert torch.allclose(oa.last_grad_norm, norm, rtol=1e-6)
        assert all(torch.equal(k, p.grad) for k, p in zip(kept, a))
    for x, y in zip(a, b):
        assert torch.allclose(x, y, rtol=1e-5, atol=1e-6)


def test_optimizer_layouts_missing_gradients_and_late_parameters():
    a, b = params(), params()
    a[0].data = a[0].data.to(memory_format=torch.channels_last)
    oa, ob = FusedAdamW(a, lr=0.01), torch.optim.AdamW(b, lr=0.01)
    for s in range(3):
        give_grads(a, s)   # contiguous gradients of a channels_last weight
        give_grads(b, s)
        if s == 0:
            a[1].grad = b[1].grad = None   # starts a step late
        oa.step()
        ob.step()
    assert [oa.state[p]["step"] for p in a] == [3, 2, 3]
    for x, y in zip(a, b):
        assert torch.allclose(x, y, rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_optimizer_resumes_bit_for_bit(bits, dtype, tmp_path):
    a = params(dtype=dtype)
    oa = FusedAdamW(a, lr=0.01, state_bits=bits, seed=4)
    give_grads(a, 0)
    oa.step()
    torch.save({"o": oa.state_dict(), "p": [p.data for p in a]},
               tmp_path / "c")
    give_grads(a, 1)
    oa.step()
    saved = torch.load(tmp_path / "c", weights_only=True)
    b = [torch.nn.Parameter(t) for t in saved["p"]]
    ob = FusedAdamW(b, lr=0.5, state_bits=bits, seed=4)
    ob.load_state_dict(saved["o"])
    give_grads(b, 1)
    ob.step()
    for x, y in zip(a, b):
        assert torch.equal(x, y)
        for k, t in oa.state[x].items():
            u = ob.state[y][k]
            assert t == u if k == "step" else (
                t.dtype == u.dtype and torch.equal(t.float(), u.float()))


@pytest.mark.parametrize("bits", [8, 32])
def test_optimizer_takes_state_of_torch_adamw(bits):
    a, b = params(), params()
    ob = torch.optim.AdamW(b, lr=0.01)
    give_grads(b, 0)
    ob.step()
    a = [torch.nn.Parameter(p.detach().clone()) for p in b]
    oa = FusedAdamW(a, lr=0.3, state_bits=bits)
    oa.load_state_dict(copy.deepcopy(ob.state_dict()))
    assert oa.param_groups[0]["state_bits"] == bits
    assert all(s["exp_avg"].dtype == torch.float32 for s in oa.state.values())
    give_grads(a, 1)
    give_grads(b, 1)
    oa.step()
    ob.step()
    for x, y in zip(a, b):
        assert torch.allclose(x, y, rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize("bits", [8, 32])
def test_loaded_state_follows_the_memory_format(bits):
    """Saved from contiguous filters, loaded for channels_last ones: the same
    moments at the same indices (8 bits: rounded once more, to half a step
    of a code, 2^-4 of the value and of sqrt(v), or of the least step)."""
    a = params()
    oa = FusedAdamW(a, lr=0.01, state_bits=bits)
    give_grads(a, 0)
    oa.step()
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    b[0].data = b[0].data.to(memory_format=torch.channels_last)
    ob = FusedAdamW(b, lr=0.01, state_bits=bits)
    ob.load_state_dict(oa.state_dict())
    s, t = oa.state[a[0]], ob.state[b[0]]
    assert t["exp_avg"].stride() == b[0].stride()
    if bits == 32:
        assert torch.equal(s["exp_avg"], t["exp_avg"])
        assert torch.equal(s["exp_avg_sq"], t["exp_avg_sq"])
    else:
        (m0,), (v0,) = adamw8bit_values(*[[s[k]] for k in (
            "exp_avg", "exp_avg_sq", "scales")])
        (m1,), (v1,) = adamw8bit_values(*[[t[k]] for k in (
            "exp_avg", "exp_avg_sq", "scales")])
        assert ((m0 - m1).abs() <= 2.0 ** -4 * m0.abs()
                + 2.0 ** -10 * t["scales"][:, 0].max()).all()
        r0, r1 = v0.sqrt(), v1.sqrt()
        assert ((r0 - r1).abs() <= 2.0 ** -5 * 1.01 * r0
                + 2.0 ** -18 * t["scales"][:, 1].max()).all()
    give_grads(b, 1)
    ob.step()


def test_optimizer_refusals():
    p = params()
    other = torch.optim.AdamW(p, lr=0.1, amsgrad=True)
    with pytest.raises(ValueError):
        FusedAdamW(p).load_state_dict(other.state_dict())
    with pytest.raises(ValueError):
        FusedAdamW(params(), state_bits=4)
    with pytest.raises(ValueError):
        FusedAdamW(params(), lr=-1.0)
    with pytest.raises(ValueError):
        FusedAdamW(params(), max_grad_norm=-1.0)
    p = torch.nn.Parameter(torch.zeros(8)[::2])
    p.grad = torch.ones(4)
    with pytest.raises(ValueError):
        FusedAdamW([p]).step()
    e = torch.nn.Embedding(5, 3, sparse=True)
    e(torch.tensor([1])).sum().backward()
    with pytest.raises(ValueError):
        FusedAdamW(e.parameters()).step()


@pytest.mark.parametrize("other", [
    lambda p: torch.optim.SGD(p, lr=0.1, momentum=0.9),
    lambda p: torch.optim.Adam(p, lr=0.1, weight_decay=0.1)])
def test_state_of_other_optimizers(other):
    """Refused, with everything as it was."""
    p = params()
    before = other(p)
    give_grads(p, 0)
    before.step()
    opt = FusedAdamW(p, lr=0.5)
    opt.step()
    kept = [opt.state[x]["exp_avg"].clone() for x in p]
    with pytest.raises(ValueError):
        opt.load_state_dict(before.state_dict())
    assert opt.param_groups[0]["lr"] == 0.5
    assert all(torch.equal(opt.state[x]["exp_avg"], k)
               for x, k in zip(p, kept))
