"""States that do not fit the parameters are refused, before anything is
loaded."""

import copy

import pytest
import torch

from moco_amd.ops import FusedAdamW


def stepped(shape, bits, seed=0):
    torch.manual_seed(seed)
    p = torch.nn.Parameter(torch.randn(shape))
    opt = FusedAdamW([p], lr=0.1, state_bits=bits)
    p.grad = torch.randn(shape)
    opt.step()
    return p, opt


def refused(opt, p, state):
    kept = copy.deepcopy(opt.state_dict())
    with pytest.raises(ValueError):
        opt.load_state_dict(state)
    now = opt.state_dict()
    assert now["param_groups"] == kept["param_groups"]
    for k, t in kept["state"][0].items():
        u = now["state"][0][k]
        assert t == u if k == "step" else torch.equal(
            t.view(torch.uint8), u.view(torch.uint8))


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("saved,shape", [
    ((4, 6), (3, 4, 6)), ((6,), (4, 6)), ((1,), (300,)), ((), (300,)),
    ((300,), (301,)), ((4, 6), (24,)), ((4, 6), (6, 4))])
def test_moments_of_another_shape(bits, saved, shape):
    """Those that would broadcast among them."""
    _, old = stepped(saved, bits)
    p, opt = stepped(shape, bits, 1)
    refused(opt, p, old.state_dict())
    refused(opt, p, {**torch.optim.AdamW([torch.nn.Parameter(torch.zeros(
        saved))]).state_dict(), "state": {0: {
            "step": torch.tensor(1.0), "exp_avg": torch.zeros(saved),
            "exp_avg_sq": torch.zeros(saved)}}})


def edited(state, **entries):
    state = copy.deepcopy(state)
    state["state"][0].update(entries)
    return state


@pytest.mark.parametrize("entry", [
    dict(scales=torch.zeros(1, 2)), dict(scales=torch.zeros(2, 2).double()),
    dict(scales=torch.zeros(4)), dict(exp_avg=torch.zeros(300)),
    dict(exp_avg=torch.zeros(300, dtype=torch.float8_e5m2)),
    dict(exp_avg_sq=torch.zeros(300)),
    dict(exp_avg_sq=torch.zeros(300, dtype=torch.int8)),
    dict(exp_avg_sq=torch.zeros(299, dtype=torch.uint8)),
    dict(scales=3.0), dict(exp_avg=3.0)])
def test_codes_without_their_scales_or_types(entry):
    p, opt = stepped((300,), 8)
    refused(opt, p, edited(opt.state_dict(), **entry))


@pytest.mark.parametrize("entry", [
    dict(exp_avg=torch.zeros(300, dtype=torch.float8_e4m3fn)),
    dict(exp_avg_sq=torch.zeros(300, dtype=torch.uint8)),
    dict(exp_avg=torch.zeros(300).double()), dict(exp_avg=None),
    dict(exp_avg=torch.zeros(300).to_sparse()),
    dict(step=-1), dict(step=torch.tensor(1.5)), dict(step=None)])
def test_moments_and_steps_that_are_none(entry):
    p, opt = stepped((300,), 32)
    refused(opt, p, edited(opt.state_dict(), **entry))


def test_a_second_parameter_of_another_shape():
    """The first one's state is not loaded either."""
    ps = [torch.nn.Parameter(torch.randn(s)) for s in ((5,), (4, 6))]
    qs = [torch.nn.Parameter(torch.randn(s)) for s in ((5,), (6,))]
    a, b = FusedAdamW(ps), FusedAdamW(qs)
    for p in ps + qs:
        p.grad = torch.randn_like(p)
    a.step()
    b.step()
    refused(a, ps[0], b.state_dict())
