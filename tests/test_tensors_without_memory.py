"""GPU tensors that only stand for one, as FakeTensorMode and make_fx use
them: their data pointer is null, and a kernel must not get it."""

import pytest
import torch
import torch.nn as nn
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

from moco_amd.ops import (adamw8bit_, adamw8bit_values, adamw_, ext,
                          grad_norm, has_ext, norm_residual)

if not has_ext():
    pytest.skip("the HIP extension is not built", allow_module_level=True)

CALLS = {
    "norm": lambda x: norm_residual(x, x),
    "norm8": lambda x: norm_residual(x, x, scale=x[0]),
    "grad_norm": lambda x: grad_norm([x]),
    "adamw": lambda x: adamw_([x], [x + 1], [x + 2], [x + 3], step=1, lr=0.1),
    "adamw8": lambda x: adamw8bit_(
        [x], [x + 1], [x.to(torch.float8_e4m3fn)], [x.to(torch.uint8)],
        [x.new_zeros(1, 2)], step=1, lr=0.1),
    "values": lambda x: adamw8bit_values(
        [x.to(torch.float8_e4m3fn)], [x.to(torch.uint8)],
        [x.new_zeros(1, 2)])}


def fake(mode):
    with mode:
        return torch.empty(4, 64, device="cuda")


@pytest.mark.parametrize("name", list(CALLS))
def test_inside_the_mode(name):
    """(Without a GPU: the check comes before anything else.)"""
    mode = FakeTensorMode()
    x = fake(mode)
    assert x.is_cuda
    with mode, pytest.raises(NotImplementedError):
        CALLS[name](x)


def test_outside_the_mode():
    x = fake(FakeTensorMode())
    no = [None] * 7
    with pytest.raises(NotImplementedError):
        norm_residual(x, x)
    for call in (lambda: ext().grad_norm([x], False),
                 lambda: ext().adamw_step([x], [x], [x], [x], None, 1, 0.1,
                                          0.9, 0.99, 0.0, 0.0, None, None, 0),
                 lambda: ext().adamw8bit_values([x], [x], [x], torch.float32)):
        with pytest.raises(NotImplementedError):
            call()
    for i in range(7):
        some = list(no)
        some[i] = x
        with pytest.raises(NotImplementedError):
            ext().norm_residual(torch.zeros(4, 64), *some, 1.0, 0, 1, 0, 0.0,
                                0.0, 0)
    with pytest.raises(NotImplementedError):
        t = [torch.zeros(4)]
        ext().adamw_step(t, t, t, t, None, 1, 0.1, 0.9, 0.99, 0.0, 0.0, 1.0,
                         x, 0)


def test_the_cpu_path_takes_them():
    with FakeTensorMode():
        r, y = norm_residual(torch.empty(4, 64), torch.empty(4, 64),
                             pre=nn.LayerNorm(64))
    assert r.shape == y.shape == (4, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(CALLS))
def test_make_fx_is_refused(name):
    """With real tensors too: it would keep the outputs as constants."""
    with pytest.raises(NotImplementedError):
        make_fx(CALLS[name])(torch.randn(4, 64, device="cuda"))


@pytest.mark.gpu
def test_backward_inside_the_mode():
    x = torch.randn(4, 64, device="cuda", requires_grad=True)
    pre = nn.RMSNorm(64, eps=1e-6, device="cuda")
    r, y = norm_residual(x, x, pre=pre)
    mode = FakeTensorMode(allow_non_fake_inputs=True)
    with mode:
        d = mode.from_tensor(torch.zeros(4, 64, device="cuda"))
        with pytest.raises(NotImplementedError):
            torch.autograd.grad(y, x, d)
    got = torch.autograd.grad(y, x, torch.ones_like(y))[0]
    assert torch.isfinite(got).all()


@pytest.mark.gpu
def test_batched_gradients_are_refused():
    x = torch.randn(4, 64, device="cuda", requires_grad=True)
    y = norm_residual(x, pre=nn.RMSNorm(64, eps=1e-6, device="cuda"))[1]
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, x, torch.ones(3, 4, 64, device="cuda"),
                            is_grads_batched=True)
