"""Which norm modules norm_residual takes: those whose own forward pass is the
formula that it computes."""

import pytest
import torch
import torch.nn as nn

from moco_amd.ops import norm_residual


class OnePlusWeight(nn.RMSNorm):
    def forward(self, x):
        return nn.functional.rms_norm(x, self.normalized_shape,
                                      1 + self.weight, self.eps)


class ChannelsFirst(nn.LayerNorm):
    def forward(self, x):
        return super().forward(x.movedim(1, -1)).movedim(-1, 1)


class Called(nn.LayerNorm):
    def __call__(self, x):
        return 2 * super().__call__(x)


def patched(width):
    mod = nn.LayerNorm(width)
    mod.forward = lambda x: 2 * x
    return mod


def hooked(register):
    def make(width):
        mod = nn.LayerNorm(width)
        getattr(mod, register)(lambda *args: None)
        return mod
    return make


@pytest.mark.parametrize("device", [
    "cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("make", [
    lambda w: OnePlusWeight(w, eps=1e-6), ChannelsFirst, Called, patched,
    hooked("register_forward_hook"), hooked("register_forward_pre_hook"),
    hooked("register_full_backward_hook"),
    hooked("register_full_backward_pre_hook")])
def test_modules_that_do_something_else_are_refused(make, device):
    x = torch.randn(2, 8, 8, 8, device=device)
    mod = make(8).to(device)
    with pytest.raises(TypeError):
        norm_residual(x, pre=mod)
    with pytest.raises(TypeError):
        norm_residual(x, x, post=mod)


class Named(nn.LayerNorm):
    """Another constructor, the same forward pass."""

    def __init__(self, width):
        super().__init__(width, eps=1e-3)


class Doubled(nn.Module):
    def forward(self, w):
        return 2 * w


def parametrized(width):
    mod = nn.RMSNorm(width, eps=1e-6)
    nn.utils.parametrize.register_parametrization(mod, "weight", Doubled())
    return mod


def unhooked(width):
    mod = nn.LayerNorm(width)
    mod.register_forward_hook(lambda *args: None).remove()
    return mod


@pytest.mark.parametrize("make", [Named, parametrized, unhooked])
def test_modules_with_the_same_forward_pass(make):
    """Two 32-bit computations of rows of 16 in another order: 64 U of entries
    under 16 at most."""
    x, mod = torch.randn(5, 16), make(16)
    y = norm_residual(x, pre=mod)[1]
    assert (y - mod(x)).abs().max() <= 64 * 2.0 ** -24 * 16
