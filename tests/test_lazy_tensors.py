"""Tensors whose memory does not hold their values: negated ones (the
imaginary part of a conjugate) and zeros without memory."""

import pytest
import torch
import torch.nn as nn

from moco_amd.ops import (adamw8bit_, adamw8bit_values, adamw_, grad_norm,
                          norm_residual)

devices = pytest.mark.parametrize("device", [
    "cpu", pytest.param("cuda", marks=pytest.mark.gpu)])


def negated(t):
    return torch._neg_view(-t)


def test_a_conjugates_imaginary_part_is_one():
    part = torch.complex(torch.ones(1), torch.ones(1)).conj().imag
    assert part.is_neg() and part.item() == -1.0
    assert negated(torch.ones(3)).is_neg()


@devices
@pytest.mark.parametrize("post,pre", [("rms", "layer"), ("layer", "rms")])
def test_norm_residual_takes_their_values(device, post, pre):
    torch.manual_seed(0)
    width = 40
    make = {"rms": lambda: nn.RMSNorm(width, eps=1e-6),
            "layer": lambda: nn.LayerNorm(width)}
    mods = [make[k]().to(device) for k in (post, pre)]
    for mod in mods:
        mod.weight.data = torch.randn(width, device=device)
    x, h, g, d_r, d_y = (torch.randn(7, width, device=device)
                         for _ in range(5))
    s = torch.randn(width, device=device)

    def run(lazy):
        leaves = [lazy(t).requires_grad_() for t in (x, h, g, s)]
        out = norm_residual(*leaves[:2], post=mods[0], pre=mods[1],
                            gate=leaves[2], gate_act="silu", scale=leaves[3])
        return (*out, *torch.autograd.grad(out, leaves,
                                           (lazy(d_r), lazy(d_y))))
    for a, b in zip(run(torch.clone), run(negated)):
        assert torch.equal(a, b)


@devices
def test_grad_norm_of_negated_and_missing_values(device):
    t = torch.randn(300, device=device)
    zeros = torch._efficientzerotensor((5,), device=device,
                                       dtype=torch.float32)
    assert torch.equal(grad_norm([negated(t), zeros]), grad_norm([t]))
    assert float(grad_norm([zeros])) == 0.0


@pytest.mark.gpu
def test_norm_residual_of_zeros_without_memory():
    x = torch.randn(3, 40, device="cuda", requires_grad=True)
    zeros = torch._efficientzerotensor((3, 40), device="cuda",
                                       dtype=torch.float32)
    pre = nn.RMSNorm(40, eps=1e-6, device="cuda")
    r, y = norm_residual(zeros, x, pre=pre)
    want = norm_residual(torch.zeros_like(x), x, pre=pre)
    assert torch.equal(r, want[0]) and torch.equal(y, want[1])
    r, y = norm_residual(x, zeros, pre=pre)
    assert torch.equal(r, x) and torch.equal(y, norm_residual(x, pre=pre)[1])


@pytest.mark.gpu
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("which", range(5))
@pytest.mark.parametrize("lazy", [negated, lambda t: torch.
                                  _efficientzerotensor(t.shape, dtype=t.dtype,
                                                       device=t.device)])
def test_adamw_refuses_them(eight, which, lazy):
    p, g, m, v = (torch.randn(600, device="cuda") for _ in range(4))
    st = [p, g, m, v]
    if eight:
        st[2:] = [m.to(torch.float8_e4m3fn), v.to(torch.uint8),
                  torch.ones(3, 2, device="cuda")]
    if which >= len(st) or (lazy is negated and
                            st[which].dtype != torch.float32):
        return
    st[which] = lazy(st[which])
    was = p.clone()
    with pytest.raises(ValueError):
        (adamw8bit_ if eight else adamw_)(*[[t] for t in st], step=1, lr=0.1)
    if eight and which >= 2:
        with pytest.raises(ValueError):
            adamw8bit_values(*[[t] for t in st[2:]])
    torch.cuda.synchronize()
    assert torch.equal(p, was)
    with pytest.raises(ValueError):
        adamw_([p], [g], [m], [v], step=1, lr=0.1, max_norm=1.0,
               total_norm=lazy(g[:1].clone()))
