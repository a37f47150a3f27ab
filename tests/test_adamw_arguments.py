"""AdamW's numbers in the forms that its checks let pass."""

import numpy as np
import pytest
import torch

from moco_amd.ops import adamw8bit_, adamw_

devices = pytest.mark.parametrize("device", [
    "cpu", pytest.param("cuda", marks=pytest.mark.gpu)])


def state(eight, device):
    torch.manual_seed(0)
    p, g = (torch.randn(600).to(device) for _ in range(2))
    out = [[p], [g], [torch.zeros_like(p)], [torch.zeros_like(p)]]
    if eight:
        out[2:] = [[out[2][0].to(torch.float8_e4m3fn)],
                   [out[3][0].to(torch.uint8)],
                   [torch.zeros(3, 2, device=device)]]
    return out


@devices
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("step", [2.0, np.int64(2), np.float32(2),
                                  torch.tensor(2.0), torch.tensor(2)])
def test_a_step_count_of_any_type(device, eight, step):
    call = adamw8bit_ if eight else adamw_
    a, b = state(eight, device), state(eight, device)
    call(*a, step=2, lr=0.1)
    call(*b, step=step, lr=0.1)
    for x, y in zip(a, b):
        assert torch.equal(x[0].view(torch.uint8), y[0].view(torch.uint8))


@devices
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("to", [np.float32, torch.tensor])
def test_numbers_of_any_type(device, eight, to):
    """Each is taken as the double that it is."""
    call = adamw8bit_ if eight else adamw_
    a, b = state(eight, device), state(eight, device)
    kw = {k: to(x) for k, x in dict(lr=0.003, eps=1e-7, weight_decay=0.1,
                                    max_norm=3.1).items()}
    betas = to(0.9), to(0.99)
    call(*a, step=3, betas=tuple(float(x) for x in betas),
         **{k: float(x) for k, x in kw.items()})
    call(*b, step=3, betas=betas, **kw)
    for x, y in zip(a, b):
        assert torch.equal(x[0].view(torch.uint8), y[0].view(torch.uint8))


@devices
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("which", [0, 2, 3, 4])
def test_a_norm_among_what_is_written(device, eight, which):
    """A workgroup might read it after another has written it."""
    if which >= (5 if eight else 4):
        return
    call = adamw8bit_ if eight else adamw_
    st = state(eight, device)
    was = [x[0].clone() for x in st]
    flat = st[which][0].view(-1).view(torch.uint8)
    at = 8 if which == 4 else 256
    norm = flat[at:at + 4].view(torch.float32)
    with pytest.raises(ValueError):
        call(*st, step=1, lr=0.1, max_norm=1.0, total_norm=norm)
    for x, y in zip(was, st):
        assert torch.equal(x.view(torch.uint8), y[0].view(torch.uint8))


@devices
@pytest.mark.parametrize("eight", [False, True])
def test_a_norm_among_the_gradients(device, eight):
    """Only read, so allowed."""
    call = adamw8bit_ if eight else adamw_
    a, b = state(eight, device), state(eight, device)
    norm = a[1][0][4]
    out = call(*a, step=1, lr=0.1, max_norm=1.0, total_norm=norm)
    call(*b, step=1, lr=0.1, max_norm=1.0, total_norm=norm.clone())
    assert out is norm or torch.equal(out, norm)
    for x, y in zip(a, b):
        assert torch.equal(x[0].view(torch.uint8), y[0].view(torch.uint8))
