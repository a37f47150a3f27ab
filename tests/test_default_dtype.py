"""torch.set_default_dtype does not reach the optimizer's state or results."""

import pytest
import torch
import torch.nn as nn

from moco_amd.ops import FusedAdamW, norm_residual


@pytest.mark.parametrize("device", [
    "cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("default", [torch.float64, torch.bfloat16])
def test_default_dtype(device, bits, default):
    torch.manual_seed(0)
    x = torch.randn(9, 48, device=device)
    pre = nn.RMSNorm(48, eps=1e-6, device=device)

    def train():
        p = nn.Parameter(x.clone())
        opt = FusedAdamW([p], lr=0.1, state_bits=bits, max_grad_norm=0.5)
        for _ in range(2):
            opt.zero_grad()
            r, y = norm_residual(p, x, pre=pre, scale=0.3)
            (r * y).sum().backward()
            opt.step()
        opt.load_state_dict(opt.state_dict())
        return [p.detach(), opt.last_grad_norm, *(
            t for k, t in opt.state[p].items() if k != "step")]

    want = train()
    old = torch.get_default_dtype()
    torch.set_default_dtype(default)
    try:
        got = train()
    finally:
        torch.set_default_dtype(old)
    for a, b in zip(want, got):
        assert a.dtype == b.dtype
        assert torch.equal(a.reshape(-1).view(torch.uint8),
                           b.reshape(-1).view(torch.uint8))
