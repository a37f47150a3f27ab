"""torch.jit.trace cannot follow the kernels' own calls: what they return
would become constants of the traced program, and what they write would be
left out of it.  On the GPU that is an error."""

import pytest
import torch
import torch.nn as nn

from moco_amd.ops import (adamw8bit_, adamw8bit_values, adamw_, grad_norm,
                          norm_residual)


def norm(x):
    return norm_residual(x, pre=nn.RMSNorm(64, eps=1e-6, device=x.device))[1]


def step(x):
    p = torch.zeros_like(x)
    adamw_([p], [x], [torch.zeros_like(x)], [torch.zeros_like(x)], step=1,
           lr=0.1)
    return p


def step8(x):
    p = torch.zeros_like(x)
    m = torch.zeros_like(x, dtype=torch.float8_e4m3fn)
    v = torch.zeros_like(x, dtype=torch.uint8)
    adamw8bit_([p], [x], [m], [v], [torch.zeros(1, 2, device=x.device)],
               step=1, lr=0.1)
    return p


def values(x):
    codes = torch.ones_like(x, dtype=torch.uint8)
    return adamw8bit_values([codes.view(torch.float8_e4m3fn)], [codes],
                            [x.new_ones(1, 2)])[1][0] * x


@pytest.mark.gpu
@pytest.mark.parametrize("call", [
    norm, step, step8, values, lambda x: grad_norm([x])])
def test_tracing_is_refused_on_the_gpu(call):
    x = torch.randn(2, 64, device="cuda")
    want = call(x)
    with pytest.raises(NotImplementedError):
        torch.jit.trace(call, (x,), check_trace=False)
    with torch.no_grad(), pytest.raises(NotImplementedError):
        torch.jit.trace(call, (x,), check_trace=False)
    assert torch.equal(call(x), want)


def test_the_cpu_path_is_traced():
    traced = torch.jit.trace(norm, (torch.randn(2, 64),), check_trace=False)
    x = torch.randn(2, 64)
    assert torch.equal(traced(x), norm(x))
