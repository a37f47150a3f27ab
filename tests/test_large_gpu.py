"""Tensors of more than 2^32 elements: places behind that get what a small
call gives them."""

import numpy as np
import pytest
import torch

from adamw_oracle import check_codes, mem, step64

pytestmark = pytest.mark.gpu

N = (1 << 32) + 5003


@pytest.fixture(autouse=True)
def room():
    if torch.cuda.mem_get_info()[0] < 120 << 30:
        pytest.skip("needs 120 GB of free device memory")
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("eight", [False, True])
def test_adamw_over_4e9_elements(eight):
    from moco_amd.ops import adamw8bit_, adamw8bit_values, adamw_, grad_norm
    dev = "cuda"
    p = torch.full((N,), 0.5, device=dev, dtype=torch.bfloat16)
    g = torch.zeros(N, device=dev, dtype=torch.bfloat16)
    # whole blocks of 256: their scales depend on nothing else
    spans = [slice(0, 4096), slice((1 << 31) - 2048, (1 << 31) + 2048),
             slice((1 << 32) - 2048, (1 << 32) + 2048),
             slice((1 << 32) + 4096, N)]
    gen = torch.Generator(device=dev).manual_seed(0)
    for s in spans:
        g[s] = torch.randn(s.stop - s.start, device=dev, generator=gen).to(
            torch.bfloat16)
    norm = grad_norm([g])
    want = np.sqrt(sum((mem(g[s]) ** 2).sum() for s in spans))
    assert abs(float(norm) - want) <= 2 * 2.0 ** -24 * want
    kw = dict(step=3, lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
    if eight:
        m = torch.zeros(N, device=dev, dtype=torch.uint8).view(
            torch.float8_e4m3fn)
        v = torch.zeros(N, device=dev, dtype=torch.uint8)
        sc = torch.zeros(-(-N // 256), 2, device=dev)
        adamw8bit_([p], [g], [m], [v], [sc], seed=1, **kw)
    else:
        m, v = (torch.zeros(N, device=dev) for _ in range(2))
        adamw_([p], [g], [m], [v], **kw)
    for s in spans:
        gs = mem(g[s])
        zero = np.zeros(len(gs))
        p2, m2, v2, dp, dm, dv = step64(
            zero + 0.5, gs, zero, zero, 3, 1e-2, (0.9, 0.99), 1e-8, 0.1, 1.0)
        assert (abs(mem(p[s]) - p2) <= dp + 2.0 ** -8 * (abs(p2) + dp)).all()
        if not eight:
            assert (abs(mem(m[s]) - m2) <= dm).all()
            assert (abs(mem(v[s]) - v2) <= dv).all()
            continue
        # the rounding hash counts elements modulo 2^32: check_codes counts
        # from 0, a seed's multiple is added for what lies before (the hash
        # adds seed * 0x6A09E667, which is odd: solved for the start)
        start = s.start & 0xFFFFFFFF
        shift = start * pow(0x6A09E667, -1, 1 << 32) & 0xFFFFFFFF
        rows = slice(s.start // 256, -(-s.stop // 256))
        check_codes(m2, np.sqrt(v2), dm, m[s], v[s], sc[rows], 0, 3,
                    1 + shift)
    if eight:
        (mv,), (vv,) = adamw8bit_values([m], [v], [sc], dtype=torch.bfloat16)
        a = adamw8bit_values([m[spans[2]]], [v[spans[2]]],
                             [sc[spans[2].start // 256:
                                 spans[2].stop // 256].contiguous()],
                             dtype=torch.bfloat16)
        assert torch.equal(mv[spans[2]], a[0][0])
        assert torch.equal(vv[spans[2]], a[1][0])


def test_norm_residual_over_4e9_elements():
    """Rows do not depend on each other: the last ones, far behind 2^32
    elements, are those of a small call."""
    from moco_amd.ops import norm_residual
    dev, width = "cuda", 4099
    rows = (1 << 32) // width + 77
    post, pre = (torch.nn.RMSNorm(width, eps=1e-6, device=dev)
                 for _ in range(2))

    def big():
        t = torch.ones(rows, width, device=dev, dtype=torch.bfloat16)
        t[-100:] = torch.randn(100, width, device=dev).to(torch.bfloat16)
        return t.requires_grad_()
    x, h = big(), big()
    r, y = norm_residual(x, h, post=post, pre=pre, scale=0.5)
    d = [torch.zeros(rows, width, device=dev, dtype=torch.bfloat16)
         for _ in range(2)]
    for t in d:
        t[-100:] = torch.randn(100, width, device=dev).to(torch.bfloat16)
    got = torch.autograd.grad((r, y), (x, h, post.weight, pre.weight), d)
    xs, hs = (t.detach()[-100:].clone().requires_grad_() for t in (x, h))
    rs, ys = norm_residual(xs, hs, post=post, pre=pre, scale=0.5)
    want = torch.autograd.grad((rs, ys), (xs, hs, post.weight, pre.weight),
                               [t[-100:] for t in d])
    assert torch.equal(r[-100:], rs) and torch.equal(y[-100:], ys)
    for a, b in zip(got[:2], want[:2]):
        assert torch.equal(a[-100:], b)
        assert not a[:1000].any()
    # the other rows add zeros: only the order of the sums differs, 100
    # terms of order one
    for a, b in zip(got[2:], want[2:]):
        assert torch.allclose(a, b, atol=200 * 2.0 ** -24 * 100)
