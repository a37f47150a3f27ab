"""AdamW and grad_norm over more tensors than a launch's table holds, more
than 65536, and more bytes than the last-level cache."""

import numpy as np
import pytest
import torch

from adamw_oracle import HALF
from moco_amd.ops import adamw8bit_, adamw_, grad_norm

pytestmark = pytest.mark.gpu

f = np.float32


@pytest.mark.parametrize("size", [3, 4099])
@pytest.mark.parametrize("types", [[t] for t in HALF] + [list(HALF)])
def test_norm_of_600_gradients(size, types):
    gen = torch.Generator().manual_seed(0)
    gs = [(torch.randn(size, generator=gen) * 10.0 ** -(i % 5)).to(
        types[i % len(types)]).cuda() for i in range(600)]
    want = np.sqrt(sum((g.double().cpu().numpy() ** 2).sum() for g in gs))
    got = grad_norm(gs)
    # the root's rounding and the one to 32 bits
    assert abs(float(got) - want) <= 2 * 2.0 ** -24 * want


def test_numbers_of_65626_tensors():
    """Two elements each, the first of which sets the scales, so that the
    second's code goes by the rounding hash of the tensor's number."""
    n, seed, step, b1, b2 = 65536 + 90, 5, 1, 0.9, 0.999
    rng = np.random.default_rng(0)
    g = rng.standard_normal((n, 2)).astype(f)
    g[:, 1] = g[:, 0] * rng.uniform(0.05, 0.95, n)
    flat = [torch.zeros(n, 2), torch.from_numpy(g),
            torch.zeros(n, 2).to(torch.float8_e4m3fn),
            torch.zeros(n, 2, dtype=torch.uint8), torch.zeros(n, 1, 2)]
    flat = [t.cuda() for t in flat]
    adamw8bit_(*[list(t.unbind(0)) for t in flat], step=step, seed=seed,
               lr=0.1, betas=(b1, b2))
    # 32-bit operations, one by one
    r = np.sqrt((g * g) * f(1 - b2))
    sr = r.max(1, keepdims=True) * f(1 / 1.9375)
    bits = (r * (f(1) / sr) * f(2.0 ** -112)).view(np.int32)
    mask = np.uint64(0xFFFFFFFF)
    x = (np.arange(n, dtype=np.uint64)[:, None] * np.uint64(0x3C6EF372)
         + np.arange(2, dtype=np.uint64)
         + np.uint64(seed * 0x6A09E667 + step * 0xA54FF53A)) & mask
    x = (x * np.uint64(0x9E3779B9)) & mask
    x ^= x >> np.uint64(15)
    x = (x * np.uint64(0xBB67AE85)) & mask
    x ^= x >> np.uint64(16)
    codes = (bits + (x >> np.uint64(13)).astype(np.int32)) >> 19
    codes = np.where(r > 0, np.clip(codes, 1, 255), 0)
    got = flat[3].cpu().numpy()
    assert len(np.unique(got[:, 1])) > 30
    assert np.array_equal(flat[4].cpu().numpy()[:, 0, 1], sr[:, 0])
    assert np.array_equal(got, codes)


def filled(n, dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(n, device="cuda", generator=gen).to(dtype)


@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("eight", [False, True])
def test_a_call_past_the_caches_is_the_same(dtype, eight):
    """A call of 300 MB against calls of a third of it: bit for bit.  Tensors
    that are left out are replaced by empty ones, which keeps the others'
    numbers."""
    size = torch.finfo(dtype).bits // 8
    n = (300 << 20) // (2 * size + (2 if eight else 8)) // 3
    sizes = [n, n + 4097, n - 255]
    ps = [filled(k, dtype, i) for i, k in enumerate(sizes)]
    gs = [filled(k, dtype, 9 + i) * 0.01 for i, k in enumerate(sizes)]
    st = [ps, gs]
    if eight:
        st += [[torch.zeros(k, device="cuda", dtype=torch.uint8).view(
            torch.float8_e4m3fn) for k in sizes],
            [torch.zeros(k, device="cuda", dtype=torch.uint8) for k in sizes],
            [torch.zeros(-(-k // 256), 2, device="cuda") for k in sizes]]
    else:
        st += [[torch.zeros(k, device="cuda") for k in sizes]
               for _ in range(2)]
    assert sum(t.nbytes for x in st for t in x) > 256 << 20
    other = [[t.clone() for t in x] for x in st]
    call = adamw8bit_ if eight else adamw_
    for step in (1, 2):
        call(*st, step=step, lr=1e-2)
        for i in range(3):
            call(*[[t if j == i else t[:0] for j, t in enumerate(x)]
                   for x in other], step=step, lr=1e-2)
    for x, y in zip(st, other):
        for a, b in zip(x, y):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("dtype", list(HALF))
def test_norm_of_300_mb(dtype):
    n = (300 << 20) // (torch.finfo(dtype).bits // 8)
    g = filled(n + 77, dtype, 0)
    want = sum(float(c.double().square().sum()) for c in g.split(1 << 24))
    want = np.sqrt(want)
    for gs in ([g], list(g.split(n // 5 + 3))):
        assert abs(float(grad_norm(gs)) - want) <= 2 * 2.0 ** -24 * want
