"""Gradients whose squares are next to the least 32-bit numbers: second
moments down to the subnormal ones, with eps = 0."""

import numpy as np
import pytest
import torch

from adamw_oracle import U, dither
from moco_amd.ops import adamw8bit_, adamw_

f = np.float32
B1, B2, LR = 0.9, 0.999, 1e-3


def gradients(n, seed):
    """1e-23 to 1e-10, every sign, some zeros.  Squares below 1.4e-45 are
    zeros in 32 bits, those below 1.2e-38 subnormal, and so is 0.001 of
    them."""
    rng = np.random.default_rng(seed)
    g = 10.0 ** rng.uniform(-23, -10, n) * rng.choice([-1, 1], n)
    g[::97] = 0.0
    return g.astype(f)


devices = pytest.mark.parametrize("device", [
    "cpu", pytest.param("cuda", marks=pytest.mark.gpu)])


@devices
@pytest.mark.parametrize("eps", [0.0, 1e-20])
def test_weights(device, eps):
    """v is that of numpy's 32-bit operations.  m / (sqrt(v) / c + eps), from
    v on: the root U, c U, the product and the sum U, the reciprocal 2U, the
    product U; under 8U of the quotient.  Where v is zero and eps too, a
    quotient is infinite, or no number."""
    n = 50_000
    g = gradients(n, 0)
    p = np.random.default_rng(1).standard_normal(n).astype(f)
    t = [torch.from_numpy(x.copy()).to(device)
         for x in (p, g, np.zeros(n, f), np.zeros(n, f))]
    adamw_(*[[x] for x in t], step=1, lr=LR, betas=(B1, B2), eps=eps,
           weight_decay=0.0)
    m = g * f(1 - B1)
    v = (g * g) * f(1 - B2)
    assert (v[v > 0] < 2.0 ** -126).any() and (v == 0).any()
    assert np.array_equal(t[2].cpu().numpy(), m)
    assert np.array_equal(t[3].cpu().numpy(), v)
    with np.errstate(all="ignore"):
        q = m.astype(float) / (np.sqrt(v.astype(float))
                               / np.sqrt(1 - B2) + eps)
    got = t[0].cpu().numpy().astype(float)
    ok = np.isfinite(q)
    if eps == 0.0:
        assert (~ok == (v == 0)).all()
    else:
        assert ok.all()
    assert (np.isfinite(got) == ok).all()
    step = LR / (1 - B1) * q[ok]
    want = p[ok] - step
    assert (abs(got[ok] - want)
            <= 9 * U * abs(step) + U * abs(want) + 2 * U * abs(p[ok])).all()


def codes(n, device):
    """Weights, no gradients yet, empty moments and scales."""
    st = [torch.ones(n), None, torch.zeros(n).to(torch.float8_e4m3fn),
          torch.zeros(n, dtype=torch.uint8), torch.zeros(-(-n // 256), 2)]
    return [None if t is None else t.to(device) for t in st]


@devices
def test_a_second_moment_above_zero_keeps_a_code(device):
    n = 20_001
    st = codes(n, device)
    g = gradients(n, 5)
    st[1] = torch.from_numpy(g.copy()).to(device)
    adamw8bit_(*[[x] for x in st], step=1, lr=LR, betas=(B1, B2))
    v = (g * g) * f(1 - B2)
    assert ((v > 0) & (v < 2.0 ** -126)).any()
    assert ((st[3].cpu().numpy() > 0) == (v > 0)).all()


@pytest.mark.gpu
def test_codes():
    """Bit for bit those of 32-bit operations over three steps.  (The CPU's
    library root is off by an ulp here and there.)"""
    n, device = 20_001, "cuda"
    rows = -(-n // 256)
    st = codes(n, device)
    m, r = np.zeros(rows * 256, f), np.zeros(rows * 256, f)
    below = 0
    for step in range(1, 4):
        g = np.zeros(rows * 256, f)
        # whole blocks of small ones, so that their scales are small too
        g[:n] = gradients(n, step) * f(2.0 ** -10)
        st[1] = torch.from_numpy(g[:n].copy()).to(device)
        adamw8bit_(*[[x] for x in st], step=step, seed=4, lr=LR,
                   betas=(B1, B2))
        m = m * f(B1) + g * f(1 - B1)
        v = (r * r) * f(B2) + (g * g) * f(1 - B2)
        r = np.sqrt(v)
        m, r = m.reshape(-1, 256), r.reshape(-1, 256)
        sm = np.maximum(abs(m).max(1, keepdims=True), f(1e-30)) * f(1 / 448)
        sr = np.maximum(r.max(1, keepdims=True), f(1e-30)) * f(1 / 1.9375)
        assert np.array_equal(st[4].cpu().numpy(), np.hstack([sm, sr]))
        mc = torch.from_numpy(np.clip(m * (f(1) / sm), f(-448), f(448))).to(
            torch.float8_e4m3fn)
        bits = (r * (f(1) / sr) * f(2.0 ** -112)).view(np.int32)
        up = (dither(rows * 256, 0, step, 4) * 2 ** 19).astype(np.int32)
        rc = np.minimum((bits + up.reshape(-1, 256)) >> 19, 255)
        rc = np.where(r > 0, np.maximum(rc, 1), 0)
        below += ((v > 0) & (v < 2.0 ** -126)).sum()
        got = st[3].cpu().numpy()
        assert ((got > 0) == (v[:n] > 0)).all()
        assert np.array_equal(got, rc.reshape(-1)[:n])
        assert torch.equal(st[2].cpu().float(), mc.float().view(-1)[:n])
        m = (mc.float().numpy() * sm).reshape(-1)
        r = ((rc.astype(np.int32) << 19).view(f) * f(2.0 ** 112)
             * sr).reshape(-1)
    assert below > 1000
