"""AdamW and its 8-bit moments from the definitions, in 64-bit numpy, with
bounds on what 32-bit arithmetic may differ by.  Shared by the CPU and the
GPU tests."""

import numpy as np
import torch

U = 2.0 ** -24          # half a step of fp32, relative
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8,
        torch.float16: 2.0 ** -11}   # of a 16-bit weight, relative
# half of the least step (fp16's subnormals)
LEAST = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}


def mem(t):
    """Elements in memory order, float64."""
    flat = t.detach().as_strided((t.numel(),), (1,)).cpu()
    if flat.dtype == torch.uint8:
        return flat.numpy().astype(np.int64)
    return flat.float().numpy().astype(np.float64)


def root_value(code):
    e, f = code // 16, code % 16
    return np.where(e == 0, f / 16 * 2.0 ** -14,
                    (1 + f / 16) * 2.0 ** (e - 15.0))


def decode(m, v, s):
    """(m, sqrt(v)) of codes in memory order."""
    rows = np.repeat(s.detach().cpu().double().numpy(), 256,
                     axis=0)[:m.numel()]
    return mem(m) * rows[:, 0], root_value(mem(v)) * rows[:, 1]


def step64(p, g, m, v, step, lr, betas, eps, wd, coef):
    """New p, m, v and how far 32-bit ones may be off.  Bounds count the
    roundings: a factor of 32 bits made from a 64-bit one U, each operation
    U, a square root of 1 ulp 2U, the clip's coefficient 3U."""
    b1, b2 = betas
    a, b = b1 * m, (1 - b1) * (g * coef)
    m2 = a + b
    v2 = b2 * v + (1 - b2) * (g * coef) ** 2
    dm = 8 * U * (abs(a) + abs(b))
    dv = 14 * U * v2
    denom = np.sqrt(v2) / np.sqrt(1 - b2 ** step) + eps
    ss = lr / (1 - b1 ** step)
    q = m2 / denom
    p2 = p * (1 - lr * wd) - ss * q
    dp = 3 * U * abs(p) + ss * (dm / denom + 18 * U * abs(q)) + U * abs(p2)
    # what 32 bits hold no smaller than
    return p2, m2, v2, dp + 1e-44, dm + 1e-44, dv + 1e-44


def dither(n, i, step, seed):
    """19 random bits of the elements of tensor i."""
    mask = 0xFFFFFFFF
    x = [(e + seed * 0x6A09E667 + step * 0xA54FF53A + i * 0x3C6EF372) & mask
         for e in range(n)]
    x = np.array(x, dtype=np.uint64)
    x = (x * np.uint64(0x9E3779B9)) & np.uint64(mask)
    x ^= x >> np.uint64(15)
    x = (x * np.uint64(0xBB67AE85)) & np.uint64(mask)
    x ^= x >> np.uint64(16)
    return (x >> np.uint64(13)).astype(np.float64) / 2 ** 19


def block_max(x):
    pad = np.pad(abs(x), (0, -len(x) % 256)).reshape(-1, 256)
    return np.maximum(pad.max(1), 1e-30)


def check_codes(m2, r2, dm, codes_m, codes_v, scales, i, step, seed):
    """The stored 8-bit moments against 64-bit m2 and r2 = sqrt(v2)."""
    n = len(m2)
    s = scales.detach().cpu().double().numpy()
    assert s.shape == (-(-n // 256), 2)
    # a maximum is off by its element's error: 8U, the product by 2U more
    assert np.allclose(s[:, 0], block_max(m2) / 448.0, rtol=1e-5, atol=0)
    assert np.allclose(s[:, 1], block_max(r2) / 1.9375, rtol=16 * U, atol=0)
    sm, sr = (np.repeat(s[:, k], 256)[:n] for k in (0, 1))
    # m: half a step of e4m3 (2^-4 of the value, at least half of 2^-9)
    q = m2 / sm
    off = abs(mem(codes_m) - q)
    assert (off <= np.maximum(abs(q) * 2.0 ** -4, 2.0 ** -10)
            + dm / sm + 8 * U * abs(q)).all()
    # sqrt(v): the code below or above, as the dither says; where the sum is
    # within 1e-3 of a code's border, either (32-bit errors are 20U of q,
    # 20U * 32 = 4e-5 of a code)
    q = r2 / sr
    e = np.floor(np.log2(np.maximum(q, 2.0 ** -14)))
    place = (e + 14) * 16 + q / 2.0 ** e * 16 + dither(n, i, step, seed)
    want = np.where(r2 > 0, np.clip(np.floor(place), 1, 255), 0)
    near = abs(place - np.round(place)) < 1e-3
    got = mem(codes_v)
    assert (near | (got == want)).all()
    assert (abs(got - want) <= 1).all()
    assert ((got > 0) == (r2 > 0)).all()
