"""norm_residual and its gradients from the formulas, in 64 bits, with bounds
on what 32-bit arithmetic may differ by.  Shared by CPU and GPU tests."""

import torch

U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8,
        torch.float16: 2.0 ** -11}


def hat_of(t, kind):
    kind_, eps = kind
    if kind_ == "layer":
        t = t - t.mean(-1, keepdim=True)
    inv = (t.square().mean(-1, keepdim=True) + eps).rsqrt()
    return t * inv, inv


def back(t, hat, inv, layer):
    out = t - hat * (t * hat).mean(-1, keepdim=True)
    return inv * (out - t.mean(-1, keepdim=True) if layer else out)


def columns(a, b=None):
    """Sum over rows of a * b, and the size that its error goes by.  a and b
    are rows from a chain that may cancel, so an entry is off by a share of
    its row's largest entry (as in check), not of itself; the product is then
    off by that share of (1 + max|a|) |b| + (1 + max|b|) |a|."""
    if b is None:
        return a.sum(0), (1 + a.abs().amax(-1, keepdim=True)
                          + 0 * a.abs()).sum(0)
    size = (1 + a.abs().amax(-1, keepdim=True)) * b.abs() + \
        (1 + b.abs().amax(-1, keepdim=True)) * a.abs()
    return (a * b).sum(0), size.sum(0)


def formula(x, h, gate, act, scale, post, pre, d_r=None, d_y=None):
    """post, pre: None or (kind, eps, weight, bias).  Returns a dict of r, y
    and the gradients, in float64; a gradient that is summed over rows comes
    with the size of its error (columns)."""
    out = {}
    one = torch.ones(1, dtype=torch.float64)
    if h is not None:
        if post:
            h_hat, h_inv = hat_of(h, post[:2])
            w1 = one if post[2] is None else post[2]
            n = h_hat * w1 + (0 if post[3] is None else post[3])
        else:
            n = h
        g = one if gate is None else gate
        sig = torch.sigmoid(g)
        a, slope = {None: (g, torch.ones_like(g)),
                    "sigmoid": (sig, sig * (1 - sig)),
                    "silu": (g * sig, sig * (1 + g * (1 - sig)))}[act]
        s = one if scale is None else scale
        r = x + s * a * n
        out["r"] = r
    else:
        r = x
    d = torch.zeros_like(x) if d_r is None else d_r
    if pre:
        r_hat, r_inv = hat_of(r, pre[:2])
        w2 = one if pre[2] is None else pre[2]
        out["y"] = r_hat * w2 + (0 if pre[3] is None else pre[3])
        if d_y is not None:
            d = d + back(d_y * w2, r_hat, r_inv, pre[0] == "layer")
            out["dw2"] = columns(d_y, r_hat)
            out["db2"] = columns(d_y)
    if d_r is None and d_y is None:
        return out
    out["dx"] = d
    if h is not None:
        dn = d * s * a
        out["dscale"] = columns(d, a * n)
        da = d * s * n
        if gate is not None and gate.shape[-1] == 1:
            da = da.sum(-1, keepdim=True)
        out["dgate"] = da * slope
        if post:
            out["dw1"] = columns(dn, h_hat)
            out["db1"] = columns(dn)
            out["dh"] = back(dn * w1, h_hat, h_inv, post[0] == "layer")
        else:
            out["dh"] = dn
    return out


def check(got, want, dtype, terms=None, rows=0, growth=1.0):
    """A result of type `dtype` against 64 bits.

    Rounding to the type: half a step.  Before it, 32 bits: the longest chain
    is the statistics of h, those of r, and the two row sums of the backward
    pass; a row sum is at most 16 + 6 + 16 additions deep (a thread's, a
    wave's, the waves'), so each of the four is off by 38 U of its terms'
    size, the elementwise operations between them by some 60 U in all, and a
    later statistic passes an earlier one's error on at most twice: under
    512 U of the largest entry (the inputs here are of order one, and so is
    what cancels).  `growth`: where a row's std is small, its errors are
    stretched by 1 / std.  A column sum (`terms`: what columns() gives)
    adds `rows` additions in the worst order.
    """
    got = got.detach().double().cpu()
    assert got.shape == want.shape
    if not want.numel():
        return
    size = 1.0 + want.abs().max() if terms is None else terms
    tol = growth * (512 + rows) * U * size
    off = (got - want).abs()
    bound = tol + HALF[dtype] * (want.abs() + tol) + \
        (2.0 ** -25 if dtype == torch.float16 else 0.0)
    assert (off <= bound).all(), float((off / bound).max())
