"""norm_residual on CPU: values and gradients of the plain path against the
formulas and against differences, and what is refused."""

import pytest
import torch
import torch.nn as nn

from moco_amd.ops import norm_residual
from norm_oracle import check, formula


def norms(kind, width, affine=True, dtype=torch.float32, seed=0):
    torch.manual_seed(seed)
    if kind is None:
        return None
    if kind == "rms":
        m = nn.RMSNorm(width, eps=1e-5, elementwise_affine=affine)
    else:
        m = nn.LayerNorm(width, eps=1e-5, elementwise_affine=affine)
    with torch.no_grad():
        for p in m.parameters():
            p.add_(torch.randn_like(p) * 0.2)
    return m.to(dtype)


def spec(mod):
    if mod is None:
        return None
    kind = "layer" if isinstance(mod, nn.LayerNorm) else "rms"
    w, b = (None if t is None else t.detach().double().cpu() for t in
            (mod.weight, getattr(mod, "bias", None)))
    return kind, mod.eps, w, b


def run_case(rows, width, x_type, h_type, post, pre, gate, act, scale,
             device="cpu", outs="ry", affine=True, w_type=torch.float32,
             layout=None):
    """One call with gradients, checked against the formulas."""
    gen = torch.Generator().manual_seed(rows * 31 + width)

    def rand(*shape, dtype):
        return torch.randn(*shape, generator=gen).to(dtype).to(device)

    x, h = rand(rows, width, dtype=x_type), rand(rows, width, dtype=h_type)
    g = None if gate is None else rand(
        rows, width if gate == "full" else 1, dtype=h_type)
    if layout is not None:
        x, h, g = layout(x, h, g)
    s = None if scale is None else (
        rand(width, dtype=w_type) * 0.3 if scale == "vector" else scale)
    post_m, pre_m = (norms(k, width, affine, w_type, i).to(device)
                     if k else None for i, k in enumerate((post, pre)))
    leaves = [t for t in (x, h, g, s) if isinstance(t, torch.Tensor)]
    leaves = [t.requires_grad_() for t in leaves]
    r, y = norm_residual(x, h, post=post_m, pre=pre_m, gate=g, gate_act=act,
                         scale=s)
    assert r.dtype == x_type and r.shape == x.shape
    d_r = rand(rows, width, dtype=x_type) if "r" in outs else None
    d_y = rand(rows, width, dtype=h_type) if "y" in outs and pre else None
    torch.autograd.backward([t for t, d in ((r, d_r), (y, d_y))
                             if d is not None],
                            [d for d in (d_r, d_y) if d is not None])

    def wide(t):
        return None if t is None else t.detach().double().cpu()

    s64 = wide(s) if isinstance(s, torch.Tensor) else (
        None if s is None else torch.tensor(s, dtype=torch.float64))
    want = formula(wide(x), wide(h), wide(g), act, s64, spec(post_m),
                   spec(pre_m), wide(d_r), wide(d_y))
    check(r, want["r"], x_type)
    if pre:
        assert y.dtype == h_type
        check(y, want["y"], h_type)
    else:
        assert y is None
    got = {"dx": x, "dh": h, "dgate": g,
           "dscale": s if isinstance(s, torch.Tensor) else None,
           "dw1": post_m and post_m.weight,
           "db1": getattr(post_m, "bias", None),
           "dw2": pre_m and pre_m.weight, "db2": getattr(pre_m, "bias", None)}
    for name, t in got.items():
        if t is None:
            continue
        if name not in want:   # no gradient reaches it
            assert t.grad is None or not t.grad.any()
            continue
        w, terms = want[name] if isinstance(want[name], tuple) else (
            want[name], None)
        check(t.grad, w, t.dtype, terms, rows)


TYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
         (torch.float16, torch.float16), (torch.float32, torch.bfloat16)]
FORMS = [("rms", "rms", "full", "silu", "vector"),
         ("layer", "layer", "row", "sigmoid", "vector"),
         ("layer", "rms", "full", None, 0.5),
         (None, "rms", None, None, None), ("rms", None, "row", "silu", None),
         (None, "layer", "full", "sigmoid", "vector")]


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("rows,width", [(1, 64), (5, 33), (40, 7), (3, 1)])
def test_against_the_formulas(types, form, rows, width):
    if width == 1 and form[2] == "row":
        form = form[:2] + ("full",) + form[3:]
    run_case(rows, width, *types, *form)


@pytest.mark.parametrize("form", FORMS)
def test_gradients_against_differences(form):
    post, pre, gate, act, scale = form
    torch.manual_seed(3)
    x, h = (torch.randn(2, 3, 6, dtype=torch.float64) for _ in range(2))
    g = None if gate is None else torch.randn(
        2, 3, 6 if gate == "full" else 1, dtype=torch.float64)
    s = torch.randn(6, dtype=torch.float64) if scale == "vector" else scale
    mods = [norms(k, 6, dtype=torch.float64, seed=i)
            for i, k in enumerate((post, pre))]
    leaves = [t.requires_grad_() for t in (x, h, g, s)
              if isinstance(t, torch.Tensor)]
    leaves += [p for m in mods if m is not None for p in m.parameters()]

    def f(*_):
        out = norm_residual(x, h, post=mods[0], pre=mods[1], gate=g,
                            gate_act=act, scale=s)
        return tuple(t for t in out if t is not None)
    assert torch.autograd.gradcheck(f, leaves)


def test_against_torch_modules():
    """The same as nn.RMSNorm and nn.LayerNorm around a sum."""
    x, h = torch.randn(2, 5, 48), torch.randn(2, 5, 48)
    a, b = norms("rms", 48), norms("layer", 48, seed=1)
    r, y = norm_residual(x, h, post=a, pre=b, scale=0.5)
    assert torch.allclose(r, x + 0.5 * a(h), atol=1e-6)
    assert torch.allclose(y, b(x + 0.5 * a(h)), atol=1e-5)


def test_first_block_has_no_branch():
    x = torch.randn(4, 32, requires_grad=True)
    m = norms("rms", 32)
    r, y = norm_residual(x, pre=m)
    assert r is x and torch.allclose(y, m(x), atol=1e-6)
    r, y = norm_residual(x, pre=m, out_dtype=torch.bfloat16)
    assert y.dtype == torch.bfloat16
    y.float().sum().backward()
    assert x.grad is not None and m.weight.grad is not None


def test_one_element_scale_and_no_affine():
    x, h = torch.randn(4, 32), torch.randn(4, 32)
    s = torch.tensor([0.25], requires_grad=True)
    m = norms("rms", 32, affine=False)
    r, y = norm_residual(x, h, post=m, scale=s)
    assert y is None and torch.allclose(r, x + 0.25 * m(h), atol=1e-6)
    r.sum().backward()
    assert torch.allclose(s.grad, m(h).sum().view(1), atol=1e-4)
    for shape in ((4, 32), (4, 1)):
        r = norm_residual(torch.zeros(shape), torch.ones(shape),
                          scale=torch.tensor(0.5))[0]
        assert torch.equal(r, torch.full(shape, 0.5))


def test_no_rows():
    x = torch.zeros(0, 16, requires_grad=True)
    m = norms("layer", 16)
    r, y = norm_residual(x, torch.zeros(0, 16), post=m, pre=m)
    (r.sum() + y.sum()).backward()
    assert r.shape == y.shape == (0, 16) and not m.weight.grad.any()


@pytest.mark.parametrize("exc,kw", [
    (ValueError, dict(branch=torch.zeros(4, 9))),
    (ValueError, dict(branch=torch.zeros(4, 8)[None])),
    (ValueError, dict(pre=nn.RMSNorm(9, eps=1e-5))),
    (ValueError, dict(pre=nn.RMSNorm((4, 8), eps=1e-5))),
    (ValueError, dict(pre=nn.RMSNorm(8))),
    (TypeError, dict(pre=nn.BatchNorm1d(8))),
    (TypeError, dict(post=nn.RMSNorm(8, eps=1e-5).double())),
    (ValueError, dict(gate=torch.zeros(4, 2))),
    (ValueError, dict(gate=torch.zeros(8))),
    (ValueError, dict(gate_act="silu")),
    (ValueError, dict(gate=torch.zeros(4, 8), gate_act="tanh")),
    (TypeError, dict(gate=torch.zeros(4, 8).bfloat16())),
    (ValueError, dict(scale=torch.zeros(4))),
    (ValueError, dict(scale=torch.zeros(4, 8))),
    (TypeError, dict(scale=torch.zeros(8).half())),
    (TypeError, dict(x=torch.zeros(4, 8).bfloat16())),
    (TypeError, dict(x=torch.zeros(4, 8, dtype=torch.int32),
                     branch=torch.zeros(4, 8, dtype=torch.int32))),
    (ValueError, dict(branch=None)),
    (ValueError, dict(branch=None, pre=nn.RMSNorm(8, eps=1e-5), scale=0.5)),
    (ValueError, dict(branch=None, pre=nn.RMSNorm(8, eps=1e-5),
                      gate=torch.zeros(4, 8))),
    (ValueError, dict(out_dtype=torch.bfloat16)),
    (ValueError, dict(branch=torch.zeros(4, 8, device="meta"))),
    (ValueError, dict(x=torch.zeros(4, 0), branch=torch.zeros(4, 0))),
    (ValueError, dict(x=torch.tensor(1.0), branch=torch.tensor(1.0))),
])
def test_refusals(exc, kw):
    kw = {"x": torch.zeros(4, 8), "branch": torch.zeros(4, 8), **kw}
    with pytest.raises(exc):
        norm_residual(kw.pop("x"), kw.pop("branch"), **kw)
