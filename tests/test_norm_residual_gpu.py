"""norm_residual on the GPU: values and gradients against the formulas in 64
bits."""

import pytest
import torch
import torch.nn as nn

from test_norm_residual_cpu import FORMS, TYPES, norms, run_case

pytestmark = pytest.mark.gpu

# one row to several per workgroup; widths around a vector of 8, and of each
# number of threads and registers per row
SIZES = [(1, 1), (1, 2048), (5, 7), (70, 8), (3, 9), (3, 64), (130, 65),
         (77, 128), (50, 129), (40, 256), (9, 257), (9, 512), (6, 513),
         (600, 200), (7, 1000), (5, 1024), (4, 1025), (3, 2048), (520, 1030),
         (3, 2056), (2, 4095), (5, 4096), (2, 4100), (2, 8192), (2, 8195),
         (3, 16383), (2, 16384)]


@pytest.mark.parametrize("types", TYPES + [(torch.float32, torch.float16)])
@pytest.mark.parametrize("form", FORMS)
def test_against_the_formulas_gpu(types, form):
    for rows, width in SIZES:
        f = form
        if width == 1 and f[2] == "row":
            f = f[:2] + ("full",) + f[3:]
        run_case(rows, width, *types, *f, device="cuda")


@pytest.mark.parametrize("outs", ["r", "y"])
@pytest.mark.parametrize("form", FORMS)
def test_one_output_used(outs, form):
    if outs == "y" or form[1] is not None:
        run_case(21, 264, torch.float32, torch.bfloat16, *form,
                 device="cuda", outs=outs)


@pytest.mark.parametrize("form", FORMS[:3])
def test_weights_of_the_blocks_type_and_none(form):
    run_case(33, 72, torch.bfloat16, torch.bfloat16, *form, device="cuda",
             w_type=torch.bfloat16)
    run_case(33, 72, torch.bfloat16, torch.bfloat16, *form, device="cuda",
             affine=False)


def test_strided_inputs():
    """Branch and gate as halves of one projection, a stream inside a wider
    buffer, rows in steps, columns in steps, and transposed."""
    def halves(x, h, g):
        hg = torch.cat([h, g], 1)
        w = h.shape[1]
        wide = torch.cat([x, x, x], 1)
        return wide[:, w:2 * w], hg[:, :w], hg[:, w:]

    def steps(x, h, g):
        def gap(t, dim):
            out = torch.zeros([2 * n if d == dim else n for d, n in
                               enumerate(t.shape)], dtype=t.dtype,
                              device=t.device)
            sl = [slice(None)] * t.dim()
            sl[dim] = slice(None, None, 2)
            out[tuple(sl)] = t
            return out[tuple(sl)]
        return gap(x, 0), gap(h, 1), gap(g, 0)

    def turned(x, h, g):
        return (x.t().contiguous().t(), h,
                g[:, :1].expand_as(g) if g.shape[1] > 1 else g)
    for layout in (halves, steps, turned):
        for width in (64, 65, 2048):
            run_case(37, width, torch.float32, torch.bfloat16, "rms", "layer",
                     "full", "silu", "vector", device="cuda", layout=layout)


def test_more_dimensions():
    """[batch, time, width], batches that lie apart, one gate per token."""
    post, pre = (norms(k, 40, seed=i).cuda() for i, k in
                 enumerate(("rms", "layer")))
    base = torch.randn(4, 9, 40, device="cuda")
    for x in (base, base[:, 2:7], base.transpose(0, 1), base[1], base[1, 2],
              base[:, :1].expand(4, 6, 40)):
        h = torch.randn(x.shape, device="cuda")
        g = torch.randn(*x.shape[:-1], 1, device="cuda")
        r, y = norm_residual_of(x, h, post, pre, g)
        want, want_y = norm_residual_of(x.cpu(), h.cpu(), copy_of(post),
                                        copy_of(pre), g.cpu())
        assert r.shape == x.shape
        assert torch.allclose(r.cpu(), want, atol=1e-5)
        assert torch.allclose(y.cpu(), want_y, atol=1e-5)


def copy_of(m):
    import copy
    return copy.deepcopy(m).cpu()


def norm_residual_of(x, h, post, pre, g):
    from moco_amd.ops import norm_residual
    return norm_residual(x, h, post=post, pre=pre, gate=g,
                         gate_act="sigmoid", scale=0.7)


def test_first_block_and_inference():
    from moco_amd.ops import norm_residual
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.randn(17, 96, device="cuda", requires_grad=True)
        m = norms("layer", 96).cuda()
        r, y = norm_residual(x, pre=m, out_dtype=dtype)
        assert r is x and y.dtype == dtype
        d = torch.randn(17, 96, device="cuda").to(dtype)
        y.backward(d)
        x2 = x.detach().double().cpu().requires_grad_()
        m2 = copy_of(m).double()
        m2.zero_grad()
        m2(x2).backward(d.double().cpu())
        tol = 1e-5 if dtype == torch.float32 else 2.0 ** -7
        assert torch.allclose(x.grad.double().cpu(), x2.grad, atol=tol)
        assert torch.allclose(m.weight.grad.double().cpu(), m2.weight.grad,
                              atol=1e-4)
        with torch.no_grad():
            again = norm_residual(x, pre=m, out_dtype=dtype)[1]
        assert torch.equal(again, y)


def test_constant_rows_and_nonfinite_rows():
    """A row without spread divides by sqrt(eps); a NaN or an infinity stays
    in its row."""
    from moco_amd.ops import norm_residual
    for kind in ("rms", "layer"):
        m, p = (norms(kind, 136, seed=i).cuda() for i in range(2))
        x = torch.randn(6, 136, device="cuda", requires_grad=True)
        h = torch.randn(6, 136, device="cuda")
        clean = norm_residual(x, h, post=m, pre=p)
        h2 = h.clone()
        h2[1] = 0.0
        h2[2, 5] = float("nan")
        h2[4, 7] = float("inf")
        h2.requires_grad_()
        r, y = norm_residual(x, h2, post=m, pre=p)
        for a, b in zip((r, y), clean):
            for row in (0, 3, 5):
                assert torch.equal(a[row], b[row])
            assert torch.isfinite(a[1]).all()
            assert torch.isnan(a[2]).any() and torch.isnan(a[4]).any()
        gx, gh = torch.autograd.grad(r.sum() + y.sum(), (x, h2))
        for t in (gx, gh):
            assert torch.isfinite(t[[0, 1, 3, 5]]).all()
        bias = m.bias if kind == "layer" else 0.0
        assert torch.allclose(r[1], x[1] + bias, atol=1e-6)


def test_no_rows_gpu():
    from moco_amd.ops import norm_residual
    x = torch.zeros(0, 16, device="cuda", requires_grad=True)
    m = norms("layer", 16).cuda()
    r, y = norm_residual(x, torch.zeros(0, 16, device="cuda"), post=m, pre=m)
    (r.sum() + y.sum()).backward()
    assert r.shape == y.shape == (0, 16) and not m.weight.grad.any()
    assert not m.bias.grad.any() and x.grad.shape == (0, 16)


def test_one_module_for_both_norms_and_one_element_scale():
    from moco_amd.ops import norm_residual
    m = norms("rms", 256).cuda()
    s = torch.tensor([0.25], device="cuda", requires_grad=True)
    x, h = (torch.randn(50, 256, device="cuda") for _ in range(2))
    r, y = norm_residual(x, h, post=m, pre=m, scale=s)
    (r.sum() + (y * x).sum()).backward()
    m2, s2 = copy_of(m).double(), s.detach().cpu().double().requires_grad_()
    m2.zero_grad()
    x2, h2 = x.cpu().double(), h.cpu().double()
    r2 = x2 + s2 * m2(h2)
    (r2.sum() + (m2(r2) * x2).sum()).backward()
    # sums over 12800 entries of order one: 1e-5 of their sizes
    assert torch.allclose(m.weight.grad.double().cpu(), m2.weight.grad,
                          atol=1e-3)
    assert torch.allclose(s.grad.double().cpu(), s2.grad, atol=0.1)


def test_one_element_scale_of_any_shape():
    from moco_amd.ops import norm_residual
    for shape in ((4, 32), (4, 1)):
        for s in (torch.tensor(0.5), torch.tensor([0.5]),
                  torch.tensor([[0.5]])):
            s = s.cuda().requires_grad_()
            r = norm_residual(torch.zeros(shape, device="cuda"),
                              torch.ones(shape, device="cuda"), scale=s)[0]
            assert torch.equal(r, torch.full_like(r, 0.5))
            r.sum().backward()
            assert s.grad.shape == s.shape
            assert float(s.grad) == r.numel()


def run_graph(x, h, post, pre, leaves, d):
    from moco_amd.ops import norm_residual
    r, y = norm_residual(x, h, post=post, pre=pre, scale=0.5)
    grads = torch.autograd.grad((r, y), leaves, d)
    # without their graph, whose nodes would stay on this call's stream
    return (r.detach(), y.detach(), *grads)


def test_streams_graphs_and_repeatability():
    """The same bits on another stream, and in each replay of a captured
    forward and backward pass, with eager work between the replays."""
    post, pre = (norms(k, 1024, seed=i).cuda() for i, k in
                 enumerate(("rms", "layer")))
    x, h = (torch.randn(700, 1024, device="cuda").requires_grad_()
            for _ in range(2))
    d = tuple(torch.randn(700, 1024, device="cuda") for _ in range(2))
    leaves = [x, h, *post.parameters(), *pre.parameters()]
    want = [t.detach().clone() for t in
            run_graph(x, h, post, pre, leaves, d)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run_graph(x, h, post, pre, leaves, d)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del got
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run_graph(x, h, post, pre, leaves, d)
    for k in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(700, 1024, device="cuda"))
        g.replay()
        torch.cuda.synchronize()
        kept = [t.detach().clone() for t in out]
        want = run_graph(x, h, post, pre, leaves, d)
        assert all(torch.equal(a, b) for a, b in zip(kept, want))
        del want


def test_refusals_gpu():
    from moco_amd.ops import norm_residual
    x = torch.zeros(2, 8, device="cuda")
    with pytest.raises(ValueError):
        norm_residual(torch.zeros(2, 16385, device="cuda"),
                      torch.zeros(2, 16385, device="cuda"))
    with pytest.raises(ValueError):
        norm_residual(x, x.cpu())
    with pytest.raises(ValueError):
        norm_residual(x, x, post=nn.RMSNorm(8, eps=1e-6))
    with pytest.raises(TypeError):
        norm_residual(x.double(), x.double())
    with pytest.raises(TypeError):
        norm_residual(x, x, gate=x.bfloat16())
    y = norm_residual(x.requires_grad_(), x)[0]
    (g,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_graph_of_a_call():
    """What autograd promises for any node: two passes over a kept graph, an
    error for a freed one and for an input changed in between, nothing for a
    frozen input, the same under checkpointing and with half its outputs."""
    from torch.utils.checkpoint import checkpoint

    from moco_amd.ops import norm_residual
    post, pre = (norms(k, 96, seed=i).cuda() for i, k in
                 enumerate(("rms", "layer")))
    gen = torch.Generator("cuda").manual_seed(5)
    x, h, gate, d = (torch.randn(33, 96, device="cuda", generator=gen)
                     for _ in range(4))
    x.requires_grad_()
    gate.requires_grad_()
    leaves = [x, gate, *post.parameters(), *pre.parameters()]

    def call(a, b, g):
        return norm_residual(a, b, post=post, pre=pre, gate=g)

    outs = call(x, h, gate)
    assert all(o.requires_grad and o.grad_fn is not None for o in outs)
    want = torch.autograd.grad(outs, leaves, (d, d), retain_graph=True)
    again = torch.autograd.grad(outs, leaves, (d, d))
    assert all(torch.equal(a, b) for a, b in zip(again, want))
    with pytest.raises(RuntimeError):
        torch.autograd.grad(outs, leaves, (d, d))
    got = torch.autograd.grad(checkpoint(call, x, h, gate,
                                         use_reentrant=False), leaves, (d, d))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # one output only, the other's gradient absent or zero
    some = torch.autograd.grad(call(x, h, gate)[1], leaves, d)
    zero = torch.autograd.grad(call(x, h, gate), leaves,
                               (torch.zeros_like(d), d))
    assert all(torch.equal(a, b) for a, b in zip(some, zero))
    # frozen inputs beside one that is not
    y = call(x.detach(), h, gate.detach())[1]
    y.backward(d)
    assert h.grad is None and x.grad is None and gate.grad is None
    assert all(p.grad is not None for p in pre.parameters())
    outs = call(x, h, gate)
    h.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(outs, leaves, (d, d))
    with torch.no_grad():
        assert not any(o.requires_grad for o in call(x, h, gate))


def test_transforms_refused():
    """Forward-mode tangents and function transforms are refused, not
    dropped."""
    import torch.autograd.forward_ad as fwAD

    from moco_amd.ops import norm_residual
    x, h, t = (torch.ones(2, 8, device="cuda") for _ in range(3))
    with fwAD.dual_level():
        for grad in (False, True):
            dual = fwAD.make_dual(h.clone().requires_grad_(grad), t)
            with pytest.raises(NotImplementedError):
                norm_residual(x, dual)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda a: norm_residual(a, h)[0].sum())(x)
