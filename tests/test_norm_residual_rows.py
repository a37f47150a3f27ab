"""norm_residual where a workgroup takes several rows: the loops over rows,
with the next row's inputs on their way, weights kept over rows, and last
turns in which only some of a workgroup's groups have a row."""

import pytest
import torch

import test_norm_residual_cpu as one_row
from norm_oracle import check

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16

# A forward grid has 262144 threads at most, rows have 8 (64 columns) to 1024
# (above 4096): two turns and the beginning of a third, of a size for each
# number of threads a row, odd widths and whole vectors.  Backward grids are
# smaller.
SIZES = [(65541, 5), (65541, 9), (65539, 64), (32771, 100), (16387, 200),
         (16385, 256), (8195, 500), (4097, 1001), (2050, 1500), (2049, 2048),
         (1027, 2100), (1025, 4096), (600, 4100), (515, 8192), (520, 8200),
         (513, 16384)]
CASES = [((BF16, BF16), ("rms", "rms", "full", "silu", "vector")),
         ((F32, BF16), ("layer", "layer", "row", "sigmoid", "vector")),
         ((F32, F32), ("layer", "rms", "full", None, 0.5)),
         ((F16, F16), ("rms", None, "row", "silu", "vector"))]


@pytest.mark.parametrize("types,form", CASES)
@pytest.mark.parametrize("rows,width", SIZES)
def test_several_turns(monkeypatch, rows, width, types, form):
    """A column sum's additions: a group's turns (a backward grid has 256
    workgroups at least, or each has one turn), a workgroup's groups (32 at
    most), and of up to 1024 workgroups 32 at a time, then those."""
    depth = -(-rows // 256) + 32 + 32 + 32

    def deep(got, want, dtype, terms=None, rows=0):
        check(got, want, dtype, terms, depth)

    monkeypatch.setattr(one_row, "check", deep)
    one_row.run_case(rows, width, *types, *form, device="cuda")


@pytest.mark.parametrize("types", [(BF16, BF16), (F32, F16)])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("rows,width", [(32775, 7), (16390, 136), (1030, 2048),
                                        (520, 4096), (260, 8192), (260, 9000)])
def test_a_row_does_not_depend_on_its_turn(types, kind, rows, width):
    """The same rows alone, and in an order that gives them other turns and
    groups: the same bits, both ways."""
    from moco_amd.ops import norm_residual
    torch.manual_seed(0)
    post, pre = (one_row.norms(kind, width, seed=i).cuda() for i in range(2))
    x, d_r = (torch.randn(rows, width, device="cuda").to(types[0])
              for _ in range(2))
    h, g, d_y = (torch.randn(rows, width, device="cuda").to(types[1])
                 for _ in range(3))

    def run(order):
        leaves = [t[order].requires_grad_() for t in (x, h, g)]
        out = norm_residual(*leaves[:2], post=post, pre=pre, gate=leaves[2],
                            gate_act="sigmoid", scale=0.5)
        return (*out, *torch.autograd.grad(out, leaves,
                                           (d_r[order], d_y[order])))

    every = torch.arange(rows, device="cuda")
    whole = run(every)
    for order in (every.flip(0), every.roll(17), every[-40:], every[:1]):
        for a, b in zip(whole, run(order)):
            assert torch.equal(a[order], b)
