"""The training-step operators in one program: a small residual encoder whose
blocks are joined by norm_residual, its loss, and AdamW steps with a clip."""

import copy

import numpy as np
import pytest
import torch
import torch.nn as nn

from adamw_oracle import check_codes, decode, mem, step64
from moco_amd.ops import FusedAdamW, norm_residual, softmax_ce_label0


class Encoder(nn.Module):
    """Two gated residual blocks between norms."""

    def __init__(self, width=48):
        super().__init__()
        self.first = nn.RMSNorm(width, eps=1e-6)
        self.blocks = nn.ModuleList(
            nn.Linear(width, 2 * width) for _ in range(2))
        self.post = nn.ModuleList(
            nn.RMSNorm(width, eps=1e-6) for _ in range(2))
        self.pre = nn.ModuleList(
            (nn.RMSNorm(width, eps=1e-6), nn.LayerNorm(width, eps=1e-6)))
        self.scale = nn.ParameterList(
            nn.Parameter(torch.full((width,), 0.5)) for _ in range(2))
        self.out = nn.Linear(width, 9)

    def forward(self, x):
        x, y = norm_residual(x, pre=self.first)
        for lin, post, pre, s in zip(self.blocks, self.post, self.pre,
                                     self.scale):
            branch, gate = lin(y).chunk(2, -1)   # strided halves
            x, y = norm_residual(x, branch, post=post, pre=pre, gate=gate,
                                 gate_act="silu", scale=s)
        return self.out(y)


def loss_of(model, x):
    return softmax_ce_label0(model(x).flatten(0, -2))


@pytest.mark.parametrize("device", [
    "cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("bits", [8, 32])
def test_gradients_and_steps(device, bits):
    torch.manual_seed(0)
    ref = Encoder().double()          # plain path in 64 bits on the CPU
    model = copy.deepcopy(ref).float().to(device)
    opt = FusedAdamW(model.parameters(), lr=1e-2, weight_decay=0.1,
                     state_bits=bits, max_grad_norm=0.05, seed=7)
    x = torch.randn(6, 5, 48)
    for step in range(1, 4):
        for p, q in zip(ref.parameters(), model.parameters()):
            p.data.copy_(q.data)
        ref.zero_grad()
        opt.zero_grad()
        loss = loss_of(model, x.to(device))
        loss.backward()
        # cross entropy of 64-bit logits (the op itself is 32-bit)
        want = nn.functional.cross_entropy(
            ref(x.double()).flatten(0, -2), torch.zeros(30, dtype=torch.long))
        want.backward()
        # the longest chain of 32-bit operations is some 2000 deep, and what
        # it sums is of order one: 2000 U = 1.2e-4 of a gradient's size
        assert abs(float(loss.detach()) - float(want.detach())) < 1e-4
        for p, q in zip(ref.parameters(), model.parameters()):
            off = (q.grad.double().cpu() - p.grad).abs().max()
            assert off <= 1.2e-4 * (1 + p.grad.abs().max())
        params = list(model.parameters())
        before = [mem(p) for p in params]
        state = [opt.state[p] for p in params]
        if step == 1:
            mv = [(np.zeros(p.numel()), np.zeros(p.numel())) for p in params]
        elif bits == 32:
            mv = [(mem(s["exp_avg"]), mem(s["exp_avg_sq"])) for s in state]
        else:
            mv = [decode(s["exp_avg"], s["exp_avg_sq"], s["scales"])
                  for s in state]
            mv = [(m, r * r) for m, r in mv]
        gs = [mem(p.grad) for p in params]
        norm = np.sqrt(sum((g ** 2).sum() for g in gs))
        opt.step()
        assert abs(float(opt.last_grad_norm) - norm) <= 2 * 2.0 ** -24 * norm
        coef = min(1.0, 0.05 / (norm + 1e-6))
        assert coef < 1
        for i, p in enumerate(params):
            p2, m2, v2, dp, dm, dv = step64(before[i], gs[i], *mv[i], step,
                                            1e-2, (0.9, 0.999), 1e-8, 0.1,
                                            coef)
            assert (abs(mem(p) - p2) <= dp).all()
            s = opt.state[p]
            if bits == 32:
                assert (abs(mem(s["exp_avg"]) - m2) <= dm).all()
                assert (abs(mem(s["exp_avg_sq"]) - v2) <= dv).all()
            else:
                check_codes(m2, np.sqrt(v2), dm, s["exp_avg"],
                            s["exp_avg_sq"], s["scales"], i, step, 7)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_bf16_blocks_under_an_fp32_stream(dtype):
    """Autocast: 16-bit branches and gates, fp32 stream, weights and
    gradients.  16-bit branches are off by half a step and so is what follows
    from them: 8 roundings deep at most, of entries of order one."""
    torch.manual_seed(0)
    ref = Encoder().double()
    model = copy.deepcopy(ref).float().cuda()
    x = torch.randn(6, 5, 48)
    with torch.autocast("cuda", dtype=dtype):
        stream, y = norm_residual(x.cuda(), pre=model.first, out_dtype=dtype)
        for lin, post, pre, s in zip(model.blocks, model.post, model.pre,
                                     model.scale):
            branch, gate = lin(y).chunk(2, -1)
            stream, y = norm_residual(stream, branch, post=post, pre=pre,
                                      gate=gate, gate_act="silu", scale=s)
            assert stream.dtype == torch.float32 and y.dtype == dtype
    y.float().square().mean().backward()
    out, want = norm_residual(x.double(), pre=ref.first)
    for lin, post, pre, s in zip(ref.blocks, ref.post, ref.pre, ref.scale):
        branch, gate = lin(want).chunk(2, -1)
        out, want = norm_residual(out, branch, post=post, pre=pre, gate=gate,
                                  gate_act="silu", scale=s)
    want.square().mean().backward()
    tol = 8 * torch.finfo(dtype).eps / 2
    assert ((y.double().cpu() - want).abs()
            <= tol * (1 + want.abs().max())).all()
    for p, q in zip(ref.parameters(), model.parameters()):
        if p.grad is None:
            continue
        off = (q.grad.double().cpu() - p.grad).abs().max()
        assert off <= tol * (1 + p.grad.abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("graph", [False, True])
def test_moco_stepper_with_adamw(bits, graph):
    """The pretraining step, eager and as a replayed graph, with AdamW run
    after each replay: every step reaches every weight."""
    from moco_amd import MoCo
    from moco_amd.engine import MoCoStepper
    from moco_amd.models.resnet import build_model
    torch.manual_seed(1)
    model = MoCo(lambda num_classes: build_model("resnet18",
                                                 num_classes=num_classes),
                 dim=128, K=64, m=0.99, T=0.2, mlp=True)
    model = model.cuda().to(memory_format=torch.channels_last)
    opt = FusedAdamW(model.parameters(), lr=1e-3, state_bits=bits,
                     max_grad_norm=1.0)
    st = MoCoStepper(model, opt, torch.device("cuda"), out_size=32,
                     use_graph=graph)
    pool = [torch.rand(4, 3, 40, 40, device="cuda") for _ in range(2)]
    for i in range(6):
        was = [p.detach().clone() for p in model.encoder_q.parameters()]
        loss, _, _ = st.step_from_raw(pool[i % 2])
        assert torch.isfinite(loss)
        assert torch.isfinite(opt.last_grad_norm) and opt.last_grad_norm > 0
        assert all(not torch.equal(a, b) for a, b in
                   zip(was, model.encoder_q.parameters()) if b.dim() > 1)
    assert st.use_graph == graph
    assert all(opt.state[p]["step"] == 6
               for p in model.encoder_q.parameters())
