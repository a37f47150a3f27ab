"""One process: captured training steps are the eager ones."""

import copy

import pytest
import torch

from moco_amd.builder import MoCo

pytestmark = pytest.mark.gpu


class Small(torch.nn.Module):
    """An encoder without convolutions: the library's may add partial sums in
    any order, and two runs of one program then differ."""

    def __init__(self, num_classes):
        super().__init__()
        self.body = torch.nn.Sequential(
            torch.nn.Flatten(), torch.nn.Linear(192, 64),
            torch.nn.BatchNorm1d(64), torch.nn.ReLU())
        self.fc = torch.nn.Linear(64, num_classes)

    def forward(self, x):
        return self.fc(self.body(x))


def test_captured_steps_are_the_eager_ones():
    """Warmup, capture and replays, once round the queue: losses, queue and
    weights bit for bit."""
    from moco_amd.engine import MoCoStepper
    from moco_amd.ops import FusedAdamW, FusedSGD
    for optimizer in (FusedSGD, FusedAdamW):
        torch.manual_seed(0)
        eager = MoCo(Small, dim=128, K=64, m=0.9, T=0.2, mlp=True).cuda()
        graph = copy.deepcopy(eager)
        steppers = [
            MoCoStepper(m, optimizer(m.parameters(), lr=0.05),
                        torch.device("cuda"), use_graph=g)
            for m, g in ((eager, False), (graph, True))]
        for _ in range(8):
            crops = [torch.randn(8, 3, 8, 8, device="cuda") for _ in range(2)]
            a = steppers[0].step(*crops)[0].detach().clone()
            b = steppers[1].step_graphed(*crops)[0].detach().clone()
            torch.cuda.synchronize()
            assert torch.equal(a, b)
            assert torch.equal(eager.queue, graph.queue)
        assert steppers[1].use_graph
        assert int(eager.queue_ptr) == int(graph.queue_ptr) == 0
        for p, q in zip(eager.parameters(), graph.parameters()):
            assert torch.equal(p, q)
