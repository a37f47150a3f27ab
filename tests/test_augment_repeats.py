"""The GPU augmentation gives equal crops for equal random numbers."""

import pytest
import torch

from moco_amd.ops import two_crop_augment

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("size,out", [(40, 32), (256, 224), (61, 57)])
@pytest.mark.parametrize("plus", [False, True])
@pytest.mark.parametrize("uint8", [False, True])
def test_equal_calls_give_equal_crops(size, out, plus, uint8):
    raw = torch.rand(16, 3, size, size, device="cuda")
    if uint8:
        raw = (raw * 255).to(torch.uint8)

    def run():
        return two_crop_augment(raw, out_size=out, aug_plus=plus,
                                generator=torch.Generator().manual_seed(3))
    want = run()
    for _ in range(20):
        assert all(torch.equal(a, b) for a, b in zip(want, run()))
