"""Tree attention over pools at any address: which kernel runs is no matter of the caller's."""
import pytest
import torch

from test_tree_attention_gpu import BF, DEV, F32, FAR, Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,hd,odd", [(BF, 64, 1), (BF, 128, 4), (BF, 96, 2), (F32, 64, 1), (F32, 64, 2), (BF, 64, 8)])
@pytest.mark.parametrize("shapes,reach", [([(300, 9), (40, 3)], None), ([(700, 50), (40, 33)], FAR)])
@pytest.mark.parametrize("which", ["k", "v"])
def test_pools_that_start_anywhere(dtype, hd, odd, shapes, reach, which):
    b = Batch(dtype, 4, 2, hd, shapes, seed=51)
    flat = torch.zeros(b.dev[which].numel() + 16, dtype=dtype, device=DEV)
    moved = flat[odd:odd + b.dev[which].numel()].view(b.dev[which].shape)
    moved.copy_(b.dev[which])
    b.dev[which] = moved
    b.check(b.run(reach=reach))
