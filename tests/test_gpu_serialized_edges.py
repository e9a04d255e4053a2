"""The serialised-cloud block on the GPU: batches of nothing."""

import pytest
import torch

from gdl_b200.serialized import SerializedBlock, morton_order

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]


@pytest.mark.parametrize("bounds", [[0], [0, 0, 0]])
def test_a_batch_without_rows(bounds):
    ptr, pos, x = torch.tensor(bounds).cuda(), torch.empty(0, 3).cuda(), torch.empty(0, 32).cuda().requires_grad_(True)
    block = SerializedBlock(32, 4, window=8).cuda()
    assert morton_order(pos, ptr).shape == (0,)
    y = block(x, pos, ptr)
    assert y.shape == (0, 32)
    y.sum().backward()
    assert x.grad.shape == (0, 32) and all(float(p.grad.abs().sum()) == 0 for p in block.parameters())
