"""The serialised-cloud block on the GPU: batches of nothing; the stream that operators run on."""

import pytest
import torch

from gdl_b200 import _native as nat
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


def test_the_raw_stream_is_the_current_one(monkeypatch):
    """With torch's shorter way to it and, where a torch lacks that, by the public one."""
    dev, side = torch.device("cuda", 0), torch.cuda.Stream()
    for raw in (nat._raw_stream, None):
        monkeypatch.setattr(nat, "_raw_stream", raw)
        for d in (dev, torch.device("cuda")):
            assert nat.stream(d) == torch.cuda.current_stream().cuda_stream
            with torch.cuda.stream(side):
                assert nat.stream(d) == side.cuda_stream
