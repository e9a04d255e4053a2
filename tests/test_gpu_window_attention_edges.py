"""Windowed attention on the GPU where single rows go wrong: maxima that keep growing, rows and columns that
hold what is not finite, rows that a bias masks throughout, extreme arguments."""

import pytest
import torch

from .attention_ref import check, reference
from .test_gpu_window_attention import DT, call, make, verify

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 72, 96, 128])
@pytest.mark.parametrize("window,sinks", [((-1, -1), 0), ((-1, 0), 0), ((150, 40), 9)])
def test_maxima_that_grow_all_along(dt, dim, window, sinks):
    """Logits rise by 16 with every 32 keys, so that a row's reference of the exponents moves in each half of
    every tile: what was written before (P of the other half, the output) is rescaled again and again."""
    c = make(40, [300, 77], 2, 1, dim, DT[dt])
    c["q"][..., 0] = dim ** 0.5
    c["k"][..., 0] = torch.cat([torch.arange(300), torch.arange(77)]).cuda()[:, None] * 0.5
    verify(c, window, sinks)


def test_bucket_sums_beside_keys_of_minus_infinity():
    """Keys with a component of -inf where every query is positive have logits of -inf: weight 0. dQ of the rows
    that see one is 0 times infinity, so the gradients' second pass runs; the bucket sums are those of the
    other keys, the same bits each time."""
    c = make(41, [700, 130], 2, 1, 64, torch.bfloat16, buckets=16)
    c["q"][..., 0] = 1.0
    at = torch.tensor([35, 45, 60, 63, 100, 127, 400, 700 + 50, 700 + 120])
    c["k"][at.cuda(), :, 0] = -float("inf")
    first = None
    for _ in range(5):
        got = call(c, (90, 70), 3)
        want = reference(c["q"], c["k"], c["v"], c["ptr_q"].tolist(), c["ptr_k"].tolist(), 90, 70, 3, 0.125, c["bias"],
                         c["pos_q"], c["pos_k"], 0.4, 4, c["dout"], True) if first is None else want
        for n in ("out", "dk", "dv", "dbias"):
            check(got[n], want[n], n)
        first = got if first is None else first
        assert torch.equal(got["dbias"], first["dbias"])
