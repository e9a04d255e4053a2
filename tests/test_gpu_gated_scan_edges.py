"""Gated scan on the GPU: many clouds of few rows, tangents."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from gdl_b200.functional import gated_scan

from .test_gpu_gated_scan import DT, call, make

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("reverse", [False, True])
def test_more_clouds_than_a_grid_has_rows(dt, reverse):
    """70000 clouds, most of them empty, of 204 rows in all: as the same rows in the clouds that have any."""
    lens = [2, 0, 1, 1] * 51
    some = make(20, lens, 6, DT[dt])
    many = dict(some, h0=torch.cat([some["h0"], torch.randn(70000 - len(lens), 6)]),
                dlast=torch.cat([some["dlast"], torch.randn(70000 - len(lens), 6)]),
                ptr=torch.cat([some["ptr"], some["ptr"][-1:].expand(70000 - len(lens))]))
    got, want = call(many, reverse), call(some, reverse)
    tol = 2.0 ** -18 + (2.0 ** -7 if dt == "bf16" else 0.0)  # another kernel's order of the same sums
    for n in want:
        a, b = got[n].detach().float(), want[n].detach().float()
        a = a[:len(b)]
        assert float((a - b).abs().max()) <= tol * 4 * float(b.abs().max()), n
    assert torch.equal(got["last"][len(lens):].cpu(), many["h0"][len(lens):])
    assert torch.equal(got["dh0"][len(lens):].cpu(), many["dlast"][len(lens):])


def test_a_tangent_is_refused_without_gradients_too():
    c = make(21, [40], 8, torch.float32)
    x, gate, decay, ptr = (c[m].cuda() for m in ("x", "gate", "decay", "ptr"))
    with torch.no_grad(), fwAD.dual_level():
        with pytest.raises((RuntimeError, NotImplementedError)):
            gated_scan(fwAD.make_dual(x, torch.ones_like(x)), gate, decay, ptr)
