"""Limits of the serialised-cloud operators that show without a GPU: refusals before a launch, workspace sizes,
extreme arguments."""

import numpy as np
import pytest
import torch

from gdl_b200 import csrc
from gdl_b200.functional import window_attention
from gdl_b200.serialized import morton_order

from .test_serialized_host import INVALID, attention, lib  # noqa: F401


@pytest.mark.parametrize("inv_radius2", [-1.0, -1e-30, float("nan"), float("inf"), -float("inf")])
def test_a_bucket_scale_below_zero_or_not_finite_is_refused(lib, inv_radius2):  # noqa: F811
    """The kernels count buckets from t = 1 + d^2 inv_radius2 >= 1: below it a table's address would lie outside."""
    a = attention(bias=4096, buckets=8, pos_q=4096, pos_k=4096, inv_radius2=inv_radius2)
    assert lib.gdl_window_attention(a, 4096, None, None, None) == INVALID
    assert lib.gdl_window_attention_backward(a, 4096, 4096, None, 4096, 4096, 4096, 4096, 4096, 4096, 1 << 40, None) == INVALID


def test_morton_order_leaves_rows_of_no_cloud_in_their_places():
    """Bounds that do not cover all rows (the operators give such rows 0): an index made of them must stay in range."""
    g = torch.Generator().manual_seed(0)
    pos = torch.rand(100, 3, generator=g)
    for bounds in ([10, 40, 40, 85], [0, 60], [30, 100], [50, 50], [0]):
        order = morton_order(pos, torch.tensor(bounds))
        assert torch.equal(order.sort()[0], torch.arange(100))
        assert torch.equal(order[:bounds[0]], torch.arange(bounds[0]))
        assert torch.equal(order[bounds[-1]:], torch.arange(bounds[-1], 100))
        for s, e in zip(bounds[:-1], bounds[1:]):  # each cloud as if it were alone
            assert torch.equal(order[s:e] - s, morton_order(pos[s:e], torch.tensor([0, e - s])))
    assert morton_order(pos[:0], torch.tensor([0, 0])).shape == (0,)
    assert torch.equal(morton_order(pos, torch.tensor([0, 30, 100], dtype=torch.int32)), morton_order(pos, torch.tensor([0, 30, 100])))


def test_bounds_on_another_gpu_are_copied(monkeypatch):
    """A kernel must not be given another GPU's memory: bounds pass as they are only on the rows' own device."""
    class Bounds:
        is_cuda, dtype, device = True, torch.int64, torch.device("cuda", 1)

        def is_contiguous(self):
            return True

    monkeypatch.setattr(csrc.nat, "to_device", lambda t, dev, dtype: ("copied", dev))
    there = Bounds()
    assert csrc._bounds(there, torch.device("cuda", 0)) == ("copied", torch.device("cuda", 0))
    assert csrc._bounds(there, torch.device("cuda", 1)) is there


def test_few_rows_of_many_clouds_are_given_a_workspace(lib):  # noqa: F811
    """The size asked for is that of the kernels that run: one launch takes few rows of up to 65533 clouds."""
    assert lib.gdl_gated_scan_workspace_size(256, 65533, 8) == 256
    assert lib.gdl_gated_scan_workspace_size(256, 65534, 8) > 65534 * 8 * 4
    assert lib.gdl_gated_scan_workspace_size(0, 70000, 8) > 70000 * 8 * 4


def test_the_workspace_of_many_sinks_is_bounded(lib):  # noqa: F811
    """Partial sums of the sinks: what the kernels that run need, and no more than three times dK and dV in f32."""
    def size(dtype=1, **over):
        a = attention(dtype=dtype, heads=4, kv_heads=4, dim=64, q_row=256, k_row=256, v_row=256, q_head=64, k_head=64, v_head=64, **over)
        return lib.gdl_window_attention_backward_workspace_size(a)

    rows = dict(n_query=131072, n_key=131072, num_clouds=1, left=256, right=256)
    plain = size(**rows)
    grads = 131072 * 4 * 64 * 2 * 4
    assert size(num_sinks=2048, **rows) - plain < 1.1 * grads       # 0.27 GB (chunks of 1024 queries: 0.54)
    assert size(num_sinks=4, **rows) - plain < 0.01 * grads         # chunks of 1024: 129 of 4 rows
    for sinks in (1, 60, 500, 10_000, 131_000, 131_072, 2 ** 31 - 1):
        for clouds in (1, 8, 20_000):
            for dtype in (0, 1):
                over = dict(rows, num_clouds=clouds)
                assert size(dtype, num_sinks=sinks, **over) - size(dtype, **over) <= 3 * grads + 512, (sinks, clouds, dtype)


def test_partial_sums_of_sinks_lie_apart():
    """The kernels' places, restated: cloud b's sinks from min(b * sinks, its first key) on; chunk i of its queries
    (first query // size + i) * sinks rows further; min(clouds * sinks, keys) rows, and (queries // size) * sinks more."""
    rng = np.random.RandomState(0)
    for _ in range(200):
        clouds, sinks, size = rng.randint(1, 30), rng.randint(1, 200), int(rng.choice([1, 7, 128]))
        nk, nq = (np.where(rng.rand(clouds) < 0.2, 0, rng.randint(0, 400, clouds)) for _ in range(2))
        k0, q0 = (np.cumsum(n) - n + rng.randint(0, 9) for n in (nk, nq))
        n_key, n_query = int(k0[-1] + nk[-1] + rng.randint(0, 9)), int(q0[-1] + nq[-1] + rng.randint(0, 9))
        most = min(clouds * sinks, n_key)
        main, chunk = np.zeros(most, int), np.zeros(n_query // size * sinks + most, int)
        for b in range(clouds):
            base, own = min(b * sinks, int(k0[b])), min(sinks, int(nk[b]))
            main[base:base + own] += 1
            assert base + own <= len(main)
            for i in range((int(nq[b]) + size - 1) // size):
                at = (int(q0[b]) // size + i) * sinks + base
                chunk[at:at + own] += 1
                assert at + own <= len(chunk)
        assert main.max(initial=0) <= 1 and chunk.max(initial=0) <= 1


def test_the_status_word_reaches_both_directions(monkeypatch):
    """What a bounded wait that gave up would write to is the caller's tensor, in the forward and in the backward."""
    seen = []

    class Lib:  # in the library's place: notes the status word that it is given
        def gdl_window_attention(self, a, *rest):
            return seen.append(a.status) or 0

        def gdl_window_attention_backward_workspace_size(self, a):
            return 256

        def gdl_window_attention_backward(self, a, *rest):
            return seen.append(a.status) or 0

    monkeypatch.setattr(csrc.nat, "load", lambda: Lib())
    monkeypatch.setattr(csrc.nat, "require_cuda", lambda *t, what: torch.device("cpu"))
    monkeypatch.setattr(csrc.nat, "stream", lambda dev: 0)
    monkeypatch.setattr(csrc, "_bounds", lambda p, dev: p)

    class Word(torch.Tensor):
        is_cuda = True

    word = torch.zeros(1, dtype=torch.int32).as_subclass(Word)
    x, ptr = torch.zeros(4, 2, 8, requires_grad=True), torch.tensor([0, 4])
    for status, want in ((word, word.data_ptr()), (None, None)):
        window_attention(x, x, x, ptr, status=status).sum().backward()
        with torch.no_grad():
            window_attention(x, x, x, ptr, status=status)
        assert seen == [want] * 3
        seen.clear()
    for bad in (torch.zeros(1, dtype=torch.int32), torch.zeros(1).as_subclass(Word), torch.zeros(0, dtype=torch.int32).as_subclass(Word)):
        with pytest.raises(csrc.nat.GdlError):
            window_attention(x, x, x, ptr, status=bad)
