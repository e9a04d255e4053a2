"""Limits of the serialised-cloud operators that show without a GPU: refusals before a launch, workspace sizes,
extreme arguments."""

import pytest

from .test_serialized_host import INVALID, attention, lib  # noqa: F401


@pytest.mark.parametrize("inv_radius2", [-1.0, -1e-30, float("nan"), float("inf"), -float("inf")])
def test_a_bucket_scale_below_zero_or_not_finite_is_refused(lib, inv_radius2):  # noqa: F811
    """The kernels count buckets from t = 1 + d^2 inv_radius2 >= 1: below it a table's address would lie outside."""
    a = attention(bias=4096, buckets=8, pos_q=4096, pos_k=4096, inv_radius2=inv_radius2)
    assert lib.gdl_window_attention(a, 4096, None, None, None) == INVALID
    assert lib.gdl_window_attention_backward(a, 4096, 4096, None, 4096, 4096, 4096, 4096, 4096, 4096, 1 << 40, None) == INVALID
