"""float32 x beside bfloat16 streams, and the other way round, in calls with many rows (rows through shared memory), at widths that are and are not multiples of eight."""
import pytest
import torch

from test_norms_gpu import BF, F, check_gated, check_residual, leave_no_memory      # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,cols", [(70001, 128), (33001, 257), (8400, 1001), (8193, 1024), (2101, 4096), (1639, 5120), (1026, 8191), (1025, 8192)])
@pytest.mark.parametrize("types", [(F, BF, BF), (BF, F, F)])
@pytest.mark.parametrize("post", [False, True])
def test_residual(rows, cols, types, post):
    check_residual(rows, cols, types, post, None if rows % 2 else 0.7, seed=rows)


@pytest.mark.parametrize("rows,cols", [(70001, 128), (110000, 77), (33001, 257), (2101, 4096)])
@pytest.mark.parametrize("types", [(F, BF, BF), (BF, F, F)])
def test_gated(rows, cols, types):
    check_gated(rows, cols, types, "silu" if rows % 2 else "sigmoid", seed=cols)
