"""The fit operators on the GPU at their ends: empty and malformed inputs, the
forms and paths that ordinary sizes do not reach, and their torch ops."""

from __future__ import annotations

import pytest
import torch

from golden_io import mb

pytestmark = pytest.mark.gpu
DEV = "cuda"
ops = mb.ops
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def _stale(n, dtype):
    """Leaves NaN in the block that the next allocation of this size gets."""
    x = torch.full((n,), float("nan"), dtype=dtype, device=DEV)
    torch.cuda.synchronize()
    del x


# ------------------------------------------------------------- log probs
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 37, 5000])
def test_log_probs_gradient_without_segments(dtype, n):
    """Every element is outside every segment: its gradient is zero."""
    x = torch.randn(n, device=DEV).to(DT[dtype])
    off = torch.zeros(1, dtype=torch.int64, device=DEV)
    got = ops.log_probs(x, off)
    _stale(n + 8, x.dtype)
    dx = ops.log_probs_backward(x, off, None, got, torch.zeros(0, device=DEV))
    assert dx.shape == x.shape and torch.count_nonzero(dx) == 0
