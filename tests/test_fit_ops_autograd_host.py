"""The fit operators' torch ops without a GPU: which outputs carry a gradient
and how their backward passes trace, on fake tensors."""

from __future__ import annotations

import importlib

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

torch_ops = importlib.import_module("hexo-shrimp-bot_b200.torch_ops")
torch_ops.define_fit()
fit = torch.ops.mantis_b200


def _cuda(*shape, dtype=torch.bfloat16, grad=False):
    return torch.empty(*shape, dtype=dtype, device="cuda", requires_grad=grad)


def _attention(dtype):
    q = _cuda(2, 4, 9, 32, dtype=dtype, grad=True)
    k, v = (_cuda(2, 2, 9, 32, dtype=dtype, grad=True) for _ in range(2))
    bias = _cuda(5, 4, dtype=torch.float32, grad=True)
    where = _cuda(3, 3, dtype=torch.int32), _cuda(9, 2, dtype=torch.int32), _cuda(2, dtype=torch.int32)
    return q, k, v, bias, *where


def _segments(dtype):
    return _cuda(40, dtype=dtype, grad=True), _cuda(5, dtype=torch.long), _cuda(4, dtype=torch.long), 3


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_outputs_that_carry_a_gradient(dtype):
    """The log-sum-exps and the unrounded output have no gradient formula, so
    they must not ask for one."""
    with FakeTensorMode():
        assert [x.requires_grad for x in fit.bucket_attention(*_attention(dtype))] == [True, False, False]
        assert [x.requires_grad for x in fit.log_probs(*_segments(dtype))] == [True, True, False, False, True]
        assert fit.dropout_add(_cuda(3, 8, grad=True), _cuda(3, 8, grad=True), 0.1, 1, 2).requires_grad


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bias_grad", [True, False])
def test_backward_ops_have_fakes(dtype, bias_grad):
    """Each backward pass is an op with a fake of its own: what tracing needs."""
    with FakeTensorMode():
        args = _attention(dtype)
        dq, dk, dv, dbias = fit.bucket_attention_backward(*args, *fit.bucket_attention(*args), args[0], None, bias_grad)
        for x, y in zip((dq, dk, dv), args):
            assert x.shape == y.shape and x.dtype == dtype
        assert dbias.dtype == torch.float32 and dbias.shape == (args[3].shape if bias_grad else (0,))
        logits, offsets, ranks, top = _segments(dtype)
        logp, entropy, lse, tops, top_logp = fit.log_probs(logits, offsets, ranks, top)
        dx = fit.log_probs_backward(logits, offsets, ranks, lse, entropy, tops, logp, None, top_logp)
        assert dx.shape == logits.shape and dx.dtype == dtype
        dy = fit.dropout_backward(_cuda(3, 8, dtype=torch.float32), 0.1, 1, 2, dtype)
        assert dy.shape == (3, 8) and dy.dtype == dtype
