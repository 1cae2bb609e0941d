"""Attention over token sequences at the edges of what a call may be: sizes, biases and scores that a test of ordinary calls
does not reach."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float32


def _K():
    from visiontransformer_amd import functional as K
    return K


@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("bias", [False, True])
def test_no_query_heads(cuda0, dtype, bias):
    """keys without a query head: their gradients are zeros, whatever the memory held before"""
    K = _K()
    q = torch.ones(2, 40, 0, 64, dtype=dtype, device=cuda0).requires_grad_()
    k, v = (torch.ones(2, 70, 3, 64, dtype=dtype, device=cuda0).requires_grad_() for _ in range(2))
    kw = {}
    if bias:
        kw = dict(bias_table=torch.zeros(4, 0, device=cuda0).requires_grad_(), bias_buckets=torch.zeros(5, dtype=torch.int32, device=cuda0))
    out = K.band_attention(q, k, v, window=(10, 0), sinks=2, **kw)
    assert out.shape == q.shape
    held = [torch.full_like(k, float("nan")) for _ in range(4)]
    del held
    grads = torch.autograd.grad(out.sum(), [q, k, v] + list(kw.values())[:1])
    for t, g in zip((q, k, v), grads):
        assert g.shape == t.shape and not g.any()
