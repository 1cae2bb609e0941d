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


@pytest.mark.parametrize("dtype", [FP, BF])
def test_equal_keys_weigh_the_same_wherever_they_stand(cuda0, dtype):
    """Scores of 2^29 and 2^29 + 64 (exact in fp32, which cannot tell 2^29 + 60 from it): the later tiles' keys all have the
    larger one, and the result is the mean of their values.  v is whole numbers below 8: sums of 186 of them are exact, the mean is
    off by the rounding of the quotient and of the probabilities, 2^-8 (bf16) or 2^-22."""
    K = _K()
    B, L, H, D = 16, 250, 16, 64
    k = torch.zeros(1, L, 1, D)
    k[..., 0] = 2.0 ** 29
    k[:, 64:, :, 1] = 64.0
    v = torch.randint(0, 8, (1, L, 1, D), generator=torch.Generator().manual_seed(2)).float()
    on = lambda t, h: t.to(dtype).to(cuda0).expand(B, L, h, D).contiguous()
    want = v[0, 64:, 0].double().mean(0)
    for n in (L, 3):
        out = K.band_attention(on(torch.ones(1, L, 1, D), H)[:, L - n:], on(k, H), on(v, H), scale=1 / 1.4426950408889634).double().cpu()
        assert bool(((out - want).abs() <= want * (2.0 ** -8 if dtype == BF else 2.0 ** -22)).all())
