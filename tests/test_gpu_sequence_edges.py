"""Attention over token sequences at the edges of what a call may be: sizes, biases and scores that a test of ordinary calls
does not reach."""
import math

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


LEVELS = {"high": [0, 80, 160, 250], "higher": [250, 250, 0, 250], "low": [-250, -200, -220, -150], "lower": [-100, -250, -250, -200]}


@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("value", [torch.finfo(FP).min, -1e30, -1e9, -1e6, -3e3, torch.finfo(FP).max, 1e9])
@pytest.mark.parametrize("levels", list(LEVELS))
@pytest.mark.parametrize("B,L,Hq,Hkv,D,table_grad", [(1, 250, 2, 1, 64, True), (2, 250, 4, 2, 30, False), (16, 250, 16, 8, 64, True), (16, 250, 16, 8, 30, False),
                                                     (16, 250, 16, 16, 128, False)])
def test_biases_far_from_zero_leave_the_softmax_of_large_scores(cuda0, B, L, Hq, Hkv, D, table_grad, levels, value, dtype):
    """A table of one finite number, however far from zero: the softmax of the scores alone, and its gradients, also where the
    scores (levels of base-2 logits by tile of 64 keys; whole numbers, exact in both types) leave fp32's exponents.  Small calls, with
    their split form, and calls that fill the chip; without gradients as well."""
    from oracle import sequence_oracle as S
    from test_gpu_sequence import _within
    K = _K()
    gen = torch.Generator().manual_seed(D)
    level = torch.tensor(LEVELS[levels], dtype=FP).repeat_interleave(64)[:L]
    k = (level.view(1, L, 1, 1) + torch.randint(-3, 4, (1, L, Hkv, D), generator=gen)).to(dtype)
    q, v, dout = torch.ones(1, L, Hq, D).to(dtype), torch.randn(1, L, Hkv, D, generator=gen).to(dtype), torch.randn(1, L, Hq, D, generator=gen).to(dtype)
    bmap = torch.randint(0, 4, (2 * 40 + 1,), generator=gen, dtype=torch.int32)
    scale = math.log(2) / D
    ref = S.attention(q.double(), k.double(), v.double(), 150, 0, 20, scale, table=torch.zeros(4, Hq, dtype=torch.float64), buckets=bmap,
                      dout=dout.double(), dtype=dtype, table_grad=table_grad)
    on = lambda t: t.to(cuda0).expand(B, -1, -1, -1).contiguous()
    leaves = [on(t).requires_grad_() for t in (q, k, v)] + [torch.full((4, Hq), value, device=cuda0).requires_grad_(table_grad)]
    kw = dict(window=(150, 0), sinks=20, scale=scale, bias_table=leaves[3], bias_buckets=bmap.to(cuda0))
    out = K.band_attention(*leaves[:3], **kw)
    grads = torch.autograd.grad(out, leaves[:4 if table_grad else 3], on(dout))
    with torch.no_grad():
        again = K.band_attention(*leaves[:3], **kw)
    for name, got in [("out", out), ("out (no grad)", again)] + list(zip(("dq", "dk", "dv"), grads)):
        want, bound = ref[name.split(" ")[0]]
        _within(name, got, want.expand(B, -1, -1, -1), bound.expand(B, -1, -1, -1))
    if table_grad:      # (B equal sequences: their sum)
        want, bound = ref["dtable"]
        _within("dtable", grads[3], B * want, B * (bound + B * S.F * want.abs()))


@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("value", [torch.finfo(FP).min, -1e9])
@pytest.mark.parametrize("levels", list(LEVELS))
@pytest.mark.parametrize("D", [30, 128])
def test_new_tokens_whose_biases_are_all_far_from_zero(cuda0, D, levels, value, dtype):
    """the same for single rows over long caches, whose keys are shared out"""
    from oracle import sequence_oracle as S
    from test_gpu_sequence import _within
    K = _K()
    gen = torch.Generator().manual_seed(D)
    L = 4000
    level = torch.tensor(LEVELS[levels], dtype=FP).repeat_interleave(1000)
    k = (level.view(1, L, 1, 1) + torch.randint(-3, 4, (1, L, 2, D), generator=gen)).to(dtype)
    q, v = torch.ones(1, 1, 4, D).to(dtype), torch.randn(1, L, 2, D, generator=gen).to(dtype)
    bmap = torch.zeros(2 * 40 + 1, dtype=torch.int32)
    scale = math.log(2) / D
    lens = torch.tensor([4000, 0, 1, 1700], dtype=torch.int32)
    four = lambda t: t.expand(4, -1, -1, -1).contiguous()
    ref = S.attention(four(q).double(), four(k).double(), four(v).double(), None, 0, 0, scale, k_lens=lens, dtype=dtype)["out"]
    with torch.no_grad():
        out = K.band_attention(four(q).to(cuda0), four(k).to(cuda0), four(v).to(cuda0), window=(None, 0), scale=scale, k_lens=lens.to(cuda0),
                               bias_table=torch.full((1, 4), value, device=cuda0), bias_buckets=bmap.to(cuda0))
    _within("out", out, *ref)


@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("B,Hq", [(1, 2), (16, 16)])
def test_rows_that_see_one_not_a_number_key_show_it(cuda0, B, Hq, bias, dtype):
    """windows of one key, and of a few: a row that sees the bad key is not finite, whether it sees another one or not; the
    others are what they are without it"""
    K = _K()
    gen = torch.Generator().manual_seed(4)
    L, at = 160, 70
    q, k, v = (torch.randn(B, L, Hq, 32, generator=gen).to(dtype).to(cuda0) for _ in range(3))
    kw = dict(bias_table=torch.zeros(1, Hq, device=cuda0), bias_buckets=torch.zeros(5, dtype=torch.int32, device=cuda0)) if bias else {}
    bad = k.clone()
    bad[:, at, :, 3] = float("nan")
    for left in (0, 4):
        clean, out = (K.band_attention(q, x, v, window=(left, 0), **kw) for x in (k, bad))
        sees = torch.arange(L, device=cuda0)
        sees = (sees >= at) & (sees <= at + left)
        assert torch.isnan(out[:, sees]).all() and torch.isfinite(out[:, ~sees]).all()
        assert float((out[:, ~sees] - clean[:, ~sees]).abs().max()) <= 2.0 ** -7 * float(v.abs().max())
    # a new token whose only visible key of a share is the bad one
    long = torch.randn(1, 4000, Hq, 32, generator=gen).to(dtype).to(cuda0)
    one = long.clone()
    one[:, 3999 - 128, :, 3] = float("nan")
    assert torch.isnan(K.band_attention(q[:1, :1], one, long, window=(128, 0), **kw)).all()
    one = long.clone()
    one[:, 0, :, 3] = float("nan")
    assert torch.isnan(K.band_attention(q[:1, :1], one, long, window=(64, 0), sinks=1, **kw)).all()
    assert torch.isfinite(K.band_attention(q[:1, :1], one, long, window=(64, 0), **kw)).all()


@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("left", [1, 2, 40])
@pytest.mark.parametrize("B,L,Hq,Hkv,D", [(2, 150, 4, 2, 64), (1, 90, 2, 2, 30), (16, 150, 16, 4, 64), (8, 200, 16, 16, 30), (8, 140, 16, 8, 128),
                                           (1, 150, 2, 1, 33)])
def test_gradients_of_scores_under_one_dominant_key(cuda0, B, L, Hq, Hkv, D, left, dtype):
    """Rows whose softmax is nearly one key: dS is small beside dP and delta, which have to agree far better than the result's own
    rounding.  q and k are small whole numbers, so that scores carry the scaling's roundings alone; with and without a
    bias that wants no gradient."""
    from oracle import sequence_oracle as S
    from test_gpu_sequence import _within
    K = _K()
    gen = torch.Generator().manual_seed(left)
    ints = lambda h, n: torch.randint(-n, n + 1, (B, L, h, D), generator=gen).to(dtype)
    q, k = ints(Hq, 1), ints(Hkv, 2)
    v, dout = torch.randn(B, L, Hkv, D, generator=gen).to(dtype), torch.randn(B, L, Hq, D, generator=gen).to(dtype)
    table, bmap = torch.randn(4, Hq, generator=gen), torch.randint(0, 4, (9,), generator=gen, dtype=torch.int32)
    for bias in (False, True):
        ref = S.attention(q.double(), k.double(), v.double(), left, 0, 0, 0.5, table=table.double() if bias else None, buckets=bmap if bias else None,
                          dout=dout.double(), dtype=dtype, table_grad=False, score_roundings=4, whole_delta=True)
        leaves = [t.to(cuda0).requires_grad_() for t in (q, k, v)]
        kw = dict(bias_table=table.to(cuda0), bias_buckets=bmap.to(cuda0)) if bias else {}
        out = K.band_attention(*leaves, window=(left, 0), scale=0.5, **kw)
        _within("out", out, *ref["out"])
        for name, g in zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, dout.to(cuda0))):
            _within(name, g, *ref[name])


@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("B,H", [(16, 16), (1, 1)])
@pytest.mark.parametrize("top", [2.0 ** 40, -2.0 ** 40, 2.0 ** 70])
def test_scores_beyond_what_fp32_tells_apart(cuda0, top, B, H, dtype):
    """Scores of `top` and, for every third key, lower by a 2^-7 of it: the mean of the others' values, though the scores' scaling
    alone rounds by thousands.  Tolerance as for equal keys."""
    K = _K()
    L, D = 250, 64
    k = torch.full((1, L, 1, D), top / D)
    low = torch.arange(L) % 3 == 1
    k[:, low] = (top - abs(top) / 128) / D
    v = torch.randint(0, 8, (1, L, 1, D), generator=torch.Generator().manual_seed(2)).float()
    on = lambda t: t.to(dtype).to(cuda0).expand(B, L, H, D).contiguous()
    assert torch.equal(k.to(dtype).float(), k)
    want = v[0, ~low, 0].double().mean(0)
    for scale in (0.125, 1 / 3, 0.7):
        out = K.band_attention(on(torch.ones(1, L, 1, D)), on(k), on(v), scale=scale).double().cpu()
        assert bool(((out - want).abs() <= want * (2.0 ** -8 if dtype == BF else 2.0 ** -22)).all()), scale


# (bf16 calls keep a row's probability of 1 up to scores of 2^15: off by 2^-9 there, which is rounded away)
@pytest.mark.parametrize("dtype,top", [(BF, 201 * 2.0 ** 7)] + [(FP, 201 * x) for x in (2.0 ** 7, 2.0 ** 13, 2.0 ** 33, -2.0 ** 13)])
@pytest.mark.parametrize("B,L,Hq,Hkv,D", [(1, 150, 2, 1, 64), (16, 150, 16, 4, 64), (8, 140, 16, 16, 30), (8, 140, 16, 8, 128)])
def test_gradients_of_rows_of_one_key_with_large_scores(cuda0, top, B, L, Hq, Hkv, D, dtype):
    """Every row's softmax is one key, 2^9 and more above the others (their probabilities are below 2^-240, zero), however the
    scaling rounds its score: the result is that key's value, dv its rows' dout added up, and the scores have no gradient at all."""
    K = _K()
    gen = torch.Generator().manual_seed(D)
    k = torch.zeros(B, L, Hkv, D)
    k[..., 0] = top - abs(top) / 201 * (25 if abs(top) < 2.0 ** 16 else 1)      # (bf16 has 8 bits: 176 and 200 of 201)
    k[:, 17, :, 0] = top
    assert torch.equal(k.to(dtype).float(), k)
    q = torch.zeros(B, L, Hq, D)
    q[..., 0] = 1.0
    v, dout = torch.randn(B, L, Hkv, D, generator=gen).to(dtype), torch.randn(B, L, Hq, D, generator=gen).to(dtype)
    G = Hq // Hkv
    total = dout.double().sum(1).view(B, Hkv, G, D).sum(2)
    bound = (L * G + 8) * 2.0 ** -24 * dout.double().abs().sum(1).view(B, Hkv, G, D).sum(2) + torch.finfo(dtype).eps / 2 * total.abs()
    for scale in (0.7, 1 / 3):
        leaves = [t.to(dtype).to(cuda0).requires_grad_() for t in (q, k, v)]
        out = K.band_attention(*leaves, scale=scale)
        assert torch.equal(out, leaves[2][:, 17:18].repeat_interleave(G, 2).expand_as(out))
        dq, dk, dv = (g.double().cpu() for g in torch.autograd.grad(out, leaves, dout.to(cuda0)))
        assert not dq.any() and not dk.any()
        assert not dv[:, :17].any() and not dv[:, 18:].any()
        assert bool(((dv[:, 17] - total).abs() <= bound).all())
