"""Attention over token sequences in calls large enough for the kernels of prompts and training batches (128 query rows a
workgroup), against the 64-bit restatement, entry by entry within its bounds.  Smaller calls, with their split forms, are
in test_gpu_sequence.py."""
import math

import pytest
import torch

from oracle import sequence_oracle as S
from test_gpu_sequence import _inputs, _layout, _within

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float32


def _K():
    from visiontransformer_amd import functional as K
    return K


def _is_large(B, Lq, Hq, Hkv):
    """the library's rule: more than 32 rows on a key head, and 128-row blocks for all 256 CUs (the dq kernel's 128-row form
    asks for the second alone)"""
    return Lq * (Hq // Hkv) > 32 and B * Hq * ((Lq + 127) // 128) >= 256


def _lengths(kind, B, Lq, Lk):
    """(q_lens, k_lens): "ragged" is a padded batch with an empty sequence and one of one token, "both" has lengths of their own"""
    if kind is None:
        return None, None
    if kind == "ragged":
        n = torch.tensor([[Lk, 0, 1, Lk // 2, Lk - 1, 65][b % 6] for b in range(B)], dtype=torch.int32)
        return n, n
    return (torch.tensor([[Lq, 5, Lq + 9, -3, 70][b % 5] for b in range(B)], dtype=torch.int32),
            torch.tensor([[Lk, 3, Lk // 2, Lk + 100, 64][b % 5] for b in range(B)], dtype=torch.int32))


def _check(dev, case, dtype, seed, buckets=0, distance=0, table_grad=True):
    K = _K()
    B, Lq, Lk, Hq, Hkv, D, left, right, sinks, lens, layout = case
    assert _is_large(B, Lq, Hq, Hkv), "this case belongs to the tests of small calls"
    q, k, v, dout, gen = _inputs((B, Lq, Hq, D), (B, Lk, Hkv, D), dtype, seed)
    ql, kl = _lengths(lens, B, Lq, Lk)
    table = bmap = None
    if buckets:
        table = torch.randn(buckets, Hq, generator=gen) * 0.7
        bmap = torch.tensor(S.bucket_map(buckets, distance, right == 0), dtype=torch.int32)
    ref = S.attention(q.double(), k.double(), v.double(), left, right, sinks, D ** -0.5, ql, kl, None if table is None else table.double(), bmap,
                      dout.double(), dtype, table_grad)
    leaves = [_layout(t, layout, dev).requires_grad_() for t in (q, k, v)]
    tab = None if table is None else table.to(dev).requires_grad_(table_grad)
    kw = dict(window=(left, right), sinks=sinks, q_lens=None if ql is None else ql.to(dev), k_lens=None if kl is None else kl.to(dev),
              bias_table=tab, bias_buckets=None if bmap is None else bmap.to(dev))
    with torch.no_grad():
        _within("out (no grad)", K.band_attention(*leaves, **kw), *ref["out"])
    out = K.band_attention(*leaves, **kw)
    _within("out", out, *ref["out"])
    if tab is not None and table_grad:
        leaves.append(tab)
    for name, g in zip(("dq", "dk", "dv", "dtable"), torch.autograd.grad(out, leaves, _layout(dout, layout, dev))):
        _within(name, g, *ref[name])


#  B   Lq   Lk   Hq  Hkv D    left  right sinks lens      layout
LARGE = [
    (16, 150, 150, 16, 4, 64, 33, 17, 2, None, "dense"),
    (8, 200, 200, 16, 16, 30, 20, 20, 4, None, "even"),
    (8, 200, 200, 16, 16, 30, 20, 20, 4, "ragged", "packed"),
    (8, 140, 260, 16, 4, 128, None, 0, 0, None, "heads first"),
    (8, 260, 140, 16, 2, 33, 10, 0, 1, None, "packed"),          # more queries than keys: the first rows see nothing
    (16, 129, 129, 16, 4, 64, None, None, 0, "ragged", "dense"),
    (5, 390, 390, 16, 8, 96, 100, 0, 70, "both", "even"),
    (8, 257, 257, 16, 16, 7, None, 0, 0, None, "packed"),
    (3, 520, 520, 32, 4, 128, 200, 50, 130, "ragged", "even"),
    (16, 190, 320, 8, 8, 32, 100, 5, 130, "both", "dense"),
    (1, 8200, 333, 8, 1, 48, 60, None, 3, None, "dense"),         # rows far ahead of the first key
]


@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("case", LARGE, ids=lambda c: "-".join(str(x) for x in c).replace(" ", "_"))
def test_large_calls(cuda0, case, dtype):
    _check(cuda0, case, dtype, 17)


LARGE_BIAS = [
    ((8, 150, 150, 16, 4, 64, None, None, 0, None, "dense"), 32, 16),
    ((8, 200, 200, 16, 16, 30, 150, 0, 4, None, "even"), 32, 128),
    ((8, 140, 260, 16, 4, 128, None, None, 0, "both", "packed"), 64, 300),
    ((8, 300, 300, 16, 8, 64, 40, 40, 70, "ragged", "heads first"), 8, 32),
    ((8, 129, 129, 16, 16, 9, 500, 0, 3, "ragged", "dense"), 16, 512),
]


@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("table_grad", [True, False])
@pytest.mark.parametrize("case,buckets,distance", LARGE_BIAS, ids=[str(i) for i in range(len(LARGE_BIAS))])
def test_large_calls_with_bias(cuda0, case, buckets, distance, table_grad, dtype):
    _check(cuda0, case, dtype, 18, buckets, distance, table_grad)


# base-2 logits by tile of 64 keys: the reference of a row is its first tile's maximum, which is moved up when sums pass 2^60
# (steps below 127), or made a running maximum in a second pass when they overflow
LEVELS = {"moved up": [0, 80, 160, 250], "moved up after the sinks": [-100, 20, 100, 60], "second pass": [0, 250, 120, 250],
          "second pass, late": [0, 20, -30, 240], "falling": [250, 100, 0, -250], "low sinks": [-250, -250, 100, 120]}


@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("D", [30, 64, 128])
@pytest.mark.parametrize("levels", list(LEVELS), ids=lambda n: n.replace(" ", "_"))
def test_large_calls_with_logits_that_climb(cuda0, levels, D, dtype):
    """Whole numbers of few bits, so that inputs are exact in both types; scale ln 2 / D makes a level a power of two.  Rows of
    sequences that see everything, and causal ones with a window that only the sinks' tile reaches."""
    K = _K()
    B, L, Hq, Hkv = 16, 250, 16, 4
    assert _is_large(B, L, Hq, Hkv)
    gen = torch.Generator().manual_seed(D)
    level = torch.tensor(LEVELS[levels], dtype=torch.float32).repeat_interleave(64)[:L]
    k = (level.view(1, L, 1, 1) + torch.randint(-3, 4, (1, L, Hkv, D), generator=gen)).to(dtype)
    q = torch.ones(1, L, Hq, D).to(dtype)
    v, dout = torch.randn(1, L, Hkv, D, generator=gen).to(dtype), torch.randn(1, L, Hq, D, generator=gen).to(dtype)
    for left, right, sinks in ((None, None, 0), (100, 0, 20)):
        ref = S.attention(q.double(), k.double(), v.double(), left, right, sinks, math.log(2) / D, dout=dout.double(), dtype=dtype)
        leaves = [t.to(cuda0).expand(B, -1, -1, -1).contiguous().requires_grad_() for t in (q, k, v)]
        out = K.band_attention(*leaves, window=(left, right), sinks=sinks, scale=math.log(2) / D)
        grads = torch.autograd.grad(out, leaves, dout.to(cuda0).expand(B, -1, -1, -1).contiguous())
        for name, got in zip(("out", "dq", "dk", "dv"), (out,) + grads):
            want, bound = ref[name]
            _within(name, got, want.expand(B, -1, -1, -1), bound.expand(B, -1, -1, -1))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("D", [30, 128])
def test_large_calls_keep_non_finite_values_with_the_rows_that_see_them(cuda0, D, dtype, bad):
    """one bad number in a key and one in a value, in a tile that rows on both sides of it read; what lies behind a sequence's
    keys is bad all through"""
    K = _K()
    B, L, Hq, Hkv, at = 16, 230, 16, 8, 100
    assert _is_large(B, L, Hq, Hkv)
    q, k, v, _, _ = _inputs((1, L, Hq, D), (1, L, Hkv, D), dtype, 8)
    ref = S.attention(q.double(), k.double(), v.double(), 20, 0, 2, D ** -0.5, None, torch.tensor([L - 9]), dtype=dtype)["out"]
    k2, v2 = k.clone(), v.clone()
    k2[0, at, 0, 3], v2[0, at, 0, 5] = bad, bad
    k2[0, at, 1, 3] = bad
    v2[0, at, 2, 5] = bad
    k2[0, L - 9:], v2[0, L - 9:] = bad, bad
    on = lambda t: t.to(cuda0).expand(B, -1, -1, -1).contiguous()
    out = K.band_attention(on(q), on(k2), on(v2), window=(20, 0), sinks=2, k_lens=torch.full((B,), L - 9, dtype=torch.int32, device=cuda0)).cpu()
    p = torch.arange(L) - 9
    sees = (p >= at) & (p <= at + 20)
    for b in (0, B - 1):
        for h in range(Hq):
            clean = ~sees if h < 6 else torch.ones_like(sees)
            _within("head %d" % h, out[b, clean, h], ref[0][0, clean, h], ref[1][0, clean, h])
            if h in (0, 1) or (h in (4, 5)):
                assert bool((~torch.isfinite(out[b, sees, h])).any(-1).all()), "rows that see the value must show it"


@pytest.mark.parametrize("step,L,hkv", [((1 << 28) + 64, 20, 1), ((1 << 24) - 64, 200, 1)], ids=["element by element", "16-byte pieces"])
def test_large_calls_over_rows_far_apart(cuda0, step, L, hkv):
    """keys and values whose rows end beyond 2^32 bytes, so far apart that a tile spans 2 GiB, and just not: the forward of
    large calls and of small ones, and the backward"""
    K = _K()
    if torch.cuda.mem_get_info(cuda0)[0] < 24 << 30:
        pytest.skip("needs 24 GiB of free device memory")
    room = torch.empty(L * step, dtype=BF, device=cuda0)
    for Hq in (256, 2):
        assert _is_large(1, L, Hq, 1) == (Hq == 256)
        q, k, v, dout, _ = _inputs((1, L, Hq, 64), (1, L, 1, 64), BF, 4)
        kg = room.as_strided((1, L, 1, 64), (0, step, 0, 1))
        vg = room.as_strided((1, L, 1, 64), (0, step, 0, 1), 4096)
        kg.copy_(k)
        vg.copy_(v)
        ref = S.attention(q.double(), k.double(), v.double(), 150, 0, 0, 0.125, dout=dout.double(), dtype=BF)
        leaves = [q.to(cuda0).requires_grad_(), kg.detach().requires_grad_(), vg.detach().requires_grad_()]
        assert leaves[1].stride(1) == step
        out = K.band_attention(*leaves, window=(150, 0))
        _within("out", out, *ref["out"])
        for name, g in zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, dout.to(cuda0))):
            _within(name, g, *ref[name])
    del room


@pytest.mark.parametrize("sinks", [3, 140])
@pytest.mark.parametrize("dtype", [FP, BF])
def test_sinks_of_many_sequences(cuda0, dtype, sinks):
    """many short windows and rows far behind their sinks: the sinks' blocks are cut by what there is to do in all"""
    K = _K()
    B, L, D = 512, 4096, 8
    q, k, v, dout, _ = _inputs((1, L, 1, D), (1, L, 1, D), dtype, 5)
    ref = S.attention(q.double(), k.double(), v.double(), 20, 0, sinks, D ** -0.5, dout=dout.double(), dtype=dtype)
    on = lambda t: t.to(cuda0).expand(B, -1, -1, -1).contiguous()
    leaves = [on(t).requires_grad_() for t in (q, k, v)]
    out = K.band_attention(*leaves, window=(20, 0), sinks=sinks)
    grads = torch.autograd.grad(out, leaves, on(dout))
    for name, got in zip(("out", "dq", "dk", "dv"), (out,) + grads):
        got = got.detach()
        assert bool((got == got[:1]).all())      # (equal sequences)
        _within(name, got[B - 1:], *ref[name])
