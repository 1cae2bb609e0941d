"""Attention over token sequences (functional.qk_norm_rotary, functional.band_attention) against the 64-bit restatement
in oracle/sequence_oracle.py, entry by entry within its bounds for the roundings of the kernels."""
import math

import pytest
import torch

from oracle import sequence_oracle as S

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float32


def _K():
    from visiontransformer_amd import functional as K
    return K


def _within(name, got, want, bound, slack=1.0):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert bool(torch.isfinite(got).all()), "%s: not finite" % name
    off = (got - want).abs()
    over = off > slack * bound + 1e-30
    assert not bool(over.any()), "%s: %d of %d entries out of bounds, worst %g against %g at %s" % (
        name, int(over.sum()), off.numel(), float(off[over].max()), float(bound[over].max()), over.nonzero()[0].tolist())


def _layout(t, kind, dev):
    """t [B, L, H, D] on the GPU in other strides, values unchanged"""
    t = t.to(dev)
    B, L, H, D = t.shape
    if kind == "heads first":
        return t.transpose(1, 2).contiguous().transpose(1, 2)
    if kind == "packed":       # beside other columns, rows that begin on odd addresses
        room = torch.full((B, L, H * D + 3 * D + 1), float("nan"), dtype=t.dtype, device=dev)
        room[:, :, 1:1 + H * D] = t.reshape(B, L, H * D)
        return room[:, :, 1:1 + H * D].view(B, L, H, D) if H * D else t
    if kind == "even":         # 4-byte aligned rows
        room = torch.full((B, L, H, D + 2), float("nan"), dtype=t.dtype, device=dev)
        room[..., :D] = t
        return room[..., :D]
    return t.contiguous()


def _inputs(shape_q, shape_k, dtype, seed, std=1.0):
    gen = torch.Generator().manual_seed(seed)
    mk = lambda s: (torch.randn(*s, generator=gen) * std).to(dtype)
    return mk(shape_q), mk(shape_k), mk(shape_k), mk(shape_q), gen


# ----------------------------------------------------------------------------------------------
# attention
# ----------------------------------------------------------------------------------------------
#  B  Lq  Lk  Hq Hkv D   left  right sinks  lens     layout
CASES = [
    (1, 1, 1, 1, 1, 64, None, None, 0, None, "dense"),
    (2, 37, 37, 2, 2, 32, None, None, 0, None, "dense"),
    (1, 128, 128, 1, 1, 64, None, 0, 0, None, "dense"),
    (1, 129, 129, 4, 2, 64, None, 0, 0, None, "heads first"),
    (2, 200, 200, 6, 6, 30, 20, 20, 4, None, "even"),
    (2, 200, 200, 6, 6, 30, 20, 20, 4, None, "packed"),
    (1, 300, 300, 4, 1, 128, 64, 0, 3, None, "dense"),
    (1, 257, 257, 2, 1, 96, 0, 0, 70, None, "heads first"),
    (1, 150, 333, 3, 1, 48, 100, 5, 130, None, "dense"),
    (1, 333, 150, 2, 2, 33, 10, 0, 1, None, "packed"),
    (3, 190, 190, 4, 2, 64, 33, 17, 2, "ragged", "dense"),
    (4, 70, 140, 4, 4, 7, None, 0, 0, "both", "packed"),
    (2, 65, 65, 2, 2, 1, 3, 3, 1, None, "packed"),
    (1, 64, 0, 2, 2, 16, None, None, 0, None, "dense"),
    (1, 260, 260, 2, 2, 64, 0, 0, 0, None, "dense"),       # every row sees itself only
    (2, 140, 140, 8, 2, 128, None, None, 0, "ragged", "even"),
]


def _lens(kind, B, Lq, Lk):
    if kind is None:
        return None, None
    if kind == "ragged":       # padded batch: an empty sequence, one token, all of it
        n = torch.tensor([Lk, 0, 1, Lk // 2][:B], dtype=torch.int32)
        return n, n
    return torch.tensor([Lq, 5, Lq + 9, -3][:B], dtype=torch.int32), torch.tensor([Lk, 3, Lk // 2, Lk + 100][:B], dtype=torch.int32)


def _check_attention(dev, case, dtype, seed, buckets=0, distance=0, table_grad=True, std=1.0):
    K = _K()
    B, Lq, Lk, Hq, Hkv, D, left, right, sinks, lens, layout = case
    q, k, v, dout, gen = _inputs((B, Lq, Hq, D), (B, Lk, Hkv, D), dtype, seed, std)
    ql, kl = _lens(lens, B, Lq, Lk)
    table = bmap = None
    if buckets:
        table = torch.randn(buckets, Hq, generator=gen) * 0.7
        bmap = torch.tensor(S.bucket_map(buckets, distance, right == 0), dtype=torch.int32)
    scale = D ** -0.5
    ref = S.attention(q.double(), k.double(), v.double(), left, right, sinks, scale, ql, kl, None if table is None else table.double(), bmap,
                      dout.double(), dtype, table_grad)
    leaves = [_layout(t, layout, dev).requires_grad_() for t in (q, k, v)]
    tab = None if table is None else table.to(dev).requires_grad_(table_grad)
    kw = dict(window=(left, right), sinks=sinks, q_lens=None if ql is None else ql.to(dev), k_lens=None if kl is None else kl.to(dev),
              bias_table=tab, bias_buckets=None if bmap is None else bmap.to(dev))
    out = K.band_attention(*leaves, **kw)
    _within("out", out, *ref["out"])
    if tab is not None and table_grad:
        leaves.append(tab)
    grads = torch.autograd.grad(out, leaves, _layout(dout, layout, dev))
    for name, g in zip(("dq", "dk", "dv", "dtable"), grads):
        _within(name, g, *ref[name])
    with torch.no_grad():      # the call without gradients may run another kernel
        _within("out (no grad)", K.band_attention(*[t.detach() for t in leaves[:3]], **kw), *ref["out"])
    return leaves, kw, out, grads


@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in c).replace(" ", "_"))
def test_attention(cuda0, case, dtype):
    _check_attention(cuda0, case, dtype, 11)


BIAS_CASES = [
    ((2, 100, 100, 2, 2, 64, None, None, 0, None, "dense"), 32, 16),
    ((1, 300, 300, 4, 2, 30, None, 0, 0, None, "even"), 32, 128),
    ((2, 260, 260, 2, 2, 64, 40, 40, 4, "ragged", "dense"), 8, 32),
    ((1, 200, 420, 3, 3, 128, None, None, 0, None, "packed"), 64, 300),
    ((1, 700, 700, 2, 1, 32, None, None, 0, None, "dense"), 16, 64),
    ((4, 70, 140, 4, 4, 48, 500, 0, 3, "both", "dense"), 64, 512),
    ((1, 5, 9, 1, 1, 64, None, None, 0, None, "dense"), 4, 2),
]


@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("case,buckets,distance", BIAS_CASES, ids=[str(i) for i in range(len(BIAS_CASES))])
def test_attention_with_bias(cuda0, case, buckets, distance, dtype):
    _check_attention(cuda0, case, dtype, 12, buckets, distance)


@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("D", [30, 64, 128])
def test_the_longest_bias_map(cuda0, dtype, D):
    """512 distances to each side: the most LDS that a call takes"""
    _check_attention(cuda0, (1, 90, 700, 2, 2, D, None, None, 0, None, "dense"), dtype, 14, 64, 512)


@pytest.mark.parametrize("dtype", [FP, BF])
def test_bias_without_its_gradient(cuda0, dtype):
    _check_attention(cuda0, BIAS_CASES[1][0], dtype, 13, 32, 128, table_grad=False)


@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("value", [float("-inf"), torch.finfo(torch.float32).min, -1e9, -1e4])
@pytest.mark.parametrize("masked", [70, 129])
@pytest.mark.parametrize("table_grad", [True, False])
def test_masks_in_a_bias_table(cuda0, dtype, value, masked, table_grad):
    """A table that masks the nearest `masked` distances of a causal call (129: all of them), so that the first rows see
    nothing else.  -inf takes those keys away: the reference leaves them out of the window.  A finite value leaves the softmax
    of the scores to rows that have nothing better and nothing to the others; the reference has it as -100, whose weight of
    4e-44 beside any other is far below its bounds."""
    K = _K()
    B, L, Hq, Hkv, D, M = 1, 300, 2, 1, 64, 128
    q, k, v, dout, gen = _inputs((B, L, Hq, D), (B, L, Hkv, D), dtype, 31)
    table = torch.randn(4, Hq, generator=gen) * 0.7
    bmap = torch.tensor([0 if -masked < d <= 0 else 1 + (d & 1) for d in range(-M, M + 1)], dtype=torch.int32)
    table[0] = value
    instead = table.double()
    instead[0] = -100.0
    gone = value == float("-inf")
    ref = S.attention(q.double(), k.double(), v.double(), None, (-masked if masked <= M else -10 ** 6) if gone else 0, 0, D ** -0.5, None, None,
                      instead, bmap, dout.double(), dtype, table_grad)
    leaves = [t.to(cuda0).requires_grad_() for t in (q, k, v)] + [table.to(cuda0).requires_grad_(table_grad)]
    kw = dict(window=(None, 0), bias_table=leaves[3], bias_buckets=bmap.to(cuda0))
    out = K.band_attention(*leaves[:3], **kw)
    grads = torch.autograd.grad(out, leaves[:4 if table_grad else 3], dout.to(cuda0))
    _within("out", out, *ref["out"])
    for name, g in zip(("dq", "dk", "dv", "dtable"), grads):
        _within(name, g, *ref[name])
    with torch.no_grad():
        _within("out (no grad)", K.band_attention(*leaves[:3], **kw), *ref["out"])
    if gone:
        rows = L if masked > M else masked
        assert not out[:, :rows].any() and not grads[0][:, :rows].any()


#  rows over a cache: B Lq Lk Hq Hkv D left right sinks
STEPS = [
    (3, 1, 1000, 4, 1, 64, None, 0, 0), (2, 1, 5000, 8, 8, 128, 1023, 0, 4), (1, 1, 1, 2, 2, 30, 5, 0, 0),
    (2, 2, 777, 6, 2, 48, 100, 0, 40), (1, 5, 3000, 16, 2, 64, 600, 0, 1), (1, 13, 2050, 4, 1, 33, None, None, 0),
    (2, 40, 4000, 2, 1, 128, 2000, 0, 4), (40, 1, 100, 1, 1, 7, 10, 0, 2), (1, 100, 100, 1, 1, 64, 30, 30, 3),
]


@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("step", STEPS, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("buckets", [0, 32])
def test_rows_over_a_cache(cuda0, step, dtype, buckets):
    """calls without gradients on few rows, ragged key lengths with zero and one among them"""
    K = _K()
    B, Lq, Lk, Hq, Hkv, D, left, right, sinks = step
    q, k, v, _, gen = _inputs((B, Lq, Hq, D), (B, Lk, Hkv, D), dtype, 5)
    kl = torch.tensor([[Lk, 0, 1, Lk // 2, 2][b % 5] for b in range(B)], dtype=torch.int32)
    table = bmap = None
    if buckets:
        table, bmap = torch.randn(buckets, Hq, generator=gen), torch.tensor(S.bucket_map(buckets, 64, True), dtype=torch.int32)
    ref = S.attention(q.double(), k.double(), v.double(), left, right, sinks, D ** -0.5, None, kl, None if table is None else table.double(),
                      bmap, None, dtype)
    put = lambda t: None if t is None else t.to(cuda0)
    for layout in ("dense", "heads first", "packed"):
        # what lies behind a sequence's keys may be anything
        kg, vg = _layout(k, layout, cuda0), _layout(v, layout, cuda0)
        for b in range(B):
            kg[b, int(kl[b]):] = float("nan")
            vg[b, int(kl[b]):] = float("inf")
        out = K.band_attention(_layout(q, layout, cuda0), kg, vg, window=(left, right), sinks=sinks, k_lens=put(kl), bias_table=put(table),
                               bias_buckets=put(bmap))
        _within(layout, out, *ref["out"])


def test_large_logits_and_running_maximum(cuda0):
    """scores in the hundreds, growing along the keys: the running maximum has to follow"""
    K = _K()
    for dtype in (FP, BF):
        _check_attention(cuda0, (1, 200, 200, 2, 2, 64, None, 0, 0, None, "dense"), dtype, 21, std=4.0)
        q = torch.ones(1, 150, 1, 32, dtype=dtype)
        k = (torch.arange(150).view(1, 150, 1, 1) / 8).expand(1, 150, 1, 32).to(dtype)
        v = torch.randn(1, 150, 1, 32, generator=torch.Generator().manual_seed(3)).to(dtype)
        for lq in (150, 1):
            ref = S.attention(q[:, :lq].double(), k.double(), v.double(), None, None, 0, 1.0, dtype=dtype)
            out = K.band_attention(q[:, :lq].to(cuda0), k.to(cuda0), v.to(cuda0), scale=1.0)
            _within("growing", out, *ref["out"])


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dtype", [FP, BF])
def test_non_finite_values_stay_with_the_rows_that_see_them(cuda0, dtype, bad):
    K = _K()
    q, k, v, _, _ = _inputs((1, 100, 2, 32), (1, 100, 2, 32), dtype, 8)
    ref = S.attention(q.double(), k.double(), v.double(), 20, 0, 2, 32 ** -0.5, dtype=dtype)["out"]
    k2, v2 = k.clone(), v.clone()
    k2[0, 40, 0, 3], v2[0, 40, 0, 5] = bad, bad
    for n in (100, 3):  # whole sequence; the last rows alone (which do not see key 40)
        out = K.band_attention(q[:, 100 - n:].to(cuda0), k2.to(cuda0), v2.to(cuda0), window=(20, 0), sinks=2).cpu()
        rows = torch.arange(100 - n, 100)
        sees = (rows >= 40) & (rows <= 60)
        for h in range(2):
            clean = ~sees if h == 0 else torch.ones_like(sees)
            _within("head %d" % h, out[0, clean, h], ref[0][0, rows[clean], h], ref[1][0, rows[clean], h])
            if h == 0 and n == 100:
                assert bool((~torch.isfinite(out[0, sees, h])).any(-1).all()), "rows that see the value must show it"


def test_padding_is_ignored_and_gets_zero_gradients(cuda0):
    K = _K()
    gen = torch.Generator().manual_seed(9)
    lens = torch.tensor([50, 0, 128], dtype=torch.int32)
    ts = [torch.randn(3, 130, 2, 32, generator=gen).to(BF) for _ in range(4)]
    for b, n in enumerate(lens.tolist()):
        for t in ts:
            t[b, n:] = float("nan")
    leaves = [t.to(cuda0).requires_grad_() for t in ts[:3]]
    out = K.band_attention(*leaves, q_lens=lens.to(cuda0), k_lens=lens.to(cuda0), window=(30, 30))
    grads = torch.autograd.grad(out, leaves, ts[3].to(cuda0))
    for b, n in enumerate(lens.tolist()):
        for t in (out,) + grads:
            assert float(t[b, n:].detach().abs().sum()) == 0.0
    clean = [torch.nan_to_num(t.double(), nan=0.0) for t in ts]
    ref = S.attention(*clean[:3], 30, 30, 0, 32 ** -0.5, lens, lens, dout=clean[3], dtype=BF)
    for name, t in zip(("out", "dq", "dk", "dv"), (out,) + grads):
        _within(name, t, *ref[name])


def test_gradients_against_differences(cuda0):
    """fp32: the loss along a random direction, central differences in 64 bits on the oracle's forward"""
    case = (2, 70, 90, 4, 2, 30, 40, 9, 3, None, "dense")
    leaves, kw, out, grads = _check_attention(cuda0, case, FP, 31, 16, 32)
    gen = torch.Generator().manual_seed(1)
    dout = _inputs((2, 70, 4, 30), (2, 90, 2, 30), FP, 31)[3]
    base = [t.detach().double().cpu() for t in leaves]
    dirs = [torch.randn(t.shape, generator=gen, dtype=torch.float64) for t in base]
    bmap = kw["bias_buckets"].cpu()

    def loss(s):
        x = [t + s * d for t, d in zip(base, dirs)]
        return float((S.attention(*x[:3], 40, 9, 3, 30 ** -0.5, table=x[3], buckets=bmap)["out"][0] * dout.double()).sum())

    h = 1e-4
    slope = (loss(h) - loss(-h)) / (2 * h)
    got = sum(float((g.double().cpu() * d).sum()) for g, d in zip(grads, dirs))
    size = sum(float((g.double().cpu() * d).abs().sum()) for g, d in zip(grads, dirs))
    # fp32 gradients: 2^-24 of the terms' absolute sum times a few dozen roundings; differences: h^2
    assert abs(got - slope) <= size * 64 * 2.0 ** -24 + 1e-6 * abs(slope), (got, slope)


@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("D", [7, 30, 64, 128])
def test_rows_that_see_one_key_have_no_gradient_of_their_scores(cuda0, dtype, D):
    """softmax of one number is constant: dq, dk and the bias' gradient are zeros, not what roundings leave"""
    K = _K()
    for L, window in ((1, (None, None)), (150, (0, 0))):
        q, k, v, dout, gen = _inputs((2, L, 4, D), (2, L, 2, D), dtype, 6)
        table = torch.randn(8, 4, generator=gen).to(cuda0).requires_grad_()
        bmap = torch.tensor(S.bucket_map(8, 16, False), dtype=torch.int32, device=cuda0)
        leaves = [t.to(cuda0).requires_grad_() for t in (q, k, v)] + [table]
        for kw in (dict(bias_table=table, bias_buckets=bmap), {}):
            out = K.band_attention(*leaves[:3], window=window, **kw)
            assert torch.equal(out, leaves[2].repeat_interleave(2, 2))
            grads = torch.autograd.grad(out, leaves if kw else leaves[:3], dout.to(cuda0))
            assert all(float(g.abs().max()) == 0.0 for i, g in enumerate(grads) if i != 2)
            t = None if not kw else table.detach().double().cpu()
            ref = S.attention(q.double(), k.double(), v.double(), *window, 0, D ** -0.5, table=t, buckets=None if t is None else bmap.cpu(),
                              dout=dout.double(), dtype=dtype)
            _within("dv", grads[2], *ref["dv"])   # (a probability of 1 is off by the rounding of its logit, which may be any size)


@pytest.mark.parametrize("dtype", [FP, BF])
def test_long_calls_of_rows_that_see_one_key(cuda0, dtype):
    """the same where the row blocks fill the chip: another forward kernel"""
    K = _K()
    q, k, v, dout, gen = _inputs((1, 4200, 8, 32), (1, 4200, 8, 32), dtype, 8)
    table = torch.randn(8, 8, generator=gen).to(cuda0).requires_grad_()
    bmap = torch.tensor(S.bucket_map(8, 16, False), dtype=torch.int32, device=cuda0)
    leaves = [t.to(cuda0).requires_grad_() for t in (q, k, v)] + [table]
    for kw in (dict(bias_table=table, bias_buckets=bmap), {}):
        out = K.band_attention(*leaves[:3], window=(0, 0), **kw)
        assert torch.equal(out, leaves[2])
        grads = torch.autograd.grad(out, leaves if kw else leaves[:3], dout.to(cuda0))
        assert all(float(g.abs().max()) == 0.0 for i, g in enumerate(grads) if i != 2)


def test_shared_heads_and_broadcast_inputs(cuda0):
    K = _K()
    gen = torch.Generator().manual_seed(2)
    one = torch.randn(1, 60, 1, 32, generator=gen).to(cuda0).requires_grad_()
    q = torch.randn(3, 60, 4, 32, generator=gen).to(cuda0)
    dout = torch.randn(3, 60, 4, 32, generator=gen)
    out = K.band_attention(q, one.expand(3, 60, 2, 32), one.expand(3, 60, 2, 32), window=(None, 0))
    (g,) = torch.autograd.grad(out, one, dout.to(cuda0))
    kv = one.detach().double().cpu().expand(3, 60, 2, 32).contiguous()
    ref = S.attention(q.double().cpu(), kv, kv.clone(), None, 0, 0, 32 ** -0.5, dout=dout.double())
    want = (ref["dk"][0] + ref["dv"][0]).sum((0, 2), keepdim=True)
    bound = (ref["dk"][1] + ref["dv"][1] + 8 * S.F * (ref["dk"][0].abs() + ref["dv"][0].abs())).sum((0, 2), keepdim=True)
    _within("shared", g, want, bound)


def test_the_same_call_gives_the_same_bits(cuda0):
    K = _K()
    q, k, v, dout, gen = _inputs((2, 500, 4, 64), (2, 500, 2, 64), BF, 3)
    table = torch.randn(32, 4, generator=gen).to(cuda0).requires_grad_()
    bmap = torch.tensor(S.bucket_map(32, 128, False), dtype=torch.int32, device=cuda0)
    leaves = [t.to(cuda0).requires_grad_() for t in (q, k, v)] + [table]
    runs = []
    for _ in range(3):
        out = K.band_attention(*leaves[:3], bias_table=table, bias_buckets=bmap)
        runs.append((out,) + torch.autograd.grad(out, leaves, dout.to(cuda0)))
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], r))


def test_offsets_beyond_32_bits(cuda0):
    """a cache whose rows lie 2^28 elements apart: 20 rows end beyond 2^32 elements (bytes: 2^33)"""
    K = _K()
    free = torch.cuda.mem_get_info(cuda0)[0]
    if free < 24 << 30:
        pytest.skip("needs 24 GiB of free device memory")
    step = (1 << 28) + 64
    room = torch.empty(20 * step, dtype=BF, device=cuda0)
    q, k, v, _, _ = _inputs((1, 20, 2, 64), (1, 20, 1, 64), BF, 4)
    kg = room.as_strided((1, 20, 1, 64), (0, step, 0, 1))
    vg = room.as_strided((1, 20, 1, 64), (0, step, 0, 1), 4096)
    kg.copy_(k)
    vg.copy_(v)
    ref = S.attention(q.double(), k.double(), v.double(), None, 0, 0, 0.125, dtype=BF)["out"]
    _within("prompt", K.band_attention(q.to(cuda0).requires_grad_(), kg, vg, window=(None, 0)), *ref)
    _within("step", K.band_attention(q[:, 19:].to(cuda0), kg, vg, window=(None, 0)), ref[0][:, 19:], ref[1][:, 19:])
    del room


def test_other_stream_and_graph_replay(cuda0):
    """forward with its split form, and a whole training pass, captured and replayed with new inputs and with eager work
    between the replays; every replay against the eager result"""
    K = _K()
    gen = torch.Generator(device=cuda0).manual_seed(5)
    mk = lambda *s: torch.randn(*s, device=cuda0, generator=gen).to(BF)
    bmap = torch.tensor(S.bucket_map(16, 64, True), dtype=torch.int32, device=cuda0)
    st = {"q1": mk(2, 1, 4, 64), "k1": mk(2, 3000, 2, 64), "v1": mk(2, 3000, 2, 64), "q": mk(2, 200, 4, 64), "k": mk(2, 200, 2, 64),
          "v": mk(2, 200, 2, 64), "g": mk(2, 200, 4, 64), "t": torch.randn(16, 4, device=cuda0, generator=gen)}
    lens = torch.tensor([3000, 1700], dtype=torch.int32, device=cuda0)

    def work(x):
        with torch.no_grad():
            step = K.band_attention(x["q1"], x["k1"], x["v1"], window=(None, 0), k_lens=lens)
        leaves = [x[n].detach().requires_grad_() for n in ("q", "k", "v", "t")]
        out = K.band_attention(*leaves[:3], window=(50, 0), sinks=2, bias_table=leaves[3], bias_buckets=bmap)
        return (step, out.detach()) + torch.autograd.grad(out, leaves, x["g"])

    side = torch.cuda.Stream(cuda0)
    side.wait_stream(torch.cuda.current_stream(cuda0))
    with torch.cuda.stream(side):
        for _ in range(2):
            warm = work(st)
    torch.cuda.current_stream(cuda0).wait_stream(side)
    for a, b in zip(warm, work(st)):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = work(st)
    for n in range(4):
        for t in st.values():
            t.copy_(torch.randn(t.shape, device=cuda0, generator=gen))
        lens.copy_(torch.tensor([3000 - 977 * n, 1 + n], dtype=torch.int32))
        graph.replay()
        got = [t.clone() for t in held]
        for a, b in zip(got, work(st)):
            assert torch.equal(a, b)
        torch.cuda.synchronize()


def test_refusals(cuda0):
    K = _K()
    z = lambda *s, dtype=FP: torch.zeros(*s, dtype=dtype, device=cuda0)
    q, k = z(2, 4, 4, 8), z(2, 6, 2, 8)
    ints = lambda n: torch.zeros(n, dtype=torch.int32, device=cuda0)
    for args, kw, text in [
        ((q, k.bfloat16(), k), {}, "bfloat16"),
        ((q.half(), k.half(), k.half()), {}, "dtype"),
        ((q[0], k, k), {}, "must be"),
        ((q, k, z(2, 5, 2, 8)), {}, "do not go together"),
        ((q, z(2, 6, 3, 8), z(2, 6, 3, 8)), {}, "over 3 key heads"),
        ((q, z(2, 6, 0, 8), z(2, 6, 0, 8)), {}, "key heads"),
        ((z(2, 4, 4, 130), z(2, 6, 2, 130), z(2, 6, 2, 130)), {}, "head dim 130"),
        ((q, k, k), dict(window=(-1, 0)), "left"),
        ((q, k, k), dict(window=(None, 1.5)), "right"),
        ((q, k, k), dict(sinks=-1), "sinks"),
        ((q, k, k), dict(scale=0.0), "scale"),
        ((q, k, k), dict(scale=float("nan")), "scale"),
        ((q, k, k), dict(k_lens=ints(3)), "k_lens"),
        ((q, k, k), dict(q_lens=torch.zeros(2, device=cuda0)), "q_lens"),
        ((q, k, k), dict(k_lens=torch.zeros(2, dtype=torch.int32)), "k_lens"),
        ((q, k, k), dict(bias_table=z(4, 4)), "go together"),
        ((q, k, k), dict(bias_table=z(4, 3), bias_buckets=ints(9)), "bias_table"),
        ((q, k, k), dict(bias_table=z(4, 4), bias_buckets=ints(8)), "2 M"),
        ((q, k, k), dict(bias_table=z(4, 4), bias_buckets=ints(1027)), "2 M"),
    ]:
        with pytest.raises(RuntimeError, match=text):
            K.band_attention(*args, **kw)
    for args, kw, text in [
        ((q, k), {}, "differ in more"),
        ((q, q.bfloat16()), {}, "bfloat16"),
        ((q, q), dict(q_weight=z(7)), "q_weight"),
        ((q, q), dict(freqs=z(5)), "need more"),
        ((q, q), dict(freqs=z(2, 3)), "need more"),
        ((q, q), dict(freqs=z(2).double()), "freqs"),
        ((q, q), dict(positions=ints(4)), "without freqs"),
        ((q, q), dict(freqs=z(2), positions=ints(5)), "positions"),
        ((q, q), dict(freqs=z(2), positions=z(4)), "positions"),
        ((z(1, 1, 1, 129), z(1, 1, 1, 129)), {}, "head dim 129"),
    ]:
        with pytest.raises(RuntimeError, match=text):
            K.qk_norm_rotary(*args, **kw)
    # a second derivative is refused, not silently wrong
    x = q.clone().requires_grad_()
    (g,) = torch.autograd.grad(K.band_attention(x, k, k).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)


def test_empty_sizes(cuda0):
    K = _K()
    z = lambda *s: torch.zeros(*s, device=cuda0)
    for B, Lq, Lk, Hq, Hkv in ((0, 4, 4, 2, 1), (2, 0, 4, 2, 1), (2, 4, 0, 2, 1), (1, 4, 4, 0, 0), (1, 0, 0, 1, 1)):
        ts = [t.requires_grad_() for t in (z(B, Lq, Hq, 8) + 1, z(B, Lk, Hkv, 8), z(B, Lk, Hkv, 8))]
        tab = z(4, Hq).requires_grad_()
        out = K.band_attention(*ts, bias_table=tab, bias_buckets=torch.zeros(5, dtype=torch.int32, device=cuda0))
        assert out.shape == (B, Lq, Hq, 8) and float(out.detach().abs().sum()) == 0.0
        for t, g in zip(ts + [tab], torch.autograd.grad(out.sum(), ts + [tab])):
            assert g.shape == t.shape and float(g.abs().sum()) == 0.0
        a, b = K.qk_norm_rotary(ts[0], z(B, Lq, Hkv, 8), z(8).requires_grad_())
        assert a.shape == ts[0].shape and b.shape == (B, Lq, Hkv, 8)
        torch.autograd.grad(a.sum() + b.sum(), ts[0])


# ----------------------------------------------------------------------------------------------
# norm + rotation
# ----------------------------------------------------------------------------------------------
#  B  L   Hq Hkv D   axes pairs interleaved layout
ROTARY = [
    (2, 5, 4, 2, 64, 1, 32, False, "dense"), (2, 5, 4, 2, 64, 1, 32, True, "heads first"),
    (1, 70, 6, 6, 30, 2, 7, False, "even"), (1, 70, 6, 6, 30, 1, 15, True, "packed"), (2, 33, 3, 1, 30, 1, 15, False, "even"),
    (1, 300, 2, 2, 128, 1, 64, False, "dense"), (1, 17, 2, 1, 128, 2, 20, True, "packed"), (2, 9, 1, 3, 127, 1, 63, False, "packed"),
    (1, 9, 2, 2, 7, 3, 1, True, "dense"), (3, 1, 2, 2, 1, 1, 0, False, "dense"), (2, 6, 5, 0, 48, 1, 8, False, "dense"),
    (2, 2100, 2, 1, 32, 1, 12, False, "dense"),
]


@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("positions", [None, "shared", "far", "far64"])
@pytest.mark.parametrize("case", ROTARY, ids=lambda c: "-".join(map(str, c)).replace(" ", "_"))
def test_qk_norm_rotary(cuda0, case, positions, dtype):
    """Bounds.  Forward: the sum of squares, the root, the product with weight and root, the rotation are some D / 2 + 16
    roundings in fp32 of numbers no larger than the pair's |u1| + |u2| (angles: below 2^-22 of a turn, 2^-19 radians
    is taken), then one rounding to the type.  Backward likewise on |du| and on r (|dn| + |n| mean|dn n|)."""
    K = _K()
    B, L, Hq, Hkv, D, axes, pairs, inter, layout = case
    gen = torch.Generator().manual_seed(D * 7 + L)
    x = {"q": torch.randn(B, L, Hq, D, generator=gen).to(dtype), "k": (3 * torch.randn(B, L, Hkv, D, generator=gen)).to(dtype)}
    g = {n: torch.randn(t.shape, generator=gen).to(dtype) for n, t in x.items()}
    w = {n: torch.randn(D, generator=gen) for n in x}
    freqs = torch.rand(axes, pairs, generator=gen) + 1e-3
    pos = None
    if positions == "shared":
        pos = torch.randint(0, 5000, (L, axes), generator=gen, dtype=torch.int32)
    elif positions:
        hi = 2 ** 31 - 1 if positions == "far" else 2 ** 28
        pos = torch.randint(-hi if positions == "far64" else 0, hi, (B, L, axes), generator=gen, dtype=torch.int64)
        hi_ok = 2 ** 28  # the stated accuracy of the reduction: positions times frequencies up to 2^28 turns
        pos = (pos % hi_ok).to(torch.int32) if positions == "far" else pos
    pd = torch.arange(L).view(1, L, 1).expand(1, L, axes) if pos is None else pos.view(-1, L, axes)
    angles = (pd.double().unsqueeze(-1) * freqs.double()).flatten(-2)
    eps = 1e-6
    kw = dict(eps=eps, interleaved=inter)
    if pairs:
        flat = axes == 1 and positions != "shared"
        kw["freqs"] = (freqs[0] if flat else freqs).to(cuda0)
        kw["positions"] = None if pos is None else (pos.squeeze(-1) if flat else pos).to(cuda0)
    leaves = {n: _layout(t, layout, cuda0).requires_grad_() for n, t in x.items()}
    ws = {n: t.to(cuda0).requires_grad_() for n, t in w.items()}
    got = dict(zip("qk", K.qk_norm_rotary(leaves["q"], leaves["k"], ws["q"], ws["k"], **kw)))
    order = [leaves["q"], leaves["k"], ws["q"], ws["k"]]
    grads = torch.autograd.grad([got["q"], got["k"]], order, [_layout(g[n], layout, cuda0) for n in "qk"])
    uo, f = S.unit(dtype), (D / 2 + 16) * S.F + 2.0 ** -19
    for i, n in enumerate("qk"):
        a, b = x[n].double().requires_grad_(), w[n].double().requires_grad_()
        y = S.rotary(a, b, angles, axes * pairs, eps, inter)
        da, db = torch.autograd.grad(y, (a, b), g[n].double())
        r = 1 / torch.sqrt((a * a).mean(-1, keepdim=True) + eps)
        u = (a * r * b).detach().abs()
        # a pair's size on both of its columns: rotating the sizes by 45 degrees' worth of both bounds each
        both = u + u.amax(-1, keepdim=True)
        _within(n, got[n], y.detach(), uo * y.detach().abs() + f * both)
        nrm = (a * r).detach().abs()
        gg = g[n].double().abs()
        du = gg + gg.amax(-1, keepdim=True)
        dn = du * b.detach().abs()
        _within("d" + n, grads[i], da, uo * da.abs() + f * r.detach() * (dn + nrm * (dn * nrm).mean(-1, keepdim=True)))
        rows = B * L * x[n].shape[2]
        _within("dw" + n, grads[2 + i], db, ((f + (rows ** 0.5 + 64) * S.F) * (du * nrm)).sum((0, 1, 2)))
    with torch.no_grad():
        again = K.qk_norm_rotary(*[t.detach() for t in order], **kw)
    assert torch.equal(again[0], got["q"]) and torch.equal(again[1], got["k"])


# ----------------------------------------------------------------------------------------------
# the operators together: sequence.BandedMSA
# ----------------------------------------------------------------------------------------------
def test_qk_norm_rotary_captured_and_replayed(cuda0):
    """a training pass in a graph, with new inputs and eager work between the replays, against the eager result"""
    K = _K()
    gen = torch.Generator(device=cuda0).manual_seed(9)
    st = {"q": torch.randn(3, 700, 6, 30, device=cuda0, generator=gen).to(BF), "k": torch.randn(3, 700, 2, 30, device=cuda0, generator=gen).to(BF),
          "wq": torch.randn(30, device=cuda0, generator=gen), "wk": torch.randn(30, device=cuda0, generator=gen)}
    freqs, pos = torch.rand(2, 7, device=cuda0, generator=gen), torch.randint(0, 64, (700, 2), device=cuda0, generator=gen)

    def work():
        leaves = [t.detach().requires_grad_() for t in st.values()]
        out = K.qk_norm_rotary(*leaves, freqs, pos)
        return [t.detach() for t in out] + list(torch.autograd.grad(out, leaves, (st["q"], st["k"])))

    side = torch.cuda.Stream(cuda0)
    side.wait_stream(torch.cuda.current_stream(cuda0))
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream(cuda0).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = work()
    for n in range(4):
        for t in st.values():
            t.copy_(torch.randn(t.shape, device=cuda0, generator=gen))
        pos.add_(17 * n)
        graph.replay()
        got = [t.clone() for t in held]
        for x, y in zip(got, work()):
            assert torch.equal(x, y)
        torch.cuda.synchronize()


def _module_in_64_bits(mod, x, positions, lens=None):
    """BandedMSA by plain tensor operations in the dtype of its (double) parameters"""
    B, L, C = x.shape
    h, g, d = mod.num_heads, mod.kv_heads, mod.head_dim
    qkv = torch.nn.functional.linear(x, mod.qkv.weight, mod.qkv.bias).unflatten(-1, (h + 2 * g, d))
    q, k, v = qkv.split((h, g, g), dim=2)
    f = mod.rotary_freqs.double()
    ang = (positions.double().view(-1, L, f.shape[0], 1) * f).flatten(-2)
    q, k = (S.rotary(t, w, ang, f.numel(), mod.eps, False) for t, w in ((q, mod.q_norm), (k, mod.k_norm)))
    rep = h // g
    k, v = k.repeat_interleave(rep, 2), v.repeat_interleave(rep, 2)
    s = torch.einsum("bihd,bjhd->bhij", q, k) * d ** -0.5
    if mod.pe is not None:
        M = mod.pe.max_distance
        rel = (torch.arange(L)[None, :] - torch.arange(L)[:, None]).clamp(-M, M) + M
        s = s + mod.pe.table()[mod.pe.buckets.long()[rel]].permute(2, 0, 1)
    vis = torch.stack([S.visible(L, L, n, n, mod.window[0], mod.window[1], mod.sinks)[0] for n in (lens or [L] * B)])[:, None]
    s = s.masked_fill(~vis, -math.inf)
    p = torch.where(vis, torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300)), 0.0)
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
    z = torch.einsum("bhij,bjhd->bihd", p, v).reshape(B, L, C)
    return torch.nn.functional.linear(z, mod.out_proj.weight, mod.out_proj.bias)


def _module(**kw):
    from visiontransformer_amd.sequence import BandedMSA
    torch.manual_seed(3)
    mod = BandedMSA(**kw)
    with torch.no_grad():
        for p in mod.parameters():
            p.add_(torch.randn_like(p) * 0.1)
    return mod


@pytest.mark.parametrize("kw,L,lens", [
    (dict(dim=180, num_heads=6, window=(40, 40), sinks=4, rotary_axes=2, num_buckets=16, max_distance=32), 144, None),
    (dict(dim=128, num_heads=4, kv_heads=2, window=(60, 0), sinks=2, num_buckets=8, max_distance=64), 130, [130, 17]),
    (dict(dim=64, num_heads=4, rotary_pairs=5), 70, [70, 0]),
])
def test_banded_msa_trains(cuda0, kw, L, lens):
    """fp32: output and every gradient against double.  Both Linears are fp32 sums of dim products, the attention's bounds are
    a few dozen roundings: 2^-24 * (2 dim + 400) of each tensor's norm is taken, some twenty times what errors of random
    sign add up to."""
    import copy
    mod = _module(**kw)
    ref = copy.deepcopy(mod).double()
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(2, L, kw["dim"], generator=gen)
    g = torch.randn(2, L, kw["dim"], generator=gen)
    axes = mod.rotary_axes
    pos = torch.stack([torch.arange(L) // 12, torch.arange(L) % 12], -1) if axes == 2 else torch.arange(L)[:, None]
    xd = x.double().requires_grad_()
    yd = _module_in_64_bits(ref, xd, pos[None], lens)
    want = torch.autograd.grad(yd, [xd] + list(ref.parameters()), g.double())
    mod = mod.to(cuda0)
    xg = x.to(cuda0).requires_grad_()
    y = mod(xg, positions=pos.to(cuda0) if axes == 2 else None, lens=None if lens is None else torch.tensor(lens, device=cuda0))
    got = torch.autograd.grad(y, [xg] + list(mod.parameters()), g.to(cuda0))
    tol = 2.0 ** -24 * (2 * kw["dim"] + 400)
    names = ["x"] + [n for n, _ in mod.named_parameters()]
    for name, a, b in [("y", y, yd)] + list(zip(names, got, want)):
        err = float((a.detach().double().cpu() - b.detach()).norm() / b.detach().norm().clamp(min=1e-30))
        assert err <= tol, (name, err, tol)


@pytest.mark.parametrize("dtype", [FP, BF])
def test_new_tokens_behind_a_cache_equal_the_whole_sequence(cuda0, dtype):
    """a padded prompt, then tokens one by one (and three at once), against the module on the whole sequences.  fp32: both
    ways compute the same sums in other orders; bf16: they differ by roundings of intermediates of 2^-8 each (projection,
    norm, probabilities, result, projection)."""
    from visiontransformer_amd.sequence import KVCache
    mod = _module(dim=128, num_heads=4, kv_heads=2, window=(20, 0), sinks=2, num_buckets=8, max_distance=64).to(cuda0).to(dtype).eval()
    assert mod.rotary_freqs.dtype == torch.float32
    gen = torch.Generator().manual_seed(2)
    lens, extra = [37, 50], 9
    x = torch.randn(2, 50 + extra, 128, generator=gen).to(dtype).to(cuda0)
    with torch.no_grad():
        cache = KVCache(2, 70, 2, 32, dtype=dtype, device=cuda0)
        cache.k.fill_(float("nan"))
        cache.v.fill_(float("nan"))
        first = mod(x[:, :50], lens=torch.tensor(lens, device=cuda0), cache=cache)
        assert cache.lens.tolist() == lens
        steps, at = [], 0
        for n in (1, 1, 3, 1, 3):
            new = torch.stack([x[b, lens[b] + at:lens[b] + at + n] for b in range(2)])
            steps.append(mod(new, cache=cache))
            at += n
        steps = torch.cat(steps, 1)
        tol = 2e-5 if dtype == FP else 5 * 2.0 ** -8
        for b in range(2):
            whole = mod(x[b:b + 1, :lens[b] + extra])[0]
            for got, want in ((first[b, :lens[b]], whole[:lens[b]]), (steps[b], whole[lens[b]:])):
                err = float((got.double() - want.double()).norm() / want.double().norm())
                assert err <= tol, (b, err)
        with pytest.raises(RuntimeError, match="capacity"):
            mod(x[:, :20], cache=cache)
    with pytest.raises(RuntimeError, match="inference"):
        mod(x[:, :1], cache=KVCache(2, 4, 2, 32, dtype=dtype, device=cuda0))


def test_banded_msa_under_autocast(cuda0):
    """fp32 parameters, bf16 autocast, a training step: finite, close to fp32 (2e-2, the bar of the package's bf16 runs)"""
    mod = _module(dim=180, num_heads=6, window=(64, 64), sinks=4, num_buckets=16, max_distance=32).to(cuda0)
    x = torch.randn(2, 200, 180, generator=torch.Generator().manual_seed(4)).to(cuda0).requires_grad_()
    g = torch.randn(2, 200, 180, generator=torch.Generator().manual_seed(5)).to(cuda0)
    outs = []
    for on in (False, True):
        with torch.autocast("cuda", dtype=BF, enabled=on):
            y = mod(x)
        outs.append([y] + list(torch.autograd.grad(y, [x] + list(mod.parameters()), g.to(y.dtype))))
    for a, b in zip(*outs):
        assert float((a.double() - b.double()).norm() / a.double().norm()) <= 2e-2
