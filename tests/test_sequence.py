"""Attention over token sequences, what needs no GPU: bucket maps, refusals of the C entry points, argument checks."""
import ctypes

import pytest
import torch

from oracle import sequence_oracle as S


@pytest.mark.parametrize("buckets,distance,causal", [(32, 128, False), (32, 128, True), (8, 64, False), (64, 300, True), (4, 2, False), (16, 512, False)])
def test_bucket_map(buckets, distance, causal):
    from visiontransformer_amd.sequence import bucket_of_distance
    got = bucket_of_distance(buckets, distance, not causal).tolist()
    assert len(got) == 2 * distance + 1
    assert got == S.bucket_map(buckets, distance, causal)
    side = buckets if causal else buckets // 2
    behind = got[:distance + 1][::-1]
    assert behind[0] == 0 and behind[-1] == side - 1
    assert all(0 <= b - a <= side for a, b in zip(behind, behind[1:]))       # never falls
    assert behind[:side // 2] == list(range(side // 2))                          # one by one nearby
    if causal:
        assert set(got[distance + 1:]) == {0}
    else:
        assert got[distance + 1:] == [b + side for b in behind[1:]]


def test_bucket_map_refusals():
    from visiontransformer_amd.sequence import bucket_of_distance
    for args in ((1, 64, False), (3, 64, True), (32, 8, True), (2, 64, True)):
        with pytest.raises(ValueError):
            bucket_of_distance(*args)


def test_expanded_bias():
    from visiontransformer_amd.sequence import BucketedPositionBias
    pe = BucketedPositionBias(3, 8, 16, bidirectional=True)
    full = pe(5, 9)
    assert full.shape == (1, 3, 5, 9)
    for i in range(5):
        for j in range(9):
            rel = max(-16, min(16, j - (4 + i)))
            assert torch.equal(full[0, :, i, j], pe.table()[int(pe.buckets[rel + 16])])


def _desc(**kw):
    from visiontransformer_amd._lib import BandDesc
    d = dict(dtype=1, B=1, Lq=4, Lk=8, Hq=4, Hkv=2, D=32, left=-1, right=0, sinks=0, scale=0.1)
    d.update(kw)
    return ctypes.byref(BandDesc(**d))


def test_refusals_of_the_c_entries():
    """before any HIP call: descriptions, null pointers, workspaces"""
    from visiontransformer_amd import _lib
    lib = _lib.load()
    buf = (ctypes.c_float * 64)()
    p = ctypes.cast(buf, ctypes.c_void_p)
    s = ctypes.byref(_lib.Strides(1, 1, 1))

    def fwd(desc, q=p, ws=None, n=0, so=s, lse=None, o32=None):
        return lib.dsw_band_attn_fwd(desc, q, s, p, s, p, s, p, so, lse, o32, ws, n, None), lib.dswin_last_error_string()

    for kw, code, text in [
        (dict(dtype=2), 2, b"dtype"), (dict(B=-1), 1, b"negative"), (dict(D=0), 2, b"head dim 0"), (dict(D=129), 2, b"head dim 129"),
        (dict(Hq=3), 1, b"3 query heads"), (dict(Hkv=0), 1, b"0 key heads"), (dict(left=-2), 1, b"window"), (dict(sinks=-1), 1, b"sinks"),
        (dict(scale=0.0), 1, b"scale"), (dict(scale=float("nan")), 1, b"scale"), (dict(scale=float("inf")), 1, b"scale"),
        (dict(Lk=(1 << 29) + 1), 2, b"tokens"), (dict(B=1 << 20, Lq=1 << 20), 2, b"row blocks"),
        (dict(bias_table=p), 1, b"bucket map"), (dict(bias_table=p, bias_buckets=p, n_buckets=4, max_distance=513), 2, b"distances"),
        (dict(bias_table=p, bias_buckets=p, n_buckets=0, max_distance=8), 1, b"bucket map"),
        (dict(bias_table=p, bias_buckets=p, n_buckets=4, max_distance=0), 2, b"distances"),
    ]:
        rc, msg = fwd(_desc(**kw))
        assert rc == code and text in msg, (kw, rc, msg)
        if "B" not in kw or kw["B"] >= 0:
            assert lib.dsw_band_attn_fwd_workspace(_desc(**kw)) == 0 and lib.dsw_band_attn_bwd_workspace(_desc(**kw)) == 0
    rc, msg = fwd(None)
    assert rc == 1 and b"null description" in msg
    rc, msg = fwd(_desc(), q=None)
    assert rc == 1 and b"null q" in msg
    rc, msg = fwd(_desc(), so=None)
    assert rc == 1 and b"null out" in msg
    rc, msg = fwd(_desc(), so=ctypes.byref(_lib.Strides(1, -1, 1)))
    assert rc == 1 and b"negative stride" in msg
    rc, msg = fwd(_desc(), o32=p)
    assert rc == 1 and b"out32" in msg
    long = _desc(Lq=1, Lk=100000)
    need = lib.dsw_band_attn_fwd_workspace(long)
    assert need > 0
    rc, msg = fwd(long, ws=p, n=need - 1)
    assert rc == 1 and b"workspace" in msg
    rc, msg = fwd(long, ws=None, n=need)
    assert rc == 1 and b"workspace" in msg
    assert fwd(_desc(B=0))[0] == 0 and fwd(_desc(Lq=0))[0] == 0        # nothing to do

    def bwd(desc, lse=p, table=None, ws=p, n=1 << 40):
        return (lib.dsw_band_attn_bwd(desc, p, s, p, s, p, s, p, s, None, p, s, lse, p, s, p, s, p, s, table, ws, n, None),
                lib.dswin_last_error_string())

    rc, msg = bwd(_desc(), lse=None)
    assert rc == 1 and b"null lse" in msg
    rc, msg = bwd(_desc(), table=p)
    assert rc == 1 and b"table" in msg
    rc, msg = bwd(_desc(), n=lib.dsw_band_attn_bwd_workspace(_desc()) - 1)
    assert rc == 1 and b"workspace" in msg
    assert bwd(_desc(B=0))[0] == 0

    def rot(dtype=1, B=1, L=4, Hq=2, Hkv=1, D=32, axes=1, pairs=8, freqs=p, q=p, st=s, pos=None, pos_bytes=0):
        return (lib.dsw_qk_norm_rotary_fwd(q, st, p, s, dtype, B, L, Hq, Hkv, D, None, None, 1e-6, freqs, axes, pairs, pos, pos_bytes, 0, 0, p, s, p, s, None),
                lib.dswin_last_error_string())

    for kw, code, text in [
        (dict(dtype=3), 2, b"dtype"), (dict(L=-1), 1, b"negative"), (dict(D=129), 2, b"head dim"), (dict(D=0), 2, b"head dim"),
        (dict(pairs=17), 1, b"need more"), (dict(axes=1 << 20, pairs=1 << 20), 1, b"need more"), (dict(freqs=None), 1, b"null freqs"),
        (dict(q=None), 1, b"null pointer"), (dict(st=None), 1, b"null strides"), (dict(B=1 << 20, L=1 << 20), 2, b"tokens"),
        (dict(Hq=4096), 2, b"heads"), (dict(pos=p, pos_bytes=2), 1, b"positions of 2 bytes"),
    ]:
        rc, msg = rot(**kw)
        assert rc == code and text in msg, (kw, rc, msg)
    assert rot(B=0)[0] == 0 and rot(Hq=0, Hkv=0)[0] == 0
    assert lib.dsw_qk_norm_rotary_blocks(1, -1, 4, 1, 1, 8, 1, 1) == 0 and lib.dsw_qk_norm_rotary_blocks(1, 2, 4, 1, 1, 8, 1, 1) == 8


def test_cpu_tensors_are_refused():
    from visiontransformer_amd import functional as K
    z = torch.zeros(1, 4, 2, 8)
    with pytest.raises(RuntimeError, match="GPU only"):
        K.band_attention(z, z, z)
    with pytest.raises(RuntimeError, match="GPU only"):
        K.qk_norm_rotary(z, z)


def test_cache_refusals_on_the_cpu():
    from visiontransformer_amd.sequence import KVCache
    c = KVCache(2, 4, 1, 8, dtype=torch.float32, device="cpu")
    z = torch.zeros(2, 3, 1, 8)
    c.append(z + 1, z + 2, torch.tensor([3, 1]))
    assert c.lens.tolist() == [3, 1]
    c.append(z[:, :1] + 5, z[:, :1] + 6)
    k, v = c.tokens()
    assert c.lens.tolist() == [4, 2] and float(k[0, 3, 0, 0]) == 5 and float(k[1, 1, 0, 0]) == 5 and float(v[1, 0, 0, 0]) == 2
    with pytest.raises(RuntimeError, match="capacity"):
        c.append(z[:, :1], z[:, :1])
    with pytest.raises(RuntimeError, match="KVCache"):
        c.append(z[:1, :1], z[:1, :1])
    with pytest.raises(RuntimeError, match="KVCache"):
        c.append(z[:, :0].half(), z[:, :0].half())


def test_cache_counts_and_refusals():
    from visiontransformer_amd.sequence import KVCache
    cache = KVCache(2, 8, 3, 4, dtype=torch.float32, device="cpu")
    k, v = torch.randn(2, 5, 3, 4), torch.randn(2, 5, 3, 4)
    cache.append(k, v, torch.tensor([2, 2 ** 33], dtype=torch.int64))       # (clamped to the batch's 5, not wrapped)
    assert cache.lens.tolist() == [2, 5] and cache.longest == 5
    cache.append(k[:, :3], v[:, :3])
    assert cache.lens.tolist() == [5, 8]
    assert torch.equal(cache.tokens()[0][0, :5], torch.cat([k[0, :2], k[0, :3]])) and torch.equal(cache.tokens()[1][1], torch.cat([v[1], v[1, :3]]))
    fresh = KVCache(2, 8, 3, 4, dtype=torch.float32, device="cpu")
    for args in ((k.requires_grad_(), v), (k.detach(), v, torch.tensor([1])), (k.detach().double(), v), (k.detach()[:1], v)):
        with pytest.raises(RuntimeError, match="KVCache"):
            fresh.append(*args)
    with pytest.raises(RuntimeError, match="capacity"):
        cache.append(k.detach()[:, :1], v[:, :1])
    with torch.no_grad():
        fresh.append(k, v)
    assert fresh.lens.tolist() == [5, 5] and not fresh.k.requires_grad
