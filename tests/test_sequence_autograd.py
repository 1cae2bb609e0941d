"""The token-sequence operators under autograd, what needs no GPU: the library's calls are recorded instead of launched."""
import pytest
import torch
from torch.autograd import forward_ad


@pytest.fixture
def calls(monkeypatch):
    """functional with CPU tensors and recorded library calls (name, arguments)"""
    from visiontransformer_amd import _lib, functional as K
    made = []
    monkeypatch.setattr(_lib, "require_cuda", lambda *tensors: None)
    monkeypatch.setattr(K, "stream", lambda device=None: 0)
    monkeypatch.setattr(K, "_call_on", lambda device, name, *args: made.append((name, args)))
    return made


def _attention(*args, **kw):
    from visiontransformer_amd import functional as K
    return K.band_attention(*args, **kw)


def _rotary(*args, **kw):
    from visiontransformer_amd import functional as K
    return K.qk_norm_rotary(*args, **kw)[0]


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("which", [0, 1, 2])
def test_forward_mode_derivatives_are_refused(calls, grad, which):
    """a dual input, with gradients enabled and without: an error, not a result without its tangent"""
    x = torch.randn(1, 4, 2, 8)
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        args = [x.clone(), x.clone(), x.clone()]
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(x))
        with pytest.raises(NotImplementedError):
            _attention(*args)
        if which < 2:
            with pytest.raises(NotImplementedError):
                _rotary(*args[:2])
        weight = forward_ad.make_dual(torch.ones(8), torch.ones(8))
        with pytest.raises(NotImplementedError):
            _rotary(x, x, weight)
        assert _attention(x, x, x).shape == _rotary(x, x).shape == x.shape      # (no dual input: an ordinary call)


def test_calls_without_gradients_save_nothing(calls):
    x = torch.randn(1, 4, 2, 8)
    for out in (_attention(x, x, x), _rotary(x, x)):
        assert out.grad_fn is None
    y = x.clone().requires_grad_()
    with torch.no_grad():
        for out in (_attention(y, x, x), _rotary(y, x)):
            assert not out.requires_grad
    for out in (_attention(y, x, x), _rotary(y, x)):
        assert out.grad_fn is not None


def test_copies_of_saved_tensors_live_until_the_launch(calls, monkeypatch):
    """a hook that returns saved tensors with a strided last dimension: the dense copies that the kernels read are alive when
    they are launched"""
    import weakref
    from visiontransformer_amd import functional as K
    given = []
    rows = K._head_rows

    def head_rows(t):
        r = rows(t)
        given.append((weakref.ref(r[0]), r[2]))
        return r

    def launch(device, name, *args):
        calls.append(name)
        if name.endswith("_bwd"):
            for alive, address in given:
                assert alive() is not None and alive().data_ptr() == address, name

    def strided(t):
        if t.dim() != 4 or t.shape[-1] != 8:      # (rows of heads only)
            return t
        return t.transpose(2, 3).contiguous().transpose(2, 3)

    monkeypatch.setattr(K, "_head_rows", head_rows)
    monkeypatch.setattr(K, "_call_on", launch)
    for run in (lambda a, b, c: _attention(a, b, c), lambda a, b, c: _rotary(a, b)):
        leaves = [torch.randn(1, 4, 2, 8, requires_grad=True) for _ in range(3)]
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, strided):
            out = run(*leaves)
        given.clear()
        out.sum().backward()
    assert [n for n in calls if n.endswith("_bwd")] == ["dsw_band_attn_bwd", "dsw_qk_norm_rotary_bwd"]


@pytest.mark.parametrize("shape,launched", [((1, 4, 5, 0, 2), True), ((1, 4, 5, 0, 0), False), ((1, 0, 5, 2, 1), True), ((1, 4, 0, 2, 1), True),
                                            ((0, 4, 5, 2, 1), False), ((1, 0, 0, 2, 1), False)])
def test_backward_is_launched_wherever_there_is_a_gradient_to_write(calls, shape, launched):
    """also without query heads: the gradients of k and v are zeros then, which the library writes"""
    B, Lq, Lk, Hq, Hkv = shape
    leaves = [torch.randn(B, n, h, 8, requires_grad=True) for n, h in ((Lq, Hq), (Lk, Hkv), (Lk, Hkv))]
    _attention(*leaves).sum().backward()
    assert ("dsw_band_attn_bwd" in [n for n, _ in calls]) == launched


def test_sizes_of_calls_without_query_heads():
    """the C entries count workspaces of such a call as of any other"""
    import ctypes
    from visiontransformer_amd import _lib
    for sinks in (0, 3):
        d = _lib.BandDesc(dtype=1, B=1, Lq=4, Lk=8, Hq=0, Hkv=2, D=32, left=-1, right=0, sinks=sinks, scale=0.1)
        assert _lib.load().dsw_band_attn_bwd_workspace(ctypes.byref(d)) == _lib.load().dsw_band_attn_fwd_workspace(ctypes.byref(d)) == 0


def test_workspace_of_a_backward_with_sinks():
    """Blocks of sinks are seen by every row; the shares of their runs must not outgrow the card's memory with the batch or the
    number of sinks.  Four runs for each resident workgroup (512 of them for narrow heads in 16 bits, else 256), rounded up
    block by block to twice as many at most; a share is 2 x 128 rows of fp32."""
    import ctypes
    from visiontransformer_amd import _lib

    def size(sinks, B=4, L=32768, H=16, D=128, left=256, dtype=1):
        d = _lib.BandDesc(dtype=dtype, B=B, Lq=L, Lk=L, Hq=H, Hkv=H, D=D, left=left, right=0, sinks=sinks, scale=0.1)
        return _lib.load().dsw_band_attn_bwd_workspace(ctypes.byref(d))

    for kw in ({}, dict(B=16), dict(B=1, H=1), dict(D=64, left=1024), dict(L=4096), dict(B=2, L=200000, H=8), dict(B=64, dtype=0)):
        for sinks in (1, 4, 128, 129, 1000, 4096, 20000):
            extra = size(sinks, **kw) - size(0, **kw)
            assert 0 <= extra <= 2 * 128 << 20, (kw, sinks, extra)
            assert sinks > 4 or extra <= 68 << 20, (kw, sinks, extra)


def test_refusals_of_what_the_rounding_leaves():
    """out_rest with fp32 tensors, in both directions, before anything is launched"""
    import ctypes
    from visiontransformer_amd import _lib
    lib = _lib.load()
    p, s = ctypes.cast((ctypes.c_float * 64)(), ctypes.c_void_p), ctypes.byref(_lib.Strides(1, 1, 1))
    d = _lib.BandDesc(dtype=0, B=1, Lq=4, Lk=8, Hq=4, Hkv=2, D=32, left=-1, right=0, sinks=0, scale=0.1, out_rest=p)
    assert lib.dsw_band_attn_fwd(ctypes.byref(d), p, s, p, s, p, s, p, s, p, None, p, 1 << 40, None) == 1
    assert b"out_rest" in lib.dswin_last_error_string()
    assert lib.dsw_band_attn_bwd(ctypes.byref(d), p, s, p, s, p, s, p, s, None, p, s, p, p, s, p, s, p, s, None, p, 1 << 40, None) == 1
    assert b"out_rest" in lib.dswin_last_error_string()


@pytest.mark.parametrize("dtype,wants,table,kept", [(torch.bfloat16, "q", False, True), (torch.bfloat16, "v", False, False), (torch.float32, "q", False, False),
                                                    (torch.bfloat16, "kt", True, False), (torch.bfloat16, "k", True, True)])
def test_what_the_rounding_leaves_is_kept_where_scores_want_gradients(calls, dtype, wants, table, kept):
    """(a table's gradient keeps the whole result in 32 bits instead)"""
    import ctypes
    ts = {n: torch.randn(1, 4, 2, 8).to(dtype).requires_grad_(n in wants) for n in "qkv"}
    tab = torch.randn(3, 2).requires_grad_("t" in wants) if table else None
    out = _attention(ts["q"], ts["k"], ts["v"], bias_table=tab, bias_buckets=torch.zeros(5, dtype=torch.int32) if table else None)
    out.sum().backward()
    from visiontransformer_amd._lib import BandDesc
    descs = [ctypes.cast(ctypes.pointer(args[0]._obj), ctypes.POINTER(BandDesc)).contents for _, args in calls]
    assert len(descs) == 2 and all(bool(d.out_rest) == kept for d in descs) and descs[0].out_rest == descs[1].out_rest


def test_bucket_numbers_are_clamped_before_they_are_narrowed(calls, monkeypatch):
    """int64 buckets beyond 32 bits: the table's ends, as for any other number outside it"""
    import ctypes
    from visiontransformer_amd import functional as K
    from visiontransformer_amd._lib import BandDesc
    seen = []

    def launch(device, name, desc, *args):
        d = ctypes.cast(ctypes.pointer(desc._obj), ctypes.POINTER(BandDesc)).contents
        seen.append(list((ctypes.c_int * 5).from_address(d.bias_buckets)))

    monkeypatch.setattr(K, "_call_on", launch)
    x = torch.zeros(1, 4, 2, 8)
    _attention(x, x, x, bias_table=torch.zeros(3, 2), bias_buckets=torch.tensor([2 ** 32, -2 ** 32 - 1, 1, 2 ** 33 + 1, -1]))
    assert seen == [[2, 0, 1, 2, 0]]
    _attention(x, x, x, bias_table=torch.zeros(3, 2), bias_buckets=torch.tensor([0, 1, 1, 2, 0], dtype=torch.int32))
    assert seen[1] == [0, 1, 1, 2, 0]


@pytest.mark.parametrize("dtype,table,kept", [(torch.float32, False, True), (torch.bfloat16, False, False), (torch.float32, True, False)])
def test_what_the_rounding_of_the_log_sum_exp_leaves_is_kept_in_fp32(calls, dtype, table, kept):
    """(with a bias it is in two parts anyway)"""
    import ctypes
    from visiontransformer_amd._lib import BandDesc
    x = torch.randn(2, 4, 3, 8).to(dtype).requires_grad_()
    kw = dict(bias_table=torch.zeros(3, 3), bias_buckets=torch.zeros(5, dtype=torch.int32)) if table else {}
    _attention(x, x, x, **kw).sum().backward()
    for name, args in calls:
        d = ctypes.cast(ctypes.pointer(args[0]._obj), ctypes.POINTER(BandDesc)).contents
        lse = args[9 if name.endswith("fwd") else 12]
        assert d.lse_rest == (lse + 4 * 2 * 3 * 4 if kept else None), name
