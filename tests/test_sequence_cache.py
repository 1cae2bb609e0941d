"""sequence.KVCache and sequence.BandedMSA on the CPU: calls that are refused, and what they leave behind."""
import pytest
import torch


@pytest.mark.parametrize("lens", [torch.tensor([1.5, 2.0]), torch.tensor([True, True]), torch.tensor([1, 2], dtype=torch.int16),
                                  torch.tensor([1, 2], device="meta")])
def test_counts_of_other_types_are_refused_before_anything_is_written(lens):
    """as band_attention refuses them, which a module calls behind the append: the cache must not have moved on by then"""
    from visiontransformer_amd.sequence import KVCache
    cache = KVCache(2, 8, 1, 4, dtype=torch.float32, device="cpu")
    cache.k.fill_(7.0)
    with pytest.raises(RuntimeError, match="KVCache: lens"):
        cache.append(torch.zeros(2, 3, 1, 4), torch.zeros(2, 3, 1, 4), lens)
    assert cache.lens.tolist() == [0, 0] and cache.longest == 0 and bool((cache.k == 7).all())


@pytest.mark.parametrize("kw", [dict(rotary_axes=0), dict(rotary_axes=0, qk_norm=False), dict(rotary_pairs=0)])
def test_positions_without_a_rotation_are_refused(kw):
    """with the norm alone they were dropped"""
    from visiontransformer_amd.sequence import BandedMSA
    with pytest.raises(RuntimeError, match="without rotation"):
        BandedMSA(64, **kw)(torch.zeros(1, 4, 64), positions=torch.arange(4))
