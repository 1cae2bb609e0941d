"""sequence.KVCache on the CPU: what a refused call leaves behind."""
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
