"""The arrays of a paged cache are those that its tensor maps were made for (no GPU needed)."""
import pytest
import torch

from yasakani_b200 import paged


@pytest.mark.parametrize("name", ["k", "v", "kmean"])
def test_the_arrays_of_a_cache_cannot_be_exchanged(name):
    """Another tensor under the same name would leave every call with the old one's addresses, whose memory may belong to someone else by then."""
    cache = paged.PagedCache.__new__(paged.PagedCache)
    with pytest.raises(AttributeError):
        setattr(cache, name, torch.zeros(1))


@pytest.mark.gpu
def test_the_arrays_can_be_read_and_written():
    k = torch.zeros((3, 2, 32, 128), dtype=torch.float16, device="cuda")
    cache = paged.PagedCache.of(k, k.clone(), k[:, :, 0].clone())
    cache.k[1] = 1.0
    cache.v.copy_(cache.k)
    assert cache.k is k and (k[1] == 1).all() and torch.equal(cache.v, k) and cache.kmean.shape == (3, 2, 128) and cache.nbytes() == 2 * k.nbytes + 3 * 2 * 128 * 2
    assert paged.PagedCache.of(k, cache.v).kmean is None
