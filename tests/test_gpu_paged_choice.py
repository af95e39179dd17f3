"""Choices whose scores are exact in fp64 in any order of summation: products that are whole numbers within a factor of 2^23 (fp16) or 2^29 (bf16) of one another, large ones
that cancel among them, and so few different scores that the border runs through many equal ones."""
import pytest
import torch

from test_gpu_paged import DT, choose, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt,big", [("f16", 2.0 ** 11), ("f16", 2.0 ** 13), ("bf16", 2.0 ** 11), ("bf16", 2.0 ** 21)])
@pytest.mark.parametrize("nh,hkv,hd", [(6, 2, 128), (16, 1, 256), (8, 8, 256)])
@pytest.mark.parametrize("blocks,take", [(300, 40), (5000, 100)])
def test_whole_numbers_and_large_ones_that_cancel(dt, big, nh, hkv, hd, blocks, take):
    from yasakani_b200 import paged
    g = torch.Generator(device="cuda").manual_seed(blocks + hd)
    whole = lambda *shape: torch.randint(-3, 4, shape, generator=g, device="cuda").float()
    km, q = whole(blocks, hkv, hd) * (torch.rand((blocks, hkv, hd), generator=g, device="cuda") < 0.05), whole(2, nh, hd)
    where = torch.randperm(hd, generator=g, device="cuda")[:hd // 4]                        # pairs of channels far apart in the order of summation
    a, b = where[:hd // 8], where[hd // 8:]
    q[..., b] = q[..., a]
    km[..., a] = big * whole(blocks, hkv, hd // 8)
    km[..., b] = -km[..., a]
    km, q = km.to(DT[dt]).contiguous(), q.to(DT[dt])
    prod = (q.double()[:, :, None].abs() @ km.double().abs().amax((0, 1))[:, None]).amax()
    assert float(prod) < 2.0 ** 53 and 9 * big <= 2.0 ** (23 if dt == "f16" else 29)        # exact: every partial sum is a whole number below 2^53
    k = torch.zeros((blocks, hkv, 16, hd), dtype=DT[dt], device="cuda")
    table = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)[None].contiguous()
    ids = torch.empty((2, hkv, take), dtype=torch.int32, device="cuda")
    cache, seq, pos = paged.PagedCache.of(k, k, km), ints([0, 0]), ints([blocks * 16 - 1, blocks * 8])
    paged.launch_select(q, cache, table, seq, pos, ids, paged.workspace(cache, 2, nh, blocks, select=True))
    assert torch.equal(ids.cpu(), choose(q, km, table, seq, pos, 16, take))
