"""Paged attention where each token can be told from its neighbours: a token that is lost, read twice or taken from another place shows, however long the row is."""
import pytest
import torch

from test_gpu_paged import DT, attend, ints

pytestmark = pytest.mark.gpu


def spots(n, shared, page):
    """Borders of tiles (64, 128 tokens), of pages and of the shared part, ends, and some in between."""
    at = {0, 1, n - 1, n - 2, n // 2, n // 3, 2 * n // 3}
    for step in (16, 64, 128, page, 1024):
        for i in (1, 2, 3, n // (2 * step), n // step - 1, n // step):
            at |= {step * i - 1, step * i}
    at |= {shared - 1, shared, shared + 1, shared + 63, shared + 64}
    return sorted(a for a in at if 0 <= a < n)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("nh,hkv,hd,page,n,shared", [
    (16, 2, 128, 64, 70001, 0), (6, 1, 256, 16, 33333, 0), (28, 4, 128, 32, 5300, 5216), (24, 4, 256, 64, 20000, 16384), (12, 1, 128, 128, 4097, 0), (24, 4, 256, 16, 2700, 2512)])
def test_each_token_counts_once(dt, nh, hkv, hd, page, n, shared):
    """Keys are zero, so every token weighs 1 / n; values are zero but for one token a row of the call, whose sequence names pages of its own there.  What comes
    out is that token's value / n, rounded twice at most (the weight is a power of two times the others' and exact): a lost token gives zero, one read twice the double."""
    g = torch.Generator(device="cuda").manual_seed(n)
    at, blocks = spots(n, shared, page), -(-n // page)
    own = [a for a in at if a >= shared]
    pages = blocks + len(own) + 1
    k = torch.zeros((pages, hkv, page, hd), dtype=DT[dt], device="cuda")
    v = torch.zeros_like(k)
    table = torch.arange(blocks, dtype=torch.int32, device="cuda").repeat(len(own) + 1, 1)
    mark = (torch.rand((len(own) + 1, hkv, hd), generator=g, device="cuda") + 1.0).to(DT[dt]) * (2 ** 12)
    for i, a in enumerate(own):                                  # a page with the token alone, in place of the common one
        table[i, a // page] = blocks + i
        v[blocks + i, :, a % page] = mark[i]
    seq = torch.arange(len(own) + 1, dtype=torch.int32, device="cuda")
    q = torch.randn((len(own) + 1, nh, hd), generator=g, device="cuda").to(DT[dt])
    h = torch.finfo(DT[dt]).eps / 2

    def check(o16, want):
        tol = (2 * h + n * 2.0 ** -23) * want + 2.0 ** -24       # sums of n equal weights in fp32; a weight, the row; the smallest fp16 numbers
        assert ((o16.double() - want).abs() <= tol).all(), float(((o16.double() - want).abs() / tol).max())

    o16, _ = attend(k, v, table, seq, ints([n - 1] * len(seq)), q, 1.0, shared=shared)
    want = (mark.double() / n).repeat_interleave(nh // hkv, 1)
    want[-1] = 0.0                                               # a row without any
    check(o16, want)
    for i, a in enumerate(own):                                  # each by itself too: its line is cut elsewhere
        if i % 4 == 0:
            o16, _ = attend(k, v, table, ints([i]), ints([n - 1]), q[i:i + 1], 1.0, shared=shared)
            check(o16, want[i:i + 1])
    for a in (a for a in at if a < shared):                      # in the shared part: for all rows
        v.zero_()
        v[a // page, :, a % page] = mark[0]
        o16, _ = attend(k, v, table, seq, ints([n - 1] * len(seq)), q, 1.0, shared=shared)
        check(o16, (mark[:1].double() / n).repeat_interleave(nh // hkv, 1).expand(o16.shape))


def test_a_pool_of_more_than_2_31_elements():
    """Pages whose elements lie beyond 31 and 32 bits: append, mean keys, choice and both attentions there give the bits that they give in a small pool."""
    from yasakani_b200 import paged
    hkv, nh, hd, page, n, shared = 4, 24, 256, 64, 700, 256
    per = hkv * page * hd
    pages = (1 << 32) // per + 40                                # 8.6 GB each for keys and values
    g = torch.Generator(device="cuda").manual_seed(7)
    high = [pages - 1, (1 << 32) // per, (1 << 31) // per, (1 << 31) // per - 1, (1 << 32) // per - 1, pages - 2, pages - 7, 0, pages - 3, pages - 11, pages - 20]
    x = torch.randn((n, nh + 2 * hkv, hd), generator=g, device="cuda").bfloat16()
    rope = torch.randn((n, 32, 2), generator=g, device="cuda")
    outs = []
    for names, size in ((list(range(11)), 11), (high, pages)):
        cache = paged.PagedCache(size, hkv, hd, page=page, dtype=torch.bfloat16, means=True)
        table = ints([names])
        seq, pos = ints([0] * n), torch.arange(n, dtype=torch.int32, device="cuda")
        q = torch.empty((n, nh, hd), dtype=torch.bfloat16, device="cuda")
        paged.launch_append(cache, table, x[:, nh:nh + hkv], x[:, nh + hkv:], seq, pos, rope, 64, q=x[:, :nh], q_out=q)
        ws = paged.workspace(cache, 2, nh, 11, shared=shared, select=True)
        two, seq, pos = q[-2:].contiguous(), ints([0, 0]), ints([n - 2, n - 1])
        ids = torch.empty((2, hkv, 5), dtype=torch.int32, device="cuda")
        paged.launch_select(two, cache, table, seq, pos, ids, ws)
        o = [torch.empty_like(two) for _ in range(3)]
        paged.launch_attention(two, cache, table, seq, pos, hd ** -0.5, o[0], ws)
        paged.launch_attention(two, cache, table, seq, pos, hd ** -0.5, o[1], ws, blocks=ids)
        paged.launch_attention(two, cache, table, seq, pos, hd ** -0.5, o[2], ws, shared=shared)
        at = torch.tensor(names, device="cuda")
        outs.append([q, ids, *o, cache.k[at], cache.v[at], cache.kmean[at]])
        if size == pages:                                        # nothing else was written: the sum of all bits is that of these pages
            for t in (cache.k, cache.v):
                rest = torch.ones(pages, dtype=torch.bool, device="cuda")
                rest[at] = False
                assert not any(bool(t[i:i + 4096][rest[i:i + 4096]].any()) for i in range(0, pages, 4096))
        del cache
    assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) if a.dtype == torch.bfloat16 else torch.equal(a, b) for a, b in zip(*outs))
    assert (outs[0][2] != 0).any() and (outs[0][3] != outs[0][2]).any()
