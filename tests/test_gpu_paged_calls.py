"""How the paged cache's operators are called: other streams, captured graphs whose rows change, calls behind one another on one workspace, tensors of
the wrong type, shape or device, a cache whose rows reach the end of its arrays."""
import pytest
import torch

from test_gpu_paged import DT, attend, check_rows, choose, ints, make_pool

pytestmark = pytest.mark.gpu


def case(dt="bf16", lengths=(300, 64, 1000, 1), nh=28, hkv=4, hd=128, page=32, seed=1, shared=0):
    k, v, table, g = make_pool(list(lengths), hkv, hd, page, DT[dt], seed=seed, shared=shared)
    kmean = torch.randn((k.shape[0], hkv, hd), generator=g, device="cuda").to(DT[dt])
    q = torch.randn((len(lengths), nh, hd), generator=g, device="cuda").to(DT[dt])
    return k, v, kmean, table, torch.arange(len(lengths), dtype=torch.int32, device="cuda"), ints(list(lengths)) - 1, q


@pytest.mark.parametrize("shared", [0, 640])
def test_another_stream_and_the_same_bits_twice(shared):
    from yasakani_b200 import paged
    k, v, kmean, table, seq, pos, q = case(lengths=[shared + n for n in (300, 64, 1000, 1)], shared=shared)
    cache = paged.PagedCache.of(k, v)
    outs = []
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for stream in (None, side, None):
        ws, o = paged.workspace(cache, 4, 28, table.shape[1], shared=shared), torch.empty_like(q)
        torch.cuda.synchronize()
        paged.launch_attention(q, cache, table, seq, pos, 0.09, o, ws, shared=shared, stream=stream)
        torch.cuda.synchronize()
        outs.append(o)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    check_rows(outs[0], q, k, v, table, seq, pos, 0.09)


def test_a_captured_step_follows_its_rows():
    """One graph of append, choice and both attentions; before each replay positions, sequences and inputs change on the device, padding rows among them."""
    from yasakani_b200 import kv4, paged
    hkv, nh, hd, page, dt, shared = 4, 24, 256, 32, torch.bfloat16, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    cache = paged.PagedCache(64, hkv, hd, page=page, dtype=dt, means=True)
    for t in (cache.k, cache.v, cache.kmean):
        t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
    order = torch.randperm(64, generator=g, device="cuda").to(torch.int32)
    table = torch.stack([torch.cat((order[:2], order[2 + 20 * i:22 + 20 * i])) for i in range(3)]).contiguous()
    rope = torch.empty((22 * page, 32, 2), dtype=torch.float32, device="cuda")
    kv4.launch_rope_table_g(rope, 22 * page, 1e6, 64)
    x = torch.randn((4, nh + 2 * hkv, hd), generator=g, device="cuda").to(dt)
    seq, pos = ints([0, 1, 2, -1]), ints([100, 200, 300, 0])
    q, o, o_shared, o_all = (torch.zeros((4, nh, hd), dtype=dt, device="cuda") for _ in range(4))
    ids = torch.zeros((4, hkv, 4), dtype=torch.int32, device="cuda")
    ws = paged.workspace(cache, 4, nh, table.shape[1], shared=shared, select=True)

    def step():
        paged.launch_append(cache, table, x[:, nh:nh + hkv], x[:, nh + hkv:], seq, pos, rope, 64, q=x[:, :nh], q_out=q)
        paged.launch_select(q, cache, table, seq, pos, ids, ws)
        paged.launch_attention(q, cache, table, seq, pos, hd ** -0.5, o, ws, blocks=ids)
        paged.launch_attention(q, cache, table, seq, pos, hd ** -0.5, o_shared, ws, shared=shared)
        paged.launch_attention(q, cache, table, seq, pos, hd ** -0.5, o_all, ws)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for s, p in (([0, 1, 2, -1], [101, 201, 301, 0]), ([2, -1, 0, 1], [31, 5, 639, 95]), ([-1, -1, -1, -1], [0, 0, 0, 0]), ([1, 1, 1, 0], [96, 97, 98, -1])):
        seq.copy_(ints(s)); pos.copy_(ints(p))
        x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        for t in (o, o_shared, o_all):
            t.fill_(3.0)
        ids.fill_(77)
        graph.replay()
        torch.cuda.synchronize()
        before = torch.full_like(o, 3.0)
        want = choose(q, cache.kmean, table, seq, pos, page, 4)
        for r, n in enumerate(s):
            if n < 0:
                want[r] = 77
        assert torch.equal(ids.cpu(), want)
        check_rows(o, q, cache.k, cache.v, table, seq, pos, hd ** -0.5, ids=ids, before=before)
        check_rows(o_shared, q, cache.k, cache.v, table, seq, pos, hd ** -0.5, before=before)
        check_rows(o_all, q, cache.k, cache.v, table, seq, pos, hd ** -0.5, before=before)
    assert kv4.device_status() == 0


def test_calls_behind_one_another_on_one_workspace():
    """A workspace for the largest call serves smaller ones at once behind it, without a wait in between."""
    from yasakani_b200 import paged
    nh, calls, big = 28, [], None
    for i, (n, shared) in enumerate(((60, 1280), (1, 0), (42, 1280), (7, 256), (300, 0), (43, 640))):
        k, v, kmean, table, seq, pos, q = case(lengths=[shared + 1 + (37 * j) % 200 for j in range(n)], seed=i, shared=shared)
        calls.append((paged.PagedCache.of(k, v), table, seq, pos, q, shared, torch.empty_like(q), k, v))
    ws = paged.workspace(calls[0][0], 300, nh, 64, shared=1280)
    torch.cuda.synchronize()
    for _ in range(2):
        for cache, table, seq, pos, q, shared, o, k, v in calls:
            paged.launch_attention(q, cache, table, seq, pos, 0.09, o, ws, shared=shared)
    torch.cuda.synchronize()
    for cache, table, seq, pos, q, shared, o, k, v in calls:
        some = list(range(0, q.shape[0], 1 + q.shape[0] // 12))
        check_rows(o[some], q[some], k, v, table, seq[some], pos[some], 0.09)


def test_queries_rotated_in_place_and_one_row():
    from yasakani_b200 import kv4, paged
    k, v, kmean, table, seq, pos, q = case("f16", lengths=(40,))
    rope = torch.empty((64, 64, 2), dtype=torch.float32, device="cuda")
    kv4.launch_rope_table_g(rope, 64, 1e6, 128)
    new = torch.randn((1, 4, 128), device="cuda").half()
    out, mine = torch.empty_like(q), q.clone()
    cache = paged.PagedCache.of(k, v)
    paged.launch_append(cache, table, new, new, seq, pos, rope, 128, q=q, q_out=out)
    paged.launch_append(cache, table, new, new, seq, pos, rope, 128, q=mine, q_out=mine)
    assert torch.equal(out, mine) and not torch.equal(out, q)
    assert torch.equal(v[int(table[0, 1]), :, 7], new[0])


def test_the_last_page_of_the_arrays():
    """Rows that end where the arrays end: nothing behind them is read or written (the guard values stay)."""
    from yasakani_b200 import paged
    page, hkv, hd = 16, 2, 128
    big = torch.full((6, hkv, page, hd), 1.0, dtype=torch.float16, device="cuda")
    k, v = big[:3], torch.randn((3, hkv, page, hd), device="cuda").half()
    k.copy_(torch.randn(k.shape, device="cuda"))
    big[3:] = float("nan")
    table, seq = ints([[0, 1, 2]]), ints([0])
    q = torch.randn((1, 4, hd), device="cuda").half()
    for pos in (47, 40, 32):
        o16, before = attend(k, v, table, seq, ints([pos]), q, 0.1)
        check_rows(o16, q, k, v, table, [0], [pos], 0.1)
        o16, before = attend(k, v, table, seq, ints([pos]), q, 0.1, shared=32)
        check_rows(o16, q, k, v, table, [0], [pos], 0.1)
    new = torch.randn((1, hkv, hd), device="cuda").half()
    paged.launch_append(paged.PagedCache.of(k, v), table, new, new, seq, ints([47]))
    assert torch.equal(k[2, :, 15], new[0]) and torch.isnan(big[3:]).all()


def test_refusals_on_the_device():
    from yasakani_b200 import Kv4Error, paged
    k, v, kmean, table, seq, pos, q = case()
    cache, o = paged.PagedCache.of(k, v, kmean), torch.empty_like(q)
    ws = paged.workspace(cache, 4, 28, table.shape[1], select=True)
    good = dict(q=q, cache=cache, table=table, seq=seq, pos=pos, qscale=0.1, o16=o, ws=ws)
    for change, error in ((dict(table=table.long()), TypeError), (dict(seq=seq.cpu()), AssertionError), (dict(pos=pos[:3]), ValueError), (dict(q=q.half()), TypeError),
                          (dict(q=q[:, :, :64]), ValueError), (dict(q=q[:3]), ValueError), (dict(o16=o[:, :27]), ValueError), (dict(ws=ws[:1024]), Kv4Error),
                          (dict(ws=ws[16:]), Kv4Error), (dict(ws=ws.cpu()), AssertionError), (dict(q=q[:, :27], o16=o[:, :27].contiguous()), Kv4Error), (dict(shared=33), Kv4Error),
                          (dict(blocks=torch.zeros((4, 4, 3), device="cuda")), TypeError), (dict(blocks=torch.zeros((4, 3, 3), dtype=torch.int32, device="cuda")), ValueError),
                          (dict(blocks=torch.zeros((4, 4, 0), dtype=torch.int32, device="cuda")), ValueError), (dict(table=table[:, ::2]), AssertionError),
                          (dict(o16=torch.empty((8, 28, 128), dtype=o.dtype, device="cuda")[::2]), AssertionError),
                          (dict(q=torch.zeros((1, 28, 128), dtype=q.dtype, device="cuda").expand(4, 28, 128)), Kv4Error)):
        with pytest.raises(error):
            paged.launch_attention(**dict(good, **change))
    with pytest.raises(Kv4Error, match="no mean keys|keeps no"):
        paged.launch_select(q, paged.PagedCache.of(k, v), table, seq, pos, torch.zeros((4, 4, 4), dtype=torch.int32, device="cuda"), ws)
    with pytest.raises(ValueError):
        paged.workspace(cache, 0, 28, 4)
    with pytest.raises(Kv4Error, match="page of 48"):
        paged.PagedCache(4, 2, 128, page=48)
    paged.launch_attention(**good)
    torch.cuda.synchronize()
    check_rows(o, q, k, v, table, seq, pos, 0.1)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="one GPU")
def test_a_cache_on_another_device_than_the_current_one():
    from yasakani_b200 import paged
    k, v, kmean, table, seq, pos, q = (t.to("cuda:1") for t in case())
    cache, o = paged.PagedCache.of(k, v), torch.empty_like(q)
    paged.launch_attention(q, cache, table, seq, pos, 0.09, o, paged.workspace(cache, 4, 28, table.shape[1]))
    torch.cuda.synchronize(1)
    assert torch.cuda.current_device() == 0
    check_rows(*(t.to("cuda:0") for t in (o, q, k, v, table)), seq.tolist(), pos.tolist(), 0.09)


@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("tiles", range(1, 10))
def test_prefix_runs_of_few_tiles_from_cold_caches(hd, tiles):
    """Each number of 128-token tiles in a run meets another phase of the prefix kernel's buffers at its end.  160 rows of 8 heads over 8 shared heads are 40
    pairs of blocks, more than half of those that fit, so a run has all the tiles; keys and values come from memory, late, and each launch has the same bits."""
    from yasakani_b200 import kv4, paged
    rows, nh, hkv, page, shared = 160, 64, 8, 32, 128 * tiles - 32 * (tiles % 2)
    k, v, _, table, seq, pos, q = case(lengths=[shared + 1 + i % 3 for i in range(rows)], nh=nh, hkv=hkv, hd=hd, page=page, shared=shared, seed=tiles)
    cache, ws = paged.PagedCache.of(k, v), paged.workspace(paged.PagedCache.of(k, v), rows, nh, table.shape[1], shared=shared)
    flush = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    outs = []
    for i in range(12):
        o = torch.full_like(q, 7.0)
        ws.fill_(0xFF)                                           # NaN wherever nothing is written
        flush.fill_(i)
        paged.launch_attention(q, cache, table, seq, pos, 0.09, o, ws, shared=shared)
        outs.append(o)
    torch.cuda.synchronize()
    assert kv4.device_status() == 0
    assert all(torch.equal(o.view(torch.int16), outs[0].view(torch.int16)) for o in outs)
    some = torch.tensor([0, 1, 15, 16, 31, 32, 80, 127, 159], device="cuda")
    check_rows(outs[0][some], q[some], k, v, table, seq[some], pos[some], 0.09)
