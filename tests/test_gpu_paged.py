"""The paged 16-bit cache against its definitions in 64 bits: append with rotation and mean keys, attention of single rows, over chosen blocks and
behind a shared part, the choice of blocks; lengths of none and one, pages that end inside a tile, garbage and non-finite values where nobody looks.

Tolerances.  h = half a step of the 16-bit type (2^-11, 2^-8), relative.  Attention: the scores are fp32 sums of exact products; a sum of n fp32 terms is off by at most
n 2^-24 of the sum of their magnitudes, so a score (in base 2) is off by e <= (HD + 4) 2^-23 * S with S = max sum |q k| * scale (tensor cores truncate: a whole step each), and a weight by
a factor 2^(2 e + 2^-21).  A weight is rounded once (h), the row once (h): |o - exact| <= h |o| + (h + 2 (2 e + 2^-20)) * sum w |v| + keys 2^-23 sum w |v|."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {"f16": torch.float16, "bf16": torch.bfloat16}


def half_step(dt):
    return torch.finfo(dt).eps / 2


def make_pool(lengths, hkv, hd, page, dt, seed, spare=3, garbage=False, width=None, shared=0):
    """Pages in any order; what lies behind a sequence's end is NaN and infinity where `garbage`."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    first = shared // page
    blocks = [max(0, -(-n // page) - first) for n in lengths]
    pages = first + sum(blocks) + spare
    order = torch.randperm(pages, generator=g, device="cuda").tolist()
    width = width or max(1, first + max(blocks))
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    common, at = order[:first], first
    k = torch.randn((pages, hkv, page, hd), generator=g, device="cuda").to(dt)
    v = torch.randn((pages, hkv, page, hd), generator=g, device="cuda").to(dt)
    for i, n in enumerate(lengths):
        mine = order[at:at + blocks[i]]
        at += blocks[i]
        have = min(first, -(-n // page)) if shared else 0
        for b, p in enumerate(common[:have] + mine):
            table[i, b] = p
        if garbage and n % page and mine:
            k[mine[-1], :, n % page:] = float("nan")
            v[mine[-1], :, n % page:] = float("inf")
    if garbage:
        for p in order[at:]:
            k[p], v[p] = float("nan"), float("nan")
    return k, v, table.cuda(), g


def exact_row(q, keys, values, qscale):
    """q [g][hd], keys / values [n][hd] in fp64 -> (o, sum w |v|, scale of the scores)."""
    if keys.shape[0] == 0:
        z = torch.zeros_like(q)
        return z, z, 0.0
    w = torch.softmax(q @ keys.T * qscale, -1)
    return w @ values, w @ values.abs(), float((q.abs() @ keys.abs().T).max() * abs(qscale) * math.log2(math.e))


def check_rows(o16, q, k, v, table, seq, pos, qscale, ids=None, before=None):
    dt, (n, nh, hd) = o16.dtype, q.shape
    hkv, page = k.shape[1], k.shape[2]
    g, h = nh // hkv, half_step(dt)
    worst = 0.0
    for r in range(n):
        s, p = int(seq[r]), int(pos[r])
        if not 0 <= s < table.shape[0]:
            assert torch.equal(o16[r].view(torch.int16), before[r].view(torch.int16)), f"padding row {r} was written"
            continue
        p = min(p, table.shape[1] * page - 1)
        for j in range(hkv):
            blocks = list(range(p // page + 1)) if p >= 0 else []
            if ids is not None:
                blocks = [b for b in ids[r, j].tolist() if 0 <= b <= (p // page if p >= 0 else -1) and b < table.shape[1]]
            kk, vv = [], []
            for b in blocks:
                pg, m = int(table[s, b]), min(page, p + 1 - b * page)
                if 0 <= pg < k.shape[0]:
                    kk.append(k[pg, j, :m].double()); vv.append(v[pg, j, :m].double())
            kk = torch.cat(kk) if kk else torch.zeros((0, hd), dtype=torch.float64, device="cuda")
            vv = torch.cat(vv) if vv else torch.zeros((0, hd), dtype=torch.float64, device="cuda")
            want, mag, S = exact_row(q[r, j * g:(j + 1) * g].double(), kk, vv, qscale)
            got = o16[r, j * g:(j + 1) * g].double()
            e = (hd + 4) * 2.0 ** -23 * S
            bound = h * want.abs() + (1 + h) * (h + 2 * (2 * e + 2.0 ** -20) + kk.shape[0] * 2.0 ** -23) * mag + 2.0 ** -24
            err = (got - want).abs()
            assert torch.isfinite(got).all(), (r, j)
            assert (err <= bound).all(), (r, j, float((err / bound).max()))
            worst = max(worst, float((err / bound).max()))
    return worst


def attend(k, v, table, seq, pos, q, qscale, shared=0, ids=None, stream=None):
    from yasakani_b200 import kv4, paged
    cache = paged.PagedCache.of(k, v)
    ws = paged.workspace(cache, q.shape[0], q.shape[1], table.shape[1], shared=shared)
    ws.fill_(0xFF)                                               # NaN wherever nothing is written
    o16 = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
    before = o16.clone()
    paged.launch_attention(q, cache, table, seq, pos, qscale, o16, ws, shared=shared, blocks=ids, stream=stream)
    torch.cuda.synchronize()
    assert kv4.device_status() == 0
    return o16, before


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ---------------------------------------------------------------------------------------------------------------- attention
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("nh,hkv,hd,page,lengths", [
    (16, 2, 128, 64, [1]),
    (24, 4, 256, 64, [64]),
    (24, 4, 256, 16, [1, 15, 16, 17, 63, 64, 65, 127, 129]),
    (28, 4, 128, 32, [500, 1, 33, 2000, 64]),
    (8, 8, 128, 128, [127, 128, 129, 700]),
    (32, 2, 256, 64, [1000, 5]),                                 # sixteen heads a kv-head
    (9, 1, 128, 16, [300, 77]),
    (1, 1, 256, 128, [4097]),
    (24, 4, 256, 64, [9000, 3, 0, 12]),
])
def test_rows_of_any_length(dt, nh, hkv, hd, page, lengths):
    k, v, table, g = make_pool(lengths, hkv, hd, page, DT[dt], seed=len(lengths) + hd, garbage=True)
    q = torch.randn((len(lengths), nh, hd), generator=g, device="cuda").to(DT[dt])
    seq, pos = torch.arange(len(lengths), dtype=torch.int32, device="cuda"), ints(lengths) - 1
    o16, before = attend(k, v, table, seq, pos, q, hd ** -0.5)
    check_rows(o16, q, k, v, table, seq, pos, hd ** -0.5, before=before)


def test_padding_rows_negative_positions_and_absent_pages():
    k, v, table, g = make_pool([200, 90, 300], 4, 128, 32, torch.bfloat16, seed=5, garbage=True)
    table[2, 3], table[2, 5] = -1, 10 ** 6                       # tokens without a page are not seen
    seq, pos = ints([0, -1, 1, 3, 2, 0, 2, -2 ** 31, 1]), ints([199, 5, 89, 4, 299, -1, 10 ** 9, 3, -2 ** 31])
    q = torch.randn((9, 28, 128), generator=g, device="cuda").bfloat16()
    k[:, :, :, :] = torch.where(torch.isfinite(k), k, 0.0)       # row 6 stands beyond the table: it sees all of its pages
    v[:, :, :, :] = torch.where(torch.isfinite(v), v, 0.0)
    o16, before = attend(k, v, table, seq, pos, q, 0.1)
    check_rows(o16, q, k, v, table, seq, pos, 0.1, before=before)
    assert (o16[5] == 0).all() and (o16[8] == 0).all()


def test_many_rows_take_several_launches_and_drafts_share_a_sequence():
    lengths = [37 + 5 * i % 90 for i in range(40)]
    k, v, table, g = make_pool(lengths, 2, 128, 16, torch.float16, seed=9, garbage=True)
    n = 1030
    seq = ints([i % 40 for i in range(n)])
    pos = ints([lengths[i % 40] - 1 - (i // 40) % 7 for i in range(n)])
    q = torch.randn((n, 4, 128), generator=g, device="cuda").half()
    o16, before = attend(k, v, table, seq, pos, q, 0.09)
    check_rows(o16[::37], q[::37], k, v, table, seq[::37], pos[::37], 0.09, before=before[::37])
    check_rows(o16[500:530], q[500:530], k, v, table, seq[500:530], pos[500:530], 0.09, before=before[500:530])


def test_large_scores_and_rows_of_a_wider_tensor():
    k, v, table, g = make_pool([777], 2, 128, 64, torch.bfloat16, seed=3)
    wide = torch.randn((1, 12, 128), generator=g, device="cuda").bfloat16() * 30
    q = wide[:, 4:8]
    for scale in (1.0, -1.0):                                     # a softmax that one key decides; scores far below zero
        o16, before = attend(k, v, table, ints([0]), ints([776]), q, scale)
        check_rows(o16, q, k, v, table, [0], [776], scale, before=before)


@pytest.mark.parametrize("shared", [0, 160])
def test_a_scale_of_zero_is_the_mean_of_the_values(shared):
    k, v, table, g = make_pool([shared + 50, shared + 7], 2, 128, 32, torch.bfloat16, seed=13, garbage=True, shared=shared)
    q = torch.randn((2, 6, 128), generator=g, device="cuda").bfloat16()
    pos = [shared + 49, shared + 6]
    o16, before = attend(k, v, table, ints([0, 1]), ints(pos), q, 0.0, shared=shared)
    check_rows(o16, q, k, v, table, [0, 1], pos, 0.0, before=before)


def test_values_that_are_not_finite_stay_in_their_channel():
    k, v, table, g = make_pool([100], 1, 128, 64, torch.float16, seed=4)
    v[int(table[0, 0]), 0, 5, 17] = float("inf")
    q = torch.randn((1, 2, 128), generator=g, device="cuda").half()
    o16, _ = attend(k, v, table, ints([0]), ints([99]), q, 0.1)
    assert torch.isinf(o16[0, :, 17]).all() and torch.isfinite(o16[0, :, :17]).all() and torch.isfinite(o16[0, :, 18:]).all()


# ---------------------------------------------------------------------------------------------------------------- a shared part
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("nh,hkv,hd,page,shared,behind", [
    (24, 4, 256, 64, 64, [0]),                                   # a row that ends with the shared part
    (24, 4, 256, 64, 1024, [1, 70, 64]),
    (28, 4, 128, 16, 16, [5, 0, 300, 16]),                       # less than a tile of keys
    (28, 4, 128, 32, 992, [(7 * i) % 90 for i in range(40)]),
    (16, 2, 128, 128, 4096, [1 + i for i in range(20)]),
    (32, 2, 256, 16, 400, [3] * 9),
    (4, 4, 128, 64, 8192, [(3 * i) % 5 for i in range(130)]),    # one head a kv-head, more rows than a tile holds
    (24, 4, 256, 32, 2592, [(11 * i) % 40 for i in range(50)]),
])
def test_rows_behind_a_shared_part(dt, nh, hkv, hd, page, shared, behind):
    lengths = [shared + n for n in behind]
    k, v, table, g = make_pool(lengths, hkv, hd, page, DT[dt], seed=shared + len(behind), garbage=True, shared=shared)
    n = len(lengths)
    q = torch.randn((n, nh, hd), generator=g, device="cuda").to(DT[dt])
    seq, pos = torch.arange(n, dtype=torch.int32, device="cuda"), ints(lengths) - 1
    o16, before = attend(k, v, table, seq, pos, q, hd ** -0.5, shared=shared)
    some = list(range(n)) if n <= 40 else list(range(0, n, 5)) + [n - 1]
    check_rows(o16[some], q[some], k, v, table, seq[some], pos[some], hd ** -0.5, before=before[some])


def test_shared_part_with_short_and_padding_rows():
    """Rows shorter than the shared part attend by themselves; padding rows and rows that see nothing stay what they are, the first ones too."""
    shared, lengths = 640, [700, 640, 641, 900]
    k, v, table, g = make_pool(lengths, 4, 128, 64, torch.bfloat16, seed=8, garbage=True, shared=shared)
    seq, pos = ints([-1, 0, 0, 1, 2, 3, 3, 3, 9, 1]), ints([699, -1, 300, 639, 640, 899, 638, 0, 640, -7])
    q = torch.randn((10, 28, 128), generator=g, device="cuda").bfloat16()
    for scale in (0.09, -0.09):
        o16, before = attend(k, v, table, seq, pos, q, scale, shared=shared)
        check_rows(o16, q, k, v, table, seq, pos, scale, before=before)
    pos[:] = -1                                                  # no row at all has the shared part
    o16, before = attend(k, v, table, seq, pos, q, 0.09, shared=shared)
    check_rows(o16, q, k, v, table, seq, pos, 0.09, before=before)


def test_shared_part_with_large_scores_and_rising_maxima():
    """The running maximum grows from tile to tile by more than the rescale's margin."""
    shared = 2048
    k, v, table, g = make_pool([shared + 10, shared + 3], 2, 128, 64, torch.float16, seed=6, shared=shared)
    for b in range(shared // 64):
        k[int(table[0, b])] *= 0.1 * (b + 1)
    q = torch.randn((2, 16, 128), generator=g, device="cuda").half() * 8
    o16, before = attend(k, v, table, ints([0, 1]), ints([shared + 9, shared + 2]), q, 0.2, shared=shared)
    check_rows(o16, q, k, v, table, [0, 1], [shared + 9, shared + 2], 0.2, before=before)


# ---------------------------------------------------------------------------------------------------------------- chosen blocks
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("nh,hkv,hd,page,lengths,take", [
    (24, 4, 256, 64, [5000, 64, 65, 1], 9), (28, 4, 128, 16, [1000, 31, 500], 7), (8, 1, 128, 128, [3000, 129], 4), (16, 2, 128, 32, [700], 60)])
def test_attention_over_chosen_blocks(dt, nh, hkv, hd, page, lengths, take):
    k, v, table, g = make_pool(lengths, hkv, hd, page, DT[dt], seed=take, garbage=True)
    n = len(lengths)
    q = torch.randn((n, nh, hd), generator=g, device="cuda").to(DT[dt])
    ids = torch.full((n, hkv, take), -1, dtype=torch.int32)
    for r, m in enumerate(lengths):
        last = (m - 1) // page
        for j in range(hkv):
            pick = torch.randperm(last + 1)[:take - 1].tolist()
            pick = (pick + [last, -5, table.shape[1] + 3, 2 ** 31 - 1])[:take]      # any order; the last twice perhaps; some that name nothing
            ids[r, j, :len(pick)] = torch.tensor(pick, dtype=torch.int32)
    seq, pos, ids = torch.arange(n, dtype=torch.int32, device="cuda"), ints(lengths) - 1, ids.cuda()
    o16, before = attend(k, v, table, seq, pos, q, hd ** -0.5, ids=ids)
    check_rows(o16, q, k, v, table, seq, pos, hd ** -0.5, ids=ids, before=before)


def choose(q, kmean, table, seq, pos, page, take):
    """The definition: fp64 scores, ties to the lowest block, the last block always."""
    n, nh, hd = q.shape
    hkv = kmean.shape[1]
    ids = torch.full((n, hkv, take), -1, dtype=torch.int32)
    for r in range(n):
        s, p = int(seq[r]), min(int(pos[r]), table.shape[1] * page - 1)
        if p < 0 or not 0 <= s < table.shape[0]:
            continue
        last = p // page
        for j in range(hkv):
            have = [b for b in range(last) if 0 <= int(table[s, b]) < kmean.shape[0]]
            if have:
                m = kmean[table[s, have].long(), j].double()
                x = (q[r, j * (nh // hkv):(j + 1) * (nh // hkv)].double() @ m.T)
                x = torch.where(torch.isnan(x), -math.inf, x).amax(0)
                have = sorted(torch.tensor(have)[torch.sort(x, descending=True, stable=True)[1][:take - 1].cpu()].tolist())
            got = have + [last]
            ids[r, j, :len(got)] = torch.tensor(got, dtype=torch.int32)
    return ids


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("nh,hkv,hd,page,lengths,take", [
    (24, 4, 256, 16, [40000, 1, 16, 17, 5000], 33), (28, 4, 128, 32, [9000, 64], 2), (16, 1, 128, 64, [70000], 1024), (1, 1, 256, 128, [1000, 130], 5)])
def test_choice_of_blocks(dt, nh, hkv, hd, page, lengths, take):
    from yasakani_b200 import paged
    k, v, table, g = make_pool(lengths, hkv, hd, page, DT[dt], seed=take + nh)
    kmean = torch.randn((k.shape[0], hkv, hd), generator=g, device="cuda").to(DT[dt])
    for a in range(3, 40, 4):                                    # blocks of equal height
        if a + 1 < table.shape[1] and table[0, a + 1] >= 0:
            kmean[int(table[0, a + 1])] = kmean[int(table[0, a])]
    if table.shape[1] > 60:
        table[0, 50] = -1                                        # no page, no candidate
        kmean[int(table[0, 51])] = float("nan")
    n = len(lengths)
    q = torch.randn((n, nh, hd), generator=g, device="cuda").to(DT[dt])
    seq, pos = torch.arange(n, dtype=torch.int32, device="cuda"), ints(lengths) - 1
    if n > 1:
        seq[1] = -1                                              # a padding row keeps what it had
    cache = paged.PagedCache.of(k, v, kmean)
    ws = paged.workspace(cache, n, nh, table.shape[1], select=True)
    ids = torch.full((n, hkv, take), 99, dtype=torch.int32, device="cuda")
    paged.launch_select(q, cache, table, seq, pos, ids, ws)
    want = choose(q, kmean, table, seq, pos, page, take)
    if n > 1:
        want[1] = 99
    assert torch.equal(ids.cpu(), want)


@pytest.mark.parametrize("blocks,take,kind", [(5000, 33, "random"), (9001, 1024, "random"), (4097, 300, "equal"), (6000, 50, "few values"), (70000, 20, "few values"),
                                              (66000, 100, "random"), (5000, 40, "not finite")])
def test_choice_among_many_blocks(blocks, take, kind):
    """More blocks than a thread block keeps in registers, or has bits for; scores that are equal, or that fp32 cannot tell apart, or does not hold."""
    from yasakani_b200 import paged
    g = torch.Generator(device="cuda").manual_seed(blocks)
    k = torch.zeros((blocks, 1, 16, 128), dtype=torch.bfloat16, device="cuda")
    kmean = torch.randn((blocks, 1, 128), generator=g, device="cuda").bfloat16()
    if kind == "equal":
        kmean[:] = kmean[0]
    if kind == "few values":
        kmean = kmean[torch.randint(0, 40, (blocks,), generator=g, device="cuda")].contiguous()
    if kind == "not finite":
        kmean[torch.randint(0, blocks, (500,), generator=g, device="cuda"), 0, 5] = float("inf")
        kmean[77, 0, 3] = float("nan")
        kmean[78, 0] = 3e38
    table = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)[None].contiguous()
    q = torch.randn((1, 3, 128), generator=g, device="cuda").bfloat16()
    cache = paged.PagedCache.of(k, k, kmean)
    ids = torch.full((1, 1, take), 99, dtype=torch.int32, device="cuda")
    paged.launch_select(q, cache, table, ints([0]), ints([blocks * 16 - 1]), ids, paged.workspace(cache, 1, 3, blocks, select=True))
    assert torch.equal(ids.cpu(), choose(q, kmean, table, [0], [blocks * 16 - 1], 16, take))


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("shift", [2, 6, 10, 13])
def test_choice_where_scores_are_differences_of_large_sums(dt, shift):
    """Channels that cancel one another by up to 2^shift: fp32 sums are off by more than neighbours differ, and the choice is that of fp64 sums all the same."""
    from yasakani_b200 import paged
    hkv, nh, hd, blocks, take = 2, 6, 128, 700, 40
    g = torch.Generator(device="cuda").manual_seed(shift)
    km, q = torch.randn((blocks, hkv, hd), generator=g, device="cuda"), torch.randn((1, nh, hd), generator=g, device="cuda")
    big = torch.randn((blocks, hkv, hd // 2), generator=g, device="cuda").abs() * 2.0 ** shift
    q[..., 1::2] = q[..., ::2]
    km[..., ::2] += big
    km[..., 1::2] -= big
    km, q = km.to(DT[dt]).contiguous(), q.to(DT[dt])
    k = torch.zeros((blocks, hkv, 16, hd), dtype=DT[dt], device="cuda")
    table = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)[None].contiguous()
    ids = torch.empty((1, hkv, take), dtype=torch.int32, device="cuda")
    cache = paged.PagedCache.of(k, k, km)
    paged.launch_select(q, cache, table, ints([0]), ints([blocks * 16 - 1]), ids, paged.workspace(cache, 1, nh, blocks, select=True))
    assert torch.equal(ids.cpu(), choose(q, km, table, [0], [blocks * 16 - 1], 16, take))


def test_choice_among_equal_scores_takes_the_lowest_blocks():
    from yasakani_b200 import paged
    k, v, table, g = make_pool([64 * 600], 2, 128, 64, torch.float16, seed=1)
    kmean = torch.zeros((k.shape[0], 2, 128), dtype=torch.float16, device="cuda")
    q = torch.randn((1, 4, 128), generator=g, device="cuda").half()
    ids = torch.empty((1, 2, 300), dtype=torch.int32, device="cuda")
    cache = paged.PagedCache.of(k, v, kmean)
    ws = paged.workspace(cache, 1, 4, 600, select=True)
    paged.launch_select(q, cache, table, ints([0]), ints([64 * 600 - 1]), ids, ws)
    want = torch.tensor(list(range(299)) + [599], dtype=torch.int32).expand(1, 2, 300)
    assert torch.equal(ids.cpu(), want)
    paged.launch_select(q, cache, table, ints([0]), ints([-1]), ids, ws)
    assert (ids == -1).all()


# ---------------------------------------------------------------------------------------------------------------- append
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("nh,hkv,hd,page,rd,starts,rows", [
    (24, 4, 256, 64, 64, [0, 100], [130, 1]), (28, 4, 128, 16, 128, [5, 0, 15], [40, 1, 1]), (3, 1, 128, 32, 16, [31, 0], [1, 64]),
    (2, 2, 256, 128, 256, [127, 0], [1, 256]), (16, 2, 128, 64, 96, [60], [10]), (4, 4, 128, 64, 0, [0], [64])])
def test_append(dt, nh, hkv, hd, page, rd, starts, rows):
    from yasakani_b200 import kv4, paged
    T, h = sum(rows), half_step(DT[dt])
    k, v, table, g = make_pool([a + b for a, b in zip(starts, rows)], hkv, hd, page, DT[dt], seed=T)
    old_k, old_v = k.clone(), v.clone()
    kmean = torch.full((k.shape[0], hkv, hd), 5.0, dtype=DT[dt], device="cuda")
    x = torch.randn((T, nh + 2 * hkv, hd), generator=g, device="cuda").to(DT[dt])
    seq = ints([i for i, m in enumerate(rows) for _ in range(m)])
    pos = ints([a + j for a, m in zip(starts, rows) for j in range(m)])
    max_ctx = 512
    rope = torch.empty((max_ctx, max(rd, 2) // 2, 2), dtype=torch.float32, device="cuda")
    if rd:
        kv4.launch_rope_table_g(rope, max_ctx, 1e6, rd)
    pad = T // 2
    if T > 2:
        seq[pad] = -1                                            # a padding row in the middle
    q_out = torch.full((T, nh, hd), 9.0, dtype=DT[dt], device="cuda")
    paged.launch_append(paged.PagedCache.of(k, v, kmean), table, x[:, nh:nh + hkv], x[:, nh + hkv:], seq, pos, rope if rd else None, rd, q=x[:, :nh], q_out=q_out)
    torch.cuda.synchronize()
    y = x.double()
    bound = torch.zeros_like(y)
    if rd:
        cs = rope.double()[pos.long()][:, None]
        a, b = y[..., :rd // 2].clone(), y[..., rd // 2:rd].clone()
        y[..., :rd // 2], y[..., rd // 2:rd] = a * cs[..., 0] - b * cs[..., 1], b * cs[..., 0] + a * cs[..., 1]
        mag = a.abs() * cs[..., 0].abs() + b.abs() * cs[..., 1].abs(), b.abs() * cs[..., 0].abs() + a.abs() * cs[..., 1].abs()
        tiny = torch.finfo(DT[dt]).smallest_normal * h           # half a step of the smallest numbers
        bound[..., :rd] = h * y[..., :rd].abs() + (1 + h) * 2.0 ** -23 * torch.cat(mag, -1) + tiny      # one rounding; two fp32 operations
    live = [i for i in range(T) if int(seq[i]) >= 0]
    want_q, got_q = y[live, :nh], q_out[live].double()
    assert ((got_q - want_q).abs() <= bound[live, :nh]).all()
    if T > 2:
        assert (q_out[pad] == 9.0).all()
    new_k, new_v = old_k.clone(), old_v.clone()
    for i in live:
        p, o = int(table[int(seq[i]), int(pos[i]) // page]), int(pos[i]) % page
        assert torch.equal(v[p, :, o], x[i, nh + hkv:])
        assert ((k[p, :, o].double() - y[i, nh:nh + hkv]).abs() <= bound[i, nh:nh + hkv]).all(), i
        new_k[p, :, o], new_v[p, :, o] = k[p, :, o], x[i, nh + hkv:]
    assert torch.equal(new_k, k) and torch.equal(new_v, v)       # nothing else was written
    want_mean = torch.full_like(kmean, 5.0)
    for i in live:
        if (int(pos[i]) + 1) % page == 0:
            p = int(table[int(seq[i]), int(pos[i]) // page])
            exact = k[p].double().mean(1)
            assert ((kmean[p].double() - exact).abs() <= h * exact.abs() + (1 + h) * (page * 2.0 ** -24) * k[p].double().abs().mean(1) + 2.0 ** -25).all()
            want_mean[p] = kmean[p]
    assert torch.equal(want_mean, kmean)


def test_means_of_pages_whose_rows_come_in_any_order():
    from yasakani_b200 import kv4, paged
    page, dt = 32, torch.bfloat16
    k, v, table, g = make_pool([200, 130, 64], 2, 128, page, dt, seed=21)
    kmean = torch.full((k.shape[0], 2, 128), 5.0, dtype=dt, device="cuda")
    rope = torch.empty((256, 64, 2), dtype=torch.float32, device="cuda")
    kv4.launch_rope_table_g(rope, 256, 1e6, 128)
    where = [(0, p) for p in range(37, 200)] + [(1, p) for p in range(10, 128)] + [(2, p) for p in (63, 31, 30)]     # pages that were begun before, that end inside, rows apart
    where = [where[i] for i in torch.randperm(len(where), generator=torch.Generator().manual_seed(1)).tolist()]
    x = torch.randn((len(where), 4, 128), generator=g, device="cuda").to(dt)
    outs = []
    for order in (list(range(len(where))), sorted(range(len(where)), key=lambda i: where[i])):
        c = [t.clone() for t in (k, v, kmean)]
        seq, pos = ints([where[i][0] for i in order]), ints([where[i][1] for i in order])
        y = x[order].contiguous()
        paged.launch_append(paged.PagedCache.of(*c), table, y[:, :2], y[:, 2:], seq, pos, rope, 128)
        torch.cuda.synchronize()
        outs.append(c)
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    full = {(s, p // page) for s, p in where if p % page == page - 1}
    for s in range(3):
        for b in range(table.shape[1]):
            pg = int(table[s, b])
            if pg < 0:
                continue
            if (s, b) not in full:
                assert (outs[0][2][pg] == 5.0).all()
                continue
            rows = outs[0][0][pg].double()
            h = half_step(dt)
            assert ((outs[0][2][pg].double() - rows.mean(1)).abs() <= h * rows.mean(1).abs() + (1 + h) * page * 2.0 ** -24 * rows.abs().mean(1) + 2.0 ** -25).all(), (s, b)


def test_append_leaves_out_rows_without_a_place():
    from yasakani_b200 import paged
    k, v, table, g = make_pool([64, 64], 2, 128, 16, torch.float16, seed=2)
    table[1, 2] = -1
    old_k, old_v = k.clone(), v.clone()
    kmean = torch.zeros((k.shape[0], 2, 128), dtype=torch.float16, device="cuda")
    x = torch.randn((6, 6, 128), generator=g, device="cuda").half()
    rope = torch.zeros((64, 64, 2), device="cuda")
    rope[..., 0] = 1.0                                           # no turn: rows are copied
    seq, pos = ints([0, 1, 0, 2, 1, 0]), ints([-1, 47, 64, 0, 63, 2 ** 31 - 1])      # negative, no page, beyond table and angles, no such sequence, one that fits
    q_out = torch.full((6, 2, 128), 9.0, dtype=torch.float16, device="cuda")
    paged.launch_append(paged.PagedCache.of(k, v, kmean), table, x[:, 2:4], x[:, 4:], seq, pos, rope, 128, q=x[:, :2], q_out=q_out)
    p = int(table[1, 3])
    old_k[p, :, 15], old_v[p, :, 15] = x[4, 2:4], x[4, 4:]
    assert torch.equal(k, old_k) and torch.equal(v, old_v)
    assert torch.equal(q_out[4], x[4, :2]) and torch.equal(q_out[1], x[1, :2])       # a position without a page still has an angle
    assert (q_out[[0, 2, 3, 5]] == 9.0).all()
    assert (kmean[[i for i in range(k.shape[0]) if i != p]] == 0).all() and not (kmean[p] == 0).all()


# ---------------------------------------------------------------------------------------------------------------- a run of all of them
@pytest.mark.parametrize("page,hd,nh,hkv,rd", [(16, 128, 28, 4, 128), (64, 256, 24, 4, 64)])
def test_a_run_as_a_server_makes_it(page, hd, nh, hkv, rd):
    """Prompts of two sequences behind a common part, then steps of one token each: append, choose, attend over all, over the chosen ones, with the common part shared."""
    from yasakani_b200 import kv4, paged
    dt, shared, prompts, steps = torch.bfloat16, 8 * page, [3 * page + 5, page - 1], 3
    g = torch.Generator(device="cuda").manual_seed(page)
    pages = 8 + 2 * 6
    cache = paged.PagedCache(pages, hkv, hd, page=page, dtype=dt, means=True)
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.stack([torch.cat((order[:8], order[8 + 6 * i:14 + 6 * i])) for i in range(2)]).contiguous()
    max_ctx = 14 * page
    rope = torch.empty((max_ctx, rd // 2, 2), dtype=torch.float32, device="cuda")
    kv4.launch_rope_table_g(rope, max_ctx, 1e6, rd)
    ws = paged.workspace(cache, 64, nh, table.shape[1], shared=shared, select=True)

    def append(seq, pos):
        x = torch.randn((len(pos), nh + 2 * hkv, hd), generator=g, device="cuda").to(dt)
        q = torch.empty((len(pos), nh, hd), dtype=dt, device="cuda")
        paged.launch_append(cache, table, x[:, nh:nh + hkv], x[:, nh + hkv:], ints(seq), ints(pos), rope, rd, q=x[:, :nh], q_out=q)
        return q

    append([0] * shared, list(range(shared)))
    for i, m in enumerate(prompts):
        append([i] * m, [shared + x for x in range(m)])
    for t in range(steps):
        seq, pos = ints([0, 1]), ints([shared + m + t for m in prompts])
        q = append([0, 1], pos.tolist())
        ids = torch.empty((2, hkv, 5), dtype=torch.int32, device="cuda")
        outs = [torch.empty_like(q) for _ in range(3)]
        paged.launch_select(q, cache, table, seq, pos, ids, ws)
        paged.launch_attention(q, cache, table, seq, pos, hd ** -0.5, outs[0], ws, blocks=ids)
        paged.launch_attention(q, cache, table, seq, pos, hd ** -0.5, outs[1], ws)
        paged.launch_attention(q, cache, table, seq, pos, hd ** -0.5, outs[2], ws, shared=shared)
        assert torch.equal(ids.cpu(), choose(q, cache.kmean, table, seq, pos, page, 5))
        check_rows(outs[0], q, cache.k, cache.v, table, seq, pos, hd ** -0.5, ids=ids)
        check_rows(outs[1], q, cache.k, cache.v, table, seq, pos, hd ** -0.5)
        check_rows(outs[2], q, cache.k, cache.v, table, seq, pos, hd ** -0.5)
    assert kv4.device_status() == 0
