"""Operators over a paged cache of 16-bit rows: what a server of many sequences asks of it, from one token to a whole prompt.

The rows of a layer lie in pages, k and v [pages][kv-heads][page][head_dim]; `table` [sequences][blocks] names the page of each block of a
sequence.  Keys are rotated when they are appended.  Sizes are those of the repository's configurations (24 / 4 heads of 256 channels with 64
rotated, 16 / 2 and 28 / 4 heads of 128), key channels scaled as there; pages lie anywhere in the pool.

  kinds   append    rows of several sequences into their pages, keys and queries rotated at each row's position, the mean key of every page
                    that a row completes                                                                                 (every step, every prompt)
          decode    one row for each of several sequences over its pages                                                 (batched token generation)
          prefix    the same where all sequences begin with the same pages                                               (one system prompt, many users)
          sparse    the pages whose mean keys score highest for each row and kv-head, then attention over those alone    (long contexts)
"""
import math

import torch

own = False

HEADS = {(16, 2, 128): (128, 1e6), (28, 4, 128): (128, 1e6), (24, 4, 256): (64, 1e7)}       # (heads, kv-heads, channels) -> rotated channels, base


def _case(kind, name, dtype, heads, page, **more):
    hq, hkv, hd = heads
    c = dict(kind=kind, dtype=dtype, hq=hq, hkv=hkv, hd=hd, page=page, **more)
    return dict(c, name=name) if name else c


def listed():
    small, wide, big = (16, 2, 128), (28, 4, 128), (24, 4, 256)
    return [
        # one new token for each of eight sequences: latency and launches
        _case("append", "append_8_tokens", "f16", small, 64, starts="900,63,4095,127,2000,17,31,512", rows="1,1,1,1,1,1,1,1"),
        # odd chunks of five prompts in one call, small pages
        _case("append", "append_ragged_1203", "bf16", wide, 16, starts="0,37,1000,15,4", rows="301,5,640,1,256"),
        # a whole prompt
        _case("append", "append_prompt_8192", "bf16", big, 64, starts="0", rows="8192"),
        # one token of a small layer at a short context
        _case("decode", "decode_hd128_4k", "f16", small, 64, contexts="4096"),
        # token generation for eight users at mixed contexts
        _case("decode", "decode_batch_8", "bf16", big, 64, contexts="2048,4096,8192,16384,32768,65536,98304,131072"),
        # many users with short, ragged contexts in small pages
        _case("decode", "decode_ragged_33", "bf16", wide, 16, contexts=",".join(str(37 + 241 * ((7 * i) % 33)) for i in range(33))),
        # a few users behind a common prompt
        _case("prefix", "prefix_8_users_4k", "f16", small, 64, shared=4096, contexts="1,300,77,1000,513,64,65,200"),
        # many users behind a long common prompt
        _case("prefix", "prefix_64_users_32k", "bf16", big, 64, shared=32768, contexts=",".join(str(1 + 97 * ((11 * i) % 64) % 1500) for i in range(64))),
        # more users than two tiles hold, a common prompt that ends inside a tile of keys
        _case("prefix", "prefix_200_users_5k", "bf16", wide, 32, shared=5216, contexts=",".join(str(1 + (53 * i) % 700) for i in range(200))),
        # one token over a long context, of which 64 pages are read
        _case("sparse", "sparse_131k", "bf16", big, 64, contexts="131072", take=64),
        # five sequences of odd lengths, smaller pages
        _case("sparse", "sparse_5_users_20k", "f16", big, 32, contexts="20011,777,12345,31999,5000", take=48),
        # sixteen long sequences
        _case("sparse", "sparse_16_users_64k", "bf16", wide, 64, contexts=",".join(str(65536 - 1000 * i) for i in range(16)), take=33),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _text(values):
    return ",".join(str(v) for v in values)


def draw(rng):
    kind, dtype = rng.choice(["append", "decode", "prefix", "sparse"]), rng.choice(["f16", "bf16"])
    heads, page = rng.choice(sorted(HEADS)), rng.choice([16, 32, 64, 128])
    if kind == "append":
        n = _log(rng, 1, 40)
        most = rng.choice([1, 8192 // n])
        return _case(kind, None, dtype, heads, page, starts=_text(rng.randint(0, 5000) for _ in range(n)), rows=_text(_log(rng, 1, most) for _ in range(n)))
    if kind == "decode":
        n = _log(rng, 1, 64)
        return _case(kind, None, dtype, heads, page, contexts=_text(_log(rng, 1, 262144 // n) for _ in range(n)))
    if kind == "prefix":
        n = _log(rng, 2, 200)
        return _case(kind, None, dtype, heads, page, shared=page * max(1, _log(rng, 128, 2000000 // n if n > 61 else 32768) // page),
                     contexts=_text(_log(rng, 1, 1000) for _ in range(n)))
    n = _log(rng, 1, 16)
    return _case(kind, None, dtype, heads, page, contexts=_text(_log(rng, 200, 262144 // n) for _ in range(n)), take=rng.randint(2, max(2, 4096 // page)))


# ---------------------------------------------------------------------------------------------------------------- inputs
def _ints(text):
    return [int(x) for x in text.split(",")]


def _dtype(case):
    return torch.float16 if case["dtype"] == "f16" else torch.bfloat16


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _key_scale(g, hkv, hd):
    lo, hi = math.log(0.5), math.log(4.0)
    return torch.exp(torch.rand((hkv, 1, hd), generator=g, device="cuda") * (hi - lo) + lo)


def _rope(n, rd, theta):
    freq = theta ** (-torch.arange(0, rd, 2, dtype=torch.float64, device="cuda") / rd)
    angle = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * freq
    return torch.stack((angle.cos(), angle.sin()), -1).float().contiguous()                 # [positions][rd / 2][cos, sin]


def _lengths(case):
    """Rows of each sequence that lie in pages of its own (behind a shared part), whole sequences' lengths."""
    if case["kind"] == "append":
        own_rows = [a + b for a, b in zip(_ints(case["starts"]), _ints(case["rows"]))]
    else:
        own_rows = _ints(case["contexts"])
    return own_rows, [n + case.get("shared", 0) for n in own_rows]


def _pool(case, g, correlated):
    """Pages in any order, filled with rows (old ones where nothing has been written yet), and the sequences' table."""
    page, hkv, hd, dt = case["page"], case["hkv"], case["hd"], _dtype(case)
    own_rows, _ = _lengths(case)
    first = case.get("shared", 0) // page
    blocks = [-(-n // page) for n in own_rows]
    pages = first + sum(blocks)
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    width = first + max(blocks)
    at = torch.arange(width, device="cuda")[None, :]
    n = torch.tensor(blocks, device="cuda")[:, None]
    begin = first + n.cumsum(0) - n
    table = torch.where(at < first, order[at.clamp(max=max(first - 1, 0))], torch.where(at - first < n, order[(begin + at - first).clamp(max=pages - 1)], -1))
    k, v = (torch.empty((pages, hkv, page, hd), dtype=dt, device="cuda") for _ in range(2))
    scale = _key_scale(g, hkv, hd)
    for p in range(0, pages, 1024):
        m = min(1024, pages - p)
        x = _randn(g, m, hkv, page, hd)
        if correlated:                                          # the tokens of a passage have something in common
            x = 0.8 * x + 0.6 * _randn(g, m, hkv, 1, hd)
        k[p:p + m], v[p:p + m] = (x * scale).to(dt), _randn(g, m, hkv, page, hd).to(dt)
    return dict(k=k, v=v, table=table.to(torch.int32).contiguous(), scale=scale)


def prepare(case, seed):
    g, kind, dt = torch.Generator(device="cuda").manual_seed(seed), case["kind"], _dtype(case)
    hq, hkv, hd, page = (case[x] for x in ("hq", "hkv", "hd", "page"))
    s = dict(kind=kind, hq=hq, page=page, shared=case.get("shared", 0), qscale=1.0 / math.sqrt(hd), **_pool(case, g, kind == "sparse"))
    _, whole = _lengths(case)
    if kind == "append":
        starts, rows = _ints(case["starts"]), _ints(case["rows"])
        s["seq"] = torch.repeat_interleave(torch.arange(len(rows), device="cuda"), torch.tensor(rows, device="cuda")).to(torch.int32)
        pos = [a + i for a, n in zip(starts, rows) for i in range(n)]
        s["pos"] = torch.tensor(pos, dtype=torch.int32, device="cuda")
        s["ends"] = torch.tensor([i for i, p in enumerate(pos) if (p + 1) % page == 0], dtype=torch.int64, device="cuda")      # rows that complete a page
        T, (rd, theta) = len(pos), HEADS[(hq, hkv, hd)]
        s["rd"], s["rope"] = rd, _rope((max(whole) + 63) // 64 * 64, rd, theta)
        qkv = _randn(g, T, hq + 2 * hkv, hd)
        qkv[:, hq:hq + hkv] *= s["scale"][:, 0]
        s["qkv"], s["q_out"] = qkv.to(dt), torch.zeros((T, hq, hd), dtype=dt, device="cuda")    # one projection's output: queries, keys, values
        s["kmean"] = torch.zeros((s["k"].shape[0], hkv, hd), dtype=dt, device="cuda")
    else:
        n = len(whole)
        s["seq"], s["pos"] = torch.arange(n, dtype=torch.int32, device="cuda"), torch.tensor(whole, dtype=torch.int32, device="cuda") - 1
        s["q"], s["o16"] = _randn(g, n, hq, hd).to(dt), torch.zeros((n, hq, hd), dtype=dt, device="cuda")
        s["take"] = case.get("take", 0)
        s["kmean"] = s["k"].float().mean(2).to(dt) if kind == "sparse" else None
        s["ids"] = torch.full((n, hkv, s["take"]), -1, dtype=torch.int32, device="cuda")
    if own:
        from yasakani_b200 import paged
        s["cache"] = paged.PagedCache.of(s["k"], s["v"], s["kmean"])
        if kind != "append":
            s["ws"] = paged.workspace(s["cache"], len(whole), hq, s["table"].shape[1], shared=s["shared"], select=kind == "sparse")
    return s


# ---------------------------------------------------------------------------------------------------------------- the plain forms
def _turn(x, cs, rd):
    """Rotates channels (c, c + rd / 2) of x [rows][heads][channels] by the rows' (cos, sin)."""
    a, b, rest = x[..., :rd // 2], x[..., rd // 2:rd], x[..., rd:]
    c, d = cs[:, None, :, 0], cs[:, None, :, 1]
    return torch.cat((a * c - b * d, b * c + a * d, rest), -1)


def _append(s):
    page, hq, rd, k = s["page"], s["hq"], s["rd"], s["k"]
    hkv, dt = k.shape[1], k.dtype
    seq, pos = s["seq"].long(), s["pos"].long()
    at, slot, cs = s["table"][seq, pos // page].long(), pos % page, s["rope"][pos]
    s["q_out"].copy_(_turn(s["qkv"][:, :hq].float(), cs, rd))
    k[at, :, slot] = _turn(s["qkv"][:, hq:hq + hkv].float(), cs, rd).to(dt)
    s["v"][at, :, slot] = s["qkv"][:, hq + hkv:]
    done = at[s["ends"]]
    s["kmean"][done] = (k[done].float().sum(2) / page).to(dt)
    return [s["q_out"], k, s["v"], s["kmean"]]


def _weights(x, see):
    """exp(x - max) over the last axis where `see`, and its sum."""
    x = torch.where(see, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - top)
    return p, p.sum(-1, keepdim=True)


def _rows_of(x, pages):
    """Rows of the pages [..., blocks] as [..., kv-heads, blocks * page, channels] in 32 bits (absent pages: the first one's)."""
    y = x[pages.clamp(min=0).long()].float().transpose(-4, -3)
    return y.reshape(*y.shape[:-3], -1, y.shape[-1])


def _attend(s):
    n, hq, hd = s["q"].shape
    hkv, page, first = s["k"].shape[1], s["page"], s["shared"] // s["page"]
    q = s["q"].float().view(n, hkv, hq // hkv, hd) * s["qscale"]
    table = s["table"][:, first:]
    keys, values = _rows_of(s["k"], table), _rows_of(s["v"], table)                         # [rows][kv-heads][tokens][channels]
    at = s["shared"] + torch.arange(keys.shape[2], device="cuda")
    see = (at[None, :] <= s["pos"][:, None])[:, None, None, :].expand(n, 1, 1, -1)
    x = q @ keys.transpose(-1, -2)
    if first:                                                                               # the common part: its rows are taken once, for all
        pages = s["table"][0, :first]
        common, common_v = _rows_of(s["k"], pages), _rows_of(s["v"], pages)                 # [kv-heads][tokens][channels]
        flat = q.transpose(0, 1).reshape(hkv, -1, hd)
        y = (flat @ common.transpose(-1, -2)).view(hkv, n, hq // hkv, -1).transpose(0, 1)
        x, see = torch.cat((y, x), -1), torch.cat((torch.ones_like(see[..., :1]).expand(n, 1, 1, s["shared"]), see), -1)
    p, total = _weights(x, see)
    o = p[..., s["shared"]:] @ values
    if first:
        flat = p[..., :s["shared"]].transpose(0, 1).reshape(hkv, -1, s["shared"])
        o = o + (flat @ common_v).view(hkv, n, hq // hkv, hd).transpose(0, 1)
    s["o16"].copy_((o / total).view(n, hq, hd))
    return s["o16"]


def _sparse(s):
    n, hq, hd = s["q"].shape
    hkv, page, take = s["k"].shape[1], s["page"], s["take"]
    last = s["pos"].long() // page                                                          # the block that is open, or just full: always taken
    means = s["kmean"][s["table"].clamp(min=0).long()].double().transpose(1, 2)             # [rows][kv-heads][blocks][channels]
    score = (s["q"].double().view(n, hkv, hq // hkv, hd) @ means.transpose(-1, -2)).amax(2)
    blocks = torch.arange(s["table"].shape[1], device="cuda")
    score = torch.where(blocks < last[:, None, None], score, -math.inf)
    order = torch.sort(score, dim=-1, descending=True, stable=True)[1][..., :take - 1]
    order = torch.where(order < last[:, None, None], order, 1 << 30)
    order = torch.cat((order, last[:, None, None].expand(n, hkv, 1)), -1).sort(-1)[0]
    got = order.shape[-1]
    s["ids"].fill_(-1)
    s["ids"][..., :got] = torch.where(order < 1 << 30, order, -1)
    ids = s["ids"].long()
    heads = torch.arange(hkv, device="cuda")[None, :, None]
    pages = torch.gather(s["table"][:, None].expand(n, hkv, -1).long(), 2, ids.clamp(min=0)).clamp(min=0)
    keys, values = (x[pages, heads].float().reshape(n, hkv, -1, hd) for x in (s["k"], s["v"]))
    at = (ids[..., None] * page + torch.arange(page, device="cuda")).reshape(n, hkv, -1)
    see = (at >= 0) & (at <= s["pos"][:, None, None])
    x = (s["q"].float().view(n, hkv, hq // hkv, hd) * s["qscale"]) @ keys.transpose(-1, -2)
    p, total = _weights(x, see[:, :, None, :])
    s["o16"].copy_((p @ values / total).view(n, hq, hd))
    return [s["ids"], s["o16"]]


# ---------------------------------------------------------------------------------------------------------------- one pass
def run(s):
    if own:
        from yasakani_b200 import paged
        if s["kind"] == "append":
            hq, hkv = s["hq"], s["k"].shape[1]
            paged.launch_append(s["cache"], s["table"], s["qkv"][:, hq:hq + hkv], s["qkv"][:, hq + hkv:], s["seq"], s["pos"], s["rope"], s["rd"],
                                q=s["qkv"][:, :hq], q_out=s["q_out"])
            return [s["q_out"], s["k"], s["v"], s["kmean"]]
        if s["kind"] == "sparse":
            paged.launch_select(s["q"], s["cache"], s["table"], s["seq"], s["pos"], s["ids"], s["ws"])
            paged.launch_attention(s["q"], s["cache"], s["table"], s["seq"], s["pos"], s["qscale"], s["o16"], s["ws"], blocks=s["ids"])
            return [s["ids"], s["o16"]]
        paged.launch_attention(s["q"], s["cache"], s["table"], s["seq"], s["pos"], s["qscale"], s["o16"], s["ws"], shared=s["shared"])
        return s["o16"]
    return _append(s) if s["kind"] == "append" else _sparse(s) if s["kind"] == "sparse" else _attend(s)


# ---------------------------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    """The definitions row by row: softmax over the keys that a row sees; the sums, angles and means as they stand."""
    s = prepare(case, seed)
    hq, hkv, hd, page = (case[x] for x in ("hq", "hkv", "hd", "page"))
    k, v, table = s["k"].double(), s["v"].double(), s["table"].long()
    seq, pos = s["seq"].tolist(), s["pos"].tolist()
    if case["kind"] == "append":
        z = torch.view_as_complex(s["rope"].double())[s["pos"].long()][:, None, :]
        x, half = s["qkv"].double(), s["rd"] // 2
        y = torch.complex(x[..., :half], x[..., half:2 * half]) * z
        x = torch.cat((torch.cat((y.real, y.imag, x[..., 2 * half:]), -1)[:, :hq + hkv], x[:, hq + hkv:]), 1)
        kmean = s["kmean"].double()
        where = table[s["seq"].long(), s["pos"].long() // page].tolist()
        flat_k, flat_v = (t.permute(0, 2, 1, 3).reshape(-1, hkv, hd).clone() for t in (k, v))           # a row for each (page, place)
        place = torch.tensor([w * page + p % page for w, p in zip(where, pos)], device="cuda")
        flat_k[place], flat_v[place] = x[:, hq:hq + hkv], x[:, hq + hkv:]
        k, v = (t.view(-1, page, hkv, hd).permute(0, 2, 1, 3).contiguous() for t in (flat_k, flat_v))
        rounded = k.to(s["k"].dtype).double()                                                           # what the cache holds
        for w, p in zip(where, pos):
            if p % page == page - 1:
                kmean[w] = rounded[w].mean(1)
        return [x[:, :hq].contiguous(), k, v, kmean]
    q, o = s["q"].double() * s["qscale"], torch.zeros((len(pos), hq, hd), dtype=torch.float64, device="cuda")
    ids = torch.full((len(pos), hkv, s["take"]), -1, dtype=torch.int64, device="cuda")
    for r, (b, p) in enumerate(zip(seq, pos)):
        for h in range(hkv):
            mine = q[r, h * (hq // hkv):(h + 1) * (hq // hkv)]
            blocks = torch.arange(p // page + 1, device="cuda")
            if case["kind"] == "sparse":
                score = (s["kmean"][table[b, :p // page], h].double() @ mine.T).amax(1) if p >= page else torch.zeros(0, device="cuda")
                best = torch.argsort(score, descending=True, stable=True)[:s["take"] - 1].sort()[0]
                blocks = torch.cat((best, blocks[-1:]))
                ids[r, h, :len(blocks)] = blocks
            rows = (blocks[:, None] * page + torch.arange(page, device="cuda")).view(-1) <= p
            keys, values = (t[table[b, blocks], h].reshape(-1, hd)[rows] for t in (k, v))
            o[r, h * (hq // hkv):(h + 1) * (hq // hkv)] = torch.softmax(mine @ keys.T, -1) @ values
    return [ids, o] if case["kind"] == "sparse" else o


# ---------------------------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    hq, hkv, hd, page, kind = (case[x] for x in ("hq", "hkv", "hd", "page", "kind"))
    row = 2 * hkv * hd                                           # bytes of one token's keys, or values
    if kind == "append":
        starts, rows = _ints(case["starts"]), _ints(case["rows"])
        T, rd = sum(rows), HEADS[(hq, hkv, hd)][0]
        done = sum((a + n) // page - a // page for a, n in zip(starts, rows))
        before = sum(a % page for a, n in zip(starts, rows) if (a + n) // page > a // page)             # rows of completed pages that were there already
        # rows in and out, each position's angles once, two indexes a row; for a page's mean the rows that this pass does not bring itself
        return {"bytes": T * (2 * (2 * row + 2 * hq * hd) + 8) + min(T, max(a + n for a, n in zip(starts, rows))) * rd * 4 + before * row + done * row,
                "flops": T * (hq + hkv) * rd * 3 + done * page * hkv * hd}
    ctx, io, shared = _ints(case["contexts"]), 4 * hq * hd, case.get("shared", 0)
    n = len(ctx)
    if kind == "sparse":
        blocks = [(c - 1) // page for c in ctx]                  # complete pages in front of the last
        seen = [min(case["take"] - 1, b) * page + c - b * page for b, c in zip(blocks, ctx)]
        return {"bytes": sum(blocks) * row + 2 * row * sum(seen) + n * (io + 4 * hkv * case["take"]), "flops": 2 * hq * hd * sum(blocks) + 4 * hq * hd * sum(seen)}
    return {"bytes": 2 * row * (sum(ctx) + shared) + n * io, "flops": 4 * hq * hd * (sum(ctx) + n * shared)}
