"""The paged cache's entries refuse what their documentation does not allow, before anything is launched (no GPU needed)."""
import ctypes as C

import pytest
import torch

from yasakani_b200 import _lib, paged

A = 1 << 20                                                      # an address that is aligned and never followed


def cache(**change):
    c = _lib.PagedCacheC(A, A, A, 100, 4, 64, 256, 1)
    c.ready = 1
    for k, v in change.items():
        setattr(c, k, v)
    return c


def rows(**change):
    r = _lib.PagedRowsC(A, 3, 16, A, A, 5)
    for k, v in change.items():
        setattr(r, k, v)
    return r


def call(name, c, r, a):
    L = _lib.load()
    rc = getattr(L, name)(C.byref(c) if c is not None else None, C.byref(r) if r is not None else None, C.byref(a) if a is not None else None, None)
    return rc, L.yskn_kv4_last_error().decode()


def append_args(**change):
    a = _lib.PagedAppendArgsC(A, A, A, A, 1024, 1024, 24 * 256, A, 4096, 64, 24)
    for k, v in change.items():
        setattr(a, k, v)
    return a


def select_args(**change):
    a = _lib.PagedSelectArgsC(A, 24 * 256, 24, 8, A, A, 1 << 40)
    for k, v in change.items():
        setattr(a, k, v)
    return a


def attn_args(**change):
    a = _lib.PagedAttnArgsC(A, 24 * 256, 24, 0.06, A, 0, None, 0, A, 1 << 40)
    for k, v in change.items():
        setattr(a, k, v)
    return a


ENTRIES = [("yskn_kv4_paged_append", append_args), ("yskn_kv4_paged_select", select_args), ("yskn_kv4_paged_attention", attn_args)]


def test_struct_layouts():
    assert _lib.PagedCacheC.dtype.offset == 40 and _lib.PagedCacheC.maps.offset == 48 and C.sizeof(_lib.PagedCacheC) == 560
    assert _lib.PagedRowsC.seq.offset == 16 and C.sizeof(_lib.PagedRowsC) == 40
    assert _lib.PagedAppendArgsC.rope.offset == 56 and C.sizeof(_lib.PagedAppendArgsC) == 80
    assert _lib.PagedSelectArgsC.ids.offset == 24 and C.sizeof(_lib.PagedSelectArgsC) == 48
    assert _lib.PagedAttnArgsC.o16.offset == 24 and _lib.PagedAttnArgsC.ids.offset == 40 and C.sizeof(_lib.PagedAttnArgsC) == 72


@pytest.mark.parametrize("name,args", ENTRIES)
@pytest.mark.parametrize("change,text", [
    (dict(k=None), "null cache array"), (dict(hd=64), "head_dim"), (dict(page=48), "page of 48"), (dict(dtype=2), "F16 or BF16"), (dict(pages=0), "bad shape"),
    (dict(kvh=0), "bad shape"), (dict(pages=1 << 24), "bad shape"), (dict(v=A + 8), "16-byte aligned"), (dict(ready=0), "paged_init")])
def test_caches_that_are_refused(name, args, change, text):
    rc, msg = call(name, cache(**change), rows(), args())
    assert rc == -1 and text in msg and msg.startswith(name)


@pytest.mark.parametrize("name,args", ENTRIES)
@pytest.mark.parametrize("change,text", [
    (dict(table=None), "null buffer"), (dict(seq=None), "null buffer"), (dict(pos=None), "null buffer"), (dict(rows=-1), "rows -1"), (dict(seqs=0), "bad table"),
    (dict(blocks=0), "bad table"), (dict(blocks=1 << 25), "bad table")])
def test_rows_that_are_refused(name, args, change, text):
    rc, msg = call(name, cache(), rows(**change), args())
    assert rc == -1 and text in msg


@pytest.mark.parametrize("name,args", ENTRIES)
def test_nothing_to_do_and_nothing_at_all(name, args):
    assert call(name, cache(), rows(rows=0), args())[0] == 0
    for c, r, a in ((None, rows(), args()), (cache(), None, args()), (cache(), rows(), None)):
        rc, msg = call(name, c, r, a)
        assert rc == -1 and "null" in msg


@pytest.mark.parametrize("change,text", [
    (dict(k_in=None), "null buffer"), (dict(q_out=None), "null buffer"), (dict(rd=8), "rotary width 8"), (dict(rd=272), "rotary width 272"), (dict(rd=-16), "rotary width"),
    (dict(rope=None), "needs a rope table"), (dict(rope_rows=0), "needs a rope table"), (dict(k_in=A + 2), "16-byte aligned"), (dict(v_stride=1028), "16-byte aligned"),
    (dict(k_stride=1016), "16-byte aligned"), (dict(q_out=A + 8), "16-byte aligned"), (dict(nh=0), "bad queries"), (dict(q_stride=23 * 256), "bad queries")])
def test_append_refuses(change, text):
    rc, msg = call("yskn_kv4_paged_append", cache(), rows(), append_args(**change))
    assert rc == -1 and text in msg


@pytest.mark.parametrize("change,text", [
    (dict(q=None), "null buffer"), (dict(ids=None), "null buffer"), (dict(take=1), "take 1"), (dict(take=1025), "take 1025"), (dict(nh=25), "25 heads"), (dict(nh=68), "68 heads"),
    (dict(q=A + 8), "16-byte aligned"), (dict(q_stride=24 * 256 + 4), "multiple of 8"), (dict(workspace_bytes=5 * 4 * 16 * 16 - 1), "workspace of"),
    (dict(workspace=None), "workspace of"), (dict(workspace=A + 64), "256-byte aligned")])
def test_select_refuses(change, text):
    rc, msg = call("yskn_kv4_paged_select", cache(), rows(), select_args(**change))
    assert rc == -1 and text in msg
    assert "mean keys" in call("yskn_kv4_paged_select", cache(kmean=None), rows(), select_args())[1]
    assert "65535" in call("yskn_kv4_paged_select", cache(), rows(rows=65536), select_args())[1]


@pytest.mark.parametrize("change,text", [
    (dict(q=None), "null buffer"), (dict(o16=None), "o16"), (dict(o16=A + 4), "o16"), (dict(nh=0), "0 heads"), (dict(nh=4 * 17), "68 heads"), (dict(shared=100), "shared part of 100"),
    (dict(shared=-64), "shared part"), (dict(shared=17 * 64), "shared part"), (dict(shared=64, ids=A, take=4), "exclude"), (dict(ids=A, take=0), "take 0"),
    (dict(workspace_bytes=1000), "workspace of"), (dict(workspace=A + 16), "256-byte aligned")])
def test_attention_refuses(change, text):
    rc, msg = call("yskn_kv4_paged_attention", cache(), rows(), attn_args(**change))
    assert rc == -1 and text in msg


def test_a_line_beyond_32_bits_is_refused():
    rc, msg = call("yskn_kv4_paged_attention", cache(kvh=1024, page=64), rows(rows=60000, blocks=1 << 20), attn_args(nh=1024, q_stride=1024 * 256))
    assert rc == -1 and "too many for one call" in msg


def test_workspace_serves_fewer_rows_and_tokens():
    L = _lib.load()
    for kvh, nh, hd in ((4, 24, 256), (4, 28, 128), (16, 16, 128), (2, 32, 256)):
        c = cache(kvh=kvh, hd=hd)
        size = lambda n, s, b=0: L.yskn_kv4_paged_workspace_bytes(C.byref(c), n, nh, s, b)
        most = 0
        for n in list(range(1, 200)) + [500, 65535]:
            for s in (0, 64, 64 * 37, 64 * 512):
                assert 0 < size(n, s) <= size(n, 64 * 512)
            assert size(n, 64 * 512) >= most
            most = size(n, 64 * 512)
        assert size(5, 0, 10 ** 6) >= 16 * 5 * kvh * 10 ** 6
    for bad in ((0, 24, 0, 0), (65536, 24, 0, 0), (1, 23, 0, 0), (1, 24, 65, 0), (1, 24, -64, 0), (1, 24, 0, -1)):
        assert L.yskn_kv4_paged_workspace_bytes(C.byref(cache()), *bad) == 0


def test_python_refuses():
    k = torch.zeros((4, 2, 64, 128), dtype=torch.bfloat16)
    with pytest.raises(AssertionError):
        paged.PagedCache.of(k, k)                                # host memory
    with pytest.raises(TypeError):
        paged.PagedCache.of(k.float(), k.float())
    with pytest.raises(TypeError):
        paged.PagedCache.of(k, k.half())
    with pytest.raises(ValueError):
        paged.PagedCache.of(k, k[:2])
    with pytest.raises(ValueError):
        paged.PagedCache.of(k, k, k[:, :, 0, :64])
    for name, n in (("paged_append", 12), ("paged_select", 9), ("paged_attention", 12)):
        with pytest.raises(TypeError):
            getattr(_lib.host, name)(1, 2, 3)
        with pytest.raises(AttributeError):
            getattr(_lib.host, name)(*[None] * n)
    with pytest.raises(TypeError):                               # no struct of a cache
        _lib.host.paged_select(b"x" * 16, k, *[torch.zeros(1, dtype=torch.int32)] * 3, k, k, k, None)
