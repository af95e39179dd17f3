"""Paged attention where one key outweighs all others by 2^20 to 2^27 and its value is zero in half of the channels, so that those channels are carried by a
long tail of small weights.

Tolerance.  As in test_gpu_paged.py, but for the rounding of a weight to 16 bits.  In bf16 it is relative (h = 2^-8) over the whole range.  fp16 has that (h = 2^-11) down to 2^-14 and
steps of 2^-24 below, and the kernels round p 2^s, s = 15 where a row attends by itself and 7 behind a shared part, against a reference that is never above the row's
largest score: a weight is off by h p + 2^-25-s, in units of the largest weight, and the row by 2^-32 sum |v| / l more, l >= 1, with the smaller s for both."""
import math

import pytest
import torch

from test_gpu_paged import DT, attend, half_step, ints

pytestmark = pytest.mark.gpu


def check(o16, q, keys, values, scale, what):
    """q [nh][hd], keys / values [kvh][n][hd] in fp64."""
    nh, hd = q.shape
    kvh, n, _ = keys.shape
    h = half_step(o16.dtype)
    x = torch.einsum("hgc,hnc->hgn", q.view(kvh, -1, hd), keys) * scale
    w = torch.softmax(x, -1)
    want, mag = (w @ values).reshape(nh, hd), (w @ values.abs()).reshape(nh, hd)
    total = values.abs().sum(1).repeat_interleave(nh // kvh, 0)
    S = float((q.view(kvh, -1, hd).abs() @ keys.abs().transpose(1, 2)).max() * abs(scale) * math.log2(math.e))
    e = (hd + 4) * 2.0 ** -23 * S
    tiny = 2.0 ** -32 * total if o16.dtype == torch.float16 else 0.0
    bound = h * want.abs() + (1 + h) * (h + 2 * (2 * e + 2.0 ** -20) + n * 2.0 ** -23) * mag + tiny + 2.0 ** -24
    err = (o16.double() - want).abs()
    assert (err <= bound).all(), (what, float((err / bound).max()))
    return want, bound


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("shared", [0, 1920])
@pytest.mark.parametrize("nh,hkv,hd", [(4, 2, 128), (24, 4, 256), (32, 2, 128), (64, 8, 128)])
@pytest.mark.parametrize("at", ["first", "middle", "last"])
@pytest.mark.parametrize("count", [1, 120])                      # a row's tokens on many CTAs; pairs that lie in one
@pytest.mark.parametrize("sink,spread", [(2.25, 0.5), (2.34375, 0.0625)])      # q k = 8 sink against 8 * [0, spread): 2^20.2 to 2^26 between them; 2^26.3 to 2^27
def test_a_long_tail_behind_one_key(dt, shared, nh, hkv, hd, at, count, sink, spread):
    page, own = 64, 130 if shared else 1500
    n, g = shared + own, torch.Generator(device="cuda").manual_seed(hd + nh + shared)
    pages = -(-n // page)
    k = torch.randn((pages, hkv, page, hd), generator=g, device="cuda") * 2.0 ** -8
    k[..., 0] = torch.rand(k.shape[:-1], generator=g, device="cuda") * spread
    v = (torch.rand(k.shape, generator=g, device="cuda") + 0.5) * 1000.0                    # of one sign: the tail adds up
    i = {"first": 0, "middle": n // 2, "last": n - 1}[at]
    k[i // page, :, i % page, 0] = sink
    v[i // page, :, i % page, :hd // 2] = 0.0
    k, v = k.to(DT[dt]), v.to(DT[dt])
    q = torch.randn((count, nh, hd), generator=g, device="cuda") * 2.0 ** -6
    q[..., 0] = 8.0
    q = q.to(DT[dt])
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None].contiguous()
    o16, _ = attend(k, v, table, ints([0] * count), ints([n - 1] * count), q, 1.0, shared=shared)
    keys, values = (t.transpose(0, 1).reshape(hkv, -1, hd)[:, :n].double() for t in (k, v))
    for r in sorted({0, count // 2, count - 1}):
        want, bound = check(o16[r], q[r].double(), keys, values, 1.0, r)
        tail = want[:, :hd // 2]
        assert (tail > 20 * bound[:, :hd // 2]).all()            # nothing at all in these channels would be far outside


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("shared", [0, 1920])
@pytest.mark.parametrize("size", [4.0, 512.0, 2048.0])
def test_scores_that_fp32_holds_in_large_steps(dt, shared, size):
    """Scores up to about 2^9, 2^23 and 2^27: at the largest an fp32 score is off by whole powers of two, so that nobody can say which of the highest keys counts, but what
    comes out is a mean of values with weights that sum to 1, each rounded by half a step at most: it lies between the least and the largest value, up to 2 h."""
    g = torch.Generator(device="cuda").manual_seed(int(size))
    n, hkv, nh, hd, h = shared + 200, 2, 14, 128, half_step(DT[dt])
    k = (torch.randn((-(-n // 64), hkv, 64, hd), generator=g, device="cuda") * size).to(DT[dt])
    v = (torch.rand(k.shape, generator=g, device="cuda") + 1.0).to(DT[dt])
    q = (torch.randn((3, nh, hd), generator=g, device="cuda") * size).to(DT[dt])
    for scale in (1.0, -1.0):
        o16, _ = attend(k, v, torch.arange(k.shape[0], dtype=torch.int32, device="cuda")[None].contiguous(), ints([0] * 3), ints([n - 1] * 3), q, scale, shared=shared)
        assert (o16 >= 1.0 - 2 * h).all() and (o16 <= 2.0 * (1 + 2 * h)).all(), (float(o16.min()), float(o16.max()))


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("shared", [0, 640])
@pytest.mark.parametrize("at", [3, 600, 700])
@pytest.mark.parametrize("what", [float("nan"), float("inf")])
def test_a_score_that_is_not_finite_is_not_lost(dt, shared, at, what):
    """A softmax with a score that is no number, or infinite, has no value: the heads that see such a key say so, rows that end in front of it and the other kv-head do not."""
    g = torch.Generator(device="cuda").manual_seed(at)
    n, hkv, nh, hd = 800, 2, 14, 128
    k = torch.randn((-(-n // 64), hkv, 64, hd), generator=g, device="cuda").to(DT[dt])
    v = torch.randn(k.shape, generator=g, device="cuda").to(DT[dt])
    k[at // 64, 1, at % 64, 5] = what
    q = torch.randn((3, nh, hd), generator=g, device="cuda").to(DT[dt])
    q[..., 5] = 1.0
    o16, _ = attend(k, v, torch.arange(k.shape[0], dtype=torch.int32, device="cuda")[None].contiguous(), ints([0] * 3), ints([n - 1, at, at - 1]), q, 0.1, shared=shared)
    assert torch.isnan(o16[:2, nh // 2:]).all()
    assert torch.isfinite(o16[:, :nh // 2]).all()
    assert torch.isfinite(o16[2]).all()
