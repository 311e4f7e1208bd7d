"""Attention over the paged cache at values that ordinary inputs do not hold: infinities and NaN that a query sees,
magnitudes at the end of f32's range, and weights far below the largest one."""
import math

import pytest
import torch

import paged_util as P
from vantablack_b200 import ops

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
DTYPES = [F32, F16, BF16]
F32_MAX = 3.4028234663852886e38


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def put(cache, which, s, t, head, d, value):
    """Position t of sequence s, in the pages and in the host's rows."""
    pages, rows = (cache.k, cache.k_rows) if which == "k" else (cache.v, cache.v_rows)
    pages[int(cache.table[s, t // cache.page]), head, t % cache.page, d] = value
    rows[s][t, head, d] = value


def bound(ref, n, dtype, extra=0.0):
    """attention_tolerance with P as exact as in decode, for sums whose steps the tensor cores may cut off (2^-23 of
    the sum so far, two steps per 16 positions) where it counts rounded ones."""
    out, a, b = ref
    return P.attention_tolerance(out, a, b, n, dtype, False) + a * (n / 8) * 2.0 ** -23 + extra


def decode(cache, q, **kw):
    got = ops.paged_attention_decode(q, cache.k, cache.v, cache.table, cache.d_lens, **kw)
    ops.check_device_error()
    return got


def decode_all(cache, q, s, **kw):
    """Every row of q as the new token of sequence s."""
    n = q.shape[0]
    got = ops.paged_attention_decode(q, cache.k, cache.v, cache.table[s:s + 1].repeat(n, 1), cache.d_lens[s:s + 1].repeat(n), **kw)
    ops.check_device_error()
    return got


def prefill(cache, q, s, n, **kw):
    """The last n tokens of sequence s alone."""
    got = ops.paged_attention_prefill(q, cache.k, cache.v, cache.table[s:s + 1], cache.d_lens[s:s + 1], i32(0, n), **kw)
    ops.check_device_error()
    return got


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_prefill_infinities_where_all_rows_see_them(dtype, hd, value):
    """In tiles that all rows see, with weights down to nothing: scores of 24 (nats) standard deviation."""
    cache = P.Cache([1000], 2, hd, 16, dtype, 75)
    at = [100, 130, 500]
    for t in at:
        put(cache, "v", 0, t, 1, 5, value)
    n = 90
    q = torch.randn(n, 8, hd, generator=torch.Generator().manual_seed(8)).to(dtype).cuda()
    scale = 24.0 / math.sqrt(hd)
    got = prefill(cache, q, 0, n, scale=scale).double().cpu()
    hit = got[:, 4:, 5]
    assert bool(torch.isnan(hit).all()) if math.isnan(value) else bool((hit == value).all())
    for t in at:
        cache.v_rows[0][t, 1, 5] = 0.0
    ref = P.attention(q.double().cpu(), cache.k_rows[0].double(), cache.v_rows[0].double(), torch.arange(910, 1000), scale)
    ok = (got - ref[0]).abs() <= P.attention_tolerance(*ref, 1000, dtype, True)
    ok[:, 4:, 5] = True
    assert bool(ok.all())


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads,n,length,window,sinks", [(8, 700, 700, 0, 0), (6, 130, 1500, 0, 0), (4, 400, 2000, 300, 4), (2, 3, 6000, 0, 0)])
def test_prefill_keeps_the_weights_exact(dtype, hd, heads, n, length, window, sinks):
    """16-bit caches: the output carries its own rounding only, not one of each weight."""
    cache = P.Cache([length], 2, hd, 16, dtype, 76)
    q = torch.randn(n, heads, hd, generator=torch.Generator().manual_seed(9)).to(dtype).cuda()
    got = prefill(cache, q, 0, n, window=window, sinks=sinks).double().cpu()
    ref = P.attention(q.double().cpu(), cache.k_rows[0].double(), cache.v_rows[0].double(), torch.arange(length - n, length),
                      hd ** -0.5, window, sinks)
    assert bool(((got - ref[0]).abs() <= bound(ref, length, dtype)).all())


# What a weight of an f16 cache is held to, as a share of the row's largest: f16 ends at steps of 2^-24, half a step
# off at most, and weights are kept times 2^15 (decode) and 2^13 (prefill, whose running maximum may lag by 2 bits).
F16_STEP = {"decode": 2.0 ** -40, "prefill": 2.0 ** -38}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nats", [12.0, 15.0, 18.0])
@pytest.mark.parametrize("where", ["first", "middle"])
def test_many_small_weights_beside_a_large_one(dtype, nats, where):
    """One key far above all others, its value 0: the output is made of the small weights alone."""
    length, hd, n = 20000, 64, 5
    cache = P.Cache([length], 1, hd, 64, dtype, 77)
    g = torch.Generator().manual_seed(10)
    at = 0 if where == "first" else 11111
    k = torch.zeros(length, 1, hd)
    k[:, 0, 1:] = 0.02 * torch.randn(length, hd - 1, generator=g)  # the others differ a little
    k[at, 0, 0] = nats
    v = torch.rand(length, 1, hd, generator=g) + 0.5
    v[at] = 0.0
    cache.k_rows[0], cache.v_rows[0] = k.to(dtype), v.to(dtype)
    t = torch.arange(length)
    pg = cache.table[0].cpu().long()[t // 64].cuda()
    cache.k[pg, :, (t % 64).cuda()] = cache.k_rows[0].cuda()
    cache.v[pg, :, (t % 64).cuda()] = cache.v_rows[0].cuda()
    q = torch.randn(n, 4, hd, generator=g)
    q[:, :, 0] = 1.0
    q = q.to(dtype).cuda()
    pos = torch.arange(length - n, length)
    ref = P.attention(q.double().cpu(), cache.k_rows[0].double(), cache.v_rows[0].double(), pos, 1.0)
    for what, got in (("prefill", prefill(cache, q, 0, n, scale=1.0)), ("decode", decode(cache, q[-1:], scale=1.0))):
        r = ref if what == "prefill" else tuple(x[-1:] for x in ref)
        small = length * F16_STEP[what] * 1.5 if dtype == F16 else 0.0
        err = (got.double().cpu() - r[0]).abs()
        tol = bound(r, length, dtype, small)
        assert bool((err <= tol).all()), f"{what}: {float((err / tol).max()):.2f} of the bound"


def test_decode_small_weights_within_a_warp():
    """As above where a warp walks its positions alone: more sequences (of one prompt's pages) than CTAs."""
    length, hd, n = 1000, 64, 320
    cache = P.Cache([length], 2, hd, 64, F16, 79)
    g = torch.Generator().manual_seed(12)
    k = torch.zeros(length, 2, hd)
    k[:, :, 1:] = 0.02 * torch.randn(length, 2, hd - 1, generator=g)
    k[3, :, 0] = 18.0
    v = torch.rand(length, 2, hd, generator=g) + 0.5
    v[3] = 0.0
    cache.k_rows[0], cache.v_rows[0] = k.to(F16), v.to(F16)
    t = torch.arange(length)
    pg = cache.table[0].cpu().long()[t // 64].cuda()
    cache.k[pg, :, (t % 64).cuda()] = cache.k_rows[0].cuda()
    cache.v[pg, :, (t % 64).cuda()] = cache.v_rows[0].cuda()
    q = torch.randn(n, 8, hd, generator=g)
    q[:, :, 0] = 1.0
    q = q.to(F16).cuda()
    got = ops.paged_attention_decode(q, cache.k, cache.v, cache.table.repeat(n, 1), cache.d_lens.repeat(n), scale=1.0)
    ops.check_device_error()
    ref = P.attention(q.double().cpu(), cache.k_rows[0].double(), cache.v_rows[0].double(), torch.full((n,), length - 1), 1.0)
    err, tol = (got.double().cpu() - ref[0]).abs(), bound(ref, length, F16, length * F16_STEP["decode"] * 1.5)
    assert bool((err <= tol).all()), f"{float((err / tol).max()):.2f} of the bound"
