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


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd,heads", [(64, 8), (128, 8), (64, 24), (128, 40)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (70, 5)])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_decode_infinities_and_nans_of_v_reach_their_values_only(dtype, hd, heads, window, sinks, value):
    """As in prefill: a query that sees a V row with such a value gets it there; every other value is as if it were 0.
    The sequences lie within one CTA, and over many."""
    cache = P.Cache([250, 40, 9001, 1], 2, hd, 16, dtype, 71)
    bad = {0: [2, 45, 249], 2: [3, 4000, 8999], 3: [0]}
    for s, at in bad.items():
        for t in at:
            put(cache, "v", s, t, 1, 5, value)
    q = torch.randn(4, heads, hd, generator=torch.Generator().manual_seed(4)).to(dtype).cuda()
    got = decode(cache, q, window=window, sinks=sinks).double().cpu()
    for s, at in bad.items():
        n = cache.lens[s]
        see = P.visible(torch.tensor([n - 1]), torch.tensor(at), window, sinks)
        assert bool(see.any())
        for t in at:
            cache.v_rows[s][t, 1, 5] = 0.0
        ref = P.attention(q[s:s + 1].double().cpu(), cache.k_rows[s].double(), cache.v_rows[s].double(), torch.tensor([n - 1]),
                          hd ** -0.5, window, sinks)
        ok = (got[s:s + 1] - ref[0]).abs() <= bound(ref, n, dtype)
        hit = got[s, heads // 2:, 5]  # kv head 1's queries
        assert bool(torch.isnan(hit).all()) if math.isnan(value) else bool((hit == value).all())
        ok[:, heads // 2:, 5] = True
        assert bool(ok.all())
    assert bool(torch.isfinite(got[1]).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_of_both_signs_make_nan(dtype):
    cache = P.Cache([300], 2, 64, 16, dtype, 72)
    put(cache, "v", 0, 20, 0, 7, math.inf)
    put(cache, "v", 0, 200, 0, 7, -math.inf)
    q = torch.randn(30, 8, 64, generator=torch.Generator().manual_seed(5)).to(dtype).cuda()
    for got in (decode(cache, q[-1:]), prefill(cache, q, 0, 30)):
        bad = ~torch.isfinite(got)
        assert bool(torch.isnan(got[:, :4, 7]).all())
        bad[:, :4, 7] = False
        assert not bool(bad.any())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("scale", [0.125, -0.2])
@pytest.mark.parametrize("what", ["decode", "prefill"])
def test_infinities_of_k(dtype, hd, scale, what):
    """A score of -inf has the weight 0: the query is as if it did not see the position.  A score of inf gives NaN.
    Positions in tiles that all rows see, at the edge, and in the rest of the cache."""
    cache = P.Cache([700, 33], 2, hd, 16, dtype, 73)
    at = [5, 300, 655]
    for t in at:
        put(cache, "k", 0, t, 1, 3, math.inf)
    n = 60 if what == "prefill" else 6
    q = torch.randn(n, 6, hd, generator=torch.Generator().manual_seed(6)).to(dtype)
    q[:, :, 3] = q[:, :, 3].abs().clamp(min=0.1) * torch.where(torch.arange(n) % 3 == 0, 1.0, -1.0).to(dtype)[:, None]
    q = q.cuda()
    if what == "prefill":
        rows, pos = prefill(cache, q, 0, n, scale=scale).double().cpu(), torch.arange(640, 700)
    else:
        rows, pos = decode_all(cache, q, 0, scale=scale).double().cpu(), torch.full((n,), 699)
    qq = q.double().cpu()
    up = (qq[:, 0, 3] * scale > 0)  # the score of such a position is +inf
    assert bool(up.any()) and not bool(up.all())
    assert bool(torch.isnan(rows[up][:, 3:]).all())
    # the others: what is left of the cache without these positions
    keep = torch.tensor([t for t in range(700) if t not in at])
    for r in torch.nonzero(~up).flatten().tolist():
        t = keep[keep <= pos[r]]
        k, v = cache.k_rows[0].double()[t, 1:], cache.v_rows[0].double()[t, 1:]
        ref = P.attention(qq[r:r + 1, 3:], k, v, torch.tensor([len(t) - 1]), scale)
        assert bool(((rows[r:r + 1, 3:] - ref[0]).abs() <= bound(ref, 700, dtype)).all()), r
    ref = P.attention(qq[:, :3], cache.k_rows[0].double()[:, :1], cache.v_rows[0].double()[:, :1], pos, scale)
    assert bool(((rows[:, :3] - ref[0]).abs() <= bound(ref, 700, dtype)).all())  # kv head 0 has none


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("huge", [F32_MAX, -F32_MAX, 3.4027e38, 1e38])
@pytest.mark.parametrize("what", ["decode", "prefill"])
def test_f32_values_at_the_end_of_the_range(hd, huge, what):
    """Finite values whose leading part would round to infinity.  V: hidden ones stay hidden, seen ones count with their
    weight.  K: a query that is 0 there is as if they were, one that is not (a score of -1e7) as if it did not see them."""
    cache = P.Cache([400, 90], 2, hd, 16, F32, 74)
    for t in (10, 390):
        put(cache, "v", 0, t, 1, 9, huge)
    for t in (30, 395):
        put(cache, "k", 0, t, 0, 2, huge)
    for head in range(2):  # the largest weight is another position's: sums of the huge values stay in range
        put(cache, "k", 0, 1, head, 0, 90.0)
    n = 50 if what == "prefill" else 4
    q = torch.randn(n, 8, hd, generator=torch.Generator().manual_seed(7))
    q[:, :, 0] = 1.0
    q[:, :, 2] = torch.where(torch.arange(n) % 2 == 0, 0.0, -1e-30 * (1 if huge > 0 else -1))[:, None]
    q = q.cuda()
    if what == "prefill":
        rows, pos = prefill(cache, q, 0, n).double().cpu(), torch.arange(350, 400)
    else:
        rows, pos = decode_all(cache, q, 0).double().cpu(), torch.full((n,), 399)
    qq = q.double().cpu()
    assert bool(torch.isfinite(rows).all())
    k, v = cache.k_rows[0].double(), cache.v_rows[0].double()
    for r in range(n):
        t = torch.arange(int(pos[r]) + 1)
        if qq[r, 0, 2] != 0:
            t = t[(t != 30) & (t != 395)]
        got = rows[r:r + 1] if qq[r, 0, 2] == 0 else rows[r:r + 1, :4]  # (kv head 0's queries)
        ref = P.attention(qq[r:r + 1, :got.shape[1]], k[t, :2 if got.shape[1] == 8 else 1], v[t, :2 if got.shape[1] == 8 else 1],
                          torch.tensor([len(t) - 1]), hd ** -0.5)
        # a leading part cut off instead of rounded: 2^-19 of the terms in place of 2^-20
        assert bool(((got - ref[0]).abs() <= bound(ref, 400, F32) + ref[1] * 2.0 ** -19).all()), r


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


def test_infinities_at_both_ends_of_a_long_context():
    """f32: two bad V rows far apart cost a look at the rows between them, not a walk of every row's thread."""
    length, n = 8704, 512
    cache = P.Cache([length], 8, 128, 64, F32, 78)
    q = torch.randn(n, 32, 128, generator=torch.Generator().manual_seed(11)).cuda()
    starts = i32(0, n)

    def time():
        best = math.inf
        for _ in range(4):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            torch.cuda.synchronize()
            a.record()
            got = ops.paged_attention_prefill(q, cache.k, cache.v, cache.table, cache.d_lens, starts)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        ops.check_device_error()
        return best, got

    clean, want = time()
    put(cache, "v", 0, 1, 1, 5, math.inf)
    put(cache, "v", 0, length - n, 1, 6, -math.inf)
    slow, got = time()
    assert bool((got[:, 4:8, 5] == math.inf).all() and (got[:, 4:8, 6] == -math.inf).all())
    got[:, 4:8, 5:7] = want[:, 4:8, 5:7]
    assert torch.equal(got, want)
    assert slow <= 10 * clean, f"{slow:.3f} ms, {clean:.3f} without"


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nats", [2.0, 5.0])
def test_large_values_where_the_maximum_grows(dtype, hd, nats):
    """V next to the end of the range at a position whose score is above all before it: its weight is 1 at most."""
    length, n = 700, 40
    cache = P.Cache([length], 2, hd, 16, dtype, 80)
    at = 600
    for head in range(2):
        for t in range(length):
            cache.k_rows[0][t, head, 0] = 0.0
        put(cache, "k", 0, at, head, 0, nats)
    pg = cache.table[0].cpu().long()[torch.arange(length) // 16].cuda()
    cache.k[pg, :, torch.arange(length).cuda() % 16, 0] = cache.k_rows[0][:, :, 0].cuda()
    put(cache, "v", 0, at, 1, 7, 3.0e38)
    q = torch.zeros(n, 8, hd)
    q[:, :, 0] = 1.0
    q[:, :, 1:] = 0.02 * torch.randn(n, 8, hd - 1, generator=torch.Generator().manual_seed(13))
    q = q.to(dtype).cuda()
    pos = torch.arange(length - n, length)
    ref = P.attention(q.double().cpu(), cache.k_rows[0].double(), cache.v_rows[0].double(), pos, 1.0)
    for r, got in ((ref, prefill(cache, q, 0, n, scale=1.0)), (tuple(x[-1:] for x in ref), decode(cache, q[-1:], scale=1.0))):
        err = (got.double().cpu() - r[0]).abs()
        assert bool(torch.isfinite(got.float()).all()) and bool((err <= bound(r, length, dtype)).all())
