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
