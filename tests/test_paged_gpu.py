"""Paged key-value cache on the GPU (vtb_cuda_paged_*) against plain 64-bit
forms: single-token and chunk attention with sliding window and sinks, append
with RoPE, page copies and compaction, and a run of them together."""
import math

import pytest
import torch

import paged_util as P
from vantablack_b200 import _lib, ops

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
DTYPES = [F32, F16, BF16]
P_ROUNDED = {"decode": False, "prefill": True}  # 16-bit prefill: P is one value of the type


def check_rows(got, cache, s, q, pos, scale, window, sinks, what):
    out, a, b = P.attention(q.double().cpu(), cache.k_rows[s].double(), cache.v_rows[s].double(), pos, scale, window,
                            sinks)
    tol = P.attention_tolerance(out, a, b, cache.lens[s], cache.dtype, P_ROUNDED[what])
    err = (got.double().cpu() - out).abs()
    assert torch.isfinite(got.float()).all(), f"sequence {s}: not finite"
    assert bool((err <= tol).all()), f"sequence {s}: error {err.max():.3g}, {float((err / tol).max()):.2f} of the bound"


def run_decode(cache, heads, hd, window=0, sinks=0, scale=None, seed=5, q=None, **kw):
    g = torch.Generator().manual_seed(seed)
    if q is None:
        q = torch.randn(len(cache.lens), heads, hd, generator=g).to(cache.dtype).cuda()
    got = ops.paged_attention_decode(q, cache.k, cache.v, cache.table, cache.d_lens, scale=scale, window=window,
                                     sinks=sinks, **kw)
    ops.check_device_error()
    for s, n in enumerate(cache.lens):
        check_rows(got[s:s + 1], cache, s, q[s:s + 1], torch.tensor([n - 1]), scale or hd ** -0.5, window, sinks, "decode")
    return q, got


# ---- decode ----

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("heads,kv", [(4, 4), (8, 1), (28, 4), (24, 2), (40, 2), (6, 2)])
def test_decode_heads(dtype, hd, heads, kv):
    run_decode(P.Cache([1, 0, 17, 64, 65, 130, 391, 16], kv, hd, 16, dtype, 1), heads, hd)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("page", [1, 2, 8, 32, 64, 256, 1024])
def test_decode_page_sizes(dtype, page):
    run_decode(P.Cache([1, 63, 300, 129], 2, 128, page, dtype, 2), 8, 128)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 3), (64, 4), (100, 0), (128, 70), (5000, 9)])
def test_decode_window(dtype, window, sinks):
    run_decode(P.Cache([1, 5, 64, 65, 133, 0, 700], 2, 64, 16, dtype, 3), 8, 64, window, sinks)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens", [[20011], [9001, 3, 0, 4097], [1] * 70, [64] * 600, [0, 0, 0]])
def test_decode_splits(dtype, lens):
    """One long sequence cut into many parts, ragged lengths, more sequences than CTAs, nothing at all."""
    run_decode(P.Cache(lens, 2, 64, 16, dtype, 4), 10, 64)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["nhd", "mixed"])
def test_decode_strides(dtype, layout):
    """Other orders of the cache's strides; q a slice of a fused projection row; out inside a larger buffer."""
    cache = P.Cache([33, 190, 2], 4, 128, 8, dtype, 5, layout=layout)
    g = torch.Generator().manual_seed(9)
    qkv = torch.randn(3, 16 + 8, 128, generator=g).to(dtype).cuda()
    buf = torch.full((3, 20, 136), 7.0, dtype=dtype, device="cuda")
    _, got = run_decode(cache, 16, 128, q=qkv[:, :16], out=buf[:, 2:18, :128])
    assert bool((buf[:, :2] == 7).all() and (buf[:, 18:] == 7).all() and (buf[:, :, 128:] == 7).all())


def test_decode_unread_entries_may_hold_anything():
    """Pages left behind by the window have been given back: their entries hold -1 and 2^30."""
    cache = P.Cache([500, 40], 2, 64, 16, BF16, 6)
    want = run_decode(cache, 8, 64, window=50, sinks=2)[1]
    cache.table[0, 1:28] = torch.tensor([-1, 2 ** 30] * 13 + [-1], dtype=torch.int32, device="cuda")
    got = run_decode(cache, 8, 64, window=50, sinks=2)[1]
    assert torch.equal(got, want)


def test_decode_scale_and_large_scores():
    """Scores far apart (the running maximum moves by hundreds) and a negative scale."""
    cache = P.Cache([300], 1, 64, 16, F32, 7)
    run_decode(cache, 4, 64, scale=3.0)
    run_decode(cache, 4, 64, scale=-0.25)


def test_decode_same_result_every_time():
    cache = P.Cache([3000, 17, 900], 4, 128, 16, BF16, 8)
    q, first = run_decode(cache, 16, 128)
    for _ in range(5):
        again = ops.paged_attention_decode(q, cache.k, cache.v, cache.table, cache.d_lens)
        assert torch.equal(again, first)


def test_decode_captured_with_growing_lengths():
    """One captured call replayed while the lengths grow: the plan is made on the device."""
    cache = P.Cache([700, 90], 2, 64, 16, BF16, 9)
    q = torch.randn(2, 8, 64, device="cuda").to(BF16)
    lens = torch.tensor([1, 1], dtype=torch.int32, device="cuda")
    ws = ops.paged_attention_workspace(BF16, 8, 2, 64)
    out = torch.empty_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        ops.paged_attention_decode(q, cache.k, cache.v, cache.table, lens, out=out, workspace=ws)
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            ops.paged_attention_decode(q, cache.k, cache.v, cache.table, lens, out=out, workspace=ws)
    for now in ([1, 1], [64, 90], [0, 65], [700, 3]):
        lens.copy_(torch.tensor(now, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        for s, n in enumerate(now):
            ref, a, b = P.attention(q[s:s + 1].double().cpu(), cache.k_rows[s][:n].double(), cache.v_rows[s][:n].double(),
                                    torch.tensor([n - 1]), 0.125)
            tol = P.attention_tolerance(ref, a, b, n, BF16, P_ROUNDED["decode"])
            assert bool(((out[s:s + 1].double().cpu() - ref).abs() <= tol).all())
    ops.check_device_error()


def test_decode_two_streams_with_a_workspace_each():
    caches = [P.Cache([2500, 40], 2, 64, 16, F32, 10 + i) for i in range(2)]
    qs = [torch.randn(2, 8, 64, device="cuda") for _ in range(2)]
    want = [ops.paged_attention_decode(q, c.k, c.v, c.table, c.d_lens) for q, c in zip(qs, caches)]
    ws = [ops.paged_attention_workspace(F32, 8, 2, 64) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                c = caches[i]
                outs[i].append(ops.paged_attention_decode(qs[i], c.k, c.v, c.table, c.d_lens, workspace=ws[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in outs[i])


def test_bad_pages_and_lengths_set_the_error_word():
    """A page id outside the cache and a length beyond the table are reported, and the next call is right."""
    cache = P.Cache([100, 20], 2, 64, 16, BF16, 11)
    q = torch.randn(2, 8, 64, device="cuda").to(BF16)
    for bad in (-1, cache.n_pages, 2 ** 31 - 1):
        table = cache.table.clone()
        table[0, 2] = bad
        good = ops.paged_attention_decode(q, cache.k, cache.v, table, cache.d_lens)
        with pytest.raises(_lib.VtbError):
            ops.check_device_error()
        ref = P.attention(q[1:].double().cpu(), cache.k_rows[1].double(), cache.v_rows[1].double(), torch.tensor([19]), 0.125)
        assert bool(((good[1:].double().cpu() - ref[0]).abs() <= P.attention_tolerance(*ref, 20, BF16, False)).all())
    ops.paged_attention_decode(q, cache.k, cache.v, cache.table, torch.tensor([2 ** 31 - 1, 20], dtype=torch.int32, device="cuda"))
    with pytest.raises(_lib.VtbError):
        ops.check_device_error()
    run_decode(cache, 8, 64)


# ---- prefill ----

def run_prefill(cache, counts, heads, hd, window=0, sinks=0, scale=None, pad=0, seed=6, **kw):
    """counts[s] new tokens at the end of each sequence; `pad` rows behind the last stay as they were."""
    g = torch.Generator().manual_seed(seed)
    total = sum(counts)
    q = torch.randn(total + pad, heads, hd, generator=g).to(cache.dtype).cuda()
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    out = torch.full((total + pad, heads, hd), 7.0, dtype=cache.dtype, device="cuda")
    got = ops.paged_attention_prefill(q, cache.k, cache.v, cache.table, cache.d_lens,
                                      torch.tensor(starts, dtype=torch.int32, device="cuda"), scale=scale, window=window,
                                      sinks=sinks, out=out, **kw)
    ops.check_device_error()
    for s, n in enumerate(counts):
        if n:
            a, b = starts[s], starts[s + 1]
            check_rows(got[a:b], cache, s, q[a:b], torch.arange(cache.lens[s] - n, cache.lens[s]),
                       scale or hd ** -0.5, window, sinks, "prefill")
    assert bool((got[total:] == 7).all())
    return q, got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("heads,kv", [(4, 4), (8, 1), (28, 4), (24, 2), (6, 2)])
def test_prefill_heads(dtype, hd, heads, kv):
    run_prefill(P.Cache([1, 0, 50, 200, 129, 300], kv, hd, 16, dtype, 21), [1, 0, 50, 77, 1, 260], heads, hd, pad=3)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("page", [1, 2, 8, 32, 128, 512])
def test_prefill_page_sizes(dtype, page):
    run_prefill(P.Cache([33, 300], 2, 128, page, dtype, 22), [33, 130], 8, 128)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 3), (64, 4), (100, 0), (128, 70), (130, 200), (5000, 9)])
def test_prefill_window(dtype, window, sinks):
    run_prefill(P.Cache([600, 5, 301], 2, 64, 16, dtype, 23), [450, 5, 20], 8, 64, window, sinks)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("counts,ctx", [([2], [9000]), ([1] * 40, list(range(40))), ([700], [0]), ([300, 1, 40], [2000, 5000, 0])])
def test_prefill_shapes(dtype, counts, ctx):
    """Few rows over a long context, many single tokens, a prompt, a mixed step."""
    run_prefill(P.Cache([a + b for a, b in zip(counts, ctx)], 2, 64, 16, dtype, 24), counts, 6, 64)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["nhd", "mixed"])
def test_prefill_strides(dtype, layout):
    run_prefill(P.Cache([150, 333], 4, 128, 8, dtype, 25, layout=layout), [150, 40], 16, 128)


@pytest.mark.parametrize("dtype", DTYPES)
def test_prefill_large_scores(dtype):
    cache = P.Cache([400], 1, 64, 16, dtype, 26)
    for scale in (2.0, -0.3):
        run_prefill(cache, [390], 4, 64, scale=scale)


@pytest.mark.parametrize("dtype", DTYPES)
def test_zero_scale_is_the_mean(dtype):
    cache = P.Cache([40, 200], 2, 64, 16, dtype, 30)
    run_prefill(cache, [40, 33], 8, 64, scale=1e-30)
    run_decode(cache, 8, 64, scale=1e-30)
    q = torch.randn(2, 8, 64, device="cuda").to(dtype)
    i32 = lambda *n: torch.tensor(n, dtype=torch.int32, device="cuda")  # noqa: E731
    got = (ops.paged_attention_decode(q, cache.k, cache.v, cache.table, cache.d_lens, scale=0.0),
           ops.paged_attention_prefill(q, cache.k, cache.v, cache.table, cache.d_lens, i32(0, 1, 2), scale=0.0))
    for s in range(2):
        mean = cache.v_rows[s].double().mean(0).repeat_interleave(4, 0)
        for g in got:
            assert torch.allclose(g[s].double().cpu(), mean, rtol=2 * P.EPS[dtype], atol=2 * P.EPS[dtype])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [2, 16])
@pytest.mark.parametrize("window,sinks", [(0, 0), (70, 5)])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_prefill_hidden_infinities_and_nans(dtype, page, window, sinks, value):
    """K and V of some tokens of the chunk are not finite: the queries that do not see them are as without them.
    (Sequence 0: 210 new tokens on 40; 1: one new token, over a split.)"""
    cache = P.Cache([250, 1300], 2, 64, page, dtype, 35)
    at = [45, 100, 101, 233]
    for t in at:
        pg, slot = int(cache.table[0, t // page]), t % page
        cache.k[pg, :, slot, 3] = value
        cache.v[pg, 1, slot, 5] = value
    g = torch.Generator().manual_seed(2)
    q = torch.randn(211, 8, 64, generator=g).to(dtype).cuda()
    got = ops.paged_attention_prefill(q, cache.k, cache.v, cache.table, cache.d_lens,
                                      torch.tensor([0, 210, 211], dtype=torch.int32, device="cuda"), window=window, sinks=sinks)
    ops.check_device_error()
    pos = torch.arange(40, 250)
    see = P.visible(pos, torch.tensor(at), window, sinks).any(1)
    assert bool(see.any()) and not bool(see.all())
    ref, a, b = P.attention(q[:210].double().cpu(), cache.k_rows[0].double(), cache.v_rows[0].double(), pos, 0.125, window, sinks)
    tol = P.attention_tolerance(ref, a, b, 250, dtype, P_ROUNDED["prefill"])
    clean = ~see
    assert bool(((got[:210].double().cpu() - ref).abs() <= tol)[clean].all())
    assert not bool(torch.isfinite(got[:210].float().cpu()[see][:, 4:]).all())  # kv head 1's queries that see them
    check_rows(got[210:], cache, 1, q[210:], torch.tensor([1299]), 0.125, window, sinks, "prefill")


def test_prefill_rows_before_the_first_position_give_zeros():
    """A chunk longer than the sequence's length: its first rows see nothing."""
    cache = P.Cache([10], 1, 64, 16, BF16, 27)
    q = torch.randn(16, 4, 64, device="cuda").to(BF16)
    got = ops.paged_attention_prefill(q, cache.k, cache.v, cache.table, cache.d_lens,
                                      torch.tensor([0, 16], dtype=torch.int32, device="cuda"))
    assert bool((got[:6] == 0).all())
    check_rows(got[6:], cache, 0, q[6:], torch.arange(10), 0.125, 0, 0, "prefill")


def test_prefill_bad_starts_set_the_error_word():
    cache = P.Cache([30, 30], 1, 64, 16, F32, 28)
    q = torch.randn(20, 2, 64, device="cuda")
    for bad in ([0, 25, 20], [-4, 10, 20], [0, 10, 21], [12, 10, 20]):
        ops.paged_attention_prefill(q, cache.k, cache.v, cache.table, cache.d_lens,
                                    torch.tensor(bad, dtype=torch.int32, device="cuda"))
        with pytest.raises(_lib.VtbError):
            ops.check_device_error()
    run_prefill(cache, [10, 10], 2, 64)


def test_prefill_of_single_tokens_equals_decode():
    cache = P.Cache([1, 70, 333], 2, 64, 16, F32, 29)
    q, got = run_decode(cache, 8, 64, 40, 3)
    pre = ops.paged_attention_prefill(q, cache.k, cache.v, cache.table, cache.d_lens,
                                      torch.arange(4, dtype=torch.int32, device="cuda"), window=40, sinks=3)
    assert torch.allclose(pre, got, rtol=2e-5, atol=2e-6)


# ---- append ----

def rope_table(n, hd, base=10000.0):
    ang = torch.arange(n).double()[:, None] / base ** (torch.arange(0, hd, 2).double() / hd)
    return torch.stack((ang.cos(), ang.sin()), -1).reshape(n, hd).float()


def rotate(x, rope, pos):
    """Interleaved pairs of x [rows, heads, hd] at positions pos, in float64 from the f32 inputs."""
    z = x.double().reshape(*x.shape[:2], -1, 2)
    c = rope[pos].double().reshape(x.shape[0], 1, -1, 2)
    return torch.stack((z[..., 0] * c[..., 0] - z[..., 1] * c[..., 1], z[..., 0] * c[..., 1] + z[..., 1] * c[..., 0]),
                       -1).reshape(x.shape), (z.abs().sum(-1, keepdim=True).expand_as(z)).reshape(x.shape)


@pytest.mark.parametrize("x,dtype", [(F32, F32), (F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("hd,page,layout", [(64, 16, "hnd"), (128, 1, "nhd"), (128, 64, "mixed")])
@pytest.mark.parametrize("with_rope", [True, False])
def test_append(x, dtype, hd, page, layout, with_rope):
    cache = P.Cache([40, 7, 90], 3, hd, page, dtype, 31, slack=5.0, layout=layout)
    g = torch.Generator().manual_seed(3)
    seq = torch.tensor([2, 0, 1, -1, 0, 2], dtype=torch.int32)
    pos = torch.tensor([89, 0, 6, 3, 39, -7], dtype=torch.int32)  # two padding rows
    rows = torch.randn(6, 7 + 6, hd, generator=g).to(x)
    rope = rope_table(90, hd)
    before_k, before_v = cache.k.cpu().clone(), cache.v.cpu().clone()
    d = rows.cuda()
    q_out = torch.full((6, 7, hd), 3.0, dtype=dtype, device="cuda")
    ops.paged_append(cache.k, cache.v, cache.table, d[:, 7:10], d[:, 10:], seq.cuda(), pos.cuda(), q=d[:, :7], q_out=q_out,
                     rope=rope.cuda() if with_rope else None)
    ops.check_device_error()
    y, size = rotate(rows[:, :10], rope, pos.clamp(min=0).long()) if with_rope else (rows[:, :10].double(), rows[:, :10].double() * 0)
    # two products and a sum in f32, then half a step of the type
    tol = size * 3 * 2.0 ** -24 + (y.abs() + size * 2.0 ** -22) * P.EPS[dtype] / 2 + (2.0 ** -25 if dtype == F16 else 0)
    want_k, want_v = before_k.clone(), before_v.clone()
    got_k, got_v = cache.k.cpu(), cache.v.cpu()
    for r in range(6):
        if seq[r] < 0 or pos[r] < 0:
            assert bool((q_out[r] == 3).all())
            continue
        pg, slot = int(cache.table[seq[r], pos[r] // page]), int(pos[r]) % page
        assert bool(((q_out[r].cpu().double() - y[r, :7]).abs() <= tol[r, :7]).all())
        assert bool(((got_k[pg, :, slot].double() - y[r, 7:]).abs() <= tol[r, 7:]).all())
        assert torch.equal(got_v[pg, :, slot], rows[r, 10:].to(dtype))
        want_k[pg, :, slot], want_v[pg, :, slot] = got_k[pg, :, slot], got_v[pg, :, slot]
    assert torch.equal(got_k, want_k) and torch.equal(got_v, want_v)  # nothing else was written


def test_append_in_place_and_without_q():
    cache = P.Cache([40], 2, 64, 16, BF16, 32, slack=0.0)
    rope = rope_table(40, 64).cuda()
    q = torch.randn(5, 4, 64, device="cuda").to(BF16)
    k, v = torch.randn(5, 2, 64, device="cuda").to(BF16), torch.randn(5, 2, 64, device="cuda").to(BF16)
    seq, pos = torch.zeros(5, dtype=torch.int32, device="cuda"), torch.arange(9, 14, dtype=torch.int32, device="cuda")
    want = ops.paged_append(cache.k, cache.v, cache.table, k, v, seq, pos, q=q, rope=rope)
    ck, cv = cache.k.clone(), cache.v.clone()
    assert ops.paged_append(cache.k, cache.v, cache.table, k, v, seq, pos, rope=rope) is None
    got = ops.paged_append(cache.k, cache.v, cache.table, k, v, seq, pos, q=q, q_out=q, rope=rope)
    assert got is q and torch.equal(q, want) and torch.equal(ck, cache.k) and torch.equal(cv, cache.v)
    none = torch.empty(0, 2, 64, device="cuda").to(BF16)
    e = torch.empty(0, dtype=torch.int32, device="cuda")
    ops.paged_append(cache.k, cache.v, cache.table, none, none, e, e)
    assert torch.equal(ck, cache.k)


@pytest.mark.parametrize("seq,pos", [(2, 0), (0, 48), (0, 40), (1, 20)])
def test_append_out_of_range_is_reported_and_not_written(seq, pos):
    """A sequence or position beyond the table, a position beyond rope (40 rows), an entry without a page."""
    cache = P.Cache([48, 10], 1, 64, 16, F32, 33, slack=0.0)
    before = cache.k.clone(), cache.v.clone()
    x = torch.randn(1, 1, 64, device="cuda")
    i = lambda n: torch.tensor([n], dtype=torch.int32, device="cuda")  # noqa: E731
    ops.paged_append(cache.k, cache.v, cache.table, x, x, i(seq), i(pos), rope=rope_table(40, 64).cuda())
    with pytest.raises(_lib.VtbError):
        ops.check_device_error()
    assert torch.equal(before[0], cache.k) and torch.equal(before[1], cache.v)


# ---- page copies ----

@pytest.mark.parametrize("dtype,hd,page,layers", [(F32, 64, 1, 1), (BF16, 128, 64, 3), (F16, 64, 8, 5), (F32, 128, 256, 2)])
@pytest.mark.parametrize("layout", ["hnd", "nhd"])
def test_copy_pages(dtype, hd, page, layers, layout):
    g = torch.Generator().manual_seed(41)
    shape = (layers, 11, 3, page, hd) if layout == "hnd" else (layers, 11, page, 3, hd)
    k, v = (torch.randn(shape, generator=g).to(dtype).cuda() for _ in range(2))
    if layout == "nhd":
        k, v = k.transpose(2, 3), v.transpose(2, 3)
    src, dst = torch.tensor([7, 7, 0, 10], dtype=torch.int32), torch.tensor([1, 3, 9, 2], dtype=torch.int32)
    want_k, want_v = k.clone(), v.clone()
    want_k[:, dst.long()], want_v[:, dst.long()] = k[:, src.long()], v[:, src.long()]
    ops.paged_copy(k, v, src.cuda(), dst.cuda())
    ops.check_device_error()
    assert torch.equal(k, want_k) and torch.equal(v, want_v)


def test_copy_one_layer_and_none():
    k, v = torch.randn(4, 1, 16, 64, device="cuda"), torch.randn(4, 1, 16, 64, device="cuda")
    i = lambda *n: torch.tensor(n, dtype=torch.int32, device="cuda")  # noqa: E731
    a, b = k.clone(), v.clone()
    ops.paged_copy(k, v, i(), i())
    assert torch.equal(a, k)
    ops.paged_copy(k, v, i(2), i(0))
    a[0], b[0] = a[2], b[2]
    assert torch.equal(a, k) and torch.equal(b, v)


def test_compaction_rewrites_tables():
    g = torch.Generator().manual_seed(42)
    k, v = torch.randn(2, 40, 2, 16, 64, generator=g).cuda(), torch.randn(2, 40, 2, 16, 64, generator=g).cuda()
    big = torch.randint(-3, 40, (300, 37), generator=g).to(torch.int32)
    big[big < 0] = -1
    table = big.cuda()
    part = table[:, 2:35]  # rows with a stride of their own
    src, dst = torch.tensor([39, 30, 33], dtype=torch.int32), torch.tensor([0, 5, 1], dtype=torch.int32)
    page_map = torch.arange(40, dtype=torch.int32)
    page_map[src.long()] = dst
    want = big.clone()
    w = want[:, 2:35]
    w[w >= 0] = page_map[w[w >= 0].long()]
    want_k = k.clone()
    want_k[:, dst.long()] = k[:, src.long()]
    ops.paged_copy(k, v, src.cuda(), dst.cuda(), page_table=part, page_map=page_map.cuda())
    ops.check_device_error()
    assert torch.equal(table.cpu(), want) and torch.equal(k, want_k)


def test_copy_bad_ids_are_reported_and_skipped():
    k, v = torch.randn(2, 4, 1, 16, 64, device="cuda"), torch.randn(2, 4, 1, 16, 64, device="cuda")
    a = k.clone()
    i = lambda *n: torch.tensor(n, dtype=torch.int32, device="cuda")  # noqa: E731
    ops.paged_copy(k, v, i(4, 1, 2), i(0, -1, 3))
    with pytest.raises(_lib.VtbError):
        ops.check_device_error()
    a[:, 3] = a[:, 2]
    assert torch.equal(a, k)
    table = torch.tensor([[0, 9, -1]], dtype=torch.int32, device="cuda")
    ops.paged_copy(k, v, i(), i(), page_table=table, page_map=i(3, 1, 2, 0))
    with pytest.raises(_lib.VtbError):
        ops.check_device_error()
    assert table.tolist() == [[3, 9, -1]]


# ---- together ----

@pytest.mark.parametrize("dtype", DTYPES)
def test_prompt_fork_decode_compact(dtype):
    """A prompt in two chunks, a fork with a private copy of the tail page, different tokens in each branch, a
    compaction, more tokens: every output against contiguous 64-bit attention over the rows that were written."""
    heads, kv, hd, page, layers = 8, 2, 64, 16, 2
    g = torch.Generator().manual_seed(51)
    k, v = (torch.full((layers, 24, kv, page, hd), float("nan"), dtype=dtype, device="cuda") for _ in range(2))
    table = torch.full((2, 6), -1, dtype=torch.int32)
    table[0, :6] = torch.tensor([20, 3, 17, 9, 22, 11])
    rope = rope_table(96, hd).cuda()
    hist = {(layer, s): ([], []) for layer in range(layers) for s in range(2)}
    lens = [0, 0]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731

    def step(counts):
        n = sum(counts)
        seq = [s for s in range(2) for _ in range(counts[s])]
        pos = [lens[s] + i for s in range(2) for i in range(counts[s])]
        for s in range(2):
            lens[s] += counts[s]
        for layer in range(layers):
            rows = torch.randn(n, heads + 2 * kv, hd, generator=g).cuda()
            tab = table.cuda()
            q = ops.paged_append(k[layer], v[layer], tab, rows[:, heads:heads + kv], rows[:, heads + kv:], i32(seq), i32(pos),
                                 q=rows[:, :heads], rope=rope)
            if max(counts) == 1 and min(counts) == 1:
                got = ops.paged_attention_decode(q, k[layer], v[layer], tab, i32(lens))
                what = "decode"
            else:
                got = ops.paged_attention_prefill(q, k[layer], v[layer], tab, i32(lens), i32([0, counts[0], n]))
                what = "prefill"
            ops.check_device_error()
            at = 0
            for s in range(2):
                for i in range(counts[s]):
                    p = lens[s] - counts[s] + i
                    pg = int(table[s, p // page])
                    hist[layer, s][0].append(k[layer, pg, :, p % page].cpu())
                    hist[layer, s][1].append(v[layer, pg, :, p % page].cpu())
                if counts[s]:
                    kk, vv = (torch.stack(x).double() for x in hist[layer, s])
                    ref, a, b = P.attention(q[at:at + counts[s]].double().cpu(), kk, vv,
                                            torch.arange(lens[s] - counts[s], lens[s]), hd ** -0.5)
                    tol = P.attention_tolerance(ref, a, b, lens[s], dtype, P_ROUNDED[what])
                    assert bool(((got[at:at + counts[s]].double().cpu() - ref).abs() <= tol).all())
                    at += counts[s]

    step([30, 0])
    step([23, 0])  # 53 positions: pages 0..2 full, 5 slots of page 3
    table[1, :4] = torch.tensor([20, 3, 17, 5])  # the fork shares the full pages
    table[1, 4:6] = torch.tensor([0, 14])
    ops.paged_copy(k, v, i32([9]), i32([5]))
    lens[1] = lens[0]
    for layer in range(layers):
        hist[layer, 1] = (list(hist[layer, 0][0]), list(hist[layer, 0][1]))
    for _ in range(13):  # both branches pass into their next page
        step([1, 1])
    src, dst = [20, 17, 22, 14], [1, 2, 4, 6]
    page_map = torch.arange(24, dtype=torch.int32)
    page_map[torch.tensor(src)] = torch.tensor(dst, dtype=torch.int32)
    tab = table.cuda()
    ops.paged_copy(k, v, i32(src), i32(dst), page_table=tab, page_map=page_map.cuda())
    for p in src:
        k[:, p], v[:, p] = math.nan, math.nan  # the pages that were left hold nothing any more
    table = tab.cpu()
    for _ in range(3):
        step([1, 1])
    step([7, 2])


def test_no_sequences_and_no_rows():
    cache = P.Cache([20, 3], 2, 64, 16, BF16, 61)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    none = torch.empty(0, 8, 64, dtype=BF16, device="cuda")
    got = ops.paged_attention_decode(none, cache.k, cache.v, cache.table[:0], cache.d_lens[:0])
    assert got.shape == none.shape
    got = ops.paged_attention_prefill(none, cache.k, cache.v, cache.table, cache.d_lens, i32([0, 0, 0]))
    assert got.shape == none.shape
    got = ops.paged_attention_prefill(none, cache.k, cache.v, cache.table[:0], cache.d_lens[:0], i32([0]))
    assert got.shape == none.shape


@pytest.mark.parametrize("dtype", DTYPES)
def test_longest_window_and_sinks(dtype):
    """The largest window and sinks an int holds see what no window sees; rows before the first position give zeros."""
    cache = P.Cache([150, 9], 2, 64, 16, dtype, 62)
    top = 2 ** 31 - 1
    for w, n in ((top, 0), (top, top), (1, top)):
        q, got = run_decode(cache, 8, 64)
        assert torch.equal(got, run_decode(cache, 8, 64, w, n)[1])
        q, got = run_prefill(cache, [140, 9], 8, 64)
        if w == top:
            assert torch.equal(got, run_prefill(cache, [140, 9], 8, 64, w, n)[1])
        else:
            run_prefill(cache, [140, 9], 8, 64, w, n)
    q = torch.randn(40, 8, 64, device="cuda").to(dtype)
    starts = torch.tensor([0, 0, 40], dtype=torch.int32, device="cuda")
    want = ops.paged_attention_prefill(q, cache.k, cache.v, cache.table, cache.d_lens, starts)
    got = ops.paged_attention_prefill(q, cache.k, cache.v, cache.table, cache.d_lens, starts, window=top, sinks=top)
    assert torch.equal(got, want) and not got[:31].any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_captured_chunk_step(dtype):
    """Append and chunk attention in one captured graph, first called there, replayed with other rows, positions and
    lengths; a second graph with its own workspace runs in between."""
    heads, kv, hd, page, n = 12, 4, 64, 8, 37
    cache = P.Cache([400, 300], kv, hd, page, dtype, 63)
    g = torch.Generator().manual_seed(64)
    side, graphs = torch.cuda.Stream(), []
    for _ in range(2):
        rows = torch.zeros(n, heads + 2 * kv, hd, device="cuda")
        seq, pos = (torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(2))
        lens, starts = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
        out = torch.empty(n, heads, hd, dtype=dtype, device="cuda")
        ws = ops.paged_attention_workspace(dtype, heads, kv, hd)
        q = torch.empty(n, heads, hd, dtype=dtype, device="cuda")
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            ops.paged_append(cache.k, cache.v, cache.table, rows[:, heads:heads + kv], rows[:, heads + kv:], seq, pos,
                             q=rows[:, :heads], q_out=q)
            ops.paged_attention_prefill(q, cache.k, cache.v, cache.table, lens, starts, out=out, workspace=ws)
        graphs.append((graph, rows, seq, pos, lens, starts, out, q))
    for turn, (first, counts) in enumerate([((300, 40), (20, 17)), ((0, 263), (0, 37)), ((50, 7), (36, 1)), ((363, 0), (37, 0))]):
        graph, rows, seq, pos, lens, starts, out, q = graphs[turn % 2]
        x = torch.randn(n, heads + 2 * kv, hd, generator=g)
        rows.copy_(x)
        seq.copy_(torch.tensor([s for s in range(2) for _ in range(counts[s])], dtype=torch.int32))
        pos.copy_(torch.tensor([first[s] + i for s in range(2) for i in range(counts[s])], dtype=torch.int32))
        now = [first[s] + counts[s] for s in range(2)]
        lens.copy_(torch.tensor(now, dtype=torch.int32))
        starts.copy_(torch.tensor([0, counts[0], n], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        at = 0
        for s in range(2):
            c = counts[s]
            cache.k_rows[s][first[s]:now[s]] = x[at:at + c, heads:heads + kv].to(dtype)
            cache.v_rows[s][first[s]:now[s]] = x[at:at + c, heads + kv:].to(dtype)
            if c:
                ref, a, b = P.attention(q[at:at + c].double().cpu(), cache.k_rows[s][:now[s]].double(),
                                        cache.v_rows[s][:now[s]].double(), torch.arange(first[s], now[s]), hd ** -0.5)
                tol = P.attention_tolerance(ref, a, b, now[s], dtype, P_ROUNDED["prefill"])
                assert bool(((out[at:at + c].double().cpu() - ref).abs() <= tol).all())
            at += c
    ops.check_device_error()


def test_default_workspaces_on_two_streams():
    """Calls without a workspace of their own on two streams at once, chunk and single-token attention."""
    caches = [P.Cache([1900, 40], 2, 128, 64, BF16, 70 + i) for i in range(2)]
    qd = [torch.randn(2, 8, 128, device="cuda").to(BF16) for _ in range(2)]
    qp = [torch.randn(50, 8, 128, device="cuda").to(BF16) for _ in range(2)]
    starts = torch.tensor([0, 30, 50], dtype=torch.int32, device="cuda")
    call = lambda i: (ops.paged_attention_decode(qd[i], caches[i].k, caches[i].v, caches[i].table, caches[i].d_lens),  # noqa: E731
                      ops.paged_attention_prefill(qp[i], caches[i].k, caches[i].v, caches[i].table, caches[i].d_lens, starts))
    want = [call(i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                outs[i].append(call(i))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(d, want[i][0]) and torch.equal(p, want[i][1]) for d, p in outs[i])
    ops.check_device_error()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [2, 16])
@pytest.mark.parametrize("window,sinks", [(0, 0), (70, 5)])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_prefill_infinities_and_nans_of_v_reach_their_values_only(dtype, page, window, sinks, value):
    """One value of some V rows is not finite: the queries that see it get it in that value, every other value is as if
    it were 0.  (Sequence 0: 210 new tokens on 40, also split over CTAs by a call of its own; the bad rows lie before the
    chunk, inside it and at its end.)"""
    cache = P.Cache([250, 1300], 2, 64, page, dtype, 36)
    at = [2, 45, 100, 101, 233, 249]
    for t in at:
        cache.v[int(cache.table[0, t // page]), 1, t % page, 5] = value
        cache.v_rows[0][t, 1, 5] = 0.0
    g = torch.Generator().manual_seed(3)
    q = torch.randn(211, 8, 64, generator=g).to(dtype).cuda()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    got = ops.paged_attention_prefill(q, cache.k, cache.v, cache.table, cache.d_lens, i32(0, 210, 211), window=window, sinks=sinks)
    alone = ops.paged_attention_prefill(q[205:210], cache.k, cache.v, cache.table[:1], cache.d_lens[:1], i32(0, 5),
                                        window=window, sinks=sinks)
    ops.check_device_error()
    for out, first in ((got[:210], 40), (alone, 245)):
        pos = torch.arange(first, 250)
        see = P.visible(pos, torch.tensor(at), window, sinks).any(1)
        x = out.double().cpu()
        ref, a, b = P.attention(q[first - 40:210].double().cpu(), cache.k_rows[0].double(), cache.v_rows[0].double(), pos, 0.125,
                                window, sinks)
        ok = (x - ref).abs() <= P.attention_tolerance(ref, a, b, 250, dtype, P_ROUNDED["prefill"])
        bad = x[see][:, 4:, 5]  # kv head 1's queries that see one
        assert bool(torch.isnan(bad).all()) if math.isnan(value) else bool((bad == value).all())
        ok[:, 4:, 5] |= see[:, None]
        assert bool(ok.all())
    check_rows(got[210:], cache, 1, q[210:], torch.tensor([1299]), 0.125, window, sinks, "prefill")
