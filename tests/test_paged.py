"""Host-side checks of the paged cache entry points: bad calls are refused
before any launch (no GPU needed)."""
import ctypes as C

import pytest

from vantablack_b200 import _lib, build


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


@pytest.fixture()
def buf():
    b = C.create_string_buffer(4096)
    return b, (C.addressof(b) + 255) & ~255


def kv_args(p, **kw):
    a = dict(k=p, v=p, type=30, n_kv_heads=2, head_dim=64, page_size=16, n_pages=4, page_stride=2048, head_stride=1024,
             slot_stride=64, page_table=p, table_stride=3, n_seqs=2, pages_per_seq=3)
    a.update(kw)
    return _lib.PagedKv(*[a[n] for n, _ in _lib.PagedKv._fields_])


def attn_args(p, lib, **kw):
    a = dict(q=p, out=p, q_row_stride=512, q_head_stride=64, out_row_stride=512, out_head_stride=64, n_heads=8, window=0,
             sinks=0, scale=0.125, lens=p, workspace=p, workspace_bytes=1 << 30)
    a.update(kw)
    return _lib.PagedAttn(*[a[n] for n, _ in _lib.PagedAttn._fields_])


def rows_args(p, **kw):
    a = dict(type=0, n_heads=8, n_rows=2, k=p, v=p, q=p, k_row_stride=128, k_head_stride=64, v_row_stride=128,
             v_head_stride=64, q_row_stride=512, q_head_stride=64, q_out=p, rope=p, n_rope=8, seq=p, pos=p)
    a.update(kw)
    return _lib.PagedRows(*[a[n] for n, _ in _lib.PagedRows._fields_])


BAD_KV = [(dict(k=None), -1), (dict(type=8), -8), (dict(head_dim=80), -8), (dict(page_size=12), -1), (dict(page_size=0), -1),
          (dict(page_size=2048), -1), (dict(n_kv_heads=0), -1), (dict(n_pages=0), -1), (dict(n_pages=1 << 31), -1),
          (dict(page_stride=-8), -1), (dict(slot_stride=65), -1), (dict(head_stride=1 << 50), -1)]
BAD_TABLE = [(dict(page_table=None), -1), (dict(n_seqs=0), -1), (dict(pages_per_seq=0), -1), (dict(table_stride=2), -1),
             (dict(pages_per_seq=(1 << 26) + 1, table_stride=1 << 30), -1)]


@pytest.mark.parametrize("bad,status", BAD_KV + BAD_TABLE)
def test_bad_cache_is_refused(lib, buf, bad, status):
    p = buf[1]
    kv = kv_args(p, **bad)
    a, r = attn_args(p, lib), rows_args(p)
    assert lib.vtb_cuda_paged_attn_decode(C.byref(kv), C.byref(a), None) == status
    assert lib.vtb_cuda_paged_attn_prefill(C.byref(kv), C.byref(a), p, 4, None) == status
    assert lib.vtb_cuda_paged_append(C.byref(kv), C.byref(r), None) == status
    if (bad, status) in BAD_KV:
        assert lib.vtb_cuda_paged_copy(C.byref(kv), 1, 0, p, p, 1, None, None, None) == status


@pytest.mark.parametrize("bad", [dict(q=None), dict(out=None), dict(q_row_stride=5), dict(out_head_stride=32), dict(n_heads=7),
                                 dict(n_heads=0), dict(n_heads=258), dict(q_row_stride=0), dict(out_row_stride=32), dict(window=-1), dict(sinks=-1), dict(sinks=4), dict(lens=None),
                                 dict(scale=float("nan")), dict(scale=float("inf"))])
def test_bad_attention_arguments_are_refused(lib, buf, bad):
    p = buf[1]
    kv, a = kv_args(p), attn_args(p, lib, **bad)
    assert lib.vtb_cuda_paged_attn_decode(C.byref(kv), C.byref(a), None) == -1
    assert lib.vtb_cuda_paged_attn_prefill(C.byref(kv), C.byref(a), p, 4, None) == -1


def test_misaligned_pointers_are_refused(lib, buf):
    p = buf[1]
    ok = kv_args(p)
    for kv, a in ((kv_args(p, k=p + 2), attn_args(p, lib)), (ok, attn_args(p, lib, q=p + 4)), (ok, attn_args(p, lib, out=p + 8)),
                  (ok, attn_args(p, lib, workspace=p + 4)), (ok, attn_args(p, lib, workspace=None))):
        assert lib.vtb_cuda_paged_attn_decode(C.byref(kv), C.byref(a), None) == -1


def test_small_workspace_is_refused(lib, buf):
    p = buf[1]
    kv, a = kv_args(p), attn_args(p, lib, workspace_bytes=0)
    assert lib.vtb_cuda_paged_attn_decode(C.byref(kv), C.byref(a), None) == -1
    assert lib.vtb_cuda_paged_attn_workspace_bytes(8, 8, 2, 64) == 0   # not a cache type
    assert lib.vtb_cuda_paged_attn_workspace_bytes(30, 7, 2, 64) == 0  # heads do not divide


def test_bad_prefill_rows_are_refused(lib, buf):
    p = buf[1]
    kv, a = kv_args(p), attn_args(p, lib)
    assert lib.vtb_cuda_paged_attn_prefill(C.byref(kv), C.byref(a), None, 4, None) == -1
    assert lib.vtb_cuda_paged_attn_prefill(C.byref(kv), C.byref(a), p, -1, None) == -1
    assert lib.vtb_cuda_paged_attn_prefill(C.byref(kv), C.byref(a), p, 1 << 40, None) == -1
    assert lib.vtb_cuda_paged_attn_prefill(C.byref(kv), C.byref(a), p, 0, None) == 0


@pytest.mark.parametrize("bad,status", [(dict(type=1), -8), (dict(type=8), -8), (dict(n_rows=-1), -1), (dict(k=None), -1),
                                        (dict(v=None), -1), (dict(k_row_stride=3), -1), (dict(v_head_stride=32), -1), (dict(q_row_stride=0), -1),
                                        (dict(q_out=None), -1), (dict(q=None), -1), (dict(n_heads=0), -1), (dict(seq=None), -1),
                                        (dict(pos=None), -1), (dict(n_rope=0), -1)])
def test_bad_rows_are_refused(lib, buf, bad, status):
    p = buf[1]
    kv, r = kv_args(p), rows_args(p, **bad)
    assert lib.vtb_cuda_paged_append(C.byref(kv), C.byref(r), None) == status


def test_no_rows_is_no_launch(lib, buf):
    p = buf[1]
    kv, r = kv_args(p), rows_args(p, n_rows=0)
    assert lib.vtb_cuda_paged_append(C.byref(kv), C.byref(r), None) == 0
    assert lib.vtb_cuda_paged_append(C.byref(kv), None, None) == -1


def test_bad_copies_are_refused(lib, buf):
    p = buf[1]
    kv = kv_args(p)
    f = lib.vtb_cuda_paged_copy
    assert f(C.byref(kv), 0, 0, p, p, 1, None, None, None) == -1
    assert f(C.byref(kv), 1, -8, p, p, 1, None, None, None) == -1
    assert f(C.byref(kv), 2, 3, p, p, 1, None, None, None) == -1
    assert f(C.byref(kv), 1, 0, None, p, 1, None, None, None) == -1
    assert f(C.byref(kv), 1, 0, p, p, -1, None, None, None) == -1
    assert f(C.byref(kv), 1, 0, p, p, 1, p, None, None) == -1
    assert f(C.byref(kv), 1, 0, p, p, 1, None, p, None) == -1
    assert f(None, 1, 0, p, p, 1, None, None, None) == -1
    assert f(C.byref(kv), 1, 0, None, None, 0, None, None, None) == 0  # nothing to do


def test_python_front_end_refuses_host_tensors(lib):
    import torch
    from vantablack_b200 import ops
    if torch.cuda.is_available():
        pytest.skip("the refusal of host tensors is the same with a GPU; covered where there is none")
    k = torch.zeros(4, 2, 16, 64)
    t = torch.zeros(2, 3, dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.paged_attention_decode(torch.zeros(2, 8, 64), k, k, t, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError):
        ops.paged_copy(k, k, t[0], t[1])


def test_packed_descriptors_have_the_c_layout(lib):
    from vantablack_b200 import ops
    for packed, c in ((ops._KV, _lib.PagedKv), (ops._ROWS, _lib.PagedRows), (ops._ATTN, _lib.PagedAttn)):
        assert packed.size == C.sizeof(c)
        vals = [0.5 if t is C.c_float else i + 1 for i, (_, t) in enumerate(c._fields_)]
        got = c.from_buffer_copy(packed.pack(*vals))
        assert [getattr(got, n) for n, _ in c._fields_] == vals


def test_counts_that_would_overflow_are_refused(lib, buf):
    p = buf[1]
    kv, a = kv_args(p), attn_args(p, lib)
    assert lib.vtb_cuda_paged_attn_prefill(C.byref(kv), C.byref(a), p, 1 << 62, None) == -1  # 4 heads a group: 2^64
    many = (1 << 31) - 1
    assert lib.vtb_cuda_paged_copy(C.byref(kv), many, 0, p, p, many, None, None, None) != 0
    kv = kv_args(p, n_kv_heads=4096, page_size=1024)
    assert lib.vtb_cuda_paged_copy(C.byref(kv), many, 0, p, p, many, None, None, None) != 0


def test_empty_list_of_rows_needs_no_address(lib, buf):
    p = buf[1]
    kv, a = kv_args(p), attn_args(p, lib, q=None, out=None)
    assert lib.vtb_cuda_paged_attn_prefill(C.byref(kv), C.byref(a), p, 0, None) == 0
    assert lib.vtb_cuda_paged_attn_prefill(C.byref(kv), C.byref(a), p, 1, None) == -1
