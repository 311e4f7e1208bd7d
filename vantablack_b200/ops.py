"""Tensor-level front end of the CUDA kernels.

Device memory and streams come from PyTorch (plumbing only); every call goes
through the C ABI of libvtbcuda.so on torch's current stream.  Weight
tensors are flat ``torch.uint8`` CUDA tensors of packed GGUF blocks.
"""
from __future__ import annotations

import ctypes as C
import functools
import struct

import torch

from . import _lib
from .synth import BF16, BLOCK_ELEMS, F16, F32, Q4_K, Q5_K, Q6_K, Q8_0, row_bytes  # noqa: F401

lib = _lib.load()


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _dev(t: torch.Tensor, name: str) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def gemv(quant: int, w: torch.Tensor, x: torch.Tensor, m: int, k: int, out: torch.Tensor | None = None,
         pdl: bool = False) -> torch.Tensor:
    """y[m] = W[m, k] . x[k] (f32)."""
    _dev(w, "w"); _dev(x, "x")
    if x.dtype != torch.float32 or x.numel() != k:
        raise ValueError("x must be f32[k]")
    if w.numel() < m * row_bytes(quant, k):
        raise ValueError("w is smaller than m rows")
    y = torch.empty(m, dtype=torch.float32, device=x.device) if out is None else out
    _lib.check(lib.vtb_cuda_gemv(quant, w.data_ptr(), x.data_ptr(), y.data_ptr(), m, k, _stream(), int(pdl)),
               "vtb_cuda_gemv")
    return y


def dequant(quant: int, w: torch.Tensor, n: int) -> torch.Tensor:
    _dev(w, "w")
    out = torch.empty(n, dtype=torch.float32, device=w.device)
    _lib.check(lib.vtb_cuda_dequant(quant, w.data_ptr(), out.data_ptr(), n, _stream()), "vtb_cuda_dequant")
    return out


def embed(quant: int, table: torch.Tensor, ids: torch.Tensor, dim: int) -> torch.Tensor:
    _dev(table, "table"); _dev(ids, "ids")
    ids = ids.to(torch.int32)
    out = torch.empty(ids.numel(), dim, dtype=torch.float32, device=table.device)
    _lib.check(lib.vtb_cuda_embed(quant, table.data_ptr(), ids.data_ptr(), out.data_ptr(), dim, ids.numel(),
                                  _stream()), "vtb_cuda_embed")
    return out


def gemv_mlx(w: torch.Tensor, scales: torch.Tensor, biases: torch.Tensor, x: torch.Tensor, m: int, k: int,
             bits: int, group: int, bf16: bool, w_off: int = 0) -> torch.Tensor:
    """MLX affine GEMV (mlx.zig matmul): y[m] = W . x.  w, scales, biases are
    flat uint8 CUDA tensors; w_off shifts the weight pointer by bytes."""
    for t, nm in ((w, "w"), (scales, "scales"), (biases, "biases"), (x, "x")):
        _dev(t, nm)
    y = torch.empty(m, dtype=torch.float32, device=x.device)
    _lib.check(lib.vtb_cuda_gemv_mlx(w.data_ptr() + w_off, scales.data_ptr(), biases.data_ptr(), x.data_ptr(),
                                     y.data_ptr(), m, k, bits, group, int(bf16), _stream()), "vtb_cuda_gemv_mlx")
    return y


def dequant_mlx(w: torch.Tensor, scales: torch.Tensor, biases: torch.Tensor, rows: int, k: int, bits: int,
                group: int, bf16: bool, w_off: int = 0) -> torch.Tensor:
    for t, nm in ((w, "w"), (scales, "scales"), (biases, "biases")):
        _dev(t, nm)
    out = torch.empty(rows, k, dtype=torch.float32, device=w.device)
    _lib.check(lib.vtb_cuda_dequant_mlx(w.data_ptr() + w_off, scales.data_ptr(), biases.data_ptr(), out.data_ptr(),
                                        rows, k, bits, group, int(bf16), _stream()), "vtb_cuda_dequant_mlx")
    return out


def sample(logits: torch.Tensor, temperature: float, top_k: int = 0, top_p: float = 0.0, u=None) -> torch.Tensor:
    """Sampler.sample (sampler.zig:44-104) per row of f32 logits [rows, n] on the
    device, with one caller-supplied uniform draw per row; logits are rewritten
    in place.  Returns int32 tokens [rows] on the device."""
    import numpy as np
    _dev(logits, "logits")
    if logits.dtype != torch.float32:
        raise ValueError("logits must be f32")
    lg = logits if logits.dim() == 2 else logits.view(1, -1)
    rows, n = lg.shape
    cfg = _lib.SamplerConfig(float(temperature), int(top_k), float(top_p), 0)
    ua = None if u is None else np.ascontiguousarray(np.atleast_1d(u), np.float32)
    if ua is not None and ua.size != rows:
        raise ValueError("one draw per row")
    tok = torch.empty(rows, dtype=torch.int32, device=logits.device)
    _lib.check(lib.vtb_cuda_sample(lg.data_ptr(), rows, n, n, C.byref(cfg),
                                   None if ua is None else ua.ctypes.data, tok.data_ptr(), _stream()),
               "vtb_cuda_sample")
    return tok


def quantize_q8_0(x: torch.Tensor):
    _dev(x, "x")
    k = x.numel()
    qs = torch.empty(k, dtype=torch.int8, device=x.device)
    d = torch.empty(k // 32, dtype=torch.float32, device=x.device)
    _lib.check(lib.vtb_cuda_quantize_q8_0(x.data_ptr(), k, qs.data_ptr(), d.data_ptr(), _stream()),
               "vtb_cuda_quantize_q8_0")
    return qs, d


def q8_0_block_dots(w: torch.Tensor, xq: torch.Tensor, m: int, k: int) -> torch.Tensor:
    _dev(w, "w"); _dev(xq, "xq")
    dots = torch.empty(m, k // 32, dtype=torch.int32, device=w.device)
    _lib.check(lib.vtb_cuda_q8_0_block_dots(w.data_ptr(), xq.data_ptr(), dots.data_ptr(), m, k, _stream()),
               "vtb_cuda_q8_0_block_dots")
    return dots


def gemv_q8_0_q8_0(w: torch.Tensor, x: torch.Tensor, m: int, k: int, out=None, scratch=None,
                   pdl: bool = False) -> torch.Tensor:
    _dev(w, "w"); _dev(x, "x")
    y = torch.empty(m, dtype=torch.float32, device=x.device) if out is None else out
    if scratch is None:
        scratch = (torch.empty(k, dtype=torch.int8, device=x.device),
                   torch.empty(k // 32, dtype=torch.float32, device=x.device))
    xq, dx = scratch
    _lib.check(lib.vtb_cuda_gemv_q8_0_q8_0(w.data_ptr(), x.data_ptr(), y.data_ptr(), m, k, xq.data_ptr(),
                                           dx.data_ptr(), _stream(), int(pdl)), "vtb_cuda_gemv_q8_0_q8_0")
    return y


def gemm(quant: int, w: torch.Tensor, acts: torch.Tensor, m: int, k: int, precise: bool = False,
         out: torch.Tensor | None = None) -> torch.Tensor:
    """out[B, m] = acts[B, k] . W^T on the tcgen05 tensor cores (prefill)."""
    _dev(w, "w"); _dev(acts, "acts")
    nb = acts.shape[0]
    if acts.dtype != torch.float32 or acts.numel() != nb * k:
        raise ValueError("acts must be f32[B, k]")
    o = torch.empty(nb, m, dtype=torch.float32, device=acts.device) if out is None else out
    wsb = lib.vtb_cuda_gemm_workspace_bytes(k, nb, int(precise))
    ws = torch.empty(wsb, dtype=torch.uint8, device=acts.device)
    _lib.check(lib.vtb_cuda_gemm(quant, w.data_ptr(), acts.data_ptr(), o.data_ptr(), m, k, nb, int(precise),
                                 ws.data_ptr(), wsb, _stream()), "vtb_cuda_gemm")
    return o


# ---- paged key-value cache ----
# A decode step makes these calls once per layer, so the host side is kept short: descriptors are packed as bytes
# (struct, in the C layouts of _lib.PagedKv / PagedRows / PagedAttn), device and stream are read as plain integers.

KV_TYPES = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
_KV = struct.Struct("@2P4i4qPq2i")
_ROWS = struct.Struct("@2iq3P6q2Pq2P")
_ATTN = struct.Struct("@2P4q3if2PN")
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _stream_of(dev: int) -> int:
    return _raw_stream(dev) if _raw_stream is not None else _stream()


def _on(dev: int, dtype: torch.dtype, **tensors) -> None:
    for name, t in tensors.items():
        if t.get_device() != dev:
            raise ValueError(f"{name} must be on the cache's device")
        if t.dtype is not dtype:
            raise ValueError(f"{name} must be {dtype}")


def _paged_kv(k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor | None):
    """The cache as the C ABI describes it; k, v [n_pages, n_kv_heads, page_size, head_dim]
    (any order of strides, so a [page, slot, head, dim] cache goes in as .transpose(1, 2); an axis of
    layers before them is left to the caller).  Returns (descriptor, device index, dtype, shape, n_seqs)."""
    dev, dt, st, shape = k.get_device(), k.dtype, k.stride(), k.shape
    if dev < 0 or dev != _current_device():
        raise ValueError("the cache must be on the current CUDA device")
    code = KV_TYPES.get(dt)
    if code is None or len(st) < 4 or st[-1] != 1:
        raise ValueError("the cache is [n_pages, n_kv_heads, page_size, head_dim], f32, f16 or bf16, dense in head_dim")
    if v.get_device() != dev or v.dtype is not dt or v.stride() != st or v.shape != shape:
        raise ValueError("k and v must agree in device, type, shape and strides")
    n_pages, n_kv, page_size, hd = shape[-4:]
    ptr = ld = n = per = 0
    if page_table is not None:
        if page_table.get_device() != dev or page_table.dtype is not torch.int32:
            _on(dev, torch.int32, page_table=page_table)
        if page_table.dim() != 2:
            raise ValueError("page_table is [n_seqs, pages per sequence]")
        n, per = page_table.shape
        ld, one = page_table.stride()
        if one != 1 and per > 1:
            raise ValueError("page_table must be dense in its rows")
        if n <= 1 and ld < per:
            ld = per
        ptr = page_table.data_ptr()
    kv = _KV.pack(k.data_ptr(), v.data_ptr(), code, n_kv, hd, page_size, n_pages, st[-4], st[-3], st[-2], ptr, ld, n, per)
    return kv, dev, dt, shape, n


def _rows(x: torch.Tensor, name: str, dev: int, dtype: torch.dtype, heads: int | None, hd: int):
    """(row stride, head stride) of [rows, heads, head_dim] rows."""
    st, shape = x.stride(), x.shape
    if x.get_device() != dev or x.dtype is not dtype:
        _on(dev, dtype, **{name: x})
    if len(st) != 3 or shape[2] != hd or (heads is not None and shape[1] != heads):
        raise ValueError(f"{name} has the wrong shape {tuple(shape)}")
    if st[2] != 1:
        raise ValueError(f"{name} must be dense in head_dim")
    return st[0], st[1] if shape[1] > 1 else hd


def _vec(x: torch.Tensor, name: str, dev: int, n: int) -> int:
    """Address of a contiguous int32 list of n entries."""
    if x.get_device() != dev or x.dtype is not torch.int32:
        _on(dev, torch.int32, **{name: x})
    if x.dim() != 1 or x.numel() != n or (n > 1 and x.stride(0) != 1):
        raise ValueError(f"{name} must be a contiguous list of {n} entries")
    return x.data_ptr()


def paged_append(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, k: torch.Tensor,
                 v: torch.Tensor, seq: torch.Tensor, pos: torch.Tensor, q: torch.Tensor | None = None,
                 q_out: torch.Tensor | None = None, rope: torch.Tensor | None = None) -> torch.Tensor | None:
    """Writes the rows k, v [rows, n_kv_heads, head_dim] (f32 or the cache's type) into the pages at position
    pos[r] of sequence seq[r] (int32; a negative one skips the row), rotated by rope [positions, head_dim] if
    given; with q [rows, n_heads, head_dim] also returns the rotated queries in the cache's type (in q_out)."""
    kv, dev, dt, shape, _ = _paged_kv(k_pages, v_pages, page_table)
    _, n_kv, _, hd = shape
    x = k.dtype
    if x is not torch.float32 and x is not dt:
        raise ValueError("rows must be f32 or of the cache's type")
    ks = _rows(k, "k", dev, x, n_kv, hd)
    vs = _rows(v, "v", dev, x, n_kv, hd)
    n = k.shape[0]
    if v.shape[0] != n:
        raise ValueError("v must have one entry per row")
    at = (_vec(seq, "seq", dev, n), _vec(pos, "pos", dev, n))
    qs, heads, q_ptr, o_ptr = (0, 0), 0, 0, 0
    if q is not None:
        qs, heads = _rows(q, "q", dev, x, None, hd), q.shape[1]
        if q.shape[0] != n:
            raise ValueError("q must have one entry per row")
        if q_out is None:
            q_out = torch.empty(n, heads, hd, dtype=dt, device=k_pages.device)
        else:
            _rows(q_out, "q_out", dev, dt, heads, hd)
            if q_out.shape[0] != n or not q_out.is_contiguous():
                raise ValueError("q_out must be contiguous [rows, n_heads, head_dim]")
        q_ptr, o_ptr = q.data_ptr(), q_out.data_ptr()
    elif q_out is not None:
        raise ValueError("q_out without q")
    turn = (0, 0)
    if rope is not None:
        _on(dev, torch.float32, rope=rope)
        if rope.dim() != 2 or rope.shape[1] != hd or not rope.is_contiguous():
            raise ValueError("rope must be contiguous f32 [positions, head_dim]")
        turn = (rope.data_ptr(), rope.shape[0])
    if n == 0:
        return q_out
    r = _ROWS.pack(KV_TYPES[x], heads, n, k.data_ptr(), v.data_ptr(), q_ptr, *ks, *vs, *qs, o_ptr, *turn, *at)
    _lib.check(lib.vtb_cuda_paged_append(kv, r, _stream_of(dev)), "vtb_cuda_paged_append")
    return q_out


@functools.lru_cache(maxsize=None)
def _workspace_bytes(dtype: torch.dtype, n_heads: int, n_kv_heads: int, head_dim: int, dev: int) -> int:
    return lib.vtb_cuda_paged_attn_workspace_bytes(KV_TYPES[dtype], n_heads, n_kv_heads, head_dim)


def paged_attention_workspace(dtype: torch.dtype, n_heads: int, n_kv_heads: int, head_dim: int,
                              device="cuda") -> torch.Tensor:
    """A workspace for the paged attention calls of one stream on `device` (calls that may overlap need one each)."""
    device = torch.device(device)
    dev = _current_device() if device.index is None else device.index
    with torch.cuda.device(dev):  # its size goes by the device's SMs
        n = _workspace_bytes(dtype, n_heads, n_kv_heads, head_dim, dev)
    return torch.empty(n, dtype=torch.uint8, device=device)


def _attn(q, k_pages, dev, dt, shape, n_seqs, lens, scale, window, sinks, out, workspace):
    _, n_kv, _, hd = shape
    qs, heads = _rows(q, "q", dev, dt, None, hd), q.shape[1]
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(q.shape)
    os = _rows(out, "out", dev, dt, heads, hd)
    if out.shape[0] != q.shape[0]:
        raise ValueError("out must have q's shape")
    if workspace is None:
        workspace = k_pages.new_empty(_workspace_bytes(dt, heads, n_kv, hd, dev), dtype=torch.uint8)
    elif workspace.get_device() != dev or workspace.dtype is not torch.uint8 or not workspace.is_contiguous():
        raise ValueError("workspace must be a contiguous uint8 tensor on the cache's device")
    a = _ATTN.pack(q.data_ptr(), out.data_ptr(), *qs, *os, heads, window, sinks, hd ** -0.5 if scale is None else scale,
                   _vec(lens, "lens", dev, n_seqs), workspace.data_ptr(), workspace.numel())
    return out, a, workspace


def paged_attention_decode(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                           lens: torch.Tensor, scale: float | None = None, window: int = 0, sinks: int = 0,
                           out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one new token per sequence, q [n_seqs, n_heads, head_dim] at position lens[s] - 1, over the
    sequence's pages.  window > 0: the last `window` positions and the first `sinks` are visible.  scale: 1 / sqrt(head_dim)
    unless given.  A sequence of length 0 gives zeros."""
    kv, dev, dt, shape, n_seqs = _paged_kv(k_pages, v_pages, page_table)
    if q.shape[0] != n_seqs:
        raise ValueError("q must have one row per sequence")
    if n_seqs == 0:
        return torch.empty_like(q) if out is None else out
    out, a, workspace = _attn(q, k_pages, dev, dt, shape, n_seqs, lens, scale, window, sinks, out, workspace)
    _lib.check(lib.vtb_cuda_paged_attn_decode(kv, a, _stream_of(dev)), "vtb_cuda_paged_attn_decode")
    return out


def paged_attention_prefill(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                            lens: torch.Tensor, starts: torch.Tensor, scale: float | None = None, window: int = 0,
                            sinks: int = 0, out: torch.Tensor | None = None,
                            workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of a chunk of new tokens per sequence: rows starts[s] .. starts[s + 1] of q
    [rows, n_heads, head_dim] are the last tokens of sequence s's lens[s] positions, whose keys and values are
    in the pages already (paged_append).  Rows that no sequence holds are left as they were."""
    kv, dev, dt, shape, n_seqs = _paged_kv(k_pages, v_pages, page_table)
    at = _vec(starts, "starts", dev, n_seqs + 1)
    if q.shape[0] == 0:
        return torch.empty_like(q) if out is None else out
    out, a, workspace = _attn(q, k_pages, dev, dt, shape, n_seqs, lens, scale, window, sinks, out, workspace)
    _lib.check(lib.vtb_cuda_paged_attn_prefill(kv, a, at, q.shape[0], _stream_of(dev)), "vtb_cuda_paged_attn_prefill")
    return out


def paged_copy(k_cache: torch.Tensor, v_cache: torch.Tensor, src: torch.Tensor, dst: torch.Tensor,
               page_table: torch.Tensor | None = None, page_map: torch.Tensor | None = None) -> None:
    """Copies page src[i] to page dst[i] (int32) in all layers of k_cache, v_cache [n_layers, n_pages, n_kv_heads,
    page_size, head_dim] (or one layer's 4-d pages); entries e >= 0 of page_table become page_map[e]."""
    layers, step = (k_cache.shape[0], k_cache.stride(0)) if k_cache.dim() == 5 else (1, 0)
    if k_cache.dim() not in (4, 5) or not layers:
        raise ValueError("the cache is [n_layers, n_pages, n_kv_heads, page_size, head_dim], or one layer's four axes")
    if (page_table is None) != (page_map is None):
        raise ValueError("page_table and page_map go together")
    kv, dev, _, shape, _ = _paged_kv(k_cache, v_cache, page_table)
    n = src.numel()
    moves = (_vec(src, "src", dev, n), _vec(dst, "dst", dev, n), n)
    tables = (page_table.data_ptr(), _vec(page_map, "page_map", dev, shape[-4])) if page_map is not None else (0, 0)
    _lib.check(lib.vtb_cuda_paged_copy(kv, layers, step, *moves, *tables, _stream_of(dev)),
               "vtb_cuda_paged_copy")


def check_device_error() -> None:
    _lib.check(lib.vtb_cuda_check_device_error(), "device error word")
