"""Tensor-level front end of the CUDA kernels.

Device memory and streams come from PyTorch (plumbing only); every call goes
through the C ABI of libvtbcuda.so on torch's current stream.  Weight
tensors are flat ``torch.uint8`` CUDA tensors of packed GGUF blocks.
"""
from __future__ import annotations

import ctypes as C

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

KV_TYPES = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}


def _on(dev: torch.device, t: torch.Tensor, name: str, dtype: torch.dtype) -> None:
    if t.device != dev:
        raise ValueError(f"{name} must be on {dev}, as the cache is")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}")


def _paged_kv(k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor | None) -> _lib.PagedKv:
    """The cache as the C ABI describes it; k, v [n_pages, n_kv_heads, page_size, head_dim]
    (any order of strides, so a [page, slot, head, dim] cache goes in as .transpose(1, 2))."""
    if not k.is_cuda or k.device.index != torch.cuda.current_device():
        raise ValueError("the cache must be on the current CUDA device")
    st = k.stride()
    if k.dim() != 4 or st[3] != 1 or k.dtype not in KV_TYPES:
        raise ValueError("the cache is [n_pages, n_kv_heads, page_size, head_dim], f32, f16 or bf16, dense in head_dim")
    _on(k.device, v, "v", k.dtype)
    if v.shape != k.shape or v.stride() != st:
        raise ValueError("k and v must agree in shape and strides")
    n_pages, n_kv, page_size, hd = k.shape
    if page_table is None:
        return _lib.PagedKv(k.data_ptr(), v.data_ptr(), KV_TYPES[k.dtype], n_kv, hd, page_size, n_pages, st[0], st[1],
                            st[2], None, 0, 0, 0)
    _on(k.device, page_table, "page_table", torch.int32)
    if page_table.dim() != 2 or (page_table.stride(1) != 1 and page_table.shape[1] > 1):
        raise ValueError("page_table is [n_seqs, pages per sequence], dense in its rows")
    n, per = page_table.shape
    ld = page_table.stride(0)
    return _lib.PagedKv(k.data_ptr(), v.data_ptr(), KV_TYPES[k.dtype], n_kv, hd, page_size, n_pages, st[0], st[1],
                        st[2], page_table.data_ptr(), ld if n > 1 else max(ld, per), n, per)


def _rows(x: torch.Tensor, name: str, dev: torch.device, dtype: torch.dtype, heads: int | None, hd: int):
    """(row stride, head stride) of [rows, heads, head_dim] rows."""
    _on(dev, x, name, dtype)
    if x.dim() != 3 or x.shape[2] != hd or (heads is not None and x.shape[1] != heads):
        raise ValueError(f"{name} has the wrong shape {tuple(x.shape)}")
    st = x.stride()
    if st[2] != 1:
        raise ValueError(f"{name} must be dense in head_dim")
    return st[0], st[1] if x.shape[1] > 1 else hd


def paged_append(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, k: torch.Tensor,
                 v: torch.Tensor, seq: torch.Tensor, pos: torch.Tensor, q: torch.Tensor | None = None,
                 q_out: torch.Tensor | None = None, rope: torch.Tensor | None = None) -> torch.Tensor | None:
    """Writes the rows k, v [rows, n_kv_heads, head_dim] (f32 or the cache's type) into the pages at position
    pos[r] of sequence seq[r] (int32; a negative one skips the row), rotated by rope [positions, head_dim] if
    given; with q [rows, n_heads, head_dim] also returns the rotated queries in the cache's type (in q_out)."""
    kv = _paged_kv(k_pages, v_pages, page_table)
    dev, n_kv, hd = k_pages.device, kv.n_kv_heads, kv.head_dim
    x = k.dtype
    if x not in (torch.float32, k_pages.dtype):
        raise ValueError("rows must be f32 or of the cache's type")
    ks = _rows(k, "k", dev, x, n_kv, hd)
    vs = _rows(v, "v", dev, x, n_kv, hd)
    n = k.shape[0]
    _on(dev, seq, "seq", torch.int32); _on(dev, pos, "pos", torch.int32)
    if v.shape[0] != n or seq.shape != (n,) or pos.shape != (n,) or not (seq.is_contiguous() and pos.is_contiguous()):
        raise ValueError("k, v, seq and pos must have one entry per row")
    qs, heads = (0, 0), 0
    if q is not None:
        qs, heads = _rows(q, "q", dev, x, None, hd), q.shape[1]
        if q.shape[0] != n:
            raise ValueError("q must have one entry per row")
        if q_out is None:
            q_out = torch.empty(n, heads, hd, dtype=k_pages.dtype, device=dev)
        _on(dev, q_out, "q_out", k_pages.dtype)
        if q_out.shape != (n, heads, hd) or not q_out.is_contiguous():
            raise ValueError("q_out must be contiguous [rows, n_heads, head_dim]")
    elif q_out is not None:
        raise ValueError("q_out without q")
    if rope is not None:
        _on(dev, rope, "rope", torch.float32)
        if rope.dim() != 2 or rope.shape[1] != hd or not rope.is_contiguous():
            raise ValueError("rope must be contiguous f32 [positions, head_dim]")
    if n == 0:
        return q_out
    r = _lib.PagedRows(KV_TYPES[x], heads, n, k.data_ptr(), v.data_ptr(), q.data_ptr() if q is not None else None,
                       *ks, *vs, *qs, q_out.data_ptr() if q is not None else None,
                       rope.data_ptr() if rope is not None else None, rope.shape[0] if rope is not None else 0,
                       seq.data_ptr(), pos.data_ptr())
    _lib.check(lib.vtb_cuda_paged_append(C.byref(kv), C.byref(r), _stream()), "vtb_cuda_paged_append")
    return q_out


def paged_attention_workspace(dtype: torch.dtype, n_heads: int, n_kv_heads: int, head_dim: int,
                              device="cuda") -> torch.Tensor:
    """A workspace for the paged attention calls of one stream (calls that may overlap need one each)."""
    n = lib.vtb_cuda_paged_attn_workspace_bytes(KV_TYPES[dtype], n_heads, n_kv_heads, head_dim)
    return torch.empty(n, dtype=torch.uint8, device=device)


def _attn(kv, q, k_pages, lens, scale, window, sinks, out, workspace):
    dev, hd = k_pages.device, kv.head_dim
    qs = _rows(q, "q", dev, k_pages.dtype, None, hd)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    os = _rows(out, "out", dev, k_pages.dtype, q.shape[1], hd)
    _on(dev, lens, "lens", torch.int32)
    if out.shape != q.shape or lens.shape != (kv.n_seqs,) or not lens.is_contiguous():
        raise ValueError("out must have q's shape, lens one entry per sequence")
    if workspace is None:
        workspace = paged_attention_workspace(k_pages.dtype, q.shape[1], kv.n_kv_heads, hd, dev)
    _on(dev, workspace, "workspace", torch.uint8)
    if scale is None:
        scale = hd ** -0.5
    return out, _lib.PagedAttn(q.data_ptr(), out.data_ptr(), *qs, *os, q.shape[1], window, sinks, scale,
                               lens.data_ptr(), workspace.data_ptr(), workspace.numel()), workspace


def paged_attention_decode(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                           lens: torch.Tensor, scale: float | None = None, window: int = 0, sinks: int = 0,
                           out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one new token per sequence, q [n_seqs, n_heads, head_dim] at position lens[s] - 1, over the
    sequence's pages.  window > 0: the last `window` positions and the first `sinks` are visible.  scale: 1 / sqrt(head_dim)
    unless given.  A sequence of length 0 gives zeros."""
    kv = _paged_kv(k_pages, v_pages, page_table)
    if q.shape[0] != kv.n_seqs:
        raise ValueError("q must have one row per sequence")
    out, a, workspace = _attn(kv, q, k_pages, lens, scale, window, sinks, out, workspace)
    _lib.check(lib.vtb_cuda_paged_attn_decode(C.byref(kv), C.byref(a), _stream()), "vtb_cuda_paged_attn_decode")
    return out


def paged_attention_prefill(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                            lens: torch.Tensor, starts: torch.Tensor, scale: float | None = None, window: int = 0,
                            sinks: int = 0, out: torch.Tensor | None = None,
                            workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of a chunk of new tokens per sequence: rows starts[s] .. starts[s + 1] of q
    [rows, n_heads, head_dim] are the last tokens of sequence s's lens[s] positions, whose keys and values are
    in the pages already (paged_append).  Rows that no sequence holds are left as they were."""
    kv = _paged_kv(k_pages, v_pages, page_table)
    _on(k_pages.device, starts, "starts", torch.int32)
    if starts.shape != (kv.n_seqs + 1,) or not starts.is_contiguous():
        raise ValueError("starts must have one entry per sequence and one more")
    out, a, workspace = _attn(kv, q, k_pages, lens, scale, window, sinks, out, workspace)
    _lib.check(lib.vtb_cuda_paged_attn_prefill(C.byref(kv), C.byref(a), starts.data_ptr(), q.shape[0], _stream()),
               "vtb_cuda_paged_attn_prefill")
    return out


def paged_copy(k_cache: torch.Tensor, v_cache: torch.Tensor, src: torch.Tensor, dst: torch.Tensor,
               page_table: torch.Tensor | None = None, page_map: torch.Tensor | None = None) -> None:
    """Copies page src[i] to page dst[i] (int32) in all layers of k_cache, v_cache [n_layers, n_pages, n_kv_heads,
    page_size, head_dim] (or one layer's 4-d pages); entries e >= 0 of page_table become page_map[e]."""
    if k_cache.dim() == 4:
        k_cache, v_cache = k_cache[None], v_cache[None]
    if k_cache.dim() != 5 or v_cache.shape != k_cache.shape or v_cache.stride() != k_cache.stride() or not k_cache.shape[0]:
        raise ValueError("the cache is [n_layers, n_pages, n_kv_heads, page_size, head_dim], k and v alike")
    if (page_table is None) != (page_map is None):
        raise ValueError("page_table and page_map go together")
    kv = _paged_kv(k_cache[0], v_cache[0], page_table)
    dev, n = k_cache.device, src.numel()
    for t, nm in ((src, "src"), (dst, "dst")):
        _on(dev, t, nm, torch.int32)
        if t.shape != (n,) or not t.is_contiguous():
            raise ValueError("src and dst must be contiguous lists of the same length")
    if page_map is not None:
        _on(dev, page_map, "page_map", torch.int32)
        if page_map.shape != (kv.n_pages,) or not page_map.is_contiguous():
            raise ValueError("page_map must have one entry per page")
    _lib.check(lib.vtb_cuda_paged_copy(C.byref(kv), k_cache.shape[0], k_cache.stride(0), src.data_ptr(), dst.data_ptr(), n,
                                       page_table.data_ptr() if page_table is not None else None,
                                       page_map.data_ptr() if page_map is not None else None, _stream()),
               "vtb_cuda_paged_copy")


def check_device_error() -> None:
    _lib.check(lib.vtb_cuda_check_device_error(), "device error word")
