"""Plain 64-bit forms of the paged cache operators, and the error bounds that
their tests hold the kernels to."""
import math

import torch

EPS = {torch.float32: 2.0 ** -23, torch.float16: 2.0 ** -10, torch.bfloat16: 2.0 ** -7}


def pages(lens, page, g, extra=3, fill=-1, per=None):
    """Shuffled page ids per sequence: (table [n_seqs, pages] int32 on the CPU, number of pages)."""
    need = [-(-n // page) for n in lens]
    n_pages = sum(need) + extra
    ids = torch.randperm(n_pages, generator=g)[: sum(need)].tolist()
    table = torch.full((len(lens), max(max(need), 1) if per is None else per), fill, dtype=torch.int32)
    for s, n in enumerate(need):
        for j in range(n):
            table[s, j] = ids.pop()
    return table, n_pages


def visible(p, t, window, sinks):
    """[len(p), len(t)] truth values: which cached positions t the query positions p see."""
    see = t[None] <= p[:, None]
    if window:
        see &= (t[None] > p[:, None] - window) | (t[None] < sinks)
    return see


def attention(q, k, v, pos, scale, window=0, sinks=0):
    """q [rows, H, hd] at positions pos over k, v [len, KV, hd], all float64.  Returns (out, a, b):
    a = sum_t p_t |v_t|, b[row, head] = the largest visible sum_d |q_d k_d| * scale."""
    rows, heads, hd = q.shape
    length, kv, _ = k.shape
    see = visible(pos, torch.arange(length), window, sinks)[:, None]  # [rows, 1, len]
    kk = k.repeat_interleave(heads // kv, 1).permute(1, 2, 0)         # [H, hd, len]
    vv = v.repeat_interleave(heads // kv, 1).transpose(0, 1)          # [H, len, hd]
    x = torch.matmul(q.transpose(0, 1), kk).transpose(0, 1) * scale   # [rows, H, len]
    b = torch.matmul(q.abs().transpose(0, 1), kk.abs()).transpose(0, 1) * abs(scale)
    b = torch.where(see, b, 0.0).amax(-1) if length else torch.zeros(rows, heads)
    x = x.masked_fill(~see, -math.inf)
    p = torch.softmax(x, -1).nan_to_num(0.0) if length else x
    p = torch.where(see, p, 0.0)
    out = torch.matmul(p.transpose(0, 1), torch.where(torch.isfinite(vv), vv, 0.0)).transpose(0, 1)
    a = torch.matmul(p.transpose(0, 1), torch.where(torch.isfinite(vv), vv, 0.0).abs()).transpose(0, 1)
    return out, a, b


def attention_tolerance(out, a, b, n, dtype, p_rounded):
    """An elementwise bound on |kernel - exact|.

    Scores: hd products summed in f32 (at most 136 roundings with scale and split, 2^-24 each, on sum |q k|), and
    for f32 inputs products of values split into 11 + 11 bits, three of four kept: 2^-20 of sum |q k|.  A score
    error e changes every weight by at most a factor e^e and the sum by as much: 2 e (plus 2^-21 for
    exponentials), each times a = sum p |v|.  The sums over n positions: steps of 16 added in f32 and joined,
    (n / 16 + 40) 2^-24, numerator and denominator, and 2^-20 for the split products (f32) or 2^-16 (P as two
    16-bit values).  `p_rounded`: P as one value of the type, half a step.  Output: half a step."""
    f32 = dtype == torch.float32
    e = b[..., None] * (136 * 2.0 ** -24 + (2.0 ** -20 if f32 else 0.0))
    rel = 2 * e + 2.0 ** -21 + 2 * (n / 16 + 40) * 2.0 ** -24 + (2.0 ** -20 if f32 else 2.0 ** -16)
    if p_rounded and not f32:
        rel = rel + EPS[dtype] / 2
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0  # f16 below its normal range: steps of 2^-24
    return a * rel + (out.abs() + a * rel) * EPS[dtype] / 2 + tiny + 1e-30


class Cache:
    """A paged cache on the GPU filled from float64 host rows; slots that hold no position get `slack`."""

    def __init__(self, lens, kv, hd, page, dtype, seed, slack=float("nan"), layout="hnd", fill=-1, dev="cuda",
                 per=None):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.page, self.dtype = lens, page, dtype
        self.table, self.n_pages = pages(lens, page, g, fill=fill, per=per)
        self.k_rows = [torch.randn(n, kv, hd, generator=g).to(dtype) for n in lens]
        self.v_rows = [torch.randn(n, kv, hd, generator=g).to(dtype) for n in lens]
        shape = (self.n_pages, kv, page, hd)
        k = torch.full(shape, slack, dtype=dtype)
        v = torch.full(shape, slack, dtype=dtype)
        for s, n in enumerate(lens):
            if n:
                t = torch.arange(n)
                pg = self.table[s].long()[t // page]
                k[pg, :, t % page] = self.k_rows[s]
                v[pg, :, t % page] = self.v_rows[s]
        if layout == "hnd":
            self.k, self.v = k.to(dev), v.to(dev)
        elif layout == "nhd":  # [page, slot, head, dim] in memory
            self.k = k.transpose(1, 2).contiguous().to(dev).transpose(1, 2)
            self.v = v.transpose(1, 2).contiguous().to(dev).transpose(1, 2)
        else:  # K and V side by side in one buffer, with a gap behind each row
            buf = torch.full((self.n_pages, kv, page, 2, hd + 8), slack, dtype=dtype)
            buf[..., 0, :hd], buf[..., 1, :hd] = k, v
            buf = buf.to(dev)
            self.k, self.v = buf[..., 0, :hd], buf[..., 1, :hd]
        self.table = self.table.to(dev)
        self.d_lens = torch.tensor(lens, dtype=torch.int32, device=dev)
