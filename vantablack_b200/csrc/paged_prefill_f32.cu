// paged_prefill_f32.cu -- chunk attention over an f32 paged cache on the 5th-
// generation tensor cores, with f32-class results.
//
// Every operand is split into two tf32 values, x = hi + lo (11 significant bits
// each, split_tf32), and a product is three: lo hi + hi lo + hi hi, what is
// left out being 2^-22 of it.  The tensor cores add to their accumulators with
// truncation, so chains are kept short: the small terms of a chain come first,
// and O is not accumulated over the tiles of positions in TMEM but added up in
// registers, one f32 FMA per tile and element, which also applies the factor
// that a grown row maximum asks for.
//
// A CTA takes up to 128 query rows of one kv head (rows = (token, head of the
// group) pairs, whole tokens), and walks the positions they see in tiles of 64:
//   S = Q K^T    A = Q hi / lo from TMEM, B = K hi / lo, K-major in shared memory
//   P = 2^(S - m) by one thread per row, hi over S and lo beside it in TMEM
//   O = P V      A = P from TMEM, B = V^T hi / lo, K-major in shared memory
// TMEM: Q hi 0, Q lo HD, S / P hi 256, P lo 320, O 384 (columns).
//
// Warps 0-3: softmax and output; 4-7: split K, and warp 4 issues the MMAs between
// its rows of two tiles; 8-11: split and transpose V (each thread a head
// dimension, so that it writes 16-byte pieces of positions).  The next tile's K
// and V wait in registers until the products of this one have read the shared
// tiles.
// Tensor work of a tile at 128 values: 48 instructions of Q K^T (46 clocks each,
// measured) and 24 of P V (67), 3.8k clocks; a tile takes 8.5k, as the softmax with
// its splits follows Q K^T and a second S has no room in TMEM at 128 values.  256
// tokens on 1797 (32 / 8 heads x 128): 100 to 105 us, 80 TFLOP/s, 240 in tf32 products.
#include <type_traits>

#include "paged.cuh"

namespace vtb {

__device__ __forceinline__ void mma_tf32_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, int acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::tf32 [%0], [%1], %2, %3, p;\n}\n"
      ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}

constexpr int FQ = 128, FN = 64, F_THREADS = 384;
// Registers per thread: softmax warps, K and V warps (168 at launch).
constexpr int F_REGS_SOFTMAX = 232, F_REGS_SPLIT = 136;
template <int HD> struct F32Prefill {
  static constexpr int KV = FN * HD * 4;                // bytes of one part (hi or lo) of a K or V tile
  static constexpr int ROWS = FQ * HD * 4;              // Q on its way in, the output on its way out
  static constexpr int SMEM = 4 * KV + ROWS + 1024 + 128;
  static constexpr int SLOT = FQ * (HD + 2);            // floats of one split's partial result
  static constexpr uint32_t S = 256, P_LO = 320, O = 384;
};
struct F32Bars {
  uint64_t q_full, k_full, k_freed, v_full, v_freed, s_full, p_full, o_full;
  uint32_t tmem;
  int bad0, bad1;  // tiles with infinities or NaN in V lie in [bad0, bad1) (take_nonfinite)
};

__device__ __forceinline__ float max3_nan(float a, float b, float c) {  // NaN if one is
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// The row's scores once more where they are NaN, from the cache in plain f32: an
// infinity in K or Q, or a finite value next to the end of f32's range, has no second
// part that adds up with the first (inf - inf), and a score of -inf has to weigh
// nothing.  x: the tile's scores, from index i0 of the span on.
template <int HD>
__device__ __noinline__ void scores_again(const AttnArgs& a, const float* q, int s, int kvh, const Span& sp, int i0, float* x) {
  for (int i = 0; i < FN; ++i) {
    if (!isnan(x[i])) continue;
    const int t = sp.pos(i0 + i);
    const char* k = a.kv.k + page_row(a.kv, __ldg(a.kv.table + s * a.kv.table_stride + (t >> a.kv.page_shift)), t) + kvh * a.kv.head_stride;
    float d = 0.f;
    for (int c = 0; c < HD; c += 4) {
      const float4 u = *reinterpret_cast<const float4*>(q + c), v = *reinterpret_cast<const float4*>(k + c * 4);
      d = fmaf(u.x, v.x, d); d = fmaf(u.y, v.y, d); d = fmaf(u.z, v.z, d); d = fmaf(u.w, v.w, d);
    }
    x[i] = a.negate ? -d : d;
  }
}

template <int HD>
__global__ void __launch_bounds__(F_THREADS, 1) paged_prefill_f32_kernel(const __grid_constant__ AttnArgs a, int splits) {
  using C = F32Prefill<HD>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  F32Bars& bar = *reinterpret_cast<F32Bars*>(smem + 4 * C::KV + C::ROWS);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t sk = smem_u32(smem), sv = sk + 2 * C::KV, sr = sk + 4 * C::KV;

  // blockIdx.x = ((row tile from the last, kv head), split): the longest rows start first
  const int split = blockIdx.x % splits, unit = blockIdx.x / splits, kvh = unit % a.n_kv, units = gridDim.x / splits;
  RowTile rt;
  if (!row_tile(a, units / a.n_kv - 1 - unit / a.n_kv, a.tile, rt)) return;
  const int nflat = rt.n * a.group, last = min(rt.f0 + a.tile, nflat) - 1, tok0 = rt.f0 / a.group;
  const Span sp = span_of(max(0, rt.ctx + tok0), rt.ctx + last / a.group, a.window, a.sinks);
  const unsigned all = (sp.n + FN - 1) / FN;
  const int j0 = (int)(all * (unsigned)split / (unsigned)splits), n = (int)(all * (unsigned)(split + 1) / (unsigned)splits) - j0;

  if (warp == 4) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&bar.tmem)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  } else if (threadIdx.x == 0) {
    bar.bad0 = 0x7fffffff;
    bar.bad1 = 0;
    mbar_init(&bar.q_full, 4);
    mbar_init(&bar.k_full, 4);
    mbar_init(&bar.v_full, 4);
    mbar_init(&bar.p_full, 4);
    mbar_init(&bar.k_freed, 1);
    mbar_init(&bar.v_freed, 1);
    mbar_init(&bar.s_full, 1);
    mbar_init(&bar.o_full, 1);
    fence_mbar_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bar.tmem;  // 0: all columns are this CTA's
  bool ok = true;                  // one answer per warp; a wait that gave up ends the warp's work

  if (warp >= 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(F_REGS_SPLIT));
    const int32_t* table = a.kv.table + rt.s * a.kv.table_stride;
    // Byte offset of the row of index i of the span in the cache.  Indexes behind the
    // span get the cache's first row: their loads need no branch (which would make
    // one wait for the other), and zeros replace the values when they are split.
    auto row_of = [&](int i) -> long long {
      if (i >= sp.n) return 0;
      const int pos = sp.pos(i);
      return page_row(a.kv, __ldg(table + (pos >> a.kv.page_shift)), pos) + kvh * a.kv.head_stride;
    };
    auto landed = [&](uint64_t* full) {
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(full);
    };
    auto st4 = [&](uint32_t addr, const uint32_t* x) {
      asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]) : "memory");
    };
    if (warp < 8) {
      // ---------------- K: 16 rows per warp, PIECES lanes to a row ----------------
      constexpr int PIECES = HD / 4, RPR = 32 / PIECES, ROUNDS = 16 / RPR;
      const int pc = lane % PIECES, r0 = (warp - 4) * 16 + lane / PIECES;
      float4 x[ROUNDS];
      auto fetch = [&](int j) {
        const long long mine = row_of((j0 + j) * FN + (warp - 4) * 16 + (lane & 15));
#pragma unroll
        for (int i = 0; i < ROUNDS; ++i) {
          const long long off = __shfl_sync(0xffffffffu, mine, i * RPR + lane / PIECES);
          x[i] = *reinterpret_cast<const float4*>(a.kv.k + off + pc * 16);
        }
      };
      // MMA issuer (warp 4): uniform registers, one elected thread
      constexpr uint32_t base = (1u << 4) | (2u << 7) | (2u << 10) | ((uint32_t)(FQ >> 4) << 24);
      const uint32_t id_s = base | (a.negate ? 1u << 13 : 0u) | ((uint32_t)(FN >> 3) << 17);
      constexpr uint32_t id_o = base | ((uint32_t)(HD >> 3) << 17);
      constexpr int PART = C::KV >> 4, KATOM = FN * 128 >> 4, VATOM = HD * 128 >> 4;  // descriptor steps
      auto wait = [&](uint64_t* b, int phase) {
        ok = ok && warp_wait(b, phase & 1);
        tc_fence_after();
      };
      auto split = [&](int j) {  // the fetched rows into the shared tile
        if (j) ok = ok && warp_wait(&bar.k_freed, (j - 1) & 1);
        if (!ok) return;
#pragma unroll
        for (int i = 0; i < ROUNDS; ++i) {
          const int r = r0 + i * RPR;
          const uint32_t d = sk + (pc >> 3) * (FN * 128) + r * 128 + (((pc & 7) ^ (r & 7)) << 4);
          const bool live = (j0 + j) * FN + r < sp.n;
          const float v[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) split_tf32(live ? v[c] : 0.f, hi[c], lo[c]);
          st4(d, hi);
          st4(d + C::KV, lo);
        }
        landed(&bar.k_full);
      };
      auto qk = [&](int j) {
        wait(&bar.k_full, j);
        if (ok && elect_one()) {  // (in order behind the product that reads P of the tile before)
          const uint64_t dk = sw128_desc(sk);
#pragma unroll
          for (int t = 0; t < 3; ++t)  // lo hi, hi lo, hi hi
#pragma unroll
            for (int kk = 0; kk < HD / 8; ++kk)
              mma_tf32_ts(C::S, (t == 0 ? HD : 0) + kk * 8, dk + (t == 1 ? PART : 0) + (kk / 4) * KATOM + (kk % 4) * 2, id_s, (t | kk) != 0);
          mma_commit(&bar.s_full);
          mma_commit(&bar.k_freed);
        }
        __syncwarp();
      };
      auto pv = [&](int j) {
        wait(&bar.v_full, j);
        wait(&bar.p_full, j);
        if (ok && elect_one()) {
          const uint64_t dv = sw128_desc(sv);
#pragma unroll
          for (int t = 0; t < 3; ++t)
#pragma unroll
            for (int kk = 0; kk < FN / 8; ++kk)
              mma_tf32_ts(C::O, (t == 0 ? C::P_LO : C::S) + kk * 8, dv + (t == 1 ? PART : 0) + (kk / 4) * VATOM + (kk % 4) * 2, id_o, (t | kk) != 0);
          mma_commit(&bar.v_freed);
          mma_commit(&bar.o_full);
        }
        __syncwarp();
      };
      if (n > 0) fetch(0);
      for (int j = 0; j < n && ok; ++j) {  // warp 4 splits its rows of tile j while the softmax of tile j - 1 runs
        split(j);
        if (warp == 4) {
          if (j) pv(j - 1);
          else wait(&bar.q_full, 0);
          qk(j);
        }
        if (j + 1 < n) fetch(j + 1);
      }
      if (warp == 4 && n > 0) pv(n - 1);
    } else {
      // ---------------- V: one head dimension per thread, POS positions of it ----------------
      constexpr int POS = FN * HD / 128;
      const int t = threadIdx.x - 256, d = t % HD, p0 = t / HD * POS;
      float x[POS];
      auto fetch = [&](int j) {
        const int i0 = (j0 + j) * FN + p0;
        long long mine[POS / 32];
#pragma unroll
        for (int b = 0; b < POS / 32; ++b) mine[b] = row_of(i0 + 32 * b + lane);
#pragma unroll
        for (int i = 0; i < POS; ++i) {
          const long long off = __shfl_sync(0xffffffffu, mine[i / 32], i % 32);
          x[i] = *reinterpret_cast<const float*>(a.kv.v + off + d * 4);
        }
      };
      auto store = [&](int j, auto half) {  // the fetched values into the shared tile
#pragma unroll
        for (int i = 0; i < POS; i += 4) {
          const int pc = (p0 + i) / 4;  // 16-byte piece of the row of dimension d
          const uint32_t at = sv + (pc >> 3) * (HD * 128) + d * 128 + (((pc & 7) ^ (d & 7)) << 4);
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const float v = (j0 + j) * FN + p0 + i + c < sp.n ? x[i + c] : 0.f;
            split_tf32(v, hi[c], lo[c], half);
          }
          st4(at, hi);
          st4(at + C::KV, lo);
        }
      };
      if (n > 0) fetch(0);
      for (int j = 0; j < n; ++j) {
        if (j) ok = warp_wait(&bar.v_freed, (j - 1) & 1);
        if (!ok) break;
        bool odd = false;  // values that have no hi and lo: infinities, NaN, and what would round to infinity
#pragma unroll
        for (int i = 0; i < POS; ++i) odd |= (__float_as_uint(x[i]) & 0x7fffffffu) >= 0x7f7ff000u;
        bool huge = false;
        if (__any_sync(0xffffffffu, odd)) {
          bool bad = false;
#pragma unroll
          for (int i = 0; i < POS; ++i)
            if ((__float_as_uint(x[i]) & 0x7f800000u) == 0x7f800000u) {
              x[i] = 0.f;
              bad = true;
            } else {
              huge |= (__float_as_uint(x[i]) & 0x7fffffffu) >= 0x7f7ff000u;
            }
          if (__any_sync(0xffffffffu, bad) && lane == 0) {
            atomicMin(&bar.bad0, j);
            atomicMax(&bar.bad1, j + 1);
          }
        }
        // At 64 values two copies of the loop beat a register to add (1024 tokens on 1024:
        // 140 us, 165), at 128 they cost registers (252, 248).
        if constexpr (HD == 64) {
          if (huge) store(j, std::integral_constant<uint32_t, 0>());
          else store(j, std::integral_constant<uint32_t, 0x1000>());
        } else {
          store(j, huge ? 0u : 0x1000u);
        }
        landed(&bar.v_full);
        if (j + 1 < n) fetch(j + 1);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(F_REGS_SOFTMAX));
    // ---------------- softmax: one row per thread ----------------
    constexpr int PIECES = HD / 4, RPR = 32 / PIECES;  // whole rows in and out, PIECES lanes to a row
    const int r = threadIdx.x, pc = lane % PIECES;
    const bool row = r < a.tile && rt.f0 + r < nflat;
    const uint32_t lanes = (uint32_t)(warp * 32) << 16, mine = sr + r * HD * 4;
    auto place = [&](int x, int piece) { return sr + x * HD * 4 + ((piece ^ (x & 7)) << 4); };
#pragma unroll 4
    for (int i = lane / PIECES; i < 32; i += RPR) {
      const int x = warp * 32 + i, t = a.token(x);
      const bool live = x < a.tile && rt.f0 + x < nflat;
      const float* q = static_cast<const float*>(a.q);
      if (live) q += (rt.r0 + tok0 + t) * a.q_row + (long long)(kvh * a.group + x - t * a.group) * a.q_head + pc * 4;
      cpa16(place(x, pc), q, live);
    }
    cpa_commit();
    cpa_wait<0>();
    __syncwarp();
#pragma unroll 1
    for (int c = 0; c < HD; c += 32) {
      uint32_t hi[32], lo[32];
#pragma unroll
      for (int i = 0; i < 32; i += 4) {
        const float4 v = lds_f4(mine + ((((c + i) / 4) ^ (r & 7)) << 4));
        split_tf32(v.x, hi[i], lo[i]);
        split_tf32(v.y, hi[i + 1], lo[i + 1]);
        split_tf32(v.z, hi[i + 2], lo[i + 2]);
        split_tf32(v.w, hi[i + 3], lo[i + 3]);
      }
      tmem_st32(lanes + c, hi);
      tmem_st32(lanes + HD + c, lo);
    }
    tmem_wait_st();
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(&bar.q_full);

    // The row sees positions [0, va) (sinks) and [vb, vc), as index ranges of the span.
    int va = 0, vb = 0, vc = 0x7fffffff;
    if (row) {
      const int p = rt.ctx + tok0 + a.token(r);
      vc = p < 0 ? 0 : p - sp.w0 + sp.ns + 1;
      if (a.window && p >= 0) {
        vb = max(0, p + 1 - a.window) - sp.w0 + sp.ns;
        va = min(a.sinks, vb);
      }
    }
    float m = -INFINITY, l = 0.f, f = 1.f, o[HD];  // o is relative to the maximum before the last factor f
#pragma unroll
    for (int i = 0; i < HD; ++i) o[i] = 0.f;
    auto take = [&]() {  // o = o f + the last tile's product
#pragma unroll
      for (int c = 0; c < HD; c += 32) {
        uint32_t x[32];
        tmem_ld32(x, lanes + C::O + c);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) o[c + i] = fmaf(o[c + i], f, __uint_as_float(x[i]));
      }
    };
    for (int j = 0; j < n; ++j) {
      if (j) {  // the last tile's product, while this tile's S is computed
        ok = warp_wait(&bar.o_full, (j - 1) & 1);
        if (!ok) break;
        tc_fence_after();
        take();
      }
      ok = warp_wait(&bar.s_full, j & 1);
      if (!ok) break;
      tc_fence_after();
      uint32_t s[FN];
      tmem_ld32(s, lanes + C::S);
      tmem_ld32(s + 32, lanes + C::S + 32);
      tmem_wait_ld();
      const int v0 = (j0 + j) * FN;
      int masked = __any_sync(0xffffffffu, v0 + FN > vc || (v0 < vb && v0 + FN > va));
      asm volatile("" : "+r"(masked));
#pragma unroll 1
      for (; masked > 0; --masked) {
#pragma unroll
        for (int c = 0; c < FN; c += 32) {  // bit i: index v0 + c + i is seen
          const uint32_t see = below(vc - v0 - c) & (below(va - v0 - c) | ~below(vb - v0 - c));
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (!(see >> i & 1)) s[c + i] = 0xff800000u;
        }
      }
      auto largest = [&]() {  // NaN if a score that is seen is NaN
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < FN; i += 4)
#pragma unroll
          for (int q = 0; q < 2; ++q) mx[q] = max3_nan(mx[q], __uint_as_float(s[i + 2 * q]), __uint_as_float(s[i + 2 * q + 1]));
        return max3_nan(mx[0], mx[1], mx[0]);
      };
      float top = largest();
      int again = __any_sync(0xffffffffu, row && isnan(top));
      asm volatile("" : "+r"(again));
#pragma unroll 1
      for (; again > 0; --again) {
        float x[FN];
#pragma unroll
        for (int i = 0; i < FN; ++i) x[i] = __uint_as_float(s[i]);
        if (row) {
          const int t = a.token(r);
          const float* q = static_cast<const float*>(a.q) + (rt.r0 + tok0 + t) * a.q_row + (long long)(kvh * a.group + r - t * a.group) * a.q_head;
          scores_again<HD>(a, q, rt.s, kvh, sp, v0, x);
        }
#pragma unroll
        for (int i = 0; i < FN; ++i) s[i] = __float_as_uint(x[i]);
        top = largest();
      }
      const float mn = fmaxf(m, top * a.scale2), b = mn == -INFINITY ? 0.f : mn;
      f = ex2(m - b);
      m = mn;
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int c = 0; c < FN; c += 16) {
        uint32_t lo[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float p = ex2(fmaf(__uint_as_float(s[c + i]), a.scale2, -b));
          sum[i & 1] += p;
          split_tf32(p, s[c + i], lo[i]);
        }
        tmem_st16(lanes + C::S + c, s + c);
        tmem_st16(lanes + C::P_LO + c, lo);
      }
      l = l * f + (sum[0] + sum[1]);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.p_full);
    }
    if (ok && n > 0) {
      ok = warp_wait(&bar.o_full, (n - 1) & 1);
      tc_fence_after();
      if (ok) take();
    }
    // ---------------- output: whole rows through shared memory ----------------
    if (ok) {
      float* part = a.part + (long long)blockIdx.x * C::SLOT;
      const int bad0 = *reinterpret_cast<volatile int*>(&bar.bad0), bad1 = *reinterpret_cast<volatile int*>(&bar.bad1);
      if (bad0 < bad1) {
        RowSums<HD> x;
#pragma unroll
        for (int i = 0; i < HD; ++i) x.o[i] = o[i];
        for (uint32_t& y : x.set) y = 0;
        x.done = row ? 0u : ~0u;
        const int p = rt.ctx + tok0 + a.token(r), pa = a.window ? a.sinks : 0, pb = a.window ? p + 1 - a.window : 0;
        // the tiles' positions: sinks, then what lies behind w0
        const int i0 = (j0 + bad0) * FN, i1 = min((j0 + bad1) * FN, sp.n), behind = sp.w0 - sp.ns;
        take_nonfinite<float, HD>(a, rt.s, kvh, i0, min(i1, sp.ns), sp.w0, pa, pb, p + 1, x);
        take_nonfinite<float, HD>(a, rt.s, kvh, max(i0, sp.ns) + behind, i1 + behind, sp.w0, pa, pb, p + 1, x);
#pragma unroll
        for (int i = 0; i < HD; ++i) o[i] = x.o[i];
      }
      const float inv = splits > 1 ? 1.f : l == 0.f ? 0.f : 1.f / l;
      __syncwarp();
#pragma unroll
      for (int i = 0; i < HD; i += 4)
        asm volatile("st.shared.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(mine + (((i / 4) ^ (r & 7)) << 4)), "f"(o[i] * inv),
                     "f"(o[i + 1] * inv), "f"(o[i + 2] * inv), "f"(o[i + 3] * inv) : "memory");
      __syncwarp();
#pragma unroll 4
      for (int i = lane / PIECES; i < 32; i += RPR) {
        const int x = warp * 32 + i, t = a.token(x);
        if (x >= a.tile || rt.f0 + x >= nflat) break;
        float* dst = splits > 1 ? part + 2 * FQ + x * HD
                                : static_cast<float*>(a.out) + (rt.r0 + tok0 + t) * a.o_row + (long long)(kvh * a.group + x - t * a.group) * a.o_head;
        *reinterpret_cast<float4*>(dst + pc * 4) = lds_f4(place(x, pc));
      }
      if (splits > 1 && row) {
        part[r] = m;
        part[FQ + r] = l;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 4) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

size_t paged_prefill_f32_workspace(int head_dim) {
  return (size_t)sm_count(current_device()) * FQ * (head_dim + 2) * sizeof(float);
}

template <int HD>
static cudaError_t launch_prefill_f32_t(AttnArgs a, cudaStream_t st) {
  using C = F32Prefill<HD>;
  static_assert(F_REGS_SOFTMAX + 2 * F_REGS_SPLIT <= 3 * 168, "register shares");
  const int dev = current_device();
  cudaError_t e = ensure_smem_attr<paged_prefill_f32_kernel<HD>>(dev, C::SMEM);
  if (e || (e = check_register_split<paged_prefill_f32_kernel<HD>>(dev, F_THREADS,
                                                                    128 * (F_REGS_SOFTMAX + 2 * F_REGS_SPLIT))))
    return e;
  set_tile(a, FQ);
  const long long units = ((long long)a.rows * a.group / a.tile + a.kv.n_seqs) * a.n_kv;
  if (units > 0x7fffffffll / 16) return cudaErrorInvalidValue;
  const int splits = prefill_splits(a, units, FN, sm_count(dev));
  paged_prefill_f32_kernel<HD><<<(unsigned)(units * splits), F_THREADS, C::SMEM, st>>>(a, splits);
  if ((e = cudaGetLastError()) || splits == 1) return e;
  return launch_dependent(paged_prefill_join_kernel<float, HD, 1>, dim3((unsigned)(units * 8)), dim3(256), 0, st, a, splits);
}

cudaError_t launch_paged_prefill_f32(int head_dim, const AttnArgs& a, cudaStream_t st) {
  return head_dim == 64 ? launch_prefill_f32_t<64>(a, st) : launch_prefill_f32_t<128>(a, st);
}

}  // namespace vtb
