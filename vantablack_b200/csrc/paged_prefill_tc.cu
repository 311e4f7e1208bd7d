// paged_prefill_tc.cu -- chunk attention over the paged cache on the 5th-
// generation tensor cores, for f16 and bf16 caches.
//
// A CTA takes 256 query rows of one kv head (rows = (token, head of the group)
// pairs in token order, as in paged_prefill_kernel) as two tiles A and B of 128,
// and walks the positions they see in tiles of 128.  Per tile of positions:
//   S = Q K^T       tcgen05.mma, both operands K-major in 128-byte-swizzled
//                   shared tiles, S (f32) in TMEM
//   P = 2^(S - m)   one thread per row: the row maximum and sum need no
//                   exchange; P (16 bits) overwrites S in TMEM
//   O += P V        tcgen05.mma with P from TMEM and V (rows of positions,
//                   MN-major) from shared memory, O (f32) in TMEM
// The two tiles alternate: while the tensor cores work on one, eight warps of
// softmax threads (four per tile) work on the other.  O is rescaled only when
// a row's maximum has grown by more than 8 (a factor of 256, which both types
// hold), which after the first tiles hardly ever happens.
//
// Warps 0-3: softmax of A; 4-7: of B; warp 8: one thread issues the MMAs; 9-11
// bring K and V into two stages each by TMA, one box per page and 64 values (4-d
// map over the page pool); pages of fewer than 8 positions, whose boxes would
// break the swizzle, are gathered row by row with cp.async.  V rows at positions
// that no query row sees (behind the last position, before the window) are
// replaced by zeros, so what lies in the rest of a page never meets P = 0.
//
// The scale is taken positive (a negative one negates Q in the first product),
// so the maximum of S is the maximum of the scaled scores.
#include <type_traits>

#include "paged.cuh"
#include "tma.cuh"

namespace vtb {

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar)) : "memory");
}
// A bounded wait of a whole warp, with one answer for all its lanes.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, unsigned parity) {
  return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity));
}
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
  return r != 0;
}
__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, int acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, int acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
      ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
// MN-major operand in 128-byte-swizzled atoms of 64 values x 8 rows: rows 8 apart
// lie 1024 bytes apart, the next 64 values `mn` bytes.
__device__ __forceinline__ uint64_t sw128_desc_mn(uint32_t saddr, uint32_t mn) {
  return (sw128_desc(saddr) & ~((uint64_t)0x3fff << 16)) | (uint64_t)(mn >> 4) << 16;
}

#define VTB_R8(v, i) "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3]), "=r"(v[i + 4]), "=r"(v[i + 5]), "=r"(v[i + 6]), "=r"(v[i + 7])
#define VTB_I8(v, i) "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3]), "r"(v[i + 4]), "r"(v[i + 5]), "r"(v[i + 6]), "r"(v[i + 7])
__device__ __forceinline__ void tmem_ld32(uint32_t* v, uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : VTB_R8(v, 0), VTB_R8(v, 8), VTB_R8(v, 16), VTB_R8(v, 24) : "r"(addr));
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};"
      ::VTB_I8(v, 0), VTB_I8(v, 8), VTB_I8(v, 16), VTB_I8(v, 24), "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// 2^x of a pair on the FMA pipe: x = n + f with n the nearest integer (f in
// [-1/2, 1/2]), a degree-4 polynomial in f (least maximum relative error for a
// constant term of 1, fitted on Chebyshev nodes: 2.9e-6), n added to the exponent.
// x <= -127, -inf among it, gives exactly 0 (f = 0 there, and 1 has an exponent of 127).
__device__ __forceinline__ void ex2_poly(f2 x, float& a, float& b) {
  float u, v;
  unpk(x, u, v);
  x = pk(fmaxf(u, -127.f), fmaxf(v, -127.f));
  const f2 magic = pk(12582912.f, 12582912.f), t = add2(x, magic), f = sub2(x, sub2(t, magic));
  f2 p = fma2(f, pk(0.009582852944731712f, 0.009582852944731712f), pk(0.055906426161527634f, 0.055906426161527634f));
  p = fma2(p, f, pk(0.24024099111557007f, 0.24024099111557007f));
  p = fma2(p, f, pk(0.6931241750717163f, 0.6931241750717163f));
  p = fma2(p, f, pk(1.f, 1.f));
  float tu, tv;
  unpk(t, tu, tv);
  unpk(p, u, v);
  a = __int_as_float(__float_as_int(u) + (__float_as_int(tu) << 23));
  b = __int_as_float(__float_as_int(v) + (__float_as_int(tv) << 23));
}

constexpr int TQ = 128, TN = 128, TC_THREADS = 384;
// Of every 16 pairs of exponentials, this many go to the FMA pipe: the special-
// function unit alone (16 results per clock and SM) would take as long as the
// products of a tile.
constexpr int POLY = 4;
// Registers per thread after the split: softmax warps, MMA and gather warps.
// setmaxnreg draws on what the CTA was launched with, so the sum of the shares
// must not pass it (checked before the launch).
constexpr int REGS_SOFTMAX = 208, REGS_OTHER = 88;
template <int HD> struct TcPrefill {
  static constexpr int ATOM = 128 * 128;                // bytes: 128 rows x 64 values
  static constexpr int TILE = (HD / 64) * ATOM;         // one operand tile
  static constexpr int SMEM = 6 * TILE + 1024 + 256;    // Q A, Q B, K x 2, V x 2; alignment; barriers
  static constexpr int SLOT = 2 * TQ * (HD + 2);        // floats of one split's partial result
};

struct TcBars {
  uint64_t q_full, k_full[2], v_full[2], v_raw[2], k0_freed, freed[2], s_full[2], p_full[2][2], done;
  uint32_t tmem;
};

template <typename T, int HD>
__global__ void __launch_bounds__(TC_THREADS, 1)
paged_prefill_tc_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ CUtensorMap map_k,
                        const __grid_constant__ CUtensorMap map_v, int splits, int box) {
  using C = TcPrefill<HD>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  TcBars& bar = *reinterpret_cast<TcBars*>(smem + 6 * C::TILE);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0 && box) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_k)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_v)) : "memory");
  }
  // blockIdx.x = ((row tile from the last, kv head), split): the longest rows start first
  const int split = blockIdx.x % splits, unit = blockIdx.x / splits, kvh = unit % a.n_kv;
  const int units = gridDim.x / splits;
  RowTile rt;
  if (!row_tile(a, units / a.n_kv - 1 - unit / a.n_kv, 2 * TQ, rt)) return;
  const int nflat = rt.n * a.group;
  const bool two = rt.f0 + TQ < nflat;  // tile B has rows
  const int last = min(rt.f0 + 2 * TQ, nflat) - 1;
  // Positions [w0, p1] and, when a window has left them behind, the first `sinks`
  // of [0, w0), in tiles at multiples of TN: `ks` sink tiles, then those from kw.
  const int p1 = rt.ctx + last / a.group, p0 = max(0, rt.ctx + rt.f0 / a.group);
  const int w0 = a.window && p0 >= a.window ? p0 + 1 - a.window : 0;
  const int kw0 = w0 / TN, ks = min((min(a.sinks, w0) + TN - 1) / TN, kw0), ke = p1 < 0 ? 0 : p1 / TN + 1;
  const int kw = ke > 0 ? kw0 : 0, all = p1 < 0 ? 0 : ks + ke - kw;
  // Tiles that this split walks; those of A end with its own last position.
  const int j0 = (int)((long long)all * split / splits), j1 = (int)((long long)all * (split + 1) / splits);
  const int pa = rt.ctx + (min(rt.f0 + TQ, nflat) - 1) / a.group;  // A's last position
  const int na = max(0, min(j1, pa < 0 ? 0 : ks + pa / TN + 1 - kw) - j0), nb = two ? j1 - j0 : 0;
  auto tile_pos = [&](int j) { return (j0 + j < ks ? j0 + j : j0 + j - ks + kw) * TN; };  // first position of tile j

  if (threadIdx.x == 0) {
    mbar_init(&bar.q_full, 8);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar.k_full[i], 3);  // the three gather warps
      mbar_init(&bar.v_full[i], 3);
      mbar_init(&bar.v_raw[i], 1);
      mbar_init(&bar.s_full[i], 1);
      mbar_init(&bar.p_full[i][0], 4);  // the tile's four warps
      mbar_init(&bar.p_full[i][1], 4);
    }
    mbar_init(&bar.k0_freed, 1);
    mbar_init(&bar.freed[0], 1);
    mbar_init(&bar.freed[1], 1);
    mbar_init(&bar.done, 1);
    fence_mbar_init();
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&bar.tmem)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // All 512 columns are this CTA's, so its block starts at column 0: TMEM
  // addresses are constants (S at w * TN, O at 256 + w * HD).
  const uint32_t tmem = bar.tmem;
  const uint32_t sq = smem_u32(smem), sk = sq + 2 * C::TILE, sv = sq + 4 * C::TILE;
  const int n = max(na, nb);

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_OTHER));
    if (warp == 8) {
      // ---------------- MMA issuer ----------------
      // The whole warp walks the loop, so addresses and descriptors stay in uniform
      // registers (a one-thread branch moves each operand over: 90 clocks per
      // instruction instead of the 64 that it runs); one elected thread issues.
      constexpr uint32_t fmt = std::is_same<T, __half>::value ? 0u : 1u;
      constexpr uint32_t base = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(TQ >> 4) << 24);
      const uint32_t id_s = base | (a.negate ? 1u << 13 : 0u) | ((uint32_t)(TN >> 3) << 17);
      constexpr uint32_t id_o = base | (1u << 16) | ((uint32_t)(HD >> 3) << 17);
      const uint64_t dq = sw128_desc(sq), dk = sw128_desc(sk), dv = sw128_desc_mn(sv, C::ATOM);
      bool ok = true;
      auto qk = [&](int w, int j) {
        const uint64_t q = dq + w * (C::TILE >> 4), k = dk + (j & 1) * (C::TILE >> 4);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk) {
            constexpr int A16 = C::ATOM >> 4;
            const int off = (kk / 4) * A16 + (kk % 4) * 2;
            mma_f16_ss(w * TN, q + off, k + off, id_s, kk != 0);
          }
          mma_commit(&bar.s_full[w]);
        }
        __syncwarp();
      };
      auto pv = [&](int w, int j, int h) {
        const uint64_t v = dv + (j & 1) * (C::TILE >> 4) + h * (TN / 32) * 128;
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < TN / 32; ++kk)
            mma_f16_ts(256 + w * HD, w * TN + (h * (TN / 32) + kk) * 8, v + kk * 128, id_o, (j | h | kk) != 0);
        }
        __syncwarp();
      };
      // freed[j & 1], phase j / 2: V tile j and K tile j + 1 have been read (k0_freed: K tile 0)
      auto release = [&](uint64_t* b) {
        if (elect_one()) mma_commit(b);
        __syncwarp();
      };
      auto wait = [&](uint64_t* b, int phase) {
        ok = ok && warp_wait(b, phase & 1);
        tc_fence_after();
      };
      wait(&bar.q_full, 0);
      if (n > 0) wait(&bar.k_full[0], 0);
      if (ok && na > 0) qk(0, 0);
      if (ok && nb > 0) qk(1, 0);
      if (ok && n > 0) release(&bar.k0_freed);
      for (int j = 0; j < n && ok; ++j) {
        wait(&bar.v_full[j & 1], j >> 1);
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const int m = w ? nb : na;
          if (j >= m || !ok) continue;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            wait(&bar.p_full[w][h], j);
            if (ok) pv(w, j, h);
          }
          if (j + 1 >= m) continue;
          if (w == 0 || j + 1 >= na) wait(&bar.k_full[(j + 1) & 1], (j + 1) >> 1);
          if (ok) qk(w, j + 1);  // in order behind the product that reads P from the same columns
        }
        if (!ok) break;
        release(&bar.freed[j & 1]);
      }
      release(&bar.done);
      warp_wait(&bar.done, 0);
    } else {
      // ---------------- K / V tiles ----------------
      const int32_t* table = a.kv.table + rt.s * a.kv.table_stride;
      // by TMA: lane i of warp 9 loads box i / ATOMS, values 64 (i % ATOMS) ...; boxes
      // in which no position is seen are left out (their pages may be gone)
      auto boxes = [&](const CUtensorMap* map, uint32_t dst, int t0, uint64_t* full) {
        constexpr int ATOMS = HD / 64;
        const int i = lane / ATOMS, at = lane % ATOMS, pos = t0 + i * box;
        const bool mine = i * box < TN && pos <= p1 && (pos + box > w0 || pos < a.sinks);
        int page = mine ? __ldg(table + (pos >> a.kv.page_shift)) : 0;
        if ((unsigned)page >= (unsigned)a.kv.n_pages) {
          flag_error(DEV_ERR_BAD_ARG);
          page = 0;
        }
        const unsigned live = __ballot_sync(0xffffffffu, mine);
        if (lane == 0) mbar_expect_tx(full, __popc(live) * box * 128);
        __syncwarp();
        if (mine)
          tma_load_4d(dst + at * C::ATOM + i * box * 128, map, at * 64, pos & ((1 << a.kv.page_shift) - 1), kvh, page, full);
      };
      // by rows: 16-byte pieces, PIECES lanes to a row
      constexpr int PIECES = HD / 8, RPW = 32 / PIECES;
      const int pc = lane % PIECES, sub = (warp - 9) * RPW + lane / PIECES;
      auto rows = [&](const char* base, uint32_t dst, int t0) {
        const char* src = base + kvh * a.kv.head_stride + pc * 16;
        const uint32_t d0 = dst + (pc >> 3) * C::ATOM;
#pragma unroll 4
        for (int r = sub; r < TN; r += 3 * RPW) {
          const int pos = t0 + r;
          const bool live = pos <= p1 && (pos >= w0 || pos < a.sinks);
          const long long off = live ? page_row(a.kv, __ldg(table + (pos >> a.kv.page_shift)), pos) : 0;
          cpa16(d0 + r * 128 + (((pc & 7) ^ (r & 7)) << 4), src + off, live);
        }
        cpa_commit();
      };
      auto landed = [&](uint64_t* full) {  // this warp's copies are in shared memory
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(full);
      };
      bool ok = true;
      unsigned edges = 0;  // phase of v_raw[i] in bit i
      for (int j = 0; j < n && ok; ++j) {
        const int t0 = tile_pos(j), i = j & 1;
        const uint32_t dk = sk + i * C::TILE, dv = sv + i * C::TILE;
        if (j == 2) ok = warp_wait(&bar.k0_freed, 0);  // (K tile j - 2 of a later one: V tile j - 1 waited for it)
        if (!ok) break;
        if (!box) {
          rows(a.kv.k, dk, t0);
        } else if (warp == 9) {
          boxes(&map_k, dk, t0, &bar.k_full[i]);
        } else if (lane == 0) {
          mbar_arrive(&bar.k_full[i]);
        }
        if (j >= 2) ok = warp_wait(&bar.freed[i], ((j >> 1) - 1) & 1);
        if (!ok) break;
        if (!box) {
          rows(a.kv.v, dv, t0);
          cpa_wait<1>();
          landed(&bar.k_full[i]);
          cpa_wait<0>();
          landed(&bar.v_full[i]);
        } else if (t0 + TN > p1 + 1 || (t0 < w0 && t0 + TN > a.sinks)) {
          // an edge tile: zeros in place of the V rows that no query row sees
          if (warp == 9) {
            if (lane == 0) mbar_arrive(&bar.v_full[i]);
            boxes(&map_v, dv, t0, &bar.v_raw[i]);
          } else {
            ok = warp_wait(&bar.v_raw[i], edges >> i & 1);
            edges ^= 1u << i;
            for (int r = sub - RPW; r < TN; r += 2 * RPW) {
              const int pos = t0 + r;
              if (pos > p1 || (pos < w0 && pos >= a.sinks))
                *reinterpret_cast<uint4*>(smem + (4 + i) * C::TILE + (pc >> 3) * C::ATOM + r * 128 + ((pc & 7) << 4)) =
                    make_uint4(0, 0, 0, 0);
            }
            landed(&bar.v_full[i]);
          }
        } else if (warp == 9) {
          boxes(&map_v, dv, t0, &bar.v_full[i]);
        } else if (lane == 0) {
          mbar_arrive(&bar.v_full[i]);
        }
      }
      cpa_wait<0>();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_SOFTMAX));
    // ---------------- softmax: one row per thread ----------------
    const int w = warp >> 2, r = threadIdx.x & 127, f = rt.f0 + w * TQ + r;
    const bool row = f < nflat;
    {  // this warp's 32 rows of Q into the swizzled tile, whole rows at a time
      constexpr int PIECES = HD / 8, RPW = 32 / PIECES;
      const int pc = lane % PIECES;
#pragma unroll 4
      for (int i = lane / PIECES; i < 32; i += RPW) {
        const int x = (warp & 3) * 32 + i, fx = rt.f0 + w * TQ + x, t = min(fx, nflat - 1) / a.group;
        const T* q = static_cast<const T*>(a.q) + (rt.r0 + t) * a.q_row + (long long)(kvh * a.group + min(fx, nflat - 1) - t * a.group) * a.q_head;
        cpa16(sq + w * C::TILE + (pc >> 3) * C::ATOM + x * 128 + (((pc & 7) ^ (x & 7)) << 4), q + pc * 8, fx < nflat);
      }
      cpa_commit();
      cpa_wait<0>();
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.q_full);
    }
    // The row sees positions [0, va) (sinks) and [vb, vc).
    const int p = rt.ctx + f / a.group;
    int va = 0, vb = 0, vc = 0x7fffffff;
    if (row) {
      vc = p + 1;
      if (a.window) {
        vb = vc - a.window;
        va = a.sinks;
      }
    }
    const int m_tiles = w ? nb : na;
    const uint32_t ts = w * TN + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t to = 256 + w * HD + ((uint32_t)((warp & 3) * 32) << 16);
    float m = -INFINITY, l = 0.f;  // the maximum that P is relative to (in units of log2), the row's sum
    bool ok = true;
    for (int j = 0; j < m_tiles; ++j) {
      ok = ok && warp_wait(&bar.s_full[w], j & 1);
      if (!ok) break;
      tc_fence_after();
      uint32_t s[TN];
#pragma unroll
      for (int c = 0; c < TN; c += 32) tmem_ld32(s + c, ts + c);
      tmem_wait_ld();
      const int v0 = tile_pos(j);
      // Few tiles need a mask.  Written as a loop because the compiler turns an `if`
      // here into 128 selects on every tile (830 of 2400 clocks).
      int masked = __any_sync(0xffffffffu, v0 + TN > vc || (v0 < vb && v0 + TN > va));
      asm volatile("" : "+r"(masked));
#pragma unroll 1
      for (; masked > 0; --masked) {
        const int xa = va - v0, xb = vb - v0, xc = vc - v0;
#pragma unroll
        for (int i = 0; i < TN; ++i)
          if (i >= xc || (i < xb && i >= xa)) s[i] = 0xff800000u;
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < TN; i += 8)
#pragma unroll
        for (int k = 0; k < 4; ++k) mx[k] = max3(mx[k], __uint_as_float(s[i + 2 * k]), __uint_as_float(s[i + 2 * k + 1]));
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale2;
      if (__any_sync(0xffffffffu, top > m + 8.f)) {
        const float mn = fmaxf(m, top), k = m == -INFINITY ? 0.f : ex2(m - mn);
        m = mn;
        l *= k;
        if (j > 0) {  // every product so far is complete: S was issued behind them
#pragma unroll 1
          for (int c = 0; c < HD; c += 32) {
            uint32_t o[32];
            tmem_ld32(o, to + c);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * k);
            tmem_st32(to + c, o);
          }
        }
      }
      const float b = m == -INFINITY ? 0.f : -m;
      const f2 scale = pk(a.scale2, a.scale2), base = pk(b, b);
      f2 sum[2] = {pk(0.f, 0.f), pk(0.f, 0.f)};
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // P in two halves: the product starts on the first
#pragma unroll
        for (int i = h * (TN / 4); i < (h + 1) * (TN / 4); ++i) {
          const f2 x = fma2(pk(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), scale, base);
          float u, v;
          if ((i * POLY) % 16 + POLY >= 16 && POLY > 0) {
            ex2_poly(x, u, v);
          } else {
            unpk(x, u, v);
            u = ex2(u);
            v = ex2(v);
          }
          sum[i & 1] = add2(sum[i & 1], pk(u, v));
          s[i] = pack2<T>(u, v);
        }
        tmem_st32(ts + h * 32, s + h * 32);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.p_full[w][h]);
      }
      l += hsum(add2(sum[0], sum[1]));
    }
    // ---------------- output ----------------
    ok = ok && warp_wait(&bar.done, 0);
    if (ok) {
      tc_fence_after();
      float* part = a.part + (long long)blockIdx.x * C::SLOT;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      // 16-bit rows go out through this warp's part of the Q tile (its products are
      // done), so that stores cover whole rows
      const uint32_t stage = sq + w * C::TILE + (warp & 3) * 32 * HD * 2;
#pragma unroll 1
      for (int c = 0; c < HD; c += 32) {
        uint32_t o[32];
        if (m_tiles > 0) {
          tmem_ld32(o, to + c);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0u;
        }
        if (splits == 1) {
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            uint32_t x[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
              x[k] = pack2<T>(__uint_as_float(o[i + 2 * k]) * inv, __uint_as_float(o[i + 2 * k + 1]) * inv);
            const int pc = (c + i) / 8;
            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(stage + lane * HD * 2 + ((pc ^ (lane & 7)) << 4)),
                         "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]) : "memory");
          }
        } else if (row) {
          float* d = part + 4 * TQ + (long long)(w * TQ + r) * HD + c;
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<float4*>(d + i) = make_float4(__uint_as_float(o[i]), __uint_as_float(o[i + 1]),
                                                            __uint_as_float(o[i + 2]), __uint_as_float(o[i + 3]));
        }
      }
      if (splits == 1) {
        __syncwarp();
        constexpr int PIECES = HD / 8, RPW = 32 / PIECES;
        const int pc = lane % PIECES;
#pragma unroll 4
        for (int i = lane / PIECES; i < 32; i += RPW) {
          const int fx = rt.f0 + w * TQ + (warp & 3) * 32 + i, t = fx / a.group;
          if (fx >= nflat) break;
          uint4 x;
          asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
                       : "r"(stage + i * HD * 2 + ((pc ^ (i & 7)) << 4)) : "memory");
          T* out = static_cast<T*>(a.out) + (rt.r0 + t) * a.o_row + (long long)(kvh * a.group + fx - t * a.group) * a.o_head;
          *reinterpret_cast<uint4*>(out + pc * 8) = x;
        }
      }
      if (splits > 1 && row) {
        part[w * TQ + r] = m_tiles > 0 ? m : -INFINITY;
        part[2 * TQ + w * TQ + r] = l;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

// Adds the splits of 256 rows, 16 rows per CTA: out = sum_i o_i 2^(m_i - M) / sum_i l_i 2^(m_i - M).
template <typename T, int HD>
__global__ void __launch_bounds__(256) paged_prefill_join_kernel(const __grid_constant__ AttnArgs a, int splits) {
  using C = TcPrefill<HD>;
  const int unit = blockIdx.x >> 4, kvh = unit % a.n_kv, units = gridDim.x >> 4;
  RowTile rt;
  const bool any = row_tile(a, units / a.n_kv - 1 - unit / a.n_kv, 2 * TQ, rt);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (!any) return;
  constexpr int LANES = HD / 8;  // threads per row, 8 values each
  for (int x = threadIdx.x; x < 16 * LANES; x += 256) {
    const int r = (blockIdx.x & 15) * 16 + x / LANES, c = (x % LANES) * 8, f = rt.f0 + r;
    if (f >= rt.n * a.group) continue;
    const float* p = a.part + (long long)unit * splits * C::SLOT;
    float M = -INFINITY, L = 0.f, acc[8] = {};
    for (int i = 0; i < splits; ++i) M = fmaxf(M, p[(long long)i * C::SLOT + r]);
    const float b = M == -INFINITY ? 0.f : M;
#pragma unroll 4
    for (int i = 0; i < splits; ++i) {
      const float* q = p + (long long)i * C::SLOT;
      const float e = exp2f(q[r] - b);
      L += q[2 * TQ + r] * e;
      const float4 u = *reinterpret_cast<const float4*>(q + 4 * TQ + (long long)r * HD + c);
      const float4 v = *reinterpret_cast<const float4*>(q + 4 * TQ + (long long)r * HD + c + 4);
      acc[0] += u.x * e; acc[1] += u.y * e; acc[2] += u.z * e; acc[3] += u.w * e;
      acc[4] += v.x * e; acc[5] += v.y * e; acc[6] += v.z * e; acc[7] += v.w * e;
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] *= inv;
    store_vec(static_cast<T*>(a.out) + (rt.r0 + f / a.group) * a.o_row + (long long)(kvh * a.group + f % a.group) * a.o_head + c, acc);
  }
}

// CTAs that a call of few row tiles spreads over: one per SM.
size_t paged_prefill_tc_workspace(int head_dim) {
  return (size_t)sm_count(current_device()) * 2 * TQ * (head_dim + 2) * sizeof(float);
}

// TMA map of a page pool, (value, slot, head, page), in boxes of 64 values x `fit` slots.
static bool page_map(CUtensorMap* map, const PagedView& kv, const char* base, bool half, int hd, int n_kv, int fit) {
  auto fn = tmap_encode_fn();
  if (!fn || !kv.page_stride || !kv.head_stride || !kv.slot_stride || kv.page_stride >= (1ll << 40)) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)hd, (cuuint64_t)1 << kv.page_shift, (cuuint64_t)n_kv, (cuuint64_t)kv.n_pages};
  const cuuint64_t strides[3] = {(cuuint64_t)kv.slot_stride, (cuuint64_t)kv.head_stride, (cuuint64_t)kv.page_stride};
  const cuuint32_t boxes[4] = {64, (cuuint32_t)fit, 1, 1}, ones[4] = {1, 1, 1, 1};
  return fn(map, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<char*>(base), dims,
            strides, boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Whether the kernel was built with the registers that its split adds up to.
template <auto KERN>
static cudaError_t check_register_split(int dev) {
  static std::atomic<int> known[VTB_MAX_DEVICES];
  if (known[dev].load(std::memory_order_relaxed)) return cudaSuccess;
  cudaFuncAttributes f;
  const cudaError_t e = cudaFuncGetAttributes(&f, KERN);
  if (e) return e;
  if (f.numRegs / 8 * 8 * TC_THREADS < 256 * REGS_SOFTMAX + 128 * REGS_OTHER) return cudaErrorInvalidConfiguration;
  known[dev].store(1, std::memory_order_relaxed);
  return cudaSuccess;
}

template <typename T, int HD>
static cudaError_t launch_prefill_tc_t(AttnArgs a, cudaStream_t st) {
  using C = TcPrefill<HD>;
  a.negate = a.scale2 < 0.f;
  a.scale2 = fmaxf(fabsf(a.scale2), 1e-36f);  // not 0: masked scores have to stay -inf
  const int dev = current_device();
  cudaError_t e = ensure_smem_attr<paged_prefill_tc_kernel<T, HD>>(dev, C::SMEM);
  if (e || (e = check_register_split<paged_prefill_tc_kernel<T, HD>>(dev))) return e;
  const long long units = ((long long)a.rows * a.group / (2 * TQ) + a.kv.n_seqs) * a.n_kv;
  if (units > 0x7fffffffll / 16) return cudaErrorInvalidValue;
  // Fewer row tiles than SMs: the positions are split too, down to two tiles of
  // positions per CTA (below that the join costs more than the split gives).
  const long long cap = (long long)a.kv.pages_per_seq << a.kv.page_shift;
  long long seen = a.window ? (long long)a.window + a.sinks + a.rows : cap;
  if (seen > cap) seen = cap;
  long long splits = sm_count(dev) / units, most = seen / (2 * TN);
  if (splits > most) splits = most;
  if (splits < 1) splits = 1;
  CUtensorMap map_k = {}, map_v = {};
  const int slots = 1 << a.kv.page_shift, fit = slots < TN ? slots : TN;
  const int box = slots >= 8 && page_map(&map_k, a.kv, a.kv.k, std::is_same<T, __half>::value, HD, a.n_kv, fit) &&
                          page_map(&map_v, a.kv, a.kv.v, std::is_same<T, __half>::value, HD, a.n_kv, fit) ? fit : 0;
  paged_prefill_tc_kernel<T, HD><<<(unsigned)(units * splits), TC_THREADS, C::SMEM, st>>>(a, map_k, map_v, (int)splits, box);
  if ((e = cudaGetLastError()) || splits == 1) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(units * 16));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_prefill_join_kernel<T, HD>, a, (int)splits);
}

cudaError_t launch_paged_prefill_tc(int type, int head_dim, const AttnArgs& a, cudaStream_t st) {
  if (type == T_F16) return head_dim == 64 ? launch_prefill_tc_t<__half, 64>(a, st) : launch_prefill_tc_t<__half, 128>(a, st);
  return head_dim == 64 ? launch_prefill_tc_t<__nv_bfloat16, 64>(a, st) : launch_prefill_tc_t<__nv_bfloat16, 128>(a, st);
}

}  // namespace vtb
