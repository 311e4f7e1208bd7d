// paged_prefill_tc.cu -- chunk attention over the paged cache on the 5th-
// generation tensor cores, for f16 and bf16 caches.
//
// One CTA per SM runs at a time and takes items one after the other.  An item is two tiles A and B of up to
// 128 query rows of one kv head (rows = (token, head of the group) pairs in token
// order, whole tokens to a tile), and the positions they see in tiles of 128.
// Per tile of positions:
//   S = Q K^T       tcgen05.mma, both operands K-major in 128-byte-swizzled
//                   shared tiles, S (f32) in TMEM
//   P = 2^(S - m)   one thread per row: the row maximum and sum need no
//                   exchange; P overwrites S in TMEM, as a sum of two 16-bit
//                   values (what the first leaves is rounded again), which keeps a
//                   weight to 2^-17 (bf16), so that the output carries its own
//                   rounding only
//   O += P V        tcgen05.mma, a product for each part of P, with P from TMEM
//                   and V (rows of positions, MN-major) from shared memory, O (f32)
//                   in TMEM
// The tiles A and B alternate on the tensor cores: while they work on one, the
// softmax threads work on the other.  O is rescaled only when a row's maximum
// has grown by more than Range::LAG bits, which after the first tiles hardly ever
// happens.
//
// Warps 0-3: softmax of A; 4-7: of B; 8: issues the MMAs; 10: brings Q, K and V
// by TMA, K and V into two stages each, one box per page and 64 values (4-d map
// over the page pool); 9 and 11: in tiles at an edge (the last positions, the
// window's start) put zeros in place of V rows at positions that no query row
// sees, so that what lies in the rest of a page never meets P = 0, and in place of
// infinities and NaN in the others (take_nonfinite).  Pages of fewer than 8 positions,
// whose boxes would break the swizzle, are gathered row by row with cp.async by
// warps 9 to 11.
//
// Bound by the chain of one row tile, not by a pipe: the softmax with its 1024 clocks
// of exponentials at the MUFU rate and the rounding of both parts of P, then P V (1024
// clocks at 128 values) and the next Q K^T (512), and the hand-overs.  A pair of row
// tiles takes 4500 to 4800 clocks per tile of positions at 128 values, 4170 at 64; to
// that a call adds 18 to 19 us, and the change from one item to the next 10 us (64) to
// 20 us (128), which no stage of the kernel has been seen to account for.  Measured
// (32 / 8 heads x 128, bf16): 2048 tokens 64 us (0.53 PFLOP/s), 8192 under a window of
// 4096 586 to 593 us (0.70); 11 chunks of 1 to 511 (32 / 4 x 64, f16) 112 to 115 us.  With
// P as one 16-bit value it was 53, 459 and 96 us, at an error against 64 bits of 0.0020
// (bf16) and 2.9e-4 (f16) of the output in place of the 0.0016 and 2.1e-4 that the
// output's rounding makes alone.
//
// The scale is taken positive (a negative one negates Q in the first product),
// so the maximum of S is the maximum of the scaled scores.
#include <type_traits>

#include "paged.cuh"
#include "tma.cuh"

namespace vtb {

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar)) : "memory");
}
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
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
      ::VTB_I8(v, 0), VTB_I8(v, 8), "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Bits 0 ... n - 1 (none for n <= 0, all for n >= 32).
__device__ __forceinline__ uint32_t below(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Infinities and NaN in V.  0 * inf is NaN, so they may not meet the weights of rows that
// do not see them, nor weights that are 0 only because they were rounded.  In tiles
// that part of the rows see, zeros go into the products in their place; in the others
// they leave a sum that is not finite.  Either way the rows that see such a position
// get its values afterwards (inf + x = inf, whatever P is): the warp, whose rows share
// the sequence and the kv head, looks through V 32 positions at a time and
// visits the ones that hold any.
// Puts them in place of what the sums x.o hold for their values.  The item sees positions
// from w0 on and the sinks, the lane's row [0, va) and [vb, vc).
template <int HD> struct RowSums {
  float o[HD];
  uint32_t set[HD / 32];  // bits of the values that such a position has given so far
  uint32_t done;          // bits of V's 16-byte pieces whose values are all NaN: nothing changes them any more
};
template <typename T, int HD>
__device__ __noinline__ void take_nonfinite(const AttnArgs& a, int s, int kvh, int t0, int t1, int w0, int va, int vb, int vc,
                                            RowSums<HD>& x) {
  constexpr int PER = 16 / sizeof(T), PIECES = HD / PER;
  constexpr uint32_t ALL = 0xffffffffu >> (32 - PIECES);
  const int32_t* table = a.kv.table + s * a.kv.table_stride;
  const char* v = a.kv.v + kvh * a.kv.head_stride;
  auto bad = [](float y) { return (__float_as_uint(y) & 0x7f800000u) == 0x7f800000u; };
  for (int b = t0; b < t1; b += 32) {
    const uint32_t skip = __reduce_and_sync(0xffffffffu, x.done);
    if ((skip & ALL) == ALL) return;
    const int mine = b + (threadIdx.x & 31);
    long long off = 0;
    uint32_t odd = 0;  // the pieces of this lane's position that hold any
    if (mine < t1 && (mine >= w0 || mine < a.sinks)) {
      off = page_row(a.kv, __ldg(table + (mine >> a.kv.page_shift)), mine);
#pragma unroll 8
      for (int p = 0; p < PIECES; ++p) {
        float y[PER];
        load_vec<T, T>(reinterpret_cast<const T*>(v + off) + p * PER, y);
        bool any = false;
#pragma unroll
        for (int k = 0; k < PER; ++k) any |= bad(y[k]);
        odd |= any ? 1u << p : 0u;
      }
      odd &= ~skip;
    }
    for (unsigned hits = __ballot_sync(0xffffffffu, odd != 0); hits; hits &= hits - 1) {
      const int l = __ffs(hits) - 1, t = b + l;
      const long long from = __shfl_sync(0xffffffffu, off, l);
      uint32_t m = __shfl_sync(0xffffffffu, odd, l);
      if (t >= vc || (t < vb && t >= va)) continue;
      for (; m; m &= m - 1) {
        const int p = __ffs(m) - 1, d = p * PER;
        float y[PER];
        load_vec<T, T>(reinterpret_cast<const T*>(v + from) + d, y);
        bool nan = true;
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          if (bad(y[k])) {
            const uint32_t bit = 1u << ((d + k) & 31);
            x.o[d + k] = x.set[(d + k) >> 5] & bit ? x.o[d + k] + y[k] : y[k];
            x.set[(d + k) >> 5] |= bit;
          }
          nan = nan && isnan(x.o[d + k]);
        }
        if (nan) x.done |= 1u << p;
      }
    }
  }
}
// Whether one of the 16-bit values in w is infinite or NaN, in bits 15 and 31 of the result.
template <typename T> __device__ __forceinline__ uint32_t nonfinite2(uint32_t w) {
  constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7c007c00u : 0x7f807f80u;
  return (w & e) + (std::is_same<T, __half>::value ? 0x04000400u : 0x00800080u);
}

constexpr int TQ = 128, TN = 128, TC_THREADS = 384;
// How far (in bits) the maximum that P is relative to may lag behind a row's own before O
// is rescaled, and the power of two that P is kept times.  bf16 has f32's range: P is at
// most 1, so a sum overflows only where the plain one does.  f16
// ends at steps of 2^-24, so weights far below the largest would be lost from the
// products, but not from the row's sum: they are kept times 2^13 (2^15 at most, with
// the lag), which holds them to 2^-38 of the largest.  4096 tokens on 4096 (32 / 8 heads
// x 128): 522 us; lag 8 and 2^7 (2^-32) 516; no lag and 2^15 (2^-40) 548.
template <typename T> struct Range { static constexpr float LAG = 8.f, UP = -8.f; };
template <> struct Range<__half> { static constexpr float LAG = 2.f, UP = 13.f; };
// Registers per thread after the split: softmax warps, MMA and gather warps.
// setmaxnreg draws on what the CTA was launched with, so the sum of the shares
// must not pass it (checked before the launch).
constexpr int REGS_SOFTMAX = 200, REGS_OTHER = 104;
template <int HD> struct TcPrefill {
  static constexpr int ATOM = 128 * 128;                // bytes: 128 rows x 64 values
  static constexpr int TILE = (HD / 64) * ATOM;         // one operand tile
  static constexpr int OUT = 8 * 32 * 128;              // output staging: 64 values of 32 rows per softmax warp
  static constexpr int SMEM = 6 * TILE + OUT + 1024 + 256;  // Q A, Q B, K x 2, V x 2; staging; alignment; barriers
  static constexpr int SLOT = 2 * TQ * (HD + 2);        // floats of one split's partial result
};

struct TcBars {
  uint4 answer[2];  // to requests for items
  uint64_t next_full[2], next_read[2];
  uint64_t q_full, q_freed, k_full[2], k_freed[2], v_full[2], v_freed[2], v_raw[2], s_full[2], p_full[2], o_full[2], done;
  uint32_t tmem;
  int mended[4];  // [i & 3] = i + 1: the CTA's i-th item has zeros in place of infinities or NaN in V
};

// One piece of work: two row tiles of a kv head over one split of the positions they see.
struct TcItem {
  RowTile rt;
  int kvh, nflat, first, p1, w0, ks, kw, j0, na, nb;  // first: position of the first row (p1: of the last)
  __device__ __forceinline__ int tiles() const { return max(na, nb); }
  // Whether some of the item's rows do not see all of the tile at t0.
  __device__ __forceinline__ bool edge(int t0, const AttnArgs& a) const {
    return t0 + TN > first + 1 || (a.window && t0 < p1 + 1 - a.window);
  }
  __device__ __forceinline__ int pos(int j) const { return (j0 + j < ks ? j0 + j : j0 + j - ks + kw) * TN; }  // first of tile j
};
// Item `i` of `items`: (row tile from the last, kv head, split), so the longest rows
// come first.  False: no such row tile.
__device__ __forceinline__ bool tc_item(const AttnArgs& a, int i, int items, int splits, TcItem& t) {
  const int split = i % splits, unit = i / splits, units = items / splits;
  t.kvh = unit % a.n_kv;
  if (!row_tile(a, units / a.n_kv - 1 - unit / a.n_kv, 2 * a.tile, t.rt)) return false;
  const RowTile& rt = t.rt;
  t.nflat = rt.n * a.group;
  // Positions [w0, p1] and, when a window has left them behind, the first `sinks`
  // of [0, w0), in tiles at multiples of TN: `ks` sink tiles, then those from kw.
  t.first = rt.ctx + rt.f0 / a.group;
  const int last = min(rt.f0 + 2 * a.tile, t.nflat) - 1, p0 = max(0, t.first);
  t.p1 = rt.ctx + last / a.group;
  t.w0 = a.window && p0 >= a.window ? p0 + 1 - a.window : 0;
  t.kw = t.w0 / TN;
  t.ks = min((min(a.sinks, t.w0) + TN - 1) / TN, t.kw);
  // Tiles that this split walks; those of A end with its own last position.
  const unsigned all = t.p1 < 0 ? 0 : t.ks + t.p1 / TN + 1 - t.kw;
  t.j0 = (int)(all * (unsigned)split / (unsigned)splits);
  const int j1 = (int)(all * (unsigned)(split + 1) / (unsigned)splits);
  const int pa = rt.ctx + (min(rt.f0 + a.tile, t.nflat) - 1) / a.group;
  t.na = max(0, min(j1, pa < 0 ? 0 : t.ks + pa / TN + 1 - t.kw) - t.j0);
  t.nb = rt.f0 + a.tile < t.nflat ? j1 - t.j0 : 0;
  return true;
}
// Work is taken as it is needed: the grid has a CTA per item, and a CTA that runs
// takes over the item of one that has not started (cluster launch control), so
// ragged batches even out without a counter in memory.  The request for the next
// item is made with the loads of this one's last tile: early enough for its first
// tiles to follow without a gap, late enough for long items to be nearly done.
__device__ __forceinline__ void request_item(uint32_t answer, uint64_t* bar) {
  mbar_expect_tx(bar, 16);
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];"
               ::"r"(answer), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ int requested_item(uint32_t answer) {  // -1: none is left
  int got, x;
  asm volatile(
      "{\n .reg .b128 h;\n .reg .pred p;\n .reg .b32 y, z, w;\n"
      " ld.shared.b128 h, [%2];\n"
      " clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n"
      " selp.s32 %0, 1, 0, p;\n mov.b32 %1, 0;\n"
      " @p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, y, z, w}, h;\n}\n"
      : "=r"(got), "=r"(x) : "r"(answer) : "memory");
  return got ? x : -1;
}

template <typename T, int HD>
__global__ void __launch_bounds__(TC_THREADS, 1)
paged_prefill_tc_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ CUtensorMap map_k,
                        const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_q, int items,
                        int splits, int box) {
  using C = TcPrefill<HD>;
  constexpr int PIECES = HD / 8, RPW = 32 / PIECES;  // 16-byte pieces of a row; rows per round of a warp
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  TcBars& bar = *reinterpret_cast<TcBars*>(smem + 6 * C::TILE + C::OUT);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t sq = smem_u32(smem), sk = sq + 2 * C::TILE, sv = sq + 4 * C::TILE;

  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&bar.tmem)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  } else if (threadIdx.x == 0) {
    for (int i = 0; i < 4; ++i) bar.mended[i] = 0;
    mbar_init(&bar.q_full, 1);
    mbar_init(&bar.q_freed, 1);
    mbar_init(&bar.done, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar.k_full[i], box ? 2 : 3);  // warp 10 twice, or warps 9 to 11
      mbar_init(&bar.v_full[i], 3);
      mbar_init(&bar.k_freed[i], 1);
      mbar_init(&bar.v_freed[i], 1);
      mbar_init(&bar.v_raw[i], 1);
      mbar_init(&bar.s_full[i], 1);
      mbar_init(&bar.p_full[i], 4);  // the tile's four warps
      mbar_init(&bar.o_full[i], 1);
      mbar_init(&bar.next_full[i], 1);
      mbar_init(&bar.next_read[i], TC_THREADS / 32);
    }
    fence_mbar_init();
  } else if (warp == 10 && lane == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_q)) : "memory");
    if (box) {
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_k)) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_v)) : "memory");
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // All 512 columns are this CTA's, so its block starts at column 0: TMEM
  // addresses are constants (S at w * TN, O at 256 + w * HD).
  const uint32_t tmem = bar.tmem;
  bool ok = true;  // one answer per warp; a wait that gave up ends the warp's work
  TcItem it;
  // The CTA's items: number 0 is its own, number q >= 1 the answer to request q (slot q & 1).
  auto phase_of = [](int q) { return (((q + 1) >> 1) - 1) & 1; };
  auto request = [&](int q) {
    if (q >= 3) ok = ok && warp_wait(&bar.next_read[q & 1], phase_of(q - 2));  // every warp has read the slot's last answer
    if (ok && lane == 0) request_item(smem_u32(&bar.answer[q & 1]), &bar.next_full[q & 1]);
  };
  auto next_item = [&](int q) -> int {
    ok = ok && warp_wait(&bar.next_full[q & 1], phase_of(q));
    if (!ok) return -1;
    const int i = requested_item(smem_u32(&bar.answer[q & 1]));
    fence_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&bar.next_read[q & 1]);
    return i;
  };

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
      auto qk = [&](int w, int kt) {
        const uint64_t q = dq + w * (C::TILE >> 4), k = dk + (kt & 1) * (C::TILE >> 4);
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
      auto pv = [&](int w, int kt, bool first) {
        const uint64_t v = dv + (kt & 1) * (C::TILE >> 4);
        if (elect_one()) {
#pragma unroll
          for (int part = 1; part >= 0; --part)  // the low part of P, then the high one
#pragma unroll
            for (int kk = 0; kk < TN / 16; ++kk)
              mma_f16_ts(256 + w * HD, w * TN + part * (TN / 2) + kk * 8, v + kk * 128, id_o, !(first && part == 1 && kk == 0));
        }
        __syncwarp();
      };
      auto signal = [&](uint64_t* b) {  // when everything issued so far is complete
        if (elect_one()) mma_commit(b);
        __syncwarp();
      };
      auto wait = [&](uint64_t* b, int phase) {
        ok = ok && warp_wait(b, phase & 1);
        tc_fence_after();
      };
      int kt = 0, np[2] = {0, 0}, nq = 0;  // position tiles, P tiles of A and B, items so far
      for (int k = 1, i = blockIdx.x; i >= 0; i = next_item(k++)) {
        if (!tc_item(a, i, items, splits, it)) continue;
        const int n = it.tiles();
        wait(&bar.q_full, nq++);
        if (n > 0) {
          wait(&bar.k_full[kt & 1], kt >> 1);
          if (ok && it.na > 0) qk(0, kt);
          if (ok && it.nb > 0) qk(1, kt);
          if (ok) signal(&bar.k_freed[kt & 1]);
          wait(&bar.v_full[kt & 1], kt >> 1);
        }
        if (ok && n < 2) signal(&bar.q_freed);
        for (int j = 0; j < n && ok; ++j, ++kt) {
          const bool more = j + 1 < n;
#pragma unroll
          for (int w = 0; w < 2; ++w) {  // A and B in turn: one's products run under the other's softmax
            const int m = w ? it.nb : it.na;
            if (j < m) {
              wait(&bar.p_full[w], np[w]++);
              if (ok) pv(w, kt, j == 0);
              if (ok && j + 1 == m) signal(&bar.o_full[w]);
            }
            // (waits for the next tile pass while the product above runs)
            if (w == 0 && more) wait(&bar.k_full[(kt + 1) & 1], (kt + 1) >> 1);
            if (w == 1 && more) wait(&bar.v_full[(kt + 1) & 1], (kt + 1) >> 1);
            if (ok && j + 1 < m) qk(w, kt + 1);  // in order behind the product that reads P from the same columns
          }
          if (!ok) break;
          if (more) signal(&bar.k_freed[(kt + 1) & 1]);
          signal(&bar.v_freed[kt & 1]);
          if (j + 2 == n) signal(&bar.q_freed);  // behind the last use of Q
        }
      }
      signal(&bar.done);
      warp_wait(&bar.done, 0);  // nothing is in flight when the columns are given back
    } else {
      // ---------------- Q rows, K / V tiles ----------------
      const int pc = lane % PIECES, sub = lane / PIECES;
      auto landed = [&](uint64_t* full) {  // this warp's writes are in shared memory
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(full);
      };
      int kt = 0, nq = 0, ni = -1;
      unsigned edges = 0;  // phase of v_raw[i] in bit i
      for (int k = 1, i = blockIdx.x; i >= 0; i = next_item(k++)) {
        const bool any = tc_item(a, i, items, splits, it);
        if (warp == 10 && (!any || it.tiles() == 0)) request(k);
        if (!any) continue;
        const RowTile& rt = it.rt;
        const int32_t* table = a.kv.table + rt.s * a.kv.table_stride;
        const int n = it.tiles(), p1 = it.p1, w0 = it.w0;
        ++ni;
        if (warp == 10) {  // Q: both tiles, a box of (64 values, group, tokens of a tile) each
          if (nq) ok = warp_wait(&bar.q_freed, (nq - 1) & 1);
          if (!ok) break;
          ++nq;
          constexpr int ATOMS = HD / 64;
          const bool two = rt.f0 + a.tile < it.nflat;
          if (lane == 0) mbar_expect_tx(&bar.q_full, (two ? 2 : 1) * ATOMS * a.tile * 128);
          __syncwarp();
          if (lane < (two ? 2 : 1) * ATOMS) {
            const int at = lane % ATOMS, tl = lane / ATOMS;
            tma_load_3d(sq + tl * C::TILE + at * C::ATOM, &map_q, at * 64, it.kvh * a.group, rt.r0 + (rt.f0 + tl * a.tile) / a.group,
                        &bar.q_full);
          }
        }
        // by TMA: lane i loads box i / ATOMS, values 64 (i % ATOMS) ...; boxes in which no
        // position is seen are left out (their pages may be gone)
        auto boxes = [&](const CUtensorMap* map, uint32_t dst, int t0, uint64_t* full) {
          constexpr int ATOMS = HD / 64;
          const int b = lane / ATOMS, at = lane % ATOMS, pos = t0 + b * box;
          const bool mine = b * box < TN && pos <= p1 && (pos + box > w0 || pos < a.sinks);
          int page = mine ? __ldg(table + (pos >> a.kv.page_shift)) : 0;
          if ((unsigned)page >= (unsigned)a.kv.n_pages) {
            flag_error(DEV_ERR_BAD_ARG);
            page = 0;
          }
          const unsigned live = __ballot_sync(0xffffffffu, mine);
          if (lane == 0) mbar_expect_tx(full, __popc(live) * box * 128);
          __syncwarp();
          if (mine)
            tma_load_4d(dst + at * C::ATOM + b * box * 128, map, at * 64, pos & ((1 << a.kv.page_shift) - 1), it.kvh, page, full);
        };
        // by rows
        auto rows = [&](const char* src, uint32_t dst, int t0) {
          src += it.kvh * a.kv.head_stride + pc * 16;
          const uint32_t d = dst + (pc >> 3) * C::ATOM;
#pragma unroll 4
          for (int r = (warp - 9) * RPW + sub; r < TN; r += 3 * RPW) {
            const int pos = t0 + r;
            const bool live = pos <= p1 && (pos >= w0 || pos < a.sinks);
            const long long off = live ? page_row(a.kv, __ldg(table + (pos >> a.kv.page_shift)), pos) : 0;
            cpa16(d + r * 128 + (((pc & 7) ^ (r & 7)) << 4), src + off, live);
          }
          cpa_commit();
        };
        // V rows of an edge tile in shared memory, this lane's piece of row r at place(r): zeros in place of infinities and NaN
        auto look = [&](auto place, int r0, auto rounds, int step) {
          uint32_t odd = 0, x[4];
          auto get = [&](uint32_t at) {
            asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(at) : "memory");
            return nonfinite2<T>(x[0]) | nonfinite2<T>(x[1]) | nonfinite2<T>(x[2]) | nonfinite2<T>(x[3]);
          };
#pragma unroll 8
          for (int i = 0; i < rounds; ++i) odd |= get(place(r0 + i * step));
          if (!__any_sync(0xffffffffu, odd & 0x80008000u)) return;
          if (lane == 0) bar.mended[ni & 3] = ni + 1;
#pragma unroll 1
          for (int i = 0; i < rounds; ++i)
            if (get(place(r0 + i * step)) & 0x80008000u) {
#pragma unroll
              for (int c = 0; c < 4; ++c) x[c] &= ~(((nonfinite2<T>(x[c]) & 0x80008000u) >> 15) * 0xffffu);
              asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};"
                           ::"r"(place(r0 + i * step)), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]) : "memory");
            }
        };
        for (int j = 0; j < n; ++j, ++kt) {
          if (warp == 10 && j + 1 == n) request(k);
          const int t0 = it.pos(j), slot = kt & 1;
          const uint32_t ak = sk + slot * C::TILE, av = sv + slot * C::TILE;
          // (with boxes warps 9 and 11 only follow the edge tiles, by v_raw)
          const bool fills = warp == 10 || !box;
          if (fills && kt >= 2) ok = warp_wait(&bar.k_freed[slot], ((kt >> 1) - 1) & 1);
          if (!ok) break;
          if (!box) {
            rows(a.kv.k, ak, t0);
          } else if (warp == 10) {
            if (lane == 0) mbar_arrive(&bar.k_full[slot]);
            boxes(&map_k, ak, t0, &bar.k_full[slot]);
          }
          if (fills && kt >= 2) ok = warp_wait(&bar.v_freed[slot], ((kt >> 1) - 1) & 1);
          if (!ok) break;
          if (!box) {
            rows(a.kv.v, av, t0);
            cpa_wait<1>();
            landed(&bar.k_full[slot]);
            cpa_wait<0>();
            if (it.edge(t0, a))
              look([&](int r) { return av + (pc >> 3) * C::ATOM + r * 128 + (((pc & 7) ^ (r & 7)) << 4); }, (warp - 9) * RPW + sub,
                   (TN - ((warp - 9) * RPW + sub) + 3 * RPW - 1) / (3 * RPW), 3 * RPW);
            landed(&bar.v_full[slot]);
          } else if (it.edge(t0, a)) {
            // an edge tile: zeros in place of the V rows that no query row sees, and a look at the others
            if (warp == 10) {
              if (lane == 0) mbar_arrive(&bar.v_full[slot]);
              boxes(&map_v, av, t0, &bar.v_raw[slot]);
            } else {
              ok = warp_wait(&bar.v_raw[slot], edges >> slot & 1);
              if (!ok) break;
              edges ^= 1u << slot;
              const int r0 = (warp == 11 ? TN / 2 : 0) + sub;
              if (t0 + TN > p1 + 1 || (t0 < w0 && t0 + TN > a.sinks))
                for (int r = r0; r < r0 + TN / 2; r += RPW) {
                  const int pos = t0 + r;
                  if (pos > p1 || (pos < w0 && pos >= a.sinks))
                    *reinterpret_cast<uint4*>(smem + (4 + slot) * C::TILE + (pc >> 3) * C::ATOM + r * 128 + ((pc & 7) << 4)) =
                        make_uint4(0, 0, 0, 0);
                }
              look([&](int r) { return av + (pc >> 3) * C::ATOM + r * 128 + ((pc & 7) << 4); }, r0,
                   std::integral_constant<int, TN / 2 / RPW>(), RPW);
              landed(&bar.v_full[slot]);
            }
          } else if (warp == 10) {
            if (lane < 2) mbar_arrive(&bar.v_full[slot]);
            boxes(&map_v, av, t0, &bar.v_full[slot]);
          }
        }
      }
      cpa_wait<0>();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_SOFTMAX));
    // ---------------- softmax: one row per thread ----------------
    const int w = warp >> 2, r = threadIdx.x & 127;
    const uint32_t ts = w * TN + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t to = 256 + w * HD + ((uint32_t)((warp & 3) * 32) << 16);
    int ns = 0, no = 0, ni = -1;  // S and O tiles, items so far
    for (int k = 1, item = blockIdx.x; item >= 0; item = next_item(k++)) {
      if (!tc_item(a, item, items, splits, it)) continue;
      ++ni;
      const RowTile& rt = it.rt;
      const int f = rt.f0 + w * a.tile + r;
      const bool row = r < a.tile && f < it.nflat;
      const int tok0 = (rt.f0 + w * a.tile) / a.group;  // the tile's first token
      // The row sees positions [0, va) (sinks) and [vb, vc).
      int va = 0, vb = 0, vc = 0x7fffffff;
      if (row) {
        vc = rt.ctx + tok0 + a.token(r) + 1;
        if (a.window) {
          vb = vc - a.window;
          va = a.sinks;
        }
      }
      const int m_tiles = w ? it.nb : it.na;
      float m = -INFINITY, l = 0.f;  // the maximum that P is relative to (in units of log2), the row's sum
      for (int j = 0; j < m_tiles; ++j) {
        ok = warp_wait(&bar.s_full[w], ns++ & 1);
        if (!ok) break;
        tc_fence_after();
        uint32_t s[TN];
#pragma unroll
        for (int c = 0; c < TN; c += 32) tmem_ld32(s + c, ts + c);
        tmem_wait_ld();
        const int v0 = it.pos(j);
        // Few tiles need a mask.  Written as a loop because the compiler turns an `if`
        // here into selects on every tile (830 of 2400 clocks).
        int masked = __any_sync(0xffffffffu, v0 + TN > vc || (v0 < vb && v0 + TN > va));
        asm volatile("" : "+r"(masked));
#pragma unroll 1
        for (; masked > 0; --masked) {
#pragma unroll
          for (int c = 0; c < TN; c += 32) {  // bit i: position v0 + c + i is seen
            const uint32_t see = below(vc - v0 - c) & (below(va - v0 - c) | ~below(vb - v0 - c));
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!(see >> i & 1)) s[c + i] = 0xff800000u;
          }
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < TN; i += 8)
#pragma unroll
          for (int q = 0; q < 4; ++q) mx[q] = max3(mx[q], __uint_as_float(s[i + 2 * q]), __uint_as_float(s[i + 2 * q + 1]));
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale2;
        if (__any_sync(0xffffffffu, top > m + Range<T>::LAG)) {
          const float mn = fmaxf(m, top), f2o = m == -INFINITY ? 0.f : ex2(m - mn);
          m = mn;
          l *= f2o;
          if (j > 0) {  // every product so far is complete: S was issued behind them
#pragma unroll 1
            for (int c = 0; c < HD; c += 32) {
              uint32_t o[32];
              tmem_ld32(o, to + c);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f2o);
              tmem_st32(to + c, o);
            }
          }
        }
        const float b = m == -INFINITY ? 0.f : Range<T>::UP - m;
        const f2 scale = pk(a.scale2, a.scale2), base = pk(b, b);
        f2 sum[2] = {pk(0.f, 0.f), pk(0.f, 0.f)};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t hi[TN / 4], lo[TN / 4];
#pragma unroll
          for (int i = 0; i < TN / 4; ++i) {
            const int c = h * (TN / 2) + 2 * i;
            const f2 x = fma2(pk(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), scale, base);
            float u, v;
            unpk(x, u, v);
            u = ex2(u);
            v = ex2(v);
            const f2 p = pk(u, v);
            sum[i & 1] = add2(sum[i & 1], p);
            hi[i] = pack2<T>(u, v);
            const float2 r = unpack2<T>(hi[i]);
            unpk(sub2(p, pk(r.x, r.y)), u, v);
            lo[i] = pack2<T>(u, v);
          }
          tmem_st32(ts + h * (TN / 4), hi);
          tmem_st32(ts + TN / 2 + h * (TN / 4), lo);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.p_full[w]);
        l += hsum(add2(sum[0], sum[1]));
      }
      // ---------------- output ----------------
      if (ok && m_tiles > 0) ok = warp_wait(&bar.o_full[w], no++ & 1);
      if (!ok) break;
      tc_fence_after();
      float* part = a.part + (long long)item * C::SLOT;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const uint32_t stage = sq + 6 * C::TILE + warp * 32 * 128;  // 64 values of this warp's 32 rows
      // Rows go out whole, 8 lanes to 128 bytes: this lane's rows are lane / 8 + 4 i.
      T* dst[8];
      if (splits == 1) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int x = (warp & 3) * 32 + (lane >> 3) + 4 * i, t = a.token(x);
          dst[i] = x < a.tile && rt.f0 + w * a.tile + x < it.nflat
                       ? static_cast<T*>(a.out) + (rt.r0 + tok0 + t) * a.o_row + (long long)(it.kvh * a.group + x - t * a.group) * a.o_head + (lane & 7) * 8
                       : nullptr;
        }
      }
      f2 zero = pk(0.f, 0.f);  // 0 as long as the row's sums are finite, NaN otherwise
#pragma unroll 1
      for (int c = 0; c < HD; c += 64) {
        uint32_t o[64];
        if (m_tiles > 0) {
          tmem_ld32(o, to + c);
          tmem_ld32(o + 32, to + c + 32);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 64; i += 2) zero = fma2(pk(__uint_as_float(o[i]), __uint_as_float(o[i + 1])), pk(0.f, 0.f), zero);
        } else {
#pragma unroll
          for (int i = 0; i < 64; ++i) o[i] = 0u;
        }
        if (splits == 1) {
#pragma unroll
          for (int i = 0; i < 64; i += 8) {
            uint32_t x[4];
#pragma unroll
            for (int q = 0; q < 4; ++q)
              x[q] = pack2<T>(__uint_as_float(o[i + 2 * q]) * inv, __uint_as_float(o[i + 2 * q + 1]) * inv);
            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(stage + lane * 128 + (((i / 8) ^ (lane & 7)) << 4)),
                         "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]) : "memory");
          }
          __syncwarp();
          uint4 x[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int y = (lane >> 3) + 4 * i;
            asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(x[i].x), "=r"(x[i].y), "=r"(x[i].z), "=r"(x[i].w)
                         : "r"(stage + y * 128 + (((lane & 7) ^ (y & 7)) << 4)) : "memory");
          }
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (dst[i]) *reinterpret_cast<uint4*>(dst[i] + c) = x[i];
          __syncwarp();
        } else if (row) {
          float* d = part + 4 * TQ + (long long)(w * TQ + r) * HD + c;
#pragma unroll
          for (int i = 0; i < 64; i += 4)
            *reinterpret_cast<float4*>(d + i) = make_float4(__uint_as_float(o[i]), __uint_as_float(o[i + 1]),
                                                            __uint_as_float(o[i + 2]), __uint_as_float(o[i + 3]));
        }
      }
      if (splits > 1 && row) {
        part[w * TQ + r] = m_tiles > 0 ? m : -INFINITY;
        part[2 * TQ + w * TQ + r] = l;
      }
      // ---------------- infinities and NaN of V (take_nonfinite): such rows once more ----------------
      const bool in_edges = m_tiles > 0 && *reinterpret_cast<volatile int*>(&bar.mended[ni & 3]) == ni + 1;
      const bool in_others = __any_sync(0xffffffffu, row && l == l && hsum(zero) != 0.f);  // (a score of NaN: NaN it stays)
      if (in_edges || in_others) {
        RowSums<HD> x;
        for (uint32_t& y : x.set) y = 0;
        x.done = row ? 0u : ~0u;
#pragma unroll 1
        for (int c = 0; c < HD; c += 32) {
          uint32_t o[32];
          tmem_ld32(o, to + c);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) x.o[c + i] = __uint_as_float(o[i]);
        }
#pragma unroll 1
        for (int j = 0; j < m_tiles; ++j) {
          const int t0 = it.pos(j);
          if (it.edge(t0, a) ? in_edges : in_others)
            take_nonfinite<T, HD>(a, rt.s, it.kvh, t0, min(t0 + TN, it.p1 + 1), it.w0, va, vb, vc, x);
        }
        if (row) {
          const int t = a.token(r);
          T* out = static_cast<T*>(a.out) + (rt.r0 + tok0 + t) * a.o_row + (long long)(it.kvh * a.group + r - t * a.group) * a.o_head;
          for (int d = 0; d < HD; ++d) {
            if (splits == 1) out[d] = from_f<T>(x.o[d] * inv);
            else part[4 * TQ + (long long)(w * TQ + r) * HD + d] = x.o[d];
          }
        }
        __syncwarp();
      }
      tc_fence_before();  // O has been read: the next item's first product (behind its P) may replace it
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

// Adds the splits of an item's TILES x 128 rows, 16 rows per CTA:
// out = sum_i o_i 2^(m_i - M) / sum_i l_i 2^(m_i - M).
template <typename T, int HD, int TILES>
__global__ void __launch_bounds__(256) paged_prefill_join_kernel(const __grid_constant__ AttnArgs a, int splits) {
  constexpr int ROWS = TILES * TQ, SLOT = ROWS * (HD + 2), CTAS = ROWS / 16, V = 16 / sizeof(T), LANES = HD / V;
  const int unit = blockIdx.x / CTAS, kvh = unit % a.n_kv, units = gridDim.x / CTAS;
  RowTile rt;
  const bool any = row_tile(a, units / a.n_kv - 1 - unit / a.n_kv, TILES * a.tile, rt);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (!any) return;
  for (int x = threadIdx.x; x < 16 * LANES; x += 256) {
    const int r = (blockIdx.x % CTAS) * 16 + x / LANES, c = (x % LANES) * V;  // row r % TQ of tile r / TQ
    const int f = rt.f0 + (r / TQ) * a.tile + r % TQ;
    if (r % TQ >= a.tile || f >= rt.n * a.group) continue;
    const float* p = a.part + (long long)unit * splits * SLOT;
    float M = -INFINITY, L = 0.f, acc[V] = {};
    for (int i = 0; i < splits; ++i) M = fmaxf(M, p[(long long)i * SLOT + r]);
    const float b = M == -INFINITY ? 0.f : M;
#pragma unroll 4
    for (int i = 0; i < splits; ++i) {
      const float* q = p + (long long)i * SLOT;
      const float e = fmaxf(exp2f(q[r] - b), TINY);
      L += q[ROWS + r] * e;
#pragma unroll
      for (int k = 0; k < V; k += 4) {
        const float4 u = *reinterpret_cast<const float4*>(q + 2 * ROWS + (long long)r * HD + c + k);
        acc[k] += u.x * e; acc[k + 1] += u.y * e; acc[k + 2] += u.z * e; acc[k + 3] += u.w * e;
      }
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] *= inv;
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

// TMA map of the query rows, (value, head, token), in boxes of 64 values x a kv head's
// group x the tokens of a tile.  (Strides of axes of one entry are never used; a
// caller may have left 0 there.)
static bool query_map(CUtensorMap* map, const AttnArgs& a, bool half, int hd) {
  auto fn = tmap_encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)a.n_kv * a.group, (cuuint64_t)a.rows};
  const cuuint64_t strides[2] = {(cuuint64_t)a.q_head * 2, (cuuint64_t)(a.q_row ? a.q_row : a.q_head) * 2};
  const cuuint32_t boxes[3] = {64, (cuuint32_t)a.group, (cuuint32_t)(TQ / a.group)}, ones[3] = {1, 1, 1};
  return fn(map, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(a.q), dims,
            strides, boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Whether the kernel was built with the registers that its split adds up to.
template <auto KERN>
static cudaError_t check_register_split(int dev, int threads, int sum) {
  static std::atomic<int> known[VTB_MAX_DEVICES];
  if (known[dev].load(std::memory_order_relaxed)) return cudaSuccess;
  cudaFuncAttributes f;
  const cudaError_t e = cudaFuncGetAttributes(&f, KERN);
  if (e) return e;
  if (f.numRegs / 8 * 8 * threads < sum) return cudaErrorInvalidConfiguration;
  known[dev].store(1, std::memory_order_relaxed);
  return cudaSuccess;
}

// Query rows of a tile of up to `rows` (whole tokens), and a positive scale.
static void set_tile(AttnArgs& a, int rows) {
  a.tile = rows / a.group * a.group;
  a.recip = 65536 / a.group + 1;
  a.negate = a.scale2 < 0.f;
  a.scale2 = fmaxf(fabsf(a.scale2), 1e-36f);  // not 0: masked scores have to stay -inf
}
// Fewer items than SMs: the positions are split too, down to two tiles of
// positions per CTA (below that the join costs more than the split gives).
static int prefill_splits(const AttnArgs& a, long long units, int tile, int sms) {
  const long long cap = (long long)a.kv.pages_per_seq << a.kv.page_shift;
  long long seen = a.window ? (long long)a.window + a.sinks + a.rows : cap;
  if (seen > cap) seen = cap;
  long long splits = sms / units;
  if (splits > seen / (2 * tile)) splits = seen / (2 * tile);
  return splits > 1 ? (int)splits : 1;
}

template <typename T, int HD>
static cudaError_t launch_prefill_tc_t(AttnArgs a, cudaStream_t st) {
  using C = TcPrefill<HD>;
  const int dev = current_device();
  cudaError_t e = ensure_smem_attr<paged_prefill_tc_kernel<T, HD>>(dev, C::SMEM);
  if (e || (e = check_register_split<paged_prefill_tc_kernel<T, HD>>(dev, TC_THREADS, 256 * REGS_SOFTMAX + 128 * REGS_OTHER)))
    return e;
  set_tile(a, TQ);
  const long long units = ((long long)a.rows * a.group / (2 * a.tile) + a.kv.n_seqs) * a.n_kv;
  if (units > 0x7fffffffll / 16) return cudaErrorInvalidValue;
  const int splits = prefill_splits(a, units, TN, sm_count(dev));
  CUtensorMap map_k = {}, map_v = {};
  const int slots = 1 << a.kv.page_shift, fit = slots < TN ? slots : TN;
  CUtensorMap map_q = {};
  if (!query_map(&map_q, a, std::is_same<T, __half>::value, HD)) return cudaErrorInvalidValue;
  const int box = slots >= 8 && page_map(&map_k, a.kv, a.kv.k, std::is_same<T, __half>::value, HD, a.n_kv, fit) &&
                          page_map(&map_v, a.kv, a.kv.v, std::is_same<T, __half>::value, HD, a.n_kv, fit) ? fit : 0;
  const long long items = units * splits;
  paged_prefill_tc_kernel<T, HD><<<(unsigned)items, TC_THREADS, C::SMEM, st>>>(a, map_k, map_v, map_q, (int)items, splits, box);
  if ((e = cudaGetLastError()) || splits == 1) return e;
  return launch_dependent(paged_prefill_join_kernel<T, HD, 2>, dim3((unsigned)(units * 16)), dim3(256), 0, st, a, splits);
}

cudaError_t launch_paged_prefill_tc(int type, int head_dim, const AttnArgs& a, cudaStream_t st) {
  if (type == T_F16) return head_dim == 64 ? launch_prefill_tc_t<__half, 64>(a, st) : launch_prefill_tc_t<__half, 128>(a, st);
  return head_dim == 64 ? launch_prefill_tc_t<__nv_bfloat16, 64>(a, st) : launch_prefill_tc_t<__nv_bfloat16, 128>(a, st);
}

}  // namespace vtb
