// paged.cuh -- shared device code of the paged key-value cache: where a
// position's rows lie, which positions a query sees, and the warp-level
// attention step over 16 cached positions.
//
// The step computes S^T = K Q^T and O^T += V^T P^T with positions (and head
// dimensions) on the 16-row side of mma.sync and 8 query vectors on its
// 8-column side, so a group of up to 8 query heads that share a kv head fills
// the instruction and every K and V element is loaded from shared memory once.
// One query token does 2 G flops per cached element, far below what the
// legacy tensor path gives at HBM rate, so mma.sync (whose operands need no
// TMEM round trip) is enough here.
#pragma once
#include <type_traits>

#include "common.cuh"

namespace vtb {

// ggml type ids of the cache and row types (F32 = 0 in common.cuh).
constexpr int T_F16 = 1, T_BF16 = 30;

struct PagedView {  // strides in bytes
  const char* k;
  const char* v;
  long long page_stride, head_stride, slot_stride;
  const int32_t* table;
  long long table_stride;  // entries
  int n_pages, n_seqs, pages_per_seq, page_shift;
};

// Bytes from the base of K (or V) to row (page of position t, t's slot); the
// page id is checked, so a bad table sets the error word instead of reading
// outside the cache (the row of page 0 is read in its place).
__device__ __forceinline__ long long page_row(const PagedView& kv, int page, int t) {
  if ((unsigned)page >= (unsigned)kv.n_pages) {
    flag_error(DEV_ERR_BAD_ARG);
    page = 0;
  }
  return page * kv.page_stride + (t & ((1 << kv.page_shift) - 1)) * kv.slot_stride;
}

// Cached length of a sequence, held within its page table.
__device__ __forceinline__ int paged_len(const PagedView& kv, const int32_t* lens, int s) {
  const int n = lens[s];
  const long long cap = (long long)kv.pages_per_seq << kv.page_shift;
  if (n > cap) {
    flag_error(DEV_ERR_BAD_ARG);
    return (int)cap;
  }
  return n < 0 ? 0 : n;
}

template <typename T> struct Elem;
template <> struct Elem<float> { static constexpr bool f32 = true; };
template <> struct Elem<__half> { static constexpr bool f32 = false; };
template <> struct Elem<__nv_bfloat16> { static constexpr bool f32 = false; };

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Two values as one packed 16-bit pair (a in the low half), rounded to nearest.
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t p);
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t p) {
  return __half22float2(*reinterpret_cast<const __half2*>(&p));
}
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t p) {
  return make_float2(__uint_as_float(p << 16), __uint_as_float(p & 0xffff0000u));
}

__device__ __forceinline__ void ldsm4(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t movm(uint32_t x) {  // transpose an 8 x 8 tile of 16-bit values
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ float4 lds_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
template <typename T>
__device__ __forceinline__ void mma16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16<__half>(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16<__nv_bfloat16>(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x = hi + lo with both in tf32 (11 significant bits): hi rounded to nearest,
// so lo's sign is free and cutting it to 11 bits (relative 2^-21 of x at most)
// has no bias.  A product of two split values drops lo * lo, 2^-22 relative.
// (half = 0 cuts hi off instead, 2 bits worse in all: for finite values from 0x7f7ff000
// on, which would round to infinity.)
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo, uint32_t half = 0x1000u) {
  hi = (__float_as_uint(x) + half) & 0xffffe000u;
  lo = __float_as_uint(x - __uint_as_float(hi)) & 0xffffe000u;
}

__device__ __forceinline__ void cpa16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cpa_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cpa_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// ---- one warp, 16 positions, NT * 8 query vectors ----
// Lane (g = lane / 4, t = lane % 4).  Scores s[nt][0..3] are (position g,
// vector 8 nt + 2t), (g, 2t + 1), (g + 8, 2t), (g + 8, 2t + 1); o[nt][j][0..3] are
// (dimension dim(j, 0), vector 2t), (same, 2t + 1), (dim(j, 1), 2t), (same, 2t + 1).
template <typename T, int HD, int NT, bool F32 = Elem<T>::f32> struct Step;

// 16-bit types: m16n8k16 with ldmatrix; rows of HD values with their 16-byte
// pieces swizzled by the row (piece ^ row % 8), so ldmatrix is conflict-free.
// P enters the second product as a sum of two 16-bit values, which keeps it
// exact to 2^-17 (bf16): the output then carries its own rounding only.  f16 ends at
// steps of 2^-24: P is kept times 2^15, which holds weights to 2^-40 of the largest
// (they would be lost from the products, but not from the sum).
template <typename T, int HD, int NT> struct Step<T, HD, NT, false> {
  static constexpr bool F = false;
  static constexpr int UP = std::is_same<T, __half>::value ? 15 : 0;
  static constexpr int PIECES = HD / 8, ROW = HD * 2;  // 16-byte pieces and bytes of a staged row
  static constexpr int QREGS = HD / 8;
  uint32_t q[NT][QREGS];

  static __device__ __forceinline__ uint32_t k_off(int r, int piece) { return r * ROW + ((piece ^ (r & 7)) << 4); }
  static __device__ __forceinline__ uint32_t v_off(int r, int piece) { return r * ROW + ((piece ^ (r & 7)) << 4); }
  // Vector 8 nt + g's values, read from `p` (null: a vector of zeros).
  __device__ __forceinline__ void load_q(int nt, const T* p, int t) {
#pragma unroll
    for (int j = 0; j < HD / 16; ++j) {
      q[nt][2 * j] = p ? *reinterpret_cast<const uint32_t*>(p + 16 * j + 2 * t) : 0u;
      q[nt][2 * j + 1] = p ? *reinterpret_cast<const uint32_t*>(p + 16 * j + 8 + 2 * t) : 0u;
    }
  }
  __device__ __forceinline__ void scores(uint32_t kbase, int lane, float (&s)[NT][4]) const {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
    const int r = lane & 15, pc = lane >> 4;
#pragma unroll
    for (int j = 0; j < HD / 16; ++j) {
      uint32_t a[4];
      ldsm4(a, kbase + k_off(r, 2 * j + pc));
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) mma16<T>(s[nt], a, q[nt][2 * j], q[nt][2 * j + 1]);
    }
  }
  // o = o * f + V^T P^T (f: the factor of each of the lane's vectors; all 1 unless `moved`)
  __device__ __forceinline__ void pv(uint32_t vbase, int lane, const float (&p)[NT][4], const float (&f)[NT][2], bool moved,
                                     float (&o)[NT][HD / 16][4]) const {
    if (moved) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < HD / 16; ++j) {
          o[nt][j][0] *= f[nt][0]; o[nt][j][2] *= f[nt][0];
          o[nt][j][1] *= f[nt][1]; o[nt][j][3] *= f[nt][1];
        }
    }
    uint32_t bh[NT][2], bl[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t hi = pack2<T>(p[nt][2 * h], p[nt][2 * h + 1]);
        const float2 r = unpack2<T>(hi);
        bh[nt][h] = movm(hi);
        bl[nt][h] = movm(pack2<T>(p[nt][2 * h] - r.x, p[nt][2 * h + 1] - r.y));
      }
    const int r = (lane & 7) + ((lane >> 4) << 3), pc = (lane >> 3) & 1;
#pragma unroll
    for (int j = 0; j < HD / 16; ++j) {
      uint32_t a[4];
      ldsm4_t(a, vbase + v_off(r, 2 * j + pc));
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        mma16<T>(o[nt][j], a, bl[nt][0], bl[nt][1]);
        mma16<T>(o[nt][j], a, bh[nt][0], bh[nt][1]);
      }
    }
  }
  static __device__ __forceinline__ int dim(int j, int hi, int g) { return 16 * j + 8 * hi + g; }
};

// f32: m16n8k8 tf32 on values split in two, three products each (hi lo, lo hi,
// hi hi): 2^-21 relative, f32-class sums, at a cost that does not grow with the
// group.  The order of the head dimensions inside a product is free as long as
// both operands share it, so a lane reads whole 16-byte pieces: score step
// (jj, cc) holds dimensions 4 (t + 4 jj) + 2 cc + {0, 1} of lane t, output tile
// (jj, cc) dimensions 4 (g + 8 jj) + 2 cc + {0, 1} of lane g.  The eight lanes of a
// 128-byte phase read 4 pieces of two rows of K, 2 pieces of four rows of V: the
// pieces are swizzled by the row so that these fall into different banks.
template <int HD, int NT> struct Step<float, HD, NT, true> {
  static constexpr bool F = true;
  static constexpr int UP = 0;
  static constexpr int PIECES = HD / 4, ROW = HD * 4;
  static constexpr int QREGS = HD / 4;
  float q[NT][QREGS];

  static __device__ __forceinline__ uint32_t k_off(int r, int piece) { return r * ROW + ((piece ^ ((r & 1) << 2)) << 4); }
  static __device__ __forceinline__ uint32_t v_off(int r, int piece) { return r * ROW + ((piece ^ (r & 6)) << 4); }
  __device__ __forceinline__ void load_q(int nt, const float* p, int t) {
#pragma unroll
    for (int jj = 0; jj < HD / 16; ++jj) {
      const float4 v = p ? *reinterpret_cast<const float4*>(p + 4 * (t + 4 * jj)) : make_float4(0.f, 0.f, 0.f, 0.f);
      q[nt][4 * jj] = v.x; q[nt][4 * jj + 1] = v.y; q[nt][4 * jj + 2] = v.z; q[nt][4 * jj + 3] = v.w;
    }
  }
  // The tensor cores add their products to the accumulator with truncation, so
  // a long chain drifts by half a last place per step, all in one direction.
  // Chains are therefore short: the small cross terms have accumulators of
  // their own, the leading ones two, and o is updated by an ordinary f32 add.
  __device__ __forceinline__ void scores(uint32_t kbase, int lane, float (&s)[NT][4]) const {
    float big[2][NT][4], small[2][NT][4];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c) big[i][nt][c] = small[i][nt][c] = 0.f;
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int jj = 0; jj < HD / 16; ++jj) {
      const float4 ka = lds_f4(kbase + k_off(g, t + 4 * jj)), kb = lds_f4(kbase + k_off(g + 8, t + 4 * jj));
      const float va[4] = {ka.x, ka.y, ka.z, ka.w}, vb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
      for (int cc = 0; cc < 2; ++cc) {
        uint32_t ah[4], al[4];
        split_tf32(va[2 * cc], ah[0], al[0]);
        split_tf32(vb[2 * cc], ah[1], al[1]);
        split_tf32(va[2 * cc + 1], ah[2], al[2]);
        split_tf32(vb[2 * cc + 1], ah[3], al[3]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          uint32_t h0, l0, h1, l1;
          split_tf32(q[nt][4 * jj + 2 * cc], h0, l0);
          split_tf32(q[nt][4 * jj + 2 * cc + 1], h1, l1);
          mma_tf32(small[0][nt], al, h0, h1);
          mma_tf32(small[1][nt], ah, l0, l1);
          mma_tf32(big[cc][nt], ah, h0, h1);
        }
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 4; ++c) s[nt][c] = (big[0][nt][c] + big[1][nt][c]) + (small[0][nt][c] + small[1][nt][c]);
  }
  __device__ __forceinline__ void pv(uint32_t vbase, int lane, const float (&p)[NT][4], const float (&f)[NT][2], bool,
                                     float (&o)[NT][HD / 16][4]) const {
    const int g = lane >> 2, t = lane & 3;
    // P^T of positions 8h + 2t, 8h + 2t + 1 for vector g: the 32-bit tile is
    // transposed as two tiles of 16-bit halves
    uint32_t bh[2][NT][2], bl[2][NT][2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const uint32_t x = __float_as_uint(p[nt][2 * h]), y = __float_as_uint(p[nt][2 * h + 1]);
        const uint32_t lo = movm(__byte_perm(x, y, 0x5410)), hi = movm(__byte_perm(x, y, 0x7632));
        split_tf32(__uint_as_float(__byte_perm(lo, hi, 0x5410)), bh[h][nt][0], bl[h][nt][0]);
        split_tf32(__uint_as_float(__byte_perm(lo, hi, 0x7632)), bh[h][nt][1], bl[h][nt][1]);
      }
#pragma unroll
    for (int jj = 0; jj < HD / 32; ++jj) {
      float c[2][NT][4];
#pragma unroll
      for (int cc = 0; cc < 2; ++cc)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) c[cc][nt][0] = c[cc][nt][1] = c[cc][nt][2] = c[cc][nt][3] = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float4 f0 = lds_f4(vbase + v_off(8 * h + 2 * t, g + 8 * jj));
        const float4 f1 = lds_f4(vbase + v_off(8 * h + 2 * t + 1, g + 8 * jj));
        const float va[4] = {f0.x, f0.y, f0.z, f0.w}, vb[4] = {f1.x, f1.y, f1.z, f1.w};
#pragma unroll
        for (int cc = 0; cc < 2; ++cc) {
          uint32_t ah[4], al[4];
          split_tf32(va[2 * cc], ah[0], al[0]);
          split_tf32(va[2 * cc + 1], ah[1], al[1]);
          split_tf32(vb[2 * cc], ah[2], al[2]);
          split_tf32(vb[2 * cc + 1], ah[3], al[3]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma_tf32(c[cc][nt], al, bh[h][nt][0], bh[h][nt][1]);
            mma_tf32(c[cc][nt], ah, bl[h][nt][0], bl[h][nt][1]);
            mma_tf32(c[cc][nt], ah, bh[h][nt][0], bh[h][nt][1]);
          }
        }
      }
#pragma unroll
      for (int cc = 0; cc < 2; ++cc)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[nt][2 * jj + cc][i] = fmaf(o[nt][2 * jj + cc][i], f[nt][i & 1], c[cc][nt][i]);
    }
  }
  static __device__ __forceinline__ int dim(int j, int hi, int g) { return 4 * (g + 8 * (j >> 1)) + 2 * (j & 1) + hi; }
};

// Online softmax of the warp's 16 scores per vector (in units of log2): m is
// the running maximum, l this lane's share of the running sum.  A row whose
// maximum is still -inf keeps p = 0.  On return s holds p, f the factors that
// o needs (all 1 unless the result is true, the same for the whole warp).  p and l
// are kept times 2^UP.
template <int NT, int UP>
__device__ __forceinline__ bool softmax_step(float (&s)[NT][4], float (&m)[NT][2], float (&l)[NT][2], float (&f)[NT][2]) {
  bool moved = false;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float x = fmaxf(s[nt][c], s[nt][c + 2]);
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, off));
      const float mn = fmaxf(m[nt][c], x), base = mn == -INFINITY ? 0.f : mn - UP;
      f[nt][c] = exp2f(m[nt][c] - (mn == -INFINITY ? 0.f : mn));
      moved |= mn != m[nt][c];
      m[nt][c] = mn;
      s[nt][c] = exp2f(s[nt][c] - base);
      s[nt][c + 2] = exp2f(s[nt][c + 2] - base);
      l[nt][c] = l[nt][c] * f[nt][c] + (s[nt][c] + s[nt][c + 2]);
    }
  return __any_sync(0xffffffffu, moved);
}

}  // namespace vtb
