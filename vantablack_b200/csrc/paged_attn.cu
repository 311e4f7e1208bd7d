// paged_attn.cu -- attention over the paged key-value cache, with a sliding
// window and sinks (first positions that stay visible): one new token per
// sequence (decode), and what the chunk (prefill) kernels share.
//
//   o = sum_t softmax_t(scale q . k_t) v_t over the visible t:
//   t <= p, t < len, and (window == 0 or t > p - window or t < sinks)
//
// for a query at position p; a query that sees nothing gives 0.
#include "paged.cuh"

namespace vtb {

struct AttnArgs {
  PagedView kv;
  const void* q;
  void* out;
  long long q_row, q_head, o_row, o_head;  // elements
  const int32_t* lens;
  const int32_t* starts;  // prefill: first row of each sequence, then the number of rows
  int rows, n_kv, group, window, sinks;
  float scale2;  // scale * log2(e): scores are kept in units of log2
  int tile;      // tensor-core prefill: query rows of a tile, and 2^16 / group + 1
  int recip;
  bool negate;   // tensor-core prefill: the scale is negative (scale2 holds its size)
  float* part;   // partial results of splits
  // Token of row x < 256 of a tile: x / group for group <= 128 (x * (recip * group - 2^16) < 2^16).
  __device__ __forceinline__ int token(int x) const { return x * recip >> 16; }
};

// A run of cached positions as one index range: `ns` sinks, then [w0, end).
struct Span {
  int ns, w0, n;
  __device__ __forceinline__ int pos(int i) const { return i < ns ? i : i - ns + w0; }
};
// Positions that queries at [p0, p1] see (p0 <= p1; p1 < 0: none).
__device__ __forceinline__ Span span_of(int p0, int p1, int window, int sinks) {
  Span s{0, 0, 0};
  if (p1 < 0) return s;
  if (window && p0 >= window) s.w0 = p0 + 1 - window;
  s.ns = min(sinks, s.w0);
  s.n = s.ns + p1 + 1 - s.w0;
  return s;
}

// Factors between maxima are not let down to 0, so that an infinity stays one in parts
// that weigh nothing (finite parts of them stay below anything that counts).
constexpr float TINY = 1.2e-38f;

// ======================= decode =======================
// HBM bound: K and V are read once.  The visible positions of every (sequence,
// kv head) are cut into tiles of 16 per warp, all tiles put in one line, and the line
// cut into equal parts, one per resident CTA: a ragged batch and a single long
// sequence load the GPU the same way, with no host knowledge of the lengths
// (a captured call stays right as they grow).  A part that covers a whole
// (sequence, kv head) writes its output; the others leave (max, sum, o) behind
// and decode_join_kernel adds them in line order, so results do not depend on
// timing.  Each of the CTA's warps streams its own 16 positions of a tile
// through a private cp.async ring, with no barrier but at a part's end.
// Measured, with the join: one sequence of 131009 (8 kv heads x 128, bf16, 537 MB)
// 93 us, the main kernel alone at 6.5 TB/s; 32 sequences of 2049 to 2560 in f32
// (604 MB) 109 to 121 us, bound by issue (52% active) and the latency of the split
// products; 61 sequences behind a window of 1024 in f16 (124 MB) 34 us, of which
// the plan, the ring's start and the join are half; 37 positions 4.7 us.

template <typename T, int HD, int NT> struct DecodeCfg {
  using S = Step<T, HD, NT>;
  // A warp's ring holds the K and V rows of 16 positions, STAGES times; for f32 at 128 values, where
  // eight warps have no room for two stages, K and V take turns in three halves (8 warps at 5.5 TB/s,
  // 6 with two whole stages at 5.0; in halves the smaller rows lose 5 to 10%).
  static constexpr int WARPS = S::F || HD == 64 ? 8 : 4, TILE = 16 * WARPS;
  static constexpr bool HALVES = S::F && HD == 128;
  static constexpr int STAGES = S::F && HD == 64 ? 2 : 3, ROWS = 16 * S::ROW, STAGE = HALVES ? ROWS : 2 * ROWS;
  static constexpr int RED = WARPS * 4 * (HD + 4) * 4;  // the warps' o of 4 query vectors
  static constexpr int SMEM = WARPS * STAGES * STAGE + RED + WARPS * 8 * 2 * 4;
  static constexpr int SLOT = NT * 8 * (HD + 2);  // floats of one partial result
};

struct Line {  // the line of all tiles, cut into `parts`: the first `rest` of them one tile longer than `each`
  long long total, each;
  int parts, rest;
  __device__ __forceinline__ long long start(int c) const { return c * each + min(c, rest); }
};
template <int TILE> __device__ __forceinline__ int seq_tiles(const AttnArgs& a, int s) {
  const int len = paged_len(a.kv, a.lens, s);
  return (span_of(len - 1, len - 1, a.window, a.sinks).n + TILE - 1) / TILE;
}
template <int TILE> __device__ __forceinline__ Line line_of(const AttnArgs& a, int units, int grid) {
  long long n = 0;
  for (int s = threadIdx.x & 31; s < a.kv.n_seqs; s += 32) n += seq_tiles<TILE>(a, s);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  n *= units;
  if (n <= grid) return Line{n, 1, (int)n, 0};
  const long long each = n < (1ll << 32) ? (unsigned)n / (unsigned)grid : n / grid;
  return Line{n, each, grid, (int)(n - each * grid)};
}
// The sequence that holds place `w` of the line, and the tiles before it.
template <int TILE> __device__ __forceinline__ int line_seq(const AttnArgs& a, int units, long long w, long long& before) {
  before = 0;
  const int lane = threadIdx.x & 31;
  for (int s0 = 0; s0 < a.kv.n_seqs; s0 += 32) {
    long long n = s0 + lane < a.kv.n_seqs ? (long long)seq_tiles<TILE>(a, s0 + lane) * units : 0, incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, before + incl > w);
    if (hit) {
      const int l = __ffs(hit) - 1;
      before += __shfl_sync(0xffffffffu, incl - n, l);
      return s0 + l;
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
  return -1;
}

template <int TILE> struct LineCursor {  // one tile of the line
  int s, u, t, nt;
  Span sp;
  __device__ __forceinline__ void enter(const AttnArgs& a) {
    const int len = paged_len(a.kv, a.lens, s);
    sp = span_of(len - 1, len - 1, a.window, a.sinks);
    nt = (sp.n + TILE - 1) / TILE;
  }
  __device__ __forceinline__ void place(long long at) {  // `at` tiles into the sequence
    u = at < (1ll << 32) ? (int)((unsigned)at / (unsigned)nt) : (int)(at / nt);
    t = (int)(at - (long long)u * nt);
  }
  __device__ __forceinline__ void next(const AttnArgs& a, int units) {
    if (++t < nt) return;
    t = 0;
    if (++u < units) return;
    u = 0;
    do ++s;
    while (s < a.kv.n_seqs && (enter(a), nt == 0));
  }
};

// One query vector's share of a warp (its 16 positions of tiles t0 ... t1) once more, in
// plain f32.  The tensor cores get P, and in f32 every operand, in two parts, where
// an infinity becomes NaN (inf * 0, inf - inf) and a finite value next to the end of
// f32's range rounds to infinity.  Either leaves a sum that is not finite, so the fast
// path looks at nothing but its sums at the end of a share.  Here scores of -inf
// have the weight 0, and infinities and NaN of V reach their value whatever the
// weight (as in prefill).  One infinity in 131072 positions (32 / 8 heads x 128, bf16):
// 0.1 -> 0.36 ms; V of NaN throughout 3.0 ms.  out: HD sums in shared memory;
// returns (max, sum).
template <typename T, int HD, int TILE, int UP>
__device__ __noinline__ float2 decode_again(const AttnArgs& a, const T* q, int s, int kvh, Span sp, int t0, int t1, float* out) {
  constexpr int PER = HD / 32;  // values per lane
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float x[PER], o[PER] = {}, m = -INFINITY, l = 0.f;
#pragma unroll
  for (int k = 0; k < PER; ++k) x[k] = to_f(q[lane * PER + k]);
  for (int t = t0; t <= t1; ++t) {
    const int base = t * TILE + warp * 16, n = min(16, sp.n - base);
    if (n <= 0) break;
    long long off = 0;  // lanes i and i + 16: row i
    float score = -INFINITY;
    if ((lane & 15) < n) {
      const int pos = sp.pos(base + (lane & 15));
      off = page_row(a.kv, a.kv.table[s * a.kv.table_stride + (pos >> a.kv.page_shift)], pos) + kvh * a.kv.head_stride;
    }
    for (int i = 0; i < n; ++i) {
      const T* k = reinterpret_cast<const T*>(a.kv.k + __shfl_sync(0xffffffffu, off, i)) + lane * PER;
      float d = 0.f;
#pragma unroll
      for (int j = 0; j < PER; ++j) d = fmaf(x[j], to_f(k[j]), d);
      d = warp_sum(d);
      if ((lane & 15) == i) score = d * a.scale2;
    }
    float top = score;
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    const float mn = fmaxf(m, top), b = mn == -INFINITY ? 0.f : mn, f = fmaxf(exp2f(m - b), TINY);
    const float p = exp2f(score - (b - UP));
    float sum = p;
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    l = l * f + sum;
    m = mn;
    float add[PER] = {};
    for (int i = 0; i < n; ++i) {
      const T* v = reinterpret_cast<const T*>(a.kv.v + __shfl_sync(0xffffffffu, off, i)) + lane * PER;
      const float w = __shfl_sync(0xffffffffu, p, i);
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const float y = to_f(v[j]);
        add[j] = fabsf(y) < INFINITY ? fmaf(w, y, add[j]) : add[j] + y;
      }
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) o[j] = o[j] * f + add[j];
  }
#pragma unroll
  for (int k = 0; k < PER; ++k) out[lane * PER + k] = o[k];
  return make_float2(m, l);
}

template <typename T, int HD, int NT>
__global__ void __launch_bounds__(DecodeCfg<T, HD, NT>::WARPS * 32, Elem<T>::f32 ? 1 : 2)
paged_decode_kernel(const __grid_constant__ AttnArgs a, int hgroups) {
  using C = DecodeCfg<T, HD, NT>;
  using S = Step<T, HD, NT>;
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  extern __shared__ __align__(128) unsigned char smem[];
  float* red = reinterpret_cast<float*>(smem + C::WARPS * C::STAGES * C::STAGE);  // [warp][4][HD + 4]
  float2* ml = reinterpret_cast<float2*>(red + C::WARPS * 4 * (HD + 4));          // [warp][8]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int units = a.n_kv * hgroups;
  T* out = static_cast<T*>(a.out);
  // sequences that see nothing
  for (int s = blockIdx.x; s < a.kv.n_seqs; s += gridDim.x)
    if (seq_tiles<C::TILE>(a, s) == 0)
      for (int i = threadIdx.x; i < a.n_kv * a.group * HD; i += C::WARPS * 32)
        out[s * a.o_row + (i / HD) * a.o_head + i % HD] = from_f<T>(0.f);
  const Line line = line_of<C::TILE>(a, units, gridDim.x);
  // What the join does for this CTA: n parts of unit (s, u), the first of them in this CTA's slot.
  int4* todo = reinterpret_cast<int4*>(a.part + 2ll * gridDim.x * C::SLOT) + blockIdx.x;
  if ((int)blockIdx.x >= line.parts) {
    if (threadIdx.x == 0) *todo = make_int4(0, 0, 0, 0);
    return;
  }
  const long long w0 = line.start(blockIdx.x), w1 = line.start(blockIdx.x + 1);
  LineCursor<C::TILE> cur;
  long long before;
  cur.s = line_seq<C::TILE>(a, units, w0, before);
  cur.enter(a);
  cur.place(w0 - before);
  LineCursor<C::TILE> ld = cur;
  const int n = (int)(w1 - w0);

  const uint32_t ring = smem_u32(smem) + warp * C::STAGES * C::STAGE;
  // The row this lane looks up for the next tile to load (rows lane & 15): its page is
  // read one tile ahead of the copies that need it.
  int row_pos = -1, row_page = 0;
  auto look = [&]() {
    const int i = ld.t * C::TILE + warp * 16 + (lane & 15);
    row_pos = -1;
    if (ld.s < a.kv.n_seqs && i < ld.sp.n) {
      row_pos = ld.sp.pos(i);
      row_page = a.kv.table[ld.s * a.kv.table_stride + (row_pos >> a.kv.page_shift)];
    }
  };
  // Stages go out in order: a tile's K and V, or its K, for which the rows are found, and then its V.
  int out_tile = 0, out_slot = 0;
  bool out_v = false;
  long long off = -1;
  auto copy = [&](uint32_t dst, const char* base, bool v) {
    constexpr int RPI = 32 / S::PIECES;  // rows per round of 32 lanes
#pragma unroll
    for (int r0 = 0; r0 < 16; r0 += RPI) {
      const int r = r0 + lane / S::PIECES, pc = lane % S::PIECES;
      const long long o = __shfl_sync(0xffffffffu, off, r), src = (o < 0 ? 0 : o) + pc * 16;
      if (C::HALVES) {
        cpa16(dst + (v ? S::v_off(r, pc) : S::k_off(r, pc)), base + src, o >= 0);
      } else {
        cpa16(dst + S::k_off(r, pc), a.kv.k + src, o >= 0);
        cpa16(dst + C::ROWS + S::v_off(r, pc), a.kv.v + src, o >= 0);
      }
    }
  };
  auto load = [&]() {
    if (out_tile < n) {
      const uint32_t dst = ring + out_slot * C::STAGE;
      if (!C::HALVES || !out_v) {
        off = row_pos < 0 ? -1 : page_row(a.kv, row_page, row_pos) + (ld.u / hgroups) * a.kv.head_stride;
        ld.next(a, units);
        if (out_tile + 1 < n) look();
      }
      copy(dst, out_v ? a.kv.v : a.kv.k, out_v);
      out_tile += !C::HALVES || out_v;
      out_v = !out_v;
      out_slot = out_slot + 1 == C::STAGES ? 0 : out_slot + 1;
    }
    cpa_commit();
  };
  look();
#pragma unroll 1
  for (int i = 0; i < C::STAGES - 1; ++i) load();
  int slot_now = 0;
  auto arrived = [&]() -> uint32_t {  // the next stage, whole; the one before it makes room for another
    cpa_wait<C::STAGES - 2>();
    __syncwarp();
    load();
    const uint32_t at = ring + slot_now * C::STAGE;
    slot_now = slot_now + 1 == C::STAGES ? 0 : slot_now + 1;
    return at;
  };

  S st;
  auto queries = [&](int s, int u) {  // the query vectors of unit u
    const T* q = static_cast<const T*>(a.q) + s * a.q_row;
    const int h0 = (u % hgroups) * NT * 8, kvh = u / hgroups;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int h = h0 + 8 * nt + g;
      st.load_q(nt, h < a.group ? q + (long long)(kvh * a.group + h) * a.q_head : nullptr, t);
    }
  };
  queries(cur.s, cur.u);
  float m[NT][2], l[NT][2], o[NT][HD / 16][4];
  bool fresh = true, first_part = true, left = false;
  for (int i = 0; i < n; ++i) {
    if (fresh) {
      fresh = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        m[nt][0] = m[nt][1] = -INFINITY;
        l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
        for (int j = 0; j < HD / 16; ++j) o[nt][j][0] = o[nt][j][1] = o[nt][j][2] = o[nt][j][3] = 0.f;
      }
    }
    const int base = cur.t * C::TILE + warp * 16;
    const bool any = base < cur.sp.n;  // (the same for the whole warp)
    float s[NT][4];
    const uint32_t kb = arrived();
    if (any) st.scores(kb, lane, s);
    const uint32_t vb = C::HALVES ? arrived() : kb + C::ROWS;
    if (any) {
      const bool in0 = base + g < cur.sp.n, in1 = base + g + 8 < cur.sp.n;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        s[nt][0] = in0 ? s[nt][0] * a.scale2 : -INFINITY;
        s[nt][1] = in0 ? s[nt][1] * a.scale2 : -INFINITY;
        s[nt][2] = in1 ? s[nt][2] * a.scale2 : -INFINITY;
        s[nt][3] = in1 ? s[nt][3] * a.scale2 : -INFINITY;
      }
      float f[NT][2];
      const bool moved = softmax_step<NT, S::UP>(s, m, l, f);
      st.pv(vb, lane, s, f, moved, o);
    }
    if (cur.t + 1 < cur.nt && i + 1 < n) {
      ++cur.t;
      continue;
    }
    // ---- end of this CTA's share of (sequence, unit): join the warps ----
    fresh = true;
    const bool whole = cur.t + 1 == cur.nt && i >= cur.nt - 1;
    const int h0 = (cur.u % hgroups) * NT * 8, kvh = cur.u / hgroups, seq = cur.s;
    if (cur.t + 1 < cur.nt && i >= cur.t) {  // begins here and goes on in the CTAs behind
      left = true;
      if (threadIdx.x == 0) {
        const long long end = w0 + i - cur.t + cur.nt;
        int parts = 1;
        while ((int)blockIdx.x + parts < line.parts && line.start(blockIdx.x + parts) < end) ++parts;
        *todo = make_int4(seq, cur.u, parts, first_part ? 0 : 1);
      }
    }
    const Span sp = cur.sp;
    const int t1 = cur.t, t0 = max(0, cur.t - i);  // the share's tiles
    cur.next(a, units);
    if (i + 1 < n) queries(cur.s, cur.u);  // on their way while the warps are joined
    float* slot = a.part + (2ll * blockIdx.x + (first_part ? 0 : 1)) * C::SLOT;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], off);
        float zero = 0.f;  // 0 if the sums of vector 2t + c are finite, NaN otherwise
#pragma unroll
        for (int j = 0; j < HD / 16; ++j) zero = fmaf(o[nt][j][c], 0.f, fmaf(o[nt][j][c + 2], 0.f, zero));
        // (16-bit scores are right as they are: a NaN among them is NaN here too)
        const unsigned odd = __ballot_sync(0xffffffffu, zero != 0.f && (S::F || l[nt][c] == l[nt][c]));
#pragma unroll 1
        for (int v = 0; odd && v < 4; ++v) {
          const int h = h0 + 8 * nt + 2 * v + c;
          if (!(odd >> v & 0x11111111u) || h >= a.group) continue;
          float* again = red + warp * 4 * (HD + 4);
          const T* q = static_cast<const T*>(a.q) + seq * a.q_row + (long long)(kvh * a.group + h) * a.q_head;
          const float2 now = decode_again<T, HD, C::TILE, S::UP>(a, q, seq, kvh, sp, t0, t1, again);
          __syncwarp();
          if (t == v) {
            m[nt][c] = now.x;
            l[nt][c] = now.y;
#pragma unroll
            for (int j = 0; j < HD / 16; ++j) {
              o[nt][j][c] = again[S::dim(j, 0, g)];
              o[nt][j][c + 2] = again[S::dim(j, 1, g)];
            }
          }
          __syncwarp();
        }
        if (g == 0) ml[warp * 8 + 2 * t + c] = make_float2(m[nt][c], l[nt][c]);
      }
      __syncthreads();
      float f[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float M = -INFINITY;
        for (int w = 0; w < C::WARPS; ++w) M = fmaxf(M, ml[w * 8 + 2 * t + c].x);
        f[c] = fmaxf(exp2f(m[nt][c] - (M == -INFINITY ? 0.f : M)), TINY);
      }
#pragma unroll
      for (int v0 = 0; v0 < 8; v0 += 4) {  // vectors v0 ... v0 + 3 of the eight
        const int heads = min(4, a.group - h0 - 8 * nt - v0);
        if (heads <= 0) break;
        if (t >> 1 == v0 >> 2) {
          float* mine = red + (warp * 4 + 2 * (t & 1)) * (HD + 4);
#pragma unroll
          for (int j = 0; j < HD / 16; ++j)
#pragma unroll
            for (int hi = 0; hi < 2; ++hi) {
              const int d = S::dim(j, hi, g);
              mine[d] = o[nt][j][2 * hi] * f[0];
              mine[HD + 4 + d] = o[nt][j][2 * hi + 1] * f[1];
            }
        }
        __syncthreads();
        for (int x = threadIdx.x; x < heads * HD; x += C::WARPS * 32) {
          const int h = x / HD, d = x % HD;
          float M = -INFINITY, L = 0.f, acc = 0.f;
          for (int w = 0; w < C::WARPS; ++w) M = fmaxf(M, ml[w * 8 + v0 + h].x);
          const float b = M == -INFINITY ? 0.f : M;
          for (int w = 0; w < C::WARPS; ++w) {
            const float2 v = ml[w * 8 + v0 + h];
            L += v.y * exp2f(v.x - b);
            acc += red[(w * 4 + h) * (HD + 4) + d];
          }
          const int hu = 8 * nt + v0 + h;  // head of the unit
          if (whole) {
            out[seq * a.o_row + (long long)(kvh * a.group + h0 + hu) * a.o_head + d] = from_f<T>(L == 0.f ? 0.f : acc / L);
          } else {
            slot[NT * 16 + hu * HD + d] = acc;
            if (d == 0) {
              slot[hu] = M;
              slot[NT * 8 + hu] = L;
            }
          }
        }
        __syncthreads();  // ml and red are free again
      }
    }
    first_part = false;
  }
  cpa_wait<0>();
  if (threadIdx.x == 0 && !left) *todo = make_int4(0, 0, 0, 0);
}

// Adds the parts of each (sequence, unit) that is cut: CTA (c, h) does what CTA c
// of the decode kernel left to do, for head h of the unit.  Latency bound (0.5 to 2
// MB, 8 to 12 us from cold caches): started early by programmatic launch, a CTA per
// head, so the loads of up to 296 parts are spread over all SMs.
constexpr int JOIN_MAX = 512;  // parts there can be (resident CTAs of a decode call)
template <typename T, int HD, int NT>
__global__ void __launch_bounds__(HD) paged_decode_join_kernel(const __grid_constant__ AttnArgs a, int hgroups) {
  using C = DecodeCfg<T, HD, NT>;
  asm volatile("griddepcontrol.launch_dependents;");
  __shared__ float weight[JOIN_MAX];
  __shared__ float red[2 * HD / 32];
  const int c = blockIdx.x, h = blockIdx.y, d = threadIdx.x, warp = d >> 5, lane = d & 31;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 job = reinterpret_cast<const int4*>(a.part + 2ll * gridDim.x * C::SLOT)[c];
  const int n = job.z, u = job.y;  // parts of the unit (0: nothing to do)
  if (n == 0 || (u % hgroups) * NT * 8 + h >= a.group) return;
  // the first part lies in slot job.w of CTA c, the others are the first ones of the CTAs behind it
  const float* first = a.part + (2ll * c + job.w) * C::SLOT;
  auto slot = [&](int i) { return i ? a.part + 2ll * (c + i) * C::SLOT : first; };
  float M = -INFINITY;
  for (int i = d; i < n; i += HD) {
    const float m = slot(i)[h];
    weight[i] = m;
    M = fmaxf(M, m);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  if (lane == 0) red[warp] = M;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < HD / 32; ++i) M = fmaxf(M, red[i]);
  const float b = M == -INFINITY ? 0.f : M;
  float L = 0.f;
  for (int i = d; i < n; i += HD) {
    const float e = fmaxf(exp2f(weight[i] - b), TINY);
    weight[i] = e;
    L += slot(i)[NT * 8 + h] * e;
  }
  L = warp_sum(L);
  if (lane == 0) red[HD / 32 + warp] = L;
  __syncthreads();
  L = 0.f;
#pragma unroll
  for (int i = 0; i < HD / 32; ++i) L += red[HD / 32 + i];
  float acc = 0.f;
#pragma unroll 8
  for (int i = 0; i < n; ++i) acc += slot(i)[NT * 16 + h * HD + d] * weight[i];
  static_cast<T*>(a.out)[job.x * a.o_row + (long long)((u / hgroups) * a.group + (u % hgroups) * NT * 8 + h) * a.o_head + d] =
      from_f<T>(L == 0.f ? 0.f : acc / L);
}

// ======================= rows of a chunk (prefill) =======================
// Rows [r0, r0 + n) of sequence s; tile `idx` of the line of all sequences' row
// tiles gives (s, first flattened row).  Bad starts set the error word.
struct RowTile {
  int s, r0, n, f0, ctx;
};
__device__ __forceinline__ int chunk_rows(const AttnArgs& a, int s, int& r0) {
  r0 = a.starts[s];
  const int r1 = a.starts[s + 1];
  if (r0 < 0 || r1 < r0 || r1 > a.rows) {
    flag_error(DEV_ERR_BAD_ARG);
    return 0;
  }
  return r1 - r0;
}
__device__ __forceinline__ bool row_tile(const AttnArgs& a, int idx, int tile, RowTile& rt) {
  const int lane = threadIdx.x & 31;
  long long before = 0;
  for (int s0 = 0; s0 < a.kv.n_seqs; s0 += 32) {
    int r0 = 0, n = 0, len = 0;
    if (s0 + lane < a.kv.n_seqs) {
      len = paged_len(a.kv, a.lens, s0 + lane);
      n = chunk_rows(a, s0 + lane, r0);
    }
    const long long tiles = ((long long)n * a.group + tile - 1) / tile;
    long long incl = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, before + incl > idx);
    if (hit) {
      const int l = __ffs(hit) - 1;
      rt.s = s0 + l;
      rt.r0 = __shfl_sync(0xffffffffu, r0, l);
      rt.n = __shfl_sync(0xffffffffu, n, l);
      rt.f0 = (int)(idx - before - __shfl_sync(0xffffffffu, incl - tiles, l)) * tile;
      rt.ctx = __shfl_sync(0xffffffffu, len, l) - rt.n;
      return true;
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
  return false;
}

// ======================= launches =======================
// Programmatic dependent launch: the kernel may start while its predecessor on
// the stream still runs, and waits for it (griddepcontrol.wait) before it reads
// or writes anything.
template <typename K, typename... A>
static cudaError_t launch_dependent(K kern, dim3 grid, dim3 block, size_t smem, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

template <typename T, int HD, int NT>
static cudaError_t launch_decode_t(const AttnArgs& a, int hgroups, int grid, cudaStream_t st) {
  using C = DecodeCfg<T, HD, NT>;
  const int dev = current_device();
  cudaError_t e = ensure_smem_attr<paged_decode_kernel<T, HD, NT>>(dev, C::SMEM);
  if (e) return e;
  // no more CTAs than tiles there can be
  const long long cap = (long long)a.kv.pages_per_seq << a.kv.page_shift;
  const long long vis = a.window && a.window + (long long)a.sinks < cap ? a.window + (long long)a.sinks : cap;
  const long long most = a.kv.n_seqs * (long long)a.n_kv * hgroups * ((vis + C::TILE - 1) / C::TILE);
  if (most < grid) grid = (int)(most > 0 ? most : 1);
  if ((e = launch_dependent(paged_decode_kernel<T, HD, NT>, dim3(grid), dim3(C::WARPS * 32), C::SMEM, st, a, hgroups))) return e;
  if (vis <= C::TILE) return cudaSuccess;  // one tile per unit: nothing is cut
  return launch_dependent(paged_decode_join_kernel<T, HD, NT>, dim3(grid, a.group < 8 * NT ? a.group : 8 * NT), dim3(HD), 0, st, a,
                          hgroups);
}

// Resident CTAs that share a decode call's line, and the workspace they need.
static int decode_grid(int type) {
  const int n = sm_count(current_device()) * (type == F32 ? 1 : 2);
  return n < JOIN_MAX ? n : JOIN_MAX;
}
size_t paged_decode_workspace(int type, int group, int head_dim) {
  const int nt = group > 8 ? 2 : 1;
  return decode_grid(type) * ((size_t)2 * nt * 8 * (head_dim + 2) * sizeof(float) + sizeof(int4));
}

cudaError_t launch_paged_decode(int type, int head_dim, const AttnArgs& a, cudaStream_t st) {
  const int nt = a.group > 8 ? 2 : 1, hgroups = (a.group + 8 * nt - 1) / (8 * nt), grid = decode_grid(type);
#define VTB_DEC(TY, HD)                                                             \
  return nt == 1 ? launch_decode_t<TY, HD, 1>(a, hgroups, grid, st) : launch_decode_t<TY, HD, 2>(a, hgroups, grid, st)
  if (type == F32) {
    if (head_dim == 64) VTB_DEC(float, 64);
    VTB_DEC(float, 128);
  }
  if (type == T_F16) {
    if (head_dim == 64) VTB_DEC(__half, 64);
    VTB_DEC(__half, 128);
  }
  if (head_dim == 64) VTB_DEC(__nv_bfloat16, 64);
  VTB_DEC(__nv_bfloat16, 128);
#undef VTB_DEC
}

}  // namespace vtb
