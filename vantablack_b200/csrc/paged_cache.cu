// paged_cache.cu -- writing and moving the pages of the key-value cache:
// append (RoPE and the cache write of new rows, forward.zig:258-269 and
// math.zig:88-104 on pages), and page copies through all layers with the page
// tables rewritten after a compaction.
#include "paged.cuh"

namespace vtb {

struct AppendArgs {
  PagedView kv;
  const void* q;
  const void* k;
  const void* v;
  long long q_row, q_head, k_row, k_head, v_row, v_head;  // elements
  void* q_out;                                            // [rows][n_heads][hd] in the cache's type
  const float* rope;  // [n_rope][hd]: (cos, sin) of each pair; null: no rotation
  const int32_t* seq;
  const int32_t* pos;
  long long rows, n_rope;
  int n_heads, n_kv, hd;
};

// 16 bytes of the cache's type per thread: 4 f32 or 8 16-bit values of one head.
template <typename X, typename T, int N>
__device__ __forceinline__ void load_vec(const X* p, float (&x)[N]) {
  constexpr int PER = 16 / sizeof(X) < N ? 16 / sizeof(X) : N;  // values per load
#pragma unroll
  for (int i = 0; i < N; i += PER) {
    if constexpr (sizeof(X) == 4) {
      const float4 v = *reinterpret_cast<const float4*>(p + i);
      x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w;
    } else {
      const uint4 v = *reinterpret_cast<const uint4*>(p + i);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = unpack2<X>(w[j]);
        x[i + 2 * j] = f.x;
        x[i + 2 * j + 1] = f.y;
      }
    }
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_vec(T* p, const float (&x)[N]) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  } else {
    uint4 v;
    v.x = pack2<T>(x[0], x[1]); v.y = pack2<T>(x[2], x[3]);
    v.z = pack2<T>(x[4], x[5]); v.w = pack2<T>(x[6], x[7]);
    *reinterpret_cast<uint4*>(p) = v;
  }
}

// HBM bound (each value read and written once): 8191 rows of 48 heads x 128, f32 to
// bf16, 302 MB in 55 us, 5.5 TB/s; 32 rows 2.3 us, launch latency.  CTA (row, part) has 256 vectors of
// a row, one per thread, so nothing is divided; its threads read the row's page
// through the same cache lines.  The rotation is the forward loop's: products and
// their difference rounded separately in f32, then one rounding to the cache's
// type.
template <typename X, typename T>
__global__ void __launch_bounds__(256) paged_append_kernel(const __grid_constant__ AppendArgs a) {
  constexpr int N = 16 / sizeof(T);
  const int shift = a.hd * (int)sizeof(T) == 512 ? 5 : a.hd * (int)sizeof(T) == 256 ? 4 : 3;  // log2 of vectors per head
  const int nq = a.q ? a.n_heads : 0, i = blockIdx.y * 256 + threadIdx.x, head = i >> shift, d = (i & ((1 << shift) - 1)) * N;
  if (head >= nq + 2 * a.n_kv) return;
  const long long row = blockIdx.x;
  const bool is_q = head < nq, is_v = head >= nq + a.n_kv;
  const X* src = is_q   ? static_cast<const X*>(a.q) + row * a.q_row + head * a.q_head
                 : is_v ? static_cast<const X*>(a.v) + row * a.v_row + (head - nq - a.n_kv) * a.v_head
                        : static_cast<const X*>(a.k) + row * a.k_row + (head - nq) * a.k_head;
  float x[N];
  load_vec<X, T>(src + d, x);
  const int pos = a.pos[row], seq = a.seq[row];
  if (pos < 0 || seq < 0) return;  // a padding row
  if (seq >= a.kv.n_seqs || pos >= (long long)a.kv.pages_per_seq << a.kv.page_shift || (a.rope && pos >= a.n_rope)) {
    flag_error(DEV_ERR_BAD_ARG);
    return;
  }
  T* dst;
  if (is_q) {
    dst = static_cast<T*>(a.q_out) + (row * a.n_heads + head) * a.hd;
  } else {
    const int page = a.kv.table[seq * a.kv.table_stride + (pos >> a.kv.page_shift)];
    if ((unsigned)page >= (unsigned)a.kv.n_pages) {
      flag_error(DEV_ERR_BAD_ARG);
      return;
    }
    dst = reinterpret_cast<T*>(const_cast<char*>(is_v ? a.kv.v : a.kv.k) + page_row(a.kv, page, pos) +
                               (is_v ? head - nq - a.n_kv : head - nq) * a.kv.head_stride);
  }
  if (a.rope && !is_v) {
    float cs[N];
    load_vec<float, float>(a.rope + (long long)pos * a.hd + d, cs);
#pragma unroll
    for (int k = 0; k < N; k += 2) {
      const float x0 = x[k], x1 = x[k + 1], c = cs[k], s = cs[k + 1];
      x[k] = __fsub_rn(__fmul_rn(x0, c), __fmul_rn(x1, s));
      x[k + 1] = __fadd_rn(__fmul_rn(x0, s), __fmul_rn(x1, c));
    }
  }
  store_vec(dst + d, x);
}

cudaError_t launch_paged_append(int in_type, int type, const AppendArgs& a, cudaStream_t st) {
  const int n = type == F32 ? 4 : 8;
  const dim3 grid((unsigned)a.rows, (((a.q ? a.n_heads : 0) + 2 * a.n_kv) * (a.hd / n) + 255) / 256);  // y <= 9216: heads are checked
#define VTB_APP(X, T) paged_append_kernel<X, T><<<grid, 256, 0, st>>>(a)
  if (type == F32) VTB_APP(float, float);
  else if (type == T_F16 && in_type == F32) VTB_APP(float, __half);
  else if (type == T_F16) VTB_APP(__half, __half);
  else if (in_type == F32) VTB_APP(float, __nv_bfloat16);
  else VTB_APP(__nv_bfloat16, __nv_bfloat16);
#undef VTB_APP
  return cudaGetLastError();
}

struct CopyArgs {
  char* k;
  char* v;
  long long layer_stride, page_stride, head_stride, slot_stride;  // bytes
  const int32_t* src;
  const int32_t* dst;
  long long moves;
  int n_layers, n_pages, page_shift, row_pieces, page_pieces;  // 16-byte pieces per (head, slot) row and per page
  int chunks;                                                  // CTAs per page
  int32_t* table;
  const int32_t* map;
  long long table_rows, table_cols, table_stride, copy_blocks;
};

// HBM bound: every piece is read and written once, eight 16-byte loads in
// flight per thread: 83 pages of 32 layers (1.39 GB moved) 217 us, 6.4 TB/s; 3 pages
// of 22 layers 3.0 us, latency.  CTAs [0, copy_blocks) copy one chunk of one page of K or V
// in one layer; the CTAs behind them rewrite the page tables.
constexpr int CP_THREADS = 256, CP_DEPTH = 8;
__global__ void __launch_bounds__(CP_THREADS) paged_copy_kernel(const __grid_constant__ CopyArgs a) {
  if (blockIdx.x >= a.copy_blocks) {
    const long long n = a.table_rows * a.table_cols, step = (gridDim.x - a.copy_blocks) * (long long)CP_THREADS;
    for (long long i = (blockIdx.x - a.copy_blocks) * (long long)CP_THREADS + threadIdx.x; i < n; i += step) {
      int32_t* e = a.table + i / a.table_cols * a.table_stride + i % a.table_cols;
      const int page = *e;
      if (page < 0) continue;  // no page
      if (page >= a.n_pages) flag_error(DEV_ERR_BAD_ARG);
      else *e = a.map[page];
    }
    return;
  }
  long long b = blockIdx.x;
  const int chunk = (int)(b % a.chunks);
  b /= a.chunks;
  const int which = (int)(b & 1);
  b >>= 1;
  const int layer = (int)(b % a.n_layers);
  const long long mv = b / a.n_layers;
  const int from = a.src[mv], to = a.dst[mv];
  if ((unsigned)from >= (unsigned)a.n_pages || (unsigned)to >= (unsigned)a.n_pages) {
    if (threadIdx.x == 0) flag_error(DEV_ERR_BAD_ARG);
    return;
  }
  char* base = (which ? a.v : a.k) + layer * a.layer_stride;
  const char* s = base + from * a.page_stride;
  char* d = base + to * a.page_stride;
  const int p0 = chunk * CP_THREADS * CP_DEPTH + threadIdx.x, slots = 1 << a.page_shift;
  uint4 x[CP_DEPTH];
  long long off[CP_DEPTH];
#pragma unroll
  for (int i = 0; i < CP_DEPTH; ++i) {
    const int p = p0 + i * CP_THREADS;
    off[i] = -1;
    if (p < a.page_pieces) {
      const int row = p / a.row_pieces;
      off[i] = (row >> a.page_shift) * a.head_stride + (row & (slots - 1)) * a.slot_stride + (p - row * a.row_pieces) * 16;
      x[i] = __ldcs(reinterpret_cast<const uint4*>(s + off[i]));
    }
  }
#pragma unroll
  for (int i = 0; i < CP_DEPTH; ++i)
    if (off[i] >= 0) __stcs(reinterpret_cast<uint4*>(d + off[i]), x[i]);
}

cudaError_t launch_paged_copy(CopyArgs a, cudaStream_t st) {
  a.chunks = (a.page_pieces + CP_THREADS * CP_DEPTH - 1) / (CP_THREADS * CP_DEPTH);
  if ((double)a.moves * a.n_layers * 2 * a.chunks > 2147483647.) return cudaErrorInvalidValue;  // (before it overflows)
  a.copy_blocks = a.moves * a.n_layers * 2 * a.chunks;
  long long extra = a.table ? (a.table_rows * a.table_cols + CP_THREADS - 1) / CP_THREADS : 0;
  if (extra > sm_count(current_device())) extra = sm_count(current_device());
  if (a.copy_blocks + extra == 0) return cudaSuccess;
  if (a.copy_blocks + extra > 0x7fffffffll) return cudaErrorInvalidValue;
  paged_copy_kernel<<<(unsigned)(a.copy_blocks + extra), CP_THREADS, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace vtb
