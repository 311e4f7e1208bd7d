// paged_api.cu -- extern "C" entry points of the paged key-value cache:
// argument checks, then one launch (two for an attention call whose sequences are
// split over CTAs).  Included after api.cu and the paged kernels.

static int paged_elem_bytes(int type) { return type == F32 ? 4 : type == T_F16 || type == T_BF16 ? 2 : 0; }
static bool mul16(long long elems, int es) { return elems * es % 16 == 0; }

// Checks the cache description and turns its strides into bytes.
static int paged_view(const VtbCudaPagedKv* kv, bool need_table, PagedView* out) {
  if (!kv || !kv->k || !kv->v) return set_err(VTB_CUDA_ERR_INVALID_ARG, "null cache");
  const int es = paged_elem_bytes(kv->type);
  if (!es) return set_err(VTB_CUDA_ERR_UNSUPPORTED, "cache type must be F32, F16 or BF16");
  if (kv->head_dim != 64 && kv->head_dim != 128) return set_err(VTB_CUDA_ERR_UNSUPPORTED, "head_dim must be 64 or 128");
  int shift = 0;
  while (shift < 10 && (1 << shift) < kv->page_size) ++shift;
  if (kv->page_size < 1 || (1 << shift) != kv->page_size)
    return set_err(VTB_CUDA_ERR_INVALID_ARG, "page_size must be a power of two in [1, 1024]");
  if (kv->n_kv_heads < 1 || kv->n_kv_heads > 4096 || kv->n_pages < 1 || kv->n_pages > INT_MAX)
    return set_err(VTB_CUDA_ERR_INVALID_ARG, "bad n_kv_heads or n_pages");
  if (!aligned16(kv->k) || !aligned16(kv->v)) return set_err(VTB_CUDA_ERR_INVALID_ARG, "cache is not 16-byte aligned");
  const int64_t st[3] = {kv->page_stride, kv->head_stride, kv->slot_stride};
  for (int64_t s : st)
    if (s < 0 || s > (int64_t(1) << 40) || !mul16(s, es))
      return set_err(VTB_CUDA_ERR_INVALID_ARG, "cache strides must be whole numbers of 16 bytes");
  if (need_table && (!kv->page_table || kv->n_seqs < 1 || kv->pages_per_seq < 1 || kv->table_stride < kv->pages_per_seq ||
                     (int64_t(kv->pages_per_seq) << shift) > (1 << 30)))
    return set_err(VTB_CUDA_ERR_INVALID_ARG, "bad page table");
  *out = PagedView{static_cast<const char*>(kv->k), static_cast<const char*>(kv->v), kv->page_stride * es,
                   kv->head_stride * es, kv->slot_stride * es, kv->page_table, kv->table_stride,
                   (int)kv->n_pages, kv->n_seqs, kv->pages_per_seq, shift};
  return VTB_CUDA_OK;
}

static int paged_rows_ok(const void* p, int64_t n, int64_t row, int64_t head, int es, int64_t hd) {
  if (n == 0) return VTB_CUDA_OK;  // (an empty list may have no address)
  if (!p) return set_err(VTB_CUDA_ERR_INVALID_ARG, "null rows");
  if (!aligned16(p) || !mul16(row, es) || !mul16(head, es) || row < (n > 1 ? hd : 0) || head < hd || row > (int64_t(1) << 40) ||
      head > (int64_t(1) << 40))
    return set_err(VTB_CUDA_ERR_INVALID_ARG, "rows must be 16-byte aligned, with strides of whole 16 bytes and at least head_dim");
  return VTB_CUDA_OK;
}

// One workspace serves both attention calls.
static size_t paged_workspace(int type, int group, int head_dim) {
  const size_t d = paged_decode_workspace(type, group, head_dim);
  const size_t p = type == F32 ? paged_prefill_f32_workspace(head_dim) : paged_prefill_tc_workspace(head_dim);
  return d > p ? d : p;
}

static int paged_attn_args(const VtbCudaPagedKv* kv, const VtbCudaPagedAttn* p, int64_t rows, AttnArgs* a) {
  if (!p) return set_err(VTB_CUDA_ERR_INVALID_ARG, "null attention arguments");
  int rc = paged_view(kv, true, &a->kv);
  if (rc) return rc;
  const int es = paged_elem_bytes(kv->type);
  if ((rc = paged_rows_ok(p->q, rows, p->q_row_stride, p->q_head_stride, es, kv->head_dim))) return rc;
  if ((rc = paged_rows_ok(p->out, rows, p->out_row_stride, p->out_head_stride, es, kv->head_dim))) return rc;
  if (p->n_heads < 1 || p->n_heads % kv->n_kv_heads || p->n_heads / kv->n_kv_heads > 128)
    return set_err(VTB_CUDA_ERR_INVALID_ARG, "n_heads must be a multiple of n_kv_heads, at most 128 times it");
  if (!p->lens) return set_err(VTB_CUDA_ERR_INVALID_ARG, "null lens");
  if (!(p->scale > -INFINITY && p->scale < INFINITY)) return set_err(VTB_CUDA_ERR_INVALID_ARG, "scale must be finite");
  if (p->window < 0 || p->sinks < 0 || (p->sinks && !p->window))
    return set_err(VTB_CUDA_ERR_INVALID_ARG, "window and sinks must not be negative, and sinks need a window");
  a->q = p->q;
  a->out = p->out;
  a->q_row = p->q_row_stride;
  a->q_head = p->q_head_stride;
  a->o_row = p->out_row_stride;
  a->o_head = p->out_head_stride;
  a->lens = p->lens;
  a->starts = nullptr;
  a->rows = kv->n_seqs;
  a->n_kv = kv->n_kv_heads;
  a->group = p->n_heads / kv->n_kv_heads;
  // positions lie below 2^30: a longer window sees the same, and nothing overflows
  a->window = p->window < (1 << 30) ? p->window : 1 << 30;
  a->sinks = p->sinks < (1 << 30) ? p->sinks : 1 << 30;
  a->tile = a->recip = 0;
  a->negate = false;
  a->scale2 = (float)((double)p->scale * 1.4426950408889634);
  if (!p->workspace || !aligned16(p->workspace) || p->workspace_bytes < paged_workspace(kv->type, a->group, kv->head_dim))
    return set_err(VTB_CUDA_ERR_INVALID_ARG, "workspace is missing, misaligned or too small");
  a->part = static_cast<float*>(p->workspace);
  return VTB_CUDA_OK;
}

extern "C" {

size_t vtb_cuda_paged_attn_workspace_bytes(int type, int32_t n_heads, int32_t n_kv_heads, int32_t head_dim) {
  if (!paged_elem_bytes(type) || n_kv_heads < 1 || n_heads < 1 || n_heads % n_kv_heads) return 0;
  return paged_workspace(type, n_heads / n_kv_heads, head_dim);
}

int vtb_cuda_paged_attn_decode(const VtbCudaPagedKv* kv, const VtbCudaPagedAttn* p, void* stream) {
  cudaGetLastError();  // drop a stale error left by an unrelated earlier call
  AttnArgs a;
  int rc = paged_attn_args(kv, p, kv ? kv->n_seqs : 0, &a);
  if (rc) return rc;
  return cuda_status(launch_paged_decode(kv->type, kv->head_dim, a, (cudaStream_t)stream));
}

int vtb_cuda_paged_attn_prefill(const VtbCudaPagedKv* kv, const VtbCudaPagedAttn* p, const int32_t* starts, int64_t n_rows,
                                void* stream) {
  cudaGetLastError();
  AttnArgs a;
  int rc = paged_attn_args(kv, p, n_rows, &a);
  if (rc) return rc;
  if (!starts || n_rows < 0 || n_rows > INT_MAX / a.group)
    return set_err(VTB_CUDA_ERR_INVALID_ARG, "bad starts or n_rows");
  if (n_rows == 0) return VTB_CUDA_OK;
  a.starts = starts;
  a.rows = (int)n_rows;
  cudaStream_t st = (cudaStream_t)stream;
  return cuda_status(kv->type == F32 ? launch_paged_prefill_f32(kv->head_dim, a, st)
                                     : launch_paged_prefill_tc(kv->type, kv->head_dim, a, st));
}

int vtb_cuda_paged_append(const VtbCudaPagedKv* kv, const VtbCudaPagedRows* r, void* stream) {
  cudaGetLastError();
  AppendArgs a;
  int rc = paged_view(kv, true, &a.kv);
  if (rc) return rc;
  if (!r) return set_err(VTB_CUDA_ERR_INVALID_ARG, "null rows");
  if (r->type != F32 && r->type != kv->type)
    return set_err(VTB_CUDA_ERR_UNSUPPORTED, "rows must be F32 or the cache's type");
  if (r->n_rows < 0 || r->n_rows > INT_MAX) return set_err(VTB_CUDA_ERR_INVALID_ARG, "bad n_rows");
  if (r->n_rows == 0) return VTB_CUDA_OK;
  const int es = paged_elem_bytes(r->type);
  if ((rc = paged_rows_ok(r->k, r->n_rows, r->k_row_stride, r->k_head_stride, es, kv->head_dim))) return rc;
  if ((rc = paged_rows_ok(r->v, r->n_rows, r->v_row_stride, r->v_head_stride, es, kv->head_dim))) return rc;
  if (r->q) {
    if ((rc = paged_rows_ok(r->q, r->n_rows, r->q_row_stride, r->q_head_stride, es, kv->head_dim))) return rc;
    if (r->n_heads < 1 || r->n_heads > 65536 || !r->q_out || !aligned16(r->q_out))
      return set_err(VTB_CUDA_ERR_INVALID_ARG, "q needs n_heads and a 16-byte aligned q_out");
  } else if (r->q_out) {
    return set_err(VTB_CUDA_ERR_INVALID_ARG, "q_out without q");
  }
  if (!r->seq || !r->pos) return set_err(VTB_CUDA_ERR_INVALID_ARG, "null seq or pos");
  if (r->rope && (!aligned16(r->rope) || r->n_rope < 1))
    return set_err(VTB_CUDA_ERR_INVALID_ARG, "rope must be 16-byte aligned, with at least one position");
  a.q = r->q; a.k = r->k; a.v = r->v;
  a.q_row = r->q_row_stride; a.q_head = r->q_head_stride;
  a.k_row = r->k_row_stride; a.k_head = r->k_head_stride;
  a.v_row = r->v_row_stride; a.v_head = r->v_head_stride;
  a.q_out = r->q_out;
  a.rope = r->rope;
  a.n_rope = r->n_rope;
  a.seq = r->seq;
  a.pos = r->pos;
  a.rows = r->n_rows;
  a.n_heads = r->n_heads;
  a.n_kv = kv->n_kv_heads;
  a.hd = kv->head_dim;
  return cuda_status(launch_paged_append(r->type, kv->type, a, (cudaStream_t)stream));
}

int vtb_cuda_paged_copy(const VtbCudaPagedKv* kv, int32_t n_layers, int64_t layer_stride, const int32_t* src,
                        const int32_t* dst, int64_t n_moves, int32_t* page_table, const int32_t* page_map, void* stream) {
  cudaGetLastError();
  PagedView v;
  int rc = paged_view(kv, false, &v);
  if (rc) return rc;
  const int es = paged_elem_bytes(kv->type);
  if (n_layers < 1 || layer_stride < 0 || layer_stride > (int64_t(1) << 42) || !mul16(layer_stride, es))
    return set_err(VTB_CUDA_ERR_INVALID_ARG, "bad n_layers or layer_stride");
  if (n_moves < 0 || n_moves > INT_MAX || (n_moves && (!src || !dst)))
    return set_err(VTB_CUDA_ERR_INVALID_ARG, "bad move list");
  if (!page_table != !page_map) return set_err(VTB_CUDA_ERR_INVALID_ARG, "page_table and page_map go together");
  if (page_table && (kv->n_seqs < 0 || kv->pages_per_seq < 0 || kv->table_stride < kv->pages_per_seq))
    return set_err(VTB_CUDA_ERR_INVALID_ARG, "bad page table");
  CopyArgs a = {};
  a.k = static_cast<char*>(kv->k);
  a.v = static_cast<char*>(kv->v);
  a.layer_stride = layer_stride * es;
  a.page_stride = v.page_stride;
  a.head_stride = v.head_stride;
  a.slot_stride = v.slot_stride;
  a.src = src;
  a.dst = dst;
  a.moves = n_moves;
  a.n_layers = n_layers;
  a.n_pages = v.n_pages;
  a.page_shift = v.page_shift;
  a.row_pieces = kv->head_dim * es / 16;
  a.page_pieces = kv->n_kv_heads * kv->page_size * a.row_pieces;
  a.table = page_table;
  a.map = page_map;
  a.table_rows = kv->n_seqs;
  a.table_cols = kv->pages_per_seq;
  a.table_stride = kv->table_stride;
  return cuda_status(launch_paged_copy(a, (cudaStream_t)stream));
}

}  // extern "C"
