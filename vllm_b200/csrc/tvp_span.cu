// Entry points of the attention over part of a row's pages (sliding window and
// sinks: K6 decode, K8 prefill) and over pages that rows share (K7): argument
// checks on the host, workspace layout, launches.
#include <climits>
#include <cmath>

#include "tvp_span.cuh"

namespace tvp {
namespace {

inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

int resolve_span_ctas(int num_ctas, int* out) {
  if (num_ctas < 0 || num_ctas > kMaxSpanCtas) return TVP_ERR_INVALID_ARGUMENT;
  if (num_ctas > 0) {
    *out = num_ctas;
    return TVP_OK;
  }
  return tvp_device_sm_count(out);
}

constexpr int kMaxStride = INT_MAX / kPage;  // token positions are 32-bit

// The kernels add up the pages that the rows see in 32 bits.
bool pages_countable(int batch, long long pages_per_row) {
  return batch * pages_per_row <= INT_MAX;
}

bool span_heads_supported(int kv_heads) {
  return kv_heads == 1 || kv_heads == 2 || kv_heads == 4 || kv_heads == kMaxKvHeads;
}

struct SpanWorkspace {
  size_t row_ranges, group_pieces, partials, pieces, total;
  int max_pieces;
};

// counters[1024][8] | row_ranges[batch] | group_pieces[groups + 1] | partials | pieces.
// The counters' place and size are the same for every call.  Pieces: one
// per CTA, or per tile of 32 rows and KV head where those are more.
SpanWorkspace span_workspace(int batch, int groups, int kv_heads, int num_ctas) {
  auto align = [](size_t x) { return (x + 255) / 256 * 256; };
  SpanWorkspace w = {};
  w.row_ranges = (size_t)kMaxSpanCtas * kMaxKvHeads * 4;
  w.group_pieces = w.row_ranges + (groups > 0 ? align((size_t)batch * sizeof(int2)) : 0);
  w.partials = align(w.group_pieces + (groups > 0 ? (size_t)groups + 1 : 0) * sizeof(int2));
  const size_t slots = groups > 0 ? (size_t)batch + num_ctas : (size_t)2 * num_ctas;
  w.pieces = align(w.partials + slots * kv_heads * kPartialFloats * 4);
  if (groups > 0) {
    const int streams = kv_heads * (batch / kTileRows + groups);
    w.max_pieces = streams > num_ctas ? streams : num_ctas;
  }
  w.total = align(w.pieces + (size_t)w.max_pieces * kPieceFloats * 4);
  return w;
}

void fill_span(const tvp_bf16* q, const tvp_bf16* k_pool, const tvp_bf16* v_pool, int num_pages,
              int layer, int kv_heads, const int32_t* tables, int table_stride, int batch,
              float scale, tvp_bf16* out, int32_t* d_error, SpanParams* p) {
  *p = SpanParams{};
  p->q = reinterpret_cast<const __nv_bfloat16*>(q);
  p->k_pool = reinterpret_cast<const __nv_bfloat16*>(k_pool);
  p->v_pool = reinterpret_cast<const __nv_bfloat16*>(v_pool);
  p->out = reinterpret_cast<__nv_bfloat16*>(out);
  p->tables = tables;
  p->layer_row_base = (long long)layer * num_pages * kPage;
  p->num_pages = num_pages;
  p->table_stride = table_stride;
  p->batch = batch;
  p->kv_heads = kv_heads;
  p->scale_log2 = scale * 1.4426950408889634f;
  p->err = d_error;
}

void fill_workspace(void* d_workspace, const SpanWorkspace& w, int num_ctas, SpanParams* p) {
  char* base = static_cast<char*>(d_workspace);
  p->counters = reinterpret_cast<int32_t*>(base);
  p->row_ranges = reinterpret_cast<int2*>(base + w.row_ranges);
  p->group_pieces = reinterpret_cast<int2*>(base + w.group_pieces);
  p->partials = reinterpret_cast<float*>(base + w.partials);
  p->pieces = reinterpret_cast<float*>(base + w.pieces);
  p->piece_target = num_ctas;
}

int map_cuda(cudaError_t e) { return e == cudaSuccess ? TVP_OK : TVP_ERR_RUNTIME; }

}  // namespace
}  // namespace tvp

using namespace tvp;

extern "C" {

size_t tvp_span_workspace_bytes(int batch, int groups, int kv_heads, int num_ctas) {
  if (batch <= 0 || groups < 0 || !span_heads_supported(kv_heads)) return 0;
  int ctas = 0;
  if (resolve_span_ctas(num_ctas, &ctas) != TVP_OK) return 0;
  return span_workspace(batch, groups, kv_heads, ctas).total;
}

int tvp_paged_window_decode_attention(const tvp_bf16* q, const tvp_bf16* k_pool,
                                      const tvp_bf16* v_pool, int num_pages, int num_layers,
                                      int layer, int kv_heads, int q_heads,
                                      const int32_t* d_block_tables, int table_stride,
                                      const int32_t* d_seq_lens, int batch, int window, int sinks,
                                      float scale, int num_ctas, void* d_workspace,
                                      size_t workspace_bytes, tvp_bf16* out, int32_t* d_error,
                                      tvp_stream_t stream) {
  int rc = check_decode_args(q, k_pool, v_pool, out, num_pages, num_layers, layer, kv_heads,
                             q_heads, d_block_tables, table_stride, d_seq_lens, batch, scale,
                             TVP_MODE_FAST, num_ctas);
  if (rc != TVP_OK) return rc;
  if (window < 1 || sinks < 0) return TVP_ERR_INVALID_ARGUMENT;
  if (table_stride > kMaxStride) return TVP_ERR_UNSUPPORTED;
  // (a window that starts inside a page sees one page more)
  const long long seen = ((long long)window + kPage - 1) / kPage + ((long long)sinks + kPage - 1) / kPage + 1;
  if (!pages_countable(batch, seen < table_stride ? seen : table_stride)) return TVP_ERR_UNSUPPORTED;
  int ctas = 0;
  if ((rc = resolve_span_ctas(num_ctas, &ctas)) != TVP_OK) return rc;
  const SpanWorkspace w = span_workspace(batch, 0, kv_heads, ctas);
  if (!d_workspace || !aligned(d_workspace, 256) || workspace_bytes < w.total)
    return TVP_ERR_WORKSPACE;
  SpanParams p;
  fill_span(q, k_pool, v_pool, num_pages, layer, kv_heads, d_block_tables, table_stride, batch,
            scale, out, d_error, &p);
  p.seq_lens = d_seq_lens;
  p.window = window;
  p.sinks = sinks;
  fill_workspace(d_workspace, w, ctas, &p);
  return map_cuda(launch_span_decode(p, false, (long long)num_layers * num_pages * kPage, ctas,
                                     static_cast<cudaStream_t>(stream)));
}

int tvp_paged_shared_prefix_decode_attention(
    const tvp_bf16* q, const tvp_bf16* k_pool, const tvp_bf16* v_pool, int num_pages,
    int num_layers, int layer, int kv_heads, int q_heads, const int32_t* d_block_tables,
    int table_stride, const int32_t* d_seq_lens, int batch, const int32_t* d_prefix_tables,
    int prefix_stride, const int32_t* d_prefix_pages, const int32_t* d_group_rows, int groups,
    float scale, int num_ctas, void* d_workspace, size_t workspace_bytes, tvp_bf16* out,
    int32_t* d_error, tvp_stream_t stream) {
  int rc = check_decode_args(q, k_pool, v_pool, out, num_pages, num_layers, layer, kv_heads,
                             q_heads, d_block_tables, table_stride, d_seq_lens, batch, scale,
                             TVP_MODE_FAST, num_ctas);
  if (rc != TVP_OK) return rc;
  if (groups < 0 || groups > 65535 || prefix_stride < 0 || !aligned(q, 16) ||
      (groups > 0 && (!d_prefix_tables || !d_prefix_pages || !d_group_rows || prefix_stride < 1)))
    return TVP_ERR_INVALID_ARGUMENT;
  if (table_stride > kMaxStride || prefix_stride > kMaxStride || !pages_countable(batch, table_stride))
    return TVP_ERR_UNSUPPORTED;
  int ctas = 0;
  if ((rc = resolve_span_ctas(num_ctas, &ctas)) != TVP_OK) return rc;
  const SpanWorkspace w = span_workspace(batch, groups, kv_heads, ctas);
  if (!d_workspace || !aligned(d_workspace, 256) || workspace_bytes < w.total)
    return TVP_ERR_WORKSPACE;
  SpanParams p;
  fill_span(q, k_pool, v_pool, num_pages, layer, kv_heads, d_block_tables, table_stride, batch,
            scale, out, d_error, &p);
  p.seq_lens = d_seq_lens;
  p.prefix_tables = d_prefix_tables;
  p.prefix_pages = d_prefix_pages;
  p.group_rows = d_group_rows;
  p.groups = groups;
  p.prefix_stride = prefix_stride;
  p.window = INT_MAX;  // without groups: everything
  fill_workspace(d_workspace, w, ctas, &p);
  const long long rows = (long long)num_layers * num_pages * kPage;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (groups > kWarpGroups && (rc = map_cuda(launch_prefix_plan(p, st))) != TVP_OK) return rc;
  if ((rc = map_cuda(launch_span_decode(p, groups > 0, rows, ctas, st))) != TVP_OK || groups == 0)
    return rc;
  if ((rc = map_cuda(launch_prefix_tiles(p, rows, w.max_pieces, st))) != TVP_OK) return rc;
  return map_cuda(launch_prefix_merge(p, st));
}

int tvp_paged_window_prefill_attention(const tvp_bf16* q, const tvp_bf16* k_pool,
                                       const tvp_bf16* v_pool, int num_pages, int num_layers,
                                       int layer, int kv_heads, int q_heads,
                                       const int32_t* d_block_tables, int table_stride,
                                       const int32_t* d_cu_q, const int32_t* d_q_pos0,
                                       int num_seqs, int max_q_len, int window, int sinks,
                                       float scale, tvp_bf16* out, int32_t* d_error,
                                       tvp_stream_t stream) {
  if (!q || !k_pool || !v_pool || !out || !d_block_tables || !d_cu_q || !d_q_pos0 ||
      num_pages <= 0 || num_layers <= 0 || layer < 0 || layer >= num_layers || table_stride <= 0 ||
      num_seqs <= 0 || num_seqs > 65535 || max_q_len < 0 || window < 1 || sinks < 0 ||
      !std::isfinite(scale))
    return TVP_ERR_INVALID_ARGUMENT;
  if (table_stride > kMaxStride) return TVP_ERR_UNSUPPORTED;
  if (max_q_len > 65535 * 32) return TVP_ERR_UNSUPPORTED;  // one grid row per 32-token tile
  if (!span_heads_supported(kv_heads) || q_heads != kv_heads * kGroup) return TVP_ERR_UNSUPPORTED;
  if ((long long)num_layers * num_pages * kPage > 0x7fffffffLL) return TVP_ERR_UNSUPPORTED;
  if (!aligned(k_pool, 16) || !aligned(v_pool, 16) || !aligned(q, 16) || !aligned(out, 16))
    return TVP_ERR_INVALID_ARGUMENT;
  if (max_q_len == 0) return TVP_OK;
  SpanParams p;
  fill_span(q, k_pool, v_pool, num_pages, layer, kv_heads, d_block_tables, table_stride, num_seqs,
            scale, out, d_error, &p);
  p.cu_q = d_cu_q;
  p.q_pos0 = d_q_pos0;
  p.window = window;
  p.sinks = sinks;
  return map_cuda(launch_window_tiles(p, (long long)num_layers * num_pages * kPage, max_q_len,
                                      num_seqs, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
