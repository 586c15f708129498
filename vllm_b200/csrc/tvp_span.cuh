// Attention over part of a row's pages and over pages that rows share: the
// parameter block of its kernels, a row's span of pages, and the split of
// shared prefixes into pieces.
#pragma once

#include "tvp_params.cuh"

namespace tvp {

constexpr int kMaxSpanCtas = 1024;
constexpr int kTileRows = 32;   // batch rows (or query tokens) of one MMA tile
constexpr int kChunkPages = 4;  // pages per key chunk of a tile
// Prefix groups up to which each CTA works the pieces out by itself; a plan saves
// that and costs a launch.  By itself / planned, us, groups of two rows behind 128
// tokens: of 8 heads 150 52 / 52, 192 67 / 65, 1000 763 / 275; of one head 150 20 / 24,
// 192 23 / 28, 1000 122 / 71.
constexpr int kWarpGroups = 192;
// One piece of a shared prefix: per row of the tile an (m, l, O) partial.
constexpr size_t kPieceFloats = (size_t)kTileRows * kPartialFloats;

struct SpanParams {
  const __nv_bfloat16* q;
  const __nv_bfloat16* k_pool;
  const __nv_bfloat16* v_pool;
  __nv_bfloat16* out;
  const int32_t* tables;
  const int32_t* seq_lens;  // decode: row b's query is its last token
  const int32_t* cu_q;      // prefill: query tokens of sequence s
  const int32_t* q_pos0;
  const int32_t* prefix_tables;
  const int32_t* prefix_pages;
  const int32_t* group_rows;
  int groups, prefix_stride;
  long long layer_row_base;
  int num_pages, table_stride, batch, kv_heads;
  int window, sinks;
  float scale_log2;
  int32_t* err;
  // workspace
  int32_t* counters;   // [kMaxSpanCtas][8]: arrivals of the row that starts in a range and leaves it
  float* partials;     // split-K partials: [2 ctas][kv_heads], or, of rows with prefixes,
                       // [row + range][kv_heads]
  // rows with prefixes
  int2* row_ranges;    // [batch]: first and last range of a row's own pages
  int2* group_pieces;  // [groups + 1]: first piece, pieces per (tile, KV head); with a plan the
                       // last entry says whether the group rows are in order
  float* pieces;       // [piece][row of the tile] partials of the shared prefixes
  int piece_target;    // pieces to aim at
};

// A row's visible pages, laid end to end: `head` pages from the row's start,
// then those from page head + skip on; a token t of them is visible when
// t < len and (t < sinks or t >= lo).
struct RowSpan {
  int pages, head, skip, len, sinks, lo;
  __device__ __forceinline__ int logical(int v) const { return v < head ? v : v + skip; }
  // Visible tokens of logical page j, bit i for token 16 j + i.
  __device__ __forceinline__ uint32_t keep(int j) const {
    const int t0 = j * kPage;
    return below(len - t0) & (below(sinks - t0) | ~below(lo - t0)) & 0xffffu;
  }
  __device__ __forceinline__ static uint32_t below(int n) {
    return n <= 0 ? 0u : n >= kPage ? 0xffffu : (1u << n) - 1u;
  }
};

// Pages of a window and sinks for a context of `len` tokens whose first query
// sees the tokens from `first_lo` on (decode: len - window).
__device__ __forceinline__ RowSpan window_span(int len, long long first_lo, int sinks) {
  RowSpan r;
  r.len = len;
  r.lo = first_lo > 0 ? (int)first_lo : 0;
  r.sinks = min(sinks, r.lo);
  const int all = (len + kPage - 1) / kPage;
  r.head = (r.sinks + kPage - 1) / kPage;
  r.skip = max(0, r.lo / kPage - r.head);
  r.pages = all - r.skip;
  return r;
}

// Group of row s: the last one that starts at or before it, if it holds it.
__device__ __forceinline__ int group_of(const SpanParams& p, int s) {
  int lo = 0, hi = p.groups;  // group_rows[lo - 1] <= s < group_rows[hi]
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(p.group_rows + mid) <= s)
      lo = mid + 1;
    else
      hi = mid;
  }
  return lo > 0 && s < __ldg(p.group_rows + lo) ? lo - 1 : -1;
}

__device__ __forceinline__ int shared_pages(const SpanParams& p, int g, bool report) {
  const int n = __ldg(p.prefix_pages + g);
  if (n >= 0 && n <= p.prefix_stride) return n;
  if (report) record_error(p.err, TVP_DEVERR_BAD_LENGTH);
  return n < 0 ? 0 : p.prefix_stride;
}

// Pages of row s that the decode kernel streams.  len 0: the row's output is
// zeros (an empty row, or one shorter than its prefix).
template <bool SHARED>
__device__ __forceinline__ RowSpan decode_span(const SpanParams& p, int s, bool report) {
  int L = __ldg(p.seq_lens + s);
  if (L < 0 || L > p.table_stride * kPage) {
    if (report) record_error(p.err, TVP_DEVERR_BAD_LENGTH);
    L = L < 0 ? 0 : p.table_stride * kPage;
  }
  if (!SHARED) return window_span(L, (long long)L - p.window, p.sinks);
  RowSpan r = window_span(L, 0, 0);
  const int g = group_of(p, s);
  if (g >= 0) {
    const int shared = shared_pages(p, g, false);
    if (L < shared * kPage) {
      if (report && L > 0) record_error(p.err, TVP_DEVERR_BAD_LENGTH);
      r.len = r.pages = 0;
    } else {
      r.skip = shared;
      r.pages -= shared;
    }
  }
  return r;
}

// True when every thread's share of the group rows is in order; all threads of
// the block call it.
__device__ __forceinline__ bool groups_in_order(const SpanParams& p) {
  bool bad = false;
  for (int i = threadIdx.x; i < p.groups; i += blockDim.x) {
    const int a = __ldg(p.group_rows + i), b = __ldg(p.group_rows + i + 1);
    bad |= a < 0 || b < a || b > p.batch;
  }
  return !__syncthreads_or(bad);
}

// The same, read from the plan where there is one.
__device__ __forceinline__ bool groups_usable(const SpanParams& p) {
  return p.groups <= kWarpGroups ? groups_in_order(p) : __ldg(&p.group_pieces[p.groups].x) != 0;
}

cudaError_t launch_prefix_plan(const SpanParams& p, cudaStream_t stream);
cudaError_t launch_span_decode(const SpanParams& p, bool shared, long long pool_rows, int num_ctas,
                               cudaStream_t stream);
cudaError_t launch_prefix_tiles(const SpanParams& p, long long pool_rows, int max_pieces,
                                cudaStream_t stream);
cudaError_t launch_prefix_merge(const SpanParams& p, cudaStream_t stream);
cudaError_t launch_window_tiles(const SpanParams& p, long long pool_rows, int max_q_len,
                                int num_seqs, cudaStream_t stream);

}  // namespace tvp
