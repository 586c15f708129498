// Attention over part of a row's pages (sliding window and sinks, K6 decode
// and K8 prefill) and over pages that rows share (K7).
//
// One kernel serves all three: a block takes one (query token, KV head), its
// warp h the query head 4 g + h.  A warp walks the visible keys 32 at a time,
// one key per lane for the scores, two channels per lane for P.V, and keeps
// the running maximum and sum of a softmax in base 2 in FP32.
#include <cmath>

#include "tvp_params.cuh"

namespace tvp {
namespace {

constexpr int kMaxSpanCtas = 1024;

struct SpanParams {
  const __nv_bfloat16* q;
  const __nv_bfloat16* k_pool;
  const __nv_bfloat16* v_pool;
  __nv_bfloat16* out;
  const int32_t* tables;
  const int32_t* seq_lens;  // decode: row b's query is its last token
  const int32_t* cu_q;      // prefill: query tokens of sequence s, else null
  const int32_t* q_pos0;
  const int32_t* prefix_tables;
  const int32_t* prefix_pages;
  const int32_t* group_rows;
  int groups, prefix_stride;
  long long layer_row_base;
  int num_pages, table_stride, batch, kv_heads;
  int window, sinks;  // window 0: everything
  float scale_log2;
  int32_t* err;
};

__global__ void __launch_bounds__(kGroup * 32) span_attention_kernel(const SpanParams p) {
  const int h = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = blockIdx.y;
  __shared__ float q_s[kGroup][kHeadDim];
  int s, token, pos;
  if (p.cu_q) {
    s = blockIdx.x;
    const int q0 = __ldg(p.cu_q + s), q1 = __ldg(p.cu_q + s + 1);
    if (q0 + (int)blockIdx.z >= q1) return;
    token = q0 + blockIdx.z;
    pos = __ldg(p.q_pos0 + s) + blockIdx.z;
    if (pos < 0 || pos / kPage >= p.table_stride) {
      if (threadIdx.x == 0) record_error(p.err, TVP_DEVERR_BAD_TOKEN);
      return;
    }
  } else {
    s = token = blockIdx.x;
    int L = __ldg(p.seq_lens + s);
    if (L < 0 || L > p.table_stride * kPage) {
      if (threadIdx.x == 0) record_error(p.err, TVP_DEVERR_BAD_LENGTH);
      L = L < 0 ? 0 : p.table_stride * kPage;
    }
    pos = L - 1;
  }
  int shared_pages = 0;
  const int32_t* shared_table = nullptr;
  for (int i = 0, last = 0; i < p.groups; ++i) {
    const int r0 = __ldg(p.group_rows + i), r1 = __ldg(p.group_rows + i + 1);
    if (r0 < last || r1 < r0 || r1 > p.batch) {
      if (threadIdx.x == 0) record_error(p.err, TVP_DEVERR_BAD_PLAN);
      return;
    }
    last = r0;
    if (s >= r0 && s < r1) {
      shared_pages = __ldg(p.prefix_pages + i);
      shared_table = p.prefix_tables + (size_t)i * p.prefix_stride;
      if (shared_pages < 0 || shared_pages > p.prefix_stride) {
        if (threadIdx.x == 0) record_error(p.err, TVP_DEVERR_BAD_LENGTH);
        shared_pages = shared_pages < 0 ? 0 : p.prefix_stride;
      }
    }
  }
  if (pos >= 0 && pos + 1 < shared_pages * kPage) {
    if (threadIdx.x == 0) record_error(p.err, TVP_DEVERR_BAD_LENGTH);
    pos = -1;
  }
  const size_t row = (size_t)token * p.kv_heads * kGroup * kHeadDim + (g * kGroup + h) * kHeadDim;
  q_s[h][lane] = __bfloat162float(p.q[row + lane]);
  q_s[h][lane + 32] = __bfloat162float(p.q[row + lane + 32]);
  __syncwarp();
  const int lo = p.window > 0 && pos + 1 > p.window ? pos + 1 - p.window : 0;
  const int sinks = min(p.sinks, lo);
  const int n = pos < 0 ? 0 : sinks + (pos + 1 - lo);  // visible keys
  float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
  const int width = p.kv_heads * kHeadDim;
  for (int base = 0; base < n; base += 32) {
    const int i = base + lane;
    const int key = i < sinks ? i : lo + (i - sinks);
    long long at = -1;
    if (i < n) {
      const int pg = key / kPage;
      const int phys = pg < shared_pages ? __ldg(shared_table + pg)
                                         : __ldg(p.tables + (size_t)s * p.table_stride + pg);
      if (phys >= 0 && phys < p.num_pages)
        at = (p.layer_row_base + (long long)phys * kPage + key % kPage) * width + g * kHeadDim;
      else
        record_error(p.err, TVP_DEVERR_BAD_PAGE);
    }
    float x = -INFINITY;
    if (at >= 0) {
      float dot = 0.f;
      for (int d = 0; d < kHeadDim; d += 2) {
        const uint32_t kk = __ldg(reinterpret_cast<const uint32_t*>(p.k_pool + at + d));
        dot = fmaf(bf16lo_to_f32(kk), q_s[h][d], dot);
        dot = fmaf(bf16hi_to_f32(kk), q_s[h][d + 1], dot);
      }
      x = dot * p.scale_log2;
    }
    float mx = x;
    for (int k = 16; k > 0; k >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, k));
    const float mn = fmaxf(m, mx);
    if (mn == -INFINITY) continue;
    const float keep = m == -INFINITY ? 0.f : exp2f(m - mn);
    const float pr = at >= 0 ? exp2f(x - mn) : 0.f;
    m = mn;
    l = l * keep + pr;
    o0 *= keep;
    o1 *= keep;
    for (int j = 0; j < 32; ++j) {
      const long long aj = __shfl_sync(0xffffffffu, at, j);
      const float pj = __shfl_sync(0xffffffffu, pr, j);
      if (aj < 0) continue;
      const uint32_t vv = __ldg(reinterpret_cast<const uint32_t*>(p.v_pool + aj + 2 * lane));
      o0 = fmaf(pj, bf16lo_to_f32(vv), o0);
      o1 = fmaf(pj, bf16hi_to_f32(vv), o1);
    }
  }
  for (int k = 16; k > 0; k >>= 1) l += __shfl_xor_sync(0xffffffffu, l, k);
  const float inv = l > 0.f ? 1.f / l : 0.f;
  *reinterpret_cast<uint32_t*>(p.out + row + 2 * lane) = pack_bf16x2(o0 * inv, o1 * inv);
}

inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

int resolve_span_ctas(int num_ctas, int* out) {
  if (num_ctas < 0 || num_ctas > kMaxSpanCtas) return TVP_ERR_INVALID_ARGUMENT;
  if (num_ctas > 0) {
    *out = num_ctas;
    return TVP_OK;
  }
  return tvp_device_sm_count(out);
}

bool span_heads_supported(int kv_heads) {
  return kv_heads == 1 || kv_heads == 2 || kv_heads == 4 || kv_heads == kMaxKvHeads;
}

// counters[1024][8] | split-K partials[2 num_ctas][kv_heads] | prefix pieces
size_t span_workspace(int batch, int groups, int kv_heads, int num_ctas) {
  size_t n = (size_t)kMaxSpanCtas * kMaxKvHeads * 4;
  n += (size_t)num_ctas * 2 * kv_heads * kPartialFloats * 4;
  if (groups > 0) {
    const size_t streams = (size_t)kv_heads * (batch / 32 + groups);
    const size_t pieces = streams > (size_t)2 * num_ctas ? streams : (size_t)2 * num_ctas;
    n += pieces * (128 * (kHeadDim + 2)) * 4;
  }
  return (n + 255) / 256 * 256;
}

int fill_span(const tvp_bf16* q, const tvp_bf16* k_pool, const tvp_bf16* v_pool, int num_pages,
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
  return TVP_OK;
}

int launched() { return cudaGetLastError() == cudaSuccess ? TVP_OK : TVP_ERR_RUNTIME; }

}  // namespace
}  // namespace tvp

using namespace tvp;

extern "C" {

size_t tvp_span_workspace_bytes(int batch, int groups, int kv_heads, int num_ctas) {
  if (batch <= 0 || groups < 0 || !span_heads_supported(kv_heads)) return 0;
  int ctas = 0;
  if (resolve_span_ctas(num_ctas, &ctas) != TVP_OK) return 0;
  return span_workspace(batch, groups, kv_heads, ctas);
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
  int ctas = 0;
  if ((rc = resolve_span_ctas(num_ctas, &ctas)) != TVP_OK) return rc;
  if (!d_workspace || !aligned(d_workspace, 256) || (workspace_bytes & 3u) ||
      workspace_bytes < span_workspace(batch, 0, kv_heads, ctas))
    return TVP_ERR_WORKSPACE;
  SpanParams p;
  fill_span(q, k_pool, v_pool, num_pages, layer, kv_heads, d_block_tables, table_stride, batch,
            scale, out, d_error, &p);
  p.seq_lens = d_seq_lens;
  p.window = window;
  p.sinks = sinks;
  span_attention_kernel<<<dim3(batch, kv_heads), kGroup * 32, 0, static_cast<cudaStream_t>(stream)>>>(p);
  return launched();
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
  int ctas = 0;
  if ((rc = resolve_span_ctas(num_ctas, &ctas)) != TVP_OK) return rc;
  if (!d_workspace || !aligned(d_workspace, 256) || (workspace_bytes & 3u) ||
      workspace_bytes < span_workspace(batch, groups, kv_heads, ctas))
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
  span_attention_kernel<<<dim3(batch, kv_heads), kGroup * 32, 0, static_cast<cudaStream_t>(stream)>>>(p);
  return launched();
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
  span_attention_kernel<<<dim3(num_seqs, kv_heads, max_q_len), kGroup * 32, 0,
                          static_cast<cudaStream_t>(stream)>>>(p);
  return launched();
}

}  // extern "C"
