// K9 — one token per row of logits from given random numbers.
//
// One block per row.  Weights w_i = exp((x_i - max) / T) are taken in FP64 and
// held as integers of 2^-44 of the largest (64-bit sums are then exact, in any
// order).  The filters cut the row at a place in its falling order (value,
// then index): the cut is found digit by digit, 8 bits of the order-preserving
// image of the logit at a time, from a histogram of counts (top-k) or of
// weights (top-p); ties at the cut go by index.  The token is found by running
// sums in index order.
#include "tvp_common.cuh"

namespace tvp {
namespace {

constexpr int kThreads = 1024;
typedef unsigned long long u64;

__device__ __forceinline__ uint32_t order_of(float x) {  // larger logit, larger image
  const uint32_t u = __float_as_uint(x == 0.f ? 0.f : x);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

struct Block {
  u64 warp[32];
  u64 hist[256];
  u64 carry;
  u64 out;
  uint32_t prefix;
};

__device__ u64 block_sum(Block& b, u64 v) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) b.warp[threadIdx.x >> 5] = v;
  __syncthreads();
  u64 s = 0;
  for (int w = 0; w < kThreads / 32; ++w) s += b.warp[w];
  return s;
}

// Exclusive prefix sum over the block's threads, and the total.
__device__ u64 block_scan(Block& b, u64 v, u64* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 x = v;
  for (int o = 1; o < 32; o <<= 1) {
    const u64 y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) b.warp[warp] = x;
  __syncthreads();
  u64 before = 0, all = 0;
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += b.warp[w];
    all += b.warp[w];
  }
  *total = all;
  return before + x - v;
}

// The kept part of a row: images above `key`, and of those equal to it the
// indices up to `last`.
struct Cut {
  uint32_t key;
  int last;
};

__global__ void __launch_bounds__(kThreads)
    sample_kernel(const float* __restrict__ logits, int vocab, long long row_stride,
                  const float* __restrict__ uniforms, const float* __restrict__ temperature,
                  const int32_t* __restrict__ top_k, const float* __restrict__ top_p,
                  const float* __restrict__ min_p, int32_t* __restrict__ tokens) {
  __shared__ Block b;
  const int row = blockIdx.x, tid = threadIdx.x;
  const float* x = logits + (size_t)row * row_stride;
  const float T = temperature ? temperature[row] : 1.f;
  const int k = top_k ? top_k[row] : 0;
  const float P = top_p ? top_p[row] : 1.f;
  const float mp = min_p ? min_p[row] : 0.f;
  const float M = mp > 0.f ? fminf(mp, 1.f) : 0.f;
  // best (image, lowest index)
  u64 best = 0;
  for (int i = tid; i < vocab; i += kThreads) {
    const float v = x[i];
    if (v > -INFINITY) {
      const u64 c = ((u64)order_of(v) << 32) | (uint32_t)~i;
      best = c > best ? c : best;
    }
  }
  for (int o = 16; o > 0; o >>= 1) {
    const u64 c = __shfl_xor_sync(0xffffffffu, best, o);
    best = c > best ? c : best;
  }
  if ((tid & 31) == 0) b.warp[tid >> 5] = best;
  __syncthreads();
  for (int w = 0; w < kThreads / 32; ++w) best = b.warp[w] > best ? b.warp[w] : best;
  if (best == 0 || !(T > 0.f)) {
    if (tid == 0) tokens[row] = best == 0 ? -1 : (int32_t)~(uint32_t)best;
    return;
  }
  const float top = x[~(uint32_t)best];
  const double inv = 1.0 / (double)T;
  auto weight = [&](float v) -> double {  // of a logit above -inf
    return v == top ? 1.0 : exp(((double)v - (double)top) * inv);
  };
  auto fixed = [&](float v) -> u64 { return (u64)__double2ll_rn(weight(v) * 17592186044416.0); };
  Cut cut = {0u, vocab};
  auto kept = [&](float v, int i) {
    if (!(v > -INFINITY)) return false;
    const uint32_t o = order_of(v);
    return o > cut.key || (o == cut.key && i <= cut.last);
  };
  // The cut where the running amount (counts or weights) in falling order
  // first reaches `want` (>= 1).
  auto find = [&](bool mass, u64 want) {
    uint32_t prefix = 0;
    u64 above = 0;  // amount of images above the prefix's range
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += kThreads) b.hist[i] = 0;
      __syncthreads();
      for (int i = tid; i < vocab; i += kThreads) {
        const float v = x[i];
        if (!kept(v, i)) continue;
        const uint32_t o = order_of(v);
        if (shift < 24 && (o >> (shift + 8)) != (prefix >> (shift + 8))) continue;
        atomicAdd(&b.hist[(o >> shift) & 255], mass ? fixed(v) : 1ull);
      }
      __syncthreads();
      if (tid == 0) {
        u64 sum = above;
        int d = 255;
        for (; d > 0 && sum + b.hist[d] < want; --d) sum += b.hist[d];
        b.carry = sum;
        b.prefix = prefix | ((uint32_t)d << shift);
      }
      __syncthreads();
      above = b.carry;
      prefix = b.prefix;
      __syncthreads();
    }
    // ties: the n-th of them in index order
    const u64 unit = mass ? fixed(__uint_as_float((prefix & 0x80000000u) ? prefix ^ 0x80000000u : ~prefix)) : 1ull;
    u64 n = unit ? (want - above + unit - 1) / unit : 1;
    u64 seen = 0;
    if (tid == 0) b.out = (u64)cut.last;
    for (int base = 0; base < vocab; base += kThreads) {
      const int i = base + tid;
      const bool tie = i < vocab && kept(x[i], i) && order_of(x[i]) == prefix;
      u64 all;
      const u64 before = block_scan(b, tie ? 1 : 0, &all);
      if (tie && seen + before + 1 == n) b.out = (u64)i;
      seen += all;
    }
    __syncthreads();
    cut.key = prefix;
    cut.last = (int)b.out;
    __syncthreads();
  };
  if (k > 0 && k < vocab) find(false, (u64)k);
  if (P < 1.f) {
    u64 part = 0;
    for (int i = tid; i < vocab; i += kThreads)
      if (kept(x[i], i)) part += fixed(x[i]);
    const u64 total = block_sum(b, part);
    const double want = ceil((double)P * (double)total);
    find(true, want < 1.0 ? 1ull : (u64)want);
  }
  auto left = [&](float v, int i) -> u64 {
    if (!kept(v, i) || (M > 0.f && weight(v) < (double)M)) return 0;
    return fixed(v);
  };
  u64 part = 0;
  for (int i = tid; i < vocab; i += kThreads) part += left(x[i], i);
  const u64 total = block_sum(b, part);
  const float u = uniforms[row];
  double at = u > 0.f ? (double)fminf(u, 1.f) * (double)total : 0.0;
  u64 point = (u64)at;  // the running sum must exceed it
  if (point >= total) point = total - 1;
  u64 seen = 0;
  for (int base = 0; base < vocab; base += kThreads) {
    const int i = base + tid;
    const u64 w = i < vocab ? left(x[i], i) : 0;
    u64 all;
    const u64 before = seen + block_scan(b, w, &all);
    if (w && before <= point && before + w > point) tokens[row] = i;
    seen += all;
    if (seen > point) return;
  }
}

}  // namespace
}  // namespace tvp

using namespace tvp;

extern "C" int tvp_sample_tokens(const float* d_logits, int rows, int vocab, long long row_stride,
                                 const float* d_uniforms, const float* d_temperature,
                                 const int32_t* d_top_k, const float* d_top_p, const float* d_min_p,
                                 int32_t* d_tokens, tvp_stream_t stream) {
  if (!d_logits || !d_uniforms || !d_tokens || rows <= 0 || vocab <= 0 || row_stride < vocab ||
      (reinterpret_cast<uintptr_t>(d_logits) & 3u))
    return TVP_ERR_INVALID_ARGUMENT;
  if (vocab > TVP_SAMPLE_MAX_VOCAB || rows > 65535) return TVP_ERR_UNSUPPORTED;
  sample_kernel<<<rows, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
      d_logits, vocab, row_stride, d_uniforms, d_temperature, d_top_k, d_top_p, d_min_p, d_tokens);
  return cudaGetLastError() == cudaSuccess ? TVP_OK : TVP_ERR_RUNTIME;
}
