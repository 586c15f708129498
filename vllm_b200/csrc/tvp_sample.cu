// K9 — one token per row of logits from given random numbers.
//
// A cluster of 8 CTAs takes a row: each keeps its eighth of the logits in
// shared memory, so the row is read once from HBM however many passes the
// filters take, and a single row streams through 8 SMs.
//
// Weights.  w_i = exp((x_i - max) / T) is held as an integer of 2^-44 of the
// largest weight, so sums are exact in any order (atomics included) and every
// CTA count gives the same token; a vocabulary of 2^19 ones sums below 2^63.
// FP32 exponentials would not do: with 2^17 logits the running sum's borders
// lie closer together than 2^-24 of the whole.  2^-t is taken in FP64: t in
// 32nds of an octave, a table of the 32 fractions and a Taylor polynomial of
// degree 5 (|f| <= 1/64 octave: the first term left out is below 2^-48).
//
// Filters.  top-k and top-p cut the row at a place in its falling order (value,
// then index).  A histogram of the distance from the maximum, 2048 buckets over
// the distances that still have weight, finds the bucket of the cut; each CTA
// bins its eighth, CTA r adds up buckets [256 r, 256 r + 256) of all eight
// through distributed shared memory.  When few enough logits lie at or above
// that bucket (a usual nucleus), CTA 0 gathers and sorts them, cuts and draws:
// 4 cluster barriers in all.  Otherwise only the cut's own bucket is gathered
// and sorted (or, when equal logits fill it, resolved by radix digits and an
// index count), and the draw goes by sums: per CTA, per warp, then within the
// warp's segment in index order.
#include <cooperative_groups.h>

#include "tvp_common.cuh"

namespace cg = cooperative_groups;

namespace tvp {
namespace {

typedef unsigned long long u64;
constexpr int kCluster = 8;
constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBuckets = 2048;
constexpr int kSegment = kBuckets / kCluster;
constexpr int kList = 2048;  // logits that CTA 0 sorts
constexpr int kFixedBits = 44;
// Distances (in units of T) past which a weight rounds to 0: 45 ln 2.
constexpr float kFar = 31.25f;

struct Cut {
  uint32_t key;  // kept: order image above it, or equal and index <= last
  int last;
};

struct alignas(16) Shared {
  u64 best[kCluster];  // by rank: (order image, ~index) of the largest logit
  float least[kCluster];
  u64 amount[kCluster];  // by rank: a sum that the step at hand exchanges
  u64 count[kCluster];
  u64 fills[kCluster];
  u64 ties[kCluster];
  u64 seg[kSegment];       // this CTA's segment of the cluster's histogram: amounts
  uint32_t seg_n[kSegment];  // and counts
  u64 warp[kWarps];
  u64 found[4];
  double pow[32];  // 2^(-j / 32)
  Cut cut;
  int fill;
};

constexpr size_t kScratchBytes = 2 * kList * 8;  // histogram, then the lists
static_assert(kScratchBytes >= kBuckets * 12, "the histogram fits the lists' place");

__device__ __forceinline__ uint32_t order_of(float x) {  // larger logit, larger image
  const uint32_t u = __float_as_uint(x);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float of_order(uint32_t o) {
  return __uint_as_float((o & 0x80000000u) ? o ^ 0x80000000u : ~o);
}

__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ u64 warp_scan(u64 v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  return v;
}

struct Sampler {
  cg::cluster_group cluster;
  Shared& s;
  const float* x;  // this CTA's logits, NaN as -inf
  unsigned char* scratch;
  int rank, begin, len;
  int tid, lane, warp;
  float top;
  double c32;   // 32 log2(e) / T
  float scale;  // buckets per unit of distance

  __device__ u64 fixed(float v) const {  // weight of a logit above -inf, in 2^-44
    if (v == top) return 1ull << kFixedBits;
    const double t = ((double)top - (double)v) * c32;
    if (!(t <= 32.0 * (kFixedBits + 1))) return 0;
    const double shifted = t + 6755399441055744.0;  // 1.5 * 2^52: rounds to an integer
    const int k = __double2loint(shifted);
    const double f = ((shifted - 6755399441055744.0) - t) * (0.6931471805599453 / 32.0);
    double y = fma(f, 1.0 / 120.0, 1.0 / 24.0);
    y = fma(y, f, 1.0 / 6.0);
    y = fma(y, f, 0.5);
    y = fma(y, f, 1.0);
    y = fma(y, f, 1.0);
    y *= s.pow[k & 31];
    // * 2^(44 - k / 32), then the integer part from the sum's mantissa
    y = fma(y, __hiloint2double((1023 + kFixedBits - (k >> 5)) << 20, 0), 4503599627370496.0);
    return (u64)__double_as_longlong(y) & 0xfffffffffffffull;
  }
  __device__ int bucket(float v) const {  // rises as v falls
    if (v == top) return 0;  // also +inf, whose distance is no number
    return (int)fminf((top - v) * scale, (float)(kBuckets - 1));
  }
  __device__ bool kept(float v, int i) const {
    if (!(v > -INFINITY)) return false;
    const uint32_t o = order_of(v);
    return o > s.cut.key || (o == s.cut.key && i <= s.cut.last);
  }

  // Exclusive sum over the block's threads (all must call), and the total.
  __device__ u64 block_scan(u64 v, u64* total) {
    const u64 inc = warp_scan(v, lane);
    __syncthreads();
    if (lane == 31) s.warp[warp] = inc;
    __syncthreads();
    const u64 w = lane < kWarps ? s.warp[lane] : 0;
    const u64 winc = warp_scan(w, lane);
    *total = __shfl_sync(0xffffffffu, winc, 31);
    const u64 before = __shfl_sync(0xffffffffu, winc - w, warp);
    return before + inc - v;
  }

  // Every CTA's value, to every CTA's `place[rank]`; a cluster barrier inside.
  // Between two calls with one place every CTA passes another cluster barrier
  // after its reads.
  __device__ void share(u64* place, u64 v) {
    if (tid < kCluster) cluster.map_shared_rank(place, tid)[rank] = v;
    cluster.sync();
  }

  // Histogram of the logits that `take` accepts, by `bin` (0 first in falling
  // order): the bin where the running amount reaches want(total); returns the
  // bin, the amount before it, and the counts before and in it.
  struct Border {
    int bin;
    u64 above, want, above_n, in_n;
  };
  template <typename Take, typename Bin, typename Want>
  __device__ Border border(bool mass, Take take, Bin bin, Want want_of) {
    u64* hist = reinterpret_cast<u64*>(scratch);
    uint32_t* hist_n = reinterpret_cast<uint32_t*>(hist + kBuckets);
    for (int i = tid; i < kBuckets; i += kThreads) {
      hist[i] = 0;
      hist_n[i] = 0;
    }
    __syncthreads();
    for (int i = tid; i < len; i += kThreads) {
      const float v = x[i];
      if (!take(v, begin + i)) continue;
      const int b = bin(v);
      atomicAdd(&hist_n[b], 1u);
      if (mass) {
        const u64 w = fixed(v);
        if (w) atomicAdd(&hist[b], w);
      }
    }
    cluster.sync();
    // This CTA's segment over all eight.
    u64 a = 0, n = 0;
    if (tid < kSegment) {
      const int b = rank * kSegment + tid;
#pragma unroll
      for (int r = 0; r < kCluster; ++r) {
        n += cluster.map_shared_rank(hist_n, r)[b];
        if (mass) a += cluster.map_shared_rank(hist, r)[b];
      }
      if (!mass) a = n;
      s.seg[tid] = a;
      s.seg_n[tid] = (uint32_t)n;
    }
    u64 all, all_n;
    block_scan(a, &all);
    block_scan(n, &all_n);
    if (tid < kCluster) cluster.map_shared_rank(s.count, tid)[rank] = all_n;
    share(s.amount, all);
    u64 total = 0;
#pragma unroll
    for (int r = 0; r < kCluster; ++r) total += s.amount[r];
    Border out;
    out.want = want_of(total);
    out.above = out.above_n = 0;
    int seg = 0;
    for (; seg < kCluster - 1 && out.above + s.amount[seg] < out.want; ++seg) {
      out.above += s.amount[seg];
      out.above_n += s.count[seg];
    }
    const u64 ba = tid < kSegment ? cluster.map_shared_rank(s.seg, seg)[tid] : 0;
    const u64 bn = tid < kSegment ? cluster.map_shared_rank(s.seg_n, seg)[tid] : 0;
    const u64 before = block_scan(ba, &all) + out.above;
    const u64 before_n = block_scan(bn, &all_n) + out.above_n;
    if (tid == 0) {  // amounts that never reach `want`: the last bin of all
      s.found[0] = kBuckets - 1;
      s.found[1] = out.above + all;
      s.found[2] = out.above_n + all_n;
      s.found[3] = 0;
    }
    __syncthreads();
    if (tid < kSegment && before < out.want && before + ba >= out.want) {
      s.found[0] = seg * kSegment + tid;
      s.found[1] = before;
      s.found[2] = before_n;
      s.found[3] = bn;
    }
    __syncthreads();
    out.bin = (int)s.found[0];
    out.above = s.found[1];
    out.above_n = s.found[2];
    out.in_n = s.found[3];
    return out;
  }

  // The logits that `take` accepts, as (order image, ~index), in CTA 0's list
  // sorted falling; n of them in the cluster (n <= kList).  Only CTA 0 returns
  // true.
  template <typename Take>
  __device__ bool gather_sorted(Take take, int n) {
    u64* mine = reinterpret_cast<u64*>(scratch);
    if (tid == 0) s.fill = 0;
    __syncthreads();
    for (int i = tid; i < len; i += kThreads) {
      const float v = x[i];
      if (!take(v, begin + i)) continue;
      mine[atomicAdd(&s.fill, 1)] = ((u64)order_of(v) << 32) | (uint32_t)~(begin + i);
    }
    __syncthreads();
    share(s.fills, (u64)s.fill);
    if (rank != 0) return false;
    u64* list = mine + kList;
    int at = 0;
    for (int r = 0; r < kCluster; ++r) {
      const u64* from = cluster.map_shared_rank(mine, r);
      const int m = (int)s.fills[r];
      for (int i = tid; i < m; i += kThreads) list[at + i] = from[i];
      at += m;
    }
    sort_falling(list, n);
    return true;
  }

  // Bitonic sort of list[0..n), padded with zeros to a power of two.
  __device__ void sort_falling(u64* list, int n) {
    int size = 2;
    while (size < n) size <<= 1;
    for (int i = n + tid; i < size; i += kThreads) list[i] = 0;
    __syncthreads();
    for (int k = 2; k <= size; k <<= 1) {
      for (int j = k >> 1; j > 0; j >>= 1) {
        for (int p = tid; p < size / 2; p += kThreads) {
          const int i = 2 * p - (p & (j - 1));
          const u64 a = list[i], b = list[i + j];
          if ((a < b) == ((i & k) == 0)) {
            list[i] = b;
            list[i + j] = a;
          }
        }
        __syncthreads();
      }
    }
  }

  // The integer that a running sum must exceed: u of `total` (> 0).
  __device__ static u64 point_of(float u, u64 total) {
    const double at = u > 0.f ? (double)fminf(u, 1.f) * (double)total : 0.0;
    const u64 p = (u64)at;
    return p < total ? p : total - 1;
  }
  // The amount that reaches `share` (< 1) of `total`, at least 1.
  __device__ static u64 want_of(float share, u64 total) {
    const double w = ceil((double)share * (double)total);
    return w < 1.0 ? 1ull : (u64)w;
  }

  // CTA 0: the token among its sorted list[0..n) (the largest logits, falling):
  // at most the first m, of these the shortest run that weighs `want` (0: the
  // share P of their whole), min-p M, draw u.
  __device__ void finish(const u64* list, int m, u64 want, float P, float M, float u,
                         int32_t* token) {
    constexpr int kEach = kList / kThreads;
    u64* by_index = reinterpret_cast<u64*>(scratch);  // the local list, read before the sort
    // weights in falling order; thread t holds kEach neighbours
    u64 w[kEach], mine = 0, total;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int i = tid * kEach + e;
      w[e] = i < m ? fixed(of_order((uint32_t)(list[i] >> 32))) : 0;
      mine += w[e];
    }
    u64 before = block_scan(mine, &total);
    if (want == 0) want = P < 1.f ? want_of(P, total) : ~0ull;
    int r = 0;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int i = tid * kEach + e;
      if (i < m && (i == 0 || before < want) && !below(list[i], M)) r = i + 1;
      before += w[e];
    }
    if (tid == 0) s.fill = 0;
    __syncthreads();
    r = __reduce_max_sync(0xffffffffu, r);
    if (lane == 0) atomicMax(&s.fill, r);
    __syncthreads();
    r = s.fill;
    // in index order: sort ~index (falling), which keeps the place in the list
    for (int i = tid; i < r; i += kThreads)
      by_index[i] = ((list[i] & 0xffffffffull) << 32) | (uint32_t)i;
    __syncthreads();
    sort_falling(by_index, r);
    mine = 0;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int i = tid * kEach + e;
      w[e] = i < r ? fixed(of_order((uint32_t)(list[(uint32_t)by_index[i]] >> 32))) : 0;
      mine += w[e];
    }
    before = block_scan(mine, &total);
    const u64 point = point_of(u, total);
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int i = tid * kEach + e;
      if (w[e] && before <= point && before + w[e] > point)
        *token = (int32_t)~(uint32_t)(by_index[i] >> 32);
      before += w[e];
    }
  }
  __device__ bool below(u64 entry, float M) const {
    return M > 0.f && below(of_order((uint32_t)(entry >> 32)), M);
  }
  __device__ bool below(float v, float M) const {  // exp((v - top) / T) < M
    return v != top && exp(((double)v - (double)top) * (c32 * (0.6931471805599453 / 32.0))) < (double)M;
  }

  // The cut in bucket `b` (gathered, sorted when it fits) or, for a bucket of
  // more logits, by radix digits of the order image and, among equal logits,
  // by index.  `need`: the amount still wanted of that bucket.
  __device__ void cut_in_bucket(bool mass, int bkt, u64 need, u64 in_n) {
    auto inside = [&](float v, int i) { return kept(v, i) && bucket(v) == bkt; };
    if (in_n <= kList) {
      if (gather_sorted(inside, (int)in_n)) {
        constexpr int kEach = kList / kThreads;
        const u64* list = reinterpret_cast<u64*>(scratch) + kList;
        u64 w[kEach], mine = 0, total;
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
          const int i = tid * kEach + e;
          w[e] = i < (int)in_n ? (mass ? fixed(of_order((uint32_t)(list[i] >> 32))) : 1) : 0;
          mine += w[e];
        }
        u64 before = block_scan(mine, &total);
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
          const int i = tid * kEach + e;
          if (w[e] && before < need && before + w[e] >= need) s.found[0] = list[i];
          before += w[e];
        }
        __syncthreads();
        if (tid < kCluster) {
          const Cut c = {(uint32_t)(s.found[0] >> 32), (int)~(uint32_t)s.found[0]};
          *cluster.map_shared_rank(&s.cut, tid) = c;
        }
      }
      cluster.sync();
      return;
    }
    uint32_t prefix = 0, mask = 0;
    u64 left = need;
    const int shifts[3] = {21, 10, 0}, bits[3] = {11, 11, 10};
    for (int d = 0; d < 3; ++d) {
      const uint32_t top_digit = (1u << bits[d]) - 1u;
      const Border at = border(
          mass, [&](float v, int i) { return inside(v, i) && (order_of(v) & mask) == prefix; },
          [&](float v) { return (int)(top_digit - ((order_of(v) >> shifts[d]) & top_digit)); },
          [&](u64) { return left; });
      prefix |= (top_digit - (uint32_t)at.bin) << shifts[d];
      mask |= top_digit << shifts[d];
      left = at.want - at.above;
    }
    // `left` of the amount of equal logits: the n-th of them by index.
    const u64 unit = mass ? fixed(of_order(prefix)) : 1;
    const u64 nth = (left + unit - 1) / unit;
    const int each = (len + kThreads - 1) / kThreads;
    const int i0 = min(tid * each, len), i1 = min(i0 + each, len);
    u64 ties = 0, all;
    for (int i = i0; i < i1; ++i) ties += kept(x[i], begin + i) && order_of(x[i]) == prefix;
    const u64 before = block_scan(ties, &all);
    share(s.ties, all);
    u64 seen = before;
    for (int r = 0; r < rank; ++r) seen += s.ties[r];
    int last = -1;
    if (seen < nth && seen + ties >= nth)
      for (int i = i0; i < i1; ++i)
        if (kept(x[i], begin + i) && order_of(x[i]) == prefix && ++seen == nth) last = begin + i;
    cluster.sync();  // every CTA has used the old cut
    if (last >= 0)
      for (int r = 0; r < kCluster; ++r) *cluster.map_shared_rank(&s.cut, r) = {prefix, last};
    cluster.sync();
  }
};

__global__ void __launch_bounds__(kThreads, 2)
    sample_kernel(const float* __restrict__ logits, int vocab, int slice, long long row_stride,
                  const float* __restrict__ uniforms, const float* __restrict__ temperature,
                  const int32_t* __restrict__ top_k, const float* __restrict__ top_p,
                  const float* __restrict__ min_p, int32_t* __restrict__ tokens) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ Shared s;
  const cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), row = blockIdx.x / kCluster;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int begin = min(rank * slice, vocab), len = min(slice, vocab - begin);
  float* x = reinterpret_cast<float*>(smem + kScratchBytes);
  if (tid < 32) s.pow[tid] = exp2(-tid / 32.0);
  if (tid == 0) s.cut = {0u, vocab};
  const float T = temperature ? temperature[row] : 1.f;
  const int k = top_k ? top_k[row] : 0;
  const float P = top_p ? top_p[row] : 1.f;
  const float mp = min_p ? min_p[row] : 0.f;
  const float M = mp > 0.f ? fminf(mp, 1.f) : 0.f;
  const float u = uniforms[row];

  // This CTA's logits into shared memory, and the row's largest and least.
  float hi = -INFINITY, lo = INFINITY;
  int hi_at = 0;
  auto put = [&](float v, int i) -> float {
    v = v != v ? -INFINITY : v + 0.f;  // -0 is +0
    if (v > hi) {  // indices rise within a thread: the lowest of equals stays
      hi = v;
      hi_at = begin + i;
    }
    if (v > -INFINITY) lo = fminf(lo, v);
    return v;
  };
  const float* src = logits + (size_t)row * row_stride + begin;
  int done = 0;
  if ((reinterpret_cast<uintptr_t>(src) & 15u) == 0) {
    const int n4 = len / 4;
    constexpr int kBatch = 8;
    for (int base = tid; base < n4; base += kBatch * kThreads) {
      float4 v[kBatch];
#pragma unroll
      for (int e = 0; e < kBatch; ++e)
        if (base + e * kThreads < n4)
          v[e] = __ldcs(reinterpret_cast<const float4*>(src) + base + e * kThreads);
#pragma unroll
      for (int e = 0; e < kBatch; ++e) {
        const int q = base + e * kThreads;
        if (q >= n4) break;
        float4 w;
        w.x = put(v[e].x, 4 * q);
        w.y = put(v[e].y, 4 * q + 1);
        w.z = put(v[e].z, 4 * q + 2);
        w.w = put(v[e].w, 4 * q + 3);
        reinterpret_cast<float4*>(x)[q] = w;
      }
    }
    done = n4 * 4;
  }
  constexpr int kBatch1 = 16;
  for (int base = done + tid; base < len; base += kBatch1 * kThreads) {
    float v[kBatch1];
#pragma unroll
    for (int e = 0; e < kBatch1; ++e)
      if (base + e * kThreads < len) v[e] = __ldcs(src + base + e * kThreads);
#pragma unroll
    for (int e = 0; e < kBatch1; ++e) {
      const int i = base + e * kThreads;
      if (i >= len) break;
      x[i] = put(v[e], i);
    }
  }
  u64 best = hi > -INFINITY ? ((u64)order_of(hi) << 32) | (uint32_t)~hi_at : 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const u64 c = __shfl_xor_sync(0xffffffffu, best, o);
    best = c > best ? c : best;
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
  }
  __shared__ float warp_lo[kWarps];
  if (lane == 0) {
    s.warp[warp] = best;
    warp_lo[warp] = lo;
  }
  __syncthreads();
  if (tid < kCluster) {
    for (int w = 0; w < kWarps; ++w) {
      best = s.warp[w] > best ? s.warp[w] : best;
      lo = fminf(lo, warp_lo[w]);
    }
    cluster.map_shared_rank(s.best, tid)[rank] = best;
    cluster.map_shared_rank(s.least, tid)[rank] = lo;
  }
  cluster.sync();
  best = s.best[0];
  lo = s.least[0];
#pragma unroll
  for (int r = 1; r < kCluster; ++r) {
    best = s.best[r] > best ? s.best[r] : best;
    lo = fminf(lo, s.least[r]);
  }
  if (best == 0 || !(T > 0.f)) {
    if (rank == 0 && tid == 0) tokens[row] = best == 0 ? -1 : (int32_t)~(uint32_t)best;
    return;
  }
  const float top = of_order((uint32_t)(best >> 32));
  // Buckets over the distances that have weight, or over the row's own range
  // where that is narrower.
  const float range = fminf(kFar * T, top - lo);
  Sampler a = {cluster, s, x, smem, rank, begin, len, tid, lane, warp, top,
               46.16624130844683 / (double)T, range > 0.f ? (float)kBuckets / range : 0.f};
  const bool by_k = k > 0 && k < vocab;
  if (by_k || P < 1.f) {
    auto any = [&](float v, int i) { return a.kept(v, i); };
    auto bin = [&](float v) { return a.bucket(v); };
    for (int filter = by_k ? 0 : 1; filter < 2; ++filter) {
      const bool mass = filter == 1;
      if (mass && !(P < 1.f)) break;
      const Sampler::Border at = a.border(mass, any, bin, [&](u64 total) {
        return mass ? Sampler::want_of(P, total) : (u64)k;
      });
      const u64 n = at.above_n + at.in_n;
      if (at.in_n == 0) continue;  // fewer logits above -inf than k
      if (n <= kList) {
        if (a.gather_sorted([&](float v, int i) { return a.kept(v, i) && a.bucket(v) <= at.bin; },
                            (int)n)) {
          // After a histogram of weights the amount wanted is known, of the
          // whole; after one of counts, top-p is of the k that are left.
          a.finish(reinterpret_cast<u64*>(smem) + kList, mass ? (int)n : min((int)n, k),
                   mass ? at.want : 0, P, M, u, tokens + row);
        }
        cluster.sync();  // CTA 0 reads the others' lists
        return;
      }
      a.cut_in_bucket(mass, at.bin, at.want - at.above, at.in_n);
    }
  }
  // The draw by sums: warps take neighbouring segments of the CTA's logits.
  auto weight = [&](int i) -> u64 {
    if (i >= len || !a.kept(x[i], begin + i) || (M > 0.f && a.below(x[i], M))) return 0;
    return a.fixed(x[i]);
  };
  const int part = (len + kWarps * 32 - 1) / (kWarps * 32) * 32;
  const int w0 = min(warp * part, len), w1 = min(w0 + part, len);
  u64 sum = 0;
  for (int i = w0 + lane; i < w1; i += 32) sum += weight(i);
  sum = warp_sum(sum);
  __syncthreads();
  if (lane == 0) s.warp[warp] = sum;
  __syncthreads();
  u64 mine = 0;
  for (int w = 0; w < kWarps; ++w) mine += s.warp[w];
  a.share(s.amount, mine);
  u64 total = 0, before = 0;
#pragma unroll
  for (int r = 0; r < kCluster; ++r) {
    if (r < rank) before += s.amount[r];
    total += s.amount[r];
  }
  const u64 point = Sampler::point_of(u, total);
  for (int w = 0; w < warp; ++w) before += s.warp[w];
  if (before > point || before + sum <= point) return;
  for (int i = w0; i < w1; i += 32) {
    const u64 w = i + lane < w1 ? weight(i + lane) : 0;
    const u64 inc = before + warp_scan(w, lane);
    if (w && inc - w <= point && inc > point) tokens[row] = begin + i + lane;
    before = __shfl_sync(0xffffffffu, inc, 31);
    if (before > point) return;
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
  auto slice_of = [](int v) { return ((v + kCluster - 1) / kCluster + 3) / 4 * 4; };
  static bool configured[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return TVP_ERR_RUNTIME;
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    if (cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)(kScratchBytes + (size_t)slice_of(TVP_SAMPLE_MAX_VOCAB) * 4)) !=
        cudaSuccess)
      return TVP_ERR_RUNTIME;
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  const int slice = slice_of(vocab);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)rows * kCluster);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kScratchBytes + (size_t)slice * 4;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kCluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, sample_kernel, d_logits, vocab, slice, row_stride, d_uniforms,
                            d_temperature, d_top_k, d_top_p, d_min_p, d_tokens) == cudaSuccess
             ? TVP_OK
             : TVP_ERR_RUNTIME;
}
