// K9 — one token per row of logits from given random numbers.
//
// A cluster of 8 CTAs takes a row: each keeps its eighth of the logits in
// shared memory, so the row is read once from HBM however many passes the
// filters take, and a single row streams through 8 SMs.
//
// Weights.  w_i = exp((x_i - max) / T) is held as an integer of 2^-44 of the
// largest weight, so sums are exact in any order (atomics included) and every
// CTA count gives the same token; a vocabulary of 2^19 ones sums below 2^63.
// Plain FP32 exponentials would not do: with 2^17 logits the running sum's
// borders lie closer together than 2^-24 of the whole.  2^-t is taken with t in
// 256ths of an octave, a table of the 256 fractions and a Taylor polynomial of
// degree 3 (|f| <= 1/512 octave: the first term left out is below 2^-42).
//
// Filters.  top-k and top-p cut the row at a place in its falling order (value,
// then index).  A histogram of the distance from the maximum, 2048 buckets over
// the distances that still have weight, finds the bucket of the cut; each CTA
// bins its eighth, CTA r adds up buckets [256 r, 256 r + 256) of all eight
// through distributed shared memory.  When few enough logits lie at or above
// that bucket (a usual nucleus), CTA 0 gathers them, cuts and draws, all by
// comparing each with each; 4 cluster barriers in all.  Otherwise only the cut's
// own bucket is gathered (or, when it holds many, resolved by radix digits and a
// count of equal logits by index), and the draw goes by sums: per CTA, per warp,
// then within the warp's segment in index order.
#include <cfloat>

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
constexpr int kBlocks = kBuckets / 32;  // two per lane of a warp
static_assert(kBlocks == 64 && kBuckets / kCluster <= kThreads, "border() deals them out so");
#ifndef TVP_STREAM_ROWS
#define TVP_STREAM_ROWS 64
#endif
constexpr int kStreamRows = TVP_STREAM_ROWS;  // from so many rows on, one CTA takes a row
constexpr int kList = 512;  // logits of a bucket that CTA 0 takes in
// Logits at or above the cut that CTA 0 finishes by itself.  Each-with-each takes
// 2 x 0.7 us for 128 and 2 x 11 us for 512; the sums take some 3 us of passes.
constexpr int kFew = 160;
constexpr int kFixedBits = 44;
// Distances (in units of T) past which a weight rounds to 0: 45 ln 2.
constexpr float kFar = 31.25f;

struct Cut {
  uint32_t key;  // kept: order image above it, or equal and index <= last
  int last;
};

// The bin where a running amount reaches `want`: the amount before it, and the
// counts before and in it (0: the amount is not reached).
struct Border {
  int bin, above_n, in_n;
  u64 above, want;
};

template <int CL>
struct alignas(16) Shared {
  static constexpr int kSegment = kBuckets / CL;
  u64 best[CL];  // by rank: (order image, ~index) of the largest logit
  float least[CL];
  u64 amount[CL];  // by rank: a sum that the step at hand exchanges
  int fills[CL];
  u64 ties[CL];
  u64 seg[CL > 1 ? kSegment : 1];         // this CTA's segment of the cluster's histogram: amounts
  uint32_t seg_n[CL > 1 ? kSegment : 1];  // and counts
  u64 sub[kBlocks];                       // every 32 buckets of the whole histogram: amounts
  uint32_t sub_n[kBlocks];                // and counts
  u64 warp[kWarps];
  float warp_lo[kWarps];
  double pow[256];
  Cut cut;
  Border border;
  int fill;
};

// 2^(-j / 256), by the Taylor series of the exponential.
struct Powers {
  double d[256];
  constexpr Powers() : d() {
    for (int j = 0; j < 256; ++j) {
      const double x = -j * (0.6931471805599453 / 256);
      double term = 1, sum = 1;
      for (int n = 1; n < 24; ++n) {
        term *= x / n;
        sum += term;
      }
      d[j] = sum;
    }
  }
};
__device__ const Powers g_powers = Powers();

constexpr size_t kScratchBytes = kBuckets * 12;  // histogram, then the lists
static_assert(kScratchBytes >= 3 * kList * 8, "the lists fit the histogram's place");

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
template <typename V>
__device__ __forceinline__ V warp_scan(V v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  return v;
}

// 64-bit sum into shared memory from two 32-bit ones: the low words' carry goes
// with the high word, which most weights do not touch.
__device__ __forceinline__ void shared_add(u64* at, u64 w) {
  uint32_t* p = reinterpret_cast<uint32_t*>(at);
  const uint32_t lo = (uint32_t)w;
  uint32_t hi = (uint32_t)(w >> 32);
  if (lo) hi += atomicAdd(p, lo) > ~lo;
  if (hi) atomicAdd(p + 1, hi);
}

template <int CL>
struct Sampler {
  Shared<CL>& s;
  const float* x;  // this CTA's logits: in shared memory (CL > 1), or the row itself
  unsigned char* scratch;
  int rank, begin, len, head;  // logits before the first aligned four of x
  int tid, lane, warp;
  float top;    // finite
  float far;    // logits below it have no weight
  double c256;  // 256 log2(e) / T
  float scale;  // buckets per unit of distance
  bool infinite;  // the row holds +inf: these count as 0, the others as -inf
  bool cutting;  // a filter has cut the row
  Cut cut;

  // The CTAs of a row: barrier, and another one's shared memory.
  __device__ static void sync() {
    if (CL > 1)
      cg::this_cluster().sync();
    else
      __syncthreads();
  }
  template <typename V>
  __device__ static V* of_rank(V* place, int r) {
    return CL > 1 ? cg::this_cluster().map_shared_rank(place, r) : place;
  }

  // A logit as the sampler takes it: NaN is -inf, -0 is +0.  Shared memory holds
  // them so.
  __device__ __forceinline__ float canon(float v) const {
    if (CL > 1) return v;
    v = v != v ? -INFINITY : v + 0.f;
    return !infinite ? v : v == INFINITY ? 0.f : -INFINITY;
  }
  __device__ __forceinline__ float at(int i) const { return canon(x[i]); }

  // Calls visit(four logits, index of the first) for the quads [q0, q1) with
  // q % kThreads == tid, q0 <= q: `step` threads apart, several loads in flight.
  template <typename Visit>
  __device__ __forceinline__ void quads(int q0, int q1, int step, Visit visit) const {
    constexpr int kBatch = CL > 1 ? 1 : 4;
    const float4* x4 = reinterpret_cast<const float4*>(x + head);
    for (int q = q0; q < q1; q += kBatch * step) {
      float4 v[kBatch];
#pragma unroll
      for (int e = 0; e < kBatch; ++e)
        if (q + e * step < q1) v[e] = x4[q + e * step];
#pragma unroll
      for (int e = 0; e < kBatch; ++e)
        if (q + e * step < q1)
          visit(make_float4(canon(v[e].x), canon(v[e].y), canon(v[e].z), canon(v[e].w)),
                head + 4 * (q + e * step));
    }
  }
  __device__ __forceinline__ int n_quads() const { return (len - head) / 4; }
  // All logits of the CTA; the ones around the quads come as a four with -inf.
  template <typename Visit>
  __device__ __forceinline__ void each_four(Visit visit) const {
    const int n4 = n_quads();
    quads(tid, n4, kThreads, visit);
    const int tail = len - head - 4 * n4;
    if (tid < head + tail) {
      const int i = tid < head ? tid : len - tail + (tid - head);
      visit(make_float4(at(i), -INFINITY, -INFINITY, -INFINITY), i);
    }
  }

  // Weight of a logit in 2^-44 of the largest's.  Without branches, so that the
  // chains of several logits overlap.  (An FP32 form that carries the products'
  // rounding errors along, good to 2^-31, measured the same time: 11 FP64
  // instructions against some 30 FP32 ones.)
  __device__ __forceinline__ u64 fixed(float v) const {
    const double t = ((double)top - (double)fmaxf(v, far)) * c256;
    const double shifted = t + 6755399441055744.0;  // 1.5 * 2^52: rounds to an integer
    const int k = __double2loint(shifted);
    const double f = ((shifted - 6755399441055744.0) - t) * (0.6931471805599453 / 256);
    double y = fma(f, 1.0 / 6.0, 0.5);
    y = fma(y, f, 1.0);
    y = fma(y, f, 1.0);
    y *= s.pow[k & 255];
    // * 2^(44 - k / 256), then the integer part from the sum's mantissa
    y = fma(y, __hiloint2double((1023 + kFixedBits - (k >> 8)) << 20, 0), 4503599627370496.0);
    return v < far ? 0ull : (u64)__double_as_longlong(y) & 0xfffffffffffffull;
  }
  __device__ __forceinline__ int bucket(float v) const {  // rises as v falls
    return (int)fminf((top - v) * scale, (float)(kBuckets - 1));
  }
  __device__ __forceinline__ bool kept(float v, int i) const {  // with a weight, that is
    if (v < far) return false;
    if (!cutting) return true;
    const uint32_t o = order_of(v);
    return o > cut.key || (o == cut.key && i <= cut.last);
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
  template <typename V>
  __device__ void share(V* place, V v) {
    if (tid < CL) of_rank(place, tid)[rank] = v;
    sync();
  }

  static constexpr int kSegment = kBuckets / CL;

  // Histogram of the logits that `take` accepts, by `bin` (0 first in falling
  // order), and the bin where the running amount reaches want(total).
  template <bool MASS, typename Take, typename Bin, typename Want>
  __device__ Border border(Take take, Bin bin, Want want_of) {
    u64* hist = reinterpret_cast<u64*>(scratch);
    uint32_t* hist_n = reinterpret_cast<uint32_t*>(hist + kBuckets);
    for (int i = tid; i < (int)(kScratchBytes / 16); i += kThreads)
      reinterpret_cast<uint4*>(scratch)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    auto add = [&](float v, u64 w, int i) {
      if (!take(v, begin + i)) return;
      const int b = bin(v);
      atomicAdd(&hist_n[b], 1u);
      if (MASS) shared_add(&hist[b], w);
    };
    each_four([&](const float4& v, int i) {
      if (fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) < far) return;
      u64 w[4] = {};
      if (MASS) {
        w[0] = fixed(v.x);
        w[1] = fixed(v.y);
        w[2] = fixed(v.z);
        w[3] = fixed(v.w);
      }
      add(v.x, w[0], i);
      add(v.y, w[1], i + 1);
      add(v.z, w[2], i + 2);
      add(v.w, w[3], i + 3);
    });
    sync();
    if (CL > 1) {
      // This CTA's segment over all, one bucket per thread of 8 warps, and the
      // sum of each warp's 32 to every CTA.
      if (tid < kSegment) {
        const int b = rank * kSegment + tid;
        uint32_t ns[CL];
        u64 as[CL];
#pragma unroll
        for (int r = 0; r < CL; ++r) {
          ns[r] = of_rank(hist_n, r)[b];
          if (MASS) as[r] = of_rank(hist, r)[b];
        }
        uint32_t n = 0;
        u64 a = 0;
#pragma unroll
        for (int r = 0; r < CL; ++r) {
          n += ns[r];
          a += MASS ? as[r] : ns[r];
        }
        s.seg[tid] = a;
        s.seg_n[tid] = n;
        a = MASS ? warp_sum(a) : 0;
        n = __reduce_add_sync(0xffffffffu, n);
        if (lane < CL) {
          of_rank(s.sub, lane)[rank * (kSegment / 32) + warp] = MASS ? a : n;
          of_rank(s.sub_n, lane)[rank * (kSegment / 32) + warp] = n;
        }
      }
    } else {
      for (int block = warp; block < kBlocks; block += kWarps) {
        const uint32_t n = __reduce_add_sync(0xffffffffu, hist_n[block * 32 + lane]);
        const u64 a = MASS ? warp_sum(hist[block * 32 + lane]) : n;
        if (lane == 0) {
          s.sub[block] = a;
          s.sub_n[block] = n;
        }
      }
    }
    sync();
    // One warp finds the 32 buckets, then the bucket.
    if (warp == 0) find_border<MASS>(want_of);
    __syncthreads();
    return s.border;
  }
  template <bool MASS, typename Want>
  __device__ __forceinline__ void find_border(Want want_of) {
    Border out;
    const u64 s0 = s.sub[2 * lane], s1 = s.sub[2 * lane + 1];
    const uint32_t n0 = s.sub_n[2 * lane], n1 = s.sub_n[2 * lane + 1];
    const u64 inc = warp_scan(s0 + s1, lane);
    const uint32_t inc_n = warp_scan(n0 + n1, lane);
    out.want = want_of(__shfl_sync(0xffffffffu, inc, 31));
    const u64 before = inc - s0 - s1;
    const uint32_t at = __ballot_sync(0xffffffffu, before < out.want && inc >= out.want);
    if (at == 0) {
      out.bin = kBuckets - 1;
      out.above = __shfl_sync(0xffffffffu, inc, 31);
      out.above_n = (int)__shfl_sync(0xffffffffu, inc_n, 31);
      out.in_n = 0;
      if (lane == 0) s.border = out;
      return;
    }
    const int src = __ffs(at) - 1;
    const bool second = before + s0 < out.want;
    const int block = 2 * src + __shfl_sync(0xffffffffu, (int)second, src);
    const u64 above = __shfl_sync(0xffffffffu, second ? before + s0 : before, src);
    const uint32_t above_n =
        __shfl_sync(0xffffffffu, second ? inc_n - n1 : inc_n - n0 - n1, src);
    u64 ba;
    uint32_t bn;
    if (CL > 1) {
      constexpr int kPer = kSegment / 32;  // blocks of a CTA
      const int place = block % kPer * 32 + lane;
      ba = of_rank(s.seg, block / kPer)[place];
      bn = of_rank(s.seg_n, block / kPer)[place];
    } else {
      const u64* hist = reinterpret_cast<const u64*>(scratch);
      bn = reinterpret_cast<const uint32_t*>(hist + kBuckets)[block * 32 + lane];
      ba = MASS ? hist[block * 32 + lane] : bn;
    }
    const u64 upto = above + warp_scan(ba, lane);
    const uint32_t upto_n = above_n + warp_scan(bn, lane);
    const int hit = __ffs(__ballot_sync(0xffffffffu, upto >= out.want)) - 1;
    out.bin = block * 32 + hit;
    out.above = __shfl_sync(0xffffffffu, upto - ba, hit);
    out.above_n = (int)__shfl_sync(0xffffffffu, upto_n - bn, hit);
    out.in_n = (int)__shfl_sync(0xffffffffu, bn, hit);
    if (lane == 0) s.border = out;
  }

  // The n (<= kList) logits that `take` accepts, as (order image, ~index), in
  // CTA 0's list, in no order.  Only CTA 0 returns true.
  __device__ u64* list() const { return reinterpret_cast<u64*>(scratch) + kList; }
  __device__ u64* weights() const { return reinterpret_cast<u64*>(scratch) + 2 * kList; }
  template <typename Take>
  __device__ bool gather(Take take, int n) {
    u64* mine = reinterpret_cast<u64*>(scratch);
    if (tid == 0) s.fill = 0;
    __syncthreads();
    if (CL == 1) mine = list();
    auto put = [&](float v, int i) {
      if (take(v, begin + i))
        mine[atomicAdd(&s.fill, 1)] = ((u64)order_of(v) << 32) | (uint32_t)~(begin + i);
    };
    each_four([&](const float4& v, int i) {
      if (fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) < far) return;
      put(v.x, i);
      put(v.y, i + 1);
      put(v.z, i + 2);
      put(v.w, i + 3);
    });
    __syncthreads();
    if (CL == 1) return true;
    share(s.fills, s.fill);
    if (rank != 0) return false;
    if (tid < n) {
      int r = 0, from = tid;
#pragma unroll
      for (int q = 0; q < CL - 1; ++q)
        if (r == q && from >= s.fills[q]) {
          from -= s.fills[q];
          ++r;
        }
      list()[tid] = of_rank(mine, r)[from];
    }
    __syncthreads();
    return true;
  }

  // The list is not sorted: an entry's place in the falling order is what lies
  // ahead of it, counted by `parts` threads per entry.
  struct Share {
    int parts, i, q;  // threads per entry, this thread's entry, its part
  };
  __device__ Share share_of(int n) const {
    int parts = 32;
    while (kThreads / parts < n) parts >>= 1;
    return {parts, tid / parts, tid % parts};
  }
  template <typename V>
  __device__ static V over_parts(V v, int parts) {
    for (int o = 1; o < parts; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
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

  // CTA 0: the token among its list of n (the largest logits): at most the
  // first k (0: all), of these the shortest run that weighs `want` (0: the share
  // P of their whole), min-p M, draw u.
  __device__ void finish(int n, int k, u64 want, float P, float M, float u, int32_t* token) {
    const u64* entries = list();
    u64* w = weights();
    if (tid < n) w[tid] = fixed(of_order((uint32_t)(entries[tid] >> 32)));
    __syncthreads();
    const Share sh = share_of(n);
    const bool mine = sh.i < n;
    const u64 me = mine ? entries[sh.i] : 0, weight = mine ? w[sh.i] : 0;
    int ahead = 0;
    u64 mass = 0, total;
    for (int j = sh.q; j < n; j += sh.parts)
      if (entries[j] > me) {
        ++ahead;
        mass += w[j];
      }
    ahead = over_parts(ahead, sh.parts);
    mass = over_parts(mass, sh.parts);
    bool keep = mine && (k == 0 || ahead < k);
    if (want == 0) {
      block_scan(keep && sh.q == 0 ? weight : 0, &total);
      want = P < 1.f ? want_of(P, total) : ~0ull;
    }
    keep = keep && (ahead == 0 || mass < want) && !below(of_order((uint32_t)(me >> 32)), M);
    block_scan(keep && sh.q == 0 ? weight : 0, &total);  // and every thread has read w
    if (mine && sh.q == 0 && !keep) w[sh.i] = 0;
    __syncthreads();
    // the running sum in index order
    u64 lower = 0;
    for (int j = sh.q; j < n; j += sh.parts) lower += (uint32_t)entries[j] > (uint32_t)me ? w[j] : 0;
    lower = over_parts(lower, sh.parts);
    const u64 point = point_of(u, total);
    if (keep && sh.q == 0 && lower <= point && lower + weight > point)
      *token = (int32_t)~(uint32_t)me;
  }
  __device__ __forceinline__ bool below(float v, float M) const {  // exp((v - top) / T) < M
    return M > 0.f && v != top &&
           exp(((double)v - (double)top) * (c256 * (0.6931471805599453 / 256))) < (double)M;
  }

  // The cut in bucket `bkt`: among its logits gathered, or, for a bucket of
  // many, by radix digits of the order image and, among equal logits, by index.
  // `need`: the amount still wanted of that bucket.
  template <bool MASS>
  __device__ void cut_in_bucket(int bkt, u64 need, int in_n) {
    auto inside = [&](float v, int i) { return bucket(v) == bkt && kept(v, i); };
    if (in_n <= kList) {
      if (gather(inside, in_n)) {
        const u64* entries = list();
        u64* w = weights();
        if (tid < in_n) w[tid] = MASS ? fixed(of_order((uint32_t)(entries[tid] >> 32))) : 1;
        __syncthreads();
        const Share sh = share_of(in_n);
        const u64 me = sh.i < in_n ? entries[sh.i] : 0;
        u64 ahead = 0;
        for (int j = sh.q; j < in_n; j += sh.parts) ahead += entries[j] > me ? w[j] : 0;
        ahead = over_parts(ahead, sh.parts);
        if (sh.i < in_n && sh.q == 0 && ahead < need && ahead + w[sh.i] >= need) {
          const Cut c = {(uint32_t)(me >> 32), (int)~(uint32_t)me};
          for (int r = 0; r < CL; ++r) *of_rank(&s.cut, r) = c;
        }
      }
      sync();
      cut = s.cut;
      cutting = true;
      return;
    }
    uint32_t prefix = 0, mask = 0;
    u64 left = need;
    const int shifts[3] = {21, 10, 0}, bits[3] = {11, 11, 10};
    for (int d = 0; d < 3; ++d) {
      const uint32_t top_digit = (1u << bits[d]) - 1u;
      const Border part = border<MASS>(
          [&](float v, int i) { return inside(v, i) && (order_of(v) & mask) == prefix; },
          [&](float v) { return (int)(top_digit - ((order_of(v) >> shifts[d]) & top_digit)); },
          [&](u64) { return left; });
      prefix |= (top_digit - (uint32_t)part.bin) << shifts[d];
      mask |= top_digit << shifts[d];
      left = part.want - part.above;
    }
    // `left` of the amount of equal logits: the n-th of them by index.
    const u64 unit = MASS ? fixed(of_order(prefix)) : 1;
    const u64 nth = (left + unit - 1) / unit;
    const int each = (len + kThreads - 1) / kThreads;
    const int i0 = min(tid * each, len), i1 = min(i0 + each, len);
    u64 ties = 0, all;
    for (int i = i0; i < i1; ++i) ties += kept(at(i), begin + i) && order_of(at(i)) == prefix;
    const u64 before = block_scan(ties, &all);
    share(s.ties, all);
    u64 seen = before;
    for (int r = 0; r < rank; ++r) seen += s.ties[r];
    int last = -1;
    if (seen < nth && seen + ties >= nth)
      for (int i = i0; i < i1; ++i)
        if (kept(at(i), begin + i) && order_of(at(i)) == prefix && ++seen == nth) last = begin + i;
    if (last >= 0)
      for (int r = 0; r < CL; ++r) *of_rank(&s.cut, r) = {prefix, last};
    sync();
    cut = s.cut;
    cutting = true;
  }

  // One filter: true when it ended the row (the token is written).
  template <bool MASS, typename Want>
  __device__ bool filter(Want want_of, int k, float P, float M, float u, int32_t* token) {
    const Border edge = border<MASS>([&](float v, int i) { return kept(v, i); },
                                   [&](float v) { return bucket(v); }, want_of);
    if (edge.in_n == 0) return false;  // fewer logits with a weight than k
    const int n = edge.above_n + edge.in_n;
    if (n > kFew) {
      cut_in_bucket<MASS>(edge.bin, edge.want - edge.above, edge.in_n);
      return false;
    }
    // After a histogram of weights the amount wanted is known, of the whole;
    // after one of counts, top-p is of the k that are left.
    if (gather([&](float v, int i) { return bucket(v) <= edge.bin && kept(v, i); }, n))
      finish(n, MASS ? 0 : k, MASS ? edge.want : 0, P, M, u, token);
    sync();  // CTA 0 reads the others' lists
    return true;
  }
};

template <int CL>
__global__ void __launch_bounds__(kThreads, 2)
    sample_kernel(const float* __restrict__ logits, int vocab, int slice, long long row_stride,
                  const float* __restrict__ uniforms, const float* __restrict__ temperature,
                  const int32_t* __restrict__ top_k, const float* __restrict__ top_p,
                  const float* __restrict__ min_p, int32_t* __restrict__ tokens) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ Shared<CL> s;
  const int rank = CL > 1 ? (int)cg::this_cluster().block_rank() : 0, row = blockIdx.x / CL;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int begin = min(rank * slice, vocab), len = min(slice, vocab - begin);
  const float* src = logits + (size_t)row * row_stride + begin;
  // Logits before the first 16-byte boundary.
  const int head = min((int)((0u - (uint32_t)(reinterpret_cast<uintptr_t>(src) >> 2)) & 3u), len);
  float* x = reinterpret_cast<float*>(smem + kScratchBytes);  // CL > 1

  // The row's largest and least logit; with CL > 1 the CTA's logits also go into
  // shared memory.
  float hi = -INFINITY, lo = INFINITY;
  int hi_at = 0;
  auto see = [&](float v, int i) {
    v = v != v ? -INFINITY : v + 0.f;  // -0 is +0
    if (v > hi || (v == hi && begin + i < hi_at)) {
      hi = v;
      hi_at = begin + i;
    }
    if (v > -INFINITY) lo = fminf(lo, v);
    return v;
  };
  const int n4 = (len - head) / 4;
  constexpr int kBatch = 8;
  for (int base = tid; base < n4; base += kBatch * kThreads) {
    float4 v[kBatch];
#pragma unroll
    for (int e = 0; e < kBatch; ++e)
      if (base + e * kThreads < n4)
        v[e] = __ldg(reinterpret_cast<const float4*>(src + head) + base + e * kThreads);
#pragma unroll
    for (int e = 0; e < kBatch; ++e) {
      const int i = head + 4 * (base + e * kThreads);
      if (base + e * kThreads >= n4) break;
      const float4 c = make_float4(see(v[e].x, i), see(v[e].y, i + 1), see(v[e].z, i + 2),
                                   see(v[e].w, i + 3));
      if (CL > 1) {
        if (head == 0) {
          *reinterpret_cast<float4*>(x + i) = c;
        } else {
          x[i] = c.x;
          x[i + 1] = c.y;
          x[i + 2] = c.z;
          x[i + 3] = c.w;
        }
      }
    }
  }
  const int tail = len - head - 4 * n4;
  if (tid < head + tail) {
    const int i = tid < head ? tid : len - tail + (tid - head);
    const float c = see(src[i], i);
    if (CL > 1) x[i] = c;
  }
  u64 best = hi > -INFINITY ? ((u64)order_of(hi) << 32) | (uint32_t)~hi_at : 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const u64 c = __shfl_xor_sync(0xffffffffu, best, o);
    best = c > best ? c : best;
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
  }
  if (lane == 0) {
    s.warp[warp] = best;
    s.warp_lo[warp] = lo;
  }
  if (tid < 256) s.pow[tid] = g_powers.d[tid];
  float T = temperature ? temperature[row] : 1.f;
  if (T > 0.f) T = fmaxf(T, 2e-36f);  // 256 log2(e) / T stays finite
  const int k = top_k ? top_k[row] : 0;
  const float P = top_p ? top_p[row] : 1.f;
  const float mp = min_p ? min_p[row] : 0.f;
  const float M = mp > 0.f ? fminf(mp, 1.f) : 0.f;
  const float u = uniforms[row];
  __syncthreads();
  if (tid < CL) {
    for (int w = 0; w < kWarps; ++w) {
      best = s.warp[w] > best ? s.warp[w] : best;
      lo = fminf(lo, s.warp_lo[w]);
    }
    Sampler<CL>::of_rank(s.best, tid)[rank] = best;
    Sampler<CL>::of_rank(s.least, tid)[rank] = lo;
  }
  Sampler<CL>::sync();
  best = s.best[0];
  lo = s.least[0];
#pragma unroll
  for (int r = 1; r < CL; ++r) {
    best = s.best[r] > best ? s.best[r] : best;
    lo = fminf(lo, s.least[r]);
  }
  if (best == 0 || !(T > 0.f)) {
    if (rank == 0 && tid == 0) tokens[row] = best == 0 ? -1 : (int32_t)~(uint32_t)best;
    return;
  }
  float top = of_order((uint32_t)(best >> 32));
  const bool infinite = top == INFINITY;
  if (infinite) {  // these share the mass: zeros among -inf
    if (CL > 1)
      for (int i = tid; i < len; i += kThreads) x[i] = x[i] == INFINITY ? 0.f : -INFINITY;
    __syncthreads();
    top = lo = 0.f;
  }
  // Buckets over the distances that have weight, or over the row's own range
  // where that is narrower.
  const float range = fminf(kFar * T, top - lo);
  Sampler<CL> a = {s, CL > 1 ? x : src, smem, rank, begin, len, CL > 1 ? 0 : head, tid, lane, warp,
                   top, fmaxf(top - kFar * T, -FLT_MAX), 369.3299304675746 / (double)T,
                   range > 0.f ? (float)kBuckets / range : 0.f, infinite, false, {}};
  if (k > 0 && k < vocab &&
      a.template filter<false>([&](u64) { return (u64)k; }, k, P, M, u, tokens + row))
    return;
  if (P < 1.f &&
      a.template filter<true>([&](u64 total) { return Sampler<CL>::want_of(P, total); }, k, P, M, u,
                              tokens + row))
    return;
  // The draw by sums: warps take neighbouring segments of the CTA's quads, the
  // first one also what comes before them, the last one what comes after.
  // min-p: logits well above and below its distance need no exponential.
  const float dist = T == INFINITY ? T : M > 0.f && M < 1.f ? (float)(-log((double)M) * T) : 0.f;
  auto stays = [&](float v, int i) {
    if (!a.kept(v, begin + i)) return false;
    const float d = top - v;
    return M == 0.f || d < dist * 0.99999f || (d <= dist * 1.00001f && !a.below(v, M));
  };
  auto weight = [&](int i) -> u64 {
    const float v = a.at(i);
    return stays(v, i) ? a.fixed(v) : 0;
  };
  const int all = a.n_quads(), part = (all + kWarps * 32 - 1) / (kWarps * 32) * 32;
  u64 sum = 0;
  a.quads(warp * part + lane, min((warp + 1) * part, all), 32, [&](const float4& v, int i) {
    const bool k0 = stays(v.x, i), k1 = stays(v.y, i + 1), k2 = stays(v.z, i + 2),
               k3 = stays(v.w, i + 3);
    if (!(k0 || k1 || k2 || k3)) return;
    const u64 f0 = a.fixed(v.x), f1 = a.fixed(v.y), f2 = a.fixed(v.z), f3 = a.fixed(v.w);
    sum += ((k0 ? f0 : 0) + (k1 ? f1 : 0)) + ((k2 ? f2 : 0) + (k3 ? f3 : 0));
  });
  // Where segment w of the CTA starts.
  auto start_of = [&](int w) {
    return w == 0 ? 0 : w == kWarps ? len : a.head + 4 * min(w * part, all);
  };
  if (warp == 0 && lane < a.head) sum += weight(lane);
  const int after = a.head + 4 * all;
  if (warp == kWarps - 1 && lane < len - after) sum += weight(after + lane);
  sum = warp_sum(sum);
  __syncthreads();
  if (lane == 0) s.warp[warp] = sum;
  __syncthreads();
  u64 mine = 0;
  for (int w = 0; w < kWarps; ++w) mine += s.warp[w];
  a.share(s.amount, mine);
  u64 total = 0, before = 0;
#pragma unroll
  for (int r = 0; r < CL; ++r) {
    if (r < rank) before += s.amount[r];
    total += s.amount[r];
  }
  const u64 point = Sampler<CL>::point_of(u, total);
  if (before > point || before + mine <= point) return;
  // The whole CTA goes over the segment that holds the point.
  int seg = 0;
  while (before + s.warp[seg] <= point) before += s.warp[seg++];
  const int s0 = start_of(seg), s1 = start_of(seg + 1);
  const int each = (s1 - s0 + kThreads - 1) / kThreads;
  const int i0 = min(s0 + tid * each, s1), i1 = min(i0 + each, s1);
  mine = 0;
  for (int i = i0; i < i1; ++i) mine += weight(i);
  u64 run = before + a.block_scan(mine, &total);
  if (run > point || run + mine <= point) return;
  for (int i = i0; i < i1; ++i) {
    const u64 w = weight(i);
    if (w && run <= point && run + w > point) tokens[row] = begin + i;
    run += w;
  }
}

}  // namespace
}  // namespace tvp

using namespace tvp;

namespace {

template <int CL>
cudaError_t launch_sampler(int rows, int vocab, long long row_stride, const float* logits,
                           const float* uniforms, const float* temperature, const int32_t* top_k,
                           const float* top_p, const float* min_p, int32_t* tokens,
                           cudaStream_t stream) {
  auto slice_of = [](int v) { return CL > 1 ? ((v + CL - 1) / CL + 3) / 4 * 4 : v; };
  auto smem_of = [](int slice) { return kScratchBytes + (CL > 1 ? (size_t)slice * 4 : 0); };
  static bool configured[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    e = cudaFuncSetAttribute(sample_kernel<CL>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)smem_of(slice_of(TVP_SAMPLE_MAX_VOCAB)));
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  const int slice = slice_of(vocab);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)rows * CL);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem_of(slice);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CL;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, sample_kernel<CL>, logits, vocab, slice, row_stride, uniforms,
                            temperature, top_k, top_p, min_p, tokens);
}

}  // namespace

extern "C" int tvp_sample_tokens(const float* d_logits, int rows, int vocab, long long row_stride,
                                 const float* d_uniforms, const float* d_temperature,
                                 const int32_t* d_top_k, const float* d_top_p, const float* d_min_p,
                                 int32_t* d_tokens, tvp_stream_t stream) {
  if (!d_logits || !d_uniforms || !d_tokens || rows <= 0 || vocab <= 0 || row_stride < vocab ||
      (reinterpret_cast<uintptr_t>(d_logits) & 3u))
    return TVP_ERR_INVALID_ARGUMENT;
  if (vocab > TVP_SAMPLE_MAX_VOCAB || rows > 65535) return TVP_ERR_UNSUPPORTED;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e =
      rows < kStreamRows
          ? launch_sampler<kCluster>(rows, vocab, row_stride, d_logits, d_uniforms, d_temperature,
                                     d_top_k, d_top_p, d_min_p, d_tokens, st)
          : launch_sampler<1>(rows, vocab, row_stride, d_logits, d_uniforms, d_temperature, d_top_k,
                              d_top_p, d_min_p, d_tokens, st);
  return e == cudaSuccess ? TVP_OK : TVP_ERR_RUNTIME;
}
