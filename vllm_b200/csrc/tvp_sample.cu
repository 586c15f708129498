// K9 — one token per row of logits from given random numbers.
//
// A cluster of CTAs takes a row: 8 or 16 that keep the logits in shared memory
// while there are few rows, so that a row is read once from HBM however many passes
// the filters take, and 4 or 2 that read them again from L2 when there are many
// (kStreamRows).
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
// bins its part, CTA r adds up its share of the buckets of all of them through
// distributed shared memory.  When few enough logits lie at or above that bucket
// (a usual nucleus), CTA 0 gathers them, cuts and draws, all by comparing each
// with each.  Otherwise only the cut's own bucket is gathered (or, when it holds
// many, resolved by radix digits and a count of equal logits by index), and the
// draw goes by sums: per CTA, per 128 neighbouring logits, then by one warp over
// the 128 at the point.  For a small top-k the histogram is one of the largest
// logits of every 32, which costs no pass over the row.
//
// What bounds it, at rows of 128256 logits: one row 8.3 us without filters, 10.5
// with top-k 50, 22 with top-p 0.9 (launch, a chain of cluster barriers of about
// 0.5 us and reads of other CTAs' shared memory, and passes of one row over 16
// SMs; the 16-CTA form also spills 184 bytes a thread at its 64 registers);
// 256 rows without filters 69 us (131 MB: 1.9 TB/s; the weights' FP64
// arithmetic takes 50 of them), with top-k 50 45 us (2.9 TB/s: the first pass
// streams at the HBM rate, the chain behind it is the same as for one row), with
// top-p 0.9 200 us (a weight into a shared-memory histogram, two 32-bit atomics,
// for each logit with one).
#include <cfloat>
#include <climits>
#include <utility>

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
constexpr int kQuads = 8;  // fours of logits per batch of a thread
constexpr int kBlocks = kBuckets / 32;  // two per lane of a warp
// Few rows: 8 CTAs keep a row in shared memory.  From kStreamRows on, 4 CTAs per
// row read it again from L2 (kStreamMany: 2), which leaves room for more rows at
// once.  Measured, us for rows of 128256 of mixed settings, 8 kept / 4 / 2
// streaming: 32 rows 32 / 46 / 76, 64 rows 50 / 51 / 77, 96 rows 69 / 60 / 71,
// 256 rows 157 / 115 / 117; of top-k 50: 32 rows 14 / 14 / 17, 64 rows
// 27 / 16 / 17, 256 rows 105 / 65 / 47.
// Shorter rows (kShortVocab) are mostly barriers, and go to 2 CTAs from kStreamShort
// rows on.  Mixed settings / top-k 50, 4 CTAs against 2: of 8000 logits 64 rows
// 23.5 / 13.5 against 21.4 / 12.3, 96 rows 30.2 / 24.1 against 22.3 / 14.3, 191 rows
// 45.3 / 36.2 against 31.7 / 24.6; of 32000 80 rows 27.1 / 23.6 against 30.3 / 14.9, 96
// rows 31.7 / 25.1 against 32.6 / 14.9, 191 rows 49.3 / 37.4 against 35.4 / 26.2; of
// 50257 96 rows 33.8 / 27.4 against 45.2 / 16.7.
// A few rows of a large vocabulary: 16 CTAs.  One row, top-p 0.9, 8 CTAs / 16: of
// 300000 logits 51 / 37 us, of 128256 25 / 22, of 50257 20.5 / 20.2, of 1000
// 9.7 / 10.3 (a larger cluster's barriers take longer); 8 rows of 128256 27.9 / 27.4
// and without filters 8.7 / 12.0, as eight such clusters do not start at once.
constexpr int kWide = 16;
constexpr int kWideRows = 4;
constexpr int kWideVocab = 65536;
static_assert(kBlocks == 64 && kBuckets / kWide % 32 == 0, "border() deals them out so");
constexpr int kStreamRows = 64;
constexpr int kStreamMany = 192;
constexpr int kStreamShort = 96;
constexpr int kShortVocab = 32768;
constexpr int kList = 512;  // logits of a bucket that CTA 0 takes in
// Logits at or above the cut that CTA 0 finishes by itself, each compared with
// each by two threads or more per logit.  Top-k 200 that way: one row 14.4 us, 256
// rows 63; by the cut and sums 17.5 and 105.  Above 256 a logit has one thread, and
// 512 took 22 us.
constexpr int kFew = 256;
// The largest top-k that starts on this way: the list holds some more than k
// logits, and one that overflows costs 6 to 9 us.
constexpr int kFewK = 224;
constexpr int kFixedBits = 44;
// A distance (in units of T) where a weight rounds to 0: from 45 ln 2 = 31.2 on.
constexpr float kFar = 33.f;
constexpr double kTwo52 = 4503599627370496.0;

struct Cut {
  float value;  // kept: logits above it, or equal and of index <= last
  int last;
};

// The bin where a running amount reaches `want`, and the amount before it; bin
// kBuckets: it is not reached.
struct Border {
  int bin;
  u64 above, want;
};

template <int CL>
struct alignas(16) Shared {
  static constexpr int kSegment = kBuckets / CL;
  float most[CL], least[CL];  // by rank: largest and least logit
  int where[CL];              // by rank: the lowest index of the largest
  u64 amount[CL];  // by rank: a sum that the step at hand exchanges
  int fills[2][CL];  // in turn: one gather() may follow another at once
  u64 ties[CL];
  u64 seg[kSegment];  // this CTA's segment of the cluster's histogram
  u64 sub[kBlocks];                // every 32 buckets of the whole histogram
  u64 warp[kWarps];
  float warp_most[kWarps], warp_least[kWarps];
  double pow[256];
  Cut cut;
  Border border;
  int fill, hits;
  int part;  // where the draw's point lies, and the sum before
  u64 run;
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

constexpr size_t kScratchBytes = kBuckets * 8 + 5120;  // histogram, then the lists
static_assert(kScratchBytes >= 3 * kList * 8 + kList * 4, "the lists fit the histogram's place");
static_assert(kScratchBytes >= (TVP_SAMPLE_MAX_VOCAB / 128 + 3) * 8, "and so do the sums");

__host__ __device__ constexpr int batches_of(int logits) {
  return (logits / 4 + kQuads * kThreads - 1) / (kQuads * kThreads);
}

__device__ __forceinline__ uint32_t order_of(float x) {  // larger logit, larger image
  const uint32_t u = __float_as_uint(x + 0.f);  // -0 is +0
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

// Exclusive sum over the block's threads (all must call), and the total; `sums`:
// shared memory, one per warp.
__device__ u64 block_scan(u64* sums, u64 v, u64* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const u64 inc = warp_scan(v, lane);
  __syncthreads();
  if (lane == 31) sums[warp] = inc;
  __syncthreads();
  const u64 w = lane < kWarps ? sums[lane] : 0;
  const u64 winc = warp_scan(w, lane);
  *total = __shfl_sync(0xffffffffu, winc, 31);
  return __shfl_sync(0xffffffffu, winc - w, warp) + inc - v;
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

template <int CL, bool RES>
struct Sampler {
  Shared<CL>& s;
  const float* x;  // this CTA's logits: in shared memory (RES), or the row itself
  const float* maxima;  // of each thread's batches
  unsigned char* scratch;
  int rank, begin, len, head;  // logits before the first aligned four of x
  int tid, lane, warp;
  float top;    // finite
  float far;    // logits at and below it have no weight
  double c256;  // 256 log2(e) / T
  double reach_p;  // min-p keeps the logits up to this far below the top
  float scale;  // buckets per unit of distance
  float least;  // what the filters have left of the row: see kept()
  int last;
  int turn;

  // The CTAs of a row: barrier, and another one's shared memory.
  __device__ static void sync() { cg::this_cluster().sync(); }
  template <typename V>
  __device__ static V* of_rank(V* place, int r) {
    return cg::this_cluster().map_shared_rank(place, r);
  }

  // A thread's batch `it` is the kQuads quads of logits (it kQuads + e) kThreads +
  // tid after the head: a warp's quads of one e are 128 neighbouring logits.
  __device__ __forceinline__ int n_quads() const { return (len - head) / 4; }
  __device__ __forceinline__ int n_batches() const {
    return (n_quads() + kQuads * kThreads - 1) / (kQuads * kThreads);
  }
  // Quads e0 .. e0 + 3 of batch `it`, -inf past the last one.
  __device__ __forceinline__ void half_batch(int it, int e0, float4 (&v)[4]) const {
    const float4* x4 = reinterpret_cast<const float4*>(x + head);
    const int n4 = n_quads();
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int q = (it * kQuads + e0 + e) * kThreads + tid;
      v[e] = q < n4 ? x4[q] : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    }
  }
  // Index of the first logit of quad e of batch `it`.
  __device__ __forceinline__ int place(int it, int e) const {
    return head + 4 * ((it * kQuads + e) * kThreads + tid);
  }
  // Calls visit(four logits, index of the first) for the CTA's logits; batches
  // whose largest is below `floor` are left out.  The logits around the quads
  // come as fours with -inf.
  template <typename Visit>
  __device__ __forceinline__ void each_four(float floor, Visit visit) const {
    const int n = n_batches();
    for (int it = 0; it < n; ++it) {
      if (maxima[it * kThreads + tid] < floor) continue;
#pragma unroll 1  // the code of a pass is fetched once per row: it had better be short
      for (int e0 = 0; e0 < kQuads; e0 += 4) {
        float4 v[4];
        half_batch(it, e0, v);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (fmaxf(fmaxf(v[e].x, v[e].y), fmaxf(v[e].z, v[e].w)) >= floor)
            visit(v[e], place(it, e0 + e));
      }
    }
    const int i = single();
    if (i >= 0) visit(make_float4(x[i], -INFINITY, -INFINITY, -INFINITY), i);
  }
  // This thread's logit among the up to 6 before and after the quads, or -1.
  __device__ __forceinline__ int single() const {
    const int tail = (len - head) & 3;
    return tid < head ? tid : tid < head + tail ? len - tail + (tid - head) : -1;
  }
  // 2^52 + the weight of a logit in 2^-44 of the largest's: the sum's mantissa
  // holds the integer.  Without branches, so that the chains of several logits
  // overlap; a logit below `far`, a NaN among them, counts as `far`, which rounds
  // to 0.  (The passes that weigh every logit are bound by instruction issue:
  // 67 per 32 logits, with masks and selects, took 77 us for 256 rows of 128256.)
  __device__ __forceinline__ double weigh(float v) const {
    const double t = ((double)top - (double)fmaxf(v, far)) * c256;
    const double shifted = t + 6755399441055744.0;  // 1.5 * 2^52: rounds to an integer
    const int k = __double2loint(shifted);
    const double f = (shifted - 6755399441055744.0) - t;
    constexpr double kStep = 0.6931471805599453 / 256;  // ln 2 per 256th of an octave
    double y = fma(f, kStep * kStep * kStep / 6, kStep * kStep / 2);
    y = fma(y, f, kStep);
    y = fma(y, f, 1.0);
    const double p = s.pow[k & 255];  // * 2^(44 - k / 256)
    const double scaled = __hiloint2double(
        __double2hiint(p) + (kFixedBits << 20) - ((k & ~255) << 12), __double2loint(p));
    return fma(y, scaled, kTwo52);
  }
  __device__ __forceinline__ u64 fixed(float v) const {
    return (u64)__double_as_longlong(weigh(v)) & 0xfffffffffffffull;
  }
  // The sum of four, exact in FP64.
  __device__ __forceinline__ double weigh4(const float4& v) const {
    return ((weigh(v.x) - kTwo52) + (weigh(v.y) - kTwo52)) +
           ((weigh(v.z) - kTwo52) + (weigh(v.w) - kTwo52));
  }
  __device__ __forceinline__ int bucket(float v) const {  // rises as v falls
    return (int)fminf((top - v) * scale, (float)(kBuckets - 1));
  }
  // No kept logit is below `least`; of those equal to it the ones up to `last`.  A
  // NaN is not kept.
  __device__ __forceinline__ bool kept(float v, int i) const {
    return v > least || (v == least && i <= last);
  }

  __device__ u64 block_scan(u64 v, u64* total) { return tvp::block_scan(s.warp, v, total); }

  // Every CTA's value, to every CTA's `place[rank]`; a cluster barrier inside.
  // Between two calls with one place every CTA passes another cluster barrier
  // after its reads.
  template <typename V>
  __device__ void share(V* place, V v) {
    if (tid < CL) of_rank(place, tid)[rank] = v;
    sync();
  }

  static constexpr int kSegment = kBuckets / CL;

  // Histogram of the kept logits that `take` accepts, by `bin` (0 first in
  // falling order), and the bin where the running amount reaches want(total).
  // With MAXIMA: of the batches' largest logits, each counted once.
  template <bool MASS, bool MAXIMA, typename Take, typename Bin, typename Want>
  __device__ Border border(Take take, Bin bin, Want want_of) {
    u64* hist = reinterpret_cast<u64*>(scratch);
    uint32_t* counts = reinterpret_cast<uint32_t*>(scratch);
    for (int i = tid; i < kBuckets * (MASS ? 8 : 4) / 16; i += kThreads)
      reinterpret_cast<uint4*>(scratch)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    auto add = [&](float v, u64 w, int i) {
      if (!kept(v, begin + i) || !take(v)) return;
      if (MASS)
        shared_add(&hist[bin(v)], w);
      else
        atomicAdd(&counts[bin(v)], 1u);
    };
    if (MAXIMA) {
      const int n = n_batches();
      for (int it = 0; it < n; ++it) {
        const float v = maxima[it * kThreads + tid];
        if (v >= far) atomicAdd(&counts[bin(v)], 1u);
      }
      const int i = single();
      if (i >= 0) add(x[i], 0, i);
    } else {
      each_four(least, [&](const float4& v, int i) {
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
    }
    sync();
    // This CTA's segment over all, and the sum of each warp's 32 buckets to
    // every CTA.
    for (int i = tid; i < kSegment; i += kThreads) {
      const int b = rank * kSegment + i;
      u64 as[CL], a = 0;
#pragma unroll
      for (int r = 0; r < CL; ++r) as[r] = MASS ? of_rank(hist, r)[b] : of_rank(counts, r)[b];
#pragma unroll
      for (int r = 0; r < CL; ++r) a += as[r];
      s.seg[i] = a;
      a = warp_sum(a);
      if (lane < CL) of_rank(s.sub, lane)[b / 32] = a;
    }
    sync();
    // One warp finds the 32 buckets, then the bucket.
    if (warp == 0) find_border(want_of);
    __syncthreads();
    return s.border;
  }
  template <typename Want>
  __device__ __forceinline__ void find_border(Want want_of) {
    Border out;
    const u64 s0 = s.sub[2 * lane], s1 = s.sub[2 * lane + 1];
    const u64 inc = warp_scan(s0 + s1, lane);
    out.want = want_of(__shfl_sync(0xffffffffu, inc, 31));
    const u64 before = inc - s0 - s1;
    const uint32_t at = __ballot_sync(0xffffffffu, before < out.want && inc >= out.want);
    if (at == 0) {
      out.bin = kBuckets;
      out.above = 0;
      if (lane == 0) s.border = out;
      return;
    }
    const int src = __ffs(at) - 1;
    const bool second = before + s0 < out.want;
    const int block = 2 * src + __shfl_sync(0xffffffffu, (int)second, src);
    const u64 above = __shfl_sync(0xffffffffu, second ? before + s0 : before, src);
    constexpr int kPer = kSegment / 32;  // blocks of a CTA
    const u64 mine = of_rank(s.seg, block / kPer)[block % kPer * 32 + lane];
    const u64 upto = above + warp_scan(mine, lane);
    const int hit = __ffs(__ballot_sync(0xffffffffu, upto >= out.want)) - 1;
    out.bin = block * 32 + hit;
    out.above = __shfl_sync(0xffffffffu, upto - mine, hit);
    if (lane == 0) s.border = out;
  }

  // The kept logits in buckets b0 .. b1, as (order image, ~index), in CTA
  // 0's list, in no order; returns how many there are in the row, or, when more
  // than `most` (<= kList), some number above that and no list.
  __device__ u64* list() const { return reinterpret_cast<u64*>(scratch) + kList; }
  __device__ u64* weights() const { return reinterpret_cast<u64*>(scratch) + 2 * kList; }
  __device__ int gather(int b0, int b1, int most) {
    u64* mine = reinterpret_cast<u64*>(scratch);
    // A logit of bucket b1 lies above `floor`, one of b0 below `ceiling` (the distance
    // is rounded, by 2^-23 of it at most, and so are the product and the quotient).
    const float reach =
        b1 < kBuckets - 1 && scale > 0.f ? (float)(b1 + 1) / scale * 1.000001f : INFINITY;
    const float floor = fmaxf(least, top - reach);
    const float ceiling = b0 > 0 ? top - (float)b0 / scale * 0.999999f : INFINITY;
    int* hits = reinterpret_cast<int*>(weights() + kList);  // batches with a logit to list
    if (tid == 0) s.fill = s.hits = 0;
    __syncthreads();
    if (b0 == 0) {  // at least one logit for each batch whose largest lies there
      int n = 0;
      for (int it = 0; it < n_batches(); ++it) {
        const float m = maxima[it * kThreads + tid];
        const bool hit = bucket(m) <= b1 && m >= least;
        n += hit && m > least;
        const uint32_t all = __ballot_sync(0xffffffffu, hit);
        if (all == 0) continue;
        int at = 0;
        if (lane == 0) at = atomicAdd(&s.hits, __popc(all));
        at = __shfl_sync(0xffffffffu, at, 0) + __popc(all & ((1u << lane) - 1u));
        if (hit && at < kList) hits[at] = it * kThreads + tid;
      }
      n = __reduce_add_sync(0xffffffffu, n);
      if (lane == 0 && n > 0) atomicAdd(&s.fill, n);
      __syncthreads();
      n = s.fill;
      __syncthreads();
      if (n <= most && tid == 0) s.fill = 0;
      __syncthreads();
    }
    auto put = [&](float v, int i) {
      if (v < floor || v > ceiling || !kept(v, begin + i) || bucket(v) < b0 || bucket(v) > b1) return;
      // past `most` the count no longer matters
      if (*const_cast<volatile int*>(&s.fill) > most) return;
      const int to = atomicAdd(&s.fill, 1);
      if (to < most) mine[to] = ((u64)order_of(v) << 32) | (uint32_t)~(begin + i);
    };
    auto put4 = [&](const float4& v, int i) {
      put(v.x, i);
      put(v.y, i + 1);
      put(v.z, i + 2);
      put(v.w, i + 3);
    };
    if (*const_cast<volatile int*>(&s.fill) <= most) {
      if (b0 == 0 && s.hits <= kList) {
        // A few batches: a lane per quad, all of them at once.  (A warp that went
        // over its own batches waited for L2 once per half batch: of 256 rows of
        // top-k 50 each took 24 us, 17 this way.)
        static_assert(kQuads == 8, "a lane per quad");
        const float4* x4 = reinterpret_cast<const float4*>(x + head);
        for (int j = tid / kQuads; j < s.hits; j += kThreads / kQuads) {
          const int it = hits[j] / kThreads, owner = hits[j] % kThreads;
          const int q = (it * kQuads + tid % kQuads) * kThreads + owner;
          if (q < n_quads()) put4(x4[q], head + 4 * q);
        }
        const int i = single();
        if (i >= 0) put(x[i], i);
      } else {
        each_four(floor, put4);
      }
    }
    __syncthreads();
    int* fills = s.fills[turn ^= 1];
    share(fills, s.fill);
    int n = 0;
#pragma unroll
    for (int r = 0; r < CL; ++r) n += fills[r];
    if (rank == 0 && n <= most) {
      if (tid < n) {
        int r = 0, from = tid;
#pragma unroll
        for (int q = 0; q < CL - 1; ++q)
          if (r == q && from >= fills[q]) {
            from -= fills[q];
            ++r;
          }
        list()[tid] = of_rank(mine, r)[from];
      }
      __syncthreads();
    }
    return n;
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
  // P of their whole), min-p, draw u.
  __device__ void finish(int n, int k, u64 want, float P, float u, int32_t* token) {
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
    keep = keep && (ahead == 0 || mass < want) && !below(of_order((uint32_t)(me >> 32)));
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
  __device__ __forceinline__ bool below(float v) const {  // exp((v - top) / T) < min-p
    return (double)top - (double)v > reach_p;
  }

  // The cut in bucket `bkt`: among its logits gathered, or, for a bucket of
  // many, by radix digits of the order image and, among equal logits, by index.
  // `need`: the amount still wanted of that bucket.
  template <bool MASS>
  __device__ void cut_in_bucket(int bkt, u64 need) {
    const int in_n = gather(bkt, bkt, kList);
    if (in_n <= kList) {
      if (rank == 0) {
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
          const Cut c = {of_order((uint32_t)(me >> 32)), (int)~(uint32_t)me};
          for (int r = 0; r < CL; ++r) *of_rank(&s.cut, r) = c;
        }
      }
      sync();
      least = s.cut.value;
      last = s.cut.last;
      return;
    }
    uint32_t prefix = 0, mask = 0;
    u64 left = need;
    const int shifts[3] = {21, 10, 0}, bits[3] = {11, 11, 10};
    for (int d = 0; d < 3; ++d) {
      const uint32_t top_digit = (1u << bits[d]) - 1u;
      const Border part = border<MASS, false>(
          [&](float v) { return bucket(v) == bkt && (order_of(v) & mask) == prefix; },
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
    for (int i = i0; i < i1; ++i) ties += kept(x[i], begin + i) && order_of(x[i]) == prefix;
    const u64 before = block_scan(ties, &all);
    share(s.ties, all);
    u64 seen = before;
    for (int r = 0; r < rank; ++r) seen += s.ties[r];
    int nth_at = -1;
    if (seen < nth && seen + ties >= nth)
      for (int i = i0; i < i1; ++i)
        if (kept(x[i], begin + i) && order_of(x[i]) == prefix && ++seen == nth) nth_at = begin + i;
    if (nth_at >= 0)
      for (int r = 0; r < CL; ++r) *of_rank(&s.cut, r) = {of_order(prefix), nth_at};
    sync();
    least = s.cut.value;
    last = s.cut.last;
  }

  // CTA 0 draws from what gather() listed; the others wait, their lists are read.
  __device__ void finish_listed(int n, int k, u64 want, float P, float u,
                                int32_t* token) {
    if (rank == 0) finish(n, k, want, P, u, token);
    sync();
  }

  // One filter, by count (the k largest) or by weight (the share P): true when
  // it ended the row (the token is written).
  template <bool MASS>
  __device__ bool filter(int k, float P, float u, int32_t* token) {
    auto any = [](float) { return true; };
    auto bin = [&](float v) { return bucket(v); };
    auto want = [&](u64 total) { return MASS ? want_of(P, total) : (u64)k; };
    if (!MASS && k <= kFewK) {
      // The k-th largest of the batches' maxima is no larger than the k-th
      // largest logit: what lies above it holds the k, and little more.
      const Border edge = border<false, true>(any, bin, want);
      if (edge.bin < kBuckets) {
        const int n = gather(0, edge.bin, kFew);
        if (n <= kFew) {
          finish_listed(n, k, 0, P, u, token);
          return true;
        }
      }
    }
    const Border edge = border<MASS, false>(any, bin, want);
    if (edge.bin == kBuckets) return false;  // fewer logits with a weight than k
    if (MASS || k <= kFewK) {
      // After a histogram of weights the amount wanted is known, of the whole;
      // after one of counts, top-p is of the k that are left.
      const int n = gather(0, edge.bin, kFew);
      if (n <= kFew) {
        finish_listed(n, MASS ? 0 : k, MASS ? edge.want : 0, P, u, token);
        return true;
      }
    }
    cut_in_bucket<MASS>(edge.bin, edge.want - edge.above);
    return false;
  }
};

// The row that the turn-th cluster takes, where not all rows run at once: of
// every kThreads rows first those that a histogram of weights goes over, then
// those of a large top-k.  Such a row takes up to 78 us of its two CTAs, the others
// 25; in the rows' own order the last of them to start ended 256 mixed rows at
// 115 us.
__device__ int in_turn(int turn, int rows, int vocab, const float* temperature,
                       const int32_t* top_k, const float* top_p) {
  __shared__ int counts[kWarps];  // rows of the first kind, and of the second << 16
  __shared__ int found;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int base = turn / kThreads * kThreads, row = base + threadIdx.x;
  const bool real = row < rows;
  const float T = real && temperature ? __ldg(temperature + row) : 1.f;
  const float P = real && top_p ? __ldg(top_p + row) : 1.f;
  const int k = real && top_k ? __ldg(top_k + row) : 0;
  const bool all = k <= 0 || k >= vocab;
  const bool weighed = real && T > 0.f && all && P < 1.f;
  const bool counted = real && T > 0.f && !all && k > kFewK;
  const uint32_t b0 = __ballot_sync(0xffffffffu, weighed), b1 = __ballot_sync(0xffffffffu, counted);
  if (lane == 0) counts[warp] = __popc(b0) | __popc(b1) << 16;
  __syncthreads();
  const int upto = warp_scan(lane < kWarps ? counts[lane] : 0, lane);
  const int total = __shfl_sync(0xffffffffu, upto, 31);
  const int lower = warp > 0 ? __shfl_sync(0xffffffffu, upto, warp - 1) : 0;
  const uint32_t mask = (1u << lane) - 1u;
  const int before0 = (lower & 0xffff) + __popc(b0 & mask), before1 = (lower >> 16) + __popc(b1 & mask);
  const int all0 = total & 0xffff, all1 = total >> 16;
  const int place = weighed   ? before0
                    : counted ? all0 + before1
                              : all0 + all1 + (int)threadIdx.x - before0 - before1;
  if (place == turn - base) found = row;
  __syncthreads();
  return found;
}

template <int CL, bool RES>
__global__ void __launch_bounds__(kThreads, 2)
    sample_kernel(const float* __restrict__ logits, int vocab, int slice, long long row_stride,
                  const float* __restrict__ uniforms, const float* __restrict__ temperature,
                  const int32_t* __restrict__ top_k, const float* __restrict__ top_p,
                  const float* __restrict__ min_p, int32_t* __restrict__ tokens) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ Shared<CL> s;
  // Another CTA's shared memory may be written once that CTA is known to run: every
  // CTA says so here, and waits for the others before its first remote store, with
  // the first pass over the row in between.
  auto started = cg::this_cluster().barrier_arrive();
  const int rank = (int)cg::this_cluster().block_rank();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = RES ? blockIdx.x / CL
                      : in_turn(blockIdx.x / CL, gridDim.x / CL, vocab, temperature, top_k, top_p);
  const int begin = min(rank * slice, vocab), len = min(slice, vocab - begin);
  const float* src = logits + (size_t)row * row_stride + begin;
  // Logits before the first 16-byte boundary.
  const int head = min((int)((0u - (uint32_t)(reinterpret_cast<uintptr_t>(src) >> 2)) & 3u), len);
  const int n4 = (len - head) / 4;
  const int batches = (n4 + kQuads * kThreads - 1) / (kQuads * kThreads);
  float* maxima = reinterpret_cast<float*>(smem + kScratchBytes);
  // RES: the copy's quads lie on 16 bytes as the row's do.
  float* x = maxima + batches_of(slice) * kThreads + ((4 - head) & 3);

  // The row's largest and least logit, and every batch's largest; with RES the
  // CTA's logits also go into shared memory.
  float top = -INFINITY, lo = INFINITY;
  for (int it = 0; it < batches; ++it) {
    const int base = it * kQuads * kThreads + tid;
    float most = -INFINITY;
    float4 v[kQuads];
#pragma unroll
    for (int e = 0; e < kQuads; ++e)
      if (base + e * kThreads < n4)
        v[e] = __ldg(reinterpret_cast<const float4*>(src + head) + base + e * kThreads);
#pragma unroll
    for (int e = 0; e < kQuads; ++e) {
      if (base + e * kThreads >= n4) break;
      const float4 c = v[e];  // a NaN loses every comparison
      most = max3(max3(most, c.x, c.y), c.z, c.w);
      lo = fminf(lo, fminf(fminf(c.x, c.y), fminf(c.z, c.w)));
      if (RES) *reinterpret_cast<float4*>(x + head + 4 * (base + e * kThreads)) = c;
    }
    maxima[it * kThreads + tid] = most;
    top = fmaxf(top, most);
  }
  const int tail = len - head - 4 * n4;
  if (tid < head + tail) {
    const int i = tid < head ? tid : len - tail + (tid - head);
    const float c = src[i];
    top = fmaxf(top, c);
    lo = fminf(lo, c);
    if (RES) x[i] = c;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
  }
  if (lane == 0) {
    s.warp_most[warp] = top;
    s.warp_least[warp] = lo;
  }
  if (tid < 256) s.pow[tid] = g_powers.d[tid];
  float T = temperature ? temperature[row] : 1.f;
  const int k = top_k ? top_k[row] : 0;
  const float P = top_p ? top_p[row] : 1.f;
  const float mp = min_p ? min_p[row] : 0.f;
  const float M = mp > 0.f ? fminf(mp, 1.f) : 0.f;
  const float u = uniforms[row];
  __syncthreads();
  for (int w = 0; w < kWarps; ++w) {
    top = fmaxf(top, s.warp_most[w]);
    lo = fminf(lo, s.warp_least[w]);
  }
  cg::this_cluster().barrier_wait(std::move(started));
  if (tid < CL) {
    Sampler<CL, RES>::of_rank(s.most, tid)[rank] = top;
    Sampler<CL, RES>::of_rank(s.least, tid)[rank] = lo;
  }
  Sampler<CL, RES>::sync();
#pragma unroll
  for (int r = 0; r < CL; ++r) {
    top = fmaxf(top, s.most[r]);
    lo = fminf(lo, s.least[r]);
  }
  if (top == -INFINITY) {
    if (rank == 0 && tid == 0) tokens[row] = -1;
    return;
  }
  if (!(T > 0.f)) {  // the lowest index of the largest
    int first = INT_MAX;
    auto look = [&](float v, int i) {
      if (v == top) first = min(first, begin + i);
    };
    const float* from = RES ? x : src;
    for (int it = 0; it < batches; ++it)
      if (maxima[it * kThreads + tid] == top)
        for (int e = 0; e < kQuads; ++e) {
          const int q = (it * kQuads + e) * kThreads + tid;
          for (int j = 0; q < n4 && j < 4; ++j) look(from[head + 4 * q + j], head + 4 * q + j);
        }
    if (tid < head + tail) {
      const int i = tid < head ? tid : len - tail + (tid - head);
      look(from[i], i);
    }
    if (tid == 0) s.fill = INT_MAX;
    __syncthreads();
    first = __reduce_min_sync(0xffffffffu, first);
    if (lane == 0) atomicMin(&s.fill, first);
    __syncthreads();
    if (tid < CL) Sampler<CL, RES>::of_rank(s.where, tid)[rank] = s.fill;
    Sampler<CL, RES>::sync();
    if (rank == 0 && tid == 0) {
      for (int r = 0; r < CL; ++r) first = min(first, s.where[r]);
      tokens[row] = first;
    }
    return;
  }
  if (top == INFINITY) {
    // These alone have weight, the same each: the filters leave the first n of
    // them, and the draw takes one of these by its place.
    const int each = (len + kThreads - 1) / kThreads;
    const int i0 = min(tid * each, len), i1 = min(i0 + each, len);
    const float* from = RES ? x : src;
    u64 count = 0, all;
    for (int i = i0; i < i1; ++i) count += from[i] == INFINITY;
    u64 seen = block_scan(s.warp, count, &all);
    if (tid < CL) Sampler<CL, RES>::of_rank(s.amount, tid)[rank] = all;
    Sampler<CL, RES>::sync();
    u64 n = 0;
    for (int r = 0; r < CL; ++r) {
      if (r < rank) seen += s.amount[r];
      n += s.amount[r];
    }
    if (k > 0) n = min(n, (u64)k);
    if (P < 1.f) n = Sampler<CL, RES>::want_of(P, n);
    const u64 place = Sampler<CL, RES>::point_of(u, n);
    for (int i = i0; i < i1; ++i)
      if (from[i] == INFINITY && seen++ == place) tokens[row] = begin + i;
    return;
  }
  // A temperature below a 512th of the top's last place gives every other logit
  // weight 0 as that 512th does, and keeps the distances' exponents in range.
  const float under = nextafterf(top, -INFINITY);
  T = fmaxf(T, (top - under) * (1.f / 512.f));
  // Rounded away from the top: to the nearest, a T of 0.045 of the top's last place left
  // `far` 22 T below it, where a weight is 3929 of 2^-44.
  const float far = fmaxf(fminf(__fsub_rd(top, __fmul_ru(kFar, T)), under), -FLT_MAX);
  // Buckets over the distances that have weight, or over the row's own range
  // where that is narrower (and not a masked row's, whose least is -inf).  Finite, so
  // that the buckets of far logits have an end in every case.
  const float range = fminf(fminf(kFar * T, top - lo), FLT_MAX);
  Sampler<CL, RES> a = {s, RES ? x : src, maxima, smem, rank, begin, len, head, tid, lane, warp,
                   top, far, 369.3299304675746 / (double)T,
               M > 0.f && T < INFINITY ? -log((double)M) * (double)T : (double)INFINITY,
                   range > 0.f ? fminf((float)kBuckets / range, FLT_MAX) : 0.f, far, INT_MAX, 0};
  if (k > 0 && k < vocab && a.template filter<false>(k, P, u, tokens + row)) return;
  if (P < 1.f && a.template filter<true>(k, P, u, tokens + row)) return;
  // The draw by sums, of every 128 neighbouring logits first.
  auto stays = [&](float v, int i) {
    return a.kept(v, begin + i) && (M == 0.f || !a.below(v));
  };
  // Nothing cut, and no weight at `far`: every logit goes into the sum as it is.
  const bool simple = a.least == far && M == 0.f && far > -FLT_MAX;
  auto weight = [&](int i) -> u64 {
    const float v = a.x[i];
    return stays(v, i) ? a.fixed(v) : 0;
  };
  // sums[0]: the logits before the quads; then one for each 32 quads; last: the
  // logits after them.
  u64* sums = reinterpret_cast<u64*>(smem);
  const int parts = (a.n_quads() + 31) / 32 + 2;
  // (min-p's distance with room for the roundings, which are large among subnormals)
  const float least =
      fmaxf(a.least, __fsub_rd(top, __fmul_ru(__double2float_ru(a.reach_p), 1.00001f)));
  for (int it = 0; it < a.n_batches(); ++it) {
    const bool active = maxima[it * kThreads + tid] >= least;  // -inf past the last quad
    const int first = 1 + it * kQuads * kWarps + warp;
    if (!__any_sync(0xffffffffu, active)) {
      if (lane < kQuads && first + lane * kWarps < parts - 1) sums[first + lane * kWarps] = 0;
      continue;
    }
#pragma unroll 1
    for (int e0 = 0; e0 < kQuads; e0 += 4) {
      float4 v[4];
      double w[4];
      if (simple) {
        a.half_batch(it, e0, v);
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = a.weigh4(v[e]);
      } else {
        a.half_batch(it, e0, v);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = a.place(it, e0 + e);
          const bool k0 = stays(v[e].x, i), k1 = stays(v[e].y, i + 1), k2 = stays(v[e].z, i + 2),
                     k3 = stays(v[e].w, i + 3);
          w[e] = 0.0;
          if (__any_sync(0xffffffffu, k0 || k1 || k2 || k3))
            w[e] = ((k0 ? a.weigh(v[e].x) - kTwo52 : 0.0) + (k1 ? a.weigh(v[e].y) - kTwo52 : 0.0)) +
                   ((k2 ? a.weigh(v[e].z) - kTwo52 : 0.0) + (k3 ? a.weigh(v[e].w) - kTwo52 : 0.0));
        }
      }
      // The warp's four sums (of 128 weights, exact in FP64) at once: lanes of bit
      // 4 take over two of them, lanes of bit 3 one of these; e is then (bit 4,
      // bit 3).
      const bool b4 = lane & 16, b3 = lane & 8;
      const double x0 = (b4 ? w[2] : w[0]) + __shfl_xor_sync(0xffffffffu, b4 ? w[0] : w[2], 16);
      const double x1 = (b4 ? w[3] : w[1]) + __shfl_xor_sync(0xffffffffu, b4 ? w[1] : w[3], 16);
      double y = (b3 ? x1 : x0) + __shfl_xor_sync(0xffffffffu, b3 ? x0 : x1, 8);
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
      const int to = first + (e0 + (lane >> 3)) * kWarps;
      if ((lane & 7) == 0 && to < parts - 1) sums[to] = (u64)(long long)y;
    }
  }
  if (tid < 2) {
    u64 w = 0;
    for (int i = tid ? a.head + 4 * a.n_quads() : 0; i < (tid ? len : a.head); ++i) w += weight(i);
    sums[tid ? parts - 1 : 0] = w;
  }
  __syncthreads();
  const int each = (parts + kThreads - 1) / kThreads;
  const int p0 = min(tid * each, parts), p1 = min(p0 + each, parts);
  u64 mine = 0, all;
  for (int p = p0; p < p1; ++p) mine += sums[p];
  u64 run = a.block_scan(mine, &all);
  a.share(s.amount, all);
  u64 total = 0, before = 0;
#pragma unroll
  for (int r = 0; r < CL; ++r) {
    if (r < rank) before += s.amount[r];
    total += s.amount[r];
  }
  const u64 point = Sampler<CL, RES>::point_of(u, total);
  run += before;
  if (run <= point && run + mine > point) {
    int p = p0;
    while (run + sums[p] <= point) run += sums[p++];
    s.part = p;
    s.run = run;
  }
  if (before > point || before + all <= point) return;
  __syncthreads();
  if (warp != 0) return;
  // One warp goes over the 128 logits (or the few around the quads) at the point.
  run = s.run;
  const int at = s.part, end = a.head + 4 * a.n_quads();
  const int i0 = at == 0 ? 0 : at == parts - 1 ? end : a.head + 128 * (at - 1);
  const int i1 = at == 0 ? a.head : at == parts - 1 ? len : min(i0 + 128, end);
  u64 w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int i = i0 + 4 * lane + e;
    w[e] = i < i1 ? weight(i) : 0;
  }
  mine = (w[0] + w[1]) + (w[2] + w[3]);
  run += warp_scan(mine, lane) - mine;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (w[e] && run <= point && run + w[e] > point) tokens[row] = begin + i0 + 4 * lane + e;
    run += w[e];
  }
}

}  // namespace
}  // namespace tvp

using namespace tvp;

namespace {

template <int CL, bool RES>
cudaError_t launch_sampler(int rows, int vocab, long long row_stride, const float* logits,
                           const float* uniforms, const float* temperature, const int32_t* top_k,
                           const float* top_p, const float* min_p, int32_t* tokens,
                           cudaStream_t stream) {
  auto slice_of = [](int v) { return ((v + CL - 1) / CL + 3) / 4 * 4; };
  auto smem_of = [](int slice) {
    return kScratchBytes + (size_t)batches_of(slice) * kThreads * 4 + (RES ? (size_t)slice * 4 + 16 : 0);
  };
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
  static bool configured[64] = {}, unfit[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    const size_t most = smem_of(slice_of(TVP_SAMPLE_MAX_VOCAB));
    e = cudaFuncSetAttribute(sample_kernel<CL, RES>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)most);
    if (e != cudaSuccess) return e;
    if (CL > kCluster) {  // more than every device takes: only where one has room
      e = cudaFuncSetAttribute(sample_kernel<CL, RES>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
      if (e != cudaSuccess) return e;
      cudaLaunchConfig_t largest = cfg;
      largest.gridDim = dim3(CL);
      largest.dynamicSmemBytes = most;
      int clusters = 0;
      e = cudaOccupancyMaxActiveClusters(&clusters, sample_kernel<CL, RES>, &largest);
      if (e != cudaSuccess) return e;
      if (clusters < 1 && (dev < 0 || dev >= 64)) return cudaErrorNotSupported;
      if (clusters < 1) unfit[dev] = true;
    }
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  if (dev >= 0 && dev < 64 && unfit[dev]) return cudaErrorNotSupported;
  return cudaLaunchKernelEx(&cfg, sample_kernel<CL, RES>, logits, vocab, slice, row_stride, uniforms,
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
  auto run = [&](auto launch) {
    return launch(rows, vocab, row_stride, d_logits, d_uniforms, d_temperature, d_top_k, d_top_p,
                  d_min_p, d_tokens, st);
  };
  cudaError_t e = cudaErrorNotSupported;
  if (rows <= kWideRows && vocab >= kWideVocab) e = run(launch_sampler<kWide, true>);
  if (e == cudaErrorNotSupported)
    e = run(rows < kStreamRows ? launch_sampler<kCluster, true>
            : rows < (vocab > kShortVocab ? kStreamMany : kStreamShort)
                ? launch_sampler<4, false>
                : launch_sampler<2, false>);
  return e == cudaSuccess ? TVP_OK : TVP_ERR_RUNTIME;
}
