// K6, and the rows' own part of K7: decode attention over a span of each row's
// pages, K2h's kernel (tvp_decode_heads.cu) with three changes.
//
//   * A row's pages are the visible ones only: its sink pages, then its window
//     (RowSpan), or what follows the shared prefix.  Hidden tokens of a page
//     that is read are masked in the scores and zeroed in the V tile.
//   * No plan launch: every CTA adds up the rows' pages itself, finds its range
//     of the T pages laid end to end and the row it starts in, and the walk
//     recomputes each row's span from its length.  One load of the lengths and a
//     block scan replace a launch per step, about 2.5 us, which is what a small
//     batch takes altogether.
//   * SHARED: a row's pieces are left as partials, which the merge kernel folds
//     together with the pieces of its group's prefix.  The CTA is half as large
//     (8 consumer warps, 4 stages), so that a CTA of the tile kernel shares the SM
//     with it: this kernel waits for HBM, that one for its exponentials.
//
// Bound by HBM: each visible token's K and V are read once (2 KiB for 8 heads).
// 256 rows of 512 to 8192 tokens, window 2048: 162 us for 997 MB, 6.15 TB/s of the
// 6.46 of a copy.  One row with a window of 256: 9.6 us, a chain of dependent reads.
// A row that is cut by ranges counts its pieces at the range it starts in: at
// most one row starts in a range and leaves it, so the counters' places do not
// depend on the batch, and a workspace serves any.
#include "tvp_span.cuh"
#include "tvp_ways.cuh"

namespace tvp {
namespace {

constexpr int kTailBarrier = 14;  // the 16 consumer warps, before the stages become merge scratch

// Shape and shared memory of a CTA.
template <int KVH, bool SHARED>
struct Shape {
  static constexpr int kSets = SHARED ? 1 : 2;  // of 8 consumer warps
  static constexpr int kStages = SHARED ? 4 : 6;
  static constexpr int kThreads = decode_threads<kSets, true>();
  // Registers: SHARED leaves the tile kernel's CTA its 30,720.
  static constexpr int kBlocks = SHARED ? 2 : 1;
  static constexpr int kConsumer = SHARED ? 96 : kConsumerRegs;
  static constexpr int kWays = kSets * kStageTiles / KVH;
  static constexpr size_t kBarsAt = (size_t)kStages * kStageBytes;
  static constexpr size_t kScratchAt = (kBarsAt + 2 * kStages * 8 + (kStages + 4) * 4 + 15) / 16 * 16;
  // senders of the widest merge level: kWays / 2 of each head
  static constexpr size_t kSetupAt = kScratchAt + (size_t)(kWays / 2 * KVH) * kStateFloats * 32 * 4;
  static constexpr size_t kSmem = kSetupAt + 256;
};

// Fold of one partial into this lane's (m, l, 8 channels) of a query head.
struct Fold {
  float m = -INFINITY, l = 0.f, o[8] = {};
  __device__ __forceinline__ void add(float pm, float pl, const float4& a, const float4& b) {
    const float M = fmaxf(m, pm);
    const float wa = m == -INFINITY ? 0.f : exp2f(m - M);
    const float wb = pm == -INFINITY ? 0.f : exp2f(pm - M);
    m = M;
    l = l * wa + pl * wb;
    o[0] = o[0] * wa + a.x * wb; o[1] = o[1] * wa + a.y * wb;
    o[2] = o[2] * wa + a.z * wb; o[3] = o[3] * wa + a.w * wb;
    o[4] = o[4] * wa + b.x * wb; o[5] = o[5] * wa + b.y * wb;
    o[6] = o[6] * wa + b.z * wb; o[7] = o[7] * wa + b.w * wb;
  }
  // n partials, the i-th at at(i), kFlight in flight at once, folded in order (256
  // rows behind 8192 tokens: 76.9 us with 8, 77.6 with 6, 80.4 with 4, 78.4 with 10).
  static constexpr int kFlight = 8;
  template <typename At>
  __device__ __forceinline__ void add_all(int n, At at, int lane) {
    const int h = lane >> 3, d = 2 * kGroup + h * kHeadDim + (lane & 7) * 8;
    for (int i = 0; i < n; i += kFlight) {
      float pm[kFlight], pl[kFlight];
      float4 a[kFlight], b[kFlight];
#pragma unroll
      for (int e = 0; e < kFlight; ++e) {
        if (i + e >= n) continue;
        const float* x = at(i + e);
        pm[e] = __ldcg(x + h);
        pl[e] = __ldcg(x + kGroup + h);
        a[e] = __ldcg(reinterpret_cast<const float4*>(x + d));
        b[e] = __ldcg(reinterpret_cast<const float4*>(x + d + 4));
      }
#pragma unroll
      for (int e = 0; e < kFlight; ++e)
        if (i + e < n) add(pm[e], pl[e], a[e], b[e]);
    }
  }
  __device__ __forceinline__ void write(__nv_bfloat16* out, int lane) const {
    const float inv = l > 0.f ? 1.f / l : 0.f;
    uint4 w;
    w.x = pack_bf16x2(o[0] * inv, o[1] * inv);
    w.y = pack_bf16x2(o[2] * inv, o[3] * inv);
    w.z = pack_bf16x2(o[4] * inv, o[5] * inv);
    w.w = pack_bf16x2(o[6] * inv, o[7] * inv);
    *reinterpret_cast<uint4*>(out + (lane >> 3) * kHeadDim + (lane & 7) * 8) = w;
  }
};

template <int KVH, bool SHARED>
__global__ void __launch_bounds__(Shape<KVH, SHARED>::kThreads, Shape<KVH, SHARED>::kBlocks)
    span_decode_kernel(const SpanParams p, const __grid_constant__ CUtensorMap k_map,
                       const __grid_constant__ CUtensorMap v_map) {
  using Cta = Shape<KVH, SHARED>;
  constexpr int kStages = Cta::kStages;
  constexpr int PS = kStageTiles / KVH;      // pages per stage
  constexpr int PERIOD = Cta::kSets * PS;    // pages between two pages of one way
  constexpr int kConsumers = Cta::kSets * kStageTiles;
  // 1 KiB alignment of the stage tiles (128-byte swizzle); checked, as in K2.
  extern __shared__ __align__(1024) unsigned char smem[];
  if (smem_addr(smem) & 1023u) {
    if (threadIdx.x == 0) record_error(p.err, TVP_DEVERR_SMEM_ALIGN);
    if (!SHARED) asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + Cta::kBarsAt);
  uint64_t* empty_bar = full_bar + kStages;
  int* stage_mask = reinterpret_cast<int*>(empty_bar + kStages);  // bit o: page o of the stage loaded
  volatile int* abort_flag = stage_mask + kStages;
  float* scratch = reinterpret_cast<float*>(smem + Cta::kScratchAt);
  int* warp_sums = reinterpret_cast<int*>(smem + Cta::kSetupAt);     // [warps]
  int* start = reinterpret_cast<int*>(smem + Cta::kSetupAt + 128);  // row and its first page

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // The tile kernel may start beside this one.
  if (SHARED) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (SHARED && !groups_usable(p)) {
    if (tid == 0 && blockIdx.x == 0) record_error(p.err, TVP_DEVERR_BAD_PLAN);
    return;
  }
  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(smem_addr(&full_bar[s]), 1);
      mbar_init(smem_addr(&empty_bar[s]), kStageTiles);  // one arrival per (page, head) tile
    }
    *abort_flag = 0;
    mbar_fence_init();
  }
  // The lengths may come from the kernel before.
  if (!SHARED) asm volatile("griddepcontrol.wait;" ::: "memory");
  // The rows' pages, added up by every CTA: thread t takes `each` rows from t * each.
  const int each = (p.batch + blockDim.x - 1) / blockDim.x;
  const int row0 = min(tid * each, p.batch), row1 = min(row0 + each, p.batch);
  int mine = 0;
  for (int s = row0; s < row1; ++s) mine += decode_span<SHARED>(p, s, blockIdx.x == 0).pages;
  int inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += y;
  }
  if (lane == 31) warp_sums[warp] = inc;
  __syncthreads();
  int before = inc - mine, total = 0;
  for (int w = 0; w < (int)blockDim.x / 32; ++w) {
    const int x = warp_sums[w];
    if (w < warp) before += x;
    total += x;
  }
  // Only min(grid, T) CTAs take pages: every range holds at least one.  Where the
  // grid has two ranges or more for each row, a whole number of them per row: rows
  // of one length, which windows make usual, are then cut at their own ends only,
  // and no CTA merges one row before it starts the next.  Their number is at most
  // twice the root of the row's pages, as a further piece costs its merge about a
  // quarter of what a further page costs the range.  One row of 251 pages 26.4 us
  // in 148 ranges, 14.4 in 32; 16 rows of 21 pages 17.8 -> 10.6; 64 of 23 pages
  // 15.4 -> 13.4; a single page pays 5.05 -> 5.35 for the rule.
  const long long T = total;
  long long C = T < (long long)gridDim.x ? T : (long long)gridDim.x;
  if (!SHARED && p.batch <= (int)gridDim.x / 2) {
    const int cuts = max(1, (int)(2.f * sqrtf((float)T / (float)p.batch) + 0.5f));
    C = min(C, (long long)(min((int)gridDim.x / p.batch, cuts) * p.batch));
  }
  const long long c = blockIdx.x;
  const int p_begin = c < C ? (int)(c * T / C) : 0;
  const int p_end = c < C ? (int)((c + 1) * T / C) : 0;
  const int n = p_end - p_begin;
  if (n > 0 && before <= p_begin && p_begin < before + mine) {
    int s = row0, first = before;
    for (;; ++s) {
      const int k = decode_span<SHARED>(p, s, false).pages;
      if (p_begin < first + k) break;
      first += k;
    }
    start[0] = s;
    start[1] = first;
  }
  __syncthreads();
  const uint32_t smem_base = smem_addr(smem);

  if (warp >= kConsumers) {
    // ------------------------------ producer ------------------------------
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kProducerRegs));
    if (warp != kConsumers) return;
    if (lane == 0) {
      prefetch_tensor_map(&k_map);
      prefetch_tensor_map(&v_map);
    }
    // Lane o < PS walks the range's pages o, o + PS, o + 2 PS, ... (row and its
    // span in registers, next page id loaded one stage ahead).
    int s = 0, first = 0, phys = 0;
    RowSpan span = {};
    int i = lane;
    auto walk = [&]() {
      const int pg = p_begin + i;
      while (pg >= first + span.pages) {
        first += span.pages;
        span = decode_span<SHARED>(p, ++s, false);
      }
      phys = __ldg(p.tables + (size_t)s * p.table_stride + span.logical(pg - first));
    };
    if (lane < PS && i < n) {
      s = start[0];
      first = start[1];
      span = decode_span<SHARED>(p, s, false);
      walk();
    }
    // The kernel before is done (the wait at the top; SHARED starts after it): what
    // it wrote to the pages is ordered before this warp's copies.
    if (!SHARED) asm volatile("fence.proxy.async.global;" ::: "memory");
    const int n_stages = (n + PS - 1) / PS;
    int stage = 0, issued = 0;
    uint32_t empty_parity = 1;
    for (int kk = 0; kk < n_stages; ++kk) {
      const int cur_phys = phys;
      const bool in_range = lane < PS && i < n;
      i += PS;
      if (lane < PS && i < n) walk();
      if (kk >= kStages) {
        int timed_out = 0;
        if (lane == 0) timed_out = !mbar_wait_bounded(smem_addr(&empty_bar[stage]), empty_parity);
        if (__shfl_sync(0xffffffffu, timed_out, 0)) {
          if (lane == 0) {
            *abort_flag = 1;
            record_error(p.err, TVP_DEVERR_TIMEOUT | TVP_DEVERR_WAIT_EMPTY);
          }
          break;
        }
      }
      const bool ok = in_range && cur_phys >= 0 && cur_phys < p.num_pages;
      if (in_range && !ok) record_error(p.err, TVP_DEVERR_BAD_PAGE);
      const uint32_t mask = __ballot_sync(0xffffffffu, ok);
      const uint32_t full = smem_addr(&full_bar[stage]);
      if (lane == 0) {
        stage_mask[stage] = (int)mask;
        mbar_arrive_expect_tx(full, (uint32_t)(__popc(mask) * KVH * 2 * kTileBytes));
      }
      __syncwarp();
      // lanes 0..PS-1: the K box of page o = lane, lanes PS..2PS-1: its V box
      // (as K2h: a 3-D page box for KVH > 1, the one-head box of the 2-D map for 1).
      const int o = lane % PS;
      const int tile_phys = __shfl_sync(0xffffffffu, cur_phys, o);
      if (lane < 2 * PS && ((mask >> o) & 1u)) {
        const bool is_v = lane >= PS;
        const uint32_t dst = smem_base + stage * kStageBytes +
                             (is_v ? kStageTiles * kTileBytes : 0) + o * KVH * kTileBytes;
        const int y = (int)(p.layer_row_base + (long long)tile_phys * kPage);
        if (KVH > 1)
          tma_load_3d(dst, is_v ? &v_map : &k_map, 0, y, 0, full);
        else
          tma_load_2d(dst, is_v ? &v_map : &k_map, 0, y, full);
      }
      issued = kk + 1;
      if (++stage == kStages) {
        stage = 0;
        empty_parity ^= 1u;
      }
    }
    drain_issued_stages<kStages>(full_bar, issued, lane, p.err);
    return;
  }

  // ------------------------------ consumers -------------------------------
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Cta::kConsumer));
  const int set = warp / kStageTiles;
  const int t = warp % kStageTiles;  // tile of the stage this warp reads
  const int o = t / KVH, h = t % KVH;
  const int way = set * PS + o;
  const TileLane tl(lane);
  const uint32_t k_off = t * kTileBytes, v_off = (kStageTiles + t) * kTileBytes;
  constexpr int kOutRow = KVH * kGroup * kHeadDim;
  auto out_of = [&](int s) { return p.out + (size_t)s * kOutRow + h * kGroup * kHeadDim; };

  int s = n > 0 ? start[0] : 0;
  int first = n > 0 ? start[1] : 0;
  RowSpan span = {};
  if (n > 0) span = decode_span<SHARED>(p, s, false);
  int pg = p_begin;
  int kbase = 0;  // range-local index of the piece's first page
  int c_kk = 0, c_stage = 0;
  uint32_t c_parity = 0;
  HeadState st;
  bool last_partial = false;  // the range ends inside a row that started earlier
  while (pg < p_end) {
    while (pg >= first + span.pages) {  // next row with pages
      first += span.pages;
      span = decode_span<SHARED>(p, ++s, false);
    }
    const int end = first + span.pages;
    const int piece_end = min(p_end, end);
    const int np = piece_end - pg;
    const bool complete = (pg == first) && (piece_end == end);

    uint32_t qb[4][2];
    load_q_frags(p.q + (size_t)s * kOutRow + h * kGroup * kHeadDim, tl, qb);
    st.reset();

    for (int i = kbase + ((way - kbase) % PERIOD + PERIOD) % PERIOD; i < kbase + np; i += PERIOD) {
      for (const int kk = i / PS; c_kk < kk; ++c_kk) {
        if (++c_stage == kStages) {
          c_stage = 0;
          c_parity ^= 1u;
        }
      }
      const int stage = c_stage;
      bool ready = false;
      if (!*abort_flag) ready = mbar_wait_bounded(smem_addr(&full_bar[stage]), c_parity);
      ready = __all_sync(0xffffffffu, ready);
      if (!ready && lane == 0 && !*abort_flag) {
        *abort_flag = 1;
        record_error(p.err, TVP_DEVERR_TIMEOUT | TVP_DEVERR_WAIT_FULL);
      }
      const bool have = ready && ((stage_mask[stage] >> o) & 1);
      uint32_t keep = 0xffffu;
      uint32_t kf[4][4], vf[4][4];
      if (have) {
        keep = span.keep(span.logical(pg - first + (i - kbase)));
        if (keep != 0xffffu) {
          zero_hidden_v_rows(smem + stage * kStageBytes + v_off, keep, lane);
          __syncwarp();
        }
        const uint32_t sb = smem_base + stage * kStageBytes;
        load_tile_frags(sb + k_off, sb + v_off, tl, kf, vf);
      }
      if (keep != 0xffffu) fence_proxy_async_smem();
      __syncwarp();
      // A stage is released only after its copies landed (a consumer that gave
      // up keeps it, so the producer cannot reuse a slot with a copy in flight).
      if (ready && lane == 0) mbar_arrive(smem_addr(&empty_bar[stage]));
      if (have)
        attend_tile_keep<true>(st, kf, vf, qb, keep != 0xffffu, (keep >> tl.tr) & 1u,
                               (keep >> (tl.tr + 8)) & 1u, p.scale_log2);
    }

    merge_ways<KVH, Cta::kWays>(st, scratch, way, h, lane);
    const int r0 = range_of_page(first, T, C), r1 = range_of_page(end - 1, T, C);
    if (SHARED) {
      if (way == 0) {
        reduce_l(st);
        // row + range: each next piece raises one of them
        write_partial(st, p.partials + ((size_t)(s + c) * KVH + h) * kPartialFloats, tl);
        if (pg == first && h == 0 && lane == 0) p.row_ranges[s] = make_int2(r0, r1);
      }
    } else {
      if (piece_end == p_end && !complete) {
        last_partial = true;  // published and merged below
        break;
      }
      if (way == 0) {
        reduce_l(st);
        if (complete)
          write_output(st, local_out(out_of(s)), tl);
        else if (publish_partial_at(
                     st, p.partials + ((size_t)partial_slot((int)c, first, T, C) * KVH + h) * kPartialFloats,
                     p.counters + r0 * kMaxKvHeads + h, r1 - r0 + 1, tl, lane))
          combine_partials<1>(p.partials, KVH, h, first, end, T, C, local_out(out_of(s)), lane);
      }
    }
    kbase += np;
    pg = piece_end;
  }
  if (SHARED) return;
  if (last_partial) {
    // The range's last piece ends inside a row that started earlier: once every
    // consumer warp has read its last tile the stages are free, and head h's
    // share of them holds the row's partials for the merge (K2h).
    named_barrier_sync(kTailBarrier, kConsumers * 32);
    if (way == 0) {
      reduce_l(st);
      const int end = first + span.pages;
      const int r0 = range_of_page(first, T, C);
      if (publish_partial_at(
              st, p.partials + ((size_t)partial_slot((int)c, first, T, C) * KVH + h) * kPartialFloats,
              p.counters + r0 * kMaxKvHeads + h, range_of_page(end - 1, T, C) - r0 + 1, tl, lane)) {
        constexpr int kShareBytes = kStages * kStageBytes / KVH;
        combine_partials_staged(p.partials, KVH, h, first, end, T, C, local_out(out_of(s)), lane,
                                reinterpret_cast<float*>(smem + (size_t)h * kShareBytes),
                                (kShareBytes - 512) / 1024);
      }
    }
  }
  // Rows without pages attend to nothing.
  if (way == 0) {
    for (int b = blockIdx.x; b < p.batch; b += gridDim.x)
      if (decode_span<SHARED>(p, b, false).pages == 0)
        *reinterpret_cast<uint4*>(out_of(b) + lane * 8) = make_uint4(0, 0, 0, 0);
  }
}

// The last step of K7: a warp per (row, KV head) folds the partials of the row's
// own pages and of its group's prefix, and writes the output; all of them read
// from L2, a few microseconds for any batch.  (Folded by the decode kernel's
// warps as they finished a row, the prefix pieces cost 2 to 3 us per row there,
// with the pipeline standing.)
constexpr int kMergeWarps = 4;  // of a block; 8: 256 rows 79.0 us instead of 78.0

template <int KVH>
__global__ void __launch_bounds__(kMergeWarps * 32) prefix_merge_kernel(const SpanParams p) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool in_order = groups_usable(p);
  const int at = blockIdx.x * kMergeWarps + warp, s = at / KVH, h = at % KVH;
  if (!in_order || s >= p.batch) {
    // Later work of the stream is behind the call's other launches through this wait.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }
  // What the call's inputs say, before the launches before this one are done.
  const RowSpan span = decode_span<true>(p, s, false);
  const int g = span.len > 0 ? group_of(p, s) : -1;
  const int t = g >= 0 ? s - __ldg(p.group_rows + g) : 0;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  Fold f;
  // The prefix's pieces, then the row's own; both counts in one round trip.
  const int2 in = g >= 0 ? __ldcg(p.group_pieces + g) : make_int2(0, 0);
  const int2 r = span.pages > 0 ? __ldcg(p.row_ranges + s) : make_int2(0, -1);
  const float* shared = p.pieces + ((size_t)(in.x + ((t / kTileRows) * KVH + h) * in.y) * kTileRows +
                                    t % kTileRows) * kPartialFloats;
  const float* own = p.partials + ((size_t)(s + r.x) * KVH + h) * kPartialFloats;
  f.add_all(in.y + r.y - r.x + 1,
            [&](int i) {
              return i < in.y ? shared + (size_t)i * kPieceFloats
                              : own + (size_t)(i - in.y) * KVH * kPartialFloats;
            },
            lane);
  f.write(p.out + ((size_t)s * KVH + h) * kGroup * kHeadDim, lane);
}

template <int KVH, bool SHARED>
cudaError_t launch(const SpanParams& p, const CUtensorMap& k_map, const CUtensorMap& v_map,
                   int num_ctas, cudaStream_t stream) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  static bool configured[64] = {};
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    // A register split that the launch's pool cannot satisfy would never return.
    cudaFuncAttributes fa;
    e = cudaFuncGetAttributes(&fa, span_decode_kernel<KVH, SHARED>);
    if (e != cudaSuccess) return e;
    constexpr int kThreads = Shape<KVH, SHARED>::kThreads;
    if (fa.numRegs * kThreads < 128 * kProducerRegs + (kThreads - 128) * Shape<KVH, SHARED>::kConsumer)
      return cudaErrorInvalidConfiguration;
    e = cudaFuncSetAttribute(span_decode_kernel<KVH, SHARED>,
                             cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)Shape<KVH, SHARED>::kSmem);
    // The tile kernel's CTAs find their shared memory beside this one's.
    if (e == cudaSuccess && SHARED)
      e = cudaFuncSetAttribute(span_decode_kernel<KVH, SHARED>,
                               cudaFuncAttributePreferredSharedMemoryCarveout,
                               cudaSharedmemCarveoutMaxShared);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)num_ctas);
  cfg.blockDim = dim3(Shape<KVH, SHARED>::kThreads);
  cfg.dynamicSmemBytes = Shape<KVH, SHARED>::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = SHARED ? 0 : 1;  // SHARED: the tile kernel beside it counts on a full wait here
  return cudaLaunchKernelEx(&cfg, span_decode_kernel<KVH, SHARED>, p, k_map, v_map);
}

template <bool SHARED>
cudaError_t launch_heads(const SpanParams& p, const CUtensorMap& k_map, const CUtensorMap& v_map,
                         int num_ctas, cudaStream_t stream) {
  switch (p.kv_heads) {
    case 1: return launch<1, SHARED>(p, k_map, v_map, num_ctas, stream);
    case 2: return launch<2, SHARED>(p, k_map, v_map, num_ctas, stream);
    case 4: return launch<4, SHARED>(p, k_map, v_map, num_ctas, stream);
    case 8: return launch<8, SHARED>(p, k_map, v_map, num_ctas, stream);
    default: return cudaErrorInvalidValue;
  }
}

template <int KVH>
cudaError_t launch_merge(const SpanParams& p, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(((long long)p.batch * KVH + kMergeWarps - 1) / kMergeWarps));
  cfg.blockDim = dim3(kMergeWarps * 32);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, prefix_merge_kernel<KVH>, p);
}

}  // namespace

cudaError_t launch_prefix_merge(const SpanParams& p, cudaStream_t stream) {
  switch (p.kv_heads) {
    case 1: return launch_merge<1>(p, stream);
    case 2: return launch_merge<2>(p, stream);
    case 4: return launch_merge<4>(p, stream);
    case 8: return launch_merge<8>(p, stream);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t launch_span_decode(const SpanParams& p, bool shared, long long pool_rows, int num_ctas,
                               cudaStream_t stream) {
  CUtensorMap k_map, v_map;
  const bool paged = p.kv_heads > 1;
  if (!(paged ? page_tensor_map(p.k_pool, pool_rows, p.kv_heads, &k_map)
              : pool_tensor_map(p.k_pool, pool_rows, p.kv_heads, &k_map)) ||
      !(paged ? page_tensor_map(p.v_pool, pool_rows, p.kv_heads, &v_map)
              : pool_tensor_map(p.v_pool, pool_rows, p.kv_heads, &v_map)))
    return cudaErrorInvalidValue;
  return shared ? launch_heads<true>(p, k_map, v_map, num_ctas, stream)
                : launch_heads<false>(p, k_map, v_map, num_ctas, stream);
}

}  // namespace tvp
