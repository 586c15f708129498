// The tcgen05 tile kernel of K8 (prefill with a sliding window and sinks) and
// of K7's shared prefixes: 32 query tokens of one KV head against a list of
// pages, 128 MMA rows 4 t + h, so every K/V byte serves 4 heads of 32 tokens.
//
//   * PREFIX: the 32 tokens are 32 rows of a group, the pages a part of its
//     prefix ("piece"); the CTA leaves (m, l, O) per (row, head) for the merge
//     kernel to fold in.  The pieces' length is the shortest that keeps their
//     number within piece_target (one CTA per SM, next to the decode kernel's: two
//     pieces per SM, one after the other, took 26.7 us instead of 18.2 for 8 rows
//     behind 8192 tokens, 78 instead of 75 for 256), so a few long prefixes and
//     many short ones both fill the GPU once; every CTA works this out from the
//     group sizes, a search of some ten steps by one warp, or, of more groups than
//     kWarpGroups, reads it from a plan.
//   * window: the tokens are a tile of a sequence's queries, the pages the ones
//     that some query of the tile sees; the CTA writes the output rows.
//
// Keys go in chunks of 4 pages (64 keys): warps 0 and 3 stream K and V boxes
// (TMA) into a ring, warp 1 issues S = Q K^T, warp 2 O += P V, two softmax sides
// of four warps (one thread per row) take the chunks in turn, each with its own
// P and O in Tensor Memory and its own running maximum and sum; they merge at
// the end.  Unlike K3's, scores stay FP32, and P is written to Tensor
// Memory (two BF16 per column) and is the MMA's A operand there: shared memory
// carries no P, whose write and reads took half of its bandwidth (per 64-key
// chunk and tile 16 KB written and 16 KB read, next to 24 KB for S, 8 KB for V
// and 16 KB from TMA).  P is BF16 as V is, since the two operands of an MMA have one
// type; its remainder as a second term would take 64 more columns, and two CTAs fill
// Tensor Memory already.  Outputs are off by 0.0019 to 0.0023 of their size (root mean
// square), 0.0017 of which is their own rounding.
// Bound by the exponentials: 8192 tokens with a window of 2048 take 182 us for 470
// million of them, 107 us of the special function unit's time.  A chunk takes a side
// 2790 cycles, of which the four sides of an SM keep that unit busy for 2048.
// A side takes a chunk's scores into registers at once, so one S of 64 columns
// serves both, and S(c + 2) is formed while chunk c is still in its
// exponentials.  (With an S per side that P overwrote, S(c + 2) had to wait for
// P V(c): a side idled 1000 of 3200 cycles per chunk.)  S(c + 1) follows when
// S(c) was read, P V(c) when P(c) was written; a side waits for P V(c - 2) before
// it rescales its O or writes P(c).
#include "tvp_span.cuh"
#include "tvp_tile.cuh"
#include "tvp_umma.cuh"

namespace tvp {
namespace {

constexpr int kRows = kTileRows * kGroup;          // 128 MMA rows
constexpr int kChunk = kChunkPages * kPage;        // 64 keys
constexpr int kStages = 4;
constexpr int kKvBytes = kChunkPages * kTileBytes;  // 8 KiB of K (or of V) per stage
constexpr int kChunkBytes = 2 * kKvBytes;
constexpr int kQBytes = kRows * 128;
constexpr int kThreads = 12 * 32;
// S: columns 0-63; P of side 0: 64-95, of side 1: 96-127; O: 128-191 and 192-255
constexpr uint32_t kTmemCols = 256;
constexpr uint32_t kColP = 64, kColO = 128;
constexpr int kLowRegs = 32;    // warps 0-3
constexpr int kHighRegs = 104;  // the softmax warps
constexpr unsigned kProducerNs = 200, kMmaNs = 40;  // sleeps of the waiting warps
// A piece of a prefix is no shorter than this: 4 rows behind 512 tokens take 12.2 us
// with 2 chunks, 12.8 with 4; one chunk each made 32 rows behind 1024 tokens 12% slower.
constexpr int kMinChunks = 2;

constexpr int kOffStages = kQBytes;
constexpr int kOffBars = kOffStages + kStages * kChunkBytes;
// q_full, o_full, drain[2], then by side: S formed, S read, P written, P V
// done; kv_full[stages], kv_empty[stages]
constexpr int kBarDrain = 2;
constexpr int kBarSFull = 4;
constexpr int kBarSRead = 6;
constexpr int kBarPFull = 8;
constexpr int kBarPvDone = 10;
constexpr int kBarKvFull = 12;
constexpr int kBarKvEmpty = kBarKvFull + kStages;
constexpr int kNumBars = kBarKvEmpty + kStages;
constexpr int kOffPlan = kOffBars + kNumBars * 8 + 16;
constexpr size_t kSmem = kOffPlan + 32;

struct Piece {
  int group, tile, head, first, last;  // pages [first, last) of the prefix
};

// Streams (tiles x KV heads) and chunks of group g; no streams without either.
__device__ __forceinline__ int2 group_work(const SpanParams& p, int g) {
  const int rows = __ldg(p.group_rows + g + 1) - __ldg(p.group_rows + g);
  const int pages = shared_pages(p, g, false);
  const int chunks = (pages + kChunkPages - 1) / kChunkPages;
  return make_int2(chunks > 0 ? (rows + kTileRows - 1) / kTileRows * p.kv_heads : 0, chunks);
}

// The shortest length of a piece, in chunks, whose pieces fit piece_target, between
// the even share and one piece per stream; count(n) is the number of pieces of n
// chunks.
template <typename Count>
__device__ __forceinline__ int piece_length(const SpanParams& p, long long streams, long long work,
                                            int most, Count count) {
  most = max(most, kMinChunks);
  if (streams >= p.piece_target) return most;
  const long long even = (work + p.piece_target - 1) / p.piece_target;
  int lo = (int)(even > kMinChunks ? even : kMinChunks), hi = max(most, lo);
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (count(mid) <= p.piece_target)
      hi = mid;
    else
      lo = mid + 1;
  }
  return lo;
}

// Piece `at` of group g, whose streams have `splits` pieces each.
__device__ __forceinline__ Piece piece_of(const SpanParams& p, int g, int chunks, int splits, int at) {
  const int stream = at / splits, j = at % splits;
  Piece out;
  out.group = g;
  out.tile = stream / p.kv_heads;
  out.head = stream % p.kv_heads;
  out.first = (int)((long long)chunks * j / splits) * kChunkPages;
  out.last = min(shared_pages(p, g, false), (int)((long long)chunks * (j + 1) / splits) * kChunkPages);
  return out;
}

// Piece `index` of the prefixes of up to kWarpGroups groups, by one warp; group < 0
// past the last.  The first block also leaves every group's first piece and count of
// pieces per stream for the merge kernel.
__device__ __forceinline__ Piece find_piece(const SpanParams& p, int index, int lane, bool publish) {
  auto sum = [](long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  };
  long long streams = 0, work = 0;
  int most = 1;
  for (int g = lane; g < p.groups; g += 32) {
    const int2 w = group_work(p, g);
    streams += w.x;
    work += (long long)w.x * w.y;
    if (w.x > 0) most = max(most, w.y);
  }
  streams = sum(streams);
  work = sum(work);
  most = __reduce_max_sync(0xffffffffu, most);
  const int length = piece_length(p, streams, work, most, [&](int n) {
    long long pieces = 0;
    for (int g = lane; g < p.groups; g += 32) {
      const int2 w = group_work(p, g);
      pieces += (long long)w.x * ((w.y + n - 1) / n);
    }
    return sum(pieces);
  });
  Piece out = {-1, 0, 0, 0, 0};
  int before = 0;
  for (int base = 0; base < p.groups; base += 32) {
    const int g = base + lane;
    const int2 w = g < p.groups ? group_work(p, g) : make_int2(0, 0);
    const int splits = (w.y + length - 1) / length;
    const int n = w.x * splits;
    int inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    const int first = before + inc - n;
    if (publish && g < p.groups) p.group_pieces[g] = make_int2(first, n > 0 ? splits : 0);
    const uint32_t who = __ballot_sync(0xffffffffu, index >= first && index < first + n);
    if (who) {
      const int src = __ffs(who) - 1;
      out = piece_of(p, base + src, __shfl_sync(0xffffffffu, w.y, src), __shfl_sync(0xffffffffu, splits, src),
                     index - __shfl_sync(0xffffffffu, first, src));
      if (!publish) return out;
    }
    before += __shfl_sync(0xffffffffu, inc, 31);
  }
  return out;
}

// The same for more groups, in two steps: one block works out every group's first
// piece, a launch before the others, and a CTA finds its group by bisection, so that
// the cost grows with the groups and not with their square.
constexpr int kPlanThreads = 1024;

__global__ void __launch_bounds__(kPlanThreads) prefix_plan_kernel(const SpanParams p) {
  __shared__ long long sums[kPlanThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // Sum over the block, in every thread; two barriers.
  auto sum = [&](long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane == 0) sums[warp] = v;
    __syncthreads();
    v = sums[lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    return v;
  };
  const bool in_order = groups_in_order(p);
  if (tid == 0) p.group_pieces[p.groups] = make_int2(in_order, 0);
  if (!in_order) return;  // the decode kernel reports it
  long long streams = 0, work = 0;
  int most = 1;
  for (int g = tid; g < p.groups; g += kPlanThreads) {
    shared_pages(p, g, true);
    const int2 w = group_work(p, g);
    streams += w.x;
    work += (long long)w.x * w.y;
    if (w.x > 0) most = max(most, w.y);
  }
  streams = sum(streams);
  work = sum(work);
  most = __reduce_max_sync(0xffffffffu, most);
  if (lane == 0) sums[warp] = most;
  __syncthreads();
  most = __reduce_max_sync(0xffffffffu, (int)sums[lane]);
  __syncthreads();
  const int length = piece_length(p, streams, work, most, [&](int n) {
    long long pieces = 0;
    for (int g = tid; g < p.groups; g += kPlanThreads) {
      const int2 w = group_work(p, g);
      pieces += (long long)w.x * ((w.y + n - 1) / n);
    }
    return sum(pieces);
  });
  int before = 0;
  for (int base = 0; base < p.groups; base += kPlanThreads) {
    const int g = base + tid;
    const int2 w = g < p.groups ? group_work(p, g) : make_int2(0, 0);
    const int splits = (w.y + length - 1) / length, n = w.x * splits;
    int inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    if (lane == 31) sums[warp] = inc;
    __syncthreads();
    int lower = 0, total = 0;
    for (int i = 0; i < kPlanThreads / 32; ++i) {
      if (i < warp) lower += (int)sums[i];
      total += (int)sums[i];
    }
    __syncthreads();
    if (g < p.groups) p.group_pieces[g] = make_int2(before + lower + inc - n, n > 0 ? splits : 0);
    before += total;
  }
}

// Piece `index` by the plan.
__device__ __forceinline__ Piece planned_piece(const SpanParams& p, int index) {
  int lo = 0, hi = p.groups;  // first piece of group lo <= index < that of group hi
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(&p.group_pieces[mid].x) <= index)
      lo = mid;
    else
      hi = mid;
  }
  const int2 in = __ldg(p.group_pieces + lo);
  const int2 w = group_work(p, lo);
  if (in.y == 0 || index - in.x >= w.x * in.y) return {-1, 0, 0, 0, 0};
  return piece_of(p, lo, w.y, in.y, index - in.x);
}

template <bool PREFIX>
__global__ void __launch_bounds__(kThreads, 2)
    span_tiles_kernel(const SpanParams p, const __grid_constant__ CUtensorMap k_map,
                      const __grid_constant__ CUtensorMap v_map) {
  // 128-byte swizzled tiles need 1 KiB alignment (checked, as in K3).
  extern __shared__ __align__(1024) unsigned char smem[];
  const uint32_t sbase = smem_addr(smem);
  if (sbase & 1023u) {
    if (threadIdx.x == 0) record_error(p.err, TVP_DEVERR_SMEM_ALIGN);
    if (PREFIX) asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int s, g, tok0, count, pos0 = 0, pos_last = 0;
  int v_begin, v_end;  // pages of the list that this CTA takes
  RowSpan span = {};   // window: from list to logical pages
  const int32_t* table;
  if (PREFIX) {
    // Launched beside the decode kernel (a programmatic dependent launch that
    // needs nothing of it).  The merge kernel waits for this grid alone, so its
    // last block, behind the ones that may have a piece, waits for the decode
    // kernel.
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (blockIdx.x == gridDim.x - 1) {
      asm volatile("griddepcontrol.wait;" ::: "memory");
      return;
    }
    if (!groups_usable(p)) return;  // the decode kernel reports it
    Piece* shared_piece = reinterpret_cast<Piece*>(smem + kOffPlan);
    if (warp == 0) {
      const bool publish = p.groups <= kWarpGroups && blockIdx.x == 0;
      const Piece mine = p.groups <= kWarpGroups ? find_piece(p, blockIdx.x, lane, publish)
                                                 : planned_piece(p, blockIdx.x);
      if (lane == 0) *shared_piece = mine;
      if (publish)
        for (int i = lane; i < p.groups; i += 32) shared_pages(p, i, true);
    }
    __syncthreads();
    const Piece piece = *shared_piece;
    if (piece.group < 0) return;
    s = piece.group;
    g = piece.head;
    const int r0 = __ldg(p.group_rows + s);
    tok0 = r0 + piece.tile * kTileRows;
    count = min(kTileRows, __ldg(p.group_rows + s + 1) - tok0);
    v_begin = piece.first;
    v_end = piece.last;
    table = p.prefix_tables + (size_t)s * p.prefix_stride;
  } else {
    s = blockIdx.x;
    g = blockIdx.y;
    const int q_begin = __ldg(p.cu_q + s), q_end = __ldg(p.cu_q + s + 1);
    const int tile = gridDim.z - 1 - blockIdx.z;  // the later tiles see the most keys
    tok0 = q_begin + tile * kTileRows;
    if (tok0 >= q_end) return;  // this sequence has fewer tiles
    count = min(kTileRows, q_end - tok0);
    const long long at0 = (long long)__ldg(p.q_pos0 + s) + tile * kTileRows;
    if (!positions_on_table(at0, count, p.table_stride)) {
      if (threadIdx.x == 0) record_error(p.err, TVP_DEVERR_BAD_TOKEN);
      return;
    }
    pos0 = (int)at0;  // position of the tile's token 0
    pos_last = pos0 + count - 1;
    span = window_span(pos_last + 1, (long long)pos0 + 1 - p.window, p.sinks);
    v_begin = 0;
    v_end = span.pages;
    table = p.tables + (size_t)s * p.table_stride;
  }
  const int n_chunks = (v_end - v_begin + kChunkPages - 1) / kChunkPages;

  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kOffBars);
  auto bar = [&](int i) { return smem_addr(&bars[i]); };
  const uint32_t q_full = bar(0), o_full = bar(1);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kNumBars);
  const int quarters = (count * kGroup + 31) / 32;  // row quarters with a real row
  if (threadIdx.x == 0) {
    mbar_init(q_full, 4);
    mbar_init(o_full, 1);
    mbar_init(bar(kBarDrain), 1);
    mbar_init(bar(kBarDrain + 1), 1);
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar(kBarSFull + b), 1);
      mbar_init(bar(kBarSRead + b), quarters);
      mbar_init(bar(kBarPFull + b), quarters);
      mbar_init(bar(kBarPvDone + b), 1);
    }
    for (int i = 0; i < kStages; ++i) {
      mbar_init(bar(kBarKvFull + i), 2);  // K and V
      mbar_init(bar(kBarKvEmpty + i), 1);
    }
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_addr(tmem_slot), kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  // Threads that meet before Tensor Memory is released: warps 1, 2 and both sides.
  constexpr int kEndThreads = 2 * 32 + 8 * 32;

  if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLowRegs));

  if (warp == 0 || warp == 3) {
    // ------------------------------ producers -----------------------------
    // Warp 0 streams K, warp 3 V: a box takes some 100 cycles to issue, and the
    // eight of a chunk by one warp took longer than its exponentials.
    const CUtensorMap* map = warp == 0 ? &k_map : &v_map;
    const uint32_t dst0 = sbase + kOffStages + (warp == 0 ? 0 : kKvBytes);
    if (lane == 0) prefetch_tensor_map(map);
    const int chunks = __shfl_sync(0xffffffffu, n_chunks, 0);
    const int x = __shfl_sync(0xffffffffu, g, 0) * kHeadDim;
    // lane i: the row of the pool that page slot i of a chunk starts at, -16 for a
    // slot past the last page or a bad id (a box wholly outside the pool arrives as
    // zeros); loaded one chunk ahead.
    auto page_row = [&](int c) {
      const int v = v_begin + c * kChunkPages + (lane & 3);
      if (v >= v_end) return -kPage;
      const int phys = __ldg(table + span.logical(v));
      if (phys >= 0 && phys < p.num_pages) return (int)(p.layer_row_base + (long long)phys * kPage);
      if (warp == 0 && lane < kChunkPages) record_error(p.err, TVP_DEVERR_BAD_PAGE);
      return -kPage;
    };
    int issued = 0, stage = 0, parity = 1;  // of the round before
    int next = page_row(0);
    for (int c = 0; c < chunks; ++c) {
      const int rows = next;
      if (c + 1 < chunks) next = page_row(c + 1);
      if (c >= kStages &&
          !__all_sync(0xffffffffu, mbar_wait_sleeping(bar(kBarKvEmpty + stage), parity, kProducerNs))) {
        if (lane == 0) record_error(p.err, TVP_DEVERR_TIMEOUT | TVP_DEVERR_WAIT_EMPTY);
        break;
      }
      int y[kChunkPages];
#pragma unroll
      for (int i = 0; i < kChunkPages; ++i) y[i] = __shfl_sync(0xffffffffu, rows, i);
      if (elect_one()) {
        const uint32_t full = bar(kBarKvFull + stage);
        mbar_arrive_expect_tx(full, kKvBytes);
#pragma unroll
        for (int i = 0; i < kChunkPages; ++i)
          tma_load_2d(dst0 + stage * kChunkBytes + i * kTileBytes, map, x, y[i], full);
      }
      __syncwarp();
      issued = c + 1;
      if (++stage == kStages) {
        stage = 0;
        parity ^= 1;
      }
    }
    drain_issued_stages<kStages>(bars + kBarKvFull, issued, lane, p.err);
    return;
  }

  if (warp <= 2) {
    // ----------------------------- MMA issuers ----------------------------
    // Warp 1 issues S(c), warp 2 P V(c): a wait takes some 300 cycles even where
    // nothing is to be waited for, and one warp after three of them per chunk held
    // every chunk up by 1550 cycles.  The whole warp waits and works out the
    // operands, one lane issues.
    constexpr uint32_t kIdS = umma_idesc_bf16_f32(kRows, kChunk, false, false);
    constexpr uint32_t kIdO = umma_idesc_bf16_f32(kRows, kHeadDim, false, true);
    const uint32_t cols = __shfl_sync(0xffffffffu, tmem, 0);
    const int chunks = __shfl_sync(0xffffffffu, n_chunks, 0);
    bool ok = true;
    auto wait = [&](uint32_t b, uint32_t parity) {
      if (ok && !__all_sync(0xffffffffu, mbar_wait_sleeping(b, parity, kMmaNs))) {
        if (lane == 0) record_error(p.err, TVP_DEVERR_TIMEOUT | TVP_DEVERR_WAIT_FULL);
        ok = false;
      }
      return ok;
    };
    int stage = 0;
    if (warp == 1) {
      // S(c) = Q K(c)^T for side c % 2, 16 channels per MMA, once S(c - 1) is in the
      // registers of its side.  Descriptors: a byte offset adds offset / 16.
      const uint64_t q_desc = umma_desc_sw128(sbase, 16, 1024);
      const uint64_t k_desc = umma_desc_sw128(sbase + kOffStages, 16, 1024);
      int parity = 0;
      wait(q_full, 0);
      for (int c = 0; ok && c < chunks; ++c) {
        if (!wait(bar(kBarKvFull + stage), parity)) break;
        if (c > 0 && !wait(bar(kBarSRead + ((c - 1) & 1)), ((c - 1) >> 1) & 1)) break;
        tc_fence_after_sync();
        const uint64_t k = k_desc + (uint32_t)(stage * (kChunkBytes >> 4));
        if (elect_one()) {
#pragma unroll
          for (int i = 0; i < kHeadDim / 16; ++i)
            umma_bf16(cols, q_desc + 2 * i, k + 2 * i, kIdS, i > 0);
          umma_commit(bar(kBarSFull + (c & 1)));
        }
        __syncwarp();
        if (++stage == kStages) {
          stage = 0;
          parity ^= 1;
        }
      }
    } else {
      // O_s += P(c) V(c) for c's side s, 16 keys (one page of V, 8 columns of P) per
      // MMA; the first chunk of each side overwrites O.  V(c) is there: P(c) comes
      // of S(c), which waited for the chunk.
      const uint64_t v_desc = umma_desc_sw128(sbase + kOffStages + kKvBytes, 0, 1024);
      for (int c = 0; ok && c < chunks; ++c) {
        const int side = c & 1;
        if (!wait(bar(kBarPFull + side), (c >> 1) & 1)) break;
        tc_fence_after_sync();
        const uint64_t v = v_desc + (uint32_t)(stage * (kChunkBytes >> 4));
        if (elect_one()) {
#pragma unroll
          for (int i = 0; i < kChunkPages; ++i)
            umma_bf16_ts(cols + kColO + 64 * side, cols + kColP + 32 * side + 8 * i,
                         v + (uint32_t)(i * (kTileBytes >> 4)), kIdO, (c >= 2 || i > 0));
          umma_commit(bar(kBarPvDone + side));
          umma_commit(bar(kBarKvEmpty + stage));
        }
        __syncwarp();
        if (++stage == kStages) stage = 0;
      }
      if (ok && elect_one()) umma_commit(o_full);
    }
    // Every MMA issued has completed before Tensor Memory is released.
    if (elect_one()) umma_commit(bar(kBarDrain + warp - 1));
    __syncwarp();
    if (!__all_sync(0xffffffffu, mbar_wait_bounded(bar(kBarDrain + warp - 1), 0)) && lane == 0)
      record_error(p.err, TVP_DEVERR_TIMEOUT | TVP_DEVERR_WAIT_DRAIN);
    __syncwarp();
    tc_fence_before_sync();
    named_barrier_sync(1, kEndThreads);
    if (warp == 1) {
      tc_fence_after_sync();
      tmem_dealloc(tmem, kTmemCols);
    }
    return;
  }

  // ------------------------------ softmax sides ----------------------------
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kHighRegs));
  const int side = (warp - 4) >> 2;  // 0: warps 4-7 (even chunks), 1: warps 8-11 (odd)
  const int quarter = warp & 3;      // TMEM lanes 32 quarter .. + 31
  const int row = quarter * 32 + lane;
  const int t = row >> 2, h = row & 3;
  const bool valid = t < count;
  const int qpos = pos0 + t;
  const int qdim = p.kv_heads * kGroup * kHeadDim;
  const int hq = g * kGroup + h;
  const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
  // The exponent's factor must be positive for the maximum of the scores to be
  // that of the products: a negative scale goes into q's sign, a zero one into q.
  const float c_log2 = p.scale_log2 == 0.f ? 1.f : fabsf(p.scale_log2);
  if (side == 0) {
    // Q row (token t, head hq) into the swizzled A tile of S = Q K^T.
    const uint4* src =
        reinterpret_cast<const uint4*>(p.q + (size_t)(tok0 + t) * qdim + hq * kHeadDim);
    const uint32_t flip = p.scale_log2 < 0.f ? 0x80008000u : 0u;
    const bool take = valid && p.scale_log2 != 0.f;
#pragma unroll
    for (int cc = 0; cc < 8; ++cc) {
      uint4 w = take ? __ldg(src + cc) : make_uint4(0, 0, 0, 0);
      w.x ^= flip; w.y ^= flip; w.z ^= flip; w.w ^= flip;
      *reinterpret_cast<uint4*>(smem + sw128_offset(row, cc)) = w;
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(q_full);
  }
  const bool active = quarter < quarters;
  float m = -INFINITY, l = 0.f;  // this side's running max (base-2 units) and normaliser
  bool ok = true;
  // The chunks that every row sees whole: those of pages [whole0, whole1), and
  // those before page sinks_whole.
  int whole0 = v_begin, whole1 = v_end, sinks_whole = 0;
  if (!PREFIX) {
    const long long low = (long long)pos_last + 1 - p.window;  // the last row sees from here on
    const int first = low > 0 ? (int)((low + kPage - 1) / kPage) : 0;  // its first whole page
    whole0 = max(span.head, first - span.skip);
    if (span.skip == 0) whole0 = first;
    whole1 = (pos0 + 1) / kPage - span.skip;
    sinks_whole = min(min(span.head, p.sinks / kPage), (pos0 + 1) / kPage);  // none in the future
  }
  // A wait of the whole warp; false when it ran out.
  auto warp_wait = [&](uint32_t b, uint32_t parity) {
    return __all_sync(0xffffffffu, mbar_wait_bounded(b, parity)) != 0;
  };
  uint32_t parity = 0;
  for (int c = side; active && c < n_chunks; c += 2) {
    ok = warp_wait(bar(kBarSFull + side), parity);
    if (!ok) break;
    tc_fence_after_sync();
    uint32_t sr[2][32];
    tmem_ld32(tmem + lane_base, sr[0]);
    tmem_ld32(tmem + 32 + lane_base, sr[1]);
    tmem_wait_ld();
    tc_fence_before_sync();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(kBarSRead + side));
    const int v0 = v_begin + c * kChunkPages;
    const bool whole = (v0 >= whole0 && v0 + kChunkPages <= whole1) ||
                       (!PREFIX && v0 + kChunkPages <= sinks_whole);
    if (!whole) {
#pragma unroll
      for (int i = 0; i < kChunkPages; ++i) {
        uint32_t keep = 0u;
        if (v0 + i < v_end) {
          keep = 0xffffu;
          if (!PREFIX) {
            const RowSpan mine = {0, 0, 0, qpos + 1, p.sinks, max(0, qpos + 1 - p.window)};
            keep = mine.keep(span.logical(v0 + i));
          }
        }
#pragma unroll
        for (int j = 0; j < kPage; ++j)
          if (!((keep >> j) & 1u)) sr[i >> 1][(i & 1) * kPage + j] = 0xff800000u;  // -inf
      }
    }
    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int j = 0; j < 32; j += 4) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        mx[e] = max3(mx[e], __uint_as_float(sr[0][j + e]), __uint_as_float(sr[1][j + e]));
    }
    const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c_log2;
    if (c >= 2) {  // P V(c - 2) is the last MMA into this side's O and out of its P
      ok = warp_wait(bar(kBarPvDone + side), parity ^ 1u);
      if (!ok) break;
      tc_fence_after_sync();
    }
    parity ^= 1u;
    // Lazy running max: rescale only when a score beats the side's max by more
    // than kLazyMargin (probabilities stay below 2^kLazyMargin).
    if (__any_sync(0xffffffffu, top > m + kLazyMargin)) {
      float alpha = 1.f;
      if (top > m + kLazyMargin) {
        alpha = m == -INFINITY ? 0.f : fast_exp2(m - top);
        m = top;
      }
      l *= alpha;
#pragma unroll 1
      for (int part = 0; c >= 2 && part < 4; ++part) {
        const uint32_t taddr = tmem + kColO + 64 * side + 16 * part + lane_base;
        uint32_t o[16];
        tmem_ld16(taddr, o);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
        tmem_st16(taddr, o);
      }
    }
    const float nbase = m == -INFINITY ? 0.f : -m;
    const uint64_t l2e2 = f2_pack(c_log2, c_log2), nb2 = f2_pack(nbase, nbase);
    uint64_t ls2[4];  // four independent paired sums
#pragma unroll
    for (int i = 0; i < 4; ++i) ls2[i] = f2_pack(0.f, 0.f);
    // P, two keys per column.
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint32_t w[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const uint64_t arg = f2_fma(f2_pack(__uint_as_float(sr[half][2 * j]),
                                            __uint_as_float(sr[half][2 * j + 1])),
                                    l2e2, nb2);
        float a0, a1;
        f2_unpack(arg, a0, a1);
        const float p0 = fast_exp2(a0), p1 = fast_exp2(a1);
        ls2[j & 3] = f2_add(ls2[j & 3], f2_pack(p0, p1));
        w[j] = pack_bf16x2(p0, p1);
      }
      tmem_st16(tmem + kColP + 32 * side + 16 * half + lane_base, w);
    }
    tmem_wait_st();
    float la, lb;
    f2_unpack(f2_add(f2_add(ls2[0], ls2[1]), f2_add(ls2[2], ls2[3])), la, lb);
    l += la + lb;
    // Tokens that no row of the tile sees may hold anything: zero them in the V
    // tile before P V reads it (P is 0 there, but 0 x NaN is not).
    if (!PREFIX && !whole && quarter == 0) {
      const RowSpan any = {0, 0, 0, pos_last + 1, p.sinks, max(0, pos0 + 1 - p.window)};
#pragma unroll
      for (int i = 0; i < kChunkPages; ++i) {
        if (v0 + i >= v_end) break;
        const uint32_t keep = any.keep(span.logical(v0 + i));
        if (keep != 0xffffu)
          zero_hidden_v_rows(smem + kOffStages + (c % kStages) * kChunkBytes + kKvBytes +
                                 i * kTileBytes, keep, lane);
      }
      fence_proxy_async_smem();
    }
    tc_fence_before_sync();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(kBarPFull + side));
  }
  const bool fin = active && ok && warp_wait(o_full, 0);
  if (active && !fin && lane == 0)
    record_error(p.err, TVP_DEVERR_TIMEOUT | TVP_DEVERR_WAIT_FULL);
  // Merge the two sides per row: side 1 hands its (max, normaliser) to side 0
  // through the Q tile, whose last reader (an S MMA) completed before o_full.
  float* xchg = reinterpret_cast<float*>(smem);
  if (side == 1 && fin) {
    xchg[2 * row] = m;
    xchg[2 * row + 1] = l;
  }
  named_barrier_sync(2, 8 * 32);
  if (side == 0 && fin) {
    const float mb = xchg[2 * row], lb = xchg[2 * row + 1];
    const float mt = fmaxf(m, mb);
    const float wa = m == -INFINITY ? 0.f : fast_exp2(m - mt);
    const float wb = mb == -INFINITY ? 0.f : fast_exp2(mb - mt);
    const float lt = l * wa + lb * wb;
    const float inv = PREFIX ? 1.f : lt > 0.f ? 1.f / lt : 0.f;
    const bool two = n_chunks > 1;  // side 1 wrote its accumulator
    float* part = PREFIX ? p.pieces + ((size_t)blockIdx.x * kTileRows + t) * kPartialFloats : nullptr;
    if (PREFIX && valid) {
      part[h] = mt;
      part[kGroup + h] = lt;
    }
    tc_fence_after_sync();
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint32_t oa[32], ob[32];
      tmem_ld32(tmem + kColO + 32 * half + lane_base, oa);
      if (two) tmem_ld32(tmem + kColO + 64 + 32 * half + lane_base, ob);
      tmem_wait_ld();
      if (!valid) continue;
      float x[32];
#pragma unroll
      for (int d = 0; d < 32; ++d) {
        x[d] = __uint_as_float(oa[d]) * wa;
        if (two) x[d] = fmaf(__uint_as_float(ob[d]), wb, x[d]);
      }
      if (PREFIX) {
        float4* dst = reinterpret_cast<float4*>(part + 2 * kGroup + h * kHeadDim + 32 * half);
#pragma unroll
        for (int d = 0; d < 8; ++d)
          dst[d] = make_float4(x[4 * d], x[4 * d + 1], x[4 * d + 2], x[4 * d + 3]);
      } else {
        uint4* dst = reinterpret_cast<uint4*>(p.out + (size_t)(tok0 + t) * qdim + hq * kHeadDim) +
                     4 * half;
#pragma unroll
        for (int cc = 0; cc < 4; ++cc)
          dst[cc] = make_uint4(pack_bf16x2(x[8 * cc] * inv, x[8 * cc + 1] * inv),
                               pack_bf16x2(x[8 * cc + 2] * inv, x[8 * cc + 3] * inv),
                               pack_bf16x2(x[8 * cc + 4] * inv, x[8 * cc + 5] * inv),
                               pack_bf16x2(x[8 * cc + 6] * inv, x[8 * cc + 7] * inv));
      }
    }
  }
  tc_fence_before_sync();
  named_barrier_sync(1, kEndThreads);
}

template <bool PREFIX>
cudaError_t launch_tiles(const SpanParams& p, long long pool_rows, dim3 grid, cudaStream_t stream) {
  static bool configured[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    // A register split that the launch's pool cannot satisfy would never return.
    cudaFuncAttributes fa;
    e = cudaFuncGetAttributes(&fa, span_tiles_kernel<PREFIX>);
    if (e != cudaSuccess) return e;
    if ((long long)fa.numRegs * kThreads < 128LL * kLowRegs + 256LL * kHighRegs)
      return cudaErrorInvalidConfiguration;
    e = cudaFuncSetAttribute(span_tiles_kernel<PREFIX>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)kSmem);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(span_tiles_kernel<PREFIX>,
                               cudaFuncAttributePreferredSharedMemoryCarveout,
                               cudaSharedmemCarveoutMaxShared);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  CUtensorMap k_map, v_map;
  if (!pool_tensor_map(p.k_pool, pool_rows, p.kv_heads, &k_map) ||
      !pool_tensor_map(p.v_pool, pool_rows, p.kv_heads, &v_map))
    return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = PREFIX ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, span_tiles_kernel<PREFIX>, p, k_map, v_map);
}

}  // namespace

cudaError_t launch_prefix_plan(const SpanParams& p, cudaStream_t stream) {
  prefix_plan_kernel<<<1, kPlanThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_prefix_tiles(const SpanParams& p, long long pool_rows, int max_pieces,
                                cudaStream_t stream) {
  return launch_tiles<true>(p, pool_rows, dim3((unsigned)max_pieces + 1), stream);
}

cudaError_t launch_window_tiles(const SpanParams& p, long long pool_rows, int max_q_len,
                                int num_seqs, cudaStream_t stream) {
  return launch_tiles<false>(
      p, pool_rows,
      dim3((unsigned)num_seqs, (unsigned)p.kv_heads, (unsigned)((max_q_len + kTileRows - 1) / kTileRows)),
      stream);
}

}  // namespace tvp
