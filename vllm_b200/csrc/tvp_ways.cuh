// Merging the online-softmax states of the consumer warps ("ways") that share
// a KV head: KVH heads on 16 consumer warps leave W = 16 / KVH ways per head
// (on 8 warps, 8 / KVH), each over pages of its own.
#pragma once

#include "tvp_tile.cuh"

namespace tvp {

constexpr int kStateFloats = 20;  // m0, m1, l0, l1, acc[16] per lane
constexpr int kMergeSlots = 8;    // senders of the widest merge level (W / 2 x KVH)

// Online-softmax state of two ways over disjoint pages, merged into `a`; the
// other way's state is read field by field from its slot (field f at f * 32).
__device__ __forceinline__ void merge_state(HeadState& a, const float* b) {
  const float mb0 = b[0 * 32], mb1 = b[1 * 32];
  const float M0 = fmaxf(a.m0, mb0), M1 = fmaxf(a.m1, mb1);
  const float wa0 = a.m0 == -INFINITY ? 0.f : exp2f(a.m0 - M0);
  const float wa1 = a.m1 == -INFINITY ? 0.f : exp2f(a.m1 - M1);
  const float wb0 = mb0 == -INFINITY ? 0.f : exp2f(mb0 - M0);
  const float wb1 = mb1 == -INFINITY ? 0.f : exp2f(mb1 - M1);
  a.m0 = M0;
  a.m1 = M1;
  a.l0 = a.l0 * wa0 + b[2 * 32] * wb0;
  a.l1 = a.l1 * wa1 + b[3 * 32] * wb1;
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    a.acc[d][0] = a.acc[d][0] * wa0 + b[(4 + 4 * d + 0) * 32] * wb0;  // columns 2hc
    a.acc[d][1] = a.acc[d][1] * wa1 + b[(4 + 4 * d + 1) * 32] * wb1;  // columns 2hc + 1
    a.acc[d][2] = a.acc[d][2] * wa0 + b[(4 + 4 * d + 2) * 32] * wb0;
    a.acc[d][3] = a.acc[d][3] * wa1 + b[(4 + 4 * d + 3) * 32] * wb1;
  }
}

// Tree merge of the W ways of KV head h into way 0.  Slots are [field][lane]
// so that a warp's stores and loads are conflict-free.  Barrier ids: 1 + h for
// the levels (participants: the ways still in the tree), 1 + KVH + h for the
// entry, which all W ways pass, so that no way of the next piece writes a slot
// that way 0 is still reading.  With two ways the one level has the
// entry's participants, and both use 1 + h.
template <int KVH, int W = 16 / KVH>
__device__ __forceinline__ void merge_ways(HeadState& st, float* scratch, int way, int h,
                                           int lane) {
  if (W == 1) return;
  named_barrier_sync(W == 2 ? 1 + h : 1 + KVH + h, W * 32);
#pragma unroll
  for (int d = W / 2; d >= 1; d >>= 1) {
    if (way >= d) {  // sender at this level (ways >= 2d have left)
      float* slot = scratch + (size_t)((way - d) * KVH + h) * kStateFloats * 32 + lane;
      slot[0 * 32] = st.m0;
      slot[1 * 32] = st.m1;
      slot[2 * 32] = st.l0;
      slot[3 * 32] = st.l1;
#pragma unroll
      for (int d4 = 0; d4 < 4; ++d4)
#pragma unroll
        for (int e = 0; e < 4; ++e) slot[(4 + 4 * d4 + e) * 32] = st.acc[d4][e];
      named_barrier_sync(1 + h, 2 * d * 32);
      return;
    }
    named_barrier_sync(1 + h, 2 * d * 32);
    merge_state(st, scratch + (size_t)(way * KVH + h) * kStateFloats * 32 + lane);
    // The next level's senders (ways [d/2, d)) overwrite slots that ways
    // [0, d/2) have just read.
    if (d > 1) named_barrier_sync(1 + h, d * 32);
  }
}

}  // namespace tvp
