// The ordering of scores as integer keys, which the kernels of grouped_topk.cu and few_tokens.cu share, and grouped_topk.cu's routing of one
// token by one warp: the group-limited selection of the largest.  The header of grouped_topk.cu has the definition.  few_tokens.cuh has
// the same choice in fewer steps (choose); the tests hold the two together, ties of experts and of groups included.
#pragma once

#include "moe_common.cuh"

namespace moe {
namespace {

__device__ __forceinline__ uint32_t ordered_bits(float v) {
  uint32_t b = __float_as_uint(v);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ uint64_t make_key(float v, uint32_t idx) {
  return ((uint64_t)ordered_bits(v) << 32) | (uint64_t)(0xFFFFFFFFu - idx);
}
// max of a 64-bit key over the warp with two 32-bit reductions (redux.sync): the largest high
// word, then the largest low word among the lanes that hold it
__device__ __forceinline__ uint64_t warp_max_u64(uint64_t k) {
  const uint32_t hi = (uint32_t)(k >> 32), lo = (uint32_t)k;
  const uint32_t mh = __reduce_max_sync(0xFFFFFFFFu, hi);
  const uint32_t ml = __reduce_max_sync(0xFFFFFFFFu, hi == mh ? lo : 0u);
  return ((uint64_t)mh << 32) | ml;
}
__device__ __forceinline__ float from_ordered_bits(uint32_t ob) {
  return __uint_as_float((ob & 0x80000000u) ? (ob ^ 0x80000000u) : ~ob);
}

// The routing of one token by one warp: `row` holds the token's E scores (element stride
// `stride1`; global or shared memory), the results go to w_row / id_row [topk].
template <typename ST, typename BT, int VPT>
__device__ __forceinline__ void route_row(const ST* row, int64_t stride1, const BT* __restrict__ bias, int E,
                                          int n_group, int topk_group, int topk, int renormalize, float scaling,
                                          int scoring_func, float* w_row, int32_t* id_row, int lane) {
  const int per_group = E / n_group;
  const float NEG_INF = __int_as_float(0xff800000);

  float u[VPT];      // unbiased score
  uint64_t key[VPT]; // ranking key of u + bias (0 = absent / consumed)
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int e = j * 32 + lane;
    if (e < E) {
      float s = ToF32<ST>::get(row[(int64_t)e * stride1]);
      if (scoring_func == 1) s = (float)(1.0 / (1.0 + exp(-(double)s)));
      u[j] = s;
      key[j] = make_key(s + ToF32<BT>::get(bias[e]), (uint32_t)e);
    } else {
      u[j] = 0.0f;
      key[j] = 0;
    }
  }

  if (n_group > 1) {
    // group of every register of this lane, computed once (-1: no expert)
    int grp[VPT];
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int e = j * 32 + lane;
      grp[j] = e < E ? e / per_group : -1;
    }
    // group score -> lane g holds the score of group g.  The two largest r of a group are found
    // on the order-preserving integer image of r (the key's high word; 0 = none): the lane's own
    // two, then the warp's largest, then the largest of what is left once its owner gave it up.
    float my_group_score = NEG_INF;
    for (int g = 0; g < n_group; ++g) {
      uint32_t b1 = 0, b2 = 0;
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        if (grp[j] == g) {
          const uint32_t ob = (uint32_t)(key[j] >> 32);
          if (ob > b1) { b2 = b1; b1 = ob; } else if (ob > b2) { b2 = ob; }
        }
      }
      const uint32_t top1 = __reduce_max_sync(0xFFFFFFFFu, b1);
      const int owner = __ffs(__ballot_sync(0xFFFFFFFFu, b1 == top1)) - 1;
      const uint32_t top2 = __reduce_max_sync(0xFFFFFFFFu, lane == owner ? b2 : b1);
      const float gs = per_group >= 2 ? from_ordered_bits(top1) + from_ordered_bits(top2) : from_ordered_bits(top1);
      if (lane == g) my_group_score = gs;
    }
    // choose topk_group groups
    uint32_t keep_mask = 0;
    uint64_t gkey = lane < n_group ? make_key(my_group_score, (uint32_t)lane) : 0;
    for (int t = 0; t < topk_group; ++t) {
      uint64_t best = warp_max_u64(gkey);
      uint32_t g = 0xFFFFFFFFu - (uint32_t)(best & 0xFFFFFFFFu);
      keep_mask |= 1u << (g & 31);
      if (gkey == best) gkey = 0;
    }
    // experts of dropped groups rank as -inf (still ordered by index)
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int e = j * 32 + lane;
      if (grp[j] >= 0 && !((keep_mask >> grp[j]) & 1u)) key[j] = make_key(NEG_INF, (uint32_t)e);
    }
  }

  // top-k extraction
  float my_w = 0.0f;
  int32_t my_id = 0;
  uint64_t local = 0;
  int local_j = 0;
#pragma unroll
  for (int j = 0; j < VPT; ++j)
    if (key[j] > local) { local = key[j]; local_j = j; }
  for (int t = 0; t < topk; ++t) {
    uint64_t best = warp_max_u64(local);
    uint32_t id = 0xFFFFFFFFu - (uint32_t)(best & 0xFFFFFFFFu);
    float wsel = 0.0f;
    if (local == best && best != 0) {
      // this lane owns the winner: fetch its unbiased value, consume it
#pragma unroll
      for (int j = 0; j < VPT; ++j)
        if (j == local_j) { wsel = u[j]; key[j] = 0; }
      local = 0;
#pragma unroll
      for (int j = 0; j < VPT; ++j)
        if (key[j] > local) { local = key[j]; local_j = j; }
    }
    wsel = __shfl_sync(0xFFFFFFFFu, wsel, id & 31);
    if (lane == t) { my_w = wsel; my_id = (int32_t)id; }
  }
  float sum = lane < topk ? my_w : 0.0f;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, off);
  if (lane < topk) {
    float w = renormalize ? my_w / (sum + 1e-20f) : my_w;
    w_row[lane] = w * scaling;
    id_row[lane] = my_id;
  }
}

}  // namespace
}  // namespace moe
