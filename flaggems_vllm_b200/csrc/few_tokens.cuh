// What the two kernels behind fused_moe_few_tokens share (few_tokens.cu: 16-bit weights; few_tokens_fp8.cu: e4m3 weights): the call's
// arguments, the routing of its tokens, the 8-bit quantisation of activations.
#pragma once

#include <type_traits>

#include "route_row.cuh"
#include "tc_common.cuh"

namespace moe {

constexpr int kTokens = 8;
constexpr int kMaxSlots = 256;   // routed experts of a call: 8 tokens x 32
constexpr int kMaxExperts = 1024, kMaxHidden = 16384, kMaxHidden8 = 8192, kMaxWidth = 1 << 22;
constexpr int64_t kFewSmem = 232448;

struct Few {
  const void *x, *residual;
  void* out;
  const void *w1, *w2, *sw1, *sw2;              // sw: shared expert
  const float *w1s, *w2s, *sw1s, *sw2s;         // block scales
  const float *scores, *bias;                   // [M, E] sigmoids, or logits of a softmax
  float* topk_w;
  int32_t* topk_ids;
  void* h;                                      // [slots][8][I], then the shared expert's [8][Is]
  uint8_t *h8, *h8_shared;                      // in 8 bits: the routed experts' rows, the shared one's
  float *h8_scale, *h8_scale_shared;            // the scales of their groups, times the routing weights
  int32_t* counters;                            // claims of W1 and W2, finished runs of W1, one unused, outputs of each group of 128
  int64_t cleared;                              // counters to clear
  int64_t x_ld, residual_ld;
  int M, E, H, I, Is, topk, n_group, topk_group, renormalize, sigmoid;
  float scaling;
  int64_t x_pitch;                              // bytes from a token's row to the next, where the kernel reads them
  int staged;                                   // whether that is in shared memory
  int32_t* status;
  unsigned long long wait_ns;
};


// the experts of a call whose weights are e4m3, behind its router (few_tokens_fp8.cu)
int few_experts_fp8(const Few& P, int dtype, cudaStream_t st);

namespace {

struct B32 {  // 32 bytes of a row
  uint32_t r[8];
};
__device__ __forceinline__ void zero(B32& v) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v.r[i] = 0;
}
// 16 bytes from p on and 16 from p + APART on, in shared or global memory
template <int APART>
__device__ __forceinline__ void load_row(B32& v, const void* p) {
  const uint4 a = *reinterpret_cast<const uint4*>(p), b = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(p) + APART);
  v.r[0] = a.x; v.r[1] = a.y; v.r[2] = a.z; v.r[3] = a.w; v.r[4] = b.x; v.r[5] = b.y; v.r[6] = b.z; v.r[7] = b.w;
}
__device__ __forceinline__ int claim(int32_t* counter) { return atomicAdd(counter, 1); }

// Returns when `want` runs of W1 are done, or the library's limit has passed (the status word says so; the caller goes on, on
// whatever is there).
__device__ __forceinline__ void wait_for_runs(const int32_t* done, int64_t want, int32_t* status, unsigned long long wait_ns) {
  unsigned long long t0 = 0;
  for (uint32_t spins = 1;; ++spins) {
    int n;
    asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(n) : "l"(done) : "memory");
    if (n >= want || ((spins & 0x3F) == 0 && tc::wait_expired(t0, status, wait_ns))) return;
  }
}

template <typename T> __device__ __forceinline__ float2 widen2(uint32_t v);
template <> __device__ __forceinline__ float2 widen2<__nv_bfloat16>(uint32_t v) { return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v)); }
template <> __device__ __forceinline__ float2 widen2<__half>(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }

// 32 values of a lane, 128 of the four lanes of a group: their e4m3 bytes and the group's scale
template <typename T>
__device__ __forceinline__ float quantise(const B32 (&v)[2], B32& q) {
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float2 f = widen2<T>(v[i >> 3].r[i & 7]);
    m = max_nan(m, max_nan(fabsf(f.x), fabsf(f.y)));
  }
  m = max_nan(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
  m = max_nan(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
  const float s = (m > kQuantEps || m != m ? m : kQuantEps) * (1.0f / kFp8Max), inv = 1.0f / s;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 a = widen2<T>(v[i >> 2].r[2 * i & 7]), b = widen2<T>(v[i >> 2].r[(2 * i + 1) & 7]);
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(div_by_scale(a.x, s, inv), div_by_scale(a.y, s, inv)), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(div_by_scale(b.x, s, inv), div_by_scale(b.y, s, inv)), __NV_SATFINITE, __NV_E4M3);
    q.r[i] = lo | hi << 16;
  }
  return s;
}

struct Shared {
  float weight[kMaxSlots + 1][kTokens];   // of every routed expert for the tokens that it has; the shared expert's are 1
  uint32_t mask[kMaxSlots + 1];           // tokens of the expert
  int32_t list[kMaxSlots];                // routed experts, ascending
  uint32_t used[kMaxExperts / 32];        // a bit for each
  float bias[kMaxExperts];
  float w[kTokens][32];
  int32_t id[kTokens][32];
  int32_t whole[kMaxSlots];               // groups of h that this block has to quantise
  int32_t slots, next1, next2, wholes;
};
// What routing needs and the kernel in front does not make
__device__ __forceinline__ void prepare_route(const Few& P, Shared& S) {
  for (int e = threadIdx.x; e < P.E; e += blockDim.x) S.bias[e] = P.bias ? P.bias[e] : 0.0f;
  for (int i = threadIdx.x; i < kMaxSlots; i += blockDim.x) S.mask[i] = 0;
  if (threadIdx.x < kMaxExperts / 32) S.used[threadIdx.x] = 0;
  __syncthreads();
}
// The choice of one token by one warp: route_row's rule and order (route_row.cuh), in fewer steps of a lone warp, which takes four or
// five clocks for each.  u: scores of expert 32 j + lane.  ranks: E words of the warp's own.
template <int VPT>
__device__ __forceinline__ void choose(const Few& P, const Shared& S, const float (&u)[VPT], uint32_t* ranks, float* w_row, int32_t* id_row, int lane) {
  uint64_t key[VPT];
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int e = j * 32 + lane;
    key[j] = e < P.E ? make_key(u[j] + S.bias[e], (uint32_t)e) : 0;
  }
  if (P.n_group > 1) {
    const int per_group = P.E / P.n_group;
#pragma unroll
    for (int j = 0; j < VPT; ++j)
      if (j * 32 + lane < P.E) ranks[j * 32 + lane] = (uint32_t)(key[j] >> 32);
    __syncwarp();
    // neighbouring lanes share a group; its two largest out of their own
    const int share = P.n_group <= 4 ? 8 : (P.n_group <= 8 ? 4 : (P.n_group <= 16 ? 2 : 1));
    const int group = lane / share;
    uint32_t b1 = 0, b2 = 0;
    if (group < P.n_group) {
      for (int i = lane % share; i < per_group; i += share) {
        const uint32_t v = ranks[group * per_group + i];
        b2 = max(b2, min(b1, v));
        b1 = max(b1, v);
      }
    }
    for (int off = 1; off < share; off <<= 1) {
      const uint32_t o1 = __shfl_xor_sync(0xFFFFFFFFu, b1, off), o2 = __shfl_xor_sync(0xFFFFFFFFu, b2, off);
      b2 = max(max(b2, o2), min(b1, o1));
      b1 = max(b1, o1);
    }
    const float score = per_group >= 2 ? from_ordered_bits(b1) + from_ordered_bits(b2) : from_ordered_bits(b1);
    const uint32_t mine = ordered_bits(score);
    int rank = 0;
    for (int q = 0; q < P.n_group; ++q) {
      const uint32_t other = __shfl_sync(0xFFFFFFFFu, mine, q * share);
      rank += other > mine || (other == mine && q < group);
    }
    const uint32_t kept = __ballot_sync(0xFFFFFFFFu, group < P.n_group && rank < P.topk_group);  // bit q share: group q
    const float inv = 1.0f / (float)per_group;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int e = j * 32 + lane, q = (int)(((float)e + 0.5f) * inv);  // e / per_group: both below 2^10
      // experts of dropped groups rank as -inf (still ordered by index)
      if (e < P.E && !((kept >> (q * share)) & 1u)) key[j] = make_key(__int_as_float(0xff800000), (uint32_t)e);
    }
  }
  float my_w = 0.0f;
  int32_t my_id = 0;
  uint64_t local = 0;
  float local_u = 0.0f;
#pragma unroll
  for (int j = 0; j < VPT; ++j)
    if (key[j] > local) { local = key[j]; local_u = u[j]; }
  for (int t = 0; t < P.topk; ++t) {
    const uint64_t best = warp_max_u64(local);
    const uint32_t id = 0xFFFFFFFFu - (uint32_t)(best & 0xFFFFFFFFu);
    const float w = __shfl_sync(0xFFFFFFFFu, local_u, id & 31);  // the lane that holds it
    if (lane == t) { my_w = w; my_id = (int32_t)id; }
    if (local == best) {  // consumed: the lane's next largest
      local = 0;
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        if (key[j] < best && key[j] > local) { local = key[j]; local_u = u[j]; }
      }
    }
  }
  float sum = lane < P.topk ? my_w : 0.0f;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, off);
  if (lane < P.topk) {
    w_row[lane] = (P.renormalize ? my_w / (sum + 1e-20f) : my_w) * P.scaling;
    id_row[lane] = my_id;
  }
}

// every token's experts, by a warp each; the list of all of them.  scratch: E words for each of eight warps
template <int VPT>
__device__ __forceinline__ void route(const Few& P, Shared& S, uint32_t* scratch) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp < P.M) {
    const float* row = P.scores + (int64_t)warp * P.E;
    float u[VPT];
#pragma unroll
    for (int j = 0; j < VPT; ++j) u[j] = j * 32 + lane < P.E ? row[j * 32 + lane] : -INFINITY;
    if (!P.sigmoid) {
      float m = u[0];
#pragma unroll
      for (int j = 1; j < VPT; ++j) m = fmaxf(m, u[j]);
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, off));
      double sum = 0.0;
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        if (j * 32 + lane < P.E) {
          const double x = exp((double)u[j] - (double)m);
          sum += x;
          u[j] = (float)x;
        }
      }
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, off);
      const double inv = 1.0 / sum;
#pragma unroll
      for (int j = 0; j < VPT; ++j) u[j] = (float)(u[j] * inv);
    }
    choose<VPT>(P, S, u, scratch + warp * P.E, S.w[warp], S.id[warp], lane);
    __syncwarp();
    if (lane < P.topk) {
      const int id = S.id[warp][lane];
      atomicOr(&S.used[id >> 5], 1u << (id & 31));
      if (blockIdx.x == 0) {
        P.topk_w[warp * P.topk + lane] = S.w[warp][lane];
        P.topk_ids[warp * P.topk + lane] = id;
      }
    }
  }
  __syncthreads();
  // an expert's place is the number of used ones below it; lane i has those of the first 32 i
  const uint32_t word = S.used[lane];
  int below = __popc(word);
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int v = __shfl_up_sync(0xFFFFFFFFu, below, off);
    if (lane >= off) below += v;
  }
  const int slots = __shfl_sync(0xFFFFFFFFu, below, 31);
  below -= __popc(word);
  if (warp < P.M) {
    const int id = lane < P.topk ? S.id[warp][lane] : 0;
    const int s = __shfl_sync(0xFFFFFFFFu, below, id >> 5) + __popc(S.used[id >> 5] & ((1u << (id & 31)) - 1));
    if (lane < P.topk) {
      S.list[s] = id;
      S.weight[s][warp] = S.w[warp][lane];
      atomicOr(&S.mask[s], 1u << warp);
    }
  }
  if (warp == 0) {
    if (lane < kTokens) S.weight[slots][lane] = 1.0f;
    if (lane == 0) {
      S.slots = slots;
      S.mask[slots] = (1u << P.M) - 1;  // nobody's slot
    }
  }
  __syncthreads();
}

}  // namespace
}  // namespace moe
