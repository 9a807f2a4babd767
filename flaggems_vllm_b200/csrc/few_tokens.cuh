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
  int x_pitch, staged;                          // bytes of a token's row in shared memory; whether the rows are there
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
// every token's experts, by a warp each; the list of all of them
template <int VPT>
__device__ __forceinline__ void route(const Few& P, Shared& S, float* scratch) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp < P.M) {
    const float* u = P.scores + (int64_t)warp * P.E;
    if (!P.sigmoid) {
      float l[VPT], m = -INFINITY;
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        l[j] = j * 32 + lane < P.E ? u[j * 32 + lane] : -INFINITY;
        m = fmaxf(m, l[j]);
      }
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, off));
      float* s = scratch + warp * P.E;
      double sum = 0.0;
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        if (j * 32 + lane < P.E) {
          const double x = exp((double)l[j] - (double)m);
          sum += x;
          l[j] = (float)x;
        }
      }
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, off);
      const double inv = 1.0 / sum;
#pragma unroll
      for (int j = 0; j < VPT; ++j)
        if (j * 32 + lane < P.E) s[j * 32 + lane] = (float)(l[j] * inv);
      __syncwarp();
      u = s;
    }
    route_row<float, float, VPT>(u, 1, S.bias, P.E, P.n_group, P.topk_group, P.topk, P.renormalize, P.scaling, 0, S.w[warp], S.id[warp], lane);
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
