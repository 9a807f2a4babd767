// Dense products with a fused epilogue, and their gradients:
//
//     z = x W^T + b,   y = act(z) + residual          x [M, K], W [N', K], y [M, N]
//     dz = dy act'(z), dx = dz W, dW = dz^T x, db = sum over rows of dz
//
// N' = N, or 2 N for the gated activation silu(z[:, :N]) * z[:, N:].  Sums, bias, activation and residual are fp32, y is rounded
// once.  z is kept for the backward pass in the operands' type: its rounding reaches the gradients through act' only, and dz has
// to be rounded to that type anyway, because it is an operand of two products; the bias' gradient sums dz before its rounding.
// The gated activation keeps z in fp32: there dz is a product of both halves of z and takes their roundings in full.
//
// All products are one form, D[r, c] = sum_k A[r, k] B[c, k], in which each operand may lie either way in memory: rows of k
// ("K-major": x and W forward, dz for dx) or rows of r or c ("MN-major": W for dx, dz and x for dW).  The tensor core takes both
// from 128-byte swizzled tiles, so nothing is transposed on the way: a box of 64 x 64 elements lands as 8 KB in both cases and
// only its descriptor differs.  Two kernels:
//
//   pair_kernel   256 x 256 (or 256 x 128) tiles by a CTA pair (cta_group::2), persistent, two accumulators, so that a tile's
//                 epilogue runs under the next tile's products: products that fill the GPU.
//   tile_kernel   128 x BN tiles, K divided over a cluster whose partial sums are added through distributed shared memory in
//                 rank order: few rows (the weights are then the 128 side, "swapped", and what counts is how many SMs stream
//                 them), and products of few tiles.
//
// Both are deterministic.  fp32 operands run on f32_kernel (CUDA cores: the tensor core has no fp32 products).
#include <cooperative_groups.h>

#include <type_traits>

#include "tc_common.cuh"

namespace cg = cooperative_groups;

namespace moe {
namespace {
using namespace tc;

// What happens to a finished sum.  m: row of y, n: column of y.
struct Epilogue {
  const void* bias;      // [N'], in the operands' type or (bias_f32) fp32; null = none
  const void* residual;  // [M, N], rows residual_ld apart; null = none
  void* y;               // [M, N]
  void* z;               // [M, N'], null = not kept
  int64_t residual_ld, y_ld, z_ld;
  int N, act, bias_f32;
};

// Distribution function of the normal distribution, Phi.  fp32 results take CUDA's; 16-bit ones, on the negative side,
// e^(-z^2 / 2) erfcx(|z| / sqrt 2) / 2 with erfcx(x) = t P(t), t = 1 / (1 + 0.51 x): the form of formula 7.1.26 in Abramowitz and
// Stegun, Handbook of Mathematical Functions, whose own coefficients keep the absolute error small.  The seven here keep the relative one
// below 2^-20 for x up to 10 (least squares reweighted towards the largest error, against erfcx in 64 bits), where Phi is below
// bf16's smallest number.  What is left is the fast exponential's error, 2^-16 of Phi at z = -13 and 2^-18 at -6; half a step is
// 2^-8 and 2^-11 of the value.  (4096 x 2048 -> 4096
// bf16 with gelu: 51.9 us, 51.3 with the published five.)
template <typename T>
__device__ __forceinline__ float normal_cdf(float z) {
  if constexpr (std::is_same<T, float>::value) {
    return normcdff(z);
  } else {
    const float t = __fdividef(1.0f, fmaf(0.36062446f, fabsf(z), 1.0f));  // 0.51 / sqrt 2
    const float p = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, 0.0944997968f, -0.359134275f), 0.35844488f), 0.0550533605f), 0.279065958f),
                                     0.284152342f), 0.287917501f);
    const float tail = 0.5f * p * __expf(-0.5f * z * z);
    return z < 0.0f ? tail : 1.0f - tail;
  }
}
// 1 / (1 + e^-z), by e^-|z|, which cannot overflow: below z = -88 too, where the result, or z times it, is still a normal number of
// fp32 and bf16.  Fast forms where the result is rounded to 16 bits.
template <typename T>
__device__ __forceinline__ float sigmoid(float z) {
  float e, q;
  if constexpr (std::is_same<T, float>::value) {
    e = expf(-fabsf(z));
    q = 1.0f / (1.0f + e);
  } else {
    e = __expf(-fabsf(z));
    q = __fdividef(1.0f, 1.0f + e);
  }
  return z < 0.0f ? e * q : q;
}
// (1 + tanh(c (z + a z^3))) / 2 is the sigmoid of twice the argument
template <typename T>
__device__ __forceinline__ float tanh_gate(float z) {
  return sigmoid<T>(1.5957691216057308f * z * fmaf(0.044715f * z, z, 1.0f));
}
template <typename T>
__device__ __forceinline__ float act_value(int act, float z) {
  switch (act) {
    case MOE_LIN_RELU: return z > 0.0f ? z : (z != z ? z : 0.0f);
    case MOE_LIN_SILU: return z * sigmoid<T>(z);
    case MOE_LIN_GELU: return z * normal_cdf<T>(z);
    case MOE_LIN_GELU_TANH: return z * tanh_gate<T>(z);
    default: return z;
  }
}
template <typename T>
__device__ __forceinline__ float act_slope(int act, float z) {
  switch (act) {
    case MOE_LIN_RELU: return z > 0.0f ? 1.0f : (z != z ? z : 0.0f);
    case MOE_LIN_SILU: {
      const float s = sigmoid<T>(z);
      return s * (1.0f + z * (1.0f - s));
    }
    case MOE_LIN_GELU: {
      const float e = std::is_same<T, float>::value ? expf(-0.5f * z * z) : __expf(-0.5f * z * z);
      return normal_cdf<T>(z) + z * (0.3989422804014327f * e);
    }
    case MOE_LIN_GELU_TANH: {  // g = sigmoid(s): (z g)' = g + z g (1 - g) s'
      const float g = tanh_gate<T>(z);
      const float h = g * (1.0f - g);
      return h == 0.0f ? g : g + z * h * (1.5957691216057308f * fmaf(0.134145f * z, z, 1.0f));  // s' overflows far out
    }
    default: return 1.0f;
  }
}
// How sums are rounded, two at a time: as results, or as the backward pass gets them.  There, those that the type cannot hold become its
// largest value, not infinity, where the slopes are 0 times infinity (far out they are 0 and 1 long before); what is no number stays
// so.  relu's slope asks for the sign: a positive sum that the type would round to zero becomes its smallest value.
struct AsResult {
  template <typename T>
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack2<T>(lo, hi); }
};
struct AsKept {
  template <typename T>
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    uint32_t r;
    if constexpr (std::is_same<T, __half>::value) asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
  }
};
struct AsKeptSign {
  template <typename T>
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    constexpr float least = std::is_same<T, __half>::value ? 0x1p-24f : 0x1p-133f;
    return AsKept::pack<T>(lo > 0.0f ? fmaxf(lo, least) : lo, hi > 0.0f ? fmaxf(hi, least) : hi);
  }
};
template <typename T, typename As>
__device__ __forceinline__ T rounded(float v) {
  if constexpr (sizeof(T) == 4) {
    return v;
  } else {
    const uint16_t h = (uint16_t)As::template pack<T>(v, 0.0f);
    return *reinterpret_cast<const T*>(&h);
  }
}
template <typename T>
__device__ __forceinline__ float bias_at(const Epilogue& E, int n) {
  if (E.bias == nullptr) return 0.0f;
  return E.bias_f32 ? reinterpret_cast<const float*>(E.bias)[n] : ToF32<T>::get(reinterpret_cast<const T*>(E.bias)[n]);
}
// the sum(s) of output (m, n) -> its value, and z where it is kept; z1: the gate's partner; add: its residual, if that is at hand
template <typename T>
__device__ __forceinline__ float value(const Epilogue& E, int64_t m, int n, float z0, float z1, const T* add = nullptr) {
  z0 += bias_at<T>(E, n);
  float v;
  if (E.act == MOE_LIN_SILU_MUL) {
    z1 += bias_at<T>(E, E.N + n);
    v = z0 * sigmoid<T>(z0) * z1;
    if (E.z) {
      float* z = reinterpret_cast<float*>(E.z) + m * E.z_ld + n;
      z[0] = z0;
      z[E.N] = z1;
    }
  } else {
    v = act_value<T>(E.act, z0);
    if (E.z) reinterpret_cast<T*>(E.z)[m * E.z_ld + n] = E.act == MOE_LIN_RELU ? rounded<T, AsKeptSign>(z0) : rounded<T, AsKept>(z0);
  }
  if (add) v += ToF32<T>::get(*add);
  else if (E.residual) v += ToF32<T>::get(reinterpret_cast<const T*>(E.residual)[m * E.residual_ld + n]);
  return v;
}
template <typename T>
__device__ __forceinline__ void finish(const Epilogue& E, int64_t m, int n, float z0, float z1, const T* add) {
  reinterpret_cast<T*>(E.y)[m * E.y_ld + n] = from_f32<T>(value<T>(E, m, n, z0, z1, add));
}

// ------------------------------------------------------------------ operand tiles
constexpr int BOX = 64 * 128;  // bytes of a box: 64 rows of 128 bytes, swizzled, either way round

// descriptor of a tile of such boxes: K-major rows follow each other; MN-major boxes are 64 rows (columns of D) each, the
// eight-k groups of a box 1024 bytes apart
__device__ __forceinline__ uint64_t box_desc(uint32_t saddr, bool mn) {
  uint64_t d = make_smem_desc(saddr);
  if (mn) d = (d & ~((uint64_t)0x3FFF << 16)) | ((uint64_t)(BOX >> 4) << 16);
  return d;
}
// what 16 elements of k are in a descriptor's address field
__device__ __forceinline__ uint64_t k_step(bool mn) { return mn ? 2048 >> 4 : 32 >> 4; }

struct Product {
  int64_t rows, cols;  // of D
  int KB;              // steps of 64 k
  int a_mn, b_mn;
  int gate;            // distance of the up rows from the gate rows in the weights (N of a gated call), else 0
  int swapped;         // rows of D are columns of y
  int split, BN, ring; // tile_kernel
  int group;           // pair_kernel: row tiles that walk the column tiles together
  int32_t* status;
  unsigned long long wait_ns;
};

// ------------------------------------------------------------------ tile_kernel
constexpr int TTHREADS = 256;
struct TAux {
  uint64_t full[12], empty[12], done;
  uint32_t tmem_base, unused;  // whole 8 bytes: the stash lies behind
};
// Two waves of blocks and more: tiles of up to 128 columns leave room for a second block on the multiprocessor, which streams while the
// first one adds up and stores (64 x 4096 -> 2 x 14336 gated 50.5 -> 44.1 us).  One wave: all of the memory is one block's ring (33 x
// 14336 -> 4096 24.8 -> 23.9).
constexpr int kRingWhole = 196608, kRingHalf = 98304;
__host__ __device__ constexpr int tile_stage(int bn) { return (128 + bn) * 128; }
__host__ __device__ constexpr int tile_stages(int bn, int ring) { return ring / tile_stage(bn) < 12 ? ring / tile_stage(bn) : 12; }
constexpr int kStash = 8192;  // residuals of a share of up to 1024 quads
constexpr size_t tile_smem(int ring) { return (size_t)ring + 1024 + sizeof(TAux) + kStash; }
static_assert(128 * 260 * 4 <= kRingWhole && 128 * 132 * 4 <= kRingHalf, "the partial tile takes the ring's place");
static_assert(2 * (tile_smem(kRingHalf) + 1024) <= 233472, "two blocks on a multiprocessor");

__device__ __forceinline__ void tmem_ld16_sync(uint32_t taddr, uint32_t* a) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]), "=r"(a[4]), "=r"(a[5]), "=r"(a[6]), "=r"(a[7]), "=r"(a[8]), "=r"(a[9]),
        "=r"(a[10]), "=r"(a[11]), "=r"(a[12]), "=r"(a[13]), "=r"(a[14]), "=r"(a[15])
      : "r"(taddr)
      : "memory");
}

// This CTA's share of the outputs of its cluster's tile, four columns of D at a time: the partial sums of all ranks in flight, added
// in rank order.  Lanes run along the rows of y.
template <typename T, int SPLIT, int THREADS = TTHREADS>
__device__ __forceinline__ void finish_share(cg::cluster_group& cluster, uint8_t* smem, const Product& P, const Epilogue& E, int rank, int64_t r0,
                                             int64_t c0, int out_rows, int out_cols, const T* stash = nullptr) {
  const int pitch = P.BN + 4, quads = out_cols / 4, share = out_rows * quads / SPLIT;  // all powers of two
  const int row_bits = __ffs(out_rows) - 1, quad_bits = __ffs(quads) - 1;
  const int up = P.gate == 0 ? 0 : (P.swapped ? 64 * pitch : P.BN / 2);
  const float* base[SPLIT];
#pragma unroll
  for (int j = 0; j < SPLIT; ++j)
    base[j] = SPLIT == 1 ? reinterpret_cast<const float*>(smem) : cluster.map_shared_rank(reinterpret_cast<const float*>(smem), j);
  const bool wide = !P.swapped && ((uintptr_t)E.y & (4 * sizeof(T) - 1)) == 0 && E.y_ld % 4 == 0;
  for (int i = rank * share + threadIdx.x; i < (rank + 1) * share; i += THREADS) {
    const int r = P.swapped ? i & (out_rows - 1) : i >> quad_bits, c = 4 * (P.swapped ? i >> row_bits : i & (quads - 1));
    if (r0 + r >= P.rows || c0 + c >= P.cols) continue;
    const int at = r * pitch + c;
    const T* add = stash ? stash + 4 * (i - rank * share) : nullptr;
    float4 v[SPLIT], u[SPLIT];
#pragma unroll
    for (int j = 0; j < SPLIT; ++j) v[j] = *reinterpret_cast<const float4*>(base[j] + at);
    if (up) {
#pragma unroll
      for (int j = 0; j < SPLIT; ++j) u[j] = *reinterpret_cast<const float4*>(base[j] + at + up);
    }
    float z0[4] = {v[0].x, v[0].y, v[0].z, v[0].w}, z1[4] = {};
#pragma unroll
    for (int j = 1; j < SPLIT; ++j) { z0[0] += v[j].x; z0[1] += v[j].y; z0[2] += v[j].z; z0[3] += v[j].w; }
    if (up) {
#pragma unroll
      for (int j = 0; j < SPLIT; ++j) { z1[0] += u[j].x; z1[1] += u[j].y; z1[2] += u[j].z; z1[3] += u[j].w; }
    }
    if (wide && c0 + c + 4 <= P.cols) {
      const int64_t m = r0 + r;
      const int n = (int)(c0 + c);
      float o[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) o[q] = value<T>(E, m, n + q, z0[q], z1[q], add ? add + q : nullptr);
      T* y = reinterpret_cast<T*>(E.y) + m * E.y_ld + n;
      if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(y) = make_float4(o[0], o[1], o[2], o[3]);
      else *reinterpret_cast<uint2*>(y) = make_uint2(pack2<T>(o[0], o[1]), pack2<T>(o[2], o[3]));
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (c0 + c + q < P.cols) finish<T>(E, P.swapped ? c0 + c + q : r0 + r, (int)(P.swapped ? r0 + r : c0 + c + q), z0[q], z1[q], add ? add + q : nullptr);
    }
  }
}

// The residual of this CTA's share, quad by quad as finish_share takes it, into shared memory while the products run: there each of
// its steps would wait for memory (33 x 14336 -> 4096 with a residual 27.4 -> 24.1 us, 501 x 1024 -> 768 13.2 -> 9.4).
template <typename T>
__device__ __forceinline__ void stash_residual(const Product& P, const Epilogue& E, int rank, int64_t r0, int64_t c0, int out_rows, int out_cols,
                                               T* stash, int t, int threads) {
  const int quads = out_cols / 4, share = out_rows * quads / P.split, row_bits = __ffs(out_rows) - 1, quad_bits = __ffs(quads) - 1;
#pragma unroll 4
  for (int k = t; k < share; k += threads) {
    const int i = rank * share + k;
    const int64_t r = r0 + (P.swapped ? i & (out_rows - 1) : i >> quad_bits), c = c0 + 4 * (P.swapped ? i >> row_bits : i & (quads - 1));
    T v[4] = {};
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (r < P.rows && c + q < P.cols) v[q] = reinterpret_cast<const T*>(E.residual)[P.swapped ? (c + q) * E.residual_ld + r : r * E.residual_ld + c + q];
#pragma unroll
    for (int q = 0; q < 4; ++q) stash[4 * k + q] = v[q];
  }
}

// One 128 x BN tile of D by the `split` CTAs of a cluster, each over its share of K.  A gated call's tile is half gate rows and
// half up rows of the weights, whichever side they are on.
template <typename T>
__global__ void __launch_bounds__(TTHREADS, 2)
tile_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const Product P, const Epilogue E) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align_1024(smem_raw);
  TAux* aux = reinterpret_cast<TAux*>(smem + P.ring);
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank();
  const int warp = __shfl_sync(0xFFFFFFFFu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int BN = P.BN, stage = tile_stage(BN), stages = tile_stages(BN, P.ring);
  const bool gate_a = P.gate != 0 && P.swapped, gate_b = P.gate != 0 && !P.swapped;
  const int out_rows = gate_a ? 64 : 128, out_cols = gate_b ? BN / 2 : BN;  // of D that the tile finishes
  const int64_t r0 = (int64_t)blockIdx.y * out_rows;
  const int64_t c0 = (int64_t)(blockIdx.x / P.split) * out_cols;
  const int kb0 = (int)((int64_t)P.KB * rank / P.split), kb1 = (int)((int64_t)P.KB * (rank + 1) / P.split);
  const uint32_t cols_alloc = BN < 32 ? 32 : BN;
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) { mbar_init(&aux->full[s], 1); mbar_init(&aux->empty[s], 1); }
    mbar_init(&aux->done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&aux->tmem_base)), "r"(cols_alloc));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = aux->tmem_base;
  pdl_wait();  // operands, weights among them, may be the kernel's in front
  pdl_trigger();
  T* stash = E.residual != nullptr && out_rows * out_cols / 4 / P.split <= kStash / 8 ? reinterpret_cast<T*>(aux + 1) : nullptr;
  if (warp == 0) {
    const bool leader = elect_lane();
    const int bbox = gate_b ? (BN / 2 < 64 ? BN / 2 : 64) : (BN < 64 ? BN : 64);  // rows of a box of B
    const int nb = BN / bbox;
    for (int kb = kb0, s = 0, ph = 1; kb < kb1; ++kb) {
      if (!mbar_wait(&aux->empty[s], ph, P.status, P.wait_ns)) break;
      if (leader) {
        uint8_t* sA = smem + (size_t)s * stage;
        mbar_expect_tx(&aux->full[s], stage);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int r = (int)r0 + (gate_a ? j * P.gate : j * 64);
          tma_load_2d(&map_a, &aux->full[s], sA + j * BOX, P.a_mn ? r : kb * 64, P.a_mn ? kb * 64 : r);
        }
        for (int j = 0; j < nb; ++j) {
          int c = (int)c0 + j * bbox;
          if (gate_b && j >= nb / 2) c += P.gate - out_cols;
          tma_load_2d(&map_b, &aux->full[s], sA + 2 * BOX + j * bbox * 128, P.b_mn ? c : kb * 64, P.b_mn ? kb * 64 : c);
        }
      }
      if (++s == stages) { s = 0; ph ^= 1; }
    }
  } else if (warp == 1) {
    const bool leader = elect_lane();
    constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    const uint32_t idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)P.a_mn << 15) | ((uint32_t)P.b_mn << 16) |
                           ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
    const uint64_t ka = k_step(P.a_mn), kb_ = k_step(P.b_mn);
    const uint64_t a0 = box_desc(smem_u32(smem), P.a_mn), b0 = box_desc(smem_u32(smem) + 2 * BOX, P.b_mn);
    bool first = true;
    for (int kb = kb0, s = 0, ph = 0; kb < kb1; ++kb) {
      if (!mbar_wait(&aux->full[s], ph, P.status, P.wait_ns)) break;
      tc_fence_after();
      if (leader) {
        const uint64_t ad = a0 + (uint64_t)(s * (stage >> 4)), bd = b0 + (uint64_t)(s * (stage >> 4));
#pragma unroll
        for (int k4 = 0; k4 < 4; ++k4) tc_mma<MMA_F16>(tmem, ad + k4 * ka, bd + k4 * kb_, idesc, first && k4 == 0 ? 0u : 1u);
        tc_commit(&aux->empty[s]);
      }
      first = false;
      if (++s == stages) { s = 0; ph ^= 1; }
    }
    if (leader) tc_commit(&aux->done);
  } else if (stash != nullptr) {
    stash_residual<T>(P, E, rank, r0, c0, out_rows, out_cols, stash, threadIdx.x - 64, TTHREADS - 64);
  }
  if (warp >= 4) {
    // every product has finished reading the ring: it now holds the partial tile, rows of BN + 4 floats (a pitch that spreads
    // 16-byte pieces over the banks down a column as well as along the lanes' rows)
    const bool ok = warp_agrees(mbar_wait(&aux->done, 0, P.status, P.wait_ns));
    tc_fence_after();
    const int row = ((warp & 3) << 5) + lane;
    float* part = reinterpret_cast<float*>(smem) + (size_t)row * (BN + 4);
    if (ok) {
#pragma unroll 1
      for (int c = 0; c < BN; c += 16) {
        uint32_t r[16];
        tmem_ld16_sync(tmem + ((uint32_t)((warp & 3) << 5) << 16) + (uint32_t)c, r);
#pragma unroll
        for (int i = 0; i < 4; ++i) reinterpret_cast<uint4*>(part + c)[i] = make_uint4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
      }
    }
    tc_fence_before();
  }
  __syncwarp();  // a wait that gave up may have ended for some lanes first
  if (P.split > 1) cluster.sync();
  else __syncthreads();
  switch (P.split) {
    case 1: finish_share<T, 1>(cluster, smem, P, E, rank, r0, c0, out_rows, out_cols, stash); break;
    case 2: finish_share<T, 2>(cluster, smem, P, E, rank, r0, c0, out_rows, out_cols, stash); break;
    case 4: finish_share<T, 4>(cluster, smem, P, E, rank, r0, c0, out_rows, out_cols, stash); break;
    default: finish_share<T, 8>(cluster, smem, P, E, rank, r0, c0, out_rows, out_cols, stash);
  }
  tc_fence_before();
  if (P.split > 1) cluster.sync();  // no CTA leaves while its partial tile may still be read
  else __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols_alloc));
  }
}

// ------------------------------------------------------------------ pair_kernel
constexpr int PTHREADS = 384, PCONS = 256;
constexpr int kPairRing = 196608;
struct PAux {
  uint64_t full[8], empty[8], tmem_full[2], tmem_empty[2];
  uint32_t tmem_base;
};
constexpr int kStagePitch = 33;  // floats of a staged row of 32 columns
constexpr int kPairStage = PCONS * kStagePitch * 4;
constexpr size_t kPairSmem = (size_t)kPairRing + kPairStage + 1024 + sizeof(PAux);
static_assert(kPairSmem <= 232448, "shared memory of one SM");

// Tile order: `group` row tiles share a walk over the column tiles, so that the pairs that run at one time read few different
// operand tiles.
__device__ __forceinline__ void tile_at(int item, int RT, int CT, int group, int& rt, int& ct) {
  const int per = group * CT, g = item / per, first = g * group;
  const int size = RT - first < group ? RT - first : group;
  const int in = item - g * per;
  rt = first + in % size;
  ct = in / size;
}

// 32 columns of 32 rows between a warp's registers (lane = row) and memory.  `wide`: the rows are whole 16-byte pieces, and each
// lane moves its own; else they go through shared memory, so that the warp reads and writes along the rows (4096 x 2048 -> 4097:
// 57 us, 232 with each lane at its own row).
struct Rows {
  int64_t m0, end;  // the warp's first row, the first row that is not there
  int n0, n;        // first column, columns that are there (n > 0)
  float* stage;     // the warp's own
  int lane;
};
template <typename S>
__device__ __forceinline__ void load_rows(const S* base, int64_t ld, bool wide, const Rows& R, float (&v)[32]) {
  if (wide && R.n == 32) {
    if (R.m0 + R.lane < R.end) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float t[8];
        load8<S>(base + (R.m0 + R.lane) * ld + R.n0 + 8 * i, t);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[8 * i + j] = t[j];
      }
    }
  } else {
    __syncwarp();
#pragma unroll 8
    for (int r = 0; r < 32; ++r)
      R.stage[r * kStagePitch + R.lane] = R.m0 + r < R.end && R.lane < R.n ? ToF32<S>::get(base[(R.m0 + r) * ld + R.n0 + R.lane]) : 0.0f;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = R.stage[R.lane * kStagePitch + i];
  }
}
template <typename S, typename As = AsResult>
__device__ __forceinline__ void store_rows(S* base, int64_t ld, bool wide, bool wide32, const Rows& R, const float (&v)[32]) {
  if (wide && R.n == 32) {
    if (R.m0 + R.lane < R.end) {
      S* p = base + (R.m0 + R.lane) * ld + R.n0;
      if constexpr (sizeof(S) == 4) {
        uint4 q[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          q[i] = make_uint4(__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]), __float_as_uint(v[4 * i + 2]), __float_as_uint(v[4 * i + 3]));
        store_row_pieces<8>(p, q, wide32);
      } else {
        uint4 q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          q[i] = make_uint4(As::template pack<S>(v[8 * i], v[8 * i + 1]), As::template pack<S>(v[8 * i + 2], v[8 * i + 3]),
                            As::template pack<S>(v[8 * i + 4], v[8 * i + 5]), As::template pack<S>(v[8 * i + 6], v[8 * i + 7]));
        store_row_pieces<4>(p, q, wide32);
      }
    }
  } else {
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 32; ++i) R.stage[R.lane * kStagePitch + i] = v[i];
    __syncwarp();
#pragma unroll 8
    for (int r = 0; r < 32; ++r)
      if (R.m0 + r < R.end && R.lane < R.n) base[(R.m0 + r) * ld + R.n0 + R.lane] = rounded<S, As>(R.stage[r * kStagePitch + R.lane]);
  }
}
// whole 16 (32) byte pieces, for columns that begin at multiples of 32
template <typename S>
__device__ __forceinline__ bool pieces(const S* base, int64_t ld, int bytes) {
  return ((uintptr_t)base & (bytes - 1)) == 0 && ld * (int64_t)sizeof(S) % bytes == 0;
}

template <typename T>
__global__ void __launch_bounds__(PTHREADS, 1)
pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const Product P, const Epilogue E) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align_1024(smem_raw);
  PAux* aux = reinterpret_cast<PAux*>(smem + kPairRing + kPairStage);
  const int warp = __shfl_sync(0xFFFFFFFFu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int cr = (int)cluster_ctarank();  // 0 leads
  const int BN = P.BN, stage = 2 * BOX + (BN / 128) * BOX, stages = BN == 256 ? 6 : 8;
  const int out_cols = P.gate ? BN / 2 : BN;
  const int RT = (int)((P.rows + 255) / 256), CT = (int)((P.cols + out_cols - 1) / out_cols);
  const int total = RT * CT, item0 = blockIdx.x / 2, step = gridDim.x / 2;
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) { mbar_init(&aux->full[s], 1); mbar_init(&aux->empty[s], 1); }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&aux->tmem_full[a], 1);
      mbar_init(&aux->tmem_empty[a], 2 * (PCONS / 32));  // the warps of both CTAs
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&aux->tmem_base)), "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::);
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // both CTAs' barriers exist before anyone signals across
  tc_fence_after();
  const uint32_t tmem_base = aux->tmem_base;
  pdl_wait();
  pdl_trigger();

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    const bool leader = elect_lane();
    if (leader) {
      asm volatile("prefetch.tensormap [%0];" ::"l"(&map_a) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(&map_b) : "memory");
    }
    uint32_t s = 0, ph = 1;
    bool alive = true;
    for (int item = item0; item < total && alive; item += step) {
      int rt, ct;
      tile_at(item, RT, CT, P.group, rt, ct);
      const int r = rt * 256 + cr * 128;
      // the pair's columns, half from each CTA: gate and up of a gated call
      const int c = P.gate ? ct * out_cols + cr * P.gate : ct * BN + cr * (BN / 2);
      for (int kb = 0; kb < P.KB; ++kb) {
        if (!mbar_wait(&aux->empty[s], ph, P.status, P.wait_ns)) { alive = false; break; }
        if (leader) {
          if (cr == 0) mbar_expect_tx(&aux->full[s], 2 * stage);  // the peer's bytes may already have been counted
          uint8_t* sA = smem + (size_t)s * stage;
#pragma unroll
          for (int j = 0; j < 2; ++j)
            tma_load_2d_pair(&map_a, &aux->full[s], sA + j * BOX, P.a_mn ? r + 64 * j : kb * 64, P.a_mn ? kb * 64 : r + 64 * j);
          for (int j = 0; j < BN / 128; ++j)
            tma_load_2d_pair(&map_b, &aux->full[s], sA + (2 + j) * BOX, P.b_mn ? c + 64 * j : kb * 64, P.b_mn ? kb * 64 : c + 64 * j);
        }
        if (++s == stages) { s = 0; ph ^= 1; }
      }
    }
  } else if (warp == 1 && cr == 0) {
    // ------------------------------------------------------------ MMA issuer
    const bool leader = elect_lane();
    constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    const uint32_t idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)P.a_mn << 15) | ((uint32_t)P.b_mn << 16) |
                           ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(256 >> 4) << 24);
    const uint64_t ka = k_step(P.a_mn), kb_ = k_step(P.b_mn);
    const uint64_t a0 = box_desc(smem_u32(smem), P.a_mn), b0 = box_desc(smem_u32(smem) + 2 * BOX, P.b_mn);
    uint64_t ad = a0, bd = b0;
    uint32_t s = 0, ph = 0, acc_it = 0;
    bool alive = true;
    for (int item = item0; item < total && alive; item += step) {
      const uint32_t a = acc_it & 1, d = tmem_base + a * 256;
      if (!mbar_wait(&aux->tmem_empty[a], ((acc_it >> 1) & 1) ^ 1, P.status, P.wait_ns)) break;
      tc_fence_after();
#pragma unroll 1
      for (int kb = 0; kb < P.KB; ++kb) {
        if (!mbar_wait(&aux->full[s], ph, P.status, P.wait_ns)) { alive = false; break; }
        tc_fence_after();
        if (leader) {
#pragma unroll
          for (int k4 = 0; k4 < 4; ++k4) tc_mma_pair<MMA_F16>(d, ad + k4 * ka, bd + k4 * kb_, idesc, kb > 0 || k4 > 0 ? 1u : 0u);
          tc_commit_pair(&aux->empty[s]);
        }
        ad += (uint64_t)(stage >> 4);
        bd += (uint64_t)(stage >> 4);
        if (++s == (uint32_t)stages) { s = 0; ad = a0; bd = b0; ph ^= 1; }
      }
      if (leader && alive) tc_commit_pair(&aux->tmem_full[a]);
      ++acc_it;
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------ epilogue: a thread has 32 columns of one row at a time
    const int h = (warp - 4) >> 2, wq = warp & 3;
    const uint32_t t_lane = tmem_base + ((uint32_t)(wq << 5) << 16);
    uint32_t acc_it = 0;
    const T* res = reinterpret_cast<const T*>(E.residual);
    T *y = reinterpret_cast<T*>(E.y), *z = reinterpret_cast<T*>(E.z);
    float* zf = reinterpret_cast<float*>(E.z);  // of a gated call
    const bool y16 = pieces(y, E.y_ld, 16), y32 = pieces(y, E.y_ld, 32), r16 = pieces(res, E.residual_ld, 16);
    const bool z16 = P.gate ? pieces(zf, E.z_ld, 16) && E.N % 4 == 0 : pieces(z, E.z_ld, 16);
    const bool z32 = P.gate ? pieces(zf, E.z_ld, 32) && E.N % 8 == 0 : pieces(z, E.z_ld, 32);
    Rows R;
    R.end = P.rows;
    R.stage = reinterpret_cast<float*>(smem + kPairRing) + (warp - 4) * 32 * kStagePitch;
    R.lane = lane;
    for (int item = item0; item < total; item += step) {
      const uint32_t a = acc_it & 1;
      if (!warp_agrees(mbar_wait_idle(&aux->tmem_full[a], (acc_it >> 1) & 1, P.status, P.wait_ns))) break;
      tc_fence_after();
      int rt, ct;
      tile_at(item, RT, CT, P.group, rt, ct);
      R.m0 = (int64_t)rt * 256 + cr * 128 + wq * 32;
      const int span = out_cols / 2;  // columns of this warp
#pragma unroll 1
      for (int q = 0; q < span; q += 32) {
        const int in = h * span + q;
        R.n0 = ct * out_cols + in;
        if (R.n0 >= P.cols || R.m0 >= R.end) break;
        R.n = (int)(P.cols - R.n0 < 32 ? P.cols - R.n0 : 32);
        // a lane reads one column's bias and hands it round: 32 loads of every lane were the epilogue's longest part (4096 x 2048 ->
        // 4096 with gelu_tanh and a bias, z kept, 96 -> 55 us)
        const float b0 = lane < R.n ? bias_at<T>(E, R.n0 + lane) : 0.0f;
        uint32_t r0[32], r1[32];
        tmem_ld32_async(t_lane + a * 256 + (uint32_t)in, r0);
        if (P.gate) tmem_ld32_async(t_lane + a * 256 + (uint32_t)(BN / 2 + in), r1);
        tmem_wait32(r0);
        if (P.gate) tmem_wait32(r1);
        float v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r0[i]);
        if (E.bias) {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] += __shfl_sync(0xFFFFFFFFu, b0, i);
        }
        if (P.gate) {
          float u[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) u[i] = __uint_as_float(r1[i]);
          if (E.bias) {
            const float b1 = lane < R.n ? bias_at<T>(E, E.N + R.n0 + lane) : 0.0f;
#pragma unroll
            for (int i = 0; i < 32; ++i) u[i] += __shfl_sync(0xFFFFFFFFu, b1, i);
          }
          if (zf) {
            store_rows<float>(zf, E.z_ld, z16, z32, R, v);
            store_rows<float>(zf + E.N, E.z_ld, z16, z32, R, u);
          }
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = v[i] * sigmoid<T>(v[i]) * u[i];
        } else {
          if (z) {
            if (E.act == MOE_LIN_RELU) store_rows<T, AsKeptSign>(z, E.z_ld, z16, z32, R, v);
            else store_rows<T, AsKept>(z, E.z_ld, z16, z32, R, v);
          }
          switch (E.act) {  // one loop each: the choice is the call's
            case MOE_LIN_NONE: break;
            case MOE_LIN_RELU:
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = act_value<T>(MOE_LIN_RELU, v[i]);
              break;
            case MOE_LIN_SILU:
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = act_value<T>(MOE_LIN_SILU, v[i]);
              break;
            case MOE_LIN_GELU:
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = act_value<T>(MOE_LIN_GELU, v[i]);
              break;
            default:
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = act_value<T>(MOE_LIN_GELU_TANH, v[i]);
          }
        }
        if (res) {
          float t[32];
          load_rows<T>(res, E.residual_ld, r16, R, t);
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] += t[i];
        }
        store_rows<T>(y, E.y_ld, y16, y32, R, v);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (cr == 1) mbar_arrive_remote(&aux->tmem_empty[a], 0);
        else mbar_arrive(&aux->tmem_empty[a]);
      }
      ++acc_it;
    }
  }
  // -------------------------------------------------------------------- teardown
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // no CTA leaves while its partner may still signal its barriers
  if (warp == 2) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512));
  }
}

// ------------------------------------------------------------------ fp32 operands
// Tiles of D of TM rows and T columns, RM x 8 outputs to a thread (tiles of 32: 4 x 4), 16 k at a time out of a ring in shared memory that asynchronous
// copies fill (each element to its place, which transposes operands with rows of k; whole 16-byte pieces where rows of r or c allow
// it); K divided over a cluster as in tile_kernel.  Half of a gated call's columns are gates, the other half the ups that go with
// them.  A copy is an address and an instruction for every element, and a tile of 128 x 128 has half as many for a product as one
// of 64 x 64.
struct F32Operand {
  const float* p;
  int64_t rs, ks;  // strides of the row (r or c) and of k, one of them 1
  int wide;        // rows of r or c in whole 16-byte pieces
};
constexpr int FSTAGES = 3;
__device__ __forceinline__ void cp_async4_or_zero(uint32_t dst, const void* src, bool yes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(yes ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// ROWS x 16 elements from (base, k0) on; zeros beyond `end` and `kend`.  gate: rows from ROWS / 2 on lie that far behind the first
template <int ROWS, int FTHREADS, int FPITCH>
__device__ __forceinline__ void f32_fill(const F32Operand& X, int64_t base, int64_t end, int64_t gate, int64_t k0, int64_t kend, uint32_t dst) {
  constexpr int ROUND = FTHREADS / 16;  // rows of a round of copies
  const int t = threadIdx.x;
  if (X.ks == 1) {
    const int k = t & 15;
    const bool in = k0 + k < kend;
    dst += (uint32_t)(k * FPITCH + (t >> 4)) * 4;
    const float* p = X.p + (base + (t >> 4)) * X.rs + k0 + k;
    int64_t left = end - base - (t >> 4);  // rows that are there from this thread's first on
    const int64_t step = ROUND * X.rs;
    if (end - base >= (gate != 0 ? ROWS / 2 : ROWS) && k0 + 16 <= kend) {  // all there: an address and a copy each
#pragma unroll
      for (int i = 0; i < ROWS / ROUND; ++i) {
        if (gate != 0 && i == ROWS / ROUND / 2) p += (gate - ROWS / 2) * X.rs;
        cp_async4(dst + 4 * ROUND * i, p);
        p += step;
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < ROWS / ROUND; ++i) {
      if (gate != 0 && i == ROWS / ROUND / 2) {
        p += (gate - ROWS / 2) * X.rs;
        left += ROWS / 2;
      }
      const bool yes = in && left > 0;
      cp_async4_or_zero(dst + 4 * ROUND * i, yes ? p : X.p, yes);
      p += step;
      left -= ROUND;
    }
  } else if (X.wide) {
    constexpr int LANES = ROWS / 4, PER = FTHREADS / LANES;  // pieces of a k, k of a round
#pragma unroll
    for (int i = 0; i < (16 + PER - 1) / PER; ++i) {
      const int k = t / LANES + PER * i, r = (t % LANES) * 4;
      if (k >= 16) break;
      const int64_t left = k0 + k < kend ? end - base - r : 0;
      const int bytes = left >= 4 ? 16 : (left > 0 ? (int)left * 4 : 0);
      cp_async16_or_zero(dst + (uint32_t)(k * FPITCH + r) * 4, bytes ? X.p + (k0 + k) * X.ks + base + r : X.p, bytes);
    }
  } else {
    constexpr int PER = FTHREADS / ROWS;
    const int r = t % ROWS;
    const bool in = base + r < end;
#pragma unroll
    for (int i = 0; i < 16 / PER; ++i) {
      const int k = t / ROWS + PER * i;
      const bool yes = in && k0 + k < kend;
      cp_async4_or_zero(dst + (uint32_t)(k * FPITCH + r) * 4, yes ? X.p + (k0 + k) * X.ks + base + r : X.p, yes);
    }
  }
}
// four neighbours of thread i's, and of eight the other four `half` behind them
template <int N>
__device__ __forceinline__ void take(const float* row, int i, int half, float (&v)[N]) {
#pragma unroll
  for (int q = 0; q < N; q += 4) {
    const float4 p = *reinterpret_cast<const float4*>(row + q / 4 * half + 4 * i);
    v[q] = p.x; v[q + 1] = p.y; v[q + 2] = p.z; v[q + 3] = p.w;
  }
}
template <int RM, int T, int FTHREADS>
__global__ void __launch_bounds__(FTHREADS, T == 32 ? 12 : (T == 64 ? 7 : 2)) f32_kernel(const F32Operand A, const F32Operand B, int64_t K, const Product P, const Epilogue E) {
  extern __shared__ __align__(16) uint8_t smem_raw[];  // FSTAGES x {A, B}[16][pitch], then the partial tile
  float* s_mem = reinterpret_cast<float*>(smem_raw);
  constexpr int TM = RM == 1 ? 8 : T, CN = T == 32 ? 4 : 8, PITCH = T + 4, TILE = 16 * PITCH;  // floats of an operand's tile
  static_assert(RM == 1 ? T == 64 && FTHREADS == 64 : FTHREADS * RM * CN == T * T, "threads");
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank();
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  // a warp is 4 x 8 threads: its 16-byte pieces of a k are 64 and 128 bytes
  const int tx = T <= 64 ? (t & 7) : (warp & 1) * 8 + (lane & 7), ty = T <= 64 ? (t >> 3) : (warp >> 1) * 4 + (lane >> 3);
  const int out_cols = P.gate ? T / 2 : T;
  const int64_t r0 = (int64_t)(blockIdx.x / P.split) * TM, c0 = (int64_t)blockIdx.y * out_cols;
  const int64_t steps = (K + 15) / 16, first = steps * rank / P.split, last = steps * (rank + 1) / P.split;
  const uint32_t s0 = smem_u32(s_mem);
  float acc[RM][CN] = {};
  auto fill = [&](int64_t step, int stage) {
    if (step < last) {
      const uint32_t dst = s0 + (uint32_t)stage * (2 * TILE * 4);
      f32_fill<TM, FTHREADS, PITCH>(A, r0, P.rows, 0, step * 16, K, dst);
      f32_fill<T, FTHREADS, PITCH>(B, c0, P.cols, P.gate, step * 16, K, dst + TILE * 4);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll 1
  for (int s = 0; s < FSTAGES - 1; ++s) fill(first + s, s);
  int to = FSTAGES - 1, from = 0;
#pragma unroll 1
  for (int64_t step = first; step < last; ++step) {
    asm volatile("cp.async.wait_group %0;" ::"n"(FSTAGES - 2) : "memory");
    __syncthreads();  // this step's tiles are there, the last one's have been read
    fill(step + FSTAGES - 1, to);
    if (++to == FSTAGES) to = 0;
    const float* sa = s_mem + from * (2 * TILE);
    const float* sb = sa + TILE;
    if (++from == FSTAGES) from = 0;
#pragma unroll 4
    for (int k = 0; k < 16; ++k) {
      float av[RM], bv[CN];
      take<CN>(sb + k * PITCH, tx, T / 2, bv);
      if constexpr (RM == 1) av[0] = sa[k * PITCH + ty];
      else take<RM>(sa + k * PITCH, ty, T / 2, av);
#pragma unroll
      for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int j = 0; j < CN; ++j) acc[i][j] = fmaf(av[i], bv[j], acc[i][j]);
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
#pragma unroll
  for (int i = 0; i < RM; ++i) {
    float* part = s_mem + (RM == 1 ? ty : (i < 4 ? 4 * ty + i : T / 2 - 4 + 4 * ty + i)) * PITCH + 4 * tx;
    *reinterpret_cast<float4*>(part) = make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
    if constexpr (CN == 8) *reinterpret_cast<float4*>(part + T / 2) = make_float4(acc[i][4], acc[i][5], acc[i][6], acc[i][7]);
  }
  if (P.split > 1) cluster.sync();
  else __syncthreads();
  uint8_t* tile = reinterpret_cast<uint8_t*>(s_mem);
  switch (P.split) {
    case 1: finish_share<float, 1, FTHREADS>(cluster, tile, P, E, rank, r0, c0, TM, out_cols); break;
    case 2: finish_share<float, 2, FTHREADS>(cluster, tile, P, E, rank, r0, c0, TM, out_cols); break;
    case 4: finish_share<float, 4, FTHREADS>(cluster, tile, P, E, rank, r0, c0, TM, out_cols); break;
    default: finish_share<float, 8, FTHREADS>(cluster, tile, P, E, rank, r0, c0, TM, out_cols);
  }
  if (P.split > 1) cluster.sync();  // no CTA leaves while its partial tile may still be read
}

// ------------------------------------------------------------------ gradient of the activation, and of the bias
// dz = dy act'(z) element by element, and per block the sums over its rows of dz in fp32, before its rounding.  A warp takes 32 V
// neighbouring columns, the block's eight warps every eighth row.  HBM-bound.
struct ActGrad {
  const void *dy, *z;
  void* dz;     // null: only sums are wanted
  float* part;  // [blocks of rows, N'], null: no bias
  int64_t M, dy_ld, z_ld, dz_ld, rows_per_block;
  int N, act;
};
template <typename T, int V>
__global__ void __launch_bounds__(256) act_grad_kernel(const ActGrad P) {
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = (blockIdx.x * 32 + lane) * V;
  const int64_t m0 = (int64_t)blockIdx.y * P.rows_per_block;
  const int64_t m1 = m0 + P.rows_per_block < P.M ? m0 + P.rows_per_block : P.M;
  const bool gated = P.act == MOE_LIN_SILU_MUL, in = n < P.N;
  float s0[V] = {}, s1[V] = {};
  auto load = [](auto type, const void* base, int64_t at, float (&v)[V]) {
    using S = decltype(type);
    const S* p = reinterpret_cast<const S*>(base) + at;
    if constexpr (V == 8) load8<S>(p, v);
    else v[0] = ToF32<S>::get(*p);
  };
  auto store = [](void* base, int64_t at, const float (&v)[V]) {
    T* p = reinterpret_cast<T*>(base) + at;
    if constexpr (V == 8 && sizeof(T) == 2)
      *reinterpret_cast<uint4*>(p) = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
    else
#pragma unroll
      for (int i = 0; i < V; ++i) p[i] = from_f32<T>(v[i]);
  };
  if (in) {
#pragma unroll 2
    for (int64_t m = m0 + warp; m < m1; m += 8) {
      float dy[V], z[V];
      load(T(), P.dy, m * P.dy_ld + n, dy);
      if (gated) {
        float u[V], du[V];
        load(float(), P.z, m * P.z_ld + n, z);
        load(float(), P.z, m * P.z_ld + P.N + n, u);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float s = sigmoid<T>(z[i]), d = dy[i];
          du[i] = __fmul_rn(d, z[i] * s);  // never part of a fused sum, whoever takes dz
          dy[i] = __fmul_rn(d * u[i], s * (1.0f + z[i] * (1.0f - s)));
          s0[i] += dy[i];
          s1[i] += du[i];
        }
        if (P.dz) {
          store(P.dz, m * P.dz_ld + n, dy);
          store(P.dz, m * P.dz_ld + P.N + n, du);
        }
      } else {
        if (P.act != MOE_LIN_NONE) {
          load(T(), P.z, m * P.z_ld + n, z);
#pragma unroll
          for (int i = 0; i < V; ++i) dy[i] = __fmul_rn(dy[i], act_slope<T>(P.act, z[i]));
        }
#pragma unroll
        for (int i = 0; i < V; ++i) s0[i] += dy[i];
        if (P.dz) store(P.dz, m * P.dz_ld + n, dy);
      }
    }
  }
  if (P.part == nullptr) return;
  __shared__ float sum[8][32 * V];
  float* out = P.part + (int64_t)blockIdx.y * (gated ? 2 * P.N : P.N);
  for (int half = 0; half <= (gated ? 1 : 0); ++half) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < V; ++i) sum[warp][lane * V + i] = half ? s1[i] : s0[i];
    __syncthreads();
    const int c = blockIdx.x * 32 * V + threadIdx.x;
    if (threadIdx.x < 32 * V && c < P.N) {
      float v = sum[0][threadIdx.x];
#pragma unroll
      for (int w = 1; w < 8; ++w) v += sum[w][threadIdx.x];
      out[half * P.N + c] = v;
    }
  }
}
// the blocks' sums in order: a warp per 32 columns would read them one behind another, so eight warps take every eighth block
template <typename BT>
__global__ void __launch_bounds__(256) bias_grad_kernel(const float* part, int64_t blocks, int64_t cols, BT* db) {
  pdl_wait();
  pdl_trigger();
  __shared__ float sum[8][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  float v = 0.0f;
  if (c < cols) {
#pragma unroll 4
    for (int64_t b = warp; b < blocks; b += 8) v += part[b * cols + c];
  }
  sum[warp][lane] = v;
  __syncthreads();
  if (warp == 0 && c < cols) {
#pragma unroll
    for (int w = 1; w < 8; ++w) v += sum[w][lane];
    db[c] = from_f32<BT>(v);
  }
}

// Rows of 16-bit elements that TMA cannot read (a pitch that is no multiple of 16 bytes, an odd address) -> rows that it can.  A
// thread writes 16 bytes at a time, put together from the aligned words that hold them: the first and the last of them may
// reach beyond the row, never beyond the words that it touches.
__global__ void __launch_bounds__(256) pitch_kernel(const uint16_t* src, int64_t src_ld, int64_t rows, int64_t cols, uint16_t* dst, int64_t dst_ld) {
  pdl_wait();
  pdl_trigger();
  const int64_t pieces = dst_ld / 8, total = rows * pieces;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / pieces, c = (i - r * pieces) * 8;
    const uintptr_t at = (uintptr_t)(src + r * src_ld + c);
    const uint32_t* w = reinterpret_cast<const uint32_t*>(at & ~(uintptr_t)3);
    const int left = cols - c < 8 ? (int)(cols - c) : 8;      // elements of this piece, > 0
    const int words = (left + ((at & 2) ? 1 : 0) + 1) / 2;  // words that hold them
    uint32_t v[5];
#pragma unroll
    for (int k = 0; k < 5; ++k) v[k] = k < words ? w[k] : 0u;
    if (at & 2) {
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = __funnelshift_r(v[k], v[k + 1], 16);
    }
    *reinterpret_cast<uint4*>(dst + r * dst_ld + c) = make_uint4(v[0], v[1], v[2], v[3]);
  }
}

// ------------------------------------------------------------------ host side
struct Matrix {  // row-major in memory: `rows` rows of `cols`, `ld` apart
  const void* p;
  int64_t rows, cols, ld;
};
bool tma_reads(const Matrix& m) { return ((uintptr_t)m.p & 15) == 0 && m.ld % 8 == 0; }
int64_t padded(int64_t cols) { return (cols + 7) / 8 * 8; }
int64_t up256(int64_t b) { return (b + 255) / 256 * 256; }

// a workspace handed out front to back
struct Space {
  uint8_t* at;
  int64_t left;
  void* take(int64_t bytes) {
    bytes = up256(bytes);
    if (bytes > left) return nullptr;
    void* p = at;
    at += bytes;
    left -= bytes;
    return p;
  }
};
int readable(Matrix& m, Space& ws, cudaStream_t st) {
  if (tma_reads(m)) return 0;
  const int64_t ld = padded(m.cols);
  void* p = ws.take(m.rows * ld * 2);
  if (!p) return fail(MOE_E_BADARG, "fused_linear: workspace too small");
  const int64_t blocks = (m.rows * (ld / 8) + 255) / 256;
  const int rc = launch_pdl(pitch_kernel, dim3((unsigned)(blocks < 8 * sm_count() ? blocks : 8 * sm_count())), 256, 0, 1, st,
                            "fused_linear (pitch)", (const uint16_t*)m.p, m.ld, m.rows, m.cols, (uint16_t*)p, ld);
  m.p = p;
  m.ld = ld;
  return rc;
}

// Which kernel, tile and split of K.  Costs in clocks of an SM that moves operands at 64 bytes per clock out of L2 and multiplies
// 128 x BN x 64 in 2 BN; a whole product also moves its bytes through HBM once.
struct Plan {
  bool pair, swapped;
  int BN, split;
};
Plan choose(int64_t rows, int64_t cols, int64_t K, bool gated, bool a_mn, int sms) {
  Plan best = {false, false, 64, 1};
  double cost = 1e300;
  const int64_t kb = (K + 63) / 64;
  auto consider = [&](Plan p, double c) {
    if (c < cost) { cost = c; best = p; }
  };
  for (int swapped = 0; swapped <= 1; ++swapped) {  // D as it is, or transposed: its columns on the 128 side
    const int64_t r = swapped ? cols : rows, c = swapped ? rows : (gated ? 2 * cols : cols);
    const int rt = gated && swapped ? 64 : 128, least = swapped && !a_mn ? 16 : 64;  // a box of MN-major rows is 64 of them
    if ((r + rt - 1) / rt > 65535) continue;
    for (int bn = least; bn <= 256 && (bn == least || bn / 2 < c); bn *= 2) {
      const int64_t tiles = (r + rt - 1) / rt * ((c + bn - 1) / bn);
      for (int s = 1; s <= 8 && s <= kb; s *= 2) {
        const double reach = (s == 8 ? 112.0 : (s == 4 ? 132.0 : 148.0)) * sms / 148.0;
        const double waves = (double)(int64_t)((double)(tiles * s) / reach + 0.9999);
        const double step = (128 + bn) * 2.0;  // never below the products' 2 bn
        consider({false, swapped != 0, bn, s}, waves * (((kb + s - 1) / s) * step + 24.0 * bn + 1500.0) + 2500.0 + (s > 1 ? 1500.0 + 8.0 * bn : 0.0));
      }
    }
  }
  for (int bn = 128; bn <= 256; bn *= 2) {
    const int ct = gated ? bn / 2 : bn;
    const int64_t tiles = (rows + 255) / 256 * ((cols + ct - 1) / ct);
    const double waves = (double)((tiles + sms / 2 - 1) / (sms / 2));
    consider({true, false, bn, 1}, waves * kb * (bn == 256 ? 512.0 : 300.0) + 4000.0 + 12.0 * bn);
  }
  return best;
}

template <typename T>
int run_product(Matrix a, Matrix b, bool a_mn, bool b_mn, int64_t rows, int64_t cols, int64_t K, bool gated, const Epilogue& E,
                int32_t* status, cudaStream_t st) {
  // a, b: the operands of D [rows, cols]; a_mn: a is [K, rows] in memory.  gated: b has 2 cols rows
  Plan p = choose(rows, cols, K, gated, a_mn, sm_count());
  const CUtensorMapDataType dt = std::is_same<T, __nv_bfloat16>::value ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  Product P = {};
  P.KB = (int)((K + 63) / 64);
  P.gate = gated ? (int)cols : 0;
  P.status = status;
  P.wait_ns = wait_limit_ns();
  P.BN = p.BN;
  P.split = p.split;
  P.swapped = p.swapped;
  P.rows = p.swapped ? cols : rows;
  P.cols = p.swapped ? rows : cols;
  if (p.swapped) { Matrix t = a; a = b; b = t; const bool q = a_mn; a_mn = b_mn; b_mn = q; }
  P.a_mn = a_mn;
  P.b_mn = b_mn;
  int bbox = 64;
  if (!p.pair) bbox = gated && !p.swapped ? (p.BN / 2 < 64 ? p.BN / 2 : 64) : (p.BN < 64 ? p.BN : 64);
  CUtensorMap ma, mb;
  int rc = make_map(&ma, a.p, dt, 2, (uint64_t)a.rows, (uint64_t)a.cols, 64, p.swapped, 128, (uint64_t)a.ld);
  if (rc) return rc;
  rc = make_map(&mb, b.p, dt, 2, (uint64_t)b.rows, (uint64_t)b.cols, b_mn ? 64 : bbox, !p.swapped, 128, (uint64_t)b.ld);
  if (rc) return rc;
  if (p.pair) {
    auto kern = pair_kernel<T>;
    rc = allow_smem((const void*)kern, (int)kPairSmem);
    if (rc) return rc;
    const int ct = gated ? p.BN / 2 : p.BN;
    const int64_t RT = (rows + 255) / 256, CT = (cols + ct - 1) / ct, tiles = RT * CT;
    if (tiles >= (1ll << 31)) return fail(MOE_E_TOOBIG, "fused_linear: too many tiles");
    // 4096 x 4096 -> 2 x 14336 gated, 8192 x 4096 -> 4096: 854, 179 us with groups of one row tile, 688, 186 of 4, 667, 194 of 8, 657, 182 of
    // 16, 654, 212 of 64; of the second the runs of one size are as far apart
    P.group = 8;
    const int pairs = sm_count() / 2;
    return launch_pdl(kern, dim3((unsigned)(2 * (tiles < pairs ? tiles : pairs))), PTHREADS, kPairSmem, 2, st, "fused_linear (pair)", ma, mb, P, E);
  }
  auto kern = tile_kernel<T>;
  rc = allow_smem((const void*)kern, (int)tile_smem(kRingWhole));
  if (rc) return rc;
  while (P.split > 1 && max_clusters((const void*)kern, P.split, TTHREADS, tile_smem(kRingWhole)) == 0) P.split /= 2;
  const int rt = gated && p.swapped ? 64 : 128, ct = gated && !p.swapped ? p.BN / 2 : p.BN;
  const dim3 grid((unsigned)((P.cols + ct - 1) / ct * P.split), (unsigned)((P.rows + rt - 1) / rt));
  P.ring = p.BN <= 128 && (int64_t)grid.x * grid.y > sm_count() ? kRingHalf : kRingWhole;
  return launch_pdl(kern, grid, TTHREADS, tile_smem(P.ring), P.split, st, "fused_linear (tile)", ma, mb, P, E);
}

int run_f32(F32Operand a, F32Operand b, int64_t rows, int64_t cols, int64_t K, bool gated, const Epilogue& E, cudaStream_t st) {
  for (F32Operand* x : {&a, &b}) x->wide = ((uintptr_t)x->p & 15) == 0 && x->ks % 4 == 0;
  Product P = {};
  P.rows = rows;
  P.cols = cols;
  P.gate = gated ? (int)cols : 0;
  // Tile and split of K, by us (fitted to 18 products from 30 x 64 x 32 to 2048 x 1024 x 1024, each tile with splits of 1 to 8, to 8 %):
  // a block alone on a multiprocessor takes `alone` for each k, `full` where others hide its waiting; `last` is its outputs, which
  // the ranks of a cluster share, `next` and `ramp` what a further block of the multiprocessor adds.  32 x 32 answers soonest (300 x
  // 501 -> 333: 11.2 us, 15.5 with tiles of 64), 128 x 128 reads least (2048 x 1024 -> 1024: 114 us, 123 of 64, 172 of 32).
  struct Tile { int t; double alone, full, last, next, ramp; };
  static const Tile tiles_of[3] = {{32, 0.0353, 0.0121, 0.9, 0.0, 0.27}, {64, 0.0775, 0.0318, 4.3, 0.92, 0.36}, {128, 0.119, 0.1015, 8.9, 0.0, 4.2}};
  const int64_t sms = sm_count();
  double best = 0.0;
  int T = 64;
  P.split = 1;
  for (const Tile& tile : tiles_of) {
    const int t = tile.t, TM = rows <= 8 ? 8 : t;
    if ((rows <= 8 && t != 64) || (t == 128 && rows <= 64)) continue;
    const int64_t across = ((gated ? 2 * cols : cols) + t - 1) / t, tiles = across * ((rows + TM - 1) / TM);
    if (across > 65535) continue;
    for (int s = 1; s <= 8 && (s == 1 || K / s >= 64); s *= 2) {
      // clusters of 8 and 4 find places on some 112 and 132 of 148 multiprocessors, further ones next to them
      const int64_t reach = s == 8 ? sms * 112 / 148 : (s == 4 ? sms * 132 / 148 : sms), blocks = tiles * s;
      const double k = (double)K / s, n = blocks > reach && blocks <= sms ? 2.0 : (double)((blocks + sms - 1) / sms);
      const double cost = (s > 1 ? 1.0 : 0.0) + fmax(tile.alone, n * tile.full) * k + tile.last / s + (n - 1.0) * (tile.next / s + tile.ramp);
      if (best == 0.0 || cost < best) { best = cost; P.split = s; T = t; }
    }
  }
  P.BN = T;
  const int TM = rows <= 8 ? 8 : T;
  const int64_t ct = ((gated ? 2 * cols : cols) + T - 1) / T, rt = (rows + TM - 1) / TM;
  if (ct > 65535 || rt * P.split >= (1ll << 31)) return fail(MOE_E_TOOBIG, "fused_linear: fp32 products of at most %d columns", 65535 * 64);
  auto go = [&](auto kern, int t, int threads) {
    const int64_t ring = (int64_t)FSTAGES * 2 * 16 * (t + 4) * 4, part = (int64_t)TM * (t + 4) * 4, smem = ring > part ? ring : part;
    const int rc = allow_smem((const void*)kern, (int)smem);
    if (rc) return rc;
    while (P.split > 1 && max_clusters((const void*)kern, P.split, threads, (size_t)smem) == 0) P.split /= 2;
    // Launched behind its predecessor's end: blocks that come while it drains crowd on the multiprocessors that are free first
    // (8192 x 512 -> 512, dW: 264 us so, 159 with each multiprocessor at its share).
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rt * P.split), (unsigned)ct);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)P.split;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = P.split > 1 ? 1 : 0;
    const cudaError_t ce = cudaLaunchKernelEx(&cfg, kern, a, b, K, P, E);
    if (ce != cudaSuccess) return fail((int)ce, "fused_linear (fp32): %s", cudaGetErrorString(ce));
    return check_launch("fused_linear (fp32)");
  };
  if (TM == 8) return go(f32_kernel<1, 64, 64>, 64, 64);
  return T == 32 ? go(f32_kernel<4, 32, 64>, 32, 64) : T == 64 ? go(f32_kernel<8, 64, 64>, 64, 64) : go(f32_kernel<8, 128, 256>, 128, 256);
}

int check_sizes(int64_t M, int64_t N, int64_t K, int dtype, int act) {
  if (dtype != MOE_BF16 && dtype != MOE_F16 && dtype != MOE_F32) return fail(MOE_E_DTYPE, "fused_linear: unsupported dtype %d", dtype);
  if (act < MOE_LIN_NONE || act > MOE_LIN_SILU_MUL) return fail(MOE_E_BADARG, "fused_linear: activation %d", act);
  if (M < 0 || N <= 0 || K <= 0) return fail(MOE_E_BADARG, "fused_linear: bad extent");
  if (M > 0x3FFFFFFF || N > 0x1FFFFFFF || K > 0x3FFFFFFF) return fail(MOE_E_TOOBIG, "fused_linear: extent beyond 2^29 columns or 2^30 rows");
  return 0;
}
int64_t width(int64_t N, int act) { return act == MOE_LIN_SILU_MUL ? 2 * N : N; }
// blocks of rows of act_grad_kernel: as many as fill the GPU, at least 32 rows each
int64_t grad_rows(int64_t M, int64_t N, int V, int sms) {
  const int64_t cb = (N + 32 * V - 1) / (32 * V);
  int64_t blocks = (8 * (int64_t)sms + cb - 1) / cb;
  if (blocks > 512) blocks = 512;
  int64_t rows = (M + blocks - 1) / blocks;
  if (rows < 32) rows = 32;
  return (rows + 7) / 8 * 8;
}
template <typename T>
int run_act_grad(ActGrad G, int V, cudaStream_t st) {
  const dim3 grid((unsigned)((G.N + 32 * V - 1) / (32 * V)), (unsigned)((G.M + G.rows_per_block - 1) / G.rows_per_block));
  if (V == 8) return launch_pdl(act_grad_kernel<T, 8>, grid, 256, 0, 1, st, "fused_linear (activation's gradient)", G);
  return launch_pdl(act_grad_kernel<T, 1>, grid, 256, 0, 1, st, "fused_linear (activation's gradient)", G);
}
template <typename BT>
int run_bias_grad(const float* part, int64_t blocks, int64_t cols, void* db, cudaStream_t st) {
  return launch_pdl(bias_grad_kernel<BT>, dim3((unsigned)((cols + 31) / 32)), 256, 0, 1, st, "fused_linear (bias' gradient)", part, blocks, cols, (BT*)db);
}

}  // namespace
}  // namespace moe

extern "C" int moe_fused_linear_workspace(const void* x, int64_t x_ld, const void* w, int64_t w_ld, int dtype, int64_t M, int64_t N,
                                          int64_t K, int act, int64_t* bytes) {
  using namespace moe;
  if (const int rc = check_sizes(M, N, K, dtype, act)) return rc;
  if (!bytes) return fail(MOE_E_BADARG, "fused_linear_workspace: null pointer");
  *bytes = 0;
  if (dtype == MOE_F32) return 0;
  if (!tma_reads({x, M, K, x_ld})) *bytes += up256(M * padded(K) * 2);
  if (!tma_reads({w, width(N, act), K, w_ld})) *bytes += up256(width(N, act) * padded(K) * 2);
  return 0;
}

extern "C" int moe_fused_linear(const void* x, int64_t x_ld, const void* w, int64_t w_ld, const void* bias, int bias_dtype,
                                const void* residual, int64_t residual_ld, int dtype, int64_t M, int64_t N, int64_t K, int act, void* y,
                                int64_t y_ld, void* z, int64_t z_ld, void* workspace, int64_t workspace_bytes, int32_t* status,
                                void* stream) {
  using namespace moe;
  if (const int rc = check_sizes(M, N, K, dtype, act)) return rc;
  if (M == 0) return 0;
  if (!x || !w || !y) return fail(MOE_E_BADARG, "fused_linear: null pointer");
  if (bias && bias_dtype != dtype && bias_dtype != MOE_F32) return fail(MOE_E_DTYPE, "fused_linear: the bias has the operands' type or fp32");
  const int64_t W = width(N, act);
  if (x_ld < K || w_ld < K || y_ld < N || (residual && residual_ld < N) || (z && z_ld < W)) return fail(MOE_E_SHAPE, "fused_linear: rows overlap");
  cudaStream_t st = (cudaStream_t)stream;
  Epilogue E = {bias, residual, y, z, residual_ld, y_ld, z_ld, (int)N, act, bias_dtype == MOE_F32};
  const bool gated = act == MOE_LIN_SILU_MUL;
  if (dtype == MOE_F32) return run_f32({(const float*)x, x_ld, 1, 0}, {(const float*)w, w_ld, 1, 0}, M, N, K, gated, E, st);
  if ((uintptr_t)workspace & 15) return fail(MOE_E_BADARG, "fused_linear: the workspace must be 16-byte aligned");
  Space ws = {(uint8_t*)workspace, workspace ? workspace_bytes : 0};
  Matrix a = {x, M, K, x_ld}, b = {w, W, K, w_ld};
  if (int rc = readable(a, ws, st)) return rc;
  if (int rc = readable(b, ws, st)) return rc;
  return dtype == MOE_BF16 ? run_product<__nv_bfloat16>(a, b, false, false, M, N, K, gated, E, status, st)
                           : run_product<__half>(a, b, false, false, M, N, K, gated, E, status, st);
}

namespace moe {
namespace {
// Elements to a thread of act_grad_kernel, and its blocks of rows
struct GradPlan {
  int V;
  int64_t rows_per_block, blocks;
};
GradPlan grad_plan(const void* dy, const void* z, int64_t z_ld, const void* dz, int dtype, int64_t M, int64_t N, int act) {
  GradPlan p;
  const int64_t W = width(N, act);
  const int eb = dtype == MOE_F32 ? 4 : 2;
  auto wide = [&](const void* q, int64_t ld) { return ((uintptr_t)q & 15) == 0 && ld * eb % 16 == 0; };
  const bool z_wide = act == MOE_LIN_SILU_MUL ? ((uintptr_t)z & 15) == 0 && z_ld % 4 == 0 : act == MOE_LIN_NONE || wide(z, z_ld);
  p.V = N % 8 == 0 && wide(dy, N) && z_wide && wide(dz, W) ? 8 : 1;
  p.rows_per_block = grad_rows(M, N, p.V, sm_count());
  p.blocks = (M + p.rows_per_block - 1) / p.rows_per_block;
  return p;
}
// The parts of the backward pass' workspace, in bytes: dz, or dy where TMA cannot read it; the bias' partial sums; x and w where TMA cannot
// read them.  dy null: wherever it lies.
struct GradSpace {
  int64_t dz, part, x, w;
  int64_t all() const { return dz + part + x + w; }
};
GradSpace grad_space(const void* dy, const void* x, int64_t x_ld, const void* w, int64_t w_ld, int dtype, int64_t M, int64_t N, int64_t K, int act,
                     bool dx, bool dw, bool db) {
  GradSpace s = {};
  const int64_t W = width(N, act);
  const bool half = dtype != MOE_F32;
  if ((dx || dw) && (act != MOE_LIN_NONE || (half && (dy == nullptr || !tma_reads({dy, M, N, N}))))) s.dz = up256(M * padded(W) * (half ? 2 : 4));
  if (db) s.part = up256(((M + 31) / 32 < 512 ? (M + 31) / 32 : 512) * W * 4);
  if (half && dw && !tma_reads({x, M, K, x_ld})) s.x = up256(M * padded(K) * 2);
  if (half && dx && !tma_reads({w, W, K, w_ld})) s.w = up256(W * padded(K) * 2);
  return s;
}
}  // namespace
}  // namespace moe

extern "C" int moe_fused_linear_grad_workspace(const void* x, int64_t x_ld, const void* w, int64_t w_ld, int dtype, int64_t M, int64_t N,
                                               int64_t K, int act, int64_t* bytes) {
  using namespace moe;
  if (const int rc = check_sizes(M, N, K, dtype, act)) return rc;
  if (!bytes) return fail(MOE_E_BADARG, "fused_linear_grad_workspace: null pointer");
  *bytes = grad_space(nullptr, x, x_ld, w, w_ld, dtype, M, N, K, act, true, true, true).all();
  return 0;
}

extern "C" int moe_fused_linear_grad_workspace_of(const void* dy, const void* x, int64_t x_ld, const void* w, int64_t w_ld, int dtype, int64_t M,
                                                  int64_t N, int64_t K, int act, int dx, int dw, int db, int64_t* bytes) {
  using namespace moe;
  if (const int rc = check_sizes(M, N, K, dtype, act)) return rc;
  if (!bytes) return fail(MOE_E_BADARG, "fused_linear_grad_workspace_of: null pointer");
  *bytes = grad_space(dy, x, x_ld, w, w_ld, dtype, M, N, K, act, dx != 0, dw != 0, db != 0).all();
  return 0;
}

extern "C" int moe_fused_linear_grad(const void* dy, const void* z, int64_t z_ld, const void* x, int64_t x_ld, const void* w, int64_t w_ld,
                                     int dtype, int64_t M, int64_t N, int64_t K, int act, void* dx, void* dw, void* db, int db_dtype,
                                     void* workspace, int64_t workspace_bytes, int32_t* status, void* stream) {
  using namespace moe;
  if (const int rc = check_sizes(M, N, K, dtype, act)) return rc;
  if (M == 0) return fail(MOE_E_BADARG, "fused_linear_grad: no rows");
  const int64_t W = width(N, act);
  if (!dy || (act != MOE_LIN_NONE && !z) || (dx && !w) || (dw && !x)) return fail(MOE_E_BADARG, "fused_linear_grad: null pointer");
  if (db && db_dtype != dtype && db_dtype != MOE_F32) return fail(MOE_E_DTYPE, "fused_linear_grad: the bias has the operands' type or fp32");
  if ((x && x_ld < K) || (w && w_ld < K) || (z && z_ld < W)) return fail(MOE_E_SHAPE, "fused_linear_grad: rows overlap");
  cudaStream_t st = (cudaStream_t)stream;
  if ((uintptr_t)workspace & 15) return fail(MOE_E_BADARG, "fused_linear_grad: the workspace must be 16-byte aligned");
  Space ws = {(uint8_t*)workspace, workspace ? workspace_bytes : 0};
  const int eb = dtype == MOE_F32 ? 4 : 2;
  const bool products = dx || dw;
  const int64_t dz_ld = act == MOE_LIN_NONE ? N : padded(W);
  void* own = products && act != MOE_LIN_NONE ? ws.take(M * dz_ld * eb) : nullptr;
  if (products && act != MOE_LIN_NONE && !own) return fail(MOE_E_BADARG, "fused_linear_grad: workspace too small");
  GradPlan g = grad_plan(dy, z, z_ld, own, dtype, M, N, act);
  if (own || db) {
    ActGrad G = {dy, z, own, nullptr, M, N, z_ld, dz_ld, g.rows_per_block, (int)N, act};
    if (db) {
      G.part = (float*)ws.take(g.blocks * W * 4);
      if (!G.part) return fail(MOE_E_BADARG, "fused_linear_grad: workspace too small");
    }
    int rc = dtype == MOE_BF16 ? run_act_grad<__nv_bfloat16>(G, g.V, st) : dtype == MOE_F16 ? run_act_grad<__half>(G, g.V, st) : run_act_grad<float>(G, g.V, st);
    if (rc) return rc;
    if (db) {
      rc = db_dtype == MOE_F32 ? run_bias_grad<float>(G.part, g.blocks, W, db, st)
           : db_dtype == MOE_BF16 ? run_bias_grad<__nv_bfloat16>(G.part, g.blocks, W, db, st) : run_bias_grad<__half>(G.part, g.blocks, W, db, st);
      if (rc) return rc;
    }
  }
  if (!products) return 0;
  const void* dz = own ? own : dy;
  Epilogue E = {};
  E.act = MOE_LIN_NONE;
  if (dtype == MOE_F32) {
    if (dx) {
      E.y = dx; E.y_ld = K; E.N = (int)K;
      if (int rc = run_f32({(const float*)dz, dz_ld, 1, 0}, {(const float*)w, 1, w_ld, 0}, M, K, W, false, E, st)) return rc;
    }
    if (dw) {
      E.y = dw; E.y_ld = K; E.N = (int)K;
      if (int rc = run_f32({(const float*)dz, 1, dz_ld, 0}, {(const float*)x, 1, x_ld, 0}, W, K, M, false, E, st)) return rc;
    }
    return 0;
  }
  Matrix d = {dz, M, W, dz_ld};
  if (int rc = readable(d, ws, st)) return rc;
  auto product = [&](const Matrix& a, const Matrix& b, bool a_mn, int64_t rows, int64_t k) {
    E.y_ld = K; E.N = (int)K;
    return dtype == MOE_BF16 ? run_product<__nv_bfloat16>(a, b, a_mn, true, rows, K, k, false, E, status, st)
                             : run_product<__half>(a, b, a_mn, true, rows, K, k, false, E, status, st);
  };
  if (dx) {
    Matrix b = {w, W, K, w_ld};
    if (int rc = readable(b, ws, st)) return rc;
    E.y = dx;
    if (int rc = product(d, b, false, M, W)) return rc;
  }
  if (dw) {
    Matrix b = {x, M, K, x_ld};
    if (int rc = readable(b, ws, st)) return rc;
    E.y = dw;
    if (int rc = product(d, b, true, W, M)) return rc;
  }
  return 0;
}
