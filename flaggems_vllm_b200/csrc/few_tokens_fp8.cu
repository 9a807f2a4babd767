// fused_moe_few_tokens with e4m3 weights (128 x 128 block scales): the kernel behind few_tokens.cu's router.
//
// The shape of the work is few_tokens.cu's: every block routes the tokens for itself, the blocks share the rows of W1 of all experts,
// then those of W2.  The products run on tcgen05 here.  mma.sync has no e4m3 of its own on sm_100: the compiler converts both operands
// for every instruction, which kept the conversion unit 86 % busy and the whole at 3.8 TB/s; tcgen05 takes e4m3 from shared memory
// as TMA puts it there, and no thread touches a weight.  One instruction multiplies 128 weight rows by 16 columns, of which the
// tokens are 8; the rest is whatever lies behind them in shared memory, in accumulator columns that nobody reads.
//
// The tensor core cannot apply 128 x 128 block scales, so each 128 k go to an accumulator of their own (16 of them, 16 columns
// each), and two groups of four warps, in turn, add  accumulator * (token's scale * weight's scale)  to eight fp32 registers a lane,
// a lane being a weight row.  8 columns make that cheap; for the layer of many tokens it would not be.
//
//   W1  a tile is up to 64 outputs of one expert: their gate rows and their up rows, in boxes of 8 rows, so that a block's run of
//       outputs, a multiple of 8, reads no row twice.  What the two groups hold is joined in shared memory at the tile's end.
//   h   is rounded to the activations' type, as in the layer of many tokens, then quantised in groups of 128 by whichever block
//       adds a group's last output: once for all blocks that read it.
//   W2  a step is 128 k of all rows of the block's run (48 or 49 of 7168), one box, with the same k of h.
//
// Warps: 0 TMA, 1 MMA, 2 TMEM, 4 to 11 the two groups.  W2's first weights are on their way while W1's results are still being
// quantised and other blocks are waited for.
#include "few_tokens.cuh"

namespace moe {
namespace {
using namespace tc;

constexpr int kConsumers = 256, kThreads = 128 + kConsumers;
constexpr int kStage1 = 128 * 128;         // W1: 128 rows of 128 bytes
constexpr int kMaxStages1 = 12, kMaxStages2 = 20;
constexpr int kAccs = 16, kAccCols = 16;   // accumulators, one of 128 k each
constexpr int kJoinBytes = 2 * 128 * kTokens * 4;

struct Aux {
  uint64_t full1[kMaxStages1], empty1[kMaxStages1], full2[kMaxStages2], empty2[kMaxStages2], acc_full[kAccs], acc_empty[kAccs];
  int32_t run1[2], run2[2];
  uint32_t tmem_base;
};
struct Few8 {
  int stages1, stages2, slot2, rows2;  // bytes of a step of W2 and its h, rows of a step
  int ring;                            // bytes
};

__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kConsumers) : "memory"); }
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async;" ::: "memory"); }
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n\ttcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
      : "r"(taddr)
      : "memory");
}

// outputs [o, o + n) of a run: up to 64 of one expert
struct Tile {
  int s, n;
  int64_t p;  // the first one inside the expert
};
__device__ __forceinline__ Tile tile_at(const Few& P, int slots, int64_t o, int64_t hi) {
  const int64_t routed = (int64_t)slots * P.I;
  Tile t;
  int64_t left;
  if (o < routed) {
    t.s = (int)((uint32_t)o / (uint32_t)P.I);
    t.p = o - (int64_t)t.s * P.I;
    left = P.I - t.p;
  } else {
    t.s = slots;
    t.p = o - routed;
    left = P.Is - t.p;
  }
  if (left > hi - o) left = hi - o;
  t.n = left < 64 ? (int)left : 64;
  return t;
}

// 8 bits: a group's scale needs all of its 128 outputs, which several blocks may have made.  Whoever adds the last ones quantises the
// group, once for all blocks that read it.  The routing weights go into the scales.  Called by the consumer threads.
template <typename T>
__device__ __forceinline__ void quantise_groups(const Few& P, Shared& S, int64_t lo, int64_t hi) {
  const int tid = threadIdx.x - 128, warp = tid >> 5, lane = tid & 31;
  const int64_t last = hi > lo ? (hi - 1) / 128 : -1;
  for (int64_t first = lo / 128; first <= last; first += kMaxSlots) {
    consumers_sync();  // this block's h is written; the list has been read
    if (tid == 0) S.wholes = 0;
    consumers_sync();
    const int64_t g = first + tid;
    if (tid < kMaxSlots && g <= last) {
      const int64_t a = g * 128 > lo ? g * 128 : lo, z = (g + 1) * 128 < hi ? (g + 1) * 128 : hi;
      const int mine = (int)(z - a);
      __threadfence();
      const int old = atomicAdd(P.counters + 4 + g, mine);
      __threadfence();
      if (old + mine == 128) S.whole[atomicAdd(&S.wholes, 1)] = (int)(g - first);
    }
    consumers_sync();
    const int n = S.wholes;
    const int64_t routed = (int64_t)S.slots * P.I;
    for (int i = warp; i < n; i += kConsumers / 32) {
      const int64_t o = (first + S.whole[i]) * 128;
      int s = S.slots;
      int64_t width = P.Is, p = o - routed;
      if (o < routed) {
        s = (int)((uint32_t)o / (uint32_t)P.I);
        width = P.I;
        p = o - (int64_t)s * P.I;
      }
      const int m = lane >> 2, c = lane & 3;
      const int64_t at = (int64_t)s * kTokens * P.I + m * width + p + c * 32;
      B32 v[2], q;
      zero(v[0]);
      zero(v[1]);
      const bool mine = (S.mask[s] >> m) & 1;
      if (mine) {
        const uint4* h = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(P.h) + at);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint4 w = __ldcg(h + j);  // other blocks' stores: past L1
          uint32_t* r = v[j >> 1].r + 4 * (j & 1);
          r[0] = w.x; r[1] = w.y; r[2] = w.z; r[3] = w.w;
        }
      }
      const float scale = quantise<T>(v, q);
      if (mine) {
        const bool shared = s == S.slots;
        const int64_t to = ((shared ? 0 : (int64_t)s * kTokens) + m) * width + p;
        uint4* d = reinterpret_cast<uint4*>((shared ? P.h8_shared : P.h8) + to + c * 32);
        d[0] = make_uint4(q.r[0], q.r[1], q.r[2], q.r[3]);
        d[1] = make_uint4(q.r[4], q.r[5], q.r[6], q.r[7]);
        if (c == 0) (shared ? P.h8_scale_shared : P.h8_scale)[to / 128] = scale * S.weight[s][m];
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 1)
few_experts8_kernel(const __grid_constant__ CUtensorMap map_w1, const __grid_constant__ CUtensorMap map_w2,
                    const __grid_constant__ CUtensorMap map_sw1, const __grid_constant__ CUtensorMap map_sw2,
                    const __grid_constant__ CUtensorMap map_h, const __grid_constant__ CUtensorMap map_sh, const Few P, const Few8 Q) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = align_1024(smem_raw);
  uint8_t* xt = ring + Q.ring;                                      // the tokens, a kilobyte for each 128 k
  const int KB = P.H / 128;
  float* xs = reinterpret_cast<float*>(xt + (KB + 1) * 1024);       // their scales [KB][8]; the kilobyte between is read as columns 8 to 15
  float* join = xs + KB * kTokens;
  Shared& S = *reinterpret_cast<Shared*>(join + kJoinBytes / 4);
  Aux* aux = reinterpret_cast<Aux*>(reinterpret_cast<uint8_t*>(&S) + (sizeof(Shared) + 15) / 16 * 16);
  const int warp = __shfl_sync(0xFFFFFFFFu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kMaxStages1; ++s) { mbar_init(&aux->full1[s], 1); mbar_init(&aux->empty1[s], 1); }
    for (int s = 0; s < kMaxStages2; ++s) { mbar_init(&aux->full2[s], 1); mbar_init(&aux->empty2[s], 1); }
    for (int s = 0; s < kAccs; ++s) { mbar_init(&aux->acc_full[s], 1); mbar_init(&aux->acc_empty[s], 4); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&aux->tmem_base)), "r"(kAccs * kAccCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  // the tokens, older than the kernel in front, in 8 bits: rows of 128 bytes in the tensor core's swizzle
  for (int i0 = warp * 8; i0 < kTokens * KB; i0 += 8 * (kThreads / 32)) {  // eight groups to a warp, four lanes each
    const int i = i0 + (lane >> 2), b = i / kTokens, m = i % kTokens, c = lane & 3;
    B32 v[2], q;
    zero(v[0]);
    zero(v[1]);
    if (m < P.M) {
      const T* p = reinterpret_cast<const T*>(P.x) + m * P.x_ld + b * 128 + c * 32;
      load_row<16>(v[0], p);
      load_row<16>(v[1], p + 16);
    }
    const float s = quantise<T>(v, q);
    uint8_t* row = xt + b * 1024 + m * 128;
    *reinterpret_cast<uint4*>(row + ((2 * c) ^ m) * 16) = make_uint4(q.r[0], q.r[1], q.r[2], q.r[3]);
    *reinterpret_cast<uint4*>(row + ((2 * c + 1) ^ m) * 16) = make_uint4(q.r[4], q.r[5], q.r[6], q.r[7]);
    if (c == 0) xs[i] = m < P.M ? s : 0.0f;
  }
  prepare_route(P, S);
  pdl_wait();  // scores and cleared counters
  pdl_trigger();
  if (threadIdx.x == 0) {
    aux->run1[0] = claim(P.counters);
    aux->run2[0] = claim(P.counters + 1);
  }
  if (P.E <= 256) route<8>(P, S, reinterpret_cast<float*>(ring));
  else route<32>(P, S, reinterpret_cast<float*>(ring));
  proxy_fence();  // the tokens are read, the scores' place is written by the other side
  tc_fence_before();
  __syncthreads();
  tc_fence_after();

  const int slots = S.slots, G = gridDim.x;
  const uint32_t tmem = aux->tmem_base;
  const int64_t outputs = (int64_t)slots * P.I + P.Is, units = outputs / 8;
  const int runs1 = G, runs2 = (P.H + 63) / 64 > G ? (P.H + 63) / 64 : G;
  const int KI = P.I / 128, KS = P.Is / 128, steps = slots * KI + KS;
  constexpr uint32_t idesc = (1u << 4) | ((uint32_t)(kAccCols >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
  const bool leader = elect_lane();  // one lane of each warp
  uint32_t s1 = 0, p1 = warp == 0 ? 1 : 0;  // W1's ring: the producer's or the MMA warp's stage and parity
  uint32_t s2 = 0, p2 = warp == 0 ? 1 : 0;
  uint32_t block = 0;                        // blocks of 128 k so far: the MMA warp's and the consumers'
  int early = 0;                             // steps of W2 whose weights are on their way
  bool alive = true;
  const int group = (warp - 4) >> 2, wq = warp & 3, tid = (int)threadIdx.x - 128;
  const uint32_t t_lane = tmem + ((uint32_t)(wq << 5) << 16);

  auto load_step = [&](int run, int i, bool weights, bool h) {  // step i of a run of W2 into stage s2
    const int lo = (int)((int64_t)P.H * run / runs2);
    const bool shared = i >= slots * KI;
    const int s = shared ? slots : i / KI, kb = shared ? i - slots * KI : i - s * KI;
    uint8_t* dst = ring + (size_t)s2 * Q.slot2;
    if (weights) {
      mbar_expect_tx(&aux->full2[s2], Q.rows2 * 128 + 1024);
      tma_load_2d(shared ? &map_sw2 : &map_w2, &aux->full2[s2], dst, kb * 128, (shared ? 0 : S.list[s] * P.H) + lo);
    }
    if (h) tma_load_2d(shared ? &map_sh : &map_h, &aux->full2[s2], dst + Q.slot2 - 1024, kb * 128, shared ? 0 : s * kTokens);
  };

  // ================================================================ W1
  for (int turn = 0;; ++turn) {
    if (turn > 0) __syncthreads();
    const int run = aux->run1[turn & 1];
    if (run >= runs1) break;
    const int64_t lo = units * run / runs1 * 8, hi = units * (run + 1) / runs1 * 8;
    if (warp == 0) {
      int next = 0;
      if (lane == 0) {
        next = claim(P.counters);
        aux->run1[(turn + 1) & 1] = next;
      }
      for (int64_t o = lo; o < hi && alive;) {
        const Tile t = tile_at(P, slots, o, hi);
        const bool shared = t.s == slots;
        const int width = shared ? P.Is : P.I, boxes = t.n / 8;
        // lane 2 u + v copies box u of the gate rows (v = 0) or of the up rows
        const int row = (int)((shared ? 0 : (int64_t)S.list[t.s] * 2 * width) + t.p) + (lane >> 1) * 8 + (lane & 1) * width;
        const uint32_t to = (uint32_t)((lane & 1) * 8192 + (lane >> 1) * 1024);
        for (int kb = 0; kb < KB; ++kb) {
          if (!warp_agrees(mbar_wait(&aux->empty1[s1], p1, P.status, P.wait_ns))) { alive = false; break; }
          if (lane == 0) mbar_expect_tx(&aux->full1[s1], boxes * 2048);
          __syncwarp();
          if (lane < 2 * boxes) tma_load_2d(shared ? &map_sw1 : &map_w1, &aux->full1[s1], ring + (size_t)s1 * kStage1 + to, kb * 128, row);
          if (++s1 == (uint32_t)Q.stages1) { s1 = 0; p1 ^= 1; }
        }
        o += t.n;
      }
      next = __shfl_sync(0xFFFFFFFFu, next, 0);
      const int run2 = aux->run2[0];
      if (next >= runs1 && run2 < runs2) {
        // W2's weights take the ring as soon as W1's products have left it
        for (int d = 0; d < Q.stages1 && alive; ++d) {
          alive = warp_agrees(mbar_wait(&aux->empty1[s1], p1, P.status, P.wait_ns));
          if (++s1 == (uint32_t)Q.stages1) { s1 = 0; p1 ^= 1; }
        }
        if (alive) {
          for (; early < Q.stages2 && early < steps; ++early) {
            if (lane == 0) load_step(run2, early, true, false);
            if (++s2 == (uint32_t)Q.stages2) s2 = 0;
          }
          s2 = 0;
        }
      }
    } else if (warp == 1) {
      const uint64_t a0 = make_smem_desc(smem_u32(ring)), b0 = make_smem_desc(smem_u32(xt));
      for (int64_t o = lo; o < hi && alive;) {
        const Tile t = tile_at(P, slots, o, hi);
        for (int kb = 0; kb < KB; ++kb, ++block) {
          const uint32_t a = block % kAccs;
          if (!mbar_wait(&aux->full1[s1], p1, P.status, P.wait_ns) ||
              !mbar_wait(&aux->acc_empty[a], ((block / kAccs) & 1) ^ 1, P.status, P.wait_ns)) { alive = false; break; }
          tc_fence_after();
          tc_mma_block_f8(leader, tmem + a * kAccCols, a0 + (uint64_t)(s1 * (kStage1 >> 4)), b0 + (uint64_t)(kb * (1024 >> 4)), idesc,
                          smem_u32(&aux->acc_full[a]), smem_u32(&aux->empty1[s1]));
          if (++s1 == (uint32_t)Q.stages1) { s1 = 0; p1 ^= 1; }
        }
        o += t.n;
      }
    } else if (warp >= 4) {
      const int row = wq * 32 + lane;
      for (int64_t o = lo; o < hi;) {
        const Tile t = tile_at(P, slots, o, hi);
        const bool shared = t.s == slots;
        const int width = shared ? P.Is : P.I;
        // this lane's row of the tile (one that is not there takes the last one's scale)
        const int64_t p = t.p + ((row & 63) < t.n ? (row & 63) : t.n - 1) + (row >= 64 ? width : 0);
        const float* ws = (shared ? P.sw1s : P.w1s + (int64_t)S.list[t.s] * (2 * width / 128) * KB) + p / 128 * KB;
        float acc[kTokens] = {};
        for (int kb = 0; kb < KB; ++kb, ++block) {
          if ((int)(block & 1) != group) continue;
          const float w = __ldg(ws + kb);
          const uint32_t a = block % kAccs;
          if (alive) alive = warp_agrees(mbar_wait(&aux->acc_full[a], (block / kAccs) & 1, P.status, P.wait_ns));
          tc_fence_after();
          uint32_t r[8];
          tmem_ld8(t_lane + a * kAccCols, r);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&aux->acc_empty[a]);
          const float4 x0 = *reinterpret_cast<const float4*>(xs + kb * kTokens), x1 = *reinterpret_cast<const float4*>(xs + kb * kTokens + 4);
          const float x[kTokens] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
#pragma unroll
          for (int m = 0; m < kTokens; ++m) acc[m] = fmaf(__uint_as_float(r[m]), x[m] * w, acc[m]);
        }
        consumers_sync();  // the last tile's sums have been read
        float4* j = reinterpret_cast<float4*>(join + (group * 128 + row) * kTokens);
        j[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
        j[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
        consumers_sync();
        const uint32_t mask = S.mask[t.s];
#pragma unroll
        for (int i = 0; i < 64 * kTokens / kConsumers; ++i) {
          const int at = tid + i * kConsumers, n = at & 63, m = at >> 6;
          if (n < t.n && ((mask >> m) & 1)) {
            const float* q = join + n * kTokens + m;
            const float gate = q[0] + q[128 * kTokens], up = q[64 * kTokens] + q[192 * kTokens];
            reinterpret_cast<T*>(P.h)[(int64_t)t.s * kTokens * P.I + (int64_t)m * width + t.p + n] = from_f32<T>(silu_mul(gate, up));
          }
        }
        o += t.n;
      }
      quantise_groups<T>(P, S, lo, hi);
      proxy_fence();  // h in 8 bits is read by TMA
      consumers_sync();
      if (tid == 0) {
        __threadfence();
        atomicAdd(P.counters + 2, 1);
      }
    }
  }

  // ================================================================ W2
  bool waited = false;
  for (int turn = 0;; ++turn) {
    if (turn > 0) __syncthreads();
    const int run = aux->run2[turn & 1];
    if (run >= runs2) break;
    const int lo = (int)((int64_t)P.H * run / runs2), hi = (int)((int64_t)P.H * (run + 1) / runs2);
    if (warp == 0) {
      if (lane == 0) {
        aux->run2[(turn + 1) & 1] = claim(P.counters + 1);
        if (!waited) wait_for_runs(P.counters + 2, runs1, P.status, P.wait_ns);
        proxy_fence();
      }
      waited = true;
      __syncwarp();
      for (int i = 0; i < steps && alive; ++i) {
        if (early > 0) {
          --early;
          if (lane == 0) load_step(run, i, false, true);
        } else {
          if (!warp_agrees(mbar_wait(&aux->empty2[s2], p2, P.status, P.wait_ns))) { alive = false; break; }
          if (lane == 0) load_step(run, i, true, true);
        }
        if (++s2 == (uint32_t)Q.stages2) { s2 = 0; p2 ^= 1; }
      }
    } else if (warp == 1) {
      const uint64_t a0 = make_smem_desc(smem_u32(ring)), b0 = make_smem_desc(smem_u32(ring) + Q.slot2 - 1024);
      for (int i = 0; i < steps && alive; ++i, ++block) {
        const uint32_t a = block % kAccs;
        if (!mbar_wait(&aux->full2[s2], p2, P.status, P.wait_ns) ||
            !mbar_wait(&aux->acc_empty[a], ((block / kAccs) & 1) ^ 1, P.status, P.wait_ns)) { alive = false; break; }
        tc_fence_after();
        const uint64_t at = (uint64_t)(s2 * (uint32_t)(Q.slot2 >> 4));
        tc_mma_block_f8(leader, tmem + a * kAccCols, a0 + at, b0 + at, idesc, smem_u32(&aux->acc_full[a]), smem_u32(&aux->empty2[s2]));
        if (++s2 == (uint32_t)Q.stages2) { s2 = 0; p2 ^= 1; }
      }
    } else if (warp >= 4) {
      if (!waited) {
        waited = true;
        if (tid == 0) wait_for_runs(P.counters + 2, runs1, P.status, P.wait_ns);
        consumers_sync();
      }
      const int row = wq * 32 + lane, r0 = lo + row < hi ? lo + row : hi - 1;  // a row that is not there takes the last one's scale
      const bool rows_here = lo + wq * 32 < hi;
      float acc[kTokens] = {};
      for (int i = 0; i < steps; ++i, ++block) {
        if ((int)(block & 1) != group) continue;
        const bool shared = i >= slots * KI;
        const int s = shared ? slots : i / KI, kb = shared ? i - slots * KI : i - s * KI, K = shared ? KS : KI;
        const uint32_t mask = S.mask[s], a = block % kAccs;
        float w = 0.0f, f = 0.0f;
        if (rows_here) {
          w = __ldg((shared ? P.sw2s : P.w2s + (int64_t)S.list[s] * KB * K) + (int64_t)(r0 / 128) * K + kb);
          if (lane < kTokens && ((mask >> lane) & 1))
            f = __ldcg((shared ? P.h8_scale_shared : P.h8_scale + (int64_t)s * kTokens * K) + lane * K + kb);
        }
        if (alive) alive = warp_agrees(mbar_wait(&aux->acc_full[a], (block / kAccs) & 1, P.status, P.wait_ns));
        tc_fence_after();
        uint32_t r[8];
        if (rows_here) tmem_ld8(t_lane + a * kAccCols, r);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&aux->acc_empty[a]);
        if (rows_here) {
#pragma unroll
          for (int m = 0; m < kTokens; ++m) {
            const float fm = __shfl_sync(0xFFFFFFFFu, f, m);
            // a token that is not the expert's takes nothing, whatever the weights and its place hold
            if ((mask >> m) & 1) acc[m] = fmaf(__uint_as_float(r[m]), fm * w, acc[m]);
          }
        }
      }
      consumers_sync();
      if (row < 64) {
        float4* j = reinterpret_cast<float4*>(join + (group * 64 + row) * kTokens);
        j[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
        j[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
      }
      consumers_sync();
#pragma unroll
      for (int i = 0; i < 64 * kTokens / kConsumers; ++i) {
        const int at = tid + i * kConsumers, n = at & 63, m = at >> 6;
        if (lo + n < hi && m < P.M) {
          float v = join[n * kTokens + m] + join[(64 + n) * kTokens + m];
          if (P.residual) v += ToF32<T>::get(reinterpret_cast<const T*>(P.residual)[m * P.residual_ld + lo + n]);
          reinterpret_cast<T*>(P.out)[(int64_t)m * P.H + lo + n] = from_f32<T>(v);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kAccs * kAccCols));
  }
}

constexpr int64_t fixed_bytes(int64_t H) {
  return 1024 + (H / 128 + 1) * 1024 + H / 128 * kTokens * 4 + kJoinBytes + (int64_t)(sizeof(Shared) + 15) / 16 * 16 + (int64_t)sizeof(Aux);
}
static_assert(fixed_bytes(kMaxHidden8) + 4 * kStage1 <= kFewSmem, "four stages at the largest hidden size");
static_assert(4 * kStage1 >= kTokens * kMaxExperts * 4, "the scores of a softmax take the ring's place");
// the tensor core reads 128 rows from a step of W2 that holds fewer: what lies behind the ring is as long
static_assert(kJoinBytes + (int64_t)sizeof(Shared) >= kStage1, "reads behind the last step stay in shared memory");

template <typename T>
int launch(const CUtensorMap (&m)[6], const Few& P, const Few8& Q, int G, cudaStream_t st) {
  auto kern = few_experts8_kernel<T>;
  const int rc = allow_smem((const void*)kern, (int)kFewSmem);
  if (rc) return rc;
  return launch_pdl(kern, dim3((unsigned)G), kThreads, (size_t)(fixed_bytes(P.H) + Q.ring), 1, st, "fused_moe_few_tokens (fp8)", m[0], m[1], m[2],
                    m[3], m[4], m[5], P, Q);
}

}  // namespace

int few_experts_fp8(const Few& P, int dtype, cudaStream_t st) {
  const int G = sm_count();
  const int64_t slots = (int64_t)P.M * P.topk < P.E ? (int64_t)P.M * P.topk : P.E;
  if ((int64_t)P.E * 2 * P.I >= (1ll << 31) || (int64_t)P.E * P.H >= (1ll << 31)) return fail(MOE_E_TOOBIG, "fused_moe_few_tokens: extent exceeds int32 coordinates");
  Few8 Q;
  const int runs2 = (P.H + 63) / 64 > G ? (P.H + 63) / 64 : G;
  Q.rows2 = (P.H + runs2 - 1) / runs2;
  Q.slot2 = (Q.rows2 * 128 + 1023) / 1024 * 1024 + 1024;
  const int64_t n1 = (kFewSmem - fixed_bytes(P.H)) / kStage1;
  Q.stages1 = (int)(n1 < kMaxStages1 ? n1 : kMaxStages1);
  Q.ring = Q.stages1 * kStage1;
  const int n2 = Q.ring / Q.slot2;
  Q.stages2 = n2 < kMaxStages2 ? n2 : kMaxStages2;
  CUtensorMap m[6];
  const CUtensorMapDataType u8 = CU_TENSOR_MAP_DATA_TYPE_UINT8;
  const bool shared = P.Is > 0;
  int rc = tc::make_map(&m[0], P.w1, u8, 1, (uint64_t)P.E * 2 * P.I, (uint64_t)P.H, 8, true);
  if (!rc) rc = tc::make_map(&m[1], P.w2, u8, 1, (uint64_t)P.E * P.H, (uint64_t)P.I, (uint32_t)Q.rows2, true);
  if (!rc) rc = shared ? tc::make_map(&m[2], P.sw1, u8, 1, (uint64_t)2 * P.Is, (uint64_t)P.H, 8, true) : (m[2] = m[0], 0);
  if (!rc) rc = shared ? tc::make_map(&m[3], P.sw2, u8, 1, (uint64_t)P.H, (uint64_t)P.Is, (uint32_t)Q.rows2, true) : (m[3] = m[1], 0);
  if (!rc) rc = tc::make_map(&m[4], P.h8, u8, 1, (uint64_t)slots * kTokens, (uint64_t)P.I, kTokens, false);
  if (!rc) rc = shared ? tc::make_map(&m[5], P.h8_shared, u8, 1, kTokens, (uint64_t)P.Is, kTokens, false) : (m[5] = m[4], 0);
  if (rc) return rc;
  return dtype == MOE_BF16 ? launch<__nv_bfloat16>(m, P, Q, G, st) : launch<__half>(m, P, Q, G, st);
}

}  // namespace moe
