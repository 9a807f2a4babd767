// fused_moe_few_tokens with e4m3 weights (128 x 128 block scales): the kernel behind few_tokens.cu's router.
//
// The shape of the work is few_tokens.cu's: every block routes the tokens for itself, the blocks share the rows of W1 of all experts,
// then those of W2.  The products run on tcgen05 here.  mma.sync has no e4m3 of its own on sm_100: the compiler converts both operands
// for every instruction, which kept the conversion unit 86 % busy and the whole at 3.8 TB/s; tcgen05 takes e4m3 from shared memory
// as TMA puts it there, and no thread touches a weight.  One instruction multiplies 128 weight rows by 16 columns, of which the
// tokens are 8; the rest is whatever lies behind them in shared memory, in accumulator columns that nobody reads.
//
// The tensor core cannot apply 128 x 128 block scales, so each 128 k go to an accumulator of their own, and two groups of four warps,
// in turn, add  accumulator * (token's scale * weight's scale)  to eight fp32 registers a lane, a lane being a weight row.  8 columns
// make that cheap; for the layer of many tokens it would not be.
//
//   W1  a tile is up to 64 outputs: their gate rows and their up rows, in units of 8, so that a block's run of outputs, a multiple
//       of 8, reads no row twice.  What the two groups hold is joined in shared memory at the tile's end.
//   h   is rounded to the activations' type, as in the layer of many tokens, then quantised in groups of 128 by whichever block
//       adds a group's last output: once for all blocks that read it.
//   W2  a K block of all rows of the block's run (48 or 49 of 7168) is one box, with the same k of h.
//
// Warps: 0 and 3 TMA, in turn, 1 MMA, 2 TMEM, 4 to 11 the two groups.  W2's first weights are on their way while W1's results are
// still being quantised and other blocks are waited for.
#include "few_tokens.cuh"

namespace moe {
namespace {
using namespace tc;

constexpr int kConsumers = 256, kThreads = 128 + kConsumers;
// A stage is what one wait, one commit and one turn of a group of consumers are for: each of these costs its thread 100 to 200 clocks
// whatever it is for, and an instruction of TMA another 90 (one K block a stage and boxes of 8 rows: 2.9 TB/s, bound by the
// thread that issues them).
constexpr int kBlocks1 = 2, kBlocks2 = 4;  // K blocks of 128 in a stage of W1, of W2
constexpr int kStage1 = kBlocks1 * 128 * 128;
constexpr int kMaxStages = 12;
constexpr int kAccs = 8, kAccCols = 16, kAccBlocks = kBlocks1 > kBlocks2 ? kBlocks1 : kBlocks2;  // a stage's blocks, 16 columns each
constexpr int kJoinBytes = 2 * 128 * kTokens * 4;

struct Aux {
  uint64_t full1[kMaxStages], empty1[kMaxStages], full2[kMaxStages], empty2[kMaxStages], acc_full[kAccs], acc_empty[kAccs];
  int32_t run1[2], run2[2], more1;
  uint32_t tmem_base;
};
struct Few8 {
  int stages1, stages2, slot2;  // bytes of a stage of W2: its blocks' rows, then their h
  int rows2, block2;            // rows of a block of W2, and its bytes, a multiple of 1024
  int ring;                     // bytes
};
// W1 as (128 bytes of k, 8 rows, K block, gate / up, 8 rows' unit): a box of 8, 4, 2 or 1 units holds what a tile's outputs need
struct Maps {
  CUtensorMap w1[4], sw1[4], w2, sw2, h, sh;
};

// a K block's products, by the lane where `yes`, into a fresh accumulator
__device__ __forceinline__ void mma_block(bool yes, uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred l, f, t;\n\t.reg .b64 a1, a2, a3, b1, b2, b3;\n\t"
      "setp.ne.b32 l, %0, 0;\n\tsetp.ne.b32 f, 0, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"
      "add.s64 a1, %2, 2;\n\tadd.s64 a2, %2, 4;\n\tadd.s64 a3, %2, 6;\n\t"
      "add.s64 b1, %3, 2;\n\tadd.s64 b2, %3, 4;\n\tadd.s64 b3, %3, 6;\n\t"
      "@l tcgen05.mma.cta_group::1.kind::f8f6f4 [%1], %2, %3, %4, f;\n\t"
      "@l tcgen05.mma.cta_group::1.kind::f8f6f4 [%1], a1, b1, %4, t;\n\t"
      "@l tcgen05.mma.cta_group::1.kind::f8f6f4 [%1], a2, b2, %4, t;\n\t"
      "@l tcgen05.mma.cta_group::1.kind::f8f6f4 [%1], a3, b3, %4, t;\n\t}"
      ::"r"((uint32_t)yes), "r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d(const CUtensorMap* map, uint64_t* bar, void* dst, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
               ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}
__device__ __forceinline__ void tma_load_5d(const CUtensorMap* map, uint64_t* bar, void* dst, int c0, int c1, int c2, int c3, int c4) {
  asm volatile("cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
               ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4)
               : "memory");
}

__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kConsumers) : "memory"); }
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async;" ::: "memory"); }
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n\ttcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
      : "r"(taddr)
      : "memory");
}

// An output of all experts' W1: its expert, its place there
struct Output {
  int s, p, width;
};
__device__ __forceinline__ Output output_at(const Few& P, int slots, int64_t o) {
  const int64_t routed = (int64_t)slots * P.I;
  if (o >= routed) return {slots, (int)(o - routed), P.Is};
  const int s = (int)((uint32_t)o / (uint32_t)P.I);
  return {s, (int)(o - (int64_t)s * P.I), P.I};
}
// Outputs of a tile that begins at o: a run is cut into equal tiles of at most 64, whatever experts they are of (every expert takes
// the same tokens).  With tiles of one expert each, a run over a border had one tile more, whose small stages bring few bytes:
// 47 us for W1 where the other blocks took 39.
__device__ __forceinline__ int tile_size(int64_t o, int64_t hi) {
  const int units = (int)((hi - o) / 8 < 1 << 20 ? (hi - o) / 8 : 1 << 20), tiles = (units + 7) / 8;
  return (units + tiles - 1) / tiles * 8;
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
few_experts8_kernel(const __grid_constant__ Maps maps, const Few P, const Few8 Q) {
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
    for (int s = 0; s < kMaxStages; ++s) {
      mbar_init(&aux->full1[s], 1);
      mbar_init(&aux->empty1[s], 1);
      mbar_init(&aux->full2[s], 1);
      mbar_init(&aux->empty2[s], 1);
    }
    for (int s = 0; s < kAccs; ++s) { mbar_init(&aux->acc_full[s], 1); mbar_init(&aux->acc_empty[s], 4); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&aux->tmem_base)), "r"(kAccs * kAccBlocks * kAccCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  // the tokens, older than the kernel in front, in 8 bits: rows of 128 bytes in the tensor core's swizzle
  for (int i = threadIdx.x; i < KB * (kTokens - P.M) * 8; i += kThreads) {  // the others' places: zeros
    const int q = i & 7, r = (i >> 3) % (kTokens - P.M) + P.M, b = (i >> 3) / (kTokens - P.M);
    *reinterpret_cast<uint4*>(xt + b * 1024 + r * 128 + q * 16) = make_uint4(0, 0, 0, 0);
    if (q == 0) xs[b * kTokens + r] = 0.0f;
  }
  const int groups = P.M * KB;
  for (int i0 = warp * 8; i0 < groups; i0 += 8 * (kThreads / 32)) {  // eight groups to a warp, four lanes each
    const int i = i0 + (lane >> 2), b = i / P.M, m = i - b * P.M, c = lane & 3;
    B32 v[2], q;
    zero(v[0]);
    zero(v[1]);
    if (i < groups) {
      const T* p = reinterpret_cast<const T*>(P.x) + m * P.x_ld + b * 128 + c * 32;
      load_row<16>(v[0], p);
      load_row<16>(v[1], p + 16);
    }
    const float s = quantise<T>(v, q);
    if (i < groups) {
      uint8_t* row = xt + b * 1024 + m * 128;
      *reinterpret_cast<uint4*>(row + ((2 * c) ^ m) * 16) = make_uint4(q.r[0], q.r[1], q.r[2], q.r[3]);
      *reinterpret_cast<uint4*>(row + ((2 * c + 1) ^ m) * 16) = make_uint4(q.r[4], q.r[5], q.r[6], q.r[7]);
      if (c == 0) xs[b * kTokens + m] = s;
    }
  }
  prepare_route(P, S);
  pdl_wait();  // scores and cleared counters
  pdl_trigger();
  if (threadIdx.x == kThreads - 32) {  // of a warp that has no token to route
    aux->run1[0] = claim(P.counters);
    aux->run2[0] = claim(P.counters + 1);
  }
  if (P.E <= 256) route<8>(P, S, reinterpret_cast<uint32_t*>(ring));
  else route<32>(P, S, reinterpret_cast<uint32_t*>(ring));
  proxy_fence();  // the tokens are read, the place of the routing is written by the other side
  tc_fence_before();
  __syncthreads();
  tc_fence_after();

  const int slots = S.slots, G = gridDim.x;
  const uint32_t tmem = aux->tmem_base;
  const int64_t outputs = (int64_t)slots * P.I + P.Is, units = outputs / 8;
  const int runs1 = G, runs2 = (P.H + 63) / 64 > G ? (P.H + 63) / 64 : G;
  const int KI = P.I / 128, KS = P.Is / 128;
  const int BI = (KI + kBlocks2 - 1) / kBlocks2, BS = (KS + kBlocks2 - 1) / kBlocks2, steps = slots * BI + BS;  // stages of a run of W2
  constexpr uint32_t idesc = (1u << 4) | ((uint32_t)(kAccCols >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
  constexpr uint32_t idesc2 = (1u << 4) | ((uint32_t)(kAccCols >> 3) << 17) | ((uint32_t)(64 >> 4) << 24);
  const bool leader = elect_lane();  // one lane of each warp
  const bool producer = warp == 0 || warp == 3;
  const uint32_t mine = warp == 3;          // the two producers take every other stage
  uint32_t s1 = 0, p1 = producer ? 1 : 0;    // W1's ring: a producer's or the MMA warp's stage and parity
  uint32_t s2 = 0, p2 = producer ? 1 : 0;
  uint32_t filled = 0;                       // stages so far: the producers'
  uint32_t batch = 0;                        // stages so far: the MMA warp's and the consumers'
  int early = 0;                             // stages of W2 whose weights are on their way
  bool alive = true;
  const int group = (warp - 4) >> 2, wq = warp & 3, tid = (int)threadIdx.x - 128;
  const uint32_t t_lane = tmem + ((uint32_t)(wq << 5) << 16);
  auto acc_at = [](uint32_t n) { return n % kAccs * (kAccBlocks * kAccCols); };

  // The accumulators of four stages at a time: each group empties its own in order, so the last one of either stands for those before.
  auto room_for = [&](uint32_t n) {
    if (n % 4 != 0) return true;
    for (uint32_t i = n + 2; i < n + 4; ++i)
      if (!mbar_wait(&aux->acc_empty[i % kAccs], ((i / kAccs) & 1) ^ 1, P.status, P.wait_ns)) return false;
    return true;
  };
  // stage i of a run of W2: expert and K blocks
  struct Step {
    int s, kb, n;
    bool shared;
  };
  auto step_at = [&](int i) {
    Step e;
    e.shared = i >= slots * BI;
    e.s = e.shared ? slots : i / BI;
    e.kb = (e.shared ? i - slots * BI : i - e.s * BI) * kBlocks2;
    const int left = (e.shared ? KS : KI) - e.kb;
    e.n = left < kBlocks2 ? left : kBlocks2;
    return e;
  };
  auto load_step = [&](int lo, int i, bool weights, bool h) {  // into stage s2
    const Step e = step_at(i);
    uint8_t* dst = ring + (size_t)s2 * Q.slot2;
    if (weights) {
      const int row = (e.shared ? 0 : S.list[e.s] * P.H) + lo;
      mbar_expect_tx(&aux->full2[s2], e.n * Q.rows2 * 128 + kBlocks2 * 1024);
      for (int j = 0; j < e.n; ++j) tma_load_2d(e.shared ? &maps.sw2 : &maps.w2, &aux->full2[s2], dst + j * Q.block2, (e.kb + j) * 128, row);
    }
    if (h) tma_load_3d(e.shared ? &maps.sh : &maps.h, &aux->full2[s2], dst + kBlocks2 * Q.block2, 0, e.shared ? 0 : e.s * kTokens, e.kb);
  };

  // ================================================================ W1
  for (int turn = 0;; ++turn) {
    if (turn > 0) __syncthreads();
    const int run = aux->run1[turn & 1];
    if (run >= runs1) break;
    const int64_t lo = units * run / runs1 * 8, hi = units * (run + 1) / runs1 * 8;
    if (producer) {
      int next = 0;
      if (warp == 0 && leader) {
        next = claim(P.counters);
        aux->run1[(turn + 1) & 1] = next;
      }
      for (int64_t o = lo; o < hi && alive;) {
        const int n = tile_size(o, hi);
        // boxes of 8, 4, 2 or 1 units of the first expert, then of the next (an expert has 16 units at least)
        const Output f = output_at(P, slots, o);
        const int all = n / 8, n0 = (f.width - f.p) / 8 < all ? (f.width - f.p) / 8 : all;
        auto boxes = [&](uint8_t* dst, uint64_t* bar, int kb, int s, int p, int count) {
          const CUtensorMap* map = s == slots ? maps.sw1 : maps.w1;
          int unit = (int)(((s == slots ? 0 : (int64_t)S.list[s] * 2 * P.I) + p) / 8);
#pragma unroll
          for (int z = 0; z < 4; ++z) {
            if (count & (8 >> z)) {
              tma_load_5d(map + z, bar, dst, 0, 0, kb, 0, unit);
              dst += (8 >> z) * (2 * kBlocks1 * 1024);
              unit += 8 >> z;
            }
          }
        };
        for (int kb = 0; kb < KB; kb += kBlocks1) {
          const bool turns = (filled++ & 1) == mine;
          if (turns && !mbar_wait(&aux->empty1[s1], p1, P.status, P.wait_ns)) { alive = false; break; }
          if (turns && leader) {
            uint8_t* dst = ring + (size_t)s1 * kStage1;
            mbar_expect_tx(&aux->full1[s1], all * (2 * kBlocks1 * 1024));
            boxes(dst, &aux->full1[s1], kb, f.s, f.p, n0);
            if (n0 < all) boxes(dst + n0 * (2 * kBlocks1 * 1024), &aux->full1[s1], kb, f.s + 1, 0, all - n0);
          }
          if (++s1 == (uint32_t)Q.stages1) { s1 = 0; p1 ^= 1; }
        }
        o += n;
      }
      // W2's weights take the ring as soon as W1's products have left it.  Which run of W2 it will be is known from the start; whether
      // another one of W1 comes first, both producers hear from the one that claimed it.
      if (warp == 0 && leader) aux->more1 = next < runs1;
      __syncwarp();  // a wait that gave up may have ended for some lanes first
      asm volatile("bar.sync 2, 64;" ::: "memory");
      const int run2 = aux->run2[0];
      if (!aux->more1 && run2 < runs2) {
        for (int d = 0; d < Q.stages1 && alive; ++d) {
          if (!mbar_wait(&aux->empty1[s1], p1, P.status, P.wait_ns)) alive = false;
          if (++s1 == (uint32_t)Q.stages1) { s1 = 0; p1 ^= 1; }
        }
        if (alive) {
          filled = 0;
          for (; early < Q.stages2 && early < steps; ++early) {
            if ((early & 1) == mine && leader) load_step((int)((int64_t)P.H * run2 / runs2), early, true, false);
            if (++s2 == (uint32_t)Q.stages2) s2 = 0;
          }
          s2 = 0;
        }
      }
    } else if (warp == 1) {
      // the eight-row groups of a tile are kBlocks1 kilobytes apart
      const uint64_t a0 = (make_smem_desc(smem_u32(ring)) & ~((uint64_t)0x3FFF << 32)) | (uint64_t)(kBlocks1 * 1024 >> 4) << 32;
      const uint64_t b0 = make_smem_desc(smem_u32(xt));
      for (int64_t o = lo; o < hi && alive;) {
        for (int kb = 0; kb < KB; kb += kBlocks1, ++batch) {
          const uint32_t a = batch % kAccs;
          if (!room_for(batch) || !mbar_wait(&aux->full1[s1], p1, P.status, P.wait_ns)) { alive = false; break; }
          tc_fence_after();
#pragma unroll
          for (int j = 0; j < kBlocks1; ++j)
            if (kb + j < KB)
              mma_block(leader, tmem + acc_at(batch) + j * kAccCols, a0 + (uint64_t)(s1 * (kStage1 >> 4) + j * 64), b0 + (uint64_t)((kb + j) * 64), idesc);
          if (leader) {
            tc_commit(&aux->acc_full[a]);
            tc_commit(&aux->empty1[s1]);
          }
          if (++s1 == (uint32_t)Q.stages1) { s1 = 0; p1 ^= 1; }
        }
        o += tile_size(o, hi);
      }
    } else if (warp >= 4) {
      const int row = wq * 32 + lane, out = (row >> 4) * 8 + (row & 7);  // eight gate rows, the up rows of the same outputs, and so on
      for (int64_t o = lo; o < hi;) {
        const int tn = tile_size(o, hi), batches = (KB + kBlocks1 - 1) / kBlocks1;
        // this lane's row of the tile (one that is not there takes the last one's scale)
        const Output q = output_at(P, slots, o + (out < tn ? out : tn - 1));
        const float* ws = (q.s == slots ? P.sw1s : P.w1s + (int64_t)S.list[q.s] * (2 * P.I / 128) * KB) + (int64_t)((q.p + (row & 8 ? q.width : 0)) / 128) * KB;
        float acc[kTokens] = {};
        const int first = ((int)(batch & 1) == group) ? 0 : 1;  // this group's stages are every other one
        float w[kBlocks1];                                      // their scales, one stage ahead
        auto fetch = [&](int i) {
#pragma unroll
          for (int j = 0; j < kBlocks1; ++j) w[j] = i * kBlocks1 + j < KB ? ws[i * kBlocks1 + j] : 0.0f;
        };
        fetch(first);
        for (int i = first; i < batches; i += 2) {
          const uint32_t n = batch + i, a = n % kAccs;
          if (alive) alive = warp_agrees(mbar_wait(&aux->acc_full[a], (n / kAccs) & 1, P.status, P.wait_ns));
          tc_fence_after();
          uint32_t r[kBlocks1][8];
#pragma unroll
          for (int j = 0; j < kBlocks1; ++j) tmem_ld8(t_lane + acc_at(n) + j * kAccCols, r[j]);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&aux->acc_empty[a]);
#pragma unroll
          for (int j = 0; j < kBlocks1; ++j) {
            const int kb = i * kBlocks1 + j;
            if (kb < KB) {
              const float4 x0 = *reinterpret_cast<const float4*>(xs + kb * kTokens), x1 = *reinterpret_cast<const float4*>(xs + kb * kTokens + 4);
              const float x[kTokens] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
#pragma unroll
              for (int m = 0; m < kTokens; ++m) acc[m] = fmaf(__uint_as_float(r[j][m]), x[m] * w[j], acc[m]);
            }
          }
          fetch(i + 2);
        }
        batch += batches;
        consumers_sync();  // the last tile's sums have been read
        float4* j = reinterpret_cast<float4*>(join + (group * 128 + row) * kTokens);
        j[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
        j[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
        consumers_sync();
#pragma unroll
        for (int i = 0; i < 64 * kTokens / kConsumers; ++i) {
          const int at = tid + i * kConsumers, n = at & 63, m = at >> 6;
          if (n < tn) {
            const Output y = output_at(P, slots, o + n);
            if ((S.mask[y.s] >> m) & 1) {
              const float* s = join + ((n >> 3) * 16 + (n & 7)) * kTokens + m;
              const float gate = s[0] + s[128 * kTokens], up = s[8 * kTokens] + s[136 * kTokens];
              reinterpret_cast<T*>(P.h)[(int64_t)y.s * kTokens * P.I + (int64_t)m * y.width + y.p] = from_f32<T>(silu_mul(gate, up));
            }
          }
        }
        o += tn;
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
    if (producer) {
      if (leader) {
        if (warp == 0) aux->run2[(turn + 1) & 1] = claim(P.counters + 1);
        if (!waited) wait_for_runs(P.counters + 2, runs1, P.status, P.wait_ns);
        proxy_fence();
      }
      waited = true;
      __syncwarp();
      if (early == 0) filled = 0;
      for (int i = 0; i < steps && alive; ++i) {
        const bool turns = (filled++ & 1) == mine, sent = early > 0;
        if (sent) --early;
        if (turns) {
          if (!sent && !mbar_wait(&aux->empty2[s2], p2, P.status, P.wait_ns)) { alive = false; break; }
          if (leader) load_step(lo, i, !sent, true);
        }
        if (++s2 == (uint32_t)Q.stages2) { s2 = 0; p2 ^= 1; }
      }
    } else if (warp == 1) {
      const uint64_t a0 = make_smem_desc(smem_u32(ring)), b0 = make_smem_desc(smem_u32(ring) + kBlocks2 * Q.block2);
      for (int i = 0; i < steps && alive; ++i, ++batch) {
        const uint32_t a = batch % kAccs;
        const int n = step_at(i).n;
        if (!room_for(batch) || !mbar_wait(&aux->full2[s2], p2, P.status, P.wait_ns)) { alive = false; break; }
        tc_fence_after();
        const uint64_t at = (uint64_t)(s2 * (uint32_t)(Q.slot2 >> 4));
#pragma unroll
        for (int j = 0; j < kBlocks2; ++j)
          if (j < n) mma_block(leader, tmem + acc_at(batch) + j * kAccCols, a0 + at + (uint64_t)(j * (Q.block2 >> 4)), b0 + at + (uint64_t)(j * 64), idesc2);
        if (leader) {
          tc_commit(&aux->acc_full[a]);
          tc_commit(&aux->empty2[s2]);
        }
        if (++s2 == (uint32_t)Q.stages2) { s2 = 0; p2 ^= 1; }
      }
    } else if (warp >= 4) {
      if (!waited) {
        waited = true;
        if (tid == 0) wait_for_runs(P.counters + 2, runs1, P.status, P.wait_ns);
        consumers_sync();
      }
      // 64 rows lie in the lower 16 lanes of each quarter.  A row that is not there takes the last one's scale
      const int row = wq * 16 + (lane & 15), r0 = lo + row < hi ? lo + row : hi - 1;
      const bool rows_here = lo + wq * 16 < hi;
      float acc[kTokens] = {};
      const int first = ((int)(batch & 1) == group) ? 0 : 1;
      // of this group's next stage: scales of the row's blocks; lane 8 j + m has token m's scale and routing weight for block j
      float w[kBlocks2] = {}, f = 0.0f;
      Step e = {};
      uint32_t mask = 0;
      auto fetch = [&](int i) {
        if (rows_here && i < steps) {
          e = step_at(i);
          const int K = e.shared ? KS : KI, m = lane & 7, j = lane >> 3;
          mask = S.mask[e.s];
          const float* ws = (e.shared ? P.sw2s : P.w2s + (int64_t)S.list[e.s] * KB * K) + (int64_t)(r0 / 128) * K + e.kb;
#pragma unroll
          for (int q = 0; q < kBlocks2; ++q) w[q] = q < e.n ? ws[q] : 0.0f;
          f = j < e.n && ((mask >> m) & 1) ? __ldcg((e.shared ? P.h8_scale_shared : P.h8_scale + (int64_t)e.s * kTokens * K) + m * K + e.kb + j) : 0.0f;
        }
      };
      fetch(first);
      for (int i = first; i < steps; i += 2) {
        const uint32_t n = batch + i, a = n % kAccs;
        if (alive) alive = warp_agrees(mbar_wait(&aux->acc_full[a], (n / kAccs) & 1, P.status, P.wait_ns));
        tc_fence_after();
        uint32_t r[kBlocks2][8];
        if (rows_here) {
#pragma unroll
          for (int j = 0; j < kBlocks2; ++j) tmem_ld8(t_lane + acc_at(n) + j * kAccCols, r[j]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&aux->acc_empty[a]);
        if (rows_here) {
#pragma unroll
          for (int j = 0; j < kBlocks2; ++j) {
            if (j < e.n) {
#pragma unroll
              for (int m = 0; m < kTokens; ++m) {
                const float fm = __shfl_sync(0xFFFFFFFFu, f, 8 * j + m);
                // a token that is not the expert's takes nothing, whatever the weights and its place hold
                if ((mask >> m) & 1) acc[m] = fmaf(__uint_as_float(r[j][m]), fm * w[j], acc[m]);
              }
            }
          }
        }
        fetch(i + 2);
      }
      batch += steps;
      consumers_sync();
      if (lane < 16) {
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
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kAccs * kAccBlocks * kAccCols));
  }
}

constexpr int64_t fixed_bytes(int64_t H) {
  return 1024 + (H / 128 + 1) * 1024 + H / 128 * kTokens * 4 + kJoinBytes + (int64_t)(sizeof(Shared) + 15) / 16 * 16 + (int64_t)sizeof(Aux);
}
static_assert(fixed_bytes(kMaxHidden8) + 4 * kStage1 <= kFewSmem, "four stages at the largest hidden size");
static_assert(4 * kStage1 >= kTokens * kMaxExperts * 4, "what routing needs takes the ring's place");
static_assert(4 * kStage1 >= 3 * kBlocks2 * (64 * 128 + 1024), "three stages of W2");
// the tensor core reads 64 rows from a block of W2 that holds fewer: what lies behind the ring is as long
static_assert(kJoinBytes + (int64_t)sizeof(Shared) >= 64 * 128, "reads behind the last block stay in shared memory");

template <typename T>
int launch(const Maps& maps, const Few& P, const Few8& Q, int G, cudaStream_t st) {
  auto kern = few_experts8_kernel<T>;
  const int rc = allow_smem((const void*)kern, (int)kFewSmem);
  if (rc) return rc;
  return launch_pdl(kern, dim3((unsigned)G), kThreads, (size_t)(fixed_bytes(P.H) + Q.ring), 1, st, "fused_moe_few_tokens (fp8)", maps, P, Q);
}

int encode(CUtensorMap* m, const void* base, int dims, const cuuint64_t* size, const cuuint64_t* stride, const cuuint32_t* box) {
  return encode_map(m, "", CU_TENSOR_MAP_DATA_TYPE_UINT8, dims, base, size, stride, box, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
}
// W1 of `experts`, [2 width, H] each
int encode_w1(CUtensorMap* m, const void* base, uint64_t experts, uint64_t width, uint64_t H) {
  const cuuint64_t size[5] = {128, 8, H / 128, 2, experts * 2 * width / 8}, stride[4] = {H, 128, width * H, 8 * H};
  for (uint32_t z = 0; z < 4; ++z) {
    const cuuint32_t box[5] = {128, 8, kBlocks1, 2, 8u >> z};
    if (const int rc = encode(m + z, base, 5, size, stride, box)) return rc;
  }
  return 0;
}
// h of `rows` rows of `width`: a box is kBlocks2 K blocks of eight rows
int encode_h(CUtensorMap* m, const void* base, uint64_t rows, uint64_t width) {
  const cuuint64_t size[3] = {128, rows, width / 128}, stride[2] = {width, 128};
  const cuuint32_t box[3] = {128, kTokens, kBlocks2};
  return encode(m, base, 3, size, stride, box);
}

}  // namespace

int few_experts_fp8(const Few& P, int dtype, cudaStream_t st) {
  const int G = sm_count();
  const int64_t slots = (int64_t)P.M * P.topk < P.E ? (int64_t)P.M * P.topk : P.E;
  if ((int64_t)P.E * 2 * P.I >= (1ll << 31) || (int64_t)P.E * P.H >= (1ll << 31)) return fail(MOE_E_TOOBIG, "fused_moe_few_tokens: extent exceeds int32 coordinates");
  Few8 Q;
  const int runs2 = (P.H + 63) / 64 > G ? (P.H + 63) / 64 : G;
  Q.rows2 = (P.H + runs2 - 1) / runs2;
  Q.block2 = (Q.rows2 * 128 + 1023) / 1024 * 1024;
  Q.slot2 = kBlocks2 * (Q.block2 + 1024);
  auto stages = [](int64_t n) { return (int)(n < kMaxStages ? n : kMaxStages); };
  Q.stages1 = stages((kFewSmem - fixed_bytes(P.H)) / kStage1);
  Q.ring = Q.stages1 * kStage1;
  Q.stages2 = stages((Q.ring + (P.H / 128 + 1) * 1024) / Q.slot2);  // W2's ring also takes the tokens' place
  Maps m;
  const CUtensorMapDataType u8 = CU_TENSOR_MAP_DATA_TYPE_UINT8;
  int rc = encode_w1(m.w1, P.w1, (uint64_t)P.E, (uint64_t)P.I, (uint64_t)P.H);
  if (!rc) rc = tc::make_map(&m.w2, P.w2, u8, 1, (uint64_t)P.E * P.H, (uint64_t)P.I, (uint32_t)Q.rows2, true);
  if (!rc) rc = encode_h(&m.h, P.h8, (uint64_t)slots * kTokens, (uint64_t)P.I);
  if (P.Is > 0) {
    if (!rc) rc = encode_w1(m.sw1, P.sw1, 1, (uint64_t)P.Is, (uint64_t)P.H);
    if (!rc) rc = tc::make_map(&m.sw2, P.sw2, u8, 1, (uint64_t)P.H, (uint64_t)P.Is, (uint32_t)Q.rows2, true);
    if (!rc) rc = encode_h(&m.sh, P.h8_shared, kTokens, (uint64_t)P.Is);
  } else {
    for (int z = 0; z < 4; ++z) m.sw1[z] = m.w1[z];
    m.sw2 = m.w2;
    m.sh = m.h;
  }
  if (rc) return rc;
  return dtype == MOE_BF16 ? launch<__nv_bfloat16>(m, P, Q, G, st) : launch<__half>(m, P, Q, G, st);
}

}  // namespace moe
