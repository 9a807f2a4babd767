// A whole layer of experts for a few tokens (up to 8) in two kernels:
//
//     logits = x Wr^T;  u = sigmoid(logits) or softmax(logits);  (w, ids) = group-limited top-k of u + bias (grouped_topk.cu's rule)
//     h_e = silu(W1_e[:I] x) * (W1_e[I:] x);   out = sum_j w_j W2_e(j) h_e(j)  [+ shared expert]  [+ residual]
//
// What it costs is reading the weights of the routed experts once; everything else is latency.  few_router_kernel forms the
// logits.  few_experts_kernel does the rest with one block per multiprocessor: every block routes the tokens for itself (a
// warp per token, a few hundred bytes of logits), then the blocks share the rows of W1 of all routed experts and of the shared
// one, and, when all of h is there, the rows of W2.
//
// Rows are shared out singly, so the blocks' parts are equal to one row: 8 experts of 2048 rows are 110.7 rows a block, where
// tiles of 128 rows would be 128 tiles for 148 multiprocessors.  Every warp copies its rows asynchronously
// into a ring of its own in shared memory, in whole lines, 12 KB a warp and 96 KB a multiprocessor in flight, and feeds warp-level
// mma.sync with 16 weight rows as M and the tokens as N = 8.  The order of k inside an instruction is free, so a lane's operand is
// whole 16-byte pieces of a row.  (No tcgen05: with 8 columns the tensor core idles either way.)  W1: a tile is 8 gate rows and the up
// rows of the same outputs, and the warps of a block divide the run of (tile, k step) evenly, joining the tiles that they share in a
// fixed order.  W2: the warps divide the run of (expert, k step), a warp keeps all rows of its block, scaled by the routing weights, in
// registers.
//
// Weights in e4m3 take few_tokens_fp8.cu behind the router.
//
// A block waits for others once, between W1 and W2.  Work is claimed from counters, and a block waits only for work that some running
// block has claimed: it needs no co-residency, and two calls on two streams cannot wait for each other.  The wait has the
// library's limit.
#include "few_tokens.cuh"

namespace moe {
namespace {
using namespace tc;

constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr int kRunTiles = 4096;  // tiles of W1 in a block's run, at most

__device__ __forceinline__ void mma8(float (&d)[4], std::integral_constant<int, 0>, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8(float (&d)[4], std::integral_constant<int, 1>, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <typename T> using Kind = std::integral_constant<int, std::is_same<T, __nv_bfloat16>::value ? 0 : 1>;

// 16 rows (lo: this lane's row of the first eight, hi: of the others) times 8 tokens over the 128 bytes that four lanes hold
template <typename KIND>
__device__ __forceinline__ void multiply(float (&d)[4], const B32& lo, const B32& hi, const B32& x) {
#pragma unroll
  for (int j = 0; j < 4; ++j) mma8(d, KIND{}, lo.r[2 * j], hi.r[2 * j], lo.r[2 * j + 1], hi.r[2 * j + 1], x.r[2 * j], x.r[2 * j + 1]);
}

// A slot holds rows of 128 bytes in pieces of 16; those of odd rows change halves, so that the eight lanes that read together (four
// pieces of two neighbouring rows) meet in no bank.  Lane 8 r + q copies piece q of rows r, r + 4, ..: whole lines.
__device__ __forceinline__ uint32_t place(int row, int piece) { return (uint32_t)(row * 128 + (piece ^ (row & 1) * 4) * 16); }
__device__ __forceinline__ void copy16(uint32_t at, const void* p) {
  asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16;" ::"r"(at), "l"(p) : "memory");
}
__device__ __forceinline__ void take16(uint32_t* r, uint32_t at) {
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
// pieces c and c + 4 of a row: what lane (row, c) multiplies
__device__ __forceinline__ void take(B32& v, uint32_t slot, int row, int c) {
  take16(v.r, slot + place(row, c));
  take16(v.r + 4, slot + place(row, c + 4));
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING> __device__ __forceinline__ void wait_copies() {  // of all lanes
  asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory");
  __syncwarp();
}

// ------------------------------------------------------------------ logits
// A block per expert; the sums are formed in the order of router_gemm's row-streaming kernel, whose bits they are.  Clears the
// counters of the kernel behind it.
template <typename XT, typename WT, int ROWS>
__global__ void __launch_bounds__(128) few_router_kernel(const XT* x, int64_t x_ld, const WT* w, int M, int E, int K,
                                                         int sigmoid, float* out, int32_t* counters, int64_t cleared) {
  pdl_wait();
  pdl_trigger();
  for (int64_t i = (int64_t)blockIdx.x * 128 + threadIdx.x; i < cleared; i += (int64_t)gridDim.x * 128) counters[i] = 0;
  const WT* row = w + (int64_t)blockIdx.x * K;
  float acc[ROWS] = {};
#pragma unroll(ROWS <= 2 ? 4 : 2)
  for (int k = threadIdx.x * 8; k < K; k += 1024) {
    float wv[8];
    load8<WT>(row + k, wv);
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      if (ROWS == 1 || r < M) {
        float xv[8];
        load8<XT>(x + r * x_ld + k, xv);
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[r] = fmaf(xv[i], wv[i], acc[r]);
      }
    }
  }
  __shared__ float part[4][ROWS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    float v = acc[r];
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, off);
    if (lane == 0) part[warp][r] = v;
  }
  __syncthreads();
  if (threadIdx.x < ROWS && threadIdx.x < M) {
    float v = part[0][threadIdx.x];
#pragma unroll
    for (int i = 1; i < 4; ++i) v += part[i][threadIdx.x];
    if (sigmoid) v = (float)(1.0 / (1.0 + exp(-(double)v)));  // grouped_topk's
    out[(int64_t)threadIdx.x * E + blockIdx.x] = v;
  }
}

// ------------------------------------------------------------------ experts
constexpr int kPartBytes = kWarps * 4 * 512;  // partial sums: two tiles of W1 a warp, four of W2
// W1's ring: a unit is a tile's 128 bytes of k, 2 KB
struct Ring1 {
  static constexpr int UNITS = 7, BYTES = UNITS * 2048;
};
// W2's: a unit is 16 rows' 128 bytes of k; a step's h comes with its first unit.  As many as fit
template <int RT> struct Ring2 {
  static constexpr int UNITS = RT == 1 ? 7 : 8, STEPS = (UNITS + RT - 1) / RT + 1, BYTES = UNITS * 2048 + STEPS * 1024;
};

// Rows [lo, hi) of all experts' W1, counted in outputs: routed experts one behind another, then the shared one.
template <typename T>
__device__ __forceinline__ void first_product(const Few& P, const Shared& S, const uint8_t* xrows, float* part, uint32_t ring, int64_t lo, int64_t hi) {
  using R = Ring1;
  using KIND = Kind<T>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int KB = P.H / 64, tiles = (int)((hi - lo + 7) / 8), total = tiles * KB;
  auto bound = [&](int w) { return (int)((int64_t)total * w / kWarps); };
  const int begin = bound(warp), end = bound(warp + 1);
  const int64_t routed = (int64_t)S.slots * P.I, row_bytes = (int64_t)P.H * 2;
  ring += (uint32_t)warp * R::BYTES;
  const int cr = lane >> 3, cq = lane & 7;  // what this lane copies: piece cq of rows cr and cr + 4
  // output o of all experts': its gate row, and how far behind it the up row is
  struct Row {
    const uint8_t* gate;
    int64_t up;
  };
  auto row_of = [&](int64_t o) {
    Row r = {nullptr, 0};
    if (o >= hi) return r;
    int64_t p;  // output inside the expert
    const uint8_t* base;
    int width;
    if (o < routed) {
      const int s = (int)((uint32_t)o / (uint32_t)P.I);
      p = o - (int64_t)s * P.I;
      const int64_t e = S.list[s];
      width = P.I;
      base = reinterpret_cast<const uint8_t*>(P.w1) + e * 2 * width * row_bytes;
    } else {
      p = o - routed;
      width = P.Is;
      base = reinterpret_cast<const uint8_t*>(P.sw1);
    }
    r.gate = base + p * row_bytes;
    r.up = width * row_bytes;
    return r;
  };
  int lt = begin / KB, lk = begin - lt * KB;  // where copying stands
  const uint8_t* src[2];
  int64_t up[2];
  auto enter = [&] {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const Row r = row_of(lo + 8 * (int64_t)lt + cr + 4 * j);
      src[j] = r.gate;
      up[j] = r.up;
    }
  };
  enter();
  auto copy = [&](uint32_t slot) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (src[j] != nullptr) {  // rows that are not there leave the slot as it was, and nobody looks at their outputs
        const uint8_t* p = src[j] + lk * 128 + cq * 16;
        copy16(slot + place(cr + 4 * j, cq), p);
        copy16(slot + 1024 + place(cr + 4 * j, cq), p + up[j]);
      }
    }
    if (++lk == KB) {
      lk = 0;
      ++lt;
      enter();
    }
  };
#pragma unroll 1
  for (int d = 0; d < R::UNITS - 1; ++d) {
    if (begin + d < end) copy(ring + d * 2048);
    commit_copies();
  }
  auto finish = [&](int tile, const float4& v) {
    const int64_t o = lo + 8 * (int64_t)tile + g;
    if (o < hi) {
      T* h;
      int64_t stride;
      if (o < routed) {
        const int s = (int)((uint32_t)o / (uint32_t)P.I);
        stride = P.I;
        h = reinterpret_cast<T*>(P.h) + s * kTokens * stride + (o - s * stride);
      } else {
        stride = P.Is;
        h = reinterpret_cast<T*>(P.h) + routed * kTokens + (o - routed);
      }
      // rounded to the activations' type, as in the layer of many tokens: h is an operand of the second product
      if (2 * c < P.M) h[2 * c * stride] = from_f32<T>(silu_mul(v.x, v.z));
      if (2 * c + 1 < P.M) h[(2 * c + 1) * stride] = from_f32<T>(silu_mul(v.y, v.w));
    }
  };
  int tile = begin / KB, kb = begin - tile * KB;
  int to = R::UNITS - 1, at = 0;  // slots
  float acc[4] = {};
  const uint8_t* xr = xrows + g * P.x_pitch + c * 16;
#pragma unroll 1
  for (int i = begin; i < end; ++i) {
    wait_copies<R::UNITS - 2>();
    if (i + R::UNITS - 1 < end) copy(ring + to * 2048);  // the slot that the last step has read
    commit_copies();
    if (++to == R::UNITS) to = 0;
    const uint32_t slot = ring + at * 2048;
    if (++at == R::UNITS) at = 0;
    B32 x, wg, wu;
    take(wg, slot, g, c);
    take(wu, slot + 1024, g, c);
    if (g < P.M) load_row<64>(x, xr + kb * 128);
    else zero(x);
    float p[4] = {};
    multiply<KIND>(p, wg, wu, x);
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] += p[j];
    if (++kb == KB || i + 1 == end) {
      const float4 v = make_float4(acc[0], acc[1], acc[2], acc[3]);
      const bool from_start = tile * KB >= begin;
      if (from_start && kb == KB) finish(tile, v);  // the warp had all of the tile
      else reinterpret_cast<float4*>(part)[(warp * 2 + from_start) * 32 + lane] = v;
      acc[0] = acc[1] = acc[2] = acc[3] = 0.0f;
      kb = 0;
      ++tile;
    }
  }
  __syncthreads();
  // a shared tile: the warp that has its start adds what the warps behind it hold, in their order
  if (end > begin && end % KB != 0) {
    const int t = end / KB;
    if (t * KB >= begin) {
      float4 v = reinterpret_cast<const float4*>(part)[(warp * 2 + 1) * 32 + lane];
      for (int w = warp + 1; w < kWarps && bound(w) < (t + 1) * KB; ++w) {
        if (bound(w) == bound(w + 1)) continue;
        const float4 q = reinterpret_cast<const float4*>(part)[w * 2 * 32 + lane];
        v.x += q.x; v.y += q.y; v.z += q.z; v.w += q.w;
      }
      finish(t, v);
    }
  }
}

// Rows [lo, hi) of W2, at most 16 RT, of all experts, and the output columns that they are.  `wait`: returns when h is there
template <typename T, int RT, typename Wait>
__device__ __forceinline__ void second_product(const Few& P, const Shared& S, float* part, uint32_t ring, int lo, int hi, Wait wait) {
  using R = Ring2<RT>;
  using KIND = Kind<T>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int KB = P.I / 64, SB = P.Is / 64, routed = S.slots * KB, total = routed + SB;
  const int begin = (int)((int64_t)total * warp / kWarps), end = (int)((int64_t)total * (warp + 1) / kWarps);
  ring += (uint32_t)warp * R::BYTES;
  const uint32_t hring = ring + R::UNITS * 2048;
  struct At {
    int s, kb, KB;
    const uint8_t* w;  // this lane's piece of row lo + cr
    int64_t row;       // bytes of a row
    const uint8_t* h;  // the expert's
  };
  const int cr = lane >> 3, cq = lane & 7;  // what this lane copies: piece cq of rows cr, cr + 4, ..
  auto enter = [&](int s, int kb) {  // expert s, S.slots = the shared one
    At a;
    a.s = s;
    a.kb = kb;
    const bool shared = s == S.slots;
    const int width = shared ? P.Is : P.I;
    a.KB = shared ? SB : KB;
    a.row = (int64_t)width * 2;
    const int64_t e = shared ? 0 : S.list[s];
    a.w = reinterpret_cast<const uint8_t*>(shared ? P.sw2 : P.w2) + (e * P.H + lo + cr) * a.row + cq * 16;
    a.h = reinterpret_cast<const uint8_t*>(P.h) + (int64_t)s * kTokens * P.I * 2;  // the shared expert's lies behind the others'
    return a;
  };
  auto locate = [&](int i) { return i < routed ? enter(i / KB, i % KB) : enter(S.slots, i - routed); };
  auto advance = [&](At& a) {
    if (++a.kb == a.KB && a.s < S.slots && (a.s + 1 < S.slots || SB > 0)) a = enter(a.s + 1, 0);
  };
  auto copy = [&](const At& a, int t, uint32_t slot) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (lo + 16 * t + 4 * j + cr < hi) copy16(slot + place(4 * j + cr, cq), a.w + (16 * t + 4 * j) * a.row + a.kb * 128);
  };
  auto copy_h = [&](const At& a, uint32_t slot) {
    const uint32_t mask = S.mask[a.s];
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if ((mask >> (4 * j + cr)) & 1) copy16(slot + place(4 * j + cr, cq), a.h + (4 * j + cr) * a.row + a.kb * 128 + cq * 16);
  };
  const int units = (end - begin) * RT;
  At ld = locate(begin < total ? begin : total - 1), at = ld;
  int lu = 0, lt = 0, to = 0, hto = 0;  // where copying stands: unit, tile of the step, slots
#pragma unroll 1
  for (; lu < R::UNITS - 1 && lu < units; ++lu) {  // weights do not wait for h
    copy(ld, lt, ring + to * 2048);
    if (++to == R::UNITS) to = 0;
    if (++lt == RT) {
      lt = 0;
      advance(ld);
    }
  }
  wait();
  {
    At a = at;
    int t = 0;
#pragma unroll 1
    for (int u = 0; u < R::UNITS - 1; ++u) {
      if (u < units) {
        if (t == 0) {
          copy_h(a, hring + hto * 1024);
          if (++hto == R::STEPS) hto = 0;
        }
        if (++t == RT) {
          t = 0;
          advance(a);
        }
      }
      commit_copies();
    }
  }
  auto next = [&] {  // one more unit on its way
    if (lu < units) {
      copy(ld, lt, ring + to * 2048);
      if (lt == 0) {
        copy_h(ld, hring + hto * 1024);
        if (++hto == R::STEPS) hto = 0;
      }
      if (++to == R::UNITS) to = 0;
      ++lu;
      if (++lt == RT) {
        lt = 0;
        advance(ld);
      }
    }
    commit_copies();
  };
  float acc[RT][4] = {};
  int from = 0, hfrom = 0;
#pragma unroll 1
  for (int i = begin; i < end; ++i) {
    const uint32_t mask = S.mask[at.s];
    const bool r0 = (mask >> (2 * c)) & 1, r1 = (mask >> (2 * c + 1)) & 1;
    const float f0 = r0 ? S.weight[at.s][2 * c] : 0.0f, f1 = r1 ? S.weight[at.s][2 * c + 1] : 0.0f;
    wait_copies<R::UNITS - 2>();
    next();
    const uint32_t hs = hring + hfrom * 1024;
    if (++hfrom == R::STEPS) hfrom = 0;
    B32 x;
    if ((mask >> g) & 1) take(x, hs, g, c);
    else zero(x);
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      if (t > 0) {
        wait_copies<R::UNITS - 2>();
        next();
      }
      B32 wa, wb;
      take(wa, ring + from * 2048, g, c);
      take(wb, ring + from * 2048, 8 + g, c);
      if (++from == R::UNITS) from = 0;
      float p[4] = {};
      multiply<KIND>(p, wa, wb, x);
      // a token that is not the expert's takes nothing, whatever the weights hold
      if (r0) { acc[t][0] = fmaf(p[0], f0, acc[t][0]); acc[t][2] = fmaf(p[2], f0, acc[t][2]); }
      if (r1) { acc[t][1] = fmaf(p[1], f1, acc[t][1]); acc[t][3] = fmaf(p[3], f1, acc[t][3]); }
    }
    advance(at);
  }
  __syncthreads();
#pragma unroll
  for (int t = 0; t < RT; ++t) reinterpret_cast<float4*>(part)[(warp * RT + t) * 32 + lane] = make_float4(acc[t][0], acc[t][1], acc[t][2], acc[t][3]);
  __syncthreads();
  for (int t = warp; t < RT; t += kWarps) {
    float v[4] = {};
#pragma unroll
    for (int k = 0; k < kWarps; ++k) {
      const float4 q = reinterpret_cast<const float4*>(part)[(k * RT + t) * 32 + lane];
      v[0] += q.x; v[1] += q.y; v[2] += q.z; v[3] += q.w;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = lo + 16 * t + 8 * (j >> 1) + g, m = 2 * c + (j & 1);
      if (r < hi && m < P.M) {
        float o = v[j];
        if (P.residual) o += ToF32<T>::get(reinterpret_cast<const T*>(P.residual)[m * P.residual_ld + r]);
        reinterpret_cast<T*>(P.out)[(int64_t)m * P.H + r] = from_f32<T>(o);
      }
    }
  }
}

template <typename T, int RT>
__global__ void __launch_bounds__(kThreads, 1) few_experts_kernel(const Few P) {
  extern __shared__ __align__(16) uint8_t smem[];
  Shared& S = *reinterpret_cast<Shared*>(smem);
  float* part = reinterpret_cast<float*>(smem + (sizeof(Shared) + 127) / 128 * 128);
  uint8_t* rest = reinterpret_cast<uint8_t*>(part) + kPartBytes;  // routing, then W1's ring and the tokens, then W2's ring
  uint8_t* xs = rest + kWarps * Ring1::BYTES;
  // the tokens, older than the kernel in front: into shared memory
  const uint8_t* xrows = xs;
  if (P.staged) {
    const int pieces = P.H / 8;
    for (int i = threadIdx.x; i < P.M * pieces; i += kThreads) {
      const int m = i / pieces, k = i - m * pieces;
      *reinterpret_cast<uint4*>(xs + m * P.x_pitch + k * 16) = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(P.x) + m * P.x_ld + k * 8);
    }
  } else {
    xrows = reinterpret_cast<const uint8_t*>(P.x);
  }
  prepare_route(P, S);
  pdl_wait();  // scores and cleared counters
  pdl_trigger();
  int mine1 = 0, mine2 = 0;  // thread 0: claimed, not begun
  if (threadIdx.x == 0) {
    mine1 = claim(P.counters);
    mine2 = claim(P.counters + 1);
  }
  if (P.E <= 256) route<8>(P, S, reinterpret_cast<uint32_t*>(rest));
  else route<32>(P, S, reinterpret_cast<uint32_t*>(rest));

  const int64_t outputs = (int64_t)S.slots * P.I + P.Is;
  const int G = gridDim.x;
  const int64_t runs1 = (outputs + (int64_t)G * kRunTiles * 8 - 1) / ((int64_t)G * kRunTiles * 8) * G;
  for (;;) {
    if (threadIdx.x == 0) S.next1 = mine1;
    __syncthreads();
    const int run = S.next1;
    if (run >= runs1) break;
    if (threadIdx.x == 0) mine1 = claim(P.counters);
    first_product<T>(P, S, xrows, part, smem_u32(rest), outputs * run / runs1, outputs * (run + 1) / runs1);
    __syncthreads();  // all of the run's h is written
    if (threadIdx.x == 0) {
      __threadfence();
      atomicAdd(P.counters + 2, 1);
    }
  }
  bool waited = false;
  auto wait = [&] {
    if (waited) return;
    waited = true;
    if (threadIdx.x == 0) wait_for_runs(P.counters + 2, runs1, P.status, P.wait_ns);
    __syncthreads();
  };
  const int runs2 = (P.H + 16 * RT - 1) / (16 * RT) > G ? (P.H + 16 * RT - 1) / (16 * RT) : G;
  for (;;) {
    if (threadIdx.x == 0) S.next2 = mine2;
    __syncthreads();
    const int run = S.next2;
    if (run >= runs2) break;
    if (threadIdx.x == 0) mine2 = claim(P.counters + 1);
    second_product<T, RT>(P, S, part, smem_u32(rest), (int)((int64_t)P.H * run / runs2), (int)((int64_t)P.H * (run + 1) / runs2), wait);
  }
}

constexpr int64_t kHead = (sizeof(Shared) + 127) / 128 * 128 + kPartBytes;
static_assert(kTokens * kMaxExperts * 4 <= kWarps * Ring1::BYTES, "what routing needs lies in front of the tokens");
static_assert(kHead + kWarps * Ring2<1>::BYTES <= kFewSmem && kHead + kWarps * Ring2<2>::BYTES <= kFewSmem &&
                  kHead + kWarps * Ring2<4>::BYTES <= kFewSmem, "ring of W2");

// ------------------------------------------------------------------ host side
struct Layout {
  int64_t counters, scores, h, h8, h8_shared, h8_scale, h8_scale_shared, bytes;
};
Layout layout(int64_t M, int E, int64_t I, int64_t Is, int topk, bool fp8) {
  auto up = [](int64_t b) { return (b + 255) / 256 * 256; };
  Layout l;
  const int64_t slots = M * topk < E ? M * topk : E, outputs = slots * I + Is;
  l.counters = 4 + (fp8 ? outputs / 128 : 0);
  l.scores = up(l.counters * 4);
  l.h = l.scores + up(M * E * 4);
  l.h8 = l.h + up(outputs * kTokens * 2);
  l.h8_shared = l.h8 + (fp8 ? up(slots * I * kTokens) : 0);
  l.h8_scale = l.h8_shared + (fp8 ? up(Is * kTokens) : 0);
  l.h8_scale_shared = l.h8_scale + (fp8 ? up(slots * I / 128 * kTokens * 4) : 0);
  l.bytes = l.h8_scale_shared + (fp8 ? up(Is / 128 * kTokens * 4) : 0);
  return l;
}

template <typename XT, typename WT>
int run_router(const Few& P, const void* w, cudaStream_t st) {
#define MOE_FEW_ROUTER(ROWS)                                                                                                             \
  launch_pdl(few_router_kernel<XT, WT, ROWS>, dim3((unsigned)P.E), 128, 0, 1, st, "fused_moe_few_tokens (router)", (const XT*)P.x, P.x_ld, \
             (const WT*)w, P.M, P.E, P.H, P.sigmoid, const_cast<float*>(P.scores), P.counters, P.cleared)
  if (P.M == 1) return MOE_FEW_ROUTER(1);
  if (P.M == 2) return MOE_FEW_ROUTER(2);
  if (P.M <= 4) return MOE_FEW_ROUTER(4);
  return MOE_FEW_ROUTER(8);
#undef MOE_FEW_ROUTER
}

template <typename T>
int run_experts(Few P, cudaStream_t st) {
  P.x_pitch = (int64_t)P.H * 2 + 64;  // neighbouring tokens' pieces lie in other banks
  const int64_t first = kHead + kWarps * Ring1::BYTES;
  int64_t smem = first + P.M * P.x_pitch;
  P.staged = smem <= kFewSmem;
  if (!P.staged) {  // the rows then come out of L1
    smem = first;
    P.x_pitch = P.x_ld * 2;  // rows may lie any distance apart
  }
  const int G = sm_count();
  const int rows = (P.H + G - 1) / G;
  auto go = [&](auto rt) {
    auto kern = few_experts_kernel<T, decltype(rt)::value>;
    const int rc = allow_smem((const void*)kern, (int)kFewSmem);
    if (rc) return rc;
    const int64_t second = kHead + kWarps * Ring2<decltype(rt)::value>::BYTES;
    return launch_pdl(kern, dim3((unsigned)G), kThreads, (size_t)(smem > second ? smem : second), 1, st, "fused_moe_few_tokens", P);
  };
  if (rows <= 16) return go(std::integral_constant<int, 1>());
  if (rows <= 32) return go(std::integral_constant<int, 2>());
  return go(std::integral_constant<int, 4>());
}

}  // namespace
}  // namespace moe

extern "C" int moe_few_tokens_workspace(int64_t M, int E, int64_t I, int64_t shared_I, int topk, int fp8, int64_t* bytes) {
  using namespace moe;
  if (M < 0 || M > kTokens || E <= 0 || E > kMaxExperts || I <= 0 || shared_I < 0 || topk <= 0 || topk > 32 || !bytes)
    return fail(MOE_E_BADARG, "few_tokens_workspace: bad extent");
  *bytes = layout(M, E, I, shared_I, topk, fp8 != 0).bytes;
  return 0;
}

extern "C" int moe_few_tokens(const void* x, int64_t x_ld, int dtype, const void* router, int router_dtype, const float* bias, const void* w1,
                              const void* w2, const float* w1_scale, const float* w2_scale, const void* shared_w1, const void* shared_w2,
                              const float* shared_w1_scale, const float* shared_w2_scale, const void* residual, int64_t residual_ld, int64_t M,
                              int E, int H, int I, int shared_I, int topk, int n_group, int topk_group, int renormalize, float scaling,
                              int sigmoid, void* out, float* topk_weights, int32_t* topk_ids, void* workspace, int64_t workspace_bytes,
                              int32_t* status, void* stream) {
  using namespace moe;
  const char* who = "fused_moe_few_tokens";
  if (dtype != MOE_BF16 && dtype != MOE_F16) return fail(MOE_E_DTYPE, "%s: activations are bf16 or f16", who);
  if (router_dtype != dtype && router_dtype != MOE_F32) return fail(MOE_E_DTYPE, "%s: the router's weights have the activations' type or fp32", who);
  if (M < 0 || M > kTokens) return fail(MOE_E_TOOBIG, "%s: at most %d tokens", who, kTokens);
  if (M == 0) return 0;
  const bool fp8 = w1_scale != nullptr;
  const int unit = fp8 ? 128 : 64;
  if (E <= 0 || E > kMaxExperts || H <= 0 || H > (fp8 ? kMaxHidden8 : kMaxHidden) || I <= 0 || I > kMaxWidth || shared_I > kMaxWidth || shared_I < 0 || H % unit || I % unit || shared_I % unit)
    return fail(MOE_E_SHAPE, "%s: at most %d experts, hidden sizes up to %d; sizes in multiples of %d", who, kMaxExperts, fp8 ? kMaxHidden8 : kMaxHidden, unit);
  if (topk <= 0 || topk > 32 || topk > E || n_group <= 0 || n_group > 32 || E % n_group || topk_group <= 0 || topk_group > n_group ||
      (int64_t)topk > (int64_t)E / n_group * topk_group)
    return fail(MOE_E_SHAPE, "%s: groups and topk do not fit the experts", who);
  if (!x || !router || !w1 || !w2 || !out || !topk_weights || !topk_ids || !workspace || (shared_I > 0) != (shared_w1 != nullptr) ||
      (shared_I > 0) != (shared_w2 != nullptr) || fp8 != (w2_scale != nullptr) || (fp8 && shared_I > 0 && (!shared_w1_scale || !shared_w2_scale)))
    return fail(MOE_E_BADARG, "%s: null pointer", who);
  if (x_ld < H || x_ld % 8 || (residual && residual_ld < H)) return fail(MOE_E_SHAPE, "%s: rows of x in whole 16-byte pieces", who);
  for (const void* p : {w1, w2, shared_w1, shared_w2})
    if ((uintptr_t)p & 31) return fail(MOE_E_BADARG, "%s: weights must be 32-byte aligned", who);
  for (const void* p : {x, router, (const void*)workspace})
    if ((uintptr_t)p & 15) return fail(MOE_E_BADARG, "%s: operands must be 16-byte aligned", who);
  const Layout l = layout(M, E, I, shared_I, topk, fp8);
  if (workspace_bytes < l.bytes) return fail(MOE_E_BADARG, "%s: workspace too small", who);
  uint8_t* ws = (uint8_t*)workspace;
  Few P = {};
  P.x = x; P.x_ld = x_ld; P.residual = residual; P.residual_ld = residual_ld; P.out = out;
  P.w1 = w1; P.w2 = w2; P.sw1 = shared_w1; P.sw2 = shared_w2;
  P.w1s = w1_scale; P.w2s = w2_scale; P.sw1s = shared_w1_scale; P.sw2s = shared_w2_scale;
  P.scores = (const float*)(ws + l.scores); P.bias = bias;
  P.topk_w = topk_weights; P.topk_ids = topk_ids;
  P.h = ws + l.h; P.h8 = ws + l.h8; P.h8_shared = ws + l.h8_shared; P.h8_scale = (float*)(ws + l.h8_scale);
  P.h8_scale_shared = (float*)(ws + l.h8_scale_shared); P.counters = (int32_t*)ws; P.cleared = l.counters;
  P.M = (int)M; P.E = E; P.H = H; P.I = I; P.Is = shared_I; P.topk = topk; P.n_group = n_group; P.topk_group = topk_group;
  P.renormalize = renormalize; P.sigmoid = sigmoid; P.scaling = scaling;
  P.status = status; P.wait_ns = wait_limit_ns();
  cudaStream_t st = (cudaStream_t)stream;
  const bool f32 = router_dtype == MOE_F32;
  int rc = dtype == MOE_BF16 ? (f32 ? run_router<__nv_bfloat16, float>(P, router, st) : run_router<__nv_bfloat16, __nv_bfloat16>(P, router, st))
                             : (f32 ? run_router<__half, float>(P, router, st) : run_router<__half, __half>(P, router, st));
  if (rc) return rc;
  if (fp8) return few_experts_fp8(P, dtype, st);
  return dtype == MOE_BF16 ? run_experts<__nv_bfloat16>(P, st) : run_experts<__half>(P, st);
}
