// The loss that keeps a router's experts evenly used, the tokens that every expert got, and the gradient of the logits.
//
//   u = l (softmax scores), log sigmoid(l) (sigmoid scores divided by their sum)      p_te = exp(u_te - max u_t) / sum_e
//   per sequence s of N_s tokens that are not padding:   c_se = routes of its tokens to expert e,   P_se = mean of p_te
//   loss = mean over the sequences with N_s > 0 of  sum_e f_se P_se,   f_se = E c_se / (k N_s)
//   dl_te = p_te (a_e - sum_j p_tj a_j) u'(l_te),   a_e = dloss f_se / (N_s sequences),   u' = 1 or 1 - sigmoid(l)
//
// The counts are held: no gradient goes through the choice.  Scores that are divided by their sum are a softmax of their
// logarithms, so one stable form serves both routers (sigmoids that all underflow have a sum of zero; their logarithms are
// finite).  A constant taken off a_e changes nothing, as p sums to one: E c - k N, a whole number, stands for E c, so that what
// is left of two nearly equal sums when the experts are nearly even is exact to fp32.  A row whose logits are all -inf has
// p = 0 and no gradient.
//
// Two launches forward, one where a block holds all rows.  Each block of the first takes a run of rows and, for every sequence in
// it, sums p and counts routes in registers and shared memory; sequence s in block c goes to slot c + s, which no other pair has (a
// walk along the rows adds one to c or to s at every step).  The second adds the slots in order, so that results are the same bits
// in every run.
// Bound: the logits are read once forward and once backward; up to some ten thousand tokens it is the launches and the chain of
// loads in a block, with many short sequences that chain once for each.  us on the device, logits not in L2, forward and backward:
// 64 x 8 fp32 3.8 + 2.8 (one launch forward), 4096 x 128 bf16 9.5 + 4.7, 8192 x 256 fp32 10.6 + 6.1, the same in 23 sequences of
// sigmoid scores 22.7 + 10.0, in 700 94 + 10.9, 65536 x 256 fp32 22.8 + 27.9 (floor 10 + 20).
#include "moe_common.cuh"

namespace moe {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kSumBlocks = 3, kGradBlocks = 2;  // of a multiprocessor, as their registers allow: one wave

struct Balance {
  const void* logits;
  int64_t ld;
  const void* ids;
  const int32_t* cu;       // [sequences + 1], null = one sequence of all rows
  const uint8_t* padding;  // [tokens], null = none
  int64_t tokens;
  int experts, topk, sequences, ids64, sigmoid;
  int rows;   // of a block
  int lanes;  // that share a token
};

// Sums of the slots, [slots, experts] and [slots]; [0]: the sequences are not in order, [1]: blocks that are done.
struct Slots {
  float* mass;
  int32_t *count, *tokens, *flags;
  double* part;  // [sequences, slices] of the loss
};

// The first sequence that ends behind row t (their number if none does), the same in every lane: 32 edges are looked at a time,
// as a search by halves waits for the memory at every step.
__device__ __forceinline__ int sequence_of(const int32_t* cu, int sequences, int64_t t) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = sequences;  // it is one of lo .. lo + n
  while (n > 0) {
    const int step = (n + 31) / 32, i = (lane + 1) * step - 1;
    const int passed = __popc(__ballot_sync(0xFFFFFFFFu, i < n && cu[lo + i + 1] <= t));
    lo += passed * step;
    n = min(step - 1, n - passed * step);
  }
  return lo;
}

// Tokens that a lane has in hand at once: their loads and the two sums over the lanes of each run beside one another.
__host__ __device__ constexpr int tokens_in_hand(int values) { return values >= 32 ? 1 : values >= 16 ? 2 : 4; }

template <typename T, int V, int CH>
__device__ __forceinline__ void load_row(const T* row, int at, int lanes, int experts, bool live, float (&l)[CH][V]) {
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int e = (at + c * lanes) * V;
#pragma unroll
    for (int i = 0; i < V; ++i) l[c][i] = -INFINITY;
    if (live && e < experts) {
      if constexpr (V == 1) {
        l[c][0] = ToF32<T>::get(row[e]);
      } else {
        const uint4 raw = *reinterpret_cast<const uint4*>(row + e);
#pragma unroll
        for (int i = 0; i < V; ++i) l[c][i] = ToF32<T>::get(reinterpret_cast<const T*>(&raw)[i]);
      }
    }
  }
}

// 2^x; what is below 2^-126 is zero.
__device__ __forceinline__ float exp2_ftz(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float log2_approx(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// l -> e of U tokens, each over `lanes` lanes (all lanes of the warp call it); the scores are p = e inv.
template <int V, int CH, int U>
__device__ __forceinline__ void scores(const float (&l)[U][CH][V], int lanes, bool sigmoid, float (&e)[U][CH][V], float (&inv)[U]) {
  if (sigmoid) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float x = l[u][c][i];
          // off by 2^-22 of one, as little as the score is then off by itself; fminf drops a NaN
          e[u][c][i] = x == x ? fmaf(log2_approx(1.0f + expf(-fabsf(x))), -0.6931471805599453f, fminf(x, 0.0f)) : x;
        }
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < V; ++i) e[u][c][i] = l[u][c][i];
  }
  float m[U], sum[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    m[u] = -INFINITY;
    sum[u] = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int i = 0; i < V; ++i) m[u] = max_nan(m[u], e[u][c][i]);
  }
  for (int off = lanes / 2; off > 0; off >>= 1)
#pragma unroll
    for (int u = 0; u < U; ++u) m[u] = max_nan(m[u], __shfl_xor_sync(0xFFFFFFFFu, m[u], off));
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const float at = m[u] == -INFINITY ? 0.0f : m[u];
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        // the difference first: with the type's lowest value in every place it is zero
        e[u][c][i] = exp2_ftz((e[u][c][i] - at) * 1.4426950408889634f);
        sum[u] += e[u][c][i];
      }
  }
  for (int off = lanes / 2; off > 0; off >>= 1)
#pragma unroll
    for (int u = 0; u < U; ++u) sum[u] += __shfl_xor_sync(0xFFFFFFFFu, sum[u], off);
#pragma unroll
  for (int u = 0; u < U; ++u) inv[u] = sum[u] == 0.0f ? 0.0f : 1.0f / sum[u];  // the sum is at least 1, or the row has no score
}

// Sum over the block, the same in every thread and run; `sh` holds a value per warp.
template <typename X>
__device__ __forceinline__ X block_sum(X v, X* sh) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, off);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  v = lane < (int)blockDim.x / 32 ? sh[lane] : X(0);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, off);
  return v;
}

// What the call gives back; null in the first of two launches.
struct Result {
  int32_t *counts, *saved;
  float* loss;
};

template <typename T, int V, int CH>
__global__ void __launch_bounds__(kThreads, V * CH > 16 ? 1 : kSumBlocks) balance_sums_kernel(const Balance b, const Slots out, const Result result, int32_t* __restrict__ status) {
  pdl_wait();
  pdl_trigger();
  constexpr int U = tokens_in_hand(V * CH);
  extern __shared__ float sh[];  // [warps, experts] of p, [experts] of routes, tokens
  __shared__ double sh_sum[kWarps];
  int32_t* hist = reinterpret_cast<int32_t*>(sh + kWarps * b.experts);
  int32_t* live_tokens = hist + b.experts;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, groups = 32 / b.lanes, step = kWarps * groups;
  const int group = lane / b.lanes, at = lane % b.lanes;
  const int64_t r0 = (int64_t)blockIdx.x * b.rows, r1 = min(b.tokens, r0 + b.rows);
  if (b.cu != nullptr && blockIdx.x == gridDim.x - 1) {  // a block more, which looks at the edges
    int bad = 0;
    for (int s = threadIdx.x; s < b.sequences; s += kThreads) bad |= b.cu[s] < 0 || b.cu[s + 1] < b.cu[s] || b.cu[s + 1] > b.tokens;
    bad = __syncthreads_or(bad);
    if (threadIdx.x == 0) {
      out.flags[0] = bad;
      out.flags[1] = 0;
      if (bad) set_status(status, MOE_ST_BAD_ROW);
    }
    return;
  }
  if (b.cu == nullptr && result.loss == nullptr && blockIdx.x == 0 && threadIdx.x < 2) out.flags[threadIdx.x] = 0;
  bool bad_id = false;
  int s = b.cu == nullptr ? 0 : sequence_of(b.cu, b.sequences, r0);
  int64_t edge = b.cu == nullptr ? 0 : b.cu[s];
  for (; s < b.sequences; ++s) {
    int64_t first = r0, last = r1;
    if (b.cu != nullptr) {
      if (edge >= r1) break;
      first = max(r0, edge);
      edge = b.cu[s + 1];
      last = min(r1, edge);
      if (first >= last) continue;
    }
    // What a sequence's part needs is asked for at once: routes, padding, the first tokens.  One load behind another, and the
    // routes before the tokens, a block of two sequences took 13 us where one of one took 7.7.
    const uint32_t routes = (uint32_t)(last * b.topk);  // check(): all routes are below 2^31
    uint32_t i0 = (uint32_t)(first * b.topk) + threadIdx.x;
    int id[4];
    auto load_ids = [&] {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t i = i0 + j * kThreads;
        id[j] = -1;
        if (i >= routes) continue;
        const bool pad = b.padding != nullptr && b.padding[i / (uint32_t)b.topk];
        const int64_t v = b.ids64 ? reinterpret_cast<const int64_t*>(b.ids)[i] : (int64_t) reinterpret_cast<const int32_t*>(b.ids)[i];
        id[j] = pad || v < 0 ? -1 : v < b.experts ? (int)v : b.experts;
      }
    };
    auto count_ids = [&] {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (id[j] >= 0 && id[j] < b.experts) atomicAdd(hist + id[j], 1);
        bad_id |= id[j] == b.experts;
      }
    };
    load_ids();
    for (int e = threadIdx.x; e <= b.experts; e += kThreads) hist[e] = 0;  // and the tokens behind
    __syncthreads();
    float acc[CH][V] = {};
    int mine = 0;
    const T* row = reinterpret_cast<const T*>(b.logits) + (first + warp * groups + group) * b.ld;
    const int64_t apart = step * b.ld;
    for (int t0 = (int)first + warp * groups + group; t0 - group < (int)last; t0 += U * step, row += U * apart) {
      float l[U][CH][V], p[U][CH][V], inv[U];
      bool live[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int t = t0 + u * step;
        live[u] = t < (int)last;
        load_row<T, V, CH>(row + u * apart, at, b.lanes, b.experts, live[u], l[u]);
        if (b.padding != nullptr && live[u]) live[u] = !b.padding[t];
      }
      if (b.padding != nullptr) {  // whatever padding holds
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < V; ++i) l[u][c][i] = live[u] ? l[u][c][i] : -INFINITY;
      }
      scores<V, CH, U>(l, b.lanes, b.sigmoid, p, inv);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        mine += live[u] && at == 0;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
          for (int i = 0; i < V; ++i) acc[c][i] = fmaf(p[u][c][i], inv[u], acc[c][i]);
      }
    }
    count_ids();
    for (i0 += 4 * kThreads; i0 - threadIdx.x < routes; i0 += 4 * kThreads) {
      load_ids();
      count_ids();
    }
    for (int off = 16; off >= b.lanes; off >>= 1)
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < V; ++i) acc[c][i] += __shfl_xor_sync(0xFFFFFFFFu, acc[c][i], off);
    mine = __reduce_add_sync(0xFFFFFFFFu, mine);
    if (lane == 0 && mine) atomicAdd(live_tokens, mine);
    if (lane < b.lanes) {
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int e = (lane + c * b.lanes) * V + i;
          if (e < b.experts) sh[warp * b.experts + e] = acc[c][i];
        }
    }
    __syncthreads();
    const int64_t slot = (int64_t)blockIdx.x + s;
    double part = 0.0;
    for (int e = threadIdx.x; e < b.experts; e += kThreads) {
      float m = sh[e];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) m += sh[w * b.experts + e];
      if (result.loss != nullptr) {
        result.counts[e] = result.saved[e] = hist[e];
        part += (double)hist[e] * (double)m;
      } else {
        out.mass[slot * b.experts + e] = m;
        out.count[slot * b.experts + e] = hist[e];
      }
    }
    if (result.loss != nullptr) {  // one block, one sequence: this was all
      const int live = *live_tokens;
      part = block_sum(part, sh_sum);
      if (threadIdx.x == 0) {
        result.saved[b.experts] = live;
        result.saved[b.experts + 1] = live > 0;
        *result.loss = live > 0 ? (float)(part * (double)b.experts / ((double)b.topk * (double)live * (double)live)) : 0.0f;
      }
    } else if (threadIdx.x == 0) {
      out.tokens[slot] = *live_tokens;
    }
    __syncthreads();
  }
  if (bad_id) set_status(status, MOE_ST_BAD_EXPERT_ID);
}

// Block (32 experts, sequence): a lane per expert, the warps share the slots.  The block that is last to end adds up the loss.
__global__ void __launch_bounds__(1024) balance_loss_kernel(const Balance b, const Slots in, const Result out) {
  pdl_wait();
  pdl_trigger();
  __shared__ float mass[32][33];
  __shared__ int32_t count[32][33];
  __shared__ double shd[32];
  __shared__ int shi[32], is_last;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x / 32;
  const int s = blockIdx.y, e = blockIdx.x * 32 + lane;
  const int bad = in.flags[0];
  int64_t first = 0, last = b.tokens;
  if (b.cu != nullptr) {  // within the rows whatever they are: what is read for bad ones is not used
    first = min(max((int64_t)b.cu[s], (int64_t)0), b.tokens);
    last = min(max((int64_t)b.cu[s + 1], first), b.tokens);
  }
  const int c0 = (int)(first / b.rows), c1 = first < last ? (int)((last - 1) / b.rows) + 1 : c0;  // blocks that hold its rows
  float m = 0.0f;
  int n = 0, live = 0;
  for (int c = c0 + threadIdx.x; c < c1; c += blockDim.x) live += in.tokens[c + s];
  for (int c = c0 + warp; c < c1; c += 14 * warps) {  // as many in flight: three slots a multiprocessor are one round of 32 warps
    float mv[14];
    int nv[14];
#pragma unroll
    for (int j = 0; j < 14; ++j) {
      const bool there = e < b.experts && c + j * warps < c1;
      const int64_t at = (int64_t)(c + j * warps + s) * b.experts + e;
      mv[j] = there ? in.mass[at] : 0.0f;
      nv[j] = there ? in.count[at] : 0;
    }
#pragma unroll
    for (int j = 0; j < 14; ++j) { m += mv[j]; n += nv[j]; }
  }
  mass[warp][lane] = m;
  count[warp][lane] = n;
  live = __reduce_add_sync(0xFFFFFFFFu, live);
  if (lane == 0) shi[warp] = live;
  __syncthreads();
  live = __reduce_add_sync(0xFFFFFFFFu, lane < warps ? shi[lane] : 0);
  if (bad) live = 0;
  double part = 0.0;
  for (int r = warp; r < 32; r += warps) {  // a warp per expert
    float total = lane < warps ? mass[lane][r] : 0.0f;
    n = lane < warps && !bad ? count[lane][r] : 0;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) total += __shfl_xor_sync(0xFFFFFFFFu, total, off);
    n = __reduce_add_sync(0xFFFFFFFFu, n);
    const int expert = blockIdx.x * 32 + r;
    if (lane == 0 && expert < b.experts) {
      out.counts[(int64_t)s * b.experts + expert] = n;
      out.saved[(int64_t)s * b.experts + expert] = n;
      part += (double)n * (double)total;
    }
  }
  if (lane == 0) shd[warp] = part;
  __syncthreads();
  if (warp == 0) {
    part = lane < warps ? shd[lane] : 0.0;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) part += __shfl_xor_sync(0xFFFFFFFFu, part, off);
    if (lane == 0) {
      in.part[(int64_t)s * gridDim.x + blockIdx.x] = live > 0 ? part * (double)b.experts / ((double)b.topk * (double)live * (double)live) : 0.0;
      if (blockIdx.x == 0) out.saved[(int64_t)b.sequences * b.experts + s] = live;
      __threadfence();
      is_last = atomicAdd(in.flags + 1, 1) == (int)(gridDim.x * gridDim.y) - 1;
    }
  }
  __syncthreads();
  if (!is_last) return;
  __threadfence();
  double sum = 0.0;
  int filled = 0;
  const int parts = b.sequences * (int)gridDim.x;
  if (parts <= 32) {  // a warp's work: no barriers
    if (warp != 0) return;
    sum = lane < parts ? __ldcg(in.part + lane) : 0.0;
    filled = lane < b.sequences && __ldcg(out.saved + (int64_t)b.sequences * b.experts + lane) > 0;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, off);
    filled = __reduce_add_sync(0xFFFFFFFFu, filled);
  } else {
    for (int i = threadIdx.x; i < parts; i += blockDim.x) sum += __ldcg(in.part + i);
    for (int i = threadIdx.x; i < b.sequences; i += blockDim.x) filled += __ldcg(out.saved + (int64_t)b.sequences * b.experts + i) > 0;
    sum = block_sum(sum, shd);
    filled = block_sum(filled, shi);
  }
  if (threadIdx.x == 0) {
    out.saved[(int64_t)b.sequences * (b.experts + 1)] = filled;
    *out.loss = bad ? __uint_as_float(0x7FC00000u) : (float)(filled > 1 ? sum / filled : sum);
  }
}

// saved and dloss may be the work of the kernel in front, which still runs when this one starts: no __restrict__, whose loads the
// compiler may take for read-only as long as the kernel lives.
template <typename T, int V, int CH>
__global__ void __launch_bounds__(kThreads, V * CH > 16 ? 1 : 2) balance_grad_kernel(const Balance b, const int32_t* saved,
                                                                const float* dloss, T* dlogits) {
  pdl_wait();
  pdl_trigger();
  constexpr int U = tokens_in_hand(V * CH);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, groups = 32 / b.lanes, step = kWarps * groups;
  const int group = lane / b.lanes, at = lane % b.lanes;
  const int64_t r0 = (int64_t)blockIdx.x * b.rows, r1 = min(b.tokens, r0 + b.rows);
  const int32_t* live_tokens = saved + (int64_t)b.sequences * b.experts;
  const double scale = (double)*dloss / (double)max(1, live_tokens[b.sequences]);
  int s = b.cu == nullptr ? 0 : sequence_of(b.cu, b.sequences, r0 + warp * groups), held = -1;
  int begin = 0, end = INT32_MAX;  // of sequence s
  if (b.cu != nullptr) {
    begin = b.cu[s];
    end = s < b.sequences ? b.cu[s + 1] : INT32_MAX;
  }
  float a[CH][V] = {};
  const T* row = reinterpret_cast<const T*>(b.logits) + (r0 + warp * groups + group) * b.ld;
  T* drow = dlogits + (r0 + warp * groups + group) * b.experts;
  const int64_t apart = step * b.ld;
  const int dapart = step * b.experts;
  for (int t0 = (int)r0 + warp * groups + group; t0 - group < (int)r1; t0 += U * step, row += U * apart, drow += U * dapart) {
    float l[U][CH][V], p[U][CH][V], inv[U];
    int own[U];  // the token's sequence, -1 = its gradient is zero
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = t0 + u * step;
      bool live = t < (int)r1;
      load_row<T, V, CH>(row + u * apart, at, b.lanes, b.experts, live, l[u]);
      if (b.padding != nullptr && live) live = !b.padding[t];
      while (end <= t) {  // ends behind the last sequence at the latest
        begin = end;
        ++s;
        end = s < b.sequences ? b.cu[s + 1] : INT32_MAX;
      }
      own[u] = live && s < b.sequences && begin <= t ? s : -1;  // what the row holds is then of no account
    }
    scores<V, CH, U>(l, b.lanes, b.sigmoid, p, inv);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (own[u] >= 0 && own[u] != held) {
        held = own[u];
        const double n = (double)max(1, live_tokens[held]);
        const float k = (float)(scale / ((double)b.topk * n * n));
        const int64_t even = (int64_t)b.topk * live_tokens[held];
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const int e = (at + c * b.lanes) * V + i;
            a[c][i] = e < b.experts ? k * (float)((int64_t)b.experts * saved[(int64_t)held * b.experts + e] - even) : 0.0f;
          }
      }
      float mean = 0.0f;
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < V; ++i) mean = fmaf(p[u][c][i], a[c][i], mean);
      for (int off = b.lanes / 2; off > 0; off >>= 1) mean += __shfl_xor_sync(0xFFFFFFFFu, mean, off);
      mean *= inv[u];
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < V; ++i) p[u][c][i] = p[u][c][i] * inv[u] * (a[c][i] - mean);
      if (b.sigmoid) {
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
          for (int i = 0; i < V; ++i) p[u][c][i] = __fdividef(p[u][c][i], 1.0f + expf(l[u][c][i]));  // 0 where the sum overflows
      }
      if (t0 + u * step < (int)r1) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          const int e = (at + c * b.lanes) * V;
          if (e >= b.experts) continue;
          uint4 raw;
          T* o = reinterpret_cast<T*>(&raw);
#pragma unroll
          for (int i = 0; i < V; ++i) o[i] = from_f32<T>(own[u] >= 0 ? p[u][c][i] : 0.0f);
          T* dst = drow + u * dapart + e;
          if constexpr (V == 1) *dst = o[0];
          else *reinterpret_cast<uint4*>(dst) = raw;
        }
      }
    }
  }
}

constexpr int kMaxExperts = 1024, kMaxTopk = 32;
constexpr int64_t kMaxRoutes = 0x7FFF0000;  // a turn behind the last token is an int too

// How the rows are shared out: a turn of a block takes the tokens that its lanes have in hand, and turns are spread over the
// multiprocessors.  `whole`: one block that has all rows ends the call, without a second launch, so it takes up to four turns (us
// forward, 2048 x 8 fp32 8.6, 2049 x 8 in five blocks 8.8).  Where there is no launch to save it only works alone, so it is not
// for sequences (2000 x 8 in 64 of them: 151 in one block, 48 in four) nor for the gradient (2048 x 8: 7.4 and 3.4, 128 x 256: 9.8
// and 4.2).
struct Plan { bool vector; int pieces, lanes, rows; int64_t blocks; };
Plan plan_of(const void* logits, int64_t ld, const void* other, int dtype, int64_t tokens, int experts, int blocks_per_sm, bool whole) {
  Plan p;
  const int size = dtype == MOE_F32 ? 4 : 2, vec = 16 / size;
  p.vector = experts % vec == 0 && ((uintptr_t)logits & 15) == 0 && ((uintptr_t)other & 15) == 0 && ld * size % 16 == 0;
  const int width = p.vector ? vec : 1, pieces = experts / width;
  // 16 values to a lane: the sums over its lanes and all else that is done once per token count half of what they do at eight
  p.pieces = (experts <= 512 ? 16 : 32) / width;
  p.lanes = 1;
  while (p.lanes * p.pieces < pieces) p.lanes *= 2;
  const int64_t turn = (int64_t)kWarps * (32 / p.lanes) * tokens_in_hand(p.pieces * width), spread = (int64_t)sm_count() * blocks_per_sm;
  int64_t rows = (tokens + spread - 1) / spread;
  if (rows < turn) rows = turn;
  if (whole && tokens <= 4 * turn) rows = tokens;
  p.rows = (int)rows;
  p.blocks = (tokens + rows - 1) / rows;
  return p;
}

int64_t up16(int64_t n) { return (n + 15) / 16 * 16; }

// Bytes of the slots for any plan of these extents, or the pointers into them.
int64_t lay_out(int64_t tokens, int experts, int sequences, int64_t blocks, void* base, Slots* out) {
  const int64_t slots = blocks + sequences, slices = (experts + 31) / 32;
  char* p = (char*)base;
  int64_t at = 0;
  auto take = [&](int64_t bytes) { const int64_t a = at; at += up16(bytes); return p + a; };
  char *part = take(8 * slices * sequences), *mass = take(4 * slots * experts), *count = take(4 * slots * experts), *tok = take(4 * slots),
       *flags = take(8);
  if (out) *out = Slots{(float*)mass, (int32_t*)count, (int32_t*)tok, (int32_t*)flags, (double*)part};
  return at;
}
int64_t most_blocks(int64_t tokens) {
  const int64_t turns = (tokens + kWarps - 1) / kWarps, spread = (int64_t)sm_count() * kSumBlocks;
  return turns < spread ? turns : spread;
}

int check(const char* who, int64_t tokens, int experts, int topk, int sequences, int dtype, int64_t ld) {
  if (tokens < 0 || experts <= 0 || topk <= 0 || sequences < 1 || ld < 0) return fail(MOE_E_BADARG, "%s: bad extent", who);
  if (dtype != MOE_F32 && dtype != MOE_F16 && dtype != MOE_BF16) return fail(MOE_E_DTYPE, "%s: unsupported dtype %d", who, dtype);
  if (experts > kMaxExperts || topk > kMaxTopk || tokens * topk > kMaxRoutes || sequences > 65535)
    return fail(MOE_E_TOOBIG, "%s: at most %d experts, %d routes per token, 65535 sequences and 2^31 - 2^16 routes", who, kMaxExperts, kMaxTopk);
  return 0;
}

}  // namespace
}  // namespace moe

// Calls F(T, V, CH) for the kernel of a plan.
#define MOE_BALANCE_PIECES(F, T, VEC, plan)                                               \
  ((plan).vector ? ((plan).pieces == 16 / VEC ? F(T, VEC, (16 / VEC)) : F(T, VEC, (32 / VEC))) \
                 : ((plan).pieces == 16 ? F(T, 1, 16) : F(T, 1, 32)))
#define MOE_BALANCE_DISPATCH(F, dtype, plan)                         \
  ((dtype) == MOE_F32 ? MOE_BALANCE_PIECES(F, float, 4, plan)        \
   : (dtype) == MOE_F16 ? MOE_BALANCE_PIECES(F, __half, 8, plan)     \
                        : MOE_BALANCE_PIECES(F, __nv_bfloat16, 8, plan))

extern "C" int moe_balance_loss_workspace(int64_t tokens, int experts, int topk, int sequences, int64_t* bytes) {
  using namespace moe;
  const int rc = check("balance_loss", tokens, experts, topk, sequences, MOE_F32, 0);
  if (rc) return rc;
  if (!bytes) return fail(MOE_E_BADARG, "balance_loss: null pointer");
  bytes[0] = lay_out(tokens, experts, sequences, most_blocks(tokens), nullptr, nullptr);
  bytes[1] = 4 * ((int64_t)sequences * (experts + 1) + 1);
  return 0;
}

extern "C" int moe_balance_loss(const void* logits, int64_t ld, int dtype, int64_t tokens, int experts, const void* topk_ids, int ids_int64,
                                int topk, int sigmoid, const int32_t* cu_seqlens, int sequences, const uint8_t* is_padding, float* loss,
                                int32_t* counts, void* saved, void* workspace, int64_t workspace_bytes, int32_t* status, void* stream) {
  using namespace moe;
  int rc = check("balance_loss", tokens, experts, topk, sequences, dtype, ld);
  if (rc) return rc;
  if (!loss || !counts || !saved || (!cu_seqlens && sequences != 1)) return fail(MOE_E_BADARG, "balance_loss: bad argument");
  cudaStream_t st = (cudaStream_t)stream;
  if (tokens == 0) {
    cudaError_t ce = cudaMemsetAsync(loss, 0, 4, st);
    if (ce == cudaSuccess) ce = cudaMemsetAsync(counts, 0, 4 * (size_t)sequences * experts, st);
    if (ce == cudaSuccess) ce = cudaMemsetAsync(saved, 0, 4 * ((size_t)sequences * (experts + 1) + 1), st);
    return ce == cudaSuccess ? 0 : fail((int)ce, "balance_loss: %s", cudaGetErrorString(ce));
  }
  if (!logits || !topk_ids || !workspace) return fail(MOE_E_BADARG, "balance_loss: null pointer");
  const Plan plan = plan_of(logits, ld, nullptr, dtype, tokens, experts, kSumBlocks, !cu_seqlens);
  Slots slots;
  if (((uintptr_t)workspace & 15) || lay_out(tokens, experts, sequences, plan.blocks, workspace, &slots) > workspace_bytes)
    return fail(MOE_E_BADARG, "balance_loss: workspace too small");
  const Balance b = {logits, ld, topk_ids, cu_seqlens, is_padding, tokens, experts, topk, sequences, ids_int64 != 0, sigmoid != 0,
                     plan.rows, plan.lanes};
  const size_t smem = 4 * ((size_t)(kWarps + 1) * experts + 1);
  const Result result = {counts, (int32_t*)saved, loss}, later = {};
  const bool whole = plan.blocks == 1 && !cu_seqlens;
#define MOE_BL(T, V, CH)                                                                                                            \
  launch_pdl(balance_sums_kernel<T, V, CH>, dim3((unsigned)plan.blocks + (cu_seqlens != nullptr)), kThreads, smem, 1, st, "balance_loss", b, slots, whole ? result : later, \
             status)
  rc = MOE_BALANCE_DISPATCH(MOE_BL, dtype, plan);
#undef MOE_BL
  if (rc || whole) return rc;
  // one sequence has its rows in all blocks, several have few each
  return launch_pdl(balance_loss_kernel, dim3((unsigned)((experts + 31) / 32), (unsigned)sequences), sequences == 1 ? 1024 : 256, 0, 1, st,
                    "balance_loss (sum)", b, slots, result);
}

extern "C" int moe_balance_loss_grad(const void* logits, int64_t ld, int dtype, int64_t tokens, int experts, int topk, int sigmoid,
                                     const int32_t* cu_seqlens, int sequences, const uint8_t* is_padding, const void* saved,
                                     const float* dloss, void* dlogits, void* stream) {
  using namespace moe;
  const int rc = check("balance_loss_grad", tokens, experts, topk, sequences, dtype, ld);
  if (rc || tokens == 0) return rc;
  if (!logits || !saved || !dloss || !dlogits || (!cu_seqlens && sequences != 1)) return fail(MOE_E_BADARG, "balance_loss_grad: bad argument");
  const Plan plan = plan_of(logits, ld, dlogits, dtype, tokens, experts, kGradBlocks, false);
  const Balance b = {logits, ld, nullptr, cu_seqlens, is_padding, tokens, experts, topk, sequences, 0, sigmoid != 0, plan.rows, plan.lanes};
  cudaStream_t st = (cudaStream_t)stream;
#define MOE_BG(T, V, CH)                                                                                                               \
  launch_pdl(balance_grad_kernel<T, V, CH>, dim3((unsigned)plan.blocks), kThreads, 0, 1, st, "balance_loss_grad", b, (const int32_t*)saved, \
             dloss, (T*)dlogits)
  return MOE_BALANCE_DISPATCH(MOE_BG, dtype, plan);
#undef MOE_BG
}
