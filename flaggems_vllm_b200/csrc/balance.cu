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
// Two launches forward.  Each block of the first takes a run of rows and, for every sequence in it, sums p and counts routes
// in registers and shared memory; sequence s in block c goes to slot c + s, which no other pair has (a walk along the rows
// adds one to c or to s at every step).  The second adds the slots in order, so that results are the same bits in every run.
// Bound: memory, one pass over the logits forward and one backward; the launches for a few thousand tokens.
#include "moe_common.cuh"

namespace moe {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;

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

// The first sequence that ends behind row t (their number if none does).
__device__ __forceinline__ int sequence_of(const int32_t* cu, int sequences, int64_t t) {
  int lo = 0, hi = sequences;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (cu[mid + 1] > t) hi = mid; else lo = mid + 1;
  }
  return lo;
}

template <typename T, int V, int CH>
__device__ __forceinline__ void load_row(const T* row, int at, int lanes, int experts, bool live, float (&l)[CH][V]) {
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int e = (at + c * lanes) * V;
    if (live && e < experts) {
      if constexpr (V == 1) {
        l[c][0] = ToF32<T>::get(row[e]);
      } else {
        const uint4 raw = *reinterpret_cast<const uint4*>(row + e);
#pragma unroll
        for (int i = 0; i < V; ++i) l[c][i] = ToF32<T>::get(reinterpret_cast<const T*>(&raw)[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) l[c][i] = -INFINITY;
    }
  }
}

// l -> p, over the `lanes` lanes of a token (all lanes of the warp call it).
template <int V, int CH>
__device__ __forceinline__ void scores(const float (&l)[CH][V], int lanes, bool sigmoid, float (&p)[CH][V]) {
  float m = -INFINITY;
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      p[c][i] = sigmoid ? fminf(l[c][i], 0.0f) - log1pf(expf(-fabsf(l[c][i]))) : l[c][i];
      if (!(l[c][i] == l[c][i])) p[c][i] = l[c][i];  // fminf drops a NaN
      m = max_nan(m, p[c][i]);
    }
  for (int off = lanes / 2; off > 0; off >>= 1) m = max_nan(m, __shfl_xor_sync(0xFFFFFFFFu, m, off));
  float sum = 0.0f;
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      // the difference first: with the type's lowest value in every place it is zero
      p[c][i] = m == -INFINITY ? 0.0f : exp2f((p[c][i] - m) * 1.4426950408889634f);
      sum += p[c][i];
    }
  for (int off = lanes / 2; off > 0; off >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, off);
  const float inv = m == -INFINITY ? 0.0f : 1.0f / sum;
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int i = 0; i < V; ++i) p[c][i] *= inv;
}

template <typename T, int V, int CH>
__global__ void __launch_bounds__(kThreads) balance_sums_kernel(const Balance b, const Slots out, int32_t* __restrict__ status) {
  pdl_wait();
  pdl_trigger();
  extern __shared__ float sh[];  // [warps, experts] of p, [experts] of routes, tokens
  int32_t* hist = reinterpret_cast<int32_t*>(sh + kWarps * b.experts);
  int32_t* live_tokens = hist + b.experts;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, groups = 32 / b.lanes;
  const int64_t r0 = (int64_t)blockIdx.x * b.rows, r1 = min(b.tokens, r0 + b.rows);
  if (blockIdx.x == 0) {
    int bad = 0;
    if (b.cu != nullptr)
      for (int s = threadIdx.x; s < b.sequences; s += kThreads) bad |= b.cu[s] < 0 || b.cu[s + 1] < b.cu[s] || b.cu[s + 1] > b.tokens;
    bad = __syncthreads_or(bad);
    if (threadIdx.x == 0) {
      out.flags[0] = bad;
      out.flags[1] = 0;
      if (bad) set_status(status, MOE_ST_BAD_ROW);
    }
  }
  bool bad_id = false;
  for (int s = b.cu == nullptr ? 0 : sequence_of(b.cu, b.sequences, r0); s < b.sequences; ++s) {
    int64_t first = r0, last = r1;
    if (b.cu != nullptr) {
      if (b.cu[s] >= r1) break;
      first = max(r0, (int64_t)b.cu[s]);
      last = min(r1, (int64_t)b.cu[s + 1]);
      if (first >= last) continue;
    }
    for (int e = threadIdx.x; e <= b.experts; e += kThreads) hist[e] = 0;  // and the tokens behind
    __syncthreads();
    const uint32_t routes = (uint32_t)(last * b.topk);  // check(): all routes are below 2^31
    for (uint32_t i = (uint32_t)(first * b.topk) + threadIdx.x; i < routes; i += kThreads) {
      if (b.padding != nullptr && b.padding[i / (uint32_t)b.topk]) continue;
      const int64_t id = b.ids64 ? reinterpret_cast<const int64_t*>(b.ids)[i] : (int64_t) reinterpret_cast<const int32_t*>(b.ids)[i];
      if (id >= 0 && id < b.experts) atomicAdd(hist + id, 1);
      else bad_id |= id >= b.experts;
    }
    float acc[CH][V] = {};
    int mine = 0;
    for (int64_t t0 = first + warp * groups; t0 < last; t0 += kWarps * groups) {
      const int64_t t = t0 + lane / b.lanes;
      const bool live = t < last && (b.padding == nullptr || !b.padding[t]);
      float l[CH][V], p[CH][V];
      load_row<T, V, CH>(reinterpret_cast<const T*>(b.logits) + t * b.ld, lane % b.lanes, b.lanes, b.experts, live, l);
      scores<V, CH>(l, b.lanes, b.sigmoid, p);
      mine += live && lane % b.lanes == 0;
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < V; ++i) acc[c][i] += p[c][i];
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
    for (int e = threadIdx.x; e < b.experts; e += kThreads) {
      float m = sh[e];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) m += sh[w * b.experts + e];
      out.mass[slot * b.experts + e] = m;
      out.count[slot * b.experts + e] = hist[e];
    }
    if (threadIdx.x == 0) out.tokens[slot] = *live_tokens;
    __syncthreads();
  }
  if (bad_id) set_status(status, MOE_ST_BAD_EXPERT_ID);
}

// Sum over the block, the same in every thread and run; `sh` holds a value per warp.
template <typename X>
__device__ __forceinline__ X block_sum(X v, X* sh) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, off);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = sh[0];
  for (int w = 1; w < (int)blockDim.x / 32; ++w) v += sh[w];
  return v;
}

// Block (sequence, 32 experts): a lane per expert, the warps share the slots.  The block that is last to end adds up the loss.
__global__ void __launch_bounds__(1024) balance_loss_kernel(const Balance b, const Slots in, int32_t* __restrict__ counts,
                                                            int32_t* __restrict__ saved, float* __restrict__ loss) {
  pdl_wait();
  pdl_trigger();
  __shared__ float mass[32][33];
  __shared__ int32_t count[32][33];
  __shared__ double shd[32];
  __shared__ int shi[32], is_last;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x / 32;
  const int s = blockIdx.y, e = blockIdx.x * 32 + lane;
  const bool bad = in.flags[0] != 0;
  int64_t first = 0, last = b.tokens;
  if (b.cu != nullptr) { first = b.cu[s]; last = b.cu[s + 1]; }
  int64_t c0 = 0, c1 = 0;  // blocks that hold rows of the sequence
  if (!bad && first < last) { c0 = first / b.rows; c1 = (last - 1) / b.rows + 1; }
  float m = 0.0f;
  int n = 0, live = 0;
#pragma unroll 4
  for (int64_t c = c0 + warp; c < c1; c += warps) {
    if (e < b.experts) {
      m += in.mass[(c + s) * b.experts + e];
      n += in.count[(c + s) * b.experts + e];
    }
    if (lane == 0) live += in.tokens[c + s];
  }
  mass[warp][lane] = m;
  count[warp][lane] = n;
  live = block_sum(live, shi);  // its barriers stand between the writes above and the reads below
  double part = 0.0;
  if (warp == 0) {
    double total = 0.0;
    n = 0;
    for (int w = 0; w < warps; ++w) { total += (double)mass[w][lane]; n += count[w][lane]; }
    if (e < b.experts) {
      counts[(int64_t)s * b.experts + e] = n;
      saved[(int64_t)s * b.experts + e] = n;
      if (live > 0) part = (double)n * total;
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) part += __shfl_xor_sync(0xFFFFFFFFu, part, off);
    if (live > 0) part *= (double)b.experts / ((double)b.topk * (double)live * (double)live);
    if (lane == 0) {
      in.part[(int64_t)s * gridDim.x + blockIdx.x] = part;
      if (blockIdx.x == 0) saved[(int64_t)b.sequences * b.experts + s] = live;
      __threadfence();
      is_last = atomicAdd(in.flags + 1, 1) == (int)(gridDim.x * gridDim.y) - 1;
    }
  }
  __syncthreads();
  if (!is_last) return;
  __threadfence();
  double sum = 0.0;
  int filled = 0;
  for (int64_t i = threadIdx.x; i < (int64_t)b.sequences * gridDim.x; i += blockDim.x) sum += __ldcg(in.part + i);
  for (int i = threadIdx.x; i < b.sequences; i += blockDim.x) filled += __ldcg(saved + (int64_t)b.sequences * b.experts + i) > 0;
  sum = block_sum(sum, shd);
  filled = block_sum(filled, shi);
  if (threadIdx.x == 0) {
    saved[(int64_t)b.sequences * (b.experts + 1)] = filled;
    *loss = bad ? __uint_as_float(0x7FC00000u) : (float)(sum / (filled > 0 ? filled : 1));
  }
}

template <typename T, int V, int CH>
__global__ void __launch_bounds__(kThreads) balance_grad_kernel(const Balance b, const int32_t* __restrict__ saved,
                                                                const float* __restrict__ dloss, T* __restrict__ dlogits) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, groups = 32 / b.lanes, at = lane % b.lanes;
  const int64_t r0 = (int64_t)blockIdx.x * b.rows, r1 = min(b.tokens, r0 + b.rows);
  const int32_t* live_tokens = saved + (int64_t)b.sequences * b.experts;
  const double scale = (double)*dloss / (double)max(1, live_tokens[b.sequences]);
  int s = b.cu == nullptr ? 0 : sequence_of(b.cu, b.sequences, r0 + warp * groups + lane / b.lanes), held = -1;
  float a[CH][V] = {};
  for (int64_t t0 = r0 + warp * groups; t0 < r1; t0 += kWarps * groups) {
    const int64_t t = t0 + lane / b.lanes;
    bool live = t < r1 && (b.padding == nullptr || !b.padding[t]);
    if (b.cu != nullptr) {
      while (s < b.sequences && b.cu[s + 1] <= t) ++s;
      live = live && s < b.sequences && b.cu[s] <= t;
    }
    float l[CH][V], p[CH][V];
    load_row<T, V, CH>(reinterpret_cast<const T*>(b.logits) + t * b.ld, at, b.lanes, b.experts, live, l);
    if (live && s != held) {
      held = s;
      const double n = (double)max(1, live_tokens[s]);
      const float k = (float)(scale / ((double)b.topk * n * n));
      const int64_t even = (int64_t)b.topk * live_tokens[s];
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int e = (at + c * b.lanes) * V + i;
          a[c][i] = e < b.experts ? k * (float)((int64_t)b.experts * saved[(int64_t)s * b.experts + e] - even) : 0.0f;
        }
    }
    scores<V, CH>(l, b.lanes, b.sigmoid, p);
    float mean = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int i = 0; i < V; ++i) mean = fmaf(p[c][i], a[c][i], mean);
    for (int off = b.lanes / 2; off > 0; off >>= 1) mean += __shfl_xor_sync(0xFFFFFFFFu, mean, off);
    if (t >= r1) continue;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int e = (at + c * b.lanes) * V;
      if (e >= b.experts) continue;
      uint4 raw;
      T* o = reinterpret_cast<T*>(&raw);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float d = p[c][i] * (a[c][i] - mean);
        if (b.sigmoid) d /= 1.0f + expf(l[c][i]);
        o[i] = from_f32<T>(live ? d : 0.0f);
      }
      T* dst = dlogits + t * b.experts + e;
      if constexpr (V == 1) *dst = o[0];
      else *reinterpret_cast<uint4*>(dst) = raw;
    }
  }
}

constexpr int kMaxExperts = 1024, kMaxTopk = 32;
constexpr int64_t kMaxTokens = 0x7FFFFFFF;

// Rows of a block: four blocks to a multiprocessor, but four turns for every warp.
int rows_of_block(int64_t tokens, int lanes) {
  const int64_t spread = (int64_t)sm_count() * 4, least = 4 * kWarps * (32 / lanes);
  const int64_t rows = (tokens + spread - 1) / spread;
  return (int)(rows > least ? rows : least);
}

struct Plan { bool vector; int lanes, rows; int64_t blocks; };
Plan plan_of(const void* logits, int64_t ld, const void* other, int dtype, int64_t tokens, int experts) {
  Plan p;
  const int size = dtype == MOE_F32 ? 4 : 2, vec = 16 / size;
  p.vector = experts % vec == 0 && ((uintptr_t)logits & 15) == 0 && ((uintptr_t)other & 15) == 0 && ld * size % 16 == 0;
  const int pieces = p.vector ? experts / vec : experts;
  p.lanes = 1;
  while (p.lanes < 32 && p.lanes < pieces) p.lanes *= 2;
  p.rows = rows_of_block(tokens, p.lanes);
  p.blocks = (tokens + p.rows - 1) / p.rows;
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
int64_t most_blocks(int64_t tokens) {  // least rows of a block: one token to a warp
  const int64_t rows = rows_of_block(tokens, 32);
  return (tokens + rows - 1) / rows;
}

int check(const char* who, int64_t tokens, int experts, int topk, int sequences, int dtype, int64_t ld) {
  if (tokens < 0 || experts <= 0 || topk <= 0 || sequences < 1 || ld < 0) return fail(MOE_E_BADARG, "%s: bad extent", who);
  if (dtype != MOE_F32 && dtype != MOE_F16 && dtype != MOE_BF16) return fail(MOE_E_DTYPE, "%s: unsupported dtype %d", who, dtype);
  if (experts > kMaxExperts || topk > kMaxTopk || tokens > kMaxTokens || tokens * topk > kMaxTokens || sequences > 65535)
    return fail(MOE_E_TOOBIG, "%s: at most %d experts, %d routes per token, 65535 sequences and 2^31 - 1 routes", who, kMaxExperts, kMaxTopk);
  return 0;
}

}  // namespace
}  // namespace moe

// Calls F(T, V, CH) for the kernels of a plan: CH pieces per lane.
#define MOE_BALANCE_PIECES(F, T, VEC, plan, experts)                                       \
  ((plan).vector ? ((experts) <= 32 * VEC ? F(T, VEC, 1) : (experts) <= 64 * VEC ? F(T, VEC, 2) : F(T, VEC, (32 / VEC))) \
                 : ((experts) <= 64 ? F(T, 1, 2) : (experts) <= 256 ? F(T, 1, 8) : F(T, 1, 32)))
#define MOE_BALANCE_DISPATCH(F, dtype, plan, experts)                                      \
  ((dtype) == MOE_F32 ? MOE_BALANCE_PIECES(F, float, 4, plan, experts)                     \
   : (dtype) == MOE_F16 ? MOE_BALANCE_PIECES(F, __half, 8, plan, experts)                  \
                        : MOE_BALANCE_PIECES(F, __nv_bfloat16, 8, plan, experts))

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
  const Plan plan = plan_of(logits, ld, nullptr, dtype, tokens, experts);
  Slots slots;
  if (((uintptr_t)workspace & 15) || lay_out(tokens, experts, sequences, plan.blocks, workspace, &slots) > workspace_bytes)
    return fail(MOE_E_BADARG, "balance_loss: workspace too small");
  const Balance b = {logits, ld, topk_ids, cu_seqlens, is_padding, tokens, experts, topk, sequences, ids_int64 != 0, sigmoid != 0,
                     plan.rows, plan.lanes};
  const size_t smem = 4 * ((size_t)(kWarps + 1) * experts + 1);
#define MOE_BL(T, V, CH) \
  launch_pdl(balance_sums_kernel<T, V, CH>, dim3((unsigned)plan.blocks), kThreads, smem, 1, st, "balance_loss", b, slots, status)
  rc = MOE_BALANCE_DISPATCH(MOE_BL, dtype, plan, experts);
#undef MOE_BL
  if (rc) return rc;
  // one sequence has its rows in all blocks, several have few each
  return launch_pdl(balance_loss_kernel, dim3((unsigned)((experts + 31) / 32), (unsigned)sequences), sequences == 1 ? 1024 : 256, 0, 1, st,
                    "balance_loss (sum)", b, slots, counts, (int32_t*)saved, loss);
}

extern "C" int moe_balance_loss_grad(const void* logits, int64_t ld, int dtype, int64_t tokens, int experts, int topk, int sigmoid,
                                     const int32_t* cu_seqlens, int sequences, const uint8_t* is_padding, const void* saved,
                                     const float* dloss, void* dlogits, void* stream) {
  using namespace moe;
  const int rc = check("balance_loss_grad", tokens, experts, topk, sequences, dtype, ld);
  if (rc || tokens == 0) return rc;
  if (!logits || !saved || !dloss || !dlogits || (!cu_seqlens && sequences != 1)) return fail(MOE_E_BADARG, "balance_loss_grad: bad argument");
  const Plan plan = plan_of(logits, ld, dlogits, dtype, tokens, experts);
  const Balance b = {logits, ld, nullptr, cu_seqlens, is_padding, tokens, experts, topk, sequences, 0, sigmoid != 0, plan.rows, plan.lanes};
  cudaStream_t st = (cudaStream_t)stream;
#define MOE_BG(T, V, CH)                                                                                                               \
  launch_pdl(balance_grad_kernel<T, V, CH>, dim3((unsigned)plan.blocks), kThreads, 0, 1, st, "balance_loss_grad", b, (const int32_t*)saved, \
             dloss, (T*)dlogits)
  return MOE_BALANCE_DISPATCH(MOE_BG, dtype, plan, experts);
#undef MOE_BG
}
