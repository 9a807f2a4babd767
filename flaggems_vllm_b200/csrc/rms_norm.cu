// Root-mean-square norm of the residual stream, with the residual's addition in front of it, an 8-bit output behind it, and
// its gradient.
//
//   h = round(x + residual)          the stream as it is stored (h = x without a residual)
//   r = 1 / sqrt(mean(h^2) + eps),  y_i = w_i h_i r
//   quantised: s = max(amax |y|, quant_eps) / qmax per group of a row or per row,  q = round(y / s)
//   dh_i = r (w_i dy_i - h_i r^2 mean(w dy h)) + (gradient that reaches the stream directly),  dw_i = sum over rows dy_i h_i r
//
// The norm is that of the rounded h, not of the sum in fp32: what the next layer adds to is what was normed, and the
// gradient, which has only h, is that of the same function.  y itself is rounded once: the quantiser takes its fp32 value.
// The gradient computes r again (the row is in registers anyway), so nothing but h is kept between the two passes.
//
// Bound: memory.  A row is read once: it stays in the registers of the threads that share it, 64 bytes to a thread (32 values of 16
// bits, 16 of fp32; four or eight where rows are not made of 16-byte pieces) so that four blocks of 256 threads, and their loads,
// are on a multiprocessor.  us on the device, 8192 x 7168 bf16 with a residual (470 MB: 72 at the rate of a copy): norm 69.7; e4m3
// in groups of 128 70.7 (411 MB: 63), e5m2 73.2, with the norm itself 82 (528 MB: 81); int8 per row 68.6; gradient 85, of which 5
// for the weight's (470 MB: 72).  16 or 64 values of bf16 to a thread instead: 3 to 6 % slower.  One token of 7168: 2.4, a launch
// and one round of loads.
#include "moe_common.cuh"

namespace moe {
namespace {

// Two 16-bit values as fp32 and back, an instruction or less per value: element by element the norm took 21 instructions per
// element and its gradient 30, and both waited for the integer pipe.
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t v);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
}
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// V consecutive elements that one thread moves at once: 32 or 16 bytes, or a single element where rows are not made of such
// pieces.  Loads and stores of 32 bytes are sm_100's own.
template <typename T, int V> struct Piece {
  static constexpr int W = V * (int)sizeof(T) / 4;
  static_assert(W == 8 || W == 4, "16 or 32 bytes");
  uint32_t raw[W] = {};
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (W == 8) {
      asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                   : "=r"(raw[0]), "=r"(raw[1]), "=r"(raw[2]), "=r"(raw[3]), "=r"(raw[4]), "=r"(raw[5]), "=r"(raw[6]), "=r"(raw[7])
                   : "l"(p));
    } else {
      set_raw(*reinterpret_cast<const uint4*>(p));
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (W == 8)
      asm volatile("st.global.v8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(raw[0]), "r"(raw[1]), "r"(raw[2]), "r"(raw[3]), "r"(raw[4]),
                   "r"(raw[5]), "r"(raw[6]), "r"(raw[7]), "l"(p)
                   : "memory");
    else
      *reinterpret_cast<uint4*>(p) = make_uint4(raw[0], raw[1], raw[2], raw[3]);
  }
  __device__ __forceinline__ void set_raw(uint4 v) { raw[0] = v.x; raw[1] = v.y; raw[2] = v.z; raw[3] = v.w; }
  __device__ __forceinline__ void get(float (&v)[V]) const {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      if constexpr (sizeof(T) == 4) {
        v[i] = __uint_as_float(raw[i]);
      } else {
        const float2 f = unpack2<T>(raw[i]);
        v[2 * i] = f.x; v[2 * i + 1] = f.y;
      }
    }
  }
  __device__ __forceinline__ void set(const float (&v)[V]) {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      if constexpr (sizeof(T) == 4) raw[i] = __float_as_uint(v[i]);
      else raw[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
    }
  }
};
template <typename T> struct Piece<T, 1> {
  T raw = from_f32<T>(0.0f);
  __device__ __forceinline__ void load(const T* p) { raw = *p; }
  __device__ __forceinline__ void store(T* p) const { *p = raw; }
  __device__ __forceinline__ void get(float (&v)[1]) const { v[0] = ToF32<T>::get(raw); }
  __device__ __forceinline__ void set(const float (&v)[1]) { raw = from_f32<T>(v[0]); }
};

// The V weights from element `at` on; the weight has the type of the rows or is fp32.
template <typename T, int V>
__device__ __forceinline__ void load_weight(const void* w, bool w_f32, int at, float (&v)[V]) {
  if (w_f32) {
    const float* p = reinterpret_cast<const float*>(w) + at;
    if constexpr (V == 1) {
      v[0] = *p;
    } else {
#pragma unroll
      for (int i = 0; i < V; i += 4) {
        const float4 f = *reinterpret_cast<const float4*>(p + i);
        v[i] = f.x; v[i + 1] = f.y; v[i + 2] = f.z; v[i + 3] = f.w;
      }
    }
  } else {
    Piece<T, V> p;
    p.load(reinterpret_cast<const T*>(w) + at);
    p.get(v);
  }
}

struct Sum { static __device__ __forceinline__ float join(float a, float b) { return a + b; } };
struct Max { static __device__ __forceinline__ float join(float a, float b) { return max_nan(a, b); } };

// N values joined over the TPR threads of a row; every thread gets the same bits (fixed order).  `sh` holds N floats per
// warp of the block; a caller that comes again puts a barrier between.  WHOLE: the block has no other rows at the time (else
// the row's threads meet at a barrier of their own).
template <class Op, int N, int TPR, bool WHOLE = true>
__device__ __forceinline__ void join_row(float (&v)[N], float* sh) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1)
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = Op::join(v[n], __shfl_xor_sync(0xFFFFFFFFu, v[n], off));
  if constexpr (TPR > 32) {
    const int warp = threadIdx.x >> 5, first = warp / (TPR / 32) * (TPR / 32);
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int n = 0; n < N; ++n) sh[warp * N + n] = v[n];
    if constexpr (WHOLE) __syncthreads();
    else asm volatile("bar.sync %0, %1;" ::"r"(first / (TPR / 32) + 1), "n"(TPR) : "memory");
    // every warp joins the warps' values again, a lane each: a dozen instructions where reading them all took four times as many
    constexpr int W = TPR / 32;
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = sh[(first + (lane & (W - 1))) * N + n];
#pragma unroll
    for (int off = W / 2; off > 0; off >>= 1)
#pragma unroll
      for (int n = 0; n < N; ++n) v[n] = Op::join(v[n], __shfl_xor_sync(0xFFFFFFFFu, v[n], off));
  }
}

// 1 / sqrt(x): the approximation and one step of Newton's method, within two roundings; 0 for infinity, NaN for NaN.
__device__ __forceinline__ float inverse_root(float x) {
  const float r = rsqrtf(x);
  const float better = r * fmaf(-0.5f * x * r, r, 1.5f);
  return x > 1e-30f && x < 1e30f ? better : r;
}

enum { kNone = -1, kE4M3 = 0, kE5M2 = 1, kInt8 = 2 };
__device__ __forceinline__ constexpr float quant_max(int format) { return format == kE4M3 ? 448.0f : format == kE5M2 ? 57344.0f : 127.0f; }

// The scale of a group from its largest magnitude.  A NaN in the group makes the scale NaN, as it makes the values it stands for.
__device__ __forceinline__ float group_scale(float amax, float eps, int format, bool ue8m0) {
  float s = max_nan(amax, eps) * (1.0f / quant_max(format));
  if (ue8m0 && s < INFINITY) {  // the smallest power of two that is not below it, nor below 1e-10: the stand-alone quantiser's rule
    s = fmaxf(s, 1e-10f);
    const uint32_t b = __float_as_uint(s);
    s = __uint_as_float((b + 0x7FFFFFu) & 0x7F800000u);
  }
  return s;
}

__device__ __forceinline__ uint8_t to_8bit(float v, int format) {  // fp8 conversions saturate and keep NaN
  if (format == kE4M3) return (uint8_t)__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
  if (format == kE5M2) return (uint8_t)__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E5M2);
  return (uint8_t)(int8_t)max(-128, min(127, __float2int_rn(v)));  // NaN gives 0; its scale is NaN
}

// A scale of zero (no floor under it, and nothing in the group) stands over zeros.
__device__ __forceinline__ float quotient(float y, float s) { return s == 0.0f ? 0.0f : y / s; }

// Four values rounded to the nearest whole number, halves to even, and cut to [-128, 127].
__device__ __forceinline__ uint32_t pack_int8(float a, float b, float c, float d) {
  uint32_t hi, out;
  asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, 0;" : "=r"(hi) : "r"(__float2int_rn(d)), "r"(__float2int_rn(c)));
  asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, %3;" : "=r"(out) : "r"(__float2int_rn(b)), "r"(__float2int_rn(a)), "r"(hi));
  return out;
}

// V quotients of one piece as bytes.
template <int V>
__device__ __forceinline__ void quantise(const float (&y)[V], float s, int format, uint8_t* dst) {
  float d[V];
  if (s > 1e-20f && s < 1e30f) {  // where div_by_scale() gives the bytes of the division
    const float inv = 1.0f / s;
#pragma unroll
    for (int i = 0; i < V; ++i) d[i] = div_by_scale(y[i], s, inv);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) d[i] = quotient(y[i], s);
  }
  uint32_t w[(V + 3) / 4] = {};
  if (format == kE4M3 && V % 4 == 0) {
#pragma unroll
    for (int i = 0; i + 3 < V; i += 4) {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(d[i], d[i + 1]), __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(d[i + 2], d[i + 3]), __NV_SATFINITE, __NV_E4M3);
      w[i / 4] = lo | hi << 16;
    }
  } else if (format == kInt8 && V % 4 == 0) {
#pragma unroll
    for (int i = 0; i + 3 < V; i += 4) w[i / 4] = pack_int8(d[i], d[i + 1], d[i + 2], d[i + 3]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) w[i / 4] |= (uint32_t)to_8bit(d[i], format) << (8 * (i & 3));
  }
  if constexpr (V == 16) *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
  else if constexpr (V == 8) *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
  else if constexpr (V == 4) *reinterpret_cast<uint32_t*>(dst) = w[0];
  else *dst = (uint8_t)w[0];
}

struct Forward {
  const void *x, *residual, *weight;  // residual: null = none
  void *y, *h;                        // y: null = not wanted; h: null without a residual
  int64_t x_ld, residual_ld, y_ld, h_ld, rows;
  int cols, w_f32;
  float eps, mean;  // mean: 1 / cols
  // 8-bit output
  uint8_t* q;
  float* scales;
  int64_t scale_ld;  // of the transposed layout
  int group, groups, format, transposed, ue8m0;
  float quant_eps;
};

__device__ __forceinline__ float* scale_at(const Forward& p, int64_t row, int group_index) {
  return p.transposed ? p.scales + (int64_t)group_index * p.scale_ld + row : p.scales + row * p.groups + group_index;
}

// One row per TPR threads, kept in registers: CH pieces of V elements per thread.  x and y (residual and h) may be the same
// memory: a thread has read its pieces before it writes them, and nobody else reads them.
template <typename T, int V, int TPR, int CH, int FORMAT, int BLOCK = (TPR > 128 ? TPR : 128)>
__global__ void __launch_bounds__(BLOCK) rms_norm_kernel(const Forward p) {
  constexpr bool QUANT = FORMAT != kNone;
  pdl_wait();
  pdl_trigger();
  __shared__ float sh[2][BLOCK / 32];
  const int t = threadIdx.x % TPR, pieces = p.cols / V;
  const int64_t row = (int64_t)blockIdx.x * (BLOCK / TPR) + threadIdx.x / TPR;
  if (row >= p.rows) return;  // whole warps, and all threads of a row: no barrier is left short
  float h[CH][V];  // the stream, then its norm
  {
    const T* x = reinterpret_cast<const T*>(p.x) + row * p.x_ld;
    Piece<T, V> a[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c)
      if (t + c * TPR < pieces) a[c].load(x + (t + c * TPR) * V);
    if (p.residual != nullptr) {
      const T* r = reinterpret_cast<const T*>(p.residual) + row * p.residual_ld;
      Piece<T, V> b[CH];
#pragma unroll
      for (int c = 0; c < CH; ++c)
        if (t + c * TPR < pieces) b[c].load(r + (t + c * TPR) * V);
      T* out = reinterpret_cast<T*>(p.h) + row * p.h_ld;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        float u[V], v[V];
        a[c].get(u);
        b[c].get(v);
#pragma unroll
        for (int i = 0; i < V; ++i) u[i] += v[i];
        a[c].set(u);
        if (t + c * TPR < pieces) a[c].store(out + (t + c * TPR) * V);
      }
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) a[c].get(h[c]);
  }
  float ss[1] = {0.0f};
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int i = 0; i < V; ++i) ss[0] = fmaf(h[c][i], h[c][i], ss[0]);
  join_row<Sum, 1, TPR, TPR == BLOCK>(ss, sh[0]);
  const float inv = inverse_root(fmaf(ss[0], p.mean, p.eps));
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    if (t + c * TPR < pieces) {
      float w[V];
      load_weight<T, V>(p.weight, p.w_f32, (t + c * TPR) * V, w);
#pragma unroll
      for (int i = 0; i < V; ++i) h[c][i] = h[c][i] * inv * w[i];
      if (!QUANT || p.y != nullptr) {
        Piece<T, V> o;
        o.set(h[c]);
        o.store(reinterpret_cast<T*>(p.y) + row * p.y_ld + (t + c * TPR) * V);
      }
    }
  }
  if constexpr (QUANT) {
    float amax[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      amax[c] = 0.0f;
#pragma unroll
      for (int i = 0; i < V; ++i) amax[c] = max_nan(amax[c], fabsf(h[c][i]));  // zero beyond the row
    }
    uint8_t* q = p.q + row * p.cols;
    if (p.group == p.cols) {
      float m[1] = {amax[0]};
#pragma unroll
      for (int c = 1; c < CH; ++c) m[0] = max_nan(m[0], amax[c]);
      join_row<Max, 1, TPR, TPR == BLOCK>(m, sh[1]);
      const float s = group_scale(m[0], p.quant_eps, FORMAT, p.ue8m0);
      if (t == 0) *scale_at(p, row, 0) = s;
#pragma unroll
      for (int c = 0; c < CH; ++c)
        if (t + c * TPR < pieces) quantise<V>(h[c], s, FORMAT, q + (t + c * TPR) * V);
    } else {
      // the pieces of a group, a power of two up to 32, lie in one warp
      const int lanes = p.group / V, shift = 31 - __clz(lanes);
      float* scales = scale_at(p, row, 0);
      const int64_t apart = p.transposed ? p.scale_ld : 1;
      for (int off = lanes / 2; off > 0; off >>= 1)
#pragma unroll
        for (int c = 0; c < CH; ++c) amax[c] = max_nan(amax[c], __shfl_xor_sync(0xFFFFFFFFu, amax[c], off));
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int piece = t + c * TPR;
        if (piece < pieces) {
          const float s = group_scale(amax[c], p.quant_eps, FORMAT, p.ue8m0);
          if ((piece & (lanes - 1)) == 0) scales[(piece >> shift) * apart] = s;
          quantise<V>(h[c], s, FORMAT, q + piece * V);
        }
      }
    }
  }
}

// N sums over a row of any length, this thread's share of them: term(i, s) adds what element i gives.  16 terms at a time are added
// in fp32 and their sum to one in fp64.  One fp32 sum over millions of columns would drift: a term of 1.21 added to 65536 loses up
// to 2^-8, the same way every time.  us for the gradient of 4096 x 8191 bf16: one sum 153; unrolled by four or eight 170-176, in
// full 157, by a count of 16 152.
template <int N, class Term>
__device__ __forceinline__ void sum_long(int cols, float (&s)[N], Term term) {
  double total[N] = {};
  int i = threadIdx.x;
  float part[N] = {};
  while (i + 15 * 256 < cols) {
#pragma unroll 16
    for (int j = 0; j < 16; ++j) term(i + 256 * j, part);
    i += 256 * 16;
#pragma unroll
    for (int n = 0; n < N; ++n) { total[n] += part[n]; part[n] = 0.0f; }
  }
  for (; i < cols; i += 256) term(i, part);
#pragma unroll
  for (int n = 0; n < N; ++n) total[n] += part[n];
#pragma unroll
  for (int n = 0; n < N; ++n) s[n] = (float)total[n];
}

// Any row length, alignment and group: a block per row, which is read again instead of kept.
template <typename T>
__global__ void __launch_bounds__(256) rms_norm_any_kernel(const Forward p) {
  pdl_wait();
  pdl_trigger();
  __shared__ float sh[2][8];
  const int64_t row = blockIdx.x;
  const T* x = reinterpret_cast<const T*>(p.x) + row * p.x_ld;
  const T* src = x;
  float ss[1];
  if (p.residual != nullptr) {
    const T* r = reinterpret_cast<const T*>(p.residual) + row * p.residual_ld;
    T* out = reinterpret_cast<T*>(p.h) + row * p.h_ld;
    sum_long(p.cols, ss, [&](int i, float (&s)[1]) {
      const T v = from_f32<T>(ToF32<T>::get(x[i]) + ToF32<T>::get(r[i]));
      out[i] = v;
      s[0] = fmaf(ToF32<T>::get(v), ToF32<T>::get(v), s[0]);
    });
    src = out;
  } else {
    sum_long(p.cols, ss, [&](int i, float (&s)[1]) { s[0] = fmaf(ToF32<T>::get(x[i]), ToF32<T>::get(x[i]), s[0]); });
  }
  join_row<Sum, 1, 256>(ss, sh[0]);  // its barrier also makes h visible to the block
  const float inv = inverse_root(fmaf(ss[0], p.mean, p.eps));
  auto norm = [&](int i) {
    const float w = p.w_f32 ? reinterpret_cast<const float*>(p.weight)[i] : ToF32<T>::get(reinterpret_cast<const T*>(p.weight)[i]);
    return ToF32<T>::get(src[i]) * inv * w;
  };
  if (p.q != nullptr) {
    uint8_t* q = p.q + row * p.cols;
    if (p.group == p.cols) {
      float m[1] = {0.0f};
      for (int i = threadIdx.x; i < p.cols; i += 256) m[0] = max_nan(m[0], fabsf(norm(i)));
      join_row<Max, 1, 256>(m, sh[1]);
      const float s = group_scale(m[0], p.quant_eps, p.format, p.ue8m0);
      if (threadIdx.x == 0) *scale_at(p, row, 0) = s;
      for (int i = threadIdx.x; i < p.cols; i += 256) q[i] = to_8bit(quotient(norm(i), s), p.format);
    } else {  // a warp per group
      const int lane = threadIdx.x & 31;
      for (int g = threadIdx.x >> 5; g < p.groups; g += 8) {
        float m[1] = {0.0f};
        for (int i = lane; i < p.group; i += 32) m[0] = max_nan(m[0], fabsf(norm(g * p.group + i)));
        join_row<Max, 1, 32>(m, nullptr);
        const float s = group_scale(m[0], p.quant_eps, p.format, p.ue8m0);
        if (lane == 0) *scale_at(p, row, g) = s;
        for (int i = lane; i < p.group; i += 32) q[g * p.group + i] = to_8bit(quotient(norm(g * p.group + i), s), p.format);
      }
    }
  }
  // y may lie over x, which nothing reads once there is an h, and without an h (no residual) y is memory of its own
  if (p.y != nullptr) {
    T* y = reinterpret_cast<T*>(p.y) + row * p.y_ld;
    for (int i = threadIdx.x; i < p.cols; i += 256) y[i] = from_f32<T>(norm(i));
  }
}

struct Backward {
  const void *dy, *dh, *h, *weight;  // dh: null = none
  void *dx;                          // null = not wanted
  float* partial;                    // [blocks, cols] sums of dw; null = not wanted
  int64_t h_ld, rows;
  int cols, w_f32;
  float eps, mean;  // mean: 1 / cols
};

// 16 bytes into shared memory behind the thread's back.
__device__ __forceinline__ void copy16(uint4* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}

// Rows made of 16-byte pieces: TPR threads to a row, THREADS / TPR rows of a block at a time, dealt out in turn; a thread keeps its
// columns' part of dw in registers over all of them.  The rows to come are on their way into shared memory meanwhile.  A thread
// fetches the pieces that it reads itself, so the copies need no barrier, only the thread's own wait: per row there is the one
// barrier of the two sums.  STAGES rows of dy, h and dh per group of threads make up to 196 KB in flight on a multiprocessor.
template <typename T, int TPR, int CH, int STAGES, int THREADS>
__global__ void __launch_bounds__(THREADS, 1) rms_norm_grad_kernel(const Backward p) {
  constexpr int V = 16 / sizeof(T), GROUPS = THREADS / TPR;
  static_assert(TPR == 32 || GROUPS <= 15, "a named barrier for each group beside the block's own");
  extern __shared__ uint4 ring[];  // [STAGES][3][CH][threads]
  __shared__ float sh[2][THREADS / 32 * 2];
  pdl_wait();
  pdl_trigger();
  const int t = threadIdx.x % TPR, group = threadIdx.x / TPR, pieces = p.cols / V;
  const int64_t row0 = (int64_t)group * gridDim.x + blockIdx.x, step = (int64_t)GROUPS * gridDim.x;
  const bool with_dh = p.dh != nullptr && p.dx != nullptr;
  auto slot = [&](int stage, int n, int c) { return ring + ((stage * 3 + n) * CH + c) * THREADS + threadIdx.x; };
  const T *h_next = reinterpret_cast<const T*>(p.h) + row0 * p.h_ld + t * V,  // this thread's pieces of the next row to fetch
          *dy_next = reinterpret_cast<const T*>(p.dy) + row0 * p.cols + t * V, *dh_next = reinterpret_cast<const T*>(p.dh) + row0 * p.cols + t * V;
  T* dx = reinterpret_cast<T*>(p.dx) + row0 * p.cols + t * V;
  const int64_t h_step = step * p.h_ld, step_elements = step * p.cols;
  auto fetch = [&](int64_t row, int stage) {
    if (row < p.rows) {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        if (t + c * TPR < pieces) {
          copy16(slot(stage, 0, c), h_next + c * TPR * V);
          copy16(slot(stage, 1, c), dy_next + c * TPR * V);
          if (with_dh) copy16(slot(stage, 2, c), dh_next + c * TPR * V);
        }
      }
      h_next += h_step;
      dy_next += step_elements;
      dh_next += step_elements;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  float dw[CH][V];
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int i = 0; i < V; ++i) dw[c][i] = 0.0f;
#pragma unroll
  for (int i = 0; i < STAGES; ++i) {
    if (!with_dh)
#pragma unroll
      for (int c = 0; c < CH; ++c) *slot(i, 2, c) = make_uint4(0, 0, 0, 0);  // and it stays so: nothing is added
    fetch(row0 + i * step, i);
  }
  int stage = 0, turn = 0;
  for (int64_t row = row0; row < p.rows; row += step, turn ^= 1) {
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      if (t + c * TPR < pieces) {
        Piece<T, V> a;
        float h[V], g[V], w[V];
        a.set_raw(*slot(stage, 0, c));
        a.get(h);
        a.set_raw(*slot(stage, 1, c));
        a.get(g);
        load_weight<T, V>(p.weight, p.w_f32, (t + c * TPR) * V, w);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          s[0] = fmaf(h[i], h[i], s[0]);
          s[1] = fmaf(w[i] * g[i], h[i], s[1]);
        }
      }
    }
    join_row<Sum, 2, TPR, TPR == THREADS>(s, sh[turn]);  // the other half is still read by threads that are a row behind
    const float inv = inverse_root(fmaf(s[0], p.mean, p.eps));
    const float k = inv * (s[1] * p.mean);  // r^2 itself is infinite for rows below 5e-20 where eps is zero
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      if (t + c * TPR < pieces) {
        Piece<T, V> a;
        float h[V], g[V], d[V], w[V];  // read again: kept in registers beside dw they would spill
        a.set_raw(*slot(stage, 0, c));
        a.get(h);
        a.set_raw(*slot(stage, 1, c));
        a.get(g);
        a.set_raw(*slot(stage, 2, c));
        a.get(d);
        load_weight<T, V>(p.weight, p.w_f32, (t + c * TPR) * V, w);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float x = h[i] * inv;
          dw[c][i] = fmaf(g[i], x, dw[c][i]);
          d[i] = fmaf(inv, fmaf(-x, k, w[i] * g[i]), d[i]);
        }
        if (p.dx != nullptr) {
          a.set(d);
          a.store(dx + c * TPR * V);
        }
      }
    }
    dx += step_elements;
    fetch(row + STAGES * step, stage);  // over what this thread alone has read, and used
    stage = stage + 1 == STAGES ? 0 : stage + 1;
  }
  if (p.partial == nullptr) return;
  asm volatile("cp.async.wait_all;" ::: "memory");
  // the groups' sums meet in shared memory, in order
  float* acc = reinterpret_cast<float*>(ring);
  for (int r = 0; r < GROUPS; ++r) {
    __syncthreads();
    if (group == r) {
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (t + c * TPR < pieces) {
            float* a = acc + (t + c * TPR) * V + i;
            *a = r == 0 ? dw[c][i] : *a + dw[c][i];
          }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < p.cols; i += THREADS) p.partial[(int64_t)blockIdx.x * p.cols + i] = acc[i];
}

// Rows that are not: element by element, straight into registers.
template <typename T, int TPR, int CH, int BLOCK = (TPR > 128 ? TPR : 128)>
__global__ void __launch_bounds__(BLOCK) rms_norm_grad_single_kernel(const Backward p) {
  pdl_wait();
  pdl_trigger();
  constexpr int RPB = BLOCK / TPR;
  __shared__ float sh[2][BLOCK / 32 * 2];
  const int t = threadIdx.x % TPR;
  float dw[CH] = {};
  int turn = 0;
  auto weight = [&](int i) {
    return p.w_f32 ? reinterpret_cast<const float*>(p.weight)[i] : ToF32<T>::get(reinterpret_cast<const T*>(p.weight)[i]);
  };
  for (int64_t row = (int64_t)(threadIdx.x / TPR) * gridDim.x + blockIdx.x; row < p.rows; row += (int64_t)gridDim.x * RPB, turn ^= 1) {
    float h[CH], g[CH], d[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int at = t + c * TPR;
      h[c] = g[c] = d[c] = 0.0f;
      if (at < p.cols) {
        h[c] = ToF32<T>::get(reinterpret_cast<const T*>(p.h)[row * p.h_ld + at]);
        g[c] = ToF32<T>::get(reinterpret_cast<const T*>(p.dy)[row * p.cols + at]);
        if (p.dh != nullptr) d[c] = ToF32<T>::get(reinterpret_cast<const T*>(p.dh)[row * p.cols + at]);
      }
    }
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      if (t + c * TPR < p.cols) {
        s[0] = fmaf(h[c], h[c], s[0]);
        s[1] = fmaf(weight(t + c * TPR) * g[c], h[c], s[1]);
      }
    }
    join_row<Sum, 2, TPR, TPR == BLOCK>(s, sh[turn]);
    const float inv = inverse_root(fmaf(s[0], p.mean, p.eps));
    const float k = inv * (s[1] * p.mean);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int at = t + c * TPR;
      if (at < p.cols) {
        const float x = h[c] * inv;
        dw[c] = fmaf(g[c], x, dw[c]);
        if (p.dx != nullptr) reinterpret_cast<T*>(p.dx)[row * p.cols + at] = from_f32<T>(fmaf(inv, fmaf(-x, k, weight(at) * g[c]), d[c]));
      }
    }
  }
  if (p.partial == nullptr) return;
  __shared__ float acc[RPB > 1 ? TPR * CH : 1];
  for (int r = 0; r < RPB; ++r) {  // the rows at a time of a block: their threads' sums meet in order
    if (RPB > 1) __syncthreads();
    if ((int)threadIdx.x / TPR == r) {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int at = t + c * TPR;
        if (at >= p.cols) continue;
        const float v = r == 0 ? dw[c] : acc[RPB > 1 ? at : 0] + dw[c];
        if (r + 1 == RPB) p.partial[(int64_t)blockIdx.x * p.cols + at] = v;
        else acc[at] = v;
      }
    }
  }
}

// dw[col] = sum over the blocks' partial sums, in order: 32 columns per block, 32 threads to a column, N parts of each in flight
// (with 5 a part of every multiprocessor is one round).  What the kernel in front writes has no __restrict__: this one may have
// started meanwhile, and loads that the compiler takes for read-only need not stay behind the wait.
template <typename W, int N>
__global__ void __launch_bounds__(1024) weight_grad_kernel(const float* partial, int parts, int cols, W* __restrict__ dw) {
  pdl_wait();
  pdl_trigger();
  __shared__ float sh[32][33];
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), r = threadIdx.x >> 5;
  float s = 0.0f;
  for (int i = r; i < parts; i += 32 * N) {
    float v[N];
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = col < cols && i + 32 * j < parts ? partial[(int64_t)(i + 32 * j) * cols + col] : 0.0f;
#pragma unroll
    for (int j = 0; j < N; ++j) s += v[j];
  }
  sh[r][threadIdx.x & 31] = s;
  __syncthreads();
  s = sh[threadIdx.x & 31][r];
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, off);
  const int out = blockIdx.x * 32 + r;
  if ((threadIdx.x & 31) == 0 && out < cols) dw[out] = from_f32<W>(s);
}

// Any row length: dx with the rows read twice, r of every row kept for the columns' kernel behind.
template <typename T>
__global__ void __launch_bounds__(256) rms_norm_grad_any_kernel(const Backward p, float* __restrict__ inv_rms) {
  pdl_wait();
  pdl_trigger();
  __shared__ float sh[16];
  const int64_t row = blockIdx.x;
  const T* h = reinterpret_cast<const T*>(p.h) + row * p.h_ld;
  const T* dy = reinterpret_cast<const T*>(p.dy) + row * p.cols;
  auto weight = [&](int i) {
    return p.w_f32 ? reinterpret_cast<const float*>(p.weight)[i] : ToF32<T>::get(reinterpret_cast<const T*>(p.weight)[i]);
  };
  float s[2];
  sum_long(p.cols, s, [&](int i, float (&s)[2]) {
    const float hv = ToF32<T>::get(h[i]);
    s[0] = fmaf(hv, hv, s[0]);
    s[1] = fmaf(weight(i) * ToF32<T>::get(dy[i]), hv, s[1]);
  });
  join_row<Sum, 2, 256>(s, sh);
  const float inv = inverse_root(fmaf(s[0], p.mean, p.eps));
  const float k = inv * (s[1] * p.mean);
  if (inv_rms != nullptr && threadIdx.x == 0) inv_rms[row] = inv;
  if (p.dx == nullptr) return;
  for (int i = threadIdx.x; i < p.cols; i += 256) {
    const float d = p.dh != nullptr ? ToF32<T>::get(reinterpret_cast<const T*>(p.dh)[row * p.cols + i]) : 0.0f;
    const float x = ToF32<T>::get(h[i]) * inv;
    reinterpret_cast<T*>(p.dx)[row * p.cols + i] = from_f32<T>(fmaf(inv, fmaf(-x, k, weight(i) * ToF32<T>::get(dy[i])), d));
  }
}
template <typename T>
__global__ void __launch_bounds__(256) weight_grad_any_kernel(const Backward p, const float* inv_rms) {
  pdl_wait();
  pdl_trigger();
  const int col = blockIdx.x * 256 + threadIdx.x;
  if (col >= p.cols) return;
  float s = 0.0f;
  for (int64_t row = blockIdx.y; row < p.rows; row += gridDim.y)
    s = fmaf(ToF32<T>::get(reinterpret_cast<const T*>(p.dy)[row * p.cols + col]),
             ToF32<T>::get(reinterpret_cast<const T*>(p.h)[row * p.h_ld + col]) * inv_rms[row], s);
  p.partial[(int64_t)blockIdx.y * p.cols + col] = s;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
bool pieces16(const void* p, int64_t ld, int size) { return aligned16(p) && ld * size % 16 == 0; }

// Threads to a row that give each all pieces that it holds, `held` of them in flight at once; 0 = the kernel for any row.
int threads_of(int pieces, int held) {
  for (int threads = 32; threads <= 1024; threads *= 2)
    if (pieces <= threads * held) return threads;
  return 0;
}

template <typename T, int V, int TPR, int CH, int FORMAT>
int launch_rows(const Forward& p, cudaStream_t st) {
  constexpr int block = TPR > 128 ? TPR : 128, at_a_time = block / TPR;
  return launch_pdl(rms_norm_kernel<T, V, TPR, CH, FORMAT>, dim3((unsigned)((p.rows + at_a_time - 1) / at_a_time)), block, 0, 1, st, "rms_norm", p);
}

template <typename T, int V, int CH, int FORMAT>
int launch_pieces(const Forward& p, cudaStream_t st) {
  const int threads = threads_of(p.cols / V, CH), lanes = p.group / V;
  // groups of a power of two of pieces within a warp, or whole rows, are quantised from registers
  const bool held = FORMAT == kNone || p.group == p.cols || (p.group % V == 0 && lanes <= 32 && (lanes & (lanes - 1)) == 0);
  switch (held ? threads : 0) {
    case 32: return launch_rows<T, V, 32, CH, FORMAT>(p, st);
    case 64: return launch_rows<T, V, 64, CH, FORMAT>(p, st);
    case 128: return launch_rows<T, V, 128, CH, FORMAT>(p, st);
    case 256: return launch_rows<T, V, 256, CH, FORMAT>(p, st);
    case 512: return launch_rows<T, V, 512, CH, FORMAT>(p, st);
    case 1024: return launch_rows<T, V, 1024, CH, FORMAT>(p, st);
  }
  if (V == 1 && held && p.cols <= 1024 * 8) return launch_rows<T, 1, 1024, 8, FORMAT>(p, st);
  return launch_pdl(rms_norm_any_kernel<T>, dim3((unsigned)p.rows), 256, 0, 1, st, "rms_norm", p);
}

// `piece`: bytes that rows and pointers are made of, 32 or 16, or fewer.  With 32 each lane's part of a group is twice as long (its
// largest value, scale and reciprocal are half the work per value) and half as many loads and stores are issued: 8192 x 7168 bf16
// in groups of 128 in 70.4 us, 77.7 in pieces of 16; the norm alone 69.5 and 71.0.
template <typename T, int FORMAT>
int launch_forward(const Forward& p, int piece, cudaStream_t st) {
  constexpr int S = sizeof(T);
  if (piece == 32 && p.group % (32 / S) == 0) return launch_pieces<T, 32 / S, 2, FORMAT>(p, st);
  if (piece >= 16) return launch_pieces<T, 16 / S, 4, FORMAT>(p, st);
  return launch_pieces<T, 1, 4, FORMAT>(p, st);
}

template <typename T>
int launch_format(const Forward& p, int piece, cudaStream_t st) {
  if (p.q == nullptr) return launch_forward<T, kNone>(p, piece, st);
  switch (p.format) {
    case kE4M3: return launch_forward<T, kE4M3>(p, piece, st);
    case kE5M2: return launch_forward<T, kE5M2>(p, piece, st);
    default: return launch_forward<T, kInt8>(p, piece, st);
  }
}

int forward(const Forward& p, int dtype, cudaStream_t st) {
  const int size = dtype == MOE_F32 ? 4 : 2;
  uint64_t bits = (uint64_t)p.cols * size | (uintptr_t)p.x | (uintptr_t)p.weight | (uintptr_t)p.y | (uintptr_t)p.q;
  if (p.rows > 1) bits |= (uint64_t)p.x_ld * size | (p.y ? (uint64_t)p.y_ld * size : 0);
  if (p.residual) {
    bits |= (uintptr_t)p.residual | (uintptr_t)p.h;
    if (p.rows > 1) bits |= (uint64_t)(p.residual_ld | p.h_ld) * size;
  }
  const int piece = bits % 32 == 0 ? 32 : bits % 16 == 0 ? 16 : 1;
  switch (dtype) {
    case MOE_F32: return launch_format<float>(p, piece, st);
    case MOE_F16: return launch_format<__half>(p, piece, st);
    default: return launch_format<__nv_bfloat16>(p, piece, st);
  }
}

constexpr int64_t kMaxRows = 0x7FFFFFFF;  // blocks of a grid

// Checks that both forward entry points share.
int check_forward(const char* who, const void* x, int dtype, int weight_dtype, const void* residual, const void* weight, int64_t rows,
                  int64_t cols, float eps, int64_t x_ld, int64_t residual_ld, void* h, int64_t h_ld) {
  if (rows < 0 || cols <= 0 || cols > (1 << 24)) return fail(MOE_E_BADARG, "%s: bad extent", who);
  if (rows > kMaxRows) return fail(MOE_E_TOOBIG, "%s: too many rows", who);
  if (dtype != MOE_F32 && dtype != MOE_F16 && dtype != MOE_BF16) return fail(MOE_E_DTYPE, "%s: unsupported dtype %d", who, dtype);
  if (weight_dtype != dtype && weight_dtype != MOE_F32) return fail(MOE_E_DTYPE, "%s: the weight is fp32 or of the rows' type", who);
  if (!(eps >= 0.0f) || !(eps < 3.0e38f)) return fail(MOE_E_BADARG, "%s: eps must be finite and not negative", who);
  if (rows == 0) return 0;
  if (!x || !weight || (residual && !h)) return fail(MOE_E_BADARG, "%s: null pointer", who);
  if (x_ld < 0 || (residual && (residual_ld < 0 || (h_ld < cols && rows > 1)))) return fail(MOE_E_BADARG, "%s: bad row distance", who);
  return 0;
}

// Blocks of the gradient, each with its part of dw: one to a multiprocessor, whose shared memory it fills, or, element by element,
// as many as make 1024 threads (8192 x 501 bf16: 28 us with two of 256 threads, 17 with eight of 128).  The parts of long rows take
// 256 MB at most, or 16 rows: two to a multiprocessor would be 20 GB for 2^24 columns, whose columns alone fill the device.
int grad_blocks(int64_t rows, int64_t cols, bool vector) {
  int64_t most = (int64_t)sm_count() * (vector ? 1 : cols <= 128 * 4 ? 8 : cols <= 256 * 4 ? 4 : 2);
  const int64_t room = (int64_t)(256 << 20) / 4 / cols;
  if (most > room) most = room > 16 ? room : 16;
  return (int)(rows < most ? rows : most);
}

template <typename W>
int sum_parts(const float* partial, int parts, int cols, W* dw, cudaStream_t st) {
  const dim3 grid((unsigned)((cols + 31) / 32));
  return parts <= 32 * 5 ? launch_pdl(weight_grad_kernel<W, 5>, grid, 1024, 0, 1, st, "rms_norm_grad (weight)", partial, parts, cols, dw)
                         : launch_pdl(weight_grad_kernel<W, 10>, grid, 1024, 0, 1, st, "rms_norm_grad (weight)", partial, parts, cols, dw);
}

template <typename T>
int launch_grad_any(const Backward& p, int parts, cudaStream_t st) {
  float* inv = p.partial ? p.partial + (int64_t)parts * p.cols : nullptr;
  const int rc = launch_pdl(rms_norm_grad_any_kernel<T>, dim3((unsigned)p.rows), 256, 0, 1, st, "rms_norm_grad", p, inv);
  if (rc || !p.partial) return rc;
  return launch_pdl(weight_grad_any_kernel<T>, dim3((unsigned)((p.cols + 255) / 256), (unsigned)parts), 256, 0, 1, st, "rms_norm_grad", p,
                    (const float*)inv);
}

template <typename T, int TPR, int CH, int STAGES, int THREADS>
int launch_grad_ring(const Backward& p, int parts, cudaStream_t st) {
  constexpr int smem = STAGES * 3 * CH * THREADS * 16;
  static_assert(smem + 1024 <= 227 * 1024, "the ring fits a multiprocessor");
  const int rc = allow_smem((const void*)rms_norm_grad_kernel<T, TPR, CH, STAGES, THREADS>, smem);
  if (rc) return rc;
  return launch_pdl(rms_norm_grad_kernel<T, TPR, CH, STAGES, THREADS>, dim3((unsigned)parts), THREADS, smem, 1, st, "rms_norm_grad", p);
}

template <typename T>
int launch_backward(const Backward& p, bool vector, int parts, cudaStream_t st) {
  if (vector) {
    const int pieces = p.cols / (16 / (int)sizeof(T));
    if (pieces <= 32 * 4) return launch_grad_ring<T, 32, 4, 2, 512>(p, parts, st);
    if (pieces <= 128 * 2) return launch_grad_ring<T, 128, 2, 2, 1024>(p, parts, st);
    if (pieces <= 256 * 2) return launch_grad_ring<T, 256, 2, 2, 1024>(p, parts, st);
    if (pieces <= 512 * 2) return launch_grad_ring<T, 512, 2, 2, 1024>(p, parts, st);
    if (pieces <= 1024 * 2) return launch_grad_ring<T, 1024, 2, 2, 1024>(p, parts, st);
    if (pieces <= 1024 * 4) return launch_grad_ring<T, 1024, 4, 1, 1024>(p, parts, st);  // one row fills the ring
    return launch_grad_any<T>(p, parts, st);
  }
#define MOE_RG(TPR, CH) \
  launch_pdl(rms_norm_grad_single_kernel<T, TPR, CH>, dim3((unsigned)parts), TPR > 128 ? TPR : 128, 0, 1, st, "rms_norm_grad", p)
  if (p.cols <= 32 * 4) return MOE_RG(32, 4);
  if (p.cols <= 64 * 4) return MOE_RG(64, 4);
  if (p.cols <= 128 * 4) return MOE_RG(128, 4);
  if (p.cols <= 256 * 4) return MOE_RG(256, 4);
  if (p.cols <= 512 * 4) return MOE_RG(512, 4);
  return launch_grad_any<T>(p, parts, st);
#undef MOE_RG
}

}  // namespace
}  // namespace moe

extern "C" int moe_rms_norm(const void* x, int64_t x_ld, const void* residual, int64_t residual_ld, const void* weight, int dtype,
                            int weight_dtype, int64_t rows, int64_t cols, float eps, void* y, int64_t y_ld, void* residual_out,
                            int64_t residual_out_ld, void* stream) {
  using namespace moe;
  const int rc = check_forward("rms_norm", x, dtype, weight_dtype, residual, weight, rows, cols, eps, x_ld, residual_ld, residual_out,
                               residual_out_ld);
  if (rc || rows == 0) return rc;
  if (!y || (y_ld < cols && rows > 1)) return fail(MOE_E_BADARG, "rms_norm: bad output");
  if (!residual && y == x) return fail(MOE_E_BADARG, "rms_norm: the output may lie over the input only with a residual");
  const bool shifted = (y == x && y_ld != x_ld) || (residual && residual_out == residual && residual_out_ld != residual_ld);
  if (residual && (y == residual_out || (shifted && rows > 1)))
    return fail(MOE_E_BADARG, "rms_norm: outputs over the inputs have their row distance, and lie apart");
  Forward p = {};
  p.x = x; p.residual = residual; p.weight = weight; p.y = y; p.h = residual ? residual_out : nullptr;
  p.x_ld = x_ld; p.residual_ld = residual_ld; p.y_ld = y_ld; p.h_ld = residual_out_ld; p.rows = rows;
  p.cols = (int)cols; p.w_f32 = weight_dtype == MOE_F32; p.eps = eps; p.mean = 1.0f / (float)cols; p.group = (int)cols; p.groups = 1;
  return forward(p, dtype, (cudaStream_t)stream);
}

extern "C" int moe_rms_norm_quant(const void* x, int64_t x_ld, const void* residual, int64_t residual_ld, const void* weight, int dtype,
                                  int weight_dtype, int64_t rows, int64_t cols, float eps, int format, int group, float quant_eps,
                                  int scale_flags, void* q, float* scales, int64_t scale_ld, void* y, void* residual_out, void* stream) {
  using namespace moe;
  const int rc = check_forward("rms_norm_quant", x, dtype, weight_dtype, residual, weight, rows, cols, eps, x_ld, residual_ld,
                               residual_out, cols);
  if (rc) return rc;
  if (format < kE4M3 || format > kInt8) return fail(MOE_E_DTYPE, "rms_norm_quant: unknown 8-bit format %d", format);
  if (group <= 0 || cols % group != 0) return fail(MOE_E_SHAPE, "rms_norm_quant: the row must be a multiple of the group size %d", group);
  if (!(quant_eps >= 0.0f) || !(quant_eps < 3.0e38f)) return fail(MOE_E_BADARG, "rms_norm_quant: quant_eps must be finite and not negative");
  if ((scale_flags & 2) && format == kInt8) return fail(MOE_E_BADARG, "rms_norm_quant: power-of-two scales are for the 8-bit floats");
  if (rows == 0) return 0;
  if (!q || !scales || ((scale_flags & 1) && scale_ld < rows)) return fail(MOE_E_BADARG, "rms_norm_quant: bad output");
  if (y && (y == x || y == residual || y == residual_out)) return fail(MOE_E_BADARG, "rms_norm_quant: the norm is written to memory of its own");
  if (residual && residual_out == residual && residual_ld != cols && rows > 1)
    return fail(MOE_E_BADARG, "rms_norm_quant: a stream over the residual has its row distance");
  Forward p = {};
  p.x = x; p.residual = residual; p.weight = weight; p.y = y; p.h = residual ? residual_out : nullptr;
  p.x_ld = x_ld; p.residual_ld = residual_ld; p.y_ld = cols; p.h_ld = cols; p.rows = rows;
  p.cols = (int)cols; p.w_f32 = weight_dtype == MOE_F32; p.eps = eps; p.mean = 1.0f / (float)cols;
  p.q = (uint8_t*)q; p.scales = scales; p.scale_ld = scale_ld; p.group = group; p.groups = (int)(cols / group); p.format = format;
  p.transposed = scale_flags & 1; p.ue8m0 = (scale_flags >> 1) & 1; p.quant_eps = quant_eps;
  return forward(p, dtype, (cudaStream_t)stream);
}

extern "C" int moe_rms_norm_grad_workspace(int64_t rows, int64_t cols, int64_t* bytes) {
  using namespace moe;
  if (rows < 0 || cols <= 0 || cols > (1 << 24) || !bytes) return fail(MOE_E_BADARG, "rms_norm_grad: bad extent");
  if (rows > kMaxRows) return fail(MOE_E_TOOBIG, "rms_norm_grad: too many rows");
  *bytes = 4 * ((int64_t)grad_blocks(rows, cols, false) * cols + rows);
  return 0;
}

extern "C" int moe_rms_norm_grad(const void* dy, const void* dresidual_out, const void* h, int64_t h_ld, const void* weight, int dtype,
                                 int weight_dtype, int64_t rows, int64_t cols, float eps, void* dx, void* dweight, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  using namespace moe;
  int rc = check_forward("rms_norm_grad", h, dtype, weight_dtype, nullptr, weight, rows, cols, eps, h_ld, 0, nullptr, 0);
  if (rc) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  if (rows == 0) {
    if (!dweight) return 0;
    const cudaError_t ce = cudaMemsetAsync(dweight, 0, (size_t)cols * (weight_dtype == MOE_F32 ? 4 : 2), st);
    return ce == cudaSuccess ? 0 : fail((int)ce, "rms_norm_grad: %s", cudaGetErrorString(ce));
  }
  if (!dy || (!dx && !dweight)) return fail(MOE_E_BADARG, "rms_norm_grad: null pointer");
  if (dx && (dx == dy || dx == h || dx == dresidual_out))  // long rows are read again for dweight when dx is written
    return fail(MOE_E_BADARG, "rms_norm_grad: dx lies apart from what it is made of");
  if (dweight && (!workspace || workspace_bytes < 4 * ((int64_t)grad_blocks(rows, cols, false) * cols + rows) || !aligned16(workspace)))
    return fail(MOE_E_BADARG, "rms_norm_grad: workspace too small");
  Backward p = {};
  p.dy = dy; p.dh = dresidual_out; p.h = h; p.weight = weight; p.dx = dx; p.partial = dweight ? (float*)workspace : nullptr;
  p.h_ld = h_ld; p.rows = rows; p.cols = (int)cols; p.w_f32 = weight_dtype == MOE_F32; p.eps = eps; p.mean = 1.0f / (float)cols;
  const int size = dtype == MOE_F32 ? 4 : 2;
  const bool vector = cols % (16 / size) == 0 && pieces16(h, h_ld, size) && aligned16(dy) && aligned16(dresidual_out) && aligned16(dx) &&
                      aligned16(weight);
  const int parts = grad_blocks(rows, cols, vector);
  rc = dtype == MOE_F32 ? launch_backward<float>(p, vector, parts, st)
       : dtype == MOE_F16 ? launch_backward<__half>(p, vector, parts, st)
                          : launch_backward<__nv_bfloat16>(p, vector, parts, st);
  if (rc || !dweight) return rc;
  const float* partial = (const float*)workspace;
  return weight_dtype == MOE_F32   ? sum_parts(partial, parts, (int)cols, (float*)dweight, st)
         : weight_dtype == MOE_F16 ? sum_parts(partial, parts, (int)cols, (__half*)dweight, st)
                                   : sum_parts(partial, parts, (int)cols, (__nv_bfloat16*)dweight, st);
}
