// Scalar pieces shared by the dense layer's kernels: types, activations and their derivatives, the epilogue.
#pragma once
#include "dense_internal.h"

namespace petdense_k {

// hipLaunchKernel itself: the launch syntax pushes and pops a configuration first, which a small call would notice
template <typename A>
struct Same {
  typedef A type;
};
template <typename... A>
inline hipError_t launch_kernel(void (*k)(A...), dim3 grid, dim3 block, size_t lds, hipStream_t s,
                                typename Same<A>::type... a) {
  void* args[] = {static_cast<void*>(&a)...};
  return hipLaunchKernel(reinterpret_cast<const void*>(k), grid, block, args, lds, s);
}

typedef float f32x4 __attribute__((ext_vector_type(4)));

// Neighbouring workgroup numbers go to different XCDs, each with its own L2: XCD x takes a contiguous run of the n
// pieces of work, [first, first + len).
__device__ __forceinline__ void run_of(int n, int x, int& first, int& len) {
  const int per = n / 8, rest = n % 8;
  first = x * per + min(x, rest);
  len = per + (x < rest ? 1 : 0);
}

// Phi(x) = erfc(-x / sqrt 2) / 2: right relative to itself in the lower tail too, where 1 + erf would cancel (5 % off
// at x = -4.9).
// 16-bit outputs: Phi(-a) = e^(-a^2/2) t P(t) with t = 1 / (1 + 0.35 a), a = |x|, and Phi(a) = 1 - Phi(-a).  P of
// degree 6 has the least largest error beside min(1e-7, 1e-5 Phi) over a <= 14 (a linear program over
// Phi(-a) e^(a^2/2)): 4e-8 absolute and 4e-6 relative, 2.1e-7 and 2^-16 with its fp32 steps (the exponent's roundings
// are a^2 2^-24 of the value), beside the 2^-9 and 2^-12 of an output that is rounded to 16 bits.  A third of the
// instructions that erfcf takes (17 of 51), and the epilogue pays them once per output.  The gradient needs the
// exponential as well (`e`).
__device__ __forceinline__ float normal_cdf_fast(float x, float& e) {
  const float t = __builtin_amdgcn_rcpf(fmaf(0.35f, fabsf(x), 1.0f));
  e = __builtin_amdgcn_exp2f(x * x * -0.72134752f);
  float p = fmaf(0.0446154723f, t, -0.184429168f);
  p = fmaf(p, t, 0.211082418f);
  p = fmaf(p, t, 0.0089271389f);
  p = fmaf(p, t, 0.143156413f);
  p = fmaf(p, t, 0.136871306f);
  p = fmaf(p, t, 0.139776456f);
  const float q = p * t * e;
  return x < 0.f ? q : 1.0f - q;
}

template <bool EXACT>
__device__ __forceinline__ float normal_cdf(float x) {
  if constexpr (EXACT) {
    return 0.5f * erfcf(x * -0.70710678118654752f);
  } else {
    float e;
    return normal_cdf_fast(x, e);
  }
}

template <bool EXACT>
__device__ __forceinline__ float sigmoid(float x) {
  if constexpr (EXACT) return 1.0f / (1.0f + expf(-x));
  return __builtin_amdgcn_rcpf(1.0f + __expf(-x));
}

template <bool EXACT>
__device__ __forceinline__ float activate(float v, int act) {
  if (act == kRelu) return v < 0.f ? 0.f : v;               // a NaN stays
  if (act == kGelu) return v * normal_cdf<EXACT>(v);
  if (act == kSilu) return v * sigmoid<EXACT>(v);
  return v;
}

// act'(v); for ReLU v may be the output as well as the pre-activation
template <bool EXACT>
__device__ __forceinline__ float activate_grad(float g, float v, int act) {
  if (act == kRelu) return v <= 0.f ? 0.f : g;
  if (act == kGelu) {
    float cdf, e;
    if constexpr (EXACT) {
      cdf = normal_cdf<true>(v);
      e = expf(-0.5f * v * v);
    } else {
      cdf = normal_cdf_fast(v, e);
    }
    return g * fmaf(v, 0.39894228040143268f * e, cdf);
  }
  if (act == kSilu) {
    const float s = sigmoid<EXACT>(v);
    return g * s * fmaf(v, 1.0f - s, 1.0f);
  }
  return g;
}

// W neighbouring values of a row, of which n exist (the others read as zero).  Whole groups are one access of any
// alignment.
template <typename T, int W>
__device__ __forceinline__ void load_row(const T* src, int n, float* v) {
  if (n >= W) {
    T w[W];
    __builtin_memcpy(w, src, sizeof(w));
#pragma unroll
    for (int q = 0; q < W; ++q) v[q] = (float)w[q];
  } else {
#pragma unroll
    for (int q = 0; q < W; ++q) v[q] = q < n ? (float)src[q] : 0.f;
  }
}
template <typename T, int W>
__device__ __forceinline__ void store_row(T* dst, int n, const float* v) {
  if (n >= W) {
    T w[W];
#pragma unroll
    for (int q = 0; q < W; ++q) w[q] = (T)v[q];
    __builtin_memcpy(dst, w, sizeof(w));
  } else {
#pragma unroll
    for (int q = 0; q < W; ++q)
      if (q < n) dst[q] = (T)v[q];
  }
}

// The bias of columns j .. j + 7, of which `n` exist.
template <typename T>
__device__ __forceinline__ void bias8(const Epilogue& e, int64_t j, int n, float* w) {
  if (e.bias_f32) load_row<float, 8>(static_cast<const float*>(e.bias) + j, n, w);
  else load_row<T, 8>(static_cast<const T*>(e.bias) + j, n, w);
}

// Eight outputs (i, j .. j + 7) of which `n` exist; `bias`: theirs, read already, or null.
template <typename T>
__device__ __forceinline__ void epilogue8(const Epilogue& e, int64_t i, int64_t j, int n, float* v,
                                          const float* bias = nullptr) {
  constexpr bool EXACT = sizeof(T) == 4;
  float w[8];
  if (e.bias) {
    if (!bias) bias8<T>(e, j, n, w);
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] += bias ? bias[q] : w[q];
  }
  if (e.res) {
    load_row<T, 8>(static_cast<const T*>(e.res) + i * e.ldr + j, n, w);
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] += w[q];
  }
  if (e.pre) {
    if (e.out_f32) store_row<float, 8>(static_cast<float*>(e.pre) + i * e.ldp + j, n, v);
    else store_row<T, 8>(static_cast<T*>(e.pre) + i * e.ldp + j, n, v);
  }
  if (e.act == kRelu) {
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = activate<EXACT>(v[q], kRelu);
  } else if (e.act == kGelu) {
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = activate<EXACT>(v[q], kGelu);
  } else if (e.act == kSilu) {
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = activate<EXACT>(v[q], kSilu);
  }
  if (e.out_f32) store_row<float, 8>(static_cast<float*>(e.out) + i * e.ldo + j, n, v);
  else store_row<T, 8>(static_cast<T*>(e.out) + i * e.ldo + j, n, v);
}

// g[q] = g[q] act'(v[q]) for W values, one uniform branch
template <bool EXACT, int W>
__device__ __forceinline__ void activate_grads(float* g, const float* v, int act) {
  if (act == kRelu) {
#pragma unroll
    for (int q = 0; q < W; ++q) g[q] = activate_grad<EXACT>(g[q], v[q], kRelu);
  } else if (act == kGelu) {
#pragma unroll
    for (int q = 0; q < W; ++q) g[q] = activate_grad<EXACT>(g[q], v[q], kGelu);
  } else if (act == kSilu) {
#pragma unroll
    for (int q = 0; q < W; ++q) g[q] = activate_grad<EXACT>(g[q], v[q], kSilu);
  }
}

// Sums 8 columns of dy act'(saved) over all rows: a thread takes every THREADS-th row; the rows meet by shuffles, the
// waves in LDS, in a fixed order.
template <typename T, int THREADS>
__device__ __forceinline__ void sum_columns8(const ColumnSum& p, int block, int t, float* red) {
  constexpr int W = 8, AHEAD = 4;
  const int j = block * W, n = p.N - j;
  const T* dy = static_cast<const T*>(p.dy) + j;
  const T* sv = static_cast<const T*>(p.saved) + j;
  float sum[W];
#pragma unroll
  for (int q = 0; q < W; ++q) sum[q] = 0.f;
  int64_t m = t;
  if (n >= W) {
    for (; m + (AHEAD - 1) * THREADS < p.M; m += AHEAD * THREADS) {
      float g[AHEAD][W], v[AHEAD][W];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        load_row<T, W>(dy + (m + u * THREADS) * p.ldy, W, g[u]);
        if (p.act != kNone) load_row<T, W>(sv + (m + u * THREADS) * p.lds, W, v[u]);
      }
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        activate_grads<sizeof(T) == 4, W>(g[u], v[u], p.act);
#pragma unroll
        for (int q = 0; q < W; ++q) sum[q] += g[u][q];
      }
    }
  }
  for (; m < p.M; m += THREADS) {
    float g[W], v[W];
    load_row<T, W>(dy + m * p.ldy, n, g);
    if (p.act != kNone) load_row<T, W>(sv + m * p.lds, n, v);
    activate_grads<sizeof(T) == 4, W>(g, v, p.act);
#pragma unroll
    for (int q = 0; q < W; ++q) sum[q] += g[q];
  }
#pragma unroll
  for (int q = 0; q < W; ++q) {
#pragma unroll
    for (int o = 1; o < 64; o *= 2) sum[q] += __shfl_xor(sum[q], o);
    if ((t & 63) == 0) red[(t >> 6) * W + q] = sum[q];
  }
  __syncthreads();
  if (t < W && t < n) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) s += red[w * W + t];
    if (p.out_type == kF32) static_cast<float*>(p.out)[j + t] = s;
    else if (p.out_type == kBF16) static_cast<__bf16*>(p.out)[j + t] = (__bf16)s;
    else static_cast<_Float16*>(p.out)[j + t] = (_Float16)s;
  }
}

// Sums 16 columns of a column join: thread t < 256 takes column t % 16 of the chunks t / 16, t / 16 + 16, .., sixteen
// loads at a time (past the last: its value again, not added); the 16 groups meet in LDS, in order.  Every thread of
// the workgroup comes here.
__device__ __forceinline__ void join_columns16(const ColumnJoin& p, int block, int t, float* red) {
  constexpr int AHEAD = 16;
  const int c = t & 15, g = t >> 4, j = block * 16 + c;
  float v = 0.f;
  if (t < 256 && j < p.N) {
    for (int k = g; k < p.chunks; k += 16 * AHEAD) {
      float w[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) w[u] = p.part[(int64_t)min(k + 16 * u, p.chunks - 1) * p.N + j];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) v += k + 16 * u < p.chunks ? w[u] : 0.f;
    }
  }
  if (t < 256) red[t] = v;
  __syncthreads();
  if (g == 0 && j < p.N) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) s += red[k * 16 + c];
    if (p.out_type == kF32) static_cast<float*>(p.out)[j] = s;
    else if (p.out_type == kBF16) static_cast<__bf16*>(p.out)[j] = (__bf16)s;
    else static_cast<_Float16*>(p.out)[j] = (_Float16)s;
  }
}

// e4m3 codes of a word's four bytes times 2^E (`scale`) as two packed words of T; exact for the blocks the checkpoint
// writes (four significant bits, E >= -117, no value past T's largest), except that fp16 rounds what is below 2^-14.
template <typename T>
__device__ __forceinline__ void restore4(unsigned w, float scale, T* out) {
  if constexpr (sizeof(T) == 4) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    const f2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, scale, false);
    const f2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, scale, true);
    out[0] = a[0]; out[1] = a[1]; out[2] = b[0]; out[3] = b[1];
  } else if constexpr (__is_same(T, __bf16)) {
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false);
    const auto b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true);
    out[0] = a[0]; out[1] = a[1]; out[2] = b[0]; out[3] = b[1];
  } else {
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, false);
    const auto b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, true);
    out[0] = a[0]; out[1] = a[1]; out[2] = b[0]; out[3] = b[1];
  }
}

// 2^(byte - 127): an exponent byte as a float's exponent field (the checkpoint writes 10 .. 247)
__device__ __forceinline__ float exponent_scale(unsigned byte) { return __uint_as_float(byte << 23); }

}  // namespace petdense_k
