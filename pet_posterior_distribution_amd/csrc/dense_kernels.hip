// The dense layer's kernels around its tiled product: the join of split products, few-row products, the activation's
// gradient with the bias gradient's column sums, and the 8-bit activation checkpoint.
#include "dense_epilogue.h"

#include <algorithm>
#include <type_traits>

namespace petdense_k {

namespace {

constexpr int64_t kSlab = (int64_t)1 << 29;     // threads of one launch (a grid holds fewer than 2^32)

inline unsigned blocks_for(int64_t n, int per) { return (unsigned)((n + per - 1) / per); }

// ---------------------------------------------------------------------------------------------------------------
// join: out = epilogue(sum over splits).  Bound by reading the parts.  A thread takes eight columns and every G-th
// split; the G sums meet in LDS, in order.  G = 8 where outputs are few and splits many: one thread after another
// would wait for memory split by split (63 x 31 outputs of 64 splits: 15.6 us with G = 1).  The first workgroups
// join a bias gradient's column sums, which saves it a launch (they take longest: last, they would end last).
// 1536 x 128 outputs of 10 parts and 128 columns of 1024 chunks: 5.2 us; 48 tiles of 256 x 256 of 5 parts and 512
// columns: 15.8 us, 79 MB.
// ---------------------------------------------------------------------------------------------------------------
template <typename T, int G>
__global__ __launch_bounds__(256) void join_kernel(Product p, ColumnJoin cols, int64_t octets, int orow, int first) {
  constexpr int PER = 256 / G;
  __shared__ f32x4 red[G > 1 ? G : 1][PER][2];
  if ((int)blockIdx.x < first) return join_columns16(cols, blockIdx.x, threadIdx.x, reinterpret_cast<float*>(red));
  const int q8 = threadIdx.x % PER, g = threadIdx.x / PER;
  const int64_t t = (int64_t)(blockIdx.x - first) * PER + q8;
  const bool live = t < octets;
  const int64_t i = live ? t / orow : 0;
  const int j = live ? (int)(t - i * orow) * 8 : 0, n = p.J - j;
  const float* src = p.part + i * p.J + j;
  const int64_t plane = (int64_t)p.I * p.J;
  float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (live) {
#pragma unroll 8
    for (int s = g; s < p.splits; s += G) {
      float w[8];
      load_row<float, 8>(src + s * plane, n, w);
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] += w[q];
    }
  }
  if constexpr (G > 1) {
    red[g][q8][0] = f32x4{v[0], v[1], v[2], v[3]};
    red[g][q8][1] = f32x4{v[4], v[5], v[6], v[7]};
    __syncthreads();
    if (g != 0 || !live) return;
    f32x4 lo = red[0][q8][0], hi = red[0][q8][1];
#pragma unroll
    for (int k = 1; k < G; ++k) {
      lo += red[k][q8][0];
      hi += red[k][q8][1];
    }
    for (int q = 0; q < 4; ++q) v[q] = lo[q], v[4 + q] = hi[q];
  } else if (!live) {
    return;
  }
  epilogue8<T>(p.e, i, j, n, v);
}

template <typename T>
__global__ __launch_bounds__(256) void join_tiles_kernel(Product p, ColumnJoin cols, int b, int ti, int tj, int first) {
  __shared__ float red[256];
  if ((int)blockIdx.y < first) {
    const int k = blockIdx.y * gridDim.x + blockIdx.x;
    if (k * 16 < cols.N) join_columns16(cols, k, threadIdx.x, red);
    return;
  }
  // split tile y; a thread takes eight columns of one of its rows
  const int per = b / 8, t = blockIdx.x * 256 + threadIdx.x, r = t / per, c = (t % per) * 8, y = blockIdx.y - first;
  int a, d;
  tile_at(p.whole + y, ti, tj, a, d);
  const int64_t i = (int64_t)a * b + r;
  const int j = d * b + c, n = p.J - j;
  if (r >= b || i >= p.I || n <= 0) return;
  const float* src = p.part + (int64_t)y * p.splits * b * b + r * b + c;
  float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) {
    float w[8];
    load_row<float, 8>(src + (int64_t)s * b * b, 8, w);
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] += w[q];
  }
  epilogue8<T>(p.e, i, j, n, v);
}

// ---------------------------------------------------------------------------------------------------------------
// One or two rows (decoding, a single sample): every value of B is read once by one workgroup, which owns 32 columns
// and, where those are enough workgroups, the whole contraction, so that one launch ends the call.  Bound by latency:
// 4 lanes share a row's 8-column pieces, 256 rows of B are in flight four deep, and the sums meet by two rotations of
// 16 lanes and once in LDS, in a fixed order.  Neighbouring columns go to one XCD, whose L2 has the other half of their
// cache lines: 1 x 8192 x 8192 bf16 in 27.6 us, 4.9 TB/s of weights (42 us with them spread).  1 x 1024 x 4096 in
// 4.4 us, where a launch alone takes 3 us.  From three rows on the sliced tiles are quicker (3 x 3608 x 4882 fp16 took
// 29 us here).
// ---------------------------------------------------------------------------------------------------------------
// v summed over the four lanes l, l + 4, l + 8, l + 12 of a row of 16, in each of them (two rotations of the row: no
// LDS, which ROWS x 8 shuffles of 16 waves would keep busy for microseconds)
__device__ __forceinline__ float sum_row4(float v) {
  const int a = __builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + 8, 0xf, 0xf, false);     // row_ror:8
  v += __int_as_float(a);
  const int b = __builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + 4, 0xf, 0xf, false);     // row_ror:4
  return v + __int_as_float(b);
}

// W neighbouring values as one access of any alignment
template <typename T, int W>
struct Octet {
  typedef T type __attribute__((ext_vector_type(W)));
  typedef type any __attribute__((aligned(sizeof(T)), may_alias));
};

// W neighbouring values of a row, all there or 0 < n < W of them.  The cut piece reads its last value again rather than
// branch, so that its loads go out together.
template <typename T, int W, bool WHOLE>
__device__ __forceinline__ void load_piece(const T* __restrict__ src, int n, T* w) {
  if constexpr (WHOLE) {
    const typename Octet<T, W>::type v = *reinterpret_cast<const typename Octet<T, W>::any*>(src);
#pragma unroll
    for (int q = 0; q < W; ++q) w[q] = v[q];
  } else {
#pragma unroll
    for (int q = 0; q < W; ++q) w[q] = src[q < n ? q : n - 1];
  }
}

template <typename T, int ROWS>
__global__ __launch_bounds__(kRowThreads) void rows_kernel(Product p) {
  constexpr int W = 8, LANES = kRowCols / W, GROUPS = kRowThreads / LANES;   // 4 lanes a row, 256 rows at a time
  constexpr int AHEAD = 4;                                                  // rows of a lane in flight
  constexpr int PARTS = kRowThreads / 16;                                   // sums of 16 lanes that meet in LDS
  __shared__ float red[PARTS][ROWS][kRowCols];
  __shared__ float sum[ROWS][kRowCols];
  const int tid = threadIdx.x, l = tid % LANES, grp = tid / LANES;
  const int groups = (p.J + kRowCols - 1) / kRowCols;
  int first, len;
  run_of(groups * p.splits, blockIdx.x % 8, first, len);
  const int piece = first + blockIdx.x / 8, split = piece / groups, j0 = (piece - split * groups) * kRowCols;
  const int j = j0 + l * W, n = p.J - j;
  const T* A = static_cast<const T*>(p.A);
  const T* B = static_cast<const T*>(p.B) + j;
  float acc[ROWS][W];
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
#pragma unroll
    for (int q = 0; q < W; ++q) acc[r][q] = 0.f;
  const int end = min(p.C, (split + 1) * p.c_per);      // this part of the contraction
  auto walk = [&](auto whole) {
    auto add = [&](const T* w, const T* x) {
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int q = 0; q < W; ++q) acc[r][q] = fmaf((float)x[r], (float)w[q], acc[r][q]);
    };
    auto fetch = [&](int c, T* w, T* x) {
      load_piece<T, W, decltype(whole)::value>(B + (int64_t)c * p.ldb, n, w);
#pragma unroll
      for (int r = 0; r < ROWS; ++r) x[r] = A[r * p.lda + c];
    };
    int c = split * p.c_per + grp;
    for (; c + (AHEAD - 1) * GROUPS < end; c += AHEAD * GROUPS) {
      T w[AHEAD][W], x[AHEAD][ROWS];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) fetch(c + u * GROUPS, w[u], x[u]);
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) add(w[u], x[u]);
    }
    for (; c < end; c += GROUPS) {
      T w[W], x[ROWS];
      fetch(c, w, x);
      add(w, x);
    }
  };
  if (n >= W) walk(std::true_type{});
  else if (n > 0) walk(std::false_type{});        // past n: sums that nothing stores
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
#pragma unroll
    for (int q = 0; q < W; ++q) {
      const float v = sum_row4(acc[r][q]);
      if ((tid & 15) < LANES) red[tid >> 4][r][l * W + q] = v;
    }
  __syncthreads();
  if (tid < ROWS * kRowCols) {
    const int r = tid / kRowCols, q = tid % kRowCols;
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < PARTS; ++k) v += red[k][r][q];
    sum[r][q] = v;
  }
  __syncthreads();
  // thread t: row t / 4, columns 8 (t % 4) ..
  if (tid < ROWS * LANES && j < p.J) {
    const int r = tid / LANES;
    float v[W];
#pragma unroll
    for (int q = 0; q < W; ++q) v[q] = sum[r][l * W + q];
    if (p.splits > 1) store_row<float, W>(p.part + ((int64_t)split * p.I + r) * p.J + j, n, v);
    else epilogue8<T>(p.e, r, j, n, v);
  }
}

template <typename T>
hipError_t rows_t(const Product& p, hipStream_t s) {
  const dim3 grid(blocks_for(p.J, kRowCols) * p.splits), block(kRowThreads);
  if (p.I == 1) return launch_kernel(rows_kernel<T, 1>, grid, block, 0, s, p);
  return launch_kernel(rows_kernel<T, 2>, grid, block, 0, s, p);
}

// ---------------------------------------------------------------------------------------------------------------
// dp = dy act'(saved), and column sums of the unrounded dp over a chunk of rows.  One pass, memory bound: a lane takes
// 8 columns, lpr lanes a row (a power of two, so that narrow layers fill the wave with rows) and two rows at a time,
// whose loads go out together; the wave's rows meet by shuffles, the block's waves in LDS, in a fixed order.
// 8192 x 4096 bf16 with GELU in 46.6 us, 4.3 TB/s; 8323 x 7910 (rows on 4 bytes) with ReLU 86 us, 4.6 TB/s.  (Four rows
// together: the same for large layers, 2 us more for small ones, whose code comes cold.)
// ---------------------------------------------------------------------------------------------------------------
template <typename T, int ACT>
__global__ __launch_bounds__(256) void act_grad_kernel(const T* dy, int64_t ldy, const T* saved, int64_t lds, T* dp,
                                                       int64_t ldd, int bare, float* part, int rows_per, int M, int N,
                                                       int lpr) {
  constexpr bool EXACT = sizeof(T) == 4;
  constexpr int W = 8, AHEAD = 2;
  __shared__ float red[4][64 * W];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int l = lane & (lpr - 1), rows = 256 / lpr;             // rows the block takes at a time
  const int j = (blockIdx.x * lpr + l) * W, n = N - j;
  const int64_t m0 = (int64_t)blockIdx.y * rows_per, m1 = min(m0 + rows_per, (int64_t)M);
  float sum[W];
#pragma unroll
  for (int q = 0; q < W; ++q) sum[q] = 0.f;
  auto walk = [&](auto whole) {
    constexpr bool WHOLE = decltype(whole)::value;
    for (int64_t m = m0 + threadIdx.x / lpr; m < m1; m += AHEAD * rows) {
      T dyv[AHEAD][W], sv[AHEAD][W];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int64_t r = min(m + u * rows, m1 - 1);            // past the chunk: its last row again, and not used
        load_piece<T, W, WHOLE>(dy + r * ldy + j, n, dyv[u]);
        if constexpr (ACT != kNone) load_piece<T, W, WHOLE>(saved + r * lds + j, n, sv[u]);
      }
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        if (m + u * rows >= m1) break;
        float g[W], v[W];
#pragma unroll
        for (int q = 0; q < W; ++q) {
          const bool there = WHOLE || q < n;
          g[q] = there ? (float)dyv[u][q] : 0.f;
          v[q] = there && ACT != kNone ? (float)sv[u][q] : 0.f;
        }
        activate_grads<EXACT, W>(g, v, ACT);
#pragma unroll
        for (int q = 0; q < W; ++q) sum[q] += g[q];
        // (columns past the last are zero: the next product may read them)
        if (dp) store_row<T, W>(dp + (m + u * rows) * ldd + j, bare ? n : W, g);
      }
    }
  };
  if (n >= W) walk(std::true_type{});
  else if (n > 0) walk(std::false_type{});
  if (!part) return;
#pragma unroll
  for (int q = 0; q < W; ++q)
    for (int o = lpr; o < 64; o *= 2) sum[q] += __shfl_xor(sum[q], o);
  if (lane < lpr) {
#pragma unroll
    for (int q = 0; q < W; ++q) red[wave][lane * W + q] = sum[q];
  }
  __syncthreads();
  for (int c = threadIdx.x; c < lpr * W; c += 256) {
    const int k = blockIdx.x * lpr * W + c;
    if (k < N) part[(int64_t)blockIdx.y * N + k] = ((red[0][c] + red[1][c]) + red[2][c]) + red[3][c];
  }
}

template <typename T, int ACT>
hipError_t act_grad_a(const T* dy, int64_t ldy, const T* saved, int64_t lds, T* dp, int64_t ldd, int bare, float* part,
                      int chunks, int M, int N, hipStream_t s) {
  const int rows_per = (M + chunks - 1) / chunks, lpr = act_grad_lanes(N);
  return launch_kernel(act_grad_kernel<T, ACT>, dim3(blocks_for(N, lpr * 8), chunks), dim3(256), 0, s, dy, ldy, saved,
                       lds, dp, ldd, bare, part, rows_per, M, N, lpr);
}

template <typename T>
hipError_t act_grad_t(const void* dy, int64_t ldy, const void* saved, int64_t lds, void* dp, int64_t ldd, int bare,
                      float* part, int chunks, int M, int N, int act, hipStream_t s) {
  auto* f = act == kRelu   ? act_grad_a<T, kRelu>
            : act == kGelu ? act_grad_a<T, kGelu>
            : act == kSilu ? act_grad_a<T, kSilu>
                           : act_grad_a<T, kNone>;
  return f(static_cast<const T*>(dy), ldy, static_cast<const T*>(saved), lds, static_cast<T*>(dp), ldd, bare, part,
           chunks, M, N, s);
}

__global__ __launch_bounds__(256) void join_columns_kernel(ColumnJoin p) {
  __shared__ float red[256];
  for (int64_t b = blockIdx.x; b * 16 < p.N; b += gridDim.x) {
    join_columns16(p, (int)b, threadIdx.x, red);
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Padded copies.  A thread moves 16 bytes; a row's last piece is filled up with zeros.  Memory bound: 2048 x 5717 and
// 5717 x 416 bf16 values in 9.4 us.
// ---------------------------------------------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void pad_kernel(PadJobs p) {
  constexpr int W = 16 / (int)sizeof(T);
  int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
#pragma unroll
  for (int q = 0; q < 3; ++q) {
    const PadJob& job = p.job[q];
    const int pieces = (int)(job.ldd / W);
    const int64_t all = (int64_t)job.rows * pieces;
    if (t < all) {
      const int64_t r = t / pieces;
      const int c = (int)(t - r * pieces) * W, n = job.n - c;
      const T* src = static_cast<const T*>(job.src) + r * job.ld + c;
      T v[W];
      if (n >= W) {
        __builtin_memcpy(v, src, 16);
      } else {
#pragma unroll
        for (int x = 0; x < W; ++x) v[x] = x < n ? src[x] : (T)0.f;
      }
      __builtin_memcpy(__builtin_assume_aligned(static_cast<T*>(job.dst) + r * job.ldd + c, 16), v, 16);
      return;
    }
    t -= all;
    if (t < 0) return;
  }
}

// ---------------------------------------------------------------------------------------------------------------
// 8-bit checkpoint.  A lane takes 8 neighbouring values, 4 lanes a block of 32; the block's largest finite magnitude
// meets over the 4 lanes by two shuffles.  Memory bound both ways: 65536 x 4096 bf16 there and back in 331 us, 1.63 GB,
// 4.9 TB/s (a copy: 5.1 TB/s).
// ---------------------------------------------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void quantize_kernel(const T* x, int64_t ldx, int64_t octets, int orow, int K,
                                                       uint8_t* codes, int64_t ldc, uint8_t* exps, int64_t lde) {
  // orow: octets of a row, rounded up to whole blocks (a multiple of 4), so the 4 lanes of a block stay together
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t m = t / orow;
  const int k = (int)(t - m * orow) * 8;
  const bool live = t < octets;
  const int n = live ? K - k : 0;                       // may be <= 0 in a row's last block
  float v[8];
  load_row<T, 8>(live ? x + m * ldx + k : x, n, v);
  float top = 0.f;
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    const float a = fabsf(v[q]);
    top = fmaxf(top, a < __builtin_inff() ? a : 0.f);   // NaN and infinities do not count
  }
  top = fmaxf(top, __shfl_xor(top, 1));
  top = fmaxf(top, __shfl_xor(top, 2));
  // least E with top <= 448 2^E (448 = 1.75 2^8): top = 1.f 2^p gives E = p - 8, one more past a fraction of 0.75.
  // A subnormal top has exponent field 0 and ends at the least E as it should.
  const unsigned b = __float_as_uint(top);
  int byte = (int)(b >> 23) - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  byte = max(byte, 127 - 117);
  const float inv = __uint_as_float((unsigned)(254 - byte) << 23);      // 2^-E, exact
  const float lim = byte == (sizeof(T) == 2 && __is_same(T, _Float16) ? 127 + 8 : 127 + 120) ? 240.f : 448.f;
  unsigned w[2] = {0, 0};
#pragma unroll
  for (int q = 0; q < 8; q += 2) {
    const float y0 = fminf(fmaxf(v[q] * inv, -lim), lim), y1 = fminf(fmaxf(v[q + 1] * inv, -lim), lim);
    const int c = __builtin_amdgcn_cvt_pk_fp8_f32(y0, y1, 0, false) & 0xffff;
    w[q >> 2] |= (unsigned)c << ((q & 2) * 8);
  }
#pragma unroll
  for (int q = 0; q < 8; ++q)
    if (!(fabsf(v[q]) < __builtin_inff())) w[q >> 2] |= 0x7fu << ((q & 3) * 8);   // no infinities: they become NaN
  if (n <= 0) return;
  uint8_t* dst = codes + m * ldc + k;
  if (n >= 8) {
    __builtin_memcpy(dst, w, 8);
  } else {
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (q < n) dst[q] = (uint8_t)(w[q >> 2] >> ((q & 3) * 8));
  }
  if ((k & 31) == 0) exps[m * lde + k / 32] = (uint8_t)byte;
}

template <typename T>
__global__ __launch_bounds__(256) void restore_kernel(const uint8_t* codes, int64_t ldc, const uint8_t* exps,
                                                      int64_t lde, int64_t octets, int orow, int K, T* x, int64_t ldx) {
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (t >= octets) return;
  const int64_t m = t / orow;
  const int k = (int)(t - m * orow) * 8, n = K - k;
  const uint8_t* src = codes + m * ldc + k;
  unsigned w[2] = {0, 0};
  if (n >= 8) {
    __builtin_memcpy(w, src, 8);
  } else {
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (q < n) w[q >> 2] |= (unsigned)src[q] << ((q & 3) * 8);
  }
  const float sc = exponent_scale(exps[m * lde + k / 32]);
  T v[8];
  restore4<T>(w[0], sc, v);
  restore4<T>(w[1], sc, v + 4);
  T* dst = x + m * ldx + k;
  if (n >= 8) {
    __builtin_memcpy(dst, v, sizeof(v));
  } else {
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (q < n) dst[q] = v[q];
  }
}

template <typename T>
hipError_t quantize_t(const void* x, int64_t ldx, int64_t M, int K, uint8_t* codes, int64_t ldc, uint8_t* exps,
                      int64_t lde, hipStream_t s) {
  const int orow = (K + 31) / 32 * 4;
  const int64_t slab = std::max<int64_t>(1, kSlab / orow);
  for (int64_t m = 0; m < M; m += slab) {
    const int64_t octets = std::min(slab, M - m) * orow;
    if (hipError_t e = launch_kernel(quantize_kernel<T>, dim3(blocks_for(octets, 256)), dim3(256), 0, s,
                                     static_cast<const T*>(x) + m * ldx, ldx, octets, orow, K, codes + m * ldc, ldc,
                                     exps + m * lde, lde))
      return e;
  }
  return hipSuccess;
}

template <typename T>
hipError_t restore_t(const uint8_t* codes, int64_t ldc, const uint8_t* exps, int64_t lde, int64_t M, int K, void* x,
                     int64_t ldx, hipStream_t s) {
  const int orow = (K + 7) / 8;
  const int64_t slab = std::max<int64_t>(1, kSlab / orow);
  for (int64_t m = 0; m < M; m += slab) {
    const int64_t octets = std::min(slab, M - m) * orow;
    if (hipError_t e = launch_kernel(restore_kernel<T>, dim3(blocks_for(octets, 256)), dim3(256), 0, s,
                                     codes + m * ldc, ldc, exps + m * lde, lde, octets, orow, K,
                                     static_cast<T*>(x) + m * ldx, ldx))
      return e;
  }
  return hipSuccess;
}

}  // namespace

#define PETDENSE_BY_TYPE(type, call)         \
  switch (type) {                            \
    case kF32: { using T = float; call; }    \
    case kBF16: { using T = __bf16; call; }  \
    default: { using T = _Float16; call; }   \
  }

template <typename T, int G>
hipError_t join_t(const Product& p, const ColumnJoin& cols, hipStream_t s) {
  const int orow = (p.J + 7) / 8;
  const int64_t octets = (int64_t)p.I * orow;
  const unsigned first = blocks_for(cols.N, 16);
  return launch_kernel(join_kernel<T, G>, dim3(first + blocks_for(octets, 256 / G)), dim3(256), 0, s, p, cols, octets,
                       orow, (int)first);
}

hipError_t join(const Product& p, const ColumnJoin& cols, int type, hipStream_t s) {
  if (p.splits > 2 && (int64_t)p.I * ((p.J + 7) / 8) < 65536)
    PETDENSE_BY_TYPE(type, return (join_t<T, 8>(p, cols, s)))
  PETDENSE_BY_TYPE(type, return (join_t<T, 1>(p, cols, s)))
}

hipError_t join_tiles(const Product& p, const ColumnJoin& cols, int type, int b, hipStream_t s) {
  const int ti = (p.I + b - 1) / b, tj = (p.J + b - 1) / b, tiles = ti * tj - p.whole;
  const unsigned row = blocks_for(b * (b / 8), 256), first = blocks_for(cols.N, 16 * row);
  PETDENSE_BY_TYPE(type, return launch_kernel(join_tiles_kernel<T>, dim3(row, first + tiles), dim3(256), 0, s, p, cols,
                                              b, ti, tj, (int)first))
}

hipError_t rows(const Product& p, int type, hipStream_t s) { PETDENSE_BY_TYPE(type, return rows_t<T>(p, s)) }

hipError_t act_grad(const void* dy, int64_t ldy, const void* saved, int64_t lds, void* dp, int64_t ldd, int bare,
                    float* part, int chunks, int M, int N, int type, int act, hipStream_t s) {
  PETDENSE_BY_TYPE(type, return act_grad_t<T>(dy, ldy, saved, lds, dp, ldd, bare, part, chunks, M, N, act, s))
}

template <typename T>
hipError_t pad_t(const PadJobs& p, hipStream_t s) {
  int64_t pieces = 0;
  for (const PadJob& j : p.job) pieces += (int64_t)j.rows * (j.ldd * (int64_t)sizeof(T) / 16);
  if (pieces >= (int64_t)1 << 32) return hipErrorInvalidValue;      // the plan copies nothing of that size
  return launch_kernel(pad_kernel<T>, dim3(blocks_for(pieces, 256)), dim3(256), 0, s, p);
}

hipError_t pad(const PadJobs& p, int type, hipStream_t s) { PETDENSE_BY_TYPE(type, return pad_t<T>(p, s)) }

hipError_t join_columns(const ColumnJoin& c, hipStream_t s) {
  const unsigned blocks = std::min(blocks_for(c.N, 16), 1u << 20);      // (2^28 columns would be 2^32 threads)
  return launch_kernel(join_columns_kernel, dim3(blocks), dim3(256), 0, s, c);
}

__global__ __launch_bounds__(256) void fill_zero_kernel(char* p, int64_t total, int n, int64_t ld, int size) {
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < total; t += (int64_t)gridDim.x * 256) {
    const int64_t r = t / n;
    char* d = p + (r * ld + (t - r * n)) * size;
    if (size == 4) *reinterpret_cast<float*>(d) = 0.f;
    else *reinterpret_cast<uint16_t*>(d) = 0;
  }
}

hipError_t fill_zero(void* p, int64_t rows, int n, int64_t ld, int size, hipStream_t s) {
  const int64_t total = rows * n;
  return launch_kernel(fill_zero_kernel, dim3((unsigned)std::min<int64_t>(4096, (total + 255) / 256)), dim3(256), 0, s,
                       static_cast<char*>(p), total, n, ld, size);
}

hipError_t quantize(const void* x, int64_t ldx, int64_t M, int K, int type, uint8_t* codes, int64_t ldc, uint8_t* exps,
                    int64_t lde, hipStream_t s) {
  PETDENSE_BY_TYPE(type, return quantize_t<T>(x, ldx, M, K, codes, ldc, exps, lde, s))
}

hipError_t restore(const uint8_t* codes, int64_t ldc, const uint8_t* exps, int64_t lde, int64_t M, int K, int type,
                   void* x, int64_t ldx, hipStream_t s) {
  PETDENSE_BY_TYPE(type, return restore_t<T>(codes, ldc, exps, lde, M, K, x, ldx, s))
}

}  // namespace petdense_k
