// The tiled matrix product of the dense layer (forward, input gradient, kernel gradient) for gfx950.
//
//   C[i][j] = sum_c A(i, c) B(c, j)
//
// A workgroup owns a BI x BJ tile of C; its waves split the tile, each holding its part in fp32 accumulators.  Per
// step the workgroup stages BC contraction values of both operands in LDS (128 bytes of each operand's row or
// BC rows), two stages deep: the loads of step t + 1 are in flight while step t is multiplied, one barrier a step.
// 16-bit operands go through v_mfma_f32_16x16x32, fp32 through v_mfma_f32_16x16x4.
//
// Operands are taken as they lie in memory:
//  - contraction-contiguous ([free][c]): a lane's fragment is 16 bytes of its row, one ds_read_b128;
//  - free-contiguous ([c][free]): the fragment runs down a column; 16-bit ones are transposed on the way out of
//    LDS by ds_read_b64_tr_b16 (16 lanes read 4 rows of 16 values and get 4 values of one column each).
// No operand is copied or transposed in memory.
//
// The fragments enter the matrix instruction with B's as the row operand, so that a lane ends with four
// neighbouring j of one i: the epilogue reads and writes four values at a time.
#pragma once
#include "dense_epilogue.h"

namespace petdense_k {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef short i16x8 __attribute__((ext_vector_type(8)));

#define PETDENSE_LDS __attribute__((address_space(3)))

__device__ void raw_buffer_load_lds(i32x4 rsrc, PETDENSE_LDS void* lds, int size, int voffset, int soffset,
                                    int offset, int aux) __asm("llvm.amdgcn.raw.buffer.load.lds");

// A stage of one operand: ROWS rows of CPR 16-byte pieces.  Piece c of row r lies at place c ^ key(r) of the row, so
// that the lanes of one LDS read, which take the same piece of several rows, meet every bank once.
template <typename T, bool FREE, int R, int BC>
struct Stage {
  static constexpr int EPC = 16 / (int)sizeof(T);                    // values of a piece
  static constexpr int ROWS = FREE ? BC : R;
  static constexpr int CPR = (FREE ? R : BC) / EPC;
  static constexpr int PIECES = ROWS * CPR;
  static constexpr int BYTES = PIECES * 16;
  __device__ static int key(int r) {
    if constexpr (!FREE) return r & 7;                               // CPR = 8
    else if constexpr (sizeof(T) == 4) return ((r >> 2) & (CPR >= 16 ? 3 : CPR / 4 - 1)) << 2;
    else if constexpr (CPR >= 16) return ((r & 3) | ((r >> 1) & 4)) << 1;
    else if constexpr (CPR == 8) return (((r >> 1) & 1) | ((r >> 2) & 2)) << 1;
    else return 0;
  }
};

template <typename T>
struct Frag;
template <>
struct Frag<__bf16> { typedef bf16x8 type; };
template <>
struct Frag<_Float16> { typedef f16x8 type; };
template <>
struct Frag<float> { typedef f32x4 type; };

template <typename T>
__device__ __forceinline__ f32x4 multiply(typename Frag<T>::type a, typename Frag<T>::type b, f32x4 c) {
  if constexpr (__is_same(T, __bf16)) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  else if constexpr (__is_same(T, _Float16)) return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  else {
#pragma unroll
    for (int q = 0; q < 4; ++q) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[q], b[q], c, 0, 0, 0);
    return c;
  }
}

// The fragment of 16 free values from r0 (a multiple of 16) and contraction group ks of the stage.  Lane (g, i) =
// (lane / 16, lane % 16) holds free value r0 + i and the contraction values 8 g .. 8 g + 7 of the group's 32
// (fp32: 4 g .. 4 g + 3 of its 16; the four instructions take one each).
template <typename T, bool FREE, int R, int BC>
__device__ __forceinline__ typename Frag<T>::type fragment(const char* st, int r0, int ks, int lane) {
  using S = Stage<T, FREE, R, BC>;
  const int g = lane >> 4, i = lane & 15;
  if constexpr (!FREE) {
    const int r = r0 + i;
    return *reinterpret_cast<const typename Frag<T>::type*>(st + (r * S::CPR + ((ks * 4 + g) ^ S::key(r))) * 16);
  } else if constexpr (sizeof(T) == 4) {
    f32x4 v;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int r = ks * 16 + g * 4 + q;
      v[q] = *reinterpret_cast<const float*>(st + (r * S::CPR + (((r0 + i) >> 2) ^ S::key(r))) * 16 + (i & 3) * 4);
    }
    return v;
  } else {
    i16x4 h[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int r = ks * 32 + g * 8 + q * 4 + (i >> 2);
      const int c = (r0 >> 3) + ((i & 3) >> 1);
      h[q] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (PETDENSE_LDS i16x4*)(st + (r * S::CPR + (c ^ S::key(r))) * 16 + (i & 1) * 8));
    }
    const i16x8 v = __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(typename Frag<T>::type, v);
  }
}

// Fills stages of one operand.  `c0` is the operand's first contraction value, `clen` the values of this part.
// LOADER kDma: rows and row starts are multiples of 16 bytes: buffer loads that write LDS themselves; a piece outside
//   the operand gets an offset past the buffer's end, and the hardware writes zeros for it.
// LOADER kReg: any alignment: through registers, loaded before the step's products and stored after them.
// Q8: the operand is e4m3 codes with exponent bytes, free-contiguous: through registers, restored to T on the way.
template <typename T, bool FREE, int R, int BC, int THREADS, int LOADER, bool Q8>
struct Filler {
  using S = Stage<T, FREE, R, BC>;
  static constexpr int N = (S::PIECES + THREADS - 1) / THREADS;      // pieces of a thread
  static_assert(S::PIECES % THREADS == 0, "every thread stages the same number of pieces");
  static_assert(!Q8 || FREE, "8-bit operands are free-contiguous");
  const char* base;      // the tile's first value at contraction value 0 of this part
  int64_t ld;            // bytes from row to row
  int limit;             // free values of the tile that exist
  int clen;
  const uint8_t* exps;   // Q8: exponent byte of the tile's first block at the part's first row
  int64_t lde;
  int voff[LOADER == kDma ? N : 1];
  u32x4 reg[LOADER == kDma ? 1 : N];

  __device__ void init(const void* p, int64_t ld_values, int f0, int f_limit, int64_t c0, int clen_,
                       const uint8_t* ex, int64_t lde_, int tid) {
    constexpr int SZ = Q8 ? 1 : (int)sizeof(T);
    ld = ld_values * SZ;
    base = static_cast<const char*>(p) + (FREE ? c0 * ld + (int64_t)f0 * SZ : f0 * ld + c0 * SZ);
    limit = f_limit - f0;
    clen = clen_;
    exps = Q8 ? ex + c0 * lde_ + f0 / 32 : nullptr;
    lde = lde_;
    if constexpr (LOADER == kDma) {
#pragma unroll
      for (int q = 0; q < N; ++q) {
        const int k = q * THREADS + tid, r = k / S::CPR, c = (k % S::CPR) ^ S::key(r);
        const bool in = FREE ? c * S::EPC < limit : r < limit;
        voff[q] = in ? (int)(r * ld) + c * 16 : (int)0x80000000;
      }
    }
  }

  // the first bytes of step t
  __device__ const char* step(int t) const {
    return base + (FREE ? (int64_t)t * BC * ld : (int64_t)t * BC * (int64_t)sizeof(T));
  }

  // begins the loads of step t (kDma: into `st`)
  __device__ __forceinline__ void begin(char* st, int t, int tid) {
    const int left = clen - t * BC;                                  // contraction values of this step that exist
    if constexpr (LOADER == kDma) {
      const unsigned long long a = reinterpret_cast<unsigned long long>(step(t));
      i32x4 rs;
      rs[0] = __builtin_amdgcn_readfirstlane((int)(a & 0xffffffffull));
      rs[1] = __builtin_amdgcn_readfirstlane((int)((a >> 32) & 0xffffull));
      rs[2] = (int)0x80000000;
      rs[3] = 0x00020000;
      const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
#pragma unroll
      for (int q = 0; q < N; ++q) {
        int o = voff[q];
        if (left < BC) {
          const int k = q * THREADS + tid, r = k / S::CPR, c = (k % S::CPR) ^ S::key(r);
          if (FREE ? r >= left : c * S::EPC >= left) o = (int)0x80000000;
        }
        raw_buffer_load_lds(rs, (PETDENSE_LDS void*)(st + (q * THREADS + wave * 64) * 16), 16, o, 0, 0, 0);
      }
    } else {
      const char* p = step(t);
#pragma unroll
      for (int q = 0; q < N; ++q) {
        const int k = q * THREADS + tid, r = k / S::CPR, c = (k % S::CPR) ^ S::key(r);
        // values of the piece that exist
        const int n = FREE ? (r < left ? limit - c * S::EPC : 0) : (r < limit ? left - c * S::EPC : 0);
        reg[q] = u32x4{0, 0, 0, 0};
        if constexpr (Q8) {
          const char* s = p + r * ld + c * S::EPC;
          unsigned w[2] = {0, 0};
          if (n >= S::EPC) __builtin_memcpy(w, s, S::EPC);
          else
            for (int v = 0; v < n; ++v) w[v >> 2] |= (unsigned)(uint8_t)s[v] << ((v & 3) * 8);
          // a step past the end keeps no exponent: its codes are zero
          const unsigned b = n > 0 ? exps[((int64_t)t * BC + r) * lde + (c * S::EPC) / 32] : 127;
          reg[q][0] = w[0];
          reg[q][1] = w[1];
          reg[q][2] = b;
        } else {
          const char* s = p + r * ld + c * 16;
          if (n >= S::EPC) {
            __builtin_memcpy(&reg[q], s, 16);
          } else if (n > 0) {
            T v[S::EPC];
#pragma unroll
            for (int x = 0; x < S::EPC; ++x) {
              v[x] = (T)0.f;
              if (x < n) __builtin_memcpy(&v[x], s + x * sizeof(T), sizeof(T));
            }
            __builtin_memcpy(&reg[q], v, 16);
          }
        }
      }
    }
  }

  // ends them: kReg: writes the registers to `st`
  __device__ __forceinline__ void end(char* st, int tid) {
    if constexpr (LOADER == kReg) {
#pragma unroll
      for (int q = 0; q < N; ++q) {
        u32x4 w = reg[q];
        if constexpr (Q8) {
          const float sc = exponent_scale(w[2]);
          T v[S::EPC];
          restore4<T>(w[0], sc, v);
          if constexpr (S::EPC == 8) restore4<T>(w[1], sc, v + 4);
          __builtin_memcpy(&w, v, 16);
        }
        *reinterpret_cast<u32x4*>(st + (q * THREADS + tid) * 16) = w;
      }
    }
  }
};

// Own loads and LDS accesses done, then a bare barrier.
__device__ __forceinline__ void step_barrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

template <typename T, int BI, int BJ, int WI, int WJ, bool FA, bool FB, int LA, int LB, bool Q8>
struct Shape {
  static constexpr int BC = 128 / (int)sizeof(T);
  static constexpr int THREADS = WI * WJ * 64;
  static constexpr int LDS = 2 * (Stage<T, FA, BI, BC>::BYTES + Stage<T, FB, BJ, BC>::BYTES);
};

// Workgroup -> tile.  Neighbouring workgroup numbers go to different XCDs, each with its own L2: every XCD gets a
// contiguous run of tiles, and a run walks bands of 4 tile rows, so that the workgroups an XCD runs together share
// rows of A and columns of B.
__device__ __forceinline__ void tile_of(int b, int ti, int tj, int& i, int& j) {
  const int n = ti * tj;
  const int per = n / 8, rest = n % 8, x = b % 8;
  const int t = x * per + min(x, rest) + b / 8;
  constexpr int BAND = 4;
  const int band = t / (BAND * tj), first = band * BAND, h = min(BAND, ti - first), r = t - first * tj;
  i = first + r % h;
  j = r / h;
}

template <typename T, int BI, int BJ, int WI, int WJ, bool FA, bool FB, int LA, int LB, bool Q8>
__global__ __launch_bounds__(WI* WJ * 64) void product_kernel(Product p) {
  using SH = Shape<T, BI, BJ, WI, WJ, FA, FB, LA, LB, Q8>;
  constexpr int BC = SH::BC, THREADS = SH::THREADS;
  using SA = Stage<T, FA, BI, BC>;
  using SB = Stage<T, FB, BJ, BC>;
  constexpr int STAGE = SA::BYTES + SB::BYTES;
  constexpr int FI = BI / WI / 16, FJ = BJ / WJ / 16, KS = 2;
  extern __shared__ char lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wi = wave / WJ, wj = wave % WJ;
  int ti, tj;
  tile_of(blockIdx.x, (p.I + BI - 1) / BI, (p.J + BJ - 1) / BJ, ti, tj);
  const int i0 = ti * BI, j0 = tj * BJ;
  const int64_t c0 = (int64_t)blockIdx.y * p.c_per;
  const int clen = (int)min((int64_t)p.c_per, p.C - c0);
  const int steps = (clen + BC - 1) / BC;

  Filler<T, FA, BI, BC, THREADS, LA, Q8> fa;
  Filler<T, FB, BJ, BC, THREADS, LB, false> fb;
  fa.init(p.A, p.lda, i0, p.I, c0, clen, p.exps, p.lde, tid);
  fb.init(p.B, p.ldb, j0, p.J, c0, clen, nullptr, 0, tid);

  f32x4 acc[FI][FJ];
#pragma unroll
  for (int x = 0; x < FI; ++x)
#pragma unroll
    for (int y = 0; y < FJ; ++y) acc[x][y] = f32x4{0.f, 0.f, 0.f, 0.f};

  fa.begin(lds, 0, tid);
  fb.begin(lds + SA::BYTES, 0, tid);
  fa.end(lds, tid);
  fb.end(lds + SA::BYTES, tid);
  for (int t = 0; t < steps; ++t) {
    char* cur = lds + (t & 1) * STAGE;
    char* nxt = lds + ((t & 1) ^ 1) * STAGE;
    step_barrier();             // step t has landed, and every wave is done with step t - 1's stage
    if (t + 1 < steps) {
      fa.begin(nxt, t + 1, tid);
      fb.begin(nxt + SA::BYTES, t + 1, tid);
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      typename Frag<T>::type a[FI], b[FJ];
#pragma unroll
      for (int y = 0; y < FJ; ++y)
        b[y] = fragment<T, FB, BJ, BC>(cur + SA::BYTES, wj * (BJ / WJ) + y * 16, ks, lane);
#pragma unroll
      for (int x = 0; x < FI; ++x) a[x] = fragment<T, FA, BI, BC>(cur, wi * (BI / WI) + x * 16, ks, lane);
#pragma unroll
      for (int x = 0; x < FI; ++x)
#pragma unroll
        for (int y = 0; y < FJ; ++y) acc[x][y] = multiply<T>(b[y], a[x], acc[x][y]);
    }
    if (t + 1 < steps) {
      fa.end(nxt, tid);
      fb.end(nxt + SA::BYTES, tid);
    }
  }

  const int g = lane >> 4, il = lane & 15;
#pragma unroll
  for (int x = 0; x < FI; ++x) {
    const int i = i0 + wi * (BI / WI) + x * 16 + il;
    if (i >= p.I) continue;
#pragma unroll
    for (int y = 0; y < FJ; ++y) {
      const int j = j0 + wj * (BJ / WJ) + y * 16 + g * 4;
      const int n = p.J - j;
      if (n <= 0) continue;
      if (p.splits > 1) {
        float* o = p.part + ((int64_t)blockIdx.y * p.I + i) * p.J + j;
        if (n >= 4 && p.J % 4 == 0) {
          *reinterpret_cast<f32x4*>(o) = acc[x][y];
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (q < n) o[q] = acc[x][y][q];
        }
      } else {
        epilogue4<T>(p.e, i, j, n, acc[x][y]);
      }
    }
  }
}

template <typename T, int BI, int BJ, int WI, int WJ, bool FA, bool FB, int LA, int LB, bool Q8>
hipError_t launch(const Product& p, hipStream_t s) {
  using SH = Shape<T, BI, BJ, WI, WJ, FA, FB, LA, LB, Q8>;
  auto k = product_kernel<T, BI, BJ, WI, WJ, FA, FB, LA, LB, Q8>;
  hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize,
                                     SH::LDS);
  if (e != hipSuccess) return e;
  const int64_t tiles = (int64_t)((p.I + BI - 1) / BI) * ((p.J + BJ - 1) / BJ);
  hipLaunchKernelGGL(k, dim3((unsigned)tiles, (unsigned)p.splits), dim3(SH::THREADS), SH::LDS, s, p);
  return hipGetLastError();
}

template <typename T, int BI, int BJ, int WI, int WJ>
hipError_t product_tile(const Product& p, int layout, int loader, int q8, hipStream_t s) {
  if constexpr (BI == 256) {      // the plan takes the largest tile only for operands that DMA can stage
    if (loader != kDma) return hipErrorInvalidValue;
    if (layout == kForward) return launch<T, BI, BJ, WI, WJ, false, true, kDma, kDma, false>(p, s);
    if (layout == kInputGrad) return launch<T, BI, BJ, WI, WJ, false, false, kDma, kDma, false>(p, s);
    return q8 ? launch<T, BI, BJ, WI, WJ, true, true, kReg, kDma, true>(p, s)
              : launch<T, BI, BJ, WI, WJ, true, true, kDma, kDma, false>(p, s);
  } else {
  if (layout == kForward)
    return loader == kDma ? launch<T, BI, BJ, WI, WJ, false, true, kDma, kDma, false>(p, s)
                          : launch<T, BI, BJ, WI, WJ, false, true, kReg, kReg, false>(p, s);
  if (layout == kInputGrad)
    return loader == kDma ? launch<T, BI, BJ, WI, WJ, false, false, kDma, kDma, false>(p, s)
                          : launch<T, BI, BJ, WI, WJ, false, false, kReg, kReg, false>(p, s);
  if (q8)
    return loader == kDma ? launch<T, BI, BJ, WI, WJ, true, true, kReg, kDma, true>(p, s)
                          : launch<T, BI, BJ, WI, WJ, true, true, kReg, kReg, true>(p, s);
  return loader == kDma ? launch<T, BI, BJ, WI, WJ, true, true, kDma, kDma, false>(p, s)
                        : launch<T, BI, BJ, WI, WJ, true, true, kReg, kReg, false>(p, s);
  }
}

template <typename T>
hipError_t product(const Product& p, int layout, int loader, int tile, int q8, hipStream_t s) {
  if (tile == kLarge) return product_tile<T, 256, 256, 2, 4>(p, layout, loader, q8, s);
  if (tile == kMid) return product_tile<T, 128, 128, 2, 2>(p, layout, loader, q8, s);
  return product_tile<T, 64, 64, 2, 2>(p, layout, loader, q8, s);
}

}  // namespace petdense_k
