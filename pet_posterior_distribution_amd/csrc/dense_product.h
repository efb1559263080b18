// The tiled matrix product of the dense layer (forward, input gradient, kernel gradient) for gfx950.
//
//   C[i][j] = sum_c A(i, c) B(c, j)
//
// A workgroup owns a BI x BJ tile of C; its waves split the tile, each holding its part in fp32 accumulators.  Per
// step the workgroup stages BC contraction values of both operands in LDS (128 bytes of each operand's row or
// BC rows), two stages deep.  16-bit operands go through v_mfma_f32_16x16x32, fp32 through v_mfma_f32_16x16x4.
// A step is two groups of products (KS = 2), and every read is one group ahead of its use:
//   group 0: read group 1's fragments while group 0 is multiplied
//   wait: group 1's fragments are in registers, the next stage has landed; barrier: so it is for every wave
//   group 1: the load of the stage after the next goes into the stage just read; read the next stage's group 0
//            fragments while group 1 is multiplied
// so neither a barrier nor LDS latency stands before a product, and a load has a whole step to land.
//
// Operands are taken as they lie in memory:
//  - contraction-contiguous ([free][c]): a lane's fragment is 16 bytes of its row, one ds_read_b128;
//  - free-contiguous ([c][free]): the fragment runs down a column; 16-bit ones are transposed on the way out of
//    LDS by ds_read_b64_tr_b16 (16 lanes read 4 rows of 16 values and get 4 values of one column each).
// No operand is copied or transposed in memory.
//
// The fragments enter the matrix instruction with B's as the row operand, so that a lane ends with four
// neighbouring j of one i: the epilogue reads and writes four values at a time.
//
// What bounds it, and what it measured (the library's product of the same operands in brackets, no epilogue):
//  - large products by the matrix units at the clock that power leaves: 8192 x 4096 x 8192 bf16 in 424 us, 1.30 PFLOP/s
//    (412 .. 423 us), its input gradient 405 us, its kernel gradient 412 us; matrix instructions in 66 % of the busy
//    cycles, no LDS bank conflict; fp32 83 % (its matrix instructions take as many cycles for a sixteenth of the work),
//    76 % with 64 x 64 tiles (6144 x 1836 x 512, 103 us);
//  - short contractions by the tile's first loads and its stores: input gradient of 12288 x 6144 x 512 in 103 us
//    (115 .. 122 us), where its operations alone take 59 us and its stores 30 us;
//  - few outputs by latency: 9 x 600 x 5000 in 4.2 us, 40 x 4100 x 64 in 4.9 us and 4.0 us for the join.
#pragma once
#include "dense_epilogue.h"

#include <algorithm>
#include <atomic>
#include <type_traits>

namespace petdense_k {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef short i16x8 __attribute__((ext_vector_type(8)));

#define PETDENSE_LDS __attribute__((address_space(3)))

// One wave's buffer load of 64 x 16 bytes straight into LDS at `lds` (wave-uniform) + 16 lane.  In assembly, because
// the compiler would put a wait for it before every LDS read that follows; the kernel waits for it itself, before the
// barrier that publishes a stage.  (No output register: nothing the compiler could reuse early.)
__device__ __forceinline__ void load_to_lds(i32x4 rsrc, unsigned lds, int voffset, int soffset) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds), "v"(voffset),
               "s"(rsrc), "s"(soffset)
               : "memory", "m0");
}

// A stage of one operand: ROWS rows of CPR 16-byte pieces.  Piece c of row r lies at place c ^ key(r) of the row, so
// that the lanes of one LDS read, which take the same piece of several rows, meet every bank once.
template <typename T, bool FREE, int R, int BC>
struct Stage {
  static constexpr int EPC = 16 / (int)sizeof(T);                    // values of a piece
  static constexpr int ROWS = FREE ? BC : R;
  static constexpr int CPR = (FREE ? R : BC) / EPC;
  static constexpr int PIECES = ROWS * CPR;
  static constexpr int BYTES = PIECES * 16;
  __host__ __device__ static constexpr int key(int r) {
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

// acc[y] += b[y] a: one row of a wave's 16 x 16 tiles.  fp32: the four instructions of a product are spread over the
// row, so that none waits for the one before it.
template <typename T, int N>
__device__ __forceinline__ void multiply_row(const typename Frag<T>::type* b, typename Frag<T>::type a, f32x4* acc) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int y = 0; y < N; ++y) acc[y] = __builtin_amdgcn_mfma_f32_16x16x4f32(b[y][q], a[q], acc[y], 0, 0, 0);
  } else {
#pragma unroll
    for (int y = 0; y < N; ++y) {
      if constexpr (__is_same(T, __bf16)) acc[y] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[y], a, acc[y], 0, 0, 0);
      else acc[y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b[y], a, acc[y], 0, 0, 0);
    }
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
// LOADER kReg: any alignment: through registers, loaded a step ahead and stored after the step's first group.
// Q8: the operand is e4m3 codes with exponent bytes, free-contiguous: through registers, restored to T on the way.
// ACT: the operand is dP = dy act'(saved), made from two sources on the way (kReg), rounded to T as a dP in memory is.
// KW > 1: the filler's wave takes every KW-th step, from step `kw`.
template <typename T, bool FREE, int R, int BC, int THREADS, int KW, int LOADER, bool Q8, bool ACT>
struct Filler {
  using S = Stage<T, FREE, R, BC>;
  static constexpr int N = (S::PIECES + THREADS - 1) / THREADS;      // pieces of a thread
  static_assert(S::PIECES % THREADS == 0, "every thread stages the same number of pieces");
  static_assert(!Q8 || FREE, "8-bit operands are free-contiguous");
  const char* base;      // the tile's first value at contraction value 0 of this part
  int64_t ld;            // bytes from row to row
  int limit;             // free values of the tile that exist
  bool brief;            // kReg: value by value: rows shorter than a piece, or exponents too far apart for its offsets
  int clen, kw;
  const uint8_t* exps;   // Q8: exponent byte of the tile's first block at the part's first row
  int64_t lde;
  // pieces of a thread: rows r0, r0 + RPQ, ..; `same`: all at one place of their rows
  static constexpr int RPQ = THREADS / S::CPR;
  static constexpr bool same() {
    for (int q = 1; q < N; ++q)
      for (int r = 0; r < RPQ; ++r)
        if (S::key(r + q * RPQ) != S::key(r)) return false;
    return true;
  }
  static constexpr bool SAME = same();
  static_assert(THREADS % S::CPR == 0, "");
  int v0;                // kDma: bytes from a step's first to the thread's first row, and with SAME to its piece
  u32x4 reg[LOADER == kDma ? 1 : N];
  const char* base2;     // ACT: the same of `saved`
  int64_t ld2;
  int act;
  u32x4 reg2[ACT ? N : 1];
  static_assert(!ACT || (LOADER == kReg && !Q8), "dP is staged through registers");

  __device__ void init(const void* p, int64_t ld_values, int f0, int f_limit, int64_t c0, int clen_, int c_all,
                       const uint8_t* ex, int64_t lde_, int kw_, int tid) {
    kw = kw_;
    brief = (FREE ? f_limit : c_all) < S::EPC || (Q8 && !exponents_fit(lde_));
    constexpr int SZ = Q8 ? 1 : (int)sizeof(T);
    ld = ld_values * SZ;
    base = static_cast<const char*>(p) + (FREE ? c0 * ld + (int64_t)f0 * SZ : f0 * ld + c0 * SZ);
    limit = f_limit - f0;
    clen = clen_;
    exps = Q8 ? ex + c0 * lde_ + f0 / 32 : nullptr;
    lde = lde_;
    if constexpr (LOADER == kDma) {
      const int r = tid / S::CPR;
      v0 = r * (int)ld + (SAME ? ((tid % S::CPR) ^ S::key(r)) * 16 : 0);
    }
  }

  __device__ void init_saved(const void* p, int64_t ld_values, int act_, int f0, int64_t c0) {
    act = act_;
    ld2 = act ? ld_values * (int64_t)sizeof(T) : ld;
    // without an activation nothing of `saved` counts: dy stands in for it
    base2 = !act ? base : static_cast<const char*>(p) + (FREE ? c0 * ld2 + (int64_t)f0 * (int64_t)sizeof(T)
                                                              : f0 * ld2 + c0 * (int64_t)sizeof(T));
  }

  // what every piece of the t-th step needs
  struct Step {
    i32x4 rs;            // kDma: the buffer that begins at the step
    const char* p;
    const char* p2;
    int t, left;         // contraction values of the step that exist (<= 0: a step past the end loads nothing)
    bool whole;          // kReg: no piece has to be cut
  };
  __device__ __forceinline__ Step at(int t) const {
    Step u;
    u.t = KW > 1 ? t * KW + kw : t;
    u.left = clen - u.t * BC;
    u.p = base + (FREE ? (int64_t)u.t * BC * ld : (int64_t)u.t * BC * (int64_t)sizeof(T));
    if constexpr (ACT) u.p2 = base2 + (FREE ? (int64_t)u.t * BC * ld2 : (int64_t)u.t * BC * (int64_t)sizeof(T));
    // free-contiguous: 16 bytes from a piece's first value may run into the next row, which then has to exist
    // (offsets within a step fit 31 bits)
    u.whole = !brief && (FREE ? u.left > BC && ld >= 16 : u.left >= BC) && ld < kMaxRowBytes &&
              (!ACT || ((!FREE || ld2 >= 16) && ld2 < kMaxRowBytes));
    if constexpr (LOADER == kDma) {
      const unsigned long long a = reinterpret_cast<unsigned long long>(u.p);
      u.rs[0] = __builtin_amdgcn_readfirstlane((int)(a & 0xffffffffull));
      u.rs[1] = __builtin_amdgcn_readfirstlane((int)((a >> 32) & 0xffffull));
      u.rs[2] = (int)0x80000000;
      u.rs[3] = 0x00020000;
    }
    return u;
  }

  // begins the load of the thread's piece q of a step into LDS at `st`
  __device__ __forceinline__ void begin(char* st, const Step& u, int q, int tid) {
    if constexpr (LOADER == kDma) {
      const int r = tid / S::CPR + q * RPQ, c = (tid % S::CPR) ^ S::key(r);
      const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
      const bool in = FREE ? r < u.left && c * S::EPC < limit : r < limit && c * S::EPC < u.left;
      load_to_lds(u.rs, (unsigned)(uintptr_t)(PETDENSE_LDS char*)st + (q * THREADS + wave * 64) * 16,
                  in ? v0 + (SAME ? 0 : c * 16) : (int)0x80000000, q * RPQ * (int)ld);
    }
  }

  // Begins the loads of a step into registers, each a whole piece of any alignment, with no branch on the lane:
  //  - whole steps: pieces past the operand's free end read its first value instead (they feed outputs that are not
  //    stored);
  //  - cut steps: a piece that ends past its row is read so that it ends with it, and shifted; what does not exist
  //    becomes zero;
  //  - `brief`: value by value, by 64-bit offsets.
  __device__ __forceinline__ void begin_reg(const Step& u, int tid) {
    if constexpr (LOADER == kReg) {
      constexpr int SZ = Q8 ? 1 : (int)sizeof(T), PB = SZ * S::EPC;        // bytes of a value and a piece in memory
      if (u.whole) {
#pragma unroll
        for (int q = 0; q < N; ++q) {
          const int k = q * THREADS + tid, r = k / S::CPR, c = (k % S::CPR) ^ S::key(r);
          const int rr = FREE ? r : min(r, limit - 1), cc = FREE && c * S::EPC >= limit ? 0 : c;
          load_piece(reg[q], u.p + (unsigned)(rr * (int)ld + cc * PB));
          if constexpr (ACT) load_piece(reg2[q], u.p2 + (unsigned)(rr * (int)ld2 + cc * PB));
          if constexpr (Q8)
            reg[q][2] = (exps + (int64_t)u.t * BC * lde)[exponent_offset(r, lde, (cc * S::EPC) / 32)];
        }
        return;
      }
      if (u.left <= 0) {
#pragma unroll
        for (int q = 0; q < N; ++q) {
          reg[q] = u32x4{0, 0, Q8 ? 127u : 0u, 0};
          if constexpr (ACT) reg2[q] = u32x4{0, 0, 0, 0};
        }
        return;
      }
      // cut steps are rare: nothing of theirs is worth a register across the others
      asm volatile("" : "+v"(tid));
#pragma unroll
      for (int q = 0; q < N; ++q) {
        const int k = q * THREADS + tid, r = k / S::CPR, c = (k % S::CPR) ^ S::key(r);
        // the piece's row (clamped to one that exists), its first value in it, and the values that follow
        const int64_t row = FREE ? min((int64_t)u.t * BC + r, (int64_t)clen - 1) : min(r, limit - 1);
        const int64_t first = (FREE ? 0 : (int64_t)u.t * BC) + c * S::EPC;
        const int64_t after = (FREE ? limit : clen) - first;
        const bool in = FREE ? r < u.left : r < limit;
        const int n = !in || after <= 0 ? 0 : after < S::EPC ? (int)after : S::EPC;
        const char* p = base + row * ld;
        const char* p2 = ACT ? base2 + row * ld2 : nullptr;
        if (brief) {
#pragma unroll 1
          for (int x = S::EPC - 1; x >= 0; --x) {
            // the values come in from the last to the first, each moving those behind it up
            const int64_t at = min(first + x, (int64_t)(FREE ? limit : clen) - 1) * SZ;
            unsigned one = 0;
            __builtin_memcpy(&one, p + at, SZ);
            push_value(reg[q], x < n ? one : 0u);
            if constexpr (ACT) {
              __builtin_memcpy(&one, p2 + at, SZ);
              push_value(reg2[q], x < n ? one : 0u);
            }
          }
        } else {
          const int64_t at = after >= S::EPC ? first : (int64_t)(FREE ? limit : clen) - S::EPC;
          const int bits = (after >= S::EPC && in ? 0 : S::EPC - n) * SZ * 8;
          load_piece(reg[q], p + at * SZ);
          shift_piece(reg[q], bits);
          if constexpr (ACT) {
            load_piece(reg2[q], p2 + at * SZ);
            shift_piece(reg2[q], bits);
          }
        }
        if constexpr (Q8) reg[q][2] = exps[row * lde + min(first, (int64_t)limit - 1) / 32];
      }
    }
  }

  __device__ __forceinline__ void load_piece(u32x4& r, const char* s) {
    if constexpr (Q8) {
      unsigned w[2] = {0, 0};
      __builtin_memcpy(w, s, S::EPC);
      r[0] = w[0];
      r[1] = w[1];
    } else {
      __builtin_memcpy(&r, s, 16);
    }
  }
  // moves the piece's values up by one and puts `v` in front
  __device__ __forceinline__ void push_value(u32x4& r, unsigned v) {
    constexpr int BITS = Q8 ? 8 : 8 * (int)sizeof(T);
#pragma unroll
    for (int w = Q8 ? 1 : 3; w >= 0; --w) {
      const unsigned below = w ? r[w - 1] : 0;
      if constexpr (BITS == 32) r[w] = w ? below : v;
      else r[w] = r[w] << BITS | (w ? below >> (32 - BITS) : v);
    }
  }
  // moves the piece's values down by `bits`, zeros behind them
  __device__ __forceinline__ void shift_piece(u32x4& r, int bits) {
    const uint64_t lo = r[0] | (uint64_t)r[1] << 32;
    if constexpr (Q8) {
      constexpr int ALL = S::EPC * 8;
      const uint64_t v = bits >= ALL ? 0 : lo >> bits;
      r[0] = (unsigned)v;
      r[1] = (unsigned)(v >> 32);
    } else {
      const uint64_t hi = r[2] | (uint64_t)r[3] << 32;
      const int b = bits & 63;
      const uint64_t lo1 = (lo >> b) | (b ? hi << (64 - b) : 0), hi1 = hi >> b;
      const uint64_t l = bits >= 128 ? 0 : bits >= 64 ? hi1 : lo1, h = bits >= 64 ? 0 : hi1;
      r = u32x4{(unsigned)l, (unsigned)(l >> 32), (unsigned)h, (unsigned)(h >> 32)};
    }
  }

  __device__ __forceinline__ void begin_all(char* st, int t, int tid) {
    const Step u = at(t);
#pragma unroll
    for (int q = 0; q < N; ++q) begin(st, u, q, tid);
    begin_reg(u, tid);
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
        } else if constexpr (ACT) {
          T d[S::EPC], v[S::EPC];
          __builtin_memcpy(d, &w, 16);
          __builtin_memcpy(v, &reg2[q], 16);
          float gf[S::EPC], vf[S::EPC];
#pragma unroll
          for (int x = 0; x < S::EPC; ++x) gf[x] = (float)d[x], vf[x] = (float)v[x];
          activate_grads<sizeof(T) == 4, S::EPC>(gf, vf, act);
#pragma unroll
          for (int x = 0; x < S::EPC; ++x) d[x] = (T)gf[x];
          __builtin_memcpy(&w, d, 16);
        }
        *reinterpret_cast<u32x4*>(st + (q * THREADS + tid) * 16) = w;
      }
    }
  }
};

// All but the last N of this wave's loads have landed, its LDS accesses are done; then, where waves share stages, a
// bare barrier.
template <int N, bool SHARED>
__device__ __forceinline__ void step_barrier() {
  if constexpr (SHARED) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
  else asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}

// A kind of tile: BI x BJ outputs, by WI x WJ waves that share the stages; or (KW > 1) by KW waves that each multiply
// the whole tile over every KW-th step, from stages of their own, and meet at the end: for few outputs with a long
// contraction, where one wave after another would wait for memory.
template <int BI_, int BJ_, int WI_, int WJ_, int KW_>
struct Kind {
  static constexpr int BI = BI_, BJ = BJ_, WI = WI_, WJ = WJ_, KW = KW_;
  static constexpr int THREADS = WI * WJ * KW * 64;
  static constexpr int LDS = 2 * KW * (BI + BJ) * 128;
  // the largest tile's workgroups stay and walk (its first loads and its stores are a large part of a tile's time;
  // smaller tiles run several workgroups on a compute unit, which hide them from each other)
  static constexpr bool STREAM = BI == 256;
  static constexpr int TURN = 16 * (BJ / WJ) * 4;                         // a wave's 16 rows of outputs in fp32
  static constexpr int LAUNCH_LDS = LDS + (STREAM ? WI * WJ * TURN : 0);
  static_assert(KW == 1 || WI * WJ == 1, "");
};
// Large: 32 products of a wave for 12 fragments (Mid: 16 for 8), but one workgroup on a compute unit: 8192 x 8192 x
//   4096's input gradient took 607 us with a tile a workgroup, 431 us with workgroups that walk.
// Mid, Small: 2 and 4 workgroups on a compute unit, which hide each other's loads and stores: 50176 x 256 x 128 in
//   13 us (its bytes: 7.6 us), 777 x 1069 x 333 through registers in 14.5 us with its join.
// Slice, Slice64: few outputs; 24576 x 1536 x 128's kernel gradient took 32 us with 4 parts of Slice64, 26 us with 16
//   of Small, 53 us with 4 of Slice, which stages twice the bytes per product; 1846 x 160 x 1680's 11 us with Small or
//   Slice64, 15 us with Slice.
typedef Kind<256, 256, 2, 4, 1> Large;
typedef Kind<128, 128, 2, 2, 1> Mid;
typedef Kind<64, 64, 2, 2, 1> Small;
typedef Kind<32, 32, 1, 1, 8> Slice;
typedef Kind<64, 64, 1, 1, 4> Slice64;

// Workgroup -> part of the contraction and tile: a part's rows are fetched by one XCD.
__device__ __forceinline__ void place_of(int b, int ti, int tj, int splits, int& split, int& i, int& j) {
  const int tiles = ti * tj;
  int first, len;
  run_of(tiles * splits, b % 8, first, len);
  const int u = first + b / 8;
  split = u / tiles;
  tile_at(u - split * tiles, ti, tj, i, j);
}

// A wave's outputs, from row i and column j on.  Its accumulators hold four neighbouring columns of a row in a lane;
// 16 rows at a time turn through LDS of the wave's own (16-byte piece c of row r at place c ^ r), so that a lane gets
// eight neighbouring outputs of a row and neighbouring lanes fill whole cache lines.  (Two swaps between rows of 16
// lanes give a lane its eight outputs without LDS, but neighbouring lanes then belong to different rows: 50176 x 256 x
// 128 took 21.5 us, not 13.2.)  A lane keeps its columns, so the bias is read once: a read for every 8 rows took
// 14 us more of 8192 x 4096 x 8192 with GELU and the pre-activation (460 us).
template <typename T, int FI, int FJ>
__device__ __forceinline__ void store_tile(const Epilogue& e, const f32x4 (&acc)[FI][FJ], int i, int j, int rows,
                                           int cols, int lane, char* own) {
  constexpr int PIECES = FJ * 4, MASK = PIECES < 16 ? PIECES - 1 : 15, OCTETS = FJ * 2, AT = 64 / OCTETS;
  static_assert(FJ == 2 || FJ == 4, "");
  constexpr int PASSES = AT < 16 ? 16 / AT : 1;                          // of AT rows
  const int g = lane >> 4, il = lane & 15, r = lane / OCTETS, c = lane % OCTETS * 2;
  const int n = cols - j - c * 4;
  // (fp32: erff and expf twice over and a bias in registers would spill the accumulators of the largest tile)
  constexpr bool LEAN = sizeof(T) == 4;
  constexpr int AT_ONCE = LEAN ? 1 : PASSES;
  float bias[8];
  if (!LEAN && e.bias && n > 0) bias8<T>(e, j + c * 4, n, bias);
#pragma unroll 1
  for (int x = 0; x < FI; ++x) {
#pragma unroll
    for (int u = 0; u < FI; ++u)
      if (u == x) {
#pragma unroll
        for (int y = 0; y < FJ; ++y)
          *reinterpret_cast<f32x4*>(own + (il * PIECES + ((y * 4 + g) ^ (il & MASK))) * 16) = acc[u][y];
      }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");     // other lanes of the wave read what this one wrote
#pragma unroll AT_ONCE
    for (int h = 0; h < PASSES; ++h) {
      const int lr = r + h * AT, row = i + x * 16 + lr;
      const f32x4 lo = *reinterpret_cast<const f32x4*>(own + (lr * PIECES + (c ^ (lr & MASK))) * 16);
      const f32x4 hi = *reinterpret_cast<const f32x4*>(own + (lr * PIECES + ((c + 1) ^ (lr & MASK))) * 16);
      float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      if (row < rows && n > 0) epilogue8<T>(e, row, j + c * 4, n, v, LEAN ? nullptr : bias);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}

// ACT_A, ACT_B: that operand is dP, made from dy and p.saved
template <typename T, typename K, bool FA, bool FB, int LA, int LB, bool Q8, bool ACT_A = false, bool ACT_B = false>
__device__ __forceinline__ void product_body(const Product& p, int block, char* lds) {
  constexpr int BI = K::BI, BJ = K::BJ, WI = K::WI, WJ = K::WJ, KW = K::KW;
  constexpr int BC = 128 / (int)sizeof(T);
  constexpr bool SHARED = KW == 1;
  constexpr int THREADS = WI * WJ * 64;                 // that share a stage
  using SA = Stage<T, FA, BI, BC>;
  using SB = Stage<T, FB, BJ, BC>;
  constexpr int STAGE = SA::BYTES + SB::BYTES;
  static_assert(2 * KW * STAGE == K::LDS, "");
  constexpr int FI = BI / WI / 16, FJ = BJ / WJ / 16, KS = 2;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int tid = SHARED ? threadIdx.x : lane;
  const int wi = SHARED ? wave / WJ : 0, wj = SHARED ? wave % WJ : 0;
  const int kw = SHARED ? 0 : __builtin_amdgcn_readfirstlane(wave);
  char* mine = lds + kw * 2 * STAGE;
  int split, ti, tj;
  place_of(block, (p.I + BI - 1) / BI, (p.J + BJ - 1) / BJ, p.splits, split, ti, tj);
  const int i0 = ti * BI, j0 = tj * BJ;
  const int64_t c0 = (int64_t)split * p.c_per;
  const int clen = (int)min((int64_t)p.c_per, p.C - c0);
  // steps of this wave; one at least, which finds nothing past the end
  const int steps = SHARED ? (clen + BC - 1) / BC : max(1, ((clen + BC - 1) / BC - kw + KW - 1) / KW);

  Filler<T, FA, BI, BC, THREADS, KW, LA, Q8, ACT_A> fa;
  Filler<T, FB, BJ, BC, THREADS, KW, LB, false, ACT_B> fb;
  fa.init(p.A, p.lda, i0, p.I, c0, clen, p.C, p.exps, p.lde, kw, tid);
  fb.init(p.B, p.ldb, j0, p.J, c0, clen, p.C, nullptr, 0, kw, tid);
  if constexpr (ACT_A) fa.init_saved(p.saved, p.lds, p.saved_act, i0, c0);
  if constexpr (ACT_B) fb.init_saved(p.saved, p.lds, p.saved_act, j0, c0);

  f32x4 acc[FI][FJ];
#pragma unroll
  for (int x = 0; x < FI; ++x)
#pragma unroll
    for (int y = 0; y < FJ; ++y) acc[x][y] = f32x4{0.f, 0.f, 0.f, 0.f};

  typename Frag<T>::type a[KS][FI], b[KS][FJ];
  const int ra = wi * (BI / WI), rb = wj * (BJ / WJ);
  // fragment f of a group: the FJ of B, then the FI of A
  auto read = [&](const char* st, int ks, int f) {
    if (f < FJ) b[ks][f] = fragment<T, FB, BJ, BC>(st + SA::BYTES, rb + f * 16, ks, lane);
    else a[ks][f - FJ] = fragment<T, FA, BI, BC>(st, ra + (f - FJ) * 16, ks, lane);
  };
  // Multiplies group ks row by row of A's fragments while it reads group kn of stage `rd` and, with LOAD, begins the
  // pieces of step `ua` / `ub` into `ld`.  A row's fragment is dead after its row, and the reads are spread so that
  // two more than FI are live at once; the last row reads nothing, which covers the last read's latency.
  constexpr int READS = FI + FJ, ROWS = FI > 1 ? FI - 1 : 1;
  constexpr std::true_type yes;
  constexpr std::false_type no;
  constexpr int NA = decltype(fa)::N, NB = decltype(fb)::N;
  auto group = [&](int ks, int kn, auto reads, const char* rd, auto loads, char* ld, const auto& ua, const auto& ub) {
#pragma unroll
    for (int x = 0; x < FI; ++x) {
      if constexpr (decltype(loads)::value) {
        if (x == 0) {
          fa.begin_reg(ua, tid);
          fb.begin_reg(ub, tid);
        }
#pragma unroll
        for (int q = 0; q < NA; ++q)
          if (q * FI / NA == x) fa.begin(ld, ua, q, tid);
#pragma unroll
        for (int q = 0; q < NB; ++q)
          if (q * FI / NB == x) fb.begin(ld + SA::BYTES, ub, q, tid);
      }
      if constexpr (decltype(reads)::value) {
#pragma unroll
        for (int f = 0; f < READS; ++f)
          if (f * ROWS / READS == x) read(rd, kn, f);
      }
      multiply_row<T, FJ>(b[ks], a[ks][x], acc[x]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  fa.begin_all(mine, 0, tid);
  fb.begin_all(mine + SA::BYTES, 0, tid);
  fa.end(mine, tid);
  fb.end(mine + SA::BYTES, tid);
  fa.begin_all(mine + STAGE, 1, tid);
  fb.begin_all(mine + STAGE + SA::BYTES, 1, tid);
  step_barrier<(LA == kDma ? NA : 0) + (LB == kDma ? NB : 0), SHARED>();
#pragma unroll
  for (int f = 0; f < READS; ++f) read(mine, 0, f);
  char* cur = mine;
  char* nxt = mine + STAGE;
  for (int t = 0; t + 1 < steps; ++t) {
    const auto ua = fa.at(t + 2);
    const auto ub = fb.at(t + 2);
    group(0, 1, yes, cur, no, nullptr, ua, ub);
    fa.end(nxt, tid);
    fb.end(nxt + SA::BYTES, tid);
    step_barrier<0, SHARED>();
    group(1, 0, yes, nxt, yes, cur, ua, ub);
    char* s = cur;
    cur = nxt;
    nxt = s;
  }
  {
    const auto ua = fa.at(steps);
    const auto ub = fb.at(steps);
    group(0, 1, yes, cur, no, nullptr, ua, ub);
    group(1, 0, no, nullptr, no, nullptr, ua, ub);
  }
  // loads into LDS past the last step (of zeros) end before the workgroup's LDS is given away
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

  // Epilogue
  Epilogue e = p.e;
  if (p.splits > 1) {
    e = Epilogue{};
    e.out = p.part + (int64_t)split * p.I * p.J;
    e.ldo = p.J;
    e.out_f32 = 1;
  }
  if constexpr (!SHARED) {
    __syncthreads();
    const int g = lane >> 4, il = lane & 15;
    // every wave's sums of the whole tile, then one octet of outputs a thread: the waves' parts added in order
    constexpr int PIECES = BJ / 4, MASK = PIECES < 16 ? PIECES - 1 : 15, PLANE = BI * BJ * 4;
#pragma unroll
    for (int x = 0; x < FI; ++x)
#pragma unroll
      for (int y = 0; y < FJ; ++y)
        *reinterpret_cast<f32x4*>(lds + kw * PLANE + ((x * 16 + il) * PIECES + ((y * 4 + g) ^ (il & MASK))) * 16) =
            acc[x][y];
    __syncthreads();
    for (int k = threadIdx.x; k < BI * (BJ / 8); k += K::THREADS) {
      const int r = k / (BJ / 8), c = (k % (BJ / 8)) * 2, key = r & MASK, i = i0 + r, j = j0 + c * 4;
      f32x4 lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        lo += *reinterpret_cast<const f32x4*>(lds + w * PLANE + (r * PIECES + (c ^ key)) * 16);
        hi += *reinterpret_cast<const f32x4*>(lds + w * PLANE + (r * PIECES + ((c + 1) ^ key)) * 16);
      }
      if (i < p.I && j < p.J) {
        float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        epilogue8<T>(e, i, j, p.J - j, v);
      }
    }
  } else {
    __syncthreads();                                      // the stages are free for the outputs
    store_tile<T>(e, acc, i0 + ra, j0 + rb, p.I, p.J, lane, lds + wave * K::TURN);
  }
}

// A product whose workgroups stay: each walks several tiles, and the loads run ahead across tiles, so that the next
// tile's first two steps land while this one's outputs are stored.  The first p.whole tiles of the walk are multiplied
// whole; the others, too few to fill the card once more, are split along the contraction (p.splits parts each): 3090 x
// 5256 x 7696's input gradient took 372 us with a last round of a third of the card, 227 us split.
// (Smaller tiles gain nothing from walking: Mid's took as long either way.)
template <typename T, typename K, bool FA, bool FB, int LA, int LB, bool Q8>
__device__ __forceinline__ void stream_body(const Product& p, char* lds) {
  constexpr int BI = K::BI, BJ = K::BJ, WI = K::WI, WJ = K::WJ, BC = 128 / (int)sizeof(T), THREADS = K::THREADS;
  static_assert(K::KW == 1, "");
  using SA = Stage<T, FA, BI, BC>;
  using SB = Stage<T, FB, BJ, BC>;
  constexpr int STAGE = SA::BYTES + SB::BYTES;
  constexpr int FI = BI / WI / 16, FJ = BJ / WJ / 16, KS = 2;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wi = wave / WJ, wj = wave % WJ;
  const int ti = (p.I + BI - 1) / BI, tj = (p.J + BJ - 1) / BJ, rest = ti * tj - p.whole;

  // this workgroup's work: every `stride`-th of its XCD's runs over the whole tiles and over the (part, tile) pairs
  const int x8 = blockIdx.x % 8, r8 = blockIdx.x / 8, stride = ((int)gridDim.x - x8 + 7) / 8;
  int first1, len1, first2, len2;
  run_of(p.whole, x8, first1, len1);
  run_of(rest * p.splits, x8, first2, len2);
  const int n1 = len1 > r8 ? (len1 - r8 + stride - 1) / stride : 0;
  const int count = n1 + (len2 > r8 ? (len2 - r8 + stride - 1) / stride : 0);
  if (count == 0) return;
  struct Item {
    int i0, j0, c0, clen, steps, slot;       // slot: place of its sums in p.part, or -1: a whole contraction
  };
  auto item = [&](int n) {
    Item m;
    int tile;
    if (n < n1) {
      tile = first1 + r8 + n * stride;
      m.slot = -1;
      m.c0 = 0;
      m.clen = p.C;
    } else {
      const int u = first2 + r8 + (n - n1) * stride, split = u / rest, q = u - split * rest;
      tile = p.whole + q;
      m.slot = p.splits > 1 ? q * p.splits + split : -1;
      m.c0 = split * p.c_per;
      m.clen = min(p.c_per, p.C - m.c0);
    }
    int a, b;
    tile_at(tile, ti, tj, a, b);
    m.i0 = a * BI;
    m.j0 = b * BJ;
    m.steps = (m.clen + BC - 1) / BC;
    return m;
  };

  Filler<T, FA, BI, BC, THREADS, 1, LA, Q8, false> fa;
  Filler<T, FB, BJ, BC, THREADS, 1, LB, false, false> fb;
  int at_item = 0, at_step = 0, at_steps;    // what is loaded next
  auto take = [&](int n) {
    const Item m = item(n);
    fa.init(p.A, p.lda, m.i0, p.I, m.c0, m.clen, p.C, p.exps, p.lde, 0, tid);
    fb.init(p.B, p.ldb, m.j0, p.J, m.c0, m.clen, p.C, nullptr, 0, 0, tid);
    at_steps = m.steps;
  };
  auto ahead = [&]() {
    if (++at_step < at_steps) return;
    at_step = 0;
    if (++at_item < count) {
      take(at_item);
    } else {
      fa.clen = fb.clen = 0;                 // nothing more: the steps that follow load nothing
      at_steps = 0x7fffffff;
    }
  };

  f32x4 acc[FI][FJ];
  typename Frag<T>::type a[KS][FI], b[KS][FJ];
  const int ra = wi * (BI / WI), rb = wj * (BJ / WJ);
  auto read = [&](const char* st, int ks, int f) {
    if (f < FJ) b[ks][f] = fragment<T, FB, BJ, BC>(st + SA::BYTES, rb + f * 16, ks, lane);
    else a[ks][f - FJ] = fragment<T, FA, BI, BC>(st, ra + (f - FJ) * 16, ks, lane);
  };
  // as in product_body: group ks multiplied row by row while group kn of `rd` is read and a step's pieces are begun
  constexpr int READS = FI + FJ, ROWS = FI > 1 ? FI - 1 : 1;
  constexpr std::true_type yes;
  constexpr std::false_type no;
  constexpr int NA = decltype(fa)::N, NB = decltype(fb)::N;
  auto group = [&](int ks, int kn, const char* rd, auto loads, char* ld, const auto& ua, const auto& ub) {
#pragma unroll
    for (int x = 0; x < FI; ++x) {
      if constexpr (decltype(loads)::value) {
        if (x == 0) {
          fa.begin_reg(ua, tid);
          fb.begin_reg(ub, tid);
        }
#pragma unroll
        for (int q = 0; q < NA; ++q)
          if (q * FI / NA == x) fa.begin(ld, ua, q, tid);
#pragma unroll
        for (int q = 0; q < NB; ++q)
          if (q * FI / NB == x) fb.begin(ld + SA::BYTES, ub, q, tid);
      }
#pragma unroll
      for (int f = 0; f < READS; ++f)
        if (f * ROWS / READS == x) read(rd, kn, f);
      multiply_row<T, FJ>(b[ks], a[ks][x], acc[x]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  take(0);
  fa.begin_all(lds, 0, tid);
  fb.begin_all(lds + SA::BYTES, 0, tid);
  ahead();
  fa.end(lds, tid);
  fb.end(lds + SA::BYTES, tid);
  fa.begin_all(lds + STAGE, at_step, tid);
  fb.begin_all(lds + STAGE + SA::BYTES, at_step, tid);
  ahead();
  step_barrier<(LA == kDma ? NA : 0) + (LB == kDma ? NB : 0), true>();
#pragma unroll
  for (int f = 0; f < READS; ++f) read(lds, 0, f);
  char* cur = lds;
  char* nxt = lds + STAGE;
  bool inside = false;                       // the last tile's outputs of this wave all exist
  for (int n = 0; n < count; ++n) {
    const Item m = item(n);
#pragma unroll
    for (int x = 0; x < FI; ++x)
#pragma unroll
      for (int y = 0; y < FJ; ++y) acc[x][y] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int t = 0; t < m.steps; ++t) {
      const auto ua = fa.at(at_step);
      const auto ub = fb.at(at_step);
      group(0, 1, cur, no, nullptr, ua, ub);
      fa.end(nxt, tid);
      fb.end(nxt + SA::BYTES, tid);
      // a tile's first step: the loads it waits for are older than the last tile's stores, of which there were FI FJ/2
      // at least where the wave's outputs all exist: as many newer accesses may still be on their way
      if (t == 0 && inside) step_barrier<FI * FJ / 2, true>();
      else step_barrier<0, true>();
      group(1, 0, nxt, yes, cur, ua, ub);
      ahead();
      char* s = cur;
      cur = nxt;
      nxt = s;
    }

    Epilogue e = p.e;
    int rows = p.I, cols = p.J, i1 = m.i0 + ra, j1 = m.j0 + rb;
    if (m.slot >= 0) {
      e = Epilogue{};
      e.out = p.part + (int64_t)m.slot * (BI * BJ);
      e.ldo = BJ;
      e.out_f32 = 1;
      rows = BI;
      cols = BJ;
      i1 = ra;
      j1 = rb;
    }
    store_tile<T>(e, acc, i1, j1, rows, cols, lane, lds + K::LDS + wave * K::TURN);
    inside = i1 + FI * 16 <= rows && j1 + FJ * 16 <= cols;
  }
  // the loads of nothing behind the last step end before the workgroup's LDS is given away
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

template <typename T, typename K, bool FA, bool FB, int LA, int LB, bool Q8>
__global__ __launch_bounds__(K::THREADS) void product_kernel(Product p) {
  extern __shared__ char lds[];
  if constexpr (K::STREAM) stream_body<T, K, FA, FB, LA, LB, Q8>(p, lds);
  else product_body<T, K, FA, FB, LA, LB, Q8>(p, blockIdx.x, lds);
}

// The backward pass's two products and the join of its column sums as one launch: the product whose workgroups take
// longer starts first (what starts last should end soon), the last workgroups join 16 columns each.  For products that
// do not fill the card: 512 x 2048 x 512 in 11.4 us, 17.7 us as launches of their own.
template <typename T, typename K, int LX, int LK, bool Q8>
__global__ __launch_bounds__(K::THREADS) void pair_kernel(Pair p) {
  extern __shared__ char lds[];
  const int b = blockIdx.x, bx = b - p.x0, bk = b - p.k0;
  if (bk >= 0 && bk < p.nk) {
    product_body<T, K, true, true, Q8 ? kReg : LK, LK, Q8>(p.k, bk, lds);
  } else if (bx >= 0 && bx < p.nx) {
    product_body<T, K, false, false, LX, LX, false>(p.x, bx, lds);
  } else {
    join_columns16(p.cols, b - p.nx - p.nk, threadIdx.x, reinterpret_cast<float*>(lds));
  }
}

// The same from dy and saved: dP is formed while it is staged, the other workgroups sum 8 columns each.  One launch
// for a small backward pass, for which the host takes longer than the device (1568 x 128 x 64 bf16: 10.3 us and 13 us a
// call, 10.6 us and 17 us as two launches); every tile that reads dP forms it again, so it is taken for at most 2^18
// values of dP.
template <typename T, typename K, bool Q8>
__global__ __launch_bounds__(K::THREADS) void fused_kernel(Pair p) {
  extern __shared__ char lds[];
  const int b = blockIdx.x, bx = b - p.x0, bk = b - p.k0;
  if (bk >= 0 && bk < p.nk) product_body<T, K, true, true, kReg, kReg, Q8, false, true>(p.k, bk, lds);
  else if (bx >= 0 && bx < p.nx) product_body<T, K, false, false, kReg, kReg, false, true, false>(p.x, bx, lds);
  else sum_columns8<T, K::THREADS>(p.sums, b - p.nx - p.nk, threadIdx.x, reinterpret_cast<float*>(lds));
}

// Marks a kernel's use of more LDS than the default, once per device.
inline hipError_t allow_lds(const void* k, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  if (hipError_t e = hipGetDevice(&dev)) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_acquire) & bit) return hipSuccess;
  if (hipError_t e = hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, bytes)) return e;
  done.fetch_or(bit, std::memory_order_release);
  return hipSuccess;
}

inline int64_t tiles_of(const Product& p, int bi, int bj) {
  return (int64_t)((p.I + bi - 1) / bi) * ((p.J + bj - 1) / bj);
}

template <typename T, typename K, bool FA, bool FB, int LA, int LB, bool Q8>
hipError_t launch(const Product& p, hipStream_t s) {
  static std::atomic<uint64_t> done{0};
  auto k = product_kernel<T, K, FA, FB, LA, LB, Q8>;
  constexpr int LDS = K::LAUNCH_LDS;
  if (hipError_t e = allow_lds(reinterpret_cast<const void*>(k), LDS, done)) return e;
  const int64_t tiles = tiles_of(p, K::BI, K::BJ);
  // workgroups that stay: as many as the card holds at once (256 compute units, 160 KB of LDS each)
  const int64_t groups = K::STREAM ? std::min<int64_t>(p.whole + (tiles - p.whole) * p.splits, 256 * (163840 / LDS))
                                    : tiles * p.splits;
  return launch_kernel(k, dim3((unsigned)groups), dim3(K::THREADS), LDS, s, p);
}

// (a pair's kernel may have one product only: the other's workgroups are none)
inline void place_pair(Pair& p, int64_t nx, int64_t nk) {
  const bool x_first = p.x.c_per > p.k.c_per;
  p.nx = (int)nx;
  p.nk = (int)nk;
  p.x0 = x_first ? 0 : p.nk;
  p.k0 = x_first ? p.nx : 0;
}

template <typename T, typename K, int LX, int LK, bool Q8>
hipError_t launch_pair(Pair p, hipStream_t s) {
  static std::atomic<uint64_t> done{0};
  auto k = pair_kernel<T, K, LX, LK, Q8>;
  if (hipError_t e = allow_lds(reinterpret_cast<const void*>(k), K::LDS, done)) return e;
  place_pair(p, tiles_of(p.x, K::BI, K::BJ) * p.x.splits, tiles_of(p.k, K::BI, K::BJ) * p.k.splits);
  return launch_kernel(k, dim3((unsigned)(p.nx + p.nk + (p.cols.N + 15) / 16)), dim3(K::THREADS), K::LDS, s, p);
}

template <typename T, typename K, bool Q8>
hipError_t launch_fused(Pair p, hipStream_t s) {
  static std::atomic<uint64_t> done{0};
  auto k = fused_kernel<T, K, Q8>;
  if (hipError_t e = allow_lds(reinterpret_cast<const void*>(k), K::LDS, done)) return e;
  place_pair(p, p.x.e.out ? tiles_of(p.x, K::BI, K::BJ) * p.x.splits : 0,
             p.k.e.out ? tiles_of(p.k, K::BI, K::BJ) * p.k.splits : 0);
  return launch_kernel(k, dim3((unsigned)(p.nx + p.nk + (p.sums.N + 7) / 8)), dim3(K::THREADS), K::LDS, s, p);
}

template <typename T, typename K>
hipError_t product_kind(const Product& p, int layout, int loader, int q8, hipStream_t s) {
  if constexpr (K::BI == 256) {      // the plan takes the largest tile only where DMA stages both operands
    if (loader != kDma) return hipErrorInvalidValue;
    if (layout == kForward) return launch<T, K, false, true, kDma, kDma, false>(p, s);
    if (layout == kInputGrad) return launch<T, K, false, false, kDma, kDma, false>(p, s);
    return q8 ? hipErrorInvalidValue : launch<T, K, true, true, kDma, kDma, false>(p, s);
  } else {
    if (layout == kForward)
      return loader == kDma ? launch<T, K, false, true, kDma, kDma, false>(p, s)
                            : launch<T, K, false, true, kReg, kReg, false>(p, s);
    if (layout == kInputGrad)
      return loader == kDma ? launch<T, K, false, false, kDma, kDma, false>(p, s)
                            : launch<T, K, false, false, kReg, kReg, false>(p, s);
    if (q8)
      return loader == kDma ? launch<T, K, true, true, kReg, kDma, true>(p, s)
                            : launch<T, K, true, true, kReg, kReg, true>(p, s);
    return loader == kDma ? launch<T, K, true, true, kDma, kDma, false>(p, s)
                          : launch<T, K, true, true, kReg, kReg, false>(p, s);
  }
}

template <typename T>
hipError_t product(const Product& p, int layout, int loader, int tile, int q8, hipStream_t s) {
  if (tile == kLarge) return product_kind<T, Large>(p, layout, loader, q8, s);
  if (tile == kMid) return product_kind<T, Mid>(p, layout, loader, q8, s);
  if (tile == kSmall) return product_kind<T, Small>(p, layout, loader, q8, s);
  if (tile == kSlice) return product_kind<T, Slice>(p, layout, loader, q8, s);
  return product_kind<T, Slice64>(p, layout, loader, q8, s);
}

template <typename T, typename K>
hipError_t pair_kind(const Pair& p, int lx, int lk, int q8, hipStream_t s) {
  if (q8) {
    if (lx == kDma && lk == kDma) return launch_pair<T, K, kDma, kDma, true>(p, s);
    if (lx != kDma && lk != kDma) return launch_pair<T, K, kReg, kReg, true>(p, s);
    return lx == kDma ? launch_pair<T, K, kDma, kReg, true>(p, s) : launch_pair<T, K, kReg, kDma, true>(p, s);
  }
  if (lx == kDma && lk == kDma) return launch_pair<T, K, kDma, kDma, false>(p, s);
  if (lx != kDma && lk != kDma) return launch_pair<T, K, kReg, kReg, false>(p, s);
  return lx == kDma ? launch_pair<T, K, kDma, kReg, false>(p, s) : launch_pair<T, K, kReg, kDma, false>(p, s);
}

template <typename T>
hipError_t pair(const Pair& p, int lx, int lk, int tile, int q8, hipStream_t s) {
  return tile == kSmall    ? pair_kind<T, Small>(p, lx, lk, q8, s)
         : tile == kSlice ? pair_kind<T, Slice>(p, lx, lk, q8, s)
                          : pair_kind<T, Slice64>(p, lx, lk, q8, s);
}

template <typename T>
hipError_t fused(const Pair& p, int tile, int q8, hipStream_t s) {
  if (tile == kSmall) return q8 ? launch_fused<T, Small, true>(p, s) : launch_fused<T, Small, false>(p, s);
  return q8 ? launch_fused<T, Slice, true>(p, s) : launch_fused<T, Slice, false>(p, s);
}

}  // namespace petdense_k
