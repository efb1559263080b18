// Internal declarations of the dense layer's operators (dense_*.hip <-> dense_api.cpp, include/petdense.h).
#pragma once
#include <hip/hip_runtime.h>
#include <cstddef>
#include <cstdint>

namespace petdense_k {

enum Type { kF32 = 0, kBF16 = 1, kF16 = 2 };
enum Act { kNone = 0, kRelu = 1, kGelu = 2, kSilu = 3 };

// What a product's accumulators go through: v + bias[j] + res[i][j], stored as `pre` if asked, then the activation.
struct Epilogue {
  const void* bias;      // [J] or null
  const void* res;       // [I][J] (row stride ldr) in the operands' type, or null
  void* out;             // [I][J] (row stride ldo)
  void* pre;             // [I][J] (row stride ldp) or null
  int64_t ldr, ldo, ldp;
  int act;
  int bias_f32, out_f32; // these are fp32 (else: the operands' type); `pre` has out's type
};

// C[i][j] = sum over c of A(i, c) B(c, j).  A is stored [I][C] or, with free-contiguous operands, [C][I];
// B likewise [J][C] or [C][J].
struct Product {
  const void* A;
  const void* B;
  int64_t lda, ldb;
  const uint8_t* exps;   // A held in 8 bits: exponent bytes [C][I / 32] (row stride lde)
  int64_t lde;
  // the operand dP = dy act'(saved), formed while it is staged: `saved` beside A (input gradient) or B (kernel
  // gradient), row stride lds
  const void* saved;
  int64_t lds;
  int saved_act;
  int I, J, C;
  int splits, c_per;     // contraction split into `splits` parts of c_per (a multiple of the k-step)
  float* part;           // their sums in fp32 when splits > 1 (the join has the epilogue then): [splits][I][J],
                         // or of a streamed product [tile - whole][splits][tile rows][tile columns]
  int whole;             // streamed products: the first tiles of the walk, a whole contraction each
  Epilogue e;
};

// Rows of a tile are reached by 32-bit offsets from its first: 256 rows at most, each shorter than this.
constexpr int64_t kMaxRowBytes = 0x7fffffff / 256;

// Whether exponent bytes, `lde` from row to row, are reached by 32-bit offsets from a step's first.
__host__ __device__ inline bool exponents_fit(int64_t lde) { return lde < kMaxRowBytes; }

// Offset of the exponent byte of block `block` in a step's row r.
__host__ __device__ inline unsigned exponent_offset(int r, int64_t lde, int block) {
  return (unsigned)(r * (int)lde + block);
}

enum Layout { kForward = 0, kInputGrad = 1, kKernelGrad = 2 };   // (A, B): (c-, j-), (c-, c-), (i-, j-contiguous)
enum Loader { kDma = 0, kReg = 1 };
enum Tile { kLarge = 0, kMid = 1, kSmall = 2, kSlice = 3, kSlice64 = 4 };

// out[n] = sum over chunks of part[chunk][n], in order
struct ColumnJoin {
  const float* part;
  void* out;
  int chunks, N;         // N = 0: nothing to join
  int out_type;
};

// out[n] = sum over rows of dy act'(saved), straight from the inputs
struct ColumnSum {
  const void* dy;
  const void* saved;
  void* out;
  int64_t ldy, lds;
  int M, N, act;         // N = 0: no sums wanted
  int out_type;
};

// The backward pass's products and its bias gradient as one launch (kSmall, kSlice, kSlice64).
struct Pair {
  Product x, k;
  ColumnJoin cols;       // pair: the sums' parts are there (act_grad)
  ColumnSum sums;        // fused: they are made here
  int nx, nk, x0, k0;    // workgroups of each, and the first of them (the launcher's)
};

// One launch of the tiled product: `q8`: A is e4m3 codes with exponent bytes (kKernelGrad only).
hipError_t product_f32(const Product& p, int layout, int loader, int tile, int q8, hipStream_t s);
hipError_t product_bf16(const Product& p, int layout, int loader, int tile, int q8, hipStream_t s);
hipError_t product_f16(const Product& p, int layout, int loader, int tile, int q8, hipStream_t s);

hipError_t pair_f32(const Pair& p, int lx, int lk, int tile, int q8, hipStream_t s);
hipError_t pair_bf16(const Pair& p, int lx, int lk, int tile, int q8, hipStream_t s);
hipError_t pair_f16(const Pair& p, int lx, int lk, int tile, int q8, hipStream_t s);
// The whole backward pass as one launch: dP is formed while the products stage it (all operands through registers).
hipError_t fused_f32(const Pair& p, int tile, int q8, hipStream_t s);
hipError_t fused_bf16(const Pair& p, int tile, int q8, hipStream_t s);
hipError_t fused_f16(const Pair& p, int tile, int q8, hipStream_t s);

// Joins split products: the sum of p.part over the splits, in order, through the epilogue; and column sums (N > 0).
hipError_t join(const Product& p, const ColumnJoin& cols, int type, hipStream_t s);
// The same for the split tiles of a streamed product with b x b tiles.
hipError_t join_tiles(const Product& p, const ColumnJoin& cols, int type, int b, hipStream_t s);

// Tile number t of the walk over ti x tj tiles: bands of 4 tile rows, column by column, so that workgroups that run
// together share rows of A and columns of B.
__host__ __device__ inline void tile_at(int t, int ti, int tj, int& i, int& j) {
  constexpr int BAND = 4;
  const int band = t / (BAND * tj), first = band * BAND, h = ti - first < BAND ? ti - first : BAND, r = t - first * tj;
  i = first + r % h;
  j = r / h;
}

// One or two rows: one pass over B ([C][J], j-contiguous), I <= kMaxRows.
constexpr int kMaxRows = 2, kRowThreads = 1024, kRowCols = 32;
hipError_t rows(const Product& p, int type, hipStream_t s);

// lanes that share a row of N columns in act_grad: a power of two
inline int act_grad_lanes(int N) {
  int l = 1;
  while (l < 64 && l * 8 < N) l *= 2;
  return l;
}

// Copies whose rows start and end on 16 bytes, zeros behind their values: DMA stages them whatever the source's
// alignment.  Up to three matrices a launch.
struct PadJob {
  const void* src;
  void* dst;
  int64_t ld, ldd;       // ldd: values of a row with its zeros, a multiple of 16 bytes
  int rows, n;           // rows = 0: no job
};
struct PadJobs {
  PadJob job[3];
};
hipError_t pad(const PadJobs& p, int type, hipStream_t s);

// dp = dy act'(saved) (dp may be null, its rows hold zeros up to a multiple of 8 columns, unless `bare`),
// part[chunk][n] = column sums of dp over the chunk's rows (may be null)
hipError_t act_grad(const void* dy, int64_t ldy, const void* saved, int64_t lds, void* dp, int64_t ldd, int bare,
                    float* part, int chunks, int M, int N, int type, int act, hipStream_t s);
hipError_t join_columns(const ColumnJoin& c, hipStream_t s);

// rows x n values of `size` bytes (row stride ld) become zero; a kernel, so that a graph can hold it
hipError_t fill_zero(void* p, int64_t rows, int n, int64_t ld, int size, hipStream_t s);

hipError_t quantize(const void* x, int64_t ldx, int64_t M, int K, int type, uint8_t* codes, int64_t ldc, uint8_t* exps,
                    int64_t lde, hipStream_t s);
hipError_t restore(const uint8_t* codes, int64_t ldc, const uint8_t* exps, int64_t lde, int64_t M, int K, int type,
                   void* x, int64_t ldx, hipStream_t s);

}  // namespace petdense_k
