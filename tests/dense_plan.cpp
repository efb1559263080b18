// The dense layer's plan on the CPU: its C entries (dense_api.cpp, which the test compiles beside this file) over
// launchers that write down what they are asked for, one line a launch, and launch nothing.
#include "dense_internal.h"

#include <cstdio>
#include <string>

namespace {
std::string g_log;

template <typename... A>
hipError_t note(const char* format, A... a) {
  char line[512];
  std::snprintf(line, sizeof line, format, a...);
  g_log += line;
  g_log += '\n';
  return hipSuccess;
}
long long L(int64_t v) { return v; }
}  // namespace

namespace petdense_k {

static hipError_t product(const Product& p, int type, int layout, int loader, int tile, int q8, const char* kind) {
  return note("%s type=%d layout=%d loader=%d tile=%d q8=%d lda=%lld ldb=%lld lde=%lld I=%d J=%d C=%d splits=%d "
              "c_per=%d whole=%d", kind, type, layout, loader, tile, q8, L(p.lda), L(p.ldb), L(p.lde), p.I, p.J, p.C,
              p.splits, p.c_per, p.whole);
}
hipError_t product_f32(const Product& p, int layout, int loader, int tile, int q8, hipStream_t) {
  return product(p, kF32, layout, loader, tile, q8, "product");
}
hipError_t product_bf16(const Product& p, int layout, int loader, int tile, int q8, hipStream_t) {
  return product(p, kBF16, layout, loader, tile, q8, "product");
}
hipError_t product_f16(const Product& p, int layout, int loader, int tile, int q8, hipStream_t) {
  return product(p, kF16, layout, loader, tile, q8, "product");
}

static hipError_t pair(const Pair& p, int type, int lx, int lk, int tile, int q8) {
  (void)product(p.x, type, kInputGrad, lx, tile, 0, "pair");
  (void)product(p.k, type, kKernelGrad, lk, tile, q8, "pair");
  return note("pair_columns N=%d", p.cols.N);
}
hipError_t pair_f32(const Pair& p, int lx, int lk, int tile, int q8, hipStream_t) {
  return pair(p, kF32, lx, lk, tile, q8);
}
hipError_t pair_bf16(const Pair& p, int lx, int lk, int tile, int q8, hipStream_t) {
  return pair(p, kBF16, lx, lk, tile, q8);
}
hipError_t pair_f16(const Pair& p, int lx, int lk, int tile, int q8, hipStream_t) {
  return pair(p, kF16, lx, lk, tile, q8);
}
hipError_t fused_f32(const Pair&, int tile, int q8, hipStream_t) { return note("fused tile=%d q8=%d", tile, q8); }
hipError_t fused_bf16(const Pair&, int tile, int q8, hipStream_t) { return note("fused tile=%d q8=%d", tile, q8); }
hipError_t fused_f16(const Pair&, int tile, int q8, hipStream_t) { return note("fused tile=%d q8=%d", tile, q8); }

hipError_t join(const Product& p, const ColumnJoin& c, int, hipStream_t) {
  return note("join I=%d J=%d splits=%d N=%d", p.I, p.J, p.splits, c.N);
}
hipError_t join_tiles(const Product& p, const ColumnJoin& c, int, int b, hipStream_t) {
  return note("join_tiles I=%d J=%d splits=%d whole=%d b=%d N=%d", p.I, p.J, p.splits, p.whole, b, c.N);
}
hipError_t join_columns(const ColumnJoin& c, hipStream_t) { return note("join_columns N=%d", c.N); }
hipError_t rows(const Product& p, int, hipStream_t) { return note("rows I=%d J=%d splits=%d", p.I, p.J, p.splits); }
hipError_t pad(const PadJobs& p, int type, hipStream_t) {
  for (const PadJob& j : p.job)
    if (j.rows) (void)note("pad type=%d rows=%d n=%d ldd=%lld", type, j.rows, j.n, L(j.ldd));
  return hipSuccess;
}
hipError_t act_grad(const void*, int64_t, const void*, int64_t, void* dp, int64_t ldd, int, float* part, int chunks,
                    int M, int N, int, int act, hipStream_t) {
  return note("act_grad M=%d N=%d dp=%d ldd=%lld part=%d chunks=%d act=%d", M, N, dp != nullptr, L(ldd),
              part != nullptr, chunks, act);
}
hipError_t fill_zero(void*, int64_t rows, int n, int64_t, int, hipStream_t) {
  return note("fill_zero rows=%lld n=%d", L(rows), n);
}
hipError_t quantize(const void*, int64_t, int64_t M, int K, int, uint8_t*, int64_t, uint8_t*, int64_t, hipStream_t) {
  return note("quantize M=%lld K=%d", L(M), K);
}
hipError_t restore(const uint8_t*, int64_t, const uint8_t*, int64_t, int64_t M, int K, int, void*, int64_t ldx,
                   hipStream_t) {
  return note("restore M=%lld K=%d ldx=%lld", L(M), K, L(ldx));
}

}  // namespace petdense_k

extern "C" {
const char* plan_log() { return g_log.c_str(); }
void plan_clear() { g_log.clear(); }
int plan_exponents_fit(int64_t lde) { return petdense_k::exponents_fit(lde); }
uint64_t plan_exponent_offset(int r, int64_t lde, int block) { return petdense_k::exponent_offset(r, lde, block); }
}
