// C-ABI implementation of the training step (include/pettrain.h), SURVEY.md 8(f) row 4.
//
// ImprovedDDPM.train_step (diffusion_model.py:533-598) on one GPU, fp32:
//   q-sample -> U-Net forward (im2col + rocBLAS GEMM per conv, activations kept)
//   -> loss + analytic output gradient -> backward through every layer
//   (weight grads A^T dY, data grads dY W^T + col2im) -> per-variable clip + Adam.
// With pettrain_set_precision(PETTRAIN_BF16) the convolutions and the condition encoder
// run on the dense layer's operators (petdense.h) instead, the inputs of their products
// held in bf16 or in 8 bits.
// The layer walk mirrors UnetConditional.call (networks.py:994-1093) at the
// shipped config; the CPU restatement of every gradient is oracle/train_ref.py.
#include "pettrain.h"
#include "petdense.h"
#include "petdiff_internal.h"
#include "petdiff_spec.h"
#include "train_internal.h"

#include <rocblas/rocblas.h>

#include <cmath>
#include <cstring>
#include <map>
#include <memory>
#include <string>
#include <vector>

using namespace petdiff;
namespace K = pettrain_k;

namespace {

thread_local std::string g_err;

int fail(int code, const std::string& msg) {
  g_err = msg;
  return code;
}

#define HIPC(expr)                                                                        \
  do {                                                                                    \
    hipError_t e_ = (expr);                                                               \
    if (e_ != hipSuccess)                                                                 \
      return fail(PETDIFF_ERR_HIP, std::string(#expr) + ": " + hipGetErrorString(e_));    \
  } while (0)

#define RBC(expr)                                                                                   \
  do {                                                                                              \
    rocblas_status s_ = (expr);                                                                     \
    if (s_ != rocblas_status_success)                                                               \
      return fail(PETDIFF_ERR_HIP, std::string(#expr) + ": " + rocblas_status_to_string(s_));      \
  } while (0)

#define CHK(expr)                    \
  do {                               \
    int r_ = (expr);                 \
    if (r_ != PETDIFF_OK) return r_; \
  } while (0)

struct Buf {
  void* p = nullptr;
  size_t bytes = 0;
  ~Buf() { if (p) (void)hipFree(p); }
  hipError_t alloc(size_t b) {
    if (b <= bytes && p) return hipSuccess;
    if (p) (void)hipFree(p);
    p = nullptr;
    bytes = 0;
    hipError_t e = hipMalloc(&p, b ? b : 16);
    if (e == hipSuccess) bytes = b;
    return e;
  }
  float* f() const { return reinterpret_cast<float*>(p); }
  int* i() const { return reinterpret_cast<int*>(p); }
  __bf16* h() const { return reinterpret_cast<__bf16*>(p); }
  uint8_t* u8() const { return reinterpret_cast<uint8_t*>(p); }
  void release() {
    if (p) (void)hipFree(p);
    p = nullptr;
    bytes = 0;
  }
};

// The input of a product that its backward pass reads again: bf16 rows, or their 8-bit checkpoint.
struct Kept {
  Buf rows, exps;
};

// a row of n values in bf16, padded so that rows start and end on 16 bytes
inline int pad8(int n) { return (n + 7) / 8 * 8; }

// Shipped-config geometry
constexpr int kDownL[4] = {48, 24, 12, 6};
constexpr int kDownCin[4] = {2, 128, 256, 512};
constexpr int kDownCout[4] = {128, 256, 512, 1024};
constexpr int kUpLc[3] = {6, 12, 24};          // coarse length (label/time length)
constexpr int kUpCin[3] = {1024, 512, 256};
constexpr int kUpCout[3] = {512, 256, 128};
constexpr int kLevelL[7] = {48, 24, 12, 6, 6, 12, 24};   // label/time length of cond level p

K::ConvIn down_in(int d) { return K::ConvIn{1, kDownCin[d], 0, kDownL[d], 0, 6, 2}; }
K::ConvIn upconv_in(int u) { return K::ConvIn{1, kUpCin[u], 0, kUpLc[u], 1, 2, 0}; }
K::ConvIn block_in(int u) { return K::ConvIn{0, kUpCout[u], kUpCout[u], 2 * kUpLc[u], 0, 6, 2}; }

}  // namespace

struct pettrain_ctx {
  petdiff_config cfg;
  pettrain_config opt;
  int device = 0, n_out = 4, T = 0, learn_mode = 2, param_mode = 0;
  std::vector<Spec> spec;
  std::map<std::string, size_t> off;
  size_t n_w = 0;
  Buf w, g, m, v, tab;
  Buf cvar, cstart, clen, vfirst, vcount, partial, vscale;
  int n_chunks = 0, n_vars = 0;
  Buf weff[7];                     // folded ConvBlock kernels: down0..3, up0..2 blocks
  rocblas_handle rb = nullptr;
  int B_cap = 0;
  // forward
  Buf t, noise, xt, emb, a_t, h_t, cond_aug, e1, e2, e3, z, lab[7], tim[7];
  Buf A_dn[4], out_dn[4], pool[3], A_uc[3], hu[3], A_bk[3], out_up[3], y4;
  // backward
  Buf dy4, dA, dpre, d_out_up[3], d_out_dn3, d_pool[3], dskip[3], dhu, dlab, dtim, dz, dh_t, da_t, de1, de2, de3,
      sse, vlb, dbias_part, stats;
  // bf16 step: convolutions 0-3 down, 4-6 up, 7-9 up blocks; encoder layers 0-3
  int precision = PETTRAIN_F32, keep = PETTRAIN_KEEP;
  Buf w16[10], b16[10], we16[4], a16, da16, dp16, gk16, work16;
  Kept in16[10], en16[4];
  Buf e16[4], de16[4];          // inputs of the encoder's layers, and the gradients of its outputs
  int64_t iter = 0;
  int last_B = 0;          // batch of the last backward pass (gradients valid)
  bool has_stats = false;  // a forward + loss ran (pettrain_last_stats valid)

  float* W(const std::string& n) const { return w.f() + off.at(n); }
  float* G(const std::string& n) const { return g.f() + off.at(n); }
};

namespace {

// Row-major C[M,N] = op(A)[M,K] op(B)[K,N] (+ beta C) on the handle's rocBLAS stream.
int gemm(pettrain_ctx* h, bool ta, bool tb, int M, int N, int Kd, const float* A, int lda, const float* B, int ldb,
         float* C, int ldc, float beta) {
  const float one = 1.0f;
  RBC(rocblas_sgemm(h->rb, tb ? rocblas_operation_transpose : rocblas_operation_none,
                    ta ? rocblas_operation_transpose : rocblas_operation_none, N, M, Kd, &one, B, ldb, A, lda, &beta,
                    C, ldc));
  return PETDIFF_OK;
}

// Augmented activations: every tensor that feeds a Dense layer or a conv GEMM carries a
// trailing column of ones (row stride K + 1), and the weight operand is the blob's
// [kernel ; bias] block (adjacent in the blob), so the GEMM adds the bias and the
// weight-gradient GEMM returns [d kernel ; d bias] in one pass.
int ensure16(pettrain_ctx* h, int B);

int ensure(pettrain_ctx* h, int B) {
  if (B <= h->B_cap) return PETDIFF_OK;
  const size_t Bz = (size_t)B, F = 4, R = Bz * 49;
  const bool f32 = h->precision == PETTRAIN_F32;
  HIPC(h->t.alloc(Bz * 4));
  HIPC(h->noise.alloc(Bz * 96 * F));
  HIPC(h->xt.alloc(Bz * 96 * F));
  HIPC(h->emb.alloc(Bz * 65 * F));
  HIPC(h->a_t.alloc(Bz * 48 * F));
  HIPC(h->h_t.alloc(Bz * 49 * F));
  if (f32) {
    HIPC(h->cond_aug.alloc(R * 55 * F));
    HIPC(h->e1.alloc(R * 257 * F));
    HIPC(h->e2.alloc(R * 129 * F));
    HIPC(h->e3.alloc(R * 65 * F));
    HIPC(h->de1.alloc(R * 256 * F));
    HIPC(h->de2.alloc(R * 128 * F));
    HIPC(h->de3.alloc(R * 64 * F));
  }
  HIPC(h->z.alloc(R * 33 * F));
  for (int p = 0; p < 7; ++p) {
    HIPC(h->lab[p].alloc(R * kLevelL[p] * F));
    HIPC(h->tim[p].alloc(Bz * kLevelL[p] * F));
  }
  size_t maxA = 0;
  for (int d = 0; d < 4; ++d) {
    const K::ConvIn ci = down_in(d);
    const size_t k = (size_t)ci.taps * ci.cfull();
    maxA = std::max(maxA, Bz * ci.lout() * k);
    if (f32) HIPC(h->A_dn[d].alloc(Bz * ci.lout() * (k + 1) * F));
    HIPC(h->out_dn[d].alloc(Bz * kDownL[d] * kDownCout[d] * F));
    if (d < 3) {
      HIPC(h->pool[d].alloc(Bz * (kDownL[d] / 2) * kDownCout[d] * F));
      HIPC(h->d_pool[d].alloc(Bz * (kDownL[d] / 2) * kDownCout[d] * F));
      HIPC(h->dskip[d].alloc(Bz * kDownL[d] * kDownCout[d] * F));
    }
  }
  for (int u = 0; u < 3; ++u) {
    const K::ConvIn uc = upconv_in(u), bk = block_in(u);
    const size_t k1 = (size_t)uc.taps * uc.cfull(), k2 = (size_t)bk.taps * bk.cfull();
    maxA = std::max(maxA, std::max(Bz * uc.lout() * k1, Bz * bk.lout() * k2));
    if (f32) HIPC(h->A_uc[u].alloc(Bz * uc.lout() * (k1 + 1) * F));
    if (f32) HIPC(h->A_bk[u].alloc(Bz * bk.lout() * (k2 + 1) * F));
    HIPC(h->hu[u].alloc(Bz * 2 * kUpLc[u] * kUpCout[u] * F));
    HIPC(h->out_up[u].alloc(Bz * 2 * kUpLc[u] * kUpCout[u] * F));
    HIPC(h->d_out_up[u].alloc(Bz * 2 * kUpLc[u] * kUpCout[u] * F));
  }
  HIPC(h->y4.alloc(Bz * 48 * h->n_out * F));
  HIPC(h->dy4.alloc(Bz * 48 * h->n_out * F));
  if (f32) HIPC(h->dA.alloc(maxA * F));
  if (f32) HIPC(h->dpre.alloc(Bz * 6144 * F));
  if (!f32) CHK(ensure16(h, B));
  HIPC(h->d_out_dn3.alloc(Bz * 6 * 1024 * F));
  HIPC(h->dhu.alloc(Bz * 6144 * F));
  HIPC(h->dlab.alloc(R * 48 * F));
  HIPC(h->dtim.alloc(Bz * 48 * F));
  HIPC(h->dz.alloc(R * 32 * F));
  HIPC(h->dh_t.alloc(Bz * 48 * F));
  HIPC(h->da_t.alloc(Bz * 48 * F));
  HIPC(h->sse.alloc(Bz * F));
  HIPC(h->vlb.alloc(Bz * F));
  HIPC(h->dbias_part.alloc(Bz * h->n_out * F));
  HIPC(h->stats.alloc(3 * sizeof(double)));
  // the ones columns (never overwritten: GEMMs write N of the N + 1 columns)
  struct { Buf* b; size_t rows; int ld; } aug[] = {{&h->emb, Bz, 65}, {&h->h_t, Bz, 49}, {&h->cond_aug, R, 55},
                                                   {&h->e1, R, 257}, {&h->e2, R, 129}, {&h->e3, R, 65},
                                                   {&h->z, R, 33}};
  for (auto& a : aug)
    if (a.b->p) HIPC(K::fill_strided(a.b->f() + (a.ld - 1), a.rows, a.ld, 1.0f, 0));
  HIPC(hipDeviceSynchronize());
  h->B_cap = B;
  return PETDIFF_OK;
}

// ---------------------------------------------------------------- bf16 step
K::ConvIn conv_in(int c) { return c < 4 ? down_in(c) : c < 7 ? upconv_in(c - 4) : block_in(c - 7); }
int conv_out(int c) { return c < 4 ? kDownCout[c] : kUpCout[(c - 4) % 3]; }
constexpr int kEncIn[4] = {54, 256, 128, 64}, kEncOut[4] = {256, 128, 64, 32};
const char* const kEncName[4] = {"cond_enc.hidden0", "cond_enc.hidden1", "cond_enc.hidden2", "cond_enc.z"};

int dense_failed(int rc) { return rc ? fail(rc, std::string("dense layer: ") + petdense_last_error()) : PETDIFF_OK; }

petdense_forward_args forward16(const void* x, int64_t ldx, const void* w, const void* bias, void* y, int64_t ldy,
                                int64_t m, int64_t k, int64_t n, int relu, int out_f32) {
  petdense_forward_args a{};
  a.x = x;
  a.ldx = ldx;
  a.kernel = w;
  a.ldk = n;
  a.bias = bias;
  a.bias_f32 = 1;
  a.y = y;
  a.ldy = ldy;
  a.m = m;
  a.k = k;
  a.n = n;
  a.dtype = PETDENSE_BF16;
  a.activation = relu ? PETDENSE_RELU : PETDENSE_NONE;
  a.out_f32 = out_f32;
  return a;
}

petdense_backward_args backward16(const void* dy, const Kept& in, bool e4m3, int64_t ldx, const void* w,
                                  const void* relu_out, void* dx, float* dk, float* db, int64_t m, int64_t k,
                                  int64_t n) {
  petdense_backward_args a{};
  a.dy = dy;
  a.lddy = n;
  a.x = in.rows.p;
  a.ldx = ldx;
  if (e4m3) {
    a.x_exponents = in.exps.u8();
    a.lde = (k + PETDENSE_BLOCK - 1) / PETDENSE_BLOCK;
  }
  a.kernel = w;
  a.ldk = n;
  a.saved = relu_out;
  a.lds = n;
  a.activation = relu_out ? PETDENSE_RELU : PETDENSE_NONE;
  a.dx = dx;
  a.lddx = k;
  a.dkernel = dk;
  a.lddk = n;
  a.dbias = db;
  a.m = m;
  a.k = k;
  a.n = n;
  a.dtype = PETDENSE_BF16;
  a.grad_f32 = 1;
  return a;
}

// The convolution's arguments with every pointer but the workspace as in a step: the workspaces' sizes go by them.
petdense_backward_args conv_backward16(pettrain_ctx* h, int c, int B, float* Gk, float* Gb) {
  const K::ConvIn ci = conv_in(c);
  const int M = B * ci.lout(), Kd = ci.taps * ci.cfull(), Kp = pad8(Kd);
  // the padding's rows of the kernel gradient would lie on the blob's next values: those go through a buffer
  float* dk = Kp == Kd ? Gk : h->gk16.f();
  return backward16(h->dp16.p, h->in16[c], h->keep == PETTRAIN_KEEP_E4M3, Kp, h->w16[c].p, nullptr, h->da16.p, dk, Gb,
                    M, Kp, conv_out(c));
}

petdense_backward_args enc_backward16(pettrain_ctx* h, int l, int R) {
  const std::string name = kEncName[l];
  // layer l's output gradient is de16[l]; its input's goes to de16[l - 1]
  petdense_backward_args a = backward16(
      h->de16[l].p, h->en16[l], h->keep == PETTRAIN_KEEP_E4M3, pad8(kEncIn[l]), h->we16[l].p,
      l < 3 ? h->e16[l + 1].p : nullptr, l ? h->de16[l - 1].p : nullptr, h->G(name + ".kernel"), h->G(name + ".bias"),
      R, kEncIn[l], kEncOut[l]);
  if (h->keep != PETTRAIN_KEEP_E4M3) a.x = h->e16[l].p;
  return a;
}

int ensure16(pettrain_ctx* h, int B) {
  const size_t Bz = (size_t)B, R = Bz * 49;
  const bool e4m3 = h->keep == PETTRAIN_KEEP_E4M3;
  size_t most = 0, grad = 0;
  for (int c = 0; c < 10; ++c) {
    const K::ConvIn ci = conv_in(c);
    const size_t M = Bz * ci.lout(), Kd = (size_t)ci.taps * ci.cfull(), Kp = pad8((int)Kd), N = conv_out(c);
    HIPC(h->w16[c].alloc(Kp * N * 2));
    HIPC(h->b16[c].alloc(N * 4));
    HIPC(h->in16[c].rows.alloc(M * Kp * (e4m3 ? 1 : 2)));
    if (e4m3) HIPC(h->in16[c].exps.alloc(M * ((Kp + PETDENSE_BLOCK - 1) / PETDENSE_BLOCK)));
    most = std::max(most, M * Kp);
    if (Kp != Kd) grad = std::max(grad, Kp * N);
  }
  if (e4m3) HIPC(h->a16.alloc(most * 2));
  HIPC(h->da16.alloc(most * 2));
  HIPC(h->dp16.alloc(Bz * 6144 * 2));
  HIPC(h->gk16.alloc(grad * 4));
  for (int l = 0; l < 4; ++l) {
    const size_t K = pad8(kEncIn[l]), N = kEncOut[l];
    HIPC(h->we16[l].alloc((size_t)kEncIn[l] * N * 2));
    HIPC(h->e16[l].alloc(R * K * 2));
    HIPC(h->de16[l].alloc(R * N * 2));
    if (e4m3) {
      HIPC(h->en16[l].rows.alloc(R * K));
      HIPC(h->en16[l].exps.alloc(R * ((kEncIn[l] + PETDENSE_BLOCK - 1) / PETDENSE_BLOCK)));
    }
  }
  return PETDIFF_OK;
}

// The products' workspace goes by the batch (a smaller one may be split where a larger one is not): it grows on demand.
hipError_t grow_work(pettrain_ctx* h, size_t need, hipStream_t s) {
  if (need <= h->work16.bytes) return hipSuccess;
  if (hipError_t e = hipStreamSynchronize(s)) return e;       // a product may still be using the old one
  return h->work16.alloc(need);
}

int run_forward16(pettrain_ctx* h, const petdense_forward_args& a, hipStream_t s) {
  const size_t need = petdense_forward_workspace(&a);
  HIPC(grow_work(h, need, s));
  return dense_failed(petdense_forward(&a, h->work16.p, h->work16.bytes, s));
}

int run_backward16(pettrain_ctx* h, const petdense_backward_args& a, hipStream_t s) {
  const size_t need = petdense_backward_workspace(&a);
  HIPC(grow_work(h, need, s));
  return dense_failed(petdense_backward(&a, h->work16.p, h->work16.bytes, s));
}

// keeps X [M][K] (row stride ld) of a product for its backward pass
int keep16(pettrain_ctx* h, const void* X, int64_t ld, int64_t M, int64_t K, Kept& in, hipStream_t s) {
  return dense_failed(petdense_checkpoint(X, ld, M, K, PETDENSE_BF16, in.rows.u8(), ld, in.exps.u8(),
                                          (K + PETDENSE_BLOCK - 1) / PETDENSE_BLOCK, s));
}

// out[M][cout] = (relu) im2col W + bias, in fp32
int conv_fwd16(pettrain_ctx* h, int c, int B, const float* lab, const float* tim, const float* x1, const float* x2,
               int relu, bool keep, float* out, hipStream_t s) {
  const K::ConvIn ci = conv_in(c);
  const int M = B * ci.lout(), Kp = pad8(ci.taps * ci.cfull()), N = conv_out(c);
  const bool e4m3 = h->keep == PETTRAIN_KEEP_E4M3;
  __bf16* A = e4m3 ? h->a16.h() : h->in16[c].rows.h();
  HIPC(K::im2col16(ci, B, lab, tim, x1, x2, A, Kp, s));
  CHK(run_forward16(h, forward16(A, Kp, h->w16[c].p, h->b16[c].p, out, N, M, Kp, N, relu, 1), s));
  if (e4m3 && keep) CHK(keep16(h, A, Kp, M, Kp, h->in16[c], s));
  return PETDIFF_OK;
}

// from dp16 (the pre-activation's gradient): kernel and bias gradients, and the input's through col2im
int conv_bwd16(pettrain_ctx* h, int c, int B, float* Gk, float* Gb, float* dlab, float* dtim, float* dx1, float* dx2,
               hipStream_t s) {
  const K::ConvIn ci = conv_in(c);
  const int Kd = ci.taps * ci.cfull(), Kp = pad8(Kd);
  CHK(run_backward16(h, conv_backward16(h, c, B, Gk, Gb), s));
  if (Kp != Kd)
    HIPC(hipMemcpyAsync(Gk, h->gk16.p, (size_t)Kd * conv_out(c) * 4, hipMemcpyDeviceToDevice, s));
  HIPC(K::col2im16(ci, B, h->da16.h(), Kp, dlab, dtim, dx1, dx2, s));
  return PETDIFF_OK;
}

// dense forward: Y[M, N] (row stride ldy) = [X | 1] [kernel ; bias], X of row stride Kd + 1
int dense_fwd(pettrain_ctx* h, const float* X, int M, int Kd, const std::string& name, int N, float* Y, int ldy,
              int relu, hipStream_t s) {
  CHK(gemm(h, false, false, M, N, Kd + 1, X, Kd + 1, h->W(name + ".kernel"), N, Y, ldy, 0.f));
  if (relu) HIPC(K::bias_act(Y, M, N, ldy, nullptr, 1, s));
  return PETDIFF_OK;
}

// dense backward: G [kernel ; bias] = [X | 1]^T dY; dX (=|+=) dY kernel^T (dX may be null)
int dense_bwd(pettrain_ctx* h, const float* X, const float* dY, int M, int Kd, const std::string& name, int N,
              float* dX, float beta) {
  CHK(gemm(h, true, false, Kd + 1, N, M, X, Kd + 1, dY, N, h->G(name + ".kernel"), N, 0.f));
  if (dX) CHK(gemm(h, false, true, M, Kd, N, dY, N, h->W(name + ".kernel"), N, dX, Kd, beta));
  return PETDIFF_OK;
}

// conv forward: out[B*Lout, cout] = [im2col | 1] [W ; bias] (relu optional)
int conv_fwd(pettrain_ctx* h, const K::ConvIn& ci, int B, const float* lab, const float* tim, const float* x1,
             const float* x2, float* A, const float* Wk, int cout, int relu, float* out, hipStream_t s) {
  HIPC(K::im2col(ci, B, lab, tim, x1, x2, A, s));
  const int M = B * ci.lout(), Kd = ci.taps * ci.cfull();
  CHK(gemm(h, false, false, M, cout, Kd + 1, A, Kd + 1, Wk, cout, out, cout, 0.f));
  if (relu) HIPC(K::bias_act(out, M, cout, cout, nullptr, 1, s));
  return PETDIFF_OK;
}

// conv backward from dpre: G [kernel ; bias] = [A | 1]^T dpre, dA = dpre W^T, col2im
int conv_bwd(pettrain_ctx* h, const K::ConvIn& ci, int B, const float* A, const float* Wk, int cout,
             const float* dpre, float* Gk, float* dlab, float* dtim, float* dx1, float* dx2, hipStream_t s) {
  const int M = B * ci.lout(), Kd = ci.taps * ci.cfull();
  CHK(gemm(h, true, false, Kd + 1, cout, M, A, Kd + 1, dpre, cout, Gk, cout, 0.f));
  CHK(gemm(h, false, true, M, Kd, cout, dpre, cout, Wk, cout, h->dA.f(), Kd, 0.f));
  HIPC(K::col2im(ci, B, h->dA.f(), dlab, dtim, dx1, dx2, s));
  return PETDIFF_OK;
}

// the residual 1x1 kernel / bias share the gradient of the centre tap / conv bias
int copy_res_grads(pettrain_ctx* h, const std::string& p, int cin_full, int cout, hipStream_t s) {
  const size_t cn = (size_t)cin_full * cout;
  HIPC(hipMemcpyAsync(h->G(p + ".res.kernel"), h->G(p + ".conv.kernel") + 2 * cn, cn * 4, hipMemcpyDeviceToDevice,
                      s));
  HIPC(hipMemcpyAsync(h->G(p + ".res.bias"), h->G(p + ".conv.bias"), (size_t)cout * 4, hipMemcpyDeviceToDevice, s));
  return PETDIFF_OK;
}

std::string level_prefix(int p) { return p < 4 ? "down" + std::to_string(p) : "up" + std::to_string(p - 4); }

// label / time projection backward of cond level p (networks.py:915-921, 958-964)
int cond_bwd(pettrain_ctx* h, int p, int B, bool first) {
  const std::string pre = level_prefix(p);
  const int L = kLevelL[p], R = B * 49;
  CHK(dense_bwd(h, h->z.f(), h->dlab.f(), R, 32, pre + ".label_proj", L, h->dz.f(), first ? 0.f : 1.f));
  CHK(dense_bwd(h, h->h_t.f(), h->dtim.f(), B, 48, pre + ".time_proj", L, h->dh_t.f(), first ? 0.f : 1.f));
  return PETDIFF_OK;
}

int forward_backward(pettrain_ctx* h, const float* x0, const float* cond, int B, const int32_t* t_in,
                     const float* noise_in, uint64_t seed, uint64_t goff, float* loss_out, hipStream_t s,
                     bool backward = true) {
  CHK(ensure(h, B));
  RBC(rocblas_set_stream(h->rb, s));
  const int R = B * 49;
  // q-sample (diffusion_model.py:542-551)
  HIPC(K::qsample(x0, t_in, noise_in, seed, goff, h->iter, B, h->T, h->tab.f(), h->t.i(), h->noise.f(), h->xt.f(),
                  s));
  // time MLP and condition encoder (networks.py:182-198, 235-258, 574-586)
  HIPC(K::time_embed(h->t.i(), B, 64, h->emb.f(), 65, s));
  CHK(dense_fwd(h, h->emb.f(), B, 64, "time_mlp", 48, h->a_t.f(), 48, 0, s));
  HIPC(K::gelu_fwd(h->a_t.f(), h->h_t.f(), B, 48, 49, s));
  const bool bf16 = h->precision == PETTRAIN_BF16;
  if (bf16) {
    HIPC(K::to_bf16(cond, R, 54, h->e16[0].h(), pad8(54), s));
    for (int l = 0; l < 4; ++l) {
      const std::string name = kEncName[l];
      HIPC(K::to_bf16(h->W(name + ".kernel"), kEncIn[l], kEncOut[l], h->we16[l].h(), kEncOut[l], s));
      CHK(run_forward16(h, forward16(h->e16[l].p, pad8(kEncIn[l]), h->we16[l].p, h->W(name + ".bias"),
                                     l < 3 ? h->e16[l + 1].p : h->z.p, l < 3 ? kEncOut[l] : 33, R, kEncIn[l],
                                     kEncOut[l], l < 3, l == 3), s));
      if (backward && h->keep == PETTRAIN_KEEP_E4M3)
        CHK(keep16(h, h->e16[l].p, pad8(kEncIn[l]), R, kEncIn[l], h->en16[l], s));
    }
  } else {
    HIPC(K::copy_rows(cond, R, 54, h->cond_aug.f(), 55, s));
    CHK(dense_fwd(h, h->cond_aug.f(), R, 54, "cond_enc.hidden0", 256, h->e1.f(), 257, 1, s));
    CHK(dense_fwd(h, h->e1.f(), R, 256, "cond_enc.hidden1", 128, h->e2.f(), 129, 1, s));
    CHK(dense_fwd(h, h->e2.f(), R, 128, "cond_enc.hidden2", 64, h->e3.f(), 65, 1, s));
    CHK(dense_fwd(h, h->e3.f(), R, 64, "cond_enc.z", 32, h->z.f(), 33, 0, s));
  }
  for (int p = 0; p < 7; ++p) {
    const std::string pre = level_prefix(p);
    CHK(dense_fwd(h, h->z.f(), R, 32, pre + ".label_proj", kLevelL[p], h->lab[p].f(), kLevelL[p], 0, s));
    CHK(dense_fwd(h, h->h_t.f(), B, 48, pre + ".time_proj", kLevelL[p], h->tim[p].f(), kLevelL[p], 0, s));
  }
  // down path (networks.py:1010-1031)
  for (int d = 0; d < 4; ++d) {
    const std::string p = "down" + std::to_string(d);
    const K::ConvIn ci = down_in(d);
    const float* xin = d == 0 ? h->xt.f() : h->pool[d - 1].f();
    if (bf16) {
      HIPC(K::fold_weff16(h->W(p + ".conv.kernel"), h->W(p + ".conv.bias"), h->W(p + ".res.kernel"),
                          h->W(p + ".res.bias"), h->w16[d].h(), h->b16[d].f(), pad8(6 * ci.cfull()), 6, 2, ci.cfull(),
                          kDownCout[d], s));
      CHK(conv_fwd16(h, d, B, h->lab[d].f(), h->tim[d].f(), xin, nullptr, 1, backward, h->out_dn[d].f(), s));
    } else {
      HIPC(K::fold_weff(h->W(p + ".conv.kernel"), h->W(p + ".conv.bias"), h->W(p + ".res.kernel"),
                        h->W(p + ".res.bias"), h->weff[d].f(), 6, 2, ci.cfull(), kDownCout[d], s));
      CHK(conv_fwd(h, ci, B, h->lab[d].f(), h->tim[d].f(), xin, nullptr, h->A_dn[d].f(), h->weff[d].f(), kDownCout[d],
                   1, h->out_dn[d].f(), s));
    }
    if (d < 3) HIPC(K::maxpool_fwd(h->out_dn[d].f(), h->pool[d].f(), B, kDownL[d], kDownCout[d], s));
  }
  // up path (networks.py:1033-1072)
  for (int u = 0; u < 3; ++u) {
    const std::string p = "up" + std::to_string(u);
    const K::ConvIn uc = upconv_in(u), bk = block_in(u);
    const float* hin = u == 0 ? h->out_dn[3].f() : h->out_up[u - 1].f();
    if (bf16) {
      HIPC(K::fold_weff16(h->W(p + ".upconv.kernel"), h->W(p + ".upconv.bias"), nullptr, nullptr, h->w16[4 + u].h(),
                          h->b16[4 + u].f(), pad8(2 * uc.cfull()), 2, 0, uc.cfull(), kUpCout[u], s));
      CHK(conv_fwd16(h, 4 + u, B, h->lab[4 + u].f(), h->tim[4 + u].f(), hin, nullptr, 0, backward, h->hu[u].f(), s));
      HIPC(K::fold_weff16(h->W(p + ".conv.kernel"), h->W(p + ".conv.bias"), h->W(p + ".res.kernel"),
                          h->W(p + ".res.bias"), h->w16[7 + u].h(), h->b16[7 + u].f(), pad8(6 * bk.cfull()), 6, 2,
                          bk.cfull(), kUpCout[u], s));
      CHK(conv_fwd16(h, 7 + u, B, nullptr, nullptr, h->out_dn[2 - u].f(), h->hu[u].f(), 1, backward, h->out_up[u].f(), s));
      continue;
    }
    CHK(conv_fwd(h, uc, B, h->lab[4 + u].f(), h->tim[4 + u].f(), hin, nullptr, h->A_uc[u].f(),
                 h->W(p + ".upconv.kernel"), kUpCout[u], 0, h->hu[u].f(), s));
    HIPC(K::fold_weff(h->W(p + ".conv.kernel"), h->W(p + ".conv.bias"), h->W(p + ".res.kernel"),
                      h->W(p + ".res.bias"), h->weff[4 + u].f(), 6, 2, bk.cfull(), kUpCout[u], s));
    CHK(conv_fwd(h, bk, B, nullptr, nullptr, h->out_dn[2 - u].f(), h->hu[u].f(), h->A_bk[u].f(), h->weff[4 + u].f(),
                 kUpCout[u], 1, h->out_up[u].f(), s));
  }
  // final Conv1D 1x1 (networks.py:1074)
  const int n_out = h->n_out;
  CHK(gemm(h, false, false, B * 48, n_out, 128, h->out_up[2].f(), 128, h->W("final.kernel"), n_out, h->y4.f(), n_out,
           0.f));
  HIPC(K::bias_act(h->y4.f(), B * 48, n_out, n_out, h->W("final.bias"), 0, s));
  // loss + d loss / d output (diffusion_model.py:498-578)
  K::LossArgs la{};
  la.y = h->y4.f();
  la.x0 = x0;
  la.noise = h->noise.f();
  la.xt = h->xt.f();
  la.t = h->t.i();
  la.tab = h->tab.f();
  la.T = h->T;
  la.B = B;
  la.n_out = n_out;
  la.learn_mode = h->learn_mode;
  la.param_mode = h->param_mode;
  la.lambda_vlb = h->opt.lambda_vlb;
  la.bin_width = (float)(2.0 * 1.34896 / std::cbrt((double)B * 48.0));    // freedman_diaconis_rule (:529-531)
  la.dy = h->dy4.f();
  la.sse = h->sse.f();
  la.vlb = h->vlb.f();
  la.dbias_part = h->dbias_part.f();
  HIPC(K::loss(la, s));
  HIPC(K::loss_finish(h->sse.f(), h->vlb.f(), h->dbias_part.f(), B, n_out, B * 96, loss_out,
                      reinterpret_cast<double*>(h->stats.p), backward ? h->G("final.bias") : nullptr, s));
  h->has_stats = true;
  if (!backward) return PETDIFF_OK;   // test_step: loss only, the gradient blob is untouched

  // ---------------- backward ----------------
  CHK(gemm(h, true, false, 128, n_out, B * 48, h->out_up[2].f(), 128, h->dy4.f(), n_out, h->G("final.kernel"), n_out,
           0.f));
  CHK(gemm(h, false, true, B * 48, 128, n_out, h->dy4.f(), n_out, h->W("final.kernel"), n_out, h->d_out_up[2].f(),
           128, 0.f));
  bool first = true;
  for (int u = 2; u >= 0; --u) {
    const std::string p = "up" + std::to_string(u);
    const K::ConvIn uc = upconv_in(u), bk = block_in(u);
    float* dhin = u == 0 ? h->d_out_dn3.f() : h->d_out_up[u - 1].f();
    if (bf16) {
      HIPC(K::pool_mask_bwd16(h->out_up[u].f(), nullptr, h->d_out_up[u].f(), h->dp16.h(), B, bk.lout(), kUpCout[u], s));
      CHK(conv_bwd16(h, 7 + u, B, h->G(p + ".conv.kernel"), h->G(p + ".conv.bias"), nullptr, nullptr,
                     h->dskip[2 - u].f(), h->dhu.f(), s));
      CHK(copy_res_grads(h, p, bk.cfull(), kUpCout[u], s));
      HIPC(K::to_bf16(h->dhu.f(), B * uc.lout(), kUpCout[u], h->dp16.h(), kUpCout[u], s));
      CHK(conv_bwd16(h, 4 + u, B, h->G(p + ".upconv.kernel"), h->G(p + ".upconv.bias"), h->dlab.f(), h->dtim.f(), dhin,
                     nullptr, s));
      CHK(cond_bwd(h, 4 + u, B, first));
      first = false;
      continue;
    }
    HIPC(K::pool_mask_bwd(h->out_up[u].f(), nullptr, h->d_out_up[u].f(), h->dpre.f(), B, bk.lout(), kUpCout[u], s));
    CHK(conv_bwd(h, bk, B, h->A_bk[u].f(), h->weff[4 + u].f(), kUpCout[u], h->dpre.f(), h->G(p + ".conv.kernel"),
                 nullptr, nullptr, h->dskip[2 - u].f(), h->dhu.f(), s));
    CHK(copy_res_grads(h, p, bk.cfull(), kUpCout[u], s));
    CHK(conv_bwd(h, uc, B, h->A_uc[u].f(), h->W(p + ".upconv.kernel"), kUpCout[u], h->dhu.f(),
                 h->G(p + ".upconv.kernel"), h->dlab.f(), h->dtim.f(), dhin, nullptr, s));
    CHK(cond_bwd(h, 4 + u, B, first));
    first = false;
  }
  for (int d = 3; d >= 0; --d) {
    const std::string p = "down" + std::to_string(d);
    const K::ConvIn ci = down_in(d);
    if (bf16) {
      const bool last = d == 3;
      HIPC(K::pool_mask_bwd16(h->out_dn[d].f(), last ? nullptr : h->d_pool[d].f(),
                              last ? h->d_out_dn3.f() : h->dskip[d].f(), h->dp16.h(), B, kDownL[d], kDownCout[d], s));
      CHK(conv_bwd16(h, d, B, h->G(p + ".conv.kernel"), h->G(p + ".conv.bias"), h->dlab.f(), h->dtim.f(),
                     d > 0 ? h->d_pool[d - 1].f() : nullptr, nullptr, s));
      CHK(copy_res_grads(h, p, ci.cfull(), kDownCout[d], s));
      CHK(cond_bwd(h, d, B, false));
      continue;
    }
    if (d == 3)
      HIPC(K::pool_mask_bwd(h->out_dn[3].f(), nullptr, h->d_out_dn3.f(), h->dpre.f(), B, 6, 1024, s));
    else
      HIPC(K::pool_mask_bwd(h->out_dn[d].f(), h->d_pool[d].f(), h->dskip[d].f(), h->dpre.f(), B, kDownL[d],
                            kDownCout[d], s));
    CHK(conv_bwd(h, ci, B, h->A_dn[d].f(), h->weff[d].f(), kDownCout[d], h->dpre.f(), h->G(p + ".conv.kernel"),
                 h->dlab.f(), h->dtim.f(), d > 0 ? h->d_pool[d - 1].f() : nullptr, nullptr, s));
    CHK(copy_res_grads(h, p, ci.cfull(), kDownCout[d], s));
    CHK(cond_bwd(h, d, B, false));
  }
  if (bf16) {
    HIPC(K::to_bf16(h->dz.f(), R, 32, h->de16[3].h(), 32, s));
    for (int l = 3; l >= 0; --l) CHK(run_backward16(h, enc_backward16(h, l, R), s));
    HIPC(K::gelu_bwd(h->dh_t.f(), h->a_t.f(), h->da_t.f(), B * 48, s));
    CHK(dense_bwd(h, h->emb.f(), h->da_t.f(), B, 64, "time_mlp", 48, nullptr, 0.f));
    h->last_B = B;
    return PETDIFF_OK;
  }
  // condition encoder backward (ReLU masks read the augmented activations)
  CHK(dense_bwd(h, h->e3.f(), h->dz.f(), R, 64, "cond_enc.z", 32, h->de3.f(), 0.f));
  HIPC(K::relu_mask(h->de3.f(), h->e3.f(), R, 64, 65, s));
  CHK(dense_bwd(h, h->e2.f(), h->de3.f(), R, 128, "cond_enc.hidden2", 64, h->de2.f(), 0.f));
  HIPC(K::relu_mask(h->de2.f(), h->e2.f(), R, 128, 129, s));
  CHK(dense_bwd(h, h->e1.f(), h->de2.f(), R, 256, "cond_enc.hidden1", 128, h->de1.f(), 0.f));
  HIPC(K::relu_mask(h->de1.f(), h->e1.f(), R, 256, 257, s));
  CHK(dense_bwd(h, h->cond_aug.f(), h->de1.f(), R, 54, "cond_enc.hidden0", 256, nullptr, 0.f));
  // time MLP backward (GELU exact)
  HIPC(K::gelu_bwd(h->dh_t.f(), h->a_t.f(), h->da_t.f(), B * 48, s));
  CHK(dense_bwd(h, h->emb.f(), h->da_t.f(), B, 64, "time_mlp", 48, nullptr, 0.f));
  h->last_B = B;
  return PETDIFF_OK;
}

}  // namespace

extern "C" {

const char* pettrain_last_error(void) { return g_err.c_str(); }

int pettrain_default_config(pettrain_config* o) {
  if (!o) return fail(PETDIFF_ERR_INVALID, "null argument");
  o->learning_rate = 2e-4f;
  o->decay_steps = 1.0f;
  o->decay_rate = 1.0f;
  o->beta_1 = 0.9f;
  o->beta_2 = 0.999f;
  o->epsilon = 1e-7f;
  o->clipnorm = 1.5f;
  o->lambda_vlb = 0.1f;
  return PETDIFF_OK;
}

int pettrain_create(const petdiff_config* cfg, const float* weights, size_t n_weights, const float* tab, int T,
                    const pettrain_config* opt, int device, pettrain_handle* out) {
  if (!cfg || !weights || !tab || !opt || !out || T <= 1) return fail(PETDIFF_ERR_INVALID, "bad arguments");
  if (!is_shipped_arch(*cfg))
    return fail(PETDIFF_ERR_UNSUPPORTED, "only the shipped UnetConditional architecture is compiled");
  if (cfg->learn_variance < 0 || cfg->learn_variance > 2 || cfg->parameterization < 0 || cfg->parameterization > 3)
    return fail(PETDIFF_ERR_INVALID, "bad learn_variance / parameterization");
  if (!(opt->decay_steps > 0.f) || !(opt->learning_rate >= 0.f))
    return fail(PETDIFF_ERR_INVALID, "bad optimizer config");
  std::unique_ptr<pettrain_ctx> h(new pettrain_ctx());
  h->cfg = *cfg;
  h->opt = *opt;
  h->device = device;
  h->T = T;
  h->learn_mode = cfg->learn_variance;
  h->param_mode = cfg->parameterization;
  h->n_out = cfg->learn_variance == PETDIFF_LEARN_FIXED ? cfg->n_par : 2 * cfg->n_par;
  h->spec = make_spec(*cfg, h->n_out);
  h->n_w = h->spec.back().off + h->spec.back().size;
  if (n_weights != h->n_w)
    return fail(PETDIFF_ERR_INVALID, "weight blob has " + std::to_string(n_weights) + " values, expected " +
                                         std::to_string(h->n_w));
  for (auto& s : h->spec) h->off[s.name] = s.off;
  HIPC(hipSetDevice(device));
  if (rocblas_create_handle(&h->rb) != rocblas_status_success) return fail(PETDIFF_ERR_HIP, "rocblas_create_handle");
  RBC(rocblas_set_atomics_mode(h->rb, rocblas_atomics_not_allowed));   // run-to-run deterministic GEMMs
  const size_t wb = h->n_w * 4;
  HIPC(h->w.alloc(wb));
  HIPC(h->g.alloc(wb));
  HIPC(h->m.alloc(wb));
  HIPC(h->v.alloc(wb));
  HIPC(hipMemcpy(h->w.p, weights, wb, hipMemcpyHostToDevice));
  HIPC(hipMemset(h->g.p, 0, wb));
  HIPC(hipMemset(h->m.p, 0, wb));
  HIPC(hipMemset(h->v.p, 0, wb));
  HIPC(h->tab.alloc((size_t)kNTab * T * 4));
  HIPC(hipMemcpy(h->tab.p, tab, (size_t)kNTab * T * 4, hipMemcpyHostToDevice));
  for (int d = 0; d < 4; ++d) HIPC(h->weff[d].alloc(((size_t)6 * down_in(d).cfull() + 1) * kDownCout[d] * 4));
  for (int u = 0; u < 3; ++u) HIPC(h->weff[4 + u].alloc(((size_t)6 * block_in(u).cfull() + 1) * kUpCout[u] * 4));
  // optimizer chunk tables
  std::vector<int> cvar, clen, vfirst, vcount;
  std::vector<long long> cstart;
  for (size_t k = 0; k < h->spec.size(); ++k) {
    vfirst.push_back((int)cvar.size());
    const Spec& s = h->spec[k];
    int n = 0;
    for (size_t o = 0; o < s.size; o += K::kChunk, ++n) {
      cvar.push_back((int)k);
      cstart.push_back((long long)(s.off + o));
      clen.push_back((int)std::min<size_t>(K::kChunk, s.size - o));
    }
    vcount.push_back(n);
  }
  h->n_chunks = (int)cvar.size();
  h->n_vars = (int)h->spec.size();
  HIPC(h->cvar.alloc(cvar.size() * 4));
  HIPC(h->clen.alloc(clen.size() * 4));
  HIPC(h->cstart.alloc(cstart.size() * 8));
  HIPC(h->vfirst.alloc(vfirst.size() * 4));
  HIPC(h->vcount.alloc(vcount.size() * 4));
  HIPC(h->partial.alloc(cvar.size() * 8));
  HIPC(h->vscale.alloc(vfirst.size() * 4));
  HIPC(hipMemcpy(h->cvar.p, cvar.data(), cvar.size() * 4, hipMemcpyHostToDevice));
  HIPC(hipMemcpy(h->clen.p, clen.data(), clen.size() * 4, hipMemcpyHostToDevice));
  HIPC(hipMemcpy(h->cstart.p, cstart.data(), cstart.size() * 8, hipMemcpyHostToDevice));
  HIPC(hipMemcpy(h->vfirst.p, vfirst.data(), vfirst.size() * 4, hipMemcpyHostToDevice));
  HIPC(hipMemcpy(h->vcount.p, vcount.data(), vcount.size() * 4, hipMemcpyHostToDevice));
  *out = h.release();
  return PETDIFF_OK;
}

void pettrain_destroy(pettrain_handle h) {
  if (!h) return;
  if (h->rb) (void)rocblas_destroy_handle(h->rb);
  delete h;
}

int pettrain_set_precision(pettrain_handle h, int precision, int keep) {
  if (!h) return fail(PETDIFF_ERR_INVALID, "null handle");
  if (precision != PETTRAIN_F32 && precision != PETTRAIN_BF16)
    return fail(PETDIFF_ERR_INVALID, "precision must be PETTRAIN_F32 or PETTRAIN_BF16");
  if (keep != PETTRAIN_KEEP && keep != PETTRAIN_KEEP_E4M3)
    return fail(PETDIFF_ERR_INVALID, "keep must be PETTRAIN_KEEP or PETTRAIN_KEEP_E4M3");
  if (keep == PETTRAIN_KEEP_E4M3 && precision != PETTRAIN_BF16)
    return fail(PETDIFF_ERR_INVALID, "8-bit checkpoints need PETTRAIN_BF16");
  if (precision == h->precision && keep == h->keep) return PETDIFF_OK;
  HIPC(hipSetDevice(h->device));
  const auto release = [](Buf* b, size_t count) {
    for (size_t i = 0; i < count; ++i) b[i].release();
  };
  // what one of the precisions alone holds
  release(h->A_dn, 4);
  release(h->A_uc, 3);
  release(h->A_bk, 3);
  release(h->w16, 10);
  release(h->b16, 10);
  release(h->we16, 4);
  release(h->e16, 4);
  release(h->de16, 4);
  for (Kept* k = h->in16; k != h->in16 + 10; ++k) {
    k->rows.release();
    k->exps.release();
  }
  for (Kept* k = h->en16; k != h->en16 + 4; ++k) {
    k->rows.release();
    k->exps.release();
  }
  for (Buf* b : {&h->cond_aug, &h->e1, &h->e2, &h->e3, &h->de1, &h->de2, &h->de3, &h->dA, &h->dpre, &h->a16, &h->da16,
                 &h->dp16, &h->gk16, &h->work16})
    b->release();
  h->B_cap = 0;                 // the next step allocates what its precision needs
  h->precision = precision;
  h->keep = keep;
  return PETDIFF_OK;
}

size_t pettrain_step_bytes(pettrain_handle h) {
  if (!h) return 0;
  size_t n = 0;
  const auto add = [&](const Buf* b, size_t count) {
    for (size_t i = 0; i < count; ++i) n += b[i].bytes;
  };
  const Buf* one[] = {&h->t, &h->noise, &h->xt, &h->emb, &h->a_t, &h->h_t, &h->cond_aug, &h->e1, &h->e2, &h->e3,
                      &h->z, &h->y4, &h->dy4, &h->dA, &h->dpre, &h->d_out_dn3, &h->dhu, &h->dlab, &h->dtim, &h->dz,
                      &h->dh_t, &h->da_t, &h->de1, &h->de2, &h->de3, &h->sse, &h->vlb, &h->dbias_part, &h->stats,
                      &h->a16, &h->da16, &h->dp16, &h->gk16, &h->work16};
  for (const Buf* b : one) add(b, 1);
  add(h->lab, 7);
  add(h->tim, 7);
  add(h->A_dn, 4);
  add(h->out_dn, 4);
  add(h->pool, 3);
  add(h->A_uc, 3);
  add(h->hu, 3);
  add(h->A_bk, 3);
  add(h->out_up, 3);
  add(h->d_out_up, 3);
  add(h->d_pool, 3);
  add(h->dskip, 3);
  add(h->w16, 10);
  add(h->b16, 10);
  add(h->we16, 4);
  add(h->e16, 4);
  add(h->de16, 4);
  for (const Kept& k : h->in16) n += k.rows.bytes + k.exps.bytes;
  for (const Kept& k : h->en16) n += k.rows.bytes + k.exps.bytes;
  return n;
}

int pettrain_compute_gradients(pettrain_handle h, const float* x0_dev, const float* cond_dev, int B,
                               const int32_t* t_dev, const float* noise_dev, uint64_t seed, uint64_t sample_offset,
                               float* loss_dev, void* stream) {
  if (!h) return fail(PETDIFF_ERR_INVALID, "null handle");
  if (B <= 0 || !x0_dev || !cond_dev) return fail(PETDIFF_ERR_INVALID, "bad arguments");
  HIPC(hipSetDevice(h->device));
  return forward_backward(h, x0_dev, cond_dev, B, t_dev, noise_dev, seed, sample_offset, loss_dev,
                          (hipStream_t)stream);
}

int pettrain_compute_loss(pettrain_handle h, const float* x0_dev, const float* cond_dev, int B, const int32_t* t_dev,
                          const float* noise_dev, uint64_t seed, uint64_t sample_offset, float* loss_dev,
                          void* stream) {
  if (!h) return fail(PETDIFF_ERR_INVALID, "null handle");
  if (B <= 0 || !x0_dev || !cond_dev) return fail(PETDIFF_ERR_INVALID, "bad arguments");
  HIPC(hipSetDevice(h->device));
  return forward_backward(h, x0_dev, cond_dev, B, t_dev, noise_dev, seed, sample_offset, loss_dev,
                          (hipStream_t)stream, false);
}

int pettrain_apply_gradients(pettrain_handle h, float grad_scale, void* stream) {
  if (!h) return fail(PETDIFF_ERR_INVALID, "null handle");
  if (h->last_B <= 0) return fail(PETDIFF_ERR_INVALID, "no gradients computed yet");
  HIPC(hipSetDevice(h->device));
  // Keras: lr from the schedule at `iterations`, then alpha in the variable dtype (fp32)
  const pettrain_config& o = h->opt;
  const float lr = (float)((double)o.learning_rate * std::pow((double)o.decay_rate, (double)h->iter / o.decay_steps));
  const float step = (float)(h->iter + 1);
  const float b1p = std::pow(o.beta_1, step), b2p = std::pow(o.beta_2, step);
  K::AdamArgs a{};
  a.w = h->w.f();
  a.g = h->g.f();
  a.m = h->m.f();
  a.v = h->v.f();
  a.cvar = h->cvar.i();
  a.cstart = reinterpret_cast<const long long*>(h->cstart.p);
  a.clen = h->clen.i();
  a.n_chunks = h->n_chunks;
  a.vfirst = h->vfirst.i();
  a.vcount = h->vcount.i();
  a.n_vars = h->n_vars;
  a.partial = reinterpret_cast<double*>(h->partial.p);
  a.vscale = h->vscale.f();
  a.grad_scale = grad_scale;
  a.clipnorm = o.clipnorm;
  a.alpha = lr * std::sqrt(1.0f - b2p) / (1.0f - b1p);
  a.beta_1 = o.beta_1;
  a.beta_2 = o.beta_2;
  a.epsilon = o.epsilon;
  HIPC(K::adam(a, (hipStream_t)stream));
  h->iter += 1;
  return PETDIFF_OK;
}

int pettrain_step(pettrain_handle h, const float* x0_dev, const float* cond_dev, int B, const int32_t* t_dev,
                  const float* noise_dev, uint64_t seed, uint64_t sample_offset, float* loss_dev, void* stream) {
  CHK(pettrain_compute_gradients(h, x0_dev, cond_dev, B, t_dev, noise_dev, seed, sample_offset, loss_dev, stream));
  return pettrain_apply_gradients(h, 1.0f, stream);
}

float* pettrain_gradients(pettrain_handle h) { return h ? h->g.f() : nullptr; }

int pettrain_get_gradients(pettrain_handle h, float* dst_dev, void* stream) {
  if (!h || !dst_dev) return fail(PETDIFF_ERR_INVALID, "bad arguments");
  HIPC(hipMemcpyAsync(dst_dev, h->g.p, h->n_w * 4, hipMemcpyDeviceToDevice, (hipStream_t)stream));
  return PETDIFF_OK;
}

int pettrain_set_gradients(pettrain_handle h, const float* src_dev, void* stream) {
  if (!h || !src_dev) return fail(PETDIFF_ERR_INVALID, "bad arguments");
  HIPC(hipMemcpyAsync(h->g.p, src_dev, h->n_w * 4, hipMemcpyDeviceToDevice, (hipStream_t)stream));
  return PETDIFF_OK;
}

int pettrain_get_weights(pettrain_handle h, float* dst_dev, void* stream) {
  if (!h || !dst_dev) return fail(PETDIFF_ERR_INVALID, "bad arguments");
  HIPC(hipMemcpyAsync(dst_dev, h->w.p, h->n_w * 4, hipMemcpyDeviceToDevice, (hipStream_t)stream));
  return PETDIFF_OK;
}

int pettrain_last_stats(pettrain_handle h, double* out3, void* stream) {
  if (!h || !out3) return fail(PETDIFF_ERR_INVALID, "bad arguments");
  if (!h->has_stats) return fail(PETDIFF_ERR_INVALID, "no step run yet");
  HIPC(hipMemcpyAsync(out3, h->stats.p, 3 * sizeof(double), hipMemcpyDeviceToHost, (hipStream_t)stream));
  HIPC(hipStreamSynchronize((hipStream_t)stream));
  return PETDIFF_OK;
}

int64_t pettrain_iterations(pettrain_handle h) { return h ? h->iter : -1; }

}  // extern "C"
