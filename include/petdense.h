/*
 * petdense.h -- C ABI of the dense layer's operators on MI355X (libpetdiff.so): the products of the denoiser's
 * training step (every Dense layer, and every Conv1D over its im2col matrix; networks.py:529-537, 666-670) with
 * their epilogues, their backward pass, and activations kept in 8 bits for it.
 *
 *   forward    P = X W + b + R,  Y = act(P)       X [m][k], W [k][n] (Keras layout), b [n], R [m][n]
 *   backward   dP = dY act'(P);  dX = dP W^T,  dW = X^T dP,  db = column sums of dP,  dR = dP
 *   checkpoint blocks of 32 values along a row share 2^E, the least (E >= -117) with max|x| <= 448 2^E over the
 *              block's finite values; a value is kept as the e4m3 code nearest to x 2^-E (ties to even), the block
 *              as the byte E + 127.  NaN and infinities become NaN.  Where 256 2^E is past the type's largest value
 *              (E = 8 for fp16, 120 for bf16 and fp32) codes end at 240, so that every finite value is restored
 *              as a finite one.
 *
 * Types: x, kernel, residual, dy and saved are of one type, PETDENSE_F32 / BF16 / F16.  Sums run in fp32 (fp32
 * products on the fp32 matrix instructions) and every output is rounded once.  In the backward pass of a 16-bit
 * layer dP is rounded to the layer's type before the two products, which take 16-bit operands; db sums the
 * unrounded dP.  ReLU and linear layers' dP are exact; the others' products carry its rounding, into an fp32 dkernel
 * too.  GELU and SiLU are evaluated to 2^-16 of themselves in 16-bit layers, to (x^2 + 8) 2^-23 in fp32 ones, lower
 * tails included.  ReLU's gradient where saved is NaN is dy.
 *
 * All pointers are device memory of the current device and belong to the caller; work runs on `stream`, in order,
 * with no synchronisation and no allocation, so every call can be captured into a graph.  Workspaces: at least
 * petdense_*_workspace bytes, 256-byte aligned, not shared by calls that may run at once (two streams, two captured
 * graphs that may replay together).  Their sizes go by every argument, which outputs are asked for and the pointers'
 * alignment included: ask with the arguments of the call.  Row strides (ld*) are in values, at least the row's
 * length; rows do not overlap.  Outputs do not alias inputs or each other, with one exception: y may be the residual
 * itself.  Sums are in a fixed order: results are the same from run to run.  A call's y, dx and dkernel, where asked
 * for, have fewer than 2^23 tiles of 64 x 64 values each (2^35 values).
 *
 * Every function returns a PETDIFF_* code (petdiff.h); petdense_last_error() names the last failure of the thread.
 */
#ifndef PETDENSE_H
#define PETDENSE_H

#include <stddef.h>
#include <stdint.h>

#include "petdiff.h"

#ifdef __cplusplus
extern "C" {
#endif

#define PETDENSE_F32 0
#define PETDENSE_BF16 1
#define PETDENSE_F16 2

#define PETDENSE_NONE 0
#define PETDENSE_RELU 1
#define PETDENSE_GELU 2    /* x (1 + erf(x / sqrt 2)) / 2, the time MLP's (networks.py:235-258) */
#define PETDENSE_SILU 3    /* x / (1 + exp(-x)) */

#define PETDENSE_BLOCK 32  /* values of a row that share an exponent byte */

typedef struct petdense_forward_args {
  const void* x;           /* [m][k] */
  const void* kernel;      /* [k][n] */
  const void* bias;        /* [n] or NULL */
  const void* residual;    /* [m][n] or NULL: added before the activation */
  void* y;                 /* [m][n] */
  void* pre;               /* [m][n] or NULL: P, in y's type (what GELU and SiLU need saved for the backward pass) */
  int64_t ldx, ldk, ldr, ldy, ldp;
  int64_t m, k, n;         /* m >= 0; k, n >= 1; all < 2^31 - 65536 */
  int dtype, activation;
  int bias_f32;            /* bias is fp32 */
  int out_f32;             /* y and pre are fp32 */
} petdense_forward_args;

typedef struct petdense_backward_args {
  const void* dy;          /* [m][n] */
  const void* x;           /* [m][k]; e4m3 codes when x_exponents is given; may be NULL when dkernel is */
  const uint8_t* x_exponents; /* [m][ceil(k / 32)] bytes E + 127, or NULL */
  const void* kernel;      /* [k][n]; may be NULL when dx is */
  const void* saved;       /* [m][n]: P for GELU and SiLU, P or Y for ReLU; ignored without an activation */
  void* dx;                /* [m][k] or NULL, of dtype */
  void* dkernel;           /* [k][n] or NULL */
  void* dbias;             /* [n] or NULL */
  void* dresidual;         /* [m][n] or NULL, of dtype */
  int64_t lddy, ldx, lde, ldk, lds, lddx, lddk, lddr;
  int64_t m, k, n;
  int dtype, activation;
  int grad_f32;            /* dkernel and dbias are fp32 (else: dtype) */
} petdense_backward_args;

size_t petdense_forward_workspace(const petdense_forward_args* a);
int petdense_forward(const petdense_forward_args* a, void* work, size_t work_bytes, void* stream);

size_t petdense_backward_workspace(const petdense_backward_args* a);
int petdense_backward(const petdense_backward_args* a, void* work, size_t work_bytes, void* stream);

/* m >= 0, k >= 1, both < 2^31 - 65536.
 * x [m][k] of dtype (row stride ldx) -> codes [m][k] bytes (row stride ldc), exponents [m][ceil(k / 32)] (lde) */
int petdense_checkpoint(const void* x, int64_t ldx, int64_t m, int64_t k, int dtype, uint8_t* codes, int64_t ldc,
                        uint8_t* exponents, int64_t lde, void* stream);
/* the values that the codes stand for, in dtype: exact, but that fp16 rounds what is below 2^-14.  Exponent bytes
 * are those that petdense_checkpoint writes for dtype. */
int petdense_restore(const uint8_t* codes, int64_t ldc, const uint8_t* exponents, int64_t lde, int64_t m, int64_t k,
                     int dtype, void* x, int64_t ldx, void* stream);

const char* petdense_last_error(void);

#ifdef __cplusplus
}
#endif
#endif /* PETDENSE_H */
