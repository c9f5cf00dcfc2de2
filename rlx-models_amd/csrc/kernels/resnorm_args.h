/* Argument block of the residual-norm kernels, shared by the host (g++) and
 * device (hipcc) compilers: plain C types only. */
#ifndef RLXQ_RESNORM_ARGS_H
#define RLXQ_RESNORM_ARGS_H
#include <stdint.h>

typedef struct rlxq_resnorm_args {
  const void* block;       /* [M, H], or NULL (zero)                          */
  const void* resid;       /* [M, H], or NULL (zero)                          */
  const void* gate;        /* [M / gate_span, H], or NULL (one)               */
  const void* post_w;      /* [H], or NULL: the block is not normalised       */
  const void* pre_w;       /* [H], or NULL: y is not written                  */
  void* sum;               /* [M, H] of resid's type, or NULL                 */
  void* y;                 /* [M, H], or NULL                                 */
  int64_t M, H, gate_span;
  float alpha, eps, w_off;
  int32_t block_bf16, resid_bf16, gate_bf16, w_bf16, y_bf16;
} rlxq_resnorm_args;

#endif
