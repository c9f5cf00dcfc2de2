/* Argument block of the low-rank adapter kernels, shared by the host (g++) and
 * device (hipcc) compilers: plain C types only. */
#ifndef RLXQ_LORA_ARGS_H
#define RLXQ_LORA_ARGS_H
#include <stdint.h>

#define RLXQ_LORA_SEGS 4   /* most column segments of a call */

typedef struct rlxq_lora_args {
  const void* x;           /* [M, K]                                          */
  const int32_t* ids;      /* [M]; outside [0, E): no adapter                 */
  const void* a;           /* [E, S * R, K]                                   */
  const void* b;           /* [E, N, R]                                       */
  const int32_t* ranks;    /* [E], or NULL (R)                                */
  const float* scales;     /* [E], or NULL (1)                                */
  const void* base;        /* [M, N], or NULL (zero)                          */
  void* y;                 /* [M, N]                                          */
  float* v;                /* [M, S * R]: scale * (A x)                       */
  int64_t M, K, N;
  int32_t R, E, S;
  int32_t x_bf16, ab_bf16, y_bf16;
  int64_t ends[RLXQ_LORA_SEGS];   /* column ends of the segments (the last N) */
} rlxq_lora_args;

#endif
