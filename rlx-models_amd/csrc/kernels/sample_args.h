/* Argument block of the sampling kernels, shared by the host (g++) and device
 * (hipcc) compilers: plain C types only. */
#ifndef RLXQ_SAMPLE_ARGS_H
#define RLXQ_SAMPLE_ARGS_H
#include <stdint.h>

#define RLXQ_SAMPLE_MAX_VOCAB (1 << 20)

typedef struct rlxq_sample_args {
  const void* logits;        /* [M, V] f32 or bf16                            */
  const float* temperature;  /* [M], or NULL (1)                              */
  const int32_t* top_k;      /* [M], or NULL (off)                            */
  const float* top_p;        /* [M], or NULL (off)                            */
  const float* min_p;        /* [M], or NULL (off)                            */
  const float* u;            /* [M]                                           */
  int32_t* tokens;           /* [M]                                           */
  float* probs;              /* [M], or NULL                                  */
  int64_t M;
  int32_t V, bf16;
} rlxq_sample_args;

#endif
