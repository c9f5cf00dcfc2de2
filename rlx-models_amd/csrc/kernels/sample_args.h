/* Argument block of the sampling kernels, shared by the host (g++) and device
 * (hipcc) compilers: plain C types only. */
#ifndef RLXQ_SAMPLE_ARGS_H
#define RLXQ_SAMPLE_ARGS_H
#include <stdint.h>

#define RLXQ_SAMPLE_MAX_VOCAB (1 << 20)
#define RLXQ_SAMPLE_CHUNK 4096   /* elements of a chunk                         */
/* A chunk's bins: steps of 1/16 in l / T down from a multiple of 2 (32 bins) at
 * or above its top, the last bin open; 16 groups of 32 */
#define RLXQ_SAMPLE_BINS 512
#define RLXQ_SAMPLE_GROUPS 16

/* What the first launch leaves of one chunk of one row. */
typedef struct rlxq_sample_chunk {
  uint64_t best;      /* largest (key, falling index) of the chunk; 0: all masked */
  double mass;        /* its weights over its own largest, times 2^48          */
  uint32_t bad;       /* holds a NaN or +inf                                   */
  uint32_t count;     /* elements that are not masked (rows with top_k)        */
  float tops[4];      /* the largest logit of each quarter                     */
  double group_mass[RLXQ_SAMPLE_GROUPS];      /* as mass (rows with a border)  */
  uint32_t group_count[RLXQ_SAMPLE_GROUPS];   /* (rows with top_k)             */
} rlxq_sample_chunk;

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
  int32_t chunks, per;       /* of a row; of a workgroup                      */
  rlxq_sample_chunk* heads;  /* [M, chunks]                                   */
  uint64_t* masses;          /* [M, chunks, BINS], each in steps of its own   */
  uint16_t* counts;          /* [M, chunks, BINS]                             */
} rlxq_sample_args;

#endif
