/* Argument block of the low-rank adapter kernels, shared by the host (g++) and
 * device (hipcc) compilers: plain C types only. */
#ifndef RLXQ_LORA_ARGS_H
#define RLXQ_LORA_ARGS_H
#include <stdint.h>

#define RLXQ_LORA_SEGS 4           /* most column segments of a call            */
#define RLXQ_LORA_MAX_RANK 256
#define RLXQ_LORA_SPLITS 8         /* most slices of K                          */
#define RLXQ_LORA_MAX_ADAPTERS 16384
#define RLXQ_LORA_ROWS 32          /* rows of a tile of the list                */
#define RLXQ_LORA_FEW 256          /* most rows whose tiles every workgroup finds */

/* Rows of one adapter that a workgroup takes together (prompts). */
typedef struct rlxq_lora_tile {
  int32_t e;               /* adapter, or -1: rows without one                */
  int32_t start, count;    /* order[start .. start + count)                   */
  int32_t pad;
} rlxq_lora_tile;

typedef struct rlxq_lora_args {
  const void* x;           /* [M, K]                                          */
  const int32_t* ids;      /* [M]; outside [0, E): no adapter                 */
  const void* a;           /* [E, S * R, K]                                   */
  const void* b;           /* [E, N, R]                                       */
  const int32_t* ranks;    /* [E], or NULL (R)                                */
  const float* scales;     /* [E], or NULL (1)                                */
  const void* base;        /* [M, N], or NULL (zero)                          */
  void* y;                 /* [M, N]                                          */
  float* v;                /* [splits, M, S * R]: A x, by slice of K          */
  int32_t* order;          /* [M]: rows by adapter (with the list)            */
  rlxq_lora_tile* tiles;   /* [max_tiles], unused ones with count 0           */
  int64_t M, K, N;
  int32_t R, E, S;
  int32_t splits, kslice;  /* slices of K, each a multiple of 128: four waves */
                           /* of whole 32s                                    */
  int32_t jblocks;         /* shrink: workgroups over S * R                   */
  int32_t cols, cblocks;   /* expand: columns a workgroup, workgroups over N  */
  int32_t max_tiles;
  int32_t vec;             /* base, y and the segments allow 16-byte accesses */
  int32_t copy;            /* rows without an adapter are base's: copied      */
  int64_t ends[RLXQ_LORA_SEGS];    /* column ends of the segments (the last N) */
  int32_t cfirst[RLXQ_LORA_SEGS];  /* expand: first workgroup of a segment    */
} rlxq_lora_args;

#endif
