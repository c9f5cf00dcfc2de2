/* Argument blocks of the MXFP4 quantiser and matmul kernels, shared by the
 * host (g++) and device (hipcc) compilers: plain C types only. */
#ifndef RLXQ_MXFP4_ARGS_H
#define RLXQ_MXFP4_ARGS_H
#include <stdint.h>

/* Quantised activations as the matmul's MFMA operand ("fragments"): for
 * `rows` (16 or 32) activation rows and one span of 64 / rows * 128 elements,
 * a chunk of 4096 code bytes and 256 scale bytes.  Lane l of a wave holds row
 * l % rows and, with g = l / rows, four of the span's blocks, b(g, j) = 4 g + j
 * (16 rows) or 4 (j / 2) + 2 g + j % 2 (32 rows, whose first half of 128
 * elements is j = 0, 1), j = 0 .. 3: the 16 code bytes of block b(g, j) at
 * 1024 j + 16 l, its scale byte at 4096 + 4 l + j.
 * Chunk (row block rb, span s) is number rb * spans + s. */
#define RLXQ_MX_CHUNK 4352

typedef struct rlxq_mx_quant_args {
  const void* x;      /* f32 or bf16 [M, K]                                  */
  uint8_t* codes;     /* [M, K / 2], or the fragment chunks (rows != 0)      */
  uint8_t* scales;    /* [M, K / 32] (rows == 0)                             */
  int64_t M, K;
  int32_t rows;       /* 0: row-major; 16 or 32: fragments                   */
  int32_t spans;      /* fragments: spans of a row (the last one padded)     */
  /* wblocks > 0: the first wblocks workgroups lay out the scales of 32 weight
   * rows each (see mx_scale_frag)                                          */
  int32_t wblocks, pad;
  const uint8_t* ws;  /* E8M0 scales [N, K / 32]                             */
  uint32_t* wsf;      /* [wblocks, spans, 64]                                */
  uint8_t* zero;      /* [wblocks]                                           */
  int64_t N;
} rlxq_mx_quant_args;

typedef struct rlxq_mx_gemm_args {
  const uint8_t* xf;  /* activation fragments                                */
  const void* x;      /* kernels that quantise them themselves: [M, K]       */
  const uint8_t* w;   /* codes [N, K / 2]                                    */
  const uint8_t* ws;  /* E8M0 scales [N, K / 32]                             */
  void* y;            /* [M, N] f32 or bf16                                  */
  const uint32_t* wsf;   /* scales of 32-row blocks in lane order (rows = 32) */
  const uint8_t* zero;   /* which of those blocks hold a scale byte 0        */
  float* part;        /* splits > 1: f32 partial sums [splits, M, N]         */
  int64_t M, N, K;
  int32_t spans;      /* spans of a row                                      */
  int32_t splits;     /* K splits over workgroups                            */
  int32_t y_bf16;
  int32_t vec;        /* whole 16-byte stores: N and y allow them              */
} rlxq_mx_gemm_args;

#endif
