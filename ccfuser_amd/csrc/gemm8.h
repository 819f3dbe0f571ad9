// Products in e4m3 with a scale for each block of 128: what the launchers and the layer call share.
#pragma once

#include "fp8.h"

namespace ccf {

struct Gemm8Args {
  const uint8_t *a;          // rows' codes [*, K]
  const float *a_scale;      // [*, KB]
  const int32_t *a_rows;     // row of `a` for sorted row j, null: j
  const uint8_t *b;          // weights' codes [E, N, K]
  const float *b_scale;      // [E, NB, KB]
  const void *bias;          // [E, N] in the output's type, or null
  const int32_t *offsets;    // [E + 1], null: one weight for rows 0 .. max_rows - 1
  int max_rows, E, N, K;
  const int32_t *c_rows;     // row of the output for sorted row j, null: j
  void *c;                   // [*, N]
  uint8_t *codes;            // or, through the GELU, codes [*, N] and scales [*, NB]
  float *scales;
};

enum { kGemm8Half = 0, kGemm8Bf16 = 1, kGemm8Gelu8 = 2 };     // the output: fp16, bf16, or GELU and 8 bits

extern int g_fp8_form;       // ccf_set_option("fp8_form"): 0 .. 6

int gemm8(const Gemm8Args &p, int out, hipStream_t stream, const char *what);

int launch_quantize_rows(const void *x, int rows, int k, int dtype, uint8_t *codes, float *scales, hipStream_t st);

}  // namespace ccf
