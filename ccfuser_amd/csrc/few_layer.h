// The MoE layer for a few tokens (few_layer.hip), as the entry points call it.
#pragma once

#include "fp8.h"

namespace ccf {

struct FewLayerArgs {
  const half_t *x;                                 // [tokens, d]
  const uint8_t *x_codes;                          // the same in 8 bits, or null
  const float *x_scales;
  const half_t *wg, *bg;
  const void *w1;                                  // [E, f, d] fp16, or codes with scales s1
  const float *s1;
  const half_t *b1;                                // or null
  const void *w2;                                  // [E, d, f]
  const float *s2;
  const half_t *b2;
  int tokens, d, f, E, k;
  int64_t *idx;                                    // [tokens, k], written; -1: no expert
  half_t *score;
  void *h;                                         // [tokens * k, f] fp16, or codes with h_scales
  float *h_scales;
  half_t *out;                                     // [tokens, d]
};

bool few_layer_fits(int tokens, int d, int f, int E, int k);
// Whether the first kernel has room for the tokens in 8 bits.
bool few_layer_fits_fp8(int tokens, int d);
int few_layer(const FewLayerArgs &p, bool fp8, ccf_stream_t stream);

}  // namespace ccf
