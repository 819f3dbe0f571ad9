// The gate's selection: which logits of a token are the k best, and their softmax.  Shared by the kernels that gate, so
// that one choice has one set of bits.
#pragma once

#include "ccf_common.h"

#include <limits.h>

namespace ccf {

constexpr int kMaxTopK = 8;
constexpr int kPart = 128;          // K elements of a part of a logit's sum

template <typename T>
__device__ inline float round_to(float v) {
  return static_cast<float>(static_cast<T>(v));
}

__device__ inline bool better(float v, int id, float bv, int bid) {
  return v > bv || (v == bv && id < bid);
}

// The k best of a token so far (k <= KS), best first; ties keep the lower expert id.
template <int KS>
struct Best {
  float v[KS];
  int id[KS];
  __device__ inline void clear() {
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      v[s] = -INFINITY;
      id[s] = INT_MAX;
    }
  }
  __device__ inline void offer(float nv, int nid, int k) {
    if constexpr (KS > 2) {                        // long lists: most offers end at the last kept entry
      float lv = v[0];
      int li = id[0];
#pragma unroll
      for (int s = 1; s < KS; ++s)
        if (s == k - 1) {
          lv = v[s];
          li = id[s];
        }
      if (!better(nv, nid, lv, li)) return;        // not among the k best
    }
    bool beats[KS];                                // short lists: no branch
#pragma unroll
    for (int s = 0; s < KS; ++s) beats[s] = better(nv, nid, v[s], id[s]);
#pragma unroll
    for (int s = KS - 1; s >= 0; --s) {
      if (s < k) {
        const int up = s > 0 ? s - 1 : 0;
        const bool ahead = s > 0 && beats[up];     // belongs further up: slot s takes its upper neighbour
        v[s] = ahead ? v[up] : (beats[s] ? nv : v[s]);
        id[s] = ahead ? id[up] : (beats[s] ? nid : id[s]);
      }
    }
  }
  // softmax over the k selected logits (slot 0 holds the maximum) and the writes
  template <typename T>
  __device__ inline void write(int t, int k, int64_t *__restrict__ idx_out, T *__restrict__ score_out) const {
    float ex[KS];
    float sum = 0.0f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      ex[s] = (s < k) ? expf(v[s] - v[0]) : 0.0f;
      sum += ex[s];
    }
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      if (s < k) {
        idx_out[static_cast<size_t>(t) * k + s] = static_cast<int64_t>(id[s]);
        score_out[static_cast<size_t>(t) * k + s] = static_cast<T>(ex[s] / sum);
      }
    }
  }
};

}  // namespace ccf
