// The whole MoE layer for a few tokens in two kernels, on experts in 16 or in 8 bits, for gfx950: one sequence being
// decoded, or a small batch of them.
//
//   1. gate, choice, FFN1 and GELU   h[t, s, :] = gelu(x[t] w1[e]^T + b1[e]) for the slots (t, s) of every chosen expert e
//   2. FFN2 and the combine          out[t] = sum over s of score[t, s] (h[t, s] w2[e]^T + b2[e])
//
// Bound by the chosen experts' weights, which are read once, and by launches.  What makes it two:
//
//   * every workgroup of the first kernel gates for itself: the logits of a few tokens are as long as the launch of a
//     kernel that would compute them (their sums and the selection are the gate's own, bit for bit);
//   * no routing: a product's columns are the tokens themselves, 16 or 32 of them, whichever of them chose the expert, so
//     no rows are listed, moved or padded; what a token gets from an expert that it did not choose is dropped;
//   * the second kernel runs all chosen experts of its 16 columns into one sum, so nothing is left to combine.
//
// In 8 bits (e4m3, a scale per block of 128) rows of x are quantised where they are read, as ccf_quantize_rows does, and
// the first kernel's workgroups have the 128 columns of a scale of h.  Wavefronts cut K among them and read straight from
// memory, 16 rows of 128 consecutive bytes at a time, two steps ahead; their sums meet in LDS in a fixed order.
#include "few_layer.h"
#include "gate_select.h"
#include "gelu.h"
#include "plan.h"

#include <type_traits>

namespace ccf {
namespace {

constexpr int kFewTokens = 32;                     // most
constexpr int kFewSlots = kFewTokens * kMaxTopK;
constexpr int kThreads = 512, kWaves = kThreads / 64;

__device__ const int4v kZeros16 = {0, 0, 0, 0};    // what lanes behind the end of K read

enum { kHalf = 0, kCodes = 1, kQuantise = 2 };     // fp16 weights; e4m3 ones, with rows in 8 bits or quantised here

__device__ __forceinline__ int8v join(int4v lo, int4v hi) { return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7); }

// 16 columns (w) by 16 tokens (x) over the 128 bytes of a step, from zero.
template <bool kFp8>
__device__ __forceinline__ float4v product(int8v w, int8v x) {
  if constexpr (kFp8) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, float4v{0, 0, 0, 0}, 0, 0, 0, 0, 0, 0);
  } else {
    typedef _Float16 half16 __attribute__((ext_vector_type(16)));
    const half16 a = __builtin_bit_cast(half16, w), b = __builtin_bit_cast(half16, x);
    const half8 a0 = __builtin_shufflevector(a, a, 0, 1, 2, 3, 4, 5, 6, 7), a1 = __builtin_shufflevector(a, a, 8, 9, 10, 11, 12, 13, 14, 15);
    const half8 b0 = __builtin_shufflevector(b, b, 0, 1, 2, 3, 4, 5, 6, 7), b1 = __builtin_shufflevector(b, b, 8, 9, 10, 11, 12, 13, 14, 15);
    const float4v c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, b0, float4v{0, 0, 0, 0}, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, b1, c, 0, 0, 0);
  }
}

// 32 bytes of a row of `bytes` from byte `at` on; zeros behind its end.
__device__ __forceinline__ int8v piece(const uint8_t *row, int at, int bytes) {
  const int4v *zeros = &kZeros16;
  const int4v *lo = at < bytes ? reinterpret_cast<const int4v *>(row + at) : zeros;
  const int4v *hi = at + 16 < bytes ? reinterpret_cast<const int4v *>(row + at + 16) : zeros;
  return join(*lo, *hi);
}

// Which experts have tokens, in ascending order, and which slot of a token each is.
struct Slots {
  unsigned mask[32];                               // of E <= 1024 experts
  int act[kFewSlots];                              // the chosen experts
  uint8_t slot[kFewSlots][kFewTokens];             // slot of token t that expert act[i] is, 255: none
  int e[kFewSlots];                                // the tokens' choice
  float score[kFewSlots];

  __device__ __forceinline__ int rank(int expert) const {
    int r = __popc(mask[expert >> 5] & ((1u << (expert & 31)) - 1));
    for (int i = 0; i < expert >> 5; ++i) r += __popc(mask[i]);
    return r;
  }
  // all threads, behind a barrier after e and score were written; how many experts were chosen
  __device__ int build(int n, int k, int E) {
    if (threadIdx.x < 32) mask[threadIdx.x] = 0;
    for (int i = threadIdx.x; i < n * kFewTokens / 4; i += blockDim.x) reinterpret_cast<unsigned *>(slot)[i] = 0xffffffffu;
    __syncthreads();
    const int q = threadIdx.x, mine = q < n ? e[q] : E;
    const bool valid = mine >= 0 && mine < E;      // (a list that NaN logits left short has entries that are no expert)
    if (valid) atomicOr(&mask[mine >> 5], 1u << (mine & 31));
    __syncthreads();
    if (valid) {
      const int r = rank(mine), t = q / k;
      act[r] = mine;
      slot[r][t] = static_cast<uint8_t>(q - t * k);
    }
    int total = 0;
    for (int i = 0; i < (E + 31) / 32; ++i) total += __popc(mask[i]);
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(total);
  }
};

// LDS of the gate: expert rows, token rows, part sums, logits
struct GateLds {
  int x, part, logit, bytes;
};
__host__ __device__ inline GateLds gate_lds(int T, int E, int nparts) {
  GateLds l;
  l.x = E * nparts * 256;
  l.part = l.x + T * nparts * 256;
  l.logit = l.part + 4 * T * E * (nparts + 1);
  l.bytes = l.logit + 4 * T * (E + 1);
  return l;
}

// The gate's choice for all tokens: chains of fused multiply-adds over parts of 128 elements from zero, the parts' sums in
// ascending order, the bias last, one rounding to fp16.  Rows lie in LDS in 16-byte pieces, piece c of part i at
// c ^ (i % 16), so that lanes on neighbouring parts read other banks.
__device__ __forceinline__ void gate_here(const FewLayerArgs &p, char *s_raw, Slots &slots) {
  const int T = p.tokens, d = p.d, E = p.E, k = p.k, nparts = (d + kPart - 1) / kPart;
  const GateLds at = gate_lds(T, E, nparts);
  float *s_part = reinterpret_cast<float *>(s_raw + at.part), *s_logit = reinterpret_cast<float *>(s_raw + at.logit);
  auto fetch = [&](const half_t *base, int rows, int to) {
    const int pieces = rows * nparts * 16;
    for (int s = threadIdx.x; s < pieces; s += kThreads) {
      const int i = s >> 4, r = i / nparts, part = i - r * nparts, c = s & 15, kk = part * kPart + c * 8;
      const half8 v = kk < d ? *reinterpret_cast<const half8 *>(base + static_cast<size_t>(r) * d + kk) : half8{0, 0, 0, 0, 0, 0, 0, 0};
      *reinterpret_cast<half8 *>(s_raw + to + i * 256 + ((c ^ (i & 15)) << 4)) = v;
    }
  };
  fetch(p.wg, E, 0);
  fetch(p.x, T, at.x);
  __syncthreads();
  const int chains = E * nparts;
  for (int q = threadIdx.x; q < T * chains; q += kThreads) {
    const int t = q / chains, chain = q - t * chains, part = chain % nparts, xi = t * nparts + part;
    const char *wr = s_raw + chain * 256, *xr = s_raw + at.x + xi * 256;
    const int len = d - part * kPart;
    float acc = 0.0f;
#pragma unroll
    for (int c = 0; c < kPart / 8; ++c) {
      const half8 wv = *reinterpret_cast<const half8 *>(wr + ((c ^ (chain & 15)) << 4));
      const half8 xv = *reinterpret_cast<const half8 *>(xr + ((c ^ (xi & 15)) << 4));
      if (c * 8 < len) {
#pragma unroll
        for (int j = 0; j < 8; ++j) acc = __builtin_fmaf(static_cast<float>(xv[j]), static_cast<float>(wv[j]), acc);
      }
    }
    s_part[(t * E + chain / nparts) * (nparts + 1) + part] = acc;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < T * E; i += kThreads) {
    const float *ps = s_part + i * (nparts + 1);
    float v = ps[0];
    for (int q = 1; q < nparts; ++q) v = v + ps[q];
    if (p.bg) v = v + static_cast<float>(p.bg[i % E]);
    s_logit[i / E * (E + 1) + i % E] = round_to<half_t>(v);
  }
  __syncthreads();
  if (static_cast<int>(threadIdx.x) < T) {
    const int t = threadIdx.x;
    Best<kMaxTopK> best;
    best.clear();
    for (int e = 0; e < E; ++e) best.offer(s_logit[t * (E + 1) + e], e, k);
    int64_t idx[kMaxTopK];
    half_t score[kMaxTopK];
    best.write<half_t>(0, k, idx, score);
#pragma unroll
    for (int s = 0; s < kMaxTopK; ++s)
      if (s < k) {
        slots.e[t * k + s] = best.id[s];
        if (blockIdx.x == 0) {                     // for the second kernel
          p.idx[t * k + s] = idx[s] < E ? idx[s] : -1;
          p.score[t * k + s] = score[s];
        }
      }
  }
}

// 16 RB tokens; a workgroup's columns: 64 of fp16 weights, whose K all eight wavefronts cut among them, 128 in 8 bits, four
// wavefronts to either half.
template <int kIn, int RB>
__global__ void __launch_bounds__(kThreads, kIn == kHalf && RB == 1 ? 4 : 2)
few_layer_up_kernel(FewLayerArgs p, bool gated) {
  constexpr bool kFp8 = kIn != kHalf;
  constexpr int CT = 4, CS = kFp8 ? 2 : 1, KS = kWaves / CS, BN = 16 * CT * CS, kLd = BN + 4;
  extern __shared__ __attribute__((aligned(16))) char s_raw[];
  __shared__ Slots slots;
  const int T = p.tokens, n = T * p.k;
  if (gated) {
    for (int q = threadIdx.x; q < n; q += kThreads) {
      const int64_t e = p.idx[q];
      const bool valid = e >= 0 && e < p.E;
      slots.e[q] = valid ? static_cast<int>(e) : p.E;
      if (!valid && blockIdx.x == 0) p.idx[q] = -1;
    }
  } else {
    gate_here(p, s_raw, slots);
  }
  __syncthreads();
  const int n_act = slots.build(n, p.k, p.E);

  float *s_part = reinterpret_cast<float *>(s_raw);                        // [KS][16 RB][kLd]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g = lane >> 4, ks = wave % KS, cs = wave / KS;
  const int row_bytes = p.d * (kFp8 ? 1 : 2), steps = (row_bytes + 127) / 128;
  const int blocks = (p.f + BN - 1) / BN, KB = scale_blocks(p.d), FB = scale_blocks(p.f);
  const int count = steps > ks ? (steps - ks + KS - 1) / KS : 0;           // steps ks, ks + KS, ...
  int token[RB];
#pragma unroll
  for (int b = 0; b < RB; ++b) token[b] = 16 * b + r16 < T ? 16 * b + r16 : T - 1;

  for (int u = blockIdx.x; u < n_act * blocks; u += gridDim.x) {
    const int i = u / blocks, n0 = (u - i * blocks) * BN, c0 = n0 + cs * 16 * CT;
    const int e = __builtin_amdgcn_readfirstlane(slots.act[i]);
    const uint8_t *w[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      const int col = c0 + 16 * c + r16;
      w[c] = static_cast<const uint8_t *>(p.w1) + (static_cast<size_t>(e) * p.f + (col < p.f ? col : p.f - 1)) * row_bytes;
    }
    const float *sb = kFp8 ? p.s1 + (static_cast<size_t>(e) * FB + (c0 / kScaleBlock < FB ? c0 / kScaleBlock : FB - 1)) * KB : nullptr;
    float4v acc[CT][RB];
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int b = 0; b < RB; ++b) acc[c][b] = float4v{0, 0, 0, 0};
    int8v wf[2][CT], xf[2][RB], xw[2][RB];         // xw: the second half of 32 elements in 16 bits
    float sx[2][RB], sw[2];
    auto fetch = [&](int q, auto B_) {             // the wavefront's step q; past the last one it again
      constexpr int buf = decltype(B_)::value;
      const int st = ks + (q < count ? q : count - 1) * KS;
#pragma unroll
      for (int c = 0; c < CT; ++c) wf[buf][c] = piece(w[c], st * 128 + 32 * g, row_bytes);
#pragma unroll
      for (int b = 0; b < RB; ++b) {
        if constexpr (kIn == kQuantise) {
          const uint8_t *row = reinterpret_cast<const uint8_t *>(p.x + static_cast<size_t>(token[b]) * p.d);
          xf[buf][b] = piece(row, st * 256 + 64 * g, 2 * p.d);
          xw[buf][b] = piece(row, st * 256 + 64 * g + 32, 2 * p.d);
        } else if constexpr (kIn == kCodes) {
          xf[buf][b] = piece(p.x_codes + static_cast<size_t>(token[b]) * p.d, st * 128 + 32 * g, p.d);
          sx[buf][b] = p.x_scales[static_cast<size_t>(token[b]) * KB + st];
        } else {
          xf[buf][b] = piece(reinterpret_cast<const uint8_t *>(p.x + static_cast<size_t>(token[b]) * p.d), st * 128 + 32 * g, row_bytes);
        }
      }
      if constexpr (kFp8) sw[buf] = sb[st];
    };
    auto multiply = [&](int q, auto B_) {
      constexpr int buf = decltype(B_)::value;
      if (q >= count) return;                      // uniform
#pragma unroll
      for (int b = 0; b < RB; ++b) {
        int8v x = xf[buf][b];
        float s = 1.0f;
        if constexpr (kIn == kQuantise) {
          typedef _Float16 half16 __attribute__((ext_vector_type(16)));
          const half16 lo = __builtin_bit_cast(half16, xf[buf][b]), hi = __builtin_bit_cast(half16, xw[buf][b]);
          float top = 0.0f;
#pragma unroll
          for (int j = 0; j < 16; ++j) top = fmaxf(top, fmaxf(fabsf(static_cast<float>(lo[j])), fabsf(static_cast<float>(hi[j]))));
          top = fmaxf(top, __shfl_xor(top, 16));
          top = fmaxf(top, __shfl_xor(top, 32));
          float inverse;
          s = block_scale(top, &inverse);
          auto four = [&](const half16 &v, int j) {
            return pack_fp8(static_cast<float>(v[j]) * inverse, static_cast<float>(v[j + 1]) * inverse,
                            static_cast<float>(v[j + 2]) * inverse, static_cast<float>(v[j + 3]) * inverse);
          };
          x = int8v{four(lo, 0), four(lo, 4), four(lo, 8), four(lo, 12), four(hi, 0), four(hi, 4), four(hi, 8), four(hi, 12)};
        } else if constexpr (kIn == kCodes) {
          s = sx[buf][b];
        }
        if constexpr (kFp8) s *= sw[buf];
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          const float4v part = product<kFp8>(wf[buf][c], x);
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[c][b][j] = kFp8 ? fmaf(part[j], s, acc[c][b][j]) : acc[c][b][j] + part[j];
        }
      }
    };
    if (count > 0) {
      constexpr std::integral_constant<int, 0> even{};
      constexpr std::integral_constant<int, 1> odd{};
      fetch(0, even);
      for (int q = 0; q < count; q += 2) {
        fetch(q + 1, odd);
        __builtin_amdgcn_sched_barrier(0);
        multiply(q, even);
        __builtin_amdgcn_sched_barrier(0);
        fetch(q + 2, even);
        __builtin_amdgcn_sched_barrier(0);
        multiply(q + 1, odd);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    __syncthreads();                               // the gate's or the last unit's LDS is read
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int b = 0; b < RB; ++b)
        *reinterpret_cast<float4v *>(s_part + (ks * 16 * RB + 16 * b + r16) * kLd + (cs * CT + c) * 16 + 4 * g) = acc[c][b];
    __syncthreads();
    // eight consecutive columns of a token to a thread
    const half_t *bias = p.b1 ? p.b1 + static_cast<size_t>(e) * p.f : nullptr;
    constexpr int kPer = BN / 8;
    for (int o = threadIdx.x; o < 16 * RB * kPer; o += kThreads) {
      const int t = o / kPer, c = (o % kPer) * 8, col = n0 + c;
      const int slot = t < T ? slots.slot[i][t] : 255;
      const bool mine = slot != 255 && col < p.f;
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = mine && bias ? static_cast<float>(bias[col + j]) : 0.0f;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const float *part = s_part + (s * 16 * RB + t) * kLd + c;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += part[j];
      }
      const size_t row = static_cast<size_t>(t) * p.k + (mine ? slot : 0);
      float top = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = mine ? gelu_erf(v[j]) : 0.0f;
        top = fmaxf(top, fabsf(v[j]));
      }
      if constexpr (kFp8) {
#pragma unroll
        for (int x = 8; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
        float inverse;
        const float scale = block_scale(top, &inverse);
        if (mine) {
          if ((o & 15) == 0) p.h_scales[row * FB + col / kScaleBlock] = scale;
          *reinterpret_cast<int2v *>(static_cast<uint8_t *>(p.h) + row * p.f + col) =
              int2v{pack_fp8(v[0] * inverse, v[1] * inverse, v[2] * inverse, v[3] * inverse),
                    pack_fp8(v[4] * inverse, v[5] * inverse, v[6] * inverse, v[7] * inverse)};
        }
      } else if (mine) {
        half8 o8;
#pragma unroll
        for (int j = 0; j < 8; ++j) o8[j] = static_cast<half_t>(v[j]);
        *reinterpret_cast<half8 *>(static_cast<half_t *>(p.h) + row * p.f + col) = o8;
      }
    }
  }
}

// 16 columns of the output, all chosen experts; the wavefronts cut the experts' K among them.  A token's results of an
// expert are scaled by its score (and the blocks' scales) as they are added.
template <bool kFp8, int RB>
__global__ void __launch_bounds__(kThreads, RB == 1 ? 4 : 2)
few_layer_down_kernel(FewLayerArgs p) {
  constexpr int kUnroll = RB == 1 ? 3 : 2, kLd = 16 + 4;
  __shared__ Slots slots;
  __shared__ float s_part[kWaves][16 * RB][kLd];
  const int T = p.tokens, n = T * p.k;
  for (int q = threadIdx.x; q < n; q += kThreads) {
    const int64_t e = p.idx[q];
    slots.e[q] = e >= 0 && e < p.E ? static_cast<int>(e) : p.E;
    slots.score[q] = static_cast<float>(p.score[q]);
  }
  __syncthreads();
  const int n_act = slots.build(n, p.k, p.E);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g = lane >> 4, n0 = blockIdx.x * 16;
  const int row_bytes = p.f * (kFp8 ? 1 : 2), steps = (row_bytes + 127) / 128;
  const int KB = scale_blocks(p.f), NB = scale_blocks(p.d);
  const int count = steps > wave ? (steps - wave + kWaves - 1) / kWaves : 0;           // of an expert: steps wave, wave + 8, ...
  const int total = count * n_act;
  const int col = n0 + r16 < p.d ? n0 + r16 : p.d - 1;
  float4v acc[RB];
#pragma unroll
  for (int b = 0; b < RB; ++b) acc[b] = float4v{0, 0, 0, 0};

  // the item that is fetched next: step `at` of chosen expert `i`
  int i = 0, at = wave;
  const uint8_t *w = nullptr, *h[RB];
  const float *sb = nullptr, *sh[RB];
  float score[RB];
  bool chose[RB], any[RB];                         // this lane's token did, one of the 16 did
  auto expert = [&]() __attribute__((always_inline)) {
    const int e = __builtin_amdgcn_readfirstlane(slots.act[i]);
    w = static_cast<const uint8_t *>(p.w2) + (static_cast<size_t>(e) * p.d + col) * row_bytes;
    if constexpr (kFp8) sb = p.s2 + (static_cast<size_t>(e) * NB + n0 / kScaleBlock) * KB;
    // lanes of tokens that did not choose it read a row of one that did
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      const int t = 16 * b + r16, slot = t < T ? slots.slot[i][t] : 255;
      chose[b] = slot != 255;
      const unsigned long long who = __ballot(chose[b]);
      any[b] = who != 0;
      const int row = chose[b] ? t * p.k + slot : 0;
      const int shared = __builtin_amdgcn_readlane(row, who ? __ffsll(who) - 1 : 0);
      const size_t r = static_cast<size_t>(chose[b] ? row : shared);
      score[b] = chose[b] ? slots.score[row] : 0.0f;
      h[b] = static_cast<const uint8_t *>(p.h) + r * row_bytes;
      if constexpr (kFp8) sh[b] = p.h_scales + r * KB;
    }
  };
  int8v wf[2][kUnroll], hf[2][kUnroll][RB];
  float sf[2][kUnroll][RB];
  bool mine[2][kUnroll][RB];
  auto fetch = [&](int q, auto B_) __attribute__((always_inline)) {        // items q ...; past the last one nothing new
    constexpr int buf = decltype(B_)::value;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (q + u < total) {                         // uniform
        if (at == wave) expert();
        wf[buf][u] = piece(w, at * 128 + 32 * g, row_bytes);
        const float b_scale = kFp8 ? sb[at] : 1.0f;
#pragma unroll
        for (int b = 0; b < RB; ++b) {
          mine[buf][u][b] = chose[b];
          sf[buf][u][b] = score[b];
          if (any[b]) {                            // uniform
            hf[buf][u][b] = piece(h[b], at * 128 + 32 * g, row_bytes);
            if constexpr (kFp8) sf[buf][u][b] *= sh[b][at] * b_scale;
          }
        }
        at += kWaves;
        if (at >= steps) {
          at = wave;
          ++i;
        }
      }
    }
  };
  auto multiply = [&](int q, auto B_) __attribute__((always_inline)) {
    constexpr int buf = decltype(B_)::value;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (q + u < total) {                         // uniform
#pragma unroll
        for (int b = 0; b < RB; ++b) {
          const float4v part = product<kFp8>(wf[buf][u], hf[buf][u][b]);
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[b][j] = mine[buf][u][b] ? fmaf(part[j], sf[buf][u][b], acc[b][j]) : acc[b][j];
        }
      }
    }
  };
  if (total > 0) {
    constexpr std::integral_constant<int, 0> even{};
    constexpr std::integral_constant<int, 1> odd{};
    fetch(0, even);
    for (int q = 0; q < total; q += 2 * kUnroll) {
      fetch(q + kUnroll, odd);
      __builtin_amdgcn_sched_barrier(0);
      multiply(q, even);
      __builtin_amdgcn_sched_barrier(0);
      fetch(q + 2 * kUnroll, even);
      __builtin_amdgcn_sched_barrier(0);
      multiply(q + kUnroll, odd);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
#pragma unroll
  for (int b = 0; b < RB; ++b) *reinterpret_cast<float4v *>(&s_part[wave][16 * b + r16][4 * g]) = acc[b];
  __syncthreads();
  for (int o = threadIdx.x; o < T * 16; o += kThreads) {
    const int t = o / 16, c = n0 + o % 16;
    if (c >= p.d) continue;
    float v = 0.0f;
    for (int s = 0; s < p.k; ++s) {
      const int e = slots.e[t * p.k + s];
      if (e < p.E && p.b2) v = fmaf(slots.score[t * p.k + s], static_cast<float>(p.b2[static_cast<size_t>(e) * p.d + c]), v);
    }
#pragma unroll
    for (int x = 0; x < kWaves; ++x) v += s_part[x][t][o % 16];
    p.out[static_cast<size_t>(t) * p.d + c] = static_cast<half_t>(v);
  }
}
}  // namespace

bool few_layer_fits(int tokens, int d, int f, int E, int k) {
  return tokens >= 1 && tokens <= kFewTokens && d > 0 && f > 0 && d % 64 == 0 && f % 64 == 0 && E >= 1 && E <= 1024 && k >= 1 &&
         k <= kMaxTopK && k <= E;
}

namespace {

template <int kIn, int RB>
int launch_up(const FewLayerArgs &p, bool gated, size_t gate_bytes, hipStream_t st) {
  constexpr int BN = kIn == kHalf ? 64 : 128, KS = kIn == kHalf ? 8 : 4;
  const size_t part = sizeof(float) * KS * 16 * RB * (BN + 4), lds = gate_bytes > part ? gate_bytes : part;
  auto kernel = few_layer_up_kernel<kIn, RB>;
  if (lds > 65536 - sizeof(Slots)) {
    hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(lds));
    if (e != hipSuccess) return fail(CCF_ERR_HIP, "few_layer: LDS attribute: %s", hipGetErrorString(e));
  }
  const int n = p.tokens * p.k;
  const long long units = static_cast<long long>(p.E < n ? p.E : n) * ((p.f + BN - 1) / BN);
  const int most = lds > 65536 || RB > 1 || kIn != kHalf ? 256 : 512;      // workgroups on the chip at once
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(units < most ? units : most)), dim3(kThreads), lds, st, p, gated);
  return check_launch("few_layer_up_kernel");
}

template <int RB>
int launch_few_layer(const FewLayerArgs &p, bool fp8, bool gated, size_t gate_bytes, hipStream_t st) {
  const int rc = !fp8 ? launch_up<kHalf, RB>(p, gated, gate_bytes, st)
                      : (p.x_codes ? launch_up<kCodes, RB>(p, gated, gate_bytes, st) : launch_up<kQuantise, RB>(p, gated, gate_bytes, st));
  if (rc) return rc;
  auto kernel = fp8 ? few_layer_down_kernel<true, RB> : few_layer_down_kernel<false, RB>;
  hipLaunchKernelGGL(kernel, dim3((p.d + 15) / 16), dim3(kThreads), 0, st, p);
  return check_launch("few_layer_down_kernel");
}

}  // namespace

int few_layer(const FewLayerArgs &p, bool fp8, ccf_stream_t stream) {
  const int nparts = (p.d + kPart - 1) / kPart;
  const long long chains = static_cast<long long>(p.tokens) * p.E * nparts;
  // gated in the first kernel: at most two chains to a thread, and operands that fit in LDS
  const bool here = chains <= 2 * kThreads && gate_lds(p.tokens, p.E, nparts).bytes <= 128 * 1024;
  if (!here) {
    int tokens_per_wg = 0;
    if (int rc = gate_forward(p.x, p.wg, p.bg, p.tokens, p.d, p.E, p.k, CCF_F16, p.idx, p.score, nullptr, stream, nullptr, 0,
                              &tokens_per_wg))
      return rc;
  }
  const size_t gate_bytes = here ? gate_lds(p.tokens, p.E, nparts).bytes : 0;
  return p.tokens > 16 ? launch_few_layer<2>(p, fp8, !here, gate_bytes, as_stream(stream))
                       : launch_few_layer<1>(p, fp8, !here, gate_bytes, as_stream(stream));
}

}  // namespace ccf
