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
// Workgroups start their sums at K places of their own, which go by the column: started together, they read the same bytes
// of rows a power of two apart, and few of the memory's channels (XXX).
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

enum { kHalf = 0, kCodes = 1, kQuantise = 2 };     // fp16 weights; e4m3 ones, with rows in 8 bits or quantised here into LDS

__device__ __forceinline__ int8v join(int4v lo, int4v hi) { return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7); }

// 16 columns (w) by 16 tokens (x) over the 128 bytes of a step: in 8 bits from zero, since a scale follows, else onto c.
template <bool kFp8>
__device__ __forceinline__ float4v product(int8v w, int8v x, float4v c = float4v{0, 0, 0, 0}) {
  if constexpr (kFp8) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, float4v{0, 0, 0, 0}, 0, 0, 0, 0, 0, 0);
  } else {
    typedef _Float16 half16 __attribute__((ext_vector_type(16)));
    const half16 a = __builtin_bit_cast(half16, w), b = __builtin_bit_cast(half16, x);
    const half8 a0 = __builtin_shufflevector(a, a, 0, 1, 2, 3, 4, 5, 6, 7), a1 = __builtin_shufflevector(a, a, 8, 9, 10, 11, 12, 13, 14, 15);
    const half8 b0 = __builtin_shufflevector(b, b, 0, 1, 2, 3, 4, 5, 6, 7), b1 = __builtin_shufflevector(b, b, 8, 9, 10, 11, 12, 13, 14, 15);
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, b0, c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, b1, c, 0, 0, 0);
  }
}

// 32 bytes of a lane's row, 16 from byte `in_step` of the step on and 16 from 64 bytes further, so that the 4 lanes of a row
// read 64 consecutive bytes at a time; zeros behind the end of the row's `bytes`, which begins at base + row.  A
// step is the 128 bytes (`span` times that) that the wavefront reads of every row; it and base are the wavefront's own.
__device__ __forceinline__ int8v piece(const uint8_t *base, uint32_t row, int step, int in_step, int bytes, int span = 1) {
  const uint8_t *at = base + step * 128;
  if ((step + span) * 128 <= bytes) {
    const int4v *both = reinterpret_cast<const int4v *>(at + (row + in_step));
    return join(both[0], both[4]);
  }
  const int left = bytes - step * 128 - in_step;
  const int4v *zeros = &kZeros16;
  const int4v *lo = left > 0 ? reinterpret_cast<const int4v *>(at + (row + in_step)) : zeros;
  const int4v *hi = left > 64 ? reinterpret_cast<const int4v *>(at + (row + in_step) + 64) : zeros;
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

// LDS of the gate: a slice of the expert rows (32 elements of every part), token rows, part sums, logits
struct GateLds {
  int x, part, logit, bytes;
};
constexpr int kSliceRow = 80;                      // a part's 64 bytes of a slice + 16: bank spread
constexpr int kGateChains = 512;                   // most parts of expert rows: their pieces are on their way in registers
__host__ __device__ inline GateLds gate_lds(int T, int E, int nparts) {
  GateLds l;
  l.x = E * nparts * kSliceRow;
  l.part = l.x + T * nparts * 256;
  l.logit = l.part + 4 * T * E * (nparts + 1);
  l.bytes = (l.logit + 4 * T * (E + 1) + 15) / 16 * 16;
  return l;
}

// The gate's choice for all tokens: chains of fused multiply-adds over parts of 128 elements from zero, the parts' sums in
// ascending order, the bias last, one rounding to fp16.  The expert rows are loaded at once, 16 bytes at a time, into
// registers and pass through LDS in four slices, so that they leave room for a second workgroup on the CU.  Token rows lie
// in LDS in 16-byte pieces, piece c of part i at c ^ (i % 16), so that lanes on neighbouring parts read other banks.
__device__ __forceinline__ void gate_here(const FewLayerArgs &p, char *s_raw, Slots &slots) {
  const int T = p.tokens, d = p.d, E = p.E, k = p.k, nparts = (d + kPart - 1) / kPart, chains = E * nparts;
  const GateLds at = gate_lds(T, E, nparts);
  const FastDiv by_parts(nparts), by_chains(chains), by_experts(E);
  float *s_part = reinterpret_cast<float *>(s_raw + at.part), *s_logit = reinterpret_cast<float *>(s_raw + at.logit);
  constexpr int kSlices = 4, kPer = kGateChains * 4 / kThreads;            // pieces of a slice to a thread
  half8 piece_of[kSlices][kPer];
#pragma unroll
  for (int s = 0; s < kSlices; ++s)
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int q = i * kThreads + threadIdx.x, chain = q >> 2, e = by_parts.div(chain);
      const int kk = (chain - e * nparts) * kPart + s * 32 + (q & 3) * 8;
      piece_of[s][i] = half8{0, 0, 0, 0, 0, 0, 0, 0};
      if (chain < chains && kk < d) piece_of[s][i] = *reinterpret_cast<const half8 *>(p.wg + static_cast<size_t>(e) * d + kk);
    }
  float bias = 0.0f;                               // of the logit that this thread adds up
  if (p.bg && static_cast<int>(threadIdx.x) < T * E) bias = static_cast<float>(p.bg[threadIdx.x - by_experts.div(threadIdx.x) * E]);
  const int x_pieces = T * nparts * 16;
#pragma unroll 4
  for (int q = threadIdx.x; q < x_pieces; q += kThreads) {
    const int i = q >> 4, t = by_parts.div(i), c = q & 15, kk = (i - t * nparts) * kPart + c * 8;
    half8 v = half8{0, 0, 0, 0, 0, 0, 0, 0};
    if (kk < d) v = *reinterpret_cast<const half8 *>(p.x + static_cast<size_t>(t) * d + kk);
    *reinterpret_cast<half8 *>(s_raw + at.x + i * 256 + ((c ^ (i & 15)) << 4)) = v;
  }
  // a thread's chains (the caller sees to it that two are enough)
  constexpr int kChains = 2;
  float acc[kChains];
  int chain_of[kChains], x_of[kChains], len_of[kChains];
  bool live[kChains];
#pragma unroll
  for (int j = 0; j < kChains; ++j) {
    const int q = j * kThreads + threadIdx.x, t = by_chains.div(q);
    live[j] = q < T * chains;
    chain_of[j] = q - t * chains;
    const int part = chain_of[j] - by_parts.div(chain_of[j]) * nparts;
    x_of[j] = t * nparts + part;
    len_of[j] = d - part * kPart;
    acc[j] = 0.0f;
  }
#pragma unroll
  for (int s = 0; s < kSlices; ++s) {
    if (s) __syncthreads();                        // the last slice is read
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int q = i * kThreads + threadIdx.x, chain = q >> 2;
      if (chain < chains) *reinterpret_cast<half8 *>(s_raw + chain * kSliceRow + (q & 3) * 16) = piece_of[s][i];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kChains; ++j) {
      if (!live[j]) continue;
      const char *wr = s_raw + chain_of[j] * kSliceRow, *xr = s_raw + at.x + x_of[j] * 256;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const half8 wv = *reinterpret_cast<const half8 *>(wr + c * 16);
        const half8 xv = *reinterpret_cast<const half8 *>(xr + (((s * 4 + c) ^ (x_of[j] & 15)) << 4));
        if (s * 32 + c * 8 < len_of[j]) {
#pragma unroll
          for (int i = 0; i < 8; ++i) acc[j] = __builtin_fmaf(static_cast<float>(xv[i]), static_cast<float>(wv[i]), acc[j]);
        }
      }
    }
  }
#pragma unroll
  for (int j = 0; j < kChains; ++j)
    if (live[j]) {
      const int row = by_parts.div(x_of[j]) * E + by_parts.div(chain_of[j]);           // token, expert
      s_part[row * (nparts + 1) + x_of[j] - by_parts.div(x_of[j]) * nparts] = acc[j];
    }
  __syncthreads();
  for (int i = threadIdx.x; i < T * E; i += kThreads) {
    const float *ps = s_part + i * (nparts + 1);
    const int t = by_experts.div(i), e = i - t * E;
    float v = ps[0];
#pragma unroll 16
    for (int q = 1; q < nparts; ++q) v = v + ps[q];
    if (p.bg) v = v + (i < kThreads ? bias : static_cast<float>(p.bg[e]));
    s_logit[t * (E + 1) + e] = round_to<half_t>(v);
  }
  __syncthreads();
  auto select = [&](auto KS_) __attribute__((always_inline)) {
    constexpr int KS = decltype(KS_)::value;       // most entries of a list
    const int t = threadIdx.x;
    Best<KS> best;
    best.clear();
#pragma unroll 8
    for (int e = 0; e < E; ++e) best.offer(s_logit[t * (E + 1) + e], e, k);
    int64_t idx[KS];
    half_t score[KS];
    best.template write<half_t>(0, k, idx, score);
#pragma unroll
    for (int s = 0; s < KS; ++s)
      if (s < k) {
        slots.e[t * k + s] = best.id[s];
        if (blockIdx.x == 0) {                     // for the second kernel
          p.idx[t * k + s] = idx[s] < E ? idx[s] : -1;
          p.score[t * k + s] = score[s];
        }
      }
  };
  if (static_cast<int>(threadIdx.x) < T) {
    if (k <= 2) select(std::integral_constant<int, 2>{});
    else select(std::integral_constant<int, kMaxTopK>{});
  }
}

// Tokens in 8 bits in LDS: rows of d codes, 16 bytes apart beyond that (16 rows on as many banks), then their scales.
struct RowsLds {
  int ld, scales, bytes;
};
__host__ __device__ inline RowsLds rows_lds(int T, int d) {
  RowsLds l;
  l.ld = (d + 127) / 128 * 128 + 16;
  l.scales = T * l.ld;
  l.bytes = (l.scales + 4 * T * scale_blocks(d) + 15) / 16 * 16;
  return l;
}

// As ccf_quantize_rows: 16 lanes to a block of 128.  Codes behind the end of K are zeros.  The caller's barrier follows.
__device__ __forceinline__ void quantise_here(const FewLayerArgs &p, char *s_rows, const RowsLds &at) {
  const int blocks = scale_blocks(p.d);
  const FastDiv by_blocks(blocks);
  const int pieces = p.tokens * blocks * 16;
  constexpr int kAhead = 4;                        // loads on their way
  for (int q0 = threadIdx.x; q0 < pieces; q0 += kAhead * kThreads) {
    half8 v[kAhead];
    int row[kAhead], col[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const int q = q0 + a * kThreads, i = q >> 4;
      row[a] = by_blocks.div(i);
      col[a] = (i - row[a] * blocks) * kScaleBlock + (q & 15) * 8;
      v[a] = half8{0, 0, 0, 0, 0, 0, 0, 0};
      if (q < pieces && col[a] < p.d) v[a] = *reinterpret_cast<const half8 *>(p.x + static_cast<size_t>(row[a]) * p.d + col[a]);
    }
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const int q = q0 + a * kThreads;
      float top = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(static_cast<float>(v[a][j])));
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
      float inverse;
      const float scale = block_scale(top, &inverse);
      auto four = [&](int j) {
        return pack_fp8(static_cast<float>(v[a][j]) * inverse, static_cast<float>(v[a][j + 1]) * inverse,
                        static_cast<float>(v[a][j + 2]) * inverse, static_cast<float>(v[a][j + 3]) * inverse);
      };
      if (q >= pieces) continue;
      *reinterpret_cast<int2v *>(s_rows + row[a] * at.ld + col[a]) = int2v{four(0), four(4)};
      if ((q & 15) == 0) *reinterpret_cast<float *>(s_rows + at.scales + 4 * (q >> 4)) = scale;
    }
  }
}

// 16 RB tokens; a workgroup's columns: 64 of fp16 weights, whose K all eight wavefronts cut among them, 128 in 8 bits, four
// wavefronts to either half.
template <int kIn, int RB>
__global__ void __launch_bounds__(kThreads, RB == 1 && kIn != kCodes ? 4 : 2)
few_layer_up_kernel(FewLayerArgs p, bool gated) {
  constexpr bool kFp8 = kIn != kHalf;
  constexpr int CT = 4, CS = kFp8 ? 2 : 1, KS = kWaves / CS, BN = 16 * CT * CS, kLd = BN + 4;
  extern __shared__ __attribute__((aligned(16))) char s_all[];             // kQuantise: the rows' codes and scales first
  __shared__ Slots slots;
  const int T = p.tokens, n = T * p.k;
  const RowsLds rows_at = rows_lds(kIn == kQuantise ? T : 0, p.d);
  char *s_raw = s_all + rows_at.bytes;
  if constexpr (kIn == kQuantise) quantise_here(p, s_all, rows_at);
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
  const uint8_t *x = kIn == kCodes ? p.x_codes : reinterpret_cast<const uint8_t *>(p.x);

  const int units = n_act * blocks;
  if (static_cast<int>(blockIdx.x) >= units) return;
  // a wavefront without a step takes part all the same: a step of another one's, not multiplied
  const int turns = count > 0 ? count : 1;

  // the item that is fetched next: the q-th of this wavefront's steps in unit u.  Its steps come in turn, from the one on
  // that the unit's columns start at.
  int u_next = blockIdx.x, q_next = 0, from_next = 0;
  const uint8_t *w = nullptr;
  const float *sb = nullptr;
  auto aim = [&]() __attribute__((always_inline)) {
    const int i = u_next / blocks, block = u_next - i * blocks;
    int c0 = block * BN + cs * 16 * CT;
    c0 = c0 < p.f ? c0 : p.f - 16 * CT;            // (f is a multiple of 64) the second half of 128 columns: never stored
    const int e = __builtin_amdgcn_readfirstlane(slots.act[i]);
    from_next = block % turns;
    w = static_cast<const uint8_t *>(p.w1) + (static_cast<size_t>(e) * p.f + c0) * row_bytes;
    if constexpr (kFp8) sb = p.s1 + (static_cast<size_t>(e) * FB + c0 / kScaleBlock) * KB;
  };
  auto step_of = [&](int from, int q) {
    const int at = from + q, st = ks + (at < turns ? at : at - turns) * KS;
    return st < steps ? st : steps - 1;
  };
  int8v wf[2][CT], xf[2][RB];
  float sx[2][RB], sw[2];
  auto fetch = [&](auto B_) __attribute__((always_inline)) {
    constexpr int buf = decltype(B_)::value;
    if (u_next >= units) return;                   // uniform
    const int st = step_of(from_next, q_next);
#pragma unroll
    for (int c = 0; c < CT; ++c) wf[buf][c] = piece(w + static_cast<size_t>(16 * c) * row_bytes, r16 * row_bytes, st, 16 * g, row_bytes);
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      if constexpr (kIn == kCodes) {
        xf[buf][b] = piece(x, token[b] * row_bytes, st, 16 * g, row_bytes);
        sx[buf][b] = p.x_scales[token[b] * KB + st];
      } else if constexpr (kIn == kHalf) {
        xf[buf][b] = piece(x, token[b] * row_bytes, st, 16 * g, row_bytes);
      }
    }
    if constexpr (kFp8) sw[buf] = sb[st];
    if (++q_next == turns) {
      q_next = 0;
      u_next += gridDim.x;
      if (u_next < units) aim();
    }
  };
  // the unit that is computed, its item; eight consecutive columns of a token to a thread in its epilogue
  constexpr int kPer = BN / 8;
  static_assert(16 * RB * kPer <= kThreads, "a thread has at most one piece of the epilogue");
  const int t_mine = threadIdx.x / kPer, c_mine = threadIdx.x % kPer * 8;
  int u = blockIdx.x, q = 0, from = 0, i = 0, n0 = 0, slot = 255;
  half8 bias;
  float4v acc[CT][RB];
  auto begin = [&]() __attribute__((always_inline)) {
    i = u / blocks;
    const int block = u - i * blocks, e = __builtin_amdgcn_readfirstlane(slots.act[i]);
    from = block % turns;
    n0 = block * BN;
    slot = t_mine < T && n0 + c_mine < p.f ? slots.slot[i][t_mine] : 255;
    bias = half8{0, 0, 0, 0, 0, 0, 0, 0};
    if (slot != 255 && p.b1) bias = *reinterpret_cast<const half8 *>(p.b1 + static_cast<size_t>(e) * p.f + n0 + c_mine);
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int b = 0; b < RB; ++b) acc[c][b] = float4v{0, 0, 0, 0};
  };
  auto multiply = [&](auto B_) __attribute__((always_inline)) {
    constexpr int buf = decltype(B_)::value;
    if (count == 0) return;                        // uniform
    const int st = step_of(from, q);
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      float s = 1.0f;
      if constexpr (kIn == kQuantise) {
        const char *row = s_all + token[b] * rows_at.ld + st * 128 + 16 * g;
        xf[buf][b] = join(*reinterpret_cast<const int4v *>(row), *reinterpret_cast<const int4v *>(row + 64));
        s = *reinterpret_cast<const float *>(s_all + rows_at.scales + 4 * (token[b] * KB + st));
      } else if constexpr (kIn == kCodes) {
        s = sx[buf][b];
      }
      if constexpr (kFp8) s *= sw[buf];
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        const float4v part = product<kFp8>(wf[buf][c], xf[buf][b], acc[c][b]);
        if constexpr (kFp8) {
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[c][b][j] = fmaf(part[j], s, acc[c][b][j]);
        } else {
          acc[c][b] = part;
        }
      }
    }
  };
  // the unit's end: the wavefronts' sums meet, GELU, h
  auto finish = [&]() __attribute__((always_inline)) {
    __syncthreads();                               // the gate's or the last unit's LDS is read
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int b = 0; b < RB; ++b)
        *reinterpret_cast<float4v *>(s_part + (ks * 16 * RB + 16 * b + r16) * kLd + (cs * CT + c) * 16 + 4 * g) = acc[c][b];
    __syncthreads();
    if (t_mine >= 16 * RB) return;
    const bool mine = slot != 255;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = static_cast<float>(bias[j]);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const float *part = s_part + (s * 16 * RB + t_mine) * kLd + c_mine;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += part[j];
    }
    const size_t row = static_cast<size_t>(t_mine) * p.k + (mine ? slot : 0);
    const int col = n0 + c_mine;
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
        if (threadIdx.x % 16 == 0) p.h_scales[row * FB + col / kScaleBlock] = scale;
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
  };
  // one item, with the next one's loads (of the next unit, at a unit's end) on their way; whether it was the last
  auto item = [&](auto B_) __attribute__((always_inline)) {
    constexpr int buf = decltype(B_)::value;
    fetch(std::integral_constant<int, buf ^ 1>{});
    __builtin_amdgcn_sched_barrier(0);
    multiply(B_);
    __builtin_amdgcn_sched_barrier(0);
    if (++q < turns) return false;
    finish();
    q = 0;
    u += gridDim.x;
    if (u >= units) return true;
    begin();
    return false;
  };
  constexpr std::integral_constant<int, 0> even{};
  constexpr std::integral_constant<int, 1> odd{};
  aim();
  fetch(even);
  begin();
  while (!item(even) && !item(odd)) {
  }
}

// CW columns of the output, all chosen experts; the wavefronts cut the experts' K among them.  With CW < 16 the 16 rows of a
// product are CW columns on 16 / CW steps of K at a time, each product with the tokens of one of them: a narrow tile loads as
// many bytes as a wide one, and there are enough of them for the chip.  A token's results of an expert are scaled by its
// score (and the blocks' scales) as they are added.
//
// Sixteen wavefronts to a workgroup, of which there is one on a CU; eight where a step has the fragments of several blocks of
// tokens or steps, which need twice the registers.
constexpr int down_waves(int RB, int CW) { return RB == 1 && CW == 16 ? 16 : 8; }

template <bool kFp8, int RB, int CW>
__global__ void __launch_bounds__(down_waves(RB, CW) * 64, down_waves(RB, CW) / 4)
few_layer_down_kernel(FewLayerArgs p) {
  constexpr int kDownWaves = down_waves(RB, CW), kLd = 16 + 4, KG = 16 / CW;
  constexpr int kUnroll = RB * KG > 4 ? 1 : 2;     // items fetched at a time
  __shared__ Slots slots;
  __shared__ float s_part[kDownWaves][16 * RB][kLd];
  const int T = p.tokens, n = T * p.k;
  for (int q = threadIdx.x; q < n; q += kDownWaves * 64) {
    const int64_t e = p.idx[q];
    slots.e[q] = e >= 0 && e < p.E ? static_cast<int>(e) : p.E;
    slots.score[q] = static_cast<float>(p.score[q]);
  }
  __syncthreads();
  const int n_act = slots.build(n, p.k, p.E);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g = lane >> 4, n0 = blockIdx.x * CW;
  const int mine_k = g * 4 / CW;                   // of the KG steps, the one that this lane's results (rows 4 g ..) are of
  const int row_bytes = p.f * (kFp8 ? 1 : 2), steps = (row_bytes + 128 * KG - 1) / (128 * KG);         // of KG blocks of 128 bytes
  const int KB = scale_blocks(p.f), NB = scale_blocks(p.d);
  const int count = steps > wave ? (steps - wave + kDownWaves - 1) / kDownWaves : 0;   // of an expert: steps wave, wave + 16, ...
  const int total = count * n_act;
  float4v acc[RB];
#pragma unroll
  for (int b = 0; b < RB; ++b) acc[b] = float4v{0, 0, 0, 0};

  // the item that is fetched next: step `at` of chosen expert `i`
  const int from = count > 0 ? wave + blockIdx.x % count * kDownWaves : 0;
  int i = 0, at = from;
  const uint8_t *w = nullptr, *h = static_cast<const uint8_t *>(p.h);
  const float *sb = nullptr;
  uint32_t h_row[RB];
  float score[RB];
  bool chose[RB], any[RB];                         // this lane's token did, one of the 16 did
  auto expert = [&]() __attribute__((always_inline)) {
    const int e = __builtin_amdgcn_readfirstlane(slots.act[i]);
    w = static_cast<const uint8_t *>(p.w2) + (static_cast<size_t>(e) * p.d + n0) * row_bytes;
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
      h_row[b] = static_cast<uint32_t>(chose[b] ? row : shared);
      score[b] = chose[b] ? slots.score[row] : 0.0f;
    }
  };
  // the biases' part of this thread's output
  const int t_mine = threadIdx.x / CW, c_mine = threadIdx.x % CW;
  static_assert(16 * RB * CW <= kDownWaves * 64, "a thread has at most one output");
  float sum = 0.0f;
  if (p.b2 && t_mine < T) {
#pragma unroll 2
    for (int s = 0; s < p.k; ++s) {
      const int e = slots.e[t_mine * p.k + s];
      if (e < p.E) sum = fmaf(slots.score[t_mine * p.k + s], static_cast<float>(p.b2[static_cast<size_t>(e) * p.d + n0 + c_mine]), sum);
    }
  }
  int8v wf[2][kUnroll], hf[2][kUnroll][RB][KG];
  float sf[2][kUnroll][RB];
  bool mine[2][kUnroll][RB];
  auto fetch = [&](int q, auto B_) __attribute__((always_inline)) {        // items q ...; past the last one nothing new
    constexpr int buf = decltype(B_)::value;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (q + u < total) {                         // uniform
        if (at == from) expert();
        wf[buf][u] = piece(w, r16 % CW * row_bytes, at * KG, r16 / CW * 128 + 16 * g, row_bytes, KG);
        const int kb = at * KG + mine_k < KB ? at * KG + mine_k : KB - 1;
        const float b_scale = kFp8 ? sb[kb] : 1.0f;
#pragma unroll
        for (int b = 0; b < RB; ++b) {
          mine[buf][u][b] = chose[b];
          sf[buf][u][b] = score[b];
          if (any[b]) {                            // uniform
#pragma unroll
            for (int j = 0; j < KG; ++j) hf[buf][u][b][j] = piece(h, h_row[b] * row_bytes, at * KG + j, 16 * g, row_bytes);
            if constexpr (kFp8) sf[buf][u][b] *= p.h_scales[h_row[b] * KB + kb] * b_scale;
          }
        }
        at += kDownWaves;
        if (at >= steps) at = wave;
        if (at == from) ++i;
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
          float4v part = product<kFp8>(wf[buf][u], hf[buf][u][b][0]);
#pragma unroll
          for (int j = 1; j < KG; ++j) {
            const float4v other = product<kFp8>(wf[buf][u], hf[buf][u][b][j]);
            part = mine_k == j ? other : part;
          }
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
  if (t_mine < T) {
#pragma unroll
    for (int x = 0; x < kDownWaves; ++x)
#pragma unroll
      for (int j = 0; j < KG; ++j) sum += s_part[x][t_mine][j * CW + c_mine];
    p.out[static_cast<size_t>(t_mine) * p.d + n0 + c_mine] = static_cast<half_t>(sum);
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
  const size_t part = sizeof(float) * KS * 16 * RB * (BN + 4);
  const size_t lds = (gate_bytes > part ? gate_bytes : part) + (kIn == kQuantise ? rows_lds(p.tokens, p.d).bytes : rows_lds(0, p.d).bytes);
  auto kernel = few_layer_up_kernel<kIn, RB>;
  if (lds > 65536 - sizeof(Slots)) {
    hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(lds));
    if (e != hipSuccess) return fail(CCF_ERR_HIP, "few_layer: LDS attribute: %s", hipGetErrorString(e));
  }
  const int n = p.tokens * p.k;
  const long long units = static_cast<long long>(p.E < n ? p.E : n) * ((p.f + BN - 1) / BN);
  const int most = lds + sizeof(Slots) > 80 * 1024 || RB > 1 || kIn == kCodes ? 256 : 512;              // workgroups on the chip at once
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(units < most ? units : most)), dim3(kThreads), lds, st, p, gated);
  return check_launch("few_layer_up_kernel");
}

template <bool kFp8, int RB>
int launch_down(const FewLayerArgs &p, hipStream_t st) {
  // the widest tiles of which there are enough for the chip
  const int cw = p.d >= 16 * 256 ? 16 : (p.d >= 8 * 256 ? 8 : 4);
  auto kernel = cw == 16 ? few_layer_down_kernel<kFp8, RB, 16> : (cw == 8 ? few_layer_down_kernel<kFp8, RB, 8> : few_layer_down_kernel<kFp8, RB, 4>);
  hipLaunchKernelGGL(kernel, dim3(p.d / cw), dim3(down_waves(RB, cw) * 64), 0, st, p);
  return check_launch("few_layer_down_kernel");
}

template <int RB>
int launch_few_layer(const FewLayerArgs &p, bool fp8, bool gated, size_t gate_bytes, hipStream_t st) {
  const int rc = !fp8 ? launch_up<kHalf, RB>(p, gated, gate_bytes, st)
                      : (p.x_codes ? launch_up<kCodes, RB>(p, gated, gate_bytes, st) : launch_up<kQuantise, RB>(p, gated, gate_bytes, st));
  if (rc) return rc;
  return fp8 ? launch_down<true, RB>(p, st) : launch_down<false, RB>(p, st);
}

// What the first kernel may keep in LDS beside its part sums (70 KB at most) and the slots.
constexpr int kMaxGateLds = 64 * 1024, kMaxRowsLds = 72 * 1024;

}  // namespace

bool few_layer_quantises(int tokens, int d) { return rows_lds(tokens, d).bytes <= kMaxRowsLds; }

int few_layer(const FewLayerArgs &p, bool fp8, ccf_stream_t stream) {
  const int nparts = (p.d + kPart - 1) / kPart;
  const long long chains = static_cast<long long>(p.E) * nparts;
  // gated in the first kernel: its expert rows in registers, at most two chains to a thread, and operands that fit in LDS
  const bool here = chains <= kGateChains && p.tokens * chains <= 2 * kThreads &&
                    gate_lds(p.tokens, p.E, nparts).bytes <= kMaxGateLds;
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
