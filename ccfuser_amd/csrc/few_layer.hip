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
//   * no routing: a product's columns are the tokens themselves, 16 of them, whichever of them chose the expert, so
//     no rows are listed, moved or padded; what a token gets from an expert that it did not choose is dropped;
//   * the second kernel runs all chosen experts of its 16 columns into one sum, so nothing is left to combine.
//
// In 8 bits (e4m3, a scale per block of 128) rows of x are quantised where they are read, as ccf_quantize_rows does, and
// the first kernel's workgroups have the 128 columns of a scale of h.  Wavefronts cut K among them, each with a stream of
// operands of its own; their sums meet in LDS in a fixed order.
//
// One token, widths 4096 and 14336, two experts: 16 bits 45 + 38 us, 5.3 and 6.2 TB/s (the gate is 5 to 8 us of the first),
// 8 bits 31 + 22 us, 3.8 and 5.3 TB/s; 1 GiB copied by the framework 5.1.
#include "few_layer.h"
#include "gate_select.h"
#include "gelu.h"
#include "plan.h"

#include <type_traits>

namespace ccf {
namespace {

// Most tokens.  With 32 the layer of any size was as fast or faster (17 tokens, us, widths 1024 / 4096, 16 experts: 16 bits 117
// and 70, 8 bits 72 and 51; 4096 / 14336, 8 experts: 367 and 314, 212 and 213): by then most experts are chosen, and a product
// that works on all tokens whichever chose the expert moves more of them than of weights.
constexpr int kFewTokens = 16;
constexpr int kFewSlots = kFewTokens * kMaxTopK;
constexpr int kThreads = 512, kWaves = kThreads / 64;

__device__ const int4v kZeros16 = {0, 0, 0, 0};    // what lanes behind the end of K read

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

// Which experts have tokens, in ascending order, and which slot of a token each is; in LDS.
struct Slots {
  unsigned *mask;                                  // [32] of E <= 1024 experts
  int *act, *e;                                    // [n] the chosen experts; the tokens' choice
  float *score;                                    // [n]
  uint8_t *slot;                                   // [n][16] slot of token t that expert act[i] is, 255: none

  __host__ __device__ static int bytes(int n) { return 128 + n * (4 + 4 + 4 + kFewTokens); }
  __device__ __forceinline__ Slots(char *at, int n)
      : mask(reinterpret_cast<unsigned *>(at)), act(reinterpret_cast<int *>(at + 128)), e(act + n),
        score(reinterpret_cast<float *>(e + n)), slot(reinterpret_cast<uint8_t *>(score + n)) {}

  __device__ __forceinline__ int of(int i, int t) const { return slot[i * kFewTokens + t]; }
  __device__ __forceinline__ int rank(int expert) const {
    int r = __popc(mask[expert >> 5] & ((1u << (expert & 31)) - 1));
    for (int i = 0; i < expert >> 5; ++i) r += __popc(mask[i]);
    return r;
  }
  // all threads, behind a barrier after e and score were written; how many experts were chosen
  __device__ __forceinline__ int build(int n, int k, int E) {
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
      slot[r * kFewTokens + t] = static_cast<uint8_t>(q - t * k);
    }
    int total = 0;
    for (int i = 0; i < (E + 31) / 32; ++i) total += __popc(mask[i]);
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(total);
  }
};

// ---- a wavefront's stream of operands
//
// Weights and tokens go to LDS by direct loads into a ring of the wavefront's own, kDepth items deep, each item the weights
// (16 rows of 128 bytes: two loads of 8 whole lines) and the tokens of one product: no barrier, the wavefront waits for its
// oldest item by the number of loads that may still be in flight.  16-byte chunk c of row r lies at c ^ (r % 8); a lane's
// fragment is chunks g and g + 4 of row r16, of either operand.  (Loads into registers touch 64 bytes of 16 rows each:
// 2 GiB of weights streamed that way came at 5.5 to 5.9 TB/s and, with the non-temporal hint, 5.2, whole lines with it at
// 6.5 to 6.8.)
//
// The loads are asm for what the compiler does not know: which LDS reads they concern.  They write no register.
template <bool kNT>
__device__ __forceinline__ void load16_to_lds(const void *base, uint32_t offset, uint32_t at) {
  if constexpr (kNT)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(at), "v"(offset), "s"(base));
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(at), "v"(offset), "s"(base));
}
__device__ __forceinline__ void load16_to_lds(const void *src, uint32_t at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(at), "v"(src));
}
__device__ __forceinline__ void load4_to_lds(const void *base, uint32_t offset, uint32_t at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(at), "v"(offset), "s"(base));
}
// All but the newest n loads have landed.
template <int n>
__device__ __forceinline__ void loads_but() {
  static_assert(n >= 0 && n < 64, "vmcnt has six bits");
  __builtin_amdgcn_s_waitcnt(0x0f70 | (n & 15) | (n >> 4) << 14);
  asm volatile("" ::: "memory");
}
// The LDS reads so far have their values: their place may be loaded into.
__device__ __forceinline__ void reads_done() {
  __builtin_amdgcn_s_waitcnt(0xc07f);
  asm volatile("" ::: "memory");
}
__device__ __forceinline__ uint32_t lds_address(const char *p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) char *)p));
}
__device__ __forceinline__ int8v fragment(const char *tile, int r, int g) {
  const char *row = tile + r * 128;
  return join(*reinterpret_cast<const int4v *>(row + ((g ^ (r & 7)) << 4)), *reinterpret_cast<const int4v *>(row + (((g ^ (r & 7)) ^ 4) << 4)));
}
__device__ __forceinline__ float scalar_load(const float *p) { return *(const __attribute__((address_space(4))) float *)p; }

// Whether weights are loaded past the caches: where more passes before they are read again than the 256 MB Infinity Cache
// holds (few.hip has the measurements).
__device__ __forceinline__ bool pass_by(int n_act, int d, int f, bool fp8) {
  return 2.0f * static_cast<float>(n_act) * static_cast<float>(d) * static_cast<float>(f) * (fp8 ? 1.0f : 2.0f) >= 320e6f;
}

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
__device__ __forceinline__ void gate_here(const FewLayerArgs &p, char *s_raw, const Slots &slots) {
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

// The caller's codes, or as ccf_quantize_rows makes them, 16 lanes to a block of 128.  Codes behind the end of K are zeros.
// The caller's barrier follows.
__device__ __forceinline__ void rows_here(const FewLayerArgs &p, char *s_rows, const RowsLds &at) {
  const int blocks = scale_blocks(p.d);
  const FastDiv by_blocks(blocks);
  const int pieces = p.tokens * blocks * 16;
  if (p.x_codes) {
    const int chunks = blocks * 8;                 // of 16 bytes, to a row
    const FastDiv by_chunks(chunks);
#pragma unroll 4
    for (int q = threadIdx.x; q < p.tokens * chunks; q += kThreads) {
      const int t = by_chunks.div(q), c = (q - t * chunks) * 16;
      int4v v = int4v{0, 0, 0, 0};
      if (c < p.d) v = *reinterpret_cast<const int4v *>(p.x_codes + static_cast<size_t>(t) * p.d + c);
      *reinterpret_cast<int4v *>(s_rows + t * at.ld + c) = v;
    }
    for (int q = threadIdx.x; q < p.tokens * blocks; q += kThreads) reinterpret_cast<float *>(s_rows + at.scales)[q] = p.x_scales[q];
    return;
  }
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

// At most 8 NX tokens.  A workgroup's columns: 16 of fp16 weights, whose K its eight wavefronts
// cut among them, 128 in 8 bits, 16 to a wavefront: the columns of a scale of h.  It takes one such unit after the other, the
// next one's operands on their way.
template <bool kFp8, int NX>
struct UpShape {
  static constexpr int CS = kFp8 ? 8 : 1, KS = kWaves / CS, BN = 16 * CS, kLd = BN + 4;
  static constexpr int kLoads = 2 + (kFp8 ? 0 : NX), kItem = 1024 * kLoads, kDepth = kFp8 ? 4 : 2;
  static constexpr int kRing = kWaves * kDepth * kItem, kPart = 4 * KS * 16 * kLd;
};

template <bool kFp8, int NX>
__global__ void __launch_bounds__(kThreads, 4)
few_layer_up_kernel(FewLayerArgs p, bool gated, int ring_bytes) {
  using S = UpShape<kFp8, NX>;
  constexpr int KS = S::KS, BN = S::BN, kLd = S::kLd;
  // the rings (first the gate's), part sums, slots, in 8 bits the tokens' codes and scales
  extern __shared__ __attribute__((aligned(1024))) char s_all[];
  const int T = p.tokens, n = T * p.k;
  float *s_part = reinterpret_cast<float *>(s_all + ring_bytes);           // [KS][16][kLd]
  Slots slots(s_all + ring_bytes + S::kPart, n);
  const RowsLds rows_at = rows_lds(kFp8 ? T : 0, p.d);
  char *s_rows = s_all + ring_bytes + S::kPart + (Slots::bytes(n) + 15) / 16 * 16;
  if constexpr (kFp8) rows_here(p, s_rows, rows_at);
  if (gated) {
    for (int q = threadIdx.x; q < n; q += kThreads) {
      const int64_t e = p.idx[q];
      const bool valid = e >= 0 && e < p.E;
      slots.e[q] = valid ? static_cast<int>(e) : p.E;
      if (!valid && blockIdx.x == 0) p.idx[q] = -1;
    }
  } else {
    gate_here(p, s_all, slots);
  }
  __syncthreads();
  const int n_act = slots.build(n, p.k, p.E);

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g = lane >> 4, ks = wave % KS, cs = wave / KS;
  const int row_bytes = p.d * (kFp8 ? 1 : 2), steps = (row_bytes + 127) / 128, tail = row_bytes % 128;
  const int blocks = (p.f + BN - 1) / BN, KB = scale_blocks(p.d), FB = scale_blocks(p.f);
  const int count = steps > ks ? (steps - ks + KS - 1) / KS : 0;           // steps ks, ks + KS, ...
  const int units = n_act * blocks;
  if (static_cast<int>(blockIdx.x) >= units) return;
  // a wavefront without a step takes part all the same: a step of another one's, not multiplied
  const int turns = count > 0 ? count : 1;
  const bool nt = pass_by(n_act, p.d, p.f, kFp8);
  const char *ring = s_all + wave * (S::kDepth * S::kItem);
  const uint32_t ring_at = __builtin_amdgcn_readfirstlane(lds_address(ring));

  // this lane's loads: chunk (lane % 8) ^ (row % 8) of row 8 j + lane / 8 of a tile
  const int chunk = (lane & 7) ^ (lane >> 3);
  const uint32_t w_lane = (lane >> 3) * row_bytes + chunk * 16;
  uint32_t x_lane[NX];
#pragma unroll
  for (int j = 0; j < NX; ++j) {
    const int t = 8 * j + (lane >> 3);             // (two blocks of tokens have all 16 each)
    x_lane[j] = (t < T ? t : T - 1) * row_bytes + chunk * 16;
  }

  // the item that is loaded next: the q-th of this wavefront's steps in unit u
  int u_next = blockIdx.x, q_next = 0, slot_next = 0, ahead = 0;
  const uint8_t *w = nullptr;
  auto aim = [&]() __attribute__((always_inline)) {
    const int i = u_next / blocks, block = u_next - i * blocks;
    int c0 = block * BN + cs * 16;
    c0 = c0 < p.f ? c0 : p.f - 16;                 // (f is a multiple of 64) the second half of 128 columns: never stored
    const int e = __builtin_amdgcn_readfirstlane(slots.act[i]);
    w = static_cast<const uint8_t *>(p.w1) + (static_cast<size_t>(e) * p.f + c0) * row_bytes;
  };
  auto step_of = [&](int q) { return ks + q * KS < steps ? ks + q * KS : steps - 1; };
  auto load_item = [&]() __attribute__((always_inline)) {
    const int st = step_of(q_next);
    const uint8_t *base = w + st * 128, *base8 = base + static_cast<size_t>(8) * row_bytes;
    uint32_t at = ring_at + slot_next * S::kItem, lane_at = w_lane;
    // chunks behind the end of a row: its step's first one again, for codes that are zeros
    if (tail && st == steps - 1) lane_at -= chunk * 16 >= tail ? chunk * 16 : 0;
    if (nt) {
      load16_to_lds<true>(base, lane_at, at);
      load16_to_lds<true>(base8, lane_at, at + 1024);
    } else {
      load16_to_lds<false>(base, lane_at, at);
      load16_to_lds<false>(base8, lane_at, at + 1024);
    }
    if constexpr (!kFp8) {
      const uint8_t *x = reinterpret_cast<const uint8_t *>(p.x) + st * 128;
#pragma unroll
      for (int j = 0; j < NX; ++j) load16_to_lds<false>(x, x_lane[j], at + 2048 + 1024 * j);
    }
    ++ahead;
    slot_next = slot_next + 1 < S::kDepth ? slot_next + 1 : 0;
    if (++q_next == turns) {
      q_next = 0;
      u_next += gridDim.x;
      if (u_next < units) aim();
    }
  };
  // the unit that is computed, its item; eight consecutive columns of a token to a thread in its epilogue
  constexpr int kPer = BN / 8;
  static_assert(16 * kPer <= kThreads, "a thread has at most one piece of the epilogue");
  const int t_mine = threadIdx.x / kPer, c_mine = threadIdx.x % kPer * 8;
  int u = blockIdx.x, q = 0, i = 0, n0 = 0, slot = 255, place = 0;
  const float *sb = nullptr;
  half8 bias;
  float4v acc;
  auto begin = [&]() __attribute__((always_inline)) {
    i = u / blocks;
    const int block = u - i * blocks, e = __builtin_amdgcn_readfirstlane(slots.act[i]);
    n0 = block * BN;
    if constexpr (kFp8) sb = p.s1 + (static_cast<size_t>(e) * FB + block) * KB;
    slot = t_mine < T && n0 + c_mine < p.f ? slots.of(i, t_mine) : 255;
    bias = half8{0, 0, 0, 0, 0, 0, 0, 0};
    if (slot != 255 && p.b1) bias = *reinterpret_cast<const half8 *>(p.b1 + static_cast<size_t>(e) * p.f + n0 + c_mine);
    acc = float4v{0, 0, 0, 0};
  };
  // the unit's end: the wavefronts' sums meet, GELU, h
  auto finish = [&]() __attribute__((always_inline)) {
    __syncthreads();                               // the last unit's part sums are read
    *reinterpret_cast<float4v *>(s_part + (ks * 16 + r16) * kLd + cs * 16 + 4 * g) = acc;
    __syncthreads();
    if (t_mine >= 16) return;
    const bool mine = slot != 255;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = static_cast<float>(bias[j]);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const float *part = s_part + (s * 16 + t_mine) * kLd + c_mine;
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

  aim();
#pragma unroll
  for (int j = 0; j < S::kDepth; ++j)
    if (u_next < units) load_item();
  begin();
  while (true) {
    if (ahead == S::kDepth) loads_but<S::kLoads *(S::kDepth - 1)>();
    else loads_but<0>();                           // the last items: none are loaded behind them
    const char *at = ring + place * S::kItem;
    place = place + 1 < S::kDepth ? place + 1 : 0;
    const int st = step_of(q);
    const int8v wf = fragment(at, r16, g);
    int8v xf;
    float sx;
    if constexpr (kFp8) {
      const int t = r16 < T ? r16 : T - 1;
      const char *row = s_rows + t * rows_at.ld + st * 128 + 16 * g;
      xf = join(*reinterpret_cast<const int4v *>(row), *reinterpret_cast<const int4v *>(row + 64));
      sx = *reinterpret_cast<const float *>(s_rows + rows_at.scales + 4 * (t * KB + st)) * scalar_load(sb + st);
    } else {
      xf = fragment(at + 2048, r16 & (8 * NX - 1), g);
    }
    reads_done();
    --ahead;
    if (u_next < units) load_item();
    if (count > 0) {                               // uniform
      const float4v part = product<kFp8>(wf, xf, acc);
      if constexpr (kFp8) {
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] = fmaf(part[j], sx, acc[j]);
      } else {
        acc = part;
      }
    }
    if (++q < turns) continue;
    finish();
    q = 0;
    u += gridDim.x;
    if (u >= units) return;
    begin();
  }
}

// CW columns of the output, all chosen experts; the wavefronts cut the experts' K among them.  With CW < 16 the 16 rows of a
// product are CW columns on KG = 16 / CW steps of K at a time, each product with the tokens of one of them: a narrow tile
// loads as many bytes as a wide one, and there are enough of them for two workgroups on every CU.  A token's results of an
// expert are scaled by its score (and the blocks' scales) as they are added.
template <bool kFp8, int NX, int CW>
struct DownShape {
  static constexpr int KG = 16 / CW, kLd = 16 + 4;
  static constexpr int kLoads = 2 + KG * NX + (kFp8 ? 1 : 0), kItem = 1024 * (2 + KG * NX) + (kFp8 ? 256 : 0);
  static constexpr int kDepth = kItem <= 3 * 1024 ? 3 : 2;
  static constexpr int kRing = kWaves * kDepth * kItem, kPart = 4 * kWaves * 16 * kLd;
};

template <bool kFp8, int NX, int CW>
__global__ void __launch_bounds__(kThreads, 4)
few_layer_down_kernel(FewLayerArgs p) {
  using S = DownShape<kFp8, NX, CW>;
  constexpr int KG = S::KG, kLd = S::kLd;
  extern __shared__ __attribute__((aligned(1024))) char s_all[];           // the rings, part sums, slots
  const int T = p.tokens, n = T * p.k;
  float *s_part = reinterpret_cast<float *>(s_all + S::kRing);             // [wavefronts][16][kLd]
  Slots slots(s_all + S::kRing + S::kPart, n);
  for (int q = threadIdx.x; q < n; q += kThreads) {
    const int64_t e = p.idx[q];
    const float score = static_cast<float>(p.score[q]);
    slots.e[q] = e >= 0 && e < p.E ? static_cast<int>(e) : p.E;
    slots.score[q] = score;
  }
  __syncthreads();
  const int n_act = slots.build(n, p.k, p.E);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g = lane >> 4, n0 = blockIdx.x * CW;
  const int mine_k = g * 4 / CW;                   // of the KG steps, the one that this lane's results (rows 4 g ..) are of
  const int row_bytes = p.f * (kFp8 ? 1 : 2), steps = (row_bytes + 128 * KG - 1) / (128 * KG);         // of KG blocks of 128 bytes
  const int KB = scale_blocks(p.f), NB = scale_blocks(p.d);
  const int count = steps > wave ? (steps - wave + kWaves - 1) / kWaves : 0;           // of an expert: steps wave, wave + 8, ...
  const int total = count * n_act;
  const bool nt = pass_by(n_act, p.d, p.f, kFp8);
  const char *ring = s_all + wave * (S::kDepth * S::kItem);
  const uint32_t ring_at = __builtin_amdgcn_readfirstlane(lds_address(ring));

  // the biases' part of this thread's output
  const int t_mine = threadIdx.x / CW, c_mine = threadIdx.x % CW;
  static_assert(16 * CW <= kThreads, "a thread has at most one output");
  float sum = 0.0f;
  if (p.b2 && t_mine < T) {
#pragma unroll 2
    for (int s = 0; s < p.k; ++s) {
      const int e = slots.e[t_mine * p.k + s];
      if (e < p.E) sum = fmaf(slots.score[t_mine * p.k + s], static_cast<float>(p.b2[static_cast<size_t>(e) * p.d + n0 + c_mine]), sum);
    }
  }

  // this lane's loads: chunk (lane % 8) ^ (row % 8) of row 8 j + lane / 8 of a tile; of the weights' the row is column
  // r % CW at step r / CW of the item's
  const int chunk = (lane & 7) ^ (lane >> 3);
  uint32_t w_lane[2];
  int w_behind[2];                                 // where the chunk lies in the item's bytes of the column
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int r = 8 * j + (lane >> 3);
    w_behind[j] = r / CW * 128 + chunk * 16;
    w_lane[j] = r % CW * row_bytes + w_behind[j];
  }
  // the item that is loaded next: step `at` of chosen expert `i`, a token that did not choose it taking a row of one that did
  int i_next = 0, at_next = wave, slot_next = 0, ahead = 0;
  const uint8_t *w = nullptr;
  uint32_t h_lane[NX], s_lane = 0;
  auto aim = [&]() __attribute__((always_inline)) {
    const int e = __builtin_amdgcn_readfirstlane(slots.act[i_next]);
    w = static_cast<const uint8_t *>(p.w2) + (static_cast<size_t>(e) * p.d + n0) * row_bytes;
    const int t16 = lane & 15, slot16 = t16 < T ? slots.of(i_next, t16) : 255;
    const int some = __builtin_amdgcn_readlane(t16 * p.k + slot16, __ffsll(__ballot(slot16 != 255)) - 1);
    auto row_of = [&](int t) {
      const int slot = t < T ? slots.of(i_next, t) : 255;
      return static_cast<uint32_t>(slot != 255 ? t * p.k + slot : some);
    };
#pragma unroll
    for (int j = 0; j < NX; ++j) h_lane[j] = row_of(8 * j + (lane >> 3)) * row_bytes + chunk * 16;
    if constexpr (kFp8) s_lane = row_of(lane % (16)) * KB;
  };
  auto load_item = [&]() __attribute__((always_inline)) {
    if (at_next == wave) aim();
    const uint8_t *base = w + static_cast<size_t>(at_next) * (128 * KG), *h = static_cast<const uint8_t *>(p.h) + at_next * (128 * KG);
    const uint32_t at = ring_at + slot_next * S::kItem;
    const int left = row_bytes - at_next * (128 * KG);         // bytes of a row from this item on
    uint32_t lane_at[2] = {w_lane[0], w_lane[1]};
    if (left < 128 * KG) {
      // chunks behind the end of a row: the item's first one again, for activations that are zeros
#pragma unroll
      for (int j = 0; j < 2; ++j) lane_at[j] -= w_behind[j] >= left ? w_behind[j] : 0;
    }
    if (nt) {
      load16_to_lds<true>(base, lane_at[0], at);
      load16_to_lds<true>(base, lane_at[1], at + 1024);
    } else {
      load16_to_lds<false>(base, lane_at[0], at);
      load16_to_lds<false>(base, lane_at[1], at + 1024);
    }
#pragma unroll
    for (int k = 0; k < KG; ++k)
#pragma unroll
      for (int j = 0; j < NX; ++j) {
        const uint32_t to = at + 2048 + 1024 * (k * NX + j);
        if (left < 128 * KG)
          load16_to_lds(128 * k + chunk * 16 < left ? h + (128 * k + h_lane[j]) : reinterpret_cast<const uint8_t *>(&kZeros16), to);
        else
          load16_to_lds<false>(h + 128 * k, h_lane[j], to);
      }
    if constexpr (kFp8) {
      // the scales of the tokens at the item's steps, token t at step k in lane 16 k + t
      const int k = lane / (16) < KG ? lane / (16) : KG - 1, kb = at_next * KG + k < KB ? at_next * KG + k : KB - 1;
      load4_to_lds(p.h_scales, 4 * (s_lane + kb), at + 1024 * (2 + KG * NX));
    }
    ++ahead;
    slot_next = slot_next + 1 < S::kDepth ? slot_next + 1 : 0;
    at_next += kWaves;
    if (at_next >= steps) {
      at_next = wave;
      ++i_next;
    }
  };
  static_assert(!kFp8 || 16 * KG <= 64, "a lane per token and step");

  // the item that is computed
  int i = 0, at = wave, place = 0;
  const float *sb = nullptr;
  float score;
  bool chose;
  float4v acc = float4v{0, 0, 0, 0};
  if (total > 0) {
    int loaded = 0;
#pragma unroll
    for (int j = 0; j < S::kDepth; ++j)
      if (loaded < total) {
        load_item();
        ++loaded;
      }
    for (int item = 0; item < total; ++item) {
      if (at == wave) {
        const int e = __builtin_amdgcn_readfirstlane(slots.act[i]);
        if constexpr (kFp8) sb = p.s2 + (static_cast<size_t>(e) * NB + n0 / kScaleBlock) * KB;
        const int t = r16, slot = t < T ? slots.of(i, t) : 255;
        chose = slot != 255;
        score = chose ? slots.score[t * p.k + slot] : 0.0f;
      }
      if (ahead == S::kDepth) loads_but<S::kLoads *(S::kDepth - 1)>();
      else loads_but<0>();
      const char *tile = ring + place * S::kItem;
      place = place + 1 < S::kDepth ? place + 1 : 0;
      const int8v wf = fragment(tile, r16, g);
      int8v hf[KG];
      float s;
#pragma unroll
      for (int k = 0; k < KG; ++k)
        hf[k] = fragment(tile + 2048 + 1024 * NX * k, r16 & (8 * NX - 1), g);
      s = score;
      if constexpr (kFp8) {
        // (weights' scales of all the item's steps, this lane's picked)
        float scale = scalar_load(sb + at * KG);
#pragma unroll
        for (int k = 1; k < KG; ++k) {
          const float other = scalar_load(sb + (at * KG + k < KB ? at * KG + k : KB - 1));
          scale = mine_k == k ? other : scale;
        }
        s *= *reinterpret_cast<const float *>(tile + 1024 * (2 + KG * NX) + 4 * (16 * mine_k + r16)) * scale;
      }
      reads_done();
      --ahead;
      if (loaded < total) {
        load_item();
        ++loaded;
      }
      float4v part = product<kFp8>(wf, hf[0]);
#pragma unroll
      for (int k = 1; k < KG; ++k) {
        const float4v other = product<kFp8>(wf, hf[k]);
        part = mine_k == k ? other : part;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j] = chose ? fmaf(part[j], s, acc[j]) : acc[j];
      at += kWaves;
      if (at >= steps) {
        at = wave;
        ++i;
      }
    }
  }
  *reinterpret_cast<float4v *>(s_part + (wave * 16 + r16) * kLd + 4 * g) = acc;
  __syncthreads();
  if (t_mine < T) {
#pragma unroll
    for (int x = 0; x < kWaves; ++x)
#pragma unroll
      for (int j = 0; j < KG; ++j) sum += s_part[(x * 16 + t_mine) * kLd + j * CW + c_mine];
    p.out[static_cast<size_t>(t_mine) * p.d + n0 + c_mine] = static_cast<half_t>(sum);
  }
}
}  // namespace

bool few_layer_fits(int tokens, int d, int f, int E, int k) {
  return tokens >= 1 && tokens <= kFewTokens && d > 0 && f > 0 && d % 64 == 0 && f % 64 == 0 && E >= 1 && E <= 1024 && k >= 1 &&
         k <= kMaxTopK && k <= E;
}

namespace {

template <typename K>
int allow_lds(K kernel, size_t lds) {
  if (lds <= 65536) return CCF_OK;
  hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                     static_cast<int>(lds));
  return e == hipSuccess ? static_cast<int>(CCF_OK) : fail(CCF_ERR_HIP, "few_layer: LDS attribute: %s", hipGetErrorString(e));
}

template <bool kFp8, int NX>
int launch_up(const FewLayerArgs &p, bool gated, size_t gate_bytes, hipStream_t st) {
  using S = UpShape<kFp8, NX>;
  const int n = p.tokens * p.k;
  const size_t ring = gate_bytes > S::kRing ? (gate_bytes + 1023) / 1024 * 1024 : S::kRing;
  const size_t lds = ring + S::kPart + (Slots::bytes(n) + 15) / 16 * 16 + (kFp8 ? rows_lds(p.tokens, p.d).bytes : 0);
  auto kernel = few_layer_up_kernel<kFp8, NX>;
  if (int rc = allow_lds(kernel, lds)) return rc;
  const long long units = static_cast<long long>(p.E < n ? p.E : n) * ((p.f + S::BN - 1) / S::BN);
  const int most = lds > 80 * 1024 ? 256 : 512;                // workgroups on the chip at once
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(units < most ? units : most)), dim3(kThreads), lds, st, p, gated,
                     static_cast<int>(ring));
  return check_launch("few_layer_up_kernel");
}

template <bool kFp8, int NX, int CW>
int launch_down_at(const FewLayerArgs &p, hipStream_t st) {
  using S = DownShape<kFp8, NX, CW>;
  const size_t lds = S::kRing + S::kPart + Slots::bytes(p.tokens * p.k);
  auto kernel = few_layer_down_kernel<kFp8, NX, CW>;
  if (int rc = allow_lds(kernel, lds)) return rc;
  hipLaunchKernelGGL(kernel, dim3(p.d / CW), dim3(kThreads), lds, st, p);
  return check_launch("few_layer_down_kernel");
}

template <bool kFp8, int NX>
int launch_down(const FewLayerArgs &p, hipStream_t st) {
  // the widest tiles of which there are two for every CU; with more than 8 tokens an item of narrow ones is mostly tokens
  if constexpr (NX == 1) {
    if (p.d < 8 * 256) return launch_down_at<kFp8, NX, 4>(p, st);
  }
  return p.d < 16 * 512 ? launch_down_at<kFp8, NX, 8>(p, st) : launch_down_at<kFp8, NX, 16>(p, st);
}

template <bool kFp8>
int launch_few_layer(const FewLayerArgs &p, bool gated, size_t gate_bytes, hipStream_t st) {
  auto run = [&](auto NX_) {
    constexpr int NX = decltype(NX_)::value;
    if (int rc = launch_up<kFp8, NX>(p, gated, gate_bytes, st)) return rc;
    return launch_down<kFp8, NX>(p, st);
  };
  return p.tokens <= 8 ? run(std::integral_constant<int, 1>{}) : run(std::integral_constant<int, 2>{});
}

// What the first kernel may keep in LDS of the gate's operands, and of tokens in 8 bits beside its rings, part sums (9 KB at
// most) and slots (4 KB).
constexpr int kMaxGateLds = 64 * 1024, kMaxRowsLds = 64 * 1024;

}  // namespace

bool few_layer_fits_fp8(int tokens, int d) { return rows_lds(tokens, d).bytes <= kMaxRowsLds; }

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
  return fp8 ? launch_few_layer<true>(p, !here, gate_bytes, as_stream(stream))
             : launch_few_layer<false>(p, !here, gate_bytes, as_stream(stream));
}

}  // namespace ccf
