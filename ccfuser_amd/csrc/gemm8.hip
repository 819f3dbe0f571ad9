// Matrix product in e4m3 with a scale for each block of 128, dense or grouped by expert, for gfx950.
//
//   y[r, n] = sum over blocks b of sa[r, b] sb[n / 128, b] (sum over k in b of a[r, k] w[n, k]) + bias[n]
//
// v_mfma_f32_16x16x128_f8f6f4 contracts one block: its result, from zero, is scaled by a row's and a weight block's scale
// and added to the sum in fp32, four fused multiply-adds for an instruction of 32 cycles.  Weights are the A operand, so a
// lane holds four consecutive columns of one row: one scale per lane and 16 rows, and stores of four columns.  (The
// instruction's own scales are powers of two per 32 elements; weights come with scales of any value.)  A lane's 32
// bytes are the same ones of either operand, in whatever order of K: all that a product needs.
//
// Two kernels.  gemm8_tile_kernel: tiles of 256, 128 or 64 rows through LDS.  It is bound by the instructions that a SIMD
// issues: at 4096 rows, 4096 -> 14336, 252 us (1.9 PFLOP/s) and 225 with the loads of operands left out; the four fused
// multiply-adds per product, which any fp32 scale needs, are most of them.  gemm8_split_kernel: a workgroup's wavefronts cut K
// among them and read straight from memory, for few rows or few tiles: bound by the weights' bytes or by a chain of loads
// (1 row, 4096 -> 14336: 14.8 us, 4.0 TB/s).
#include "gemm8.h"
#include "gelu.h"

#include <type_traits>
#include <utility>

namespace ccf {
int g_fp8_form = 0;          // 0: by form_of's rule, else a Form for every call
namespace {

__device__ const int4v kZeros16 = {0, 0, 0, 0};              // what lanes behind the end of K read

__device__ __forceinline__ float4v mfma8(int8v a, int8v b) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, float4v{0, 0, 0, 0}, 0, 0, 0, 0, 0, 0);
}

__device__ __forceinline__ int8v join(int4v lo, int4v hi) { return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7); }

// f(0), f(1), ... f(N - 1), each index a constant
template <int... I, class F>
__device__ __forceinline__ void in_turn(std::integer_sequence<int, I...>, F f) {
  (f(std::integral_constant<int, I>{}), ...);
}

struct Tile {
  int e, row0, rows, m, n;   // expert (-1: none), first sorted row, rows of the expert from it on, tile indices
};

// Tile `t` of the grouped product in tiles of BM rows: expert by expert, inside one in groups of 8 tiles of rows, columns
// outside, so that neighbours share both operands.  The experts' tiles are counted 64 experts at a time.
template <int BM>
__device__ __forceinline__ Tile find_tile(const Gemm8Args &p, int pid, int grid, int n_tiles) {
  const int lane = threadIdx.x & 63;
  auto span = [&](int e, int &lo, int &hi) {
    lo = hi = 0;
    if (e < p.E) {
      lo = p.offsets ? p.offsets[e] : 0;
      hi = p.offsets ? p.offsets[e + 1] : p.max_rows;
      lo = lo < p.max_rows ? lo : p.max_rows;
      hi = hi < p.max_rows ? hi : p.max_rows;
    }
  };
  int total = 0;
  for (int e0 = 0; e0 < p.E; e0 += 64) {
    int lo, hi;
    span(e0 + lane, lo, hi);
    int mt = hi > lo ? (hi - lo + BM - 1) / BM : 0;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mt += __shfl_xor(mt, o);
    total += mt;
  }
  total = __builtin_amdgcn_readfirstlane(total) * n_tiles;
  // workgroup ids go round the 8 XCDs: each XCD takes a run of tiles, which share operands in its L2
  const int per = (total + 7) / 8;
  int t = (pid & 7) * per + (pid >> 3);
  Tile r{-1, 0, 0, 0, 0};
  if ((pid >> 3) >= per || t >= total) return r;
  int before = 0;
  for (int e0 = 0; e0 < p.E; e0 += 64) {
    int lo, hi;
    span(e0 + lane, lo, hi);
    const int mt = hi > lo ? (hi - lo + BM - 1) / BM : 0;
    int upto = mt;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(upto, o);
      upto += lane >= o ? v : 0;
    }
    const unsigned long long past = __ballot((before + upto) * n_tiles > t);
    if (past) {
      const int who = __ffsll(past) - 1;
      const int mts = __builtin_amdgcn_readlane(mt, who);
      t -= (before + __builtin_amdgcn_readlane(upto, who) - mts) * n_tiles;
      const int group = t / (8 * n_tiles), in = t - group * 8 * n_tiles;
      const int gm = mts - group * 8 < 8 ? mts - group * 8 : 8;
      r.e = e0 + who;
      r.n = in / gm;
      r.m = group * 8 + in - r.n * gm;
      r.row0 = __builtin_amdgcn_readlane(lo, who) + r.m * BM;
      r.rows = __builtin_amdgcn_readlane(hi, who) - r.row0;
      return r;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  return r;
}

// ------------------------------------------------------------------ tiles through LDS
//
// BM rows x BN columns, WM x WN wavefronts; a K step is a block of 128, staged by direct loads into one of NS LDS places
// while another is multiplied (two; of the 64-row tile in one group three, so that a load has two steps to land).  16-byte
// chunks of a row lie at chunk ^ (row % 8), which the loads' global addresses apply, and a lane's two chunks are g and g + 4
// (g = lane / 16): a read then takes 5 cycles of a wavefront (256 bytes each), with 2 g and 2 g + 1 9, unswizzled 17.  The
// scales of a step come the same way, a lane per row, and lie by row.
//
// A wavefront reads its rows' fragments once a step and its columns' one by one, each ahead of its products.  The step's one
// barrier stands in front of its last columns, whose fragments are in registers by then: behind it this step's place is free
// for the loads of the step NS on, and the next step's rows are read between the last products.  So the matrix cores run
// through the steps, and a load has a whole step to land.
//
// KS = 2: two groups of such wavefronts take every other block each, with places of their own, and their sums meet in LDS at
// the tile's end: half as many steps, for a CU that has one small tile (512 rows, 4096 -> 1024: 17 us for 21.5).
template <int BM, int BN, int WM, int WN, int NS, int KS>
struct TileShape {
  static constexpr int kWaves = WM * WN, kThreads = KS * kWaves * 64;       // (wavefronts of a group)
  static constexpr int TT = BM / WM / 16, CT = BN / WN / 16;       // 16 x 16 products of a wavefront: rows, columns
  static constexpr int kRowsBytes = (BM + BN) * kScaleBlock;       // a place: codes, then scales of rows, then of columns
  static constexpr int kStage = kRowsBytes + 4 * (BM + 64);
  static constexpr int kLoadsX = BM / 8 / kWaves, kLoadsW = BN / 8 / kWaves;      // loads of 1 KB per wavefront and step
  static constexpr int kLoads = kLoadsX + kLoadsW;
  static constexpr int kPlace = KS * kStage, kMeet = KS > 1 ? 4 * BM * BN : 0, kMap = NS * kPlace + kMeet;
  static_assert(kWaves >= BM / 64 + 1, "a wavefront more than the rows' scales take loads the columns'");
};

// Direct loads to LDS at byte `at` + 16 (or 4) * lane.  In asm so that the compiler, which cannot tell the two places
// apart, does not wait for them in front of every LDS read: they write no register, and the step's own wait and barrier
// stand between them and any read of what they bring.
__device__ __forceinline__ void load16_to_lds(const void *src, uint32_t at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(at), "v"(src));
}
// The same at a 32-bit offset from an address that the wavefront shares.
__device__ __forceinline__ void load16_to_lds(const void *base, uint32_t offset, uint32_t at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(at), "v"(offset), "s"(base));
}
__device__ __forceinline__ void load4_to_lds(const void *src, uint32_t at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(at), "v"(src));
}

// Rows of an expert beyond its 256-row tiles cost as much as a whole one however few they are: up to kLeftRows of them may
// go to a launch of smaller tiles.
enum { kAll = 0, kWhole = 1, kLeft = 2 };            // all rows; without those; those alone
constexpr int kWholeRows = 256, kLeftRows = 64;

// The experts' tiles in LDS, for a workgroup that runs several: first[e] tiles of rows in front of expert e's, the first row
// of it and, E further, the one behind its last.
template <int BM>
struct TileMap {
  const int *first, *row;    // [E + 1], [2 E]
  int E, n_tiles;

  // all threads; the caller's barrier follows.  Of every expert's rows those that `part` says
  __device__ __forceinline__ static void build(const Gemm8Args &p, int part, int *first, int *row) {
    if (threadIdx.x >= 64) return;
    const int lane = threadIdx.x;
    int before = 0;
    for (int e0 = 0; e0 < p.E; e0 += 64) {
      int lo = 0, hi = 0;
      if (e0 + lane < p.E) {
        lo = p.offsets ? p.offsets[e0 + lane] : 0;
        hi = p.offsets ? p.offsets[e0 + lane + 1] : p.max_rows;
        lo = lo < p.max_rows ? lo : p.max_rows;
        hi = hi < p.max_rows ? hi : p.max_rows;
        const int over = hi > lo ? (hi - lo) % kWholeRows : 0;
        const bool few = over <= kLeftRows;          // rows beyond whole tiles that tiles of their own take
        if (part == kWhole && few) hi -= over;
        if (part == kLeft) lo = few ? hi - over : hi;
      }
      int upto = hi > lo ? (hi - lo + BM - 1) / BM : 0;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int v = __shfl_up(upto, o);
        upto += lane >= o ? v : 0;
      }
      if (e0 + lane < p.E) {
        if (e0 + lane == 0) first[0] = 0;
        first[e0 + lane + 1] = before + upto;
        row[e0 + lane] = lo;
        row[p.E + e0 + lane] = hi;
      }
      before += __builtin_amdgcn_readlane(upto, 63);
    }
  }

  __device__ __forceinline__ int total() const { return __builtin_amdgcn_readfirstlane(first[E]) * n_tiles; }

  // tile t of total(): inside an expert in groups of 8 tiles of rows, columns outside, so that neighbours share both operands
  __device__ __forceinline__ Tile find(int t) const {
    const int lane = threadIdx.x & 63;
    int e0 = 0;
    unsigned long long past = 0;
    for (; e0 < E; e0 += 64) {
      past = __ballot(e0 + lane < E && first[e0 + lane + 1] * n_tiles > t);
      if (past) break;
    }
    const int e = e0 + __ffsll(past) - 1;
    const int f = __builtin_amdgcn_readfirstlane(first[e]), mts = __builtin_amdgcn_readfirstlane(first[e + 1]) - f;
    t -= f * n_tiles;
    const int group = t / (8 * n_tiles), in = t - group * 8 * n_tiles;
    const int gm = mts - group * 8 < 8 ? mts - group * 8 : 8;
    Tile r;
    r.e = e;
    r.n = in / gm;
    r.m = group * 8 + in - r.n * gm;
    r.row0 = __builtin_amdgcn_readfirstlane(row[e]) + r.m * BM;
    r.rows = __builtin_amdgcn_readfirstlane(row[E + e]) - r.row0;
    return r;
  }
};

// out[j], j the source's 16 lanes: afterwards the 16 lanes `g` of all four hold what was in[g] of the lanes 16 j ...
__device__ __forceinline__ void transpose_rows_of_16(uint32_t (&v)[4]) {
  typedef unsigned uint2v __attribute__((ext_vector_type(2)));
  uint2v a = __builtin_amdgcn_permlane16_swap(v[0], v[1], false, false), b = __builtin_amdgcn_permlane16_swap(v[2], v[3], false, false);
  uint2v c = __builtin_amdgcn_permlane32_swap(a.x, b.x, false, false), d = __builtin_amdgcn_permlane32_swap(a.y, b.y, false, false);
  v[0] = c.x;
  v[1] = d.x;
  v[2] = c.y;
  v[3] = d.y;
}

// Where a lane's loads of a tile's first step start, row i * 8 * waves + 8 * wave + lane / 8 of the stage: the tile's rows in
// units of 16 bytes from p.a, its columns in bytes from the expert's weight; the scales of row 64 wave + lane, or of column
// 128 lane, in floats.  (A function, and its caller's
// advance not another: as closures they kept their captures in memory.)
template <class S, int BM, int BN>
__device__ __forceinline__ void tile_sources(const Gemm8Args &p, const Tile &tile, int wave, int lane, int chunk, int KB, int NB,
                                             uint32_t (&src)[S::kLoads], uint32_t &scale_src) {
  asm("" : "+v"(lane));                              // what follows from it is made here, not kept over the steps
  const int rows = tile.rows < BM ? tile.rows : BM, n0 = tile.n * BN;
  const uint32_t chunks = p.K / 16;
  auto a_row = [&](int r) {                          // past the end: the last row again, never stored
    const int j = tile.row0 + (r < rows ? r : rows - 1);
    return static_cast<uint32_t>(p.a_rows ? p.a_rows[j] : j);
  };
#pragma unroll
  for (int i = 0; i < S::kLoadsX; ++i) src[i] = a_row((i * S::kWaves + wave) * 8 + (lane >> 3)) * chunks + chunk;
#pragma unroll
  for (int i = 0; i < S::kLoadsW; ++i) {
    const int n = n0 + (i * S::kWaves + wave) * 8 + (lane >> 3);
    src[S::kLoadsX + i] = (static_cast<uint32_t>(n < p.N ? n : p.N - 1) * chunks + chunk) * 16;
  }
  if (wave < BM / 64) {
    scale_src = a_row(wave * 64 + lane) * KB;
  } else {
    const int nb = (n0 + lane * kScaleBlock) / kScaleBlock;
    scale_src = static_cast<uint32_t>(tile.e * NB + (nb < NB ? nb : NB - 1)) * KB;
  }
}

// On to the step behind `next`'s next_step, which is loaded; e < 0: there is none.
template <class S, int BM, int BN, int KS>
__device__ __forceinline__ void advance(const Gemm8Args &p, const TileMap<BM> &map, int end, int slots, int ks, int wave, int lane, int chunk,
                                        int KB, int NB, Tile &next, int &next_step, int &t_next, int &ahead,
                                        const uint8_t *&a, const uint8_t *&b,
                                        uint32_t (&src)[S::kLoads], uint32_t &scale_src) {
  ++ahead;
  a += KS * kScaleBlock;
  b += KS * kScaleBlock;
  if (++next_step * KS < KB) return;
  next_step = 0;
  t_next += slots;
  if (t_next < end) {
    next = map.find(t_next);
    a = p.a + ks * kScaleBlock;
    b = p.b + static_cast<size_t>(next.e) * p.N * p.K + ks * kScaleBlock;
    tile_sources<S, BM, BN>(p, next, wave, lane, chunk, KB, NB, src, scale_src);
  } else {
    next.e = -1;
  }
}

// Persistent: a workgroup per CU (or two, of small tiles) runs tiles one behind the other, and the steps of all of them are
// one stream: the next tile's first loads are on their way while this one's last products and its epilogue run.
template <int BM, int BN, int WM, int WN, int NS, int KS, int kOut>
__global__ void __launch_bounds__(KS * WM * WN * 64, 2)
gemm8_tile_kernel(Gemm8Args p, int n_tiles, int part) {
  using S = TileShape<BM, BN, WM, WN, NS, KS>;
  using Out = std::conditional_t<kOut == kGemm8Bf16, bf16_t, half_t>;
  extern __shared__ __attribute__((aligned(1024))) char s_tile[];          // the places, where the groups meet, the tile map
  int *s_map = reinterpret_cast<int *>(s_tile + S::kMap);
  TileMap<BM>::build(p, part, s_map, s_map + p.E + 1);
  __syncthreads();
  const TileMap<BM> map{s_map, s_map + p.E + 1, p.E, n_tiles};
  // workgroup ids go round the 8 XCDs: each XCD takes a run of tiles, which share operands in its L2
  const int total = map.total(), per = (total + 7) / 8, slots = gridDim.x / 8;
  const int end = ((blockIdx.x & 7) + 1) * per < total ? ((blockIdx.x & 7) + 1) * per : total;
  int t_next = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if (t_next >= end) return;

  const int lane = threadIdx.x & 63, wave_all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ks = KS > 1 ? wave_all / S::kWaves : 0, wave = KS > 1 ? wave_all % S::kWaves : wave_all;
  const int r16 = lane & 15, g = lane >> 4;
  const int wm = wave / WN, wn = wave % WN;
  const int KB = scale_blocks(p.K), NB = scale_blocks(p.N), tail = p.K % kScaleBlock;
  auto block_of = [&](int n) __attribute__((always_inline)) { return n / kScaleBlock < NB ? n / kScaleBlock : NB - 1; };

  const int chunk = (lane & 7) ^ (lane >> 3);        // of a row, that this lane's loads take to place lane % 8
  uint32_t src[S::kLoads], scale_src;
  const bool scales_of_rows = wave < BM / 64, scales_of_columns = wave == BM / 64;       // lane i: of column 128 i
  const float *scale_base = p.b_scale;
  if (scales_of_rows) scale_base = p.a_scale;
  // the step whose loads are issued next: tile `next` (e < 0: there is none), block KS next_step + ks
  int t_now = t_next, next_step = 0, ahead = 0;        // ahead: steps loaded beyond the one that is computed
  Tile next = map.find(t_next);
  const uint8_t *a = p.a + ks * kScaleBlock, *b = p.b + static_cast<size_t>(next.e) * p.N * p.K + ks * kScaleBlock;
  tile_sources<S, BM, BN>(p, next, wave, lane, chunk, KB, NB, src, scale_src);
  char *s_mine = s_tile + ks * S::kStage;
  const uint32_t lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char *)s_mine));
  // Its loads in four parts: a wavefront that issues all at once waits for the queue, and its products with it.  A wavefront
  // of few products, which are done before its instructions are issued, has fewer of those with all loads in one.
  constexpr int kParts = S::TT >= 4 ? 4 : 1;
  constexpr std::integral_constant<int, 0> kFirst{};
  auto load_part = [&](int place, auto PART) __attribute__((always_inline)) {
    constexpr int quarter = decltype(PART)::value;
    const uint32_t at = __builtin_amdgcn_readfirstlane(lds + place * S::kPlace + wave * 1024);
    // (a group that has no block left loads the last one, for nothing)
    const int kb = KS * next_step + ks, over = KS > 1 && kb >= KB ? kb - KB + 1 : 0;
    const uint8_t *rows = a - over * kScaleBlock, *columns = b - over * kScaleBlock;
    constexpr int lo = quarter * S::kLoads / kParts, hi = (quarter + 1) * S::kLoads / kParts;
    if (tail && kb - over == KB - 1) {
      // chunks behind the end of K: zeros for the rows, and for the columns the block's first chunk again (what is no
      // number there is no number in the sum anyway)
      const bool behind = chunk * 16 >= tail;
#pragma unroll
      for (int i = lo; i < hi; ++i) {
        const uint8_t *q = rows + (static_cast<uint64_t>(src[i]) << 4);
        if (i < S::kLoadsX) load16_to_lds(behind ? reinterpret_cast<const uint8_t *>(&kZeros16) : q, at + i * S::kWaves * 1024);
        else load16_to_lds(columns, src[i] - (behind ? chunk * 16 : 0), at + i * S::kWaves * 1024);
      }
    } else {
#pragma unroll
      for (int i = lo; i < hi; ++i) {
        if (i < S::kLoadsX) load16_to_lds(rows + (static_cast<uint64_t>(src[i]) << 4), at + i * S::kWaves * 1024);
        else load16_to_lds(columns, src[i], at + i * S::kWaves * 1024);
      }
    }
    if (quarter == 0 && (scales_of_rows || scales_of_columns))          // the wavefronts' 64 scales each, one behind the other
      load4_to_lds(scale_base + (kb - over) + scale_src,
                   __builtin_amdgcn_readfirstlane(lds + place * S::kPlace + S::kRowsBytes + wave * 256));
  };

  const int x_at = (wm * (BM / WM) + r16) * kScaleBlock + (g ^ (r16 & 7)) * 16;
  const int w_at = (BM + wn * (BN / WN) + r16) * kScaleBlock + (g ^ (r16 & 7)) * 16;
  const int sa_at = S::kRowsBytes + 4 * (wm * (BM / WM) + r16), sb_at = S::kRowsBytes + 4 * (BM + wn * (BN / WN) / kScaleBlock);
  auto fragment = [&](const char *place, int at, int i) __attribute__((always_inline)) {
    return join(*reinterpret_cast<const int4v *>(place + at + i * 16 * kScaleBlock),
                *reinterpret_cast<const int4v *>(place + (at ^ 64) + i * 16 * kScaleBlock));
  };
  // Fragments of columns are read kRing - 1 ahead of their products, and a product's result is scaled three products later.
  // With four rows' fragments to a column's one that is ahead enough; with fewer a column's products do not cover an LDS read,
  // and three columns' do.
  constexpr int kRing = S::TT >= 4 ? 2 : 4, kLate = 3, Q = S::CT * S::TT;
  static_assert(S::CT % kRing == 0 && Q % (kLate + 1) == 0 && S::CT - kRing >= 4, "rings turn whole times in a step");
  float4v acc[S::CT][S::TT], product[kLate + 1];
  int8v x[S::TT], w[kRing], x_next[S::TT];
  float sa[S::TT], sb, s[S::TT];                     // scales as read for the coming step; of the step whose results are scaled
  auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < S::CT; ++c)
#pragma unroll
      for (int t = 0; t < S::TT; ++t) acc[c][t] = float4v{0, 0, 0, 0};
#pragma unroll
    for (int q = 0; q <= kLate; ++q) product[q] = float4v{0, 0, 0, 0};
#pragma unroll
    for (int t = 0; t < S::TT; ++t) s[t] = 0.0f;
  };
  auto scaled = [&](int q) __attribute__((always_inline)) {          // of the step's Q products, in their order
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float4v &sum = acc[q / S::TT][q % S::TT];
      sum[i] = fmaf(product[q % (kLate + 1)][i], s[q % S::TT], sum[i]);
    }
  };
  // the sums of columns c exist here: without that the compiler puts all scalings of a step off behind its branch, and
  // keeps their inputs in registers that there are not
  auto settled = [&](int c) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < S::TT; ++t) asm volatile("" : "+v"(acc[c][t]));
  };
  // the coming step's loads have landed (those of the ahead - 1 steps behind it may be on their way), all LDS reads are done
  const bool more_loads = scales_of_rows || scales_of_columns;
  auto meet = [&]() __attribute__((always_inline)) {
    auto wait = [](auto N) __attribute__((always_inline)) {
      constexpr int n = decltype(N)::value;
      static_assert(n < 64, "vmcnt has six bits");
      __builtin_amdgcn_s_waitcnt(0x0070 | (n & 15) | (n >> 4) << 14);      // vmcnt(n) lgkmcnt(0)
    };
    if (NS == 2 || ahead <= 1) wait(std::integral_constant<int, 0>{});
    else in_turn(std::make_integer_sequence<int, NS - 2>{}, [&](auto I) __attribute__((always_inline)) {
      constexpr int behind = decltype(I)::value + 1;
      if (ahead != behind + 1) return;
      if (more_loads) wait(std::integral_constant<int, behind * (S::kLoads + 1)>{});
      else wait(std::integral_constant<int, behind * S::kLoads>{});
    });
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };

  Tile tile = next;
#pragma unroll
  for (int i = 0; i < NS - 1; ++i)
    if (next.e >= 0) {
      in_turn(std::make_integer_sequence<int, kParts>{}, [&](auto I) __attribute__((always_inline)) { load_part(i, I); });
      advance<S, BM, BN, KS>(p, map, end, slots, ks, wave, lane, chunk, KB, NB, next, next_step, t_next, ahead, a, b, src, scale_src);
    }
  auto on = [&]() __attribute__((always_inline)) {
    advance<S, BM, BN, KS>(p, map, end, slots, ks, wave, lane, chunk, KB, NB, next, next_step, t_next, ahead, a, b, src, scale_src);
  };
  auto begin_load = [&](int place) __attribute__((always_inline)) {
    --ahead;                                         // (which counted the step that comes)
    if (next.e < 0) return;
    load_part(place, kFirst);
    if constexpr (kParts == 1) on();
  };
  meet();
  begin_load(NS - 1);
  sb = *reinterpret_cast<const float *>(s_mine + sb_at);
#pragma unroll
  for (int t = 0; t < S::TT; ++t) {
    x[t] = fragment(s_mine, x_at, t);
    sa[t] = *reinterpret_cast<const float *>(s_mine + sa_at + 64 * t);
  }
#pragma unroll
  for (int c = 0; c < kRing - 1; ++c) w[c] = fragment(s_mine, w_at, c);
  clear();

  int place = 0, step = 0;
  while (true) {
    const char *now = s_mine + place * S::kPlace;
    const int coming = place + 1 < NS ? place + 1 : 0;
    const char *next_place = s_mine + coming * S::kPlace;            // behind the last step: read for nothing
    in_turn(std::make_integer_sequence<int, S::CT>{}, [&](auto C) __attribute__((always_inline)) {
      constexpr int c = decltype(C)::value, c_ahead = c + kRing - 1;
      constexpr bool at_meet = c == S::CT - kRing + 1, rows_here = S::TT >= 4 && c == S::CT - 1;
      if constexpr (at_meet) {
        meet();                                      // the next step's loads have landed, this one's place is read
        begin_load(place);
        if constexpr (S::TT < 4) {
#pragma unroll
          for (int t = 0; t < S::TT; ++t) {
            x_next[t] = fragment(next_place, x_at, t);
            sa[t] = *reinterpret_cast<const float *>(next_place + sa_at + 64 * t);
          }
          sb = *reinterpret_cast<const float *>(next_place + sb_at);
        }
      }
      if constexpr (!rows_here) w[c_ahead % kRing] = fragment(c_ahead < S::CT ? now : next_place, w_at, c_ahead % S::CT);
#pragma unroll
      for (int t = 0; t < S::TT; ++t) {
        const int q = c * S::TT + t;
        if (q == kLate) {
#pragma unroll
          for (int i = 0; i < S::TT; ++i) s[i] = KS == 1 || KS * step + ks < KB ? sa[i] * sb : 0.0f;
        }
        product[q % (kLate + 1)] = mfma8(w[c % kRing], x[t]);
        scaled((q + Q - kLate) % Q);
        if constexpr (rows_here) {
          x[t] = fragment(next_place, x_at, t);
          sa[t] = *reinterpret_cast<const float *>(next_place + sa_at + 64 * t);
        }
      }
      if constexpr (rows_here) {
        w[0] = fragment(next_place, w_at, 0);
        sb = *reinterpret_cast<const float *>(next_place + sb_at);
      } else if constexpr (S::TT >= 4) {
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
#pragma unroll
        for (int t = 0; t < S::TT; ++t) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
        }
      }
      settled(((Q + (c + 1) * S::TT - kLate) / S::TT + S::CT - 1) % S::CT);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (kParts > 1 && c < kParts) {
        if (next.e >= 0) {
          if constexpr (c < kParts - 1) load_part(place ? place - 1 : NS - 1, std::integral_constant<int, c + 1>{});
          else on();
        }
      }
    });
    if constexpr (S::TT < 4) {
#pragma unroll
      for (int t = 0; t < S::TT; ++t) x[t] = x_next[t];
    }
    place = coming;
    if (++step * KS < KB) continue;

    // the tile's end.  A lane holds one row and, in every product, four consecutive columns; of four products' columns it
    // stores 16 consecutive ones, which it gets from the lanes that hold the same row
#pragma unroll
    for (int q = Q - kLate; q < Q; ++q) scaled(q);
    if constexpr (KS > 1) {
      static_assert(KS == 2, "two groups meet");
      // (written again only behind barriers of the next tile's steps)
      float4v *at = reinterpret_cast<float4v *>(s_tile + NS * S::kPlace) + wave * Q * 64 + lane;
      if (ks == 1) {
#pragma unroll
        for (int q = 0; q < Q; ++q) at[q * 64] = acc[q / S::TT][q % S::TT];
      }
      __builtin_amdgcn_s_waitcnt(0xc07f);            // lgkmcnt(0)
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (ks == 0) {
#pragma unroll
        for (int q = 0; q < Q; ++q) acc[q / S::TT][q % S::TT] += at[q * 64];
      }
    }
    if (KS == 1 || ks == 0) {
    const int rows = tile.rows < BM ? tile.rows : BM, n0 = tile.n * BN;
    const Out *bias = p.bias ? static_cast<const Out *>(p.bias) + static_cast<size_t>(tile.e) * p.N : nullptr;
    const int col0 = n0 + wn * (BN / WN), nb = block_of(col0);       // a wavefront's columns share a scale
    typedef Out out4 __attribute__((ext_vector_type(4)));
    out4 b4[S::CT];
#pragma unroll
    for (int c = 0; c < S::CT; ++c) {
      const int col = col0 + 16 * c + 4 * g;
      b4[c] = bias && col < p.N ? *reinterpret_cast<const out4 *>(bias + col) : out4{0, 0, 0, 0};
    }
#pragma unroll
    for (int t = 0; t < S::TT; ++t) {
      const int r = wm * (BM / WM) + t * 16 + r16;
      const bool mine = r < rows;
      const int j = tile.row0 + (mine ? r : 0);
      const size_t crow = static_cast<size_t>(p.c_rows ? p.c_rows[j] : j);
      if constexpr (kOut == kGemm8Gelu8) {
        float top = 0.0f;
#pragma unroll
        for (int c = 0; c < S::CT; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float v = gelu_erf(acc[c][t][i] + static_cast<float>(b4[c][i]));
            v = col0 + 16 * c + 4 * g < p.N ? v : 0.0f;
            acc[c][t][i] = v;
            top = fmaxf(top, fabsf(v));
          }
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        float inverse;
        const float scale = block_scale(top, &inverse);
        if (mine && g == 0 && col0 < p.N) p.scales[crow * NB + nb] = scale;
#pragma unroll
        for (int q = 0; q < S::CT; q += 4) {
          uint32_t v[4];
#pragma unroll
          for (int c = 0; c < 4; ++c)
            v[c] = static_cast<uint32_t>(pack_fp8(acc[q + c][t][0] * inverse, acc[q + c][t][1] * inverse,
                                                  acc[q + c][t][2] * inverse, acc[q + c][t][3] * inverse));
          transpose_rows_of_16(v);
          const int col = col0 + 16 * (q + g);
          uint8_t *at = p.codes + crow * p.N + col;          // 8-byte aligned
          if (mine && col < p.N) *reinterpret_cast<int2v *>(at) = int2v{static_cast<int>(v[0]), static_cast<int>(v[1])};
          if (mine && col + 8 < p.N) *reinterpret_cast<int2v *>(at + 8) = int2v{static_cast<int>(v[2]), static_cast<int>(v[3])};
        }
      } else {
#pragma unroll
        for (int q = 0; q < S::CT; q += 4) {
          uint32_t lo[4], hi[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            out4 o;
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = static_cast<Out>(acc[q + c][t][i] + static_cast<float>(b4[q + c][i]));
            const int2v words = __builtin_bit_cast(int2v, o);
            lo[c] = words[0];
            hi[c] = words[1];
          }
          transpose_rows_of_16(lo);
          transpose_rows_of_16(hi);
          const int col = col0 + 16 * (q + g);
          int4v *at = reinterpret_cast<int4v *>(static_cast<Out *>(p.c) + crow * p.N + col);
          auto word = [](uint32_t v) { return static_cast<int>(v); };
          if (mine && col < p.N) at[0] = int4v{word(lo[0]), word(hi[0]), word(lo[1]), word(hi[1])};
          if (mine && col + 8 < p.N) at[1] = int4v{word(lo[2]), word(hi[2]), word(lo[3]), word(hi[3])};
        }
      }
    }
    }
    t_now += slots;
    if (t_now >= end) return;
    tile = map.find(t_now);
    step = 0;
    clear();
  }
}

// ------------------------------------------------------- K cut over the wavefronts of a workgroup
//
// 16 TT rows x 16 CT CS columns; KS = 8 / CS wavefronts take every KS-th block of K each, straight from memory, and their
// sums meet in LDS.  Two blocks are on their way while one is multiplied.
//
// In: uint8_t for rows in 8 bits, or half_t or bf16_t for rows that are quantised here, each block of 128 by the four lanes
// that hold it, to the codes of ccf_quantize_rows.  Every workgroup does that again, but hides it behind its weights' loads,
// where a launch for it costs 3.5 us.
template <int TT, int CT, int CS>
struct SplitShape {
  static constexpr int kWaves = 8, KS = kWaves / CS, BM = 16 * TT, BN = 16 * CT * CS, kLd = BN + 4;
  static constexpr size_t kLds = sizeof(float) * KS * BM * kLd;
};

template <int TT, int CT, int CS, int kOut, class In>
__global__ void __launch_bounds__(512, 2)
gemm8_split_kernel(Gemm8Args p, int n_tiles) {
  constexpr bool kCodes = sizeof(In) == 1;
  static_assert(kCodes || TT == 1, "a block of 16 rows is quantised at a time");
  typedef std::conditional_t<kCodes, half_t, In> Raw;
  typedef Raw raw8 __attribute__((ext_vector_type(8)));
  using S = SplitShape<TT, CT, CS>;
  using Out = std::conditional_t<kOut == kGemm8Bf16, bf16_t, half_t>;
  extern __shared__ __attribute__((aligned(16))) float s_part[];           // [KS][BM][kLd]
  const Tile tile = find_tile<S::BM>(p, blockIdx.x, gridDim.x, n_tiles);
  if (tile.e < 0) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g = lane >> 4, ks = wave % S::KS, cs = wave / S::KS;
  const int KB = scale_blocks(p.K), NB = scale_blocks(p.N);
  const int rows = tile.rows < S::BM ? tile.rows : S::BM, n0 = tile.n * S::BN, c0 = n0 + cs * 16 * CT;
  const In *x[TT];
  const float *sa[TT];
#pragma unroll
  for (int t = 0; t < TT; ++t) {
    const int r = 16 * t + r16, j = tile.row0 + (r < rows ? r : rows - 1);
    const size_t row = static_cast<size_t>(p.a_rows ? p.a_rows[j] : j);
    x[t] = reinterpret_cast<const In *>(p.a) + row * p.K + 32 * g;
    sa[t] = p.a_scale + row * KB;
  }
  const uint8_t *w[CT];
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    const int n = c0 + 16 * c + r16;
    w[c] = p.b + (static_cast<size_t>(tile.e) * p.N + (n < p.N ? n : p.N - 1)) * p.K + 32 * g;
  }
  int nb = c0 / kScaleBlock;
  nb = nb < NB ? nb : NB - 1;
  const float *sb = p.b_scale + (static_cast<size_t>(tile.e) * NB + nb) * KB;
  float4v acc[CT][TT];
#pragma unroll
  for (int c = 0; c < CT; ++c)
#pragma unroll
    for (int t = 0; t < TT; ++t) acc[c][t] = float4v{0, 0, 0, 0};

  const int count = KB > ks ? (KB - ks + S::KS - 1) / S::KS : 0;           // blocks ks, ks + KS, ...
  int8v wf[2][CT], xf[2][TT];
  raw8 raw[2][4];
  float sf[2][TT];
  auto piece = [&](const uint8_t *q, int kb) {
    const uint8_t *at = q + static_cast<size_t>(kb) * kScaleBlock;
    const int left = p.K - kb * kScaleBlock - 32 * g;                      // codes of the row from this lane's first on
    const int4v *lo = reinterpret_cast<const int4v *>(left > 0 ? at : reinterpret_cast<const uint8_t *>(&kZeros16));
    const int4v *hi = reinterpret_cast<const int4v *>(left > 16 ? at + 16 : reinterpret_cast<const uint8_t *>(&kZeros16));
    return join(*lo, *hi);
  };
  auto whole = [&](const uint8_t *q, int kb) {
    const int4v *at = reinterpret_cast<const int4v *>(q + static_cast<size_t>(kb) * kScaleBlock);
    return join(at[0], at[1]);
  };
  auto fetch = [&](int i, auto B_) {                                       // the wavefront's block i; past the last one it again
    constexpr int buf = decltype(B_)::value;
    const int kb = ks + (i < count ? i : count - 1) * S::KS;
    const float b = sb[kb];
    if ((kb + 1) * kScaleBlock <= p.K) {                                   // uniform
#pragma unroll
      for (int c = 0; c < CT; ++c) wf[buf][c] = whole(w[c], kb);
      if constexpr (kCodes) {
#pragma unroll
        for (int t = 0; t < TT; ++t) xf[buf][t] = whole(x[t], kb);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) raw[buf][q] = *reinterpret_cast<const raw8 *>(x[0] + static_cast<size_t>(kb) * kScaleBlock + 8 * q);
      }
    } else {
#pragma unroll
      for (int c = 0; c < CT; ++c) wf[buf][c] = piece(w[c], kb);
      if constexpr (kCodes) {
#pragma unroll
        for (int t = 0; t < TT; ++t) xf[buf][t] = piece(x[t], kb);
      } else {
        const int left = p.K - kb * kScaleBlock - 32 * g;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const In *at = x[0] + static_cast<size_t>(kb) * kScaleBlock + 8 * q;
          raw[buf][q] = *reinterpret_cast<const raw8 *>(left > 8 * q ? at : reinterpret_cast<const In *>(&kZeros16));
        }
      }
    }
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      if constexpr (kCodes) sf[buf][t] = sa[t][kb] * b;
      else sf[buf][t] = b;
    }
  };
  auto quantise = [&](auto B_) {                                           // raw[buf] to codes, their scale into sf
    constexpr int buf = decltype(B_)::value;
    float top = 0.0f;
#pragma unroll
    for (int q = 0; q < 32; ++q) top = fmaxf(top, fabsf(static_cast<float>(raw[buf][q / 8][q % 8])));
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    float inverse;
    sf[buf][0] = block_scale(top, &inverse) * sf[buf][0];
    auto v = [&](int q) { return static_cast<float>(raw[buf][q / 8][q % 8]) * inverse; };
#pragma unroll
    for (int q = 0; q < 8; ++q) xf[buf][0][q] = pack_fp8(v(4 * q), v(4 * q + 1), v(4 * q + 2), v(4 * q + 3));
  };
  auto multiply = [&](int i, auto B_) {
    constexpr int buf = decltype(B_)::value;
    if (i >= count) return;                                                // uniform
    if constexpr (!kCodes) quantise(B_);
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      float4v part[TT];
#pragma unroll
      for (int t = 0; t < TT; ++t) part[t] = mfma8(wf[buf][c], xf[buf][t]);
#pragma unroll
      for (int t = 0; t < TT; ++t)
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[c][t][q] = fmaf(part[t][q], sf[buf][t], acc[c][t][q]);
    }
  };
  if (count > 0) {
    constexpr std::integral_constant<int, 0> even{};
    constexpr std::integral_constant<int, 1> odd{};
    fetch(0, even);
    for (int i = 0; i < count; i += 2) {
      fetch(i + 1, odd);
      __builtin_amdgcn_sched_barrier(0);
      multiply(i, even);
      __builtin_amdgcn_sched_barrier(0);
      fetch(i + 2, even);
      __builtin_amdgcn_sched_barrier(0);
      multiply(i + 1, odd);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
#pragma unroll
  for (int c = 0; c < CT; ++c)
#pragma unroll
    for (int t = 0; t < TT; ++t)
      *reinterpret_cast<float4v *>(s_part + (ks * S::BM + 16 * t + r16) * S::kLd + (cs * CT + c) * 16 + 4 * g) = acc[c][t];
  __syncthreads();
  // eight consecutive columns to a thread, 16 threads to a scale's block
  const Out *bias = p.bias ? static_cast<const Out *>(p.bias) + static_cast<size_t>(tile.e) * p.N : nullptr;
  constexpr int kPer = S::BN / 8;
  for (int i = threadIdx.x; i < S::BM * kPer; i += 512) {
    const int r = i / kPer, c = (i % kPer) * 8, col = n0 + c;
    const bool mine = r < rows && col < p.N;
    float v[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = 0.0f;
#pragma unroll
    for (int k = 0; k < S::KS; ++k) {
      const float *part = s_part + (k * S::BM + r) * S::kLd + c;
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] += part[q];
    }
    if (bias && mine) {
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] += static_cast<float>(bias[col + q]);
    }
    const int j = tile.row0 + r;
    const size_t crow = mine && p.c_rows ? static_cast<size_t>(p.c_rows[j]) : static_cast<size_t>(j);
    if constexpr (kOut == kGemm8Gelu8) {
      float top = 0.0f;
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        v[q] = mine ? gelu_erf(v[q]) : 0.0f;
        top = fmaxf(top, fabsf(v[q]));
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
      float inverse;
      const float scale = block_scale(top, &inverse);
      if (mine) {
        if ((i & 15) == 0) p.scales[crow * NB + col / kScaleBlock] = scale;
        *reinterpret_cast<int2v *>(p.codes + crow * p.N + col) =
            int2v{pack_fp8(v[0] * inverse, v[1] * inverse, v[2] * inverse, v[3] * inverse),
                  pack_fp8(v[4] * inverse, v[5] * inverse, v[6] * inverse, v[7] * inverse)};
      }
    } else if (mine) {
      typedef Out out8 __attribute__((ext_vector_type(8)));
      out8 o;
#pragma unroll
      for (int q = 0; q < 8; ++q) o[q] = static_cast<Out>(v[q]);
      *reinterpret_cast<out8 *>(static_cast<Out *>(p.c) + crow * p.N + col) = o;
    }
  }
}

// Workgroups: every tile that the rows may make, in whole rounds of the XCDs.
long long grid_of(const Gemm8Args &p, int bm, int n_tiles) {
  const long long m = p.max_rows / bm + (p.offsets ? (p.E < p.max_rows ? p.E : p.max_rows) : 1);
  return (m * n_tiles + 7) / 8 * 8;
}

int allow_lds(const void *kernel, size_t lds, const char *what) {
  if (lds <= 65536) return CCF_OK;
  hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds));
  return e == hipSuccess ? static_cast<int>(CCF_OK) : fail(CCF_ERR_HIP, "%s: LDS attribute: %s", what, hipGetErrorString(e));
}

// Compute units of the current device, in whole rounds of the 8 XCDs.
int compute_units() {
  static thread_local int cached_dev = -1, cached = 0;
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return 0;
  if (dev != cached_dev) {
    int cus = 0;
    if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess) return 0;
    cached = cus / 8 * 8;
    cached_dev = dev;
  }
  return cached;
}

template <int BM, int BN, int WM, int WN, int NS, int KS, int kOut>
int launch_tiles(const Gemm8Args &p, int part, hipStream_t st, const char *what) {
  using S = TileShape<BM, BN, WM, WN, NS, KS>;
  auto kernel = gemm8_tile_kernel<BM, BN, WM, WN, NS, KS, kOut>;
  const size_t lds = S::kMap + 4 * (3 * p.E + 1);
  const int cus = compute_units(), n_tiles = (p.N + BN - 1) / BN;
  CCF_REQUIRE(cus > 0, CCF_ERR_HIP, "%s: no device", what);
  if (int rc = allow_lds(reinterpret_cast<const void *>(kernel), lds, what)) return rc;
  const long long tiles = part == kLeft ? (static_cast<long long>(n_tiles) * (p.offsets ? p.E : 1) + 7) / 8 * 8 : grid_of(p, BM, n_tiles);
  const long long most = static_cast<long long>(cus) * (160 * 1024 / lds);             // workgroups on the chip at once
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(tiles < most ? tiles : most)), dim3(S::kThreads), lds, st, p, n_tiles, part);
  return check_launch(what);
}

template <int TT, int CT, int CS, int kOut, class In = uint8_t>
int launch_split(const Gemm8Args &p, hipStream_t st, const char *what) {
  using S = SplitShape<TT, CT, CS>;
  auto kernel = gemm8_split_kernel<TT, CT, CS, kOut, In>;
  const int n_tiles = (p.N + S::BN - 1) / S::BN;
  const long long grid = grid_of(p, S::BM, n_tiles);
  CCF_REQUIRE(grid < (1ll << 28), CCF_ERR_SHAPE, "%s: too many tiles", what);
  if (int rc = allow_lds(reinterpret_cast<const void *>(kernel), S::kLds, what)) return rc;
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(grid)), dim3(512), S::kLds, st, p, n_tiles);
  return check_launch(what);
}

// The form by sizes; the experts' row counts are on the device, so their loads are taken as even, and a quarter more.  The
// limits are where measured times cross (us, K -> N, rows of an expert; weights cycled through a graph's replays):
//   K over wavefronts, for at most 16 rows, where one round of workgroups holds them and K is long: 4096 -> 14336, 1 row
//   14.7 and tiles of 64 in two groups 18.4; 8192 -> 2048 of 8 experts, 8 rows 26 and 31; but 4096 -> 1024, 32 rows 19.5 and
//   16.6, 768 -> 2048 7.8 and 6.7, and in two rounds (14336 -> 4096 of 8, 2 rows) 86 and, tiles of 64, 77.
//   Tiles of 64, while there are few tiles: 4096 -> 1024, 512 rows 22, of 128 28, of 256 51; 4096 -> 14336, 333 rows 47, 41, 56;
//   in two groups while a CU has one at most: 17 for 22, 4096 -> 1024 of 8 experts, 139 rows 20 for 23; with a tile on each of
//   256 CUs that wait for weights (14336 -> 4096 of 8) 96 for 77.
//   Tiles of 256 with the rest as a launch of its own, where the whole tiles alone fill the chip: 4096 -> 14336 of 8, 512
//   rows 364, all in tiles of 256 394, of 128 397; but 4096 -> 1024, 4096 rows 56, 54, 32.
//   Tiles of 256, where tiles of 128 go over a round: 4096 -> 14336, 700 rows 60, of 128 68; 512 rows 56 and 45.
enum Form { kSplit = 1, kTiles256, kTiles128, kTiles64, kTilesAndRest, kTiles64Halves };
constexpr long long kOneEach = 192;                  // of 256 CUs have a tile: few enough that two groups to a CU pay
Form form_of(const Gemm8Args &p) {
  constexpr long long kCus = 256;
  const bool grouped = p.offsets != nullptr;
  const long long owners = grouped ? (p.E < p.max_rows ? p.E : p.max_rows) : 1;
  const long long rows = (p.max_rows + owners - 1) / owners, likely = grouped ? rows + rows / 4 : rows;
  auto tiles = [&](int bm, int bn) { return owners * ((likely + bm - 1) / bm) * ((p.N + bn - 1) / bn); };
  if (p.K >= 2048 && (grouped ? 2 * rows : rows) <= 16 && owners * ((p.N + 63) / 64) <= kCus) return kSplit;
  if (owners * (rows / kWholeRows) * ((p.N + 255) / 256) >= kCus) {
    const long long rest = rows % kWholeRows;
    return grouped || (rest > 0 && rest <= kLeftRows) ? kTilesAndRest : kTiles256;          // an empty launch is 4 us
  }
  if (tiles(64, 128) <= kOneEach) return kTiles64Halves;
  if (likely <= 64 || tiles(64, 128) <= 448) return kTiles64;
  if (likely > 128 && tiles(128, 128) >= 640) return kTiles256;
  return kTiles128;
}

template <int kOut>
int gemm8_out(const Gemm8Args &p, hipStream_t st, const char *what) {
  // (the 8-bit output wants all 128 columns of a scale in one workgroup)
  constexpr int CS = kOut == kGemm8Gelu8 ? 2 : 1;
  switch (g_fp8_form ? static_cast<Form>(g_fp8_form) : form_of(p)) {
    case kSplit: return launch_split<1, 4, CS, kOut>(p, st, what);
    case kTiles256: return launch_tiles<256, 256, 4, 2, 2, 1, kOut>(p, kAll, st, what);
    case kTiles128: return launch_tiles<128, 128, 4, 1, 2, 1, kOut>(p, kAll, st, what);
    case kTiles64: return launch_tiles<64, 128, 4, 1, 3, 1, kOut>(p, kAll, st, what);
    case kTiles64Halves: return launch_tiles<64, 128, 4, 1, 2, 2, kOut>(p, kAll, st, what);
    case kTilesAndRest: break;
  }
  if (int rc = launch_tiles<256, 256, 4, 2, 2, 1, kOut>(p, kWhole, st, what)) return rc;
  // (one expert in four has so few rows left, loads being arbitrary)
  const long long left = (p.offsets ? (p.E + 3) / 4 : 1) * static_cast<long long>((p.N + 127) / 128);
  return left <= kOneEach ? launch_tiles<64, 128, 4, 1, 2, 2, kOut>(p, kLeft, st, what)
                          : launch_tiles<64, 128, 4, 1, 3, 1, kOut>(p, kLeft, st, what);
}

}  // namespace

int gemm8(const Gemm8Args &p, int out, hipStream_t st, const char *what) {
  if (p.max_rows == 0 || p.E == 0) return CCF_OK;
  if (out == kGemm8Half) return gemm8_out<kGemm8Half>(p, st, what);
  if (out == kGemm8Bf16) return gemm8_out<kGemm8Bf16>(p, st, what);
  return gemm8_out<kGemm8Gelu8>(p, st, what);
}

namespace {

int check_product(const Gemm8Args &p, const char *what) {
  CCF_REQUIRE(p.max_rows >= 0 && p.E > 0 && p.N > 0 && p.K > 0, CCF_ERR_ARG, "%s: bad size", what);
  CCF_REQUIRE(p.E <= 1024, CCF_ERR_SHAPE, "%s: num_expert=%d beyond 1024", what, p.E);
  CCF_REQUIRE(p.K % 16 == 0 && p.N % 8 == 0, CCF_ERR_SHAPE, "%s: contraction of %d and %d columns: multiples of 16 and 8 are needed",
              what, p.K, p.N);
  // the tile kernel counts 16-byte chunks of the rows, and bytes of an expert's weights, in 32 bits
  CCF_REQUIRE(p.max_rows < (1 << 30) && static_cast<long long>(p.max_rows) * (p.K / 16) < (1ll << 32) &&
                  static_cast<long long>(p.N) * p.K < (1ll << 32), CCF_ERR_SHAPE,
              "%s: %d rows of %d and %d columns: rows times contraction reaches 2^36 or columns times contraction 2^32", what,
              p.max_rows, p.K, p.N);
  if (p.max_rows == 0) return CCF_OK;
  CCF_REQUIRE(p.a && p.a_scale && p.b && p.b_scale && (p.c || (p.codes && p.scales)), CCF_ERR_ARG, "%s: null pointer", what);
  CCF_REQUIRE(aligned16(p.a) && aligned16(p.b) && aligned16(p.c) && aligned16(p.codes) && aligned16(p.bias), CCF_ERR_ARG,
              "%s: rows must be 16-byte aligned", what);
  return CCF_OK;
}

// Whether a dense product of rows in 16 bits takes the kernel that quantises them itself: at most 16 rows, cut over K.
bool quantises(const Gemm8Args &p) {
  return p.max_rows <= 16 && (g_fp8_form ? g_fp8_form == kSplit : form_of(p) == kSplit);
}

size_t codes_bytes(int rows, int k) { return (static_cast<size_t>(rows) * k + 255) / 256 * 256; }

}  // namespace
}  // namespace ccf

extern "C" size_t ccf_linear_fp8_workspace_bytes(int rows, int k) {
  if (rows <= 0 || k <= 0) return 256;
  return ccf::codes_bytes(rows, k) + sizeof(float) * rows * ccf::scale_blocks(k);
}

extern "C" int ccf_linear_fp8_rows(const void *x, int x_dtype, int rows, int k, const void *w_codes, const float *w_scales, int n,
                                   const void *bias, int dtype, void *y, void *workspace, size_t workspace_bytes, ccf_stream_t stream) {
  using namespace ccf;
  CCF_REQUIRE(dtype == CCF_F16 || dtype == CCF_BF16, CCF_ERR_UNSUPPORTED, "linear_fp8: output of type %d", dtype);
  CCF_REQUIRE(x_dtype == CCF_F16 || x_dtype == CCF_BF16 || x_dtype == CCF_F32, CCF_ERR_UNSUPPORTED, "linear_fp8: rows of type %d", x_dtype);
  CCF_REQUIRE(rows == 0 || workspace, CCF_ERR_WORKSPACE, "linear_fp8: no workspace");
  CCF_REQUIRE(aligned16(workspace), CCF_ERR_ARG, "linear_fp8: workspace must be 16-byte aligned");
  uint8_t *codes = static_cast<uint8_t *>(workspace);
  Gemm8Args p{codes, nullptr, nullptr, static_cast<const uint8_t *>(w_codes), w_scales, bias, nullptr, rows, 1, n, k, nullptr, y,
              nullptr, nullptr};
  float *scales = rows > 0 && k > 0 ? reinterpret_cast<float *>(codes + codes_bytes(rows, k)) : nullptr;
  p.a_scale = scales;
  if (int rc = check_product(p, "linear_fp8")) return rc;
  if (rows == 0) return CCF_OK;
  CCF_REQUIRE(x, CCF_ERR_ARG, "linear_fp8: null pointer");
  CCF_REQUIRE(reinterpret_cast<uintptr_t>(x) % (x_dtype == CCF_F32 ? 4 : 2) == 0, CCF_ERR_ARG, "linear_fp8: x is not aligned to its type");
  CCF_REQUIRE(workspace_bytes >= ccf_linear_fp8_workspace_bytes(rows, k), CCF_ERR_WORKSPACE, "linear_fp8: workspace too small");
  const hipStream_t st = as_stream(stream);
  if (x_dtype != CCF_F32 && aligned16(x) && quantises(p)) {
    p.a = static_cast<const uint8_t *>(x);
    auto run = [&](auto in, auto out) {
      return launch_split<1, 4, 1, decltype(out)::value, decltype(in)>(p, st, "linear_fp8");
    };
    constexpr std::integral_constant<int, kGemm8Half> half{};
    constexpr std::integral_constant<int, kGemm8Bf16> bf{};
    if (x_dtype == CCF_F16) return dtype == CCF_F16 ? run(half_t{}, half) : run(half_t{}, bf);
    return dtype == CCF_F16 ? run(bf16_t{}, half) : run(bf16_t{}, bf);
  }
  if (int rc = launch_quantize_rows(x, rows, k, x_dtype, codes, scales, st)) return rc;
  return gemm8(p, dtype == CCF_F16 ? kGemm8Half : kGemm8Bf16, st, "linear_fp8");
}

extern "C" int ccf_linear_fp8(const void *x_codes, const float *x_scales, int rows, int k, const void *w_codes,
                              const float *w_scales, int n, const void *bias, int dtype, void *y, ccf_stream_t stream) {
  using namespace ccf;
  CCF_REQUIRE(dtype == CCF_F16 || dtype == CCF_BF16, CCF_ERR_UNSUPPORTED, "linear_fp8: output of type %d", dtype);
  const Gemm8Args p{static_cast<const uint8_t *>(x_codes), x_scales, nullptr, static_cast<const uint8_t *>(w_codes), w_scales, bias,
                    nullptr, rows, 1, n, k, nullptr, y, nullptr, nullptr};
  if (int rc = check_product(p, "linear_fp8")) return rc;
  return gemm8(p, dtype == CCF_F16 ? kGemm8Half : kGemm8Bf16, as_stream(stream), "linear_fp8");
}

extern "C" int ccf_ffn1_fp8(const void *x_codes, const float *x_scales, const int32_t *src_row, const int32_t *offsets, int max_rows,
                            int num_expert, int d_model, int d_ffn, const void *w1_codes, const float *w1_scales, const void *b1,
                            void *h_codes, float *h_scales, ccf_stream_t stream) {
  using namespace ccf;
  const Gemm8Args p{static_cast<const uint8_t *>(x_codes), x_scales, src_row, static_cast<const uint8_t *>(w1_codes), w1_scales, b1,
                    offsets, max_rows, num_expert, d_ffn, d_model, nullptr, nullptr, static_cast<uint8_t *>(h_codes), h_scales};
  if (int rc = check_product(p, "ffn1_fp8")) return rc;
  CCF_REQUIRE(offsets || max_rows == 0, CCF_ERR_ARG, "ffn1_fp8: null pointer");
  return gemm8(p, kGemm8Gelu8, as_stream(stream), "ffn1_fp8");
}

extern "C" int ccf_ffn2_fp8(const void *h_codes, const float *h_scales, const int32_t *dst_row, const int32_t *offsets, int max_rows,
                            int num_expert, int d_model, int d_ffn, const void *w2_codes, const float *w2_scales, const void *b2,
                            void *y, ccf_stream_t stream) {
  using namespace ccf;
  const Gemm8Args p{static_cast<const uint8_t *>(h_codes), h_scales, nullptr, static_cast<const uint8_t *>(w2_codes), w2_scales, b2,
                    offsets, max_rows, num_expert, d_model, d_ffn, dst_row, y, nullptr, nullptr};
  if (int rc = check_product(p, "ffn2_fp8")) return rc;
  CCF_REQUIRE(offsets || max_rows == 0, CCF_ERR_ARG, "ffn2_fp8: null pointer");
  return gemm8(p, kGemm8Half, as_stream(stream), "ffn2_fp8");
}
