// Root-mean-square norm with the residual's addition and an output in 8 bits, and its backward, for gfx950 (HBM-bound).
//
//   total = x + residual, rounded to the rows' type: the residual stream that the next block reads
//   y     = total * rstd * weight,  rstd = 1 / sqrt(mean(total^2) + eps)
//   codes, scales: y in e4m3 with a scale for each block of 128 columns, from the fp32 value (one rounding; y itself is
//   another one of the same value)
//
// The norm is taken of the rounded total, so that a caller who adds first gets the same bits and the backward, which is
// given the total, differentiates what the forward computed.  Sums, rstd and products are fp32.
//
//   grad_x = grad_total + rstd (g w - total rstd^2 mean(g w total)),  grad_weight = sum over rows of g total rstd
//
// One pass: a row stays in the registers of its threads (8 consecutive elements each, 16 lanes to a scale's block) between
// the loads, the sum and the stores.  Rows too long for that are read again.  The backward keeps a thread's columns of the
// weight gradient in registers over all rows of a workgroup, and a second launch adds the workgroups' sums in order.
//
// Measured, bf16 with a residual, 16384 x 4096: forward 98.8 us, 5.4 TB/s (1 GiB copied: 5.1); backward with both gradients
// 139.7 us, 3.8 TB/s (of its four streams one is written); quantize_rows 31.9 us, 6.3 TB/s.  8 x 14336 x 4096 fp16 weights to
// 8 bits 279 us, 5.1 TB/s.  One row of 4096: 3.9, 6.5 and 2.8 us, a launch's own time.
#include "fp8.h"

#include <type_traits>

namespace ccf {
namespace {

// 8 elements at any address: rows of odd length start anywhere, and the hardware takes unaligned wide accesses
template <typename T>
struct Vec8 {
  typedef T type __attribute__((ext_vector_type(8)));
  struct __attribute__((packed, aligned(sizeof(T) < 4 ? sizeof(T) : 4))) Any {
    type v;
  };
};

template <typename T>
__device__ __forceinline__ void load8(const T *p, int n, float (&out)[8]) {        // n valid elements, zeros behind them
  if (n >= 8) {
    const typename Vec8<T>::type v = reinterpret_cast<const typename Vec8<T>::Any *>(p)->v;
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = static_cast<float>(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = i < n ? static_cast<float>(p[i]) : 0.0f;
  }
}

template <typename T>
__device__ __forceinline__ void store8(T *p, int n, const float (&in)[8]) {
  if (n >= 8) {
    typename Vec8<T>::type v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = static_cast<T>(in[i]);
    reinterpret_cast<typename Vec8<T>::Any *>(p)->v = v;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = static_cast<T>(in[i]);
  }
}

__device__ __forceinline__ void store_codes(uint8_t *p, int n, const float (&v)[8], float inverse) {
  const int lo = pack_fp8(v[0] * inverse, v[1] * inverse, v[2] * inverse, v[3] * inverse);
  const int hi = pack_fp8(v[4] * inverse, v[5] * inverse, v[6] * inverse, v[7] * inverse);
  if (n >= 8) {
    struct __attribute__((packed, aligned(1))) Any {
      int lo, hi;
    };
    *reinterpret_cast<Any *>(p) = Any{lo, hi};
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = static_cast<uint8_t>((i < 4 ? lo : hi) >> (8 * (i & 3)));
  }
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// Largest magnitude of the 16 lanes (128 elements) around this one.
__device__ __forceinline__ float block_top(const float (&v)[8]) {
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[i]));
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  return top;
}

// Sum over the TPR threads of a row; s_sum holds one float per wavefront.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float *s_sum) {
  v = wave_sum(v);
  if constexpr (TPR > 64) {
    if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int i = 0; i < TPR / 64; ++i) v += s_sum[i];
  }
  return v;
}

struct NormArgs {
  const void *x, *residual, *weight;
  int rows, d;
  float eps;
  void *y, *total;
  uint8_t *codes;
  float *scales, *rstd;
};

// TPR threads per row (a workgroup holds 256 / TPR rows when TPR < 256), NV chunks of 8 elements per thread; kLong: rows
// beyond TPR * NV * 8 elements, read a second time.
template <typename T, typename W, int TPR, int NV, bool kLong>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR)
rms_norm_kernel(NormArgs p) {
  constexpr int kRows = TPR < 256 ? 256 / TPR : 1;
  __shared__ float s_sum[TPR / 64 < 1 ? 1 : TPR / 64];
  const int lane = threadIdx.x % TPR;
  const int row = blockIdx.x * kRows + threadIdx.x / TPR;
  if (row >= p.rows) return;                       // whole wavefronts; with a barrier below a workgroup has one row
  const size_t at = static_cast<size_t>(row) * p.d;
  const T *x = static_cast<const T *>(p.x) + at, *res = p.residual ? static_cast<const T *>(p.residual) + at : nullptr;
  const W *w = static_cast<const W *>(p.weight);
  T *total = p.total ? static_cast<T *>(p.total) + at : nullptr, *y = p.y ? static_cast<T *>(p.y) + at : nullptr;
  float v[NV][8];
  auto fetch = [&](int c0, bool first) {           // chunks c0 + ... of the row: added, rounded and, the first time, written
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (c0 + i * TPR + lane) * 8, n = p.d - c;
      if (n > 0) {
        load8(x + c, n, v[i]);
        if (res) {
          float r[8];
          load8(res + c, n, r);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[i][j] = static_cast<float>(static_cast<T>(v[i][j] + r[j]));
          if (first && total) store8(total + c, n, v[i]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
      }
    }
  };
  float sum = 0.0f;
  const int chunks = (p.d + 7) / 8;
  const int span = kLong ? chunks : 1;             // kLong: several turns over the row
  for (int c0 = 0; c0 < span; c0 += TPR * NV) {
    fetch(c0, true);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) sum = fmaf(v[i][j], v[i][j], sum);
  }
  sum = row_sum<TPR>(sum, s_sum);
  const float rstd = 1.0f / sqrtf(sum / static_cast<float>(p.d) + p.eps);
  if (p.rstd && lane == 0) p.rstd[row] = rstd;
  const int blocks = scale_blocks(p.d);
  for (int c0 = 0; c0 < span; c0 += TPR * NV) {
    if constexpr (kLong) fetch(c0, false);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (c0 + i * TPR + lane) * 8, n = p.d - c;
      float g[8], o[8];
      if (n > 0) {
        load8(w + c, n, g);
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = v[i][j] * rstd * g[j];
        if (y) store8(y + c, n, o);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = 0.0f;
      }
      if (p.codes) {
        float inverse;
        const float scale = block_scale(block_top(o), &inverse);
        if (n > 0) {
          store_codes(p.codes + at + c, n, o, inverse);
          if ((lane & 15) == 0) p.scales[static_cast<size_t>(row) * blocks + c / kScaleBlock] = scale;
        }
      }
    }
  }
}

template <typename T, typename W>
int launch_norm(const NormArgs &p, hipStream_t st) {
  // a row's threads: a wavefront up to 1024 elements, so that several rows share a workgroup and none needs a barrier
  const int d = p.d;
  void (*kernel)(NormArgs);
  int tpr;
  if (d <= 512) kernel = rms_norm_kernel<T, W, 64, 1, false>, tpr = 64;
  else if (d <= 1024) kernel = rms_norm_kernel<T, W, 64, 2, false>, tpr = 64;
  else if (d <= 2048) kernel = rms_norm_kernel<T, W, 256, 1, false>, tpr = 256;
  else if (d <= 4096) kernel = rms_norm_kernel<T, W, 256, 2, false>, tpr = 256;
  else if (d <= 8192) kernel = rms_norm_kernel<T, W, 512, 2, false>, tpr = 512;
  else if (d <= 16384) kernel = rms_norm_kernel<T, W, 1024, 2, false>, tpr = 1024;
  else kernel = rms_norm_kernel<T, W, 1024, 2, true>, tpr = 1024;
  const int rows_wg = tpr < 256 ? 256 / tpr : 1;
  hipLaunchKernelGGL(kernel, dim3((p.rows + rows_wg - 1) / rows_wg), dim3(tpr < 256 ? 256 : tpr), 0, st, p);
  return check_launch("rms_norm_kernel");
}

struct NormBwdArgs {
  const void *grad_y, *total, *weight, *grad_total;
  const float *rstd;
  int rows, d, rows_wg;                            // rows of a workgroup
  void *grad_x;
  float *partial;                                  // [workgroups][d] or null
};

template <typename T, typename W, int TPR, int NV>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR)
rms_norm_backward_kernel(NormBwdArgs p) {
  constexpr int kRows = TPR < 256 ? 256 / TPR : 1;   // rows at a time
  __shared__ float s_sum[2][TPR / 64 < 1 ? 1 : TPR / 64];
  extern __shared__ float s_part[];                // kRows > 1: [kRows][TPR * NV * 8]
  const int lane = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  float w[NV][8], gw[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + lane) * 8, n = p.d - c;
#pragma unroll
    for (int j = 0; j < 8; ++j) w[i][j] = gw[i][j] = 0.0f;
    if (n > 0) load8(static_cast<const W *>(p.weight) + c, n, w[i]);
  }
  const int first = blockIdx.x * p.rows_wg, last = first + p.rows_wg < p.rows ? first + p.rows_wg : p.rows;
  int turn = 0;
  for (int r0 = first; r0 < last; r0 += kRows, ++turn) {
    const int row = r0 + sub;
    const bool live = row < last;
    const size_t at = static_cast<size_t>(live ? row : last - 1) * p.d;
    const float rstd = p.rstd[live ? row : last - 1];
    float g[NV][8], t[NV][8];
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * 8, n = p.d - c;
#pragma unroll
      for (int j = 0; j < 8; ++j) g[i][j] = t[i][j] = 0.0f;
      if (n > 0) {
        load8(static_cast<const T *>(p.grad_y) + at + c, n, g[i]);
        load8(static_cast<const T *>(p.total) + at + c, n, t[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (live) gw[i][j] = fmaf(g[i][j], t[i][j] * rstd, gw[i][j]);
        g[i][j] *= w[i][j];
        sum = fmaf(g[i][j], t[i][j], sum);
      }
    sum = row_sum<TPR>(sum, s_sum[turn & 1]);      // two places in turn: one barrier a row
    const float c1 = -rstd * rstd * (sum / static_cast<float>(p.d));
    if (p.grad_x && live) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * TPR + lane) * 8, n = p.d - c;
        if (n <= 0) continue;
        float o[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = rstd * fmaf(c1, t[i][j], g[i][j]);
        if (p.grad_total) {
          float gt[8];
          load8(static_cast<const T *>(p.grad_total) + at + c, n, gt);
#pragma unroll
          for (int j = 0; j < 8; ++j) o[j] += gt[j];
        }
        store8(static_cast<T *>(p.grad_x) + at + c, n, o);
      }
    }
  }
  if (!p.partial) return;
  float *out = p.partial + static_cast<size_t>(blockIdx.x) * p.d;
  if constexpr (kRows > 1) {
    constexpr int kRow = TPR * NV * 8;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) s_part[sub * kRow + (i * 8 + j) * TPR + lane] = gw[i][j];
    __syncthreads();
    for (int q = threadIdx.x; q < kRow; q += 256) {
      float v = s_part[q];
#pragma unroll
      for (int r = 1; r < kRows; ++r) v += s_part[r * kRow + q];
      const int l = q % TPR, ij = q / TPR, c = ((ij >> 3) * TPR + l) * 8 + (ij & 7);
      if (c < p.d) out[c] = v;
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * 8, n = p.d - c;
      if (n > 0) store8(out + c, n, gw[i]);
    }
  }
}

// Rows too long for registers: two turns over the row, the weight gradient by a second kernel over columns.
template <typename T, typename W>
__global__ void __launch_bounds__(1024)
rms_norm_backward_long_kernel(NormBwdArgs p) {
  __shared__ float s_sum[16];
  const int row = blockIdx.x;
  const size_t at = static_cast<size_t>(row) * p.d;
  const T *gy = static_cast<const T *>(p.grad_y) + at, *tt = static_cast<const T *>(p.total) + at;
  const float rstd = p.rstd[row];
  float sum = 0.0f;
  for (int c = threadIdx.x * 8; c < p.d; c += 8192) {
    float g[8], t[8], w[8];
    load8(gy + c, p.d - c, g);
    load8(tt + c, p.d - c, t);
    load8(static_cast<const W *>(p.weight) + c, p.d - c, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) sum = fmaf(g[j] * w[j], t[j], sum);
  }
  sum = row_sum<1024>(sum, s_sum);
  const float c1 = -rstd * rstd * (sum / static_cast<float>(p.d));
  for (int c = threadIdx.x * 8; c < p.d; c += 8192) {
    float g[8], t[8], w[8];
    load8(gy + c, p.d - c, g);
    load8(tt + c, p.d - c, t);
    load8(static_cast<const W *>(p.weight) + c, p.d - c, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) g[j] = rstd * fmaf(c1, t[j], g[j] * w[j]);
    if (p.grad_total) {
      float gt[8];
      load8(static_cast<const T *>(p.grad_total) + at + c, p.d - c, gt);
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] += gt[j];
    }
    store8(static_cast<T *>(p.grad_x) + at + c, p.d - c, g);
  }
}

template <typename T>
__global__ void __launch_bounds__(256)
rms_norm_weight_long_kernel(NormBwdArgs p) {
  const int c = (blockIdx.x * 256 + threadIdx.x) * 8;
  if (c >= p.d) return;
  const int first = blockIdx.y * p.rows_wg, last = first + p.rows_wg < p.rows ? first + p.rows_wg : p.rows;
  float gw[8] = {};
  for (int row = first; row < last; ++row) {
    const size_t at = static_cast<size_t>(row) * p.d + c;
    const float rstd = p.rstd[row];
    float g[8], t[8];
    load8(static_cast<const T *>(p.grad_y) + at, p.d - c, g);
    load8(static_cast<const T *>(p.total) + at, p.d - c, t);
#pragma unroll
    for (int j = 0; j < 8; ++j) gw[j] = fmaf(g[j], t[j] * rstd, gw[j]);
  }
  store8(p.partial + static_cast<size_t>(blockIdx.y) * p.d + c, p.d - c, gw);
}

// grad_weight[c] = sum over the workgroups' rows of partial, in a fixed order: a wavefront's lanes are 64 columns, the
// wavefronts take every 16th row, their sums meet in LDS.
template <typename W>
__global__ void __launch_bounds__(1024)
rms_norm_weight_kernel(const float *__restrict__ partial, int n, int d, W *__restrict__ out) {
  __shared__ float s_sum[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
  float v = 0.0f;
  if (c < d) {
    int r = wave;
    for (; r + 48 < n; r += 64) {                  // four loads on their way
      const float a = partial[static_cast<size_t>(r) * d + c], b = partial[static_cast<size_t>(r + 16) * d + c];
      const float e = partial[static_cast<size_t>(r + 32) * d + c], f = partial[static_cast<size_t>(r + 48) * d + c];
      v += a;
      v += b;
      v += e;
      v += f;
    }
    for (; r < n; r += 16) v += partial[static_cast<size_t>(r) * d + c];
  }
  s_sum[wave][lane] = v;
  __syncthreads();
  if (wave == 0 && c < d) {
    for (int i = 1; i < 16; ++i) v += s_sum[i][lane];
    out[c] = static_cast<W>(v);
  }
}

constexpr int kNormLong = 16384;                   // longest row that stays in registers

// Rows of a workgroup of the backward: few enough workgroups that their partial sums (one row of fp32 each) are a small
// part of the traffic, enough to fill the chip.
int backward_rows(int rows, int d) {
  const int at_once = d <= 1024 ? 4 : 1;
  const int wgs = d > kNormLong ? 64 : (d <= 2048 ? 1024 : 768);
  int per = (rows + wgs - 1) / wgs;
  return (per + at_once - 1) / at_once * at_once;
}

template <typename T, typename W>
int launch_norm_backward(const NormBwdArgs &p, void *grad_weight, hipStream_t st) {
  const int d = p.d, wgs = (p.rows + p.rows_wg - 1) / p.rows_wg;
  if (d > kNormLong) {
    if (p.grad_x) {
      hipLaunchKernelGGL((rms_norm_backward_long_kernel<T, W>), dim3(p.rows), dim3(1024), 0, st, p);
      if (int rc = check_launch("rms_norm_backward_long_kernel")) return rc;
    }
    if (grad_weight) {
      hipLaunchKernelGGL(rms_norm_weight_long_kernel<T>, dim3((d + 2047) / 2048, wgs), dim3(256), 0, st, p);
      if (int rc = check_launch("rms_norm_weight_long_kernel")) return rc;
    }
  } else {
    void (*kernel)(NormBwdArgs);
    int tpr, nv = 2;
    if (d <= 512) kernel = rms_norm_backward_kernel<T, W, 64, 1>, tpr = 64, nv = 1;
    else if (d <= 1024) kernel = rms_norm_backward_kernel<T, W, 64, 2>, tpr = 64;
    else if (d <= 2048) kernel = rms_norm_backward_kernel<T, W, 256, 1>, tpr = 256, nv = 1;
    else if (d <= 4096) kernel = rms_norm_backward_kernel<T, W, 256, 2>, tpr = 256;
    else if (d <= 8192) kernel = rms_norm_backward_kernel<T, W, 512, 2>, tpr = 512;
    else kernel = rms_norm_backward_kernel<T, W, 1024, 2>, tpr = 1024;
    const size_t lds = tpr < 256 ? sizeof(float) * 256 * nv * 8 : 0;
    hipLaunchKernelGGL(kernel, dim3(wgs), dim3(tpr < 256 ? 256 : tpr), lds, st, p);
    if (int rc = check_launch("rms_norm_backward_kernel")) return rc;
  }
  if (!grad_weight) return CCF_OK;
  hipLaunchKernelGGL(rms_norm_weight_kernel<W>, dim3((d + 63) / 64), dim3(1024), 0, st, p.partial, wgs, d,
                     static_cast<W *>(grad_weight));
  return check_launch("rms_norm_weight_kernel");
}

// f(rows' type, weight's type) for the pairs that there are: one type, or 16-bit rows and an fp32 weight
template <typename F>
int with_types(int dtype, int weight_dtype, F f) {
  if (dtype == CCF_F16 && weight_dtype == CCF_F16) return f(half_t(), half_t());
  if (dtype == CCF_F16 && weight_dtype == CCF_F32) return f(half_t(), float());
  if (dtype == CCF_BF16 && weight_dtype == CCF_BF16) return f(bf16_t(), bf16_t());
  if (dtype == CCF_BF16 && weight_dtype == CCF_F32) return f(bf16_t(), float());
  if (dtype == CCF_F32 && weight_dtype == CCF_F32) return f(float(), float());
  return fail(CCF_ERR_UNSUPPORTED, "rms_norm: rows of type %d with a weight of type %d", dtype, weight_dtype);
}

bool aligned_to(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
size_t type_bytes(int dtype) { return dtype == CCF_F32 ? 4 : 2; }

// ------------------------------------------------------------------ rows and weights to 8 bits
template <typename T>
__global__ void __launch_bounds__(256)
quantize_rows_kernel(const T *__restrict__ x, long long pieces, int k, int blocks, uint8_t *__restrict__ codes,
                     float *__restrict__ scales) {
  // 16 lanes to a block of 128 elements
  for (long long i = blockIdx.x * 16ll + (threadIdx.x >> 4); i < pieces; i += gridDim.x * 16ll) {
    const long long row = i / blocks;
    const int b = static_cast<int>(i - row * blocks), c = b * kScaleBlock + (threadIdx.x & 15) * 8, n = k - c;
    float v[8] = {}, inverse;
    const size_t at = static_cast<size_t>(row) * k + c;
    if (n > 0) load8(x + at, n, v);
    const float scale = block_scale(block_top(v), &inverse);
    if (n > 0) store_codes(codes + at, n, v, inverse);
    if ((threadIdx.x & 15) == 0) scales[i] = scale;
  }
}

// One workgroup per block of 128 x 128: 16 lanes to a row, 16 rows at a time, the values kept in registers.
template <typename T>
__global__ void __launch_bounds__(256)
quantize_weight_kernel(const T *__restrict__ w, int n, int k, int nb, int kb, uint8_t *__restrict__ codes,
                       float *__restrict__ scales) {
  __shared__ float s_top[4];
  const long long blk = blockIdx.x;
  const int bk = static_cast<int>(blk % kb), bn = static_cast<int>(blk / kb % nb);
  const size_t e = static_cast<size_t>(blk / kb / nb);
  const int c = bk * kScaleBlock + (threadIdx.x & 15) * 8, left = k - c;
  float v[8][8], top = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = bn * kScaleBlock + i * 16 + (threadIdx.x >> 4);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
    if (r < n && left > 0) load8(w + (e * n + r) * k + c, left, v[i]);
    top = fmaxf(top, block_top(v[i]));
  }
  top = fmaxf(top, __shfl_xor(top, 16));
  top = fmaxf(top, __shfl_xor(top, 32));
  if ((threadIdx.x & 63) == 0) s_top[threadIdx.x >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf(s_top[0], s_top[1]), fmaxf(s_top[2], s_top[3]));
  float inverse;
  const float scale = block_scale(top, &inverse);
  if (threadIdx.x == 0) scales[blk] = scale;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = bn * kScaleBlock + i * 16 + (threadIdx.x >> 4);
    if (r < n && left > 0) store_codes(codes + (e * n + r) * k + c, left, v[i], inverse);
  }
}

template <typename F>
int with_type(int dtype, const char *what, F f) {
  if (dtype == CCF_F16) return f(half_t());
  if (dtype == CCF_BF16) return f(bf16_t());
  if (dtype == CCF_F32) return f(float());
  return fail(CCF_ERR_UNSUPPORTED, "%s: type %d", what, dtype);
}

}  // namespace

int launch_quantize_rows(const void *x, int rows, int k, int dtype, uint8_t *codes, float *scales, hipStream_t st) {
  if (rows == 0) return CCF_OK;
  const int blocks = scale_blocks(k);
  const long long pieces = static_cast<long long>(rows) * blocks, wgs = (pieces + 15) / 16;
  return with_type(dtype, "quantize_rows", [&](auto t) {
    using T = decltype(t);
    hipLaunchKernelGGL(quantize_rows_kernel<T>, dim3(static_cast<unsigned>(wgs < 16384 ? wgs : 16384)), dim3(256), 0, st,
                       static_cast<const T *>(x), pieces, k, blocks, codes, scales);
    return check_launch("quantize_rows_kernel");
  });
}

}  // namespace ccf

extern "C" int ccf_rms_norm(const void *x, const void *residual, const void *weight, int rows, int d, float eps, int dtype,
                            int weight_dtype, void *y, void *total, void *codes, float *scales, float *rstd,
                            ccf_stream_t stream) {
  using namespace ccf;
  CCF_REQUIRE(rows >= 0 && d > 0 && d <= (1 << 24), CCF_ERR_ARG, "rms_norm: bad size");
  if (rows == 0) return CCF_OK;                    // tensors of no rows have no address
  CCF_REQUIRE(x && weight && (y || codes), CCF_ERR_ARG, "rms_norm: null pointer");
  CCF_REQUIRE((codes == nullptr) == (scales == nullptr), CCF_ERR_ARG, "rms_norm: codes and scales go together");
  CCF_REQUIRE(!residual == !total, CCF_ERR_ARG, "rms_norm: a residual and its total go together");
  CCF_REQUIRE(eps >= 0.0f, CCF_ERR_ARG, "rms_norm: eps below zero");
  const size_t a = type_bytes(dtype);
  CCF_REQUIRE(aligned_to(x, a) && aligned_to(residual, a) && aligned_to(y, a) && aligned_to(total, a) &&
                  aligned_to(weight, type_bytes(weight_dtype)) && aligned_to(scales, 4) && aligned_to(rstd, 4),
              CCF_ERR_ARG, "rms_norm: a pointer is not aligned to its type");
  return with_types(dtype, weight_dtype, [&](auto t, auto w) {
    return launch_norm<decltype(t), decltype(w)>(
        NormArgs{x, residual, weight, rows, d, eps, y, total, static_cast<uint8_t *>(codes), scales, rstd}, as_stream(stream));
  });
}

extern "C" size_t ccf_rms_norm_backward_workspace_bytes(int rows, int d) {
  if (rows <= 0 || d <= 0) return 0;
  const int per = ccf::backward_rows(rows, d);
  return sizeof(float) * static_cast<size_t>((rows + per - 1) / per) * d;
}

extern "C" int ccf_rms_norm_backward(const void *grad_y, const void *total, const void *weight, const float *rstd,
                                     const void *grad_total, int rows, int d, int dtype, int weight_dtype, void *grad_x,
                                     void *grad_weight, void *workspace, size_t workspace_bytes, ccf_stream_t stream) {
  using namespace ccf;
  CCF_REQUIRE(rows >= 0 && d > 0 && d <= (1 << 24), CCF_ERR_ARG, "rms_norm_backward: bad size");
  if (rows == 0 && !grad_weight) return CCF_OK;
  CCF_REQUIRE(weight && (grad_x || grad_weight) && (rows == 0 || (grad_y && total && rstd)), CCF_ERR_ARG,
              "rms_norm_backward: null pointer");
  const size_t need = grad_weight ? ccf_rms_norm_backward_workspace_bytes(rows, d) : 0;
  CCF_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), CCF_ERR_WORKSPACE,
              "rms_norm_backward: workspace of %zu bytes needed, %zu given", need, workspace_bytes);
  const size_t a = type_bytes(dtype);
  CCF_REQUIRE(aligned_to(grad_y, a) && aligned_to(total, a) && aligned_to(grad_total, a) && aligned_to(grad_x, a) &&
                  aligned_to(weight, type_bytes(weight_dtype)) && aligned_to(grad_weight, type_bytes(weight_dtype)) &&
                  aligned_to(rstd, 4) && aligned_to(workspace, 4),
              CCF_ERR_ARG, "rms_norm_backward: a pointer is not aligned to its type");
  return with_types(dtype, weight_dtype, [&](auto t, auto w) {
    using W = decltype(w);
    if (rows == 0) {
      hipLaunchKernelGGL(rms_norm_weight_kernel<W>, dim3((d + 63) / 64), dim3(1024), 0, as_stream(stream),
                         static_cast<const float *>(nullptr), 0, d, static_cast<W *>(grad_weight));
      return check_launch("rms_norm_weight_kernel");
    }
    return launch_norm_backward<decltype(t), W>(
        NormBwdArgs{grad_y, total, weight, grad_total, rstd, rows, d, backward_rows(rows, d), grad_x,
                    grad_weight ? static_cast<float *>(workspace) : nullptr},
        grad_weight, as_stream(stream));
  });
}

extern "C" int ccf_quantize_rows(const void *x, int rows, int k, int dtype, void *codes, float *scales, ccf_stream_t stream) {
  using namespace ccf;
  CCF_REQUIRE(rows >= 0 && k > 0, CCF_ERR_ARG, "quantize_rows: bad size");
  CCF_REQUIRE(rows == 0 || (x && codes && scales), CCF_ERR_ARG, "quantize_rows: null pointer");
  CCF_REQUIRE(aligned_to(x, type_bytes(dtype)) && aligned_to(scales, 4), CCF_ERR_ARG,
              "quantize_rows: a pointer is not aligned to its type");
  return launch_quantize_rows(x, rows, k, dtype, static_cast<uint8_t *>(codes), scales, as_stream(stream));
}

extern "C" int ccf_quantize_weight(const void *w, int num_expert, int n, int k, int dtype, void *codes, float *scales,
                                   ccf_stream_t stream) {
  using namespace ccf;
  CCF_REQUIRE(num_expert >= 0 && n > 0 && k > 0, CCF_ERR_ARG, "quantize_weight: bad size");
  CCF_REQUIRE(num_expert == 0 || (w && codes && scales), CCF_ERR_ARG, "quantize_weight: null pointer");
  CCF_REQUIRE(aligned_to(w, type_bytes(dtype)) && aligned_to(scales, 4), CCF_ERR_ARG,
              "quantize_weight: a pointer is not aligned to its type");
  const int nb = scale_blocks(n), kb = scale_blocks(k);
  const long long wgs = static_cast<long long>(num_expert) * nb * kb;
  CCF_REQUIRE(wgs < (1ll << 31), CCF_ERR_SHAPE, "quantize_weight: too many blocks");
  if (wgs == 0) return CCF_OK;
  return with_type(dtype, "quantize_weight", [&](auto t) {
    using T = decltype(t);
    hipLaunchKernelGGL(quantize_weight_kernel<T>, dim3(static_cast<unsigned>(wgs)), dim3(256), 0, as_stream(stream),
                       static_cast<const T *>(w), n, k, nb, kb, static_cast<uint8_t *>(codes), scales);
    return check_launch("quantize_weight_kernel");
  });
}
