// Layer norm over the last dimension, forward and backward, with the reduction of the weight's and bias' gradients.
//
//   forward    mean = sum x / C,  var = sum (x - mean)^2 / C,  y = (x - mean) rstd w + b
//   backward   xh = (x - mean) rstd,  g = dy w,  dx = rstd (g - mean(g) - xh mean(g xh)),
//              dw = sum_rows dy xh,  db = sum_rows dy
//
// Bound by HBM: the forward pass must read x and write y, the backward pass must read x and dy and write dx.
#include <cuda_bf16.h>

#include <algorithm>

#include "../../include/symplex_b200.h"
#include "host_api.h"
#include "sm100_ptx.cuh"

namespace sx {
namespace {

constexpr int LN_THREADS = 256;
constexpr int LN_PARTS = 320;      // upper bound of the partial rows a column reduction is split into
constexpr int LN_COL_TILE = 32;    // columns of one CTA of the column reductions

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum of v over the CTA, the same value in every thread. `red` is a shared array of 32 floats.
__device__ __forceinline__ float cta_sum(float v, float* red) {
  v = warp_sum(v);
  __syncthreads();  // the previous use of red is over
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  const int warps = blockDim.x >> 5;
  float s = (threadIdx.x & 31) < warps ? red[threadIdx.x & 31] : 0.0f;
  return warp_sum(s);
}

// One CTA per row, the row read three times (twice from L2): rows of any length and alignment.
template <typename T, typename W>
__global__ void __launch_bounds__(LN_THREADS)
ln_forward_any_kernel(const T* x, const W* __restrict__ w, const W* __restrict__ b, T* y, float* __restrict__ mean_out,
                      float* __restrict__ rstd_out, long long rows, long long cols, long long ldx, long long ldy, float eps) {
  __shared__ float red[32];
  pdl_launch_dependents();
  pdl_wait_prior_grids();
  const float inv = 1.0f / (float)cols;
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = x + r * ldx;
    T* yr = y + r * ldy;
    float s = 0.0f;
    for (long long c = threadIdx.x; c < cols; c += LN_THREADS) s += float(xr[c]);
    const float mean = cta_sum(s, red) * inv;
    float q = 0.0f;
    for (long long c = threadIdx.x; c < cols; c += LN_THREADS) {
      const float d = float(xr[c]) - mean;
      q = fmaf(d, d, q);
    }
    const float rstd = 1.0f / sqrtf(cta_sum(q, red) * inv + eps);
    if (threadIdx.x == 0) {
      if (mean_out != nullptr) mean_out[r] = mean;
      if (rstd_out != nullptr) rstd_out[r] = rstd;
    }
    for (long long c = threadIdx.x; c < cols; c += LN_THREADS) {
      float v = (float(xr[c]) - mean) * rstd;
      if (w != nullptr) v *= float(w[c]);
      if (b != nullptr) v += float(b[c]);
      yr[c] = T(v);
    }
  }
}

// dx of one row per CTA, rows of any length and alignment.
template <typename T, typename W>
__global__ void __launch_bounds__(LN_THREADS)
ln_backward_dx_any_kernel(const T* dy, const T* __restrict__ x, const float* __restrict__ mean_in,
                          const float* __restrict__ rstd_in, const W* __restrict__ w, T* dx, long long rows, long long cols,
                          long long lddy, long long ldx, long long lddx) {
  __shared__ float red[32];
  pdl_launch_dependents();
  pdl_wait_prior_grids();
  const float inv = 1.0f / (float)cols;
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    const float mean = mean_in[r], rstd = rstd_in[r];
    const T* xr = x + r * ldx;
    const T* dyr = dy + r * lddy;
    float s1 = 0.0f, s2 = 0.0f;
    for (long long c = threadIdx.x; c < cols; c += LN_THREADS) {
      const float g = w != nullptr ? float(dyr[c]) * float(w[c]) : float(dyr[c]);
      s1 += g;
      s2 = fmaf(g, (float(xr[c]) - mean) * rstd, s2);
    }
    const float c1 = cta_sum(s1, red) * inv;
    const float c2 = cta_sum(s2, red) * inv;
    for (long long c = threadIdx.x; c < cols; c += LN_THREADS) {
      const float g = w != nullptr ? float(dyr[c]) * float(w[c]) : float(dyr[c]);
      const float xh = (float(xr[c]) - mean) * rstd;
      dx[r * lddx + c] = T(rstd * (g - c1 - xh * c2));
    }
  }
}

// Column sums of dy * xh and dy over one slab of rows: CTA (column tile, slab) -> part[slab][2][cols].
template <typename T>
__global__ void __launch_bounds__(LN_THREADS)
ln_backward_columns_kernel(const T* __restrict__ dy, const T* __restrict__ x, const float* __restrict__ mean_in,
                           const float* __restrict__ rstd_in, float* __restrict__ part, long long rows, long long cols,
                           long long lddy, long long ldx, int slabs) {
  __shared__ float sw[8][LN_COL_TILE], sb[8][LN_COL_TILE];
  pdl_launch_dependents();
  pdl_wait_prior_grids();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long tiles = (cols + LN_COL_TILE - 1) / LN_COL_TILE;
  for (long long t = blockIdx.x; t < tiles * slabs; t += gridDim.x) {
    const long long slab = t / tiles;
    const long long c = (t - slab * tiles) * LN_COL_TILE + lane;
    const long long r0 = rows * slab / slabs, r1 = rows * (slab + 1) / slabs;
    float dw = 0.0f, db = 0.0f;
    if (c < cols) {
      for (long long r = r0 + warp; r < r1; r += 8) {
        const float d = float(dy[r * lddy + c]);
        dw = fmaf(d, (float(x[r * ldx + c]) - mean_in[r]) * rstd_in[r], dw);
        db += d;
      }
    }
    __syncthreads();  // the previous tile's sums have been read
    sw[warp][lane] = dw;
    sb[warp][lane] = db;
    __syncthreads();
    if (warp == 0 && c < cols) {
      for (int i = 1; i < 8; ++i) {
        dw += sw[i][lane];
        db += sb[i][lane];
      }
      part[(slab * 2) * cols + c] = dw;
      part[(slab * 2 + 1) * cols + c] = db;
    }
  }
}

// dweight / dbias from the partial rows, always in the same order: eight interleaved chains, then their sum.
template <typename W>
__global__ void __launch_bounds__(LN_THREADS)
ln_backward_finish_kernel(const float* __restrict__ part, W* __restrict__ dw, W* __restrict__ db, long long cols, int parts) {
  __shared__ float s[2][8][LN_COL_TILE];
  pdl_launch_dependents();
  pdl_wait_prior_grids();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long c = (long long)blockIdx.x * LN_COL_TILE + lane;
  float a = 0.0f, d = 0.0f;
  if (c < cols) {
    for (int i = warp; i < parts; i += 8) {
      a += part[(long long)(2 * i) * cols + c];
      d += part[(long long)(2 * i + 1) * cols + c];
    }
  }
  s[0][warp][lane] = a;
  s[1][warp][lane] = d;
  __syncthreads();
  if (warp < 2 && c < cols) {
    float v = s[warp][0][lane];
    for (int i = 1; i < 8; ++i) v += s[warp][i][lane];
    W* dst = warp == 0 ? dw : db;
    if (dst != nullptr) dst[c] = W(v);
  }
}

struct LnShape {
  long long rows, cols, ldx, ldy, ldd;
};

template <typename T, typename W>
int forward(const void* x, const void* w, const void* b, void* y, float* mean, float* rstd, const LnShape& s, float eps,
            int num_sms, cudaStream_t stream) {
  const unsigned grid = (unsigned)std::min<long long>(s.rows, (long long)num_sms * 64);
  cudaError_t e = launch_kernel_ex(ln_forward_any_kernel<T, W>, grid, LN_THREADS, 0, stream, 1, pdl_enabled(),
                                   static_cast<const T*>(x), static_cast<const W*>(w), static_cast<const W*>(b),
                                   static_cast<T*>(y), mean, rstd, s.rows, s.cols, s.ldx, s.ldy, eps);
  if (e != cudaSuccess) return launch_failed(e, "layer norm launch failed");
  count_launches(1);
  return SX_OK;
}

template <typename T, typename W>
int backward(const void* dy, const void* x, const float* mean, const float* rstd, const void* w, void* dx, void* dw,
             void* db, const LnShape& s, float* part, int num_sms, cudaStream_t stream) {
  cudaError_t e;
  const bool pdl = pdl_enabled();
  if (dw != nullptr || db != nullptr) {
    // before dx: dx may overwrite dy
    const long long tiles = (s.cols + LN_COL_TILE - 1) / LN_COL_TILE;
    int slabs = 0;
    if (s.rows > 0) {
      slabs = (int)std::min<long long>(std::min<long long>(LN_PARTS, (s.rows + 7) / 8), std::max<long long>(1, num_sms * 8LL / tiles));
      e = launch_kernel_ex(ln_backward_columns_kernel<T>, (unsigned)std::min<long long>(tiles * slabs, num_sms * 8LL), LN_THREADS, 0,
                           stream, 1, pdl, static_cast<const T*>(dy), static_cast<const T*>(x), mean, rstd, part, s.rows,
                           s.cols, s.ldd, s.ldx, slabs);
      if (e != cudaSuccess) return launch_failed(e, "layer norm backward launch failed");
      count_launches(1);
    }
    e = launch_kernel_ex(ln_backward_finish_kernel<W>, (unsigned)tiles, LN_THREADS, 0, stream, 1, pdl, (const float*)part,
                         static_cast<W*>(dw), static_cast<W*>(db), s.cols, slabs);
    if (e != cudaSuccess) return launch_failed(e, "layer norm backward launch failed");
    count_launches(1);
  }
  if (dx != nullptr && s.rows > 0) {
    e = launch_kernel_ex(ln_backward_dx_any_kernel<T, W>, (unsigned)std::min<long long>(s.rows, (long long)num_sms * 64),
                         LN_THREADS, 0, stream, 1, pdl, static_cast<const T*>(dy), static_cast<const T*>(x), mean, rstd,
                         static_cast<const W*>(w), static_cast<T*>(dx), s.rows, s.cols, s.ldd, s.ldx, s.ldy);
    if (e != cudaSuccess) return launch_failed(e, "layer norm backward launch failed");
    count_launches(1);
  }
  return SX_OK;
}

int check_shape(int64_t rows, int64_t cols, int32_t dtype, int32_t param_dtype) {
  if (rows < 0 || cols <= 0) return fail_fmt(SX_ERR_INVALID, "layer norm needs rows >= 0 and cols >= 1");
  if (cols > 0x7fffffffLL) return fail_fmt(SX_ERR_INVALID, "dimension exceeds 2^31-1");
  if (dtype != SYMPLEX_DT_F32 && dtype != SYMPLEX_DT_BF16)
    return fail_fmt(SX_ERR_INVALID, "dtype %d not supported (F32=9, BF16=11)", dtype);
  if (param_dtype != dtype && param_dtype != SYMPLEX_DT_F32)
    return fail_fmt(SX_ERR_INVALID, "param_dtype must be dtype or F32");
  return SX_OK;
}

// Base pointers must be aligned to their element.
bool element_aligned(const void* p, int32_t dtype) {
  return reinterpret_cast<uintptr_t>(p) % (dtype == SYMPLEX_DT_F32 ? 4 : 2) == 0;
}

}  // namespace
}  // namespace sx

using namespace sx;

extern "C" {

int symplex_b200_layer_norm(const void* x, const void* weight, const void* bias, void* y, float* mean, float* rstd,
                            int64_t rows, int64_t cols, int64_t ldx, int64_t ldy, int32_t dtype, int32_t param_dtype,
                            double eps, void* stream) {
  int rc = check_shape(rows, cols, dtype, param_dtype);
  if (rc != SX_OK) return rc;
  LnShape s{rows, cols, ldx ? ldx : cols, ldy ? ldy : cols, 0};
  if (s.ldx < cols || s.ldy < cols) return fail_fmt(SX_ERR_INVALID, "leading dimension too small");
  if (!(eps >= 0.0)) return fail_fmt(SX_ERR_INVALID, "eps must not be negative");
  if (rows == 0) return SX_OK;
  if (x == nullptr || y == nullptr) return fail_fmt(SX_ERR_INVALID, "null pointer");
  if (!element_aligned(x, dtype) || !element_aligned(y, dtype) || !element_aligned(weight, param_dtype) ||
      !element_aligned(bias, param_dtype) || !element_aligned(mean, SYMPLEX_DT_F32) || !element_aligned(rstd, SYMPLEX_DT_F32))
    return fail_fmt(SX_ERR_INVALID, "a pointer is not aligned to its element type");
  int sms = 0;
  if ((rc = current_device_sms(&sms)) != SX_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == SYMPLEX_DT_F32) return forward<float, float>(x, weight, bias, y, mean, rstd, s, (float)eps, sms, st);
  if (param_dtype == SYMPLEX_DT_F32)
    return forward<__nv_bfloat16, float>(x, weight, bias, y, mean, rstd, s, (float)eps, sms, st);
  return forward<__nv_bfloat16, __nv_bfloat16>(x, weight, bias, y, mean, rstd, s, (float)eps, sms, st);
}

size_t symplex_b200_layer_norm_backward_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  return (size_t)std::min<int64_t>(rows, LN_PARTS) * 2 * (size_t)cols * sizeof(float);
}

int symplex_b200_layer_norm_backward(const void* dy, const void* x, const float* mean, const float* rstd,
                                     const void* weight, void* dx, void* dweight, void* dbias, int64_t rows,
                                     int64_t cols, int64_t lddy, int64_t ldx, int64_t lddx, int32_t dtype,
                                     int32_t param_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_shape(rows, cols, dtype, param_dtype);
  if (rc != SX_OK) return rc;
  LnShape s{rows, cols, ldx ? ldx : cols, lddx ? lddx : cols, lddy ? lddy : cols};
  if (s.ldx < cols || s.ldy < cols || s.ldd < cols) return fail_fmt(SX_ERR_INVALID, "leading dimension too small");
  const bool params = dweight != nullptr || dbias != nullptr;
  if (dx == nullptr && !params) return SX_OK;
  if (rows > 0 && (dy == nullptr || x == nullptr || mean == nullptr || rstd == nullptr))
    return fail_fmt(SX_ERR_INVALID, "null pointer");
  if (!element_aligned(x, dtype) || !element_aligned(dy, dtype) || !element_aligned(dx, dtype) ||
      !element_aligned(weight, param_dtype) || !element_aligned(dweight, param_dtype) || !element_aligned(dbias, param_dtype) ||
      !element_aligned(mean, SYMPLEX_DT_F32) || !element_aligned(rstd, SYMPLEX_DT_F32))
    return fail_fmt(SX_ERR_INVALID, "a pointer is not aligned to its element type");
  if (params) {
    const size_t need = symplex_b200_layer_norm_backward_workspace_bytes(rows, cols);
    if (need > workspace_bytes || (need && workspace == nullptr))
      return fail_fmt(SX_ERR_INVALID, "workspace too small: need %zu bytes, got %zu", need, workspace_bytes);
    if (reinterpret_cast<uintptr_t>(workspace) % 256) return fail_fmt(SX_ERR_INVALID, "workspace must be 256-byte aligned");
  }
  int sms = 0;
  if ((rc = current_device_sms(&sms)) != SX_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  float* part = static_cast<float*>(workspace);
  if (dtype == SYMPLEX_DT_F32)
    return backward<float, float>(dy, x, mean, rstd, weight, dx, dweight, dbias, s, part, sms, st);
  if (param_dtype == SYMPLEX_DT_F32)
    return backward<__nv_bfloat16, float>(dy, x, mean, rstd, weight, dx, dweight, dbias, s, part, sms, st);
  return backward<__nv_bfloat16, __nv_bfloat16>(dy, x, mean, rstd, weight, dx, dweight, dbias, s, part, sms, st);
}

}  // extern "C"
