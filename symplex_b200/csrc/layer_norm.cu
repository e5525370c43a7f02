// Layer norm over the last dimension, forward and backward, with the reduction of the weight's and bias' gradients.
//
//   forward    mean = sum x / C,  var = sum (x - mean)^2 / C,  y = (x - mean) rstd w + b
//   backward   xh = (x - mean) rstd,  g = dy w,  dx = rstd (g - mean(g) - xh mean(g xh)),
//              dw = sum_rows dy xh,  db = sum_rows dy
//
// Bound by HBM: the forward pass must read x and write y, the backward pass must read x and dy and write dx.
//
// A row is held in registers by a power of two of threads, at most 16 values each (16-byte vectors where the rows allow it, else
// single values): read once, its deviations squared from the registers. Persistent CTAs walk over the rows and fetch the next row
// while they reduce this one. In the backward pass a thread keeps its 16 columns' share of dw and db in registers over all rows of
// its CTA, so the sums over rows cost no traffic but one partial row per CTA, joined by a second, small kernel. Rows of more than
// 16384 values (8192 backward) take the kernels that read a row several times.
#include <cuda_bf16.h>

#include <algorithm>
#include <initializer_list>

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

// ------------------------------------------------------------------ rows in registers
template <typename T, int VEC>
struct LnRaw {
  uint4 v;
  __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void unpack(float (&f)[VEC]) const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  }
  static __device__ __forceinline__ void store(T* p, const float (&f)[VEC]) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
    } else {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
      *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
};
template <typename T>
struct LnRaw<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = *p; }
  __device__ __forceinline__ void unpack(float (&f)[1]) const { f[0] = float(v); }
  static __device__ __forceinline__ void store(T* p, const float (&f)[1]) { *p = T(f[0]); }
};

// VEC consecutive parameters (of the input's type or float).
template <typename W, int VEC>
__device__ __forceinline__ void load_params(const W* p, float (&f)[VEC]) {
  if constexpr (VEC == 1) {
    f[0] = float(*p);
  } else if constexpr (sizeof(W) == 4) {
#pragma unroll
    for (int i = 0; i < VEC; i += 4) {
      const float4 x = __ldg(reinterpret_cast<const float4*>(p + i));
      f[i] = x.x; f[i + 1] = x.y; f[i + 2] = x.z; f[i + 3] = x.w;
    }
  } else {
    LnRaw<W, VEC> r;
    r.load(p);
    r.unpack(f);
  }
}

// kN sums over the tpr threads of a row, the same values in every thread. `red`: this row group's [32][kN] floats for this call; the
// caller alternates between two of them, and the barrier in between keeps a use of one apart from the next use of the same.
template <int kN>
__device__ __forceinline__ void row_sum(float (&v)[kN], float* red, int tpr, int group) {
#pragma unroll
  for (int i = 0; i < kN; ++i) v[i] = warp_sum(v[i]);
  if (tpr == 32) return;
  const int lane = threadIdx.x & 31, warp = (threadIdx.x & (tpr - 1)) >> 5, warps = tpr >> 5;
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < kN; ++i) red[warp * kN + i] = v[i];
  }
  asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(tpr) : "memory");  // at most 8 groups of 64 threads
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    float s = lane < warps ? red[lane * kN + i] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    v[i] = s;
  }
}

template <typename T, typename W, int VEC, int NV, int BLOCK>
__global__ void __launch_bounds__(BLOCK)
ln_forward_kernel(const T* x, const W* __restrict__ w, const W* __restrict__ b, T* y, float* __restrict__ mean_out,
                  float* __restrict__ rstd_out, long long rows, int cols, long long ldx, long long ldy, float eps, int tpr) {
  __shared__ float red[BLOCK / 32 * 2 * 2 + 64];
  const int group = threadIdx.x / tpr, t = threadIdx.x & (tpr - 1);
  const long long groups = (long long)gridDim.x * (BLOCK / tpr);
  float* const my_red = red + group * (tpr >> 5) * 2;
  const int nvec = cols / VEC;
  const float inv = 1.0f / (float)cols;
  pdl_launch_dependents();
  pdl_wait_prior_grids();
  LnRaw<T, VEC> next[NV];
  auto fetch = [&](long long r) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (t + i * tpr < nvec) next[i].load(x + r * ldx + (long long)(t + i * tpr) * VEC);
  };
  long long r = (long long)blockIdx.x * (BLOCK / tpr) + group;
  if (r < rows) fetch(r);
  for (; r < rows; r += groups) {
    float f[NV][VEC];
    float s[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (t + i * tpr < nvec) {
        next[i].unpack(f[i]);
#pragma unroll
        for (int j = 0; j < VEC; ++j) s[0] += f[i][j];
      }
    }
    if (r + groups < rows) fetch(r + groups);
    row_sum(s, my_red, tpr, group);
    const float mean = s[0] * inv;
    float q[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (t + i * tpr < nvec) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          f[i][j] -= mean;
          q[0] = fmaf(f[i][j], f[i][j], q[0]);
        }
      }
    }
    row_sum(q, my_red + (tpr >> 5), tpr, group);
    const float rstd = 1.0f / sqrtf(q[0] * inv + eps);
    if (t == 0) {
      if (mean_out != nullptr) mean_out[r] = mean;
      if (rstd_out != nullptr) rstd_out[r] = rstd;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = t + i * tpr;
      if (v < nvec) {
        float p[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) f[i][j] *= rstd;
        if (w != nullptr) {
          load_params<W, VEC>(w + v * VEC, p);
#pragma unroll
          for (int j = 0; j < VEC; ++j) f[i][j] *= p[j];
        }
        if (b != nullptr) {
          load_params<W, VEC>(b + v * VEC, p);
#pragma unroll
          for (int j = 0; j < VEC; ++j) f[i][j] += p[j];
        }
        LnRaw<T, VEC>::store(y + r * ldy + (long long)v * VEC, f[i]);
      }
    }
  }
}

// dx, and this CTA's share of dw and db as row blockIdx.x of part[grid][2][cols] (part null: dx only; dx null: those only).
template <typename T, typename W, int VEC, int NV, int BLOCK, bool kAhead>
__global__ void __launch_bounds__(BLOCK)
ln_backward_kernel(const T* dy, const T* __restrict__ x, const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
                   const W* __restrict__ w, T* dx, float* __restrict__ part, long long rows, int cols, long long lddy, long long ldx,
                   long long lddx, int tpr) {
  extern __shared__ float joined[];  // [2][cols], where several row groups are joined
  __shared__ float red[2][BLOCK / 32 * 2];
  const int group = threadIdx.x / tpr, t = threadIdx.x & (tpr - 1), per_cta = BLOCK / tpr;
  const long long groups = (long long)gridDim.x * per_cta;
  const int nvec = cols / VEC;
  const float inv = 1.0f / (float)cols;
  pdl_launch_dependents();
  pdl_wait_prior_grids();
  LnRaw<T, VEC> nx[NV], nd[NV];
  float nmean = 0.0f, nrstd = 0.0f;
  auto fetch = [&](long long r) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (t + i * tpr < nvec) {
        nx[i].load(x + r * ldx + (long long)(t + i * tpr) * VEC);
        nd[i].load(dy + r * lddy + (long long)(t + i * tpr) * VEC);
      }
    }
    nmean = mean_in[r];
    nrstd = rstd_in[r];
  };
  float dw[NV][VEC] = {}, db[NV][VEC] = {};
  long long r = (long long)blockIdx.x * per_cta + group;
  if (kAhead && r < rows) fetch(r);
  int buf = 0;
  for (; r < rows; r += groups, buf ^= 1) {
    if (!kAhead) fetch(r);
    const float mean = nmean, rstd = nrstd;
    float xh[NV][VEC], g[NV][VEC];
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = t + i * tpr;
      if (v < nvec) {
        nx[i].unpack(xh[i]);
        nd[i].unpack(g[i]);
        float p[VEC];
        if (w != nullptr) load_params<W, VEC>(w + v * VEC, p);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          xh[i][j] = (xh[i][j] - mean) * rstd;
          dw[i][j] = fmaf(g[i][j], xh[i][j], dw[i][j]);
          db[i][j] += g[i][j];
          if (w != nullptr) g[i][j] *= p[j];
          s[0] += g[i][j];
          s[1] = fmaf(g[i][j], xh[i][j], s[1]);
        }
      }
    }
    if (kAhead && r + groups < rows) fetch(r + groups);
    if (dx == nullptr) continue;
    row_sum(s, red[buf] + group * (tpr >> 5) * 2, tpr, group);
    const float c1 = s[0] * inv, c2 = s[1] * inv;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = t + i * tpr;
      if (v < nvec) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) g[i][j] = rstd * (g[i][j] - c1 - xh[i][j] * c2);
        LnRaw<T, VEC>::store(dx + r * lddx + (long long)v * VEC, g[i]);
      }
    }
  }
  if (part == nullptr) return;
  float* const out = part + (long long)blockIdx.x * 2 * cols;
  for (int turn = 0; turn < per_cta; ++turn) {  // group after group, always in the same order
    if (per_cta > 1) __syncthreads();
    if (group == turn) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = t + i * tpr;
        if (v < nvec) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const int c = v * VEC + j;
            float a = dw[i][j], d = db[i][j];
            if (turn > 0) {
              a += joined[c];
              d += joined[cols + c];
            }
            if (turn == per_cta - 1) {
              out[c] = a;
              out[cols + c] = d;
            } else {
              joined[c] = a;
              joined[cols + c] = d;
            }
          }
        }
      }
    }
  }
}

// Threads of a row: the smallest power of two (a warp at least) that holds it with `most` values a thread; where there are fewer rows
// than SMs, enough that a thread has one vector.
int threads_per_row(long long vectors, int most_vectors, int limit, bool few) {
  int t = 32;
  while (t < limit && (long long)t * (few ? 1 : most_vectors) < vectors) t *= 2;
  return t;
}

struct LnShape {
  long long rows, cols, ldx, ldy, ldd;
};

bool all_aligned(std::initializer_list<const void*> ps, std::initializer_list<long long> strides_bytes) {
  uintptr_t a = 0;
  for (const void* p : ps) a |= reinterpret_cast<uintptr_t>(p);
  for (long long s : strides_bytes) a |= (uintptr_t)s;
  return a % 16 == 0;
}

template <typename T, typename W, int VEC, int NV>
cudaError_t forward_rows(const void* x, const void* w, const void* b, void* y, float* mean, float* rstd, const LnShape& s, float eps, int tpr,
                         int num_sms, cudaStream_t stream) {
  auto go = [&](auto kern, int block, int ctas_per_sm) {
    const long long per_cta = block / tpr;
    const unsigned grid = (unsigned)std::min<long long>((s.rows + per_cta - 1) / per_cta, (long long)num_sms * ctas_per_sm);
    return launch_kernel_ex(kern, grid, block, 0, stream, 1, pdl_enabled(), static_cast<const T*>(x), static_cast<const W*>(w),
                            static_cast<const W*>(b), static_cast<T*>(y), mean, rstd, s.rows, (int)s.cols, s.ldx, s.ldy, eps, tpr);
  };
  return tpr <= 256 ? go(ln_forward_kernel<T, W, VEC, NV, 256>, 256, 4) : go(ln_forward_kernel<T, W, VEC, NV, 1024>, 1024, 1);
}

template <typename T, typename W>
int forward(const void* x, const void* w, const void* b, void* y, float* mean, float* rstd, const LnShape& s, float eps,
            int num_sms, cudaStream_t stream) {
  constexpr int VEC = 16 / sizeof(T), MOST = 16 / VEC;
  const long long eb = sizeof(T);
  const bool vec = s.cols % VEC == 0 && all_aligned({x, y, w, b}, {s.ldx * eb, s.ldy * eb});
  const bool few = s.rows <= num_sms;
  cudaError_t e;
  if (vec && s.cols <= 1024 * 16) {
    const int tpr = threads_per_row(s.cols / VEC, MOST, 1024, few);
    const long long nv = (s.cols / VEC + tpr - 1) / tpr;
    if (nv <= 1) e = forward_rows<T, W, VEC, 1>(x, w, b, y, mean, rstd, s, eps, tpr, num_sms, stream);
    else if (nv <= 2) e = forward_rows<T, W, VEC, 2>(x, w, b, y, mean, rstd, s, eps, tpr, num_sms, stream);
    else e = forward_rows<T, W, VEC, MOST>(x, w, b, y, mean, rstd, s, eps, tpr, num_sms, stream);
  } else if (!vec && s.cols <= 1024 * 16) {
    const int tpr = threads_per_row(s.cols, 8, 1024, few);
    const long long nv = (s.cols + tpr - 1) / tpr;
    if (nv <= 1) e = forward_rows<T, W, 1, 1>(x, w, b, y, mean, rstd, s, eps, tpr, num_sms, stream);
    else if (nv <= 8) e = forward_rows<T, W, 1, 8>(x, w, b, y, mean, rstd, s, eps, tpr, num_sms, stream);
    else e = forward_rows<T, W, 1, 16>(x, w, b, y, mean, rstd, s, eps, tpr, num_sms, stream);
  } else {
    const unsigned grid = (unsigned)std::min<long long>(s.rows, (long long)num_sms * 64);
    e = launch_kernel_ex(ln_forward_any_kernel<T, W>, grid, LN_THREADS, 0, stream, 1, pdl_enabled(), static_cast<const T*>(x),
                         static_cast<const W*>(w), static_cast<const W*>(b), static_cast<T*>(y), mean, rstd, s.rows, s.cols, s.ldx, s.ldy,
                         eps);
  }
  if (e != cudaSuccess) return launch_failed(e, "layer norm launch failed");
  count_launches(1);
  return SX_OK;
}

template <typename T, typename W, int VEC, int NV>
int backward_rows(const void* dy, const void* x, const float* mean, const float* rstd, const void* w, void* dx, float* part, const LnShape& s,
                  int tpr, int num_sms, cudaStream_t stream, int* parts) {
  constexpr int BLOCK = 512;
  auto kern = ln_backward_kernel<T, W, VEC, NV, BLOCK, true>;
  const long long per_cta = BLOCK / tpr;
  const size_t smem = per_cta > 1 && part != nullptr ? (size_t)s.cols * 8 : 0;
  SX_ENSURE_DYN_SMEM(kern, 64 * 1024);
  *parts = (int)std::min<long long>((s.rows + per_cta - 1) / per_cta, std::min(num_sms, LN_PARTS));
  const cudaError_t e = launch_kernel_ex(kern, (unsigned)*parts, BLOCK, smem, stream, 1, pdl_enabled(), static_cast<const T*>(dy),
                                         static_cast<const T*>(x), mean, rstd, static_cast<const W*>(w), static_cast<T*>(dx), part, s.rows,
                                         (int)s.cols, s.ldd, s.ldx, s.ldy, tpr);
  if (e != cudaSuccess) return launch_failed(e, "layer norm backward launch failed");
  count_launches(1);
  return SX_OK;
}

template <typename T, typename W>
int backward(const void* dy, const void* x, const float* mean, const float* rstd, const void* w, void* dx, void* dw,
             void* db, const LnShape& s, float* part, int num_sms, cudaStream_t stream) {
  const bool pdl = pdl_enabled();
  const bool params = dw != nullptr || db != nullptr;
  const long long tiles = (s.cols + LN_COL_TILE - 1) / LN_COL_TILE;
  int parts = 0;
  cudaError_t e;
  if (s.rows > 0 && s.cols <= 512 * 16) {
    constexpr int VEC = 16 / sizeof(T), MOST = 16 / VEC;
    const long long eb = sizeof(T);
    const bool few = s.rows <= num_sms;
    float* to = params ? part : nullptr;
    int rc;
    if (s.cols % VEC == 0 && all_aligned({x, dy, dx, w}, {s.ldx * eb, s.ldd * eb, s.ldy * eb})) {
      const int tpr = threads_per_row(s.cols / VEC, MOST, 512, few);
      const long long nv = (s.cols / VEC + tpr - 1) / tpr;
      rc = nv <= 1   ? backward_rows<T, W, VEC, 1>(dy, x, mean, rstd, w, dx, to, s, tpr, num_sms, stream, &parts)
           : nv <= 2 ? backward_rows<T, W, VEC, 2>(dy, x, mean, rstd, w, dx, to, s, tpr, num_sms, stream, &parts)
                     : backward_rows<T, W, VEC, MOST>(dy, x, mean, rstd, w, dx, to, s, tpr, num_sms, stream, &parts);
    } else {
      const int tpr = threads_per_row(s.cols, 4, 512, few);
      const long long nv = (s.cols + tpr - 1) / tpr;
      rc = nv <= 1   ? backward_rows<T, W, 1, 1>(dy, x, mean, rstd, w, dx, to, s, tpr, num_sms, stream, &parts)
           : nv <= 4 ? backward_rows<T, W, 1, 4>(dy, x, mean, rstd, w, dx, to, s, tpr, num_sms, stream, &parts)
                     : backward_rows<T, W, 1, 16>(dy, x, mean, rstd, w, dx, to, s, tpr, num_sms, stream, &parts);
    }
    if (rc != SX_OK || !params) return rc;
  } else if (s.rows > 0) {
    if (params) {  // before dx: dx may overwrite dy
      parts = (int)std::min<long long>(std::min<long long>(LN_PARTS, (s.rows + 7) / 8), std::max<long long>(1, num_sms * 8LL / tiles));
      e = launch_kernel_ex(ln_backward_columns_kernel<T>, (unsigned)std::min<long long>(tiles * parts, num_sms * 8LL), LN_THREADS, 0, stream,
                           1, pdl, static_cast<const T*>(dy), static_cast<const T*>(x), mean, rstd, part, s.rows, s.cols, s.ldd, s.ldx, parts);
      if (e != cudaSuccess) return launch_failed(e, "layer norm backward launch failed");
      count_launches(1);
    }
    if (dx != nullptr) {
      e = launch_kernel_ex(ln_backward_dx_any_kernel<T, W>, (unsigned)std::min<long long>(s.rows, (long long)num_sms * 64), LN_THREADS, 0,
                           stream, 1, pdl, static_cast<const T*>(dy), static_cast<const T*>(x), mean, rstd, static_cast<const W*>(w),
                           static_cast<T*>(dx), s.rows, s.cols, s.ldd, s.ldx, s.ldy);
      if (e != cudaSuccess) return launch_failed(e, "layer norm backward launch failed");
      count_launches(1);
    }
  }
  if (params) {
    e = launch_kernel_ex(ln_backward_finish_kernel<W>, (unsigned)tiles, LN_THREADS, 0, stream, 1, pdl, (const float*)part,
                         static_cast<W*>(dw), static_cast<W*>(db), s.cols, parts);
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
