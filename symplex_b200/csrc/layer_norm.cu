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
#include <atomic>
#include <initializer_list>
#include <type_traits>

#include "../../include/symplex_b200.h"
#include "byte_rows.h"
#include "gemm_params.h"
#include "host_api.h"
#include "sm100_ptx.cuh"

namespace sx {
namespace {

constexpr int LN_THREADS = 256;
// Rows of single values (no 16-byte vectors) that are held in registers: longer ones are faster in the kernels that read a row
// several times and put more rows on an SM (bf16, device: forward of 2048 x 7777 57 us in registers, 38 so;
// backward 128 and 80; forward of 16384 x 1001 47 us in registers, 56 so).
constexpr long long LN_SINGLE_FORWARD = 2048, LN_SINGLE_BACKWARD = 2048;
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
#pragma unroll 8
    for (int c = threadIdx.x; c < (int)cols; c += LN_THREADS) s += float(xr[c]);
    const float mean = cta_sum(s, red) * inv;
    float q = 0.0f;
#pragma unroll 8
    for (int c = threadIdx.x; c < (int)cols; c += LN_THREADS) {
      const float d = float(xr[c]) - mean;
      q = fmaf(d, d, q);
    }
    const float rstd = 1.0f / sqrtf(cta_sum(q, red) * inv + eps);
    if (threadIdx.x == 0) {
      if (mean_out != nullptr) mean_out[r] = mean;
      if (rstd_out != nullptr) rstd_out[r] = rstd;
    }
#pragma unroll 4
    for (int c = threadIdx.x; c < (int)cols; c += LN_THREADS) {
      float v = (float(xr[c]) - mean) * rstd;
      if (w != nullptr) v *= float(w[c]);
      if (b != nullptr) v += float(b[c]);
      yr[c] = T(v);
    }
  }
}

// dweight / dbias from the partial rows, always in the same order: 32 interleaved chains (a warp each, eight loads in flight a lane),
// then their sum. Few columns a CTA and many warps, because what it costs is the latency of the chains.
template <typename W>
__global__ void __launch_bounds__(1024)
ln_backward_finish_kernel(const float* __restrict__ part, W* __restrict__ dw, W* __restrict__ db, long long cols, int parts) {
  __shared__ float s[2][32][LN_COL_TILE + 1];
  pdl_launch_dependents();
  pdl_wait_prior_grids();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long c = (long long)blockIdx.x * LN_COL_TILE + lane;
  float a = 0.0f, d = 0.0f;
  if (c < cols) {
    for (int i = warp; i < parts; i += 4 * 32) {
      float x[4], y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool in = i + 32 * j < parts;
        const float* p = part + (long long)(2 * (in ? i + 32 * j : i)) * cols + c;
        x[j] = in ? p[0] : 0.0f;
        y[j] = in ? p[cols] : 0.0f;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        a += x[j];
        d += y[j];
      }
    }
  }
  s[0][warp][lane] = a;
  s[1][warp][lane] = d;
  __syncthreads();
  // warp w adds up column w: 32 chains across its lanes
  const long long col = (long long)blockIdx.x * LN_COL_TILE + warp;
  a = warp_sum(s[0][lane][warp]);
  d = warp_sum(s[1][lane][warp]);
  if (lane == 0 && col < cols) {
    if (dw != nullptr) dw[col] = W(a);
    if (db != nullptr) db[col] = W(d);
  }
}

// ------------------------------------------------------------------ rows in registers
// VEC values of a thread, in pairs: one instruction of the packed fp32 unit for two of them.
template <int VEC>
struct Fv {
  unsigned long long p[VEC / 2];
  static __device__ __forceinline__ unsigned long long pair(float a, float b) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
  }
  static __device__ __forceinline__ float2 split(unsigned long long v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
  }
  __device__ __forceinline__ void fill(float s) {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) p[i] = pair(s, s);
  }
  __device__ __forceinline__ void add(const Fv& o) {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) asm("add.rn.f32x2 %0, %0, %1;" : "+l"(p[i]) : "l"(o.p[i]));
  }
  __device__ __forceinline__ void mul(const Fv& o) {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(p[i]) : "l"(o.p[i]));
  }
  // this = a * b, without a copy of a
  __device__ __forceinline__ void product(const Fv& a, const Fv& b) {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(p[i]) : "l"(a.p[i]), "l"(b.p[i]));
  }
  // this += a * b
  __device__ __forceinline__ void fma(const Fv& a, const Fv& b) {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(p[i]) : "l"(a.p[i]), "l"(b.p[i]));
  }
  // sums over all values are kept in one pair
  using Sum = unsigned long long;
  static __device__ __forceinline__ Sum zero() { return 0ull; }
  static __device__ __forceinline__ float total(Sum s) {
    const float2 v = split(s);
    return v.x + v.y;
  }
  __device__ __forceinline__ void sum_into(Sum& s) const {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) asm("add.rn.f32x2 %0, %0, %1;" : "+l"(s) : "l"(p[i]));
  }
  __device__ __forceinline__ void dot_into(Sum& s, const Fv& o) const {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(s) : "l"(p[i]), "l"(o.p[i]));
  }
  __device__ __forceinline__ float get(int j) const {
    const float2 v = split(p[j / 2]);
    return j & 1 ? v.y : v.x;
  }
};
template <>
struct Fv<1> {
  float p;
  __device__ __forceinline__ void fill(float s) { p = s; }
  __device__ __forceinline__ void add(const Fv& o) { p += o.p; }
  __device__ __forceinline__ void mul(const Fv& o) { p *= o.p; }
  __device__ __forceinline__ void product(const Fv& a, const Fv& b) { p = a.p * b.p; }
  __device__ __forceinline__ void fma(const Fv& a, const Fv& b) { p = fmaf(a.p, b.p, p); }
  using Sum = float;
  static __device__ __forceinline__ Sum zero() { return 0.0f; }
  static __device__ __forceinline__ float total(Sum s) { return s; }
  __device__ __forceinline__ void sum_into(Sum& s) const { s += p; }
  __device__ __forceinline__ void dot_into(Sum& s, const Fv& o) const { s = fmaf(p, o.p, s); }
  __device__ __forceinline__ float get(int) const { return p; }
};

template <typename T, int VEC>
struct LnRaw {
  uint4 v;
  __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void unpack(Fv<VEC>& f) const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 2; ++i) f.p[i] = Fv<VEC>::pair(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) f.p[i] = Fv<VEC>::pair(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    }
  }
  static __device__ __forceinline__ void store(T* p, const Fv<VEC>& f) {
    uint32_t w[4];
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float2 v = Fv<VEC>::split(f.p[i]);
        w[2 * i] = __float_as_uint(v.x);
        w[2 * i + 1] = __float_as_uint(v.y);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 h = __float22bfloat162_rn(Fv<VEC>::split(f.p[i]));
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <typename T>
struct LnRaw<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = *p; }
  __device__ __forceinline__ void unpack(Fv<1>& f) const { f.p = float(v); }
  static __device__ __forceinline__ void store(T* p, const Fv<1>& f) { *p = T(f.p); }
};

// VEC consecutive parameters (of the input's type or float).
template <typename W, int VEC>
__device__ __forceinline__ void load_params(const W* p, Fv<VEC>& f) {
  if constexpr (VEC == 1) {
    f.p = float(*p);
  } else if constexpr (sizeof(W) == 4) {
#pragma unroll
    for (int i = 0; i < VEC; i += 4) {
      const float4 x = __ldg(reinterpret_cast<const float4*>(p + i));
      f.p[i / 2] = Fv<VEC>::pair(x.x, x.y);
      f.p[i / 2 + 1] = Fv<VEC>::pair(x.z, x.w);
    }
  } else {
    LnRaw<W, VEC> r;
    r.load(p);
    r.unpack(f);
  }
}

// Parameters staged in shared memory as floats, the 4-float pieces of a vector nvec * 16 bytes apart (so that neighbouring lanes read
// neighbouring 16 bytes). Persistent CTAs unpack them once instead of once a row.
template <typename W, int VEC>
__device__ __forceinline__ void stage_params(const W* p, float* to, int nvec) {
  if constexpr (VEC > 1) {
    for (int v = threadIdx.x; v < nvec; v += blockDim.x) {
      Fv<VEC> f;
      load_params<W, VEC>(p + (long long)v * VEC, f);
#pragma unroll
      for (int h = 0; h < VEC / 4; ++h) {
        const float2 a = Fv<VEC>::split(f.p[2 * h]), b = Fv<VEC>::split(f.p[2 * h + 1]);
        reinterpret_cast<float4*>(to)[h * nvec + v] = make_float4(a.x, a.y, b.x, b.y);
      }
    }
  }
}
template <int VEC>
__device__ __forceinline__ void staged_params(const float* from, int nvec, int v, Fv<VEC>& f) {
  if constexpr (VEC > 1) {
#pragma unroll
    for (int h = 0; h < VEC / 4; ++h) {
      const float4 x = reinterpret_cast<const float4*>(from)[h * nvec + v];
      f.p[2 * h] = Fv<VEC>::pair(x.x, x.y);
      f.p[2 * h + 1] = Fv<VEC>::pair(x.z, x.w);
    }
  }
}

// v^-1/2: the hardware's estimate and one step of Newton's method, which leaves two roundings' error; 1 / sqrt as the formula has it
// where the step would meet an infinity (v = 0) or a NaN.
__device__ __forceinline__ float inverse_root(float v) {
  const float y = rsqrtf(v);
  const float z = fmaf(fmaf(-v * y, y, 1.0f), 0.5f * y, y);
  return y < 3.402823466e38f && v < 1e30f ? z : y;
}

// ---- backward for rows that do not fit into registers: dx with one CTA a row, which reads it twice (the second time from L2), and the
// column sums by a kernel of their own, which reads x and dy again.
template <typename T, typename W, int VEC>
__global__ void __launch_bounds__(512)
ln_backward_dx_any_kernel(const T* dy, const T* __restrict__ x, const float* __restrict__ mean_in,
                          const float* __restrict__ rstd_in, const W* __restrict__ w, T* dx, long long rows, long long cols,
                          long long lddy, long long ldx, long long lddx) {
  __shared__ float red[32];
  pdl_launch_dependents();
  pdl_wait_prior_grids();
  const float inv = 1.0f / (float)cols;
  const long long nvec = cols / VEC;
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    Fv<VEC> km, kr;
    km.fill(-mean_in[r]);
    kr.fill(rstd_in[r]);
    const T* xr = x + r * ldx;
    const T* dyr = dy + r * lddy;
    auto values = [&](long long v, Fv<VEC>& xm, Fv<VEC>& g) {
      LnRaw<T, VEC> a, d;
      a.load(xr + v * VEC);
      d.load(dyr + v * VEC);
      a.unpack(xm);
      d.unpack(g);
      xm.add(km);
      if (w != nullptr) {
        Fv<VEC> p;
        load_params<W, VEC>(w + v * VEC, p);
        g.mul(p);
      }
    };
    typename Fv<VEC>::Sum s0 = Fv<VEC>::zero(), s1 = Fv<VEC>::zero();
#pragma unroll 4
    for (long long v = threadIdx.x; v < nvec; v += 512) {
      Fv<VEC> xm, g;
      values(v, xm, g);
      g.sum_into(s0);
      g.dot_into(s1, xm);
    }
    const float rstd = rstd_in[r];
    Fv<VEC> k1, k2;
    k1.fill(-cta_sum(Fv<VEC>::total(s0), red) * inv);
    k2.fill(-(cta_sum(Fv<VEC>::total(s1), red) * rstd) * inv * rstd);
#pragma unroll 4
    for (long long v = threadIdx.x; v < nvec; v += 512) {
      Fv<VEC> xm, g;
      values(v, xm, g);
      g.add(k1);
      g.fma(xm, k2);
      g.mul(kr);
      LnRaw<T, VEC>::store(dx + r * lddx + v * VEC, g);
    }
  }
}

// Column sums of dy * xh and dy over one slab of rows: CTA (32 vectors of columns, slab) -> part[slab][2][cols].
template <typename T, int VEC>
__global__ void __launch_bounds__(LN_THREADS)
ln_backward_columns_kernel(const T* __restrict__ dy, const T* __restrict__ x, const float* __restrict__ mean_in,
                           const float* __restrict__ rstd_in, float* __restrict__ part, long long rows, long long cols,
                           long long lddy, long long ldx, int slabs) {
  __shared__ float sw[8][32 * VEC + 1], sb[8][32 * VEC + 1];
  pdl_launch_dependents();
  pdl_wait_prior_grids();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long nvec = cols / VEC, tiles = (nvec + 31) / 32;
  for (long long t = blockIdx.x; t < tiles * slabs; t += gridDim.x) {
    const long long slab = t / tiles;
    const long long v = (t - slab * tiles) * 32 + lane;
    const long long r0 = rows * slab / slabs, r1 = rows * (slab + 1) / slabs;
    Fv<VEC> dw, db;
    dw.fill(0.0f);
    db.fill(0.0f);
    if (v < nvec) {
#pragma unroll 4
      for (long long r = r0 + warp; r < r1; r += 8) {
        LnRaw<T, VEC> a, d;
        a.load(x + r * ldx + v * VEC);
        d.load(dy + r * lddy + v * VEC);
        Fv<VEC> xm, g, k;
        a.unpack(xm);
        d.unpack(g);
        db.add(g);
        k.fill(-mean_in[r]);
        xm.add(k);
        k.fill(rstd_in[r]);
        g.mul(k);
        dw.fma(g, xm);
      }
    }
    __syncthreads();  // the previous tile's sums have been read
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      sw[warp][j * 32 + lane] = dw.get(j);
      sb[warp][j * 32 + lane] = db.get(j);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < 32 * VEC; e += LN_THREADS) {
      const long long c = ((t - slab * tiles) * 32 + (e & 31)) * VEC + (e >> 5);
      if (c >= cols) continue;
      float a = 0.0f, d = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        a += sw[i][e];
        d += sb[i][e];
      }
      part[(slab * 2) * cols + c] = a;
      part[(slab * 2 + 1) * cols + c] = d;
    }
  }
}

// kN sums over the tpr threads of a row, the same values in every thread (kTpr: tpr where it is known, else 0). `red`: this row group's
// kN * warps floats for this call; the caller alternates between two such places, and the barrier in between keeps a use of one
// apart from the next use of the same.
template <int kN, int kTpr>
__device__ __forceinline__ void row_sum(float (&v)[kN], float* red, int tpr, int group) {
#pragma unroll
  for (int i = 0; i < kN; ++i) v[i] = warp_sum(v[i]);
  if ((kTpr ? kTpr : tpr) == 32) return;
  const int lane = threadIdx.x & 31, warp = (threadIdx.x & ((kTpr ? kTpr : tpr) - 1)) >> 5, warps = (kTpr ? kTpr : tpr) >> 5;
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < kN; ++i) red[i * warps + warp] = v[i];
  }
  asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(kTpr ? kTpr : tpr) : "memory");  // at most 8 groups
  if constexpr (kTpr == 128 || kTpr == 256) {  // four or eight values: read by everyone, shorter than another round of shuffles
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const float4 a = *reinterpret_cast<const float4*>(red + i * warps);
      v[i] = (a.x + a.y) + (a.z + a.w);
      if constexpr (kTpr == 256) {
        const float4 b = *reinterpret_cast<const float4*>(red + i * warps + 4);
        v[i] += (b.x + b.y) + (b.z + b.w);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < kN; ++i) v[i] = warp_sum(lane < warps ? red[i * warps + lane] : 0.0f);
  }
}

template <typename T, typename W, int VEC, int NV, int BLOCK, bool kStage, int kTpr>
__global__ void __launch_bounds__(BLOCK)
ln_forward_kernel(const T* x, const W* __restrict__ w, const W* __restrict__ b, T* y, float* __restrict__ mean_out,
                  float* __restrict__ rstd_out, long long rows, int cols, long long ldx, long long ldy, float eps, int tpr_) {
  const int tpr = kTpr ? kTpr : tpr_;
  extern __shared__ float4 staged[];  // kStage: the weights, the biases
  __shared__ __align__(16) float red[BLOCK / 32 * 2];
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
  const float* const ws = reinterpret_cast<const float*>(staged);
  const float* const bs = ws + (w != nullptr ? cols : 0);
  if constexpr (kStage) {
    if (w != nullptr) stage_params<W, VEC>(w, reinterpret_cast<float*>(staged), nvec);
    if (b != nullptr) stage_params<W, VEC>(b, reinterpret_cast<float*>(staged) + (w != nullptr ? cols : 0), nvec);
    __syncthreads();
  }
  for (; r < rows; r += groups) {
    Fv<VEC> f[NV], k;
    typename Fv<VEC>::Sum sum = Fv<VEC>::zero();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (t + i * tpr < nvec) {
        next[i].unpack(f[i]);
        f[i].sum_into(sum);
      }
    }
    if (r + groups < rows) fetch(r + groups);
    float s[1] = {Fv<VEC>::total(sum)};
    row_sum<1, kTpr>(s, my_red, tpr, group);
    const float mean = s[0] * inv;
    k.fill(-mean);
    sum = Fv<VEC>::zero();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (t + i * tpr < nvec) {
        f[i].add(k);
        f[i].dot_into(sum, f[i]);
      }
    }
    float q[1] = {Fv<VEC>::total(sum)};
    row_sum<1, kTpr>(q, my_red + (tpr >> 5), tpr, group);
    const float rstd = inverse_root(q[0] * inv + eps);
    if (t == 0) {
      if (mean_out != nullptr) mean_out[r] = mean;
      if (rstd_out != nullptr) rstd_out[r] = rstd;
    }
    k.fill(rstd);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = t + i * tpr;
      if (v < nvec) {
        Fv<VEC> p;
        f[i].mul(k);
        if (w != nullptr) {
          if constexpr (kStage) staged_params<VEC>(ws, nvec, v, p);
          else load_params<W, VEC>(w + v * VEC, p);
          f[i].mul(p);
        }
        if (b != nullptr) {
          if constexpr (kStage) staged_params<VEC>(bs, nvec, v, p);
          else load_params<W, VEC>(b + v * VEC, p);
          f[i].add(p);
        }
        LnRaw<T, VEC>::store(y + r * ldy + (long long)v * VEC, f[i]);
      }
    }
  }
}

// dx, and this CTA's share of dw and db as row blockIdx.x of part[grid][2][cols] (part null: dx only; dx null: those only).
template <typename T, typename W, int VEC, int NV, int BLOCK, int kTpr>
__global__ void __launch_bounds__(BLOCK, 1)
ln_backward_kernel(const T* dy, const T* __restrict__ x, const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
                   const W* __restrict__ w, T* dx, float* __restrict__ part, long long rows, int cols, long long lddy, long long ldx,
                   long long lddx, int tpr_) {
  const int tpr = kTpr ? kTpr : tpr_;
  extern __shared__ float joined[];  // [group][2][cols]: 512 threads with at most 16 columns each or 1024 with 8, 64 KB
  __shared__ __align__(16) float red[2][BLOCK / 32 * 2];
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
  Fv<VEC> dw[NV], db[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    dw[i].fill(0.0f);
    db[i].fill(0.0f);
  }
  long long r = (long long)blockIdx.x * per_cta + group;
  if (r < rows) fetch(r);
  int buf = 0;
  for (; r < rows; r += groups, buf ^= 1) {
    const float mean = nmean, rstd = nrstd;
    Fv<VEC> xm[NV], g[NV], km, kr;  // x - mean; rstd is multiplied where it is needed: dw, the sum of g xh, and dx
    km.fill(-mean);
    kr.fill(rstd);
    typename Fv<VEC>::Sum s0 = Fv<VEC>::zero(), s1 = Fv<VEC>::zero();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = t + i * tpr;
      if (v < nvec) {
        nx[i].unpack(xm[i]);
        nd[i].unpack(g[i]);
        xm[i].add(km);
        db[i].add(g[i]);
        Fv<VEC> p;
        p.product(g[i], kr);
        dw[i].fma(p, xm[i]);
        if (w != nullptr) {
          load_params<W, VEC>(w + v * VEC, p);
          g[i].mul(p);
        }
        g[i].sum_into(s0);
        g[i].dot_into(s1, xm[i]);
      }
    }
    if (r + groups < rows) fetch(r + groups);
    if (dx == nullptr) continue;
    float s[2] = {Fv<VEC>::total(s0), Fv<VEC>::total(s1)};
    row_sum<2, kTpr>(s, red[buf] + group * (tpr >> 5) * 2, tpr, group);
    Fv<VEC> k1, k2;
    k1.fill(-s[0] * inv);
    k2.fill(-(s[1] * rstd) * inv * rstd);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = t + i * tpr;
      if (v < nvec) {
        g[i].add(k1);
        g[i].fma(xm[i], k2);
        g[i].mul(kr);
        LnRaw<T, VEC>::store(dx + r * lddx + (long long)v * VEC, g[i]);
      }
    }
  }
  if (part == nullptr) return;
  float* const out = part + (long long)blockIdx.x * 2 * cols;
  // The groups' shares side by side in shared memory, then their sum, group after group.
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = t + i * tpr;
    if (v < nvec) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        joined[(2 * group) * cols + v * VEC + j] = dw[i].get(j);
        joined[(2 * group + 1) * cols + v * VEC + j] = db[i].get(j);
      }
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * cols; c += blockDim.x) {
    float a = joined[c];
    for (int k = 1; k < per_cta; ++k) a += joined[2 * k * cols + c];
    out[c] = a;
  }
}

// The same for 16-byte aligned rows of some length, through shared memory: every row group has a ring of LN_RING rows (x and dy), filled
// by one of its threads with bulk copies two rows ahead, and the weights stand there as floats. In registers the next row can only be
// fetched once this one has been unpacked, which is too late for HBM. Waits are bounded: a group whose wait ran out goes on without
// waiting (in bounds), and the status word says so.
constexpr int LN_RING = 3;
constexpr int LN_RING_BYTES = 220 * 1024;
constexpr long long LN_RING_COLS = 1024;  // shorter rows: registers

template <typename T, typename W, int VEC, int NV, int kTpr>
__global__ void __launch_bounds__(512, 1)
ln_backward_ring_kernel(const T* dy, const T* __restrict__ x, const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
                        const W* __restrict__ w, T* dx, float* __restrict__ part, long long rows, int cols, long long lddy, long long ldx,
                        long long lddx, int* status, unsigned long long wait_ns) {
  extern __shared__ float4 ring_smem[];  // weights [cols]; [group][LN_RING][x row, dy row], at the end [group][2][cols] floats
  __shared__ __align__(16) float red[2][512 / 32 * 2];
  __shared__ uint64_t full[512 / kTpr * LN_RING];
  __shared__ int abort_flag;
  const int group = threadIdx.x / kTpr, t = threadIdx.x & (kTpr - 1), per_cta = blockDim.x / kTpr;
  const long long groups = (long long)gridDim.x * per_cta;
  const int nvec = cols / VEC;
  const int row_bytes = cols * int(sizeof(T));
  const float inv = 1.0f / (float)cols;
  float* const ws = reinterpret_cast<float*>(ring_smem);
  uint8_t* const rings = reinterpret_cast<uint8_t*>(ws + (w != nullptr ? cols : 0));
  uint64_t* const bars = full + group * LN_RING;
  uint8_t* const ring = rings + (size_t)group * LN_RING * 2 * row_bytes;
  if (t == 0) {
    for (int i = 0; i < LN_RING; ++i) mbar_init(&bars[i], 1);
    if (group == 0) abort_flag = 0;
    fence_mbar_init();
  }
  pdl_launch_dependents();
  pdl_wait_prior_grids();
  bool ok = true;
  auto fetch = [&](long long r, int slot) {  // thread 0 of the group
    mbar_arrive_expect_tx(&bars[slot], 2 * row_bytes);
    bulk_load_1d(ring + (size_t)slot * 2 * row_bytes, x + r * ldx, row_bytes, &bars[slot]);
    bulk_load_1d(ring + (size_t)slot * 2 * row_bytes + row_bytes, dy + r * lddy, row_bytes, &bars[slot]);
  };
  const long long r0 = (long long)blockIdx.x * per_cta + group;
  if (t == 0) {
    for (int i = 0; i < LN_RING - 1; ++i)
      if (r0 + i * groups < rows) fetch(r0 + i * groups, i);
  }
  if (w != nullptr) stage_params<W, VEC>(w, ws, nvec);
  __syncthreads();
  Fv<VEC> dw[NV], db[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    dw[i].fill(0.0f);
    db[i].fill(0.0f);
  }
  int buf = 0, slot = 0;
  uint32_t phase = 0;
  float nmean = 0.0f, nrstd = 0.0f;
  if (r0 < rows) {
    nmean = mean_in[r0];
    nrstd = rstd_in[r0];
  }
  for (long long r = r0; r < rows; r += groups, buf ^= 1) {
    if (ok && !mbar_wait(&bars[slot], phase, &abort_flag, wait_ns)) ok = false;
    const float rstd = nrstd;
    Fv<VEC> xm[NV], g[NV], km, kr;
    km.fill(-nmean);
    kr.fill(nrstd);
    if (r + groups < rows) {
      nmean = mean_in[r + groups];
      nrstd = rstd_in[r + groups];
    }
    const T* xs = reinterpret_cast<const T*>(ring + (size_t)slot * 2 * row_bytes);
    const T* ds = reinterpret_cast<const T*>(ring + (size_t)slot * 2 * row_bytes + row_bytes);
    typename Fv<VEC>::Sum s0 = Fv<VEC>::zero(), s1 = Fv<VEC>::zero();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = t + i * kTpr;
      if (v < nvec) {
        LnRaw<T, VEC> rx, rd;
        rx.load(xs + v * VEC);
        rd.load(ds + v * VEC);
        rx.unpack(xm[i]);
        rd.unpack(g[i]);
        xm[i].add(km);
        db[i].add(g[i]);
        Fv<VEC> p;
        p.product(g[i], kr);
        dw[i].fma(p, xm[i]);
        if (w != nullptr) {
          staged_params<VEC>(ws, nvec, v, p);
          g[i].mul(p);
        }
        g[i].sum_into(s0);
        g[i].dot_into(s1, xm[i]);
      }
    }
    float s[2] = {Fv<VEC>::total(s0), Fv<VEC>::total(s1)};
    row_sum<2, kTpr>(s, red[buf] + group * (kTpr >> 5) * 2, kTpr, group);
    // Behind this barrier the whole group has the row in registers, and the row before it is long done with: the slot of that one
    // takes the row after next.
    const int free_slot = slot == 0 ? LN_RING - 1 : slot - 1;
    if (t == 0 && ok && r + (LN_RING - 1) * groups < rows) fetch(r + (LN_RING - 1) * groups, free_slot);
    if (dx != nullptr) {
      Fv<VEC> k1, k2;
      k1.fill(-s[0] * inv);
      k2.fill(-(s[1] * rstd) * inv * rstd);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = t + i * kTpr;
        if (v < nvec) {
          g[i].add(k1);
          g[i].fma(xm[i], k2);
          g[i].mul(kr);
          LnRaw<T, VEC>::store(dx + r * lddx + (long long)v * VEC, g[i]);
        }
      }
    }
    if (++slot == LN_RING) { slot = 0; phase ^= 1; }
  }
  __syncthreads();
  if (threadIdx.x == 0 && abort_flag != 0) {
    const uint64_t from = globaltimer_ns();  // copies that were issued get a bounded time to land
    while (globaltimer_ns() - from < 1000000ull) __nanosleep(1000);
    if (status != nullptr) atomicExch(status, int(ST_WAIT_TIMEOUT));
  }
  if (part == nullptr) return;
  float* const joined = reinterpret_cast<float*>(rings);  // the rings are not used any more
  float* const out = part + (long long)blockIdx.x * 2 * cols;
  // The groups' shares side by side in shared memory, then their sum, group after group.
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = t + i * kTpr;
    if (v < nvec) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        joined[(2 * group) * cols + v * VEC + j] = dw[i].get(j);
        joined[(2 * group + 1) * cols + v * VEC + j] = db[i].get(j);
      }
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * cols; c += blockDim.x) {
    float a = joined[c];
    for (int k = 1; k < per_cta; ++k) a += joined[2 * k * cols + c];
    out[c] = a;
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

// One call of f with the number of threads as a constant.
template <typename F>
auto with_threads(int tpr, F&& f) {
  switch (tpr) {
    case 32: return f(std::integral_constant<int, 32>{});
    case 64: return f(std::integral_constant<int, 64>{});
    case 128: return f(std::integral_constant<int, 128>{});
    case 256: return f(std::integral_constant<int, 256>{});
    case 512: return f(std::integral_constant<int, 512>{});
    default: return f(std::integral_constant<int, 1024>{});
  }
}

template <typename T, typename W, int VEC, int NV>
cudaError_t forward_rows(const void* x, const void* w, const void* b, void* y, float* mean, float* rstd, const LnShape& s, float eps, int tpr,
                         int num_sms, cudaStream_t stream) {
  auto go = [&](auto kern, int block, int ctas_per_sm, size_t smem) {
    const long long per_cta = block / tpr;
    const unsigned grid = (unsigned)std::min<long long>((s.rows + per_cta - 1) / per_cta, (long long)num_sms * ctas_per_sm);
    return launch_kernel_ex(kern, grid, block, smem, stream, 1, pdl_enabled(), static_cast<const T*>(x), static_cast<const W*>(w),
                            static_cast<const W*>(b), static_cast<T*>(y), mean, rstd, s.rows, (int)s.cols, s.ldx, s.ldy, eps, tpr);
  };
  if constexpr (VEC > 1) {
    return with_threads(tpr, [&](auto n) -> cudaError_t {
      constexpr int TPR = decltype(n)::value;
      constexpr int BLOCK = TPR >= 512 ? 1024 : 512;  // at most 8 groups that need a barrier
      // Parameters staged once per CTA where a group sees several rows (NV = 1 is the form for few rows or short ones).
      const size_t smem = ((w != nullptr ? 1 : 0) + (b != nullptr ? 1 : 0)) * (size_t)s.cols * 4;
      if constexpr (NV > 1) {
        if (s.rows >= 8LL * num_sms * (1024 / TPR) && smem > 0) {
          auto kern = ln_forward_kernel<T, W, VEC, NV, BLOCK, true, TPR>;
          static std::atomic<uint32_t> raised{0};  // once per device and instance
          int dev = 0;
          cudaGetDevice(&dev);
          if (!((raised.load(std::memory_order_relaxed) >> (dev & 31)) & 1u)) {
            const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * 16384 * 4);
            if (e != cudaSuccess) return e;
            raised.fetch_or(1u << (dev & 31));
          }
          return go(kern, BLOCK, smem <= 100 * 1024 ? 1024 / BLOCK : 1, smem);
        }
      }
      return go(ln_forward_kernel<T, W, VEC, NV, BLOCK, false, TPR>, BLOCK, 1024 / BLOCK, 0);
    });
  }
  return tpr <= 256 ? go(ln_forward_kernel<T, W, VEC, NV, 256, false, 0>, 256, 8, 0)
                    : go(ln_forward_kernel<T, W, VEC, NV, 1024, false, 0>, 1024, 1, 0);
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
    else e = forward_rows<T, W, VEC, MOST>(x, w, b, y, mean, rstd, s, eps, tpr, num_sms, stream);
  } else if (!vec && s.cols <= LN_SINGLE_FORWARD) {
    const int tpr = threads_per_row(s.cols, 4, 1024, few);
    const long long nv = (s.cols + tpr - 1) / tpr;
    e = nv <= 1 ? forward_rows<T, W, 1, 1>(x, w, b, y, mean, rstd, s, eps, tpr, num_sms, stream)
                : forward_rows<T, W, 1, 4>(x, w, b, y, mean, rstd, s, eps, tpr, num_sms, stream);
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

template <typename T, typename W, int VEC, int NV, int BLOCK = 512>
int backward_rows(const void* dy, const void* x, const float* mean, const float* rstd, const void* w, void* dx, float* part, const LnShape& s,
                  int tpr, int num_sms, cudaStream_t stream, int* parts) {
  const long long per_cta = BLOCK / tpr;
  const size_t smem = part != nullptr ? (size_t)(BLOCK / tpr) * s.cols * 8 : 0;
  *parts = (int)std::min<long long>((s.rows + per_cta - 1) / per_cta, std::min(num_sms, LN_PARTS));
  // n: the threads of a row as a constant, 0 in the form for single values
  auto go = [&](auto n) -> int {
    constexpr int TPR = decltype(n)::value <= BLOCK ? decltype(n)::value : BLOCK;
    auto kern = ln_backward_kernel<T, W, VEC, NV, BLOCK, TPR>;
    SX_ENSURE_DYN_SMEM(kern, 128 * 1024);
    const cudaError_t e = launch_kernel_ex(kern, (unsigned)*parts, BLOCK, smem, stream, 1, pdl_enabled(), static_cast<const T*>(dy),
                                           static_cast<const T*>(x), mean, rstd, static_cast<const W*>(w), static_cast<T*>(dx), part,
                                           s.rows, (int)s.cols, s.ldd, s.ldx, s.ldy, tpr);
    if (e != cudaSuccess) return launch_failed(e, "layer norm backward launch failed");
    count_launches(1);
    return SX_OK;
  };
  if constexpr (VEC > 1) return with_threads(tpr, go);
  return go(std::integral_constant<int, 0>{});
}

// Row groups of a CTA of the ring kernel (0: the rows are too long, or too short, for it).
int ring_groups(const LnShape& s, int eb, int tpr, int num_sms) {
  if (s.cols < LN_RING_COLS || tpr < 64) return 0;
  const long long ring = LN_RING * 2 * s.cols * eb;
  const long long fit = std::min<long long>(512 / tpr, (LN_RING_BYTES - 4 * s.cols) / ring);
  return (int)std::min(fit, (s.rows + num_sms - 1) / num_sms);
}

template <typename T, typename W, int VEC, int NV>
int backward_ring(const void* dy, const void* x, const float* mean, const float* rstd, const void* w, void* dx, float* part, const LnShape& s,
                  int tpr, int groups, const DeviceInfo& dev, cudaStream_t stream, int* parts) {
  // (the rings, 12 or 24 bytes a column and group, are also large enough for the sums at the end, 8 bytes)
  const size_t smem = (size_t)groups * LN_RING * 2 * s.cols * sizeof(T) + (w != nullptr ? (size_t)s.cols * 4 : 0);
  *parts = (int)std::min<long long>((s.rows + groups - 1) / groups, std::min(dev.num_sms, LN_PARTS));
  return with_threads(tpr, [&](auto n) -> int {
    constexpr int TPR = decltype(n)::value < 64 ? 64 : decltype(n)::value > 512 ? 512 : decltype(n)::value;
    auto kern = ln_backward_ring_kernel<T, W, VEC, NV, TPR>;
    SX_ENSURE_DYN_SMEM(kern, LN_RING_BYTES);
    const cudaError_t e = launch_kernel_ex(kern, (unsigned)*parts, (unsigned)(groups * TPR), smem, stream, 1, pdl_enabled(),
                                           static_cast<const T*>(dy), static_cast<const T*>(x), mean, rstd, static_cast<const W*>(w),
                                           static_cast<T*>(dx), part, s.rows, (int)s.cols, s.ldd, s.ldx, s.ldy, dev.status,
                                           wait_limit_ns_option());
    if (e != cudaSuccess) return launch_failed(e, "layer norm backward launch failed");
    count_launches(1);
    return SX_OK;
  });
}

template <typename T, typename W>
int backward(const void* dy, const void* x, const float* mean, const float* rstd, const void* w, void* dx, void* dw,
             void* db, const LnShape& s, float* part, const DeviceInfo& dev, cudaStream_t stream) {
  const int num_sms = dev.num_sms;
  constexpr int VEC = 16 / sizeof(T), MOST = 16 / VEC;
  const bool pdl = pdl_enabled();
  const bool params = dw != nullptr || db != nullptr;
  const long long tiles = (s.cols + LN_COL_TILE - 1) / LN_COL_TILE, eb = sizeof(T);
  const bool few = s.rows <= num_sms;
  const bool vec = s.cols % VEC == 0 && all_aligned({x, dy, dx, w}, {s.ldx * eb, s.ldd * eb, s.ldy * eb});
  float* to = params ? part : nullptr;
  int parts = 0, rc = SX_OK;
  cudaError_t e;
  const int tpr = vec ? threads_per_row(s.cols / VEC, MOST, 512, few) : std::max(128, threads_per_row(s.cols, 4, 1024, few));
  const long long nv = ((vec ? s.cols / VEC : s.cols) + tpr - 1) / tpr;
  if (s.rows > 0 && s.cols <= (vec ? 512 * 16 : LN_SINGLE_BACKWARD)) {
    const int ring = vec ? ring_groups(s, sizeof(T), tpr, num_sms) : 0;
    if (ring > 0)
      rc = nv <= 1 ? backward_ring<T, W, VEC, 1>(dy, x, mean, rstd, w, dx, to, s, tpr, ring, dev, stream, &parts)
                   : backward_ring<T, W, VEC, MOST>(dy, x, mean, rstd, w, dx, to, s, tpr, ring, dev, stream, &parts);
    else if (vec)
      rc = nv <= 1 ? backward_rows<T, W, VEC, 1>(dy, x, mean, rstd, w, dx, to, s, tpr, num_sms, stream, &parts)
                   : backward_rows<T, W, VEC, MOST>(dy, x, mean, rstd, w, dx, to, s, tpr, num_sms, stream, &parts);
    else
      rc = nv <= 1 ? backward_rows<T, W, 1, 1, 1024>(dy, x, mean, rstd, w, dx, to, s, tpr, num_sms, stream, &parts)
                   : backward_rows<T, W, 1, 4, 1024>(dy, x, mean, rstd, w, dx, to, s, tpr, num_sms, stream, &parts);
    if (rc != SX_OK || !params) return rc;
  } else if (s.rows > 0) {
    auto any = [&](auto n) -> cudaError_t {
      constexpr int V = decltype(n)::value;
      cudaError_t err = cudaSuccess;
      if (params) {  // before dx: dx may overwrite dy
        const long long vtiles = (s.cols / V + 31) / 32;
        parts = (int)std::min<long long>(std::min<long long>(LN_PARTS, (s.rows + 31) / 32), std::max<long long>(1, num_sms * 8LL / vtiles));
        err = launch_kernel_ex(ln_backward_columns_kernel<T, V>, (unsigned)std::min<long long>(vtiles * parts, num_sms * 8LL), LN_THREADS, 0,
                               stream, 1, pdl, static_cast<const T*>(dy), static_cast<const T*>(x), mean, rstd, part, s.rows, s.cols, s.ldd,
                               s.ldx, parts);
        if (err != cudaSuccess) return err;
        count_launches(1);
      }
      if (dx != nullptr) {
        err = launch_kernel_ex(ln_backward_dx_any_kernel<T, W, V>, (unsigned)std::min<long long>(s.rows, (long long)num_sms * 64), 512, 0, stream,
                               1, pdl, static_cast<const T*>(dy), static_cast<const T*>(x), mean, rstd, static_cast<const W*>(w),
                               static_cast<T*>(dx), s.rows, s.cols, s.ldd, s.ldx, s.ldy);
        if (err != cudaSuccess) return err;
        count_launches(1);
      }
      return err;
    };
    e = vec ? any(std::integral_constant<int, VEC>{}) : any(std::integral_constant<int, 1>{});
    if (e != cudaSuccess) return launch_failed(e, "layer norm backward launch failed");
  }
  if (params) {
    e = launch_kernel_ex(ln_backward_finish_kernel<W>, (unsigned)tiles, 1024u, 0, stream, 1, pdl, (const float*)part,
                         static_cast<W*>(dw), static_cast<W*>(db), s.cols, parts);
    if (e != cudaSuccess) return launch_failed(e, "layer norm backward launch failed");
    count_launches(1);
  }
  return SX_OK;
}

int check_shape(int64_t rows, int64_t cols, int32_t dtype, int32_t param_dtype) {
  if (rows < 0 || cols <= 0) return fail_fmt(SX_ERR_INVALID, "layer norm needs rows >= 0 and cols >= 1");
  if (cols > 0x3fffffffLL) return fail_fmt(SX_ERR_INVALID, "cols exceeds 2^30-1");
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
  const long long eb = dtype == SYMPLEX_DT_F32 ? 4 : 2, params = cols * (param_dtype == SYMPLEX_DT_F32 ? 4 : 2);
  const ByteRows out{y, rows, cols * eb, s.ldy * eb};
  const bool in_place = x == y && (s.ldx == s.ldy || rows == 1);
  if ((!in_place && share_bytes(out, {x, rows, cols * eb, s.ldx * eb})) || share_bytes(out, one_row(weight, params)) ||
      share_bytes(out, one_row(bias, params)))
    return fail_fmt(SX_ERR_INVALID, "y overlaps x (and is not x itself), weight or bias");
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
  DeviceInfo dev;
  if ((rc = current_device(&dev)) != SX_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  float* part = static_cast<float*>(workspace);
  if (dtype == SYMPLEX_DT_F32)
    return backward<float, float>(dy, x, mean, rstd, weight, dx, dweight, dbias, s, part, dev, st);
  if (param_dtype == SYMPLEX_DT_F32)
    return backward<__nv_bfloat16, float>(dy, x, mean, rstd, weight, dx, dweight, dbias, s, part, dev, st);
  return backward<__nv_bfloat16, __nv_bfloat16>(dy, x, mean, rstd, weight, dx, dweight, dbias, s, part, dev, st);
}

}  // extern "C"
