// Softmax cross entropy of a linear head (l = x W^T over a large vocabulary) and its gradients, logits never kept.
//
//   forward    per row t: lse = log sum_v exp l_tv,  loss = lse - l_t,target
//   backward   G_tv = (exp(l_tv - lse_t) - [v = target_t]) s_t,  dx = G W,  dW = G^T x
//
// A part of a row is (m, s): its largest logit m and s = sum exp(l - m); parts join by rescaling to the larger m. Powers
// are taken as 2^((l - m) log2 e) of the difference, not as one multiply-add of l and a scaled m: that would round m log2 e
// once, an error that grows with |m| and, where a part's logits are all near the type's lowest value, overflows.
//
// This file: the row-wise kernels, the pieces of the vocabulary through the general GEMM, and the C entry points.
#include <cuda_bf16.h>

#include <algorithm>

#include "../../include/symplex_b200.h"
#include "host_api.h"
#include "sm100_ptx.cuh"

namespace sx {
namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

struct RowPart {
  float m, s;
};

// Join two parts of one row. A part without any mass (m = -inf: no columns, or all logits -inf) adds nothing.
__device__ __forceinline__ RowPart join(RowPart a, RowPart b) {
  const float m = fmaxf(a.m, b.m);
  if (m == -INFINITY) return {m, a.s + b.s};  // s is 0, or NaN where a logit was
  return {m, a.s * exp2f((a.m - m) * LOG2E) + b.s * exp2f((b.m - m) * LOG2E)};
}

// One CTA per row of a piece of logits L[T, ld]: its part of the row, and the target's logit if it is in the piece.
__global__ void __launch_bounds__(256)
ce_piece_rows_kernel(const float* __restrict__ L, long long ld, int cols, long long v0, const long long* __restrict__ targets,
                     float2* __restrict__ part, float* __restrict__ target_logit) {
  __shared__ float2 red[8];
  pdl_launch_dependents();
  pdl_wait_prior_grids();
  const long long t = blockIdx.x;
  const float* row = L + t * ld;
  float top = -INFINITY;
  bool nan = false;
  for (int c = threadIdx.x; c < cols; c += 256) {
    const float v = row[c];
    top = fmaxf(top, v);
    nan = nan || v != v;
  }
  RowPart r{top, 0.0f};
  if (top != -INFINITY) {
    for (int c = threadIdx.x; c < cols; c += 256) r.s += exp2f((row[c] - top) * LOG2E);
  }
  if (nan) r.s = __int_as_float(0x7fc00000);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) r = join(r, {__shfl_xor_sync(0xffffffffu, r.m, o), __shfl_xor_sync(0xffffffffu, r.s, o)});
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = make_float2(r.m, r.s);
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 8; ++w) r = join(r, {red[w].x, red[w].y});
    part[t] = make_float2(r.m, r.s);
    const long long at = targets[t] - v0;
    if (at >= 0 && at < cols) target_logit[t] = row[at];
  }
}

// One warp per row: the parts [parts][T] joined, lse and the row's loss.
__global__ void __launch_bounds__(256)
ce_finish_kernel(const float2* __restrict__ part, int parts, const float* __restrict__ target_logit,
                 const long long* __restrict__ targets, float* __restrict__ loss, float* __restrict__ lse, long long T, long long V,
                 long long ignore) {
  pdl_launch_dependents();
  pdl_wait_prior_grids();
  const int lane = threadIdx.x & 31;
  const long long t = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (t >= T) return;
  RowPart r{-INFINITY, 0.0f};
  for (int i = lane; i < parts; i += 32) {
    const float2 p = part[(long long)i * T + t];
    r = join(r, {p.x, p.y});
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) r = join(r, {__shfl_xor_sync(0xffffffffu, r.m, o), __shfl_xor_sync(0xffffffffu, r.s, o)});
  if (lane == 0) {
    const float l = fmaf(log2f(r.s), LN2, r.m);
    lse[t] = l;
    const long long at = targets[t];
    loss[t] = at == ignore ? 0.0f : (at < 0 || at >= V) ? __int_as_float(0x7fc00000) : l - target_logit[t];
  }
}

// Sum of v over the CTA (1024 threads), in thread 0.
template <typename S>
__device__ __forceinline__ S cta_total(S v, S* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x < 32) {
    v = red[threadIdx.x];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  }
  __syncthreads();
  return v;
}

// One CTA: the rows' losses summed in 64 bits, divided by the counted rows for a mean.
__global__ void __launch_bounds__(1024)
ce_reduce_kernel(const float* __restrict__ row_loss, const long long* __restrict__ targets, float* __restrict__ loss, long long T,
                 long long ignore, int mean) {
  __shared__ double sred[32];
  __shared__ long long cred[32];
  pdl_launch_dependents();
  pdl_wait_prior_grids();
  double s = 0.0;
  long long n = 0;
  for (long long t = threadIdx.x; t < T; t += 1024) {
    s += row_loss[t];
    n += targets[t] != ignore ? 1 : 0;
  }
  s = cta_total(s, sred);
  n = cta_total(n, cred);
  if (threadIdx.x == 0) *loss = (float)(mean ? s / (double)n : s);
}

// One CTA: 1 / counted rows (0 where there are none: no row has a gradient then).
__global__ void __launch_bounds__(1024)
ce_count_kernel(const long long* __restrict__ targets, float* __restrict__ inv_count, long long T, long long ignore) {
  __shared__ long long cred[32];
  pdl_launch_dependents();
  pdl_wait_prior_grids();
  long long n = 0;
  for (long long t = threadIdx.x; t < T; t += 1024) n += targets[t] != ignore ? 1 : 0;
  n = cta_total(n, cred);
  if (threadIdx.x == 0) *inv_count = n > 0 ? (float)(1.0 / (double)n) : 0.0f;
}

// G and its transpose from a piece of logits: 32 x 32 tiles, the transpose through shared memory.
template <typename T>
__global__ void __launch_bounds__(256)
ce_piece_grad_kernel(const float* __restrict__ L, long long ld, int cols, long long v0, const long long* __restrict__ targets,
                     const float* __restrict__ lse, const float* __restrict__ dloss, int per_row, const float* __restrict__ inv_count,
                     T* __restrict__ G, long long ldg, T* __restrict__ GT, long long ldt, long long rows, long long V, long long ignore) {
  __shared__ T tile[32][33];
  pdl_launch_dependents();
  pdl_wait_prior_grids();
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  const long long row_tiles = (rows + 31) / 32, tiles = row_tiles * ((cols + 31) / 32);
  for (long long i = blockIdx.x; i < tiles; i += gridDim.x) {
    const long long r0 = i % row_tiles * 32;
    const int c0 = int(i / row_tiles) * 32;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const long long r = r0 + y + 8 * j;
      const int c = c0 + x;
      float g = 0.0f;
      if (r < rows && c < cols) {
        const long long at = targets[r];
        if (at != ignore) {
          float s = dloss[per_row ? r : 0];
          if (inv_count != nullptr) s *= *inv_count;
          g = (exp2f((L[r * ld + c] - lse[r]) * LOG2E) - (at == v0 + c ? 1.0f : 0.0f)) * s;
          // The fp32 products round operands to tf32 by adding to their bits, which carries the NaN that arithmetic
          // makes (all mantissa bits set) into the sign: a quiet NaN with a short mantissa survives.
          if (at < 0 || at >= V || g != g) g = __int_as_float(0x7fc00000);
        }
        G[r * ldg + c] = T(g);
      }
      tile[y + 8 * j][x] = T(g);
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = c0 + y + 8 * j;
      const long long r = r0 + x;
      if (r < rows && c < cols) GT[c * ldt + r] = tile[x][y + 8 * j];
    }
    __syncthreads();
  }
}

__global__ void __launch_bounds__(256)
ce_round_kernel(const float* __restrict__ in, __nv_bfloat16* __restrict__ out, long long n) {
  pdl_launch_dependents();
  pdl_wait_prior_grids();
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) out[i] = __nv_bfloat16(in[i]);
}

// ------------------------------------------------------------------ host side
size_t up256(size_t x) { return (x + 255) & ~size_t(255); }
long long up(long long x, long long m) { return (x + m - 1) / m * m; }

struct Problem {
  long long T, H, V, ldx, ldw;
  bool bf16;
  int eb;
  long long ignore;
  int reduction;
};

// Columns of one piece: T x piece fp32 logits of about PIECE_BYTES.
constexpr long long PIECE_BYTES = 256ll << 20;
long long piece_columns(long long T, long long V) {
  const long long c = PIECE_BYTES / 4 / std::max<long long>(T, 1) / 256 * 256;
  return std::min(up(V, 8), std::max<long long>(256, c));
}

symplex_gemm_desc product(const Problem& p, long long M, long long N, long long K, bool out_f32, int b_layout, long long lda,
                          long long ldb, long long ldc) {
  symplex_gemm_desc d;
  symplex_b200_gemm_desc_init(&d, M, N, K, p.bf16 ? SYMPLEX_DT_BF16 : SYMPLEX_DT_F32,
                              out_f32 || !p.bf16 ? SYMPLEX_DT_F32 : SYMPLEX_DT_BF16);
  d.b_layout = b_layout;
  d.lda = lda;
  d.ldb = ldb;
  d.ldc = ldc;
  return d;
}

// Everything the two passes keep in the workspace.
struct Layout {
  long long piece, ldl, ldt;
  int parts;
  size_t logits, part, target_logit, row_loss, inv_count, G, GT, acc[2], gemm, gemm_bytes, total;
};

Layout layout(const Problem& p, bool backward) {
  Layout w{};
  w.piece = piece_columns(p.T, p.V);
  w.ldl = up(w.piece, 8);
  w.ldt = up(p.T, 8);
  w.parts = (int)((p.V + w.piece - 1) / w.piece);
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t at = off;
    off = up256(off + bytes);
    return at;
  };
  w.logits = take((size_t)p.T * w.ldl * 4);
  if (!backward) {
    w.part = take((size_t)w.parts * p.T * sizeof(float2));
    w.target_logit = take((size_t)p.T * 4);
    w.row_loss = take((size_t)p.T * 4);
  } else {
    w.inv_count = take(4);
    w.G = take((size_t)p.T * w.ldl * p.eb);
    w.GT = take((size_t)w.piece * w.ldt * p.eb);
    w.acc[0] = take((size_t)p.T * p.H * 4);
    w.acc[1] = take((size_t)p.T * p.H * 4);
  }
  // The products' own scratch, at the size of a full piece.
  auto need = [&](const symplex_gemm_desc& d) { w.gemm_bytes = std::max(w.gemm_bytes, symplex_b200_gemm_workspace_bytes(&d)); };
  need(product(p, p.T, w.piece, p.H, true, SYMPLEX_COL_MAJOR, p.ldx, p.ldw, w.ldl));
  if (backward) {
    need(product(p, p.T, p.H, w.piece, true, SYMPLEX_ROW_MAJOR, w.ldl, p.ldw, p.H));
    need(product(p, w.piece, p.H, p.T, false, SYMPLEX_ROW_MAJOR, w.ldt, p.ldx, p.H));
  }
  w.gemm = take(w.gemm_bytes);
  w.total = off;
  return w;
}

int check(Problem* p, int64_t T, int64_t H, int64_t V, int64_t ldx, int64_t ldw, int32_t dtype, int64_t ignore, int32_t reduction) {
  if (T < 0 || H <= 0 || V <= 0) return fail_fmt(SX_ERR_INVALID, "the loss needs T >= 0, H >= 1 and V >= 1");
  if (T > 0x3fffffffLL || H > 0x3fffffffLL || V > 0x3fffffffLL) return fail_fmt(SX_ERR_INVALID, "dimension exceeds 2^30-1");
  if (dtype != SYMPLEX_DT_F32 && dtype != SYMPLEX_DT_BF16)
    return fail_fmt(SX_ERR_INVALID, "dtype %d not supported (F32=9, BF16=11)", dtype);
  if (reduction < SYMPLEX_LOSS_NONE || reduction > SYMPLEX_LOSS_SUM) return fail_fmt(SX_ERR_INVALID, "reduction %d not supported", reduction);
  *p = Problem{T, H, V, ldx ? ldx : H, ldw ? ldw : H, dtype == SYMPLEX_DT_BF16, dtype == SYMPLEX_DT_BF16 ? 2 : 4, ignore, reduction};
  if (p->ldx < H || p->ldw < H) return fail_fmt(SX_ERR_INVALID, "leading dimension too small");
  return SX_OK;
}

int check_workspace(size_t need, const void* ws, size_t bytes) {
  if (need > bytes || (need && ws == nullptr)) return fail_fmt(SX_ERR_INVALID, "workspace too small: need %zu bytes, got %zu", need, bytes);
  if (reinterpret_cast<uintptr_t>(ws) % 256) return fail_fmt(SX_ERR_INVALID, "workspace must be 256-byte aligned");
  return SX_OK;
}

bool aligned_to(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

#define CE_LAUNCH(kern, grid, block, ...)                                                                             \
  do {                                                                                                                \
    const cudaError_t e__ = launch_kernel_ex(kern, (unsigned)(grid), block, 0, stream, 1, pdl_enabled(), __VA_ARGS__); \
    if (e__ != cudaSuccess) return launch_failed(e__, "loss kernel launch failed");                                   \
    count_launches(1);                                                                                                \
  } while (0)

int forward(const Problem& p, const void* x, const void* W, const long long* targets, float* loss, float* lse, uint8_t* ws,
            cudaStream_t stream) {
  const Layout w = layout(p, false);
  float* logits = reinterpret_cast<float*>(ws + w.logits);
  float2* part = reinterpret_cast<float2*>(ws + w.part);
  float* target_logit = reinterpret_cast<float*>(ws + w.target_logit);
  float* row_loss = p.reduction == SYMPLEX_LOSS_NONE ? loss : reinterpret_cast<float*>(ws + w.row_loss);
  for (int i = 0; i < w.parts; ++i) {
    const long long v0 = i * w.piece, n = std::min(w.piece, p.V - v0);
    const symplex_gemm_desc d = product(p, p.T, n, p.H, true, SYMPLEX_COL_MAJOR, p.ldx, p.ldw, w.ldl);
    const int rc = symplex_b200_gemm_ws(&d, x, static_cast<const uint8_t*>(W) + (size_t)v0 * p.ldw * p.eb, logits, nullptr, nullptr,
                                        ws + w.gemm, w.gemm_bytes, stream);
    if (rc != SX_OK) return rc;
    CE_LAUNCH(ce_piece_rows_kernel, p.T, 256, (const float*)logits, w.ldl, (int)n, v0, targets, part + i * p.T, target_logit);
  }
  CE_LAUNCH(ce_finish_kernel, (p.T + 7) / 8, 256, (const float2*)part, w.parts, (const float*)target_logit, targets, row_loss, lse, p.T, p.V,
            p.ignore);
  if (p.reduction != SYMPLEX_LOSS_NONE)
    CE_LAUNCH(ce_reduce_kernel, 1, 1024, (const float*)row_loss, targets, loss, p.T, p.ignore, p.reduction == SYMPLEX_LOSS_MEAN ? 1 : 0);
  return SX_OK;
}

int backward(const Problem& p, const float* dloss, const void* x, const void* W, const long long* targets, const float* lse, void* dx,
             void* dW, uint8_t* ws, int num_sms, cudaStream_t stream) {
  const Layout w = layout(p, true);
  float* logits = reinterpret_cast<float*>(ws + w.logits);
  float* inv_count = nullptr;
  if (p.reduction == SYMPLEX_LOSS_MEAN) {
    inv_count = reinterpret_cast<float*>(ws + w.inv_count);
    CE_LAUNCH(ce_count_kernel, 1, 1024, targets, inv_count, p.T, p.ignore);
  }
  const int per_row = p.reduction == SYMPLEX_LOSS_NONE ? 1 : 0;
  float* acc[2] = {reinterpret_cast<float*>(ws + w.acc[0]), reinterpret_cast<float*>(ws + w.acc[1])};
  for (int i = 0; i < w.parts; ++i) {
    const long long v0 = i * w.piece, n = std::min(w.piece, p.V - v0);
    const uint8_t* Wp = static_cast<const uint8_t*>(W) + (size_t)v0 * p.ldw * p.eb;
    symplex_gemm_desc d = product(p, p.T, n, p.H, true, SYMPLEX_COL_MAJOR, p.ldx, p.ldw, w.ldl);
    int rc = symplex_b200_gemm_ws(&d, x, Wp, logits, nullptr, nullptr, ws + w.gemm, w.gemm_bytes, stream);
    if (rc != SX_OK) return rc;
    const long long tiles = (p.T + 31) / 32 * ((n + 31) / 32);
    const unsigned grid = (unsigned)std::min<long long>(tiles, num_sms * 8LL);
    if (p.bf16)
      CE_LAUNCH(ce_piece_grad_kernel<__nv_bfloat16>, grid, 256, (const float*)logits, w.ldl, (int)n, v0, targets, lse, dloss, per_row,
                (const float*)inv_count, reinterpret_cast<__nv_bfloat16*>(ws + w.G), w.ldl, reinterpret_cast<__nv_bfloat16*>(ws + w.GT),
                w.ldt, p.T, p.V, p.ignore);
    else
      CE_LAUNCH(ce_piece_grad_kernel<float>, grid, 256, (const float*)logits, w.ldl, (int)n, v0, targets, lse, dloss, per_row,
                (const float*)inv_count, reinterpret_cast<float*>(ws + w.G), w.ldl, reinterpret_cast<float*>(ws + w.GT), w.ldt, p.T,
                p.V, p.ignore);
    // dx: pieces add up in 32 bits, from one accumulator into the other; fp32 ends in dx itself
    d = product(p, p.T, p.H, n, true, SYMPLEX_ROW_MAJOR, w.ldl, p.ldw, p.H);
    d.beta = i ? 1.0f : 0.0f;
    float* to = !p.bf16 && i == w.parts - 1 ? static_cast<float*>(dx) : acc[i & 1];
    rc = symplex_b200_gemm_ws(&d, ws + w.G, Wp, to, nullptr, i ? acc[(i & 1) ^ 1] : nullptr, ws + w.gemm, w.gemm_bytes, stream);
    if (rc != SX_OK) return rc;
    d = product(p, n, p.H, p.T, false, SYMPLEX_ROW_MAJOR, w.ldt, p.ldx, p.H);
    rc = symplex_b200_gemm_ws(&d, ws + w.GT, x, static_cast<uint8_t*>(dW) + (size_t)v0 * p.H * p.eb, nullptr, nullptr, ws + w.gemm,
                              w.gemm_bytes, stream);
    if (rc != SX_OK) return rc;
  }
  if (p.bf16)
    CE_LAUNCH(ce_round_kernel, std::min<long long>((p.T * p.H + 255) / 256, num_sms * 16LL), 256, (const float*)acc[(w.parts - 1) & 1],
              static_cast<__nv_bfloat16*>(dx), p.T * p.H);
  return SX_OK;
}

}  // namespace
}  // namespace sx

using namespace sx;

extern "C" {

size_t symplex_b200_linear_cross_entropy_workspace_bytes(int64_t T, int64_t H, int64_t V, int32_t dtype) {
  Problem p;
  if (check(&p, T, H, V, 0, 0, dtype, 0, 0) != SX_OK || T == 0) return 0;
  return layout(p, false).total;
}

int symplex_b200_linear_cross_entropy(const void* x, const void* W, const int64_t* targets, float* loss, float* lse,
                                      int64_t T, int64_t H, int64_t V, int64_t ldx, int64_t ldw, int32_t dtype,
                                      int64_t ignore_index, int32_t reduction, void* workspace, size_t workspace_bytes,
                                      void* stream) {
  Problem p;
  int rc = check(&p, T, H, V, ldx, ldw, dtype, ignore_index, reduction);
  if (rc != SX_OK) return rc;
  if (T == 0 && reduction == SYMPLEX_LOSS_NONE) return SX_OK;
  if (loss == nullptr || (T > 0 && (x == nullptr || W == nullptr || targets == nullptr || lse == nullptr)))
    return fail_fmt(SX_ERR_INVALID, "null pointer");
  if (!aligned_to(x, p.eb) || !aligned_to(W, p.eb) || !aligned_to(targets, 8) || !aligned_to(loss, 4) || !aligned_to(lse, 4))
    return fail_fmt(SX_ERR_INVALID, "a pointer is not aligned to its element type");
  if ((rc = check_workspace(symplex_b200_linear_cross_entropy_workspace_bytes(T, H, V, dtype), workspace, workspace_bytes)) != SX_OK) return rc;
  DeviceInfo dev;
  if ((rc = current_device(&dev)) != SX_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const long long* tg = reinterpret_cast<const long long*>(targets);
  if (T == 0) {
    cudaStream_t stream = st;
    CE_LAUNCH(ce_reduce_kernel, 1, 1024, (const float*)nullptr, tg, loss, 0LL, (long long)ignore_index, reduction == SYMPLEX_LOSS_MEAN ? 1 : 0);
    return SX_OK;
  }
  return forward(p, x, W, tg, loss, lse, static_cast<uint8_t*>(workspace), st);
}

size_t symplex_b200_linear_cross_entropy_backward_workspace_bytes(int64_t T, int64_t H, int64_t V, int32_t dtype) {
  Problem p;
  if (check(&p, T, H, V, 0, 0, dtype, 0, 0) != SX_OK || T == 0) return 0;
  return layout(p, true).total;
}

int symplex_b200_linear_cross_entropy_backward(const float* dloss, const void* x, const void* W, const int64_t* targets,
                                               const float* lse, void* dx, void* dW, int64_t T, int64_t H, int64_t V,
                                               int64_t ldx, int64_t ldw, int32_t dtype, int64_t ignore_index,
                                               int32_t reduction, void* workspace, size_t workspace_bytes, void* stream) {
  Problem p;
  int rc = check(&p, T, H, V, ldx, ldw, dtype, ignore_index, reduction);
  if (rc != SX_OK) return rc;
  if (dW == nullptr || (T > 0 && (dloss == nullptr || x == nullptr || W == nullptr || targets == nullptr || lse == nullptr || dx == nullptr)))
    return fail_fmt(SX_ERR_INVALID, "null pointer");
  if (!aligned_to(x, p.eb) || !aligned_to(W, p.eb) || !aligned_to(targets, 8) || !aligned_to(dloss, 4) || !aligned_to(lse, 4) ||
      !aligned_to(dx, p.eb) || !aligned_to(dW, p.eb))
    return fail_fmt(SX_ERR_INVALID, "a pointer is not aligned to its element type");
  if ((rc = check_workspace(symplex_b200_linear_cross_entropy_backward_workspace_bytes(T, H, V, dtype), workspace, workspace_bytes)) != SX_OK)
    return rc;
  DeviceInfo dev;
  if ((rc = current_device(&dev)) != SX_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (T == 0) {
    const cudaError_t e = cudaMemsetAsync(dW, 0, (size_t)V * H * p.eb, st);
    return e == cudaSuccess ? SX_OK : launch_failed(e, "cudaMemsetAsync");
  }
  return backward(p, dloss, x, W, reinterpret_cast<const long long*>(targets), lse, dx, dW, static_cast<uint8_t*>(workspace), dev.num_sms, st);
}

}  // extern "C"
