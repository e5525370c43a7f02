// Softmax cross entropy of a linear head (l = x W^T over a large vocabulary) and its gradients, logits never kept.
//
//   forward    per row t: lse = log sum_v exp l_tv,  loss = lse - l_t,target
//   backward   G_tv = (exp(l_tv - lse_t) - [v = target_t]) s_t,  dx = G W,  dW = G^T x
//
// A part of a row is (m, s): its largest logit m and s = sum exp(l - m); parts join by rescaling to the larger m. Powers
// are taken as 2^((l - m) log2 e) of the difference, not as one multiply-add of l and a scaled m: that would round m log2 e
// once, an error that grows with |m| and, where a part's logits are all near the type's lowest value, overflows.
//
// bf16 runs on the kernels of ce_pair_sm100.cu: the forward pass reduces each tile of logits where it is computed, the backward
// pass writes G for a piece of the vocabulary and multiplies it with W and x in one launch. fp32 takes pieces of the vocabulary
// through the 3xTF32 product with the operands split once (W's pieces as they come), logits of one piece at a time in scratch.
//
// This file: the row-wise kernels, the passes put together, and the C entry points.
#include <cuda_bf16.h>

#include <algorithm>

#include "../../include/symplex_b200.h"
#include "ce_params.h"
#include "ce_tiles.h"
#include "host_api.h"
#include "sm100_ptx.cuh"

namespace sx {
namespace {

constexpr float LOG2E = CE_LOG2E;
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
                     float2* __restrict__ part, float* __restrict__ target_logit, unsigned* __restrict__ done) {
  __shared__ float2 red[8];
  const long long t = blockIdx.x;
  if (t == 0 && threadIdx.x == 0) *done = 0;
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

// Sum of v over the CTA's kThreads threads, in thread 0.
template <int kThreads, typename S>
__device__ __forceinline__ S cta_total(S v, S* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x < 32) {
    v = threadIdx.x < kThreads / 32 ? red[threadIdx.x] : S(0);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  }
  __syncthreads();
  return v;
}

// Four rows per CTA, 64 threads on the parts [parts][T] of each (four rows make whole sectors of 32 bytes; 61 rows of 286 parts have
// 16 CTAs at work on them): lse and the row's loss. With `sum`, the CTA that finishes last sums the rows' losses, in 64 bits and in
// the order of the rows, and divides by the counted ones for a mean; the kernel before this one has set `done` to 0.
__global__ void __launch_bounds__(256)
ce_finish_kernel(const float2* __restrict__ part, int parts, const float* __restrict__ target_logit,
                 const long long* __restrict__ targets, float* __restrict__ row_loss, float* __restrict__ lse, long long T, long long V,
                 long long ignore, float* __restrict__ sum, int mean, unsigned* __restrict__ done) {
  __shared__ float2 red[8][4];
  __shared__ int last;
  __shared__ double sred[32];
  __shared__ long long cred[32];
  const int mine = threadIdx.x & 3;
  const long long t = (long long)blockIdx.x * 4 + mine;
  RowPart r{-INFINITY, 0.0f};
  if (t < T) {
    constexpr int AHEAD = 6;
    for (int i0 = threadIdx.x >> 2; i0 < parts; i0 += 64 * AHEAD) {
      float2 p[AHEAD];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k)
        p[k] = i0 + 64 * k < parts ? part[(long long)(i0 + 64 * k) * T + t] : make_float2(-INFINITY, 0.0f);
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) r = join(r, {p[k].x, p[k].y});
    }
  }
#pragma unroll
  for (int o = 16; o > 2; o >>= 1) r = join(r, {__shfl_xor_sync(0xffffffffu, r.m, o), __shfl_xor_sync(0xffffffffu, r.s, o)});
  if ((threadIdx.x & 31) < 4) red[threadIdx.x >> 5][mine] = make_float2(r.m, r.s);
  __syncthreads();
  if (threadIdx.x < 4 && t < T) {
    for (int w = 1; w < 8; ++w) r = join(r, {red[w][mine].x, red[w][mine].y});
    const float l = fmaf(log2f(r.s), LN2, r.m);
    lse[t] = l;
    const long long at = targets[t];
    row_loss[t] = at == ignore ? 0.0f : (at < 0 || at >= V) ? __int_as_float(0x7fc00000) : l - target_logit[t];
  }
  if (sum == nullptr) return;
  if (threadIdx.x < 4) __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    last = atomicAdd(done, 1u) == gridDim.x - 1;
    __threadfence();
  }
  __syncthreads();
  if (!last) return;
  double s = 0.0;
  long long n = 0;
  for (long long i = threadIdx.x; i < T; i += 256) {
    s += __ldcg(row_loss + i);
    n += targets[i] != ignore ? 1 : 0;
  }
  s = cta_total<256>(s, sred);
  n = cta_total<256>(n, cred);
  if (threadIdx.x == 0) *sum = (float)(mean ? s / (double)n : s);
}

// The sum over no rows, or their mean.
__global__ void ce_nothing_kernel(float* loss, int mean) {
  *loss = mean ? __int_as_float(0x7fc00000) : 0.0f;
}

// One CTA: what every counted row's gradient is multiplied with, dloss or dloss / counted rows (0 where no row counts: there is
// no gradient then).
__global__ void __launch_bounds__(1024)
ce_scale_kernel(const long long* __restrict__ targets, const float* __restrict__ dloss, float* __restrict__ scale, long long T,
                long long ignore, int mean) {
  __shared__ long long cred[32];
  long long n = 0;
  if (mean) {
    for (long long t = threadIdx.x; t < T; t += 1024) n += targets[t] != ignore ? 1 : 0;
    n = cta_total<1024>(n, cred);
  }
  if (threadIdx.x == 0) *scale = !mean ? *dloss : n > 0 ? (float)((double)*dloss / (double)n) : 0.0f;
}

// x with the ignored rows 0, for the backward pass: such a row may hold anything (NaN of a padded sequence), and G's zeros do not keep
// it out of G^T x. One warp a row, bf16 (fp32 does it where it splits x). 1999 x 768 bf16: 3 us of 440.
__global__ void __launch_bounds__(256)
ce_counted_rows_kernel(const uint16_t* __restrict__ x, long long ldx, int vec, const long long* __restrict__ targets, long long ignore,
                       uint16_t* __restrict__ to, long long ld, long long T, int H, int copies) {
  const int lane = threadIdx.x & 31;
  for (long long t = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); t < T; t += (long long)gridDim.x * 8) {
    const bool counted = targets[t] != ignore;
    const uint16_t* from = x + t * ldx;
    for (int k = 0; k < copies; ++k) {
      uint16_t* row = to + (k * T + t) * ld;
      int c = 0;
      if (vec) {
        for (int i = lane; i < H / 8; i += 32)
          reinterpret_cast<uint4*>(row)[i] = counted ? __ldg(reinterpret_cast<const uint4*>(from) + i) : make_uint4(0, 0, 0, 0);
        c = H / 8 * 8;
      }
      for (c += lane; c < H; c += 32) row[c] = counted ? from[c] : 0;
    }
  }
}

__device__ __forceinline__ float tf32_part(float x) {
  uint32_t r;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
  return __uint_as_float(r);
}

// fp32: G and its transpose from a piece of logits, both as the {hi, lo} tf32 planes the products read (hi = tf32(g), lo =
// tf32(g - hi)): G in parts of `chunk` columns (a multiple of 32), [part][2][rows][chunk], the columns of the last part past the
// piece 0; G^T [2][cols][ldt], planes plane_t values apart. Tiles of 32 rows x 128 columns, four values a thread at a time, the transpose
// through shared memory. 509 x 8192: 16 us (32 x 32 tiles, single values: 25).
constexpr int GT_PITCH = 33;
__global__ void __launch_bounds__(256)
ce_piece_grad_kernel(const float* __restrict__ L, long long ld, int cols, long long v0, const long long* __restrict__ targets,
                     const float* __restrict__ lse, const float* __restrict__ dloss, const float* __restrict__ scale,
                     float* __restrict__ G, int chunk, float* __restrict__ GT, long long ldt, long long plane_t,
                     long long rows, long long V, long long ignore) {
  __shared__ float tile[128 * GT_PITCH];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int padded = (cols + chunk - 1) / chunk * chunk;  // columns of all parts
  const long long row_tiles = (rows + 31) / 32, tiles = row_tiles * ((padded + 127) / 128);
  for (long long i = blockIdx.x; i < tiles; i += gridDim.x) {
    const long long r0 = i % row_tiles * 32;
    const int c0 = int(i / row_tiles) * 128, c = c0 + 4 * x;  // this thread's four columns: in one part, chunk is a multiple of 32
    const int part = c / chunk;
    float* const g_part = G + (long long)part * 2 * rows * chunk + (c - part * chunk);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const long long r = r0 + y + 8 * j;
      float g[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      if (r < rows && c < padded) {
        const long long at = targets[r];
        if (c < cols && at != ignore) {  // a piece's rows are a multiple of 8 values apart: four of them are there
          const float s = scale != nullptr ? *scale : dloss[r];
          const float l = lse[r];
          const float4 v = *reinterpret_cast<const float4*>(L + r * ld + c);
          const float w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (c + k >= cols) continue;
            g[k] = (exp2f((w[k] - l) * LOG2E) - (at == v0 + c + k ? 1.0f : 0.0f)) * s;
            if (at < 0 || at >= V) g[k] = __int_as_float(0x7fc00000);
          }
        }
        float hi[4], lo[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          hi[k] = tf32_part(g[k]);
          lo[k] = tf32_part(g[k] - hi[k]);
        }
        *reinterpret_cast<float4*>(g_part + r * chunk) = make_float4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<float4*>(g_part + (rows + r) * chunk) = make_float4(lo[0], lo[1], lo[2], lo[3]);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) tile[(4 * x + k) * GT_PITCH + y + 8 * j] = g[k];
    }
    __syncthreads();
    // four rows of one column: 8 neighbouring threads write its 128 bytes
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int e = threadIdx.x + 256 * j, ct = e >> 3, rt = (e & 7) * 4;
      const long long r = r0 + rt;
      if (r < rows && c0 + ct < cols) {  // rows of G^T are padded to a multiple of 8 values, with the zeros of rows past the last
        float hi[4], lo[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float g = tile[ct * GT_PITCH + rt + k];
          hi[k] = tf32_part(g);
          lo[k] = tf32_part(g - hi[k]);
        }
        float* const to = GT + (long long)(c0 + ct) * ldt + r;
        *reinterpret_cast<float4*>(to) = make_float4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<float4*>(to + plane_t) = make_float4(lo[0], lo[1], lo[2], lo[3]);
      }
    }
    __syncthreads();
  }
}

// An fp32 operand that is read in both orders, as {hi, lo} planes: `to` [2][rows][ld_to] and `trans` in parts of `chunk` rows,
// [part][2][cols][chunk], 0 past the last row. With targets, rows to be ignored are 0 whatever they hold. Tiles as above. Reading W once
// instead of once for each order: 14 us against 23 of the 509 x 512 x 8192 backward pass.
__global__ void __launch_bounds__(256)
ce_split_both_kernel(const float* __restrict__ in, long long ld, int vec, long long rows, int cols, const long long* __restrict__ targets,
                     long long ignore, float* __restrict__ to, long long ld_to, float* __restrict__ trans, long long chunk) {
  __shared__ float tile[128 * GT_PITCH];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  const long long padded = (rows + chunk - 1) / chunk * chunk;
  const long long row_tiles = (padded + 31) / 32, tiles = row_tiles * ((cols + 127) / 128);
  for (long long i = blockIdx.x; i < tiles; i += gridDim.x) {
    const long long r0 = i % row_tiles * 32;
    const int c0 = int(i / row_tiles) * 128, c = c0 + 4 * x;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const long long r = r0 + y + 8 * j;
      float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      if (r < rows && c < ld_to) {
        if (targets == nullptr || targets[r] != ignore) {
          const float* from = in + r * ld + c;
          if (vec && c + 4 <= cols) {
            const float4 w = __ldg(reinterpret_cast<const float4*>(from));
            v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
          } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (c + k < cols) v[k] = __ldg(from + k);
          }
        }
        float hi[4], lo[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          hi[k] = tf32_part(v[k]);
          lo[k] = tf32_part(v[k] - hi[k]);
        }
        *reinterpret_cast<float4*>(to + r * ld_to + c) = make_float4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<float4*>(to + (rows + r) * ld_to + c) = make_float4(lo[0], lo[1], lo[2], lo[3]);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) tile[(4 * x + k) * GT_PITCH + y + 8 * j] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int e = threadIdx.x + 256 * j, ct = e >> 3, rt = (e & 7) * 4;
      const long long r = r0 + rt;
      if (r < padded && c0 + ct < cols) {  // four rows are in one part: chunk is a multiple of 8
        const long long part = r / chunk;
        float hi[4], lo[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float v = tile[ct * GT_PITCH + rt + k];
          hi[k] = tf32_part(v);
          lo[k] = tf32_part(v - hi[k]);
        }
        float* const at = trans + ((part * 2) * cols + c0 + ct) * chunk + (r - part * chunk);
        *reinterpret_cast<float4*>(at) = make_float4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<float4*>(at + cols * chunk) = make_float4(lo[0], lo[1], lo[2], lo[3]);
      }
    }
    __syncthreads();
  }
}

// out = (add ? out : 0) + scale * the sum of `chunks` accumulators of n values each, in their order.
template <typename T>
__global__ void __launch_bounds__(256)
ce_join_kernel(const float* __restrict__ acc, int chunks, long long n, const float* __restrict__ scale, T* out, int add) {
  const float f = scale != nullptr ? *scale : 1.0f;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    float v = 0.0f;
    for (int c = 0; c < chunks; ++c) v += acc[c * n + i];
    v *= f;
    out[i] = add ? T(float(out[i]) + v) : T(v);
  }
}

// ------------------------------------------------------------------ host side
size_t up256(size_t x) { return (x + 255) & ~size_t(255); }
long long up(long long x, long long m) { return (x + m - 1) / m * m; }

struct Problem {
  const void *x, *W;  // looked at for their alignment only where a workspace is sized
  long long T, H, V, ldx, ldw;
  bool bf16;
  int eb;
  long long ignore;
  int reduction;

  // bf16 backward, few tokens: G in two bf16 parts. A row of G holds one large entry, the target's, whose rounding moves the whole row
  // of dx and the target's row of dW; over many tokens that adds a fifth to the results' own rounding, over one it may be as large as
  // that (error of the gradients of one token 2.6e-3, 1.6e-3 in two parts). The second part is T more rows of G (and of x), for which a
  // tile has room: 1 x 2048 x 32768 120 us either way; 100 x 1024 x 32768 would take 85 us instead of 73.
  bool two_parts() const { return bf16 && T <= 64; }
  long long g_rows() const { return two_parts() ? 2 * T : T; }

  // bf16 operands that TMA cannot read in place go through a padded copy.
  bool copy(const void* p, long long ld) const { return bf16 && (ld % 8 != 0 || reinterpret_cast<uintptr_t>(p) % 16 != 0); }
  bool copy_x() const { return copy(x, ldx); }
  bool copy_w() const { return copy(W, ldw); }
};

// Columns of the vocabulary worked through at a time.
// bf16 backward: G [T, piece] in bf16 of about 128 MB, so that most of it is still in L2 (126 MB) when the products read it,
// but at least 8192 columns: dx makes a round trip through its fp32 accumulator once a piece, 8 T H bytes beside 6 T H piece
// flops. fp32: logits of a piece of about 64 MB, with G and its transpose in two planes each four times that.
long long piece_columns(const Problem& p, bool backward) {
  const long long T = std::max<long long>(p.T, 1);
  if (p.bf16 && !backward) return up(p.V, 8);
  if (p.bf16) {
    const long long most = std::max<long long>(8192, (64ll << 20) / T / 256 * 256);
    return p.V <= most ? up(p.V, 8) : ce_piece_of_waves(T, p.V, most);
  }
  return std::min(up(p.V, 8), std::max<long long>(256, (16ll << 20) / T / 256 * 256));
}

// Everything the two passes keep in the workspace (offsets in bytes).
struct Layout {
  long long hp, tp, piece;  // padded H and T, columns of a piece (a multiple of 8)
  int pieces, parts;
  int chunks;         // parts that the vocabulary is cut into for dx, each with an accumulator
  long long chunk;    // fp32: columns of one
  size_t xcopy, wcopy, part, target_logit, row_loss, done, scale, G, acc;
  size_t xs, xts, ws, wts, logits, GT;  // fp32: operand planes, a piece's logits, G^T
  size_t total;
};

// fp32: columns of a tile of dx.
int dx_tile(long long H) { return H > 64 ? 128 : 64; }

Layout layout(const Problem& p, bool backward) {
  Layout w{};
  w.hp = up(p.H, 8);
  w.tp = up(p.T, 8);
  w.piece = piece_columns(p, backward);
  w.pieces = (int)((p.V + w.piece - 1) / w.piece);
  w.parts = p.bf16 ? ce_parts_most(p.T, p.V) : w.pieces;
  w.chunks = 1;
  w.chunk = up(w.piece, 32);
  if (backward && p.bf16) {
    // counted as the kernel cuts them: parts of as many k-blocks each, the last one shorter
    const long long nkb = (std::min(w.piece, p.V) + 63) / 64, c = ce_dx_chunks(p.g_rows(), p.H, std::min(w.piece, p.V)), kb = (nkb + c - 1) / c;
    w.chunks = (int)((nkb + kb - 1) / kb);
  }
  if (backward && !p.bf16) {
    // dx = G W has T / 128 x H / 128 tiles over the whole piece: cut into parts of 512 columns or more, as many as one wave of tiles
    // takes (509 x 512 x 8192: 160 tiles of 64 columns, two waves, took 71 us of the pass' 183; 144 of 128 columns, one wave: 141 in all; 126 with the passes since)
    const long long tiles = ((p.T + 127) / 128) * ((p.H + dx_tile(p.H) - 1) / dx_tile(p.H));
    const long long want = std::min<long long>(148 / tiles, w.piece / 512);
    if (want > 1) {
      w.chunk = up((w.piece + want - 1) / want, 32);
      w.chunks = (int)((w.piece + w.chunk - 1) / w.chunk);
    }
  }
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t at = off;
    off = up256(off + bytes);
    return at;
  };
  if (backward ? p.bf16 : p.copy_x()) w.xcopy = take((size_t)(backward ? p.g_rows() : p.T) * w.hp * 2);
  if (p.copy_w()) w.wcopy = take((size_t)w.piece * w.hp * 2);
  if (!p.bf16) {
    w.xs = take((size_t)2 * p.T * w.hp * 4);
    w.ws = take((size_t)2 * w.piece * w.hp * 4);
    w.logits = take((size_t)p.T * w.piece * 4);
  }
  if (!backward) {
    w.part = take((size_t)w.parts * p.T * sizeof(float2));
    w.target_logit = take((size_t)p.T * 4);
    w.row_loss = take((size_t)p.T * 4);
    w.done = take(4);
  } else {
    w.scale = take(4);
    const long long cols = p.bf16 ? w.piece : w.chunks * w.chunk;
    w.G = take((size_t)p.g_rows() * cols * (p.bf16 ? 2 : 8));
    if (w.chunks > 1 || p.two_parts()) w.acc = take((size_t)w.chunks * p.g_rows() * p.H * 4);
    else if (w.pieces > 1) w.acc = take((size_t)p.T * p.H * 4 * (p.bf16 ? 1 : 2));  // fp32: from one accumulator into the other
    if (!p.bf16) {
      w.xts = take((size_t)2 * p.H * w.tp * 4);
      w.wts = take((size_t)2 * p.H * cols * 4);
      w.GT = take((size_t)2 * w.piece * w.tp * 4);
    }
  }
  w.total = off;
  return w;
}

int check(Problem* p, const void* x, const void* W, int64_t T, int64_t H, int64_t V, int64_t ldx, int64_t ldw, int32_t dtype, int64_t ignore,
          int32_t reduction) {
  if (T < 0 || H <= 0 || V <= 0) return fail_fmt(SX_ERR_INVALID, "the loss needs T >= 0, H >= 1 and V >= 1");
  if (T > 0x3fffffffLL || H > 0x3fffffffLL || V > 0x3fffffffLL) return fail_fmt(SX_ERR_INVALID, "dimension exceeds 2^30-1");
  if (dtype != SYMPLEX_DT_F32 && dtype != SYMPLEX_DT_BF16)
    return fail_fmt(SX_ERR_INVALID, "dtype %d not supported (F32=9, BF16=11)", dtype);
  if (reduction < SYMPLEX_LOSS_NONE || reduction > SYMPLEX_LOSS_SUM) return fail_fmt(SX_ERR_INVALID, "reduction %d not supported", reduction);
  *p = Problem{x, W, T, H, V, ldx ? ldx : H, ldw ? ldw : H, dtype == SYMPLEX_DT_BF16, dtype == SYMPLEX_DT_BF16 ? 2 : 4, ignore, reduction};
  if (p->ldx < H || p->ldw < H) return fail_fmt(SX_ERR_INVALID, "leading dimension too small");
  return SX_OK;
}

int check_workspace(size_t need, const void* ws, size_t bytes) {
  if (need > bytes || (need && ws == nullptr)) return fail_fmt(SX_ERR_INVALID, "workspace too small: need %zu bytes, got %zu", need, bytes);
  if (reinterpret_cast<uintptr_t>(ws) % 256) return fail_fmt(SX_ERR_INVALID, "workspace must be 256-byte aligned");
  return SX_OK;
}

bool aligned_to(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// In plain stream order, like the tensor-core kernels of these passes: none of them has a griddepcontrol.wait.
#define CE_LAUNCH(kern, grid, block, ...)                                                                             \
  do {                                                                                                                \
    const cudaError_t e__ = launch_kernel_ex(kern, (unsigned)(grid), block, 0, stream, 1, false, __VA_ARGS__);         \
    if (e__ != cudaSuccess) return launch_failed(e__, "loss kernel launch failed");                                   \
    count_launches(1);                                                                                                \
  } while (0)

int prep(int rc) {
  if (rc != SX_OK) return launch_failed(cudaGetLastError(), "operand preparation launch failed");
  count_launches(1);
  return SX_OK;
}
#define CE_TRY(call)                  \
  do {                                \
    const int rc__ = (call);          \
    if (rc__ != SX_OK) return rc__;   \
  } while (0)

// x, or rows [v0, v0 + n) of W, where TMA can read it.
int readable(bool copy, const void* p, long long rows, long long cols, long long ld, uint8_t* to, cudaStream_t stream, CeMatrix* out) {
  if (!copy) {
    *out = CeMatrix{p, rows, cols, ld};
    return SX_OK;
  }
  const long long ldc = up(cols, 8);
  CE_TRY(prep(launch_repack_16(p, ld, 0, to, ldc, (int)rows, (int)cols, 1, stream)));
  *out = CeMatrix{to, rows, cols, ldc};
  return SX_OK;
}

// fp32: C[M, N] = A B^T + R from operands in {hi, lo} planes, both K contiguous.
int split_product(const CeCommon& c, const float* A, long long lda, long long plane_a, const float* B, long long ldb, long long plane_b, float* C,
                  long long ldc, const float* R, long long M, long long N, long long K, cudaStream_t stream, int batch = 1, int bn = 0) {
  TcGemmArgs g{};
  g.M = M; g.N = N; g.K = K;
  g.batch = batch;
  g.A = A; g.lda = lda; g.a_plane_stride = plane_a;
  g.B = B; g.ldb = ldb; g.b_plane_stride = plane_b;
  g.C = C; g.ldc = ldc; g.c_batch_stride = M * ldc;
  g.alpha = 1.0f;
  g.beta = R != nullptr ? 1.0f : 0.0f;
  g.residual = R;
  g.status = c.status;
  g.num_sms = c.num_sms;
  g.wait_limit_ns = c.wait_limit_ns;
  // the general product's rule: 128-column tiles where they fill the chip
  g.bn = bn ? bn : N > 64 && ((M + 127) / 128) * ((N + 127) / 128) * batch >= c.num_sms ? 128 : 64;
  const int rc = launch_gemm_tf32x3(g, stream);
  if (rc == SX_ERR_EXEC) return launch_failed(cudaGetLastError(), "loss product launch failed");
  if (rc == SX_OK) count_launches(1);
  return rc;
}

int forward(const Problem& p, const CeCommon& dev, const long long* targets, float* loss, float* lse, uint8_t* ws, cudaStream_t stream) {
  const Layout w = layout(p, false);
  float2* part = reinterpret_cast<float2*>(ws + w.part);
  float* target_logit = reinterpret_cast<float*>(ws + w.target_logit);
  float* row_loss = p.reduction == SYMPLEX_LOSS_NONE ? loss : reinterpret_cast<float*>(ws + w.row_loss);
  unsigned* done = reinterpret_cast<unsigned*>(ws + w.done);
  int parts = w.parts;
  if (p.bf16) {
    CeForward f{};
    CE_TRY(readable(p.copy_x(), p.x, p.T, p.H, p.ldx, ws + w.xcopy, stream, &f.x));
    CE_TRY(readable(p.copy_w(), p.W, p.V, p.H, p.ldw, ws + w.wcopy, stream, &f.W));
    f.targets = targets;
    f.part = part;
    f.target_logit = target_logit;
    f.done = done;
    CE_TRY(launch_ce_forward(dev, f, stream, &parts));
  } else {
    float *xs = reinterpret_cast<float*>(ws + w.xs), *wsp = reinterpret_cast<float*>(ws + w.ws), *logits = reinterpret_cast<float*>(ws + w.logits);
    CE_TRY(prep(launch_split_tf32(static_cast<const float*>(p.x), p.ldx, 0, xs, (int)p.T, (int)p.H, (int)w.hp, 1, stream)));
    for (int i = 0; i < w.pieces; ++i) {
      const long long v0 = i * w.piece, n = std::min(w.piece, p.V - v0);
      CE_TRY(prep(launch_split_tf32(static_cast<const float*>(p.W) + v0 * p.ldw, p.ldw, 0, wsp, (int)n, (int)p.H, (int)w.hp, 1, stream)));
      CE_TRY(split_product(dev, xs, w.hp, p.T * w.hp, wsp, w.hp, n * w.hp, logits, w.piece, nullptr, p.T, n, p.H, stream));
      CE_LAUNCH(ce_piece_rows_kernel, p.T, 256, (const float*)logits, w.piece, (int)n, v0, targets, part + i * p.T, target_logit, done);
    }
  }
  const bool all = p.reduction != SYMPLEX_LOSS_NONE;
  CE_LAUNCH(ce_finish_kernel, (p.T + 3) / 4, 256, (const float2*)part, parts, (const float*)target_logit, targets, row_loss, lse, p.T, p.V,
            p.ignore, all ? loss : nullptr, p.reduction == SYMPLEX_LOSS_MEAN ? 1 : 0, done);
  return SX_OK;
}

int backward(const Problem& p, const CeCommon& dev, const float* dloss, const long long* targets, const float* lse, void* dx, void* dW,
             uint8_t* ws, cudaStream_t stream) {
  const Layout w = layout(p, true);
  const bool per_row = p.reduction == SYMPLEX_LOSS_NONE;
  float* scale = nullptr;
  if (!per_row) {
    scale = reinterpret_cast<float*>(ws + w.scale);
    CE_LAUNCH(ce_scale_kernel, 1, 1024, targets, dloss, scale, p.T, p.ignore, p.reduction == SYMPLEX_LOSS_MEAN ? 1 : 0);
  }
  if (p.bf16) {
    const int vec = p.ldx % 8 == 0 && reinterpret_cast<uintptr_t>(p.x) % 16 == 0;
    CE_LAUNCH(ce_counted_rows_kernel, std::min<long long>((p.T + 7) / 8, dev.num_sms * 8LL), 256, static_cast<const uint16_t*>(p.x), p.ldx, vec, targets,
              p.ignore, reinterpret_cast<uint16_t*>(ws + w.xcopy), w.hp, p.T, (int)p.H, p.two_parts() ? 2 : 1);
    const CeMatrix x{ws + w.xcopy, p.T, p.H, w.hp}, xs{ws + w.xcopy, p.g_rows(), p.H, w.hp};
    float* acc = reinterpret_cast<float*>(ws + w.acc);
    for (int i = 0; i < w.pieces; ++i) {
      const long long v0 = i * w.piece, n = std::min(w.piece, p.V - v0);
      CeMatrix Wp;
      CE_TRY(readable(p.copy_w(), static_cast<const uint8_t*>(p.W) + (size_t)v0 * p.ldw * 2, n, p.H, p.ldw, ws + w.wcopy, stream, &Wp));
      CeGrad g{};
      g.x = x;
      g.W = Wp;
      g.G = ws + w.G;
      g.ldg = w.piece;
      g.lo = p.two_parts();
      g.targets = targets;
      g.lse = lse;
      g.dloss = per_row ? dloss : nullptr;
      g.v0 = v0;
      g.V = p.V;
      g.ignore = p.ignore;
      CE_TRY(launch_ce_grad(dev, g, stream));
      // One factor for all rows is left out of G, where rounding it would move every large entry (the targets', close to
      // -factor) the same way, and multiplied into the results' fp32 sums instead.
      CeProducts d{};
      d.G = CeMatrix{ws + w.G, p.g_rows(), n, w.piece};
      d.x = xs;
      d.W = Wp;
      d.acc = acc;
      d.chunks = w.chunks;
      d.first = i == 0;
      d.last = i == w.pieces - 1;
      d.dx = p.two_parts() ? nullptr : dx;
      d.dW = static_cast<uint8_t*>(dW) + (size_t)v0 * p.H * 2;
      d.scale = scale;
      CE_TRY(launch_ce_products(dev, d, stream));
    }
    if (w.chunks > 1 || p.two_parts())  // [chunk][part of G][T][H]
      CE_LAUNCH(ce_join_kernel<__nv_bfloat16>, std::min<long long>((p.T * p.H + 255) / 256, dev.num_sms * 8LL), 256, (const float*)acc, w.chunks * (p.two_parts() ? 2 : 1),
                p.T * p.H, (const float*)scale, static_cast<__nv_bfloat16*>(dx), 0);
    return SX_OK;
  }
  auto at = [&](size_t off) { return reinterpret_cast<float*>(ws + off); };
  float *xs = at(w.xs), *xts = at(w.xts), *wsp = at(w.ws), *wts = at(w.wts), *logits = at(w.logits), *G = at(w.G), *GT = at(w.GT);
  float* acc[2] = {at(w.acc), at(w.acc) + p.T * p.H};  // one chunk: accumulators of pieces
  auto split_both = [&](const float* in, long long ld, long long rows, const long long* tg, float* to, float* trans, long long chunk) -> int {
    const int v = ld % 4 == 0 && reinterpret_cast<uintptr_t>(in) % 16 == 0;
    const long long tiles = ((rows + chunk - 1) / chunk * chunk + 31) / 32 * ((p.H + 127) / 128);
    CE_LAUNCH(ce_split_both_kernel, std::min<long long>(tiles, dev.num_sms * 8LL), 256, in, ld, v, rows, (int)p.H, tg, p.ignore, to, w.hp, trans, chunk);
    return SX_OK;
  };
  CE_TRY(split_both(static_cast<const float*>(p.x), p.ldx, p.T, targets, xs, xts, w.tp));
  for (int i = 0; i < w.pieces; ++i) {
    const long long v0 = i * w.piece, n = std::min(w.piece, p.V - v0);
    const float* Wp = static_cast<const float*>(p.W) + v0 * p.ldw;
    // W in both orders; W^T, for dx, in parts of the vocabulary
    const int chunks = (int)((n + w.chunk - 1) / w.chunk);
    CE_TRY(split_both(Wp, p.ldw, n, nullptr, wsp, wts, w.chunk));
    CE_TRY(split_product(dev, xs, w.hp, p.T * w.hp, wsp, w.hp, n * w.hp, logits, w.piece, nullptr, p.T, n, p.H, stream));
    const long long tiles = (p.T + 31) / 32 * ((chunks * w.chunk + 127) / 128);
    CE_LAUNCH(ce_piece_grad_kernel, std::min<long long>(tiles, dev.num_sms * 8LL), 256, (const float*)logits, w.piece, (int)n, v0, targets, lse,
              dloss, (const float*)scale, G, (int)w.chunk, GT, w.tp, n * w.tp, p.T, p.V, p.ignore);
    if (w.chunks > 1) {
      CE_TRY(split_product(dev, G, w.chunk, p.T * w.chunk, wts, w.chunk, p.H * w.chunk, acc[0], p.H, nullptr, p.T, p.H, w.chunk, stream, chunks, dx_tile(p.H)));
      CE_LAUNCH(ce_join_kernel<float>, std::min<long long>((p.T * p.H + 255) / 256, dev.num_sms * 8LL), 256, (const float*)acc[0], chunks, p.T * p.H,
                (const float*)nullptr, static_cast<float*>(dx), i > 0 ? 1 : 0);
    } else {
      float* to = i == w.pieces - 1 ? static_cast<float*>(dx) : acc[i & 1];
      CE_TRY(split_product(dev, G, w.chunk, p.T * w.chunk, wts, w.chunk, p.H * w.chunk, to, p.H, i ? acc[(i & 1) ^ 1] : nullptr, p.T, p.H, n, stream));
    }
    CE_TRY(split_product(dev, GT, w.tp, n * w.tp, xts, w.tp, p.H * w.tp, static_cast<float*>(dW) + v0 * p.H, p.H, nullptr, n, p.H, p.T, stream));
  }
  return SX_OK;
}

}  // namespace
}  // namespace sx

using namespace sx;

extern "C" {

size_t symplex_b200_linear_cross_entropy_workspace_bytes(const void* x, const void* W, int64_t T, int64_t H, int64_t V, int64_t ldx,
                                                         int64_t ldw, int32_t dtype) {
  Problem p;
  if (check(&p, x, W, T, H, V, ldx, ldw, dtype, 0, 0) != SX_OK || T == 0) return 0;
  return layout(p, false).total;
}

int symplex_b200_linear_cross_entropy(const void* x, const void* W, const int64_t* targets, float* loss, float* lse,
                                      int64_t T, int64_t H, int64_t V, int64_t ldx, int64_t ldw, int32_t dtype,
                                      int64_t ignore_index, int32_t reduction, void* workspace, size_t workspace_bytes,
                                      void* stream) {
  Problem p;
  int rc = check(&p, x, W, T, H, V, ldx, ldw, dtype, ignore_index, reduction);
  if (rc != SX_OK) return rc;
  if (T == 0 && reduction == SYMPLEX_LOSS_NONE) return SX_OK;
  if (loss == nullptr || (T > 0 && (x == nullptr || W == nullptr || targets == nullptr || lse == nullptr)))
    return fail_fmt(SX_ERR_INVALID, "null pointer");
  if (!aligned_to(x, p.eb) || !aligned_to(W, p.eb) || !aligned_to(targets, 8) || !aligned_to(loss, 4) || !aligned_to(lse, 4))
    return fail_fmt(SX_ERR_INVALID, "a pointer is not aligned to its element type");
  if ((rc = check_workspace(symplex_b200_linear_cross_entropy_workspace_bytes(x, W, T, H, V, ldx, ldw, dtype), workspace, workspace_bytes)) != SX_OK) return rc;
  DeviceInfo info;
  if ((rc = current_device(&info)) != SX_OK) return rc;
  const CeCommon dev{info.num_sms, info.status, wait_limit_ns_option()};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const long long* tg = reinterpret_cast<const long long*>(targets);
  if (T == 0) {
    cudaStream_t stream = st;
    CE_LAUNCH(ce_nothing_kernel, 1, 1, loss, reduction == SYMPLEX_LOSS_MEAN ? 1 : 0);
    return SX_OK;
  }
  return forward(p, dev, tg, loss, lse, static_cast<uint8_t*>(workspace), st);
}

size_t symplex_b200_linear_cross_entropy_backward_workspace_bytes(const void* x, const void* W, int64_t T, int64_t H, int64_t V,
                                                                  int64_t ldx, int64_t ldw, int32_t dtype) {
  Problem p;
  if (check(&p, x, W, T, H, V, ldx, ldw, dtype, 0, 0) != SX_OK || T == 0) return 0;
  return layout(p, true).total;
}

int symplex_b200_linear_cross_entropy_backward(const float* dloss, const void* x, const void* W, const int64_t* targets,
                                               const float* lse, void* dx, void* dW, int64_t T, int64_t H, int64_t V,
                                               int64_t ldx, int64_t ldw, int32_t dtype, int64_t ignore_index,
                                               int32_t reduction, void* workspace, size_t workspace_bytes, void* stream) {
  Problem p;
  int rc = check(&p, x, W, T, H, V, ldx, ldw, dtype, ignore_index, reduction);
  if (rc != SX_OK) return rc;
  if (dW == nullptr || (T > 0 && (dloss == nullptr || x == nullptr || W == nullptr || targets == nullptr || lse == nullptr || dx == nullptr)))
    return fail_fmt(SX_ERR_INVALID, "null pointer");
  if (!aligned_to(x, p.eb) || !aligned_to(W, p.eb) || !aligned_to(targets, 8) || !aligned_to(dloss, 4) || !aligned_to(lse, 4) ||
      !aligned_to(dx, p.eb) || !aligned_to(dW, p.eb))
    return fail_fmt(SX_ERR_INVALID, "a pointer is not aligned to its element type");
  if ((rc = check_workspace(symplex_b200_linear_cross_entropy_backward_workspace_bytes(x, W, T, H, V, ldx, ldw, dtype), workspace, workspace_bytes)) != SX_OK)
    return rc;
  DeviceInfo info;
  if ((rc = current_device(&info)) != SX_OK) return rc;
  const CeCommon dev{info.num_sms, info.status, wait_limit_ns_option()};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (T == 0) {
    const cudaError_t e = cudaMemsetAsync(dW, 0, (size_t)V * H * p.eb, st);
    return e == cudaSuccess ? SX_OK : launch_failed(e, "cudaMemsetAsync");
  }
  return backward(p, dev, dloss, reinterpret_cast<const long long*>(targets), lse, dx, dW, static_cast<uint8_t*>(workspace), st);
}

}  // extern "C"
