// Products of a few rows with 4-bit weights that carry a scale (and a zero) per group of consecutive k:
//
//   C[m][n] = act(sum_g scale[n][g] * sum_{k in g} (code[n][k] - zero[n][g]) * A[m][k] + bias[n])
//
// Bound by HBM: N K / 2 bytes of codes, read once for every 16 rows of A.
//
// int4_mma_kernel: the rows of W are the M side of mma.sync m16n8k16, the rows of A (up to 8 per fragment) its N side. A code
// becomes bf16 exactly - four masked bits under the exponent of 128 read 128 + code, minus (128 + zero) - so the products are
// exact and each group's sum is scaled once, in fp32. Which k a fragment slot stands for is free as long as both operands agree:
// a lane takes 8 consecutive k of its row (one 32-bit word), whose nibbles j and j + 4 fall into the halves of one register
// (pairs (k0,k4), (k1,k5), ...), and the same pairs of A are put together with byte permutes. No shuffle, no shared memory on
// the way in. 4-bit products are far below what even the warp-level tensor path delivers, so the tcgen05 path has nothing to
// add here: what has to be fast is the dequantisation, 11 instructions for 8 codes.
#include <cuda_bf16.h>

#include <algorithm>

#include "../../include/symplex_b200.h"
#include "epilogue.cuh"
#include "host_api.h"
#include "sm100_ptx.cuh"

namespace sx {
namespace {

// One value of the activation set with the accurate device functions.
__device__ __forceinline__ float activate(float x, int act) {
  switch (act) {
    case ACT_RELU: return fmaxf(x, 0.0f);
    case ACT_GELU: return 0.5f * x * (1.0f + tanhf(0.7978845608028654f * (x + 0.044715f * x * x * x)));
    case ACT_SIGMOID: return 1.0f / (1.0f + expf(-x));
    case ACT_TANH: return tanhf(x);
    case ACT_SILU: return x / (1.0f + expf(-x));
    default: return x;
  }
}

struct Int4Args {
  const __nv_bfloat16* A;
  const uint8_t* codes;
  const void* scales;
  const uint8_t* zeros;
  const float* bias;
  void* C;
  int M, N, K, group, groups, group_log2;  // group_log2: -1 where group is no power of two
  long long lda, ldq, ldc;
  int act;
};

// ------------------------------------------------------------------ fast path
constexpr int MV_WARPS = 8;
constexpr int MV_TILE = 32;  // rows of W per warp: two m16 tiles share every fragment of A
constexpr int MV_K = 128;    // k of one step
constexpr int MV_AHEAD = 2;  // steps in flight per warp: 2 KB of codes each, and 16 warps an SM
constexpr int MV_STAGE_BYTES = 88 * 1024;  // shared memory of a CTA for A, if all of A fits: two CTAs an SM

__device__ __forceinline__ uint32_t ldg_stream_32(const void* p) {
  uint32_t v;
  asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 ldg_stream_64(const void* p) {
  uint2 v;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}
__device__ __forceinline__ uint4 ldg_stream_128(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16_zero(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t sub_bf16x2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// Eight codes -> four registers (k0,k4), (k1,k5), (k2,k6), (k3,k7) of code - zero; zero2 = (128 + zero) twice.
__device__ __forceinline__ void dequant8(uint32_t w, uint32_t zero2, uint32_t (&out)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) out[j] = sub_bf16x2(((w >> (4 * j)) & 0x000f000fu) | 0x43004300u, zero2);
}

// What a warp holds of one step of 128 k for its 32 rows: per row slot (g, g + 8, g + 16, g + 24) four words of codes and the
// scales (and zeros) of the step's groups, packed as they lie in memory. kGW = 128, 64 or 32 is how many k share a scale within
// a step: a lane's words are laid out so that the four lanes of a row stay inside one group for every pair of MMAs.
template <int kGW, typename ST, bool kZeros>
struct MvStep {
  static constexpr int GROUPS = MV_K / kGW;
  static constexpr int SCALE_WORDS = (GROUPS * int(sizeof(ST)) + 3) / 4;
  uint32_t c[4][4];
  uint32_t s[4][SCALE_WORDS];
  uint32_t z[4];

  __device__ __forceinline__ float scale(int r, int j) const {
    if constexpr (sizeof(ST) == 4) return __uint_as_float(s[r][j]);
    return __uint_as_float(j & 1 ? s[r][j / 2] & 0xffff0000u : s[r][j / 2] << 16);  // bf16: the high half of a float
  }
  // 128 + zero, twice, in bf16
  __device__ __forceinline__ uint32_t zero2(int r, int j) const {
    if constexpr (!kZeros) return 0x43084308u;
    return __byte_perm(z[r], 0x00000043u, 0x4040u + 0x0101u * j);
  }

  // row: this lane's four rows, at the first byte of the lane's share of step 0. k0: first k of the step, t: lane in the quad. Words
  // past K repeat the row's beginning (A is 0 there). s_vec: the step's groups are GROUPS whole scales in a row, aligned.
  __device__ __forceinline__ void load(const Int4Args& p, const uint8_t* const (&row)[4], const uint32_t (&srow)[4], int k0, int t, int s_vec) {
#pragma unroll
    for (int h = 0; h < GROUPS; ++h) {
      const int k = k0 + h * kGW + t * (kGW / 4);
      const long long at = k < p.K ? k0 / 2 + h * (kGW / 2) : 0;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if constexpr (kGW == 128) {
          const uint4 v = ldg_stream_128(row[r] + at);
          c[r][0] = v.x; c[r][1] = v.y; c[r][2] = v.z; c[r][3] = v.w;
        } else if constexpr (kGW == 64) {
          const uint2 v = ldg_stream_64(row[r] + at);
          c[r][2 * h] = v.x; c[r][2 * h + 1] = v.y;
        } else {
          c[r][h] = ldg_stream_32(row[r] + at);
        }
      }
    }
    const ST* scales = static_cast<const ST*>(p.scales);
    if (GROUPS > 1 && s_vec) {
      const uint32_t g = k0 / kGW;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if constexpr (SCALE_WORDS == 1) {
          s[r][0] = __ldg(reinterpret_cast<const uint32_t*>(scales + (srow[r] + g)));
        } else if constexpr (SCALE_WORDS == 2) {
          const uint2 v = __ldg(reinterpret_cast<const uint2*>(scales + (srow[r] + g)));
          s[r][0] = v.x; s[r][1] = v.y;
        } else {
          const uint4 v = __ldg(reinterpret_cast<const uint4*>(scales + (srow[r] + g)));
          s[r][0] = v.x; s[r][1] = v.y; s[r][2] = v.z; s[r][3] = v.w;
        }
        if constexpr (kZeros && GROUPS == 2) z[r] = __ldg(reinterpret_cast<const uint16_t*>(p.zeros + (srow[r] + g)));
        if constexpr (kZeros && GROUPS == 4) z[r] = __ldg(reinterpret_cast<const uint32_t*>(p.zeros + (srow[r] + g)));
      }
      return;
    }
#pragma unroll
    for (int j = 0; j < GROUPS; ++j) {
      const int k = min(k0 + j * kGW, p.K - 1);
      const uint32_t g = p.group_log2 >= 0 ? k >> p.group_log2 : k / p.group;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if constexpr (sizeof(ST) == 4) {
          s[r][j] = __ldg(reinterpret_cast<const uint32_t*>(scales) + (srow[r] + g));
        } else {
          const uint32_t v = __ldg(reinterpret_cast<const uint16_t*>(scales) + (srow[r] + g));
          s[r][j / 2] = j & 1 ? s[r][j / 2] | (v << 16) : v;
        }
        if constexpr (kZeros) {
          const uint32_t v = __ldg(p.zeros + (srow[r] + g));
          z[r] = j ? z[r] | (v << (8 * j)) : v;
        }
      }
    }
  }
};

// A in shared memory: rows of 16-byte blocks of 8 k, each block as the pairs the dequantised words have, (k0,k4) (k1,k5) (k2,k6)
// (k3,k7); block b of a row stands at b ^ ((b >> 3) & 1), and rows are MvPad blocks longer than their k: the eight lanes of a
// quarter warp (two rows, four shares of a group) then read eight different bank groups. Row `rows` is zeros, for lanes whose row
// of A does not exist.
template <int kGW> constexpr int MvPad = kGW == 128 ? 2 : kGW == 64 ? 1 : 4;

__device__ __forceinline__ void stage_a(const Int4Args& p, uint4* to, int pitch, int m0, int rows, int k0, int kn, int a_vec) {
  const int blocks = kn >> 3;
  for (int e = threadIdx.x; e < blocks * (rows + 1); e += MV_WARPS * 32) {
    const int m = e / blocks, b = e - m * blocks;
    const int k = k0 + 8 * b;
    uint4 x = make_uint4(0, 0, 0, 0);
    if (m < rows && k < p.K) {  // K is a multiple of 8: a block is inside or outside
      const __nv_bfloat16* a = p.A + (m0 + m) * p.lda + k;
      if (a_vec) {
        x = __ldg(reinterpret_cast<const uint4*>(a));
      } else {
        const uint16_t* u = reinterpret_cast<const uint16_t*>(a);
        x.x = u[0] | (uint32_t(u[1]) << 16);
        x.y = u[2] | (uint32_t(u[3]) << 16);
        x.z = u[4] | (uint32_t(u[5]) << 16);
        x.w = u[6] | (uint32_t(u[7]) << 16);
      }
    }
    to[m * pitch + (b ^ ((b >> 3) & 1))] = make_uint4(__byte_perm(x.x, x.z, 0x5410), __byte_perm(x.x, x.z, 0x7632),
                                                      __byte_perm(x.y, x.w, 0x5410), __byte_perm(x.y, x.w, 0x7632));
  }
}

struct MvPlan {
  int kw_log2;      // warps that share a row tile, each with every kw-th step
  int chunk_steps;  // steps whose A is staged at a time, a multiple of kw * MV_AHEAD; all of them where A fits
  int pitch;        // 16-byte blocks from one staged row to the next
  int a_vec, s_vec, out_bf16;
};

template <int kGW, int kNB, typename ST, bool kZeros>
__global__ void __launch_bounds__(MV_WARPS * 32, 2)
int4_mma_kernel(const Int4Args p, const MvPlan plan) {
  using Step = MvStep<kGW, ST, kZeros>;
  constexpr int WPG = kGW / 32;  // words of a lane per group of a step
  extern __shared__ uint4 a_smem[];
  __shared__ float red[MV_WARPS][MV_TILE][8 * kNB + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int kw = 1 << plan.kw_log2;
  const int my_k = warp & (kw - 1), my_r = warp >> plan.kw_log2;
  const int rows_cta = (MV_WARPS >> plan.kw_log2) * MV_TILE;
  const long long n0 = (long long)blockIdx.x * rows_cta + my_r * MV_TILE;
  const int m0 = blockIdx.y * (8 * kNB);
  const int m_here = min(8 * kNB, p.M - m0);

  const uint8_t* row[4];
  uint32_t srow[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const long long n = min(n0 + g + 8 * r, (long long)p.N - 1);  // rows past the end repeat the last one and are not written
    row[r] = p.codes + n * p.ldq + t * (kGW / 8);
    srow[r] = (uint32_t)n * (uint32_t)p.groups;  // checked by the host: N * groups < 2^32
  }
  const int steps = (p.K + MV_K - 1) / MV_K;
  pdl_launch_dependents();
  pdl_wait_prior_grids();
  Step buf[MV_AHEAD];
#pragma unroll
  for (int i = 0; i < MV_AHEAD; ++i)
    if (my_k + i * kw < steps) buf[i].load(p, row, srow, (my_k + i * kw) * MV_K, t, plan.s_vec);

  const int buf_blocks = plan.pitch * (m_here + 1);
  const int chunk_k = plan.chunk_steps * MV_K;
  stage_a(p, a_smem, plan.pitch, m0, m_here, 0, chunk_k, plan.a_vec);
  __syncthreads();

  const uint4* arow[kNB];
  float acc[kNB][2][4] = {};
  // one step; block: first 16-byte block of the step inside the staged rows (a multiple of 16)
  auto compute = [&](const Step& st, int k0, int block) {
#pragma unroll
    for (int j = 0; j < Step::GROUPS; ++j) {
      float part[kNB][2][4];
      uint32_t zero2[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) zero2[r] = st.zero2(r, j);
#pragma unroll
      for (int i = 0; i < WPG; ++i) {
        const int w = j * WPG + i;
        const int b = j * (kGW / 8) + t * (kGW / 32) + i;  // this lane's block of the step
        uint4 x[kNB];
#pragma unroll
        for (int nb = 0; nb < kNB; ++nb) x[nb] = arow[nb][block + (b ^ ((b >> 3) & 1))];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          uint32_t lo[4], hi[4];  // rows g and g + 8 of this m16 tile
          dequant8(st.c[2 * mt][w], zero2[2 * mt], lo);
          dequant8(st.c[2 * mt + 1][w], zero2[2 * mt + 1], hi);
#pragma unroll
          for (int nb = 0; nb < kNB; ++nb) {
            if (i == 0) mma_bf16_zero(part[nb][mt], lo[0], hi[0], lo[1], hi[1], x[nb].x, x[nb].y);
            else mma_bf16(part[nb][mt], lo[0], hi[0], lo[1], hi[1], x[nb].x, x[nb].y);
            mma_bf16(part[nb][mt], lo[2], hi[2], lo[3], hi[3], x[nb].z, x[nb].w);
          }
        }
      }
      // A group that lies past K whole has sums of 0 and repeats a scale, which may be anything: 0 * inf must not count.
      if (Step::GROUPS == 1 || k0 + j * kGW < p.K) {
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          const float s0 = st.scale(2 * mt, j), s1 = st.scale(2 * mt + 1, j);
#pragma unroll
          for (int nb = 0; nb < kNB; ++nb) {
            acc[nb][mt][0] = fmaf(s0, part[nb][mt][0], acc[nb][mt][0]);
            acc[nb][mt][1] = fmaf(s0, part[nb][mt][1], acc[nb][mt][1]);
            acc[nb][mt][2] = fmaf(s1, part[nb][mt][2], acc[nb][mt][2]);
            acc[nb][mt][3] = fmaf(s1, part[nb][mt][3], acc[nb][mt][3]);
          }
        }
      }
    }
  };

  for (int c = 0, s0 = 0; s0 < steps; ++c, s0 += plan.chunk_steps) {
    // Behind the barrier chunk c is staged and nobody reads chunk c - 1 any more: its buffer takes chunk c + 1.
    if (c > 0) __syncthreads();
    if (s0 + plan.chunk_steps < steps)
      stage_a(p, a_smem + ((c + 1) & 1) * buf_blocks, plan.pitch, m0, m_here, (s0 + plan.chunk_steps) * MV_K, chunk_k, plan.a_vec);
#pragma unroll
    for (int b = 0; b < kNB; ++b) arow[b] = a_smem + (c & 1) * buf_blocks + min(8 * b + g, m_here) * plan.pitch;
    const int end = min(s0 + plan.chunk_steps, steps);
    for (int u = s0 + my_k; u < end; u += MV_AHEAD * kw) {
#pragma unroll
      for (int i = 0; i < MV_AHEAD; ++i) {
        const int v = u + i * kw;
        if (v < end) {
          compute(buf[i], v * MV_K, (v - s0) * (MV_K / 8));
          if (v + MV_AHEAD * kw < steps) buf[i].load(p, row, srow, (v + MV_AHEAD * kw) * MV_K, t, plan.s_vec);
        }
      }
    }
  }

#pragma unroll
  for (int nb = 0; nb < kNB; ++nb)
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int i = 0; i < 4; ++i) red[warp][16 * mt + g + 8 * (i >> 1)][8 * nb + 2 * t + (i & 1)] = acc[nb][mt][i];
  __syncthreads();
  for (int e = threadIdx.x; e < m_here * rows_cta; e += MV_WARPS * 32) {
    const int m = e / rows_cta, r = e - m * rows_cta;
    const long long n = (long long)blockIdx.x * rows_cta + r;
    if (n >= p.N) continue;
    float v = 0.0f;
    for (int i = 0; i < kw; ++i) v += red[(r / MV_TILE) * kw + i][r % MV_TILE][m];  // a fixed order
    if (p.bias != nullptr) v += p.bias[n];
    v = activate(v, p.act);
    const long long at = (m0 + m) * p.ldc + n;
    if (plan.out_bf16) static_cast<__nv_bfloat16*>(p.C)[at] = __nv_bfloat16(v);
    else static_cast<float*>(p.C)[at] = v;
  }
}

// ------------------------------------------------------------------ any K, stride and alignment
constexpr int MV_ROWS = 8;  // rows of A of one warp's accumulators

// One warp per row of W, codes byte by byte: any K, stride and alignment.
template <typename ST, typename OutT>
__global__ void __launch_bounds__(256)
int4_matvec_any_kernel(const Int4Args p) {
  pdl_launch_dependents();
  pdl_wait_prior_grids();
  const int lane = threadIdx.x & 31;
  const long long n = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (n >= p.N) return;
  const ST* scales = static_cast<const ST*>(p.scales) + n * p.groups;
  const uint8_t* zeros = p.zeros ? p.zeros + n * p.groups : nullptr;
  for (int m0 = 0; m0 < p.M; m0 += MV_ROWS) {
    float acc[MV_ROWS] = {};
    for (int g = 0; g < p.groups; ++g) {
      const int k1 = min(p.K, (g + 1) * p.group);
      const int z = zeros ? zeros[g] : 8;
      float part[MV_ROWS] = {};
      for (int k = g * p.group + 2 * lane; k < k1; k += 64) {
        const int byte = p.codes[n * p.ldq + (k >> 1)];
        const float q0 = float((byte & 15) - z), q1 = float((byte >> 4) - z);
#pragma unroll
        for (int m = 0; m < MV_ROWS; ++m) {
          if (m0 + m >= p.M) break;
          const __nv_bfloat16* a = p.A + (m0 + m) * p.lda + k;
          part[m] = fmaf(q0, float(a[0]), part[m]);
          if (k + 1 < k1) part[m] = fmaf(q1, float(a[1]), part[m]);
        }
      }
      const float s = float(scales[g]);
#pragma unroll
      for (int m = 0; m < MV_ROWS; ++m) acc[m] = fmaf(s, part[m], acc[m]);
    }
#pragma unroll
    for (int m = 0; m < MV_ROWS; ++m) {
      if (m0 + m >= p.M) break;
      float v = acc[m];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if (lane == 0) {
        if (p.bias != nullptr) v += p.bias[n];
        static_cast<OutT*>(p.C)[(m0 + m) * p.ldc + n] = OutT(activate(v, p.act));
      }
    }
  }
}

// One warp per group of weights.
template <typename T, typename ST>
__global__ void __launch_bounds__(256)
int4_quantize_kernel(const T* __restrict__ W, uint8_t* __restrict__ codes, ST* __restrict__ scales, uint8_t* __restrict__ zeros,
                     long long N, int K, int group, int groups, long long ldw) {
  pdl_launch_dependents();
  pdl_wait_prior_grids();
  const int lane = threadIdx.x & 31;
  const long long ldq = ((long long)K + 1) / 2;
  for (long long i = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); i < N * groups; i += (long long)gridDim.x * 8) {
    const long long n = i / groups;
    const int g = int(i - n * groups);
    const int k0 = g * group, k1 = min(K, k0 + group);
    const T* row = W + n * ldw;
    float lo = 0.0f, hi = 0.0f;
    bool bad = false;
    for (int k = k0 + lane; k < k1; k += 32) {
      const float v = float(row[k]);
      lo = fminf(lo, v);
      hi = fmaxf(hi, v);
      bad = bad || !(fabsf(v) <= 3.402823466e38f);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    bad = __any_sync(0xffffffffu, bad);
    // hi / 15 - lo / 15 does not overflow where hi - lo would
    float s = zeros != nullptr ? __fdiv_rn(hi, 15.0f) - __fdiv_rn(lo, 15.0f) : __fdiv_rn(fmaxf(hi, -lo), 7.0f);
    s = float(ST(s));
    if (s == 0.0f) s = 1.0f;
    int z = 8;
    if (zeros != nullptr) z = min(15, max(0, __float2int_rn(__fdiv_rn(-lo, s))));
    if (bad) s = __int_as_float(0x7fc00000);  // a weight that is not finite: the group answers NaN
    if (lane == 0) {
      scales[i] = ST(s);
      if (zeros != nullptr) zeros[i] = (uint8_t)z;
    }
    for (int k = k0 + 2 * lane; k < k1; k += 64) {
      auto code = [&](int kk) -> int {
        if (kk >= k1 || bad) return kk >= k1 ? 0 : z;
        return min(15, max(0, __float2int_rn(__fdiv_rn(float(row[kk]), s)) + z));
      };
      codes[n * ldq + (k >> 1)] = (uint8_t)(code(k) | (code(k + 1) << 4));
    }
  }
}

int check_int4(int64_t N, int64_t K, int64_t group, int32_t scale_dtype) {
  if (N < 0 || K <= 0) return fail_fmt(SX_ERR_INVALID, "4-bit weights need N >= 0 and K >= 1");
  if (N > 0x40000000LL || K > 0x20000000LL) return fail_fmt(SX_ERR_INVALID, "N exceeds 2^30 or K 2^29");
  if (group <= 0 || group % 32 != 0 || group > 0x20000000LL)
    return fail_fmt(SX_ERR_INVALID, "group must be a positive multiple of 32 and at most 2^29, got %lld", (long long)group);
  if (scale_dtype != SYMPLEX_DT_F32 && scale_dtype != SYMPLEX_DT_BF16)
    return fail_fmt(SX_ERR_INVALID, "scale_dtype %d not supported (F32=9, BF16=11)", scale_dtype);
  return SX_OK;
}

bool aligned_to(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
int bytes_of(int32_t dtype) { return dtype == SYMPLEX_DT_F32 ? 4 : 2; }

template <int kGW, int kNB, typename ST, bool kZeros>
int matvec_mma(const Int4Args& a, bool out_bf16, int sms, cudaStream_t stream) {
  auto kern = int4_mma_kernel<kGW, kNB, ST, kZeros>;
  constexpr int GROUPS = MV_K / kGW;
  MvPlan plan{};
  // Warps per row tile: enough warps for the chip's loads in flight (12 a SM), never more than there are steps.
  const long long tiles = (a.N + MV_TILE - 1) / MV_TILE;
  const int steps = (a.K + MV_K - 1) / MV_K;
  while (plan.kw_log2 < 3 && (2 << plan.kw_log2) <= steps && (tiles << plan.kw_log2) < sms * 12LL) ++plan.kw_log2;
  const int round = MV_AHEAD << plan.kw_log2;
  const int rows = std::min(a.M, 8 * kNB) + 1;
  auto bytes = [&](int n) { return (size_t)rows * (n * (MV_K / 8) + MvPad<kGW>) * 16; };
  plan.chunk_steps = (steps + round - 1) / round * round;
  size_t smem = bytes(plan.chunk_steps);
  if (smem > MV_STAGE_BYTES) {  // in chunks of 8 steps (16 where 8 warps share a tile), two buffers
    plan.chunk_steps = std::max(8, round);
    smem = 2 * bytes(plan.chunk_steps);
  }
  plan.pitch = plan.chunk_steps * (MV_K / 8) + MvPad<kGW>;
  plan.a_vec = a.lda % 8 == 0 && reinterpret_cast<uintptr_t>(a.A) % 16 == 0;
  plan.s_vec = a.group == kGW && a.groups % GROUPS == 0 && reinterpret_cast<uintptr_t>(a.scales) % (GROUPS * sizeof(ST)) == 0 &&
               reinterpret_cast<uintptr_t>(a.zeros) % GROUPS == 0;
  plan.out_bf16 = out_bf16 ? 1 : 0;
  SX_ENSURE_DYN_SMEM(kern, 160 * 1024);
  const int rows_cta = (MV_WARPS >> plan.kw_log2) * MV_TILE;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((a.N + rows_cta - 1) / rows_cta), (unsigned)((a.M + 8 * kNB - 1) / (8 * kNB)), 1);
  cfg.blockDim = dim3(MV_WARPS * 32, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a, plan);
  if (e != cudaSuccess) return launch_failed(e, "4-bit product launch failed");
  count_launches(1);
  return SX_OK;
}

template <int kGW, typename ST>
int matvec_gw(const Int4Args& a, bool out_bf16, int sms, cudaStream_t stream) {
  if (a.M <= 8)
    return a.zeros ? matvec_mma<kGW, 1, ST, true>(a, out_bf16, sms, stream) : matvec_mma<kGW, 1, ST, false>(a, out_bf16, sms, stream);
  return a.zeros ? matvec_mma<kGW, 2, ST, true>(a, out_bf16, sms, stream) : matvec_mma<kGW, 2, ST, false>(a, out_bf16, sms, stream);
}

template <typename ST>
int matvec(const Int4Args& a, bool out_bf16, int sms, cudaStream_t stream) {
  // The widest load whose lanes' shares stay inside one group, as far as the rows' alignment allows.
  const uintptr_t at = reinterpret_cast<uintptr_t>(a.codes) | (uintptr_t)a.ldq;
  if (a.K % 32 == 0 && at % 4 == 0 && (long long)a.N * a.groups < (1ll << 32)) {
    if (a.group % 128 == 0 && at % 16 == 0) return matvec_gw<128, ST>(a, out_bf16, sms, stream);
    if (a.group % 64 == 0 && at % 8 == 0) return matvec_gw<64, ST>(a, out_bf16, sms, stream);
    return matvec_gw<32, ST>(a, out_bf16, sms, stream);
  }
  const cudaError_t e = out_bf16 ? launch_kernel_ex(int4_matvec_any_kernel<ST, __nv_bfloat16>, (unsigned)((a.N + 7) / 8), 256, 0, stream, 1,
                                                    pdl_enabled(), a)
                                 : launch_kernel_ex(int4_matvec_any_kernel<ST, float>, (unsigned)((a.N + 7) / 8), 256, 0, stream, 1,
                                                    pdl_enabled(), a);
  if (e != cudaSuccess) return launch_failed(e, "4-bit product launch failed");
  count_launches(1);
  return SX_OK;
}

template <typename T, typename ST>
int quantize(const void* W, uint8_t* codes, void* scales, uint8_t* zeros, int64_t N, int64_t K, int64_t group, int64_t ldw, int sms,
             cudaStream_t stream) {
  const long long groups = (K + group - 1) / group;
  const unsigned grid = (unsigned)std::min<long long>((N * groups + 7) / 8, (long long)sms * 64);
  cudaError_t e = launch_kernel_ex(int4_quantize_kernel<T, ST>, grid, 256, 0, stream, 1, pdl_enabled(), static_cast<const T*>(W),
                                   codes, static_cast<ST*>(scales), zeros, (long long)N, (int)K, (int)group, (int)groups,
                                   (long long)ldw);
  if (e != cudaSuccess) return launch_failed(e, "4-bit quantiser launch failed");
  count_launches(1);
  return SX_OK;
}

}  // namespace
}  // namespace sx

using namespace sx;

extern "C" {

int symplex_b200_int4_matvec(const void* A, const uint8_t* codes, const void* scales, const uint8_t* zeros,
                             const float* bias, void* C, int64_t M, int64_t N, int64_t K, int64_t group, int64_t lda,
                             int64_t ldq, int64_t ldc, int32_t scale_dtype, int32_t out_dtype, int32_t activation,
                             void* stream) {
  int rc = check_int4(N, K, group, scale_dtype);
  if (rc != SX_OK) return rc;
  if (M < 0 || M > SYMPLEX_B200_INT4_MAX_M)
    return fail_fmt(SX_ERR_INVALID, "M must be in 0..%d, got %lld", SYMPLEX_B200_INT4_MAX_M, (long long)M);
  if (out_dtype != SYMPLEX_DT_F32 && out_dtype != SYMPLEX_DT_BF16)
    return fail_fmt(SX_ERR_INVALID, "out_dtype %d not supported (F32=9, BF16=11)", out_dtype);
  if (activation < SYMPLEX_ACT_NONE || activation > SYMPLEX_ACT_SILU)
    return fail_fmt(SX_ERR_INVALID, "activation %d not supported", activation);
  Int4Args a{};
  a.M = (int)M; a.N = (int)N; a.K = (int)K;
  a.group = (int)group;
  a.groups = (int)((K + group - 1) / group);
  a.group_log2 = (group & (group - 1)) == 0 ? __builtin_ctzll((unsigned long long)group) : -1;
  a.lda = lda ? lda : K;
  a.ldq = ldq ? ldq : (K + 1) / 2;
  a.ldc = ldc ? ldc : N;
  if (a.lda < K || a.ldq < (K + 1) / 2 || a.ldc < N) return fail_fmt(SX_ERR_INVALID, "leading dimension too small");
  if (M == 0 || N == 0) return SX_OK;
  if (A == nullptr || codes == nullptr || scales == nullptr || C == nullptr) return fail_fmt(SX_ERR_INVALID, "null pointer");
  if (!aligned_to(A, 2) || !aligned_to(scales, bytes_of(scale_dtype)) || !aligned_to(C, bytes_of(out_dtype)) || !aligned_to(bias, 4))
    return fail_fmt(SX_ERR_INVALID, "a pointer is not aligned to its element type");
  a.A = static_cast<const __nv_bfloat16*>(A);
  a.codes = codes;
  a.scales = scales;
  a.zeros = zeros;
  a.bias = bias;
  a.C = C;
  a.act = activation;
  int sms = 0;
  if ((rc = current_device_sms(&sms)) != SX_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool out_bf16 = out_dtype == SYMPLEX_DT_BF16;
  return scale_dtype == SYMPLEX_DT_F32 ? matvec<float>(a, out_bf16, sms, st) : matvec<__nv_bfloat16>(a, out_bf16, sms, st);
}

int symplex_b200_int4_quantize(const void* W, uint8_t* codes, void* scales, uint8_t* zeros, int64_t N, int64_t K,
                               int64_t group, int64_t ldw, int32_t dtype, int32_t scale_dtype, void* stream) {
  int rc = check_int4(N, K, group, scale_dtype);
  if (rc != SX_OK) return rc;
  if (dtype != SYMPLEX_DT_F32 && dtype != SYMPLEX_DT_BF16)
    return fail_fmt(SX_ERR_INVALID, "dtype %d not supported (F32=9, BF16=11)", dtype);
  if (ldw == 0) ldw = K;
  if (ldw < K) return fail_fmt(SX_ERR_INVALID, "leading dimension too small");
  if (N == 0) return SX_OK;
  if (W == nullptr || codes == nullptr || scales == nullptr) return fail_fmt(SX_ERR_INVALID, "null pointer");
  if (!aligned_to(W, bytes_of(dtype)) || !aligned_to(scales, bytes_of(scale_dtype)))
    return fail_fmt(SX_ERR_INVALID, "a pointer is not aligned to its element type");
  int sms = 0;
  if ((rc = current_device_sms(&sms)) != SX_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == SYMPLEX_DT_F32)
    return scale_dtype == SYMPLEX_DT_F32 ? quantize<float, float>(W, codes, scales, zeros, N, K, group, ldw, sms, st)
                                         : quantize<float, __nv_bfloat16>(W, codes, scales, zeros, N, K, group, ldw, sms, st);
  return scale_dtype == SYMPLEX_DT_F32 ? quantize<__nv_bfloat16, float>(W, codes, scales, zeros, N, K, group, ldw, sms, st)
                                       : quantize<__nv_bfloat16, __nv_bfloat16>(W, codes, scales, zeros, N, K, group, ldw, sms, st);
}

}  // extern "C"
