// Products of a few rows with 4-bit weights that carry a scale (and a zero) per group of consecutive k:
//
//   C[m][n] = act(sum_g scale[n][g] * sum_{k in g} (code[n][k] - zero[n][g]) * A[m][k] + bias[n])
//
// Bound by HBM: N K / 2 bytes of codes, read once for every 16 rows of A.
//
// int4_mma_kernel: the rows of W are the M side of mma.sync m16n8k16, the rows of A (up to 8 per fragment) its N side. A code less
// its zero becomes bf16 exactly (dequant8 below), so the products are exact and each group's sum is scaled once, in fp32. Which k a
// fragment slot stands for is free as long as both operands agree: a lane takes 8 consecutive k of its row (one 32-bit word), whose
// nibbles j and j + 4 fall into the halves of one register (pairs (k0,k4), (k1,k5), ...), and A is laid out in the same pairs.
// 4-bit products are far below what even the warp-level tensor path delivers, so the tcgen05 path has nothing to add here: what has to
// be fast is the dequantisation, 9 instructions for 8 codes.
#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>

#include "../../include/symplex_b200.h"
#include "byte_rows.h"
#include "epilogue.cuh"
#include "host_api.h"
#include "sm100_ptx.cuh"

namespace sx {
namespace {

// One value of the activation set with the accurate device functions.
__device__ __forceinline__ float activate(float x, int act) {
  switch (act) {
    case ACT_RELU: return x > 0.0f || x != x ? x : 0.0f;  // a NaN stays one (fmaxf would answer 0)
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
constexpr int MV_WARPS = 16;
constexpr int MV_TILE = 32;  // rows of W per tile: two m16 tiles share every fragment of A
constexpr int MV_K = 128;    // k of one step
constexpr int MV_RING = 2;   // steps of codes in flight per warp, 2 KB each: 64 KB an SM (three steps: within 3 %, but 32 KB less for A)
constexpr int MV_STEP_BYTES = MV_TILE * MV_K / 2;
constexpr int MV_RING_BYTES = MV_WARPS * MV_RING * MV_STEP_BYTES;
constexpr int MV_SMEM = 227 * 1024;
constexpr int MV_CLUSTER_MOST = 8;
constexpr int MV_CLUSTER_KW = 1;  // log2 of the fewest warps on a tile in a cluster (16 x 28672 x 8192 in groups of 128: 56 us, 62 with 2)

// 16 bytes global -> shared, past L1; `bytes` 0 writes zeros without reading.
__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kN>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kN) : "memory");
}
// The warps of one of `groups` groups (1, 2, 4 or 8: barriers `groups` to 2 groups - 1, so that no barrier ever has two sizes).
__device__ __forceinline__ void group_barrier(int group, int groups) {
  asm volatile("bar.sync %0, %1;" ::"r"(groups + group), "r"(32 * MV_WARPS / groups) : "memory");
}
__device__ __forceinline__ void cluster_arrive() {
  __syncwarp();  // both barriers are the whole warp's
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 ld_cluster(uint32_t addr, uint32_t rank) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(mapa_u32(addr, rank)) : "memory");
  return v;
}
__device__ __forceinline__ void add(float4& a, const float4& b) {
  a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 r = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&r);
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
__device__ __forceinline__ uint32_t fma_bf16x2(uint32_t a, uint32_t b, uint32_t c) {
  const __nv_bfloat162 r = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b),
                                   *reinterpret_cast<const __nv_bfloat162*>(&c));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// Eight codes -> four registers (k0,k4), (k1,k5), (k2,k6), (k3,k7) of code - zero, the second and fourth a quarter of it.
//   0x430q is 128 + q; less zero2 = 128 + zero.
//   0x00q0 is 16 q 2^-133 (subnormal numbers and the first binade are one run of equal steps), times 2^127 a quarter of q; plus
//   quarter2 = -zero / 4. All exact. One shift for both pairs of a kind, where the first form alone takes three
// (16 x 28672 x 8192 in groups of 128: 51.7 us, 54.9 with the first form).
// The mask and the exponent are registers: one three-input operation each, where two immediates would take two.
__device__ __forceinline__ void dequant8(uint32_t w, uint32_t zero2, uint32_t quarter2, uint32_t mask, uint32_t base, uint32_t (&out)[4]) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    uint32_t v;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(v) : "r"(w), "r"(mask), "r"(base));  // (w & mask) | base
    out[2 * j] = sub_bf16x2(v, zero2);
    out[2 * j + 1] = fma_bf16x2(w & 0x00f000f0u, 0x7f007f00u, quarter2);
    w >>= 8;
  }
}

// The scales (and zeros) of one step of 128 k for a lane's four rows (g, g + 8, g + 16, g + 24), packed as they lie in memory.
// kGW = 128, 64 or 32 is how many k share a scale within a step.
template <int kGW, typename ST, bool kZeros>
struct MvScales {
  static constexpr int GROUPS = MV_K / kGW;
  static constexpr int SCALE_WORDS = (GROUPS * int(sizeof(ST)) + 3) / 4;
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

  // srow: the rows' first groups, k0: first k of the step; s_vec: its groups are GROUPS whole scales in a row, aligned.
  __device__ __forceinline__ void load(const Int4Args& p, const uint32_t (&srow)[4], int k0, int s_vec) {
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

struct MvPlan {
  int tiles;
  int kw_log2;     // warps that share a tile, each with every kw-th step; MV_WARPS / kw tiles are worked on at a time
  int cluster;     // CTAs that share tiles, each with `steps` of their steps
  int steps;
  int rows;        // rows of A of a CTA
  int pitch;       // 16-byte blocks from one staged row of A to the next
  int a_vec, s_vec, c_vec, out_bf16;
};

// A in shared memory: rows of 16-byte blocks of 8 k, each block as the pairs the dequantised words have, (k0,k4) (k1,k5) (k2,k6)
// (k3,k7); block b of a row stands at b ^ ((b >> 3) & 1), and rows are MvPad blocks longer than their k: the eight lanes of a
// quarter warp (two rows, four shares of a group) then read eight different bank groups.
template <int kGW> constexpr int MvPad = kGW == 128 ? 2 : kGW == 64 ? 1 : 4;

// Even k at a quarter, as the odd ones' codes are; a sum's factor of 4 is put back at its end. Exact but for magnitudes below 2^-124.
__device__ __forceinline__ uint32_t quarter(uint32_t pair) { return fma_bf16x2(pair, 0x3e803e80u, 0x80008000u); }
__device__ __forceinline__ uint4 pairs_of(const uint4& x) {
  return make_uint4(quarter(__byte_perm(x.x, x.z, 0x5410)), __byte_perm(x.x, x.z, 0x7632), quarter(__byte_perm(x.y, x.w, 0x5410)),
                    __byte_perm(x.y, x.w, 0x7632));
}

__device__ __forceinline__ void stage_a(const Int4Args& p, const MvPlan& plan, uint4* to, int m0, int rows, int k0) {
  const int blocks = plan.steps * (MV_K / 8);
  for (int m = 0; m < rows; ++m) {
    const __nv_bfloat16* row = p.A + (long long)(m0 + m) * p.lda + k0;
    for (int b = threadIdx.x; b < blocks; b += MV_WARPS * 32) {
      uint4 x = make_uint4(0, 0, 0, 0);
      if (k0 + 8 * b < p.K) {  // K is a multiple of 8: a block is inside or outside
        if (plan.a_vec) {
          x = __ldg(reinterpret_cast<const uint4*>(row + 8 * b));
        } else {
          const uint16_t* u = reinterpret_cast<const uint16_t*>(row + 8 * b);
          x.x = u[0] | (uint32_t(u[1]) << 16);
          x.y = u[2] | (uint32_t(u[3]) << 16);
          x.z = u[4] | (uint32_t(u[5]) << 16);
          x.w = u[6] | (uint32_t(u[7]) << 16);
        }
      }
      to[m * plan.pitch + (b ^ ((b >> 3) & 1))] = pairs_of(x);
    }
  }
}

// Work of a CTA: its tiles t0 .. t1 in rounds of MV_WARPS / kw tiles; where half of them or fewer are left for the last round, 2 kw
// or more warps share each. The warps' sums of a tile are joined in shared memory.
//
// Measured (16 x 28672 x 8192, groups of 64 with zeros): 64 us, 2.0 TB/s; 1 x 28672 x 8192, groups of 128: 31 us, 3.9 TB/s. HBM would
// take 20 and 18: the ALU, the shared-memory pipe and the issue of instructions are each about half busy, with the four warps a
// scheduler that 128 registers leave.
//
// Where all of A does not fit into shared memory, a cluster of 2, 4 or 8 CTAs shares its tiles: each has a stretch of k, with that
// stretch of A, for all of them. A round's sums stay in the CTA that made them until the next round is done, when every CTA of the
// cluster has arrived with its own; then each of them takes a share of the outputs and adds up what the others hold.
//
// Where a cluster of 8 does not hold A either, fewer rows of A are taken in a pass over W. (A in slabs that every CTA replaces as it
// goes through k: 81 us for the first case above, the barriers between slabs and the copies of A.)
template <int kGW, int kNB, typename ST, bool kZeros>
__global__ void __launch_bounds__(MV_WARPS * 32, 1)
int4_mma_kernel(const Int4Args p, const MvPlan plan) {
  using Scales = MvScales<kGW, ST, kZeros>;
  constexpr int GROUPS = Scales::GROUPS;
  constexpr int WPG = kGW / 32;  // words of a lane per group of a step
  constexpr int RED_PITCH = MV_TILE + 4;  // floats from one row of A to the next: the lanes of a store meet every bank once
  constexpr int RED_WARP = 8 * kNB * RED_PITCH;
  extern __shared__ uint4 dyn_smem[];
  constexpr int ROUND_SUMS = (MV_WARPS >> MV_CLUSTER_KW) * MV_TILE * 8 * kNB;  // of a CTA in a cluster
  float* const red = reinterpret_cast<float*>(dyn_smem + MV_RING_BYTES / 16);  // [warp][row of A][row of the tile]
  float* const sums = red + MV_WARPS * RED_WARP;                               // cluster: [round mod 2][tile][row of A][row of the tile]
  uint4* const a_smem = reinterpret_cast<uint4*>(sums + (plan.cluster > 1 ? 2 * ROUND_SUMS : 0));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int rank = plan.cluster > 1 ? (int)cluster_ctarank() : 0;
  const int m0 = blockIdx.y * plan.rows;
  const int m_here = min(plan.rows, p.M - m0);
  const int first = rank * plan.steps;  // this CTA's steps
  const int steps = min((p.K + MV_K - 1) / MV_K, first + plan.steps);
  const int crowd = blockIdx.x / plan.cluster, crowds = gridDim.x / plan.cluster;
  const int t0 = (int)((long long)plan.tiles * crowd / crowds), t1 = (int)((long long)plan.tiles * (crowd + 1) / crowds);
  // log2 of the warps on each tile in the round that begins at tile b < t1
  auto round_kw = [&](int b) {
    const int left = t1 - b, base = plan.kw_log2;
    if (left >= MV_WARPS >> base) return base;
    return 4 - (32 - __clz(left - 1));  // the most warps that leave one for every tile
  };

  // The warp's ring of codes: a step is 32 rows of 64 bytes, 16-byte block q of a row at q ^ f with f = the bits of row / 2 in reverse,
  // so that every read below (16, 8 or 4 bytes a lane) meets each bank once.
  const uint32_t ring = smem_u32(dyn_smem) + warp * (MV_RING * MV_STEP_BYTES);
  const uint32_t f = ((g >> 2) & 1) | (g & 2);  // row / 2 = (g >> 1) mod 4 for all four rows
  const uint32_t put = ring + g * 64 + ((t ^ f) << 4);

  // This warp's next tile and first step in the rounds from the one at `round` (moved on to it) on; tile t1: none.
  auto after = [&](int& round, int& tile, int& step) {
    for (; round < t1;) {
      const int kwl = round_kw(round);
      tile = round + (warp >> kwl);
      step = first + (warp & ((1 << kwl) - 1));
      if (tile < t1 && step < steps) return kwl;
      round += MV_WARPS >> kwl;
    }
    tile = t1;
    return 0;
  };
  // The step whose codes are fetched next runs ahead of the one being multiplied by the ring.
  int far_round = t0, far_kw = 0, far_tile = 0, far_step = 0;
  const uint8_t* row[4];  // this lane's share of the fetched tile's rows
  auto far_rows = [&]() {
    far_kw = after(far_round, far_tile, far_step);
    if (far_tile >= t1) return;
#pragma unroll
    for (int r = 0; r < 4; ++r)  // rows past the end repeat the last one and are not written
      row[r] = p.codes + (long long)min(far_tile * MV_TILE + g + 8 * r, p.N - 1) * p.ldq + 16 * t;
  };
  auto fetch = [&](uint32_t slot) {
    if (far_tile < t1) {
      const int bytes = far_step * MV_K + 32 * t < p.K ? 16 : 0;  // K is a multiple of 32: a block is inside or outside
      const long long at = bytes ? (long long)far_step * (MV_K / 2) : 0;
#pragma unroll
      for (int r = 0; r < 4; ++r) cp_async_16(put + slot + r * 512, row[r] + at, bytes);
      far_step += 1 << far_kw;
      if (far_step >= steps) {
        far_round += MV_WARPS >> far_kw;
        far_rows();
      }
    }
    cp_async_commit();
  };
  // So do the scales, by one step.
  uint32_t srow[4];
  auto scale_rows = [&](int tile) {
#pragma unroll
    for (int r = 0; r < 4; ++r) srow[r] = (uint32_t)min(tile * MV_TILE + g + 8 * r, p.N - 1) * (uint32_t)p.groups;  // host: N * groups < 2^32
  };

  pdl_launch_dependents();
  pdl_wait_prior_grids();
  far_rows();
  Scales sc;
  if (far_tile < t1) {
    scale_rows(far_tile);
    sc.load(p, srow, far_step * MV_K, plan.s_vec);
  }
#pragma unroll
  for (int i = 0; i < MV_RING; ++i) fetch(i * MV_STEP_BYTES);
  stage_a(p, plan, a_smem, m0, m_here, first * MV_K);
  __syncthreads();

  auto write = [&](int tile, int m, int r, float4 sum) {  // four outputs of row m, from row r of the tile on
    const int n = tile * MV_TILE + r;
    float v[4] = {sum.x, sum.y, sum.z, sum.w};
    const long long at = (m0 + m) * p.ldc + n;
    const bool all = n + 4 <= p.N;
    if (p.bias != nullptr) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (all || n + i < p.N) v[i] += p.bias[n + i];
    }
    if (p.act != ACT_NONE) {
#pragma unroll 1
      for (int i = 0; i < 4; ++i) v[i] = activate(v[i], p.act);
    }
    if (all && plan.c_vec) {
      if (plan.out_bf16) *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.C) + at) = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
      else *reinterpret_cast<float4*>(static_cast<float*>(p.C) + at) = make_float4(v[0], v[1], v[2], v[3]);
      return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (n + i >= p.N) break;
      if (plan.out_bf16) static_cast<__nv_bfloat16*>(p.C)[at + i] = __nv_bfloat16(v[i]);
      else static_cast<float*>(p.C)[at + i] = v[i];
    }
  };
  // Cluster: this CTA's share of the outputs of a round, once every CTA has arrived with its sums.
  int held_tile = -1, held_n = 0, held_buf = 0;
  auto write_held = [&]() {
    cluster_wait();
    for (int e = rank * (MV_WARPS * 32) + threadIdx.x; e < held_n * (8 * kNB) * (MV_TILE / 4); e += plan.cluster * MV_WARPS * 32) {
      const int m = e / (MV_TILE / 4) % (8 * kNB);
      if (m >= m_here) continue;
      const uint32_t at = smem_u32(sums + held_buf * ROUND_SUMS + 4 * e);
      float4 v = ld_cluster(at, 0);
      for (int i = 1; i < plan.cluster; ++i) add(v, ld_cluster(at, i));
      write(held_tile + e / (8 * kNB * (MV_TILE / 4)), m, 4 * e % MV_TILE, v);
    }
  };

  // Where a lane finds its blocks of A in a step: two bases, for the even and odd ones among its words, because of the exchange of
  // neighbours in every other eight blocks. Rows of A that do not exist repeat the last one; their sums are not written.
  int a_base[kNB][2];
#pragma unroll
  for (int nb = 0; nb < kNB; ++nb)
#pragma unroll
    for (int i = 0; i < 2; ++i)
      a_base[nb][i] = min(8 * nb + g, m_here - 1) * plan.pitch + (kGW == 128 ? 4 * t + (i ^ (t >> 1)) : kGW == 64 ? 2 * t + i : t ^ i);
  uint32_t mask = 0x000f000fu, base128 = 0x43004300u;
  asm volatile("" : "+r"(mask), "+r"(base128));
  uint32_t slot = 0;
  for (int b0 = t0, kwl; b0 < t1; b0 += MV_WARPS >> kwl) {
    kwl = round_kw(b0);
    const int kw = 1 << kwl, RG = MV_WARPS >> kwl;
    const int mk = warp & (kw - 1), rg = warp >> kwl;
    const int tile = b0 + rg;
    float acc[kNB][2][4] = {};
    if (tile < t1) {
      const uint4* a0 = a_smem + mk * (MV_K / 8);
      for (int v = first + mk; v < steps; v += kw, a0 += kw * (MV_K / 8)) {
        cp_async_wait<MV_RING - 1>();
        __syncwarp();
        uint32_t codes[4][4];
        const uint32_t base = ring + slot + g * 64;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if constexpr (kGW == 128) {
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(codes[r][0]), "=r"(codes[r][1]), "=r"(codes[r][2]), "=r"(codes[r][3])
                         : "r"(base + ((t ^ f) << 4) + r * 512));
          } else if constexpr (kGW == 64) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
              asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];"
                           : "=r"(codes[r][2 * h]), "=r"(codes[r][2 * h + 1])
                           : "r"(base + ((((2 * h) | (t >> 1)) ^ f) << 4) + ((t & 1) << 3) + r * 512));
          } else {
#pragma unroll
            for (int h = 0; h < 4; ++h)
              asm volatile("ld.shared.u32 %0, [%1];" : "=r"(codes[r][h]) : "r"(base + ((h ^ f) << 4) + (t << 2) + r * 512));
          }
        }
        const Scales cur = sc;
        if (v + kw < steps) {
          sc.load(p, srow, (v + kw) * MV_K, plan.s_vec);
        } else {
          int round2 = b0 + RG, tile2, step2;
          after(round2, tile2, step2);
          if (tile2 < t1) {
            scale_rows(tile2);
            sc.load(p, srow, step2 * MV_K, plan.s_vec);
          }
        }
#pragma unroll
        for (int j = 0; j < GROUPS; ++j) {
          float part[kNB][2][4];
          uint32_t zero2[4], quarter2[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            zero2[r] = cur.zero2(r, j);
            quarter2[r] = kZeros ? fma_bf16x2(zero2[r], 0xbe80be80u, 0x42004200u) : 0xc000c000u;  // 32 - (128 + zero) / 4
          }
#pragma unroll
          for (int i = 0; i < WPG; ++i) {
            const int w = j * WPG + i;
            uint4 x[kNB];
#pragma unroll
            for (int nb = 0; nb < kNB; ++nb) {
              if constexpr (kGW == 128) x[nb] = a0[a_base[nb][i & 1] + (i & 2)];
              else if constexpr (kGW == 64) x[nb] = a0[a_base[nb][i ^ j] + 8 * j];
              else x[nb] = a0[a_base[nb][j >> 1] + 4 * j];
            }
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
              uint32_t lo[4], hi[4];  // rows g and g + 8 of this m16 tile
              dequant8(codes[2 * mt][w], zero2[2 * mt], quarter2[2 * mt], mask, base128, lo);
              dequant8(codes[2 * mt + 1][w], zero2[2 * mt + 1], quarter2[2 * mt + 1], mask, base128, hi);
#pragma unroll
              for (int nb = 0; nb < kNB; ++nb) {
                if (i == 0) mma_bf16_zero(part[nb][mt], lo[0], hi[0], lo[1], hi[1], x[nb].x, x[nb].y);
                else mma_bf16(part[nb][mt], lo[0], hi[0], lo[1], hi[1], x[nb].x, x[nb].y);
                mma_bf16(part[nb][mt], lo[2], hi[2], lo[3], hi[3], x[nb].z, x[nb].w);
              }
            }
          }
          // A group that lies past K whole has sums of 0 and repeats a scale, which may be anything: 0 * inf must not count.
          if (GROUPS == 1 || v * MV_K + j * kGW < p.K) {
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
              const float sc0 = cur.scale(2 * mt, j), sc1 = cur.scale(2 * mt + 1, j);
#pragma unroll
              for (int nb = 0; nb < kNB; ++nb) {
                acc[nb][mt][0] = fmaf(sc0, part[nb][mt][0], acc[nb][mt][0]);
                acc[nb][mt][1] = fmaf(sc0, part[nb][mt][1], acc[nb][mt][1]);
                acc[nb][mt][2] = fmaf(sc1, part[nb][mt][2], acc[nb][mt][2]);
                acc[nb][mt][3] = fmaf(sc1, part[nb][mt][3], acc[nb][mt][3]);
              }
            }
          }
        }
        __syncwarp();  // every lane has its words: the slot takes the step after the ring's last
        fetch(slot);
        slot = slot == (MV_RING - 1) * MV_STEP_BYTES ? 0 : slot + MV_STEP_BYTES;
      }
    }
    // The tile's sums over the warps that share it, always in the order of the warps.
    if (plan.cluster > 1 && held_tile >= 0) write_held();  // and now nobody needs the sums of the round before that any more
    if (tile < t1) {
#pragma unroll
      for (int nb = 0; nb < kNB; ++nb)
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            red[warp * RED_WARP + (8 * nb + 2 * t + (i & 1)) * RED_PITCH + 16 * mt + g + 8 * (i >> 1)] = acc[nb][mt][i];
      if (kw == 1) __syncwarp();
      else group_barrier(rg, RG);
      const float* const from = red + rg * kw * RED_WARP;
      for (int e = mk * 32 + lane; e < m_here * (MV_TILE / 4); e += 32 * kw) {
        const int m = e / (MV_TILE / 4), r = 4 * e % MV_TILE;
        const float* at = from + m * RED_PITCH + r;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (kw >= 4) {
          for (int i = 0; i < kw; i += 4) {
#pragma unroll
            for (int k = 0; k < 4; ++k) add(v, *reinterpret_cast<const float4*>(at + (i + k) * RED_WARP));
          }
        } else {
          for (int i = 0; i < kw; ++i) add(v, *reinterpret_cast<const float4*>(at + i * RED_WARP));
        }
        v.x *= 4.0f; v.y *= 4.0f; v.z *= 4.0f; v.w *= 4.0f;
        if (plan.cluster > 1) *reinterpret_cast<float4*>(sums + (held_buf ^ 1) * ROUND_SUMS + (rg * 8 * kNB + m) * MV_TILE + r) = v;
        else write(tile, m, r, v);
      }
      if (kw == 1) __syncwarp();  // red is free again
      else group_barrier(rg, RG);
    }
    if (plan.cluster > 1) {
      held_tile = b0;
      held_n = min(RG, t1 - b0);
      held_buf ^= 1;
      cluster_arrive();
    }
  }
  if (plan.cluster > 1) {
    if (held_tile >= 0) write_held();
    cluster_arrive();  // no CTA leaves while its sums are being read
    cluster_wait();
  }
  cp_async_wait<0>();
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

// Shared memory of a CTA for `rows` rows of A and `steps` steps, alone or in a cluster.
template <int kGW>
size_t mv_smem(int rows, int steps, bool cluster) {
  const int nb = rows > 8 ? 2 : 1;
  const size_t joined = (size_t)MV_WARPS * (MV_TILE + 4) * 8 * nb * 4, held = cluster ? 2 * (MV_WARPS >> MV_CLUSTER_KW) * MV_TILE * 8 * nb * 4 : 0;
  return MV_RING_BYTES + joined + held + (size_t)rows * (steps * (MV_K / 8) + MvPad<kGW>) * 16;
}
// The smallest cluster whose CTAs hold `rows` rows of A between them; 0: none does.
template <int kGW>
int mv_cluster(int rows, int steps) {
  for (int c = 1; c <= MV_CLUSTER_MOST; c *= 2)
    if (mv_smem<kGW>(rows, (steps + c - 1) / c, c > 1) <= MV_SMEM) return c;
  return 0;
}

template <int kGW, int kNB, typename ST, bool kZeros>
int matvec_mma(const Int4Args& a, int rows, int cluster, bool out_bf16, int sms, cudaStream_t stream) {
  auto kern = int4_mma_kernel<kGW, kNB, ST, kZeros>;
  constexpr int GROUPS = MV_K / kGW;
  const int mblocks = (a.M + rows - 1) / rows, steps = (a.K + MV_K - 1) / MV_K;
  SX_ENSURE_DYN_SMEM(kern, MV_SMEM);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  MvPlan plan{};
  plan.tiles = (a.N + MV_TILE - 1) / MV_TILE;
  plan.rows = rows;
  plan.cluster = cluster;
  plan.steps = (steps + cluster - 1) / cluster;
  int crowds = std::max(1, sms / mblocks / cluster);
  plan.pitch = plan.steps * (MV_K / 8) + MvPad<kGW>;
  plan.a_vec = a.lda % 8 == 0 && reinterpret_cast<uintptr_t>(a.A) % 16 == 0;
  plan.s_vec = a.group == kGW && a.groups % GROUPS == 0 && reinterpret_cast<uintptr_t>(a.scales) % (GROUPS * sizeof(ST)) == 0 &&
               reinterpret_cast<uintptr_t>(a.zeros) % GROUPS == 0;
  plan.out_bf16 = out_bf16 ? 1 : 0;
  plan.c_vec = a.ldc % 4 == 0 && reinterpret_cast<uintptr_t>(a.C) % (out_bf16 ? 8 : 16) == 0;
  cfg.blockDim = dim3(MV_WARPS * 32, 1, 1);
  cfg.dynamicSmemBytes = mv_smem<kGW>(rows, plan.steps, cluster > 1);
  cfg.stream = stream;
  cfg.attrs = attr;
  if (plan.cluster > 1) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = plan.cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.numAttrs = 1;
    // A processing cluster of the GPU may have SMs left over that make no whole cluster; each device has its own.
    constexpr int DEVICES = 16;  // current_device_sms takes no more
    static std::atomic<int> resident[DEVICES][MV_CLUSTER_MOST + 1];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || dev < 0 || dev >= DEVICES) return launch_failed(e, "device of a 4-bit product");
    int n = resident[dev][plan.cluster].load(std::memory_order_relaxed);
    if (n == 0) {
      cfg.gridDim = dim3(plan.cluster, 1, 1);
      cudaLaunchConfig_t most = cfg;
      most.dynamicSmemBytes = MV_SMEM;
      e = cudaOccupancyMaxActiveClusters(&n, kern, &most);
      if (e != cudaSuccess || n <= 0) return launch_failed(e, "cluster size not supported");
      resident[dev][plan.cluster].store(n, std::memory_order_relaxed);
    }
    crowds = std::max(1, std::min(crowds, n / mblocks));
  }
  crowds = std::min(crowds, plan.tiles);
  cfg.gridDim = dim3((unsigned)(crowds * plan.cluster), (unsigned)mblocks, 1);
  // Warps on a tile: those with which the rounds of a CTA (or cluster) take the fewest steps, two counted for joining the sums
  // (5 x 50257 x 2048: 23.0 us with two, 23.2 with four, 30 with 16; 1 x 28672 x 8192: 31 with four, 33 with two).
  const int each = plan.tiles / crowds;
  double least = 1e30;
  for (int kwl = cluster > 1 ? MV_CLUSTER_KW : 0; kwl <= 4; ++kwl) {
    double cost = 0;
    for (int n : {each, each + (plan.tiles % crowds ? 1 : 0)}) {
      const int whole = n / (MV_WARPS >> kwl), left = n % (MV_WARPS >> kwl);
      cost += whole * (double)((plan.steps + (1 << kwl) - 1) / (1 << kwl) + 2);
      if (left > 0) {
        int kw = 1 << kwl;
        while (MV_WARPS / (2 * kw) >= left) kw *= 2;
        cost += (plan.steps + kw - 1) / kw + 2;
      }
    }
    if (cost < least) least = cost, plan.kw_log2 = kwl;
  }
  if (pdl_enabled() && cluster == 1) {  // clusters start in plain stream order (a microsecond of 40 or more)
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
  }
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a, plan);
  if (e != cudaSuccess) return launch_failed(e, "4-bit product launch failed");
  count_launches(1);
  return SX_OK;
}

template <int kGW, typename ST>
int matvec_gw(const Int4Args& a, int rows, int cluster, bool out_bf16, int sms, cudaStream_t stream) {
  if (rows <= 8)
    return a.zeros ? matvec_mma<kGW, 1, ST, true>(a, rows, cluster, out_bf16, sms, stream)
                   : matvec_mma<kGW, 1, ST, false>(a, rows, cluster, out_bf16, sms, stream);
  return a.zeros ? matvec_mma<kGW, 2, ST, true>(a, rows, cluster, out_bf16, sms, stream)
                 : matvec_mma<kGW, 2, ST, false>(a, rows, cluster, out_bf16, sms, stream);
}

template <typename ST>
int matvec(const Int4Args& a, bool out_bf16, int sms, cudaStream_t stream) {
  // The fast path reads rows of codes in 16-byte blocks; which of its forms goes by the group.
  const uintptr_t at = reinterpret_cast<uintptr_t>(a.codes) | (uintptr_t)a.ldq;
  if (a.K % 32 == 0 && at % 16 == 0 && (long long)a.N * a.groups < (1ll << 32)) {
    const int steps = (a.K + MV_K - 1) / MV_K, gw = a.group % 128 == 0 ? 128 : a.group % 64 == 0 ? 64 : 32;
    // Up to 16 rows of A in a pass over W, as even as they go; fewer where even a cluster does not hold them. K is beyond 300000 where not
    // one fits.
    const int passes = (a.M + 15) / 16;
    for (int rows = (a.M + passes - 1) / passes; rows > 0; rows = rows > 8 ? 8 : rows / 2) {
      const int cluster = gw == 128 ? mv_cluster<128>(rows, steps) : gw == 64 ? mv_cluster<64>(rows, steps) : mv_cluster<32>(rows, steps);
      if (cluster == 0) continue;
      if (gw == 128) return matvec_gw<128, ST>(a, rows, cluster, out_bf16, sms, stream);
      if (gw == 64) return matvec_gw<64, ST>(a, rows, cluster, out_bf16, sms, stream);
      return matvec_gw<32, ST>(a, rows, cluster, out_bf16, sms, stream);
    }
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
  const ByteRows out{C, M, N * bytes_of(out_dtype), a.ldc * bytes_of(out_dtype)};
  const long long sums = N * a.groups;
  if (share_bytes(out, {A, M, K * 2, a.lda * 2}) || share_bytes(out, {codes, N, (K + 1) / 2, a.ldq}) ||
      share_bytes(out, one_row(scales, sums * bytes_of(scale_dtype))) || share_bytes(out, one_row(zeros, sums)) || share_bytes(out, one_row(bias, N * 4)))
    return fail_fmt(SX_ERR_INVALID, "C overlaps an operand, which other columns of the product still read");
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
