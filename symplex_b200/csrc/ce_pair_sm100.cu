// Tensor-core kernels of the linear head's loss, bf16: logits on CTA pairs (tcgen05.mma.cta_group::2) that never leave the
// SM, and the two products of the gradient.
//
//   CE_LSE     l = x W^T tile by tile; the epilogue turns each row's stretch of a tile into (largest, sum of exponentials)
//              straight from tensor memory and picks out the target's logit. Nothing of size T x V is written.
//   CE_GRAD    the same product again for a piece of the vocabulary; the epilogue writes G = (exp(l - lse) - 1hot) s in bf16.
//   CE_PROD    dx += G W (A = G as stored) and dW = G^T x (A = G read MN-major, no transpose pass) as ONE list of tiles:
//              both need G alone, their tiles differ in length (n against T k-blocks), and together they fill the pairs of the
//              chip where dx by itself would leave the last wave mostly idle.
//
// Roles, barriers and tile shapes are those of the general pair kernel (gemm_pair_sm100.cu): warp 0 TMA, warp 1 MMA issue (leader CTA
// only), then the epilogue warps; kMB = 1: 256 x 256 tiles with two alternating accumulators, kMB = 2: 512 x 256 tiles. All waits are
// bounded; on a timeout every role unwinds and the status word says so.
//
// What bounds it: the tensor pipe (2 T V H flops forward, 6 T V H backward with the logits computed again).
#include <cuda_bf16.h>

#include <algorithm>

#include "ce_params.h"
#include "ce_tiles.h"
#include "epilogue.cuh"
#include "gemm_params.h"
#include "host_api.h"
#include "options.h"
#include "sm100_ptx.cuh"

namespace sx {
namespace {

enum CeMode : int { CE_LSE = 0, CE_GRAD = 1, CE_PROD = 2 };

// kMB = 1, 2: row blocks of 128 per CTA of a pair. kMB = 0: one CTA by itself, 128 rows.
template <int kMB>
struct CeCfg {
  static constexpr int ROWS = 128 * kMB;  // rows of A per CTA
  static constexpr int BM = 2 * ROWS;
  static constexpr int BN = 256;
  static constexpr int BK = 64;
  static constexpr int A_BYTES = ROWS * 128;
  static constexpr int B_BYTES = 128 * 128;  // this CTA's 128 of the 256 columns
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGES = kMB == 1 ? 6 : 4;
  static constexpr int EPI_WARPS = 4 * kMB;
  static constexpr int TMEM_COLS = 512;
};

// At most 128 tokens. A pair's tile would be filled up to 256 rows with nothing, and its MMAs then take as long as W's rows take to
// arrive (512 cycles for 16 KB per SM, 9 TB/s with no pause): one CTA has half the rows to multiply (1 x 4096 x 65536: 150 us on
// pairs, 94 us alone, 5.7 TB/s; 37 x 1024 x 50257: 32 and 25 us, 26 since the kernels start in plain stream order). Columns of a tile, rows of A that
// are copied and stages are set at launch: the tiles share the vocabulary out evenly, and the stages fill shared memory. The MMA
// reads 128 rows of A from a stage whatever was copied; the rows behind the copied ones are other data, and nobody reads their sums.
template <>
struct CeCfg<0> {
  static constexpr int ROWS = 128;
  static constexpr int BM = 128;
  static constexpr int BN = 256;  // at most
  static constexpr int BK = 64;
  static constexpr int STAGES = 12;  // at most
  static constexpr int EPI_WARPS = 4;
  static constexpr int TMEM_COLS = 512;
};

// One product: tiles of [M, N] over K.
struct CeJob {
  int M, N, K, m_tiles, n_tiles, group_m;
  int chunks, chunk_kb;  // k cut into parts of chunk_kb k-blocks, each a list of tiles of its own (CE_PROD's dx; else 1)
};

struct CeKernelParams {
  CeJob job[2];     // job 1: CE_PROD only
  int first_extra;  // CE_PROD: job-1 tiles given ahead to the pairs that got one job-0 tile fewer
  int* status;
  unsigned long long wait_limit_ns;
  const long long* targets;
  long long v0, V, ignore;
  float2* part;
  float* target_logit;
  unsigned* done;   // CE_LSE: set to 0 for the kernel behind this one
  const float* lse;
  const float* dloss;
  const float* scale;
  int lo;           // CE_GRAD: G's rounding errors are written too, through out1
  int dx_add;       // CE_PROD: job 0 adds to what the accumulators hold
  const float* dx_acc;
  int dx_bf16;      // CE_PROD: job 0 writes bf16 dx (last piece, one chunk), else the fp32 accumulators
  int bn, a_bytes, stages;  // kMB = 0: columns of a tile, bytes of A in a stage, stages
  int tma_out[2];   // outputs written by TMA (16-byte aligned rows), else element by element
  void* out[2];
};

struct CeTile {
  int job, m0, n0, chunk, kb0, kb;  // k-blocks kb0 .. kb0 + kb
};

// The tiles of one pair, in order. CE_LSE / CE_GRAD: every pairs-th tile. CE_PROD: every pairs-th tile of job 0 (dx); the pairs that
// got one fewer of those take `extra` tiles of job 1 (dW) each instead, and the rest of job 1 is dealt out evenly.
template <int kMode, int kMB>
struct CeWork {
  using Cfg = CeCfg<kMB>;
  const CeKernelParams& p;
  int pair, pairs, stage, next, end, stride;

  __host__ __device__ CeWork(const CeKernelParams& p_, int pair_, int pairs_) : p(p_), pair(pair_), pairs(pairs_), stage(0) {
    next = pair;
    end = p.job[0].m_tiles * p.job[0].n_tiles * p.job[0].chunks;
    stride = pairs;
  }
  __host__ __device__ bool get(CeTile* t) {
    if constexpr (kMode == CE_PROD) {
      while (next >= end) {
        const int t0 = p.job[0].m_tiles * p.job[0].n_tiles * p.job[0].chunks, t1 = p.job[1].m_tiles * p.job[1].n_tiles;
        const int full = t0 % pairs;  // pairs 0 .. full-1 have one job-0 tile more
        if (stage == 0) {
          stage = 1;
          next = pair >= full ? pair - full : p.first_extra;
          end = p.first_extra;
          stride = pairs - full;
        } else if (stage == 1) {
          stage = 2;
          next = p.first_extra + pair;
          end = t1;
          stride = pairs;
        } else {
          return false;
        }
      }
    } else if (next >= end) {
      return false;
    }
    const int job = kMode == CE_PROD && stage > 0 ? 1 : 0;
    const CeJob& j = p.job[job];
    const int per_chunk = j.m_tiles * j.n_tiles;
    const int chunk = kMode == CE_PROD ? next / per_chunk : 0;
    const int at = kMode == CE_PROD ? next - chunk * per_chunk : next;
    const int band = j.group_m * j.n_tiles;  // bands of group_m tile rows, column by column: operands of a band stay in L2
    const int g = at / band;
    const int first_m = g * j.group_m;
    const int gsz = j.m_tiles - first_m < j.group_m ? j.m_tiles - first_m : j.group_m;
    const int in_band = at - g * band;
    const int all = (j.K + Cfg::BK - 1) / Cfg::BK;
    t->job = job;
    t->m0 = (first_m + in_band % gsz) * Cfg::BM;
    t->n0 = (in_band / gsz) * (kMB == 0 ? p.bn : Cfg::BN);
    t->chunk = chunk;
    t->kb0 = kMode == CE_PROD ? chunk * j.chunk_kb : 0;
    t->kb = kMode == CE_PROD ? (all - t->kb0 < j.chunk_kb ? all - t->kb0 : j.chunk_kb) : all;
    next += stride;
    return true;
  }
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 16 columns of this warp's 32 rows, a row a lane; waits for them.
__device__ __forceinline__ void tmem_get_32x16(uint32_t taddr, uint32_t (&r)[16]) {
  __syncwarp();
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
               "tcgen05.wait::ld.sync.aligned;"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                 "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(taddr)
               : "memory");
}

// 16-byte chunk `chunk` (of 8) of a lane's row of a 128-byte-swizzled staging tile of 32 rows x 128 bytes, one row per lane (the layout
// of a SWIZZLE_128B tensor map).
__device__ __forceinline__ uint8_t* staged_at(uint8_t* tile, int lane, int chunk) { return tile + lane * 128 + ((chunk ^ (lane & 7)) << 4); }
// 32 values of one row: bf16 fills four chunks from `chunk` on, fp32 all eight.
__device__ __forceinline__ void stage_bf16(const float (&v)[32], uint8_t* tile, int lane, int chunk) {
#pragma unroll
  for (int c = 0; c < 4; ++c) *reinterpret_cast<uint4*>(staged_at(tile, lane, chunk + c)) = EpilogueCtx<__nv_bfloat16>::pack8_bf16(v + 8 * c);
}
__device__ __forceinline__ void stage_f32(const float (&v)[32], uint8_t* tile, int lane) {
#pragma unroll
  for (int c = 0; c < 8; ++c)
    *reinterpret_cast<float4*>(staged_at(tile, lane, c)) = make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
}

// The accumulators round every sum towards 0: a logit loses about 2^-26 of itself for each 16 k, and the loss, which all logits move the
// same way, 2e-10 H of itself (measured: 8e-7 at H = 4096, 1.6e-6 at 8192; with 3000 words, whose loss is smaller, 1.1e-6 and 2.6e-6).
// Where all products of a logit have one sign (a row that is sure of its target) it is 6e-6 at 2048 and 1.5e-5 at 4096 (segments: 1.1e-6).
// kSegments (CE_LSE and CE_GRAD, kMB 0 and 1): k in segments of 512, each from zero into the next accumulator; twice the epilogue warps,
// half of a tile's columns each, add them up in registers with rounded sums. 1e-7 at any H. Both passes of a problem take the same form:
// the target's entry of G is exp(l - lse) - 1, of which an l with the bias beside an lse without it leaves nothing right where 1 - p is
// small (T = 2100, H = 4104, rows of 1 - p = 1e-5 to 1e-3: G off by 3e-4, by 1e-6 in the same form).
template <int kMB, bool kSegments>
constexpr int CE_EPI_WARPS = kSegments ? 8 : CeCfg<kMB>::EPI_WARPS;
// Shared memory: operand stages, then a staging tile of 32 x 128 bytes for each epilogue warp that writes through one.
constexpr int CE_STAGING_BYTES = 32 * 128;
template <int kMode, int kMB, bool kSegments>
__host__ __device__ constexpr int ce_stage_room() {
  if constexpr (kMB > 0) return CeCfg<kMB>::STAGES * CeCfg<kMB>::STAGE_BYTES;
  else return (kMode == CE_GRAD && kSegments ? 192 : 200) * 1024;
}
template <int kMode, int kMB, bool kSegments>
constexpr int CE_DYN_SMEM = ce_stage_room<kMode, kMB, kSegments>() + (kMode == CE_LSE ? 0 : CE_EPI_WARPS<kMB, kSegments> * CE_STAGING_BYTES) + 1024;

template <int kMode, int kMB, bool kSegments>
__global__ void __launch_bounds__(64 + 32 * CE_EPI_WARPS<kMB, kSegments>, 1)
ce_pair_kernel(const __grid_constant__ CUtensorMap tmA0, const __grid_constant__ CUtensorMap tmB0,
               const __grid_constant__ CUtensorMap tmA1, const __grid_constant__ CUtensorMap tmB1,
               const __grid_constant__ CUtensorMap out0, const __grid_constant__ CUtensorMap out1,
               const __grid_constant__ CeKernelParams p) {
  using Cfg = CeCfg<kMB>;
  using Work = CeWork<kMode, kMB>;
  constexpr int BN = Cfg::BN, BK = Cfg::BK;
  constexpr bool kPair = kMB > 0;
  constexpr int kGroup = kPair ? 2 : 1;  // CTAs that share a tile
  int STAGES, STAGE_BYTES, A_BYTES;
  if constexpr (kPair) {
    STAGES = Cfg::STAGES, STAGE_BYTES = Cfg::STAGE_BYTES, A_BYTES = Cfg::A_BYTES;
  } else {
    STAGES = p.stages, A_BYTES = p.a_bytes, STAGE_BYTES = p.a_bytes + p.bn * 128;
  }

  extern __shared__ uint8_t dyn_smem[];
  __shared__ uint64_t full_bar[Cfg::STAGES], empty_bar[Cfg::STAGES], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_base_slot;
  __shared__ int abort_flag;

  uint8_t* tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dyn_smem) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t cta_rank = kPair ? cluster_ctarank() : 0;  // 0 = leader
  const uint64_t wait_ns = p.wait_limit_ns;
  const int pair_id = blockIdx.x / kGroup;
  const int num_pairs = gridDim.x / kGroup;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);   // leader: its producer's arrive.expect_tx (bytes of both CTAs)
      mbar_init(&empty_bar[s], 1);  // one tcgen05.commit per use
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], kGroup * CE_EPI_WARPS<kMB, kSegments>);  // every epilogue warp of both CTAs
    }
    abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc<kGroup>(&tmem_base_slot, Cfg::TMEM_COLS);
    tmem_relinquish<kGroup>();
  }
  tc_fence_before_sync();
  __syncwarp();
  if constexpr (kPair) cluster_sync_all();
  else __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = tmem_base_slot;
  if (kMode == CE_LSE && blockIdx.x == 0 && threadIdx.x == 0) *p.done = 0;

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer (both CTAs)
    if (lane == 0) {
      tma_prefetch_desc(&tmA0);
      tma_prefetch_desc(&tmB0);
      if constexpr (kMode == CE_PROD) {
        tma_prefetch_desc(&tmA1);
        tma_prefetch_desc(&tmB1);
      }
      int stage = 0;
      uint32_t phase = 0;
      uint32_t armed = 0, armed_phase = 0;  // leader: stages whose copies (of both CTAs) may still be in flight
      bool ok = true;
      CeTile t;
      for (Work w(p, pair_id, num_pairs); ok && w.get(&t);) {
        const int my_m0 = t.m0 + int(cta_rank) * Cfg::ROWS;
        const int my_n0 = t.n0 + int(cta_rank) * 128;
        for (int kb = t.kb0; kb < t.kb0 + t.kb; ++kb) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1, &abort_flag, wait_ns)) { ok = false; break; }
          uint8_t* sa = tiles + stage * STAGE_BYTES;
          uint8_t* sb = sa + A_BYTES;
          if (cta_rank == 0) {
            mbar_arrive_expect_tx(&full_bar[stage], kGroup * STAGE_BYTES);
            armed |= 1u << stage;
            armed_phase = (armed_phase & ~(1u << stage)) | (phase << stage);
          }
          const uint32_t leader_full = kPair ? mapa_u32(smem_u32(&full_bar[stage]), 0) : 0;
          if constexpr (!kPair) {
            tma_load_3d(sa, &tmA0, &full_bar[stage], kb * BK, t.m0, 0);
            tma_load_3d(sb, &tmB0, &full_bar[stage], kb * BK, t.n0, 0);
          } else if constexpr (kMode != CE_PROD) {
            tma_load_3d_pair(sa, &tmA0, leader_full, kb * BK, my_m0, 0);
            tma_load_3d_pair(sb, &tmB0, leader_full, kb * BK, my_n0, 0);
          } else {
            if (t.job == 0) {
              tma_load_3d_pair(sa, &tmA0, leader_full, kb * BK, my_m0, 0);
            } else {  // MN-major: boxes of [64 k][64 m], 8192 bytes each
#pragma unroll
              for (int c = 0; c < Cfg::ROWS / 64; ++c)
                tma_load_3d_pair(sa + c * (BK * 128), &tmA1, leader_full, my_m0 + c * 64, kb * BK, 0);
            }
            const CUtensorMap* tb = t.job == 0 ? &tmB0 : &tmB1;
            tma_load_3d_pair(sb, tb, leader_full, my_n0, kb * BK, 0);
            tma_load_3d_pair(sb + BK * 128, tb, leader_full, my_n0 + 64, kb * BK, 0);
          }
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
      if (!ok) {
        // Unwinding: copies in flight get a bounded time to land (the partner, which has no barrier of its own to watch, a
        // fixed grace period) before the CTAs meet at the cluster barrier below.
        const uint64_t t0 = globaltimer_ns();
        if (cta_rank == 0) {
          for (int s = 0; s < STAGES; ++s) {
            if (!(armed & (1u << s))) continue;
            while (!mbar_try_wait(&full_bar[s], (armed_phase >> s) & 1u)) {
              if (globaltimer_ns() - t0 > 2000000ull) break;
            }
          }
        } else {
          while (globaltimer_ns() - t0 < 100000ull) __nanosleep(1000);
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (leader CTA only)
    if (lane == 0 && cta_rank == 0) {
      constexpr uint64_t k_major = make_smem_desc_hi(16, 1024);
      constexpr uint64_t mn_major = make_smem_desc_hi(BK * 128, 1024);  // chunks of 64 columns 8192 bytes apart
      constexpr int KSTEPS = BK / 16;
      constexpr bool kBmn = kMode == CE_PROD;
      constexpr uint64_t b_hi = kBmn ? mn_major : k_major;
      constexpr uint32_t b_kstep = kBmn ? 16 * 128 : 32;
      int stage = 0;
      uint32_t phase = 0;
      int slot = 0;
      uint32_t acc_phase = 0;
      bool ok = true;
      auto advance = [&](int& s, uint32_t& ph) {
        if (++s == STAGES) { s = 0; ph ^= 1; }
      };
      CeTile t;
      for (Work w(p, pair_id, num_pairs); ok && w.get(&t);) {
        const bool a_mn = kMode == CE_PROD && t.job == 1;
        const uint32_t idesc = !kPair ? make_idesc(1, false, false, 128, p.bn) : a_mn ? make_idesc(1, true, kBmn, 256, BN) : make_idesc(1, false, kBmn, 256, BN);
        const uint64_t a_hi = a_mn ? mn_major : k_major;
        const uint32_t a_kstep = a_mn ? 16 * 128 : 32;
        const int nk = t.kb;
        // four MMAs (one 64-wide k-block) of row block `mb` into accumulator `acc`
        auto issue = [&](int acc, int mb, int s, uint32_t accumulate) {
          const uint32_t a_addr = smem_u32(tiles + s * STAGE_BYTES) + mb * (128 * 128);
          const uint32_t b_addr = smem_u32(tiles + s * STAGE_BYTES) + A_BYTES;
#pragma unroll
          for (int k = 0; k < KSTEPS; ++k)
            umma<kGroup, 0>(tmem_base + acc * BN, smem_desc(a_hi, a_addr + k * a_kstep), smem_desc(b_hi, b_addr + k * b_kstep), idesc,
                       accumulate | (k != 0 ? 1u : 0u));
        };
        auto commit = [&](uint64_t* bar) {
          if constexpr (kPair) umma_commit_pair(bar, 3);
          else umma_commit(bar);
        };
        if constexpr (kMB <= 1) {
          const int length = kSegments ? CE_SEGMENT : nk;
          for (int k0 = 0; ok && k0 < nk; k0 += length) {
            if (!mbar_wait<true>(&acc_empty[slot], acc_phase ^ 1, &abort_flag, wait_ns)) { ok = false; break; }
            tc_fence_after_sync();
            for (int kb = k0; kb < min(k0 + length, nk); ++kb) {
              if (!mbar_wait(&full_bar[stage], phase, &abort_flag, wait_ns)) { ok = false; break; }
              tc_fence_after_sync();
              issue(slot, 0, stage, kb != k0 ? 1u : 0u);
              commit(&empty_bar[stage]);
              advance(stage, phase);
            }
            if (!ok) break;
            commit(&acc_full[slot]);
            if (++slot == 2) { slot = 0; acc_phase ^= 1; }
          }
          if (!ok) break;
        } else {
          // The tile's two row blocks share every B stage; the first and last SKEW k-blocks are issued block-major, so block 0
          // is done 4 SKEW MMAs early and the next tile starts on it while block 1 is still being drained.
          constexpr int SKEW = 2;
          const int head_end = min(SKEW, nk);
          const int tail_begin = max(head_end, nk - SKEW);
          auto group = [&](int g0, int g1) {
            for (int mb = 0; mb < 2 && ok; ++mb) {
              if (g0 == 0) {
                if (!mbar_wait<true>(&acc_empty[mb], acc_phase ^ 1, &abort_flag, wait_ns)) { ok = false; break; }
                tc_fence_after_sync();
              }
              int s = stage;
              uint32_t ph = phase;
              for (int kb = g0; kb < g1; ++kb) {
                if (mb == 0) {
                  if (!mbar_wait(&full_bar[s], ph, &abort_flag, wait_ns)) { ok = false; break; }
                  tc_fence_after_sync();
                }
                issue(mb, mb, s, kb != 0 ? 1u : 0u);
                if (mb == 1) commit(&empty_bar[s]);
                advance(s, ph);
              }
              if (ok && g1 == nk) commit(&acc_full[mb]);
            }
            for (int kb = g0; kb < g1; ++kb) advance(stage, phase);
          };
          group(0, head_end);
          for (int kb = head_end; ok && kb < tail_begin; ++kb) {
            if (!mbar_wait(&full_bar[stage], phase, &abort_flag, wait_ns)) { ok = false; break; }
            tc_fence_after_sync();
            const uint32_t a_addr = smem_u32(tiles + stage * STAGE_BYTES);
            const uint32_t b_addr = a_addr + A_BYTES;
#pragma unroll
            for (int k = 0; k < KSTEPS; ++k) {
#pragma unroll
              for (int mb = 0; mb < 2; ++mb)
                umma<2, 0>(tmem_base + mb * BN, smem_desc(a_hi, a_addr + mb * (128 * 128) + k * a_kstep),
                           smem_desc(b_hi, b_addr + k * b_kstep), idesc, 1u);
            }
            commit(&empty_bar[stage]);
            advance(stage, phase);
          }
          if (ok && tail_begin < nk) group(tail_begin, nk);
          if (!ok) break;
          acc_phase ^= 1;
        }
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue (both CTAs)
    const int q = warp & 3;  // TMEM lane quarter this warp may read
    const int half = kMB <= 1 && !kSegments ? 0 : (warp - 2) >> 2;
    constexpr int kBlocks = kMB == 2 ? 2 : 1;
    constexpr int kHalves = kMB == 2 || kSegments ? 2 : 1;
    constexpr int STRIPS = (BN / 32) / kHalves;  // 32-column strips per warp and accumulator
    uint8_t* staging = tiles + ce_stage_room<kMode, kMB, kSegments>() + (warp - 2) * CE_STAGING_BYTES;
    int slot = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    const float scale = kMode == CE_PROD && p.scale != nullptr ? *p.scale : 1.0f;
    bool stored = false;  // this warp has TMA stores that may be reading its staging tile
    CeTile t;
    for (Work w(p, pair_id, num_pairs); ok && w.get(&t);) {
      const CeJob& job = p.job[t.job];
      const int n_end = kPair ? job.N : min(job.N, t.n0 + p.bn);  // columns of this tile end here at the latest
#pragma unroll 1
      for (int blk = 0; blk < kBlocks; ++blk) {
        if constexpr (kMB == 2) slot = blk;
        const int row0 = t.m0 + int(cta_rank) * Cfg::ROWS + blk * 128 + q * 32;  // this warp's first row
        const int row = row0 + lane;
        const bool row_ok = row < job.M;
        // What the row needs besides its logits, fetched while the accumulator is still being computed.
        int at = -1;  // the target's column in this product
        float lse = 0.0f, rs = 1.0f;
        bool counted = true;
        if constexpr (kMode != CE_PROD) {
          const long long tg = row_ok ? p.targets[row] : -1;
          if (tg >= p.v0 && tg < p.v0 + n_end) at = int(tg - p.v0);
          if constexpr (kMode == CE_GRAD) {
            counted = row_ok && tg != p.ignore;
            if (row_ok) {
              lse = p.lse[row];
              if (p.dloss != nullptr) rs = p.dloss[row];
              if (tg < 0 || tg >= p.V) rs = __int_as_float(0x7fc00000);
            }
          }
        }
        float m = -INFINITY, s = 0.0f;
        // One strip of logits into the row's part.
        auto lse_strip = [&](float (&v)[32], int cb) {
          if (cb + 32 > n_end) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (cb + j >= n_end) v[j] = -INFINITY;
          }
          const int a = at - cb;
          if (a >= 0 && a < 32) {
            float l = 0.0f;
#pragma unroll
            for (int j = 0; j < 32; ++j) l = a == j ? v[j] : l;
            p.target_logit[row] = l;
          }
          float top = v[0];
#pragma unroll
          for (int j = 1; j < 32; ++j) top = fmaxf(top, v[j]);  // a NaN is passed over here and meets the sum below
          const float nm = fmaxf(m, top);
          if (nm == -INFINITY) {  // no mass so far: -inf - -inf must not become NaN, a NaN must stay one
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (v[j] != v[j]) s = v[j];
          } else {
            float add = 0.0f;
#pragma unroll
            for (int j = 0; j < 32; ++j) add += ex2((v[j] - nm) * CE_LOG2E);
            s = fmaf(s, ex2((m - nm) * CE_LOG2E), add);
            m = nm;
          }
        };
        // CE_GRAD: two strips of logits (bits of floats) -> a block of 64 columns of G.
        auto grad_block = [&](const uint32_t (&a0)[32], const uint32_t (&a1)[32], int col0) {
          const bool second = col0 + 32 < n_end;
          auto put = [&](const CUtensorMap* to, bool lo) {
            auto entry = [&](uint32_t bits, float minus) {
              float g = (ex2((__uint_as_float(bits) - lse) * CE_LOG2E) - minus) * rs;
              if (lo) g -= float(__nv_bfloat16(g));
              return counted ? g : 0.0f;
            };
            auto strip = [&](const uint32_t (&r)[32], int cb, int chunk) {
#pragma unroll
              for (int c = 0; c < 4; ++c) {  // eight values at a time: the segmented form has 128 logits in registers
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = entry(r[8 * c + j], 0.0f);
                *reinterpret_cast<uint4*>(staged_at(staging, lane, chunk + c)) = EpilogueCtx<__nv_bfloat16>::pack8_bf16(v);
              }
              const int a = at - cb;
              if (a >= 0 && a < 32) {
                uint32_t l = 0;
#pragma unroll
                for (int j = 0; j < 32; ++j) l = a == j ? r[j] : l;
                *reinterpret_cast<__nv_bfloat16*>(staged_at(staging, lane, chunk + (a >> 3)) + 2 * (a & 7)) = __nv_bfloat16(entry(l, 1.0f));
              }
            };
            if (stored && lane == 0) bulk_wait_group_read<0>();  // the previous block has left the staging tile
            __syncwarp();
            strip(a0, col0, 0);
            if (second) strip(a1, col0 + 32, 4);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_3d(to, staging, col0, row0, 0);
              bulk_commit_group();
            }
            stored = true;
          };
          put(&out0, false);
          if (kMB == 0 && p.lo) put(&out1, true);
        };
        if constexpr (kSegments) {
          float l[STRIPS][32];
#pragma unroll
          for (int c = 0; c < STRIPS; ++c)
#pragma unroll
            for (int j = 0; j < 32; ++j) l[c][j] = 0.0f;
          for (int k0 = 0; ok && k0 < t.kb; k0 += CE_SEGMENT) {
            if (!mbar_wait_warp(&acc_full[slot], acc_phase, &abort_flag, wait_ns)) { ok = false; break; }
            tc_fence_after_sync();
#pragma unroll
            for (int c = 0; c < 2 * STRIPS; ++c) {
              uint32_t r[16];
              tmem_get_32x16(tmem_base + (uint32_t(q * 32) << 16) + slot * BN + half * STRIPS * 32 + c * 16, r);
#pragma unroll
              for (int j = 0; j < 16; ++j) l[c / 2][c % 2 * 16 + j] += __uint_as_float(r[j]);
            }
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) {
              if constexpr (kPair) mbar_arrive_cluster(mapa_u32(smem_u32(&acc_empty[slot]), 0));
              else mbar_arrive(&acc_empty[slot]);
            }
            if (++slot == 2) { slot = 0; acc_phase ^= 1; }
          }
          if (!ok) break;
          if constexpr (kMode == CE_LSE) {
#pragma unroll
            for (int c = 0; c < STRIPS; ++c) {
              const int cb = t.n0 + (half * STRIPS + c) * 32;
              if (cb < n_end) lse_strip(l[c], cb);
            }
            if (row_ok) p.part[((long long)(kPair ? t.n0 / BN : t.n0 / p.bn) * 2 + half) * job.M + row] = make_float2(m, s);
          } else {
#pragma unroll
            for (int c = 0; c < STRIPS; c += 2) {
              const int cb = t.n0 + (half * STRIPS + c) * 32;
              if (cb >= n_end) continue;
              uint32_t a0[32], a1[32];
#pragma unroll
              for (int j = 0; j < 32; ++j) a0[j] = __float_as_uint(l[c][j]), a1[j] = __float_as_uint(l[c + 1][j]);
              grad_block(a0, a1, cb);
            }
          }
          continue;
        }
        if (!mbar_wait_warp(&acc_full[slot], acc_phase, &abort_flag, wait_ns)) { ok = false; break; }
        tc_fence_after_sync();
#pragma unroll 1
        for (int c = half * STRIPS; c < (half + 1) * STRIPS; c += 2) {
          uint32_t r0[32], r1[32];
          const uint32_t taddr = tmem_base + (uint32_t(q * 32) << 16) + slot * BN + c * 32;
          tmem_ld_32x32(taddr, r0);
          tmem_ld_32x32(taddr + 32, r1);
          tmem_ld_wait();
          const int col0 = t.n0 + c * 32;
          if (col0 >= n_end) continue;
          const bool second = col0 + 32 < n_end;
          float v[32];

          if constexpr (kMode == CE_LSE) {
            auto strip = [&](const uint32_t (&r)[32], int cb) {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
              lse_strip(v, cb);
            };
            strip(r0, col0);
            if (second) strip(r1, col0 + 32);
          } else if constexpr (kMode == CE_GRAD) {
            grad_block(r0, r1, col0);
          } else {
            const bool f32 = t.job == 0 && !p.dx_bf16;
            const CUtensorMap* om = t.job == 0 ? &out0 : &out1;
            const bool tma = p.tma_out[t.job] != 0;
            auto strip = [&](const uint32_t (&r)[32], int cb) {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
              if (t.job == 0 && p.dx_add && row_ok) {
                const float* a = p.dx_acc + ((long long)t.chunk * job.M + row) * job.N + cb;
                if (cb + 32 <= job.N && (job.N & 3) == 0) {
#pragma unroll
                  for (int j = 0; j < 8; ++j) {
                    const float4 x = *reinterpret_cast<const float4*>(a + 4 * j);
                    v[4 * j] += x.x; v[4 * j + 1] += x.y; v[4 * j + 2] += x.z; v[4 * j + 3] += x.w;
                  }
                } else {
#pragma unroll
                  for (int j = 0; j < 32; ++j)
                    if (cb + j < job.N) v[j] += a[j];
                }
              }
              if (!f32) {
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] *= scale;
              }
            };
            auto plain = [&](int cb) {  // rows that a TMA store cannot take
              if (!row_ok) return;
              const long long off = ((long long)t.chunk * job.M + row) * job.N + cb;
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                if (cb + j >= job.N) break;
                if (f32) static_cast<float*>(p.out[0])[off + j] = v[j];
                else static_cast<__nv_bfloat16*>(p.out[t.job])[off + j] = __nv_bfloat16(v[j]);
              }
            };
            strip(r0, col0);
            if (!tma) {
              plain(col0);
              if (second) {
                strip(r1, col0 + 32);
                plain(col0 + 32);
              }
              continue;
            }
            if (stored && lane == 0) bulk_wait_group_read<0>();
            __syncwarp();
            if (f32) {  // one 128-byte block per strip
              stage_f32(v, staging, lane);
              if (second) {
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                  tma_store_3d(om, staging, col0, row0, t.chunk);
                  bulk_commit_group();
                }
                strip(r1, col0 + 32);
                if (lane == 0) bulk_wait_group_read<0>();
                __syncwarp();
                stage_f32(v, staging, lane);
              }
            } else {
              stage_bf16(v, staging, lane, 0);
              if (second) {
                strip(r1, col0 + 32);
                stage_bf16(v, staging, lane, 4);
              }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_3d(om, staging, f32 && second ? col0 + 32 : col0, row0, t.chunk);
              bulk_commit_group();
            }
            stored = true;
          }
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          if constexpr (kPair) mbar_arrive_cluster(mapa_u32(smem_u32(&acc_empty[slot]), 0));  // leader's barrier
          else mbar_arrive(&acc_empty[slot]);
        }
        if constexpr (kMode == CE_LSE) {
          if (row_ok) p.part[(long long)(kPair ? t.n0 / BN * kMB + half : t.n0 / p.bn) * job.M + row] = make_float2(m, s);
        }
      }
      if constexpr (kSegments) {
      } else if constexpr (kMB <= 1) {
        if (++slot == 2) { slot = 0; acc_phase ^= 1; }
      } else {
        acc_phase ^= 1;
      }
    }
    if (stored && lane == 0) bulk_wait_group<0>();  // every store of this warp has been performed
  }

  // Both CTAs stay until every remote barrier signal and paired MMA has landed.
  tc_fence_before_sync();
  __syncwarp();
  if constexpr (kPair) cluster_sync_all();
  else __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc<kGroup>(tmem_base, Cfg::TMEM_COLS);
  }
  if (threadIdx.x == 0 && abort_flag != 0 && p.status != nullptr) atomicExch(p.status, int(ST_WAIT_TIMEOUT));
}

// ------------------------------------------------------------------ host side

int map_of(CUtensorMap* out, const CeMatrix& m, uint32_t box_cols, uint32_t box_rows) {
  const uint64_t dims[3] = {(uint64_t)m.cols, (uint64_t)m.rows, 1};
  const uint64_t strides[2] = {(uint64_t)m.ld * 2, (uint64_t)m.rows * m.ld * 2};
  const uint32_t box[3] = {box_cols, box_rows, 1};
  return encode_tensor_map_3d(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, m.p, dims, strides, box);
}

int out_map(CUtensorMap* out, const void* p, long long rows, long long cols, long long ld, bool f32, int planes = 1) {
  const int eb = f32 ? 4 : 2;
  const uint64_t dims[3] = {(uint64_t)cols, (uint64_t)rows, (uint64_t)planes};
  const uint64_t strides[2] = {(uint64_t)ld * eb, (uint64_t)rows * ld * eb};
  const uint32_t box[3] = {(uint32_t)(128 / eb), 32, 1};
  return encode_tensor_map_3d(out, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, p, dims, strides, box);
}

CeJob job_of(long long M, long long N, long long K, int mb) {
  CeJob j;
  j.M = (int)M; j.N = (int)N; j.K = (int)K;
  const int bm = mb > 0 ? 256 * mb : 128;
  j.m_tiles = (int)((M + bm - 1) / bm);
  j.n_tiles = (int)((N + 255) / 256);
  j.group_m = mb == 2 ? 4 : 8;
  j.chunks = 1;
  j.chunk_kb = (int)((K + 63) / 64);
  return j;
}

template <int kMode, int kMB, bool kSegments = false>
int launch(const CUtensorMap (&in)[4], const CUtensorMap (&out)[2], const CeKernelParams& p, long long tiles, int num_sms, cudaStream_t stream) {
  auto kern = ce_pair_kernel<kMode, kMB, kSegments>;
  constexpr int THREADS = 64 + 32 * CE_EPI_WARPS<kMB, kSegments>;
  constexpr int DYN_SMEM = CE_DYN_SMEM<kMode, kMB, kSegments>;
  SX_ENSURE_DYN_SMEM(kern, DYN_SMEM);
  constexpr int kGroup = kMB > 0 ? 2 : 1;
  // In plain stream order, not as a programmatic dependent: one of two things that a hang of unknown cause had in common (2 us more for
  // the smallest calls).
  const unsigned groups = (unsigned)std::min<long long>(tiles, num_sms / kGroup);
  const cudaError_t e = launch_kernel_ex(kern, kGroup * groups, THREADS, DYN_SMEM, stream, kGroup, false, in[0], in[1], in[2], in[3],
                                         out[0], out[1], p);
  if (e != cudaSuccess) return launch_failed(e, "loss kernel launch failed");
  count_launches(1);
  return SX_OK;
}

CeKernelParams common(const CeCommon& c) {
  CeKernelParams p{};
  p.status = c.status;
  p.wait_limit_ns = c.wait_limit_ns;
  return p;
}

}  // namespace

int ce_dx_chunks(long long T, long long H, long long n) {
  // dx has T / 512 x H / 256 tiles of n / 64 k-blocks each. Where these are fewer than the 74 CTA pairs, the longest of them would
  // outlast everything else (1999 x 768 tokens: 12 tiles of 524 k-blocks, 290 us of a product of 330): as many parts as make a wave,
  // none shorter than 16 k-blocks.
  const long long tiles = ((T + 511) / 512) * ((H + 255) / 256), nkb = (n + 63) / 64;
  if (tiles >= 74) return 1;
  return (int)std::max<long long>(1, std::min((74 + tiles - 1) / tiles, nkb / 16));
}
long long ce_piece_of_waves(long long T, long long V, long long most) {
  const long long m = (T + 511) / 512, columns = (V + 255) / 256;
  auto waves = [&](long long c) { return (m * c + 73) / 74; };
  long long best = most / 256;
  double least = 1e30;
  for (long long c = most / 256; c >= most / 512 && c > 0; --c) {
    const double cost = columns / c * (waves(c) + 0.5) + (columns % c ? waves(columns % c) + 0.5 : 0);
    if (cost < least) least = cost, best = c;
  }
  return best * 256;
}

// The logits' product of either pass: operands, tile shape (chosen here alone, by one look at the options), and the kernel for it. `parts`:
// how many parts the forward pass writes of a row.
template <int kMode>
static int launch_logits(const CeCommon& c, const CeMatrix& x, const CeMatrix& W, const CUtensorMap (&out)[2], CeKernelParams* p, cudaStream_t stream,
                         int* parts) {
  const CeTiles tiling = kMode == CE_LSE ? ce_forward_tiles(x.rows, W.rows, x.cols, c.num_sms, (int)options().pair_mode.load(std::memory_order_relaxed))
                                         : ce_gradient_tiles(x.rows, p->V, x.cols, W.rows, p->lo != 0, c.num_sms, (int)options().pair_mode.load(std::memory_order_relaxed));
  const int mb = tiling.mb;
  const bool segments = tiling.segments;
  uint32_t a_rows = 128 * mb, b_rows = 128;
  p->job[0] = job_of(x.rows, W.rows, x.cols, mb);
  if (mb == 0) {
    a_rows = (uint32_t)(x.rows + 15) / 16 * 16;
    b_rows = (uint32_t)tiling.bn;
    p->bn = tiling.bn;
    p->a_bytes = (int)a_rows * 128;
    const int room = segments ? ce_stage_room<kMode, 0, true>() : ce_stage_room<kMode, 0, false>();
    p->stages = std::min(CeCfg<0>::STAGES, room / (p->a_bytes + p->bn * 128));
    p->job[0].n_tiles = (int)((W.rows + p->bn - 1) / p->bn);
  }
  if constexpr (kMode == CE_LSE) *parts = ce_parts(tiling, W.rows);
  CUtensorMap in[4] = {};
  int rc = map_of(&in[0], x, 64, a_rows);
  if (rc == SX_OK) rc = map_of(&in[1], W, 64, b_rows);
  if (rc != SX_OK) return rc;
  const long long tiles = (long long)p->job[0].m_tiles * p->job[0].n_tiles;
  if (tiles > 0x7fffffffLL) return set_last_error(SX_ERR_INVALID, "the problem has more than 2^31-1 tiles");
  if (segments) return mb == 0 ? launch<kMode, 0, true>(in, out, *p, tiles, c.num_sms, stream) : launch<kMode, 1, true>(in, out, *p, tiles, c.num_sms, stream);
  if (mb == 0) return launch<kMode, 0>(in, out, *p, tiles, c.num_sms, stream);
  if constexpr (kMode == CE_GRAD) {
    if (mb == 1) return launch<kMode, 1>(in, out, *p, tiles, c.num_sms, stream);
  }
  return launch<kMode, 2>(in, out, *p, tiles, c.num_sms, stream);
}

int launch_ce_forward(const CeCommon& c, const CeForward& a, cudaStream_t stream, int* parts) {
  CeKernelParams p = common(c);
  p.targets = a.targets;
  p.V = a.W.rows;
  p.part = a.part;
  p.target_logit = a.target_logit;
  p.done = a.done;
  return launch_logits<CE_LSE>(c, a.x, a.W, {CUtensorMap{}, CUtensorMap{}}, &p, stream, parts);
}

int launch_ce_grad(const CeCommon& c, const CeGrad& a, cudaStream_t stream) {
  CUtensorMap to[2] = {};
  int rc = out_map(&to[0], a.G, a.x.rows, a.W.rows, a.ldg, false);
  if (rc == SX_OK && a.lo) rc = out_map(&to[1], static_cast<const uint16_t*>(a.G) + a.x.rows * a.ldg, a.x.rows, a.W.rows, a.ldg, false);
  if (rc != SX_OK) return rc;
  CeKernelParams p = common(c);
  p.lo = a.lo ? 1 : 0;
  p.targets = a.targets;
  p.lse = a.lse;
  p.dloss = a.dloss;
  p.v0 = a.v0;
  p.V = a.V;
  p.ignore = a.ignore;
  return launch_logits<CE_GRAD>(c, a.x, a.W, to, &p, stream, nullptr);
}

// The tiles of both products in one shape. Returns how long the busiest pair works, in k-blocks of 256 x 256.
static double products_plan(long long T, long long H, long long n, int mb, int chunks, int num_sms, CeKernelParams* p) {
  p->job[0] = job_of(T, H, n, mb);
  p->job[1] = job_of(n, H, T, mb);
  // The widest piece (the first one) sets how many accumulators there are; a narrower one may fill fewer of them.
  const long long nkb = (n + 63) / 64, tkb = (T + 63) / 64;
  p->job[0].chunk_kb = (int)((nkb + chunks - 1) / chunks);
  p->job[0].chunks = (int)((nkb + p->job[0].chunk_kb - 1) / p->job[0].chunk_kb);
  const long long t0 = (long long)p->job[0].m_tiles * p->job[0].n_tiles * p->job[0].chunks, t1 = (long long)p->job[1].m_tiles * p->job[1].n_tiles;
  const long long pairs = std::min<long long>(t0 + t1, num_sms / 2), full = t0 % pairs;
  p->first_extra = 0;
  if (full != 0) {
    const long long each = (p->job[0].chunk_kb + tkb / 2) / tkb;  // dW tiles that take as long as one of dx
    p->first_extra = (int)std::min<long long>(t1, each * (pairs - full));
  }
  const double tile0 = p->job[0].chunk_kb + 4, tile1 = tkb + 4;  // with the start and end of a tile
  double most = 0;
  for (long long i = 0; i < pairs; ++i) {
    const long long n0 = t0 / pairs + (i < full), rest = t1 - p->first_extra;
    const long long ahead = i >= full && p->first_extra ? (p->first_extra + pairs - 1 - i) / (pairs - full) : 0;
    most = std::max(most, n0 * tile0 + (ahead + rest / pairs + (i < rest % pairs)) * tile1);
  }
  return most * mb / (mb == 1 ? 0.80 : 0.84);
}

int launch_ce_products(const CeCommon& c, const CeProducts& a, cudaStream_t stream) {
  const long long T = a.x.rows, H = a.x.cols, n = a.W.rows;
  CeKernelParams p = common(c);
  // 256-row or 512-row tiles, whichever get done first (us of a whole backward pass, vocabulary 50257: 8192 x 512 1225 / 1574,
  // 4096 x 1024 1058 / 1124, 4096 x 2048 1909 / 1872, 8192 x 4096 7226 / 6910).
  const int64_t mode = options().pair_mode.load(std::memory_order_relaxed);
  int mb = mode == 1 || mode == 2 ? (int)mode : 1;
  const double time = products_plan(T, H, n, mb, a.chunks, c.num_sms, &p);
  if (mode != 1 && mode != 2 && std::min(T, n) > 256) {
    CeKernelParams q = p;
    if (products_plan(T, H, n, 2, a.chunks, c.num_sms, &q) < time) p = q, mb = 2;
  }
  CUtensorMap in[4], out[2] = {};
  int rc = map_of(&in[0], a.G, 64, 128 * mb);          // dx: A = G, k = vocabulary
  if (rc == SX_OK) rc = map_of(&in[1], a.W, 64, 64);   //     B = W, MN-major
  if (rc == SX_OK) rc = map_of(&in[2], a.G, 64, 64);   // dW: A = G^T, MN-major, k = tokens
  if (rc == SX_OK) rc = map_of(&in[3], a.x, 64, 64);   //     B = x, MN-major
  if (rc != SX_OK) return rc;
  p.scale = a.scale;
  p.dx_acc = a.acc;
  p.dx_add = a.first ? 0 : 1;
  p.dx_bf16 = a.chunks == 1 && a.last && a.dx != nullptr;
  p.out[0] = p.dx_bf16 ? a.dx : a.acc;
  p.out[1] = a.dW;
  for (int j = 0; j < 2; ++j) {
    const bool f32 = j == 0 && !p.dx_bf16;
    p.tma_out[j] = (H * (f32 ? 4 : 2)) % 16 == 0 && reinterpret_cast<uintptr_t>(p.out[j]) % 16 == 0;
    if (p.tma_out[j] && (rc = out_map(&out[j], p.out[j], j == 0 ? T : n, H, H, f32, j == 0 ? p.job[0].chunks : 1)) != SX_OK) return rc;
  }
  const long long t0 = (long long)p.job[0].m_tiles * p.job[0].n_tiles * p.job[0].chunks, t1 = (long long)p.job[1].m_tiles * p.job[1].n_tiles;
  if (t0 + t1 > 0x3fffffffLL) return set_last_error(SX_ERR_INVALID, "the problem has more than 2^30-1 tiles");
  return mb == 2 ? launch<CE_PROD, 2>(in, out, p, t0 + t1, c.num_sms, stream) : launch<CE_PROD, 1>(in, out, p, t0 + t1, c.num_sms, stream);
}

}  // namespace sx
