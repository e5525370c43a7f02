// Interface between the C entry points of the linear head's loss (linear_cross_entropy.cu) and its tensor-core kernels
// (ce_pair_sm100.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace sx {

constexpr float CE_LOG2E = 1.4426950408889634f;

// A bf16 matrix of `rows` rows of `cols` values, `ld` values apart; base 16-byte aligned, ld a multiple of 8.
struct CeMatrix {
  const void* p;
  long long rows, cols, ld;
};

struct CeCommon {
  int num_sms;
  int* status;
  unsigned long long wait_limit_ns;
};

// Forward: every row's part (largest logit, sum of exp(l - largest)) of every tile column, and the targets' logits.
struct CeForward {
  CeMatrix x, W;  // [T, H], [V, H]
  const long long* targets;
  float2* part;  // [parts][T], room for ce_parts_most
  float* target_logit;
  unsigned* done;  // set to 0
};
int launch_ce_forward(const CeCommon& c, const CeForward& a, cudaStream_t stream, int* parts);  // parts: those that it writes

// G[t][v] = (exp(x W^T - lse) - [v0 + v = target]) * (dloss ? dloss[t] : 1), 0 in ignored rows, NaN where the target is none.
struct CeGrad {
  CeMatrix x, W;  // [T, H], the piece of W: [n, H]
  void* G;        // bf16 [T, ldg], ldg a multiple of 8, 16-byte aligned
  long long ldg;
  bool lo;  // T <= 128 only: G's rounding errors follow in another T rows, bf16 as well
  const long long* targets;
  const float* lse;
  const float* dloss;  // per row, or null
  long long v0, V, ignore;
};
int launch_ce_grad(const CeCommon& c, const CeGrad& a, cudaStream_t stream);

// dx (+)= G W and dW = G^T x of one piece, times *scale where scale is not null. dx goes to `chunks` fp32 accumulators [T, H] in a row
// (its k, the vocabulary, cut into as many parts), to which pieces after the first one add. With one chunk the last piece writes
// bf16 dx = (acc + G W) * scale instead where dx is given; else the accumulators are joined afterwards.
struct CeProducts {
  CeMatrix G, x, W;  // [T, n], [T, H], [n, H]
  float* acc;
  int chunks;
  bool first, last;
  void* dx;
  void* dW;  // [n, H] packed
  const float* scale;
};
int launch_ce_products(const CeCommon& c, const CeProducts& a, cudaStream_t stream);
// Chunks for a problem whose widest piece has n columns, on a device with 148 SMs (the workspace is sized without one).
int ce_dx_chunks(long long T, long long H, long long n);
// Columns of a piece, at most `most` (a multiple of 256): those with which the pieces' logits take the fewest waves of tiles, half
// a wave counted for each piece's start and end.
long long ce_piece_of_waves(long long T, long long V, long long most);

}  // namespace sx
