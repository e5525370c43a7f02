// Products of a few rows with 4-bit weights that carry a scale (and a zero) per group of consecutive k:
//
//   C[m][n] = act(sum_g scale[n][g] * sum_{k in g} (code[n][k] - zero[n][g]) * A[m][k] + bias[n])
//
// Bound by HBM: N K / 2 bytes of codes, read once whatever M is, up to about a hundred rows.
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
  int M, N, K, group, groups;
  long long lda, ldq, ldc;
  int act;
};

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

template <typename ST, typename OutT>
int matvec(const Int4Args& a, cudaStream_t stream) {
  cudaError_t e = launch_kernel_ex(int4_matvec_any_kernel<ST, OutT>, (unsigned)((a.N + 7) / 8), 256, 0, stream, 1, pdl_enabled(), a);
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
  if (scale_dtype == SYMPLEX_DT_F32)
    return out_dtype == SYMPLEX_DT_F32 ? matvec<float, float>(a, st) : matvec<float, __nv_bfloat16>(a, st);
  return out_dtype == SYMPLEX_DT_F32 ? matvec<__nv_bfloat16, float>(a, st) : matvec<__nv_bfloat16, __nv_bfloat16>(a, st);
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
