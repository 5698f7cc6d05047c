// Products of block-scaled 8-bit codes: C[m][n] = sum_k a[m,k] b[n,k], the
// values being code * 2^e with one e for 128 neighbours along k.
//
// 64 x 64 tiles on the FP32 pipe, 32 values of k at a time: values are
// restored while they are staged in shared memory, so any operand layout and
// any sizes take the same code.
#include "f64e_fp8.cuh"
#include "f64e_fp8.h"

namespace f64e {

namespace {

constexpr int kT = 64, kKc = 32;

__device__ __forceinline__ float value_at(const Fp8Operand& o, int64_t r, int64_t k) {
  const uint32_t q = o.kmajor ? o.q[r * o.ld + k] : o.q[k * o.ld + r];
  const float2 v = o.code == F64E_E4M3 ? values2<F64E_E4M3>(q) : values2<F64E_E5M2>(q);
  return v.x * scale_of_byte(o.s[(r >> o.s_shift) * o.s_row + (k / kFp8Block) * o.s_kb]);
}

__global__ void __launch_bounds__(256) fp8_gemm_simple_kernel(const Fp8GemmArgs g) {
  __shared__ float sa[kKc][kT + 1], sb[kKc][kT + 1];
  const int64_t ntn = (g.N + kT - 1) / kT;
  const int64_t m0 = (int64_t)(blockIdx.x / ntn) * kT, n0 = (int64_t)(blockIdx.x % ntn) * kT;
  const int tm = threadIdx.x >> 4, tn = threadIdx.x & 15;
  float acc[4][4] = {};
  for (int64_t k0 = 0; k0 < g.K; k0 += kKc) {
    for (int i = threadIdx.x; i < kT * kKc; i += 256) {
      // neighbouring threads read along the operand's contiguous direction
      const int ra = g.a.kmajor ? i / kKc : i % kT, ka = g.a.kmajor ? i % kKc : i / kT;
      sa[ka][ra] = (m0 + ra < g.M && k0 + ka < g.K) ? value_at(g.a, m0 + ra, k0 + ka) : 0.f;
      const int rb = g.b.kmajor ? i / kKc : i % kT, kb = g.b.kmajor ? i % kKc : i / kT;
      sb[kb][rb] = (n0 + rb < g.N && k0 + kb < g.K) ? value_at(g.b, n0 + rb, k0 + kb) : 0.f;
    }
    __syncthreads();
    for (int k = 0; k < kKc; k++)
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] = fmaf(sa[k][tm + 16 * i], sb[k][tn + 16 * j], acc[i][j]);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int64_t m = m0 + tm + 16 * i, n = n0 + tn + 16 * j;
      if (m >= g.M || n >= g.N) continue;
      const int64_t at = m * g.ldo + n;
      if (g.out_type == F64E_F32)
        static_cast<float*>(g.out)[at] = acc[i][j];
      else if (g.out_type == F64E_F16)
        static_cast<__half*>(g.out)[at] = __float2half_rn(acc[i][j]);
      else
        static_cast<__nv_bfloat16*>(g.out)[at] = __float2bfloat16_rn(acc[i][j]);
    }
}

}  // namespace

cudaError_t launch_fp8_gemm(const Fp8GemmArgs& g, cudaStream_t s) {
  const int64_t tiles = ((g.M + kT - 1) / kT) * ((g.N + kT - 1) / kT);
  fp8_gemm_simple_kernel<<<(unsigned)tiles, 256, 0, s>>>(g);
  return cudaGetLastError();
}

}  // namespace f64e
