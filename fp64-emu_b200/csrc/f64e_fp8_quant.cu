// Block quantisation to 8-bit floating point and back.
//
// Both kernels are bound by memory: rows reads e bytes a value (e = 2 or 4)
// and writes 1 + 1/128; the squares kernel does the same and, asked for row
// and column blocks at once, writes 2 (1 + 1/128) for one read.
#include "f64e_fp8.cuh"
#include "f64e_fp8.h"

namespace f64e {

namespace {

constexpr int kThreads = 256;

// Largest finite magnitude of a block is wanted; the first pass takes the
// largest of all, and only a block that holds a non-finite value pays for a
// second look.
template <int T>
__device__ __forceinline__ uint32_t max8(const uint32_t* w) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) m = max(m, mag<T>(w, i));
  return m;
}
template <int T>
__device__ __forceinline__ uint32_t max8_finite(const uint32_t* w) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const uint32_t v = mag<T>(w, i);
    if (v < kInfBits) m = max(m, v);
  }
  return m;
}

// Maximum over the 16 lanes that hold one 128-value row block.
__device__ __forceinline__ uint32_t max_half_warp(uint32_t m) {
#pragma unroll
  for (int o = 8; o; o >>= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
  return m;
}

// --------------------------------------------------------------- rows ----
// Half a warp holds a block: eight values a lane, one 16-byte load each (two
// in 32 bits).  A CTA covers 16 rows by four blocks, all its loads in flight
// before the first reduction.
constexpr int kRowBlocks = 4, kRowPasses = 4, kRowsPerPass = kThreads / (16 * kRowBlocks);

template <int T, int CODE>
__global__ void __launch_bounds__(kThreads) fp8_quant_rows_kernel(const Fp8QuantArgs a, int64_t nkb, int64_t ngroups,
                                                                  bool vec) {
  const int half = threadIdx.x >> 4, l = threadIdx.x & 15;
  const int64_t kb = (blockIdx.x % ngroups) * kRowBlocks + (half & (kRowBlocks - 1));
  const int64_t row0 = (blockIdx.x / ngroups) * (kRowsPerPass * kRowPasses) + half / kRowBlocks;
  const int64_t col = kb * kFp8Block + l * 8;
  const int64_t padded = (a.cols + 15) & ~(int64_t)15;
  const typename Elem<T>::type* x = static_cast<const typename Elem<T>::type*>(a.x);
  uint32_t w[kRowPasses][Elem<T>::kWords];
#pragma unroll
  for (int u = 0; u < kRowPasses; u++) {
    const int64_t r = row0 + u * kRowsPerPass;
    load8<T>(x + r * a.ldx + col, r < a.rows ? a.cols - col : 0, vec, w[u]);
  }
#pragma unroll
  for (int u = 0; u < kRowPasses; u++) {
    const int64_t r = row0 + u * kRowsPerPass;
    uint32_t m = max_half_warp(max8<T>(w[u]));
    const bool special = m >= kInfBits;
    if (__any_sync(0xFFFFFFFFu, special)) {
      const uint32_t f = max_half_warp(max8_finite<T>(w[u]));
      if (special) m = f;
    }
    const int e = scale_exponent<CODE>(m);
    const uint2 c = codes8<T, CODE>(w[u], inverse_scale(e), special);
    if (r < a.rows) {
      if (col < padded) *reinterpret_cast<uint2*>(a.q + r * a.ldq + col) = c;
      if (l == 0 && kb < nkb) a.s[r * nkb + kb] = (uint8_t)(e + 127);
    }
  }
}

// ------------------------------------------------------------ squares ----
// A CTA keeps a 128 x 128 square in registers: thread (g, l), g = half-warp,
// holds eight columns 8 l.. of the rows g, g + 16, ..; the value is read once
// for both block directions.  Column maxima: over the thread's rows, the two
// half-warps of a warp, then the eight warps through shared memory.
constexpr int kSqRows = kFp8Block / (kThreads / 16);

template <int T, int CODE, int MODE>  // MODE 0: column blocks, 1: column and row blocks, 2: square blocks
__global__ void __launch_bounds__(kThreads) fp8_quant_squares_kernel(const Fp8QuantArgs a, int64_t nkb, bool vec) {
  __shared__ uint32_t s_max[kThreads / 32][kFp8Block];
  const int g = threadIdx.x >> 4, l = threadIdx.x & 15, warp = threadIdx.x >> 5;
  const int64_t kb = blockIdx.x % nkb, rb = blockIdx.x / nkb;
  const int64_t col = kb * kFp8Block + l * 8;
  const int64_t padded = (a.cols + 15) & ~(int64_t)15;
  const typename Elem<T>::type* x = static_cast<const typename Elem<T>::type*>(a.x);
  uint32_t w[kSqRows][Elem<T>::kWords];
#pragma unroll
  for (int u = 0; u < kSqRows; u++) {
    const int64_t r = rb * kFp8Block + u * (kThreads / 16) + g;
    load8<T>(x + r * a.ldx + col, r < a.rows ? a.cols - col : 0, vec, w[u]);
  }

  // Maxima of the eight columns over the square, every thread's copy.
  auto column_maxima = [&](bool finite_only, uint32_t* cm) {
#pragma unroll
    for (int i = 0; i < 8; i++) cm[i] = 0;
#pragma unroll
    for (int u = 0; u < kSqRows; u++)
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const uint32_t v = mag<T>(w[u], i);
        if (!finite_only || v < kInfBits) cm[i] = max(cm[i], v);
      }
#pragma unroll
    for (int i = 0; i < 8; i++) cm[i] = max(cm[i], __shfl_xor_sync(0xFFFFFFFFu, cm[i], 16));
    if ((threadIdx.x & 31) < 16) {
      *reinterpret_cast<uint4*>(&s_max[warp][l * 8]) = make_uint4(cm[0], cm[1], cm[2], cm[3]);
      *reinterpret_cast<uint4*>(&s_max[warp][l * 8 + 4]) = make_uint4(cm[4], cm[5], cm[6], cm[7]);
    }
    __syncthreads();
#pragma unroll
    for (int v = 0; v < kThreads / 32; v++) {
      const uint4 p = *reinterpret_cast<const uint4*>(&s_max[v][l * 8]);
      const uint4 q = *reinterpret_cast<const uint4*>(&s_max[v][l * 8 + 4]);
      cm[0] = max(cm[0], p.x);
      cm[1] = max(cm[1], p.y);
      cm[2] = max(cm[2], p.z);
      cm[3] = max(cm[3], p.w);
      cm[4] = max(cm[4], q.x);
      cm[5] = max(cm[5], q.y);
      cm[6] = max(cm[6], q.z);
      cm[7] = max(cm[7], q.w);
    }
    __syncthreads();
  };
  auto all_of = [&](const uint32_t* cm) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) m = max(m, cm[i]);
    return max_half_warp(m);
  };

  uint32_t cm[8];
  column_maxima(false, cm);
  const bool special = all_of(cm) >= kInfBits;   // the same in every thread
  uint32_t fin[8];
#pragma unroll
  for (int i = 0; i < 8; i++) fin[i] = cm[i];
  if (special) column_maxima(true, fin);

  if (MODE == 2) {
    const int e = scale_exponent<CODE>(all_of(fin));
    const float r = inverse_scale(e);
#pragma unroll
    for (int u = 0; u < kSqRows; u++) {
      const int64_t row = rb * kFp8Block + u * (kThreads / 16) + g;
      const uint2 c = codes8<T, CODE>(w[u], r, special);
      if (row < a.rows && col < padded) *reinterpret_cast<uint2*>(a.q + row * a.ldq + col) = c;
    }
    if (threadIdx.x == 0) a.s[rb * nkb + kb] = (uint8_t)(e + 127);
    return;
  }

  float r[8];
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const int e = scale_exponent<CODE>(fin[i]);
    r[i] = inverse_scale(e);
    if (g == 0 && col + i < a.cols) a.sc[rb * a.cols + col + i] = (uint8_t)(e + 127);
  }
#pragma unroll
  for (int u = 0; u < kSqRows; u++) {
    const int64_t row = rb * kFp8Block + u * (kThreads / 16) + g;
    uint32_t c[4];
#pragma unroll
    for (int i = 0; i < 4; i++)
      c[i] = code2<CODE>(Elem<T>::get(w[u], 2 * i) * r[2 * i], Elem<T>::get(w[u], 2 * i + 1) * r[2 * i + 1]);
    if (special) {
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const float v = Elem<T>::get(w[u], i);
        if ((__float_as_uint(v) & 0x7FFFFFFFu) == kInfBits)
          c[i >> 1] = (c[i >> 1] & ~(0xFFu << (8 * (i & 1)))) | (code_of_inf<CODE>(v < 0.f) << (8 * (i & 1)));
      }
    }
    if (row < a.rows && col < padded)
      *reinterpret_cast<uint2*>(a.qc + row * a.ldq + col) = make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
  }
  if (MODE == 1) {
#pragma unroll
    for (int u = 0; u < kSqRows; u++) {
      const int64_t row = rb * kFp8Block + u * (kThreads / 16) + g;
      uint32_t m = max_half_warp(max8<T>(w[u]));
      const bool sp = m >= kInfBits;
      if (__any_sync(0xFFFFFFFFu, sp)) {
        const uint32_t f = max_half_warp(max8_finite<T>(w[u]));
        if (sp) m = f;
      }
      const int e = scale_exponent<CODE>(m);
      const uint2 c = codes8<T, CODE>(w[u], inverse_scale(e), sp);
      if (row < a.rows) {
        if (col < padded) *reinterpret_cast<uint2*>(a.q + row * a.ldq + col) = c;
        if (l == 0) a.s[row * nkb + kb] = (uint8_t)(e + 127);
      }
    }
  }
}

// --------------------------------------------------------- dequantise ----
// Sixteen codes a thread; a row block or square gives them one scale.
template <int CODE, int T>
__global__ void __launch_bounds__(kThreads) fp8_dequant_kernel(const Fp8DequantArgs a, int64_t nvec, bool vec_in,
                                                               bool vec_out) {
  const int64_t id = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int64_t r = id / nvec, c = (id - r * nvec) * 16;
  if (r >= a.rows) return;
  const int64_t n = a.cols - c;
  const uint8_t* q = a.q + r * a.ldq + c;
  uint32_t w[4] = {0, 0, 0, 0};
  if (vec_in && n >= 16) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(q));
    w[0] = v.x;
    w[1] = v.y;
    w[2] = v.z;
    w[3] = v.w;
  } else {
#pragma unroll
    for (int i = 0; i < 16; i++)
      if (i < n) w[i >> 2] |= (uint32_t)__ldg(q + i) << (8 * (i & 3));
  }
  const uint8_t* s = a.s + (a.blocks == F64E_BLOCKS_ROW ? r : r / kFp8Block) * a.s_row;
  const bool per_col = a.blocks == F64E_BLOCKS_COL;
  const float one = per_col ? 1.0f : scale_of_byte(__ldg(s + c / kFp8Block * a.s_col));
  float f[16];
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const float2 v = values2<CODE>((w[i >> 1] >> (16 * (i & 1))) & 0xFFFFu);
    f[2 * i] = v.x;
    f[2 * i + 1] = v.y;
  }
#pragma unroll
  for (int i = 0; i < 16; i++) f[i] *= per_col ? (i < n ? scale_of_byte(__ldg(s + (c + i) * a.s_col)) : 0.0f) : one;
  typename Elem<T>::type* o = static_cast<typename Elem<T>::type*>(a.out) + r * a.cols + c;
  if (vec_out && n >= 16) {
    if (T == F64E_F32) {
#pragma unroll
      for (int i = 0; i < 4; i++)
        reinterpret_cast<float4*>(o)[i] = make_float4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]);
    } else {
#pragma unroll
      for (int i = 0; i < 2; i++) {
        uint32_t p[4];
#pragma unroll
        for (int j = 0; j < 4; j++)
          p[j] = Elem<T>::bits(f[8 * i + 2 * j]) | (Elem<T>::bits(f[8 * i + 2 * j + 1]) << 16);
        reinterpret_cast<uint4*>(o)[i] = make_uint4(p[0], p[1], p[2], p[3]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; i++)
      if (i < n) {
        if (T == F64E_F32)
          reinterpret_cast<uint32_t*>(o)[i] = Elem<T>::bits(f[i]);
        else
          reinterpret_cast<uint16_t*>(o)[i] = (uint16_t)Elem<T>::bits(f[i]);
      }
  }
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
bool aligned16(const void* p, int64_t pitch_bytes) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && pitch_bytes % 16 == 0;
}

template <int T, int CODE>
cudaError_t rows_of(const Fp8QuantArgs& a, cudaStream_t s) {
  const int64_t nkb = ceil_div(a.cols, kFp8Block), ng = ceil_div(nkb, kRowBlocks);
  const int64_t grid = ng * ceil_div(a.rows, kRowsPerPass * kRowPasses);
  const bool vec = aligned16(a.x, a.ldx * (int64_t)sizeof(typename Elem<T>::type));
  fp8_quant_rows_kernel<T, CODE><<<(unsigned)grid, kThreads, 0, s>>>(a, nkb, ng, vec);
  return cudaGetLastError();
}
template <int T, int CODE>
cudaError_t squares_of(const Fp8QuantArgs& a, int tile, cudaStream_t s) {
  const int64_t nkb = ceil_div(a.cols, kFp8Block);
  const unsigned grid = (unsigned)(nkb * ceil_div(a.rows, kFp8Block));
  const bool vec = aligned16(a.x, a.ldx * (int64_t)sizeof(typename Elem<T>::type));
  if (tile)
    fp8_quant_squares_kernel<T, CODE, 2><<<grid, kThreads, 0, s>>>(a, nkb, vec);
  else if (a.q)
    fp8_quant_squares_kernel<T, CODE, 1><<<grid, kThreads, 0, s>>>(a, nkb, vec);
  else
    fp8_quant_squares_kernel<T, CODE, 0><<<grid, kThreads, 0, s>>>(a, nkb, vec);
  return cudaGetLastError();
}
template <int CODE, int T>
cudaError_t dequant_of(const Fp8DequantArgs& a, cudaStream_t s) {
  const int64_t nvec = ceil_div(a.cols, 16);
  const unsigned grid = (unsigned)ceil_div(nvec * a.rows, kThreads);
  const bool vin = aligned16(a.q, a.ldq), vout = aligned16(a.out, a.cols * (int64_t)sizeof(typename Elem<T>::type));
  fp8_dequant_kernel<CODE, T><<<grid, kThreads, 0, s>>>(a, nvec, vin, vout);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_fp8_quant_rows(const Fp8QuantArgs& a, int x_type, int code, cudaStream_t s) {
  const bool e4 = code == F64E_E4M3;
  switch (x_type) {
    case F64E_F32: return e4 ? rows_of<F64E_F32, F64E_E4M3>(a, s) : rows_of<F64E_F32, F64E_E5M2>(a, s);
    case F64E_F16: return e4 ? rows_of<F64E_F16, F64E_E4M3>(a, s) : rows_of<F64E_F16, F64E_E5M2>(a, s);
    default: return e4 ? rows_of<F64E_BF16, F64E_E4M3>(a, s) : rows_of<F64E_BF16, F64E_E5M2>(a, s);
  }
}

cudaError_t launch_fp8_quant_squares(const Fp8QuantArgs& a, int x_type, int code, int tile, cudaStream_t s) {
  const bool e4 = code == F64E_E4M3;
  switch (x_type) {
    case F64E_F32: return e4 ? squares_of<F64E_F32, F64E_E4M3>(a, tile, s) : squares_of<F64E_F32, F64E_E5M2>(a, tile, s);
    case F64E_F16: return e4 ? squares_of<F64E_F16, F64E_E4M3>(a, tile, s) : squares_of<F64E_F16, F64E_E5M2>(a, tile, s);
    default: return e4 ? squares_of<F64E_BF16, F64E_E4M3>(a, tile, s) : squares_of<F64E_BF16, F64E_E5M2>(a, tile, s);
  }
}

cudaError_t launch_fp8_dequant(const Fp8DequantArgs& a, int code, int out_type, cudaStream_t s) {
  const bool e4 = code == F64E_E4M3;
  switch (out_type) {
    case F64E_F32: return e4 ? dequant_of<F64E_E4M3, F64E_F32>(a, s) : dequant_of<F64E_E5M2, F64E_F32>(a, s);
    case F64E_F16: return e4 ? dequant_of<F64E_E4M3, F64E_F16>(a, s) : dequant_of<F64E_E5M2, F64E_F16>(a, s);
    default: return e4 ? dequant_of<F64E_E4M3, F64E_BF16>(a, s) : dequant_of<F64E_E5M2, F64E_BF16>(a, s);
  }
}

}  // namespace f64e
