// Block quantisation to 8-bit floating point and back.
//
// All three kernels are bound by memory: quantising reads e bytes a value (e =
// 2 or 4) and writes 1 + 1/128, or twice that for row and column blocks from
// one read; restoring is the reverse.  An SM must then handle about 6 values a
// cycle, some 16 instructions a value at most, so a thread works on sixteen
// neighbouring values at a time: one or two loads, packed magnitudes, and the
// scale's arithmetic shared by all of them.
// Where rows do not start on 16-byte boundaries (VEC = false) a quantising
// thread takes every eighth value instead, so that neighbouring lanes still
// touch neighbouring elements, and codes are put in order in shared memory.
#include "f64e_fp8.cuh"
#include "f64e_fp8.h"

namespace f64e {

namespace {

constexpr int kThreads = 256;

// Lanes l = 0..7 hold one 128-value row block: the maximum over them.
__device__ __forceinline__ float max_over_block(float m) {
#pragma unroll
  for (int o = 4; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
  return m;
}
// Exponent of the row block these lanes hold; its infinities are NaN after.
template <int T, int CODE>
__device__ __forceinline__ int row_exponent(uint32_t* w) {
  float m = max_over_block(max16<T>(w));
  if (__any_sync(0xFFFFFFFFu, is_inf(m))) {
    infs_to_nan<T>(w);
    m = max_over_block(max16<T>(w));
  }
  return scale_exponent<CODE>(m);
}

// Column of a thread's i-th value within its 128, from lane l of eight.
template <bool VEC>
__device__ __forceinline__ int col_of(int l, int i) {
  return VEC ? l * 16 + i : i * 8 + l;
}
template <int T, bool VEC>
__device__ __forceinline__ void load_row(const typename Elem<T>::type* row, int l, int64_t n, bool wide, uint32_t* w) {
  if (VEC && n >= (l + 1) * 16)
    load16<T>(row + l * 16, wide, w);
  else
    load16_some<T>(row + (VEC ? l * 16 : l), VEC ? 1 : 8, n - (VEC ? l * 16 : l), w);
}

// --------------------------------------------------------------- rows ----
// A warp covers four neighbouring blocks (512 columns) of four rows.
constexpr int kRowPasses = 4;

template <int T, int CODE, bool VEC>
__global__ void __launch_bounds__(kThreads) fp8_quant_rows_kernel(const Fp8QuantArgs a, int nkb, int ngroups,
                                                                  bool wide) {
  __shared__ __align__(16) uint8_t s_codes[VEC ? 1 : kThreads / 32][VEC ? 16 : 512];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane & 7;
  const int kb = (int)(blockIdx.x % ngroups) * 4 + (lane >> 3);
  const int64_t row0 = ((int64_t)(blockIdx.x / ngroups) * (kThreads / 32) + warp) * kRowPasses;
  const int64_t col = (int64_t)kb * kFp8Block, padded = (a.cols + 15) & ~(int64_t)15;
  const typename Elem<T>::type* x = static_cast<const typename Elem<T>::type*>(a.x) + row0 * a.ldx + col;
  uint8_t* q = a.q + row0 * a.ldq + col + l * 16;
  uint8_t* s = a.s + row0 * nkb + kb;
  uint32_t w[kRowPasses][Elem<T>::kWords];
  launch_next();
  launch_wait();
#pragma unroll
  for (int u = 0; u < kRowPasses; u++)
    load_row<T, VEC>(x + u * a.ldx, l, row0 + u < a.rows ? a.cols - col : 0, wide, w[u]);
#pragma unroll
  for (int u = 0; u < kRowPasses; u++) {
    const int e = row_exponent<T, CODE>(w[u]);
    const float r = inverse_scale(e);
    uint32_t c[8];
    codes16<T, CODE>(w[u], [&](int) { return r; }, c);
    uint4 v;
    if (VEC) {
      v = row_of_codes(c);
    } else {
      uint8_t* st = s_codes[warp % (VEC ? 1 : kThreads / 32)] + (lane >> 3) * (VEC ? 0 : 128);
#pragma unroll
      for (int i = 0; i < 16; i++) st[(VEC ? 0 : i * 8) + l] = (uint8_t)(c[i >> 1] >> (8 * (i & 1)));
      __syncwarp();
      v = *reinterpret_cast<const uint4*>(st + l * (VEC ? 0 : 16));
      __syncwarp();
    }
    if (row0 + u < a.rows && kb < nkb) {
      if (col + l * 16 < padded) *reinterpret_cast<uint4*>(q + u * a.ldq) = v;
      if (l == 0) s[(int64_t)u * nkb] = (uint8_t)(e + 127);
    }
  }
}

// ------------------------------------------------------------ squares ----
// A CTA keeps a 128 x 128 square in registers, a thread sixteen columns of the
// four rows 4 g .. 4 g + 3, so one read serves both block directions.  Column
// maxima: packed over the thread's rows and the four threads of a warp that
// share its columns, then over the eight warps in shared memory, where one
// thread a column turns them into the scale.
// Transposed codes leave through shared memory: a thread's four rows of a
// column are one 32-bit word there.
enum { kCols = 0, kRowsCols = 1, kTile = 2, kRowsColsT = 3 };

struct SquareSmem {
  float max[kThreads / 32][kFp8Block];
  float inv[kFp8Block];
};

// Row-major codes of the thread's four rows, codes(u, c) giving those of row u.
// VEC = false puts them in order in `tile` (the whole CTA calls it).
template <bool VEC, typename F>
__device__ __forceinline__ void store_rows(uint8_t* q, int64_t ldq, int64_t rows, int64_t row0, int64_t col,
                                           int64_t padded, int g, int l, uint8_t* tile, F codes) {
  uint32_t c[8];
  if (VEC) {
    uint8_t* p = q + (row0 + 4 * g) * ldq + col + l * 16;
#pragma unroll
    for (int u = 0; u < 4; u++) {
      codes(u, c);
      if (row0 + 4 * g + u < rows && col + l * 16 < padded) *reinterpret_cast<uint4*>(p + u * ldq) = row_of_codes(c);
    }
  } else {
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 4; u++) {
      codes(u, c);
#pragma unroll
      for (int i = 0; i < 16; i++) tile[(4 * g + u) * 128 + i * 8 + l] = (uint8_t)(c[i >> 1] >> (8 * (i & 1)));
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const int r = u * 32 + (threadIdx.x >> 3);
      if (row0 + r < rows && col + l * 16 < padded)
        *reinterpret_cast<uint4*>(q + (row0 + r) * ldq + col + l * 16) =
            *reinterpret_cast<const uint4*>(tile + r * 128 + l * 16);
    }
  }
}
// The same codes with rows contiguous: qt[col][row], pitch ldt.
template <bool VEC>
__device__ __forceinline__ void store_columns(uint8_t* qt, int64_t ldt, int64_t cols, int64_t padded_rows, int64_t row0,
                                              int64_t col, int g, int l, uint8_t* tile, const uint32_t (&c)[4][8]) {
  uint32_t* words = reinterpret_cast<uint32_t*>(tile);   // [128 columns][32 words], words XORed by 4 x (column / 16)
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 8; k++) {
    const uint32_t x = __byte_perm(c[0][k], c[1][k], 0x5140), y = __byte_perm(c[2][k], c[3][k], 0x5140);
    const int c0 = col_of<VEC>(l, 2 * k), c1 = col_of<VEC>(l, 2 * k + 1);
    words[c0 * 32 + (g ^ ((c0 >> 4) << 2))] = __byte_perm(x, y, 0x5410);
    words[c1 * 32 + (g ^ ((c1 >> 4) << 2))] = __byte_perm(x, y, 0x7632);
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < 4; u++) {
    const int cc = u * 32 + (threadIdx.x >> 3), ch = threadIdx.x & 7;
    if (col + cc < cols && row0 + ch * 16 < padded_rows)
      *reinterpret_cast<uint4*>(qt + (col + cc) * ldt + row0 + ch * 16) =
          *reinterpret_cast<const uint4*>(tile + cc * 128 + ((ch ^ (cc >> 4)) << 4));
  }
}

template <int T, int CODE, int MODE, bool VEC>
__global__ void __launch_bounds__(kThreads, T == F64E_F32 || MODE == kRowsCols ? 2 : MODE == kRowsColsT ? 3 : 4)
    fp8_quant_squares_kernel(const Fp8QuantArgs a, int nkb, bool wide) {
  using E = Elem<T>;
  __shared__ SquareSmem sm;
  __shared__ __align__(16) uint8_t tile[!VEC || MODE == kRowsColsT ? 128 * 128 : 16];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane & 7, g = threadIdx.x >> 3;
  const int kb = (int)(blockIdx.x % nkb);
  const int64_t rb = blockIdx.x / nkb, row0 = rb * kFp8Block, col = (int64_t)kb * kFp8Block;
  const int64_t padded = (a.cols + 15) & ~(int64_t)15;
  const typename E::type* x = static_cast<const typename E::type*>(a.x) + (row0 + 4 * g) * a.ldx + col;
  uint32_t w[4][E::kWords];
  launch_next();
  launch_wait();
#pragma unroll
  for (int u = 0; u < 4; u++)
    load_row<T, VEC>(x + u * a.ldx, l, row0 + 4 * g + u < a.rows ? a.cols - col : 0, wide, w[u]);

  // Rows are unpacked one after the other, each time anew: all 64 values kept
  // as floats would leave an SM one CTA instead of three.
  auto one_row = [](uint32_t (&r)[E::kWords]) {
#pragma unroll
    for (int k = 0; k < E::kWords; k++) asm volatile("" : "+r"(r[k])::"memory");
  };

  if (MODE == kTile) {
    float m;
    while (true) {   // a second time after infinities
      m = 0.f;
#pragma unroll
      for (int u = 0; u < 4; u++) m = fmaxf(m, max16<T>(w[u]));
#pragma unroll
      for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
      if (lane == 0) sm.inv[warp] = m;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kThreads / 32; i++) m = fmaxf(m, sm.inv[i]);
      if (!is_inf(m)) break;
      __syncthreads();
#pragma unroll
      for (int u = 0; u < 4; u++) infs_to_nan<T>(w[u]);
    }
    const int e = scale_exponent<CODE>(m);
    const float r = inverse_scale(e);
    store_rows<VEC>(a.q, a.ldq, a.rows, row0, col, padded, g, l, tile, [&](int u, uint32_t* c) {
      one_row(w[u]);
      codes16<T, CODE>(w[u], [&](int) { return r; }, c);
    });
    if (threadIdx.x == 0) a.s[rb * nkb + kb] = (uint8_t)(e + 127);
    return;
  }

  if (MODE == kRowsCols || MODE == kRowsColsT) {
    store_rows<VEC>(a.q, a.ldq, a.rows, row0, col, padded, g, l, tile, [&](int u, uint32_t* c) {
      one_row(w[u]);
      const int e = row_exponent<T, CODE>(w[u]);
      const float r = inverse_scale(e);
      codes16<T, CODE>(w[u], [&](int) { return r; }, c);
      const int64_t row = row0 + 4 * g + u;
      if (l == 0 && row < a.rows) a.s[row * nkb + kb] = (uint8_t)(e + 127);
    });
  }

  while (true) {   // a second time after infinities (the rows above left none)
    typename E::mag m[E::kWords];
#pragma unroll
    for (int k = 0; k < E::kWords; k++) {
      m[k] = E::zero();
#pragma unroll
      for (int u = 0; u < 4; u++) m[k] = E::max_mag(m[k], w[u][k]);
      m[k] = E::max_of(m[k], E::shfl(m[k], 8));
      m[k] = E::max_of(m[k], E::shfl(m[k], 16));
    }
#pragma unroll
    for (int k = 0; k < E::kWords; k++)
      if ((lane >> 3) == k * 4 / E::kWords) {   // each of the four writes a quarter
        if constexpr (T == F64E_F32) {
          sm.max[warp][col_of<VEC>(l, k)] = m[k];
        } else {
          sm.max[warp][col_of<VEC>(l, 2 * k)] = E::lo(m[k]);
          sm.max[warp][col_of<VEC>(l, 2 * k + 1)] = E::hi(m[k]);
        }
      }
    __syncthreads();
    float top = 0.f;
    if (threadIdx.x < kFp8Block) {
#pragma unroll
      for (int i = 0; i < kThreads / 32; i++) top = fmaxf(top, sm.max[i][threadIdx.x]);
    }
    if (MODE == kCols && __syncthreads_or(is_inf(top))) {
#pragma unroll
      for (int u = 0; u < 4; u++) infs_to_nan<T>(w[u]);
      continue;
    }
    if (threadIdx.x < kFp8Block) {
      const int e = scale_exponent<CODE>(top);
      sm.inv[threadIdx.x] = inverse_scale(e);
      if (col + threadIdx.x < a.cols) a.sc[rb * a.cols + col + threadIdx.x] = (uint8_t)(e + 127);
    }
    __syncthreads();
    break;
  }
  float r[16];
  if (VEC) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float4 v = *reinterpret_cast<const float4*>(&sm.inv[l * 16 + 4 * i]);
      r[4 * i] = v.x;
      r[4 * i + 1] = v.y;
      r[4 * i + 2] = v.z;
      r[4 * i + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; i++) r[i] = sm.inv[i * 8 + l];
  }
  auto codes = [&](int u, uint32_t* c) {
    one_row(w[u]);
    codes16<T, CODE>(w[u], [&](int i) { return r[i]; }, c);
  };
  if (MODE == kRowsColsT) {
    uint32_t c[4][8];
#pragma unroll
    for (int u = 0; u < 4; u++) codes(u, c[u]);
    store_columns<VEC>(a.qc, a.ldt, a.cols, (a.rows + 15) & ~(int64_t)15, row0, col, g, l, tile, c);
  } else {
    store_rows<VEC>(a.qc, a.ldq, a.rows, row0, col, padded, g, l, tile, codes);
  }
}

// --------------------------------------------------------- dequantise ----
// Sixteen columns of up to four rows of one row block a thread (rows g, g +
// 32, .. of the 128), so column scales are read once for the four.
template <int CODE, int T>
__global__ void __launch_bounds__(kThreads) fp8_dequant_kernel(const Fp8DequantArgs a, int ncb, bool wide) {
  const int l = threadIdx.x & 7, g = threadIdx.x >> 3;
  const int64_t rb = blockIdx.x / ncb, cb = blockIdx.x % ncb, col = cb * kFp8Block + l * 16;
  const int64_t n = a.cols - col;   // columns from here on: none, some, or sixteen and more
  const uint8_t* q = a.q + (rb * kFp8Block + g) * a.ldq + col;
  uint32_t w[4][4];
  launch_next();
  launch_wait();
  if (n <= 0) return;
#pragma unroll
  for (int u = 0; u < 4; u++) {
    w[u][0] = w[u][1] = w[u][2] = w[u][3] = 0;
    if (rb * kFp8Block + g + 32 * u >= a.rows) continue;
    const uint8_t* p = q + (int64_t)(32 * u) * a.ldq;
    if (n >= 16) {
      const uint4 v = *reinterpret_cast<const uint4*>(p);
      w[u][0] = v.x;
      w[u][1] = v.y;
      w[u][2] = v.z;
      w[u][3] = v.w;
    } else {
#pragma unroll
      for (int i = 0; i < 16; i++)
        if (i < n) w[u][i >> 2] |= (uint32_t)p[i] << (8 * (i & 3));
    }
  }
  const bool per_col = a.blocks == F64E_BLOCKS_COL;
  float sc[16];
  if (per_col) {
    const uint8_t* s = a.s + rb * a.s_row + col * a.s_col;
#pragma unroll
    for (int i = 0; i < 16; i++) sc[i] = i < n ? scale_of_byte(s[i * a.s_col]) : 0.f;
  }
#pragma unroll
  for (int u = 0; u < 4; u++) {
    const int64_t row = rb * kFp8Block + g + 32 * u;
    if (row >= a.rows) break;
    if (!per_col) {
      const float one = scale_of_byte(a.s[(a.blocks == F64E_BLOCKS_ROW ? row : rb) * a.s_row + cb * a.s_col]);
#pragma unroll
      for (int i = 0; i < 16; i++) sc[i] = one;
    }
    float f[16];
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float2 v = values2<CODE>((w[u][i >> 1] >> (16 * (i & 1))) & 0xFFFFu);
      f[2 * i] = v.x * sc[2 * i];
      f[2 * i + 1] = v.y * sc[2 * i + 1];
    }
    typename Elem<T>::type* o = static_cast<typename Elem<T>::type*>(a.out) + row * a.cols + col;
    if (n >= 16) {
      uint32_t b[Elem<T>::kWords];
#pragma unroll
      for (int i = 0; i < Elem<T>::kWords; i++)
        b[i] = T == F64E_F32 ? Elem<T>::bits(f[i]) : Elem<T>::pack(f[(2 * i) & 15], f[(2 * i + 1) & 15]);
      uint32_t* ow = reinterpret_cast<uint32_t*>(o);
      if (wide) {
#pragma unroll
        for (int i = 0; i < Elem<T>::kWords; i += 8)
          asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(ow + i), "r"(b[i]), "r"(b[i + 1]),
                       "r"(b[i + 2]), "r"(b[i + 3]), "r"(b[i + 4]), "r"(b[i + 5]), "r"(b[i + 6]), "r"(b[i + 7])
                       : "memory");
      } else {
#pragma unroll
        for (int i = 0; i < Elem<T>::kWords; i += 4)
          *reinterpret_cast<uint4*>(ow + i) = make_uint4(b[i], b[i + 1], b[i + 2], b[i + 3]);
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
}

// Rows that start anywhere: a warp writes 32 neighbouring elements of a row at
// a time (thread: columns lane, lane + 32, .. of sixteen rows).
template <int CODE, int T>
__global__ void __launch_bounds__(kThreads) fp8_dequant_any_kernel(const Fp8DequantArgs a, int ncb) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t rb = blockIdx.x / ncb, cb = blockIdx.x % ncb, col = cb * kFp8Block + lane;
  const int64_t row0 = rb * kFp8Block + warp * 16;
  const int n = (int)min((int64_t)16, a.rows - row0);
  launch_next();
  launch_wait();
  const bool per_col = a.blocks == F64E_BLOCKS_COL;
  float sc[4];
#pragma unroll
  for (int i = 0; i < 4; i++)
    sc[i] = per_col && col + 32 * i < a.cols ? scale_of_byte(a.s[rb * a.s_row + (col + 32 * i) * a.s_col]) : 0.f;
  constexpr int U = 8;   // rows read before they are written: loads do not pass stores
  const uint8_t* q = a.q + row0 * a.ldq + col;
  typename Elem<T>::type* o = static_cast<typename Elem<T>::type*>(a.out) + row0 * a.cols + col;
  bool there[4];
#pragma unroll
  for (int i = 0; i < 4; i++) there[i] = col + 32 * i < a.cols;
  for (int u0 = 0; u0 < n; u0 += U) {
    uint32_t c[U][4];
    float one[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const bool row = u0 + u < n;
      one[u] = per_col || !row ? 0.f
                               : scale_of_byte(a.s[(a.blocks == F64E_BLOCKS_ROW ? row0 + u0 + u : rb) * a.s_row + cb * a.s_col]);
#pragma unroll
      for (int i = 0; i < 4; i++) c[u][i] = row && there[i] ? q[32 * i] : 0;
      q += a.ldq;
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (u0 + u >= n) break;
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (there[i]) {
          const float f = values2<CODE>(c[u][i]).x * (per_col ? sc[i] : one[u]);
          if (T == F64E_F32)
            reinterpret_cast<uint32_t*>(o)[32 * i] = Elem<T>::bits(f);
          else
            reinterpret_cast<uint16_t*>(o)[32 * i] = (uint16_t)Elem<T>::bits(f);
        }
      o += a.cols;
    }
  }
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
bool aligned(const void* p, int64_t pitch_bytes, int64_t to) {
  return reinterpret_cast<uintptr_t>(p) % to == 0 && pitch_bytes % to == 0;
}

template <int T, int CODE>
cudaError_t rows_of(const Fp8QuantArgs& a, cudaStream_t s) {
  const int nkb = (int)ceil_div(a.cols, kFp8Block), ng = (nkb + 3) / 4;
  const unsigned grid = (unsigned)(ng * ceil_div(a.rows, kThreads / 32 * kRowPasses));
  const int64_t pitch = a.ldx * (int64_t)sizeof(typename Elem<T>::type);
  const bool wide = aligned(a.x, pitch, 32);
  if (aligned(a.x, pitch, 16))
    return fp8_launch(fp8_quant_rows_kernel<T, CODE, true>, grid, kThreads, 0, 0, s, a, nkb, ng, wide);
  return fp8_launch(fp8_quant_rows_kernel<T, CODE, false>, grid, kThreads, 0, 0, s, a, nkb, ng, wide);
}
template <int T, int CODE, int MODE>
cudaError_t squares_mode(const Fp8QuantArgs& a, cudaStream_t s) {
  const int nkb = (int)ceil_div(a.cols, kFp8Block);
  const unsigned grid = (unsigned)(nkb * ceil_div(a.rows, kFp8Block));
  const int64_t pitch = a.ldx * (int64_t)sizeof(typename Elem<T>::type);
  const bool wide = aligned(a.x, pitch, 32);
  if (aligned(a.x, pitch, 16))
    return fp8_launch(fp8_quant_squares_kernel<T, CODE, MODE, true>, grid, kThreads, 0, 0, s, a, nkb, wide);
  return fp8_launch(fp8_quant_squares_kernel<T, CODE, MODE, false>, grid, kThreads, 0, 0, s, a, nkb, wide);
}
template <int T, int CODE>
cudaError_t squares_of(const Fp8QuantArgs& a, int tile, cudaStream_t s) {
  if (tile) return squares_mode<T, CODE, kTile>(a, s);
  if (!a.q) return squares_mode<T, CODE, kCols>(a, s);
  return a.ldt ? squares_mode<T, CODE, kRowsColsT>(a, s) : squares_mode<T, CODE, kRowsCols>(a, s);
}
template <int CODE, int T>
cudaError_t dequant_of(const Fp8DequantArgs& a, cudaStream_t s) {
  const int ncb = (int)ceil_div(a.cols, kFp8Block);
  const unsigned grid = (unsigned)(ncb * ceil_div(a.rows, kFp8Block));
  const int64_t pitch = a.cols * (int64_t)sizeof(typename Elem<T>::type);
  const bool wide = aligned(a.out, pitch, 32);
  if (aligned(a.q, a.ldq, 16) && aligned(a.out, pitch, 16))
    return fp8_launch(fp8_dequant_kernel<CODE, T>, grid, kThreads, 0, 0, s, a, ncb, wide);
  return fp8_launch(fp8_dequant_any_kernel<CODE, T>, grid, kThreads, 0, 0, s, a, ncb);
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
