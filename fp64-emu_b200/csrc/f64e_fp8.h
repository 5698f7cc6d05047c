// Host-side launchers of the 8-bit floating-point operators (block
// quantisation, products of block-scaled codes).  All launches go to the
// caller's stream; none allocates memory.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace f64e {

// Launch with programmatic stream serialization (launch_wait, launch_next in
// f64e_fp8.cuh) and, where cluster > 0, in clusters.
template <typename... P, typename... A>
cudaError_t fp8_launch(void (*kernel)(P...), unsigned grid, unsigned block, size_t smem, unsigned cluster,
                       cudaStream_t s, A... args) {
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3(block, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 0 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}

constexpr int kFp8Block = 128;  // values that share one scale

// ---- quantisation (f64e_fp8_quant.cu) ----
struct Fp8QuantArgs {
  const void* x;        // [rows, cols], row pitch ldx elements
  int64_t rows, cols, ldx;
  uint8_t* q;           // codes [rows][ldq]: blocks along the row (or square blocks)
  uint8_t* s;           // scales [rows][ceil(cols / 128)], or [ceil(rows / 128)][ceil(cols / 128)]
  uint8_t* qc;          // codes [rows][ldq]: blocks along the column
  uint8_t* sc;          // scales [ceil(rows / 128)][cols]
  int64_t ldq;          // row pitch of q and qc: a multiple of 16, at least cols
  int64_t ldt;          // not 0: qc holds the column codes transposed, [cols][ldt]
};
// x_type F64E_F32 / F16 / BF16, code F64E_E4M3 / E5M2.
cudaError_t launch_fp8_quant_rows(const Fp8QuantArgs& a, int x_type, int code, cudaStream_t s);
// 128 x 128 squares held in registers: tile != 0 writes q / s with one scale
// per square; otherwise qc / sc, and q / s too when q is not null (only then
// may qc be transposed).
cudaError_t launch_fp8_quant_squares(const Fp8QuantArgs& a, int x_type, int code, int tile, cudaStream_t s);

struct Fp8DequantArgs {
  const uint8_t* q;
  const uint8_t* s;
  int64_t rows, cols, ldq;
  int64_t s_row, s_col;   // scale strides (bytes) per row block and per column block
  int blocks;             // F64E_BLOCKS_*
  void* out;              // [rows][cols], contiguous
};
cudaError_t launch_fp8_dequant(const Fp8DequantArgs& a, int code, int out_type, cudaStream_t s);

// ---- products (f64e_fp8_gemm.cu) ----
// One operand as the product sees it: `rows` output rows (or columns) by K
// contracted values.  kmajor: codes [rows][ld], else [K][ld].  The scale of
// (row r, contraction block kb) is s[(r >> s_shift) * s_row + kb * s_kb].
enum { kScaleBytes = 0, kScaleWords = 1, kScaleRows = 2, kScaleTile = 3 };
struct Fp8Operand {
  const uint8_t* q;
  int64_t ld;
  const uint8_t* s;
  int64_t s_row, s_kb;
  int s_shift;   // 0, or 7: one scale for 128 rows
  int s_mode;    // how the products' kernels gather them (fp8_scale_mode)
  int code;
  int kmajor;
};
struct Fp8GemmArgs {
  Fp8Operand a, b;
  int64_t M, N, K;
  void* out;      // [M][ldo]
  int64_t ldo;
  int out_type;
  uint64_t wait_limit_ns;
  int sms;
};
// Scratch bytes the product needs (0: none).
int64_t fp8_gemm_workspace(const Fp8GemmArgs& g);
cudaError_t launch_fp8_gemm(const Fp8GemmArgs& g, void* workspace, cudaStream_t s);
// The same product on one-CTA tiles whose K is split over a cluster
// (f64e_fp8_split.cu), for few rows or columns.
// Launches it unless the estimate of its cycles exceeds other_cost, or the
// smaller operand is not K-major; done says which.
cudaError_t launch_fp8_split(const Fp8GemmArgs& g, int64_t other_cost, bool* done, cudaStream_t s);
// y = quantised(x) @ w^T for a few rows of x (at most kFusedRows) of up to
// kFusedMaxK values (what TMEM holds of the parts of 32-bit sums, over the
// largest split): x is quantised in row blocks by the CTAs that contract it.
constexpr int kFusedRows = 16;
constexpr int64_t kFusedMaxK = 442368;
struct Fp8LinearArgs {
  Fp8GemmArgs g;   // b: the weights; a unused
  const void* x;   // [M][ldx] of type x_type; the output has the same type
  int64_t ldx;
  int x_type;
};
cudaError_t launch_fp8_linear_few(const Fp8LinearArgs& a, cudaStream_t s);

// Host helpers shared by the two.
bool fp8_encode_2d(CUtensorMap* map, CUtensorMapDataType type, void* base, int64_t inner, int64_t outer,
                   int64_t pitch_bytes, int box_inner, int box_outer, CUtensorMapSwizzle swizzle);
bool fp8_encode_codes(CUtensorMap* map, const Fp8Operand& o, int64_t rows, int64_t K, int box_rows);
// whole_squares: tiles start at multiples of 128 rows.
int fp8_scale_mode(const Fp8Operand& o, int64_t rows, bool whole_squares);

// The device's status words of these products, cleared by the read; synchronizes.
cudaError_t read_fp8_split_status(int* status, cudaStream_t s);
cudaError_t read_fp8_status(int* status, cudaStream_t s);
// One thread runs a bounded wait out, which records its site in the pairs' word
// (kWaitSelfTest) or the split products' (kWaitSelfTestSplit).
cudaError_t launch_fp8_wait_selftest(uint64_t limit_ns, cudaStream_t s);
cudaError_t launch_fp8_split_wait_selftest(uint64_t limit_ns, cudaStream_t s);

}  // namespace f64e
