// C ABI of the 8-bit floating-point operators (declared in include/f64e.h).
#include <algorithm>

#include "f64e.h"
#include "f64e_fp8.h"

namespace f64e {
int report_error(int code, const char* msg);
int begin_call();
int device_sms(int* sms);
uint64_t wait_limit_ns();
}  // namespace f64e

using namespace f64e;

namespace {

constexpr int64_t kMaxDim = (int64_t)1 << 30;   // tile coordinates are 32-bit

int bad(const char* msg) { return report_error(F64E_ERR_ARGUMENT, msg); }
int cuda_error(cudaError_t e) { return report_error(F64E_ERR_CUDA, cudaGetErrorString(e)); }
int64_t round_up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }
int64_t blocks_of(int64_t n) { return (n + kFp8Block - 1) / kFp8Block; }

const char* check_types(int x_type, int code) {
  if (x_type != F64E_F32 && x_type != F64E_F16 && x_type != F64E_BF16) return "fp8: element type must be F32, F16 or BF16";
  if (code != F64E_E4M3 && code != F64E_E5M2) return "fp8: code must be E4M3 or E5M2";
  return nullptr;
}

const char* check_matrix(int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 0) return "fp8: negative dimension";
  if (rows > kMaxDim || cols > kMaxDim) return "fp8: dimension too large";
  // a CTA for 32 x 512 or 128 x 128 values
  if (blocks_of(rows) * blocks_of(cols) > 0x7FFFFFFF || (rows + 31) / 32 * ((cols + 511) / 512) > 0x7FFFFFFF)
    return "fp8: matrix too large";
  return nullptr;
}

const char* check_codes(const void* q, int64_t ldq, int64_t cols) {
  if (ldq < cols) return "fp8: row pitch of the codes is below their columns";
  if (ldq % 16 != 0 || (reinterpret_cast<uintptr_t>(q) & 15)) return "fp8: codes need 16-byte aligned rows";
  return nullptr;
}

// Kernels read and write whole elements: an address inside one would fault.
const char* check_elements(const void* x, int type) {
  return reinterpret_cast<uintptr_t>(x) % (type == F64E_F32 ? 4 : 2) ? "fp8: values are not aligned to their type" : nullptr;
}

// Sizes, types and pitches of a product; fills everything but the pointers.
int check_problem(const f64e_fp8_problem* p, Fp8GemmArgs* g) {
  if (!p) return bad("fp8: null problem");
  if (const char* m = check_types(p->out_type, p->a.code)) return bad(m);
  if (const char* m = check_types(p->out_type, p->b.code)) return bad(m);
  if (p->M < 0 || p->N < 0 || p->K < 0) return bad("fp8: negative dimension");
  if (p->M > kMaxDim || p->N > kMaxDim || p->K > kMaxDim) return bad("fp8: dimension too large");
  if (blocks_of(p->M) * blocks_of(p->N) > 0x7FFFFFFF / 2 || blocks_of(p->K) * blocks_of(std::min(p->M, p->N)) > 0x7FFFFFFF)
    return bad("fp8: product too large");
  if (p->ldo < p->N) return bad("fp8: row pitch of the output is below its columns");
  const f64e_fp8_operand* in[2] = {&p->a, &p->b};
  Fp8Operand* o[2] = {&g->a, &g->b};
  const int64_t rows[2] = {p->M, p->N};
  for (int i = 0; i < 2; i++) {
    if (in[i]->tile != 0 && in[i]->tile != 1) return bad("fp8: tile must be 0 or 1");
    if (in[i]->k_major != 0 && in[i]->k_major != 1) return bad("fp8: k_major must be 0 or 1");
    if (const char* m = check_codes(nullptr, in[i]->ld, in[i]->k_major ? p->K : rows[i])) return bad(m);
    o[i]->kmajor = in[i]->k_major;
    o[i]->ld = in[i]->ld;
    o[i]->s_row = in[i]->scale_row;
    o[i]->s_kb = in[i]->scale_block;
    o[i]->s_shift = in[i]->tile ? 7 : 0;
    o[i]->code = in[i]->code;
  }
  g->M = p->M;
  g->N = p->N;
  g->K = p->K;
  g->ldo = p->ldo;
  g->out_type = p->out_type;
  return F64E_OK;
}

}  // namespace

extern "C" {

int f64e_fp8_quantize(const void* x, int32_t x_type, int64_t rows, int64_t cols, int64_t ldx, int32_t blocks,
                      int32_t code, void* q, int64_t ldq, void* scale, void* stream) {
  begin_call();
  if (const char* m = check_types(x_type, code)) return bad(m);
  if (blocks != F64E_BLOCKS_ROW && blocks != F64E_BLOCKS_COL && blocks != F64E_BLOCKS_TILE)
    return bad("fp8: blocks must be ROW, COL or TILE");
  if (const char* m = check_matrix(rows, cols)) return bad(m);
  if (rows == 0 || cols == 0) return F64E_OK;
  if (!x || !q || !scale) return bad("fp8: null pointer");
  if (ldx < cols) return bad("fp8: row pitch of x is below its columns");
  if (const char* m = check_elements(x, x_type)) return bad(m);
  if (const char* m = check_codes(q, ldq, cols)) return bad(m);
  int sms = 0;
  if (const int rc = device_sms(&sms)) return rc;
  Fp8QuantArgs a{};
  a.x = x;
  a.rows = rows;
  a.cols = cols;
  a.ldx = ldx;
  a.ldq = ldq;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (blocks == F64E_BLOCKS_COL) {
    a.qc = static_cast<uint8_t*>(q);
    a.sc = static_cast<uint8_t*>(scale);
    e = launch_fp8_quant_squares(a, x_type, code, 0, s);
  } else {
    a.q = static_cast<uint8_t*>(q);
    a.s = static_cast<uint8_t*>(scale);
    e = blocks == F64E_BLOCKS_ROW ? launch_fp8_quant_rows(a, x_type, code, s)
                                  : launch_fp8_quant_squares(a, x_type, code, 1, s);
  }
  return e == cudaSuccess ? F64E_OK : cuda_error(e);
}

int f64e_fp8_quantize_both(const void* x, int32_t x_type, int64_t rows, int64_t cols, int64_t ldx, int32_t code,
                           void* q_row, void* scale_row, int64_t ldq, void* q_col, void* scale_col, int32_t transposed,
                           int64_t ld_col, void* stream) {
  begin_call();
  if (const char* m = check_types(x_type, code)) return bad(m);
  if (const char* m = check_matrix(rows, cols)) return bad(m);
  if (rows == 0 || cols == 0) return F64E_OK;
  if (!x || !q_row || !scale_row || !q_col || !scale_col) return bad("fp8: null pointer");
  if (ldx < cols) return bad("fp8: row pitch of x is below its columns");
  if (const char* m = check_elements(x, x_type)) return bad(m);
  if (const char* m = check_codes(q_row, ldq, cols)) return bad(m);
  if (transposed != 0 && transposed != 1) return bad("fp8: transposed must be 0 or 1");
  if (const char* m = check_codes(q_col, ld_col, transposed ? rows : cols)) return bad(m);
  if (!transposed && ld_col != ldq) return bad("fp8: row and column codes need the same pitch");
  int sms = 0;
  if (const int rc = device_sms(&sms)) return rc;
  Fp8QuantArgs a{};
  a.x = x;
  a.rows = rows;
  a.cols = cols;
  a.ldx = ldx;
  a.ldq = ldq;
  a.ldt = transposed ? ld_col : 0;
  a.q = static_cast<uint8_t*>(q_row);
  a.s = static_cast<uint8_t*>(scale_row);
  a.qc = static_cast<uint8_t*>(q_col);
  a.sc = static_cast<uint8_t*>(scale_col);
  const cudaError_t e = launch_fp8_quant_squares(a, x_type, code, 0, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? F64E_OK : cuda_error(e);
}

int f64e_fp8_dequantize(const void* q, int32_t code, int64_t rows, int64_t cols, int64_t ldq, int32_t blocks,
                        const void* scale, int64_t scale_row, int64_t scale_col, void* out, int32_t out_type,
                        void* stream) {
  begin_call();
  if (const char* m = check_types(out_type, code)) return bad(m);
  if (blocks != F64E_BLOCKS_ROW && blocks != F64E_BLOCKS_COL && blocks != F64E_BLOCKS_TILE)
    return bad("fp8: blocks must be ROW, COL or TILE");
  if (const char* m = check_matrix(rows, cols)) return bad(m);
  if (rows == 0 || cols == 0) return F64E_OK;
  if (!q || !scale || !out) return bad("fp8: null pointer");
  if (ldq < cols) return bad("fp8: row pitch of the codes is below their columns");
  if (const char* m = check_elements(out, out_type)) return bad(m);
  int sms = 0;
  if (const int rc = device_sms(&sms)) return rc;
  Fp8DequantArgs a{};
  a.q = static_cast<const uint8_t*>(q);
  a.s = static_cast<const uint8_t*>(scale);
  a.rows = rows;
  a.cols = cols;
  a.ldq = ldq;
  a.s_row = scale_row;
  a.s_col = scale_col;
  a.blocks = blocks;
  a.out = out;
  const cudaError_t e = launch_fp8_dequant(a, code, out_type, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? F64E_OK : cuda_error(e);
}

size_t f64e_fp8_workspace_size(const f64e_fp8_problem* p) {
  begin_call();
  Fp8GemmArgs g{};
  if (check_problem(p, &g)) return 0;
  return (size_t)fp8_gemm_workspace(g);
}

int f64e_fp8_gemm(const f64e_fp8_problem* p, const void* A, const void* a_scale, const void* B, const void* b_scale,
                  void* out, void* workspace, size_t workspace_bytes, void* stream) {
  begin_call();
  Fp8GemmArgs g{};
  if (const int rc = check_problem(p, &g)) return rc;
  if (p->M == 0 || p->N == 0) return F64E_OK;
  if (p->K == 0) return bad("fp8: K must be at least 1");
  if (!A || !a_scale || !B || !b_scale || !out) return bad("fp8: null pointer");
  if ((reinterpret_cast<uintptr_t>(A) & 15) || (reinterpret_cast<uintptr_t>(B) & 15))
    return bad("fp8: codes need 16-byte aligned rows");
  if (const char* m = check_elements(out, p->out_type)) return bad(m);
  g.a.q = static_cast<const uint8_t*>(A);
  g.a.s = static_cast<const uint8_t*>(a_scale);
  g.b.q = static_cast<const uint8_t*>(B);
  g.b.s = static_cast<const uint8_t*>(b_scale);
  g.out = out;
  const int64_t need = fp8_gemm_workspace(g);
  if (need > 0 && (!workspace || workspace_bytes < (size_t)need || (reinterpret_cast<uintptr_t>(workspace) & 255)))
    return report_error(F64E_ERR_WORKSPACE, "fp8: workspace missing, too small or not 256-byte aligned");
  g.wait_limit_ns = wait_limit_ns();
  if (const int rc = device_sms(&g.sms)) return rc;
  const cudaError_t e = launch_fp8_gemm(g, workspace, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? F64E_OK : cuda_error(e);
}

size_t f64e_fp8_linear_workspace_size(int64_t M, int64_t K) {
  begin_call();
  if (check_matrix(M, K)) {
    bad(check_matrix(M, K));
    return 0;
  }
  if (M <= kFusedRows && K <= kFusedMaxK) return 0;
  return (size_t)(round_up(M * round_up(K, 16), 256) + M * blocks_of(K));
}

int f64e_fp8_linear(const f64e_fp8_problem* p, const void* x, int64_t ldx, const void* w, const void* w_scale,
                    void* out, void* workspace, size_t workspace_bytes, void* stream) {
  begin_call();
  if (!p) return bad("fp8: null problem");
  f64e_fp8_problem q = *p;   // the operand a: x's codes, row blocks
  q.a.ld = round_up(std::max<int64_t>(q.K, 1), 16);
  q.a.code = F64E_E4M3;
  q.a.tile = 0;
  q.a.k_major = 1;
  q.a.scale_row = blocks_of(q.K);
  q.a.scale_block = 1;
  Fp8LinearArgs a{};
  if (const int rc = check_problem(&q, &a.g)) return rc;
  if (const char* m = check_matrix(q.M, q.K)) return bad(m);
  if (ldx < q.K) return bad("fp8: row pitch of x is below its columns");
  if (q.M == 0 || q.N == 0) return F64E_OK;
  if (q.K == 0) return bad("fp8: K must be at least 1");
  if (!x || !w || !w_scale || !out) return bad("fp8: null pointer");
  if (reinterpret_cast<uintptr_t>(w) & 15) return bad("fp8: codes need 16-byte aligned rows");
  for (const void* v : {x, static_cast<const void*>(out)})
    if (const char* m = check_elements(v, q.out_type)) return bad(m);
  if (q.M > kFusedRows || q.K > kFusedMaxK) {
    const size_t need = f64e_fp8_linear_workspace_size(q.M, q.K);
    if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255))
      return report_error(F64E_ERR_WORKSPACE, "fp8: workspace missing, too small or not 256-byte aligned");
    uint8_t* codes = static_cast<uint8_t*>(workspace);
    uint8_t* scales = codes + round_up(q.M * q.a.ld, 256);
    if (const int rc = f64e_fp8_quantize(x, q.out_type, q.M, q.K, ldx, F64E_BLOCKS_ROW, F64E_E4M3, codes, q.a.ld,
                                         scales, stream))
      return rc;
    return f64e_fp8_gemm(&q, codes, scales, w, w_scale, out, nullptr, 0, stream);
  }
  a.g.b.q = static_cast<const uint8_t*>(w);
  a.g.b.s = static_cast<const uint8_t*>(w_scale);
  a.g.out = out;
  a.g.wait_limit_ns = wait_limit_ns();
  a.x = x;
  a.ldx = ldx;
  a.x_type = q.out_type;
  if (const int rc = device_sms(&a.g.sms)) return rc;
  const cudaError_t e = launch_fp8_linear_few(a, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? F64E_OK : cuda_error(e);
}

int f64e_fp8_wait_selftest(int32_t split, uint64_t limit_ns, void* stream) {
  begin_call();
  if (split != 0 && split != 1) return bad("fp8: split must be 0 or 1");
  if (limit_ns == 0 || limit_ns > 10000000000ULL) return bad("fp8: limit must be in (0, 10 s]");
  int sms = 0;
  if (const int rc = device_sms(&sms)) return rc;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = split ? launch_fp8_split_wait_selftest(limit_ns, s) : launch_fp8_wait_selftest(limit_ns, s);
  return e == cudaSuccess ? F64E_OK : cuda_error(e);
}

int f64e_fp8_status(void* stream, int32_t* status) {
  begin_call();
  if (!status) return bad("fp8: null argument");
  int sms = 0;
  if (const int rc = device_sms(&sms)) return rc;
  const cudaError_t e = read_fp8_status(status, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? F64E_OK : cuda_error(e);
}

}  // extern "C"
