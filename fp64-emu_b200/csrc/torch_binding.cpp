// torch op binding of the B200 fp64-emu library, namespace fp64_emu_b200.
//
// The five product ops keep the reference's schemas exactly
// (torch-ext/torch_binding.cpp:7-12 of CharlesCNorton/fp64-emu) and its
// argument checks and messages (fp64_emu_cuda/fp64_emu.cu:1583-1704); the
// work is done by the C ABI in include/f64e.h with a workspace from torch's
// caching allocator on the current stream.  A few extra ops expose the
// two-phase form used by the partitioned multi-GPU path and test aids.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/core/AutogradState.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <tuple>
#include <vector>

#include "f64e.h"

namespace {

std::vector<int32_t> host_primes(const at::Tensor& primes_cpu) {
  auto pc = primes_cpu.to(at::kCPU, at::kInt).contiguous();
  return std::vector<int32_t>(pc.data_ptr<int32_t>(), pc.data_ptr<int32_t>() + pc.numel());
}

void check(int rc) { TORCH_CHECK(rc == F64E_OK, "fp64_emu: ", f64e_last_error()); }

at::Tensor make_ws(const f64e_problem& p, const at::Tensor& like) {
  const size_t n = f64e_workspace_size(&p);
  TORCH_CHECK(n > 0, "fp64_emu: ", f64e_last_error());
  return at::empty({(int64_t)n}, like.options().dtype(at::kByte));
}

void* stream_of() { return at::cuda::getCurrentCUDAStream().stream(); }

void check_out(const at::Tensor& out, const at::Tensor& A, at::IntArrayRef shape, const char* msg) {
  TORCH_CHECK(out.dtype() == at::kDouble && out.sizes() == shape && out.is_contiguous(), msg);
  TORCH_CHECK(out.is_cuda() && out.device() == A.device(), "out must be on the device of A");
}

f64e_problem problem(int64_t batch, int64_t M, int64_t N, int64_t K, bool b_kn, const std::vector<int32_t>& pr,
                     bool exact, int64_t bits, bool use_corr) {
  f64e_problem p;
  p.batch = batch;
  p.M = M;
  p.N = N;
  p.K = K;
  p.b_layout = b_kn ? F64E_B_KN : F64E_B_NK;
  p.nprimes = (int32_t)pr.size();
  p.primes = pr.data();
  p.exact = exact ? 1 : 0;
  p.bits = (int32_t)bits;
  p.use_corr = use_corr ? 1 : 0;
  p.slab_cols = 0;
  return p;
}

int64_t maxp() { return f64e_maxp(); }

// out[m,n] = A[m,k] @ B[n,k]^T (reference fp64_emu_mm, fp64_emu.cu:1583-1608).
void mm(at::Tensor& out, const at::Tensor& A, const at::Tensor& B, const at::Tensor& primes_cpu,
        const at::Tensor& inv_cpu, const at::Tensor& mu_cpu, bool exact, int64_t bits, bool use_corr) {
  (void)inv_cpu;
  (void)mu_cpu;
  TORCH_CHECK(A.is_cuda() && B.is_cuda() && A.dtype() == at::kDouble && B.dtype() == at::kDouble,
              "A,B must be f64 CUDA");
  TORCH_CHECK(A.dim() == 2 && B.dim() == 2 && A.is_contiguous() && B.is_contiguous(), "2D contig");
  const int64_t M = A.size(0), K = A.size(1), N = B.size(0);
  TORCH_CHECK(B.size(1) == K, "expect B as [N, K]");
  check_out(out, A, {M, N}, "out f64 [M,N]");
  TORCH_CHECK((int)primes_cpu.numel() <= f64e_maxp(), "too many primes");
  TORCH_CHECK(K <= (int64_t)128 * 65536, "K bound: 128 segments of 65536");
  TORCH_CHECK(bits >= 16 && bits <= 53, "bits must be in [16, 53]");
  const c10::cuda::CUDAGuard guard(A.device());
  const auto pr = host_primes(primes_cpu);
  const f64e_problem p = problem(1, M, N, K, false, pr, exact, bits, use_corr);
  at::Tensor ws = make_ws(p, A);
  check(f64e_mm(out.data_ptr<double>(), A.data_ptr<double>(), B.data_ptr<double>(), M, N, K, pr.data(),
                (int32_t)pr.size(), exact, bits, use_corr, ws.data_ptr(), ws.numel(), stream_of()));
}

// out[m,n] = A[m,k] @ Bt[k,n] (reference fp64_emu_mm_nt, fp64_emu.cu:1613-1632).
void mm_nt(at::Tensor& out, const at::Tensor& A, const at::Tensor& Bt, const at::Tensor& primes_cpu,
           const at::Tensor& inv_cpu, const at::Tensor& mu_cpu, bool exact, int64_t bits, bool use_corr) {
  (void)inv_cpu;
  (void)mu_cpu;
  TORCH_CHECK(A.is_cuda() && Bt.is_cuda() && A.dtype() == at::kDouble && Bt.dtype() == at::kDouble,
              "A,Bt must be f64 CUDA");
  TORCH_CHECK(A.dim() == 2 && Bt.dim() == 2 && A.is_contiguous() && Bt.is_contiguous(), "2D contig");
  const int64_t M = A.size(0), K = A.size(1), N = Bt.size(1);
  TORCH_CHECK(Bt.size(0) == K, "expect Bt as [K, N]");
  check_out(out, A, {M, N}, "out f64 [M,N]");
  TORCH_CHECK((int)primes_cpu.numel() <= f64e_maxp(), "too many primes");
  TORCH_CHECK(K <= 131071, "K bound for int32 modular GEMM");
  TORCH_CHECK(bits >= 16 && bits <= 53, "bits must be in [16, 53]");
  const c10::cuda::CUDAGuard guard(A.device());
  const auto pr = host_primes(primes_cpu);
  const f64e_problem p = problem(1, M, N, K, true, pr, exact, bits, use_corr);
  at::Tensor ws = make_ws(p, A);
  check(f64e_mm_nt(out.data_ptr<double>(), A.data_ptr<double>(), Bt.data_ptr<double>(), M, N, K, pr.data(),
                   (int32_t)pr.size(), exact, bits, use_corr, ws.data_ptr(), ws.numel(), stream_of()));
}

// out[b] = A[b] @ B[b]^T (reference fp64_emu_bmm, fp64_emu.cu:1637-1662).
void bmm(at::Tensor& out, const at::Tensor& A, const at::Tensor& B, const at::Tensor& primes_cpu,
         const at::Tensor& inv_cpu, const at::Tensor& mu_cpu, bool exact, int64_t bits, bool use_corr) {
  (void)inv_cpu;
  (void)mu_cpu;
  TORCH_CHECK(A.is_cuda() && B.is_cuda() && A.dtype() == at::kDouble && B.dtype() == at::kDouble,
              "A,B must be f64 CUDA");
  TORCH_CHECK(A.dim() == 3 && B.dim() == 3 && A.is_contiguous() && B.is_contiguous(), "3D contig");
  const int64_t batch = A.size(0), M = A.size(1), K = A.size(2), N = B.size(1);
  TORCH_CHECK(B.size(0) == batch && B.size(2) == K, "expect B as [batch, N, K]");
  check_out(out, A, {batch, M, N}, "out f64 [batch,M,N]");
  const int64_t NP = primes_cpu.numel() + (use_corr ? 2 : 0);
  TORCH_CHECK((int)primes_cpu.numel() <= f64e_maxp(), "too many primes");
  TORCH_CHECK(NP * batch <= 65535, "(nprimes + 2) * batch exceeds the launch z-extent");
  TORCH_CHECK(K <= (int64_t)128 * 65536, "K bound: 128 segments of 65536");
  TORCH_CHECK(bits >= 16 && bits <= 53, "bits must be in [16, 53]");
  const c10::cuda::CUDAGuard guard(A.device());
  const auto pr = host_primes(primes_cpu);
  const f64e_problem p = problem(batch, M, N, K, false, pr, exact, bits, use_corr);
  at::Tensor ws = make_ws(p, A);
  check(f64e_bmm(out.data_ptr<double>(), A.data_ptr<double>(), B.data_ptr<double>(), batch, M, N, K, pr.data(),
                 (int32_t)pr.size(), exact, bits, use_corr, ws.data_ptr(), ws.numel(), stream_of()));
}

// out[b] = A[b] @ Bt[b] (reference fp64_emu_bmm_nt, fp64_emu.cu:1665-1686).
void bmm_nt(at::Tensor& out, const at::Tensor& A, const at::Tensor& Bt, const at::Tensor& primes_cpu,
            const at::Tensor& inv_cpu, const at::Tensor& mu_cpu, bool exact, int64_t bits, bool use_corr) {
  (void)inv_cpu;
  (void)mu_cpu;
  TORCH_CHECK(A.is_cuda() && Bt.is_cuda() && A.dtype() == at::kDouble && Bt.dtype() == at::kDouble,
              "A,Bt must be f64 CUDA");
  TORCH_CHECK(A.dim() == 3 && Bt.dim() == 3 && A.is_contiguous() && Bt.is_contiguous(), "3D contig");
  const int64_t batch = A.size(0), M = A.size(1), K = A.size(2), N = Bt.size(2);
  TORCH_CHECK(Bt.size(0) == batch && Bt.size(1) == K, "expect Bt as [batch, K, N]");
  check_out(out, A, {batch, M, N}, "out f64 [batch,M,N]");
  const int64_t NP = primes_cpu.numel() + (use_corr ? 2 : 0);
  TORCH_CHECK((int)primes_cpu.numel() <= f64e_maxp(), "too many primes");
  TORCH_CHECK(NP * batch <= 65535, "(nprimes + 2) * batch exceeds the launch z-extent");
  TORCH_CHECK(K <= 131071, "K bound for int32 modular GEMM");
  TORCH_CHECK(bits >= 16 && bits <= 53, "bits must be in [16, 53]");
  const c10::cuda::CUDAGuard guard(A.device());
  const auto pr = host_primes(primes_cpu);
  const f64e_problem p = problem(batch, M, N, K, true, pr, exact, bits, use_corr);
  at::Tensor ws = make_ws(p, A);
  check(f64e_bmm_nt(out.data_ptr<double>(), A.data_ptr<double>(), Bt.data_ptr<double>(), batch, M, N, K,
                    pr.data(), (int32_t)pr.size(), exact, bits, use_corr, ws.data_ptr(), ws.numel(), stream_of()));
}

// mm with phase timings (reference fp64_emu_mm_timed, fp64_emu.cu:1688-1704).
void mm_timed(at::Tensor& out, at::Tensor& times, const at::Tensor& A, const at::Tensor& B,
              const at::Tensor& primes_cpu, const at::Tensor& inv_cpu, const at::Tensor& mu_cpu, bool exact,
              int64_t bits, bool use_corr) {
  (void)inv_cpu;
  (void)mu_cpu;
  TORCH_CHECK(A.size(1) <= 131071, "K bound for int32 modular GEMM");
  TORCH_CHECK(bits >= 16 && bits <= 53, "bits must be in [16, 53]");
  TORCH_CHECK(A.is_cuda() && B.is_cuda() && A.dtype() == at::kDouble && B.dtype() == at::kDouble,
              "A,B must be f64 CUDA");
  TORCH_CHECK(A.dim() == 2 && B.dim() == 2 && A.is_contiguous() && B.is_contiguous(), "2D contig");
  TORCH_CHECK(B.size(1) == A.size(1), "expect B as [N, K]");
  TORCH_CHECK(times.device().is_cpu() && times.dtype() == at::kFloat && times.numel() >= 4 &&
                  times.is_contiguous(),
              "times must be a CPU float32 tensor of 4");
  const int64_t M = A.size(0), K = A.size(1), N = B.size(0);
  check_out(out, A, {M, N}, "out f64 [M,N]");
  const c10::cuda::CUDAGuard guard(A.device());
  const auto pr = host_primes(primes_cpu);
  const f64e_problem p = problem(1, M, N, K, false, pr, exact, bits, use_corr);
  at::Tensor ws = make_ws(p, A);
  check(f64e_mm_timed(out.data_ptr<double>(), times.data_ptr<float>(), A.data_ptr<double>(), B.data_ptr<double>(),
                      M, N, K, pr.data(), (int32_t)pr.size(), exact, bits, use_corr, ws.data_ptr(), ws.numel(),
                      stream_of()));
}

// ---- two-phase and test-aid ops ----

f64e_problem problem_of(const at::Tensor& A, const at::Tensor& B, bool b_kn, const std::vector<int32_t>& pr,
                        bool exact, int64_t bits, bool use_corr) {
  TORCH_CHECK(A.dim() == B.dim() && (A.dim() == 2 || A.dim() == 3), "A and B must both be 2-D or 3-D");
  const bool batched = A.dim() == 3;
  const int64_t batch = batched ? A.size(0) : 1;
  const int64_t M = A.size(-2), K = A.size(-1);
  const int64_t N = b_kn ? B.size(-1) : B.size(-2);
  TORCH_CHECK((b_kn ? B.size(-2) : B.size(-1)) == K, "inner dimensions differ");
  TORCH_CHECK(!batched || B.size(0) == batch, "batch sizes differ");
  return problem(batch, M, N, K, b_kn, pr, exact, bits, use_corr);
}

int64_t workspace_bytes(const at::Tensor& A, const at::Tensor& B, const at::Tensor& primes_cpu, bool b_kn,
                        bool use_corr, int64_t slab_cols) {
  const auto pr = host_primes(primes_cpu);
  f64e_problem p = problem_of(A, B, b_kn, pr, true, 53, use_corr);
  p.slab_cols = slab_cols;
  const size_t n = f64e_workspace_size(&p);
  TORCH_CHECK(n > 0, "fp64_emu: ", f64e_last_error());
  return (int64_t)n;
}

void gemm_phase(at::Tensor& out, at::Tensor& ws, const at::Tensor& A, const at::Tensor& B,
                const at::Tensor& primes_cpu, bool b_kn, bool exact, int64_t bits, bool use_corr, int64_t phases,
                bool checked, int64_t slab_cols, const std::vector<int64_t>* events = nullptr,
                int32_t* launches = nullptr) {
  TORCH_CHECK(A.is_cuda() && B.is_cuda() && A.dtype() == at::kDouble && B.dtype() == at::kDouble,
              "A,B must be f64 CUDA");
  TORCH_CHECK(A.is_contiguous() && B.is_contiguous() && out.is_contiguous() && ws.is_contiguous(), "contig");
  TORCH_CHECK(ws.is_cuda() && ws.device() == A.device() && out.device() == A.device(), "same device");
  const auto pr = host_primes(primes_cpu);
  f64e_problem p = problem_of(A, B, b_kn, pr, exact, bits, use_corr);
  p.slab_cols = slab_cols;
  TORCH_CHECK(out.dtype() == at::kDouble && out.numel() == p.batch * p.M * p.N, "out f64 of batch*M*N");
  const c10::cuda::CUDAGuard guard(A.device());
  const size_t nb = (size_t)ws.numel() * ws.element_size();
  if (checked)
    check(f64e_gemm_checked(&p, A.data_ptr<double>(), B.data_ptr<double>(), out.data_ptr<double>(), ws.data_ptr(),
                            nb, stream_of()));
  else if (events) {
    std::vector<void*> ev(events->size());
    for (size_t i = 0; i < ev.size(); i++) ev[i] = reinterpret_cast<void*>((*events)[i]);
    check(f64e_gemm_ev(&p, A.data_ptr<double>(), B.data_ptr<double>(), out.data_ptr<double>(), ws.data_ptr(), nb,
                       stream_of(), (int)phases, ev.data(), (int32_t)ev.size(), launches));
  } else {
    check(f64e_gemm(&p, A.data_ptr<double>(), B.data_ptr<double>(), out.data_ptr<double>(), ws.data_ptr(), nb,
                    stream_of(), (int)phases));
  }
}

void gemm_ws(at::Tensor& out, at::Tensor& ws, const at::Tensor& A, const at::Tensor& B,
             const at::Tensor& primes_cpu, bool b_kn, bool exact, int64_t bits, bool use_corr, int64_t phases,
             int64_t slab_cols) {
  gemm_phase(out, ws, A, B, primes_cpu, b_kn, exact, bits, use_corr, phases, false, slab_cols);
}

// gemm_ws that brackets each modular-GEMM launch with two of the given CUDA
// events (raw cudaEvent_t handles, e.g. torch.cuda.Event.cuda_event) and
// returns the number of GEMM launches.
int64_t gemm_ws_ev(at::Tensor& out, at::Tensor& ws, const at::Tensor& A, const at::Tensor& B,
                   const at::Tensor& primes_cpu, bool b_kn, bool exact, int64_t bits, bool use_corr, int64_t phases,
                   int64_t slab_cols, at::IntArrayRef events) {
  for (const int64_t e : events) TORCH_CHECK(e != 0, "events must be created (record them once first)");
  const std::vector<int64_t> ev(events.begin(), events.end());
  int32_t launches = 0;
  gemm_phase(out, ws, A, B, primes_cpu, b_kn, exact, bits, use_corr, phases, false, slab_cols, &ev, &launches);
  return launches;
}

// Host-resident product: A, B and out are CPU tensors (page-locked for the
// copies to overlap); the device buffers and workspace come from torch's
// caching allocator on the current device and stream.  The result blocks are
// copied back while later blocks compute; the call returns once out holds
// the product.
void gemm_host(at::Tensor& out, const at::Tensor& A, const at::Tensor& B, const at::Tensor& primes_cpu, bool b_kn,
               bool exact, int64_t bits, bool use_corr) {
  TORCH_CHECK(!A.is_cuda() && !B.is_cuda() && !out.is_cuda(), "host product: A, B and out must be CPU tensors");
  TORCH_CHECK(A.dtype() == at::kDouble && B.dtype() == at::kDouble && out.dtype() == at::kDouble, "f64 tensors");
  TORCH_CHECK(A.is_contiguous() && B.is_contiguous() && out.is_contiguous(), "contig");
  TORCH_CHECK(bits >= 16 && bits <= 53, "bits must be in [16, 53]");
  const auto pr = host_primes(primes_cpu);
  const f64e_problem p = problem_of(A, B, b_kn, pr, exact, bits, use_corr);
  TORCH_CHECK(out.numel() == p.batch * p.M * p.N, "out f64 of batch*M*N");
  const auto dev = at::TensorOptions().device(at::kCUDA, c10::cuda::current_device()).dtype(at::kDouble);
  at::Tensor Ad = at::empty(A.sizes(), dev), Bd = at::empty(B.sizes(), dev), Cd = at::empty(out.sizes(), dev);
  const size_t nb = f64e_workspace_size(&p);
  TORCH_CHECK(nb > 0, "fp64_emu: ", f64e_last_error());
  at::Tensor ws = at::empty({(int64_t)nb}, dev.dtype(at::kByte));
  check(f64e_gemm_host(&p, A.data_ptr<double>(), B.data_ptr<double>(), out.data_ptr<double>(), Ad.data_ptr<double>(),
                       Bd.data_ptr<double>(), Cd.data_ptr<double>(), ws.data_ptr(), nb, stream_of()));
  const cudaError_t e = cudaStreamSynchronize(static_cast<cudaStream_t>(stream_of()));
  TORCH_CHECK(e == cudaSuccess, "fp64_emu: ", cudaGetErrorString(e));
}

// One product of fp64_emu.HostStream, queued without a host wait: the
// operand copies on streams[0], the product on streams[1], the result copy on
// streams[2] (raw cudaStream_t handles of the slot's device).  events (raw
// cudaEvent_t, created): [caller, loaded, computed, done]; the three streams
// first wait for what the caller's current stream queued before the call,
// and when the slot held an earlier product (used) the copies into its
// device operands wait until that product has read them and the product
// waits until its result has left the device.
void host_submit(at::Tensor& out, const at::Tensor& A, const at::Tensor& B, at::Tensor& Ad, at::Tensor& Bd,
                 at::Tensor& Cd, at::Tensor& ws, const at::Tensor& primes_cpu, bool b_kn, bool exact, int64_t bits,
                 bool use_corr, at::IntArrayRef streams, at::IntArrayRef events, bool used) {
  TORCH_CHECK(!A.is_cuda() && !B.is_cuda() && !out.is_cuda(), "host submit: A, B and out must be CPU tensors");
  TORCH_CHECK(Ad.is_cuda() && Bd.is_cuda() && Cd.is_cuda() && ws.is_cuda(), "host submit: device buffers");
  TORCH_CHECK(Bd.device() == Ad.device() && Cd.device() == Ad.device() && ws.device() == Ad.device(),
              "host submit: device buffers on one device");
  for (const at::Tensor* t : std::initializer_list<const at::Tensor*>{&out, &A, &B, &Ad, &Bd, &Cd})
    TORCH_CHECK(t->dtype() == at::kDouble && t->is_contiguous(), "host submit: contiguous f64 tensors");
  TORCH_CHECK(A.sizes() == Ad.sizes() && B.sizes() == Bd.sizes() && out.sizes() == Cd.sizes(),
              "host submit: host and device shapes differ");
  TORCH_CHECK(ws.is_contiguous(), "host submit: contiguous workspace");
  TORCH_CHECK(streams.size() == 3 && events.size() == 4, "host submit: 3 streams and 4 events");
  for (const int64_t e : events) TORCH_CHECK(e != 0, "events must be created (record them once first)");
  TORCH_CHECK(bits >= 16 && bits <= 53, "bits must be in [16, 53]");
  const auto pr = host_primes(primes_cpu);
  const f64e_problem p = problem_of(Ad, Bd, b_kn, pr, exact, bits, use_corr);
  const c10::cuda::CUDAGuard guard(Ad.device());
  cudaStream_t h2d = reinterpret_cast<cudaStream_t>(streams[0]), comp = reinterpret_cast<cudaStream_t>(streams[1]),
               d2h = reinterpret_cast<cudaStream_t>(streams[2]);
  cudaEvent_t caller = reinterpret_cast<cudaEvent_t>(events[0]), loaded = reinterpret_cast<cudaEvent_t>(events[1]),
              computed = reinterpret_cast<cudaEvent_t>(events[2]), done = reinterpret_cast<cudaEvent_t>(events[3]);
  cudaError_t e = cudaEventRecord(caller, static_cast<cudaStream_t>(stream_of()));
  for (cudaStream_t st : {h2d, comp, d2h})
    if (e == cudaSuccess) e = cudaStreamWaitEvent(st, caller, 0);
  if (used && e == cudaSuccess) e = cudaStreamWaitEvent(h2d, computed, 0);
  if (used && e == cudaSuccess) e = cudaStreamWaitEvent(comp, done, 0);
  if (e == cudaSuccess)
    e = cudaMemcpyAsync(Ad.data_ptr(), A.data_ptr(), (size_t)A.numel() * 8, cudaMemcpyHostToDevice, h2d);
  if (e == cudaSuccess)
    e = cudaMemcpyAsync(Bd.data_ptr(), B.data_ptr(), (size_t)B.numel() * 8, cudaMemcpyHostToDevice, h2d);
  if (e == cudaSuccess) e = cudaEventRecord(loaded, h2d);
  if (e == cudaSuccess) e = cudaStreamWaitEvent(comp, loaded, 0);
  TORCH_CHECK(e == cudaSuccess, "fp64_emu: ", cudaGetErrorString(e));
  check(f64e_gemm(&p, Ad.data_ptr<double>(), Bd.data_ptr<double>(), Cd.data_ptr<double>(), ws.data_ptr(),
                  (size_t)ws.numel() * ws.element_size(), comp, F64E_PHASE_ALL));
  e = cudaEventRecord(computed, comp);
  if (e == cudaSuccess) e = cudaStreamWaitEvent(d2h, computed, 0);
  if (e == cudaSuccess)
    e = cudaMemcpyAsync(out.data_ptr(), Cd.data_ptr(), (size_t)out.numel() * 8, cudaMemcpyDeviceToHost, d2h);
  if (e == cudaSuccess) e = cudaEventRecord(done, d2h);
  TORCH_CHECK(e == cudaSuccess, "fp64_emu: ", cudaGetErrorString(e));
}

void gemm_checked(at::Tensor& out, at::Tensor& ws, const at::Tensor& A, const at::Tensor& B,
                  const at::Tensor& primes_cpu, bool b_kn, bool exact, int64_t bits, bool use_corr) {
  gemm_phase(out, ws, A, B, primes_cpu, b_kn, exact, bits, use_corr, F64E_PHASE_ALL, true, 0);
}

int64_t status(const at::Tensor& ws) {
  TORCH_CHECK(ws.is_cuda(), "workspace must be CUDA");
  const c10::cuda::CUDAGuard guard(ws.device());
  int32_t st = 0;
  check(f64e_status(ws.data_ptr(), stream_of(), &st));
  return st;
}

at::Tensor debug_fetch(const at::Tensor& ws, const at::Tensor& A, const at::Tensor& B, const at::Tensor& primes_cpu,
                       bool b_kn, bool use_corr, int64_t which) {
  const auto pr = host_primes(primes_cpu);
  const f64e_problem p = problem_of(A, B, b_kn, pr, true, 53, use_corr);
  const c10::cuda::CUDAGuard guard(ws.device());
  const size_t cap = (size_t)ws.numel();
  at::Tensor host = at::empty({(int64_t)cap}, at::TensorOptions().dtype(at::kByte));
  size_t n = 0;
  check(f64e_debug_fetch(&p, ws.data_ptr(), (int)which, host.data_ptr(), cap, &n, stream_of()));
  return host.narrow(0, 0, (int64_t)n).clone();
}

void set_wait_limit_ns(int64_t ns) { f64e_set_wait_limit_ns((uint64_t)ns); }

int64_t wait_selftest(at::Tensor& ws, int64_t limit_ns) {
  TORCH_CHECK(ws.is_cuda() && ws.is_contiguous(), "workspace must be a contiguous CUDA tensor");
  TORCH_CHECK(limit_ns > 0, "limit must be positive");
  const c10::cuda::CUDAGuard guard(ws.device());
  int32_t st = 0;
  check(f64e_wait_selftest(ws.data_ptr(), (size_t)ws.numel() * ws.element_size(), (uint64_t)limit_ns, stream_of(),
                           &st));
  return st;
}

// ---- 8-bit floating-point operators ----

int fp8_type(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return F64E_F32;
    case at::kHalf: return F64E_F16;
    case at::kBFloat16: return F64E_BF16;
    default: return -1;
  }
}
int fp8_code(at::ScalarType t) {
  return t == at::kFloat8_e4m3fn ? F64E_E4M3 : t == at::kFloat8_e5m2 ? F64E_E5M2 : -1;
}
// Shapes of a product's operands: A [M, K] B [N, K], A [M, K] B [K, N], A [K, M] B [K, N].
enum { kFp8NT = 0, kFp8NN = 1, kFp8TN = 2 };
int64_t fp8_blocks(int64_t n) { return (n + 127) / 128; }
c10::SymInt fp8_blocks(const c10::SymInt& n) { return (n + 127) / 128; }

void fp8_check_float(const at::Tensor& x, const char* what) {
  TORCH_CHECK(fp8_type(x.scalar_type()) >= 0, what, " must be float32, float16 or bfloat16");
}
void fp8_check_cuda(const at::Tensor& t, const char* what) { TORCH_CHECK(t.is_cuda(), what, " must be a CUDA tensor"); }

// Rows of x with unit stride (x itself, or a copy).
at::Tensor fp8_rows(const at::Tensor& x) {
  return (x.stride(1) == 1 || x.size(1) <= 1) && (x.stride(0) >= x.size(1) || x.size(0) <= 1) ? x : x.contiguous();
}
int64_t fp8_pitch(const at::Tensor& x) { return x.size(0) <= 1 ? std::max<int64_t>(x.size(1), 1) : x.stride(0); }

// A new tensor on x's device (current by the caller's guard) straight from the
// allocator: these operators' small calls cost as much on the host as on the GPU.
at::Tensor fp8_empty(const at::Tensor& x, at::IntArrayRef sizes, at::ScalarType type) {
  if (!x.is_cuda()) return at::empty(sizes, x.options().dtype(type));
  return at::detail::empty_cuda(sizes, type, x.device(), std::nullopt);
}
// Codes [rows, cols] whose rows start on 16-byte boundaries.
at::Tensor fp8_new_codes(const at::Tensor& x, int64_t rows, int64_t cols, at::ScalarType code) {
  const int64_t ld = (cols + 15) / 16 * 16;
  at::Tensor q = fp8_empty(x, {rows, ld}, code);
  return ld == cols ? q : q.as_strided({rows, cols}, {ld, 1});
}
int64_t fp8_code_pitch(int64_t cols) { return (cols + 15) / 16 * 16; }

std::tuple<at::Tensor, at::Tensor> fp8_quantize(const at::Tensor& x, int64_t blocks, at::ScalarType code) {
  TORCH_CHECK(x.dim() == 2, "x must be a matrix");
  fp8_check_float(x, "x");
  TORCH_CHECK(fp8_code(code) >= 0, "the code must be float8_e4m3fn or float8_e5m2");
  TORCH_CHECK(blocks >= F64E_BLOCKS_ROW && blocks <= F64E_BLOCKS_TILE, "blocks must be row, col or tile");
  fp8_check_cuda(x, "x");
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t R = x.size(0), C = x.size(1);
  const at::Tensor xr = fp8_rows(x);
  at::Tensor q = fp8_new_codes(x, R, C, code);
  at::Tensor s = fp8_empty(x, {blocks == F64E_BLOCKS_ROW ? R : fp8_blocks(R), blocks == F64E_BLOCKS_COL ? C : fp8_blocks(C)},
                           at::kFloat8_e8m0fnu);
  check(f64e_fp8_quantize(xr.data_ptr(), fp8_type(x.scalar_type()), R, C, fp8_pitch(xr), (int32_t)blocks,
                          fp8_code(code), q.data_ptr(), fp8_code_pitch(C), s.data_ptr(), stream_of()));
  return {q, s};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> fp8_quantize_both(const at::Tensor& x, at::ScalarType code,
                                                                             bool transposed) {
  TORCH_CHECK(x.dim() == 2, "x must be a matrix");
  fp8_check_float(x, "x");
  TORCH_CHECK(fp8_code(code) >= 0, "the code must be float8_e4m3fn or float8_e5m2");
  fp8_check_cuda(x, "x");
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t R = x.size(0), C = x.size(1);
  const at::Tensor xr = fp8_rows(x);
  at::Tensor q = fp8_new_codes(x, R, C, code);
  at::Tensor qc = transposed ? fp8_new_codes(x, C, R, code).t() : fp8_new_codes(x, R, C, code);
  at::Tensor s = fp8_empty(x, {R, fp8_blocks(C)}, at::kFloat8_e8m0fnu);
  at::Tensor sc = fp8_empty(x, {fp8_blocks(R), C}, at::kFloat8_e8m0fnu);
  check(f64e_fp8_quantize_both(xr.data_ptr(), fp8_type(x.scalar_type()), R, C, fp8_pitch(xr), fp8_code(code),
                               q.data_ptr(), s.data_ptr(), fp8_code_pitch(C), qc.data_ptr(), sc.data_ptr(), transposed,
                               fp8_code_pitch(transposed ? R : C), stream_of()));
  return {q, s, qc, sc};
}

at::Tensor fp8_dequantize(const at::Tensor& q, const at::Tensor& s, int64_t blocks, at::ScalarType dtype) {
  TORCH_CHECK(q.dim() == 2 && s.dim() == 2, "codes and scales must be matrices");
  TORCH_CHECK(fp8_code(q.scalar_type()) >= 0, "codes must be float8_e4m3fn or float8_e5m2");
  TORCH_CHECK(s.scalar_type() == at::kFloat8_e8m0fnu, "scales must be float8_e8m0fnu (powers of two)");
  TORCH_CHECK(fp8_type(dtype) >= 0, "the result must be float32, float16 or bfloat16");
  TORCH_CHECK(blocks >= F64E_BLOCKS_ROW && blocks <= F64E_BLOCKS_TILE, "blocks must be row, col or tile");
  const int64_t R = q.size(0), C = q.size(1);
  TORCH_CHECK(s.size(0) == (blocks == F64E_BLOCKS_ROW ? R : fp8_blocks(R)) &&
                  s.size(1) == (blocks == F64E_BLOCKS_COL ? C : fp8_blocks(C)),
              "scales do not have one entry per block");
  fp8_check_cuda(q, "codes");
  TORCH_CHECK(s.device() == q.device(), "codes and scales must be on one device");
  const c10::cuda::CUDAGuard guard(q.device());
  const at::Tensor qr = fp8_rows(q);
  at::Tensor out = fp8_empty(q, {R, C}, dtype);
  check(f64e_fp8_dequantize(qr.data_ptr(), fp8_code(q.scalar_type()), R, C, fp8_pitch(qr), (int32_t)blocks,
                            s.data_ptr(), s.stride(0), s.stride(1), out.data_ptr(), fp8_type(dtype), stream_of()));
  return out;
}

// One operand of a product: codes whose rows start on 16-byte boundaries (a
// copy is made when they do not), scales as strides.  kdim: the contracted
// dimension of q.
struct Fp8Held {
  at::Tensor q;
  f64e_fp8_operand o;
};
void fp8_check_operand(const at::Tensor& q, const at::Tensor& s, int kdim, const char* name) {
  TORCH_CHECK(q.dim() == 2 && s.dim() == 2, name, ": codes and scales must be matrices");
  TORCH_CHECK(fp8_code(q.scalar_type()) >= 0, name, ": codes must be float8_e4m3fn or float8_e5m2");
  TORCH_CHECK(s.scalar_type() == at::kFloat8_e8m0fnu, name, ": scales must be float8_e8m0fnu (powers of two)");
  const c10::SymInt r = q.sym_size(1 - kdim), k = q.sym_size(kdim), sr = s.sym_size(1 - kdim), sk = s.sym_size(kdim);
  TORCH_CHECK(sk == fp8_blocks(k) && (sr == r || sr == fp8_blocks(r)), name, ": scales of shape ", s.sym_sizes(),
              " do not fit codes of shape ", q.sym_sizes(), " with blocks of 128 along the contracted dimension");
}
// Whether the rows of the stored codes start on 16-byte boundaries, with
// `fast` the contiguous dimension.
bool fp8_aligned(const at::Tensor& q, int fast) {
  const int64_t n = q.size(fast), m = q.size(1 - fast);
  return (n <= 1 || q.stride(fast) == 1) && (m <= 1 || (q.stride(1 - fast) % 16 == 0 && q.stride(1 - fast) >= n)) &&
         (reinterpret_cast<uintptr_t>(q.data_ptr()) & 15) == 0;
}
Fp8Held fp8_hold(const at::Tensor& q, const at::Tensor& s, int kdim) {
  Fp8Held h;
  int fast = 1;
  h.q = q;
  if (!fp8_aligned(q, 1)) {
    if (fp8_aligned(q, 0)) {
      fast = 0;
    } else {
      h.q = fp8_new_codes(q, q.size(0), q.size(1), q.scalar_type());
      h.q.copy_(q);
    }
  }
  h.o.ld = h.q.size(1 - fast) <= 1 ? fp8_code_pitch(h.q.size(fast)) : h.q.stride(1 - fast);
  h.o.k_major = fast == kdim;
  h.o.code = fp8_code(q.scalar_type());
  h.o.tile = s.size(1 - kdim) == q.size(1 - kdim) ? 0 : 1;
  h.o.scale_row = s.stride(1 - kdim);
  h.o.scale_block = s.stride(kdim);
  return h;
}

at::Tensor fp8_mm(const at::Tensor& a, const at::Tensor& b, const at::Tensor& sa, const at::Tensor& sb, int64_t layout,
                  at::ScalarType dtype) {
  TORCH_CHECK(layout >= kFp8NT && layout <= kFp8TN, "layout must be 0 (NT), 1 (NN) or 2 (TN)");
  const int ka = layout == kFp8TN ? 0 : 1, kb = layout == kFp8NT ? 1 : 0;
  fp8_check_operand(a, sa, ka, "A");
  fp8_check_operand(b, sb, kb, "B");
  TORCH_CHECK(a.size(ka) == b.size(kb), "inner dimensions differ");
  TORCH_CHECK(a.size(ka) >= 1, "the inner dimension must be at least 1");
  TORCH_CHECK(fp8_type(dtype) >= 0, "the result must be float32, float16 or bfloat16");
  fp8_check_cuda(a, "A");
  TORCH_CHECK(b.device() == a.device() && sa.device() == a.device() && sb.device() == a.device(),
              "operands and scales must be on one device");
  const c10::cuda::CUDAGuard guard(a.device());
  const Fp8Held ha = fp8_hold(a, sa, ka), hb = fp8_hold(b, sb, kb);
  f64e_fp8_problem p;
  p.M = a.size(1 - ka);
  p.N = b.size(1 - kb);
  p.K = a.size(ka);
  p.out_type = fp8_type(dtype);
  p.ldo = p.N;
  p.a = ha.o;
  p.b = hb.o;
  at::Tensor out = fp8_empty(a, {p.M, p.N}, dtype);
  const size_t nb = f64e_fp8_workspace_size(&p);
  const at::Tensor ws = nb ? fp8_empty(a, {(int64_t)nb}, at::kByte) : at::Tensor();
  check(f64e_fp8_gemm(&p, ha.q.data_ptr(), sa.data_ptr(), hb.q.data_ptr(), sb.data_ptr(), out.data_ptr(),
                      nb ? ws.data_ptr() : nullptr, nb, stream_of()));
  return out;
}

// Status of the 8-bit products on a device (f64e_fp8_status).
int64_t fp8_status(int64_t device) {
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
  int32_t st = 0;
  check(f64e_fp8_status(stream_of(), &st));
  return st;
}

void fp8_wait_selftest(int64_t device, bool split, int64_t limit_ns) {
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
  check(f64e_fp8_wait_selftest(split, (uint64_t)limit_ns, stream_of()));
}

// ---- a layer held in 8 bits ----
// Sizes are read as symbols wherever the layer's autograd kernel comes by: it
// also runs while a compiler traces it, and a number read there would tie the
// traced program to the batch size at hand.
void fp8_check_linear(const at::Tensor& x, const at::Tensor& w, const std::optional<at::Tensor>& ws) {
  TORCH_CHECK(x.dim() >= 1 && w.dim() == 2, "x must have at least one dimension and w two");
  fp8_check_float(x, "x");
  TORCH_CHECK(x.sym_size(-1) == w.sym_size(1), "x's last dimension and w's differ");
  TORCH_CHECK(w.sym_size(0) >= 1 && w.sym_size(1) >= 1, "w must not be empty");
  if (ws.has_value()) {
    fp8_check_operand(w, *ws, 1, "w");
    TORCH_CHECK(ws->sym_size(0) == fp8_blocks(w.sym_size(0)), "w: kept weights need one scale per 128 x 128 square");
  } else {
    fp8_check_float(w, "w");
  }
  TORCH_CHECK(w.device() == x.device() && (!ws.has_value() || ws->device() == x.device()),
              "x, w and its scales must be on one device");
}
std::vector<int64_t> fp8_out_sizes(const at::Tensor& x, int64_t n) {
  std::vector<int64_t> v = x.sizes().vec();
  v.back() = n;
  return v;
}

at::Tensor fp8_linear(const at::Tensor& x, const at::Tensor& w, const std::optional<at::Tensor>& ws) {
  fp8_check_linear(x, w, ws);
  fp8_check_cuda(x, "x");
  const c10::cuda::CUDAGuard guard(x.device());
  const at::Tensor xr = fp8_rows(x.dim() == 2 ? x : x.reshape({-1, x.size(-1)}));
  at::Tensor wq, wsc;
  if (ws.has_value()) {
    wq = w;
    wsc = *ws;
  } else {
    std::tie(wq, wsc) = fp8_quantize(w, F64E_BLOCKS_TILE, at::kFloat8_e4m3fn);
  }
  const Fp8Held hw = fp8_hold(wq, wsc, 1);
  f64e_fp8_problem p{};
  p.M = xr.size(0);
  p.N = w.size(0);
  p.K = w.size(1);
  p.out_type = fp8_type(x.scalar_type());
  p.ldo = p.N;
  p.b = hw.o;
  const size_t nb = f64e_fp8_linear_workspace_size(p.M, p.K);
  const at::Tensor work = nb ? fp8_empty(x, {(int64_t)nb}, at::kByte) : at::Tensor();
  at::Tensor y = fp8_empty(x, fp8_out_sizes(x, p.N), x.scalar_type());
  check(f64e_fp8_linear(&p, xr.data_ptr(), fp8_pitch(xr), hw.q.data_ptr(), wsc.data_ptr(), y.data_ptr(),
                        nb ? work.data_ptr() : nullptr, nb, stream_of()));
  return y;
}

// The same with gradients.  What the backward pass needs of x is kept in 8
// bits with blocks along the rows of x (the tokens), the direction the weight
// gradient contracts, and those contiguous, so that product takes x's codes as
// the K-major operand it needs; the operators are called through the dispatcher, so a
// tracer sees them.
using Two = std::tuple<at::Tensor, at::Tensor>;
using Four = std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor>;
Two call_quantize(const at::Tensor& x, int64_t blocks) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("fp64_emu_b200::fp8_quantize", "")
                       .typed<Two(const at::Tensor&, int64_t, at::ScalarType)>();
  return op.call(x, blocks, at::kFloat8_e4m3fn);
}
Four call_quantize_both(const at::Tensor& x, bool transposed) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("fp64_emu_b200::fp8_quantize_both", "")
                       .typed<Four(const at::Tensor&, at::ScalarType, bool)>();
  return op.call(x, at::kFloat8_e4m3fn, transposed);
}
at::Tensor call_mm(const at::Tensor& a, const at::Tensor& b, const at::Tensor& sa, const at::Tensor& sb,
                   int64_t layout, at::ScalarType dtype) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("fp64_emu_b200::fp8_mm", "")
                       .typed<at::Tensor(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                                         int64_t, at::ScalarType)>();
  return op.call(a, b, sa, sb, layout, dtype);
}
at::Tensor call_linear(const at::Tensor& x, const at::Tensor& w, const std::optional<at::Tensor>& ws) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("fp64_emu_b200::fp8_linear", "")
                       .typed<at::Tensor(const at::Tensor&, const at::Tensor&, const std::optional<at::Tensor>&)>();
  return op.call(x, w, ws);
}

// x [..., K] as a matrix, and rows [n, N] with x's leading dimensions.
at::Tensor fp8_matrix(const at::Tensor& x) {
  return x.dim() == 2 ? x : x.reshape_symint({c10::SymInt(-1), x.sym_size(-1)});
}
at::Tensor fp8_shaped_like(const at::Tensor& rows, const at::Tensor& x) {
  if (x.dim() == 2) return rows;
  std::vector<c10::SymInt> v = x.sym_sizes().vec();
  v.back() = rows.sym_size(1);
  return rows.view_symint(v);
}

struct Fp8Linear : public torch::autograd::Function<Fp8Linear> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w,
                            const std::optional<at::Tensor>& ws) {
    at::AutoDispatchBelowADInplaceOrView below;
    const at::Tensor x2 = fp8_matrix(x);
    const bool want_w = w.requires_grad() && !ws.has_value();
    at::Tensor q, s, qc, sc, wq = w, wsc;
    if (want_w)
      std::tie(q, s, qc, sc) = call_quantize_both(x2, true);
    else
      std::tie(q, s) = call_quantize(x2, F64E_BLOCKS_ROW);
    if (ws.has_value())
      wsc = *ws;
    else
      std::tie(wq, wsc) = call_quantize(w, F64E_BLOCKS_TILE);
    at::Tensor y = call_mm(q, wq, s, wsc, kFp8NT, x.scalar_type());
    const bool want_x = x.requires_grad();
    ctx->save_for_backward({want_x ? wq : at::Tensor(), want_x ? wsc : at::Tensor(), qc, sc});
    ctx->saved_data["x_type"] = (int64_t)x.scalar_type();
    ctx->saved_data["w_type"] = (int64_t)w.scalar_type();
    return fp8_shaped_like(y, x);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    // Asked for straight away; a gradient that comes with a graph of its own (a
    // layer or a loss behind this one) is taken, see once().
    TORCH_CHECK(!(at::GradMode::is_enabled() && grads[0].requires_grad() && grads[0].is_leaf()), kNoSecond);
    at::AutoDispatchBelowADInplaceOrView below;
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &wq = saved[0], &wsc = saved[1], &qc = saved[2], &sc = saved[3];
    const bool want_x = wq.defined(), want_w = qc.defined();
    at::Tensor dx, dw;
    if (grads[0].defined() && (want_x || want_w)) {
      const at::Tensor g = fp8_matrix(grads[0]);
      at::Tensor q, s, gc, gsc;
      if (want_x && want_w)
        std::tie(q, s, gc, gsc) = call_quantize_both(g, true);
      else if (want_x)
        std::tie(q, s) = call_quantize(g, F64E_BLOCKS_ROW);
      else
        std::tie(gc, gsc) = call_quantize(g, F64E_BLOCKS_COL);
      if (want_x) {
        dx = call_mm(q, wq, s, wsc, kFp8NN, (at::ScalarType)ctx->saved_data["x_type"].toInt());
        dx = fp8_shaped_like(dx, grads[0]);
      }
      if (want_w) {
        const auto wt = (at::ScalarType)ctx->saved_data["w_type"].toInt();
        dw = TORCH_GUARD_OR_TRUE(g.sym_size(0).sym_gt(0))
                 ? call_mm(gc, qc, gsc, sc, kFp8TN, wt)
                 : at::zeros_symint({g.sym_size(1), qc.sym_size(1)}, g.options().dtype(wt));
      }
    }
    return {once(dx), once(dw), at::Tensor()};
  }

 private:
  static constexpr const char* kNoSecond = "linear_fp8 has no second derivative";
  // Where a graph of the backward pass is asked for (create_graph): dx depends
  // on w and dy, dw on x and dy, so a gradient is not a constant, and
  // differentiating it ends with an error instead of leaving it out.
  static at::Tensor once(at::Tensor grad) {
    if (!grad.defined() || !at::GradMode::is_enabled()) return grad;
    grad.set_requires_grad(true);
    return torch::autograd::DelayedError(kNoSecond, 1).apply({grad})[0];
  }
};

// A tangent would be lost below this kernel: the result would count as a constant.
void fp8_check_no_tangent(const at::Tensor& t) {
  TORCH_CHECK(!t._fw_grad(/*level=*/0).defined(), "linear_fp8 has no forward-mode derivative");
}

at::Tensor fp8_linear_autograd(const at::Tensor& x, const at::Tensor& w, const std::optional<at::Tensor>& ws) {
  if (c10::AutogradState::get_tls_state().get_fw_grad_mode()) {
    fp8_check_no_tangent(x);
    fp8_check_no_tangent(w);
  }
  if (at::GradMode::is_enabled() && (x.requires_grad() || (w.requires_grad() && !ws.has_value()))) {
    fp8_check_linear(x, w, ws);   // the device is asked for by the operators it calls: shapes alone (meta) pass
    return Fp8Linear::apply(x, w, ws);
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return call_linear(x, w, ws);
}

}  // namespace

TORCH_LIBRARY(fp64_emu_b200, ops) {
  ops.def("fp64_emu_maxp() -> int");
  ops.def(
      "fp64_emu_mm(Tensor! out, Tensor A, Tensor B, Tensor primes_cpu, Tensor inv_cpu, Tensor mu_cpu, bool exact, "
      "int bits=53, bool use_corr=True) -> ()");
  ops.def(
      "fp64_emu_bmm(Tensor! out, Tensor A, Tensor B, Tensor primes_cpu, Tensor inv_cpu, Tensor mu_cpu, bool exact, "
      "int bits=53, bool use_corr=True) -> ()");
  ops.def(
      "fp64_emu_mm_nt(Tensor! out, Tensor A, Tensor Bt, Tensor primes_cpu, Tensor inv_cpu, Tensor mu_cpu, bool "
      "exact, int bits=53, bool use_corr=True) -> ()");
  ops.def(
      "fp64_emu_bmm_nt(Tensor! out, Tensor A, Tensor Bt, Tensor primes_cpu, Tensor inv_cpu, Tensor mu_cpu, bool "
      "exact, int bits=53, bool use_corr=True) -> ()");
  ops.def(
      "fp64_emu_mm_timed(Tensor! out, Tensor! times, Tensor A, Tensor B, Tensor primes_cpu, Tensor inv_cpu, Tensor "
      "mu_cpu, bool exact, int bits=53, bool use_corr=True) -> ()");
  ops.def(
      "fp64_emu_workspace_bytes(Tensor A, Tensor B, Tensor primes_cpu, bool b_kn, bool use_corr, int slab_cols=0) "
      "-> int");
  ops.def(
      "fp64_emu_gemm_ws(Tensor! out, Tensor! ws, Tensor A, Tensor B, Tensor primes_cpu, bool b_kn, bool exact, "
      "int bits, bool use_corr, int phases, int slab_cols=0) -> ()");
  ops.def(
      "fp64_emu_gemm_ws_ev(Tensor! out, Tensor! ws, Tensor A, Tensor B, Tensor primes_cpu, bool b_kn, bool exact, "
      "int bits, bool use_corr, int phases, int slab_cols, int[] events) -> int");
  ops.def(
      "fp64_emu_gemm_host(Tensor! out, Tensor A, Tensor B, Tensor primes_cpu, bool b_kn, bool exact, int bits, "
      "bool use_corr) -> ()");
  ops.def(
      "fp64_emu_host_submit(Tensor! out, Tensor A, Tensor B, Tensor! Ad, Tensor! Bd, Tensor! Cd, Tensor! ws, "
      "Tensor primes_cpu, bool b_kn, bool exact, int bits, bool use_corr, int[] streams, int[] events, bool used) "
      "-> ()");
  ops.def(
      "fp64_emu_gemm_checked(Tensor! out, Tensor! ws, Tensor A, Tensor B, Tensor primes_cpu, bool b_kn, bool "
      "exact, int bits, bool use_corr) -> ()");
  ops.def("fp64_emu_status(Tensor ws) -> int");
  ops.def(
      "fp64_emu_debug_fetch(Tensor ws, Tensor A, Tensor B, Tensor primes_cpu, bool b_kn, bool use_corr, int which) "
      "-> Tensor");
  ops.def("fp64_emu_set_wait_limit_ns(int ns) -> ()");
  ops.def("fp64_emu_wait_selftest(Tensor! ws, int limit_ns) -> int");
  ops.def("fp8_quantize(Tensor x, int blocks, ScalarType code) -> (Tensor, Tensor)");
  ops.def("fp8_quantize_both(Tensor x, ScalarType code, bool transposed) -> (Tensor, Tensor, Tensor, Tensor)");
  ops.def("fp8_dequantize(Tensor q, Tensor s, int blocks, ScalarType dtype) -> Tensor");
  ops.def("fp8_mm(Tensor a, Tensor b, Tensor sa, Tensor sb, int layout, ScalarType dtype) -> Tensor");
  ops.def("fp8_linear(Tensor x, Tensor w, Tensor? ws=None) -> Tensor");
  ops.def("fp8_status(int device) -> int");
  ops.def("fp8_wait_selftest(int device, bool split, int limit_ns) -> ()");
  ops.impl("fp8_wait_selftest", &fp8_wait_selftest);
  ops.impl("fp8_status", &fp8_status);
  ops.impl("fp64_emu_maxp", &maxp);
  ops.impl("fp64_emu_workspace_bytes", &workspace_bytes);
  ops.impl("fp64_emu_set_wait_limit_ns", &set_wait_limit_ns);
}

// The host product's tensors live on the CPU; its work runs on the current CUDA device.
TORCH_LIBRARY_IMPL(fp64_emu_b200, CPU, ops) { ops.impl("fp64_emu_gemm_host", &gemm_host); }

TORCH_LIBRARY_IMPL(fp64_emu_b200, CUDA, ops) {
  ops.impl("fp64_emu_mm", &mm);
  ops.impl("fp64_emu_bmm", &bmm);
  ops.impl("fp64_emu_mm_nt", &mm_nt);
  ops.impl("fp64_emu_bmm_nt", &bmm_nt);
  ops.impl("fp64_emu_mm_timed", &mm_timed);
  ops.impl("fp64_emu_gemm_ws", &gemm_ws);
  ops.impl("fp64_emu_gemm_ws_ev", &gemm_ws_ev);
  ops.impl("fp64_emu_gemm_checked", &gemm_checked);
  ops.impl("fp64_emu_host_submit", &host_submit);   // CPU operands, CUDA buffers: the CUDA key
  ops.impl("fp64_emu_status", &status);
  ops.impl("fp64_emu_debug_fetch", &debug_fetch);
  ops.impl("fp64_emu_wait_selftest", &wait_selftest);
}

// The 8-bit operators check shapes and types before they ask for the device;
// on the CPU they end with that refusal.
#define F64E_FP8_IMPLS(ops)                        \
  ops.impl("fp8_quantize", &fp8_quantize);         \
  ops.impl("fp8_quantize_both", &fp8_quantize_both); \
  ops.impl("fp8_dequantize", &fp8_dequantize);     \
  ops.impl("fp8_mm", &fp8_mm);                     \
  ops.impl("fp8_linear", &fp8_linear);
TORCH_LIBRARY_IMPL(fp64_emu_b200, CUDA, ops) { F64E_FP8_IMPLS(ops) }
TORCH_LIBRARY_IMPL(fp64_emu_b200, CPU, ops) { F64E_FP8_IMPLS(ops) }
#undef F64E_FP8_IMPLS

// Codes and scales carry no gradient; the layer has its own.
TORCH_LIBRARY_IMPL(fp64_emu_b200, Autograd, ops) {
  ops.impl("fp8_quantize", torch::CppFunction::makeFallthrough());
  ops.impl("fp8_quantize_both", torch::CppFunction::makeFallthrough());
  ops.impl("fp8_dequantize", torch::CppFunction::makeFallthrough());
  ops.impl("fp8_mm", torch::CppFunction::makeFallthrough());
  ops.impl("fp8_linear", &fp8_linear_autograd);
}
