// Products of block-scaled 8-bit codes: C[m][n] = sum_k a[m,k] b[n,k], the
// values being code * 2^e with one e for 128 neighbours along k.
//
// The codes go to the tensor cores as they are (tcgen05.mma kind::mxf8f6f4,
// FP32 accumulators in TMEM); the scales go with them, so nothing is
// multiplied or added on the CUDA cores before the one rounding of the output.
// Operands may be stored with k contiguous (K-major) or with m / n contiguous
// (MN-major): both are legal for 8-bit operands, so the three products of a
// layer and its gradients read the same tensors without a transposed copy.
#include <algorithm>
#include <map>
#include <mutex>

#include "f64e_fp8.cuh"
#include "f64e_fp8.h"

namespace f64e {

// First wait that ran out in a product on this device (kWait*), 0 if none.
__device__ int g_fp8_status;

namespace {

// ------------------------------------------------------------- epilogue --
// A warp's 32 rows x 128 bytes of output, staged in shared memory so that
// eight neighbouring lanes write one row's 128 bytes (16-byte chunks XORed
// with the row: both sides free of bank conflicts).
template <int OUT>
struct OutOf;
template <>
struct OutOf<F64E_F32> {
  static constexpr int kCols = 32;   // columns of a 128-byte row
};
template <>
struct OutOf<F64E_F16> {
  static constexpr int kCols = 64;
};
template <>
struct OutOf<F64E_BF16> {
  static constexpr int kCols = 64;
};

template <int OUT>
__device__ __forceinline__ uint32_t pack2(uint32_t lo, uint32_t hi) {
  if (OUT == F64E_F16) {
    const __half2 h = __floats2half2_rn(__uint_as_float(lo), __uint_as_float(hi));
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __nv_bfloat162 h = __floats2bfloat162_rn(__uint_as_float(lo), __uint_as_float(hi));
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Rows [0, rows) x columns [0, cols) of the staged block to out (row pitch
// ldo elements); vec: 16-byte stores are aligned.
template <int OUT>
__device__ __forceinline__ void store_staged(const uint8_t* stage, int lane, char* out, int64_t ldo, int rows,
                                             int cols, bool vec) {
  constexpr int ES = OUT == F64E_F32 ? 4 : 2, COLS = OutOf<OUT>::kCols, PER = 16 / ES;
  if (vec) {
    const int ch = lane & 7;
#pragma unroll
    for (int t = 0; t < 8; t++) {
      const int r = t * 4 + (lane >> 3);
      const uint8_t* s = stage + r * 128 + ((ch ^ (r & 7)) << 4);
      const uint4 v = *reinterpret_cast<const uint4*>(s);
      char* o = out + (int64_t)r * ldo * ES + ch * 16;
      if (r < rows) {
        if (ch * PER + PER <= cols) {
          *reinterpret_cast<uint4*>(o) = v;
        } else {
#pragma unroll
          for (int i = 0; i < PER; i++)
            if (ch * PER + i < cols) {
              if (ES == 4)
                reinterpret_cast<uint32_t*>(o)[i] = reinterpret_cast<const uint32_t*>(s)[i];
              else
                reinterpret_cast<uint16_t*>(o)[i] = reinterpret_cast<const uint16_t*>(s)[i];
            }
        }
      }
    }
  } else {
#pragma unroll 4
    for (int r = 0; r < 32; r++) {
      if (r >= rows) break;
#pragma unroll
      for (int h = 0; h < COLS / 32; h++) {
        const int c = h * 32 + lane, ch = c / PER;
        const uint8_t* s = stage + r * 128 + ((ch ^ (r & 7)) << 4) + (c % PER) * ES;
        char* o = out + ((int64_t)r * ldo + c) * ES;
        if (c < cols) {
          if (ES == 4)
            *reinterpret_cast<uint32_t*>(o) = *reinterpret_cast<const uint32_t*>(s);
          else
            *reinterpret_cast<uint16_t*>(o) = *reinterpret_cast<const uint16_t*>(s);
        }
      }
    }
  }
}

// 32 FP32 accumulators of this lane's row into its staged row, from column
// `half` * 32 on (half = 0 only, in 32 bits).
template <int OUT>
__device__ __forceinline__ void stage32(uint8_t* stage, int lane, int half, const uint32_t (&v)[32]) {
  uint8_t* row = stage + lane * 128;
  if (OUT == F64E_F32) {
#pragma unroll
    for (int i = 0; i < 8; i++)
      *reinterpret_cast<uint4*>(row + ((i ^ (lane & 7)) << 4)) =
          make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++)
      *reinterpret_cast<uint4*>(row + (((half * 4 + i) ^ (lane & 7)) << 4)) =
          make_uint4(pack2<OUT>(v[8 * i], v[8 * i + 1]), pack2<OUT>(v[8 * i + 2], v[8 * i + 3]),
                     pack2<OUT>(v[8 * i + 4], v[8 * i + 5]), pack2<OUT>(v[8 * i + 6], v[8 * i + 7]));
  }
}

// --------------------------------------------------------------- scales --
// The scale word of row r: bytes of blocks 4 j .. 4 j + 3, 0 outside the
// operand (its codes read as zeros there, and 0 is a finite scale).
__device__ __forceinline__ uint32_t scale_word(const Fp8Operand& o, int64_t rows, int nkb, int64_t r, int j,
                                               bool words) {
  if (r >= rows) return 0;
  const uint8_t* p = o.s + (r >> o.s_shift) * o.s_row + (int64_t)(4 * j) * o.s_kb;
  const int n = nkb - 4 * j;
  if (words && n >= 4) return __ldg(reinterpret_cast<const uint32_t*>(p));
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; i++)
    if (i < n) w |= (uint32_t)__ldg(p + i * o.s_kb) << (8 * i);
  return w;
}
// The atom of rows r0 .. r0 + 127 (a warp; lane = row of the atom).
__device__ __forceinline__ uint4 scale_atom(const Fp8Operand& o, int64_t rows, int nkb, int64_t r0, int j, int lane,
                                            bool words) {
  return make_uint4(scale_word(o, rows, nkb, r0 + lane, j, words), scale_word(o, rows, nkb, r0 + lane + 32, j, words),
                    scale_word(o, rows, nkb, r0 + lane + 64, j, words),
                    scale_word(o, rows, nkb, r0 + lane + 96, j, words));
}

struct GemmK {
  Fp8Operand a, b;
  int M, N, nkb;
  int64_t ldo;
  char* out;
  uint64_t wait_limit_ns;
  uint32_t idesc;
  int a_words, b_words;   // scales may be read four at a time
  int vec;                // 16-byte stores of the output are aligned
};

// --------------------------------------------------------------- CTA pair --
// A cluster of two CTAs on two SMs computes a 256 x 256 tile: CTA r holds rows
// [128 r, +128) of A's and of B's half tiles, and the leader's tcgen05.mma
// works on both.  Per SM and K = 32 step the tensor core then reads 8 KB of
// shared memory for 2^20 products; a lone CTA's 128 x 256 tile reads 12.
//   warp 0      TMA: 128 x 128 boxes of A and B, 128-byte swizzle, 5 stages
//   warp 1      TMEM owner; the leader's elected thread issues scale copies
//               and MMAs and commits stages and tiles to both CTAs
//   warps 2, 3  scales: gathered into atoms for 4 blocks of k at a time
//   warps 4..7  epilogue: 128 TMEM lanes, 32 columns at a time
// Every wait is bounded; one that runs out records its site and unwinds the
// CTA: copies and MMAs in flight are waited for before TMEM is freed (see the
// end of the kernel).
constexpr int BK = kFp8Block, BN = 256, PBM = 256, PHALF = 128, STAGES = 5, SF_STAGES = 4, PGROUP_M = 8;
constexpr int PTHREADS = 256;
constexpr uint32_t TILE_BYTES = PHALF * BK, STAGE_BYTES = 2 * TILE_BYTES;
constexpr uint32_t ATOM = 512, SF_BYTES = 3 * ATOM;   // A's rows, B's rows 0-127, 128-255
constexpr uint32_t STAGING = 4 * 32 * 128;
constexpr size_t PSMEM = 1024 + (size_t)STAGES * STAGE_BYTES + STAGING + SF_STAGES * SF_BYTES + 256;
constexpr uint32_t TMEM_COLS = 512, SF_COL = 256, SF_COLS = 12;   // scales: two buffers of 4 + 8 columns

enum : int { kWaitScales = 6, kWaitScalesFree = 7 };

__device__ __forceinline__ void tile_origin(int tile, int ntm, int ntn, int& m0, int& n0) {
  const int gsz = PGROUP_M * ntn;
  const int gi = tile / gsz, o = tile - gi * gsz;
  const int mf = gi * PGROUP_M, mh = min(PGROUP_M, ntm - mf);
  m0 = (mf + o % mh) * PBM;
  n0 = (o / mh) * BN;
}

template <int OUT>
__global__ void __launch_bounds__(PTHREADS, 1)
    fp8_gemm_pair_kernel(const __grid_constant__ CUtensorMap tmapA, const __grid_constant__ CUtensorMap tmapB,
                         const __grid_constant__ GemmK g) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_s = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw_s + 1023u) & ~1023u) - raw_s);
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * TILE_BYTES;
  uint8_t* staging = smem + STAGES * STAGE_BYTES;
  uint8_t* sSF = staging + STAGING;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(sSF + SF_STAGES * SF_BYTES);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* sf_full = empty_bar + STAGES;
  uint64_t* sf_empty = sf_full + SF_STAGES;
  uint64_t* acc_full = sf_empty + SF_STAGES;
  uint64_t* acc_empty = acc_full + 1;
  uint64_t* drain_bar = acc_empty + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile uint32_t* peer_issued = reinterpret_cast<volatile uint32_t*>(tmem_slot + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int cluster = blockIdx.x >> 1, nclusters = gridDim.x >> 1;
  const int ntm = (g.M + PBM - 1) / PBM, ntn = (g.N + BN - 1) / BN, ntiles = ntm * ntn;
  int* status = &g_fp8_status;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; s++) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int s = 0; s < SF_STAGES; s++) {
      mbar_init(&sf_full[s], 4);   // two loader warps of both CTAs
      mbar_init(&sf_empty[s], 1);
    }
    mbar_init(acc_full, 1);
    mbar_init(acc_empty, 2 * 4);   // the epilogue warps of both CTAs
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    *peer_issued = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmapA);
    tma_prefetch_desc(&tmapB);
  }
  __syncwarp();
  // TMEM: allocated by both CTAs once both run, the permit given up once both
  // have it (see residue_gemm_pair_kernel).
  cluster_sync();
  if (warp == 1) tmem_alloc_pair(tmem_slot, TMEM_COLS);
  tc_fence_before();
  __syncwarp();
  cluster_sync();
  tc_fence_after();
  if (warp == 1) tmem_relinquish_pair();
  const uint32_t tmem = *tmem_slot;
  const uint64_t lim = g.wait_limit_ns;
  const uint32_t full0 = mapa_shared(smem_u32(full_bar), 0);
  const uint32_t sffull0 = mapa_shared(smem_u32(sf_full), 0);
  const uint32_t accempty0 = mapa_shared(smem_u32(acc_empty), 0);

  uint32_t issued = 0;
  bool producer = false;
  if (warp == 0) {
    producer = elect_one();
    if (producer) {
      uint32_t j = 0;
      bool ok = true;
      for (int tile = cluster; tile < ntiles && ok; tile += nclusters) {
        int m0, n0;
        tile_origin(tile, ntm, ntn, m0, n0);
        const int ra = m0 + PHALF * (int)rank, rb = n0 + PHALF * (int)rank;
        for (int kb = 0; kb < g.nkb; kb++, j++) {
          const uint32_t s = j % STAGES, ph = (j / STAGES) & 1;
          if (!mbar_wait_poll(&empty_bar[s], ph ^ 1, lim, status, kWaitEmpty) || *abort_flag) {
            *abort_flag = 1;
            ok = false;
            break;
          }
          const int k = kb * BK;
          if (leader) mbar_arrive_expect_tx(&full_bar[s], 2 * STAGE_BYTES);
          tma_load_2d_pair(sA + s * TILE_BYTES, &tmapA, g.a.kmajor ? k : ra, g.a.kmajor ? ra : k, full0 + 8 * s);
          tma_load_2d_pair(sB + s * TILE_BYTES, &tmapB, g.b.kmajor ? k : rb, g.b.kmajor ? rb : k, full0 + 8 * s);
        }
      }
      issued = j;
      if (!leader) st_cluster_u32(mapa_shared(smem_u32((const void*)peer_issued), 0), j);
    }
  } else if (warp == 1) {
    if (leader && elect_one()) {
      uint32_t j = 0, it = 0, gr = 0;
      uint32_t last[2] = {0, 0};   // one past the last stage that used each scale buffer
      const uint32_t a_step = g.a.kmajor ? 32 : 32 * BK, b_step = g.b.kmajor ? 32 : 32 * BK;
      bool ok = true;
      for (int tile = cluster; tile < ntiles && ok; tile += nclusters, it++) {
        if (!mbar_wait_poll(acc_empty, (it & 1) ^ 1, lim, status, kWaitAccEmpty) || *abort_flag) {
          *abort_flag = 1;
          break;
        }
        tc_fence_after();
        uint32_t sf = 0;
        for (int kb = 0; kb < g.nkb; kb++, j++) {
          if ((kb & 3) == 0) {
            const uint32_t ss = gr % SF_STAGES, buf = gr & 1;
            bool got = mbar_wait_poll(&sf_full[ss], (gr / SF_STAGES) & 1, lim, status, kWaitScales);
            // The buffer's earlier MMAs have completed: by the ring (a stage
            // is filled again only after them), else by their own commit.
            if (got && last[buf] + STAGES > j + 1 && last[buf] > 0) {
              const uint32_t p = last[buf] - 1;
              got = mbar_wait_poll(&empty_bar[p % STAGES], (p / STAGES) & 1, lim, status, kWaitScales);
            }
            if (!got || *abort_flag) {
              *abort_flag = 1;
              ok = false;
              break;
            }
          }
          const uint32_t s = j % STAGES, ph = (j / STAGES) & 1;
          if (!mbar_wait_poll(&full_bar[s], ph, lim, status, kWaitFull) || *abort_flag) {
            *abort_flag = 1;
            ok = false;
            break;
          }
          tc_fence_after();
          if ((kb & 3) == 0) {
            const uint32_t ss = gr % SF_STAGES, buf = gr & 1, sa = smem_u32(sSF + ss * SF_BYTES);
            sf = tmem + SF_COL + buf * SF_COLS;
            copy_scales_pair(sf, smem_desc_scales(sa));
            copy_scales_pair(sf + 4, smem_desc_scales(sa + ATOM));
            copy_scales_pair(sf + 8, smem_desc_scales(sa + 2 * ATOM));
            tc_commit_pair(&sf_empty[ss], 0x3);
            gr++;
          }
          last[(gr - 1) & 1] = j + 1;
          const uint32_t a_addr = smem_u32(sA + s * TILE_BYTES), b_addr = smem_u32(sB + s * TILE_BYTES);
          const uint32_t id = g.idesc | idesc_scale_byte(kb & 3);
#pragma unroll
          for (int kk = 0; kk < BK / 32; kk++)
            mma_mx_pair(tmem, smem_desc_sw128(a_addr + kk * a_step), smem_desc_sw128(b_addr + kk * b_step), id, sf,
                        sf + 4, (kb | kk) != 0);
          tc_commit_pair(&empty_bar[s], 0x3);
        }
        if (ok) tc_commit_pair(acc_full, 0x3);
      }
      tc_commit_pair(drain_bar, 0x1);
      mbar_wait_poll(drain_bar, 0, drain_limit(lim), status, kWaitDrain);
    }
  } else if (warp < 4) {
    // Scales: warp 2 gathers A's atom (this CTA's rows), warp 3 both of B's.
    uint32_t gr = 0;
    bool ok = true;
    for (int tile = cluster; tile < ntiles && ok; tile += nclusters) {
      int m0, n0;
      tile_origin(tile, ntm, ntn, m0, n0);
      for (int kb = 0; kb < g.nkb; kb += 4, gr++) {
        const uint32_t ss = gr % SF_STAGES;
        uint8_t* dst = sSF + ss * SF_BYTES + lane * 16;
        uint4 u, v;
        if (warp == 2) {
          u = scale_atom(g.a, g.M, g.nkb, m0 + PHALF * (int)rank, kb >> 2, lane, g.a_words);
        } else {
          u = scale_atom(g.b, g.N, g.nkb, n0, kb >> 2, lane, g.b_words);
          v = scale_atom(g.b, g.N, g.nkb, n0 + 128, kb >> 2, lane, g.b_words);
        }
        if (!mbar_wait_poll(&sf_empty[ss], ((gr / SF_STAGES) & 1) ^ 1, lim, status, kWaitScalesFree) || *abort_flag) {
          *abort_flag = 1;
          ok = false;
          break;
        }
        if (warp == 2) {
          *reinterpret_cast<uint4*>(dst) = u;
        } else {
          *reinterpret_cast<uint4*>(dst + ATOM) = u;
          *reinterpret_cast<uint4*>(dst + 2 * ATOM) = v;
        }
        fence_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(sffull0 + 8 * ss);
      }
    }
  } else {
    const int q = warp & 3;
    constexpr int ES = OUT == F64E_F32 ? 4 : 2, COLS = OutOf<OUT>::kCols;
    uint8_t* stage = staging + q * (32 * 128);
    uint32_t it = 0;
    for (int tile = cluster; tile < ntiles; tile += nclusters, it++) {
      int m0, n0;
      tile_origin(tile, ntm, ntn, m0, n0);
      if (!mbar_wait_poll(acc_full, it & 1, lim, status, kWaitAccFull) || *abort_flag) {
        *abort_flag = 1;
        break;
      }
      tc_fence_after();
      const int row0 = m0 + PHALF * (int)rank + q * 32;
      const int rows = min(32, g.M - row0);
      const uint32_t taddr = tmem + ((uint32_t)(q * 32) << 16);
#pragma unroll 1
      for (int c = 0; c < BN; c += COLS) {
#pragma unroll
        for (int h = 0; h < COLS / 32; h++) {
          uint32_t v[32];
          tmem_ld_32x32b_x32(taddr + c + h * 32, v);
          tmem_wait_ld();
          stage32<OUT>(stage, lane, h, v);
        }
        if (c + COLS >= BN) {   // the tile has left TMEM
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(accempty0);
        }
        __syncwarp();
        store_staged<OUT>(stage, lane, g.out + ((int64_t)row0 * g.ldo + n0 + c) * ES, g.ldo, rows, g.N - n0 - c, g.vec);
        __syncwarp();
      }
    }
  }

  tc_fence_before();
  __syncwarp();
  cluster_sync();   // the peer's stage count is visible; the leader's MMAs have drained
  if (producer && leader) {
    // Every copy of the pair lands before either CTA releases its shared
    // memory: the accounting of residue_gemm_pair_kernel.
    const uint32_t jp = *peer_issued;
    const uint32_t jmax = issued > jp ? issued : jp;
    const uint32_t lo = jmax > (uint32_t)STAGES ? jmax - STAGES : 0;
    for (uint32_t jj = lo; jj < jmax; jj++) {
      const uint32_t s = jj % STAGES;
      if (jj >= issued) mbar_arrive_expect_tx(&full_bar[s], STAGE_BYTES);
      else if (jj >= jp) mbar_complete_tx(&full_bar[s], STAGE_BYTES);
      mbar_wait_poll(&full_bar[s], (jj / STAGES) & 1, drain_limit(lim), status, kWaitDrain);
    }
  }
  __syncwarp();
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, TMEM_COLS);
  }
}

// Codes as TMA sees them: 128 x 128-byte boxes of a [outer][inner] byte matrix
// with row pitch ld (a multiple of 16), zeros outside.
bool encode_codes(CUtensorMap* map, const void* base, int64_t outer, int64_t inner, int64_t ld) {
  using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static EncodeFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult qr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &qr) != cudaSuccess ||
        qr != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeFn>(f);
  }();
  if (!fn) return false;
  const cuuint64_t gdim[2] = {(cuuint64_t)inner, (cuuint64_t)outer};
  const cuuint64_t gstride[1] = {(cuuint64_t)ld};
  const cuuint32_t box[2] = {128, 128};
  const cuuint32_t estride[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), gdim, gstride, box, estride,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool scale_words(const Fp8Operand& o) {
  return o.s_kb == 1 && o.s_row % 4 == 0 && (reinterpret_cast<uintptr_t>(o.s) & 3) == 0;
}

template <int OUT>
cudaError_t launch_pair(const CUtensorMap& ta, const CUtensorMap& tb, const GemmK& k, int sms, cudaStream_t s) {
  const int64_t tiles = (int64_t)((k.M + PBM - 1) / PBM) * ((k.N + BN - 1) / BN);
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(2 * (sms / 2), 1, 1);
  cfg.blockDim = dim3(PTHREADS, 1, 1);
  cfg.dynamicSmemBytes = PSMEM;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  // per device: the shared-memory opt-in and the resident cluster count
  static std::mutex mtx;
  static std::map<int, int> clusters_of;
  std::unique_lock<std::mutex> lk(mtx);
  int& max_clusters = clusters_of.emplace(dev, -1).first->second;
  if (max_clusters < 0) {
    e = cudaFuncSetAttribute(fp8_gemm_pair_kernel<OUT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PSMEM);
    if (e != cudaSuccess) return e;
    int n = 0;
    e = cudaOccupancyMaxActiveClusters(&n, fp8_gemm_pair_kernel<OUT>, &cfg);
    if (e != cudaSuccess) return e;
    max_clusters = std::max(n, 1);
  }
  cfg.gridDim = dim3(2 * (unsigned)std::min<int64_t>(tiles, max_clusters), 1, 1);
  lk.unlock();
  return cudaLaunchKernelEx(&cfg, fp8_gemm_pair_kernel<OUT>, ta, tb, k);
}

}  // namespace

cudaError_t launch_fp8_gemm(const Fp8GemmArgs& g, cudaStream_t s) {
  CUtensorMap ta, tb;
  const bool ok = encode_codes(&ta, g.a.q, g.a.kmajor ? g.M : g.K, g.a.kmajor ? g.K : g.M, g.a.ld) &&
                  encode_codes(&tb, g.b.q, g.b.kmajor ? g.N : g.K, g.b.kmajor ? g.K : g.N, g.b.ld);
  if (!ok) return cudaErrorInvalidValue;
  GemmK k;
  k.a = g.a;
  k.b = g.b;
  k.M = (int)g.M;
  k.N = (int)g.N;
  k.nkb = (int)((g.K + BK - 1) / BK);
  k.ldo = g.ldo;
  k.out = static_cast<char*>(g.out);
  k.wait_limit_ns = g.wait_limit_ns;
  k.idesc = idesc_mx(PBM, BN, g.a.code, g.b.code, !g.a.kmajor, !g.b.kmajor);
  k.a_words = scale_words(g.a);
  k.b_words = scale_words(g.b);
  k.vec = (reinterpret_cast<uintptr_t>(g.out) & 15) == 0 && g.ldo * (g.out_type == F64E_F32 ? 4 : 2) % 16 == 0;
  switch (g.out_type) {
    case F64E_F32: return launch_pair<F64E_F32>(ta, tb, k, g.sms, s);
    case F64E_F16: return launch_pair<F64E_F16>(ta, tb, k, g.sms, s);
    default: return launch_pair<F64E_BF16>(ta, tb, k, g.sms, s);
  }
}

cudaError_t read_fp8_status(int* status, cudaStream_t s) {
  static const int zero = 0;
  cudaError_t e = cudaMemcpyFromSymbolAsync(status, g_fp8_status, sizeof(int), 0, cudaMemcpyDeviceToHost, s);
  if (e == cudaSuccess) e = cudaMemcpyToSymbolAsync(g_fp8_status, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, s);
  return e == cudaSuccess ? cudaStreamSynchronize(s) : e;
}

}  // namespace f64e
