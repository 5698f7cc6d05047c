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
#include <type_traits>

#include "f64e_fp8.cuh"
#include "f64e_fp8.h"

namespace f64e {

// First wait that ran out in a product on this device (kWait*), 0 if none.
__device__ int g_fp8_status;

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeFn encode_fn() {
  static EncodeFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult qr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &qr) != cudaSuccess ||
        qr != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeFn>(f);
  }();
  return fn;
}
bool fp8_encode_2d(CUtensorMap* map, CUtensorMapDataType type, void* base, int64_t inner, int64_t outer,
               int64_t pitch_bytes, int box_inner, int box_outer, CUtensorMapSwizzle swizzle) {
  const EncodeFn fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t gdim[2] = {(cuuint64_t)inner, (cuuint64_t)outer};
  const cuuint64_t gstride[1] = {(cuuint64_t)pitch_bytes};
  const cuuint32_t box[2] = {(cuuint32_t)box_inner, (cuuint32_t)box_outer};
  const cuuint32_t estride[2] = {1, 1};
  return fn(map, type, 2, base, gdim, gstride, box, estride, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// An operand as TMA sees it: boxes of 128 values of k by box_rows rows (128 when
// MN-major) of a byte matrix with pitch ld (a multiple of 16), 128-byte
// swizzle, zeros outside.
bool fp8_encode_codes(CUtensorMap* map, const Fp8Operand& o, int64_t rows, int64_t K, int box_rows) {
  return fp8_encode_2d(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, const_cast<uint8_t*>(o.q), o.kmajor ? K : rows,
                   o.kmajor ? rows : K, o.ld, 128, o.kmajor ? box_rows : 128, CU_TENSOR_MAP_SWIZZLE_128B);
}
int fp8_scale_mode(const Fp8Operand& o, int64_t rows, bool whole_squares) {
  if (o.s_shift && whole_squares) return kScaleTile;
  const bool base = (reinterpret_cast<uintptr_t>(o.s) & 3) == 0;
  if (base && o.s_kb == 1 && o.s_row % 4 == 0) return kScaleWords;
  if (base && !o.s_shift && o.s_row == 1 && o.s_kb % 4 == 0 && rows % 4 == 0) return kScaleRows;
  return kScaleBytes;
}

namespace {

// ------------------------------------------------------------- epilogue --
// A warp stages 2 KB of output rows in shared memory, 64 bytes of 32 rows (or
// 128 bytes of 16), 16-byte pieces XORed with the row number as in TMA's
// swizzle, which keeps the writes free of bank conflicts.  From there a TMA
// store takes them, or, where the output's rows are not on 16-byte boundaries,
// the warp itself, neighbouring lanes writing neighbouring elements.
constexpr uint32_t kStage = 2048;

template <int OUT>
struct OutOf {
  static constexpr int kBytes = OUT == F64E_F32 ? 4 : 2;
};

template <int RB>   // bytes of a staged row: 64 or 128
__device__ __forceinline__ uint32_t staged_at(int row, int piece) {
  return (uint32_t)(row * RB + ((RB == 64 ? piece ^ ((row >> 1) & 3) : piece ^ (row & 7)) << 4));
}

// The staged rows to out (row pitch ldo elements), of which `rows` rows and
// `cols` columns exist, W bytes a lane.
template <int OUT, int RB, int W>
__device__ __forceinline__ void store_staged(const uint8_t* stage, int lane, char* out, int64_t ldo, int rows,
                                             int cols) {
  constexpr int ES = OutOf<OUT>::kBytes, LANES = RB / W;                 // lanes of a row
  constexpr int ROWS = (int)kStage / RB, AT = 32 / LANES < 1 ? 1 : 32 / LANES;   // staged rows, rows written at once
  constexpr int U = W == 8 ? 2 : ES == 4 ? 4 : 8;                        // rows read before they are written
  using Word = std::conditional_t<W == 8, uint2, std::conditional_t<W == 4, uint32_t, uint16_t>>;
  const int at = lane % LANES * W, r0 = lane / LANES;
  const int left = cols - at / ES;   // elements of this lane that exist
  if (left <= 0) return;
  char* o = out + (int64_t)r0 * ldo * ES + at;
#pragma unroll
  for (int t = 0; t < ROWS / AT; t += U) {
    Word v[U];
#pragma unroll
    for (int u = 0; u < U; u++)
      v[u] = *reinterpret_cast<const Word*>(stage + staged_at<RB>((t + u) * AT + r0, at >> 4) + (at & 15));
#pragma unroll
    for (int u = 0; u < U; u++, o += AT * ldo * ES) {
      if ((t + u) * AT + r0 >= rows) continue;
      if (left * ES >= W) {
        *reinterpret_cast<Word*>(o) = v[u];
      } else {
#pragma unroll
        for (int i = 0; i < W / ES; i++)
          if (i < left) {
            if (ES == 4)
              reinterpret_cast<uint32_t*>(o)[i] = reinterpret_cast<const uint32_t*>(&v[u])[i];
            else
              reinterpret_cast<uint16_t*>(o)[i] = reinterpret_cast<const uint16_t*>(&v[u])[i];
          }
      }
    }
  }
}

// 64 / kBytes accumulators of this lane's row into its staged row.
template <int OUT>
__device__ __forceinline__ void stage_row(uint8_t* stage, int lane, const float* v) {
#pragma unroll
  for (int i = 0; i < 4; i++)
    if (OUT == F64E_F32)
      *reinterpret_cast<float4*>(stage + staged_at<64>(lane, i)) =
          make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    else
      *reinterpret_cast<uint4*>(stage + staged_at<64>(lane, i)) =
          make_uint4(Elem<OUT>::pack(v[8 * i], v[8 * i + 1]), Elem<OUT>::pack(v[8 * i + 2], v[8 * i + 3]),
                     Elem<OUT>::pack(v[8 * i + 4], v[8 * i + 5]), Elem<OUT>::pack(v[8 * i + 6], v[8 * i + 7]));
}
// The same of a transposed tile: this lane's accumulators are one column of
// the staged rows (32 columns).
template <int OUT>
__device__ __forceinline__ void stage_column(uint8_t* stage, int lane, const float* v) {
  constexpr int ES = OutOf<OUT>::kBytes, RB = 32 * ES, N = (int)kStage / RB;
  const int ch = lane * ES / 16, at = lane * ES % 16;
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    if (OUT == F64E_F32) {
      *reinterpret_cast<float*>(stage + staged_at<RB>(i, ch) + at) = v[i];
      *reinterpret_cast<float*>(stage + staged_at<RB>(i + 1, ch) + at) = v[i + 1];
    } else {
      const uint32_t p = Elem<OUT>::pack(v[i], v[i + 1]);
      *reinterpret_cast<uint16_t*>(stage + staged_at<RB>(i, ch) + at) = (uint16_t)p;
      *reinterpret_cast<uint16_t*>(stage + staged_at<RB>(i + 1, ch) + at) = (uint16_t)(p >> 16);
    }
  }
}

// The kernel's view of a product: a tile has rows of operand a and columns of
// operand b.  out element (row, col) is at row * ldo + col, or transposed.
struct GemmK {
  Fp8Operand a, b;
  int M, N, nkb;
  int64_t ldo;
  char* out;
  uint64_t wait_limit_ns;
  uint32_t idesc;
  int tma_out;            // the output's rows start and end on 16-byte boundaries
  int store_bytes;        // else: the boundaries they do start on, 2, 4 or 8
};

// --------------------------------------------------------------- CTA pair --
// A cluster of two CTAs on two SMs computes a 256 x 256 tile: CTA r holds rows
// [128 r, +128) of A's and of B's half tiles, and the leader's tcgen05.mma
// works on both, so an SM stages 32 KB for 128 values of k where a lone CTA's
// 128 x 256 tile would stage 48.
//   warp 0       TMA: 128 x 128 boxes of A and B, 5 stages
//   warp 1       TMEM owner; the leader's elected thread issues scale copies
//                and MMAs and commits stages and sums to both CTAs
//   warps 2, 3   scales: gathered into atoms for 4 blocks of k at a time
//   warps 4..11  epilogue: two warps for each 32 TMEM lanes, half the columns
//                each
// TMEM holds two accumulators, so MMAs run on while a tile is drained.  They
// and the scales exceed its 512 columns: the accumulators overlap by 32
// columns, which the epilogue drains first.
// Operand storage: the tensor cores read an MN-major A as fast as a K-major
// one, but take 1.6 times as long over an MN-major B (measured without the
// copies, 4096^3: 96 us against 59).  Such products are therefore computed transposed, with the
// operands' roles exchanged (TRANS), or after a transposition of one operand
// (launch_fp8_gemm).
// Sums: the tensor core truncates what an addition shifts out, an error that
// grows with the number of additions (part_blocks in f64e_fp8_split.cu has the
// measurements).  An accumulator therefore restarts after kChunk blocks of k
// for 32-bit outputs and kLongChunk for 16-bit ones, whose own rounding is far
// larger, and the parts are added in registers (PARTS; 16-bit outputs of up to
// kLongChunk blocks are stored straight from their one accumulator).
// Every wait is bounded; one that runs out records its site and unwinds the
// CTA: copies and MMAs in flight are waited for before TMEM is freed (see the
// end of the kernel).
constexpr int BK = kFp8Block, BN = 256, PBM = 256, PHALF = 128, STAGES = 5, SF_STAGES = 4, PGROUP_M = 8;
constexpr int EPI_WARPS = 8, PTHREADS = 32 * (4 + EPI_WARPS);
constexpr int kChunk = 16, kLongChunk = 1024;   // 2048 and 131072 values of k
constexpr uint32_t ATOM = 512, SF_BYTES = 3 * ATOM;   // A's rows, B's rows 0-127, 128-255
constexpr uint32_t TILE_BYTES = PHALF * BK, STAGE_BYTES = 2 * TILE_BYTES;
constexpr uint32_t TMEM_COLS = 512, ACC_COLS = 224, SF_COL = 480, SF_COLS = 12;   // scales: two buffers of 4 + 8
constexpr size_t PSMEM = 1024 + (size_t)STAGES * STAGE_BYTES + 2 * EPI_WARPS * kStage + SF_STAGES * SF_BYTES + 256;

__device__ __forceinline__ void tile_origin(int tile, int ntm, int ntn, int& m0, int& n0) {
  const int gsz = PGROUP_M * ntn;
  const int gi = tile / gsz, o = tile - gi * gsz;
  const int mf = gi * PGROUP_M, mh = min(PGROUP_M, ntm - mf);
  m0 = (mf + o % mh) * PBM;
  n0 = (o / mh) * BN;
}

template <int OUT, bool TRANS, bool PARTS>
__global__ void __launch_bounds__(PTHREADS, 1)
    fp8_gemm_pair_kernel(const __grid_constant__ CUtensorMap tmapA, const __grid_constant__ CUtensorMap tmapB,
                         const __grid_constant__ CUtensorMap tmapO, const __grid_constant__ GemmK g) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_s = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw_s + 1023u) & ~1023u) - raw_s);
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * TILE_BYTES;
  uint8_t* staging = smem + STAGES * STAGE_BYTES;
  uint8_t* sSF = staging + 2 * EPI_WARPS * kStage;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(sSF + SF_STAGES * SF_BYTES);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* sf_full = empty_bar + STAGES;
  uint64_t* sf_peer = sf_full + SF_STAGES;
  uint64_t* sf_empty = sf_peer + SF_STAGES;
  uint64_t* acc_full = sf_empty + SF_STAGES;
  uint64_t* acc_empty = acc_full + 1;
  uint64_t* drain_bar = acc_empty + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile uint32_t* peer_issued = reinterpret_cast<volatile uint32_t*>(tmem_slot + 2);
  volatile uint32_t* all_done = reinterpret_cast<volatile uint32_t*>(tmem_slot + 3);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int cluster = blockIdx.x >> 1, nclusters = gridDim.x >> 1;
  const int ntm = (g.M + PBM - 1) / PBM, ntn = (g.N + BN - 1) / BN, ntiles = ntm * ntn;
  const int chunk = !PARTS ? g.nkb : OUT == F64E_F32 ? kChunk : kLongChunk;   // blocks of k per accumulator
  int* status = &g_fp8_status;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; s++) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int s = 0; s < SF_STAGES; s++) {
      mbar_init(&sf_full[s], 2);   // the two loader warps
      mbar_init(&sf_peer[s], 1);   // the other CTA's scales (leader)
      mbar_init(&sf_empty[s], 1);
    }
    mbar_init(acc_full, 1);
    mbar_init(acc_empty, 2 * EPI_WARPS);   // the epilogue warps of both CTAs
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    *peer_issued = 0;
    *all_done = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmapA);
    tma_prefetch_desc(&tmapB);
  }
  // What can start early does: the first scales are gathered (two dependent
  // loads) while the CTAs of the pair meet and are handed over by the barrier
  // of the TMEM allocation; copies begin when both CTAs' barriers are known to
  // be set up.  One after the other, the first MMA came 3.5 us into the kernel.
  const uint64_t lim = g.wait_limit_ns;
  int m0, n0;
  tile_origin(cluster, ntm, ntn, m0, n0);
  uint32_t raw_a[4], raw_b[8];   // scales on their way (warp 2: this CTA's rows of A, warp 3: B's)
  auto gather = [&](int kb) {
    if (warp == 2)
      load_scales<1>(g.a, g.M, g.nkb, m0 + PHALF * (int)rank, kb >> 2, lane, raw_a);
    else
      load_scales<2>(g.b, g.N, g.nkb, n0, kb >> 2, lane, raw_b);
  };
  __syncwarp();
  cluster_arrive_relaxed();
  launch_next();
  launch_wait();
  if (warp == 2 || warp == 3) gather(0);
  cluster_wait();
  const uint32_t full0 = mapa_shared(smem_u32(full_bar), 0);
  const uint32_t sfpeer0 = mapa_shared(smem_u32(sf_peer), 0);
  const uint32_t accempty0 = mapa_shared(smem_u32(acc_empty), 0);
  auto stage_scales = [&](uint32_t ss) {
    if (warp == 2) {
      finish_scales<1>(g.a, raw_a);
      store_scales<1>(g.a, lane, raw_a, sSF + ss * SF_BYTES);
    } else {
      finish_scales<2>(g.b, raw_b);
      store_scales<2>(g.b, lane, raw_b, sSF + ss * SF_BYTES + ATOM);
    }
    fence_async_shared();
    __syncwarp();
  };
  auto load = [&](uint32_t s, int kb) {
    const int k = kb * BK, ra = m0 + PHALF * (int)rank, rb = n0 + PHALF * (int)rank;
    if (leader) mbar_arrive_expect_tx(&full_bar[s], 2 * STAGE_BYTES);
    tma_load_2d_pair(sA + s * TILE_BYTES, &tmapA, g.a.kmajor ? k : ra, g.a.kmajor ? ra : k, full0 + 8 * s);
    tma_load_2d_pair(sB + s * TILE_BYTES, &tmapB, g.b.kmajor ? k : rb, g.b.kmajor ? rb : k, full0 + 8 * s);
  };
  // TMEM: allocated by both CTAs once both run, the permit given up at the end
  // (see residue_gemm_pair_kernel).
  const bool uses_tmem = warp == 1 || warp >= 4;
  __syncwarp();
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, TMEM_COLS);
    tc_fence_before();
    __syncwarp();
  }
  if (warp == 2 || warp == 3) stage_scales(0);
  cluster_arrive();
  const bool producer = warp == 0 && elect_one();
  const int head = min(STAGES, g.nkb);   // blocks loaded ahead
  if (producer)
    for (int kb = 0; kb < head; kb++) load(kb, kb);
  if (uses_tmem) {
    cluster_wait();
    tc_fence_after();
  }
  const uint32_t tmem = uses_tmem ? *tmem_slot : 0;

  uint32_t issued = 0;
  if (warp == 0) {
    if (producer) {
      uint32_t j = head;
      bool ok = true;
      for (int tile = cluster; tile < ntiles && ok; tile += nclusters) {
        tile_origin(tile, ntm, ntn, m0, n0);
        for (int kb = tile == cluster ? head : 0; kb < g.nkb; kb++, j++) {
          const uint32_t s = j % STAGES, ph = (j / STAGES) & 1;
          if (!mbar_wait_poll(&empty_bar[s], ph ^ 1, lim, status, kWaitEmpty) || *abort_flag) {
            *abort_flag = 1;
            ok = false;
            break;
          }
          load(s, kb);
        }
      }
      issued = j;
      if (!leader) st_cluster_u32(mapa_shared(smem_u32((const void*)peer_issued), 0), j);
    }
  } else if (warp == 1) {
    if (leader) {
      // The whole warp runs the loop, so its counters and descriptors are
      // uniform; one thread issues.  A block of k has 512 cycles before the
      // tensor cores run dry, which the loop must not exceed: stage counters
      // instead of divisions, descriptors by addition, and no check of the
      // abort flag where a wait would notice.
      const bool issuer = elect_one();
      // K = 32 further on: 32 bytes along a K-major row, 32 rows of an MN-major box (in 16-byte units)
      const uint32_t a_step = (g.a.kmajor ? 32 : 32 * PHALF) >> 4, b_step = (g.b.kmajor ? 32 : 32 * PHALF) >> 4;
      const uint64_t desc_a = smem_desc_sw128(smem_u32(sA)), desc_b = smem_desc_sw128(smem_u32(sB));
      const uint64_t desc_sf = smem_desc_scales(smem_u32(sSF));
      uint32_t s = 0, ph = 0;        // stage and its parity
      uint32_t ss = 0, sph = 0;      // scale stage and its parity
      uint32_t j = 0, prev = 0;      // stages so far; where the previous group of 4 began
      uint32_t it = 0, gr = 0;
      bool ok = true;
      for (int tile = cluster; tile < ntiles && ok; tile += nclusters) {
        for (int kb = 0; kb < g.nkb && ok; it++) {   // an accumulator
          if (!warp_all(mbar_wait_poll(acc_empty, (it & 1) ^ 1, lim, status, kWaitAccEmpty) && !*abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t d_tmem = tmem + (it & 1) * ACC_COLS;
          const int end = min(kb + chunk, g.nkb);
          uint32_t accumulate = 0;
          while (kb < end && ok) {   // a group of 4 blocks
            // Its scales, both CTAs' (group 0's came with the allocation's barrier).
            if (gr > 0) {
              const uint32_t par = sph ^ (ss == 0);
              ok = warp_all(mbar_wait_poll(&sf_full[ss], par, lim, status, kWaitScales) &&
                            mbar_wait_poll<true>(&sf_peer[ss], par, lim, status, kWaitScales));
            }
            // Two buffers in TMEM: the MMAs of the group before the last have
            // completed, by the ring (a stage is filled again only after
            // them) or, after short groups, by their own commit.
            if (ok && prev + STAGES > j + 1 && prev > 0) {
              const uint32_t p = prev - 1;
              ok = warp_all(mbar_wait_poll(&empty_bar[p % STAGES], (p / STAGES) & 1, lim, status, kWaitScales));
            }
            prev = j;
            const uint32_t sf = tmem + SF_COL + (gr & 1) * SF_COLS;
            const int last = min(kb + 4, end);
            for (uint32_t i = 0; kb < last && ok; kb++, i++, j++) {
              if (!warp_all(mbar_wait_poll(&full_bar[s], ph, lim, status, kWaitFull))) {
                ok = false;
                break;
              }
              if (issuer) {
                if (i == 0) {
                  const uint64_t d = desc_sf + ss * (SF_BYTES >> 4);
                  tc_fence_after();
                  copy_scales_pair(sf, d);
                  copy_scales_pair(sf + 4, d + (ATOM >> 4));
                  copy_scales_pair(sf + 8, d + (2 * ATOM >> 4));
                  tc_commit_pair(&sf_empty[ss], 0x3);
                }
                const uint64_t da = desc_a + s * (TILE_BYTES >> 4), db = desc_b + s * (TILE_BYTES >> 4);
                const uint32_t id = g.idesc | idesc_scale_byte(i);
                mma_mx_pair(d_tmem, da, db, id, sf, sf + 4, accumulate);
#pragma unroll
                for (int kk = 1; kk < BK / 32; kk++)
                  mma_mx_pair(d_tmem, da + kk * a_step, db + kk * b_step, id, sf, sf + 4, 1);
                tc_commit_pair(&empty_bar[s], 0x3);
              }
              accumulate = 1;
              if (++s == STAGES) {
                s = 0;
                ph ^= 1;
              }
            }
            gr++;
            if (++ss == SF_STAGES) {
              ss = 0;
              sph ^= 1;
            }
          }
          if (ok && issuer) tc_commit_pair(acc_full, 0x3);
        }
      }
      if (!ok) *abort_flag = 1;
      // Every copy was waited for above and every MMA is waited for here: both
      // CTAs may then leave at the next barrier.
      if (issuer) {
        tc_commit_pair(drain_bar, 0x1);
        if (mbar_wait_poll(drain_bar, 0, drain_limit(lim), status, kWaitDrain) && ok)
          for (uint32_t r = 0; r < 2; r++) st_cluster_u32(mapa_shared(smem_u32((const void*)all_done), r), 1);
      }
    } else {
      // The other CTA passes on to the leader which of its scales are in place:
      // a release at cluster scope takes too long (550 cycles or more) for the
      // warps that gather them.
      uint32_t ss = 1, par = 0;
      for (int tile = cluster; tile < ntiles; tile += nclusters)
        for (int kb = tile == cluster ? 4 : 0; kb < g.nkb; kb += 4) {
          if (!warp_all(mbar_wait_poll(&sf_full[ss], par ^ (ss == 0), lim, status, kWaitScales) && !*abort_flag)) {
            *abort_flag = 1;
            tile = ntiles;
            break;
          }
          if (lane == 0) mbar_arrive_cluster(sfpeer0 + 8 * ss);
          if (++ss == SF_STAGES) {
            ss = 0;
            par ^= 1;
          }
        }
    }
  } else if (warp < 4) {
    // Scales, a group of 4 blocks after the other; the next group's loads are
    // issued before this one's place is waited for.
    int tile = cluster, kb = 0;
    auto advance = [&]() {   // to the next group; its loads
      kb += 4;
      if (kb >= g.nkb) {
        kb = 0;
        tile += nclusters;
        if (tile < ntiles) tile_origin(tile, ntm, ntn, m0, n0);
      }
      if (tile < ntiles) gather(kb);
      return tile < ntiles;
    };
    uint32_t ss = 1, par = 1;   // group 0 is in place
    for (bool more = advance(); more;) {
      uint32_t now_a[4], now_b[8];
#pragma unroll
      for (int i = 0; i < 4; i++) now_a[i] = raw_a[i];
#pragma unroll
      for (int i = 0; i < 8; i++) now_b[i] = raw_b[i];
      if (warp == 2)
        finish_scales<1>(g.a, now_a);
      else
        finish_scales<2>(g.b, now_b);
      more = advance();
      if (!warp_all(mbar_wait_poll(&sf_empty[ss], par, lim, status, kWaitScalesFree) && !*abort_flag)) {
        *abort_flag = 1;
        break;
      }
      if (warp == 2)
        store_scales<1>(g.a, lane, now_a, sSF + ss * SF_BYTES);
      else
        store_scales<2>(g.b, lane, now_b, sSF + ss * SF_BYTES + ATOM);
      fence_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sf_full[ss]);
      if (++ss == SF_STAGES) {
        ss = 0;
        par ^= 1;
      }
    }
  } else {
    // Epilogue: warp q of 4 by lanes, half h of the columns.  A warp arrives on
    // acc_empty once per accumulator, after its first 32 columns of it: by then
    // it has left the other accumulator, and the columns both share (the last
    // of the first accumulator, the first of the second) are in registers,
    // since the half that holds them starts there.
    const int q = warp & 3, h = (warp - 4) >> 2;
    constexpr int ES = OutOf<OUT>::kBytes, COLS = 64 / ES, NP = BN / 2 / COLS;   // columns and number of a warp's passes
    uint32_t it = 0, puts = 0;
    bool ok = true;
    for (int tile = cluster; tile < ntiles && ok; tile += nclusters) {
      tile_origin(tile, ntm, ntn, m0, n0);
      const int row0 = m0 + PHALF * (int)rank + q * 32;
      auto column = [&](int p) { return h * (BN / 2) + (h ? NP - 1 - p : p) * COLS; };
      auto release = [&]() {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster_relaxed(accempty0);
      };
      auto put = [&](int p, const float* v) {
        constexpr int RB = TRANS ? 32 * ES : 64;
        const int col0 = n0 + column(p);
        // Nothing to write; and every block that takes a buffer has a store,
        // which the wait below counts on.
        if (row0 >= g.M || col0 >= g.N) return;
        uint8_t* stage = staging + (2 * (warp - 4) + (puts++ & 1)) * kStage;
        if (g.tma_out) {   // the store before the last has been read
          if (lane == 0) tma_store_wait_read<1>();
          __syncwarp();
        }
        if (TRANS)
          stage_column<OUT>(stage, lane, v);
        else
          stage_row<OUT>(stage, lane, v);
        if (g.tma_out) {
          fence_async_shared();
          __syncwarp();
          if (lane == 0) tma_store_2d(&tmapO, TRANS ? row0 : col0, TRANS ? col0 : row0, stage);
        } else {
          __syncwarp();
          const int orow = TRANS ? col0 : row0, ocol = TRANS ? row0 : col0;
          const int rows = TRANS ? g.N - col0 : g.M - row0, cols = TRANS ? g.M - row0 : g.N - col0;
          char* o = g.out + ((int64_t)orow * g.ldo + ocol) * ES;
          if (g.store_bytes == 8)
            store_staged<OUT, RB, 8>(stage, lane, o, g.ldo, rows, cols);
          else if (g.store_bytes == 4)
            store_staged<OUT, RB, 4>(stage, lane, o, g.ldo, rows, cols);
          else if (ES == 2)
            store_staged<OUT, RB, 2>(stage, lane, o, g.ldo, rows, cols);
          __syncwarp();
        }
      };
      float sum[PARTS ? NP : 1][COLS];
      for (int kb = 0; kb < g.nkb; kb += chunk, it++) {
        if (!warp_all(mbar_wait_poll(acc_full, it & 1, lim, status, kWaitAccFull) && !*abort_flag)) {
          *abort_flag = 1;
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t taddr = tmem + ((uint32_t)(q * 32) << 16) + (it & 1) * ACC_COLS;
#pragma unroll
        for (int p = 0; p < NP; p++) {
          if constexpr (PARTS) {
#pragma unroll
            for (int c = 0; c < COLS; c += 16) {
              uint32_t v[16];
              tmem_ld_32x32b_x16(taddr + column(p) + c, v);
              tmem_wait_ld();
              if (p * COLS + c == 16) release();   // 32 columns
#pragma unroll
              for (int k = 0; k < 16; k++)
                sum[p][c + k] = kb == 0 ? __uint_as_float(v[k]) : sum[p][c + k] + __uint_as_float(v[k]);
            }
          } else {
            uint32_t v[32];
            tmem_ld_32x32b_x32(taddr + column(p), v);
            tmem_wait_ld();
            if (p == 0) release();
            put(p, reinterpret_cast<const float*>(v));
          }
        }
      }
      if (PARTS && ok) {
#pragma unroll
        for (int p = 0; p < NP; p++) put(p, sum[p]);
      }
    }
    if (lane == 0) tma_store_wait();   // shared memory outlives the stores
  }

  if (!uses_tmem) cluster_wait();   // the allocation's barrier
  tc_fence_before();
  __syncwarp();
  cluster_sync();   // the leader's MMAs have drained; the peer's stage count is visible
  if (!*all_done) {
    // A wait ran out.  Every copy of the pair lands before either CTA releases
    // its shared memory: the accounting of residue_gemm_pair_kernel.
    if (producer && leader) {
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
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_relinquish_pair();
    tmem_dealloc_pair(tmem, TMEM_COLS);
  }
}

// The output in boxes of one staged block.
template <int OUT, bool TRANS>
bool encode_out(CUtensorMap* map, const GemmK& k) {
  constexpr int ES = OutOf<OUT>::kBytes, RB = TRANS ? 32 * ES : 64;
  return fp8_encode_2d(map, ES == 4 ? CU_TENSOR_MAP_DATA_TYPE_UINT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, k.out,
                   TRANS ? k.M : k.N, TRANS ? k.N : k.M, k.ldo * ES, RB / ES, (int)kStage / RB,
                   RB == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int OUT, bool TRANS, bool PARTS>
cudaError_t launch_pair(const GemmK& k, int64_t K, int sms, cudaStream_t s) {
  CUtensorMap ta, tb;
  CUtensorMap to = {};
  if (!fp8_encode_codes(&ta, k.a, k.M, K, 128) || !fp8_encode_codes(&tb, k.b, k.N, K, 128) ||
      (k.tma_out && !encode_out<OUT, TRANS>(&to, k)))
    return cudaErrorInvalidValue;
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
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  // per device: the shared-memory opt-in and the resident cluster count
  static std::mutex mtx;
  static std::map<int, int> clusters_of;
  std::unique_lock<std::mutex> lk(mtx);
  int& max_clusters = clusters_of.emplace(dev, -1).first->second;
  if (max_clusters < 0) {
    e = cudaFuncSetAttribute(fp8_gemm_pair_kernel<OUT, TRANS, PARTS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PSMEM);
    if (e != cudaSuccess) return e;
    int n = 0;
    e = cudaOccupancyMaxActiveClusters(&n, fp8_gemm_pair_kernel<OUT, TRANS, PARTS>, &cfg);
    if (e != cudaSuccess) return e;
    max_clusters = std::max(n, 1);
  }
  const int64_t tiles = (int64_t)((k.M + PBM - 1) / PBM) * ((k.N + BN - 1) / BN);
  const unsigned grid = 2 * (unsigned)std::min<int64_t>(tiles, max_clusters);
  lk.unlock();
  return fp8_launch(fp8_gemm_pair_kernel<OUT, TRANS, PARTS>, grid, PTHREADS, PSMEM, 2, s, ta, tb, to, k);
}

template <int OUT>
cudaError_t launch_out(const GemmK& k, bool trans, int64_t K, int sms, cudaStream_t s) {
  if (OUT == F64E_F32 || k.nkb > kLongChunk)
    return trans ? launch_pair<OUT, true, true>(k, K, sms, s) : launch_pair<OUT, false, true>(k, K, sms, s);
  constexpr bool parts = OUT == F64E_F32;   // no such instance without parts
  return trans ? launch_pair<OUT, true, parts>(k, K, sms, s) : launch_pair<OUT, false, parts>(k, K, sms, s);
}

// ------------------------------------------------------ transposed copies --
// [K][rows] codes to [rows][ldt], zeros up to ldt (K rounded up to 16): squares
// of 128 x 128 through shared memory, 4 x 4 bytes transposed in registers.
__global__ void __launch_bounds__(256) fp8_transpose_kernel(const uint8_t* q, int64_t ld, int64_t rows, int64_t K,
                                                            uint8_t* t, int64_t ldt, int64_t nrb) {
  __shared__ uint32_t sm[128][33];   // [row][k / 4], one word of padding
  const int64_t r0 = (blockIdx.x % nrb) * 128, k0 = (blockIdx.x / nrb) * 128;
  const int rg = threadIdx.x & 31, kg0 = threadIdx.x >> 5;   // 4 rows by 4 k each
  uint32_t w[4][4];
  launch_next();
  launch_wait();
#pragma unroll
  for (int u = 0; u < 4; u++)
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int64_t k = k0 + (u * 8 + kg0) * 4 + i, r = r0 + rg * 4;
      const uint8_t* p = q + k * ld + r;
      uint32_t v = 0;
      if (k < K) {
        if (r + 4 <= rows) {
          v = *reinterpret_cast<const uint32_t*>(p);
        } else {
#pragma unroll
          for (int b = 0; b < 4; b++)
            if (r + b < rows) v |= (uint32_t)p[b] << (8 * b);
        }
      }
      w[u][i] = v;
    }
#pragma unroll
  for (int u = 0; u < 4; u++) {
    const uint32_t a = __byte_perm(w[u][0], w[u][1], 0x5140), b = __byte_perm(w[u][2], w[u][3], 0x5140);
    const uint32_t c = __byte_perm(w[u][0], w[u][1], 0x7362), d = __byte_perm(w[u][2], w[u][3], 0x7362);
    const int kg = u * 8 + kg0;
    sm[rg * 4][kg] = __byte_perm(a, b, 0x5410);
    sm[rg * 4 + 1][kg] = __byte_perm(a, b, 0x7632);
    sm[rg * 4 + 2][kg] = __byte_perm(c, d, 0x5410);
    sm[rg * 4 + 3][kg] = __byte_perm(c, d, 0x7632);
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < 4; u++) {
    const int row = u * 32 + (threadIdx.x >> 3), ch = threadIdx.x & 7;
    const int64_t r = r0 + row, k = k0 + ch * 16;
    if (r < rows && k < ldt)
      *reinterpret_cast<uint4*>(t + r * ldt + k) =
          make_uint4(sm[row][ch * 4], sm[row][ch * 4 + 1], sm[row][ch * 4 + 2], sm[row][ch * 4 + 3]);
  }
}

int64_t round16(int64_t v) { return (v + 15) & ~(int64_t)15; }

// Whether one of two MN-major operands is transposed first: where the time won
// on the tensor cores (waves of tiles times blocks of k) exceeds a launch and
// a pass over the smaller operand.
bool transpose_first(int64_t M, int64_t N, int64_t K, int sms) {
  const int64_t tiles = ((M + PBM - 1) / PBM) * ((N + BN - 1) / BN);
  const int64_t waves = (tiles + sms / 2 - 1) / (sms / 2);
  return waves * ((K + BK - 1) / BK) >= 32;
}

}  // namespace

// Decided for 148 SMs whatever the device: the size is asked for without one,
// and the product decides by the same call.
int64_t fp8_gemm_workspace(const Fp8GemmArgs& g) {
  constexpr int kSms = 148;
  if (g.a.kmajor || g.b.kmajor || !transpose_first(g.M, g.N, g.K, kSms)) return 0;
  return std::min(g.M, g.N) * round16(g.K);
}

cudaError_t launch_fp8_gemm(const Fp8GemmArgs& g, void* workspace, cudaStream_t s) {
  // Fewer tiles than CTA pairs: perhaps smaller tiles with K split over more of
  // the SMs.  What a wave of pairs takes, in cycles: 600 a block of k (512 of
  // MMAs), 11000 to start and to write the last tile, and what rows of the
  // output that are not on 16-byte boundaries add (measured: 777 x 2043 x 1234
  // in 32 bits 17.2 us, 13.8 with 2048 columns, 11.4 on tiles of 128 x 112).
  const int es = g.out_type == F64E_F32 ? 4 : 2;
  const bool tma_out =
      (reinterpret_cast<uintptr_t>(g.out) & 15) == 0 && g.ldo * es % 16 == 0 && g.N * es % 16 == 0;
  if (((g.M + PBM - 1) / PBM) * ((g.N + BN - 1) / BN) <= g.sms / 2) {
    bool done = false;
    const int64_t pairs_cost = (g.K + BK - 1) / BK * 600 + 11000 + (tma_out ? 0 : es == 4 ? 8000 : 3000);
    const cudaError_t e = launch_fp8_split(g, pairs_cost, &done, s);
    if (e != cudaSuccess || done) return e;
  }
  GemmK k;
  k.a = g.a;
  k.b = g.b;
  const int64_t need = fp8_gemm_workspace(g);
  if (need > 0) {
    const bool a_side = g.M < g.N;
    Fp8Operand& o = a_side ? k.a : k.b;
    const int64_t rows = a_side ? g.M : g.N, nrb = (rows + 127) / 128;
    uint8_t* t = static_cast<uint8_t*>(workspace);
    const cudaError_t e = fp8_launch(fp8_transpose_kernel, (unsigned)(nrb * ((g.K + 127) / 128)), 256, 0, 0, s, o.q, o.ld,
                                     rows, g.K, t, round16(g.K), nrb);
    if (e != cudaSuccess) return e;
    o.q = t;
    o.ld = round16(g.K);
    o.kmajor = 1;
  }
  const bool trans = !k.b.kmajor && k.a.kmajor;   // the MN-major operand takes A's place
  if (trans) std::swap(k.a, k.b);
  k.M = (int)(trans ? g.N : g.M);
  k.N = (int)(trans ? g.M : g.N);
  k.nkb = (int)((g.K + BK - 1) / BK);
  k.ldo = g.ldo;
  k.out = static_cast<char*>(g.out);
  k.wait_limit_ns = g.wait_limit_ns;
  k.idesc = idesc_mx(PBM, BN, k.a.code, k.b.code, !k.a.kmajor, !k.b.kmajor);
  k.a.s_mode = fp8_scale_mode(k.a, k.M, true);
  k.b.s_mode = fp8_scale_mode(k.b, k.N, true);
  // A TMA store clips a row's end at 16 bytes: the output's columns must fill
  // them (with a wider pitch, what follows would be overwritten).
  k.tma_out = tma_out;
  const int64_t pitch = g.ldo * es;
  k.store_bytes = 8;
  while (reinterpret_cast<uintptr_t>(g.out) % k.store_bytes || pitch % k.store_bytes) k.store_bytes /= 2;
  switch (g.out_type) {
    case F64E_F32: return launch_out<F64E_F32>(k, trans, g.K, g.sms, s);
    case F64E_F16: return launch_out<F64E_F16>(k, trans, g.K, g.sms, s);
    default: return launch_out<F64E_BF16>(k, trans, g.K, g.sms, s);
  }
}

// Nothing arrives at the barrier and nothing else is in flight: the kernel returns.
__global__ void fp8_wait_selftest_kernel(uint64_t limit_ns) {
  __shared__ __align__(8) uint64_t bar;
  if (elect_one()) {
    mbar_init(&bar, 1);
    fence_barrier_init();
    mbar_wait_poll(&bar, 0, limit_ns, &g_fp8_status, kWaitSelfTest);
  }
}
cudaError_t launch_fp8_wait_selftest(uint64_t limit_ns, cudaStream_t s) {
  fp8_wait_selftest_kernel<<<1, 32, 0, s>>>(limit_ns);
  return cudaGetLastError();
}

cudaError_t read_fp8_status(int* status, cudaStream_t s) {
  static const int zero = 0;
  int split = 0;
  cudaError_t e = read_fp8_split_status(&split, s);
  if (e == cudaSuccess) e = cudaMemcpyFromSymbolAsync(status, g_fp8_status, sizeof(int), 0, cudaMemcpyDeviceToHost, s);
  if (e == cudaSuccess) e = cudaMemcpyToSymbolAsync(g_fp8_status, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  if (e == cudaSuccess && !*status) *status = split;
  return e;
}

}  // namespace f64e
