// Products of block-scaled 8-bit codes with few rows or columns: a served
// layer on a handful of tokens, a small batch.
//
// A CTA computes 128 rows of the large ("wide") operand by up to 128 columns of
// the small ("thin") one, and a cluster of up to eight CTAs shares the tile's K,
// so that a product with few tiles still draws on most SMs: bound by reading
// the wide operand, it needs their copies in flight (10 stages of 16 KB each),
// not their tensor cores.  The partial sums meet in shared memory:
// every CTA adds a share of the tile, in the order of the K ranges, so results
// do not depend on timing and no scratch or second launch is needed.
//
// With x in 16 or 32 bits (a served layer on up to kFusedRows tokens), the
// CTAs quantise the blocks of x they contract themselves: row blocks are 128
// values of k, so a block is quantised within one step of the K loop.
//   warp 0       TMA: 128 x 128 boxes of the wide operand (and the thin one's)
//   warp 1       TMEM owner; one thread issues scale copies and MMAs (tcgen05,
//                cta_group::1)
//   warps 2, 3   scales of the wide and the thin operand, four blocks of k a
//                gather
//   warps 4..    quantisation of x (eight warps); epilogue (four)
// Every wait is bounded; one that runs out records its site, and the CTA goes
// on to the cluster barriers without storing.
#include <algorithm>
#include <array>
#include <map>
#include <mutex>

#include "f64e_fp8.cuh"
#include "f64e_fp8.h"

namespace f64e {

// First wait that ran out in one of these kernels on this device, 0 if none.
__device__ int g_fp8_split_status;

namespace {

constexpr int kBlock = kFp8Block, kRows = 128;
constexpr int kMaxStages = 10, kMaxSplit = 8, kMaxCols = 128;
constexpr uint32_t kWideBytes = kRows * kBlock, kAtom = 512;
constexpr uint32_t kRing = 190 * 1024;   // shared memory for stages
// More than half an SM's shared memory: no two kernels of this library that
// hold TMEM share an SM.  A CTA that waited for TMEM held by a CTA of another
// cluster, which waits at its cluster barrier for a CTA that waits in turn,
// would wait for good.
constexpr size_t kMinSmem = 120 * 1024;
// Floats from one column of partial sums to the next: four rows of eight
// neighbouring columns lie in different banks.
constexpr int kPitch = kRows + 4;
// Accumulators of a CTA: each holds part_blocks() blocks of k at most.  Parts
// that TMEM holds beside one another wait there for the end; more of them take
// turns in two accumulators, and the epilogue's warps, idle until then, add
// each part to a sum kept in TMEM too.
constexpr int kTurnParts = 3;            // two accumulators and the sum

struct SplitArgs {
  Fp8Operand w, x;      // wide, thin (fused: x's codes and scales unused)
  int rows, cols;       // extents of the wide and the thin operand
  int nkb;              // blocks of k
  int bn, nst, split;   // columns of a tile, stages, CTAs per tile
  int tiles_r;          // tiles along the wide operand
  int nacc;             // accumulators (their sums are added at the end), or:
  int turns;            // blocks of a part, where parts take turns in two of them; 0
  uint32_t tmem_cols, idesc;
  char* out;
  int64_t out_r, out_c;   // output strides (elements) along rows and columns
  int vec;                // four rows of a column may be stored at once
  const void* xf;         // fused: x [cols][ldx]
  int64_t ldx, K;
  int x_vec, x_wide;
  uint32_t ring;          // bytes of shared memory before the scales: stages, then partial sums
  uint64_t wait_limit_ns;
};

__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// Warps that quantise x, the epilogue's four among them.
template <int XT>
constexpr int kQuantWarps = XT >= 0 ? 8 : 4;

// XT: type of x when the kernel quantises it, -1 for codes.  TURNS: parts take
// turns in two accumulators (an instance of its own: that code inline cost the
// others, 8 us kernels whose instructions are fetched anew each time, 0.1 us).
template <int OUT, int XT, bool TURNS>
__global__ void __launch_bounds__(32 * (4 + kQuantWarps<XT>), 1)
    fp8_split_kernel(const __grid_constant__ CUtensorMap tmapW, const __grid_constant__ CUtensorMap tmapX,
                     const __grid_constant__ SplitArgs g) {
  constexpr bool FUSED = XT >= 0;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_s = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw_s + 1023u) & ~1023u) - raw_s);
  const uint32_t thin_bytes = g.bn * kBlock, stage_bytes = kWideBytes + thin_bytes;
  uint8_t* sSF = smem + g.ring;
  uint64_t* full = reinterpret_cast<uint64_t*>(sSF + g.nst * 2 * kAtom);
  uint64_t* empty = full + kMaxStages;
  uint64_t* sf_full = empty + kMaxStages;
  uint64_t* acc_full = sf_full + kMaxStages;
  uint64_t* part_full = acc_full + 1;   // [2], and the part's accumulator read: [2]
  uint64_t* part_empty = part_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(part_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)(blockIdx.x % g.split), tile = (int)(blockIdx.x / g.split);
  const int r0 = (tile % g.tiles_r) * kRows, c0 = (tile / g.tiles_r) * g.bn;
  const int kb0 = (int)((int64_t)g.nkb * rank / g.split), kb1 = (int)((int64_t)g.nkb * (rank + 1) / g.split);
  const int cols = min(g.bn, g.cols - c0);
  const int turns = TURNS ? g.turns : 0;
  const int per = turns ? turns : (kb1 - kb0 + g.nacc - 1) / g.nacc;   // blocks per accumulator
  const uint64_t lim = g.wait_limit_ns;
  int* status = &g_fp8_split_status;

  // Before the CTA meets: the copies that need no free stage, the first scales
  // and the first blocks of x are on their way, and TMEM is allocated.
  const int n = kb1 - kb0, head = min(n, g.nst);
  auto load = [&](int i, int s) {
    const int k = (kb0 + i) * kBlock;
    uint8_t* st = smem + s * stage_bytes;
    mbar_arrive_expect_tx(&full[s], FUSED ? kWideBytes : stage_bytes);
    tma_load_2d(st, &tmapW, g.w.kmajor ? k : r0, g.w.kmajor ? r0 : k, &full[s]);
    if (!FUSED) tma_load_2d(st + kWideBytes, &tmapX, k, c0, &full[s]);
  };
  uint32_t raw[4] = {};   // scales on their way (warp 2: wide, warp 3: thin)
  auto gather = [&](int kb) {
    if (warp == 2)
      load_scales<1>(g.w, g.rows, g.nkb, r0, kb >> 2, lane, raw);
    else
      load_scales<1>(g.x, g.cols, g.nkb, c0, kb >> 2, lane, raw);
  };
  // Blocks of x in registers: warp 4 + b takes every QW-th block of k, from
  // the b-th on, of all rows: rows 4 p + lane / 8, eight lanes a block.
  constexpr int QW = kQuantWarps<XT>;
  constexpr int PASSES = kFusedRows / 4;
  using EX = Elem<FUSED ? XT : F64E_BF16>;
  const int l = lane & 7;
  uint32_t v[PASSES][EX::kWords];
  auto load_x = [&](int i) {
    if constexpr (FUSED) {
      const int64_t k = (int64_t)(kb0 + i) * kBlock + l * 16;
      const typename EX::type* x = static_cast<const typename EX::type*>(g.xf) + (int64_t)(c0 + (lane >> 3)) * g.ldx + k;
      const bool whole = g.x_vec && (int64_t)(kb0 + i + 1) * kBlock <= g.K;
#pragma unroll
      for (int p = 0; p < PASSES; p++) {
        if (p * 4 >= cols) break;
        const bool row = p * 4 + (lane >> 3) < cols;
        if (whole) {
          if (row) load16<XT>(x + p * 4 * g.ldx, g.x_wide, v[p]);
        } else {
          load16_some<XT>(x + p * 4 * g.ldx, 1, row ? g.K - k : 0, v[p]);
        }
      }
    }
  };
  launch_next();
  if (warp == 0) {
    if (elect_one()) {
      for (int s = 0; s < g.nst; s++) mbar_init(&full[s], 1);
      fence_barrier_init();
      launch_wait();
      for (int i = 0; i < head; i++) load(i, i);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      for (int s = 0; s < g.nst; s++) mbar_init(&empty[s], 1);
      mbar_init(acc_full, 1);
      for (int i = 0; i < 2 && TURNS; i++) {
        mbar_init(&part_full[i], 1);
        mbar_init(&part_empty[i], 4);   // the epilogue's warps
      }
      *abort_flag = 0;
      fence_barrier_init();
    }
    __syncwarp();
    tmem_alloc(tmem_slot, g.tmem_cols);
    tmem_relinquish();
    tc_fence_before();
  } else if (warp < 4) {
    if (warp == 2 && lane == 0) {
      for (int s = 0; s < g.nst; s++) mbar_init(&sf_full[s], 2);
      fence_barrier_init();
    }
    launch_wait();
    if (warp == 2 || !FUSED) gather(kb0);
  } else {
    launch_wait();
    if (warp - 4 < n) load_x(warp - 4);
  }
  launch_wait();
  __syncwarp();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_slot);

  if (warp == 0) {
    if (elect_one()) {
      int i = head, s = 0;
      uint32_t par = 0;
      for (; i < n; i++) {
        if (!mbar_wait_poll(&empty[s], par, lim, status, kWaitEmpty) || *abort_flag) {
          *abort_flag = 1;
          break;
        }
        load(i, s);
        if (++s == g.nst) {
          s = 0;
          par ^= 1;
        }
      }
      // Every copy has landed before the CTA goes on (the MMAs waited for
      // them too, unless a wait ran out).
      for (int j = max(0, i - g.nst); j < i; j++)
        mbar_wait_poll(&full[j % g.nst], (j / g.nst) & 1, drain_limit(lim), status, kWaitDrain);
    }
  } else if (warp == 1) {
    // One thread: with the whole warp in the loop, which needs a vote on every
    // wait, 48 x 4096 x 4096 took 8.6 us, not 8.2, a layer's 1 x 4096 x 4096 7.4, not 7.0.
    if (elect_one()) {
      const uint32_t w_step = (g.w.kmajor ? 32 : 32 * kRows) >> 4;
      const uint32_t sf_base = tmem + g.bn * g.nacc;
      int s = 0, left = 0;
      uint32_t ph = 0, d_tmem = tmem - g.bn, accumulate = 0;
      int part = -1;   // where they take turns: the part at work
      for (int kb = kb0; kb < kb1; kb++) {
        if (left == 0) {
          if (TURNS) {
            if (part >= 0) tc_commit(&part_full[part & 1]);
            part++;
            // the accumulator's last part but one has been read
            if (part >= 2 &&
                !mbar_wait_poll(&part_empty[part & 1], ((part >> 1) + 1) & 1, lim, status, kWaitAccEmpty)) {
              *abort_flag = 1;
              break;
            }
            tc_fence_after();
            d_tmem = tmem + (part & 1) * g.bn;
          } else {
            d_tmem += g.bn;
          }
          accumulate = 0;
          left = per;
        }
        left--;
        if (!mbar_wait_poll(&sf_full[s], ph, lim, status, kWaitScales) ||
            !mbar_wait_poll(&full[s], ph, lim, status, kWaitFull)) {
          *abort_flag = 1;
          break;
        }
        const uint32_t st = smem_u32(smem + s * stage_bytes), sf = smem_u32(sSF + s * 2 * kAtom);
        const uint32_t sfa = sf_base + s * 8, id = g.idesc | idesc_scale_byte(kb & 3);
        copy_scales(sfa, smem_desc_scales(sf));
        copy_scales(sfa + 4, smem_desc_scales(sf + kAtom));
        const uint64_t dw = smem_desc_sw128(st), dx = smem_desc_sw128(st + kWideBytes);
        mma_mx(d_tmem, dw, dx, id, sfa, sfa + 4, accumulate);
#pragma unroll
        for (int kk = 1; kk < kBlock / 32; kk++) mma_mx(d_tmem, dw + kk * w_step, dx + kk * 2, id, sfa, sfa + 4, 1);
        tc_commit(&empty[s]);
        accumulate = 1;
        if (++s == g.nst) {
          s = 0;
          ph ^= 1;
        }
      }
      tc_commit(acc_full);   // every MMA issued has completed when it arrives
      mbar_wait_poll(acc_full, 0, drain_limit(lim), status, kWaitDrain);
    }
  } else if (warp == 2 || (warp == 3 && !FUSED)) {
    // Scale words for four blocks of k at a time, written to every stage that
    // uses them; the next four's loads are issued once the first is handed over
    // (a wait for some loads is one for all).  (Stages are counted,
    // not divided for: this warp's steps are near the pace of the copies.)
    const Fp8Operand& o = warp == 2 ? g.w : g.x;
    uint32_t now[4], par = 1;
    int s = 0;
    for (int kb = kb0; kb < kb1; kb++) {
      const bool first = kb == kb0 || (kb & 3) == 0;
      if (first) {
#pragma unroll
        for (int j = 0; j < 4; j++) now[j] = raw[j];
        finish_scales<1>(o, now);
      }
      if (!warp_all(mbar_wait_poll(&empty[s], par, lim, status, kWaitScalesFree))) {
        *abort_flag = 1;
        break;
      }
      store_scales<1>(o, lane, now, sSF + (s * 2 + warp - 2) * kAtom);
      fence_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sf_full[s]);
      if (first && (kb | 3) + 1 < kb1) gather((kb | 3) + 1);
      if (++s == g.nst) {
        s = 0;
        par ^= 1;
      }
    }
  } else if (warp >= 4) {
    if constexpr (FUSED) {
      // One warp a block: a lone warp issues an instruction every few cycles,
      // so warps that each took a quarter of every block's rows, with all
      // the arithmetic of a scale for each, set the kernel's pace on few rows
      // (8192^2, one row: 1450 cycles a block of k, copies 800).
      int s = warp - 4;
      uint32_t par = 1;
      while (s >= g.nst) {
        s -= g.nst;
        par ^= 1;
      }
      for (int i = warp - 4; i < n; i += QW) {
        uint4 code[PASSES];
        uint8_t scale[PASSES];
#pragma unroll
        for (int p = 0; p < PASSES; p++) {
          if (p * 4 >= cols) break;
          float m = max16<XT>(v[p]);
#pragma unroll
          for (int o = 4; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
          if (__any_sync(0xFFFFFFFFu, is_inf(m))) {
            infs_to_nan<XT>(v[p]);
            m = max16<XT>(v[p]);
#pragma unroll
            for (int o = 4; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
          }
          const int e = scale_exponent<F64E_E4M3>(m);
          const float r = inverse_scale(e);
          uint32_t c[8];
          codes16<XT, F64E_E4M3>(v[p], [&](int) { return r; }, c);
          code[p] = row_of_codes(c);
          scale[p] = (uint8_t)(e + 127);
        }
        if (i + QW < n) load_x(i + QW);
        if (!warp_all(mbar_wait_poll(&empty[s], par, lim, status, kWaitScalesFree))) {
          *abort_flag = 1;
          break;
        }
        uint8_t* st = smem + s * stage_bytes + kWideBytes;
        uint8_t* sf = sSF + s * 2 * kAtom + kAtom + ((kb0 + i) & 3);
#pragma unroll
        for (int p = 0; p < PASSES; p++) {
          if (p * 4 >= cols) break;
          const int t = p * 4 + (lane >> 3);
          *reinterpret_cast<uint4*>(st + t * kBlock + ((l ^ (t & 7)) << 4)) = code[p];
          if (l == 0) sf[t * 16] = scale[p];
        }
        fence_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sf_full[s]);
        for (s += QW; s >= g.nst; par ^= 1) s -= g.nst;
      }
    }
    const int q = warp & 3;
    const uint32_t taddr = tmem + ((uint32_t)(q * 32) << 16);
    bool done = warp < 8;
    const int parts = n <= per ? 1 : (n + per - 1) / per;
    // What the end adds: all parts in their order, or the sum kept so far and the last part.
    const int terms = TURNS ? min(parts, 2) : parts;
    uint32_t term0 = taddr, term_step = g.bn;
    if (TURNS && parts > 1) {
      term0 += 2 * g.bn;
      term_step = ((parts - 1) & 1) * g.bn - 2 * g.bn;
    }
    if (TURNS) {
      // All parts but the last: the first to the sum's columns, others added.
      for (int a = 0; a + 1 < parts && done; a++) {
        const int i = a & 1;
        done = warp_all(mbar_wait_poll(&part_full[i], (a >> 1) & 1, lim, status, kWaitAccFull) && !*abort_flag);
        if (!done) {
          *abort_flag = 1;
          break;
        }
        tc_fence_after();
        for (int c = 0; c < cols; c += 16) {
          uint32_t v[16], w[16];
          tmem_ld_32x32b_x16(taddr + i * g.bn + c, v);
          if (a > 0) tmem_ld_32x32b_x16(taddr + 2 * g.bn + c, w);
          tmem_wait_ld();
          if (a > 0) {
#pragma unroll
            for (int k = 0; k < 16; k++) v[k] = __float_as_uint(__uint_as_float(w[k]) + __uint_as_float(v[k]));
          }
          tmem_st_32x32b_x16(taddr + 2 * g.bn + c, v);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&part_empty[i]);
      }
    }
    // Partial sums to shared memory, by columns of 128 rows; the stages are free:
    // every MMA has completed.
    done = done && warp_all(mbar_wait_poll(acc_full, 0, drain_limit(lim), status, kWaitAccFull) && !*abort_flag);
    if (done) {
      tc_fence_after();
      float* part = reinterpret_cast<float*>(smem) + q * 32 + lane;   // column pitch kPitch
      if (parts == 1 && g.bn % 32 == 0) {   // one accumulator, 32 columns at a time
        for (int c = 0; c < cols; c += 32) {
          uint32_t v[32];
          tmem_ld_32x32b_x32(taddr + c, v);
          tmem_wait_ld();
#pragma unroll
          for (int k = 0; k < 32; k++) part[(c + k) * kPitch] = __uint_as_float(v[k]);
        }
      } else {
        for (int c = 0; c < cols; c += 16) {
          float sum[16];
          for (int a = 0; a < terms; a++) {
            uint32_t v[16];
            tmem_ld_32x32b_x16(term0 + a * term_step + c, v);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 16; k++) sum[k] = a == 0 ? __uint_as_float(v[k]) : sum[k] + __uint_as_float(v[k]);
          }
#pragma unroll
          for (int k = 0; k < 16; k++) part[(c + k) * kPitch] = sum[k];
        }
      }
      tc_fence_before();
    }
  }

  __syncwarp();
  if (g.split > 1)
    cluster_sync();
  else
    __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, g.tmem_cols);
  }
  // This CTA's share of the tile: four rows of a column a thread, neighbouring
  // threads along the output's contiguous direction, four items in flight.
  const int items = cols * (kRows / 4);
  const int i0 = (int)((int64_t)items * rank / g.split), i1 = (int)((int64_t)items * (rank + 1) / g.split);
  if (!*abort_flag) {
    constexpr int NT = 32 * (4 + QW), U = 4;
    const uint32_t base = smem_u32(smem);
    for (int i = i0 + (int)threadIdx.x; i < i1; i += NT * U) {
      float4 v[U];
      int c[U], r[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int j = min(i + u * NT, i1 - 1);
        c[u] = g.out_c == 1 ? j % cols : j / (kRows / 4);
        r[u] = (g.out_c == 1 ? j / cols : j % (kRows / 4)) * 4;
        v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
      for (int p0 = 0; p0 < g.split; p0 += 4) {   // four CTAs' sums in flight, added in order
        float4 w[4][U];
#pragma unroll
        for (int p = 0; p < 4; p++) {
          if (p0 + p >= g.split) break;
          const uint32_t from = mapa_shared(base, p0 + p);
#pragma unroll
          for (int u = 0; u < U; u++) w[p][u] = ld_cluster_f4(from + (c[u] * kPitch + r[u]) * 4);
        }
#pragma unroll
        for (int p = 0; p < 4; p++) {
          if (p0 + p >= g.split) break;
#pragma unroll
          for (int u = 0; u < U; u++) {
            v[u].x += w[p][u].x;
            v[u].y += w[p][u].y;
            v[u].z += w[p][u].z;
            v[u].w += w[p][u].w;
          }
        }
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        if (i + u * NT >= i1) break;
        const int row = r0 + r[u];
        typename Elem<OUT>::type* o = reinterpret_cast<typename Elem<OUT>::type*>(g.out) + (int64_t)row * g.out_r +
                                      (int64_t)(c0 + c[u]) * g.out_c;
        const float f[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
        if (g.vec && row + 4 <= g.rows) {
          if (OUT == F64E_F32)
            *reinterpret_cast<float4*>(o) = v[u];
          else
            *reinterpret_cast<uint2*>(o) = make_uint2(Elem<OUT>::pack(f[0], f[1]), Elem<OUT>::pack(f[2], f[3]));
        } else {
#pragma unroll
          for (int k = 0; k < 4; k++)
            if (row + k < g.rows) {
              if (OUT == F64E_F32)
                reinterpret_cast<uint32_t*>(o)[k * g.out_r] = Elem<OUT>::bits(f[k]);
              else
                reinterpret_cast<uint16_t*>(o)[k * g.out_r] = (uint16_t)Elem<OUT>::bits(f[k]);
            }
        }
      }
    }
  }
  __syncwarp();   // the loop's trips differ by lane, and the barrier is one for whole warps
  if (g.split > 1) cluster_sync();   // the peers have read this CTA's sums
}

template <int OUT, int XT, bool TURNS>
cudaError_t launch_kernel(const CUtensorMap& tw, const CUtensorMap& tx, const SplitArgs& k, int tiles, size_t smem,
                          cudaStream_t s) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  {
    // the shared-memory opt-in is a per-device attribute of the kernel
    static std::mutex mtx;
    static std::map<int, bool> done;
    std::lock_guard<std::mutex> lk(mtx);
    if (!done[dev]) {
      e = cudaFuncSetAttribute(fp8_split_kernel<OUT, XT, TURNS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               227 * 1024);
      if (e != cudaSuccess) return e;
      done[dev] = true;
    }
  }
  return fp8_launch(fp8_split_kernel<OUT, XT, TURNS>, (unsigned)(tiles * k.split), 32 * (4 + kQuantWarps<XT>), smem,
                    k.split, s, tw, tx, k);
}

template <int OUT>
cudaError_t launch_codes(const CUtensorMap& tw, const CUtensorMap& tx, const SplitArgs& k, int tiles, size_t smem,
                         cudaStream_t s) {
  return k.turns ? launch_kernel<OUT, -1, true>(tw, tx, k, tiles, smem, s)
                 : launch_kernel<OUT, -1, false>(tw, tx, k, tiles, smem, s);
}

// held[n]: clusters of n CTAs that the current device holds at once (a
// cluster's CTAs share a GPC, so fewer than its SMs divided by n).  Asked once.
cudaError_t resident_clusters(int sms, const int** held) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  static std::mutex mtx;
  static std::map<int, std::array<int, kMaxSplit + 1>> known;
  std::lock_guard<std::mutex> lk(mtx);
  auto it = known.find(dev);
  if (it == known.end()) {
    std::array<int, kMaxSplit + 1> h{};
    const size_t smem = 200 * 1024;   // any amount above half an SM's gives the same answer
    e = cudaFuncSetAttribute(fp8_split_kernel<F64E_BF16, -1, false>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             227 * 1024);
    if (e != cudaSuccess) return e;
    for (int n = 1; n <= kMaxSplit; n++) {
      cudaLaunchConfig_t cfg = {};
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = n;
      attr[0].val.clusterDim.y = 1;
      attr[0].val.clusterDim.z = 1;
      cfg.gridDim = dim3((unsigned)(sms / n * n), 1, 1);
      cfg.blockDim = dim3(32 * (4 + kQuantWarps<-1>), 1, 1);
      cfg.dynamicSmemBytes = smem;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      int c = 0;
      e = cudaOccupancyMaxActiveClusters(&c, fp8_split_kernel<F64E_BF16, -1, false>, &cfg);
      if (e != cudaSuccess) return e;
      h[n] = std::max(c, 1);
    }
    it = known.emplace(dev, h).first;
  }
  *held = it->second.data();
  return cudaSuccess;
}

// How a product is cut: columns of a tile (a multiple of 16) and CTAs that
// share a tile's K.
struct Plan {
  int bn = 0, split = 0;
  int64_t cost = -1;   // cycles, estimated
};

// The cut of least time.  A CTA takes, a block of k, some 500 cycles (its MMA
// warp's loop) or all CTAs' copies of 16 KB and bn x 128 bytes at 5300 bytes a
// cycle (the L2's rate); 7500 to start and to end, 12 a column to put its sums
// down and 32 to fetch the others' (16 bytes a cycle between SMs).  Tiles have
// up to 128 columns: with 256, stages of 48 KB leave too few in flight (1024 x
// 2048 x 2048 14.6 us against 11.7).  Measured, both sides of a choice: 1024^3
// 7.7 us with 64 columns, 8.7 with 128; 8 x 2048 x 8192 9.1 us with 7 CTAs a
// tile, 14.3 with 8, of whose clusters the device holds one too few at once.
// most: blocks of k that a CTA may take at most (0: any number).
cudaError_t plan_tiles(int64_t rows, int64_t cols, int64_t nkb, int sms, int64_t most, Plan* best) {
  const int* held_of = nullptr;
  const cudaError_t e = resident_clusters(sms, &held_of);
  if (e != cudaSuccess) return e;
  const int64_t t0 = (cols + kMaxCols - 1) / kMaxCols;
  for (int64_t t = t0; t <= 2 * t0; t += t0) {
    const int64_t bn = ((cols + t - 1) / t + 15) / 16 * 16;
    if (t > t0 && bn < 48) break;
    const int64_t tiles = (rows + kRows - 1) / kRows * ((cols + bn - 1) / bn);
    for (int s = 1; s <= kMaxSplit && s <= nkb; s++) {
      if (most > 0 && (nkb + s - 1) / s > most) continue;
      const int64_t held = held_of[s];
      const int64_t ctas = std::min(tiles, held) * s;
      const int64_t block = std::max<int64_t>(500, ctas * (kWideBytes + bn * kBlock) / 5300);
      const int64_t cost =
          (tiles + held - 1) / held * ((nkb + s - 1) / s * block + 7500 + 12 * bn + 32 * bn * (s - 1) / s);
      if (best->cost < 0 || cost < best->cost) *best = {(int)bn, s, cost};
    }
  }
  return cudaSuccess;
}

// Blocks of k that one accumulator may hold.  The tensor core truncates what an
// addition shifts out, always towards zero: measured on random 2048 x 2048 x K,
// sums in one accumulator come out too small by 7e-8 of themselves at K = 2048
// (a 32-bit product of torch is off by 6e-8), 6e-6 at 65536, 4e-5 at 262144 and
// 2e-4 at 2^20, as much as rounding to float16 (2.1e-4).  Parts of 2048 values
// for 32-bit outputs, and of 131072 for 16-bit ones: too small by 1.6e-5.
constexpr int part_blocks(int out_type) { return out_type == F64E_F32 ? 16 : 1024; }

int stages_of(int bn, int per_cta) {
  return (int)std::min<int64_t>({kMaxStages, per_cta, (int64_t)(kRing / (kWideBytes + bn * kBlock + 2 * kAtom))});
}
// Accumulators of bn columns that TMEM holds beside the stages' scales.
int held_parts(int bn, int stages) { return (512 - stages * 8) / bn; }
static_assert((512 - 8 * (int)(kRing / (kWideBytes + kMaxCols * kBlock + 2 * kAtom))) / kMaxCols >= kTurnParts &&
                  (512 - 8 * kMaxStages) / 16 * 16 * kMaxSplit * kBlock >= kFusedMaxK,
              "three accumulators fit beside any stages, and all parts of a fused product beside one another");

// k.rows x k.cols of k.w and k.x.
cudaError_t launch(SplitArgs k, int out_type, int x_type, int64_t K, const Plan& plan, cudaStream_t s) {
  CUtensorMap tw, tx = {};
  if (!fp8_encode_codes(&tw, k.w, k.rows, K, kRows) ||
      (x_type < 0 && !fp8_encode_codes(&tx, k.x, k.cols, K, plan.bn)))
    return cudaErrorInvalidValue;
  k.nkb = (int)((K + kBlock - 1) / kBlock);
  k.K = K;
  k.bn = plan.bn;
  k.split = plan.split;
  k.tiles_r = (k.rows + kRows - 1) / kRows;
  const int tiles = k.tiles_r * ((k.cols + k.bn - 1) / k.bn);
  const int per_cta = (k.nkb + k.split - 1) / k.split;
  const size_t stage = kWideBytes + (size_t)k.bn * kBlock;
  k.nst = stages_of(k.bn, per_cta);
  const int sf_cols = k.nst * 8;
  k.nacc = (per_cta + part_blocks(out_type) - 1) / part_blocks(out_type);
  if (k.nacc > held_parts(k.bn, k.nst)) {
    if (x_type >= 0) return cudaErrorInvalidValue;   // excluded by the plan
    k.nacc = kTurnParts;
    k.turns = part_blocks(out_type);
  }
  k.tmem_cols = 32;
  while ((int)k.tmem_cols < k.bn * k.nacc + sf_cols) k.tmem_cols *= 2;
  k.idesc = idesc_mx(kRows, k.bn, k.w.code, k.x.code, !k.w.kmajor, 0);
  k.w.s_mode = fp8_scale_mode(k.w, k.rows, true);
  if (x_type < 0) k.x.s_mode = fp8_scale_mode(k.x, k.cols, k.bn >= k.cols || k.bn % 128 == 0);
  const int es = out_type == F64E_F32 ? 4 : 2;
  k.vec = k.out_r == 1 && reinterpret_cast<uintptr_t>(k.out) % (4 * es) == 0 && k.out_c % 4 == 0;
  k.ring = (uint32_t)std::max((size_t)k.nst * stage, (size_t)k.bn * kPitch * 4);
  const size_t smem =
      std::max(kMinSmem, 1024 + (size_t)k.ring + (size_t)k.nst * 2 * kAtom + (3 * kMaxStages + 5) * 8 + 16);
  if (x_type >= 0) {
    switch (x_type) {
      case F64E_F32: return launch_kernel<F64E_F32, F64E_F32, false>(tw, tx, k, tiles, smem, s);
      case F64E_F16: return launch_kernel<F64E_F16, F64E_F16, false>(tw, tx, k, tiles, smem, s);
      default: return launch_kernel<F64E_BF16, F64E_BF16, false>(tw, tx, k, tiles, smem, s);
    }
  }
  switch (out_type) {
    case F64E_F32: return launch_codes<F64E_F32>(tw, tx, k, tiles, smem, s);
    case F64E_F16: return launch_codes<F64E_F16>(tw, tx, k, tiles, smem, s);
    default: return launch_codes<F64E_BF16>(tw, tx, k, tiles, smem, s);
  }
}

}  // namespace

cudaError_t launch_fp8_split(const Fp8GemmArgs& g, int64_t other_cost, bool* done, cudaStream_t s) {
  *done = false;
  if (!(g.M <= g.N ? g.a : g.b).kmajor) return cudaSuccess;
  Plan plan;
  const cudaError_t e =
      plan_tiles(std::max(g.M, g.N), std::min(g.M, g.N), (g.K + kBlock - 1) / kBlock, g.sms, 0, &plan);
  if (e != cudaSuccess || plan.cost > other_cost) return e;
  *done = true;
  SplitArgs k = {};
  const bool a_thin = g.M <= g.N;
  k.w = a_thin ? g.b : g.a;
  k.x = a_thin ? g.a : g.b;
  k.rows = (int)(a_thin ? g.N : g.M);
  k.cols = (int)(a_thin ? g.M : g.N);
  k.out = static_cast<char*>(g.out);
  k.out_r = a_thin ? 1 : g.ldo;
  k.out_c = a_thin ? g.ldo : 1;
  k.wait_limit_ns = g.wait_limit_ns;
  return launch(k, g.out_type, -1, g.K, plan, s);
}

cudaError_t launch_fp8_linear_few(const Fp8LinearArgs& a, cudaStream_t s) {
  const Fp8GemmArgs& g = a.g;
  SplitArgs k = {};
  k.w = g.b;
  k.x.code = F64E_E4M3;
  k.x.kmajor = 1;
  k.rows = (int)g.N;
  k.cols = (int)g.M;
  k.out = static_cast<char*>(g.out);
  k.out_r = 1;
  k.out_c = g.ldo;
  k.xf = a.x;
  k.ldx = a.ldx;
  const int64_t pitch = a.ldx * (a.x_type == F64E_F32 ? 4 : 2);
  const uintptr_t x = reinterpret_cast<uintptr_t>(a.x);
  k.x_vec = x % 16 == 0 && (pitch % 16 == 0 || g.M == 1);
  k.x_wide = x % 32 == 0 && (pitch % 32 == 0 || g.M == 1);
  k.wait_limit_ns = g.wait_limit_ns;
  Plan plan;
  // Its warps 4 to 7 quantise x until the end, so its parts are all kept.
  const int64_t most = (int64_t)held_parts(16, kMaxStages) * part_blocks(a.x_type);
  const cudaError_t e = plan_tiles(g.N, g.M, (g.K + kBlock - 1) / kBlock, g.sms, most, &plan);
  return e == cudaSuccess ? launch(k, a.x_type, a.x_type, g.K, plan, s) : e;
}

// Nothing arrives at the barrier and nothing else is in flight: the kernel returns.
__global__ void fp8_split_wait_selftest_kernel(uint64_t limit_ns) {
  __shared__ __align__(8) uint64_t bar;
  if (elect_one()) {
    mbar_init(&bar, 1);
    fence_barrier_init();
    mbar_wait_poll(&bar, 0, limit_ns, &g_fp8_split_status, kWaitSelfTestSplit);
  }
}
cudaError_t launch_fp8_split_wait_selftest(uint64_t limit_ns, cudaStream_t s) {
  fp8_split_wait_selftest_kernel<<<1, 32, 0, s>>>(limit_ns);
  return cudaGetLastError();
}

cudaError_t read_fp8_split_status(int* status, cudaStream_t s) {
  static const int zero = 0;
  cudaError_t e = cudaMemcpyFromSymbolAsync(status, g_fp8_split_status, sizeof(int), 0, cudaMemcpyDeviceToHost, s);
  if (e == cudaSuccess)
    e = cudaMemcpyToSymbolAsync(g_fp8_split_status, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, s);
  return e == cudaSuccess ? cudaStreamSynchronize(s) : e;
}

}  // namespace f64e
