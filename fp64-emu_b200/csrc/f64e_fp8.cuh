// Device-side building blocks of the 8-bit floating-point operators: element
// types, codes, power-of-two block scales.
//
// A block's scale is 2^e with e the smallest integer for which every finite
// value fits, amax <= FMAX * 2^e, and at least -127; its code is the
// round-to-nearest-even 8-bit float of x * 2^-e.  A power of two costs nothing
// against a free scale in relative precision (a float's rounding error does
// not depend on its exponent), keeps x * 2^-e and code * 2^e exact, makes the
// codes independent of how the scale is computed, and is the form the tensor
// cores multiply by themselves (ue8m0).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "f64e.h"
#include "f64e_device.cuh"
#include "f64e_fp8.h"

namespace f64e {

// --------------------------------------------------- overlapping launches --
// These kernels are launched with programmatic stream serialization: a kernel
// may be set up while the one before it in the stream drains.  It reads and
// writes global memory only after launch_wait(), when that kernel has
// completed; launch_next() lets the next one be set up.  Loads of what an
// earlier kernel wrote are plain ld.global: the non-coherent path (__ldg) may
// hold lines from before that kernel's end, since no kernel begins in between.
__device__ __forceinline__ void launch_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void launch_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// ------------------------------------------------------------ scale bytes --
// FMAX = 1.75 * 2^emax in both codes: e = p - emax for a largest magnitude
// m * 2^p with m in [1, 1.75], one more above.  Subnormal magnitudes give
// exponents below -127 whatever their leading bit, so the field serves as p.
template <int CODE>
__device__ __forceinline__ int scale_exponent(float amax) {
  const uint32_t amax_bits = __float_as_uint(amax);
  constexpr int emax = CODE == F64E_E4M3 ? 8 : 15;
  if (amax_bits == 0) return 0;
  const int p = (int)(amax_bits >> 23) - 127;
  const int e = p - emax + ((amax_bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return e < -127 ? -127 : e;
}
// 2^-e for e in [-127, 120]: a normal number.
__device__ __forceinline__ float inverse_scale(int e) { return __uint_as_float((uint32_t)(127 - e) << 23); }
// 2^(b - 127), b = 0 a subnormal; b = 255 stands for NaN.
__device__ __forceinline__ float scale_of_byte(uint32_t b) {
  return b == 255u ? __uint_as_float(0x7FFFFFFFu) : (b ? __uint_as_float(b << 23) : __uint_as_float(0x00400000u));
}

// ------------------------------------------------------------------ codes --
// Two codes from two scaled values, `lo` in the low byte.  Finite values are
// within FMAX by the choice of the scale; a NaN becomes a NaN code (and an
// infinity would become the largest finite one, see infs_to_nan).
template <int CODE>
__device__ __forceinline__ uint32_t code2(float lo, float hi) {
  uint16_t r;
  if (CODE == F64E_E4M3)
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
template <int CODE>
__device__ __forceinline__ float2 values2(uint32_t codes) {
  uint32_t h;
  if (CODE == F64E_E4M3)
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)codes));
  else
    asm("cvt.rn.f16x2.e5m2x2 %0, %1;" : "=r"(h) : "h"((uint16_t)codes));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// --------------------------------------------------------------- elements --
// Sixteen elements of a thread as 32-bit words (two 16-bit elements a word),
// their largest magnitude, and their values.  NaN never counts as a largest
// magnitude.
template <int T>
struct Elem;
template <>
struct Elem<F64E_F32> {
  using type = float;
  static constexpr int kWords = 16;
  using mag = float;   // magnitudes of one word
  __device__ static mag zero() { return 0.f; }
  __device__ static mag max_mag(mag m, uint32_t w) { return fmaxf(m, fabsf(__uint_as_float(w))); }
  __device__ static mag max_of(mag a, mag b) { return fmaxf(a, b); }
  __device__ static mag shfl(mag a, int o) { return __shfl_xor_sync(0xFFFFFFFFu, a, o); }
  __device__ static float get(const uint32_t* w, int i) { return __uint_as_float(w[i]); }
  __device__ static uint32_t bits(float v) { return __float_as_uint(v); }
  __device__ static uint32_t pack(float, float) { return 0; }   // two elements never share a word
};
template <typename H2>
struct Elem16 {
  static constexpr int kWords = 8;
  using mag = H2;
  __device__ static mag max_mag(mag m, uint32_t w) {
    w &= 0x7FFF7FFFu;
    return __hmax2(m, *reinterpret_cast<const H2*>(&w));
  }
  __device__ static mag max_of(mag a, mag b) { return __hmax2(a, b); }
  __device__ static mag shfl(mag a, int o) {
    const uint32_t w = __shfl_xor_sync(0xFFFFFFFFu, *reinterpret_cast<const uint32_t*>(&a), o);
    return *reinterpret_cast<const H2*>(&w);
  }
  __device__ static mag zero() {
    const uint32_t w = 0;
    return *reinterpret_cast<const H2*>(&w);
  }
};
template <>
struct Elem<F64E_F16> : Elem16<__half2> {
  using type = __half;
  __device__ static float get(const uint32_t* w, int i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i >> 1]));
    return (i & 1) ? f.y : f.x;
  }
  __device__ static float lo(__half2 m) { return __low2float(m); }
  __device__ static float hi(__half2 m) { return __high2float(m); }
  __device__ static uint32_t bits(float v) { return (uint32_t)__half_as_ushort(__float2half_rn(v)); }
  __device__ static uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <>
struct Elem<F64E_BF16> : Elem16<__nv_bfloat162> {
  using type = __nv_bfloat16;
  __device__ static float get(const uint32_t* w, int i) {
    return __uint_as_float((i & 1) ? (w[i >> 1] & 0xFFFF0000u) : (w[i >> 1] << 16));
  }
  __device__ static float lo(__nv_bfloat162 m) { return __low2float(m); }
  __device__ static float hi(__nv_bfloat162 m) { return __high2float(m); }
  __device__ static uint32_t bits(float v) { return (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(v)); }
  __device__ static uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

// Sixteen contiguous elements at p, all there: 32-byte loads where `wide`
// (p 32-byte aligned), else 16-byte loads.
template <int T>
__device__ __forceinline__ void load16(const typename Elem<T>::type* p, bool wide, uint32_t* w) {
  if (wide) {
#pragma unroll
    for (int i = 0; i < Elem<T>::kWords; i += 8)
      asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
          : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3]), "=r"(w[i + 4]), "=r"(w[i + 5]), "=r"(w[i + 6]),
            "=r"(w[i + 7])
          : "l"(reinterpret_cast<const uint32_t*>(p) + i)
          : "memory");
  } else {
#pragma unroll
    for (int i = 0; i < Elem<T>::kWords; i += 4) {
      const uint4 v = reinterpret_cast<const uint4*>(p)[i / 4];
      w[i] = v.x;
      w[i + 1] = v.y;
      w[i + 2] = v.z;
      w[i + 3] = v.w;
    }
  }
}
// Elements p[0], p[step], .. p[15 step], of which those with index below n
// exist; the others read as zero.
template <int T>
__device__ __forceinline__ void load16_some(const typename Elem<T>::type* p, int step, int64_t n, uint32_t* w) {
  if (Elem<T>::kWords == 16) {
#pragma unroll
    for (int i = 0; i < 16; i++) w[i % Elem<T>::kWords] = i * step < n ? reinterpret_cast<const uint32_t*>(p)[i * step] : 0;
  } else {
    const uint16_t* u = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      const uint32_t lo = i * step < n ? u[i * step] : 0;
      const uint32_t hi = (i + 1) * step < n ? u[(i + 1) * step] : 0;
      w[i / 2] = lo | (hi << 16);
    }
  }
}

// Largest magnitude of sixteen elements, as a float.
__device__ __forceinline__ float fold(float m) { return m; }
__device__ __forceinline__ float fold(__half2 m) { return fmaxf(__low2float(m), __high2float(m)); }
__device__ __forceinline__ float fold(__nv_bfloat162 m) { return fmaxf(__low2float(m), __high2float(m)); }
template <int T>
__device__ __forceinline__ float max16(const uint32_t* w) {
  typename Elem<T>::mag m = Elem<T>::zero();
#pragma unroll
  for (int i = 0; i < Elem<T>::kWords; i++) m = Elem<T>::max_mag(m, w[i]);
  return fold(m);
}
__device__ __forceinline__ bool is_inf(float m) { return __float_as_uint(m) == 0x7F800000u; }
// Infinities among sixteen elements become NaN: no scale could hold them, and
// as NaN they neither count as magnitudes nor saturate.  Where a block's
// largest magnitude is infinite it is taken again after this.
template <int T>
__device__ __forceinline__ void infs_to_nan(uint32_t* w) {
#pragma unroll
  for (int i = 0; i < Elem<T>::kWords; i++) {
    if (T == F64E_F32) {
      if ((w[i] & 0x7FFFFFFFu) == 0x7F800000u) w[i] = 0x7FFFFFFFu;
    } else {
      constexpr uint32_t inf = T == F64E_F16 ? 0x7C00u : 0x7F80u;
      if ((w[i] & 0x7FFFu) == inf) w[i] |= 0x7FFFu;
      if (((w[i] >> 16) & 0x7FFFu) == inf) w[i] |= 0x7FFF0000u;
    }
  }
}

// Codes of sixteen elements, two a word: element i scaled by r(i).
template <int T, int CODE, typename R>
__device__ __forceinline__ void codes16(const uint32_t* w, R r, uint32_t* c) {
#pragma unroll
  for (int i = 0; i < 8; i++)
    c[i] = code2<CODE>(Elem<T>::get(w, 2 * i) * r(2 * i), Elem<T>::get(w, 2 * i + 1) * r(2 * i + 1));
}
// The words of sixteen neighbouring codes.
__device__ __forceinline__ uint4 row_of_codes(const uint32_t* c) {
  return make_uint4(c[0] | (c[1] << 16), c[2] | (c[3] << 16), c[4] | (c[5] << 16), c[6] | (c[7] << 16));
}

// ------------------------------------------------ block-scaled tcgen05 --
// Everything below serves products of 8-bit codes whose 128-value blocks carry
// power-of-two scales: the tensor cores take a scale per 32 values of k, read
// from TMEM, so the four K = 32 instructions of a 128-value block read the
// same one and the sums stay in one FP32 accumulator over all of K.

// Bounded wait like mbar_wait, polling without sleeps (nothing else runs
// beside these kernels' CTAs).  CLUSTER: acquires at cluster scope, for a
// barrier that orders the other CTA's shared-memory writes; the acquire costs
// some 270 cycles, so the waits on copies and MMAs, every block of k, go without.
template <bool CLUSTER>
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  if (!CLUSTER) return mbar_try_wait(bar, parity);
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, "
      "0, p;\n}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
template <bool CLUSTER = false>
__device__ __forceinline__ bool mbar_wait_poll(uint64_t* bar, uint32_t parity, uint64_t limit_ns, int* status,
                                               int site) {
  if (mbar_test<CLUSTER>(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  while (true) {
#pragma unroll 1
    for (int i = 0; i < 64; i++)
      if (mbar_test<CLUSTER>(bar, parity)) return true;
    if (globaltimer_ns() - t0 > limit_ns) {
      record_status(status, site);
      return false;
    }
  }
}
// What a wait gave, for the whole warp: true where all of its lanes have what
// they waited for.  A lane that gives up, or reads the abort flag a moment
// later than its neighbours, must not part from them: tcgen05 loads, barriers
// and __syncwarp behind the wait need all 32.  Nor may the lane that issues run
// ahead of one that still waits, which could miss the phase it waits for.  So
// every wait that is not one elected thread's goes through this vote.
__device__ __forceinline__ bool warp_all(bool ok) { return __all_sync(0xFFFFFFFFu, ok) != 0; }

// 128 x 128-byte box of a 2-D map at (x, y): x along the contiguous direction.
__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
      "[%4];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}
// The same, counted on an mbarrier of either CTA of the pair (no multicast).
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* map, int x, int y,
                                                 uint32_t bar_cluster_addr) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
      "%3}], [%4];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar_cluster_addr)
      : "memory");
}

// Box of shared memory to a 2-D map at (x, y), clipped at its extents; done
// (shared memory read) when the thread's bulk groups say so.
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, int x, int y, const void* src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y), "r"(smem_u32(src))
               : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
template <int LEFT>
__device__ __forceinline__ void tma_store_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(LEFT) : "memory");
}
__device__ __forceinline__ void tma_store_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// Arrival on an mbarrier of either CTA that orders no memory (what it signals
// is a tcgen05.ld that has completed): a release at cluster scope would wait
// 550 cycles for the warp's stores.
__device__ __forceinline__ void mbar_arrive_cluster_relaxed(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// The two halves of a cluster barrier; a warp's lanes may reach them apart.
// The relaxed arrival orders nothing but barriers set up before fence_barrier_init().
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory"); }
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// Generic-proxy writes to shared memory made visible to the tensor cores.
__device__ __forceinline__ void fence_async_shared() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// 16 columns of this warp's 32 lanes (see tmem_ld_32x32b_x32).
__device__ __forceinline__ void tmem_ld_32x32b_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
        "=r"(r[15])
      : "r"(taddr));
}

__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Instruction descriptor of kind::mxf8f6f4 with ue8m0 scales (bit 23): types
// at bits 7-9 / 10-12 (0 e4m3, 1 e5m2), transposes (operand stored with M or N
// contiguous) at bits 15 / 16, N >> 3 at bits 17-22, M >> 7 at bits 27-28.
// The byte of the scale word each operand uses is added per instruction: B's
// at bits 4-5, A's at bits 29-30.
__host__ __device__ constexpr uint32_t idesc_mx(int M, int N, int a_code, int b_code, int a_mn, int b_mn) {
  return ((uint32_t)a_code << 7) | ((uint32_t)b_code << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) |
         ((uint32_t)(N >> 3) << 17) | (1u << 23) | ((uint32_t)(M >> 7) << 27);
}
__device__ __forceinline__ uint32_t idesc_scale_byte(uint32_t i) { return (i << 4) | (i << 29); }

// Shared-memory descriptor of a scale atom: 32 rows of 16 bytes, 8-row core
// matrices 128 bytes apart, no swizzle.  Row r holds the words of tile rows
// r, r + 32, r + 64, r + 96, a word the scales of four neighbouring blocks.
__device__ __forceinline__ uint64_t smem_desc_scales(uint32_t saddr) {
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (uint64_t)(128 >> 4) << 16 | (uint64_t)(128 >> 4) << 32 |
         (uint64_t)1 << 46;
}

// A scale atom to four TMEM columns, in every 32-lane quarter.
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
// D[tmem] (+)= (A * scale)[smem] * (B * scale)[smem]^T, K = 32.
__device__ __forceinline__ void mma_mx(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                       uint32_t sfa_tmem, uint32_t sfb_tmem, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
      " tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n}" ::"r"(
          d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa_tmem), "r"(sfb_tmem), "r"(accumulate)
      : "memory");
}

// A scale atom to four TMEM columns, in every 32-lane quarter of both CTAs, each from its own shared memory.
__device__ __forceinline__ void copy_scales_pair(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
// D[tmem] (+)= (A * scale)[smem] * (B * scale)[smem]^T, K = 32.
__device__ __forceinline__ void mma_mx_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                       uint32_t sfa_tmem, uint32_t sfb_tmem, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
      " tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n}" ::"r"(
          d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa_tmem), "r"(sfb_tmem), "r"(accumulate)
      : "memory");
}

enum : int { kWaitScales = 6, kWaitScalesFree = 7, kWaitSelfTestSplit = 10 };   // status sites, beside kWait*

// --------------------------------------------------------------- scales --
// Gathering the scales of `N` atoms (128 rows each, from r0) for blocks 4 j ..
// 4 j + 3 of k, a warp, in two steps: loads into raw[4 N] registers, none of
// which depends on a branch or on another, and, when the atoms' place is free,
// the atoms themselves.  Taken one word after the other the scales, not the
// MMAs, set the pace of a product with column scales on both sides.  Rows and blocks outside the operand read
// a neighbour's scale: their codes are zeros, and no store uses them.
//   kScaleWords  four blocks' scales are one aligned word
//   kScaleRows   four rows' scales are one aligned word (column blocks)
//   kScaleTile   one scale for all rows of an atom
//   kScaleBytes  any strides
template <int N>
__device__ __forceinline__ void load_scales(const Fp8Operand& o, int rows, int nkb, int r0, int j, int lane,
                                            uint32_t* raw) {
  if (o.s_mode == kScaleRows) {
#pragma unroll
    for (int n = 0; n < N; n++) {
      const uint8_t* p = o.s + min(r0 + n * 128 + lane * 4, rows - 4);
#pragma unroll
      for (int i = 0; i < 4; i++)
        raw[4 * n + i] = *reinterpret_cast<const uint32_t*>(p + (int64_t)min(4 * j + i, nkb - 1) * o.s_kb);
    }
  } else if (o.s_mode == kScaleTile) {
#pragma unroll
    for (int n = 0; n < N; n++) {
      const uint8_t* p = o.s + (int64_t)(min(r0 + n * 128, rows - 1) >> 7) * o.s_row;
#pragma unroll
      for (int i = 0; i < 4; i++) raw[4 * n + i] = p[(int64_t)min(4 * j + i, nkb - 1) * o.s_kb];
    }
  } else {
    const uint8_t* p[4 * N];
#pragma unroll
    for (int w = 0; w < 4 * N; w++)
      p[w] = o.s + (int64_t)(min(r0 + w * 32 + lane, rows - 1) >> o.s_shift) * o.s_row;
    if (o.s_mode == kScaleWords && 4 * j + 4 <= nkb) {
#pragma unroll
      for (int w = 0; w < 4 * N; w++) raw[w] = *reinterpret_cast<const uint32_t*>(p[w] + 4 * j);
    } else {
      uint32_t b[4 * N][4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int64_t at = (int64_t)min(4 * j + i, nkb - 1) * o.s_kb;
#pragma unroll
        for (int w = 0; w < 4 * N; w++) b[w][i] = p[w][at];
      }
#pragma unroll
      for (int w = 0; w < 4 * N; w++) raw[w] = b[w][0] | (b[w][1] << 8) | (b[w][2] << 16) | (b[w][3] << 24);
    }
  }
}
// What was loaded as the atoms' words: row n * 128 + lane + 32 w in raw[4 n + w],
// or, in kScaleRows, row n * 128 + 4 lane + w.
template <int N>
__device__ __forceinline__ void finish_scales(const Fp8Operand& o, uint32_t (&raw)[4 * N]) {
  if (o.s_mode != kScaleRows && o.s_mode != kScaleTile) return;
#pragma unroll
  for (int n = 0; n < N; n++) {
    uint32_t* v = raw + 4 * n;
    const uint32_t a = __byte_perm(v[0], v[1], 0x5140), b = __byte_perm(v[2], v[3], 0x5140);
    const uint32_t c = __byte_perm(v[0], v[1], 0x7362), d = __byte_perm(v[2], v[3], 0x7362);
    v[0] = __byte_perm(a, b, 0x5410);
    if (o.s_mode == kScaleTile) {
      v[1] = v[2] = v[3] = v[0];
    } else {
      v[1] = __byte_perm(a, b, 0x7632);
      v[2] = __byte_perm(c, d, 0x5410);
      v[3] = __byte_perm(c, d, 0x7632);
    }
  }
}
template <int N>
__device__ __forceinline__ void store_scales(const Fp8Operand& o, int lane, const uint32_t* words, uint8_t* atoms) {
#pragma unroll
  for (int n = 0; n < N; n++) {
    const uint32_t* v = words + 4 * n;
    if (o.s_mode == kScaleRows) {
      uint32_t* w = reinterpret_cast<uint32_t*>(atoms + n * 512 + (lane & 7) * 64 + (lane >> 3) * 4);
      w[0] = v[0];
      w[4] = v[1];
      w[8] = v[2];
      w[12] = v[3];
    } else {
      *reinterpret_cast<uint4*>(atoms + n * 512 + lane * 16) = make_uint4(v[0], v[1], v[2], v[3]);
    }
  }
}

}  // namespace f64e
