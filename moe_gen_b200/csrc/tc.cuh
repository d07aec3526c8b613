// Device helpers shared by the tensor-core kernels: mbarriers with bounded waits, TMA loads, tcgen05 wrappers,
// shared-memory descriptors, FP8 conversion.  sm_100a only.
#pragma once
#include <cuda_fp8.h>

#include "common.cuh"

namespace mg {

constexpr unsigned long long WAIT_LIMIT_NS = 2000000000ull;

// ---- PTX wrappers ---------------------------------------------------------------------
__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ uint32_t mbar_try_wait(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok;
}
// nanoseconds; the two halves are read separately and the high half checked, so that a carry of the low
// half between the reads cannot produce a value that is off by 2^32 ns
__device__ __forceinline__ unsigned long long global_timer() {
  uint32_t hi, lo, hi2;
  do {
    asm volatile("mov.u32 %0, %%globaltimer_hi;" : "=r"(hi));
    asm volatile("mov.u32 %0, %%globaltimer_lo;" : "=r"(lo));
    asm volatile("mov.u32 %0, %%globaltimer_hi;" : "=r"(hi2));
  } while (hi != hi2);
  return (static_cast<unsigned long long>(hi) << 32) | lo;
}
// The limit of a bounded wait has run out.  The 64-bit timer is read as two halves; a read that straddles
// a carry of the low half can come out far too small or too large, so the difference is taken as a
// signed number (a reading below t0 never counts) and an expiry must be seen by two readings in a row.
__device__ __forceinline__ bool timed_out(unsigned long long t0, unsigned long long limit_ns) {
  const long long d1 = static_cast<long long>(global_timer() - t0);
  if (d1 <= static_cast<long long>(limit_ns)) return false;
  const long long d2 = static_cast<long long>(global_timer() - t0);
  return d2 > static_cast<long long>(limit_ns) && d2 >= d1;
}
// Bounded wait.  Returns false if the wait ran out or another role already gave up.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag,
                                          int32_t* status, int where,
                                          unsigned long long limit_ns = WAIT_LIMIT_NS) {
  if (mbar_try_wait(bar, parity)) return true;
  const unsigned long long t0 = global_timer();
  uint32_t spins = 0;
  while (true) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((++spins & 63u) == 0u) {
      if (*abort_flag) return false;
      if (timed_out(t0, limit_ns)) {
        *abort_flag = 1;
        if (atomicCAS(status, MG_DEV_OK, MG_DEV_WAIT_TIMEOUT) == MG_DEV_OK) status[1] = where;
        return false;
      }
    }
  }
}
// The same for the roles that a whole warp plays, which leave their loops by this vote only: another role may raise the
// flag, and the limit run out, between the readings of two lanes, and a lane that left on its own would wait at the
// kernel's closing barrier for lanes that wait for it in a warp-wide instruction, without a limit.
__device__ __forceinline__ bool mbar_wait_warp(uint32_t bar, uint32_t parity, volatile int* abort_flag, int32_t* status,
                                               int where, unsigned long long limit_ns = WAIT_LIMIT_NS) {
  return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity, abort_flag, status, where, limit_ns)) != 0;
}
// The same with the common case, a barrier that all lanes find complete, kept to one vote.
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, volatile int* abort_flag, int32_t* status, int where) {
  return __all_sync(0xFFFFFFFFu, mbar_try_wait(bar, parity)) || mbar_wait_warp(bar, parity, abort_flag, status, where);
}
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int c0, int c1,
                                            uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
// the box of a load, into L2 only
__device__ __forceinline__ void tma_prefetch_3d(const CUtensorMap* map, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global.tile [%0, {%1, %2, %3}];" ::"l"(map), "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}
__device__ __forceinline__ void tma_prefetch_4d(const CUtensorMap* map, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.prefetch.tensor.4d.L2.global.tile [%0, {%1, %2, %3, %4}];" ::"l"(map), "r"(c0), "r"(c1), "r"(c2),
               "r"(c3)
               : "memory");
}
__device__ __forceinline__ void st_cluster(uint32_t cluster_addr, int v) {
  asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(cluster_addr), "r"(v) : "memory");
}
// mbar_wait for what a thread of the other CTA has written (mbar_arrive_cluster)
__device__ __forceinline__ bool mbar_wait_cluster(uint32_t bar, uint32_t parity, volatile int* abort_flag, int32_t* status,
                                                  int where, unsigned long long limit_ns = WAIT_LIMIT_NS) {
  if (!mbar_wait(bar, parity, abort_flag, status, where, limit_ns)) return false;
  asm volatile("fence.acq_rel.cluster;" ::: "memory");
  return true;
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, int c0, int c1, uint32_t src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(c0),
               "r"(c1), "r"(src)
               : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}

// L2 residency hints for data that is written once and read many times before it is overwritten
__device__ __forceinline__ uint64_t policy_evict_last() {
  uint64_t pol;
  asm volatile("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(pol));
  return pol;
}
__device__ __forceinline__ void tma_load_2d_hint(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar,
                                                 uint64_t pol) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4}], [%2], %5;"
      ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1), "l"(pol)
      : "memory");
}
__device__ __forceinline__ void st_global_hint16(void* ptr, const uint4& v, uint64_t pol) {
  asm volatile("st.global.L2::cache_hint.v4.b32 [%0], {%1, %2, %3, %4}, %5;" ::"l"(ptr), "r"(v.x), "r"(v.y), "r"(v.z),
               "r"(v.w), "l"(pol)
               : "memory");
}
// One thread of a converged warp.  Single-thread roles choose their thread with this and not by a lane number: the
// compiler knows of an elected region that it is one thread, keeps the operands of TMA and tcgen05 instructions in
// uniform registers and issues them back to back; under `lane == 0` it moves each operand over per instruction.
// Measured, four M256 N32 K16 MMAs with A in tensor memory and two commits: 67 against 273 cycles.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred P;\n\telect.sync _|P, 0xffffffff;\n\tselp.u32 %0, 1, 0, P;\n\t}" : "=r"(p));
  return p != 0u;
}
__device__ __forceinline__ void tc_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
               : "memory");
}
__device__ __forceinline__ void tc_mma_bf16(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                            uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tc_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tc_ld_wait() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// K-major, 128B-swizzled operand tile: rows of 128 bytes, 8-row groups group_bytes apart.
__device__ __forceinline__ uint64_t make_smem_desc(uint32_t saddr, uint32_t group_bytes = 1024) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);        // start address, 16-byte units
  d |= static_cast<uint64_t>(1) << 16;                        // leading byte offset (unused here)
  d |= static_cast<uint64_t>(group_bytes >> 4) << 32;         // stride byte offset between 8-row groups
  d |= static_cast<uint64_t>(1) << 46;                        // descriptor version (Blackwell)
  d |= static_cast<uint64_t>(2) << 61;                        // SWIZZLE_128B
  return d;
}
// exp off by 2 + 1.2 |g| units of 2^-23, the quotient by 2 more: far below the bf16 rounding (2^-8) of the product that follows
__device__ __forceinline__ float silu_f(float g) { return __fdividef(g, 1.0f + __expf(-g)); }

// 16 FP8 values -> 16 bf16 (two 16-byte chunks), each bf16(float(q) * s)
__device__ __forceinline__ void convert16(const uint4& q, float s, uint4& lo, uint4& hi) {
  const __nv_fp8x2_storage_t* p = reinterpret_cast<const __nv_fp8x2_storage_t*>(&q);
  uint32_t o[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    __half2_raw hr = __nv_cvt_fp8x2_to_halfraw2(p[i], __NV_E4M3);
    float2 f = __half22float2(*reinterpret_cast<__half2*>(&hr));
    const float2 r = __fmul2_rn(f, make_float2(s, s));      // one instruction for the two products
    __nv_bfloat162 b = __floats2bfloat162_rn(r.x, r.y);
    o[i] = *reinterpret_cast<uint32_t*>(&b);
  }
  lo = make_uint4(o[0], o[1], o[2], o[3]);
  hi = make_uint4(o[4], o[5], o[6], o[7]);
}

// ---- rows of bf16 -----------------------------------------------------------------------
__device__ __forceinline__ void unpack8(const uint4& v, float* f) {
  const __nv_bfloat162* p = reinterpret_cast<const __nv_bfloat162*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 t = __bfloat1622float2(p[i]);
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}
// Rows of the kernel before this one, or of another GPU during this forward: an ordinary (coherent) load, kept in its place.
// Free to move the loads, the compiler holds all addresses in 64 registers and half the warps fit: combine of 65536 tokens
// of the V3 shape 2.37 ms, with 32 registers 1.43; of 32768 tokens of V2-236B 0.79 and 0.56.
__device__ __forceinline__ uint4 ld_row(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ uint4 pack8(const float* f) {
  uint4 v;
  __nv_bfloat162* p = reinterpret_cast<__nv_bfloat162*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) p[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
  return v;
}
__device__ __forceinline__ float round_bf16(float f) {
  return __bfloat162float(__float2bfloat16_rn(f));
}

// ---- rows of bytes ----------------------------------------------------------------------
// A row x is held as integers q in [-127, 127] and one scale: m = max(max|x|, 2^-100), scale = m / 127, inv = 127 / m (fp32,
// correctly rounded quotients), q = the integer nearest to x * inv, ties to even.  The product is rounded once: the fused
// multiply-add with 1.5 * 2^23 leaves the integer of the exact product in its low bits.  2^-100 keeps inv finite; rows below
// it, rows of zeros among them, come out as zeros.  A row that holds an infinity or a NaN has scale NaN and q = 0, so that
// every product of the row is NaN.
constexpr float kQuantFloor = 7.888609052210118e-31f;       // 2^-100

__device__ __forceinline__ void row_scale(uint32_t amax_bits, float& scale, float& inv) {
  const float m = fmaxf(__uint_as_float(amax_bits << 16), kQuantFloor);
  const bool finite = amax_bits < 0x7F80u;
  scale = finite ? __fdiv_rn(m, 127.0f) : __int_as_float(0x7FC00000);
  inv = finite ? __fdiv_rn(127.0f, m) : 0.0f;
}
// the two bf16 of a word -> their integers in the low bytes of lo and hi
__device__ __forceinline__ void quantise2(uint32_t pair, float inv, uint32_t& lo, uint32_t& hi) {
  lo = __float_as_uint(__fmaf_rn(__uint_as_float(pair << 16), inv, 12582912.0f));
  hi = __float_as_uint(__fmaf_rn(__uint_as_float(pair & 0xFFFF0000u), inv, 12582912.0f));
}
__device__ __forceinline__ uint32_t quantise4(uint32_t a, uint32_t b, float inv) {
  uint32_t q[4];
  quantise2(a, inv, q[0], q[1]);
  quantise2(b, inv, q[2], q[3]);
  return __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
}
// largest |x| of a 16-byte vector's halves and m's, as bf16 bits (an infinity or NaN is larger than any number)
__device__ __forceinline__ uint32_t amax8(uint32_t m, const uint4& a) {
  return __vmaxu2(__vmaxu2(m, a.x & 0x7FFF7FFFu),
                  __vmaxu2(a.y & 0x7FFF7FFFu, __vmaxu2(a.z & 0x7FFF7FFFu, a.w & 0x7FFF7FFFu)));
}
__device__ __forceinline__ uint2 quantise8(const uint4& a, float inv) {
  return inv == 0.0f ? make_uint2(0u, 0u) : make_uint2(quantise4(a.x, a.y, inv), quantise4(a.z, a.w, inv));
}

// ---- SM pairs (cta_group::2) -----------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_ctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t map_to_cta(uint32_t saddr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
  return r;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
// both CTAs of the pair issue it; the completion bytes are counted on the leader's barrier
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"(map), "r"(bar & 0xFEFFFFFFu), "r"(c0), "r"(c1)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(dst), "l"(map), "r"(bar & 0xFEFFFFFFu), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
__device__ __forceinline__ void tma_load_4d_pair(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3,
                                                 uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(dst), "l"(map), "r"(bar & 0xFEFFFFFFu), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
__device__ __forceinline__ void tc_commit_pair(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
      ::"r"(bar), "h"(static_cast<uint16_t>(3))
      : "memory");
}
// A CTA of a pair leaves only when the releases of all its slots have arrived: the leader's commits signal both CTAs, and one still
// on its way would find another block's shared memory.  Waits as if the n slots were filled once more, from slot i and phase ph on.
__device__ __forceinline__ void drain_slots(uint64_t* released, uint32_t i, uint32_t ph, uint32_t n, volatile int* abort_flag,
                                            int32_t* status, int where) {
  for (uint32_t left = n; left > 0 && mbar_wait(smem_u32(&released[i]), ph ^ 1u, abort_flag, status, where); --left)
    if (++i == n) { i = 0; ph ^= 1u; }
}
__device__ __forceinline__ void tc_mma_bf16_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                                 uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 2-D tensor map of a row-major matrix, from the handle's cache (gemm.cu)
enum TensorMapKind : uint32_t {
  TM_BF16 = 0,        // boxes of 64 bf16, SWIZZLE_128B: MMA operand tiles
  TM_FP8_ROWS = 1,    // boxes of 64 bytes, unswizzled
  TM_OUT_PIECE = 2,   // boxes of 32 bf16, SWIZZLE_64B: the epilogue's stores
  TM_OUT_16 = 3,      // boxes of 16 bf16, unswizzled: the SwiGLU stores of the weight-lane kernel
};

int encode_2d(const Handle* h, CUtensorMap* map, const void* base, uint64_t rows, uint64_t cols, uint32_t box_rows,
              TensorMapKind kind);

// tensor map of up to four dimensions, SWIZZLE_128B, of bytes or bf16: extents, strides in bytes of all but the inner one,
// box (gemm.cu; not cached)
int encode_map(CUtensorMap* map, const void* base, bool bytes, int rank, const uint64_t (&dims)[4],
               const uint64_t (&strides)[3], const uint32_t (&box)[4]);

}  // namespace mg
