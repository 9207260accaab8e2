// sm_100a building blocks of the attention kernels on the 5th-generation tensor
// cores: mbarriers with bounded waits, TMA tile loads, tcgen05 matrix
// products, tensor-memory loads and stores, packed fp32 arithmetic.
#pragma once

#include <cuda.h>

#include "common.cuh"

namespace pse {
namespace t5 {

constexpr uint32_t kSpinLimit = 1u << 18;  // tries, a few microseconds each

// The bound of a role's waits, and the flag by which the CTA's other roles learn
// that one of them has expired.
struct Waits {
  volatile int* abort_flag;
  uint32_t tries;
};
// The bound for the next launch's products: kSpinLimit, unless a test has set
// another.  The other roles keep kSpinLimit in their code and give up with the
// products (with a bound from the arguments in every wait, 64 short trees took 51.5 us
// instead of 50.7).
uint32_t wait_tries();

__device__ __forceinline__ uint32_t su32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// ---------------------------------------------------------------- mbarriers
__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(su32(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(su32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(su32(bar)) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// Bounded wait that also gives up once another role of the CTA has.  (Each try
// suspends the thread in hardware for a while.  The loop is this short because
// it stands in some thirty places: kernels whose warps walk different code
// spend their time fetching it when it outgrows the instruction cache.)
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, const Waits& w) {
#pragma unroll 1
  for (uint32_t n = 0; n < w.tries; ++n) {
    if (mbar_try_wait(bar, parity)) return true;
    if (*w.abort_flag) return false;
  }
  *w.abort_flag = 1;
  return false;
}
// The same for a whole warp: every lane gets the same answer.  All lanes poll:
// the warp has to arrive converged at the .aligned tensor-memory accesses that
// follow, and a poll by one lane joined by a vote does not ensure that.
__device__ __forceinline__ bool mbar_wait_warp(uint32_t bar, uint32_t parity, const Waits& w) {
  const bool ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, w));
  __syncwarp();
  return ok;
}
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, const Waits& w) {
  return mbar_wait(su32(bar), parity, w);
}
__device__ __forceinline__ bool mbar_wait_warp(uint64_t* bar, uint32_t parity, const Waits& w) {
  return mbar_wait_warp(su32(bar), parity, w);
}
// Waits for three barriers at once (repeat one for fewer): their polls are on
// their way together.
__device__ __forceinline__ bool mbar_wait3_warp(uint32_t a, uint32_t pa, uint32_t b, uint32_t pb, uint32_t c, uint32_t pc,
                                                const Waits& w) {
  bool ok = false;
#pragma unroll 1
  for (uint32_t n = 0; n < w.tries; ++n) {
    const bool x = mbar_try_wait(a, pa), y = mbar_try_wait(b, pb), z = mbar_try_wait(c, pc);
    if (x && y && z) {
      ok = true;
      break;
    }
    if (*w.abort_flag) break;
  }
  if (!ok) *w.abort_flag = 1;
  ok = __all_sync(0xffffffffu, ok);
  __syncwarp();
  return ok;
}
// Bounded wait of the exit path (no abort check).
__device__ __forceinline__ void mbar_drain(uint32_t bar, uint32_t parity) {
  for (uint32_t n = 0; n < kSpinLimit; ++n) {
    if (mbar_try_wait(bar, parity)) return;
    if (n >= 64) __nanosleep(64);
  }
}
__device__ __forceinline__ void mbar_drain(uint64_t* bar, uint32_t parity) { mbar_drain(su32(bar), parity); }

// ---------------------------------------------------------------- TMA
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(su32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(su32(bar))
      : "memory");
}

// From a converged warp, issued by its elected lane (see mma_ss below).
__device__ __forceinline__ void tma_load_2d(uint32_t elected, uint32_t dst, const CUtensorMap* map, int x, int y,
                                            uint32_t bar) {
  asm volatile(
      "{\n .reg .pred e;\n setp.ne.b32 e, %5, 0;\n"
      " @e cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
      "[%4];\n}\n" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar), "r"(elected)
      : "memory");
}

// Whether a [tokens, heads, hd] bf16 view can be read through a 3-D tensor map.
inline bool tma_rows(const char* p, int64_t tok, int64_t head, int heads, int hd) {
  if (heads == 1) head = hd;  // the stride of an axis of one is not used
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && tok % 8 == 0 && head % 8 == 0 && tok >= hd && head >= hd &&
         tok < (1ll << 38) && head < (1ll << 38);
}

// ---------------------------------------------------------------- tensor cores
// Shared-memory operand descriptors, 128-byte swizzle.  K-major: rows 128 B
// apart, 8-row groups 1024 B apart, a 16-element K step 32 B inside the row.
__device__ __forceinline__ uint64_t desc_kmajor(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
         (uint64_t)2 << 61;
}
// MN-major (V as the B operand of P V): 64 columns x 8 keys per 1024 B atom,
// atoms `lbo` bytes apart along the columns, 1024 B along the keys.
__device__ __forceinline__ uint64_t desc_mnmajor(uint32_t addr, uint32_t lbo) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | (uint64_t)((lbo >> 4) & 0x3FFF) << 16 | (uint64_t)(1024 >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// bf16 x bf16 -> fp32, M = 128, N = n; b_mn: B is MN-major.
__host__ __device__ constexpr uint32_t instr_desc(int n, int b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(128 >> 4) << 24);
}
// The products and commits below are called by a whole converged warp with the
// same operands in every lane and issued by the lane that elect_one picked:
// operands that are uniform over the warp stay in uniform registers, where
// the instruction wants them.  Issued from a branch of one lane, every operand
// is moved there first, about 130 clocks per product against 64 of the product.
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t e;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(e));
  return e;
}
__device__ __forceinline__ void mma_ss(uint32_t elected, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p, e;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 e, %5, 0;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(elected)
      : "memory");
}
// A in tensor memory: row r is lane r, 16-bit elements two to a column.
__device__ __forceinline__ void mma_ts(uint32_t elected, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                       uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p, e;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 e, %5, 0;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(elected)
      : "memory");
}
// The barrier's arrival waits for every tcgen05 operation the elected thread issued before.
__device__ __forceinline__ void mma_commit(uint32_t elected, uint32_t bar) {
  asm volatile(
      "{\n .reg .pred e;\n setp.ne.b32 e, %1, 0;\n"
      " @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(bar),
      "r"(elected)
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t elected, uint64_t* bar) { mma_commit(elected, su32(bar)); }

// S = Q K^T (M = N = 128) over head_dim HD: both operands as HD / 64 column
// halves of 16 KB.
template <int HD>
__device__ __forceinline__ void issue_scores(uint32_t elected, uint32_t d, uint32_t q, uint32_t k) {
  const uint64_t a = desc_kmajor(q), b = desc_kmajor(k);
#pragma unroll
  for (int kk = 0; kk < HD / 16; ++kk) {
    const uint64_t off = ((kk >> 2) * (128 * 128) + (kk & 3) * 32) >> 4;
    mma_ss(elected, d, a + off, b + off, instr_desc(128, 0), kk > 0);
  }
}
// O += P V for keys 64 h .. 64 h + 63 of a tile (N = HD), P in tensor memory, V
// MN-major; fresh: the first product overwrites O.
template <int HD>
__device__ __forceinline__ void issue_values(uint32_t elected, uint32_t o, uint32_t p, uint32_t v, int h, bool fresh) {
  const uint64_t b = desc_mnmajor(v + h * 8192, HD == 128 ? 128u * 128u : 1024u);
  p += 32 * h;
#pragma unroll
  for (int kk = 0; kk < 4; ++kk)
    mma_ts(elected, o, p + 8 * kk, b + ((kk * 2048) >> 4), instr_desc(HD, 1), kk > 0 || !fresh);
}

#define PSE_T5_R32(r)                                                                                               \
  "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),       \
      "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),        \
      "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),       \
      "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
#define PSE_T5_W32(r)                                                                                               \
  "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),      \
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),   \
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),   \
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])

// 32 consecutive columns of this thread's lane (the load needs tmem_wait_ld).
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : PSE_T5_R32(r)
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      PSE_T5_W32(r)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// Orders this thread's shared-memory writes before later asynchronous reads (MMA, TMA).
__device__ __forceinline__ void fence_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ---------------------------------------------------------------- arithmetic
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The largest of three, NaN if any is.
__device__ __forceinline__ float fmax3_nan(float a, float b, float c) {
  float y;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
  return v;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

}  // namespace t5
}  // namespace pse
