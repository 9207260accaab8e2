// The softmax of one 128 x 128 score tile, shared by the prompt and tree
// kernels: scores come from tensor memory, weights go back there as bf16.
#pragma once

#include "tcgen05.cuh"

namespace pse {
namespace tile {

using namespace t5;

constexpr int kKeys = 128;

// A query row's running statistics, in units of log2: weights are taken
// against `m`, a maximum of the row's scores so far that is raised only when
// the true maximum has passed it by more than 8.  The weights stay below 2^8,
// the output then needs no rescaling in most tiles, and the quotient O / l is
// the same whatever reference both were taken against.
struct RowState {
  float m, l;
  __device__ void reset() {
    m = -INFINITY;
    l = 0.f;
  }
};

// One tile of one row (this thread's TMEM lane).  s_col: the 128 score columns,
// whose first 64 columns receive the weights, two bf16 to a column.  o_col: the
// row's HD output columns, rescaled here when `first` is false and the
// reference maximum moved.  masked (warp-uniform): only keys whose bit is set
// in vis[0..3] take part.  half_done[h] is arrived on (once per warp) when the
// weights of keys 64 h .. 64 h + 63 stand in tensor memory.
//
// The weights are rounded to bf16 for the tensor cores (the sum l adds them
// unrounded in fp32): 2^-8 of a weight at most, as much as the bf16 result's
// own rounding.
template <int HD>
__device__ __forceinline__ void softmax_tile(uint32_t lane_base, uint32_t s_col, uint32_t o_col, float sl2, bool first,
                                             bool masked, const uint32_t* vis, RowState& row, uint64_t* half0,
                                             uint64_t* half1) {
  uint32_t u[kKeys];
  float* s = reinterpret_cast<float*>(u);
#pragma unroll
  for (int c = 0; c < kKeys / 32; ++c) tmem_ld32(lane_base + s_col + 32 * c, u + 32 * c);
  tmem_wait_ld();
  if (masked) {
#pragma unroll
    for (int c = 0; c < kKeys; ++c) s[c] = (vis[c >> 5] >> (c & 31)) & 1u ? s[c] : -INFINITY;
  }
  float m4[4];
#pragma unroll
  for (int x = 0; x < 4; ++x) m4[x] = fmax3_nan(s[x], s[x + 4], s[x + 8]);
#pragma unroll
  for (int c = 12; c + 8 <= kKeys; c += 8) {
#pragma unroll
    for (int x = 0; x < 4; ++x) m4[x] = fmax3_nan(m4[x], s[c + x], s[c + 4 + x]);
  }
#pragma unroll
  for (int x = 0; x < 4; ++x) m4[x] = fmax3_nan(m4[x], s[kKeys - 4 + x], s[kKeys - 4 + x]);
  const float mx = fmax3_nan(fmax3_nan(m4[0], m4[1], m4[2]), m4[3], m4[3]) * sl2;
  // a NaN or +inf among the scores: the row's result is NaN
  if (!(mx < INFINITY)) row.l = __int_as_float(0x7fffffff);
  float corr = 1.f;
  if (mx > row.m + 8.f) {
    corr = ex2(row.m - mx);  // 0 from -inf
    row.m = mx;
  }
  row.l *= corr;
  if (!first && __any_sync(0xffffffffu, corr != 1.f)) {
    // every product issued before these scores has retired (their commit
    // covers it), so the output can be rescaled in place
#pragma unroll 1
    for (int c = 0; c < HD / 32; ++c) {
      uint32_t o[32];
      tmem_ld32(lane_base + o_col + 32 * c, o);
      tmem_wait_ld();
#pragma unroll
      for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * corr);
      tmem_st32(lane_base + o_col + 32 * c, o);
    }
  }
  const float neg = row.m == -INFINITY ? 0.f : -row.m;
  const uint64_t sc2 = pack2(sl2, sl2), neg2 = pack2(neg, neg);
  uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t p[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const int c = 64 * h + 2 * i;
      float lo, hi;
      unpack2(fma2(pack2(s[c], s[c + 1]), sc2, neg2), lo, hi);
      lo = ex2(lo);
      hi = ex2(hi);
      sum[i & 1] = add2(sum[i & 1], pack2(lo, hi));
      p[i] = pack_bf16(lo, hi);
    }
    tmem_st32(lane_base + s_col + 32 * h, p);
    tmem_wait_st();
    fence_before();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(h == 0 ? half0 : half1);
  }
  float a, b, c, d;
  unpack2(sum[0], a, b);
  unpack2(sum[1], c, d);
  row.l += (a + b) + (c + d);
}

// The same in rolled loops of 32 columns, the scores read twice: a quarter of the
// code and of the registers.  For kernels whose warps come back to a tile after
// much other code: there the instructions' own way through the caches counts (64
// trees of 5 to 26 nodes: 54 us, and 77 with the unrolled form above).
template <int HD>
__device__ __forceinline__ void softmax_tile_small(uint32_t lane_base, uint32_t s_col, uint32_t o_col, float sl2,
                                                   bool first, bool masked, uint32_t vis0, uint32_t vis1, uint32_t vis2,
                                                   uint32_t vis3, RowState& row, uint32_t half0) {
  const uint32_t sa = lane_base + s_col;
  float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
  for (int c = 0; c < kKeys; c += 32) {
    uint32_t u[32];
    float* f = reinterpret_cast<float*>(u);
    tmem_ld32(sa + c, u);
    tmem_wait_ld();
    if (masked) {
      // hidden scores become -inf where they stand, for the second pass
#pragma unroll
      for (int i = 0; i < 32; ++i) f[i] = vis0 >> i & 1u ? f[i] : -INFINITY;
      tmem_st32(sa + c, u);
      vis0 = vis1;
      vis1 = vis2;
      vis2 = vis3;
    }
#pragma unroll
    for (int i = 0; i < 32; i += 8) {
#pragma unroll
      for (int y = 0; y < 4; ++y) m4[y] = fmax3_nan(m4[y], f[i + y], f[i + 4 + y]);
    }
  }
  if (masked) tmem_wait_st();
  const float mx = fmax3_nan(fmax3_nan(m4[0], m4[1], m4[2]), m4[3], m4[3]) * sl2;
  // a NaN or +inf among the scores: the row's result is NaN
  if (!(mx < INFINITY)) row.l = __int_as_float(0x7fffffff);
  float corr = 1.f;
  if (mx > row.m + 8.f) {
    corr = ex2(row.m - mx);  // 0 from -inf
    row.m = mx;
  }
  row.l *= corr;
  if (!first && __any_sync(0xffffffffu, corr != 1.f)) {
    // every product issued before these scores has retired (their commit
    // covers it), so the output can be rescaled in place
#pragma unroll 1
    for (int c = 0; c < HD; c += 16) {
      uint32_t o[16];
      tmem_ld16(lane_base + o_col + c, o);
      tmem_wait_ld();
#pragma unroll
      for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * corr);
      tmem_st16(lane_base + o_col + c, o);
    }
  }
  const float neg = row.m == -INFINITY ? 0.f : -row.m;
  const uint64_t sc2 = pack2(sl2, sl2), neg2 = pack2(neg, neg);
  uint64_t sum[2] = {0ull, 0ull};
#pragma unroll 1
  for (int c = 0; c < kKeys; c += 32) {
    uint32_t u[32], p[16];
    const float* f = reinterpret_cast<const float*>(u);
    tmem_ld32(sa + c, u);
    tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float lo, hi;
      unpack2(fma2(pack2(f[2 * i], f[2 * i + 1]), sc2, neg2), lo, hi);
      lo = ex2(lo);
      hi = ex2(hi);
      sum[i & 1] = add2(sum[i & 1], pack2(lo, hi));
      p[i] = pack_bf16(lo, hi);
    }
    // over columns that have been read: chunk c's weights lie under chunk c / 2
    tmem_st16(sa + c / 2, p);
    if (c & 32) {
      tmem_wait_st();
      fence_before();
      __syncwarp();
      if ((threadIdx.x & 31) == 0) mbar_arrive(half0 + (c >> 6) * 8);
    }
  }
  float a, b, c, d;
  unpack2(sum[0], a, b);
  unpack2(sum[1], c, d);
  row.l += (a + b) + (c + d);
}

// 32 columns of an output row, scaled and rounded; vec: the row is 16-byte aligned.
__device__ __forceinline__ void store_row32(__nv_bfloat16* dst, const float* o, float inv, bool vec) {
#pragma unroll
  for (int x = 0; x < 32; x += 8) {
    uint4 w;
    w.x = pack_bf16(o[x] * inv, o[x + 1] * inv);
    w.y = pack_bf16(o[x + 2] * inv, o[x + 3] * inv);
    w.z = pack_bf16(o[x + 4] * inv, o[x + 5] * inv);
    w.w = pack_bf16(o[x + 6] * inv, o[x + 7] * inv);
    if (vec) {
      *reinterpret_cast<uint4*>(dst + x) = w;
    } else {
      unsigned short* d = reinterpret_cast<unsigned short*>(dst + x);
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const uint32_t v = y == 0 ? w.x : y == 1 ? w.y : y == 2 ? w.z : w.w;
        d[2 * y] = (unsigned short)v;
        d[2 * y + 1] = (unsigned short)(v >> 16);
      }
    }
  }
}

// A whole warp: sets the infinities and NaN among n vectors of 8 bf16 (n a
// multiple of 256) in shared memory to zero, visible to later products; returns
// whether there were any.
__device__ __forceinline__ bool clear_nonfinite(uint4* v, int n) {
  const int lane = threadIdx.x & 31;
  const __nv_bfloat162 zero = __floats2bfloat162_rn(0.f, 0.f);
  bool bad = false;
#pragma unroll 1
  for (int i = lane; i < n; i += 256) {
    // 0 x value, summed: NaN if any value is not finite, else a zero
    __nv_bfloat162 z = zero;
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const uint4 w = v[i + 32 * x];
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const uint32_t b = y == 0 ? w.x : y == 1 ? w.y : y == 2 ? w.z : w.w;
        z = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&b), zero, z);
      }
    }
    bad |= !(__low2float(z) == 0.f && __high2float(z) == 0.f);
  }
  bad = __any_sync(0xffffffffu, bad);
  if (bad) {
    uint32_t* w = reinterpret_cast<uint32_t*>(v);
#pragma unroll 1
    for (int i = lane; i < 4 * n; i += 32) {
      uint32_t x = w[i];
      if ((x & 0x7f80u) == 0x7f80u) x &= 0xffff0000u;
      if ((x & 0x7f800000u) == 0x7f800000u) x &= 0x0000ffffu;
      w[i] = x;
    }
    fence_proxy();
  }
  __syncwarp();
  return bad;
}

}  // namespace tile
}  // namespace pse
