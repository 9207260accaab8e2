// One query tile of attention on the CUDA cores in fp32, for the shapes and
// types the tensor-core kernels do not take (fp32 pools, head sizes other than
// 64 and 128, unaligned rows).
//
// 256 threads as 16 x 16: thread (ty, tx) holds RPT rows' scores of keys tx,
// tx + 16, tx + 32, tx + 48 and, of the output, the 4-column chunks tx, tx + 16,
// ... of the same rows, so a row's maximum and sum stay within 16 lanes.  Q, K,
// V and the weights of a tile stand in shared memory as fp32 with rows padded
// by 4 floats (16 lanes reading 16 rows' vectors touch every bank once per
// quarter warp).  One pass over the keys with a running maximum and sum.
//
// Products in pairs of columns (two fp32 results an instruction), a tile's loads
// together, masks as bits per row.  8 prompts of 1000 tokens, 12 heads of 64: 480
// us, 26 TFLOP/s (1080 us and 11 with 16 query rows per block instead of 64); bound
// by the instructions of the two blocks, 16 warps, that a multiprocessor holds (2.3
// a clock), and by a tile's loads, which nothing is multiplied under.  Few short
// prompts leave a block alone on its multiprocessor, its 8 warps waiting in turn for
// each tile's loads and for each other: the five tiles of 300 tokens take 37 to 47 us.
#pragma once

#include "tcgen05.cuh"

namespace pse {
namespace simt {

using t5::fma2;
using t5::mul2;
using t5::pack2;
using t5::unpack2;

constexpr int kThreads = 256;
constexpr int BK = 64;

// Up to 4 elements of a row as fp32 (zeros past n).
template <typename T>
__device__ __forceinline__ float4 load4(const T* p, int n, bool vec) {
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (vec && n >= 4) {
    if constexpr (sizeof(T) == 4) {
      v = *reinterpret_cast<const float4*>(p);
    } else {
      const uint2 u = *reinterpret_cast<const uint2*>(p);
      const __nv_bfloat162 a = *reinterpret_cast<const __nv_bfloat162*>(&u.x);
      const __nv_bfloat162 b = *reinterpret_cast<const __nv_bfloat162*>(&u.y);
      v = make_float4(__bfloat162float(a.x), __bfloat162float(a.y), __bfloat162float(b.x), __bfloat162float(b.y));
    }
  } else {
    if (n > 0) v.x = to_f32(p[0]);
    if (n > 1) v.y = to_f32(p[1]);
    if (n > 2) v.z = to_f32(p[2]);
    if (n > 3) v.w = to_f32(p[3]);
  }
  return v;
}

template <int RPT>
__host__ __device__ constexpr size_t smem_floats(int hd) {
  const int ld = (hd + 3) / 4 * 4 + 4;
  return (size_t)(16 * RPT + 2 * BK) * ld + (size_t)16 * RPT * (BK + 4);
}

// NC: 64-column groups of the head (head_dim <= 64 NC).
template <int RPT, int NC>
struct Tile {
  static constexpr int BQ = 16 * RPT;
  int hd, ld, tx, ty;
  float *q, *k, *v, *p;
  uint64_t o[RPT][NC][2];  // pairs of columns
  float m[RPT], l[RPT];

  __device__ void init(float* smem, int head_dim) {
    hd = head_dim;
    ld = (hd + 3) / 4 * 4 + 4;
    tx = threadIdx.x & 15;
    ty = threadIdx.x >> 4;
    q = smem;
    k = q + BQ * ld;
    v = k + BK * ld;
    p = v + BK * ld;
  }
  __device__ void reset() {
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      m[i] = -INFINITY;
      l[i] = 0.f;
#pragma unroll
      for (int c = 0; c < NC; ++c) o[i][c][0] = o[i][c][1] = 0ull;
    }
  }
  // Q from row(r) (nullptr: zeros), scaled.  Here and below a thread's loads are on
  // their way together: one after the other their latency was most of a short
  // item's time.
  template <typename T, typename F>
  __device__ void fill_q(F row, bool vec, float scale) {
    const int c4 = (hd + 3) / 4;
#pragma unroll 1
    for (int e0 = threadIdx.x; e0 < BQ * c4; e0 += RPT * kThreads) {
      float4 x[RPT];
#pragma unroll
      for (int i = 0; i < RPT; ++i) {
        const int e = min(e0 + i * kThreads, BQ * c4 - 1), r = e / c4, d = (e - r * c4) * 4;
        const T* src = row(r);
        x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (src) x[i] = load4<T>(src + d, hd - d, vec);
      }
#pragma unroll
      for (int i = 0; i < RPT; ++i) {
        const int e = e0 + i * kThreads, r = e / c4, d = (e - r * c4) * 4;
        if (e < BQ * c4)
          *reinterpret_cast<float4*>(q + (size_t)r * ld + d) =
              make_float4(x[i].x * scale, x[i].y * scale, x[i].z * scale, x[i].w * scale);
      }
    }
  }
  // BK rows of K and V; rows(r, ks, vs) sets their pointers (or leaves nullptr: zeros)
  template <typename T, typename F>
  __device__ void fill_kv(F rows, bool kvec, bool vvec) {
    const int c4 = (hd + 3) / 4;
#pragma unroll 1
    for (int e0 = threadIdx.x; e0 < BK * c4; e0 += 4 * kThreads) {
      float4 x[4], y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = min(e0 + i * kThreads, BK * c4 - 1), r = e / c4, d = (e - r * c4) * 4;
        const T *ks = nullptr, *vs = nullptr;
        rows(r, ks, vs);
        x[i] = y[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (ks) {
          x[i] = load4<T>(ks + d, hd - d, kvec);
          y[i] = load4<T>(vs + d, hd - d, vvec);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = e0 + i * kThreads, r = e / c4, d = (e - r * c4) * 4;
        if (e < BK * c4) {
          *reinterpret_cast<float4*>(k + (size_t)r * ld + d) = x[i];
          *reinterpret_cast<float4*>(v + (size_t)r * ld + d) = y[i];
        }
      }
    }
  }
  // One tile of BK keys (K, V and Q filled, a barrier passed).  visible(i), asked
  // only when `masked`, has a bit for each key that this thread's row i sees;
  // weights of hidden keys take no part, so what stands in a hidden key's V does
  // not matter.
  template <typename F>
  __device__ void step(bool masked, F visible) {
    // (sums of the even and of the odd columns)
    uint64_t s2[RPT][4];
#pragma unroll
    for (int i = 0; i < RPT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) s2[i][j] = 0ull;
    const int c4 = (hd + 3) / 4;
#pragma unroll 4
    for (int c = 0; c < c4; ++c) {
      ulonglong2 a[RPT], b[4];
#pragma unroll
      for (int i = 0; i < RPT; ++i) a[i] = *reinterpret_cast<const ulonglong2*>(q + (size_t)(ty * RPT + i) * ld + 4 * c);
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j] = *reinterpret_cast<const ulonglong2*>(k + (size_t)(tx + 16 * j) * ld + 4 * c);
#pragma unroll
      for (int i = 0; i < RPT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s2[i][j] = fma2(a[i].x, b[j].x, fma2(a[i].y, b[j].y, s2[i][j]));
    }
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      float s[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float odd;
        unpack2(s2[i][j], s[j], odd);
        s[j] += odd;
      }
      uint64_t vis = ~0ull;
      if (masked) {
        vis = visible(i) >> tx;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (!(vis >> (16 * j) & 1ull)) s[j] = -INFINITY;
      }
      float mx = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
#pragma unroll
      for (int w = 8; w > 0; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
      const float mn = fmaxf(m[i], mx), ms = mn == -INFINITY ? 0.f : mn;
      const float corr = exp2f(m[i] - ms);
      m[i] = mn;
      l[i] *= corr;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        o[i][c][0] = mul2(o[i][c][0], pack2(corr, corr));
        o[i][c][1] = mul2(o[i][c][1], pack2(corr, corr));
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float w = exp2f(s[j] - ms);
        l[i] += w;
        // (a hidden key's zero is negative: a seen key's weight may underflow)
        p[(ty * RPT + i) * (BK + 4) + tx + 16 * j] = masked && !(vis >> (16 * j) & 1ull) ? -0.f : w;
      }
    }
    __syncwarp();  // a row's weights are written and read by one half warp
    if (masked)
      values<true>();
    else
      values<false>();
  }
  // o += p v.  Columns past the head's are computed and not used (their reads end
  // inside the tile's memory).  MASKED: a hidden key's weight (-0) takes no part,
  // which matters where V is infinite or NaN.
  template <bool MASKED>
  __device__ __forceinline__ void values() {
#pragma unroll 4
    for (int kk = 0; kk < BK; kk += 4) {
      float4 w[RPT];
#pragma unroll
      for (int i = 0; i < RPT; ++i) w[i] = *reinterpret_cast<const float4*>(p + (ty * RPT + i) * (BK + 4) + kk);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(v + (size_t)(kk + x) * ld + 4 * (tx + 16 * c));
          bool skip = false;
          if (MASKED) {
            float f[4];
            unpack2(b.x, f[0], f[1]);
            unpack2(b.y, f[2], f[3]);
            skip = !(fabsf(f[0]) + fabsf(f[1]) + fabsf(f[2]) + fabsf(f[3]) < INFINITY);
          }
#pragma unroll
          for (int i = 0; i < RPT; ++i) {
            const float y = x == 0 ? w[i].x : x == 1 ? w[i].y : x == 2 ? w[i].z : w[i].w;
            if (skip && __float_as_uint(y) == 0x80000000u) continue;
            o[i][c][0] = fma2(pack2(y, y), b.x, o[i][c][0]);
            o[i][c][1] = fma2(pack2(y, y), b.y, o[i][c][1]);
          }
        }
      }
    }
  }
  // columns 4 (tx + 16 c) .. + 3 of the thread's row i
  __device__ float4 out(int i, int c) const {
    float4 x;
    unpack2(o[i][c][0], x.x, x.y);
    unpack2(o[i][c][1], x.z, x.w);
    return x;
  }
  // the row's sum over its 16 lanes
  __device__ float row_sum(int i) const {
    float x = l[i];
#pragma unroll
    for (int w = 8; w > 0; w >>= 1) x += __shfl_xor_sync(0xffffffffu, x, w);
    return x;
  }
};

template <typename T>
__device__ __forceinline__ void store4(T* p, int n, float4 v) {
  if (n > 0) p[0] = from_f32<T>(v.x);
  if (n > 1) p[1] = from_f32<T>(v.y);
  if (n > 2) p[2] = from_f32<T>(v.z);
  if (n > 3) p[3] = from_f32<T>(v.w);
}

}  // namespace simt
}  // namespace pse
