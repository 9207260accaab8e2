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
#pragma once

#include "common.cuh"

namespace pse {
namespace simt {

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
  float4 o[RPT][NC];
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
      for (int c = 0; c < NC; ++c) o[i][c] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
  }
  // rows of `dst` from row_ptr(r) (nullptr: zeros); scale applied to the values
  template <typename T, typename F>
  __device__ void fill(float* dst, int rows, F row_ptr, bool vec, float scale) {
    const int c4 = (hd + 3) / 4;
    for (int e = threadIdx.x; e < rows * c4; e += kThreads) {
      const int r = e / c4, d = (e - r * c4) * 4;
      const T* src = row_ptr(r);
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (src) x = load4<T>(src + d, hd - d, vec);
      if (scale != 1.f) {
        x.x *= scale;
        x.y *= scale;
        x.z *= scale;
        x.w *= scale;
      }
      *reinterpret_cast<float4*>(dst + (size_t)r * ld + d) = x;
    }
  }
  // One tile of BK keys (K, V and Q filled, a barrier passed).  visible(row,
  // key) is asked only when `masked`; weights of hidden keys take no part, so
  // what stands in a hidden key's V does not matter.
  template <typename F>
  __device__ void step(bool masked, F visible) {
    float s[RPT][4];
#pragma unroll
    for (int i = 0; i < RPT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
    const int c4 = (hd + 3) / 4;
    for (int c = 0; c < c4; ++c) {
      float4 a[RPT], b[4];
#pragma unroll
      for (int i = 0; i < RPT; ++i) a[i] = *reinterpret_cast<const float4*>(q + (size_t)(ty * RPT + i) * ld + 4 * c);
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j] = *reinterpret_cast<const float4*>(k + (size_t)(tx + 16 * j) * ld + 4 * c);
#pragma unroll
      for (int i = 0; i < RPT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          s[i][j] = fmaf(a[i].x, b[j].x, fmaf(a[i].y, b[j].y, fmaf(a[i].z, b[j].z, fmaf(a[i].w, b[j].w, s[i][j]))));
    }
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      if (masked) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (!visible(ty * RPT + i, tx + 16 * j)) s[i][j] = -INFINITY;
      }
      float mx = fmaxf(fmaxf(s[i][0], s[i][1]), fmaxf(s[i][2], s[i][3]));
#pragma unroll
      for (int w = 8; w > 0; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
      const float mn = fmaxf(m[i], mx), ms = mn == -INFINITY ? 0.f : mn;
      const float corr = exp2f(m[i] - ms);
      m[i] = mn;
      l[i] *= corr;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        o[i][c].x *= corr;
        o[i][c].y *= corr;
        o[i][c].z *= corr;
        o[i][c].w *= corr;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float w = exp2f(s[i][j] - ms);
        l[i] += w;
        p[(ty * RPT + i) * (BK + 4) + tx + 16 * j] = w;
      }
    }
    __syncwarp();  // a row's weights are written and read by one half warp
    for (int kk = 0; kk < BK; kk += 4) {
      float4 w[RPT];
#pragma unroll
      for (int i = 0; i < RPT; ++i) w[i] = *reinterpret_cast<const float4*>(p + (ty * RPT + i) * (BK + 4) + kk);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const int d = 4 * (tx + 16 * c);
          if (d >= hd) continue;
          const float4 b = *reinterpret_cast<const float4*>(v + (size_t)(kk + x) * ld + d);
#pragma unroll
          for (int i = 0; i < RPT; ++i) {
            const float y = x == 0 ? w[i].x : x == 1 ? w[i].y : x == 2 ? w[i].z : w[i].w;
            if (masked && y == 0.f) continue;
            o[i][c].x = fmaf(y, b.x, o[i][c].x);
            o[i][c].y = fmaf(y, b.y, o[i][c].y);
            o[i][c].z = fmaf(y, b.z, o[i][c].z);
            o[i][c].w = fmaf(y, b.w, o[i][c].w);
          }
        }
      }
    }
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
