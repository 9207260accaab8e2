// Rotary positions: y1 = x1 cos a - x2 sin a, y2 = x2 cos a + x1 sin a with
// a = position * f_i for pair i of the first rotary_dim elements of each head,
// pairs (i, i + rotary_dim/2) or (2i, 2i + 1), the rest of the head copied;
// optionally with the append of the turned K and the V into the paged cache
// (the reference has learned positions, engine/model.py:174-181, and copies K
// and V afterwards, engine/paged_cache.py:131-136).
//
// Bound by HBM: every element is read once and written once.  A thread owns
// one unit of a head, two 16-byte vectors (V pairs), for kHeads heads of one
// token, and issues all its loads first; while they are in flight the block
// computes its tokens' sines and cosines, each once, into shared memory (105 us
// where each thread computed its own, 62 so, at the size below: 5.4 TB/s; 65 and
// 5.1 where every call has other inputs).  The
// angle is kept in turns and reduced in fp64 (one multiply, one rounding, one
// subtraction), so the fp32 sine and cosine are those of the exact angle at any
// int32 position; no table is read.
#include "common.cuh"

namespace pse {
namespace {

// Heads of a token whose loads a thread has in flight together.  Two, with
// registers held to 48, so that 1280 threads stay resident (64 with the append, and
// 1024): 61.9 us at 16384 tokens, 32 + 8 heads of 128 in bf16, against 81.4 with
// four heads at 96 registers and 74.4 with one.
constexpr int kHeads = 2;

struct View {
  char* p;
  int64_t tok, head;  // strides in elements
};

struct RotaryArgs {
  View q, q_out, k, k_out, v;
  int q_heads, kv_heads;
  const double* turns;
  float factor;
  int hd, rd, interleaved;
  const int32_t* positions;
  int64_t tokens;
  int units, groups;  // units per head, head groups per token
  int copy_rest;      // q / k elements past rotary_dim must be copied too
  // append
  pse_block_state st;
  char *k_pool, *v_pool;
  const int32_t* slots;
  const int32_t* cache_pos;
};

template <int BYTES>
struct Raw;
template <>
struct Raw<16> { using type = uint4; };
template <>
struct Raw<8> { using type = uint2; };
template <>
struct Raw<4> { using type = uint32_t; };
template <>
struct Raw<2> { using type = uint16_t; };

template <typename T, int V>
union Vec {
  typename Raw<V * sizeof(T)>::type raw;
  T e[V];
  __device__ Vec() {}
};

// The fractional turn is exact to 2^-53 of a turn times the position, and
// sincospif takes it without a further reduction.
__device__ __forceinline__ void turn(double turns, int pos, float factor, float* c, float* s) {
  const double x = turns * (double)pos;
  const float f = (float)(x - rint(x));
  sincospif(2.f * f, s, c);
  *c *= factor;
  *s *= factor;
}

template <typename T, int V, bool APPEND>
__global__ void __launch_bounds__(256, APPEND ? 4 : 5) rotary_kernel(const RotaryArgs a) {
  extern __shared__ float cs[];  // per token of the block: rd / 2 cosines, rd / 2 sines
  using R = typename Raw<V * sizeof(T)>::type;
  pdl_wait();
  pdl_trigger();
  const int per_tok = a.units * a.groups;
  const int tpb = max(1, (int)blockDim.x / per_tok), half = a.rd / 2;
  const int n_heads = a.q_heads + a.kv_heads + (APPEND ? a.kv_heads : 0);
  const int n_rot = a.rd / (2 * V);  // units that turn
  const int64_t t0 = (int64_t)blockIdx.x * tpb;
  for (int e = threadIdx.x; e < tpb * per_tok || e < (int)blockDim.x; e += blockDim.x) {
    const int tb = e / per_tok;
    const int64_t t = t0 + tb;
    const bool work = tb < tpb && t < a.tokens;
    const int r = e - tb * per_tok, g = r / a.units, u = r - g * a.units;
    // element offsets of the unit's two vectors: a turned unit's partners, or
    // two neighbouring vectors that are copied
    const bool rot = u < n_rot;
    const int lo = rot && !a.interleaved ? u * V : u * 2 * V;
    const int hi = rot && !a.interleaved ? half + u * V : u * 2 * V + V;
    Vec<T, V> x[kHeads], y[kHeads];
    if (work) {
#pragma unroll
      for (int j = 0; j < kHeads; ++j) {
        const int h = g + j * a.groups;
        if (h >= n_heads) continue;
        const T* src;
        int l = lo, m = hi;
        if (h < a.q_heads) {
          src = reinterpret_cast<const T*>(a.q.p) + t * a.q.tok + h * a.q.head;
        } else if (h < a.q_heads + a.kv_heads) {
          src = reinterpret_cast<const T*>(a.k.p) + t * a.k.tok + (h - a.q_heads) * a.k.head;
        } else {
          src = reinterpret_cast<const T*>(a.v.p) + t * a.v.tok + (h - a.q_heads - a.kv_heads) * a.v.head;
          l = u * 2 * V;
          m = l + V;
        }
        x[j].raw = *reinterpret_cast<const R*>(src + l);
        y[j].raw = *reinterpret_cast<const R*>(src + m);
      }
    }
    int64_t page = -1;  // element offset of (block, head 0, row) in the pools, -1: nowhere
    if (APPEND && work) {
      const int slot = a.slots[t], pos = a.cache_pos[t];
      if (slot >= 0 && slot < a.st.num_slots && pos >= 0) {
        const int bi = pos / a.st.block_size;
        // blocks that were never reserved (pool exhausted) drop the token
        if (bi < a.st.nblocks[slot]) {
          const int blk = a.st.block_table[(int64_t)slot * a.st.max_blocks + bi];
          if (blk >= 0 && blk < a.st.num_blocks)
            page = ((int64_t)blk * a.kv_heads * a.st.block_size + pos % a.st.block_size) * a.hd;
        }
      }
    }
    if (e == threadIdx.x) {
      // the block's sines and cosines, once each, while the loads are in flight
      for (int i = threadIdx.x; i < tpb * half; i += blockDim.x) {
        const int k = i / half, p = i - k * half;
        if (t0 + k < a.tokens) turn(__ldg(a.turns + p), a.positions[t0 + k], a.factor, &cs[2 * k * half + p], &cs[2 * k * half + half + p]);
      }
      __syncthreads();
    }
    if (!work) continue;
    const float* c = cs + 2 * tb * half + u * V;
    const float* s = c + half;
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {
      const int h = g + j * a.groups;
      if (h >= n_heads) continue;
      const bool is_v = h >= a.q_heads + a.kv_heads;
      if (rot && !is_v) {
        if (a.interleaved) {
          // pair i of the unit: elements 2i and 2i + 1 of the two vectors in a row
#pragma unroll
          for (int i = 0; i < V; ++i) {
            T& e0 = 2 * i < V ? x[j].e[(2 * i) % V] : y[j].e[(2 * i) % V];
            T& e1 = 2 * i + 1 < V ? x[j].e[(2 * i + 1) % V] : y[j].e[(2 * i + 1) % V];
            const float p = to_f32(e0), w = to_f32(e1);
            e0 = from_f32<T>(p * c[i] - w * s[i]);
            e1 = from_f32<T>(w * c[i] + p * s[i]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float p = to_f32(x[j].e[i]), w = to_f32(y[j].e[i]);
            x[j].e[i] = from_f32<T>(p * c[i] - w * s[i]);
            y[j].e[i] = from_f32<T>(w * c[i] + p * s[i]);
          }
        }
      }
      auto put = [&](T* dst, int l, int m) {
        *reinterpret_cast<R*>(dst + l) = x[j].raw;
        *reinterpret_cast<R*>(dst + m) = y[j].raw;
      };
      if (h < a.q_heads) {
        if (rot || (a.copy_rest & 1)) put(reinterpret_cast<T*>(a.q_out.p) + t * a.q_out.tok + h * a.q_out.head, lo, hi);
      } else if (!is_v) {
        const int hk = h - a.q_heads;
        if (a.k_out.p && (rot || (a.copy_rest & 2)))
          put(reinterpret_cast<T*>(a.k_out.p) + t * a.k_out.tok + hk * a.k_out.head, lo, hi);
        if (APPEND && page >= 0)
          put(reinterpret_cast<T*>(a.k_pool) + page + (int64_t)hk * a.st.block_size * a.hd, lo, hi);
      } else if (APPEND && page >= 0) {
        const int hk = h - a.q_heads - a.kv_heads;
        put(reinterpret_cast<T*>(a.v_pool) + page + (int64_t)hk * a.st.block_size * a.hd, u * 2 * V, u * 2 * V + V);
      }
    }
  }
}

bool aligned(const View& v, int64_t esz, int bytes) {
  return !v.p || (reinterpret_cast<uintptr_t>(v.p) % bytes == 0 && (v.tok * esz) % bytes == 0 &&
                  (v.head * esz) % bytes == 0);
}

template <typename T, int V, bool APPEND>
int launch(RotaryArgs a, cudaStream_t s) {
  const int n_heads = a.q_heads + a.kv_heads + (APPEND ? a.kv_heads : 0);
  a.units = a.hd / (2 * V);
  a.groups = ceil_div(n_heads, kHeads);
  const int64_t per_tok = (int64_t)a.units * a.groups;
  if (per_tok >= (1 << 30)) return PSE_EINVAL;
  const int tpb = per_tok >= 256 ? 1 : (int)(256 / per_tok);
  const int threads = per_tok >= 256 ? 256 : ceil_div((int)per_tok * tpb, 32) * 32;
  const int64_t grid = (a.tokens + tpb - 1) / tpb;
  if (grid > 0x7fffffffll) return PSE_EINVAL;
  const size_t smem = (size_t)(threads / per_tok > tpb ? threads / per_tok : tpb) * a.rd * sizeof(float);
  if (smem > 48 * 1024) return PSE_EINVAL;  // (head_dim far beyond any layout here)
  const cudaError_t e = launch_pdl(rotary_kernel<T, V, APPEND>, dim3((unsigned)grid), dim3(threads), smem, s, a);
  return e == cudaSuccess ? PSE_OK : (int)e;
}

template <typename T, bool APPEND>
int dispatch(const RotaryArgs& a, cudaStream_t s) {
  // the widest vector that every base, stride and unit boundary allows
  auto fits = [&](int v) {
    const int bytes = v * (int)sizeof(T);
    bool ok = a.rd / 2 % v == 0 && (a.hd - a.rd) % (2 * v) == 0;
    for (const View* w : {&a.q, &a.q_out, &a.k, &a.k_out, &a.v}) ok = ok && aligned(*w, sizeof(T), bytes);
    if (APPEND)
      ok = ok && reinterpret_cast<uintptr_t>(a.k_pool) % bytes == 0 && reinterpret_cast<uintptr_t>(a.v_pool) % bytes == 0;
    return ok;
  };
  constexpr int V16 = 16 / sizeof(T);
  if (fits(V16)) return launch<T, V16, APPEND>(a, s);
  if (fits(V16 / 2)) return launch<T, V16 / 2, APPEND>(a, s);
  return launch<T, 1, APPEND>(a, s);
}

View view(const pse_head_view& v) { return View{reinterpret_cast<char*>(v.data), v.tok_stride, v.head_stride}; }

int fill(RotaryArgs& a, const pse_rotary_spec& r, const pse_head_view& q, const pse_head_view& q_out,
         const pse_head_view& k, const pse_head_view& k_out, const int32_t* positions, int64_t tokens) {
  if (tokens < 0 || r.head_dim <= 0 || r.head_dim % 2 || r.rotary_dim < 0 || r.rotary_dim % 2 ||
      r.rotary_dim > r.head_dim || q.heads < 0 || k.heads < 0 || q.heads > (1 << 20) || k.heads > (1 << 20))
    return PSE_EINVAL;
  if (tokens == 0 || q.heads + k.heads == 0) return PSE_OK;
  if (!positions || (r.rotary_dim > 0 && !r.turns) || (q.heads > 0 && (!q.data || !q_out.data || q_out.heads != q.heads)) ||
      (k.heads > 0 && !k.data) || (k_out.data && k_out.heads != k.heads))
    return PSE_EINVAL;
  a.q = view(q);
  a.q_out = view(q_out);
  a.k = view(k);
  a.k_out = view(k_out);
  a.v = View{nullptr, 0, 0};
  a.q_heads = q.heads;
  a.kv_heads = k.heads;
  a.turns = r.turns;
  a.factor = r.factor;
  a.hd = r.head_dim;
  a.rd = r.rotary_dim;
  a.interleaved = r.interleaved != 0;
  a.positions = positions;
  a.tokens = tokens;
  auto same = [](const View& x, const View& y) { return x.p == y.p && x.tok == y.tok && x.head == y.head; };
  a.copy_rest = (same(a.q, a.q_out) ? 0 : 1) | (same(a.k, a.k_out) ? 0 : 2);
  return PSE_OK;
}

}  // namespace
}  // namespace pse

using namespace pse;

extern "C" int pse_rotary(pse_rotary_spec r, const pse_head_view* views, const int32_t* positions, int64_t tokens,
                          int32_t dtype, void* stream) {
  if (!views) return PSE_EINVAL;
  const pse_head_view &q = views[0], &q_out = views[1], &k = views[2], &k_out = views[3];
  RotaryArgs a{};
  const int rc = fill(a, r, q, q_out, k, k_out, positions, tokens);
  if (rc != PSE_OK) return rc;
  if (dtype != PSE_F32 && dtype != PSE_BF16) return PSE_EINVAL;
  if (tokens == 0 || q.heads + k.heads == 0) return PSE_OK;
  if (k.heads > 0 && !k_out.data) return PSE_EINVAL;
  return dtype == PSE_BF16 ? dispatch<__nv_bfloat16, false>(a, (cudaStream_t)stream)
                           : dispatch<float, false>(a, (cudaStream_t)stream);
}

extern "C" int pse_rotary_append(pse_block_state st, pse_kv_layer kv, pse_rotary_spec r, const pse_head_view* views,
                                 const int32_t* positions, const int32_t* slots, const int32_t* cache_pos,
                                 int64_t tokens, void* stream) {
  if (!views) return PSE_EINVAL;
  const pse_head_view &q = views[0], &q_out = views[1], &k = views[2], &k_out = views[3], &v = views[4];
  RotaryArgs a{};
  const int rc = fill(a, r, q, q_out, k, k_out, positions, tokens);
  if (rc != PSE_OK) return rc;
  if (!st.block_table || !st.nblocks || st.block_size <= 0 || st.max_blocks <= 0 || !kv.k_pool || !kv.v_pool ||
      kv.kv_heads != k.heads || kv.head_dim != r.head_dim || v.heads != k.heads || k.heads <= 0)
    return PSE_EINVAL;
  if (kv.dtype != PSE_F32 && kv.dtype != PSE_BF16) return PSE_EINVAL;
  if (tokens == 0) return PSE_OK;
  if (!v.data || !slots || !cache_pos) return PSE_EINVAL;
  a.v = view(v);
  a.st = st;
  a.k_pool = reinterpret_cast<char*>(kv.k_pool);
  a.v_pool = reinterpret_cast<char*>(kv.v_pool);
  a.slots = slots;
  a.cache_pos = cache_pos;
  return kv.dtype == PSE_BF16 ? dispatch<__nv_bfloat16, true>(a, (cudaStream_t)stream)
                              : dispatch<float, true>(a, (cudaStream_t)stream);
}
