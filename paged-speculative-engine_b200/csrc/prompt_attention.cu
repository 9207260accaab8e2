// Causal attention over packed prompts of different lengths: token i of a
// prompt attends to its tokens 0..i (engine/model.py:99-116 without the
// padding), O_i = sum_j softmax_j(q_i . k_j scale) v_j, query head h reading
// K/V head h / (q_heads / kv_heads).
//
// Work is planned on the host (the lengths are known there when the prompts
// are packed): an item is one prompt, one K/V head and two query tiles of
// 128 / group tokens each, the group's heads side by side in a tile; the items
// are dealt to the CTAs longest first, each to the CTA with the least work so
// far, which needs no counter on the device and gives the same order of
// operations in every call.
#include <algorithm>
#include <queue>
#include <vector>

#include "simt_attention.cuh"

namespace pse {
namespace prompt {

struct Args {
  const char *q, *k, *v;
  char* out;
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head, o_tok, o_head;  // elements
  int64_t tokens;
  int q_heads, kv_heads, group, hd;
  float scale_log2;
  const int32_t* plan;  // [n_cta + 1] first items, padding, then int4 {first token, length, first query token, K/V head}
  int n_cta, n_items;
  int32_t* status;
};

// Tokens of one query tile: at most 128 rows of (token, group head).
__host__ __device__ inline int tile_tokens(int group) { return group >= 128 ? 1 : 128 / group; }
__host__ __device__ inline int plan_items_at(int n_cta) { return (n_cta + 4) / 4 * 4; }

// ---------------------------------------------------------------- CUDA cores
template <typename T, int NC>
__global__ void __launch_bounds__(simt::kThreads) prompt_simt_kernel(const Args a) {
  extern __shared__ float smem[];
  const int subs = ceil_div(2 * tile_tokens(a.group) * a.group, 64);
  const int4 it = reinterpret_cast<const int4*>(a.plan + plan_items_at(a.n_cta))[blockIdx.x / subs];
  const int tok0 = it.x, len = it.y, hk = it.w;
  // an item that the tensors do not hold is skipped (a plan made for others)
  if (tok0 < 0 || len < 0 || it.z < 0 || (int64_t)tok0 + len > a.tokens || hk < 0 || hk >= a.kv_heads) return;
  const int64_t r0 = (int64_t)it.z * a.group + (blockIdx.x % subs) * 64;
  const int64_t r_end = (int64_t)min(len, it.z + 2 * tile_tokens(a.group)) * a.group;
  const int nr = (int)min((int64_t)64, r_end - r0);
  if (nr <= 0) return;
  simt::Tile<4, NC> t;
  t.init(smem, a.hd);
  t.reset();
  auto vec = [&](const char* p, int64_t tok, int64_t head) {
    return reinterpret_cast<uintptr_t>(p) % (4 * sizeof(T)) == 0 && tok % 4 == 0 && head % 4 == 0;
  };
  const T* q = reinterpret_cast<const T*>(a.q);
  const T* k = reinterpret_cast<const T*>(a.k) + hk * a.k_head;
  const T* v = reinterpret_cast<const T*>(a.v) + hk * a.v_head;
  t.template fill<T>(
      t.q, 64,
      [&](int r) -> const T* {
        if (r >= nr) return nullptr;
        const int64_t rr = r0 + r;
        return q + (tok0 + rr / a.group) * a.q_tok + (hk * a.group + rr % a.group) * a.q_head;
      },
      vec(a.q, a.q_tok, a.q_head), a.scale_log2);
  const int kmax = (int)((r0 + nr - 1) / a.group) + 1;  // keys the last row sees
  const bool kvec = vec(a.k, a.k_tok, a.k_head), vvec = vec(a.v, a.v_tok, a.v_head);
  for (int k0 = 0; k0 < kmax; k0 += simt::BK) {
    __syncthreads();
    t.template fill<T>(
        t.k, simt::BK,
        [&](int r) -> const T* { return k0 + r < kmax ? k + (int64_t)(tok0 + k0 + r) * a.k_tok : nullptr; }, kvec, 1.f);
    t.template fill<T>(
        t.v, simt::BK,
        [&](int r) -> const T* { return k0 + r < kmax ? v + (int64_t)(tok0 + k0 + r) * a.v_tok : nullptr; }, vvec, 1.f);
    __syncthreads();
    t.step(k0 + simt::BK > (int)(r0 / a.group) + 1,
           [&](int r, int key) { return k0 + key <= (int)((r0 + r) / a.group); });
  }
  T* out = reinterpret_cast<T*>(a.out);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float L = t.row_sum(i);
    const int r = t.ty * 4 + i;
    if (r >= nr) continue;
    const int64_t rr = r0 + r;
    T* dst = out + (tok0 + rr / a.group) * a.o_tok + (hk * a.group + rr % a.group) * a.o_head;
    // a sum of zero (every score -inf) gives zero
    const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int d = 4 * (t.tx + 16 * c);
      float4 x = t.o[i][c];
      x.x *= inv;
      x.y *= inv;
      x.z *= inv;
      x.w *= inv;
      if (d < a.hd) simt::store4(dst + d, a.hd - d, x);
    }
  }
}

template <typename T, int NC>
int launch_simt(const Args& a, cudaStream_t s) {
  auto kern = prompt_simt_kernel<T, NC>;
  const size_t smem = simt::smem_floats<4>(a.hd) * sizeof(float);
  static const cudaError_t opt = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                      (int)(simt::smem_floats<4>(64 * NC) * sizeof(float)));
  if (opt != cudaSuccess) return (int)opt;
  const int64_t subs = ceil_div(2 * tile_tokens(a.group) * a.group, 64);
  if (subs * a.n_items > 0x7fffffffll) return PSE_EINVAL;
  kern<<<(unsigned)(subs * a.n_items), simt::kThreads, smem, s>>>(a);
  PSE_LAUNCH_CHECK();
  return PSE_OK;
}

template <typename T>
int simt_attention(const Args& a, cudaStream_t s) {
  if (a.hd <= 64) return launch_simt<T, 1>(a, s);
  if (a.hd <= 128) return launch_simt<T, 2>(a, s);
  return launch_simt<T, 4>(a, s);
}

// ---------------------------------------------------------------- planning
struct Item {
  int32_t tok0, len, w0, hk;
  int64_t cost;
};

int make_plan(const int32_t* lens, int32_t n, int32_t q_heads, int32_t kv_heads, int32_t n_cta, int32_t* out,
              int64_t cap, int64_t* n_ints) {
  if (n < 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads || n_cta <= 0 || n_cta > 65536 || !n_ints ||
      (n > 0 && !lens))
    return PSE_EINVAL;
  const int per = 2 * tile_tokens(q_heads / kv_heads);
  int64_t total = 0, items = 0;
  for (int32_t i = 0; i < n; ++i) {
    if (lens[i] < 0) return PSE_EINVAL;
    total += lens[i];
    items += ((int64_t)lens[i] + per - 1) / per * kv_heads;
  }
  if (total > 0x7fffffffll || items > 0x1fffffffll) return PSE_EINVAL;
  *n_ints = plan_items_at(n_cta) + 4 * items;
  if (!out) return PSE_OK;
  if (cap < *n_ints) return PSE_EWORKSPACE;
  std::vector<Item> all;
  all.reserve((size_t)items);
  int32_t tok0 = 0;
  for (int32_t i = 0; i < n; ++i) {
    for (int32_t w0 = 0; w0 < lens[i]; w0 += per)
      for (int32_t h = 0; h < kv_heads; ++h) {
        const int64_t keys = std::min<int64_t>((int64_t)w0 + per, lens[i]);
        // key tiles, and two tiles' time for an item's start and end
        all.push_back(Item{tok0, lens[i], w0, h, (keys + 127) / 128 + 2});
      }
    tok0 += lens[i];
  }
  std::stable_sort(all.begin(), all.end(), [](const Item& x, const Item& y) { return x.cost > y.cost; });
  using Load = std::pair<int64_t, int32_t>;  // (work so far, CTA)
  std::priority_queue<Load, std::vector<Load>, std::greater<Load>> heap;
  for (int32_t c = 0; c < n_cta; ++c) heap.push({0, c});
  std::vector<int32_t> owner(all.size());
  std::vector<int32_t> count((size_t)n_cta + 1, 0);
  for (size_t e = 0; e < all.size(); ++e) {
    Load x = heap.top();
    heap.pop();
    owner[e] = x.second;
    ++count[(size_t)x.second + 1];
    x.first += all[e].cost;
    heap.push(x);
  }
  for (int32_t c = 0; c < n_cta; ++c) count[(size_t)c + 1] += count[(size_t)c];
  for (int c = 0; c < plan_items_at(n_cta); ++c) out[c] = c <= n_cta ? count[(size_t)c] : 0;
  std::vector<int32_t> at(count.begin(), count.end() - 1);
  int32_t* dst = out + plan_items_at(n_cta);
  for (size_t e = 0; e < all.size(); ++e) {
    int32_t* p = dst + 4 * (int64_t)at[(size_t)owner[e]]++;
    p[0] = all[e].tok0;
    p[1] = all[e].len;
    p[2] = all[e].w0;
    p[3] = all[e].hk;
  }
  return PSE_OK;
}

}  // namespace prompt
}  // namespace pse

using namespace pse;

extern "C" int pse_prompt_plan(const int32_t* lens, int32_t n, int32_t q_heads, int32_t kv_heads, int32_t n_cta,
                               int32_t* plan, int64_t plan_ints, int64_t* n_ints) {
  try {
    return prompt::make_plan(lens, n, q_heads, kv_heads, n_cta, plan, plan_ints, n_ints);
  } catch (const std::bad_alloc&) {
    return PSE_EINVAL;
  }
}

extern "C" int pse_prompt_attention(pse_head_view q, pse_head_view k, pse_head_view v, pse_head_view out,
                                    int64_t tokens, int32_t head_dim, int32_t dtype, float scale, const int32_t* plan,
                                    int32_t n_cta, int64_t n_items, int32_t* status, void* stream) {
  if (tokens < 0 || tokens > 0x7fffffffll || head_dim <= 0 || head_dim > 256 || n_cta <= 0 || n_items < 0 ||
      n_items > 0x1fffffffll || (dtype != PSE_F32 && dtype != PSE_BF16) || q.heads <= 0 || k.heads <= 0 ||
      q.heads % k.heads || v.heads != k.heads || out.heads != q.heads)
    return PSE_EINVAL;
  if (tokens == 0 || n_items == 0) return PSE_OK;
  if (!q.data || !k.data || !v.data || !out.data || !plan || reinterpret_cast<uintptr_t>(plan) % 16) return PSE_EINVAL;
  prompt::Args a{};
  a.q = (const char*)q.data;
  a.k = (const char*)k.data;
  a.v = (const char*)v.data;
  a.out = (char*)out.data;
  a.q_tok = q.tok_stride;
  a.q_head = q.head_stride;
  a.k_tok = k.tok_stride;
  a.k_head = k.head_stride;
  a.v_tok = v.tok_stride;
  a.v_head = v.head_stride;
  a.o_tok = out.tok_stride;
  a.o_head = out.head_stride;
  a.tokens = tokens;
  a.q_heads = q.heads;
  a.kv_heads = k.heads;
  a.group = q.heads / k.heads;
  a.hd = head_dim;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.plan = plan;
  a.n_cta = n_cta;
  a.n_items = (int)n_items;
  a.status = status;
  return dtype == PSE_BF16 ? prompt::simt_attention<__nv_bfloat16>(a, (cudaStream_t)stream)
                           : prompt::simt_attention<float>(a, (cudaStream_t)stream);
}
