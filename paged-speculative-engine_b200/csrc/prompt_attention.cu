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
// operations in every call.  (The CUDA-core kernel has a block per 64 rows of an
// item instead; its blocks start in the list's order, one CTA's items after the
// other's, not the longest first.)
#include <algorithm>
#include <atomic>
#include <queue>
#include <vector>

#include "attention_tile.cuh"
#include "simt_attention.cuh"
#include "tmap_cache.h"

namespace pse {

namespace t5 {
namespace {
std::atomic<uint32_t> g_wait_tries{kSpinLimit};
}
uint32_t wait_tries() { return g_wait_tries.load(std::memory_order_relaxed); }
}  // namespace t5

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
  bool out_vec;  // output rows are 16-byte aligned
  uint32_t wait_tries;  // of the products
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
  // rows (token, group head) of the item, token-major, from r0; token t of the
  // prompt's is it.z + row / group
  const int r0 = (int)(blockIdx.x % subs) * 64;
  const int nr = min(64, min(len - it.z, 2 * tile_tokens(a.group)) * a.group - r0);
  if (nr <= 0) return;
  const int first = it.z + r0 / a.group, last = it.z + (r0 + nr - 1) / a.group;  // its tokens
  simt::Tile<4, NC> t;
  t.init(smem, a.hd);
  t.reset();
  auto vec = [&](const char* p, int64_t tok, int64_t head) {
    return reinterpret_cast<uintptr_t>(p) % (4 * sizeof(T)) == 0 && tok % 4 == 0 && head % 4 == 0;
  };
  const T* q = reinterpret_cast<const T*>(a.q);
  const T* k = reinterpret_cast<const T*>(a.k) + hk * a.k_head;
  const T* v = reinterpret_cast<const T*>(a.v) + hk * a.v_head;
  t.template fill_q<T>(
      [&](int r) -> const T* {
        if (r >= nr) return nullptr;
        const int w = (r0 + r) / a.group;
        return q + (int64_t)(tok0 + it.z + w) * a.q_tok + (int64_t)(hk * a.group + (r0 + r - w * a.group)) * a.q_head;
      },
      vec(a.q, a.q_tok, a.q_head), a.scale_log2);
  int token[4];  // of this thread's rows
#pragma unroll
  for (int i = 0; i < 4; ++i) token[i] = it.z + (r0 + t.ty * 4 + i) / a.group;
  const bool kvec = vec(a.k, a.k_tok, a.k_head), vvec = vec(a.v, a.v_tok, a.v_head);
#pragma unroll 1
  for (int k0 = 0; k0 <= last; k0 += simt::BK) {
    __syncthreads();
    t.template fill_kv<T>(
        [&](int r, const T*& ks, const T*& vs) {
          if (k0 + r > last) return;
          ks = k + (int64_t)(tok0 + k0 + r) * a.k_tok;
          vs = v + (int64_t)(tok0 + k0 + r) * a.v_tok;
        },
        kvec, vvec);
    __syncthreads();
    t.step(k0 + simt::BK > first + 1, [&](int i) -> uint64_t {
      const int n = token[i] + 1 - k0;  // keys of the tile up to its own
      return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1;
    });
  }
  T* out = reinterpret_cast<T*>(a.out);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float L = t.row_sum(i);
    const int r = t.ty * 4 + i;
    if (r >= nr) continue;
    T* dst = out + (int64_t)(tok0 + token[i]) * a.o_tok +
             (int64_t)(hk * a.group + (r0 + r - (token[i] - it.z) * a.group)) * a.o_head;
    // a sum of zero (every score -inf) gives zero
    const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int d = 4 * (t.tx + 16 * c);
      float4 x = t.out(i, c);
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

// ---------------------------------------------------------------- tensor cores
// bf16, head_dim 64 or 128.  A CTA per multiprocessor works through its list of
// items.  A query tile is 128 rows, (token, group head) token-major; an item's
// two tiles are two streams that share every 128-key K/V tile:
//   warps 0-3, 4-7  the softmax of stream 0 and 1, a thread per row
//                   (attention_tile.cuh), and the item's output
//   warp 8          TMA: K and V tiles through a ring of slots
//   warp 9          the products: S = Q K^T into tensor memory, O += P V with
//                   P there (over S's columns), V MN-major
//   warp 10         looks through V tiles that some row must not see in whole
//   warp 11         TMA: Q tiles, so that the ring runs on into the next item
// While a stream's softmax runs, the tensor cores work on the other stream.
//
// Measured: three prompts of 5003 to 8192 tokens, 32 + 8 heads of 128: 900 us in
// bursts of 20 calls at full clock, 1200 TFLOP/s of the 1660 that a large matrix
// product reaches so; 1048 us and 1030 TFLOP/s of 1370 in a loop of calls, where the
// power cap holds the clock.  What is lost are the hand-overs between the softmax
// warps and the products (each some 200 clocks of a tile's 2800) and the work beyond
// the diagonal.  Heads of 64 need twice the exponentials per product: 2048 token
// prompts 640 TFLOP/s (600 in a loop), the exponential pipe 61% busy.  24 prompts of
// 17 to 1500 tokens, heads of 64, take 71 us: 8 or 9 items to a CTA with 31 us of
// exponentials, the rest hand-overs and items' beginnings and ends (an item's queries
// are loaded when the scores of the item before have retired, and its first softmax
// waits for them).  One prompt of 37 tokens 5.1 us, all of it latency.
// Tried and slower: a third of the exponentials by a polynomial on the FMA units,
// 96 + 32 keys instead of 64 + 64 to a hand-over, a warp per stream for the products,
// weights apart from the scores.
//
// A hidden key has weight zero, but 0 x inf is NaN in a product, and a tile at
// the causal edge or the prompt's end holds V rows of later tokens or of the
// next prompt.  Warp 10 zeroes the infinities and NaN of such a tile before the
// product sees it and marks the tile; at the item's end a row adds the marked
// tiles' non-finite values of the keys it does see.
using namespace t5;

constexpr int kTcThreads = 384;
constexpr int kHalfBytes = 128 * 128;  // 64 columns of a 128-row tile
constexpr int kGuards = 8;             // barriers of tiles on their way through warp 10
constexpr uint32_t kColS = 0, kColO = 256;

template <int HD>
__host__ __device__ constexpr int n_slots() { return HD == 128 ? 5 : 8; }

template <int HD>
constexpr size_t tc_smem_bytes() {
  return 1024 + (size_t)2 * 128 * HD * 2 + (size_t)n_slots<HD>() * 128 * HD * 2 + 512;
}

struct TcItem {
  int tok0, len, w0, hk;
  int n[2], n_max;
  int guard0;  // first tile that its first row does not see in whole
};

__device__ __forceinline__ TcItem decode(const Args& a, int e, int tpt) {
  const int4 x = __ldg(reinterpret_cast<const int4*>(a.plan + plan_items_at(a.n_cta)) + e);
  TcItem it;
  it.tok0 = x.x;
  it.len = x.y;
  it.w0 = x.z;
  it.hk = x.w;
  const bool ok = it.tok0 >= 0 && it.len >= 0 && it.w0 >= 0 && (int64_t)it.tok0 + it.len <= a.tokens && it.hk >= 0 &&
                  it.hk < a.kv_heads;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const int first = it.w0 + s * tpt;
    it.n[s] = ok && first < it.len ? (min(first + tpt, it.len) + 127) >> 7 : 0;
  }
  it.n_max = max(it.n[0], it.n[1]);
  it.guard0 = (it.w0 + 1) >> 7;
  return it;
}

template <int HD>
__global__ void __launch_bounds__(kTcThreads, 1)
    prompt_tc_kernel(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk,
                     const __grid_constant__ CUtensorMap tmv, const Args a) {
  constexpr int NS = n_slots<HD>();
  constexpr int kTileBytes = 128 * HD * 2, kHalves = HD / 64;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* q_s = smem;                     // [2 streams][128 x HD]
  uint8_t* ring = q_s + 2 * kTileBytes;    // [NS][128 x HD]: K and V tiles in turn
  uint64_t* slot_full = reinterpret_cast<uint64_t*>(ring + NS * kTileBytes);
  uint64_t* slot_empty = slot_full + NS;
  uint64_t* guard_full = slot_empty + NS;  // [kGuards] a guarded V tile landed
  uint64_t* q_full = guard_full + kGuards;
  uint64_t* q_empty = q_full + 1;
  uint64_t* s_full = q_empty + 1;          // [2] a stream's scores stand in tensor memory
  uint64_t* p_half = s_full + 2;           // [2][2] half of a stream's weights stand there
  uint64_t* o_full = p_half + 4;           // [2] a stream's last product of the item retired
  uint64_t* o_empty = o_full + 2;          // [2] its output has been read
  uint64_t* final_bar = o_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(final_bar + 1);
  int* abort_flag = reinterpret_cast<int*>(tmem_slot + 1);
  int* poison = abort_flag + 1;            // [kGuards] items' marked tiles, bit j: tile guard0 + j
  int* last_bar = poison + kGuards;        // [NS + 1] per slot (and Q): barrier and parity of its last copy
  const Waits waits{abort_flag, kSpinLimit};

  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // uniform
  if (tid == 0) {
    prefetch_map(&tmq);
    prefetch_map(&tmk);
    prefetch_map(&tmv);
    for (int i = 0; i < NS; ++i) {
      mbar_init(&slot_full[i], 1);
      mbar_init(&slot_empty[i], 1);
    }
    for (int i = 0; i < kGuards; ++i) mbar_init(&guard_full[i], 1);
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&p_half[2 * s], 4);
      mbar_init(&p_half[2 * s + 1], 4);
      mbar_init(&o_full[s], 1);
      mbar_init(&o_empty[s], 4);
    }
    mbar_init(final_bar, 1);
    *abort_flag = 0;
    for (int i = 0; i <= NS; ++i) last_bar[i] = -1;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(su32(tmem_slot)), "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_trigger();
  const int tpt = tile_tokens(a.group);
  const int e0 = __ldg(a.plan + blockIdx.x), e1 = min(__ldg(a.plan + blockIdx.x + 1), a.n_items);

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    if (warp == 8) {
      // -------------------------------------------------------------- copies
      if (lane == 0) {
        int c = 0, g = 0;
        bool run = true;
        auto load = [&](const CUtensorMap* map, int hk, int tok, bool guarded) -> bool {
          const int s = c % NS;
          if (!mbar_wait(&slot_empty[s], ((c / NS) & 1) ^ 1, waits)) return false;
          uint64_t* bar = guarded ? &guard_full[g % kGuards] : &slot_full[s];
          last_bar[s] = guarded ? (NS + g % kGuards) * 2 + ((g / kGuards) & 1) : s * 2 + ((c / NS) & 1);
          mbar_expect_tx(bar, kTileBytes);
#pragma unroll
          for (int h = 0; h < kHalves; ++h)
            tma_load_3d(ring + s * kTileBytes + h * kHalfBytes, map, h * 64, hk, tok, bar);
          ++c;
          if (guarded) ++g;
          return true;
        };
#pragma unroll 1
        for (int e = e0; run && e < e1; ++e) {
          const TcItem it = decode(a, e, tpt);
          if (it.n_max == 0) continue;
#pragma unroll 1
          for (int j = 0; run && j < it.n_max; ++j)
            run = load(&tmk, it.hk, it.tok0 + j * 128, false) && load(&tmv, it.hk, it.tok0 + j * 128, j >= it.guard0);
        }
      }
    } else if (warp == 11) {
      // -------------------------------------------------------------- queries
      if (lane == 0) {
        int nq = 0;
#pragma unroll 1
        for (int e = e0; e < e1; ++e) {
          const TcItem it = decode(a, e, tpt);
          if (it.n_max == 0) continue;
          if (!mbar_wait(q_empty, (nq & 1) ^ 1, waits)) break;
          const int streams = it.n[1] > 0 ? 2 : 1;
          last_bar[NS] = nq & 1;
          mbar_expect_tx(q_full, streams * kHalves * tpt * a.group * 128);
#pragma unroll 1
          for (int s = 0; s < streams; ++s)
#pragma unroll 1
            for (int h = 0; h < kHalves; ++h)
              tma_load_3d(q_s + s * kTileBytes + h * kHalfBytes, &tmq, h * 64, it.hk * a.group,
                          it.tok0 + it.w0 + s * tpt, q_full);
          ++nq;
        }
      }
    } else if (warp == 9) {
      // -------------------------------------------------------------- products
      const uint32_t el = elect_one();
      const Waits tries{abort_flag, a.wait_tries};
      const uint32_t full0 = su32(slot_full), ring0 = su32(ring), q0 = su32(q_s);
      const uint32_t part0 = su32(p_half);
      int slot = 0;
      uint32_t fill = 0;
      uint32_t parts = 0, outs = 3;
      uint32_t nq = 0;
      bool run = true;
      auto next_slot = [&](int& i, uint32_t& par) {
        i = slot;
        par = fill;
        if (++slot == NS) {
          slot = 0;
          fill ^= 1;
        }
      };
#pragma unroll 1
      for (int e = e0; run && e < e1; ++e) {
        const TcItem it = decode(a, e, tpt);
        if (it.n_max == 0) continue;
        const int n0 = it.n[0], n1 = it.n[1], n = it.n_max;
        int k, v = 0;
        uint32_t kp, vp = 0;
        next_slot(k, kp);
        run = mbar_wait3_warp(su32(q_full), nq, full0 + 8 * k, kp, full0 + 8 * k, kp, tries);
        nq ^= 1;
        if (!run) break;
        fence_after();
        issue_scores<HD>(el, tmem + kColS, q0, ring0 + k * kTileBytes);
        mma_commit(el, &s_full[0]);
        if (n1 > 0) {
          issue_scores<HD>(el, tmem + kColS + 128, q0 + kTileBytes, ring0 + k * kTileBytes);
          mma_commit(el, &s_full[1]);
        }
        mma_commit(el, &slot_empty[k]);
        if (n == 1) mma_commit(el, q_empty);
#pragma unroll 1
        for (int j = 0; run && j < n; ++j) {
          next_slot(v, vp);
          const bool more = j + 1 < n;
          if (more) next_slot(k, kp);
          const uint32_t vbar = full0 + 8 * v, kbar = more ? full0 + 8 * k : vbar;
          if (!more) kp = vp;
          bool here = false;  // the tile's V and the next K have been awaited
          auto stream = [&](int s, int ns) {
            if (j >= ns || !run) return;
            const uint32_t s_col = tmem + kColS + s * 128, o_col = tmem + kColO + s * 128, part = part0 + 16 * s;
            const uint32_t np = parts >> s & 1u;
            if (j == 0) run = mbar_wait_warp(&o_empty[s], outs >> s & 1u, tries);
            run = run && (here ? mbar_wait_warp(part, np, tries) : mbar_wait3_warp(part, np, vbar, vp, kbar, kp, tries));
            here = true;
            if (!run) return;
            fence_after();
            issue_values<HD>(el, o_col, s_col, ring0 + v * kTileBytes, 0, j == 0);
            run = mbar_wait_warp(part + 8, np, tries);
            if (!run) return;
            fence_after();
            issue_values<HD>(el, o_col, s_col, ring0 + v * kTileBytes, 1, false);
            parts ^= 1u << s;
            if (j + 1 == ns) {
              mma_commit(el, &o_full[s]);
              outs ^= 1u << s;
            } else {
              issue_scores<HD>(el, s_col, q0 + s * kTileBytes, ring0 + k * kTileBytes);
              mma_commit(el, &s_full[s]);
            }
          };
          stream(0, n0);
          stream(1, n1);
          if (!run) break;
          mma_commit(el, &slot_empty[v]);
          if (more) mma_commit(el, &slot_empty[k]);
          if (j + 2 == n) mma_commit(el, q_empty);
        }
        // a stream that has no part in this item holds nothing up above: however
        // many such items follow, its output of an earlier one is read (and that
        // item's word in `poison` with it) before this warp goes on
        if (n1 == 0 && run) run = mbar_wait_warp(&o_empty[1], outs >> 1 & 1u, tries);
      }
      mma_commit(el, final_bar);
    } else if (warp == 10) {
      // -------------------------------------------------------------- guard
      int c = 0, g = 0, items = 0;
      bool run = true;
#pragma unroll 1
      for (int e = e0; run && e < e1; ++e) {
        const TcItem it = decode(a, e, tpt);
        if (it.n_max == 0) continue;
        int marks = 0;
#pragma unroll 1
        for (int j = it.guard0; j < it.n_max; ++j, ++g) {
          if (!mbar_wait_warp(&guard_full[g % kGuards], (g / kGuards) & 1, waits)) {
            run = false;
            break;
          }
          const int s = (c + 2 * j + 1) % NS;
          if (tile::clear_nonfinite(reinterpret_cast<uint4*>(ring + s * kTileBytes), kTileBytes / 16))
            marks |= 1 << (j - it.guard0);
          if (lane == 0) {
            poison[items % kGuards] = marks;
            mbar_arrive(&slot_full[s]);
          }
        }
        c += 2 * it.n_max;
        ++items;
      }
    }
  } else {
    // ---------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int s = warp >> 2, r = tid & 127;
    const uint32_t lane_base = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
    const int rt = r / a.group, rg = r - rt * a.group;
    int nt = 0, items = 0, no = 0;  // tiles, items and outputs of this stream
    bool run = true;
#pragma unroll 1
    for (int e = e0; run && e < e1; ++e) {
      const TcItem it = decode(a, e, tpt);
      if (it.n_max == 0) continue;
      const int item = items++;
      if (it.n[s] == 0) continue;
      const int tok = it.w0 + s * tpt + rt;  // this row's token within its prompt
      const bool valid = rt < tpt && tok < it.len;
      const int lim = valid ? tok + 1 : 0x7fffffff;  // keys [0, lim) are visible
      const bool any_valid = __any_sync(0xffffffffu, valid);
      tile::RowState row;
      row.reset();
#pragma unroll 1
      for (int j = 0; j < it.n[s]; ++j, ++nt) {
        if (!mbar_wait_warp(&s_full[s], nt & 1, waits)) {
          run = false;
          break;
        }
        fence_after();
        if (!any_valid) {
          // no row of this warp is anyone's: its weights may be anything
          if (lane == 0) {
            mbar_arrive(&p_half[2 * s]);
            mbar_arrive(&p_half[2 * s + 1]);
          }
          continue;
        }
        const int left = lim - j * 128;
        const bool masked = __any_sync(0xffffffffu, left < 128);
        uint32_t vis[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int n = left - 32 * x;
          vis[x] = n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u;
        }
        tile::softmax_tile<HD>(lane_base, kColS + s * 128, kColO + s * 128, a.scale_log2, j == 0, masked, vis, row,
                               &p_half[2 * s], &p_half[2 * s + 1]);
      }
      if (!run || !mbar_wait_warp(&o_full[s], no & 1, waits)) break;
      ++no;
      fence_after();
      const int marks = it.guard0 < it.n_max ? poison[item % kGuards] : 0;
      // a row whose weights are all zero (every score -inf) gives zero
      const float inv = row.l == 0.f ? 0.f : 1.f / row.l;
      __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(a.out) + (int64_t)(it.tok0 + tok) * a.o_tok +
                           (int64_t)(it.hk * a.group + rg) * a.o_head;
#pragma unroll 1
      for (int h = 0; h < HD / 32; ++h) {
        uint32_t u[32];
        float* o = reinterpret_cast<float*>(u);
        tmem_ld32(lane_base + kColO + s * 128 + 32 * h, u);
        tmem_wait_ld();
        if (h == HD / 32 - 1) {
          fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&o_empty[s]);
        }
        if (marks && valid) {
          const __nv_bfloat16* v = reinterpret_cast<const __nv_bfloat16*>(a.v) + it.hk * a.v_head + 32 * h;
#pragma unroll 1
          for (int key = it.guard0 * 128; key < lim; ++key) {
            if (!(marks >> ((key >> 7) - it.guard0) & 1)) continue;
#pragma unroll
            for (int x = 0; x < 32; ++x) {
              const float y = __bfloat162float(v[(int64_t)(it.tok0 + key) * a.v_tok + x]);
              if (!isfinite(y)) o[x] += y;
            }
          }
        }
        if (valid) {
          tile::store_row32(dst + 32 * h, o, inv, a.out_vec);
        }
      }
    }
  }

  __syncthreads();
  if (*waits.abort_flag) {
    if (tid == 0 && a.status) atomicOr(a.status, PSE_STATUS_TIMEOUT);
    if (tid == 0) {
      // copies still on their way land before the shared memory goes
      for (int i = 0; i < NS; ++i)
        if (last_bar[i] >= 0) {
          const int b = last_bar[i] >> 1;
          mbar_drain(b < NS ? &slot_full[b] : &guard_full[b - NS], last_bar[i] & 1);
        }
      if (last_bar[NS] >= 0) mbar_drain(q_full, last_bar[NS]);
    }
  }
  if (warp == 9) {
    if (lane == 0) mbar_drain(final_bar, 0);
    __syncwarp();
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
}

Map3Cache g_maps;

bool tc_eligible(const Args& a) {
  return (a.hd == 64 || a.hd == 128) && a.group <= 128 && a.scale_log2 > 0.f &&
         tma_rows(a.q, a.q_tok, a.q_head, a.q_heads, a.hd) && tma_rows(a.k, a.k_tok, a.k_head, a.kv_heads, a.hd) &&
         tma_rows(a.v, a.v_tok, a.v_head, a.kv_heads, a.hd);
}

template <int HD>
int launch_tc(const Args& a, cudaStream_t s) {
  auto kern = prompt_tc_kernel<HD>;
  constexpr size_t smem = tc_smem_bytes<HD>();
  static_assert(smem <= 227 * 1024, "shared memory");
  static const cudaError_t opt = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (opt != cudaSuccess) return (int)opt;
  auto key = [&](const char* p, int64_t tok, int64_t head, int heads, uint32_t b1, uint32_t b2) {
    return Map3Key{reinterpret_cast<uint64_t>(p), (uint64_t)HD, (uint64_t)heads, (uint64_t)a.tokens,
                   (uint64_t)(heads == 1 ? HD : head) * 2, (uint64_t)tok * 2, b1, b2};
  };
  CUtensorMap mq, mk, mv;
  int rc = g_maps.get(key(a.q, a.q_tok, a.q_head, a.q_heads, a.group, tile_tokens(a.group)), PSE_EINVAL, &mq);
  if (rc == 0) rc = g_maps.get(key(a.k, a.k_tok, a.k_head, a.kv_heads, 1, 128), PSE_EINVAL, &mk);
  if (rc == 0) rc = g_maps.get(key(a.v, a.v_tok, a.v_head, a.kv_heads, 1, 128), PSE_EINVAL, &mv);
  if (rc) return rc;
  // with fewer items than CTAs the plan gives them to the first ones
  const int grid = a.n_items < a.n_cta ? a.n_items : a.n_cta;
  const cudaError_t e = launch_pdl(kern, dim3(grid), dim3(kTcThreads), smem, s, mq, mk, mv, a);
  return e == cudaSuccess ? PSE_OK : (int)e;
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

extern "C" int pse_attention_wait_tries(int32_t tries) {
  t5::g_wait_tries.store(tries < 0 ? t5::kSpinLimit : (uint32_t)tries, std::memory_order_relaxed);
  return PSE_OK;
}

extern "C" int pse_prompt_attention(const pse_head_view* views, int64_t tokens, int32_t head_dim, int32_t dtype,
                                    float scale, const int32_t* plan, int32_t n_cta, int64_t n_items, int32_t* status,
                                    void* stream) {
  if (!views) return PSE_EINVAL;
  const pse_head_view &q = views[0], &k = views[1], &v = views[2], &out = views[3];
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
  a.wait_tries = t5::wait_tries();
  a.out_vec = reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && a.o_tok % 8 == 0 && a.o_head % 8 == 0;
  if (dtype == PSE_BF16 && prompt::tc_eligible(a))
    return head_dim == 64 ? prompt::launch_tc<64>(a, (cudaStream_t)stream)
                          : prompt::launch_tc<128>(a, (cudaStream_t)stream);
  return dtype == PSE_BF16 ? prompt::simt_attention<__nv_bfloat16>(a, (cudaStream_t)stream)
                           : prompt::simt_attention<float>(a, (cudaStream_t)stream);
}
