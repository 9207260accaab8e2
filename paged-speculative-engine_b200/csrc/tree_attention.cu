// Attention of drafted token trees over the paged cache: query node n of a row
// attends to the row's whole context and to the nodes that its mask names
// (engine/model.py:99-116 with the mask of a token tree; the reference lists
// trees as future work, README.md:210-214).  Any tree per row: the masks are
// bits, one word per 64 nodes, and rows may hold different numbers of nodes.
//
// The context's K/V is read from HBM once per request, which bounds the call
// until a K/V head has about 256 query rows (nodes x group).
#include "simt_attention.cuh"
#include "tree_partition.cuh"

namespace pse {
namespace tree {

constexpr int kMaxCtas = 2 * kNumSMs;
constexpr int kCounterBytes = 4 * 512;

struct Args {
  Rows rows;
  const int32_t* block_table;
  const int32_t* nblocks;
  int max_blocks, block_size, num_blocks;
  const char *k_pool, *v_pool;
  int hd;
  const char* q;
  int64_t q_tok, q_head;
  char* out;
  int64_t o_tok, o_head;
  const int64_t* masks;
  int words;
  int block_nodes;
  float scale_log2;
  int32_t* counters;  // [kMaxCtas], zero between calls
  float* parts;       // [ctas][2][block rows][hd + 2]
  int32_t* status;
};

// Which of its CTA's two partial results a segment writes: the first segment's
// item may be cut at its start, the last one's at its end.
__device__ __forceinline__ float* part(const Args& a, int cta, bool starts_item, int rows) {
  return a.parts + ((int64_t)cta * 2 + (starts_item ? 1 : 0)) * rows * (a.hd + 2);
}

// ---------------------------------------------------------------- CUDA cores
template <typename T, int RPT, int NC>
__global__ void __launch_bounds__(simt::kThreads) tree_simt_kernel(const Args a) {
  extern __shared__ float smem[];
  __shared__ long long tmp[40];
  __shared__ int last;
  constexpr int BQ = 16 * RPT, TILE = simt::BK;
  const Span span = my_span<TILE>(a.rows, a.block_nodes, tmp);
  if ((int)blockIdx.x >= span.ctas) return;
  simt::Tile<RPT, NC> t;
  t.init(smem, a.hd);
  const int group = a.rows.group, hd = a.hd;
  auto aligned = [&](const char* p, int64_t tok, int64_t head) {
    return reinterpret_cast<uintptr_t>(p) % (4 * sizeof(T)) == 0 && tok % 4 == 0 && head % 4 == 0;
  };
  const bool qvec = aligned(a.q, a.q_tok, a.q_head);
  const bool kvec = aligned(a.k_pool, hd, hd), vvec = aligned(a.v_pool, hd, hd);
  Walk<TILE> walk(a.rows, span, a.block_nodes);
  Segment g;
  while (walk.next(g)) {
    // rows of the block: (node, group head), node-major; a group above BQ heads
    // takes its rows BQ at a time
    const int node0 = g.block * a.block_nodes;
    const int nr = min(a.block_nodes, g.r.nodes - node0) * group;
    const int32_t* table = a.block_table + (int64_t)max(g.r.slot, 0) * a.max_blocks;
    const int held = g.r.slot >= 0 ? min(a.nblocks[g.r.slot], a.max_blocks) : 0;
    t.reset();
    __syncthreads();
    t.template fill<T>(
        t.q, BQ,
        [&](int r) -> const T* {
          if (r >= nr) return nullptr;
          return reinterpret_cast<const T*>(a.q) + (int64_t)(g.r.n0 + node0 + r / group) * a.q_tok +
                 (int64_t)(g.hk * group + r % group) * a.q_head;
        },
        qvec, a.scale_log2);
    const int keys = g.r.ctx + g.r.nodes;
    for (int tile = g.t0; tile < g.t1; ++tile) {
      const int k0 = tile * TILE;
      __syncthreads();
      auto at = [&](const char* pool, int r) -> const T* {
        const int key = k0 + r;
        if (key >= keys) return nullptr;
        const int bi = key / a.block_size;
        if (bi >= held) return nullptr;
        const int blk = table[bi];
        if (blk < 0 || blk >= a.num_blocks) return nullptr;
        return reinterpret_cast<const T*>(pool) +
               (((int64_t)blk * a.rows.kv_heads + g.hk) * a.block_size + key % a.block_size) * hd;
      };
      t.template fill<T>(t.k, TILE, [&](int r) { return at(a.k_pool, r); }, kvec, 1.f);
      t.template fill<T>(t.v, TILE, [&](int r) { return at(a.v_pool, r); }, vvec, 1.f);
      __syncthreads();
      t.step(k0 + TILE > g.r.ctx || g.r.slot < 0, [&](int r, int key) {
        if (r >= nr || k0 + key >= keys) return false;
        const int64_t* m = a.masks + (int64_t)(g.r.n0 + node0 + r / group) * a.words;
        return (visible32(m, a.words, g.r, k0 + (key & ~31)) >> (key & 31) & 1u) != 0u;
      });
    }
    T* out = reinterpret_cast<T*>(a.out);
    auto out_row = [&](int r) {
      return out + (int64_t)(g.r.n0 + node0 + r / group) * a.o_tok + (int64_t)(g.hk * group + r % group) * a.o_head;
    };
    const bool whole = g.t0 == 0 && g.t1 == g.tiles;
    float* mine = part(a, blockIdx.x, g.t0 == 0, BQ);
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      const float L = t.row_sum(i);
      const int r = t.ty * RPT + i;
      if (r >= nr) continue;
      const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int d = 4 * (t.tx + 16 * c);
        if (d >= hd) continue;
        float4 x = t.o[i][c];
        if (whole) {
          x.x *= inv;
          x.y *= inv;
          x.z *= inv;
          x.w *= inv;
          simt::store4(out_row(r) + d, hd - d, x);
        } else {
          simt::store4(mine + (int64_t)r * (hd + 2) + d, hd - d, x);
        }
      }
      if (!whole && t.tx == 0) {
        mine[(int64_t)r * (hd + 2) + hd] = t.m[i];
        mine[(int64_t)r * (hd + 2) + hd + 1] = L;
      }
    }
    if (whole) continue;
    const int c1 = owner(span, g.first), c2 = owner(span, g.first + g.tiles - 1);
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last = atomicAdd(a.counters + c1, 1) == c2 - c1;
    __syncthreads();
    if (!last) continue;
    __threadfence();
    if (threadIdx.x == 0) a.counters[c1] = 0;
    for (int e = threadIdx.x; e < nr * hd; e += simt::kThreads) {
      const int r = e / hd, d = e - r * hd;
      float M = -INFINITY;
      for (int c = c1; c <= c2; ++c)
        M = fmaxf(M, __ldcg(part(a, c, c == c1, BQ) + (int64_t)r * (hd + 2) + hd));
      const float ms = M == -INFINITY ? 0.f : M;
      float L = 0.f, x = 0.f;
      for (int c = c1; c <= c2; ++c) {
        const float* p = part(a, c, c == c1, BQ) + (int64_t)r * (hd + 2);
        const float f = exp2f(__ldcg(p + hd) - ms);
        if (f != 0.f) {
          L += __ldcg(p + hd + 1) * f;
          x += __ldcg(p + d) * f;
        }
      }
      out_row(r)[d] = from_f32<T>(L == 0.f ? 0.f : x / L);
    }
    __syncthreads();
  }
}

int simt_rows(int rows) { return rows <= 16 ? 1 : 4; }

template <typename T, int RPT, int NC>
int launch_simt(const Args& a, int grid, cudaStream_t s) {
  auto kern = tree_simt_kernel<T, RPT, NC>;
  const size_t smem = simt::smem_floats<RPT>(a.hd) * sizeof(float);
  static const cudaError_t opt = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                      (int)(simt::smem_floats<RPT>(64 * NC) * sizeof(float)));
  if (opt != cudaSuccess) return (int)opt;
  kern<<<grid, simt::kThreads, smem, s>>>(a);
  PSE_LAUNCH_CHECK();
  return PSE_OK;
}

template <typename T, int RPT>
int simt_nc(const Args& a, int grid, cudaStream_t s) {
  if (a.hd <= 64) return launch_simt<T, RPT, 1>(a, grid, s);
  if (a.hd <= 128) return launch_simt<T, RPT, 2>(a, grid, s);
  return launch_simt<T, RPT, 4>(a, grid, s);
}

template <typename T>
int simt_attention(Args& a, int max_nodes, cudaStream_t s) {
  const int rpt = simt_rows(max_nodes * a.rows.group);
  a.block_nodes = 16 * rpt / a.rows.group;
  return rpt == 1 ? simt_nc<T, 1>(a, kMaxCtas, s) : simt_nc<T, 4>(a, kMaxCtas, s);
}

// Node ancestors: bit m of node n's mask for m = n and every node on the way
// to the root; depth = edges to the root context's first node.
__global__ void masks_kernel(const int32_t* parents, const int32_t* node_off, int rows, int n_nodes, int words,
                             unsigned long long* masks, int32_t* depths) {
  const int i = blockIdx.x;
  const int n0 = node_off[i], n = node_off[i + 1] - n0;
  if (n0 < 0 || n < 0 || (int64_t)n0 + n > n_nodes) return;
  for (int j = threadIdx.x; j < n; j += blockDim.x) {
    unsigned long long* m = masks + (int64_t)(n0 + j) * words;
    for (int w = 0; w < words; ++w) m[w] = 0ull;
    int depth = -1;
    // parents precede their children, so the walk falls strictly and ends
    for (int at = j; at >= 0 && at < 64 * words;) {
      m[at >> 6] |= 1ull << (at & 63);
      ++depth;
      const int up = parents[n0 + at];
      if (up >= at) break;
      at = up;
    }
    depths[n0 + j] = depth;
  }
}

}  // namespace tree
}  // namespace pse

using namespace pse;

extern "C" int pse_tree_masks(const int32_t* parents, const int32_t* node_off, int32_t rows, int32_t n_nodes,
                              int32_t words, int64_t* masks, int32_t* depths, void* stream) {
  if (rows < 0 || n_nodes < 0 || words <= 0) return PSE_EINVAL;
  if (rows == 0 || n_nodes == 0) return PSE_OK;
  if (!parents || !node_off || !masks || !depths) return PSE_EINVAL;
  tree::masks_kernel<<<rows, 64, 0, (cudaStream_t)stream>>>(parents, node_off, rows, n_nodes, words,
                                                            (unsigned long long*)masks, depths);
  PSE_LAUNCH_CHECK();
  return PSE_OK;
}

extern "C" size_t pse_token_tree_workspace(int32_t head_dim) {
  if (head_dim <= 0) return 0;
  // two partial results of up to 64 rows per CTA
  return (size_t)tree::kCounterBytes + (size_t)tree::kMaxCtas * 2 * 64 * (head_dim + 2) * 4;
}

extern "C" int pse_token_tree_attention(pse_block_state st, pse_kv_layer kv, pse_head_view q, pse_head_view out,
                                        const int32_t* slots, const int32_t* ctx, const int32_t* node_off,
                                        int32_t rows, int32_t n_nodes, int32_t max_nodes, const int64_t* masks,
                                        int32_t words, float scale, void* workspace, size_t workspace_bytes,
                                        void* stream) {
  if (!st.block_table || !st.nblocks || !st.status || st.block_size <= 0 || st.max_blocks <= 0 || st.num_slots <= 0 ||
      !kv.k_pool || !kv.v_pool || kv.kv_heads <= 0 || kv.head_dim <= 0 || kv.head_dim > 256 || rows < 0 ||
      n_nodes < 0 || max_nodes < 0 || words <= 0 || max_nodes > 64ll * words || q.heads <= 0 ||
      q.heads % kv.kv_heads || out.heads != q.heads || q.heads / kv.kv_heads > 64)
    return PSE_EINVAL;
  if (kv.dtype != PSE_F32 && kv.dtype != PSE_BF16) return PSE_EINVAL;
  if (rows == 0 || n_nodes == 0 || max_nodes == 0) return PSE_OK;
  if (!q.data || !out.data || !slots || !ctx || !node_off || !masks || !workspace ||
      reinterpret_cast<uintptr_t>(workspace) % 16)
    return PSE_EINVAL;
  if (workspace_bytes < pse_token_tree_workspace(kv.head_dim)) return PSE_EWORKSPACE;
  tree::Args a{};
  a.rows.slots = slots;
  a.rows.ctx = ctx;
  a.rows.node_off = node_off;
  a.rows.rows = rows;
  a.rows.num_slots = st.num_slots;
  a.rows.n_nodes = n_nodes;
  a.rows.kv_heads = kv.kv_heads;
  a.rows.group = q.heads / kv.kv_heads;
  a.rows.max_keys = (int64_t)st.max_blocks * st.block_size;
  if (a.rows.max_keys > 0x7fffff00ll) a.rows.max_keys = 0x7fffff00ll;
  a.block_table = st.block_table;
  a.nblocks = st.nblocks;
  a.max_blocks = st.max_blocks;
  a.block_size = st.block_size;
  a.num_blocks = st.num_blocks;
  a.k_pool = (const char*)kv.k_pool;
  a.v_pool = (const char*)kv.v_pool;
  a.hd = kv.head_dim;
  a.q = (const char*)q.data;
  a.q_tok = q.tok_stride;
  a.q_head = q.head_stride;
  a.out = (char*)out.data;
  a.o_tok = out.tok_stride;
  a.o_head = out.head_stride;
  a.masks = masks;
  a.words = words;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.counters = (int32_t*)workspace;
  a.parts = (float*)((char*)workspace + tree::kCounterBytes);
  a.status = st.status;
  return kv.dtype == PSE_BF16 ? tree::simt_attention<__nv_bfloat16>(a, max_nodes, (cudaStream_t)stream)
                              : tree::simt_attention<float>(a, max_nodes, (cudaStream_t)stream);
}
