// Attention of drafted token trees over the paged cache: query node n of a row
// attends to the row's whole context and to the nodes that its mask names
// (engine/model.py:99-116 with the mask of a token tree; the reference lists
// trees as future work, README.md:210-214).  Any tree per row: the masks are
// bits, one word per 64 nodes, and rows may hold different numbers of nodes.
//
// The context's K/V is read from HBM once per request, which bounds the call
// until a K/V head has about 256 query rows (nodes x group).  Measured, in bursts of
// 20 calls (and in a loop of calls, where the power cap holds the clock): 16
// requests of 16384 tokens, 8 K/V heads of 128: 8 nodes (32 rows) 177 us (201), 6.1
// TB/s, 93% of a copy's rate; 32 nodes (128 rows) 194 us (223); 64 nodes (256 rows)
// 271 us (326), 1014 TFLOP/s, the products and the softmax in turn.  At head_dim 64 a
// row of scores costs twice as many exponentials for its bytes, and the softmax
// warps bound the call: 64 requests of 2048 tokens with 26 nodes 85 us (89), 3.4
// TB/s; with 6 nodes 68 us (72), 4.0 TB/s.  A small tree (8 nodes, 300 tokens) takes
// 11 us, of which 5 pass before the first scores stand (launch, the split of the
// work, the first loads) and 3 in the join: the split leaves no item whole there.
#include "attention_tile.cuh"
#include "simt_attention.cuh"
#include "tmap_cache.h"
#include "tree_partition.cuh"

namespace pse {
namespace tree {

struct Cut;
constexpr int kMaxWorkers = 2 * kNumSMs;
constexpr size_t kCutBytes = 8192;  // a Cut per worker

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
  Cut* cuts;     // [workers]
  float* parts;  // [workers][2][part_rows * part_width(hd)]
  int part_rows;
  int32_t* status;
  bool out_vec;  // output rows are 16-byte aligned
  uint32_t wait_tries;  // of the products
};

// Partial results of cut items: per worker two blocks of `part_rows` rows, first
// the output four columns at a time (a float4 of every row, then the next four
// columns: threads with a row each write and read them side by side), then a
// (maximum, sum) per row.  A worker's first segment, if it begins inside an item,
// uses the first block; a segment that begins an item and does not end it,
// necessarily the worker's last, uses the second.
__host__ __device__ constexpr int part_width(int hd) { return (hd + 3) / 4 * 4 + 2; }  // floats per row
__device__ __forceinline__ float* part(const Args& a, int cta, bool starts_item) {
  return a.parts + ((int64_t)cta * 2 + (starts_item ? 1 : 0)) * a.part_rows * part_width(a.hd);
}
__device__ __forceinline__ float4* part_cols(const Args& a, float* block, int r, int col) {  // col: a multiple of 4
  return reinterpret_cast<float4*>(block) + col / 4 * a.part_rows + r;
}
__device__ __forceinline__ float2* part_stats(const Args& a, float* block, int r) {
  return reinterpret_cast<float2*>(block + a.part_rows * (part_width(a.hd) - 2)) + r;
}

// What the join needs of the item that worker c begins and does not end.
struct Cut {
  int last;    // the item's last worker (-1: worker c cuts nothing)
  int node0;   // its first query node
  int nodes;   // and their number
  int hk;
};

// A warp per 32 rows and 8 columns of a cut item, a row per lane: the parts are
// summed in the order of their workers.  Every block reads all cuts and numbers
// their tasks, so these are spread over the whole GPU whatever was cut where.
// (A warp per row with its lanes over the columns, the parts row by row, took 10 us
// more where 64 rows-per-head trees of 2048 tokens leave 31 thousand cut rows: the
// parts' writer, a thread per row, then writes 16 bytes to each of 32 lines.)
constexpr int kJoinThreads = 512;

template <typename T>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const Args a, int workers, int tile_rows, int tile_pitch) {
  __shared__ int scan_tmp[33];
  __shared__ int first_chunk[kJoinThreads];  // chunks of 32 rows of the cuts before
  __shared__ int4 cuts[kJoinThreads];
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, lane = tid & 31, group = a.rows.group, hd = a.hd;
  int4 mine = make_int4(-1, 0, 0, 0);
  if (tid < workers) mine = __ldcg(reinterpret_cast<const int4*>(a.cuts + tid));
  int total;
  const int before = block_exclusive_scan(mine.x >= 0 ? ceil_div(mine.z * group, 32) : 0, scan_tmp, &total);
  first_chunk[tid] = before;
  cuts[tid] = mine;
  __syncthreads();
  const int warps = gridDim.x * (kJoinThreads / 32), col_groups = ceil_div(hd, 8);
#pragma unroll 1
  for (int task = blockIdx.x * (kJoinThreads / 32) + (tid >> 5); task < total * col_groups; task += warps) {
    const int chunk = task / col_groups, col = 8 * (task - chunk * col_groups);
    // the last cut whose chunks begin at or before this one (cuts without rows
    // share their successor's beginning)
    int c1 = 0;
#pragma unroll
    for (int step = kJoinThreads / 2; step > 0; step >>= 1)
      if (first_chunk[c1 + step] <= chunk) c1 += step;
    const int4 cut = cuts[c1];
    const int n = cut.x - c1 + 1;
    const int row = 32 * (chunk - first_chunk[c1]) + lane;
    if (row >= cut.z * group) continue;
    const int r = row / tile_rows * tile_pitch + row % tile_rows;
    const bool second = col + 4 < hd;
    // worker c1 holds the item's beginning in its second block, the others theirs
    // in their first
    auto block = [&](int i) { return part(a, c1 + i, i == 0); };
    // four parts on their way at a time
    float2 ml[4];
    float4 x[4], y[4];
    auto load = [&](int i0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ml[i] = make_float2(-INFINITY, 0.f);
        x[i] = y[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i0 + i >= n) continue;
        float* p = block(i0 + i);
        ml[i] = __ldcg(part_stats(a, p, r));
        x[i] = __ldcg(part_cols(a, p, r, col));
        if (second) y[i] = __ldcg(part_cols(a, p, r, col + 4));
      }
    };
    load(0);
    float M = fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x));
#pragma unroll 1
    for (int i = 4; i < n; ++i) M = fmaxf(M, __ldcg(part_stats(a, block(i), r)).x);
    const float ms = M == -INFINITY ? 0.f : M;
    float L = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int i0 = 0; i0 < n; i0 += 4) {
      if (i0 > 0) load(i0);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i0 + i >= n) break;
        const float f = exp2f(ml[i].x - ms);
        // (a part that saw nothing is all zeros; an infinity or NaN that a row sees
        // reaches it from the smallest part too)
        L += ml[i].y * f;
        const float v[8] = {x[i].x, x[i].y, x[i].z, x[i].w, y[i].x, y[i].y, y[i].z, y[i].w};
#pragma unroll
        for (int d = 0; d < 8; ++d) acc[d] = fmaf(v[d], f, acc[d]);
      }
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    T* dst = reinterpret_cast<T*>(a.out) + (int64_t)(cut.y + row / group) * a.o_tok +
             (int64_t)(cut.w * group + row % group) * a.o_head + col;
#pragma unroll
    for (int d = 0; d < 8; ++d) acc[d] *= inv;
    if (sizeof(T) == 2 && a.out_vec && col + 8 <= hd) {
      *reinterpret_cast<uint4*>(dst) = make_uint4(t5::pack_bf16(acc[0], acc[1]), t5::pack_bf16(acc[2], acc[3]),
                                                  t5::pack_bf16(acc[4], acc[5]), t5::pack_bf16(acc[6], acc[7]));
    } else {
#pragma unroll
      for (int d = 0; d < 8; ++d)
        if (col + d < hd) dst[d] = from_f32<T>(acc[d]);
    }
  }
}

template <typename T>
int launch_join(const Args& a, int workers, int tile_rows, int tile_pitch, cudaStream_t s) {
  static_assert(kMaxWorkers <= kJoinThreads, "a thread per cut");
  const cudaError_t e =
      launch_pdl(join_kernel<T>, dim3(2 * kNumSMs), dim3(kJoinThreads), 0, s, a, workers, tile_rows, tile_pitch);
  return e == cudaSuccess ? PSE_OK : (int)e;
}

// ---------------------------------------------------------------- CUDA cores
template <typename T, int RPT, int NC>
__global__ void __launch_bounds__(simt::kThreads) tree_simt_kernel(const Args a) {
  extern __shared__ float smem[];
  __shared__ int tmp[40];
  constexpr int TILE = simt::BK;
  pdl_trigger();
  Span span;
  const Split split = my_span<TILE>(a.rows, a.block_nodes, tmp, span);
  Cut cut{-1, 0, 0, 0};
  simt::Tile<RPT, NC> t;
  t.init(smem, a.hd);
  const int group = a.rows.group, hd = a.hd;
  auto aligned = [&](const char* p, int64_t tok, int64_t head) {
    return reinterpret_cast<uintptr_t>(p) % (4 * sizeof(T)) == 0 && tok % 4 == 0 && head % 4 == 0;
  };
  const bool qvec = aligned(a.q, a.q_tok, a.q_head);
  const bool kvec = aligned(a.k_pool, hd, hd), vvec = aligned(a.v_pool, hd, hd);
  int rt[RPT];  // the node of each of this thread's rows
#pragma unroll
  for (int i = 0; i < RPT; ++i) rt[i] = (t.ty * RPT + i) / group;
  Walk<TILE> walk;
  walk.start(a.rows, span, a.block_nodes);
  Segment g;
  while (walk.next(g)) {
    // rows of the block: (node, group head), node-major
    const int node0 = g.block * a.block_nodes;
    const int nr = min(a.block_nodes, g.r.nodes - node0) * group;
    const int32_t* table = a.block_table + (int64_t)max(g.r.slot, 0) * a.max_blocks;
    const int held = g.r.slot >= 0 ? min(a.nblocks[g.r.slot], a.max_blocks) : 0;
    t.reset();
    __syncthreads();
    t.template fill_q<T>(
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
      t.template fill_kv<T>(
          [&](int r, const T*& ks, const T*& vs) {
            const int key = k0 + r;
            if (key >= keys) return;
            const int bi = key / a.block_size;
            if (bi >= held) return;
            const int blk = __ldg(table + bi);
            if (blk < 0 || blk >= a.num_blocks) return;
            const int64_t at = (((int64_t)blk * a.rows.kv_heads + g.hk) * a.block_size + (key - bi * a.block_size)) * hd;
            ks = reinterpret_cast<const T*>(a.k_pool) + at;
            vs = reinterpret_cast<const T*>(a.v_pool) + at;
          },
          kvec, vvec);
      __syncthreads();
      t.step(k0 + TILE > g.r.ctx || g.r.slot < 0, [&](int i) -> uint64_t {
        if (t.ty * RPT + i >= nr) return 0ull;
        const uint32_t* m = reinterpret_cast<const uint32_t*>(a.masks + (int64_t)(g.r.n0 + node0 + rt[i]) * a.words);
        const auto word = [&](int w) { return __ldg(m + w); };
        const uint32_t lo = visible32(word, a.words, g.r.slot, g.r.ctx, g.r.nodes, k0);
        return lo | (uint64_t)visible32(word, a.words, g.r.slot, g.r.ctx, g.r.nodes, k0 + 32) << 32;
      });
    }
    T* out = reinterpret_cast<T*>(a.out);
    auto out_row = [&](int r) {
      return out + (int64_t)(g.r.n0 + node0 + r / group) * a.o_tok + (int64_t)(g.hk * group + r % group) * a.o_head;
    };
    const bool whole = g.t0 == 0 && g.t1 == g.tiles;
    float* mine = part(a, blockIdx.x, g.t0 == 0);
    if (g.t0 == 0 && !whole)
      cut = Cut{owner(split, g.first + g.tiles - 1), g.r.n0 + node0, min(a.block_nodes, g.r.nodes - node0), g.hk};
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
        float4 x = t.out(i, c);
        if (whole) {
          x.x *= inv;
          x.y *= inv;
          x.z *= inv;
          x.w *= inv;
          simt::store4(out_row(r) + d, hd - d, x);
        } else {
          *part_cols(a, mine, r, d) = x;
        }
      }
      if (!whole && t.tx == 0) *part_stats(a, mine, r) = make_float2(t.m[i], L);
    }
  }
  if (threadIdx.x == 0) *reinterpret_cast<int4*>(a.cuts + blockIdx.x) = make_int4(cut.last, cut.node0, cut.nodes, cut.hk);
}

// Rows per thread: blocks of 16 query rows up to 32, of 64 above.  16 against 64, 8
// requests of 500 tokens and 12 K/V heads: 26 rows 51 and 63 us, 33 rows 70 and 62,
// 48 rows 71 and 64, 63 rows 94 and 69; 16 requests of 2000 tokens and 8 K/V heads: 24
// rows 206 and 218 us, 40 rows 301 and 219, 56 rows 400 and 221, 104 rows 684 and 413.
int simt_rows(int rows, int group) { return rows <= 32 && group <= 16 ? 1 : 4; }

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
  const int rpt = simt_rows(max_nodes * a.rows.group, a.rows.group);
  a.block_nodes = 16 * rpt / a.rows.group;
  a.part_rows = 16 * rpt;
  if (!countable(a.rows, simt::BK, a.block_nodes)) return PSE_EINVAL;
  const int rc = rpt == 1 ? simt_nc<T, 1>(a, kMaxWorkers, s) : simt_nc<T, 4>(a, kMaxWorkers, s);
  return rc == PSE_OK ? launch_join<T>(a, kMaxWorkers, a.part_rows, a.part_rows, s) : rc;
}

// ---------------------------------------------------------------- tensor cores
// bf16 pools, head_dim 64 or 128, pages of 16, 32, 64 or 128 tokens.  A query
// tile is 128 rows, (node, group head) node-major, and has a stream: four softmax
// warps with 256 columns of tensor memory.
//   NQ = 1 (at most 128 rows per K/V head): a CTA has one stream, and a
//          multiprocessor two CTAs, each a worker of its own: while one's softmax
//          runs or its output is written, the other loads and multiplies;
//   NQ = 2: one CTA with two streams, the two query tiles of an item, which share
//          every K/V tile (the second one idles through a block whose last nodes
//          fill one tile).
// Warps (h = 4 NQ):
//   0 .. h - 1  the softmax (attention_tile.cuh), a thread per row, and the output
//   h, h + 4    K, and V pages by TMA into a ring of 128-key slots (a copy takes
//               its warp some 50 clocks to issue, and a tile of 16-token pages is
//               16 copies; two streams leave one warp the time for both)
//   h + 1       the products
//   h + 2       clears V tiles that hold nodes (or what stands after them) of
//               infinities and NaN before the product, as in prompt_attention.cu
//   h + 3       Q tiles, so that the ring runs on into the next segment, and what
//               the softmax and product warps have to know of it (Seg)
// NQ = 1 keeps its softmax in rolled loops (softmax_tile_small).  Slower, 64 trees
// of 26 nodes over 2048 tokens (85 us): scores of 64 keys in two buffers, two tiles
// ahead of the values (89); halves of 64 scores in registers, 8 warps (91).
using namespace t5;

constexpr int kHalfBytes = 128 * 128;
constexpr int kGuards = 8;

template <int NQ>
__host__ __device__ constexpr int n_threads() { return 32 * (4 * NQ + (NQ == 1 ? 5 : 4)); }
// two CTAs share a multiprocessor's 227 KB when NQ = 1: at head_dim 128 a K and a
// V tile each, whose loads still pass behind the other tile's softmax
template <int HD, int NQ>
__host__ __device__ constexpr int n_slots() { return HD == 128 ? (NQ == 1 ? 2 : 5) : (NQ == 1 ? 5 : 10); }

template <int HD, int NQ>
constexpr size_t tc_smem_bytes() {
  return 1024 + (size_t)(NQ + n_slots<HD, NQ>()) * 128 * HD * 2 + 512;
}

// A segment as the softmax and product warps read it from shared memory when
// they need it: held in registers it would not fit beside a row of scores.
struct Seg {
  int q0, nodes;           // the block's first query, and its nodes
  int hk, slot, ctx, row_nodes;
  int t0, t1, tiles, first;
  int g0;                  // tiles from here on hold keys that some node may not see
};
constexpr int kSegs = 4;

template <int HD, int NQ>
__global__ void __launch_bounds__(n_threads<NQ>(), NQ == 1 ? 2 : 1)
    tree_tc_kernel(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk,
                   const __grid_constant__ CUtensorMap tmv, const Args a) {
  constexpr int NS = n_slots<HD, NQ>(), kHelp = 4 * NQ;
  constexpr int kTileBytes = 128 * HD * 2, kHalves = HD / 64;
  constexpr uint32_t kColO = 128 * NQ, kTmem = 256 * NQ;
  extern __shared__ uint8_t smem_raw[];
  __shared__ int span_tmp[40];
  __shared__ Seg segs[kSegs];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* q_s = smem;                      // [NQ][128 x HD]
  uint8_t* ring = q_s + NQ * kTileBytes;    // [NS][128 x HD]: K and V tiles in turn
  uint64_t* slot_full = reinterpret_cast<uint64_t*>(ring + NS * kTileBytes);
  uint64_t* slot_empty = slot_full + NS;
  uint64_t* guard_full = slot_empty + NS;   // [kGuards] a guarded V tile landed
  uint64_t* q_full = guard_full + kGuards;
  uint64_t* q_empty = q_full + 1;
  uint64_t* s_full = q_empty + 1;           // [NQ] a stream's scores stand
  uint64_t* p_half = s_full + 2;            // [NQ][2] half of its weights stand
  uint64_t* o_full = p_half + 4;            // [NQ] its last product of the segment retired
  uint64_t* o_empty = o_full + 2;           // [NQ] its output has been read
  uint64_t* final_bar = o_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(final_bar + 1);
  int* abort_flag = reinterpret_cast<int*>(tmem_slot + 1);
  int* poison = abort_flag + 1;             // [kGuards] segments' marked tiles, bit j: tile g0 + j
  int* last_bar = poison + kGuards;         // [NS + 1] per slot (and Q): barrier and parity of its last copy
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
    for (int s = 0; s < NQ; ++s) {
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
  if (warp == kHelp + 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(su32(tmem_slot)), "r"(kTmem));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_trigger();  // the join's blocks stand ready wherever this kernel's have ended
  Span span;
  const Split split = my_span<128>(a.rows, a.block_nodes, span_tmp, span);
  const int group = a.rows.group, tpt = 128 / group;
  auto guard_from = [&](const Segment& x) { return max(x.t0, x.r.slot < 0 ? 0 : x.r.ctx >> 7); };
  bool run = true;

  // (two streams hold a row of scores in registers: the other warps give some up)
  if (NQ == 2 && warp >= kHelp) asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
  if (warp < kHelp) {
    // ---------------------------------------------------------------- softmax
    if (NQ == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int s = NQ == 1 ? 0 : warp >> 2, r = tid & 127;
    const uint32_t lane_base = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
    const int rt = r / group, rg = r - rt * group;
    const int total = span.end - span.begin;
    int done = 0, items = 0;  // tiles and segments of this stream
    int cut = -1;             // Cut::last of the item that the worker's last segment begins
#pragma unroll 1
    while (run && done < total) {
      // a segment is known here once its first scores stand
      run = mbar_wait_warp(&s_full[s], done & 1, waits);
      if (!run) break;
      const Seg& x = segs[items % kSegs];
      const int node = s * tpt + rt;  // within the block
      const bool valid = rt < tpt && node < x.nodes;
      const bool any_valid = __any_sync(0xffffffffu, valid);
      const uint32_t* mask =
          reinterpret_cast<const uint32_t*>(a.masks) + (int64_t)(x.q0 + (valid ? node : 0)) * (2 * a.words);
      // the first word of the mask (all of it, up to 64 nodes)
      const uint2 head = __ldg(reinterpret_cast<const uint2*>(mask));
      auto bits = [&](int key0) {
        return visible32([&](int i) { return i == 0 ? head.x : i == 1 ? head.y : __ldg(mask + i); }, a.words, x.slot,
                         x.ctx, x.row_nodes, key0);
      };
      tile::RowState row;
      row.reset();
      const int t0 = x.t0, t1 = x.t1;
#pragma unroll 1
      for (int t = t0; t < t1; ++t, ++done) {
        const bool masked = t >= x.g0;
        uint32_t vis[4] = {0u, 0u, 0u, 0u};
        if (masked && valid) {
#pragma unroll
          for (int y = 0; y < 4; ++y) vis[y] = bits(t * 128 + 32 * y);
        }
        if (t > t0) run = mbar_wait_warp(&s_full[s], done & 1, waits);
        if (!run) break;
        fence_after();
        if (!any_valid) {
          // no row of this warp is anyone's: its weights may be anything
          if (lane == 0) {
            mbar_arrive(&p_half[2 * s]);
            mbar_arrive(&p_half[2 * s + 1]);
          }
          continue;
        }
        if (NQ == 1)
          tile::softmax_tile_small<HD>(lane_base, s * 128, kColO + s * 128, a.scale_log2, t == t0, masked, vis[0], vis[1],
                                       vis[2], vis[3], row, su32(&p_half[2 * s]));
        else
          tile::softmax_tile<HD>(lane_base, s * 128, kColO + s * 128, a.scale_log2, t == t0, masked, vis, row,
                                 &p_half[2 * s], &p_half[2 * s + 1]);
      }
      if (!run || !mbar_wait_warp(&o_full[s], items & 1, waits)) break;
      fence_after();
      const int marks = x.g0 < t1 ? poison[items % kGuards] : 0;
      const bool whole = t0 == 0 && t1 == x.tiles;
      // a row whose weights are all zero (nothing visible, or every score -inf) gives zero
      const float inv = whole ? (row.l == 0.f ? 0.f : 1.f / row.l) : 1.f;
      float* mine = part(a, blockIdx.x, t0 == 0);
      const int prow = s * 128 + r;
      if (t0 == 0 && !whole) {
        cut = owner(split, x.first + x.tiles - 1);
        if (tid == 0) *reinterpret_cast<int4*>(a.cuts + blockIdx.x) = make_int4(cut, x.q0, x.nodes, x.hk);
      }
      __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(a.out) + (int64_t)(x.q0 + node) * a.o_tok +
                           (int64_t)(x.hk * group + rg) * a.o_head;
#pragma unroll 1
      for (int col = 0; col < HD; col += 32) {
        uint32_t u[32];
        float* o = reinterpret_cast<float*>(u);
        if (any_valid) {
          tmem_ld32(lane_base + kColO + s * 128 + col, u);
          tmem_wait_ld();
        }
        if (marks && valid) {
          const int keys = min(x.ctx + x.row_nodes, t1 * 128);
#pragma unroll 1
          for (int key = x.g0 * 128; key < keys; ++key) {
            if (!(marks >> min((key >> 7) - x.g0, 31) & 1) || !(bits(key & ~31) >> (key & 31) & 1u)) continue;
            const int bi = key / a.block_size;
            if (x.slot < 0 || bi >= min(a.nblocks[x.slot], a.max_blocks)) continue;
            const int blk = a.block_table[(int64_t)x.slot * a.max_blocks + bi];
            if (blk < 0 || blk >= a.num_blocks) continue;
            const __nv_bfloat16* v =
                reinterpret_cast<const __nv_bfloat16*>(a.v_pool) +
                (((int64_t)blk * a.rows.kv_heads + x.hk) * a.block_size + key % a.block_size) * HD + col;
#pragma unroll
            for (int y = 0; y < 32; ++y) {
              const float f = __bfloat162float(v[y]);
              if (!isfinite(f)) o[y] += f;
            }
          }
        }
        if (valid && whole) {
          tile::store_row32(dst + col, o, inv, a.out_vec);
        } else if (valid) {
#pragma unroll
          for (int y = 0; y < 8; ++y)
            __stcg(part_cols(a, mine, prow, col + 4 * y), make_float4(o[4 * y], o[4 * y + 1], o[4 * y + 2], o[4 * y + 3]));
        }
      }
      if (!whole && valid) __stcg(part_stats(a, mine, prow), make_float2(row.m, row.l));
      // the output and the segment's description have been read
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&o_empty[s]);
      ++items;
    }
    if (cut < 0 && tid == 0) *reinterpret_cast<int4*>(a.cuts + blockIdx.x) = make_int4(-1, 0, 0, 0);
  } else if (warp == kHelp + 1) {
    // ---------------------------------------------------------------- products
    const uint32_t el = elect_one();
    const uint32_t full0 = su32(slot_full), empty0 = su32(slot_empty), ring0 = su32(ring), q0 = su32(q_s);
    const uint32_t part0 = su32(p_half);
    int slot = 0;                  // next slot of the ring, and the parity of its fill
    uint32_t fill = 0;
    uint32_t parts = 0, outs = 3;  // per stream (bit): parity of its next weights, of its last output's reading
    int segment = 0;
    auto next_slot = [&](int& i, uint32_t& par) {
      i = slot;
      par = fill;
      if (++slot == NS) {
        slot = 0;
        fill ^= 1;
      }
    };
#pragma unroll 1
    for (int left = span.end - span.begin; run && left > 0;) {
      int k, v = 0, nt = 0;
      uint32_t kp, vp = 0;
      // step i: the values of tile i, then the scores of tile i + 1, stream by stream
#pragma unroll 1
      for (int i = -1; run && i < nt; ++i) {
        if (i >= 0) next_slot(v, vp);
        const bool more = i + 1 < nt || i < 0;
        const uint32_t vbar = full0 + 8 * v;
        if (more) {
          next_slot(k, kp);
        } else {
          k = v;
          kp = vp;
        }
        const uint32_t kbar = full0 + 8 * k;
        if (i < 0) {
          run = mbar_wait3_warp(su32(q_full), segment & 1, kbar, kp, kbar, kp, Waits{abort_flag, a.wait_tries});
          if (!run) break;
          const Seg& x = segs[segment++ % kSegs];
          nt = x.t1 - x.t0;
          left -= nt;
        }
#pragma unroll
        for (int s = 0; s < NQ; ++s) {
          if (!run) break;
          const uint32_t s_col = tmem + s * 128, o_col = tmem + kColO + s * 128;
          if (i >= 0) {
            const uint32_t part = part0 + 16 * s, par = parts >> s & 1u;
            // the output of the segment before has been read
            if (i == 0) run = mbar_wait_warp(&o_empty[s], outs >> s & 1u, waits);
            run = run && (s == 0 ? mbar_wait3_warp(part, par, vbar, vp, kbar, kp, waits)
                                 : mbar_wait_warp(part, par, waits));
            if (!run) break;
            fence_after();
            issue_values<HD>(el, o_col, s_col, ring0 + v * kTileBytes, 0, i == 0);
            run = mbar_wait_warp(part + 8, par, waits);
            if (!run) break;
            fence_after();
            issue_values<HD>(el, o_col, s_col, ring0 + v * kTileBytes, 1, false);
            parts ^= 1u << s;
            if (!more) {
              mma_commit(el, &o_full[s]);
              outs ^= 1u << s;
            }
          }
          if (more) {
            fence_after();
            issue_scores<HD>(el, s_col, q0 + s * kTileBytes, ring0 + k * kTileBytes);
            mma_commit(el, &s_full[s]);
          }
        }
        if (!run) break;
        if (i >= 0) mma_commit(el, empty0 + 8 * v);
        if (more) mma_commit(el, empty0 + 8 * k);
        if (i + 2 == nt) mma_commit(el, q_empty);
      }
    }
    mma_commit(el, final_bar);
  } else {
    Walk<128> walk;
    walk.start(a.rows, span, a.block_nodes);
    Segment g;
    if (warp == kHelp || (NQ == 1 && warp == kHelp + 4)) {
      // -------------------------------------------------------------- pages
      // NQ = 1: this warp's K or V tiles, every second slot; NQ = 2: both in turn
      const int kv0 = warp == kHelp ? 0 : 1, kv1 = NQ == 1 ? kv0 : 1;
      const int bs = a.block_size, ppt = 128 / bs, tpc = 32 / ppt, oob = a.num_blocks * a.rows.kv_heads * bs;
      const uint32_t el = elect_one();
      const uint32_t empty0 = su32(slot_empty), full0 = su32(slot_full), guard0 = su32(guard_full), ring0 = su32(ring);
      int gd = 0, slot = kv0;
      uint32_t fill = 0;
#pragma unroll 1
      while (run && walk.next(g)) {
        const int g0 = guard_from(g), keys = g.r.ctx + g.r.nodes;
        const int32_t* table = a.block_table + (int64_t)max(g.r.slot, 0) * a.max_blocks;
        const int held = g.r.slot >= 0 ? a.nblocks[g.r.slot] : 0;
        // the pool rows of 32 pages (32 / ppt tiles), a page per lane, and of the next
        // 32; the first ones' loads and that of `held` do not wait for each other
        auto page = [&](int j) -> int {
          const int pi = g.t0 * ppt + j;
          if (g.r.slot < 0 || pi >= g.t1 * ppt || pi >= a.max_blocks || pi * bs >= keys) return oob;
          const int b = __ldg(table + pi);
          return pi < held && b >= 0 && b < a.num_blocks ? (b * a.rows.kv_heads + g.hk) * bs : oob;
        };
        int cur = page(lane), nxt = page(32 + lane);
#pragma unroll 1
        for (int t = g.t0; run && t < g.t1; ++t) {
          const int i = t - g.t0, src = (i & (tpc - 1)) * ppt;
          if (i > 0 && src == 0) {
            cur = nxt;
            nxt = page(32 * (i / tpc + 1) + lane);
          }
          int y[8];
#pragma unroll
          for (int p = 0; p < 8; ++p) y[p] = __shfl_sync(0xffffffffu, cur, (src + p) & 31);
#pragma unroll 1
          for (int kv = kv0; kv <= kv1; ++kv) {
            run = mbar_wait_warp(empty0 + 8 * slot, fill ^ 1, waits);
            if (!run) break;
            const bool guarded = kv == 1 && t >= g0;
            const uint32_t bar = guarded ? guard0 + 8 * (gd % kGuards) : full0 + 8 * slot;
            if (el) {
              last_bar[slot] = guarded ? (NS + gd % kGuards) * 2 + ((gd / kGuards) & 1) : slot * 2 + (int)fill;
              mbar_expect_tx(bar, kTileBytes);
            }
            __syncwarp();
            const uint32_t dst = ring0 + slot * kTileBytes;
            const CUtensorMap* map = kv ? &tmv : &tmk;
#pragma unroll
            for (int p = 0; p < 8; ++p) {
              if (p >= ppt) break;
#pragma unroll
              for (int h = 0; h < kHalves; ++h)
                tma_load_2d(el, dst + h * kHalfBytes + p * bs * 128, map, h * 64, y[p], bar);
            }
            if (guarded) ++gd;
            slot += NQ == 1 ? 2 : 1;
            if (slot >= NS) {
              slot -= NS;
              fill ^= 1;
            }
          }
        }
      }
    } else if (warp == kHelp + 3) {
      // -------------------------------------------------------------- queries
      if (lane == 0) {
        int n = 0;
#pragma unroll 1
        while (walk.next(g)) {
          if (!mbar_wait(q_empty, (n & 1) ^ 1, waits)) break;
          // (the segment kSegs before has been written out: the one before this
          // has made its last scores, which came after its own first product,
          // and that after the reading of the output before it)
          Seg& x = segs[n % kSegs];
          const int node0 = g.block * a.block_nodes;
          x.q0 = g.r.n0 + node0;
          x.nodes = min(a.block_nodes, g.r.nodes - node0);
          x.hk = g.hk;
          x.slot = g.r.slot;
          x.ctx = g.r.ctx;
          x.row_nodes = g.r.nodes;
          x.t0 = g.t0;
          x.t1 = g.t1;
          x.tiles = g.tiles;
          x.first = g.first;
          x.g0 = guard_from(g);
          last_bar[NS] = n & 1;
          ++n;
          const int tiles = NQ == 2 && x.nodes > tpt ? 2 : 1;
          mbar_expect_tx(q_full, tiles * kHalves * tpt * group * 128);
#pragma unroll 1
          for (int i = 0; i < tiles * kHalves; ++i)
            tma_load_3d(q_s + i * kHalfBytes, &tmq, (i % kHalves) * 64, g.hk * group,
                        g.r.n0 + node0 + i / kHalves * tpt, q_full);
        }
      }
    } else {
      // -------------------------------------------------------------- guard
      int gd = 0, tiles = 0, items = 0;
#pragma unroll 1
      while (run && walk.next(g)) {
        const int g0 = guard_from(g);
        int marks = 0;
#pragma unroll 1
        for (int t = g0; t < g.t1; ++t, ++gd) {
          run = mbar_wait_warp(&guard_full[gd % kGuards], (gd / kGuards) & 1, waits);
          if (!run) break;
          const int s = (2 * (tiles + t - g.t0) + 1) % NS;
          if (tile::clear_nonfinite(reinterpret_cast<uint4*>(ring + s * kTileBytes), kTileBytes / 16))
            marks |= 1 << min(t - g0, 31);
          if (lane == 0) {
            poison[items % kGuards] = marks;
            mbar_arrive(&slot_full[s]);
          }
        }
        tiles += g.t1 - g.t0;
        ++items;
      }
    }
  }

  __syncthreads();
  if (*waits.abort_flag && tid == 0) {
    atomicOr(a.status, PSE_STATUS_TIMEOUT);
    for (int i = 0; i < NS; ++i)
      if (last_bar[i] >= 0) {
        const int b = last_bar[i] >> 1;
        mbar_drain(b < NS ? &slot_full[b] : &guard_full[b - NS], last_bar[i] & 1);
      }
    if (last_bar[NS] >= 0) mbar_drain(q_full, last_bar[NS]);
  }
  if (warp == kHelp + 1) {
    if (lane == 0) mbar_drain(final_bar, 0);
    __syncwarp();
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmem));
  }
}

Map3Cache g_q_maps;
TmapCache g_pool_maps;

bool tc_eligible(const Args& a, int q_heads) {
  const int64_t pool_rows = (int64_t)a.num_blocks * a.rows.kv_heads * a.block_size;
  return (a.hd == 64 || a.hd == 128) &&
         (a.block_size == 16 || a.block_size == 32 || a.block_size == 64 || a.block_size == 128) && a.num_blocks > 0 &&
         a.scale_log2 > 0.f && (reinterpret_cast<uintptr_t>(a.k_pool) | reinterpret_cast<uintptr_t>(a.v_pool)) % 16 == 0 &&
         pool_rows + a.block_size < (1ll << 31) && tma_rows(a.q, a.q_tok, a.q_head, q_heads, a.hd);
}

template <int HD, int NQ>
int launch_tc(Args& a, int q_heads, cudaStream_t s) {
  auto kern = tree_tc_kernel<HD, NQ>;
  constexpr size_t smem = tc_smem_bytes<HD, NQ>();
  static_assert(smem + 640 <= 227 * 1024, "shared memory");
  static const cudaError_t opt = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (opt != cudaSuccess) return (int)opt;
  const int tpt = 128 / a.rows.group, ctas = NQ == 1 ? 2 * kNumSMs : kNumSMs;
  a.block_nodes = NQ * tpt;
  CUtensorMap mq, mk, mv;
  int rc = g_q_maps.get(Map3Key{reinterpret_cast<uint64_t>(a.q), (uint64_t)HD, (uint64_t)q_heads,
                                (uint64_t)a.rows.n_nodes, (uint64_t)(q_heads == 1 ? HD : a.q_head) * 2,
                                (uint64_t)a.q_tok * 2, (uint32_t)a.rows.group, (uint32_t)tpt},
                        PSE_EINVAL, &mq);
  const uint64_t pool_rows = (uint64_t)a.num_blocks * a.rows.kv_heads * a.block_size;
  if (rc == 0) rc = g_pool_maps.get(a.k_pool, HD, pool_rows, HD * 2, 64u, a.block_size, PSE_EINVAL, &mk);
  if (rc == 0) rc = g_pool_maps.get(a.v_pool, HD, pool_rows, HD * 2, 64u, a.block_size, PSE_EINVAL, &mv);
  if (rc) return rc;
  a.part_rows = 128 * NQ;
  if (!countable(a.rows, 128, a.block_nodes)) return PSE_EINVAL;
  const cudaError_t e = launch_pdl(kern, dim3(ctas), dim3(n_threads<NQ>()), smem, s, mq, mk, mv, a);
  if (e != cudaSuccess) return (int)e;
  return launch_join<__nv_bfloat16>(a, ctas, tpt * a.rows.group, 128, s);
}

template <int HD>
int tc_attention(Args& a, int q_heads, int max_nodes, cudaStream_t s) {
  // (64 nodes of 4 heads over 16384 tokens, 12 requests: 209 us; with one stream per
  // CTA, which reads each K/V tile once per 128 rows, 285.  The other way round, 64
  // trees of 5 to 26 nodes: 68 us on two streams, of which one has no rows, 54 on one.)
  return max_nodes > 128 / a.rows.group ? launch_tc<HD, 2>(a, q_heads, s)
                                        : launch_tc<HD, 1>(a, q_heads, s);
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
  // two partial results per CTA: of 64 rows on the CUDA cores, of 256 on the tensor cores
  const size_t simt = (size_t)tree::kMaxWorkers * 64, tc = (size_t)kNumSMs * 256;
  return tree::kCutBytes + (head_dim <= 128 && tc > simt ? tc : simt) * 2 * tree::part_width(head_dim) * 4;
}

extern "C" int pse_token_tree_attention(pse_block_state st, pse_kv_layer kv, const pse_head_view* views,
                                        const int32_t* slots, const int32_t* ctx, const int32_t* node_off,
                                        int32_t rows, int32_t n_nodes, int32_t max_nodes, const int64_t* masks,
                                        int32_t words, float scale, void* workspace, size_t workspace_bytes,
                                        void* stream) {
  if (!views) return PSE_EINVAL;
  const pse_head_view &q = views[0], &out = views[1];
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
  a.rows.max_nodes = max_nodes;
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
  a.cuts = (tree::Cut*)workspace;
  a.parts = (float*)((char*)workspace + tree::kCutBytes);
  a.status = st.status;
  a.wait_tries = t5::wait_tries();
  a.out_vec = reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && a.o_tok % 8 == 0 && a.o_head % 8 == 0;
  if (kv.dtype == PSE_BF16 && tree::tc_eligible(a, q.heads))
    return a.hd == 64 ? tree::tc_attention<64>(a, q.heads, max_nodes, (cudaStream_t)stream)
                      : tree::tc_attention<128>(a, q.heads, max_nodes, (cudaStream_t)stream);
  return kv.dtype == PSE_BF16 ? tree::simt_attention<__nv_bfloat16>(a, max_nodes, (cudaStream_t)stream)
                              : tree::simt_attention<float>(a, max_nodes, (cudaStream_t)stream);
}
