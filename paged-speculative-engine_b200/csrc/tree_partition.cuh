// How the work of one token-tree attention call is split over its workers, the
// CTAs.
//
// Row i (a request) has nodes_i queries per head over ctx_i + nodes_i keys.  Its
// items are (query block, K/V head), each a run of ceil(keys / tile) key tiles.
// The tiles of all items of all rows, in order, form one line of T tiles; worker
// c of G takes T / G of them (the first T mod G one more), so every worker has
// the same number of tiles whatever the lengths are, and nothing about them has
// to be known on the host.  An item whose tiles all fall to one worker is
// finished there.  An item cut by the workers' bounds leaves one partial result
// per worker (maximum, sum and unnormalised output) in the workspace, which a
// second, small kernel joins in the order of the workers.  (Joining by the last
// of them to arrive saves that launch but leaves an item's rows to one CTA:
// 158 us instead of 95 at 64 requests of 128 to 4096 tokens, all else equal.)
#pragma once

#include "common.cuh"

namespace pse {
namespace tree {

struct Rows {
  const int32_t* slots;
  const int32_t* ctx;
  const int32_t* node_off;  // [rows + 1]
  int rows, num_slots, n_nodes, max_nodes, kv_heads, group;
  int64_t max_keys;  // keys a block table can hold
};

struct Row {
  int slot, ctx, n0, nodes;  // nodes == 0: no work
};

__device__ __forceinline__ Row read_row(const Rows& a, int i) {
  Row r;
  r.slot = a.slots[i];
  r.ctx = a.ctx[i];
  r.n0 = a.node_off[i];
  r.nodes = a.node_off[i + 1] - r.n0;
  if (r.n0 < 0 || r.nodes < 0 || r.nodes > a.max_nodes || (int64_t)r.n0 + r.nodes > a.n_nodes) r.nodes = 0;
  if (r.slot < 0 || r.slot >= a.num_slots) r.slot = -1;
  // a context the table cannot hold is not one: its nodes see nothing
  if (r.ctx < 0 || (int64_t)r.ctx + r.nodes > a.max_keys) {
    r.ctx = 0;
    r.slot = -1;
  }
  return r;
}

// Query blocks of `block_rows` rows (node, group head) per K/V head.
__device__ __forceinline__ int q_blocks(const Rows& a, const Row& r, int block_nodes) {
  return (r.nodes + block_nodes - 1) / block_nodes;
}

template <int TILE>
__device__ __forceinline__ int key_tiles(const Row& r) {
  return r.nodes > 0 ? (r.ctx + r.nodes + TILE - 1) / TILE : 0;
}

// All counts of tiles fit 31 bits (the entry point checks the largest that the
// block table allows): 64-bit divisions took longer than the loads of a tile.
struct Split {
  int per, extra;    // tiles per worker; the first `extra` workers have one more
  int workers;       // workers that have tiles
};
struct Span {
  int begin, end;    // a worker's tiles
  int row, off;      // row of the first tile, and its offset within the row
  Row r;             // that row
};

template <int TILE>
__device__ __forceinline__ int row_weight(const Rows& a, const Row& r, int block_nodes) {
  return r.nodes > 0 ? key_tiles<TILE>(r) * q_blocks(a, r, block_nodes) * a.kv_heads : 0;
}

// The span of this CTA, worker blockIdx.x of gridDim.x.  All threads of the CTA;
// `tmp` holds 40 ints of shared memory.
template <int TILE>
__device__ Split my_span(const Rows& a, int block_nodes, int* tmp, Span& x) {
  const int per = (a.rows + blockDim.x - 1) / blockDim.x;
  const int lo = min(a.rows, (int)threadIdx.x * per), hi = min(a.rows, lo + per);
  int mine = 0, first = 0;
  Row r{-1, 0, 0, 0};  // row lo
#pragma unroll 1
  for (int i = lo; i < hi; ++i) {
    const Row ri = read_row(a, i);
    const int w = row_weight<TILE>(a, ri, block_nodes);
    if (i == lo) {
      first = w;
      r = ri;
    }
    mine += w;
  }
  // exclusive prefix over the threads
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = (blockDim.x + 31) / 32;
  const int inc = warp_inclusive_scan(mine);
  if (lane == 31) tmp[warp] = inc;
  __syncthreads();
  int before = inc - mine, total = 0;
#pragma unroll 1
  for (int w = 0; w < nw; ++w) {
    const int y = tmp[w];
    before += w < warp ? y : 0;
    total += y;
  }
  Split s;
  s.workers = min((int)gridDim.x, total);
  s.per = s.workers > 0 ? total / s.workers : 0;
  s.extra = total - s.per * s.workers;
  const int c = blockIdx.x;
  x.begin = x.end = x.row = x.off = 0;
  x.r = Row{-1, 0, 0, 0};
  if (c < s.workers) {
    x.begin = s.per * c + min(c, s.extra);
    x.end = x.begin + s.per + (c < s.extra ? 1 : 0);
    if (x.begin >= before && x.begin < before + mine) {
      int at = x.begin - before, i = lo, w = first;
#pragma unroll 1
      while (at >= w) {
        at -= w;
        r = read_row(a, ++i);
        w = row_weight<TILE>(a, r, block_nodes);
      }
      tmp[32] = i;
      tmp[33] = at;
      tmp[34] = r.slot;
      tmp[35] = r.ctx;
      tmp[36] = r.n0;
      tmp[37] = r.nodes;
    }
  }
  __syncthreads();
  if (c < s.workers) {
    x.row = tmp[32];
    x.off = tmp[33];
    x.r = Row{tmp[34], tmp[35], tmp[36], tmp[37]};
  }
  return s;
}

// The worker that has tile x.
__device__ __forceinline__ int owner(const Split& s, int x) {
  const int cut = s.extra * (s.per + 1);
  return x < cut ? x / (s.per + 1) : s.extra + (x - cut) / s.per;
}

// One run of tiles of one item, within one worker.
struct Segment {
  int hk, block;          // the item: K/V head and query block
  Row r;
  int t0, t1, tiles;      // key tiles [t0, t1) of the item's `tiles`
  int first;              // the item's first tile on the line
};

// Whether the tiles of any call of these sizes can be counted in 31 bits.
inline bool countable(const Rows& a, int tile, int block_nodes) {
  const int64_t tiles = (a.max_keys + tile - 1) / tile, blocks = (a.max_nodes + block_nodes - 1) / block_nodes;
  return (double)tiles * (double)blocks * a.kv_heads * a.rows < 2147483647.0;
}

// Walks a worker's segments.
template <int TILE>
struct Walk {
  const Rows* rows;
  int block_nodes, at, end, row, off, w, nt, nb;  // next tile on the line, ...; the row's weight, tiles, blocks
  Row r;
  __device__ __forceinline__ void start(const Rows& a, const Span& span, int bn) {
    rows = &a;
    block_nodes = bn;
    at = span.begin;
    end = span.end;
    row = span.row;
    off = span.off;
    r = span.r;
    weigh();
  }
  __device__ __forceinline__ void weigh() {
    nt = key_tiles<TILE>(r);
    nb = q_blocks(*rows, r, block_nodes);
    w = nt * nb * rows->kv_heads;
  }
  __device__ bool next(Segment& g) {
    if (at >= end) return false;
#pragma unroll 1
    while (off >= w) {
      off -= w;
      if (++row >= rows->rows) return false;
      r = read_row(*rows, row);
      weigh();
    }
    const int item = off / nt;
    g.r = r;
    g.tiles = nt;
    g.t0 = off - item * nt;
    g.t1 = min(nt, g.t0 + (end - at));
    // the blocks of one K/V head side by side: they read the same keys
    g.hk = item / nb;
    g.block = item - g.hk * nb;
    g.first = at - g.t0;
    at += g.t1 - g.t0;
    off += g.t1 - g.t0;
    return true;
  }
};

// 32 keys' visibility for one query node, bit b for key `key0 + b`: every key
// below the context, then the nodes its mask names; word(i): the mask's i-th 32
// bits (i < 2 words).
template <typename F>
__device__ __forceinline__ uint32_t visible32(F word, int words, int slot, int ctx, int nodes, int key0) {
  if (slot < 0) return 0u;
  const int d = key0 - ctx;
  if (d <= -32) return 0xffffffffu;
  uint32_t bits = d < 0 ? (1u << -d) - 1u : 0u;
  // node bits [max(d, 0), d + 32) of the mask, nodes past the tree never
  const int n0 = max(d, 0), sh = n0 - d;
  if (n0 < nodes) {
    const int w = n0 >> 5, b = n0 & 31, nw = 2 * words;
    const uint32_t lo = w < nw ? word(w) : 0u, up = w + 1 < nw ? word(w + 1) : 0u;
    uint32_t x = __funnelshift_r(lo, up, b);
    const int left = nodes - n0;
    if (left < 32) x &= (1u << left) - 1u;
    bits |= x << sh;
  }
  return bits;
}

}  // namespace tree
}  // namespace pse
