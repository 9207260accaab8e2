// How the work of one token-tree attention call is split over the CTAs.
//
// Row i (a request) has nodes_i queries per head over ctx_i + nodes_i keys.  Its
// items are (query block, K/V head), each a run of ceil(keys / tile) key tiles.
// The tiles of all items of all rows, in order, form one line of T tiles; CTA
// c of G takes the tiles [c T / G, (c + 1) T / G), so every CTA has the same
// number of tiles (within one) whatever the lengths are, and nothing about
// them has to be known on the host.  An item whose tiles all fall to one CTA
// is finished there.  An item cut by CTA boundaries leaves one partial result
// per CTA (maximum, sum and unnormalised output) in the workspace, which a
// second, small kernel joins in the order of the CTAs.  (Joining by the last CTA
// to arrive saves that launch but leaves the rows of an item to one warp each
// 32, serially: 158 us instead of %JOIN% at 64 requests of 128 to 4096 tokens.)
#pragma once

#include "common.cuh"

namespace pse {
namespace tree {

struct Rows {
  const int32_t* slots;
  const int32_t* ctx;
  const int32_t* node_off;  // [rows + 1]
  int rows, num_slots, n_nodes, kv_heads, group;
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
  if (r.n0 < 0 || r.nodes < 0 || (int64_t)r.n0 + r.nodes > a.n_nodes) r.nodes = 0;
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

struct Span {
  long long begin, end, total;  // this CTA's tiles, all tiles
  int ctas;                     // CTAs that have tiles
  int row;                      // row of the first tile
  long long off;                // its offset within the row
};

// All threads of the CTA; `tmp` holds 40 long longs of shared memory.
template <int TILE>
__device__ Span my_span(const Rows& a, int block_nodes, long long* tmp) {
  const int per = (a.rows + blockDim.x - 1) / blockDim.x;
  const int lo = min(a.rows, (int)threadIdx.x * per), hi = min(a.rows, lo + per);
  auto weight = [&](int i) -> long long {
    const Row r = read_row(a, i);
    return (long long)key_tiles<TILE>(r) * q_blocks(a, r, block_nodes) * a.kv_heads;
  };
  long long mine = 0, first = 0;
  for (int i = lo; i < hi; ++i) {
    const long long w = weight(i);
    if (i == lo) first = w;
    mine += w;
  }
  // exclusive prefix over the threads
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = (blockDim.x + 31) / 32;
  long long inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long n = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += n;
  }
  if (lane == 31) tmp[warp] = inc;
  __syncthreads();
  long long before = inc - mine, total = 0;
  for (int w = 0; w < nw; ++w) {
    if (w < warp) before += tmp[w];
    total += tmp[w];
  }
  Span s;
  s.total = total;
  s.ctas = (int)min((long long)gridDim.x, total);
  const int c = blockIdx.x;
  s.begin = s.end = 0;
  s.row = 0;
  s.off = 0;
  if (c < s.ctas) {
    s.begin = total * c / s.ctas;
    s.end = total * (c + 1) / s.ctas;
    if (s.begin >= before && s.begin < before + mine) {
      long long at = s.begin - before;
      int i = lo;
      long long w = first;
      while (at >= w) {
        at -= w;
        w = weight(++i);
      }
      tmp[32] = i;
      tmp[33] = at;
    }
  }
  __syncthreads();
  if (c < s.ctas) {
    s.row = (int)tmp[32];
    s.off = tmp[33];
  }
  __syncthreads();
  return s;
}

// The CTA that has tile x.
__device__ __forceinline__ int owner(const Span& s, long long x) { return (int)(((x + 1) * s.ctas - 1) / s.total); }

// One run of tiles of one item, within one CTA.
struct Segment {
  int row, hk, block;     // the item
  Row r;
  int t0, t1, tiles;      // key tiles [t0, t1) of the item's `tiles`
  long long first;        // the item's first tile on the line
};

// Walks a CTA's segments.
template <int TILE>
struct Walk {
  const Rows& a;
  const Span& s;
  int block_nodes;
  long long at;  // next tile on the line
  int row;
  long long off;
  __device__ Walk(const Rows& rows, const Span& span, int bn)
      : a(rows), s(span), block_nodes(bn), at(span.begin), row(span.row), off(span.off) {}
  __device__ bool next(Segment& g) {
    if (at >= s.end) return false;
    Row r = read_row(a, row);
    int nt = key_tiles<TILE>(r);
    long long w = (long long)nt * q_blocks(a, r, block_nodes) * a.kv_heads;
    while (off >= w) {
      off -= w;
      if (++row >= a.rows) return false;
      r = read_row(a, row);
      nt = key_tiles<TILE>(r);
      w = (long long)nt * q_blocks(a, r, block_nodes) * a.kv_heads;
    }
    const long long item = off / nt;
    g.row = row;
    g.r = r;
    g.tiles = nt;
    g.t0 = (int)(off - item * nt);
    g.t1 = (int)min((long long)nt, g.t0 + (s.end - at));
    // the blocks of one K/V head side by side: they read the same keys
    const int nb = q_blocks(a, r, block_nodes);
    g.hk = (int)(item / nb);
    g.block = (int)(item % nb);
    g.first = at - g.t0;
    at += g.t1 - g.t0;
    off += g.t1 - g.t0;
    return true;
  }
};

// 32 keys' visibility for one query node, bit b for key `key0 + b`: every key
// below the context, then the nodes its mask names.
__device__ __forceinline__ uint32_t visible32(const int64_t* mask, int words, const Row& r, int key0) {
  if (r.slot < 0) return 0u;
  const int d = key0 - r.ctx;
  if (d <= -32) return 0xffffffffu;
  uint32_t bits = d < 0 ? (1u << -d) - 1u : 0u;
  // node bits [max(d, 0), d + 32) of the mask, nodes past the tree never
  const int n0 = max(d, 0), sh = n0 - d;
  if (n0 < r.nodes) {
    const uint32_t* m = reinterpret_cast<const uint32_t*>(mask);
    const int w = n0 >> 5, b = n0 & 31, nw = 2 * words;
    const uint32_t lo = w < nw ? __ldg(m + w) : 0u, up = w + 1 < nw ? __ldg(m + w + 1) : 0u;
    uint32_t x = __funnelshift_r(lo, up, b);
    const int left = r.nodes - n0;
    if (left < 32) x &= (1u << left) - 1u;
    bits |= x << sh;
  }
  return bits;
}

}  // namespace tree
}  // namespace pse
