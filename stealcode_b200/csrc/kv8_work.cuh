// kv8_work.cuh -- how an attention call's work is shared out over the blocks
// of a launch.
//
// For one (sequence, kv head) the query rows are the pairs (token, query
// head of that kv head), token-major; an item is ROWS of them, and its keys
// are the tiles of TILE consecutive tokens that hold a token some row sees:
// tiles [0, a) of the first `sinks` tokens, then tiles [b, c) of the window.
// Every item counts OVER units (its queries, its result) and one for each
// tile; all items' units, one after the other, are cut into equal contiguous
// shares, one per block, whatever the sequences' lengths: a block computes
// whole items and at most two parts of items (the end of one, the start of
// another).  Parts go to the workspace; the block that finishes an item last
// joins its parts in order, so the result does not depend on who was last.
#pragma once

#include "kv8.cuh"

namespace sc {
namespace kv8 {

struct WorkGrid {
  int group;       // query heads per kv head
  uint32_t magic;  // 2^21 / group, rounded up
  int per_seq;     // items per sequence and kv head, at most
  int entries;     // m * per_seq
  int min_share;   // units; fewer blocks work when there are few
  int32_t *count;  // [blocks] parts done of the item that starts in a block
  float *parts;    // [2 * blocks] parts
};

struct Entry {
  int i, s;         // entry of the batch, sequence (-1: none)
  int64_t row0;     // first packed token
  int first;        // position of that token
  int r0, r1;       // rows [r0, r1) of the sequence
  int j0, h0;       // row r0's token (from row0) and query head
  int p_lo, p_hi;   // positions of the first and the last row
  int a, b, c;
  unsigned bad;     // status bits of what is wrong with entry i
  __device__ __forceinline__ int tiles() const { return a + c - b; }
  __device__ __forceinline__ int steps() const { return max(1, tiles()); }  // an item without keys has a result too
  __device__ __forceinline__ int tile(int x) const { return x < a ? x : b + x - a; }
  // Token and query head of row r0 + k, k < 256: (h0 + k) / group by a product
  // with 2^21 / group rounded up, exact as (h0 + k) * group < 1280 * 1024 < 2^21.
  __device__ __forceinline__ void row(const WorkGrid &g, int k, int &j, int &h) const {
    const uint32_t x = (uint32_t)(h0 + k), d = x * g.magic >> 21;
    j = j0 + (int)d;
    h = (int)(x - d * (uint32_t)g.group);
  }
};

// False when entry e has no rows.
template <int ROWS, int TILE>
__device__ __forceinline__ bool get_entry(const AttendArgs &p, const WorkGrid &g, int e, Entry &o) {
  o.i = (int)((uint32_t)e / (uint32_t)g.per_seq);
  int count;
  o.bad = p.b.rows(o.i, o.row0, count) ? 0u : (unsigned)kBadRows;
  o.r0 = (e - o.i * g.per_seq) * ROWS;
  const int rows = count * g.group;
  if (o.r0 >= rows) return false;
  o.r1 = min(rows, o.r0 + ROWS);
  o.s = p.b.seq(o.i, p.c.n_seqs);
  if (o.s < 0) o.bad = kBadSeq;
  const int len = o.s < 0 ? 0 : seq_length(p.c, o.s);
  o.first = len - count;
  o.j0 = (int)((uint32_t)o.r0 / (uint32_t)g.group);
  o.h0 = o.r0 - o.j0 * g.group;
  int j, h;
  o.row(g, o.r1 - 1 - o.r0, j, h);
  o.p_lo = o.first + o.j0;
  o.p_hi = o.first + j;
  o.a = o.b = o.c = 0;
  if (o.p_hi >= 0) {
    o.c = o.p_hi / TILE + 1;
    if (p.window > 0) {
      o.b = max(0, max(o.p_lo, 0) - p.window + 1) / TILE;
      o.a = min((min(p.sinks, o.p_hi + 1) + TILE - 1) / TILE, o.b);
    }
  }
  return true;
}

// A block's share [pos, end) of all units and the entry that holds pos.
struct Share {
  int64_t pos, end, total;
  int blocks;       // blocks that have a share
  int e;            // entry
  int64_t at;       // first unit of entry e
};

// The block whose share holds unit `pos`.
__device__ __forceinline__ int block_of(int64_t pos, int64_t total, int blocks) {
  return (int)(((pos + 1) * blocks - 1) / total);
}

struct ShareScratch {
  int64_t warp[32];
  int e;
  int64_t at;
};

// All threads of the block call; false when the block has nothing to do.
template <int ROWS, int TILE, int OVER, int THREADS>
__device__ bool find_share(const AttendArgs &p, const WorkGrid &g, ShareScratch &sh, Share &o) {
  const int tid = (int)threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (g.entries + THREADS - 1) / THREADS;
  const int e0 = min(tid * per, g.entries), e1 = min(e0 + per, g.entries);
  int64_t mine = 0;
  unsigned bad = 0;
  Entry en;
  for (int e = e0; e < e1; e++) {
    if (get_entry<ROWS, TILE>(p, g, e, en)) mine += (int64_t)(OVER + en.steps()) * p.c.kv;
    bad |= en.bad;
  }
  if (bad && blockIdx.x == 0) atomicOr(p.c.status, bad);
  int64_t x = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += y;
  }
  if (lane == 31) sh.warp[warp] = x;
  __syncthreads();
  int64_t before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; w++) {
    if (w < warp) before += sh.warp[w];
    total += sh.warp[w];
  }
  const int64_t start = before + x - mine;
  o.total = total;
  const int64_t most = (total + g.min_share - 1) / g.min_share;
  o.blocks = (int)(most < (int64_t)gridDim.x ? most : (int64_t)gridDim.x);
  if ((int)blockIdx.x >= o.blocks) return false;
  o.pos = (int64_t)blockIdx.x * total / o.blocks;
  o.end = ((int64_t)blockIdx.x + 1) * total / o.blocks;
  if (o.pos >= start && o.pos < start + mine) {
    int64_t at = start;
    for (int e = e0; e < e1; e++) {
      if (!get_entry<ROWS, TILE>(p, g, e, en)) continue;
      const int64_t n = (int64_t)(OVER + en.steps()) * p.c.kv;
      if (o.pos < at + n) {
        sh.e = e;
        sh.at = at;
        break;
      }
      at += n;
    }
  }
  __syncthreads();
  o.e = sh.e;
  o.at = sh.at;
  return o.pos < o.end;
}

// One piece of the share: tiles [t0, t1) of an item.
struct Piece {
  int head;
  int t0, t1;
  bool whole, starts;  // the whole item; the piece holds the item's first tile
  int c0, parts;       // block in which the item starts, and its parts
};

// Moves to the share's next piece (entry in `en`); false at its end.  Tile t
// of an item is unit OVER + t: a share that holds only the first OVER units
// of an item has no piece of it.
template <int ROWS, int TILE, int OVER>
__device__ __forceinline__ bool next_piece(const AttendArgs &p, const WorkGrid &g, Share &o, Entry &en, Piece &q) {
  while (o.pos < o.end) {
    if (!get_entry<ROWS, TILE>(p, g, o.e, en)) {
      o.e = (en.i + 1) * g.per_seq;  // the sequence has no more rows
      continue;
    }
    const int steps = en.steps(), cost = OVER + steps;
    const int64_t n = (int64_t)cost * p.c.kv;
    if (o.pos >= o.at + n) {
      o.at += n;
      o.e++;
      continue;
    }
    q.head = (int)((uint32_t)(o.pos - o.at) / (uint32_t)cost);
    const int64_t s0 = o.at + (int64_t)q.head * cost + OVER;  // unit of tile 0
    const int64_t end = o.end < s0 + steps ? o.end : s0 + steps;
    q.t0 = o.pos > s0 ? (int)(o.pos - s0) : 0;
    q.t1 = (int)(end - s0);
    o.pos = end;
    if (q.t1 <= q.t0) continue;
    q.starts = q.t0 == 0;
    q.whole = q.starts && q.t1 == steps;
    q.c0 = q.starts ? (int)blockIdx.x : block_of(s0, o.total, o.blocks);
    q.parts = (q.t1 == steps ? (int)blockIdx.x : block_of(s0 + steps - 1, o.total, o.blocks)) - q.c0 + 1;
    return true;
  }
  return false;
}

// Workspace slot of part k of the item that starts in block c0.
__device__ __forceinline__ int part_slot(int c0, int k) { return k == 0 ? 2 * c0 + 1 : 2 * (c0 + k); }

// Bytes (0, 1) or (2, 3) of a word of codes, each with its top bit flipped
// (code + 128), as two f16: 0x6400 | u is 1024 + u.
__device__ __forceinline__ uint32_t two_f16(uint32_t w, uint32_t sel) {
  const uint32_t u = __byte_perm(w, 0x64646464u, sel);
  const __half2 h = __hsub2(*reinterpret_cast<const __half2 *>(&u), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t *>(&h);
}
constexpr uint32_t kLow = 0x4140, kHigh = 0x4342;

__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float log2_approx(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;constexpr int kMaxBlocks = 4096;  // counters at the start of the workspace

}  // namespace kv8
}  // namespace sc
