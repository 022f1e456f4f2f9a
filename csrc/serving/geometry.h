// Which rows, tokens and pages a workgroup has. Plain arithmetic, for the
// kernels and for host checks of it: no result points outside the arrays that
// its arguments describe, whatever `starts`, `lens` and `table` hold.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "serving.h"

namespace serving {

constexpr int kTile = 64;  // tokens that a wave takes at once

// The last of 0 .. count - 1 whose first(i) is not over `at`; 0 if there is
// none. first() does not fall. On the device all lanes of a wave ask for the
// same: few places are counted at once, since each step of a search waits for
// memory.
template <typename First>
__host__ __device__ inline int last_at_most(int count, int64_t at, First first) {
#if defined(__HIP_DEVICE_COMPILE__)
  if (count <= 512) {
    int found = 0;
    for (int i = 0; i < count; i += 64) {
      const int lane = i + (threadIdx.x & 63);
      found += __popcll(__ballot(lane < count && first(lane < count ? lane : 0) <= at));
    }
    return found > 0 ? found - 1 : 0;
  }
#endif
  int lo = 0, hi = count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first(mid) <= at) lo = mid; else hi = mid;
  }
  return lo;
}

// ---- attention -------------------------------------------------------------

// Rows of a sequence are (token, head) pairs, `row_tile` of them a workgroup.
struct Place {
  int b, row0, count, len;  // sequence (batch: the rows behind the last one), its first row, its rows' tokens, its length
  int tile, local, rows;    // which tile, its first (token, head) row, rows in it
  int first, last;          // positions of the first and the last of them
  int lo, hi, splits;       // tokens seen: [lo, hi); workgroups with any
  bool broken;              // longer than its row of the table: its results are NaN
  bool keep;                // rows behind the last sequence whose output stays as it was
};

// Rows of a tile are a power of two.
__host__ __device__ inline int tile_shift(const AttentionArgs& a) { return __builtin_ctz(a.row_tile); }

// Where sequences have few rows, each has `per` slots. Otherwise those of
// sequence b start at starts[b] group / row_tile + b: enough for its tiles,
// whatever the lengths, and a rule that a search can invert.
__host__ __device__ inline int64_t first_slot(const AttentionArgs& a, int group, int b) {
  return ((int64_t)a.c.starts[b] * group >> tile_shift(a)) + b;
}

__host__ __device__ inline int64_t slot_count(const AttentionArgs& a) {
  const int group = a.q_heads / a.c.heads;
  if (a.per) return (int64_t)a.c.batch * a.per;
  return ((int64_t)a.c.rows * group >> tile_shift(a)) + a.c.batch + 1;
}

// The rest of `p` from b, count and tile.
__host__ __device__ inline void fill_place(const AttentionArgs& a, int group, Place& p) {
  const int room = a.c.blocks * a.c.page;
  p.len = p.b < a.c.batch ? a.c.lens[p.b] : 0;
  p.broken = p.len > room;
  if (p.broken) p.len = room;
  if (p.len < 0) p.len = 0;
  p.local = p.tile * a.row_tile;
  const int all = p.count * group;
  p.rows = all - p.local < a.row_tile ? all - p.local : a.row_tile;
  const int before = p.len - p.count;
  p.first = before + p.local / group;
  p.last = before + (p.local + p.rows - 1) / group;
  p.hi = p.last + 1 > 0 ? p.last + 1 : 0;
  p.lo = a.window && p.first - a.window + 1 > 0 ? p.first - a.window + 1 : 0;
  const int start = p.lo & ~(kTile - 1);
  const int n = p.hi > start ? (int)((uint32_t)(p.hi - start - 1) / (uint32_t)a.chunk) + 1 : 1;
  p.splits = n < a.splits ? n : a.splits;
}

// The rows of sequence p.b; false if it has none.
__host__ __device__ inline bool rows_of(const CacheArgs& c, Place& p) {
  if (!c.starts) {
    p.row0 = p.b;
    p.count = 1;
    return p.b < c.rows;
  }
  p.row0 = c.starts[p.b];
  const int next = p.b < c.batch ? c.starts[p.b + 1] : c.rows;
  if (p.row0 < 0 || next <= p.row0 || next > c.rows) return false;
  p.count = next - p.row0;
  return true;
}

// Whether a pass takes a sequence of `count` tokens.
__host__ __device__ inline bool takes(const AttentionArgs& a, int group, int count) {
  const int64_t rows = (int64_t)count * group;
  return rows > a.few && rows <= a.many;
}

// The tile of a slot; false if it has none.
__host__ __device__ inline bool place_of_slot(const AttentionArgs& a, int group, int slot, Place& p) {
  const CacheArgs& c = a.c;
  if (a.per) {
    p.b = slot / a.per;
    p.tile = slot - p.b * a.per;
  } else {
    p.b = last_at_most(c.batch + 1, slot, [&](int i) { return first_slot(a, group, i); });
    const int64_t tile = slot - first_slot(a, group, p.b);
    if (tile < 0 || tile > 0x7FFFFFFF) return false;
    p.tile = (int)tile;
  }
  if (!rows_of(c, p)) return false;
  if ((int64_t)p.tile * a.row_tile >= (int64_t)p.count * group) return false;
  if (p.b == c.batch ? a.tail == kLeaveTail : !takes(a, group, p.count)) return false;
  p.keep = p.b == c.batch && a.tail == kTailLse;
  fill_place(a, group, p);
  return true;
}

// ---- append ----------------------------------------------------------------

// A page that gets tokens: its slots [from, to) get rows src, src + 1, ...
struct PageWrite {
  int pid, from, to, src;
};

// Slots of sequence b start at starts[b] / page + 2 b.
__host__ __device__ inline int64_t append_slots(const CacheArgs& c) {
  return c.starts ? (int64_t)c.rows / c.page + 2 * (int64_t)c.batch : c.batch;
}

__host__ __device__ inline bool page_of_slot(const CacheArgs& c, int slot, PageWrite& w) {
  int b, row0, count, nth;
  if (c.starts) {
    b = last_at_most(c.batch, slot, [&](int i) { return (int64_t)c.starts[i] / c.page + 2 * i; });
    row0 = c.starts[b];
    const int next = c.starts[b + 1];
    if (row0 < 0 || next <= row0 || next > c.rows) return false;
    count = next - row0;
    nth = slot - (row0 / c.page + 2 * b);
    if (nth < 0) return false;
  } else {
    b = row0 = slot;
    count = 1;
    nth = 0;
  }
  const int len = c.lens[b];
  if (len <= 0) return false;
  const int first = len - count;  // position of the first new token
  const int begin = first > 0 ? first : 0;
  const int block = begin / c.page + nth;
  if (block > (len - 1) / c.page || block >= c.blocks) return false;
  w.pid = c.table[b * c.ldt + block];
  if (w.pid < 0 || w.pid >= c.pages) return false;
  const int base = block * c.page;
  w.from = begin > base ? begin - base : 0;
  w.to = len - base < c.page ? len - base : c.page;
  w.src = row0 + base + w.from - first;
  return true;
}

}  // namespace serving
