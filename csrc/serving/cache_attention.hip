// Attention over a paged cache held in 8 bits (e4m3, one scale for each page
// and head), for single tokens and for chunks of tokens:
//
//   s_j = c q . K_j ks_j,  out = sum_j softmax(s)_j V_j vs_j,  lse = log sum e^s
//
// over the positions j that a row sees: up to its own, and not further back
// than the window. Bound by the bytes of the cached codes for single tokens,
// by the matrix instructions for long chunks.
//
// Both products are formed transposed, so that no operand crosses lanes:
// S^T = K Q^T leaves query row l % 16 and tokens 16 (l / 16) .. + 15 of 64 in
// lane l, since the rows of K that a matrix instruction takes are chosen as
// tokens 16 a + 8 c + 4 h + i (a, i: the lane's row 4 a + i). This is just the
// order in which O^T = V^T P^T takes its second operand, and a lane's running
// maximum and its factors belong to its own query row. Keys lie [token][dim]
// and values [dim][token], so that both are read 16 bytes a lane.
//
// Codes become q's type for the scores and fp16 for the values: both hold e4m3
// exactly. The weights are rounded to fp16 (2^-11; bf16 would show in bf16
// results). They are p vs over a reference that follows the largest p vs so far,
// so that weights down to 2^-21 of it keep their 11 bits: a context may be
// shared by a million tokens beside a single large one. Sums are fp32.
//
// Of few rows, a workgroup's 4 waves take turns at tiles of 64 tokens and join
// in LDS; of many, they have rows of their own and share the tiles. Long
// contexts are split over workgroups in chunks of a fixed number of tokens, whose
// results a second launch joins in their order.
//
// Measured, kernel and join: 64 contexts of 8000 to 16384 tokens, 64 heads on 8 of
// 128: 275 + 6 us, 5.7 TB/s of the 6.3 that a plain read reaches (all heads of a
// page on one die took it from 323 to 302, fewer workgroups to 280: split()); 32
// of up to 4100 tokens: 32 + 3 us, bound by the latency of a workgroup's few tiles. A
// prompt of 4096 causal tokens, 32 heads on 8: 215 us, 0.64 PFLOP/s; 4 chunks of 512
// tokens on 8192: 304 us, 0.88 PFLOP/s, bound by the vector unit's share of the
// softmax beside the matrix instructions.
#include <type_traits>

#include "device.h"
#include "geometry.h"
#include "serving.h"

namespace serving {
namespace {

constexpr int kWaves = 4;

template <typename T>
struct Codes;
template <>
struct Codes<__bf16> {
  static __device__ __forceinline__ bf16x8 widen(uint32_t lo, uint32_t hi) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false);
    const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false);
    const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  }
};
template <>
struct Codes<_Float16> {
  static __device__ __forceinline__ f16x8 widen(uint32_t lo, uint32_t hi) {
    const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, false);
    const f16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, true);
    const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, false);
    const f16x2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, true);
    return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  }
};

// 0xFF in the bytes below the n-th of a dword.
__device__ __forceinline__ uint32_t bytes_below(int n) {
  return n <= 0 ? 0u : n >= 4 ? ~0u : (1u << (8 * n)) - 1u;
}
// 0x80 in the bytes that hold e4m3's NaN.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {
  return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
}

template <typename T>
__device__ __forceinline__ void store4(T* to, f32x4 v) {
  typedef T t4 __attribute__((ext_vector_type(4)));
  t4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = (T)v[i];
  *reinterpret_cast<t4*>(to) = r;
}

// How a lane's 16 tokens, all of one page, weigh in: a score's power of two is
// unit q . K + log, with the value's scale in it, and `back` takes that out of
// the sum again. The scale of a page that no row sees (not `within`) is left out:
// it may be anything, and a score of -inf would not keep it from the sum.
struct Weighing {
  float unit, log, back;
  __device__ __forceinline__ Weighing(bool known, bool within, float ks, float vs, float scale) {
    unit = known ? ks * scale * kLog2e : __builtin_nanf("");
    const float v = known && within ? vs : 1.f;
    log = __builtin_amdgcn_logf(v);
    back = 1.f / v;
  }
};

// What weights are relative to, in powers of two: 2^7 under the largest so far
// when it moves, and it moves only where a weight would pass 2^15. So the largest
// weights fill fp16's range (65504), and those with 11 bits reach down to 2^-21 of
// the largest, with fewer bits to 2^-31.
__device__ __forceinline__ float reference(float top, float best) {
  return best > top + 15.f ? best - 7.f : top;
}

// Codes that one workgroup reads once pass by the L2.
template <int QT>
__device__ __forceinline__ u32x4 load16(const uint8_t* p) {
  if constexpr (QT == 1) return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
  return *reinterpret_cast<const u32x4*>(p);
}

// The same number, but one that the compiler does not know to be: what depends
// on it is worked out where it stands, not ahead of a loop, where it would take
// more scalar registers than there are.
__device__ __forceinline__ int anew(int v) {
  asm volatile("" : "+s"(v));
  return v;
}

constexpr int waves_of(int dt, int qt) { return dt * qt <= 4 ? 3 : dt * qt <= 8 ? 2 : 1; }

// DT tiles of 16 dimensions, all of them there if kWhole; QT tiles of 16 query
// rows.
template <typename T, int DT, int QT, bool kWhole>
__global__ __launch_bounds__(kWaves * 64, waves_of(DT, QT)) void attention_kernel(AttentionArgs a) {
  using x8 = typename Mat<T>::x8;
  constexpr int KB = DT / 4;  // blocks of 64 dimensions
  const CacheArgs& c = a.c;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, g = lane >> 4;
  const int group = a.q_heads / c.heads;
  // Workgroups go to the 8 dies in turn. All heads of a slot and split follow
  // one another on one die: their codes are neighbours in every page.
  const int turn = blockIdx.x >> 3, h = turn % c.heads;
  const int64_t job = (int64_t)(turn / c.heads) * 8 + (blockIdx.x & 7);
  const int slots = (int)slot_count(a);
  const int split = (int)(job / slots), slot = (int)(job - (int64_t)split * slots);
  if (split >= a.splits) return;

  Place p;
  if (!place_of_slot(a, group, slot, p)) return;
  if (split >= p.splits) return;

  const int page = c.page, dim = kWhole ? DT * 16 : c.dim;
  const int shift = 31 - __clz(page);
  const int begin = (p.lo & ~(kTile - 1)) + split * a.chunk;
  const int end = split == p.splits - 1 || begin + a.chunk > p.hi ? p.hi : begin + a.chunk;
  const int32_t* table = c.table + (p.b < c.batch ? p.b * c.ldt : 0);

  // the lane's query rows, their positions, and their operands
  x8 q[QT][KB * 2];
  int pos[QT], low[QT];  // a row sees the positions low + 1 .. pos
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int i = t * 16 + r < p.rows ? t * 16 + r : p.rows - 1;
    const int tok = (p.local + i) / group, head = h * group + (p.local + i) % group;
    pos[t] = p.len - p.count + tok;
    low[t] = a.window ? pos[t] - a.window : -1;
    const T* src = (const T*)a.q + (int64_t)(p.row0 + tok) * a.q_row + head * a.q_head;
#pragma unroll
    for (int k = 0; k < KB * 2; ++k) {
      const int d = (k >> 1) * 64 + g * 16 + (k & 1) * 8;
      q[t][k] = bits_as<x8>(u32x4{0, 0, 0, 0});
      if (kWhole || d < dim) q[t][k] = *reinterpret_cast<const x8*>(src + d);
    }
  }

  f32x4 acc[QT][DT];
  float top[QT], sum[QT];
  // Keys of the next tile come while this one's weights are formed, and this
  // tile's values while its scores are: each takes the registers that the other
  // has left. Page numbers come a tile ahead of the keys.
  struct Pages {
    int pid;     // of the lane's 16 tokens, within range
    bool known;  // whether it was; if not, what sees it is NaN
  };
  auto look_up = [&](int base) {
    const int blk = (base + g * 16) >> shift;
    const int pid = table[blk < c.blocks ? blk : c.blocks - 1];
    const bool known = blk < c.blocks && (uint32_t)pid < (uint32_t)c.pages && !p.broken;
    return Pages{(uint32_t)pid < (uint32_t)c.pages ? pid : 0, known};
  };
  u32x4 kr[4][KB], vr[DT];
  float ks, vs;
  auto load_keys = [&](int base, const Pages& at) {
    const int dim = kWhole ? DT * 16 : anew(c.dim);
    const int pid = __shfl(at.pid, (r >> 2) << 4);
    const int tok = ((base + ((r >> 2) << 4)) & (page - 1)) + (r & 3);
    const uint8_t* from = c.k + (((int64_t)pid * c.heads + h) * page + tok) * dim + g * 16;
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
      for (int k = 0; k < KB; ++k) {
        // lanes past the last dimension, where the queries are 0, read the same
        // token's first ones: another's NaN would not stay with it
        const uint8_t* here = from + m * 4 * dim + (kWhole || k * 64 + g * 16 < dim ? k * 64 : -g * 16);
        kr[m][k] = *reinterpret_cast<const u32x4*>(here);
      }
    const int64_t ph = (int64_t)at.pid * c.heads + h;
    ks = c.k_scale[ph];
    vs = c.v_scale[ph];
  };
  auto load_values = [&](int base, const Pages& at) {
    const int dim = kWhole ? DT * 16 : anew(c.dim), page = anew(c.page);
    const uint8_t* from = c.v + (((int64_t)at.pid * c.heads + h) * dim + r) * page + ((base + g * 16) & (page - 1));
#pragma unroll
    for (int d = 0; d < DT; ++d)
      vr[d] = load16<QT>(from + (kWhole ? d : min(d, (dim >> 4) - 1)) * 16 * page);
  };

  // Takes the wave's tiles. A tile at the edge of what the rows see may hold
  // NaN among the values of some of them: then `sweep` says so, and the second
  // form, which keeps a NaN from the rows that do not see it, starts over.
  auto sweep = [&](auto careful) {
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      top[t] = -kInf;
      sum[t] = 0.f;
#pragma unroll
      for (int d = 0; d < DT; ++d) acc[t][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    int base = begin + wave * kTile;
    if (base >= end) return false;
    bool odd = false;
    Pages here = look_up(base);
    load_keys(base, here);
    Pages next = look_up(base + kWaves * kTile < end ? base + kWaves * kTile : base);
#pragma unroll 1
    for (; base < end; base += kWaves * kTile) {
      const int tok0 = base + g * 16;  // the lane's 16 tokens for P and V
      load_values(base, here);
      Weighing by(here.known, tok0 < end && tok0 + 16 > p.lo, ks, vs, a.scale);

      f32x4 s[QT][4] = {};
#pragma unroll
      for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int k = 0; k < KB; ++k) {
          const x8 lo = Codes<T>::widen(kr[m][k][0], kr[m][k][1]), hi = Codes<T>::widen(kr[m][k][2], kr[m][k][3]);
#pragma unroll
          for (int t = 0; t < QT; ++t) {
            s[t][m] = Mat<T>::mfma(lo, q[t][2 * k], s[t][m]);
            s[t][m] = Mat<T>::mfma(hi, q[t][2 * k + 1], s[t][m]);
          }
        }
      const int ahead = base + kWaves * kTile < end ? base + kWaves * kTile : base;  // the last reads its own again
      load_keys(ahead, next);
      here = next;
      next = look_up(ahead + kWaves * kTile < end ? ahead + kWaves * kTile : ahead);

      const bool edge = base + kTile > p.first + 1 || (a.window && base <= p.last - a.window);
      if (edge) {
#pragma unroll
        for (int t = 0; t < QT; ++t)
#pragma unroll
          for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int j = tok0 + m * 4 + i;
              const bool in = (j <= pos[t]) & (j > low[t]);
              s[t][m][i] = in ? s[t][m][i] * by.unit : -kInf;
            }
        by.unit = 1.f;  // masked behind the unit: an unknown page's NaN stays with the rows that see it
      }
      f16x8 pw[QT][2];
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        float best = -kInf;
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
          for (int i = 0; i < 4; ++i) best = fmaxf(best, s[t][m][i]);
        best = __builtin_fmaf(best, by.unit, by.log);
        best = fmaxf(best, __shfl_xor(best, 16));
        best = fmaxf(best, __shfl_xor(best, 32));
        const float now = reference(top[t], best);
        if (__any(now != top[t])) {
          const float f = now == -kInf ? 0.f : __builtin_amdgcn_exp2f(top[t] - now);
          sum[t] *= f;
#pragma unroll
          for (int d = 0; d < DT; ++d) acc[t][d] *= f;
          top[t] = now;
        }
        const float off = by.log - (now == -kInf ? 0.f : now);
        float part = 0.f;
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][m][i], by.unit, off));
            part += e;
            pw[t][m >> 1][(m & 1) * 4 + i] = (_Float16)e;
          }
        sum[t] = __builtin_fmaf(part, by.back, sum[t]);
      }
      if (edge) {
        // values that no row sees are whatever the page held before
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t keep = bytes_below(p.hi - tok0 - 4 * w) & ~bytes_below(p.lo - tok0 - 4 * w);
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            vr[d][w] &= keep;
            odd |= nan_bytes(vr[d][w]) != 0;
          }
        }
        if constexpr (careful) {
          f16x8 seen[QT][2];
#pragma unroll
          for (int t = 0; t < QT; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i)
              seen[t][i >> 3][i & 7] = (tok0 + i <= pos[t]) & (tok0 + i > low[t]) ? (_Float16)1.f : (_Float16)0.f;
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            f32x4 hits[QT] = {};
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const uint32_t w0 = nan_bytes(vr[d][2 * x]) >> 7, w1 = nan_bytes(vr[d][2 * x + 1]) >> 7;
              vr[d][2 * x] &= ~(w0 * 0xFFu);
              vr[d][2 * x + 1] &= ~(w1 * 0xFFu);
              f16x8 is;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                is[i] = (_Float16)(float)(w0 >> (8 * i) & 1u);
                is[4 + i] = (_Float16)(float)(w1 >> (8 * i) & 1u);
              }
#pragma unroll
              for (int t = 0; t < QT; ++t) hits[t] = Mat<_Float16>::mfma(is, seen[t][x], hits[t]);
            }
#pragma unroll
            for (int t = 0; t < QT; ++t)
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (hits[t][i] > 0.f) acc[t][d][i] = __builtin_nanf("");
          }
        }
      }
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const f16x8 v = Codes<_Float16>::widen(vr[d][2 * x], vr[d][2 * x + 1]);
#pragma unroll
          for (int t = 0; t < QT; ++t) acc[t][d] = Mat<_Float16>::mfma(v, pw[t][x], acc[t][d]);
        }
    }
    return __any(odd) != 0;
  };
  if (sweep(std::false_type{})) sweep(std::true_type{});

  // the waves' parts: against one reference, then summed in the waves' order
  __shared__ float tops[kWaves][QT][16], sums[kWaves][QT][16];
  __shared__ f32x4 part[kWaves][DT][64];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    sum[t] += __shfl_xor(sum[t], 16);
    sum[t] += __shfl_xor(sum[t], 32);
    if (g == 0) {
      tops[wave][t][r] = top[t];
      sums[wave][t][r] = sum[t];
    }
  }
  __syncthreads();
  const bool whole = p.splits == 1;
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    float all = tops[0][t][r];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) all = fmaxf(all, tops[w][t][r]);
    const float ref = all == -kInf ? 0.f : all;
    float total = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) total += sums[w][t][r] * __builtin_amdgcn_exp2f(tops[w][t][r] - ref);
    if (p.broken) total = __builtin_nanf("");
    const float f = __builtin_amdgcn_exp2f(top[t] - ref);
    if (t) __syncthreads();
#pragma unroll
    for (int d = 0; d < DT; ++d) part[wave][d][lane] = acc[t][d] * f;
    __syncthreads();
    const int i = t * 16 + r;
    if (i < p.rows) {
      const int tok = (p.local + i) / group, head = h * group + (p.local + i) % group;
      if (whole) {
        const float inv = total != 0.f ? 1.f / total : 0.f;
        T* out = (T*)a.out + (int64_t)(p.row0 + tok) * a.o_row + head * a.o_head + g * 4;
#pragma unroll
        for (int d = wave; d < DT; d += kWaves) {
          f32x4 o = part[0][d][lane];
#pragma unroll
          for (int w = 1; w < kWaves; ++w) o += part[w][d][lane];
          if ((kWhole || d * 16 < dim) && !p.keep) store4(out + d * 16, o * inv);
        }
        if (wave == 0 && g == 0)
          a.lse[(int64_t)(p.row0 + tok) * a.q_heads + head] = (all + __builtin_amdgcn_logf(total)) * kLn2;
      } else {
        float* to = a.work + (((int64_t)slot * c.heads + h) * a.splits + split) * a.row_tile * (dim + 2);
        float* row = to + (int64_t)i * dim + g * 4;
#pragma unroll
        for (int d = wave; d < DT; d += kWaves) {
          f32x4 o = part[0][d][lane];
#pragma unroll
          for (int w = 1; w < kWaves; ++w) o += part[w][d][lane];
          if (kWhole || d * 16 < dim) *reinterpret_cast<f32x4*>(row + d * 16) = o;
        }
        if (wave == 0 && g == 0) {
          to[(int64_t)a.row_tile * dim + 2 * i] = all;
          to[(int64_t)a.row_tile * dim + 2 * i + 1] = total;
        }
      }
    }
  }
}

// Many rows: 4 waves with 32 rows each share the tiles of 64 tokens. A wave
// fetches and widens a quarter of a tile, in the order of the matrix
// instruction's operands, into one half of the LDS while all work on the other.
// So codes are read and widened once for 128 rows; a tile then costs a wave 32
// LDS reads of 1 KB for 64 matrix instructions, about the same time each.
template <int DT>
struct Staged {
  static constexpr int kKeys = DT * 2, kValues = DT * 2;  // operands of 1 KB
  static constexpr int kHalf = (kKeys + kValues) * 64;    // in 16 bytes
  static constexpr size_t kBytes = 2 * (size_t)kHalf * 16;
};

template <typename T, int DT, bool kWhole>
__global__ __launch_bounds__(kWaves * 64, DT <= 8 ? 2 : 1) void attention_rows_kernel(AttentionArgs a) {
  using x8 = typename Mat<T>::x8;
  constexpr int KB = DT / 4, QT = 2, VQ = DT / kWaves;
  extern __shared__ u32x4 staged[];
  __shared__ int flagged;
  const CacheArgs& c = a.c;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, g = lane >> 4;
  const int group = a.q_heads / c.heads;
  const int turn = blockIdx.x >> 3, h = turn % c.heads;
  const int64_t job = (int64_t)(turn / c.heads) * 8 + (blockIdx.x & 7);
  const int slots = (int)slot_count(a);
  const int split = (int)(job / slots), slot = (int)(job - (int64_t)split * slots);
  if (split >= a.splits) return;
  Place p;
  if (!place_of_slot(a, group, slot, p)) return;
  if (split >= p.splits) return;

  const int page = c.page, dim = kWhole ? DT * 16 : c.dim;
  const int shift = 31 - __clz(page);
  const int begin = (p.lo & ~(kTile - 1)) + split * a.chunk;
  const int end = split == p.splits - 1 || begin + a.chunk > p.hi ? p.hi : begin + a.chunk;
  const int32_t* table = c.table + (p.b < c.batch ? p.b * c.ldt : 0);

  x8 q[QT][KB * 2];
  int pos[QT], low[QT];
  const int mine = wave * 32;  // the wave's first row of the tile
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int i = mine + t * 16 + r < p.rows ? mine + t * 16 + r : p.rows - 1;
    const int tok = (p.local + i) / group, head = h * group + (p.local + i) % group;
    pos[t] = p.len - p.count + tok;
    low[t] = a.window ? pos[t] - a.window : -1;
    const T* src = (const T*)a.q + (int64_t)(p.row0 + tok) * a.q_row + head * a.q_head;
#pragma unroll
    for (int k = 0; k < KB * 2; ++k) {
      const int d = (k >> 1) * 64 + g * 16 + (k & 1) * 8;
      q[t][k] = bits_as<x8>(u32x4{0, 0, 0, 0});
      if (kWhole || d < dim) q[t][k] = *reinterpret_cast<const x8*>(src + d);
    }
  }
  // what the wave's rows see: nothing for a wave without rows
  const int last_row = mine + 31 < p.rows ? mine + 31 : p.rows - 1;
  const int w_first = p.len - p.count + (p.local + mine) / group;
  const int w_last = mine < p.rows ? p.len - p.count + (p.local + last_row) / group : -1;
  const int w_low = a.window ? w_first - a.window : -1;  // positions up to it are seen by none

  f32x4 acc[QT][DT];
  float top[QT], sum[QT];
  u32x4 kr[KB], vr[VQ];
  float ks, vs, ks_next, vs_next;
  bool known, known_next;
  auto look_up = [&](int base, bool& is) {
    const int blk = (base + g * 16) >> shift;
    const int pid = table[blk < c.blocks ? blk : c.blocks - 1];
    is = blk < c.blocks && (uint32_t)pid < (uint32_t)c.pages && !p.broken;
    return (uint32_t)pid < (uint32_t)c.pages ? pid : 0;
  };
  // the wave's quarter: token rows m = wave of the keys, VQ tiles of dimensions
  auto fetch = [&](int base, int pid) {
    const int pid_k = __shfl(pid, (r >> 2) << 4);
    const int tok = ((base + ((r >> 2) << 4)) & (page - 1)) + (r & 3) + wave * 4;
    const uint8_t* key = c.k + (((int64_t)pid_k * c.heads + h) * page + tok) * dim;
#pragma unroll
    for (int k = 0; k < KB; ++k)
      kr[k] = *reinterpret_cast<const u32x4*>(key + (kWhole || k * 64 + g * 16 < dim ? k * 64 + g * 16 : 0));
    const uint8_t* value = c.v + (((int64_t)pid * c.heads + h) * dim + r) * page + ((base + g * 16) & (page - 1));
#pragma unroll
    for (int d = 0; d < VQ; ++d)
      vr[d] = *reinterpret_cast<const u32x4*>(value + (kWhole || (wave * VQ + d) * 16 < dim ? wave * VQ + d : 0) * 16 * page);
    const int64_t ph = (int64_t)pid * c.heads + h;
    ks_next = c.k_scale[ph];
    vs_next = c.v_scale[ph];
  };

  auto sweep = [&](auto careful) {
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      top[t] = -kInf;
      sum[t] = 0.f;
#pragma unroll
      for (int d = 0; d < DT; ++d) acc[t][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    bool odd = false;
    // Values that no row sees become 0; NaN among the others is told, and in the
    // careful form taken out.
    auto put = [&](int base, int half) {
      u32x4* to = staged + half * Staged<DT>::kHalf;
#pragma unroll
      for (int k = 0; k < KB; ++k) {
        to[((wave * KB + k) * 2) * 64 + lane] = bits_as<u32x4>(Codes<T>::widen(kr[k][0], kr[k][1]));
        to[((wave * KB + k) * 2 + 1) * 64 + lane] = bits_as<u32x4>(Codes<T>::widen(kr[k][2], kr[k][3]));
      }
      to += Staged<DT>::kKeys * 64;
      if (base + kTile > p.first + 1 || (a.window && base <= p.last - a.window)) {
        const int tok0 = base + g * 16;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t keep = bytes_below(p.hi - tok0 - 4 * w) & ~bytes_below(p.lo - tok0 - 4 * w);
#pragma unroll
          for (int d = 0; d < VQ; ++d) {
            vr[d][w] &= keep;
            const uint32_t nan = nan_bytes(vr[d][w]);
            odd |= nan != 0;
            if constexpr (careful) vr[d][w] &= ~((nan >> 7) * 0xFFu);
          }
        }
      }
#pragma unroll
      for (int d = 0; d < VQ; ++d)
#pragma unroll
        for (int x = 0; x < 2; ++x)
          to[((wave * VQ + d) * 2 + x) * 64 + lane] =
              bits_as<u32x4>(Codes<_Float16>::widen(vr[d][2 * x], vr[d][2 * x + 1]));
    };

    if (begin < end) {
      int pid = look_up(begin, known_next);
      fetch(begin, pid);
      int beyond = begin + kTile < end ? begin + kTile : begin;
      bool known_beyond;
      pid = look_up(beyond, known_beyond);
      put(begin, 0);
      ks = ks_next, vs = vs_next, known = known_next;
      __syncthreads();
      int half = 0;
#pragma unroll 1
      for (int base = begin; base < end; base += kTile, half ^= 1) {
        const bool more = base + kTile < end;
        fetch(beyond, pid);  // the last tile is fetched again and left
        known_next = known_beyond;
        const int next = beyond;
        beyond = beyond + kTile < end ? beyond + kTile : beyond;
        pid = look_up(beyond, known_beyond);
        const u32x4* at = staged + half * Staged<DT>::kHalf + lane;

        if (base <= w_last && base + kTile - 1 > w_low) {
          const int tok0 = base + g * 16;
          Weighing by(known, tok0 < end && tok0 + 16 > p.lo, ks, vs, a.scale);
          f32x4 s[QT][4] = {};
#pragma unroll
          for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int k = 0; k < KB * 2; ++k) {
              const x8 key = bits_as<x8>(at[(m * KB * 2 + k) * 64]);
#pragma unroll
              for (int t = 0; t < QT; ++t) s[t][m] = Mat<T>::mfma(key, q[t][k], s[t][m]);
            }
          if (base + kTile > w_first + 1 || (a.window && base <= w_last - a.window)) {
#pragma unroll
            for (int t = 0; t < QT; ++t)
#pragma unroll
              for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const int j = tok0 + m * 4 + i;
                  const bool in = (j <= pos[t]) & (j > low[t]);
                  s[t][m][i] = in ? s[t][m][i] * by.unit : -kInf;
                }
            by.unit = 1.f;
          }
          f16x8 pw[QT][2];
#pragma unroll
          for (int t = 0; t < QT; ++t) {
            float best = -kInf;
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
              for (int i = 0; i < 4; ++i) best = fmaxf(best, s[t][m][i]);
            best = __builtin_fmaf(best, by.unit, by.log);
            best = fmaxf(best, __shfl_xor(best, 16));
            best = fmaxf(best, __shfl_xor(best, 32));
            const float now = reference(top[t], best);
            if (__any(now != top[t])) {
              const float f = now == -kInf ? 0.f : __builtin_amdgcn_exp2f(top[t] - now);
              sum[t] *= f;
#pragma unroll
              for (int d = 0; d < DT; ++d) acc[t][d] *= f;
              top[t] = now;
            }
            const float off = by.log - (now == -kInf ? 0.f : now);
            float part = 0.f;
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][m][i], by.unit, off));
                part += e;
                pw[t][m >> 1][(m & 1) * 4 + i] = (_Float16)e;
              }
            sum[t] = __builtin_fmaf(part, by.back, sum[t]);
          }
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const f16x8 v = bits_as<f16x8>(at[(Staged<DT>::kKeys + d * 2 + x) * 64]);
#pragma unroll
              for (int t = 0; t < QT; ++t) acc[t][d] = Mat<_Float16>::mfma(v, pw[t][x], acc[t][d]);
            }
          if constexpr (careful) {
            // which rows see a NaN among this tile's values, from the page itself
#pragma unroll 1
            for (int d = 0; d < DT; ++d) {
              if (d * 16 >= dim) break;
              bool is;
              const int here = look_up(base, is);
              const u32x4 raw = *reinterpret_cast<const u32x4*>(
                  c.v + (((int64_t)here * c.heads + h) * dim + d * 16 + r) * page + (tok0 & (page - 1)));
              f32x4 hits[QT] = {};
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                const uint32_t w0 = nan_bytes(raw[2 * x]) >> 7, w1 = nan_bytes(raw[2 * x + 1]) >> 7;
                f16x8 bad;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  bad[i] = (_Float16)(float)(w0 >> (8 * i) & 1u);
                  bad[4 + i] = (_Float16)(float)(w1 >> (8 * i) & 1u);
                }
#pragma unroll
                for (int t = 0; t < QT; ++t) {
                  f16x8 seen;
#pragma unroll
                  for (int i = 0; i < 8; ++i) {
                    const int j = tok0 + x * 8 + i;
                    seen[i] = (j <= pos[t]) & (j > low[t]) ? (_Float16)1.f : (_Float16)0.f;
                  }
                  hits[t] = Mat<_Float16>::mfma(bad, seen, hits[t]);
                }
              }
#pragma unroll
              for (int dd = 0; dd < DT; ++dd)
                if (dd == d)
#pragma unroll
                  for (int t = 0; t < QT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                      if (hits[t][i] > 0.f) acc[t][dd][i] = __builtin_nanf("");
            }
          }
        }
        if (more) put(next, half ^ 1);
        ks = ks_next, vs = vs_next, known = known_next;
        __syncthreads();
      }
    }
    return odd;
  };

  if (threadIdx.x == 0) flagged = 0;
  __syncthreads();
  if (__any(sweep(std::false_type{})) && lane == 0) flagged = 1;
  __syncthreads();
  if (flagged) sweep(std::true_type{});

#pragma unroll
  for (int t = 0; t < QT; ++t) {
    sum[t] += __shfl_xor(sum[t], 16);
    sum[t] += __shfl_xor(sum[t], 32);
    if (p.broken) sum[t] = __builtin_nanf("");
    const int i = mine + t * 16 + r;
    if (i >= p.rows) continue;
    if (p.splits == 1) {
      const int tok = (p.local + i) / group, head = h * group + (p.local + i) % group;
      const float inv = sum[t] != 0.f ? 1.f / sum[t] : 0.f;
      T* out = (T*)a.out + (int64_t)(p.row0 + tok) * a.o_row + head * a.o_head + g * 4;
#pragma unroll
      for (int d = 0; d < DT; ++d)
        if ((kWhole || d * 16 < dim) && !p.keep) store4(out + d * 16, acc[t][d] * inv);
      if (g == 0) a.lse[(int64_t)(p.row0 + tok) * a.q_heads + head] = (top[t] + __builtin_amdgcn_logf(sum[t])) * kLn2;
    } else {
      float* to = a.work + (((int64_t)slot * c.heads + h) * a.splits + split) * a.row_tile * (dim + 2);
      float* row = to + (int64_t)i * dim + g * 4;
#pragma unroll
      for (int d = 0; d < DT; ++d)
        if (kWhole || d * 16 < dim) *reinterpret_cast<f32x4*>(row + d * 16) = acc[t][d];
      if (g == 0) {
        to[(int64_t)a.row_tile * dim + 2 * i] = top[t];
        to[(int64_t)a.row_tile * dim + 2 * i + 1] = sum[t];
      }
    }
  }
}

// Joins the splits of 16 rows of a slot and head, 16 lanes a row: lane j of them
// has split j's reference and sum (a pass for each 16 splits) and the dimensions
// 4 j .. + 3 of each 64. The loads of up to 8 splits wait together (a pass of one
// context of 16384 tokens in 32 splits: 17 us, with two at a time 29); of two
// splits no more are asked for, which leaves room for more rows at once (4 us of
// 119 with chunks of up to 256 tokens).
template <typename T, int kParts, int kBatch>
__global__ __launch_bounds__(256) void join_kernel(AttentionArgs a) {
  const CacheArgs& c = a.c;
  const int lane = threadIdx.x & 63, j = lane & 15, dim = c.dim;
  const int group = a.q_heads / c.heads, pieces = a.row_tile / 16;
  const int piece = blockIdx.x % pieces;
  const int job = blockIdx.x / pieces, h = job % c.heads, slot = job / c.heads;
  Place p;
  if (!place_of_slot(a, group, slot, p)) return;
  if (p.splits == 1 || piece * 16 >= p.rows) return;  // written whole, or nothing there
  const int row = piece * 16 + (threadIdx.x >> 4);
  const bool live = row < p.rows;
  const int i = live ? row : p.rows - 1;

  const int64_t step = (int64_t)a.row_tile * (dim + 2);
  const float* from = a.work + ((int64_t)slot * c.heads + h) * a.splits * step;
  const float* heads = from + (int64_t)a.row_tile * dim + 2 * i;
  const float* mine = from + (int64_t)i * dim;
  float all = -kInf, total = 0.f;
  f32x4 o[kParts] = {};
  for (int first = 0; first < p.splits; first += 16) {
    const int n = p.splits - first < 16 ? p.splits - first : 16;
    const float* at = heads + (first + (j < n ? j : 0)) * step;
    const float top = at[0], sum = at[1];
    const float* src = mine + first * step;
    f32x4 held[kBatch][kParts];
    auto fetch = [&](int begin) {
#pragma unroll
      for (int s = 0; s < kBatch; ++s)
        if (begin + s < n) {
#pragma unroll
          for (int q = 0; q < kParts; ++q)
            held[s][q] = *reinterpret_cast<const f32x4*>(src + (begin + s) * step + (q * 64 + j * 4 < dim ? q * 64 + j * 4 : 0));
        }
    };
    fetch(0);
    float best = j < n ? top : -kInf;
#pragma unroll
    for (int x = 1; x < 16; x <<= 1) best = fmaxf(best, __shfl_xor(best, x));
    const float now = fmaxf(all, best), ref = now == -kInf ? 0.f : now;
    const float old = __builtin_amdgcn_exp2f(all - ref);
    const float f = j < n ? __builtin_amdgcn_exp2f(top - ref) : 0.f;
    float part = j < n ? sum * f : 0.f;
#pragma unroll
    for (int x = 1; x < 16; x <<= 1) part += __shfl_xor(part, x);
    total = total * old + part;
    all = now;
#pragma unroll
    for (int q = 0; q < kParts; ++q) o[q] *= old;
#pragma unroll 1
    for (int begin = 0; begin < n; begin += kBatch) {
#pragma unroll
      for (int s = 0; s < kBatch; ++s) {
        const float w = __shfl(f, (lane & 48) + begin + s);
        if (begin + s < n) {
#pragma unroll
          for (int q = 0; q < kParts; ++q) o[q] += held[s][q] * w;
        }
      }
      if (begin + kBatch < n) fetch(begin + kBatch);
    }
  }
  if (!live) return;
  const int tok = (p.local + i) / group, head = h * group + (p.local + i) % group;
  const float inv = total != 0.f ? 1.f / total : 0.f;
  T* out = (T*)a.out + (int64_t)(p.row0 + tok) * a.o_row + head * a.o_head + j * 4;
#pragma unroll
  for (int q = 0; q < kParts; ++q)
    if (q * 64 + j * 4 < dim) store4(out + q * 64, o[q] * inv);
  if (j == 0) a.lse[(int64_t)(p.row0 + tok) * a.q_heads + head] = (all + __builtin_amdgcn_logf(total)) * kLn2;
}

constexpr int kManyRows = 128;

template <typename T, int DT, bool kWhole>
hipError_t launch(const AttentionArgs& a, hipStream_t stream) {
  const int64_t jobs = slot_count(a) * a.splits;
  const dim3 grid((unsigned)((jobs + 7) / 8 * 8 * a.c.heads)), block(kWaves * 64);
  if (a.row_tile == kManyRows) {
    auto kernel = attention_rows_kernel<T, DT, kWhole>;
    constexpr size_t bytes = Staged<DT>::kBytes;
    if (bytes > 65536 - 64) {
      const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
      if (e != hipSuccess) return e;
    }
    kernel<<<grid, block, bytes, stream>>>(a);
  } else if (DT <= 8 && a.row_tile == 32) {
    attention_kernel<T, DT <= 8 ? DT : 8, 2, kWhole><<<grid, block, 0, stream>>>(a);
  } else {
    attention_kernel<T, DT, 1, kWhole><<<grid, block, 0, stream>>>(a);
  }
  if (hipError_t e = hipGetLastError()) return e;
  if (a.splits > 1) {
    auto kernel = a.splits == 2 ? join_kernel<T, DT / 4, 2> : join_kernel<T, DT / 4, DT <= 8 ? 8 : 4>;
    kernel<<<dim3((unsigned)(slot_count(a) * a.c.heads * (a.row_tile / 16))), 256, 0, stream>>>(a);
  }
  return hipGetLastError();
}

template <typename T, int DT>
hipError_t by_width(const AttentionArgs& a, hipStream_t stream) {
  return a.c.dim == DT * 16 ? launch<T, DT, true>(a, stream) : launch<T, DT, false>(a, stream);
}

template <typename T>
hipError_t by_dim(const AttentionArgs& a, hipStream_t stream) {
  if (a.c.dim <= 64) return by_width<T, 4>(a, stream);
  if (a.c.dim <= 128) return by_width<T, 8>(a, stream);
  return by_width<T, 16>(a, stream);
}

// Splits a pass's contexts; returns its floats of workspace.
int64_t split(AttentionArgs& a, int64_t per_seq) {
  const int64_t slots = slot_count(a), work = slots * a.c.heads;
  int64_t longest = a.longest < 1 ? 1 : a.longest > 1 << 30 ? 1 << 30 : a.longest;
  if (a.window && longest > a.window + kTile + per_seq) longest = a.window + kTile + per_seq;
  // Four rounds of workgroups on the card (2 fit a compute unit) even out their
  // lengths; more only add their beginnings and ends (64 contexts of 8-16k
  // tokens: 285 us with 2048, 302 with 4096, 326 with 8192). Chunks are two
  // tiles a wave at least, and a context of four or fewer is not split, since a
  // join takes 3.5 us and its launch. Where many rows share a workgroup, one
  // round will do.
  // Where chunks of four tiles a wave make one or two rounds of workgroups, they
  // are taken (4 contexts of 16384, 8 heads: 31 us, with two tiles 35.5; of 9000,
  // half a round: 27.3 and 25.9).
  const int64_t unit = kTile * kWaves, longer = 4 * unit, round = 512;
  const bool rounds = a.row_tile != kManyRows && work * (longest / longer) >= round &&
                      work * ((longest + longer - 1) / longer) <= 2 * round;
  const int64_t least = rounds ? longer : 2 * unit;
  const int64_t target = a.row_tile == kManyRows ? 768 : 2048;
  int64_t splits = longest <= 4 * unit ? 1 : target / (work > 0 ? work : 1);
  const int64_t most = (longest + least - 1) / least;
  splits = splits < 1 ? 1 : splits > most ? most : splits;
  if (splits > 256) splits = 256;
  a.chunk = (int)(((longest + splits - 1) / splits + unit - 1) / unit * unit);
  a.splits = (int)((longest + a.chunk - 1) / a.chunk);
  return a.splits == 1 ? 0 : work * a.splits * a.row_tile * (a.c.dim + 2);
}

}  // namespace

AttentionPlan plan_attention(const AttentionArgs& all) {
  AttentionPlan plan{};
  const int group = all.q_heads / all.c.heads;
  const int64_t rows = (int64_t)all.c.rows * group;
  const int64_t mean = all.c.starts ? rows / (all.c.batch > 0 ? all.c.batch : 1) : group;
  constexpr int kFew = 64;  // rows that waves with tokens of their own still serve better
  auto add = [&](int row_tile, int per, int few, int many, int64_t per_seq) {
    AttentionArgs& a = plan.pass[plan.passes++];
    a = all;
    a.row_tile = row_tile;
    a.few = few;
    a.many = many;
    a.per = per;
    a.tail = per == 0 ? all.tail : kLeaveTail;
    a.work = all.work ? all.work + plan.floats : nullptr;
    plan.floats += split(a, per_seq);
  };
  const int most = 0x7FFFFFFF;
  const int pair = all.c.dim <= 128 ? 32 : 16;  // two tiles of rows, if registers allow
  if (!all.c.starts) {
    const int tile = group > kFew ? kManyRows : group > 16 ? pair : 16;
    add(tile, (group + tile - 1) / tile, 0, most, mean);
  } else if (mean <= 16 || rows <= kFew) {
    add(16, 0, 0, most, mean);
  } else if (all.c.batch == 1) {
    add(kManyRows, 0, 0, most, mean);
  } else {
    add(pair, kFew / pair, 0, kFew, kFew);
    add(kManyRows, 0, kFew, most, mean);
  }
  return plan;
}

hipError_t launch_cache_attention(const AttentionArgs& all, hipStream_t stream) {
  const AttentionPlan plan = plan_attention(all);
  for (int i = 0; i < plan.passes; ++i) {
    const AttentionArgs& a = plan.pass[i];
    const hipError_t e = a.dtype == kBF16 ? by_dim<__bf16>(a, stream) : by_dim<_Float16>(a, stream);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace serving
