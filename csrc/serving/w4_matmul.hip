// y[m, n] = sum_k x[m, k] (q[n, k] - z[n, g]) s[n, g], g = k / group: the
// product of a decode batch with weights held in 4 bits.
//
// Bound by the bytes of the codes, which are read once: a tile of 16 rows by
// 128 columns is 1 KB, one 16-byte load of a wave, and lies in the order in
// which the lanes feed the matrix instruction. The weights are its first
// operand, so that up to 16 tokens ride along as columns at no further cost.
//
// A nibble q becomes the operand's type by putting it into the top mantissa
// bits of 16.0: 16 + q exactly, for bf16 and fp16 alike, two codes in two
// instructions. A second product with a constant takes the offset (and the
// zero point, where all are 8) off again inside the fp32 accumulator; it is one
// for all weight rows and gives the sum of x that zero points are times. Each
// product is of x with a whole number of at most 5 bits, and nothing is rounded
// before the fp32 sum of a group, which its scale multiplies. On its way the sum
// of 128 columns comes to 24 128 + 31 32 = 2^12 times the largest x, whatever its
// result, so x has to be under 2^115 for it to stay within fp32.
//
// The 8 waves of a workgroup split the columns and join their sums in LDS, in
// the waves' order, so that results do not depend on timing. 16 waves are slower
// even where there are few tiles of rows (16 x 1024 x 8192: 12.5 us against 11.5).
//
// What the tokens cost beside the codes decides the rest (us, measured):
// - Every load occupies the address path for 16 cycles, however little it
//   fetches, as long as a load of 1 KB of codes. So scales and zero points come
//   through LDS, and the tokens of few long rows too, up to 32 KB (1 x 8192 x 8192:
//   10.1 with them in LDS, 12.4 without). Rows are staged one after another, so more
//   and shorter ones lose by it (4 x 16384 x 1024: 5.7 and 4.9; 16 x 4096 x 1024: 6.3
//   and 4.3), unless 16-byte loads do not fit them: LDS saves their packing.
// - Tokens that do not fit are read by every workgroup through the L2, which is
//   what a compute unit's second workgroup waits for: 16 x 8192 tokens by 256
//   tiles of rows take 12.1, by 257 to 512 tiles 20.8, but with two tiles a
//   workgroup 13.1. So one workgroup a unit has all its tiles, up to 8 (16 x 28672
//   x 8192: 28; with four tiles, 448 workgroups, 34), 4 of 64 tokens. Of fewer than
//   8 tokens, two workgroups with a tile each take 9.5, one with two 10.2 (5 x 5000
//   x 5000). Tokens in LDS: two tiles a workgroup from 512 tiles on (1 x 28672 x
//   8192: 25.8, with one 27.8; 1 x 8192 x 8192: 10.5 and 9.7).
// - Rows of tokens a power of two apart fall on the same channels of the L2. A
//   launch before lays tokens out in the order of the loads, which pays from two
//   tiles of tokens on (64 x 16384 x 8192: 34 with it, 44 without), but not for one
//   (16 x 28672 x 8192: 29.5 with it, 28 without), and not for up to 128 KB of
//   tokens, where its launch is what a call costs (32 x 4096 x 2048: a call 12.2 with
//   it, 8.2 without; replayed from a graph 6.7 and 7.9). It also takes rows that
//   16-byte loads do not fit.
// - Workgroups that read the same tokens, or rows of weights a power of two apart,
//   at the same time wait for the same channels: they start a block of columns
//   apart (32 x 16384 x 8192: 23.4 with the packing, 26.3 without; 16 x 32768 x
//   8192: 31.4, 36.7). For one tile of tokens and few tiles of rows it only costs
//   (16 x 8192 x 8192: 13.8 instead of 13.2).
// - The codes pass by the L2 (non-temporal): 5% at the largest sizes.
#include "device.h"
#include "serving.h"

namespace serving {
namespace {

constexpr int W = 8;  // waves of a workgroup

// 8 codes of a dword in the order of 8 consecutive columns, plus 16 each. The
// instruction that masks and sets bits takes no constants: its mask lives in a
// vector register and its base in a scalar one, made once.
template <typename T>
struct Decoder {
  static constexpr bool kHalf = __is_same(T, _Float16);
  static constexpr int kTop = kHalf ? 6 : 3;  // lowest of the 4 bits in a half dword
  uint32_t mask = kHalf ? 0x03C003C0u : 0x00780078u;
  uint32_t base = kHalf ? 0x4C004C00u : 0x41804180u;
  __device__ __forceinline__ Decoder() {
    asm("" : "+v"(mask));
    asm("" : "+s"(base));
  }
  __device__ __forceinline__ typename Mat<T>::x8 operator()(uint32_t w) const {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int up = kTop - 4 * i;
      r[i] = ((up >= 0 ? w << (up & 31) : w >> (-up & 31)) & mask) | base;
    }
    return bits_as<typename Mat<T>::x8>(r);
  }
};

template <typename T>
__device__ __forceinline__ typename Mat<T>::x8 splat8(float v) {
  typename Mat<T>::x8 r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = (T)v;
  return r;
}

// LDS of a workgroup: scales and zero points of its tiles, then the tokens if
// they are few; the waves' sums take its place at the end.
template <typename T, int MT, int NT>
struct Lds {
  int groups, scales, zeros, x, pitch;  // bytes, and elements of a token's row
  size_t size;
  __host__ __device__ Lds(const W4Args& a, bool with_x) {
    groups = (a.k + a.group - 1) / a.group;
    scales = NT * groups * 16 * (int)sizeof(T);
    zeros = a.zeros ? NT * groups * 16 : 0;
    // 16 bytes more than whole blocks: rows start in different banks
    pitch = (a.k + 127) / 128 * 128 + 8;
    x = with_x ? (a.m < 16 * MT ? a.m : 16 * MT) * pitch * (int)sizeof(T) : 0;
    size = (size_t)scales + zeros + x;
    const size_t sums = (size_t)W * NT * MT * 1024;
    if (size < sums) size = sums;
  }
};

// Where the lanes of a matrix instruction find their tokens in memory: the
// caller's rows, or packed ones. Elements.
struct Tokens {
  const void* x;
  int64_t row;       // from a lane's row to the next (packed: from lane to lane)
  int64_t tile;      // from a tile of 16 tokens to the next
  int64_t chunk;     // from a workgroup's tiles to the next one's
  int step, block;   // from 32 columns to the next, from 128 to the next
  int columns, packed;
};

// What is read for columns past the last.
__device__ const u32x4 kNothing = {0, 0, 0, 0};

// MT tiles of 16 tokens, NT tiles of 16 weight rows, groups of G columns. kX:
// tokens come through LDS, else from memory.
template <typename T, int MT, int NT, int G, bool kZeros, bool kX>
__global__ __launch_bounds__(W * 64) void w4_kernel(W4Args a, Tokens from) {
  using x8 = typename Mat<T>::x8;
  typedef T t4 __attribute__((ext_vector_type(4)));
  // Of 64 tokens, groups of 128 columns are summed by halves, whose tokens are
  // all in registers at once.
  constexpr int kPart = MT > 2 && G > 64 ? 64 : G;
  constexpr int kSubs = 128 / kPart;  // parts of a block of 128 columns
  constexpr int kSteps = kPart / 32;  // matrix instructions of a part
  extern __shared__ u32x4 lds[];
  const Lds<T, MT, NT> plan(a, kX);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, g = lane >> 4;
  const int tiles = (a.n + 15) >> 4, blocks = (a.k + 127) >> 7;
  const int groups = plan.groups;
  const int tile0 = blockIdx.x * NT, m0 = blockIdx.y * 16 * MT;

  const u32x4* codes[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int tile = tile0 + nt < tiles ? tile0 + nt : tiles - 1;
    codes[nt] = (const u32x4*)a.codes + (int64_t)tile * blocks * 64 + lane;
  }
  const T* x[MT];
  if constexpr (!kX) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {  // tokens past the last are another's: their results go nowhere
      const int m = mt * 16 + r, last = a.m - m0 - 1;
      x[mt] = (const T*)from.x + blockIdx.y * from.chunk;
      x[mt] += from.packed ? mt * from.tile + lane * 8 : (m < last ? m : last) * from.row + g * 8;
    }
  }
  // The next turn's codes come from memory while this one's are at work, and
  // its tokens, kRing steps ahead, into the registers that a step leaves.
  constexpr bool kTurns = MT * NT > 8;
  constexpr int kRing = kX || MT <= 2 || (kTurns && !kZeros) ? 4 : 2;
  u32x4 now[NT], next[NT];
  x8 xf[MT][kRing];
  auto load_codes = [&](int b) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) next[nt] = __builtin_nontemporal_load(codes[nt] + (int64_t)b * 64);
  };
  auto load_x = [&](int b, int j) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const T* p = x[mt] + (int64_t)b * from.block + j * from.step;
      if constexpr (MT == 1)  // more are packed, with zeros behind the last column
        p = b * 128 + j * 32 + g * 8 < from.columns ? p : (const T*)&kNothing;
      xf[mt][j % kRing] = *reinterpret_cast<const x8*>(p);
    }
  };
  // Turn i's block of columns: where it pays, workgroups of a die begin a block
  // apart.
  const int apart = MT > 1 || NT % 4 == 0 ? (int)(blockIdx.x >> 3) % blocks : 0;
  auto block_of = [&](int i) { return i + apart < blocks ? i + apart : i + apart - blocks; };
  if (wave < blocks) {
    load_codes(block_of(wave));
    if constexpr (!kX) {
#pragma unroll
      for (int j = 0; j < kRing; ++j) load_x(block_of(wave), j);
    }
  }

  // scales, zero points and few tokens are small pieces scattered over lanes:
  // read from memory each would cost a load as long as one of codes
  char* base = reinterpret_cast<char*>(lds);
  T* scales = reinterpret_cast<T*>(base);
  uint8_t* zeros = reinterpret_cast<uint8_t*>(base + plan.scales);
  T* xs = reinterpret_cast<T*>(base + plan.scales + plan.zeros);
  {
    const int rest = (tiles - tile0 < NT ? tiles - tile0 : NT) * groups * 16;  // of the tiles that are there
    const T* sc = (const T*)a.scales + (int64_t)tile0 * groups * 16;
    for (int i = threadIdx.x * 4; i < rest; i += W * 256)
      *reinterpret_cast<u32x2*>(scales + i) = *reinterpret_cast<const u32x2*>(sc + i);
    if constexpr (kZeros) {
      const uint8_t* z = a.zeros + (int64_t)tile0 * groups * 16;
      for (int i = threadIdx.x * 4; i < rest; i += W * 256)
        *reinterpret_cast<uint32_t*>(zeros + i) = *reinterpret_cast<const uint32_t*>(z + i);
    }
    if constexpr (kX) {
      const int rows = a.m - m0 < 16 * MT ? a.m - m0 : 16 * MT;
      const bool whole = a.k % 8 == 0 && a.ldx % 8 == 0 && (uintptr_t)a.x % 16 == 0;
      for (int row = 0; row < rows; ++row) {
        const T* src = (const T*)a.x + (int64_t)(m0 + row) * a.ldx;
        for (int k = threadIdx.x * 8; k < blocks * 128; k += W * 512) {
          x8 v = bits_as<x8>(u32x4{0, 0, 0, 0});
          if (whole) {
            if (k < a.k) v = *reinterpret_cast<const x8*>(src + k);
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (k + i < a.k) v[i] = src[k + i];
          }
          *reinterpret_cast<x8*>(xs + row * plan.pitch + k) = v;
        }
      }
    }
  }
  __syncthreads();
  int at[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int last = a.m - m0 - 1;
    at[mt] = (mt * 16 + r < last ? mt * 16 + r : last) * plan.pitch + g * 8;
  }

  f32x4 acc[NT][MT] = {};
  const Decoder<T> decode;
  const x8 offset = splat8<T>(kZeros ? -16.f : -24.f);  // 24: 16 + 8
#pragma unroll 1
  for (int turn = wave; turn < blocks; turn += W) {
    const int b = block_of(turn);
    const int after = block_of(turn + W < blocks ? turn + W : turn);  // the last turn reads its own again
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) now[nt] = next[nt];
    if constexpr (kX) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int j = 0; j < 4; ++j) xf[mt][j] = *reinterpret_cast<const x8*>(xs + at[mt] + b * 128 + j * 32);
    }
    load_codes(after);
#pragma unroll
    for (int s = 0; s < kSubs; ++s) {
      int grp = b * (128 / G) + s * kPart / G;
      if (grp >= groups) grp = groups - 1;  // columns past the last: x is 0
      f32x4 z[MT] = {};
      auto add = [&](int nt, const f32x4* part) {
        const int place = (nt * groups + grp) * 16 + g * 4;
        const t4 sc = bits_as<t4>(*reinterpret_cast<const u32x2*>(scales + place));
        uint32_t zp = 0;
        if constexpr (kZeros) zp = *reinterpret_cast<const uint32_t*>(zeros + place);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float v = part[mt][i];
            if constexpr (kZeros)  // z is -16 times the sum of x
              v = __builtin_fmaf((float)(zp >> (8 * i) & 255u), z[mt][i] * 0.0625f, v);
            acc[nt][mt][i] = __builtin_fmaf((float)sc[i], v, acc[nt][mt][i]);
          }
      };
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int j = 0; j < kSteps; ++j) z[mt] = Mat<T>::mfma(offset, xf[mt][(s * kSteps + j) % kRing], z[mt]);
      if constexpr (kTurns) {
        // a tile of rows at a time, the sums of the one before being scaled
        // meanwhile: those of all tiles at once take more registers than there are
        f32x4 part[2][MT];
#pragma unroll
        for (int nt = 0; nt <= NT; ++nt) {
          if (nt < NT) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) part[nt & 1][mt] = z[mt];
#pragma unroll
            for (int j = s * kSteps; j < (s + 1) * kSteps; ++j) {
              const x8 w = decode(now[nt][j]);
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) part[nt & 1][mt] = Mat<T>::mfma(w, xf[mt][j % kRing], part[nt & 1][mt]);
            }
          }
          if (nt > 0) add(nt - 1, part[nt - 1 & 1]);
          if (nt == NT - 1) {
#pragma unroll
            for (int j = s * kSteps; j < (s + 1) * kSteps; ++j) load_x(j + kRing < 4 ? b : after, (j + kRing) % 4);
          }
        }
      } else {
        f32x4 part[NT][MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) part[nt][mt] = z[mt];
#pragma unroll
        for (int j = s * kSteps; j < (s + 1) * kSteps; ++j) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const x8 w = decode(now[nt][j]);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) part[nt][mt] = Mat<T>::mfma(w, xf[mt][j % kRing], part[nt][mt]);
          }
          if constexpr (!kX) load_x(j + kRing < 4 ? b : after, (j + kRing) % 4);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) add(nt, part[nt]);
      }
      if constexpr (MT > 2 || MT * NT > 4) __builtin_amdgcn_sched_barrier(0);  // registers
    }
  }

  __syncthreads();  // what was staged has been used
  f32x4* sums = reinterpret_cast<f32x4*>(lds);  // [W][NT MT][64]
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) sums[(wave * NT * MT + nt * MT + mt) * 64 + lane] = acc[nt][mt];
  __syncthreads();
  for (int f = wave; f < NT * MT; f += W) {
    f32x4 s = sums[f * 64 + lane];
#pragma unroll
    for (int w = 1; w < W; ++w) s += sums[(w * NT * MT + f) * 64 + lane];
    const int m = m0 + (f % MT) * 16 + r;
    const int n = (tile0 + f / MT) * 16 + g * 4;
    if (m < a.m) {
      T* y = (T*)a.y + (int64_t)m * a.ldy + n;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < a.n) y[i] = (T)s[i];
    }
  }
}

// Tokens in the order of the matrix instruction's loads, 1 KB for 16 tokens and
// 32 columns; columns and tokens past the last are 0. A thread has 8 columns of
// a token, a wave 512 in a row, so that reads spread over the channels.
template <typename T>
__global__ __launch_bounds__(256) void pack_kernel(W4Args a, T* to, int mts, bool whole) {
  typedef typename Mat<T>::x8 x8;
  const int parts = (a.k + 127) / 128 * 16;  // of a token
  const int part = blockIdx.x * 256 + threadIdx.x;
  if (part >= parts) return;
  const int m = blockIdx.y, k = part * 8;
  x8 v = bits_as<x8>(u32x4{0, 0, 0, 0});
  if (m < a.m) {
    const T* src = (const T*)a.x + m * a.ldx + k;
    if (whole) {
      if (k < a.k) v = *reinterpret_cast<const x8*>(src);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (k + i < a.k) v[i] = src[i];
    }
  }
  const int chunk = m / (16 * mts), tile = m / 16 % mts;
  const int64_t piece = (int64_t)chunk * (parts / 4) * mts + (int64_t)(part / 4) * mts + tile;
  *reinterpret_cast<x8*>(to + piece * 512 + ((part % 4) * 16 + m % 16) * 8) = v;
}

int token_tiles(int m) { return m <= 16 ? 1 : m <= 32 ? 2 : 4; }
bool whole_loads(const W4Args& a) { return a.k % 8 == 0 && a.ldx % 8 == 0 && (uintptr_t)a.x % 16 == 0; }
bool through_lds(const W4Args& a) {
  return a.m <= 16 && (int64_t)a.m * a.k <= 16384 && (a.k >= 1024 * a.m || !whole_loads(a));
}
bool packs(const W4Args& a) {
  const bool small = (int64_t)a.m * a.k <= 65536 && a.k % 128 == 0;  // and no columns past the last
  return !through_lds(a) && !(whole_loads(a) && (a.m <= 16 || small));
}

template <typename T, int MT, int NT, int G, bool kZeros, bool kX>
hipError_t launch(const W4Args& a, hipStream_t stream) {
  const int tiles = (a.n + 15) / 16, blocks = (a.k + 127) / 128;
  const int chunks = (a.m + 16 * MT - 1) / (16 * MT);
  Tokens from{a.x, a.ldx, 0, 16 * MT * a.ldx, 32, 128, a.k, 0};
  if (!kX && packs(a)) {
    const int pieces = blocks * 4 * MT;
    pack_kernel<T><<<dim3((blocks * 16 + 255) / 256, chunks * 16 * MT), 256, 0, stream>>>(a, (T*)a.work, MT, whole_loads(a));
    if (hipError_t e = hipGetLastError()) return e;
    from = Tokens{a.work, 8, 512, (int64_t)pieces * 512, MT * 512, MT * 2048, blocks * 128, 1};
  }
  const Lds<T, MT, NT> plan(a, kX);
  auto kernel = w4_kernel<T, MT, NT, G, kZeros, kX>;
  if (plan.size > 65536) {
    const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)plan.size);
    if (e != hipSuccess) return e;
  }
  kernel<<<dim3((tiles + NT - 1) / NT, chunks), W * 64, plan.size, stream>>>(a, from);
  return hipGetLastError();
}

template <typename T, int MT, int NT, bool kX>
hipError_t by_group(const W4Args& a, hipStream_t stream) {
  if (a.zeros) {
    if (a.group == 32) return launch<T, MT, NT, 32, true, kX>(a, stream);
    if (a.group == 64) return launch<T, MT, NT, 64, true, kX>(a, stream);
    return launch<T, MT, NT, 128, true, kX>(a, stream);
  }
  if (a.group == 32) return launch<T, MT, NT, 32, false, kX>(a, stream);
  if (a.group == 64) return launch<T, MT, NT, 64, false, kX>(a, stream);
  return launch<T, MT, NT, 128, false, kX>(a, stream);
}

// Tiles of rows of a workgroup: as many as let one round of workgroups, one for
// each compute unit, do, and in more rounds as few as leave those even. The
// tokens of up to 7 rows cost little enough for two workgroups a unit.
template <int kMost>
int row_tiles(const W4Args& a) {
  const int tiles = (a.n + 15) / 16, units = 256;
  if (a.m < 8 && tiles <= 2 * units) return 1;
  // their scales have to leave room in the LDS
  const int fit = 147456 / ((a.k + a.group - 1) / a.group * 48);
  const int most = fit < 1 ? 1 : fit < kMost ? fit : kMost;
  const int rounds = (tiles + units * most - 1) / (units * most);
  return (tiles + units * rounds - 1) / (units * rounds);
}

template <typename T, int MT>
hipError_t by_rows(const W4Args& a, hipStream_t stream) {
  constexpr int kMost = MT > 2 ? 4 : 8;  // registers
  switch (row_tiles<kMost>(a)) {
    case 1: return by_group<T, MT, 1, false>(a, stream);
    case 2: return by_group<T, MT, 2, false>(a, stream);
    case 3: return by_group<T, MT, 3, false>(a, stream);
    case 4: return by_group<T, MT, 4, false>(a, stream);
  }
  if constexpr (kMost > 4) {
    switch (row_tiles<kMost>(a)) {
      case 5: return by_group<T, MT, 5, false>(a, stream);
      case 6: return by_group<T, MT, 6, false>(a, stream);
      case 7: return by_group<T, MT, 7, false>(a, stream);
      case 8: return by_group<T, MT, 8, false>(a, stream);
    }
  }
  return hipErrorInvalidValue;
}

template <typename T>
hipError_t by_tokens(const W4Args& a, hipStream_t stream) {
  if (through_lds(a)) return a.n > 8192 ? by_group<T, 1, 2, true>(a, stream) : by_group<T, 1, 1, true>(a, stream);
  switch (token_tiles(a.m)) {
    case 1: return by_rows<T, 1>(a, stream);
    case 2: return by_rows<T, 2>(a, stream);
    default: return by_rows<T, 4>(a, stream);
  }
}

}  // namespace

int64_t w4_workspace(const W4Args& a) {
  if (!packs(a)) return 0;
  const int mts = token_tiles(a.m);
  return (int64_t)((a.m + 16 * mts - 1) / (16 * mts)) * ((a.k + 127) / 128) * 4 * mts * 1024;
}

hipError_t launch_w4_matmul(const W4Args& a, hipStream_t stream) {
  return a.dtype == kBF16 ? by_tokens<__bf16>(a, stream) : by_tokens<_Float16>(a, stream);
}

}  // namespace serving
