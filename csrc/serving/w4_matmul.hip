// y[m, n] = sum_k x[m, k] (q[n, k] - z[n, g]) s[n, g], g = k / group: the
// product of a decode batch with weights held in 4 bits.
//
// Bound by the bytes of the codes, which are read once: a tile of 16 rows by
// 128 columns is 1 KB, one 16-byte load of a wave, and lies in the order in
// which the lanes feed the matrix instruction. The weights are its first
// operand, so that up to 16 tokens ride along as columns at no further cost.
//
// A nibble q becomes the operand's type by putting it into the top mantissa
// bits of 16.0: 16 + q exactly, for bf16 and fp16 alike, two codes an
// instruction pair. A second product with the constant -(16 + z) takes the
// offset off again inside the fp32 accumulator, so each product is of x with
// a whole number of at most 5 bits and nothing is rounded before the sum. A
// group's scale multiplies its fp32 sum.
//
// The waves of a workgroup split the columns and join their sums in LDS, in
// the waves' order, so that results do not depend on timing.
#include "device.h"
#include "serving.h"

namespace serving {
namespace {

// 8 codes of a dword in the order of 8 consecutive columns, plus 16 each.
template <typename T>
__device__ __forceinline__ typename Mat<T>::x8 decode8(uint32_t w);

template <>
__device__ __forceinline__ bf16x8 decode8<__bf16>(uint32_t w) {
  u32x4 r;
  r[0] = ((w << 3) & 0x00780078u) | 0x41804180u;
  r[1] = ((w >> 1) & 0x00780078u) | 0x41804180u;
  r[2] = ((w >> 5) & 0x00780078u) | 0x41804180u;
  r[3] = ((w >> 9) & 0x00780078u) | 0x41804180u;
  return bits_as<bf16x8>(r);
}

template <>
__device__ __forceinline__ f16x8 decode8<_Float16>(uint32_t w) {
  u32x4 r;
  r[0] = ((w << 6) & 0x03C003C0u) | 0x4C004C00u;
  r[1] = ((w << 2) & 0x03C003C0u) | 0x4C004C00u;
  r[2] = ((w >> 2) & 0x03C003C0u) | 0x4C004C00u;
  r[3] = ((w >> 6) & 0x03C003C0u) | 0x4C004C00u;
  return bits_as<f16x8>(r);
}

template <typename T>
__device__ __forceinline__ typename Mat<T>::x8 splat8(float v) {
  typename Mat<T>::x8 r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = (T)v;
  return r;
}

// 8 values of row `x` from column k on; columns past the last are 0.
template <typename T, bool kVec>
__device__ __forceinline__ typename Mat<T>::x8 load_x8(const T* x, int k, int cols, bool live) {
  typename Mat<T>::x8 r = bits_as<typename Mat<T>::x8>(u32x4{0, 0, 0, 0});
  if constexpr (kVec) {
    if (live && k < cols) r = *reinterpret_cast<const typename Mat<T>::x8*>(x + k);
  } else {
    if (live) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (k + i < cols) r[i] = x[k + i];
    }
  }
  return r;
}

// MT tiles of 16 tokens, NT tiles of 16 weight rows, groups of G columns.
template <typename T, int MT, int NT, int G, bool kZeros, bool kVec, int W>
__global__ __launch_bounds__(W * 64) void w4_kernel(W4Args a) {
  using x8 = typename Mat<T>::x8;
  constexpr int kSubs = 128 / G;      // groups of a block of 128 columns
  constexpr int kSteps = G / 32;      // matrix instructions of a group
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, g = lane >> 4;
  const int tiles = (a.n + 15) >> 4, blocks = (a.k + 127) >> 7;
  const int groups = (a.k + G - 1) / G;
  const int tile0 = blockIdx.x * NT, m0 = blockIdx.y * 16 * MT;

  const T* x[MT];
  bool live[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int m = m0 + mt * 16 + r;
    live[mt] = m < a.m;
    x[mt] = (const T*)a.x + (int64_t)(live[mt] ? m : 0) * a.ldx;
  }
  const u32x4* codes[NT];
  const T* scales[NT];
  const uint8_t* zeros[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int tile = tile0 + nt < tiles ? tile0 + nt : tiles - 1;
    codes[nt] = (const u32x4*)a.codes + (int64_t)tile * blocks * 64 + lane;
    scales[nt] = (const T*)a.scales + (int64_t)tile * groups * 16 + g * 4;
    zeros[nt] = kZeros ? a.zeros + (int64_t)tile * groups * 16 + r : nullptr;
  }

  f32x4 acc[NT][MT] = {};
  const x8 eight = splat8<T>(-24.f);  // -(16 + 8)
  for (int b = wave; b < blocks; b += W) {
    u32x4 c[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) c[nt] = codes[nt][(int64_t)b * 64];
    x8 xf[MT][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        xf[mt][j] = load_x8<T, kVec>(x[mt], b * 128 + j * 32 + g * 8, a.k, live[mt]);
#pragma unroll
    for (int s = 0; s < kSubs; ++s) {
      int grp = b * kSubs + s;
      if (grp >= groups) grp = groups - 1;  // columns past the last: x is 0
      f32x4 part[NT][MT];
      if constexpr (!kZeros) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          f32x4 z = {};
#pragma unroll
          for (int j = 0; j < kSteps; ++j) z = Mat<T>::mfma(eight, xf[mt][s * kSteps + j], z);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) part[nt][mt] = z;
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if constexpr (kZeros) {
          const x8 off = splat8<T>(-16.f - (float)zeros[nt][grp * 16]);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            f32x4 z = {};
#pragma unroll
            for (int j = 0; j < kSteps; ++j) z = Mat<T>::mfma(off, xf[mt][s * kSteps + j], z);
            part[nt][mt] = z;
          }
        }
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
          const x8 w = decode8<T>(c[nt][s * kSteps + j]);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
            part[nt][mt] = Mat<T>::mfma(w, xf[mt][s * kSteps + j], part[nt][mt]);
        }
        const u32x2 raw = *reinterpret_cast<const u32x2*>(scales[nt] + grp * 16);
        typedef T t4 __attribute__((ext_vector_type(4)));
        const t4 sc = bits_as<t4>(raw);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[nt][mt][i] += (float)sc[i] * part[nt][mt][i];
      }
    }
  }

  __shared__ f32x4 sums[W][NT * MT][64];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) sums[wave][nt * MT + mt][lane] = acc[nt][mt];
  __syncthreads();
  for (int f = wave; f < NT * MT; f += W) {
    f32x4 s = sums[0][f][lane];
#pragma unroll
    for (int w = 1; w < W; ++w) s += sums[w][f][lane];
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

template <typename T, int MT, int NT, int G, bool kZeros, bool kVec>
hipError_t launch(const W4Args& a, hipStream_t stream) {
  constexpr int W = 8;
  const int tiles = (a.n + 15) / 16;
  const dim3 grid((tiles + NT - 1) / NT, (a.m + 16 * MT - 1) / (16 * MT));
  w4_kernel<T, MT, NT, G, kZeros, kVec, W><<<grid, W * 64, 0, stream>>>(a);
  return hipGetLastError();
}

template <typename T, int MT, int NT, int G, bool kZeros>
hipError_t by_load(const W4Args& a, hipStream_t stream) {
  const bool vec = a.k % 8 == 0 && a.ldx % 8 == 0 && (uintptr_t)a.x % 16 == 0;
  return vec ? launch<T, MT, NT, G, kZeros, true>(a, stream) : launch<T, MT, NT, G, kZeros, false>(a, stream);
}

template <typename T, int MT, int NT>
hipError_t by_group(const W4Args& a, hipStream_t stream) {
  if (a.zeros) {
    if (a.group == 32) return by_load<T, MT, NT, 32, true>(a, stream);
    if (a.group == 64) return by_load<T, MT, NT, 64, true>(a, stream);
    return by_load<T, MT, NT, 128, true>(a, stream);
  }
  if (a.group == 32) return by_load<T, MT, NT, 32, false>(a, stream);
  if (a.group == 64) return by_load<T, MT, NT, 64, false>(a, stream);
  return by_load<T, MT, NT, 128, false>(a, stream);
}

template <typename T>
hipError_t by_tokens(const W4Args& a, hipStream_t stream) {
  if (a.m <= 16) return by_group<T, 1, 1>(a, stream);
  if (a.m <= 32) return by_group<T, 2, 1>(a, stream);
  return by_group<T, 4, 1>(a, stream);
}

}  // namespace

hipError_t launch_w4_matmul(const W4Args& a, hipStream_t stream) {
  return a.dtype == kBF16 ? by_tokens<__bf16>(a, stream) : by_tokens<_Float16>(a, stream);
}

}  // namespace serving
