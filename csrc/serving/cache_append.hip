// Writes new keys and values into a paged cache held in 8 bits, with one scale
// for each page and head.
//
// A scale is the smallest power of two that brings the page's largest
// magnitude within 448 (not under 2^-64): e4m3 holds 4 significant bits at any
// such scale, so a finer one would not be more exact, and a page whose scale
// grows is re-rounded by an exact shift of its exponents, which loses bits
// only where codes become subnormal. Infinities are held as +-448, NaN as NaN,
// and neither counts for the scale.
//
// Of a run of tokens, one workgroup owns a page and head: it finds the largest
// magnitude of keys and values, settles both scales, re-rounds what the page
// held where a scale grew, and writes the new codes, the values' by way of LDS,
// where a tile of them is turned so that memory gets whole words of a column.
// Bound by the bytes of the new tokens: 24.6 k tokens of 8 heads by 128 take 40
// us, 3.8 TB/s read and written of the 4.9 that a large copy reaches. Of single
// tokens, one wave owns a sequence's head, half of it the key and half the
// value; 256 of them take 7 us, bound by the chain of loads from the length to
// the page's scale. Where a scale grows, the half wave re-rounds its page a dword a
// lane and turn: 15 us more for a page of 64 tokens by 128, 90 for 128 by 256.
#include "device.h"
#include "geometry.h"
#include "serving.h"

namespace serving {
namespace {

constexpr int kThreads = 256;
constexpr float kMax8 = 448.f;

__device__ __forceinline__ float scale_for(float amax) {
  const int e = (int)((bits_as<uint32_t>(amax) + 0x1FFFFFu) >> 23) - 127 - 8;
  return bits_as<float>((uint32_t)((e < -64 ? -64 : e) + 127) << 23);
}

__device__ __forceinline__ uint32_t encode2(float a, float b) {
  // clamp that lets NaN through
  a = a != a ? a : fminf(fmaxf(a, -kMax8), kMax8);
  b = b != b ? b : fminf(fmaxf(b, -kMax8), kMax8);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false) & 0xFFFFu;
}

// The 4 codes of a dword times an exact power of two, rounded again.
__device__ __forceinline__ uint32_t recode4(uint32_t w, float f) {
  const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false);
  const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
  return encode2(lo[0] * f, lo[1] * f) | encode2(hi[0] * f, hi[1] * f) << 16;
}

__device__ __forceinline__ float finite_magnitude(float x) {
  const float m = fabsf(x);
  return m < kInf ? m : 0.f;
}

// 8 values; `whole` where 16 bytes can be read at once.
template <typename T>
__device__ __forceinline__ typename Mat<T>::x8 load8(const T* p, bool whole) {
  typename Mat<T>::x8 v;
  if (whole) return *reinterpret_cast<const typename Mat<T>::x8*>(p);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = p[i];
  return v;
}

template <typename X>
__device__ __forceinline__ float most_of(X v, float m) {
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, finite_magnitude((float)v[i]));
  return m;
}

// The codes of 8 values, times an exact power of two first.
template <typename X>
__device__ __forceinline__ u32x2 encode8(X v, float f) {
  u32x2 r;
#pragma unroll
  for (int w = 0; w < 2; ++w)
    r[w] = encode2((float)v[4 * w] * f, (float)v[4 * w + 1] * f) |
           encode2((float)v[4 * w + 2] * f, (float)v[4 * w + 3] * f) << 16;
  return r;
}

// ---- single tokens: a wave for a sequence's head -----------------------------

template <typename T>
__global__ __launch_bounds__(kThreads) void append_one_kernel(AppendArgs a, bool whole) {
  typedef typename Mat<T>::x8 x8;
  const CacheArgs& c = a.c;
  const int lane = threadIdx.x & 63, half = lane >> 5, d = (lane & 31) * 8;
  const int64_t job = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  const int b = (int)(job / c.heads), h = (int)(job - (int64_t)b * c.heads);
  if (b >= c.batch) return;
  const int page = c.page, dim = c.dim;
  const bool mine = d < dim;
  // the token does not wait for its page
  const T* src = half ? (const T*)a.v_new + b * a.v_row + h * a.v_head : (const T*)a.k_new + b * a.k_row + h * a.k_head;
  x8 x = bits_as<x8>(u32x4{0, 0, 0, 0});
  if (mine) x = load8(src + d, whole);

  PageWrite w;
  if (!page_of_slot(c, b, w)) return;
  const int64_t ph = (int64_t)w.pid * c.heads + h;
  float* scales = half ? c.v_scale : c.k_scale;
  const float old = scales[ph];
  float most = most_of(x, 0.f);
#pragma unroll
  for (int i = 1; i < 32; i <<= 1) most = fmaxf(most, __shfl_xor(most, i));
  float scale = scale_for(most);
  uint8_t* to = (half ? c.v : c.k) + ph * page * dim;
  if (w.from > 0) {
    scale = fmaxf(scale, old);
    if (scale != old) {
      const float f = old / scale;
      uint32_t* held = (uint32_t*)to;
      for (int i = lane & 31; i < page * dim / 4; i += 32) held[i] = recode4(held[i], f);
      __threadfence();  // of these words other lanes write some bytes next
    }
  }
  if ((lane & 31) == 0) scales[ph] = scale;
  if (!mine) return;
  const u32x2 codes = encode8(x, 1.f / scale);
  if (half) {
#pragma unroll
    for (int i = 0; i < 8; ++i) to[(d + i) * page + w.from] = (uint8_t)(codes[i >> 2] >> (8 * (i & 3)));
  } else {
    *reinterpret_cast<u32x2*>(to + w.from * dim + d) = codes;
  }
}

// ---- runs of tokens: a workgroup for a page and head -------------------------

constexpr int kTurn = 64;  // tokens whose values are turned at once

// kHeld: pieces of 8 values that a thread keeps of a page's keys, and as many of
// its values; 0: they are read twice.
template <typename T, int kHeld>
__global__ __launch_bounds__(kThreads) void append_kernel(AppendArgs a, bool whole) {
  typedef typename Mat<T>::x8 x8;
  const CacheArgs& c = a.c;
  __shared__ float shared[2][kThreads / 64];
  __shared__ uint32_t turned[256 * (kTurn / 4 + 1)];  // [dim][token], rows a word apart from whole banks
  const int h = blockIdx.x % c.heads, page = c.page, dim = c.dim;
  PageWrite w;
  if (!page_of_slot(c, blockIdx.x / c.heads, w)) return;

  const T* kn = (const T*)a.k_new + (int64_t)w.src * a.k_row + h * a.k_head;
  const T* vn = (const T*)a.v_new + (int64_t)w.src * a.v_row + h * a.v_head;
  const int row = dim / 8;  // pieces of a token
  const int n = (w.to - w.from) * row;
  // piece i: token i / row; by a rounded-up reciprocal, exact for i < 2^17
  const uint32_t inverse = (1u << 24) / row + 1;
  auto token_of = [&](int i) { return (int)((uint64_t)i * inverse >> 24); };
  auto key = [&](int i) { const int t = token_of(i); return load8(kn + t * a.k_row + (i - t * row) * 8, whole); };
  auto value = [&](int i) { const int t = token_of(i); return load8(vn + t * a.v_row + (i - t * row) * 8, whole); };

  x8 ks[kHeld ? kHeld : 1], vs[kHeld ? kHeld : 1];
  float km = 0.f, vm = 0.f;
  if constexpr (kHeld != 0) {
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
      const int i = threadIdx.x + j * kThreads;
      ks[j] = vs[j] = bits_as<x8>(u32x4{0, 0, 0, 0});
      if (i < n) {
        ks[j] = key(i);
        vs[j] = value(i);
      }
    }
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
      km = most_of(ks[j], km);
      vm = most_of(vs[j], vm);
    }
  } else {
    for (int i = threadIdx.x; i < n; i += kThreads) {
      km = most_of(key(i), km);
      vm = most_of(value(i), vm);
    }
  }
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) {
    km = fmaxf(km, __shfl_xor(km, i));
    vm = fmaxf(vm, __shfl_xor(vm, i));
  }
  if ((threadIdx.x & 63) == 0) {
    shared[0][threadIdx.x >> 6] = km;
    shared[1][threadIdx.x >> 6] = vm;
  }
  const int64_t ph = (int64_t)w.pid * c.heads + h;
  const float k_old = c.k_scale[ph], v_old = c.v_scale[ph];
  __syncthreads();  // every thread has read the old scales
#pragma unroll
  for (int i = 0; i < kThreads / 64; ++i) {
    km = fmaxf(km, shared[0][i]);
    vm = fmaxf(vm, shared[1][i]);
  }
  float k_scale = scale_for(km), v_scale = scale_for(vm);
  if (w.from > 0) {  // the page holds tokens before these
    k_scale = fmaxf(k_scale, k_old);
    v_scale = fmaxf(v_scale, v_old);
  }
  if (threadIdx.x == 0) {
    c.k_scale[ph] = k_scale;
    c.v_scale[ph] = v_scale;
  }
  uint8_t* kc = c.k + ph * page * dim;
  uint8_t* vc = c.v + ph * page * dim;
  if (w.from > 0 && k_scale != k_old) {
    const float f = k_old / k_scale;
    uint32_t* held = (uint32_t*)kc;
    for (int i = threadIdx.x; i < page * dim / 4; i += kThreads) held[i] = recode4(held[i], f);
  }
  if (w.from > 0 && v_scale != v_old) {
    const float f = v_old / v_scale;
    uint32_t* held = (uint32_t*)vc;
    for (int i = threadIdx.x; i < page * dim / 4; i += kThreads) held[i] = recode4(held[i], f);
  }
  __syncthreads();

  const float ki = 1.f / k_scale, vi = 1.f / v_scale;  // exact
  auto put_key = [&](int i, x8 x) { *reinterpret_cast<u32x2*>(kc + w.from * dim + i * 8) = encode8(x, ki); };
  if constexpr (kHeld != 0) {
#pragma unroll
    for (int j = 0; j < kHeld; ++j)
      if (threadIdx.x + j * kThreads < n) put_key(threadIdx.x + j * kThreads, ks[j]);
  } else {
    for (int i = threadIdx.x; i < n; i += kThreads) put_key(i, key(i));
  }
  // values: kTurn slots of the page at a time, turned in LDS
  uint8_t* bytes = reinterpret_cast<uint8_t*>(turned);
  constexpr int kPitch = kTurn + 4;
  for (int base = w.from & ~(kTurn - 1); base < w.to; base += kTurn) {
    const int lo = w.from > base ? w.from - base : 0;
    const int hi = w.to - base < kTurn ? w.to - base : kTurn;
    auto put_value = [&](int i, x8 x) {
      const int t = token_of(i), at = w.from + t - base;
      if (at < 0 || at >= kTurn) return;
      const u32x2 codes = encode8(x, vi);
      const int d = (i - t * row) * 8;
#pragma unroll
      for (int e = 0; e < 8; ++e) bytes[(d + e) * kPitch + at] = (uint8_t)(codes[e >> 2] >> (8 * (e & 3)));
    };
    if constexpr (kHeld != 0) {
#pragma unroll
      for (int j = 0; j < kHeld; ++j)
        if (threadIdx.x + j * kThreads < n) put_value(threadIdx.x + j * kThreads, vs[j]);
    } else {
      const int begin = (base + lo - w.from) * row, end = (base + hi - w.from) * row;
      for (int i = begin + threadIdx.x; i < end; i += kThreads) put_value(i, value(i));
    }
    __syncthreads();
    const int words = (page < kTurn ? page : kTurn) / 4;
    for (int i = threadIdx.x; i < dim * words; i += kThreads) {
      const int d = i / words, t = (i - d * words) * 4;
      if (t + 4 <= lo || t >= hi) continue;
      uint8_t* to = vc + d * page + base + t;
      const uint32_t word = turned[(d * kPitch + t) / 4];
      if (t >= lo && t + 4 <= hi) {
        *reinterpret_cast<uint32_t*>(to) = word;
      } else {
        for (int e = 0; e < 4; ++e)
          if (t + e >= lo && t + e < hi) to[e] = (uint8_t)(word >> (8 * e));
      }
    }
    __syncthreads();
  }
}

template <typename T>
hipError_t launch(const AppendArgs& a, hipStream_t stream) {
  const CacheArgs& c = a.c;
  const bool whole = (uintptr_t)a.k_new % 16 == 0 && (uintptr_t)a.v_new % 16 == 0 &&
                     (a.k_row | a.k_head | a.v_row | a.v_head) % 8 == 0;
  if (!c.starts) {
    const int64_t jobs = (int64_t)c.batch * c.heads;
    append_one_kernel<T><<<dim3((unsigned)((jobs + 3) / 4)), kThreads, 0, stream>>>(a, whole);
    return hipGetLastError();
  }
  const dim3 grid((unsigned)(append_slots(c) * c.heads));
  const int pieces = c.page * c.dim / 8;
  if (pieces <= kThreads)
    append_kernel<T, 1><<<grid, kThreads, 0, stream>>>(a, whole);
  else if (pieces <= 4 * kThreads)
    append_kernel<T, 4><<<grid, kThreads, 0, stream>>>(a, whole);
  else
    append_kernel<T, 0><<<grid, kThreads, 0, stream>>>(a, whole);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_cache_append(const AppendArgs& a, hipStream_t stream) {
  return a.dtype == kBF16 ? launch<__bf16>(a, stream) : launch<_Float16>(a, stream);
}

}  // namespace serving
