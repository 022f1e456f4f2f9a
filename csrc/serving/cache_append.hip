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
// One workgroup owns a page and head that gets tokens: it finds the largest
// magnitude of keys and values, settles both scales, re-rounds what the page
// held where a scale grew, and writes the new codes. Bound by the bytes of the
// new tokens, and by the launch for a decode step.
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

// Largest finite magnitude of the workgroup's values, for keys and values.
__device__ f32x2 block_max(f32x2 v, float (*shared)[2]) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    v[0] = fmaxf(v[0], __shfl_xor(v[0], d));
    v[1] = fmaxf(v[1], __shfl_xor(v[1], d));
  }
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) {
    shared[wave][0] = v[0];
    shared[wave][1] = v[1];
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    v[0] = fmaxf(v[0], shared[w][0]);
    v[1] = fmaxf(v[1], shared[w][1]);
  }
  return v;
}

__device__ __forceinline__ float finite_magnitude(float x) {
  const float m = fabsf(x);
  return m < kInf ? m : 0.f;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void append_kernel(AppendArgs a) {
  const CacheArgs& c = a.c;
  __shared__ float shared[kThreads / 64][2];
  const int h = blockIdx.y, page = c.page, dim = c.dim;
  PageWrite w;
  if (!page_of_slot(c, blockIdx.x, w)) return;
  const int from = w.from;

  const T* kn = (const T*)a.k_new + (int64_t)w.src * a.k_row + h * a.k_head;
  const T* vn = (const T*)a.v_new + (int64_t)w.src * a.v_row + h * a.v_head;
  const int n = (w.to - from) * dim;
  f32x2 most = {0.f, 0.f};
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int t = i / dim, d = i - t * dim;
    most[0] = fmaxf(most[0], finite_magnitude((float)kn[t * a.k_row + d]));
    most[1] = fmaxf(most[1], finite_magnitude((float)vn[t * a.v_row + d]));
  }
  most = block_max(most, shared);

  const int64_t ph = (int64_t)w.pid * c.heads + h;
  float ks = scale_for(most[0]), vs = scale_for(most[1]);
  float k_old = ks, v_old = vs;
  if (from > 0) {  // the page holds tokens before these
    k_old = c.k_scale[ph];
    v_old = c.v_scale[ph];
    ks = fmaxf(ks, k_old);
    vs = fmaxf(vs, v_old);
  }
  __syncthreads();  // every thread has read the old scales
  if (threadIdx.x == 0) {
    c.k_scale[ph] = ks;
    c.v_scale[ph] = vs;
  }
  uint8_t* kc = c.k + ph * page * dim;
  uint8_t* vc = c.v + ph * page * dim;
  if (ks != k_old) {
    const float f = k_old / ks;
    uint32_t* held = (uint32_t*)kc;
    for (int i = threadIdx.x; i < page * dim / 4; i += kThreads) held[i] = recode4(held[i], f);
  }
  if (vs != v_old) {
    const float f = v_old / vs;
    uint32_t* held = (uint32_t*)vc;
    for (int i = threadIdx.x; i < page * dim / 4; i += kThreads) held[i] = recode4(held[i], f);
  }
  __syncthreads();
  const float ki = 1.f / ks, vi = 1.f / vs;  // exact
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int t = i / dim, d = i - t * dim;
    const uint32_t code = encode2((float)kn[t * a.k_row + d] * ki, (float)vn[t * a.v_row + d] * vi);
    kc[(from + t) * dim + d] = (uint8_t)code;
    vc[d * page + from + t] = (uint8_t)(code >> 8);
  }
}

}  // namespace

hipError_t launch_cache_append(const AppendArgs& a, hipStream_t stream) {
  const CacheArgs& c = a.c;
  const dim3 grid((unsigned)append_slots(c), c.heads);
  if (a.dtype == kBF16)
    append_kernel<__bf16><<<grid, kThreads, 0, stream>>>(a);
  else
    append_kernel<_Float16><<<grid, kThreads, 0, stream>>>(a);
  return hipGetLastError();
}

}  // namespace serving
