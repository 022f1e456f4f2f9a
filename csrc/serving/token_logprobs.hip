// Of each row of logits x and its given token t: log p(t), the entropy of p,
// the number of tokens above t, and the top alternatives, p = softmax(x).
//
// Bound by one read of the logits. A wave takes a span of consecutive logits
// in registers, finds their largest m, and then, with u = (x - m) log2 e, sums
// 2^u and 2^u u and counts x > x_t. On the way it leaves the largest of each 64
// consecutive logits (one 128-byte line of 16-bit ones): no other trace of the alternatives is needed,
// since the k best logits, by value and then by lower index, lie in the k best
// spans by their largest and then by lower index, and in these in the k best
// groups of 64. A second launch, or of few rows the same workgroup, joins a row's
// spans in a fixed order and reads only those groups again.
//
// Sums are fp32 over at most 4096 values a span, 64 a lane.
//
// 2048 x 130001 bf16, 5 alternatives: 110 us, 4.8 TB/s of the 6.3 that a plain
// read reaches, and 11 us for the joins. What bounds it is the vector unit: 11
// instructions a value, the exponential at a quarter of the rate, keep it busy
// 88% of the time. One row of 32000 with 20 alternatives takes 10.5 us, most of them
// for its join, a chain of dependent loads and selections in one workgroup.
#include "device.h"
#include "serving.h"

namespace serving {
namespace {

constexpr int kUnits = 8;  // 16-byte loads of a lane

template <typename T>
struct Shape {
  static constexpr int kVec = 16 / (int)sizeof(T);      // values of a load
  static constexpr int kSpan = kUnits * 64 * kVec;      // of a wave
  static constexpr int kGroups = kSpan / 64;
  static constexpr int kLanes = 64 / kVec;              // lanes of a group
};

// Workspace of a row: per span {reference, sum, weighted sum, count}, then
// the spans' largest, then the groups' largest.
struct Layout {
  int spans, groups;
  int64_t row;  // floats of a row
  __host__ __device__ Layout(int vocab, int span) {
    spans = (vocab + span - 1 + 7) / span;  // a row may start within a 16-byte line
    groups = span / 64;
    row = (int64_t)spans * (5 + groups);
  }
  __device__ float* stats(float* w, int64_t r, int s) const { return w + r * row + s * 4; }
  __device__ float* tops(float* w, int64_t r) const { return w + r * row + spans * 4; }
  __device__ float* group(float* w, int64_t r, int s) const { return w + r * row + spans * 5 + (int64_t)s * groups; }
};

__device__ __forceinline__ void unpack(u32x4 v, float* f, const __bf16*) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = bits_as<float>(v[i] << 16);
    f[2 * i + 1] = bits_as<float>(v[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ void unpack(u32x4 v, float* f, const _Float16*) {
  const f16x8 h = bits_as<f16x8>(v);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = (float)h[i];
}
__device__ __forceinline__ void unpack(u32x4 v, float* f, const float*) {
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = bits_as<float>(v[i]);
}

// Larger of a lane's and another's; NaN gives way.
__device__ __forceinline__ float max_xor(float v, int mask) { return fmaxf(v, __shfl_xor(v, mask)); }

// Largest of kLanes neighbours (8 or 16), in all of them; a NaN stays.
template <int kControl>
__device__ __forceinline__ float max_dpp(float v) {
  const int other = __builtin_amdgcn_update_dpp(0, bits_as<int>(v), kControl, 0xF, 0xF, true);
  return __builtin_elementwise_maximum(v, bits_as<float>(other));
}
template <int kLanes>
__device__ __forceinline__ float group_max(float v) {
  v = max_dpp<0xB1>(v);   // lane ^ 1
  v = max_dpp<0x4E>(v);   // lane ^ 2
  v = max_dpp<0x141>(v);  // the other 4 of 8, mirrored
  if constexpr (kLanes == 16) v = max_dpp<0x140>(v);  // the other 8 of 16, mirrored
  return v;
}

// Whole numbers in the order of the values: -0 equals 0, NaN is above all.
__device__ __forceinline__ uint32_t order_of(float f) {
  if (f != f) return 0xFFFFFFFFu;
  const uint32_t b = bits_as<uint32_t>(f + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t order) {
  return bits_as<float>(order & 0x80000000u ? order & 0x7FFFFFFFu : ~order);  // all ones: NaN
}

// A wave's span of a row, left in row `at` of `work`.
template <typename T>
__device__ __forceinline__ void take_span(const LogprobArgs& a, const Layout& lay, int64_t row, int span, float* work, int64_t at) {
  using S = Shape<T>;
  constexpr int V = S::kVec;
  const int lane = threadIdx.x & 63;
  const T* x = (const T*)a.logits + row * a.ld;
  const int shift = (int)(((uintptr_t)x / sizeof(T)) % V);
  const int first = span * S::kSpan + lane * V - shift;  // index of the lane's first value

  u32x4 raw[kUnits];
  if (span * S::kSpan - shift >= 0 && (span + 1) * S::kSpan - shift <= a.vocab) {
#pragma unroll
    for (int u = 0; u < kUnits; ++u) raw[u] = *reinterpret_cast<const u32x4*>(x + first + u * 64 * V);
  } else {
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int e = first + u * 64 * V;
      if (e >= 0 && e + V <= a.vocab) {
        raw[u] = *reinterpret_cast<const u32x4*>(x + e);
      } else {  // the row's ends: nothing outside it is read
        T part[V];
#pragma unroll
        for (int i = 0; i < V; ++i) part[i] = (e + i >= 0 && e + i < a.vocab) ? x[e + i] : (T)-kInf;
        __builtin_memcpy(&raw[u], part, 16);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  const int64_t t = a.targets[row];
  const bool known = t >= 0 && t < a.vocab;
  const float xt = known ? (float)x[t] : kInf;

  // The two passes over the registers unpack them anew: kept, the values
  // would take the registers of three waves in five.
  auto again = [&] {
#pragma unroll
    for (int u = 0; u < kUnits; ++u) asm volatile("" : "+v"(raw[u]));
  };
  float best[kUnits];  // of the lane's group of 64 values
  float m = -kInf;
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    float f[V];
    unpack(raw[u], f, (const T*)nullptr);
    float b = f[0];
#pragma unroll
    for (int i = 1; i < V; ++i) b = __builtin_elementwise_maximum(b, f[i]);  // a NaN stays
    best[u] = group_max<S::kLanes>(b);
    m = __builtin_elementwise_maximum(m, best[u]);
  }
  if constexpr (S::kLanes == 8) m = max_dpp<0x140>(m);
  m = __builtin_elementwise_maximum(m, __shfl_xor(m, 16));
  m = __builtin_elementwise_maximum(m, __shfl_xor(m, 32));
  again();

  const float ref = m == -kInf ? 0.f : m;
  float sum = 0.f, weighted = 0.f;
  int above = 0;
  if (fabsf(ref) < 0x1p20f) {
    // u = x log2 e - m log2 e in one step. The product with m is off by a
    // rounding, the same for all values, and comes off the sums again: `off` is
    // half a step of 2^20 log2 e at most, 2^-4, so that 2^off is near 1. From 2^31
    // on it passes 2^7, where 2^off leaves fp32. What lies below -1e38 (masks,
    // -inf) is at 0 either way.
    const float shift = ref * kLog2e, off = __builtin_fmaf(ref, kLog2e, -shift);
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      float f[V];
      unpack(raw[u], f, (const T*)nullptr);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        // the middle of three: a maximum in one instruction
        const float d = __builtin_fmaf(__builtin_amdgcn_fmed3f(f[i], -1e38f, kInf), kLog2e, -shift);
        const float p = __builtin_amdgcn_exp2f(d);
        sum += p;
        weighted = __builtin_fmaf(p, d, weighted);
        above += __popcll(__ballot(f[i] > xt));
      }
      __builtin_amdgcn_sched_barrier(0);  // registers
    }
    const float back = __builtin_amdgcn_exp2f(-off);
    weighted = (weighted - off * sum) * back;
    sum *= back;
    if (m == -kInf) sum = weighted = 0.f;
  } else {
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      float f[V];
      unpack(raw[u], f, (const T*)nullptr);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float d = (f[i] - ref) * kLog2e;
        const float p = __builtin_amdgcn_exp2f(d);
        sum += p;
        weighted = __builtin_fmaf(p, fmaxf(d, -256.f), weighted);  // 2^-256 is 0: no 0 x inf
        above += __popcll(__ballot(f[i] > xt));
      }
    }
  }
  if (m != m) sum = m;  // a NaN among the values: the row's
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    sum += __shfl_xor(sum, d);
    weighted += __shfl_xor(weighted, d);
  }
  if (lane == 0) {
    f32x4 s;
    s[0] = m == -kInf ? -kInf : ref;
    s[1] = sum;
    s[2] = weighted;
    s[3] = bits_as<float>(above);
    float* to = lay.stats(work, at, span);
#pragma unroll
    for (int i = 0; i < 4; ++i) to[i] = s[i];
    lay.tops(work, at)[span] = m;
  }
  if (a.top && lane % S::kLanes == 0) {
    float* to = lay.group(work, at, span) + lane / S::kLanes;
#pragma unroll
    for (int u = 0; u < kUnits; ++u) to[u * (64 / S::kLanes)] = best[u];
  }
}

template <typename T>
__global__ __launch_bounds__(256, 5) void spans_kernel(LogprobArgs a) {
  const Layout lay(a.vocab, Shape<T>::kSpan);
  const int span = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (span >= lay.spans) return;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) take_span<T>(a, lay, row, span, a.work, row);
}

// Lists of (order, place) in LDS, one list a wave; a key is larger where the
// value is, and among equal values where the place is lower. A list holds the
// groups, or where they are many the spans, then at most 64 members of each of
// `top` parts.
constexpr int kDirect = 1024;
inline int list_size(const Layout& lay, int top) {
  const int64_t groups = (int64_t)lay.spans * lay.groups;
  const int first = groups <= kDirect ? (int)groups : lay.spans;
  return top == 0 ? 0 : first > 64 * top ? first : 64 * top;
}

__device__ __forceinline__ uint64_t key_of(uint32_t order, uint32_t place) {
  return (uint64_t)order << 32 | (uint32_t)~place;
}

constexpr int kRow = 256;  // threads of a row's join

// What select_top() needs in LDS.
struct Selection {
  uint64_t most[kRow];
  int place[kRow];
  int counts[kRow / 64];
};

// Sorts out the `want` largest of list[0..n), all different, into out[0..want)
// in falling order; list is used up. All kRow threads.
__device__ void select_top(uint64_t* list, int n, int want, uint64_t* out, Selection& use) {
  const int me = threadIdx.x, wave = me >> 6;
  if (n > kRow) {
    // Of `lists` lists, the want-th of their largest is a floor under the want
    // largest of all, and seldom far under them where lists are three times as
    // many or more. Its search costs lists^2 / kRow steps, so there are no more.
    const int lists = want <= 24 ? 64 : want <= 48 ? 128 : 256;
    const int id = me & (lists - 1);
    uint64_t mine = 0;
    for (int i = me; i < n; i += kRow) mine = list[i] > mine ? list[i] : mine;
    use.most[me] = mine;
    use.place[me] = 0;
    __syncthreads();
    for (int i = id; i < kRow; i += lists) mine = use.most[i] > mine ? use.most[i] : mine;
    __syncthreads();
    if (me < lists) use.most[me] = mine;
    __syncthreads();
    const int share = lists * lists / kRow, first = me / lists * share;
    int place = 0;
#pragma unroll 8
    for (int j = 0; j < share; ++j) place += use.most[first + j] > mine;
    atomicAdd(&use.place[id], place);
    __syncthreads();
    if (me < lists && use.place[me] == want - 1) use.most[0] = mine;
    __syncthreads();
    const uint64_t low = use.most[0];
    int kept = 0;
    for (int i = 0; i < n; i += kRow) {
      const uint64_t key = i + me < n ? list[i + me] : 0;
      const bool in = i + me < n && key >= low;
      const uint64_t mask = __ballot(in);
      if ((me & 63) == 0) use.counts[wave] = __popcll(mask);
      __syncthreads();  // also: every thread has read this part of the list
      int at = kept;
#pragma unroll
      for (int w = 0; w < kRow / 64; ++w) {
        if (w < wave) at += use.counts[w];
        kept += use.counts[w];
      }
      if (in) list[at + __popcll(mask & ((1ull << (me & 63)) - 1))] = key;
      __syncthreads();
    }
    n = kept;
  }
  for (int i = me; i < n; i += kRow) {
    const uint64_t key = list[i];
    int place = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) place += list[j] > key;
    if (place < want) out[place] = key;
  }
}

// Joins the spans of a row, left in row `from` of `work`. All kRow threads; 64 do
// if there are no alternatives to find.
template <typename T>
__device__ __forceinline__ void join_row(const LogprobArgs& a, const Layout& lay, int64_t row, float* work, int64_t from_row) {
  using S = Shape<T>;
  const int me = threadIdx.x, lane = me & 63, wave = me >> 6;
  const T* x = (const T*)a.logits + row * a.ld;
  const int64_t t = a.targets[row];  // early: two loads that wait for one another
  const bool known = t >= 0 && t < a.vocab;
  const float xt = known ? (float)x[t] : 0.f;

  extern __shared__ uint64_t list[];  // list_size()
  __shared__ uint64_t out[3][kMaxTop];
  __shared__ Selection use;
  __shared__ int found;
  // groups of 64 where they are few enough to go through at once, else spans
  const bool direct = (int64_t)lay.spans * lay.groups <= kDirect;
  int n = direct ? lay.spans * lay.groups : lay.spans;
  if (a.top) {
    const float* from = direct ? lay.group(work, from_row, 0) : lay.tops(work, from_row);
    for (int i = me; i < n; i += kRow) list[i] = key_of(order_of(from[i]), i);
  }

  // the spans' sums against one reference, each lane's in the spans' order; all
  // waves alike
  const float* stats = lay.stats(work, from_row, 0);
  float ref = -kInf;
  for (int s = lane; s < lay.spans; s += 64) ref = fmaxf(ref, stats[s * 4]);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) ref = max_xor(ref, d);
  float sum = 0.f, weighted = 0.f;
  int64_t above = 0;
  for (int s = lane; s < lay.spans; s += 64) {
    const float r = stats[s * 4], q = stats[s * 4 + 1], w = stats[s * 4 + 2];
    above += bits_as<int>(stats[s * 4 + 3]);
    if (r == -kInf && !(q != q)) continue;  // nothing allowed in this span
    const float d = (r - ref) * kLog2e;
    const float f = __builtin_amdgcn_exp2f(d);
    sum += q * f;
    weighted += f * __builtin_fmaf(q, d < -256.f ? -256.f : d, w);
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    sum += __shfl_xor(sum, d);
    weighted += __shfl_xor(weighted, d);
    above += __shfl_xor(above, d);
  }
  const float log_sum = __builtin_amdgcn_logf(sum) * kLn2;
  const bool empty = ref == -kInf && !(sum != sum);  // every token masked
  auto logp = [&](float v) { return empty ? -kInf : (v - ref) - log_sum; };
  if (me == 0) {
    a.logprob[row] = known ? logp(xt) : t < 0 ? 0.f : __builtin_nanf("");
    a.entropy[row] = empty ? 0.f : log_sum - weighted / sum * kLn2;
    a.rank[row] = known ? above : -1;
  }
  if (a.top == 0) return;

  const int want = a.top;
  const int shift = (int)(((uintptr_t)x / sizeof(T)) % S::kVec);
  int got = 0;
#pragma unroll 1
  for (int level = direct ? 1 : 0, first_level = level; level <= 2; ++level) {
    if (level > first_level) {
      // members of the last level's parts, a part a wave and turn; those under
      // its least are left out, and what else a part's turn finds follows in the
      // list wherever the waves get to (the keys order it)
      const int parts = got;
      const int size = level == 1 ? S::kGroups : 64;
      const uint32_t least = parts == want ? (uint32_t)(out[level - 1][parts - 1] >> 32) : 0u;
      constexpr int kBatch = 4;
      if (me == 0) found = 0;
      __syncthreads();
#pragma unroll 1
      for (int first = wave; first < parts; first += kBatch * (kRow / 64)) {
        uint32_t place[kBatch];
        float value[kBatch];
        bool in[kBatch];
#pragma unroll
        for (int q = 0; q < kBatch; ++q) {  // loads without a branch, so that none waits for another
          const int p = first + q * (kRow / 64);
          const uint32_t part = ~(uint32_t)out[level - 1][p < parts ? p : parts - 1];
          place[q] = part * size + lane - (level == 1 ? 0 : shift);
          in[q] = p < parts && lane < size && (level == 1 || place[q] < (uint32_t)a.vocab);
        }
        if (level == 1) {
          const float* from = lay.group(work, from_row, 0);
#pragma unroll
          for (int q = 0; q < kBatch; ++q) value[q] = from[in[q] ? place[q] : 0];
        } else {
          T raw[kBatch];
#pragma unroll
          for (int q = 0; q < kBatch; ++q) raw[q] = x[in[q] ? place[q] : 0];
#pragma unroll
          for (int q = 0; q < kBatch; ++q) value[q] = (float)raw[q];
        }
#pragma unroll
        for (int q = 0; q < kBatch; ++q) {
          const uint32_t order = order_of(value[q]);
          const bool kept = in[q] && order >= least;
          const uint64_t mask = __ballot(kept);
          int at = 0;
          if (lane == 0 && mask) at = atomicAdd(&found, __popcll(mask));
          at = __builtin_amdgcn_readfirstlane(at);
          if (kept) list[at + __popcll(mask & ((1ull << lane) - 1))] = key_of(order, place[q]);
        }
      }
      __syncthreads();
      n = found;
    }
    __syncthreads();
    got = n < want ? n : want;
    select_top(list, n, got, out[level], use);
    __syncthreads();
  }
  for (int i = me; i < want; i += kRow) {
    const uint64_t key = out[2][i];
    a.top_ids[row * want + i] = ~(uint32_t)key;
    a.top_logprobs[row * want + i] = logp(value_of((uint32_t)(key >> 32)));
  }
}

template <typename T>
__global__ __launch_bounds__(kRow) void rows_kernel(LogprobArgs a) {
  const Layout lay(a.vocab, Shape<T>::kSpan);
  join_row<T>(a, lay, blockIdx.x, a.work, blockIdx.x);
}

// Few rows of few spans: a workgroup takes a row's spans, a wave each, and joins
// them from the LDS, which saves a launch and the workspace (a pass of 256 x 32000
// bf16 with 20 alternatives: 13.1 us, 257 rows in two launches 18.0). Of more rows
// than compute units, workgroups wait for the joins of others (512 x 1000: 25.8 in
// one launch, 17.3 in two), and with two spans a wave a row is slower too (1 x
// 130001: 23.9, 17.1). Both ways compute the same.
constexpr int kFewSpans = 16;
template <typename T>
__global__ __launch_bounds__(kFewSpans * 64) void row_kernel(LogprobArgs a) {
  using S = Shape<T>;
  __shared__ float work[kFewSpans * (5 + S::kGroups)];
  const Layout lay(a.vocab, S::kSpan);
  const int wave = threadIdx.x >> 6;
  if (wave < lay.spans) take_span<T>(a, lay, blockIdx.x, wave, work, 0);
  __syncthreads();
  if (wave >= kRow / 64) return;  // barriers wait for the waves that are left
  join_row<T>(a, lay, blockIdx.x, work, 0);
}

bool in_one(int64_t rows, const Layout& lay) { return rows <= 256 && lay.spans <= kFewSpans; }

template <typename T>
hipError_t launch(const LogprobArgs& a, hipStream_t stream) {
  const Layout lay(a.vocab, Shape<T>::kSpan);
  const size_t lds = sizeof(uint64_t) * list_size(lay, a.top);
  if (in_one(a.rows, lay)) {
    row_kernel<T><<<dim3((unsigned)a.rows), kFewSpans * 64, lds, stream>>>(a);
    return hipGetLastError();
  }
  const int across = (lay.spans + 3) / 4;
  const int64_t down = (1 << 24) / across - 1;  // a launch has fewer than 2^32 threads
  const int64_t most = down < 65535 ? down : 65535;
  const dim3 grid(across, (unsigned)(a.rows < most ? a.rows : most));
  spans_kernel<T><<<grid, 256, 0, stream>>>(a);
  if (hipError_t e = hipGetLastError()) return e;
  rows_kernel<T><<<dim3((unsigned)a.rows), a.top ? kRow : 64, lds, stream>>>(a);
  return hipGetLastError();
}

}  // namespace

int64_t logprob_workspace(int64_t rows, int vocab, int dtype) {
  const int span = dtype == kF32 ? Shape<float>::kSpan : Shape<__bf16>::kSpan;
  const Layout lay(vocab, span);
  return in_one(rows, lay) ? 0 : rows * lay.row;
}

hipError_t launch_token_logprobs(const LogprobArgs& a, hipStream_t stream) {
  if (a.dtype == kBF16) return launch<__bf16>(a, stream);
  if (a.dtype == kF16) return launch<_Float16>(a, stream);
  return launch<float>(a, stream);
}

}  // namespace serving
