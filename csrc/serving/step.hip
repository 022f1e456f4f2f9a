// The serving diagnostic: 32 sequences of 65 to 2000 tokens take one step
// through a projection to queries, keys and values (6144 x 4096 in 4 bits), the
// append, the attention (32 heads on 8 cached ones of 128, pages of 64), an
// output projection (4096 x 4096), a head (32768 x 4096) and the log
// probabilities with 5 alternatives.
//
// Weights, prompts and tokens come from a hash that host and device share, so
// that an oracle needs no copy of the 4-bit weights. Each operator is checked
// against its own inputs as they were on the device, at places drawn from the
// seed; bounds are those of the types' roundings. A second run from the same
// state has to give the same bits everywhere.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <stdexcept>

#include "device.h"
#include "serving.h"
#include "step.h"

namespace serving {
namespace {

constexpr int kBatch = 32, kWidth = 4096, kQHeads = 32, kHeads = 8, kDim = 128, kPage = 64;
constexpr int kGroup = 128, kVocab = 32768, kTop = 5, kLongest = 2000;
constexpr int kQkv = (kQHeads + 2 * kHeads) * kDim, kOut = kQHeads * kDim;
constexpr int kBlocks = (kLongest + kPage) / kPage;

void check(hipError_t e, const char* what) {
  if (e != hipSuccess) throw std::runtime_error(std::string(what) + " failed: " + hipGetErrorString(e));
}

__host__ __device__ inline uint32_t hash(uint32_t a, uint32_t b) {
  uint32_t h = a * 0x9E3779B1u ^ (b + 0x7F4A7C15u) * 0x85EBCA77u;
  h ^= h >> 15;
  h *= 0x2C1B3C6Du;
  h ^= h >> 12;
  h *= 0x297A2D39u;
  return h ^ h >> 15;
}
// Whole numbers -7..7 over 4: bf16 holds them exactly.
__host__ __device__ inline float small_value(uint32_t h) { return (float)((int)(h % 15u) - 7) * 0.25f; }
__host__ __device__ inline float scale_value(uint32_t h) { return (float)(1 + h % 4u) * 0x1p-9f; }

__global__ void fill_bytes(uint32_t* to, int64_t words, uint32_t seed) {
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < words; i += (int64_t)gridDim.x * blockDim.x)
    to[i] = hash(seed, (uint32_t)i);
}
__global__ void fill_values(__bf16* to, int64_t n, uint32_t seed, bool scales) {
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
    const uint32_t h = hash(seed, (uint32_t)i);
    to[i] = (__bf16)(scales ? scale_value(h) : small_value(h));
  }
}

struct Buffer {
  void* p = nullptr;
  size_t bytes = 0;
  explicit Buffer(size_t n) : bytes(n) { check(hipMalloc(&p, n ? n : 16), "hipMalloc"); }
  ~Buffer() { (void)hipFree(p); }
  Buffer(const Buffer&) = delete;
  Buffer& operator=(const Buffer&) = delete;
  template <typename T>
  T* as() const { return static_cast<T*>(p); }
  template <typename T>
  std::vector<T> read() const {
    std::vector<T> v(bytes / sizeof(T));
    check(hipMemcpy(v.data(), p, v.size() * sizeof(T), hipMemcpyDeviceToHost), "hipMemcpy");
    return v;
  }
  template <typename T>
  void write(const std::vector<T>& v) {
    check(hipMemcpy(p, v.data(), v.size() * sizeof(T), hipMemcpyHostToDevice), "hipMemcpy");
  }
};

struct Stream {
  hipStream_t s = nullptr;
  Stream() { check(hipStreamCreate(&s), "hipStreamCreate"); }
  ~Stream() { (void)hipStreamDestroy(s); }
};
struct Event {
  hipEvent_t e = nullptr;
  Event() { check(hipEventCreate(&e), "hipEventCreate"); }
  ~Event() { (void)hipEventDestroy(e); }
};

// The device the caller had is current again behind the check.
struct OnDevice {
  int before = 0;
  explicit OnDevice(int device) {
    check(hipGetDevice(&before), "hipGetDevice");
    check(hipSetDevice(device), "hipSetDevice");
  }
  ~OnDevice() { (void)hipSetDevice(before); }
};

double of_bf16(uint16_t b) {
  const uint32_t w = (uint32_t)b << 16;
  float f;
  std::memcpy(&f, &w, 4);
  return f;
}
double of_e4m3(uint8_t c) {
  const int e = c >> 3 & 15, m = c & 7;
  if ((c & 127) == 127) return NAN;
  const double v = e ? std::ldexp(8 + m, e - 10) : std::ldexp(m, -9);
  return c & 128 ? -v : v;
}
// Half a step of e4m3 at magnitude v (v at most 448).
double half_step_e4m3(double v) { return std::ldexp(1.0, std::max(v > 0 ? std::ilogb(v) : -6, -6) - 4); }

struct Weights {
  int n, k;
  uint32_t seed;
  Buffer codes, scales;
  Weights(int n_, int k_, uint32_t seed_, hipStream_t s)
      : n(n_), k(k_), seed(seed_), codes((size_t)(n_ / 16) * (k_ / 128) * 1024), scales((size_t)n_ / 16 * (k_ / kGroup) * 32) {
    fill_bytes<<<1024, 256, 0, s>>>(codes.as<uint32_t>(), (int64_t)codes.bytes / 4, seed);
    fill_values<<<256, 256, 0, s>>>(scales.as<__bf16>(), (int64_t)scales.bytes / 2, seed + 1, true);
    check(hipGetLastError(), "fill");
  }
  W4Args args(const void* x, void* y, void* work) const {
    W4Args a{};
    a.x = x;
    a.codes = codes.as<uint8_t>();
    a.scales = scales.p;
    a.y = y;
    a.ldx = k;
    a.ldy = n;
    a.m = kBatch;
    a.n = n;
    a.k = k;
    a.group = kGroup;
    a.dtype = kBF16;
    a.work = work;
    return a;
  }
  double weight(int row, int col) const {
    const int b = col / 128, c = col % 128, j = c / 32, g = c % 32 / 8, e = c % 8;
    const int nibble = e / 2 + 4 * (e % 2);
    const int64_t word = ((((int64_t)(row / 16) * (k / 128) + b) * 64 + g * 16 + row % 16) * 16) / 4 + j;
    const int q = hash(seed, (uint32_t)word) >> (4 * nibble) & 15;
    const int64_t at = ((int64_t)(row / 16) * (k / kGroup) + col / kGroup) * 16 + row % 16;
    return (q - 8) * (double)scale_value(hash(seed + 1, (uint32_t)at));
  }
};

class Checker {
 public:
  Checker(StepResult& r, double offset) : r_(r), offset_(offset) {}
  void near(const char* what, double got, double want, double bound) {
    ++r_.checked;
    want += offset_;
    if (std::isfinite(got) && std::fabs(got - want) <= bound) return;
    char text[160];
    std::snprintf(text, sizeof text, "%s: %.9g, expected %.9g within %.3g", what, got, want, bound);
    fail(text);
  }
  void same(const char* what, int64_t got, int64_t want) {
    ++r_.checked;
    if (got == want) return;
    char text[160];
    std::snprintf(text, sizeof text, "%s: %lld, expected %lld", what, (long long)got, (long long)want);
    fail(text);
  }
  void bits(const char* what, const std::vector<uint8_t>& a, const std::vector<uint8_t>& b) {
    int64_t off = 0;
    for (size_t i = 0; i < a.size(); ++i) off += a[i] != b[i];
    r_.checked += (int64_t)a.size();
    if (!off) return;
    char text[160];
    std::snprintf(text, sizeof text, "%s: %lld bytes differ between two runs", what, (long long)off);
    r_.failures += off - 1;
    fail(text);
  }

 private:
  void fail(const char* text) {
    ++r_.failures;
    if (r_.messages.size() < 8) r_.messages.emplace_back(text);
  }
  StepResult& r_;
  double offset_;
};

}  // namespace

StepResult run_step(int device, int iters, uint32_t seed, double oracle_offset) {
  StepResult result;
  Checker verify(result, oracle_offset);
  OnDevice on(device);
  Stream stream;
  const hipStream_t s = stream.s;

  Weights qkv(kQkv, kWidth, seed + 10, s), proj(kWidth, kOut, seed + 20, s), head(kVocab, kWidth, seed + 30, s);
  Buffer x((size_t)kBatch * kWidth * 2), y((size_t)kBatch * kQkv * 2), o((size_t)kBatch * kOut * 2);
  Buffer hidden((size_t)kBatch * kWidth * 2), logits((size_t)kBatch * kVocab * 2);
  Buffer lse((size_t)kBatch * kQHeads * 4);
  fill_values<<<256, 256, 0, s>>>(x.as<__bf16>(), kBatch * kWidth, seed + 40, false);

  // lengths 64 .. kLongest - 1 before the step; pages dealt out by the hash
  std::vector<int32_t> before(kBatch), lens(kBatch), starts(kBatch + 1, 0), table(kBatch * kBlocks);
  for (int b = 0; b < kBatch; ++b) {
    before[b] = 64 + (kLongest - 65) * b / (kBatch - 1);
    lens[b] = before[b] + 1;
    starts[b + 1] = starts[b] + before[b];
  }
  for (int i = 0; i < kBatch * kBlocks; ++i) table[i] = i;
  for (int i = kBatch * kBlocks - 1; i > 0; --i) std::swap(table[i], table[hash(seed + 50, i) % (uint32_t)(i + 1)]);
  const int pages = kBatch * kBlocks;
  const size_t cells = (size_t)pages * kHeads * kPage * kDim;
  Buffer kc(cells), vc(cells), ks((size_t)pages * kHeads * 4), vs((size_t)pages * kHeads * 4);
  Buffer d_before(kBatch * 4), d_lens(kBatch * 4), d_starts((kBatch + 1) * 4), d_table(table.size() * 4);
  d_before.write(before);
  d_lens.write(lens);
  d_starts.write(starts);
  d_table.write(table);
  fill_bytes<<<1024, 256, 0, s>>>(kc.as<uint32_t>(), (int64_t)cells / 4, seed + 60);  // an earlier owner's
  fill_bytes<<<1024, 256, 0, s>>>(vc.as<uint32_t>(), (int64_t)cells / 4, seed + 61);

  CacheArgs cache{};
  cache.k = kc.as<uint8_t>();
  cache.v = vc.as<uint8_t>();
  cache.k_scale = ks.as<float>();
  cache.v_scale = vs.as<float>();
  cache.table = d_table.as<int32_t>();
  cache.ldt = kBlocks;
  cache.pages = pages;
  cache.heads = kHeads;
  cache.page = kPage;
  cache.dim = kDim;
  cache.batch = kBatch;
  cache.blocks = kBlocks;

  AppendArgs prompt{};
  prompt.c = cache;
  prompt.c.lens = d_before.as<int32_t>();
  prompt.c.starts = d_starts.as<int32_t>();
  prompt.c.rows = starts[kBatch];
  Buffer prompts((size_t)prompt.c.rows * 2 * kHeads * kDim * 2);
  fill_values<<<1024, 256, 0, s>>>(prompts.as<__bf16>(), (int64_t)prompts.bytes / 2, seed + 70, false);
  prompt.k_new = prompts.p;
  prompt.v_new = prompts.as<__bf16>() + kHeads * kDim;
  prompt.k_row = prompt.v_row = 2 * kHeads * kDim;
  prompt.k_head = prompt.v_head = kDim;
  prompt.dtype = kBF16;
  check(launch_cache_append(prompt, s), "cache_append");

  AppendArgs token{};
  token.c = cache;
  token.c.lens = d_lens.as<int32_t>();
  token.c.rows = kBatch;
  token.k_new = y.as<__bf16>() + kOut;
  token.v_new = y.as<__bf16>() + kOut + kHeads * kDim;
  token.k_row = token.v_row = kQkv;
  token.k_head = token.v_head = kDim;
  token.dtype = kBF16;

  AttentionArgs attention{};
  attention.c = token.c;
  attention.q = y.p;
  attention.out = o.p;
  attention.lse = lse.as<float>();
  attention.q_row = kQkv;
  attention.q_head = attention.o_head = kDim;
  attention.o_row = kOut;
  attention.q_heads = kQHeads;
  attention.scale = 1.f / std::sqrt((float)kDim);
  attention.dtype = kBF16;
  attention.longest = kLongest;
  Buffer split(plan_attention(attention).floats * 4);
  attention.work = split.as<float>();

  std::vector<int64_t> targets(kBatch);
  for (int b = 0; b < kBatch; ++b) targets[b] = hash(seed + 80, b) % kVocab;
  Buffer d_targets(kBatch * 8), logprob(kBatch * 4), entropy(kBatch * 4), rank(kBatch * 8);
  Buffer top_ids(kBatch * kTop * 8), top_logprobs(kBatch * kTop * 4);
  Buffer spans(logprob_workspace(kBatch, kVocab, kBF16) * 4);
  d_targets.write(targets);
  LogprobArgs tokens{};
  tokens.logits = logits.p;
  tokens.targets = d_targets.as<int64_t>();
  tokens.logprob = logprob.as<float>();
  tokens.entropy = entropy.as<float>();
  tokens.rank = rank.as<int64_t>();
  tokens.top_ids = top_ids.as<int64_t>();
  tokens.top_logprobs = top_logprobs.as<float>();
  tokens.work = spans.as<float>();
  tokens.ld = kVocab;
  tokens.rows = kBatch;
  tokens.vocab = kVocab;
  tokens.top = kTop;
  tokens.dtype = kBF16;

  const W4Args w_qkv0 = qkv.args(x.p, y.p, nullptr), w_proj0 = proj.args(o.p, hidden.p, nullptr),
               w_head0 = head.args(hidden.p, logits.p, nullptr);
  Buffer pack(std::max({w4_workspace(w_qkv0), w4_workspace(w_proj0), w4_workspace(w_head0), (int64_t)16}));
  const W4Args w_qkv = qkv.args(x.p, y.p, pack.p), w_proj = proj.args(o.p, hidden.p, pack.p),
               w_head = head.args(hidden.p, logits.p, pack.p);

  Event mark[5];
  double spent[4] = {};
  auto step = [&](bool timed) {
    auto at = [&](int i) {
      if (timed) check(hipEventRecord(mark[i].e, s), "hipEventRecord");
    };
    at(0);
    check(launch_w4_matmul(w_qkv, s), "w4_matmul");
    at(1);
    check(launch_cache_append(token, s), "cache_append");
    check(launch_cache_attention(attention, s), "cache_attention");
    at(2);
    check(launch_w4_matmul(w_proj, s), "w4_matmul");
    check(launch_w4_matmul(w_head, s), "w4_matmul");
    at(3);
    check(launch_token_logprobs(tokens, s), "token_logprobs");
    at(4);
    if (!timed) return;
    check(hipEventSynchronize(mark[4].e), "hipEventSynchronize");
    for (int i = 0; i < 4; ++i) {
      float ms = 0;
      check(hipEventElapsedTime(&ms, mark[i].e, mark[i + 1].e), "hipEventElapsedTime");
      spent[i] += ms;
    }
  };
  auto outputs = [&] {
    std::vector<std::vector<uint8_t>> v;
    for (const Buffer* b : {&y, &o, &lse, &hidden, &logits, &logprob, &entropy, &rank, &top_ids, &top_logprobs})
      v.push_back(b->read<uint8_t>());
    return v;
  };

  step(false);
  check(hipStreamSynchronize(s), "hipStreamSynchronize");
  const auto first = outputs();
  step(false);
  check(hipStreamSynchronize(s), "hipStreamSynchronize");
  const auto second = outputs();
  const char* names[] = {"projections", "attention", "lse", "hidden", "logits", "logprob", "entropy", "rank", "top ids", "top logprobs"};
  for (size_t i = 0; i < first.size(); ++i) verify.bits(names[i], first[i], second[i]);

  const int steps = iters < 1 ? 1 : iters;
  Event begin, end;
  check(hipEventRecord(begin.e, s), "hipEventRecord");
  for (int i = 0; i < steps; ++i) step(false);
  check(hipEventRecord(end.e, s), "hipEventRecord");
  check(hipEventSynchronize(end.e), "hipEventSynchronize");
  float ms = 0;
  check(hipEventElapsedTime(&ms, begin.e, end.e), "hipEventElapsedTime");
  for (int i = 0; i < steps; ++i) step(true);
  int64_t held = 0;
  for (int b = 0; b < kBatch; ++b) held += lens[b];
  const double product_bytes = (double)(qkv.codes.bytes + proj.codes.bytes + head.codes.bytes);
  const double cache_bytes = (double)held * kHeads * kDim * 2, logit_bytes = (double)logits.bytes;
  result.ms = ms / steps;
  result.gbps = (product_bytes + cache_bytes + logit_bytes) / result.ms / 1e6;
  result.product_gbps = product_bytes / ((spent[0] + spent[2]) / steps) / 1e6;
  result.attention_gbps = cache_bytes / (spent[1] / steps) / 1e6;
  result.logprob_gbps = logit_bytes / (spent[3] / steps) / 1e6;

  // ---- oracles, each on the operator's own inputs ----
  const auto hx = x.read<uint16_t>(), hy = y.read<uint16_t>(), ho = o.read<uint16_t>(), hh = hidden.read<uint16_t>(),
             hl = logits.read<uint16_t>();
  constexpr double kHalf = 0x1p-9;  // half a step of bf16
  auto product = [&](const char* what, const Weights& w, const std::vector<uint16_t>& in, const std::vector<uint16_t>& out) {
    for (int i = 0; i < 96; ++i) {
      const int m = hash(seed + 90, i) % kBatch, n = i < 4 ? (i & 1 ? w.n - 1 : 0) : (int)(hash(seed + 91, i) % (uint32_t)w.n);
      double want = 0, size = 0;
      for (int k = 0; k < w.k; ++k) {
        const double v = of_bf16(in[(size_t)m * w.k + k]);
        want += v * w.weight(n, k);
        size += std::fabs(v) * 47 * 0x1p-7;  // with 16 + q and 24, at the largest scale
      }
      // fp32 sums of a group's 2 x 128 terms, then of the groups and the waves
      const double sums = (2 * kGroup + w.k / kGroup + 16) * 0x1p-24 * size;
      verify.near(what, of_bf16(out[(size_t)m * w.n + n]), want, 2 * kHalf * std::fabs(want) + sums + 1e-30);
    }
  };
  product("projection", qkv, hx, hy);
  product("output projection", proj, ho, hh);
  product("head", head, hh, hl);

  const auto hks = ks.read<float>(), hvs = vs.read<float>();
  std::vector<uint8_t> page_k((size_t)kPage * kDim), page_v((size_t)kPage * kDim);
  const auto hlse = lse.read<float>();
  for (int i = 0; i < 6; ++i) {
    const int b = i == 0 ? 0 : i == 1 ? kBatch - 1 : (int)(hash(seed + 100, i) % kBatch), h = hash(seed + 101, i) % kHeads;
    const int len = lens[b];
    std::vector<double> K((size_t)len * kDim), V((size_t)len * kDim);
    for (int block = 0; block * kPage < len; ++block) {
      const int64_t ph = (int64_t)table[b * kBlocks + block] * kHeads + h;
      check(hipMemcpy(page_k.data(), kc.as<uint8_t>() + ph * kPage * kDim, page_k.size(), hipMemcpyDeviceToHost), "hipMemcpy");
      check(hipMemcpy(page_v.data(), vc.as<uint8_t>() + ph * kPage * kDim, page_v.size(), hipMemcpyDeviceToHost), "hipMemcpy");
      for (int t = 0; t < kPage && block * kPage + t < len; ++t)
        for (int d = 0; d < kDim; ++d) {
          K[(size_t)(block * kPage + t) * kDim + d] = of_e4m3(page_k[t * kDim + d]) * hks[ph];
          V[(size_t)(block * kPage + t) * kDim + d] = of_e4m3(page_v[d * kPage + t]) * hvs[ph];
        }
    }
    // what the append left of a prompt's token and of the step's
    for (int which = 0; which < 2; ++which) {
      const int t = which ? len - 1 : (int)(hash(seed + 102, i) % (uint32_t)before[b]);
      const int64_t ph = (int64_t)table[b * kBlocks + t / kPage] * kHeads + h;
      for (int d = 0; d < kDim; ++d) {
        const int64_t row = starts[b] + t;
        const double k_in = which ? of_bf16(hy[(size_t)b * kQkv + kOut + h * kDim + d])
                                  : small_value(hash(seed + 70, (uint32_t)((row * 2 * kHeads + h) * kDim + d)));
        const double v_in = which ? of_bf16(hy[(size_t)b * kQkv + kOut + (kHeads + h) * kDim + d])
                                  : small_value(hash(seed + 70, (uint32_t)((row * 2 * kHeads + kHeads + h) * kDim + d)));
        // a prompt's code is rounded again where its page's scale has grown
        const double f = which ? 1.01 : 2.01;
        verify.near("cached key", K[(size_t)t * kDim + d], k_in, f * hks[ph] * half_step_e4m3(std::fabs(k_in) / hks[ph]));
        verify.near("cached value", V[(size_t)t * kDim + d], v_in, f * hvs[ph] * half_step_e4m3(std::fabs(v_in) / hvs[ph]));
      }
    }
    const int q = h * (kQHeads / kHeads) + (int)(hash(seed + 103, i) % (kQHeads / kHeads));
    std::vector<double> score(len);
    double top = -INFINITY, size = 0;
    for (int t = 0; t < len; ++t) {
      double dot = 0, mag = 0;
      for (int d = 0; d < kDim; ++d) {
        const double p = of_bf16(hy[(size_t)b * kQkv + q * kDim + d]) * K[(size_t)t * kDim + d];
        dot += p;
        mag += std::fabs(p);
      }
      score[t] = dot * attention.scale;
      size = std::max(size, mag * attention.scale);
      top = std::max(top, score[t]);
    }
    double total = 0;
    for (int t = 0; t < len; ++t) total += std::exp(score[t] - top);
    const double want_lse = top + std::log(total);
    // a score's fp32 sum and power; the weights' sum; fp16 weights
    const double rel = std::expm1((size * (kDim + 8) + std::fabs(top) * 4) * 0x1p-24) + 0x1p-21 + (len + 8) * 0x1p-24;
    verify.near("lse", hlse[(size_t)b * kQHeads + q], want_lse, rel + std::fabs(want_lse) * 0x1p-22);
    for (int d = 0; d < kDim; ++d) {
      double want = 0, mass = 0, largest = 0;
      for (int t = 0; t < len; ++t) {
        const double p = std::exp(score[t] - want_lse), v = V[(size_t)t * kDim + d];
        want += p * v;
        mass += p * std::fabs(v);
        largest = std::max(largest, p * std::fabs(v));
      }
      verify.near("attention", of_bf16(ho[(size_t)b * kOut + q * kDim + d]), want,
                  2 * kHalf * std::fabs(want) + mass * (0x1p-11 + 2 * rel) + (mass + 1) * len * 0x1p-24 + 1e-30);
    }
  }

  const auto hlp = logprob.read<float>(), hent = entropy.read<float>(), htop = top_logprobs.read<float>();
  const auto hrank = rank.read<int64_t>(), hids = top_ids.read<int64_t>();
  for (int b = 0; b < kBatch; b += 5) {
    std::vector<double> v(kVocab);
    double top = -INFINITY, total = 0, mean = 0;
    for (int i = 0; i < kVocab; ++i) top = std::max(top, v[i] = of_bf16(hl[(size_t)b * kVocab + i]));
    for (int i = 0; i < kVocab; ++i) total += std::exp(v[i] - top);
    for (int i = 0; i < kVocab; ++i) mean += std::exp(v[i] - top) / total * (v[i] - top);
    const double norm = top + std::log(total), bound = 128 * 0x1p-24;
    int64_t above = 0;
    for (int i = 0; i < kVocab; ++i) above += v[i] > v[targets[b]];
    const double lp = v[targets[b]] - norm;
    verify.near("logprob", hlp[b], lp, bound + (std::fabs(lp) + 20) * 0x1p-22);
    verify.near("entropy", hent[b], std::log(total) - mean, bound * 24 + 20 * 0x1p-20);
    verify.same("rank", hrank[b], above);
    std::vector<int> order(kVocab);
    for (int i = 0; i < kVocab; ++i) order[i] = i;
    std::partial_sort(order.begin(), order.begin() + kTop, order.end(),
                      [&](int p, int q) { return v[p] != v[q] ? v[p] > v[q] : p < q; });
    for (int i = 0; i < kTop; ++i) {
      verify.same("alternative", hids[(size_t)b * kTop + i], order[i]);
      const double want = v[order[i]] - norm;
      verify.near("alternative's logprob", htop[(size_t)b * kTop + i], want, bound + (std::fabs(want) + 20) * 0x1p-22);
    }
  }
  return result;
}

}  // namespace serving
