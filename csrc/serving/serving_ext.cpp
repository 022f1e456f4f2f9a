// Python binding of the serving operators. Pointers, sizes and streams come as
// whole numbers from gpud_amd/diag/serving.py, which has checked them; errors
// of the runtime leave as exceptions.
#include <hip/hip_runtime.h>
#include <pybind11/pybind11.h>

#include <pybind11/stl.h>

#include <stdexcept>
#include <string>
#include <vector>

#include "geometry.h"
#include "serving.h"
#include "step.h"

namespace py = pybind11;
using namespace serving;

namespace {

template <typename T>
T* ptr(uintptr_t p) {
  return reinterpret_cast<T*>(p);
}

// Makes `device` current for a launch and the caller's again behind it.
class OnDevice {
 public:
  explicit OnDevice(int device) {
    check(hipGetDevice(&before_), "hipGetDevice");
    if (before_ != device) {
      check(hipSetDevice(device), "hipSetDevice");
      moved_ = true;
    }
  }
  ~OnDevice() {
    if (moved_) (void)hipSetDevice(before_);
  }
  OnDevice(const OnDevice&) = delete;
  OnDevice& operator=(const OnDevice&) = delete;

  static void check(hipError_t e, const char* what) {
    if (e != hipSuccess) throw std::runtime_error(std::string(what) + " failed: " + hipGetErrorString(e));
  }

 private:
  int before_ = 0;
  bool moved_ = false;
};

hipStream_t stream_of(uintptr_t s) { return reinterpret_cast<hipStream_t>(s); }

W4Args w4_args(uintptr_t x, int64_t ldx, int m, int n, int k, int group, int dtype) {
  W4Args a{};
  a.x = ptr<void>(x);
  a.ldx = ldx;
  a.m = m;
  a.n = n;
  a.k = k;
  a.group = group;
  a.dtype = dtype;
  return a;
}

int64_t w4_work(uintptr_t x, int64_t ldx, int m, int n, int k, int group, int dtype) {
  return w4_workspace(w4_args(x, ldx, m, n, k, group, dtype));
}

void w4_matmul(int device, uintptr_t stream, uintptr_t x, int64_t ldx, int m, int n, int k, int group, int dtype,
               uintptr_t codes, uintptr_t scales, uintptr_t zeros, uintptr_t y, int64_t ldy, uintptr_t work) {
  W4Args a = w4_args(x, ldx, m, n, k, group, dtype);
  a.codes = ptr<uint8_t>(codes);
  a.scales = ptr<void>(scales);
  a.zeros = ptr<uint8_t>(zeros);
  a.y = ptr<void>(y);
  a.ldy = ldy;
  a.work = ptr<void>(work);
  OnDevice on(device);
  OnDevice::check(launch_w4_matmul(a, stream_of(stream)), "w4_matmul");
}

CacheArgs cache_args(const py::tuple& t) {
  CacheArgs c{};
  c.k = ptr<uint8_t>(t[0].cast<uintptr_t>());
  c.v = ptr<uint8_t>(t[1].cast<uintptr_t>());
  c.k_scale = ptr<float>(t[2].cast<uintptr_t>());
  c.v_scale = ptr<float>(t[3].cast<uintptr_t>());
  c.table = ptr<int32_t>(t[4].cast<uintptr_t>());
  c.lens = ptr<int32_t>(t[5].cast<uintptr_t>());
  c.starts = ptr<int32_t>(t[6].cast<uintptr_t>());
  c.ldt = t[7].cast<int64_t>();
  c.pages = t[8].cast<int>();
  c.heads = t[9].cast<int>();
  c.page = t[10].cast<int>();
  c.dim = t[11].cast<int>();
  c.batch = t[12].cast<int>();
  c.blocks = t[13].cast<int>();
  c.rows = t[14].cast<int>();
  return c;
}

void cache_append(int device, uintptr_t stream, const py::tuple& cache, uintptr_t k, int64_t k_row, int64_t k_head,
                  uintptr_t v, int64_t v_row, int64_t v_head, int dtype) {
  AppendArgs a{};
  a.c = cache_args(cache);
  a.k_new = ptr<void>(k);
  a.k_row = k_row;
  a.k_head = k_head;
  a.v_new = ptr<void>(v);
  a.v_row = v_row;
  a.v_head = v_head;
  a.dtype = dtype;
  OnDevice on(device);
  OnDevice::check(launch_cache_append(a, stream_of(stream)), "cache_append");
}

int64_t attention_floats(int rows, int batch, int heads, int q_heads, int dim, bool ragged, int window, int64_t longest) {
  AttentionArgs a{};
  static const int32_t some = 0;
  a.c.rows = rows;
  a.c.batch = batch;
  a.c.heads = heads;
  a.c.dim = dim;
  a.c.starts = ragged ? &some : nullptr;  // only whether it is there counts
  a.q_heads = q_heads;
  a.window = window;
  a.longest = longest;
  return plan_attention(a).floats;
}

void cache_attention(int device, uintptr_t stream, const py::tuple& cache, uintptr_t q, int64_t q_row, int64_t q_head,
                     uintptr_t out, int64_t o_row, int64_t o_head, uintptr_t lse, uintptr_t work, int q_heads,
                     int window, int64_t longest, bool fill_tail, float scale, int dtype) {
  AttentionArgs a{};
  a.c = cache_args(cache);
  a.q = ptr<void>(q);
  a.q_row = q_row;
  a.q_head = q_head;
  a.out = ptr<void>(out);
  a.o_row = o_row;
  a.o_head = o_head;
  a.lse = ptr<float>(lse);
  a.work = ptr<float>(work);
  a.q_heads = q_heads;
  a.window = window;
  a.longest = longest;
  a.fill_tail = fill_tail;
  a.scale = scale;
  a.dtype = dtype;
  OnDevice on(device);
  OnDevice::check(launch_cache_attention(a, stream_of(stream)), "cache_attention");
}

void token_logprobs(int device, uintptr_t stream, uintptr_t logits, int64_t ld, uintptr_t targets, uintptr_t logprob,
                    uintptr_t entropy, uintptr_t rank, uintptr_t top_ids, uintptr_t top_logprobs, uintptr_t work,
                    int64_t rows, int vocab, int top, int dtype) {
  LogprobArgs a{};
  a.logits = ptr<void>(logits);
  a.ld = ld;
  a.targets = ptr<int64_t>(targets);
  a.logprob = ptr<float>(logprob);
  a.entropy = ptr<float>(entropy);
  a.rank = ptr<int64_t>(rank);
  a.top_ids = ptr<int64_t>(top_ids);
  a.top_logprobs = ptr<float>(top_logprobs);
  a.work = ptr<float>(work);
  a.rows = rows;
  a.vocab = vocab;
  a.top = top;
  a.dtype = dtype;
  OnDevice on(device);
  OnDevice::check(launch_token_logprobs(a, stream_of(stream)), "token_logprobs");
}

// What the kernels derive from host copies of lengths, starts and tables, for
// checks on the host: (row, head, slot, split, lo, hi) of every row that a
// workgroup of attention has, and (slot, page, from, to, src) of every append.
std::vector<std::vector<int64_t>> attention_places(const std::vector<int32_t>& starts, const std::vector<int32_t>& lens,
                                                   int rows, int heads, int q_heads, int page, int blocks, int window,
                                                   int64_t max_seq_len, bool fill_tail) {
  AttentionArgs all{};
  all.c.starts = starts.empty() ? nullptr : starts.data();
  all.c.lens = lens.data();
  all.c.batch = (int)lens.size();
  all.c.rows = rows;
  all.c.heads = heads;
  all.c.page = page;
  all.c.blocks = blocks;
  all.c.dim = 128;
  all.q_heads = q_heads;
  all.window = window;
  all.fill_tail = fill_tail;
  all.longest = max_seq_len;
  const int group = q_heads / heads;
  std::vector<std::vector<int64_t>> got;
  const AttentionPlan plan = plan_attention(all);
  for (int pass = 0; pass < plan.passes; ++pass) {
    const AttentionArgs& a = plan.pass[pass];
    for (int64_t slot = 0; slot < slot_count(a); ++slot) {
      Place p;
      if (!place_of_slot(a, group, (int)slot, p)) continue;
      for (int split = 0; split < p.splits; ++split) {
        const int begin = (p.lo & ~(kTile - 1)) + split * a.chunk;
        const int end = split == p.splits - 1 || begin + a.chunk > p.hi ? p.hi : begin + a.chunk;
        for (int i = 0; i < p.rows; ++i)
          got.push_back({p.row0 + (p.local + i) / group, (p.local + i) % group, slot, split, begin, end});
      }
    }
  }
  return got;
}

std::vector<std::vector<int64_t>> append_places(const std::vector<int32_t>& starts, const std::vector<int32_t>& lens,
                                                const std::vector<int32_t>& table, int rows, int page, int blocks,
                                                int pages) {
  CacheArgs c{};
  c.starts = starts.empty() ? nullptr : starts.data();
  c.lens = lens.data();
  c.table = table.data();
  c.ldt = blocks;
  c.batch = (int)lens.size();
  c.rows = rows;
  c.page = page;
  c.blocks = blocks;
  c.pages = pages;
  if ((int64_t)table.size() != (int64_t)c.batch * blocks) throw std::invalid_argument("table");
  std::vector<std::vector<int64_t>> got;
  for (int64_t slot = 0; slot < append_slots(c); ++slot) {
    PageWrite w;
    if (page_of_slot(c, (int)slot, w)) got.push_back({slot, w.pid, w.from, w.to, w.src});
  }
  return got;
}

py::dict step(int device, int iters, uint32_t seed, double oracle_offset) {
  if (iters <= 0 || iters > 100000) throw std::invalid_argument("iters");
  StepResult r;
  {
    py::gil_scoped_release release;
    r = run_step(device, iters, seed, oracle_offset);
  }
  py::dict d;
  d["ms_per_step"] = r.ms;
  d["gbps"] = r.gbps;
  d["product_gbps"] = r.product_gbps;
  d["attention_gbps"] = r.attention_gbps;
  d["logprob_gbps"] = r.logprob_gbps;
  d["checked"] = r.checked;
  d["verified"] = r.failures == 0;
  d["verify_failures"] = r.failures;
  d["messages"] = r.messages;
  return d;
}

}  // namespace

PYBIND11_MODULE(_serving, m) {
  m.doc() = "gpud_amd CDNA4 serving-step operators (4-bit products, 8-bit cache, token log probabilities)";
  m.def("w4_workspace", &w4_work);
  m.def("w4_matmul", &w4_matmul);
  m.def("cache_append", &cache_append);
  m.def("attention_workspace", &attention_floats);
  m.def("cache_attention", &cache_attention);
  m.def("logprob_workspace", &logprob_workspace);
  m.def("serving_step", &step, py::arg("device") = 0, py::arg("iters") = 20, py::arg("seed") = 1,
        py::arg("oracle_offset") = 0.0,
        "One token step of a synthetic served model, checked against host oracles; returns rates + verification");
  m.def("attention_places", &attention_places);
  m.def("append_places", &append_places);
  m.def("token_logprobs", &token_logprobs);
  m.attr("MAX_COLUMNS") = kMaxColumns;
  m.attr("MAX_TOP") = kMaxTop;
  m.attr("MAX_VOCAB") = kMaxVocab;
}
