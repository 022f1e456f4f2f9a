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

// The launches are called once an operator and step of a program, so they take
// their whole numbers straight from the interpreter.
class Numbers {
 public:
  Numbers(PyObject* const* args, Py_ssize_t count, Py_ssize_t wanted) : args_(args) {
    if (count != wanted) throw std::invalid_argument("wrong number of arguments");
  }
  int64_t whole() {
    PyObject* o = args_[at_++];
    const int64_t v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw py::error_already_set();
    return v;
  }
  int small() { return (int)whole(); }
  // of a tensor that may be missing
  template <typename T = void>
  T* pointer() { return ptr<T>((uintptr_t)whole()); }
  // of one that has to be there: a tensor may have a shape and no memory
  template <typename T = void>
  T* memory() {
    T* p = pointer<T>();
    if (!p) throw std::domain_error("a tensor has no memory");
    return p;
  }
  double real() {
    const double v = PyFloat_AsDouble(args_[at_++]);
    if (v == -1 && PyErr_Occurred()) throw py::error_already_set();
    return v;
  }

 private:
  PyObject* const* args_;
  Py_ssize_t at_ = 0;
};

template <typename F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (py::error_already_set& e) {
    e.restore();
  } catch (const std::invalid_argument& e) {
    PyErr_SetString(PyExc_TypeError, e.what());
  } catch (const std::domain_error& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}
PyObject* none() { Py_RETURN_NONE; }

W4Args w4_args(Numbers& n) {
  W4Args a{};
  a.x = n.memory();
  a.ldx = n.whole();
  a.m = n.small();
  a.n = n.small();
  a.k = n.small();
  a.group = n.small();
  a.dtype = n.small();
  return a;
}

PyObject* w4_work(PyObject*, PyObject* const* args, Py_ssize_t count) {
  return guarded([&] {
    Numbers n(args, count, 7);
    return PyLong_FromLongLong(w4_workspace(w4_args(n)));
  });
}

PyObject* w4_matmul(PyObject*, PyObject* const* args, Py_ssize_t count) {
  return guarded([&] {
    Numbers n(args, count, 15);
    W4Args a = w4_args(n);
    a.codes = n.memory<uint8_t>();
    a.scales = n.memory();
    a.zeros = n.pointer<uint8_t>();
    a.y = n.memory();
    a.ldy = n.whole();
    a.work = w4_workspace(a) ? n.memory() : n.pointer();
    OnDevice on(n.small());
    OnDevice::check(launch_w4_matmul(a, stream_of(n.whole())), "w4_matmul");
    return none();
  });
}

CacheArgs cache_args(Numbers& n) {
  CacheArgs c{};
  c.k = n.memory<uint8_t>();
  c.v = n.memory<uint8_t>();
  c.k_scale = n.memory<float>();
  c.v_scale = n.memory<float>();
  c.table = n.pointer<int32_t>();
  c.lens = n.memory<int32_t>();
  c.starts = n.pointer<int32_t>();
  c.ldt = n.whole();
  c.pages = n.small();
  c.heads = n.small();
  c.page = n.small();
  c.dim = n.small();
  c.batch = n.small();
  c.blocks = n.small();
  c.rows = n.small();
  if (c.blocks && !c.table) throw std::domain_error("block_table has no memory");
  return c;
}

PyObject* cache_append(PyObject*, PyObject* const* args, Py_ssize_t count) {
  return guarded([&] {
    Numbers n(args, count, 24);
    AppendArgs a{};
    a.c = cache_args(n);
    a.k_new = n.memory();
    a.k_row = n.whole();
    a.k_head = n.whole();
    a.v_new = n.memory();
    a.v_row = n.whole();
    a.v_head = n.whole();
    a.dtype = n.small();
    OnDevice on(n.small());
    OnDevice::check(launch_cache_append(a, stream_of(n.whole())), "cache_append");
    return none();
  });
}

PyObject* attention_floats(PyObject*, PyObject* const* args, Py_ssize_t count) {
  return guarded([&] {
    Numbers n(args, count, 8);
    AttentionArgs a{};
    static const int32_t some = 0;
    a.c.rows = n.small();
    a.c.batch = n.small();
    a.c.heads = n.small();
    a.q_heads = n.small();
    a.c.dim = n.small();
    a.c.starts = n.whole() ? &some : nullptr;  // only whether it is there counts
    a.window = n.small();
    a.longest = n.whole();
    return PyLong_FromLongLong(plan_attention(a).floats);
  });
}

PyObject* cache_attention(PyObject*, PyObject* const* args, Py_ssize_t count) {
  return guarded([&] {
    Numbers n(args, count, 31);
    AttentionArgs a{};
    a.c = cache_args(n);
    a.q = n.memory();
    a.q_row = n.whole();
    a.q_head = n.whole();
    a.out = n.memory();
    a.o_row = n.whole();
    a.o_head = n.whole();
    a.lse = n.memory<float>();
    a.work = n.pointer<float>();
    a.q_heads = n.small();
    a.window = n.small();
    a.longest = n.whole();
    a.tail = n.small() ? kFillTail : kTailLse;
    a.scale = (float)n.real();
    a.dtype = n.small();
    if (!a.work && plan_attention(a).floats) throw std::domain_error("the workspace has no memory");
    OnDevice on(n.small());
    OnDevice::check(launch_cache_attention(a, stream_of(n.whole())), "cache_attention");
    return none();
  });
}

PyObject* logprob_floats(PyObject*, PyObject* const* args, Py_ssize_t count) {
  return guarded([&] {
    Numbers n(args, count, 3);
    const int64_t rows = n.whole();
    const int vocab = n.small();
    return PyLong_FromLongLong(logprob_workspace(rows, vocab, n.small()));
  });
}

PyObject* token_logprobs(PyObject*, PyObject* const* args, Py_ssize_t count) {
  return guarded([&] {
    Numbers n(args, count, 15);
    LogprobArgs a{};
    a.logits = n.memory();
    a.ld = n.whole();
    a.targets = n.memory<int64_t>();
    a.logprob = n.memory<float>();
    a.entropy = n.memory<float>();
    a.rank = n.memory<int64_t>();
    a.top_ids = n.pointer<int64_t>();
    a.top_logprobs = n.pointer<float>();
    a.work = n.pointer<float>();
    a.rows = n.whole();
    a.vocab = n.small();
    a.top = n.small();
    a.dtype = n.small();
    if ((a.top && !(a.top_ids && a.top_logprobs)) || (!a.work && logprob_workspace(a.rows, a.vocab, a.dtype)))
      throw std::domain_error("a tensor has no memory");
    OnDevice on(n.small());
    OnDevice::check(launch_token_logprobs(a, stream_of(n.whole())), "token_logprobs");
    return none();
  });
}

#define FAST(name, f) {name, (PyCFunction)(void (*)(void))f, METH_FASTCALL, nullptr}
PyMethodDef launches[] = {
    FAST("w4_workspace", w4_work),
    FAST("w4_matmul", w4_matmul),
    FAST("cache_append", cache_append),
    FAST("attention_workspace", attention_floats),
    FAST("cache_attention", cache_attention),
    FAST("logprob_workspace", logprob_floats),
    FAST("token_logprobs", token_logprobs),
    {nullptr, nullptr, 0, nullptr},
};
#undef FAST

// What the kernels derive from host copies of lengths, starts and tables, for
// checks on the host: (row, head, slot, split, lo, hi) of every row that a
// workgroup of attention has, and (slot, page, from, to, src) of every append.
std::vector<std::vector<int64_t>> attention_places(const std::vector<int32_t>& starts, const std::vector<int32_t>& lens,
                                                   int rows, int heads, int q_heads, int page, int blocks, int window,
                                                   int64_t max_seq_len, bool fill_tail, int dim) {
  AttentionArgs all{};
  all.c.starts = starts.empty() ? nullptr : starts.data();
  all.c.lens = lens.data();
  all.c.batch = (int)lens.size();
  all.c.rows = rows;
  all.c.heads = heads;
  all.c.page = page;
  all.c.blocks = blocks;
  all.c.dim = dim;
  all.q_heads = q_heads;
  all.window = window;
  all.tail = fill_tail ? kFillTail : kLeaveTail;
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
  if (PyModule_AddFunctions(m.ptr(), launches) != 0) throw py::error_already_set();
  m.def("serving_step", &step, py::arg("device") = 0, py::arg("iters") = 20, py::arg("seed") = 1,
        py::arg("oracle_offset") = 0.0,
        "One token step of a synthetic served model, checked against host oracles; returns rates + verification");
  m.def("attention_places", &attention_places, py::arg("starts"), py::arg("lens"), py::arg("rows"), py::arg("heads"),
        py::arg("q_heads"), py::arg("page"), py::arg("blocks"), py::arg("window"), py::arg("max_seq_len"),
        py::arg("fill_tail"), py::arg("dim") = 128);
  m.def("append_places", &append_places);
  m.attr("MAX_COLUMNS") = kMaxColumns;
  m.attr("MAX_TOKENS") = kMaxTokens;
  m.attr("MAX_TOP") = kMaxTop;
  m.attr("MAX_VOCAB") = kMaxVocab;
}
