// The hot path from Python to the C entry points of the serving operators.
//
// Arguments are checked in Python (the operators' modules), once for each signature: shapes,
// strides, types, devices and options.  What they decide, the filled-in parameter struct, is
// then kept here under that signature, and a call whose signature is known allocates its
// outputs, puts in the addresses and calls the library: 5 us for a rotation or an append, 11 for
// upkeep, 13 for attention, instead of 17 to 70 (attention 39).  Any other call (a new signature,
// another current device, an address that is not aligned) is answered with None and takes the
// Python path.  Nothing is kept by address.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>
#include <string>
#include <unordered_map>
#include <vector>

#include "dsa_b200.h"

namespace {

enum Op { kAttn, kRotary, kAppend, kUpkeep, kOps };

typedef int (*Entry)(const void*, void*);
Entry g_entry[kOps];
PyObject* g_check;                        // raises for a code that is not DSA_OK
std::unordered_map<int, int*> g_report;   // report flag of each device

struct Plan {
  std::string params, extra;   // the struct; upkeep: the array of caches, attention: which of
                               // query and query_rope are copied first
  int64_t ws_bytes;
};
std::unordered_map<std::string, Plan> g_plans[kOps];
constexpr size_t kMostPlans = 1024;

// A signature, appended to piece by piece.  What an argument may be (None, a number, a tensor, a
// text, a list) is written before it, so that no two kinds give the same bytes.
struct Key {
  std::string s;
  void raw(const void* p, size_t n) { s.append(static_cast<const char*>(p), n); }
  void num(int64_t v) { raw(&v, sizeof v); }
  void real(double v) { raw(&v, sizeof v); }
  void none() { s.push_back('n'); }
  void number(int64_t v) {
    s.push_back('i');
    num(v);
  }
  void text(const char* p, int64_t n) {
    s.push_back('s');
    num(n);
    raw(p, n);
  }
  void list(int64_t n) {
    s.push_back('l');
    num(n);
  }
  void tensor(const at::Tensor& t) {
    const auto sizes = t.sizes(), strides = t.strides();
    s.push_back('t');
    num(((int64_t)t.scalar_type() << 40) | ((int64_t)(t.get_device() + 1) << 8) | (int64_t)sizes.size());
    raw(sizes.data(), sizes.size() * 8);
    raw(strides.data(), strides.size() * 8);
  }
};

const at::Tensor* tensor_of(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

// A tensor or None; false for anything else.
bool maybe_tensor(PyObject* o, Key& key, const at::Tensor** out) {
  *out = nullptr;
  if (o == Py_None) {
    key.none();
    return true;
  }
  *out = tensor_of(o);
  if (!*out || !(*out)->defined() || (*out)->layout() != at::kStrided) return false;
  key.tensor(**out);
  return true;
}

bool tensors_of(PyObject* list, Key& key, std::vector<const at::Tensor*>& out) {
  if (!PyList_Check(list) && !PyTuple_Check(list)) return false;
  PyObject** items = PySequence_Fast_ITEMS(list);
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(list);
  key.list(n);
  out.resize(n);
  for (Py_ssize_t i = 0; i < n; ++i)
    if (!maybe_tensor(items[i], key, &out[i]) || !out[i]) return false;
  return true;
}

bool number(PyObject* o, Key& key) {
  if (o == Py_None) {
    key.none();
    return true;
  }
  if (!PyLong_Check(o)) return false;
  int over = 0;
  key.number(PyLong_AsLongLongAndOverflow(o, &over));
  return !over;
}

uint64_t at_of(const at::Tensor* t) { return reinterpret_cast<uint64_t>(t->data_ptr()); }
template <typename T>
T* ptr(const at::Tensor* t) { return t ? static_cast<T*>(t->data_ptr()) : nullptr; }

// What the signatures of the four operators are made of; false when the Python path has to look.
struct AttnArgs {
  Key key;
  const at::Tensor *q, *qr, *k, *kr, *table, *act_k, *act_q;
  bool stats;
  bool read(PyObject* const* a) {
    if (!maybe_tensor(a[0], key, &q) || !maybe_tensor(a[1], key, &qr) || !maybe_tensor(a[2], key, &k) ||
        !maybe_tensor(a[3], key, &kr) || !maybe_tensor(a[4], key, &table) ||
        !maybe_tensor(a[5], key, &act_k) || !maybe_tensor(a[6], key, &act_q) || !PyFloat_Check(a[7]) ||
        !number(a[8], key) || !q || !qr || !k || !kr || !table || !act_k)
      return false;
    key.real(PyFloat_AS_DOUBLE(a[7]));
    stats = a[9] == Py_True;
    return true;
  }
};
struct RotaryArgs {
  Key key;
  const at::Tensor *x, *table, *positions;
  bool read(PyObject* const* a) {
    if (!maybe_tensor(a[0], key, &x) || !maybe_tensor(a[1], key, &table) || !maybe_tensor(a[2], key, &positions) ||
        !x || !table || !positions || !PyUnicode_Check(a[3]) || !number(a[4], key))
      return false;
    Py_ssize_t n;
    const char* layout = PyUnicode_AsUTF8AndSize(a[3], &n);
    if (!layout) {
      PyErr_Clear();
      return false;
    }
    key.text(layout, n);
    key.number((a[5] == Py_True ? 1 : 0) + (a[6] == a[0] ? 2 : 0));
    return (a[5] == Py_True || a[5] == Py_False) && (a[6] == Py_None || a[6] == a[0]);
  }
};
struct AppendArgs {
  Key key;
  std::vector<const at::Tensor*> tokens, caches;
  const at::Tensor *block_table, *starts, *counts, *table;
  bool read(PyObject* const* a) {
    if (!tensors_of(a[0], key, tokens) || !tensors_of(a[1], key, caches) ||
        !maybe_tensor(a[2], key, &block_table) || !maybe_tensor(a[3], key, &starts) ||
        !maybe_tensor(a[4], key, &counts) || !maybe_tensor(a[5], key, &table) || !block_table || !starts ||
        tokens.size() != caches.size() || tokens.size() > DSA_APPEND_MAX_ENTRIES || tokens.empty())
      return false;
    if (a[6] == Py_None) {
      key.none();
      return true;
    }
    if (!PyList_Check(a[6]) && !PyTuple_Check(a[6])) return false;
    PyObject** items = PySequence_Fast_ITEMS(a[6]);
    key.list(PySequence_Fast_GET_SIZE(a[6]));
    for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(a[6]); ++i) {
      if (items[i] == Py_None) {
        key.none();
        continue;
      }
      if (!PyTuple_Check(items[i]) || PyTuple_GET_SIZE(items[i]) != 2) return false;
      PyObject* layout = PyTuple_GET_ITEM(items[i], 0);
      Py_ssize_t n;
      const char* s = PyUnicode_Check(layout) ? PyUnicode_AsUTF8AndSize(layout, &n) : nullptr;
      if (!s) {
        PyErr_Clear();
        return false;
      }
      key.text(s, n);
      if (!number(PyTuple_GET_ITEM(items[i], 1), key)) return false;
    }
    return true;
  }
};
struct UpkeepArgs {
  Key key;
  std::vector<const at::Tensor*> caches;
  const at::Tensor *state[3], *first, *second;
  bool read(PyObject* const* a) {
    if (!number(a[0], key) || !tensors_of(a[1], key, caches)) return false;
    for (int i = 0; i < 3; ++i)
      if (!maybe_tensor(a[2 + i], key, &state[i])) return false;
    return maybe_tensor(a[5], key, &first) && maybe_tensor(a[6], key, &second) && number(a[7], key);
  }
};

// The plan of a signature, if the lead tensor's device is the current one; and its report flag.
const Plan* find(Op op, const Key& key, const at::Tensor& lead, int** report) {
  const auto it = g_plans[op].find(key.s);
  if (it == g_plans[op].end()) return nullptr;
  const int index = (int)lead.get_device();
  if (index < 0 || c10::cuda::current_device() != index) return nullptr;
  const auto flag = g_report.find(index);
  if (flag == g_report.end()) return nullptr;
  *report = flag->second;
  return &it->second;
}

// Calls the entry; false with a Python error set if it fails.
bool call(Op op, const void* params, const at::Tensor& lead, const char* what) {
  const int rc = g_entry[op](params, c10::cuda::getCurrentCUDAStream(lead.get_device()).stream());
  if (rc == DSA_OK) return true;
  PyObject* r = PyObject_CallFunction(g_check, "is", rc, what);
  if (r) {   // (check raises)
    Py_DECREF(r);
    PyErr_SetString(PyExc_RuntimeError, what);
  }
  return false;
}

// f(), its C++ exceptions turned into the Python ones that torch's own functions raise (its
// OutOfMemoryError, which callers look for, among them).
template <typename F>
PyObject* guarded(F f) {
  HANDLE_TH_ERRORS
  return f();
  END_HANDLE_TH_ERRORS
}

PyObject* attn(PyObject*, PyObject* const* argv, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    AttnArgs a;
    int* report;
    if (n != 10 || !a.read(argv)) Py_RETURN_NONE;
    const Plan* plan = find(kAttn, a.key, *a.q, &report);
    if (!plan) Py_RETURN_NONE;
    const bool copy_q = plan->extra[0], copy_qr = plan->extra[1];
    if (((copy_q ? 0 : at_of(a.q)) | (copy_qr ? 0 : at_of(a.qr)) | at_of(a.k) | at_of(a.kr)) % 16) Py_RETURN_NONE;
    const at::Tensor q = copy_q ? a.q->clone(at::MemoryFormat::Contiguous) : *a.q;
    const at::Tensor qr = copy_qr ? a.qr->clone(at::MemoryFormat::Contiguous) : *a.qr;
    DsaAttnPagedParams p;
    std::memcpy(&p, plan->params.data(), sizeof p);
    const auto f32 = a.q->options().dtype(at::kFloat);
    at::Tensor out = at::empty(a.q->sizes(), a.q->options());
    const int64_t shape[4] = {p.batch, 1, p.s1, p.n1};
    at::Tensor top = a.stats ? at::empty(shape, f32) : at::zeros(shape, f32);
    at::Tensor sum = a.stats ? at::empty(shape, f32) : at::zeros(shape, f32);
    at::Tensor ws = at::empty({plan->ws_bytes}, a.q->options().dtype(at::kByte));
    p.query = q.data_ptr();
    p.query_rope = qr.data_ptr();
    p.key_cache = a.k->data_ptr();
    p.key_rope_cache = a.kr->data_ptr();
    p.block_table = ptr<const int32_t>(a.table);
    p.act_k = ptr<const int32_t>(a.act_k);
    p.act_q = ptr<const int32_t>(a.act_q);
    p.out = out.data_ptr();
    if (a.stats) {
      p.softmax_max = ptr<float>(&top);
      p.softmax_sum = ptr<float>(&sum);
    }
    p.error_flag = report;
    p.workspace = ws.data_ptr();
    if (!call(kAttn, &p, *a.q, "dsa_attn_paged")) return nullptr;
    PyObject* r = PyTuple_New(3);
    if (!r) return nullptr;
    PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(out));
    PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(top));
    PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(sum));
    return r;
  });
}

PyObject* rotary(PyObject*, PyObject* const* argv, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    RotaryArgs a;
    int* report;
    if (n != 7 || !a.read(argv)) Py_RETURN_NONE;
    const Plan* plan = find(kRotary, a.key, *a.x, &report);
    if (!plan) Py_RETURN_NONE;
    DsaRotaryParams p;
    std::memcpy(&p, plan->params.data(), sizeof p);
    at::Tensor out = argv[6] == Py_None ? at::empty(a.x->sizes(), a.x->options()) : *a.x;   // or in place
    p.x = a.x->data_ptr();
    p.out = out.data_ptr();
    p.positions = ptr<const int32_t>(a.positions);
    p.table = ptr<const float>(a.table);
    p.error_flag = report;
    if (!call(kRotary, &p, *a.x, "dsa_rotary")) return nullptr;
    if (argv[6] == Py_None) return THPVariable_Wrap(out);
    Py_INCREF(argv[6]);
    return argv[6];
  });
}

PyObject* append(PyObject*, PyObject* const* argv, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    AppendArgs a;
    int* report;
    if (n != 7 || !a.read(argv)) Py_RETURN_NONE;
    const Plan* plan = find(kAppend, a.key, *a.caches[0], &report);
    if (!plan) Py_RETURN_NONE;
    DsaCacheAppendParams p;
    std::memcpy(&p, plan->params.data(), sizeof p);
    uint64_t low = p.dim ? at_of(a.table) : 0;
    for (size_t i = 0; i < a.tokens.size(); ++i) {
      low |= at_of(a.tokens[i]) | at_of(a.caches[i]);
      p.rows[i].src = a.tokens[i]->data_ptr();
      p.rows[i].cache = a.caches[i]->data_ptr();
    }
    if (low % 16) Py_RETURN_NONE;
    p.table = p.dim ? ptr<const float>(a.table) : nullptr;
    p.block_table = ptr<const int32_t>(a.block_table);
    p.starts = ptr<const int32_t>(a.starts);
    p.counts = ptr<const int32_t>(a.counts);
    p.error_flag = report;
    if (!call(kAppend, &p, *a.caches[0], "dsa_cache_append")) return nullptr;
    Py_RETURN_TRUE;
  });
}

PyObject* upkeep(PyObject*, PyObject* const* argv, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    UpkeepArgs a;
    int* report;
    if (n != 8 || !a.read(argv) || (!a.state[0] && a.caches.empty())) Py_RETURN_NONE;
    const at::Tensor& lead = a.state[0] ? *a.state[0] : *a.caches[0];
    const Plan* plan = find(kUpkeep, a.key, lead, &report);
    if (!plan) Py_RETURN_NONE;
    DsaPagesParams p;
    std::memcpy(&p, plan->params.data(), sizeof p);
    std::vector<DsaPageCache> caches(a.caches.size());
    std::memcpy(caches.data(), plan->extra.data(), plan->extra.size());
    for (size_t i = 0; i < caches.size(); ++i) {
      caches[i].data = a.caches[i]->data_ptr();
      if (at_of(a.caches[i]) % 16) Py_RETURN_NONE;
    }
    at::Tensor out[3], ws;
    for (int i = 0; i < 3; ++i)
      if (a.state[i] && a.state[0]) out[i] = at::empty(a.state[i]->sizes(), a.state[i]->options());
    if (a.state[0]) ws = at::empty({plan->ws_bytes}, lead.options().dtype(at::kByte));
    p.block_table = ptr<const int32_t>(a.state[0]);
    p.seq_lengths = ptr<const int32_t>(a.state[1]);
    p.ref_counts = ptr<const int32_t>(a.state[2]);
    p.block_table_out = out[0].defined() ? ptr<int32_t>(&out[0]) : nullptr;
    p.seq_lengths_out = out[1].defined() ? ptr<int32_t>(&out[1]) : nullptr;
    p.ref_counts_out = out[2].defined() ? ptr<int32_t>(&out[2]) : nullptr;
    p.first = ptr<const int32_t>(a.first);
    p.second = ptr<const int32_t>(a.second);
    p.caches = caches.data();
    p.error_flag = report;
    p.workspace = ws.defined() ? ws.data_ptr() : nullptr;
    if (!call(kUpkeep, &p, lead, "dsa_pages")) return nullptr;
    PyObject* r = PyTuple_New(3);
    if (!r) return nullptr;
    for (int i = 0; i < 3; ++i) {
      PyObject* o = Py_None;
      if (out[i].defined()) o = THPVariable_Wrap(out[i]);
      else Py_INCREF(o);
      PyTuple_SET_ITEM(r, i, o);
    }
    return r;
  });
}

// keep(op, the operator's arguments..., params bytes, extra bytes, workspace bytes)
PyObject* keep(PyObject*, PyObject* const* argv, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n < 5) Py_RETURN_FALSE;
    const long op = PyLong_AsLong(argv[0]);
    if (PyErr_Occurred()) return nullptr;
    PyObject *params = argv[n - 3], *extra = argv[n - 2];
    if (op < 0 || op >= kOps || !PyBytes_Check(params) || !PyBytes_Check(extra)) Py_RETURN_FALSE;
    static const Py_ssize_t kArgs[kOps] = {10, 7, 7, 8};
    static const size_t kSize[kOps] = {sizeof(DsaAttnPagedParams), sizeof(DsaRotaryParams),
                                       sizeof(DsaCacheAppendParams), sizeof(DsaPagesParams)};
    if (n != kArgs[op] + 4 || (size_t)PyBytes_GET_SIZE(params) != kSize[op]) Py_RETURN_FALSE;
    Key key;
    bool ok = false;
    size_t more = 0;   // extra bytes
    if (op == kAttn) { AttnArgs a; ok = a.read(argv + 1); key = a.key; more = 2; }
    if (op == kRotary) { RotaryArgs a; ok = a.read(argv + 1); key = a.key; }
    if (op == kAppend) { AppendArgs a; ok = a.read(argv + 1); key = a.key; }
    if (op == kUpkeep) { UpkeepArgs a; ok = a.read(argv + 1); key = a.key; more = a.caches.size() * sizeof(DsaPageCache); }
    if (!ok || (size_t)PyBytes_GET_SIZE(extra) != more) Py_RETURN_FALSE;
    Plan plan;
    plan.params.assign(PyBytes_AS_STRING(params), PyBytes_GET_SIZE(params));
    plan.extra.assign(PyBytes_AS_STRING(extra), PyBytes_GET_SIZE(extra));
    plan.ws_bytes = PyLong_AsLongLong(argv[n - 1]);
    if (PyErr_Occurred()) return nullptr;
    if (g_plans[op].size() >= kMostPlans) g_plans[op].clear();
    g_plans[op][key.s] = std::move(plan);
    Py_RETURN_TRUE;
  });
}

// connect(entry addresses of the four operators, check): called once
PyObject* connect(PyObject*, PyObject* args) {
  unsigned long long e[kOps];
  PyObject* check;
  if (!PyArg_ParseTuple(args, "KKKKO", &e[0], &e[1], &e[2], &e[3], &check)) return nullptr;
  for (int i = 0; i < kOps; ++i) g_entry[i] = reinterpret_cast<Entry>(e[i]);
  Py_INCREF(check);
  g_check = check;
  Py_RETURN_NONE;
}

// set_report(device index, address of its report flag)
PyObject* set_report(PyObject*, PyObject* args) {
  int index;
  unsigned long long p;
  if (!PyArg_ParseTuple(args, "iK", &index, &p)) return nullptr;
  g_report[index] = reinterpret_cast<int*>(p);
  Py_RETURN_NONE;
}

PyMethodDef g_methods[] = {
    {"attn", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attn)), METH_FASTCALL, nullptr},
    {"rotary", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rotary)), METH_FASTCALL, nullptr},
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(append)), METH_FASTCALL, nullptr},
    {"upkeep", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(upkeep)), METH_FASTCALL, nullptr},
    {"keep", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(keep)), METH_FASTCALL, nullptr},
    {"connect", connect, METH_VARARGS, nullptr},
    {"set_report", set_report, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, g_methods};

}  // namespace

// What the module was compiled against: another torch may have another ABI, whose symbols resolve all
// the same.  The text is what build.py looks for in the built file.
#define DSA_TORCH_STAMP "dsa binding for torch "
static const char g_stamp[] = DSA_TORCH_STAMP DSA_TORCH_VERSION;

PyMODINIT_FUNC PyInit__binding(void) {
  PyObject* m = PyModule_Create(&g_module);
  if (m && PyModule_AddStringConstant(m, "TORCH_VERSION", g_stamp + sizeof(DSA_TORCH_STAMP) - 1) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
