// Host-side bookkeeping of LUMA.step for large parameter sets (the Python
// extension module luma_amd._luma_host).
//
// A step over the same parameters and gradient layout as the previous step
// re-uses its tensor table and only needs the current gradient and parameter
// pointers (the reference re-reads p.grad every step, optimizer.py:425-455).
// Reading p.grad, data_ptr() and the dtype of every parameter from Python
// costs about 1.2 us per tensor (24 ms for 20,000 tensors).  Here the same
// checks read the tensors' C++ objects directly.  Those objects lie scattered
// in host memory, so the walk is bound by memory latency: it runs in stages
// over arrays (parameter object -> TensorImpl -> autograd meta -> gradient
// TensorImpl -> data pointers) with software prefetch a few tensors ahead,
// and large sets are split over a few threads of a pool that lives as long as
// the process (made on first use, made again in a forked child).  The worker
// threads only read C++ objects while the calling thread holds the GIL, so
// nothing they read can change under them.  The module computes nothing of
// the step itself: the step runs in libluma_hip.so.
#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <pybind11/numpy.h>
#include <pybind11/pybind11.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <unistd.h>

#include <algorithm>
#include <cmath>
#include <condition_variable>
#include <cstdint>
#include <cstring>
#include <functional>
#include <mutex>
#include <optional>
#include <string>
#include <thread>
#include <vector>

#include "../../include/luma.h"

namespace py = pybind11;

namespace {

// Gradient element type codes of the C ABI (LUMA_GRAD_*).
int grad_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return 0;
    case at::kBFloat16: return 1;
    case at::kHalf: return 2;
    default: return -1;
  }
}

constexpr int64_t kAhead = 8;             // prefetch distance, in tensors
constexpr int64_t kPerThread = 2048;      // parameters per thread, at least
constexpr int kMaxThreads = 8;            // the calling thread and up to 7 workers

// Workers that run part t of a job for t = 1 .. parts-1 while the calling
// thread runs part 0.  One job at a time (the callers hold the GIL).
class Pool {
 public:
  // The pool of this process; empty (run() then does every part on the
  // calling thread) when no thread could be started.
  static Pool &get() {
    static Pool *pool = nullptr;
    static pid_t owner = 0;
    if (!pool || owner != getpid()) {
      // a forked child inherits the memory but not the threads: it makes
      // its own pool (the parent's stays unused in the child)
      pool = new Pool(kMaxThreads - 1);
      owner = getpid();
    }
    return *pool;
  }

  void run(int parts, const std::function<void(int)> &fn) {
    const int use = std::min<int>(parts - 1, (int)threads_.size());
    {
      std::lock_guard<std::mutex> lock(mu_);
      fn_ = &fn;
      use_ = use;
      pending_ = use;
      ++gen_;
    }
    if (use > 0) wake_.notify_all();
    for (int t = use + 1; t < parts; ++t) fn(t);   // parts no worker took
    fn(0);
    std::unique_lock<std::mutex> lock(mu_);
    done_.wait(lock, [&] { return pending_ == 0; });
    fn_ = nullptr;
  }

 private:
  explicit Pool(int n) {
    for (int i = 0; i < n; ++i) {
      try {
        threads_.emplace_back([this, i] { loop(i + 1); });
      } catch (...) {
        break;
      }
    }
    for (std::thread &t : threads_) t.detach();
  }

  void loop(int part) {
    uint64_t seen = 0;
    for (;;) {
      const std::function<void(int)> *fn;
      {
        std::unique_lock<std::mutex> lock(mu_);
        wake_.wait(lock, [&] { return gen_ != seen; });
        seen = gen_;
        if (part > use_) continue;
        fn = fn_;
      }
      (*fn)(part);
      std::lock_guard<std::mutex> lock(mu_);
      if (--pending_ == 0) done_.notify_one();
    }
  }

  std::vector<std::thread> threads_;
  std::mutex mu_;
  std::condition_variable wake_, done_;
  const std::function<void(int)> *fn_ = nullptr;
  int use_ = 0, pending_ = 0;
  uint64_t gen_ = 0;
};

inline void prefetch(const void *p) { __builtin_prefetch(p, 0, 3); }

inline void prefetch_impl(const c10::TensorImpl *t) {
  const char *c = reinterpret_cast<const char *>(t);
  for (int off = 0; off < (int)sizeof(c10::TensorImpl); off += 64) prefetch(c + off);
}

// The Python types a planned parameter may have: torch.Tensor and
// torch.nn.Parameter (set at module import).
PyTypeObject *g_tensor_type = nullptr;
PyTypeObject *g_param_type = nullptr;

constexpr int kMaxCands = 8;   // cached pointer sets compared during a refresh

struct Plan {
  PyObject *const *params;   // planned parameter objects
  const uint8_t *has_grad;   // per parameter
  const int64_t *row_param;  // per row: index in params (increasing)
  const int32_t *grad_dtype; // per row
  const int64_t *layout_at;  // per row: offset in layout of [ndim, sizes..., strides...]
  const int64_t *layout;
  char *table;               // tensor table rows
  int64_t row_bytes, grad_off, param_off;
  int64_t device;
  int n_cands;               // cached (grad, param) pointer sets, one pair per row
  const uint64_t *cands[kMaxCands];
};

// Checks parameters [a, b) and the rows [ra, rb) that step them, writing
// the rows' pointers.  0: mismatch, 1: pointers unchanged, 2: some moved.
// *same: bit k cleared when a row's new pointers differ from cands[k]'s.
int check_range(const Plan &P, int64_t a, int64_t b, int64_t ra, int64_t rb,
                uint32_t *same) noexcept {
  try {
    const int64_t n = b - a;
    std::vector<const c10::TensorImpl *> pimpl(n), gimpl(n);
    std::vector<const c10::AutogradMetaInterface *> meta(n);
    for (int64_t i = 0; i < n; ++i) {
      if (i + kAhead < n) prefetch(P.params[a + i + kAhead]);
      PyObject *obj = P.params[a + i];
      if (Py_TYPE(obj) != g_tensor_type && Py_TYPE(obj) != g_param_type) return 0;
      pimpl[i] = THPVariable_Unpack(obj).unsafeGetTensorImpl();
    }
    for (int64_t i = 0; i < n; ++i) {
      if (i + kAhead < n) prefetch_impl(pimpl[i + kAhead]);
      meta[i] = pimpl[i]->autograd_meta();
    }
    for (int64_t i = 0; i < n; ++i) {
      if (i + kAhead < n && meta[i + kAhead]) {
        prefetch(meta[i + kAhead]);
        prefetch(reinterpret_cast<const char *>(meta[i + kAhead]) + 64);
      }
      const c10::TensorImpl *g = nullptr;
      if (meta[i]) {
        const at::Tensor &grad = meta[i]->grad();
        if (grad.defined()) g = grad.unsafeGetTensorImpl();
      }
      if ((g != nullptr) != (P.has_grad[a + i] != 0)) return 0;
      gimpl[i] = g;
    }
    bool changed = false;
    for (int64_t r = ra; r < rb; ++r) {
      if (r + kAhead < rb && gimpl[P.row_param[r + kAhead] - a])
        prefetch_impl(gimpl[P.row_param[r + kAhead] - a]);
      const int64_t j = P.row_param[r] - a;
      const c10::TensorImpl *p = pimpl[j], *g = gimpl[j];
      if (!g) return 0;
      // A tensor subclass (e.g. a DTensor) handles its own dispatch, and one
      // with a custom device or sizes policy answers is_cuda(), device(),
      // dim() and sizes() in Python, which needs the GIL that the calling
      // thread holds while the workers run: so the key set (a plain field)
      // is checked before anything else is asked of either tensor.
      if (g->key_set().has(c10::DispatchKey::Python) || p->key_set().has(c10::DispatchKey::Python) ||
          g->key_set().has(c10::DispatchKey::PythonTLSSnapshot) ||
          p->key_set().has(c10::DispatchKey::PythonTLSSnapshot))
        return 0;
      if (grad_code(g->dtype().toScalarType()) != P.grad_dtype[r]) return 0;
      if (p->dtype().toScalarType() != at::kFloat || !p->is_cuda() || !g->is_cuda() ||
          p->device().index() != P.device || g->device().index() != P.device)
        return 0;
      if (g->layout() != at::kStrided || p->layout() != at::kStrided || g->is_neg() ||
          p->is_neg())
        return 0;
      const int64_t *lay = P.layout + P.layout_at[r];
      const int64_t nd = lay[0];
      if (p->dim() != nd || g->dim() != nd) return 0;
      const c10::IntArrayRef ps = p->sizes(), pst = p->strides(), gs = g->sizes(),
                             gst = g->strides();
      for (int64_t d = 0; d < nd; ++d)
        if (ps[d] != lay[1 + d] || gs[d] != lay[1 + d] || pst[d] != lay[1 + nd + d] ||
            gst[d] != lay[1 + nd + d])
          return 0;
      if (!g->has_storage() || !p->has_storage()) return 0;
      const uint64_t ga = (uint64_t)(uintptr_t)g->data(), pa = (uint64_t)(uintptr_t)p->data();
      char *row = P.table + r * P.row_bytes;
      uint64_t *gp = reinterpret_cast<uint64_t *>(row + P.grad_off);
      uint64_t *pp = reinterpret_cast<uint64_t *>(row + P.param_off);
      changed |= (*gp != ga) | (*pp != pa);
      *gp = ga;
      *pp = pa;
      for (int k = 0; k < P.n_cands; ++k)
        if (((*same >> k) & 1u) && (P.cands[k][2 * r] != ga || P.cands[k][2 * r + 1] != pa))
          *same &= ~(1u << k);
    }
    return changed ? 2 : 1;
  } catch (...) {
    return 0;   // an unusual tensor: the caller rebuilds the table, which reports it
  }
}

}  // namespace

// Re-validates a planned step and writes the current pointers into its
// tensor table.
//   groups     -- the optimizer's param_groups (list of dicts with "params")
//   planned    -- the flat parameter list of the plan (same objects, same order)
//   has_grad   -- uint8 per planned parameter: 1 where it had a gradient
//   row_param  -- int64 per table row: index of the row's parameter in planned
//                 (increasing)
//   layout_at, layout -- per table row, [ndim, sizes..., strides...] of the
//                 planned parameter (its Q_m and gradient have the same)
//   gdtype     -- int32 per table row: the planned gradient dtype code
//   table      -- address of the tensor table (LumaTensor rows), its row
//                 size and the byte offsets of the grad and param fields
//   device     -- the planned CUDA device index
//   cands      -- optional: up to 8 (n_rows, 2) uint64 arrays of gradient and
//                 parameter pointers (pointer sets whose tables the caller
//                 keeps on the device)
// Returns 0 when anything differs from the plan (a parameter added, removed
// or replaced by another object, a gradient that appeared or disappeared, a
// gradient of another dtype, shape, layout or device, a tensor subclass, or
// a parameter whose storage was replaced by one of another dtype or layout);
// the table is then to be rebuilt, whatever this call wrote into it.
// Otherwise 1 when every pointer was already in the table, 2 when some moved,
// plus bit 2 + k when every row's new pointers equal cands[k]'s (compared
// while they are written, so the caller need not scan the table again).
template <typename T>
using carray = py::array_t<T, py::array::c_style | py::array::forcecast>;

int refresh(py::list groups, py::list planned, carray<uint8_t> has_grad,
            carray<int64_t> row_param, carray<int64_t> layout_at, carray<int64_t> layout,
            carray<int32_t> gdtype, uintptr_t table, int64_t row_bytes, int64_t grad_off,
            int64_t param_off, int64_t device, py::object cands) {
  const int64_t n_params = (int64_t)planned.size();
  const int64_t n_rows = row_param.shape(0);
  if (has_grad.ndim() != 1 || row_param.ndim() != 1 || layout_at.ndim() != 1 ||
      layout.ndim() != 1 || gdtype.ndim() != 1 || has_grad.shape(0) != n_params ||
      layout_at.shape(0) != n_rows || gdtype.shape(0) != n_rows)
    return 0;
  const int64_t *rp = row_param.data();
  const int64_t *lat = layout_at.data();
  const int64_t *lay = layout.data();
  const int64_t n_layout = layout.shape(0);
  for (int64_t r = 0; r < n_rows; ++r) {
    if (rp[r] < 0 || rp[r] >= n_params || (r > 0 && rp[r] <= rp[r - 1])) return 0;
    if (lat[r] < 0 || lat[r] >= n_layout || lay[lat[r]] < 0 ||
        lat[r] + 1 + 2 * lay[lat[r]] > n_layout)
      return 0;
  }
  // same parameter objects in the same order
  PyObject *const *pl = n_params ? &PyList_GET_ITEM(planned.ptr(), 0) : nullptr;
  int64_t k = 0;
  for (py::handle g : groups) {
    PyObject *params = PyDict_GetItemString(g.ptr(), "params");
    if (!params || !PyList_Check(params)) return 0;
    const Py_ssize_t n = PyList_GET_SIZE(params);
    if (k + n > n_params) return 0;
    for (Py_ssize_t i = 0; i < n; ++i)
      if (PyList_GET_ITEM(params, i) != pl[k + i]) return 0;
    k += n;
  }
  if (k != n_params || !g_tensor_type || !g_param_type) return 0;

  Plan P{pl, has_grad.data(), rp, gdtype.data(), lat, lay,
         reinterpret_cast<char *>(table), row_bytes, grad_off, param_off, device, 0, {}};
  // the candidate arrays (held here for the call's duration); one of another
  // shape is never a match and never read (its bit starts cleared)
  std::vector<carray<uint64_t>> held;
  uint32_t usable = 0;
  if (!cands.is_none()) {
    const py::list cl = cands.cast<py::list>();
    for (py::handle h : cl) {
      if (P.n_cands == kMaxCands) break;
      held.push_back(h.cast<carray<uint64_t>>());
      const carray<uint64_t> &c = held.back();
      const bool fits = c.ndim() == 2 && c.shape(0) == n_rows && c.shape(1) == 2;
      P.cands[P.n_cands] = fits ? c.data() : nullptr;
      if (fits) usable |= 1u << P.n_cands;
      ++P.n_cands;
    }
  }
  const int T = (int)std::min<int64_t>(kMaxThreads, std::max<int64_t>(1, n_params / kPerThread));
  std::vector<int> res(T, 1);
  std::vector<uint32_t> same(T, usable);
  const std::function<void(int)> part = [&](int t) {
    const int64_t a = n_params * t / T, b = n_params * (t + 1) / T;
    const int64_t ra = std::lower_bound(rp, rp + n_rows, a) - rp;
    const int64_t rb = std::lower_bound(rp, rp + n_rows, b) - rp;
    res[t] = check_range(P, a, b, ra, rb, &same[t]);
  };
  if (T == 1)
    part(0);
  else
    Pool::get().run(T, part);
  int out = 1;
  uint32_t match = usable;
  for (int t = 0; t < T; ++t) {
    if (res[t] == 0) return 0;
    if (res[t] == 2) out = 2;
    match &= same[t];
  }
  return out | (int)(match << 2);
}

// Whether the gradient and parameter pointers of the table's rows are those
// of cols (one (grad, param) pair per row; the table has at least as many
// rows).  Stops at the first difference: a table that matches no cached
// pointer set costs one row per cached set.
bool same_pointers(uintptr_t table, int64_t row_bytes, int64_t grad_off, int64_t param_off,
                   carray<uint64_t> cols) {
  if (cols.ndim() != 2 || cols.shape(1) != 2)
    throw py::value_error("same_pointers: cols must be an (n, 2) array");
  const int64_t n = cols.shape(0);
  const uint64_t *c = cols.data();
  const char *t = reinterpret_cast<const char *>(table);
  for (int64_t r = 0; r < n; ++r) {
    const char *row = t + r * row_bytes;
    uint64_t g, p;
    std::memcpy(&g, row + grad_off, sizeof g);
    std::memcpy(&p, row + param_off, sizeof p);
    if (g != c[2 * r] || p != c[2 * r + 1]) return false;
  }
  return true;
}

// state["step"] += 1 for every state dict of the list.  The dicts of one
// plan usually hold the same count object, so the sum is formed once per
// distinct object.  The dicts lie scattered in memory: each one, and then its
// key table, is prefetched a few dicts ahead.
void bump_steps(py::list states) {
  static PyObject *key = PyUnicode_InternFromString("step");
  py::object last_v, last_nv;
  py::object one = py::int_(1);
  for (Py_ssize_t i = 0; i < PyList_GET_SIZE(states.ptr()); ++i) {
    // (the size is read again each time: a count object's __add__ could
    // change the list)
    const Py_ssize_t n = PyList_GET_SIZE(states.ptr());
    if (i + 2 * kAhead < n) prefetch(PyList_GET_ITEM(states.ptr(), i + 2 * kAhead));
    if (i + kAhead < n) {
      PyObject *a = PyList_GET_ITEM(states.ptr(), i + kAhead);
      if (PyDict_CheckExact(a)) {
        const char *keys = reinterpret_cast<const char *>(((PyDictObject *)a)->ma_keys);
        prefetch(keys);
        prefetch(keys + 64);
      }
    }
    PyObject *d = PyList_GET_ITEM(states.ptr(), i);
    if (!PyDict_Check(d)) throw py::type_error("bump_steps: a state is not a dict");
    PyObject *v = PyDict_GetItemWithError(d, key);
    if (!v) {
      if (PyErr_Occurred()) throw py::error_already_set();
      throw py::key_error("step");
    }
    if (v != last_v.ptr()) {
      PyObject *nv = PyNumber_Add(v, one.ptr());
      if (!nv) throw py::error_already_set();
      last_v = py::reinterpret_borrow<py::object>(v);
      last_nv = py::reinterpret_steal<py::object>(nv);
    }
    if (PyDict_SetItem(d, key, last_nv.ptr()) != 0) throw py::error_already_set();
  }
}

// The gradients of a list of tensors, or the tensors themselves, as rows of the
// C ABI's LumaGrad table (the walk of check_range: in stages, with prefetch).
struct GradRow {
  uint64_t data;
  int64_t numel;
  int32_t dtype, first_tile;
};
static_assert(sizeof(GradRow) == sizeof(LumaGrad), "LumaGrad");
constexpr int64_t kGradTile = LUMA_GRAD_TILE;

// One part's *count rows, their first_tile within the part; false for a tensor
// that the kernels cannot take as it is.  *device: the CUDA device of all of them
// (-1 for none).  impls: takes the rows' tensors, or null.
bool grad_range(PyObject *const *objs, int64_t n, bool of_grad, GradRow *rows,
                const c10::TensorImpl **impls, int64_t *count, int64_t *device) noexcept {
  int64_t dev = -1, tiles = 0;     // (not *device: its neighbours are other threads')
  GradRow *row = rows;
  try {
    std::vector<const c10::TensorImpl *> impl(n);
    for (int64_t i = 0; i < n; ++i) {
      if (i + kAhead < n) prefetch(objs[i + kAhead]);
      if (Py_TYPE(objs[i]) != g_tensor_type && Py_TYPE(objs[i]) != g_param_type) return false;
      impl[i] = THPVariable_Unpack(objs[i]).unsafeGetTensorImpl();
    }
    if (of_grad) {
      std::vector<const c10::AutogradMetaInterface *> meta(n);
      for (int64_t i = 0; i < n; ++i) {
        if (i + kAhead < n) prefetch_impl(impl[i + kAhead]);
        meta[i] = impl[i]->autograd_meta();
      }
      for (int64_t i = 0; i < n; ++i) {
        if (i + kAhead < n && meta[i + kAhead]) {
          prefetch(meta[i + kAhead]);
          prefetch(reinterpret_cast<const char *>(meta[i + kAhead]) + 64);
        }
        impl[i] = nullptr;
        if (meta[i]) {
          const at::Tensor &grad = meta[i]->grad();
          if (grad.defined()) impl[i] = grad.unsafeGetTensorImpl();
        }
      }
    }
    for (int64_t i = 0; i < n; ++i) {
      if (i + kAhead < n && impl[i + kAhead]) prefetch_impl(impl[i + kAhead]);
      const c10::TensorImpl *g = impl[i];
      if (!g) continue;
      if (g->key_set().has(c10::DispatchKey::Python) ||
          g->key_set().has(c10::DispatchKey::PythonTLSSnapshot) || !g->is_cuda() ||
          g->layout() != at::kStrided || g->is_neg() || !g->has_storage())
        return false;
      const int code = grad_code(g->dtype().toScalarType());
      if (code < 0 || !g->is_non_overlapping_and_dense()) return false;
      if (dev >= 0 && g->device().index() != dev) return false;
      dev = g->device().index();
      if (g->numel() == 0) continue;
      const uint64_t p = (uint64_t)(uintptr_t)g->data();
      if (!p) return false;
      if (tiles > INT32_MAX) return false;
      if (impls) *impls++ = g;
      *row++ = {p, g->numel(), code, (int32_t)tiles};
      tiles += (g->numel() - 1) / kGradTile + 1;
    }
    if (tiles > INT32_MAX) return false;
    *device = dev;
    *count = row - rows;
    return true;
  } catch (...) {
    return false;   // an unusual tensor: the caller looks at it
  }
}

// Records that the kernels will write to these tensors, as torch's in-place
// operations do (what autograd has saved of them is then stale).  By the calling
// thread, an increment for each tensor: 20,000 views of one buffer, which share one
// counter, take 200 us, by eight threads that take its line from each other 390.
void bump_versions(const c10::TensorImpl *const *impls, int64_t n) {
  auto at = [&](int64_t i) { return const_cast<c10::TensorImpl *>(impls[i]); };
  uint32_t seen = 0;
  constexpr int64_t kRun = 64;
  for (int64_t a = 0; a < n; a += kRun) {
    const int64_t b = std::min(n, a + kRun);
    // (an atomic increment waits for all loads before it: a run's lines first)
    for (int64_t i = a; i < b; ++i)
      if (!at(i)->is_inference()) seen += (uint32_t)at(i)->version_counter().current_version();
    for (int64_t i = a; i < b; ++i)
      if (!at(i)->is_inference()) at(i)->bump_version();
  }
  asm volatile("" ::"r"(seen));
}

// Whether no two rows share memory.
bool disjoint(const GradRow *rows, int64_t n) {
  auto end = [](const GradRow &r) { return r.data + (uint64_t)r.numel * (r.dtype == 0 ? 4 : 2); };
  bool up = true, down = true;
  for (int64_t i = 1; i < n && (up || down); ++i) {
    up &= end(rows[i - 1]) <= rows[i].data;
    down &= end(rows[i]) <= rows[i - 1].data;
  }
  if (up || down) return true;
  std::vector<std::pair<uint64_t, uint64_t>> spans(n);
  for (int64_t i = 0; i < n; ++i) spans[i] = {rows[i].data, end(rows[i])};
  std::sort(spans.begin(), spans.end());
  for (int64_t i = 1; i < n; ++i)
    if (spans[i].first < spans[i - 1].second) return false;
  return true;
}

// Writes the rows of the tensors in objs (of_grad: of their gradients, those
// without one left out) to `table`, which has room for one per object.  Returns
// (rows, device index or -1 for no rows), or None when one of them is a
// subclass, sparse, not dense, of another type or device, or (apart) shares
// memory with another: the caller then looks at each.  apart: they will be written to.
py::object grad_rows(py::list objs, bool of_grad, bool apart, uintptr_t table) {
  const int64_t n = (int64_t)objs.size();
  PyObject *const *o = n ? &PyList_GET_ITEM(objs.ptr(), 0) : nullptr;
  GradRow *rows = reinterpret_cast<GradRow *>(table);
  const int T = (int)std::min<int64_t>(kMaxThreads, std::max<int64_t>(1, n / kPerThread));
  int64_t device[kMaxThreads], count[kMaxThreads];
  bool ok[kMaxThreads];
  std::vector<const c10::TensorImpl *> impls(apart ? n : 0);
  const std::function<void(int)> job = [&](int t) {
    const int64_t a = n * t / T, b = n * (t + 1) / T;
    ok[t] = grad_range(o + a, b - a, of_grad, rows + a, apart ? impls.data() + a : nullptr,
                       &count[t], &device[t]);
  };
  if (T == 1)
    job(0);
  else
    Pool::get().run(T, job);
  int64_t dev = -1, at = 0, tiles = 0;
  for (int t = 0; t < T; ++t) {
    if (!ok[t] || (device[t] >= 0 && dev >= 0 && device[t] != dev)) return py::none();
    if (device[t] >= 0) dev = device[t];
    // the part's rows behind those of the parts before it
    const GradRow *from = rows + n * t / T;
    int64_t last = tiles;
    for (int64_t i = 0; i < count[t]; ++i) {
      GradRow r = from[i];
      const int64_t first = tiles + r.first_tile;
      last = first + (r.numel - 1) / kGradTile + 1;
      if (last > INT32_MAX) return py::none();
      r.first_tile = (int32_t)first;
      if (apart) impls[at] = impls[n * t / T + i];
      rows[at++] = r;
    }
    tiles = last;
  }
  if (apart) {
    if (!disjoint(rows, at)) return py::none();
    bump_versions(impls.data(), at);
  }
  return py::make_tuple(at, dev);
}

// -- calls of the library -------------------------------------------------------
// The eager paths of the operators beside the step: their allocations, the
// library's calls and linear_cross_entropy's autograd node (from Python they take
// 120 us of a call of the latter whose kernels take 45, and 20 of a clipping of
// 50 tensors whose kernels take 10).  The entry points come from the caller
// (bind), which checked the library's ABI.
struct Library {
  int64_t (*workspace)(const LumaXentArgs *, int32_t) = nullptr;
  int (*forward)(const LumaXentArgs *, void *) = nullptr;
  int (*backward)(const LumaXentArgs *, void *) = nullptr;
  int (*norm)(const LumaNormArgs *, void *) = nullptr;
  int (*clip)(const LumaNormArgs *, void *) = nullptr;
  const char *(*error)() = nullptr;
  PyObject *stream = nullptr;    // torch's current stream of a device, as an address
} g_lib;

void bind(uintptr_t workspace, uintptr_t forward, uintptr_t backward, uintptr_t norm,
          uintptr_t clip, uintptr_t error, py::object stream) {
  g_lib = {reinterpret_cast<int64_t (*)(const LumaXentArgs *, int32_t)>(workspace),
           reinterpret_cast<int (*)(const LumaXentArgs *, void *)>(forward),
           reinterpret_cast<int (*)(const LumaXentArgs *, void *)>(backward),
           reinterpret_cast<int (*)(const LumaNormArgs *, void *)>(norm),
           reinterpret_cast<int (*)(const LumaNormArgs *, void *)>(clip),
           reinterpret_cast<const char *(*)()>(error), stream.release().ptr()};
}

void *current_stream(int64_t device) {
  py::gil_scoped_acquire gil;    // (the backward runs on autograd's thread)
  return reinterpret_cast<void *>(py::handle(g_lib.stream)(device).cast<uintptr_t>());
}

// The norm of the tensors in objs or (clip) of their gradients, which are then
// clipped by max_norm: the norm as a float32 scalar, or None for what grad_rows
// cannot take, no rows and lists that need a device table (more than `most`).
py::object grad_norm(py::list objs, bool clip, int32_t norm, double max_norm, int64_t most) {
  const int64_t n = (int64_t)objs.size();
  if (n > most || n == 0 || !g_lib.norm) return py::none();
  std::vector<GradRow> rows(n);
  std::vector<const c10::TensorImpl *> impls(clip ? n : 0);
  int64_t count = 0, device = -1;
  if (!grad_range(&PyList_GET_ITEM(objs.ptr(), 0), n, clip, rows.data(),
                  clip ? impls.data() : nullptr, &count, &device) ||
      count == 0 || (clip && !disjoint(rows.data(), count)))
    return py::none();
  if (clip) bump_versions(impls.data(), count);
  const c10::Device dev(c10::kCUDA, (c10::DeviceIndex)device);
  const c10::DeviceGuard guard(dev);
  const at::Tensor partials =
      at::empty({LUMA_NORM_PARTIALS}, at::TensorOptions().dtype(at::kDouble).device(dev));
  at::Tensor total = at::empty({}, at::TensorOptions().dtype(at::kFloat).device(dev));
  LumaNormArgs a{};
  a.grads = reinterpret_cast<const LumaGrad *>(rows.data());
  a.n = (int32_t)count;
  a.norm = norm;
  a.max_norm = max_norm;
  a.partials = partials.mutable_data_ptr<double>();
  a.total = total.mutable_data_ptr<float>();
  const int rc = (clip ? g_lib.clip : g_lib.norm)(&a, current_stream(device));
  TORCH_CHECK(rc == 0, g_lib.error());
  return py::cast(total);
}

// t, or a copy, with elements of a row next to each other and rows apart.
at::Tensor rows_of(const at::Tensor &t) {
  const bool plain = !t.is_neg() && !t._is_zerotensor() && (t.size(1) <= 1 || t.stride(1) == 1) &&
                     (t.size(0) <= 1 || (t.stride(0) >= t.size(1) && t.stride(0) <= 1 << 21));
  return plain ? t : t.contiguous();
}

LumaXentArgs xent_args(const at::Tensor &hidden, const at::Tensor &weight,
                       const at::Tensor &target, const at::Tensor &stats, int64_t ignore,
                       int64_t reduction) {
  LumaXentArgs a{};
  a.hidden = hidden.const_data_ptr();
  a.weight = weight.const_data_ptr();
  a.target = target.const_data_ptr<int64_t>();
  a.n = hidden.size(0);
  a.h = hidden.size(1);
  a.v = weight.size(0);
  a.ld_hidden = a.n > 1 ? hidden.stride(0) : a.h;
  a.ld_weight = a.v > 1 ? weight.stride(0) : a.h;
  a.ignore_index = ignore;
  a.dtype = grad_code(hidden.scalar_type());
  a.reduction = (int32_t)reduction;
  a.stats = stats.mutable_data_ptr<float>();
  return a;
}

void xent_call(LumaXentArgs &a, bool backward, const at::Tensor &like) {
  const c10::DeviceGuard guard(like.device());
  const int64_t bytes = g_lib.workspace(&a, backward);
  TORCH_CHECK(bytes >= 0, g_lib.error());
  const at::Tensor workspace =
      at::empty({std::max<int64_t>(bytes, 1)}, like.options().dtype(at::kByte));
  a.workspace = workspace.mutable_data_ptr();
  a.workspace_bytes = bytes;
  const int rc = (backward ? g_lib.backward : g_lib.forward)(
      &a, current_stream(like.device().index()));
  TORCH_CHECK(rc == 0, g_lib.error());
}

// A gradient under create_graph=True: depends on the operands, and says so when it
// is differentiated.
struct XentOnce : torch::autograd::Function<XentOnce> {
  static at::Tensor forward(torch::autograd::AutogradContext *, const at::Tensor &grad,
                            const at::Tensor &, const at::Tensor &, const at::Tensor &) {
    return grad.detach();
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *,
                                                 torch::autograd::variable_list) {
    TORCH_CHECK(false, "linear_cross_entropy: its gradients cannot be differentiated again");
  }
};

// The custom op of the backward, which loss.py registers.
const auto &backward_op() {
  static const auto op =
      c10::Dispatcher::singleton()
          .findSchemaOrThrow("luma_amd::linear_cross_entropy_backward", "")
          .typed<std::tuple<at::Tensor, at::Tensor>(
              const at::Tensor &, const at::Tensor &, const at::Tensor &, const at::Tensor &,
              const at::Tensor &, int64_t, int64_t, bool, bool)>();
  return op;
}

struct Xent : torch::autograd::Function<Xent> {
  static at::Tensor forward(torch::autograd::AutogradContext *ctx, const at::Tensor &hidden,
                            const at::Tensor &weight, const at::Tensor &target, int64_t ignore,
                            int64_t reduction) {
    const int64_t n = hidden.size(0);
    const auto f32 = hidden.options().dtype(at::kFloat);
    at::Tensor loss, stats;
    const std::vector<int64_t> shape =
        reduction == LUMA_XENT_NONE ? std::vector<int64_t>{n} : std::vector<int64_t>{};
    if (n == 0) {
      loss = at::full(shape, reduction == LUMA_XENT_MEAN ? NAN : 0.0, f32);
      stats = at::zeros({1}, f32);
    } else {
      loss = at::empty(shape, f32);
      stats = at::empty({2 * n + 1}, f32);
      const at::Tensor x = rows_of(hidden), w = rows_of(weight), t = target.contiguous();
      LumaXentArgs a = xent_args(x, w, t, stats, ignore, reduction);
      a.loss = loss.mutable_data_ptr<float>();
      xent_call(a, false, hidden);
    }
    ctx->save_for_backward({hidden, weight, target, stats});
    ctx->saved_data["ignore"] = ignore;
    ctx->saved_data["reduction"] = reduction;
    ctx->set_materialize_grads(false);
    return loss;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx,
                                                 torch::autograd::variable_list grads) {
    const bool want_hidden = ctx->needs_input_grad(0), want_weight = ctx->needs_input_grad(1);
    at::Tensor d_hidden, d_weight;
    if (grads[0].defined() && (want_hidden || want_weight)) {
      const auto saved = ctx->get_saved_variables();
      const at::Tensor &hidden = saved[0], &weight = saved[1], &target = saved[2];
      const int64_t ignore = ctx->saved_data["ignore"].toInt();
      const int64_t reduction = ctx->saved_data["reduction"].toInt();
      {
        at::AutoDispatchBelowADInplaceOrView below;
        if (c10::impl::dispatch_mode_enabled() ||
            c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch)) {
          // (a tracer or another mode, begun since the forward, watches the operators
          // called: it is given one, which holds the kernels)
          std::tie(d_hidden, d_weight) =
              backward_op().call(grads[0], hidden, weight, target, saved[3], ignore, reduction,
                                 want_hidden, want_weight);
          if (!want_hidden) d_hidden.reset();
          if (!want_weight) d_weight.reset();
        } else {
          if (want_hidden) d_hidden = at::empty(hidden.sizes(), hidden.options());
          if (want_weight) d_weight = at::empty(weight.sizes(), weight.options());
          if (hidden.size(0) == 0) {
            if (want_weight) d_weight.zero_();
          } else {
            const at::Tensor x = rows_of(hidden), w = rows_of(weight), t = target.contiguous();
            const at::Tensor g = grads[0].to(at::kFloat).contiguous();
            LumaXentArgs a = xent_args(x, w, t, saved[3], ignore, reduction);
            a.grad_loss = g.const_data_ptr<float>();
            a.d_hidden = want_hidden ? d_hidden.mutable_data_ptr() : nullptr;
            a.d_weight = want_weight ? d_weight.mutable_data_ptr() : nullptr;
            xent_call(a, true, hidden);
          }
        }
      }
      if (at::GradMode::is_enabled())
        for (at::Tensor *d : {&d_hidden, &d_weight})
          if (d->defined()) *d = XentOnce::apply(*d, hidden, weight, grads[0]);
    }
    return {d_hidden, d_weight, at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

// linear_cross_entropy of plain tensors; None where its arguments do not fit (the
// caller then says which).
py::object xent(const at::Tensor &hidden, const at::Tensor &weight, const at::Tensor &target,
                int64_t ignore, int64_t reduction) {
  if (!g_lib.forward || !hidden.is_cuda() || weight.device() != hidden.device() ||
      target.device() != hidden.device() || hidden.layout() != at::kStrided ||
      weight.layout() != at::kStrided || target.layout() != at::kStrided)
    return py::none();
  const int64_t d = hidden.dim();
  if (d < 1 || weight.dim() != 2 || weight.size(0) == 0 || weight.size(1) == 0 ||
      hidden.size(d - 1) != weight.size(1) || grad_code(hidden.scalar_type()) < 0 ||
      weight.scalar_type() != hidden.scalar_type() || target.scalar_type() != at::kLong ||
      target.sizes() != hidden.sizes().slice(0, d - 1))
    return py::none();
  if (d == 2) return py::cast(Xent::apply(hidden, weight, target, ignore, reduction));
  const at::Tensor loss = Xent::apply(hidden.reshape({-1, weight.size(1)}), weight,
                                      target.reshape({-1}), ignore, reduction);
  return py::cast(reduction == LUMA_XENT_NONE ? loss.view(target.sizes()) : loss);
}

// -- the residual stream's operators and the policy loss ---------------------------

// The entry points of dropout, the norm and the policy loss, both ways.
struct More {
  int (*dropout)(const LumaDropoutArgs *, void *) = nullptr;
  int64_t (*norm_workspace)(const LumaLayerNormArgs *) = nullptr;
  int (*norm_forward)(const LumaLayerNormArgs *, void *) = nullptr;
  int (*norm_backward)(const LumaLayerNormArgs *, void *) = nullptr;
  int64_t (*policy_workspace)(const LumaPolicyArgs *) = nullptr;
  int (*policy_forward)(const LumaPolicyArgs *, void *) = nullptr;
  int (*policy_backward)(const LumaPolicyArgs *, void *) = nullptr;
} g_more;

void bind_more(const std::vector<uintptr_t> &at) {
  TORCH_CHECK(at.size() == 7, "bind_more: seven entry points");
  g_more = {reinterpret_cast<int (*)(const LumaDropoutArgs *, void *)>(at[0]),
            reinterpret_cast<int64_t (*)(const LumaLayerNormArgs *)>(at[1]),
            reinterpret_cast<int (*)(const LumaLayerNormArgs *, void *)>(at[2]),
            reinterpret_cast<int (*)(const LumaLayerNormArgs *, void *)>(at[3]),
            reinterpret_cast<int64_t (*)(const LumaPolicyArgs *)>(at[4]),
            reinterpret_cast<int (*)(const LumaPolicyArgs *, void *)>(at[5]),
            reinterpret_cast<int (*)(const LumaPolicyArgs *, void *)>(at[6])};
}

typedef std::optional<at::Tensor> MaybeTensor;
typedef torch::autograd::AutogradContext Context;
typedef torch::autograd::variable_list Variables;

const at::ScalarType kTypes[] = {at::kFloat, at::kBFloat16, at::kHalf};   // by LUMA_GRAD_*

bool given(const MaybeTensor &t) { return t.has_value() && t->defined(); }

at::Tensor value(const MaybeTensor &t) { return given(t) ? *t : at::Tensor(); }

MaybeTensor maybe(const at::Tensor &t) { return t.defined() ? MaybeTensor(t) : std::nullopt; }

// A tensor beside `like`, its memory not set.
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor &like) {
  return at::empty(sizes, like.options().dtype(type));
}

// Whether a tracer or another mode watches the operators that are called.
bool watched() {
  return c10::impl::dispatch_mode_enabled() ||
         c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch);
}

// t with memory that holds its values.
at::Tensor resolved(const at::Tensor &t) {
  if (t._is_zerotensor()) return at::zeros(t.sizes(), t.options());
  return t.is_neg() ? t.resolve_neg() : t;
}

at::Tensor dense(const at::Tensor &t) { return resolved(t).contiguous(); }

// t (or a copy) as rows of its last dimension, elements of a row next to each other.
at::Tensor as_rows(const at::Tensor &t) {
  const int64_t h = t.size(t.dim() - 1);
  at::Tensor r = resolved(t);
  if (r.dim() != 2) r = r.reshape({-1, h});
  return h > 1 && r.stride(1) != 1 ? r.contiguous() : r;
}

int64_t ld_of(const at::Tensor &rows) {
  return rows.size(0) > 1 ? rows.stride(0) : rows.size(1);
}

void run(int rc) { TORCH_CHECK(rc == 0, g_lib.error()); }

// A gradient under create_graph=True: depends on what it was formed of, and says so
// when it is differentiated.
struct Once : torch::autograd::Function<Once> {
  static at::Tensor forward(Context *ctx, const at::Tensor &grad, std::string name,
                            const MaybeTensor &, const MaybeTensor &, const MaybeTensor &,
                            const MaybeTensor &) {
    ctx->saved_data["name"] = name;
    return grad.detach();
  }
  static Variables backward(Context *ctx, Variables) {
    TORCH_CHECK(false, ctx->saved_data["name"].toStringRef(),
                ": its gradients cannot be differentiated again");
  }
};

void once(std::initializer_list<at::Tensor *> grads, const char *name, const at::Tensor &a,
          const at::Tensor &b = {}, const at::Tensor &c = {}, const at::Tensor &d = {}) {
  if (!at::GradMode::is_enabled()) return;
  for (at::Tensor *g : grads)
    if (g->defined())
      *g = Once::apply(*g, std::string(name), maybe(a), maybe(b), maybe(c), maybe(d));
}

// What a call of dropout is drawn from.
struct Draws {
  at::Tensor seed_at;
  double p;
  int64_t seed, call;

  LumaDropout args() const {
    LumaDropout d{};
    d.seed_at = seed_at.defined() ? seed_at.const_data_ptr<int64_t>() : nullptr;
    d.seed = (uint64_t)seed;
    d.p = p;
    d.call = (uint32_t)call;
    return d;
  }
};

// (with x's device the current one)
void dropout_call(const at::Tensor &x, const at::Tensor &residual, const at::Tensor &y,
                  const Draws &d) {
  LumaDropoutArgs a{};
  a.x = x.const_data_ptr();
  a.residual = residual.defined() ? residual.const_data_ptr() : nullptr;
  a.y = y.mutable_data_ptr();
  a.numel = x.numel();
  a.in = grad_code(x.scalar_type());
  a.out = grad_code(y.scalar_type());
  a.drop = d.args();
  run(g_more.dropout(&a, current_stream(x.device().index())));
}

// An operator of the package, by its name.
template <typename F>
auto op_of(const char *name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}

at::Tensor dropped(const at::Tensor &x, const MaybeTensor &residual, const Draws &d) {
  const c10::DeviceGuard guard(x.device());
  const at::Tensor &like = given(residual) ? *residual : x;
  at::Tensor y = fresh(x.sizes(), like.scalar_type(), x);
  dropout_call(dense(x), given(residual) ? dense(*residual) : at::Tensor(), y, d);
  return y;
}

// Dropout's gradient for its result's, of type code.
at::Tensor dropped_grad(const at::Tensor &grad, const Draws &d, int64_t code) {
  if (watched()) {
    static const auto op = op_of<at::Tensor(const at::Tensor &, const MaybeTensor &, double, int64_t,
                                            int64_t, int64_t)>("luma_amd::dropout_backward");
    return op.call(grad, maybe(d.seed_at), d.p, d.seed, d.call, code);
  }
  const c10::DeviceGuard guard(grad.device());
  const at::Tensor d_x = fresh(grad.sizes(), kTypes[code], grad);
  dropout_call(dense(grad), at::Tensor(), d_x, d);
  return d_x;
}

struct Dropout : torch::autograd::Function<Dropout> {
  static at::Tensor forward(Context *ctx, const at::Tensor &x, const MaybeTensor &residual,
                            const MaybeTensor &seed_at, double p, int64_t seed, int64_t call) {
    const Draws d{value(seed_at), p, seed, call};
    const at::Tensor y = dropped(x, residual, d);
    ctx->save_for_backward({d.seed_at});
    ctx->saved_data["p"] = p;
    ctx->saved_data["numbers"] =
        std::vector<int64_t>{seed, call, grad_code(x.scalar_type()), given(residual)};
    ctx->set_materialize_grads(false);
    return y;
  }

  static Variables backward(Context *ctx, Variables grads) {
    const auto numbers = ctx->saved_data["numbers"].toIntVector();
    const bool residual = numbers[3];
    at::Tensor d_x, d_residual;
    if (grads[0].defined()) {
      if (residual && ctx->needs_input_grad(1)) d_residual = grads[0];
      if (ctx->needs_input_grad(0)) {
        at::AutoDispatchBelowADInplaceOrView below;
        const Draws d{ctx->get_saved_variables()[0], ctx->saved_data["p"].toDouble(), numbers[0],
                      numbers[1]};
        d_x = dropped_grad(grads[0], d, numbers[2]);
      }
      once({&d_x}, "dropout", grads[0]);
    }
    return {d_x, d_residual, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

// Whether a call of these (some may be null) is one that autograd records, or, of
// tensors with a tangent, refuses.
bool differentiable(std::initializer_list<const at::Tensor *> tensors) {
  const bool grad = at::GradMode::is_enabled();
  for (const at::Tensor *t : tensors)
    if (t && ((grad && t->requires_grad()) || t->_fw_grad(0).defined())) return true;
  return false;
}

const at::Tensor *pointer(const MaybeTensor &t) { return given(t) ? &*t : nullptr; }

bool same_place(const at::Tensor &t, const at::Tensor &like) {
  return t.layout() == at::kStrided && t.device() == like.device();
}

bool fit_draws(const at::Tensor &x, const MaybeTensor &seed_at, double p, int64_t call) {
  return p >= 0.0 && p <= 1.0 && call >= 0 && call <= (int64_t)UINT32_MAX &&
         (!given(seed_at) || (same_place(*seed_at, x) && seed_at->scalar_type() == at::kLong &&
                              seed_at->numel() == 1));
}

// dropout of plain tensors; None where its arguments do not fit (the caller then
// says which) and for no elements.
py::object dropout(const at::Tensor &x, const MaybeTensor &residual, const MaybeTensor &seed_at,
                   double p, int64_t seed, int64_t call) {
  if (!g_more.dropout || !x.is_cuda() || x.layout() != at::kStrided || x.numel() == 0 ||
      grad_code(x.scalar_type()) < 0 || !fit_draws(x, seed_at, p, call))
    return py::none();
  if (given(residual) && (!same_place(*residual, x) || residual->sizes() != x.sizes() ||
                          (residual->scalar_type() != x.scalar_type() &&
                           residual->scalar_type() != at::kFloat)))
    return py::none();
  if (!differentiable({&x, pointer(residual)}))
    return py::cast(dropped(x, residual, {value(seed_at), p, seed, call}));
  return py::cast(Dropout::apply(x, residual, seed_at, p, seed, call));
}

// The sizes, types and draws of a call of layer_norm or add_layer_norm.
LumaLayerNormArgs norm_args(int64_t n, int64_t h, int64_t stream, int64_t branch, int64_t param,
                            double eps, const Draws &d) {
  LumaLayerNormArgs a{};
  a.n = n;
  a.h = h;
  a.stream = (int32_t)stream;
  a.branch = (int32_t)branch;
  a.param = (int32_t)param;
  a.eps = eps;
  a.drop = d.args();
  return a;
}

// y and, with a residual, the sum; (keep) each row's mean and 1 / deviation.
struct Normed {
  at::Tensor y, total, stats;
};

int64_t param_code(const MaybeTensor &weight, const MaybeTensor &bias) {
  return given(weight) ? grad_code(weight->scalar_type())
         : given(bias) ? grad_code(bias->scalar_type())
                       : LUMA_GRAD_F32;
}

Normed normed(const at::Tensor &x, const MaybeTensor &residual, const MaybeTensor &weight,
              const MaybeTensor &bias, double eps, const Draws &d, int64_t branch, bool keep) {
  const c10::DeviceGuard guard(x.device());
  const bool adds = given(residual);
  const at::Tensor &like = adds ? *residual : x;
  const int64_t h = x.size(x.dim() - 1), n = x.numel() / h;
  LumaLayerNormArgs a = norm_args(n, h, grad_code(like.scalar_type()), branch,
                                  param_code(weight, bias), eps, d);
  const at::Tensor xs = as_rows(x), rs = adds ? as_rows(*residual) : at::Tensor();
  const at::Tensor w = given(weight) ? dense(*weight) : at::Tensor();
  const at::Tensor b = given(bias) ? dense(*bias) : at::Tensor();
  Normed o;
  o.y = fresh(x.sizes(), kTypes[branch], x);
  a.x = xs.const_data_ptr();
  a.ld_x = ld_of(xs);
  if (adds) {
    o.total = fresh(x.sizes(), like.scalar_type(), x);
    a.residual = rs.const_data_ptr();
    a.ld_residual = ld_of(rs);
    a.total = o.total.mutable_data_ptr();
  }
  a.weight = w.defined() ? w.const_data_ptr() : nullptr;
  a.bias = b.defined() ? b.const_data_ptr() : nullptr;
  a.y = o.y.mutable_data_ptr();
  if (keep) {
    o.stats = fresh({2 * n}, at::kFloat, x);
    a.stats = o.stats.mutable_data_ptr<float>();
  }
  run(g_more.norm_forward(&a, current_stream(x.device().index())));
  return o;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  // y, or y and the sum.
  static Variables forward(Context *ctx, const at::Tensor &x, const MaybeTensor &residual,
                           const MaybeTensor &weight, const MaybeTensor &bias,
                           const MaybeTensor &seed_at, double eps, double p, int64_t seed,
                           int64_t call, int64_t branch) {
    const bool adds = given(residual);
    const Draws d{value(seed_at), p, seed, call};
    const Normed o = normed(x, residual, weight, bias, eps, d, branch, true);
    ctx->save_for_backward({adds ? o.total : x, value(weight), o.stats, d.seed_at});
    ctx->saved_data["p"] = p;
    // (last which inputs there are: a gradient's number counts those alone)
    ctx->saved_data["numbers"] =
        std::vector<int64_t>{seed, call, branch, param_code(weight, bias),
                             1 | adds << 1 | given(weight) << 2 | given(bias) << 3};
    ctx->set_materialize_grads(false);
    return adds ? Variables{o.y, o.total} : Variables{o.y};
  }

  static Variables backward(Context *ctx, Variables grads) {
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &s = saved[0], &weight = saved[1], &stats = saved[2];
    const auto numbers = ctx->saved_data["numbers"].toIntVector();
    const Draws d{saved[3], ctx->saved_data["p"].toDouble(), numbers[0], numbers[1]};
    const int64_t branch = numbers[2], param = numbers[3], inputs = numbers[4];
    const bool adds = inputs >> 1 & 1;
    bool want[4];
    for (int i = 0, edge = 0; i < 4; ++i)
      want[i] = (inputs >> i & 1) && ctx->needs_input_grad(edge++);
    at::Tensor out[4];      // of x, residual, weight, bias
    at::Tensor d_y = grads[0], d_total = adds ? grads[1] : at::Tensor();
    const int64_t stream = grad_code(s.scalar_type());
    // (without draws the sum's gradient is that of both)
    const bool one = adds && d.p == 0.0 && stream == branch;
    if (!d_y.defined() && d_total.defined()) {
      // The sum alone was used: its norm has no part in the gradients, whether those of
      // its rows are numbers or not.
      at::AutoDispatchBelowADInplaceOrView below;
      d_total = d_total.to(s.scalar_type());
      if (want[0]) out[0] = one ? d_total : dropped_grad(d_total, d, branch);
      if (want[1]) out[1] = d_total;
      for (int i = 2; i < 4; ++i)
        if (want[i]) out[i] = at::zeros({s.size(s.dim() - 1)}, s.options().dtype(kTypes[param]));
    } else if (d_y.defined()) {
      at::AutoDispatchBelowADInplaceOrView below;
      const bool want_x = want[0] && !one, want_r = want[1] || (one && want[0]);
      if (watched()) {
        static const auto op =
            op_of<std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor>(
                const at::Tensor &, const MaybeTensor &, const at::Tensor &, const MaybeTensor &,
                const at::Tensor &, const MaybeTensor &, double, int64_t, int64_t, int64_t, int64_t,
                bool, bool, bool, bool, bool)>("luma_amd::layer_norm_backward");
        std::tie(out[0], out[1], out[2], out[3]) =
            op.call(d_y, maybe(d_total), s, maybe(weight), stats, maybe(d.seed_at), d.p, d.seed,
                    d.call, branch, param, adds, want_x, want_r, want[2], want[3]);
        const bool keep[4] = {want_x, want_r, want[2], want[3]};
        for (int i = 0; i < 4; ++i)
          if (!keep[i]) out[i].reset();
      } else {
        const int64_t h = s.size(s.dim() - 1), n = s.numel() / h;
        LumaLayerNormArgs a = norm_args(n, h, stream, branch, param, 0.0, d);
        const at::Tensor ss = as_rows(s), dy = dense(d_y.to(kTypes[branch]));
        const at::Tensor w = weight.defined() ? dense(weight) : at::Tensor();
        const at::Tensor dt = d_total.defined() ? dense(d_total.to(s.scalar_type())) : at::Tensor();
        const c10::DeviceGuard guard(s.device());
        if (want_x) out[0] = fresh(s.sizes(), kTypes[adds ? branch : stream], s);
        if (want_r) out[1] = fresh(s.sizes(), kTypes[stream], s);
        if (want[2]) out[2] = fresh({h}, kTypes[param], s);
        if (want[3]) out[3] = fresh({h}, kTypes[param], s);
        a.x = ss.const_data_ptr();
        a.ld_x = ld_of(ss);
        if (adds) a.total = const_cast<void *>(ss.const_data_ptr());
        a.weight = w.defined() ? w.const_data_ptr() : nullptr;
        a.stats = const_cast<float *>(stats.const_data_ptr<float>());
        a.d_y = dy.const_data_ptr();
        a.d_total = dt.defined() ? dt.const_data_ptr() : nullptr;
        void **to[4] = {&a.d_x, &a.d_residual, &a.d_weight, &a.d_bias};
        for (int i = 0; i < 4; ++i) *to[i] = out[i].defined() ? out[i].mutable_data_ptr() : nullptr;
        at::Tensor workspace;
        if (want[2] || want[3]) {
          const int64_t bytes = g_more.norm_workspace(&a);
          TORCH_CHECK(bytes >= 0, g_lib.error());
          workspace = fresh({bytes}, at::kByte, s);
          a.workspace = workspace.mutable_data_ptr();
          a.workspace_bytes = bytes;
        }
        run(g_more.norm_backward(&a, current_stream(s.device().index())));
      }
      if (one && want[0]) out[0] = out[1];
      if (one && !want[1]) out[1].reset();
    }
    once({&out[0], &out[1], &out[2], &out[3]}, adds ? "add_layer_norm" : "layer_norm", s, weight,
         grads[0], adds ? grads[1] : at::Tensor());
    return {out[0], out[1], out[2], out[3], at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(),
            at::Tensor(), at::Tensor()};
  }
};

// layer_norm and (with a residual) add_layer_norm of plain tensors: y, or y and the
// sum; None where the arguments do not fit (the caller then says which) and for no
// elements.  branch: y's LUMA_GRAD_*.
py::object layer_norm(const at::Tensor &x, const MaybeTensor &residual, const MaybeTensor &weight,
                      const MaybeTensor &bias, const MaybeTensor &seed_at, double eps, double p,
                      int64_t seed, int64_t call, int64_t branch) {
  if (!g_more.norm_forward || !x.is_cuda() || x.layout() != at::kStrided || x.dim() < 1 ||
      x.numel() == 0 || grad_code(x.scalar_type()) < 0 || branch < 0 || branch > 2 ||
      !(eps >= 0.0) || !fit_draws(x, seed_at, p, call))
    return py::none();
  const bool adds = given(residual);
  const at::Tensor &like = adds ? *residual : x;
  if (adds && (!same_place(like, x) || like.sizes() != x.sizes())) return py::none();
  const int64_t stream = grad_code(like.scalar_type());
  if (stream < 0 || (stream != branch && stream != LUMA_GRAD_F32)) return py::none();
  if (adds && grad_code(x.scalar_type()) != branch) return py::none();
  const MaybeTensor *const params[2] = {&weight, &bias};
  for (const MaybeTensor *t : params)
    if (given(*t)) {
      const int64_t code = grad_code((*t)->scalar_type());
      if (!same_place(**t, x) || (*t)->dim() != 1 || (*t)->size(0) != x.size(x.dim() - 1) ||
          (code != LUMA_GRAD_F32 && code != branch) ||
          (given(weight) && given(bias) && weight->scalar_type() != bias->scalar_type()))
        return py::none();
    }
  if (!differentiable({&x, &like, pointer(weight), pointer(bias)})) {
    const Normed o = normed(x, residual, weight, bias, eps, {value(seed_at), p, seed, call}, branch,
                            false);
    return adds ? py::object(py::make_tuple(o.y, o.total)) : py::cast(o.y);
  }
  const Variables out = LayerNorm::apply(x, residual, weight, bias, seed_at, eps, p, seed, call,
                                         branch);
  return adds ? py::object(py::make_tuple(out[0], out[1])) : py::cast(out[0]);
}

// The operands of a policy loss as rows.
struct PolicyRows {
  at::Tensor logp, old, ref, advantage, mask;
};

LumaPolicyArgs policy_args(const at::Tensor &logp, const at::Tensor &old,
                           const at::Tensor &advantage, const at::Tensor &mask,
                           const at::Tensor &ref, const at::Tensor &share, double low, double high,
                           double kl, int64_t reduction, PolicyRows &r) {
  const bool each = advantage.dim() == logp.dim();
  r.logp = as_rows(logp);
  r.old = as_rows(old);
  if (ref.defined()) r.ref = as_rows(ref);
  if (mask.defined()) r.mask = as_rows(mask);
  r.advantage = each ? as_rows(advantage) : dense(advantage);
  LumaPolicyArgs a{};
  a.logp = r.logp.const_data_ptr();
  a.old_logp = r.old.const_data_ptr();
  a.ref_logp = ref.defined() ? r.ref.const_data_ptr() : nullptr;
  a.advantage = r.advantage.const_data_ptr<float>();
  a.mask = mask.defined() ? static_cast<const uint8_t *>(r.mask.const_data_ptr()) : nullptr;
  a.rows = r.logp.size(0);
  a.length = r.logp.size(1);
  a.ld_logp = ld_of(r.logp);
  a.ld_old = ld_of(r.old);
  a.ld_ref = ref.defined() ? ld_of(r.ref) : 0;
  a.ld_mask = mask.defined() ? ld_of(r.mask) : 0;
  a.ld_advantage = each ? ld_of(r.advantage) : 1;
  a.advantage_each = each;
  a.dtype = grad_code(logp.scalar_type());
  a.reduction = (int32_t)reduction;
  a.clip_low = low;
  a.clip_high = high;
  a.kl_weight = kl;
  a.share = share.defined() ? share.mutable_data_ptr<float>() : nullptr;
  return a;
}

// The loss, (figures) its figures, (keep) the rows' shares of a mean.
struct PolicyLoss {
  at::Tensor loss, stats, share;
};

PolicyLoss policy_of(const at::Tensor &logp, const at::Tensor &old, const at::Tensor &advantage,
                     const MaybeTensor &mask, const MaybeTensor &ref, double low, double high,
                     double kl, int64_t reduction, bool keep, bool figures) {
  const c10::DeviceGuard guard(logp.device());
  const int64_t rows = logp.numel() / logp.size(logp.dim() - 1);
  PolicyLoss o;
  o.loss = fresh(reduction == LUMA_XENT_NONE ? logp.sizes() : at::IntArrayRef(), at::kFloat,
                 logp);
  if (figures) o.stats = fresh({LUMA_POLICY_STATS}, at::kFloat, logp);
  if (keep) o.share = fresh({rows + 1}, at::kFloat, logp);
  PolicyRows r;
  LumaPolicyArgs a = policy_args(logp, old, advantage, value(mask), value(ref), o.share, low, high,
                                 kl, reduction, r);
  a.loss = o.loss.mutable_data_ptr<float>();
  a.stats = figures ? o.stats.mutable_data_ptr<float>() : nullptr;
  const int64_t bytes = g_more.policy_workspace(&a);
  TORCH_CHECK(bytes >= 0, g_lib.error());
  at::Tensor workspace;
  if (bytes) {
    workspace = fresh({bytes}, at::kByte, logp);
    a.workspace = workspace.mutable_data_ptr();
    a.workspace_bytes = bytes;
  }
  run(g_more.policy_forward(&a, current_stream(logp.device().index())));
  return o;
}

struct Policy : torch::autograd::Function<Policy> {
  static Variables forward(Context *ctx, const at::Tensor &logp, const at::Tensor &old,
                           const at::Tensor &advantage, const MaybeTensor &mask,
                           const MaybeTensor &ref, double low, double high, double kl,
                           int64_t reduction, bool figures) {
    const PolicyLoss o = policy_of(logp, old, advantage, mask, ref, low, high, kl, reduction, true,
                                   figures);
    ctx->save_for_backward({logp, old, advantage, value(mask), value(ref), o.share});
    ctx->saved_data["low"] = low;
    ctx->saved_data["high"] = high;
    ctx->saved_data["kl"] = kl;
    ctx->saved_data["reduction"] = reduction;
    ctx->set_materialize_grads(false);
    if (!figures) return {o.loss};
    ctx->mark_non_differentiable({o.stats});
    return {o.loss, o.stats};
  }

  static Variables backward(Context *ctx, Variables grads) {
    at::Tensor d_logp;
    if (grads[0].defined() && ctx->needs_input_grad(0)) {
      const auto saved = ctx->get_saved_variables();
      const at::Tensor &logp = saved[0];
      const double low = ctx->saved_data["low"].toDouble();
      const double high = ctx->saved_data["high"].toDouble();
      const double kl = ctx->saved_data["kl"].toDouble();
      const int64_t reduction = ctx->saved_data["reduction"].toInt();
      {
        at::AutoDispatchBelowADInplaceOrView below;
        if (watched()) {
          static const auto op =
              op_of<at::Tensor(const at::Tensor &, const at::Tensor &, const at::Tensor &,
                               const at::Tensor &, const MaybeTensor &, const MaybeTensor &,
                               const at::Tensor &, double, double, double, int64_t)>(
                  "luma_amd::policy_loss_backward");
          d_logp = op.call(grads[0], logp, saved[1], saved[2], maybe(saved[3]), maybe(saved[4]),
                           saved[5], low, high, kl, reduction);
        } else {
          const c10::DeviceGuard guard(logp.device());
          const at::Tensor g = dense(grads[0].to(at::kFloat));
          d_logp = fresh(logp.sizes(), logp.scalar_type(), logp);
          PolicyRows r;
          LumaPolicyArgs a = policy_args(logp, saved[1], saved[2], saved[3], saved[4], saved[5],
                                         low, high, kl, reduction, r);
          a.grad_loss = g.const_data_ptr<float>();
          a.d_logp = d_logp.mutable_data_ptr();
          run(g_more.policy_backward(&a, current_stream(logp.device().index())));
        }
      }
      once({&d_logp}, "policy_loss", logp, grads[0]);
    }
    return {d_logp, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(),
            at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

// policy_loss of plain tensors: the loss, or with its figures; None where its arguments do
// not fit (the caller then says which) and for no tokens.
py::object policy_loss(const at::Tensor &logp, const at::Tensor &old, const at::Tensor &advantage,
                       const MaybeTensor &mask, const MaybeTensor &ref, double low, double high,
                       double kl, int64_t reduction, bool figures) {
  const int64_t d = logp.dim();
  if (!g_more.policy_forward || !logp.is_cuda() || logp.layout() != at::kStrided || d < 1 ||
      logp.numel() == 0 || grad_code(logp.scalar_type()) < 0 || !same_place(old, logp) ||
      old.scalar_type() != logp.scalar_type() || old.sizes() != logp.sizes() ||
      !same_place(advantage, logp) || advantage.scalar_type() != at::kFloat ||
      (advantage.sizes() != logp.sizes() && advantage.sizes() != logp.sizes().slice(0, d - 1)) ||
      !(low >= 0.0 && low <= 1.0) || !(high >= 0.0) || kl != kl)
    return py::none();
  if (given(mask) && (!same_place(*mask, logp) || mask->scalar_type() != at::kBool ||
                      mask->sizes() != logp.sizes()))
    return py::none();
  if (given(ref) && (!same_place(*ref, logp) || ref->scalar_type() != logp.scalar_type() ||
                     ref->sizes() != logp.sizes()))
    return py::none();
  if (!differentiable({&logp, &old, &advantage, pointer(ref)})) {
    const PolicyLoss o = policy_of(logp, old, advantage, mask, ref, low, high, kl, reduction, false,
                                   figures);
    return figures ? py::object(py::make_tuple(o.loss, o.stats)) : py::cast(o.loss);
  }
  // (what requires a gradient and gets none stays out of the graph)
  auto constant = [](const at::Tensor &t) { return t.requires_grad() ? t.detach() : t; };
  const Variables out = Policy::apply(logp, constant(old), constant(advantage), mask,
                                      given(ref) ? MaybeTensor(constant(*ref)) : ref, low, high, kl,
                                      reduction, figures);
  return figures ? py::object(py::make_tuple(out[0], out[1])) : py::cast(out[0]);
}

PYBIND11_MODULE(_luma_host, m) {
  m.doc() = "Host-side bookkeeping of LUMA.step (pointer refresh of a planned step) and of the "
            "gradient norm (its table); the eager calls of the operators beside the step.";
  py::object torch = py::module_::import("torch");
  g_tensor_type = reinterpret_cast<PyTypeObject *>(torch.attr("Tensor").ptr());
  g_param_type = reinterpret_cast<PyTypeObject *>(torch.attr("nn").attr("Parameter").ptr());
  // the module holds them for its lifetime
  Py_INCREF(g_tensor_type);
  Py_INCREF(g_param_type);
  m.def("refresh", &refresh, py::arg("groups"), py::arg("planned"), py::arg("has_grad"),
        py::arg("row_param"), py::arg("layout_at"), py::arg("layout"), py::arg("gdtype"),
        py::arg("table"), py::arg("row_bytes"), py::arg("grad_off"), py::arg("param_off"),
        py::arg("device"), py::arg("cands") = py::none());
  m.def("same_pointers", &same_pointers);
  m.def("bump_steps", &bump_steps);
  m.def("grad_rows", &grad_rows);
  m.def("xent", &xent);
  m.def("grad_norm", &grad_norm);
  m.def("bind", &bind);
  m.def("bind_more", &bind_more);
  m.def("dropout", &dropout);
  m.def("layer_norm", &layer_norm);
  m.def("policy_loss", &policy_loss);
  // the torch whose headers this module was compiled against: it reads
  // TensorImpl fields in that version's inline layout
  m.attr("torch_version") = LUMA_TORCH_VERSION;
}
