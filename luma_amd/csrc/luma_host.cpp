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

PYBIND11_MODULE(_luma_host, m) {
  m.doc() = "Host-side bookkeeping of LUMA.step (pointer refresh of a planned step) and of the "
            "gradient norm (its table); linear_cross_entropy's eager calls.";
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
  // the torch whose headers this module was compiled against: it reads
  // TensorImpl fields in that version's inline layout
  m.attr("torch_version") = LUMA_TORCH_VERSION;
}
