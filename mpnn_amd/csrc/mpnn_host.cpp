// Host side of the entry points that take many tensors or are called once per decoded token: argument checks, pointer tables
// and output allocation in C++.  From Python an attribute of a tensor costs 50-150 ns and a ctypes call 3 us: checking and
// tabulating the six lists of an optimizer step over 118 tensors took 270 us, the beam calls 12-30 us - many times what the
// kernels behind them take at those sizes.  The kernels are reached through the C ABI (include/mpnn_hip.h); mpnn_amd/_lib.py
// hands over the addresses of the library's functions (bind).
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/ge.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <climits>
#include <memory>
#include <string>
#include <utility>
#include <vector>

#include "mpnn_hip.h"

namespace {

struct Error {
  PyObject* type;
  std::string text;
};
[[noreturn]] void value_error(std::string s) { throw Error{PyExc_ValueError, std::move(s)}; }
[[noreturn]] void runtime_error(std::string s) { throw Error{PyExc_RuntimeError, std::move(s)}; }
[[noreturn]] void type_error(std::string s) { throw Error{PyExc_TypeError, std::move(s)}; }

decltype(&mpnn_beam_select) f_select;
decltype(&mpnn_beam_select_workspace) f_select_ws;
decltype(&mpnn_beam_reorder) f_reorder;
decltype(&mpnn_grad_sumsq_parts) f_parts;
decltype(&mpnn_adamw_mixed) f_adamw;
decltype(&mpnn_last_error) f_error;

void check_rc(int rc, const char* name) {
  if (rc) runtime_error(std::string(name) + " failed (code " + std::to_string(rc) + "): " + f_error());
}

// ---- arguments ----
const at::Tensor& tensor(PyObject* o, const char* what, const char* name) {
  if (!THPVariable_Check(o)) type_error(std::string("mpnn_amd.") + what + ": " + name + " must be a tensor");
  return THPVariable_Unpack(o);
}
std::string str(const c10::Device& d) { return d.str(); }

const at::Tensor& on_gpu(PyObject* o, const char* what, const char* name, const c10::Device* dev = nullptr) {
  const at::Tensor& t = tensor(o, what, name);
  if (!t.is_cuda())
    runtime_error(std::string("mpnn_amd.") + what + ": `" + name + "` must be on a ROCm device (got " + str(t.device()) +
                  "); the HIP path has no CPU fallback");
  if (dev && t.device() != *dev)
    runtime_error(std::string("mpnn_amd.") + what + ": `" + name + "` is on " + str(t.device()) + ", the other tensors on " +
                  str(*dev));
  return t;
}

long long integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    type_error("mpnn_amd: an integer was expected");
  }
  return v;
}
double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    type_error("mpnn_amd: a number was expected");
  }
  return v;
}
bool whole(const at::Tensor& t) { return t.scalar_type() == at::kInt || t.scalar_type() == at::kLong; }

// the items of a list or tuple (borrowed)
struct Items {
  PyObject* seq;
  PyObject** at;
  Py_ssize_t n;
  explicit Items(PyObject* o) : seq(PySequence_Fast(o, "a list of tensors was expected")) {
    if (!seq) {
      PyErr_Clear();
      type_error("mpnn_amd: a list of tensors was expected");
    }
    at = PySequence_Fast_ITEMS(seq);
    n = PySequence_Fast_GET_SIZE(seq);
  }
  ~Items() { Py_DECREF(seq); }
  Items(const Items&) = delete;
};

void* stream_of(const c10::Device& d) { return (void*)c10::hip::getCurrentHIPStream(d.index()).stream(); }
void touched(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

template <typename F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (const Error& e) {
    PyErr_SetString(e.type, e.text.c_str());
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// ---- beam_select(logits, scores, bias, forced, n_out) ----
at::Tensor rows(const at::Tensor& t) { return t.size(-1) == 1 || t.stride(-1) == 1 ? t : t.contiguous(); }

PyObject* py_select(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    if (n_args != 5) type_error("beam_select: five arguments");
    const char* what = "beam_select";
    const at::Tensor& given = on_gpu(a[0], what, "logits");
    const c10::Device dev = given.device();
    const at::Tensor& sc = on_gpu(a[1], what, "scores", &dev);
    const auto type = given.scalar_type();
    const int dt = type == at::kFloat ? 0 : type == at::kBFloat16 ? 1 : type == at::kHalf ? 2 : -1;
    if (given.dim() != 3 || dt < 0) value_error("mpnn_amd.beam_select: logits must be [B, W, V] in fp32, bf16 or fp16");
    const long long B = given.size(0), W = given.size(1), V = given.size(2);
    if (sc.dim() != 2 || sc.size(0) != B || sc.size(1) != W || sc.scalar_type() != at::kFloat)
      value_error("mpnn_amd.beam_select: scores must be fp32 [" + std::to_string(B) + ", " + std::to_string(W) + "]");
    const long long n = a[4] == Py_None ? W : integer(a[4]);
    if (W < 1 || W > 256 || n < 1 || n > 256 || V < 1 || V > (1 << 22) || B >= (1LL << 31))
      value_error("mpnn_amd.beam_select: 1..256 beams, 1..256 hypotheses kept, 1..2^22 tokens (got " + std::to_string(W) + ", " +
                  std::to_string(n) + ", " + std::to_string(V) + ")");
    const c10::OptionalDeviceGuard guard(dev);
    const at::Tensor logits = rows(given), scores = sc.contiguous();
    at::Tensor bias, forced;
    if (a[2] != Py_None) {
      const at::Tensor& t = on_gpu(a[2], what, "bias", &dev);
      if (t.scalar_type() != at::kFloat) value_error("mpnn_amd.beam_select: bias must be fp32");
      if (t.dim() < 1 || t.size(-1) != V)
        value_error("mpnn_amd.beam_select: bias must end in the " + std::to_string(V) + " tokens");
      bias = rows(t).expand({B, W, V});
    }
    if (a[3] != Py_None) {
      const at::Tensor& t = on_gpu(a[3], what, "forced", &dev);
      if (!whole(t)) value_error("mpnn_amd.beam_select: forced must be integers");
      forced = t.to(at::kLong);
      if (forced.dim() == 1) forced = forced.unsqueeze(1);
      forced = forced.expand({B, W}).contiguous();
    }
    const auto as_long = given.options().dtype(at::kLong);
    at::Tensor out = at::empty({B, n}, given.options().dtype(at::kFloat)), parent = at::empty({B, n}, as_long),
               token = at::empty({B, n}, as_long);
    if (B) {
      const long long need = f_select_ws(dt, (int)B, (int)W, (int)V, (int)n);
      at::Tensor ws;
      if (need > 0) ws = at::empty({need}, given.options().dtype(at::kByte));
      check_rc(f_select(logits.const_data_ptr(), dt, logits.stride(0), logits.stride(1), scores.const_data_ptr<float>(),
                        bias.defined() ? bias.const_data_ptr<float>() : nullptr, bias.defined() ? bias.stride(0) : 0,
                        bias.defined() ? bias.stride(1) : 0, forced.defined() ? forced.const_data_ptr<int64_t>() : nullptr,
                        (int)B, (int)W, (int)V, (int)n, out.data_ptr<float>(), parent.data_ptr<int64_t>(),
                        token.data_ptr<int64_t>(), need > 0 ? ws.data_ptr() : nullptr, need > 0 ? need : 0, stream_of(dev)),
               "mpnn_beam_select");
    }
    PyObject* r = PyTuple_New(3);
    if (!r) return nullptr;
    PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(out));
    PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(parent));
    PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(token));
    return r;
  });
}

// ---- beam_reorder ----
struct Layout {
  bool regular;
  long long n_mid, stride_mid, run;   // elements
};

// the dimensions behind [B, W] as one strided dimension of contiguous runs; by_position: the first of them is that dimension
Layout state_layout(const at::Tensor& x, bool by_position) {
  long long n[2] = {1, 1}, s[2] = {0, 0};   // dimensions that do not merge, outermost first; more than two: irregular
  int k = 0;
  for (int64_t d = 2; d < x.dim(); ++d) {
    const long long size = x.size(d), stride = x.stride(d);
    const bool fixed = by_position && d == 2;
    if (size == 1 && !fixed) continue;
    const bool may_merge = k > 0 && !(by_position && k == 1);
    if (may_merge && s[k - 1] == size * stride) {
      n[k - 1] *= size;
      s[k - 1] = stride;
      continue;
    }
    if (k == 2) return {false, 0, 0, 0};
    n[k] = size;
    s[k] = stride;
    ++k;
  }
  const int head = by_position ? 1 : 0;
  long long run = 1;
  if (k > head && s[k - 1] == 1) run = n[--k];
  if (k > 1) return {false, 0, 0, 0};
  return k == 1 ? Layout{true, n[0], s[0], run} : Layout{true, 1, 0, run};
}

// elements from the first to behind the last; 0 if two indices share one
long long state_span(const at::Tensor& x) {
  std::vector<std::pair<long long, long long>> dims;
  for (int64_t d = 0; d < x.dim(); ++d)
    if (x.size(d) > 1) dims.emplace_back(x.stride(d), x.size(d));
  std::sort(dims.begin(), dims.end());
  long long extent = 1;
  for (const auto& d : dims) {
    if (d.first < extent) return 0;
    extent += d.first * (d.second - 1);
  }
  return extent;
}

// a state's rows: runs of bytes at up to three strides, the widest first, each at least what lies inside it spans (state_span)
struct Rows {
  int n = 0;
  long long stride[3], count[3], extent[4];   // extent[i]: bytes from level i's first to behind its last; [n]: the run
};
struct Span {
  long long begin, end;               // bytes
  Rows rows;
};

Span state_rows(const at::Tensor& x, const Layout& l, long long extent) {
  const long long item = x.element_size(), begin = (long long)x.const_data_ptr();
  std::pair<long long, long long> dims[3] = {{x.stride(0), x.size(0)}, {x.stride(1), x.size(1)}, {l.stride_mid, l.n_mid}};
  std::sort(dims, dims + 3, [](const auto& a, const auto& b) { return a.first > b.first; });
  Span s = {begin, begin + extent * item, {}};
  Rows& r = s.rows;
  for (const auto& d : dims)
    if (d.second > 1) {
      r.stride[r.n] = d.first * item;
      r.count[r.n++] = d.second;
    }
  r.extent[r.n] = l.run * item;
  for (int i = r.n - 1; i >= 0; --i) r.extent[i] = r.stride[i] * (r.count[i] - 1) + r.extent[i + 1];
  return s;
}

long long floor_div(long long x, long long y) { return x / y - (x % y < 0); }

// a's rows from level i on, b's from level j on d bytes behind them: do they share a byte?  The level with the wider stride is
// taken apart (both, if they are equal: what counts is then the distance of two blocks); `left`: steps until it says yes.
bool meet(const Rows& a, int i, const Rows& b, int j, long long d, int& left) {
  if (d >= a.extent[i] || -d >= b.extent[j]) return false;
  if ((i == a.n && j == b.n) || --left < 0) return true;
  const long long sa = i < a.n ? a.stride[i] : 0, sb = j < b.n ? b.stride[j] : 0, s = std::max(sa, sb);
  const int da = sa == s, db = sb == s;
  const long long lo = std::max(da ? 1 - a.count[i] : 0, floor_div(-b.extent[j + db] - d, s) + 1);
  const long long hi = std::min(db ? b.count[j] - 1 : 0, -floor_div(d - a.extent[i + da], s) - 1);
  for (long long k = lo; k <= hi; ++k)
    if (meet(a, i + da, b, j + db, d + k * s, left)) return true;
  return false;
}

// two states share no byte though their ranges meet: rows of one lie between those of the other
bool apart(const Span& x, const Span& y) {
  const Rows &a = x.rows, &b = y.rows;
  const long long d = y.begin - x.begin;
  // all strides are multiples of the smallest, and the runs lie side by side in it
  const long long m = std::min(a.n ? a.stride[a.n - 1] : LLONG_MAX, b.n ? b.stride[b.n - 1] : LLONG_MAX);
  bool even = m < LLONG_MAX;
  for (int i = 0; i < a.n; ++i) even &= a.stride[i] % m == 0;
  for (int i = 0; i < b.n; ++i) even &= b.stride[i] % m == 0;
  if (even) {
    const long long r = d - floor_div(d, m) * m;
    if (r >= a.extent[a.n] && r + b.extent[b.n] <= m) return true;
  }
  int left = 4096;
  return !meet(a, 0, b, 0, d, left);
}

PyObject* py_reorder(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    if (n_args != 4) type_error("beam_reorder: four arguments");
    const char* what = "beam_reorder";
    const at::Tensor& given = on_gpu(a[1], what, "parent");
    const c10::Device dev = given.device();
    if (given.dim() != 2 || !whole(given)) value_error("mpnn_amd.beam_reorder: parent must be integers [B, W]");
    const long long B = given.size(0), W = given.size(1);
    if (W < 1 || W > 256 || B > 65535)
      value_error("mpnn_amd.beam_reorder: 1..256 beams and at most 65535 groups (got " + std::to_string(W) + ", " +
                  std::to_string(B) + ")");
    const bool positions = a[2] != Py_None;
    if (a[3] != Py_None && !positions) value_error("mpnn_amd.beam_reorder: rank needs a length");
    PyObject* single[1] = {a[0]};
    const bool one = THPVariable_Check(a[0]);
    std::unique_ptr<Items> list;
    if (!one) list = std::make_unique<Items>(a[0]);
    PyObject** items = one ? single : list->at;
    const Py_ssize_t n = one ? 1 : list->n;
    long long L = -1;
    std::vector<mpnn_beam_state> table;
    std::vector<Span> spans;
    table.reserve(n);
    spans.reserve(n);
    for (Py_ssize_t i = 0; i < n; ++i) {
      const at::Tensor& x = on_gpu(items[i], what, "states", &dev);
      if (x.dim() < 2 || x.size(0) != B || x.size(1) != W)
        value_error("mpnn_amd.beam_reorder: a state must be [" + std::to_string(B) + ", " + std::to_string(W) + ", ...]");
      if (x.requires_grad()) runtime_error("mpnn_amd.beam_reorder moves states in place: they may not require gradients");
      if (positions) {
        if (x.dim() < 3 || (L >= 0 && x.size(2) != L))
          value_error("mpnn_amd.beam_reorder: with a length, every state must be [B, W, positions, ...]");
        L = x.size(2);
      }
      if (x.numel() == 0) continue;
      const Layout lay = state_layout(x, positions);
      if (!lay.regular || lay.n_mid >= (1LL << 31))
        value_error("mpnn_amd.beam_reorder: a state's rows must be contiguous, or one strided dimension of contiguous runs");
      const long long extent = state_span(x);
      if (!extent) value_error("mpnn_amd.beam_reorder: rows of a state share memory");
      const long long item = x.element_size();
      const long long sb = B > 1 ? x.stride(0) * item : 0, sw = W > 1 ? x.stride(1) * item : 0, sm = lay.stride_mid * item;
      char* data = (char*)x.data_ptr();
      table.push_back({data, sb, sw, sm, lay.run * item, (int)lay.n_mid});
      spans.push_back(state_rows(x, lay, extent));
    }
    std::sort(spans.begin(), spans.end(), [](const Span& x, const Span& y) { return x.begin < y.begin; });
    for (size_t i = 0; i < spans.size(); ++i)
      for (size_t j = i + 1; j < spans.size() && spans[j].begin < spans[i].end; ++j)
        if (!apart(spans[i], spans[j])) value_error("mpnn_amd.beam_reorder: two states share memory");
    const c10::OptionalDeviceGuard guard(dev);
    // an index that lies in a state would change while it is read
    auto beside_states = [&](at::Tensor t) {
      const long long begin = (long long)t.const_data_ptr(), end = begin + t.numel() * t.element_size();
      for (const Span& s : spans)
        if (begin < s.end && s.begin < end) return t.clone();
      return t;
    };
    long long all = -1;
    at::Tensor lengths, rank;
    if (positions) {
      if (THPVariable_Check(a[2])) {
        lengths = on_gpu(a[2], what, "length", &dev);
        if (lengths.dim() != 1 || lengths.size(0) != B || !whole(lengths))
          value_error("mpnn_amd.beam_reorder: length must be an int or integers [" + std::to_string(B) + "]");
      } else {
        all = integer(a[2]);
      }
    }
    if (a[3] != Py_None) {
      rank = on_gpu(a[3], what, "rank", &dev);
      if (!whole(rank) || (L >= 0 && (rank.dim() != 2 || rank.size(0) != B || rank.size(1) != L)))
        value_error("mpnn_amd.beam_reorder: rank must be integers [" + std::to_string(B) + ", " + std::to_string(L) + "]");
    }
    // The library compares in 32 bits.  Positions without a rank are below 2^31, so clamping a length changes nothing; where a
    // rank, or the length it is compared with, has 64 bits, the comparison's result takes its place: 0 < 1 moves, 1 < 1 stays.
    constexpr long long most = 0x7fffffff;
    int length_all = -1;
    if (positions && !table.empty()) {
      if (rank.defined() && (rank.scalar_type() == at::kLong ||
                             (lengths.defined() ? lengths.scalar_type() == at::kLong : all < 0 || all > most))) {
        at::Tensor stays = at::empty(rank.sizes(), rank.options().dtype(at::kInt));
        if (lengths.defined()) at::ge_out(stays, rank, lengths.unsqueeze(1));
        else at::ge_out(stays, rank.to(at::kLong), at::Scalar((int64_t)all));
        rank = stays;
        lengths.reset();
        length_all = 1;
      } else {
        if (rank.defined()) rank = beside_states(rank.contiguous());
        if (!lengths.defined()) length_all = (int)std::max(0LL, std::min(all, most));
        else if (lengths.scalar_type() == at::kLong) lengths = lengths.clamp(0, most).to(at::kInt);
        else lengths = beside_states(lengths.contiguous());
      }
    }
    if (!table.empty()) {
      const at::Tensor parent = beside_states(given.to(at::kLong).contiguous());
      check_rc(f_reorder((int)table.size(), table.data(), parent.const_data_ptr<int64_t>(), (int)B, (int)W, length_all,
                         lengths.defined() ? lengths.const_data_ptr<int>() : nullptr,
                         rank.defined() ? rank.const_data_ptr<int>() : nullptr, stream_of(dev)),
               "mpnn_beam_reorder");
      for (Py_ssize_t i = 0; i < n; ++i) touched(THPVariable_Unpack(items[i]));
    }
    Py_INCREF(a[0]);
    return a[0];
  });
}

// ---- optimizer ----
constexpr int kBlock = 64, kParts = 256;

// Tensors cut from a few buffers, or made list by list, first: lists are a few ascending runs, and where no two runs meet, no two
// tensors do.  (No time that shows in a step of 300 tensors; Ranges, which takes any, 5-6 us for the default model's 118 tensors
// and their state, as the allocator deals them out.)
struct Runs {
  static constexpr int kMost = 24;
  static constexpr long long kGap = 16384;   // a larger one may hold another list
  const char *begin[kMost], *end[kMost];
  int n = 0;
  // false: more runs than this holds
  bool add(const void* p, long long bytes) {
    const char* b = (const char*)p;
    if (n && b >= end[n - 1] && b - end[n - 1] <= kGap) {
      end[n - 1] = b + bytes;
      return true;
    }
    if (n == kMost) return false;
    begin[n] = b;
    end[n++] = b + bytes;
    return true;
  }
  // whether some run of this one meets another, or one of `read`
  bool meet(const Runs& read) const {
    for (int i = 0; i < n; ++i) {
      for (int j = 0; j < i; ++j)
        if (begin[i] < end[j] && begin[j] < end[i]) return true;
      for (int j = 0; j < read.n; ++j)
        if (begin[i] < read.end[j] && read.begin[j] < end[i]) return true;
    }
    return false;
  }
};

// Any tensors: their byte ranges, kept as ascending runs, merged into one.
struct Ranges {
  using Range = std::pair<const char*, const char*>;
  std::vector<Range> at;
  std::vector<size_t> run;            // where each run begins
  void add(const void* p, long long bytes) {
    const char* begin = (const char*)p;
    if (at.empty() || begin < at.back().second) run.push_back(at.size());
    at.emplace_back(begin, begin + bytes);
  }
  // into one ascending run; false if two share a byte
  bool sort() {
    std::vector<std::pair<size_t, size_t>> part;   // begin, end of the runs
    for (size_t i = 0; i < run.size(); ++i) part.emplace_back(run[i], i + 1 < run.size() ? run[i + 1] : at.size());
    std::sort(part.begin(), part.end(), [&](const auto& x, const auto& y) { return at[x.first].first < at[y.first].first; });
    std::vector<Range> out;
    std::vector<size_t> edge = {0};
    out.reserve(at.size());
    for (const auto& x : part) {
      out.insert(out.end(), at.begin() + x.first, at.begin() + x.second);
      edge.push_back(out.size());
    }
    for (; edge.size() > 2;) {
      std::vector<size_t> next = {0};
      for (size_t i = 0; i + 1 < edge.size(); i += 2) {
        const size_t end = edge[std::min(i + 2, edge.size() - 1)];
        if (edge[i + 1] < end && out[edge[i + 1]].first < out[edge[i + 1] - 1].second)
          std::inplace_merge(out.begin() + edge[i], out.begin() + edge[i + 1], out.begin() + end);
        next.push_back(end);
      }
      edge.swap(next);
    }
    at.swap(out);
    run.assign(at.empty() ? 0 : 1, 0);
    for (size_t i = 1; i < at.size(); ++i)
      if (at[i].first < at[i - 1].second) return false;
    return true;
  }
  // of a sorted one: whether any range of `r` shares a byte with it
  bool meets(const Ranges& r) const {
    for (size_t i = 0; i < r.run.size(); ++i) {
      const size_t end = i + 1 < r.run.size() ? r.run[i + 1] : r.at.size();
      auto w = std::upper_bound(at.begin(), at.end(), r.at[r.run[i]].first,
                                [](const char* x, const Range& y) { return x < y.second; });   // the first to end behind it
      if (w == at.end() || w->first >= r.at[end - 1].second) continue;
      for (size_t j = r.run[i]; j < end; ++j) {
        while (w != at.end() && w->second <= r.at[j].first) ++w;
        if (w == at.end()) break;
        if (w->first < r.at[j].second) return true;
      }
    }
    return false;
  }
};

// the addresses of an optimizer step; ms[i] and vs[i] NULL where the moments have no scales
struct StepLists {
  Py_ssize_t n;
  float* const* p;
  const float* const* g;
  void* const* m;
  void* const* v;
  float* const* ms;
  float* const* vs;
  const long long* numel;
  long long bytes(Py_ssize_t i) const { return (ms[i] ? 1 : 4) * numel[i]; }
  long long scale_bytes(Py_ssize_t i) const { return (numel[i] + kBlock - 1) / kBlock * 4; }
};

// whether a look at runs shows that no tensors of a step meet
bool plainly_apart(const StepLists& l) {
  Runs read, written;
  for (Py_ssize_t i = 0; i < l.n; ++i)
    if (!read.add(l.g[i], 4 * l.numel[i])) return false;
  for (Py_ssize_t i = 0; i < l.n; ++i)
    if (!written.add(l.p[i], 4 * l.numel[i])) return false;
  for (const auto x : {l.m, l.v})
    for (Py_ssize_t i = 0; i < l.n; ++i)
      if (!written.add(x[i], l.bytes(i))) return false;
  for (const auto x : {l.ms, l.vs})
    for (Py_ssize_t i = 0; i < l.n; ++i)
      if (x[i] && !written.add(x[i], l.scale_bytes(i))) return false;
  return !written.meet(read);
}

// What a step writes would otherwise be written, or read as a gradient, by two workgroups at once.  NULL, or what is wrong.
const char* shared_memory(const StepLists& l) {
  if (plainly_apart(l)) return nullptr;
  Ranges writes, reads;
  writes.at.reserve(5 * l.n);
  for (Py_ssize_t i = 0; i < l.n; ++i) writes.add(l.p[i], 4 * l.numel[i]);
  for (const auto x : {l.m, l.v})
    for (Py_ssize_t i = 0; i < l.n; ++i) writes.add(x[i], l.bytes(i));
  for (const auto x : {l.ms, l.vs})
    for (Py_ssize_t i = 0; i < l.n; ++i)
      if (x[i]) writes.add(x[i], l.scale_bytes(i));
  reads.at.reserve(l.n);
  for (Py_ssize_t i = 0; i < l.n; ++i) reads.add(l.g[i], 4 * l.numel[i]);
  if (!writes.sort()) return "two parameters, moments or scales share memory";
  if (writes.meets(reads)) return "a gradient shares memory with what the step writes";
  return nullptr;
}

void check_dense(const at::Tensor& t, const char* what) {
  const c10::TensorImpl* x = t.unsafeGetTensorImpl();
  if (!x->is_cuda() || x->dtype() != caffe2::TypeMeta::fromScalarType(at::kFloat) || !x->is_contiguous())
    runtime_error(std::string("mpnn_amd.optim: ") + what +
                  " must be contiguous fp32 tensors on a ROCm device (the HIP path has no CPU fallback)");
}

at::Tensor sumsq_parts(Py_ssize_t n, const float* const* p, const long long* numel, const c10::Device& dev) {
  at::Tensor parts = at::empty({kParts}, at::TensorOptions().device(dev).dtype(at::kDouble));
  check_rc(f_parts((int)n, p, numel, parts.data_ptr<double>(), stream_of(dev)), "mpnn_grad_sumsq_parts");
  return parts;
}

// grad_sumsq_parts(grads) -> float64 [256]
at::Tensor sumsq_parts(const Items& grads) {
  std::vector<const float*> p(grads.n);
  std::vector<long long> numel(grads.n);
  c10::Device dev(c10::kCPU);
  for (Py_ssize_t i = 0; i < grads.n; ++i) {
    const at::Tensor& g = tensor(grads.at[i], "optim", "gradients");
    check_dense(g, "gradients");
    if (i == 0) dev = g.device();
    if (g.device() != dev) runtime_error("mpnn_amd.optim: all tensors must be on one device");
    p[i] = g.const_data_ptr<float>();
    numel[i] = g.numel();
  }
  const c10::OptionalDeviceGuard guard(dev);
  return sumsq_parts(grads.n, p.data(), numel.data(), dev);
}

PyObject* py_parts(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    if (n_args != 1) type_error("grad_sumsq_parts: one argument");
    const Items grads(a[0]);
    if (!grads.n) value_error("mpnn_amd.optim: no gradients");
    return THPVariable_Wrap(sumsq_parts(grads));
  });
}

// adamw(params, grads, exp_avgs, exp_avg_sqs, scales, sq_scales, step, lr, beta1, beta2, eps, weight_decay, seed, first,
//       max_norm, parts) -> squared norm (float32 [1]) or None.  parts None with max_norm > 0: the norm of these gradients.
PyObject* py_adamw(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    if (n_args != 16) type_error("adamw: sixteen arguments");
    const Items P(a[0]), G(a[1]), M(a[2]), V(a[3]), A(a[4]), S(a[5]);
    const Py_ssize_t n = P.n;
    if (G.n != n || M.n != n || V.n != n || A.n != n || S.n != n)
      value_error("mpnn_amd.optim.adamw_step: lists of different lengths");
    if (!n) Py_RETURN_NONE;
    const long long step = integer(a[6]);
    if (step < 1 || step >= (1LL << 31)) value_error("mpnn_amd.optim.adamw_step: step counts from 1");
    std::vector<float*> p(n), ms(n), vs(n);
    std::vector<const float*> g(n);
    std::vector<void*> m(n), v(n);
    std::vector<long long> numel(n);
    const c10::Device dev = tensor(P.at[0], "optim", "parameters").device();
    const char* name = "optim.adamw_step";
    const auto fp32 = caffe2::TypeMeta::fromScalarType(at::kFloat), fp8 = caffe2::TypeMeta::fromScalarType(at::kFloat8_e4m3fn);
    for (Py_ssize_t i = 0; i < n; ++i) {
      const at::Tensor &tp = tensor(P.at[i], name, "params"), &tg = tensor(G.at[i], name, "grads"),
                       &tm = tensor(M.at[i], name, "exp_avgs"), &tv = tensor(V.at[i], name, "exp_avg_sqs");
      check_dense(tp, "parameters");
      check_dense(tg, "gradients");
      const c10::TensorImpl *xp = tp.unsafeGetTensorImpl(), *xg = tg.unsafeGetTensorImpl(), *xm = tm.unsafeGetTensorImpl(),
                            *xv = tv.unsafeGetTensorImpl();
      const long long k = xp->numel();
      const bool wide = A.at[i] != Py_None;
      if (wide != (S.at[i] != Py_None))
        value_error("mpnn_amd.optim.adamw_step: both moments of a tensor have scales, or none");
      if (!k) value_error("mpnn_amd.optim.adamw_step: empty tensor");
      if (xg->numel() != k || xm->numel() != k || xv->numel() != k)
        value_error("mpnn_amd.optim.adamw_step: parameter, gradient and moments differ in size");
      const auto want = wide ? fp8 : fp32;
      if (xm->dtype() != want || xv->dtype() != want || !xm->is_contiguous() || !xv->is_contiguous())
        value_error("mpnn_amd.optim.adamw_step: moments must be contiguous fp32 tensors without scales, or float8_e4m3fn with "
                    "scales");
      if (xp->device() != dev || xg->device() != dev || xm->device() != dev || xv->device() != dev)
        runtime_error("mpnn_amd.optim.adamw_step: all tensors must be on one device");
      p[i] = (float*)tp.data_ptr();
      g[i] = (const float*)tg.const_data_ptr();
      m[i] = tm.data_ptr();
      v[i] = tv.data_ptr();
      numel[i] = k;
      ms[i] = vs[i] = nullptr;
      if (wide) {
        const at::Tensor &ta = tensor(A.at[i], name, "exp_avg_scales"), &ts = tensor(S.at[i], name, "exp_avg_sq_scales");
        const long long blocks = (k + kBlock - 1) / kBlock;
        for (const at::Tensor* t : {&ta, &ts}) {
          const c10::TensorImpl* x = t->unsafeGetTensorImpl();
          if (x->dtype() != fp32 || x->numel() != blocks || !x->is_contiguous() || x->device() != dev)
            value_error("mpnn_amd.optim.adamw_step: scales must be contiguous fp32 tensors of one element for each 64 of the "
                        "parameter, on its device");
        }
        ms[i] = (float*)ta.data_ptr();
        vs[i] = (float*)ts.data_ptr();
      }
    }
    if (const char* refusal = shared_memory({n, p.data(), g.data(), m.data(), v.data(), ms.data(), vs.data(), numel.data()}))
      value_error(std::string("mpnn_amd.optim.adamw_step: ") + refusal);
    const double max_norm = number(a[14]);
    const c10::OptionalDeviceGuard guard(dev);
    at::Tensor parts, sumsq;
    if (max_norm > 0) {
      if (a[15] != Py_None) {
        parts = on_gpu(a[15], name, "parts", &dev);
        if (parts.numel() != kParts || parts.scalar_type() != at::kDouble || !parts.is_contiguous())
          value_error("mpnn_amd.optim.adamw_step: parts come from grad_sumsq_parts");
      } else {
        parts = sumsq_parts(n, g.data(), numel.data(), dev);
      }
      sumsq = at::empty({1}, at::TensorOptions().device(dev).dtype(at::kFloat));
    }
    const double lr = number(a[7]), b1 = number(a[8]), b2 = number(a[9]), eps = number(a[10]), decay = number(a[11]);
    check_rc(f_adamw((int)n, p.data(), g.data(), m.data(), v.data(), ms.data(), vs.data(), numel.data(), lr, b1, b2, eps, decay,
                     (int)step, (uint32_t)integer(a[12]), (int)integer(a[13]),
                     parts.defined() ? parts.const_data_ptr<double>() : nullptr, max_norm > 0 ? max_norm : 0.0,
                     sumsq.defined() ? sumsq.data_ptr<float>() : nullptr, stream_of(dev)),
             "mpnn_adamw_mixed");
    for (Py_ssize_t i = 0; i < n; ++i)
      for (const Items* l : {&P, &M, &V, &A, &S})
        if (l->at[i] != Py_None) touched(THPVariable_Unpack(l->at[i]));
    if (sumsq.defined()) return THPVariable_Wrap(sumsq);
    Py_RETURN_NONE;
  });
}

// ---- the library's functions, in the order _lib.py hands them over ----
PyObject* py_bind(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    if (n_args != 6) type_error("bind: six addresses");
    f_select = (decltype(f_select))integer(a[0]);
    f_select_ws = (decltype(f_select_ws))integer(a[1]);
    f_reorder = (decltype(f_reorder))integer(a[2]);
    f_parts = (decltype(f_parts))integer(a[3]);
    f_adamw = (decltype(f_adamw))integer(a[4]);
    f_error = (decltype(f_error))integer(a[5]);
    Py_RETURN_NONE;
  });
}

// layout rules of beam_reorder on any tensor (unit tests without a GPU): (n_mid, stride_mid, run) or None, span or None
PyObject* py_layout(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    if (n_args != 2) type_error("state_layout: two arguments");
    const Layout l = state_layout(tensor(a[0], "state_layout", "state"), PyObject_IsTrue(a[1]) == 1);
    if (!l.regular) Py_RETURN_NONE;
    return Py_BuildValue("(LLL)", l.n_mid, l.stride_mid, l.run);
  });
}
PyObject* py_span(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    if (n_args != 1) type_error("state_span: one argument");
    const long long s = state_span(tensor(a[0], "state_span", "state"));
    if (!s) Py_RETURN_NONE;
    return PyLong_FromLongLong(s);
  });
}

// whether beam_reorder may move the two states in one call: None where one of them is refused by itself
PyObject* py_apart(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    if (n_args != 3) type_error("states_apart: three arguments");
    Span s[2];
    for (int i = 0; i < 2; ++i) {
      const at::Tensor& t = tensor(a[i], "states_apart", "state");
      const Layout l = state_layout(t, PyObject_IsTrue(a[2]) == 1);
      const long long extent = state_span(t);
      if (!l.regular || !extent || !t.numel()) Py_RETURN_NONE;
      s[i] = state_rows(t, l, extent);
    }
    const Span &x = s[0].begin <= s[1].begin ? s[0] : s[1], &y = s[0].begin <= s[1].begin ? s[1] : s[0];
    return PyBool_FromLong(y.begin >= x.end || apart(x, y));
  });
}

// shared_memory of tensors on any device (unit tests without a GPU): params, grads, exp_avgs, exp_avg_sqs, scales, sq_scales
PyObject* py_share(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    if (n_args != 6) type_error("shared_memory: six arguments");
    std::vector<void*> at[6];
    std::vector<long long> numel;
    for (int k = 0; k < 6; ++k) {
      const Items l(a[k]);
      if (k && (size_t)l.n != at[0].size()) value_error("shared_memory: lists of different lengths");
      for (Py_ssize_t i = 0; i < l.n; ++i) {
        const at::Tensor* t = l.at[i] == Py_None ? nullptr : &tensor(l.at[i], "shared_memory", "tensors");
        at[k].push_back(t ? t->data_ptr() : nullptr);
        if (k == 0) numel.push_back(t->numel());
      }
    }
    const char* refusal = shared_memory({(Py_ssize_t)numel.size(), (float**)at[0].data(), (const float**)at[1].data(), at[2].data(),
                                         at[3].data(), (float**)at[4].data(), (float**)at[5].data(), numel.data()});
    if (!refusal) Py_RETURN_NONE;
    return PyUnicode_FromString(refusal);
  });
}

PyMethodDef methods[] = {
    {"bind", (PyCFunction)(void (*)(void))py_bind, METH_FASTCALL, "addresses of the HIP library's functions"},
    {"beam_select", (PyCFunction)(void (*)(void))py_select, METH_FASTCALL, "mpnn_amd.beam_select, arguments in order"},
    {"beam_reorder", (PyCFunction)(void (*)(void))py_reorder, METH_FASTCALL, "mpnn_amd.beam_reorder, arguments in order"},
    {"grad_sumsq_parts", (PyCFunction)(void (*)(void))py_parts, METH_FASTCALL, "partial sums of squares over gradients"},
    {"adamw", (PyCFunction)(void (*)(void))py_adamw, METH_FASTCALL, "mpnn_amd.optim.adamw_step, arguments in order"},
    {"state_layout", (PyCFunction)(void (*)(void))py_layout, METH_FASTCALL, "layout of a state behind its beams"},
    {"shared_memory", (PyCFunction)(void (*)(void))py_share, METH_FASTCALL, "why an optimizer step over these tensors is refused"},
    {"states_apart", (PyCFunction)(void (*)(void))py_apart, METH_FASTCALL, "whether two states share no byte"},
    {"state_span", (PyCFunction)(void (*)(void))py_span, METH_FASTCALL, "elements a state spans"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", "host side of mpnn_amd's many-tensor entry points", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&module); }
