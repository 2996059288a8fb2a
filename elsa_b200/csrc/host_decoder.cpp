// Native host path of the decoder operators (rotary positions, shared-prefix and differential attention): what host.cpp does for the
// attention operators.  Their smallest calls are one or two launches of a few microseconds; through Python and ctypes a call takes
// 25 to 35 us of host time, and a training step with a Python autograd.Function over 150; here 6 to 10, and about 80.
//
// A call that is not plain (see host_common.h), or whose arguments would be refused, gives None: the Python operator takes its
// general path, which also raises the errors.
#include "host_common.h"

#include <cmath>
#include <cstring>

#include <torch/csrc/autograd/functions/basic_ops.h>

namespace elsa_host {

decltype(&elsa_strerror) f_strerror = nullptr;
decltype(&elsa_last_cuda_error) f_last_cuda_error = nullptr;

namespace {

using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

decltype(&elsa_rotary) f_rotary = nullptr;
decltype(&elsa_shared_prefix_workspace_bytes) f_prefix_ws = nullptr;
decltype(&elsa_shared_prefix_attention) f_prefix = nullptr;
decltype(&elsa_differential_workspace_bytes_for) f_diff_ws = nullptr;
decltype(&elsa_differential_forward) f_diff = nullptr;
decltype(&elsa_differential_backward_workspace_bytes) f_diff_bwd_ws = nullptr;
decltype(&elsa_differential_backward) f_diff_bwd = nullptr;

constexpr int64_t kMostSize = (1 << 30) - 1;        // of any axis

// element strides of all axes but the last into `st` (0 for an axis of one); false where the rows are not contiguous or an axis is too long
bool row_strides(const at::Tensor& t, int64_t* st) {
  const auto sz = t.sizes();
  const auto s = t.strides();
  const int64_t dim = t.dim();
  if (sz[dim - 1] > 1 && s[dim - 1] != 1) return false;
  for (int64_t i = 0; i < dim; ++i)
    if (sz[i] > kMostSize) return false;
  for (int64_t i = 0; i + 1 < dim; ++i) st[i] = sz[i] > 1 ? s[i] : 0;
  return true;
}

// an uninitialised [b, h, n, d] tensor in the axis order in memory of a view with these strides
at::Tensor new_like(const at::Tensor& like, const int64_t* st, int64_t b, int64_t h, int64_t n, int64_t d) {
  return st[1] && st[2] && st[1] < st[2] ? new_bnhd(like, b, h, n, d) : new_tensor({b, h, n, d}, like, like.scalar_type());
}

void* stream_of(c10::Device dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }

int64_t bits_of(double x) {
  int64_t i;
  std::memcpy(&i, &x, sizeof i);
  return i;
}
double of_bits(int64_t i) {
  double x;
  std::memcpy(&x, &i, sizeof x);
  return x;
}

// ---- autograd ---------------------------------------------------------------------------------------------------------
enum Kind { kRotary = 0, kDifferential = 1 };
variable_list gradients(const std::vector<int64_t>& numbers, const std::vector<at::Tensor>& saved, const variable_list& grads);

// One node for both operators: its numbers (the first is the kind) and saved tensors say what the backward needs.
struct DecoderBackward : public torch::autograd::Node {
  std::vector<int64_t> numbers;
  std::vector<SavedVariable> saved;
  int out_at = -1;                                  // which saved tensor is the node's own output

  std::string name() const override { return numbers[0] == kRotary ? "RotaryEmbeddingBackward" : "DifferentialAttentionBackward"; }

  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable& s : saved) s.reset_data();
  }

  std::vector<at::Tensor> unpack() {
    std::vector<at::Tensor> t;
    for (size_t i = 0; i < saved.size(); ++i) t.push_back(static_cast<int>(i) == out_at ? saved[i].unpack(shared_from_this()) : saved[i].unpack());
    return t;
  }

  static bool none(const variable_list& grads) {
    for (const at::Tensor& g : grads)
      if (g.defined()) return false;
    return true;
  }
  // (q alone, or q and k: as many as were turned)
  static size_t inputs(const std::vector<int64_t>& numbers, const variable_list& grads) { return numbers[0] == kRotary ? grads.size() : 4; }

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    if (none(grads)) return variable_list(inputs(numbers, grads));
    const std::vector<at::Tensor> t = unpack();     // (runs the user's hooks, with autograd in force)
    variable_list result;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      result = gradients(numbers, t, grads);
    }
    if (at::GradMode::is_enabled()) {
      // create_graph: the gradients have none of their own, and say so when one is asked for
      auto error = std::make_shared<torch::autograd::Error>(name() + " is not differentiable twice", torch::autograd::edge_list());
      for (at::Tensor& r : result)
        if (r.defined()) torch::autograd::set_history(r, error);
    }
    return result;
  }

  // Compiled autograd: the node is one opaque call of its graph, on the saved tensors and the numbers.
  void compiled_args(torch::dynamo::autograd::CompiledNodeArgs& args) const override {
    args.collect(numbers);
    for (size_t i = 0; i < saved.size(); ++i) args.collect(saved[i], static_cast<int>(i) == out_at);
  }

  variable_list apply_with_saved(const variable_list& grads, torch::dynamo::autograd::SwapSavedVariables& swap) override {
    for (SavedVariable& s : saved) swap.before(s);
    const std::vector<at::Tensor> t = unpack();
    torch::dynamo::autograd::PackedArgs packed;
    std::vector<at::TypePtr> schema;
    auto add = [&](const auto& x) {
      packed.pack(x);
      schema.emplace_back(torch::dynamo::autograd::IValuePacker<std::decay_t<decltype(x)>>::packed_type());
    };
    add(numbers);
    for (const at::Tensor& x : t) add(x);
    const auto& compiler = torch::dynamo::autograd::getPyCompilerInterface();
    const std::string fn = compiler->bind_function(swap.get_py_compiler(), name(), numbers[0] == kRotary ? &call_packed<2> : &call_packed<7>, schema,
                                                   /*is_custom_function=*/true, /*is_traceable=*/false);
    variable_list result = compiler->call_function(
        swap.get_py_compiler(), "apply_functional", fn, grads, packed.vec(),
        torch::dynamo::autograd::IValuePacker<std::vector<std::optional<torch::autograd::InputMetadata>>>::pack(
            torch::dynamo::autograd::get_input_metadata(next_edges())));
    for (SavedVariable& s : saved) swap.after(s);
    return result;
  }

  template <int N>
  static variable_list call_packed(const variable_list& grads, const std::vector<c10::IValue>& values) {
    torch::dynamo::autograd::PackedArgs packed(values);
    const auto numbers = packed.unpack<std::vector<int64_t>>();
    std::vector<at::Tensor> t(N);
    for (at::Tensor& x : t) x = packed.unpack<at::Tensor>();
    if (none(grads)) return variable_list(inputs(numbers, grads));
    at::AutoDispatchBelowADInplaceOrView below;
    return gradients(numbers, t, grads);
  }
};

template <typename... V>
std::shared_ptr<DecoderBackward> new_node(std::vector<int64_t> numbers, const V&... inputs) {
  std::shared_ptr<DecoderBackward> node(new DecoderBackward(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(inputs...));
  node->numbers = std::move(numbers);
  return node;
}

// ---- rotary positions -------------------------------------------------------------------------------------------------
struct Positions {
  const void* p = nullptr;
  int bytes = 0;
  int64_t sb = 0, sn = 0;
};
Positions positions_of(const at::Tensor& t) {
  Positions p;
  if (!t.defined()) return p;
  p.p = t.const_data_ptr();
  p.bytes = static_cast<int>(t.element_size());
  p.sb = t.dim() == 2 && t.size(0) > 1 ? t.stride(0) : 0;
  p.sn = t.stride(t.dim() - 1);
  return p;
}

// x (one or two of q and k, [B, H, N, D], some element in each) turned into new tensors
void turn(const at::Tensor* x, at::Tensor* y, int count, const at::Tensor& frequencies, const at::Tensor& positions, double magnitude, bool interleaved,
          bool inverse) {
  int64_t st[2][6];
  for (int i = 0; i < count; ++i) {
    const at::Tensor& t = x[i];
    row_strides(t, st[i]);
    y[i] = new_like(t, st[i], t.size(0), t.size(1), t.size(2), t.size(3));
    row_strides(y[i], st[i] + 3);
  }
  const at::Tensor& q = x[0];
  const Positions p = positions_of(positions);
  c10::cuda::CUDAGuard guard(q.device());
  check_status(f_rotary(data_of(q), data_of(y[0]), st[0], static_cast<int>(q.size(1)), count > 1 ? data_of(x[1]) : nullptr,
                        count > 1 ? data_of(y[1]) : nullptr, count > 1 ? st[1] : nullptr, count > 1 ? static_cast<int>(x[1].size(1)) : 0,
                        frequencies.const_data_ptr<double>(), p.p, p.bytes, p.sb, p.sn, magnitude, dtype_code(q.scalar_type()),
                        static_cast<int>(q.size(0)), static_cast<int>(q.size(2)), static_cast<int>(q.size(3)),
                        static_cast<int>(2 * frequencies.size(0)), interleaved, inverse, stream_of(q.device())),
               "elsa_rotary");
}

// numbers: kind, interleaved, magnitude, frequencies, the type of the positions and their sizes; saved: frequencies, positions (undefined: none)
variable_list rotary_gradients(const std::vector<int64_t>& numbers, const std::vector<at::Tensor>& saved, const variable_list& grads) {
  variable_list result(grads.size());
  at::Tensor x[2], y[2];
  int at[2], count = 0;
  for (int i = 0; i < static_cast<int>(grads.size()); ++i) {
    if (!grads[i].defined()) continue;
    int64_t st[3];
    x[count] = row_strides(grads[i], st) ? grads[i] : grads[i].contiguous();
    at[count++] = i;
  }
  const c10::Device dev = x[0].device();
  check_unpacked(saved[0], {numbers[3]}, at::kDouble, dev);
  const at::Tensor frequencies = saved[0].contiguous();
  if (numbers.size() > 5) check_unpacked(saved[1], at::IntArrayRef(numbers).slice(5), static_cast<at::ScalarType>(numbers[4]), dev);
  turn(x, y, count, frequencies, saved[1], of_bits(numbers[2]), numbers[1] != 0, true);
  for (int i = 0; i < count; ++i) result[at[i]] = y[i];
  return result;
}

bool rotary_covers(const at::Tensor& q, const at::Tensor& k, const at::Tensor& f, const at::Tensor& pos) {
  int64_t st[3];
  auto operand = [&](const at::Tensor& t) { return plain(t) && t.dim() == 4 && t.numel() > 0 && row_strides(t, st); };
  if (!operand(q) || dtype_code(q.scalar_type()) < 0 || q.size(1) > 1024 || q.size(3) > 1024) return false;
  if (k.defined() && (!operand(k) || k.scalar_type() != q.scalar_type() || k.device() != q.device() || k.size(0) != q.size(0) ||
                      k.size(2) != q.size(2) || k.size(3) != q.size(3) || k.size(1) > 1024))
    return false;
  if (!plain(f) || f.dim() != 1 || f.scalar_type() != at::kDouble || f.device() != q.device() || !f.is_contiguous() || f.requires_grad() || f.size(0) < 1 ||
      2 * f.size(0) > std::min<int64_t>(q.size(3), 256))
    return false;
  if (pos.defined()) {
    if (!plain(pos) || (pos.scalar_type() != at::kInt && pos.scalar_type() != at::kLong) || pos.device() != q.device() || pos.dim() < 1 ||
        pos.dim() > 2 || pos.size(pos.dim() - 1) != q.size(2) || (pos.dim() == 2 && pos.size(0) != 1 && pos.size(0) != q.size(0)))
      return false;
  }
  return !modes_active();
}

// ---- differential attention -------------------------------------------------------------------------------------------
struct Diff {                 // the problem, as the C ABI wants it
  int batch, heads, kv_heads, nq, nk, d, dv, dt, causal;
  double scale;
};

struct Lam {
  const void* p;
  int dtype, stride;
};
Lam lam_of(const at::Tensor& t) {
  return {t.const_data_ptr(), dtype_code(t.scalar_type()), t.dim() == 1 && t.size(0) > 1 ? static_cast<int>(t.stride(0)) : 0};
}

bool diff_covers(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& lam, Diff* c) {
  int64_t st[3];
  for (const at::Tensor* t : {&q, &k, &v})
    if (!plain(*t) || t->dim() != 4 || t->numel() == 0 || t->scalar_type() != q.scalar_type() || t->device() != q.device() || !row_strides(*t, st)) return false;
  c->dt = dtype_code(q.scalar_type());
  if (c->dt < 0 || q.size(1) % 2 || k.size(1) % 2 || q.size(1) > 65535 || q.size(0) > 65535) return false;
  c->batch = static_cast<int>(q.size(0)); c->heads = static_cast<int>(q.size(1) / 2); c->kv_heads = static_cast<int>(k.size(1) / 2);
  c->nq = static_cast<int>(q.size(2)); c->nk = static_cast<int>(k.size(2)); c->d = static_cast<int>(q.size(3)); c->dv = static_cast<int>(v.size(3));
  if (k.size(0) != c->batch || v.size(0) != c->batch || k.size(3) != c->d || v.size(1) != c->kv_heads || v.size(2) != c->nk ||
      c->kv_heads == 0 || c->heads % c->kv_heads || c->d > 128 || c->dv > 128)
    return false;
  if (!plain(lam) || dtype_code(lam.scalar_type()) < 0 || lam.device() != q.device() || lam.dim() > 1 ||
      (lam.dim() == 1 && lam.size(0) != 1 && lam.size(0) != c->heads) || (lam.dim() == 1 && lam.size(0) > 1 && (lam.stride(0) < 1 || lam.stride(0) > kMostSize)))
    return false;
  if (c->scale == 0.0) c->scale = 1.0 / std::sqrt(static_cast<double>(c->d));      // (the default)
  return !modes_active();
}

bool lengths_cover(const at::Tensor& t, const at::Tensor& q) {
  return !t.defined() || (plain(t) && t.scalar_type() == at::kInt && t.device() == q.device() && t.dim() == 1 && t.size(0) == q.size(0) && t.is_contiguous());
}

// Rows on 16-byte boundaries, in place or copied; other head dims as they are (copied where rows are not contiguous).
at::Tensor for_tiles(const at::Tensor& t) {
  View v;
  int64_t st[3];
  if (t.size(3) % 8 == 0) return in_place_view(t, &v) ? t : aligned(t);
  return row_strides(t, st) ? t : t.contiguous();
}

at::Tensor diff_forward(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& lam, const at::Tensor& lengths, const Diff& c,
                        const at::Tensor& out2, const at::Tensor& lse) {
  int64_t st[12];
  row_strides(q, st);
  row_strides(k, st + 3);
  row_strides(v, st + 6);
  at::Tensor out = new_like(q, st, c.batch, c.heads, c.nq, c.dv);
  row_strides(out, st + 9);
  c10::cuda::CUDAGuard guard(q.device());
  const int* n = lengths.defined() ? lengths.const_data_ptr<int>() : nullptr;
  const int64_t bytes = f_diff_ws(data_of(q), data_of(k), data_of(v), n, data_of(out), st, c.dt, c.batch, c.heads, c.kv_heads, c.nq, c.nk, c.d, c.dv);
  TORCH_CHECK_VALUE(bytes >= 0, "elsa_b200: unsupported problem size for differential_attention");
  c10::DataPtr ws;                                      // (the tiles need none)
  if (bytes > 0) ws = workspace(bytes);
  const Lam l = lam_of(lam);
  check_status(f_diff(data_of(q), data_of(k), data_of(v), l.p, l.dtype, l.stride, n, data_of(out), st, out2.defined() ? data_of(out2) : nullptr,
                      lse.defined() ? lse.mutable_data_ptr<float>() : nullptr, ws.get(), bytes, c.dt, c.batch, c.heads, c.kv_heads, c.nq, c.nk, c.d, c.dv,
                      c.causal, c.scale, stream_of(q.device())),
               "elsa_differential_forward");
  return out;
}

// numbers: kind, batch, heads, kv_heads, nq, nk, d, dv, dtype code, causal, scale, gradient of lam?, lam's type and sizes; saved: q, k, v, lam, out, out2, lse
variable_list diff_gradients(const std::vector<int64_t>& numbers, const std::vector<at::Tensor>& saved, const variable_list& grads) {
  Diff c{};
  int* fields[] = {&c.batch, &c.heads, &c.kv_heads, &c.nq, &c.nk, &c.d, &c.dv, &c.dt, &c.causal};
  for (int i = 0; i < 9; ++i) *fields[i] = static_cast<int>(numbers[1 + i]);
  c.scale = of_bits(numbers[10]);
  const at::ScalarType dtype = c.dt == ELSA_F32 ? at::kFloat : c.dt == ELSA_F16 ? at::kHalf : at::kBFloat16;
  at::Tensor go = grads[0];
  const c10::Device dev = go.device();
  const int64_t B = c.batch, H = c.heads, G = c.kv_heads, N = c.nq, M = c.nk, D = c.d, V = c.dv;
  check_unpacked(saved[0], {B, 2 * H, N, D}, dtype, dev);
  check_unpacked(saved[1], {B, 2 * G, M, D}, dtype, dev);
  check_unpacked(saved[2], {B, G, M, V}, dtype, dev);
  check_unpacked(saved[3], at::IntArrayRef(numbers).slice(13), static_cast<at::ScalarType>(numbers[12]), dev);
  check_unpacked(saved[4], {B, H, N, V}, dtype, dev);
  check_unpacked(saved[5], {B, H, N, V}, dtype, dev);
  check_unpacked(saved[6], {2, B, H, N}, at::kFloat, dev);
  if (go.scalar_type() != dtype) go = go.to(dtype);
  c10::cuda::CUDAGuard guard(dev);
  const at::Tensor q = for_tiles(saved[0]), k = for_tiles(saved[1]), v = for_tiles(saved[2]), lam = saved[3].contiguous(), out = for_tiles(saved[4]);
  const at::Tensor out2 = aligned(saved[5]), lse = aligned(saved[6]);
  go = for_tiles(go);
  variable_list result(4);
  result[0] = new_tensor(q.sizes(), q, dtype);
  result[1] = new_tensor(k.sizes(), k, dtype);
  result[2] = new_tensor(v.sizes(), v, dtype);
  if (numbers[11]) result[3] = new_tensor(lam.sizes(), lam, lam.scalar_type());
  int64_t st[24];
  int i = 0;
  for (const at::Tensor* t : std::initializer_list<const at::Tensor*>{&q, &k, &v, &out, &go, &result[0], &result[1], &result[2]})
    row_strides(*t, st + 3 * i++);
  const int64_t need = f_diff_bwd_ws(c.dt, c.batch, c.heads, c.kv_heads, c.nq, c.nk, c.d, c.dv);
  TORCH_CHECK_VALUE(need >= 0, "elsa_b200: unsupported problem size for differential_attention");
  const int64_t bytes = std::max<int64_t>(need, 256);
  c10::DataPtr ws = workspace(bytes);
  const Lam l = lam_of(lam);
  check_status(f_diff_bwd(data_of(q), data_of(k), data_of(v), l.p, l.dtype, l.stride, data_of(out), data_of(out2), lse.const_data_ptr<float>(), data_of(go),
                          data_of(result[0]), data_of(result[1]), data_of(result[2]), numbers[11] ? data_of(result[3]) : nullptr, st, ws.get(), bytes, c.dt,
                          c.batch, c.heads, c.kv_heads, c.nq, c.nk, c.d, c.dv, c.causal, c.scale, stream_of(dev)),
               "elsa_differential_backward");
  return result;
}

variable_list gradients(const std::vector<int64_t>& numbers, const std::vector<at::Tensor>& saved, const variable_list& grads) {
  return numbers[0] == kRotary ? rotary_gradients(numbers, saved, grads) : diff_gradients(numbers, saved, grads);
}

bool get_double(PyObject* o, double* x) {
  *x = PyFloat_AsDouble(o);
  return !(*x == -1.0 && PyErr_Occurred());
}
constexpr double kDefaultScale = 0.0;               // what None stands for; 0 itself is refused, like every number that is not positive and finite in fp32
bool get_scale(PyObject* o, double* x, bool* refused) {
  *refused = false;
  *x = kDefaultScale;
  if (o == Py_None) return true;
  if (!get_double(o, x)) return false;
  *refused = !(*x >= 0x1p-126 && *x <= 0x1p127);
  return true;
}

}  // namespace

// rotary(q, k, frequencies, positions, interleaved, magnitude)
PyObject* py_rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 6, "rotary takes 6 arguments");
  at::Tensor x[2], y[2], f, pos;
  double magnitude;
  const int interleaved = PyObject_IsTrue(a[4]);
  if (interleaved < 0 || !get_double(a[5], &magnitude)) return nullptr;
  if (!get_tensor(a[0], &x[0]) || !get_tensor(a[1], &x[1]) || !get_tensor(a[2], &f) || !get_tensor(a[3], &pos) || !x[0].defined() || !f.defined()) Py_RETURN_NONE;
  const int count = x[1].defined() ? 2 : 1;
  {
    NoGil no_gil;
    if (rotary_covers(x[0], x[1], f, pos)) {
      const bool record = at::GradMode::is_enabled() && (x[0].requires_grad() || (count > 1 && x[1].requires_grad()));
      {
        at::AutoDispatchBelowADInplaceOrView below;
        turn(x, y, count, f, pos, magnitude, interleaved != 0, false);
      }
      if (record) {
        std::vector<int64_t> numbers{kRotary, interleaved, bits_of(magnitude), f.size(0), pos.defined() ? static_cast<int64_t>(pos.scalar_type()) : 0};
        if (pos.defined()) numbers.insert(numbers.end(), pos.sizes().begin(), pos.sizes().end());
        auto node = count > 1 ? new_node(std::move(numbers), x[0], x[1]) : new_node(std::move(numbers), x[0]);
        node->saved.emplace_back(f, false);
        node->saved.emplace_back(pos, false);
        for (int i = 0; i < count; ++i) torch::autograd::set_history(y[i], node);
      }
    }
  }
  if (!y[0].defined()) Py_RETURN_NONE;
  if (count == 1) return THPVariable_Wrap(std::move(y[0]));
  PyObject* pair = PyTuple_New(2);
  if (!pair) return nullptr;
  for (int i = 0; i < 2; ++i) PyTuple_SET_ITEM(pair, i, THPVariable_Wrap(std::move(y[i])));
  return pair;
  END_HANDLE_TH_ERRORS
}

// shared_prefix(q, k_prefix, v_prefix, k, v, lengths, scale)
PyObject* py_shared_prefix(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 7, "shared_prefix takes 7 arguments");
  at::Tensor t[5], lengths, out;
  double scale;
  for (int i = 0; i < 5; ++i)
    if (!get_tensor(a[i], &t[i]) || !t[i].defined()) Py_RETURN_NONE;
  if (!get_tensor(a[5], &lengths)) Py_RETURN_NONE;
  bool refused;
  if (!get_scale(a[6], &scale, &refused)) return nullptr;
  if (refused) Py_RETURN_NONE;
  {
    NoGil no_gil;
    const at::Tensor &q = t[0], &kp = t[1], &vp = t[2], &k = t[3], &v = t[4];
    int64_t st[16];
    bool covered = !modes_active();
    for (int i = 0; covered && i < 5; ++i)
      covered = plain(t[i]) && t[i].dim() == (i == 1 || i == 2 ? 3 : 4) && t[i].scalar_type() == q.scalar_type() && t[i].device() == q.device();
    covered = covered && q.numel() > 0 && dtype_code(q.scalar_type()) >= 0 && k.sizes() == v.sizes() && kp.sizes() == vp.sizes() && k.size(0) == q.size(0) &&
              k.size(3) == q.size(3) && kp.size(0) == k.size(1) && kp.size(2) == q.size(3) && k.size(1) > 0 && q.size(1) % k.size(1) == 0 && q.size(3) <= 128 &&
              q.size(0) <= 0x7fffffff && lengths_cover(lengths, q) && row_strides(q, st) && row_strides(kp, st + 3) && row_strides(vp, st + 5) &&
              row_strides(k, st + 7) && row_strides(v, st + 10);
    if (covered) {
      if (scale == kDefaultScale) scale = 1.0 / std::sqrt(static_cast<double>(q.size(3)));
      at::AutoDispatchBelowADInplaceOrView below;
      const int batch = static_cast<int>(q.size(0)), heads = static_cast<int>(q.size(1)), kv_heads = static_cast<int>(k.size(1)), nq = static_cast<int>(q.size(2));
      const int d = static_cast<int>(q.size(3)), np = static_cast<int>(kp.size(1)), no = static_cast<int>(k.size(2)), dt = dtype_code(q.scalar_type());
      c10::cuda::CUDAGuard guard(q.device());
      const int64_t need = f_prefix_ws(dt, batch, heads, kv_heads, nq, d, np, no);
      if (need >= 0) {
        out = new_like(q, st, batch, heads, nq, d);
        row_strides(out, st + 13);
        const int64_t bytes = std::max<int64_t>(need, 256);
        c10::DataPtr ws = workspace(bytes);
        check_status(f_prefix(data_of(q), data_of(kp), data_of(vp), data_of(k), data_of(v), data_of(out), st,
                              lengths.defined() ? lengths.const_data_ptr<int>() : nullptr, ws.get(), bytes, dt, batch, heads, kv_heads, nq, d, np, no, scale,
                              stream_of(q.device())),
                     "elsa_shared_prefix_attention");
      }
    }
  }
  if (!out.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// differential(q, k, v, lam, causal, scale, lengths, train)
PyObject* py_differential(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 8, "differential takes 8 arguments");
  at::Tensor q, k, v, lam, lengths, out;
  Diff c{};
  const int causal = PyObject_IsTrue(a[4]);
  bool refused;
  if (causal < 0 || !get_scale(a[5], &c.scale, &refused)) return nullptr;
  if (refused) Py_RETURN_NONE;
  c.causal = causal;
  if (!get_tensor(a[0], &q) || !get_tensor(a[1], &k) || !get_tensor(a[2], &v) || !get_tensor(a[3], &lam) || !get_tensor(a[6], &lengths) || !q.defined() ||
      !k.defined() || !v.defined() || !lam.defined())
    Py_RETURN_NONE;
  {
    NoGil no_gil;
    if (diff_covers(q, k, v, lam, &c) && lengths_cover(lengths, q)) {
      const bool record = a[7] == Py_True && at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad() || lam.requires_grad());
      at::Tensor qs = q, ks = k, vs = v, out2, lse;
      {
        at::AutoDispatchBelowADInplaceOrView below;
        if (record) {
          qs = for_tiles(q); ks = for_tiles(k); vs = for_tiles(v);
          out2 = new_tensor({c.batch, c.heads, c.nq, c.dv}, q, q.scalar_type());
          lse = new_tensor({2, c.batch, c.heads, c.nq}, q, at::kFloat);
        }
        out = diff_forward(qs, ks, vs, lam, lengths, c, out2, lse);
      }
      if (record) {
        std::vector<int64_t> numbers{kDifferential, c.batch, c.heads, c.kv_heads, c.nq, c.nk, c.d, c.dv, c.dt, c.causal, bits_of(c.scale), lam.requires_grad(),
                                     static_cast<int64_t>(lam.scalar_type())};
        numbers.insert(numbers.end(), lam.sizes().begin(), lam.sizes().end());
        auto node = new_node(std::move(numbers), q, k, v, lam);
        for (const at::Tensor* t : std::initializer_list<const at::Tensor*>{&qs, &ks, &vs, &lam}) node->saved.emplace_back(*t, false);
        torch::autograd::set_history(out, node);
        node->saved.emplace_back(out, true);
        node->out_at = 4;
        node->saved.emplace_back(out2, false);
        node->saved.emplace_back(lse, false);
      }
    }
  }
  if (!out.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

void bind_decoder(const std::function<void*(const char*)>& at_name) {
  f_rotary = reinterpret_cast<decltype(f_rotary)>(at_name("elsa_rotary"));
  f_prefix_ws = reinterpret_cast<decltype(f_prefix_ws)>(at_name("elsa_shared_prefix_workspace_bytes"));
  f_prefix = reinterpret_cast<decltype(f_prefix)>(at_name("elsa_shared_prefix_attention"));
  f_diff_ws = reinterpret_cast<decltype(f_diff_ws)>(at_name("elsa_differential_workspace_bytes_for"));
  f_diff = reinterpret_cast<decltype(f_diff)>(at_name("elsa_differential_forward"));
  f_diff_bwd_ws = reinterpret_cast<decltype(f_diff_bwd_ws)>(at_name("elsa_differential_backward_workspace_bytes"));
  f_diff_bwd = reinterpret_cast<decltype(f_diff_bwd)>(at_name("elsa_differential_backward"));
}

}  // namespace elsa_host
