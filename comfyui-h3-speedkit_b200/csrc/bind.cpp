// PyTorch binding of the operators that are called once per token: argument checks,
// outputs, workspace, stream and launch in one call of a few microseconds (a chain
// of Python checks and ctypes took 26 to 43 us on the host, more than the kernels of
// short inputs).  The work itself is libh3sk_b200.so's C entry points.
//
// A broken contract raises ValueError before anything is allocated or launched (operands as
// the other operators take them: plain tensors without a gradient); a CUDA error code raises
// RuntimeError.  Every operand is recorded on the current
// stream of its device, and the caller's own outputs count as modified.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstring>
#include <optional>
#include <string>
#include <utility>
#include <vector>

#include "../../include/h3sk_b200.h"

namespace py = pybind11;
using at::Tensor;
using Maybe = std::optional<Tensor>;

namespace {

[[noreturn]] void refuse(const std::string& text) { throw py::value_error(text); }
void need(bool ok, const char* text) {
  if (!ok) refuse(text);
}

struct Named {
  const char* name;
  const Tensor* t;
};
using List = std::vector<Named>;

void add(List& list, const char* name, const Tensor& t) { list.push_back({name, &t}); }
void add(List& list, const char* name, const Maybe& t) {
  if (t) list.push_back({name, &*t});
}

const void* ptr(const Tensor& t) { return t.data_ptr(); }
const void* ptr(const Maybe& t) { return t ? t->data_ptr() : nullptr; }
void* out_ptr(const Tensor& t) { return t.data_ptr(); }
const int* ints(const Maybe& t) { return static_cast<const int*>(ptr(t)); }

bool aligned(const Tensor& t, uintptr_t n) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & (n - 1)) == 0; }

// BF16 0, FP16 1, else -1
int type_of(const Tensor& t) {
  return t.scalar_type() == at::kBFloat16 ? 0 : t.scalar_type() == at::kHalf ? 1 : -1;
}

bool normal_positive(double x) {
  const float f = static_cast<float>(x);
  return std::isfinite(x) && std::isfinite(f) && f >= FLT_MIN;
}

// Tensors whose memory is their value: torch.Tensor itself, not a subclass (a Parameter, a
// wrapper), nothing that is negated or conjugated on reading, or zero without memory.
void original(const Maybe& t) {
  if (!t) return;
  const py::object object = py::reinterpret_steal<py::object>(THPVariable_Wrap(*t));
  need(reinterpret_cast<PyObject*>(Py_TYPE(object.ptr())) == THPVariableClass && !t->is_neg() && !t->is_conj() &&
           !t->_is_zerotensor() && t->layout() == at::kStrided,
       "All operands must be original plain Torch tensors");
}
template <typename... Operands>
void originals(const Operands&... operands) {
  (original(operands), ...);
}

// One device, nothing that carries a gradient: recorded, to be recorded, or a forward-mode
// tangent.  The device itself is checked last, so that the other rules hold on a host
// without a GPU too.
void plain(const List& operands) {
  const auto device = operands[0].t->device();
  for (const Named& o : operands) {
    if (o.t->device() != device) refuse("All operands must use one CUDA device");
    if (o.t->requires_grad() || o.t->_fw_grad(0).defined())
      refuse("Inference only; detach only after validating model autograd policy");
  }
}

// [first byte, one past the last byte] that a strided tensor can reach.
std::pair<const char*, const char*> span(const Tensor& t) {
  const char* p = static_cast<const char*>(t.data_ptr());
  if (t.numel() == 0) return {p, p};
  int64_t reach = 1;
  for (int64_t i = 0; i < t.dim(); ++i) reach += (t.size(i) - 1) * t.stride(i);
  return {p, p + reach * t.element_size()};
}
bool overlap(const Tensor& a, const Tensor& b) {
  const auto x = span(a), y = span(b);
  return x.first < x.second && y.first < y.second && x.first < y.second && y.first < x.second;
}

// No two indices reach one address: each stride clears the extent of the smaller ones.
bool no_self_overlap(const Tensor& t) {
  if (t.is_contiguous()) return true;
  std::vector<std::pair<int64_t, int64_t>> d;
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.size(i) > 1) d.push_back({t.stride(i), t.size(i)});
  std::sort(d.begin(), d.end());
  int64_t reach = 0;
  for (const auto& [stride, size] : d) {
    if (stride <= reach) return false;
    reach += stride * (size - 1);
  }
  return true;
}

void check_device(const Tensor& t) {
  need(t.is_cuda(), "All operands must use one CUDA device");
  const auto* p = at::cuda::getDeviceProperties(t.device().index());
  if (p->major != 10 || p->minor != 0) throw std::runtime_error("Only the intended B200 (sm_100) device is supported");
}

// Enqueue on the current stream of the operands' device.
template <typename Go>
void enqueue(const List& operands, const List& written, const char* what, const char* (*error)(int), Go&& go) {
  const auto device = operands[0].t->device();
  const c10::cuda::OptionalCUDAGuard guard(device);
  const auto stream = c10::cuda::getCurrentCUDAStream(device.index());
  for (const Named& o : operands) {
    if (o.t->numel()) c10::cuda::CUDACachingAllocator::recordStream(o.t->storage().data_ptr(), stream);
  }
  const int code = go(reinterpret_cast<uintptr_t>(stream.stream()));
  for (const Named& o : written)
    if (!o.t->is_inference()) o.t->unsafeGetTensorImpl()->bump_version();
  if (code) throw std::runtime_error(std::string(what) + ": CUDA error " + std::to_string(code) + ": " + error(code));
}

// ---- residual RMS norm to 8 bits -------------------------------------------------------

constexpr int64_t kMaxWidth = 16384;

bool rows_ok(const Tensor& t, int64_t m, int64_t k, at::ScalarType type) {
  return t.dim() == 2 && t.size(0) == m && t.size(1) == k && t.scalar_type() == type && (t.stride(1) == 1 || k == 1) &&
         (t.stride(0) >= k || m <= 1);
}

py::tuple rms_quant(const Tensor& x, const Tensor& weight, const Maybe& residual, double eps, int code, const Maybe& residual_out,
                    const Maybe& out, const Maybe& out_scale) {
  originals(x, weight, residual, residual_out, out, out_scale);
  const int type = type_of(x);
  need(x.dim() == 2 && type >= 0, "x requires BF16 or FP16 [M,K]");
  const int64_t m = x.size(0), k = x.size(1);
  need(k >= 1 && k <= kMaxWidth && m <= 0x7fffffff && rows_ok(x, m, k, x.scalar_type()),
       "x requires unit columns, rows apart by K or more, 1 <= K <= 16384");
  need(weight.dim() == 1 && weight.size(0) == k && weight.is_contiguous() &&
           (weight.scalar_type() == x.scalar_type() || weight.scalar_type() == at::kFloat),
       "weight requires contiguous [K] of x's type or FP32");
  need(normal_positive(eps), "Epsilon must be finite, positive, normal FP32");
  need(residual || !residual_out, "residual_out needs a residual");
  List ins, outs;
  add(ins, "x", x);
  add(ins, "weight", weight);
  add(ins, "residual", residual);
  add(outs, "out", out);
  add(outs, "out_scale", out_scale);
  add(outs, "residual_out", residual_out);
  List all = ins;
  all.insert(all.end(), outs.begin(), outs.end());
  plain(all);
  need(!residual || rows_ok(*residual, m, k, x.scalar_type()),
       "residual requires [M,K] of x's type, unit columns, rows apart by K or more");
  need(!residual_out || rows_ok(*residual_out, m, k, x.scalar_type()),
       "residual_out requires [M,K] of x's type, unit columns, rows apart by K or more");
  const auto code_type = code ? at::kFloat8_e4m3fn : at::kChar;
  need(!out || (out->dim() == 2 && out->size(0) == m && out->size(1) == k && out->scalar_type() == code_type && out->is_contiguous()),
       "out requires contiguous [M,K] of dtype");
  need(!out_scale || (out_scale->dim() == 2 && out_scale->size(0) == m && out_scale->size(1) == 1 &&
                      out_scale->scalar_type() == at::kFloat && out_scale->is_contiguous()),
       "out_scale requires contiguous FP32 [M,1]");
  for (size_t i = 0; i < outs.size(); ++i) {
    for (const Named& in : ins) {
      // h may take the place of an input it is computed from, value for value
      const bool place = residual_out && outs[i].t == &*residual_out && in.t != &weight &&
                         in.t->data_ptr() == outs[i].t->data_ptr() && in.t->strides() == outs[i].t->strides();
      if (!place && overlap(*in.t, *outs[i].t)) refuse(std::string("Output ") + outs[i].name + " overlaps input " + in.name);
    }
    for (size_t j = 0; j < i; ++j)
      if (overlap(*outs[j].t, *outs[i].t)) refuse(std::string("Output ") + outs[i].name + " overlaps output " + outs[j].name);
  }
  need(!residual_out || no_self_overlap(*residual_out), "residual_out must not overlap itself");
  check_device(x);
  const Tensor q = out ? *out : at::empty({m, k}, x.options().dtype(code_type));
  const Tensor s = out_scale ? *out_scale : at::empty({m, 1}, x.options().dtype(at::kFloat));
  const Tensor h = !residual ? x : residual_out ? *residual_out : at::empty({m, k}, x.options());
  List used = {{"x", &x}, {"weight", &weight}, {"q", &q}, {"s", &s}};
  if (residual) {
    add(used, "residual", residual);
    add(used, "h", h);
  }
  const auto row = [&](const Tensor& t) { return std::max(t.stride(0), k); };
  enqueue(used, outs, "residual_rms_quant", h3_rms_quant_error, [&](uintptr_t stream) {
    return h3_rms_quant_run(ptr(x), ptr(residual), ptr(weight), residual ? out_ptr(h) : nullptr, out_ptr(q),
                            static_cast<float*>(out_ptr(s)), m, k, row(x), residual ? row(*residual) : 0, residual ? row(h) : 0,
                            static_cast<float>(eps), type, weight.scalar_type() == at::kFloat ? 2 : type, code, stream);
  });
  return py::make_tuple(q, s, h);
}

// ---- rotary positions --------------------------------------------------------------------

constexpr int64_t kMaxPairs = 128, kMaxDim = 256;

// The pairs' frequencies (turns per position) and axes, made once for a model's sections.
struct Axes {
  std::vector<double> turns;
  std::vector<int> axis;
  int64_t axes;
  Axes(const std::vector<int64_t>& sections, const std::vector<double>& thetas) : axes(int64_t(sections.size())) {
    int64_t pairs = 0;
    need(!sections.empty() && sections.size() <= 255 && thetas.size() == sections.size(),
         "theta must be positive and finite, one number or one for each axis");
    for (size_t a = 0; a < sections.size(); ++a) {
      need(sections[a] >= 0, "sections requires the pairs of each axis, whole numbers from 0");
      need(std::isfinite(thetas[a]) && thetas[a] > 0, "theta must be positive and finite, one number or one for each axis");
      pairs += std::min(sections[a], kMaxPairs + 1);
    }
    need(pairs >= 1 && pairs <= kMaxPairs, "sections must sum to 1 to 128 pairs");
    for (size_t a = 0; a < sections.size(); ++a)
      for (int64_t i = 0; i < sections[a]; ++i) {
        turns.push_back(std::pow(thetas[a], -double(i) / double(sections[a])) / (2 * M_PI));
        axis.push_back(int(a));
      }
  }
  int pairs() const { return int(turns.size()); }
};

void check_positions(const Tensor& positions, const Axes& axes) {
  need(positions.dim() == 2 && (positions.scalar_type() == at::kInt || positions.scalar_type() == at::kFloat) &&
           positions.is_contiguous() && positions.size(1) == axes.axes,
       "positions requires contiguous INT32 or FP32 [T,A], one column for each of sections");
}

bool heads_ok(const Tensor& t, int64_t tokens, int64_t dim, at::ScalarType type) {
  return t.dim() == 3 && t.size(0) == tokens && t.size(2) == dim && t.scalar_type() == type && t.size(1) <= 65535 &&
         t.stride(2) == 1;
}

// Two [T,H,D] slices with one token stride that keep to different columns of the rows
// (slices of one projection interleave in memory).
bool slices_apart(const Tensor& a, const Tensor& b) {
  if (a.dim() != 3 || b.dim() != 3 || a.element_size() != b.element_size() || a.stride(0) != b.stride(0)) return false;
  const int64_t e = a.element_size(), width = a.stride(0) * e;
  if (width <= 0) return false;
  const auto columns = [&](const Tensor& t) { return ((t.size(1) - 1) * t.stride(1) + t.size(2)) * e; };
  const int64_t na = columns(a), nb = columns(b);
  int64_t lo = (static_cast<const char*>(b.data_ptr()) - static_cast<const char*>(a.data_ptr())) % width;
  if (lo < 0) lo += width;
  // b's columns begin behind a's and end before a's next row begins
  return lo >= na && lo + nb <= width;
}

py::tuple rope_axes(const Tensor& q, const Maybe& k, const Tensor& positions, const Axes& axes, bool interleaved, bool inverse,
                    const Maybe& q_weight, const Maybe& k_weight, double eps, const Maybe& q_out, const Maybe& k_out) {
  originals(q, k, positions, q_weight, k_weight, q_out, k_out);
  check_positions(positions, axes);
  const int type = type_of(q);
  need(q.dim() == 3 && type >= 0, "q requires BF16 or FP16 [T,H,D]");
  const int64_t tokens = q.size(0), hq = q.size(1), dim = q.size(2), pairs = axes.pairs();
  if (dim % 2 || dim < 2 || dim > kMaxDim || 2 * pairs > dim)
    refuse("The head width must be even, up to 256 and hold the " + std::to_string(pairs) + " pairs of sections");
  need(heads_ok(q, tokens, dim, q.scalar_type()), "q requires [T,H,D] with unit channels");
  need(!k || heads_ok(*k, tokens, dim, q.scalar_type()), "k requires [T,H,D] of q's type and tokens with unit channels");
  need(positions.size(0) == tokens, "positions requires a row for every token");
  need(normal_positive(eps), "Epsilon must be finite, positive, normal FP32");
  need(k || (!k_weight && !k_out), "k_weight and k_out need k");
  need(!k || bool(q_weight) == bool(k_weight), "q_weight and k_weight are given together");
  const Maybe* weights[2] = {&q_weight, &k_weight};
  for (const Maybe* w : weights)
    need(!*w || ((*w)->dim() == 1 && (*w)->size(0) == dim && (*w)->is_contiguous() &&
                 ((*w)->scalar_type() == q.scalar_type() || (*w)->scalar_type() == at::kFloat) &&
                 (!q_weight || (*w)->scalar_type() == q_weight->scalar_type())),
         "Norm weights require contiguous [D] of q's type or FP32, both alike");
  List ins, outs;
  add(ins, "q", q);
  add(ins, "k", k);
  add(ins, "q_weight", q_weight);
  add(ins, "k_weight", k_weight);
  add(ins, "positions", positions);
  add(outs, "q_out", q_out);
  add(outs, "k_out", k_out);
  List all = ins;
  all.insert(all.end(), outs.begin(), outs.end());
  plain(all);
  for (const Named& o : outs) {
    const Tensor& src = o.t == (q_out ? &*q_out : nullptr) ? q : *k;
    if (o.t->sizes() != src.sizes() || !heads_ok(*o.t, tokens, dim, q.scalar_type()) || !no_self_overlap(*o.t))
      refuse(std::string(o.name) + " requires the shape and type of what it takes, unit channels, not overlapping itself");
    for (const Named& other : all) {
      const bool place = other.t == &src && other.t->data_ptr() == o.t->data_ptr() && other.t->strides() == o.t->strides();
      if (other.t != o.t && !place && overlap(*o.t, *other.t) && !slices_apart(*o.t, *other.t))
        refuse(std::string("Output ") + o.name + " overlaps " + other.name);
    }
  }
  check_device(q);
  const Tensor qo = q_out ? *q_out : at::empty({tokens, hq, dim}, q.options());
  const Tensor ko = !k ? Tensor() : k_out ? *k_out : at::empty({tokens, k->size(1), dim}, q.options());
  H3RopeArgs a;
  std::memset(&a, 0, sizeof(a));
  a.q = ptr(q), a.k = ptr(k), a.q_out = out_ptr(qo), a.k_out = k ? out_ptr(ko) : nullptr;
  a.q_weight = ptr(q_weight), a.k_weight = ptr(k_weight), a.positions = ptr(positions);
  a.turns = axes.turns.data(), a.axis = axes.axis.data();
  a.tokens = tokens;
  a.q_stride_t = q.stride(0), a.q_stride_h = q.stride(1), a.qo_stride_t = qo.stride(0), a.qo_stride_h = qo.stride(1);
  if (k) a.k_stride_t = k->stride(0), a.k_stride_h = k->stride(1), a.ko_stride_t = ko.stride(0), a.ko_stride_h = ko.stride(1);
  a.q_heads = int(hq), a.k_heads = k ? int(k->size(1)) : 0, a.dim = int(dim), a.pairs = int(pairs), a.axes = int(axes.axes);
  a.float_positions = positions.scalar_type() == at::kFloat;
  a.type = type, a.weight_type = q_weight && q_weight->scalar_type() == at::kFloat ? 2 : type;
  a.interleaved = interleaved, a.inverse = inverse, a.eps = static_cast<float>(eps);
  List used = ins;
  add(used, "qo", qo);
  if (k) add(used, "ko", ko);
  enqueue(used, outs, "rope_axes", h3_rope_error, [&](uintptr_t stream) { return h3_rope_axes_run(&a, stream); });
  return py::make_tuple(qo, k ? py::cast(ko) : py::none());
}

Tensor rope_table(const Tensor& positions, const Axes& axes, const Maybe& out) {
  originals(positions, out);
  check_positions(positions, axes);
  const int64_t tokens = positions.size(0), pairs = axes.pairs();
  const std::vector<int64_t> shape = {1, tokens, 1, pairs, 2, 2};
  List all;
  add(all, "positions", positions);
  add(all, "out", out);
  plain(all);
  if (out) {
    need(out->sizes() == at::IntArrayRef(shape) && out->scalar_type() == at::kBFloat16 && out->is_contiguous() && aligned(*out, 8),
         "out requires contiguous BF16 [1,T,1,P,2,2], 8B alignment");
    need(!overlap(positions, *out), "Output out overlaps positions");
  }
  check_device(positions);
  const Tensor table = out ? *out : at::empty(shape, positions.options().dtype(at::kBFloat16));
  enqueue({{"positions", &positions}, {"table", &table}}, out ? List{{"out", &table}} : List{}, "rope_table", h3_rope_error,
          [&](uintptr_t stream) {
            return h3_rope_table_run(ptr(positions), axes.turns.data(), axes.axis.data(), out_ptr(table), tokens, int(pairs),
                                     int(axes.axes), positions.scalar_type() == at::kFloat, stream);
          });
  return table;
}

// ---- attention under masks ------------------------------------------------------------------

constexpr int64_t kMaxLength = int64_t(1) << 30;

struct View {   // [B, S, H, D] of a 3-D or 4-D tensor; strides 0 for dimensions of one element,
                // and where there is none at all
  int64_t size[4], stride[3];
  explicit View(const Tensor& t) {
    const int64_t d = t.dim() - 4;   // -1: one sequence
    for (int i = 0; i < 4; ++i) size[i] = i + d < 0 ? 1 : t.size(i + d);
    for (int i = 0; i < 3; ++i) stride[i] = i + d < 0 || size[i] <= 1 || t.numel() == 0 ? 0 : t.stride(i + d);
  }
};

void check_layout(const char* name, const Tensor& t, const View& v) {
  if (t.numel() == 0) return;
  if (t.stride(-1) != 1 || !aligned(t, 16) || v.stride[0] % 8 || v.stride[1] % 8 || v.stride[2] % 8)
    refuse(std::string(name) + " requires unit channels, strides in multiples of 8 and 16-byte alignment");
}

void check_counts(const char* name, const Maybe& t, int64_t n) {
  if (t && (t->scalar_type() != at::kInt || t->dim() != 1 || t->size(0) != n || !t->is_contiguous()))
    refuse(std::string(name) + " requires contiguous INT32 [" + std::to_string(n) + "]");
}

py::object masked_attention(const Tensor& q, const Tensor& k, const Tensor& v, std::optional<double> scale_arg, double softcap,
                            const Maybe& slopes, bool causal, const Maybe& prefix, const Maybe& q_offsets, const Maybe& k_offsets,
                            const Maybe& q_lengths, const Maybe& k_lengths, const Maybe& out_arg, const Maybe& lse_arg,
                            bool return_lse) {
  originals(q, k, v, slopes, prefix, q_offsets, k_offsets, q_lengths, k_lengths, out_arg, lse_arg);
  const int type = type_of(q);
  const bool flat = q.dim() == 3;
  for (const Tensor* t : {&q, &k, &v})
    need((flat || q.dim() == 4) && type >= 0 && t->dim() == q.dim() && t->scalar_type() == q.scalar_type(),
         "q, k and v require BF16 or FP16 [B,S,H,D] or [S,H,D], all alike");
  const View qv(q), kv(k), vv(v);
  const int64_t b = qv.size[0], sq = qv.size[1], hq = qv.size[2], d = qv.size[3], sk = kv.size[1], hk = kv.size[2];
  need(kv.size[0] == b && kv.size[3] == d && k.sizes() == v.sizes() && (d == 64 || d == 128),
       "k and v require [B,Sk,Hk,D] of one shape, q [B,Sq,Hq,D], D 64 or 128");
  need(hk >= 1 && hq >= 1 && hq % hk == 0 && hq <= 65535 && b <= (1 << 20) && std::max(sq, sk) <= kMaxLength,
       "Hq must be a positive multiple of Hk, up to 65535; lengths up to 2^30");
  check_layout("q", q, qv);
  check_layout("k", k, kv);
  check_layout("v", v, vv);
  need(!(sq > 1 && qv.stride[1] == 0) && !(hq > 1 && qv.stride[2] == 0) && !(sk > 1 && (kv.stride[1] == 0 || vv.stride[1] == 0)),
       "Only heads of k and v and batches may be expanded");
  const double scale = scale_arg ? *scale_arg : 1.0 / std::sqrt(double(d));
  need(normal_positive(scale) && normal_positive(3 * scale) && std::isfinite(static_cast<float>(3 * softcap)) &&
           (softcap == 0 || (normal_positive(softcap) && std::isfinite(static_cast<float>(scale / softcap * 3)))),
       "scale must be positive and finite, softcap finite and not negative, their ratio finite");
  int64_t documents = 0;
  if (q_offsets || k_offsets) {
    need(q_offsets && k_offsets && b == 1 && !q_lengths && !k_lengths,
         "q_offsets and k_offsets are given together, for one sequence without lengths");
    documents = q_offsets->numel() - 1;
    need(documents >= 1 && documents < kMaxLength, "q_offsets requires contiguous INT32 [N + 1] of at least one document");
    check_counts("q_offsets", q_offsets, documents + 1);
    check_counts("k_offsets", k_offsets, documents + 1);
  }
  check_counts("q_lengths", q_lengths, b);
  check_counts("k_lengths", k_lengths, b);
  need(!prefix || causal, "prefix widens a causal mask: pass causal=True");
  check_counts("prefix", prefix, documents ? documents : b);
  need(!slopes || (slopes->scalar_type() == at::kFloat && slopes->dim() == 1 && slopes->size(0) == hq && slopes->is_contiguous()),
       "slopes requires contiguous FP32 [Hq]");
  if (out_arg) {
    need(out_arg->sizes() == q.sizes() && out_arg->scalar_type() == q.scalar_type(), "out requires q's shape and type");
    check_layout("out", *out_arg, View(*out_arg));
    need(no_self_overlap(*out_arg), "out must not overlap itself");
  }
  if (lse_arg) {
    const std::vector<int64_t> shape = flat ? std::vector<int64_t>{hq, sq} : std::vector<int64_t>{b, hq, sq};
    need(lse_arg->scalar_type() == at::kFloat && lse_arg->sizes() == at::IntArrayRef(shape) && lse_arg->is_contiguous(),
         "lse requires contiguous FP32 [B,Hq,Sq] ([Hq,Sq] for one sequence)");
  }
  List ins, outs;
  add(ins, "q", q);
  add(ins, "k", k);
  add(ins, "v", v);
  add(ins, "slopes", slopes);
  add(ins, "q_offsets", q_offsets);
  add(ins, "k_offsets", k_offsets);
  add(ins, "q_lengths", q_lengths);
  add(ins, "k_lengths", k_lengths);
  add(ins, "prefix", prefix);
  add(outs, "out", out_arg);
  add(outs, "lse", lse_arg);
  List all = ins;
  all.insert(all.end(), outs.begin(), outs.end());
  plain(all);
  for (const Named& o : outs)
    for (const Named& other : all)
      if (other.t != o.t && overlap(*o.t, *other.t)) refuse(std::string("Output ") + o.name + " overlaps " + other.name);
  check_device(q);

  const Tensor out = out_arg ? *out_arg : at::empty(q.sizes(), q.options());
  Tensor lse;
  if (lse_arg)
    lse = *lse_arg;
  else if (return_lse)
    lse = flat ? at::empty({hq, sq}, q.options().dtype(at::kFloat)) : at::empty({b, hq, sq}, q.options().dtype(at::kFloat));
  // rows of no sequence are zero in new outputs; one new and one given: the new one is
  // zeroed beforehand, so that the given one keeps its rows
  const bool gaps = documents || q_lengths;
  const bool fill = gaps && !out_arg && !lse_arg;
  if (gaps && !fill) {
    if (!out_arg) out.zero_();
    if (!lse_arg && lse.defined()) lse.zero_();
  }
  const View ov(out);
  H3MaskedAttentionArgs a;
  std::memset(&a, 0, sizeof(a));
  a.q = ptr(q), a.k = ptr(k), a.v = ptr(v), a.out = out_ptr(out);
  a.lse = lse.defined() ? static_cast<float*>(out_ptr(lse)) : nullptr;
  a.slopes = static_cast<const float*>(ptr(slopes));
  a.q_offsets = ints(q_offsets), a.k_offsets = ints(k_offsets), a.q_lengths = ints(q_lengths), a.k_lengths = ints(k_lengths);
  a.prefix = ints(prefix);
  a.q_stride_b = qv.stride[0], a.q_stride_s = qv.stride[1], a.q_stride_h = qv.stride[2];
  a.k_stride_b = kv.stride[0], a.k_stride_s = kv.stride[1], a.k_stride_h = kv.stride[2];
  a.v_stride_b = vv.stride[0], a.v_stride_s = vv.stride[1], a.v_stride_h = vv.stride[2];
  a.o_stride_b = ov.stride[0], a.o_stride_s = ov.stride[1], a.o_stride_h = ov.stride[2];
  a.batch = int(b), a.q_len = int(sq), a.k_len = int(sk), a.q_heads = int(hq), a.k_heads = int(hk), a.dim = int(d);
  a.type = type, a.documents = int(documents), a.causal = causal, a.fill = fill;
  a.scale = static_cast<float>(scale), a.softcap = static_cast<float>(softcap);
  List used = ins;
  add(used, "out", out);
  if (lse.defined()) add(used, "lse", lse);
  const c10::cuda::OptionalCUDAGuard guard(q.device());
  Tensor workspace;
  const int64_t bytes = h3_masked_attention_workspace(&a);
  if (bytes > 0) {
    workspace = at::empty({bytes}, q.options().dtype(at::kByte));
    a.workspace = out_ptr(workspace), a.workspace_bytes = uint64_t(bytes);
    add(used, "workspace", workspace);
  }
  enqueue(used, outs, "masked_attention", h3_masked_attention_error,
          [&](uintptr_t stream) { return h3_masked_attention_run(&a, stream); });
  if (!lse.defined()) return py::cast(out);
  return py::make_tuple(out, lse);
}

}  // namespace

PYBIND11_MODULE(h3sk_torch, m) {
  // the argument blocks go to the library by address
  if (h3_rope_args_size() != sizeof(H3RopeArgs) || h3_masked_attention_args_size() != sizeof(H3MaskedAttentionArgs))
    throw std::runtime_error("H3 SpeedKit B200 library and binding were built from different argument blocks; build both again");
  py::class_<Axes>(m, "Axes").def(py::init<const std::vector<int64_t>&, const std::vector<double>&>());
  m.def("rms_quant", &rms_quant);
  m.def("rope_axes", &rope_axes);
  m.def("rope_table", &rope_table);
  m.def("masked_attention", &masked_attention);
}
