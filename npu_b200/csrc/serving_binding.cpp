// Python binding of the serving operators (npu_b200._serving): the argument
// checks, output and workspace allocation and the call of the C ABI in one
// step. A call through ctypes costs 13 to 24 us of host time for these
// argument lists, several times what a single-token kernel runs; through this
// module it costs 4.6 to 5.5. npu_b200.api documents the functions.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <optional>
#include <sstream>

#include "b2attn.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

template <typename... Args>
[[noreturn]] void refuse(const Args&... args) {
  std::ostringstream s;
  (s << ... << args);
  throw py::value_error(s.str());
}

// Raises B2AError for a status that is not B2A_OK.
void check(int rc, const char* what) {
  if (rc != B2A_OK) py::module_::import("npu_b200._lib").attr("check")(rc, what);
}

void need_cuda(const char* name, const Tensor& t, const c10::Device* device = nullptr) {
  if (!t.is_cuda()) refuse(name, " must be a CUDA tensor (no CPU path exists)");
  if (device && t.device() != *device) refuse(name, " must be on the inputs' device");
}

void need_bf16(const char* name, const Tensor& t, int ndim, const c10::Device* device = nullptr) {
  need_cuda(name, t, device);
  if (t.scalar_type() != at::kBFloat16) refuse(name, " must be bfloat16, got ", t.scalar_type());
  if (t.dim() != ndim) refuse(name, " must have ", ndim, " dims, got shape ", t.sizes());
  if (t.stride(-1) != 1) refuse(name, " needs a contiguous last (head_dim) dimension");
}

void need_int32(const char* name, const Tensor& t, int64_t numel, const c10::Device& device) {
  if (t.scalar_type() != at::kInt || t.device() != device || t.numel() != numel || !t.is_contiguous())
    refuse(name, " must be a contiguous int32 tensor of ", numel, " on the inputs' device");
}

void need_table(const Tensor& t, int64_t batch, const c10::Device& device) {
  if (t.scalar_type() != at::kInt || t.device() != device || t.dim() != 2 || t.size(0) != batch || t.stride(1) != 1)
    refuse("block_table must be an int32 tensor [", batch,
           ", pages] on the inputs' device with a contiguous last dim");
}

void need_gate(const Tensor& t, const Tensor& q) {
  if (t.device() != q.device()) refuse("gate must be a CUDA tensor on q's device");
  if (t.scalar_type() != at::kFloat && t.scalar_type() != at::kBFloat16) refuse("gate must be float32 or bfloat16");
  if (t.sizes() != q.sizes() || t.stride(-1) != 1)
    refuse("gate must be ", q.sizes(), " with a contiguous last dim, got ", t.sizes());
}

// int arguments of the C ABI.
int as_int(const char* name, int64_t v) {
  if (v < INT_MIN || v > INT_MAX) refuse(name, " is too large: ", v);
  return (int)v;
}

// A new tensor on like's device, by the allocator of torch's current stream
// (without the dispatcher, which takes as long as the allocation).
Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}

Tensor output(const OptTensor& out, at::IntArrayRef sizes, at::ScalarType type, const Tensor& like, const char* what) {
  if (!out) return empty(sizes, type, like);
  if (out->scalar_type() != type || out->sizes() != sizes || (out->size(-1) > 1 && out->stride(-1) != 1) ||
      out->device() != like.device())
    refuse(what);
  return *out;
}

at::ScalarType float_type(const char* name, at::ScalarType type) {
  if (type != at::kFloat && type != at::kBFloat16) refuse(name, " must be float32 or bfloat16");
  return type;
}

void* pointer(const OptTensor& t) { return t ? t->data_ptr() : nullptr; }

struct Strides {
  long long s[3];
  explicit Strides(const Tensor& t, int n) {
    for (int i = 0; i < n; ++i) s[i] = t.stride(i);
  }
  operator const long long*() const { return s; }
};

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

py::object prefill_varlen(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cu_q, const OptTensor& cu_k,
                          std::optional<double> scale, bool causal, at::ScalarType out_dtype, const OptTensor& out,
                          bool return_lse, const OptTensor& gate) {
  need_bf16("q", q, 3);
  const c10::Device device = q.device();
  need_bf16("k", k, 3, &device);
  need_bf16("v", v, 3, &device);
  const int64_t Nq = q.size(0), Hq = q.size(1), D = q.size(2), Nk = k.size(0), Hkv = k.size(1);
  if (k.size(2) != D || v.sizes() != k.sizes())
    refuse("shape mismatch q", q.sizes(), " k", k.sizes(), " v", v.sizes());
  const int64_t B = cu_q.numel() - 1;
  if (B < 1) refuse("cu_seqlens_q must hold at least two offsets");
  need_int32("cu_seqlens_q", cu_q, B + 1, device);
  if (cu_k)
    need_int32("cu_seqlens_k", *cu_k, B + 1, device);
  else if (Nk != Nq)
    refuse("k has ", Nk, " rows and q ", Nq, ": cu_seqlens_k is needed");
  float_type("out_dtype", out_dtype);
  if (gate) need_gate(*gate, q);
  const c10::cuda::CUDAGuard guard(device);
  Tensor o = output(out, q.sizes(), out_dtype, q,
                    "out must match [Nq, Hq, D], out_dtype and q's device, with a contiguous last dim");
  OptTensor lse;
  if (return_lse) lse = empty({Hq, Nq}, at::kFloat, q);
  const Strides gs(gate ? *gate : q, 2);
  check(b2a_prefill_varlen(q.data_ptr(), k.data_ptr(), v.data_ptr(), pointer(gate), o.data_ptr(),
                           static_cast<float*>(pointer(lse)), cu_q.data_ptr<int>(),
                           (cu_k ? *cu_k : cu_q).data_ptr<int>(), as_int("B", B), as_int("Nq", Nq), as_int("Nk", Nk),
                           as_int("Hq", Hq), as_int("Hkv", Hkv), as_int("D", D), Strides(q, 2), Strides(k, 2),
                           Strides(v, 2), gs, Strides(o, 2), gate && gate->scalar_type() == at::kBFloat16,
                           (float)scale.value_or(1.0 / std::sqrt((double)D)), causal, out_dtype == at::kFloat,
                           stream_of(q)),
        "b2a_prefill_varlen");
  if (return_lse) return py::make_tuple(o, *lse);
  return py::cast(o);
}

Tensor decode_paged(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages, const Tensor& table,
                    const Tensor& seqlens, std::optional<double> scale, at::ScalarType out_dtype,
                    const OptTensor& workspace, const OptTensor& out, const OptTensor& gate) {
  need_bf16("q", q, 3);
  const c10::Device device = q.device();
  need_bf16("k_pages", k_pages, 4, &device);
  need_bf16("v_pages", v_pages, 4, &device);
  const int64_t B = q.size(0), Hq = q.size(1), D = q.size(2), n_pages = k_pages.size(0), Hkv = k_pages.size(1),
                page = k_pages.size(2);
  if (k_pages.size(3) != D || v_pages.sizes() != k_pages.sizes())
    refuse("shape mismatch q", q.sizes(), " k_pages", k_pages.sizes(), " v_pages", v_pages.sizes());
  need_table(table, B, device);
  need_int32("seqlens", seqlens, B, device);
  float_type("out_dtype", out_dtype);
  if (gate) need_gate(*gate, q);
  const c10::cuda::CUDAGuard guard(device);
  Tensor o = output(out, q.sizes(), out_dtype, q,
                    "out must match [B, Hq, D], out_dtype and q's device, with a contiguous last dim");
  if (B == 0) return o;
  const size_t need =
      b2a_decode_paged_workspace_bytes(as_int("B", B), as_int("Hq", Hq), as_int("Hkv", Hkv), as_int("D", D));
  // Scratch taken here goes back when the call returns; what reuses it on this
  // stream runs after this call's kernels.
  c10::DataPtr taken;
  void* ws;
  if (workspace) {
    if (workspace->device() != device || !workspace->is_contiguous() || workspace->nbytes() < need)
      refuse("workspace must be a contiguous CUDA tensor of at least ", need, " bytes on q's device");
    ws = workspace->data_ptr();
  } else {
    taken = c10::cuda::CUDACachingAllocator::get()->allocate(std::max<size_t>(need, 16));
    ws = taken.get();
  }
  const Strides gs(gate ? *gate : q, 2);
  check(b2a_decode_paged(q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), table.data_ptr<int>(), table.stride(0),
                         as_int("table width", table.size(1)), seqlens.data_ptr<int>(), pointer(gate), o.data_ptr(),
                         (int)B, (int)Hq, (int)Hkv, as_int("n_pages", n_pages), as_int("page", page), (int)D,
                         Strides(q, 2), Strides(k_pages, 3), Strides(v_pages, 3), gs, Strides(o, 2),
                         gate && gate->scalar_type() == at::kBFloat16,
                         (float)scale.value_or(1.0 / std::sqrt((double)D)), out_dtype == at::kFloat, ws, need,
                         stream_of(q)),
        "b2a_decode_paged");
  return o;
}

py::object rope_append_paged(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cos, const Tensor& sin,
                             const Tensor& k_pages, const Tensor& v_pages, const Tensor& table, const Tensor& cu,
                             int64_t start_pos, const OptTensor& start, const OptTensor& seqlens_out,
                             const OptTensor& q_out, const OptTensor& q_norm, const OptTensor& k_norm, double eps,
                             std::optional<int64_t> rope_dim, bool return_kv) {
  for (auto [name, t] : {std::pair<const char*, const Tensor*>{"q", &q}, {"k", &k}, {"v", &v}})
    if (!t->is_cuda() || t->dim() != 3 || t->stride(-1) != 1)
      refuse(name, " must be a CUDA [N, H, D] tensor with a contiguous last dim");
  const c10::Device device = q.device();
  const at::ScalarType type = q.scalar_type();
  const int64_t N = q.size(0), Hq = q.size(1), D = q.size(2), Hkv = k.size(1);
  if (k.size(0) != N || k.size(2) != D || v.sizes() != k.sizes())
    refuse("shape mismatch q", q.sizes(), " k", k.sizes(), " v", v.sizes());
  if ((type != at::kFloat && type != at::kBFloat16) || k.scalar_type() != type || v.scalar_type() != type)
    refuse("q, k, v must share one dtype, float32 or bfloat16");
  if (k.device() != device || v.device() != device || cos.device() != device || sin.device() != device)
    refuse("q, k, v, cos and sin must be on one device");
  const int64_t rope = rope_dim.value_or(D);
  if ((cos.scalar_type() != at::kFloat && cos.scalar_type() != type) || sin.scalar_type() != cos.scalar_type() ||
      !cos.is_contiguous() || !sin.is_contiguous() || cos.dim() != 2 || cos.size(1) != rope ||
      sin.sizes() != cos.sizes())
    refuse("cos/sin must be contiguous [max_pos, rope_dim] tensors, float32 or in q's dtype");
  need_bf16("k_pages", k_pages, 4, &device);
  need_bf16("v_pages", v_pages, 4, &device);
  if (k_pages.size(1) != Hkv || k_pages.size(3) != D || v_pages.sizes() != k_pages.sizes())
    refuse("cache shape ", k_pages.sizes(), " does not fit k", k.sizes());
  const int64_t B = cu.numel() - 1;
  if (B < 1) refuse("cu_seqlens must hold at least two offsets");
  need_int32("cu_seqlens", cu, B + 1, device);
  need_table(table, B, device);
  if (start) need_int32("start_pos_per_batch", *start, B, device);
  if (seqlens_out) need_int32("seqlens_out", *seqlens_out, B, device);
  if (start && seqlens_out && start->data_ptr<int>() < seqlens_out->data_ptr<int>() + B &&
      seqlens_out->data_ptr<int>() < start->data_ptr<int>() + B)
    refuse("seqlens_out must not overlap start_pos_per_batch: the positions are read while it is written");
  for (auto [name, w] : {std::pair<const char*, const OptTensor*>{"q_norm", &q_norm}, {"k_norm", &k_norm}})
    if (*w && ((*w)->scalar_type() != type || (*w)->device() != device || (*w)->dim() != 1 || (*w)->size(0) != D ||
               !(*w)->is_contiguous()))
      refuse(name, " must be a contiguous [D] tensor in q's dtype on q's device");
  const c10::cuda::CUDAGuard guard(device);
  const char* wants = "q_out must be a contiguous bf16 [N, Hq, D] tensor on q's device";
  if (q_out && !q_out->is_contiguous()) refuse(wants);
  Tensor qo = output(q_out, q.sizes(), at::kBFloat16, q, wants);
  const bool bf16 = type == at::kBFloat16;
  OptTensor ko, vo;
  if (return_kv) ko = empty({N, Hkv, D}, at::kBFloat16, q);
  if (return_kv && !bf16) vo = empty({N, Hkv, D}, at::kBFloat16, q);
  auto result = [&]() -> py::object {
    if (return_kv) return py::make_tuple(qo, *ko, bf16 ? v : *vo);
    return py::cast(qo);
  };
  if (N == 0) {  // the lengths are the positions
    if (seqlens_out && start) seqlens_out->copy_(*start);
    if (seqlens_out && !start) seqlens_out->fill_(start_pos);
    return result();
  }
  check(b2a_rope_append_paged(q.data_ptr(), k.data_ptr(), v.data_ptr(), Strides(q, 2), Strides(k, 2), Strides(v, 2),
                              bf16, pointer(q_norm), pointer(k_norm), (float)eps, cos.data_ptr(), sin.data_ptr(),
                              cos.scalar_type() == at::kFloat, as_int("max_pos", cos.size(0)),
                              as_int("rope_dim", rope), qo.data_ptr(), pointer(ko), pointer(vo), k_pages.data_ptr(),
                              v_pages.data_ptr(), Strides(k_pages, 3), Strides(v_pages, 3), table.data_ptr<int>(),
                              table.stride(0), as_int("table width", table.size(1)),
                              as_int("n_pages", k_pages.size(0)), as_int("page", k_pages.size(2)),
                              cu.data_ptr<int>(), as_int("B", B), as_int("N", N), as_int("Hq", Hq),
                              as_int("Hkv", Hkv), as_int("D", D), as_int("start_pos", start_pos),
                              static_cast<int*>(pointer(start)), static_cast<int*>(pointer(seqlens_out)),
                              stream_of(q)),
        "b2a_rope_append_paged");
  return result();
}

// A sampling setting: a number for every row, or a per-row tensor.
template <typename T>
struct Setting {
  const T* rows = nullptr;
  double all = 0;
  Setting(const char* name, const py::handle& value, int64_t R, const c10::Device& device) {
    if (THPVariable_Check(value.ptr())) {
      const Tensor& t = THPVariable_Unpack(value.ptr());
      const at::ScalarType type = std::is_same_v<T, float> ? at::kFloat : at::kInt;
      if (t.scalar_type() != type || t.device() != device || t.dim() != 1 || t.size(0) != R || !t.is_contiguous())
        refuse(name, " must be a number or a contiguous ", type, " tensor [", R, "] on the logits' device");
      rows = t.data_ptr<T>();
    } else {
      try {
        all = value.cast<double>();
      } catch (const py::cast_error&) {
        refuse(name, " must be a number or a tensor [", R, "] on the logits' device");
      }
    }
  }
};

Tensor sample(const Tensor& logits, const OptTensor& noise, const py::handle& temperature, const py::handle& top_k,
              const py::handle& top_p, const py::handle& min_p, const OptTensor& out) {
  const bool bf16 = logits.scalar_type() == at::kBFloat16;
  if (!logits.is_cuda() || logits.dim() != 2 || logits.stride(1) != 1 || (logits.scalar_type() != at::kFloat && !bf16))
    refuse("logits must be a CUDA float32 or bfloat16 tensor [R, V] with a contiguous last dim");
  const int64_t R = logits.size(0), V = logits.size(1);
  const c10::Device device = logits.device();
  if (noise && (noise->scalar_type() != at::kFloat || noise->device() != device || noise->sizes() != logits.sizes() ||
                noise->stride(1) != 1))
    refuse("noise must be a float32 tensor [", R, ", ", V, "] on the logits' device with a contiguous last dim");
  const Setting<float> t("temperature", temperature, R, device), p("top_p", top_p, R, device),
      m("min_p", min_p, R, device);
  const Setting<int> k("top_k", top_k, R, device);
  if (std::isnan(k.all)) refuse("top_k must not be NaN");
  if (!noise && (t.rows || t.all > 0)) refuse("a temperature above 0 needs noise");
  const c10::cuda::CUDAGuard guard(device);
  Tensor o = output(out, {R}, at::kLong, logits, "out must be a contiguous int64 tensor [R] on the logits' device");
  if (R == 0) return o;
  check(b2a_sample(logits.data_ptr(), logits.stride(0), bf16, static_cast<float*>(pointer(noise)),
                   noise ? noise->stride(0) : 0, as_int("R", R), as_int("V", V), t.rows, (float)t.all, k.rows,
                   (int)std::min(std::max(k.all, -1.0), 2147483647.0), p.rows, (float)p.all, m.rows, (float)m.all,
                   reinterpret_cast<long long*>(o.data_ptr<int64_t>()), stream_of(logits)),
        "b2a_sample");
  return o;
}

}  // namespace

PYBIND11_MODULE(_serving, m) {
  m.def("prefill_varlen", &prefill_varlen);
  m.def("decode_paged", &decode_paged);
  m.def("rope_append_paged", &rope_append_paged);
  m.def("sample", &sample);
}
