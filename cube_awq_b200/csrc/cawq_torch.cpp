// cawq_torch.cpp — compiled host path of the module forward and of the layer
// operators (torch binding).
//
// AWQGEMMLinear.forward (src/modules/awq_gemm.rs:146-232) is called once per
// layer per token; at decode sizes its host work is of the order of the
// kernel's own device time. This extension holds a layer's tensors and the
// constant arguments of its cawq_gemm call, and its forward does, in C++: the
// input checks, one allocation of the output through torch's caching
// allocator on the input's device, the current stream, and the C call. The
// Python module keeps the reference's API and messages: whenever an input
// does not fit (wrong dtype, device, rank, K, layout), forward returns None
// and the module takes its general path, which raises the reference's errors.
//
// The layer operators (norm, rotary append, attention) have the same in plain
// functions: checks, allocation, the device and its current stream, one C
// call. They too return None for arguments that do not fit, and the Python
// functions of layer_ops.py then say what is wrong.
//
// Nothing here computes: the kernels are libcube_awq.so's.
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <cmath>

#include "cube_awq.h"

namespace {

struct Layer {
  at::Tensor qweight, qzeros, scales, bias;  // held, so their storage stays alive
  const uint32_t* qw = nullptr;
  const uint32_t* qz = nullptr;
  const void* sc = nullptr;
  const void* b = nullptr;
  int64_t k = 0, n = 0, g = 0;
  c10::ScalarType dtype = c10::ScalarType::Float;
  cawq_dtype code = CAWQ_F32;
  cawq_order order = CAWQ_ORDER_AWQ;
  c10::DeviceIndex device = 0;

  Layer(at::Tensor qweight_, at::Tensor qzeros_, at::Tensor scales_,
        c10::optional<at::Tensor> bias_, int64_t group_size, int64_t order_)
      : qweight(std::move(qweight_)), qzeros(std::move(qzeros_)), scales(std::move(scales_)) {
    TORCH_CHECK(qweight.is_cuda() && qzeros.is_cuda() && scales.is_cuda(),
                "layer tensors must be on a GPU");
    TORCH_CHECK(qweight.is_contiguous() && qzeros.is_contiguous() && scales.is_contiguous(),
                "layer tensors must be contiguous");
    TORCH_CHECK(qweight.dim() == 2 && scales.dim() == 2, "qweight and scales must be 2-D");
    if (bias_.has_value()) {
      bias = *bias_;
      TORCH_CHECK(bias.is_cuda() && bias.is_contiguous() && bias.scalar_type() == scales.scalar_type(),
                  "bias must be a contiguous GPU tensor in the scales' dtype");
      b = bias.data_ptr();
    }
    dtype = scales.scalar_type();
    switch (dtype) {
      case c10::ScalarType::Float: code = CAWQ_F32; break;
      case c10::ScalarType::Half: code = CAWQ_F16; break;
      case c10::ScalarType::BFloat16: code = CAWQ_BF16; break;
      default: TORCH_CHECK(false, "scales must be float32, float16 or bfloat16");
    }
    order = order_ == 1 ? CAWQ_ORDER_NATURAL : CAWQ_ORDER_AWQ;
    k = qweight.size(0);
    n = qweight.size(1) * 8;
    g = group_size;
    device = scales.get_device();
    qw = static_cast<const uint32_t*>(qweight.data_ptr());
    qz = static_cast<const uint32_t*>(qzeros.data_ptr());
    sc = scales.data_ptr();
  }

  // out = x · deq(W) (+ bias) for a contiguous [rows, K] input of the layer's
  // dtype on its device; None for any other input (the caller's general path
  // then checks it and raises); an int status if the C call failed.
  py::object forward(const at::Tensor& x) const {
    if (!x.is_cuda() || x.dim() != 2 || x.scalar_type() != dtype || x.get_device() != device ||
        x.size(1) != k || !x.is_contiguous())
      return py::none();
    const int64_t rows = x.size(0);
    at::Tensor out = at::empty({rows, n}, x.options());
    if (rows == 0) return py::cast(out);
    cudaStream_t s = c10::cuda::getCurrentCUDAStream(device).stream();
    const cawq_status st = cawq_gemm(x.data_ptr(), qw, qz, sc, b, out.data_ptr(),
                                     static_cast<size_t>(rows), static_cast<size_t>(k),
                                     static_cast<size_t>(n), static_cast<size_t>(g), code, code,
                                     order, static_cast<size_t>(n), s);
    if (st != CAWQ_OK) return py::int_(static_cast<int>(st));
    return py::cast(out);
  }
};

// ------------------------------------------------------- layer operators
using OptTensor = c10::optional<at::Tensor>;

bool float_code(c10::ScalarType t, cawq_dtype* code) {
  switch (t) {
    case c10::ScalarType::Float: *code = CAWQ_F32; return true;
    case c10::ScalarType::Half: *code = CAWQ_F16; return true;
    case c10::ScalarType::BFloat16: *code = CAWQ_BF16; return true;
    default: return false;
  }
}

struct On {  // the device and type that every operand of a call must have
  c10::DeviceIndex device;
  bool here(const at::Tensor& t) const { return t.is_cuda() && t.get_device() == device; }
};

// Row stride of a [rows, d] operand with a unit column stride (a contiguous
// tensor of any rank counts as one); false if it is neither.
bool rows_of(const at::Tensor& t, const On& on, c10::ScalarType type, c10::IntArrayRef shape,
             int64_t d, size_t* ld) {
  if (!on.here(t) || t.scalar_type() != type || t.sizes() != shape) return false;
  if (t.is_contiguous()) {
    *ld = static_cast<size_t>(d);
    return true;
  }
  if (t.dim() != 2 || (d > 1 && t.stride(1) != 1) || t.stride(0) < d) return false;
  *ld = static_cast<size_t>(t.stride(0));
  return true;
}

// (y, h), or (y8, scales, h) with `fp8`
py::object rms_norm_any(const at::Tensor& x, const at::Tensor& weight, double eps,
                        const OptTensor& residual, const OptTensor& out_, const OptTensor& scales_,
                        const OptTensor& res_out_, bool fp8) {
  cawq_dtype code;
  if (!x.is_cuda() || x.dim() < 1 || !float_code(x.scalar_type(), &code)) return py::none();
  const On on{x.get_device()};
  const int64_t d = x.size(-1);
  if (d <= 0 || (res_out_ && !residual)) return py::none();
  const int64_t rows = x.numel() / d;
  const auto type = x.scalar_type();
  const auto ytype = fp8 ? c10::ScalarType::Float8_e4m3fn : type;
  size_t ld_x, ld_r = 0, ld_y, ld_h = 0;
  if (!rows_of(x, on, type, x.sizes(), d, &ld_x) || !on.here(weight) || weight.dim() != 1 ||
      weight.size(0) != d || weight.scalar_type() != type || !weight.is_contiguous())
    return py::none();
  if (residual && !rows_of(*residual, on, type, x.sizes(), d, &ld_r)) return py::none();
  const c10::cuda::CUDAGuard guard(on.device);
  at::Tensor y = out_ ? *out_ : at::empty(x.sizes(), x.options().dtype(ytype));
  if (!rows_of(y, on, ytype, x.sizes(), d, &ld_y)) return py::none();
  at::Tensor h, scales;
  if (residual) {
    h = res_out_ ? *res_out_ : at::empty(x.sizes(), x.options());
    if (!rows_of(h, on, type, x.sizes(), d, &ld_h)) return py::none();
  }
  const auto lead = x.sizes().slice(0, x.dim() - 1);
  if (fp8) {
    scales = scales_ ? *scales_ : at::empty(lead, x.options().dtype(c10::ScalarType::Float));
    if (!on.here(scales) || scales.scalar_type() != c10::ScalarType::Float ||
        scales.sizes() != lead || !scales.is_contiguous())
      return py::none();
  }
  void* s = c10::cuda::getCurrentCUDAStream(on.device).stream();
  const void* rp = residual ? residual->data_ptr() : nullptr;
  void* hp = residual ? h.data_ptr() : nullptr;
  const size_t n = static_cast<size_t>(rows), dd = static_cast<size_t>(d);
  const cawq_status st =
      fp8 ? cawq_rms_norm_fp8(x.data_ptr(), weight.data_ptr(), rp, y.data_ptr(),
                              static_cast<float*>(scales.data_ptr()), hp, n, dd, ld_x, ld_r, ld_y,
                              ld_h, static_cast<float>(eps), code, s)
          : cawq_rms_norm(x.data_ptr(), weight.data_ptr(), rp, y.data_ptr(), hp, n, dd, ld_x, ld_r,
                          ld_y, ld_h, static_cast<float>(eps), code, s);
  if (st != CAWQ_OK) return py::int_(static_cast<int>(st));
  const py::object ho = residual ? py::cast(h) : py::none();
  if (fp8) return py::make_tuple(y, scales, ho);
  return py::make_tuple(y, ho);
}

bool paged(const at::Tensor& k, const at::Tensor& v, const at::Tensor& table,
           const at::Tensor& lens, const OptTensor& q_start, const On& on, c10::ScalarType type,
           cawq_paged_kv* kv) {
  const auto i32 = c10::ScalarType::Int;
  if (!on.here(k) || !on.here(v) || !on.here(table) || !on.here(lens)) return false;
  if (k.dim() != 4 || k.sizes() != v.sizes() || k.scalar_type() != type ||
      v.scalar_type() != type)
    return false;
  if (k.numel() > 0 && (k.stride(3) != 1 || k.strides() != v.strides())) return false;
  if (lens.dim() != 1 || lens.scalar_type() != i32 || !lens.is_contiguous()) return false;
  const int64_t batch = lens.size(0);
  if (table.dim() != 2 || table.scalar_type() != i32 || table.size(0) != batch ||
      (table.size(1) > 1 && table.stride(1) != 1))
    return false;
  if (q_start && (!on.here(*q_start) || q_start->scalar_type() != i32 || q_start->dim() != 1 ||
                  q_start->size(0) != batch + 1 || !q_start->is_contiguous()))
    return false;
  kv->k = k.data_ptr();
  kv->v = v.data_ptr();
  kv->pages = static_cast<size_t>(k.size(0));
  kv->n_kv = static_cast<size_t>(k.size(1));
  kv->page_size = static_cast<size_t>(k.size(2));
  kv->head_dim = static_cast<size_t>(k.size(3));
  kv->stride_page = static_cast<size_t>(k.stride(0));
  kv->stride_head = static_cast<size_t>(k.stride(1));
  kv->stride_token = static_cast<size_t>(k.stride(2));
  kv->block_table = static_cast<const int32_t*>(table.data_ptr());
  kv->batch = static_cast<size_t>(batch);
  kv->table_width = static_cast<size_t>(table.size(1));
  kv->ld_table = batch > 1 ? static_cast<size_t>(table.stride(0)) : kv->table_width;
  kv->seq_lens = static_cast<const int32_t*>(lens.data_ptr());
  kv->q_start = q_start ? static_cast<const int32_t*>(q_start->data_ptr()) : nullptr;
  return true;
}

// Token stride of a [tokens, heads, d] operand with dense heads; false where
// tokens share memory (a stride of 0 would mean "dense" to the C call).
bool heads_of(const at::Tensor& t, const On& on, c10::ScalarType type, int64_t tokens,
              int64_t heads, int64_t d, size_t* ld) {
  if (!on.here(t) || t.scalar_type() != type || t.dim() != 3 || t.size(0) != tokens ||
      t.size(1) != heads || t.size(2) != d)
    return false;
  if (t.numel() > 0 && (t.stride(2) != 1 || (heads > 1 && t.stride(1) != d))) return false;
  if (tokens > 1 && t.stride(0) < heads * d) return false;
  *ld = static_cast<size_t>(tokens > 1 ? t.stride(0) : heads * d);
  return true;
}

bool half_code(const at::Tensor& q, cawq_dtype* code) {
  return q.is_cuda() && q.dim() == 3 && float_code(q.scalar_type(), code) && *code != CAWQ_F32;
}

py::object rope_append(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                       const at::Tensor& rope, const at::Tensor& k_cache,
                       const at::Tensor& v_cache, const at::Tensor& table, const at::Tensor& lens,
                       const OptTensor& q_start, const OptTensor& out_) {
  cawq_dtype code;
  if (!half_code(q, &code)) return py::none();
  const On on{q.get_device()};
  const auto type = q.scalar_type();
  cawq_paged_kv kv;
  if (!paged(k_cache, v_cache, table, lens, q_start, on, type, &kv)) return py::none();
  const int64_t tokens = q.size(0), n_q = q.size(1), n_kv = k_cache.size(1), d = k_cache.size(3);
  size_t ld_q, ld_k, ld_v, ld_o;
  if (!heads_of(q, on, type, tokens, n_q, d, &ld_q) ||
      !heads_of(k, on, type, tokens, n_kv, d, &ld_k) ||
      !heads_of(v, on, type, tokens, n_kv, d, &ld_v) || !on.here(rope) ||
      rope.scalar_type() != c10::ScalarType::Float || rope.dim() != 2 || rope.size(1) != d ||
      !rope.is_contiguous())
    return py::none();
  const c10::cuda::CUDAGuard guard(on.device);
  at::Tensor out = out_ ? *out_ : at::empty(q.sizes(), q.options());
  if (!heads_of(out, on, type, tokens, n_q, d, &ld_o)) return py::none();
  const cawq_status st = cawq_rope_append(
      q.data_ptr(), k.data_ptr(), v.data_ptr(), static_cast<const float*>(rope.data_ptr()),
      static_cast<size_t>(rope.size(0)), out.data_ptr(), &kv, static_cast<size_t>(tokens),
      static_cast<size_t>(n_q), ld_q, ld_k, ld_v, ld_o, code,
      c10::cuda::getCurrentCUDAStream(on.device).stream());
  if (st != CAWQ_OK) return py::int_(static_cast<int>(st));
  return py::cast(out);
}

// q_start: attention_prefill; without it: attention_decode
py::object attention(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                     const at::Tensor& table, const at::Tensor& lens, const OptTensor& q_start,
                     c10::optional<double> scale, c10::optional<int64_t> window, int64_t sinks,
                     const OptTensor& out_) {
  cawq_dtype code;
  const int64_t win = window.value_or(0);
  if (!half_code(q, &code) || win < 0 || sinks < 0) return py::none();
  const On on{q.get_device()};
  const auto type = q.scalar_type();
  cawq_paged_kv kv;
  if (!paged(k_cache, v_cache, table, lens, q_start, on, type, &kv)) return py::none();
  const int64_t tokens = q.size(0), n_q = q.size(1), d = k_cache.size(3);
  size_t ld_q, ld_o;
  if (!heads_of(q, on, type, tokens, n_q, d, &ld_q) || (!q_start && tokens != lens.size(0)))
    return py::none();
  const c10::cuda::CUDAGuard guard(on.device);
  at::Tensor out = out_ ? *out_ : at::empty(q.sizes(), q.options());
  if (!heads_of(out, on, type, tokens, n_q, d, &ld_o)) return py::none();
  // from torch's allocator on the current stream, so it is this call's alone
  const size_t need =
      cawq_attention_workspace(&kv, static_cast<size_t>(tokens), static_cast<size_t>(n_q));
  at::Tensor ws;
  if (need)
    ws = at::empty({static_cast<int64_t>(need)}, q.options().dtype(c10::ScalarType::Byte));
  void* wp = need ? ws.data_ptr() : nullptr;
  const float sc =
      static_cast<float>(scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(d)));
  void* s = c10::cuda::getCurrentCUDAStream(on.device).stream();
  const size_t nq = static_cast<size_t>(n_q);
  const cawq_status st =
      q_start ? cawq_attention_prefill(q.data_ptr(), out.data_ptr(), &kv,
                                       static_cast<size_t>(tokens), nq, ld_q, ld_o, sc,
                                       static_cast<size_t>(win), static_cast<size_t>(sinks), code,
                                       wp, need, s)
              : cawq_attention_decode(q.data_ptr(), out.data_ptr(), &kv, nq, ld_q, ld_o, sc,
                                      static_cast<size_t>(win), static_cast<size_t>(sinks), code,
                                      wp, need, s);
  if (st != CAWQ_OK) return py::int_(static_cast<int>(st));
  return py::cast(out);
}

}  // namespace

PYBIND11_MODULE(_cawq_torch, m) {
  m.doc() = "compiled host path of the cube_awq_b200 module forward";
  py::class_<Layer>(m, "Layer")
      .def(py::init<at::Tensor, at::Tensor, at::Tensor, c10::optional<at::Tensor>, int64_t,
                    int64_t>(),
           py::arg("qweight"), py::arg("qzeros"), py::arg("scales"), py::arg("bias"),
           py::arg("group_size"), py::arg("order"))
      .def("forward", &Layer::forward);
  m.def("rms_norm", [](const at::Tensor& x, const at::Tensor& w, double eps, const OptTensor& r,
                       const OptTensor& out, const OptTensor& res_out) {
    return rms_norm_any(x, w, eps, r, out, c10::nullopt, res_out, false);
  });
  m.def("rms_norm_fp8", [](const at::Tensor& x, const at::Tensor& w, double eps,
                           const OptTensor& r, const OptTensor& out, const OptTensor& scales,
                           const OptTensor& res_out) {
    return rms_norm_any(x, w, eps, r, out, scales, res_out, true);
  });
  m.def("rope_append", &rope_append);
  m.def("attention", &attention);
}
