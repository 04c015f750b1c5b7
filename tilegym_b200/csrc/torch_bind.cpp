// The ordinary call of the decode-time operators without Python's share of it: tensors are looked at, outputs allocated and
// descriptors filled in C++, then the C entry point is called.  Every function here returns None for whatever is not
// ordinary - another type, a layout that needs a copy, inputs that want gradients, an error code - and the caller goes on with
// the Python path, which has the checks, the copies and the errors.  One decode-sized call takes 5.5 to 7 us of host time instead of 13 to 18.
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>

#include <optional>

#include "../../include/tilegym_b200.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

int32_t code_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return TG_F32;
    case at::kHalf: return TG_F16;
    case at::kBFloat16: return TG_BF16;
    case at::kInt: return TG_I32;
    case at::kLong: return TG_I64;
    case at::kFloat8_e4m3fn: return TG_F8E4M3;
    case at::kDouble: return TG_F64;
    default: return -1;
  }
}

struct Desc {
  TgTensorDesc d = {};
  const TgTensorDesc* p = nullptr;
  Desc() = default;
  explicit Desc(const Tensor& t) { fill(t); }
  explicit Desc(const OptTensor& t) {
    if (t) fill(*t);
  }
  Desc(const Tensor& t, int64_t rows, int64_t cols) {  // a contiguous tensor as a matrix
    d.ptr = reinterpret_cast<uint64_t>(t.data_ptr());
    d.ndim = 2;
    d.shape[0] = rows;
    d.shape[1] = d.strides[0] = cols;
    d.strides[1] = 1;
    d.dtype = code_of(t.scalar_type());
    p = &d;
  }
  Desc(const Desc&) = delete;
  Desc& operator=(const Desc&) = delete;
  void fill(const Tensor& t) {
    if (t.dim() > 5) return;
    d.ptr = reinterpret_cast<uint64_t>(t.data_ptr());
    d.ndim = static_cast<int32_t>(t.dim());
    for (int i = 0; i < d.ndim; ++i) {
      d.shape[i] = t.size(i);
      d.strides[i] = t.stride(i);
    }
    d.dtype = code_of(t.scalar_type());
    p = &d;
  }
};

bool is_16bit(const Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf; }
bool aligned(const Tensor& t) { return (reinterpret_cast<uint64_t>(t.data_ptr()) & 15u) == 0; }
bool wants_grad(const Tensor& t) { return (t.requires_grad() && at::GradMode::is_enabled()) || t._fw_grad(0).defined(); }  // or has a tangent
bool on(const Tensor& t, int64_t dev) { return t.is_cuda() && t.get_device() == dev; }
bool heads(const Tensor& t, int64_t dev) {
  return on(t, dev) && t.dim() == 3 && is_16bit(t) && t.stride(2) == 1 && t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 && aligned(t) && !wants_grad(t);
}
bool table(const Tensor& t, int64_t dev) { return on(t, dev) && t.scalar_type() == at::kInt && t.is_contiguous(); }
uint64_t stream_of(int64_t dev) { return reinterpret_cast<uint64_t>(c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream()); }
// The C call without the interpreter's lock: a launch may wait for room in a full queue, and other threads go on meanwhile.
template <typename F>
int32_t unlocked(F&& call) {
  py::gil_scoped_release released;
  return call();
}
Tensor like(const Tensor& t) { return at::empty(t.sizes(), t.options()); }

struct Cache {
  Desc k, v, ks, vs;
  Cache(const Tensor& a, const Tensor& b, const Tensor& c, const Tensor& d) : k(a), v(b), ks(c), vs(d) {}
};
bool cache_on(const Tensor& a, const Tensor& b, const Tensor& c, const Tensor& d, int64_t dev) { return on(a, dev) && on(b, dev) && on(c, dev) && on(d, dev); }

py::object rms_norm_quant(const Tensor& x, const Tensor& w, double eps, const OptTensor& residual, double offset, bool inplace) {
  if (!x.is_cuda() || !is_16bit(x) || x.dim() < 1 || !x.is_contiguous() || !aligned(x) || wants_grad(x)) return py::none();
  const int64_t dev = x.get_device(), hidden = x.size(-1);
  if (hidden < 128 || hidden % 128 != 0 || !on(w, dev) || w.dim() != 1 || w.size(0) != hidden || !w.is_contiguous() || !aligned(w)) return py::none();
  if (inplace && !residual) return py::none();
  if (residual && (!on(*residual, dev) || residual->scalar_type() != x.scalar_type() || residual->sizes() != x.sizes() ||
                   !residual->is_contiguous() || !aligned(*residual) || wants_grad(*residual)))
    return py::none();
  const int64_t rows = x.numel() / hidden;
  auto sizes = x.sizes().vec();
  Tensor y = at::empty(sizes, x.options().dtype(at::kFloat8_e4m3fn));
  sizes.back() = hidden / 128;
  Tensor s = at::empty(sizes, x.options().dtype(at::kFloat));
  Tensor h;
  if (residual) h = inplace ? *residual : like(x);
  const Desc dy(y, rows, hidden), ds(s, rows, hidden / 128), dx(x, rows, hidden), dw(w);
  std::optional<Desc> dh, dr;
  if (residual) {
    dh.emplace(h, rows, hidden);
    dr.emplace(*residual, rows, hidden);
  }
  const int32_t rc = unlocked([&] {
    return tg_rms_norm_quant(dy.p, ds.p, dh ? dh->p : nullptr, dx.p, dr ? dr->p : nullptr, dw.p, static_cast<float>(eps),
                             static_cast<float>(offset), static_cast<int32_t>(dev), stream_of(dev));
  });
  if (rc != TG_OK) return py::none();
  if (residual) return py::make_tuple(y, s, h);
  return py::make_tuple(y, s);
}

py::object apply_rope(const Tensor& q, const OptTensor& k, const Tensor& positions, const Tensor& inv_freq, bool interleaved, double magnitude,
                      bool inplace) {
  if (!q.is_cuda()) return py::none();
  const int64_t dev = q.get_device();
  if (!heads(q, dev) || (k && !heads(*k, dev)) || !on(positions, dev) || !positions.is_contiguous() || !on(inv_freq, dev) ||
      inv_freq.scalar_type() != at::kDouble || !inv_freq.is_contiguous())
    return py::none();
  const Tensor qo = inplace ? q : like(q);
  const OptTensor ko = !k ? OptTensor() : OptTensor(inplace ? *k : like(*k));
  const Desc dqo(qo), dko(ko), dq(q), dk(k), dp(positions), df(inv_freq);
  const int32_t rc = unlocked([&] {
    return tg_apply_rope(dqo.p, dko.p, dq.p, dk.p, dp.p, df.p, interleaved, static_cast<float>(magnitude), static_cast<int32_t>(dev),
                         stream_of(dev));
  });
  if (rc != TG_OK) return py::none();
  return py::make_tuple(qo, ko);
}

// (rotated queries or None,), or None
py::object kv_cache_write(const Tensor& kc, const Tensor& vc, const Tensor& ks, const Tensor& vs, const Tensor& k, const Tensor& v, const Tensor& block_table,
                          const Tensor& seq_lens, const OptTensor& cu, const OptTensor& inv_freq, const OptTensor& q, bool interleaved, double magnitude) {
  if (!k.is_cuda()) return py::none();
  const int64_t dev = k.get_device();
  if (!heads(k, dev) || !heads(v, dev) || !cache_on(kc, vc, ks, vs, dev) || !table(block_table, dev) || !table(seq_lens, dev) ||
      (cu && !table(*cu, dev)) || (q && !heads(*q, dev)) ||
      (inv_freq && (!on(*inv_freq, dev) || inv_freq->scalar_type() != at::kDouble || !inv_freq->is_contiguous())))
    return py::none();
  const OptTensor qo = q ? OptTensor(like(*q)) : OptTensor();
  const Cache c(kc, vc, ks, vs);
  const Desc dk(k), dv(v), dt(block_table), dl(seq_lens), dc(cu), dqo(qo), dq(q), df(inv_freq);
  const int32_t rc = unlocked([&] {
    return tg_kv_cache_write(c.k.p, c.v.p, c.ks.p, c.vs.p, dk.p, dv.p, dt.p, dl.p, dc.p, dqo.p, dq.p, df.p, interleaved,
                             static_cast<float>(magnitude), static_cast<int32_t>(dev), stream_of(dev));
  });
  if (rc != TG_OK) return py::none();
  return py::make_tuple(qo);
}

py::object paged_attention(const Tensor& q, const Tensor& kc, const Tensor& vc, const Tensor& ks, const Tensor& vs, const Tensor& block_table,
                           const Tensor& seq_lens, const OptTensor& cu, int64_t max_q_len, double scale, int64_t window, int64_t sinks,
                           const OptTensor& out, int64_t workspace_bytes) {
  if (!q.is_cuda()) return py::none();
  const int64_t dev = q.get_device(), top = 0x7fffffff;
  if (!heads(q, dev) || !cache_on(kc, vc, ks, vs, dev) || !table(block_table, dev) || !table(seq_lens, dev) || (cu && !table(*cu, dev)) ||
      (out && (!on(*out, dev) || out->sizes() != q.sizes())) || max_q_len < 1 || max_q_len > top || window < 0 || window > top || sinks < 0 || sinks > top)
    return py::none();
  const Tensor o = out ? *out : like(q);
  Tensor ws;
  if (workspace_bytes > 0) ws = at::empty({workspace_bytes}, q.options().dtype(at::kByte));
  const Cache c(kc, vc, ks, vs);
  const Desc dq(q), dout(o), dt(block_table), dl(seq_lens), dc(cu);
  const int32_t rc = unlocked([&] {
    return tg_paged_attention(dout.p, dq.p, c.k.p, c.v.p, c.ks.p, c.vs.p, dt.p, dl.p, dc.p, static_cast<int32_t>(max_q_len),
                              static_cast<float>(scale), static_cast<int32_t>(window), static_cast<int32_t>(sinks),
                              workspace_bytes > 0 ? reinterpret_cast<uint64_t>(ws.data_ptr()) : 0, static_cast<uint64_t>(workspace_bytes),
                              static_cast<int32_t>(dev), stream_of(dev));
  });
  if (rc != TG_OK) return py::none();
  return py::cast(o);
}

}  // namespace

PYBIND11_MODULE(_bind, m) {
  m.attr("torch_version") = TG_TORCH_VERSION;  // the one it was built for: it is not called under another
  m.def("rms_norm_quant", &rms_norm_quant);
  m.def("apply_rope", &apply_rope);
  m.def("kv_cache_write", &kv_cache_write);
  m.def("paged_attention", &paged_attention);
}
