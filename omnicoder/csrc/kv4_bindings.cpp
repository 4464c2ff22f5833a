// Tensor-level bindings of the 4-bit key / value cache kernels: every shape,
// type, stride and device is checked here; the kernels assume them.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "kv4.h"

namespace omni {

namespace {

using OptTensor = c10::optional<at::Tensor>;

// at::empty without the dispatcher: 0.25 us less of the 4 to 6 that a call takes on the host.
at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const at::Device& dev) {
  return at::detail::empty_cuda(sizes, type, dev, c10::nullopt);
}

cudaStream_t stream() { return at::cuda::getCurrentCUDAStream().stream(); }

int kv4_type(at::ScalarType t, const char* what) {
  if (t == at::kFloat) return KV4_F32;
  if (t == at::kHalf) return KV4_F16;
  TORCH_CHECK(t == at::kBFloat16, what, ": fp32, fp16 or bf16 values");
  return KV4_BF16;
}

bool is_pos64(const at::Tensor& t, const char* what) {
  TORCH_CHECK(t.scalar_type() == at::kLong || t.scalar_type() == at::kInt, what, ": int32 or int64 positions");
  return t.scalar_type() == at::kLong;
}

// The kernels copy 16-byte pieces of whole rows, and 32 rows at a time.
Kv4Cache cache_of(const at::Tensor& c, const at::Tensor& p, const at::Device& dev, const char* what) {
  TORCH_CHECK(c.is_cuda() && c.device() == dev && p.device() == dev, what, ": cache tensors on ", dev);
  TORCH_CHECK(c.scalar_type() == at::kByte && c.dim() == 4 && p.scalar_type() == at::kBFloat16 && p.dim() == 5 &&
                  p.size(4) == 2 && p.size(0) == c.size(0) && p.size(1) == c.size(1) && p.size(2) == c.size(2),
              what, ": codes uint8 [B, Hk, L, W / 2], params bf16 [B, Hk, L, W / g, 2]");
  const int64_t W = 2 * c.size(3), G = p.size(3);
  TORCH_CHECK(G > 0 && W % G == 0 && (W / G == 16 || W / G == 32 || W / G == 64) && W <= 1024, what,
              ": rows of at most 1024 dims in groups of 16, 32 or 64");
  TORCH_CHECK(c.size(2) % 32 == 0 && c.size(2) < (1 << 30), what, ": the number of rows must be a multiple of 32");
  TORCH_CHECK(c.stride(3) == 1 && c.stride(2) == c.size(3) && p.stride(4) == 1 && p.stride(3) == 2 &&
                  p.stride(2) == 2 * G,
              what, ": the rows of a head must be contiguous");
  Kv4Cache o{reinterpret_cast<uint8_t*>(c.data_ptr()), reinterpret_cast<uint8_t*>(p.data_ptr()), c.stride(0),
             c.stride(1), 2 * p.stride(0), 2 * p.stride(1)};
  const uintptr_t places = reinterpret_cast<uintptr_t>(o.codes) | reinterpret_cast<uintptr_t>(o.params) |
                           (uintptr_t)o.c_b | (uintptr_t)o.c_h | (uintptr_t)o.p_b | (uintptr_t)o.p_h;
  TORCH_CHECK(c.numel() == 0 || places % 16 == 0, what, ": heads and sequences must start on 16-byte boundaries");
  return o;
}

void fill_io(Kv4IO& a, const at::Tensor& pos, const at::Tensor& kc, const at::Tensor& kp, const OptTensor& vc,
             const OptTensor& vp, int64_t row_offset, const char* what) {
  const auto dev = kc.device();
  a.cache[0] = cache_of(kc, kp, dev, what);
  a.count = 1;
  if (vc.has_value()) {
    TORCH_CHECK(vp.has_value() && vc->sizes() == kc.sizes() && vp->sizes() == kp.sizes(), what,
                ": k and v caches of one shape");
    a.cache[1] = cache_of(*vc, *vp, dev, what);
    a.count = 2;
  }
  a.pos64 = is_pos64(pos, what);
  TORCH_CHECK(pos.dim() == 2 && pos.device() == dev && pos.is_contiguous() && pos.size(0) == kc.size(0), what,
              ": contiguous positions [B, T] on the cache's device");
  a.pos = pos.data_ptr();
  a.B = (int)kc.size(0);
  a.T = (int)pos.size(1);
  a.Hk = (int)kc.size(1);
  a.L = (int)kc.size(2);
  a.W = 2 * (int)kc.size(3);
  a.group = a.W / (int)kp.size(3);
  a.row_offset = row_offset;
  TORCH_CHECK(kc.size(0) <= 65535 && pos.size(1) * kc.size(1) * (kc.size(3) / 4) < (int64_t(1) << 31), what,
              ": at most 65535 sequences and 2^34 values of one");
}

}  // namespace

void kv4_write_t(const at::Tensor& pos, const at::Tensor& k, const at::Tensor& kc, const at::Tensor& kp,
                 const OptTensor& v, const OptTensor& vc, const OptTensor& vp, int64_t row_offset) {
  const char* what = "kv4_write";
  const c10::cuda::CUDAGuard g(kc.device());
  TORCH_CHECK(v.has_value() == vc.has_value(), what, ": v together with its cache");
  for (const at::Tensor* t : {&kc, &kp, vc.has_value() ? &*vc : &kc, vp.has_value() ? &*vp : &kp})
    TORCH_CHECK(t->is_non_overlapping_and_dense() || (t->stride(0) != 0 && t->stride(1) != 0), what,
                ": sequences of an expanded cache share their rows");
  Kv4IO a{};
  at::Tensor p = pos.contiguous(), keep[2];
  fill_io(a, p, kc, kp, vc, vp, row_offset, what);
  TORCH_CHECK(a.count == 1 || a.cache[0].codes == nullptr ||
                  (a.cache[0].codes != a.cache[1].codes && a.cache[0].params != a.cache[1].params),
              what, ": k and v need caches of their own");
  a.type = kv4_type(k.scalar_type(), what);
  for (int i = 0; i < a.count; ++i) {
    at::Tensor x = i == 0 ? k : *v;
    TORCH_CHECK(x.device() == kc.device() && x.scalar_type() == k.scalar_type() && x.dim() == 4 && x.size(0) == a.B &&
                    x.size(1) == a.T && x.size(2) == a.Hk && x.size(3) == a.W,
                what, ": rows [B, T, Hk, W] of one type on the cache's device");
    const int64_t align = 16 / (int64_t)x.element_size();
    if (x.stride(3) != 1 || x.stride(0) % align || x.stride(1) % align || x.stride(2) % align ||
        reinterpret_cast<uintptr_t>(x.data_ptr()) % 16)
      x = x.clone(at::MemoryFormat::Contiguous);
    keep[i] = x;
    a.rows[i] = Kv4Rows{x.data_ptr(), x.stride(0), x.stride(1), x.stride(2)};
  }
  if (a.B == 0 || a.T == 0 || a.Hk == 0) return;
  kv4_write(a, stream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

std::vector<at::Tensor> kv4_read_t(const at::Tensor& pos, const at::Tensor& kc, const at::Tensor& kp,
                                   const OptTensor& vc, const OptTensor& vp, int64_t row_offset, at::ScalarType dtype) {
  const char* what = "kv4_read";
  const c10::cuda::CUDAGuard g(kc.device());
  Kv4IO a{};
  at::Tensor p = pos.contiguous();
  fill_io(a, p, kc, kp, vc, vp, row_offset, what);
  a.type = kv4_type(dtype, what);
  std::vector<at::Tensor> out;
  for (int i = 0; i < a.count; ++i) {
    out.push_back(empty({a.B, a.T, a.Hk, a.W}, dtype, kc.device()));
    a.rows[i] = Kv4Rows{out[i].data_ptr(), out[i].stride(0), out[i].stride(1), out[i].stride(2)};
  }
  if (a.B == 0 || a.T == 0 || a.Hk == 0) return out;
  kv4_read(a, stream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return out;
}

at::Tensor kv4_attend_t(const at::Tensor& q_in, const at::Tensor& kc, const at::Tensor& kp, const OptTensor& vc,
                        const OptTensor& vp, const at::Tensor& q_pos_in, const at::Tensor& kv_len_in, int64_t window,
                        double scale, int64_t latent_v_dim, int64_t sink_rows, int64_t n_sink) {
  const char* what = "decode_attention (4-bit cache)";
  const c10::cuda::CUDAGuard g(kc.device());
  at::Tensor q = q_in.contiguous(), q_pos = q_pos_in.contiguous(), kv_len = kv_len_in.contiguous();
  TORCH_CHECK(q.device() == kc.device() && q.dim() == 4, what, ": q [B, Tn, H, W] on the cache's device");
  TORCH_CHECK(q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf, what, ": q in bf16 or fp16");
  if (reinterpret_cast<uintptr_t>(q.data_ptr()) % 16) q = q.clone();
  Kv4Attend a{};
  a.q = q.data_ptr();
  a.type = kv4_type(q.scalar_type(), what);
  a.k = cache_of(kc, kp, kc.device(), what);
  a.B = (int)q.size(0);
  a.Tn = (int)q.size(1);
  a.H = (int)q.size(2);
  a.W = (int)q.size(3);
  a.Hk = (int)kc.size(1);
  a.L = (int)kc.size(2);
  a.group = 2 * (int)kc.size(3) / (int)kp.size(3);
  TORCH_CHECK(kc.size(0) == a.B && 2 * kc.size(3) == a.W && a.Hk > 0 && a.H % a.Hk == 0, what,
              ": codes [B, Hk, L, W / 2] of q's B and W, H a multiple of Hk");
  if (vc.has_value()) {
    TORCH_CHECK(latent_v_dim == 0 && vp.has_value() && vc->sizes() == kc.sizes() && vp->sizes() == kp.sizes(), what,
                ": k and v caches of one shape");
    a.v = cache_of(*vc, *vp, kc.device(), what);
    a.V = a.W;
  } else {
    TORCH_CHECK(a.Hk == 1 && latent_v_dim > 0 && latent_v_dim <= a.W && latent_v_dim % a.group == 0, what,
                ": a latent cache has one head and whole groups as its value");
    a.V = (int)latent_v_dim;
  }
  a.pos64 = is_pos64(q_pos, what);
  a.len64 = is_pos64(kv_len, what);
  TORCH_CHECK(q_pos.device() == kc.device() && q_pos.dim() == 2 && q_pos.size(0) == a.B && q_pos.size(1) == a.Tn &&
                  kv_len.device() == kc.device() && kv_len.dim() == 1 && kv_len.size(0) == a.B,
              what, ": q_pos [B, Tn] and kv_len [B] on the cache's device");
  TORCH_CHECK(0 <= n_sink && n_sink <= sink_rows && sink_rows <= a.L && window >= 0, what,
              ": 0 <= n_sink <= sink_rows <= L, window >= 0");
  TORCH_CHECK((int64_t)a.B * a.Tn * a.H < (int64_t(1) << 31) && a.B <= 65535, what, ": too many query rows");
  a.q_pos = q_pos.data_ptr();
  a.kv_len = kv_len.data_ptr();
  a.window = (int)std::min<int64_t>(window, 1 << 30);
  a.scale = (float)scale;
  a.sink_rows = (int)sink_rows;
  a.n_sink = (int)n_sink;
  auto out = empty({a.B, a.Tn, a.H, a.V}, q.scalar_type(), kc.device());
  if (out.numel() == 0) return out;
  if (a.L == 0) return out.zero_();
  a.out = out.data_ptr();
  const Kv4Plan plan = kv4_plan(a);
  at::Tensor ws;
  if (plan.floats > 0) {
    ws = empty({(int64_t)plan.floats}, at::kFloat, kc.device());
    a.part = ws.data_ptr<float>();
  }
  kv4_attend(a, plan, stream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return out;
}

void register_kv4(pybind11::module_& m) {
  m.def("kv4_write", &kv4_write_t);
  m.def("kv4_read", &kv4_read_t);
  m.def("kv4_attend", &kv4_attend_t);
}

}  // namespace omni
