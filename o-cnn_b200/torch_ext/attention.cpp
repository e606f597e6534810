// The operators of an attention layer over octree nodes, as `ocnn.nn` has them: rotary positions, the residual's addition
// with the root-mean-square norm, attention over a window of nodes and its form for one new node.  Each with its
// gradient as one native autograd node.  Data are rows of heads, [n, heads, dim], with any strides whose last is 1.
#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <cmath>
#include <vector>

#include "ocnn_b200.h"

torch::Tensor ocnn_tc_status(c10::Device device);      // (ocnn_nn.cpp)

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using std::vector;

#define OCNN_CALL(expr)                                                      \
  do {                                                                       \
    int status__ = (expr);                                                   \
    TORCH_CHECK(status__ == OCNN_OK, "ocnn_b200: ", ocnn_last_error());      \
  } while (0)

void* current_stream() { return at::cuda::getCurrentCUDAStream().stream(); }

int dtype_of(const Tensor& t, const char* who) {
  if (t.scalar_type() == torch::kFloat32) return OCNN_F32;
  if (t.scalar_type() == torch::kBFloat16) return OCNN_BF16;
  TORCH_CHECK(t.scalar_type() == torch::kFloat16, who, ": data must be float32, bfloat16 or float16");
  return OCNN_F16;
}

void need_like(const Tensor& t, const Tensor& like, const char* name, const char* who) {
  TORCH_CHECK(t.device() == like.device() && t.scalar_type() == like.scalar_type(), who, ": ", name, " is on ",
              t.device(), " in ", t.scalar_type(), ", the data on ", like.device(), " in ", like.scalar_type());
}

// The kernels read whole rows: the last dimension is contiguous, the others may have any stride that a view gives them.
// (An expanded tensor, one row for all, is written out: tiles are not fetched at strides of 0.)
Tensor rows_of(const Tensor& t) {
  bool ok = t.size(-1) == 1 || t.stride(-1) == 1;
  for (int i = 0; i + 1 < t.dim(); ++i) ok = ok && (t.stride(i) != 0 || t.size(i) == 1);
  return ok ? t : t.contiguous();
}

// Gradients are formed by kernels: they have no graph of their own.
void once_only(const char* who) {
  TORCH_CHECK(!at::GradMode::is_enabled(), who, ": its gradient cannot be differentiated again (create_graph)");
}

// Nor do forward-mode derivatives pass through them, and neither a tracer nor a torch.func transform would see what they do.
void plain_call(std::initializer_list<Tensor> tensors, const char* who) {
  constexpr c10::DispatchKeySet transforms = c10::DispatchKeySet(c10::DispatchKey::FuncTorchBatched) |
                                             c10::DispatchKeySet(c10::DispatchKey::FuncTorchGradWrapper);
  TORCH_CHECK(!torch::jit::tracer::isTracing(), who, ": it cannot be traced (torch.jit.trace)");
  for (const Tensor& t : tensors) {
    if (!t.defined()) continue;
    TORCH_CHECK(!t.key_set().has_any(transforms), who, ": it cannot be transformed (torch.func)");
    TORCH_CHECK(!t._fw_grad(0).defined(), who, ": it has no forward-mode derivative");
  }
}

Tensor empty_rows(const Tensor& like) { return torch::empty(like.sizes(), like.options()); }

// ---- rotary positions -----------------------------------------------------------------------------------------
Tensor rotary_call(const Tensor& data, const Tensor& positions, const Tensor& freqs, const vector<int64_t>& sections,
                   bool interleaved, bool inverse) {
  const char* who = "octree_rotary";
  TORCH_CHECK(data.is_cuda(), who, ": the data tensor must be a CUDA tensor (there is no CPU path)");
  TORCH_CHECK(data.dim() == 3, who, ": data must have shape [n, heads, dim]");
  const int dtype = dtype_of(data, who);
  int64_t pairs = 0;
  for (int64_t s : sections) {
    TORCH_CHECK(s >= 0 && s <= data.size(2) / 2, who, ": a section holds 0 to dim / 2 pairs of channels");
    pairs += s;
  }
  TORCH_CHECK(data.size(2) >= 2 && data.size(2) % 2 == 0 && pairs <= data.size(2) / 2, who, ": sections of ", pairs,
              " pairs in heads of ", data.size(2), " channels");
  TORCH_CHECK(positions.device() == data.device() && freqs.device() == data.device(), who,
              ": positions and freqs must be on the data's device");
  const bool f = positions.scalar_type() == torch::kFloat32;
  TORCH_CHECK(f || positions.scalar_type() == torch::kInt32, who, ": positions must be int32 or float32");
  TORCH_CHECK(positions.dim() == 2 && positions.size(0) == data.size(0) && positions.size(1) == (int64_t)sections.size(),
              who, ": positions must have shape [n, axes], one axis per section");
  TORCH_CHECK(freqs.scalar_type() == torch::kFloat64 && freqs.dim() == 1 && freqs.size(0) == pairs, who,
              ": freqs must hold one float64 per pair of channels");
  c10::cuda::CUDAGuard guard(data.device());
  const Tensor x = rows_of(data), pos = positions.contiguous(), fr = freqs.contiguous();
  Tensor y = empty_rows(data);
  if (x.numel() == 0) return y;
  const int64_t stride[2] = {x.stride(0), x.stride(1)};
  const vector<int> sec(sections.begin(), sections.end());
  OCNN_CALL(ocnn_octree_rotary(x.data_ptr(), stride, y.data_ptr(), pos.data_ptr(), f, fr.data_ptr<double>(),
                               (int)sec.size(), sec.data(), x.size(0), (int)x.size(1), (int)x.size(2), interleaved,
                               inverse, dtype, current_stream()));
  return y;
}

struct Rotary : public torch::autograd::Function<Rotary> {
  static Tensor forward(AutogradContext* ctx, const Tensor& data, const Tensor& positions, const Tensor& freqs,
                        const vector<int64_t>& sections, bool interleaved) {
    at::AutoDispatchBelowADInplaceOrView guard;
    ctx->save_for_backward({positions, freqs});
    ctx->saved_data["sections"] = sections;
    ctx->saved_data["interleaved"] = interleaved;
    return rotary_call(data, positions, freqs, sections, interleaved, false);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once_only("octree_rotary");
    const auto saved = ctx->get_saved_variables();
    return {rotary_call(grads[0], saved[0], saved[1], ctx->saved_data["sections"].toIntVector(),
                        ctx->saved_data["interleaved"].toBool(), true),
            Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor octree_rotary(const Tensor& data, const Tensor& positions, const Tensor& freqs, const vector<int64_t>& sections,
                     bool interleaved) {
  plain_call({data}, "octree_rotary");
  if (at::GradMode::is_enabled() && data.requires_grad())
    return Rotary::apply(data, positions, freqs, sections, interleaved);
  return rotary_call(data, positions, freqs, sections, interleaved, false);
}

// ---- residual and root-mean-square norm ---------------------------------------------------------------------------
// Rows of the last dimension, whatever the others: as [rows, channels] with one stride (a copy where there is none).
Tensor flat_rows(const Tensor& t) {
  if (t.dim() == 2) return rows_of(t);
  return t.contiguous().view({-1, t.size(-1)});
}

vector<Tensor> norm_call(const Tensor& data, const c10::optional<Tensor>& residual, const Tensor& weight, double eps) {
  const char* who = "add_rms_norm";
  TORCH_CHECK(data.is_cuda(), who, ": the data tensor must be a CUDA tensor (there is no CPU path)");
  TORCH_CHECK(data.dim() >= 1 && data.size(-1) >= 1, who, ": data must be rows of channels");
  const int dtype = dtype_of(data, who);
  const int64_t channels = data.size(-1);
  TORCH_CHECK(channels < (1LL << 31), who, ": too many channels");
  const bool has = residual.has_value() && residual->defined();
  if (has) {
    need_like(*residual, data, "the residual", who);
    TORCH_CHECK(residual->sizes() == data.sizes(), who, ": the residual's shape is not the data's");
  }
  TORCH_CHECK(weight.device() == data.device() && weight.dim() == 1 && weight.size(0) == channels, who,
              ": the weight must hold one value per channel, on the data's device");
  TORCH_CHECK(weight.scalar_type() == torch::kFloat32 || weight.scalar_type() == data.scalar_type(), who,
              ": the weight must be float32 or of the data's type");
  c10::cuda::CUDAGuard guard(data.device());
  const Tensor x = flat_rows(data), r = has ? flat_rows(*residual) : Tensor(), w = weight.contiguous();
  Tensor y = empty_rows(data), sum = has ? empty_rows(data) : Tensor();
  OCNN_CALL(ocnn_add_rms_norm(x.data_ptr(), x.stride(0), has ? r.data_ptr() : nullptr, has ? r.stride(0) : 0,
                              w.data_ptr(), dtype_of(w, who), has ? sum.data_ptr() : nullptr, y.data_ptr(), x.size(0),
                              (int)channels, (float)eps, dtype, current_stream()));
  return {y, sum};
}

struct AddRmsNorm : public torch::autograd::Function<AddRmsNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& data, const c10::optional<Tensor>& residual,
                               const Tensor& weight, double eps) {
    at::AutoDispatchBelowADInplaceOrView guard;
    vector<Tensor> out = norm_call(data, residual, weight, eps);
    const bool has = out[1].defined();
    ctx->save_for_backward({data, weight, has ? *residual : Tensor()});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["has"] = has;
    ctx->set_materialize_grads(false);
    if (!has) return {out[0]};
    return {out[0], out[1]};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const char* who = "add_rms_norm";
    once_only(who);
    const auto saved = ctx->get_saved_variables();
    const bool has = ctx->saved_data["has"].toBool();
    const Tensor& weight = saved[1];
    // (positions among the tensor inputs that were given)
    const bool need_x = ctx->needs_input_grad(0) || (has && ctx->needs_input_grad(1));
    const bool need_w = ctx->needs_input_grad(has ? 2 : 1);
    variable_list res(4);
    const Tensor gy = grads[0], gs = has ? grads[1] : Tensor();
    if ((!gy.defined() && !gs.defined()) || (!need_x && !need_w)) return res;
    c10::cuda::CUDAGuard guard(weight.device());
    const Tensor s = flat_rows(saved[0]), r = has ? flat_rows(saved[2]) : Tensor(), w = weight.contiguous();
    const int64_t rows = s.size(0), channels = s.size(1);
    const Tensor fy = gy.defined() ? flat_rows(gy) : Tensor(), fs = gs.defined() ? flat_rows(gs) : Tensor();
    Tensor g = need_x ? empty_rows(saved[0]) : Tensor(), gw = need_w ? torch::empty_like(w) : Tensor(), ws;
    const size_t bytes = need_w ? ocnn_add_rms_norm_backward_workspace_bytes((int)channels) : 0;
    if (bytes > 0) ws = torch::empty({(int64_t)bytes}, s.options().dtype(torch::kUInt8));
    OCNN_CALL(ocnn_add_rms_norm_backward(
        s.data_ptr(), s.stride(0), has ? r.data_ptr() : nullptr, has ? r.stride(0) : 0, w.data_ptr(), dtype_of(w, who), fy.defined() ? fy.data_ptr() : nullptr,
        fy.defined() ? fy.stride(0) : 0, fs.defined() ? fs.data_ptr() : nullptr, fs.defined() ? fs.stride(0) : 0,
        need_x ? g.data_ptr() : nullptr, need_w ? gw.data_ptr() : nullptr, rows, (int)channels,
        (float)ctx->saved_data["eps"].toDouble(), dtype_of(s, who), bytes > 0 ? ws.data_ptr() : nullptr, bytes,
        current_stream()));
    if (ctx->needs_input_grad(0)) res[0] = g;
    if (has && ctx->needs_input_grad(1)) res[1] = g;
    res[2] = gw;
    return res;
  }
};

// (norm, sum): sum is data + residual, data itself without a residual.
vector<Tensor> add_rms_norm(const Tensor& data, const c10::optional<Tensor>& residual, const Tensor& weight, double eps) {
  const bool has = residual.has_value() && residual->defined();
  plain_call({data, weight, has ? *residual : Tensor()}, "add_rms_norm");
  vector<Tensor> out;
  if (at::GradMode::is_enabled() && (data.requires_grad() || weight.requires_grad() || (has && residual->requires_grad())))
    out = AddRmsNorm::apply(data, residual, weight, eps);
  else
    out = norm_call(data, residual, weight, eps);
  return {out[0], has ? out[1] : data};
}

// ---- attention ------------------------------------------------------------------------------------------------------
struct Operands {
  Tensor q, k, v, offsets, mask;
  ocnn_attention a;
};

Operands operands(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& offsets, const Tensor& mask,
                  int64_t window, int64_t sinks, bool causal, double scale) {
  const char* who = "octree_attention";
  TORCH_CHECK(q.is_cuda(), who, ": the data tensor must be a CUDA tensor (there is no CPU path)");
  TORCH_CHECK(q.dim() == 3 && k.dim() == 3 && v.dim() == 3, who, ": q, k and v must have shape [n, heads, dim]");
  need_like(k, q, "k", who);
  need_like(v, q, "v", who);
  TORCH_CHECK(k.sizes() == v.sizes() && k.size(0) == q.size(0) && k.size(2) == q.size(2), who, ": q is ", q.sizes(),
              ", k ", k.sizes(), ", v ", v.sizes());
  TORCH_CHECK(q.size(1) >= 1 && k.size(1) >= 1 && q.size(1) % k.size(1) == 0, who, ": ", q.size(1), " heads over ",
              k.size(1), " key heads");
  TORCH_CHECK(q.size(2) >= 1 && q.size(2) <= 128, who, ": heads of ", q.size(2), " channels (1 to 128)");
  TORCH_CHECK(q.size(0) < (1LL << 31), who, ": too many nodes");
  TORCH_CHECK(window >= 0 && window < (1LL << 31) && sinks >= 0 && sinks <= 64, who, ": window ", window, " with ", sinks,
              " first nodes (0 or more; 0 to 64)");
  TORCH_CHECK(offsets.device() == q.device() && offsets.scalar_type() == torch::kInt32 && offsets.dim() == 1 &&
                  offsets.size(0) >= 1 && offsets.size(0) < (1LL << 31),
              who, ": offsets must hold batch + 1 int32 values, on the data's device");
  Operands o;
  o.q = rows_of(q);
  o.k = rows_of(k);
  o.v = rows_of(v);
  o.offsets = offsets.contiguous();
  if (mask.defined()) {
    TORCH_CHECK(mask.device() == q.device() && mask.scalar_type() == torch::kBool && mask.dim() == 1 &&
                    mask.size(0) == q.size(0),
                who, ": the mask must hold one bool per node, on the data's device");
    o.mask = mask.contiguous();
  }
  ocnn_attention& a = o.a;
  a = {};
  a.q_dev = o.q.data_ptr();
  a.k_dev = o.k.data_ptr();
  a.v_dev = o.v.data_ptr();
  for (int i = 0; i < 2; ++i) {
    a.q_stride[i] = o.q.stride(i);
    a.k_stride[i] = o.k.stride(i);
    a.v_stride[i] = o.v.stride(i);
  }
  a.offsets_dev = o.offsets.data_ptr<int32_t>();
  a.mask_dev = mask.defined() ? reinterpret_cast<const uint8_t*>(o.mask.data_ptr()) : nullptr;
  a.batch = (int)offsets.size(0) - 1;
  a.n = (int)q.size(0);
  a.heads = (int)q.size(1);
  a.kv_heads = (int)k.size(1);
  a.dim = (int)q.size(2);
  a.window = (int)window;
  a.sinks = (int)sinks;
  a.causal = causal;
  a.dtype = dtype_of(q, who);
  a.scale = (float)scale;
  return o;
}

Tensor attention_call(const Operands& o, Tensor* lse) {
  c10::cuda::CUDAGuard guard(o.q.device());
  const Tensor status = ocnn_tc_status(o.q.device());
  Tensor out = torch::empty({o.q.size(0), o.q.size(1), o.q.size(2)}, o.q.options());
  if (lse != nullptr)
    *lse = torch::empty({(int64_t)ocnn_octree_attention_saved_bytes(&o.a) / 4 + 1}, o.q.options().dtype(torch::kFloat32));
  OCNN_CALL(ocnn_octree_attention(&o.a, out.data_ptr(), lse != nullptr ? lse->data_ptr<float>() : nullptr,
                                  status.data_ptr<int32_t>(), current_stream()));
  return out;
}

struct Attention : public torch::autograd::Function<Attention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& offsets,
                        const c10::optional<Tensor>& mask, int64_t window, int64_t sinks, bool causal,
                        double scale) {
    at::AutoDispatchBelowADInplaceOrView guard;
    const Operands o = operands(q, k, v, offsets, mask.has_value() ? *mask : Tensor(), window, sinks, causal, scale);
    Tensor lse;
    Tensor out = attention_call(o, &lse);
    ctx->save_for_backward({q, k, v, offsets, mask.has_value() ? *mask : Tensor(), out, lse});
    ctx->saved_data["window"] = window;
    ctx->saved_data["sinks"] = sinks;
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["scale"] = scale;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once_only("octree_attention");
    const auto saved = ctx->get_saved_variables();
    const Operands o = operands(saved[0], saved[1], saved[2], saved[3], saved[4], ctx->saved_data["window"].toInt(),
                                ctx->saved_data["sinks"].toInt(), ctx->saved_data["causal"].toBool(),
                                ctx->saved_data["scale"].toDouble());
    c10::cuda::CUDAGuard guard(o.q.device());
    const Tensor g = rows_of(grads[0]), status = ocnn_tc_status(o.q.device());
    // (the queries' kernel forms what the keys' needs; keys and values are one kernel)
    const bool keys = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
    Tensor dq = empty_rows(saved[0]), dk = keys ? empty_rows(saved[1]) : Tensor(), dv = keys ? empty_rows(saved[2]) : Tensor();
    const size_t bytes = ocnn_octree_attention_backward_workspace_bytes(&o.a);
    const Tensor ws = torch::empty({(int64_t)bytes}, o.q.options().dtype(torch::kUInt8));
    const int64_t stride[2] = {g.stride(0), g.stride(1)};
    OCNN_CALL(ocnn_octree_attention_backward(&o.a, saved[5].data_ptr(), saved[6].data_ptr<float>(), g.data_ptr(), stride,
                                             dq.data_ptr(), keys ? dk.data_ptr() : nullptr, keys ? dv.data_ptr() : nullptr,
                                             ws.data_ptr(), bytes,
                                             status.data_ptr<int32_t>(), current_stream()));
    variable_list res(9);
    res[0] = dq;
    res[1] = dk;
    res[2] = dv;
    return res;
  }
};

Tensor octree_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& offsets, int64_t window,
                        int64_t sinks, bool causal, const c10::optional<Tensor>& mask, c10::optional<double> scale) {
  plain_call({q, k, v}, "octree_attention");
  const double s = scale.has_value() ? *scale : q.dim() == 3 && q.size(2) > 0 ? 1.0 / std::sqrt((double)q.size(2)) : 1.0;
  if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad()))
    return Attention::apply(q, k, v, offsets, mask, window, sinks, causal, s);
  return attention_call(operands(q, k, v, offsets, mask.has_value() ? *mask : Tensor(), window, sinks, causal, s), nullptr);
}

Tensor octree_attention_step(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& k_cache,
                             const Tensor& v_cache, const Tensor& lengths, int64_t window, int64_t sinks,
                             c10::optional<double> scale) {
  const char* who = "octree_attention_step";
  plain_call({q, k, v, k_cache, v_cache}, who);
  TORCH_CHECK(q.is_cuda(), who, ": the data tensor must be a CUDA tensor (there is no CPU path)");
  TORCH_CHECK(q.dim() == 3 && k.dim() == 3 && v.dim() == 3, who, ": q, k and v must have shape [batch, heads, dim]");
  TORCH_CHECK(!(at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad() ||
                                               k_cache.requires_grad() || v_cache.requires_grad())),
              who, ": it has no gradient (call it under torch.no_grad())");
  need_like(k, q, "k", who);
  need_like(v, q, "v", who);
  need_like(k_cache, q, "k_cache", who);
  need_like(v_cache, q, "v_cache", who);
  const int64_t b = q.size(0), kv = k.size(1), dim = q.size(2);
  TORCH_CHECK(k.sizes() == v.sizes() && k.size(0) == b && k.size(2) == dim, who, ": q is ", q.sizes(), ", k ", k.sizes(),
              ", v ", v.sizes());
  TORCH_CHECK(q.size(1) >= 1 && kv >= 1 && q.size(1) % kv == 0, who, ": ", q.size(1), " heads over ", kv, " key heads");
  TORCH_CHECK(k_cache.dim() == 4 && k_cache.sizes() == v_cache.sizes() && k_cache.size(0) == b && k_cache.size(1) >= 1 &&
                  k_cache.size(2) == kv && k_cache.size(3) == dim && k_cache.size(1) < (1LL << 31),
              who, ": the caches must have shape [batch, capacity, key heads, dim]: they are ", k_cache.sizes(), " and ",
              v_cache.sizes());
  const int64_t size = q.element_size();
  TORCH_CHECK(dim >= 1 && dim <= 128 && dim * size % 16 == 0, who, ": heads of ", dim,
              " channels (multiples of 16 bytes, up to 128 channels)");
  TORCH_CHECK(window >= 0 && window < (1LL << 31) && sinks >= 0 && sinks <= 64, who, ": window ", window, " with ", sinks,
              " first nodes (0 or more; 0 to 64)");
  TORCH_CHECK(lengths.device() == q.device() && lengths.scalar_type() == torch::kInt32 && lengths.dim() == 1 &&
                  lengths.size(0) == b,
              who, ": lengths must hold one int32 per sequence, on the data's device");
  auto aligned = [&](const Tensor& t) {
    bool ok = t.stride(-1) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
    for (int i = 0; i + 1 < t.dim(); ++i) ok = ok && t.stride(i) * size % 16 == 0;
    return ok;
  };
  // The caches are written in place: no copy can stand in for them, and no two of their places may be one.
  for (const Tensor* t : {&k_cache, &v_cache}) {
    TORCH_CHECK(aligned(*t), who, ": the caches' rows must be contiguous and start on 16-byte boundaries");
    TORCH_CHECK(at::has_internal_overlap(*t) != at::MemOverlap::Yes, who, ": the caches' places must not overlap");
  }
  TORCH_CHECK(k_cache.numel() == 0 || k_cache.data_ptr() != v_cache.data_ptr(), who, ": the caches are the same memory");
  c10::cuda::CUDAGuard guard(q.device());
  auto row = [&](const Tensor& t) { return aligned(t) ? t : t.clone(at::MemoryFormat::Contiguous); };
  const Tensor qr = row(q), kr = row(k), vr = row(v), len = lengths.contiguous();
  Tensor out = torch::empty({b, q.size(1), dim}, q.options());
  if (b == 0) return out;
  ocnn_attention_cache c = {};
  c.k_dev = k_cache.data_ptr();
  c.v_dev = v_cache.data_ptr();
  for (int i = 0; i < 3; ++i) {
    c.k_stride[i] = k_cache.stride(i);
    c.v_stride[i] = v_cache.stride(i);
  }
  c.lengths_dev = len.data_ptr<int32_t>();
  c.batch = (int)b;
  c.capacity = (int)k_cache.size(1);
  c.kv_heads = (int)kv;
  c.dim = (int)dim;
  c.dtype = dtype_of(q, who);
  const int64_t qs[2] = {qr.stride(0), qr.stride(1)}, ks[2] = {kr.stride(0), kr.stride(1)},
                vs[2] = {vr.stride(0), vr.stride(1)};
  OCNN_CALL(ocnn_octree_attention_step(&c, qr.data_ptr(), qs, kr.data_ptr(), ks, vr.data_ptr(), vs, out.data_ptr(),
                                       (int)q.size(1), (int)window, (int)sinks,
                                       (float)(scale.has_value() ? *scale : 1.0 / std::sqrt((double)dim)),
                                       current_stream()));
  for (const Tensor* t : {&k_cache, &v_cache})
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
  return out;
}

}  // namespace

void bind_attention(py::module_& m) {
  m.def("octree_rotary", &octree_rotary, py::arg("data"), py::arg("positions"), py::arg("freqs"), py::arg("sections"),
        py::arg("interleaved") = false);
  m.def("add_rms_norm", &add_rms_norm, py::arg("data"), py::arg("residual"), py::arg("weight"), py::arg("eps"));
  m.def("octree_attention", &octree_attention, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("offsets"),
        py::arg("window"), py::arg("sinks"), py::arg("causal"), py::arg("mask"), py::arg("scale"));
  m.def("octree_attention_step", &octree_attention_step, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("k_cache"),
        py::arg("v_cache"), py::arg("lengths"), py::arg("window"), py::arg("sinks"), py::arg("scale"));
}
