// Entry points of the attention over a window of nodes: checks, and which kernels take a call.
#include <cmath>

#include "attention.cuh"

namespace ocnn {
namespace {

int size_of(int dtype) { return dtype == OCNN_F32 ? 4 : 2; }

int check(const ocnn_attention* a, const char* who) {
  OCNN_REQUIRE(a != nullptr, "%s: null pointer", who);
  OCNN_REQUIRE(a->n >= 0 && a->n <= INT_MAX - 1024 && a->batch >= 0 && a->heads >= 1 && a->kv_heads >= 1 && a->dim >= 1, "%s: bad sizes", who);
  OCNN_REQUIRE(a->dtype >= OCNN_F32 && a->dtype <= OCNN_F16, "%s: bad dtype %d", who, a->dtype);
  OCNN_REQUIRE(a->heads % a->kv_heads == 0, "%s: %d heads over %d key heads", who, a->heads, a->kv_heads);
  OCNN_REQUIRE(a->window >= 0 && a->sinks >= 0, "%s: window and sinks must not be negative", who);
  if (a->dim > kMaxHeadDim || a->sinks > kMaxSinks)
    return fail(OCNN_ERR_UNSUPPORTED, "%s: heads of %d channels with %d first nodes (up to %d and %d)", who, a->dim,
                a->sinks, kMaxHeadDim, kMaxSinks);
  if (a->batch > kMaxSequences || a->heads > 65535)                   // (heads: the grid's y)
    return fail(OCNN_ERR_UNSUPPORTED, "%s: %d sequences, %d heads (up to %d and 65535)", who, a->batch, a->heads, kMaxSequences);
  OCNN_REQUIRE(a->n == 0 || (a->q_dev && a->k_dev && a->v_dev && a->offsets_dev), "%s: null pointer", who);
  return OCNN_OK;
}

AttnArgs args_of(const ocnn_attention* p) {
  AttnArgs a = {};
  a.q = p->q_dev, a.q_row = p->q_stride[0], a.q_head = p->q_stride[1];
  a.k = p->k_dev, a.k_row = p->k_stride[0], a.k_head = p->k_stride[1];
  a.v = p->v_dev, a.v_row = p->v_stride[0], a.v_head = p->v_stride[1];
  a.offsets = p->offsets_dev, a.mask = p->mask_dev;
  a.batch = p->batch, a.n = p->n, a.heads = p->heads, a.kv_heads = p->kv_heads, a.dim = p->dim;
  // a window as long as the batch is none
  a.window = p->window == 0 || p->window > p->n ? p->n : p->window;
  a.sinks = a.window == p->n ? 0 : p->sinks;
  a.causal = p->causal != 0;
  a.scale = p->scale;
  a.scale_log2 = p->scale * 1.4426950408889634f;
  return a;
}

// Whether rows of `elements` values can be read from p at these strides in one access each.
bool on_boundary(const void* p, const int64_t stride[2], int dim, int elements, int size) {
  return reinterpret_cast<uintptr_t>(p) % (elements * size) == 0 && stride[0] % elements == 0 &&
         stride[1] % elements == 0 && dim % elements == 0;
}
bool all_on_boundary(const ocnn_attention* a, int elements) {
  const int size = size_of(a->dtype);
  return on_boundary(a->q_dev, a->q_stride, a->dim, elements, size) &&
         on_boundary(a->k_dev, a->k_stride, a->dim, elements, size) &&
         on_boundary(a->v_dev, a->v_stride, a->dim, elements, size);
}

// 16-bit rows in whole pieces of 16 bytes, at strides that a tensor map takes (positive, below 2^40 bytes; nodes up to 2^31
// bytes apart, others run on the CUDA cores), and a positive scale (a tile's maximum is taken before it).
bool map_strides(const int64_t stride[2], int n, int heads) {
  return (n == 1 || (stride[0] > 0 && stride[0] < (1 << 30))) && (heads == 1 || (stride[1] > 0 && stride[1] < (1LL << 38)));
}
bool on_tensor_cores(const ocnn_attention* a) {
  return a->dtype != OCNN_F32 && all_on_boundary(a, 8) && a->scale > 0.f && a->scale < INFINITY &&
         map_strides(a->q_stride, a->n, a->heads) && map_strides(a->k_stride, a->n, a->kv_heads) &&
         map_strides(a->v_stride, a->n, a->kv_heads);
}

size_t chunk_words(const ocnn_attention* a) { return ((size_t)grad_chunks(a->n) + 31) / 32 * 32; }
size_t delta_floats(const ocnn_attention* a) { return ((size_t)a->heads * a->n + 31) / 32 * 32; }

}  // namespace
}  // namespace ocnn

using namespace ocnn;

extern "C" {

int ocnn_octree_attention(const ocnn_attention* p, void* out_dev, float* lse_dev, int32_t* status_dev, void* stream) {
  const int status = check(p, "ocnn_octree_attention");
  if (status != OCNN_OK || p->n == 0) return status;
  OCNN_REQUIRE(out_dev && status_dev, "ocnn_octree_attention: null pointer");
  const AttnArgs a = args_of(p);
  if (on_tensor_cores(p) && (reinterpret_cast<uintptr_t>(out_dev) | reinterpret_cast<uintptr_t>(lse_dev)) % 16 == 0)
    return attn_tc_forward(a, p->dtype, out_dev, lse_dev, status_dev, (cudaStream_t)stream);
  return attn_simt_forward(a, p->dtype, out_dev, lse_dev, all_on_boundary(p, 4), (cudaStream_t)stream);
}

size_t ocnn_octree_attention_saved_bytes(const ocnn_attention* p) {
  if (check(p, "ocnn_octree_attention_saved_bytes") != OCNN_OK || p->n == 0) return 0;
  const AttnArgs a = args_of(p);
  return attn_lse_floats(a) * sizeof(float) + (p->dtype == OCNN_F32 ? 0 : (size_t)a.n * a.heads * a.dim * 2);
}

size_t ocnn_octree_attention_backward_workspace_bytes(const ocnn_attention* p) {
  if (check(p, "ocnn_octree_attention_backward_workspace_bytes") != OCNN_OK || p->n == 0) return 0;
  const AttnArgs a = args_of(p);
  return (chunk_words(p) + delta_floats(p) + (size_t)far_slots(a) * a.kv_heads * a.sinks * 2 * a.dim) * sizeof(float);
}

int ocnn_octree_attention_backward(const ocnn_attention* p, const void* out_dev, const float* lse_dev,
                                   const void* grad_dev, const int64_t grad_stride[2], void* dq_dev, void* dk_dev,
                                   void* dv_dev, void* workspace_dev, size_t workspace_bytes, int32_t* status_dev,
                                   void* stream) {
  const int status = check(p, "ocnn_octree_attention_backward");
  if (status != OCNN_OK || p->n == 0) return status;
  OCNN_REQUIRE(out_dev && lse_dev && grad_dev && grad_stride && dq_dev && (dk_dev == nullptr) == (dv_dev == nullptr) && status_dev,
               "ocnn_octree_attention_backward: null pointer");
  const size_t need = ocnn_octree_attention_backward_workspace_bytes(p);
  if (workspace_dev == nullptr || workspace_bytes < need)
    return fail(OCNN_ERR_CAPACITY, "ocnn_octree_attention_backward: %zu bytes of workspace are needed", need);
  const AttnArgs a = args_of(p);
  AttnGrad g = {};
  g.out = out_dev, g.grad = grad_dev, g.grad_row = grad_stride[0], g.grad_head = grad_stride[1];
  g.lse = lse_dev;
  g.largest = (unsigned*)workspace_dev;
  g.delta = (float*)workspace_dev + chunk_words(p);
  g.far = g.delta + delta_floats(p);
  g.dq = dq_dev, g.dk = dk_dev, g.dv = dv_dev;
  if (on_tensor_cores(p) && map_strides(grad_stride, a.n, a.heads) && on_boundary(grad_dev, grad_stride, p->dim, 8, 2) &&
      (reinterpret_cast<uintptr_t>(out_dev) | reinterpret_cast<uintptr_t>(lse_dev) | reinterpret_cast<uintptr_t>(dq_dev) |
       reinterpret_cast<uintptr_t>(dk_dev) | reinterpret_cast<uintptr_t>(dv_dev)) % 16 == 0)
    return attn_tc_backward(a, g, p->dtype, status_dev, (cudaStream_t)stream);
  const bool vec = all_on_boundary(p, 4) && on_boundary(grad_dev, grad_stride, p->dim, 4, size_of(p->dtype)) &&
                   reinterpret_cast<uintptr_t>(out_dev) % (4 * size_of(p->dtype)) == 0;
  return attn_simt_backward(a, g, p->dtype, vec, (cudaStream_t)stream);
}

}  // extern "C"
