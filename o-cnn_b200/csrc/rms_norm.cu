// The residual's addition and the root-mean-square norm behind it, over rows of C channels:
//     s = x + r,   y = s * rsqrt(mean(s^2) + eps) * w
// and the gradient, with u = s * rsqrt(...), from gy and gs:
//     g = gs + rsqrt(...) * (w gy - u mean(w gy u)),   gw = sum over rows of gy u
// (g is the gradient of both x and r).  Sums are held in fp32, and s is never rounded before it is used: the backward pass
// reads x and r again, not the s that was stored (one row more; from a bf16 s the weight's gradient, which is fp32,
// was off by 1.9e-3).  It forms the statistics anew, in the same pass over the row as the mean of w gy u, so nothing is
// kept between the two.
//
// Bound: HBM.  Forward 2 rows read and 2 written, backward 4 read and 1 written.  A row is taken by as few lanes as hold
// it in one vector each (8 channels of 16 bits or 4 of 32), so that a warp has several rows in flight and the statistics are
// a few shuffles; wider ones by a warp with two or four vectors a lane, one of more than 4 vectors x 32 lanes by a block,
// and one that even a block cannot keep in registers is read twice (the second time from L2).  gw: every thread keeps the sums of its own channels over
// the rows of its block, a block's sums go to a slot of the workspace, and a second launch adds the slots in order.
#include <atomic>

#include "common.cuh"

namespace ocnn {
namespace {

constexpr int kNormThreads = 256;

struct NormArgs {
  const void *x, *r, *w, *gy, *gs;
  void *sum, *y, *g;
  long long rows, x_row, r_row, gy_row, gs_row;
  float* partial;
  int channels, w_f32;
  float eps;
};

template <typename T, int V>
struct alignas(sizeof(T) * V) NormPack { T x[V]; };
__device__ __forceinline__ float norm_f32(float x) { return x; }
__device__ __forceinline__ float norm_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float norm_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ void norm_set(float& y, float x) { y = x; }
__device__ __forceinline__ void norm_set(__nv_bfloat16& y, float x) { y = __float2bfloat16(x); }
__device__ __forceinline__ void norm_set(__half& y, float x) { y = __float2half(x); }

template <typename T, int V>
__device__ __forceinline__ void norm_load(const void* base, long long at, float (&f)[V]) {
  const NormPack<T, V> p = *reinterpret_cast<const NormPack<T, V>*>((const T*)base + at);
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = norm_f32(p.x[i]);
}
template <typename T, int V>
__device__ __forceinline__ void norm_store(void* base, long long at, const float (&f)[V]) {
  NormPack<T, V> p;
#pragma unroll
  for (int i = 0; i < V; ++i) norm_set(p.x[i], f[i]);
  *reinterpret_cast<NormPack<T, V>*>((T*)base + at) = p;
}
template <typename T, int V>
__device__ __forceinline__ void norm_weight(const NormArgs& a, int c, float (&f)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i)
    f[i] = a.w_f32 ? ((const float*)a.w)[c + i] : norm_f32(((const T*)a.w)[c + i]);
}

// x + r (x alone without r) of row i from channel c on
template <typename T, int V>
__device__ __forceinline__ void norm_sum(const NormArgs& a, long long i, int c, float (&s)[V]) {
  norm_load<T, V>(a.x, i * a.x_row + c, s);
  if (a.r == nullptr) return;
  float r[V];
  norm_load<T, V>(a.r, i * a.r_row + c, r);
#pragma unroll
  for (int e = 0; e < V; ++e) s[e] += r[e];
}

// Sums over the LANES threads of a row, to all of them.  LANES = kNormThreads: the whole block.
template <int LANES, int COUNT>
__device__ __forceinline__ void norm_reduce(float (&x)[COUNT]) {
  constexpr int W = LANES < 32 ? LANES : 32;
#pragma unroll
  for (int c = 0; c < COUNT; ++c)
#pragma unroll
    for (int m = W / 2; m > 0; m >>= 1) x[c] += __shfl_xor_sync(0xffffffffu, x[c], m);
  if constexpr (LANES > 32) {
    __shared__ float part[COUNT][LANES / 32];
    __syncthreads();
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int c = 0; c < COUNT; ++c) part[c][threadIdx.x >> 5] = x[c];
    __syncthreads();
#pragma unroll
    for (int c = 0; c < COUNT; ++c) {
      x[c] = 0.f;
#pragma unroll
      for (int w = 0; w < LANES / 32; ++w) x[c] += part[c][w];
    }
  }
}

// One row by LANES threads, K vectors of V channels each in registers (K = 0: any number of channels, read twice).
template <typename T, int V, int LANES, int K>
__global__ void __launch_bounds__(kNormThreads) rms_norm_kernel(const NormArgs a) {
  grid_dependency_trigger();
  grid_dependency_wait();
  constexpr int kRows = kNormThreads / LANES;
  const int lane = threadIdx.x % LANES;
  const float inv_c = 1.f / (float)a.channels;
  float w[K > 0 ? K : 1][V];
#pragma unroll
  for (int k = 0; k < K; ++k)
    if ((lane + k * LANES) * V < a.channels) norm_weight<T, V>(a, (lane + k * LANES) * V, w[k]);
  for (long long i = (long long)blockIdx.x * kRows + threadIdx.x / LANES;; i += (long long)gridDim.x * kRows) {
    // (every lane of a warp, or thread of a block, takes part in the sums as long as one of them has a row)
    if (i - threadIdx.x / LANES >= a.rows) break;
    const bool live = i < a.rows;
    float total[1] = {0.f};
    if constexpr (K > 0) {
      float s[K][V];
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = (lane + k * LANES) * V;
        const bool in = live && c < a.channels;
#pragma unroll
        for (int e = 0; e < V; ++e) s[k][e] = 0.f;
        if (!in) continue;
        norm_sum<T, V>(a, i, c, s[k]);
#pragma unroll
        for (int e = 0; e < V; ++e) total[0] = fmaf(s[k][e], s[k][e], total[0]);
      }
      norm_reduce<LANES, 1>(total);
      const float inv = rsqrtf(total[0] * inv_c + a.eps);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = (lane + k * LANES) * V;
        if (!live || c >= a.channels) continue;
        if (a.sum != nullptr) norm_store<T, V>(a.sum, i * a.channels + c, s[k]);
#pragma unroll
        for (int e = 0; e < V; ++e) s[k][e] = s[k][e] * inv * w[k][e];
        norm_store<T, V>(a.y, i * a.channels + c, s[k]);
      }
    } else {
      for (int c = lane * V; live && c < a.channels; c += LANES * V) {
        float s[V];
        norm_sum<T, V>(a, i, c, s);
#pragma unroll
        for (int e = 0; e < V; ++e) total[0] = fmaf(s[e], s[e], total[0]);
      }
      norm_reduce<LANES, 1>(total);
      const float inv = rsqrtf(total[0] * inv_c + a.eps);
      for (int c = lane * V; live && c < a.channels; c += LANES * V) {
        float s[V], w[V];
        norm_sum<T, V>(a, i, c, s);
        if (a.sum != nullptr) norm_store<T, V>(a.sum, i * a.channels + c, s);
        norm_weight<T, V>(a, c, w);
#pragma unroll
        for (int e = 0; e < V; ++e) s[e] = s[e] * inv * w[e];
        norm_store<T, V>(a.y, i * a.channels + c, s);
      }
    }
  }
}

template <typename T, int V, int LANES, int K>
__global__ void __launch_bounds__(kNormThreads) rms_norm_backward_kernel(const NormArgs a) {
  grid_dependency_trigger();
  grid_dependency_wait();
  constexpr int kRows = kNormThreads / LANES;
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const float inv_c = 1.f / (float)a.channels;
  float* slot = a.partial + (long long)blockIdx.x * a.channels;
  if constexpr (K > 0) {
    float gw[K][V] = {}, w[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (lane + k * LANES) * V;
#pragma unroll
      for (int e = 0; e < V; ++e) w[k][e] = 0.f;
      if (c < a.channels) norm_weight<T, V>(a, c, w[k]);
    }
    for (long long i = (long long)blockIdx.x * kRows + group;; i += (long long)gridDim.x * kRows) {
      if (i - group >= a.rows) break;
      const bool live = i < a.rows;
      float s[K][V], gy[K][V], gs[K][V], total[2] = {0.f, 0.f};
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = (lane + k * LANES) * V;
#pragma unroll
        for (int e = 0; e < V; ++e) s[k][e] = gy[k][e] = gs[k][e] = 0.f;
        if (!live || c >= a.channels) continue;
        norm_sum<T, V>(a, i, c, s[k]);
        if (a.gy != nullptr) norm_load<T, V>(a.gy, i * a.gy_row + c, gy[k]);
        if (a.gs != nullptr) norm_load<T, V>(a.gs, i * a.gs_row + c, gs[k]);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          total[0] = fmaf(s[k][e], s[k][e], total[0]);
          total[1] = fmaf(s[k][e], w[k][e] * gy[k][e], total[1]);
        }
      }
      norm_reduce<LANES, 2>(total);
      const float inv = rsqrtf(total[0] * inv_c + a.eps), along = total[1] * inv * inv_c;      // mean(w gy u)
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = (lane + k * LANES) * V;
        if (!live || c >= a.channels) continue;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float u = s[k][e] * inv;
          gw[k][e] = fmaf(gy[k][e], u, gw[k][e]);
          gs[k][e] = fmaf(inv, w[k][e] * gy[k][e] - u * along, gs[k][e]);
        }
        if (a.g != nullptr) norm_store<T, V>(a.g, i * a.channels + c, gs[k]);
      }
    }
    if (a.partial == nullptr) return;
    // the block's rows side by side, in order
    extern __shared__ float part[];                        // [kRows][LANES * K * V]
    constexpr int kWide = LANES * K * V;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < V; ++e) part[group * kWide + (lane + k * LANES) * V + e] = gw[k][e];
    __syncthreads();
    for (int c = threadIdx.x; c < a.channels; c += kNormThreads) {
      float x = 0.f;
      for (int g = 0; g < kRows; ++g) x += part[g * kWide + c];
      slot[c] = x;
    }
  } else {
    // rows of any width: every thread owns its channels of the slot, and adds to them row by row
    if (a.partial != nullptr)
      for (int c = lane * V; c < a.channels; c += LANES * V)
        for (int e = 0; e < V; ++e) slot[c + e] = 0.f;
    for (long long i = blockIdx.x; i < a.rows; i += gridDim.x) {
      float total[2] = {0.f, 0.f};
      for (int c = lane * V; c < a.channels; c += LANES * V) {
        float s[V], gy[V] = {}, w[V];
        norm_sum<T, V>(a, i, c, s);
        if (a.gy != nullptr) norm_load<T, V>(a.gy, i * a.gy_row + c, gy);
        norm_weight<T, V>(a, c, w);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          total[0] = fmaf(s[e], s[e], total[0]);
          total[1] = fmaf(s[e], w[e] * gy[e], total[1]);
        }
      }
      norm_reduce<LANES, 2>(total);
      const float inv = rsqrtf(total[0] * inv_c + a.eps), along = total[1] * inv * inv_c;
      for (int c = lane * V; c < a.channels; c += LANES * V) {
        float s[V], gy[V] = {}, gs[V] = {}, w[V];
        norm_sum<T, V>(a, i, c, s);
        if (a.gy != nullptr) norm_load<T, V>(a.gy, i * a.gy_row + c, gy);
        if (a.gs != nullptr) norm_load<T, V>(a.gs, i * a.gs_row + c, gs);
        norm_weight<T, V>(a, c, w);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float u = s[e] * inv;
          if (a.partial != nullptr) slot[c + e] = fmaf(gy[e], u, slot[c + e]);
          gs[e] = fmaf(inv, w[e] * gy[e] - u * along, gs[e]);
        }
        if (a.g != nullptr) norm_store<T, V>(a.g, i * a.channels + c, gs);
      }
    }
  }
}

// gw[c] = the blocks' sums, in order: 32 channels per block, 32 runs of slots side by side.
template <typename T>
__global__ void __launch_bounds__(1024) rms_norm_weight_kernel(const float* partial, int slots, int channels, void* gw,
                                                               int w_f32) {
  grid_dependency_trigger();
  grid_dependency_wait();
  __shared__ float part[32][33];
  const int lane = threadIdx.x & 31, run = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float x = 0.f;
  if (c < channels) {
#pragma unroll 8
    for (int s = run; s < slots; s += 32) x += partial[(long long)s * channels + c];
  }
  part[run][lane] = x;
  __syncthreads();
  float y = part[lane][run];                     // (warp `run` adds channel `run`)
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) y += __shfl_xor_sync(0xffffffffu, y, m);
  const int out = blockIdx.x * 32 + run;
  if (lane == 0 && out < channels) {
    if (w_f32) ((float*)gw)[out] = y;
    else norm_set(((T*)gw)[out], y);
  }
}

// Blocks of a backward pass, each of which leaves a slot of sums: its rows, at most as many as run at once (592 blocks where
// 444 run leave a half-empty second wave: 68 us against 56 for 250 k rows of 128 channels of 16 bits) and kNormBlocks per SM.
// `blocks` below: a forward pass where it is NULL, else where a backward pass says how many it took.
constexpr int kNormBlocks = 6;

template <typename T, int V, int LANES, int K>
int norm_launch(const NormArgs& a, int* blocks_out, cudaStream_t st) {
  constexpr int kRows = kNormThreads / LANES;
  if (blocks_out == nullptr) {
    const long long need = (a.rows + kRows - 1) / kRows, cap = 16LL * sm_count();
    OCNN_CUDA_OK(launch_chained(rms_norm_kernel<T, V, LANES, K>, dim3((unsigned)(need < cap ? need : cap)),
                                dim3(kNormThreads), 0, st, a));
    OCNN_LAUNCH_OK("rms_norm_kernel");
    return OCNN_OK;
  }
  const size_t smem = K > 0 && a.partial != nullptr ? (size_t)kRows * LANES * K * V * 4 : 0;
  static std::atomic<int> at_once{0};
  int per_sm = at_once.load(std::memory_order_relaxed);
  if (per_sm == 0) {
    OCNN_CUDA_OK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, rms_norm_backward_kernel<T, V, LANES, K>, kNormThreads,
                                                               (size_t)kRows * LANES * K * V * 4));
    per_sm = per_sm < 1 ? 1 : per_sm < kNormBlocks ? per_sm : kNormBlocks;
    at_once.store(per_sm, std::memory_order_relaxed);
  }
  const long long need = (a.rows + kRows - 1) / kRows, cap = (long long)per_sm * sm_count();
  const int blocks = *blocks_out = (int)(need < cap ? need : cap);
  OCNN_CUDA_OK(launch_chained(rms_norm_backward_kernel<T, V, LANES, K>, dim3(blocks), dim3(kNormThreads), smem, st, a));
  OCNN_LAUNCH_OK("rms_norm_backward_kernel");
  return OCNN_OK;
}

// Lanes per row: the fewest of which each has one vector (with two, twice the registers hold half the rows: the gradient of
// 61 k rows of 96 fp32 channels 30 us against 20); a whole warp, then a block, with up to four.
template <typename T, int V>
int norm_by_width(const NormArgs& a, int* blocks, cudaStream_t st) {
  const int vectors = (a.channels + V - 1) / V;
  if (vectors <= 4) return norm_launch<T, V, 4, 1>(a, blocks, st);
  if (vectors <= 8) return norm_launch<T, V, 8, 1>(a, blocks, st);
  if (vectors <= 16) return norm_launch<T, V, 16, 1>(a, blocks, st);
  if (vectors <= 32) return norm_launch<T, V, 32, 1>(a, blocks, st);
  if (vectors <= 64) return norm_launch<T, V, 32, 2>(a, blocks, st);
  if (vectors <= 128) return norm_launch<T, V, 32, 4>(a, blocks, st);
  if (vectors <= 4 * kNormThreads) return norm_launch<T, V, kNormThreads, 4>(a, blocks, st);
  return norm_launch<T, V, kNormThreads, 0>(a, blocks, st);
}

template <typename T>
int norm_by_vector(const NormArgs& a, int* blocks, cudaStream_t st) {
  constexpr int kMost = 16 / sizeof(T);
  uintptr_t bits = (uintptr_t)a.x | (uintptr_t)a.r | (uintptr_t)a.gy | (uintptr_t)a.gs |
                   (uintptr_t)a.sum | (uintptr_t)a.y | (uintptr_t)a.g;
  for (long long stride : {a.x_row, a.r_row, a.gy_row, a.gs_row, (long long)a.channels})
    bits |= (uintptr_t)(stride * (long long)sizeof(T));
  if (bits % 16 == 0) return norm_by_width<T, kMost>(a, blocks, st);
  if (bits % 8 == 0) return norm_by_width<T, kMost / 2>(a, blocks, st);
  return norm_by_width<T, 1>(a, blocks, st);
}

int norm_by_type(const NormArgs& a, int dtype, int* blocks, cudaStream_t st) {
  if (dtype == OCNN_F32) return norm_by_vector<float>(a, blocks, st);
  if (dtype == OCNN_BF16) return norm_by_vector<__nv_bfloat16>(a, blocks, st);
  return norm_by_vector<__half>(a, blocks, st);
}

}  // namespace
}  // namespace ocnn

using namespace ocnn;

extern "C" {

int ocnn_add_rms_norm(const void* x_dev, int64_t x_row, const void* residual_dev, int64_t residual_row,
                      const void* weight_dev, int weight_dtype, void* sum_dev, void* y_dev, int64_t rows, int channels,
                      float eps, int dtype, void* stream) {
  OCNN_REQUIRE(rows >= 0 && channels >= 1 && dtype >= OCNN_F32 && dtype <= OCNN_F16,
               "ocnn_add_rms_norm: %lld rows of %d channels, dtype %d", (long long)rows, channels, dtype);
  OCNN_REQUIRE(weight_dtype == OCNN_F32 || weight_dtype == dtype, "ocnn_add_rms_norm: the weight's type is neither fp32 nor the data's");
  if (rows == 0) return OCNN_OK;
  OCNN_REQUIRE(x_dev && weight_dev && y_dev, "ocnn_add_rms_norm: null pointer");
  NormArgs a = {};
  a.x = x_dev, a.x_row = x_row, a.r = residual_dev, a.r_row = residual_dev ? residual_row : x_row;
  a.w = weight_dev, a.w_f32 = weight_dtype == OCNN_F32;
  a.sum = sum_dev, a.y = y_dev, a.rows = rows, a.channels = channels, a.eps = eps;
  return norm_by_type(a, dtype, nullptr, (cudaStream_t)stream);
}

size_t ocnn_add_rms_norm_backward_workspace_bytes(int channels) {
  return channels > 0 ? (size_t)kNormBlocks * sm_count() * channels * sizeof(float) : 0;
}

int ocnn_add_rms_norm_backward(const void* x_dev, int64_t x_row, const void* residual_dev, int64_t residual_row,
                               const void* weight_dev, int weight_dtype,
                               const void* grad_y_dev, int64_t grad_y_row, const void* grad_sum_dev,
                               int64_t grad_sum_row, void* grad_x_dev, void* grad_weight_dev, int64_t rows,
                               int channels, float eps, int dtype, void* workspace_dev, size_t workspace_bytes,
                               void* stream) {
  OCNN_REQUIRE(rows >= 0 && channels >= 1 && dtype >= OCNN_F32 && dtype <= OCNN_F16,
               "ocnn_add_rms_norm_backward: %lld rows of %d channels, dtype %d", (long long)rows, channels, dtype);
  OCNN_REQUIRE(weight_dtype == OCNN_F32 || weight_dtype == dtype, "ocnn_add_rms_norm_backward: the weight's type is neither fp32 nor the data's");
  cudaStream_t st = (cudaStream_t)stream;
  if (rows == 0) {
    if (grad_weight_dev != nullptr)
      OCNN_CUDA_OK(cudaMemsetAsync(grad_weight_dev, 0, (size_t)channels * (weight_dtype == OCNN_F32 ? 4 : 2), st));
    return OCNN_OK;
  }
  OCNN_REQUIRE(x_dev && weight_dev, "ocnn_add_rms_norm_backward: null pointer");
  if (grad_weight_dev != nullptr &&
      (workspace_dev == nullptr || workspace_bytes < ocnn_add_rms_norm_backward_workspace_bytes(channels)))
    return fail(OCNN_ERR_CAPACITY, "ocnn_add_rms_norm_backward: %zu bytes of workspace are needed",
                ocnn_add_rms_norm_backward_workspace_bytes(channels));
  NormArgs a = {};
  a.x = x_dev, a.x_row = x_row, a.r = residual_dev, a.r_row = residual_dev ? residual_row : x_row;
  a.w = weight_dev, a.w_f32 = weight_dtype == OCNN_F32;
  a.gy = grad_y_dev, a.gy_row = grad_y_dev ? grad_y_row : x_row;
  a.gs = grad_sum_dev, a.gs_row = grad_sum_dev ? grad_sum_row : x_row;
  a.g = grad_x_dev, a.rows = rows, a.channels = channels, a.eps = eps;
  a.partial = grad_weight_dev != nullptr ? (float*)workspace_dev : nullptr;
  int blocks = 0;
  const int status = norm_by_type(a, dtype, &blocks, st);
  if (status != OCNN_OK || grad_weight_dev == nullptr) return status;
  auto sum = dtype == OCNN_F32 ? rms_norm_weight_kernel<float>
             : dtype == OCNN_BF16 ? rms_norm_weight_kernel<__nv_bfloat16> : rms_norm_weight_kernel<__half>;
  OCNN_CUDA_OK(launch_chained(sum, dim3(ceil_div(channels, 32)), dim3(1024), 0, st, (const float*)a.partial, blocks,
                              channels, grad_weight_dev, weight_dtype == OCNN_F32 ? 1 : 0));
  OCNN_LAUNCH_OK("rms_norm_weight_kernel");
  return OCNN_OK;
}

}  // extern "C"
