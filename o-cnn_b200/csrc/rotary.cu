// Rotary positions with several axes: channels of every head turned in pairs by the node's position.
//
//     angle(i, t) = position[i][axis(t)] * freq[t],   t < pairs
//     y1 = x1 cos - x2 sin,  y2 = x2 cos + x1 sin     (inverse: -sin; the gradient is the inverse turn)
//
// Pair t is channels (t, t + dim / 2), or (2t, 2t + 1) when interleaved; pairs behind the last axis' pass through.
// Bound: HBM, every channel read and written once.  The angles of a node are the same for all its heads: a block forms
// the cosines and sines of its nodes once, in shared memory.  An angle is formed and brought into one turn in 64 bits
// (a position of 2^16 times a frequency of 1 has lost 2^-8 of a turn in 32), sine and cosine of the rest in 32.
#include "common.cuh"

namespace ocnn {
namespace {

constexpr int kMaxAxes = 8, kMaxPairs = 256, kRotThreads = 256;

struct RotaryArgs {
  const void *x, *positions;
  void* y;
  const double* freqs;
  long long rows, row, head;
  int heads, dim, axes, pairs, rows_per_block, float_positions, inverse, head_items;
  int begin[kMaxAxes + 1];                  // axis a turns the pairs [begin[a], begin[a + 1])
};

template <typename T, int V>
struct alignas(sizeof(T) * V) Pack { T x[V]; };

template <typename T>
__device__ __forceinline__ float rot_f32(T x);
template <>
__device__ __forceinline__ float rot_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ float rot_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float rot_f32<__half>(__half x) { return __half2float(x); }
__device__ __forceinline__ void rot_set(float& y, float x) { y = x; }
__device__ __forceinline__ void rot_set(__nv_bfloat16& y, float x) { y = __float2bfloat16(x); }
__device__ __forceinline__ void rot_set(__half& y, float x) { y = __float2half(x); }

// An item is V pairs of one head of one node.  Pairs side by side: two runs of V channels, half a head apart;
// interleaved: one run of 2V channels (as two packs).
template <typename T, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const RotaryArgs a) {
  extern __shared__ float2 turn[];          // [rows_per_block][pairs]
  const long long r0 = (long long)blockIdx.x * a.rows_per_block;
  const int rows = (int)min((long long)a.rows_per_block, a.rows - r0);
  for (int e = threadIdx.x; e < rows * a.pairs; e += kRotThreads) {
    const int r = e / a.pairs, t = e - r * a.pairs;
    int axis = 0;
    while (t >= a.begin[axis + 1]) ++axis;
    const long long at = (r0 + r) * a.axes + axis;
    const double pos = a.float_positions ? (double)((const float*)a.positions)[at] : (double)((const int*)a.positions)[at];
    const double turns = pos * (a.freqs[t] * 0.15915494309189535);      // 1 / 2 pi
    float s, c;
    sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
    turn[e] = make_float2(c, a.inverse ? -s : s);
  }
  __syncthreads();
  const int half = a.dim >> 1, runs = half / V, row_items = a.heads * runs, items = rows * row_items;
  for (int e0 = threadIdx.x; e0 < items; e0 += 2 * kRotThreads) {
    Pack<T, V> lo[2], hi[2];
    const T* src[2];
    T* dst[2];
    int at[2], first[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int e = e0 + u * kRotThreads;
      if (e >= items) break;
      const int r = e / row_items, rest = e - r * row_items, h = rest / runs, t = (rest - h * runs) * V;
      first[u] = t;
      at[u] = r * a.pairs + t;
      const int c = INTERLEAVED ? 2 * t : t;
      src[u] = (const T*)a.x + (r0 + r) * a.row + h * a.head + c;
      dst[u] = (T*)a.y + ((r0 + r) * a.heads + h) * a.dim + c;
      lo[u] = *reinterpret_cast<const Pack<T, V>*>(src[u]);
      hi[u] = *reinterpret_cast<const Pack<T, V>*>(src[u] + (INTERLEAVED ? V : half));
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (e0 + u * kRotThreads >= items) break;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (first[u] + i >= a.pairs) break;   // (behind the last axis' pairs: as they are, whatever they are)
        const float2 w = turn[at[u] + i];
        // interleaved: pair i is elements 2i, 2i + 1 of the run of 2V
        T& x1 = INTERLEAVED ? (2 * i < V ? lo[u].x[(2 * i) % V] : hi[u].x[(2 * i) % V]) : lo[u].x[i];
        T& x2 = INTERLEAVED ? (2 * i + 1 < V ? lo[u].x[(2 * i + 1) % V] : hi[u].x[(2 * i + 1) % V]) : hi[u].x[i];
        const float f1 = rot_f32(x1), f2 = rot_f32(x2);
        rot_set(x1, f1 * w.x - f2 * w.y);
        rot_set(x2, f2 * w.x + f1 * w.y);
      }
      *reinterpret_cast<Pack<T, V>*>(dst[u]) = lo[u];
      *reinterpret_cast<Pack<T, V>*>(dst[u] + (INTERLEAVED ? V : half)) = hi[u];
    }
  }
}

template <typename T, int V>
int rotary_launch(RotaryArgs& a, bool interleaved, cudaStream_t st) {
  // nodes per block: four items a thread, but no more than 16 KB of cosines and sines, and enough blocks for the SMs
  const int row_items = a.heads * (a.dim / 2 / V);
  long long r = (4 * kRotThreads + row_items - 1) / row_items;
  if (a.pairs > 0 && r * a.pairs > 2048) r = 2048 / a.pairs;
  const long long spread = (a.rows + 4LL * sm_count() - 1) / (4LL * sm_count());
  if (r > spread) r = spread;
  if (r < 1) r = 1;
  a.rows_per_block = (int)r;
  const long long blocks = (a.rows + r - 1) / r;
  OCNN_REQUIRE(blocks < (1LL << 31), "ocnn_octree_rotary: too many rows");
  const size_t smem = (size_t)r * a.pairs * sizeof(float2);
  if (interleaved) rotary_kernel<T, V, true><<<(unsigned)blocks, kRotThreads, smem, st>>>(a);
  else rotary_kernel<T, V, false><<<(unsigned)blocks, kRotThreads, smem, st>>>(a);
  OCNN_LAUNCH_OK("rotary_kernel");
  return OCNN_OK;
}

// The widest run of pairs that divides half a head and keeps every access aligned (16 bytes at most).
template <typename T>
int rotary_by_width(RotaryArgs& a, bool interleaved, cudaStream_t st) {
  const uintptr_t bits = (uintptr_t)a.x | (uintptr_t)a.y | (uintptr_t)(a.row * (long long)sizeof(T)) |
                         (uintptr_t)(a.head * (long long)sizeof(T));
  auto fits = [&](int v) { return (a.dim / 2) % v == 0 && bits % (v * sizeof(T)) == 0; };
  if constexpr (sizeof(T) == 2)
    if (fits(8)) return rotary_launch<T, 8>(a, interleaved, st);
  if (fits(4)) return rotary_launch<T, 4>(a, interleaved, st);
  if (fits(2)) return rotary_launch<T, 2>(a, interleaved, st);
  return rotary_launch<T, 1>(a, interleaved, st);
}

}  // namespace
}  // namespace ocnn

using namespace ocnn;

extern "C" int ocnn_octree_rotary(const void* x_dev, const int64_t x_stride[2], void* y_dev, const void* positions_dev,
                                  int float_positions, const double* freqs_dev, int axes, const int* sections,
                                  int64_t rows, int heads, int dim, int interleaved, int inverse, int dtype,
                                  void* stream) {
  OCNN_REQUIRE(rows >= 0 && heads >= 1 && dim >= 2 && dim % 2 == 0,
               "ocnn_octree_rotary: %lld rows of %d heads of %d channels (an even number)", (long long)rows, heads, dim);
  OCNN_REQUIRE(dtype >= OCNN_F32 && dtype <= OCNN_F16, "ocnn_octree_rotary: bad dtype %d", dtype);
  OCNN_REQUIRE(axes >= 1 && axes <= kMaxAxes && sections != nullptr, "ocnn_octree_rotary: 1 to %d axes", kMaxAxes);
  RotaryArgs a = {};
  for (int i = 0; i < axes; ++i) {
    OCNN_REQUIRE(sections[i] >= 0 && sections[i] <= dim / 2 - a.pairs,
                 "ocnn_octree_rotary: the sections hold more than the %d pairs of a head", dim / 2);
    a.begin[i] = a.pairs;
    a.pairs += sections[i];
  }
  a.begin[axes] = a.pairs;
  if (dim / 2 > kMaxPairs)
    return fail(OCNN_ERR_UNSUPPORTED, "ocnn_octree_rotary: heads of more than %d channels", 2 * kMaxPairs);
  if (rows == 0) return OCNN_OK;
  OCNN_REQUIRE(x_dev && y_dev && (a.pairs == 0 || (positions_dev && freqs_dev)), "ocnn_octree_rotary: null pointer");
  a.x = x_dev, a.y = y_dev, a.positions = positions_dev, a.freqs = freqs_dev;
  a.rows = rows, a.row = x_stride[0], a.head = x_stride[1];
  a.heads = heads, a.dim = dim, a.axes = axes, a.float_positions = float_positions, a.inverse = inverse;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == OCNN_F32) return rotary_by_width<float>(a, interleaved != 0, st);
  if (dtype == OCNN_BF16) return rotary_by_width<__nv_bfloat16>(a, interleaved != 0, st);
  return rotary_by_width<__half>(a, interleaved != 0, st);
}
