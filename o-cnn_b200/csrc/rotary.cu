// Rotary positions with several axes: channels of every head turned in pairs by the node's position.
//
//     angle(i, t) = position[i][axis(t)] * freq[t],   t < pairs
//     y1 = x1 cos - x2 sin,  y2 = x2 cos + x1 sin     (inverse: -sin; the gradient is the inverse turn)
//
// Pair t is channels (t, t + dim / 2), or (2t, 2t + 1) when interleaved; pairs behind the last axis' pass through.
// Bound: HBM, every channel read and written once.  The angles of a node are the same for all its heads: a block forms
// the cosines and sines of its nodes once, in shared memory.  An angle is formed and brought into one turn in 64 bits
// (a position of 2^16 times a frequency of 1 has lost 2^-8 of a turn in 32), sine and cosine of the rest in 32.
#include <cstring>

#include "common.cuh"

namespace ocnn {
namespace {

constexpr int kMaxAxes = 8, kMaxPairs = 256, kRotThreads = 256;

struct RotaryArgs {
  const void *x, *positions;
  void* y;
  const double* freqs;
  long long rows, row, head;
  int heads, dim, axes, pairs, rows_per_block, float_positions, inverse;
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

// 16 bytes at a time, the first to leave the caches when something else needs the room.
template <typename P>
__device__ __forceinline__ P read_once(const void* p) {
  P x;
  if constexpr (sizeof(P) == 16) {
    const uint4 w = __ldcs(reinterpret_cast<const uint4*>(p));
    memcpy(&x, &w, 16);
  } else {
    x = *reinterpret_cast<const P*>(p);
  }
  return x;
}
template <typename P>
__device__ __forceinline__ void write_once(void* p, const P& x) {
  if constexpr (sizeof(P) == 16) {
    uint4 w;
    memcpy(&w, &x, 16);
    __stcs(reinterpret_cast<uint4*>(p), w);
  } else {
    *reinterpret_cast<P*>(p) = x;
  }
}

// One item at a time on six blocks per SM: 250 k nodes of 16 heads of 32 in bf16 104 us, 61 k of 8 heads of 24 in fp32 22
// (two items, which leave four blocks: 106 and 26; without that hint to the caches 110 and 23).
// An item is V pairs of one head of one node.  Pairs side by side: two runs of V channels, half a head apart;
// interleaved: one run of 2V channels (as two packs).
template <typename T, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(kRotThreads, 6) rotary_kernel(const RotaryArgs a) {
  extern __shared__ float2 turn[];          // [rows_per_block][pairs]
  const long long r0 = (long long)blockIdx.x * a.rows_per_block;
  const int rows = (int)min((long long)a.rows_per_block, a.rows - r0);
  for (int e = threadIdx.x; e < rows * a.pairs; e += blockDim.x) {
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
  // A thread has one item of a row, in every rows_at_a_time-th row (or, of rows with more items than threads, several).
  const int half = a.dim >> 1, runs = half / V, row_items = a.heads * runs;
  const int across = min(row_items, (int)blockDim.x), step = blockDim.x / across;
  for (int item = threadIdx.x % across; item < row_items; item += across) {
    const int h = item / runs, t = (item - h * runs) * V, c = INTERLEAVED ? 2 * t : t, live = min(V, a.pairs - t);
    const int mine = threadIdx.x / across;
    const T* src = (const T*)a.x + (r0 + mine) * a.row + h * a.head + c;
    T* dst = (T*)a.y + ((r0 + mine) * a.heads + h) * a.dim + c;
    const long long src_step = step * a.row, dst_step = (long long)step * a.heads * a.dim;
    for (int r = mine; r < rows; r += step, src += src_step, dst += dst_step) {
      Pack<T, V> lo = read_once<Pack<T, V>>(src), hi = read_once<Pack<T, V>>(src + (INTERLEAVED ? V : half));
      const float2* w = turn + r * a.pairs + t;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (i >= live) break;                   // (behind the last axis' pairs: as they are, whatever they are)
        // interleaved: pair i is elements 2i, 2i + 1 of the run of 2V
        T& x1 = INTERLEAVED ? (2 * i < V ? lo.x[(2 * i) % V] : hi.x[(2 * i) % V]) : lo.x[i];
        T& x2 = INTERLEAVED ? (2 * i + 1 < V ? lo.x[(2 * i + 1) % V] : hi.x[(2 * i + 1) % V]) : hi.x[i];
        const float f1 = rot_f32(x1), f2 = rot_f32(x2);
        rot_set(x1, f1 * w[i].x - f2 * w[i].y);
        rot_set(x2, f2 * w[i].x + f1 * w[i].y);
      }
      write_once(dst, lo);
      write_once(dst + (INTERLEAVED ? V : half), hi);
    }
  }
}

template <typename T, int V>
int rotary_launch(RotaryArgs& a, bool interleaved, cudaStream_t st) {
  // As many threads as make whole rows (256 at most), and nodes per block: eight a thread, but no more than 16 KB of
  // cosines and sines, and enough blocks for the SMs.
  const int row_items = a.heads * (a.dim / 2 / V);
  const int threads = row_items >= kRotThreads ? kRotThreads : kRotThreads / row_items * row_items;
  const int step = row_items >= kRotThreads ? 1 : kRotThreads / row_items;
  long long r = 8LL * step;
  if (a.pairs > 0 && r * a.pairs > 2048) r = 2048 / a.pairs;
  const long long spread = (a.rows + 4LL * sm_count() - 1) / (4LL * sm_count());
  if (r > spread) r = spread;
  if (r < 1) r = 1;
  a.rows_per_block = (int)r;
  const long long blocks = (a.rows + r - 1) / r;
  OCNN_REQUIRE(blocks < (1LL << 31), "ocnn_octree_rotary: too many rows");
  const size_t smem = (size_t)r * a.pairs * sizeof(float2);
  if (interleaved) rotary_kernel<T, V, true><<<(unsigned)blocks, threads, smem, st>>>(a);
  else rotary_kernel<T, V, false><<<(unsigned)blocks, threads, smem, st>>>(a);
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
