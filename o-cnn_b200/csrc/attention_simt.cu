// Attention over a window of nodes on the CUDA cores: fp32 data, and 16-bit data in shapes or alignments that the
// tensor-core kernels do not take.
#include "attention.cuh"

namespace ocnn {
namespace {

constexpr int kB = 64;                        // queries and keys per tile
constexpr int kThreads = 256;                 // 16 x 16: thread (ty, tx) has rows 4 ty .. 4 ty + 3, columns tx + 16 c
constexpr int kPad = 4;                       // a row of DP + 4 floats: 16 rows 16 bytes each hit distinct banks

// Bound: instruction issue (fp32 products have no tensor pipe of their accuracy here) and, between a tile's barriers, the
// latency of its loads, which other thread blocks cover: of up to 32 channels three per SM (80 registers), of 64 two.
// Blocks of 16 columns that none of a warp's eight rows sees are left out.  Forward and gradients of 20 k nodes, 4 heads of
// 24, window 64: 316 us (90 + 110 + 134 one by one from cold caches); two blocks per SM and every column of a tile computed: 380.
template <int DP> constexpr int kPerSm = DP == 32 ? 3 : DP == 64 ? 2 : 1;

// Rows of a [n, heads, dim] tensor as floats, zeros for row < 0 and behind dim.  `index` gives the row for 0 .. kB - 1.
template <typename T, int DP, typename Index>
__device__ __forceinline__ void load_rows(float* dst, const void* base, long long row, long long head_offset, int dim,
                                          bool vec, Index index) {
  const T* src = (const T*)base + head_offset;
  for (int e = threadIdx.x; e < kB * (DP / 4); e += kThreads) {
    const int r = e / (DP / 4), d = (e % (DP / 4)) * 4, i = index(r);
    float x[4] = {};
    if (i >= 0 && d < dim) {
      const T* p = src + i * row + d;
      if (vec) {
        if constexpr (sizeof(T) == 4) {
          const float4 w = *reinterpret_cast<const float4*>(p);
          x[0] = w.x, x[1] = w.y, x[2] = w.z, x[3] = w.w;
        } else {
          const uint2 w = *reinterpret_cast<const uint2*>(p);
          const T* t = reinterpret_cast<const T*>(&w);
#pragma unroll
          for (int c = 0; c < 4; ++c) x[c] = to_f32(t[c]);
        }
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (d + c < dim) x[c] = to_f32(p[c]);
      }
    }
    *reinterpret_cast<float4*>(dst + r * (DP + kPad) + d) = make_float4(x[0], x[1], x[2], x[3]);
  }
}

// Which blocks of 16 columns hold anything that one of the warp's eight rows sees: bit c for columns 16 c .. 16 c + 15.
// `seen`: bit 4 r + c where the thread's row r sees its column tx + 16 c.
__device__ __forceinline__ unsigned live_columns(unsigned seen) {
  unsigned live = 0;
#pragma unroll
  for (int c = 0; c < 4; ++c) live |= __any_sync(0xffffffffu, (seen & (0x1111u << c)) != 0) ? 1u << c : 0u;
  return live;
}

// acc[r][c] = A row (4 ty + r) . B row (tx + 16 (c0 + c)), even and odd channels side by side in one instruction, for
// kDotCols blocks of columns: of 32 channels two at a time, since the sums of four do not fit the registers of three
// thread blocks per SM.
template <int DP> constexpr int kDotCols = DP == 32 ? 2 : 4;
template <int DP>
__device__ __forceinline__ void tile_dot(const float* A, const float* B, int dim, int c0, float (&acc)[4][kDotCols<DP>]) {
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  uint64_t sum[4][kDotCols<DP>] = {};
#pragma unroll 1
  for (int d = 0; d < dim; d += 4) {                     // (rows hold zeros behind dim)
    ulonglong2 x[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) x[r] = *reinterpret_cast<const ulonglong2*>(A + (4 * ty + r) * (DP + kPad) + d);
#pragma unroll
    for (int c = 0; c < kDotCols<DP>; ++c) {
      const ulonglong2 y = *reinterpret_cast<const ulonglong2*>(B + (tx + 16 * (c0 + c)) * (DP + kPad) + d);
#pragma unroll
      for (int r = 0; r < 4; ++r) sum[r][c] = fma2(x[r].y, y.y, fma2(x[r].x, y.x, sum[r][c]));
    }
  }
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int c = 0; c < kDotCols<DP>; ++c) {
      const float2 f = unpair(sum[r][c]);
      acc[r][c] = f.x + f.y;
    }
}
template <int DP>
__device__ __forceinline__ bool any_live(unsigned live, int c0) { return (live >> c0 & ((1u << kDotCols<DP>) - 1)) != 0; }

constexpr int kPRow = kB + 4;
// out = P B, where P has a row of kB columns per row of the tile and B a row of DP channels per column.  A thread sums
// channels in fours, 4 l + 64 q with l = tx, so that a value of P is used for four at a time.  Of 32 channels there are
// only eight fours: lanes tx and tx + 8 take the same one and every second four columns each, and exchange halves at the end.
template <int DP> constexpr int kOutPairs = DP == 32 ? 2 : DP / 32;
template <int DP>
struct OutTile { uint64_t sum[4][kOutPairs<DP>]; };
template <int DP>
__device__ __forceinline__ void tile_mul(const float* P, const float* B, unsigned live, OutTile<DP>& out) {
  constexpr int kSplit = DP == 32 ? 2 : 1;
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  const int l = DP == 32 ? tx & 7 : tx, shift = DP == 32 ? 4 * (tx >> 3) : 0;
#pragma unroll 1
  for (int j0 = 0; j0 < kB; j0 += 16) {
    if (!(live >> (j0 / 16) & 1)) continue;
#pragma unroll 1
    for (int jj = 0; jj < 16; jj += 4 * kSplit) {
      const int j = j0 + jj + shift;
      float4 p[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) p[r] = *reinterpret_cast<const float4*>(P + (4 * ty + r) * kPRow + j);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        ulonglong2 v[kOutPairs<DP> / 2];
#pragma unroll
        for (int q = 0; q < kOutPairs<DP> / 2; ++q)
          v[q] = *reinterpret_cast<const ulonglong2*>(B + (j + k) * (DP + kPad) + 4 * l + 64 * q);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float x = k == 0 ? p[r].x : k == 1 ? p[r].y : k == 2 ? p[r].z : p[r].w;
          const uint64_t xx = pair(x, x);
#pragma unroll
          for (int q = 0; q < kOutPairs<DP> / 2; ++q) {
            out.sum[r][2 * q] = fma2(xx, v[q].x, out.sum[r][2 * q]);
            out.sum[r][2 * q + 1] = fma2(xx, v[q].y, out.sum[r][2 * q + 1]);
          }
        }
      }
    }
  }
}
// A thread's share of row r, DP / 16 channels: the c-th is channel out_col(c).
template <int DP>
__device__ __forceinline__ int out_col(int c) {
  const int tx = threadIdx.x & 15;
  return DP == 32 ? 4 * (tx & 7) + 2 * (tx >> 3) + c : 4 * tx + 64 * (c >> 2) + (c & 3);
}
template <int DP>
__device__ __forceinline__ void out_row(const OutTile<DP>& out, int r, float (&x)[DP / 16]) {
  if (DP == 32) {
    const bool upper = (threadIdx.x & 8) != 0;
    const float2 low = unpair(out.sum[r][0]), high = unpair(out.sum[r][1]);
    x[0] = (upper ? high.x : low.x) + __shfl_xor_sync(0xffffffffu, upper ? low.x : high.x, 8);
    x[1] = (upper ? high.y : low.y) + __shfl_xor_sync(0xffffffffu, upper ? low.y : high.y, 8);
  } else {
#pragma unroll
    for (int q = 0; q < DP / 32; ++q) {
      const float2 f = unpair(out.sum[r][q]);
      x[2 * q] = f.x;
      x[2 * q + 1] = f.y;
    }
  }
}

__device__ __forceinline__ float row_max(float x) {
#pragma unroll
  for (int m = 8; m > 0; m >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, m));
  return x;
}
__device__ __forceinline__ float row_sum(float x) {
#pragma unroll
  for (int m = 8; m > 0; m >>= 1) x += __shfl_xor_sync(0xffffffffu, x, m);
  return x;
}

template <int DP>
constexpr size_t smem_bytes(int tiles, int p_tiles) {
  return (size_t)(tiles * kB * (DP + kPad) + p_tiles * kB * kPRow) * 4;
}

// The keys of the query tile at r0 and each row's (rows[] in shared memory), by all threads of the block.
__device__ __forceinline__ TileKeys query_tile(const AttnArgs& a, int r0, RowKeys* rows, int* ext) {
  if (threadIdx.x == 0) {
    ext[0] = INT_MAX;
    ext[1] = 0;
  }
  __syncthreads();
  if (threadIdx.x < kB) {
    const int i = r0 + threadIdx.x;
    const RowKeys r = attn_row_keys(a, i, attn_span(a, i));
    rows[threadIdx.x] = r;
    if (r.hi > r.lo) {
      atomicMin(&ext[0], r.lo);
      atomicMax(&ext[1], max(r.hi, r.first));
    }
    // (the first nodes of the first row's sequence; an empty row's are none)
    if (threadIdx.x == 0) {
      ext[2] = r.start;
      ext[3] = r.start;
    }
  }
  __syncthreads();
  if (threadIdx.x < kB) {
    const RowKeys r = rows[threadIdx.x];
    if (r.start == ext[2] && r.hi > r.lo) atomicMax(&ext[3], r.first);
  }
  __syncthreads();
  TileKeys t;
  t.lo = ext[0];
  t.first = ext[2];
  t.n_first = ext[1] > ext[0] ? max(0, min(ext[3], t.lo) - t.first) : 0;
  t.n = t.n_first + max(0, ext[1] - (ext[1] > 0 ? t.lo : 0));
  return t;
}

// One tile of 64 queries of one head: a pass over the keys that they see, with a running maximum and sum per row.
template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, kPerSm<DP>) attn_simt_kernel(const AttnArgs a, T* out, float* lse, bool vec) {
  extern __shared__ float smem[];
  float* sq = smem;
  float* sk = sq + kB * (DP + kPad);
  float* sv = sk + kB * (DP + kPad);
  float* sp = sv + kB * (DP + kPad);
  __shared__ RowKeys rows[kB];
  __shared__ int ext[4], redo[kB];
  const int r0 = blockIdx.x * kB, h = blockIdx.y, hk = h / (a.heads / a.kv_heads);
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  const TileKeys keys = query_tile(a, r0, rows, ext);
  load_rows<T, DP>(sq, a.q, a.q_row, h * a.q_head, a.dim, vec, [&](int r) { return r0 + r < a.n ? r0 + r : -1; });

  OutTile<DP> acc = {};
  float top[4], total[4] = {};
  unsigned ever = 0;                                         // as `seen`, of all tiles so far
#pragma unroll
  for (int r = 0; r < 4; ++r) top[r] = -INFINITY;
  for (int t0 = 0; t0 < keys.n; t0 += kB) {
    // a hidden key's row reads as zeros: what lies there has no say
    auto row_of = [&](int t) {
      if (t0 + t >= keys.n) return -1;
      const int j = keys.key(t0 + t);
      return a.mask != nullptr && a.mask[j] == 0 ? -1 : j;
    };
    __syncthreads();
    load_rows<T, DP>(sk, a.k, a.k_row, hk * a.k_head, a.dim, vec, row_of);
    load_rows<T, DP>(sv, a.v, a.v_row, hk * a.v_head, a.dim, vec, row_of);
    int j[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) j[c] = row_of(tx + 16 * c);
    __syncthreads();
    unsigned seen = 0;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const RowKeys rk = rows[4 * ty + r];
#pragma unroll
      for (int c = 0; c < 4; ++c) seen |= j[c] >= 0 && attn_sees(rk, j[c]) ? 1u << (4 * r + c) : 0u;
    }
    ever |= seen;
    const unsigned live = live_columns(seen);
    if (live == 0) continue;
    float s[4][4];
#pragma unroll
    for (int c0 = 0; c0 < 4; c0 += kDotCols<DP>) {
      float x[4][kDotCols<DP>] = {};
      if (any_live<DP>(live, c0)) tile_dot<DP>(sq, sk, a.dim, c0, x);
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < kDotCols<DP>; ++c)
          s[r][c0 + c] = seen >> (4 * r + c0 + c) & 1 ? x[r][c] * a.scale_log2 : -INFINITY;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float m = -INFINITY;
#pragma unroll
      for (int c = 0; c < 4; ++c) m = fmaxf(m, s[r][c]);
      m = fmaxf(top[r], row_max(m));
      const float base = m == -INFINITY ? 0.f : m;          // a row that has seen nothing yet
      const float keep = exp2_approx(top[r] - base);
      top[r] = m;
      float sum = 0.f;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float p = exp2_approx(s[r][c] - base);
        sp[(4 * ty + r) * kPRow + tx + 16 * c] = p;
        sum += p;
      }
      total[r] = total[r] * keep + sum;
#pragma unroll
      for (int q = 0; q < kOutPairs<DP>; ++q) acc.sum[r][q] = fma2(acc.sum[r][q], pair(keep, keep), 0);
    }
    __syncwarp();                                            // (a row of P is written and read by one half warp)
    tile_mul<DP>(sp, sv, live, acc);
  }
  T* rest = attn_rest<T>(a, lse);
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int i = r0 + 4 * ty + r;
    const bool sees = (__ballot_sync(0xffffffffu, (ever >> (4 * r) & 15u) != 0) >> (tid & 16) & 0xffffu) != 0;
    float sum = row_sum(total[r]);
    if (sees && sum == 0.f) sum = NAN;                       // scores of -inf alone have no softmax
    const float inv = sees ? 1.f / sum : 0.f;
    bool bad = false;
    float x[DP / 16];
    out_row<DP>(acc, r, x);
    if (i < a.n) {
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) {
        bad |= not_finite(x[c]);
        const int d = out_col<DP>(c);
        if (d >= a.dim) continue;
        const long long at = ((long long)i * a.heads + h) * a.dim + d;
        const float y = sees ? x[c] * inv : 0.f;
        out[at] = from_f32<T>(y);
        if (sizeof(T) == 2 && rest != nullptr) rest[at] = from_f32<T>(rounded_off<T>(y));
      }
      if (tx == 0 && lse != nullptr) lse[(long long)h * a.n + i] = sees ? top[r] + log2f(sum) : INFINITY;
    }
    // (a sum that is no number is the row's own doing: a hidden key is not in it)
    const unsigned any = __ballot_sync(0xffffffffu, bad && !not_finite(sum));
    if (tx == 0) redo[4 * ty + r] = (any >> (tid & 16)) & 0xffffu;
  }
  __syncthreads();
  for (int r = tid >> 5; r < kB; r += kThreads / 32)
    if (redo[r] != 0 && r0 + r < a.n && !attn_row_is_spoilt<T>(a, r0 + r, h, out)) attn_forward_row<T>(a, r0 + r, h, out, lse);
}

// Gradient of the queries of one tile, and delta_i = dO_i . o_i for the keys' gradients.
//     p = exp2(s - lse), ds = p (dO . v - delta), dq = scale sum_j ds k_j
template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, kPerSm<DP>) attn_simt_dq_kernel(const AttnArgs a, const AttnGrad g, bool vec) {
  extern __shared__ float smem[];
  float* sq = smem;
  float* sg = sq + kB * (DP + kPad);
  float* sk = sg + kB * (DP + kPad);
  float* sv = sk + kB * (DP + kPad);
  float* sp = sv + kB * (DP + kPad);
  __shared__ RowKeys rows[kB];
  __shared__ int ext[4], redo[kB];
  const int r0 = blockIdx.x * kB, h = blockIdx.y, hk = h / (a.heads / a.kv_heads);
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  const TileKeys keys = query_tile(a, r0, rows, ext);
  auto query = [&](int r) { return r0 + r < a.n ? r0 + r : -1; };
  load_rows<T, DP>(sq, a.q, a.q_row, h * a.q_head, a.dim, vec, query);
  load_rows<T, DP>(sg, g.grad, g.grad_row, h * g.grad_head, a.dim, vec, query);
  load_rows<T, DP>(sk, g.out, (long long)a.heads * a.dim, (long long)h * a.dim, a.dim, vec, query);
  __syncthreads();
  float lse[4], delta[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int i = r0 + 4 * ty + r;
    lse[r] = i < a.n ? g.lse[(long long)h * a.n + i] : INFINITY;
    float x = 0.f;
    for (int d = tx; d < DP; d += 16) {
      float o = sk[(4 * ty + r) * (DP + kPad) + d];
      if (sizeof(T) == 2 && i < a.n && d < a.dim) o += to_f32(attn_rest<T>(a, g.lse)[((long long)i * a.heads + h) * a.dim + d]);
      x = fmaf(sg[(4 * ty + r) * (DP + kPad) + d], o, x);
    }
    delta[r] = row_sum(x);
    if (tx == 0 && i < a.n) g.delta[(long long)h * a.n + i] = delta[r];
  }
  OutTile<DP> acc = {};
  for (int t0 = 0; t0 < keys.n; t0 += kB) {
    auto row_of = [&](int t) {
      if (t0 + t >= keys.n) return -1;
      const int j = keys.key(t0 + t);
      return a.mask != nullptr && a.mask[j] == 0 ? -1 : j;
    };
    __syncthreads();
    load_rows<T, DP>(sk, a.k, a.k_row, hk * a.k_head, a.dim, vec, row_of);
    load_rows<T, DP>(sv, a.v, a.v_row, hk * a.v_head, a.dim, vec, row_of);
    int j[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) j[c] = row_of(tx + 16 * c);
    __syncthreads();
    unsigned seen = 0;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const RowKeys rk = rows[4 * ty + r];
#pragma unroll
      for (int c = 0; c < 4; ++c) seen |= j[c] >= 0 && attn_sees(rk, j[c]) ? 1u << (4 * r + c) : 0u;
    }
    const unsigned live = live_columns(seen);
    if (live == 0) continue;
#pragma unroll
    for (int c0 = 0; c0 < 4; c0 += kDotCols<DP>) {
      if (!any_live<DP>(live, c0)) continue;
      float s[4][kDotCols<DP>], dp[4][kDotCols<DP>];
      tile_dot<DP>(sq, sk, a.dim, c0, s);
      tile_dot<DP>(sg, sv, a.dim, c0, dp);
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < kDotCols<DP>; ++c)
          sp[(4 * ty + r) * kPRow + tx + 16 * (c0 + c)] =
              seen >> (4 * r + c0 + c) & 1 ? exp2_approx(s[r][c] * a.scale_log2 - lse[r]) * (dp[r][c] - delta[r]) : 0.f;
    }
    __syncwarp();
    tile_mul<DP>(sp, sk, live, acc);
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int i = r0 + 4 * ty + r;
    bool bad = false;
    float x[DP / 16];
    out_row<DP>(acc, r, x);
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) {
      const int d = out_col<DP>(c);
      bad |= not_finite(x[c]);
      if (i < a.n && d < a.dim) ((T*)g.dq)[((long long)i * a.heads + h) * a.dim + d] = from_f32<T>(x[c] * a.scale);
    }
    const unsigned any = __ballot_sync(0xffffffffu, bad && !attn_query_is_spoilt(lse[r], delta[r]));
    if (tx == 0) redo[4 * ty + r] = (any >> (tid & 16)) & 0xffffu;
  }
  __syncthreads();
  for (int r = tid >> 5; r < kB; r += kThreads / 32)
    if (redo[r] != 0 && r0 + r < a.n) attn_dq_row<T>(a, g, r0 + r, h);
}

// Gradients of the keys and values of one tile of 64 keys: over the nodes that see them from within the window, head
// by head of the group; what the far pass has summed for first nodes is added at the end.
//     dv_j = sum_i p_ij dO_i, dk_j = scale sum_i ds_ij q_i
template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, kPerSm<DP>) attn_simt_dkv_kernel(const AttnArgs a, const AttnGrad g, bool vec) {
  extern __shared__ float smem[];
  float* sk = smem;
  float* sv = sk + kB * (DP + kPad);
  float* sq = sv + kB * (DP + kPad);
  float* sg = sq + kB * (DP + kPad);
  float* sp = sg + kB * (DP + kPad);
  float* sd = sp + kB * kPRow;
  __shared__ KeyRows rows[kB];
  __shared__ int ext[2], redo[kB];
  const int k0 = blockIdx.x * kB, hk = blockIdx.y, group = a.heads / a.kv_heads;
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  if (tid == 0) {
    ext[0] = INT_MAX;
    ext[1] = 0;
  }
  __syncthreads();
  if (tid < kB) {
    const int j = k0 + tid;
    const KeyRows r = j < a.n ? attn_key_rows(a, j, attn_span(a, j)) : KeyRows{0, 0};
    rows[tid] = r;
    if (r.hi > r.lo) {
      atomicMin(&ext[0], r.lo);
      atomicMax(&ext[1], r.hi);
    }
  }
  __syncthreads();
  auto key = [&](int t) { return rows[t].hi > rows[t].lo ? k0 + t : -1; };
  load_rows<T, DP>(sk, a.k, a.k_row, hk * a.k_head, a.dim, vec, key);
  load_rows<T, DP>(sv, a.v, a.v_row, hk * a.v_head, a.dim, vec, key);
  OutTile<DP> dk = {}, dv = {};
  for (int hg = 0; hg < group; ++hg) {
    const int h = hk * group + hg;
    for (int i0 = ext[0]; i0 < ext[1]; i0 += kB) {
      auto query = [&](int t) { return i0 + t < ext[1] ? i0 + t : -1; };
      __syncthreads();
      load_rows<T, DP>(sq, a.q, a.q_row, h * a.q_head, a.dim, vec, query);
      load_rows<T, DP>(sg, g.grad, g.grad_row, h * g.grad_head, a.dim, vec, query);
      float lse[4], delta[4];
      int i[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        i[c] = query(tx + 16 * c);
        lse[c] = i[c] >= 0 ? g.lse[(long long)h * a.n + i[c]] : 0.f;
        delta[c] = i[c] >= 0 ? g.delta[(long long)h * a.n + i[c]] : 0.f;
      }
      __syncthreads();
      unsigned seen = 0;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const KeyRows kr = rows[4 * ty + r];
#pragma unroll
        for (int c = 0; c < 4; ++c) seen |= i[c] >= kr.lo && i[c] < kr.hi ? 1u << (4 * r + c) : 0u;
      }
      const unsigned live = live_columns(seen);
      if (live == 0) continue;
#pragma unroll
      for (int c0 = 0; c0 < 4; c0 += kDotCols<DP>) {
        if (!any_live<DP>(live, c0)) continue;
        float s[4][kDotCols<DP>], dp[4][kDotCols<DP>];
        tile_dot<DP>(sk, sq, a.dim, c0, s);
        tile_dot<DP>(sv, sg, a.dim, c0, dp);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int c = 0; c < kDotCols<DP>; ++c) {
            const int at = (4 * ty + r) * kPRow + tx + 16 * (c0 + c);
            const bool see = seen >> (4 * r + c0 + c) & 1;
            const float p = see ? exp2_approx(s[r][c] * a.scale_log2 - lse[c0 + c]) : 0.f;
            sp[at] = p;
            sd[at] = see ? p * (dp[r][c] - delta[c0 + c]) : 0.f;
          }
      }
      __syncwarp();
      tile_mul<DP>(sp, sg, live, dv);
      tile_mul<DP>(sd, sq, live, dk);
    }
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int j = k0 + 4 * ty + r;
    const float* far = j < a.n ? far_sums(a, g, j, hk) : nullptr;
    bool bad_dk = false, bad_dv = false;
    float dk_row[DP / 16], dv_row[DP / 16];
    out_row<DP>(dk, r, dk_row);
    out_row<DP>(dv, r, dv_row);
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) {
      const int d = out_col<DP>(c);
      float x = dk_row[c], y = dv_row[c];
      bad_dk |= not_finite(x);
      bad_dv |= not_finite(y);
      if (j >= a.n || d >= a.dim) continue;
      x += far != nullptr ? far[d] : 0.f;
      y += far != nullptr ? far[a.dim + d] : 0.f;
      ((T*)g.dk)[((long long)j * a.kv_heads + hk) * a.dim + d] = from_f32<T>(x * a.scale);
      ((T*)g.dv)[((long long)j * a.kv_heads + hk) * a.dim + d] = from_f32<T>(y);
    }
    const unsigned any_dk = __ballot_sync(0xffffffffu, bad_dk), any_dv = __ballot_sync(0xffffffffu, bad_dv);
    if (tx == 0) redo[4 * ty + r] = ((any_dk >> (tid & 16)) & 0xffffu ? 1 : 0) + ((any_dv >> (tid & 16)) & 0xffffu ? 2 : 0);
  }
  __syncthreads();
  for (int r = tid >> 5; r < kB; r += kThreads / 32) {
    if (k0 + r >= a.n) continue;
    const bool dk_too = (redo[r] & 1) && !attn_key_is_spoilt<T>(a, g, k0 + r, hk, false);
    const bool dv_too = (redo[r] & 2) && !attn_key_is_spoilt<T>(a, g, k0 + r, hk, true);
    if (dk_too || dv_too) attn_dkv_row<T>(a, g, k0 + r, hk, dk_too, dv_too);
  }
}

// The far pass: what the nodes beyond the window add to the gradients of their sequence's first nodes, kFarSinks of them
// at a time.  A block takes kFarRows nodes of one key head; a row (a query head of a node) is read once by LPR lanes,
// 16 bytes of q and dO each, which keep their channels of the sums, so that a warp has 32 / LPR rows under way.
constexpr int kFarSinks = 4;

template <typename T>
__device__ __forceinline__ void far_load(const T* p, int left, bool vec, float (&x)[16 / sizeof(T)]) {
  constexpr int V = 16 / sizeof(T);
  if (vec) {
    uint4 w = make_uint4(0, 0, 0, 0);
    if (left > 0) w = *reinterpret_cast<const uint4*>(p);
    const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
    for (int c = 0; c < V; ++c) x[c] = to_f32(e[c]);
  } else {
#pragma unroll
    for (int c = 0; c < V; ++c) x[c] = c < left ? to_f32(p[c]) : 0.f;
  }
}

template <typename T, int LPR>
__global__ void __launch_bounds__(256, 2) attn_far_kernel(const AttnArgs a, const AttnGrad g, bool vec) {
  constexpr int V = 16 / sizeof(T), kRows = 256 / LPR;        // rows of a block at a time
  const int hk = blockIdx.y, group = a.heads / a.kv_heads, tid = threadIdx.x, sub = tid % LPR, row = tid / LPR;
  const int r0 = blockIdx.x * kFarRows, r1 = min(a.n, r0 + kFarRows), d0 = sub * V, left = a.dim - d0;
  __shared__ float part[8][2 * kMaxHeadDim];
  for (int i0 = r0; i0 < r1;) {
    const Span s = attn_span(a, i0);
    if (s.end <= s.start) {                        // outside of every sequence: on to the first one, or to the end
      const int begin = attn_offset(a, 0);
      i0 = i0 < begin ? begin : r1;
      continue;
    }
    if (s.end - s.start <= a.window) {             // nobody here sees a first node from far
      i0 = s.end;
      continue;
    }
    const int end = min(r1, s.end), sinks = min(a.sinks, s.end - s.start), slot = blockIdx.x + far_number(a, s);
    for (int t0 = 0; t0 < sinks; t0 += kFarSinks) {
      float k[kFarSinks][V], v[kFarSinks][V], dk[kFarSinks][V] = {}, dv[kFarSinks][V] = {};
      bool kept[kFarSinks];
#pragma unroll
      for (int t = 0; t < kFarSinks; ++t) {
        const int j = s.start + t0 + t;
        kept[t] = t0 + t < sinks && (a.mask == nullptr || a.mask[j] != 0);
        far_load<T>((const T*)a.k + j * a.k_row + hk * a.k_head + d0, kept[t] ? left : 0, vec, k[t]);
        far_load<T>((const T*)a.v + j * a.v_row + hk * a.v_head + d0, kept[t] ? left : 0, vec, v[t]);
      }
      // the rows that see the first of them from far; the others' turn comes a node later each
      const int from = s.end - s.start - t0 > a.window ? max(i0, s.start + t0 + a.window) : end;
      const int count = (end - from) * group;
      for (int e = row; e - row < count; e += kRows) {         // (all lanes of a warp go round together)
        const bool in = e < count;
        const int i = from + (in ? e / group : 0), h = hk * group + (in ? e % group : 0);
        float q[V], o[V];
        far_load<T>((const T*)a.q + i * a.q_row + h * a.q_head + d0, in ? left : 0, vec, q);
        far_load<T>((const T*)g.grad + i * g.grad_row + h * g.grad_head + d0, in ? left : 0, vec, o);
        const float lse = in ? g.lse[(long long)h * a.n + i] : 0.f, delta = in ? g.delta[(long long)h * a.n + i] : 0.f;
#pragma unroll
        for (int t = 0; t < kFarSinks; ++t) {
          if (t0 + t >= sinks) break;
          float x = 0.f, y = 0.f;
#pragma unroll
          for (int c = 0; c < V; ++c) {
            x = fmaf(q[c], k[t][c], x);
            y = fmaf(o[c], v[t][c], y);
          }
#pragma unroll
          for (int m = LPR / 2; m > 0; m >>= 1) {
            x += __shfl_xor_sync(0xffffffffu, x, m);
            y += __shfl_xor_sync(0xffffffffu, y, m);
          }
          const bool seen = in && kept[t] && i - (s.start + t0 + t) >= a.window;
          const float p = seen ? exp2f(x * a.scale_log2 - lse) : 0.f, ds = seen ? p * (y - delta) : 0.f;
#pragma unroll
          for (int c = 0; c < V; ++c) {
            dk[t][c] += seen ? ds * q[c] : 0.f;
            dv[t][c] += seen ? p * o[c] : 0.f;
          }
        }
      }
#pragma unroll
      for (int t = 0; t < kFarSinks; ++t) {
        if (t0 + t >= sinks) break;
#pragma unroll
        for (int c = 0; c < V; ++c)
#pragma unroll
          for (int m = LPR; m < 32; m <<= 1) {
            dk[t][c] += __shfl_xor_sync(0xffffffffu, dk[t][c], m);
            dv[t][c] += __shfl_xor_sync(0xffffffffu, dv[t][c], m);
          }
        __syncthreads();
        if ((tid & 31) < LPR) {
#pragma unroll
          for (int c = 0; c < V; ++c) {
            if (c >= left) break;
            part[tid >> 5][d0 + c] = dk[t][c];
            part[tid >> 5][a.dim + d0 + c] = dv[t][c];
          }
        }
        __syncthreads();
        float* dst = far_slot(a, g, slot, hk, t0 + t);
        for (int e = tid; e < 2 * a.dim; e += 256) {
          float x = 0.f;
#pragma unroll
          for (int w = 0; w < 8; ++w) x += part[w][e];
          dst[e] = x;
        }
      }
    }
    i0 = s.end;
  }
}

template <typename T>
int far_launch(const AttnArgs& a, const AttnGrad& g, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  auto on = [&](const void* p, long long row, long long head) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && row % V == 0 && head % V == 0;
  };
  const bool vec = a.dim % V == 0 && on(a.q, a.q_row, a.q_head) && on(a.k, a.k_row, a.k_head) &&
                   on(a.v, a.v_row, a.v_head) && on(g.grad, g.grad_row, g.grad_head);
  const dim3 grid(ceil_div(a.n, kFarRows), a.kv_heads);
  if (a.dim <= 4 * V) attn_far_kernel<T, 4><<<grid, 256, 0, st>>>(a, g, vec);
  else if (a.dim <= 8 * V) attn_far_kernel<T, 8><<<grid, 256, 0, st>>>(a, g, vec);
  else if (a.dim <= 16 * V) attn_far_kernel<T, 16><<<grid, 256, 0, st>>>(a, g, vec);
  else attn_far_kernel<T, 32><<<grid, 256, 0, st>>>(a, g, vec);
  OCNN_LAUNCH_OK("attn_far_kernel");
  return OCNN_OK;
}

template <typename T, int DP>
int forward_launch(const AttnArgs& a, void* out, float* lse, bool vec, cudaStream_t st) {
  static PerDeviceOnce once;
  const size_t bytes = smem_bytes<DP>(3, 1);
  const int status = once.run([&]() -> int {
    OCNN_CUDA_OK(cudaFuncSetAttribute(attn_simt_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    return OCNN_OK;
  });
  if (status != OCNN_OK) return status;
  attn_simt_kernel<T, DP><<<dim3(ceil_div(a.n, kB), a.heads), kThreads, bytes, st>>>(a, (T*)out, lse, vec);
  OCNN_LAUNCH_OK("attn_simt_kernel");
  return OCNN_OK;
}

template <typename T, int DP>
int backward_launch(const AttnArgs& a, const AttnGrad& g, bool vec, cudaStream_t st) {
  static PerDeviceOnce once;
  const size_t dq_bytes = smem_bytes<DP>(4, 1), dkv_bytes = smem_bytes<DP>(4, 2);
  const int status = once.run([&]() -> int {
    OCNN_CUDA_OK(cudaFuncSetAttribute(attn_simt_dq_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)dq_bytes));
    OCNN_CUDA_OK(cudaFuncSetAttribute(attn_simt_dkv_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)dkv_bytes));
    return OCNN_OK;
  });
  if (status != OCNN_OK) return status;
  attn_simt_dq_kernel<T, DP><<<dim3(ceil_div(a.n, kB), a.heads), kThreads, dq_bytes, st>>>(a, g, vec);
  OCNN_LAUNCH_OK("attn_simt_dq_kernel");
  if (g.dk == nullptr) return OCNN_OK;
  if (a.sinks > 0) {
    int far = far_launch<T>(a, g, st);
    if (far == OCNN_OK) far = attn_far_join(a, g, st);
    if (far != OCNN_OK) return far;
  }
  attn_simt_dkv_kernel<T, DP><<<dim3(ceil_div(a.n, kB), a.kv_heads), kThreads, dkv_bytes, st>>>(a, g, vec);
  OCNN_LAUNCH_OK("attn_simt_dkv_kernel");
  return OCNN_OK;
}

template <typename F>
int by_type(int dtype, int dim, F f) {
  auto width = [&](auto t) {
    using T = decltype(t);
    if (dim <= 32) return f(t, std::integral_constant<int, 32>());
    if (dim <= 64) return f(t, std::integral_constant<int, 64>());
    return f(T(), std::integral_constant<int, 128>());
  };
  if (dtype == OCNN_F32) return width(float());
  if (dtype == OCNN_BF16) return width(__nv_bfloat16());
  return width(__half());
}

}  // namespace

int attn_simt_forward(const AttnArgs& a, int dtype, void* out, float* lse, bool vec, cudaStream_t st) {
  return by_type(dtype, a.dim, [&](auto t, auto dp) -> int {
    return forward_launch<decltype(t), decltype(dp)::value>(a, out, lse, vec, st);
  });
}
int attn_simt_backward(const AttnArgs& a, const AttnGrad& g, int dtype, bool vec, cudaStream_t st) {
  return by_type(dtype, a.dim, [&](auto t, auto dp) -> int {
    return backward_launch<decltype(t), decltype(dp)::value>(a, g, vec, st);
  });
}

}  // namespace ocnn
