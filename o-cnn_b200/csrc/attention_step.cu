// Attention of one new node per sequence against a cache of the nodes before it.
//
// Sequence b stands at position p = lengths[b]: its key and value go into the cache, and its queries see the positions
// p - window + 1 .. p and the first `sinks`.  A cache of `capacity` places holds position x at place x while x < sinks
// and at sinks + (x - sinks) mod (capacity - sinks) from there on, so one that has room for sinks + window nodes serves a
// sequence of any length.
//
// Bound: HBM (every visible row of the cache is read once for all query heads that share it).  A cluster of CTAs takes a
// sequence's key head, each CTA a stretch of the visible positions, each warp its rows with a running maximum and sum;
// the parts are joined in shared memory, first the warps', then the CTAs' through the cluster's: one launch, no
// workspace, the same bits every time.
// float16 holds nothing below 2^-24: the rounded p, at most 1, is kept at 2^15 p there.
//   16-bit caches: every warp copies its rows, 16 at a time, into a ring of its own (cp.async, one row after the other:
//   rolled caches and the new row need no case of their own) and multiplies them with mma.sync, 16 query heads at a time.
//   On the CUDA cores, a product and a shuffle per value for each query head, 64 sequences of 4100 rows, 16 heads over 4
//   of 128, took 510 us, with a bulk copy per row (about 65 cycles each, one after the other) 302 us, now 119.
//   fp32 caches: a warp reads whole rows, 16 bytes a lane, on the CUDA cores.
#include <cooperative_groups.h>

#include "attention.cuh"
#include "mma.cuh"

namespace ocnn {
namespace {

namespace cg = cooperative_groups;

struct StepArgs {
  const void *q, *k, *v;
  long long q_row, q_head, k_row, k_head, v_row, v_head;
  void *kc, *vc;
  long long kc_seq, kc_pos, kc_head, vc_seq, vc_pos, vc_head;
  void* out;
  const int* lengths;
  int batch, heads, kv_heads, dim, capacity, window, sinks, rolls;
  float scale_log2;
};

// What a sequence's new node sees: its visible positions as a list, the first ones, then the window.
struct StepKeys {
  int p, lo, n_first, n;
  bool live, full;
  __device__ __forceinline__ StepKeys(const StepArgs& a, int b) {
    p = a.lengths[b];
    full = !a.rolls && p >= a.capacity;                        // no room: the output says so, the cache stays
    live = p >= 0 && !full;
    lo = live && p >= a.window ? p - a.window + 1 : 0;
    n_first = min(a.sinks, lo);
    n = live ? n_first + p - lo + 1 : 0;
  }
  __device__ __forceinline__ int position(int t) const { return t < n_first ? t : lo + t - n_first; }
};
__device__ __forceinline__ int step_place(const StepArgs& a, int x) {
  return x < a.capacity ? x : a.sinks + (x - a.sinks) % max(a.capacity - a.sinks, 1);
}

constexpr int kStepThreads = 256, kStepWarps = kStepThreads / 32, kStepUnroll = 4;

template <typename T>
struct Vec16 { static constexpr int n = 16 / sizeof(T); };

template <typename T>
__device__ __forceinline__ void unpack16(const uint4& w, float (&x)[Vec16<T>::n]) {
  const T* t = reinterpret_cast<const T*>(&w);
#pragma unroll
  for (int i = 0; i < Vec16<T>::n; ++i) x[i] = to_f32(t[i]);
}

// G query heads (a power of two; those behind the group's last do nothing) against LPK lanes per row.
template <typename T, int G, int LPK>
__global__ void __launch_bounds__(kStepThreads) attn_step_kernel(const StepArgs a) {
  constexpr int V = Vec16<T>::n, kRows = 32 / LPK;             // rows a warp reads at a time
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
  const int group = a.heads / a.kv_heads, chunks = (group + G - 1) / G;
  const int hk = blockIdx.y / chunks, g0 = (blockIdx.y % chunks) * G, b = blockIdx.z;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, sub = lane % LPK, row = lane / LPK;
  __shared__ float so[kStepWarps][G][LPK * V];
  __shared__ float sm[kStepWarps][G], sl[kStepWarps][G];
  const StepKeys keys(a, b);
  const int d0 = sub * V;
  const bool in = d0 < a.dim;

  float q[G][V], acc[G][V] = {}, top[G], total[G] = {};
#pragma unroll
  for (int g = 0; g < G; ++g) {
    top[g] = -INFINITY;
    uint4 w = make_uint4(0, 0, 0, 0);
    if (in && g0 + g < group)
      w = *reinterpret_cast<const uint4*>((const T*)a.q + b * a.q_row + (hk * group + g0 + g) * a.q_head + d0);
    unpack16<T>(w, q[g]);
#pragma unroll
    for (int i = 0; i < V; ++i) q[g][i] *= a.scale_log2;
  }
  const T* kc = (const T*)a.kc + b * a.kc_seq + hk * a.kc_head + d0;
  const T* vc = (const T*)a.vc + b * a.vc_seq + hk * a.vc_head + d0;
  const T* kn = (const T*)a.k + b * a.k_row + hk * a.k_head + d0;
  const T* vn = (const T*)a.v + b * a.v_row + hk * a.v_head + d0;
  const int per = (keys.n + parts - 1) / parts, end = min(keys.n, (part + 1) * per);
  constexpr int kStride = kStepWarps * kRows;
  for (int t0 = part * per + warp * kRows + row; t0 - row < end; t0 += kStride * kStepUnroll) {
    uint4 kw[kStepUnroll], vw[kStepUnroll];
#pragma unroll
    for (int u = 0; u < kStepUnroll; ++u) {
      const int t = t0 + u * kStride;
      kw[u] = vw[u] = make_uint4(0, 0, 0, 0);
      if (t < end && in) {
        const int x = keys.position(t), place = step_place(a, x);
        const bool newest = x == keys.p;                       // (its place in the cache is being written)
        kw[u] = *reinterpret_cast<const uint4*>(newest ? kn : kc + place * a.kc_pos);
        vw[u] = *reinterpret_cast<const uint4*>(newest ? vn : vc + place * a.vc_pos);
      }
    }
    float s[kStepUnroll][G];
#pragma unroll
    for (int u = 0; u < kStepUnroll; ++u) {
      float k[V];
      unpack16<T>(kw[u], k);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        float x = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) x = fmaf(q[g][i], k[i], x);
#pragma unroll
        for (int m = LPK / 2; m > 0; m >>= 1) x += __shfl_xor_sync(0xffffffffu, x, m);
        s[u][g] = t0 + u * kStride < end ? x : -INFINITY;
      }
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float m = top[g];
#pragma unroll
      for (int u = 0; u < kStepUnroll; ++u) m = fmaxf(m, s[u][g]);
      const float base = m == -INFINITY ? 0.f : m, keep = exp2f(top[g] - base);
      top[g] = m;
      total[g] *= keep;
#pragma unroll
      for (int i = 0; i < V; ++i) acc[g][i] *= keep;
#pragma unroll
      for (int u = 0; u < kStepUnroll; ++u) {
        s[u][g] = exp2f(s[u][g] - base);
        total[g] += s[u][g];
      }
    }
#pragma unroll
    for (int u = 0; u < kStepUnroll; ++u) {
      float v[V];
      unpack16<T>(vw[u], v);
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int i = 0; i < V; ++i) acc[g][i] = fmaf(s[u][g], v[i], acc[g][i]);
    }
  }
  // the rows a warp read side by side
#pragma unroll
  for (int g = 0; g < G; ++g) {
#pragma unroll
    for (int x = LPK; x < 32; x <<= 1) {
      const float m = fmaxf(top[g], __shfl_xor_sync(0xffffffffu, top[g], x)), base = m == -INFINITY ? 0.f : m;
      const float keep = exp2f(top[g] - base);
      total[g] *= keep;
      total[g] += __shfl_xor_sync(0xffffffffu, total[g], x);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        acc[g][i] *= keep;
        acc[g][i] += __shfl_xor_sync(0xffffffffu, acc[g][i], x);
      }
      top[g] = m;
    }
    if (row == 0) {
#pragma unroll
      for (int i = 0; i < V; ++i) so[warp][g][d0 + i] = acc[g][i];
      if (sub == 0) {
        sm[warp][g] = top[g];
        sl[warp][g] = total[g];
      }
    }
  }
  __syncthreads();
  // the warps of the CTA, into warp 0's place (each value by the thread that owns it)
  for (int e = tid; e < G * LPK * V; e += kStepThreads) {
    const int g = e / (LPK * V), d = e % (LPK * V);
    float m = -INFINITY, x = 0.f;
#pragma unroll
    for (int w = 0; w < kStepWarps; ++w) m = fmaxf(m, sm[w][g]);
    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int w = 0; w < kStepWarps; ++w) x += exp2f(sm[w][g] - base) * so[w][g][d];
    so[0][g][d] = x;
  }
  float m = -INFINITY, l = 0.f;
  if (tid < G) {
    for (int w = 0; w < kStepWarps; ++w) m = fmaxf(m, sm[w][tid]);
    for (int w = 0; w < kStepWarps; ++w) l += exp2f(sm[w][tid] - (m == -INFINITY ? 0.f : m)) * sl[w][tid];
  }
  __syncthreads();
  if (tid < G) {
    sm[0][tid] = m;
    sl[0][tid] = l;
  }
  cluster.sync();
  // the CTAs of the cluster: each writes its share of the heads' channels
  const int each = (G * LPK * V + parts - 1) / parts;
  for (int e = part * each + tid; e < min(G * LPK * V, (part + 1) * each); e += kStepThreads) {
    const int g = e / (LPK * V), d = e % (LPK * V);
    if (g0 + g >= group || d >= a.dim) continue;
    float m = -INFINITY, x = 0.f, l = 0.f;
    for (int c = 0; c < parts; ++c) m = fmaxf(m, *cluster.map_shared_rank(&sm[0][g], c));
    const float base = m == -INFINITY ? 0.f : m;
    for (int c = 0; c < parts; ++c) {
      const float f = exp2f(*cluster.map_shared_rank(&sm[0][g], c) - base);
      l += f * *cluster.map_shared_rank(&sl[0][g], c);
      x += f * *cluster.map_shared_rank(&so[0][g][d], c);
    }
    const float y = keys.full ? __int_as_float(0x7fc00000) : keys.n == 0 ? 0.f : x / l;
    ((T*)a.out)[((long long)b * a.heads + hk * group + g0 + g) * a.dim + d] = from_f32<T>(y);
  }
  if (part == 0 && g0 == 0 && keys.live && tid < 2 * LPK && in) {    // (lanes 0 .. 2 LPK - 1 hold every d0 twice)
    const int place = step_place(a, keys.p);
    T* dst = tid < LPK ? (T*)a.kc + b * a.kc_seq + place * a.kc_pos + hk * a.kc_head
                       : (T*)a.vc + b * a.vc_seq + place * a.vc_pos + hk * a.vc_head;
    *reinterpret_cast<uint4*>(dst + d0) = *reinterpret_cast<const uint4*>(tid < LPK ? kn : vn);
  }
  cluster.sync();                                              // (no CTA leaves while its shared memory is read)
}

// ---- 16-bit caches ------------------------------------------------------------------------------------------------
constexpr int kMmaWarps = 4, kMmaHeads = 16, kMmaRows = 16;    // warps, query heads of a CTA, rows of a tile

template <int DP>
struct StepShape {
  static constexpr int kPitch = DP * 2 + 16;                   // (an odd number of 16-byte pieces: ldmatrix meets no bank twice)
  static constexpr int kTile = 2 * kMmaRows * kPitch;          // K, then V
  static constexpr int kTiles = DP > 64 ? 2 : 3;               // of a warp's ring
  static constexpr int kRing = kMmaWarps * kTiles * kTile, kJoin = kMmaWarps * kMmaHeads * (DP + 2) * 4;
  static constexpr int kBytes = kRing > kJoin ? kRing : kJoin;
};

template <bool HALF, int DP>
__global__ void __launch_bounds__(32 * kMmaWarps) attn_step_mma_kernel(const StepArgs a) {
  using Shape = StepShape<DP>;
  using T = typename std::conditional<HALF, __half, __nv_bfloat16>::type;
  constexpr int KS = DP / 16, kThreads = 32 * kMmaWarps, kChunks = DP / 8, kStep = 32 / kChunks;
  constexpr float up = HALF ? 15.f : 0.f;                        // (p is kept at 2^up p, and so is its sum)
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
  const int group = a.heads / a.kv_heads, chunks = (group + kMmaHeads - 1) / kMmaHeads;
  const int hk = blockIdx.y / chunks, g0 = (blockIdx.y % chunks) * kMmaHeads, b = blockIdx.z;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  extern __shared__ __align__(128) uint8_t smem[];
  const StepKeys keys(a, b);
  // this CTA's stretch of the list, in whole rounds of its warps
  constexpr int kRound = kMmaWarps * kMmaRows;
  const int rounds = (keys.n + kRound - 1) / kRound, per = (rounds + parts - 1) / parts * kRound;
  const int t_begin = min(part * per, keys.n), t_end = min(t_begin + per, keys.n);
  const int ksteps = (a.dim + 15) / 16, full = a.dim / 8;

  uint8_t* ring = smem + warp * Shape::kTiles * Shape::kTile;
  const uint8_t* kc = (const uint8_t*)((const T*)a.kc + b * a.kc_seq + hk * a.kc_head);
  const uint8_t* vc = (const uint8_t*)((const T*)a.vc + b * a.vc_seq + hk * a.vc_head);
  const uint8_t* kn = (const uint8_t*)((const T*)a.k + b * a.k_row + hk * a.k_head);
  const uint8_t* vn = (const uint8_t*)((const T*)a.v + b * a.v_row + hk * a.v_head);
  auto fetch = [&](int i) {                                     // tile i of this warp, if there is one
    const int t0 = t_begin + i * kRound + warp * kMmaRows;
    if (t0 < t_end) {
      const int x = keys.position(min(t0 + (lane & 15), t_end - 1));
      const int where = t0 + (lane & 15) < t_end ? (x == keys.p ? -1 : step_place(a, x)) : -2;   // -1: the new row, -2: none
      const uint32_t dst = smem_u32(ring + i % Shape::kTiles * Shape::kTile);
      const int c = lane % kChunks;
#pragma unroll
      for (int it = 0; it < kMmaRows / kStep; ++it) {
        const int r = it * kStep + lane / kChunks, place = __shfl_sync(0xffffffffu, where, r);
        if (c >= 2 * ksteps) continue;                          // (zeros up to a multiple of 16 channels, and in rows there are none of)
        const uint32_t bytes = place >= -1 && c < full ? 16u : 0u;
        const uint8_t* k = place < 0 ? kn : kc + place * (a.kc_pos * 2);
        const uint8_t* v = place < 0 ? vn : vc + place * (a.vc_pos * 2);
        cp_async16(dst + r * Shape::kPitch + c * 16, bytes != 0 ? k + c * 16 : kn, bytes);
        cp_async16(dst + (kMmaRows + r) * Shape::kPitch + c * 16, bytes != 0 ? v + c * 16 : vn, bytes);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < Shape::kTiles - 1; ++i) fetch(i);

  uint32_t q[KS][4];
#pragma unroll
  for (int k = 0; k < KS; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int g = g0 + (lane >> 2) + 8 * (e & 1), d = 16 * k + 2 * (lane & 3) + 8 * (e >> 1);
      q[k][e] = g < group && d < a.dim
                    ? *reinterpret_cast<const uint32_t*>((const T*)a.q + b * a.q_row + (hk * group + g) * a.q_head + d)
                    : 0u;
    }
  float o[2 * KS][4] = {}, top[2] = {-INFINITY, -INFINITY}, total[2] = {};
  for (int i = 0; t_begin + i * kRound < t_end; ++i) {
    fetch(i + Shape::kTiles - 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(Shape::kTiles - 1) : "memory");
    __syncwarp();
    const int t0 = t_begin + i * kRound + warp * kMmaRows;
    if (t0 < t_end) {
      const uint32_t kb = smem_u32(ring + i % Shape::kTiles * Shape::kTile);
      float sc[2][4] = {};
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        if (k >= ksteps) break;
        uint32_t f[4];
        ldmatrix4(rows_frag(kb, Shape::kPitch) + 32 * k, f);
        mma16816<HALF>(sc[0], q[k], f[0], f[1]);
        mma16816<HALF>(sc[1], q[k], f[2], f[3]);
      }
      uint32_t w[4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {                              // query heads lane / 4 and lane / 4 + 8
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int t = t0 + 8 * (e >> 1) + 2 * (lane & 3) + (e & 1);
          x[e] = t < t_end ? sc[e >> 1][2 * h + (e & 1)] * a.scale_log2 : -INFINITY;
        }
        float m = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = fmaxf(top[h], fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2)));
        const float base = m == -INFINITY ? 0.f : m;
        if (__any_sync(0xffffffffu, m != top[h])) {
          const float keep = exp2_approx(top[h] - base);
          top[h] = m;
          total[h] *= keep;
#pragma unroll
          for (int n = 0; n < 2 * KS; ++n) {
            o[n][2 * h] *= keep;
            o[n][2 * h + 1] *= keep;
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = exp2_approx(x[e] + (up - base));
          total[h] += x[e];
        }
        // (rounded to the data's type for the product; the sum is of the unrounded values)
        w[h] = pack2(x[0], x[1], HALF);
        w[2 + h] = pack2(x[2], x[3], HALF);
      }
      const uint32_t vb = columns_frag(kb + kMmaRows * Shape::kPitch, Shape::kPitch);
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        if (k >= ksteps) break;
        uint32_t f[4];
        ldmatrix4t(vb + 32 * k, f);
        mma16816<HALF>(o[2 * k], w, f[0], f[1]);
        mma16816<HALF>(o[2 * k + 1], w, f[2], f[3]);
      }
    }
    __syncwarp();                                               // (the tile is read: the next copies may go there)
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  // ---------------- the warps' parts, in the rings' place ----------------
  __syncthreads();
  float* so = reinterpret_cast<float*>(smem);                   // [warp][head][DP], then maxima and sums
  float* sm = so + kMmaWarps * kMmaHeads * DP;
  float* sl = sm + kMmaWarps * kMmaHeads;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int head = (lane >> 2) + 8 * h;
    float l = total[h];
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if ((lane & 3) == 0) {
      sm[warp * kMmaHeads + head] = top[h];
      sl[warp * kMmaHeads + head] = l;
    }
#pragma unroll
    for (int n = 0; n < 2 * KS; ++n)
      *reinterpret_cast<float2*>(so + (warp * kMmaHeads + head) * DP + 8 * n + 2 * (lane & 3)) =
          make_float2(o[n][2 * h], o[n][2 * h + 1]);
  }
  __syncthreads();
  const int heads = min(kMmaHeads, group - g0);
  for (int e = tid; e < heads * DP; e += kThreads) {            // into warp 0's place, each value by the thread that owns it
    const int head = e / DP;
    float m = -INFINITY, x = 0.f;
#pragma unroll
    for (int w = 0; w < kMmaWarps; ++w) m = fmaxf(m, sm[w * kMmaHeads + head]);
    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int w = 0; w < kMmaWarps; ++w) x += exp2f(sm[w * kMmaHeads + head] - base) * so[w * kMmaHeads * DP + e];
    so[e] = x;
  }
  float m = -INFINITY, l = 0.f;
  if (tid < heads) {
    for (int w = 0; w < kMmaWarps; ++w) m = fmaxf(m, sm[w * kMmaHeads + tid]);
    for (int w = 0; w < kMmaWarps; ++w) l += exp2f(sm[w * kMmaHeads + tid] - (m == -INFINITY ? 0.f : m)) * sl[w * kMmaHeads + tid];
  }
  __syncthreads();
  if (tid < heads) {
    sm[tid] = m;
    sl[tid] = l;
  }
  if (parts > 1) cluster.sync();
  else __syncthreads();
  // ---------------- the CTAs' parts: each writes its share of the channels ----------------
  const int each = (heads * a.dim + parts - 1) / parts;
  for (int e = part * each + tid; e < min(heads * a.dim, (part + 1) * each); e += kThreads) {
    const int head = e / a.dim, d = e - head * a.dim;
    float m = -INFINITY, x = 0.f, l = 0.f;
    for (int c = 0; c < parts; ++c) m = fmaxf(m, *cluster.map_shared_rank(sm + head, c));
    const float base = m == -INFINITY ? 0.f : m;
    for (int c = 0; c < parts; ++c) {
      const float f = exp2f(*cluster.map_shared_rank(sm + head, c) - base);
      l += f * *cluster.map_shared_rank(sl + head, c);
      x += f * *cluster.map_shared_rank(so + head * DP + d, c);
    }
    const float y = keys.full ? __int_as_float(0x7fc00000) : keys.n == 0 ? 0.f : x / l;
    ((T*)a.out)[((long long)b * a.heads + hk * group + g0 + head) * a.dim + d] = from_f32<T>(y);
  }
  if (part == 0 && g0 == 0 && keys.live && tid < a.dim / 4) {   // the new row: dim / 8 pieces of K, then of V
    const int piece = tid % full * 16, place = step_place(a, keys.p);
    const bool v = tid >= full;
    uint8_t* dst = (v ? (uint8_t*)((T*)a.vc + b * a.vc_seq + place * a.vc_pos + hk * a.vc_head)
                      : (uint8_t*)((T*)a.kc + b * a.kc_seq + place * a.kc_pos + hk * a.kc_head)) + piece;
    *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>((v ? vn : kn) + piece);
  }
  if (parts > 1) cluster.sync();                                // (no CTA leaves while its shared memory is read)
}

template <bool HALF, int DP>
int step_mma_launch(const StepArgs& a, int parts, cudaStream_t st) {
  auto kernel = attn_step_mma_kernel<HALF, DP>;
  static PerDeviceOnce once;
  const int status = once.run([&]() -> int {
    OCNN_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    OCNN_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, StepShape<DP>::kBytes));
    return OCNN_OK;
  });
  if (status != OCNN_OK) return status;
  const int chunks = ceil_div(a.heads / a.kv_heads, kMmaHeads);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(parts, a.kv_heads * chunks, a.batch);
  cfg.blockDim = dim3(32 * kMmaWarps);
  cfg.dynamicSmemBytes = StepShape<DP>::kBytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = parts;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = parts > 1 ? 1 : 0;
  OCNN_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, a));
  OCNN_LAUNCH_OK("attn_step_mma_kernel");
  return OCNN_OK;
}
template <bool HALF>
int step_mma_by_width(const StepArgs& a, int parts, cudaStream_t st) {
  if (a.dim <= 32) return step_mma_launch<HALF, 32>(a, parts, st);
  if (a.dim <= 64) return step_mma_launch<HALF, 64>(a, parts, st);
  return step_mma_launch<HALF, 128>(a, parts, st);
}

template <typename T, int G, int LPK>
int step_launch(const StepArgs& a, int parts, cudaStream_t st) {
  static PerDeviceOnce once;
  const int status = once.run([&]() -> int {
    OCNN_CUDA_OK(cudaFuncSetAttribute(attn_step_kernel<T, G, LPK>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    return OCNN_OK;
  });
  if (status != OCNN_OK) return status;
  const int chunks = ceil_div(a.heads / a.kv_heads, G);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(parts, a.kv_heads * chunks, a.batch);
  cfg.blockDim = dim3(kStepThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = parts;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  OCNN_CUDA_OK(cudaLaunchKernelEx(&cfg, attn_step_kernel<T, G, LPK>, a));
  OCNN_LAUNCH_OK("attn_step_kernel");
  return OCNN_OK;
}

template <typename T, int LPK>
int step_by_group(const StepArgs& a, int parts, cudaStream_t st) {
  const int group = a.heads / a.kv_heads;
  if (group == 1) return step_launch<T, 1, LPK>(a, parts, st);
  if (group == 2) return step_launch<T, 2, LPK>(a, parts, st);
  if (group <= 4) return step_launch<T, 4, LPK>(a, parts, st);
  return step_launch<T, 8, LPK>(a, parts, st);
}

template <typename T>
int step_by_width(const StepArgs& a, int parts, cudaStream_t st) {
  constexpr int V = Vec16<T>::n, kMost = kMaxHeadDim / V;        // 16 lanes a row of 128, fp32: 32
  if (a.dim <= kMost / 4 * V) return step_by_group<T, kMost / 4>(a, parts, st);
  if (a.dim <= kMost / 2 * V) return step_by_group<T, kMost / 2>(a, parts, st);
  return step_by_group<T, kMost>(a, parts, st);
}

bool on16(const void* p, std::initializer_list<long long> strides, int size) {
  bool ok = reinterpret_cast<uintptr_t>(p) % 16 == 0;
  for (long long s : strides) ok = ok && s * size % 16 == 0;
  return ok;
}

}  // namespace
}  // namespace ocnn

using namespace ocnn;

extern "C" int ocnn_octree_attention_step(const ocnn_attention_cache* c, const void* q_dev, const int64_t q_stride[2],
                                          const void* k_dev, const int64_t k_stride[2], const void* v_dev,
                                          const int64_t v_stride[2], void* out_dev, int heads, int window, int sinks,
                                          float scale, void* stream) {
  OCNN_REQUIRE(c != nullptr && c->batch >= 0 && c->capacity >= 1 && c->kv_heads >= 1 && c->dim >= 1,
               "ocnn_octree_attention_step: bad cache");
  OCNN_REQUIRE(c->dtype >= OCNN_F32 && c->dtype <= OCNN_F16, "ocnn_octree_attention_step: bad dtype %d", c->dtype);
  OCNN_REQUIRE(heads >= 1 && heads % c->kv_heads == 0, "ocnn_octree_attention_step: %d heads over %d key heads", heads,
               c->kv_heads);
  OCNN_REQUIRE(window >= 0 && sinks >= 0, "ocnn_octree_attention_step: window and sinks must not be negative");
  const int size = c->dtype == OCNN_F32 ? 4 : 2;
  if (c->batch > 65535 || heads > 65535)                       // (the grid's y and z)
    return fail(OCNN_ERR_UNSUPPORTED, "ocnn_octree_attention_step: %d sequences, %d heads (up to 65535 each)", c->batch, heads);
  if (c->dim > kMaxHeadDim || c->dim * size % 16 != 0)
    return fail(OCNN_ERR_UNSUPPORTED, "ocnn_octree_attention_step: heads of %d channels (multiples of 16 bytes up to %d)",
                c->dim, kMaxHeadDim);
  if (c->batch == 0) return OCNN_OK;
  OCNN_REQUIRE(q_dev && k_dev && v_dev && out_dev && c->k_dev && c->v_dev && c->lengths_dev,
               "ocnn_octree_attention_step: null pointer");
  OCNN_REQUIRE(on16(q_dev, {q_stride[0], q_stride[1]}, size) && on16(k_dev, {k_stride[0], k_stride[1]}, size) &&
                   on16(v_dev, {v_stride[0], v_stride[1]}, size) &&
                   on16(c->k_dev, {c->k_stride[0], c->k_stride[1], c->k_stride[2]}, size) &&
                   on16(c->v_dev, {c->v_stride[0], c->v_stride[1], c->v_stride[2]}, size),
               "ocnn_octree_attention_step: rows must start on 16-byte boundaries");
  StepArgs a = {};
  a.q = q_dev, a.q_row = q_stride[0], a.q_head = q_stride[1];
  a.k = k_dev, a.k_row = k_stride[0], a.k_head = k_stride[1];
  a.v = v_dev, a.v_row = v_stride[0], a.v_head = v_stride[1];
  a.kc = c->k_dev, a.kc_seq = c->k_stride[0], a.kc_pos = c->k_stride[1], a.kc_head = c->k_stride[2];
  a.vc = c->v_dev, a.vc_seq = c->v_stride[0], a.vc_pos = c->v_stride[1], a.vc_head = c->v_stride[2];
  a.out = out_dev;
  a.lengths = c->lengths_dev;
  a.batch = c->batch, a.heads = heads, a.kv_heads = c->kv_heads, a.dim = c->dim, a.capacity = c->capacity;
  a.window = window == 0 ? INT_MAX : window;
  a.sinks = window == 0 ? 0 : sinks;
  a.rolls = window > 0 && (long long)window + sinks <= c->capacity;
  a.scale_log2 = scale * 1.4426950408889634f;
  // CTAs per sequence and key head, doubled until the grid has four per SM, as long as each still has 64 rows to read.  (At 128
  // channels three fit an SM: the 64 sequences above are 1024 CTAs on 444 places, 2.3 rounds.  More parts took 122 us.)
  const bool f32 = c->dtype == OCNN_F32;
  const long long pairs = (long long)a.batch * a.kv_heads;
  const long long most = a.rolls ? (long long)window + sinks : c->capacity;
  int parts = 1;
  while (parts < 16 && pairs * parts < 4LL * sm_count() && most >= 2LL * parts * 64) parts *= 2;
  cudaStream_t st = (cudaStream_t)stream;
  if (f32) return step_by_width<float>(a, parts, st);
  return c->dtype == OCNN_F16 ? step_mma_by_width<true>(a, parts, st) : step_mma_by_width<false>(a, parts, st);
}
