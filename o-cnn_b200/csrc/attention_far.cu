// What the nodes beyond the window add to the gradients of their sequence's first nodes (see far_slot in attention.cuh), for
// 16-bit data: for the sequence's first nodes j (up to 16 at a time) and all far rows i of a block,
//     s = k_j . q_i,  dP = v_j . dO_i,  p = exp2(scale s - lse_i),  ds = p (dP - delta_i);  dv_j += p dO_i,  dk_j += ds q_i
// A warp takes 16 rows (query heads of nodes) at a time into a ring of its own and forms the four products with mma.sync,
// the first nodes as the operand's 16 rows; p and ds are rounded to the data's type for the second two, as everywhere in
// the gradients.  Bound: reading q and dO once more (65 k nodes, 16 heads of 128: 0.54 GB).  On the CUDA cores, a product
// and a chain of shuffles per row and first node, this took 890 us there with four first nodes, now 190.
#include "attention.cuh"
#include "mma.cuh"

namespace ocnn {
namespace {

constexpr int kFarWarps = 4, kFarTile = 16;

template <int DP>
struct FarShape {
  static constexpr int kPitch = DP * 2 + 16;                   // (an odd number of 16-byte pieces: ldmatrix meets no bank twice)
  static constexpr int kTile = 2 * kFarTile * kPitch;          // q, then dO
  static constexpr int kRing = kFarWarps * 2 * kTile, kJoin = kFarWarps * 16 * DP * 4;
  static constexpr int kBytes = kRing > kJoin ? kRing : kJoin;
};

template <bool HALF, int DP>
__global__ void __launch_bounds__(32 * kFarWarps) attn_far_mma_kernel(const AttnArgs a, const AttnGrad g) {
  using Shape = FarShape<DP>;
  using T = typename std::conditional<HALF, __half, __nv_bfloat16>::type;
  constexpr int KS = DP / 16, kThreads = 32 * kFarWarps, kChunks = DP / 8, kStep = 32 / kChunks;
  extern __shared__ __align__(128) uint8_t smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int hk = blockIdx.y, group = a.heads / a.kv_heads;
  const int r0 = blockIdx.x * kFarRows, r1 = min(a.n, r0 + kFarRows);
  const int ksteps = (a.dim + 15) / 16, full = a.dim / 8;
  // p is kept at p * prob_up, ds at ds * kept_at, as in the other kernels
  constexpr float prob_up = HALF ? kProbUp : 1.f, prob_log = HALF ? kProbUpLog : 0.f;
  const float kept_at = HALF ? grad_scale_of(g.largest, r0, r1) : 1.f, after = kept_at / prob_up;
  uint8_t* ring = smem + warp * 2 * Shape::kTile;
  const uint8_t* qb = (const uint8_t*)((const T*)a.q + (long long)hk * group * a.q_head);
  const uint8_t* gb = (const uint8_t*)((const T*)g.grad + (long long)hk * group * g.grad_head);
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
    for (int t0 = 0; t0 < sinks; t0 += 16) {
      const int first = s.start + t0, many = min(16, sinks - t0);
      // rows that see the first of these nodes from far (the others' begin a node later each), heads side by side
      const int from = s.end - first > a.window ? max(i0, first + a.window) : end;
      const int count = max(0, end - from) * group;
      uint32_t k[KS][4], v[KS][4];
#pragma unroll
      for (int c = 0; c < KS; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int t = (lane >> 2) + 8 * (e & 1), d = 16 * c + 2 * (lane & 3) + 8 * (e >> 1), j = first + t;
          const bool live = count > 0 && t < many && d < a.dim && (a.mask == nullptr || a.mask[j] != 0);
          k[c][e] = live ? *reinterpret_cast<const uint32_t*>((const T*)a.k + j * a.k_row + hk * a.k_head + d) : 0u;
          v[c][e] = live ? *reinterpret_cast<const uint32_t*>((const T*)a.v + j * a.v_row + hk * a.v_head + d) : 0u;
        }
      bool kept[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int t = (lane >> 2) + 8 * h;
        kept[h] = t < many && (a.mask == nullptr || a.mask[first + t] != 0);
      }
      float dk[2 * KS][4] = {}, dv[2 * KS][4] = {};
      // a lane knows row (lane mod 16) of a tile: its node, its place and its statistics
      struct Row { int i, h; float lse, delta; };
      auto row_of = [&](int tile) {
        const int e = tile * kFarTile + (lane & 15);
        Row r = {-1, 0, 0.f, 0.f};
        if (e < count) {
          r.i = from + e / group;
          r.h = e - (r.i - from) * group;
          const long long at = (long long)(hk * group + r.h) * a.n + r.i;
          r.lse = g.lse[at];
          r.delta = g.delta[at];
        }
        return r;
      };
      auto fetch = [&](const Row& row, int place) {
        const uint32_t dst = smem_u32(ring + place * Shape::kTile);
        const int c = lane % kChunks;
#pragma unroll
        for (int it = 0; it < kFarTile / kStep; ++it) {
          const int r = it * kStep + lane / kChunks;
          const int i = __shfl_sync(0xffffffffu, row.i, r), h = __shfl_sync(0xffffffffu, row.h, r);
          if (c >= 2 * ksteps) continue;
          const bool live = i >= 0 && c < full;
          cp_async16(dst + r * Shape::kPitch + c * 16, live ? qb + (i * a.q_row + h * a.q_head) * 2 + c * 16 : qb, live ? 16u : 0u);
          cp_async16(dst + (kFarTile + r) * Shape::kPitch + c * 16,
                     live ? gb + (i * g.grad_row + h * g.grad_head) * 2 + c * 16 : gb, live ? 16u : 0u);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
      const int tiles = (count + kFarTile - 1) / kFarTile;
      Row row = row_of(warp);
      if (warp < tiles) fetch(row, 0);
      for (int tile = warp, n = 0; tile < tiles; tile += kFarWarps, ++n) {
        const Row ahead = row_of(tile + kFarWarps);
        if (tile + kFarWarps < tiles) {
          fetch(ahead, (n + 1) & 1);
          asm volatile("cp.async.wait_group 1;" ::: "memory");
        } else {
          asm volatile("cp.async.wait_group 0;" ::: "memory");
        }
        __syncwarp();
        const uint32_t qs = smem_u32(ring + (n & 1) * Shape::kTile), gs = qs + kFarTile * Shape::kPitch;
        float sc[2][4] = {}, dp[2][4] = {};
#pragma unroll
        for (int c = 0; c < KS; ++c) {
          if (c >= ksteps) break;
          uint32_t f[4];
          ldmatrix4(rows_frag(qs, Shape::kPitch) + 32 * c, f);
          mma16816<HALF>(sc[0], k[c], f[0], f[1]);
          mma16816<HALF>(sc[1], k[c], f[2], f[3]);
          ldmatrix4(rows_frag(gs, Shape::kPitch) + 32 * c, f);
          mma16816<HALF>(dp[0], v[c], f[0], f[1]);
          mma16816<HALF>(dp[1], v[c], f[2], f[3]);
        }
        uint32_t pw[4], dw[4];
#pragma unroll
        for (int half = 0; half < 2; ++half) {                   // rows 0-7, 8-15
          float p[2][2], ds[2][2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int r = 8 * half + 2 * (lane & 3) + e;
            const int i = __shfl_sync(0xffffffffu, row.i, r);
            const float lse = __shfl_sync(0xffffffffu, row.lse, r), delta = __shfl_sync(0xffffffffu, row.delta, r);
#pragma unroll
            for (int h = 0; h < 2; ++h) {                        // first nodes lane / 4, lane / 4 + 8
              const bool seen = kept[h] && i >= 0 && i - (first + (lane >> 2) + 8 * h) >= a.window;
              const float x = seen ? exp2_approx(sc[half][2 * h + e] * a.scale_log2 + (prob_log - lse)) : 0.f;
              p[h][e] = x;
              ds[h][e] = seen ? x * ((dp[half][2 * h + e] - delta) * after) : 0.f;
            }
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            pw[2 * half + h] = pack2(p[h][0], p[h][1], HALF);
            dw[2 * half + h] = pack2(ds[h][0], ds[h][1], HALF);
          }
        }
#pragma unroll
        for (int c = 0; c < KS; ++c) {
          if (c >= ksteps) break;
          uint32_t f[4];
          ldmatrix4t(columns_frag(gs, Shape::kPitch) + 32 * c, f);
          mma16816<HALF>(dv[2 * c], pw, f[0], f[1]);
          mma16816<HALF>(dv[2 * c + 1], pw, f[2], f[3]);
          ldmatrix4t(columns_frag(qs, Shape::kPitch) + 32 * c, f);
          mma16816<HALF>(dk[2 * c], dw, f[0], f[1]);
          mma16816<HALF>(dk[2 * c + 1], dw, f[2], f[3]);
        }
        __syncwarp();                                            // (the tile is read: the next copies may go there)
        row = ahead;
      }
      // the warps' sums, dK and then dV, in order
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        __syncthreads();
        float* part = reinterpret_cast<float*>(smem);            // [warp][first node][DP]
#pragma unroll
        for (int c = 0; c < 2 * KS; ++c)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            *reinterpret_cast<float2*>(part + (warp * 16 + (lane >> 2) + 8 * h) * DP + 8 * c + 2 * (lane & 3)) =
                which == 0 ? make_float2(dk[c][2 * h], dk[c][2 * h + 1]) : make_float2(dv[c][2 * h], dv[c][2 * h + 1]);
        __syncthreads();
        for (int e = tid; e < many * a.dim; e += kThreads) {
          const int t = e / a.dim, d = e - t * a.dim;
          float x = 0.f;
#pragma unroll
          for (int w = 0; w < kFarWarps; ++w) x += part[(w * 16 + t) * DP + d];
          far_slot(a, g, slot, hk, t0 + t)[which * a.dim + d] = x * (which == 0 ? 1.f / kept_at : 1.f / prob_up);
        }
      }
      __syncthreads();
    }
    i0 = s.end;
  }
}

template <bool HALF, int DP>
int far_mma_launch(const AttnArgs& a, const AttnGrad& g, cudaStream_t st) {
  auto kernel = attn_far_mma_kernel<HALF, DP>;
  static PerDeviceOnce once;
  const int status = once.run([&]() -> int {
    OCNN_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, FarShape<DP>::kBytes));
    return OCNN_OK;
  });
  if (status != OCNN_OK) return status;
  kernel<<<dim3(ceil_div(a.n, kFarRows), a.kv_heads), 32 * kFarWarps, FarShape<DP>::kBytes, st>>>(a, g);
  OCNN_LAUNCH_OK("attn_far_mma_kernel");
  return OCNN_OK;
}
template <bool HALF>
int far_mma_by_width(const AttnArgs& a, const AttnGrad& g, cudaStream_t st) {
  if (a.dim <= 32) return far_mma_launch<HALF, 32>(a, g, st);
  if (a.dim <= 64) return far_mma_launch<HALF, 64>(a, g, st);
  return far_mma_launch<HALF, 128>(a, g, st);
}

// Adds a first node's slots up into the first of them: a block per sequence, key head and first node; its threads are runs
// of slots x channels.
constexpr int kJoinThreads = 512;
__global__ void __launch_bounds__(kJoinThreads) attn_far_join_kernel(const AttnArgs a, const AttnGrad g) {
  __shared__ float part[kJoinThreads];
  const int b = blockIdx.x, hk = blockIdx.y, t = blockIdx.z, width = 2 * a.dim, runs = kJoinThreads / width;
  const Span s = {attn_offset(a, b), attn_offset(a, b + 1), b};
  const int j = s.start + t;
  if (j >= s.end) return;
  const FarSlots f = far_slots_of(a, j, s);
  if (f.count < 2) return;
  const int run = threadIdx.x / width, e = threadIdx.x - run * width;
  float x = 0.f;
  if (run < runs) {
#pragma unroll 8
    for (int k = run; k < f.count; k += runs) x += far_slot(a, g, f.first + k, hk, t)[e];
  }
  part[threadIdx.x] = x;
  __syncthreads();
  if (run == 0) {
    for (int k = 1; k < runs; ++k) x += part[k * width + e];
    far_slot(a, g, f.first, hk, t)[e] = x;
  }
}

}  // namespace

int attn_far_join(const AttnArgs& a, const AttnGrad& g, cudaStream_t st) {
  if (a.batch == 0) return OCNN_OK;
  attn_far_join_kernel<<<dim3(a.batch, a.kv_heads, a.sinks), kJoinThreads, 0, st>>>(a, g);
  OCNN_LAUNCH_OK("attn_far_join_kernel");
  return OCNN_OK;
}

int attn_far_mma(const AttnArgs& a, const AttnGrad& g, int dtype, cudaStream_t st) {
  return dtype == OCNN_F16 ? far_mma_by_width<true>(a, g, st) : far_mma_by_width<false>(a, g, st);
}

}  // namespace ocnn
