// Gradients of the attention over a window of nodes on the tensor cores, 16-bit data.
//
//     p = exp2(scale s - lse),  ds = p (dO . v - delta),  delta_i = dO_i . o_i
//     dq_i = scale sum_j ds_ij k_j,   dk_j = scale sum_i ds_ij q_i,   dv_j = sum_i p_ij dO_i
//
// Two kernels, one over tiles of queries and one over tiles of keys, each forming s, dO . v and p for itself: seven
// products instead of five, but every sum stays in tensor memory, in one order, and is written once; one kernel would
// have to add dq into fp32 in global memory, with atomics whose order changes the result.
//   queries: S = Q K^T, dP = dO V^T -> dS (tensor memory, in S's place) -> dQ += dS K
//   keys:    S' = K Q^T, dP' = V dO^T -> P', dS' (in place) -> dV += P' dO, dK += dS' Q
// P and dS are rounded to the data's type, which is what the products take.  Roles and tiles as in attention_tc.cu.
#include "attention_tc.cuh"

namespace ocnn {
namespace {

enum : int { kErrGradLoad = 21, kErrGradSlot = 22, kErrGradS = 23, kErrGradP = 24, kErrGradDone = 25, kErrGradTile = 26 };

constexpr int kBN = 64;                        // columns of a block: keys, or rows of queries
constexpr int kMaxStages = 6;

struct GradArgs {
  CUtensorMap q, grad, k, v;                   // dq: Q, dO by tile, K, V by block; dkv: Q, dO by block
  AttnArgs a;
  AttnGrad g;
  int* status;
  int pack_log, stages, wide;
};

constexpr int tmem_columns(int need) { return need <= 64 ? 64 : need <= 128 ? 128 : need <= 256 ? 256 : 512; }

template <int DP, int W>
struct DqShape {
  static constexpr int kThreads = 160 * W + 32;
  static constexpr int kPieces = DP / 64 > 0 ? DP / 64 : 1;
  static constexpr int kTile = 128 * kRowBytes * kPieces;                // Q, then dO
  static constexpr int kBlock = kBN * kRowBytes * kPieces;               // K, then V
  static constexpr int kAcc = 2 * kBN + DP;                              // S, dP, dQ
  static constexpr int kCols = tmem_columns(W * kAcc);
  static constexpr size_t smem(int stages) { return (size_t)W * 2 * kTile + (size_t)stages * 2 * kBlock + 1024 + 384; }
};

template <int DP, int W, bool HALF, bool MASKED, int CTAS>
__global__ void __launch_bounds__(DqShape<DP, W>::kThreads, CTAS) attn_tc_dq_kernel(const __grid_constant__ GradArgs p) {
  using Shape = DqShape<DP, W>;
  using T = typename std::conditional<HALF, __half, __nv_bfloat16>::type;
  const AttnArgs& a = p.a;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* stq = smem;
  uint8_t* skv = stq + W * 2 * Shape::kTile;
  uint64_t* full = reinterpret_cast<uint64_t*>(skv + p.stages * 2 * Shape::kBlock);
  uint64_t* empty = full + kMaxStages;
  uint64_t* clean = empty + kMaxStages;                                    // (the stage's rows are cleared)
  uint64_t* qfull = clean + kMaxStages;
  uint64_t* sfull = qfull + 1;
  uint64_t* dsfull = sfull + W;
  uint64_t* dqdone = dsfull + W;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(dqdone + W);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  BlockRange* ranges = reinterpret_cast<BlockRange*>(tmem_holder + 2);

  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const int nodes = 128 >> p.pack_log, pack = 1 << p.pack_log, r0 = blockIdx.x * (W * nodes);
  const int group = a.heads / a.kv_heads, per_kv = group >> p.pack_log;
  const int hk = blockIdx.y / per_kv, h0 = hk * group + (blockIdx.y % per_kv) * pack;
  if (tid == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), W);
      mbar_init(smem_u32(&clean[s]), 1);
    }
    mbar_init(smem_u32(qfull), 1);
    for (int t = 0; t < W; ++t) {
      mbar_init(smem_u32(&sfull[t]), 1);
      mbar_init(smem_u32(&dsfull[t]), 128);
      mbar_init(smem_u32(&dqdone[t]), 1);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 4 * W) tmem_alloc(tmem_holder, Shape::kCols);
  grid_dependency_wait();
  const WarpOffsets offsets(a);
  Span f, l;
  const TileKeys tile_keys = attn_tile_keys(a, offsets, r0, r0 + W * nodes, f, l);
  const KeyBlocks<kBN> keys(tile_keys);
  const int blocks = keys.count;
  if (W > 1 && warp < W) {
    Span x, y;
    const BlockRange r = block_range<kBN>(keys, attn_tile_keys(a, offsets, r0 + warp * nodes, r0 + (warp + 1) * nodes, x, y));
    if (lane == 0) ranges[warp] = r;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  auto active = [&](int t, int b) { return W == 1 || in_range(ranges[t], b); };
  const int ksteps = (a.dim + 15) / 16, end = min(a.n, offsets.end(a));
  const bool cleared = MASKED || (end < a.n && keys.reaches(end));   // (see clear_rows)

  if (warp < 4 * W) {
    // ---------------- rows ----------------
    const int t = warp >> 2, row = tid & 127;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16) + t * Shape::kAcc, acc = lanes + 2 * kBN;
    const int i = r0 + t * nodes + (row >> p.pack_log), h = h0 + (row & (pack - 1));
    const bool in = i < a.n;
    const RowKeys r = in ? attn_row_keys(a, i, attn_span_near(a, i, f, l)) : RowKeys{0, 0, 0, 0};
    const float lse = in ? p.g.lse[(long long)h * a.n + i] : INFINITY;
    float delta = 0.f, largest = 0.f;
    if (in) {
      const T* go = (const T*)p.g.grad + i * p.g.grad_row + h * p.g.grad_head;
      const T* o = (const T*)p.g.out + ((long long)i * a.heads + h) * a.dim;
      const T* rest = attn_rest<T>(a, p.g.lse) + ((long long)i * a.heads + h) * a.dim;
      for (int d = 0; d < a.dim; d += 8) {
        const uint4 x = *reinterpret_cast<const uint4*>(go + d), y = *reinterpret_cast<const uint4*>(o + d);
        const uint4 z = *reinterpret_cast<const uint4*>(rest + d);
        const uint32_t *xs = &x.x, *ys = &y.x, *zs = &z.x;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 u = unpack2(xs[e], HALF), v = unpack2(ys[e], HALF), w = unpack2(zs[e], HALF);
          delta = fmaf(u.x, v.x + w.x, delta);
          delta = fmaf(u.y, v.y + w.y, delta);
          if (HALF) {
            if (!not_finite(u.x)) largest = fmaxf(largest, fabsf(u.x));
            if (!not_finite(u.y)) largest = fmaxf(largest, fabsf(u.y));
          }
        }
      }
      p.g.delta[(long long)h * a.n + i] = delta;
    }
    if (HALF) {
      const unsigned most = __reduce_max_sync(0xffffffffu, __float_as_uint(largest));
      // (a warp's nodes are in one chunk; a maximum is the same in any order)
      const int chunk = (r0 + t * nodes + (((warp & 3) * 32) >> p.pack_log)) >> kChunkLog;
      if (lane == 0 && most != 0) atomicMax(p.g.largest + chunk, most);
    }
    const float kept_at = HALF ? grad_scale(largest) : 1.f;                 // dS of this row is kept at dS * kept_at
    const FullBlocks whole(keys, r, MASKED, std::integral_constant<int, kBN>());
    const uint64_t c2 = pair(a.scale_log2, a.scale_log2), lse2 = pair(-lse, -lse), delta2 = pair(-delta * kept_at, -delta * kept_at),
                   kept2 = pair(kept_at, kept_at);
    int done = 0;
    bool alive = true;
    KeptKeys<kBN> kept, ahead;
    if (MASKED && blocks > 0) ahead.ask(a, keys.key(0), a.n);
    for (int b = 0; b < blocks && alive; ++b) {
      if (MASKED) {
        kept = ahead;
        if (b + 1 < blocks) ahead.ask(a, keys.key(b + 1), a.n);
      }
      if (!active(t, b)) continue;
      alive = mbar_wait(smem_u32(&sfull[t]), done & 1, abort_flag, p.status, kErrGradS);
      alive = __all_sync(0xffffffffu, alive);
      if (!alive) break;
      tc_fence_after();
      float s[kBN], dp[kBN];
      tmem_load<kBN>(lanes, s);
      tmem_load<kBN>(lanes + kBN, dp);
      const int j = keys.key(b);
      const bool first = keys.is_first(b), all = whole.has(b);
      uint32_t bits[2];
      if (!all) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          bits[k] = first ? seen_first(keys, r, 32 * k) : seen_bits(a, r, j + 32 * k);
          if (MASKED) bits[k] &= kept.bits(k);
        }
      }
      tmem_wait_ld();
#pragma unroll
      for (int e = 0; e < kBN; e += 2) {
        const float2 x = unpair(fma2(pair(s[e], s[e + 1]), c2, lse2));
        const float2 ds = unpair(mul2(pair(exp2_approx(x.x), exp2_approx(x.y)), fma2(pair(dp[e], dp[e + 1]), kept2, delta2)));
        s[e] = ds.x;
        s[e + 1] = ds.y;
      }
      if (!all) {
#pragma unroll
        for (int e = 0; e < kBN; ++e)
          if (!((bits[e / 32] >> (e & 31)) & 1)) s[e] = 0.f;
      }
      uint32_t w[kBN / 2];
#pragma unroll
      for (int e = 0; e < kBN / 2; ++e) w[e] = pack16<HALF>(s[2 * e], s[2 * e + 1]);
      tmem_store<kBN / 2>(lanes, w);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(smem_u32(&dsfull[t]));
      ++done;
    }
    if (done > 0 && alive) {
      alive = mbar_wait(smem_u32(&dqdone[t]), (done - 1) & 1, abort_flag, p.status, kErrGradDone);
      alive = __all_sync(0xffffffffu, alive);
      tc_fence_after();
    }
    if (alive) {
      bool bad = false;
      const float up = a.scale / kept_at;
      T* dst = (T*)p.g.dq + ((long long)i * a.heads + h) * a.dim;
#pragma unroll 2
      for (int d = 0; d < a.dim; d += 16) {
        float x[16] = {};
        if (done > 0) {
          tmem_ld16(acc + d, reinterpret_cast<uint32_t(&)[16]>(x));
          tmem_wait_ld();
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          x[e] *= up;
          bad |= not_finite(x[e]);
        }
        if (in) store_row<HALF>(dst, d, a.dim, p.wide, x);
      }
      unsigned redo = __ballot_sync(0xffffffffu, bad && in && !attn_query_is_spoilt(lse, delta));
      while (redo != 0) {
        const int at = __ffs(redo) - 1;
        redo &= redo - 1;
        attn_dq_row<T>(a, p.g, __shfl_sync(0xffffffffu, i, at), __shfl_sync(0xffffffffu, h, at));
      }
    }
  } else if (warp < 5 * W) {
    // ---------------- products: a warp per tile, one thread of it issues ----------------
    if (blocks > 0) {
      const int t = warp - 4 * W;
      const bool leader = elect_one();
      const uint32_t idesc_s = attn_idesc<HALF>(kBN, false), idesc_o = attn_idesc<HALF>(16 * ksteps, true);
      const uint32_t q = smem_u32(stq + t * 2 * Shape::kTile), kv = smem_u32(skv), d = tmem + t * Shape::kAcc;
      BlockRange range;
      if (W > 1) range = ranges[t];
      auto needs = [&](int b) { return W == 1 || in_range(range, b); };
      int n = 0, stage = 0;
      uint32_t phase = 0;
      bool alive = mbar_wait(smem_u32(qfull), 0, abort_flag, p.status, kErrGradTile);
      uint64_t* ready = cleared ? clean : full;
      auto scores = [&](int s) {
        tc_fence_after();
        if (leader) {
          const uint32_t k = kv + s * 2 * Shape::kBlock;
          product_channels<DP / 16, 128, kBN>(d, q, k, ksteps, idesc_s);
          product_channels<DP / 16, 128, kBN>(d + kBN, q + Shape::kTile, k + Shape::kBlock, ksteps, idesc_s);
          umma_commit(smem_u32(&sfull[t]));
        }
      };
      // S and dP need their place: the product that reads dS through.
      auto next_scores = [&](int s) {
        if (n > 0) alive = mbar_wait(smem_u32(&dqdone[t]), (n - 1) & 1, abort_flag, p.status, kErrGradDone);
        if (alive) scores(s);
      };
      if (alive) alive = mbar_wait(smem_u32(&ready[0]), 0, abort_flag, p.status, kErrGradLoad);
      if (alive && needs(0)) scores(0);
      for (int b = 0; b < blocks && alive; ++b) {
        const int next = stage + 1 == p.stages ? 0 : stage + 1;
        const uint32_t next_phase = next == 0 ? phase ^ 1u : phase;
        const bool more = b + 1 < blocks;
        // (all asked before the first is waited for)
        const uint32_t loaded = mbar_ask(smem_u32(&ready[next]), next_phase);
        const uint32_t formed = mbar_ask(smem_u32(&dsfull[t]), n & 1);
        if (more && !loaded) alive = mbar_wait(smem_u32(&ready[next]), next_phase, abort_flag, p.status, kErrGradLoad);
        if (alive && needs(b)) {
          if (!formed) alive = mbar_wait(smem_u32(&dsfull[t]), n & 1, abort_flag, p.status, kErrGradP);
          if (!alive) break;
          tc_fence_after();
          if (leader) {
            product_rows<kBN>(d + 2 * kBN, d, kv + stage * 2 * Shape::kBlock, idesc_o, n == 0);
            umma_commit(smem_u32(&dqdone[t]));
          }
          ++n;
        }
        if (alive && leader && b + p.stages < blocks) umma_commit(smem_u32(&empty[stage]));
        if (alive && more && needs(b + 1)) next_scores(next);
        stage = next;
        phase = next_phase;
      }
      if (!alive)
        for (int it = 0; it < 64; ++it) __nanosleep(1000);       // (products under way end before tensor memory is freed)
    }
  } else if (blocks > 0) {
    // ---------------- copies ----------------
    if (lane == 0) {
      mbar_arrive_expect_tx(smem_u32(qfull), 2 * W * tile_bytes<128>(a.dim));
      for (int t = 0; t < W; ++t) {
        const uint32_t dst = smem_u32(stq + t * 2 * Shape::kTile);
        tma_tile<Shape::kPieces, 128>(dst, &p.q, a.dim, h0, r0 + t * nodes, smem_u32(qfull));
        tma_tile<Shape::kPieces, 128>(dst + Shape::kTile, &p.grad, a.dim, h0, r0 + t * nodes, smem_u32(qfull));
      }
    }
    int stage = 0, cstage = 0;
    uint32_t phase = 1, cphase = 0, words[2];
    bool alive = true;
    for (int b = 0; b < blocks + (cleared ? 1 : 0) && alive; ++b) {
      if (b < blocks) {
        if (b >= p.stages) alive = mbar_wait(smem_u32(&empty[stage]), phase, abort_flag, p.status, kErrGradSlot);
        if (!alive) break;
        if (lane == 0) {
          const uint32_t dst = smem_u32(skv + stage * 2 * Shape::kBlock), bar = smem_u32(&full[stage]);
          mbar_arrive_expect_tx(bar, 2 * tile_bytes<kBN>(a.dim));
          tma_tile<Shape::kPieces, kBN>(dst, &p.k, a.dim, hk, keys.key(b), bar);
          tma_tile<Shape::kPieces, kBN>(dst + Shape::kBlock, &p.v, a.dim, hk, keys.key(b), bar);
        }
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      KeptKeys<kBN> kept;
      if (cleared && b < blocks) kept.ask(a, keys.key(b), end);
      // the stage before has landed or is about to: its K (V is read for dP only, and a hidden key's dP is not)
      if (cleared && b > 0) {
        alive = mbar_wait(smem_u32(&full[cstage]), cphase, abort_flag, p.status, kErrGradLoad);
        alive = __all_sync(0xffffffffu, alive);
        if (!alive) break;
        clear_rows<Shape::kPieces, kBN>(skv + cstage * 2 * Shape::kBlock, [&](int k) { return words[k]; });
        proxy_fence();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&clean[cstage]));
        if (++cstage == p.stages) {
          cstage = 0;
          cphase ^= 1u;
        }
      }
      if (cleared) {
#pragma unroll
        for (int k = 0; k < 2; ++k) words[k] = kept.bits(k);
      }
    }
    if (!alive)
      for (int it = 0; it < 64; ++it) __nanosleep(1000);         // (copies under way end before the CTA does)
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 4 * W)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)Shape::kCols) : "memory");
}

// The nodes that see the keys [k0, k1) from within the window, whatever the mask says, by a whole warp; f and l: the
// sequences of the first and the last key that is in one.
__device__ __forceinline__ KeyRows attn_tile_rows(const AttnArgs& a, const WarpOffsets& offsets, int k0, int k1, Span& f, Span& l) {
  const int x = max(k0, offsets.begin()), y = min(min(k1, a.n), offsets.end(a)) - 1;
  f = l = Span{0, 0, 0};
  if (x > y) return KeyRows{0, 0};
  f = offsets.span(a, x);
  l = y < f.end ? f : offsets.span(a, y);
  return KeyRows{attn_rows_of_key(a, x, f).lo, attn_rows_of_key(a, y, l).hi};
}

template <int DP, int G>
struct DkvShape {
  static constexpr int kThreads = 128 * G + 64;
  static constexpr int kPieces = DP / 64 > 0 ? DP / 64 : 1;
  static constexpr int kTile = 128 * kRowBytes * kPieces;                // K, then V
  static constexpr int kBlock = kBN * kRowBytes * kPieces;               // Q, then dO
  static constexpr int kCols = tmem_columns(G * 2 * kBN + 2 * DP);         // S' and dP' of G blocks, dK, dV
  static constexpr size_t smem(int stages) {
    return (size_t)2 * kTile + (size_t)stages * 2 * kBlock + G * 4 * kBN * sizeof(float) + 1024 + 384;
  }
};

// One tile of 128 keys.  A block is kBN rows of queries: kBN / pack nodes, pack heads each; G groups of four warps take
// the blocks in turn, each with S' and dP' of its own.
template <int DP, int G, bool HALF, int CTAS>
__global__ void __launch_bounds__(DkvShape<DP, G>::kThreads, CTAS) attn_tc_dkv_kernel(const __grid_constant__ GradArgs p) {
  using Shape = DkvShape<DP, G>;
  using T = typename std::conditional<HALF, __half, __nv_bfloat16>::type;
  const AttnArgs& a = p.a;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* skv = smem;
  uint8_t* sqg = skv + 2 * Shape::kTile;
  float* stats = reinterpret_cast<float*>(sqg + p.stages * 2 * Shape::kBlock);       // [G][2][-lse, -delta][kBN]
  uint64_t* full = reinterpret_cast<uint64_t*>(stats + G * 4 * kBN);
  uint64_t* empty = full + kMaxStages;
  uint64_t* clean = empty + kMaxStages;                                    // (the stage's rows are cleared)
  uint64_t* kvfull = clean + kMaxStages;
  uint64_t* sfull = kvfull + 1;
  uint64_t* pfull = sfull + G;
  uint64_t* done = pfull + G;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(done + G);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const int k0 = blockIdx.x * 128, hk = blockIdx.y, group = a.heads / a.kv_heads;
  if (tid == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
      mbar_init(smem_u32(&clean[s]), 1);
    }
    mbar_init(smem_u32(kvfull), 128 * G);
    for (int t = 0; t < G; ++t) {
      mbar_init(smem_u32(&sfull[t]), 1);
      mbar_init(smem_u32(&pfull[t]), 128);
      mbar_init(smem_u32(&done[t]), 1);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 4 * G) tmem_alloc(tmem_holder, Shape::kCols);
  grid_dependency_wait();
  const WarpOffsets offsets(a);
  Span f, l;
  const KeyRows span = attn_tile_rows(a, offsets, k0, k0 + 128, f, l);
  const int pack = 1 << p.pack_log, nodes = kBN >> p.pack_log;             // nodes of a block
  const int per_head = (max(0, span.hi - span.lo) + nodes - 1) >> (6 - p.pack_log);   // blocks of `pack` heads
  const int blocks = per_head * (group >> p.pack_log);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  constexpr int kAcc = G * 2 * kBN;                                        // dK, then dV
  const int ksteps = (a.dim + 15) / 16, end = min(a.n, offsets.end(a));
  const bool cleared = end < a.n && span.hi == end;                        // (its last block holds nobody's nodes)
  // (blocks go head by head: no division where there is only one run of them)
  auto run_of = [&](int b) { return b < per_head ? 0 : b / per_head; };
  auto first_node = [&](int b) { return span.lo + (b - run_of(b) * per_head) * nodes; };
  auto first_head = [&](int b) { return hk * group + run_of(b) * pack; };

  if (warp < 4 * G) {
    // ---------------- rows: keys ----------------
    const int t = warp >> 2, row = tid & 127, j = k0 + row;
    const uint32_t quarter = tmem + ((uint32_t)((warp & 3) * 32) << 16), lanes = quarter + t * 2 * kBN;
    if (blocks > 0) {
      auto kept = [&](int r) { return k0 + r < a.n && (a.mask == nullptr || a.mask[k0 + r] != 0); };
      const T *k = (const T*)a.k + hk * a.k_head, *v = (const T*)a.v + hk * a.v_head;
      copy_tile<DP, 128, 128 * G>(smem_u32(skv), tid, a.dim, a.k,
                                  [&](int r) { return (const uint8_t*)(k + (k0 + r) * a.k_row); }, kept);
      copy_tile<DP, 128, 128 * G>(smem_u32(skv + Shape::kTile), tid, a.dim, a.k,
                                  [&](int r) { return (const uint8_t*)(v + (k0 + r) * a.v_row); }, kept);
      cp_async_arrive(smem_u32(kvfull));
    }
    const KeyRows kr = j < a.n ? attn_key_rows(a, j, attn_span_near(a, j, f, l)) : KeyRows{0, 0};
    const uint64_t c2 = pair(a.scale_log2, a.scale_log2);
    // P' is kept at P' * prob_up, dS' at dS' * kept_at
    constexpr float prob_up = HALF ? kProbUp : 1.f, prob_log = HALF ? kProbUpLog : 0.f;
    const float kept_at = HALF && blocks > 0 ? grad_scale_of(p.g.largest, span.lo, span.hi) : 1.f, after = kept_at / prob_up;
    const uint64_t after2 = pair(after, after);
    // lse and delta of a block's rows: two threads a row fetch them a block ahead
    auto fetch = [&](int b) {
      const int r = row & (kBN - 1), i = first_node(b) + (r >> p.pack_log);
      if (b >= blocks || i >= span.hi) return row < kBN ? -INFINITY : 0.f;
      const long long at = (long long)(first_head(b) + (r & (pack - 1))) * a.n + i;
      return row < kBN ? prob_log - p.g.lse[at] : -p.g.delta[at] * after;
    };
    float ahead = t < blocks ? fetch(t) : 0.f;
    int n = 0;
    bool alive = true;
    // (a group's warps meet at the barrier in every block, one that has given up too)
    for (int b = t; b < blocks; b += G, ++n) {
      float* st = stats + (t * 2 + (n & 1)) * (2 * kBN);
      st[row] = ahead;
      asm volatile("bar.sync %0, 128;" ::"r"(1 + t) : "memory");
      ahead = fetch(b + G);
      const int i0 = first_node(b);
      const int lo = (max(kr.lo, i0) - i0) << p.pack_log, hi = (max(min(kr.hi, i0 + nodes), i0) - i0) << p.pack_log;
      if (alive) alive = mbar_wait(smem_u32(&sfull[t]), n & 1, abort_flag, p.status, kErrGradS);
      alive = __all_sync(0xffffffffu, alive);
      if (alive) {
        tc_fence_after();
        const uint32_t bits[2] = {bit_run(lo, hi), bit_run(lo - 32, hi - 32)};
        const bool all = __all_sync(0xffffffffu, (bits[0] & bits[1]) == 0xffffffffu);
        auto form = [&](auto every) {
          constexpr bool ALL = decltype(every)::value;
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float s[32], dp[32];
            tmem_load<32>(lanes + 32 * k, s);
            tmem_load<32>(lanes + kBN + 32 * k, dp);
            tmem_wait_ld();
            uint32_t w[16], v[16];
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              const ulonglong2 lse = *reinterpret_cast<const ulonglong2*>(st + 32 * k + e);
              const ulonglong2 delta = *reinterpret_cast<const ulonglong2*>(st + kBN + 32 * k + e);
#pragma unroll
              for (int u = 0; u < 4; u += 2) {
                const float2 x = unpair(fma2(pair(s[e + u], s[e + u + 1]), c2, u == 0 ? lse.x : lse.y));
                float px = exp2_approx(x.x), py = exp2_approx(x.y);
                if (!ALL) {
                  if (!((bits[k] >> (e + u)) & 1)) px = 0.f;
                  if (!((bits[k] >> (e + u + 1)) & 1)) py = 0.f;
                }
                float2 ds = unpair(mul2(pair(px, py), fma2(pair(dp[e + u], dp[e + u + 1]), after2, u == 0 ? delta.x : delta.y)));
                if (!ALL) {
                  // (a hidden row's dP may be anything)
                  if (!((bits[k] >> (e + u)) & 1)) ds.x = 0.f;
                  if (!((bits[k] >> (e + u + 1)) & 1)) ds.y = 0.f;
                }
                w[(e + u) / 2] = pack16<HALF>(px, py);
                v[(e + u) / 2] = pack16<HALF>(ds.x, ds.y);
              }
            }
            // P' lies where the scores of the first 32 columns lay, dS' likewise: all read by now
            tmem_st16(lanes + 16 * k, w);
            tmem_st16(lanes + kBN + 16 * k, v);
          }
        };
        if (all) form(std::true_type());
        else form(std::false_type());
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(smem_u32(&pfull[t]));
      }
    }
    // The accumulators are through with the last block of every group of warps.  (Its own first: behind that, every other
    // group's barrier is in the phase of its last block, or past it.)
    for (int k = 0; k < G && alive; ++k) {
      const int u = (t + k) % G, count = blocks > u ? (blocks - u + G - 1) / G : 0;
      if (count > 0) alive = mbar_wait(smem_u32(&done[u]), (count - 1) & 1, abort_flag, p.status, kErrGradDone);
    }
    alive = __all_sync(0xffffffffu, alive);
    tc_fence_after();
    if (alive) {
      const bool in = j < a.n;
      const float* far = in ? far_sums(a, p.g, j, hk) : nullptr;
      // group 0 writes dK, the last one dV (both, where there is one)
#pragma unroll 1
      for (int which = t == 0 ? 0 : 1; which <= (t == G - 1 ? 1 : 0); ++which) {
        const float f = which == 0 ? a.scale : 1.f, back = which == 0 ? 1.f / kept_at : 1.f / prob_up;
        bool bad = false;
        T* dst = (T*)(which == 0 ? p.g.dk : p.g.dv) + ((long long)j * a.kv_heads + hk) * a.dim;
#pragma unroll 2
        for (int d = 0; d < a.dim; d += 16) {
          float x[16] = {};
          if (blocks > 0) {
            tmem_ld16(quarter + kAcc + which * DP + d, reinterpret_cast<uint32_t(&)[16]>(x));
            tmem_wait_ld();
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) x[e] *= back;
          if (far != nullptr) {
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (d + e < a.dim) x[e] += far[which * a.dim + d + e];
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            x[e] *= f;
            bad |= not_finite(x[e]);
          }
          if (in) store_row<HALF>(dst, d, a.dim, p.wide, x);
        }
        unsigned redo = __ballot_sync(0xffffffffu, bad && in);
        __syncwarp();
        while (redo != 0) {
          const int rj = __shfl_sync(0xffffffffu, j, __ffs(redo) - 1);
          redo &= redo - 1;
          if (!attn_key_is_spoilt<T>(a, p.g, rj, hk, which == 1)) attn_dkv_row<T>(a, p.g, rj, hk, which == 0, which == 1);
        }
      }
    }
  } else if (warp == 4 * G) {
    // ---------------- products: one thread of the warp issues ----------------
    if (blocks > 0) {
      const bool leader = elect_one();
      const uint32_t idesc_s = attn_idesc<HALF>(kBN, false), idesc_o = attn_idesc<HALF>(16 * ksteps, true);
      bool alive = mbar_wait(smem_u32(kvfull), 0, abort_flag, p.status, kErrGradTile);
      proxy_fence();                                  // (K and V came by cp.async)
      const uint32_t qg = smem_u32(sqg), k = smem_u32(skv);
      int ahead = 0, ahead_stage = 0;
      uint32_t ahead_phase = 0;
      auto scores = [&]() {                            // of the next block that has none yet
        const int t = ahead % G, n = ahead / G;
        const uint32_t bar = smem_u32(&(cleared ? clean : full)[ahead_stage]), held = smem_u32(&done[t]);
        const uint32_t loaded = mbar_ask(bar, ahead_phase), free = n > 0 ? mbar_ask(held, (n - 1) & 1) : 1u;
        if (alive && !loaded) alive = mbar_wait(bar, ahead_phase, abort_flag, p.status, kErrGradLoad);
        // (S' and dP' lie where P' and dS' do: the products that read those have to be through)
        if (alive && !free) alive = mbar_wait(held, (n - 1) & 1, abort_flag, p.status, kErrGradDone);
        if (!alive) return;
        tc_fence_after();
        if (leader) {
          const uint32_t q = qg + ahead_stage * 2 * Shape::kBlock, d = tmem + t * 2 * kBN;
          product_channels<DP / 16, 128, kBN>(d, k, q, ksteps, idesc_s);
          product_channels<DP / 16, 128, kBN>(d + kBN, k + Shape::kTile, q + Shape::kBlock, ksteps, idesc_s);
          umma_commit(smem_u32(&sfull[t]));
        }
        ++ahead;
        if (++ahead_stage == p.stages) {
          ahead_stage = 0;
          ahead_phase ^= 1u;
        }
      };
      while (alive && ahead < blocks && ahead < G) scores();
      int stage = 0;
      for (int b = 0; b < blocks && alive; ++b) {
        const int t = b % G;
        alive = mbar_wait(smem_u32(&pfull[t]), (b / G) & 1, abort_flag, p.status, kErrGradP);
        if (!alive) break;
        tc_fence_after();
        if (leader) {
          const uint32_t q = qg + stage * 2 * Shape::kBlock, d = tmem + t * 2 * kBN;
          product_rows<kBN>(tmem + kAcc + DP, d, q + Shape::kBlock, idesc_o, b == 0);    // dV += P' dO
          product_rows<kBN>(tmem + kAcc, d + kBN, q, idesc_o, b == 0);                   // dK += dS' Q
          umma_commit(smem_u32(&done[t]));
          if (b + p.stages < blocks) umma_commit(smem_u32(&empty[stage]));
        }
        if (++stage == p.stages) stage = 0;
        if (ahead < blocks) scores();
      }
      if (!alive)
        for (int it = 0; it < 64; ++it) __nanosleep(1000);       // (products under way end before tensor memory is freed)
    }
  } else {
    // ---------------- copies of Q and dO ----------------
    // (rows behind the nodes that see the tile are hidden from all of its keys)
    int stage = 0, cstage = 0;
    uint32_t phase = 1, cphase = 0;
    bool alive = true;
    for (int b = 0; b < blocks + (cleared ? 1 : 0); ++b) {
      if (b < blocks) {
        if (b >= p.stages) alive = mbar_wait(smem_u32(&empty[stage]), phase, abort_flag, p.status, kErrGradSlot);
        if (!alive) break;
        if (lane == 0) {
          const uint32_t dst = smem_u32(sqg + stage * 2 * Shape::kBlock), bar = smem_u32(&full[stage]);
          mbar_arrive_expect_tx(bar, 2 * tile_bytes<kBN>(a.dim));
          tma_tile<Shape::kPieces, kBN>(dst, &p.q, a.dim, first_head(b), first_node(b), bar);
          tma_tile<Shape::kPieces, kBN>(dst + Shape::kBlock, &p.grad, a.dim, first_head(b), first_node(b), bar);
        }
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (cleared && b > 0) {
        alive = mbar_wait(smem_u32(&full[cstage]), cphase, abort_flag, p.status, kErrGradLoad);
        alive = __all_sync(0xffffffffu, alive);
        if (!alive) break;
        const int live = (end - first_node(b - 1)) << p.pack_log;           // rows before the batch's end
        if (live < kBN) {
          for (int qg = 0; qg < 2; ++qg)
            clear_rows<Shape::kPieces, kBN>(sqg + (cstage * 2 + qg) * Shape::kBlock,
                                            [&](int k) { return bit_run(0, live - 32 * k); });
          proxy_fence();
          __syncwarp();
        }
        if (lane == 0) mbar_arrive(smem_u32(&clean[cstage]));
        if (++cstage == p.stages) {
          cstage = 0;
          cphase ^= 1u;
        }
      }
    }
    if (!alive)
      for (int it = 0; it < 64; ++it) __nanosleep(1000);         // (copies under way end before the CTA does)
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 4 * G)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)Shape::kCols) : "memory");
}

template <typename Shape, int CTAS>
int stages_for() {
  constexpr size_t kMost = (227 * 1024) / CTAS - 1024;
  static_assert(Shape::smem(3) <= kMost, "with a mask, three stages at least: one is cleared while two are read");
  int stages = kMaxStages;
  while (Shape::smem(stages) > kMost) --stages;
  return stages;
}

template <int DP, int W, int G, bool HALF, int CTAS_Q, int CTAS_K>
int grad_launch(GradArgs& p, cudaStream_t st) {
  using Dq = DqShape<DP, W>;
  using Dkv = DkvShape<DP, G>;
  auto dq = attn_tc_dq_kernel<DP, W, HALF, false, CTAS_Q>, dq_masked = attn_tc_dq_kernel<DP, W, HALF, true, CTAS_Q>;
  auto dkv = attn_tc_dkv_kernel<DP, G, HALF, CTAS_K>;
  const int stages_q = stages_for<Dq, CTAS_Q>(), stages_k = stages_for<Dkv, CTAS_K>();
  static PerDeviceOnce once;
  int status = once.run([&]() -> int {
    OCNN_CUDA_OK(cudaFuncSetAttribute(dq, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Dq::smem(stages_q)));
    OCNN_CUDA_OK(cudaFuncSetAttribute(dq_masked, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Dq::smem(stages_q)));
    OCNN_CUDA_OK(cudaFuncSetAttribute(dkv, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Dkv::smem(stages_k)));
    return OCNN_OK;
  });
  if (status != OCNN_OK) return status;
  const AttnArgs& a = p.a;
  constexpr int dtype = HALF ? OCNN_F16 : OCNN_BF16;
  const int pack = 1 << p.pack_log;
  auto queries = [&](int rows) -> int {
    const int s = attn_map(&p.q, a.q, dtype, a.dim, a.heads, a.n, a.q_row, a.q_head, pack, rows >> p.pack_log);
    return s != OCNN_OK ? s : attn_map(&p.grad, p.g.grad, dtype, a.dim, a.heads, a.n, p.g.grad_row, p.g.grad_head, pack,
                                       rows >> p.pack_log);
  };
  status = queries(128);
  if (status == OCNN_OK) status = attn_map(&p.k, a.k, dtype, a.dim, a.kv_heads, a.n, a.k_row, a.k_head, 1, kBN);
  if (status == OCNN_OK) status = attn_map(&p.v, a.v, dtype, a.dim, a.kv_heads, a.n, a.v_row, a.v_head, 1, kBN);
  if (status != OCNN_OK) return status;
  p.stages = stages_q;
  p.wide = wide_rows(p.g.dq, a.dim);
  if (a.mask != nullptr) dq = dq_masked;
  if (HALF) OCNN_CUDA_OK(cudaMemsetAsync(p.g.largest, 0, grad_chunks(a.n) * sizeof(unsigned), st));
  OCNN_CUDA_OK(launch_chained(dq, dim3(ceil_div(a.n, W * 128 >> p.pack_log), a.heads >> p.pack_log), dim3(Dq::kThreads),
                              Dq::smem(stages_q), st, p));
  OCNN_LAUNCH_OK("attn_tc_dq_kernel");
  if (p.g.dk == nullptr) return OCNN_OK;
  if (p.a.sinks > 0) {
    const int far = attn_far_mma(p.a, p.g, HALF ? OCNN_F16 : OCNN_BF16, st);
    if (far != OCNN_OK) return far;
    const int joined = attn_far_join(p.a, p.g, st);
    if (joined != OCNN_OK) return joined;
  }
  status = queries(kBN);
  if (status != OCNN_OK) return status;
  p.stages = stages_k;
  p.wide = wide_rows(p.g.dk, a.dim) && wide_rows(p.g.dv, a.dim);
  OCNN_CUDA_OK(launch_chained(dkv, dim3(ceil_div(p.a.n, 128), p.a.kv_heads), dim3(Dkv::kThreads), Dkv::smem(stages_k), st, p));
  OCNN_LAUNCH_OK("attn_tc_dkv_kernel");
  return OCNN_OK;
}

template <bool HALF>
int grad_by_width(GradArgs& p, cudaStream_t st) {
  if (p.a.dim <= 32) return grad_launch<32, 1, 1, HALF, 2, 2>(p, st);
  if (p.a.dim <= 64) return grad_launch<64, 1, 1, HALF, 2, 2>(p, st);
  return grad_launch<128, 2, 2, HALF, 1, 1>(p, st);
}

}  // namespace

int attn_tc_backward(const AttnArgs& a, const AttnGrad& g, int dtype, int* status, cudaStream_t st) {
  GradArgs p;
  p.a = a;
  p.g = g;
  p.status = status;
  p.pack_log = attn_pack_log(a);
  return dtype == OCNN_F16 ? grad_by_width<true>(p, st) : grad_by_width<false>(p, st);
}

}  // namespace ocnn
