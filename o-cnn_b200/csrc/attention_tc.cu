// Attention over a window of nodes on the tensor cores, 16-bit data: forward pass.
//
// A CTA takes W tiles of 128 rows against the keys that they see, in blocks of BN keys.  A row is a query head of a node:
// P heads that share a key head stand side by side (P the largest power of two in the group), so that 128 / P nodes share
// each copy of keys and values and the tile's windows overlap more.  Per block and tile
//     S = Q K^T (tensor memory) -> p = exp2(S scale - m) -> P (tensor memory, in S's place) -> O += P V
// with 128 threads per tile, one row each, between the two products.  m is the row's reference: its running maximum, but
// moved only when a block exceeds it by more than 8 (any reference gives the same quotient as long as nothing overflows,
// and 2^8 is far from that), so O is hardly ever scaled.  P is rounded to the data's type, which is what the product takes;
// its sum is of the unrounded values.  float16 holds nothing below 2^-24: there p is kept at 2^7 p, 2^15 at most (10^5 keys at
// 2^-25 of the strongest would add nothing otherwise, 0.3 % of their values).  Scores have two places, so that a block's are
// ready when its rows come to it.
//
// Roles: 4 W warps of rows, W warps that issue products (one thread of each), one warp that brings Q and the blocks of K
// and V by TMA into a ring of slots (and clears the rows that the mask hides: see clear_rows).
#include "attention_tc.cuh"

namespace ocnn {
namespace {

struct AttnFwdArgs {
  CUtensorMap q, k, v;
  AttnArgs a;
  void* out;
  float* lse;
  int* status;
  int pack_log, stages, wide;
};

enum : int { kErrAttnQ = 11, kErrAttnLoad = 12, kErrAttnSlot = 13, kErrAttnP = 14, kErrAttnS = 15, kErrAttnO = 16 };

constexpr int kMaxStages = 6;

// NB: places for a tile's scores (1: none ahead of its rows; more CTAs per SM cover the wait).
template <int DP, int W, int BN, int NB>
struct FwdShape {
  static constexpr int kThreads = 160 * W + 32;                          // rows, products, copies
  static constexpr int kPieces = DP / 64 > 0 ? DP / 64 : 1;
  static constexpr int kTileQ = 128 * kRowBytes * kPieces;
  static constexpr int kBlock = BN * kRowBytes * kPieces;                // K, then V
  static constexpr int kAcc = NB * BN + DP;                              // places for S, and O
  static constexpr int kCols = W * kAcc <= 128 ? 128 : W * kAcc <= 256 ? 256 : 512;
  static constexpr size_t smem(int stages) { return (size_t)W * kTileQ + (size_t)stages * 2 * kBlock + 1024 + 512; }
};

template <int DP, int W, int BN, int NB, bool HALF, bool MASKED, int CTAS>
__global__ void __launch_bounds__(FwdShape<DP, W, BN, NB>::kThreads, CTAS)
    attn_tc_kernel(const __grid_constant__ AttnFwdArgs p) {
  using Shape = FwdShape<DP, W, BN, NB>;
  using T = typename std::conditional<HALF, __half, __nv_bfloat16>::type;
  const AttnArgs& a = p.a;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* sq = smem;
  uint8_t* skv = sq + W * Shape::kTileQ;
  uint64_t* full = reinterpret_cast<uint64_t*>(skv + p.stages * 2 * Shape::kBlock);
  uint64_t* empty = full + kMaxStages;
  uint64_t* clean = empty + kMaxStages;                                     // (the slot's rows are cleared)
  uint64_t* qfull = clean + kMaxStages;
  uint64_t* sfull = qfull + 1;                                             // [tile][place]
  uint64_t* pfull = sfull + NB * W;
  uint64_t* pvdone = pfull + NB * W;
  uint64_t* ofull = pvdone + W;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(ofull + W);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  BlockRange* ranges = reinterpret_cast<BlockRange*>(tmem_holder + 2);

  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const int nodes = 128 >> p.pack_log, pack = 1 << p.pack_log;             // of a tile
  const int r0 = blockIdx.x * (W * nodes);
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
      for (int k = 0; k < NB; ++k) {
        mbar_init(smem_u32(&sfull[NB * t + k]), 1);
        mbar_init(smem_u32(&pfull[NB * t + k]), 128);
      }
      mbar_init(smem_u32(&pvdone[t]), 1);
      mbar_init(smem_u32(&ofull[t]), 1);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 4 * W) tmem_alloc(tmem_holder, Shape::kCols);
  grid_dependency_wait();
  const WarpOffsets offsets(a);
  Span f, l;
  const TileKeys tile_keys = attn_tile_keys(a, offsets, r0, r0 + W * nodes, f, l);
  const KeyBlocks<BN> keys(tile_keys);
  const int blocks = keys.count;
  if (W > 1 && warp < W) {
    Span x, y;
    const BlockRange r = block_range<BN>(keys, attn_tile_keys(a, offsets, r0 + warp * nodes, r0 + (warp + 1) * nodes, x, y));
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
    const uint32_t quarter = tmem + ((uint32_t)((warp & 3) * 32) << 16) + t * Shape::kAcc, acc = quarter + NB * BN;
    const int i = r0 + t * nodes + (row >> p.pack_log), h = h0 + (row & (pack - 1));
    const RowKeys r = i < a.n ? attn_row_keys(a, i, attn_span_near(a, i, f, l)) : RowKeys{0, 0, 0, 0};
    const FullBlocks whole(keys, r, MASKED, std::integral_constant<int, BN>());
    const float c = a.scale_log2;
    const uint64_t c2 = pair(c, c);
    constexpr float up = HALF ? 7.f : 0.f;                                 // (p is kept at 2^up p, and so is its sum)
    float ref = -INFINITY, total = 0.f;                                    // the reference, in powers of two
    uint32_t seen = r.hi > r.lo;                                           // (a node in a sequence sees itself, unless hidden)
    if (MASKED) seen = 0;
    int done = 0;
    bool alive = true;
    KeptKeys<BN> kept, ahead;
    if (MASKED && blocks > 0) ahead.ask(a, keys.key(0), a.n);
    for (int b = 0; b < blocks && alive; ++b) {
      if (MASKED) {
        kept = ahead;
        if (b + 1 < blocks) ahead.ask(a, keys.key(b + 1), a.n);
      }
      if (!active(t, b)) continue;
      const int place = done % NB, j = keys.key(b);
      const uint32_t lanes = quarter + place * BN;
      const bool first = keys.is_first(b);
      const bool all = whole.has(b);
      uint32_t bits[BN / 32];
      if (!all) {
#pragma unroll
        for (int k = 0; k < BN / 32; ++k) {
          bits[k] = first ? seen_first(keys, r, 32 * k) : seen_bits(a, r, j + 32 * k);
          if (MASKED) bits[k] &= kept.bits(k);
          if (MASKED) seen |= bits[k];
        }
      }
      alive = mbar_wait(smem_u32(&sfull[NB * t + place]), (done / NB) & 1, abort_flag, p.status, kErrAttnS);
      alive = __all_sync(0xffffffffu, alive);
      if (!alive) break;
      tc_fence_after();
      float s[BN];
      tmem_load<BN>(lanes, s);
      tmem_wait_ld();
      if (!all) {
        // (a hidden score is -inf, c > 0: its p is 0)
#pragma unroll
        for (int e = 0; e < BN; ++e)
          if (!((bits[e / 32] >> (e & 31)) & 1)) s[e] = -INFINITY;
      }
      float tops[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
      for (int e = 4; e < BN; e += 2) tops[(e / 2) & 3] = max3(tops[(e / 2) & 3], s[e], s[e + 1]);
      const float top = max3(fmaxf(tops[0], tops[1]), tops[2], tops[3]) * c;
      const bool move = top > ref + 8.f;                                   // (from -inf too)
      if (__any_sync(0xffffffffu, move)) {
        const float keep = move ? exp2_approx(ref - top) : 1.f;
        if (move) {
          ref = top;
          total *= keep;
        }
        if (done > 0) {
          // (the last block's product may still be adding to O)
          alive = mbar_wait(smem_u32(&pvdone[t]), (done - 1) & 1, abort_flag, p.status, kErrAttnO);
          alive = __all_sync(0xffffffffu, alive);
          if (!alive) break;
          tc_fence_after();
#pragma unroll 1
          for (int d = 0; d < a.dim; d += 16) {
            uint32_t o[16];
            tmem_ld16(acc + d, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
            tmem_st16(acc + d, o);
          }
        }
      }
      const float base = ref == -INFINITY ? 0.f : ref;
      const uint64_t base2 = pair(up - base, up - base);
      uint64_t sums[2] = {pair(total, 0.f), 0};
#pragma unroll
      for (int k = 0; k < BN / 32; ++k) {
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float2 x = unpair(fma2(pair(s[32 * k + 2 * e], s[32 * k + 2 * e + 1]), c2, base2));
          const float px = exp2_approx(x.x), py = exp2_approx(x.y);
          sums[e & 1] = add2(sums[e & 1], pair(px, py));
          w[e] = pack16<HALF>(px, py);
        }
        tmem_st16(lanes + 16 * k, w);                                      // (where the scores lay: all read)
      }
      const float2 sum = unpair(add2(sums[0], sums[1]));
      total = sum.x + sum.y;
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(smem_u32(&pfull[NB * t + place]));
      ++done;
    }
    // ---------------- O / sum ----------------
    if (done > 0 && alive) alive = mbar_wait(smem_u32(&ofull[t]), 0, abort_flag, p.status, kErrAttnO);
    alive = __all_sync(0xffffffffu, alive);
    tc_fence_after();
    if (alive) {
      const bool none = seen == 0;
      if (!none && total == 0.f) total = NAN;                              // scores of -inf alone have no softmax
      const float inv = none ? 0.f : 1.f / total;
      bool bad = false;
      T* dst = (T*)p.out + ((long long)i * a.heads + h) * a.dim;
#pragma unroll 2
      for (int d = 0; d < a.dim; d += 16) {
        float x[16] = {};
        if (done > 0) {
          tmem_ld16(acc + d, reinterpret_cast<uint32_t(&)[16]>(x));
          tmem_wait_ld();
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          x[e] = none ? 0.f : x[e] * inv;
          bad |= not_finite(x[e]);
        }
        if (i < a.n) store_row<HALF>(dst, d, a.dim, p.wide, x);
      }
      if (p.lse != nullptr) {                  // (a loop of its own: in the one above, a pass without it took 1 % longer)
        T* rest = attn_rest<T>(a, p.lse) + ((long long)i * a.heads + h) * a.dim;
#pragma unroll 1
        for (int d = 0; d < a.dim; d += 16) {
          float x[16] = {};
          if (done > 0) {
            tmem_ld16(acc + d, reinterpret_cast<uint32_t(&)[16]>(x));
            tmem_wait_ld();
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) x[e] = none ? 0.f : rounded_off<T>(x[e] * inv);
          if (i < a.n) store_row<HALF>(rest, d, a.dim, p.wide, x);
        }
      }
      if (i < a.n && p.lse != nullptr) p.lse[(long long)h * a.n + i] = none ? INFINITY : ref + (log2f(total) - up);
      // (a total that is no number is the row's own doing: a hidden key is not in it)
      unsigned redo = __ballot_sync(0xffffffffu, bad && i < a.n && !not_finite(total));
      __syncwarp();
      while (redo != 0) {
        const int at = __ffs(redo) - 1, ri = __shfl_sync(0xffffffffu, i, at), rh = __shfl_sync(0xffffffffu, h, at);
        redo &= redo - 1;
        if (!attn_row_is_spoilt<T>(a, ri, rh, (const T*)p.out)) attn_forward_row<T>(a, ri, rh, (T*)p.out, p.lse);
      }
    }
  } else if (warp < 5 * W) {
    // ---------------- products: a warp per tile ----------------
    // (The whole warp walks the loop, so that descriptors are formed in uniform registers; one thread of it issues.)
    if (blocks > 0) {
      const int t = warp - 4 * W;
      const bool leader = elect_one();
      const uint32_t idesc_s = attn_idesc<HALF>(BN, false), idesc_o = attn_idesc<HALF>(16 * ksteps, true);
      const uint32_t q = smem_u32(sq + t * Shape::kTileQ), kv = smem_u32(skv), d = tmem + t * Shape::kAcc;
      uint64_t* ready = cleared ? clean : full;
      BlockRange range;
      if (W > 1) range = ranges[t];
      auto needs = [&](int b) { return W == 1 || in_range(range, b); };
      int scored = 0, n = 0, stage = 0;
      uint32_t phase = 0;
      bool alive = mbar_wait(smem_u32(qfull), 0, abort_flag, p.status, kErrAttnQ);
      auto scores = [&](int s) {
        // The place's last P has to be through.  (The last product that was issued is waited for: without a gap it is that one,
        // and behind blocks that this tile passes over an older one may be two phases back, where its parity would be wrong.)
        if (scored >= NB) alive = mbar_wait(smem_u32(&pvdone[t]), (n - 1) & 1, abort_flag, p.status, kErrAttnO);
        if (!alive) return;
        tc_fence_after();
        if (leader) {
          product_channels<DP / 16, 128, BN>(d + scored % NB * BN, q, kv + s * 2 * Shape::kBlock, ksteps, idesc_s);
          umma_commit(smem_u32(&sfull[NB * t + scored % NB]));
        }
        ++scored;
      };
      if (alive) alive = mbar_wait(smem_u32(&ready[0]), 0, abort_flag, p.status, kErrAttnLoad);
      if (alive && needs(0)) scores(0);
      for (int b = 0; b < blocks && alive; ++b) {
        const int next = stage + 1 == p.stages ? 0 : stage + 1;
        const uint32_t next_phase = next == 0 ? phase ^ 1u : phase;
        const bool more = b + 1 < blocks;
        if (more) alive = mbar_wait(smem_u32(&ready[next]), next_phase, abort_flag, p.status, kErrAttnLoad);
        if (NB > 1 && alive && more && needs(b + 1)) scores(next);
        if (alive && needs(b)) {
          alive = mbar_wait(smem_u32(&pfull[NB * t + n % NB]), (n / NB) & 1, abort_flag, p.status, kErrAttnP);
          if (!alive) break;
          tc_fence_after();
          if (leader) {
            product_rows<BN>(d + NB * BN, d + n % NB * BN, kv + stage * 2 * Shape::kBlock + Shape::kBlock, idesc_o, n == 0);
            umma_commit(smem_u32(&pvdone[t]));
          }
          ++n;
        }
        if (alive && leader && b + p.stages < blocks) umma_commit(smem_u32(&empty[stage]));
        if (NB == 1 && alive && more && needs(b + 1)) scores(next);
        stage = next;
        phase = next_phase;
      }
      if (leader) umma_commit(smem_u32(&ofull[t]));              // (a barrier of its own: rows cannot tell pvdone's phases apart)
      if (!alive)
        for (int it = 0; it < 64; ++it) __nanosleep(1000);       // (products under way end before tensor memory is freed)
    }
  } else if (blocks > 0) {
    // ---------------- copies ----------------
    if (lane == 0) {
      mbar_arrive_expect_tx(smem_u32(qfull), W * tile_bytes<128>(a.dim));
      for (int t = 0; t < W; ++t)
        tma_tile<Shape::kPieces, 128>(smem_u32(sq + t * Shape::kTileQ), &p.q, a.dim, h0, r0 + t * nodes, smem_u32(qfull));
    }
    int stage = 0, cstage = 0;
    uint32_t phase = 1, cphase = 0, words[BN / 32];
    bool alive = true;
    for (int b = 0; b < blocks + (cleared ? 1 : 0) && alive; ++b) {
      if (b < blocks) {
        if (b >= p.stages) alive = mbar_wait(smem_u32(&empty[stage]), phase, abort_flag, p.status, kErrAttnSlot);
        if (!alive) break;
        if (lane == 0) {
          const uint32_t dst = smem_u32(skv + stage * 2 * Shape::kBlock), bar = smem_u32(&full[stage]);
          mbar_arrive_expect_tx(bar, 2 * tile_bytes<BN>(a.dim));
          tma_tile<Shape::kPieces, BN>(dst, &p.k, a.dim, hk, keys.key(b), bar);
          tma_tile<Shape::kPieces, BN>(dst + Shape::kBlock, &p.v, a.dim, hk, keys.key(b), bar);
        }
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      KeptKeys<BN> kept;
      if (cleared && b < blocks) kept.ask(a, keys.key(b), end);
      // the stage before has landed or is about to: its V (a hidden key's score is not read)
      if (cleared && b > 0) {
        alive = mbar_wait(smem_u32(&full[cstage]), cphase, abort_flag, p.status, kErrAttnLoad);
        alive = __all_sync(0xffffffffu, alive);
        if (!alive) break;
        clear_rows<Shape::kPieces, BN>(skv + (cstage * 2 + 1) * Shape::kBlock, [&](int k) { return words[k]; });
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
        for (int k = 0; k < BN / 32; ++k) words[k] = kept.bits(k);
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

template <int DP, int W, int BN, int NB, bool HALF, bool MASKED, int CTAS>
int fwd_launch_kernel(AttnFwdArgs& p, cudaStream_t st) {
  using Shape = FwdShape<DP, W, BN, NB>;
  constexpr size_t kMost = (227 * 1024) / CTAS - 1024;
  constexpr int dtype = HALF ? OCNN_F16 : OCNN_BF16;
  int stages = kMaxStages;
  static_assert(Shape::smem(3) <= kMost, "with a mask, three stages at least: one is cleared while two are read");
  while (Shape::smem(stages) > kMost) --stages;
  p.stages = stages;
  const size_t bytes = Shape::smem(stages);
  const AttnArgs& a = p.a;
  int status = attn_map(&p.q, a.q, dtype, a.dim, a.heads, a.n, a.q_row, a.q_head, 1 << p.pack_log, 128 >> p.pack_log);
  if (status == OCNN_OK) status = attn_map(&p.k, a.k, dtype, a.dim, a.kv_heads, a.n, a.k_row, a.k_head, 1, BN);
  if (status == OCNN_OK) status = attn_map(&p.v, a.v, dtype, a.dim, a.kv_heads, a.n, a.v_row, a.v_head, 1, BN);
  if (status != OCNN_OK) return status;
  static PerDeviceOnce once;
  status = once.run([&]() -> int {
    OCNN_CUDA_OK(cudaFuncSetAttribute(attn_tc_kernel<DP, W, BN, NB, HALF, MASKED, CTAS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)bytes));
    return OCNN_OK;
  });
  if (status != OCNN_OK) return status;
  const int nodes = W * 128 >> p.pack_log;
  OCNN_CUDA_OK(launch_chained(attn_tc_kernel<DP, W, BN, NB, HALF, MASKED, CTAS>,
                              dim3(ceil_div(a.n, nodes), a.heads >> p.pack_log), dim3(Shape::kThreads), bytes, st, p));
  OCNN_LAUNCH_OK("attn_tc_kernel");
  return OCNN_OK;
}

template <int DP, int W, int BN, int NB, bool HALF, int CTAS>
int fwd_launch(AttnFwdArgs& p, cudaStream_t st) {
  return p.a.mask != nullptr ? fwd_launch_kernel<DP, W, BN, NB, HALF, true, CTAS>(p, st)
                             : fwd_launch_kernel<DP, W, BN, NB, HALF, false, CTAS>(p, st);
}

template <bool HALF>
int fwd_by_width(AttnFwdArgs& p, cudaStream_t st) {
  // Up to 64 channels a tile's tensor memory is a quarter of the SM's with one place for scores, and three CTAs share an SM:
  // 60 k nodes, 8 heads of 32, window 256: 161 us; with two places and two CTAs 178.  At 128 channels there is room for two
  // tiles, which share their copies of K and V and have two places each.
  if (p.a.dim <= 32) return fwd_launch<32, 1, 64, 1, HALF, 3>(p, st);
  if (p.a.dim <= 64) return fwd_launch<64, 1, 64, 1, HALF, 3>(p, st);
  return fwd_launch<128, 2, 64, 2, HALF, 1>(p, st);
}

}  // namespace

int attn_tc_forward(const AttnArgs& a, int dtype, void* out, float* lse, int* status, cudaStream_t st) {
  AttnFwdArgs p;
  p.a = a;
  p.out = out;
  p.lse = lse;
  p.status = status;
  p.pack_log = attn_pack_log(a);
  p.wide = wide_rows(out, a.dim) && wide_rows(lse, a.dim);
  return dtype == OCNN_F16 ? fwd_by_width<true>(p, st) : fwd_by_width<false>(p, st);
}

}  // namespace ocnn
