// Attention over a window of nodes on the tensor cores, 16-bit data: forward pass.
//
// A CTA takes W tiles of 128 rows against the keys that they see, in blocks of BN keys.  A row is a query head of a node:
// P heads that share a key head stand side by side (P the largest power of two in the group), so that 128 / P nodes share
// each copy of keys and values and the tile's windows overlap more.  Per block and tile
//     S = Q K^T (tensor memory) -> p = exp2(S scale - m) -> P (tensor memory, in S's place) -> O += P V
// with 128 threads per tile, one row each, between the two products.  m is the row's reference: its running maximum, but
// moved only when a block exceeds it by more than 8 (any reference gives the same quotient as long as nothing overflows,
// and 2^8 is far from that), so O is hardly ever scaled.  P is rounded to the data's type, which is what the product takes;
// its sum is of the unrounded values.
//
// Roles: 4 W warps of rows (they load Q, form P and write O), one warp that copies K and V blocks into a ring of slots
// (16 bytes per cp.async: any strides, zeros for keys that the mask hides), one thread that issues the products.
#include "attention_tc.cuh"

namespace ocnn {
namespace {

struct AttnFwdArgs {
  AttnArgs a;
  void* out;
  float* lse;
  int* status;
  int pack_log, slots;
};

enum : int { kErrAttnQ = 11, kErrAttnLoad = 12, kErrAttnSlot = 13, kErrAttnP = 14, kErrAttnS = 15, kErrAttnO = 16 };

template <int DP, int W, int BN>
struct FwdShape {
  static constexpr int kLoad = DP > 64 ? 2 : 1;                            // warps that copy
  static constexpr int kThreads = 128 * W + 32 * W + 32 * kLoad;         // rows, products, copies
  static constexpr int kPieces = DP / 64 > 0 ? DP / 64 : 1;
  static constexpr int kTileQ = 128 * kRowBytes * kPieces;
  static constexpr int kSlot = BN * kRowBytes * kPieces;
  static constexpr int kAcc = BN + DP;                                   // S and O of a tile
  static constexpr int kCols = W * kAcc <= 64 ? 64 : W * kAcc <= 128 ? 128 : W * kAcc <= 256 ? 256 : 512;
  static constexpr size_t smem(int slots) { return (size_t)W * kTileQ + (size_t)slots * kSlot + 1024 + 512; }
};

template <int DP, int W, int BN, bool HALF, int CTAS>
__global__ void __launch_bounds__(FwdShape<DP, W, BN>::kThreads, CTAS) attn_tc_kernel(const AttnFwdArgs p) {
  using Shape = FwdShape<DP, W, BN>;
  using T = typename std::conditional<HALF, __half, __nv_bfloat16>::type;
  constexpr int kMaxSlots = 8;
  const AttnArgs& a = p.a;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* sq = smem;
  uint8_t* skv = sq + W * Shape::kTileQ;
  uint64_t* full = reinterpret_cast<uint64_t*>(skv + p.slots * Shape::kSlot);
  uint64_t* empty = full + kMaxSlots;
  uint64_t* qfull = empty + kMaxSlots;
  uint64_t* sfull = qfull + 1;
  uint64_t* pfull = sfull + W;
  uint64_t* pvdone = pfull + W;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(pvdone + W);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  int* ranges = reinterpret_cast<int*>(tmem_holder + 2);                   // per tile: first and last block, first nodes

  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const int nodes = 128 >> p.pack_log, pack = 1 << p.pack_log;             // of a tile
  const int r0 = blockIdx.x * (W * nodes);
  const int group = a.heads / a.kv_heads, per_kv = group >> p.pack_log;
  const int hk = blockIdx.y / per_kv, h0 = hk * group + (blockIdx.y % per_kv) * pack;

  if (tid == 0) {
    for (int s = 0; s < p.slots; ++s) {
      mbar_init(smem_u32(&full[s]), 32 * Shape::kLoad);
      mbar_init(smem_u32(&empty[s]), W);
    }
    mbar_init(smem_u32(qfull), 128 * W);
    for (int t = 0; t < W; ++t) {
      mbar_init(smem_u32(&sfull[t]), 1);
      mbar_init(smem_u32(&pfull[t]), 128);
      mbar_init(smem_u32(&pvdone[t]), 1);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 4 * W) tmem_alloc(tmem_holder, Shape::kCols);
  const TileKeys keys = attn_tile_keys(a, r0, r0 + W * nodes);
  const int blocks = (keys.n + BN - 1) / BN;
  if (W > 1 && tid < W) {
    // the blocks that tile t needs: an interval, and the first block where it holds first nodes that the tile sees
    const TileKeys k = attn_tile_keys(a, r0 + tid * nodes, r0 + (tid + 1) * nodes);
    const int at = k.lo - keys.lo + keys.n_first, end = at + k.n - k.n_first;
    ranges[3 * tid] = k.n > 0 ? at / BN : 0;
    ranges[3 * tid + 1] = k.n > 0 ? (end + BN - 1) / BN : 0;
    ranges[3 * tid + 2] = k.n > 0 && keys.n_first > 0 && k.first == keys.first;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  auto active = [&](int t, int b) {
    if (W == 1) return true;
    return (b >= ranges[3 * t] && b < ranges[3 * t + 1]) || (b == 0 && ranges[3 * t + 2] != 0);
  };
  const int ksteps = (a.dim + 15) / 16;

  if (warp < 4 * W) {
    // ---------------- rows ----------------
    const int t = warp >> 2, row = tid & 127;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16) + t * Shape::kAcc, acc = lanes + BN;
    if (blocks > 0) {
      const int node = r0 + t * nodes;
      const PackedRows q = {(const uint8_t*)((const T*)a.q + h0 * a.q_head), (int)(a.q_row * 2), p.pack_log, a.q_head * 2};
      copy_tile<DP, 128, 128>(smem_u32(sq + t * Shape::kTileQ), row, a.dim, a.q, [&](int r) { return q(node, r); },
                              [&](int r) { return node + (r >> p.pack_log) < a.n; });
      cp_async_arrive(smem_u32(qfull));
    }
    const int i = r0 + t * nodes + (row >> p.pack_log), h = h0 + (row & (pack - 1));
    const RowKeys r = i < a.n ? attn_row_keys(a, i, attn_span(a, i)) : RowKeys{0, 0, 0, 0};
    const float c = a.scale_log2;
    float ref = -INFINITY, total = 0.f;                                    // the reference, in powers of two
    int done = 0;
    bool alive = true;
    for (int b = 0; b < blocks && alive; ++b) {
      if (!active(t, b)) continue;
      uint32_t bits[BN / 32];
#pragma unroll
      for (int k = 0; k < BN / 32; ++k) {
        bits[k] = seen_bits(a, keys, r, b * BN + 32 * k);
        if (a.mask != nullptr) {
          const int at = b * BN + 32 * k + lane;
          bits[k] &= __ballot_sync(0xffffffffu, at < keys.n && a.mask[keys.key(at)] != 0);
        }
      }
      alive = mbar_wait(smem_u32(&sfull[t]), done & 1, abort_flag, p.status, kErrAttnS);
      alive = __all_sync(0xffffffffu, alive);
      if (!alive) break;
      tc_fence_after();
      float s[BN];
      tmem_load<BN>(lanes, s);
      bool all = true;
#pragma unroll
      for (int k = 0; k < BN / 32; ++k) all = all && bits[k] == 0xffffffffu;
      all = __all_sync(0xffffffffu, all);
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
      const uint64_t c2 = pair(c, c), base2 = pair(-base, -base);
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
      mbar_arrive(smem_u32(&pfull[t]));
      ++done;
    }
    // ---------------- O / sum ----------------
    bool bad = false;
    if (done > 0 && alive) {
      alive = mbar_wait(smem_u32(&pvdone[t]), (done - 1) & 1, abort_flag, p.status, kErrAttnO);
      alive = __all_sync(0xffffffffu, alive);
      tc_fence_after();
    }
    if (alive) {
      const bool empty_row = total == 0.f;
      const float inv = empty_row ? 0.f : 1.f / total;
      bad = not_finite(total);
      T* dst = (T*)p.out + ((long long)i * a.heads + h) * a.dim;
#pragma unroll 1
      for (int d = 0; d < a.dim; d += 16) {
        uint32_t o[16];
        if (done > 0) {
          tmem_ld16(acc + d, o);
          tmem_wait_ld();
        }
        uint32_t w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = empty_row ? 0.f : __uint_as_float(o[2 * e]) * inv;
          const float y = empty_row ? 0.f : __uint_as_float(o[2 * e + 1]) * inv;
          bad |= not_finite(x) | (d + 2 * e + 1 < a.dim && not_finite(y));
          w[e] = pack16<HALF>(x, y);
        }
        if (i < a.n) {
          // (dim is a multiple of 8, rows start on 16-byte boundaries)
          *reinterpret_cast<uint4*>(dst + d) = make_uint4(w[0], w[1], w[2], w[3]);
          if (d + 8 < a.dim) *reinterpret_cast<uint4*>(dst + d + 8) = make_uint4(w[4], w[5], w[6], w[7]);
        }
      }
      if (i < a.n && p.lse != nullptr) p.lse[(long long)h * a.n + i] = empty_row ? INFINITY : ref + log2f(total);
      unsigned redo = __ballot_sync(0xffffffffu, bad && i < a.n);
      while (redo != 0) {
        const int at = __ffs(redo) - 1;
        redo &= redo - 1;
        attn_forward_row<T>(a, __shfl_sync(0xffffffffu, i, at), __shfl_sync(0xffffffffu, h, at), (T*)p.out, p.lse);
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
      uint32_t full_phase = 0;                                             // per slot
      int n = 0;
      bool alive = mbar_wait(smem_u32(qfull), 0, abort_flag, p.status, kErrAttnQ);
      auto wait_slot = [&](int s) {
        if (alive) alive = mbar_wait(smem_u32(&full[s]), (full_phase >> s) & 1, abort_flag, p.status, kErrAttnLoad);
        full_phase ^= 1u << s;
        proxy_fence();
      };
      auto scores = [&](int slot) {
        tc_fence_after();
        if (leader) {
          product_channels<DP / 16, 128, BN>(d, q, kv + slot * Shape::kSlot, ksteps, idesc_s);
          umma_commit(smem_u32(&sfull[t]));
        }
      };
      int slot = 0;
      auto next = [&](int s) { return s + 1 == p.slots ? 0 : s + 1; };
      wait_slot(slot);
      if (alive && active(t, 0)) scores(slot);
      if (alive && leader) umma_commit(smem_u32(&empty[slot]));
      for (int b = 0; b < blocks && alive; ++b) {
        const int vs = next(slot), ks = next(vs);
        const bool more = b + 1 < blocks;
        wait_slot(vs);
        if (more) wait_slot(ks);
        if (alive && active(t, b)) {
          alive = mbar_wait(smem_u32(&pfull[t]), n & 1, abort_flag, p.status, kErrAttnP);
          if (!alive) break;
          tc_fence_after();
          if (leader) {
            product_rows<BN>(d + BN, d, kv + vs * Shape::kSlot, idesc_o, n == 0);
            umma_commit(smem_u32(&pvdone[t]));
          }
          ++n;
        }
        if (alive && more && leader) umma_commit(smem_u32(&empty[vs]));
        // (S lies where P does: the product that reads P has to be through)
        if (alive && more && active(t, b + 1)) {
          if (n > 0) alive = mbar_wait(smem_u32(&pvdone[t]), (n - 1) & 1, abort_flag, p.status, kErrAttnO);
          if (alive) scores(ks);
        }
        if (alive && more && leader) umma_commit(smem_u32(&empty[ks]));
        slot = ks;
      }
      if (!alive)
        for (int it = 0; it < 64; ++it) __nanosleep(1000);       // (products under way end before tensor memory is freed)
    }
  } else {
    // ---------------- copies of K and V ----------------
    const int thread = tid - 160 * W;
    const uint8_t* const base[2] = {(const uint8_t*)((const T*)a.k + hk * a.k_head),
                                    (const uint8_t*)((const T*)a.v + hk * a.v_head)};
    const int stride[2] = {(int)(a.k_row * 2), (int)(a.v_row * 2)};
    int slot = 0;
    uint32_t empty_phase = 0;
    bool alive = true;
    for (int b = 0; b < blocks && alive; ++b) {
      uint32_t kept[BN / 32];
#pragma unroll
      for (int k = 0; k < BN / 32; ++k) {
        const int at = b * BN + 32 * k + lane;
        kept[k] = __ballot_sync(0xffffffffu, at < keys.n && (a.mask == nullptr || a.mask[keys.key(at)] != 0));
      }
      const int j0 = keys.lo - keys.n_first + b * BN, nf = keys.n_first - b * BN, early = keys.first - j0;
#pragma unroll 1
      for (int kv = 0; kv < 2 && alive; ++kv) {
        if (2 * b + kv >= p.slots) {
          alive = mbar_wait(smem_u32(&empty[slot]), (empty_phase >> slot) & 1, abort_flag, p.status, kErrAttnSlot);
          alive = __all_sync(0xffffffffu, alive);
          empty_phase ^= 1u << slot;
          if (!alive) break;
        }
        copy_tile<DP, BN, 32 * Shape::kLoad>(
            smem_u32(skv + slot * Shape::kSlot), thread, a.dim, base[0],
            [&](int r) { return base[kv] + (long long)(j0 + r + (r < nf ? early : 0)) * stride[kv]; },
            [&](int r) { return ((r < 32 ? kept[0] : r < 64 ? kept[1] : r < 96 ? kept[BN / 32 - 2] : kept[BN / 32 - 1]) >> (r & 31)) & 1; });
        cp_async_arrive(smem_u32(&full[slot]));
        slot = slot + 1 == p.slots ? 0 : slot + 1;
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 4 * W)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)Shape::kCols) : "memory");
}

template <int DP, int W, int BN, bool HALF, int CTAS>
int fwd_launch(AttnFwdArgs& p, cudaStream_t st) {
  using Shape = FwdShape<DP, W, BN>;
  constexpr size_t kMost = (227 * 1024) / CTAS - 1024;
  int slots = 8;
  while (slots > 3 && Shape::smem(slots) > kMost) --slots;
  p.slots = slots;
  const size_t bytes = Shape::smem(slots);
  static PerDeviceOnce once;
  const int status = once.run([&]() -> int {
    OCNN_CUDA_OK(cudaFuncSetAttribute(attn_tc_kernel<DP, W, BN, HALF, CTAS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)bytes));
    return OCNN_OK;
  });
  if (status != OCNN_OK) return status;
  const int nodes = W * 128 >> p.pack_log;
  attn_tc_kernel<DP, W, BN, HALF, CTAS><<<dim3(ceil_div(p.a.n, nodes), p.a.heads >> p.pack_log), Shape::kThreads, bytes, st>>>(p);
  OCNN_LAUNCH_OK("attn_tc_kernel");
  return OCNN_OK;
}

template <bool HALF>
int fwd_by_width(AttnFwdArgs& p, cudaStream_t st) {
  if (p.a.dim <= 32) return fwd_launch<32, 1, 64, HALF, 3>(p, st);
  if (p.a.dim <= 64) return fwd_launch<64, 1, 64, HALF, 3>(p, st);
  return fwd_launch<128, 2, 128, HALF, 1>(p, st);
}

}  // namespace

int attn_tc_forward(const AttnArgs& a, int dtype, void* out, float* lse, int* status, cudaStream_t st) {
  AttnFwdArgs p = {a, out, lse, status, attn_pack_log(a), 0};
  return dtype == OCNN_F16 ? fwd_by_width<true>(p, st) : fwd_by_width<false>(p, st);
}

}  // namespace ocnn
