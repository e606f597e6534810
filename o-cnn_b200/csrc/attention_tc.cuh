// What the tensor-core attention kernels share: tiles in shared memory, probabilities through tensor memory.
//
// A tile of rows (queries, keys, values, gradients) lies as [64 channels][row] pieces of 128 bytes, swizzled: as it is the
// K-major operand of a product over channels (scores), and, read the other way, the MN-major operand of a product over
// rows (probabilities times values).  So one copy of K, V, Q or dO serves both of its products.
#pragma once

#include <cuda.h>

#include "attention.cuh"
#include "tc.cuh"

namespace ocnn {
namespace {

constexpr int kRowBytes = 128;                 // 64 channels of 16 bits

// MN-major, 128-byte swizzle: 64 contiguous channels per row, eight rows per 1024-byte atom (the stride between atoms along
// the rows), pieces of 64 channels `piece` bytes apart (the leading stride).
__device__ __forceinline__ uint64_t smem_desc_mn128(uint32_t addr, uint32_t piece) {
  return (uint64_t)((addr & 0x3ffffu) >> 4) | ((uint64_t)(piece >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}

// One thread of the warp, the same every time.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\tselp.u32 %0, 1, 0, e;\n\t}" : "=r"(p));
  return p != 0;
}

// D[tmem] (+)= A[tmem] B[smem]
__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,"
      "%29,%30,%31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
        "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]),
      "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]),
      "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Whether a phase is complete, asked ahead of the wait for it: the answer of a barrier takes some 200 cycles however long ago
// it was complete, and asked early it comes while other work goes on.
__device__ __forceinline__ uint32_t mbar_ask(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok;
}

// The calling thread's arrival on `bar` once its copies so far have landed.
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

// Copies of ROWS rows of `dim` channels by LANES threads, zeros up to the next multiple of 16 and for rows that are not
// live.  row(r): where row r starts.
template <int DP, int ROWS, int LANES, typename Row, typename Live>
__device__ __forceinline__ void copy_tile(uint32_t dst, int lane, int dim, const void* any, Row row, Live live) {
  constexpr int kChunks = DP / 8, kStep = LANES / kChunks;
  static_assert(LANES % kChunks == 0 && ROWS % kStep == 0, "every lane has whole pieces");
  const int c = lane % kChunks, sub = lane / kChunks;
  if (c >= (dim + 15) / 16 * 2) return;
  const bool in = c < (dim >> 3);
  const uint32_t base = dst + (c >> 3) * (ROWS * kRowBytes) + sub * kRowBytes, x = (c & 7) ^ (sub & 7);
#pragma unroll 8
  for (int it = 0; it < ROWS / kStep; ++it) {
    const int r = it * kStep + sub;
    const bool ok = in && live(r);
    cp_async16(base + it * (kStep * kRowBytes) + ((x ^ ((it * kStep) & 7)) << 4), ok ? row(r) + c * 16 : any,
               ok ? 16u : 0u);
  }
}

// ---- tiles by TMA ---------------------------------------------------------------------------------------------
// A box of 64 channels x `heads` heads x `nodes` nodes of a [n, heads, dim] tensor: (node, head) rows, swizzled as above;
// what lies outside of the tensor reads as zeros.
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* map, int channel, int head, int node, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(map), "r"(channel), "r"(head), "r"(node), "r"(bar)
      : "memory");
}
template <int PIECES, int ROWS>
__device__ __forceinline__ void tma_tile(uint32_t dst, const CUtensorMap* map, int dim, int head, int node, uint32_t bar) {
#pragma unroll
  for (int c = 0; c < PIECES; ++c)
    if (c == 0 || 64 * c < dim) tma_box(dst + c * (ROWS * kRowBytes), map, 64 * c, head, node, bar);
}
// Bytes that a tile's boxes bring.
template <int ROWS>
__device__ __forceinline__ uint32_t tile_bytes(int dim) { return (uint32_t)(dim > 64 ? 2 : 1) * ROWS * kRowBytes; }

inline int attn_map(CUtensorMap* map, const void* base, int dtype, int dim, int heads, int n, long long row, long long head,
                    int box_heads, int box_nodes) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static const Encode encode = [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &found) != cudaSuccess) fn = nullptr;
    return (Encode)fn;
  }();
  if (encode == nullptr) return fail(OCNN_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
  const cuuint64_t dims[3] = {(cuuint64_t)dim, (cuuint64_t)heads, (cuuint64_t)n};
  // (the stride of a dimension of one is whatever its tensor says: any will do)
  const cuuint64_t strides[2] = {heads == 1 ? 16 : (cuuint64_t)head * 2, n == 1 ? 16 : (cuuint64_t)row * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_nodes}, steps[3] = {1, 1, 1};
  const CUresult rc = encode(map, dtype == OCNN_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                             const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (rc != CUDA_SUCCESS) return fail(OCNN_ERR_CUDA, "cuTensorMapEncodeTiled: error %d", (int)rc);
  return OCNN_OK;
}

// ---- the keys of a tile of queries ------------------------------------------------------------------------------
// The keys that the nodes [r0, r1) see between them (TileKeys), by a whole warp.  Windows move on with the nodes, so the
// first and the last node that are in a sequence say it all; their sequences go to f and l.
__device__ __forceinline__ TileKeys attn_tile_keys(const AttnArgs& a, const WarpOffsets& offsets, int r0, int r1, Span& f, Span& l) {
  TileKeys t = {0, 0, 0, 0};
  const int x = max(r0, offsets.begin()), y = min(min(r1, a.n), offsets.end(a)) - 1;
  f = l = Span{0, 0, 0};
  if (x > y) return t;
  f = offsets.span(a, x);
  l = y < f.end ? f : offsets.span(a, y);
  const RowKeys rx = attn_row_keys(a, x, f), ry = attn_row_keys(a, y, l);
  t.lo = rx.lo;
  if (a.sinks > 0) {
    t.first = f.start;                         // (the last of the tile's nodes in the first one's sequence sees most of them)
    t.n_first = max(0, min(attn_row_keys(a, min(y, f.end - 1), f).first, t.lo) - f.start);
  }
  t.n = t.n_first + max(0, max(ry.hi, ry.first) - t.lo);
  return t;
}
// They are taken in blocks of BN consecutive keys: one for the first nodes, where they lie before the windows, and the
// windows' interval cut from its begin.
template <int BN>
struct KeyBlocks {
  int first, n_first, lo, count;
  __device__ __forceinline__ explicit KeyBlocks(const TileKeys& t)
      : first(t.first), n_first(t.n_first), lo(t.lo), count((t.n_first > 0) + (t.n - t.n_first + BN - 1) / BN) {}
  __device__ __forceinline__ bool is_first(int b) const { return b == 0 && n_first > 0; }
  __device__ __forceinline__ bool reaches(int end) const { return count > 0 && key(count - 1) + BN > end; }
  __device__ __forceinline__ int key(int b) const { return is_first(b) ? first : lo + (b - (n_first > 0)) * BN; }
};

__device__ __forceinline__ uint32_t bit_run(int lo, int hi) {      // bits [lo, hi), within 0 .. 32
  lo = max(lo, 0);
  hi = min(hi, 32);
  return hi > lo ? (0xffffffffu >> (32 - (hi - lo))) << lo : 0u;
}
// Which of the 32 keys from j on row r sees, in a block of the windows' interval; in the block of first nodes, from column c on.
__device__ __forceinline__ uint32_t seen_bits(const AttnArgs& a, const RowKeys& r, int j) {
  uint32_t w = bit_run(r.lo - j, r.hi - j);
  if (a.sinks > 0) w |= bit_run(r.start - j, r.first - j);
  return w;
}
template <int BN>
__device__ __forceinline__ uint32_t seen_first(const KeyBlocks<BN>& k, const RowKeys& r, int c) {
  return r.first > r.start && r.start == k.first ? bit_run(-c, min(k.n_first, r.first - r.start) - c) : 0u;
}
// Which keys of a block the mask keeps, of those before node `end`: read for a block ahead (`ask`), and then formed into a bit
// per key by the whole warp (`bits`, for 32 keys each).
template <int BN>
struct KeptKeys {
  unsigned char mine[BN / 32];
  __device__ __forceinline__ void ask(const AttnArgs& a, int j, int end) {
#pragma unroll
    for (int k = 0; k < BN / 32; ++k) {
      const int at = j + 32 * k + (threadIdx.x & 31);
      mine[k] = at >= end ? 0 : a.mask == nullptr ? 1 : a.mask[at];
    }
  }
  __device__ __forceinline__ uint32_t bits(int k) const { return __ballot_sync(0xffffffffu, mine[k] != 0); }
};

// Zeros in the rows of a tile that `kept` (32 rows from 32 k on) leaves out, by a whole warp: what lies there, behind the
// mask or behind the last sequence, may not be a number, and a product with a probability of 0 would be none.
template <int PIECES, int BN, typename Kept>
__device__ __forceinline__ void clear_rows(uint8_t* tile, Kept kept) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int k = 0; k < BN / 32; ++k) {
    const uint32_t bits = kept(k);
    for (int r = lane >> 3; r < 32; r += 4) {
      if ((bits >> r) & 1) continue;
#pragma unroll
      for (int c = 0; c < PIECES; ++c)
        *reinterpret_cast<uint4*>(tile + c * (BN * kRowBytes) + (32 * k + r) * kRowBytes + (lane & 7) * 16) =
            make_uint4(0, 0, 0, 0);
    }
  }
}
// Blocks [from, to) of the windows' interval of which every row of the warp sees every key.
struct FullBlocks {
  int from, to;
  template <int BN>
  __device__ __forceinline__ FullBlocks(const KeyBlocks<BN>& k, const RowKeys& r, bool masked, std::integral_constant<int, BN>) {
    const int lo = __reduce_max_sync(0xffffffffu, r.lo), hi = __reduce_min_sync(0xffffffffu, r.hi);
    const int shift = k.n_first > 0;
    from = shift + (max(lo - k.lo, 0) + BN - 1) / BN;
    to = masked || hi <= k.lo ? 0 : shift + (hi - k.lo) / BN;
  }
  __device__ __forceinline__ bool has(int b) const { return b >= from && b < to; }
};

// Which blocks a tile of several that share their copies needs: an interval, those of first nodes that lie in the shared
// interval but not in its own, and the block of first nodes.
struct BlockRange { int from, to, first_from, first_to, first; };
template <int BN>
__device__ __forceinline__ BlockRange block_range(const KeyBlocks<BN>& all, const TileKeys& own) {
  BlockRange r = {0, 0, 0, 0, 0};
  const int shift = all.n_first > 0;
  if (own.n > own.n_first) {
    r.from = shift + (own.lo - all.lo) / BN;
    r.to = shift + (own.lo - all.lo + own.n - own.n_first + BN - 1) / BN;
  }
  if (own.n_first > 0) {
    const int x = max(own.first, all.lo), y = own.first + own.n_first;
    if (y > x) {
      r.first_from = shift + (x - all.lo) / BN;
      r.first_to = shift + (y - all.lo + BN - 1) / BN;
    }
    r.first = all.n_first > 0 && own.first == all.first;
  }
  return r;
}
__device__ __forceinline__ bool in_range(const BlockRange& r, int b) {
  return (b >= r.from && b < r.to) || (b >= r.first_from && b < r.first_to) || (b == 0 && r.first != 0);
}

// Two fp32 values as one 16-bit pair: `lo` in the lower half.
template <bool HALF>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  uint32_t w;
  if constexpr (HALF) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
  return w;
}

// Products over the channels (KS steps of 16 at most, `ksteps` of them): D[128 x n] = A B^T, both tiles as copied.
template <int KS, int ROWS_A, int ROWS_B>
__device__ __forceinline__ void product_channels(uint32_t d, uint32_t a, uint32_t b, int ksteps, uint32_t idesc) {
  const uint64_t da = smem_desc_sw128(a), db = smem_desc_sw128(b);
  auto step = [&](int k) {
    umma_bf16(d, da + (k >> 2) * (ROWS_A * kRowBytes >> 4) + (k & 3) * 2, db + (k >> 2) * (ROWS_B * kRowBytes >> 4) + (k & 3) * 2,
              idesc, k > 0 ? 1u : 0u);
  };
  if (ksteps == KS) {
#pragma unroll
    for (int k = 0; k < KS; ++k) step(k);
  } else {
#pragma unroll
    for (int k = 0; k < KS; ++k)
      if (k < ksteps) step(k);
  }
}
// Products over a block's rows: D[128 x channels] (+)= P[128 x ROWS] B, P in tensor memory.
template <int ROWS>
__device__ __forceinline__ void product_rows(uint32_t d, uint32_t p, uint32_t b, uint32_t idesc, bool first) {
  const uint64_t db = smem_desc_mn128(b, ROWS * kRowBytes);
#pragma unroll
  for (int k = 0; k < ROWS / 16; ++k) umma_ts(d, p + 8 * k, db + k * (16 * kRowBytes >> 4), idesc, !first || k > 0 ? 1u : 0u);
}

// ---- values by twos and threes (sm_100) -----------------------------------------------------------------------
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// N columns of tensor memory, all under way at once.
template <int N>
__device__ __forceinline__ void tmem_load(uint32_t addr, float (&v)[N]) {
#pragma unroll
  for (int k = 0; k < N / 32; ++k) tmem_ld32(addr + 32 * k, reinterpret_cast<uint32_t(&)[32]>(v[32 * k]));
}
template <int N>
__device__ __forceinline__ void tmem_store(uint32_t addr, const uint32_t (&v)[N]) {
#pragma unroll
  for (int k = 0; k < N / 16; ++k) tmem_st16(addr + 16 * k, reinterpret_cast<const uint32_t(&)[16]>(v[16 * k]));
}

// 16 channels of a result row from channel d on, of which those below dim count.
template <bool HALF>
__device__ __forceinline__ void store_row(void* row, int d, int dim, bool wide, const float (&x)[16]) {
  uint4 w[2];
  uint32_t* u = reinterpret_cast<uint32_t*>(w);
#pragma unroll
  for (int e = 0; e < 8; ++e) u[e] = pack16<HALF>(x[2 * e], x[2 * e + 1]);
  uint8_t* dst = (uint8_t*)row + d * 2;
  if (wide) {
    st_global_32B(dst, w[0], w[1]);
  } else {
    *reinterpret_cast<uint4*>(dst) = w[0];
    if (d + 8 < dim) *reinterpret_cast<uint4*>(dst + 16) = w[1];
  }
}
inline bool wide_rows(const void* p, int dim) { return dim % 16 == 0 && reinterpret_cast<uintptr_t>(p) % 32 == 0; }

// An instruction descriptor: fp32 accumulator, 128 rows, n columns; B K-major or MN-major.
template <bool HALF>
__device__ __forceinline__ uint32_t attn_idesc(int n, bool b_mn) {
  const uint32_t ab = HALF ? 0u : 1u;
  return (1u << 4) | (ab << 7) | (ab << 10) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}

}  // namespace
}  // namespace ocnn
