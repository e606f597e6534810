// What the tensor-core attention kernels share: tiles in shared memory, probabilities through tensor memory.
//
// A tile of rows (queries, keys, values, gradients) lies as [64 channels][row] pieces of 128 bytes, swizzled: as it is the
// K-major operand of a product over channels (scores), and, read the other way, the MN-major operand of a product over
// rows (probabilities times values).  So one copy of K, V, Q or dO serves both of its products.
#pragma once

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

// The calling thread's arrival on `bar` once its copies so far have landed.
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

// Copies of ROWS rows of `dim` channels by LANES threads, zeros up to the next multiple of 16 and for rows that are not
// live.  row(r): where row r starts.  A lane has one piece of every kStep-th row, so that all but the row's address is known
// before the loop (one warp per CTA makes all its copies: with a division and 64-bit products per piece it was the copies'
// instructions that bounded every kernel here).
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

// The rows of a tile that are (node, head) pairs, 1 << pack_log heads of each node side by side.
struct PackedRows {
  const uint8_t* base;               // node 0, first head
  int row, pack_log;                 // bytes from node to node
  long long head;
  __device__ __forceinline__ const uint8_t* operator()(int node, int r) const {
    return base + (long long)(node + (r >> pack_log)) * row + (r & ((1 << pack_log) - 1)) * head;
  }
};

// The keys that the nodes [r0, r1) see between them.  Windows move on with the nodes, so the first and the last node
// that are in a sequence say it all.
__device__ __forceinline__ TileKeys attn_tile_keys(const AttnArgs& a, int r0, int r1) {
  TileKeys t = {0, 0, 0, 0};
  const int f = max(r0, attn_offset(a, 0)), l = min(min(r1, a.n), attn_offset(a, a.batch)) - 1;
  if (f > l) return t;
  const Span sf = attn_span(a, f);
  const RowKeys rf = attn_row_keys(a, f, sf), rl = attn_row_keys(a, l, attn_span(a, l));
  t.lo = rf.lo;
  if (a.sinks > 0) {
    const int i = min(l, sf.end - 1);          // the last node of the first one's sequence
    t.first = sf.start;
    t.n_first = max(0, min(attn_row_keys(a, i, sf).first, t.lo) - sf.start);
  }
  t.n = t.n_first + max(0, max(rl.hi, rl.first) - t.lo);
  return t;
}

__device__ __forceinline__ uint32_t bit_run(int lo, int hi) {      // bits [lo, hi), within 0 .. 32
  lo = max(lo, 0);
  hi = min(hi, 32);
  return hi > lo ? (0xffffffffu >> (32 - (hi - lo))) << lo : 0u;
}
// Which of the keys with list indices t .. t + 31 row r sees.
__device__ __forceinline__ uint32_t seen_bits(const AttnArgs& a, const TileKeys& k, const RowKeys& r, int t) {
  const int base = k.lo - k.n_first + t;       // the key of column 0, behind the first nodes
  uint32_t w = bit_run(r.lo - base, r.hi - base);
  if (a.sinks > 0 && r.first > r.start) {
    w |= bit_run(max(r.start - base, k.n_first - t), r.first - base);
    if (r.start == k.first) w |= bit_run(-t, min(k.n_first, r.first - r.start) - t);
  }
  return w;
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
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    if (k >= ksteps) break;
    umma_bf16(d, da + (k >> 2) * (ROWS_A * kRowBytes >> 4) + (k & 3) * 2, db + (k >> 2) * (ROWS_B * kRowBytes >> 4) + (k & 3) * 2,
              idesc, k > 0 ? 1u : 0u);
  }
}
// Products over a block's rows: D[128 x channels] (+)= P[128 x ROWS] B, P in tensor memory.
template <int ROWS>
__device__ __forceinline__ void product_rows(uint32_t d, uint32_t p, uint32_t b, uint32_t idesc, bool first) {
  const uint64_t db = smem_desc_mn128(b, ROWS * kRowBytes);
#pragma unroll
  for (int k = 0; k < ROWS / 16; ++k) umma_ts(d, p + 8 * k, db + k * (16 * kRowBytes >> 4), idesc, !first || k > 0 ? 1u : 0u);
}

// ---- two fp32 values per instruction (sm_100) -------------------------------------------------------------------
__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(x), "f"(y));
  return p;
}
__device__ __forceinline__ float2 unpair(uint64_t p) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p));
  return f;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
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

// An instruction descriptor: fp32 accumulator, 128 rows, n columns; B K-major or MN-major.
template <bool HALF>
__device__ __forceinline__ uint32_t attn_idesc(int n, bool b_mn) {
  const uint32_t ab = HALF ? 0u : 1u;
  return (1u << 4) | (ab << 7) | (ab << 10) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}

}  // namespace
}  // namespace ocnn
