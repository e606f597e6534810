// What the attention kernels share: which keys a node sees, and which nodes see a key.
//
// The batch is packed: node i belongs to the sequence b with offsets[b] <= i < offsets[b + 1] (a shape's nodes of a
// level, in Morton order).  It sees key j of its own sequence when
//     causal:      j <= i  and  (i - j < window  or  j - start < sinks)
//     both ways:   |i - j| < window  or  j - start < sinks
// and the mask (if any) keeps j.  So a node's keys are a window [lo, hi) and the sequence's first nodes
// [start, first); seen from a key, its nodes are an interval too, and, for a first node, those far behind it.
#pragma once

#include <climits>
#include <type_traits>

#include "common.cuh"

namespace ocnn {

constexpr int kMaxSequences = 1 << 24;         // (the search in steps of 32 stays below 2^31)
constexpr int kMaxSinks = 64;                 // first nodes that stay visible: "a few" (the far pass keeps their sums)
constexpr int kMaxHeadDim = 128;

// The operands as the kernels take them; strides in elements.
struct AttnArgs {
  const void *q, *k, *v;
  long long q_row, q_head, k_row, k_head, v_row, v_head;
  const int* offsets;
  const unsigned char* mask;                  // of keys, or NULL
  int batch, n, heads, kv_heads, dim, window, sinks, causal;
  float scale_log2;                           // scale * log2(e): scores are kept in powers of two
  float scale;
};

// What the backward pass has besides.  out, dq, dk, dv: contiguous; lse (in powers of two, +inf for a row that sees
// nothing) and delta: [heads][n].
// Behind lse, of 16-bit data: what rounding took from out, [n][heads][dim] in the data's type.  delta = dO . o enters every ds,
// and formed from the rounded o it was, at windows of 16, the larger part of the gradients' error (1.6 times that of results
// that are only rounded once; with the rest added back 1.45).
__host__ __device__ inline size_t attn_lse_floats(const AttnArgs& a) { return ((size_t)a.heads * a.n + 31) / 32 * 32; }
template <typename T>
__host__ __device__ inline T* attn_rest(const AttnArgs& a, const float* lse) {
  return lse == nullptr || sizeof(T) == 4 ? nullptr : (T*)(const_cast<float*>(lse) + attn_lse_floats(a));
}

struct AttnGrad {
  const void *out, *grad;
  long long grad_row, grad_head;
  const float* lse;
  float *delta, *far;
  unsigned* largest;                          // float16: per 256 nodes the largest |dO| (its bits), by the queries' kernel
  void *dq, *dk, *dv;                         // dk and dv NULL: not asked for
};

// float16 holds nothing below 2^-24, and p of a long sequence and dO of a mean loss are small: the operands of the gradients'
// second products are kept at powers of two, which the results are divided by.  p: at 2^10 p.  ds: at the power that
// brings the largest |dO| to 8 .. 16 (a sum of 128 products with values of up to 32 stays in range), for dq the row's own, for
// a tile of keys the largest of the nodes that see it, by chunks of 256 nodes.
constexpr float kProbUp = 1024.f, kProbUpLog = 10.f;
constexpr int kChunkLog = 8;
__device__ __forceinline__ float grad_scale(float largest) {       // 8 * 2^-e for 2^e <= largest < 2^(e + 1)
  if (!(largest > 0.f)) return 1.f;
  const int e = min(max((int)(__float_as_uint(largest) >> 23) - 127, -100), 100);
  return __uint_as_float((unsigned)(127 + 3 - e) << 23);
}
inline int grad_chunks(int n) { return ceil_div(n, 1 << kChunkLog); }
// The scale for rows [lo, hi), by a whole warp.
__device__ __forceinline__ float grad_scale_of(const unsigned* largest, int lo, int hi) {
  unsigned most = 0;
  for (int c = (lo >> kChunkLog) + (threadIdx.x & 31); c <= (hi - 1) >> kChunkLog; c += 32) most = max(most, largest[c]);
  return grad_scale(__uint_as_float(__reduce_max_sync(0xffffffffu, most)));
}

// Heads of a node that stand side by side in a tensor-core tile: the largest power of two in the group.
inline int attn_pack_log(const AttnArgs& a) {
  const int group = a.heads / a.kv_heads;
  int log = 0;
  while (log < 5 && (group >> log) % 2 == 0) ++log;
  return log;
}

int attn_tc_forward(const AttnArgs& a, int dtype, void* out, float* lse, int* status, cudaStream_t st);
int attn_tc_backward(const AttnArgs& a, const AttnGrad& g, int dtype, int* status, cudaStream_t st);
int attn_far_mma(const AttnArgs& a, const AttnGrad& g, int dtype, cudaStream_t st);   // 16-bit rows on 16-byte boundaries
int attn_simt_forward(const AttnArgs& a, int dtype, void* out, float* lse, bool vec, cudaStream_t st);
int attn_simt_backward(const AttnArgs& a, const AttnGrad& g, int dtype, bool vec, cudaStream_t st);

// Sequence of node i: [start, end), empty for a node outside of every sequence.  Offsets are clamped to [0, n], so
// that no offset makes a kernel leave its tensors.
struct Span { int start, end, seq; };
__device__ __forceinline__ int attn_offset(const AttnArgs& a, int b) { return min(max(a.offsets[b], 0), a.n); }
__device__ __forceinline__ Span attn_span(const AttnArgs& a, int i) {
  int lo = 0, hi = a.batch;                   // the last b with offsets[b] <= i
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (attn_offset(a, mid) <= i) lo = mid;
    else hi = mid - 1;
  }
  Span s = {0, 0, lo};
  if (i >= a.n || lo >= a.batch) return s;
  const int start = attn_offset(a, lo), end = attn_offset(a, lo + 1);
  if (i < start || i >= end) return s;
  s.start = start;
  s.end = end;
  return s;
}

// The same by whole warps, for several nodes: a warp reads the offsets once, a lane each (a search node by node is a chain of
// loads); of more than 32 it keeps every step-th and looks at 32 at a time from there.
struct WarpOffsets {
  int mine, step;                                        // offset of sequence lane * step, clamped
  __device__ __forceinline__ explicit WarpOffsets(const AttnArgs& a) {
    step = 1;
    while (step * 32 < a.batch + 1) step *= 32;
    const int b = (threadIdx.x & 31) * step;
    mine = b <= a.batch ? attn_offset(a, b) : INT_MAX;
  }
  __device__ __forceinline__ int begin() const { return __shfl_sync(0xffffffffu, mine, 0); }
  __device__ __forceinline__ int end(const AttnArgs& a) const {
    return step == 1 ? __shfl_sync(0xffffffffu, mine, a.batch) : attn_offset(a, a.batch);
  }
  __device__ __forceinline__ Span span(const AttnArgs& a, int i) const {
    unsigned under = __ballot_sync(0xffffffffu, mine <= i);
    int last = under == 0 ? 0 : (31 - __clz(under)) * step;
    for (int s = step / 32; s >= 1; s /= 32) {
      const int b = last + (threadIdx.x & 31) * s;
      under = __ballot_sync(0xffffffffu, b <= a.batch && attn_offset(a, min(b, a.batch)) <= i);
      last = under == 0 ? last : last + (31 - __clz(under)) * s;
    }
    Span s = {0, 0, last};
    if (i >= a.n || last >= a.batch) return s;
    const int start = step == 1 ? __shfl_sync(0xffffffffu, mine, last) : attn_offset(a, last);
    const int end = step == 1 ? __shfl_sync(0xffffffffu, mine, last + 1) : attn_offset(a, last + 1);
    if (i < start || i >= end) return s;
    s.start = start;
    s.end = end;
    return s;
  }
};
// Node i's, where the nodes of a tile are known to lie between those of spans f and l.
__device__ __forceinline__ Span attn_span_near(const AttnArgs& a, int i, const Span& f, const Span& l) {
  if (i >= f.start && i < f.end) return f;
  if (i >= l.start && i < l.end) return l;
  return attn_span(a, i);
}

// What node i sees: [lo, hi) and [start, first).
struct RowKeys { int lo, hi, start, first; };
__device__ __forceinline__ RowKeys attn_row_keys(const AttnArgs& a, int i, const Span& s) {
  RowKeys r = {0, 0, 0, 0};
  if (s.end <= s.start) return r;
  r.lo = max(s.start, i - a.window + 1);
  r.hi = a.causal ? i + 1 : i + min(s.end - i, a.window);
  r.start = s.start;
  r.first = s.start + min(a.sinks, (a.causal ? i + 1 : s.end) - s.start);
  return r;
}
__device__ __forceinline__ bool attn_sees(const RowKeys& r, int j) {
  return (j >= r.lo && j < r.hi) || (j >= r.start && j < r.first);
}

// The nodes that see key j from within the window: [lo, hi).  A first node is seen by every node before it too (both
// ways); the nodes from j + window on, which see it as a first node only, are left to the far pass.
struct KeyRows { int lo, hi; };
__device__ __forceinline__ KeyRows attn_rows_of_key(const AttnArgs& a, int j, const Span& s) {
  KeyRows r = {0, 0};
  if (s.end <= s.start) return r;
  r.lo = a.causal ? j : (j - s.start < a.sinks ? s.start : max(s.start, j - a.window + 1));
  r.hi = j + min(s.end - j, a.window);
  return r;
}
__device__ __forceinline__ KeyRows attn_key_rows(const AttnArgs& a, int j, const Span& s) {
  return a.mask != nullptr && a.mask[j] == 0 ? KeyRows{0, 0} : attn_rows_of_key(a, j, s);
}

// The keys that the nodes [r0, r1) see between them: the first nodes of r0's sequence where they lie before the windows,
// then one interval.  (Only r0's: the first nodes of a sequence that starts behind r0 lie in the interval.)
struct TileKeys {
  int first, n_first;                         // [first, first + n_first)
  int lo, n;                                  // then [lo, lo + n - n_first); n keys in all
  __device__ __forceinline__ int key(int t) const { return t < n_first ? first + t : lo + (t - n_first); }
};

template <typename T>
__device__ __forceinline__ float to_f32(T x) { return (float)x; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x) { return (T)x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16(x); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half(x); }

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two fp32 values per instruction (sm_100).
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

__device__ __forceinline__ bool not_finite(float x) { return !(fabsf(x) <= 3.402823466e38f); }

template <typename T>
__device__ __forceinline__ float rounded_off(float x) {
  const float r = x - to_f32(from_f32<T>(x));
  return not_finite(r) ? 0.f : r;
}

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) x += __shfl_xor_sync(0xffffffffu, x, m);
  return x;
}

// ---- rows key by key ----------------------------------------------------------------------------------------
// A tile multiplies a hidden pair's probability, 0, by whatever the hidden value is: 0 x inf is not 0.  A row whose
// result is not finite is therefore formed once more by its warp, from the keys that it sees only (where one of those
// is not finite the result is none either, however small its probability).  A row without a visible key is zeros; one whose
// visible scores are all -inf has no softmax: NaN.
//
// That is slow, a pair at a time, and a training step that overflows has such rows everywhere.  So it is done only where a
// hidden value can have been the cause: not where the row's statistics are no numbers themselves (every channel is none then),
// nor where every spoilt channel of the result has a visible value that spoils it.  Forward and gradients of 65 k nodes, 16 heads
// of 128, windows of 1024, float16: 3.7 ms, with dO all inf 4.6, not 1300; with one value of dO inf, which 200 keys around its
// window have beside them hidden, 49.
//
// The calling lane's channels (lane + 32 c) of a row that are no numbers, a bit each.
template <typename T>
__device__ __forceinline__ unsigned spoilt_channels(const T* row, int dim) {
  unsigned bits = 0;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int d = (threadIdx.x & 31) + 32 * c;
    if (d < dim && not_finite(to_f32(row[d]))) bits |= 1u << c;
  }
  return bits;
}
// Whether visible values account for every spoilt channel of row i's result, `out` as its tile left it.
template <typename T>
__device__ bool attn_row_is_spoilt(const AttnArgs& a, int i, int h, const T* out) {
  const RowKeys r = attn_row_keys(a, i, attn_span(a, i));
  const int hk = h / (a.heads / a.kv_heads);
  unsigned open = spoilt_channels(out + ((long long)i * a.heads + h) * a.dim, a.dim);
  const int n_first = max(0, min(r.first, r.lo) - r.start), behind = max(r.hi, r.first);
  for (int t = 0; t < n_first + behind - r.lo; ++t) {
    const int j = t < n_first ? r.start + t : r.lo + t - n_first;
    if (!attn_sees(r, j) || (a.mask != nullptr && a.mask[j] == 0)) continue;
    open &= ~spoilt_channels((const T*)a.v + j * a.v_row + hk * a.v_head, a.dim);
    if (!__any_sync(0xffffffffu, open != 0)) return true;
  }
  return false;
}
template <typename T>
__device__ void attn_forward_row(const AttnArgs& a, int i, int h, T* out, float* lse) {
  const int lane = threadIdx.x & 31;
  const RowKeys r = attn_row_keys(a, i, attn_span(a, i));
  const int hk = h / (a.heads / a.kv_heads);
  const T* q = (const T*)a.q + i * a.q_row + h * a.q_head;
  float qv[4], acc[4] = {};
#pragma unroll
  for (int c = 0; c < 4; ++c) qv[c] = lane + 32 * c < a.dim ? to_f32(q[lane + 32 * c]) : 0.f;
  float top = -INFINITY, total = 0.f;
  bool sees = false;
  const int n_first = max(0, min(r.first, r.lo) - r.start), behind = max(r.hi, r.first);
  for (int t = 0; t < n_first + behind - r.lo; ++t) {
    const int j = t < n_first ? r.start + t : r.lo + t - n_first;
    if (!attn_sees(r, j) || (a.mask != nullptr && a.mask[j] == 0)) continue;
    sees = true;
    const T* k = (const T*)a.k + j * a.k_row + hk * a.k_head;
    const T* v = (const T*)a.v + j * a.v_row + hk * a.v_head;
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (lane + 32 * c < a.dim) s += qv[c] * to_f32(k[lane + 32 * c]);
    s = warp_sum(s) * a.scale_log2;
    const float last = top;
    // (fmaxf passes a NaN score by, the exponential does not: it stays in the sum whatever the maximum is)
    top = fmaxf(top, s);
    const float base = top == -INFINITY ? 0.f : top, keep = exp2f(last - base), p = exp2f(s - base);
    total = total * keep + p;
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (lane + 32 * c < a.dim) acc[c] = acc[c] * keep + p * to_f32(v[lane + 32 * c]);
  }
  if (sees && total == 0.f) total = NAN;
  T* rest = attn_rest<T>(a, lse);
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (lane + 32 * c < a.dim) {
      const long long at = ((long long)i * a.heads + h) * a.dim + lane + 32 * c;
      const float x = sees ? acc[c] / total : 0.f;
      out[at] = from_f32<T>(x);
      if (rest != nullptr) rest[at] = from_f32<T>(rounded_off<T>(x));
    }
  if (lse != nullptr && lane == 0)
    lse[(long long)h * a.n + i] = sees ? top + log2f(total) : INFINITY;
}

// Gradient of query i of head h from the keys that it sees, and of key j from the queries that see it: as
// attn_forward_row, for rows whose result in a tile is not finite.  Not for a query whose statistics are no numbers while it
// sees something (lse is +inf where it does not): its dq is none in any channel.
__device__ __forceinline__ bool attn_query_is_spoilt(float lse, float delta) {
  return lse != INFINITY && (not_finite(lse) || not_finite(delta));
}
template <typename T>
__device__ __forceinline__ void attn_row(const void* base, long long at, int dim, float (&x)[4]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int c = 0; c < 4; ++c) x[c] = lane + 32 * c < dim ? to_f32(((const T*)base)[at + lane + 32 * c]) : 0.f;
}
__device__ __forceinline__ float attn_dot(const float (&x)[4], const float (&y)[4]) {
  return warp_sum(x[0] * y[0] + x[1] * y[1] + x[2] * y[2] + x[3] * y[3]);
}
template <typename T>
__device__ void attn_dq_row(const AttnArgs& a, const AttnGrad& g, int i, int h) {
  const int lane = threadIdx.x & 31, hk = h / (a.heads / a.kv_heads);
  const RowKeys r = attn_row_keys(a, i, attn_span(a, i));
  const float lse = g.lse[(long long)h * a.n + i], delta = g.delta[(long long)h * a.n + i];
  float q[4], go[4], acc[4] = {};
  attn_row<T>(a.q, i * a.q_row + h * a.q_head, a.dim, q);
  attn_row<T>(g.grad, i * g.grad_row + h * g.grad_head, a.dim, go);
  const int n_first = max(0, min(r.first, r.lo) - r.start), behind = max(r.hi, r.first);
  for (int t = 0; t < n_first + behind - r.lo; ++t) {
    const int j = t < n_first ? r.start + t : r.lo + t - n_first;
    if (!attn_sees(r, j) || (a.mask != nullptr && a.mask[j] == 0)) continue;
    float k[4], v[4];
    attn_row<T>(a.k, j * a.k_row + hk * a.k_head, a.dim, k);
    attn_row<T>(a.v, j * a.v_row + hk * a.v_head, a.dim, v);
    const float p = exp2f(attn_dot(q, k) * a.scale_log2 - lse), ds = p * (attn_dot(go, v) - delta);
#pragma unroll
    for (int c = 0; c < 4; ++c) acc[c] += ds * k[c];
  }
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (lane + 32 * c < a.dim)
      ((T*)g.dq)[((long long)i * a.heads + h) * a.dim + lane + 32 * c] = from_f32<T>(acc[c] * a.scale);
}
// Whether the queries that see key j account for every spoilt channel of its gradient (dv's as the tile left it): one whose
// statistics are no numbers spoils all of dk, and of dv the channels where its dO is none, or all.  (Where dO or a visible value
// is no number, delta is none.)
template <typename T>
__device__ bool attn_key_is_spoilt(const AttnArgs& a, const AttnGrad& g, int j, int hk, bool of_dv) {
  const int lane = threadIdx.x & 31, group = a.heads / a.kv_heads;
  const Span s = attn_span(a, j);
  const KeyRows r = attn_key_rows(a, j, s);
  const int end = r.hi > r.lo && j - s.start < a.sinks ? s.end : r.hi;
  unsigned open = of_dv ? spoilt_channels((const T*)g.dv + ((long long)j * a.kv_heads + hk) * a.dim, a.dim) : 0;
  for (int h = hk * group; h < (hk + 1) * group; ++h) {
    for (int i0 = r.lo; i0 < end; i0 += 32) {
      const bool in = i0 + lane < end;
      const float lse = in ? g.lse[(long long)h * a.n + i0 + lane] : 0.f, delta = in ? g.delta[(long long)h * a.n + i0 + lane] : 0.f;
      unsigned rows = __ballot_sync(0xffffffffu, not_finite(lse) || not_finite(delta));
      if (rows != 0 && (!of_dv || __any_sync(0xffffffffu, not_finite(lse)))) return true;
      for (; rows != 0; rows &= rows - 1) {
        const int i = i0 + __ffs(rows) - 1;
        open &= ~spoilt_channels((const T*)g.grad + i * g.grad_row + h * g.grad_head, a.dim);
        if (!__any_sync(0xffffffffu, open != 0)) return true;
      }
    }
  }
  return false;
}
template <typename T>
__device__ void attn_dkv_row(const AttnArgs& a, const AttnGrad& g, int j, int hk, bool write_dk, bool write_dv) {
  const int lane = threadIdx.x & 31, group = a.heads / a.kv_heads;
  const Span s = attn_span(a, j);
  const KeyRows r = attn_key_rows(a, j, s);
  const int end = r.hi > r.lo && j - s.start < a.sinks ? s.end : r.hi;        // (a first node: to the sequence's end)
  float k[4], v[4], dk[4] = {}, dv[4] = {};
  attn_row<T>(a.k, j * a.k_row + hk * a.k_head, a.dim, k);
  attn_row<T>(a.v, j * a.v_row + hk * a.v_head, a.dim, v);
  for (int h = hk * group; h < (hk + 1) * group; ++h) {
    for (int i = r.lo; i < end; ++i) {
      float q[4], go[4];
      attn_row<T>(a.q, i * a.q_row + h * a.q_head, a.dim, q);
      attn_row<T>(g.grad, i * g.grad_row + h * g.grad_head, a.dim, go);
      const float p = exp2f(attn_dot(q, k) * a.scale_log2 - g.lse[(long long)h * a.n + i]);
      if (write_dk) {
        const float ds = p * (attn_dot(go, v) - g.delta[(long long)h * a.n + i]);
#pragma unroll
        for (int c = 0; c < 4; ++c) dk[c] += ds * q[c];
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) dv[c] += p * go[c];
    }
  }
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const long long at = ((long long)j * a.kv_heads + hk) * a.dim + lane + 32 * c;
    if (lane + 32 * c >= a.dim) continue;
    if (write_dk) ((T*)g.dk)[at] = from_f32<T>(dk[c] * a.scale);
    if (write_dv) ((T*)g.dv)[at] = from_f32<T>(dv[c]);
  }
}

// ---- first nodes seen from far behind -----------------------------------------------------------------------
// What the nodes behind the window add to the gradients of their sequence's first nodes comes from all over the
// sequence.  It is summed in blocks of kFarRows nodes, each block's share of a sequence in a slot of its own, and the
// slots are added up in order: no atomics, the same bits every time.  Slot = block + the sequence's number: along the packed
// batch either the block or the sequence moves on, so no two pairs share one.  Only sequences longer than the window have
// anything from far: where there cannot be as many as the batch holds, start / (window + 1) numbers them instead, which is another
// one for each (10^5 short sequences of 10 nodes under a window of 1000: 4905 slots, not 103907).
constexpr int kFarRows = 256;
__host__ __device__ inline bool far_by_start(const AttnArgs& a) { return a.batch > a.n / (a.window + 1) + 1; }
inline int far_slots(const AttnArgs& a) {
  return ceil_div(a.n, kFarRows) + (far_by_start(a) ? a.n / (a.window + 1) + 1 : a.batch);
}
__device__ __forceinline__ int far_number(const AttnArgs& a, const Span& s) {
  return far_by_start(a) ? s.start / (a.window + 1) : s.seq;
}
__device__ __forceinline__ float* far_slot(const AttnArgs& a, const AttnGrad& g, int slot, int hk, int sink) {
  return g.far + (((long long)slot * a.kv_heads + hk) * a.sinks + sink) * (2 * a.dim);
}
// Key j's slots: the first one's number, and how many there are (0: nobody sees it from far).  A kernel of their own adds
// them up into the first, which the gradients' kernel reads.
struct FarSlots { int first, count; };
__device__ __forceinline__ FarSlots far_slots_of(const AttnArgs& a, int j, const Span& s) {
  if (j - s.start >= a.sinks || s.end - j <= a.window || (a.mask != nullptr && a.mask[j] == 0)) return {0, 0};
  const int first = (j + a.window) / kFarRows;
  return {first + far_number(a, s), (s.end - 1) / kFarRows - first + 1};
}
// The sums of dK's channels for key j, then of dV's; NULL where nobody sees it from far.
__device__ __forceinline__ const float* far_sums(const AttnArgs& a, const AttnGrad& g, int j, int hk) {
  if (a.sinks == 0) return nullptr;
  const Span s = attn_span(a, j);
  const FarSlots f = far_slots_of(a, j, s);
  return f.count > 0 ? far_slot(a, g, f.first, hk, j - s.start) : nullptr;
}
int attn_far_join(const AttnArgs& a, const AttnGrad& g, cudaStream_t st);

}  // namespace ocnn
