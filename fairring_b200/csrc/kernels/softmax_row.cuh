// One sweep over a row of logits: its maximum m, S = sum of exp((x - m) / T) and, where the entropy is wanted,
// A = sum of exp((x - m) / T) * log2(exp((x - m) / T)).  Shared by the kernels that ask a language-model head's
// logits for probabilities.
//
// A row is the elements up to its first 16-byte boundary, 16-byte vectors, and what is left behind them.  Few rows are taken by a
// block each or, fewer still, by the blocks of a cluster, a slice each, of which the first merges what they found, in the
// order of the slices; many by blocks that stay and take row after row; many short ones by a warp each.  Which it is depends on
// the sizes alone, and so does the order of every sum.
//
// What bounds it: the bytes, and next to them the exponentials (16 a clock and multiprocessor: 9
// TB/s of bf16 logits) and the instructions around them.  8192 rows of 51200 bf16 logits: 132 us,
// 6.4 TB/s; 61 instructions of a warp for 32 vectors of 8, of them 9 for the special function unit,
// 23 for the multiply-add pipe, 18 integer and comparisons, 4 loads and stores; 60 % of the issue
// slots.  fp32 logits need half of that a byte: 2046 rows of 50265 in 70 us, 5.9 TB/s, 6 us above
// the copy rate.  So the instructions are kept few: no comparison of the maximum a value but one a
// batch, in the logits' own type; two fp32 operations in one instruction (157 us at the time, 164
// without); no test for what masked rows need.  A polynomial in place of some exponentials costs
// more issue slots than it frees (157 -> 178).
//
// exp() is 2^((x - m) * c) with c = log2(e) / T, as one fused multiply-add of x, c and the rounded
// m * c; what that rounding changes all exponentials by is put right at the row's end.  The
// exponential's own error is 2^-22 of a probability.  That form needs |m * c| < 2^20.  A thread's m
// starts at -2^20 / c.  A row whose largest value is above has a sum of 1 or more, but for
// roundings.  One whose largest value is below (masked with the type's lowest value or with minus
// infinity throughout, say) has lost its smaller values to zero, and all of them from 126 / c below
// on: its sum is smaller than 1/2 unless it has lost nothing that fp32 sees, and it is looked at
// again, slowly, as are rows above that range and those with a NaN.
#pragma once

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <map>
#include <mutex>
#include <utility>

#include "local_kernels.h"

namespace fairring {
namespace softmax_row {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kBatch = 4;        // 16-byte vectors in flight per thread
constexpr int kMostSlices = 8;   // blocks of a cluster: what every device grants
constexpr unsigned kAll = 0xffffffffu;
constexpr float kLn2 = 0.693147180559945309f;
// exp2() of it is zero, and times it still is: in place of minus infinity where the exponent is a factor.
constexpr float kLowExponent = -256.f;
constexpr float kPlainRange = 1048576.f;

template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int kElems = 4;
  static constexpr uint32_t kMinusInf = 0xff800000u;
  static __device__ __forceinline__ void get(const uint4& r, float2 (&v)[2]) {
    v[0] = make_float2(__uint_as_float(r.x), __uint_as_float(r.y));
    v[1] = make_float2(__uint_as_float(r.z), __uint_as_float(r.w));
  }
  static __device__ __forceinline__ uint4 set(const float2 (&v)[2]) {
    return make_uint4(__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x), __float_as_uint(v[1].y));
  }
  static __device__ __forceinline__ float max(const uint4& r) {
    return fmaxf(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)), fmaxf(__uint_as_float(r.z), __uint_as_float(r.w)));
  }
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int kElems = 8;
  static constexpr uint32_t kMinusInf = 0xff80ff80u;
  static __device__ __forceinline__ void get(const uint4& r, float2 (&v)[4]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
  }
  static __device__ __forceinline__ uint4 set(const float2 (&v)[4]) {
    uint4 r;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[i].x, v[i].y);
    return r;
  }
  static __device__ __forceinline__ float max(const uint4& r) {  // packed: half the comparisons
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&r);
    const float2 m = __bfloat1622float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
    return fmaxf(m.x, m.y);
  }
};
template <> struct Vec<__half> {
  static constexpr int kElems = 8;
  static constexpr uint32_t kMinusInf = 0xfc00fc00u;
  static __device__ __forceinline__ void get(const uint4& r, float2 (&v)[4]) {
    const __half2* h = reinterpret_cast<const __half2*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __half22float2(h[i]);
  }
  static __device__ __forceinline__ uint4 set(const float2 (&v)[4]) {
    uint4 r;
    __half2* h = reinterpret_cast<__half2*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(v[i].x, v[i].y);
    return r;
  }
  static __device__ __forceinline__ float max(const uint4& r) {
    const __half2* h = reinterpret_cast<const __half2*>(&r);
    const float2 m = __half22float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
    return fmaxf(m.x, m.y);
  }
};

// The largest of a batch, compared in the type that the values have.
template <typename T> __device__ __forceinline__ float batchMax(const uint4 (&now)[kBatch]) {
  float top = Vec<T>::max(now[0]);
  for (int u = 1; u < kBatch; ++u) top = fmaxf(top, Vec<T>::max(now[u]));
  return top;
}

__device__ __forceinline__ float toFloat(float v) { return v; }
__device__ __forceinline__ float toFloat(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float toFloat(__half v) { return __half2float(v); }
__device__ __forceinline__ void fromFloat(float* p, float v) { *p = v; }
__device__ __forceinline__ void fromFloat(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void fromFloat(__half* p, float v) { *p = __float2half_rn(v); }

// 2^v; results below the smallest normal number are zero.
__device__ __forceinline__ float exp2Of(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ uint64_t packed(float2 v) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(v.x), "f"(v.y));
  return r;
}
__device__ __forceinline__ float2 unpacked(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(packed(a)), "l"(packed(b)));
  return unpacked(r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(packed(a)), "l"(packed(b)));
  return unpacked(r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(packed(a)), "l"(packed(b)), "l"(packed(c)));
  return unpacked(r);
}

template <typename T> __device__ __forceinline__ T* rowOf(const LogitRows& x, T* data, int64_t r) {
  const int64_t outer = x.inner == x.rows ? 0 : r / x.inner;
  return data + outer * x.outer_stride + (r - outer * x.inner) * x.row_stride;
}

// A row: `head` elements, `nvec` aligned 16-byte vectors, `tail` elements.
template <typename T> struct RowParts {
  int head, nvec, tail;
  __device__ __forceinline__ RowParts(const T* row, int vocab) {
    constexpr int E = Vec<T>::kElems;
    const int off = (int)(reinterpret_cast<uintptr_t>(row) & 15u) / (int)sizeof(T);
    head = min(vocab, (E - off) % E);
    nvec = (vocab - head) / E;
    tail = vocab - head - nvec * E;
  }
};

// Slice `rank` of `slices` of a row: vectors [v0, v1), which with the row's head and tail are the columns [c0, c1).
template <typename T> struct Slice {
  const T* row;
  int head, v0, v1, c0, c1;
  __device__ __forceinline__ Slice(const T* row_, int vocab, int rank, int slices) : row(row_) {
    constexpr int E = Vec<T>::kElems;
    const RowParts<T> parts(row, vocab);
    head = parts.head;
    const int each = (parts.nvec + slices - 1) / slices;
    v0 = min(parts.nvec, rank * each);
    v1 = min(parts.nvec, v0 + each);
    c0 = rank == 0 ? 0 : head + v0 * E;
    c1 = rank == slices - 1 ? vocab : head + v1 * E;
  }
  __device__ __forceinline__ int firstCol() const { return head + v0 * Vec<T>::kElems; }
  __device__ __forceinline__ int lastCol() const { return head + v1 * Vec<T>::kElems; }
  // The columns before and behind the vectors, fewer than 2 * kElems of them; -1 past the last.
  __device__ __forceinline__ int looseCol(int i) const {
    const int before = firstCol() - c0;
    const int col = i < before ? c0 + i : lastCol() + i - before;
    return col < c1 ? col : -1;
  }
};

// m * c, rounded wherever it stands: never a part of a fused multiply-add.
__device__ __forceinline__ float scaled(float m, float c) { return __fmul_rn(m, c); }

// The sums of a row or a part of it, while it is swept relative to the rounded m * c, in the end to m itself.
struct Sums {
  float m, s, a;
  // Makes them 2^d times what they are, which raises every exponent by d.
  template <bool kEntropy> __device__ __forceinline__ void shift(float d) {
    const float f = exp2Of(d);
    if (kEntropy) a = f * fmaf(fmaxf(d, kLowExponent), s, a);
    s *= f;
  }
  static __device__ __forceinline__ Sums none(float c) { return {-kPlainRange / c, 0.f, 0.f}; }
  template <bool kEntropy> __device__ __forceinline__ void merge(Sums o, float c) {
    const float top = fmaxf(m, o.m), at = scaled(top, c);
    shift<kEntropy>(scaled(m, c) - at);
    o.template shift<kEntropy>(scaled(o.m, c) - at);
    m = top;
    s += o.s;
    if (kEntropy) a += o.a;
  }
  template <bool kEntropy> __device__ __forceinline__ void add(float v, float c) {
    const float top = fmaxf(m, v), at = scaled(top, c), d = fmaf(v, c, -at), e = exp2Of(d);
    shift<kEntropy>(scaled(m, c) - at);
    m = top;
    s += e;
    if (kEntropy) a = fmaf(e, fmaxf(d, kLowExponent), a);
  }
  // Relative to m; false for a row that has to be looked at again.
  template <bool kEntropy> __device__ __forceinline__ bool settle(float c) {
    shift<kEntropy>(-fmaf(m, c, -scaled(m, c)));
    return scaled(m, c) < kPlainRange && s >= 0.5f && s < INFINITY;
  }
};

// A thread's share of a row, from the first of its vectors on.  A batch is summed by itself and
// then added: a sum of V logits is 16 + V / 4096 additions long at most in place of V / 512, each
// 2^-24 off.  Rows of 2^20 equal logits but for one a thread came out 3e-5 off and are now 1e-6;
// 8192 x 51200 bf16 takes 132 us either way.  The running sums are single numbers, since pairs
// spilled registers where the entropy and largest entries are asked for (191 -> 203 us).
struct ThreadSums {
  float m, at;  // at = m * c
  float s, a;
  __device__ __forceinline__ explicit ThreadSums(float c) : m(-kPlainRange / c), at(scaled(m, c)), s(0.f), a(0.f) {}
  // Adds the first n vectors of a batch whose largest value is `top`; all lanes of a warp have the same n.
  template <typename T, bool kEntropy, bool kWhole>
  __device__ __forceinline__ void add(const uint4 (&now)[kBatch], float top, int n, float c) {
    constexpr int E = Vec<T>::kElems;
    if (!kWhole && n <= 0) return;
    m = fmaxf(m, top);
    const float before = at;
    at = scaled(m, c);
    const float d = before - at, f = exp2Of(d);
    if (kEntropy) a = f * fmaf(fmaxf(d, kLowExponent), s, a);
    s *= f;
    float2 bs, ba;  // the batch's own
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (!kWhole && u > 0 && u >= n) break;
      float2 v[E / 2];
      Vec<T>::get(now[u], v);
#pragma unroll
      for (int k = 0; k < E / 2; ++k) {
        const float2 d = fma2(v[k], make_float2(c, c), make_float2(-at, -at));
        const float2 e = make_float2(exp2Of(d.x), exp2Of(d.y));
        bs = u == 0 && k == 0 ? e : add2(bs, e);
        if (kEntropy) {
          const float2 low = make_float2(fmaxf(d.x, kLowExponent), fmaxf(d.y, kLowExponent));
          ba = u == 0 && k == 0 ? mul2(e, low) : fma2(e, low, ba);
        }
      }
    }
    if (kEntropy) a += ba.x + ba.y;
    s += bs.x + bs.y;
  }
  __device__ __forceinline__ Sums sums() const { return {m, s, a}; }
};

// (x - m) * c of two values, for the backward kernels, too large by excess(m, c).
struct Exponent {
  float scale, minus, shift;
  static __device__ __forceinline__ float excess(float m, float c) {
    const float at = __fmul_rn(m, c);
    return fabsf(at) < kPlainRange ? fmaf(m, c, -at) : 0.f;
  }
  __device__ __forceinline__ Exponent(float m, float c) {
    const float at = __fmul_rn(m, c);
    const bool plain = fabsf(at) < kPlainRange;  // else the difference is taken first, and its product is exact enough
    minus = plain ? 0.f : -m;
    scale = c;
    shift = plain ? -at : 0.f;
  }
  __device__ __forceinline__ float2 operator()(float2 v) const {
    return fma2(add2(v, make_float2(minus, minus)), make_float2(scale, scale), make_float2(shift, shift));
  }
};

// A barrier of a warp or a block.
template <int kWidth> __device__ __forceinline__ void syncWidth() {
  if constexpr (kWidth == 32)
    __syncwarp();
  else
    __syncthreads();
}

// Backward: rows in pieces of kBatch vectors for each of a warp's threads, numbered through all rows.  The numbers are of 32
// bits, since a division of 64 takes as long as a vector: 2^31 rows, and 2 KB of logits to each piece past a row's first.
struct Pieces {
  unsigned total, a_row;
  // False if there are too many.
  template <typename T> bool cut(const LogitRows& x) {
    constexpr int per_piece = 32 * kBatch * Vec<T>::kElems;
    const int64_t each = ((int64_t)x.vocab + per_piece - 1) / per_piece;
    if (each > (int64_t)(UINT32_MAX - kThreads) / x.rows) return false;
    a_row = (unsigned)each;
    total = (unsigned)(x.rows * each);
    return true;
  }
  unsigned blocks() const { return (total + kWarps - 1) / kWarps; }
  static __device__ __forceinline__ unsigned mine() { return blockIdx.x * kWarps + threadIdx.x / 32; }
};

// What a kernel does with a batch, that from vector i on, before it is summed; returns its largest value.
// kUnroll: the batches that a turn of the loop takes.
struct NoHook {
  static constexpr int kUnroll = 1;
  template <typename P> __device__ __forceinline__ void begin(const P&) {}
  __device__ __forceinline__ void end() {}
  __device__ __forceinline__ void arrived(uint4*, int) {}
  template <typename T> __device__ __forceinline__ float batch(uint4 (&now)[kBatch], bool, int, const Slice<T>&) {
    return batchMax<T>(now);
  }
};

// This thread's share of the slice, by kWidth threads that all go through the same number of batches.  The next batch is on its
// way while this one is used.
template <typename T, bool kEntropy, int kWidth, class Hook>
__device__ __forceinline__ Sums scan(const Slice<T>& sl, float c, Hook& hook) {
  constexpr int U = kBatch;
  constexpr uint32_t w = Vec<T>::kMinusInf;
  const uint4* vecs = reinterpret_cast<const uint4*>(sl.row + sl.head);
  const int whole = (sl.v1 - sl.v0) / (U * kWidth), left = sl.v1 - sl.v0 - whole * (U * kWidth);
  int i = sl.v0 + (int)threadIdx.x % kWidth;
  uint4 raw[U], now[U];
  auto fetch = [&](int b) {
    if (b < whole) {
#pragma unroll
      for (int u = 0; u < U; ++u) raw[u] = __ldg(vecs + i + u * kWidth);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
        raw[u] = i + u * kWidth < sl.v1 ? __ldg(vecs + i + u * kWidth) : make_uint4(w, w, w, w);
    }
  };
  ThreadSums acc(c);
  if (whole > 0 || left > 0) fetch(0);
#pragma unroll Hook::kUnroll
  for (int b = 0; b < whole; ++b) {
#pragma unroll
    for (int u = 0; u < U; ++u) now[u] = raw[u];
    i += U * kWidth;
    if (b + 1 < whole || left > 0) fetch(b + 1);
    acc.add<T, kEntropy, true>(now, hook.batch(now, b == 0, i - U * kWidth, sl), U, c);
  }
  if (left > 0)
    acc.add<T, kEntropy, false>(raw, hook.batch(raw, whole == 0, i, sl), (sl.v1 - (i - (int)(threadIdx.x & 31)) + kWidth - 1) / kWidth, c);
  return acc.sums();
}

// Two sweeps over a row for what the fast one cannot do, by `warps` warps: the largest value, and this
// lane's share of the sums, relative to it.  A warp takes 1024 columns at once, of which a lane has every
// 32nd; leave.of(base), by all lanes, has a bit for each of the lane's that is to be left out.  Summed
// in 64 bits: a warp that does a whole row of 2^20 logits adds 2^15 to each sum.
constexpr unsigned kChunk = 1024;
template <typename T, class Leave, class Take>
__device__ __forceinline__ void eachAgain(const T* row, int vocab, int warp, int warps,
                                          const Leave& leave, Take&& take) {
  for (unsigned base = warp * kChunk; base < (unsigned)vocab; base += warps * kChunk) {
    const unsigned out = leave.of(base);
#pragma unroll 16
    for (unsigned j = 0; j < 32; ++j) {
      const unsigned col = base + 32 * j + (threadIdx.x & 31);
      take(col < (unsigned)vocab && !(out >> j & 1u) ? toFloat(row[col]) : -INFINITY);
    }
  }
}
template <typename T, bool kEntropy, class Leave>
__device__ __noinline__ Sums lookAgain(const T* row, int vocab, int warp, int warps, float c,
                                       float top, Leave leave) {
  const float ref = top == -INFINITY ? 0.f : top;
  double s = 0, a = 0;
  eachAgain(row, vocab, warp, warps, leave, [&](float v) {
    const float d = (v - ref) * c, e = exp2Of(d);
    s += e;
    if (kEntropy) a += e * fmaxf(d, kLowExponent);
  });
  return {top, (float)s, (float)a};
}
template <typename T, class Leave>
__device__ __noinline__ float largestOf(const T* row, int vocab, int warp, int warps, Leave leave) {
  float top = -INFINITY;
  eachAgain(row, vocab, warp, warps, leave, [&](float v) { top = fmaxf(top, v); });
  return top;
}

__device__ __forceinline__ float warpMax(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kAll, v, o));
  return v;
}
template <typename V> __device__ __forceinline__ V warpSum(V v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}

// A warp's sums from its lanes', in every lane.
template <bool kEntropy> __device__ __forceinline__ Sums warpSums(Sums acc, float c) {
  const float m = warpMax(acc.m);
  acc.shift<kEntropy>(scaled(acc.m, c) - scaled(m, c));
  return {m, warpSum(acc.s), kEntropy ? warpSum(acc.a) : 0.f};
}

// The block's sums from those of its first kThreads threads, in every thread; what others bring is not added.  `scratch`: one of
// them a warp, in shared memory.
template <bool kEntropy> __device__ __forceinline__ Sums blockSums(Sums acc, float c, Sums* scratch) {
  acc = warpSums<kEntropy>(acc, c);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = acc;
  __syncthreads();
  acc = scratch[0];
#pragma unroll
  for (int i = 1; i < kWarps; ++i) acc.merge<kEntropy>(scratch[i], c);
  return acc;
}

// A row's sums, relative to m, by a whole block, its first kThreads threads, or a whole warp, where the sweep's did not settle.
template <typename T, bool kEntropy, class Leave>
__device__ __noinline__ Sums blockAgain(const T* row, int vocab, float c, Sums* scratch, Leave leave) {
  const int mine = threadIdx.x < kThreads ? vocab : 0, warp = threadIdx.x >> 5;
  float top = warpMax(largestOf(row, mine, warp, kWarps, leave));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5].m = top;
  __syncthreads();
  for (int i = 0; i < kWarps; ++i) top = fmaxf(top, scratch[i].m);
  Sums acc = lookAgain<T, kEntropy>(row, mine, warp, kWarps, c, top, leave);
  acc.s = warpSum(acc.s);
  acc.a = warpSum(acc.a);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = acc;
  __syncthreads();
  acc.s = acc.a = 0.f;
  for (int i = 0; i < kWarps; ++i) acc.s += scratch[i].s, acc.a += scratch[i].a;
  return acc;
}
template <typename T, bool kEntropy, class Leave>
__device__ __noinline__ Sums warpAgain(const T* row, int vocab, float c, Leave leave) {
  const float top = warpMax(largestOf(row, vocab, 0, 1, leave));
  Sums acc = lookAgain<T, kEntropy>(row, vocab, 0, 1, c, top, leave);
  acc.s = warpSum(acc.s);
  acc.a = warpSum(acc.a);
  return acc;
}
struct LeaveNone {
  __device__ __forceinline__ unsigned of(unsigned) const { return 0; }
};

// The row's sums from those of the slices' blocks, in the threads of block 0.  Every block of the cluster calls
// it, and none leaves before clusterDone().
template <bool kEntropy> __device__ __forceinline__ Sums clusterSums(Sums mine, float c, Sums* shared) {
  namespace cg = cooperative_groups;
  const cg::cluster_group cluster = cg::this_cluster();
  if (threadIdx.x == 0) *shared = mine;
  cluster.sync();
  if (cluster.block_rank() != 0) return mine;
  for (unsigned r = 1; r < cluster.num_blocks(); ++r) mine.merge<kEntropy>(*cluster.map_shared_rank(shared, r), c);
  return mine;
}
__device__ __forceinline__ void clusterDone() { cooperative_groups::this_cluster().sync(); }

// Into how many slices `rows` rows are cut, as a power of two: as many as keep two blocks a multiprocessor busy, but not so many that a
// block's slice is less than half a batch.  Three blocks where the slices stay long: 200 rows of 128003 fp32 logits with the rest
// 38.8 us in one slice each and 29.6 in two, 100 rows 21.6 in two and 17.7 in four; but 48 rows of 51200 bf16 logits with 20 entries
// 11.1 in four and 13.3 in eight, 200 rows of 8192 fp32 logits 5.6 in one and 6.5 in two.
constexpr int kLongSlice = 56 * 1024;  // bytes
inline int slicesFor(int64_t rows, int vocab, int elem_size, int sm_count) {
  const int64_t bytes = (int64_t)vocab * elem_size;
  int n = 1;
  while (n < kMostSlices && rows * n * 2 <= (bytes / (n * 2) >= kLongSlice ? 3 : 2) * (int64_t)sm_count &&
         bytes / 16 / (n * 2) >= kThreads * kBatch / 2)
    n *= 2;
  return n;
}

// The status is the launch's own: cudaGetLastError() would also return, and clear, an error that the host program has pending from
// something else.
inline cudaError_t ownStatus(cudaError_t e) {
  if (e != cudaSuccess) (void)cudaGetLastError();  // reported here, so not once more by whoever asks next
  return e;
}
template <typename... Params, typename... Args>
cudaError_t launchBlocks(void (*kernel)(Params...), unsigned blocks, int threads, int cluster, size_t shared, cudaStream_t stream,
                         Args... args) {
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(blocks);
  config.blockDim = dim3((unsigned)threads);
  config.dynamicSmemBytes = shared;
  config.stream = stream;
  cudaLaunchAttribute attribute = {};
  attribute.id = cudaLaunchAttributeClusterDimension;
  attribute.val.clusterDim.x = (unsigned)cluster;
  attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
  config.attrs = &attribute;
  config.numAttrs = cluster > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&config, kernel, Params(args)...);
  if (e == cudaSuccess) noteLocalLaunch();
  return ownStatus(e);
}
// Lets a kernel's launches have that much shared memory.  Said once for a kernel, a device and a size, since saying it clears the
// error that may be pending, and never less than before: another thread may be about to launch with that.
inline cudaError_t allowShared(const void* kernel, size_t bytes) {
  static std::mutex mutex;
  static std::map<std::pair<const void*, int>, size_t> allowed;
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return ownStatus(e);
  const std::lock_guard<std::mutex> lock(mutex);
  size_t& most = allowed[{kernel, device}];
  if (bytes <= most) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess) most = bytes;
  return ownStatus(e);
}

template <typename... Params, typename... Args>
cudaError_t launchSlices(void (*kernel)(Params...), int64_t rows, int slices, int threads, size_t shared, cudaStream_t stream,
                         Args... args) {
  return launchBlocks(kernel, (unsigned)(rows * slices), threads, slices, shared, stream, args...);
}

// ---- many rows -----------------------------------------------------------------
// With a block per row the memory idles while a block starts and while it finishes its row, three to four
// microseconds of the ten that the row itself takes.  So where there are many rows the blocks stay, three a multiprocessor, and take
// row after row (8192 x 51200 bf16: 157 -> 134 us; with the rows dealt out in advance 142) in three roles:
//  - one warp fetches rows: it asks the hardware for a block that has not started yet and takes over that block's rows,
//    so that blocks which get more of the memory's bandwidth do more of them; it prepares what needs no look at the logits;
//  - eight warps sweep: every thread copies its own vectors to shared memory, kDepth - 1 batches ahead and
//    across the ends of rows, and waits for its own copies alone;
//  - one warp finishes rows while the next ones are swept.
// Read alone, 51200 bf16 logits a row, us and above the copy rate: 592 rows 19.6 (10.2), 1000 23.9
// (8.0), 2048 41.5 (9.0), 4096 71.8 (6.7), 8192 132.1 (1.9): the start, and the last rows of each
// block.
constexpr int kManyRows = 4;  // for each multiprocessor: 700 rows of 32003 fp32 logits 25.5 us by a block each, 21.5 here; 515 even, 300 the other way
constexpr int kDepth = 3;     // two batches of 16 KB on their way for each of the three blocks; one more gained nothing
constexpr int kRowThreads = kThreads + 64;  // sweep, then the warp that fetches, then the one that finishes
constexpr int kSlots = 3;                   // rows between being fetched and being finished; 4 to 6: 134 -> 136 us, with the rest 155 -> 171
constexpr uint32_t kPatience = 4000000000u;  // nanoseconds after which a wait is given up,
constexpr uint32_t kMostStep = 10000000u;    // and those that count of any one try
static_assert(kPatience + kMostStep > kPatience, "what has been waited does not start again");

__device__ __forceinline__ uint32_t sharedAddress(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void barrierInit(uint64_t* bar, int arrivals) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(sharedAddress(bar)), "r"(arrivals) : "memory");
}
__device__ __forceinline__ void barrierArrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(sharedAddress(bar)) : "memory");
}
__device__ __forceinline__ bool barrierTry(uint64_t* bar, unsigned parity) {
  uint32_t done;
  asm volatile(
      "{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
      : "=r"(done)
      : "r"(sharedAddress(bar)), "r"(parity)
      : "memory");
  return done != 0;
}
__device__ __forceinline__ uint32_t nanoseconds() {  // modulo 2^32
  uint32_t t;
  asm volatile("mov.u32 %0, %globaltimer_lo;" : "=r"(t));
  return t;
}
// False if the wait is given up.  What a block waits for is done by its own warps, so a block that was stopped (by a debugger, or
// for another context) finds it as it was: that time is no reason to give up.
__device__ __forceinline__ bool barrierWait(uint64_t* bar, unsigned parity) {
  if (barrierTry(bar, parity)) return true;
  uint32_t waited = 0, before = nanoseconds();
  while (!barrierTry(bar, parity)) {
    const uint32_t now = nanoseconds();
    waited += min(now - before, kMostStep);
    before = now;
    if (waited > kPatience) return false;
  }
  return true;
}
__device__ __forceinline__ void copyAhead(uint4* to, const uint4* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(sharedAddress(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void commitCopies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft> __device__ __forceinline__ void waitCopies() { asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory"); }

// A place in the sequence of slots.
struct Place {
  int slot = 0;
  unsigned parity = 0;
  __device__ __forceinline__ void next() {
    if (++slot == kSlots) slot = 0, parity ^= 1;
  }
};

// The rows that a block has taken.  Whoever gives up a wait has the block stop; what it has taken and not finished is NaN.
struct HandOver {
  alignas(16) uint4 answer;
  uint64_t answered;
  // The row is there; what its sweep needs is (the hook waits for that); what its finish needs is; its sums are; the slot is free.
  uint64_t ready[kSlots], marked[kSlots], prepared[kSlots], full[kSlots], empty[kSlots];
  Sums sums[kSlots][kWarps];
  int row[kSlots];  // -1: there are no more
  int failed;
  // By one thread, before a barrier of the block.
  __device__ __forceinline__ void init() {
    barrierInit(&answered, 1);
    for (int i = 0; i < kSlots; ++i) {
      barrierInit(&ready[i], 1);
      barrierInit(&marked[i], 1);
      barrierInit(&prepared[i], 1);
      barrierInit(&full[i], kWarps);
      barrierInit(&empty[i], 1);
    }
    failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __device__ __forceinline__ bool gaveUp() const { return *static_cast<const volatile int*>(&failed) != 0; }
  // All lanes of a warp; false once somebody gave up.
  __device__ __forceinline__ bool wait(uint64_t* bar, unsigned parity) {
    if (!gaveUp() && !barrierWait(bar, parity)) *static_cast<volatile int*>(&failed) = 1;
    __syncwarp();
    return !gaveUp();
  }
  __device__ __forceinline__ int rowAt(const Place& p) { return wait(&ready[p.slot], p.parity) ? row[p.slot] : -1; }
  // By one thread: asks for the block that would start next; the one before must have been answered with one.
  __device__ __forceinline__ void ask() {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], 16;" ::"r"(sharedAddress(&answered)) : "memory");
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                     sharedAddress(&answer)),
                 "r"(sharedAddress(&answered))
                 : "memory");
  }
  // By a warp: the number of the block that will not start, -1 if all have, or kNoAnswer.  Waits whoever has given up: the answer
  // comes to this block's memory.
  static constexpr int kNoAnswer = -2;
  __device__ __forceinline__ int answerOf(unsigned parity) {
    if (!__all_sync(kAll, barrierWait(&answered, parity))) {
      *static_cast<volatile int*>(&failed) = 1;
      return kNoAnswer;
    }
    int block;
    uint32_t ok;
    asm volatile(
        "{\n.reg .pred p;\n.reg .b128 r;\nld.shared.b128 r, [%2];\n"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\nselp.u32 %1, 1, 0, p;\nmov.u32 %0, 0;\n"
        "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %0, r;\n}"
        : "=r"(block), "=r"(ok)
        : "r"(sharedAddress(&answer))
        : "memory");
    __syncwarp();
    return ok ? block : -1;
  }
  // The row's sums in every lane of a warp; the columns outside the vectors are added here.
  // `left_out`: a bit for each of those that is not to be.
  template <typename T, bool kEntropy>
  __device__ __forceinline__ Sums take(int slot, const Slice<T>& sl, float c, unsigned left_out) const {
    const int lane = threadIdx.x & 31;
    Sums acc = lane < kWarps ? sums[slot][lane] : Sums::none(c);
    const int col = lane < 2 * Vec<T>::kElems && !(left_out >> lane & 1u) ? sl.looseCol(lane) : -1;
    if (col >= 0) acc.add<kEntropy>(toFloat(sl.row[col]), c);
    return warpSums<kEntropy>(acc, c);
  }
};

using Ring = uint4[kDepth][kBatch][kThreads];

// How many rows a block of the grid stands for: as many as make up 64 KB, so that asking for them does not cost more than they do,
// but so few that there are four blocks for each of those that stay.
inline int rowsABlock(const LogitRows& x, int elem_size, int sm_count) {
  const int64_t by_size = (65536 + (int64_t)x.vocab * elem_size - 1) / ((int64_t)x.vocab * elem_size), by_rows = x.rows / (12 * sm_count);
  const int64_t n = by_size < by_rows ? by_size : by_rows;
  return n < 1 ? 1 : n < 32 ? (int)n : 32;
}

// The fetching warp's part.  `counts(r)`, by one lane, says that a row does not count as far as that is seen at once, else skip(r), by
// one lane too.  prepare(r, place), by all, says for the others whether they do; mark(r, place) comes once the row's copies may begin.
// lose(r), by one lane, leaves NaN: of every row before it is handed on, of those that a block which gives up has taken, and, where
// that is not known since the hardware did not answer, of all: whoever has done one of them may have written it before or after.
// Copies run kDepth - 1 batches ahead, so as many rows: nothing that a row's copies wait for may itself wait for one of the
// kSlots - 1 rows before it.
static_assert(kSlots >= kDepth, "a row's copies begin while the row kDepth - 1 before it is swept");
template <class Counts, class Skip, class Lose, class Prepare, class Mark>
__device__ __forceinline__ void fetchRows(Counts&& counts, int64_t rows, int rows_a_block, HandOver& out, Skip&& skip, Lose&& lose,
                                          Prepare&& prepare, Mark&& mark) {
  const int lane = threadIdx.x & 31;
  Place place;
  unsigned parity = 0;
  for (int block = blockIdx.x; block >= 0; parity ^= 1) {
    if (lane == 0) out.ask();
    const int64_t first = (int64_t)block * rows_a_block, mine = first + lane;
    const bool some = lane < rows_a_block && mine < rows, yes = some && counts((int)mine);
    if (some && !yes) skip((int)mine);
    unsigned mask = __ballot_sync(kAll, yes);
    for (; mask != 0; mask &= mask - 1) {
      const int r = (int)first + __ffs(mask) - 1;
      if (!__all_sync(kAll, out.wait(&out.empty[place.slot], place.parity ^ 1))) break;
      if (!prepare(r, place)) {
        if (lane == 0) skip(r);
        continue;
      }
      __syncwarp();
      if (lane == 0) {
        lose(r);
        out.row[place.slot] = r;
        barrierArrive(&out.ready[place.slot]);
      }
      mark(r, place);
      __syncwarp();
      if (lane == 0) barrierArrive(&out.prepared[place.slot]);
      place.next();
    }
    block = out.answerOf(parity);
    if (__any_sync(kAll, out.gaveUp())) {
      if (mask >> lane & 1u) lose((int)mine);
      const int64_t next = (int64_t)block * rows_a_block + lane;
      if (block >= 0 && lane < rows_a_block && next < rows) lose((int)next);
      if (block == HandOver::kNoAnswer)
        for (int64_t r = lane; r < rows; r += 32) lose((int)r);
      return;
    }
  }
  if (!out.wait(&out.empty[place.slot], place.parity ^ 1)) return;
  if (lane == 0) {
    out.row[place.slot] = -1;
    barrierArrive(&out.ready[place.slot]);
  }
}

// The sweeping warps' part, threads 0 to kThreads - 1.  The hook sees a thread's part of batch b of a row in shared memory
// before it is read.
template <typename T, bool kEntropy, class Hook>
__device__ __forceinline__ void sweepRows(const T* logits, const LogitRows& x, float c, Ring& ring, HandOver& out, Hook& hook) {
  constexpr int U = kBatch;
  constexpr uint32_t w = Vec<T>::kMinusInf;
  const int tid = threadIdx.x;
  Place ahead, at;              // the row that is copied and the one that is summed
  const uint4* from = nullptr;  // of the row that is copied: this thread's next vector,
  int whole = 0, left = -1;     // the batches that all threads have, and the vectors behind those; < 0: the row is through
  bool more = true;
  auto open = [&] {
    const int r = out.rowAt(ahead);
    more = r >= 0;
    if (!more) return;
    ahead.next();
    const T* row = rowOf(x, logits, r);
    const RowParts<T> parts(row, x.vocab);
    from = reinterpret_cast<const uint4*>(row + parts.head) + tid;
    whole = parts.nvec / (U * kThreads);
    left = parts.nvec - whole * (U * kThreads);
    if (whole > 0 && left == 0) left = -1;
  };
  auto issue = [&](int slot) {
    if (whole == 0 && left < 0 && more) open();
    uint4* to = &ring[slot][0][tid];
    if (__any_sync(kAll, whole > 0)) {
#pragma unroll
      for (int u = 0; u < U; ++u) copyAhead(to + u * kThreads, from + u * kThreads);
      from += U * kThreads;
      --whole;
    } else if (left >= 0) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (tid + u * kThreads < left) copyAhead(to + u * kThreads, from + u * kThreads);
      left = -1;
    }
    commitCopies();
  };
#pragma unroll
  for (int d = 0; d < kDepth - 1; ++d) issue(d);
  int slot = 0;
  uint4 now[U];
  auto take = [&](int b) {  // the row's batch b; the place of the one before it, whose values have been used, is filled again
    waitCopies<kDepth - 2>();
    uint4* place = &ring[slot][0][tid];
    hook.arrived(place, b);
#pragma unroll
    for (int u = 0; u < U; ++u) now[u] = place[u * kThreads];
    issue(slot == 0 ? kDepth - 1 : slot - 1);
    slot = slot + 1 == kDepth ? 0 : slot + 1;
  };
  for (;; at.next()) {
    const int r = out.rowAt(at);
    if (r < 0) break;
    const Slice<T> sl(rowOf(x, logits, r), x.vocab, 0, 1);
    hook.begin(at);
    ThreadSums mine(c);
    const int batches = sl.v1 / (U * kThreads), rest = sl.v1 - batches * (U * kThreads);
    for (int b = 0; b < batches; ++b) {
      take(b);
      mine.add<T, kEntropy, true>(now, hook.batch(now, b == 0, tid + b * (U * kThreads), sl), U, c);
    }
    if (rest > 0 || batches == 0) {
      take(batches);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (tid + u * kThreads >= rest) now[u] = make_uint4(w, w, w, w);
      mine.add<T, kEntropy, false>(now, hook.batch(now, batches == 0, tid + batches * (U * kThreads), sl),
                                   (rest - (tid & ~31) + kThreads - 1) / kThreads, c);
    }
    hook.end();
    const Sums acc = warpSums<kEntropy>(mine.sums(), c);
    __syncwarp();  // what every lane has read of the row's slot and its marks before the arrival of one
    if ((tid & 31) == 0) {
      out.sums[at.slot][tid >> 5] = acc;
      barrierArrive(&out.full[at.slot]);
    }
  }
  waitCopies<0>();
}

// The finishing warp's part: finish(r, place), which waits for the row's sums.
template <class Finish> __device__ __forceinline__ void finishRows(HandOver& out, Finish&& finish) {
  for (Place at;; at.next()) {
    const int r = out.rowAt(at);
    if (r < 0) return;
    finish(r, at);
    __syncwarp();
    if ((threadIdx.x & 31) == 0) barrierArrive(&out.empty[at.slot]);
  }
}

template <typename... Params, typename... Args>
cudaError_t launchRows(void (*kernel)(Params...), int64_t rows, int rows_a_block, size_t shared, cudaStream_t stream, Args... args) {
  const cudaError_t e = allowShared(reinterpret_cast<const void*>(kernel), shared);
  if (e != cudaSuccess) return e;
  return launchBlocks(kernel, (unsigned)((rows + rows_a_block - 1) / rows_a_block), kRowThreads, 1, shared, stream, args...);
}

// Whether rows are many enough for that: several for each of the blocks that stay.
inline bool manyRows(int64_t rows, int sm_count) { return rows >= kManyRows * (int64_t)sm_count; }

// ---- many short rows -------------------------------------------------------------
// A short row is one warp's, which sweeps and finishes it: no thread waits for another warp, and a multiprocessor has 32 rows on the
// way.  Up to 16 KB wherever rows are many: 8192 x 1000 bf16 52 -> 6.2 us, the divergence 67 -> 11.  Up to 32 KB with eight rows
// a multiprocessor, since with fewer the longest rows take longest: 8192 x 12000 53 -> 45 and 70 -> 51, 8192 x 16000 59 -> 58 and
// 74 -> 63, 1500 x 12000 14.9 -> 13.8 and 19.3 -> 16.2, but 600 x 16000 10.9 -> 14.0 and 14.2 -> 16.3.
constexpr int kShortBytes = 32768, kVeryShortBytes = 16384;
inline bool shortRows(const LogitRows& x, int elem_size, int sm_count) {
  const int64_t bytes = (int64_t)x.vocab * elem_size;
  return bytes <= kShortBytes && x.rows >= (bytes <= kVeryShortBytes ? 1 : 2) * kManyRows * (int64_t)sm_count;
}
template <typename... Params, typename... Args>
cudaError_t launchShort(void (*kernel)(Params...), int64_t rows, size_t shared, cudaStream_t stream, Args... args) {
  return launchBlocks(kernel, (unsigned)((rows + kWarps - 1) / kWarps), kThreads, 1, shared, stream, args...);
}

}  // namespace softmax_row
}  // namespace fairring
