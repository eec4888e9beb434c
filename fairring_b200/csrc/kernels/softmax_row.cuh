// One sweep over a row of logits: its maximum m, S = sum of exp((x - m) / T) and, where the entropy is wanted,
// A = sum of exp((x - m) / T) * log2(exp((x - m) / T)).  Shared by the kernels that ask a language-model head's
// logits for probabilities.
//
// A row is the elements up to its first 16-byte boundary, 16-byte vectors, and what is left behind them.  A
// block takes a row or, where there are few rows, the blocks of a cluster take a slice of it each and the first
// one merges what they found, in the order of the slices.
//
// exp() is 2^((x - m) * c) with c = log2(e) / T, as one fused multiply-add of x, c and the rounded m * c; what that
// rounding changes all exponentials by is put right at the row's end.  The exponential's own error is 2^-22 of a
// probability.  That form needs |m * c| < 2^20.  A thread's m starts at -2^20 / c, below which nothing is seen of a row unless
// all of it is there; such rows (masked with the type's lowest value throughout, or with minus infinity), those above and those with
// a NaN come out of the sweep with a sum that is no positive number and are looked at again, slowly.
#pragma once

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

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

// Threads that finish a row together: all of a block, or some warps of it under a barrier of their own.
struct BlockGroup {
  static constexpr int kSize = kThreads;
  static __device__ __forceinline__ int rank() { return threadIdx.x; }
  static __device__ __forceinline__ void sync() { __syncthreads(); }
};
template <int kFirst, int kCount, int kBarrier> struct PartGroup {
  static constexpr int kSize = kCount;
  static __device__ __forceinline__ int rank() { return (int)threadIdx.x - kFirst; }
  static __device__ __forceinline__ void sync() { asm volatile("bar.sync %0, %1;" ::"n"(kBarrier), "n"(kCount) : "memory"); }
};

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
    return scaled(m, c) < kPlainRange && s > 0.f && s < INFINITY;
  }
};

// A thread's share of a row, from the first of its vectors on.
struct ThreadSums {
  float m, at;  // at = m * c
  float2 s, a;
  __device__ __forceinline__ explicit ThreadSums(float c) : m(-kPlainRange / c), at(scaled(m, c)), s{0.f, 0.f}, a{0.f, 0.f} {}
  // Adds the first n vectors of a batch whose largest value is `top`; all lanes of a warp have the same n.
  template <typename T, bool kEntropy, bool kWhole>
  __device__ __forceinline__ void add(const uint4 (&now)[kBatch], float top, int n, float c) {
    constexpr int E = Vec<T>::kElems;
    m = fmaxf(m, top);
    const float before = at;
    at = scaled(m, c);
    const float d = before - at, f = exp2Of(d);
    if (kEntropy) a = mul2(fma2(make_float2(fmaxf(d, kLowExponent), fmaxf(d, kLowExponent)), s, a), make_float2(f, f));
    s = mul2(s, make_float2(f, f));
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (!kWhole && u >= n) break;
      float2 v[E / 2];
      Vec<T>::get(now[u], v);
#pragma unroll
      for (int k = 0; k < E / 2; ++k) {
        const float2 d = fma2(v[k], make_float2(c, c), make_float2(-at, -at));
        const float2 e = make_float2(exp2Of(d.x), exp2Of(d.y));
        s = add2(s, e);
        if (kEntropy) a = fma2(e, make_float2(fmaxf(d.x, kLowExponent), fmaxf(d.y, kLowExponent)), a);
      }
    }
  }
  __device__ __forceinline__ Sums sums() const { return {m, s.x + s.y, a.x + a.y}; }
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

// What a kernel does with a batch, that from vector i on, before it is summed; returns its largest value.
struct NoHook {
  __device__ __forceinline__ void begin(int, unsigned) {}
  __device__ __forceinline__ void end() {}
  __device__ __forceinline__ void arrived(uint4*, int) {}
  template <typename T> __device__ __forceinline__ float batch(uint4 (&now)[kBatch], bool, int, const Slice<T>&) {
    return batchMax<T>(now);
  }
};

// This thread's share of the slice.  All threads of a block go through the same number of batches.  The next batch is on its
// way while this one is used.
template <typename T, bool kEntropy, class Hook>
__device__ __forceinline__ Sums scan(const Slice<T>& sl, float c, Hook& hook) {
  constexpr int U = kBatch;
  constexpr uint32_t w = Vec<T>::kMinusInf;
  const uint4* vecs = reinterpret_cast<const uint4*>(sl.row + sl.head);
  uint4 raw[U];
  auto fetch = [&](int i) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      raw[u] = i + u * kThreads < sl.v1 ? __ldg(vecs + i + u * kThreads) : make_uint4(w, w, w, w);
  };
  ThreadSums acc(c);
  const int batches = (sl.v1 - sl.v0 + U * kThreads - 1) / (U * kThreads);
  int i = sl.v0 + (int)threadIdx.x;
  fetch(i);
  for (int b = 0; b < batches; ++b, i += U * kThreads) {
    uint4 now[U];
#pragma unroll
    for (int u = 0; u < U; ++u) now[u] = raw[u];
    fetch(i + U * kThreads);
    acc.add<T, kEntropy, false>(now, hook.batch(now, b == 0, i, sl), (sl.v1 - (i & ~31) + kThreads - 1) / kThreads, c);
  }
  return acc.sums();
}

// Two sweeps over a row for what the fast one cannot do, by `size` threads: this one's share of it, relative to m.
template <typename T, bool kEntropy, class Leave>
__device__ __noinline__ Sums lookAgain(const T* row, int vocab, int rank, int size, float c, float top, Leave leave) {
  const float ref = top == -INFINITY ? 0.f : top;
  Sums acc = {top, 0.f, 0.f};
  for (int col = rank; col < vocab; col += size) {
    if (leave(col)) continue;
    const float d = (toFloat(row[col]) - ref) * c, e = exp2Of(d);
    acc.s += e;
    if (kEntropy) acc.a = fmaf(e, fmaxf(d, kLowExponent), acc.a);
  }
  return acc;
}
template <typename T, class Leave>
__device__ __noinline__ float largestOf(const T* row, int vocab, int rank, int size, Leave leave) {
  float top = -INFINITY;
  for (int col = rank; col < vocab; col += size)
    if (!leave(col)) top = fmaxf(top, toFloat(row[col]));
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

// The block's sums from its threads', in every thread.  `scratch`: kWarps of them in shared memory.
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

// A row's sums, relative to m, by a whole block or a whole warp, where the sweep's did not settle.
template <typename T, bool kEntropy, class Leave>
__device__ __noinline__ Sums blockAgain(const T* row, int vocab, float c, Sums* scratch, Leave leave) {
  float top = warpMax(largestOf(row, vocab, (int)threadIdx.x, kThreads, leave));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5].m = top;
  __syncthreads();
  for (int i = 0; i < kWarps; ++i) top = fmaxf(top, scratch[i].m);
  Sums acc = lookAgain<T, kEntropy>(row, vocab, (int)threadIdx.x, kThreads, c, top, leave);
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
  const int lane = threadIdx.x & 31;
  const float top = warpMax(largestOf(row, vocab, lane, 32, leave));
  Sums acc = lookAgain<T, kEntropy>(row, vocab, lane, 32, c, top, leave);
  acc.s = warpSum(acc.s);
  acc.a = warpSum(acc.a);
  return acc;
}
struct LeaveNone {
  __device__ __forceinline__ bool operator()(int) const { return false; }
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

// Into how many slices `rows` rows are cut, as a power of two: as many as keep two blocks a multiprocessor busy, but not
// so many that a block's slice is less than half a batch.
inline int slicesFor(int64_t rows, int vocab, int elem_size, int sm_count) {
  const int64_t vecs = (int64_t)vocab * elem_size / 16;
  int n = 1;
  while (n < kMostSlices && rows * n * 2 <= 2 * (int64_t)sm_count && vecs / (n * 2) >= kThreads * kBatch / 2) n *= 2;
  return n;
}

template <typename... Params, typename... Args>
cudaError_t launchSlices(void (*kernel)(Params...), int64_t rows, int slices, size_t shared, cudaStream_t stream,
                         Args... args) {
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)(rows * slices));
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = shared;
  config.stream = stream;
  cudaLaunchAttribute attribute = {};
  attribute.id = cudaLaunchAttributeClusterDimension;
  attribute.val.clusterDim.x = (unsigned)slices;
  attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
  config.attrs = &attribute;
  config.numAttrs = slices > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&config, kernel, Params(args)...);
  noteLocalLaunch();
  return e;
}

// ---- many rows -----------------------------------------------------------------
// With a block per row the memory idles while a block starts and while it finishes its row, three to four
// microseconds of the ten that the row itself takes (8192 x 51200 bf16: 144 us for the log probabilities, 4.6 to 5.8 TB/s).
// So where there are many rows the blocks stay and take row after row in three roles:
//  - eight warps sweep: every thread copies its own vectors to shared memory, kDepth - 1 batches ahead and
//    across the ends of rows, and waits for its own copies alone;
//  - they hand each row's sums over and go on without waiting;
//  - the other warps finish rows: what needs no sums they do while the row is swept.
constexpr int kManyRows = 4;  // for each multiprocessor
constexpr int kDepth = 3;
constexpr int kSpins = 1 << 20;  // tries, each of which the hardware lets sleep; then the wait is given up

__device__ __forceinline__ uint32_t sharedAddress(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void barrierInit(uint64_t* bar, int arrivals) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(sharedAddress(bar)), "r"(arrivals) : "memory");
}
__device__ __forceinline__ void barrierArrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(sharedAddress(bar)) : "memory");
}
__device__ __forceinline__ bool barrierWait(uint64_t* bar, unsigned parity) {
  for (int i = 0; i < kSpins; ++i) {
    uint32_t done;
    asm volatile(
        "{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
        : "=r"(done)
        : "r"(sharedAddress(bar)), "r"(parity)
        : "memory");
    if (done) return true;
  }
  return false;
}
__device__ __forceinline__ void copyAhead(uint4* to, const uint4* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(sharedAddress(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void commitCopies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft> __device__ __forceinline__ void waitCopies() { asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory"); }

// The rows of this block that count, in order, as every warp finds them for itself: a lane looks at one of the next 32.
template <class Counts> struct RowWalk {
  const Counts& counts;
  const unsigned rows;
  unsigned base;      // the row of lane 0
  unsigned mask = 0;  // of those not yet taken
  int row = -1;       // the current one; -1: none left
  __device__ __forceinline__ RowWalk(const Counts& counts_, int64_t rows_)
      : counts(counts_), rows((unsigned)rows_), base(blockIdx.x - 32 * gridDim.x) {}
  template <class Skip> __device__ __forceinline__ void next(Skip&& skip) {
    while (mask == 0) {
      base += 32 * gridDim.x;
      if (base >= rows) {
        base -= 32 * gridDim.x;
        row = -1;
        return;
      }
      const unsigned mine = base + (threadIdx.x & 31) * gridDim.x;
      const bool some = mine < rows, yes = some && counts((int)mine);
      if (some && !yes) skip((int)mine);
      mask = __ballot_sync(kAll, yes);
    }
    row = (int)(base + (__ffs(mask) - 1) * gridDim.x);
    mask &= mask - 1;
  }
  __device__ __forceinline__ void next() {
    next([](int) {});
  }
};

// What the sweeping warps hand over, for as many rows as may be unfinished at once.
template <int kRows> struct HandOver {
  // The row's listed tokens are marked; its sums are there; the buffer is free for another row.
  uint64_t ready[kRows], full[kRows], empty[kRows];
  Sums sums[kRows][kWarps];
  int failed;
  // By one thread, before a barrier of the block.
  __device__ __forceinline__ void init() {
    for (int i = 0; i < kRows; ++i) {
      barrierInit(&ready[i], 1);
      barrierInit(&full[i], kWarps);
      barrierInit(&empty[i], 1);
    }
    failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // All lanes of a warp.  Once a wait was given up nobody waits any more, and the block's rows become NaN.
  __device__ __forceinline__ void wait(uint64_t* bar, unsigned parity) {
    if (!gaveUp() && !barrierWait(bar, parity)) *static_cast<volatile int*>(&failed) = 1;
    __syncwarp();
  }
  // The row's sums in every lane of a warp; the columns outside the vectors are added here.
  // `left_out`: a bit for each of those that is not to be.
  template <typename T, bool kEntropy>
  __device__ __forceinline__ Sums take(int buffer, const Slice<T>& sl, float c, unsigned left_out) const {
    const int lane = threadIdx.x & 31;
    Sums acc = lane < kWarps ? sums[buffer][lane] : Sums::none(c);
    const int col = lane < 2 * Vec<T>::kElems && !(left_out >> lane & 1u) ? sl.looseCol(lane) : -1;
    if (col >= 0) acc.add<kEntropy>(toFloat(sl.row[col]), c);
    return warpSums<kEntropy>(acc, c);
  }
  __device__ __forceinline__ bool gaveUp() const { return *static_cast<const volatile int*>(&failed) != 0; }
};

using Ring = uint4[kDepth][kBatch][kThreads];

// The sweeping warps' part, threads 0 to kThreads - 1.  The hook sees a thread's part of batch b of a row in shared memory
// before it is read.
template <typename T, bool kEntropy, int kRows, class Hook, class Counts>
__device__ __forceinline__ void sweepRows(const T* logits, const LogitRows& x, const Counts& counts, float c, Ring& ring,
                                          HandOver<kRows>& out, Hook& hook) {
  constexpr int U = kBatch;
  constexpr uint32_t w = Vec<T>::kMinusInf;
  const int tid = threadIdx.x;
  RowWalk<Counts> ahead(counts, x.rows), at(counts, x.rows);  // the row that is copied and the one that is summed
  const uint4* from = nullptr;  // of the row that is copied: this thread's next vector,
  int whole = 0, left = 0;      // the batches that all threads have, and the vectors from this thread's on behind those; < 0: no row
  auto open = [&] {
    ahead.next();
    left = -kThreads;
    if (ahead.row < 0) return;
    const T* row = rowOf(x, logits, ahead.row);
    const RowParts<T> parts(row, x.vocab);
    from = reinterpret_cast<const uint4*>(row + parts.head) + tid;
    whole = parts.nvec / (U * kThreads);
    left = parts.nvec - whole * (U * kThreads);
  };
  auto issue = [&](int slot) {
    uint4* to = &ring[slot][0][tid];
    if (__any_sync(kAll, whole > 0)) {
#pragma unroll
      for (int u = 0; u < U; ++u) copyAhead(to + u * kThreads, from + u * kThreads);
      from += U * kThreads;
      if (--whole == 0 && left == 0) open();
    } else if (left >= 0) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (tid + u * kThreads < left) copyAhead(to + u * kThreads, from + u * kThreads);
      open();
    }
    commitCopies();
  };
  open();
#pragma unroll
  for (int d = 0; d < kDepth - 1; ++d) issue(d);
  int slot = 0, buffer = 0;
  unsigned parity = 0;
  uint4 now[U];
  auto take = [&](int b) {  // the row's batch b, whose turn it is; the place of the one before it, whose values have been used, is filled again
    waitCopies<kDepth - 2>();
    uint4* place = &ring[slot][0][tid];
    hook.arrived(place, b);
#pragma unroll
    for (int u = 0; u < U; ++u) now[u] = place[u * kThreads];
    issue(slot == 0 ? kDepth - 1 : slot - 1);
    slot = slot + 1 == kDepth ? 0 : slot + 1;
  };
  for (at.next(); at.row >= 0; at.next()) {
    const Slice<T> sl(rowOf(x, logits, at.row), x.vocab, 0, 1);
    out.wait(&out.empty[buffer], parity ^ 1);
    hook.begin(buffer, parity);
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
    if ((tid & 31) == 0) {
      out.sums[buffer][tid >> 5] = acc;
      barrierArrive(&out.full[buffer]);
    }
    if (++buffer == kRows) buffer = 0, parity ^= 1;
  }
  waitCopies<0>();
}

// A finishing warp's or group's part: finish(row, buffer, parity) for those of the rows that count whose number is `which`
// modulo `each`, skip(row) by single lanes for those that do not.
template <int kRows, class Counts, class Finish, class Skip>
__device__ __forceinline__ void finishRows(const Counts& counts, int64_t rows, int which, int each, Finish&& finish, Skip&& skip) {
  RowWalk<Counts> at(counts, rows);
  int buffer = 0, turn = 0;
  unsigned parity = 0;
  for (at.next(skip); at.row >= 0; at.next(skip)) {
    if (turn == which) finish(at.row, buffer, parity);
    if (++turn == each) turn = 0;
    if (++buffer == kRows) buffer = 0, parity ^= 1;
  }
}

template <typename... Params, typename... Args>
cudaError_t launchResident(void (*kernel)(Params...), int64_t rows, int threads, int blocks_per_sm, size_t shared,
                           int sm_count, cudaStream_t stream, Args... args) {
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)shared);
  if (e != cudaSuccess) return e;
  // Those that stay, or one for six rows: blocks do not get equal shares of the memory's bandwidth, and the hardware
  // hands out the later ones to whoever is done.
  const int64_t stay = (int64_t)blocks_per_sm * sm_count, blocks = rows / 6 > stay ? rows / 6 : stay;
  kernel<<<(unsigned)(rows < blocks ? rows : blocks), threads, shared, stream>>>(Params(args)...);
  noteLocalLaunch();
  return cudaGetLastError();
}

// Whether rows are many enough for that: several for each of the blocks that stay.
inline bool manyRows(int64_t rows, int sm_count) { return rows >= kManyRows * (int64_t)sm_count; }

}  // namespace softmax_row
}  // namespace fairring
