// One sweep over a row of logits: its maximum m, S = sum of exp((x - m) / T) and, where the entropy is wanted,
// A = sum of exp((x - m) / T) * log2(exp((x - m) / T)).  Shared by the kernels that ask a language-model head's
// logits for probabilities.
//
// A row is the elements up to its first 16-byte boundary, 16-byte vectors, and what is left behind them.  A
// block takes a row or, where there are few rows, the blocks of a cluster take a slice of it each and the first
// one merges what they found, in the order of the slices.
//
// exp() is 2^((x - m) * c) with c = log2(e) / T.  The difference is taken before the product: m * c of a row
// that is masked with the type's lowest value throughout would be minus infinity.  The exponential's own error
// is 2^-22 of a probability, the two roundings before it 2^-23 of the exponent.
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

struct Sums {
  float m = -INFINITY, s = 0.f, a = 0.f;
  // What differences are taken from: never -inf, whose difference from itself is NaN.
  static __device__ __forceinline__ float reference(float m) { return m == -INFINITY ? 0.f : m; }
  // The sums relative to `ref`, which is at least m.
  template <bool kEntropy> __device__ __forceinline__ void rescale(float ref, float c) {
    const float d = (m - ref) * c, f = exp2Of(d);
    if (kEntropy) a = f * fmaf(fmaxf(d, kLowExponent), s, a);
    s *= f;
  }
  template <bool kEntropy> __device__ __forceinline__ void merge(Sums o, float c) {
    const float top = fmaxf(m, o.m), ref = reference(top);
    rescale<kEntropy>(ref, c);
    o.template rescale<kEntropy>(ref, c);
    s += o.s;
    if (kEntropy) a += o.a;
    m = top;
  }
  template <bool kEntropy> __device__ __forceinline__ void add(float v, float c) {
    Sums o;
    o.m = v;
    o.s = v == -INFINITY ? 0.f : 1.f;
    if (v != v) o.m = -INFINITY, o.s = v;
    merge<kEntropy>(o, c);
  }
  template <bool kEntropy> __device__ __forceinline__ Sums fromLane(int lane_mask) const {
    Sums o;
    o.m = __shfl_xor_sync(kAll, m, lane_mask);
    o.s = __shfl_xor_sync(kAll, s, lane_mask);
    if (kEntropy) o.a = __shfl_xor_sync(kAll, a, lane_mask);
    return o;
  }
};

// What a kernel may do with a batch of vectors before they are summed: nothing.
struct NoHook {
  template <typename V> __device__ __forceinline__ void mask(uint4 (&)[kBatch], int, const V&) {}
  template <typename V>
  __device__ __forceinline__ void batch(int, const uint4 (&)[kBatch], const float (&)[kBatch], float, int, const V&) {}
};

// This thread's sums over its share of the slice.  All threads of a block go through the same number of batches.
// The next batch is on its way while this one is used.
template <typename T, bool kEntropy, class Hook>
__device__ __forceinline__ Sums scan(const Slice<T>& sl, float c, Hook& hook) {
  constexpr int E = Vec<T>::kElems, U = kBatch;
  constexpr uint32_t w = Vec<T>::kMinusInf;
  const uint4* vecs = reinterpret_cast<const uint4*>(sl.row + sl.head);
  uint4 raw[U];
  auto fetch = [&](int i) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      raw[u] = i + u * kThreads < sl.v1 ? __ldg(vecs + i + u * kThreads) : make_uint4(w, w, w, w);
  };
  Sums acc;
  const int batches = (sl.v1 - sl.v0 + U * kThreads - 1) / (U * kThreads);
  int i = sl.v0 + (int)threadIdx.x;
  fetch(i);
  for (int b = 0; b < batches; ++b, i += U * kThreads) {
    uint4 now[U];
#pragma unroll
    for (int u = 0; u < U; ++u) now[u] = raw[u];
    fetch(i + U * kThreads);
    hook.mask(now, i, sl);
    float vmax[U], top = acc.m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      vmax[u] = Vec<T>::max(now[u]);
      top = fmaxf(top, vmax[u]);
    }
    hook.batch(b, now, vmax, top, i, sl);
    const float ref = Sums::reference(top);
    const float2 minus = make_float2(-ref, -ref), cc = make_float2(c, c);
    float2 s2 = make_float2(0.f, 0.f), a2 = s2;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float2 v[E / 2];
      Vec<T>::get(now[u], v);
#pragma unroll
      for (int k = 0; k < E / 2; ++k) {
        const float2 d = mul2(add2(v[k], minus), cc);
        const float2 e = make_float2(exp2Of(d.x), exp2Of(d.y));
        s2 = add2(s2, e);
        if (kEntropy) a2 = fma2(e, make_float2(fmaxf(d.x, kLowExponent), fmaxf(d.y, kLowExponent)), a2);
      }
    }
    acc.rescale<kEntropy>(ref, c);
    acc.s += s2.x + s2.y;
    if (kEntropy) acc.a += a2.x + a2.y;
    acc.m = top;
  }
  return acc;
}

// The block's sums from its threads', in every thread.  `scratch`: kWarps of them in shared memory.
template <bool kEntropy> __device__ __forceinline__ Sums blockSums(Sums acc, float c, Sums* scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) acc.merge<kEntropy>(acc.fromLane<kEntropy>(o), c);
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = acc;
  __syncthreads();
  acc = scratch[0];
#pragma unroll
  for (int i = 1; i < kWarps; ++i) acc.merge<kEntropy>(scratch[i], c);
  return acc;
}

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

}  // namespace softmax_row
}  // namespace fairring
