// Log probabilities of given tokens under the softmax of a row of logits, the distribution's entropy and its
// largest entries (sm_100a); the gradient of the first two.
//
// With z = x / T, m and S of softmax_row.cuh:  log p_v = (z_v - max z) - log S,  H = log S - A ln 2 / S, a sum of two
// terms that are not negative.  Backward:  dx_v = 1/T [ g (1[v = t] - p_v) - h p_v (log p_v + H) ].
#include <cmath>

#include "softmax_row.cuh"

namespace fairring {
namespace {

using namespace softmax_row;

constexpr int kMostTop = kMostTopTokens;
constexpr int kKeptVecs = 1024;  // vectors that may hold one of the largest
constexpr int kList = 1024;      // candidates that are sorted; at least kMostSlices * kMostTop

// Order of logits as unsigned integers: NaN above everything, both zeros alike.
__device__ __forceinline__ uint32_t keyOf(float v) {
  if (v != v) return 0xffffffffu;
  const uint32_t b = __float_as_uint(v + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float valueOf(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
// A larger logit, then a smaller column, is the larger entry; no entry is 0.
__device__ __forceinline__ uint64_t entryOf(float v, int col) { return (uint64_t)keyOf(v) << 32 | (uint32_t)~col; }

struct TopShared {
  uint4 vec[kKeptVecs];
  int at[kKeptVecs];
  uint64_t list[kList];
  float bound[2][kWarps];
  unsigned hist[256];
  unsigned kept, listed, digit, left;
};

// Falling order of 32 values, one per lane.
__device__ __forceinline__ float sortedLanes(float v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size *= 2)
#pragma unroll
    for (int step = size / 2; step > 0; step /= 2) {
      const float o = __shfl_xor_sync(kAll, v, step);
      const bool larger = ((lane & step) == 0) == ((lane & size) == 0 || size == 32);
      v = larger ? fmaxf(v, o) : fminf(v, o);
    }
  return v;
}

// Keeps the vectors of the sweep that may hold one of the k largest.  If every warp has seen r = ceil(k / warps)
// values of `bound` or more, one in each of r lanes, k values of the row are that large.  So each warp
// sorts its lanes' maxima and gives its r-th; the smallest of these is the bound, renewed after batches 1, 2, 4, ...
// A vector below it is out.  What passes is a few hundred vectors of a row, against 8 compares per logit that
// picking single logits costs.
struct TopHook {
  TopShared* shared;
  int rank_in_warp;  // r - 1
  float bound = -INFINITY;
  int renewals = 0;
  template <typename V> __device__ __forceinline__ void mask(uint4 (&)[kBatch], int, const V&) {}
  __device__ __forceinline__ void renew(float top) {
    float* mine = shared->bound[renewals++ & 1];
    const float r = __shfl_sync(kAll, sortedLanes(top), rank_in_warp);
    if ((threadIdx.x & 31) == 0) mine[threadIdx.x >> 5] = r;
    __syncthreads();
    float b = mine[0];
#pragma unroll
    for (int i = 1; i < kWarps; ++i) b = fminf(b, mine[i]);
    bound = b;
  }
  __device__ __forceinline__ bool passes(float v) const { return v >= bound && v > -INFINITY; }
  template <typename V>
  __device__ __forceinline__ void batch(int b, const uint4 (&now)[kBatch], const float (&vmax)[kBatch], float top, int i,
                                        const V&) {
    if ((b & (b + 1)) == 0) renew(top);
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
      if (passes(vmax[u])) {
        const unsigned pos = atomicAdd(&shared->kept, 1u);
        if (pos < kKeptVecs) {
          shared->vec[pos] = now[u];
          shared->at[pos] = i + u * kThreads;
        }
      }
  }
};

// The first `n` entries of the list in falling order; those up to the next power of two are overwritten.
__device__ __forceinline__ void sortList(uint64_t* list, int n) {
  int size = 2;
  while (size < n) size *= 2;
  for (int i = n + (int)threadIdx.x; i < size; i += kThreads) list[i] = 0;
  __syncthreads();
  for (int block = 2; block <= size; block *= 2)
    for (int step = block / 2; step > 0; step /= 2) {
      for (int i = threadIdx.x; i < size / 2; i += kThreads) {
        const int a = 2 * i - (i & (step - 1)), b = a + step;
        const uint64_t x = list[a], y = list[b];
        if ((x < y) == ((a & block) == 0)) list[a] = y, list[b] = x;
      }
      __syncthreads();
    }
}

// The `want` largest of the slice's entries, into the list in any order, by a radix select that reads the slice six
// times and more: for rows where the bound lets too much pass (ties, falling or rising logits) and those with NaN.
template <typename T> __device__ void selectExactly(const Slice<T>& sl, int want, TopShared* sh) {
  uint32_t prefix = 0;
  unsigned left = want;
  for (int shift = 24; shift >= 0; shift -= 8) {
    sh->hist[threadIdx.x] = 0;
    __syncthreads();
    for (int col = sl.c0 + (int)threadIdx.x; col < sl.c1; col += kThreads) {
      const uint32_t key = keyOf(toFloat(sl.row[col]));
      if (shift == 24 || key >> (shift + 8) == prefix) atomicAdd(&sh->hist[key >> shift & 255u], 1u);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      int digit = 255;
      unsigned more = left;
      while (digit > 0 && sh->hist[digit] < more) more -= sh->hist[digit--];
      sh->digit = digit;
      sh->left = more;
    }
    __syncthreads();
    prefix = prefix << 8 | sh->digit;
    left = sh->left;
    __syncthreads();
  }
  // `prefix` is the key of the last one; `left` of those that equal it are taken, the first ones.
  if (threadIdx.x == 0) sh->listed = 0;
  __syncthreads();
  for (int col = sl.c0 + (int)threadIdx.x; col < sl.c1; col += kThreads) {
    const float v = toFloat(sl.row[col]);
    if (keyOf(v) > prefix) sh->list[atomicAdd(&sh->listed, 1u)] = entryOf(v, col);
  }
  const unsigned larger = want - left;
  unsigned taken = 0;
  for (int base = sl.c0; base < sl.c1 && taken < left; base += kThreads) {
    const int col = base + (int)threadIdx.x;
    const float v = col < sl.c1 ? toFloat(sl.row[col]) : 0.f;
    const bool equal = col < sl.c1 && keyOf(v) == prefix;
    const unsigned votes = __ballot_sync(kAll, equal);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh->hist[threadIdx.x >> 5] = __popc(votes);
    __syncthreads();
    unsigned before = taken + __popc(votes & ((1u << (threadIdx.x & 31)) - 1u)), all = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w < (int)(threadIdx.x >> 5)) before += sh->hist[w];
      all += sh->hist[w];
    }
    if (equal && before < left) sh->list[larger + before] = entryOf(v, col);
    taken += all;
  }
  __syncthreads();
}

// The slice's largest entries, at most k, in falling order at the start of the list; zeros behind them up to k.
template <typename T>
__device__ void sliceTop(const Slice<T>& sl, int k, float top, bool nan, TopHook& hook, TopShared* sh) {
  constexpr int E = Vec<T>::kElems;
  const int want = min(k, sl.c1 - sl.c0);
  hook.renew(top);
  const unsigned kept = sh->kept;
  if (kept <= kKeptVecs) {
    for (unsigned j = threadIdx.x; j < kept; j += kThreads) {
      float2 v[E / 2];
      Vec<T>::get(sh->vec[j], v);
      const int col = sl.head + sh->at[j] * E;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float x = e & 1 ? v[e / 2].y : v[e / 2].x;
        if (hook.passes(x)) {
          const unsigned pos = atomicAdd(&sh->listed, 1u);
          if (pos < kList) sh->list[pos] = entryOf(x, col + e);
        }
      }
    }
    const int col = threadIdx.x < 2 * E ? sl.looseCol(threadIdx.x) : -1;
    if (col >= 0) {
      const float x = toFloat(sl.row[col]);
      if (hook.passes(x)) {
        const unsigned pos = atomicAdd(&sh->listed, 1u);
        if (pos < kList) sh->list[pos] = entryOf(x, col);
      }
    }
  }
  __syncthreads();
  int n = sh->listed;
  __syncthreads();
  if (nan || kept > kKeptVecs || n > kList || n < want) {
    selectExactly(sl, want, sh);
    n = want;
  }
  sortList(sh->list, max(n, 1));
  for (int i = max(n, 1) + (int)threadIdx.x; i < k; i += kThreads) sh->list[i] = 0;
  if (n == 0 && threadIdx.x == 0) sh->list[0] = 0;
  __syncthreads();
}

// The k largest of the row from the slices' lists, in block 0.  clusterSums() has waited for the lists.
__device__ __forceinline__ void clusterTop(int k, TopShared* sh) {
  namespace cg = cooperative_groups;
  const cg::cluster_group cluster = cg::this_cluster();
  const int slices = cluster.num_blocks();
  if (slices == 1 || cluster.block_rank() != 0) return;
  for (int i = threadIdx.x; i < (slices - 1) * k; i += kThreads) {
    const int r = 1 + i / k;
    sh->list[r * k + (i - (r - 1) * k)] = cluster.map_shared_rank(sh, r)->list[i - (r - 1) * k];
  }
  __syncthreads();
  sortList(sh->list, slices * k);
}

// One row per cluster.  Kept for the backward: the row's maximum and S; S is -1 where the row does not count
// and NaN where its token is none.
template <typename T, bool kEntropy, bool kTop>
__global__ void __launch_bounds__(kThreads, kTop ? 3 : 4)
token_log_probs_fwd_kernel(const T* __restrict__ logits, LogitRows x, const int64_t* __restrict__ tokens, float c,
                           float inv_t, float* __restrict__ log_probs, float* __restrict__ entropy,
                           float2* __restrict__ stats, int k, float* __restrict__ top_log_probs,
                           int64_t* __restrict__ top_tokens) {
  namespace cg = cooperative_groups;
  __shared__ Sums scratch[kWarps], mine;
  const cg::cluster_group cluster = cg::this_cluster();
  const int slices = cluster.num_blocks(), rank = cluster.block_rank();
  const int64_t r = blockIdx.x / slices;
  const int64_t t = tokens != nullptr ? tokens[r] : 0;
  if (t < 0) {
    if (rank != 0) return;
    if (threadIdx.x == 0) {
      if (log_probs != nullptr) log_probs[r] = 0.f;
      if (kEntropy) entropy[r] = 0.f;
      if (stats != nullptr) stats[r] = make_float2(0.f, -1.f);
    }
    if (kTop)
      for (int i = threadIdx.x; i < k; i += kThreads) {
        top_log_probs[r * k + i] = -INFINITY;
        top_tokens[r * k + i] = -1;
      }
    return;
  }
  const Slice<T> sl(rowOf(x, logits, r), x.vocab, rank, slices);
  Sums acc;
  TopShared* sh = nullptr;
  TopHook hook;
  if constexpr (kTop) {
    extern __shared__ __align__(16) unsigned char dynamic[];
    sh = reinterpret_cast<TopShared*>(dynamic);
    hook.shared = sh;
    hook.rank_in_warp = (k + kWarps - 1) / kWarps - 1;
    if (threadIdx.x == 0) sh->kept = sh->listed = 0;
    __syncthreads();
    acc = scan<T, kEntropy>(sl, c, hook);
  } else {
    NoHook none;
    acc = scan<T, kEntropy>(sl, c, none);
  }
  const float top = acc.m;
  if (threadIdx.x < 2 * Vec<T>::kElems) {
    const int col = sl.looseCol(threadIdx.x);
    if (col >= 0) acc.add<kEntropy>(toFloat(sl.row[col]), c);
  }
  acc = blockSums<kEntropy>(acc, c, scratch);
  if constexpr (kTop) sliceTop(sl, k, top, acc.s != acc.s, hook, sh);
  if (slices > 1) {
    acc = clusterSums<kEntropy>(acc, c, &mine);
    if constexpr (kTop) clusterTop(k, sh);
    clusterDone();
    if (rank != 0) return;
  }
  const float low = logf(acc.s);
  if (threadIdx.x == 0) {
    const bool known = t < x.vocab;
    if (log_probs != nullptr)
      log_probs[r] = known ? fmaf(toFloat(sl.row[t]) - acc.m, inv_t, -low) : __int_as_float(0x7fffffff);
    if (kEntropy) entropy[r] = low - acc.a / acc.s * kLn2;
    if (stats != nullptr) stats[r] = make_float2(acc.m, known ? acc.s : __int_as_float(0x7fffffff));
  }
  if constexpr (kTop)
    for (int i = threadIdx.x; i < k; i += kThreads) {
      const uint64_t entry = sh->list[i];
      top_log_probs[r * k + i] = fmaf(valueOf((uint32_t)(entry >> 32)) - acc.m, inv_t, -low);
      top_tokens[r * k + i] = (int)~(uint32_t)entry;
    }
}

// A block does one batch of vectors of one row, so that all blocks are alike whatever the vocabulary.
template <typename T, bool kEntropy>
__global__ void __launch_bounds__(kThreads)
token_log_probs_bwd_kernel(const T* __restrict__ logits, LogitRows x, T* __restrict__ grad,
                           const int64_t* __restrict__ tokens, const float2* __restrict__ stats,
                           const float* __restrict__ entropy, const float* __restrict__ g_log_probs, int64_t g_stride,
                           const float* __restrict__ g_entropy, int64_t h_stride, float c, float inv_t,
                           int64_t pieces_total, int pieces) {
  constexpr int E = Vec<T>::kElems, U = kBatch;
  for (int64_t w = blockIdx.x; w < pieces_total; w += gridDim.x) {
    const int64_t r = w / pieces;
    const int piece = (int)(w - r * pieces);
    const T* row = rowOf(x, logits, r);
    T* out = rowOf(x, grad, r);
    const RowParts<T> parts(row, x.vocab);
    const int first = piece * U * kThreads + (int)threadIdx.x;
    const uint4* vecs = reinterpret_cast<const uint4*>(row + parts.head);
    uint4* vout = reinterpret_cast<uint4*>(out + parts.head);
    const float2 st = stats[r];
    const bool counts = !(st.y == -1.f);
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      raw[u] = counts && first + u * kThreads < parts.nvec ? __ldg(vecs + first + u * kThreads) : make_uint4(0, 0, 0, 0);
    const float g = g_log_probs != nullptr ? g_log_probs[r * g_stride] * inv_t : 0.f;
    const float h = kEntropy ? g_entropy[r * h_stride] * inv_t : 0.f;
    const int64_t t64 = tokens != nullptr ? tokens[r] : -1;
    const int t = t64 < x.vocab ? (int)t64 : -1;
    // g (1[v = t] - p) - h p (log p + H) with p = e / S and log p = u ln 2 - log S, u the exponent of e
    const float per_s = 1.f / st.y;
    const float a = -(kEntropy ? fmaf(h, entropy[r] - logf(st.y), g) : g) * per_s, b = -h * kLn2 * per_s;
    auto of = [&](float2 v) {
      const float2 d = mul2(add2(v, make_float2(-st.x, -st.x)), make_float2(c, c));
      const float2 e = make_float2(exp2Of(d.x), exp2Of(d.y));
      if (!kEntropy) return mul2(e, make_float2(a, a));
      return mul2(e, fma2(make_float2(fmaxf(d.x, kLowExponent), fmaxf(d.y, kLowExponent)), make_float2(b, b), make_float2(a, a)));
    };
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = first + u * kThreads;
      if (i >= parts.nvec) continue;
      uint4 result = make_uint4(0, 0, 0, 0);
      if (counts) {
        float2 v[E / 2];
        Vec<T>::get(raw[u], v);
        const int at = t - (parts.head + i * E);
#pragma unroll
        for (int k = 0; k < E / 2; ++k) v[k] = of(v[k]);
        if ((unsigned)at < (unsigned)E) {
#pragma unroll
          for (int k = 0; k < E / 2; ++k) {
            if (at == 2 * k) v[k].x += g;
            if (at == 2 * k + 1) v[k].y += g;
          }
        }
        result = Vec<T>::set(v);
      }
      vout[i] = result;
    }
    if (piece == 0 && threadIdx.x < 2 * E) {
      const int i = threadIdx.x, col = i < parts.head ? i : i + parts.nvec * E;
      if (col < x.vocab)
        fromFloat(out + col, counts ? of(make_float2(toFloat(row[col]), 0.f)).x + (col == t ? g : 0.f) : 0.f);
    }
  }
}

template <typename T>
cudaError_t forwardOf(const void* logits, const LogitRows& x, const TokenLogProbsArgs& a, int sm_count, cudaStream_t stream) {
  const int slices = slicesFor(x.rows, x.vocab, sizeof(T), sm_count);
  const T* data = static_cast<const T*>(logits);
  const float inv_t = (float)(1.0 / a.temperature), c = (float)(1.4426950408889634 / a.temperature);
  const size_t shared = a.k > 0 ? sizeof(TopShared) : 0;
  auto run = [&](auto kernel) {
    return launchSlices(kernel, x.rows, slices, shared, stream, data, x, a.tokens, c, inv_t, a.log_probs, a.entropy,
                        reinterpret_cast<float2*>(a.stats), a.k, a.top_log_probs, a.top_tokens);
  };
  if (a.k > 0) return a.entropy != nullptr ? run(token_log_probs_fwd_kernel<T, true, true>) : run(token_log_probs_fwd_kernel<T, false, true>);
  return a.entropy != nullptr ? run(token_log_probs_fwd_kernel<T, true, false>) : run(token_log_probs_fwd_kernel<T, false, false>);
}

template <typename T>
cudaError_t backwardOf(const void* logits, const LogitRows& x, void* grad, const TokenLogProbsGrads& a, cudaStream_t stream) {
  constexpr int per_piece = kThreads * kBatch * Vec<T>::kElems;
  const int pieces = (int)(((int64_t)x.vocab + per_piece - 1) / per_piece);
  const int64_t total = x.rows * pieces;
  const unsigned blocks = (unsigned)(total < (1 << 30) ? total : (1 << 30));
  const float inv_t = (float)(1.0 / a.temperature), c = (float)(1.4426950408889634 / a.temperature);
  auto run = [&](auto kernel) {
    kernel<<<blocks, kThreads, 0, stream>>>(static_cast<const T*>(logits), x, static_cast<T*>(grad), a.tokens,
                                            reinterpret_cast<const float2*>(a.stats), a.entropy, a.g_log_probs, a.g_stride,
                                            a.g_entropy, a.h_stride, c, inv_t, total, pieces);
    noteLocalLaunch();
    return cudaGetLastError();
  };
  return a.g_entropy != nullptr ? run(token_log_probs_bwd_kernel<T, true>) : run(token_log_probs_bwd_kernel<T, false>);
}

}  // namespace

cudaError_t launchTokenLogProbs(const void* logits, const LogitRows& x, const TokenLogProbsArgs& a, int sm_count,
                                cudaStream_t stream) {
  if (x.rows <= 0) return cudaSuccess;
  if (x.vocab <= 0 || x.rows > INT32_MAX || a.k < 0 || a.k > kMostTop || a.k > x.vocab) return cudaErrorInvalidValue;
  switch (x.type) {
    case LogitType::kBFloat16: return forwardOf<__nv_bfloat16>(logits, x, a, sm_count, stream);
    case LogitType::kHalf: return forwardOf<__half>(logits, x, a, sm_count, stream);
    default: return forwardOf<float>(logits, x, a, sm_count, stream);
  }
}

cudaError_t launchTokenLogProbsBackward(const void* logits, const LogitRows& x, void* grad, const TokenLogProbsGrads& a,
                                        cudaStream_t stream) {
  if (x.rows <= 0) return cudaSuccess;
  if (x.vocab <= 0 || x.rows > INT32_MAX) return cudaErrorInvalidValue;
  // A vector of the logits becomes a vector of the gradient.
  if ((reinterpret_cast<uintptr_t>(logits) ^ reinterpret_cast<uintptr_t>(grad)) & 15u) return cudaErrorMisalignedAddress;
  switch (x.type) {
    case LogitType::kBFloat16: return backwardOf<__nv_bfloat16>(logits, x, grad, a, stream);
    case LogitType::kHalf: return backwardOf<__half>(logits, x, grad, a, stream);
    default: return backwardOf<float>(logits, x, grad, a, stream);
  }
}

}  // namespace fairring
