// Divergence of a student's distribution over the vocabulary from a teacher's largest log probabilities (sm_100a),
// forward and backward.
//
// The student is p = softmax(x / T).  Without the rest the teacher is q = softmax of its listed values / T, and
// L = sum q_k (log q_k - log p_k), dx_v = 1/T (p_v - q_v).  With it q_k = exp of the listed values, what they leave,
// q_r = 1 - sum q_k, is the probability of all tokens that are not listed, whose share of the student is p_r, and
// L = sum q_k (log q_k - log p_k) + q_r (log q_r - log p_r); with Q = q_r + sum q_k
//   dx_v = 1/T (Q p_v - q_v) for a listed token, 1/T (p_v / p_r) (Q p_r - q_r) for any other.
// p_r is summed from the tokens that are not listed: 1 - sum p_k would lose it where the teacher's tokens are likely.
#include "softmax_row.cuh"

namespace fairring {
namespace {

using namespace softmax_row;

static_assert(kMostTeacherTokens <= kThreads, "a thread per listed token");

struct Teacher {
  int token[kMostTeacherTokens];    // -1: padding
  float given[kMostTeacherTokens];  // the teacher's value
  float logit[kMostTeacherTokens];  // the student's
  float q[kMostTeacherTokens];
  bool first[kMostTeacherTokens];  // no entry before it names the same token
  double log_total;                // what turns the values into log probabilities
  double mass;                     // sum of q
};

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

// Takes the listed tokens' logits out of the sweep: one bit per column of the slice, a vector's bits in one byte.
struct RestHook {
  const unsigned char* bits;
  int shift;  // bit of the slice's column c0, so that a vector's bits start at a multiple of its length
  template <typename T> __device__ __forceinline__ unsigned of(int pos) const {
    return bits[pos >> 3] >> (pos & 7) & ((1u << Vec<T>::kElems) - 1u);
  }
  template <typename T> __device__ __forceinline__ void mask(uint4 (&now)[kBatch], int i, const Slice<T>& sl) {
    constexpr int E = Vec<T>::kElems;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int v = i + u * kThreads;
      if (v >= sl.v1) continue;
      const unsigned listed = of<T>(sl.head + v * E - sl.c0 + shift);
      if (listed == 0) continue;
      float2 x[E / 2];
      Vec<T>::get(now[u], x);
#pragma unroll
      for (int e = 0; e < E / 2; ++e) {
        if (listed >> (2 * e) & 1u) x[e].x = -INFINITY;
        if (listed >> (2 * e + 1) & 1u) x[e].y = -INFINITY;
      }
      now[u] = Vec<T>::set(x);
    }
  }
  template <typename V>
  __device__ __forceinline__ void batch(int, const uint4 (&)[kBatch], const float (&)[kBatch], float, int, const V&) {}
};

// The teacher's probabilities, by one warp.
template <bool kRest> __device__ __forceinline__ void teacherOf(Teacher& te, int k, float inv_t) {
  const int lane = threadIdx.x & 31;
  if constexpr (kRest) {
    double mass = 0;
    for (int i = lane; i < k; i += 32) {
      const float q = te.token[i] >= 0 ? expf(te.given[i]) : 0.f;
      te.q[i] = q;
      mass += q;
    }
    mass = warpSum(mass);
    if (lane == 0) te.mass = mass, te.log_total = 0;
  } else {
    float top = -INFINITY, total = 0.f;
    for (int i = lane; i < k; i += 32)
      if (te.token[i] >= 0) top = fmaxf(top, te.given[i]);
    top = warpMax(top);
    for (int i = lane; i < k; i += 32) {
      const float q = te.token[i] >= 0 ? expf((te.given[i] - top) * inv_t) : 0.f;
      te.q[i] = q;
      total += q;
    }
    total = warpSum(total);
    for (int i = lane; i < k; i += 32) te.q[i] /= total;
    if (lane == 0) te.mass = 1, te.log_total = (double)top * inv_t + log((double)total);
  }
}

// One row per cluster.  Kept for the backward: the maximum that its sweep takes differences from and the factor of
// those exponentials, the same for the listed tokens; the last is -1 where the row does not count.  The listed
// tokens with the probabilities of equal ones added up, each once, are written to `merged`.
template <typename T, bool kRest>
__global__ void __launch_bounds__(kThreads, 4)
distillation_fwd_kernel(const T* __restrict__ logits, LogitRows x, const int64_t* __restrict__ tokens,
                        const float* __restrict__ log_probs, int k, float c, double inv_t, float* __restrict__ loss,
                        float4* __restrict__ stats, int2* __restrict__ merged) {
  namespace cg = cooperative_groups;
  __shared__ Teacher te;
  __shared__ Sums scratch[kWarps], mine;
  extern __shared__ __align__(16) unsigned bits[];
  const cg::cluster_group cluster = cg::this_cluster();
  const int slices = cluster.num_blocks(), rank = cluster.block_rank();
  const int64_t r = blockIdx.x / slices;
  const int tid = threadIdx.x;
  const T* row = rowOf(x, logits, r);
  const Slice<T> sl(row, x.vocab, rank, slices);
  bool counts = false, outside = false;
  if (tid < k) {
    const int64_t t = tokens[r * k + tid];
    const float given = log_probs[r * k + tid];
    outside = t >= x.vocab;
    te.token[tid] = t < 0 || outside ? -1 : (int)t;
    te.given[tid] = given;
    counts = t >= 0 && (kRest || !(given == -INFINITY));
    if (rank == 0) te.logit[tid] = t < 0 || outside ? 0.f : toFloat(row[t]);
  }
  RestHook hook;
  if constexpr (kRest) {
    hook.bits = reinterpret_cast<const unsigned char*>(bits);
    hook.shift = (Vec<T>::kElems - (sl.firstCol() - sl.c0) % Vec<T>::kElems) % Vec<T>::kElems;
    for (int i = tid; i < (sl.c1 - sl.c0 + hook.shift + 31) / 32; i += kThreads) bits[i] = 0;
  }
  counts = __syncthreads_or(counts);
  outside = __syncthreads_or(outside);
  if (!counts) {
    if (rank == 0 && tid == 0) {
      loss[r] = 0.f;
      stats[r] = make_float4(0.f, 0.f, 0.f, -1.f);
    }
    return;
  }
  if constexpr (kRest) {
    if (tid < k) {
      const int t = te.token[tid], pos = t - sl.c0 + hook.shift;
      if (t >= sl.c0 && t < sl.c1) atomicOr(&bits[pos >> 5], 1u << (pos & 31));
    }
    __syncthreads();
  }
  if (rank == 0 && tid < 32) teacherOf<kRest>(te, k, (float)inv_t);
  Sums acc;
  if constexpr (kRest) {
    acc = scan<T, false>(sl, c, hook);
  } else {
    NoHook none;
    acc = scan<T, false>(sl, c, none);
  }
  if (tid < 2 * Vec<T>::kElems) {
    const int col = sl.looseCol(tid);
    bool listed = false;
    if constexpr (kRest) {
      const int pos = col - sl.c0 + hook.shift;
      listed = col >= 0 && (bits[pos >> 5] >> (pos & 31) & 1u);
    }
    if (col >= 0 && !listed) acc.add<false>(toFloat(row[col]), c);
  }
  acc = blockSums<false>(acc, c, scratch);
  if (slices > 1) {
    acc = clusterSums<false>(acc, c, &mine);
    clusterDone();
    if (rank != 0) return;
  }
  if (tid < k) {
    const int t = te.token[tid];
    float q = 0.f;
    bool first = t >= 0;
    for (int j = 0; j < k; ++j)
      if (te.token[j] == t) {
        q += te.q[j];
        first = first && j >= tid;
      }
    te.first[tid] = first;
    if (merged != nullptr) merged[r * k + tid] = make_int2(first ? t : -1, __float_as_int(q));
  }
  __syncthreads();
  if (tid >= 32) return;
  // All probabilities' maximum and sum; the sweep's are those of the rest.
  float m = acc.m, s = acc.s;
  if constexpr (kRest) {
    for (int i = tid; i < k; i += 32)
      if (te.first[i]) m = fmaxf(m, te.logit[i]);
    m = warpMax(m);
    float sum = 0.f;
    for (int i = tid; i < k; i += 32)
      if (te.first[i]) sum += exp2Of((te.logit[i] - m) * c);
    s = acc.s * exp2Of((acc.m - m) * c) + warpSum(sum);
  }
  // A divergence is a small difference of large logarithms: those are kept in 64 bits.
  const double lse = (double)m * inv_t + log((double)s);
  double sum = 0;
  for (int i = tid; i < k; i += 32) {
    const float q = te.q[i];
    if (te.token[i] >= 0 && !(q == 0.f)) {
      const double log_q = kRest ? (double)te.given[i] : (double)te.given[i] * inv_t - te.log_total;
      sum += q * (log_q - ((double)te.logit[i] * inv_t - lse));
    }
  }
  sum = warpSum(sum);
  if (tid != 0) return;
  const float nan = __int_as_float(0x7fffffff);
  if constexpr (kRest) {
    const double q_rest = 1.0 - te.mass < kLeastRest ? 0.0 : 1.0 - te.mass;  // NaN stays
    if (!(q_rest == 0)) sum += q_rest * (log(q_rest) - ((double)acc.m * inv_t + log((double)acc.s) - lse));
    const double all = te.mass + q_rest, p_rest = (double)(acc.s * exp2Of((acc.m - m) * c)) / s;
    const bool some = !(acc.s == 0.f);
    stats[r] = outside ? make_float4(nan, nan, nan, nan)
                       : make_float4(some ? acc.m : 0.f, some ? (float)((all * p_rest - q_rest) / acc.s) : 0.f, m, (float)(all / s));
  } else {
    stats[r] = outside ? make_float4(nan, nan, nan, nan) : make_float4(m, 1.f / s, m, 1.f / s);
  }
  loss[r] = outside ? nan : (float)sum;
}

__global__ void __launch_bounds__(1024)
distillation_mean_kernel(const float* __restrict__ loss, const float4* __restrict__ stats, int64_t rows,
                         float* __restrict__ mean, float* __restrict__ count) {
  __shared__ double sums[32], numbers[32];
  double s = 0, n = 0;
  for (int64_t r = threadIdx.x; r < rows; r += 1024) {
    s += loss[r];
    n += stats[r].w < 0.f ? 0 : 1;
  }
  s = warpSum(s);
  n = warpSum(n);
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = s, numbers[threadIdx.x >> 5] = n;
  __syncthreads();
  if (threadIdx.x >= 32) return;
  s = warpSum(sums[threadIdx.x]);
  n = fmax(warpSum(numbers[threadIdx.x]), 1.0);
  if (threadIdx.x == 0) {
    *mean = (float)(s / n);
    *count = (float)n;
  }
}

// A block does one batch of vectors of one row and then, over what it has written, the listed tokens among them.
template <typename T>
__global__ void __launch_bounds__(kThreads)
distillation_bwd_kernel(const T* __restrict__ logits, LogitRows x, T* grad, const float4* __restrict__ stats,
                        const int2* __restrict__ merged, int k, float c, float inv_t, const float* __restrict__ upstream,
                        int64_t stride, const float* __restrict__ count, int64_t pieces_total, int pieces) {
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
    const float4 st = stats[r];
    const bool counts = !(st.w < 0.f);
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      raw[u] = counts && first + u * kThreads < parts.nvec ? __ldg(vecs + first + u * kThreads) : make_uint4(0, 0, 0, 0);
    int2 mine = make_int2(-1, 0);
    float logit = 0.f;
    if (counts && (int)threadIdx.x < k) {
      mine = merged[r * k + threadIdx.x];
      const int v = (mine.x - parts.head) / E / (U * kThreads);
      const bool vector = mine.x >= parts.head && mine.x < parts.head + parts.nvec * E;
      if (mine.x >= 0 && (vector ? v : 0) != piece) mine.x = -1;
      if (mine.x >= 0) logit = toFloat(row[mine.x]);
    }
    const float up = upstream[r * stride] * inv_t, g = count != nullptr ? up / *count : up;
    const float f = st.y * g;
    auto of = [&](float2 v) {
      const float2 d = mul2(add2(v, make_float2(-st.x, -st.x)), make_float2(c, c));
      return mul2(make_float2(exp2Of(d.x), exp2Of(d.y)), make_float2(f, f));
    };
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = first + u * kThreads;
      if (i >= parts.nvec) continue;
      uint4 result = make_uint4(0, 0, 0, 0);
      if (counts) {
        float2 v[E / 2];
        Vec<T>::get(raw[u], v);
#pragma unroll
        for (int e = 0; e < E / 2; ++e) v[e] = of(v[e]);
        result = Vec<T>::set(v);
      }
      vout[i] = result;
    }
    if (piece == 0 && threadIdx.x < 2 * E) {
      const int i = threadIdx.x, col = i < parts.head ? i : i + parts.nvec * E;
      if (col < x.vocab) fromFloat(out + col, counts ? of(make_float2(toFloat(row[col]), 0.f)).x : 0.f);
    }
    if (counts) {
      __syncthreads();  // the block's stores before those of the listed tokens
      if (mine.x >= 0) fromFloat(out + mine.x, fmaf(exp2Of((logit - st.z) * c), st.w, -__int_as_float(mine.y)) * g);
    }
  }
}

template <typename T>
cudaError_t forwardOf(const void* logits, const LogitRows& x, const DistillationArgs& a, float* loss, float* stats,
                      void* merged, int sm_count, cudaStream_t stream) {
  const int slices = slicesFor(x.rows, x.vocab, sizeof(T), sm_count);
  const float c = (float)(1.4426950408889634 / a.temperature);
  auto run = [&](auto kernel, size_t shared) {
    return launchSlices(kernel, x.rows, slices, shared, stream, static_cast<const T*>(logits), x, a.tokens, a.log_probs, a.k,
                        c, 1.0 / a.temperature, loss, reinterpret_cast<float4*>(stats), static_cast<int2*>(merged));
  };
  if (!a.rest) return run(distillation_fwd_kernel<T, false>, 0);
  // The widest slice in whole vectors, its row's head and tail, and the shift of its first bit.
  constexpr int E = Vec<T>::kElems;
  const size_t shared = ((((int64_t)x.vocab / E + slices - 1) / slices * E + 3 * E) / 32 + 1) * 4;
  if (shared > 32 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(distillation_fwd_kernel<T, true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (int)shared);
    if (e != cudaSuccess) return e;
  }
  return run(distillation_fwd_kernel<T, true>, shared);
}

template <typename T>
cudaError_t backwardOf(const void* logits, const LogitRows& x, void* grad, const float* stats, const void* merged, int k,
                       double temperature, const float* upstream, int64_t stride, const float* count, cudaStream_t stream) {
  constexpr int per_piece = kThreads * kBatch * Vec<T>::kElems;
  const int pieces = (int)(((int64_t)x.vocab + per_piece - 1) / per_piece);
  const int64_t total = x.rows * pieces;
  const unsigned blocks = (unsigned)(total < (1 << 30) ? total : (1 << 30));
  distillation_bwd_kernel<T><<<blocks, kThreads, 0, stream>>>(
      static_cast<const T*>(logits), x, static_cast<T*>(grad), reinterpret_cast<const float4*>(stats),
      static_cast<const int2*>(merged), k, (float)(1.4426950408889634 / temperature), (float)(1.0 / temperature), upstream,
      stride, count, total, pieces);
  noteLocalLaunch();
  return cudaGetLastError();
}

}  // namespace

cudaError_t launchDistillation(const void* logits, const LogitRows& x, const DistillationArgs& a, float* loss, float* stats,
                               void* merged, int sm_count, cudaStream_t stream) {
  if (x.rows <= 0) return cudaSuccess;
  if (x.vocab <= 0 || x.rows > INT32_MAX || a.k <= 0 || a.k > kMostTeacherTokens || (a.rest && x.vocab > kMostRestVocab))
    return cudaErrorInvalidValue;
  switch (x.type) {
    case LogitType::kBFloat16: return forwardOf<__nv_bfloat16>(logits, x, a, loss, stats, merged, sm_count, stream);
    case LogitType::kHalf: return forwardOf<__half>(logits, x, a, loss, stats, merged, sm_count, stream);
    default: return forwardOf<float>(logits, x, a, loss, stats, merged, sm_count, stream);
  }
}

cudaError_t launchDistillationMean(const float* loss, const float* stats, int64_t rows, float* mean, float* count,
                                   cudaStream_t stream) {
  distillation_mean_kernel<<<1, 1024, 0, stream>>>(loss, reinterpret_cast<const float4*>(stats), rows, mean, count);
  noteLocalLaunch();
  return cudaGetLastError();
}

cudaError_t launchDistillationBackward(const void* logits, const LogitRows& x, void* grad, const float* stats,
                                       const void* merged, int k, double temperature, const float* upstream, int64_t stride,
                                       const float* count, cudaStream_t stream) {
  if (x.rows <= 0) return cudaSuccess;
  if (x.vocab <= 0 || x.rows > INT32_MAX || k <= 0 || k > kMostTeacherTokens) return cudaErrorInvalidValue;
  // A vector of the logits becomes a vector of the gradient.
  if ((reinterpret_cast<uintptr_t>(logits) ^ reinterpret_cast<uintptr_t>(grad)) & 15u) return cudaErrorMisalignedAddress;
  switch (x.type) {
    case LogitType::kBFloat16:
      return backwardOf<__nv_bfloat16>(logits, x, grad, stats, merged, k, temperature, upstream, stride, count, stream);
    case LogitType::kHalf:
      return backwardOf<__half>(logits, x, grad, stats, merged, k, temperature, upstream, stride, count, stream);
    default:
      return backwardOf<float>(logits, x, grad, stats, merged, k, temperature, upstream, stride, count, stream);
  }
}

}  // namespace fairring
