// Log probabilities of given tokens under the softmax of a row of logits, the distribution's entropy and its
// largest entries (sm_100a); the gradient of the first two.
//
// With z = x / T, m and S of softmax_row.cuh:  log p_v = (z_v - max z) - log S,  H = log S - A ln 2 / S, a sum of two
// terms that are not negative.  Backward:  dx_v = 1/T [ g (1[v = t] - p_v) - h p_v (log p_v + H) ].
//
// Forward one read of the logits, backward one read and one write.  4 x 1024 x 51200 bf16 with the
// entropy, a quarter of the rows not counting: forward 68 us, backward 120 (6.1 TB/s; both together
// 163 us at the copy rate); 8192 x 51200 with the 64 largest entries 188 us (131 at the copy rate).
#include <cfloat>
#include <cmath>

#include "softmax_row.cuh"

namespace fairring {
namespace {

using namespace softmax_row;

constexpr int kMostTop = kMostTopTokens;
constexpr int kGroups = 8;    // largest values that a sweeping thread leaves of a row
constexpr int kQueue = 512;   // groups of columns that are looked into
constexpr int kList = 1024;   // candidates that are ranked
constexpr int kShortList = 256;  // of a row that one warp has
static_assert(kList >= kMostSlices * kMostTop, "the slices' results are candidates");

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

// Where the entries that are asked for are found: the sweep leaves the largest value of every thread's groups of columns, from these
// comes a bound, and only the groups that reach it are read again, from L2.  It is the block's own work, with the row's
// candidates in shared memory, five blocks a multiprocessor.  2048 rows of 51200 bf16 logits: 41.8 million instructions of a warp with 64
// entries, 35.8 with one, 25.0 for the log probabilities alone.  Warps of blocks that stay doing this behind the sweep were
// slower (274 us and more against 220 then), and so was keeping vectors above a bound while sweeping (245 against 208).
struct Groups {
  float top[kGroups][kThreads];
};
// Of kWidth threads, a block's or a warp's.
template <int kEntries> struct Candidates {
  alignas(16) uint64_t list[kEntries];
  uint64_t best[kMostTop];  // the result, in falling order
  unsigned hist[256];
  unsigned listed, digit, left;
};
struct TopWork : Candidates<kList> {
  int queue[kQueue];
  float bound[kWarps];
  unsigned above[kWarps], queued;
};

// Falling order of 32 values, one per lane.
__device__ __forceinline__ float sortedLanes(float v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size *= 2)
#pragma unroll
    for (int step = size / 2; step > 0; step /= 2) {
      const float o = __shfl_xor_sync(kAll, v, step);
      const bool larger = ((lane & step) == 0) == (size == 32 || (lane & size) == 0);
      v = larger ? fmaxf(v, o) : fminf(v, o);
    }
  return v;
}

// While a row is swept every thread leaves the largest value of each of its groups: what it has of one batch, or of `span`
// batches that follow one another in a row of more than kGroups.
struct TopHook {
  static constexpr int kUnroll = 2;  // no copies of the batch that has arrived: 194 -> 188 us; the other kernels lose by it
  Groups* groups;
  int span, g = 0, in = 0;
  float top = -INFINITY;
  template <typename T> static __device__ __forceinline__ int batches(const Slice<T>& sl) {
    return (sl.v1 - sl.v0 + kBatch * kThreads - 1) / (kBatch * kThreads);
  }
  template <typename T> static __device__ __forceinline__ int spanOf(const Slice<T>& sl) {
    return max(1, (batches(sl) + kGroups - 1) / kGroups);
  }
  template <typename T>
  __device__ __forceinline__ float batch(const uint4 (&now)[kBatch], bool first, int, const Slice<T>& sl) {
    if (first) span = spanOf(sl);
    const float largest = batchMax<T>(now);
    top = fmaxf(top, largest);
    if (++in == span) {
      groups->top[g][threadIdx.x] = top;
      ++g;
      in = 0;
      top = -INFINITY;
    }
    return largest;
  }
  __device__ __forceinline__ void end() {
    if (in > 0) groups->top[g][threadIdx.x] = top;
  }
};

// The `want` largest of the first n entries of the list, in falling order, to `best`.
template <int kWidth, int kEntries> __device__ __forceinline__ void rankList(Candidates<kEntries>& work, int n, int want) {
  const int tid = threadIdx.x % kWidth;
  uint64_t* list = work.list;
  if (n <= (kWidth == 32 ? 64 : 2 * kWidth)) {  // every entry counts those above it, two threads an entry where there are threads enough
    if (tid == 0 && (n & 1)) list[n] = 0;
    if (n & 1) syncWidth<kWidth>();
    const bool split = 2 * n <= kWidth;
    const int pairs = (n + 1) / 2, from = split && (tid & 1) ? pairs / 2 : 0, to = split && !(tid & 1) ? pairs / 2 : pairs;
    for (int i = split ? tid / 2 : tid; i < (split ? kWidth / 2 : (n + 31) / 32 * 32); i += kWidth) {
      const uint64_t mine = i < n ? list[i] : 0;
      int above = 0;
#pragma unroll 4
      for (int j = from; j < to; ++j) {
        const ulonglong2 two = reinterpret_cast<const ulonglong2*>(list)[j];
        above += two.x > mine;
        above += two.y > mine;
      }
      if (split) above += __shfl_xor_sync(kAll, above, 1);
      if (i < n && above < want) work.best[above] = mine;
    }
    syncWidth<kWidth>();
    return;
  }
  int size = 2;
  while (size < n) size *= 2;
  for (int i = n + tid; i < size; i += kWidth) list[i] = 0;
  syncWidth<kWidth>();
  for (int block = 2; block <= size; block *= 2)
    for (int step = block / 2; step > 0; step /= 2) {
      for (int i = tid; i < size / 2; i += kWidth) {
        const int a = 2 * i - (i & (step - 1)), b = a + step;
        const uint64_t x = list[a], y = list[b];
        if ((x < y) == ((a & block) == 0)) list[a] = y, list[b] = x;
      }
      syncWidth<kWidth>();
    }
  for (int i = tid; i < want; i += kWidth) work.best[i] = list[i];
  syncWidth<kWidth>();
}

// The `want` largest of the slice's entries, to the list in any order, by a radix select that reads the slice six
// times and more: for rows where the bound lets too much pass (ties, rising logits) and those with NaN.
template <int kWidth, typename T, int kEntries>
__device__ __noinline__ void selectExactly(const Slice<T>& sl, int want, Candidates<kEntries>& work) {
  const int tid = threadIdx.x % kWidth, lane = threadIdx.x & 31;
  uint32_t prefix = 0;
  unsigned left = want;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += kWidth) work.hist[i] = 0;
    syncWidth<kWidth>();
    for (int col = sl.c0 + tid; col < sl.c1; col += kWidth) {
      const uint32_t key = keyOf(toFloat(sl.row[col]));
      if (shift == 24 || key >> (shift + 8) == prefix) atomicAdd(&work.hist[key >> shift & 255u], 1u);
    }
    syncWidth<kWidth>();
    if (tid == 0) {
      int digit = 255;
      unsigned more = left;
      while (digit > 0 && work.hist[digit] < more) more -= work.hist[digit--];
      work.digit = digit;
      work.left = more;
    }
    syncWidth<kWidth>();
    prefix = prefix << 8 | work.digit;
    left = work.left;
    syncWidth<kWidth>();
  }
  // `prefix` is the key of the last one; `left` of those that equal it are taken, the first ones.
  if (tid == 0) work.listed = 0;
  syncWidth<kWidth>();
  for (int col = sl.c0 + tid; col < sl.c1; col += kWidth) {
    const float v = toFloat(sl.row[col]);
    if (keyOf(v) > prefix) work.list[atomicAdd(&work.listed, 1u)] = entryOf(v, col);
  }
  const unsigned larger = want - left;
  unsigned taken = 0;
  for (int base = sl.c0; base < sl.c1 && taken < left; base += kWidth) {
    const int col = base + tid;
    const float v = col < sl.c1 ? toFloat(sl.row[col]) : 0.f;
    const bool equal = col < sl.c1 && keyOf(v) == prefix;
    const unsigned votes = __ballot_sync(kAll, equal);
    syncWidth<kWidth>();
    if (lane == 0) work.hist[tid >> 5] = __popc(votes);
    syncWidth<kWidth>();
    unsigned before = taken + __popc(votes & ((1u << lane) - 1u)), all = 0;
    for (int w = 0; w < kWidth / 32; ++w) {
      if (w < tid >> 5) before += work.hist[w];
      all += work.hist[w];
    }
    if (equal && before < left) work.list[larger + before] = entryOf(v, col);
    taken += all;
  }
  syncWidth<kWidth>();
}

// The slice's largest entries, at most k, in falling order, to `best`, zeros behind them up to k.  The sweep is over for all of the
// block, and work.queued, work.listed and work.above are 0.
//
// If k of the threads' largest values are as large as `bound`, k values of the slice are.  Each of w warps sorts those of its threads
// and gives its r-th, r = ceil(k / w): that many are as large as the smallest of these, and the largest of them that k values
// reach is the bound.  Groups below it are out, a hundred or two of the 2048 are looked into again, and what they have above the bound, again a hundred or
// two values, is ranked.
template <typename T>
__device__ __forceinline__ void sliceTop(const Slice<T>& sl, int k, bool nan, const Groups& groups, TopWork& work) {
  constexpr int E = Vec<T>::kElems;
  const int tid = threadIdx.x, lane = tid & 31, want = min(k, sl.c1 - sl.c0);
  const int batches = TopHook::batches(sl), span = TopHook::spanOf(sl), number = (batches + span - 1) / span;
  float value[kGroups], top = -INFINITY;
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    value[g] = g < number ? groups.top[g][tid] : -INFINITY;
    top = fmaxf(top, value[g]);
  }
  const int warps = min(kWarps, (sl.v1 - sl.v0) / 32), of_each = warps > 0 ? (k + warps - 1) / warps : k;  // warps that are all at work
  const float mine = __shfl_sync(kAll, sortedLanes(top), (of_each - 1) & 31);
  if (lane == 0) work.bound[tid >> 5] = tid >> 5 < warps ? mine : INFINITY;
  __syncthreads();
  unsigned above = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const unsigned votes = __ballot_sync(kAll, top >= work.bound[w]);
    if (lane == w) above = __popc(votes);
  }
  if (lane < kWarps) atomicAdd(&work.above[lane], above);
  __syncthreads();
  float bound = -FLT_MAX;
#pragma unroll
  for (int w = 0; w < kWarps; ++w)
    if ((int)work.above[w] >= k) bound = fmaxf(bound, work.bound[w]);
  // (minus infinity is left to the other way)
  // A thread's groups side by side in the queue, those of a warp after one addition to its length.
  unsigned pass = 0;
#pragma unroll
  for (int g = 0; g < kGroups; ++g) pass |= value[g] >= bound ? 1u << g : 0u;
  int pos = __popc(pass);
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int below = __shfl_up_sync(kAll, pos, o);
    if (lane >= o) pos += below;
  }
  int at = 0;
  if (lane == 31) at = atomicAdd(&work.queued, (unsigned)pos);
  pos += __shfl_sync(kAll, at, 31) - __popc(pass);
  for (; pass != 0; pass &= pass - 1, ++pos) {
    if (pos < kQueue) work.queue[pos] = (__ffs(pass) - 1) * kThreads + tid;
  }
  __syncthreads();
  const int queued = work.queued;
  const bool fits = queued <= kQueue;
  const uint4* all = reinterpret_cast<const uint4*>(sl.row + sl.head);
  // kBatch threads a group, one for each of the vectors that a batch has of it; two rounds of groups at once.
  constexpr int kRound = kThreads / kBatch, kAhead = 2;
  for (int first = 0; first < queued && fits; first += kAhead * kRound)
    for (int batch = 0; batch < span; ++batch) {
      uint4 raw[kAhead];
      int vec[kAhead];
#pragma unroll
      for (int s = 0; s < kAhead; ++s) {
        const int q = first + s * kRound + tid / kBatch;
        vec[s] = sl.v1;
        if (q < queued) {
          const int id = work.queue[q];
          vec[s] = sl.v0 + ((id / kThreads * span + batch) * kBatch + tid % kBatch) * kThreads + id % kThreads;
        }
        constexpr uint32_t w = Vec<T>::kMinusInf;
        raw[s] = vec[s] < sl.v1 ? all[vec[s]] : make_uint4(w, w, w, w);  // swept not long ago: from L2
      }
#pragma unroll
      for (int s = 0; s < kAhead; ++s) {
        if (first + s * kRound >= queued) break;
        float2 v[E / 2];
        Vec<T>::get(raw[s], v);
        unsigned mask = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) mask |= (e & 1 ? v[e / 2].y : v[e / 2].x) >= bound ? 1u << e : 0u;
        for (;;) {  // a value of every lane that has one
          const unsigned votes = __ballot_sync(kAll, mask != 0);
          if (votes == 0) break;
          unsigned pos = 0;
          if (lane == 0) pos = atomicAdd(&work.listed, (unsigned)__popc(votes));
          pos = __shfl_sync(kAll, pos, 0) + __popc(votes & ((1u << lane) - 1u));
          if (mask != 0 && pos < kList) {
            const int col = sl.head + vec[s] * E + __ffs(mask) - 1;
            work.list[pos] = entryOf(toFloat(sl.row[col]), col);
          }
          mask &= mask - 1;
        }
      }
    }
  const int loose = tid < 2 * E ? sl.looseCol(tid) : -1;
  if (loose >= 0) {
    const float v = toFloat(sl.row[loose]);
    const unsigned pos = v >= bound ? atomicAdd(&work.listed, 1u) : kList;
    if (pos < kList) work.list[pos] = entryOf(v, loose);
  }
  __syncthreads();
  int n = work.listed;
  __syncthreads();
  if (nan || !fits || n > kList || n < want) {
    if (want > 0) selectExactly<kThreads>(sl, want, work);
    n = want;
  }
  for (int i = want + tid; i < k; i += kThreads) work.best[i] = 0;
  rankList<kThreads>(work, n, want);
}

// The k largest of the row from the slices' results, in block 0.  clusterSums() has waited for those.
__device__ __forceinline__ void clusterTop(int k, TopWork& work) {
  namespace cg = cooperative_groups;
  const cg::cluster_group cluster = cg::this_cluster();
  const int slices = cluster.num_blocks();
  if (cluster.block_rank() != 0) return;
  for (int i = threadIdx.x; i < slices * k; i += kThreads) {
    const int r = i / k;
    work.list[i] = cluster.map_shared_rank(&work, r)->best[i - r * k];
  }
  __syncthreads();
  rankList<kThreads>(work, slices * k, k);
}

// The same for a row that one warp has.  Its groups are `span` of a lane's vectors, a power of two.
struct WarpTopHook {
  static constexpr int kUnroll = 1;
  float (*groups)[32];
  int span = 1, at = 0;  // `at`: the vector that comes next
  float top = -INFINITY;
  template <typename T> static __device__ __forceinline__ int vectors(const Slice<T>& sl) { return (sl.v1 - sl.v0 + 31) / 32; }
  template <typename T> static __device__ __forceinline__ int spanOf(const Slice<T>& sl) {
    int span = 1;
    while (span * kGroups < vectors(sl)) span *= 2;
    return span;
  }
  template <typename T> __device__ __forceinline__ float batch(const uint4 (&now)[kBatch], bool first, int, const Slice<T>& sl) {
    const int lane = threadIdx.x & 31;
    if (first) span = spanOf(sl);
    float m[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) m[u] = Vec<T>::max(now[u]);
    const float low = fmaxf(m[0], m[1]), high = fmaxf(m[2], m[3]), largest = fmaxf(low, high);
    if (span >= kBatch) {
      top = fmaxf(top, largest);
      if ((at + kBatch) % span == 0) groups[at / span][lane] = top, top = -INFINITY;
    } else if (span == 2) {
      groups[at / 2][lane] = low;
      groups[at / 2 + 1][lane] = high;
    } else {
#pragma unroll
      for (int u = 0; u < kBatch; ++u) groups[at + u][lane] = m[u];
    }
    at += kBatch;
    return largest;
  }
  __device__ __forceinline__ void end() {
    if (at % span != 0) groups[at / span][threadIdx.x & 31] = top;
  }
};
static_assert(kBatch == 4 && kGroups == 8, "a batch is one group, two, or a part of one");

// Its k largest entries.  The bound is the k-th of the lanes' largest, or for more entries the best of the groups' as the warps' above.
constexpr int kFew = 24;  // 20 entries of 8192 x 1000: 18 us so, 23 by the groups
template <typename T>
__device__ __forceinline__ void warpTop(const Slice<T>& sl, int k, bool nan, const float (*groups)[32], Candidates<kShortList>& work) {
  constexpr int E = Vec<T>::kElems;
  const int lane = threadIdx.x & 31, vectors = WarpTopHook::vectors(sl), span = WarpTopHook::spanOf(sl);
  const int number = (vectors + span - 1) / span, at_work = (sl.v1 - sl.v0) / 32;  // vectors that every lane has
  float value[kGroups], top = -INFINITY;
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    value[g] = g < number ? groups[g][lane] : -INFINITY;
    top = fmaxf(top, value[g]);
  }
  float bound = -FLT_MAX;
  if (k <= kFew) {
    if (at_work > 0) bound = fmaxf(bound, __shfl_sync(kAll, sortedLanes(top), k - 1));
  } else {
    const int full = (at_work + span - 1) / span, of_each = full > 0 ? (k + full - 1) / full : 33;
#pragma unroll 1
    for (int g = 0; g < full && of_each <= 32; ++g) {
      const float mine = __shfl_sync(kAll, sortedLanes(groups[g][lane]), of_each - 1);
      int above = 0;
#pragma unroll
      for (int h = 0; h < kGroups; ++h) above += __popc(__ballot_sync(kAll, value[h] >= mine));
      if (above >= k) bound = fmaxf(bound, mine);
    }
  }
  // Every lane looks again into its own groups that reach the bound.
  const uint4* all = reinterpret_cast<const uint4*>(sl.row + sl.head);
  int listed = 0;
  auto list = [&](unsigned mask, auto colOf) {
    int pos = __popc(mask);
    if (!__any_sync(kAll, mask != 0)) return;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int below = __shfl_up_sync(kAll, pos, o);
      if (lane >= o) pos += below;
    }
    const int found = __shfl_sync(kAll, pos, 31);
    for (pos += listed - __popc(mask); mask != 0; mask &= mask - 1, ++pos) {
      const int col = colOf(__ffs(mask) - 1);
      if (pos < kShortList) work.list[pos] = entryOf(toFloat(sl.row[col]), col);
    }
    listed += found;
    __syncwarp();
  };
#pragma unroll 1
  for (int b = 0; b < vectors; b += kBatch) {
    bool pass[kBatch], any = false;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      pass[u] = b + u < vectors && sl.v0 + (b + u) * 32 + lane < sl.v1 && groups[(b + u) / span][lane] >= bound;
      any |= pass[u];
    }
    if (!__any_sync(kAll, any)) continue;
    uint4 raw[kBatch];
    constexpr uint32_t w = Vec<T>::kMinusInf;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) raw[u] = pass[u] ? all[sl.v0 + (b + u) * 32 + lane] : make_uint4(w, w, w, w);
    unsigned mask = 0;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      float2 v[E / 2];
      Vec<T>::get(raw[u], v);
#pragma unroll
      for (int e = 0; e < E; ++e) mask |= (e & 1 ? v[e / 2].y : v[e / 2].x) >= bound ? 1u << (u * E + e) : 0u;
    }
    list(mask, [&](int bit) { return sl.head + (sl.v0 + (b + bit / E) * 32 + lane) * E + bit % E; });
  }
  const int loose = lane < 2 * E ? sl.looseCol(lane) : -1;
  list(loose >= 0 && toFloat(sl.row[loose]) >= bound ? 1u : 0u, [&](int) { return loose; });
  int n = listed;
  if (nan || n > kShortList || n < k) {
    selectExactly<32>(sl, k, work);
    n = k;
  }
  rankList<32>(work, n, k);
}

// What one row leaves; any pointer but `tokens` may be null.  Kept for the backward: m and S as its exponents need it, which is
// -1 where the row does not count and NaN where its token is none.
struct Outputs {
  const int64_t* tokens;
  float* log_probs;
  float* entropy;
  float2* stats;
  int k;
  float* top_log_probs;
  int64_t* top_tokens;

  __device__ __forceinline__ void skipped(int64_t r) const {  // by one thread
    if (log_probs != nullptr) log_probs[r] = 0.f;
    if (entropy != nullptr) entropy[r] = 0.f;
    if (stats != nullptr) stats[r] = make_float2(0.f, -1.f);
    for (int i = 0; i < k; ++i) {
      top_log_probs[r * k + i] = -INFINITY;
      top_tokens[r * k + i] = -1;
    }
  }
  // By one thread: what stays if nobody comes to finish the row.
  __device__ __forceinline__ void broken(int64_t r) const {
    const float nan = __int_as_float(0x7fffffff);
    if (log_probs != nullptr) log_probs[r] = nan;
    if (entropy != nullptr) entropy[r] = nan;
    if (stats != nullptr) stats[r] = make_float2(0.f, nan);
  }
  // By one thread; `logit` is the token's.
  template <bool kEntropy>
  __device__ __forceinline__ void values(int64_t r, const Sums& acc, bool known, float logit, float c, float inv_t) const {
    const float low = logf(acc.s), nan = __int_as_float(0x7fffffff);
    if (log_probs != nullptr) log_probs[r] = known ? fmaf(logit - acc.m, inv_t, -low) : nan;
    if (kEntropy) entropy[r] = low - acc.a / acc.s * kLn2;
    if (stats != nullptr) stats[r] = make_float2(acc.m, known ? acc.s * exp2Of(Exponent::excess(acc.m, c)) : nan);
  }
  // By a block or a warp.
  template <int kWidth> __device__ __forceinline__ void largest(int64_t r, const Sums& acc, const uint64_t* best, float inv_t) const {
    const float low = logf(acc.s);
    for (int i = (int)threadIdx.x % kWidth; i < k; i += kWidth) {
      const uint64_t entry = best[i];
      top_log_probs[r * k + i] = fmaf(valueOf((uint32_t)(entry >> 32)) - acc.m, inv_t, -low);
      top_tokens[r * k + i] = (int)~(uint32_t)entry;
    }
  }
};

struct TopSlices {
  TopWork work;
  Groups groups;
};

// Few rows: one per cluster.
template <typename T, bool kEntropy, bool kTop>
__global__ void __launch_bounds__(kThreads, kTop ? 5 : 4)
token_log_probs_slices_kernel(const T* __restrict__ logits, LogitRows x, Outputs out, float c, float inv_t) {
  namespace cg = cooperative_groups;
  extern __shared__ __align__(16) unsigned char dynamic[];
  __shared__ Sums scratch[kWarps], mine;
  const cg::cluster_group cluster = cg::this_cluster();
  const int slices = cluster.num_blocks(), rank = cluster.block_rank();
  const int64_t r = blockIdx.x / slices;
  const int64_t t = out.tokens != nullptr ? out.tokens[r] : 0;
  if (t < 0) {
    if (rank == 0 && threadIdx.x == 0) out.skipped(r);
    return;
  }
  const Slice<T> sl(rowOf(x, logits, r), x.vocab, rank, slices);
  const bool known = t < x.vocab;
  float logit = 0.f;
  if (rank == 0 && threadIdx.x == 0 && known) logit = toFloat(sl.row[t]);
  Sums acc;
  TopSlices* top = reinterpret_cast<TopSlices*>(dynamic);
  if constexpr (kTop) {
    TopHook hook;
    hook.groups = &top->groups;
    if (threadIdx.x == 0) top->work.listed = top->work.queued = 0;
    if (threadIdx.x < kWarps) top->work.above[threadIdx.x] = 0;
    acc = scan<T, kEntropy, kThreads>(sl, c, hook);
    hook.end();
  } else {
    NoHook none;
    acc = scan<T, kEntropy, kThreads>(sl, c, none);
  }
  if (threadIdx.x < 2 * Vec<T>::kElems) {
    const int col = sl.looseCol(threadIdx.x);
    if (col >= 0) acc.add<kEntropy>(toFloat(sl.row[col]), c);
  }
  acc = blockSums<kEntropy>(acc, c, scratch);
  if constexpr (kTop) sliceTop(sl, out.k, acc.s != acc.s, top->groups, top->work);
  if (slices > 1) {
    acc = clusterSums<kEntropy>(acc, c, &mine);
    if constexpr (kTop) clusterTop(out.k, top->work);
    clusterDone();
    if (rank != 0) return;
  }
  if (!acc.template settle<kEntropy>(c)) acc = blockAgain<T, kEntropy>(sl.row, x.vocab, c, scratch, LeaveNone());
  if (threadIdx.x == 0) out.values<kEntropy>(r, acc, known, logit, c, inv_t);
  if constexpr (kTop) out.template largest<kThreads>(r, acc, top->work.best, inv_t);
}

// Many short rows: one per warp.
struct ShortTop {
  Candidates<kShortList> work;
  float groups[kGroups][32];
};
template <typename T, bool kEntropy, bool kTop>
__global__ void __launch_bounds__(kThreads, 4)
token_log_probs_short_kernel(const T* __restrict__ logits, LogitRows x, Outputs out, float c, float inv_t) {
  extern __shared__ __align__(16) unsigned char dynamic[];
  const int lane = threadIdx.x & 31;
  const int64_t r = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (r >= x.rows) return;
  const int64_t t = out.tokens != nullptr ? out.tokens[r] : 0;
  if (t < 0) {
    if (lane == 0) out.skipped(r);
    return;
  }
  const Slice<T> sl(rowOf(x, logits, r), x.vocab, 0, 1);
  const bool known = t < x.vocab;
  const float logit = known ? toFloat(sl.row[t]) : 0.f;
  ShortTop* top = reinterpret_cast<ShortTop*>(dynamic) + (threadIdx.x >> 5);
  Sums acc;
  if constexpr (kTop) {
    WarpTopHook hook;
    hook.groups = top->groups;
    acc = scan<T, kEntropy, 32>(sl, c, hook);
    hook.end();
  } else {
    NoHook none;
    acc = scan<T, kEntropy, 32>(sl, c, none);
  }
  const int col = lane < 2 * Vec<T>::kElems ? sl.looseCol(lane) : -1;
  if (col >= 0) acc.add<kEntropy>(toFloat(sl.row[col]), c);
  acc = warpSums<kEntropy>(acc, c);
  if constexpr (kTop) warpTop(sl, out.k, acc.s != acc.s, top->groups, top->work);
  if (!acc.template settle<kEntropy>(c)) acc = warpAgain<T, kEntropy>(sl.row, x.vocab, c, LeaveNone());
  if (lane == 0) out.values<kEntropy>(r, acc, known, logit, c, inv_t);
  if constexpr (kTop) out.template largest<32>(r, acc, top->work.best, inv_t);
}

// One warp is slow with long rows and many entries, but a multiprocessor has 32 of them: up to 1 KB for each row that a
// multiprocessor gets, and 24 KB.  bf16, 20 entries: 8192 x 1000 85 -> 18 us, 8192 x 8000 94 -> 62, 2500 x 4000 29 -> 18,
// 600 x 1000 10 -> 6; but 8192 x 16000 110 -> 118, 1200 x 8000 17 -> 26.  More entries than 64 overflow a warp's list where
// rows are not short (8192 x 8000, 128 entries: 165 -> 341).
inline bool shortTop(const LogitRows& x, int k, int elem_size, int sm_count) {
  const int64_t bytes = (int64_t)x.vocab * elem_size;
  return k <= 64 && manyRows(x.rows, sm_count) && bytes <= 24 * 1024 && bytes <= 1024 * (x.rows / sm_count);
}

// Many rows: the blocks stay.
struct Rows {
  Ring ring;
  HandOver hand;
};
template <typename T, bool kEntropy>
__global__ void __launch_bounds__(kRowThreads, 3)
token_log_probs_rows_kernel(const T* __restrict__ logits, LogitRows x, Outputs out, float c, float inv_t, int rows_a_block) {
  extern __shared__ __align__(16) unsigned char dynamic[];
  Rows& shared = *reinterpret_cast<Rows*>(dynamic);
  HandOver& hand = shared.hand;
  if (threadIdx.x == 0) hand.init();
  __syncthreads();
  const int64_t* tokens = out.tokens;
  if (threadIdx.x < kThreads) {
    NoHook none;
    sweepRows<T, kEntropy>(logits, x, c, shared.ring, hand, none);
    return;
  }
  const int lane = threadIdx.x & 31;
  if (threadIdx.x < kThreads + 32) {
    fetchRows(
        [&](int r) { return tokens == nullptr || tokens[r] >= 0; }, x.rows, rows_a_block, hand, [&](int r) { out.skipped(r); },
        [&](int r) { out.broken(r); }, [](int, const Place&) { return true; }, [](int, const Place&) {});
    return;
  }
  finishRows(hand, [&](int r, const Place& at) {
    const Slice<T> sl(rowOf(x, logits, r), x.vocab, 0, 1);
    const int64_t t = tokens != nullptr ? tokens[r] : 0;
    const bool known = t < x.vocab;
    const float logit = known ? toFloat(sl.row[t]) : 0.f;
    if (!hand.wait(&hand.full[at.slot], at.parity)) return;
    Sums acc = hand.template take<T, kEntropy>(at.slot, sl, c, 0);
    if (!acc.template settle<kEntropy>(c)) acc = warpAgain<T, kEntropy>(sl.row, x.vocab, c, LeaveNone());
    if (lane == 0) out.values<kEntropy>(r, acc, known, logit, c, inv_t);
  });
}

// A warp does one batch of vectors of one row, so that all are alike whatever the vocabulary; a
// block a batch of 16 KB left threads idle at the row's end: 4 x 1024 x 51200 125 -> 121 us, 8192 x
// 8200 bf16 58 -> 44, 8192 x 1000 22 -> 7.  Six blocks a multiprocessor (40 registers, of which
// types of 16 bits spill three, one with the entropy); with five (48, no spills) 8192 x 20000 fp32
// takes 190 us for 187, 4096 x 51200 fp16 126 for 123, 8192 x 51200 bf16 247 for 246, 8192 x 1000
// bf16 5.7 for 6.5, all without the entropy.
template <typename T, bool kEntropy>
__global__ void __launch_bounds__(kThreads, 6)
token_log_probs_bwd_kernel(const T* __restrict__ logits, LogitRows x, T* __restrict__ grad,
                           const int64_t* __restrict__ tokens, const float2* __restrict__ stats,
                           const float* __restrict__ entropy, const float* __restrict__ g_log_probs, int64_t g_stride,
                           const float* __restrict__ g_entropy, int64_t h_stride, float c, float inv_t, Pieces pieces) {
  constexpr int E = Vec<T>::kElems, U = kBatch, kWidth = 32;
  const int tid = threadIdx.x % kWidth;
  const unsigned w = pieces.mine();
  if (w >= pieces.total) return;
  const int64_t r = w / pieces.a_row;
  const int piece = (int)(w % pieces.a_row);
  const T* row = rowOf(x, logits, r);
  T* out = rowOf(x, grad, r);
  const RowParts<T> parts(row, x.vocab);
  const int first = piece * U * kWidth + tid;
  const uint4* vecs = reinterpret_cast<const uint4*>(row + parts.head);
  uint4* vout = reinterpret_cast<uint4*>(out + parts.head);
  const float2 st = stats[r];
  const bool counts = !(st.y == -1.f);
  uint4 raw[U];
#pragma unroll
  for (int u = 0; u < U; ++u)
    raw[u] = counts && first + u * kWidth < parts.nvec ? __ldg(vecs + first + u * kWidth) : make_uint4(0, 0, 0, 0);
  const float g = g_log_probs != nullptr ? g_log_probs[r * g_stride] * inv_t : 0.f;
  const float h = kEntropy ? g_entropy[r * h_stride] * inv_t : 0.f;
  const int64_t t64 = tokens != nullptr ? tokens[r] : -1;
  const int t = t64 < x.vocab ? (int)t64 : -1;
  // g (1[v = t] - p) - h p (log p + H) with p = e / S and log p = u ln 2 - log S, u the exponent of e
  const float per_s = 1.f / st.y;
  const float a = -(kEntropy ? fmaf(h, entropy[r] - logf(st.y), g) : g) * per_s, b = -h * kLn2 * per_s;
  const Exponent exponent(st.x, c);
  auto of = [&](float2 v) {
    const float2 d = exponent(v), e = make_float2(exp2Of(d.x), exp2Of(d.y));
    if (!kEntropy) return mul2(e, make_float2(a, a));
    return mul2(e, fma2(make_float2(fmaxf(d.x, kLowExponent), fmaxf(d.y, kLowExponent)), make_float2(b, b), make_float2(a, a)));
  };
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = first + u * kWidth;
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
  if (piece == 0 && tid < 2 * E) {
    const int i = tid, col = i < parts.head ? i : i + parts.nvec * E;
    if (col < x.vocab)
      fromFloat(out + col, counts ? of(make_float2(toFloat(row[col]), 0.f)).x + (col == t ? g : 0.f) : 0.f);
  }
}

template <typename T, bool kEntropy>
cudaError_t forwardOf(const T* logits, const LogitRows& x, const Outputs& out, double temperature, int sm_count, cudaStream_t stream) {
  const float inv_t = (float)(1.0 / temperature), c = (float)(1.4426950408889634 / temperature);
  if (out.k == 0 && shortRows(x, sizeof(T), sm_count))
    return launchShort(token_log_probs_short_kernel<T, kEntropy, false>, x.rows, 0, stream, logits, x, out, c, inv_t);
  if (out.k > 0 && shortTop(x, out.k, sizeof(T), sm_count))
    return launchShort(token_log_probs_short_kernel<T, kEntropy, true>, x.rows, kWarps * sizeof(ShortTop), stream, logits, x, out, c, inv_t);
  if (out.k == 0 && manyRows(x.rows, sm_count)) {
    const int rows_a_block = rowsABlock(x, sizeof(T), sm_count);
    return launchRows(token_log_probs_rows_kernel<T, kEntropy>, x.rows, rows_a_block, sizeof(Rows), stream, logits, x, out, c, inv_t,
                      rows_a_block);
  }
  const int slices = slicesFor(x.rows, x.vocab, sizeof(T), sm_count);
  if (out.k > 0)
    return launchSlices(token_log_probs_slices_kernel<T, kEntropy, true>, x.rows, slices, kThreads,
                        sizeof(TopSlices), stream, logits, x, out, c, inv_t);
  return launchSlices(token_log_probs_slices_kernel<T, kEntropy, false>, x.rows, slices, kThreads, 0, stream, logits, x, out, c, inv_t);
}

template <typename T>
cudaError_t forwardOf(const void* logits, const LogitRows& x, const TokenLogProbsArgs& a, int sm_count, cudaStream_t stream) {
  const Outputs out{a.tokens, a.log_probs, a.entropy, reinterpret_cast<float2*>(a.stats), a.k, a.top_log_probs, a.top_tokens};
  const T* data = static_cast<const T*>(logits);
  return a.entropy != nullptr ? forwardOf<T, true>(data, x, out, a.temperature, sm_count, stream)
                              : forwardOf<T, false>(data, x, out, a.temperature, sm_count, stream);
}

template <typename T>
cudaError_t backwardOf(const void* logits, const LogitRows& x, void* grad, const TokenLogProbsGrads& a, cudaStream_t stream) {
  Pieces pieces;
  if (!pieces.template cut<T>(x)) return cudaErrorInvalidValue;
  const float inv_t = (float)(1.0 / a.temperature), c = (float)(1.4426950408889634 / a.temperature);
  auto run = [&](auto kernel) {
    return launchBlocks(kernel, pieces.blocks(), kThreads, 1, 0, stream, static_cast<const T*>(logits), x, static_cast<T*>(grad), a.tokens,
                        reinterpret_cast<const float2*>(a.stats), a.entropy, a.g_log_probs, a.g_stride, a.g_entropy, a.h_stride, c,
                        inv_t, pieces);
  };
  return a.g_entropy != nullptr ? run(token_log_probs_bwd_kernel<T, true>) : run(token_log_probs_bwd_kernel<T, false>);
}

}  // namespace

cudaError_t launchTokenLogProbs(const void* logits, const LogitRows& x, const TokenLogProbsArgs& a, int sm_count,
                                cudaStream_t stream) {
  if (x.rows <= 0) return cudaSuccess;
  if (x.vocab <= 0 || x.vocab > kMostVocab || x.rows > INT32_MAX || a.k < 0 || a.k > kMostTop || a.k > x.vocab) return cudaErrorInvalidValue;
  switch (x.type) {
    case LogitType::kBFloat16: return forwardOf<__nv_bfloat16>(logits, x, a, sm_count, stream);
    case LogitType::kHalf: return forwardOf<__half>(logits, x, a, sm_count, stream);
    default: return forwardOf<float>(logits, x, a, sm_count, stream);
  }
}

cudaError_t launchTokenLogProbsBackward(const void* logits, const LogitRows& x, void* grad, const TokenLogProbsGrads& a,
                                        cudaStream_t stream) {
  if (x.rows <= 0) return cudaSuccess;
  if (x.vocab <= 0 || x.vocab > kMostVocab || x.rows > INT32_MAX) return cudaErrorInvalidValue;
  // A vector of the logits becomes a vector of the gradient.
  if ((reinterpret_cast<uintptr_t>(logits) ^ reinterpret_cast<uintptr_t>(grad)) & 15u) return cudaErrorMisalignedAddress;
  switch (x.type) {
    case LogitType::kBFloat16: return backwardOf<__nv_bfloat16>(logits, x, grad, a, stream);
    case LogitType::kHalf: return backwardOf<__half>(logits, x, grad, a, stream);
    default: return backwardOf<float>(logits, x, grad, a, stream);
  }
}

}  // namespace fairring
