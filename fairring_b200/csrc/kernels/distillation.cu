// Divergence of a student's distribution over the vocabulary from a teacher's largest log probabilities (sm_100a),
// forward and backward.
//
// The student is p = softmax(x / T).  Without the rest the teacher is q = softmax of its listed values / T, and
// L = sum q_k (log q_k - log p_k), dx_v = 1/T (p_v - q_v).  With it q_k = exp of the listed values, what they leave,
// q_r = 1 - sum q_k, is the probability of all tokens that are not listed, whose share of the student is p_r, and
// L = sum q_k (log q_k - log p_k) + q_r (log q_r - log p_r); with Q = q_r + sum q_k
//   dx_v = 1/T (Q p_v - q_v) for a listed token, 1/T (p_v / p_r) (Q p_r - q_r) for any other.
// p_r is summed from the tokens that are not listed: 1 - sum p_k would lose it where the teacher's tokens are likely.
//
// Forward one read of the logits, backward one read and one write; the listed tokens' own logits
// are read apart, and their gradients written over those of the sweep.  8192 x 51200 bf16, 64
// tokens: forward 139 us, 149 while the last gradient is still written back from L2, backward 254
// (6.6 TB/s; both together 391 us at the copy rate); 2 x 1024 x 51200 with the rest 45 or 48 and 61
// (91).
#include "softmax_row.cuh"

namespace fairring {
namespace {

using namespace softmax_row;

// What the teacher says of one row, and the student of the tokens that it names.
struct Teacher {
  int token[kMostTeacherTokens];  // -1: padding or no token
  float q[kMostTeacherTokens];
  float logit[kMostTeacherTokens];
  bool first[kMostTeacherTokens];  // no entry before it names the same token
  float log_terms, total;          // sum of q log q is the first less the mass's share of log(total)
  bool outside;                    // a token is past the vocabulary
};

// What of the loss needs no sums: of the listed tokens sum q (log q + log total), the sum of q (x - ref), that of q, and with the
// rest the maximum and the sum of their own exponentials.  A divergence is a small difference of large logarithms: sums are taken of
// differences to the largest, and what those leave out is put together in 64 bits.
struct Listed {
  float log_terms, total, ref, from_ref, mass, m, s;
};

// Whether the bit was set before.
__device__ __forceinline__ bool setBit(unsigned* bits, unsigned at) {
  return atomicOr(&bits[at >> 5], 1u << (at & 31)) >> (at & 31) & 1u;
}

struct Given {
  const int64_t* tokens;
  const float* log_probs;
  int k;
};

// The columns that the sweep leaves out, for a second look at a row.  Every lane has some of the listed
// tokens, and those of a chunk are few: a look through all of them for each column took 52 ms where 2048
// rows of 51200 bf16 logits had all but the 64 listed ones masked.
struct LeaveListed {
  const Teacher* te;
  int k;
  __device__ __forceinline__ unsigned of(unsigned base) const {
    const unsigned lane = threadIdx.x & 31;
    unsigned out = 0;
    for (int first = 0; first < k; first += 32) {
      const int i = first + (int)lane;
      const unsigned at = i < k ? (unsigned)te->token[i] - base : kChunk;  // -1 is past every chunk
      for (unsigned hits = __ballot_sync(kAll, at < kChunk); hits != 0; hits &= hits - 1) {
        const unsigned col = __shfl_sync(kAll, at, __ffs(hits) - 1);
        if ((col & 31) == lane) out |= 1u << (col >> 5);
      }
    }
    return out;
  }
};

// Takes the listed tokens' logits out of the sweep: a bit for each column of the slice's vectors, so that the bits of what one
// thread has of a batch are one word (16 bits of fp32 logits), and a word for the columns outside the vectors.
template <typename T, int kWidth = kThreads> struct Marks {
  static constexpr int E = Vec<T>::kElems, kBits = kBatch * E;
  // Whole batches, and at least one: a row without a vector is swept as a batch of none.
  static constexpr __host__ __device__ __forceinline__ int words(int vecs) {
    const int batches = (vecs + kBatch * kWidth - 1) / (kBatch * kWidth);
    return (batches > 0 ? batches : 1) * kWidth * kBits / 32;
  }
  static __device__ __forceinline__ bool loose(const Slice<T>& sl, int col) { return col < sl.firstCol() || col >= sl.lastCol(); }
  static __device__ __forceinline__ unsigned looseBit(const Slice<T>& sl, int col) {
    return 1u << (col < sl.firstCol() ? col - sl.c0 : col - sl.lastCol() + sl.firstCol() - sl.c0);
  }
  static __device__ __forceinline__ unsigned place(const Slice<T>& sl, int col) {
    const unsigned v = (unsigned)(col - sl.firstCol()) / E, e = (unsigned)(col - sl.firstCol()) % E;
    return (v / (kBatch * kWidth) * kWidth + v % kWidth) * kBits + v / kWidth % kBatch * E + e;
  }
};
template <int kWidth> struct RestHook {
  static constexpr int kUnroll = 1;
  const unsigned* bits;
  // Those of what this thread has of batch b.
  template <typename T> __device__ __forceinline__ unsigned listed(int b) const {
    const int unit = b * kWidth + (int)threadIdx.x % kWidth;
    return Marks<T>::kBits == 32 ? bits[unit] : reinterpret_cast<const unsigned short*>(bits)[unit];
  }
  template <typename T> __device__ __forceinline__ float batch(uint4 (&now)[kBatch], bool, int i, const Slice<T>& sl) {
    constexpr int E = Vec<T>::kElems;
    const unsigned mine = listed<T>((i - sl.v0) / (kBatch * kWidth));
    if (__any_sync(kAll, mine != 0)) {
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        if (!__any_sync(kAll, (mine >> (u * E) & ((1u << E) - 1u)) != 0)) continue;
        float2 x[E / 2];
        Vec<T>::get(now[u], x);
#pragma unroll
        for (int e = 0; e < E / 2; ++e) {
          if (mine >> (u * E + 2 * e) & 1u) x[e].x = -INFINITY;
          if (mine >> (u * E + 2 * e + 1) & 1u) x[e].y = -INFINITY;
        }
        now[u] = Vec<T>::set(x);
      }
    }
    return batchMax<T>(now);
  }
};

// Whether a row counts, by one warp: one does that has a listed token and, without the rest, one that the teacher gives some
// probability.
template <bool kRest> __device__ __forceinline__ bool countsAtAll(const Given& given, int64_t r) {
  bool some = false;
  for (int first = 0; first < given.k && !some; first += 32) {
    const int i = first + (threadIdx.x & 31);
    some = i < given.k && given.tokens[r * given.k + i] >= 0 && (kRest || !(given.log_probs[r * given.k + i] == -INFINITY));
    some = __any_sync(kAll, some);
  }
  return some;
}

// The entries of row r, the teacher's probabilities and the student's logits, by one warp.
template <typename T, bool kRest>
__device__ __forceinline__ void loadTeacher(Teacher& te, const Given& given, int64_t r, const T* row, int vocab, float inv_t) {
  const int lane = threadIdx.x & 31, k = given.k;
  bool outside = false;
  float top = -INFINITY, total = 0.f, terms = 0.f;
#pragma unroll 2
  for (int i = lane; i < k; i += 32) {
    const int64_t t = given.tokens[r * k + i];
    const float value = given.log_probs[r * k + i];
    const bool known = t >= 0 && t < vocab;
    outside |= t >= vocab;
    te.token[i] = known ? (int)t : -1;
    te.q[i] = known ? value : -INFINITY;
    te.logit[i] = known ? toFloat(row[t]) : 0.f;
    if (known) top = fmaxf(top, value);
  }
  outside = __any_sync(kAll, outside);
  top = kRest ? 0.f : warpMax(top);
  if (top == -INFINITY) top = 0.f;
  const float scale = kRest ? 1.f : inv_t;
  // What is stored becomes the exponential, which is divided by the total when that is known.
  for (int i = lane; i < k; i += 32) {
    const float d = (te.q[i] - top) * scale, e = expf(d);
    te.q[i] = e;
    total += e;
    if (!(e == 0.f)) terms = fmaf(e, d, terms);
  }
  terms = warpSum(terms);
  float per_total = 1.f;
  if constexpr (!kRest) {
    total = warpSum(total);
    per_total = 1.f / total;
    for (int i = lane; i < k; i += 32) te.q[i] *= per_total;
  }
  if (lane == 0) te.log_terms = terms * per_total, te.total = kRest ? 1.f : total, te.outside = outside;
  __syncwarp();
}

// Marks the listed tokens of a row, by one warp; returns the bits of those outside the vectors, and whether a token may be named
// more than once.
template <int kWidth, typename T>
__device__ __forceinline__ unsigned markListed(const Teacher& te, int k, const Slice<T>& sl, unsigned* bits, bool& twice) {
  unsigned loose = 0;
  bool again = false;
  for (int i = threadIdx.x & 31; i < k; i += 32) {
    const int t = te.token[i];
    if (t < 0) continue;
    if (Marks<T, kWidth>::loose(sl, t))
      loose |= Marks<T, kWidth>::looseBit(sl, t), again = true;  // perhaps: there are few
    else
      again |= setBit(bits, Marks<T, kWidth>::place(sl, t));
  }
  twice = __any_sync(kAll, again);
  return __reduce_or_sync(kAll, loose);
}

// Whether a token is named more than once, by one warp.  Its bit is that of its number's end: where another token had set it, that
// token is looked for among all.  `bits`: `words` of zeros, a power of two, as they are again afterwards.
constexpr int kNameWords = 1024;
static_assert(kMostTeacherTokens <= kThreads, "a thread an entry");
__device__ __forceinline__ bool namedTwice(const Teacher& te, int k, unsigned* bits, int words) {
  const int lane = threadIdx.x & 31;
  bool twice = false;
  for (int first = 0; first < k; first += 32) {
    const int i = first + lane, t = i < k ? te.token[i] : -1;
    const bool set = t >= 0 && setBit(bits, t & (32 * words - 1));
    for (unsigned mask = __ballot_sync(kAll, set); mask != 0; mask &= mask - 1) {
      const int wanted = __shfl_sync(kAll, t, __ffs(mask) - 1);
      unsigned found = 0;
      for (int j = lane; j < k; j += 32) found += te.token[j] == wanted;
      twice |= __reduce_add_sync(kAll, found) > 1;
    }
  }
  __syncwarp();
  for (int i = lane; i < k; i += 32)
    if (te.token[i] >= 0) bits[(te.token[i] >> 5) & (words - 1)] = 0;
  __syncwarp();
  return twice;
}

// Which entries are the first to name their token, and for the backward the listed tokens, each once, with the sum of what its
// entries have, by one warp.  `twice`: a token may be named more than once.
__device__ __forceinline__ void mergeTeacher(Teacher& te, int k, bool twice, int2* pairs) {
  for (int i = threadIdx.x & 31; i < k; i += 32) {
    const int t = te.token[i];
    float q = te.q[i];
    bool first = t >= 0;
    if (twice) {
      q = 0.f;
      for (int j = 0; j < k; ++j)
        if (te.token[j] == t) {
          q += te.q[j];
          first = first && j >= i;
        }
    }
    te.first[i] = first;
    if (pairs != nullptr) pairs[i] = make_int2(first ? t : -1, __float_as_int(q));
  }
  __syncwarp();
}

// By one warp.
template <bool kRest> __device__ __forceinline__ Listed listedOf(const Teacher& te, int k, float c) {
  const int lane = threadIdx.x & 31;
  Listed l = {te.log_terms, te.total, -INFINITY, 0.f, 0.f, -INFINITY, 0.f};
  for (int i = lane; i < k; i += 32)
    if (te.token[i] >= 0) l.ref = fmaxf(l.ref, te.logit[i]);
  l.ref = warpMax(l.ref);
  if (kRest) l.m = l.ref;
  if (l.ref == -INFINITY) l.ref = 0.f;
  for (int i = lane; i < k; i += 32) {
    const float q = te.q[i], x = te.logit[i] - l.ref;
    if (te.token[i] >= 0 && !(q == 0.f)) {
      l.from_ref = fmaf(q, x, l.from_ref);
      l.mass += q;
    }
    if (kRest && te.first[i]) l.s += exp2Of(x * c);
  }
  l.from_ref = warpSum(l.from_ref);
  l.mass = warpSum(l.mass);
  if (kRest) l.s = warpSum(l.s);
  return l;
}

// Loss and what the backward needs, from that and the sums of the sweep, by one thread.  Kept: the maximum that the sweep takes
// differences from and the factor of those exponentials, the same for the listed tokens; the last is -1 where the row does
// not count.
template <bool kRest>
__device__ __forceinline__ void finishRow(const Listed& l, const Sums& acc, bool broken, float c, double inv_t, float* loss,
                                          float4* stats) {
  // All probabilities' maximum and sum; the sweep's are those of the rest.
  float m = acc.m, s = acc.s, above = 1.f;
  if constexpr (kRest) {
    m = fmaxf(acc.m, l.m);
    above = acc.s == 0.f ? 0.f : exp2Of((acc.m - m) * c);
    s = acc.s * above + (l.s == 0.f ? 0.f : l.s * exp2Of((l.m - m) * c));
  }
  // Differences are taken before the temperature and the logarithm come in: beside logits of 2^53 and more a logarithm is nothing.
  const double log_s = log((double)s), mass = l.mass;
  double sum = l.log_terms - l.from_ref * inv_t;
  if (!(mass == 0)) sum -= mass * (log((double)l.total) + (((double)l.ref - m) * inv_t - log_s));
  const float nan = __int_as_float(0x7fffffff);
  float4 st = make_float4(m, 1.f / s, m, 1.f / s);
  if constexpr (kRest) {
    const double q_rest = 1.0 - mass < kLeastRest ? 0.0 : 1.0 - mass;  // NaN stays
    if (!(q_rest == 0)) sum += q_rest * (log(q_rest) - (((double)acc.m - m) * inv_t + (log((double)acc.s) - log_s)));
    const double all = mass + q_rest, p_rest = (double)(acc.s * above) / s;
    const bool some = !(acc.s == 0.f);
    st = make_float4(some ? acc.m : 0.f, some ? (float)((all * p_rest - q_rest) / acc.s) : 0.f, m, (float)(all / s));
  }
  st.y *= exp2Of(-Exponent::excess(st.x, c));
  st.w *= exp2Of(-Exponent::excess(st.z, c));
  *stats = broken ? make_float4(nan, nan, nan, nan) : st;
  *loss = broken ? nan : (float)sum;
}

__device__ __forceinline__ void skipRow(float* loss, float4* stats) {
  *loss = 0.f;
  *stats = make_float4(0.f, 0.f, 0.f, -1.f);
}

// Few rows: one per cluster.  Eight warps sweep, and one of the first block reads the teacher meanwhile.
constexpr int kSliceThreads = kThreads + 32;
template <typename T, bool kRest>
__global__ void __launch_bounds__(kSliceThreads, 4)
distillation_slices_kernel(const T* __restrict__ logits, LogitRows x, Given given, float c, double inv_t,
                           float* __restrict__ loss, float4* __restrict__ stats, int2* __restrict__ pairs) {
  namespace cg = cooperative_groups;
  __shared__ Teacher te;
  __shared__ Sums scratch[kWarps + 1], mine;
  __shared__ Listed listed;
  __shared__ unsigned loose;
  extern __shared__ __align__(16) unsigned names[];
  unsigned* bits = names + kNameWords;  // with the rest
  const cg::cluster_group cluster = cg::this_cluster();
  const int slices = cluster.num_blocks(), rank = cluster.block_rank();
  const int64_t r = blockIdx.x / slices;
  const int tid = threadIdx.x, k = given.k;
  const T* row = rowOf(x, logits, r);
  const Slice<T> sl(row, x.vocab, rank, slices);
  if (tid == 0) loose = 0;
  if (rank == 0)
    for (int i = tid; i < kNameWords; i += kSliceThreads) names[i] = 0;
  if constexpr (kRest)
    for (int i = tid; i < Marks<T>::words(sl.v1 - sl.v0); i += kSliceThreads) bits[i] = 0;
  int64_t t = -1;  // this thread's entry: there are no more than kThreads
  if (tid < k) t = given.tokens[r * k + tid];
  if (!__syncthreads_or(t >= 0 && (kRest || !(given.log_probs[r * k + tid] == -INFINITY)))) {
    if (rank == 0 && tid == 0) skipRow(loss + r, stats + r);
    return;
  }
  if constexpr (kRest) {
    if (t >= sl.c0 && t < sl.c1) {
      if (Marks<T>::loose(sl, (int)t))
        atomicOr(&loose, Marks<T>::looseBit(sl, (int)t));
      else
        setBit(bits, Marks<T>::place(sl, (int)t));
    }
    __syncthreads();
  }
  Sums acc = Sums::none(c);
  if (tid >= kThreads) {
    if (rank == 0) {
      loadTeacher<T, kRest>(te, given, r, row, x.vocab, (float)inv_t);
      if (kRest || pairs != nullptr)
        mergeTeacher(te, k, namedTwice(te, k, names, kNameWords), pairs != nullptr ? pairs + r * k : nullptr);
      const Listed l = listedOf<kRest>(te, k, c);
      if (tid == kThreads) listed = l;  // blockSums() has all wait for that
    }
  } else {
    if constexpr (kRest) {
      RestHook<kThreads> hook;
      hook.bits = bits;
      acc = scan<T, false, kThreads>(sl, c, hook);
    } else {
      NoHook none;
      acc = scan<T, false, kThreads>(sl, c, none);
    }
    const int col = tid < 2 * Vec<T>::kElems && !(loose >> tid & 1u) ? sl.looseCol(tid) : -1;
    if (col >= 0) acc.add<false>(toFloat(row[col]), c);
  }
  acc = blockSums<false>(acc, c, scratch);
  if (slices > 1) {
    acc = clusterSums<false>(acc, c, &mine);
    clusterDone();
  }
  if (rank != 0) return;
  if (!acc.settle<false>(c)) {
    if constexpr (kRest)
      acc = blockAgain<T, false>(row, x.vocab, c, scratch, LeaveListed{&te, k});
    else
      acc = blockAgain<T, false>(row, x.vocab, c, scratch, LeaveNone());
  }
  if (tid == 0) finishRow<kRest>(listed, acc, te.outside, c, inv_t, loss + r, stats + r);
}

// Many short rows: one per warp.
template <typename T> struct ShortRow {
  Teacher teacher;
  static constexpr int kWords = Marks<T, 32>::words(kShortBytes / 16);
  unsigned bits[kWords];
};
template <typename T, bool kRest>
__global__ void __launch_bounds__(kThreads, 4)
distillation_short_kernel(const T* __restrict__ logits, LogitRows x, Given given, float c, double inv_t, float* __restrict__ loss,
                          float4* __restrict__ stats, int2* __restrict__ pairs) {
  extern __shared__ __align__(16) unsigned char dynamic[];
  ShortRow<T>& mine = reinterpret_cast<ShortRow<T>*>(dynamic)[threadIdx.x >> 5];
  Teacher& te = mine.teacher;
  const int lane = threadIdx.x & 31, k = given.k;
  const int64_t r = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (r >= x.rows) return;
  if (!countsAtAll<kRest>(given, r)) {
    if (lane == 0) skipRow(loss + r, stats + r);
    return;
  }
  const T* row = rowOf(x, logits, r);
  const Slice<T> sl(row, x.vocab, 0, 1);
  loadTeacher<T, kRest>(te, given, r, row, x.vocab, (float)inv_t);
  constexpr int names = 128;  // words, a power of two
  static_assert(names <= ShortRow<T>::kWords);
  for (int i = lane; i < (kRest ? Marks<T, 32>::words(sl.v1) : names); i += 32) mine.bits[i] = 0;
  __syncwarp();
  unsigned left_out = 0;
  bool twice = false;
  if (kRest)
    left_out = markListed<32>(te, k, sl, mine.bits, twice);
  else if (pairs != nullptr)
    twice = namedTwice(te, k, mine.bits, names);
  if (kRest || pairs != nullptr) mergeTeacher(te, k, twice, pairs != nullptr ? pairs + r * k : nullptr);
  Sums acc;
  if constexpr (kRest) {
    RestHook<32> hook;
    hook.bits = mine.bits;
    acc = scan<T, false, 32>(sl, c, hook);
  } else {
    NoHook none;
    acc = scan<T, false, 32>(sl, c, none);
  }
  const Listed l = listedOf<kRest>(te, k, c);
  const int col = lane < 2 * Vec<T>::kElems && !(left_out >> lane & 1u) ? sl.looseCol(lane) : -1;
  if (col >= 0) acc.add<false>(toFloat(row[col]), c);
  acc = warpSums<false>(acc, c);
  if (!acc.settle<false>(c)) {
    if constexpr (kRest)
      acc = warpAgain<T, false>(row, x.vocab, c, LeaveListed{&te, k});
    else
      acc = warpAgain<T, false>(row, x.vocab, c, LeaveNone());
  }
  if (lane == 0) finishRow<kRest>(l, acc, te.outside, c, inv_t, loss + r, stats + r);
}

// Many rows: the blocks stay.  With the rest the fetching warp marks the listed tokens of a row while the row before it is
// swept, in place of those of the row before that.
// A row that needs no more than finishRow(), which is done for 32 of them at once.
struct Pending {
  Listed listed;
  Sums sums;
  int row;
  bool outside;
};
struct DistillRows {
  Ring ring;
  HandOver hand;
  Teacher teacher[kSlots];
  unsigned loose[kSlots];  // the listed columns outside the vectors
  Pending pending[32];
  alignas(16) unsigned bits[1];  // kNameWords; with the rest, twice as many words as the kernel is told
};
template <typename T> struct RestRowsHook : RestHook<kThreads> {
  const unsigned* all;
  HandOver* hand;
  int words_a_row, turn = 1;
  __device__ __forceinline__ void begin(const Place& at) {
    hand->wait(&hand->marked[at.slot], at.parity);
    turn ^= 1;
    bits = all + turn * words_a_row;
  }
  __device__ __forceinline__ void end() {}
  __device__ __forceinline__ void arrived(uint4* place, int b) {
    constexpr int E = Vec<T>::kElems;
    for (unsigned mine = this->template listed<T>(b); mine != 0; mine &= mine - 1) {
      const int at = __ffs(mine) - 1;
      fromFloat(reinterpret_cast<T*>(place + at / E * kThreads) + at % E, -INFINITY);
    }
  }
  __device__ __forceinline__ float batch(uint4 (&now)[kBatch], bool, int, const Slice<T>&) { return batchMax<T>(now); }
};
template <typename T, bool kRest>
__global__ void __launch_bounds__(kRowThreads, 3)
distillation_rows_kernel(const T* __restrict__ logits, LogitRows x, Given given, float c, double inv_t,
                         float* __restrict__ loss, float4* __restrict__ stats, int2* __restrict__ pairs, int words, int rows_a_block) {
  extern __shared__ __align__(16) unsigned char dynamic[];
  DistillRows& shared = *reinterpret_cast<DistillRows*>(dynamic);
  HandOver& hand = shared.hand;
  if (threadIdx.x == 0) hand.init();
  for (int i = threadIdx.x; i < (kRest ? 2 * words : kNameWords); i += kRowThreads) shared.bits[i] = 0;
  __syncthreads();
  if (threadIdx.x < kThreads) {
    if constexpr (kRest) {
      RestRowsHook<T> hook;
      hook.all = shared.bits;
      hook.hand = &hand;
      hook.words_a_row = words;
      sweepRows<T, false>(logits, x, c, shared.ring, hand, hook);
    } else {
      NoHook none;
      sweepRows<T, false>(logits, x, c, shared.ring, hand, none);
    }
    return;
  }
  const int lane = threadIdx.x & 31, k = given.k;
  if (threadIdx.x < kThreads + 32) {
    Place before;  // the row before the last
    int fetched = 0, marked = -1, marked_before = -1;  // the rows whose listed tokens are marked
    fetchRows(
        [](int) { return true; }, x.rows, rows_a_block, hand, [&](int r) { skipRow(loss + r, stats + r); },
        [&](int r) {
          const float nan = __int_as_float(0x7fffffff);
          loss[r] = nan, stats[r] = make_float4(nan, nan, nan, nan);
        },
        [&](int r, const Place& at) {
          if (!countsAtAll<kRest>(given, r)) return false;
          // The marks are waited for, so what can be done before the row is handed on is.
          if (kRest) loadTeacher<T, kRest>(shared.teacher[at.slot], given, r, rowOf(x, logits, r), x.vocab, (float)inv_t);
          return true;
        },
        [&](int r, const Place& at) {
          Teacher& te = shared.teacher[at.slot];
          const T* row = rowOf(x, logits, r);
          if (!kRest) loadTeacher<T, kRest>(te, given, r, row, x.vocab, (float)inv_t);
          bool twice = false;
          if constexpr (kRest) {
            unsigned* bits = shared.bits + (fetched & 1) * words;
            if (fetched >= 2) {  // swept: its marks go
              hand.wait(&hand.full[before.slot], before.parity);
              const Slice<T> sl(rowOf(x, logits, marked_before), x.vocab, 0, 1);
              const Teacher& old = shared.teacher[before.slot];
              for (int i = lane; i < k; i += 32)
                if (old.token[i] >= 0 && !Marks<T>::loose(sl, old.token[i])) bits[Marks<T>::place(sl, old.token[i]) >> 5] = 0;
              before.next();
              __syncwarp();
            }
            marked_before = marked;
            marked = r;
            const unsigned loose = markListed<kThreads>(te, k, Slice<T>(row, x.vocab, 0, 1), bits, twice);
            __syncwarp();  // every lane's marks before the arrival of one
            if (lane == 0) {
              shared.loose[at.slot] = loose;
              barrierArrive(&hand.marked[at.slot]);
            }
            ++fetched;
          } else if (pairs != nullptr) {
            twice = namedTwice(te, k, shared.bits, kNameWords);
          }
          if (kRest || pairs != nullptr) mergeTeacher(te, k, twice, pairs != nullptr ? pairs + (int64_t)r * k : nullptr);
        });
    return;
  }
  int pending = 0;
  auto flush = [&] {
    __syncwarp();
    if (lane < pending) {
      const Pending& p = shared.pending[lane];
      finishRow<kRest>(p.listed, p.sums, p.outside, c, inv_t, loss + p.row, stats + p.row);
    }
    __syncwarp();
    pending = 0;
  };
  finishRows(hand, [&](int r, const Place& at) {
    const T* row = rowOf(x, logits, r);
    const Slice<T> sl(row, x.vocab, 0, 1);
    const Teacher& te = shared.teacher[at.slot];
    if (!hand.wait(&hand.prepared[at.slot], at.parity)) return;
    const Listed l = listedOf<kRest>(te, k, c);
    if (!hand.wait(&hand.full[at.slot], at.parity)) return;
    Sums acc = hand.template take<T, false>(at.slot, sl, c, kRest ? shared.loose[at.slot] : 0);
    if (!acc.settle<false>(c)) {
      if constexpr (kRest)
        acc = warpAgain<T, false>(row, x.vocab, c, LeaveListed{&te, k});
      else
        acc = warpAgain<T, false>(row, x.vocab, c, LeaveNone());
    }
    if (lane == 0) shared.pending[pending] = {l, acc, r, te.outside};
    if (++pending == 32) flush();
  });
  flush();
}

__global__ void __launch_bounds__(1024)
distillation_mean_kernel(const float* __restrict__ loss, const float4* __restrict__ stats, int64_t rows,
                         float* __restrict__ mean, float* __restrict__ count) {
  __shared__ double sums[32], numbers[32];
  double s = 0, n = 0;
#pragma unroll 8
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

// A block does one batch of vectors of one row and then, over what it has written, the listed tokens among them.  What they need is
// made in the forward, each token once: looking for tokens that are named twice here cost 254 -> 314 us.  The two forms of the exponent as
// two loops save an instruction a pair and cost the sixth block (42 registers): 256 -> 273 us.
template <typename T>
__global__ void __launch_bounds__(kThreads)
distillation_bwd_kernel(const T* __restrict__ logits, LogitRows x, T* grad, const float4* __restrict__ stats,
                        const int2* __restrict__ pairs, int k, float c, float inv_t, const float* __restrict__ upstream,
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
      mine = pairs[r * k + threadIdx.x];
      if ((unsigned)mine.x >= (unsigned)x.vocab) mine.x = -1;  // a row that was given up has whatever the memory held
      const int v = (mine.x - parts.head) / E / (U * kThreads);
      const bool vector = mine.x >= parts.head && mine.x < parts.head + parts.nvec * E;
      if (mine.x >= 0 && (vector ? v : 0) != piece) mine.x = -1;
      if (mine.x >= 0) logit = toFloat(row[mine.x]);
    }
    const float up = upstream[r * stride] * inv_t, g = count != nullptr ? up / *count : up;
    const float f = st.y * g;
    const Exponent exponent(st.x, c);
    auto of = [&](float2 v) {
      const float2 d = exponent(v);
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
      if (mine.x >= 0) fromFloat(out + mine.x, fmaf(exp2Of(Exponent(st.z, c)(make_float2(logit, 0.f)).x), st.w, -__int_as_float(mine.y)) * g);
    }
  }
}

// The same by a warp a piece, which looks through all listed tokens.
template <typename T>
__global__ void __launch_bounds__(kThreads, 5)
distillation_short_bwd_kernel(const T* __restrict__ logits, LogitRows x, T* grad, const float4* __restrict__ stats,
                              const int2* __restrict__ pairs, int k, float c, float inv_t, const float* __restrict__ upstream,
                              int64_t stride, const float* __restrict__ count, Pieces pieces) {
  constexpr int E = Vec<T>::kElems, U = kBatch;
  const int lane = threadIdx.x & 31;
  const unsigned w = pieces.mine();
  if (w >= pieces.total) return;
  const int64_t r = w / pieces.a_row;
  const int piece = (int)(w % pieces.a_row);
  const T* row = rowOf(x, logits, r);
  T* out = rowOf(x, grad, r);
  const RowParts<T> parts(row, x.vocab);
  const int first = piece * U * 32 + lane;
  const uint4* vecs = reinterpret_cast<const uint4*>(row + parts.head);
  uint4* vout = reinterpret_cast<uint4*>(out + parts.head);
  const float4 st = stats[r];
  const bool counts = !(st.w < 0.f);
  uint4 raw[U];
#pragma unroll
  for (int u = 0; u < U; ++u)
    raw[u] = counts && first + u * 32 < parts.nvec ? __ldg(vecs + first + u * 32) : make_uint4(0, 0, 0, 0);
  // The i-th listed token if it is this piece's, and its logit.
  auto listed = [&](int i, float& logit) {
    int2 pair = pairs[r * k + i];
    if ((unsigned)pair.x >= (unsigned)x.vocab) pair.x = -1;  // as above
    const int v = (pair.x - parts.head) / E / (U * 32);
    const bool vector = pair.x >= parts.head && pair.x < parts.head + parts.nvec * E;
    if (pair.x >= 0 && (vector ? v : 0) != piece) pair.x = -1;
    if (pair.x >= 0) logit = toFloat(row[pair.x]);
    return pair;
  };
  int2 mine = make_int2(-1, 0);
  float logit = 0.f;
  if (counts && lane < k) mine = listed(lane, logit);
  const float up = upstream[r * stride] * inv_t, g = count != nullptr ? up / *count : up;
  const float f = st.y * g;
  const Exponent exponent(st.x, c);
  auto of = [&](float2 v) {
    const float2 d = exponent(v);
    return mul2(make_float2(exp2Of(d.x), exp2Of(d.y)), make_float2(f, f));
  };
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = first + u * 32;
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
  if (piece == 0 && lane < 2 * E) {
    const int i = lane, col = i < parts.head ? i : i + parts.nvec * E;
    if (col < x.vocab) fromFloat(out + col, counts ? of(make_float2(toFloat(row[col]), 0.f)).x : 0.f);
  }
  if (counts) {
    __syncwarp();  // the stores of the piece before those of the listed tokens
    auto put = [&] {
      if (mine.x >= 0) fromFloat(out + mine.x, fmaf(exp2Of(Exponent(st.z, c)(make_float2(logit, 0.f)).x), st.w, -__int_as_float(mine.y)) * g);
    };
    put();
    for (int i = lane + 32; i < k; i += 32) {
      mine = listed(i, logit);
      put();
    }
  }
}

template <typename T, bool kRest>
cudaError_t forwardOf(const T* logits, const LogitRows& x, const DistillationArgs& a, float* loss, float4* stats, int2* pairs,
                      int sm_count, cudaStream_t stream) {
  const float c = (float)(1.4426950408889634 / a.temperature);
  const double inv_t = 1.0 / a.temperature;
  const Given given{a.tokens, a.log_probs, a.k};
  if (shortRows(x, sizeof(T), sm_count))
    return launchShort(distillation_short_kernel<T, kRest>, x.rows, kWarps * sizeof(ShortRow<T>), stream, logits, x, given, c, inv_t,
                       loss, stats, pairs);
  const int words = kRest ? Marks<T>::words(x.vocab / Vec<T>::kElems) : 0;
  const size_t stay = sizeof(DistillRows) + (kRest ? 2 * (size_t)words : kNameWords) * 4;
  // Two blocks of the form that stays have to fit on a multiprocessor; with up to 57344 tokens of 16 bits three do.
  if (manyRows(x.rows, sm_count) && stay <= 112 * 1024) {
    const int rows_a_block = rowsABlock(x, sizeof(T), sm_count);
    return launchRows(distillation_rows_kernel<T, kRest>, x.rows, rows_a_block, stay, stream, logits, x, given, c, inv_t, loss, stats,
                      pairs, words, rows_a_block);
  }
  const int slices = slicesFor(x.rows, x.vocab, sizeof(T), sm_count);
  const size_t shared = 4 * (kNameWords + (kRest ? Marks<T>::words((x.vocab / Vec<T>::kElems + slices - 1) / slices) : 0));
  if (shared > 32 * 1024) {
    const cudaError_t e = allowShared(reinterpret_cast<const void*>(&distillation_slices_kernel<T, kRest>), shared);
    if (e != cudaSuccess) return e;
  }
  return launchSlices(distillation_slices_kernel<T, kRest>, x.rows, slices, kSliceThreads, shared, stream, logits, x, given, c, inv_t, loss,
                      stats, pairs);
}

template <typename T>
cudaError_t forwardOf(const void* logits, const LogitRows& x, const DistillationArgs& a, float* loss, float* stats,
                      void* pairs_, int sm_count, cudaStream_t stream) {
  const T* data = static_cast<const T*>(logits);
  float4* st = reinterpret_cast<float4*>(stats);
  int2* pairs = static_cast<int2*>(pairs_);
  return a.rest ? forwardOf<T, true>(data, x, a, loss, st, pairs, sm_count, stream)
                : forwardOf<T, false>(data, x, a, loss, st, pairs, sm_count, stream);
}

template <typename T>
cudaError_t backwardOf(const void* logits, const LogitRows& x, void* grad, const float* stats, const void* pairs, int k,
                       double temperature, const float* upstream, int64_t stride, const float* count, cudaStream_t stream) {
  constexpr int per_piece = kThreads * kBatch * Vec<T>::kElems;
  const int pieces = (int)(((int64_t)x.vocab + per_piece - 1) / per_piece);
  const int64_t total = x.rows * pieces;
  const float c = (float)(1.4426950408889634 / temperature), inv_t = (float)(1.0 / temperature);
  const float4* st = reinterpret_cast<const float4*>(stats);
  const int2* listed = static_cast<const int2*>(pairs);
  // Short rows that leave a quarter of the blocks' threads idle.  16 tokens, bf16: 8192 x 1000 20.3 -> 6.9 us, 8192 x 4000 25.7 -> 20.7,
  // 8192 x 8200 52.8 -> 45.8; but 8192 x 16384, which fills the blocks, 77 -> 86, and 4000 fp32 logits 36 -> 40.
  Pieces warps;
  if (warps.template cut<T>(x) && warps.a_row <= 16 && (int)warps.a_row < 6 * pieces)
    return launchBlocks(distillation_short_bwd_kernel<T>, warps.blocks(), kThreads, 1, 0, stream, static_cast<const T*>(logits), x,
                        static_cast<T*>(grad), st, listed, k, c, inv_t, upstream, stride, count, warps);
  return launchBlocks(distillation_bwd_kernel<T>, (unsigned)(total < (1 << 30) ? total : (1 << 30)), kThreads, 1, 0, stream,
                      static_cast<const T*>(logits), x, static_cast<T*>(grad), st, listed, k, c, inv_t, upstream, stride, count, total,
                      pieces);
}

}  // namespace

cudaError_t launchDistillation(const void* logits, const LogitRows& x, const DistillationArgs& a, float* loss, float* stats,
                               void* pairs, int sm_count, cudaStream_t stream) {
  if (x.rows <= 0) return cudaSuccess;
  if (x.vocab <= 0 || x.vocab > kMostVocab || x.rows > INT32_MAX || a.k <= 0 || a.k > kMostTeacherTokens || (a.rest && x.vocab > kMostRestVocab))
    return cudaErrorInvalidValue;
  switch (x.type) {
    case LogitType::kBFloat16: return forwardOf<__nv_bfloat16>(logits, x, a, loss, stats, pairs, sm_count, stream);
    case LogitType::kHalf: return forwardOf<__half>(logits, x, a, loss, stats, pairs, sm_count, stream);
    default: return forwardOf<float>(logits, x, a, loss, stats, pairs, sm_count, stream);
  }
}

cudaError_t launchDistillationMean(const float* loss, const float* stats, int64_t rows, float* mean, float* count,
                                   cudaStream_t stream) {
  return launchBlocks(distillation_mean_kernel, 1, 1024, 1, 0, stream, loss, reinterpret_cast<const float4*>(stats), rows, mean, count);
}

cudaError_t launchDistillationBackward(const void* logits, const LogitRows& x, void* grad, const float* stats,
                                       const void* pairs, int k, double temperature, const float* upstream, int64_t stride,
                                       const float* count, cudaStream_t stream) {
  if (x.rows <= 0) return cudaSuccess;
  if (x.vocab <= 0 || x.vocab > kMostVocab || x.rows > INT32_MAX || k <= 0 || k > kMostTeacherTokens) return cudaErrorInvalidValue;
  // A vector of the logits becomes a vector of the gradient.
  if ((reinterpret_cast<uintptr_t>(logits) ^ reinterpret_cast<uintptr_t>(grad)) & 15u) return cudaErrorMisalignedAddress;
  switch (x.type) {
    case LogitType::kBFloat16:
      return backwardOf<__nv_bfloat16>(logits, x, grad, stats, pairs, k, temperature, upstream, stride, count, stream);
    case LogitType::kHalf:
      return backwardOf<__half>(logits, x, grad, stats, pairs, k, temperature, upstream, stride, count, stream);
    default:
      return backwardOf<float>(logits, x, grad, stats, pairs, k, temperature, upstream, stride, count, stream);
  }
}

}  // namespace fairring
