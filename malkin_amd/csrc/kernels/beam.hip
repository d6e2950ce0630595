// Beam search's selection: per group of rows of logits, the k best of score + log softmax over all rows and tokens.
//
// A row's order does not need its sum: k_beam_rows reads the logits once, in segments, and leaves each segment's k best,
// sorted, with its maximum and the sum of exp(z - max) in 64 bits (candidates of two beams are often nearer to each other
// than a 32-bit sum is exact). k_beam_merge adds a row's sums and merges the sorted lists of a group. Neither sorts: a lower
// bound of the k-th best thins the candidates out, first in a segment (the k-th best of the maxima of 64 to 256 parts of it),
// then over the lists (the r-th best of their p-th elements, where (p + 1) r >= k), and what is left finds its place by
// counting what is better.
//
// What bounds it: for one request of four beams (12.4 us) the latency of two launches (5.6 and 6.7 us) and of their chains of
// loads, barriers and 64-bit exponentials; for 24 of them (22 us; about 42 MB of logits, those of ended beams are not read) the first
// launch, 16.3 us or 2.6 TB/s, with about 20 vector instructions a logit, half of them for its exponential.
#include <algorithm>
#include <cfloat>

#include "ctx.h"
#include "exp64.h"
#include "ops.h"

namespace mk {
namespace {

constexpr int kThreads = 256;
constexpr int kMergeThreads = 512;
constexpr int kMaxLists = kMergeThreads;  // that one merge takes
constexpr int kMergeCap = 1536;           // candidates that it ranks

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v4a __attribute__((ext_vector_type(4), aligned(4)));

struct Cand {
  float z;
  int32_t id;  // -1: none
};
struct Stat {
  double sum;  // of exp(z - max)
  float max;   // -inf: no candidate at all
  int32_t pad;
};

struct Beams {
  const float* logits;
  int64_t stride;
  const float* scores;
  const int32_t* done;
  int n_vocab, segs, len, k, beams, eos;  // len: logits of a segment
};

__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= FLT_MAX; }
// Larger logit first, then the lower token.
__device__ __forceinline__ bool ahead(float a, int ia, float b, int ib) { return a > b || (a == b && ia < ib); }

// Order-preserving bits of a float that is not NaN (0 of either sign the same).
__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t u = __float_as_uint(f + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key); }
// A candidate as one number: of two, the larger one is ahead.
__device__ __forceinline__ uint64_t rank_key(float z, int id) { return (uint64_t)order_key(z) << 32 | (uint32_t)~id; }

// One segment of a row, at most kThreads * 4 Q logits. The k-th largest of the maxima of PARTS parts of it is a bound (k <= MOST <=
// PARTS): at most (k - 1) parts hold anything larger. Of logits that are equal to it there can be any number; where the list
// does not hold them, those of the first whole rounds of 4 kThreads logits are taken that have enough.
template <int Q, int PARTS, int MOST>
__global__ __launch_bounds__(kThreads) void k_beam_rows(Beams B, Stat* __restrict__ stats, Cand* __restrict__ cands) {
  constexpr int kRound = 4 * kThreads, SHARE = kThreads / PARTS, CAP = (MOST - 1) * SHARE * 4 * Q + MOST + kRound;
  __shared__ double table[kTable];
  __shared__ __align__(16) float part_v[PARTS];
  __shared__ float wave_max[kThreads / 64];
  __shared__ uint32_t bound;
  __shared__ int n_cand;
  __shared__ double wave_sum[kThreads / 64];
  __shared__ uint64_t list[CAP];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, row = blockIdx.x / B.segs, seg = blockIdx.x % B.segs;
  const float* l = B.logits + row * B.stride;
  const int first = seg * B.len, end = min(first + B.len, B.n_vocab);
  const float start = B.scores[row];
  const int over = B.done ? B.done[row] : 0;
  if (!finite(start) || over) return;  // nobody reads what would be written
  float z[4 * Q];
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    const int at = first + q * kRound + 4 * tid;
    v4f f = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    if (at + 4 <= end) f = *reinterpret_cast<const v4a*>(l + at);
    else
#pragma unroll
      for (int e = 0; e < 3; ++e)
        if (at + e < end) f[e] = l[at + e];
#pragma unroll
    for (int e = 0; e < 4; ++e) z[4 * q + e] = f[e];
  }
  load_table(table);
  auto id_of = [&](int e) { return first + e / 4 * kRound + 4 * tid + e % 4; };
  float best = -INFINITY;
#pragma unroll
  for (int e = 0; e < 4 * Q; ++e) {
    z[e] = clean(z[e]);
    best = fmaxf(best, z[e]);
  }
  float part = best;  // of SHARE neighbouring threads
#pragma unroll
  for (int o = 1; o < SHARE; o <<= 1) part = fmaxf(part, __shfl_xor(part, o));
  float top = part;
#pragma unroll
  for (int o = 32; o >= SHARE; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  if (lane == 0) wave_max[w] = top;
  if (tid % SHARE == 0) part_v[tid / SHARE] = part;
  if (tid == 0) bound = 0xFFFFFFFFu, n_cand = 0;
  __syncthreads();
  top = wave_max[0];
#pragma unroll
  for (int i = 1; i < kThreads / 64; ++i) top = fmaxf(top, wave_max[i]);
  {  // every thread counts a share of the parts' maxima that are larger than its own part's
    int more = 0;
#pragma unroll 4
    for (int j = PARTS / SHARE * (tid % SHARE); j < PARTS / SHARE * (tid % SHARE + 1); j += 4) {
      const v4f v = *reinterpret_cast<const v4f*>(part_v + j);
#pragma unroll
      for (int e = 0; e < 4; ++e) more += v[e] > part;
    }
#pragma unroll
    for (int o = 1; o < SHARE; o <<= 1) more += __shfl_xor(more, o);
    if (more < B.k && tid % SHARE == 0) atomicMin(&bound, order_key(part));
  }
  double sum = 0.0;
  if (top > -INFINITY) {
    constexpr double c = kTable * 1.4426950408889634074, least = -63000.0 / c;  // below 2^-984 there is nothing
#pragma unroll
    for (int e = 0; e < 4 * Q; ++e) {
      const Power p = pow2_of(fmax((double)z[e] - (double)top, least), c, table);
      sum = __builtin_fma(p.factor, p.rest, sum);
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
  if (lane == 0) wave_sum[w] = sum;
  __syncthreads();
  const uint32_t key = bound;  // fewer than k parts: of -inf
  const float limit = of_key(key);
  auto put = [&](int e) {
    const int at = atomicAdd(&n_cand, 1);
    if (at < CAP) list[at] = rank_key(z[e], id_of(e));
  };
  if (best >= limit && best > -INFINITY)
#pragma unroll
    for (int e = 0; e < 4 * Q; ++e)
      if (z[e] >= limit && z[e] > -INFINITY) put(e);
  __syncthreads();
  if (n_cand > CAP) {
    __syncthreads();
    if (tid == 0) n_cand = 0;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 4 * Q; ++e)
      if (z[e] > limit) put(e);
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      __syncthreads();
      const bool want = n_cand < B.k;
      __syncthreads();
      if (want)
#pragma unroll
        for (int e = 4 * q; e < 4 * q + 4; ++e)
          if (z[e] == limit) put(e);
    }
    __syncthreads();
  }
  const int n = n_cand;
  Cand* out = cands + ((int64_t)row * B.segs + seg) * B.k;
  // Each one's place: how many are ahead of it, counted by four threads.
  for (int i = tid >> 2; i < n; i += kThreads / 4) {
    const uint64_t c = list[i];
    int before = 0;
#pragma unroll 8
    for (int j = tid & 3; j < n; j += 4) before += list[j] > c;
    before += __shfl_xor(before, 1);
    before += __shfl_xor(before, 2);
    if (before < B.k && (tid & 3) == 0) out[before] = Cand{of_key((uint32_t)(c >> 32)), (int32_t)~(uint32_t)c};
  }
  for (int i = n + tid; i < B.k; i += kThreads) out[i] = Cand{-INFINITY, -1};
  if (tid == 0) {
    double s = wave_sum[0];
    for (int i = 1; i < kThreads / 64; ++i) s += wave_sum[i];
    stats[(int64_t)row * B.segs + seg] = Stat{s, top, 0};
  }
}

struct Entry {
  double score;
  float z;
  int32_t id, beam;  // beam INT32_MAX: none
};
__device__ __forceinline__ bool ahead(const Entry& a, const Entry& b) {
  if (a.beam == b.beam) return ahead(a.z, a.id, b.z, b.id);
  return a.score > b.score || (a.score == b.score && a.beam < b.beam);
}

// One group: beams x segs sorted lists, at most kMaxLists. ROW: a group is one row, whose k best and sum become one list.
template <bool ROW>
__global__ __launch_bounds__(kMergeThreads) void k_beam_merge(Beams B, const Stat* __restrict__ stats,
                                                              const Cand* __restrict__ cands, Stat* __restrict__ row_stat,
                                                              Cand* __restrict__ row_cand, float* __restrict__ out_scores,
                                                              int32_t* __restrict__ out_seq, int32_t* __restrict__ out_tokens) {
  constexpr int kAhead = 4, kNext = 8;
  __shared__ double lse[64];
  __shared__ Entry list[kMergeCap], bound;
  __shared__ __align__(16) float heads[kMaxLists];
  __shared__ int place[kMergeCap], n_cand;
  __shared__ uint32_t least_key;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, group = blockIdx.x;
  const int beams = ROW ? 1 : B.beams, lists = beams * B.segs, k = B.k;
  const int64_t row0 = (int64_t)group * beams;
  const Entry none{-INFINITY, -INFINITY, -1, INT32_MAX};
  // This thread's list, its first elements asked for at once, beside everything else that the addresses are known of (what lies
  // where nothing was written is not looked at).
  const int beam = tid / B.segs;
  const bool in = tid < lists;
  const Cand* from = cands + (row0 * B.segs + (in ? tid : 0)) * k;
  Cand c[kAhead];
#pragma unroll
  for (int j = 0; j < kAhead; ++j) c[j] = from[min(j, k - 1)];
  const int64_t row = row0 + (in ? beam : 0);
  const float score = B.scores[row];
  const int done = B.done ? B.done[row] : 0;
  // Sums of the rows, a group of lanes for each: as many lanes as it has segments, at most a wave.
  int width = 1;
  while (width < B.segs && width < 64) width <<= 1;
  for (int b0 = w * (64 / width); b0 < beams; b0 += kMergeThreads / width) {
    const int b = b0 + lane / width, at = lane % width;
    const int64_t r = row0 + min(b, beams - 1);
    const Stat* s = stats + r * B.segs;
    const Stat first = s[min(at, B.segs - 1)];
    const float its = B.scores[r];
    const int end = B.done ? B.done[r] : 0;
    const bool live = b < beams && finite(its) && !end;  // nothing was written for the others
    Stat one{0.0, -INFINITY, 0};
    for (int i = at; i < B.segs && live; i += width) {
      const Stat t = i == at ? first : s[i];
      const float m = fmaxf(one.max, t.max);
      if (m == -INFINITY) continue;
      one = one.max == -INFINITY ? t : Stat{one.sum * exp((double)one.max - (double)m) + t.sum * exp((double)t.max - (double)m), m, 0};
    }
    float top = one.max;
    for (int o = width / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    double sum = one.max > -INFINITY ? one.sum * exp((double)one.max - (double)top) : 0.0;
    for (int o = width / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    if (live && at == 0) {
      if (ROW) row_stat[row0] = Stat{sum, top, 0};
      lse[b] = (double)top + log(sum);
    }
  }
  const bool mine = in && finite(score), over = mine && done;
  if (ROW && (!finite(score) || done)) return;
  const double start = ROW ? 0.0 : (double)score;
  if (tid == 0) bound = none, n_cand = 0, least_key = 0xFFFFFFFFu;
  for (int i = tid; i < kMergeCap; i += kMergeThreads) place[i] = 0;
  __syncthreads();
  auto entry = [&](int j, const Cand& v) {
    if (!mine || j >= k) return none;
    if (over) return tid % B.segs == 0 && j == 0 ? Entry{start, 0.0f, B.eos, beam} : none;
    return v.id < 0 ? none : Entry{(double)v.z - lse[beam] + start, v.z, v.id, beam};
  };
  auto put = [&](const Entry& e) {
    const int at = atomicAdd(&n_cand, 1);
    if (at < kMergeCap) list[at] = e;
  };
  // A bound by the lists' element p, rounded: (p + 1) r >= k, and at least r of them are as large as the r-th. Rounding keeps
  // the order, so nothing among the k best is smaller, rounded, than that.
  const int p0 = (k + lists - 1) / lists - 1, r0 = (k + p0) / (p0 + 1);
  const Entry head = entry(p0, p0 == 0 ? c[0] : from[min(p0, k - 1)]);
  const float mark = (float)head.score;
  if (in) heads[tid] = mark;
  for (int i = lists + tid; i < (lists + 3) / 4 * 4; i += kMergeThreads) heads[i] = -INFINITY;
  __syncthreads();
  if (in) {
    int more = 0;
#pragma unroll 8
    for (int j = 0; j < lists; j += 4) {
      const v4f v = *reinterpret_cast<const v4f*>(heads + j);
#pragma unroll
      for (int e = 0; e < 4; ++e) more += v[e] > mark;
    }
    if (more < r0) atomicMin(&least_key, order_key(mark));  // the r-th is the least of those
  }
  __syncthreads();
  const float least = of_key(least_key);
  {
    bool go = true;
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const Entry e = entry(j, c[j]);
      go = go && e.beam != INT32_MAX && (float)e.score >= least;
      if (go) put(e);
    }
    for (int j0 = kAhead; go && j0 < k; j0 += kNext) {  // a good beam's list has many: asked for together
      Cand more[kNext];
#pragma unroll
      for (int j = 0; j < kNext; ++j) more[j] = from[min(j0 + j, k - 1)];
#pragma unroll
      for (int j = 0; j < kNext; ++j) {
        const Entry e = entry(j0 + j, more[j]);
        go = go && e.beam != INT32_MAX && (float)e.score >= least;
        if (go) put(e);
      }
    }
  }
  __syncthreads();
  if (n_cand > kMergeCap) {
    // Many that are equal: bounds in the order's own terms, by the elements p = 0, 1, 3, .. of the lists. They leave at most
    // k (log2 k + 2): of the lists' elements p .. 2 p, fewer than k / (p + 1) + 1 each.
    Entry* all = list;
    for (int p = 0;; p = min(2 * p + 1, k - 1)) {
      const int r = (k + p) / (p + 1);
      __syncthreads();
      const Entry e = entry(p, from[min(p, k - 1)]);
      if (in) all[tid] = e;
      __syncthreads();
      if (in && r <= lists && e.beam != INT32_MAX) {
        int before = 0;
        for (int j = 0; j < lists; ++j) before += ahead(all[j], e);
        if (before == r - 1 && ahead(e, bound)) bound = e;  // one thread's
      }
      if (p == k - 1) break;
    }
    if (tid == 0) n_cand = 0;
    __syncthreads();
    const Entry last = bound;
    for (int j = 0; j < k; ++j) {
      const Entry e = entry(j, from[j]);
      if (e.beam == INT32_MAX || ahead(last, e)) break;
      put(e);
    }
    __syncthreads();
  }
  // Each one's place: how many are ahead of it, counted by several threads where there are few.
  const int n = min(n_cand, kMergeCap), parts = max(1, min(16, kMergeThreads / max(n, 1)));
  for (int at = tid; at < n * parts; at += kMergeThreads) {
    const int i = at / parts;
    const Entry e = list[i];
    int before = 0;
    auto count = [&](int j, double s) {  // of one beam's, the scores have the logits' order
      if (s > e.score || (s == e.score && ahead(list[j], e))) ++before;
    };
    int j = at % parts;
    for (; j + 3 * parts < n; j += 4 * parts) {
      double s[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) s[u] = list[j + u * parts].score;
#pragma unroll
      for (int u = 0; u < 4; ++u) count(j + u * parts, s[u]);
    }
    for (; j < n; j += parts) count(j, list[j].score);
    if (before) atomicAdd(&place[i], before);
  }
  __syncthreads();
  for (int i = tid; i < max(n, k); i += kMergeThreads) {
    const Entry e = i < n ? list[i] : none;
    const int to = i < n ? place[i] : i;
    if (to >= k) continue;
    if (ROW) {
      row_cand[row0 * k + to] = Cand{e.z, e.id};
    } else {
      const int64_t at = (int64_t)group * k + to;
      out_scores[at] = (float)e.score, out_seq[at] = i < n ? (int32_t)(row0 + e.beam) : -1, out_tokens[at] = e.id;
    }
  }
}

constexpr int kSmallSeg = kThreads * 4 * 4, kLargeSeg = kThreads * 4 * 8;

// Longer segments where there are many rows and few candidates of each: 96 rows of 151936 logits, k 4, 23.5 us with long ones
// and 24.5 with short ones, k 16 25.1 and 26.5; 4 rows 13.7 and 13.1, 56 rows 20.8 and 20.3.
int seg_of(int rows, int n_vocab, int k) {
  return k <= 16 && (int64_t)rows * n_vocab > (int64_t)kLargeSeg * 1024 ? kLargeSeg : kSmallSeg;
}

}  // namespace

size_t beam_workspace(int n_group, int beams, int n_vocab, int k) {
  const int64_t rows = (int64_t)n_group * beams, lists = rows * ((n_vocab + kSmallSeg - 1) / kSmallSeg + 1);
  return (size_t)lists * (sizeof(Stat) + (size_t)k * sizeof(Cand));
}

void beam_select(hipStream_t s, const float* logits, int64_t stride, int n_group, int beams, int n_vocab, const float* scores,
                 const int32_t* done, int eos, int k, float* out_scores, int32_t* out_seq, int32_t* out_tokens,
                 void* workspace) {
  const int rows = n_group * beams, seg = seg_of(rows, n_vocab, k), segs = (n_vocab + seg - 1) / seg;
  // Segments of one length: a short one at the end would have fewer parts than k, and rank all that it has (32 rows of 151936
  // logits, k 64: 25 us instead of 16).
  const int len = (n_vocab + segs - 1) / segs, whole = (len + 3) / 4 * 4;
  Beams B{logits, stride, scores, done, n_vocab, segs, whole, k, beams, eos};
  Stat* stats = static_cast<Stat*>(workspace);
  Stat* row_stat = stats + (int64_t)rows * segs;
  Cand* cands = reinterpret_cast<Cand*>(row_stat + rows);
  Cand* row_cand = cands + (int64_t)rows * segs * k;
  auto go = [&]<int Q, int PARTS, int MOST>() {
    hipLaunchKernelGGL((k_beam_rows<Q, PARTS, MOST>), dim3((unsigned)(rows * segs)), dim3(kThreads), 0, s, B, stats, cands);
    check_launch("beam_select rows");
  };
  const bool large = seg == kLargeSeg;
  // As many parts as k needs: a thread compares its own with all others. 160 rows of 32003 logits, k 64: 26 us with 128, 29.6
  // with 256; 32 rows of 151936, k 16: 18.2 with 64, 19.1 with 128.
  if (k <= 16) large ? go.template operator()<8, 64, 16>() : go.template operator()<4, 64, 16>();
  else if (k <= 64) go.template operator()<4, 128, 64>();
  else go.template operator()<4, 256, 128>();
  if ((int64_t)beams * segs > kMaxLists) {  // a list per row first
    hipLaunchKernelGGL(k_beam_merge<true>, dim3((unsigned)rows), dim3(kMergeThreads), 0, s, B, stats, cands, row_stat,
                       row_cand, nullptr, nullptr, nullptr);
    check_launch("beam_select lists");
    B.segs = 1, stats = row_stat, cands = row_cand;
  }
  hipLaunchKernelGGL(k_beam_merge<false>, dim3((unsigned)n_group), dim3(kMergeThreads), 0, s, B, stats, cands, nullptr, nullptr,
                     out_scores, out_seq, out_tokens);
  check_launch("beam_select merge");
}

}  // namespace mk
