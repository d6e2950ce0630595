// Beam search's selection: per group of rows of logits, the k best of score + log softmax over all rows and tokens.
//
// A row's order does not need its sum: k_beam_rows reads the logits once, in segments, and leaves each segment's k best,
// sorted, with its maximum and the sum of exp(z - max) in 64 bits (candidates of two beams are often nearer to each other
// than a 32-bit sum is exact). k_beam_merge adds a row's sums and merges the sorted lists of a group. Neither sorts: a lower
// bound of the k-th best thins the candidates out, first in a segment (the k-th best of the maxima of 64 or 256 parts of it),
// then over the lists (the r-th best of their p-th elements, where (p + 1) r >= k), and what is left finds its place by
// counting what is better.
//
// What bounds it: the logits' bytes, beside about 25 vector instructions a logit (12 of them 64-bit); for one request the
// latency of two launches and of the merge's chain.
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
  int n_vocab, segs, k, beams, eos;
};

__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= FLT_MAX; }
// Larger logit first, then the lower token.
__device__ __forceinline__ bool ahead(float a, int ia, float b, int ib) { return a > b || (a == b && ia < ib); }

// One segment of kThreads * 4 Q logits of a row. PARTS: of which the maxima bound the k-th best: 64 (of 4 threads) or one per
// thread; k <= PARTS. Only the k parts with the first maxima hold candidates, so at most CAP of them.
template <int Q, int PARTS>
__global__ __launch_bounds__(kThreads) void k_beam_rows(Beams B, Stat* __restrict__ stats, Cand* __restrict__ cands) {
  constexpr int kSeg = kThreads * 4 * Q, kMost = PARTS == 64 ? 16 : 128, CAP = kMost * (kThreads / PARTS) * 4 * Q;
  __shared__ double table[kTable];
  __shared__ float part_v[PARTS], wave_max[kThreads / 64], bound_v;
  __shared__ int part_i[PARTS], bound_i, n_cand;
  __shared__ double wave_sum[kThreads / 64];
  __shared__ Cand list[CAP];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, row = blockIdx.x / B.segs, seg = blockIdx.x % B.segs;
  if (!finite(B.scores[row]) || (B.done && B.done[row])) return;  // nobody reads what would be written
  load_table(table);
  const float* l = B.logits + row * B.stride;
  const int first = seg * kSeg;
  float z[4 * Q];
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    const int at = first + q * (4 * kThreads) + 4 * tid;
    if (at + 4 <= B.n_vocab) {
      const v4f f = *reinterpret_cast<const v4a*>(l + at);
#pragma unroll
      for (int e = 0; e < 4; ++e) z[4 * q + e] = f[e];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) z[4 * q + e] = at + e < B.n_vocab ? l[at + e] : -INFINITY;
    }
  }
  auto id_of = [&](int e) { return first + e / 4 * (4 * kThreads) + 4 * tid + e % 4; };
  float best = -INFINITY;
  int best_i = INT32_MAX;
#pragma unroll
  for (int e = 0; e < 4 * Q; ++e) {
    z[e] = clean(z[e]);
    if (z[e] > best) best = z[e], best_i = id_of(e);
  }
  float top = best;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  if (lane == 0) wave_max[w] = top;
  if (PARTS == 64) {
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      const float v = __shfl_xor(best, o);
      const int i = __shfl_xor(best_i, o);
      if (ahead(v, i, best, best_i)) best = v, best_i = i;
    }
    if (tid % 4 == 0) part_v[tid / 4] = best, part_i[tid / 4] = best_i;
  } else {
    part_v[tid] = best, part_i[tid] = best_i;
  }
  if (tid == 0) bound_v = -INFINITY, bound_i = INT32_MAX, n_cand = 0;
  __syncthreads();
  top = wave_max[0];
#pragma unroll
  for (int i = 1; i < kThreads / 64; ++i) top = fmaxf(top, wave_max[i]);
  if (tid < PARTS) {
    const float v = part_v[tid];
    const int i = part_i[tid];
    int before = 0;
#pragma unroll 8
    for (int j = 0; j < PARTS; ++j) before += ahead(part_v[j], part_i[j], v, i);
    if (before == B.k - 1 && v > -INFINITY) bound_v = v, bound_i = i;
  }
  double sum = 0.0;
  if (top > -INFINITY) {
#pragma unroll
    for (int e = 0; e < 4 * Q; ++e) {
      const double d = ((double)z[e] - (double)top) * (kTable * 1.4426950408889634074);
      const bool in = d > -63000.0;  // below 2^-984 there is nothing
      const Power p = pow2(in ? d : 0.0, table);
      sum += in ? p.factor * p.rest : 0.0;
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
  if (lane == 0) wave_sum[w] = sum;
  __syncthreads();
  const float bv = bound_v;
  const int bi = bound_i;
#pragma unroll
  for (int e = 0; e < 4 * Q; ++e)
    if (z[e] > -INFINITY && !ahead(bv, bi, z[e], id_of(e))) list[atomicAdd(&n_cand, 1)] = Cand{z[e], id_of(e)};
  __syncthreads();
  const int n = n_cand;
  Cand* out = cands + ((int64_t)row * B.segs + seg) * B.k;
  for (int i = tid; i < n; i += kThreads) {
    const Cand c = list[i];
    int before = 0;
    for (int j = 0; j < n; ++j) before += ahead(list[j].z, list[j].id, c.z, c.id);
    if (before < B.k) out[before] = c;
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
  __shared__ double lse[64];
  __shared__ Entry heads[kMaxLists], list[kMergeCap], bound;
  __shared__ int n_cand;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, group = blockIdx.x;
  const int beams = ROW ? 1 : B.beams, lists = beams * B.segs, k = B.k;
  const int64_t row0 = (int64_t)group * beams;
  auto alive = [&](int b) { return finite(B.scores[row0 + b]); };
  auto ended = [&](int b) { return B.done && B.done[row0 + b]; };
  if (ROW && (!alive(0) || ended(0))) return;
  const Entry none{-INFINITY, -INFINITY, -1, INT32_MAX};
  for (int b = w; b < beams; b += kMergeThreads / 64) {
    if (!alive(b) || ended(b)) continue;  // nothing was written for it
    const Stat* s = stats + (row0 + b) * B.segs;
    float top = -INFINITY;
    for (int i = lane; i < B.segs; i += 64) top = fmaxf(top, s[i].max);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    double sum = 0.0;
    for (int i = lane; i < B.segs; i += 64)
      if (s[i].max > -INFINITY) sum += s[i].sum * exp((double)s[i].max - (double)top);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    if (lane == 0) {
      if (ROW) row_stat[row0] = Stat{sum, top, 0};
      lse[b] = (double)top + log(sum);
    }
  }
  // This thread's list.
  const int beam = tid / B.segs;
  const bool mine = tid < lists && alive(beam);
  const bool over = mine && ended(beam);
  const Cand* from = cands + (row0 * B.segs + tid) * k;
  if (tid == 0) bound = none;
  __syncthreads();
  auto entry = [&](int j) {
    if (!mine || j >= k) return none;
    const double start = ROW ? 0.0 : (double)B.scores[row0 + beam];
    if (over) return tid % B.segs == 0 && j == 0 ? Entry{start, 0.0f, B.eos, beam} : none;
    const Cand c = from[j];
    return c.id < 0 ? none : Entry{(double)c.z - lse[beam] + start, c.z, c.id, beam};
  };
  // A bound by the lists' element p: (p + 1) r >= k, and at least r of them are as good as the r-th best.
  auto bound_by = [&](int p) {
    const int r = (k + p) / (p + 1);
    if (tid < lists) heads[tid] = entry(p);
    __syncthreads();
    if (tid < lists && r <= lists) {
      const Entry e = heads[tid];
      if (e.beam != INT32_MAX) {
        int before = 0;
#pragma unroll 4
        for (int j = 0; j < lists; ++j) before += ahead(heads[j], e);
        if (before == r - 1 && ahead(e, bound)) bound = e;  // one thread's
      }
    }
    if (tid == 0) n_cand = 0;
    __syncthreads();
  };
  auto collect = [&] {
    const Entry least = bound;
    for (int j = 0; j < k; ++j) {
      const Entry e = entry(j);
      if (e.beam == INT32_MAX || ahead(least, e)) break;
      const int at = atomicAdd(&n_cand, 1);
      if (at < kMergeCap) list[at] = e;
    }
    __syncthreads();
  };
  bound_by((k + lists - 1) / lists - 1);
  collect();
  if (n_cand > kMergeCap) {
    // Bounds of p = 0, 1, 3, .. leave at most k (log2 k + 2) candidates: of the lists' elements p .. 2 p, fewer than
    // k / (p + 1) + 1 each.
    for (int p = 0;; p = min(2 * p + 1, k - 1)) {
      bound_by(p);
      if (p == k - 1) break;
    }
    collect();
  }
  const int n = min(n_cand, kMergeCap);
  for (int i = tid; i < n; i += kMergeThreads) {
    const Entry e = list[i];
    int before = 0;
    for (int j = 0; j < n; ++j) before += ahead(list[j], e);
    if (before >= k) continue;
    if (ROW) {
      row_cand[row0 * k + before] = Cand{e.z, e.id};
    } else {
      const int64_t at = (int64_t)group * k + before;
      out_scores[at] = (float)e.score, out_seq[at] = (int32_t)(row0 + e.beam), out_tokens[at] = e.id;
    }
  }
  for (int i = n + tid; i < k; i += kMergeThreads) {
    if (ROW) {
      row_cand[row0 * k + i] = Cand{-INFINITY, -1};
    } else {
      const int64_t at = (int64_t)group * k + i;
      out_scores[at] = -INFINITY, out_seq[at] = out_tokens[at] = -1;
    }
  }
}

constexpr int kSmallSeg = kThreads * 4 * 4, kLargeSeg = kThreads * 4 * 8;

// Longer segments where there are many rows.
int seg_of(int rows, int n_vocab) {
  return (int64_t)rows * n_vocab > (int64_t)kLargeSeg * 1024 ? kLargeSeg : kSmallSeg;
}
int segs_of(int rows, int n_vocab) { return (n_vocab + seg_of(rows, n_vocab) - 1) / seg_of(rows, n_vocab); }

}  // namespace

size_t beam_workspace(int n_group, int beams, int n_vocab, int k) {
  const int64_t rows = (int64_t)n_group * beams, lists = rows * ((n_vocab + kSmallSeg - 1) / kSmallSeg + 1);
  return (size_t)lists * (sizeof(Stat) + (size_t)k * sizeof(Cand));
}

void beam_select(hipStream_t s, const float* logits, int64_t stride, int n_group, int beams, int n_vocab, const float* scores,
                 const int32_t* done, int eos, int k, float* out_scores, int32_t* out_seq, int32_t* out_tokens,
                 void* workspace) {
  const int rows = n_group * beams, segs = segs_of(rows, n_vocab);
  Beams B{logits, stride, scores, done, n_vocab, segs, k, beams, eos};
  Stat* stats = static_cast<Stat*>(workspace);
  Stat* row_stat = stats + (int64_t)rows * segs;
  Cand* cands = reinterpret_cast<Cand*>(row_stat + rows);
  Cand* row_cand = cands + (int64_t)rows * segs * k;
  auto go = [&]<int Q, int PARTS>() {
    hipLaunchKernelGGL((k_beam_rows<Q, PARTS>), dim3((unsigned)(rows * segs)), dim3(kThreads), 0, s, B, stats, cands);
    check_launch("beam_select rows");
  };
  const bool large = seg_of(rows, n_vocab) == kLargeSeg;
  if (k <= 16) large ? go.template operator()<8, 64>() : go.template operator()<4, 64>();
  else large ? go.template operator()<8, 256>() : go.template operator()<4, 256>();
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
