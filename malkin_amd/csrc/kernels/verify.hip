// Verification of drafted tokens against the target's probabilities, the random numbers given (speculative sampling):
// draft j of a lane is accepted iff Q_j(d) > 0 and u_j Q_j(d) < P_j(d), up to the first refusal; the next token is drawn
// from max(P_j - Q_j, 0) there, or from the last row's P where every draft was accepted. P and Q are softmax(logits / T)
// over the whole vocabulary (mk_verify), or what mk_sample_draw makes of rows cut to their top k (mk_verify_topk).
//
// Whole vocabulary: every probability, sum and running sum is held in 64 bits. The draw walks a running sum over
// 150 thousand tokens, whose steps are as small as the rounding of 32-bit sums: in 32 bits about one draw in a hundred
// would land on a neighbouring token. Three launches: k_rows reads every row once, in segments of 4096 logits (their
// maximum, its first place, and the sum of exp((z - max) / T)); k_excess makes each lane's decisions from those (every
// workgroup of a lane for itself: a few hundred numbers) and sums the excess over 1024 tokens at a time of the row that
// the next token comes from; k_pick finds the block and the token.
#include <cfloat>

#include "ctx.h"
#include "ops.h"

namespace mk {
namespace {

constexpr int kThreads = 256;
constexpr int kQuads = 4;                     // logits per thread, in fours
constexpr int kBlock = 64 * 4 * kQuads;       // logits per wave, contiguous
constexpr int kSeg = kThreads / 64 * kBlock;  // logits per segment
constexpr int kMaxDraft = MK_VERIFY_MAX_DRAFT;

typedef float v4f __attribute__((ext_vector_type(4)));

struct Stat {  // a segment of a row, or a row
  double sum;  // of exp((z - max) / T); T <= 0: unused
  float max;
  int32_t at;  // first place of max; -1: nothing but -inf
};
struct Choice {  // of a lane
  int32_t n_acc;
  int32_t refused;  // a draft was: the excess over Q counts
  int32_t draft;    // that draft
  int32_t pad;
  Stat p, q;
};

// NaN counts as -inf, +inf as the largest float.
__device__ __forceinline__ float clean(float z) { return fminf(fmaxf(z, -INFINITY), FLT_MAX); }

// 2^t for t <= about 1000: t = n + f, |f| <= 1/2, and the series of e^(f ln 2) to f^11, whose remainder is below
// (ln 2 / 2)^12 / 12! = 7e-15 of it. Below 2^-1074 (-inf included) it is 0.
__device__ __forceinline__ double pow2(double t) {
  t = fmax(t, -1100.0);
  const double n = __builtin_rint(t), f = t - n;
  constexpr double c[12] = {1.0,
                            6.931471805599453094e-1,
                            2.402265069591007123e-1,
                            5.550410866482157995e-2,
                            9.618129107628477232e-3,
                            1.333355814642844343e-3,
                            1.540353039338160996e-4,
                            1.525273380405984028e-5,
                            1.321548679014430949e-6,
                            1.017808600923969973e-7,
                            7.054911620801123330e-9,
                            4.445538271870811498e-10};
  double p = c[11];
#pragma unroll
  for (int i = 10; i >= 0; --i) p = __builtin_fma(p, f, c[i]);
  return __builtin_amdgcn_ldexp(p, (int)n);
}

// Logits to powers of two: log2(e) / T; 0 where T <= 0.
__device__ __forceinline__ double per_unit(const mk_verify_lane& l) {
  return l.temperature > 0.0f ? 1.4426950408889634074 / (double)l.temperature : 0.0;
}
__device__ __forceinline__ double weight(float z, float max, double c) {
  return pow2(((double)z - (double)fmaxf(max, -FLT_MAX)) * c);
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m);
  return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) v = fmaxf(v, __shfl_xor(v, m));
  return v;
}
// A value per lane (none: at -1), joined over the wave: the maximum, its first place, the sums brought to it.
__device__ __forceinline__ Stat wave_join(Stat s, double c) {
  Stat r;
  r.max = wave_max(s.at < 0 ? -INFINITY : s.max);
  int at = s.at >= 0 && s.max == r.max ? s.at : INT32_MAX;
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) at = min(at, __shfl_xor(at, m));
  r.at = at == INT32_MAX ? -1 : at;
  r.sum = c > 0.0 ? wave_sum(s.at < 0 ? 0.0 : s.sum * weight(s.max, r.max, c)) : 0.0;
  return r;
}
// The same of a row's segments, by one wave.
__device__ __forceinline__ Stat row_stat(const Stat* s, int segs, double c) {
  const int lane = threadIdx.x & 63;
  const Stat none{0.0, -INFINITY, -1};
  Stat a = wave_join(lane < segs ? s[lane] : none, c);
  for (int i = 64; i < segs; i += 64) {  // lane 63 carries the earlier ones
    const Stat b = i + lane < segs && lane < 63 ? s[i + lane] : none;
    a = wave_join(lane == 63 ? a : b, c);
    if (i + 63 < segs) {
      const Stat last = s[i + 63];
      a = wave_join(lane == 0 ? a : lane == 1 ? last : none, c);
    }
  }
  return a;
}

struct Rows {
  const float* p;
  int64_t p_stride;
  int n_rows;
  const float* q;  // NULL: every draft is certain
  int64_t q_stride;
  int n_drafts, V;
  bool vec;
};

// A lane whose parameters do not fit the call is left out: accepted -1, tokens -1.
__device__ __forceinline__ bool lane_ok(const mk_verify_lane& l, int max_draft, int n_rows, int n_drafts) {
  return l.n_draft >= 0 && l.n_draft <= max_draft && l.row >= 0 && l.row < n_rows - l.n_draft && l.first >= 0 &&
         l.first <= n_drafts - l.n_draft;
}

// Logit of place i (quad, value) of this thread in a segment.
__device__ __forceinline__ int place(int seg, int quad, int e) {
  return seg * kSeg + (threadIdx.x >> 6) * kBlock + quad * 256 + (threadIdx.x & 63) * 4 + e;
}
// A segment's logits, a wave's 1024 contiguous (past the row: -inf). vec: rows are 16-byte aligned, V a multiple of 4.
__device__ __forceinline__ void load_segment(const float* row, int seg, int V, bool vec, float (&z)[kQuads][4]) {
  if (vec) {
#pragma unroll
    for (int i = 0; i < kQuads; ++i) {
      const int at = place(seg, i, 0);
      const v4f v = *reinterpret_cast<const v4f*>(row + (at < V ? at : 0));
#pragma unroll
      for (int e = 0; e < 4; ++e) z[i][e] = at < V ? clean(v[e]) : -INFINITY;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kQuads; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int at = place(seg, i, e);
        z[i][e] = at < V ? clean(row[at]) : -INFINITY;
      }
  }
}

// Grid (lanes x (2 max_draft + 1), segments): rows j <= max_draft of a lane are the target's, the others the draft's.
__global__ __launch_bounds__(kThreads) void k_rows(Rows R, const mk_verify_lane* __restrict__ lanes, int max_draft,
                                                   Stat* __restrict__ stats) {
  const int per = 2 * max_draft + 1, li = blockIdx.x / per, j = blockIdx.x % per, seg = blockIdx.y;
  const mk_verify_lane L = lanes[li];
  if (!lane_ok(L, max_draft, R.n_rows, R.n_drafts)) return;
  const bool draft = j > max_draft;
  const int jj = draft ? j - max_draft - 1 : j;
  if (draft ? (jj >= L.n_draft || !R.q) : jj > L.n_draft) return;
  const float* row = draft ? R.q + (int64_t)(L.first + jj) * R.q_stride : R.p + (int64_t)(L.row + jj) * R.p_stride;
  float z[kQuads][4];
  load_segment(row, seg, R.V, R.vec, z);
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < kQuads; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) m = fmaxf(m, z[i][e]);
  m = wave_max(m);  // each wave against its own maximum: no barrier before the end
  const double c = per_unit(L);
  double sum = 0.0;
  int at = m == -INFINITY ? -1 : 0;
  if (c > 0.0) {
    if (at == 0) {
      const double md = (double)m;
#pragma unroll
      for (int i = 0; i < kQuads; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum += pow2(((double)z[i][e] - md) * c);
    }
    sum = wave_sum(sum);
  } else if (at == 0) {
    at = INT32_MAX;
#pragma unroll
    for (int i = 0; i < kQuads; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) at = z[i][e] == m ? min(at, place(seg, i, e)) : at;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) at = min(at, __shfl_xor(at, o));
  }
  __shared__ Stat ws[kThreads / 64];
  const int lane = threadIdx.x & 63;
  if (lane == 0) ws[threadIdx.x >> 6] = Stat{sum, m, at};
  __syncthreads();
  if (threadIdx.x >= 64) return;
  const Stat s = wave_join(lane < kThreads / 64 ? ws[lane] : Stat{0.0, -INFINITY, -1}, c);
  if (lane == 0) stats[(int64_t)blockIdx.x * gridDim.y + seg] = s;
}

// P(x) of a row from its statistics.
__device__ __forceinline__ double prob(const Stat& s, float z, int x, double c) {
  if (s.at < 0) return 0.0;
  return c > 0.0 ? weight(z, s.max, c) / s.sum : x == s.at ? 1.0 : 0.0;
}

// What of token x the next token is drawn by.
__device__ __forceinline__ double excess(const Choice& c, float zp, float zq, bool has_q, int x, double unit) {
  const double p = prob(c.p, zp, x, unit);
  if (!c.refused) return p;
  const double q = has_q ? prob(c.q, zq, x, unit) : x == c.draft ? 1.0 : 0.0;
  return fmax(p - q, 0.0);
}

__global__ __launch_bounds__(kThreads) void k_excess(Rows R, const mk_verify_lane* __restrict__ lanes, int max_draft,
                                                     const int32_t* __restrict__ drafts, const double* __restrict__ u,
                                                     const Stat* __restrict__ stats, Choice* __restrict__ choices,
                                                     double* __restrict__ sums, int32_t* __restrict__ accepted,
                                                     int32_t* __restrict__ tokens, float* __restrict__ probs) {
  const int li = blockIdx.x, segs = gridDim.y, seg = blockIdx.y, per = 2 * max_draft + 1;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const mk_verify_lane L = lanes[li];
  int32_t* tok = tokens + (int64_t)li * (max_draft + 1);
  float* pr = probs ? probs + (int64_t)li * (max_draft + 1) : nullptr;
  if (!lane_ok(L, max_draft, R.n_rows, R.n_drafts)) {
    if (seg == 0) {
      for (int j = threadIdx.x; j <= max_draft; j += kThreads) {
        tok[j] = -1;
        if (pr) pr[j] = 0.0f;
      }
      if (threadIdx.x == 0) accepted[li] = -1;
    }
    return;
  }
  const double unit = per_unit(L);
  __shared__ Stat row_s[2 * kMaxDraft + 1];
  __shared__ int stop_s;
  if (threadIdx.x == 0) stop_s = L.n_draft;
  const int rows = L.n_draft + 1 + (R.q ? L.n_draft : 0);
  for (int r = w; r < rows; r += kThreads / 64) {
    const int j = r <= L.n_draft ? r : max_draft + r - L.n_draft;
    const Stat a = row_stat(stats + ((int64_t)li * per + j) * segs, segs, unit);
    if (lane == 0) row_s[r] = a;
  }
  __syncthreads();
  for (int j = threadIdx.x; j < L.n_draft; j += kThreads) {
    const int d = drafts[L.first + j];
    double p = 0.0, q = 1.0;
    if (d >= 0 && d < R.V) {
      p = prob(row_s[j], clean(R.p[(int64_t)(L.row + j) * R.p_stride + d]), d, unit);
      if (R.q) q = prob(row_s[L.n_draft + 1 + j], clean(R.q[(int64_t)(L.first + j) * R.q_stride + d]), d, unit);
    }
    if (!(q > 0.0 && u[L.first + j] * q < p)) atomicMin(&stop_s, j);
    if (seg == 0 && pr) pr[j] = (float)p;  // past the refusal cleared below
  }
  __syncthreads();
  Choice c;
  c.n_acc = stop_s;
  c.refused = c.n_acc < L.n_draft;
  c.draft = c.refused ? drafts[L.first + c.n_acc] : -1;
  c.p = row_s[c.n_acc];
  c.q = c.refused && R.q ? row_s[L.n_draft + 1 + c.n_acc] : Stat{0.0, -INFINITY, -1};
  if (seg == 0) {
    for (int j = threadIdx.x; j <= max_draft; j += kThreads) {
      tok[j] = j < c.n_acc ? drafts[L.first + j] : -1;
      if (pr && j >= c.n_acc) pr[j] = 0.0f;
    }
    if (threadIdx.x == 0) {
      accepted[li] = c.n_acc;
      choices[li] = c;
    }
  }
  const bool both = c.refused && R.q;
  float zp[kQuads][4], zq[kQuads][4];
  load_segment(R.p + (int64_t)(L.row + c.n_acc) * R.p_stride, seg, R.V, R.vec, zp);
  if (both) load_segment(R.q + (int64_t)(L.first + c.n_acc) * R.q_stride, seg, R.V, R.vec, zq);
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < kQuads; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int x = place(seg, i, e);
      if (x < R.V) sum += excess(c, zp[i][e], both ? zq[i][e] : 0.0f, R.q != nullptr, x, unit);
    }
  sum = wave_sum(sum);
  if (lane == 0) sums[((int64_t)li * segs + seg) * (kThreads / 64) + w] = sum;
}

// The inclusive running sum over the workgroup's threads, and in `total` that of all.
__device__ __forceinline__ double block_scan(double v, double* wave_s, double& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double t = __shfl_up(v, o);
    if (lane >= o) v += t;
  }
  __syncthreads();  // the last scan's sums have been read
  if (lane == 63) wave_s[w] = v;
  __syncthreads();
  total = 0.0;
#pragma unroll
  for (int i = 0; i < kThreads / 64; ++i) {
    if (i == w) v += total;
    total += wave_s[i];
  }
  return v;
}

// The first token in order whose running sum reaches v times the total; one workgroup per lane.
__global__ __launch_bounds__(kThreads) void k_pick(Rows R, const mk_verify_lane* __restrict__ lanes, int max_draft,
                                                   const double* __restrict__ u_next,
                                                   const Choice* __restrict__ choices, const double* __restrict__ sums,
                                                   int blocks, int32_t* __restrict__ tokens,
                                                   float* __restrict__ probs) {
  const int li = blockIdx.x, tid = threadIdx.x;
  const mk_verify_lane L = lanes[li];
  if (!lane_ok(L, max_draft, R.n_rows, R.n_drafts)) return;
  Choice c = choices[li];
  const double unit = per_unit(L);
  const float* prow = R.p + (int64_t)(L.row + c.n_acc) * R.p_stride;
  const float* qrow = c.refused && R.q ? R.q + (int64_t)(L.first + c.n_acc) * R.q_stride : nullptr;
  __shared__ double wave_s[kThreads / 64];
  __shared__ int found_s, last_s;
  const double* lane_sums = sums + (int64_t)li * blocks;
  double total = 0.0;
  for (int b0 = 0; b0 < blocks; b0 += kThreads) {
    double t;
    block_scan(b0 + tid < blocks ? lane_sums[b0 + tid] : 0.0, wave_s, t);
    total += t;
  }
  // Nothing over Q: P itself, whose blocks have no sums at hand.
  const bool walk = !(total > 0.0) && c.refused;
  if (walk) c.refused = 0, qrow = nullptr, total = 1.0;
  const double goal = u_next[li] * total;
  // The block: the first whose running sum reaches the goal (rounding aside, the last with anything).
  double run = 0.0;
  int first = 0, end = blocks;
  if (!walk) {
    int block = -1, last = -1;
    double before = 0.0;
    for (int b0 = 0; b0 < blocks && block < 0; b0 += kThreads) {
      const double s = b0 + tid < blocks ? lane_sums[b0 + tid] : 0.0;
      double t;
      const double scan = block_scan(s, wave_s, t);
      if (tid == 0) found_s = INT32_MAX, last_s = -1;
      __syncthreads();
      if (s > 0.0) {
        atomicMax(&last_s, b0 + tid);
        if (before + scan >= goal) atomicMin(&found_s, b0 + tid);
      }
      __syncthreads();
      if (last_s >= 0) last = last_s;
      if (found_s != INT32_MAX) block = found_s;
      before += t;
    }
    if (block < 0) block = last;
    if (block >= 0) {
      // What lies before it, summed in the same order by every thread.
      for (int b0 = 0; b0 < block; b0 += kThreads) {
        double t;
        block_scan(b0 + tid < block ? lane_sums[b0 + tid] : 0.0, wave_s, t);
        run += t;
      }
      first = block, end = block + 1;
    } else {
      end = 0;
    }
  }
  int pick = -1, last = -1;
  for (int b = first; b < end && pick < 0; ++b) {
    // Four consecutive tokens per thread.
    double r[4], mine = 0.0;
    const int x0 = b * kBlock + 4 * tid;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int x = x0 + e;
      r[e] = x < R.V ? excess(c, clean(prow[x]), qrow ? clean(qrow[x]) : 0.0f, R.q != nullptr, x, unit) : 0.0;
      mine += r[e];
    }
    double t;
    double upto = run + (block_scan(mine, wave_s, t) - mine);
    if (tid == 0) found_s = INT32_MAX, last_s = -1;
    __syncthreads();
    int hit = INT32_MAX, tail = -1;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      upto += r[e];
      if (r[e] > 0.0) {
        tail = x0 + e;
        if (upto >= goal && hit == INT32_MAX) hit = x0 + e;
      }
    }
    if (hit != INT32_MAX) atomicMin(&found_s, hit);
    if (tail >= 0) atomicMax(&last_s, tail);
    __syncthreads();
    if (found_s != INT32_MAX) pick = found_s;
    if (last_s >= 0) last = last_s;
    run += t;
  }
  if (pick < 0) pick = last;  // rounding left the goal above the whole sum: the last token with any
  if (tid == 0) {
    tokens[(int64_t)li * (max_draft + 1) + c.n_acc] = pick;
    if (probs)
      probs[(int64_t)li * (max_draft + 1) + c.n_acc] =
          pick < 0 ? 0.0f : (float)prob(c.p, clean(prow[pick]), pick, unit);
  }
}
static_assert(kBlock == 4 * kThreads, "a block of tokens is four per thread");

// ---- rows cut to their top k ----

constexpr int kMaxK = 1024, kTopkThreads = 512;

struct Cands {
  const float* values;
  const int32_t* ids;
  int k, n;  // candidates per row, rows
};
struct Head {  // what of a row of candidates is kept: the first `keep`, of total weight `sum`
  double sum;
  int32_t keep;
};

__device__ __forceinline__ double cand_weight(float v, float top, float t) {
  return (double)(float)exp((double)((v - top) / t));
}

// One wave: the kept head (sampler.cpp:37-56), 64 candidates at a time, their running sums by a scan.
__device__ __forceinline__ Head head_of(const float* v, int k, const mk_verify_lane& L) {
  const int lane = threadIdx.x & 63;
  if (!(L.temperature > 0.0f)) return Head{1.0, 1};
  const float top = v[0];
  double all = 0.0;
  for (int c = 0; c < k; c += 64)
    all += wave_sum(c + lane < k ? cand_weight(v[c + lane], top, L.temperature) : 0.0);
  const double floor_w = (double)L.min_p * cand_weight(top, top, L.temperature), nucleus = (double)L.top_p * all;
  double run = 0.0;
  for (int c = 0; c < k; c += 64) {
    const int i = c + lane;
    const double w = i < k ? cand_weight(v[i], top, L.temperature) : 0.0;
    double scan = w;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double t = __shfl_up(scan, o);
      if (lane >= o) scan += t;
    }
    scan += run;
    const uint64_t below = __ballot(i < k && i > 0 && w < floor_w), reach = __ballot(i < k && scan >= nucleus);
    const int b = below ? __builtin_ctzll(below) : 64, e = reach ? __builtin_ctzll(reach) : 64;
    if (b < 64 || e < 64) {
      // Candidate b is not kept, candidate e is the last; one that is both is below the floor.
      const int last = b <= e ? b - 1 : e;  // in this chunk; -1: the chunk before's last
      return Head{last < 0 ? run : __shfl(scan, last), c + last + 1};
    }
    run = __shfl(scan, min(63, k - 1 - c));
  }
  return Head{run, k};
}

__device__ __forceinline__ float cand_prob(const Head& h, float v, float top, int i, float t) {
  if (i >= h.keep) return 0.0f;
  return t > 0.0f ? (float)(cand_weight(v, top, t) / h.sum) : 1.0f;
}

// Probability of token d in a row (sampler.cpp prob_in), by one wave.
__device__ __forceinline__ float prob_in(const float* v, const int32_t* ids, const Head& h, int d, float t) {
  const int lane = threadIdx.x & 63;
  for (int c = 0; c < h.keep; c += 64) {
    const uint64_t hit = __ballot(c + lane < h.keep && ids[c + lane] == d);
    if (hit) {
      const int i = c + __builtin_ctzll(hit);
      return cand_prob(h, v[i], v[0], i, t);
    }
  }
  return 0.0f;
}

// One workgroup per lane: the rows' heads in turn over the waves, each with the probability of the draft it judges;
// then wave 0 draws the next token.
__global__ __launch_bounds__(kTopkThreads) void k_verify_topk(Cands P, Cands Q, const mk_verify_lane* __restrict__ lanes,
                                                              int max_draft, int n_drafts,
                                                              const int32_t* __restrict__ drafts,
                                                              const double* __restrict__ u,
                                                              const double* __restrict__ u_next,
                                                              int32_t* __restrict__ accepted,
                                                              int32_t* __restrict__ tokens, float* __restrict__ probs) {
  const int li = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const mk_verify_lane L = lanes[li];
  int32_t* tok = tokens + (int64_t)li * (max_draft + 1);
  float* pr = probs ? probs + (int64_t)li * (max_draft + 1) : nullptr;
  const bool ok = lane_ok(L, max_draft, P.n, n_drafts);
  __shared__ int stop_s;
  __shared__ Head head_s[2 * kMaxDraft + 1];  // target rows, then draft rows
  __shared__ float prob_s[2 * kMaxDraft + 1];
  __shared__ int32_t q_id[kMaxK];
  __shared__ float q_pr[kMaxK];
  if (tid == 0) stop_s = ok ? L.n_draft : -1;
  const float t = L.temperature;
  const int rows = ok ? L.n_draft + 1 + (Q.values ? L.n_draft : 0) : 0;
  for (int r = w; r < rows; r += kTopkThreads / 64) {
    const bool draft = r > L.n_draft;
    const int j = draft ? r - L.n_draft - 1 : r, k = draft ? Q.k : P.k;
    const int64_t at = draft ? (int64_t)(L.first + j) * Q.k : (int64_t)(L.row + j) * P.k;
    const float* v = (draft ? Q.values : P.values) + at;
    const Head h = head_of(v, k, L);
    const float p = j < L.n_draft ? prob_in(v, (draft ? Q.ids : P.ids) + at, h, drafts[L.first + j], t) : 0.0f;
    if (lane == 0) head_s[r] = h, prob_s[r] = p;
  }
  __syncthreads();
  if (ok)
    for (int j = tid; j < L.n_draft; j += kTopkThreads) {
      const float p = prob_s[j], q = Q.values ? prob_s[L.n_draft + 1 + j] : 1.0f;
      if (!(q > 0.0f && u[L.first + j] * (double)q < (double)p)) atomicMin(&stop_s, j);
    }
  __syncthreads();
  const int n_acc = stop_s;
  for (int j = tid; j <= max_draft; j += kTopkThreads) {
    if (j == n_acc) continue;
    tok[j] = j < n_acc ? drafts[L.first + j] : -1;
    if (pr) pr[j] = j < n_acc ? prob_s[j] : 0.0f;
  }
  if (tid == 0) accepted[li] = n_acc;
  if (!ok) return;
  const bool refused = n_acc < L.n_draft;
  // The draft's probabilities at the refusal, by candidate.
  int q_n = 0;
  if (refused && Q.values) {
    const int64_t at = (int64_t)(L.first + n_acc) * Q.k;
    const Head qh = head_s[L.n_draft + 1 + n_acc];
    q_n = qh.keep;
    for (int i = tid; i < q_n; i += kTopkThreads) {
      q_id[i] = Q.ids[at + i];
      q_pr[i] = cand_prob(qh, Q.values[at + i], Q.values[at], i, t);
    }
  } else if (refused) {
    q_n = 1;
    if (tid == 0) q_id[0] = drafts[L.first + n_acc], q_pr[0] = 1.0f;
  }
  // What each target candidate is drawn by (at most kMaxK: kept in LDS).
  __shared__ float left_s[kMaxK];
  const float* pv = P.values + (int64_t)(L.row + n_acc) * P.k;
  const int32_t* pi = P.ids + (int64_t)(L.row + n_acc) * P.k;
  const Head ph = head_s[n_acc];
  __syncthreads();
  for (int i = tid; i < ph.keep; i += kTopkThreads) {
    const int id = pi[i];
    float q = 0.0f;
    for (int k = 0; k < q_n; ++k)
      if (q_id[k] == id) q = q_pr[k];
    left_s[i] = fmaxf(cand_prob(ph, pv[i], pv[0], i, t) - q, 0.0f);
  }
  __syncthreads();
  if (w != 0) return;
  double total = 0.0;
  bool over = true;
  auto left = [&](int i) {
    return i >= ph.keep ? 0.0 : over ? (double)left_s[i] : (double)cand_prob(ph, pv[i], pv[0], i, t);
  };
  for (;;) {
    total = 0.0;
    for (int c = 0; c < ph.keep; c += 64) total += wave_sum(left(c + lane));
    if (total > 0.0 || !over) break;
    over = false;  // nothing is left over the draft's probabilities: the row itself
  }
  const double goal = u_next[li] * total;
  double run = 0.0;
  int pick = -1, last = -1;
  for (int c = 0; c < ph.keep && pick < 0; c += 64) {
    const double r = left(c + lane);
    double scan = r;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double s = __shfl_up(scan, o);
      if (lane >= o) scan += s;
    }
    scan += run;
    const uint64_t some = __ballot(r > 0.0), hit = __ballot(r > 0.0 && scan >= goal);
    if (some) last = c + 63 - __builtin_clzll(some);
    if (hit) pick = c + __builtin_ctzll(hit);
    run = __shfl(scan, 63);
  }
  if (pick < 0) pick = last;
  if (lane == 0) {
    tok[n_acc] = pick < 0 ? -1 : pi[pick];
    if (pr) pr[n_acc] = pick < 0 ? 0.0f : cand_prob(ph, pv[pick], pv[0], pick, t);
  }
}

int segments(int V) { return (V + kSeg - 1) / kSeg; }
size_t up16(size_t n) { return (n + 15) & ~(size_t)15; }

}  // namespace

size_t verify_workspace(int n_lanes, int max_draft, int n_vocab) {
  const size_t segs = segments(n_vocab), lanes = n_lanes;
  return lanes * (2 * (size_t)max_draft + 1) * segs * sizeof(Stat) + up16(lanes * sizeof(Choice)) +
         lanes * segs * (kThreads / 64) * sizeof(double);
}

void verify(hipStream_t s, const float* p, int64_t p_stride, int n_rows, const float* q, int64_t q_stride, int n_drafts,
            int n_vocab, const mk_verify_lane* lanes, int n_lanes, int max_draft, const int32_t* drafts, const double* u,
            const double* u_next, int32_t* accepted, int32_t* tokens, float* probs, void* workspace) {
  const int segs = segments(n_vocab), per = 2 * max_draft + 1;
  Stat* stats = static_cast<Stat*>(workspace);
  Choice* choices = reinterpret_cast<Choice*>(stats + (size_t)n_lanes * per * segs);
  double* sums = reinterpret_cast<double*>(reinterpret_cast<uint8_t*>(choices) + up16(n_lanes * sizeof(Choice)));
  auto aligned = [](const float* x, int64_t stride) { return !x || (((uintptr_t)x & 15) == 0 && (stride & 3) == 0); };
  const Rows R{p, p_stride, n_rows, q, q_stride, n_drafts, n_vocab,
               (n_vocab & 3) == 0 && aligned(p, p_stride) && aligned(q, q_stride)};
  hipLaunchKernelGGL(k_rows, dim3(n_lanes * per, segs), dim3(kThreads), 0, s, R, lanes, max_draft, stats);
  check_launch("verify rows");
  hipLaunchKernelGGL(k_excess, dim3(n_lanes, segs), dim3(kThreads), 0, s, R, lanes, max_draft, drafts, u, stats, choices,
                     sums, accepted, tokens, probs);
  check_launch("verify excess");
  hipLaunchKernelGGL(k_pick, dim3(n_lanes), dim3(kThreads), 0, s, R, lanes, max_draft, u_next, choices, sums,
                     segs * (kThreads / 64), tokens, probs);
  check_launch("verify pick");
}

void verify_topk(hipStream_t s, const float* p_values, const int32_t* p_ids, int p_k, int n_rows, const float* q_values,
                 const int32_t* q_ids, int q_k, int n_drafts, const mk_verify_lane* lanes, int n_lanes, int max_draft,
                 const int32_t* drafts, const double* u, const double* u_next, int32_t* accepted, int32_t* tokens,
                 float* probs) {
  hipLaunchKernelGGL(k_verify_topk, dim3(n_lanes), dim3(kTopkThreads), 0, s, Cands{p_values, p_ids, p_k, n_rows},
                     Cands{q_values, q_ids, q_k, n_drafts}, lanes, max_draft, n_drafts, drafts, u, u_next, accepted,
                     tokens, probs);
  check_launch("verify_topk");
}

}  // namespace mk
