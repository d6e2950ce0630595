// Verification of drafted tokens against the target's probabilities, the random numbers given (speculative sampling):
// draft j of a lane is accepted iff Q_j(d) > 0 and u_j Q_j(d) < P_j(d), up to the first refusal; the next token is drawn
// from max(P_j - Q_j, 0) there, or from the last row's P where every draft was accepted. P and Q are softmax(logits / T)
// over the whole vocabulary (mk_verify), or what mk_sample_draw makes of rows cut to their top k (mk_verify_topk).
//
// Whole vocabulary: every probability, sum and running sum is held in 64 bits. The draw walks a running sum over
// 150 thousand tokens, whose steps are as small as the rounding of 32-bit sums: in 32 bits about one draw in a hundred
// would land on a neighbouring token. Three launches: k_rows reads every row once, in segments of 4096 logits (their
// maximum, its first place, and the sum of exp((z - max) / T)); k_excess makes each lane's decisions from those (every
// workgroup of a lane for itself: a few hundred numbers) and sums the excess of its segment of the row that the next
// token comes from; k_pick finds the segment and the token.
#include <cfloat>

#include "ctx.h"
#include "ops.h"

namespace mk {
namespace {

constexpr int kThreads = 256;
constexpr int kPer = 16;               // logits per thread
constexpr int kSeg = kThreads * kPer;  // logits per segment
constexpr int kMaxDraft = MK_VERIFY_MAX_DRAFT;

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
__device__ __forceinline__ float clean(float z) { return z != z ? -INFINITY : fminf(z, FLT_MAX); }

__device__ __forceinline__ double weight(float z, float max, double inv_t) {
  return z == -INFINITY ? 0.0 : exp(((double)z - (double)max) * inv_t);
}

// The larger maximum, at its first place; sums brought to it.
__device__ __forceinline__ Stat join(const Stat& a, const Stat& b, double inv_t) {
  if (a.at < 0) return b;
  if (b.at < 0) return a;
  Stat r;
  r.max = fmaxf(a.max, b.max);
  r.at = a.max == b.max ? min(a.at, b.at) : a.max > b.max ? a.at : b.at;
  r.sum = inv_t > 0.0 ? a.sum * weight(a.max, r.max, inv_t) + b.sum * weight(b.max, r.max, inv_t) : 0.0;
  return r;
}
__device__ __forceinline__ Stat shfl_xor(const Stat& s, int m) {
  return Stat{__shfl_xor(s.sum, m), __shfl_xor(s.max, m), __shfl_xor(s.at, m)};
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m);
  return v;
}

struct Rows {
  const float* p;
  int64_t p_stride;
  int n_rows;
  const float* q;  // NULL: every draft is certain
  int64_t q_stride;
  int n_drafts, V;
};

// A lane whose parameters do not fit the call is left out: accepted -1, tokens -1.
__device__ __forceinline__ bool lane_ok(const mk_verify_lane& l, int max_draft, int n_rows, int n_drafts) {
  return l.n_draft >= 0 && l.n_draft <= max_draft && l.row >= 0 && l.row < n_rows - l.n_draft && l.first >= 0 &&
         l.first <= n_drafts - l.n_draft;
}

// Thread i's logits i, i + 256, .. of a segment (past the row: -inf).
__device__ __forceinline__ void load_segment(const float* row, int seg, int V, float (&z)[kPer]) {
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int at = seg * kSeg + i * kThreads + (int)threadIdx.x;
    z[i] = at < V ? clean(row[at]) : -INFINITY;
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
  float z[kPer];
  load_segment(row, seg, R.V, z);
  float m = z[0];
#pragma unroll
  for (int i = 1; i < kPer; ++i) m = fmaxf(m, z[i]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  __shared__ float ms[4];
  __shared__ double ss[4];
  __shared__ int as[4];
  const int w = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) ms[w] = m;
  __syncthreads();
  m = fmaxf(fmaxf(ms[0], ms[1]), fmaxf(ms[2], ms[3]));
  const double inv_t = L.temperature > 0.0f ? 1.0 / (double)L.temperature : 0.0;
  double sum = 0.0;
  int at = INT32_MAX;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (z[i] == m) at = min(at, seg * kSeg + i * kThreads + (int)threadIdx.x);
    if (inv_t > 0.0) sum += weight(z[i], m, inv_t);
  }
  sum = wave_sum(sum);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) at = min(at, __shfl_xor(at, o));
  if ((threadIdx.x & 63) == 0) ss[w] = sum, as[w] = at;
  __syncthreads();
  if (threadIdx.x == 0)
    stats[(int64_t)blockIdx.x * gridDim.y + seg] =
        Stat{(ss[0] + ss[1]) + (ss[2] + ss[3]), m,
             m == -INFINITY ? -1 : min(min(as[0], as[1]), min(as[2], as[3]))};
}

// P(x) of a row from its statistics.
__device__ __forceinline__ double prob(const Stat& s, float z, int x, double inv_t) {
  if (s.at < 0) return 0.0;
  return inv_t > 0.0 ? weight(z, s.max, inv_t) / s.sum : x == s.at ? 1.0 : 0.0;
}

// What of token x the next token is drawn by.
__device__ __forceinline__ double excess(const Choice& c, float zp, float zq, bool has_q, int x, double inv_t) {
  const double p = prob(c.p, zp, x, inv_t);
  if (!c.refused) return p;
  const double q = has_q ? prob(c.q, zq, x, inv_t) : x == c.draft ? 1.0 : 0.0;
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
  const double inv_t = L.temperature > 0.0f ? 1.0 / (double)L.temperature : 0.0;
  __shared__ Stat row_s[2 * kMaxDraft + 1];
  __shared__ int stop_s;
  if (threadIdx.x == 0) stop_s = L.n_draft;
  // Rows of the lane in turn over the waves: their segments joined.
  const int rows = L.n_draft + 1 + (R.q ? L.n_draft : 0);
  for (int r = w; r < rows; r += 4) {
    const int j = r <= L.n_draft ? r : max_draft + r - L.n_draft;
    const Stat* s = stats + ((int64_t)li * per + j) * segs;
    Stat a{0.0, -INFINITY, -1};
    for (int i = lane; i < segs; i += 64) a = join(a, s[i], inv_t);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) a = join(a, shfl_xor(a, o), inv_t);
    if (lane == 0) row_s[r] = a;
  }
  __syncthreads();
  for (int j = threadIdx.x; j < L.n_draft; j += kThreads) {
    const int d = drafts[L.first + j];
    double p = 0.0, q = 1.0;
    if (d >= 0 && d < R.V) {
      p = prob(row_s[j], clean(R.p[(int64_t)(L.row + j) * R.p_stride + d]), d, inv_t);
      if (R.q) q = prob(row_s[L.n_draft + 1 + j], clean(R.q[(int64_t)(L.first + j) * R.q_stride + d]), d, inv_t);
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
  float zp[kPer], zq[kPer];
  load_segment(R.p + (int64_t)(L.row + c.n_acc) * R.p_stride, seg, R.V, zp);
  if (both) load_segment(R.q + (int64_t)(L.first + c.n_acc) * R.q_stride, seg, R.V, zq);
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int x = seg * kSeg + i * kThreads + (int)threadIdx.x;
    if (x < R.V) sum += excess(c, zp[i], both ? zq[i] : 0.0f, R.q != nullptr, x, inv_t);
  }
  sum = wave_sum(sum);
  __shared__ double ss[4];
  if (lane == 0) ss[w] = sum;
  __syncthreads();
  if (threadIdx.x == 0) sums[(int64_t)li * segs + seg] = (ss[0] + ss[1]) + (ss[2] + ss[3]);
}

// The first token in order whose running sum reaches v times the total; one workgroup per lane.
__global__ __launch_bounds__(kThreads) void k_pick(Rows R, const mk_verify_lane* __restrict__ lanes, int max_draft,
                                                   const double* __restrict__ u_next,
                                                   const Choice* __restrict__ choices, const double* __restrict__ sums,
                                                   int segs, int32_t* __restrict__ tokens, float* __restrict__ probs) {
  const int li = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const mk_verify_lane L = lanes[li];
  if (!lane_ok(L, max_draft, R.n_rows, R.n_drafts)) return;
  Choice c = choices[li];
  const double inv_t = L.temperature > 0.0f ? 1.0 / (double)L.temperature : 0.0;
  const double v = u_next[li];
  const float* prow = R.p + (int64_t)(L.row + c.n_acc) * R.p_stride;
  const float* qrow = c.refused && R.q ? R.q + (int64_t)(L.first + c.n_acc) * R.q_stride : nullptr;
  __shared__ double ss[4];
  __shared__ int pick_s, last_s;
  const double* lane_sums = sums + (int64_t)li * segs;
  double total = 0.0;
  for (int i = 0; i < segs; ++i) total += lane_sums[i];
  bool walk = false;  // P itself, segment by segment: no segment sums of it are at hand
  if (!(total > 0.0) && c.refused) {
    c.refused = 0;
    qrow = nullptr;
    walk = true;
    total = 1.0;
  }
  const double goal = v * total;
  double run = 0.0;
  int pick = -1, last = -1;
  for (int seg = 0; seg < segs && pick < 0; ++seg) {
    // Past segments whose sum stays below the goal, unless none follows with anything in it.
    if (!walk) {
      const double s = lane_sums[seg];
      if (!(s > 0.0)) continue;
      bool more = false;
      if (!(run + s >= goal))
        for (int k = seg + 1; k < segs && !more; ++k) more = lane_sums[k] > 0.0;
      if (more) {
        run += s;
        continue;
      }
    }
    // Thread i holds 16 consecutive tokens; their running sums through the waves.
    double r[kPer];
    double mine = 0.0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int x = seg * kSeg + tid * kPer + i;
      r[i] = x < R.V ? excess(c, clean(prow[x]), qrow ? clean(qrow[x]) : 0.0f, R.q != nullptr, x, inv_t) : 0.0;
      mine += r[i];
    }
    double scan = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double t = __shfl_up(scan, o);
      if (lane >= o) scan += t;
    }
    if (tid == 0) pick_s = INT32_MAX, last_s = -1;
    __syncthreads();
    if (lane == 63) ss[w] = scan;
    __syncthreads();
    double before = run + (scan - mine);
    for (int k = 0; k < w; ++k) before += ss[k];
    int hit = INT32_MAX, tail = -1;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      before += r[i];
      const int x = seg * kSeg + tid * kPer + i;
      if (r[i] > 0.0) {
        tail = x;
        if (before >= goal && hit == INT32_MAX) hit = x;
      }
    }
    if (hit != INT32_MAX) atomicMin(&pick_s, hit);
    if (tail >= 0) atomicMax(&last_s, tail);
    __syncthreads();
    if (pick_s != INT32_MAX) pick = pick_s;
    if (last_s >= 0) last = last_s;
    run += ((ss[0] + ss[1]) + ss[2]) + ss[3];
    __syncthreads();
  }
  if (pick < 0) pick = last;  // rounding left the goal above the whole sum: the last token with any
  if (tid == 0) {
    tokens[(int64_t)li * (max_draft + 1) + c.n_acc] = pick;
    if (probs)
      probs[(int64_t)li * (max_draft + 1) + c.n_acc] =
          pick < 0 ? 0.0f : (float)prob(c.p, clean(prow[pick]), pick, inv_t);
  }
}

// ---- rows cut to their top k ----

constexpr int kMaxK = 1024;

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

// One workgroup per lane: wave w decides drafts w, w + 4, ..; wave 0 draws the next token.
__global__ __launch_bounds__(kThreads) void k_verify_topk(Cands P, Cands Q, const mk_verify_lane* __restrict__ lanes,
                                                          int max_draft, int n_drafts,
                                                          const int32_t* __restrict__ drafts,
                                                          const double* __restrict__ u,
                                                          const double* __restrict__ u_next,
                                                          int32_t* __restrict__ accepted, int32_t* __restrict__ tokens,
                                                          float* __restrict__ probs) {
  const int li = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const mk_verify_lane L = lanes[li];
  int32_t* tok = tokens + (int64_t)li * (max_draft + 1);
  float* pr = probs ? probs + (int64_t)li * (max_draft + 1) : nullptr;
  const bool ok = lane_ok(L, max_draft, P.n, n_drafts);
  __shared__ int stop_s;
  __shared__ float pd_s[kMaxDraft];
  __shared__ int32_t q_id[kMaxK];
  __shared__ float q_pr[kMaxK];
  if (tid == 0) stop_s = ok ? L.n_draft : -1;
  __syncthreads();
  const float t = L.temperature;
  if (ok)
    for (int j = w; j < L.n_draft; j += 4) {
      const int d = drafts[L.first + j];
      const float* pv = P.values + (int64_t)(L.row + j) * P.k;
      const float p = prob_in(pv, P.ids + (int64_t)(L.row + j) * P.k, head_of(pv, P.k, L), d, t);
      float q = 1.0f;
      if (Q.values) {
        const float* qv = Q.values + (int64_t)(L.first + j) * Q.k;
        q = prob_in(qv, Q.ids + (int64_t)(L.first + j) * Q.k, head_of(qv, Q.k, L), d, t);
      }
      if (lane == 0) {
        pd_s[j] = p;
        if (!(q > 0.0f && u[L.first + j] * (double)q < (double)p)) atomicMin(&stop_s, j);
      }
    }
  __syncthreads();
  const int n_acc = stop_s;
  for (int j = tid; j <= max_draft; j += kThreads) {
    if (j == n_acc) continue;
    tok[j] = j < n_acc ? drafts[L.first + j] : -1;
    if (pr) pr[j] = j < n_acc ? pd_s[j] : 0.0f;
  }
  if (tid == 0) accepted[li] = n_acc;
  if (!ok) return;
  const bool refused = n_acc < L.n_draft;
  const float* pv = P.values + (int64_t)(L.row + n_acc) * P.k;
  const int32_t* pi = P.ids + (int64_t)(L.row + n_acc) * P.k;
  // The draft's probabilities at the refusal, by candidate.
  int q_n = 0;
  if (refused && Q.values) {
    const float* qv = Q.values + (int64_t)(L.first + n_acc) * Q.k;
    const Head qh = head_of(qv, Q.k, L);
    q_n = qh.keep;
    for (int i = tid; i < q_n; i += kThreads) {
      q_id[i] = Q.ids[(int64_t)(L.first + n_acc) * Q.k + i];
      q_pr[i] = cand_prob(qh, qv[i], qv[0], i, t);
    }
  } else if (refused) {
    q_n = 1;
    if (tid == 0) q_id[0] = drafts[L.first + n_acc], q_pr[0] = 1.0f;
  }
  __syncthreads();
  if (w != 0) return;
  const Head ph = head_of(pv, P.k, L);
  auto left = [&](int i, bool over) {
    const float p = cand_prob(ph, pv[i], pv[0], i, t);
    float q = 0.0f;
    if (over)
      for (int k = 0; k < q_n; ++k)
        if (q_id[k] == pi[i]) q = q_pr[k];
    return fmaxf(p - q, 0.0f);
  };
  double total = 0.0;
  bool over = refused;
  for (;;) {
    total = 0.0;
    for (int c = 0; c < ph.keep; c += 64) total += wave_sum(c + lane < ph.keep ? (double)left(c + lane, over) : 0.0);
    if (total > 0.0 || !over) break;
    over = false;  // nothing is left over the draft's probabilities: the row itself
  }
  const double goal = u_next[li] * total;
  double run = 0.0;
  int pick = -1, last = -1;
  for (int c = 0; c < ph.keep && pick < 0; c += 64) {
    const double r = c + lane < ph.keep ? (double)left(c + lane, over) : 0.0;
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
         lanes * segs * sizeof(double);
}

void verify(hipStream_t s, const float* p, int64_t p_stride, int n_rows, const float* q, int64_t q_stride, int n_drafts,
            int n_vocab, const mk_verify_lane* lanes, int n_lanes, int max_draft, const int32_t* drafts, const double* u,
            const double* u_next, int32_t* accepted, int32_t* tokens, float* probs, void* workspace) {
  const int segs = segments(n_vocab), per = 2 * max_draft + 1;
  Stat* stats = static_cast<Stat*>(workspace);
  Choice* choices = reinterpret_cast<Choice*>(stats + (size_t)n_lanes * per * segs);
  double* sums = reinterpret_cast<double*>(reinterpret_cast<uint8_t*>(choices) + up16(n_lanes * sizeof(Choice)));
  const Rows R{p, p_stride, n_rows, q, q_stride, n_drafts, n_vocab};
  hipLaunchKernelGGL(k_rows, dim3(n_lanes * per, segs), dim3(kThreads), 0, s, R, lanes, max_draft, stats);
  check_launch("verify rows");
  hipLaunchKernelGGL(k_excess, dim3(n_lanes, segs), dim3(kThreads), 0, s, R, lanes, max_draft, drafts, u, stats, choices,
                     sums, accepted, tokens, probs);
  check_launch("verify excess");
  hipLaunchKernelGGL(k_pick, dim3(n_lanes), dim3(kThreads), 0, s, R, lanes, max_draft, u_next, choices, sums, segs,
                     tokens, probs);
  check_launch("verify pick");
}

void verify_topk(hipStream_t s, const float* p_values, const int32_t* p_ids, int p_k, int n_rows, const float* q_values,
                 const int32_t* q_ids, int q_k, int n_drafts, const mk_verify_lane* lanes, int n_lanes, int max_draft,
                 const int32_t* drafts, const double* u, const double* u_next, int32_t* accepted, int32_t* tokens,
                 float* probs) {
  hipLaunchKernelGGL(k_verify_topk, dim3(n_lanes), dim3(kThreads), 0, s, Cands{p_values, p_ids, p_k, n_rows},
                     Cands{q_values, q_ids, q_k, n_drafts}, lanes, max_draft, n_drafts, drafts, u, u_next, accepted,
                     tokens, probs);
  check_launch("verify_topk");
}

}  // namespace mk
