// Verification of drafted tokens against the target's probabilities, the random numbers given (speculative sampling):
// draft j of a lane is accepted iff Q_j(d) > 0 and u_j Q_j(d) < P_j(d), up to the first refusal; the next token is drawn
// from max(P_j - Q_j, 0) there, or from the last row's P where every draft was accepted. P and Q are softmax(logits / T)
// over the whole vocabulary (mk_verify), or what mk_sample_draw makes of rows cut to their top k (mk_verify_topk).
//
// Whole vocabulary: every probability, sum and running sum is held in 64 bits. The draw walks a running sum over
// 150 thousand tokens, whose steps are as small as the rounding of 32-bit sums: in 32 bits about one draw in a hundred
// would land on a neighbouring token. Two launches: k_rows reads every row once, in segments of 4096 logits (their
// maximum, its first place, and the sum of exp((z - max) / T)); k_excess makes each lane's decisions from those (every
// workgroup of a lane for itself: a few hundred numbers) and sums the excess over 256 tokens at a time of the row that
// the next token comes from; a lane's last workgroup to finish finds the block and the token.
//
// Measured (k_rows + k_excess, 151936 tokens): one lane of 4 drafts with a draft model 5 + 13 us, which is latency (a chain
// of about eight loads from memory); 24 lanes of up to 8 drafts 40 + 19 us: 37 million logits, 150 MB, at 3.7 TB/s with
// the vector units issuing in 67 % of the cycles (about 20 instructions a logit, 12 of them 64-bit); 16 lanes of up to 5
// drafts without a model 15 + 17.6 us.
#include <cfloat>

#include "ctx.h"
#include "exp64.h"
#include "ops.h"

namespace mk {
namespace {

constexpr int kThreads = 256;
constexpr int kQuads = 4;                         // logits per thread, in fours
constexpr int kBlock = 64 * 4;                    // logits of a wave's fours
constexpr int kSeg = kThreads / 64 * kQuads * kBlock;  // logits per segment, a wave's contiguous
constexpr int kMaxDraft = MK_VERIFY_MAX_DRAFT;

typedef float v4f __attribute__((ext_vector_type(4)));

struct Stat {  // part of a row, or a row
  double sum;  // of exp((z - max) / T); T <= 0: unused
  float max;   // T > 0: near the maximum, what the sum is against; else the maximum
  int32_t at;  // T <= 0: first place of max; -1: nothing but -inf
};
struct Choice {  // of a lane
  int n_acc;
  bool refused;  // a draft was: the excess over Q counts
  int draft;     // that draft
  Stat p, q;     // sum: its inverse
};

// Logits to 64ths of a power of two: 64 log2(e) / T; 0 where T <= 0 (an infinite T counts as the largest).
__device__ __forceinline__ double per_unit(const mk_verify_lane& l) {
  return l.temperature > 0.0f ? 64 * 1.4426950408889634074 / (double)fminf(l.temperature, FLT_MAX) : 0.0;
}
constexpr double kLeast = -63000.0;  // in such 64ths: below 2^-984 there is nothing
// exp((z - max) / T), c its per_unit; 0 for z of -inf.
__device__ __forceinline__ double weight(float z, float max, double c, const double* table) {
  const double d = ((double)z - (double)max) * c;
  const bool in = d > kLeast;
  const Power v = pow2(in ? d : 0.0, table);
  return in ? v.factor * v.rest : 0.0;
}
// Moves between lanes in registers (DPP): lanes that have no source, or are masked, get `none`.
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp(float v, float none) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, none), __builtin_bit_cast(int, v),
                                                               CTRL, ROWS, 0xF, false));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp(double v, double none) {
  const v2u a = __builtin_bit_cast(v2u, v), b = __builtin_bit_cast(v2u, none);
  v2u r;
  r[0] = __builtin_amdgcn_update_dpp((int)b[0], (int)a[0], CTRL, ROWS, 0xF, false);
  r[1] = __builtin_amdgcn_update_dpp((int)b[1], (int)a[1], CTRL, ROWS, 0xF, false);
  return __builtin_bit_cast(double, r);
}
// The inclusive running sum over the wave's lanes: within rows of 16 (row_shr 1, 2, 4, 8), then row 0's and 2's ends on
// rows 1 and 3 (row_bcast:15), then lane 31's on rows 2 and 3 (row_bcast:31).
__device__ __forceinline__ double wave_scan(double v) {
  v += dpp<0x111, 0xF>(v, 0.0);
  v += dpp<0x112, 0xF>(v, 0.0);
  v += dpp<0x114, 0xF>(v, 0.0);
  v += dpp<0x118, 0xF>(v, 0.0);
  v += dpp<0x142, 0xA>(v, 0.0);
  return v + dpp<0x143, 0xC>(v, 0.0);
}
__device__ __forceinline__ double last_lane(double v) {
  v2u a = __builtin_bit_cast(v2u, v);
  a[0] = __builtin_amdgcn_readlane(a[0], 63), a[1] = __builtin_amdgcn_readlane(a[1], 63);
  return __builtin_bit_cast(double, a);
}
__device__ __forceinline__ double wave_sum(double v) { return last_lane(wave_scan(v)); }
__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, dpp<0x111, 0xF>(v, -INFINITY));
  v = fmaxf(v, dpp<0x112, 0xF>(v, -INFINITY));
  v = fmaxf(v, dpp<0x114, 0xF>(v, -INFINITY));
  v = fmaxf(v, dpp<0x118, 0xF>(v, -INFINITY));
  v = fmaxf(v, dpp<0x142, 0xA>(v, -INFINITY));
  v = fmaxf(v, dpp<0x143, 0xC>(v, -INFINITY));
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
// The statistics of s[0 .. n - 1] together (at -1: nothing), by a row of 16 lanes: the maximum, its first place, the
// sums brought to it (added in another order in every lane: lane 0's is used).
__device__ __forceinline__ Stat join16(const Stat* s, int n, double c, const double* table) {
  const int lane = threadIdx.x & 15;
  Stat r{0.0, -INFINITY, -1};
  for (int i = lane; i < n; i += 16)
    if (s[i].at >= 0) r.max = fmaxf(r.max, s[i].max);
  r.max = fmaxf(r.max, dpp<0x128, 0xF>(r.max, -INFINITY));  // row_ror 8, 4, 2, 1
  r.max = fmaxf(r.max, dpp<0x124, 0xF>(r.max, -INFINITY));
  r.max = fmaxf(r.max, dpp<0x122, 0xF>(r.max, -INFINITY));
  r.max = fmaxf(r.max, dpp<0x121, 0xF>(r.max, -INFINITY));
  if (r.max == -INFINITY) return r;
  if (c > 0.0) {
    r.at = 0;
    for (int i = lane; i < n; i += 16)
      if (s[i].at >= 0) r.sum += s[i].sum * weight(s[i].max, r.max, c, table);
    r.sum += dpp<0x128, 0xF>(r.sum, 0.0);
    r.sum += dpp<0x124, 0xF>(r.sum, 0.0);
    r.sum += dpp<0x122, 0xF>(r.sum, 0.0);
    r.sum += dpp<0x121, 0xF>(r.sum, 0.0);
  } else {
    int at = INT32_MAX;
    for (int i = lane; i < n; i += 16)
      if (s[i].at >= 0 && s[i].max == r.max) at = min(at, s[i].at);
#pragma unroll
    for (int m = 8; m > 0; m >>= 1) at = min(at, __shfl_xor(at, m, 16));
    r.at = at;
  }
  return r;
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

// Place of this thread's four logits `quad` of a segment of N per thread.
template <int N = kQuads>
__device__ __forceinline__ int place(int seg, int quad) {
  return ((seg * (kThreads / 64) + (threadIdx.x >> 6)) * N + quad) * kBlock + (threadIdx.x & 63) * 4;
}
// Four logits (past the row: -inf). VEC: rows are 16-byte aligned, V a multiple of 4.
template <bool VEC>
__device__ __forceinline__ v4f load4(const float* row, int at, int V) {
  v4f v;
  if constexpr (VEC) {
    v = *reinterpret_cast<const v4f*>(row + (at < V ? at : 0));
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = row[at + e < V ? at + e : 0];
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = clean(v[e]);
  if (__builtin_expect((at & ~(kBlock - 1)) + kBlock > V, 0)) {  // a wave's last logits
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = at + e < V ? v[e] : -INFINITY;
  }
  return v;
}

// Grid lanes x `per` rows x `spans` spans of `span` segments: rows j <= max_draft of a lane are the target's, the others
// the draft's (per = max_draft + 1: there are none). A row's spans are neighbours, so that rows that a lane does not have
// idle every XCD and shader engine alike (with spans the slow dimension 24 lanes of up to eight drafts took 64 us in all
// instead of 61, 16 lanes without draft rows 42 instead of 39). Each thread sums against the first maximum that it meets
// (64 bits reach 2^900 past it), asks for a segment's logits while the one before is summed, and the threads' sums meet
// once per span.
template <bool VEC>
__global__ __launch_bounds__(kThreads) void k_rows(Rows R, const mk_verify_lane* __restrict__ lanes, int max_draft,
                                                   int per, int span, int spans, Stat* __restrict__ stats,
                                                   uint32_t* __restrict__ arrived) {
  const int at_row = blockIdx.x / spans, at_span = blockIdx.x % spans, li = at_row / per, j = at_row % per;
  const mk_verify_lane L = lanes[li];
  if (!lane_ok(L, max_draft, R.n_rows, R.n_drafts)) return;
  if (j == 0 && at_span == 0 && threadIdx.x == 0) arrived[li] = 0;  // for k_excess
  const bool draft = j > max_draft;
  const int jj = draft ? j - max_draft - 1 : j;
  if (draft ? jj >= L.n_draft : jj > L.n_draft) return;
  const float* row = draft ? R.q + (int64_t)(L.first + jj) * R.q_stride : R.p + (int64_t)(L.row + jj) * R.p_stride;
  const int seg0 = at_span * span, seg1 = min(seg0 + span, (R.V + kSeg - 1) / kSeg);
  v4f z[kQuads], next[kQuads];
#pragma unroll
  for (int i = 0; i < kQuads; ++i) z[i] = load4<VEC>(row, place(seg0, i), R.V);
  __shared__ double table[kTable];
  load_table(table);
  const double c = per_unit(L);
  const float reach = 346.0f * L.temperature;  // a maximum further than 2^499 up is a new one to sum against
  float m = -INFINITY;
  double sum = 0.0;
  int at = -1;
  __syncthreads();
#pragma unroll 1
  for (int seg = seg0; seg < seg1; ++seg) {
    if (seg + 1 < seg1)
#pragma unroll
      for (int i = 0; i < kQuads; ++i) next[i] = load4<VEC>(row, place(seg + 1, i), R.V);
    float top = z[0][0];
#pragma unroll
    for (int i = 0; i < kQuads; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) top = fmaxf(top, z[i][e]);
    if (top > m && (m == -INFINITY || c == 0.0 || top - m > reach)) {
      sum = m == -INFINITY ? 0.0 : sum * weight(m, top, c, table);
      m = top, at = INT32_MAX;
#pragma unroll
      for (int i = kQuads - 1; i >= 0; --i)
#pragma unroll
        for (int e = 3; e >= 0; --e) at = z[i][e] == m ? place(seg, i) + e : at;
    }
    if (c > 0.0 && m > -INFINITY) {
      const double md = (double)m;
#pragma unroll
      for (int i = 0; i < kQuads; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const Power v = pow2(fmax(((double)z[i][e] - md) * c, kLeast), table);
          sum = __builtin_fma(v.factor, v.rest, sum);
        }
    }
#pragma unroll
    for (int i = 0; i < kQuads; ++i) z[i] = next[i];
  }
  // A wave's threads, then the waves.
  const int lane = threadIdx.x & 63;
  const float wm = wave_max(m);
  if (c > 0.0) {
    sum = wave_sum(m == -INFINITY ? 0.0 : sum * weight(m, wm, c, table));
    at = wm == -INFINITY ? INT32_MAX : 0;
  } else {
    at = m == wm && at >= 0 ? at : INT32_MAX;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) at = min(at, __shfl_xor(at, o));
  }
  __shared__ Stat ws[kThreads / 64];
  if (lane == 0) ws[threadIdx.x >> 6] = Stat{sum, wm, at == INT32_MAX ? -1 : at};
  __syncthreads();
  if (threadIdx.x >= 16) return;
  const Stat s = join16(ws, kThreads / 64, c, table);
  if (threadIdx.x == 0) stats[blockIdx.x] = s;
}

// P(x) of a row from its statistics (sum: its inverse).
__device__ __forceinline__ double prob(const Stat& s, float z, int x, double c, const double* table) {
  if (s.at < 0) return 0.0;
  return c > 0.0 ? weight(z, s.max, c, table) * s.sum : x == s.at ? 1.0 : 0.0;
}

// What of token x the next token is drawn by.
__device__ __forceinline__ double excess(const Choice& c, float zp, float zq, bool has_q, int x, double unit,
                                         const double* table) {
  const double p = prob(c.p, zp, x, unit, table);
  if (!c.refused) return p;
  const double q = has_q ? prob(c.q, zq, x, unit, table) : x == c.draft ? 1.0 : 0.0;
  return fmax(p - q, 0.0);
}

// Sums of the excess, which other workgroups of the lane read: stored and read past the caches that XCDs do not share.
__device__ __forceinline__ void put(double* p, double v) {
  __hip_atomic_store(reinterpret_cast<uint64_t*>(p), __builtin_bit_cast(uint64_t, v), __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ double get(const double* p) {
  return __builtin_bit_cast(double, __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED,
                                                      __HIP_MEMORY_SCOPE_AGENT));
}

// The first token in order whose running sum reaches v times the total, by one wave: there is nothing to wait for but its
// loads (one lane, its segments whole, 19.7 us in all; by four waves, a token per thread, with eight barriers 25.6). sums: of blocks of 256
// tokens.
template <bool VEC>
__device__ __forceinline__ int pick_token(const Rows& R, const float* prow, const float* qrow, Choice& c, double unit,
                                          double v, const double* sums, int blocks, const double* table) {
  const int lane = threadIdx.x & 63;
  // Lane i has the sums of `each` neighbouring blocks; their running sum and total.
  const int each = (blocks + 63) / 64, b0 = min(lane * each, blocks), b1 = min(b0 + each, blocks);
  constexpr int kKept = 10;  // in registers, of vocabularies up to 163840
  double kept[kKept], mine = 0.0;
#pragma unroll
  for (int i = 0; i < kKept; ++i) kept[i] = b0 + i < b1 ? get(sums + b0 + i) : 0.0;
#pragma unroll
  for (int i = 0; i < kKept; ++i) mine += kept[i];
  for (int b = b0 + kKept; b < b1; ++b) mine += get(sums + b);
  const double upto = wave_scan(mine);
  double total = last_lane(upto), run = 0.0;
  // Nothing over Q: P itself, whose blocks have no sums at hand.
  const bool walk = !(total > 0.0) && c.refused;
  if (walk) c.refused = 0, total = 1.0;
  const double goal = v * total;
  // The block: the first whose running sum reaches the goal (rounding aside, the last with anything), and what lies
  // before it.
  int first = 0, end = blocks;
  if (!walk) {
    int block = -1, last = -1;
    double before = upto - mine, block_run = 0.0, last_run = 0.0;
    auto look = [&](int b, double s) {
      if (s > 0.0) {
        last = b, last_run = before;
        if (block < 0 && before + s >= goal) block = b, block_run = before;
      }
      before += s;
    };
#pragma unroll
    for (int i = 0; i < kKept; ++i) look(b0 + i, kept[i]);
    for (int b = b0 + kKept; b < b1; ++b) look(b, get(sums + b));
    const uint64_t hit = __ballot(block >= 0), some = __ballot(last >= 0);
    if (!some) return -1;
    const int from = hit ? __builtin_ctzll(hit) : 63 - __builtin_clzll(some);
    first = __builtin_amdgcn_readlane(hit ? block : last, from), end = first + 1;
    run = __shfl(hit ? block_run : last_run, from);
  }
  int last = -1;
#pragma unroll 1
  for (int b = first; b < end; ++b) {  // four tokens a lane
    const int x = b * kBlock + 4 * lane;
    const v4f zp = load4<VEC>(prow, x, R.V), zq = load4<VEC>(qrow, x, R.V);
    double r[4];
    int some = -1, pick = -1;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      r[e] = excess(c, zp[e], zq[e], R.q != nullptr, x + e, unit, table);
      some = r[e] > 0.0 ? e : some;
    }
#pragma unroll
    for (int e = 1; e < 4; ++e) r[e] += r[e - 1];
    const double scan = wave_scan(r[3]), before = run + (scan - r[3]);
#pragma unroll
    for (int e = 3; e >= 0; --e)  // a running sum that has grown
      if (r[e] > (e ? r[e - 1] : 0.0) && before + r[e] >= goal) pick = e;
    const uint64_t hit = __ballot(pick >= 0), any = __ballot(some >= 0);
    if (hit) {
      const int from = __builtin_ctzll(hit);
      return b * kBlock + 4 * from + __builtin_amdgcn_readlane(pick, from);
    }
    if (any) {
      const int from = 63 - __builtin_clzll(any);
      last = b * kBlock + 4 * from + __builtin_amdgcn_readlane(some, from);
    }
    run += last_lane(scan);
  }
  return last;  // rounding may leave the goal above the whole sum: the last token with any
}

// Grid (lanes, segments of N quads per thread). The lane's last workgroup to have its sums in memory draws the token.
template <bool VEC, int N>
__global__ __launch_bounds__(kThreads) void k_excess(Rows R, const mk_verify_lane* __restrict__ lanes, int max_draft,
                                                     const int32_t* __restrict__ drafts, const double* __restrict__ u,
                                                     const double* __restrict__ u_next, const Stat* __restrict__ stats,
                                                     int per, int spans, double* __restrict__ sums,
                                                     uint32_t* __restrict__ arrived, int32_t* __restrict__ accepted,
                                                     int32_t* __restrict__ tokens, float* __restrict__ probs) {
  const int li = blockIdx.x, segs = gridDim.y, seg = blockIdx.y, tid = threadIdx.x;
  const int lane = tid & 63, w = tid >> 6;
  const mk_verify_lane L = lanes[li];
  int32_t* tok = tokens + (int64_t)li * (max_draft + 1);
  float* pr = probs ? probs + (int64_t)li * (max_draft + 1) : nullptr;
  if (!lane_ok(L, max_draft, R.n_rows, R.n_drafts)) {
    if (seg == 0) {
      for (int j = tid; j <= max_draft; j += kThreads) {
        tok[j] = -1;
        if (pr) pr[j] = 0.0f;
      }
      if (tid == 0) accepted[li] = -1;
    }
    return;
  }
  __shared__ double table[kTable];
  load_table(table);
  const double unit = per_unit(L), v = u_next[li];
  // Thread j's draft (at most 256: one each), asked for before the rows' statistics.
  static_assert(kMaxDraft <= kThreads, "a draft per thread");
  int d = -1;
  float zp_d = -INFINITY, zq_d = -INFINITY;
  double u_d = 0.0;
  if (tid < L.n_draft) {
    d = drafts[L.first + tid], u_d = u[L.first + tid];
    if (d >= 0 && d < R.V) {
      zp_d = R.p[(int64_t)(L.row + tid) * R.p_stride + d];
      if (R.q) zq_d = R.q[(int64_t)(L.first + tid) * R.q_stride + d];
    }
  }
  __shared__ Stat row_s[2 * kMaxDraft + 1];
  __shared__ int stop_s, d_s[kMaxDraft + 1], last_s;
  if (tid == 0) stop_s = L.n_draft;
  __syncthreads();
  // Sixteen lanes a row.
  const int rows = L.n_draft + 1 + (R.q ? L.n_draft : 0);
  for (int r = tid >> 4; r < rows; r += kThreads / 16) {
    const int j = r <= L.n_draft ? r : max_draft + r - L.n_draft;
    Stat a = join16(stats + ((int64_t)li * per + j) * spans, spans, unit, table);
    if (a.at >= 0 && unit > 0.0) a.sum = 1.0 / a.sum;
    if ((tid & 15) == 0) row_s[r] = a;
  }
  __syncthreads();
  float p_d = 0.0f;
  if (tid < L.n_draft) {
    double p = 0.0, q = 1.0;
    if (d >= 0 && d < R.V) {
      p = prob(row_s[tid], clean(zp_d), d, unit, table);
      if (R.q) q = prob(row_s[L.n_draft + 1 + tid], clean(zq_d), d, unit, table);
    }
    if (!(q > 0.0 && u_d * q < p)) atomicMin(&stop_s, tid);
    p_d = (float)p;
    d_s[tid] = d;
  }
  __syncthreads();
  Choice c;
  c.n_acc = stop_s;
  c.refused = c.n_acc < L.n_draft;
  c.draft = c.refused ? d_s[c.n_acc] : -1;
  c.p = row_s[c.n_acc];
  c.q = c.refused && R.q ? row_s[L.n_draft + 1 + c.n_acc] : Stat{0.0, -INFINITY, -1};
  const bool both = c.refused && R.q;
  const float* prow = R.p + (int64_t)(L.row + c.n_acc) * R.p_stride;
  const float* qrow = both ? R.q + (int64_t)(L.first + c.n_acc) * R.q_stride : prow;
  v4f zp[N], zq[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    zp[i] = load4<VEC>(prow, place<N>(seg, i), R.V);
    zq[i] = load4<VEC>(qrow, place<N>(seg, i), R.V);
  }
  if (seg == 0) {
    for (int j = tid; j <= max_draft; j += kThreads) {
      if (j == c.n_acc) continue;
      tok[j] = j < c.n_acc ? d : -1;
      if (pr) pr[j] = j < c.n_acc ? p_d : 0.0f;
    }
    if (tid == 0) accepted[li] = c.n_acc;
  }
  const int blocks = segs * (kThreads / 64 * N);
  double* lane_sums = sums + (int64_t)li * blocks;
  double sum[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    sum[i] = 0.0;
    const int x = place<N>(seg, i);
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[i] += excess(c, zp[i][e], zq[i][e], R.q != nullptr, x + e, unit, table);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) sum[i] = wave_sum(sum[i]);
  if (lane == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) put(lane_sums + seg * (kThreads / 64 * N) + w * N + i, sum[i]);
  // Every wave's sums have reached memory before the lane's counter says so.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0)
    last_s = __hip_atomic_fetch_add(arrived + li, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)segs - 1;
  __syncthreads();
  if (!last_s || w) return;
  const int pick = pick_token<VEC>(R, prow, qrow, c, unit, v, lane_sums, blocks, table);
  if (tid == 0) {
    tok[c.n_acc] = pick;
    if (pr) pr[c.n_acc] = pick < 0 ? 0.0f : (float)prob(c.p, clean(prow[pick]), pick, unit, table);
  }
}

// ---- rows cut to their top k ----

constexpr int kMaxK = 1024, kTopkThreads = 512;

struct Cands {
  const float* values;
  const int32_t* ids;
  int k, n;  // candidates per row, rows
};
struct Head {  // what of a row of candidates is kept: the first `keep`, of total weight `sum`; 0: nothing but -inf
  double sum;
  int32_t keep;
  int32_t first;  // the highest candidate, behind those of NaN, which mk_topk puts ahead of the others
  float top;      // its logit
};

// A candidate of v against the highest one, both clean: one of -inf has no weight (top is finite).
__device__ __forceinline__ double cand_weight(float v, float top, float t) {
  return (double)(float)exp((double)((v - top) / t));
}

// One wave: the kept head (sampler.cpp:37-56), 64 candidates at a time, their running sums by a scan. t: the lane's
// temperature, at most FLT_MAX; 0: greedy.
__device__ __forceinline__ Head head_of(const float* v, int k, const mk_verify_lane& L, float t) {
  const int lane = threadIdx.x & 63;
  auto logit = [&](int i) { return i < k ? clean(v[i]) : -INFINITY; };
  const float z0 = logit(lane);
  int from = 0;
  float z = z0;
  uint64_t some = __ballot(z > -INFINITY);
  while (!some) {
    if ((from += 64) >= k) return Head{1.0, 0, 0, 0.0f};
    z = logit(from + lane), some = __ballot(z > -INFINITY);
  }
  const int first = from + __builtin_ctzll(some);
  const float top =
      __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, z), __builtin_ctzll(some)));
  if (!(t > 0.0f)) return Head{1.0, first + 1, first, top};
  const double w0 = cand_weight(z0, top, t);
  double all = wave_sum(w0);
  for (int c = 64; c < k; c += 64) all += wave_sum(cand_weight(logit(c + lane), top, t));
  const double floor_w = (double)L.min_p, nucleus = (double)L.top_p * all;  // the first weight is 1
  double run = 0.0;
  for (int c = 0; c < k; c += 64) {
    const int i = c + lane;
    z = c ? logit(i) : z0;
    const double w = c ? cand_weight(z, top, t) : w0, scan = wave_scan(w) + run;
    const uint64_t below = __ballot(i > first && z > -INFINITY && w < floor_w),
                   reach = __ballot(i < k && i >= first && scan >= nucleus);
    const int b = below ? __builtin_ctzll(below) : 64, e = reach ? __builtin_ctzll(reach) : 64;
    if (b < 64 || e < 64) {
      // Candidate b is not kept, candidate e is the last; one that is both is below the floor.
      const int last = b <= e ? b - 1 : e;  // in this chunk; -1: the chunk before's last
      return Head{last < 0 ? run : __shfl(scan, last), c + last + 1, first, top};
    }
    run = __shfl(scan, min(63, k - 1 - c));
  }
  return Head{run, k, first, top};
}

// Candidate i's probability in the row v.
__device__ __forceinline__ float cand_prob(const Head& h, const float* v, int i, float t) {
  if (i >= h.keep) return 0.0f;
  return t > 0.0f ? (float)(cand_weight(clean(v[i]), h.top, t) / h.sum) : i == h.first ? 1.0f : 0.0f;
}

// Probability of token d in a row (sampler.cpp prob_in), by one wave.
__device__ __forceinline__ float prob_in(const float* v, const int32_t* ids, const Head& h, int d, float t) {
  const int lane = threadIdx.x & 63;
  for (int c = 0; c < h.keep; c += 64) {
    const uint64_t hit = __ballot(c + lane < h.keep && ids[c + lane] == d);
    if (hit) {
      const int i = c + __builtin_ctzll(hit);
      return cand_prob(h, v, i, t);
    }
  }
  return 0.0f;
}

// One workgroup per lane: the rows' heads in turn over the waves, each with the probability of the draft it judges;
// then wave 0 draws the next token. Latency: 32 lanes of up to 8 drafts and 40 candidates a row 7.9 us a pass.
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
  const float t = L.temperature > 0.0f ? fminf(L.temperature, FLT_MAX) : 0.0f;
  const int rows = ok ? L.n_draft + 1 + (Q.values ? L.n_draft : 0) : 0;
  for (int r = w; r < rows; r += kTopkThreads / 64) {
    const bool draft = r > L.n_draft;
    const int j = draft ? r - L.n_draft - 1 : r, k = draft ? Q.k : P.k;
    const int64_t at = draft ? (int64_t)(L.first + j) * Q.k : (int64_t)(L.row + j) * P.k;
    const float* v = (draft ? Q.values : P.values) + at;
    const Head h = head_of(v, k, L, t);
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
      q_pr[i] = cand_prob(qh, Q.values + at, i, t);
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
    left_s[i] = fmaxf(cand_prob(ph, pv, i, t) - q, 0.0f);
  }
  __syncthreads();
  if (w != 0) return;
  double total = 0.0;
  bool over = true;
  auto left = [&](int i) {
    return i >= ph.keep ? 0.0 : over ? (double)left_s[i] : (double)cand_prob(ph, pv, i, t);
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
    const double scan = wave_scan(r) + run;
    const uint64_t some = __ballot(r > 0.0), hit = __ballot(r > 0.0 && scan >= goal);
    if (some) last = c + 63 - __builtin_clzll(some);
    if (hit) pick = c + __builtin_ctzll(hit);
    run = __shfl(scan, 63);
  }
  if (pick < 0) pick = last;
  if (lane == 0) {
    tok[n_acc] = pick < 0 ? -1 : pi[pick];
    if (pr) pr[n_acc] = pick < 0 ? 0.0f : cand_prob(ph, pv, pick, t);
  }
}

int segments(int V) { return (V + kSeg - 1) / kSeg; }
// Segments a workgroup of k_rows takes: one where rows are few, more once they fill the CUs eight times over (24 lanes of
// eight drafts, 151936 tokens: 2 segments 47 us, 4 40, 8 42).
int span_of(int64_t rows, int segs) { return (int)std::min<int64_t>(8, std::max<int64_t>(1, rows * segs / 2048)); }
// A lane's rows in k_rows' grid, and its workgroups per row.
struct Spans {
  int per, span, spans;
};
Spans spans_of(int n_rows, bool q, int n_drafts, int n_vocab, int n_lanes, int max_draft) {
  Spans s;
  const int segs = segments(n_vocab);
  s.per = q ? 2 * max_draft + 1 : max_draft + 1;
  s.span = span_of(std::min<int64_t>((int64_t)n_lanes * s.per, (int64_t)n_rows + (q ? n_drafts : 0)), segs);
  s.spans = (segs + s.span - 1) / s.span;
  return s;
}

}  // namespace

size_t verify_workspace(int n_lanes, int max_draft, int n_vocab) {
  const size_t segs = segments(n_vocab), lanes = n_lanes;
  return lanes * (2 * (size_t)max_draft + 1) * segs * sizeof(Stat) + lanes * segs * (kSeg / kBlock) * sizeof(double) +
         lanes * sizeof(uint32_t);
}

bool verify_fits(int n_rows, bool q, int n_drafts, int n_vocab, int n_lanes, int max_draft) {
  const Spans s = spans_of(n_rows, q, n_drafts, n_vocab, n_lanes, max_draft);
  return std::max<int64_t>((int64_t)n_lanes * s.per * s.spans, n_lanes) * kThreads < (1ll << 32);
}
bool verify_topk_fits(int n_lanes) { return (int64_t)n_lanes * kTopkThreads < (1ll << 32); }

void verify(hipStream_t s, const float* p, int64_t p_stride, int n_rows, const float* q, int64_t q_stride, int n_drafts,
            int n_vocab, const mk_verify_lane* lanes, int n_lanes, int max_draft, const int32_t* drafts, const double* u,
            const double* u_next, int32_t* accepted, int32_t* tokens, float* probs, void* workspace) {
  const int segs = segments(n_vocab);
  const auto [per, span, spans] = spans_of(n_rows, q, n_drafts, n_vocab, n_lanes, max_draft);
  Stat* stats = static_cast<Stat*>(workspace);
  double* sums = reinterpret_cast<double*>(stats + (size_t)n_lanes * per * segs);
  uint32_t* arrived = reinterpret_cast<uint32_t*>(sums + (size_t)n_lanes * segs * (kSeg / kBlock));
  auto aligned = [](const float* x, int64_t stride) { return !x || (((uintptr_t)x & 15) == 0 && (stride & 3) == 0); };
  const Rows R{p, p_stride, n_rows, q, q_stride, n_drafts, n_vocab};
  auto go = [&]<bool VEC>() {
    hipLaunchKernelGGL(k_rows<VEC>, dim3((unsigned)(n_lanes * per * spans)), dim3(kThreads), 0, s, R, lanes, max_draft,
                       per, span, spans, stats, arrived);
    check_launch("verify rows");
    auto excess = [&]<int N>() {
      hipLaunchKernelGGL((k_excess<VEC, N>), dim3(n_lanes, (segs * kQuads + N - 1) / N), dim3(kThreads), 0, s, R, lanes,
                         max_draft, drafts, u, u_next, stats, per, spans, sums, arrived, accepted, tokens, probs);
      check_launch("verify excess");
    };
    // Half as much per workgroup where those would not fill the CUs once: with 8 drafts and 151936 tokens, 1 lane 19.7 us
    // instead of 22.6 and 4 lanes 27.1 instead of 28.8, but 8 lanes 36.9 both ways and 16 lanes 53.7 instead of 45.5.
    if ((int64_t)n_lanes * segs < 256) excess.template operator()<kQuads / 2>();
    else excess.template operator()<kQuads>();
  };
  if ((n_vocab & 3) == 0 && aligned(p, p_stride) && aligned(q, q_stride)) go.template operator()<true>();
  else go.template operator()<false>();
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
