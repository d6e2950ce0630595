// The pages of the 4-bit cache (include/malkin_hip.h): forking, resizing with copies of shared last pages, compaction.
//
// What a sequence holds is a row of page numbers, so that going on from another sequence copies numbers and counts holders;
// bytes are copied only where a shared page that is not full is to be written, and in compaction. Results do not depend on
// the order in which threads run: counts change by sums of whole numbers, and free pages are handed out by running sums over
// the entries and over the pool, lowest number first, in one workgroup. What bounds a call is that workgroup's chain of four
// or five loads that wait for each other and as many barriers (8.5 us for 64 entries; with 512 threads the same, with 256
// 9.4) and then the copies' bytes, which a second launch moves with the whole chip: 4.7 us for 64 last pages of 28 layers,
// 92 us for the 436 MB read and written of a compaction (4.7 TB/s).
#include <algorithm>

#include "ctx.h"
#include "ops.h"

namespace mk {
namespace {

constexpr int kThreads = 256;
constexpr int kPlan = 1024;      // threads of the one workgroup that hands out pages
constexpr int kMaxEntries = 4096;  // of a resize
constexpr int kScan = 16;        // pages per thread and step of a walk over the pool

__device__ __forceinline__ int pages_of(int rows, int shift) { return (int)(((int64_t)rows + (1 << shift) - 1) >> shift); }

// Rows that sequence s holds, never more than its entries of the table.
__device__ __forceinline__ int held(const Kv4Pool& P, int s) {
  const int64_t room = (int64_t)P.max_pages << P.shift;
  return (int)min((int64_t)max(P.len[s], 0), room);
}

// ---- fork ----

// Per entry: its source's pages as they are before the call, to the workspace, and the counts of holders. A count reaches its
// new value by additions alone, so entries need no order. head[i]: rows, -1 where the entry has no effect.
__global__ __launch_bounds__(kThreads) void k_fork_take(Kv4Pool P, const int32_t* __restrict__ dst,
                                                        const int32_t* __restrict__ src, int n, int32_t* __restrict__ head,
                                                        int32_t* __restrict__ rows) {
  const int i = blockIdx.x, tid = threadIdx.x;
  const int d = dst ? dst[i] : i, s = src[i];
  bool ok = d >= 0 && d < P.n_seq;
  if (dst && ok) {
    bool again = false;
    for (int j = i + 1 + tid; j < n; j += kThreads) again |= dst[j] == d;
    ok = !__syncthreads_or(again);
  }
  const bool from = s >= 0 && s < P.n_seq;
  if (!ok || s == d) {
    if (tid == 0) head[i] = -1;
    return;
  }
  const int len = from ? held(P, s) : 0, m = pages_of(len, P.shift), old = pages_of(held(P, d), P.shift);
  for (int j = tid; j < max(m, old); j += kThreads) {
    const int a = j < m ? P.table[(int64_t)s * P.max_pages + j] : -1;
    const int b = j < old ? P.table[(int64_t)d * P.max_pages + j] : -1;
    rows[(int64_t)i * P.max_pages + j] = a;
    if (a == b) continue;
    if (a >= 0 && a < P.n_page) atomicAdd(P.refs + a, 1);
    if (b >= 0 && b < P.n_page) atomicAdd(P.refs + b, -1);
  }
  if (tid == 0) head[i] = len;
}

__global__ __launch_bounds__(kThreads) void k_fork_put(Kv4Pool P, const int32_t* __restrict__ dst, int n,
                                                       const int32_t* __restrict__ head, const int32_t* __restrict__ rows) {
  const int i = blockIdx.x, len = head[i];
  if (len < 0) return;
  const int d = dst ? dst[i] : i;
  const int m = max(pages_of(len, P.shift), pages_of(held(P, d), P.shift));
  for (int j = threadIdx.x; j < m; j += kThreads) P.table[(int64_t)d * P.max_pages + j] = rows[(int64_t)i * P.max_pages + j];
  __syncthreads();  // every thread has read the old length
  if (threadIdx.x == 0) P.len[d] = len;
}

// The same by one workgroup, the sources' pages in LDS between: a launch less where there is little to move. 64 entries of 46
// pages 4.4 us instead of 3.1 and 2.7; a step with 192 entries of 80 pages 26.5, with two launches 22.2.
constexpr int kFewEntries = 1024, kFewNumbers = 4096;
__global__ __launch_bounds__(kPlan) void k_fork_few(Kv4Pool P, const int32_t* __restrict__ dst, const int32_t* __restrict__ src,
                                                    int n) {
  extern __shared__ int32_t lds[];
  int32_t *d_s = lds, *s_s = d_s + n, *new_s = s_s + n, *old_s = new_s + n, *rows = old_s + n;
  const int tid = threadIdx.x;
  for (int i = tid; i < n; i += kPlan) {
    d_s[i] = dst ? dst[i] : i;
    s_s[i] = src[i];
  }
  __syncthreads();
  for (int i = tid; i < n; i += kPlan) {
    const int d = d_s[i], s = s_s[i];
    bool ok = d >= 0 && d < P.n_seq && s != d;
    if (dst && d >= 0 && d < P.n_seq)
      for (int j = i + 1; j < n && ok; ++j) ok = d_s[j] != d;
    new_s[i] = ok ? (s >= 0 && s < P.n_seq ? held(P, s) : 0) : -1;
    old_s[i] = ok ? held(P, d) : 0;
  }
  __syncthreads();
  for (int at = tid; at < n * P.max_pages; at += kPlan) {
    const int i = at / P.max_pages, j = at - i * P.max_pages;
    if (new_s[i] < 0) continue;
    const int a = j < pages_of(new_s[i], P.shift) ? P.table[(int64_t)s_s[i] * P.max_pages + j] : -1;
    const int b = j < pages_of(old_s[i], P.shift) ? P.table[(int64_t)d_s[i] * P.max_pages + j] : -1;
    rows[at] = a;
    if (a == b) continue;
    if (a >= 0 && a < P.n_page) atomicAdd(P.refs + a, 1);
    if (b >= 0 && b < P.n_page) atomicAdd(P.refs + b, -1);
  }
  __syncthreads();
  for (int at = tid; at < n * P.max_pages; at += kPlan) {
    const int i = at / P.max_pages, j = at - i * P.max_pages;
    if (new_s[i] >= 0 && j < pages_of(max(new_s[i], old_s[i]), P.shift)) P.table[(int64_t)d_s[i] * P.max_pages + j] = rows[at];
  }
  for (int i = tid; i < n; i += kPlan)
    if (new_s[i] >= 0) P.len[d_s[i]] = new_s[i];
}

// ---- copies ----

struct Move {
  int32_t src, dst, rows;
};

// Rows 0 .. rows - 1 of page src to page dst, a wave per (move, head of a layer).
template <int D>
__device__ __forceinline__ void copy_head(const Kv4Pool& P, const Move& m, int head, int lane) {
  constexpr int kPieces = D / 32, G = D / 32;  // 16-byte pieces of a row, groups
  const int64_t from = ((int64_t)m.src * P.heads + head) << P.shift, to = ((int64_t)m.dst * P.heads + head) << P.shift;
  const uint4 *kf = reinterpret_cast<const uint4*>(P.k) + from * kPieces, *vf = reinterpret_cast<const uint4*>(P.v) + from * kPieces;
  uint4 *kt = reinterpret_cast<uint4*>(P.k) + to * kPieces, *vt = reinterpret_cast<uint4*>(P.v) + to * kPieces;
  for (int i = lane; i < m.rows * kPieces; i += 64) {
    const uint4 a = kf[i], b = vf[i];
    kt[i] = a, vt[i] = b;
  }
  const uint16_t *sf = P.ks + from * G, *wf = P.vs + from * G;
  uint16_t *st = P.ks + to * G, *wt = P.vs + to * G;
  for (int i = lane; i < m.rows * G; i += 64) {
    const int at = (i / m.rows << P.shift) + i % m.rows;
    const uint16_t a = sf[i], b = wf[at];
    st[i] = a, wt[at] = b;
  }
}

template <int D>
__global__ __launch_bounds__(kThreads) void k_copy_pages(Kv4Pool P, const int32_t* __restrict__ count,
                                                         const Move* __restrict__ moves) {
  const int lane = threadIdx.x & 63;
  const int64_t items = (int64_t)*count * P.heads;
  for (int64_t it = (int64_t)blockIdx.x * (kThreads / 64) + threadIdx.x / 64; it < items; it += (int64_t)gridDim.x * (kThreads / 64)) {
    const Move m = moves[it / P.heads];
    copy_head<D>(P, m, (int)(it % P.heads), lane);
  }
}

// ---- in one workgroup ----

// Exclusive running sum over the workgroup's threads, and the total. part: kPlan / 64 + 1 words of LDS, free again after the
// caller's next barrier.
template <typename T>
__device__ __forceinline__ T block_scan(T v, T* part, T& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  T x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const T y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 63) part[w] = x;
  __syncthreads();
  T before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kPlan / 64; ++i) {
    const T p = part[i];
    before += i < w ? p : 0;
    all += p;
  }
  total = all;
  return before + x - v;
}

__device__ __forceinline__ int refs_now(const int32_t* p) { return (int)ld_coh_u32(reinterpret_cast<const uint32_t*>(p)); }

// What becomes of an entry.
enum { kSkip = 0, kShrink = 1, kGrow = 2 };
constexpr int kFreeInLds = 1024;  // free pages that are kept at hand

__global__ __launch_bounds__(kPlan) void k_resize_plan(Kv4Pool P, const int32_t* __restrict__ seq,
                                                       const int32_t* __restrict__ new_len, int n, int32_t* __restrict__ status,
                                                       int32_t* __restrict__ count, Move* __restrict__ moves, int32_t* free_list) {
  extern __shared__ int32_t lds[];
  int32_t *seq_s = lds, *len_s = seq_s + n, *new_s = len_s + n, *last_s = new_s + n;
  __shared__ int part[kPlan / 64], free_s[kFreeInLds];
  __shared__ int64_t part64[kPlan / 64];
  __shared__ uint8_t kind_s[kMaxEntries];
  __shared__ int cut;  // the first entry that wants pages and finds too few
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, in_page = (1 << P.shift) - 1;
  const int E = (n + kPlan - 1) / kPlan, i0 = tid * E;  // a thread's entries follow each other
  const int64_t room = (int64_t)P.max_pages << P.shift;
  if (seq) {
    for (int i = tid; i < n; i += kPlan) seq_s[i] = seq[i];
    __syncthreads();
  }
  if (tid == 0) cut = INT32_MAX;
  bool shrinks = false;
  for (int i = tid; i < n; i += kPlan) {
    const int s = seq ? seq_s[i] : i, now = held(P, min(max(s, 0), P.n_seq - 1)), L = new_len[i];  // both loads at once
    bool ok = s >= 0 && s < P.n_seq && L >= 0 && L <= room;
    if (seq) {
      for (int j = i + 1; j < n && ok; ++j) ok = seq_s[j] != s;
    } else {
      seq_s[i] = i;
    }
    new_s[i] = L;
    const int len = ok ? now : 0;
    const int kind = !ok ? kSkip : L > len ? kGrow : kShrink;
    int last = -1;
    if (kind == kGrow && len & in_page) {
      last = P.table[(int64_t)s * P.max_pages + (len >> P.shift)];
      if (last >= P.n_page) last = -1;
    }
    len_s[i] = len, last_s[i] = max(last, -1), kind_s[i] = (uint8_t)kind;
    shrinks |= kind == kShrink && L < len;
  }
  if (__syncthreads_or(shrinks)) {  // shorter ends, a wave per entry
    for (int i = w; i < n; i += kPlan / 64) {
      if (kind_s[i] != kShrink) continue;
      const int s = seq_s[i], had = pages_of(len_s[i], P.shift), has = pages_of(new_s[i], P.shift);
      for (int j = has + lane; j < had; j += 64) {
        int32_t* at = P.table + (int64_t)s * P.max_pages + j;
        const int p = *at;
        if (p >= 0 && p < P.n_page) atomicAdd(P.refs + p, -1);
        *at = -1;
      }
      if (lane == 0) P.len[s] = new_s[i];
    }
    __syncthreads();  // the counts have been taken down
  }
  // The first pages of the pool, asked for beside the counts of the last pages.
  auto free_of = [&](int p0) {
    uint32_t free = 0;
#pragma unroll
    for (int e = 0; e < kScan; ++e) {
      const int p = p0 + kScan * tid + e;
      const int r = refs_now(P.refs + min(p, P.n_page - 1));
      free |= (uint32_t)(p < P.n_page && r <= 0) << e;
    }
    return free;
  };
  uint32_t free = kScan * (tid & ~63) < P.n_page ? free_of(0) : 0;
  // Copies and pages wanted, and where each entry's begin in the list of free pages and in that of the copies. More than the
  // pool has counts as one more than that. prior: the entry before this one that is the last to leave the page which this one
  // keeps, with what it needs (-1: none).
  int copies[kMaxEntries / kPlan], needs[kMaxEntries / kPlan], prior[kMaxEntries / kPlan];
  int64_t mine = 0;
#pragma unroll
  for (int e = 0; e < kMaxEntries / kPlan; ++e) {
    copies[e] = needs[e] = 0, prior[e] = -1;
    const int i = i0 + e;
    if (e >= E || i >= n || kind_s[i] != kGrow) continue;
    if (last_s[i] >= 0) {
      const int holders = refs_now(P.refs + last_s[i]);
      int before = 0;
      if (holders > 1)
        for (int j = 0; j < i; ++j)
          if (last_s[j] == last_s[i]) ++before, prior[e] = j;
      copies[e] = before < holders - 1;
    }
    needs[e] = min(copies[e] + pages_of(new_s[i], P.shift) - pages_of(len_s[i], P.shift), P.n_page + 1);
    mine += ((int64_t)needs[e] << 16) + copies[e];
  }
  int64_t all = 0;
  const int64_t before = block_scan(mine, part64, all);
  const int64_t wanted = all >> 16;
  // The first free pages of the pool, as many as are wanted.
  int found = 0;
  for (int p0 = 0; p0 < P.n_page && found < wanted; p0 += kScan * kPlan) {
    if (p0) free = free_of(p0);
    int here = 0, to = found + block_scan((int)__popc(free), part, here);
#pragma unroll
    for (int e = 0; e < kScan; ++e)
      if (free >> e & 1) {
        if (to < wanted) {
          if (to < kFreeInLds) free_s[to] = p0 + kScan * tid + e;
          else free_list[to] = p0 + kScan * tid + e;
        }
        ++to;
      }
    found += here;
  }
  // An entry that wants pages has them if those up to it all do, so one number says which do. One that keeps a page because
  // all who share it leave, keeps it only if the last of them does.
  if (found < wanted) {
    int64_t end = before >> 16;
#pragma unroll
    for (int e = 0; e < kMaxEntries / kPlan; ++e) {
      end += needs[e];
      if (needs[e] && end > found) atomicMin(&cut, i0 + e);
    }
  }
  __syncthreads();  // the list is written
  auto page_at = [&](int64_t i) { return i < kFreeInLds ? free_s[i] : free_list[i]; };
  int64_t run = before >> 16;
  int slot = (int)(before & 0xFFFF);
#pragma unroll
  for (int e = 0; e < kMaxEntries / kPlan; ++e) {
    const int i = i0 + e;
    if (e >= E || i >= n) continue;
    const int kind = kind_s[i];
    const bool fits = kind == kGrow && (needs[e] ? i : prior[e]) < cut;
    if (copies[e]) {  // one that does not fit stays in the list, with no rows
      Move m{0, 0, 0};
      if (fits) {
        const int p = page_at(run), s = seq_s[i], len = len_s[i];
        m = Move{last_s[i], p, len & in_page};
        P.table[(int64_t)s * P.max_pages + (len >> P.shift)] = p;
        atomicAdd(P.refs + m.src, -1);
        atomicAdd(P.refs + p, 1);
      }
      moves[slot++] = m;
    }
    status[i] = kind == kSkip ? -1 : kind == kGrow && !fits;
    if (fits) P.len[seq_s[i]] = new_s[i];
    last_s[i] = fits ? (int)run + copies[e] : -1;  // its first new page in the list
    run += needs[e];
  }
  if (tid == 0) *count = (int)(all & 0xFFFF);
  // Does any entry have new pages? Then a wave per entry puts them down.
  if (!__syncthreads_or(wanted > (all & 0xFFFF))) return;
  for (int i = w; i < n; i += kPlan / 64) {
    if (last_s[i] < 0) continue;
    const int s = seq_s[i], had = pages_of(len_s[i], P.shift), has = pages_of(new_s[i], P.shift);
    for (int j = lane; j < has - had; j += 64) {
      const int p = page_at(last_s[i] + j);
      P.table[(int64_t)s * P.max_pages + had + j] = p;
      atomicAdd(P.refs + p, 1);
    }
  }
}

// ---- compaction ----

// moves: hole j of the first n_live pages gets the j-th page in use beyond them. to[p]: where page p >= n_live went.
__global__ __launch_bounds__(kPlan) void k_compact_plan(Kv4Pool P, int32_t* __restrict__ n_live, int32_t* __restrict__ count,
                                                        Move* __restrict__ moves, int32_t* __restrict__ to) {
  __shared__ int part[kPlan / 64];
  const int tid = threadIdx.x;
  int live = 0;
  for (int p = tid; p < P.n_page; p += kPlan) live += P.refs[p] > 0;
  int total = 0;
  block_scan(live, part, total);
  int holes = 0, movers = 0;  // found so far
  for (int p0 = 0; p0 < P.n_page; p0 += kScan * kPlan) {
    int hole = 0, mover = 0;
    uint32_t used = 0;
#pragma unroll
    for (int e = 0; e < kScan; ++e) {
      const int p = p0 + kScan * tid + e;
      if (p < P.n_page && P.refs[p] > 0) used |= 1u << e, mover += p >= total;
      else if (p < total) ++hole;
      else if (p < P.n_page) to[p] = p;  // nobody's
    }
    int all_h = 0, all_m = 0;
    int h = holes + block_scan(hole, part, all_h);
    int m = movers + block_scan(mover, part, all_m);
#pragma unroll
    for (int e = 0; e < kScan; ++e) {
      const int p = p0 + kScan * tid + e;
      if (used >> e & 1) {
        if (p >= total) moves[m++].src = p;
      } else if (p < total) {
        moves[h++].dst = p;
      }
    }
    holes += all_h, movers += all_m;
  }
  __syncthreads();
  for (int j = tid; j < holes; j += kPlan) {
    const int src = moves[j].src, dst = moves[j].dst;
    moves[j].rows = 1 << P.shift;
    to[src] = dst;
    P.refs[dst] = P.refs[src];
    P.refs[src] = 0;
  }
  if (tid == 0) *count = holes, *n_live = total;
}

template <int D>
__global__ __launch_bounds__(kThreads) void k_compact_move(Kv4Pool P, const int32_t* __restrict__ n_live,
                                                           const int32_t* __restrict__ count, const Move* __restrict__ moves,
                                                           const int32_t* __restrict__ to) {
  const int lane = threadIdx.x & 63, live = *n_live;
  const int64_t entries = (int64_t)P.n_seq * P.max_pages;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < entries; i += (int64_t)gridDim.x * kThreads) {
    const int p = P.table[i];
    if (p >= live && p < P.n_page) P.table[i] = to[p];
  }
  const int64_t items = (int64_t)*count * P.heads;
  for (int64_t it = (int64_t)blockIdx.x * (kThreads / 64) + threadIdx.x / 64; it < items; it += (int64_t)gridDim.x * (kThreads / 64))
    copy_head<D>(P, moves[it / P.heads], (int)(it % P.heads), lane);
}

constexpr int kHead = 16;  // bytes before a list: its length

unsigned copy_wgs(int64_t moves, int heads) {
  const int64_t wgs = (moves * heads + kThreads / 64 - 1) / (kThreads / 64);
  return (unsigned)std::max<int64_t>(1, std::min<int64_t>(wgs, 8 * device_cus()));
}

}  // namespace

size_t kv4_fork_workspace(int n, int max_pages) { return (size_t)n * (max_pages + 1ull) * 4; }

void kv4_fork(hipStream_t s, const Kv4Pool& P, const int32_t* dst, const int32_t* src, int n, void* workspace) {
  if (n <= kFewEntries && (int64_t)n * P.max_pages <= kFewNumbers) {
    allow_lds<k_fork_few>(4 * (4 * kFewEntries + kFewNumbers));
    hipLaunchKernelGGL(k_fork_few, dim3(1), dim3(kPlan), (size_t)n * (4 + P.max_pages) * 4, s, P, dst, src, n);
    check_launch("kv4_fork few");
    return;
  }
  int32_t *head = static_cast<int32_t*>(workspace), *rows = head + n;
  hipLaunchKernelGGL(k_fork_take, dim3((unsigned)n), dim3(kThreads), 0, s, P, dst, src, n, head, rows);
  check_launch("kv4_fork take");
  hipLaunchKernelGGL(k_fork_put, dim3((unsigned)n), dim3(kThreads), 0, s, P, dst, n, head, rows);
  check_launch("kv4_fork put");
}

size_t kv4_resize_workspace(int n, int n_page) { return kHead + (size_t)n * sizeof(Move) + (size_t)n_page * 4; }

void kv4_resize(hipStream_t s, const Kv4Pool& P, int D, const int32_t* seq, const int32_t* new_len, int n, int32_t* status,
                void* workspace) {
  int32_t* count = static_cast<int32_t*>(workspace);
  Move* moves = reinterpret_cast<Move*>(count + kHead / 4);
  int32_t* free_list = reinterpret_cast<int32_t*>(moves + n);
  allow_lds<k_resize_plan>(16 * kMaxEntries);
  hipLaunchKernelGGL(k_resize_plan, dim3(1), dim3(kPlan), (size_t)n * 16, s, P, seq, new_len, n, status, count, moves, free_list);
  check_launch("kv4_resize plan");
  auto go = [&]<int D_>() {
    hipLaunchKernelGGL(k_copy_pages<D_>, dim3(copy_wgs(n, P.heads)), dim3(kThreads), 0, s, P, count, moves);
  };
  if (D == 128) go.template operator()<128>();
  else go.template operator()<64>();
  check_launch("kv4_resize copies");
}

size_t kv4_compact_workspace(int n_page) { return kHead + (size_t)n_page * (sizeof(Move) + 4); }

void kv4_compact(hipStream_t s, const Kv4Pool& P, int D, int32_t* n_live, void* workspace) {
  int32_t* count = static_cast<int32_t*>(workspace);
  Move* moves = reinterpret_cast<Move*>(count + kHead / 4);
  int32_t* to = reinterpret_cast<int32_t*>(moves + P.n_page);
  hipLaunchKernelGGL(k_compact_plan, dim3(1), dim3(kPlan), 0, s, P, n_live, count, moves, to);
  check_launch("kv4_compact plan");
  auto go = [&]<int D_>() {
    hipLaunchKernelGGL(k_compact_move<D_>, dim3(copy_wgs(P.n_page, P.heads)), dim3(kThreads), 0, s, P, n_live, count, moves, to);
  };
  if (D == 128) go.template operator()<128>();
  else go.template operator()<64>();
  check_launch("kv4_compact move");
}

}  // namespace mk
