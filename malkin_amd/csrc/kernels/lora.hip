// Low-rank adapters of many requests at once beside a shared projection: y[t] = base[t] + scale_a B_a (A_a x[t]), the
// adapter a = ids[t] chosen per token. A is [rank][cols], B [rows][rank] (the layouts of a GGUF adapter's lora_a and
// lora_b), both in one of three types; x, base, y and every sum are fp32.
//
// Two launches: k_shrink makes h = A x for every token, the columns split over workgroups (partial sums in the
// workspace, added in a fixed order by the next launch), k_expand adds scale B h to base. Both take the tokens of an
// aligned 64-token window that share an adapter together, as the 16 columns of up to four v_mfma_f32_16x16x4_f32
// (weights as its 16 rows, so that a lane ends with four consecutive ranks or rows of one token): an adapter's weights
// are read once per window that it occurs in. The products run on fp32 matrix instructions, which need no roundings of x
// or h; the rest is memory: x, base and y are read and written once.
//
// Measured (shrink + expand): 8 tokens with an adapter each, rank 16, 4096 -> 6144: 4.7 + 5.4 us, latency; 64 tokens over
// 24 adapters of rank up to 64, 5120 -> 7168: 7.3 + 10.0 us, latency; 512 tokens over 3 adapters, rank 32, 4096 -> 24576:
// 9.4 us, its workgroups on two fifths of the CUs, and 22.9 us, of which base and y are 100 MB, 4.4 TB/s.
#include <type_traits>

#include "ctx.h"
#include "ops.h"

namespace mk {
namespace {

typedef float v4f __attribute__((ext_vector_type(4)));

constexpr int kWindow = 64;     // tokens that are grouped by adapter
constexpr int kShrinkWaves = 8;
constexpr int kThreads = 256;   // of k_expand: 4 waves
constexpr int kRowBlock = 256;  // rows of y per k_expand workgroup, 64 per wave
constexpr int kStep = 32;       // columns per wave and step of k_shrink: 8 per lane
constexpr int kFewSlots = 16;

struct F16 { uint16_t v; };
struct BF16 { uint16_t v; };
__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(F16 v) { return (float)__builtin_bit_cast(_Float16, v.v); }
__device__ __forceinline__ float to_f(BF16 v) { return __builtin_bit_cast(float, (uint32_t)v.v << 16); }

// The table's pointers are to global memory, which the compiler cannot know.
template <typename T>
using global = const __attribute__((address_space(1))) T;
template <typename T>
__device__ __forceinline__ global<T>* to_global(const void* p) {
  return (global<T>*)(uintptr_t)p;
}

// N values (4 or 8) from p on, the first `valid` of them (the others 0): vec: p is aligned to 16 bytes or to N values, and
// valid is 0 or N. p[0] can always be read.
template <int N>
__device__ __forceinline__ void get(global<float>* p, int valid, bool vec, float (&r)[N]) {
  if (vec) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const v4f v = *reinterpret_cast<global<v4f>*>(p + (valid ? i : 0));
#pragma unroll
      for (int k = 0; k < 4; ++k) r[i + k] = v[k];
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = p[i < valid ? i : 0];
  }
#pragma unroll
  for (int i = 0; i < N; ++i) r[i] = i < valid ? r[i] : 0.0f;
}
template <int N, typename T>
__device__ __forceinline__ void get(global<T>* p, int valid, bool vec, float (&r)[N]) {
  typedef uint32_t words __attribute__((ext_vector_type(N / 2)));
  global<uint16_t>* q = reinterpret_cast<global<uint16_t>*>(p);
  words v;
  if (vec) {
    v = *reinterpret_cast<global<words>*>(q);
  } else {
#pragma unroll
    for (int i = 0; i < N / 2; ++i)
      v[i] = (uint32_t)q[2 * i < valid ? 2 * i : 0] | (uint32_t)q[2 * i + 1 < valid ? 2 * i + 1 : 0] << 16;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) r[i] = i < valid ? to_f(T{(uint16_t)(v[i / 2] >> (16 * (i & 1)))}) : 0.0f;
}
// Values at .. at + 3 of a row of `rank`, as they lie in memory; 0 past its end. VEC: rank is a multiple of four, the row
// aligned to four values.
template <typename T>
struct Raw {
  typedef uint2 type;
};
template <>
struct Raw<float> {
  typedef v4f type;
};
template <bool VEC>
__device__ __forceinline__ v4f get_raw(global<float>* row, int at, int rank) {
  float r[4];
  get<4>(row + (at < rank ? at : 0), max(min(rank - at, 4), 0), VEC, r);
  return v4f{r[0], r[1], r[2], r[3]};
}
template <bool VEC, typename T>
__device__ __forceinline__ uint2 get_raw(global<T>* row, int at, int rank) {
  typedef uint32_t two __attribute__((ext_vector_type(2)));
  global<uint16_t>* q = reinterpret_cast<global<uint16_t>*>(row);
  two v;
  if constexpr (VEC) {
    v = *reinterpret_cast<global<two>*>(q + (at < rank ? at : 0));
    if (at >= rank) v = two{0, 0};
  } else {
    uint32_t e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      e[i] = q[at + i < rank ? at + i : 0];
      e[i] = at + i < rank ? e[i] : 0;
    }
    v = two{e[0] | e[1] << 16, e[2] | e[3] << 16};
  }
  return make_uint2(v[0], v[1]);
}
template <typename T>
__device__ __forceinline__ void from_raw(const v4f& v, float (&r)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = v[i];
}
template <typename T>
__device__ __forceinline__ void from_raw(const uint2& v, float (&r)[4]) {
  r[0] = to_f(T{(uint16_t)v.x}), r[1] = to_f(T{(uint16_t)(v.x >> 16)});
  r[2] = to_f(T{(uint16_t)v.y}), r[3] = to_f(T{(uint16_t)(v.y >> 16)});
}
__device__ __forceinline__ int within(int64_t left, int n) { return left <= 0 ? 0 : left < n ? (int)left : n; }

// What a workgroup does: tokens[0 .. count - 1] (in LDS) of a window, their adapter (rank 0: none). Count 0: nothing.
struct Group {
  int count;
  mk_lora_adapter a;
};

// Slot j of a window is its j-th distinct adapter, in the order of their first tokens, where there are few slots (few
// adapters in the table); with kWindow slots it is the group that token j is the first of. Slots are the grid's slow
// dimension: workgroups are dealt to the XCDs and their shader engines in turn, and slots that a window does not have,
// recurring at a fixed distance, would leave whole engines without work (3 adapters, 512 tokens: 87 us instead of 30).
__device__ __forceinline__ Group group_of(int window, int j, int slots, int n, const int32_t* ids,
                                          const mk_lora_adapter* adapters, int n_adapters, int max_rank, int* tokens) {
  const int lane = threadIdx.x & 63, t0 = window * kWindow, u = t0 + lane;
  const int got = u < n ? ids[u] : -1;
  const int v = got >= 0 && got < n_adapters ? got : -1;
  uint64_t left = __ballot(u < n), mask = 0;
  Group g;
  g.a = mk_lora_adapter{nullptr, nullptr, 0.0f, 0};
  g.count = 0;
  int own = -1;
  if (slots == kWindow) {
    if (!((left >> j) & 1)) return g;
    own = __builtin_amdgcn_readlane(v, j);
    mask = __ballot(v == own) & left;
    if (mask & ((1ull << j) - 1)) return g;
  } else {
    for (int i = 0; i <= j; ++i) {
      if (!left) return g;
      own = __builtin_amdgcn_readlane(v, __builtin_ctzll(left));
      mask = __ballot(v == own) & left;
      left &= ~mask;
    }
  }
  if (own >= 0) {
    g.a = adapters[own];
    if (g.a.rank < 1 || g.a.rank > max_rank || !g.a.a || !g.a.b) g.a.rank = 0;
  }
  g.count = __popcll(mask);
  if ((mask >> lane) & 1) tokens[__popcll(mask & ((1ull << lane) - 1))] = u;  // every wave the same
  __syncthreads();
  return g;
}

// Partial sums h[split][t][r] over columns split * per .. of ranks r0 .. r0 + 31. A lane holds eight consecutive columns
// of two rank rows and of a token in each of NT tiles, one per MFMA.
template <typename T, int NT>
__device__ void shrink(const Group& g, const int* tokens, const float* __restrict__ x, int64_t x_stride, int64_t cols,
                       int r0, int64_t k0, int64_t k1, bool x_vec, float* __restrict__ h, int r_pad,
                       v4f (*part)[8][64]) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, li = lane & 15, lq = lane >> 4;
  const bool vec = x_vec && (cols & 7) == 0 && ((uintptr_t)g.a.a & 15) == 0;  // columns come in eights
  const int tiles = (g.count + 15) / 16;
  global<float>* xr[NT];
  int on[NT];  // all ones: the column is a token
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    on[i] = 16 * i + li < g.count ? -1 : 0;
    xr[i] = to_global<float>(x + tokens[min(16 * i + li, g.count - 1)] * x_stride);
  }
  const bool two = r0 + 16 < g.a.rank;
  global<T>* a[2];
  int row_on[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    row_on[i] = r0 + 16 * i + li < g.a.rank ? -1 : 0;
    a[i] = to_global<T>(g.a.a) + (int64_t)min(r0 + 16 * i + li, g.a.rank - 1) * cols;
  }
  v4f acc[2][NT];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int k = 0; k < NT; ++k) acc[i][k] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  auto walk = [&](auto vec_) __attribute__((always_inline)) {
    constexpr bool V = decltype(vec_)::value;
#pragma unroll 2
    for (int64_t k = k0 + kStep * w; k < k1; k += kStep * kShrinkWaves) {
      const int valid = within(k1 - k - 8 * lq, 8);
      const int64_t at = valid ? k + 8 * lq : k0;
      float av[2][8], xv[NT][8];
#pragma unroll
      for (int i = 0; i < 2; ++i) get<8>(a[i] + at, valid & row_on[i], V, av[i]);
#pragma unroll
      for (int i = 0; i < NT; ++i) get<8>(xr[i] + at, valid & on[i], V, xv[i]);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (j && !two) break;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          if (i >= tiles) break;
#pragma unroll
          for (int e = 0; e < 8; ++e)
            acc[j][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(av[j][e], xv[i][e], acc[j][i], 0, 0, 0);
        }
      }
    }
  };
  if (vec) walk(std::true_type{});
  else walk(std::false_type{});
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int k = 0; k < NT; ++k) part[w][i * NT + k][lane] = acc[i][k];
  __syncthreads();
  // The waves' sums, a wave per (rank tile, token tile) in turn.
#pragma unroll 1
  for (int j = w; j < 2 * NT; j += kShrinkWaves) {
    const int i = j / NT, k = j % NT, c = 16 * k + li;
    if (c < g.count && (i == 0 || two))
      *reinterpret_cast<v4f*>(h + (int64_t)tokens[c] * r_pad + r0 + 16 * i + 4 * lq) =
          ((part[0][j][lane] + part[1][j][lane]) + (part[2][j][lane] + part[3][j][lane])) +
          ((part[4][j][lane] + part[5][j][lane]) + (part[6][j][lane] + part[7][j][lane]));
  }
}

template <typename T>
__global__ __launch_bounds__(64 * kShrinkWaves) void k_shrink(const mk_lora_adapter* __restrict__ adapters, int n_adapters,
                                                     int max_rank, const int32_t* __restrict__ ids, int windows, int slots,
                                                     const float* __restrict__ x, int64_t x_stride, int n, int64_t cols,
                                                     int64_t per, bool x_vec, float* __restrict__ h, int r_pad) {
  __shared__ int tokens[kWindow];
  __shared__ v4f part[kShrinkWaves][8][64];
  const Group g = group_of(blockIdx.x % windows, blockIdx.y, slots, n, ids, adapters, n_adapters, max_rank, tokens);
  const int r0 = 32 * blockIdx.z, split = blockIdx.x / windows;
  if (!g.count || r0 >= g.a.rank) return;
  const int64_t k0 = split * per, k1 = min(cols, k0 + per);
  h += (int64_t)split * n * r_pad;
  if (g.count <= 16) shrink<T, 1>(g, tokens, x, x_stride, cols, r0, k0, k1, x_vec, h, r_pad, part);
  else shrink<T, 4>(g, tokens, x, x_stride, cols, r0, k0, k1, x_vec, h, r_pad, part);
}

// y = base + scale B h. A wave takes 64 rows of B in four MFMA tiles, and the group's tokens 16 at a time; the products go
// through LDS, so that base is read and y written 256 bytes of a token at a time. (512 rows per workgroup: 8 / 64 / 512
// tokens as above 9.8 / 21.4 / 43 us a pass instead of 9.6 / 17.0 / 38.3, and no room for rank 512.) The code is kept short
// (rolled loops): a workgroup runs most of it once, and instruction fetches that miss would cost more than the arithmetic.
// YV: rows of y and base are aligned to four floats, and of a multiple of four. The loop over the tokens has no branches of
// a lane's own but its stores: with them every turn waited for the stores of the one before (512 tokens as above 38 us
// instead of 31.6, 310 tokens of rank 64 48 instead of 35, when they were taken out). Three workgroups per CU for 16-bit
// adapters, at the cost of one spilled register with YV and eleven without (64 / 512 tokens 17.0 / 38.3 us; two, without
// spills, 19.2 / 43, four 21.7 / 60), two for fp32, whose weights take twice the registers (245 tokens of rank 62, 4096 -> 4096,
// 27 us; three, with spills, 36).
template <typename T, bool YV>
__global__ __launch_bounds__(kThreads, sizeof(T) == 4 ? 2 : 3) void k_expand(const mk_lora_adapter* __restrict__ adapters, int n_adapters,
                                                     int max_rank, const int32_t* __restrict__ ids, int windows, int slots,
                                                     int n, int64_t rows, const float* __restrict__ h, int r_pad, int splits,
                                                     const float* base, int64_t base_stride, float* y,
                                                     int64_t y_stride) {
  constexpr int kOut = 64 + 4;  // a token's stride in `out`
  __shared__ int tokens[kWindow];
  __shared__ __align__(16) float out_s[4][16 * kOut];
  extern __shared__ __align__(16) float hs[];  // [16 or 64][r_pad + 4]: the group's h, scaled
  const Group g = group_of(blockIdx.x % windows, blockIdx.y, slots, n, ids, adapters, n_adapters, max_rank, tokens);
  const int rank = g.a.rank;
  if (!g.count || (!rank && base == y)) return;
  const int hst = r_pad + 4, w = threadIdx.x >> 6, lane = threadIdx.x & 63, li = lane & 15, lq = lane >> 4;
  const int64_t row0 = (int64_t)(blockIdx.x / windows) * kRowBlock + 64 * w, row = row0 + 4 * li;
  const int valid = within(rows - row, 4);
  const bool b_vec = (rank & 3) == 0 && ((uintptr_t)g.a.b & (4 * sizeof(T) - 1)) == 0;
  // A tile of tokens (those past the last: the last) and its base; lane: token 4 k + lq, four rows from 4 li.
  auto load_base = [&](int c0, v4f(&v)[4], int(&tok)[4]) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < 4; ++k) tok[k] = tokens[min(c0 + 4 * k + lq, g.count - 1)];
    if (base) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        global<float>* p = to_global<float>(base + tok[k] * base_stride + (valid ? row : 0));
        if constexpr (YV) {
          v[k] = *reinterpret_cast<global<v4f>*>(p);
        } else {
          float q[4];
          get<4>(p, valid, false, q);
          v[k] = v4f{q[0], q[1], q[2], q[3]};
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    }
  };
  // 64 ranks of the wave's rows of B, four of a row per lane and step, as they lie in memory.
  typedef typename Raw<T>::type raw;
  raw bw[4][4];
  global<T>* b[4];
  auto load_b = [&](int r) __attribute__((always_inline)) {
    if (b_vec) {
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        if (r + 16 * s >= rank) break;
#pragma unroll
        for (int i = 0; i < 4; ++i) bw[s][i] = get_raw<true>(b[i], r + 16 * s + 4 * lq, rank);
      }
    } else {
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        if (r + 16 * s >= rank) break;
#pragma unroll
        for (int i = 0; i < 4; ++i) bw[s][i] = get_raw<false>(b[i], r + 16 * s + 4 * lq, rank);
      }
    }
  };
  // What does not wait for h is asked for first.
  v4f now[4], later[4];
  int tok[4], tok1[4];
  load_base(0, now, tok);
  if (rank) {
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = to_global<T>(g.a.b) + min(row0 + 16 * i + li, rows - 1) * rank;
    load_b(0);
    // h: its partial sums in order, four ranks a thread; where a group has few, 2^f threads take every 2^f-th split and
    // are added across lanes.
    const int quads = (rank + 15) / 16 * 4, used = g.count * quads, items = (g.count + 15) / 16 * 16 * quads;
    int f = 0;
    while (f < 4 && (used << (f + 1)) <= kThreads) ++f;
    const int part = threadIdx.x & ((1 << f) - 1);
#pragma unroll 1
    for (int i0 = 0; i0 < used; i0 += kThreads >> f) {
      const int i = i0 + (threadIdx.x >> f), c = i / quads, r = 4 * (i - c * quads);
      v4f s = {0.0f, 0.0f, 0.0f, 0.0f};
      if (i < used) {
        const float* at = h + (int64_t)tokens[c] * r_pad + r;
        const int64_t step = (int64_t)n * r_pad;
#pragma unroll 8
        for (int p = part; p < splits; p += 1 << f) s += *reinterpret_cast<const v4f*>(at + p * step);
      }
#pragma unroll 1
      for (int m = 1; m < 1 << f; m <<= 1)
#pragma unroll
        for (int k = 0; k < 4; ++k) s[k] += __shfl_xor(s[k], m);
      // Ranks past the last are 0 times x in h, which is NaN where x is infinite, and meet B's padding of 0.
#pragma unroll
      for (int k = 0; k < 4; ++k) s[k] = r + k < rank ? s[k] * g.a.scale : 0.0f;
      if (i < used && part == 0) *reinterpret_cast<v4f*>(hs + c * hst + r) = s;
    }
    for (int i = used + threadIdx.x; i < items; i += kThreads)
      *reinterpret_cast<v4f*>(hs + i / quads * hst + 4 * (i % quads)) = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    __syncthreads();
  }
  if (row0 >= rows) return;
  float* out = out_s[w];
#pragma unroll 1
  for (int c0 = 0; c0 < g.count; c0 += 16) {
    if (c0 + 16 < g.count) load_base(c0 + 16, later, tok1);
    if (rank) {
      v4f acc[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
      for (int r = 0; r < rank; r += 64) {
        if (r || (c0 && rank > 64)) load_b(r);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          if (r + 16 * s >= rank) break;
          const v4f hv = *reinterpret_cast<const v4f*>(hs + (c0 + li) * hst + r + 16 * s + 4 * lq);
          float bv[4][4];
#pragma unroll
          for (int i = 0; i < 4; ++i) from_raw<T>(bw[s][i], bv[i]);
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(bv[i][k], hv[k], acc[i], 0, 0, 0);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) *reinterpret_cast<v4f*>(out + li * kOut + 16 * i + 4 * lq) = acc[i];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // a wave's LDS accesses happen in order
#pragma unroll
      for (int k = 0; k < 4; ++k) now[k] += *reinterpret_cast<const v4f*>(out + (4 * k + lq) * kOut + 4 * li);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool on = c0 + 4 * k + lq < g.count;
      float* to = y + tok[k] * y_stride + row;
      if constexpr (YV) {
        if (on && valid) *reinterpret_cast<v4f*>(to) = now[k];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (on && e < valid) to[e] = now[k][e];
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) now[k] = later[k], tok[k] = tok1[k];
  }
}

int rank_pad(int max_rank) { return (max_rank + 15) & ~15; }

// Column splits of the first product, of at least two steps of every wave each: more make the sum over them in k_expand
// long, fewer the chain of steps (8 / 64 / 512 tokens as above 9.6 / 17.0 / 38.3 us a pass, with at most 4 splits 10.5 /
// 22.1 / 45.8, with at most 8 9.6 / 18.8 / 38.3, with at least one step 9.2 / 20.3 / 35.9; 245 fp32 tokens of rank 62, 4096 ->
// 4096, 27.3, with one step 33.6; 310 tokens of rank 64 over 8 adapters, 12288 -> 4096, 35.0, with 8 splits 34.7, with 12
// 40.2, and in fp32 45.0, 38.7 and 43.3).
constexpr int kMostSplits = 16, kWantedWindows = 256;  // splits times windows
int most_splits(int64_t cols) {
  return (int)std::max<int64_t>(1, std::min<int64_t>(kMostSplits, cols / (2 * kStep * kShrinkWaves)));
}
int windows_of(int n) { return (n - 1) / kWindow + 1; }  // n > 0
int splits_of(int n, int64_t cols) {
  const int windows = windows_of(n);
  return std::min(most_splits(cols), (kWantedWindows + windows - 1) / windows);
}
int64_t blocks_of(int64_t rows) { return (rows + kRowBlock - 1) / kRowBlock; }

bool aligned16(const void* p, int64_t stride) { return ((uintptr_t)p & 15) == 0 && (stride & 3) == 0; }

}  // namespace

// The most of any batch up to n: fewer tokens have more splits, and s of them up to (kWantedWindows - 1) / (s - 1) windows.
size_t lora_workspace(int n, int max_rank, int64_t cols) {
  int64_t sums = n;
  for (int s = 2; s <= most_splits(cols); ++s)
    sums = std::max(sums, s * std::min<int64_t>(n, (kWantedWindows - 1) / (s - 1) * kWindow));
  return (size_t)sums * rank_pad(max_rank) * sizeof(float);
}

size_t lora_need(int n, int max_rank, int64_t rows, int64_t cols) {
  const int64_t windows = windows_of(n);
  require(std::max(windows * splits_of(n, cols) * 64 * kShrinkWaves, windows * blocks_of(rows) * kThreads) < (1ll << 32),
          "mk_lora: too many tokens");
  return (size_t)splits_of(n, cols) * n * rank_pad(max_rank) * sizeof(float);
}

void lora(hipStream_t s, int type, const mk_lora_adapter* adapters, int n_adapters, int max_rank, const int32_t* ids,
          const float* x, int64_t x_stride, int n, int64_t rows, int64_t cols, const float* base, int64_t base_stride,
          float* y, int64_t y_stride, void* workspace) {
  const int splits = splits_of(n, cols), r_pad = rank_pad(max_rank);
  const int64_t step = kStep * kShrinkWaves, per = ((cols + splits - 1) / splits + step - 1) / step * step;
  const bool x_vec = aligned16(x, x_stride);
  const bool y_vec = (rows & 3) == 0 && aligned16(y, y_stride) && (!base || aligned16(base, base_stride));
  float* h = static_cast<float*>(workspace);
  const int slots = n_adapters < kFewSlots - 1 ? n_adapters + 1 : kWindow;
  const int windows = windows_of(n);
  const unsigned used = std::min(slots, n);
  const dim3 g1((unsigned)(windows * splits), used, (r_pad + 31) / 32), g2((unsigned)(windows * blocks_of(rows)), used);
  const size_t lds = (size_t)(n <= 16 ? 16 : kWindow) * (r_pad + 4) * sizeof(float);
  auto go = [&]<typename T>() {
    if (n_adapters > 0) {
      hipLaunchKernelGGL(k_shrink<T>, g1, dim3(64 * kShrinkWaves), 0, s, adapters, n_adapters, max_rank, ids, windows,
                         slots, x, x_stride, n, cols, per, x_vec, h, r_pad);
      check_launch("lora shrink");
    }
    auto expand = [&]<bool YV>() {
      allow_lds<k_expand<T, YV>>(kWindow * (512 + 4) * sizeof(float));
      hipLaunchKernelGGL((k_expand<T, YV>), g2, dim3(kThreads), lds, s, adapters, n_adapters, max_rank, ids, windows, slots,
                         n, rows, h, r_pad, splits, base, base_stride, y, y_stride);
    };
    if (y_vec) expand.template operator()<true>();
    else expand.template operator()<false>();
    check_launch("lora expand");
  };
  if (type == MK_F32) go.template operator()<float>();
  else if (type == MK_F16) go.template operator()<F16>();
  else go.template operator()<BF16>();
}

}  // namespace mk
