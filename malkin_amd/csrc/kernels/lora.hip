// Low-rank adapters of many requests at once beside a shared projection: y[t] = base[t] + scale_a B_a (A_a x[t]), the
// adapter a = ids[t] chosen per token. A is [rank][cols], B [rows][rank] (the layouts of a GGUF adapter's lora_a and
// lora_b), both in one of three types; x, base, y and every sum are fp32.
//
// Two launches: k_shrink makes h = A x for every token, the columns split over workgroups (partial sums in the
// workspace, added in a fixed order by the next launch), k_expand adds scale B h to base. Both take the tokens of an
// aligned 16-token tile that share an adapter together, as the 16 columns of v_mfma_f32_16x16x4_f32 (weights as its 16
// rows): the workgroup of a token runs if the token is the first of its tile with its adapter and leaves at once
// otherwise, so a tile costs one pass over each adapter that occurs in it.
#include "ctx.h"
#include "ops.h"

namespace mk {
namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));

constexpr int kTile = 16;      // tokens of a tile
constexpr int kThreads = 256;  // 4 waves
constexpr int kRowBlock = 256; // rows of y per k_expand workgroup, 64 per wave

struct F16 { uint16_t v; };
struct BF16 { uint16_t v; };
__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(F16 v) { return (float)__builtin_bit_cast(_Float16, v.v); }
__device__ __forceinline__ float to_f(BF16 v) { return __builtin_bit_cast(float, (uint32_t)v.v << 16); }

// Four consecutive values, from an address aligned to their size.
__device__ __forceinline__ void load4(const float* p, float (&r)[4]) {
  const float4 v = *reinterpret_cast<const float4*>(p);
  r[0] = v.x, r[1] = v.y, r[2] = v.z, r[3] = v.w;
}
__device__ __forceinline__ void load4(const F16* p, float (&r)[4]) {
  const v4h v = *reinterpret_cast<const v4h*>(p);
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = (float)v[i];
}
__device__ __forceinline__ void load4(const BF16* p, float (&r)[4]) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  r[0] = __builtin_bit_cast(float, v.x << 16), r[1] = __builtin_bit_cast(float, v.x & 0xFFFF0000u);
  r[2] = __builtin_bit_cast(float, v.y << 16), r[3] = __builtin_bit_cast(float, v.y & 0xFFFF0000u);
}

// What a workgroup does with token t's tile: the adapter (-1: none), its entry, and the tile's tokens that take it
// (0: another token's workgroup covers t).
struct Group {
  int id, t0;
  uint32_t tokens;
  mk_lora_adapter a;
};
__device__ __forceinline__ Group group_of(int t, int n, const int32_t* ids, const mk_lora_adapter* adapters,
                                          int n_adapters, int max_rank) {
  Group g;
  g.t0 = t & ~(kTile - 1);
  g.a = mk_lora_adapter{nullptr, nullptr, 0.0f, 0};
  const int u = g.t0 + (threadIdx.x & 15);
  const int mine = u < n ? ids[u] : -1;
  const int v = mine >= 0 && mine < n_adapters ? mine : -1;
  const int own = __shfl(v, t - g.t0, 16);
  g.tokens = (uint32_t)__ballot(u < n && v == own) & 0xFFFFu;
  if (g.tokens & ((1u << (t - g.t0)) - 1)) g.tokens = 0;
  g.id = __builtin_amdgcn_readfirstlane(own);
  if (g.id >= 0) {
    g.a = adapters[g.id];
    if (g.a.rank < 1 || g.a.rank > max_rank || !g.a.a || !g.a.b) g.a.rank = 0;
  }
  return g;
}

// Partial sums h[split][t][r] of columns split * per .. over ranks 16 blockIdx.z ..: MFMA rows are ranks, columns
// tokens; a lane holds eight consecutive columns of its rank row and of its token, one per MFMA.
template <typename T>
__global__ __launch_bounds__(kThreads) void k_shrink(const mk_lora_adapter* __restrict__ adapters, int n_adapters,
                                                     int max_rank, const int32_t* __restrict__ ids,
                                                     const float* __restrict__ x, int64_t x_stride, int n, int64_t cols,
                                                     int per, bool x_vec, float* __restrict__ h, int r_pad) {
  const int t = blockIdx.x;
  const Group g = group_of(t, n, ids, adapters, n_adapters, max_rank);
  const int r0 = 16 * blockIdx.z;
  if (!g.tokens || r0 >= g.a.rank) return;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, li = lane & 15, lq = lane >> 4;
  const T* a = static_cast<const T*>(g.a.a) + (int64_t)min(r0 + li, g.a.rank - 1) * cols;
  const float* xr = x + (int64_t)min(g.t0 + li, n - 1) * x_stride;
  const bool row_on = r0 + li < g.a.rank, tok_on = (g.tokens >> li) & 1;
  const bool vec = x_vec && (cols & 7) == 0 && ((uintptr_t)g.a.a & 15) == 0;
  const int64_t k0 = (int64_t)blockIdx.y * per, k1 = min(cols, k0 + per);
  v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int64_t k = k0 + 32 * w; k < k1; k += 32 * 4) {
    const int64_t at = k + 8 * lq;
    float av[8], xv[8];
    if (vec) {
      const bool in = at < k1;  // per and cols are multiples of 8
      float q[4];
#pragma unroll
      for (int u = 0; u < 8; u += 4) {
        load4(a + (in ? at + u : 0), q);
#pragma unroll
        for (int i = 0; i < 4; ++i) av[u + i] = row_on && in ? q[i] : 0.0f;
        load4(xr + (in ? at + u : 0), q);
#pragma unroll
        for (int i = 0; i < 4; ++i) xv[u + i] = tok_on && in ? q[i] : 0.0f;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool in = at + i < k1;
        av[i] = row_on && in ? to_f(a[at + i]) : 0.0f;
        xv[i] = tok_on && in ? xr[at + i] : 0.0f;
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(av[i], xv[i], acc, 0, 0, 0);
  }
  __shared__ v4f part[4][64];
  part[w][lane] = acc;
  __syncthreads();
  if (w == 0 && tok_on) {
    const v4f s = (part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]);
    *reinterpret_cast<v4f*>(h + ((int64_t)blockIdx.y * n + g.t0 + li) * r_pad + r0 + 4 * lq) = s;
  }
}

// y = base + scale B h for 256 rows: MFMA rows are rows of B, columns tokens, so a lane ends with four consecutive
// rows of one token.
template <typename T>
__global__ __launch_bounds__(kThreads) void k_expand(const mk_lora_adapter* __restrict__ adapters, int n_adapters,
                                                     int max_rank, const int32_t* __restrict__ ids, int n, int64_t rows,
                                                     const float* __restrict__ h, int r_pad, int splits,
                                                     const float* base, int64_t base_stride, float* y, int64_t y_stride,
                                                     bool y_vec) {
  const int t = blockIdx.x;
  const Group g = group_of(t, n, ids, adapters, n_adapters, max_rank);
  if (!g.tokens) return;
  const int rank = g.a.rank;
  if (rank == 0 && base == y) return;
  extern __shared__ __align__(16) float hs[];  // [16][r_pad + 4]: the tile's h, scaled
  const int hst = r_pad + 4;
  const int rank16 = (rank + 15) & ~15;
  for (int i = threadIdx.x; i < kTile * rank16; i += kThreads) {
    const int tok = i / rank16, r = i % rank16;
    float s = 0.0f;
    if (((g.tokens >> tok) & 1) && r < rank)
      for (int p = 0; p < splits; ++p) s += h[((int64_t)p * n + g.t0 + tok) * r_pad + r];
    hs[tok * hst + r] = s * g.a.scale;
  }
  __syncthreads();
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, li = lane & 15, lq = lane >> 4;
  const bool b_vec = (rank & 3) == 0 && ((uintptr_t)g.a.b & (4 * sizeof(T) - 1)) == 0;
  const bool tok_on = (g.tokens >> li) & 1;
  for (int tile = 0; tile < 4; ++tile) {
    const int64_t row0 = (int64_t)blockIdx.y * kRowBlock + 64 * w + 16 * tile;
    if (row0 >= rows) break;
    const T* b = static_cast<const T*>(g.a.b) + min(row0 + li, rows - 1) * rank;
    v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int r = 0; r < rank; r += 16) {
      const int at = r + 4 * lq;
      float bv[4];
      if (b_vec) {
        load4(b + min(at, rank - 4), bv);
        if (at >= rank) bv[0] = bv[1] = bv[2] = bv[3] = 0.0f;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) bv[i] = at + i < rank ? to_f(b[at + i]) : 0.0f;
      }
      const float4 hv = *reinterpret_cast<const float4*>(hs + li * hst + at);
      acc = __builtin_amdgcn_mfma_f32_16x16x4f32(bv[0], hv.x, acc, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_f32_16x16x4f32(bv[1], hv.y, acc, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_f32_16x16x4f32(bv[2], hv.z, acc, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_f32_16x16x4f32(bv[3], hv.w, acc, 0, 0, 0);
    }
    if (!tok_on) continue;
    const int64_t row = row0 + 4 * lq;
    const float* bp = base ? base + (g.t0 + li) * base_stride + row : nullptr;
    float* yp = y + (g.t0 + li) * y_stride + row;
    if (y_vec) {
      if (row >= rows) continue;
      v4f v = bp ? *reinterpret_cast<const v4f*>(bp) : v4f{0.0f, 0.0f, 0.0f, 0.0f};
      if (rank) v += acc;
      *reinterpret_cast<v4f*>(yp) = v;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (row + i < rows) {
          float v = bp ? bp[i] : 0.0f;
          if (rank) v += acc[i];
          yp[i] = v;
        }
    }
  }
}

int rank_pad(int max_rank) { return (max_rank + 15) & ~15; }

// Column splits of the first product: enough workgroups for the CUs twice over, of at least 256 columns each.
int splits_of(int n, int64_t cols) {
  const int tiles = (n + kTile - 1) / kTile;
  return (int)std::max<int64_t>(1, std::min<int64_t>({16, (512 + tiles - 1) / tiles, cols / 256}));
}

bool aligned16(const void* p, int64_t stride) { return ((uintptr_t)p & 15) == 0 && (stride & 3) == 0; }

}  // namespace

size_t lora_workspace(int n, int max_rank, int64_t cols) {
  return (size_t)splits_of(n, cols) * n * rank_pad(max_rank) * sizeof(float);
}

void lora(hipStream_t s, int type, const mk_lora_adapter* adapters, int n_adapters, int max_rank, const int32_t* ids,
          const float* x, int64_t x_stride, int n, int64_t rows, int64_t cols, const float* base, int64_t base_stride,
          float* y, int64_t y_stride, void* workspace) {
  const int splits = splits_of(n, cols), r_pad = rank_pad(max_rank);
  const int per = (int)(((cols + splits - 1) / splits + 31) / 32 * 32);
  const bool x_vec = aligned16(x, x_stride);
  const bool y_vec = (rows & 3) == 0 && aligned16(y, y_stride) && (!base || aligned16(base, base_stride));
  float* h = static_cast<float*>(workspace);
  const dim3 g1(n, splits, r_pad / 16), g2(n, (unsigned)((rows + kRowBlock - 1) / kRowBlock));
  const size_t lds = (size_t)kTile * (r_pad + 4) * sizeof(float);
  auto go = [&]<typename T>() {
    hipLaunchKernelGGL(k_shrink<T>, g1, dim3(kThreads), 0, s, adapters, n_adapters, max_rank, ids, x, x_stride, n,
                       cols, per, x_vec, h, r_pad);
    check_launch("lora shrink");
    hipLaunchKernelGGL(k_expand<T>, g2, dim3(kThreads), lds, s, adapters, n_adapters, max_rank, ids, n, rows, h, r_pad,
                       splits, base, base_stride, y, y_stride, y_vec);
    check_launch("lora expand");
  };
  if (type == MK_F32) go.template operator()<float>();
  else if (type == MK_F16) go.template operator()<F16>();
  else go.template operator()<BF16>();
}

}  // namespace mk
