// Attention over the 4-bit cache in pages: out = sum_j p_j v_j, p = softmax(scale q.k_j), k = s (n - 8) and v likewise, exact in
// fp16.
//
// Rows and keys. A query row is a (token, query head); the rows of one KV head and of up to 16 / G tokens of one sequence that
// follow each other (G query heads per KV head) are a block of at most 16 rows that reads the same keys, 64 at a time. A tile's
// 16-key chunks lie in one page each.
//
// Arithmetic. v_mfma_f32_16x16x32_f16 with the fp32 side in two fp16 parts, hi = fp16(x) and lo = fp16(x - hi): 2^-23 of x is
// kept. A row of q is first brought to a largest value of 2^13 .. 2^14 by a power of two; the weights are shifted so that the
// largest was 2^10 when the shift was set, so a lo part holds 2^-35 of it. Scores, statistics and outputs are fp32.
//
// S = K Q^T has keys in its rows and query rows in its columns: a lane's 16 scores belong to one query row, and the weights are,
// as they lie, the second operand of O^T = V^T P^T. V^T comes from the transposing 4-bit LDS read. A lane's elements of a key,
// in the order that its numbers come out of a word, are the order in which q's elements are multiplied; the same goes for the
// keys of V. Each wave takes every NW-th tile through a K and a V buffer of its own, which direct copies fill: a buffer's next
// tile is asked for as soon as this one is in registers, and the waves meet only to add their results.
#include <algorithm>

#include "ctx.h"
#include "ops.h"

namespace mk {
namespace {

typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v4a __attribute__((ext_vector_type(4), aligned(4)));
typedef int v2i __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) v2i lds_v2i;

constexpr float kNone = -3e38f;  // shift of a row that has seen no key
constexpr float kLog2e = 1.44269504088896341f;
constexpr int kTile = 64, kChunk = 16;
constexpr int kFew = 16;      // query rows of a block
constexpr int kIds = 1024;    // pages of chunks held in LDS at a time

// A block of rows of one KV head, and how many keys its tokens see at most.
struct Block {
  int t0, m, keys;  // tokens t0 .. t0 + m - 1
  int g, h0, per;   // KV head, first query head, heads per token
  __device__ __forceinline__ int rows() const { return m * per; }
  __device__ __forceinline__ int token(int r) const { return t0 + r / per; }
  __device__ __forceinline__ int head(int r) const { return h0 + r % per; }
};

__device__ __forceinline__ int keys_of(const Kv4Attn& A, int t) {
  const int s = A.seq[t];
  return s >= 0 && s < A.kv.n_seq ? max(0, min(A.n_keys[t], A.max_keys)) : 0;
}

__device__ __forceinline__ void fence() { asm volatile("" ::: "memory"); }
__device__ __forceinline__ void wait_lds() {
  fence();
  __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
  fence();
}

// x as hi + lo.
__device__ __forceinline__ void split8(const float (&x)[8], v8h& hi, v8h& lo) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const v2f f = {x[i], x[i + 1]};
    const v2h h = __builtin_convertvector(f, v2h);
    const v2f g = {x[i] - (float)h[0], x[i + 1] - (float)h[1]};
    const v2h l = __builtin_convertvector(g, v2h);
    hi[i] = h[0], hi[i + 1] = h[1], lo[i] = l[0], lo[i + 1] = l[1];
  }
}

// Eight numbers of a word as n - 8, exactly, in the order 0, 4, 1, 5, 2, 6, 3, 7: a number under the exponent of 1024 reads
// 1024 + n in the lowest four bits of the fraction, under that of 64 reads 64 + n four bits further up.
__device__ __forceinline__ void less8(uint32_t w, v2h (&r)[4]) {
  const v2h a = {(_Float16)1032.0f, (_Float16)1032.0f}, b = {(_Float16)72.0f, (_Float16)72.0f};
  r[0] = __builtin_bit_cast(v2h, (w & 0x000F000Fu) | 0x64006400u) - a;
  r[1] = __builtin_bit_cast(v2h, (w & 0x00F000F0u) | 0x54005400u) - b;
  w >>= 8;
  r[2] = __builtin_bit_cast(v2h, (w & 0x000F000Fu) | 0x64006400u) - a;
  r[3] = __builtin_bit_cast(v2h, (w & 0x00F000F0u) | 0x54005400u) - b;
}
__device__ __forceinline__ v8h join8(const v2h (&r)[4]) {
  return v8h{r[0][0], r[0][1], r[1][0], r[1][1], r[2][0], r[2][1], r[3][0], r[3][1]};
}
// Place of the e-th of eight elements (or keys) in that order.
__device__ __forceinline__ constexpr int place(int e) { return (e & 1) * 4 + (e >> 1); }

template <int D>
struct Geo {
  static constexpr int kSteps = D / 32;            // MFMAs over a row: lane qd of four holds its elements D / 4 qd + ..
  static constexpr int kDt = D / 16;               // 16-element tiles of a row
  static constexpr int kRow = D / 2, kGroups = D / 32;
  static constexpr int kBytes = kTile * kRow;      // of K or V
  static constexpr int kScales = kTile * kGroups * 2;
  static constexpr int kCopies = kBytes / 1024 + kScales / 256;
  static constexpr int kWave = 2 * (kBytes + kScales);
  static constexpr int kStride = D + 4;            // of a row of results
};

// What a wave holds of its rows: this lane's is row lane % 16; o[i][j] is its element 16 i + 4 (lane / 16) + j.
template <int D>
struct Acc {
  v4f o[Geo<D>::kDt];
  float m, l;  // weights are 2^(score - m), l this lane's sum of them
};

// One wave's copies and products. Everything here is the wave's own: no barrier.
template <int D>
struct Walk {
  using G_ = Geo<D>;
  const Kv4Attn& A;
  int g, lane, li, qd;
  uint8_t *ks_s, *k_s, *v_s, *vs_s;
  uint32_t k_off, v_off;  // this lane's part of a copy
  v8h hi[G_::kSteps], lo[G_::kSteps];
  float rf;        // score, in bits, of one unit of a product
  int lim, least;  // keys that this lane's row sees, and that every row of the block sees

  __device__ __forceinline__ Walk(const Kv4Attn& a, uint8_t* lds) : A(a) {
    lane = threadIdx.x & 63, li = lane & 15, qd = lane >> 4;
    k_s = lds, v_s = k_s + G_::kBytes, ks_s = v_s + G_::kBytes, vs_s = ks_s + G_::kScales;
    if constexpr (D == 128) {
      k_off = li * 64 + 16 * qd;
      v_off = (lane >> 2) * 64 + 16 * ((lane & 3) ^ (lane >> 4));
    } else {
      k_off = (lane & 31) * 16;
      v_off = ((lane & 31) >> 1) * 32 + 16 * ((lane & 1) ^ ((lane >> 4) & 1));
    }
  }

  // This lane's row of q, scaled, in two parts.
  __device__ __forceinline__ void load_q(const Block& b, const float* q, int64_t q_stride) {
    g = b.g;
    const int r = min(li, b.rows() - 1), t = b.token(r);
    const float* qr = q + t * q_stride + (int64_t)b.head(r) * D + D / 4 * qd;
    float x[G_::kSteps][8], top = 0.0f;
#pragma unroll
    for (int s = 0; s < G_::kSteps; ++s) {
      float y[8];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const v4f f = *reinterpret_cast<const v4a*>(qr + 8 * s + 4 * c);
#pragma unroll
        for (int e = 0; e < 4; ++e) y[4 * c + e] = f[e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) x[s][e] = y[place(e)], top = fmaxf(top, fabsf(y[e]));
    }
    lim = keys_of(A, t);
    least = lim;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) least = min(least, __shfl_xor(least, o));
    least = __builtin_amdgcn_readfirstlane(least);
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    int ex = 0;
    if (top > 0.0f && top < INFINITY) ex = min(14 - __builtin_amdgcn_frexp_expf(top), 100);
    rf = __builtin_ldexpf(A.scale * kLog2e, -ex);
#pragma unroll
    for (int s = 0; s < G_::kSteps; ++s) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[s][e] = __builtin_ldexpf(x[s][e], ex);
      split8(x[s], hi[s], lo[s]);
    }
  }

  // First row of the tile's chunk c in the pool, less its row in the page, and that row. Chunks without a page: page 0's.
  struct Place {
    int64_t first;
    int r;
  };
  __device__ __forceinline__ Place where(const int* ids, int key, int c) const {
    const int p = max(__builtin_amdgcn_readfirstlane(ids[c]), 0);
    return Place{A.kv.first_row(p, g), (key + kChunk * c) & ((1 << A.kv.shift) - 1)};
  }
  // ids: the tile's four chunks' pages; key: its first key.
  __device__ __forceinline__ void issue_k(const int* ids, int key) const {
    Place at[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) at[c] = where(ids, key, c);
    if constexpr (D == 128) {
#pragma unroll
      for (int c = 0; c < 4; ++c) lds_copy16(A.kv.k + (at[c].first + at[c].r) * 64, k_off, k_s + 1024 * c);
#pragma unroll
      for (int c = 0; c < 4; c += 2) {
        const int64_t row = lane < 32 ? at[c].first + at[c].r : at[c + 1].first + at[c + 1].r;
        lds_copy4(reinterpret_cast<const uint8_t*>(A.kv.ks) + row * 8 + 4 * (lane & 31), ks_s + 128 * c);
      }
    } else {
#pragma unroll
      for (int c = 0; c < 4; c += 2) {
        const int64_t row = lane < 32 ? at[c].first + at[c].r : at[c + 1].first + at[c + 1].r;
        lds_copy16(A.kv.k + row * 32 + k_off, k_s + 512 * c);
      }
      const int64_t a = lane & 16 ? at[1].first + at[1].r : at[0].first + at[0].r;
      const int64_t b = lane & 16 ? at[3].first + at[3].r : at[2].first + at[2].r;
      lds_copy4(reinterpret_cast<const uint8_t*>(A.kv.ks) + (lane < 32 ? a : b) * 4 + 4 * li, ks_s);
    }
  }
  // The scales of V in LDS: [chunk][group][key].
  __device__ __forceinline__ void issue_v(const int* ids, int key) const {
    Place at[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) at[c] = where(ids, key, c);
    auto scales = [&](int c) { return at[c].first * G_::kGroups + at[c].r; };
    const int in = ((lane >> 3) & (G_::kGroups - 1)) << A.kv.shift;
    if constexpr (D == 128) {
#pragma unroll
      for (int c = 0; c < 4; ++c) lds_copy16(A.kv.v + (at[c].first + at[c].r) * 64, v_off, v_s + 1024 * c);
#pragma unroll
      for (int c = 0; c < 4; c += 2)
        lds_copy4(A.kv.vs + (lane < 32 ? scales(c) : scales(c + 1)) + in + 2 * (lane & 7), vs_s + 128 * c);
    } else {
#pragma unroll
      for (int c = 0; c < 4; c += 2) {
        const int64_t row = lane < 32 ? at[c].first + at[c].r : at[c + 1].first + at[c + 1].r;
        lds_copy16(A.kv.v + row * 32 + v_off, v_s + 512 * c);
      }
      const int64_t a = lane & 16 ? scales(1) : scales(0), b = lane & 16 ? scales(3) : scales(2);
      lds_copy4(A.kv.vs + (lane < 32 ? a : b) + in + 2 * (lane & 7), vs_s);
    }
  }

  // One tile: keys key .. key + 63, of which those below `end` count (end <= the block's keys). next: the pages of the wave's
  // next tile at key `next_key`, or NULL.
  __device__ __forceinline__ void tile(Acc<D>& acc, bool& fresh, const int* ids, int key, int end, const int* next, int next_key) const {
    wait_vm<G_::kCopies>();  // this tile's K; its V may be under way
    fence();
    int have = 0;  // chunks that have a page
#pragma unroll
    for (int c = 0; c < 4; ++c) have |= (__builtin_amdgcn_readfirstlane(ids[c]) >= 0) << c;
    const bool whole = key + kTile <= min(least, end) && have == 15;
    v4f s[4];
    {
      uint32_t w[4][G_::kSteps];
      _Float16 sc[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if constexpr (D == 128) {
          const uint4 x = *reinterpret_cast<const uint4*>(k_s + 1024 * c + 16 * lane);
          w[c][0] = x.x, w[c][1] = x.y, w[c][2] = x.z, w[c][3] = x.w;
          sc[c] = reinterpret_cast<const _Float16*>(ks_s)[(kChunk * c + li) * 4 + qd];
        } else {
          const uint2 x = *reinterpret_cast<const uint2*>(k_s + (kChunk * c + li) * 32 + 8 * qd);
          w[c][0] = x.x, w[c][1] = x.y;
          sc[c] = reinterpret_cast<const _Float16*>(ks_s)[(kChunk * c + li) * 2 + (qd >> 1)];
        }
      }
      wait_lds();  // K is in registers, and its place free for the next tile's
      if (next) issue_k(next, next_key);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        s[c] = v4f{};
        const v2h f = {sc[c], sc[c]};
#pragma unroll
        for (int i = 0; i < G_::kSteps; ++i) {
          v2h r[4];
          less8(w[c][i], r);
#pragma unroll
          for (int j = 0; j < 4; ++j) r[j] *= f;
          const v8h a = join8(r);
          s[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, hi[i], s[c], 0, 0, 0);
          s[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, lo[i], s[c], 0, 0, 0);
        }
      }
    }
    // Register i of chunk c is key 16 c + 4 qd + i.
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      s[c] *= rf;
      if (!whole)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int k = key + kChunk * c + 4 * qd + i;
          s[c][i] = k < min(lim, end) && (have >> c & 1) ? s[c][i] : -INFINITY;
        }
    }
    float p[16], sum, top;
    auto weights = [&] __attribute__((always_inline)) {
      sum = top = 0.0f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        p[i] = __builtin_amdgcn_exp2f(s[i / 4][i % 4] - acc.m);
        sum += p[i];
        top = fmaxf(top, p[i]);
      }
    };
    if (!fresh) weights();
    // The first tile, and one whose weights leave fp16: a new shift, 10 below the largest score (that score itself where 10
    // is not exact beside it).
    if (fresh || __ballot(top > 32768.0f)) {
      float z = -INFINITY;
#pragma unroll
      for (int i = 0; i < 16; ++i) z = fmaxf(z, s[i / 4][i % 4]);
      z = fmaxf(z, __shfl_xor(z, 16));
      z = fmaxf(z, __shfl_xor(z, 32));
      const float m = fmaxf(acc.m, fabsf(z) < 0x1p24f ? z - 10.0f : z);
      const float f = __builtin_amdgcn_exp2f(acc.m - m);
      acc.m = m, acc.l *= f;
      if (!fresh) {
#pragma unroll
        for (int i = 0; i < G_::kDt; ++i) acc.o[i] *= f;
      }
      fresh = false;
      weights();
    }
    acc.l += sum;
    v8h ph[2], pl[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = p[8 * u + e];
      split8(y, ph[u], pl[u]);
    }
    if (next) wait_vm<G_::kCopies>();  // this tile's V; the next one's K may be under way
    else wait_vm<0>();
    fence();
    // A lane gives the address of a key's 16 elements and gets an element's 16 keys: number 8 u + x is the key of weight
    // 8 u + e with place(e) = x, which is 16 (2 u + e / 4) + 4 qd + e % 4.
    v2i vv[G_::kDt];
    v4h sc[G_::kGroups][4];
    {
      const int x = li & 7, e = 2 * (x & 3) + (x >> 2), k = 16 * (2 * (li >> 3) + (e >> 2)) + 4 * qd + (e & 3);
      const int turn = D == 128 ? (k >> 2) & 3 : (k >> 3) & 1;
#pragma unroll
      for (int i = 0; i < G_::kDt; ++i)
        vv[i] = __builtin_amdgcn_ds_read_tr4_b64_v2i32((lds_v2i*)(v_s + k * G_::kRow + 16 * ((i >> 1) ^ turn) + 8 * (i & 1)));
    }
#pragma unroll
    for (int n = 0; n < G_::kGroups; ++n)
#pragma unroll
      for (int c = 0; c < 4; ++c) sc[n][c] = *reinterpret_cast<const v4h*>(vs_s + ((c * G_::kGroups + n) * 16 + 4 * qd) * 2);
    wait_lds();
    if (next) issue_v(next, next_key);
    if (!whole) {  // a weight of 0 does not undo what lies in a place that nothing was written to
#pragma unroll
      for (int n = 0; n < G_::kGroups; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (key + kChunk * c + 4 * qd + i >= end || !(have >> c & 1)) sc[n][c][i] = (_Float16)0.0f;
    }
#pragma unroll
    for (int i = 0; i < G_::kDt; ++i)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        v2h r[4];
        less8((uint32_t)vv[i][u], r);
        const v4h a = sc[i / 2][2 * u], b = sc[i / 2][2 * u + 1];
        r[0] *= v2h{a[0], a[1]}, r[1] *= v2h{a[2], a[3]}, r[2] *= v2h{b[0], b[1]}, r[3] *= v2h{b[2], b[3]};
        const v8h x = join8(r);
        acc.o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, ph[u], acc.o[i], 0, 0, 0);
        acc.o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, pl[u], acc.o[i], 0, 0, 0);
      }
  }
};

// Tiles [ta, tb) of a block by the workgroup's NW waves; then put(row, element, its four values as weighted sums, l, m) by the
// 16 threads that share a row, 64 / .. elements each.
template <int D, int NW, class Put>
__device__ __forceinline__ void run_block(const Kv4Attn& A, const Block& b, int ta, int tb, const float* q, int64_t q_stride,
                                          uint8_t* smem, int* ids, v2f (*ml)[kFew], Put put) {
  using G_ = Geo<D>;
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int end = min(b.keys, tb * kTile), seq = A.seq[b.t0];
  Walk<D> walk(A, smem + w * G_::kWave);
  walk.load_q(b, q, q_stride);
  Acc<D> acc;
#pragma unroll
  for (int i = 0; i < G_::kDt; ++i) acc.o[i] = v4f{};
  acc.m = kNone, acc.l = 0.0f;
  bool fresh = true;
  for (int t0 = ta; t0 < tb; t0 += kIds / 4) {  // pages of as many tiles as LDS holds
    const int t1 = min(tb, t0 + kIds / 4);
    __syncthreads();
    for (int i = tid; i < 4 * (t1 - t0); i += NW * 64) {
      const int key = t0 * kTile + kChunk * i;
      ids[i] = key < end ? A.kv.page_of(seq, key) : -1;
    }
    __syncthreads();
    auto pages = [&](int t) { return ids + 4 * (t - t0); };
    int t = t0 + w;
    if (t < t1) walk.issue_k(pages(t), t * kTile), walk.issue_v(pages(t), t * kTile);
    for (; t < t1; t += NW) {
      const bool more = t + NW < t1;
      walk.tile(acc, fresh, pages(t), t * kTile, end, more ? pages(t + NW) : nullptr, (t + NW) * kTile);
    }
  }
  // The waves' parts of each row, brought to their largest shift and added.
  float l = acc.l + __shfl_xor(acc.l, 16);
  l += __shfl_xor(l, 32);
  __syncthreads();
  float* ob = reinterpret_cast<float*>(smem);
  if (walk.qd == 0) ml[w][walk.li] = v2f{acc.m, l};
#pragma unroll
  for (int i = 0; i < G_::kDt; ++i)
    *reinterpret_cast<v4f*>(ob + (w * kFew + walk.li) * G_::kStride + 16 * i + 4 * walk.qd) = acc.o[i];
  __syncthreads();
  for (int r = tid >> 4; r < b.rows(); r += NW * 4) {
    float f[NW], top = kNone, sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NW; ++i) top = fmaxf(top, ml[i][r][0]);
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      f[i] = __builtin_amdgcn_exp2f(ml[i][r][0] - top);
      sum = fma_(f[i], ml[i][r][1], sum);
    }
#pragma unroll
    for (int d0 = 0; d0 < D; d0 += 64) {
      const int d = d0 + 4 * (tid & 15);
      v4f a = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < NW; ++i) a += f[i] * *reinterpret_cast<const v4f*>(ob + (i * kFew + r) * G_::kStride + d);
      put(r, d, a, sum, top);
    }
  }
}

template <int D, int NW>
struct FewLds {
  static constexpr int kRing = NW * Geo<D>::kWave, kOut = NW * kFew * Geo<D>::kStride * 4;
  static constexpr int kBytes = kRing > kOut ? kRing : kOut;
};

// Four values of a row of the output, by the threads of a row together.
template <int D>
__device__ __forceinline__ void put_row(const Kv4Attn& A, float* out, int64_t out_stride, BlockQ8* xq, int t, int head, int d,
                                        const float (&y)[4]) {
  *reinterpret_cast<v4a*>(out + t * out_stride + (int64_t)head * D + d) = v4a{y[0], y[1], y[2], y[3]};
  if (xq) quantize_block_lanes_n<4>(y, (d & 31) / 4, xq + (((int64_t)t * A.H + head) * D + d) / 32);
}

// The tokens from t on that a block may have with it, tq at most.
__device__ __forceinline__ Block block_at(const Kv4Attn& A, int t, int tq, int j) {
  const int G = A.H / A.kv.KV, hs = (G + kFew - 1) / kFew, sub = j % hs;
  Block b{t, 1, keys_of(A, t), j / hs, j / hs * G + kFew * sub, min(G - kFew * sub, kFew)};
  const int s = A.seq[t];
  while (b.m < tq && t + b.m < A.n && (t + b.m) % tq && A.seq[t + b.m] == s) b.keys = max(b.keys, keys_of(A, t + b.m)), ++b.m;
  return b;
}

// A workgroup per token and KV head (per 16 of its query heads); the first token of its sequence, or of tq tokens, leads a
// block and the others' workgroups leave.
template <int D, int NW>
__global__ __launch_bounds__(NW * 64) void k_kv4_whole(Kv4Attn A, const float* __restrict__ q, int64_t q_stride,
                                                       float* __restrict__ out, int64_t out_stride, BlockQ8* __restrict__ xq) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int ids[kIds];
  __shared__ v2f ml[NW][kFew];
  const int G = A.H / A.kv.KV, hs = (G + kFew - 1) / kFew, J = A.kv.KV * hs, tq = max(1, kFew / G);
  const int t = blockIdx.x / J;
  if (t % tq && A.seq[t - 1] == A.seq[t]) return;
  const Block b = block_at(A, t, tq, blockIdx.x % J);
  run_block<D, NW>(A, b, 0, (b.keys + kTile - 1) / kTile, q, q_stride, smem, ids, ml, [&](int r, int d, v4f a, float l, float m) {
    const float n = l == 0.0f ? 1.0f : l;  // no key: zeros
    const float y[4] = {a[0] / n, a[1] / n, a[2] / n, a[3] / n};
    put_row<D>(A, out, out_stride, xq, b.token(r), b.head(r), d, y);
  });
}

}  // namespace

size_t attention_kv4_workspace(int n, int H, int KV, int D, int max_keys, int max_run) { return 0; }

size_t attention_kv4_need(const Kv4Attn& A, int D) { return 0; }

void attention_kv4(hipStream_t s, const Kv4Attn& A, int D, const float* q, int64_t q_stride, float* out, int64_t out_stride,
                   BlockQ8* xq, void* workspace) {
  const int G = A.H / A.kv.KV, J = A.kv.KV * ((G + kFew - 1) / kFew);
  auto go = [&]<int D_>() {
    constexpr int NW = 4;
    allow_lds<k_kv4_whole<D_, NW>>(FewLds<D_, NW>::kBytes);
    hipLaunchKernelGGL((k_kv4_whole<D_, NW>), dim3((unsigned)((int64_t)A.n * J)), dim3(NW * 64), (FewLds<D_, NW>::kBytes), s, A, q,
                       q_stride, out, out_stride, xq);
    check_launch("attention_kv4");
  };
  if (D == 128) go.template operator()<128>();
  else go.template operator()<64>();
}

}  // namespace mk
