// Attention over the 4-bit cache in pages: out = sum_j p_j v_j, p = softmax(scale q.k_j), k = s (n - 8) and v likewise, in fp16.
//
// Rows and keys. A query row is a (token, query head); the rows of one KV head and of neighbouring tokens of one sequence are a
// block of at most 16 or 32 rows that reads the same keys, 64 at a time. A tile's 16-key chunks lie in one page each.
//
// Split. Where a call has few keys a workgroup takes a block, and that is all. Otherwise as many workgroups as the chip holds
// share all blocks' tiles evenly, whatever the sequences' lengths: each takes a contiguous run of them, writes the blocks that lie
// whole in its run, and leaves partial results of the first and the last one, which a second launch adds. A run's place follows
// from the tokens' lengths alone, by a running sum that every workgroup makes for itself.
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
//
// What bounds it: long documents the vector instructions that turn 4 bits into fp16 factors, 13 for eight values and as many for K
// as for V, which is 416 of a tile's 560 to 700 (16 or 32 rows); two waves a SIMD cover them with matrix instructions in part.
// Four users with 5 drafted tokens each take 125 us, 3.0 TB/s of the cache's bytes, where the copies alone take 63; vector
// instructions are issued in 53 % of the cycles, the matrix units work in 31. Other calls reach no unit's limit, but wait:
// 24 users of up to 6000 keys 38 us (33 % and 11, 2.6 TB/s), of which 12 are spent before the first and after the last tile and
// 5 on joining; 512 tokens of three prompts 77 us (36 % and 17), 21 of them for setting up and ending each workgroup's two or
// three blocks and 10 on joining.
// Blocks of 128 rows, whose four waves take a tile's numbers out of 4 bits once for all of them, took 78 us there, but 69 for a
// prompt of 300 tokens by itself, which takes 31 here, so that form is not kept.
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
constexpr int kSet = 16;      // query rows of an MFMA
constexpr int kIds = 1024;    // pages of chunks held in LDS at a time

// How tokens and heads are taken together: R rows of a block, which are all G query heads of a KV head (G <= R) for up to tq
// tokens; J blocks per run of tokens.
struct Shape {
  int G, tq, J;
};
__host__ __device__ inline Shape shape_of(int H, int KV, int R, int max_run) {
  const int G = H / KV, tq = R / G;
  return Shape{G, max_run < 1 ? 1 : max_run < tq ? max_run : tq, KV};
}

// A block of rows of one KV head, and how many keys its tokens see at most.
struct Block {
  int t0, m, keys;  // tokens t0 .. t0 + m - 1
  int seq, mine;    // their sequence; keys of token t0 + lane, lane < m
  int g, h0, per;   // KV head, first query head, heads per token
  int inv;          // 2^16 / per, rounded up
  __device__ __forceinline__ int rows() const { return m * per; }
  __device__ __forceinline__ int turn(int r) const { return r * inv >> 16; }  // r / per, for r < 2^8
  __device__ __forceinline__ int token(int r) const { return t0 + turn(r); }
  __device__ __forceinline__ int head(int r) const { return h0 + r - turn(r) * per; }
  __device__ __forceinline__ int tiles() const { return (keys + kTile - 1) / kTile; }
};
__device__ __forceinline__ void set_heads(Block& b, const Shape& S, int j) {
  b.g = j, b.h0 = j * S.G, b.per = S.G;
  b.inv = (65535 + b.per) / b.per;
}

// Both loads go at once.
__device__ __forceinline__ int keys_of(const Kv4Attn& A, int s, int k) {
  return s >= 0 && s < A.kv.n_seq ? max(0, min(k, A.max_keys)) : 0;
}
__device__ __forceinline__ int keys_of(const Kv4Attn& A, int t) {
  const int s = A.seq[t], k = A.n_keys[t];
  return keys_of(A, s, k);
}
__device__ __forceinline__ bool starts(const Kv4Attn& A, int t) { return t == 0 || A.seq[t] != A.seq[t - 1]; }
// The first token of the run of its sequence's that t is in, found by a wave.
__device__ __forceinline__ int run_start(const Kv4Attn& A, int t) {
  const int lane = threadIdx.x & 63;
  for (;; t -= 64) {
    const uint64_t at = __ballot(t - lane >= 0 && starts(A, t - lane));
    if (at) return t - __builtin_ctzll(at);
  }
}
// The block that token t leads: it and the tokens of its sequence that follow, tq at most, found by a wave.
__device__ __forceinline__ void set_tokens(Block& b, const Kv4Attn& A, int t, int tq) {
  const int lane = threadIdx.x & 63, i = min(t + lane, A.n - 1);
  const int s = A.seq[i], k = A.n_keys[i];
  b.seq = __builtin_amdgcn_readfirstlane(s);
  const uint64_t same = __ballot(lane < tq && t + lane < A.n && s == b.seq);
  b.t0 = t, b.m = __builtin_ctzll(~same);
  int keys = b.mine = lane < b.m ? keys_of(A, s, k) : 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) keys = max(keys, __shfl_xor(keys, o));
  b.keys = __builtin_amdgcn_readfirstlane(keys);
}

__device__ __forceinline__ void fence() { asm volatile("" ::: "memory"); }
__device__ __forceinline__ void wait_lds() {
  fence();
  __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
  fence();
}

// x as hi + lo, two at a time: the difference is taken from the halves as they lie.
__device__ __forceinline__ void split2(float a, float b, v2h& hi, v2h& lo) {
  hi = __builtin_convertvector((v2f{a, b}), v2h);
  uint32_t r;
  asm("v_fma_mixlo_f16 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]\n\t"
      "v_fma_mixhi_f16 %0, %1, -1.0, %3 op_sel:[1,0,0] op_sel_hi:[1,0,0]"
      : "=&v"(r)
      : "v"(__builtin_bit_cast(uint32_t, hi)), "v"(a), "v"(b));
  lo = __builtin_bit_cast(v2h, r);
}
__device__ __forceinline__ void split8(const float (&x)[8], v8h& hi, v8h& lo) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    v2h h, l;
    split2(x[i], x[i + 1], h, l);
    hi[i] = h[0], hi[i + 1] = h[1], lo[i] = l[0], lo[i + 1] = l[1];
  }
}

// Eight numbers of a word as n - 8, exactly, in the order 0, 4, 1, 5, 2, 6, 3, 7: a number under the exponent of 1024 reads
// 1024 + n in the lowest four bits of the fraction, under that of 64 reads 64 + n four bits further up. Masks and exponents are
// kept in registers, one scalar and one vector, which an and-or takes together (as literals each would be an instruction).
struct Unpack {
  uint32_t mask_a, mask_b, exp_a, exp_b;
  __device__ __forceinline__ Unpack() {
    asm("s_mov_b32 %0, 0x000F000F" : "=s"(mask_a));
    asm("s_mov_b32 %0, 0x00F000F0" : "=s"(mask_b));
    asm("v_mov_b32 %0, 0x64006400" : "=v"(exp_a));
    asm("v_mov_b32 %0, 0x54005400" : "=v"(exp_b));
  }
  __device__ __forceinline__ void less8(uint32_t w, v2h (&r)[4]) const {
    const v2h a = {(_Float16)1032.0f, (_Float16)1032.0f}, b = {(_Float16)72.0f, (_Float16)72.0f};
    r[0] = __builtin_bit_cast(v2h, (w & mask_a) | exp_a) - a;
    r[1] = __builtin_bit_cast(v2h, (w & mask_b) | exp_b) - b;
    w >>= 8;
    r[2] = __builtin_bit_cast(v2h, (w & mask_a) | exp_a) - a;
    r[3] = __builtin_bit_cast(v2h, (w & mask_b) | exp_b) - b;
  }
};
__device__ __forceinline__ v8h join8(const v2h (&r)[4]) {
  return v8h{r[0][0], r[0][1], r[1][0], r[1][1], r[2][0], r[2][1], r[3][0], r[3][1]};
}
// Place of the e-th of eight elements (or keys) in that order.
__device__ __forceinline__ constexpr int place(int e) { return (e & 1) * 4 + (e >> 1); }

template <int D, int NR, int NW>
struct Geo {
  static constexpr int kR = NR * kSet;             // rows of a block
  static constexpr int kSteps = D / 32;            // MFMAs over a row: lane qd of four holds its elements D / 4 qd + ..
  static constexpr int kDt = D / 16;               // 16-element tiles of a row
  static constexpr int kRow = D / 2, kGroups = D / 32;
  static constexpr int kBytes = kTile * kRow;      // of K or V
  static constexpr int kScales = kTile * kGroups * 2;
  static constexpr int kCopies = kBytes / 1024 + kScales / 256;
  static constexpr int kWave = 2 * (kBytes + kScales);
  static constexpr int kQ = kSteps * NR * 2 * 1024;  // q: [step][set][hi, lo][lane] 16 bytes
  static constexpr int kStride = 64 + 4;             // of a row of results, 64 elements at a time
  static constexpr int kOut = NW * kR * kStride * 4;
  static constexpr int kRing = NW * kWave > kOut ? NW * kWave : kOut;
  static constexpr int kLds = kQ + kRing;
};

// What a wave holds of its rows: this lane's of set n is row 16 n + lane % 16; o[i][j] is its element 16 i + 4 (lane / 16) + j.
template <int D, int NR>
struct Acc {
  v4f o[NR][D / 16];
  float m[NR], l[NR];  // weights are 2^(score - m), l this lane's sum of them
};

// Where a tile's four chunks lie: numbers of 16 rows among all rows of the pool (those without a page: 0).
struct Place {
  uint32_t at[4];
  int have;  // chunks that have a page
};
constexpr uint32_t kNoChunk = 0xFFFFFFFFu;

// One wave's copies and products. Everything here is the wave's own: no barrier.
template <int D, int NR, int NW>
struct Walk {
  using G_ = Geo<D, NR, NW>;
  const Kv4Attn& A;
  int lane, li, qd;
  const uint8_t* q_s;
  uint8_t *ks_s, *k_s, *v_s, *vs_s;
  uint32_t k_off, v_off, vs_off;  // this lane's part of a copy
  Unpack un;
  float rf[NR];           // score, in bits, of one unit of a product
  // Scores past 2^16 bits (a bit of `wide` per set): the shift's own rounding would count beside them. They are rounded to fp32
  // first (by rg; rf is 1 then).
  float rg[NR];
  int wide;
  int lim[NR], least;     // keys that this lane's rows see, and that every row of the block sees

  __device__ __forceinline__ Walk(const Kv4Attn& a, uint8_t* smem, int w) : A(a) {
    lane = threadIdx.x & 63, li = lane & 15, qd = lane >> 4, wide = 0;
    q_s = smem;
    vs_off = (((lane >> 3) & (G_::kGroups - 1)) << A.kv.shift) + 2 * (lane & 7);
    k_s = smem + G_::kQ + w * G_::kWave, v_s = k_s + G_::kBytes, ks_s = v_s + G_::kBytes, vs_s = ks_s + G_::kScales;
    if constexpr (D == 128) {
      k_off = li * 64 + 16 * qd;
      v_off = (lane >> 2) * 64 + 16 * ((lane & 3) ^ (lane >> 4));
    } else {
      k_off = (lane & 31) * 16;
      v_off = ((lane & 31) >> 1) * 32 + 16 * ((lane & 1) ^ ((lane >> 4) & 1));
    }
  }

  __device__ __forceinline__ Place find(const uint32_t* ids) const {
    const uint4 id = *reinterpret_cast<const uint4*>(ids);
    Place p;
    p.at[0] = __builtin_amdgcn_readfirstlane(id.x), p.at[1] = __builtin_amdgcn_readfirstlane(id.y);
    p.at[2] = __builtin_amdgcn_readfirstlane(id.z), p.at[3] = __builtin_amdgcn_readfirstlane(id.w);
    p.have = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const bool in = p.at[c] != kNoChunk;
      p.have |= in << c, p.at[c] = in ? p.at[c] : 0u;
    }
    return p;
  }
  // This lane's of two or of four chunks, for copies whose lanes have them side by side.
  __device__ __forceinline__ uint32_t of2(const Place& p, int c) const { return lane < 32 ? p.at[c] : p.at[c + 1]; }
  __device__ __forceinline__ uint32_t of4(const Place& p) const {
    const uint32_t a = lane & 16 ? p.at[1] : p.at[0], b = lane & 16 ? p.at[3] : p.at[2];
    return lane < 32 ? a : b;
  }
  __device__ __forceinline__ void issue_k(const Place& p) const {
    const uint8_t* ks = reinterpret_cast<const uint8_t*>(A.kv.ks);
    if constexpr (D == 128) {
#pragma unroll
      for (int c = 0; c < 4; ++c) lds_copy16(A.kv.k + (uint64_t)p.at[c] * 1024, k_off, k_s + 1024 * c);
#pragma unroll
      for (int c = 0; c < 4; c += 2) lds_copy4(ks + (uint64_t)of2(p, c) * 128 + 4 * (lane & 31), ks_s + 128 * c);
    } else {
#pragma unroll
      for (int c = 0; c < 4; c += 2) lds_copy16(A.kv.k + (uint64_t)of2(p, c) * 512 + k_off, k_s + 512 * c);
      lds_copy4(ks + (uint64_t)of4(p) * 64 + 4 * li, ks_s);
    }
  }
  // The scales of V in LDS: [chunk][group][key]. A page's are its groups' one after the other.
  __device__ __forceinline__ const uint16_t* scales_at(uint32_t chunk) const {
    const uint32_t in = chunk & ((1u << (A.kv.shift - 4)) - 1);
    return A.kv.vs + (uint64_t)(chunk - in) * (kChunk * G_::kGroups) + kChunk * in + vs_off;
  }
  __device__ __forceinline__ void issue_v(const Place& p) const {
    if constexpr (D == 128) {
#pragma unroll
      for (int c = 0; c < 4; ++c) lds_copy16(A.kv.v + (uint64_t)p.at[c] * 1024, v_off, v_s + 1024 * c);
#pragma unroll
      for (int c = 0; c < 4; c += 2) lds_copy4(scales_at(of2(p, c)), vs_s + 128 * c);
    } else {
#pragma unroll
      for (int c = 0; c < 4; c += 2) lds_copy16(A.kv.v + (uint64_t)of2(p, c) * 512 + v_off, v_s + 512 * c);
      lds_copy4(scales_at(of4(p)), vs_s);
    }
  }

  // One tile: keys key .. key + 63, of which those below `end` count (end <= the block's keys) and whose chunk has a page.
  // more: `next` is the wave's next tile, whose copies are asked for.
  __device__ __forceinline__ void tile(Acc<D, NR>& acc, bool& fresh, int have, int key, int end, bool more, const Place& next) {
    wait_vm<G_::kCopies>();  // this tile's K; its V may be under way
    fence();
    const bool whole = key + kTile <= min(least, end) && have == 15;
    v4f s[NR][4];
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
      if (more) issue_k(next);
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[n][c] = v4f{};
#pragma unroll
      for (int i = 0; i < G_::kSteps; ++i) {
        v8h hi[NR], lo[NR];
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          const v8h* from = reinterpret_cast<const v8h*>(q_s) + (i * NR + n) * 128 + lane;
          hi[n] = from[0], lo[n] = from[64];
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          v2h r[4];
          un.less8(w[c][i], r);
          const v2h f = {sc[c], sc[c]};
#pragma unroll
          for (int j = 0; j < 4; ++j) r[j] *= f;
          const v8h a = join8(r);
#pragma unroll
          for (int n = 0; n < NR; ++n) s[n][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, hi[n], s[n][c], 0, 0, 0);
#pragma unroll
          for (int n = 0; n < NR; ++n) s[n][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, lo[n], s[n][c], 0, 0, 0);
        }
      }
    }
    // Register i of chunk c is key 16 c + 4 qd + i.
    v8h ph[NR][2], pl[NR][2];
    const bool first = fresh;
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      if (wide >> n & 1)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[n][c] *= rg[n];
      if (!whole)
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int k = key + kChunk * c + 4 * qd + i;
            s[n][c][i] = k < min(lim[n], end) && (have >> c & 1) ? s[n][c][i] : -INFINITY;
          }
      float p[16], sum;
      auto weights = [&] __attribute__((always_inline)) {
        sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          p[i] = __builtin_amdgcn_exp2f(fma_(s[n][i / 4][i % 4], rf[n], -acc.m[n]));
          sum += p[i];
        }
      };
      if (!first) weights();
      // The first tile, and one whose weights may leave fp16: a new shift, 10 below the largest score (that score itself where
      // 10 is not exact beside it).
      if (first || __ballot(sum > 32768.0f)) {
        auto largest = [&] __attribute__((always_inline)) {
          float z = -INFINITY;
#pragma unroll
          for (int i = 0; i < 16; ++i) z = fmaxf(z, s[n][i / 4][i % 4] * rf[n]);
          z = fmaxf(z, __shfl_xor(z, 16));
          return fmaxf(z, __shfl_xor(z, 32));
        };
        float z = largest();
        if (!(wide >> n & 1) && __ballot(fabsf(z) > 65536.0f && z > -INFINITY)) {
          wide |= 1 << n, rg[n] = rf[n], rf[n] = 1.0f;
#pragma unroll
          for (int c = 0; c < 4; ++c) s[n][c] *= rg[n];
          z = largest();
        }
        const float m = fmaxf(acc.m[n], fabsf(z) < 0x1p24f ? z - 10.0f : z);
        const float f = __builtin_amdgcn_exp2f(acc.m[n] - m);
        acc.m[n] = m, acc.l[n] *= f;
        if (!first) {
#pragma unroll
          for (int i = 0; i < G_::kDt; ++i) acc.o[n][i] *= f;
        }
        weights();
      }
      acc.l[n] += sum;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = p[8 * u + e];
        split8(y, ph[n][u], pl[n][u]);
      }
    }
    fresh = false;
    if (more) wait_vm<G_::kCopies>();  // this tile's V; the next one's K may be under way
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
    if (more) issue_v(next);
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
        un.less8((uint32_t)vv[i][u], r);
        const v4h a = sc[i / 2][2 * u], b = sc[i / 2][2 * u + 1];
        r[0] *= v2h{a[0], a[1]}, r[1] *= v2h{a[2], a[3]}, r[2] *= v2h{b[0], b[1]}, r[3] *= v2h{b[2], b[3]};
        const v8h x = join8(r);
#pragma unroll
        for (int n = 0; n < NR; ++n) acc.o[n][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, ph[n][u], acc.o[n][i], 0, 0, 0);
#pragma unroll
        for (int n = 0; n < NR; ++n) acc.o[n][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, pl[n][u], acc.o[n][i], 0, 0, 0);
      }
  }
};

template <int NR, int NW>
struct Shared {  // beside the dynamic part
  uint32_t ids[kIds];  // chunks' places
  v2f ml[NW][NR * kSet];  // and, before, the largest values of q's rows: NW >= 4 / NR, 4 steps at most
};

// Tiles [ta, tb) of a block by the workgroup's NW waves; then put(row, element, its next four as weighted sums, l, m) by the 16
// threads that share a row, 64 elements at a time. Ends with every thread's own reads of LDS: a barrier comes before it is
// written again.
template <int D, int NR, int NW, class Put>
__device__ __forceinline__ void run_block(const Kv4Attn& A, const Block& b, int ta, int tb, const float* q, int64_t q_stride,
                                          uint8_t* smem, Shared<NR, NW>& sh, Put put) {
  using G_ = Geo<D, NR, NW>;
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int end = min(b.keys, tb * kTile), seq = b.seq;
  Walk<D, NR, NW> walk(A, smem, w);
  const int li = walk.li, qd = walk.qd, lane = walk.lane;
  // q: waves take (step, set) pairs in turn; a row's largest value is the waves' together.
  constexpr int kPairs = G_::kSteps * NR, kMine = (kPairs + NW - 1) / NW;
  float x[kMine][8];
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int at = min(w + NW * i, kPairs - 1), s = at / NR, r = min(at % NR * kSet + li, b.rows() - 1);
    const float* qr = q + b.token(r) * q_stride + (int64_t)b.head(r) * D + D / 4 * qd + 8 * s;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const v4f f = *reinterpret_cast<const v4a*>(qr + 4 * c);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[i][4 * c + e] = f[e];
    }
  }
  // Rows beyond the block's are copies of the last one, whose results nobody reads.
  walk.least = INT32_MAX;
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    walk.lim[n] = __shfl(b.mine, b.turn(min(n * kSet + li, b.rows() - 1)));
    walk.least = min(walk.least, walk.lim[n]);
  }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) walk.least = min(walk.least, __shfl_xor(walk.least, o));
  walk.least = __builtin_amdgcn_readfirstlane(walk.least);
  auto load_ids = [&](int t0, int t1) {
    for (int i = tid; i < 4 * (t1 - t0); i += NW * 64) {
      const int key = t0 * kTile + kChunk * i;
      const int p = key < end ? A.kv.page_of(seq, key) : -1;
      sh.ids[i] = p < 0 ? kNoChunk : (uint32_t)((A.kv.first_row(p, b.g) + (key & ((1 << A.kv.shift) - 1))) >> 4);
    }
  };
  __syncthreads();  // LDS is free
  load_ids(ta, min(tb, ta + kIds / 4));
  float* top_s = reinterpret_cast<float*>(sh.ml);  // [step][row]
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int at = w + NW * i;
    float top = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[i][e]));
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    if (at < kPairs && qd == 0) top_s[at / NR * G_::kR + at % NR * kSet + li] = top;
  }
  __syncthreads();
  // The first tile's copies go while q is made ready.
  auto find = [&](int t, int t0) { return walk.find(sh.ids + 4 * (t - t0)); };
  Place at{};
  if (ta + w < tb) {
    at = find(ta + w, ta);
    walk.issue_k(at), walk.issue_v(at);
  }
  int ex[NR];
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    float top = 0.0f;
#pragma unroll
    for (int s = 0; s < G_::kSteps; ++s) top = fmaxf(top, top_s[s * G_::kR + n * kSet + li]);
    ex[n] = top > 0.0f && top < INFINITY ? min(14 - __builtin_amdgcn_frexp_expf(top), 100) : 0;
    walk.rf[n] = __builtin_ldexpf(A.scale * kLog2e, -ex[n]);
  }
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int at = w + NW * i;
    if (at >= kPairs) continue;
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = __builtin_ldexpf(x[i][place(e)], ex[at % NR]);
    v8h hi, lo;
    split8(y, hi, lo);
    v8h* to = reinterpret_cast<v8h*>(smem) + at * 128 + lane;
    to[0] = hi, to[64] = lo;
  }
  __syncthreads();
  Acc<D, NR> acc;
#pragma unroll
  for (int n = 0; n < NR; ++n) {
#pragma unroll
    for (int i = 0; i < G_::kDt; ++i) acc.o[n][i] = v4f{};
    acc.m[n] = kNone, acc.l[n] = 0.0f;
  }
  bool fresh = true;
  for (int t0 = ta; t0 < tb; t0 += kIds / 4) {  // pages of as many tiles as LDS holds
    const int t1 = min(tb, t0 + kIds / 4);
    if (t0 > ta) {
      __syncthreads();
      load_ids(t0, t1);
      __syncthreads();
    }
    int t = t0 + w;
    if (t >= t1) continue;
    if (t0 > ta) {
      at = find(t, t0);
      walk.issue_k(at), walk.issue_v(at);
    }
    for (;;) {
      const bool more = t + NW < t1;
      const int have = at.have;
      if (more) at = find(t + NW, t0);
      walk.tile(acc, fresh, have, t * kTile, end, more, at);
      if (!more) break;
      t += NW;
    }
  }
  // The waves' parts of each row, brought to their largest shift and added.
  float* ob = reinterpret_cast<float*>(smem + G_::kQ);
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    float l = acc.l[n] + __shfl_xor(acc.l[n], 16);
    l += __shfl_xor(l, 32);
    if (qd == 0) sh.ml[w][n * kSet + li] = v2f{acc.m[n], l};
  }
#pragma unroll
  for (int d0 = 0; d0 < D; d0 += 64) {
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<v4f*>(ob + (w * G_::kR + n * kSet + li) * G_::kStride + 16 * i + 4 * qd) = acc.o[n][d0 / 16 + i];
    __syncthreads();
#pragma unroll 1
    for (int r = tid >> 4; r < b.rows(); r += NW * 4) {
      float f[NW], top = kNone, sum = 0.0f;
#pragma unroll
      for (int i = 0; i < NW; ++i) top = fmaxf(top, sh.ml[i][r][0]);
#pragma unroll
      for (int i = 0; i < NW; ++i) {
        f[i] = __builtin_amdgcn_exp2f(sh.ml[i][r][0] - top);
        sum = fma_(f[i], sh.ml[i][r][1], sum);
      }
      v4f a = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < NW; ++i) a += f[i] * *reinterpret_cast<const v4f*>(ob + (i * G_::kR + r) * G_::kStride + 4 * (tid & 15));
      put(r, d0 + 4 * (tid & 15), a, sum, top);
    }
  }
}

// Four values of a row of the output, by the threads of a row together.
struct Out {
  float* out;
  int64_t stride;
  BlockQ8* xq;
};
template <int D>
__device__ __forceinline__ void put_row(const Kv4Attn& A, const Out& O, int t, int head, int d, v4f a, float l) {
  const float n = l == 0.0f ? 1.0f : 1.0f / l;  // no key: zeros
  const float y[4] = {a[0] * n, a[1] * n, a[2] * n, a[3] * n};
  *reinterpret_cast<v4a*>(O.out + t * O.stride + (int64_t)head * D + d) = v4a{y[0], y[1], y[2], y[3]};
  if (O.xq) quantize_block_lanes_n<4>(y, (d & 31) / 4, O.xq + (((int64_t)t * A.H + head) * D + d) / 32);
}

// A workgroup per token and J; the first token of its sequence, or of tq tokens, leads a block and the others' workgroups leave.
template <int D, int NR, int NW>
__global__ __launch_bounds__(NW * 64) void k_kv4_whole(Kv4Attn A, const float* __restrict__ q, int64_t q_stride, Out O) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ __align__(16) Shared<NR, NW> sh;
  const Shape S = shape_of(A.H, A.kv.KV, NR * kSet, A.max_run);
  const int t = blockIdx.x / S.J;
  if (S.tq > 1 && (t - run_start(A, t)) % S.tq) return;
  Block b;
  set_tokens(b, A, t, S.tq);
  set_heads(b, S, blockIdx.x % S.J);
  run_block<D, NR, NW>(A, b, 0, b.tiles(), q, q_stride, smem, sh,
                       [&](int r, int d, v4f a, float l, float m) { put_row<D>(A, O, b.token(r), b.head(r), d, a, l); });
}

// ---- even shares of all tiles ----

constexpr int kShare = 4;  // waves of a workgroup that takes a share
// Tiles of a share. One user, 8000 keys: 18.5 us, with 2 23, with 8 20.2; 4 x 5 drafts, 3000 keys: 26.7, 29.4 and 28.7.
constexpr int kLeast = 4;

// Per (token, j): the workgroups whose runs hold its block, first (where it begins) and last (-1: written whole), and the row
// that the token's first head has in it.
struct Record {
  int first, last, row;
};
// Partial results of workgroup w: slot 2 w of a block that began before its run, 2 w + 1 of one that begins in it and ends after.
struct Parts {
  float* o;    // [slot][row][D]
  v2f* ml;     // [slot][row] shift and sum
  Record* rec; // [token][J]
};

// Exclusive running sum (and total) over 256 threads, or the largest before; part: 4 words of LDS.
template <bool MAX, typename T>
__device__ __forceinline__ T scan256(T v, T* part, T& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const T none = MAX ? (T)-1 : (T)0;
  auto op = [](T a, T b) { return MAX ? (a > b ? a : b) : a + b; };
  T x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const T y = __shfl_up(x, o);
    if (lane >= o) x = op(x, y);
  }
  T before = __shfl_up(x, 1);
  if (lane == 0) before = none;
  __syncthreads();
  if (lane == 63) part[w] = x;
  __syncthreads();
  total = none;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i < w) before = op(before, part[i]);
    total = op(total, part[i]);
  }
  return before;
}

// Tokens that a thread looks at together where there are more than 256 (a 512-token prompt, 2600 keys: 72 us, one at a time 76;
// 120 drafted tokens: 46, four at a time 49).
template <int NR>
constexpr int kTokens = NR == 1 ? 1 : 4;

template <int D, int NR>
__global__ __launch_bounds__(kShare * 64, 2) void k_kv4_share(Kv4Attn A, const float* __restrict__ q, int64_t q_stride,
                                                                            Out O, Parts P) {
  constexpr int R = NR * kSet, kTok = kTokens<NR>, kOnce = 256 * kTok;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ __align__(16) Shared<NR, kShare> sh;
  __shared__ int part[4], start_t;
  __shared__ int64_t start_off;
  const int tid = threadIdx.x, w = blockIdx.x;
  const Shape S = shape_of(A.H, A.kv.KV, R, A.max_run);
  // kOnce tokens at a time, kTok to a thread (one, where there are few): the tiles of the blocks that they lead, and the running
  // sum of those.
  static_assert(2 * 4 * (kOnce + R) <= Geo<D, NR, kShare>::kLds);
  int *tok_seq = reinterpret_cast<int*>(smem), *tok_keys = tok_seq + kOnce + R;
  const int per = A.n > 256 ? kTok : 1;
  int run = 0, tiles[kTok], before = 0, all = 0;
  auto look = [&](int c0) {
    const int prior = A.seq[max(c0 - 1, 0)];
    __syncthreads();
    for (int i = tid; i < 256 * per + R; i += 256) {
      const int t = c0 + i, s = A.seq[min(t, A.n - 1)], k = A.n_keys[min(t, A.n - 1)];
      tok_seq[i] = s, tok_keys[i] = t < A.n ? keys_of(A, s, k) : 0;
    }
    __syncthreads();
    auto begins = [&](int i) { return c0 + i == 0 || (c0 + i < A.n && tok_seq[i] != (i ? tok_seq[i - 1] : prior)); };
    int from = -1, last;
#pragma unroll
    for (int e = 0; e < kTok; ++e)
      if (e < per && begins(per * tid + e)) from = c0 + per * tid + e;
    from = scan256<true>(from, part, last);  // the last run's first token before this thread's; of an earlier kOnce: none
    if (from < 0) from = run;
    int sum = 0;
#pragma unroll
    for (int e = 0; e < kTok; ++e) {
      const int i = per * tid + e, t = c0 + i;
      tiles[e] = 0;
      if (e >= per) continue;
      if (begins(i)) from = t;
      if (t < A.n && (t - from) % S.tq == 0) {
        int keys = tok_keys[i];
        for (int m = 1; m < S.tq && t + m < A.n && tok_seq[i + m] == tok_seq[i]; ++m) keys = max(keys, tok_keys[i + m]);
        tiles[e] = (keys + kTile - 1) / kTile;
      }
      sum += tiles[e];
    }
    before = scan256<false>(sum, part, all);
    if (last >= 0) run = last;
  };
  int64_t total = 0;
  for (int c0 = 0; c0 < A.n; c0 += kOnce) look(c0), total += all;
  // No share is smaller than kLeast tiles, or than a block where those are small on average (a prompt of 300 tokens: 31 us, with
  // kLeast 44: two blocks a workgroup instead of one).
  const int least = (int)max<int64_t>(1, min<int64_t>(total * S.tq / A.n, kLeast));
  const int64_t share = max<int64_t>((total * S.J + gridDim.x - 1) / gridDim.x, least), a = w * share, b = min(a + share, total * S.J);
  if (a >= b) return;
  // The block that holds tile a is one of exactly one thread's.
  run = 0, total = 0;
  bool found = false;
  for (int c0 = 0; c0 < A.n && !found; c0 += kOnce) {
    if (A.n > kOnce) look(c0);
    int64_t off = (total + before) * S.J;
#pragma unroll
    for (int e = 0; e < kTok; ++e) {
      if (off <= a && a < off + (int64_t)tiles[e] * S.J) start_t = c0 + per * tid + e, start_off = off;
      off += (int64_t)tiles[e] * S.J;
    }
    total += all;
    found = a < total * S.J;
  }
  if (!found) return;  // lengths that changed in between, which no caller may do: every loop ends all the same
  __syncthreads();
  // Blocks follow each other by (token, j); tile a is tile k0 of block j of those that token t leads.
  int t = start_t;
  Block blk;
  set_tokens(blk, A, t, S.tq);
  int j = (int)((a - start_off) / blk.tiles()), k0 = (int)((a - start_off) % blk.tiles());
  for (int64_t at = a; at < b;) {
    const int tiles = blk.tiles();
    if (j == S.J || tiles == 0) {  // the next tokens'
      t += blk.m, j = 0;
      if (t >= A.n) return;  // as above
      set_tokens(blk, A, t, S.tq);
      continue;
    }
    const int k1 = (int)min<int64_t>(tiles, k0 + (b - at));
    set_heads(blk, S, j);
    // A block that begins here and ends before the next workgroup's run is written whole.
    const bool begins = k0 == 0, whole = begins && at + tiles <= a + share;
    if (begins) {
      const int end = whole ? -1 : (int)((at + tiles - 1) / share);
      for (int i = tid; i < blk.m; i += kShare * 64) P.rec[(int64_t)(t + i) * S.J + j] = Record{w, end, i * blk.per};
    }
    const int64_t slot = 2 * (int64_t)w + begins;
    run_block<D, NR, kShare>(A, blk, k0, k1, q, q_stride, smem, sh, [&](int r, int d, v4f v, float l, float m) {
      if (whole) {
        put_row<D>(A, O, blk.token(r), blk.head(r), d, v, l);
      } else {
        *reinterpret_cast<v4f*>(P.o + (slot * R + r) * D + d) = v;
        if (d == 0) P.ml[slot * R + r] = v2f{m, l};
      }
    });
    at += k1 - k0;
    ++j, k0 = 0;
  }
}

// W waves per query row: the parts of rows that several workgroups had, added; zeros for rows without keys. Wave w of a row takes
// every W-th part, and asks for kAhead of them before their weights are known.
template <int D, int R, int W>
__global__ __launch_bounds__(256) void k_kv4_join(Kv4Attn A, Out O, Parts P) {
  constexpr int E = D / 64, kAhead = 8;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, w = wave % W;
  const int64_t row = (int64_t)blockIdx.x * (4 / W) + wave / W;
  if (row >= (int64_t)A.n * A.H) return;
  const Shape S = shape_of(A.H, A.kv.KV, R, A.max_run);
  const int t = (int)(row / A.H), head = (int)(row % A.H);
  const Record rec = P.rec[(int64_t)t * S.J + head / S.G];  // what it says counts where there are keys
  const bool any = keys_of(A, t) > 0;
  if (any && rec.last < 0) return;
  float v[E], sum = 0.0f;
#pragma unroll
  for (int k = 0; k < E; ++k) v[k] = 0.0f;
  if (any) {
    const int r = rec.row + head % S.G, parts = rec.last - rec.first + 1;
    auto slot = [&](int i) { return (2 * ((int64_t)rec.first + i) + (i == 0)) * R + r; };
    auto read = [&](int i0, float (&x)[kAhead][E]) {
#pragma unroll
      for (int e = 0; e < kAhead; ++e)
        if (i0 + W * e < parts)
#pragma unroll
          for (int k = 0; k < E; ++k) x[e][k] = P.o[slot(i0 + W * e) * D + E * lane + k];
    };
    float x[kAhead][E];
    read(w, x);
    v2f ml = lane < parts ? P.ml[slot(lane)] : v2f{kNone, 0.0f};
    float top = ml[0];
    for (int i = 64 + lane; i < parts; i += 64) top = fmaxf(top, P.ml[slot(i)][0]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    for (int i0 = 0; i0 < parts; i0 += 64) {
      if (i0) ml = i0 + lane < parts ? P.ml[slot(i0 + lane)] : v2f{kNone, 0.0f};
      const float f = __builtin_amdgcn_exp2f(ml[0] - top);
      sum = fma_(f, ml[1], sum);
      const int m = min(64, parts - i0);
      for (int i = w; i < m; i += W * kAhead) {
        if (i0 + i != w) read(i0 + i, x);
#pragma unroll
        for (int e = 0; e < kAhead; ++e)
          if (i + W * e < m) {
            const float fe = __shfl(f, i + W * e);
#pragma unroll
            for (int k = 0; k < E; ++k) v[k] = fma_(fe, x[e][k], v[k]);
          }
      }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
  }
  if constexpr (W > 1) {
    __shared__ float part[W - 1][D];
    static_assert(W == 4, "one row per workgroup");
    if (w)
#pragma unroll
      for (int k = 0; k < E; ++k) part[w - 1][E * lane + k] = v[k];
    __syncthreads();
    if (w) return;
#pragma unroll
    for (int i = 0; i < W - 1; ++i)
#pragma unroll
      for (int k = 0; k < E; ++k) v[k] += part[i][E * lane + k];
  }
  const float n = sum == 0.0f ? 1.0f : sum;
#pragma unroll
  for (int k = 0; k < E; ++k) v[k] = v[k] / n;
  float* to = O.out + t * O.stride + (int64_t)head * D + E * lane;
#pragma unroll
  for (int k = 0; k < E; ++k) to[k] = v[k];
  if (O.xq) quantize_block_lanes_n<E>(v, lane % (32 / E), O.xq + (row * D + E * lane) / 32);
}

// How a call is cut.
struct Cut {
  int sets;   // 16-row sets of a block
  int wgs;    // workgroups that share all tiles; 0: one per block
  int waves;  // of a workgroup that has a block to itself
};
// A workgroup of eight waves per block up to kWholeKeys keys, with kMany workgroups one of four waves: tokens that lead no block
// have workgroups too, which leave at once but need their place on a CU before (16 x 4 drafts over 200 keys 10 us, with eight
// waves 15.7; over 900 keys, 24 x 5, 21 and 18.7). 32 query heads on 8: 8 users, 1000 keys 12.5 us, in shares 18.8 (four waves
// 14.6); one user, 2000 keys 18.9, in shares 13.7; 64 users, 1000 keys 22, in shares 33 (eight waves 25.8).
// Up to kWholeKeysMany keys where kMany blocks have work. 64 users of 600 to 3000 keys 47 us, in shares 54; all of 3000 57 and
// 58.5; one of 3000 among such of 375 32 and 26.5, but up to 2000 keys as long (23.8), and with 128 users 33 and 36; of 800 to
// 4000 keys 60 and 61.5, one of 4000 among short ones 40.5 and 28.5. Fewer blocks: 16 x 4 drafts over 3000 keys 45.7 and 28.5,
// 8 x 8 41.2 and 30.4, over 1500 keys 25.1 and 26.7.
constexpr int kWholeKeys = 1024, kWholeKeysMany = 3200, kMany = 512;
// Workgroups that share all tiles: two a CU, which leaves a wave 256 registers. Three of 168 took 41.6 us where two take 39.5 (24
// users of up to 6000 keys), 49 where 42.6 (one user of 100000), and as long for 64 users of 4000.
constexpr int kShares = 2 * 256;
// Up to so many rows are joined by four waves each: 4 x 5 drafts over 120000 keys 6 us, by one 13; 16384 rows of a prompt 10,
// by four 24.
constexpr int kJoinRows = 2048;

Cut cut_of(int n, int H, int KV, int max_keys, int max_run) {
  const int64_t rows = std::min<int64_t>(std::max(max_run, 1), n) * (H / KV);
  Cut c{rows > kSet ? 2 : 1, 0, 8};
  const Shape S = shape_of(H, KV, c.sets * kSet, max_run);
  const int64_t wgs = (int64_t)n * S.J, blocks = (int64_t)((n + S.tq - 1) / S.tq) * S.J;  // launched, and with work
  if (wgs >= kMany) c.waves = 4;
  if (rows <= 2 * kSet && max_keys <= (blocks >= kMany ? kWholeKeysMany : kWholeKeys)) return c;
  c.wgs = kShares;
  return c;
}

template <int D>
size_t parts_bytes(const Cut& c, int n, int H, int KV) {
  const size_t rows = 2ull * c.wgs * c.sets * kSet;
  return rows * (D * sizeof(float) + sizeof(v2f)) + (size_t)n * KV * sizeof(Record);
}

}  // namespace

// Never less for a larger call: the larger of both kinds of blocks, the records those of the smaller ones, also where this call
// has no parts and a larger one may.
size_t attention_kv4_workspace(int n, int H, int KV, int D, int max_keys, int max_run) {
  const Cut one{1, kShares, 0}, two{2, kShares, 0};
  return std::max(D == 128 ? parts_bytes<128>(one, n, H, KV) : parts_bytes<64>(one, n, H, KV),
                  D == 128 ? parts_bytes<128>(two, n, H, KV) : parts_bytes<64>(two, n, H, KV));
}

size_t attention_kv4_need(const Kv4Attn& A, int D) {
  const Cut c = cut_of(A.n, A.H, A.kv.KV, A.max_keys, A.max_run);
  return c.wgs == 0 ? 0 : D == 128 ? parts_bytes<128>(c, A.n, A.H, A.kv.KV) : parts_bytes<64>(c, A.n, A.H, A.kv.KV);
}

void attention_kv4(hipStream_t s, const Kv4Attn& A, int D, const float* q, int64_t q_stride, float* out, int64_t out_stride,
                   BlockQ8* xq, void* workspace) {
  const Cut c = cut_of(A.n, A.H, A.kv.KV, A.max_keys, A.max_run);
  const Out O{out, out_stride, xq};
  auto go = [&]<int D_, int NR>() {
    const Shape S = shape_of(A.H, A.kv.KV, NR * kSet, A.max_run);
    auto whole = [&]<int NW>() {
      constexpr auto lds = Geo<D_, NR, NW>::kLds;
      allow_lds<k_kv4_whole<D_, NR, NW>>(lds);
      hipLaunchKernelGGL((k_kv4_whole<D_, NR, NW>), dim3((unsigned)((int64_t)A.n * S.J)), dim3(NW * 64), lds, s, A, q, q_stride, O);
      check_launch("attention_kv4 whole");
    };
    if (c.wgs == 0) return c.waves == 8 ? whole.template operator()<8>() : whole.template operator()<4>();
    constexpr int R = NR * kSet, lds = Geo<D_, NR, kShare>::kLds;
    Parts P;
    P.o = static_cast<float*>(workspace);
    P.ml = reinterpret_cast<v2f*>(P.o + 2ull * c.wgs * R * D_);
    P.rec = reinterpret_cast<Record*>(P.ml + 2ull * c.wgs * R);
    allow_lds<k_kv4_share<D_, NR>>(lds);
    hipLaunchKernelGGL((k_kv4_share<D_, NR>), dim3((unsigned)c.wgs), dim3(kShare * 64), lds, s, A, q, q_stride, O, P);
    check_launch("attention_kv4 shares");
    const int64_t rows = (int64_t)A.n * A.H;
    if (rows <= kJoinRows) hipLaunchKernelGGL((k_kv4_join<D_, R, 4>), dim3((unsigned)rows), dim3(256), 0, s, A, O, P);
    else hipLaunchKernelGGL((k_kv4_join<D_, R, 1>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, A, O, P);
    check_launch("attention_kv4 join");
  };
  if (D == 128) c.sets == 1 ? go.template operator()<128, 1>() : go.template operator()<128, 2>();
  else c.sets == 1 ? go.template operator()<64, 1>() : go.template operator()<64, 2>();
}

}  // namespace mk
