// Attention of a batch whose sequences share a prefix: key j < n_prefix of every token is row j of one sequence of the
// prefix's cache, the others rows of the token's own sequence. out = sum_j p_j vs_j v_j, p = softmax(scale ks_j q.k_j).
//
// Rows and keys. A query row is a (token, query head); the rows of one KV head read the same prefix, so a workgroup takes
// 32 of them (all tokens' heads in turn) over one chunk of the prefix's keys. A sequence's own keys are read by its own
// tokens only: there a workgroup takes the rows of up to 32 / G neighbouring tokens of one sequence over one chunk of its
// own rows. Both kinds are one launch (k_prefix_parts); each leaves a partial output with its softmax statistics, which
// k_prefix_join adds.
//
// Arithmetic. An int8 key or value is exact in fp16, so the products run on v_mfma_f32_32x32x16_f16 with the fp32 side
// split into two fp16 parts, hi = fp16(x) and lo = fp16(x - hi): the products keep 2^-23 of x at a quarter of the fp32
// matrix instructions' time. A row of q is first brought to a largest value of 2^13 .. 2^14 by a power of two. The
// softmax weights are shifted so that the largest p vs is about 2^6: a weight's lo part then lies within fp16 down to
// 2^-17 of the largest, and what fp16 cannot hold of smaller ones is below 2^-30 of it. Scores, statistics and outputs
// are fp32.
//
// S = K Q^T has the keys in its rows and the query rows in its columns: a lane's 16 scores belong to one query row, the
// statistics are one register, and the weights are, as they lie, the second operand of O^T = V^T P^T. V^T comes from the
// transposing LDS read. Each of a workgroup's four waves takes every fourth 32-key tile through a K and a V buffer of its
// own, which direct copies fill: a buffer's next tile is asked for as soon as this one is in registers, and no barrier
// stands between the preparation of q and the addition of the waves' results. q's fp16 parts lie in LDS, read beside
// each MFMA: that leaves registers for three waves per SIMD (when it was chosen, 62 users over 8192 + 1024 keys took 48 us a
// pass, and with q in registers, two waves and a second K and V buffer 56).
//
// What bounds it. A 32 x 32 tile of head_dim 128 takes 32 MFMAs (32 cycles each) and about 330 vector instructions (160
// of them make fp16 of int8, 48 split the weights, 90 are the softmax), which overlap with MFMAs of other waves in part: 62
// users x 32 heads over 8192 + 1024 keys 45 us, 2.2 TB/s and 600 TFLOP/s of matrix instructions, the vector units issuing in
// 61 % of the cycles, the matrix units at work in 36 %, both in 21 %; 512 prompt tokens behind 2048 61 us, 620 TFLOP/s, 66,
// 38 and 23 % (on another card 44 and 57 us); the join 4 .. 9 us. A few tokens behind a few hundred keys take 7 us and 3.6 us
// to join, which is the latency of the launches and of the loads that wait for each other.
#include "ctx.h"
#include "ops.h"

namespace mk {
namespace {

typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef int v2i __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v2i lds_v2i;

constexpr int kThreads = 256, kWaves = 4;
constexpr int kRows = 32;        // query rows per workgroup
constexpr int kKeys = 32;        // keys per tile
constexpr float kNone = -3e38f;      // shift of a row that has seen no key
constexpr float kLeast = 0x1p-100f;  // value scales below this count as this for the shift, so that sums of 2^-m stay finite
constexpr float kLog2e = 1.44269504088896341f;

// Chunks of the prefix's and of the own keys; a part's index is its prefix chunk, or np + its own chunk.
struct Split {
  int np, cp, no, co;
  int tiles;      // row tiles of a KV head over the prefix
  int64_t parts;  // rows of partial outputs
};

// Statistics of a row's part: its weights are 2^(score - base - m), l their sum. base is 0 but for rows of very large
// scores; no key: kNone, kNone, 0.
struct __align__(16) Sum {
  float base, m, l, pad;
  // The shift relative to another base, the largest of the parts'.
  __device__ __forceinline__ float above(float b) const { return (base - b) + m; }
};

template <int D>
struct Geo {
  static constexpr int kSteps = D / 16;        // MFMAs' k steps over a row
  static constexpr int kDt = D / 32;           // 32-value tiles of a row
  static constexpr int kPieces = D / 16;       // 16-byte pieces of a row
  static constexpr int kTileBytes = kKeys * D;
  static constexpr int kCopies = kTileBytes / 1024;
  static constexpr int kShift = D == 128 ? 1 : 2;          // rows per 64 LDS banks, as a shift
  static constexpr int kQSteps = kSteps / kWaves;          // steps of q that a wave prepares
  static constexpr int kQBytes = kSteps * 2 * 1024;        // q: [step][hi, lo][lane] 16 bytes
  static constexpr int kWaveBytes = 2 * kTileBytes + 2 * 8 * kKeys;  // K, V, two tiles' scales
  static constexpr int kOutStride = 64 + 4;                // 64 values of a row at a time
  static constexpr int kOutBytes = kWaves * kRows * kOutStride * 4;
  static constexpr int kRing = kWaves * kWaveBytes > kOutBytes ? kWaves * kWaveBytes : kOutBytes;
  static constexpr int kLds = kQBytes + kRing;
};

// The piece of row `key` that lies in slot s, and the slot that holds piece s: rows whose LDS banks coincide hold their
// pieces in different slots.
template <int D>
__device__ __forceinline__ int swizzle(int key, int s) {
  return s ^ ((key >> Geo<D>::kShift) & (Geo<D>::kPieces - 1));
}

// Eight int8 as fp16, exactly: the byte x + 128 under the exponent of 1024 reads 1024 + 128 + x.
__device__ __forceinline__ v8h cvt8(uint32_t a, uint32_t b) {
  const v2h off = {(_Float16)1152.0f, (_Float16)1152.0f};
  a ^= 0x80808080u, b ^= 0x80808080u;
  v2h r[4];
  r[0] = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, a, 0x04010400u)) - off;
  r[1] = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u)) - off;
  r[2] = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u)) - off;
  r[3] = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u)) - off;
  return v8h{r[0][0], r[0][1], r[1][0], r[1][1], r[2][0], r[2][1], r[3][0], r[3][1]};
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

__device__ __forceinline__ void fence() { asm volatile("" ::: "memory"); }

template <int D>
__global__ __launch_bounds__(kThreads, 3) void k_prefix_parts(PrefixAttn A, Split S, const float* __restrict__ q,
                                                              int64_t q_stride, float* __restrict__ po, Sum* __restrict__ pml) {
  using G_ = Geo<D>;
  const int G = A.H / A.KV, tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int li = lane & 31, h = lane >> 5;
  const int n_pre = S.tiles * A.KV * S.np;
  // Which rows, keys and cache: row r (0 .. rows - 1) is token t0 + r / G + .., see `token` and `head` below.
  int part, g, first, rows, seq = 0, k0, k1;  // first: the first row among the KV head's rows t * G + i
  const int8_t *kb, *vb;
  const float *ksb, *vsb;
  if ((int)blockIdx.x < n_pre) {
    // Each XCD a contiguous run: the row tiles of one (KV head, chunk) read its keys into one L2.
    const int it = xcd_run((int)blockIdx.x, n_pre), pair = it / S.tiles;
    part = pair % S.np, g = pair / S.np;
    first = it % S.tiles * kRows, rows = min(kRows, A.n * G - first);
    k0 = part * S.cp, k1 = min(A.n_prefix, k0 + S.cp);
    const int64_t row = (int64_t)g * A.pre_ctx;
    kb = A.pre.k + row * D, vb = A.pre.v + row * D, ksb = A.pre.ks + row, vsb = A.pre.vs + row;
  } else {
    // Token t leads the run of its sequence's tokens up to the next multiple of 32 / G; other tokens' workgroups leave, as
    // do those of chunks past a sequence's end. Both are the slow dimensions (first the tokens at those multiples, then
    // the ones after them): workgroups are dealt to XCDs and their shader engines in turn, and idle ones at a fixed
    // distance would leave whole engines without work.
    const int tq = kRows / G, blocks = (A.n + tq - 1) / tq, per = blocks * A.KV;
    const int it = (int)blockIdx.x - n_pre, c = it / per % S.no, t = it % per / A.KV * tq + it / per / S.no;
    g = it % A.KV, part = S.np + c;
    if (t >= A.n) return;
    seq = A.seq[t];
    if (seq < 0 || seq >= A.n_seq || (t % tq && A.seq[t - 1] == seq)) return;
    int m = 1;
    while ((t + m) % tq && t + m < A.n && A.seq[t + m] == seq) ++m;
    first = t * G, rows = m * G;
    k0 = c * S.co, k1 = min(max(A.max_keys - A.n_prefix, 0), k0 + S.co);
    const int64_t row = ((int64_t)seq * A.KV + g) * A.n_ctx + A.row0;
    kb = A.kv.k + row * D, vb = A.kv.v + row * D, ksb = A.kv.ks + row, vsb = A.kv.vs + row;
  }
  const bool own = part >= S.np;
  // This lane's query row: its token, head and values, in the order of its half of a K row's bytes: byte b of a row is
  // element 16 (b % (D / 16)) + b / (D / 16); step j, value e of half h is byte D / 2 h + 8 j + e. A wave prepares a
  // quarter of the steps, which it asks for before anything is waited for.
  const int r = first + min(li, rows - 1), t = r / G, head = g * G + r % G;
  float x[G_::kQSteps][8];
  {
    const float* qr = q + t * q_stride + head * D;
#pragma unroll
    for (int j = 0; j < G_::kQSteps; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int byte = D / 2 * h + 8 * (G_::kQSteps * w + j) + e;
        x[j][e] = qr[16 * (byte % (D / 16)) + byte / (D / 16)];
      }
  }
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ Sum ml[kWaves][kRows];
  uint8_t* kt_s = smem + G_::kQBytes + w * G_::kWaveBytes;
  uint8_t* vt_s = kt_s + G_::kTileBytes;
  auto scales_s = [&](int st) { return vt_s + G_::kTileBytes + st * (8 * kKeys); };
  // This lane's part of a whole tile's copies.
  uint32_t off[G_::kCopies];
#pragma unroll
  for (int c = 0; c < G_::kCopies; ++c) {
    const int at = c * 64 + lane, key = at / G_::kPieces;
    off[c] = key * D + 16 * swizzle<D>(key, at % G_::kPieces);
  }
  auto copy = [&](const int8_t* from, int kt, uint8_t* to) __attribute__((always_inline)) {
    const int base = k0 + kt * kKeys, last = k1 - 1 - base;  // keys past the end: the last one again
#pragma unroll
    for (int c = 0; c < G_::kCopies; ++c) {
      uint32_t o = off[c];
      if (last < kKeys - 1) {
        const int at = c * 64 + lane, key = at / G_::kPieces;
        o = min(key, last) * D + 16 * swizzle<D>(key, at % G_::kPieces);
      }
      lds_copy16(from + (int64_t)base * D, o, to + 1024 * c);
    }
  };
  constexpr int kKeyCopies = G_::kCopies + 1;
  auto issue_k = [&](int kt, int st) __attribute__((always_inline)) {
    copy(kb, kt, kt_s);
    const int base = k0 + kt * kKeys;
    lds_copy4((h ? vsb : ksb) + base + min(li, k1 - 1 - base), scales_s(st));
  };
  auto issue_v = [&](int kt) __attribute__((always_inline)) { copy(vb, kt, vt_s); };
  // The prefix's first tile does not wait for the tokens' keys either.
  const bool early = !own && k0 + w * kKeys < k1;
  if (early) issue_k(w, 0), issue_v(w);
  // Its keys (of this kind). Columns without a row, and rows without any key, whose results nobody reads, see every key.
  int lim = INT32_MAX, most = 0;
  {
    const int s = A.seq[t];
    const int keys = s >= 0 && s < A.n_seq ? min(A.n_keys[t], A.max_keys) : 0;
    const bool live = li < rows && keys > 0;
    if (live) lim = own ? keys - A.n_prefix : keys;
    most = live ? max(lim, 0) : 0;
  }
  int least = lim;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    most = max(most, __shfl_xor(most, o));
    least = min(least, __shfl_xor(least, o));
  }
  k1 = min(k1, __builtin_amdgcn_readfirstlane(most));
  least = min(__builtin_amdgcn_readfirstlane(least), k1);  // tiles up to here are whole for every row
  if (k0 >= k1) {
    wait_vm<0>();  // LDS is not left with a copy under way
    return;
  }
  const int tiles = (k1 - k0 + kKeys - 1) / kKeys;
  if (!early && w < tiles) issue_k(w, 0), issue_v(w);

  float rf;  // score, in bits, of one unit of a product
  {
    float top = 0.0f;
#pragma unroll
    for (int j = 0; j < G_::kQSteps; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[j][e]));
    top = fmaxf(top, __shfl_xor(top, 32));
    float* top_s = reinterpret_cast<float*>(ml);
    if (h == 0) top_s[w * kRows + li] = top;
    lds_barrier();
#pragma unroll
    for (int i = 0; i < kWaves; ++i) top = fmaxf(top, top_s[i * kRows + li]);
    int ex = 0;
    if (top > 0.0f && top < INFINITY) ex = min(14 - __builtin_amdgcn_frexp_expf(top), 100);
    rf = __builtin_ldexpf(A.scale * kLog2e, -ex);
#pragma unroll
    for (int j = 0; j < G_::kQSteps; ++j) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[j][e] = __builtin_ldexpf(x[j][e], ex);
      v8h hi, lo;
      split8(x[j], hi, lo);
      v8h* to = reinterpret_cast<v8h*>(smem + (G_::kQSteps * w + j) * 2048) + lane;
      to[0] = hi, to[64] = lo;
    }
    lds_barrier();
  }
  const v8h* qs = reinterpret_cast<const v8h*>(smem) + lane;

  v16f o[G_::kDt];
#pragma unroll
  for (int i = 0; i < G_::kDt; ++i) o[i] = v16f{};
  float m = kNone, l = 0.0f;  // shift and sum of this half's weights 2^(score - m)
  bool fresh = true;
  // Scores past 2^16 bits (`wide`): a shift's own rounding would count beside the 6 bits and the value scale in it. They
  // are rounded to fp32 first (rg) and taken relative to `ms`, the row's largest when it left the range.
  bool wide = false;
  float rg = 1.0f, ms = 0.0f;

  int st = 0;
  auto tile = [&](int kt) __attribute__((always_inline)) {
    const int base = k0 + kt * kKeys;
    const bool more = kt + kWaves < tiles;
    wait_vm<G_::kCopies>();  // this tile's K and scales; its V may be under way
    fence();
    v4u k[G_::kSteps / 2];
#pragma unroll
    for (int i = 0; i < G_::kSteps / 2; ++i)
      k[i] = *reinterpret_cast<const v4u*>(kt_s + li * D + 16 * swizzle<D>(li, h * (G_::kPieces / 2) + i));
    fence();
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): K is in registers, and its place free for the next tile's
    fence();
    if (more) issue_k(kt + kWaves, st ^ 1);
    v16f s = {};
#pragma unroll
    for (int i = 0; i < G_::kSteps / 2; ++i) {
      const v8h a = cvt8(k[i][0], k[i][1]), b = cvt8(k[i][2], k[i][3]);
      s = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qs[256 * i], s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qs[256 * i + 64], s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x16_f16(b, qs[256 * i + 128], s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x16_f16(b, qs[256 * i + 192], s, 0, 0, 0);
    }
    // Register i of a half is key 8 (i / 4) + 4 h + i % 4 of the tile.
    const float* sc = reinterpret_cast<const float*>(scales_s(st));
    float vs[16], p[16], x[16];
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const v4f a = *reinterpret_cast<const v4f*>(sc + 2 * i + 4 * h);
      const v4f b = *reinterpret_cast<const v4f*>(sc + kKeys + 2 * i + 4 * h);
#pragma unroll
      for (int k = 0; k < 4; ++k) s[i + k] *= a[k], vs[i + k] = b[k];
    }
    if (wide) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = s[i] * rg - ms;
    }
    if (base + kKeys > least) {  // some row ends in this tile: what it must not see has no weight and no value
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const bool in = base + 8 * (i / 4) + 4 * h + i % 4 < min(lim, k1);
        s[i] = in ? s[i] : -INFINITY;
        vs[i] = in ? vs[i] : 0.0f;
      }
    }
    float sum, top;
    auto weights = [&] __attribute__((always_inline)) {
      sum = top = 0.0f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        p[i] = __builtin_amdgcn_exp2f(fma_(s[i], rf, -m));
        x[i] = p[i] * vs[i];
        sum += p[i];
        top = fmaxf(top, x[i]);
      }
    };
    if (!fresh) weights();
    // The first tile, and one whose weights leave fp16 or whose sum nears fp32's end: a new shift.
    if (fresh || __ballot(top > 32768.0f || !(sum < 0x1p114f))) {
      auto shift = [&] __attribute__((always_inline)) {
        float z = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) z = fmaxf(z, fma_(s[i], rf, __builtin_amdgcn_logf(fmaxf(vs[i], kLeast))));
        return fmaxf(m, fmaxf(z, __shfl_xor(z, 32)) - 6.0f);
      };
      float m1 = shift();
      if (__ballot(fabsf(m1) > 65536.0f && m1 > kNone)) {
        if (!wide) {
          wide = true, rg = rf, rf = 1.0f;
#pragma unroll
          for (int i = 0; i < 16; ++i) s[i] *= rg;
        }
        float z = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) z = fmaxf(z, s[i]);
        z = fmaxf(z, __shfl_xor(z, 32));
        if (z > 65536.0f || (m == kNone && z < -65536.0f && z > -INFINITY)) {
          ms += z, m = m == kNone ? m : m - z;
#pragma unroll
          for (int i = 0; i < 16; ++i) s[i] -= z;
        }
        m1 = shift();
      }
      const float f = __builtin_amdgcn_exp2f(m - m1);
      m = m1, l *= f;
      if (!fresh) {
#pragma unroll
        for (int i = 0; i < G_::kDt; ++i) o[i] *= f;
      }
      fresh = false;
      weights();
    }
    l += sum;
    v8h ph[2], pl[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = x[8 * u + e];
      split8(y, ph[u], pl[u]);
    }
    if (more) wait_vm<kKeyCopies>();  // this tile's V; the next tile's K may be under way
    else wait_vm<0>();
    fence();
    // ds_read_b64_tr_b8: lane i of 16 reads 8 bytes, (row i / 2, half i % 2) of an 8 x 16 byte tile, and gets the
    // tile's column i. Row e of step u is the key of weight 8 u + e.
    v2i vv[2][G_::kDt];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int e = (lane & 15) >> 1, key = 16 * u + 8 * (e >> 2) + 4 * h + (e & 3);
#pragma unroll
      for (int i = 0; i < G_::kDt; ++i)
        vv[u][i] = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
            (lds_v2i*)(vt_s + key * D + 16 * swizzle<D>(key, 2 * i + ((lane >> 4) & 1)) + 8 * (lane & 1)));
    }
    fence();
    __builtin_amdgcn_s_waitcnt(0xC07F);  // as K
    fence();
    if (more) issue_v(kt + kWaves);
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < G_::kDt; ++i) {
        const v8h a = cvt8((uint32_t)vv[u][i][0], (uint32_t)vv[u][i][1]);
        o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ph[u], o[i], 0, 0, 0);
        o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, pl[u], o[i], 0, 0, 0);
      }
    st ^= 1;
  };
  for (int kt = w; kt < tiles; kt += kWaves) tile(kt);
  l += __shfl_xor(l, 32);

  // The waves' parts of each row, brought to their largest shift and added.
  wait_vm<0>();  // a copy issued before the rows' keys were known may still be under way
  __syncthreads();
  float* ob = reinterpret_cast<float*>(smem + G_::kQBytes);
  if (h == 0) ml[w][li] = Sum{m == kNone ? kNone : ms, m, l, 0.0f};
  const int row = tid >> 3, x8 = tid & 7, rr = first + min(row, rows - 1);
  const int64_t at = ((int64_t)part * A.n + rr / G) * A.H + g * G + rr % G;
  float f[kWaves];
#pragma unroll
  for (int d0 = 0; d0 < G_::kDt; d0 += 2) {  // 64 values at a time
    if (d0) lds_barrier();
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int a = 0; a < 4; ++a)
        *reinterpret_cast<v4f*>(ob + (w * kRows + li) * G_::kOutStride + 32 * i + 8 * a + 4 * h) =
            v4f{o[d0 + i][4 * a], o[d0 + i][4 * a + 1], o[d0 + i][4 * a + 2], o[d0 + i][4 * a + 3]};
    lds_barrier();
    if (row >= rows) continue;
    if (d0 == 0) {
      float base = kNone, top = -INFINITY, sum = 0.0f;
#pragma unroll
      for (int i = 0; i < kWaves; ++i) base = fmaxf(base, ml[i][row].base);
#pragma unroll
      for (int i = 0; i < kWaves; ++i) top = fmaxf(top, f[i] = ml[i][row].above(base));
#pragma unroll
      for (int i = 0; i < kWaves; ++i) {
        f[i] = __builtin_amdgcn_exp2f(f[i] - top);
        sum = fma_(f[i], ml[i][row].l, sum);
      }
      if (x8 == 0) pml[at] = Sum{base, top, sum, 0.0f};
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int d = 4 * (x8 + 8 * i);
      v4f a = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < kWaves; ++k)
        a += f[k] * *reinterpret_cast<const v4f*>(ob + (k * kRows + row) * G_::kOutStride + d);
      *reinterpret_cast<v4f*>(po + at * D + 32 * d0 + d) = a;
    }
  }
}

// W waves per query row: the parts that its keys reach, added. Wave w of a row takes every W-th part, at most kAhead of them,
// and asks for all at once.
template <int D, int W, int kAhead>
__global__ __launch_bounds__(kThreads) void k_prefix_join(PrefixAttn A, Split S, const float* __restrict__ po,
                                                          const Sum* __restrict__ pml, float* __restrict__ out,
                                                          int64_t out_stride, BlockQ8* __restrict__ xq) {
  constexpr int E = D / 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, w = wave % W, row = blockIdx.x * (4 / W) + wave / W;
  if (row >= A.n * A.H) return;
  const int t = row / A.H, head = row % A.H, parts = S.np + S.no;
  // Parts that the row's keys do not reach hold nothing of use, and have no weight.
  const int64_t step = (int64_t)A.n * A.H;
  const float* mine_o = po + (int64_t)row * D + E * lane;
  float ahead[kAhead][E];
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    if (W * i + w < parts)
#pragma unroll
      for (int k = 0; k < E; ++k) ahead[i][k] = mine_o[(W * i + w) * step * D + k];
  Sum mine = lane < parts ? pml[lane * step + row] : Sum{};
  const int seq = A.seq[t];
  const int keys = seq >= 0 && seq < A.n_seq ? max(0, min(A.n_keys[t], A.max_keys)) : 0;
  const bool live = lane < S.np ? lane * S.cp < min(keys, A.n_prefix)
                                : lane < parts && (int64_t)A.n_prefix + (int64_t)(lane - S.np) * S.co < keys;
  if (!live) mine = Sum{kNone, kNone, 0.0f, 0.0f};
  const uint64_t all = __ballot(live);
  float v[E], sum = 1.0f;
#pragma unroll
  for (int i = 0; i < E; ++i) v[i] = 0.0f;
  if (all) {
    float base = mine.base;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) base = fmaxf(base, __shfl_xor(base, o));
    const float mm = mine.above(base);
    float top = mm;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    const float f = __builtin_amdgcn_exp2f(mm - top);
    sum = f * mine.l;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if ((all >> (W * i + w)) & 1) {
        const float fi = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), W * i + w));
#pragma unroll
        for (int k = 0; k < E; ++k) v[k] = fma_(fi, ahead[i][k], v[k]);
      }
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
#pragma unroll
  for (int k = 0; k < E; ++k) v[k] = v[k] / sum;
  float* to = out + t * out_stride + head * D + E * lane;
#pragma unroll
  for (int k = 0; k < E; ++k) to[k] = v[k];
  if (xq) quantize_block_lanes_n<E>(v, lane % (32 / E), xq + ((int64_t)row * D + E * lane) / 32);
}

constexpr int kMaxPre = 48, kMaxOwn = 16;  // a row's parts fit one wave's lanes
// Workgroups wanted of each kind; times are us a pass, 32 / 8 heads of 128 where none are named.
//
// The prefix's are long and set up once (q, the join of their waves): about one per CU. 256, or 192 / 384 / 512: 62 users
// over 8192 + 1024 keys 50, 50 / 54 / 53; 16 users over 4000 + 300 16.9, 15.5 / 16.9 / 21.1; 16 x 5 drafts of 40 heads over
// 1999 + 301 23.5, 32.2 / 25.0 / 26.6; 40 users over 12000 + 300 35.4, 41.9 / 38.3 / 35.4; 12 users over 8000 + 300 17.7,
// 18.7 / 19.8 / 22.4. Fewer leave CUs without work where the row tiles do not divide them; more are set up more often, and
// gain with the many drafts of many users (45 x 3 over 5851 + 1498 83, 83 / 71 / 68).
//
// The own rows' are as many as there are (token run, KV head) pairs, and split only where those do not fill the CUs twice.
// 512, or 256 / 128: 8 users over 1500 + 600 keys 13.5, 14.5 / 13.9; 12 users over 8000 + 300 17.7, 17.2 / 18.4; 16 users over
// 4000 + 300 16.9, 16.0 / 17.1; 10 x 5 drafts over 92 + 1361 22.1, 27.4 with 256. A run ends at a multiple of 32 / G tokens or
// where the next sequence begins, so with n_seq sequences, each one's tokens together, there are at most n G / 32 + n_seq of
// them; with n counted instead 45 x 3 drafts of 4 / 2 heads over 5851 + 1498 take 29 instead of 22.2, 57 x 7 over 4743 + 1157
// 35.5 instead of 31.3 and 10 x 5 of 32 / 8 heads over 92 + 1361 27.4 instead of 22.1 (other orders are only slower).
//
// Long chunks of the prefix go two to a CU, or nearly, where a third place is left for the own rows': 400 prompt tokens of
// 16 / 8 heads behind 8000 keys 86 instead of 94, 150 of 40 / 8 heads behind 9000 93 instead of 104. Each condition costs a
// call where it is left out: the third place 57 x 7 drafts of 16 / 8 heads over 4743 + 1157 80 instead of 77 (but 45 x 3 of 32 /
// 8 heads over 5851 + 1498 68 instead of 83), chunks from 512 keys on 57 x 7 of 8 / 2 heads 47 instead of 40, less than one
// and a half per CU the same 44 instead of 40 and 40 users over 12000 + 300 37 instead of 35.4.
constexpr int kWantedPre = 256, kWantedOwn = 512, kLongChunk = 1536;

int chunk(int keys, int chunks) {  // keys per chunk, whole tiles for the four waves
  const int c = (keys + chunks - 1) / chunks;
  return std::max(1, (c + kWaves * kKeys - 1) / (kWaves * kKeys)) * kWaves * kKeys;
}

Split split_of(int n, int H, int KV, int n_prefix, int max_keys, int n_seq) {
  Split s{};
  const int G = H / KV, tq = std::max(1, kRows / G);
  s.tiles = (int)(((int64_t)n * G + kRows - 1) / kRows);
  const int pre = std::min(n_prefix, max_keys), own = std::max(0, max_keys - n_prefix);
  const int64_t pre_wgs = (int64_t)s.tiles * KV;
  const int64_t own_wgs = std::min<int64_t>(n, (n + (int64_t)tq - 1) / tq + std::max(n_seq, 0)) * KV;
  s.co = chunk(own, (int)std::min<int64_t>(kMaxOwn, std::max<int64_t>(1, kWantedOwn / own_wgs)));
  s.no = (own + s.co - 1) / s.co;
  int64_t chunks = std::max<int64_t>(1, kWantedPre / pre_wgs);
  const int64_t more = std::min<int64_t>(2 * kWantedPre / pre_wgs, pre / kLongChunk);
  if (2 * more * pre_wgs >= 3 * kWantedPre && more * pre_wgs + own_wgs <= 3 * kWantedPre)
    chunks = std::max(chunks, more);
  s.cp = chunk(pre, (int)std::min<int64_t>(kMaxPre, chunks));
  s.np = (pre + s.cp - 1) / s.cp;
  s.parts = (int64_t)(s.np + s.no) * n * H;
  return s;
}

// Workgroups of k_prefix_parts, and of the join, whose rows have several waves where there are many parts.
int64_t parts_wgs(const PrefixAttn& A, const Split& S) {
  const int tq = kRows / (A.H / A.KV);
  return (int64_t)S.tiles * A.KV * S.np + ((int64_t)A.n + tq - 1) / tq * tq * A.KV * S.no;
}
int join_waves(const Split& S) { return S.np + S.no <= 24 ? 1 : 4; }
int64_t join_wgs(const PrefixAttn& A, const Split& S) { return ((int64_t)A.n * A.H * join_waves(S) + 3) / 4; }

}  // namespace

// The most that split_of gives up to n tokens and up to max_keys keys, whatever n_seq is: fewer tokens have more parts, in
// all too (32 / 8 heads behind 2048 + 1024 keys: 64 tokens 24576 rows of parts, 65 14560). A row has c chunks of a kind
// only where the wanted workgroups allow that many of so few tokens, and where the keys fill c of the least length.
size_t attention_prefix_workspace(int n, int H, int KV, int D, int n_prefix, int max_keys) {
  const int64_t G = H / KV, tq = std::max<int64_t>(1, kRows / G), least = kWaves * kKeys;
  const int64_t pre = std::min(n_prefix, max_keys), own = std::max(0, max_keys - n_prefix);
  int64_t parts_pre = 0, parts_own = 0;  // times tokens
  for (int64_t c = 1; c <= std::min<int64_t>(kMaxPre, (pre + least - 1) / least); ++c) {
    const int64_t wgs = (c * kLongChunk <= pre ? 2 : 1) * kWantedPre / c;
    parts_pre = std::max(parts_pre, c * (c == 1 ? n : std::min<int64_t>(n, wgs / KV * kRows / G)));
  }
  for (int64_t c = 1; c <= std::min<int64_t>(kMaxOwn, (own + least - 1) / least); ++c)
    parts_own = std::max(parts_own, c * (c == 1 ? n : std::min<int64_t>(n, kWantedOwn / c / KV * tq)));
  return (size_t)((parts_pre + parts_own) * H) * (D * sizeof(float) + sizeof(Sum));
}

size_t attention_prefix_need(const PrefixAttn& A, int D) {
  const Split S = split_of(A.n, A.H, A.KV, A.n_prefix, A.max_keys, A.n_seq);
  require(std::max(parts_wgs(A, S), join_wgs(A, S)) * kThreads < (1ll << 32), "mk_attention_prefix: too many rows");
  return (size_t)S.parts * (D * sizeof(float) + sizeof(Sum));
}

void attention_prefix(hipStream_t s, const PrefixAttn& A, int D, const float* q, int64_t q_stride, float* out,
                      int64_t out_stride, BlockQ8* xq, void* workspace) {
  const Split S = split_of(A.n, A.H, A.KV, A.n_prefix, A.max_keys, A.n_seq);
  float* po = static_cast<float*>(workspace);
  Sum* pml = reinterpret_cast<Sum*>(po + S.parts * D);
  const int64_t wgs = parts_wgs(A, S);
  auto go = [&]<int D_>() {
    if (wgs > 0) {
      allow_lds<k_prefix_parts<D_>>(Geo<D_>::kLds);
      hipLaunchKernelGGL(k_prefix_parts<D_>, dim3((unsigned)wgs), dim3(kThreads), Geo<D_>::kLds, s, A, S, q, q_stride, po,
                         pml);
      check_launch("attention_prefix parts");
    }
    auto join = [&]<int W, int kAhead>() {
      hipLaunchKernelGGL((k_prefix_join<D_, W, kAhead>), dim3((unsigned)join_wgs(A, S)), dim3(kThreads), 0, s, A, S, po, pml,
                         out, out_stride, xq);
      check_launch("attention_prefix join");
    };
    // One round trip whatever the number of parts; with eight asked for at once and the others four at a time, one token
    // behind 8682 keys (35 parts of 8 rows) took 18.4 us a pass instead of 12.6, 16 tokens behind 4000 + 300 (19 parts of
    // 512 rows) 17.0 instead of 16.2. Four waves from nine parts on: 17.5 there, 24 parts ahead for one wave everywhere: the
    // registers of the small ones.
    if (S.np + S.no <= 8) join.template operator()<1, 8>();
    else if (join_waves(S) == 1) join.template operator()<1, 24>();
    else join.template operator()<4, 16>();
  };
  if (D == 128) go.template operator()<128>();
  else go.template operator()<64>();
}

}  // namespace mk
