// Rotary tables with scaled frequencies; norm, rotation and the 4-bit write into the cache's pages; rows read back.
//
// A group of 32 elements x becomes x ~ s (n - 8): m is the element furthest from 0 and s = m / -8, so that m is -8 steps of s
// exactly (before s is rounded) and the other side has 7. s keeps 8 significant bits: s (n - 8) then has at most 11, which
// fp16 holds, and attention multiplies by it without a rounding. An error of s is no error of a value: n is chosen for the s
// that is stored.
//
// What bounds them: tables the memory (131072 positions 14.7 us, 4.6 TB/s, near a copy); the write of a few tokens the launch (8 of
// them 4.4 us); that of a prompt the loads that a head waits for one after the other: its elements beside position, row and
// sequence, then page, length and tables. 1500 tokens of 16 + 2 x 8 heads take 13.5 us for 39 MB, 2.9 of a copy's 5.5 TB/s, with
// vector instructions in 27 % of the cycles (four heads a group of lanes took as long); their rows read back 4.4 us. A head's
// row is 16 lanes of 8 elements (8 for head_dim 64); a group's extremes are exchanged in registers, the halves of a rotation
// through LDS, which only a head's own lanes share (no barrier).
#include <algorithm>
#include <cmath>

#include "ctx.h"
#include "kv4.h"
#include "ops.h"

namespace mk {
namespace {

constexpr int kThreads = 256;
constexpr int kPer = 8;  // elements per lane

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v4a __attribute__((ext_vector_type(4), aligned(4)));  // in the caller's memory: any stride, any row
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

// ---- tables ----

struct Turns {
  double per_pos[128];  // turns of element pair i per position
};

// Four table entries per thread. The angle is brought to [-pi/4, pi/4] in 64 bits (a far position has thousands of turns);
// the series of sine and cosine there are cut where they are below 2^-28.
__global__ __launch_bounds__(kThreads) void k_rope_tables(Turns T, int half, const float* __restrict__ divide, int64_t first,
                                                          int64_t total, float mul, float* __restrict__ cos_t,
                                                          float* __restrict__ sin_t) {
  __shared__ double turns[128];
  for (int i = threadIdx.x; i < half; i += kThreads) turns[i] = T.per_pos[i] / (divide ? (double)divide[i] : 1.0);
  __syncthreads();
  for (int64_t at = 4 * ((int64_t)blockIdx.x * kThreads + threadIdx.x); at < total; at += 4ll * kThreads * gridDim.x) {
    float c[4], s[4];
    int64_t pos = at / half;
    int i = (int)(at - pos * half);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const double t = 4.0 * ((double)(first + pos) * turns[i]);  // quarter turns
      const double n = __builtin_rint(t);
      const float x = (float)(t - n) * 1.57079632679489662f, x2 = x * x;
      const int quarter = (int)((int64_t)n & 3);
      float p = fma_(x2, 1.0f / 362880, -1.0f / 5040);
      p = fma_(p, x2, 1.0f / 120);
      p = fma_(p, x2, -1.0f / 6);
      const float sn = fma_(p * x2, x, x);
      float q = fma_(x2, -1.0f / 3628800, 1.0f / 40320);
      q = fma_(q, x2, -1.0f / 720);
      q = fma_(q, x2, 1.0f / 24);
      q = fma_(q, x2, -0.5f);
      const float cs = fma_(q, x2, 1.0f);
      const float a = quarter & 1 ? sn : cs, b = quarter & 1 ? cs : sn;
      c[e] = (quarter == 1 || quarter == 2 ? -a : a) * mul;
      s[e] = (quarter & 2 ? -b : b) * mul;
      if (++i == half) i = 0, ++pos;
    }
    if (at + 4 <= total) {
      *reinterpret_cast<v4a*>(cos_t + at) = v4a{c[0], c[1], c[2], c[3]};
      *reinterpret_cast<v4a*>(sin_t + at) = v4a{s[0], s[1], s[2], s[3]};
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (at + e < total) cos_t[at + e] = c[e], sin_t[at + e] = s[e];
    }
  }
}

// ---- norm, rotation, 4-bit rows ----

// The scale of a group whose extremes are hi and lo (include/malkin_hip.h): m / -8 to 8 significant bits, then to fp16.
__device__ __forceinline__ _Float16 scale_of(double hi, double lo) {
  const double m = hi >= -lo ? hi : lo;
  const double s = fmin(fmax(m * -0.125, -4096.0), 4096.0);
  uint64_t u = __builtin_bit_cast(uint64_t, s);
  u = (u + ((1ull << 44) - 1) + (u >> 45 & 1)) & ~((1ull << 45) - 1);  // to nearest, ties to even
  return (_Float16)(float)__builtin_bit_cast(double, u);
}

__device__ __forceinline__ double fma_(double a, double b, double c) { return __builtin_fma(a, b, c); }
typedef double v4d __attribute__((ext_vector_type(4)));

struct Rope {
  const float *cos_t, *sin_t;
  const float *q_norm, *k_norm;
  const int32_t *rpos, *seq, *kv_row;
  const int32_t* len;  // rows that sequences hold, or null
  float eps;
  int half, n_pos, pairs, n, H;  // half: pairs of elements that rotate
};

// Norm and rotation of a lane's eight elements. FAST: they rotate with eight neighbours, or with each other, all of them or none.
// mine: the head's row in LDS.
template <int D, bool FAST, class T>
__device__ __forceinline__ void turn_row(const Rope& R, T (&x)[kPer], const float* w, int pos, int l, T* mine) {
  typedef T v4 __attribute__((ext_vector_type(4)));
  constexpr int L = D / kPer;
  if (w) {
    T acc = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) acc = fma_(x[e], x[e], acc);
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) acc += __shfl_xor(acc, o, L);
    const T s = (T)1 / sqrt(acc / (T)D + (T)R.eps);
#pragma unroll
    for (int e = 0; e < kPer; ++e) x[e] = x[e] * s * (T)w[kPer * l + e];
  }
  const float *ct = R.cos_t + (int64_t)pos * R.half, *st = R.sin_t + (int64_t)pos * R.half;
  if (R.pairs) {
    const int i0 = kPer / 2 * l;
    auto turn = [&](int e, T c, T s) {
      const T a = x[2 * e], b = x[2 * e + 1];
      x[2 * e] = fma_(a, c, -(b * s));
      x[2 * e + 1] = fma_(a, s, b * c);
    };
    if constexpr (FAST) {
      if (i0 < R.half) {
        const v4f c = *reinterpret_cast<const v4a*>(ct + i0), s = *reinterpret_cast<const v4a*>(st + i0);
#pragma unroll
        for (int e = 0; e < kPer / 2; ++e) turn(e, (T)c[e], (T)s[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < kPer / 2; ++e)
        if (i0 + e < R.half) turn(e, (T)ct[i0 + e], (T)st[i0 + e]);
    }
    return;
  }
#pragma unroll
  for (int c = 0; c < 2; ++c)
    *reinterpret_cast<v4*>(mine + kPer * l + 4 * c) = v4{x[4 * c], x[4 * c + 1], x[4 * c + 2], x[4 * c + 3]};
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  if constexpr (FAST) {  // a lane's elements are all of one half, or none rotates
    const int i0 = kPer * l;
    if (i0 >= 2 * R.half) return;
    const bool up = i0 >= R.half;
    const int i = up ? i0 - R.half : i0, other = up ? i0 - R.half : i0 + R.half;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const v4f cv = *reinterpret_cast<const v4a*>(ct + i + 4 * c), sv = *reinterpret_cast<const v4a*>(st + i + 4 * c);
      const v4 y = *reinterpret_cast<const v4*>(mine + other + 4 * c);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const T s = (T)(up ? sv[e] : -sv[e]);
        x[4 * c + e] = fma_(x[4 * c + e], (T)cv[e], y[e] * s);
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int i0 = kPer * l + e;
      if (i0 < 2 * R.half) {
        const bool up = i0 >= R.half;
        const int i = up ? i0 - R.half : i0;
        const T s = (T)(up ? st[i] : -st[i]);
        x[e] = fma_(x[e], (T)ct[i], mine[up ? i : i0 + R.half] * s);
      }
    }
  }
}

// One (token, head) per D / 8 lanes: lane l holds elements 8 l .. 8 l + 7. Keys are turned, and keys and values brought to their
// steps, in 64 bits: a number next to the border between two of them would else go with the rounding (one in a million does).
template <int D, bool FAST>
__global__ __launch_bounds__(kThreads) void k_rope_kv4(Rope R, Kv4 kv, const float* q, const float* __restrict__ k,
                                                       const float* __restrict__ v, int64_t stride, float* q_out,
                                                       int64_t q_out_stride) {
  constexpr int L = D / kPer;  // lanes per head
  __shared__ __align__(32) double sh[kThreads / L][D];
  const int l = threadIdx.x % L, nh = R.H + 2 * kv.KV;
  const int64_t it = (int64_t)blockIdx.x * (kThreads / L) + threadIdx.x / L;
  if (it >= (int64_t)R.n * nh) return;  // all lanes of a head
  const int t = (int)(it / nh), hh = (int)(it % nh);
  const bool is_q = hh < R.H, is_v = hh >= R.H + kv.KV;
  const int head = is_q ? hh : is_v ? hh - R.H - kv.KV : hh - R.H;
  const float* src = (is_q ? q : is_v ? v : k) + t * stride + (int64_t)head * D + kPer * l;
  float f[kPer];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const v4f y = *reinterpret_cast<const v4a*>(src + 4 * c);
#pragma unroll
    for (int e = 0; e < 4; ++e) f[4 * c + e] = y[e];
  }
  const int pos = R.rpos[t], row = R.kv_row[t], sq = R.seq[t], p = kv.page_of(sq, row);
  // A row past its sequence's may be one of somebody who holds the page too. The length comes with the page's number.
  const int len = R.len ? R.len[min(max(sq, 0), kv.n_seq - 1)] : INT32_MAX;
  if (p < 0 || row >= len || pos < 0 || pos >= R.n_pos) return;
  if (is_q) {
    turn_row<D, FAST, float>(R, f, R.q_norm, pos, l, reinterpret_cast<float*>(sh[threadIdx.x / L]));
    float* to = q_out + t * q_out_stride + (int64_t)head * D + kPer * l;
#pragma unroll
    for (int c = 0; c < 2; ++c) *reinterpret_cast<v4a*>(to + 4 * c) = v4a{f[4 * c], f[4 * c + 1], f[4 * c + 2], f[4 * c + 3]};
    return;
  }
  double x[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) x[e] = (double)f[e];
  if (!is_v) turn_row<D, FAST, double>(R, x, R.k_norm, pos, l, sh[threadIdx.x / L]);
  double hi = -INFINITY, lo = INFINITY;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    if (x[e] != x[e]) x[e] = 0.0;
    hi = fmax(hi, x[e]), lo = fmin(lo, x[e]);
  }
#pragma unroll
  for (int o = 1; o < kKv4Group / kPer; o <<= 1) hi = fmax(hi, __shfl_xor(hi, o)), lo = fmin(lo, __shfl_xor(lo, o));
  const _Float16 s = scale_of(hi, lo);
  const double inv = s != (_Float16)0.0f ? 1.0 / (double)s : 0.0;
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    const double y = x[e] * inv;
    double n = __builtin_rint(y);
    if (fabs(fabs(y - n) - 0.5) < 0x1p-40) n = __builtin_rint(x[e] / (double)s);  // in the middle, as far as inv says
    w |= (uint32_t)((int)fmin(fmax(n, -8.0), 7.0) + 8) << (4 * e);
  }
  const int64_t first = kv.first_row(p, head);
  const int r = row & ((1 << kv.shift) - 1), grp = l / (kKv4Group / kPer);
  *reinterpret_cast<uint32_t*>((is_v ? kv.v : kv.k) + (first + r) * (D / 2) + 4 * l) = w;
  if (l % (kKv4Group / kPer) == 0) {
    const uint16_t b = __builtin_bit_cast(uint16_t, s);
    if (is_v) kv.vs[first * (D / kKv4Group) + ((int64_t)grp << kv.shift) + r] = b;
    else kv.ks[(first + r) * (D / kKv4Group) + grp] = b;
  }
}

// One row of a head and side per D / 8 lanes.
template <int D>
__global__ __launch_bounds__(kThreads) void k_kv4_rows(Kv4 kv, const int32_t* __restrict__ seq, const int32_t* __restrict__ rows,
                                                       int n, _Float16* __restrict__ k_out, _Float16* __restrict__ v_out) {
  constexpr int L = D / kPer;
  const int l = threadIdx.x % L;
  const int64_t it = (int64_t)blockIdx.x * (kThreads / L) + threadIdx.x / L;
  const int i = (int)(it / (2 * kv.KV)), hh = (int)(it % (2 * kv.KV)), g = hh >> 1;
  if (i >= n) return;
  const bool is_v = hh & 1;
  _Float16* out = is_v ? v_out : k_out;
  if (!out) return;
  const int row = rows[i], p = kv.page_of(seq[i], row);
  v8h y = {};
  if (p >= 0) {
    const int64_t first = kv.first_row(p, g);
    const int r = row & ((1 << kv.shift) - 1), grp = l / (kKv4Group / kPer);
    const uint32_t w = *reinterpret_cast<const uint32_t*>((is_v ? kv.v : kv.k) + (first + r) * (D / 2) + 4 * l);
    const uint16_t b = is_v ? kv.vs[first * (D / kKv4Group) + ((int64_t)grp << kv.shift) + r] : kv.ks[(first + r) * (D / kKv4Group) + grp];
    const _Float16 s = __builtin_bit_cast(_Float16, b);
#pragma unroll
    for (int e = 0; e < kPer; ++e) y[e] = (_Float16)((int)(w >> (4 * e) & 15) - 8) * s;
  }
  *reinterpret_cast<v8h*>(out + ((int64_t)i * kv.KV + g) * D + kPer * l) = y;
}

}  // namespace

void rope_tables(hipStream_t s, const mk_rope& r, const float* divide, int64_t first, int n_pos, float* cos_t, float* sin_t) {
  Turns T{};
  const int half = r.dim / 2;
  const double d = r.dim, factor = r.factor;
  double base = r.base, mul = 1.0;
  if (r.scaling == MK_ROPE_NTK) base *= std::pow(factor, d / (d - 2));
  double low = 0, high = 0;
  if (r.scaling == MK_ROPE_YARN) {
    // The pair that makes beta turns over the trained context.
    auto pair_of = [&](double beta) { return d * std::log(r.n_orig / (2 * M_PI * beta)) / (2 * std::log(base)); };
    low = std::max(std::floor(pair_of(r.beta_fast)), 0.0), high = std::min(std::ceil(pair_of(r.beta_slow)), d - 1);
    mul = r.attn_factor != 0.0 ? r.attn_factor : 0.1 * std::log(factor) + 1;
  }
  for (int i = 0; i < half; ++i) {
    double f = std::pow(base, -2 * i / d);
    if (r.scaling == MK_ROPE_LINEAR) f /= factor;
    if (r.scaling == MK_ROPE_YARN) {
      const double ramp = std::min(std::max((i - low) / std::max(high - low, 0.001), 0.0), 1.0);
      f = f / factor * ramp + f * (1 - ramp);
    }
    T.per_pos[i] = f / (2 * M_PI);
  }
  const int64_t total = (int64_t)n_pos * half, wgs = (total + 4 * kThreads - 1) / (4 * kThreads);
  hipLaunchKernelGGL(k_rope_tables, dim3((unsigned)std::min<int64_t>(wgs, 8 * device_cus())), dim3(kThreads), 0, s, T, half,
                     divide, first, total, (float)mul, cos_t, sin_t);
  check_launch("rope_tables");
}

void rope_kv4(hipStream_t s, const Kv4& kv, int D, const float* q, const float* k, const float* v, int64_t stride, int n, int H,
              const float* q_norm, const float* k_norm, float eps, bool pairs, int rope_dim, const float* cos_t,
              const float* sin_t, int n_pos, const int32_t* rpos, const int32_t* seq, const int32_t* kv_row, const int32_t* len,
              float* q_out, int64_t q_out_stride) {
  const Rope R{cos_t, sin_t, q_norm, k_norm, rpos, seq, kv_row, len, eps, rope_dim / 2, n_pos, pairs, n, H};
  const int64_t items = (int64_t)n * (H + 2 * kv.KV), per = kThreads / (D / kPer), wgs = (items + per - 1) / per;
  const bool fast = R.half % (pairs ? kPer / 2 : kPer) == 0;
  auto go = [&]<int D_, bool F>() {
    hipLaunchKernelGGL((k_rope_kv4<D_, F>), dim3((unsigned)wgs), dim3(kThreads), 0, s, R, kv, q, k, v, stride, q_out,
                       q_out_stride);
  };
  if (D == 128) fast ? go.template operator()<128, true>() : go.template operator()<128, false>();
  else fast ? go.template operator()<64, true>() : go.template operator()<64, false>();
  check_launch("rope_kv4");
}

void kv4_rows(hipStream_t s, const Kv4& kv, int D, const int32_t* seq, const int32_t* rows, int n, void* k_out, void* v_out) {
  const int64_t items = 2ll * n * kv.KV, per = kThreads / (D / kPer), wgs = (items + per - 1) / per;
  auto go = [&]<int D_>() {
    hipLaunchKernelGGL(k_kv4_rows<D_>, dim3((unsigned)wgs), dim3(kThreads), 0, s, kv, seq, rows, n,
                       static_cast<_Float16*>(k_out), static_cast<_Float16*>(v_out));
  };
  if (D == 128) go.template operator()<128>();
  else go.template operator()<64>();
  check_launch("kv4_rows");
}

}  // namespace mk
