// Attention of a batch whose sequences share a prefix: key j < n_prefix of every token is row j of one sequence of the
// prefix's cache, the others rows of the token's own sequence. Softmax statistics and sums are fp32.
#include "ctx.h"
#include "ops.h"

namespace mk {
namespace {

// One wave per (token, query head), one key at a time.
template <int D>
__global__ __launch_bounds__(64) void k_prefix_attention(PrefixAttn A, const float* __restrict__ q, int64_t q_stride,
                                                         float* __restrict__ out, int64_t out_stride,
                                                         BlockQ8* __restrict__ xq) {
  constexpr int E = D / 64;
  const int t = blockIdx.x / A.H, h = blockIdx.x % A.H, g = h / (A.H / A.KV), lane = threadIdx.x;
  const int seq = A.seq[t];
  const int keys = seq >= 0 && seq < A.n_seq ? min(A.n_keys[t], A.max_keys) : 0;
  // Byte b of a K row is element 16 (b % (D / 16)) + b / (D / 16).
  float qv[E], o[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int b = E * lane + i;
    qv[i] = q[t * q_stride + h * D + 16 * (b % (D / 16)) + b / (D / 16)] * A.scale;
    o[i] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  for (int j = 0; j < keys; ++j) {
    const bool pre = j < A.n_prefix;
    const int64_t row = pre ? (int64_t)g * A.pre_ctx + j
                            : ((int64_t)seq * A.KV + g) * A.n_ctx + A.row0 + (j - A.n_prefix);
    const KvLayer& L = pre ? A.pre : A.kv;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) s = fma_(qv[i], (float)L.k[row * D + E * lane + i], s);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off);
    s *= L.ks[row];
    const float m1 = fmaxf(m, s), r = expf(m - m1), p = expf(s - m1), pv = p * L.vs[row];
    l = fma_(l, r, p);
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = fma_(o[i], r, pv * (float)L.v[row * D + E * lane + i]);
    m = m1;
  }
  float* row = out + t * out_stride + h * D;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    o[i] = keys > 0 ? o[i] / l : 0.0f;
    row[E * lane + i] = o[i];
  }
  if (xq) quantize_block_lanes_n<E>(o, lane % (32 / E), xq + ((int64_t)t * A.H * D + h * D + E * lane) / 32);
}

}  // namespace

size_t attention_prefix_workspace(int n, int H, int KV, int D, int n_prefix, int max_keys) { return 0; }

void attention_prefix(hipStream_t s, const PrefixAttn& A, int D, const float* q, int64_t q_stride, float* out,
                      int64_t out_stride, BlockQ8* xq, void* workspace) {
  const dim3 grid((unsigned)(A.n * A.H));
  if (D == 128)
    hipLaunchKernelGGL(k_prefix_attention<128>, grid, dim3(64), 0, s, A, q, q_stride, out, out_stride, xq);
  else
    hipLaunchKernelGGL(k_prefix_attention<64>, grid, dim3(64), 0, s, A, q, q_stride, out, out_stride, xq);
  check_launch("attention_prefix");
}

}  // namespace mk
