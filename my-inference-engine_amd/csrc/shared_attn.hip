// Attention of packed new tokens over a paged cache.
//
// One work-group per (token, query head); its four waves take every fourth key and meet in LDS.  A
// lane holds two of the head's dims, a score is the sum of the lanes' products, and each wave keeps
// the running maximum m, sum l and output O of the softmax:
//   m' = max(m, s), l' = l e^(m - m') + e^(s - m'), O' = O e^(m - m') + e^(s - m') v.
#include "cache_ops.h"

namespace mi_fa2 {

constexpr int kShWaves = 4;

template <typename E>
__global__ __launch_bounds__(64 * kShWaves) void shared_attn_kernel(const SharedParams p) {
  const int token = blockIdx.x, h = blockIdx.y, hk = h / p.group;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // the row that holds the token: cu_q[b] <= token < cu_q[b + 1]
  int lo = 0, hi = p.B;
  while (hi - lo > 1) {
    const int m = (lo + hi) >> 1;
    if (p.cu_q[m] <= token) lo = m; else hi = m;
  }
  const int b = lo, q0 = p.cu_q[b], n = p.cu_q[b + 1] - q0;
  if (token < q0 || token >= q0 + n) return;
  const int kv = clamp_len(p.kv_lens[b], p.max_kv);
  const int seen = p.causal ? min(kv, kv - n + 1 + (token - q0)) : kv;

  const uint32_t qw = *reinterpret_cast<const uint32_t*>(p.q + token * p.q_st + h * p.q_sh + 2 * lane);
  const float qa = E::lo(qw), qb = E::hi(qw);
  float m = -INFINITY, l = 0.f, oa = 0.f, ob = 0.f;
  for (int j = wave; j < seen; j += kShWaves) {
    const int blk = p.table[b * p.bt_stride + (j >> p.bs_shift)];
    const bool in = (unsigned)blk < (unsigned)p.num_blocks;
    const int64_t slot = ((int64_t)blk << p.bs_shift) + (j & ((1 << p.bs_shift) - 1));
    const int64_t at = slot * p.kv_st + hk * p.kv_sh + 2 * lane;
    const uint32_t kw = in ? *reinterpret_cast<const uint32_t*>(p.k + at) : 0;
    const uint32_t vw = in ? *reinterpret_cast<const uint32_t*>(p.v + at) : 0;
    float s = qa * E::lo(kw) + qb * E::hi(kw);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
    s *= p.scale_log2;
    const float mn = fmaxf(m, s), mu = mn == -INFINITY ? 0.f : mn;
    const float a = exp2_fast(m - mu), w = exp2_fast(s - mu);
    l = l * a + w;
    oa = oa * a + w * E::lo(vw);
    ob = ob * a + w * E::hi(vw);
    m = mn;
  }
  __shared__ float sm[kShWaves], sl[kShWaves], so[kShWaves][kHeadDim];
  if (lane == 0) {
    sm[wave] = m;
    sl[wave] = l;
  }
  so[wave][2 * lane] = oa;
  so[wave][2 * lane + 1] = ob;
  __syncthreads();
  if (wave != 0) return;
  float M = -INFINITY, L = 0.f;
  oa = ob = 0.f;
  for (int w = 0; w < kShWaves; ++w) M = fmaxf(M, sm[w]);
  const float Mu = M == -INFINITY ? 0.f : M;
  for (int w = 0; w < kShWaves; ++w) {
    const float f = exp2_fast(sm[w] - Mu);
    L += sl[w] * f;
    oa += so[w][2 * lane] * f;
    ob += so[w][2 * lane + 1] * f;
  }
  const float inv = L > 0.f ? 1.f / L : 0.f;
  *reinterpret_cast<uint32_t*>(p.o + token * p.o_st + h * p.o_sh + 2 * lane) =
      E::pack2(oa * inv, ob * inv);
  if (p.lse && lane == 0)
    p.lse[h * p.l_sh + token * p.l_st] = L > 0.f ? (M + __builtin_log2f(L)) * kLn2 : -INFINITY;
}

hipError_t launch_shared(const SharedParams& p, int dtype, hipStream_t stream) {
  const dim3 grid(p.total_q, p.Hq), block(64 * kShWaves);
  if (dtype == 0)
    hipLaunchKernelGGL((shared_attn_kernel<BF16>), grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL((shared_attn_kernel<FP16>), grid, block, 0, stream, p);
  return hipGetLastError();
}

}  // namespace mi_fa2
