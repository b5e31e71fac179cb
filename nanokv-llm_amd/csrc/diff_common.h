// Differential attention: what its decode and prefill kernels share. Heads stand in pairs; maps
// m = 0, 1 of query pair h attend with q head 2h + m over K head 2p + m of KV pair p = h / G, both
// to the pair's value, its two V heads side by side:
//   A_m = softmax(scale q_m K_m^T) [V_2p | V_2p+1]            (0 for a row that sees no key)
//   o   = A_0 - lambda A_1,  lambda = exp(lq1.lk1) - exp(lq2.lk2) + lambda_init
//   out = (1 - lambda_init) * o / sqrt(mean(o^2) + eps) * w
#pragma once

#include "nkv_common.h"

namespace nkv {

// What the operators add to an attention's arguments.
struct DiffArgs {
  const float* lambdas;  // [4, dim]: lq1, lk1, lq2, lk2
  const bf16_t* weight;  // [2 dim] in the output's type, or null: ones
  float init, eps;
};

// lambda, by the whole wave. In fp32 as the weights are: the products' sums are of order 1.
template <int DIM>
__device__ __forceinline__ float diff_lambda(const DiffArgs& d) {
  static_assert(DIM == 64 || DIM == 128, "head_dim 64 or 128");
  const int lane = threadIdx.x & 63;
  float s1 = 0.f, s2 = 0.f;
#pragma unroll
  for (int i = 0; i < DIM / 64; ++i) {
    const float* l = d.lambdas + lane + 64 * i;
    s1 = fmaf(l[0], l[DIM], s1);
    s2 = fmaf(l[2 * DIM], l[3 * DIM], s2);
  }
  return expf(wave_sum(s1)) - expf(wave_sum(s2)) + d.init;
}

// N consecutive weights (N = 2 or 4).
template <int N, bool H16>
__device__ __forceinline__ void diff_weight(const bf16_t* w, float (&v)[N]) {
  static_assert(N % 2 == 0, "pairs");
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const uint32_t x = w ? *reinterpret_cast<const uint32_t*>(w + i) : 0u;
    v[i] = w ? e16_lo<H16>(x) : 1.f;
    v[i + 1] = w ? e16_hi<H16>(x) : 1.f;
  }
}

// The checks of both entry points; `what` begins their messages.
int diff_check(const char* what, int32_t kv_type, int32_t n_q_heads, int32_t n_kv_heads,
               int32_t head_dim, float scale, float k_scale, float v_scale, const float* lambdas,
               float lambda_init, const void* norm_weight, float eps);

}  // namespace nkv
