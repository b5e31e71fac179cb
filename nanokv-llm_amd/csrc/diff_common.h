// Differential attention: what its decode and prefill kernels share. Heads stand in pairs; maps
// m = 0, 1 of query pair h attend with q head 2h + m over K head 2p + m of KV pair p = h / G, both
// to the pair's value, its two V heads side by side:
//   A_m = softmax(scale q_m K_m^T) [V_2p | V_2p+1]            (0 for a row that sees no key)
//   o   = A_0 - lambda A_1,  lambda = exp(lq1.lk1) - exp(lq2.lk2) + lambda_init
//   out = (1 - lambda_init) * o / sqrt(mean(o^2) + eps) * w
#pragma once

#include "decode_stream.h"

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

// o = A_0 - lambda A_1 held N dims a lane, D in all: normalised and stored by the whole wave.
template <int D, bool H16>
__device__ __forceinline__ void diff_store(const DiffArgs& d, const float (&o)[D / 64],
                                           const float (&w)[D / 64], bf16_t* op) {
  constexpr int N = D / 64;
  float ss = 0.f, x[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    ss = fmaf(o[i], o[i], ss);
    x[i] = o[i] * w[i];
  }
  store_dims<N, H16>(op, x, (1.f - d.init) / sqrtf(wave_sum(ss) * (1.f / D) + d.eps));
}

// The end of one (sequence b, query pair h) of a decode stream over pairs (DIFF): the partials of
// its two maps, merged by 2 x WAVES waves (`wave` of them) of a workgroup that all call it, those
// with live = false for nothing but the barrier.
template <int D, int WAVES>
struct DiffLds {
  MergeLds<D, WAVES> merge[2];
  float second[D / 64][64];
};
template <int D, bool H16, int WAVES, typename Seqs>
__device__ __forceinline__ void diff_combine(const Seqs seqs, const int b, const int h,
                                             const bool live, const int wave, int32_t Hq,
                                             int32_t P, int32_t NCG,
                                             const float* __restrict__ part,
                                             const i32x4v_t* __restrict__ desc,
                                             const DiffArgs& diff, bf16_t* __restrict__ out,
                                             int64_t out_row_stride, DiffLds<D, WAVES>& lds) {
  constexpr int N = D / 64;
  const int lane = threadIdx.x & 63;
  const int map = wave / WAVES;
  float lambda = 0.f, w[N], o[N], l = 0.f;
  bool holds = false;
  if (live) {
    if (wave == 0) {
      lambda = diff_lambda<D / 2>(diff);
      diff_weight<N, H16>(diff.weight ? diff.weight + N * lane : nullptr, w);
    }
    holds = decode_merge<D, WAVES>(seqs, b, 2 * h + map, Hq, P, NCG, part, desc, wave % WAVES,
                                   &lds.merge[map], o, l);
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  if (holds && map == 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) lds.second[i][lane] = o[i] * inv;
  }
  __syncthreads();
  if (!live || wave > 0) return;
#pragma unroll
  for (int i = 0; i < N; ++i) o[i] = fmaf(-lambda, lds.second[i][lane], o[i] * inv);
  diff_store<D, H16>(diff, o, w, out + seqs.row(b) * out_row_stride + (int64_t)h * D + N * lane);
}

// The checks of both entry points; `what` begins their messages.
int diff_check(const char* what, int32_t kv_type, int32_t n_q_heads, int32_t n_kv_heads,
               int32_t head_dim, float scale, float k_scale, float v_scale, const float* lambdas,
               float lambda_init, const void* norm_weight, float eps);

}  // namespace nkv
