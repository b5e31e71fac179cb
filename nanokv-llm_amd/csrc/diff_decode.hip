// Differential attention of one new token per sequence over the paged K/V cache (the formulas:
// diff_common.h). No counterpart in the reference; it stands beside the decode of
// nanokvllm/layers/attention.py:104-107 over the same cache.
//
// MI355X design (HBM-bound: every K/V byte is read once): two K heads beside each other in a
// token's row are one head of twice the dims, and their V heads are the value that both maps share.
// So the pair is streamed by the decode kernel's waves as one KV head of 128 or 256 dims with 2 G
// query columns, of which the even ones are scored against the row's first half and the odd ones
// against the second (decode_stream, DIFF): each V row is read once for both maps. Run as four
// ordinary attentions (two maps, each over both halves of the value) K and V would be read twice.
// head_dim 256 would be a KV head of 512 dims, for which the stream has no instance (a wave's piece
// of a row is at most 512 bytes), and 64 KiB a tile in the prefill, whose ring takes four: refused.
// The combine merges the partials of a pair's two rows in the halves of one workgroup, and
// subtracts, normalises and scales them in the wave that holds the first.
// 64 sequences of 2048..8192 tokens (Hq 32, Hk 8, head_dim 128): 199 us and 7.5 for the combine;
// the call 204 us, 6.2 TB/s, each byte of K and V read once. An fp8 pool: 119 us, 5.3 TB/s;
// head_dim 64: 110 us, 5.7 TB/s, fp8 69 us, 4.6 TB/s.
#include "diff_common.h"

#include <math.h>

namespace nkv {

// One workgroup per (sequence, query pair): 2 x WAVES waves, WAVES for each map. D: dims of the
// value (twice the head_dim).
template <int D, bool H16, int WAVES>
__global__ __launch_bounds__(128 * WAVES) void diff_decode_combine_kernel(
    const int32_t* __restrict__ context_lens, int32_t Hq, int32_t P, int32_t NCG,
    const float* __restrict__ part, const i32x4v_t* __restrict__ desc, const DiffArgs diff,
    bf16_t* __restrict__ out, int64_t out_row_stride) {
  __shared__ DiffLds<D, WAVES> lds;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  diff_combine<D, H16, WAVES>(DecodeSeqs{context_lens, 0}, (int)blockIdx.x / (Hq / 2),
                              (int)blockIdx.x % (Hq / 2), true, wave, Hq, P, NCG, part, desc, diff,
                              out, out_row_stride, lds);
}

int diff_check(const char* what, int32_t kv_type, int32_t n_q_heads, int32_t n_kv_heads,
               int32_t head_dim, float scale, float k_scale, float v_scale, const float* lambdas,
               float lambda_init, const void* norm_weight, float eps) {
  NKV_REQUIRE(kv_type == NKV_KV_BF16 || kv_type == NKV_KV_F16 || kv_type == NKV_KV_FP8,
              NKV_EINVAL, "%s: kv_type %d is none of NKV_KV_*", what, kv_type);
  NKV_REQUIRE(n_q_heads > 0 && n_kv_heads > 0 && n_q_heads % 2 == 0 && n_kv_heads % 2 == 0 &&
                  n_q_heads % n_kv_heads == 0,
              NKV_EINVAL, "%s: heads stand in pairs, whole groups of query pairs to a KV pair "
              "(got Hq=%d, Hk=%d)", what, n_q_heads, n_kv_heads);
  NKV_REQUIRE(head_dim == 64 || head_dim == 128, NKV_EUNSUPPORTED,
              "%s: head_dim must be 64 or 128 (got %d)", what, head_dim);
  NKV_REQUIRE(n_q_heads / n_kv_heads <= NKV_DIFF_MAX_GROUP, NKV_EUNSUPPORTED,
              "%s: %d query pairs to a KV pair, above %d", what, n_q_heads / n_kv_heads,
              NKV_DIFF_MAX_GROUP);
  NKV_REQUIRE(scale > 0.f && isfinite(scale) && k_scale > 0.f && v_scale > 0.f &&
                  isfinite(k_scale) && isfinite(v_scale),
              NKV_EINVAL, "%s: scales must be finite and > 0", what);
  NKV_REQUIRE(isfinite(lambda_init) && eps > 0.f && isfinite(eps), NKV_EINVAL,
              "%s: lambda_init must be finite and eps > 0", what);
  NKV_REQUIRE(lambdas && (reinterpret_cast<uintptr_t>(lambdas) & 3u) == 0 &&
                  (reinterpret_cast<uintptr_t>(norm_weight) & 7u) == 0,
              NKV_EINVAL, "%s: lambdas must be given, norm_weight 8-byte aligned", what);
  return NKV_OK;
}

}  // namespace nkv

extern "C" size_t nkv_diff_decode_workspace_bytes(int32_t batch, int32_t n_q_heads,
                                                  int32_t head_dim, int32_t max_blocks_per_seq,
                                                  int32_t block_size) {
  if (head_dim != 64 && head_dim != 128) return 0;
  return nkv_paged_decode_workspace_bytes(batch, n_q_heads, 2 * head_dim, max_blocks_per_seq,
                                          block_size);
}

extern "C" int nkv_diff_decode(int32_t kv_type, const void* q, int64_t q_row_stride,
                               const void* k_cache, const void* v_cache,
                               const int32_t* block_tables, int64_t bt_row_stride,
                               const int32_t* context_lens, int32_t batch, int32_t n_q_heads,
                               int32_t n_kv_heads, int32_t head_dim, int32_t block_size,
                               int32_t max_blocks_per_seq, int64_t n_blocks, float scale,
                               float k_scale, float v_scale, const float* lambdas,
                               float lambda_init, const void* norm_weight, float eps, void* out,
                               int64_t out_row_stride, void* workspace, size_t workspace_bytes,
                               void* stream) {
  using namespace nkv;
  clear_error();
  int rc = diff_check("diff_decode", kv_type, n_q_heads, n_kv_heads, head_dim, scale, k_scale,
                      v_scale, lambdas, lambda_init, norm_weight, eps);
  if (rc) return rc;
  if (batch == 0) return NKV_OK;
  // each lane stores its dims, 4 or 8 bytes
  NKV_REQUIRE(batch < 0 || (out && (reinterpret_cast<uintptr_t>(out) & 7u) == 0 &&
                             out_row_stride >= (int64_t)n_q_heads * head_dim &&
                             out_row_stride % 4 == 0),
              NKV_EINVAL, "diff_decode: out must be 8-byte aligned with a row stride >= Hq*D that "
              "is a multiple of 4");
  NKV_REQUIRE((int64_t)batch * n_q_heads < (1ll << 31), NKV_EUNSUPPORTED,
              "diff_decode: too many rows");
  const bool f16 = kv_type == NKV_KV_F16;
  if (kv_type != NKV_KV_FP8) k_scale = v_scale = 1.f;
  DecodeParts p;
  rc = decode_split_pairs(kv_type, q, q_row_stride, k_cache, v_cache, block_tables, bt_row_stride,
                          context_lens, batch, n_q_heads, n_kv_heads / 2, 2 * head_dim, block_size,
                          max_blocks_per_seq, n_blocks, scale, k_scale, v_scale, workspace,
                          workspace_bytes, stream, &p);
  if (rc) return rc;
  const DiffArgs diff{lambdas, (const bf16_t*)norm_weight, lambda_init, eps};
  const dim3 grid((unsigned)(batch * (n_q_heads / 2)));
#define NKV_DIFF_COMBINE(D, H16, W)                                                             \
  hipLaunchKernelGGL((diff_decode_combine_kernel<D, H16, W>), grid, dim3(128 * W), 0,           \
                     as_stream(stream), context_lens, n_q_heads, n_kv_heads / 2, p.ncg, p.part, \
                     p.desc, diff, (bf16_t*)out, out_row_stride)
#define NKV_DIFF_COMBINE_T(D, W)            \
  do {                                      \
    if (f16) NKV_DIFF_COMBINE(D, true, W);  \
    else NKV_DIFF_COMBINE(D, false, W);     \
  } while (0)
  if (head_dim == 64) {
    if (p.wide) NKV_DIFF_COMBINE_T(128, 4);
    else NKV_DIFF_COMBINE_T(128, 1);
  } else {
    if (p.wide) NKV_DIFF_COMBINE_T(256, 4);
    else NKV_DIFF_COMBINE_T(256, 1);
  }
#undef NKV_DIFF_COMBINE_T
#undef NKV_DIFF_COMBINE
  return check_launch("nkv_diff_decode");
}
