// Attention of one new token per sequence (GQA) over the block-scaled K/V cache (scaled_cache.h).
//
// Reference: beside flash_attn_with_kvcache(q.unsqueeze(1), k_cache, v_cache, cache_seqlens,
// block_table, softmax_scale, causal=True) at nanokvllm/layers/attention.py:104-107.
//   out_h = softmax(scale * q_h . K) V    over the sequence's keys, K and V = code * 2^e
//
// MI355X design (HBM-bound: every code is read once). The batch's tiles of 32 tokens are one stream
// per KV head, cut into equal ranges over the resident waves (as paged_decode.hip cuts its chunks,
// whose combine merges the partials). A wave takes one KV head: a tile of it is 32 D bytes of K and as
// many of V, each consecutive in memory, in the lanes' order for the matrix instructions. So codes
// go from their load straight into the products: no LDS, no transposition.
//   S^T = K q^T      v_mfma_f32_16x16x32_bf16, A = 16 keys, B = up to 16 of the group's query heads
//   O^T += V^T P^T   the same, A = 16 dims x 32 keys, B = the lane's own eight weights
// v_cvt_scalef32_pk_bf16_fp8 widens two codes and applies the tile's scale, exactly, on the way. The
// running maximum is only raised when a score exceeds it by more than kLazy (log2), so that most
// tiles need no exchange between lanes.
// 64 sequences, 638 MB of codes (Hq 32, Hk 8, D 128): 105 us and 4.7 for the combine, 5.8 TB/s; one of
// 246 MB 41 and 4.6. Loads that the caches keep: 123 us; a ring twice as deep, or K's place refilled
// before V's products: the same.
#include "decode_stream.h"
#include "scaled_cache.h"

#include <math.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

namespace nkv {

constexpr float kLazy = 8.f;  // log2 headroom before the running maximum is raised

template <int D>
__global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(2)))
void scaled_decode_kernel(
    const bf16_t* __restrict__ q, int64_t q_row_stride, const char* __restrict__ k_cache,
    const char* __restrict__ v_cache, const int32_t* __restrict__ block_tables,
    int64_t bt_row_stride, const int32_t* __restrict__ context_lens, int32_t batch, int32_t Hk,
    int32_t G, int32_t NCG, int32_t block_size, int32_t max_blocks, int64_t n_blocks,
    int32_t min_chunks, float scale_log2, float* __restrict__ part, i32x4v_t* __restrict__ desc) {
  constexpr int kI = D / 64;             // 1 KiB loads of 16 keys (K), half those of the tile's V
  constexpr int kLoads = 2 * kI;         // of a tile's K, and of its V
  constexpr int kDb = D / 16;            // 16-dim blocks of O^T
  constexpr int kRing = D == 128 ? 2 : 4;  // tiles in flight: 16 KiB of K and V a wave
  const int lane = threadIdx.x & 63;
  const int g4 = lane >> 4;
  const int col = lane & 15;
  const DecodeSeqs seqs{context_lens, batch};
  const int max_tokens = max_blocks * block_size;
  const int tiles_per_block = block_size / kTileRows;
  const int tile_bytes = kTileRows * (Hk * D + kRowPad);

  // this wave's KV head, column group and range (paged_decode.hip)
  const int NP = Hk * NCG;
  const int grp = (int)blockIdx.x % NP;
  const int kvh = grp / NCG;
  const int cg = grp - kvh * NCG;
  const int cols = NCG > 1 ? min(kMaxCols, G - cg * kMaxCols) : G;
  const int qh0 = kvh * G + cg * kMaxCols;
  const int wi = (int)blockIdx.x / NP;
  const int Wh = (int)gridDim.x / NP;
  float* gpart = part + (int64_t)(Wh + batch) * qh0 * part_row(D);
  SeqCursor cur;
  cur.cb = 0;
  cur.base = 0;
  seq_load<kTileRows>(cur, seqs, max_tokens);
  int T = cur.tot;
  if (batch > 64) {
    int more = 0;
#pragma unroll 4
    for (int s = 64 + lane; s < batch; s += 64)
      more += seq_chunks<kTileRows>(seqs.keys(s), max_tokens);
    T += __builtin_amdgcn_readlane(wave_incl_scan(more), 63);
  }
  const int C = max((T + Wh - 1) / Wh, min_chunks);
  const int k_begin = wi * C;
  if (k_begin >= T) return;
  const int k_end = min(T, k_begin + C);
  const int code_off = kvh * (kTileRows * D) + lane * 16;
  const int scale_off = kTileRows * Hk * D + kvh;

  for (int k = k_begin; k < k_end;) {
    // the sequence that holds tile k of the stream
    while (k >= cur.base + cur.tot) {
      cur.base += cur.tot;
      cur.cb += 64;
      seq_load<kTileRows>(cur, seqs, max_tokens);
    }
    const int ln =
        __builtin_amdgcn_readfirstlane(__builtin_ctzll(__ballot(cur.base + cur.incl > k)));
    const int b = cur.cb + ln;
    const int ctx = __builtin_amdgcn_readlane(cur.ctx, ln);
    const int nc = __builtin_amdgcn_readlane(cur.nc, ln);
    const int g0 = cur.base + __builtin_amdgcn_readlane(cur.incl, ln) - nc;
    const int c_lo = k - g0;
    const int n_seg = min(nc - c_lo, k_end - k);
    const int w_first = g0 / C;  // first wave of the segment

    // q^T as the B operand: column col, dims 64 i + 16 g4 + 0..15 (columns past the group's re-read
    // its first head and are discarded)
    u32x4_t qreg[2 * kI];
    {
      const u32x4_t* qp = reinterpret_cast<const u32x4_t*>(
          q + b * q_row_stride + (int64_t)(qh0 + (col < cols ? col : 0)) * D + g4 * 16);
#pragma unroll
      for (int i = 0; i < kI; ++i) {
        qreg[2 * i] = qp[8 * i];
        qreg[2 * i + 1] = qp[8 * i + 1];
      }
    }
    const int32_t* bt_row = block_tables + (int64_t)b * bt_row_stride;
    f32x4_t acc[kDb];  // O^T: lane l -> column l%16, dims 16*db + 4*(l/16) .. +3
#pragma unroll
    for (int db = 0; db < kDb; ++db) acc[db] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    float m_run = -INFINITY, mb = 0.f, l_run = 0.f;  // mb: m_run, or 0 while there is no key

    // windows of at most 64 cache blocks (block ids one per lane)
    const int win_cap = (kWinBlocks - 1) * tiles_per_block;
    for (int wc = 0; wc < n_seg; wc += win_cap) {
      const int wlo = c_lo + wc;                // first tile of the window
      const int wn = min(n_seg - wc, win_cap);  // tiles in the window
      const int blk0 = wlo / tiles_per_block;
      int blk_id = -1;
      {
        const int bi = blk0 + lane;
        if (bi < max_blocks && bi * tiles_per_block < wlo + wn) {
          const int id = bt_row[bi];
          NKV_DBG(id < 0 || id >= n_blocks, NKV_DEBUG_BLOCK);  // every block here is needed
          blk_id = (id >= 0 && id < n_blocks) ? id : -1;
        }
      }

      u32x4_t kreg[kRing][kLoads], vreg[kRing][kLoads];
      uint32_t kscale[kRing], vscale[kRing];  // words of the scale bytes
      int nv[kRing];  // keys of the tile in each ring slot (0: masked)
      auto issue = [&](int j, int s) {
        const int tile = wlo + j;
        const int blk = tile / tiles_per_block;
        const int pb = __builtin_amdgcn_readlane(blk_id, min(blk - blk0, 63));
        const int keys = j < wn ? min(max(ctx - tile * kTileRows, 0), kTileRows) : 0;
        nv[s] = pb >= 0 ? keys : 0;
        const int64_t at = (int64_t)(pb < 0 ? 0 : pb) * tiles_per_block + tile % tiles_per_block;
        const uint32_t bytes = nv[s] > 0 ? (uint32_t)tile_bytes : 0;
        const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc(
            (void*)(k_cache + at * tile_bytes), (short)0, bytes, kBufferFlags);
        const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc(
            (void*)(v_cache + at * tile_bytes), (short)0, bytes, kBufferFlags);
        kscale[s] = __builtin_amdgcn_raw_buffer_load_b32(rk, scale_off & ~3, 0, 0);
#pragma unroll
        for (int p = 0; p < kLoads; ++p)
          kreg[s][p] = __builtin_bit_cast(
              u32x4_t,
              __builtin_amdgcn_raw_buffer_load_b128(rk, code_off + p * 1024, 0, kStreamPolicy));
        vscale[s] = __builtin_amdgcn_raw_buffer_load_b32(rv, scale_off & ~3, 0, 0);
#pragma unroll
        for (int p = 0; p < kLoads; ++p)
          vreg[s][p] = __builtin_bit_cast(
              u32x4_t,
              __builtin_amdgcn_raw_buffer_load_b128(rv, code_off + p * 1024, 0, kStreamPolicy));
      };

      auto consume = [&](int s, auto refill, int nxt) {
        const int n = nv[s];  // the refill below overwrites the slot's count
        // S^T: lane -> column col, tokens 8 g4 + 4 t + 0..3
        const float ks = scale_of(stored_scale(byte_of(kscale[s], scale_off)));
        f32x4_t st[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          f32x4_t a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < kI; ++i) {
            const u32x4_t c = kreg[s][t * kI + i];
            a = mfma_16x16x32<false>(codes_to_bf16(c[0], c[1], ks), qreg[2 * i], a);
            a = mfma_16x16x32<false>(codes_to_bf16(c[2], c[3], ks), qreg[2 * i + 1], a);
          }
          st[t] = a;
        }
        float sv[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) sv[e] = st[e >> 2][e & 3] * scale_log2;
        if (n < kTileRows) {  // uniform: the sequence's last tile, or none
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (8 * g4 + e >= n) sv[e] = -INFINITY;
          // codes behind the end may be anything, NaN too: a zero weight would not hide them
          const int m = min(max(n - 8 * g4, 0), 8);
          const uint64_t keep = m >= 8 ? ~0ull : (1ull << (8 * m)) - 1;
#pragma unroll
          for (int p = 0; p < kLoads; ++p) {
            vreg[s][p][0] &= (uint32_t)keep;
            vreg[s][p][1] &= (uint32_t)(keep >> 32);
            vreg[s][p][2] &= (uint32_t)keep;
            vreg[s][p][3] &= (uint32_t)(keep >> 32);
          }
        }
        const float top = fmax3(fmax3(sv[0], sv[1], sv[2]), fmax3(sv[3], sv[4], sv[5]),
                                fmax3(sv[6], sv[7], -INFINITY));
        if (__builtin_amdgcn_ballot_w64(top > m_run + kLazy) != 0) {
          const float cm = col_max4(top);
          const bool raise = cm > m_run + kLazy;
          const float alpha = raise ? fast_exp2(m_run - cm) : 1.f;  // exp2(-inf) = 0
          m_run = raise ? cm : m_run;
          mb = m_run == -INFINITY ? 0.f : m_run;
          l_run *= alpha;
#pragma unroll
          for (int db = 0; db < kDb; ++db) acc[db] *= alpha;
        }
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = fast_exp2(sv[e] - mb);
        // Weights are rounded to bf16, as the product takes them, each by 2^-8 of it at most. Outputs are
        // off from 64 bits by 0.0014 - 0.0020 (relative), with weights of 32 bits by 0.0014 - 0.0018: most
        // of both is their own rounding. The sum is that of the rounded weights, which multiply V.
        const u32x4_t pb = {cvt_pk16<false>(p[0], p[1]), cvt_pk16<false>(p[2], p[3]),
                            cvt_pk16<false>(p[4], p[5]), cvt_pk16<false>(p[6], p[7])};
#pragma unroll
        for (int e = 0; e < 4; ++e) l_run = sum2_16<false>(pb[e], l_run);
        const float vs = scale_of(stored_scale(byte_of(vscale[s], scale_off)));
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
          const u32x4_t c = vreg[s][j];
          acc[2 * j] = mfma_16x16x32<false>(codes_to_bf16(c[0], c[1], vs), pb, acc[2 * j]);
          acc[2 * j + 1] = mfma_16x16x32<false>(codes_to_bf16(c[2], c[3], vs), pb, acc[2 * j + 1]);
        }
        if constexpr (decltype(refill)::value) {
          __builtin_amdgcn_sched_barrier(0);
          issue(nxt, s);
          __builtin_amdgcn_sched_barrier(0);
        }
      };

      const int n_groups = (wn + kRing - 1) / kRing;
#pragma unroll
      for (int s = 0; s < kRing; ++s) issue(s, s);
      for (int gi = 0; gi + 1 < n_groups; ++gi) {
#pragma unroll
        for (int s = 0; s < kRing; ++s)
          consume(s, std::integral_constant<bool, true>{}, (gi + 1) * kRing + s);
      }
#pragma unroll
      for (int s = 0; s < kRing; ++s) consume(s, std::integral_constant<bool, false>{}, 0);
    }

    // the segment's partial and, from the wave that ends it, its descriptor
    l_run = col_sum4(l_run);
    const int prow0 = (wi + b) * cols;
    if (col < cols) {
      float* pr = gpart + (int64_t)(prow0 + col) * part_row(D);
#pragma unroll
      for (int db = 0; db < kDb; ++db)
        *reinterpret_cast<f32x4_t*>(&pr[db * 16 + g4 * 4]) = acc[db];
      if (g4 == 0) *reinterpret_cast<float2*>(&pr[D]) = float2{m_run, l_run};
    }
    if (c_lo + n_seg == nc && lane == 0) {
      const int64_t first = (int64_t)(Wh + batch) * qh0 + (int64_t)(w_first + b) * cols;
      desc[((int64_t)b * Hk + kvh) * NCG + cg] =
          i32x4v_t{(int32_t)first, wi - w_first + 1, cols, 0};
    }
    k += n_seg;
  }
}

// As many one-wave workgroups as are resident at once, at most kWavesPerCU per CU (the workspace
// bound assumes no more).
template <int D>
static int scaled_decode_grid() {
  static std::atomic<int> cached[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) dev = 0;
  int n = cached[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    int per_cu = 0;
    if (hipOccupancyMaxActiveBlocksPerMultiprocessor(
            &per_cu, reinterpret_cast<const void*>(scaled_decode_kernel<D>), 64, 0) != hipSuccess ||
        per_cu <= 0)
      per_cu = kWavesPerCU;
    n = device_cus() * std::min(per_cu, kWavesPerCU);
    cached[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

int scaled_check_heads(const char* what, int64_t n_q_heads, int64_t n_kv_heads, int64_t most,
                       double scale) {
  NKV_REQUIRE(n_kv_heads > 0 && n_q_heads > 0 && n_q_heads % n_kv_heads == 0, NKV_EINVAL,
              "%s: n_q_heads must be a multiple of n_kv_heads (got %lld, %lld)", what,
              (long long)n_q_heads, (long long)n_kv_heads);
  NKV_REQUIRE(n_q_heads / n_kv_heads <= most, NKV_EUNSUPPORTED, "%s: GQA group %lld above %lld",
              what, (long long)(n_q_heads / n_kv_heads), (long long)most);
  NKV_REQUIRE(scale > 0 && isfinite((float)scale), NKV_EINVAL, "%s: scale must be finite and > 0",
              what);
  return NKV_OK;
}

}  // namespace nkv

extern "C" int nkv_scaled_decode(const nkv_scaled_decode_args* args) {
  using namespace nkv;
  clear_error();
  NKV_REQUIRE(args, NKV_EINVAL, "scaled_decode: null arguments");
  const nkv_scaled_decode_args& g = *args;
  NKV_REQUIRE(g.batch >= 0 && g.n_blocks >= 0, NKV_EINVAL, "scaled_decode: bad sizes (batch=%lld)",
              (long long)g.batch);
  int rc = scaled_check("scaled_decode", g.k_cache, g.v_cache, g.n_kv_heads, g.head_dim);
  if (rc) return rc;
  rc = scaled_check_heads("scaled_decode", g.n_q_heads, g.n_kv_heads, kMaxGroup, g.scale);
  if (rc) return rc;
  if (g.batch == 0) return NKV_OK;
  rc = scaled_check_tables("scaled_decode", g.block_tables, g.bt_row_stride, g.max_blocks_per_seq,
                           g.block_size, g.n_blocks);
  if (rc) return rc;
  const int64_t row = g.n_q_heads * g.head_dim;
  NKV_REQUIRE(g.q && g.context_lens && g.out && aligned16(g.q) &&
                  (reinterpret_cast<uintptr_t>(g.out) & 3u) == 0,
              NKV_EINVAL, "scaled_decode: null or misaligned pointer");
  NKV_REQUIRE(g.q_row_stride >= row && g.q_row_stride % 8 == 0 && g.out_row_stride >= row &&
                  g.out_row_stride % 2 == 0,
              NKV_EINVAL, "scaled_decode: row strides must cover Hq*D, q's in multiples of 8, "
              "out's of 2");
  const int64_t max_tiles = g.max_blocks_per_seq * (g.block_size / kTileRows);
  NKV_REQUIRE(g.batch < (1ll << 30) / max_tiles, NKV_EUNSUPPORTED,
              "scaled_decode: too many tiles in one call");
  const int32_t batch = (int32_t)g.batch, Hq = (int32_t)g.n_q_heads, Hk = (int32_t)g.n_kv_heads,
                D = (int32_t)g.head_dim, B = (int32_t)g.block_size,
                width = (int32_t)g.max_blocks_per_seq;
  const int group = Hq / Hk, ncg = decode_ncg(group), np = Hk * ncg;
  // ranges of at least two tiles, and no more partials a row than the combine holds
  const int32_t min_tiles = decode_min_chunks(max_tiles, 2);
  const int resident = D == 64 ? scaled_decode_grid<64>() : scaled_decode_grid<128>();
  const int64_t waves = std::min<int64_t>(std::max(1, resident / np),
                                          decode_useful_waves(batch, width, B));
  const size_t desc_b = decode_desc_bytes(batch, np);
  const size_t need = desc_b + decode_part_bytes(waves, batch, Hq, D);
  NKV_REQUIRE(g.workspace && aligned16(g.workspace) && g.workspace_bytes >= (int64_t)need,
              NKV_EWORKSPACE, "scaled_decode: workspace needs %zu bytes, 16-byte aligned (got %lld)",
              need, (long long)g.workspace_bytes);
  NKV_REQUIRE((waves + batch) * Hq < (1ll << 31) && waves * np < (1ll << 31), NKV_EUNSUPPORTED,
              "scaled_decode: too many partial rows");
  i32x4v_t* desc = static_cast<i32x4v_t*>(g.workspace);
  float* part = reinterpret_cast<float*>(static_cast<char*>(g.workspace) + desc_b);
#define NKV_SCALED_DECODE(D)                                                                      \
  hipLaunchKernelGGL((scaled_decode_kernel<D>), dim3((unsigned)(waves * np)), dim3(64), 0,        \
                     as_stream(g.stream), (const bf16_t*)g.q, g.q_row_stride,                     \
                     (const char*)g.k_cache, (const char*)g.v_cache, g.block_tables,              \
                     g.bt_row_stride, g.context_lens, batch, Hk, group, ncg, B, width,            \
                     g.n_blocks, min_tiles, (float)g.scale * kLog2e, part, desc)
  if (D == 64) NKV_SCALED_DECODE(64);
  else NKV_SCALED_DECODE(128);
#undef NKV_SCALED_DECODE
  rc = check_launch("nkv_scaled_decode");
  if (rc) return rc;
  return nkv_paged_decode_combine(g.context_lens, batch, Hq, Hk, D, B, width, g.out,
                                  g.out_row_stride, g.workspace, (size_t)g.workspace_bytes,
                                  g.stream);
}
