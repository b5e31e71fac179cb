// Varlen causal attention over the block-scaled K/V cache (scaled_cache.h): prompts, chunks behind a
// prefix, drafts checked against their context.
//
// Reference: beside flash_attn_varlen_func(..., causal=True, block_table) at
// nanokvllm/layers/attention.py:96-102 (bottom-right causal alignment: query j of a sequence with Lq
// queries and Lk keys sees keys 0 .. Lk-Lq+j).
//   out_j = softmax(scale * q_j . K) V    over the keys that it sees, K and V = code * 2^e
//
// MI355X design (MFMA-bound). Workgroup = (sequence, tile of queries, KV head, part of the keys) x 4
// waves; a tile's rows are its queries for all G heads of the KV head (row r: query r / G, head r % G),
// 16 * RG of them a wave. Keys advance 64 a step, two tiles of the cache: each wave brings one tile's K
// or V codes into registers while the step before computes, widens them to bf16 with the tile's scale
// (exactly, v_cvt_scalef32_pk_bf16_fp8) and writes them to one of two LDS stages. Codes come in the
// lanes' order for the matrix instructions, so that the loads, the LDS writes and the LDS reads are all
// 1 KiB of consecutive bytes a wave: no swizzle, no transposing read, no bank conflict.
//   S^T = K q^T      v_mfma_f32_16x16x32_bf16, A = 16 keys from LDS, B = q in registers
//   O^T += V^T P^T   the same, A = 16 dims x 32 keys from LDS, B = the lane's own eight weights
// Where the tiles are fewer than the chip's workgroups the keys of each are cut into `parts` equal
// ranges, whose partial rows a second launch merges.
#include "launch_rules.h"
#include "scaled_cache.h"

#include <math.h>

#include <algorithm>
#include <type_traits>

namespace nkv {

constexpr int kStep = 64;      // keys a step
constexpr float kLazy = 8.f;   // log2 headroom before the running maximum is raised
constexpr int kMaxParts = 64;  // of a tile's keys
constexpr int prefill_part_row(int D) { return D + 4; }  // floats of a partial row: O, m, l, 2 pad

struct ScaledPrefillArgs {
  const bf16_t* q;
  int64_t q_row_stride;
  const char *k_cache, *v_cache;
  const int32_t *cu_q, *cu_k, *block_tables;
  int64_t bt_row_stride;
  int32_t Hk, G, block_size, max_blocks, n_blocks, n_seqs, n_tiles, parts;
  int64_t total_q;  // rows of q and out
  float scale_log2;
  bf16_t* out;
  int64_t out_row_stride;
  float* part;  // [row of q][query head][parts] partial rows
};

// Zeroes for NaN, and ones where there was one.
__device__ __forceinline__ u32x4_t split_nan(u32x4_t v, u32x4_t& ones) {
  u32x4_t clean;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const uint32_t lo = (v[w] & 0x7fffu) > 0x7f80u ? 0xffffu : 0u;
    const uint32_t hi = (v[w] & 0x7fff0000u) > 0x7f800000u ? 0xffff0000u : 0u;
    clean[w] = v[w] & ~(lo | hi);
    ones[w] = 0x3f803f80u & (lo | hi);
  }
  return clean;
}

template <int D, int RG>
__global__ __launch_bounds__(256, 2) void scaled_prefill_kernel(const ScaledPrefillArgs a) {
  constexpr int kI = D / 64;
  constexpr int kLoads = 2 * kI;          // 1 KiB loads of a cache tile's K, and of its V
  constexpr int kKs = D / 32;             // k-steps of S^T
  constexpr int kDb = D / 16;             // 16-dim blocks of O^T
  constexpr int kHalfB = kTileRows * D * 2;  // bytes of a cache tile's K or V in LDS
  constexpr int kStageB = 4 * kHalfB;     // K of two tiles, then V of two
  __shared__ __attribute__((aligned(1024))) char ring[2 * kStageB];
  __shared__ int nan_in[2][2];  // a stage's V tiles hold NaN (of steps that mask keys)

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g4 = lane >> 4;
  const int col = lane & 15;
  const int G = a.G, Hk = a.Hk;
  const int QT = 64 * RG / G;  // queries per tile

  const int kvh = blockIdx.x % Hk;
  int rest = blockIdx.x / Hk;
  const int z = rest % a.parts;
  rest /= a.parts;
  const int tile = a.n_tiles - 1 - rest % a.n_tiles;  // largest first
  const int seq = rest / a.n_tiles;
  const int q0 = a.cu_q[seq], Lq = a.cu_q[seq + 1] - q0;
  const int Lk = a.cu_k[seq + 1] - a.cu_k[seq];
  NKV_DBG(tid == 0 && tile == 0 && (Lq < 0 || Lk < 0 || Lq > Lk), NKV_DEBUG_LENGTH);
  const int j0 = tile * QT;
  if (j0 >= Lq || q0 < 0 || (int64_t)q0 + Lq > a.total_q) return;  // uniform
  const int diag = Lk - Lq;  // query j sees keys <= diag + j
  const int last_key = min(Lk - 1, diag + j0 + QT - 1);
  const int n_steps = last_key >= 0 ? last_key / kStep + 1 : 0;
  const int per = (n_steps + a.parts - 1) / a.parts;
  const int s_lo = min(z * per, n_steps), s_end = min(s_lo + per, n_steps);

  // ---- loads: wave w brings the codes of cache tile 2 s + w / 2, K (even w) or V
  const bool is_v = wave & 1;
  const int half = wave >> 1;
  const char* cache = is_v ? a.v_cache : a.k_cache;
  const int tiles_per_block = a.block_size / kTileRows;
  const int64_t tile_bytes = (int64_t)kTileRows * (Hk * D + kRowPad);
  const int code_off = kvh * (kTileRows * D) + lane * 16;
  const int scale_off = kTileRows * Hk * D + kvh;
  const int32_t* bt = a.block_tables + (int64_t)seq * a.bt_row_stride;
  int bt_base = 0, bt_lane = -1;  // lane i: entry bt_base + i of the table row
  auto load_window = [&]() {
    const int e = bt_base + lane;
    const int id = e < a.max_blocks ? bt[e] : -1;
    NKV_DBG((int64_t)e * a.block_size < Lk && (e >= a.max_blocks || id < 0 || id >= a.n_blocks),
            e >= a.max_blocks ? NKV_DEBUG_LENGTH : NKV_DEBUG_BLOCK);
    bt_lane = (id >= 0 && id < a.n_blocks) ? id : -1;
  };
  int c_blk = (2 * s_lo + half) / tiles_per_block;  // block and tile in it of the step loaded next
  int c_in = (2 * s_lo + half) % tiles_per_block;
  bt_base = c_blk & ~63;
  load_window();
  u32x4_t code[kLoads];
  int scale_in = 0;
  auto issue = [&](int s) __attribute__((always_inline)) {
    const int n = s < s_end ? min(Lk - (2 * s + half) * kTileRows, kTileRows) : 0;
    const int pb = __builtin_amdgcn_readlane(bt_lane, c_blk - bt_base);
    const bool ok = n > 0 && pb >= 0;  // else zeros
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
        (void*)(cache + (ok ? (int64_t)pb * tiles_per_block + c_in : 0) * tile_bytes), (short)0,
        ok ? (uint32_t)tile_bytes : 0u, kBufferFlags);
    scale_in = (int)__builtin_amdgcn_raw_buffer_load_b8(r, scale_off, 0, 0);
#pragma unroll
    for (int p = 0; p < kLoads; ++p)
      code[p] = __builtin_bit_cast(
          u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(r, code_off + p * 1024, 0, 0));
    c_in += 2;
    while (c_in >= tiles_per_block) {  // at most twice: blocks of one tile
      c_in -= tiles_per_block;
      ++c_blk;
    }
    if (c_blk - bt_base >= 64) {  // uniform
      bt_base = c_blk & ~63;
      load_window();
    }
  };
  // a step masks keys of some row (uniform)
  auto is_edge = [&](int s) { return s * kStep + kStep - 1 > diag + j0 || s * kStep + kStep > Lk; };
  // the codes of the last issue(), step s's, widened into a stage
  auto commit = [&](int s, int stage) __attribute__((always_inline)) {
    char* at = ring + stage * kStageB + (is_v ? 2 * kHalfB : 0) + half * kHalfB + lane * 16;
    const float scale = scale_of(stored_scale(scale_in));
    if (is_v) {
      const int n = Lk - (2 * s + half) * kTileRows;
      if (n < kTileRows) {
        // codes behind the end may be anything, NaN too: a zero weight would not hide them
        const int m = min(max(n - 8 * g4, 0), 8);
        const uint64_t keep = m >= 8 ? ~0ull : (1ull << (8 * m)) - 1;
#pragma unroll
        for (int p = 0; p < kLoads; ++p) {
          code[p][0] &= (uint32_t)keep;
          code[p][1] &= (uint32_t)(keep >> 32);
          code[p][2] &= (uint32_t)keep;
          code[p][3] &= (uint32_t)(keep >> 32);
        }
      }
      if (is_edge(s)) {
        uint32_t found = 0;  // bytes x111 1111
#pragma unroll
        for (int p = 0; p < kLoads; ++p)
#pragma unroll
          for (int w = 0; w < 4; ++w) found |= ((code[p][w] & 0x7f7f7f7fu) + 0x01010101u);
        const bool any = __ballot((found & 0x80808080u) != 0) != 0;
        if (lane == 0) nan_in[stage][half] = any;
      }
    }
#pragma unroll
    for (int p = 0; p < kLoads; ++p) {
      *reinterpret_cast<u32x4_t*>(at + p * 2048) = codes_to_bf16(code[p][0], code[p][1], scale);
      *reinterpret_cast<u32x4_t*>(at + p * 2048 + 1024) =
          codes_to_bf16(code[p][2], code[p][3], scale);
    }
  };

  // ---- this wave's row groups: head and query of this lane's row (rows past the tile's queries
  // take query Lq: attended like the others, never stored)
  const bool idle = wave * (16 * RG) >= min(QT, Lq - j0) * G;  // only brings its share of the codes
  int head[RG], jrow[RG];
  u32x4_t qreg[RG][kKs];
  f32x4_t acc[RG][kDb];  // O^T: lane l -> row l%16, dims 16*db + 4*(l/16) .. +3
  float m_run[RG], l_run[RG], mb[RG];  // mb: m_run, or 0 while the row has seen no key
#pragma unroll
  for (int rr = 0; rr < RG; ++rr) {
    const int r = (wave * RG + rr) * 16 + col;
    const bool real = r < QT * G;
    head[rr] = real ? r % G : 0;
    jrow[rr] = real ? j0 + r / G : Lq;
    const int jc = jrow[rr] < Lq ? jrow[rr] : j0;
    const u32x4_t* qp = reinterpret_cast<const u32x4_t*>(
        a.q + (int64_t)(q0 + jc) * a.q_row_stride + (int64_t)(kvh * G + head[rr]) * D + g4 * 16);
#pragma unroll
    for (int i = 0; i < kI; ++i) {
      qreg[rr][2 * i] = qp[8 * i];
      qreg[rr][2 * i + 1] = qp[8 * i + 1];
    }
#pragma unroll
    for (int db = 0; db < kDb; ++db) acc[rr][db] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    m_run[rr] = -INFINITY;
    l_run[rr] = 0.f;
    mb[rr] = 0.f;
  }

  auto compute = [&](int s, int stage) __attribute__((always_inline)) {
    const char* kt = ring + stage * kStageB + lane * 16;
    const char* vt = kt + 2 * kHalfB;
    // S^T of quarter h: tokens 32 (h / 2) + 8 g4 + 4 (h % 2) + 0..3 of the step
    float sv[RG][16];
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      u32x4_t ka[kKs];
#pragma unroll
      for (int ks = 0; ks < kKs; ++ks)
        ka[ks] = *reinterpret_cast<const u32x4_t*>(kt + (h * kKs + ks) * 1024);
#pragma unroll
      for (int rr = 0; rr < RG; ++rr) {
        f32x4_t x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < kKs; ++ks) x = mfma_16x16x32<false>(ka[ks], qreg[rr][ks], x);
#pragma unroll
        for (int r = 0; r < 4; ++r) sv[rr][4 * h + r] = x[r];
      }
    }
    const bool edge = is_edge(s);
    int lim[RG];  // last key that the row sees, from the lane's first of the step on
#pragma unroll
    for (int rr = 0; rr < RG; ++rr) lim[rr] = min(diag + jrow[rr], Lk - 1) - s * kStep - 8 * g4;
    if (edge) {
#pragma unroll
      for (int rr = 0; rr < RG; ++rr)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if ((e >> 3) * kTileRows + (e & 7) > lim[rr]) sv[rr][e] = -INFINITY;
    }
    // the maxima are only raised where a row's exceeds its running one by kLazy
    float top[RG];
    bool raise_any = false;
#pragma unroll
    for (int rr = 0; rr < RG; ++rr) {
      const float* v = sv[rr];
      top[rr] = fmax3(fmax3(fmax3(v[0], v[1], v[2]), fmax3(v[3], v[4], v[5]),
                            fmax3(v[6], v[7], v[8])),
                      fmax3(v[9], v[10], v[11]), fmax3(fmax3(v[12], v[13], v[14]), v[15], -INFINITY));
      raise_any = raise_any || top[rr] * a.scale_log2 > m_run[rr] + kLazy;
    }
    if (__builtin_amdgcn_ballot_w64(raise_any) != 0) {
#pragma unroll
      for (int rr = 0; rr < RG; ++rr) {
        const float cm = col_max4(top[rr]) * a.scale_log2;
        const bool raise = cm > m_run[rr] + kLazy;
        const float alpha = raise ? fast_exp2(m_run[rr] - cm) : 1.f;  // exp2(-inf) = 0
        m_run[rr] = raise ? cm : m_run[rr];
        mb[rr] = m_run[rr] == -INFINITY ? 0.f : m_run[rr];
        l_run[rr] *= alpha;
#pragma unroll
        for (int db = 0; db < kDb; ++db) acc[rr][db] *= alpha;
      }
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      u32x4_t pb[RG];
#pragma unroll
      for (int rr = 0; rr < RG; ++rr) {
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
          p[e] = fast_exp2(fmaf(sv[rr][8 * c + e], a.scale_log2, -mb[rr]));
        pb[rr] = u32x4_t{cvt_pk16<false>(p[0], p[1]), cvt_pk16<false>(p[2], p[3]),
                         cvt_pk16<false>(p[4], p[5]), cvt_pk16<false>(p[6], p[7])};
        // the sum is that of the rounded weights, which multiply V
#pragma unroll
        for (int e = 0; e < 4; ++e) l_run[rr] = sum2_16<false>(pb[rr][e], l_run[rr]);
      }
      if (edge && nan_in[stage][c]) {  // uniform, rare
        // rows that do not see a key must not see its NaN: count those that each row sees
#pragma unroll
        for (int db = 0; db < kDb; ++db) {
          u32x4_t ones;
          const u32x4_t va = split_nan(
              *reinterpret_cast<const u32x4_t*>(vt + (c * kDb + db) * 1024), ones);
#pragma unroll
          for (int rr = 0; rr < RG; ++rr) {
            u32x4_t seen;
#pragma unroll
            for (int w = 0; w < 4; ++w)
              seen[w] = (c * kTileRows + 2 * w <= lim[rr] ? 0x3f80u : 0u) |
                        (c * kTileRows + 2 * w + 1 <= lim[rr] ? 0x3f800000u : 0u);
            const f32x4_t n = mfma_16x16x32<false>(ones, seen, f32x4_t{0.f, 0.f, 0.f, 0.f});
            acc[rr][db] = mfma_16x16x32<false>(va, pb[rr], acc[rr][db]);
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[rr][db][r] = n[r] > 0.f ? NAN : acc[rr][db][r];
          }
        }
        continue;
      }
#pragma unroll
      for (int db = 0; db < kDb; ++db) {
        const u32x4_t va = *reinterpret_cast<const u32x4_t*>(vt + (c * kDb + db) * 1024);
#pragma unroll
        for (int rr = 0; rr < RG; ++rr)
          acc[rr][db] = mfma_16x16x32<false>(va, pb[rr], acc[rr][db]);
      }
    }
  };

  if (s_lo < s_end) {
    issue(s_lo);
    commit(s_lo, 0);
    __syncthreads();
    auto step = [&](int s, auto st) {
      constexpr int kStage = decltype(st)::value;
      issue(s + 1);
      if (!idle) compute(s, kStage);
      if (s + 1 < s_end) commit(s + 1, 1 - kStage);
      __syncthreads();
    };
    for (int s = s_lo;;) {
      step(s, std::integral_constant<int, 0>{});
      if (++s >= s_end) break;
      step(s, std::integral_constant<int, 1>{});
      if (++s >= s_end) break;
    }
  }
  if (idle) return;

#pragma unroll
  for (int rr = 0; rr < RG; ++rr) {
    const float l = col_sum4(l_run[rr]);
    if (jrow[rr] >= Lq) continue;
    const int64_t row = q0 + jrow[rr];
    const int h = kvh * G + head[rr];
    if (a.parts > 1) {
      float* pr = a.part + ((row * (Hk * G) + h) * a.parts + z) * prefill_part_row(D);
#pragma unroll
      for (int db = 0; db < kDb; ++db)
        *reinterpret_cast<f32x4_t*>(pr + db * 16 + g4 * 4) = acc[rr][db];
      if (g4 == 0) *reinterpret_cast<float2*>(pr + D) = float2{m_run[rr], l};
      continue;
    }
    const float inv = l != 0.f ? 1.f / l : 0.f;
    bf16_t* op = a.out + row * a.out_row_stride + (int64_t)h * D + g4 * 4;
#pragma unroll
    for (int db = 0; db < kDb; ++db)
      *reinterpret_cast<uint2*>(op + db * 16) =
          uint2{cvt_pk16<false>(acc[rr][db][0] * inv, acc[rr][db][1] * inv),
                cvt_pk16<false>(acc[rr][db][2] * inv, acc[rr][db][3] * inv)};
  }
}

// One wave per (row of q, query head): its partials merged.
template <int D>
__global__ __launch_bounds__(256) void scaled_merge_kernel(const ScaledPrefillArgs a,
                                                           int32_t max_rows) {
  constexpr int N = D / 64;
  const int lane = threadIdx.x & 63;
  const int Hq = a.Hk * a.G;
  const int64_t unit =
      (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int64_t row = unit / Hq;
  if (row >= a.total_q) return;
  const int h = (int)(unit - row * Hq);
  // rows of no sequence, and those past the tiles that were launched, are left as they are
  bool mine = false;
  for (int s = lane; s < a.n_seqs; s += 64) {
    const int b = a.cu_q[s], e = a.cu_q[s + 1];
    mine = mine || (b >= 0 && row >= b && row < e && e <= a.total_q && row - b < max_rows);
  }
  if (__ballot(mine) == 0) return;
  const float* p = a.part + (row * Hq + h) * a.parts * prefill_part_row(D);
  float2 ml = {-INFINITY, 0.f};
  if (lane < a.parts) ml = *reinterpret_cast<const float2*>(p + lane * prefill_part_row(D) + D);
  const float M = wave_max(ml.x);
  const float w = ml.x == -INFINITY && ml.y == 0.f ? 0.f : fast_exp2(ml.x - M);
  const float L = wave_sum(w * ml.y);
  float o[N] = {};
  for (int z = 0; z < a.parts; ++z) {
    const float wz = __shfl(w, z, 64);
    float v[N];
    load_dims<N>(p + z * prefill_part_row(D) + N * lane, v);
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = fmaf(wz, v[i], o[i]);
  }
  store_dims<N, false>(a.out + row * a.out_row_stride + (int64_t)h * D + N * lane, o,
                       L != 0.f ? 1.f / L : 0.f);
}

struct ScaledPrefillPlan {
  int groups, parts;
};
static ScaledPrefillPlan scaled_prefill_plan(int64_t n_seqs, int64_t total_q, int64_t max_q,
                                             int64_t max_k, int32_t Hk, int g) {
  ScaledPrefillPlan p;
  const int cus = device_cus();
  p.groups = plain_groups(n_seqs, total_q, max_q, Hk, g, 2, cus);
  const BatchMix m = batch_mix(n_seqs, total_q, max_q);
  const int64_t qt = 64 * p.groups / g;
  const int64_t tiles =
      std::min(m.prompts * ((max_q + qt - 1) / qt), m.prompt_rows / qt + m.prompts) + m.rows;
  const int64_t steps = (max_k + kStep - 1) / kStep;
  p.parts = (int)std::max<int64_t>(
      1, std::min<int64_t>({2 * cus / std::max<int64_t>(1, tiles * Hk), steps / 4, kMaxParts}));
  return p;
}

}  // namespace nkv

extern "C" size_t nkv_scaled_prefill_workspace_bytes(int32_t n_seqs, int64_t total_q,
                                                     int64_t max_seqlen_q, int64_t max_seqlen_k,
                                                     int32_t n_q_heads, int32_t n_kv_heads,
                                                     int32_t head_dim) {
  using namespace nkv;
  if (n_seqs <= 0 || total_q <= 0 || max_seqlen_q <= 0 || n_kv_heads <= 0 ||
      n_q_heads % n_kv_heads != 0 || n_q_heads / n_kv_heads <= 0 ||
      n_q_heads / n_kv_heads > NKV_SCALED_MAX_GROUP || !scaled_dim_ok(head_dim))
    return 0;
  const ScaledPrefillPlan p = scaled_prefill_plan(n_seqs, total_q, max_seqlen_q, max_seqlen_k,
                                                  n_kv_heads, n_q_heads / n_kv_heads);
  if (p.parts == 1) return 0;
  return (size_t)total_q * n_q_heads * p.parts * prefill_part_row(head_dim) * sizeof(float);
}

extern "C" int nkv_scaled_prefill(const void* q, int64_t q_row_stride, int64_t total_q,
                                  const void* k_cache, const void* v_cache,
                                  const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k,
                                  const int32_t* block_tables, int64_t bt_row_stride,
                                  int32_t max_blocks_per_seq, int32_t n_seqs, int64_t max_seqlen_q,
                                  int64_t max_seqlen_k, int32_t n_q_heads, int32_t n_kv_heads,
                                  int32_t head_dim, int32_t block_size, int64_t n_blocks,
                                  float scale, void* out, int64_t out_row_stride, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  using namespace nkv;
  clear_error();
  NKV_REQUIRE(n_seqs >= 0 && total_q >= 0 && total_q < (1ll << 31) && max_seqlen_q >= 0 &&
                  n_q_heads > 0 && n_kv_heads > 0 && n_blocks >= 0,
              NKV_EINVAL, "scaled_prefill: bad sizes (%d sequences, %lld rows, Hq=%d, Hk=%d)",
              n_seqs, (long long)total_q, n_q_heads, n_kv_heads);
  NKV_REQUIRE(n_q_heads % n_kv_heads == 0, NKV_EINVAL,
              "scaled_prefill: n_q_heads %% n_kv_heads != 0 (%d, %d)", n_q_heads, n_kv_heads);
  const int g = n_q_heads / n_kv_heads;
  NKV_REQUIRE(g <= NKV_SCALED_MAX_GROUP, NKV_EUNSUPPORTED, "scaled_prefill: GQA group %d above %d",
              g, NKV_SCALED_MAX_GROUP);
  int rc = scaled_check("scaled_prefill", k_cache, v_cache, n_kv_heads, head_dim);
  if (rc) return rc;
  NKV_REQUIRE(block_size > 0 && block_size % kTileRows == 0, NKV_EUNSUPPORTED,
              "scaled_prefill: block_size must be a multiple of %d (got %d)", kTileRows,
              block_size);
  NKV_REQUIRE(max_blocks_per_seq > 0 && bt_row_stride >= max_blocks_per_seq, NKV_EINVAL,
              "scaled_prefill: bad block table width/stride (%d, %lld)", max_blocks_per_seq,
              (long long)bt_row_stride);
  NKV_REQUIRE(n_blocks < (1ll << 31) && max_blocks_per_seq <= INT32_MAX / block_size,
              NKV_EUNSUPPORTED, "scaled_prefill: blocks and lengths must fit 32 bits");
  NKV_REQUIRE(scale > 0.f && isfinite(scale), NKV_EINVAL,
              "scaled_prefill: scale must be finite and > 0");
  if (n_seqs == 0 || total_q == 0 || max_seqlen_q == 0) return NKV_OK;
  const int64_t row = (int64_t)n_q_heads * head_dim;
  NKV_REQUIRE(q && cu_seqlens_q && cu_seqlens_k && block_tables && out && aligned16(q) &&
                  (reinterpret_cast<uintptr_t>(out) & 7u) == 0,
              NKV_EINVAL, "scaled_prefill: null or misaligned pointer");
  NKV_REQUIRE(q_row_stride >= row && q_row_stride % 8 == 0 && out_row_stride >= row &&
                  out_row_stride % 4 == 0,
              NKV_EINVAL, "scaled_prefill: row strides must cover Hq*D, q's in multiples of 8, "
              "out's of 4");
  ScaledPrefillPlan p =
      scaled_prefill_plan(n_seqs, total_q, max_seqlen_q, workspace ? max_seqlen_k : 0, n_kv_heads, g);
  if (p.parts > 1) {
    const size_t need =
        (size_t)total_q * n_q_heads * p.parts * prefill_part_row(head_dim) * sizeof(float);
    NKV_REQUIRE(aligned16(workspace) && workspace_bytes >= need, NKV_EWORKSPACE,
                "scaled_prefill: workspace needs %zu bytes, 16-byte aligned (got %zu)", need,
                workspace_bytes);
  }
  const int64_t qt = 64 * p.groups / g;
  const int64_t tiles = plain_tiles(n_seqs, max_seqlen_q, qt);
  const int64_t grid = n_seqs * tiles * n_kv_heads * p.parts;
  NKV_REQUIRE(tiles < (1ll << 31) && grid < (1ll << 31), NKV_EUNSUPPORTED,
              "scaled_prefill: too many tiles in one call");
  const ScaledPrefillArgs a{(const bf16_t*)q, q_row_stride, (const char*)k_cache,
                            (const char*)v_cache, cu_seqlens_q, cu_seqlens_k, block_tables,
                            bt_row_stride, n_kv_heads, g, block_size, max_blocks_per_seq,
                            (int32_t)n_blocks, n_seqs, (int32_t)tiles, p.parts, total_q,
                            scale * kLog2e,
                            (bf16_t*)out, out_row_stride, (float*)workspace};
#define NKV_SCALED_PREFILL(D, RG)                                                          \
  hipLaunchKernelGGL((scaled_prefill_kernel<D, RG>), dim3((unsigned)grid), dim3(256), 0, \
                     as_stream(stream), a)
  if (head_dim == 64) {
    if (p.groups == 1) NKV_SCALED_PREFILL(64, 1);
    else NKV_SCALED_PREFILL(64, 2);
  } else {
    if (p.groups == 1) NKV_SCALED_PREFILL(128, 1);
    else NKV_SCALED_PREFILL(128, 2);
  }
#undef NKV_SCALED_PREFILL
  rc = check_launch("nkv_scaled_prefill");
  if (rc || p.parts == 1) return rc;
  const dim3 merge((unsigned)((total_q * n_q_heads + 3) / 4));
  const int32_t max_rows = (int32_t)std::min<int64_t>(tiles * qt, INT32_MAX);
  if (head_dim == 64)
    hipLaunchKernelGGL((scaled_merge_kernel<64>), merge, dim3(256), 0, as_stream(stream), a,
                       max_rows);
  else
    hipLaunchKernelGGL((scaled_merge_kernel<128>), merge, dim3(256), 0, as_stream(stream), a,
                       max_rows);
  return check_launch("nkv_scaled_prefill");
}
