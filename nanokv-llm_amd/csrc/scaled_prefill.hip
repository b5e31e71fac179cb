// Varlen causal attention over the block-scaled K/V cache (scaled_cache.h): prompts, chunks behind a
// prefix, drafts checked against their context.
//
// Reference: beside flash_attn_varlen_func(..., causal=True, block_table) at
// nanokvllm/layers/attention.py:96-102 (bottom-right causal alignment: query j of a sequence with Lq
// queries and Lk keys sees keys 0 .. Lk-Lq+j).
//   out_j = softmax(scale * q_j . K) V    over the keys that it sees, K and V = code * 2^e
//
// MI355X design (MFMA- and issue-bound). Workgroup = (sequence, tile of queries, KV head) x 4 waves; a
// tile's rows are its queries for all G heads of the KV head (row r: query r / G, head r % G), 16 * RG of
// them a wave. Keys advance 64 a step, two tiles of the cache. Each wave brings one tile's K or V codes
// straight into a ring of four steps in LDS (buffer_load ... lds, three steps ahead, one barrier a step)
// and every wave widens them to bf16 with the tile's scale as it reads them (exactly,
// v_cvt_scalef32_pk_bf16_fp8). Codes stand in memory in the lanes' order for the matrix instructions, so
// that the loads and the LDS reads are 1 KiB of consecutive bytes a wave: no swizzle, no transposing
// read, no bank conflict; and the ring holds a byte a value, half of what widened tiles would take.
//   S^T = K q^T      v_mfma_f32_16x16x32_bf16, A = 16 keys from LDS, B = q in registers
//   O^T += V^T P^T   the same, A = 16 dims x 32 keys from LDS, B = the lane's own eight weights
// Each wave widens for itself, so the more rows it has the less that counts: of 392 us (4 chunks of
// 1500 - 2048 behind up to 6000 keys, Hq 32, Hk 8, D 128, RG 2, q's products 104 us) K's widening took
// 35, V's 29 and the exponentials 34. RG 3 with the longest sequences first: 342 us, 1.01 PFLOP/s.
// Products of K's codes as they are (v_mfma_scale_f32_16x16x128_f8f6f4, q as the sum of two E4M3 codes)
// take as long in the matrix cores, and save only the widening: 341 us against 346, and 7.9 us against
// 7.1 for one prompt of 77, which q's taking apart costs; not taken.
//
// SPLIT: where few tiles would leave the chip idle, the workgroups that fit it at once take equal ranges
// of all the key steps, and a second launch merges the rows whose keys were cut. Units of few rows
// (single tokens, drafts) give a wave's rows to two waves, one for each cache tile of a step, joined in
// LDS at the unit's end: 2 chunks of 400 with 30 tokens behind up to 8000 keys (Hq 16, Hk 4, D 128) 91
// us against 109, 4 drafts behind 9000 - 30000 (Hq 32, Hk 8) 50 against 53 (46 now), of which the codes
// alone take 25.
#include "launch_rules.h"
#include "lds_tiles.h"
#include "scaled_cache.h"

#include <float.h>
#include <math.h>

#include <algorithm>
#include <type_traits>

namespace nkv {

constexpr int kStep = 64;      // keys a step
constexpr float kLazy = 8.f;   // log2 headroom before the running maximum is raised
constexpr int64_t kMostSeqs = 1 << 20, kMostRows = 1 << 30;  // the plan's products stay in 64 bits
constexpr int part_floats(int D) { return D + 4; }  // of a partial row: O, m, l, 2 pad

struct ScaledPrefillArgs {
  const bf16_t* q;
  int64_t q_row_stride;
  const char *k_cache, *v_cache;
  const int32_t *cu_q, *cu_k, *block_tables;
  int64_t bt_row_stride;
  int32_t Hk, G, block_size, max_blocks, n_blocks, n_seqs, n_tiles, sort;
  int64_t total_q;  // rows of q and out
  float scale_log2;
  bf16_t* out;
  int64_t out_row_stride;
  // split launches: what a workgroup's range left unfinished
  i32x4_t* desc;  // one per workgroup: {parts, first row of q, queries, KV head}
  float* part;    // two tiles of partial rows per workgroup
};

// A sequence's queries and keys; none where its rows are not all rows of q.
__device__ __forceinline__ void seq_lengths(const ScaledPrefillArgs& a, int s, int& q0, int& Lq,
                                            int& Lk) {
  q0 = a.cu_q[s];
  Lq = a.cu_q[s + 1] - q0;
  Lk = a.cu_k[s + 1] - a.cu_k[s];
  NKV_DBG(Lq < 0 || Lk < 0 || Lq > Lk, NKV_DEBUG_LENGTH);
  if (q0 < 0 || (int64_t)q0 + Lq > a.total_q) Lq = 0;
}

// The ranges of a split launch. The units of a KV head (sequence, tile) stand in one stream, a unit as
// long as its keys cost; range w is [w C, (w+1) C), a cut near a unit's end moved to that end. Every
// workgroup finds its own range from the lengths: the units' costs are series that sum in closed form.
struct Cursor {
  int seq, tile, q0, Lq, Lk;  // the current unit
  int u0;                     // its position in the stream
  int C, T, x, x_end;         // range length, stream length, the range's begin and end
};
constexpr int kSnap = 2;        // steps
// What a unit's start and end cost, counted before its first step. 0 / 2 / 3 / 4 / 6, us: drafts 50.5 /
// 48.3 / 47.9 / 47.5 / 47.7, 30 tokens and two chunks 36.8 / 34.8 / 34.5 / 34.4 / 36.0, 8 drafts behind
// up to 4000 29.3 / 27.0 / 27.0 / 26.3 / 26.1, 4 chunks of 128 63.6 / 59.4 / 60.1 / 59.8 / 62.1.
constexpr int kUnitSteps = 3;
constexpr int kLeastSteps = 4;  // shortest range
template <int RG>
__device__ __forceinline__ int key_cost(int rows) {
  return kStepBase + (rows + 16 * RG - 1) / (16 * RG);
}
__device__ __forceinline__ int tile_steps(int Lq, int Lk, int qt, int t) {
  const int last = Lk - Lq + min(Lq, (t + 1) * qt) - 1;
  return last >= 0 ? min(last, Lk - 1) / kStep + 1 : 1;  // an empty one is masked whole
}
// Keys of tile t as the stream counts them, and the cost of the tiles before tile t, all full.
__device__ __forceinline__ int tile_keys(int Lq, int Lk, int qt, int t) {
  return max(Lk - Lq, 0) + min(Lq, (t + 1) * qt) + kUnitSteps * kStep;
}
template <int RG>
__device__ __forceinline__ int cost_before(int Lq, int Lk, int qt, int t, int G) {
  return key_cost<RG>(qt * G) * (t * (max(Lk - Lq, 0) + kUnitSteps * kStep) + qt * (t * (t + 1) / 2));
}
template <int RG>
__device__ __forceinline__ bool split_begin(const ScaledPrefillArgs& a, int qt, Cursor& c) {
  const int lane = threadIdx.x & 63;
  int q0 = 0, Lq = 0, Lk = 0, cost = 0, incl = 0;
  const auto load = [&](int cb) {  // lane: sequence cb + lane
    Lq = Lk = cost = 0;
    if (cb + lane < a.n_seqs) seq_lengths(a, cb + lane, q0, Lq, Lk);
    if (Lq > 0) {
      const int t = (Lq - 1) / qt;
      cost = cost_before<RG>(Lq, Lk, qt, t, a.G) +
             tile_keys(Lq, Lk, qt, t) * key_cost<RG>((Lq - t * qt) * a.G);
    }
    incl = wave_incl_scan(cost);
    return __builtin_amdgcn_readlane(incl, 63);
  };
  c.T = 0;
  for (int cb = 0; cb < a.n_seqs; cb += 64) c.T += load(cb);
  const int ranges = (int)gridDim.x / a.Hk;
  c.C = max((c.T + ranges - 1) / ranges, kLeastSteps * kStep * kFullStep);
  c.x = (int)blockIdx.x / a.Hk * c.C;
  c.x_end = c.x + c.C;
  if (c.x >= c.T) return false;
  int base = 0, cb = 0;
  if (a.n_seqs > 64) load(0);
  for (int tot; c.x >= base + (tot = __builtin_amdgcn_readlane(incl, 63)); load(cb)) {
    base += tot;
    cb += 64;
    if (cb >= a.n_seqs) return false;
  }
  const int ln = __builtin_amdgcn_readfirstlane(__builtin_ctzll(__ballot(base + incl > c.x)));
  c.seq = cb + ln;
  c.q0 = __builtin_amdgcn_readlane(q0, ln);
  c.Lq = __builtin_amdgcn_readlane(Lq, ln);
  c.Lk = __builtin_amdgcn_readlane(Lk, ln);
  c.u0 = base + __builtin_amdgcn_readlane(incl - cost, ln);
  c.tile = -1;  // the last that begins at x or before
  for (int t0 = 0; t0 * qt < c.Lq; t0 += 64) {
    const int t = t0 + lane;
    c.tile += __builtin_popcountll(__ballot(
        t * qt < c.Lq && c.u0 + cost_before<RG>(c.Lq, c.Lk, qt, t, a.G) <= c.x));
  }
  c.tile = max(c.tile, 0);
  c.u0 += cost_before<RG>(c.Lq, c.Lk, qt, c.tile, a.G);
  return true;
}
// A whole launch's tile. Either every sequence has n_tiles places (few of them empty), or the tiles stand
// in line, a sequence's from its last (the longest) on: up to 64 sequences as they come or, if `sort`,
// the longest first; more at place cu_q[s] / qt + s, which leaves each room for its tiles and is found
// by trying 64 sequences at a time. A workgroup without a tile keeps its LDS from another for a few us:
// with as many places for each sequence as the longest needs, a chunk of 512 among 40 single tokens
// took 79 us where this takes 38, and four prompts of 512 among 60 95 and 41 (Hq 32, Hk 8, D 128).
__device__ __forceinline__ bool whole_begin(const ScaledPrefillArgs& a, int qt, Cursor& c) {
  const int lane = threadIdx.x & 63;
  int b = (int)blockIdx.x / a.Hk;
  if (a.n_tiles > 0) {
    c.seq = b / a.n_tiles;
    c.tile = a.n_tiles - 1 - b % a.n_tiles;
    seq_lengths(a, c.seq, c.q0, c.Lq, c.Lk);
    return c.tile * qt < c.Lq;
  }
  if (a.n_seqs > 64) {
    int lo = 0, step = 1;  // a sequence that stands at b or before; the last one is within 64 steps
    while ((int64_t)step * 64 < a.n_seqs) step *= 64;
    for (;; step /= 64) {
      const int s = (int)min((int64_t)lo + (int64_t)lane * step, (int64_t)a.n_seqs);
      const bool before = s < a.n_seqs && max(a.cu_q[s], 0) / qt + s <= b;
      lo += (__builtin_popcountll(__ballot(before) | 1) - 1) * step;
      if (step == 1) break;
    }
    c.seq = __builtin_amdgcn_readfirstlane(min(lo, a.n_seqs - 1));
    seq_lengths(a, c.seq, c.q0, c.Lq, c.Lk);
    c.tile = (c.Lq + qt - 1) / qt - 1 - (b - (c.q0 / qt + c.seq));
    return c.Lq > 0 && c.tile >= 0 && c.tile * qt < c.Lq;
  }
  int q0 = 0, Lq = 0, Lk = 0, before = 0;
  if (lane < a.n_seqs) seq_lengths(a, lane, q0, Lq, Lk);
  const int n = Lq > 0 ? (Lq + qt - 1) / qt : 0;
  if (a.sort) {
    for (int i = 0; i < a.n_seqs; ++i) {
      const int other = __builtin_amdgcn_readlane(Lk, i), tiles = __builtin_amdgcn_readlane(n, i);
      before += other > Lk || (other == Lk && i < lane) ? tiles : 0;
    }
  } else {
    before = wave_incl_scan(n) - n;
  }
  const uint64_t at = __ballot((uint32_t)(b - before) < (uint32_t)n);
  if (at == 0) return false;
  const int ln = __builtin_ctzll(at);
  c.seq = ln;
  c.q0 = __builtin_amdgcn_readlane(q0, ln);
  c.Lq = __builtin_amdgcn_readlane(Lq, ln);
  c.Lk = __builtin_amdgcn_readlane(Lk, ln);
  c.tile = __builtin_amdgcn_readlane(n - 1 + before, ln) - b;
  return true;
}
// The unit after the current one, which ends at u1 (false at the end of the stream).
__device__ __forceinline__ bool split_next(const ScaledPrefillArgs& a, int qt, int u1, Cursor& c) {
  c.u0 = u1;
  if (u1 >= c.T || u1 >= c.x_end) return false;
  if (++c.tile * qt < c.Lq) return true;
  c.tile = 0;
  do {
    if (++c.seq >= a.n_seqs) return false;
    seq_lengths(a, c.seq, c.q0, c.Lq, c.Lk);
  } while (c.Lq <= 0);
  return true;
}

// N KiB (16 bytes a lane each) from desc + code_off to consecutive LDS bytes at codes_at (an
// instruction's offset moves both addresses) and 256 bytes (4 a lane) from desc + scale_off to scales_at.
// Written as asm so that the compiler adds no wait for it before a barrier; the ring's own s_waitcnt does.
template <int N>
__device__ __forceinline__ void fetch_tile(i32x4_t desc, uint32_t codes_at, uint32_t code_off,
                                           uint32_t scales_at, uint32_t scale_off) {
  static_assert(N == 2 || N == 4, "a tile of codes");
  if constexpr (N == 2)
    asm volatile(NKV_LDS_AT
                 "buffer_load_dwordx4 %1, %2, 0 offen lds\n\t"
                 "buffer_load_dwordx4 %1, %2, 0 offen offset:0x400 lds\n\t"
                 "s_mov_b32 m0, %3\n\ts_nop 0\n\t"
                 "buffer_load_dword %4, %2, 0 offen lds"
                 :
                 : "s"(codes_at), "v"(code_off), "s"(desc), "s"(scales_at), "v"(scale_off)
                 : "memory", "m0");
  else
    asm volatile(NKV_LDS_AT
                 "buffer_load_dwordx4 %1, %2, 0 offen lds\n\t"
                 "buffer_load_dwordx4 %1, %2, 0 offen offset:0x400 lds\n\t"
                 "buffer_load_dwordx4 %1, %2, 0 offen offset:0x800 lds\n\t"
                 "buffer_load_dwordx4 %1, %2, 0 offen offset:0xc00 lds\n\t"
                 "s_mov_b32 m0, %3\n\ts_nop 0\n\t"
                 "buffer_load_dword %4, %2, 0 offen lds"
                 :
                 : "s"(codes_at), "v"(code_off), "s"(desc), "s"(scales_at), "v"(scale_off)
                 : "memory", "m0");
}

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

// A workgroup's tile, or (SPLIT) the units of its range. (RG 3 at head_dim 128 takes all 256 registers
// and spills four.)
template <int D, int RG, bool SPLIT>
__global__ __launch_bounds__(256, 2) void scaled_prefill_kernel(const ScaledPrefillArgs a) {
  constexpr int kI = D / 64;
  constexpr int kLoads = 2 * kI;           // 1 KiB loads of a cache tile's K, and of its V
  constexpr int kKs = D / 32;              // k-steps of S^T
  constexpr int kDb = D / 16;              // 16-dim blocks of O^T
  constexpr int kTileB = kTileRows * D;    // bytes of a head's codes of a cache tile
  constexpr int kCodesB = 4 * kTileB;      // of a step: K, V of the first cache tile, of the second
  constexpr int kStageB = kCodesB + 1024;  // and a word (64 copies) with the scale of each
  constexpr int kStages = 4;               // steps in LDS: one computed, three on their way
  __shared__ __attribute__((aligned(1024))) char ring[kStages * kStageB];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g4 = lane >> 4;
  const int col = lane & 15;
  const int G = a.G, Hk = a.Hk;
  const int QT = 64 * RG / G;  // queries per tile
  const int kvh = blockIdx.x % Hk;
  // loads: wave w brings the codes of cache tile 2 s + w / 2, K (even w) or V
  const int half = wave >> 1;
  const char* cache = (wave & 1) ? a.v_cache : a.k_cache;
  const int tiles_per_block = a.block_size / kTileRows;
  const int tile_bytes = kTileRows * (Hk * D + kRowPad);
  const uint32_t code_off = (uint32_t)(kvh * kTileB + lane * 16);
  const uint32_t scale_off = (uint32_t)(kTileRows * Hk * D + kvh);
  const uint32_t ring_at =
      (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)ring + (uint32_t)wave * kTileB;

  Cursor cur;
  if constexpr (SPLIT) {
    if (tid == 0) a.desc[blockIdx.x] = i32x4_t{0, 0, 0, 0};  // no unit cut at this range's end
    if (!split_begin<RG>(a, QT, cur)) return;                // uniform
  } else {
    if (!whole_begin(a, QT, cur)) return;  // uniform
  }
  int u1 = 0;        // the unit's end in the stream
  bool cut = false;  // the range ends inside the unit
  do {
  const auto uni = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
  const int q0 = uni(cur.q0), Lq = uni(cur.Lq), Lk = uni(cur.Lk);
  const int j0 = uni(cur.tile) * QT;
  const int diag = Lk - Lq;  // query j sees keys <= diag + j
  const int last_key = min(Lk - 1, diag + j0 + QT - 1);
  int s_lo = 0, s_end = last_key >= 0 ? last_key / kStep + 1 : 0;
  [[maybe_unused]] int lead = 0, snap = 0;
  if constexpr (SPLIT) {
    const int kc = key_cost<RG>(min(QT, Lq - j0) * G), sc = kStep * kc;
    lead = kUnitSteps * sc;
    snap = kSnap * sc;
    u1 = cur.u0 + tile_keys(Lq, Lk, QT, cur.tile) * kc;
    s_end = tile_steps(Lq, Lk, QT, cur.tile);
    cut = false;
    if (cur.x >= cur.u0 + lead + snap) {  // the range's begin lies in its first unit
      if (cur.x > u1 - snap) continue;  // which is the range's before (the condition steps on)
      s_lo = (cur.x - cur.u0 - lead + sc - 1) / sc;
    }
    if (cur.x_end < u1) {                     // the range ends within this unit
      if (cur.x_end < cur.u0 + lead + snap) return;  // which is the next range's
      cut = cur.x_end <= u1 - snap;
    }
    if (cut) s_end = min(s_end, (cur.x_end - cur.u0 - lead + sc - 1) / sc);
    // (within the tile also where lengths beyond the call's maxima have overflown the stream)
    s_end = uni(s_end);
    s_lo = max(min(uni(s_lo), s_end), 0);
  }

  // ---- this wave's row groups: head and query of this lane's row (rows past the tile's queries
  // take query Lq: attended like the others, never stored)
  const int rows = min(QT, Lq - j0) * G;
  // few rows: waves 0 and 1 attend to them in the even cache tiles, 2 and 3 in the odd ones
  const bool by_keys = SPLIT && rows <= 2 * (16 * RG);
  const int rwave = by_keys ? wave & 1 : wave;
  const bool idle = rwave * (16 * RG) >= rows;  // only brings its share of the codes
  int jrow[RG];
  u32x4_t qreg[RG][kKs];
#pragma unroll
  for (int rr = 0; rr < RG; ++rr) {
    const int r = (rwave * RG + rr) * 16 + col;
    const bool real = r < QT * G;
    const int head = real ? r % G : 0;
    jrow[rr] = real ? j0 + r / G : Lq;
    const int jc = jrow[rr] < Lq ? jrow[rr] : j0;
    const u32x4_t* qp = reinterpret_cast<const u32x4_t*>(
        a.q + (int64_t)(q0 + jc) * a.q_row_stride + (int64_t)(kvh * G + head) * D + g4 * 16);
#pragma unroll
    for (int i = 0; i < kI; ++i) {
      qreg[rr][2 * i] = qp[8 * i];
      qreg[rr][2 * i + 1] = qp[8 * i + 1];
    }
  }

  // ---- the ring
  const int32_t* bt = a.block_tables + (int64_t)uni(cur.seq) * a.bt_row_stride;
  int c_blk = (2 * s_lo + half) / tiles_per_block;  // block and tile in it of the step loaded next
  int c_in = (2 * s_lo + half) - c_blk * tiles_per_block;
  int c_left = min(Lk, s_end * kStep) - (2 * s_lo + half) * kTileRows;  // keys from there on
  int c_stage = 0;
  int bt_base = c_blk & ~63, bt_lane = -1;  // lane i: entry bt_base + i of the table row
  auto load_window = [&]() {
    const int e = bt_base + lane;
    const int id = e < a.max_blocks ? bt[e] : -1;
    NKV_DBG((int64_t)e * a.block_size < Lk && (e >= a.max_blocks || id < 0 || id >= a.n_blocks),
            e >= a.max_blocks ? NKV_DEBUG_LENGTH : NKV_DEBUG_BLOCK);
    bt_lane = (id >= 0 && id < a.n_blocks) ? id : -1;
  };
  load_window();
  auto issue = [&]() __attribute__((always_inline)) {
    const int pb = __builtin_amdgcn_readlane(bt_lane, c_blk - bt_base);
    const bool ok = c_left > 0 && pb >= 0;  // else zeros
    const int64_t at = ((int64_t)(ok ? pb : 0) * tiles_per_block + c_in) * tile_bytes;
    const i32x4_t desc = buffer_desc(cache + at, ok ? (uint32_t)tile_bytes : 0u);
    const uint32_t to = ring_at + (uint32_t)c_stage * kStageB;
    fetch_tile<kLoads>(desc, to, code_off, to - (uint32_t)wave * kTileB + kCodesB + wave * 256,
                       scale_off & ~3u);
    c_stage = c_stage + 1 == kStages ? 0 : c_stage + 1;
    c_left -= kStep;
    c_in += 2;  // at most two blocks on
    const int n = (c_in >= tiles_per_block) + (c_in >= 2 * tiles_per_block);
    c_in -= n * tiles_per_block;
    c_blk = uni(c_blk + n);
    if (c_blk - bt_base >= 64) {  // uniform; once per 64 blocks
      bt_base = c_blk & ~63;
      load_window();
    }
  };
  f32x4_t acc[RG][kDb];  // O^T: lane l -> row l%16, dims 16*db + 4*(l/16) .. +3
  float m_run[RG], l_run[RG];
#pragma unroll
  for (int rr = 0; rr < RG; ++rr) {
#pragma unroll
    for (int db = 0; db < kDb; ++db) acc[rr][db] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    m_run[rr] = -FLT_MAX;  // finite: a masked key's weight is exp2(-inf - m), 0, from the first on
    l_run[rr] = 0.f;
    // q is in registers before the ring's first loads: a wait for it later would wait for them too
#pragma unroll
    for (int ks = 0; ks < kKs; ++ks) asm volatile("" ::"v"(qreg[rr][ks]));
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the last unit's stores
#pragma unroll
  for (int st = 0; st < kStages - 1; ++st) issue();

  // NC cache tiles of step s, from tile t0 on
  auto compute = [&](int s, int stage, int t0, auto nc_c, auto edge_c)
                     __attribute__((always_inline)) {
    constexpr int NC = decltype(nc_c)::value;
    constexpr bool EDGE = decltype(edge_c)::value;
    const char* kt = ring + stage * kStageB + t0 * (2 * kTileB) + lane * 16;
    const char* st = ring + stage * kStageB + kCodesB + t0 * 512 + lane * 4;
    const int at = s * kStep + t0 * kTileRows + 8 * g4;  // the lane's first key
    float scale[2 * NC];  // K, V of each cache tile
#pragma unroll
    for (int w = 0; w < 2 * NC; ++w)
      scale[w] = scale_of(stored_scale(byte_of(
          uni((int)*reinterpret_cast<const uint32_t*>(st + w * 256)), (int)scale_off)));
    // S^T of half h of a tile: tokens 32 (h / 2) + 8 g4 + 4 (h % 2) + 0..3 from the first tile's on
    float sv[RG][8 * NC];
#pragma unroll
    for (int h = 0; h < 2 * NC; ++h) {
      u32x4_t ka[kKs];
#pragma unroll
      for (int i = 0; i < kI; ++i) {
        const u32x4_t c = *reinterpret_cast<const u32x4_t*>(
            kt + (h >> 1) * (2 * kTileB) + ((h & 1) * kI + i) * 1024);
        ka[2 * i] = codes_to_bf16(c[0], c[1], scale[h & 2]);
        ka[2 * i + 1] = codes_to_bf16(c[2], c[3], scale[h & 2]);
      }
#pragma unroll
      for (int rr = 0; rr < RG; ++rr) {
        f32x4_t x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < kKs; ++ks) x = mfma_16x16x32<false>(ka[ks], qreg[rr][ks], x);
#pragma unroll
        for (int r = 0; r < 4; ++r) sv[rr][4 * h + r] = x[r];
      }
    }
    [[maybe_unused]] int lim[RG];  // last key that the row sees, from the lane's first on
    if constexpr (EDGE) {
#pragma unroll
      for (int rr = 0; rr < RG; ++rr) {
        lim[rr] = min(diag + jrow[rr], Lk - 1) - at;
#pragma unroll
        for (int e = 0; e < 8 * NC; ++e)
          if ((e >> 3) * kTileRows + (e & 7) > lim[rr]) sv[rr][e] = -INFINITY;
      }
    }
    // the maxima are only raised where a row's exceeds its running one by kLazy
    float top[RG];
    bool raise_any = false;
#pragma unroll
    for (int rr = 0; rr < RG; ++rr) {
      const float* v = sv[rr];
      if constexpr (NC == 1)
        top[rr] = fmax3(fmax3(v[0], v[1], v[2]), fmax3(v[3], v[4], v[5]), fmaxf(v[6], v[7]));
      else
        top[rr] = fmax3(fmax3(fmax3(v[0], v[1], v[2]), fmax3(v[3], v[4], v[5]),
                              fmax3(v[6], v[7], v[8])),
                        fmax3(v[9], v[10], v[11]),
                        fmax3(fmax3(v[12], v[13], v[14]), v[15], -INFINITY));
      raise_any = raise_any || top[rr] * a.scale_log2 > m_run[rr] + kLazy;
    }
    if (__builtin_amdgcn_ballot_w64(raise_any) != 0) {
#pragma unroll
      for (int rr = 0; rr < RG; ++rr) {
        const float cm = col_max4(top[rr]) * a.scale_log2;
        const bool raise = cm > m_run[rr] + kLazy;
        const float alpha = raise ? fast_exp2(m_run[rr] - cm) : 1.f;
        m_run[rr] = raise ? cm : m_run[rr];
        l_run[rr] *= alpha;
#pragma unroll
        for (int db = 0; db < kDb; ++db) acc[rr][db] *= alpha;
      }
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      u32x4_t pb[RG];
#pragma unroll
      for (int rr = 0; rr < RG; ++rr) {
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
          p[e] = fast_exp2(fmaf(sv[rr][8 * c + e], a.scale_log2, -m_run[rr]));
        pb[rr] = u32x4_t{cvt_pk16<false>(p[0], p[1]), cvt_pk16<false>(p[2], p[3]),
                         cvt_pk16<false>(p[4], p[5]), cvt_pk16<false>(p[6], p[7])};
        // weights are rounded to bf16, as the product takes them (2^-8 of each at most); the sum is that
        // of the rounded ones, which multiply V
#pragma unroll
        for (int e = 0; e < 4; ++e) l_run[rr] = sum2_16<false>(pb[rr][e], l_run[rr]);
      }
      const char* vt = kt + kTileB + c * (2 * kTileB);
      if constexpr (EDGE) {
        // codes behind the end may be anything, NaN too, which a zero weight would not hide; and
        // rows that do not see a key must not see its NaN: those that each row sees are counted
        const int m = min(max(Lk - at - c * kTileRows, 0), 8);
        const uint32_t keep0 = m >= 4 ? ~0u : (1u << (8 * m)) - 1;
        const uint32_t keep1 = m >= 8 ? ~0u : m > 4 ? (1u << (8 * (m - 4))) - 1 : 0u;
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
          u32x4_t code = *reinterpret_cast<const u32x4_t*>(vt + j * 1024);
          code &= u32x4_t{keep0, keep1, keep0, keep1};
          uint32_t found = 0;  // bytes x111 1111
#pragma unroll
          for (int w = 0; w < 4; ++w) found |= (code[w] & 0x7f7f7f7fu) + 0x01010101u;
          const bool nan = __ballot((found & 0x80808080u) != 0) != 0;
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int db = 2 * j + u;
            u32x4_t va = codes_to_bf16(code[2 * u], code[2 * u + 1], scale[2 * c + 1]);
            if (nan) {  // uniform, rare
              u32x4_t ones;
              va = split_nan(va, ones);
#pragma unroll
              for (int rr = 0; rr < RG; ++rr) {
                u32x4_t seen;
#pragma unroll
                for (int w = 0; w < 4; ++w)
                  seen[w] = (c * kTileRows + 2 * w <= lim[rr] ? 0x3f80u : 0u) |
                            (c * kTileRows + 2 * w + 1 <= lim[rr] ? 0x3f800000u : 0u);
                const f32x4_t n = mfma_16x16x32<false>(ones, seen, f32x4_t{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[rr][db][r] = n[r] > 0.f ? NAN : acc[rr][db][r];
              }
            }
#pragma unroll
            for (int rr = 0; rr < RG; ++rr)
              acc[rr][db] = mfma_16x16x32<false>(va, pb[rr], acc[rr][db]);
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
          const u32x4_t code = *reinterpret_cast<const u32x4_t*>(vt + j * 1024);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const u32x4_t va = codes_to_bf16(code[2 * u], code[2 * u + 1], scale[2 * c + 1]);
#pragma unroll
            for (int rr = 0; rr < RG; ++rr)
              acc[rr][2 * j + u] = mfma_16x16x32<false>(va, pb[rr], acc[rr][2 * j + u]);
          }
        }
      }
    }
  };

  // steps from s_edge on mask keys of some row
  const int s_edge = max(0, min(diag + j0 + 1, Lk)) / kStep;
  int stage = 0;
  auto steps = [&](int t0, auto nc_c) __attribute__((always_inline)) {
    auto step = [&](int s, auto edge_c) __attribute__((always_inline)) {
      // this wave's loads of step s have landed, then everyone's have, and everyone is done with step
      // s - 1, whose stage takes the step kStages - 1 ahead
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"((kStages - 2) * (kLoads + 1)) : "memory");
      __syncthreads();
      issue();
      if (!idle) compute(s, stage, t0, nc_c, edge_c);
      stage = stage + 1 == kStages ? 0 : stage + 1;
    };
    int s = s_lo;
    for (; s < min(s_edge, s_end); ++s) step(s, std::integral_constant<bool, false>{});
    for (; s < s_end; ++s) step(s, std::integral_constant<bool, true>{});
  };
  if (by_keys) steps(wave >> 1, std::integral_constant<int, 1>{});
  else steps(0, std::integral_constant<int, 2>{});
  // no load into LDS outlives the workgroup, or meets the next unit's
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  if constexpr (SPLIT) {
    __syncthreads();
    if (by_keys) {  // the odd tiles' sums join the even ones'
      float* mine = reinterpret_cast<float*>(ring) + rwave * (RG * (kDb + 1) * 4 * 64) + lane * 4;
      if (wave >= 2 && !idle) {
#pragma unroll
        for (int rr = 0; rr < RG; ++rr) {
          float* x = mine + rr * ((kDb + 1) * 4 * 64);
#pragma unroll
          for (int db = 0; db < kDb; ++db) *reinterpret_cast<f32x4_t*>(x + db * 256) = acc[rr][db];
          *reinterpret_cast<float2*>(x + kDb * 256) = float2{m_run[rr], l_run[rr]};
        }
      }
      __syncthreads();
      if (wave < 2 && !idle) {
#pragma unroll
        for (int rr = 0; rr < RG; ++rr) {
          const float* x = mine + rr * ((kDb + 1) * 4 * 64);
          const float2 ml = *reinterpret_cast<const float2*>(x + kDb * 256);
          const float m = fmaxf(m_run[rr], ml.x);
          const float w0 = fast_exp2(m_run[rr] - m), w1 = fast_exp2(ml.x - m);
          m_run[rr] = m;
          l_run[rr] = l_run[rr] * w0 + ml.y * w1;
#pragma unroll
          for (int db = 0; db < kDb; ++db) {
            const f32x4_t o = *reinterpret_cast<const f32x4_t*>(x + db * 256);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[rr][db][e] = fmaf(o[e], w1, acc[rr][db][e] * w0);
          }
        }
      }
      __syncthreads();
      if (wave >= 2) continue;
    }
  }
  if (idle) continue;

  const bool part = SPLIT && (cut || s_lo > 0);
#pragma unroll
  for (int rr = 0; rr < RG; ++rr) {
    const float l = col_sum4(l_run[rr]);
    if (jrow[rr] >= Lq) continue;
    if constexpr (SPLIT) {
      if (part) {  // to one of two slots: the end of a unit begun before, or a unit's begin
        float* pr = a.part + (((int64_t)blockIdx.x * 2 + (s_lo == 0)) * (64 * RG) +
                              (rwave * RG + rr) * 16 + col) * part_floats(D);
#pragma unroll
        for (int db = 0; db < kDb; ++db)
          *reinterpret_cast<f32x4_t*>(pr + db * 16 + g4 * 4) = acc[rr][db];
        if (g4 == 0) *reinterpret_cast<float2*>(pr + D) = float2{m_run[rr], l};
        continue;
      }
    }
    const float inv = l != 0.f ? 1.f / l : 0.f;
    const int head = (rwave * RG + rr) * 16 + col - (jrow[rr] - j0) * G;
    bf16_t* op = a.out + (int64_t)(q0 + jrow[rr]) * a.out_row_stride +
                 (int64_t)(kvh * G + head) * D + g4 * 4;
#pragma unroll
    for (int db = 0; db < kDb; ++db)
      *reinterpret_cast<uint2*>(op + db * 16) =
          uint2{cvt_pk16<false>(acc[rr][db][0] * inv, acc[rr][db][1] * inv),
                cvt_pk16<false>(acc[rr][db][2] * inv, acc[rr][db][3] * inv)};
  }
  if constexpr (SPLIT) {
    if (part && s_lo == 0 && tid == 0) {  // the unit's first part: describe it to the merge
      const int w0 = (cur.u0 + lead + snap + cur.C - 1) / cur.C;  // the unit's first cut
      a.desc[blockIdx.x] =
          i32x4_t{(u1 - snap) / cur.C - w0 + 2, q0 + j0, min(QT, Lq - j0), kvh};
    }
  }
  } while (SPLIT && !cut && split_next(a, QT, u1, cur));
}

// Merges the parts of the units that ranges cut: descriptor x (of the workgroup that holds a unit's
// first part; part p > 0 is in the first slot of the workgroup p * Hk after it), four rows of its tile a
// wave, 16 lanes each. Lane c of a row owns dims 4 c + 64 i .. + 3, eight parts in flight. (A row a
// wave: 11 us where this takes 6, for the four times as many workgroups to hand out.)
template <int D>
__global__ __launch_bounds__(256) void scaled_merge_kernel(const ScaledPrefillArgs a,
                                                           int32_t tile_rows) {
  constexpr int kI = D / 64;
  constexpr int kInFlight = 8;
  const i32x4_t d = a.desc[blockIdx.x];
  const int r = blockIdx.y * 16 + (int)threadIdx.x / 16, c4 = (int)threadIdx.x % 16 * 4;
  if (d[0] < 2 || r >= d[2] * a.G) return;
  const int64_t tile = (int64_t)tile_rows * part_floats(D);
  const float* first = a.part + ((int64_t)blockIdx.x * 2 + 1) * tile + r * part_floats(D);
  const float* next = first - tile;  // + p * 2 * Hk tiles
  const int parts = min(d[0], (int)(gridDim.x - 1 - blockIdx.x) / a.Hk + 1);
  float M = -FLT_MAX, L = 0.f;
  f32x4_t o[kI] = {};
  for (int p0 = 0; p0 < parts; p0 += kInFlight) {
    float2 ml[kInFlight];
    f32x4_t v[kInFlight][kI];
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      const int p = min(p0 + u, parts - 1);
      const float* row = p == 0 ? first : next + (int64_t)p * 2 * a.Hk * tile;
      ml[u] = *reinterpret_cast<const float2*>(row + D);
#pragma unroll
      for (int i = 0; i < kI; ++i) v[u][i] = *reinterpret_cast<const f32x4_t*>(row + c4 + 64 * i);
    }
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      const float m = ml[u].x, l = ml[u].y;
      if (p0 + u >= parts) break;
      const float top = fmaxf(M, m);  // (finite, as each m is from the start)
      const float alpha = fast_exp2(M - top), w = fast_exp2(m - top);
      M = top;
      L = fmaf(w, l, L * alpha);
#pragma unroll
      for (int i = 0; i < kI; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] = fmaf(w, v[u][i][e], o[i][e] * alpha);
    }
  }
  const float inv = L != 0.f ? 1.f / L : 0.f;
  bf16_t* op = a.out + (int64_t)(d[1] + r / a.G) * a.out_row_stride +
               (int64_t)(d[3] * a.G + r % a.G) * D + c4;
#pragma unroll
  for (int i = 0; i < kI; ++i)
    *reinterpret_cast<uint2*>(op + 64 * i) =
        uint2{cvt_pk16<false>(o[i][0] * inv, o[i][1] * inv),
              cvt_pk16<false>(o[i][2] * inv, o[i][3] * inv)};
}

struct ScaledPrefillPlan {
  int groups;      // row groups a wave
  bool split;
  int64_t tiles;   // whole: places of a sequence (0: the tiles stand in line)
  bool sort;       // whole: sequences by length
  int64_t grid;    // workgroups
  size_t bytes(int D) const {  // of the workspace
    return split ? grid * (sizeof(i32x4_t) + 2 * 64 * groups * part_floats(D) * sizeof(float)) : 0;
  }
};
// How a call is launched, from its sizes alone.
//
// Split or whole. Whole, the longest tile sets the time, about 0.65 us a step of its own, and the chip is
// left idle in part; split, the steps are spread evenly, for about 8 us of ranges, partial rows and
// their merge (12 steps; 18 with two row groups). Tiles that the chip holds at once: split where the idle
// part is longer (tiles taken for three quarters of the longest). A few more than it holds make a
// second turn: where their prefixes make them as long as the first, split too; without prefixes, and
// with more tiles, the order by length fills the gaps. In graphs, whole / split, us (Hq 32, Hk 8, D 128
// but where noted):
//   1 draft of 8 behind 500 - 1000 / 2000 - 4000 / 8000 - 16000   16.7 / 16.7, 47.2 / 15.8, 170 / 25.9
//   8 drafts behind up to 1000 / 2000 / 4000                     21.2 / 16.8, 35.9 / 20.0, 63.8 / 27.3
//   32 behind up to 2000, 64 and 128 up to 4000                  37.3 / 35.0, 98 / 95, 183 / 175
//   1 chunk of 512 behind up to 4000 / 16000, of 1500 up to 6000  56.3 / 52.7, 179 / 124, 191 / 155
//   4 chunks of 128 / 256 / 300 behind up to 4000                89.8 / 60.2, 98.1 / 93.6, 94.7 / 80.3
//   8 chunks of 128 behind up to 2000 / 6000                     55.6 / 60.9, 126 / 115
//   a prompt of 1024 / 2048 / 4096                               23.0 / 34.8, 54.8 / 64.6, 141 / 169
//   2 chunks of 400 behind up to 1000 / 8000, 30 tokens (16, 4, 64)  22.8 / 26.7, 104 / 58.7
//   a chunk of 512 behind up to 1000 and 40 tokens, 8000 and 30  37.6 / 46.2, 142 / 117
//
// (Two points lie on the slower side: 128 drafts and four chunks of 256 go whole, 183 and 98.1.)
//
// Row groups a wave. More of them read, widen and wait for the keys less often; fewer fill the chip
// sooner. Whole, 1 / 2 / 3 groups, us (Hk 8; workgroups of one group):
//   512 (256)       13.8 / 18.4 / 24.9        4096 (2048)               172 / 143 / 145
//   1024 (512)      23.9 / 29.7 / 39.1        2 of 2048 + 4000 (2048)   371 / 284 / 315
//   2048 (1024)     56.9 / 55.7 / 70.7        8 of 1024 + 1000 (3600)   252 / 205 / 203
//     + 6000        254 / 207 / 262           8192 (4096)               623 / 483 / 456
// At head_dim 64 (four workgroups of one group to a CU, three of two, two of three) 1 / 2 / 3 / 4:
//   1024 (512)      17.1 / 21.6 / 27.1 / 32.1     4096 (2048)   97 / 92 / 99 / 111
//   2048 (1024)     35.9 / 39.2 / 48.6 / 56.8     8192 (4096)   357 / 297 / 304 / 300
// Split, two groups cost less where the tiles are many: 4 chunks of 128 66.3 / 59.5, 1 of 512 behind
// 16000 154 / 122, but 2 of 64 30.5 / 33.6 and 4 drafts 48.3 / 50.9.
//
// Order. Workgroups are handed out in turn, the last of them ends alone: longest sequences first, tiles
// from the last, 342 us for the chunks above and 430 as they come. (Tiles of all sequences in turn: 620,
// since their keys do not fit the L2 together.)
static ScaledPrefillPlan scaled_prefill_plan(int64_t n_seqs, int64_t total_q, int64_t max_q,
                                             int64_t max_k, int32_t Hk, int g, int D) {
  const int cus = device_cus();
  max_q = std::min(max_q, total_q);  // no sequence has more
  max_k = std::min<int64_t>(std::max<int64_t>(max_k, 0), INT32_MAX);
  const BatchMix m = batch_mix(n_seqs, total_q, max_q);
  const auto queries = [&](int groups) -> int64_t { return 64 * groups / g; };  // of a tile
  const auto tiles = [&](int groups) -> int64_t {  // that hold queries
    const int64_t qt = queries(groups);
    return std::min(m.prompts * ((max_q + qt - 1) / qt), m.prompt_rows / qt + m.prompts) + m.rows;
  };
  // workgroups that are resident at once: by the ring's LDS (69 KiB, 36 at head_dim 64), or registers
  const auto resident = [&](int groups) { return cus * (D == 128 ? 2 : groups == 1 ? 4 : 3); };
  const int least = g > 64 ? 2 : 1;
  ScaledPrefillPlan p;
  p.groups = least;
  const int64_t size = std::min<int64_t>(tiles(least) * Hk, INT32_MAX);
  const int64_t steps = (max_k + kStep - 1) / kStep;
  const int64_t prefix = max_k > max_q ? (max_k - max_q) / kStep : 0, chip = resident(least);
  const bool many = size >= cus / 2 && max_q * g > 64;
  p.split = size <= chip ? 4 * (steps - (many ? 18 : 12)) * chip > 3 * size * steps
                         : 2 * size <= 3 * chip && (2 * chip - size) * prefix > 24 * chip;
  if (p.split) {
    if (many) p.groups = 2;
  } else {
    if (2 * size > 3 * resident(1)) p.groups = 2;
    if (D == 128 && p.groups == 2 && 7 * queries(2) <= 5 * queries(3) &&
        2 * tiles(2) * Hk > 5 * resident(2))
      p.groups = 3;
  }
  const int64_t qt = queries(p.groups);
  const int64_t most = std::min(n_seqs * ((max_q + qt - 1) / qt), total_q / qt + n_seqs);
  if (p.split)
    // (a tile's keys are its queries' at least, in a sequence of fewer keys too)
    p.split = resident(p.groups) >= Hk &&
              key_split_fits(most, std::max(max_k, max_q) + kUnitSteps * kStep);
  const int64_t each = plain_tiles(n_seqs, max_q, qt), line = n_seqs > 64 ? total_q / qt + n_seqs : most;
  p.sort = !p.split && n_seqs > 1 && n_seqs <= 64 && most * Hk > resident(p.groups);
  p.tiles = !p.split && !p.sort && n_seqs * each <= line ? each : 0;
  p.grid = (p.split ? resident(p.groups) / Hk : p.tiles > 0 ? n_seqs * each : line) * Hk;
  return p;
}

}  // namespace nkv

extern "C" size_t nkv_scaled_prefill_workspace_bytes(int32_t n_seqs, int64_t total_q,
                                                     int64_t max_seqlen_q, int64_t max_seqlen_k,
                                                     int32_t n_q_heads, int32_t n_kv_heads,
                                                     int32_t head_dim) {
  using namespace nkv;
  if (n_seqs <= 0 || n_seqs > kMostSeqs || total_q <= 0 || total_q > kMostRows ||
      max_seqlen_q <= 0 || n_kv_heads <= 0 || n_kv_heads > NKV_SCALED_MAX_HEADS ||
      n_q_heads % n_kv_heads != 0 || n_q_heads / n_kv_heads <= 0 ||
      n_q_heads / n_kv_heads > NKV_SCALED_MAX_GROUP || !scaled_dim_ok(head_dim))
    return 0;
  const ScaledPrefillPlan p = scaled_prefill_plan(n_seqs, total_q, max_seqlen_q, max_seqlen_k,
                                                  n_kv_heads, n_q_heads / n_kv_heads, head_dim);
  return p.bytes(head_dim);
}

extern "C" int nkv_scaled_prefill(const nkv_scaled_prefill_args* args) {
  using namespace nkv;
  clear_error();
  NKV_REQUIRE(args, NKV_EINVAL, "scaled_prefill: null arguments");
  const nkv_scaled_prefill_args& g = *args;
  NKV_REQUIRE(g.n_seqs <= kMostSeqs, NKV_EUNSUPPORTED, "scaled_prefill: too many sequences (%lld)",
              (long long)g.n_seqs);
  NKV_REQUIRE(g.n_seqs >= 0 && g.total_q >= 0 && g.total_q <= kMostRows &&
                  g.max_seqlen_q >= 0 && g.n_blocks >= 0,
              NKV_EINVAL, "scaled_prefill: bad sizes (%lld sequences, %lld rows)",
              (long long)g.n_seqs, (long long)g.total_q);
  int rc = scaled_check("scaled_prefill", g.k_cache, g.v_cache, g.n_kv_heads, g.head_dim);
  if (rc) return rc;
  rc = scaled_check_heads("scaled_prefill", g.n_q_heads, g.n_kv_heads, NKV_SCALED_MAX_GROUP, g.scale);
  if (rc) return rc;
  if (g.n_seqs == 0 || g.total_q == 0 || g.max_seqlen_q == 0) return NKV_OK;
  rc = scaled_check_tables("scaled_prefill", g.block_tables, g.bt_row_stride, g.max_blocks_per_seq,
                           g.block_size, g.n_blocks);
  if (rc) return rc;
  const int64_t row = g.n_q_heads * g.head_dim;
  NKV_REQUIRE(g.q && g.cu_seqlens_q && g.cu_seqlens_k && g.out && aligned16(g.q) &&
                  (reinterpret_cast<uintptr_t>(g.out) & 7u) == 0,
              NKV_EINVAL, "scaled_prefill: null or misaligned pointer");
  NKV_REQUIRE(g.q_row_stride >= row && g.q_row_stride % 8 == 0 && g.out_row_stride >= row &&
                  g.out_row_stride % 4 == 0,
              NKV_EINVAL, "scaled_prefill: row strides must cover Hq*D, q's in multiples of 8, "
              "out's of 4");
  const int32_t Hk = (int32_t)g.n_kv_heads, group = (int32_t)(g.n_q_heads / g.n_kv_heads);
  const ScaledPrefillPlan p = scaled_prefill_plan(g.n_seqs, g.total_q, g.max_seqlen_q,
                                                  g.workspace ? g.max_seqlen_k : 0, Hk, group,
                                                  (int)g.head_dim);
  const size_t need = p.bytes((int)g.head_dim);
  NKV_REQUIRE(!p.split || (aligned16(g.workspace) && g.workspace_bytes >= (int64_t)need),
              NKV_EWORKSPACE, "scaled_prefill: workspace needs %zu bytes, 16-byte aligned (got %lld)",
              need, (long long)g.workspace_bytes);
  NKV_REQUIRE(p.grid < (1ll << 24), NKV_EUNSUPPORTED,  // threads of a launch are 32 bits
              "scaled_prefill: too many tiles in one call");
  i32x4_t* desc = static_cast<i32x4_t*>(g.workspace);
  const ScaledPrefillArgs a{(const bf16_t*)g.q, g.q_row_stride, (const char*)g.k_cache,
                            (const char*)g.v_cache, g.cu_seqlens_q, g.cu_seqlens_k, g.block_tables,
                            g.bt_row_stride, Hk, group, (int32_t)g.block_size,
                            (int32_t)g.max_blocks_per_seq, (int32_t)g.n_blocks, (int32_t)g.n_seqs,
                            (int32_t)p.tiles, (int32_t)p.sort, g.total_q,
                            (float)g.scale * kLog2e, (bf16_t*)g.out, g.out_row_stride, desc,
                            p.split ? reinterpret_cast<float*>(desc + p.grid) : nullptr};
  const dim3 grid((unsigned)p.grid);
#define NKV_SCALED_PREFILL_S(D, RG, SPLIT)                                                       \
  hipLaunchKernelGGL((scaled_prefill_kernel<D, RG, SPLIT>), grid, dim3(256), 0,       \
                     as_stream(g.stream), a)
#define NKV_SCALED_PREFILL(D, RG)                       \
  do {                                                  \
    if (p.split) NKV_SCALED_PREFILL_S(D, RG, true);     \
    else NKV_SCALED_PREFILL_S(D, RG, false);            \
  } while (0)
  if (g.head_dim == 64) {
    if (p.groups == 1) NKV_SCALED_PREFILL(64, 1);
    else NKV_SCALED_PREFILL(64, 2);
  } else {
    if (p.groups == 1) NKV_SCALED_PREFILL(128, 1);
    else if (p.groups == 2) NKV_SCALED_PREFILL(128, 2);
    else NKV_SCALED_PREFILL_S(128, 3, false);
  }
#undef NKV_SCALED_PREFILL
#undef NKV_SCALED_PREFILL_S
  rc = check_launch("nkv_scaled_prefill");
  if (rc || !p.split) return rc;
  const int32_t tile_rows = 64 * p.groups;
  const dim3 merge((unsigned)p.grid, (unsigned)(tile_rows / 16));
  if (g.head_dim == 64)
    hipLaunchKernelGGL((scaled_merge_kernel<64>), merge, dim3(256), 0, as_stream(g.stream), a,
                       tile_rows);
  else
    hipLaunchKernelGGL((scaled_merge_kernel<128>), merge, dim3(256), 0, as_stream(g.stream), a,
                       tile_rows);
  return check_launch("nkv_scaled_prefill");
}
