// Differential attention of many query rows (prompts, chunks of them, decode rows among them)
// over the paged K/V cache or contiguous K/V: bf16/fp16 MFMA, fp32 softmax. The formulas are in
// diff_common.h; causal, aligned to the bottom right. No counterpart in the reference; it stands
// beside the varlen attention of nanokvllm/layers/attention.py:96-102 over the same cache.
//
// MI355X design (MFMA-bound):
//  * Workgroup = (sequence, tile of queries, KV pair, range of keys). A tile's R rows are its
//    queries for all G query pairs of the KV pair, query-major, and each row is computed twice,
//    once for each map: the first half of the waves takes map 0, the other half map 1 of the same
//    rows. Both read the same V tile (the pair's value of 2 D dims), and each its own half of
//    every K row, so that K and V are fetched once for both maps and no product is made with the
//    other map's keys.
//  * Keys advance in steps of 64. A step's K and V rows (2 D dims each: the pair's two heads lie
//    beside each other) go straight into LDS, one step ahead or more, with the chunk permutation
//    of lds_tiles.h; fp8 codes pass through registers and are widened on the way.
//  * head_dim 64: four waves of three row groups, two workgroups a CU, which drift apart by
//    themselves. head_dim 128: eight waves of two row groups, one workgroup a CU, the maps' waves
//    half a step apart (see the half steps below).
//  * S^T = K Q^T (A: 16 keys from LDS, B: the wave's Q^T, held in registers) leaves a lane with one
//    row's scores of 4 keys in every 16; the weights, packed to 16 bits, are the B operand of
//    O^T += V^T P^T, its A operand read transposed from LDS. A row's running maximum is raised only
//    when it grows by more than kDiffLazy (log2), its sum is over the rounded weights. Weights in
//    16 bits are what the matrix cores take beside V as the cache holds it; summing them as rounded
//    lets the roundings' common part cancel. Relative error against 64 bits 0.0020 to 0.0023, where
//    32 bits throughout, with the output rounded, have 0.0017.
//  * The end of a tile: map 1's waves leave A_1 in LDS (the tiles' ring, free by then), map 0's
//    waves subtract, take the mean square over the row's 2 D dims (in the row's 4 lanes), normalise
//    and store. Two row groups at head_dim 128 take all 256 VGPRs there and spill 28 to 34 more,
//    behind the step loop: 31 KB a tile, as much as the call with four chunks below writes beyond
//    its output (86 MB against 58). No other instance spills.
//  * Few tiles: the tiles' keys are cut into ranges of the same number of steps, about as many in
//    all as workgroups are resident, a partial row (O, m, l) is written for each and map, and a
//    second kernel merges and ends them. Tiles of one range are ended by the first kernel.
//  * Sequences that bring one token, among prompts: the first workgroups' waves stream their K/V as
//    the decode kernel does, beside the tiles that keep the matrix cores; a tile for one query
//    would multiply 96 or 128 rows for it. The second kernel merges them too.
// Tiles are numbered over the batch without gaps (their number per sequence is known on the device
// only), each sequence's last ones first: they see the most keys.
#include "diff_common.h"
#include "launch_rules.h"
#include "lds_tiles.h"

#include <algorithm>
#include <type_traits>

namespace nkv {

constexpr int kDiffStep = 64;        // keys per step
constexpr float kDiffLazy = 8.f;     // log2 headroom before a running maximum is raised
constexpr int kDiffMinSteps = 4;     // shortest range of a cut tile
constexpr int kDiffMergeWaves = 4;
// Weight of a decode row against a tile where workgroups are shared out between them (diff_plan);
// half of it with fp8. An empirical choice, and it weighs a row by no length, since the host knows
// none but the longest. Us with 0.3 / 0.6 / 1.33 (Hq 32, Hk 8, bf16, 40 rows
// beside two chunks of 512; then fp8, 20 rows beside two of up to 2048), head_dim 128:
//   rows of 50-300:    137 / 136 / 172    293 / 293 / 293
//   rows of 300-4000:  158 / 166 / 175    808 / 427 / 304
//   rows of 6000-8000: 388 / 297 / 233   2275 / 1156 / 512
// and at head_dim 64: 98 / 95 / 74, 99 / 123 / 95, 187 / 158 / 150; 128 / 128 / 131, 265 / 148 /
// 142, 702 / 368 / 188. Few rows of long contexts beside long chunks wait for their streams.
constexpr double kDiffRowShare = 0.6;

// Waves of a workgroup, and 16-row groups of a wave at most. At head_dim 128 a step's tiles take
// 64 KiB, so one workgroup is resident and brings both waves of each SIMD itself. With fp8 the
// codes wait in 16 registers a lane until they are widened, and two groups then spilled
// (1006 us, one 980: four chunks of up to 2048 tokens over up to 6000, Hq 32, Hk 8);
// with one, each fragment read from LDS serves one product where 16-bit caches' serve two (675
// us). Codes that wait in LDS would leave the registers free; not built.
constexpr int diff_waves(int D) { return D == 128 ? 8 : 4; }
constexpr int diff_groups(int D, bool f8) { return D == 128 ? (f8 ? 1 : 2) : 3; }
constexpr int diff_rows(int D, int rg) { return 8 * diff_waves(D) * rg; }  // of a tile
constexpr int diff_part_row(int D) { return 2 * D + 4; }  // floats: O, m, l, 2 pad

struct DiffPrefillArgs {
  const bf16_t* q;
  int64_t q_row_stride;
  const void *k, *v;
  int64_t k_row_stride, v_row_stride;
  const int32_t *cu_q, *cu_k, *block_tables;
  int64_t bt_row_stride;
  int32_t P, G, block_size, max_blocks, n_limit, n_seqs, total_q;
  // workgroups for a pair at a time (0: tiles stay whole), and the most ranges and tiles of a cut
  // batch
  int32_t target, range_cap, tile_cap;
  float cus;
  float scale_log2, v_scale;
  DiffArgs diff;
  bf16_t* out;
  int64_t out_row_stride;
  // of cut tiles: {ranges, the first one, first row of q, rows}; [tile_cap]: tiles
  i32x4_t* tile_desc;
  float* part;
  // decode rows apart from the tiles: the first row_groups workgroups stream them (0: they are
  // tiles)
  int32_t row_groups, ncg, min_chunks, max_tokens;
  i32x4v_t* row_desc;
  float* row_part;
};

// A range of a tile of the batch: queries j0 .. of a sequence (row q0 of q), the key steps of range
// sp of `ranges`.
struct DiffTile {
  int seq, q0, Lq, kb0, Lk, j0;
  int id, n_steps, ranges, sp;
};

__device__ __forceinline__ int diff_steps(int Lq, int Lk, int QT, int tile) {
  const int last = min(Lk - 1, Lk - Lq + min(Lq, (tile + 1) * QT) - 1);
  return last >= 0 ? last / kDiffStep + 1 : 0;
}

// Range x of a pair, by the whole wave; false past the last one. The tiles of a sequence have as
// many places for ranges as its last one needs, so that a lane knows its sequence's number without
// a loop; the others' last places stay empty. n_tiles: all tiles, 0 where none is cut.
template <int D, int RG>
__device__ __forceinline__ bool diff_range(const DiffPrefillArgs& a, int QT, int x, DiffTile& d,
                                           int& n_tiles) {
  // A step of a workgroup alone on its CU, and of one of two on it (at head_dim 128 one is
  // resident). Measured with 256 and 512 workgroups, from 4096 keys to 12288, 16-bit caches
  // (fp8): head_dim 64, one row group 0.70 and 1.01 us (0.92, 1.29), three 1.33 and 2.10 (1.67,
  // 2.40); head_dim 128, one 1.56 (1.89), two 2.48. Only their ratio to what follows matters, and
  // one table serves all types. Then what a range's partial rows (101 KB at head_dim 64 with
  // three groups, 266 at 128 with two) cost of the chip's time, written and read again, and what
  // the merge takes beside that: fitted to whole calls.
  constexpr float kStepUs[2] = {D == 64 ? (RG == 1 ? 0.8f : 1.6f) : (RG == 1 ? 1.4f : 2.2f),
                                D == 64 ? (RG == 1 ? 1.1f : 2.1f) : (RG == 1 ? 1.4f : 2.2f)};
  constexpr float kRangeUs = D == 64 ? 0.01f * RG : 0.02f * RG, kMergeUs = 6.f;
  const int lane = threadIdx.x & 63;
  int q0 = 0, Lq = 0, kb0 = 0, Lk = 0, nt = 0, hi = 0, at = -1;
  auto load = [&](int cb) {  // lane: sequence cb + lane
    if (cb == at) return;
    at = cb;
    const int s = cb + lane;
    Lq = 0;
    if (s < a.n_seqs) {
      q0 = a.cu_q[s];
      Lq = a.cu_q[s + 1] - q0;
      kb0 = a.cu_k[s];
      Lk = a.cu_k[s + 1] - kb0;
      NKV_DBG(x == 0 && (Lq < 0 || Lk < 0 || Lq > Lk || q0 < 0 || q0 + Lq > a.total_q),
              NKV_DEBUG_LENGTH);
      Lk = max(Lk, 0);
      if (q0 < 0 || q0 > a.total_q - Lq) Lq = 0;  // rows outside q
      if (a.row_groups > 0 && Lq == 1) Lq = 0;    // not a tile
    }
    nt = Lq > 0 ? (Lq - 1) / QT + 1 : 0;
    hi = nt > 0 ? diff_steps(Lq, Lk, QT, nt - 1) : 0;
  };
  int R = INT32_MAX;  // steps of a range
  n_tiles = 0;
  if (a.target > 0) {
    // Lane k tries ranges of 1 / (k + 1) of the longest tile and takes the time until all are
    // through: steps, slower where two workgroups share a CU, and the partial rows, which all go
    // through memory twice.
    int longest = 0, tiles = 0;
    for (int cb = 0; cb < a.n_seqs; cb += 64) {  // uniform
      load(cb);
      longest = max(longest, hi);
      tiles += nt;
    }
    longest = (int)wave_max((float)longest);  // exact: below 2^24 steps of 64 keys, or near enough
    tiles = __builtin_amdgcn_readlane(wave_incl_scan(tiles), 63);
    const int mine = max(kDiffMinSteps, (longest + lane) / (lane + 1));
    const float per = 1.f / (float)mine;
    float T = 0.f, made = 0.f, places = 0.f;
    for (int cb = 0; cb < a.n_seqs; cb += 64) {
      load(cb);
      const int lo = nt > 0 ? diff_steps(Lq, Lk, QT, 0) : 0;
      for (uint64_t left = __ballot(nt > 0); left; left &= left - 1) {  // sequences with tiles
        const int ln = __builtin_ctzll(left);
        const float n = (float)__builtin_amdgcn_readlane(nt, ln);
        const float last = (float)__builtin_amdgcn_readlane(hi, ln);
        const float first = (float)__builtin_amdgcn_readlane(lo, ln);
        const float most = fmaxf(1.f, ceilf(last * per));
        T += n * 0.5f * (last + first);
        made += n * 0.5f * (most + fmaxf(1.f, ceilf(first * per)));
        places += n * most;
      }
    }
    const float m = (float)a.target, range = (float)min(mine, longest);
    const float groups = made * (float)a.P;
    const float step = groups <= a.cus ? kStepUs[0] : kStepUs[1];
    float cost = step * (made <= m ? range : T / m + 0.5f * range);
    if (lane > 0) cost += kMergeUs + groups * kRangeUs;
    if (lane > 0 && (places > (float)a.range_cap || (longest + lane - 1) / lane <= kDiffMinSteps))
      cost = INFINITY;  // too many, or what the lane before tries
    const float best = -wave_max(-cost);
    const int k = __builtin_ctzll(__ballot(cost == best) | 1ull << 63);
    // k = 0: whole tiles; as they are, too, for another batch than the plan was for (the places,
    // counted exactly: the workgroups and the partial rows are for range_cap)
    if (k > 0 && tiles <= a.tile_cap) {
      R = __builtin_amdgcn_readlane(mine, k);
      int exact = 0;
      for (int cb = 0; cb < a.n_seqs; cb += 64) {
        load(cb);
        exact += __builtin_amdgcn_readlane(wave_incl_scan(nt * max(1, (hi + R - 1) / R)), 63);
      }
      if (exact > a.range_cap) R = INT32_MAX;
      else n_tiles = tiles;
    }
  }
  int base = 0, tiles = 0;
  for (int cb = 0; cb < a.n_seqs; cb += 64) {  // uniform
    load(cb);
    const int places = R == INT32_MAX ? 1 : max(1, (hi + R - 1) / R);
    const int incl = wave_incl_scan(nt * places);
    const int total = __builtin_amdgcn_readlane(incl, 63);
    const int tile_incl = wave_incl_scan(nt);
    if (x < base + total) {
      const int ln =
          __builtin_amdgcn_readfirstlane(__builtin_ctzll(__ballot(base + incl > x)));
      d.seq = cb + ln;
      d.q0 = __builtin_amdgcn_readlane(q0, ln);
      d.Lq = __builtin_amdgcn_readlane(Lq, ln);
      d.kb0 = __builtin_amdgcn_readlane(kb0, ln);
      d.Lk = __builtin_amdgcn_readlane(Lk, ln);
      const int tn = __builtin_amdgcn_readlane(nt, ln);
      const int pl = __builtin_amdgcn_readlane(places, ln);
      const int rest = x - (base + __builtin_amdgcn_readlane(incl, ln) - tn * pl);
      const int k = __builtin_amdgcn_readfirstlane(rest / pl);  // the sequence's last tile first
      d.sp = rest - k * pl;
      d.id = tiles + __builtin_amdgcn_readlane(tile_incl, ln) - tn + k;
      d.j0 = (tn - 1 - k) * QT;
      d.n_steps = diff_steps(d.Lq, d.Lk, QT, tn - 1 - k);
      d.ranges = pl == 1 ? 1
                         : __builtin_amdgcn_readfirstlane(max(1, (d.n_steps + R - 1) / R));
      return true;
    }
    base += total;
    tiles += __builtin_amdgcn_readlane(tile_incl, 63);
  }
  return false;
}

// The batch's decode rows that lie within q.
struct OneDiffSeqs : OneRowSeqs {
  int32_t total_q;
  __device__ __forceinline__ int keys(int s) const {
    const int r = cu_q[s];
    return r >= 0 && r < total_q ? OneRowSeqs::keys(s) : 0;
  }
};

// The partial rows of range x of pair p, map 0's then map 1's.
template <int D, int RG>
__device__ __forceinline__ float* diff_part(const DiffPrefillArgs& a, int x, int p) {
  return a.part + ((int64_t)x * a.P + p) * (2 * diff_rows(D, RG) * diff_part_row(D));
}

template <bool F8, int D, bool H16, bool PAGED, int RG>
__global__ __launch_bounds__(64 * diff_waves(D), 2) void diff_prefill_kernel(
    const DiffPrefillArgs a) {
  static_assert(!(F8 && (H16 || !PAGED)), "fp8 caches are paged and read with bf16 queries");
  constexpr int kWaves = diff_waves(D), kRG = RG;
  constexpr bool kPing = kWaves == 8;
  constexpr int kV = 2 * D;                     // dims of a K or V row of the pair
  constexpr int kEl = F8 ? 1 : 2;               // bytes per cache element
  constexpr int kRB = kV * 2;                   // bytes of a staged (16-bit) row
  constexpr int kNC = kV / 8;                   // 16-byte chunks per staged row
  constexpr int kTileB = kDiffStep * kRB;       // bytes of a K or V tile
  constexpr int kTiles = kPing ? 5 : 4;         // places in the ring
  [[maybe_unused]] constexpr int kStageB = 2 * kTileB;  // a step's K and V tiles
  constexpr int kKs = D / 32;                   // k-steps of S^T (of one map's K head)
  constexpr int kDb = kV / 16;                  // 16-dim blocks of O^T
  constexpr int kWR = kDiffStep / kWaves;       // rows of a tile that a wave brings
  constexpr int kRpl = 1024 / kRB;              // rows per 1 KiB load into LDS
  constexpr int kNl = kWR / kRpl;               // such loads per wave per tile
  constexpr int kLpr8 = kV / 16;                // F8: lanes per row (16 codes each)
  constexpr int kRpl8 = 64 / kLpr8;             // F8: rows per load
  constexpr int kNl8 = kWR / kRpl8;             // F8: loads per wave per tile
  static_assert(kNl >= 1 && kNl8 >= 1, "a wave brings whole loads");
  static_assert(kWaves / 2 * kRG * kDb * 1024 <= kTiles * kTileB, "A_1 fits the ring");
  constexpr int kRowLds = PAGED ? 2 * decode_lds_elems<F8, 1, kV>() : 0;  // bytes a wave
  __shared__ __attribute__((aligned(1024))) char
      ring[kWaves * kRowLds > kTiles * kTileB ? kWaves * kRowLds : kTiles * kTileB];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g4 = lane >> 4;
  const int col = lane & 15;
  const int map = wave / (kWaves / 2);
  const int wi = wave % (kWaves / 2);  // which rows
  const int G = a.G, P = a.P;
  const int QT = diff_rows(D, RG) / G;  // queries per tile

  if constexpr (PAGED) {
    if ((int)blockIdx.x < a.row_groups) {
      decode_stream<F8, 1, kV, H16, true>(
          OneDiffSeqs{{a.cu_q, a.cu_k, a.n_seqs, a.max_tokens}, a.total_q},
          (int)blockIdx.x * kWaves + wave, a.row_groups * kWaves,
          reinterpret_cast<bf16_t*>(ring + wave * kRowLds), a.q, a.q_row_stride, a.k, a.v,
          a.block_tables, a.bt_row_stride, P, 2 * G, a.ncg, a.block_size, a.max_blocks, a.n_limit,
          a.min_chunks, a.scale_log2, a.v_scale, a.row_part, a.row_desc);
      return;
    }
  }
  const int p = ((int)blockIdx.x - a.row_groups) % P;
  const int x = ((int)blockIdx.x - a.row_groups) / P;
  DiffTile d;
  int n_tiles;
  const bool some = diff_range<D, RG>(a, QT, x, d, n_tiles);
  if (a.target > 0 && p == 0 && tid == 0) {
    if (x == 0) a.tile_desc[a.tile_cap] = i32x4_t{n_tiles, 0, 0, 0};
    if (some && d.sp == 0 && d.id < a.tile_cap)
      a.tile_desc[d.id] = i32x4_t{d.ranges, x, d.q0 + d.j0, min(QT, d.Lq - d.j0) * a.G};
  }
  if (!some || d.sp >= d.ranges) return;  // uniform
  const int j0 = d.j0, Lq = d.Lq, Lk = d.Lk;
  const int n_rows = min(QT, Lq - j0) * G;
  // equal ranges but for one step; into scalar registers (the divisions are vector code)
  const int each = d.n_steps / d.ranges, more = d.n_steps - each * d.ranges;
  const int s_lo = __builtin_amdgcn_readfirstlane(d.sp * each + min(d.sp, more));
  const int s_end = __builtin_amdgcn_readfirstlane(s_lo + each + (d.sp < more ? 1 : 0));
  const int diag = Lk - Lq;  // query j sees keys <= diag + j

  // ---- the wave's share of a step's K and V rows: kWR consecutive keys, which lie in one block
  const uint32_t row_b = (uint32_t)a.k_row_stride * kEl;
  const uint32_t row_bv = (uint32_t)a.v_row_stride * kEl;
  const int lrow = lane / kNC;
  uint32_t vol[kNl];
#pragma unroll
  for (int h = 0; h < kNl; ++h) {
    const int r = kRpl * h + lrow;
    vol[h] = (uint32_t)r * row_b + (uint32_t)p * kRB +
             (uint32_t)((lane % kNC) ^ chunk_swz<kV>(r + kWR * wave)) * 16u;
  }
  const uint32_t ring_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)ring +
                             (uint32_t)wave * (kWR * kRB);
  const int f8_row0 = lane / kLpr8;
  const int f8_c = lane % kLpr8;
  const uint32_t f8_off = (uint32_t)p * kV + (uint32_t)f8_c * 16u;
  [[maybe_unused]] u32x4_t kq[kNl8], vq[kNl8];  // F8: the next step's codes

  const int32_t* bt = PAGED ? a.block_tables + (int64_t)d.seq * a.bt_row_stride : nullptr;
  int bt_base = 0;   // lane i holds entry bt_base + i of the table row
  int bt_lane = -1;
  auto load_window = [&]() {
    const int e = bt_base + lane;
    const int id = e < a.max_blocks ? bt[e] : -1;
    NKV_DBG((int64_t)e * a.block_size < Lk && (e >= a.max_blocks || id < 0 || id >= a.n_limit),
            e >= a.max_blocks ? NKV_DEBUG_LENGTH : NKV_DEBUG_BLOCK);
    bt_lane = (id >= 0 && id < a.n_limit) ? id : -1;
  };
  int c_t0 = s_lo * kDiffStep + kWR * wave;  // first key of the rows loaded next
  int c_blk = 0, c_off = 0;                  // their block and place in it
  if constexpr (PAGED) {
    c_blk = c_t0 / a.block_size;
    c_off = c_t0 - c_blk * a.block_size;
    bt_base = c_blk & ~63;
    load_window();
  }
  const int k_lim = min(Lk, s_end * kDiffStep);
  // The rows of the next step: their K into the tile at byte `at` of the ring, and then their V.
  int64_t row0 = 0;
  int nv = 0;  // valid ones of the wave's rows
  auto issue_k = [&](uint32_t at) {
    nv = min(kWR, k_lim - c_t0);
    if constexpr (PAGED) {
      const int pb = __builtin_amdgcn_readlane(bt_lane, c_blk - bt_base);
      nv = pb < 0 ? 0 : nv;
      row0 = (int64_t)pb * a.block_size + c_off;
    } else {
      const int r0 = d.kb0 + c_t0;
      NKV_DBG(nv > 0 && (r0 < 0 || r0 > a.n_limit - nv), NKV_DEBUG_BLOCK);
      nv = (r0 < 0 || r0 > a.n_limit - nv) ? 0 : nv;  // outside the K/V rows
      row0 = r0;
    }
    nv = max(nv, 0);
    row0 = nv > 0 ? row0 : 0;
    const char* kp = static_cast<const char*>(a.k) + row0 * a.k_row_stride * kEl;
    if constexpr (F8) {  // into registers; widened into the stage by commit()
      const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc(
          (void*)kp, (short)0, (uint32_t)nv * row_b, kBufferFlags);
#pragma unroll
      for (int f = 0; f < kNl8; ++f)
        kq[f] = __builtin_bit_cast(
            u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(
                         rk, (uint32_t)(kRpl8 * f + f8_row0) * row_b + f8_off, 0, 0));
    } else {
      const i32x4_t dk = buffer_desc(kp, (uint32_t)nv * row_b);
#pragma unroll
      for (int h = 0; h < kNl; ++h)
        load_to_lds(dk, ring_base + at + 1024u * h, vol[h]);
    }
    c_t0 += kDiffStep;
    if constexpr (PAGED) {  // blocks crossed: at most 4 (blocks are a multiple of 16)
      const int B = a.block_size, v = c_off + kDiffStep;
      const int n = (v >= B) + (v >= 2 * B) + (v >= 3 * B) + (v >= 4 * B);
      c_off = v - n * B;
      c_blk = __builtin_amdgcn_readfirstlane(c_blk + n);
    }
  };
  auto issue_v = [&](uint32_t at) {
    const char* vp = static_cast<const char*>(a.v) + row0 * a.v_row_stride * kEl;
    if constexpr (F8) {
      const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc(
          (void*)vp, (short)0, (uint32_t)nv * row_bv, kBufferFlags);
#pragma unroll
      for (int f = 0; f < kNl8; ++f)
        vq[f] = __builtin_bit_cast(
            u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(
                         rv, (uint32_t)(kRpl8 * f + f8_row0) * row_bv + f8_off, 0, 0));
    } else {
      const i32x4_t dv = buffer_desc(vp, (uint32_t)nv * row_bv);
#pragma unroll
      for (int h = 0; h < kNl; ++h)
        load_to_lds(dv, ring_base + at + 1024u * h,
                    vol[h] + (uint32_t)(kRpl * h + lrow) * (row_bv - row_b));
    }
  };
  auto refill_window = [&]() {  // uniform; once per 64 blocks
    if constexpr (PAGED) {
      if (c_blk - bt_base >= 64) {
        bt_base = c_blk & ~63;
        load_window();
      }
    }
  };
  // F8: codes in registers, widened into the wave's rows of an LDS tile. Lanes in the second half
  // of a row write their pair's second chunk first, so that each 16-byte write instruction covers
  // distinct banks.
  const bool f8_swap = f8_c >= kLpr8 / 2;
  auto commit = [&](const u32x4_t (&codes)[kNl8], char* tile) {
    char* at = tile + wave * (kWR * kRB);
#pragma unroll
    for (int f = 0; f < kNl8; ++f) {
      const int r = kRpl8 * f + f8_row0;
      const int off = r * kRB + ((2 * f8_c) ^ chunk_swz<kV>(r + kWR * wave)) * 16;
      u32x4_t lo, hi, c = codes[f];
      if (f8_swap) c = u32x4_t{c[2], c[3], c[0], c[1]};
      fp8x16_to_bf16(c, lo, hi);
      *reinterpret_cast<u32x4_t*>(at + off + (f8_swap ? 16 : 0)) = lo;
      *reinterpret_cast<u32x4_t*>(at + off + (f8_swap ? 0 : 16)) = hi;
    }
  };
  if (s_lo < s_end) {
    issue_k(0);
    issue_v(kTileB);
    refill_window();
  }

  // ---- the wave's rows: query pair and query of this lane's row in each group (query-major; rows
  // past the tile's are attended like its first one and never stored)
  const bool active = wi * (16 * kRG) < n_rows;  // uniform over the wave
  int pair[kRG], jrow[kRG];
  u32x4_t qreg[kRG][kKs];
#pragma unroll
  for (int rr = 0; rr < kRG; ++rr) {
    const int r = (wi * kRG + rr) * 16 + col;
    const bool real = r < n_rows;
    pair[rr] = real ? r % G : 0;
    jrow[rr] = real ? j0 + r / G : Lq;
    const u32x4_t* qp = reinterpret_cast<const u32x4_t*>(
        a.q + (int64_t)(d.q0 + (real ? jrow[rr] : j0)) * a.q_row_stride +
        (int64_t)(2 * (p * G + pair[rr]) + map) * D + g4 * 8);
#pragma unroll
    for (int ks = 0; ks < kKs; ++ks) qreg[rr][ks] = qp[ks * 4];
  }

  // LDS read offsets (bytes from a tile's start). K A operand, 16-key quarter h: row 16h + col,
  // dims map * D + 32 ks + 8 g4: chunk map * D/8 + 4 ks + g4 before the permutation, an XOR like
  // the place of ks in it, so that one register holds them all.
  const uint32_t ko = (uint32_t)col * kRB +
                      (uint32_t)((map * (D / 8) + g4) ^ chunk_swz<kV>(col)) * 16u;
  // V^T by ds_read_b64_tr_b16: lane 16g + 4r + c reads row 4g + r (and +16), dims 16 db + 4c .. +3:
  // chunk 2 db + c/2, half c%2. The low three bits of db likewise; the rows' permutation has no
  // more.
  const int vrow = 4 * g4 + (col >> 2);
  const uint32_t vo = (uint32_t)vrow * kRB + (uint32_t)chunk_swz<kV>(vrow) * 16u +
                      (uint32_t)(col & 3) * 8u;

  f32x4_t acc[kRG][kDb];  // O^T: lane l -> row l%16, dims 16 db + 4(l/16) .. +3
  float m_run[kRG], l_run[kRG], mb_run[kRG];  // mb_run: m_run, or 0 while the row sees no key
#pragma unroll
  for (int rr = 0; rr < kRG; ++rr) {
#pragma unroll
    for (int db = 0; db < kDb; ++db) acc[rr][db] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    m_run[rr] = -INFINITY;
    l_run[rr] = 0.f;
    mb_run[rr] = 0.f;
  }
  // the uses pin the loads of Q here, so that no wait for them lands inside the loop
#pragma unroll
  for (int rr = 0; rr < kRG; ++rr)
#pragma unroll
    for (int ks = 0; ks < kKs; ++ks) asm volatile("" ::"v"(qreg[rr][ks]));
  const char* lds = (const char*)(__attribute__((address_space(3))) char*)ring;
  float sv[kRG][16];     // a step's scores
  u32x4_t pb[2][kRG];    // and its weights, 32 keys at a time
  // S^T of a K tile; `between` runs among its products. Two k-steps' reads are issued before the
  // products of the two before, and the barriers keep them there: the compiler would wait for each
  // read right after it.
  auto scores = [&](uint32_t kt, auto between) {
    constexpr int kN = 4 * kKs / 2;
    u32x4_t ka[2][2];
    auto read = [&](int i, u32x4_t (&x)[2]) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
        x[j] = *reinterpret_cast<const u32x4_t*>(lds + ((kt + ko) ^ (2 * i % kKs + j) * 64u) +
                                                 2 * i / kKs * (16 * kRB));
    };
    read(0, ka[0]);
    f32x4_t x[kRG];
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      if (i + 1 < kN) read(i + 1, ka[(i + 1) & 1]);
      __builtin_amdgcn_sched_barrier(0);
      if (i == 2) between();
      if (2 * i % kKs == 0) {
#pragma unroll
        for (int rr = 0; rr < kRG; ++rr) x[rr] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      }
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int rr = 0; rr < kRG; ++rr)
          x[rr] = mfma_16x16x32<H16>(ka[i & 1][j], qreg[rr][2 * i % kKs + j], x[rr]);
      if (2 * (i + 1) % kKs == 0) {
#pragma unroll
        for (int rr = 0; rr < kRG; ++rr)
#pragma unroll
          for (int e = 0; e < 4; ++e) sv[rr][2 * i / kKs * 4 + e] = x[rr][e];
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // masks step s and raises the running maxima
  auto maxima = [&](int s) {
    const bool edge = (s * kDiffStep + kDiffStep - 1 > diag + j0) ||
                      (s * kDiffStep + kDiffStep > Lk);  // uniform
    if (edge) {
#pragma unroll
      for (int rr = 0; rr < kRG; ++rr) {
        const int lim = min(diag + jrow[rr], Lk - 1);  // the row's last visible key
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (s * kDiffStep + 16 * (e / 4) + 4 * g4 + e % 4 > lim) sv[rr][e] = -INFINITY;
      }
    }
    // a lane tests its own scores against the headroom; only when some lane's exceed it does the
    // wave take the rows' maxima and rescale
    float lmax[kRG];
    bool lraise = false;
#pragma unroll
    for (int rr = 0; rr < kRG; ++rr) {
      const float* x = sv[rr];
      lmax[rr] = fmax3(fmax3(fmax3(x[0], x[1], x[2]), fmax3(x[3], x[4], x[5]),
                             fmax3(x[6], x[7], x[8])),
                       fmax3(x[9], x[10], x[11]),
                       fmax3(fmax3(x[12], x[13], x[14]), x[15], -INFINITY));
      lraise = lraise || (lmax[rr] * a.scale_log2 > m_run[rr] + kDiffLazy);
    }
    if (__builtin_amdgcn_ballot_w64(lraise) != 0) {
#pragma unroll
      for (int rr = 0; rr < kRG; ++rr) {
        const float cm = col_max4(lmax[rr]) * a.scale_log2;
        const bool raise = cm > m_run[rr] + kDiffLazy;
        const float alpha = raise ? fast_exp2(m_run[rr] - cm) : 1.f;
        m_run[rr] = raise ? cm : m_run[rr];
        mb_run[rr] = m_run[rr] == -INFINITY ? 0.f : m_run[rr];
        l_run[rr] *= alpha;
#pragma unroll
        for (int db = 0; db < kDb; ++db) acc[rr][db] *= alpha;
      }
    }
  };
  // the weights of 32 keys: k-slot j of lane group g is key 32c+4g+j (j<4), or 32c+16+4g+(j-4)
  auto weights = [&](int c) {
#pragma unroll
    for (int rr = 0; rr < kRG; ++rr) {
      float w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        w[e] = fast_exp2(fmaf(sv[rr][8 * c + e], a.scale_log2, -mb_run[rr]));  // -inf -> 0
      pb[c][rr] = u32x4_t{cvt_pk16<H16>(w[0], w[1]), cvt_pk16<H16>(w[2], w[3]),
                          cvt_pk16<H16>(w[4], w[5]), cvt_pk16<H16>(w[6], w[7])};
#pragma unroll
      for (int e = 0; e < 4; ++e) l_run[rr] = sum2_16<H16>(pb[c][rr][e], l_run[rr]);
    }
  };
  // O^T += V^T P^T: V^T of kVg 16-dim blocks at a time, the next ones' reads in flight
  constexpr int kVg = 4;
  auto values = [&](uint32_t vt) {
    u32x4_t va[2][kVg];
    auto read = [&](int g, u32x4_t (&x)[kVg]) {
#pragma unroll
      for (int i = 0; i < kVg; ++i) {
        const int db = (g * kVg + i) % kDb;
        const char* at = lds + ((vt + vo) ^ (db & 7) * 32u) + (db & 8) * 32 +
                         g * kVg / kDb * (32 * kRB);
        const i16x4_t v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t*)at);
        const i16x4_t v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t*)(at + 16 * kRB));
        x[i] = u32x4_t{__builtin_bit_cast(uint2, v0).x, __builtin_bit_cast(uint2, v0).y,
                       __builtin_bit_cast(uint2, v1).x, __builtin_bit_cast(uint2, v1).y};
      }
    };
    read(0, va[0]);
#pragma unroll
    for (int g = 0; g < 2 * kDb / kVg; ++g) {
      if (g + 1 < 2 * kDb / kVg) read(g + 1, va[(g + 1) & 1]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < kVg; ++i)
#pragma unroll
        for (int rr = 0; rr < kRG; ++rr)
          acc[rr][(g * kVg + i) % kDb] = mfma_16x16x32<H16>(
              va[g & 1][i], pb[g * kVg / kDb][rr], acc[rr][(g * kVg + i) % kDb]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  const int n = s_end - s_lo;
  if constexpr (kPing) {
    // Half steps, a barrier after each. Waves w and w + 4, on one SIMD, are of different maps, and
    // map 1's are half a step behind: while one's softmax keeps the vector unit busy, the other's
    // products have the matrix cores. Tiles are numbered K 0, V 0, K 1, V 1 ..: in half step h the
    // waves of map 0 work on tile h (scores of a K tile, products of a V tile), those of map 1 on
    // tile h - 1. Tile i lies in place i % kTiles of the ring, which is free from half step
    // i + 2 - kTiles on, and is fetched from then on until the end of half step i - 1: three half
    // steps with five places; fp8 codes, which wait in registers, two. Four chunks of up to 2048
    // tokens over up to 6000 (Hq 32, Hk 8): whole steps with a barrier each 690 us, half steps and
    // four places 685, five 660 to 678 in several runs; without the fetches 602, without the
    // softmax too 554.
    constexpr int kAhead = F8 ? 2 : 3;
    auto next = [](uint32_t at) { return at + kTileB == kTiles * kTileB ? 0u : at + kTileB; };
    uint32_t rd = 0, wr = 2 * kTileB;  // places read and fetched next
    [[maybe_unused]] uint32_t cm = 0;  // F8: and written next
    auto fetch = [&](auto v_c) {
      if constexpr (decltype(v_c)::value) {
        issue_v(wr);
      } else {
        issue_k(wr);
      }
      wr = next(wr);
    };
    // the tile after the one that map 0 has now is in LDS; kAhead - 1 fetches may be in flight
    auto landed = [&](auto v_c) {
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"((kAhead - 1) * (F8 ? kNl8 : kNl)) : "memory");
      if constexpr (F8) {
        commit(decltype(v_c)::value ? vq : kq, ring + cm);
        cm = next(cm);
      }
    };
    using K = std::integral_constant<bool, false>;
    using V = std::integral_constant<bool, true>;
    using First = std::conditional_t<kAhead == 2, K, V>;  // what an even half step fetches
    using Second = std::conditional_t<kAhead == 2, V, K>;
    if (n > 0) {
      if constexpr (kAhead == 3) fetch(K{});
      refill_window();
      landed(K{});
      __syncthreads();
      if (map == 1) {  // half step 0
        fetch(First{});
        refill_window();
        landed(V{});
        __syncthreads();
      }
      auto run = [&](auto map_c) {
        using Scores = std::conditional_t<decltype(map_c)::value == 0, First, Second>;
        using Values = std::conditional_t<decltype(map_c)::value == 0, Second, First>;
        using Next = std::conditional_t<decltype(map_c)::value == 0, V, K>;  // lands with scores
        using After = std::conditional_t<decltype(map_c)::value == 0, K, V>;
        for (int s = s_lo; s < s_end; ++s) {
          if (active) {
            scores(rd, [&] { fetch(Scores{}); });
            maxima(s);
            weights(0);
            weights(1);
          } else {
            fetch(Scores{});
          }
          rd = next(rd);
          refill_window();
          landed(Next{});
          __syncthreads();
          fetch(Values{});
          if (active) values(rd);
          rd = next(rd);
          refill_window();
          landed(After{});
          __syncthreads();
        }
      };
      if (map == 0) {
        run(std::integral_constant<int, 0>{});
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();  // map 1's last half step
      } else {
        run(std::integral_constant<int, 1>{});
      }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load into LDS is left in flight
    __syncthreads();
  } else {
    auto landed = [&](int stage) {  // the wave's rows of the stage are in LDS
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      if constexpr (F8) {
        commit(kq, ring + stage * kStageB);
        commit(vq, ring + stage * kStageB + kTileB);
      }
    };
    if (n > 0) landed(0);
    __syncthreads();
    auto step = [&](auto stage_c, int s) {
      constexpr int ST = decltype(stage_c)::value;
      constexpr uint32_t kt = ST * kStageB;
      auto fetch = [&] {
        issue_k((ST ^ 1) * kStageB);
        issue_v((ST ^ 1) * kStageB + kTileB);
      };
      if constexpr (F8) fetch();
      if (active) {
        scores(kt, [&] {
          if constexpr (!F8) fetch();
        });
        maxima(s);
        weights(0);
        weights(1);
        values(kt + kTileB);
      } else if constexpr (!F8) {
        fetch();
      }
      // the next step's rows landed (each wave waits for its own), then the barrier publishes them
      // and frees this stage
      landed(ST ^ 1);
      __syncthreads();
      refill_window();
    };
    for (int s = s_lo; s < s_end; s += 2) {
      step(std::integral_constant<int, 0>{}, s);
      if (s + 1 >= s_end) break;
      step(std::integral_constant<int, 1>{}, s + 1);
    }
  }

  // ---- the end
  float l[kRG];
#pragma unroll
  for (int rr = 0; rr < kRG; ++rr) {
    l[rr] = col_sum4(l_run[rr]);
    if (l[rr] == 0.f) {  // no key seen: zero, also beside values that are not finite (0 * inf)
#pragma unroll
      for (int db = 0; db < kDb; ++db) acc[rr][db] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
  }
  if (d.ranges > 1) {  // a part: O, m and l as they are
    if (!active) return;
    float* rows = diff_part<D, RG>(a, x, p) + (int64_t)map * (diff_rows(D, RG) * diff_part_row(D));
#pragma unroll
    for (int rr = 0; rr < kRG; ++rr) {
      if (jrow[rr] >= Lq) continue;
      float* pr = rows + ((wi * kRG + rr) * 16 + col) * diff_part_row(D);
#pragma unroll
      for (int db = 0; db < kDb; ++db)
        *reinterpret_cast<f32x4_t*>(pr + db * 16 + g4 * 4) = acc[rr][db];
      if (g4 == 0) *reinterpret_cast<float2*>(pr + kV) = float2{m_run[rr], l[rr]};
    }
    return;
  }
  float inv[kRG];
#pragma unroll
  for (int rr = 0; rr < kRG; ++rr) inv[rr] = l[rr] > 0.f ? a.v_scale / l[rr] : 0.f;
  // the ring is free: A_1, lane by lane as it is held
  f32x4_t* other = reinterpret_cast<f32x4_t*>(ring) + wi * (kRG * kDb * 64) + lane;
  if (map == 1 && active) {
#pragma unroll
    for (int rr = 0; rr < kRG; ++rr)
#pragma unroll
      for (int db = 0; db < kDb; ++db) other[(rr * kDb + db) * 64] = acc[rr][db] * inv[rr];
  }
  __syncthreads();
  if (map == 1 || !active) return;
  const float lambda = diff_lambda<D>(a.diff);
#pragma unroll
  for (int rr = 0; rr < kRG; ++rr) {
    float ss = 0.f;
#pragma unroll
    for (int db = 0; db < kDb; ++db) {
      const f32x4_t x = acc[rr][db] * inv[rr] - other[(rr * kDb + db) * 64] * lambda;
      acc[rr][db] = x;
      ss += (x[0] * x[0] + x[1] * x[1]) + (x[2] * x[2] + x[3] * x[3]);
    }
    inv[rr] = (1.f - a.diff.init) / sqrtf(col_sum4(ss) * (1.f / kV) + a.diff.eps);
  }
#pragma unroll
  for (int db = 0; db < kDb; ++db) {
    float w[4];
    const int dim = db * 16 + g4 * 4;
    diff_weight<4, H16>(a.diff.weight ? a.diff.weight + dim : nullptr, w);
#pragma unroll
    for (int rr = 0; rr < kRG; ++rr) {
      if (jrow[rr] >= Lq) continue;
      bf16_t* op = a.out + (int64_t)(d.q0 + jrow[rr]) * a.out_row_stride +
                   (int64_t)(p * G + pair[rr]) * kV + dim;
      float o[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = acc[rr][db][e] * w[e];
      store_dims<4, H16>(op, o, inv[rr]);
    }
  }
}

// Merges and ends the rows of tiles that have several ranges (workgroups below tile_groups); and
// the decode rows, two waves for each (sequence, query pair). A wave has kMergeRows rows of a tile
// at once, both maps of each: at head_dim 64 the halves of the wave have a map each, 4 dims a lane;
// at 128 every lane has 4 dims of both. kMergeFly ranges' loads are in flight. (One row a wave:
// 17 us over the 50 MB of two prompts of 512 tokens, Hq 32, Hk 8, head_dim 64.)
constexpr int kMergeRows = 4;
template <int D, bool H16, int RG>
__global__ __launch_bounds__(64 * kDiffMergeWaves) void diff_merge_kernel(
    const DiffPrefillArgs a, const int32_t tile_groups) {
  constexpr int kMaps = D / 64;  // of a lane
  constexpr int kMergeFly = 4 / kMaps;
  constexpr int kV = 2 * D;
  constexpr int kRow = diff_part_row(D);
  constexpr int kRowGroups = diff_rows(D, RG) / (kDiffMergeWaves * kMergeRows);  // of a tile
  static_assert(diff_rows(D, RG) % (kDiffMergeWaves * kMergeRows) == 0, "whole workgroups");
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int G = a.G, P = a.P;
  if ((int)blockIdx.x >= tile_groups) {
    __shared__ DiffLds<kV, 1> lds[kDiffMergeWaves / 2];
    const OneDiffSeqs seqs{{a.cu_q, a.cu_k, a.n_seqs, a.max_tokens}, a.total_q};
    const int id = ((int)blockIdx.x - tile_groups) * (kDiffMergeWaves / 2) + wave / 2;
    const int b = id / (P * G), r = b < a.n_seqs ? a.cu_q[b] : -1;
    const bool live = r >= 0 && r < a.total_q && a.cu_q[b + 1] - r == 1;
    diff_combine<kV, H16, 1>(seqs, b, id % (P * G), live, wave % 2, 2 * P * G, P, a.ncg,
                             a.row_part, a.row_desc, a.diff, a.out, a.out_row_stride,
                             lds[wave / 2]);
    return;
  }
  const int p = blockIdx.x % P;
  const int t = blockIdx.x / P / kRowGroups;
  const int r0 = ((int)(blockIdx.x / P % kRowGroups) * kDiffMergeWaves + wave) * kMergeRows;
  const i32x4_t d = a.tile_desc[t];
  const int ranges = d[0], rows = d[3];
  if (t >= a.tile_desc[a.tile_cap][0] || ranges < 2 || r0 >= rows) return;
  const float lambda = diff_lambda<D>(a.diff);
  const int dim = lane * 4 % kV;
  float w[4];
  diff_weight<4, H16>(a.diff.weight ? a.diff.weight + dim : nullptr, w);
  const int64_t map_f = (int64_t)diff_rows(D, RG) * kRow;
  const int64_t range_f = 2 * map_f * P;
  // the lane's map (the first of them) of row r0
  const float* part = diff_part<D, RG>(a, d[1], p) + (int64_t)r0 * kRow +
                      (kMaps == 1 ? (lane >> 5) * map_f : 0);
  float M[kMergeRows][kMaps], L[kMergeRows][kMaps];
  f32x4_t o[kMergeRows][kMaps];
#pragma unroll
  for (int i = 0; i < kMergeRows; ++i)
#pragma unroll
    for (int m = 0; m < kMaps; ++m) {
      M[i][m] = -INFINITY;
      L[i][m] = 0.f;
      o[i][m] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
  for (int s0 = 0; s0 < ranges; s0 += kMergeFly) {
    float2 ml[kMergeFly][kMergeRows][kMaps];
    f32x4_t v[kMergeFly][kMergeRows][kMaps];
#pragma unroll
    for (int u = 0; u < kMergeFly; ++u) {
      const float* range = part + min(s0 + u, ranges - 1) * range_f;
#pragma unroll
      for (int i = 0; i < kMergeRows; ++i)
#pragma unroll
        for (int m = 0; m < kMaps; ++m) {  // rows past the tile's: its last one again
          const float* row = range + min(i, rows - 1 - r0) * kRow + m * map_f;
          ml[u][i][m] = *reinterpret_cast<const float2*>(row + kV);
          v[u][i][m] = *reinterpret_cast<const f32x4_t*>(row + dim);
        }
    }
#pragma unroll
    for (int u = 0; u < kMergeFly; ++u) {
      if (s0 + u >= ranges) continue;  // uniform
#pragma unroll
      for (int i = 0; i < kMergeRows; ++i)
#pragma unroll
        for (int m = 0; m < kMaps; ++m) {
          // a range of no visible key has m = -inf, l = 0: weight 0 unless all have
          const float top = fmaxf(M[i][m], ml[u][i][m].x);
          const float mb = top == -INFINITY ? 0.f : top;
          const float alpha = fast_exp2(M[i][m] - mb), wu = fast_exp2(ml[u][i][m].x - mb);
          M[i][m] = top;
          L[i][m] = fmaf(wu, ml[u][i][m].y, L[i][m] * alpha);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            o[i][m][e] = fmaf(wu, v[u][i][m][e], o[i][m][e] * alpha);
        }
    }
  }
#pragma unroll
  for (int i = 0; i < kMergeRows; ++i) {
    const int r = r0 + i;
    if (r >= rows) break;  // uniform
    float x[4], ss = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float a0 = o[i][0][e] * (L[i][0] > 0.f ? a.v_scale / L[i][0] : 0.f);
      float a1;
      if constexpr (kMaps == 2) a1 = o[i][1][e] * (L[i][1] > 0.f ? a.v_scale / L[i][1] : 0.f);
      else a1 = __shfl_xor(a0, 32, 64);  // map 1 for the lower half
      x[e] = fmaf(-lambda, a1, a0);
      ss = fmaf(x[e], x[e], ss);
      x[e] *= w[e];
    }
#pragma unroll
    for (int s = kMaps == 2 ? 32 : 16; s > 0; s >>= 1) ss += __shfl_xor(ss, s, 64);
    const float norm = (1.f - a.diff.init) / sqrtf(ss * (1.f / kV) + a.diff.eps);
    if (kMaps == 2 || lane < 32)
      store_dims<4, H16>(a.out + (int64_t)(d[2] + r / G) * a.out_row_stride +
                             (int64_t)(p * G + r % G) * kV + dim,
                         x, norm);
  }
}

// Tiles that a batch can have.
static int64_t diff_max_tiles(int64_t total_q, int64_t n_seqs, int qt) {
  return total_q / qt + n_seqs;
}

// 16-row groups of a wave: one where the tiles then are no more than the CUs, since fewer rows a
// step are a shorter step, else as many as fit. One prompt of 300 / 900 tokens (Hq 16, Hk 8), us:
// head_dim 128 37.5 -> 25.1 / 56.7 -> 41.5, 64 24.5 -> 16.6 / 38.5 -> 25.4. Not at head_dim 64
// beside decode rows, which leave no CU idle (two chunks of 512 beside 30, fp8: 57 -> 76; at 128
// 146 -> 131 for one of 300 beside 100).
static int diff_choose(int64_t n_seqs, int64_t total_q, int64_t max_seqlen_q, int P, int G, int D,
                       bool f8) {
  const int most = diff_groups(D, f8), rows = diff_rows(D, 1);
  if (most == 1 || G > rows) return most;
  const BatchMix mix = batch_mix(n_seqs, total_q, std::max<int64_t>(max_seqlen_q, 1));
  const bool known = max_seqlen_q > 1;
  const int64_t tiles = known ? diff_max_tiles(mix.prompt_rows, mix.prompts, rows / G)
                              : diff_max_tiles(total_q, n_seqs, rows / G);
  if (D == 64 && known && mix.rows > 0) return most;
  return tiles * P <= device_cus() ? 1 : most;
}

// What a launch with a workspace does: into how many ranges a tile's keys are cut, and how many
// workgroups stream the decode rows.
struct DiffPlan {
  int64_t target, range_cap, tile_cap;
  int rg, row_groups, ncg;
  size_t tile_bytes, part_bytes, desc_bytes, row_bytes;
  size_t bytes() const { return tile_bytes + part_bytes + desc_bytes + row_bytes; }
};
static DiffPlan diff_plan(int64_t n_seqs, int64_t total_q, int64_t max_seqlen_q,
                          int64_t max_seqlen_k, int P, int G, int D, bool f8, bool paged) {
  DiffPlan d{};
  d.rg = diff_choose(n_seqs, total_q, max_seqlen_q, P, G, D, f8);
  const int rows_of = diff_rows(D, d.rg), qt = rows_of / G;
  const BatchMix mix = batch_mix(n_seqs, total_q, std::max<int64_t>(max_seqlen_q, 1));
  const int64_t resident = (int64_t)device_cus() * (D == 128 ? 1 : 2);
  int64_t tiles = diff_max_tiles(total_q, n_seqs, qt);  // that the batch has, about
  int64_t slots = resident;
  // (max_seqlen_q = 1 with more rows than sequences: padding, or not known)
  if (paged && mix.rows > 0 && (max_seqlen_q > 1 || (max_seqlen_q == 1 && total_q <= n_seqs))) {
    // A row's step of 64 keys is bound by its K/V bytes (half of them with fp8), a tile's by the
    // matrix cores: each gets workgroups by kDiffRowShare, whatever its length and head_dim.
    tiles = mix.prompts > 0 ? diff_max_tiles(mix.prompt_rows, mix.prompts, qt) : 0;
    const double rows = (double)mix.rows * kDiffRowShare * (f8 ? 0.5 : 1.0);
    d.ncg = decode_ncg(2 * G);
    const int np = P * d.ncg;  // groups of waves
    const int64_t least = (np + diff_waves(D) - 1) / diff_waves(D);
    d.row_groups = (int)std::max<int64_t>(
        least, std::min<int64_t>((int64_t)(resident * rows / (rows + (double)tiles)),
                                 mix.rows * P * std::max<int64_t>(1, max_seqlen_k / 64) /
                                         diff_waves(D) + 1));
    slots = std::max<int64_t>(resident - d.row_groups, 1);
    const int64_t waves = (int64_t)d.row_groups * diff_waves(D) / np;  // of a group
    d.desc_bytes = (size_t)n_seqs * P * d.ncg * sizeof(i32x4v_t);
    d.row_bytes = (size_t)((waves + n_seqs) * 2 * G * P) * part_row(2 * D) * sizeof(float);
  }
  if (tiles > 0 && tiles * P < slots && max_seqlen_k >= 2 * kDiffStep * kDiffMinSteps) {
    d.target = std::max<int64_t>(1, slots / P);
    d.range_cap = d.target + d.target / 2 + tiles;
    d.tile_cap = tiles;
    d.tile_bytes = (size_t)(tiles + 1) * sizeof(i32x4_t);
    d.part_bytes = (size_t)d.range_cap * P * 2 * rows_of * diff_part_row(D) * sizeof(float);
  }
  return d;
}

// Workgroups of a launch: the decode rows', and those of the ranges, or of the tiles where a batch
// has more of them than its plan.
static int64_t diff_groups_of(const DiffPrefillArgs& a, int64_t tiles) {
  return a.row_groups + std::max<int64_t>(a.range_cap, tiles) * a.P;
}

template <bool F8, int D, bool H16, bool PAGED, int RG>
static void diff_launch(const DiffPrefillArgs& a, int64_t tiles, hipStream_t s) {
  hipLaunchKernelGGL((diff_prefill_kernel<F8, D, H16, PAGED, RG>),
                     dim3((unsigned)diff_groups_of(a, tiles)), dim3(64 * diff_waves(D)), 0, s, a);
  const int64_t groups =
      (int64_t)a.tile_cap * a.P * (diff_rows(D, RG) / (kDiffMergeWaves * kMergeRows));
  const int64_t rows =
      a.row_groups > 0 ? ((int64_t)a.n_seqs * a.P * a.G + kDiffMergeWaves / 2 - 1) /
                             (kDiffMergeWaves / 2)
                       : 0;
  if (groups + rows > 0)
    hipLaunchKernelGGL((diff_merge_kernel<D, H16, RG>), dim3((unsigned)(groups + rows)),
                       dim3(64 * kDiffMergeWaves), 0, s, a, (int32_t)groups);
}
template <bool F8, int D, bool H16, bool PAGED>
static void diff_launch(const DiffPrefillArgs& a, int64_t tiles, int rg, hipStream_t s) {
  if (rg == 1) diff_launch<F8, D, H16, PAGED, 1>(a, tiles, s);
  else diff_launch<F8, D, H16, PAGED, diff_groups(D, F8)>(a, tiles, s);
}

}  // namespace nkv

extern "C" size_t nkv_diff_prefill_workspace_bytes(int32_t kv_type, int32_t n_seqs,
                                                   int64_t total_q, int64_t max_seqlen_q,
                                                   int64_t max_seqlen_k, int32_t n_q_heads,
                                                   int32_t n_kv_heads, int32_t head_dim,
                                                   int32_t paged) {
  using namespace nkv;
  if (n_seqs <= 0 || total_q <= 0 || n_kv_heads <= 0 || n_kv_heads % 2 || n_q_heads <= 0 ||
      n_q_heads % n_kv_heads || n_q_heads / n_kv_heads > NKV_DIFF_MAX_GROUP ||
      (head_dim != 64 && head_dim != 128))
    return 0;
  return diff_plan(n_seqs, total_q, max_seqlen_q, max_seqlen_k, n_kv_heads / 2,
                   n_q_heads / n_kv_heads, head_dim, kv_type == NKV_KV_FP8, paged != 0)
      .bytes();
}

extern "C" int nkv_diff_prefill(int32_t kv_type, const void* q, int64_t q_row_stride,
                                int64_t total_q, const void* k, const void* v,
                                int64_t k_row_stride, int64_t v_row_stride,
                                const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k,
                                const int32_t* block_tables, int64_t bt_row_stride,
                                int32_t max_blocks_per_seq, int32_t n_seqs, int64_t max_seqlen_q,
                                int64_t max_seqlen_k, int32_t n_q_heads, int32_t n_kv_heads,
                                int32_t head_dim, int32_t block_size, int64_t n_rows, float scale,
                                float k_scale, float v_scale, const float* lambdas,
                                float lambda_init, const void* norm_weight, float eps, void* out,
                                int64_t out_row_stride, void* workspace, size_t workspace_bytes,
                                void* stream) {
  using namespace nkv;
  clear_error();
  int rc = diff_check("diff_prefill", kv_type, n_q_heads, n_kv_heads, head_dim, scale, k_scale,
                      v_scale, lambdas, lambda_init, norm_weight, eps);
  if (rc) return rc;
  const bool paged = block_tables != nullptr, f8 = kv_type == NKV_KV_FP8;
  const int G = n_q_heads / n_kv_heads, P = n_kv_heads / 2;
  const int64_t row = (int64_t)n_kv_heads * head_dim;
  NKV_REQUIRE(n_seqs >= 0 && total_q >= 0 && n_rows >= 0 && total_q < (1ll << 31), NKV_EINVAL,
              "diff_prefill: bad sizes (n_seqs=%d, total_q=%lld, n_rows=%lld)", n_seqs,
              (long long)total_q, (long long)n_rows);
  if (n_seqs == 0 || total_q == 0) return NKV_OK;
  NKV_REQUIRE(q && k && v && cu_seqlens_q && cu_seqlens_k && out, NKV_EINVAL,
              "diff_prefill: null pointer");
  NKV_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) &&
                  (reinterpret_cast<uintptr_t>(out) & 7u) == 0,
              NKV_EINVAL, "diff_prefill: q, k and v must be 16-byte aligned, out 8-byte");
  NKV_REQUIRE(q_row_stride >= (int64_t)n_q_heads * head_dim && q_row_stride % 8 == 0 &&
                  out_row_stride >= (int64_t)n_q_heads * head_dim && out_row_stride % 4 == 0,
              NKV_EINVAL, "diff_prefill: row strides must be >= Hq*D, q's a multiple of 8, out's "
              "of 4");
  NKV_REQUIRE(k_row_stride >= row && v_row_stride >= row && k_row_stride % 8 == 0 &&
                  v_row_stride % 8 == 0 && k_row_stride < (1 << 24) && v_row_stride < (1 << 24),
              NKV_EINVAL, "diff_prefill: k and v row strides must be multiples of 8 from Hk*D to "
              "2^24");
  if (paged) {
    NKV_REQUIRE(block_size > 0 && block_size % 16 == 0, NKV_EUNSUPPORTED,
                "diff_prefill: block_size must be a multiple of 16 (got %d)", block_size);
    NKV_REQUIRE(max_blocks_per_seq > 0 && bt_row_stride >= max_blocks_per_seq, NKV_EINVAL,
                "diff_prefill: bad block table width/stride (%d, %lld)", max_blocks_per_seq,
                (long long)bt_row_stride);
    NKV_REQUIRE(k_row_stride == row && v_row_stride == row, NKV_EINVAL,
                "diff_prefill: paged rows are Hk*D apart");
    NKV_REQUIRE(n_rows / block_size < (1ll << 31), NKV_EUNSUPPORTED,
                "diff_prefill: too many blocks");
  } else {
    NKV_REQUIRE(!f8, NKV_EUNSUPPORTED, "diff_prefill: fp8 rows must be paged");
    NKV_REQUIRE(n_rows < (1ll << 31), NKV_EUNSUPPORTED, "diff_prefill: too many K/V rows");
  }
  DiffPrefillArgs a{};
  const int rg = diff_choose(n_seqs, total_q, max_seqlen_q, P, G, head_dim, f8);
  const int64_t tiles = diff_max_tiles(total_q, n_seqs, diff_rows(head_dim, rg) / G);
  if (workspace) {
    const DiffPlan d = diff_plan(n_seqs, total_q, max_seqlen_q, max_seqlen_k, P, G, head_dim, f8,
                                 paged);
    NKV_REQUIRE(workspace_bytes >= d.bytes() && aligned16(workspace), NKV_EWORKSPACE,
                "diff_prefill: workspace needs %zu bytes, 16-byte aligned (got %zu)", d.bytes(),
                workspace_bytes);
    char* ws = static_cast<char*>(workspace);
    a.target = (int32_t)d.target;
    a.cus = (float)std::max(1, device_cus() - d.row_groups);
    a.range_cap = (int32_t)d.range_cap;
    a.tile_cap = (int32_t)d.tile_cap;
    a.tile_desc = reinterpret_cast<i32x4_t*>(ws);
    ws += d.tile_bytes;
    a.part = reinterpret_cast<float*>(ws);
    if (d.row_groups > 0) {
      const int64_t max_chunks = decode_max_chunks(max_blocks_per_seq, block_size);
      NKV_REQUIRE((int64_t)max_blocks_per_seq * block_size < (1ll << 30) &&
                      max_chunks * n_seqs * P < (1ll << 31),
                  NKV_EUNSUPPORTED, "diff_prefill: too many keys in one call");
      a.row_groups = d.row_groups;
      a.ncg = d.ncg;
      a.min_chunks = decode_min_chunks(max_chunks, kMinChunks);
      a.max_tokens = max_blocks_per_seq * block_size;
      a.row_desc = reinterpret_cast<i32x4v_t*>(ws + d.part_bytes);
      a.row_part = reinterpret_cast<float*>(ws + d.part_bytes + d.desc_bytes);
    }
  }
  NKV_REQUIRE((tiles + (int64_t)a.range_cap) * P * diff_rows(head_dim, rg) < (1ll << 30) &&
                  (int64_t)n_seqs * n_q_heads < (1ll << 30),
              NKV_EUNSUPPORTED, "diff_prefill: too many tiles");
  a.q = (const bf16_t*)q;
  a.q_row_stride = q_row_stride;
  a.k = k;
  a.v = v;
  a.k_row_stride = k_row_stride;
  a.v_row_stride = v_row_stride;
  a.cu_q = cu_seqlens_q;
  a.cu_k = cu_seqlens_k;
  a.block_tables = block_tables;
  a.bt_row_stride = bt_row_stride;
  a.P = P;
  a.G = G;
  a.block_size = block_size;
  a.max_blocks = max_blocks_per_seq;
  a.n_limit = (int32_t)(paged ? n_rows / block_size : n_rows);
  a.n_seqs = n_seqs;
  a.total_q = (int32_t)total_q;
  a.scale_log2 = scale * (f8 ? k_scale : 1.f) * kLog2e;
  a.v_scale = f8 ? v_scale : 1.f;
  a.diff = DiffArgs{lambdas, (const bf16_t*)norm_weight, lambda_init, eps};
  a.out = (bf16_t*)out;
  a.out_row_stride = out_row_stride;
  hipStream_t s = as_stream(stream);
#define NKV_DIFF_LAUNCH(D)                                            \
  do {                                                                \
    if (f8) diff_launch<true, D, false, true>(a, tiles, rg, s);       \
    else if (kv_type == NKV_KV_F16)                                   \
      paged ? diff_launch<false, D, true, true>(a, tiles, rg, s)      \
            : diff_launch<false, D, true, false>(a, tiles, rg, s);    \
    else                                                              \
      paged ? diff_launch<false, D, false, true>(a, tiles, rg, s)     \
            : diff_launch<false, D, false, false>(a, tiles, rg, s);   \
  } while (0)
  if (head_dim == 64) NKV_DIFF_LAUNCH(64);
  else NKV_DIFF_LAUNCH(128);
#undef NKV_DIFF_LAUNCH
  return check_launch("nkv_diff_prefill");
}
