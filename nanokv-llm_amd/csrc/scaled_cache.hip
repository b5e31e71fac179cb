// The block-scaled K/V cache (scaled_cache.h): storing new rows into it and reading rows back.
//
// Reference: the store stands beside store_kvcache (nanokvllm/layers/attention.py:10-40), the cache
// beside the pool of ModelRunner.allocate_kv_cache (nanokvllm/engine/model_runner.py:133-152), which
// holds the model's dtype; reading back has no counterpart.
//
// A store takes a tile of a head at a time: over the rows that the call writes,
//   need = scale of max |x|,    e = need               if the tile's first row is among them
//                               e = max(e_old, need)   else, and where e grew the other rows' codes
//                                                      become E4M3(code * 2^(e_old - e))
//   code = E4M3(clamp(x * 2^-e, -448, 448)), to nearest even; NaN stays NaN.
// MI355X design: one wave to a tile and 128 elements of its rows (a head of 128, two of 64), K and V
// apart. Lane (x, y) holds dims 8x .. 8x+7 of tokens 8y .. 8y+7 in registers: one pass over the
// memory for the maximum and the codes, and both orders of codes are packed from the block that the
// lane holds (K's eight dims of a token, V's eight tokens of a dim), with no exchange. A tile that is
// written whole goes through LDS, which makes 1 KiB of consecutive bytes of each store instead of 32
// pieces of 16 (15800 rows of Hk 8, D 128: 25 us instead of 28, 3.9 TB/s). The tile's
// owner is the wave whose token begins a run of tokens of that tile in slot_mapping, which skipped
// tokens between them do not end.
#include "scaled_cache.h"

#include <algorithm>

namespace nkv {

constexpr int kGap = 32;         // so many skipped tokens end a run
// Neighbouring workgroups take windows a 37th of the list apart: with a tile's run in every fourth window
// those with work would else go to two of the eight XCDs (8 prompts of 512, Hk 8, D 128: 16.6 us, now
// 9.4; 16 of 2000: 52.7, now 37.4).
constexpr unsigned kScatter = 37;
constexpr int kScaledWaves = 4;  // of a workgroup: as many heads (or pairs), of K or V

int scaled_check(const char* what, const void* k_cache, const void* v_cache, int64_t n_kv_heads,
                 int64_t head_dim) {
  NKV_REQUIRE(scaled_dim_ok(head_dim), NKV_EUNSUPPORTED, "%s: head_dim must be 64 or 128 (got %lld)",
              what, (long long)head_dim);
  NKV_REQUIRE(n_kv_heads > 0 && n_kv_heads <= NKV_SCALED_MAX_HEADS, NKV_EUNSUPPORTED,
              "%s: 1 to %d KV heads (got %lld)", what, NKV_SCALED_MAX_HEADS, (long long)n_kv_heads);
  NKV_REQUIRE(k_cache && v_cache && aligned16(k_cache) && aligned16(v_cache), NKV_EINVAL,
              "%s: caches must be given, 16-byte aligned", what);
  return NKV_OK;
}
int scaled_check_tables(const char* what, const int32_t* block_tables, int64_t bt_row_stride,
                        int64_t max_blocks, int64_t block_size, int64_t n_blocks) {
  NKV_REQUIRE(block_size > 0 && block_size % kTileRows == 0, NKV_EUNSUPPORTED,
              "%s: block_size must be a multiple of %d (got %lld)", what, kTileRows,
              (long long)block_size);
  NKV_REQUIRE(max_blocks > 0 && bt_row_stride >= max_blocks, NKV_EINVAL,
              "%s: bad block table width/stride (%lld, %lld)", what, (long long)max_blocks,
              (long long)bt_row_stride);
  NKV_REQUIRE(n_blocks <= INT32_MAX && block_size < (1ll << 30) &&
                  max_blocks < (1ll << 30) / block_size,
              NKV_EUNSUPPORTED, "%s: max_blocks_per_seq * block_size too large", what);
  NKV_REQUIRE(block_tables, NKV_EINVAL, "%s: null block_tables", what);
  return NKV_OK;
}

// What a wave works on: 128 elements of a row of heads, of K or of V.
template <int D>
struct Unit {
  static constexpr int kHeads = 128 / D;
  static constexpr int kLanes = D / 8;  // of a head, eight dims each
  int h0, head, hx, x, y;
  bool is_v, live;
  __device__ __forceinline__ Unit(int unit, int units, int Hk) {
    const int lane = threadIdx.x & 63;
    x = lane & 15;
    y = lane >> 4;
    is_v = unit >= units / 2;
    h0 = (is_v ? unit - units / 2 : unit) * kHeads;
    head = h0 + x / kLanes;
    hx = x % kLanes;
    live = head < Hk;
  }
};
static int scaled_units(int Hk, int D) { return 2 * ((Hk * D + 127) / 128); }

__device__ __forceinline__ uint32_t abs_max2(uint32_t m, uint32_t w) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t,
                            __builtin_elementwise_max(__builtin_bit_cast(u16x2, m),
                                                      __builtin_bit_cast(u16x2, w & 0x7fff7fffu)));
}
__device__ __forceinline__ uint32_t drop_not_finite(uint32_t w) {
  if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u;
  if ((w & 0x7f800000u) == 0x7f800000u) w &= 0xffffu;
  return w;
}

// Two values to two codes in the low (or high) half of a word.
template <bool HIGH, bool SPECIAL>
__device__ __forceinline__ uint32_t put_codes(float a, float b, uint32_t old) {
  if constexpr (SPECIAL) {
    a = fp8_clamp(a);
    b = fp8_clamp(b);
  }
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, (int)old, HIGH);
}

// The codes of the lane's block into the head's tile (or its copy in LDS). SPECIAL: there may be
// values past +-448 or NaN among them. all: every row of the lane's eight is written.
template <int D, bool SPECIAL>
__device__ __forceinline__ void write_codes(const Unit<D>& un, const u32x4_t (&row)[8],
                                            const int (&src)[8], bool all, float inv, char* tile) {
  const auto value = [&](int k, int d) {
    const uint32_t w = row[k][d >> 1];
    return ((d & 1) ? bf16_hi(w) : bf16_lo(w)) * inv;
  };
  if (un.is_v) {
#pragma unroll
    for (int d = 0; d < 8; ++d) {
      uint32_t c[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        c[h] = put_codes<false, SPECIAL>(value(4 * h, d), value(4 * h + 1, d), 0);
        c[h] = put_codes<true, SPECIAL>(value(4 * h + 2, d), value(4 * h + 3, d), c[h]);
      }
      char* p = tile + v_piece(un.y, 8 * un.hx + d);
      if (all) {
        *reinterpret_cast<uint2*>(p) = uint2{c[0], c[1]};
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (src[k] >= 0) p[k] = (char)(c[k >> 2] >> (8 * (k & 3)));
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      uint32_t c[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        c[h] = put_codes<false, SPECIAL>(value(k, 4 * h), value(k, 4 * h + 1), 0);
        c[h] = put_codes<true, SPECIAL>(value(k, 4 * h + 2), value(k, 4 * h + 3), c[h]);
      }
      if (src[k] >= 0)
        *reinterpret_cast<uint2*>(tile + k_piece<D>(8 * un.y + k, un.hx)) = uint2{c[0], c[1]};
    }
  }
}

// The codes of a tile's 128 elements (`heads` heads of them live) times 2^-(growth of their head).
template <int D>
__device__ __forceinline__ void rescale(char* codes, const int (&shrink)[2], int heads) {
  constexpr int kPieces = kTileRows * D / 1024;  // of a head, 1 KiB each
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int h = 0; h < 128 / D; ++h) {
    if (h >= heads || shrink[h] == 0) continue;  // uniform
    const float f = __int_as_float((127 - min(shrink[h], 126)) << 23);
    u32x4_t* p = reinterpret_cast<u32x4_t*>(codes + h * (kTileRows * D)) + lane;
    u32x4_t w[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) w[i] = p[64 * i];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i][j], false);
        const auto b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i][j], true);
        uint32_t c = put_codes<false, false>(a[0] * f, a[1] * f, 0);
        w[i][j] = put_codes<true, false>(b[0] * f, b[1] * f, c);
      }
      p[64 * i] = w[i];
    }
  }
}

// Workgroup (window, unit group): the runs that begin among tokens [w0, w0 + window).
template <int D>
__global__ __launch_bounds__(64 * kScaledWaves) void scaled_store_kernel(
    const bf16_t* __restrict__ key, int64_t key_row_stride, const bf16_t* __restrict__ value,
    int64_t value_row_stride, char* __restrict__ k_cache, char* __restrict__ v_cache,
    const int32_t* __restrict__ slot_mapping, int64_t n_tokens, int32_t Hk, int64_t n_slots,
    int32_t units, int32_t window) {
  __shared__ int32_t rows[kScaledWaves][kTileRows];  // the token of each row of the tile, or -1
  __shared__ __attribute__((aligned(16))) char staged[kScaledWaves][kTileRows * 128];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int unit = blockIdx.y * kScaledWaves + wave;
  if (unit >= units) return;
  const Unit<D> un(unit, units, Hk);
  const bf16_t* src = un.is_v ? value : key;
  const int64_t stride = un.is_v ? value_row_stride : key_row_stride;
  char* cache = un.is_v ? v_cache : k_cache;
  const int64_t tile_bytes = (int64_t)kTileRows * (Hk * D + kRowPad);

  const auto tile_of = [&](int64_t t) -> int {  // -1: skipped, -2: no token
    if (t < 0 || t >= n_tokens) return -2;
    const int64_t s = slot_mapping[t];
    NKV_DBG(s < -1 || s >= n_slots, NKV_DEBUG_SLOT);
    return s >= 0 && s < n_slots ? (int)(s / kTileRows) : -1;
  };
  // lanes kGap ..: the window; a run goes on over fewer than kGap skipped tokens
  const uint32_t wi = window == 1 ? blockIdx.x
                                  : blockIdx.x % kScatter * (gridDim.x / kScatter) +
                                        blockIdx.x / kScatter;
  const int64_t w0 = (int64_t)wi * window - kGap;
  const int mine = lane < kGap + window ? tile_of(w0 + lane) : -2;
  const uint64_t before = __ballot(mine >= 0) & ((1ull << lane) - 1);
  const int last = before ? 63 - __builtin_clzll(before) : 0;
  const int last_tile = __shfl(mine, last, 64);
  uint64_t begins = __ballot(lane >= kGap && mine >= 0 &&
                             (!before || last < lane - kGap || last_tile != mine));

  for (; begins; begins &= begins - 1) {
    const int ln = __builtin_ctzll(begins);
    const int64_t t0 = w0 + ln;
    const int tile = __builtin_amdgcn_readlane(mine, ln);
    // the run's tokens by row; of two for a row the later one stays
    if (lane < kTileRows) rows[wave][lane] = -1;
    __builtin_amdgcn_wave_barrier();
    int skipped = 0;  // tokens since the run's last
    for (int64_t at = t0;;) {
      const int tl = tile_of(at + lane);
      const uint64_t out = ~__ballot(tl == tile);
      const int n = out ? __builtin_ctzll(out) : 64;
      if (lane < n) atomicMax(&rows[wave][slot_mapping[at + lane] % kTileRows], (int)(at + lane));
      if (n > 0) skipped = 0;
      at += n;
      if (n == 64) continue;
      const uint64_t next = ~__ballot(tl == -1) >> n;
      const int k = next ? __builtin_ctzll(next) : 64 - n;
      skipped += k;
      at += k;
      if (k == 0 || skipped >= kGap) break;
    }
    __builtin_amdgcn_wave_barrier();
    int from[8];
    bool all = true;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      from[k] = rows[wave][8 * un.y + k];
      all = all && from[k] >= 0;
    }
    const bool first = rows[wave][0] >= 0;
    __builtin_amdgcn_wave_barrier();
    char* base = cache + tile * tile_bytes;
    char* scales = base + kTileRows * Hk * D;
    const int old = un.live ? stored_scale((uint8_t)scales[un.head]) : kMinScale;
    u32x4_t row[8];
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      row[k] = u32x4_t{0, 0, 0, 0};
      if (from[k] >= 0 && un.live)
        row[k] = *reinterpret_cast<const u32x4_t*>(src + from[k] * stride + un.h0 * D + 8 * un.x);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k)
#pragma unroll
      for (int w = 0; w < 4; ++w) m = abs_max2(m, row[k][w]);
    uint32_t a = max(m & 0xffffu, m >> 16);
    bool special = __ballot(a >= 0x7f80u) != 0;
    if (special) {
      m = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int w = 0; w < 4; ++w) m = abs_max2(m, drop_not_finite(row[k][w]));
      a = max(m & 0xffffu, m >> 16);
    }
    // over the head's lanes and the four groups of tokens
#pragma unroll
    for (int o = 1; o < 64; o <<= 1)
      if (o < Unit<D>::kLanes || o >= 16) a = max(a, (uint32_t)__shfl_xor((int)a, o, 64));
    const int need = scale_byte(__uint_as_float(a << 16));
    const int e = first ? need : max(old, need);
    special = special || __ballot(e == kMaxScale) != 0;
    char* codes = base + un.h0 * (kTileRows * D);
    if (__ballot(all) == ~0ull) {
      // a whole tile: put together in LDS, written as 1 KiB of consecutive bytes at a time
      char* mine_at = staged[wave] + (un.head - un.h0) * (kTileRows * D);
      if (special) write_codes<D, true>(un, row, from, true, inverse_scale(e), mine_at);
      else write_codes<D, false>(un, row, from, true, inverse_scale(e), mine_at);
      __builtin_amdgcn_wave_barrier();
      const int pieces = min(Unit<D>::kHeads, Hk - un.h0) * (kTileRows * D / 1024);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < pieces)
          *reinterpret_cast<u32x4_t*>(codes + i * 1024 + lane * 16) =
              *reinterpret_cast<const u32x4_t*>(staged[wave] + i * 1024 + lane * 16);
      if (un.live && un.y == 0 && un.hx == 0) scales[un.head] = (char)e;
      __builtin_amdgcn_wave_barrier();
      continue;
    }
    if (!first) {
      const int grown = e - old;
      if (__ballot(un.live && grown > 0)) {
        const int shrink[2] = {__builtin_amdgcn_readlane(grown, 0),
                               __builtin_amdgcn_readlane(grown, Unit<D>::kLanes % 16)};
        rescale<D>(codes, shrink, min(Unit<D>::kHeads, Hk - un.h0));
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // other lanes' bytes go into those words
      }
    }
    if (un.live) {
      char* to = base + un.head * (kTileRows * D);
      if (special) write_codes<D, true>(un, row, from, all, inverse_scale(e), to);
      else write_codes<D, false>(un, row, from, all, inverse_scale(e), to);
      if (un.y == 0 && un.hx == 0) scales[un.head] = (char)e;
    }
  }
}

// ---------------------------------------------------------------- reading back
// HBM-bound: 414 MB read and written (12 sequences, Hk 8, D 128) in 82 us, 5.04 TB/s, a copy's rate. The
// wave's place in a tile is the store's, so that V's codes turn back into rows within the lane.
// Workgroup (tile, unit group): a tile of what sequence i holds at positions [start, start + n), n its
// share of cu_seqlens. Every workgroup finds its sequence and tile itself.
template <int D>
__global__ __launch_bounds__(64 * kScaledWaves) void scaled_read_kernel(
    const char* __restrict__ k_cache, const char* __restrict__ v_cache,
    const int32_t* __restrict__ block_tables, int64_t bt_row_stride,
    const int32_t* __restrict__ cu_seqlens, const int32_t* __restrict__ starts, int32_t n_seqs,
    int64_t n_tokens, int32_t Hk, int32_t block_size, int32_t max_blocks, int64_t n_blocks,
    int32_t units, bf16_t* __restrict__ k_out, bf16_t* __restrict__ v_out) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int unit = blockIdx.y * kScaledWaves + wave;
  if (unit >= units) return;
  const Unit<D> un(unit, units, Hk);

  // the sequence that holds tile blockIdx.x of all of them
  int cb = 0, base = 0, at = 0, n = 0, tiles = 0, incl = 0;
  uint32_t start = 0;  // positions may reach past 2^31: no table does
  for (;; cb += 64) {
    if (cb >= n_seqs) return;
    const int s = cb + lane;
    n = tiles = 0;
    if (s < n_seqs) {
      at = cu_seqlens[s];
      n = cu_seqlens[s + 1] - at;
      const int from = starts ? starts[s] : 0;
      start = (uint32_t)from;
      // rows outside the outputs or of no position: none (the grid counts n_tokens rows)
      const bool ok = at >= 0 && n > 0 && from >= 0 && (int64_t)at + n <= n_tokens;
      NKV_DBG(!ok && n != 0, NKV_DEBUG_LENGTH);
      if (!ok) n = 0;
      if (n > 0) tiles = (int)((start + n - 1) / kTileRows - start / kTileRows) + 1;
    }
    incl = wave_incl_scan(tiles);
    const int tot = __builtin_amdgcn_readlane(incl, 63);
    if ((int)blockIdx.x < base + tot) break;
    base += tot;
  }
  const int ln = __builtin_ctzll(__ballot(base + incl > (int)blockIdx.x));
  at = __builtin_amdgcn_readlane(at, ln);
  n = __builtin_amdgcn_readlane(n, ln);
  start = (uint32_t)__builtin_amdgcn_readlane((int)start, ln);
  const int first = base + __builtin_amdgcn_readlane(incl - tiles, ln);
  const uint32_t t0 = (start / kTileRows + (blockIdx.x - first)) * kTileRows;  // the tile's position
  const uint32_t bi = t0 / (uint32_t)block_size;
  const int id = bi < (uint32_t)max_blocks ? block_tables[(int64_t)(cb + ln) * bt_row_stride + bi] : -1;
  const bool valid = id >= 0 && id < n_blocks;
  NKV_DBG(!valid, bi < (uint32_t)max_blocks ? NKV_DEBUG_BLOCK : NKV_DEBUG_LENGTH);
  if (!un.live) return;

  u32x4_t row[8] = {};  // of token 8 y + k: dims 8 hx .. + 7
  if (valid) {
    const char* tile = (un.is_v ? v_cache : k_cache) +
                       ((int64_t)id * (block_size / kTileRows) + t0 % block_size / kTileRows) *
                           (kTileRows * (int64_t)(Hk * D + kRowPad));
    const float scale = scale_of(stored_scale((uint8_t)tile[kTileRows * Hk * D + un.head]));
    const char* codes = tile + un.head * (kTileRows * D);
    uint2 c[8];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      c[k] = *reinterpret_cast<const uint2*>(
          codes + (un.is_v ? v_piece(un.y, 8 * un.hx + k) : k_piece<D>(8 * un.y + k, un.hx)));
    u32x4_t w[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) w[k] = codes_to_bf16(c[k].x, c[k].y, scale);
    if (un.is_v) {  // w[d]: eight tokens of dim d
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int d = 0; d < 8; d += 2)
          row[k][d / 2] = __builtin_amdgcn_perm(w[d + 1][k / 2], w[d][k / 2],
                                                (k & 1) ? 0x07060302u : 0x05040100u);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) row[k] = w[k];
    }
  }
  bf16_t* out = (un.is_v ? v_out : k_out) + un.h0 * D + 8 * un.x;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int j = (int)(t0 + 8 * un.y + k - start);
    if (j >= 0 && j < n)
      __builtin_nontemporal_store(
          row[k], reinterpret_cast<u32x4_t*>(out + ((int64_t)at + j) * Hk * D));
  }
}

}  // namespace nkv

extern "C" int nkv_scaled_store(const nkv_scaled_store_args* args) {
  using namespace nkv;
  clear_error();
  NKV_REQUIRE(args, NKV_EINVAL, "scaled_store: null arguments");
  const nkv_scaled_store_args& g = *args;
  NKV_REQUIRE(g.n_tokens >= 0 && g.n_tokens < (1ll << 31) && g.n_slots >= 0, NKV_EINVAL,
              "scaled_store: bad sizes (%lld tokens, %lld slots)", (long long)g.n_tokens,
              (long long)g.n_slots);
  // a launch has fewer than 2^32 threads, 256 for each eight tokens
  NKV_REQUIRE(g.n_tokens <= (1 << 27) - 1024, NKV_EUNSUPPORTED,
              "scaled_store: at most 2^27 - 1024 tokens (got %lld)", (long long)g.n_tokens);
  if (g.n_tokens == 0) return NKV_OK;
  const int rc = scaled_check("scaled_store", g.k_cache, g.v_cache, g.n_kv_heads, g.head_dim);
  if (rc) return rc;
  const int64_t row = g.n_kv_heads * g.head_dim;
  NKV_REQUIRE(g.n_slots % kTileRows == 0, NKV_EINVAL,
              "scaled_store: the slots must be whole tiles of %d (got %lld)", kTileRows,
              (long long)g.n_slots);
  NKV_REQUIRE(g.key && g.value && g.slot_mapping && aligned16(g.key) && aligned16(g.value),
              NKV_EINVAL, "scaled_store: null or misaligned pointer");
  NKV_REQUIRE(g.key_row_stride >= row && g.value_row_stride >= row && g.key_row_stride % 8 == 0 &&
                  g.value_row_stride % 8 == 0,
              NKV_EINVAL, "scaled_store: row strides must be multiples of 8 covering the row");
  const int Hk = (int)g.n_kv_heads, units = scaled_units(Hk, (int)g.head_dim);
  // Tokens a wave looks at. Runs in one window follow each other (2.5 us each), and a wave without one
  // costs its dispatch (about 0.9 ns of the chip). 1 / 4 / 8 / 16 tokens (Hk 8, D 128), us:
  //   256 tokens of as many sequences (4096 of these products)   7.5 / 16.0 / 27.5 / 51
  //   1024, 2048 (16384, 32768)      19.1 / 24.5 / 31.6, 34.2 / 37.8 / 44.3
  //   8 prompts of 512 (65536)       73.8 / 10.4 / 9.4 / 7.9
  //   16 of 500 (128000)             46.3 / 15.8 / 14.0 / 13.4
  //   16 of 2000 (512000)            480 / 43.2 / 37.3 / 34.2
  // A list of prompts may hold single tokens too, whose windows should not outlast the rest. The rule knows
  // the list's length alone: 1024 and 2048 single tokens take the four of a list of prompts (24.5 and 37.8
  // us, one each 19.1 and 34.2).
  const int64_t waves = g.n_tokens * units;
  const int window = waves <= 8192 ? 1 : waves <= 131072 ? 4 : 8;
  int64_t windows = (g.n_tokens + window - 1) / window;
  if (window > 1) windows = (windows + kScatter - 1) / kScatter * kScatter;
  const dim3 grid((unsigned)windows, (unsigned)((units + kScaledWaves - 1) / kScaledWaves));
#define NKV_SCALED_STORE(D)                                                                      \
  hipLaunchKernelGGL((scaled_store_kernel<D>), grid, dim3(64 * kScaledWaves), 0,                 \
                     as_stream(g.stream), (const bf16_t*)g.key, g.key_row_stride,                \
                     (const bf16_t*)g.value, g.value_row_stride, (char*)g.k_cache,               \
                     (char*)g.v_cache, g.slot_mapping, g.n_tokens, Hk, g.n_slots, units, window)
  if (g.head_dim == 64) NKV_SCALED_STORE(64);
  else NKV_SCALED_STORE(128);
#undef NKV_SCALED_STORE
  return check_launch("nkv_scaled_store");
}

extern "C" int nkv_scaled_read(const nkv_scaled_read_args* args) {
  using namespace nkv;
  clear_error();
  NKV_REQUIRE(args, NKV_EINVAL, "scaled_read: null arguments");
  const nkv_scaled_read_args& g = *args;
  NKV_REQUIRE(g.n_seqs >= 0 && g.n_tokens >= 0 && g.n_blocks >= 0, NKV_EINVAL,
              "scaled_read: bad sizes (%lld sequences, %lld tokens)", (long long)g.n_seqs,
              (long long)g.n_tokens);
  // 64 sequences' tiles add up within 32 bits, whatever cu_seqlens holds
  NKV_REQUIRE(g.n_seqs <= (1 << 20) && g.n_tokens <= (1 << 27), NKV_EUNSUPPORTED,
              "scaled_read: at most 2^20 sequences and 2^27 tokens (got %lld, %lld)",
              (long long)g.n_seqs, (long long)g.n_tokens);
  if (g.n_seqs == 0 || g.n_tokens == 0) return NKV_OK;
  int rc = scaled_check("scaled_read", g.k_cache, g.v_cache, g.n_kv_heads, g.head_dim);
  if (rc) return rc;
  rc = scaled_check_tables("scaled_read", g.block_tables, g.bt_row_stride, g.max_blocks_per_seq,
                           g.block_size, g.n_blocks);
  if (rc) return rc;
  NKV_REQUIRE(g.cu_seqlens && g.k_out && g.v_out && aligned16(g.k_out) && aligned16(g.v_out),
              NKV_EINVAL, "scaled_read: null or misaligned pointer");
  const int Hk = (int)g.n_kv_heads, units = scaled_units(Hk, (int)g.head_dim);
  // n rows reach into at most n / 32 + 2 tiles
  const int64_t tiles = g.n_tokens / kTileRows + 2 * std::min<int64_t>(g.n_seqs, g.n_tokens);
  const dim3 grid((unsigned)tiles, (unsigned)((units + kScaledWaves - 1) / kScaledWaves));
#define NKV_SCALED_READ(D)                                                                        \
  hipLaunchKernelGGL((scaled_read_kernel<D>), grid, dim3(64 * kScaledWaves), 0,                   \
                     as_stream(g.stream), (const char*)g.k_cache, (const char*)g.v_cache,         \
                     g.block_tables, g.bt_row_stride, g.cu_seqlens, g.starts, (int32_t)g.n_seqs,  \
                     g.n_tokens, Hk, (int32_t)g.block_size, (int32_t)g.max_blocks_per_seq,        \
                     g.n_blocks, units, (bf16_t*)g.k_out, (bf16_t*)g.v_out)
  if (g.head_dim == 64) NKV_SCALED_READ(64);
  else NKV_SCALED_READ(128);
#undef NKV_SCALED_READ
  return check_launch("nkv_scaled_read");
}
