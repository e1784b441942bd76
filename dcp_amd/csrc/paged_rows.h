// The kernel of many rows (prompts, and prefixes that many requests share) and how its work is laid out.
#pragma once

#include <algorithm>

#include "paged_common.h"
#include "quantized_cache.h"

namespace dcp {

// sum + the two weights of a pair.
template <int DTYPE>
__device__ __forceinline__ float add_pair(uint32_t pair, float sum) {
  if constexpr (DTYPE == DCP_DTYPE_BF16) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pair), __builtin_bit_cast(bf16x2, 0x3f803f80u), sum, false);
  } else {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, pair), f16x2{1.0f16, 1.0f16}, sum, false);
  }
}

// 16 bytes a lane from memory into LDS at lds_at + 16 * lane (ordered by the caller, as KvTile's loads).  STREAM: read once, so it is
// to take no room in the caches: four contexts of 131072 keys 363 us without and 321 with it.
template <bool STREAM>
__device__ __forceinline__ void load_async_piece(uint32_t lds_at, const uint16_t* from) {
  if constexpr (STREAM)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off nt"
                 :
                 : "s"(__builtin_amdgcn_readfirstlane(lds_at)), "v"(from)
                 : "memory");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                 :
                 : "s"(__builtin_amdgcn_readfirstlane(lds_at)), "v"(from)
                 : "memory");
}

// The row tile of work item `rank` of a kv head (negative index: there is none), and which piece of its keys.  For up to 64 requests, one a lane.
struct RankedTile {
  RowTile tile;
  int share, n_shares;
};
// Tiles of the shortest piece.  us at 2, 3 and 4: 3 requests of 13 tokens of 1000 keys 17.7, 18.1, 18.8; 2 of 100 tokens of 1000 25.9, 23.8, 23.5.
constexpr int kMinTilesPerPiece = 3;
template <int BM>
__device__ __forceinline__ RankedTile find_ranked_tile(PagedArgs& p, SourceArgs& src, int rank) {
  const int lane = threadIdx.x & 63, b = min(lane, src.batch - 1);
  const TokenRange tokens = tokens_of(p, src, b);
  const int n_keys = keys_of(p, src, b), n_rows = lane < src.batch ? tokens.n * p.group : 0, at0 = n_keys - tokens.n;
  const int n_tiles = (n_rows + BM - 1) / BM;
  const int room = src.table_width * p.page_size / kRowsBN;
  const int most = p.window > 0 ? min((int)(((uint32_t)p.window + (uint32_t)p.n_starting) / kRowsBN), room) + 1 : room + 1;  // what a row can see
  auto total = [&](int n) { return __builtin_amdgcn_readlane(wave_scan(n), 63); };
  auto found = [&](int at, int index, int share, int n_shares) {
    auto of = [&](int x) { return __builtin_amdgcn_readlane(x, at); };
    return RankedTile{{at, of(index), {of(tokens.begin), of(tokens.n)}, of(n_keys)}, share, n_shares};
  };
  const int all = total(n_tiles);
  // Where there are fewer row tiles than workgroups, those of a request are cut into pieces of about `length` key tiles, the least that leaves
  // a workgroup for every piece: between an equal share of all key tiles and what that is if every row tile needs one piece more.  Half as many
  // workgroups where pieces are short: there is less to be joined then, and a workgroup that has a CU to itself takes three quarters of the time a
  // tile (us, all and half: 10 requests of 40 tokens of 2000 keys, 2 kv heads, 31.4 and 27.1; where pieces are longer than 6 tiles all are better, 24
  // of 40 tokens of up to 4000 44 and 84).
  const int places = src.by_few ? divide(p.n_few, p.by_heads) : 0;
  if (all < places) {
    const float tiles = (float)min(min((n_keys + kRowsBN - 1) / kRowsBN, most + 1), 1 << 20);
    const float sum = (float)total(n_tiles * (int)tiles);  // (less than 2^30)
    auto pieces = [&](float length) { return n_tiles * max((int)ceilf(tiles * __builtin_amdgcn_rcpf(length)), 1); };
    auto shortest = [&](int places) {
      float enough = max(sum / (float)(places - all), 1.0f), least = max(sum / (float)places, 1.0f);
      for (int i = 0; i < 4; ++i) {
        const float length = 0.5f * (enough + least);
        if (total(pieces(length)) <= places) enough = length;
        else least = length;
      }
      return enough;
    };
    float length = shortest(places);
    if (length <= 6.0f && all < places / 2) length = shortest(places / 2);
    const int n = pieces(max(length, (float)kMinTilesPerPiece)), ends = wave_scan(n);
    if (rank >= __builtin_amdgcn_readlane(ends, 63)) return {{0, -1, {0, 0}, 0}, 0, 0};
    const int at = __builtin_amdgcn_readfirstlane(__popcll(__ballot(ends <= rank)));
    const int in_request = rank - __builtin_amdgcn_readlane(ends - n, at), of_request = __builtin_amdgcn_readlane(n_tiles, at);
    const int each = __builtin_amdgcn_readlane(n, at) / of_request, from_last = in_request / each;
    return found(at, n_tiles - 1 - from_last, in_request - from_last * each, each);
  }
  // Otherwise the row tiles that see the most keys come first, by steps of 64: the last ones to start are the shortest, so that no CU is left
  // with a long one (32 requests of 500 tokens behind up to 2000 keys, lengths spread over a factor of 16: 115 us in the order of the requests, 84
  // so; 12 prompts of up to 1024 60 and 53).  A request's tiles that see more than 64 t keys are its last ones, and their number is known
  // from its lengths; t is found by halving.
  auto seeing_more = [&](int t) {  // tiles of the lane's request, all of them for t = 0
    const uint32_t first = kRowsBN * t > at0 ? (uint32_t)(kRowsBN * t) - (uint32_t)at0 : 0;  // the first token that sees more
    const int n = first < (uint32_t)tokens.n ? max(n_tiles - (int)first * p.group / BM, 0) : 0;
    return t == 0 ? n_tiles : t < most ? n : 0;
  };
  if (rank >= all) return {{0, -1, {0, 0}, 0}, 0, 0};
  int t = 0;
  for (int step = 1 << (31 - __builtin_clz(most)); step > 0; step >>= 1)
    if (t + step < most && total(seeing_more(t + step)) > rank) t += step;
  const int longer = seeing_more(t + 1), here = seeing_more(t) - longer;
  const int left = rank - total(longer), ends = wave_scan(here);
  const int at = __builtin_amdgcn_readfirstlane(__popcll(__ballot(ends <= left)));
  return found(at, n_tiles - 1 - (longer + left - (ends - here)), 0, 1);
}

// ---------------------------------------------------------------------------
// The kernel of rows: a workgroup of 4 waves owns 64 RT rows of one (request, kv head), 128 over a cache of 16 bits, a wave 16 RT of them, and
// walks its share of the 64-key tiles that any of them sees.  K and V tiles go from memory straight into LDS (KvTile), two stages each, K a tile
// ahead of V: S^T of tile t + 1 is multiplied while tile t is exponentiated, MFMA by MFMA in one stream, O^T += V^T P^T
// of tile t follows as a dense run that the SIMD's other wave fills with its own arithmetic.
// ---------------------------------------------------------------------------
constexpr float kNoMax = -3.0e38f;  // the reference of a row that has seen nothing: below every score, and a weight of -inf against it is 0
constexpr float kMaxTileSum = 16384.0f;  // of a lane's weights against a reference that is not their maximum: fp16 can hold them

// LDS of the kernel: two stages of K and of V, and where the 16-key groups of 2 x 64 tiles are.
constexpr int kTableTiles = 64;
template <int D>
struct RowsLds {
  static constexpr int TILE = KvTile<D>::SIZE * 2;
  static constexpr int OFFSETS = 4 * TILE;                     // int64 [2 * kTableTiles][4]: of a group, in the cache
  static constexpr int ABSENT = OFFSETS + 2 * kTableTiles * 4 * 8;  // int [2 * kTableTiles][4]: it is not there (its offset is then 0)
  static constexpr int ANY_ABSENT = ABSENT + 2 * kTableTiles * 4 * 4;  // int [2][4 waves]: one of the half's groups is not
  static constexpr int BYTES = ANY_ABSENT + 2 * 4 * 4;
};

// CORRECTED: O is divided by the sum of the rounded weights instead of theirs (l / rounded times as much), so that rounding a weight that
// outweighs the others cancels, lse as it was.  Prefixes have it in every launch: what the host says of the longest lengths chooses the
// launch, and is not to choose the rounding.  rms error against 64 bits in bf16 (0.0017 is the result's own rounding): one token a
// request 0.0023 -> 0.0019, 64 tokens each 0.0023 -> 0.0020.  Beside a prefix's chain of tiles the second sum costs nothing (64 requests of
// one token on a prefix of 32768 74.3 and 74.6 us), where products bound it 3-4 % (32 requests of 256 tokens on one of 4096 663 and 690, 4
// of 2048 on 16384 2105 and 2178).  Own keys have it not: a prompt of 8192 481 and 521 us, for an error of 0.0023 and 0.0022.
// In 4 bits requests of up to kQuantFewRows rows have it: those that the kernel of few rows takes where none longer is beside them, so that a token's
// rounding is that of the token alone.  31 single tokens of up to 8000 keys and a prompt of 500 80 us and 83, prompts without such as before
// (one of 8192 492; were they corrected as well 504, at head size 64 351 and 380).
//
// QUANT: the cache is held in 4 bits.  Wave w brings the tile's 16-key group w through registers: the codes of K of tile t + 3 and of V of
// tile t + 2 are asked for in iteration t, and those of the tiles before them, there by then, go into LDS as 16 bits, a row's
// piece between two products.
template <int DTYPE, int D, bool CORRECTED, bool QUANT = false, int RT = 2>
__device__ __forceinline__ void paged_rows(PagedArgs& p, SourceArgs& src, int item, char* lds) {
  typedef KvTile<D> Tile;
  constexpr int KS = D / 32, DT = D / 16, LPW = Tile::LPW, BM = 64 * RT;
  typedef RowsLds<D> Lds;
  constexpr int TILE_BYTES = Lds::TILE;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);

  // ---- which rows, which share of their keys ---------------------------------
  const bool ranked = QUANT && src.batch <= 64;
  RowTile tile;
  int kv_head, share, most_shares = src.n_shares, first_piece = 0;
  if (ranked) {
    const int rank = divide(item, p.by_heads);
    kv_head = item - rank * p.n_heads_kv;
    const RankedTile at = find_ranked_tile<BM>(p, src, rank);
    tile = at.tile;
    share = at.share;
    most_shares = at.n_shares;
    first_piece = kv_head * divide(p.n_few, p.by_heads) + rank - share;
  } else {
    const RowItem at = row_item(item, src.n_tiles, src.xcd_group, p.n_heads_kv, src.n_shares);
    if (at.share < 0) return;
    kv_head = __builtin_amdgcn_readfirstlane(at.kv_head);
    share = __builtin_amdgcn_readfirstlane(at.share);
    tile = find_row_tile<BM>(p, src, __builtin_amdgcn_readfirstlane(at.place));
  }
  const TokenRange tokens = tile.tokens;
  const int n_rows = tokens.n * p.group;  // (at most n_tokens * group, which the host has checked)
  auto token_of = [&](int row) { return QUANT ? divide(row, p.by_group) : row / p.group; };
  const int row0 = tile.index * BM;
  if (tile.index < 0) return;
  // In 4 bits a wave without rows brings its part of the tiles and does no more, and a CU's second workgroup has its first rows on other SIMDs: one
  // prompt of 500 tokens beside 31 single tokens behind up to 8000 keys 94 us -> 80.
  const int w_rows = QUANT ? w ^ (item >> 8 & 1) << 1 : w;
  const bool idle = QUANT && row0 + w_rows * (16 * RT) >= n_rows;
  const bool corrected = CORRECTED || (QUANT && n_rows <= kQuantFewRows);
  const bool prefix = src.cu_groups != nullptr;
  const int n_keys = tile.n_keys, window = prefix ? 0 : p.window, n_starting = p.n_starting;
  // token i of the request is at position n_keys - n + i; every token is past all of a prefix
  const int first_tok = token_of(row0), last_tok = token_of(min(row0 + BM, n_rows) - 1);
  const int at0 = prefix ? n_keys - 1 : n_keys - tokens.n, step = prefix ? 0 : 1;
  const KeyGroups groups(window, n_starting, max(at0 + first_tok * step, 0), at0 + last_tok * step);
  const int n_groups = __builtin_amdgcn_readfirstlane(groups.hull_end > 0 ? groups.count() : 0);
  const int tiles_all = (n_groups + 3) / 4, n_shares = min(most_shares, max(1, tiles_all / kMinTilesPerShare));
  int t_begin = 0, t_end = 0;
  if (ranked & (share >= n_shares)) return;
  if (share < n_shares) {
    if (QUANT && n_shares == 1) {
      t_end = tiles_all;
    } else {
      t_begin = __builtin_amdgcn_readfirstlane((int)((int64_t)tiles_all * share / n_shares));
      t_end = __builtin_amdgcn_readfirstlane((int)((int64_t)tiles_all * (share + 1) / n_shares));
    }
  }

  // ---- tiles: lane l brings pieces of rows of the tile's 16-key group l / 16, LPW of K and of V ---------
  constexpr int CH = D / 8;
  const int lane_row = Tile::row_of(w * LPW, lane / CH) & 15;  // of load 0; the others are LOAD_ROWS further each
  const uint16_t* k_lane = reinterpret_cast<const uint16_t*>(p.k) + ((int64_t)kv_head * p.head_stride + lane_row * p.token_stride + lane % CH * 8);
  const int64_t load_step = Tile::LOAD_ROWS * p.token_stride;
  const int64_t v_from_k = reinterpret_cast<const uint16_t*>(p.v) - reinterpret_cast<const uint16_t*>(p.k);
  const uint32_t k_at = lds_address(lds), v_at = k_at + 2 * TILE_BYTES;
  auto k_stage = [&](int t) { return reinterpret_cast<const uint16_t*>(lds + (t & 1) * TILE_BYTES); };
  auto v_stage = [&](int t) { return reinterpret_cast<const uint16_t*>(lds + (2 + (t & 1)) * TILE_BYTES); };
  auto load_k = [&](int t, int64_t off, int i) {
    load_async_piece<false>(Tile::group_lds_at(k_at + (t & 1) * TILE_BYTES, w, i), k_lane + off + i * load_step);
  };
  auto load_v = [&](int t, int64_t off, int i) {
    load_async_piece<false>(Tile::group_lds_at(v_at + (t & 1) * TILE_BYTES, w, i), k_lane + off + (v_from_k + i * load_step));
  };
  // the first key of group i of the list
  auto group_key = [&](int i) { return i < n_groups ? groups.at(i) * 16 : kNoKey; };
  // Where the groups are: a thread looks one up of the 64 tiles that begin with tile t_begin + rel, half a list ahead of its use.  (One
  // tile at a time, by the lanes that load it, the divisions and 64-bit products were 40 % of the loop's instructions.)
  int64_t* offsets = reinterpret_cast<int64_t*>(lds + Lds::OFFSETS);
  int* absent = reinterpret_cast<int*>(lds + Lds::ABSENT);
  int* any_absent = reinterpret_cast<int*>(lds + Lds::ANY_ABSENT);
  struct Entry {
    int key, in_page, page;
  };
  auto read_entry = [&](int rel) -> Entry {
    PagedArgs& p = fresh_kernel_args<PagedParams>();
    const int i = (t_begin + rel) * 4 + tid, key = i < 4 * t_end ? group_key(i) : kNoKey;
    if (key == kNoKey) return {key, 0, -1};
    const int entry = QUANT ? divide(key / 16, p.by_page) : key / p.page_size;
    return {key, key - entry * p.page_size, src.block_table[tile.b * src.table_stride + entry]};
  };
  auto look_up = [&](int rel, Entry entry) {
    PagedArgs& p = fresh_kernel_args<PagedParams>();
    const bool there = (unsigned)entry.page < (unsigned)p.n_pages;
    const int at = (rel * 4 + tid) % (2 * kTableTiles * 4);
    offsets[at] = !there ? 0 : entry.page * p.page_stride + (QUANT ? (int64_t)(entry.in_page / 16) * QuantTile<D>::BYTES : entry.in_page * p.token_stride);
    absent[at] = !there;
    const bool any = __any(!there & (entry.key != kNoKey));  // (what is past the end is no tile of anybody's)
    if (lane == 0) any_absent[rel / kTableTiles % 2 * 4 + w] = any;
  };
  auto offset_of = [&](int t) { return offsets[((t - t_begin) * 4 + g) % (2 * kTableTiles * 4)]; };

  Entry first_entry = {kNoKey, 0, -1};
  if (t_begin < t_end) first_entry = read_entry(0);

  // ---- this lane's rows: n of each of the wave's two row tiles (past the last one: the last one again, not written) ------
  int last_key[RT];                          // the last key it sees
  u32x4 q[RT][KS];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = min(row0 + w_rows * (16 * RT) + rt * 16 + n, n_rows - 1), tok = token_of(r), head = kv_head * p.group + (QUANT ? r - tok * p.group : r % p.group);
    const uint16_t* from = reinterpret_cast<const uint16_t*>(p.q) + (tokens.begin + tok) * p.q_token + head * p.q_head + Tile::element16(g);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) q[rt][ks] = *reinterpret_cast<const u32x4*>(from + Tile::step16(ks));
    last_key[rt] = at0 + tok * step;
  }
  // of the wave's rows (they do not decrease from lane to lane and tile to tile)
  const int first_last = __builtin_amdgcn_readlane(last_key[0], 0), last_last = __builtin_amdgcn_readlane(last_key[RT - 1], 15);
  if (t_begin < t_end) look_up(0, first_entry);  // (asked for before the rows, there before them)
  const int reach = window > 0 ? window : 0x7fffffff;  // a query sees the keys less than this before its last
  const float scale = p.scale_log2;

  // ---- running state ---------------------------------------------------------------
  f32x4 o[RT][DT];
  float m_run[RT], l_run[RT], lsum[RT];
  float l_rounded[RT];  // the sum of the rounded weights
  float alpha[RT];  // what O^T has to be multiplied by before the tile is added
  bool rescale = false;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    m_run[rt] = kNoMax;
    alpha[rt] = 1.0f;
    l_run[rt] = l_rounded[rt] = 0.0f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[rt][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  bool anchored = false;  // every row of the wave has a reference maximum
  u32x4 pb[RT][2];        // P^T of the current tile, packed
  const int k_rd = Tile::row_base16(n, g), v_rd = Tile::col_base16(lane);

  // Tiles that every row of the wave sees all of, by number: [0, full_first) in the first tokens, [full_begin, full_end) in the
  // window.  Any other is masked.
  const int shift = groups.n_first - groups.begin;
  const int full_first = min(n_starting / 16, max(first_last + 1, 0) / 16) / 4;
  const int full_begin = (max(groups.n_first, (max(last_last - reach + 1, 0) + 15) / 16 + shift) + 3) / 4;
  const int full_count = max((max(first_last + 1, 0) / 16 + shift) / 4 - full_begin, 0);
  auto is_full = [&](int t) {
    const int* any = any_absent + (t - t_begin) / kTableTiles % 2 * 4;
    const int bad = any[0] | any[1] | any[2] | any[3];
    return (((unsigned)t < (unsigned)full_first) | ((unsigned)(t - full_begin) < (unsigned)full_count)) & (__builtin_amdgcn_readfirstlane(bad) == 0);
  };
  auto mask = [&](int t, f32x4 (&s)[RT][4]) {
    if constexpr (QUANT) {
      // A key's distance to the row's last one is from 0 up to the window, in one unsigned comparison; or it is a first token.
      const bool first = group_key(t * 4) < n_starting;
#pragma unroll
      for (int kt = 0; kt < 4; ++kt) {
        const int key0 = absent[((t - t_begin) * 4 + kt) % (2 * kTableTiles * 4)] ? kNoKey : group_key(t * 4 + kt);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const int last = max(last_key[rt], -1), to_last = last - key0 - 4 * g;  // (kNoKey: far below 0)
          if (first) {
            const int to_first = min(n_starting - 1, last) - key0 - 4 * g;
#pragma unroll
            for (int e = 0; e < 4; ++e) s[rt][kt][e] = ((unsigned)(to_last - e) < (unsigned)reach) | (e <= to_first) ? s[rt][kt][e] : -INFINITY;
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) s[rt][kt][e] = (unsigned)(to_last - e) < (unsigned)reach ? s[rt][kt][e] : -INFINITY;
          }
        }
      }
      return;
    }
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
      const bool there = absent[((t - t_begin) * 4 + kt) % (2 * kTableTiles * 4)] == 0;
      const int key0 = group_key(t * 4 + kt);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = key0 + 4 * g + e;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const bool visible = (key <= last_key[rt]) & ((key < n_starting) | (last_key[rt] - key < reach)) & there;
          s[rt][kt][e] = visible ? s[rt][kt][e] : -INFINITY;
        }
      }
    }
  };
  // The maximum step: the row's reference raised to the tile's maximum, what was summed before taken relative to it.
  auto raise = [&](const f32x4 (&s)[RT][4]) {
    bool without = false;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float mx = -INFINITY;
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int e = 0; e < 4; ++e) mx = fmaxf(mx, s[rt][kt][e]);
      const float m_new = fmaxf(m_run[rt], rows_max(mx * scale));
      alpha[rt] = fast_exp2(m_run[rt] - m_new);
      l_run[rt] *= alpha[rt];
      m_run[rt] = m_new;
      lsum[rt] = 0.0f;
      without |= m_new == kNoMax;
    }
    anchored = !__any(without);
    rescale = __any((alpha[0] != 1.0f) | (alpha[RT - 1] != 1.0f));
  };
  // Two elements of the lane's 32 weights: pair i is of row tile i / 8, key tile i / 2 % 4.  Weights are rounded to the storage type
  // for the product (half a step each); their sum is of the unrounded ones.
  auto weigh = [&](const f32x4 (&s)[RT][4], int i) {
    const int rt = i / 8, kt = i / 2 % 4, e = i % 2 * 2;
    const float x0 = fast_exp2(fmaf(s[rt][kt][e], scale, -m_run[rt])), x1 = fast_exp2(fmaf(s[rt][kt][e + 1], scale, -m_run[rt]));
    lsum[rt] += x0 + x1;
    pb[rt][kt / 2][2 * (kt % 2) + e / 2] = pack2<DTYPE>(x0, x1);
  };

  f32x4 s_a[RT][4], s_b[RT][4];
  // S^T of a tile from stage k; `between(i)` goes between its 4 * KS operands
  auto multiply_qk = [&](const uint16_t* k, f32x4 (&s)[RT][4], auto between) {
    constexpr int N = 4 * KS, AHEAD = 2;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int kt = 0; kt < 4; ++kt) s[rt][kt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    u32x4 a[4];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) a[i] = Tile::read_row16(k, k_rd, i & 3, i >> 2);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i + AHEAD < N) a[(i + AHEAD) & 3] = Tile::read_row16(k, k_rd, (i + AHEAD) & 3, (i + AHEAD) >> 2);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) s[rt][i & 3] = mfma_16x16x32<DTYPE>(a[i & 3], q[rt][i >> 2], s[rt][i & 3]);
      between(i);
      __builtin_amdgcn_sched_barrier(0);  // keeps the operand reads from being hoisted into more registers
    }
  };
  auto multiply_pv = [&](const uint16_t* v) {
    constexpr int N = 2 * DT, AHEAD = 2;
    u32x4 a[4];
    float rounded[RT] = {};
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) a[i] = Tile::read_col16(v, v_rd, i / DT, i % DT);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i + AHEAD < N) a[(i + AHEAD) & 3] = Tile::read_col16(v, v_rd, (i + AHEAD) / DT, (i + AHEAD) % DT);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        o[rt][i % DT] = mfma_16x16x32<DTYPE>(a[i & 3], pb[rt][i / DT], o[rt][i % DT]);
#pragma unroll
        for (int x = i * 8 / N; CORRECTED && x < (i + 1) * 8 / N; ++x) rounded[rt] = add_pair<DTYPE>(pb[rt][x / 4][x % 4], rounded[rt]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int rt = 0; CORRECTED && rt < RT; ++rt) l_rounded[rt] += rounded[rt];
    if (QUANT && corrected) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int x = 0; x < 8; ++x) l_rounded[rt] = add_pair<DTYPE>(pb[rt][x / 4][x % 4], l_rounded[rt]);
    }
  };

  // ---- key loop ------------------------------------------------------------------------
  // Tile t's V is cleared where nobody sees it; by the wave that brought it, after its loads have landed.
  auto clear_v = [&](int t) {
    const int key0 = group_key(t * 4 + g);
    const bool there = absent[((t - t_begin) * 4 + g) % (2 * kTableTiles * 4)] == 0;
#pragma unroll
    for (int i = 0; i < LPW; ++i)
      if (!(there & groups.sees(key0 + lane_row + Tile::LOAD_ROWS * i)))
        *reinterpret_cast<u32x4*>(lds + (2 + (t & 1)) * TILE_BYTES + (Tile::group_lds_at(0, w, i) + 16 * lane)) = u32x4{0, 0, 0, 0};
  };
  // In 4 bits: the wave's group of K of tile t + 2 and of V of tile t + 1, in iteration t.
  const char* quant_head = reinterpret_cast<const char*>(p.k) + kv_head * p.head_stride;
  QuantGroup<D> codes;
  auto quant_at = [&](int t) { return quant_head + uniform64(offsets[((t - t_begin) * 4 + w) % (2 * kTableTiles * 4)]); };
  const int k_put = Tile::at(16 * w + n, g * (D / 4)), v_put = Tile::at(16 * w + 4 * g, n * (D / 16));
  auto put_k = [&](int t, int i) {  // eight elements of the lane's quarter of a row
    *reinterpret_cast<u32x4*>(lds + (t & 1) * TILE_BYTES + (k_put + 8 * i) * 2) = eight_of_codes<DTYPE>(codes.k[i], exponent_scale(codes.k_exp, 0));
  };
  auto put_v = [&](int t, int j) {  // the lane's sixteenth of a row
    char* to = lds + (2 + (t & 1)) * TILE_BYTES + (v_put + (D == 128 ? j * 4 * Tile::GROUP_STRIDE : (j & 1) * 4 * Tile::GROUP_STRIDE + (j >> 1) * D)) * 2;
    const float scale = exponent_scale(codes.v_exp, j);
    if constexpr (D == 128) {
      *reinterpret_cast<u32x4*>(to) = eight_of_codes<DTYPE>(codes.v[j], scale);
    } else {
      const uint32_t x = codes.v[j / 2];
      *reinterpret_cast<u32x2*>(to) = j % 2 ? u32x2{two_of_codes<DTYPE, 2>(x, scale), two_of_codes<DTYPE, 3>(x, scale)}
                                            : u32x2{two_of_codes<DTYPE, 0>(x, scale), two_of_codes<DTYPE, 1>(x, scale)};
    }
  };
  auto clear_codes = [&](int t) {  // of V, where nobody sees it
    const int key0 = group_key(t * 4 + w) + 4 * g;
    const bool there = absent[((t - t_begin) * 4 + w) % (2 * kTableTiles * 4)] == 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (!(there & groups.sees(key0 + j))) codes.clear_v(j);
  };
  bool full_next = false;  // is tile t + 1 full
  int64_t off_next = 0;  // of tile t + 1, whose K is there and whose V is asked for in iteration t
  auto iteration = [&](int t, f32x4 (&s_cur)[RT][4], f32x4 (&s_nxt)[RT][4]) {
    bool full;
    if constexpr (QUANT) {
      full = full_next;
      full_next = is_full(t + 1);
      if (__builtin_expect(!full_next, 0)) clear_codes(t + 1);
    } else {
      wait_loads();
      full = is_full(t);
      if (__builtin_expect(!full, 0)) clear_v(t);
    }
    if (__builtin_expect((t - t_begin) % kTableTiles == kTableTiles / 2, 0)) {
      const int rel = (t - t_begin) / kTableTiles * kTableTiles + kTableTiles;
      look_up(rel, read_entry(rel));
    }
    __syncthreads();  // K of tile t + 1 and V of tile t are there; nobody reads K of tile t or V of tile t - 1 any more
    // The loads of K of tile t + 2 and V of tile t + 1 go out between the products, unconditionally: past the end a page that there
    // is comes into a stage that nobody reads any more.
    const int64_t off_k = QUANT ? 0 : offset_of(t + 2);
    const char *k_from = nullptr, *v_from = nullptr;
    if constexpr (QUANT) {
      k_from = quant_at(t + 3);
      v_from = quant_at(t + 2);
    }
    if (QUANT && idle) {
#pragma unroll
      for (int i = 0; i < KS; ++i) put_k(t, i);
#pragma unroll
      for (int j = 0; j < 4; ++j) put_v(t + 1, j);
      codes.load_k(k_from, lane_here());
      codes.load_v(v_from, lane_here());
      return;
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) lsum[rt] = 0.0f;
    bool taken = false;  // the tile's maximum
    rescale = false;
    if constexpr (QUANT) {
      if (__builtin_expect(!full, 0)) mask(t, s_cur);
    }
    if (__builtin_expect(!((QUANT || full) & anchored), 0)) {
      if (!QUANT && !full) mask(t, s_cur);
      raise(s_cur);
      taken = true;
    }
    // Where every row has a reference and sees the whole tile (in 4 bits: or not, the masked weights are 0), its weights are taken against that without looking for its own
    // maximum; the lanes' sums tell afterwards whether that was safe, and if not it is done again.
    __builtin_amdgcn_s_setprio(2);
    constexpr int N = 4 * KS, NL = 2 * LPW;
    multiply_qk(k_stage(t + 1), s_nxt, [&](int i) {
#pragma unroll
      for (int x = i * 8 * RT / N; x < (i + 1) * 8 * RT / N; ++x) weigh(s_cur, x);
      if constexpr (QUANT) {
        if (i < KS) put_k(t, i);
        else if (i < KS + 4) put_v(t + 1, i - KS);
        else if (i == KS + 4) codes.load_k(k_from, lane_here());
        else if (i == KS + 5) codes.load_v(v_from, lane_here());
      } else {
        if (i < LPW) load_k(t, off_k, i);
        else if (i < NL) load_v(t + 1, off_next, i - LPW);
      }
    });
    if (__builtin_expect(!taken & __any(!((lsum[0] < kMaxTileSum) & (lsum[RT - 1] < kMaxTileSum))), 0)) {
      raise(s_cur);
#pragma unroll
      for (int i = 0; i < 8 * RT; ++i) weigh(s_cur, i);
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) l_run[rt] += lsum[rt];
    if (__builtin_expect(rescale, 0)) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        if (CORRECTED || QUANT) l_rounded[rt] *= alpha[rt];
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[rt][dt][e] *= alpha[rt];
      }
    }
    __builtin_amdgcn_s_setprio(1);
    multiply_pv(v_stage(t));
    __builtin_amdgcn_s_setprio(0);
    off_next = off_k;
  };
  if (t_begin < t_end) {
    __syncthreads();
    if constexpr (QUANT) {
      QuantGroup<D> next;
      codes.load_k(quant_at(t_begin), lane);
      codes.load_v(quant_at(t_begin), lane);
      next.load_k(quant_at(t_begin + 1), lane);
      next.load_v(quant_at(t_begin + 1), lane);
      full_next = is_full(t_begin);
      if (!full_next) clear_codes(t_begin);
#pragma unroll
      for (int i = 0; i < KS; ++i) put_k(t_begin, i);
#pragma unroll
      for (int j = 0; j < 4; ++j) put_v(t_begin, j);
      codes = next;
#pragma unroll
      for (int i = 0; i < KS; ++i) put_k(t_begin + 1, i);
      codes.load_k(quant_at(t_begin + 2), lane);
    } else {
      const int64_t off0 = offset_of(t_begin);
      off_next = offset_of(t_begin + 1);
#pragma unroll
      for (int i = 0; i < LPW; ++i) load_k(t_begin, off0, i);
#pragma unroll
      for (int i = 0; i < LPW; ++i) load_v(t_begin, off0, i);
#pragma unroll
      for (int i = 0; i < LPW; ++i) load_k(t_begin + 1, off_next, i);
      wait_loads();
    }
    __syncthreads();
    multiply_qk(k_stage(t_begin), s_a, [](int) {});
    for (int t = t_begin; t < t_end; t += 2) {
      iteration(t, s_a, s_b);
      if (t + 1 >= t_end) break;
      iteration(t + 1, s_b, s_a);
    }
    wait_loads();  // what was asked for past the end must land before the workgroup's LDS is anybody else's
  }

  // ---- results ---------------------------------------------------------------------
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const float l = rows_sum(l_run[rt]), m = l == 0.0f ? -INFINITY : m_run[rt];
    if (corrected) {
      const float rounded = rows_sum(l_rounded[rt]), correction = rounded == 0.0f ? 1.0f : l / rounded;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[rt][dt][e] *= correction;
    }
    const int r = row0 + w_rows * (16 * RT) + rt * 16 + n;
    if (r >= n_rows) continue;
    const int tok = token_of(r);
    const int64_t token = tokens.begin + tok, head = kv_head * p.group + (QUANT ? r - tok * p.group : r % p.group);
    if (ranked && src.by_few) {
      if ((g == 0) & (share == 0)) p.cuts[token * p.n_heads_q + head] = cut_of(first_piece, n_shares, 0, r - row0);
      if (n_shares > 1) {
        const int64_t at = (int64_t)(first_piece + share) * 2 * BM + (r - row0);
        if (g == 0) p.slot_sums[at] = f32x2{m, l};
        float* to = p.slot_out + at * D + 4 * g;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4*>(to + 16 * dt) = o[rt][dt];
        continue;
      }
    } else if (!p.direct) {
      const int64_t at = ((int64_t)(src.first_share + share) * p.n_tokens + token) * p.n_heads_q + head;
      if (g == 0) p.partial_sums[at] = f32x2{m, l};
      if (share >= n_shares) continue;  // (nothing is read of a share without weights)
      float* to = p.partial_out + at * D + 4 * g;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4*>(to + 16 * dt) = o[rt][dt];
      continue;
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) store_row_piece<DTYPE>(p, token, head, 16 * dt + 4 * g, o[rt][dt], m, l);
  }
}

// ---- host ---------------------------------------------------------------------------

// Tiles of `rows` rows of one kv head: every request may have a partial one.  (Of the last one, tile floor(first_row / rows) + batch - 1 + i with
// i < ceil(its rows / rows).)
template <typename Args>
int64_t row_tiles(const Args& x, int batch, int rows = kRowsBM) {
  return ((int64_t)x.n_tokens * (x.n_heads_q / x.n_heads_kv) - 1) / rows + batch;
}
// Row tiles that go to one XCD together: of one request (or prefix), 16 at most and about equal.  us, single tiles and groups:
// two prompts of 2048 behind 14336 keys 330 and 265, 16 of 100 behind 900 54 and 43, one of 8192 from its start 520 and 502.
template <typename Args>
int row_group(const Args& x, int batch, int rows = kRowsBM) {
  const int each = std::max((int)(row_tiles(x, batch, rows) / batch), 1), n = (each + 15) / 16;
  return (each + n - 1) / n;
}
// Shares of a tile's keys: the number that by these figures takes least (us, head size 128, at the longest lengths).  A workgroup begins
// and ends in 7 and takes 1.1 a tile where it has a CU to itself, 2.0 where two share one; the shares are written and
// read at 3 TB/s, in a kernel that takes 3.5 more.  Measured, us by shares: a prompt of 1024 (256 workgroups at one share) 29 at 1, 41 at 2,
// 49 at 4; 3 of 13 tokens of 542 keys 18 at 1 and 16 at 4; 300 tokens behind 8192 keys 152 at 1, 90 at 2, 68 at 4, 60 at 6, 82 at 16;
// 64 requests on a prefix of 32768 106 at 8, 75 at 16, 81 at 32; 83 on one of 13447 47 at 8, 35 at 16 and 43 at 21, where an XCD has 33
// workgroups for its 32 CUs; 64 tokens behind 131072 keys 2490 at 1, 337 at 8, 198 at 16, 162 at 32.
struct RowShares {
  int n;
  double us;
};
template <typename Args>
RowShares row_shares(const Args& x, int batch, int64_t max_keys, bool joined_anyway, int tile_rows = kRowsBM) {
  // (about as many tiles as have rows: row_tiles has room for more)
  const int64_t rows = (int64_t)x.n_tokens * (x.n_heads_q / x.n_heads_kv);
  const int64_t row_tiles_there = std::max<int64_t>((rows + tile_rows - 1) / tile_rows, batch), group = row_group(x, batch, tile_rows);
  const int64_t groups = (row_tiles_there + group - 1) / group * x.n_heads_kv;
  const int64_t tiles = (max_keys + kRowsBN - 1) / kRowsBN;
  const int most = (int)std::min<int64_t>(std::max<int64_t>(tiles / kMinTilesPerShare, 1), 64), n_cu = device_cu_count();
  const double share_us = (double)x.n_tokens * x.n_heads_q * (x.head_dim + 2) * sizeof(float) * 2 / 3e6;
  RowShares best = {1, 1e30};
  for (int s = 1; s <= most; ++s) {
    const int64_t n_wg = xcd_grid_size(groups * s, 1) * group, rounds = (n_wg + 2 * n_cu - 1) / (2 * n_cu);
    const double us = rounds * (7 + (double)tiles / s * (n_wg <= n_cu ? 1.0 + 0.1 * x.head_dim / 128 : 0.5 + 1.5 * x.head_dim / 128)) + (s > 1 || joined_anyway ? s * share_us : 0) +
                      (s > 1 && !joined_anyway ? 3.5 : 0);
    if (us < best.us) best = {s, us};
  }
  return best;
}

}  // namespace dcp
