// Attention over a paged K/V cache for gfx950: causal or with a sliding window and first tokens that stay visible, for any
// number of new tokens a request, and for batches that share long prefixes.
//
//   out = softmax(scale q K^T) V over the visible keys, lse = log sum exp
//
// A query's row is one (token, q head).  The rows of a kv head's group and of neighbouring tokens read the same keys, so they are
// taken together: row r of a request stands for token r / group and head r % group of the kv head.
//
// Two kernels, by how many rows a request has for a kv head (at most, as far as the host knows): the kernel of few rows (up to 32:
// answering token by token), which the keys' bytes bound, and the kernel of rows (prompts, and prefixes that many requests
// share), which the matrix instructions bound.  Both form the products transposed, so that a lane holds one row:
//
//   S^T[key, row] = K Q^T      A = rows of K, B = Q in registers
//   O^T[d,   row] = V^T P^T    A = columns of V (transposing LDS reads), B = P^T straight from the S^T accumulators
//
// with 16x16x32 products: lane l = 16 g + n holds row n of 16 and keys 4 g .. 4 g + 3 of 16 (of O^T: those of d).
//
// Keys are taken in groups of 16 that lie in one page (page sizes are multiples of 16): a page is looked up once a group.  A window
// and the first tokens are two runs of groups laid end to end; nothing in between is read.  What lies in a group and is
// seen by no row (behind the last key, between the first tokens and the window, in a page that is not one) may hold anything: its
// scores are masked by selection, and its V cleared in LDS by the lanes that brought it, since a weight of zero does not
// make a NaN vanish.
#include <math.h>

#include <algorithm>

#include "attn_common.h"
#include "record.h"

namespace dcp {

// Keys that rows look at: the requests' own, or prefixes that requests share.
struct PagedSource {
  const int32_t* block_table;
  const int32_t* key_lens;
  const int32_t* cu_groups;  // prefixes: their requests; null for the requests' own keys
  int64_t table_stride;
  int table_width, batch;    // of prefixes or requests
  int first_share, n_shares; // see PagedParams::partial_out
  int n_tiles, xcd_group;    // row tiles of a kv head (kernel of rows); as many neighbouring work items are on one XCD
  int by_few;                // the kernel of few rows takes it and may cut it (own keys)
};

struct PagedParams {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  float* lse;
  const int32_t* cu_seqlens_q;  // null: one token a request
  int64_t q_token, q_head, out_token, out_head;  // element strides
  int64_t page_stride, token_stride, head_stride;
  PagedSource own, prefix;  // (prefix.batch 0: none)
  int n_pages, page_size;
  int n_requests, n_tokens;  // of q
  int n_heads_q, n_heads_kv, group;
  int window, n_starting;  // of the own keys; window 0: none
  float scale_log2;
  int direct;  // a row whose keys one workgroup takes is finished there
  // Shares of a row's keys, joined afterwards: [share][token][q head], O relative to the maximum, the maximum (log2 domain) and
  // the sum of the weights.  The own keys have shares [0, own.n_shares), the prefixes those that follow.
  float* partial_out;
  f32x2* partial_sums;
  // The kernel of few rows: pieces of the units that are cut between workgroups, and where a row's pieces are (cut_of):
  // [token][q head]
  int2* cuts;
  float* slot_out;   // [workgroup][2][head of the workgroup][rows][D]
  f32x2* slot_sums;  // [workgroup][2][head of the workgroup][rows]
  int few_rows, few_heads_log2;  // rows of a unit; kv heads a workgroup takes at once: 1, 2 or 4
  int few_whole;                 // a workgroup takes a unit
  int n_few, few_first;     // workgroups; of paged_both_kernel those before the ones of rows
  int merge_sets;           // of lanes that share a row in the merge, a power of two
};
typedef KernArgs<PagedParams> PagedArgs;
typedef KernArgs<PagedSource> SourceArgs;

// The tokens of request (or prefix) b.  Cut to the tensor, whatever the tables say.
struct TokenRange {
  int begin, n;
};
__device__ __forceinline__ int first_token(PagedArgs& p, SourceArgs& src, int b) {
  int r = b;
  if (src.cu_groups != nullptr) r = min(max(src.cu_groups[b], 0), p.n_requests);
  if (p.cu_seqlens_q != nullptr) r = p.cu_seqlens_q[r];
  return min(max(r, 0), p.n_tokens);
}
__device__ __forceinline__ TokenRange tokens_of(PagedArgs& p, SourceArgs& src, int b) {
  const int begin = first_token(p, src, b);
  return {begin, max(first_token(p, src, b + 1) - begin, 0)};
}
// Its keys: those that its row of pages has room for.
__device__ __forceinline__ int keys_of(PagedArgs& p, SourceArgs& src, int b) {
  return min(max(src.key_lens[b], 0), p.n_pages > 0 ? src.table_width * p.page_size : 0);
}

// The 16-key groups that rows at positions [first, last] see: [0, n_first) and then [begin, end).
struct KeyGroups {
  int n_first, begin, end;
  int window_begin, hull_end, n_starting;  // keys from hull_end on, and between the first ones and the window, are seen by none
  __device__ __forceinline__ KeyGroups(int window, int starting, int first, int last) {
    n_starting = starting;
    hull_end = last + 1;
    end = (hull_end + 15) / 16;
    window_begin = window > 0 ? max(first - window + 1, 0) : 0;
    begin = window_begin / 16;
    n_first = min(starting / 16 + (starting % 16 != 0), end);
    if (n_first >= begin) begin = n_first = 0;  // one run
  }
  __device__ __forceinline__ int count() const { return n_first + end - begin; }
  __device__ __forceinline__ int at(int i) const { return i < n_first ? i : i - n_first + begin; }
  __device__ __forceinline__ bool sees(int key) const { return (key < hull_end) & ((key < n_starting) | (key >= window_begin)); }
  __device__ __forceinline__ bool sees_all_of_16(int key) const {
    return (key + 15 < hull_end) & ((key + 15 < n_starting) | (key >= window_begin));
  }
};
constexpr int kNoKey = 0x7fffff00;  // of a group that is not there: past every row's last key

__device__ __forceinline__ float rows_max(float x) {  // over the lanes of one n: the four groups of 16 lanes
  const unsigned u = __float_as_uint(x);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return halves_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float rows_sum(float x) {
  const unsigned u = __float_as_uint(x);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return halves_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

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

// The result of a row's 4 elements, from the sum of the weights.
template <int DTYPE>
__device__ __forceinline__ void store_row_piece(PagedArgs& p, int64_t token, int64_t head, int d, f32x4 o, float m, float l) {
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  *reinterpret_cast<u32x2*>(reinterpret_cast<uint16_t*>(p.out) + token * p.out_token + head * p.out_head + d) =
      u32x2{pack2<DTYPE>(o[0] * inv, o[1] * inv), pack2<DTYPE>(o[2] * inv, o[3] * inv)};
  if (d == 0) p.lse[head * p.n_tokens + token] = l == 0.0f ? INFINITY : (m + log2f(l)) * kLn2;
}

// ---------------------------------------------------------------------------
// The kernel of rows: a workgroup of 4 waves owns 128 rows of one (request, kv head), a wave 32 of them, and walks its share of the
// 64-key tiles that any of them sees.  K and V tiles go from memory straight into LDS (KvTile), two stages each, K a tile
// ahead of V: S^T of tile t + 1 is multiplied while tile t is exponentiated, MFMA by MFMA in one stream, O^T += V^T P^T
// of tile t follows as a dense run that the SIMD's other wave fills with its own arithmetic.
// ---------------------------------------------------------------------------
constexpr int kRowsThreads = 256, kRowsBM = 128, kRowsBN = 64;
constexpr int kMinTilesPerShare = 2;
constexpr float kNoMax = -3.0e38f;  // the reference of a row that has seen nothing: below every score, and a weight of -inf against it is 0
constexpr float kMaxTileSum = 16384.0f;  // of a lane's weights against a reference that is not their maximum: fp16 can hold them

// Sum over the wave's lanes up to and with this one.
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);   // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);   // row_shr:2
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);   // row_shr:4
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);   // row_shr:8
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31 into rows 2 and 3
  return x;
}

// The row tile of place `place`, the last one first: tile number `index` of request b's (negative: there is none).
struct RowTile {
  int b, index;
  TokenRange tokens;
  int n_keys;
};
__device__ __forceinline__ RowTile find_row_tile(PagedArgs& p, SourceArgs& src, int place) {
  const int lane = threadIdx.x & 63;
  // Up to 64 requests are counted.  Of more, request b's tiles begin at number floor(first_row / 128) + b: that leaves room for its last,
  // partial one, and needs no sum over the requests before it, but its places without a tile lie among the others, and CUs with two tiles
  // beside CUs with none (24 requests of 128 rows on 1024 keys, nearly half of the places empty: 40 us, counted 35; 64 of 64 rows on 4096 267
  // and 213).
  auto start = [&](int first, int b) { return (int)((int64_t)first * p.group / kRowsBM) + b; };
  const bool counted = src.batch <= 64;
  int tile = src.n_tiles - 1 - place, lo = 0, hi = src.batch;  // the last request that begins at or before the tile; 64 candidates a step
  while (hi - lo > 64) {
    const int step = (hi - lo + 63) / 64, b = lo + lane * step;
    const bool before = b < hi && start(first_token(p, src, b), b) <= tile;
    const int n = __popcll(__ballot(before));
    if (n > 1) lo += (n - 1) * step;
    hi = min(lo + step, hi);
  }
  // A lane looks at one request, and at all there is to know of it: another trip to memory for the one that is found is a microsecond.
  const int b = min(lo + lane, hi - 1);
  const TokenRange tokens = tokens_of(p, src, b);
  const int n_keys = keys_of(p, src, b), n_tiles = (tokens.n * p.group + kRowsBM - 1) / kRowsBM;
  int first_tile = start(tokens.begin, b), passed;
  if (counted) {
    const int ends = wave_scan(lane < hi ? n_tiles : 0);
    tile = __builtin_amdgcn_readlane(ends, 63) - 1 - place;
    first_tile = ends - n_tiles;
    passed = __popcll(__ballot((lane < hi) & (ends <= tile)));
  } else {
    passed = max(__popcll(__ballot((lo + lane < hi) & (first_tile <= tile))) - 1, 0);
  }
  const int at = __builtin_amdgcn_readfirstlane(min(passed, hi - lo - 1));
  auto of = [&](int x) { return __builtin_amdgcn_readlane(x, at); };
  const int index = of(tile - first_tile);
  return {of(b), (tile >= 0) & (index < of(n_tiles)) ? index : -1, {of(tokens.begin), of(tokens.n)}, of(n_keys)};
}

// Which work item workgroup `wg` takes.  The items of a group, `group` neighbouring row tiles of a kv head, read the same keys and go to one
// XCD (workgroup ids go round the eight), whose L2 then reads them once.  From one round of eight groups to the next the XCDs
// move on by one, so that the groups of one kv head do not all go to the same XCD where there are eight.  The tiles of a request's last
// tokens, which see the most, come first, places without a tile last.
struct RowItem {
  int place, kv_head, share;  // share: -1 for none
};
__device__ __forceinline__ RowItem row_item(int wg, int n_tiles, int group, int n_heads_kv, int n_shares) {
  const int per_round = kNumXcd * group, round = wg / per_round, in_round = wg - round * per_round;
  int i = round * kNumXcd + (in_round + round) % kNumXcd;  // the group
  const int kv_head = i % n_heads_kv;
  i /= n_heads_kv;
  const int place = i / n_shares * group + in_round / kNumXcd, share = i % n_shares;
  return {place, kv_head, place < n_tiles ? share : -1};
}
inline int64_t row_workgroups(int64_t n_tiles, int group, int n_heads_kv, int n_shares) {
  return xcd_grid_size((n_tiles + group - 1) / group * n_heads_kv * n_shares, 1) * group;
}

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
template <int DTYPE, int D, bool CORRECTED>
__device__ __forceinline__ void paged_rows(PagedArgs& p, SourceArgs& src, int item, char* lds) {
  typedef KvTile<D> Tile;
  constexpr int KS = D / 32, DT = D / 16, RT = 2, LPW = Tile::LPW;
  typedef RowsLds<D> Lds;
  constexpr int TILE_BYTES = Lds::TILE;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);

  // ---- which rows, which share of their keys ---------------------------------
  const RowItem at = row_item(item, src.n_tiles, src.xcd_group, p.n_heads_kv, src.n_shares);
  if (at.share < 0) return;
  const int place = __builtin_amdgcn_readfirstlane(at.place), kv_head = __builtin_amdgcn_readfirstlane(at.kv_head);
  const int share = __builtin_amdgcn_readfirstlane(at.share);
  const RowTile tile = find_row_tile(p, src, place);
  const TokenRange tokens = tile.tokens;
  const int n_rows = tokens.n * p.group;  // (at most n_tokens * group, which the host has checked)
  const int row0 = tile.index * kRowsBM;
  if (tile.index < 0) return;
  const bool prefix = src.cu_groups != nullptr;
  const int n_keys = tile.n_keys, window = prefix ? 0 : p.window, n_starting = p.n_starting;
  // token i of the request is at position n_keys - n + i; every token is past all of a prefix
  const int first_tok = row0 / p.group, last_tok = (min(row0 + kRowsBM, n_rows) - 1) / p.group;
  const int at0 = prefix ? n_keys - 1 : n_keys - tokens.n, step = prefix ? 0 : 1;
  const KeyGroups groups(window, n_starting, max(at0 + first_tok * step, 0), at0 + last_tok * step);
  const int n_groups = __builtin_amdgcn_readfirstlane(groups.hull_end > 0 ? groups.count() : 0);
  const int tiles_all = (n_groups + 3) / 4, n_shares = min(src.n_shares, max(1, tiles_all / kMinTilesPerShare));
  int t_begin = 0, t_end = 0;
  if (share < n_shares) {
    t_begin = __builtin_amdgcn_readfirstlane((int)((int64_t)tiles_all * share / n_shares));
    t_end = __builtin_amdgcn_readfirstlane((int)((int64_t)tiles_all * (share + 1) / n_shares));
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
    const int entry = key / p.page_size;
    return {key, key - entry * p.page_size, src.block_table[tile.b * src.table_stride + entry]};
  };
  auto look_up = [&](int rel, Entry entry) {
    PagedArgs& p = fresh_kernel_args<PagedParams>();
    const bool there = (unsigned)entry.page < (unsigned)p.n_pages;
    const int at = (rel * 4 + tid) % (2 * kTableTiles * 4);
    offsets[at] = there ? entry.page * p.page_stride + entry.in_page * p.token_stride : 0;
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
    const int r = min(row0 + w * 32 + rt * 16 + n, n_rows - 1), tok = r / p.group, head = kv_head * p.group + r % p.group;
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
    rescale = __any((alpha[0] != 1.0f) | (alpha[1] != 1.0f));
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
  int64_t off_next = 0;  // of tile t + 1, whose K is there and whose V is asked for in iteration t
  auto iteration = [&](int t, f32x4 (&s_cur)[RT][4], f32x4 (&s_nxt)[RT][4]) {
    wait_loads();
    const bool full = is_full(t);
    if (__builtin_expect(!full, 0)) clear_v(t);
    if (__builtin_expect((t - t_begin) % kTableTiles == kTableTiles / 2, 0)) {
      const int rel = (t - t_begin) / kTableTiles * kTableTiles + kTableTiles;
      look_up(rel, read_entry(rel));
    }
    __syncthreads();  // K of tile t + 1 and V of tile t are there; nobody reads K of tile t or V of tile t - 1 any more
    // The loads of K of tile t + 2 and V of tile t + 1 go out between the products, unconditionally: past the end a page that there
    // is comes into a stage that nobody reads any more.
    const int64_t off_k = offset_of(t + 2);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) lsum[rt] = 0.0f;
    bool taken = false;  // the tile's maximum
    rescale = false;
    if (__builtin_expect(!(full & anchored), 0)) {
      if (!full) mask(t, s_cur);
      raise(s_cur);
      taken = true;
    }
    // Where every row has a reference and sees the whole tile, its weights are taken against that without looking for its own
    // maximum; the lanes' sums tell afterwards whether that was safe, and if not it is done again.
    __builtin_amdgcn_s_setprio(2);
    constexpr int N = 4 * KS, NL = 2 * LPW;
    multiply_qk(k_stage(t + 1), s_nxt, [&](int i) {
      constexpr int PAIRS = 16 / N;
#pragma unroll
      for (int x = 0; x < PAIRS; ++x) weigh(s_cur, i * PAIRS + x);
      if (i < LPW) load_k(t, off_k, i);
      else if (i < NL) load_v(t + 1, off_next, i - LPW);
    });
    if (__builtin_expect(!taken & __any(!((lsum[0] < kMaxTileSum) & (lsum[1] < kMaxTileSum))), 0)) {
      raise(s_cur);
#pragma unroll
      for (int i = 0; i < 16; ++i) weigh(s_cur, i);
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) l_run[rt] += lsum[rt];
    if (__builtin_expect(rescale, 0)) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        if (CORRECTED) l_rounded[rt] *= alpha[rt];
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
    const int64_t off0 = offset_of(t_begin);
    off_next = offset_of(t_begin + 1);
#pragma unroll
    for (int i = 0; i < LPW; ++i) load_k(t_begin, off0, i);
#pragma unroll
    for (int i = 0; i < LPW; ++i) load_v(t_begin, off0, i);
#pragma unroll
    for (int i = 0; i < LPW; ++i) load_k(t_begin + 1, off_next, i);
    wait_loads();
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
    if constexpr (CORRECTED) {
      const float rounded = rows_sum(l_rounded[rt]), correction = rounded == 0.0f ? 1.0f : l / rounded;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[rt][dt][e] *= correction;
    }
    const int r = row0 + w * 32 + rt * 16 + n;
    if (r >= n_rows) continue;
    const int64_t token = tokens.begin + r / p.group, head = kv_head * p.group + r % p.group;
    if (!p.direct) {
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

// ---------------------------------------------------------------------------
// The kernel of few rows: the waves of a workgroup share no tile.  Each takes tiles of 32 keys of its own, K and V into its own part of
// LDS, and waits for nobody until its share of the keys is done.  (K straight into registers, in the layout of the product,
// takes no LDS and no reads of it, but its 16 lanes of a row's end lie in 16 rows: a CU's loads went at a fifth of its rate, a tile took a
// lone workgroup 3.5 us instead of 2.3, and all of them 2-10 % more.)
//
// Work is cut by length, not by request: the tiles of all (request, rows, kv heads) units are laid end to end and every workgroup
// takes the same number of them, whatever the lengths are (they are known on the device only).  A unit inside one workgroup's
// share is finished there; of one that is cut each piece goes to the workgroup's slot (0: the share begins in the unit, 1: it
// ends in it) and the merge joins them.
//
// Several kv heads at once: in a cache by token ([page][token][head]) a head's row is 256 bytes, and four heads' waves
// side by side read 1 KiB of a token at about the same time: four contexts of 131072 keys 344 us by one head and 321 by four (in a
// cache by head 319 and 335).  With few tiles a workgroup the waves take turns at one head's tiles instead, which makes the chain of
// tiles shorter.
// ---------------------------------------------------------------------------
// What the merge needs to know of a row: the workgroup that begins its unit, how many the unit is cut over, the slot of the first
// piece (the others are in slot 0) and the row in the slots.
__device__ __forceinline__ int2 cut_of(int wg, int n_pieces, int slot, int row) { return int2{wg, n_pieces | row << 20 | slot << 28}; }
constexpr int kFewBN = 32;
constexpr int kFewMaxBatch = 1 << 16;

// What request b is to the kernel.
struct FewRequest {
  int first_tok, n_tok, n_keys, n_tiles;
  __device__ __forceinline__ KeyGroups groups(PagedArgs& p) const {
    return KeyGroups(p.window, p.n_starting, max(n_keys - n_tok, 0), n_keys - 1);
  }
  __device__ __forceinline__ FewRequest() {}
  __device__ __forceinline__ FewRequest(PagedArgs& p, int b) {
    const TokenRange tokens = tokens_of(p, p.own, b);
    first_tok = tokens.begin;
    n_tok = tokens.n;
    n_keys = keys_of(p, p.own, b);
    n_tiles = max((groups(p).count() + 1) / 2, 1);  // (a request without keys has its rows written all the same)
  }
  __device__ __forceinline__ int units(PagedArgs& p, int rows) const {
    return (n_tok * p.group + rows - 1) / rows * (p.n_heads_kv >> p.few_heads_log2);
  }
  __device__ __forceinline__ FewRequest of_lane(int lane) const {
    FewRequest r;
    r.first_tok = __builtin_amdgcn_readlane(first_tok, lane);
    r.n_tok = __builtin_amdgcn_readlane(n_tok, lane);
    r.n_keys = __builtin_amdgcn_readlane(n_keys, lane);
    r.n_tiles = __builtin_amdgcn_readlane(n_tiles, lane);
    return r;
  }
};

__device__ __forceinline__ int64_t lane_value(int64_t x, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane((int)x, lane), hi = __builtin_amdgcn_readlane((int)(x >> 32), lane);
  return (int64_t)(((uint64_t)hi << 32) | lo);
}

// LDS of the kernel.  V of 32 keys: load r of a tile brings rows r, r + LOADS, ... side by side (1 KiB), 32 bytes of padding between
// loads: eight consecutive rows then lie in eight different 32-byte bank windows for the transposing reads.
template <int D, int RT, int NW>
struct FewLds {
  static constexpr int ROWS = 16 * RT, LOADS = kFewBN * D * 2 / 1024, LOAD_BYTES = 1024 + 32, STAGE = LOADS * LOAD_BYTES;
  static constexpr int O_STRIDE = D + 4;  // floats: rows of a wave's result, which takes the place of its K and as much of its V as it needs
  static constexpr int WAVE = 2 * STAGE > ROWS * O_STRIDE * 4 ? 2 * STAGE : ROWS * O_STRIDE * 4;
  static constexpr int SUMS = NW * WAVE;                  // float [wave][row][2]
  static constexpr int CHUNKS = SUMS + NW * ROWS * 2 * 4; // int [batch / 64]
  static constexpr int BYTES = CHUNKS + kFewMaxBatch / 64 * 4;
};

template <int DTYPE, int D, int RT, int NW>
__device__ __forceinline__ void paged_few(int wg, char* lds) {
  // (the arguments are read anew wherever another part of the work begins: kept in scalar registers throughout they do not fit)
  PagedArgs& p0 = fresh_kernel_args<PagedParams>();
  typedef FewLds<D, RT, NW> Lds;
  constexpr int KS = D / 32, DT = D / 16, ROWS = Lds::ROWS, LOADS = Lds::LOADS;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  float(*sums)[ROWS][2] = reinterpret_cast<float(*)[ROWS][2]>(lds + Lds::SUMS);
  int* chunk_sums = reinterpret_cast<int*>(lds + Lds::CHUNKS);

  // ---- this workgroup's share of all tiles (the host has checked that their number fits 32 bits), or its unit -----------
  const int n_chunks = (p0.own.batch + 63) / 64;
  const bool whole_units = p0.few_whole != 0;
  // Shares are counted in turns of the waves at a head's tiles: a cut inside one would cost both of its sides a whole one.  (One context
  // of 1500 keys, 8 heads, which 47 tiles a head then fit no better: counted in tiles 14.4 us, in turns 11.4.)
  const int turns_log2 = (NW == 8 ? 3 : 2) - p0.few_heads_log2, turns = 1 << turns_log2;
  auto requests_of = [&](int chunk, int& work) {
    PagedArgs& p = fresh_kernel_args<PagedParams>();
    const int b = chunk * 64 + lane;
    FewRequest r;
    r.first_tok = r.n_tok = r.n_keys = 0;
    r.n_tiles = 1;
    work = 0;
    if (b < p.own.batch) {
      r = FewRequest(p, b);
      work = r.units(p, ROWS) * (whole_units ? 1 : (r.n_tiles + turns - 1) >> turns_log2);
    }
    return r;
  };
  int total = 0, before = 0, chunk = 0, work;
  FewRequest requests = requests_of(0, work);
  int scan = wave_scan(work);  // the chunk's tiles (or units) up to and with the lane's request
  if (n_chunks == 1) {
    total = __builtin_amdgcn_readlane(scan, 63);
  } else {
    for (int i = w; i < n_chunks; i += NW) {
      int more;
      requests_of(i, more);
      more = wave_scan(more);
      if (lane == 63) chunk_sums[i] = more;
    }
    __syncthreads();
    for (int i = 0; i < n_chunks; i += 64) total += __builtin_amdgcn_readlane(wave_scan(i + lane < n_chunks ? chunk_sums[i + lane] : 0), 63);
  }
  const int per = whole_units ? 1 : (total - 1) / p0.n_few + 1;
  const int begin = (int)min((int64_t)wg * per, (int64_t)total), end = (int)min((int64_t)begin + per, (int64_t)total);
  if (begin >= end) return;
  if (n_chunks > 1) {
    for (int i = 0; i < n_chunks; i += 64) {
      const int ends = before + wave_scan(i + lane < n_chunks ? chunk_sums[i + lane] : 0);
      const int passed = __popcll(__ballot(ends <= begin));
      if (passed > 0) before = __builtin_amdgcn_readlane(ends, passed - 1);
      chunk = i + passed;
      if (passed < 64) break;
    }
    chunk = __builtin_amdgcn_readfirstlane(min(chunk, n_chunks - 1));
    requests = requests_of(chunk, work);
    scan = wave_scan(work);
  }
  int index = __builtin_amdgcn_readfirstlane(min(__popcll(__ballot(before + scan <= begin)), 63));  // in the chunk

  char* my_lds = lds + w * Lds::WAVE;  // K of a tile and V of a tile
  const uint32_t k_at = lds_address(lds) + w * Lds::WAVE, v_at = k_at + Lds::STAGE;
  int at = begin;
  while (at < end) {
    if (index == 64) {
      before += __builtin_amdgcn_readlane(scan, 63);
      if (++chunk >= n_chunks) break;
      requests = requests_of(chunk, work);
      scan = wave_scan(work);
      index = 0;
    }
    const int unit_end = before + __builtin_amdgcn_readlane(scan, index);
    if (at >= unit_end) {  // (no rows, or done)
      ++index;
      continue;
    }
    PagedArgs& p = fresh_kernel_args<PagedParams>();
    // the workgroup's kv heads at once, the waves that take turns at a head's tiles, and which of each the wave is
    const int heads = 1 << p.few_heads_log2, head_groups = p.n_heads_kv >> p.few_heads_log2;
    const int my_head = w & (heads - 1), my_turn = w >> p.few_heads_log2;
    const FewRequest request = requests.of_lane(index);
    const int b = chunk * 64 + index, in_request = at - (unit_end - __builtin_amdgcn_readlane(work, index));
    if (in_request < 0) break;  // (tables whose tokens are many times those there are: their sums wrap)
    const int unit_turns = whole_units ? 1 : (request.n_tiles + turns - 1) >> turns_log2;
    const int unit = __builtin_amdgcn_readfirstlane(in_request / unit_turns);
    const int first_turn = in_request - unit * unit_turns, taken = min(unit_turns - first_turn, end - at);
    const int t_begin = whole_units ? 0 : first_turn * turns, t_end = whole_units ? request.n_tiles : min(request.n_tiles, t_begin + taken * turns);
    at += taken;
    const int kv_head0 = unit % head_groups * heads, kv_head = kv_head0 + my_head, row0 = unit / head_groups * ROWS;
    const KeyGroups groups = request.groups(p);
    const int n_groups = request.n_keys > 0 ? groups.count() : 0, n_rows = request.n_tok * p.group;

    // ---- where the wave's next 32 tiles are: lane 2 i + j holds the 16-key group j of the i-th of them ------------
    int64_t lane_off = 0;
    int lane_key = kNoKey;
    auto look_up = [&](int step) {
      PagedArgs& p = fresh_kernel_args<PagedParams>();
      const int group = 2 * (t_begin + my_turn + turns * (step + (lane >> 1))) + (lane & 1);
      lane_off = 0;
      lane_key = kNoKey;
      if (group < n_groups && group < 2 * t_end) {
        const int key = groups.at(group) * 16, entry = key / p.page_size;
        const int page = p.own.block_table[b * p.own.table_stride + entry];
        if ((unsigned)page < (unsigned)p.n_pages) {
          lane_key = key;
          lane_off = page * p.page_stride + (int64_t)(key - entry * p.page_size) * p.token_stride;
        }
      }
    };
    // what a lane brings of a tile's K and V: a piece of LOADS rows of its half's group
    constexpr int CH = D / 8;
    const int lane_row = lane / CH % (16 / LOADS) * LOADS;  // of load 0
    const int64_t token_stride = p.token_stride;
    const uint16_t* k_lane = reinterpret_cast<const uint16_t*>(p.k) + (kv_head * p.head_stride + lane_row * token_stride + lane % CH * 8);
    const int64_t v_from_k = reinterpret_cast<const uint16_t*>(p.v) - reinterpret_cast<const uint16_t*>(p.k);
    const int n_steps = n_groups > 0 && t_begin + my_turn < t_end ? (t_end - t_begin - my_turn + turns - 1) / turns : 0;
    int64_t off = 0;  // where the lane's group of the next tile is
    int next_key[2], tile_key[2];
    auto place = [&](int step) {
      if (step % 32 == 0) look_up(step);
      const int from = 2 * (step % 32);
      const int64_t off0 = lane_value(lane_off, from), off1 = lane_value(lane_off, from + 1);
      off = lane >= 32 ? off1 : off0;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) next_key[kt] = __builtin_amdgcn_readlane(lane_key, from + kt);
    };
    auto issue = [&](uint32_t at, int64_t from_k) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the last reads of what is there are done
#pragma unroll
      for (int r = 0; r < LOADS; ++r) load_async_piece<true>(at + r * Lds::LOAD_BYTES, k_lane + off + (from_k + r * token_stride));
    };
    if (n_steps > 0) {
      place(0);
      issue(k_at, 0);
      issue(v_at, v_from_k);
    }

    // ---- this lane's rows --------------------------------------------------------------
    int last_key[RT], first_key[RT];
    int w_last = 0x7fffffff, w_first = 0;
    u32x4 q[RT][KS];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int r = row0 + rt * 16 + n, tok = r / p.group, head = kv_head * p.group + r % p.group;
      const bool live = r < n_rows;
      const uint16_t* from = reinterpret_cast<const uint16_t*>(p.q) + (request.first_tok + tok) * p.q_token + head * p.q_head + 8 * g;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        q[rt][ks] = u32x4{0, 0, 0, 0};
        if (live) q[rt][ks] = *reinterpret_cast<const u32x4*>(from + 32 * ks);
      }
      last_key[rt] = live ? request.n_keys - request.n_tok + tok : 0x7fffffff;
      first_key[rt] = live && p.window > 0 ? max(last_key[rt] - p.window + 1, 0) : 0;
      w_last = min(w_last, wave_min(last_key[rt]));
      w_first = max(w_first, wave_max(first_key[rt]));
    }
    f32x4 o[RT][DT];
    float m_run[RT], l_run[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      m_run[rt] = -INFINITY;
      l_run[rt] = 0.0f;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[rt][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    auto row_at = [](int row) { return row % LOADS * Lds::LOAD_BYTES + row / LOADS * (D * 2); };  // 16 rows further: 512 bytes
    const int k_rd = row_at(n) + 16 * g, v_rd = row_at(4 * g + (n >> 2)) + 8 * (n & 3);
    for (int step = 0; step < n_steps; ++step) {
      // K and V of the next tile are asked for as soon as those of this one have been read, and waited for on their own: under
      // way are K of a tile while V is at work and V while K is.
      __builtin_amdgcn_s_waitcnt(0x0F70 | LOADS);  // all loads but the last LOADS, which are V's
      asm volatile("" ::: "memory");
      const bool more = step + 1 < n_steps;
      bool whole = true, full = true;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        const int key = tile_key[kt] = next_key[kt];
        whole = whole & groups.sees_all_of_16(key);
        full = full & (key + 15 <= w_last) & ((key >= w_first) | (key + 15 < p.n_starting));
      }
      f32x4 s[RT][2];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) s[rt][kt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const u32x4 a = *reinterpret_cast<const u32x4*>(my_lds + k_rd + 512 * kt + 64 * ks);
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) s[rt][kt] = mfma_16x16x32<DTYPE>(a, q[rt][ks], s[rt][kt]);
        }
      }
      if (more) {
        place(step + 1);
        issue(k_at, 0);
      }
      if (!(whole & full)) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = tile_key[kt] + 4 * g + e;
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
              const bool visible = (key <= last_key[rt]) & ((key < p.n_starting) | (key >= first_key[rt])) & (tile_key[kt] != kNoKey);
              s[rt][kt][e] = visible ? s[rt][kt][e] : -INFINITY;
            }
            __builtin_amdgcn_sched_barrier(0);  // (all conditions at once need more scalar registers than there are)
          }
      }
      u32x4 pb[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        float mx = fmaxf(s[rt][0][0], s[rt][1][0]);
#pragma unroll
        for (int e = 1; e < 4; ++e) mx = fmaxf(mx, fmaxf(s[rt][0][e], s[rt][1][e]));
        mx = rows_max(mx * p.scale_log2);
        const float m_new = fmaxf(m_run[rt], mx);
        if (__any(m_new != m_run[rt])) {
          const float alpha = m_new == -INFINITY ? 1.0f : fast_exp2(m_run[rt] - m_new);
          l_run[rt] *= alpha;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[rt][dt][e] *= alpha;
          m_run[rt] = m_new;
        }
        const float m_use = m_new == -INFINITY ? 0.0f : m_new;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          float x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[e] = fast_exp2(fmaf(s[rt][kt][e], p.scale_log2, -m_use));
            l_run[rt] += x[e];
          }
          // Rounded for the product, summed unrounded, and not CORRECTED: the reference is the row's maximum, whose weight of 1 is
          // exact, and the second sum changed neither the time nor the error (0.0018 in bf16).
          pb[rt][2 * kt] = pack2<DTYPE>(x[0], x[1]);
          pb[rt][2 * kt + 1] = pack2<DTYPE>(x[2], x[3]);
        }
      }
      if (more) __builtin_amdgcn_s_waitcnt(0x0F70 | LOADS);  // (the last LOADS are the next K)
      else wait_loads();
      asm volatile("" ::: "memory");
      if (!whole) {
        const int key0 = lane >= 32 ? tile_key[1] : tile_key[0];
#pragma unroll
        for (int r = 0; r < LOADS; ++r)
          if (!((key0 != kNoKey) & groups.sees(key0 + lane_row + r)))
            *reinterpret_cast<u32x4*>(my_lds + Lds::STAGE + r * Lds::LOAD_BYTES + 16 * lane) = u32x4{0, 0, 0, 0};
        asm volatile("" ::: "memory");
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
        const uint32_t from = v_at + v_rd + 32 * dt;
        const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)from));
        const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)(from + 512)));
        const u32x4 a = {lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) o[rt][dt] = mfma_16x16x32<DTYPE>(a, pb[rt], o[rt][dt]);
      }
      if (more) issue(v_at, v_from_k);
    }

    // ---- the waves' results joined --------------------------------------------------
    asm volatile("" ::: "memory");
    float* mine = reinterpret_cast<float*>(my_lds);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const float l = rows_sum(l_run[rt]);
      if (g == 0) {
        sums[w][rt * 16 + n][0] = m_run[rt];
        sums[w][rt * 16 + n][1] = l;
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4*>(mine + (rt * 16 + n) * Lds::O_STRIDE + 16 * dt + 4 * g) = o[rt][dt];
    }
    __syncthreads();
    PagedArgs& p_out = fresh_kernel_args<PagedParams>();
    const bool cut = taken < unit_turns;
    const int slot = at - taken == begin ? 0 : 1;
    const int n_cut = (at - taken + unit_turns - 1) / per - wg + 1;  // (of a unit that begins here: it ends so many workgroups on)
    const int group = p_out.group;
    constexpr int PIECES = D / 4;  // of a row
    for (int i = tid; i < heads * ROWS * PIECES; i += NW * 64) {
      const int piece = i % PIECES, row = i / PIECES % ROWS, of = i / PIECES / ROWS, r = row0 + row;
      if (r >= n_rows) continue;
      float m = -INFINITY;
      for (int x = of; x < NW; x += heads) m = fmaxf(m, sums[x][row][0]);
      const float m_use = m == -INFINITY ? 0.0f : m;
      f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
      float l = 0.0f;
      for (int x = of; x < NW; x += heads) {
        const float weight = fast_exp2(sums[x][row][0] - m_use);
        l += weight * sums[x][row][1];
        const f32x4 o4 = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds + x * Lds::WAVE) + row * Lds::O_STRIDE + 4 * piece);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] += weight * o4[e];
      }
      const int64_t token = request.first_tok + r / group, head = (kv_head0 + of) * group + r % group;
      if ((piece == 0) & (t_begin == 0) & !whole_units) p_out.cuts[token * p_out.n_heads_q + head] = cut_of(wg, n_cut, slot, of * ROWS + row);
      if (cut) {
        const int64_t to = (((int64_t)wg * 2 + slot) * heads + of) * ROWS + row;
        *reinterpret_cast<f32x4*>(p_out.slot_out + to * D + 4 * piece) = acc;
        if (piece == 0) p_out.slot_sums[to] = f32x2{m, l};
      } else if (!p_out.direct) {
        const int64_t to = ((int64_t)p_out.own.first_share * p_out.n_tokens + token) * p_out.n_heads_q + head;
        *reinterpret_cast<f32x4*>(p_out.partial_out + to * D + 4 * piece) = acc;
        if (piece == 0) p_out.partial_sums[to] = f32x2{m, l};
      } else {
        store_row_piece<DTYPE>(p_out, token, head, 4 * piece, acc, m, l);
      }
    }
    __syncthreads();  // nobody's part of LDS is filled again before all have read it
  }
}

// ---- kernels --------------------------------------------------------------------------
template <int DTYPE, int D, bool CORRECTED>
__global__ __launch_bounds__(kRowsThreads, 2) void paged_rows_kernel(const PagedParams) {
  __shared__ __attribute__((aligned(16))) char lds[RowsLds<D>::BYTES];
  PagedArgs& p = fresh_kernel_args<PagedParams>();
  paged_rows<DTYPE, D, CORRECTED>(p, p.own, blockIdx.x, lds);
}

template <int DTYPE, int D, int RT, int NW>
__global__ __launch_bounds__(NW * 64, 2) void paged_few_kernel(const PagedParams) {
  __shared__ __attribute__((aligned(16))) char lds[FewLds<D, RT, NW>::BYTES];
  paged_few<DTYPE, D, RT, NW>(blockIdx.x, lds);
}

// The requests' own keys and prefixes of many rows in one launch: a workgroup of the one starts where one of the other has ended, without
// a kernel's end and another's start between them.  p.few_first workgroups of few rows come first, then those of rows, then the other
// few: all of the few, or one a CU, so that a CU has one of each kind, of which one waits for memory and the other for products.  (In
// turns it is the CUs that take turns: of an XCD's every second has two of rows.)
template <int DTYPE, int D, int RT>
__global__ __launch_bounds__(256, 2) void paged_both_kernel(const PagedParams) {
  __shared__ __attribute__((aligned(16))) char lds[std::max(FewLds<D, RT, 4>::BYTES, RowsLds<D>::BYTES)];
  PagedArgs& p = fresh_kernel_args<PagedParams>();
  const int wg = blockIdx.x, before = p.few_first, n_rows = gridDim.x - p.n_few;
  const bool few = (wg < before) | (wg >= before + n_rows);
  const int i = wg < before ? wg : few ? wg - n_rows : wg - before;
  if (few) paged_few<DTYPE, D, RT, 4>(i, lds);
  else paged_rows<DTYPE, D, true>(p, p.prefix, i, lds);
}

// The merge: out = sum_i 2^(m_i - m) O_i / sum_i 2^(m_i - m) l_i over a row's parts, rounded once.  The parts are the pieces
// of a unit that the kernel of few rows has cut, or shares of the own keys, and the shares of a prefix.  D / 4 lanes hold a
// row in 16-byte pieces; as many sets of such lanes as p.merge_sets take parts of one row in turn (a wave that went through 128
// parts alone took 17 us), the other sets of the workgroup take other rows (a workgroup for each of 32768 rows of two parts 27 us).
constexpr int kPagedMergeThreads = 256;
template <int DTYPE, int D>
__global__ __launch_bounds__(kPagedMergeThreads) void paged_merge_kernel(const PagedParams) {
  PagedArgs& p = fresh_kernel_args<PagedParams>();
  constexpr int PIECES = D / 4, SETS = kPagedMergeThreads / PIECES;
  __shared__ f32x4 acc_lds[SETS][PIECES];
  __shared__ f32x2 sums_lds[SETS];
  const int tid = threadIdx.x, piece = tid % PIECES, set = tid / PIECES, row_sets = p.merge_sets, turn = set % row_sets;
  const int64_t n_rows = (int64_t)p.n_tokens * p.n_heads_q;  // (fits 32 bits)
  const int64_t row64 = (int64_t)blockIdx.x * (SETS / row_sets) + set / row_sets;
  const int row = (int)min(row64, n_rows - 1), token = row / p.n_heads_q, head = row % p.n_heads_q;
  // Every trip to memory here is as long as the sums themselves, so there are three: where the row's parts are and which groups share
  // prefixes; the parts and which tokens the groups and requests have; the stores.  The parts are read before it is known whether the row
  // has any: whatever the entry of a row of no request holds, it is kept to the slots there are, and shares there are of every row.
  int2 cut = {0, 1};
  if (p.own.by_few) cut = p.cuts[row];
  const bool prefixes = p.prefix.batch > 0;
  int first = 0, end = p.n_requests, prefix_first = 0, prefix_end = 0;  // requests, then tokens
  if (prefixes) {
    prefix_first = min(max(p.prefix.cu_groups[0], 0), end);
    prefix_end = min(max(p.prefix.cu_groups[p.prefix.batch], 0), end);
  }
  if (p.cu_seqlens_q != nullptr) {
    const int32_t* cu = p.cu_seqlens_q;
    const int a = cu[first], b = cu[end], c = cu[prefix_first], d = cu[prefix_end];
    first = a; end = b; prefix_first = c; prefix_end = d;
  }
  cut.x = min(max(cut.x, 0), p.n_few);
  const int n_pieces = min(cut.y & 0xfffff, p.n_few - cut.x), n_cut = n_pieces > 1 ? n_pieces : 0;
  const int n_own = n_cut > 0 ? n_cut : p.direct ? 0 : p.own.n_shares;  // (no memory for shares where rows are done at once)
  const int n_parts = n_own + (prefixes ? p.prefix.n_shares : 0);
  const int slot_rows = p.few_rows << p.few_heads_log2, slot_row = min(cut.y >> 20 & 0xff, slot_rows - 1), slot = cut.y >> 28 & 1;
  const bool has_prefix = prefixes && token >= prefix_first && token < prefix_end;
  // rows of no request are left as they were; one that has no parts is done where it was computed
  const bool mine = row64 < n_rows && token >= first && token < end && n_parts > 0;
  // (kept in registers: a choice between two of the arguments was made by loading the chosen one, for every part anew)
  typedef __attribute__((address_space(1))) const f32x4 GlobalOut;
  typedef __attribute__((address_space(1))) const f32x2 GlobalSums;
  GlobalOut *slot_out = (GlobalOut*)p.slot_out, *partial_out = (GlobalOut*)p.partial_out;
  GlobalSums *slot_sums = (GlobalSums*)p.slot_sums, *partial_sums = (GlobalSums*)p.partial_sums;
  asm("" : "+s"(slot_out), "+s"(partial_out), "+s"(slot_sums), "+s"(partial_sums));
  // where part i is
  const int prefix_shift = p.prefix.first_share - n_own;
  auto part = [&](int i, GlobalSums*& sums) -> GlobalOut* {
    const bool in_slot = i < n_cut;
    const int64_t at = in_slot ? ((int64_t)(cut.x + i) * 2 + (i == 0 ? slot : 0)) * slot_rows + slot_row
                               : (int64_t)(i < n_own ? i : i + prefix_shift) * n_rows + row;
    sums = (in_slot ? slot_sums : partial_sums) + at;
    return (in_slot ? slot_out : partial_out) + at * PIECES + piece;
  };
  float m = -INFINITY, l = 0.0f;
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  constexpr int AT_ONCE = 8;
  for (int i0 = turn; i0 < n_parts; i0 += row_sets * AT_ONCE) {
    f32x2 ml[AT_ONCE];
    f32x4 o4[AT_ONCE];
#pragma unroll
    for (int x = 0; x < AT_ONCE; ++x) {
      ml[x] = f32x2{-INFINITY, 0.0f};
      o4[x] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if (i0 + x * row_sets < n_parts) {
        GlobalSums* sums;
        o4[x] = *part(i0 + x * row_sets, sums);
        ml[x] = *sums;
      }
    }
    float m_new = m;
#pragma unroll
    for (int x = 0; x < AT_ONCE; ++x) {
      if (i0 + x * row_sets >= n_own && !has_prefix) ml[x] = f32x2{-INFINITY, 0.0f};
      m_new = fmaxf(m_new, ml[x][0]);
    }
    const float m_use = m_new == -INFINITY ? 0.0f : m_new, old = fast_exp2(m - m_use);
    l *= old;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] *= old;
#pragma unroll
    for (int x = 0; x < AT_ONCE; ++x) {
      const float weight = fast_exp2(ml[x][0] - m_use);
      l += weight * ml[x][1];
      // (nothing is written of a share without weights; one that is not a number stays one)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += weight == 0.0f ? 0.0f : weight * o4[x][e];
    }
    m = m_new;
  }
  if (row_sets > 1) {
    acc_lds[set][piece] = acc;
    if (piece == 0) sums_lds[set] = f32x2{m, l};
    __syncthreads();
    if (turn > 0) return;
    m = -INFINITY;
    for (int x = set; x < set + row_sets; ++x) m = fmaxf(m, sums_lds[x][0]);
    const float m_use = m == -INFINITY ? 0.0f : m;
    l = 0.0f;
    acc = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int x = set; x < set + row_sets; ++x) {
      const float weight = fast_exp2(sums_lds[x][0] - m_use);
      l += weight * sums_lds[x][1];
      const f32x4 o4 = acc_lds[x][piece];
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += weight * o4[e];
    }
  }
  if (mine) store_row_piece<DTYPE>(p, token, head, 4 * piece, acc, m, l);
}

// ---- host ---------------------------------------------------------------------------

// How a call is laid out: which kernel takes which keys, and what of the workspace is whose.
struct PagedPlan {
  bool few = false;    // the kernel of few rows takes the requests' own keys
  bool whole = false;  // a workgroup takes a unit of it; otherwise an equal share of all tiles
  int waves = 4;       // of a workgroup of it
  int rows = 16, heads = 1, n_few = 0;  // rows of a unit, kv heads of a workgroup, workgroups
  int few_first = 0;                    // those before a prefix's
  int n_own = 1, n_prefix = 0;          // shares
  size_t cuts = 0, slots = 0, shares = 0;  // bytes
  size_t bytes() const { return cuts + slots + shares; }
};

// Keys that a request's queries see, of the longest there are.
static int64_t seen_keys(const dcp_paged_attn_args& x) {
  return x.window > 0 ? std::min<int64_t>(x.max_seqlen_k, (int64_t)x.max_seqlen_q + x.window + x.n_starting) : x.max_seqlen_k;
}
// Row tiles of one kv head: every request may have a partial one.  (Of the last one, tile floor(first_row / 128) + batch - 1 + i with
// i < ceil(rows / 128).)
static int64_t row_tiles(const dcp_paged_attn_args& x, int batch) {
  return ((int64_t)x.n_tokens * (x.n_heads_q / x.n_heads_kv) - 1) / kRowsBM + batch;
}
// Row tiles that go to one XCD together: of one request (or prefix), 16 at most and about equal.  us, single tiles and groups:
// two prompts of 2048 behind 14336 keys 330 and 265, 16 of 100 behind 900 54 and 43, one of 8192 from its start 520 and 502.
static int row_group(const dcp_paged_attn_args& x, int batch) {
  const int each = std::max((int)(row_tiles(x, batch) / batch), 1), n = (each + 15) / 16;
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
static RowShares row_shares(const dcp_paged_attn_args& x, int batch, int64_t max_keys, bool joined_anyway) {
  // (about as many tiles as have rows: row_tiles has room for more)
  const int64_t rows = (int64_t)x.n_tokens * (x.n_heads_q / x.n_heads_kv);
  const int64_t row_tiles_there = std::max<int64_t>((rows + kRowsBM - 1) / kRowsBM, batch), group = row_group(x, batch);
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
static PagedPlan plan_paged(const dcp_paged_attn_args& x) {
  PagedPlan plan;
  const auto up16 = [](size_t n) { return (n + 15) / 16 * 16; };
  const int group = x.n_heads_q / x.n_heads_kv;
  const int64_t keys = seen_keys(x);
  // The kernel of few rows: of requests with up to 32.  Its sums of tiles have to fit 32 bits whatever the lengths are.
  const int64_t own_rows = (int64_t)x.max_seqlen_q * group, all_rows = (int64_t)x.n_tokens * group;
  plan.rows = own_rows <= 16 ? 16 : 32;
  // (as many units as there can be, and about as many as there are)
  const int64_t most_units = (all_rows + (int64_t)x.batch * (plan.rows - 1)) / plan.rows * x.n_heads_kv;
  const int64_t units = std::max<int64_t>(x.batch, all_rows / plan.rows) * x.n_heads_kv;
  plan.few = own_rows <= 32 && x.batch <= kFewMaxBatch && (double)most_units * ((double)x.table_width * x.page_size / kFewBN + 2) < 2e9;
  const RowShares prefix_shares = x.n_prefixes > 0 ? row_shares(x, x.n_prefixes, x.max_prefix_len, true) : RowShares{0, 0};
  double few_us = 0;
  if (plan.few) {
    // Whole units where they are short: the chain of one's tiles (of a fourth of them) against what cutting costs, a second kernel and
    // more, and, as far as that goes, against the equal shares' time (of lengths that are half the longest on average, at 5.4 TB/s).
    // us, whole and cut, 8 kv heads of 128: 1 request of 100 keys 6.8 and 9.5, of 512 9.5 and 10.9, of 1024 15 and 11; 16 of 300 11 and 13, of
    // 1024 20 and 21, of up to 1024 18 and 15; 32 of 512 16 and 21, of 1400 34 and 42, of up to 1400 25 and 27, of 2048 48 and 52, of up
    // to 2048 33 and 30; 64 of up to 200 11 and 16, of up to 1400 37 and 40.  Beside a prefix's shares, which are joined anyway, also
    // where these take as long: 64 requests of up to 1024 own keys on a prefix of 32768 80 and 87, but 4 of up to 2000 on one of 2000 33 and 18.
    const double unit_us = keys * (0.004 + 0.007 * x.head_dim / 128);
    few_us = 0.5 * units * keys * x.head_dim * 4 / 5.4e6;
    plan.whole = unit_us < std::max(5.5 + std::min(0.6 * few_us, 10.5), keys <= 2048 ? prefix_shares.us - 6 : 0.0);
    const int slots = 2 * device_cu_count();
    // Of eight waves where a CU has at most one and could hold two (head size 64): 32 windows of 1016 keys 14.1, of four 14.6; 16 of
    // 2048 20.6 and 22.2, of 256 7.4 and 7.0.
    plan.waves = plan.whole && x.head_dim == 64 && x.n_prefixes == 0 && units <= device_cu_count() && keys > 512 ? 8 : 4;
    // Heads at once, a wave or two for each: of whole units while there are more than the CUs hold and a wave's chain stays short,
    // which its start and end outlast (us, one, two and four heads: 128 requests of 16 keys 15, 9.6 and 9.9, of 256 31.5, 27.9 and 28.0; 512 of
    // 64 64, 44 and 35, of up to 512 105, 82 and 87; 64 of 64 8.2, 8.7 and 10.8); of equal shares four from 64 tiles a workgroup on.
    const int64_t tiles = (int64_t)x.batch * ((keys + kFewBN - 1) / kFewBN) * x.n_heads_kv / slots;
    while (plan.heads < 4 && x.n_heads_kv % (2 * plan.heads) == 0 &&
           (plan.whole ? units / plan.heads > slots && 2 * plan.heads * keys <= 1280 : tiles >= 64))
      plan.heads *= 2;
    plan.n_few = plan.whole ? (int)(most_units / plan.heads) : slots;
    if (!plan.whole) {
      plan.cuts = up16((size_t)x.n_tokens * x.n_heads_q * sizeof(int2));
      plan.slots = (size_t)plan.n_few * 2 * plan.heads * plan.rows * (x.head_dim + 2) * sizeof(float);
    }
  } else {
    plan.n_own = row_shares(x, x.batch, keys, x.n_prefixes > 0).n;
  }
  if (x.n_prefixes > 0) {
    plan.n_prefix = prefix_shares.n;
    // All of the few first where theirs is most of the time: the prefix's then fill what they leave at their end.  us, all first and one
    // a CU first: 64 requests of up to 1024 own keys on a prefix of 32768 84 and 75, of 64 own keys 77 and 66; 256 of up to 600 on 8192
    // 114 and 97; 128 of up to 2000 on 8192 110 and 115; 64 of up to 6000 on 16384 122 and 125.
    plan.few_first = few_us < 1.5 * prefix_shares.us ? std::min(plan.n_few, device_cu_count()) : plan.n_few;
  }
  if (plan.n_own + plan.n_prefix > 1) plan.shares = (size_t)(plan.n_own + plan.n_prefix) * x.n_tokens * x.n_heads_q * (x.head_dim + 2) * sizeof(float);
  return plan;
}

// One of the kernels of a storage type and a head size.
#define DCP_PAGED_KERNEL(kernel, ...)                                                                   \
  (x.dtype == DCP_DTYPE_BF16 ? (x.head_dim == 128 ? kernel<DCP_DTYPE_BF16, 128, ##__VA_ARGS__>          \
                                                  : kernel<DCP_DTYPE_BF16, 64, ##__VA_ARGS__>)          \
                             : (x.head_dim == 128 ? kernel<DCP_DTYPE_FP16, 128, ##__VA_ARGS__>          \
                                                  : kernel<DCP_DTYPE_FP16, 64, ##__VA_ARGS__>))

namespace {

// What a caller may have wrong, before anything is launched.
int check_paged(const dcp_paged_attn_args& x) {
  if (x.dtype != DCP_DTYPE_BF16 && x.dtype != DCP_DTYPE_FP16) return fail(DCP_ERR_UNSUPPORTED, "paged_attn: dtype %d unsupported (bf16 and fp16 only)", x.dtype);
  if (x.head_dim != 64 && x.head_dim != 128) return fail(DCP_ERR_UNSUPPORTED, "paged_attn: head_dim %d unsupported (64 or 128)", x.head_dim);
  DCP_REQUIRE(x.n_tokens >= 0 && x.batch >= 0 && x.n_pages >= 0 && x.n_prefixes >= 0, "paged_attn: negative size");
  DCP_REQUIRE(x.n_heads_q > 0 && x.n_heads_kv > 0 && x.n_heads_q % x.n_heads_kv == 0, "paged_attn: n_heads_q %d must be a multiple of n_heads_kv %d",
              x.n_heads_q, x.n_heads_kv);
  DCP_REQUIRE(x.softmax_scale > 0.0f, "paged_attn: softmax_scale must be positive");
  DCP_REQUIRE(x.window >= 0 && x.n_starting >= 0, "paged_attn: negative window or number of first tokens");
  DCP_REQUIRE(x.n_prefixes == 0 || x.window == 0, "paged_attn: no window where there are shared prefixes");
  DCP_REQUIRE(x.page_size > 0 && x.page_size % 16 == 0, "paged_attn: page_size %d must be a positive multiple of 16", x.page_size);
  DCP_REQUIRE(x.table_width > 0 && x.table_stride >= 0 && (x.n_prefixes == 0 || (x.prefix_width > 0 && x.prefix_stride >= 0)),
              "paged_attn: empty block tables");
  DCP_REQUIRE(std::max((int64_t)x.table_width, (int64_t)(x.n_prefixes ? x.prefix_width : 0)) * x.page_size < kNoKey - 64, "paged_attn: too many keys a request");
  DCP_REQUIRE(x.page_stride % 8 == 0 && x.token_stride % 8 == 0 && x.head_stride % 8 == 0 && x.q_token_stride % 8 == 0 && x.q_head_stride % 8 == 0 &&
                  x.out_token_stride % 4 == 0 && x.out_head_stride % 4 == 0, "paged_attn: q, k, v strides must be multiples of 8 elements (out: 4)");
  DCP_REQUIRE(x.page_stride >= 0 && x.token_stride >= 0 && x.head_stride >= 0 && x.q_token_stride >= 0 && x.q_head_stride >= 0 &&
                  x.out_token_stride > 0 && x.out_head_stride > 0, "paged_attn: negative stride");
  DCP_REQUIRE(((reinterpret_cast<uintptr_t>(x.q) | reinterpret_cast<uintptr_t>(x.k_cache) | reinterpret_cast<uintptr_t>(x.v_cache) |
                reinterpret_cast<uintptr_t>(x.out)) & 15) == 0, "paged_attn: q, k, v and out must be 16-byte aligned");
  DCP_REQUIRE((int64_t)x.n_tokens * x.n_heads_q < ((int64_t)1 << 31) - 256, "paged_attn: too many queries");
  DCP_REQUIRE(x.cu_seqlens_q != nullptr || x.n_tokens == x.batch, "paged_attn: without cu_seqlens_q every request has one token, got %d for %d",
              x.n_tokens, x.batch);
  if (x.n_tokens == 0 || x.batch == 0) return DCP_OK;
  DCP_REQUIRE(x.q && x.out && x.lse && x.block_table && x.seq_lens && (x.n_pages == 0 || (x.k_cache && x.v_cache)) &&
                  (x.n_prefixes == 0 || (x.prefix_table && x.prefix_lens && x.cu_groups)), "paged_attn: null argument");
  DCP_REQUIRE(x.max_seqlen_q > 0 && x.max_seqlen_k > 0 && (x.n_prefixes == 0 || x.max_prefix_len > 0), "paged_attn: the longest lengths must be positive");
  // (every kernel's work items: at most 64 shares of a row tile)
  DCP_REQUIRE((row_tiles(x, x.batch) + row_tiles(x, x.n_prefixes)) * x.n_heads_kv < ((int64_t)1 << 31) - (1 << 20), "paged_attn: too many rows");
  return DCP_OK;
}

int paged_attn(const dcp_paged_attn_args& x, void* workspace, size_t workspace_bytes, void* stream) {
  DCP_RECORDED(paged_attn(x, workspace, workspace_bytes, stream));
  if (const int status = check_paged(x)) return status;
  if (x.n_tokens == 0 || x.batch == 0) return DCP_OK;
  const PagedPlan plan = plan_paged(x);
  const size_t needed = plan.bytes();
  DCP_REQUIRE(needed == 0 || (workspace && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0 && workspace_bytes >= needed),
              "paged_attn: workspace of %zu bytes is missing, not 16-byte aligned or smaller than the %zu needed", workspace_bytes, needed);
  PagedParams p = {};
  p.q = x.q; p.k = x.k_cache; p.v = x.v_cache; p.out = x.out; p.lse = x.lse;
  p.cu_seqlens_q = x.cu_seqlens_q;
  p.q_token = x.q_token_stride; p.q_head = x.q_head_stride; p.out_token = x.out_token_stride; p.out_head = x.out_head_stride;
  p.page_stride = x.page_stride; p.token_stride = x.token_stride; p.head_stride = x.head_stride;
  p.own = {x.block_table, x.seq_lens, nullptr, x.table_stride, x.table_width, x.batch, 0, plan.n_own, (int)row_tiles(x, x.batch), 1, plan.few && !plan.whole};
  if (x.n_prefixes > 0)
    p.prefix = {x.prefix_table, x.prefix_lens, x.cu_groups, x.prefix_stride, x.prefix_width, x.n_prefixes, plan.n_own, plan.n_prefix,
                (int)row_tiles(x, x.n_prefixes), 1, 0};
  p.n_pages = x.n_pages; p.page_size = x.page_size;
  p.n_requests = x.batch; p.n_tokens = x.n_tokens;
  p.n_heads_q = x.n_heads_q; p.n_heads_kv = x.n_heads_kv; p.group = x.n_heads_q / x.n_heads_kv;
  p.window = x.window; p.n_starting = x.n_starting;
  p.scale_log2 = x.softmax_scale * kLog2e;
  p.direct = plan.n_own + plan.n_prefix == 1;
  char* at = reinterpret_cast<char*>(workspace);
  p.cuts = reinterpret_cast<int2*>(at);
  p.slot_out = reinterpret_cast<float*>(at + plan.cuts);
  p.slot_sums = reinterpret_cast<f32x2*>(p.slot_out + (size_t)plan.n_few * 2 * plan.heads * plan.rows * x.head_dim);
  p.partial_out = reinterpret_cast<float*>(at + plan.cuts + plan.slots);
  p.partial_sums = reinterpret_cast<f32x2*>(p.partial_out + (size_t)(plan.n_own + plan.n_prefix) * x.n_tokens * x.n_heads_q * x.head_dim);
  p.few_rows = plan.rows; p.few_heads_log2 = plan.heads / 2; p.few_whole = plan.whole; p.merge_sets = 1; p.n_few = plan.n_few; p.few_first = plan.few_first;

  int status = DCP_OK;
  const auto launch = [&](auto kernel, const char* name, int64_t n_wg, int threads) {
    if (status != DCP_OK || n_wg == 0) return;
    if (n_wg >= (int64_t)1 << 31) {
      status = fail(DCP_ERR_ARG, "paged_attn: too many work items");
      return;
    }
    KernelTimer timer(name, stream);
    hipLaunchKernelGGL(kernel, dim3((unsigned)n_wg), dim3(threads), 0, (hipStream_t)stream, p);
    status = check_launch(name);
  };
  // A kernel of rows' workgroups
  const auto row_items = [&](PagedSource& src) {
    src.xcd_group = row_group(x, src.batch);
    return row_workgroups(src.n_tiles, src.xcd_group, x.n_heads_kv, src.n_shares);
  };
  if (plan.few && x.n_prefixes > 0) {
    const int64_t n_wg = row_items(p.prefix) + p.n_few;
    if (plan.rows == 16) launch(DCP_PAGED_KERNEL(paged_both_kernel, 1), "paged_both_kernel", n_wg, 256);
    else launch(DCP_PAGED_KERNEL(paged_both_kernel, 2), "paged_both_kernel", n_wg, 256);
  } else if (plan.few && plan.waves == 8) {
    launch(x.dtype == DCP_DTYPE_BF16 ? (plan.rows == 16 ? paged_few_kernel<DCP_DTYPE_BF16, 64, 1, 8> : paged_few_kernel<DCP_DTYPE_BF16, 64, 2, 8>)
                                     : (plan.rows == 16 ? paged_few_kernel<DCP_DTYPE_FP16, 64, 1, 8> : paged_few_kernel<DCP_DTYPE_FP16, 64, 2, 8>),
           "paged_few_kernel", p.n_few, 512);
  } else if (plan.few) {
    if (plan.rows == 16) launch(DCP_PAGED_KERNEL(paged_few_kernel, 1, 4), "paged_few_kernel", p.n_few, 256);
    else launch(DCP_PAGED_KERNEL(paged_few_kernel, 2, 4), "paged_few_kernel", p.n_few, 256);
  } else {
    launch(DCP_PAGED_KERNEL(paged_rows_kernel, false), "paged_rows_kernel", row_items(p.own), kRowsThreads);
    if (x.n_prefixes > 0) {
      std::swap(p.own, p.prefix);  // (the kernel takes what it finds there)
      launch(DCP_PAGED_KERNEL(paged_rows_kernel, true), "paged_rows_kernel", row_items(p.own), kRowsThreads);
      std::swap(p.own, p.prefix);
    }
  }
  if (p.own.by_few || !p.direct) {
    // eight parts a set of lanes, as far as the longest lengths tell how many there are
    const int64_t units = std::max<int64_t>((int64_t)x.batch * x.n_heads_kv / plan.heads, 1);
    const int64_t parts = (plan.few && !plan.whole ? plan.n_few / units + 2 : plan.n_own) + plan.n_prefix;
    const int sets = kPagedMergeThreads / (x.head_dim / 4);
    while (p.merge_sets < sets && parts > 8 * p.merge_sets) p.merge_sets *= 2;
    launch(DCP_PAGED_KERNEL(paged_merge_kernel), "paged_merge_kernel", ((int64_t)x.n_tokens * x.n_heads_q * p.merge_sets + sets - 1) / sets, kPagedMergeThreads);
  }
  return status;
}

}  // namespace
}  // namespace dcp

using namespace dcp;

extern "C" size_t dcp_paged_attn_workspace_bytes(const dcp_paged_attn_args* args) {
  if (args == nullptr || check_paged(*args) != DCP_OK || args->n_tokens == 0 || args->batch == 0) return 0;
  return plan_paged(*args).bytes();
}

extern "C" int dcp_paged_attn(const dcp_paged_attn_args* args, void* workspace, size_t workspace_bytes, void* stream) {
  DCP_REQUIRE(args != nullptr, "paged_attn: null argument");
  return paged_attn(*args, workspace, workspace_bytes, stream);
}
