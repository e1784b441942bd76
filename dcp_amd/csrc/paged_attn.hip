// Attention over a paged K/V cache for gfx950: causal or with a sliding window and first tokens that stay visible, for any
// number of new tokens a request, and for batches that share a long prefix.
//
//   out = softmax(scale q K^T) V over the visible keys, lse = log sum exp
//
// A query's row is one (token, q head).  The rows of a kv head's group and of neighbouring tokens read the same keys, so they are
// taken together: row r of a request stands for token r / group and head r % group of the kv head.
//
// The kernel of rows (paged_rows_kernel): a workgroup of 4 waves owns 128 rows of one (request, kv head), a wave 32 of them,
// and walks its share of the key tiles (64 keys) that any of them sees.  K and V tiles go from memory straight into LDS
// (KvTile), two stages; both products are transposed, as in the forward kernel of the plans:
//
//   S^T[key, row] = K Q^T      A = K rows from LDS, B = Q in registers
//   O^T[d,   row] = V^T P^T    A = V columns from LDS, B = P^T straight from the S^T accumulators
//
// Keys are taken in groups of 16 that lie in one page (page sizes are multiples of 16), so a lane looks up one page a tile:
// the lanes' 16-key group is the same for all of a wave's loads of a tile.  The window and the first tokens are two runs of such
// groups laid end to end; nothing in between is read.
#include <math.h>

#include <algorithm>

#include "attn_common.h"
#include "record.h"

namespace dcp {

struct PagedAttnParams {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  float* lse;
  const int32_t* block_table;  // of the requests, or of the shared prefixes
  const int32_t* key_lens;
  const int32_t* cu_seqlens_q;  // null: one token a request
  const int32_t* cu_groups;     // prefixes: the requests of a prefix; null otherwise
  int64_t table_stride;
  int64_t q_token, q_head, out_token, out_head;  // element strides
  int64_t page_stride, token_stride, head_stride;
  int table_width, n_pages, page_size;
  int batch;     // requests, or prefixes
  int n_tokens;  // of q
  int n_requests;
  int n_heads_q, n_heads_kv, group;
  int window, n_starting;  // window 0: none
  float scale_log2;
  int n_tiles, n_splits;  // row tiles of a kv head; shares of a tile's keys
  // shares, unless a tile has one and nothing is to be merged: [share][token][q head], O relative to the maximum
  float* partial_out;
  f32x2* partial_sums;  // the maximum (log2 domain) and the sum of the weights
  int first_share, direct;
};

constexpr int kRowsThreads = 256, kRowsBM = 128, kRowsBN = 64;
constexpr int kMinTilesPerShare = 4;

// The tokens of request (or prefix) b.  Cut to the tensor, whatever the tables say.
struct TokenRange {
  int begin, n;
};
__device__ __forceinline__ int first_token(const PagedAttnParams& p, int b) {
  int r = b;
  if (p.cu_groups != nullptr) r = min(max(p.cu_groups[b], 0), p.n_requests);
  if (p.cu_seqlens_q != nullptr) r = p.cu_seqlens_q[r];
  return min(max(r, 0), p.n_tokens);
}
__device__ __forceinline__ TokenRange tokens_of(const PagedAttnParams& p, int b) {
  const int begin = first_token(p, b);
  return {begin, max(first_token(p, b + 1) - begin, 0)};
}

// Row tile `tile` belongs to request b and is its tile number `index`.  Request b's tiles begin at number
// floor(first_row / 128) + b: that leaves room for its last, partial one, and needs no sum over the requests before it.
struct RowTile {
  int b, index;
};
__device__ __forceinline__ RowTile find_row_tile(const PagedAttnParams& p, int tile) {
  const int lane = threadIdx.x & 63;
  auto start = [&](int b) { return (int)((int64_t)first_token(p, b) * p.group / kRowsBM) + b; };
  int lo = 0, hi = p.batch;  // the last request that begins at or before the tile; 64 candidates a step
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64, b = lo + lane * step;
    const bool before = b < hi && start(b) <= tile;
    const int n = __popcll(__ballot(before));
    if (n > 1) lo += (n - 1) * step;
    hi = min(lo + step, hi);
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  return {lo, tile - __builtin_amdgcn_readfirstlane(start(lo))};
}

// The 16-key groups that rows at positions [first, last] see: [0, n_first) and then [begin, end).
struct KeyGroups {
  int n_first, begin, end;
  int window_begin, hull_end;  // keys from hull_end on, and between the first ones and the window, are seen by none
  __device__ __forceinline__ KeyGroups(const PagedAttnParams& p, int first, int last) {
    hull_end = last + 1;
    end = (hull_end + 15) / 16;
    window_begin = p.window > 0 ? max(first - p.window + 1, 0) : 0;
    begin = window_begin / 16;
    n_first = min((int)(((int64_t)p.n_starting + 15) / 16), end);
    if (n_first >= begin) begin = n_first = 0;  // one run
  }
  __device__ __forceinline__ int count() const { return n_first + end - begin; }
  __device__ __forceinline__ int at(int i) const { return i < n_first ? i : i - n_first + begin; }
  __device__ __forceinline__ bool sees(const PagedAttnParams& p, int key) const {
    return key < hull_end && (key < p.n_starting || key >= window_begin);
  }
};

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

// 16 bytes a lane from memory into LDS at lds_at + 16 * lane (ordered by the caller, as KvTile's loads)
__device__ __forceinline__ void load_async_piece(uint32_t lds_at, const uint16_t* from) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :
               : "s"(__builtin_amdgcn_readfirstlane(lds_at)), "v"(from)
               : "memory");
}

// The same for what is read once (it takes no room in the caches).
__device__ __forceinline__ void load_async_piece_nt(uint32_t lds_at, const uint16_t* from) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off nt"
               :
               : "s"(__builtin_amdgcn_readfirstlane(lds_at)), "v"(from)
               : "memory");
}

template <int DTYPE, int D>
__global__ __launch_bounds__(kRowsThreads, 2) void paged_rows_kernel(const PagedAttnParams p) {
  typedef KvTile<D> Tile;
  constexpr int KS = D / 32, DT = D / 16, RT = 2, BN = kRowsBN;
  __shared__ __attribute__((aligned(16))) uint16_t k_lds[2][Tile::SIZE];
  __shared__ __attribute__((aligned(16))) uint16_t v_lds[2][Tile::SIZE];
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);

  // ---- which rows, which share of their keys ---------------------------------
  int item = __builtin_amdgcn_readfirstlane(blockIdx.x);
  const int tile_number = item % p.n_tiles;
  item /= p.n_tiles;
  const int kv_head = __builtin_amdgcn_readfirstlane(item % p.n_heads_kv), share = __builtin_amdgcn_readfirstlane(item / p.n_heads_kv);
  const RowTile tile = find_row_tile(p, tile_number);
  const TokenRange tokens = tokens_of(p, tile.b);
  const int n_rows = tokens.n * p.group;  // (at most n_tokens * group, which the host has checked)
  const int row0 = tile.index * kRowsBM;
  if (row0 >= n_rows) return;
  const bool prefix = p.cu_groups != nullptr;
  const int n_keys = (int)min((int64_t)max(p.key_lens[tile.b], 0), p.n_pages > 0 ? (int64_t)p.table_width * p.page_size : 0);
  // token i of the request is at position n_keys - n + i; every token is past all of a prefix
  const int first_tok = row0 / p.group, last_tok = min(row0 + kRowsBM, n_rows) - 1;
  const int at0 = prefix ? n_keys - 1 : n_keys - tokens.n;
  const int step = prefix ? 0 : 1;
  const KeyGroups groups(p, max(at0 + first_tok * step, 0), at0 + last_tok / p.group * step);
  const int n_groups = groups.hull_end > 0 ? groups.count() : 0;
  const int tiles_all = (n_groups + 3) / 4;
  const int n_shares = min(p.n_splits, max(1, tiles_all / kMinTilesPerShare));
  int t_begin = 0, t_end = 0;
  if (share < n_shares) {
    t_begin = __builtin_amdgcn_readfirstlane((int)((int64_t)tiles_all * share / n_shares));
    t_end = __builtin_amdgcn_readfirstlane((int)((int64_t)tiles_all * (share + 1) / n_shares));
  }

  // ---- this lane's rows: n of each of the wave's two row tiles ------------------
  int64_t q_at[RT], out_row[RT];
  int last_key[RT], first_key[RT];  // the last key it sees; the first of its window
  bool live[RT];
  int w_last = 0x7fffffff, w_first = 0;  // what every row of the wave sees: keys up to w_last, from w_first on
  int w_hull = -1;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = row0 + w * 32 + rt * 16 + n;
    live[rt] = r < n_rows;
    const int tok = r / p.group, head = kv_head * p.group + r % p.group;
    q_at[rt] = (int64_t)(tokens.begin + tok) * p.q_token + head * p.q_head;
    out_row[rt] = (int64_t)(tokens.begin + tok) * p.n_heads_q + head;
    last_key[rt] = live[rt] ? at0 + tok * step : 0x7fffffff;  // (a row that is not there sees anything, with a zero q)
    first_key[rt] = live[rt] && p.window > 0 ? max(last_key[rt] - p.window + 1, 0) : 0;
    w_last = min(w_last, wave_min(last_key[rt]));
    w_first = max(w_first, wave_max(first_key[rt]));
    w_hull = max(w_hull, wave_max(live[rt] ? last_key[rt] : -1));
  }
  u32x4 q[RT][KS];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      q[rt][ks] = u32x4{0, 0, 0, 0};
      if (live[rt]) q[rt][ks] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(p.q) + q_at[rt] + Tile::element16(g) + Tile::step16(ks));
    }

  // ---- running state ---------------------------------------------------------------
  f32x4 o[RT][DT];
  float m_run[RT], l_run[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    m_run[rt] = -INFINITY;
    l_run[rt] = 0.0f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[rt][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  // ---- tiles: lane l brings pieces of rows of the tile's 16-key group l / 16 ---------
  const int32_t* table = p.block_table + (int64_t)tile.b * p.table_stride;
  const uint16_t* k_base = reinterpret_cast<const uint16_t*>(p.k) + kv_head * p.head_stride;
  const uint16_t* v_base = reinterpret_cast<const uint16_t*>(p.v) + kv_head * p.head_stride;
  constexpr int CH = D / 8;
  const int piece = lane % CH;
  auto row_in_group = [&](int i) { return Tile::row_of(w * Tile::LPW + Tile::group_of_load(i), lane / CH) & 15; };
  // the first key of the lane's group of tile t, -1 behind the last group
  auto group_key = [&](int t) { return t * 4 + g < n_groups ? groups.at(t * 4 + g) * 16 : -1; };
  auto look_up = [&](int t) { return t < t_end && group_key(t) >= 0 ? table[group_key(t) / p.page_size] : -1; };
  auto request = [&](int t, int page, int stage) {
    const int key = group_key(t);
    const bool there = key >= 0 && (unsigned)page < (unsigned)p.n_pages;
    const int64_t off = there ? page * p.page_stride + key % p.page_size * p.token_stride : 0;
#pragma unroll
    for (int i = 0; i < Tile::LPW; ++i) {
      const int64_t at = off + row_in_group(i) * p.token_stride + piece * 8;
      load_async_piece(Tile::group_lds_at(lds_address(k_lds[stage]), w, i), k_base + at);
      load_async_piece(Tile::group_lds_at(lds_address(v_lds[stage]), w, i), v_base + at);
    }
    return there;
  };
  const int k_rd = Tile::row_base16(n, g), v_rd = Tile::col_base16(lane);

  int page_next = look_up(t_begin + 1);
  bool there = false, there_next = false;
  if (t_begin < t_end) there_next = request(t_begin, look_up(t_begin), 0);
  for (int t = t_begin; t < t_end; ++t) {
    const int stage = (t - t_begin) & 1;
    there = there_next;
    wait_loads();
    // What no row sees (behind the last key, between the first tokens and the window, in a page that is not one) may
    // hold anything, and a weight of zero does not make a NaN vanish: its V is cleared by the lanes that brought it.
    const int key0 = group_key(t);
    const bool whole = there && key0 + 15 < groups.hull_end && (key0 + 15 < p.n_starting || key0 >= groups.window_begin);
    if (__any(!whole)) {
#pragma unroll
      for (int i = 0; i < Tile::LPW; ++i) {
        if (!(there && groups.sees(p, key0 + row_in_group(i))))
          *reinterpret_cast<u32x4*>(reinterpret_cast<char*>(v_lds[stage]) + (Tile::group_lds_at(0, w, i) + 16 * lane)) = u32x4{0, 0, 0, 0};
      }
    }
    __syncthreads();  // the tile is there, and nobody reads the other stage any more
    if (t + 1 < t_end) there_next = request(t + 1, page_next, stage ^ 1);
    page_next = look_up(t + 2);

    // the tile's four groups: their first keys, and whether they are there
    int group_keys[4];
    const uint64_t there_mask = __ballot(there);
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
      group_keys[kt] = __builtin_amdgcn_readlane(key0, 16 * kt);
      if (!(there_mask >> (16 * kt) & 1)) group_keys[kt] = 0x7fffff00;  // (past every row's last key)
    }
    bool full = true, seen = false;
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
      const int key = group_keys[kt];
      full = full && key + 15 <= w_last && (key >= w_first || key + 15 < p.n_starting);
      seen = seen || key <= w_hull;
    }
    if (!seen) continue;

    f32x4 s[RT][4];
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) s[rt][kt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const u32x4 a = Tile::read_row16(k_lds[stage], k_rd, kt, ks);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) s[rt][kt] = mfma_16x16x32<DTYPE>(a, q[rt][ks], s[rt][kt]);
      }
    }
    if (!full) {
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = group_keys[kt] + 4 * g + e;
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            const bool visible = key <= last_key[rt] && (key < p.n_starting || key >= first_key[rt]) && group_keys[kt] < 0x7fffff00;
            s[rt][kt][e] = visible ? s[rt][kt][e] : -INFINITY;
          }
        }
    }
    u32x4 pb[RT][2];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float mx = -INFINITY;
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int e = 0; e < 4; ++e) mx = fmaxf(mx, s[rt][kt][e]);
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
      float sum = 0.0f;
#pragma unroll
      for (int kt = 0; kt < 4; ++kt) {
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = fast_exp2(fmaf(s[rt][kt][e], p.scale_log2, -m_use));
          sum += x[e];
        }
        // weights are rounded to the storage type for the product (half a step each); their sum is of the unrounded ones
        pb[rt][kt / 2][2 * (kt % 2)] = pack2<DTYPE>(x[0], x[1]);
        pb[rt][kt / 2][2 * (kt % 2) + 1] = pack2<DTYPE>(x[2], x[3]);
      }
      l_run[rt] += sum;
    }
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const u32x4 a = Tile::read_col16(v_lds[stage], v_rd, s2, dt);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) o[rt][dt] = mfma_16x16x32<DTYPE>(a, pb[rt][s2], o[rt][dt]);
      }
  }

  // ---- results ---------------------------------------------------------------------
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const float l = rows_sum(l_run[rt]);
    if (!live[rt]) continue;
    if (!p.direct) {
      const int64_t at = (int64_t)(p.first_share + share) * p.n_tokens * p.n_heads_q + out_row[rt];
      if (g == 0) p.partial_sums[at] = f32x2{m_run[rt], l};
      if (share >= n_shares) continue;  // (nothing is read of a share without weights)
      float* to = p.partial_out + at * D + 4 * g;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4*>(to + 16 * dt) = o[rt][dt];
      continue;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const int64_t token = out_row[rt] / p.n_heads_q, head = out_row[rt] % p.n_heads_q;
    uint16_t* to = reinterpret_cast<uint16_t*>(p.out) + token * p.out_token + head * p.out_head + 4 * g;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      *reinterpret_cast<u32x2*>(to + 16 * dt) = u32x2{pack2<DTYPE>(o[rt][dt][0] * inv, o[rt][dt][1] * inv),
                                                      pack2<DTYPE>(o[rt][dt][2] * inv, o[rt][dt][3] * inv)};
    if (g == 0) p.lse[head * p.n_tokens + token] = l == 0.0f ? INFINITY : (m_run[rt] + log2f(l)) * kLn2;
  }
}

// ---------------------------------------------------------------------------
// The kernel of few rows: answering token by token.  A request has few rows a kv head (tokens * group, at most 32), so the
// keys' bytes bound it and what counts is how many of them are under way.  The waves of a workgroup share no tile:
// each takes tiles of 32 keys of its own, every fourth, K straight into registers in the layout of the product, V into its own
// part of LDS, both a tile ahead, and waits for nobody until its share of the keys is done.
//
// Work is cut by length, not by request: the tiles of all (request, rows, kv head) units are laid end to end and every
// workgroup takes the same number of them, whatever the lengths are (they are known on the device only).  A unit inside one
// workgroup's share is finished there; of one that is cut each piece goes to the workgroup's slot (0: the share begins in the
// unit, 1: it ends in it) and the merge kernel joins them.
// ---------------------------------------------------------------------------
struct PagedFewParams {
  PagedAttnParams a;
  int2* cuts;        // [token][q head]: see cut_of
  float* slot_out;   // [workgroup][2][head of the workgroup][rows][D]
  f32x2* slot_sums;  // [workgroup][2][head of the workgroup][rows]
  int heads;         // kv heads a workgroup takes at once: 1, 2 or 4, as many to each of which it has 4 / heads waves
};
// What the merge needs to know of a row: the workgroup that begins its unit, how many the unit is cut over, the slot of the first
// piece (the others are in slot 0) and the row in the slots.
__device__ __forceinline__ int2 cut_of(int wg, int n_pieces, int slot, int row) { return int2{wg, n_pieces | row << 20 | slot << 28}; }
constexpr int kFewThreads = 256, kFewWaves = 4, kFewBN = 32;
constexpr int kFewMaxBatch = 1 << 16;

// What request b is to the kernel.
struct FewRequest {
  int first_tok, n_tok, n_keys, n_chunks, n_tiles;
  template <typename P>
  __device__ __forceinline__ FewRequest(const P& p, int b, int rows) {
    const TokenRange tokens = tokens_of(p, b);
    first_tok = tokens.begin;
    n_tok = tokens.n;
    n_keys = (int)min((int64_t)max(p.key_lens[b], 0), p.n_pages > 0 ? (int64_t)p.table_width * p.page_size : 0);
    n_chunks = (n_tok * p.group + rows - 1) / rows;
    const KeyGroups groups(p, max(n_keys - n_tok, 0), n_keys - 1);
    n_tiles = max((groups.count() + 1) / 2, 1);  // (a request without keys has its rows written all the same)
  }
  __device__ __forceinline__ int64_t work(int head_groups) const { return (int64_t)n_chunks * head_groups * n_tiles; }
};

// Sum over the wave's lanes up to and with this one.
__device__ __forceinline__ int64_t wave_scan(int64_t x) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int off = 1; off < 64; off *= 2) {
    const int64_t y = __shfl_up(x, off);
    if (lane >= off) x += y;
  }
  return x;
}
__device__ __forceinline__ int64_t lane_value(int64_t x, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane((int)x, lane), hi = __builtin_amdgcn_readlane((int)(x >> 32), lane);
  return (int64_t)(((uint64_t)hi << 32) | lo);
}

template <int DTYPE, int D, int RT>
__global__ __launch_bounds__(kFewThreads, 2) void paged_few_kernel(const PagedFewParams params) {
  const PagedAttnParams& p = params.a;
  constexpr int KS = D / 32, DT = D / 16, ROWS = 16 * RT;
  // V of 32 keys: load r of a tile brings rows r, r + LOADS, ... side by side (1 KiB), 32 bytes of padding between loads: eight
  // consecutive rows then lie in eight different 32-byte bank windows for the transposing reads.
  constexpr int LOADS = kFewBN * D * 2 / 1024, LOAD_BYTES = 1024 + 32, STAGE = LOADS * LOAD_BYTES;
  constexpr int O_STRIDE = D + 4;  // floats: rows of the joined result, a wave's
  constexpr int WAVE_BYTES = 2 * STAGE > ROWS * O_STRIDE * 4 ? 2 * STAGE : ROWS * O_STRIDE * 4;
  __shared__ __attribute__((aligned(16))) char lds[kFewWaves][WAVE_BYTES];
  __shared__ float sums_lds[kFewWaves][ROWS][2];
  __shared__ int64_t chunk_lds[kFewMaxBatch / 64];
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);

  const int heads = params.heads, head_groups = p.n_heads_kv / heads, turns = kFewWaves / heads;
  const int my_head = w % heads, my_turn = w / heads;  // of the workgroup's heads; of the waves that share its tiles

  // ---- this workgroup's share of all tiles -----------------------------------------
  auto work_of = [&](int b) -> int64_t { return b < p.batch ? FewRequest(p, b, ROWS).work(head_groups) : 0; };
  int64_t total, per, begin, end, before;  // before: tiles before the chunk of 64 requests in which the share begins
  int chunk = 0;
  const int n_chunks = (p.batch + 63) / 64;
  int64_t scan = wave_scan(work_of(lane));
  if (n_chunks == 1) {
    total = lane_value(scan, 63);
  } else {
    for (int i = w; i < n_chunks; i += kFewWaves) {
      const int64_t sum = wave_scan(work_of(i * 64 + lane));
      if (lane == 63) chunk_lds[i] = sum;
    }
    __syncthreads();
    total = 0;
    for (int i = 0; i < n_chunks; i += 64) total += lane_value(wave_scan(i + lane < n_chunks ? chunk_lds[i + lane] : 0), 63);
  }
  per = max((total + gridDim.x - 1) / gridDim.x, (int64_t)turns);
  begin = min((int64_t)blockIdx.x * per, total);
  end = min(begin + per, total);
  if (begin >= end) return;
  before = 0;
  if (n_chunks > 1) {
    for (int i = 0; i < n_chunks; i += 64) {
      const int64_t sums = before + wave_scan(i + lane < n_chunks ? chunk_lds[i + lane] : 0);
      const int passed = __popcll(__ballot(sums <= begin));
      if (passed > 0) before = lane_value(sums, passed - 1);
      chunk = i + passed;
      if (passed < 64) break;
    }
    chunk = __builtin_amdgcn_readfirstlane(min(chunk, n_chunks - 1));
    scan = wave_scan(work_of(chunk * 64 + lane));
  }
  const int passed = min(__popcll(__ballot(before + scan <= begin)), 63);
  int b = __builtin_amdgcn_readfirstlane(chunk * 64 + passed);
  int64_t b_start = before + (passed > 0 ? lane_value(scan, passed - 1) : 0);

  const uint32_t v_at = lds_address(lds[w]);
  int64_t at = begin;
  while (at < end) {
    const FewRequest request(p, b, ROWS);
    const int64_t work = request.work(head_groups);
    if (at >= b_start + work) {  // (no rows, or done)
      b_start += work;
      if (++b >= p.batch) break;
      continue;
    }
    const int unit = __builtin_amdgcn_readfirstlane((int)((at - b_start) / request.n_tiles));
    const int t_begin = __builtin_amdgcn_readfirstlane((int)(at - b_start - (int64_t)unit * request.n_tiles));
    const int t_end = __builtin_amdgcn_readfirstlane((int)min((int64_t)request.n_tiles, t_begin + (end - at)));
    const int slot = at == begin ? 0 : 1;
    const int n_cut = t_begin == 0 ? (int)((at + request.n_tiles - 1) / per) - (int)blockIdx.x + 1 : 0;
    at += t_end - t_begin;
    const int kv_head0 = unit % head_groups * heads, kv_head = kv_head0 + my_head, row0 = unit / head_groups * ROWS;
    const KeyGroups groups(p, max(request.n_keys - request.n_tok, 0), request.n_keys - 1);
    const int n_groups = request.n_keys > 0 ? groups.count() : 0;

    // ---- this lane's rows --------------------------------------------------------------
    int64_t out_row[RT];
    int last_key[RT], first_key[RT];
    bool live[RT];
    int w_last = 0x7fffffff, w_first = 0;
    u32x4 q[RT][KS];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int r = row0 + rt * 16 + n;
      live[rt] = r < request.n_tok * p.group;
      const int tok = r / p.group, head = kv_head * p.group + r % p.group;
      out_row[rt] = (int64_t)(request.first_tok + tok) * p.n_heads_q + head;
      last_key[rt] = live[rt] ? request.n_keys - request.n_tok + tok : 0x7fffffff;
      first_key[rt] = live[rt] && p.window > 0 ? max(last_key[rt] - p.window + 1, 0) : 0;
      const uint16_t* from = reinterpret_cast<const uint16_t*>(p.q) + (request.first_tok + tok) * p.q_token + head * p.q_head + 8 * g;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        q[rt][ks] = u32x4{0, 0, 0, 0};
        if (live[rt]) q[rt][ks] = *reinterpret_cast<const u32x4*>(from + 32 * ks);
      }
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

    // ---- where the wave's next 32 tiles are: lane 2 i + j holds the 16-key group j of the i-th of them ------------
    const int32_t* table = p.block_table + (int64_t)b * p.table_stride;
    const uint16_t* k_base = reinterpret_cast<const uint16_t*>(p.k) + kv_head * p.head_stride;
    const uint16_t* v_base = reinterpret_cast<const uint16_t*>(p.v) + kv_head * p.head_stride;
    constexpr int kNoKey = 0x7fffff00;  // of a group that is not there: past every row's last key
    int64_t lane_off = 0;
    int lane_key = kNoKey;
    auto look_up = [&](int step) {
      const int group = 2 * (t_begin + my_turn + turns * (step + (lane >> 1))) + (lane & 1);
      lane_off = 0;
      lane_key = kNoKey;
      if (group < n_groups && group < 2 * t_end) {
        const int key = groups.at(group) * 16, index = key / p.page_size;
        const int page = table[index];
        if ((unsigned)page < (unsigned)p.n_pages) {
          lane_key = key;
          lane_off = page * p.page_stride + (int64_t)(key - index * p.page_size) * p.token_stride;
        }
      }
    };
    // what a lane brings of a tile: K of key n of each group, 8 elements from 32 ks + 8 g; V rows of its half's group
    constexpr int CH = D / 8;
    const int64_t k_lane = n * p.token_stride + 8 * g;
    const int v_row = lane / CH % (16 / LOADS) * LOADS;  // of load 0, in the group of the lane's half
    const int64_t v_lane = v_row * p.token_stride + lane % CH * 8;
    const int n_steps = n_groups > 0 && t_begin + my_turn < t_end ? (t_end - t_begin - my_turn + turns - 1) / turns : 0;
    u32x4 k[2][KS];  // K of the tile at hand, and once its products are formed of the next one
    int64_t off[2];  // where its two groups are
    int next_key[2], tile_key[2];
    auto place = [&](int step) {
      if (step % 32 == 0) look_up(step);
      const int src = 2 * (step % 32);
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        off[kt] = lane_value(lane_off, src + kt);
        next_key[kt] = __builtin_amdgcn_readlane(lane_key, src + kt);
      }
    };
    auto issue_v = [&](int stage) {
      const uint16_t* v = v_base + (lane >= 32 ? off[1] : off[0]) + v_lane;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the stage's last reads are done
#pragma unroll
      for (int r = 0; r < LOADS; ++r) load_async_piece_nt(v_at + stage * STAGE + r * LOAD_BYTES, v + r * p.token_stride);
    };
    auto issue_k = [&]() {
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) k[kt][ks] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(k_base + off[kt] + k_lane + 32 * ks));
    };
    const int v_rd = ((4 * g + (n >> 2)) % LOADS) * LOAD_BYTES + ((4 * g + (n >> 2)) / LOADS) * (D * 2) + 8 * (n & 3);
    if (n_steps > 0) {
      place(0);
      issue_v(0);
      issue_k();
    }
    for (int step = 0; step < n_steps; ++step) {
      const int stage = step & 1;
      wait_loads();
      asm volatile("" ::: "memory");
      tile_key[0] = next_key[0];
      tile_key[1] = next_key[1];
      const bool more = step + 1 < n_steps;
      if (more) {
        place(step + 1);
        issue_v(stage ^ 1);
      }
      bool whole = true, full = true;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        const int key = tile_key[kt];
        whole = whole && key + 15 < groups.hull_end && (key + 15 < p.n_starting || key >= groups.window_begin);
        full = full && key + 15 <= w_last && (key >= w_first || key + 15 < p.n_starting);
      }
      if (!whole) {  // V of keys that nobody sees may be anything: cleared by the lanes that brought it
        const int key0 = lane >= 32 ? tile_key[1] : tile_key[0];
#pragma unroll
        for (int r = 0; r < LOADS; ++r)
          if (!(key0 != kNoKey && groups.sees(p, key0 + v_row + r)))
            *reinterpret_cast<u32x4*>(lds[w] + stage * STAGE + r * LOAD_BYTES + 16 * lane) = u32x4{0, 0, 0, 0};
        asm volatile("" ::: "memory");
      }
      f32x4 s[RT][2];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          s[rt][kt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) s[rt][kt] = mfma_16x16x32<DTYPE>(k[kt][ks], q[rt][ks], s[rt][kt]);
        }
      if (more) issue_k();
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
          pb[rt][2 * kt] = pack2<DTYPE>(x[0], x[1]);  // (rounded for the product, summed unrounded, as above)
          pb[rt][2 * kt + 1] = pack2<DTYPE>(x[2], x[3]);
        }
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
        const uint32_t from = v_at + stage * STAGE + v_rd + 32 * dt;
        const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)from));
        const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)(from + 512)));  // rows 16 further
        const u32x4 a = {lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) o[rt][dt] = mfma_16x16x32<DTYPE>(a, pb[rt], o[rt][dt]);
      }
    }

    // ---- the four waves' results joined --------------------------------------------------
    asm volatile("" ::: "memory");
    float* mine = reinterpret_cast<float*>(lds[w]);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const float l = rows_sum(l_run[rt]);
      if (g == 0) {
        sums_lds[w][rt * 16 + n][0] = m_run[rt];
        sums_lds[w][rt * 16 + n][1] = l;
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4*>(mine + (rt * 16 + n) * O_STRIDE + 16 * dt + 4 * g) = o[rt][dt];
    }
    __syncthreads();
    const bool cut = t_end - t_begin < request.n_tiles;
    constexpr int PIECES = D / 4;  // of a row
    for (int i = tid; i < heads * ROWS * PIECES; i += kFewThreads) {
      const int piece = i % PIECES, row = i / PIECES % ROWS, of = i / PIECES / ROWS, r = row0 + row;
      if (r >= request.n_tok * p.group) continue;
      float m = -INFINITY;
      for (int x = of; x < kFewWaves; x += heads) m = fmaxf(m, sums_lds[x][row][0]);
      const float m_use = m == -INFINITY ? 0.0f : m;
      f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
      float l = 0.0f;
      for (int x = of; x < kFewWaves; x += heads) {
        const float weight = fast_exp2(sums_lds[x][row][0] - m_use);
        l += weight * sums_lds[x][row][1];
        const f32x4 o4 = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds[x]) + row * O_STRIDE + 4 * piece);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] += weight * o4[e];
      }
      const int64_t token = request.first_tok + r / p.group, head = (kv_head0 + of) * p.group + r % p.group;
      if (piece == 0 && t_begin == 0) params.cuts[token * p.n_heads_q + head] = cut_of((int)blockIdx.x, n_cut, slot, of * ROWS + row);
      if (cut || !p.direct) {
        const int64_t to = cut ? (((int64_t)blockIdx.x * 2 + slot) * heads + of) * ROWS + row : (int64_t)p.first_share * p.n_tokens * p.n_heads_q + token * p.n_heads_q + head;
        *reinterpret_cast<f32x4*>((cut ? params.slot_out : p.partial_out) + to * D + 4 * piece) = acc;
        if (piece == 0) (cut ? params.slot_sums : p.partial_sums)[to] = f32x2{m, l};
      } else {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        *reinterpret_cast<u32x2*>(reinterpret_cast<uint16_t*>(p.out) + token * p.out_token + head * p.out_head + 4 * piece) =
            u32x2{pack2<DTYPE>(acc[0] * inv, acc[1] * inv), pack2<DTYPE>(acc[2] * inv, acc[3] * inv)};
        if (piece == 0) p.lse[head * p.n_tokens + token] = l == 0.0f ? INFINITY : (m + log2f(l)) * kLn2;
      }
    }
    __syncthreads();  // nobody's part of LDS is filled again before all have read it
  }
}

// ---------------------------------------------------------------------------
// The merge: out = sum_i 2^(m_i - m) O_i / sum_i 2^(m_i - m) l_i over a row's parts, rounded once.  The parts are the pieces of a unit
// that the kernel of few rows has cut, or the shares of the kernel of rows, or one or the other and the shares of a
// prefix.  A workgroup takes a row: D / 4 lanes hold it in 16-byte pieces, and the 1024 / D sets of such lanes take parts in turn (a
// wave that went through 128 parts alone took 17 us).
// ---------------------------------------------------------------------------
struct PagedMergeParams {
  PagedFewParams few;       // few.cuts null: the kernel of rows has made the shares
  const int32_t* cu_groups; // null: no prefixes
  int n_prefixes, n_own, n_shares, rows;  // shares of the requests' own keys; with those of the prefixes, which come behind them; rows of a chunk
};
constexpr int kPagedMergeThreads = 256;
template <int DTYPE, int D>
__global__ __launch_bounds__(kPagedMergeThreads) void paged_merge_kernel(const PagedMergeParams params) {
  const PagedAttnParams& p = params.few.a;
  constexpr int PIECES = D / 4, SETS = kPagedMergeThreads / PIECES;
  __shared__ f32x4 acc_lds[SETS][PIECES];
  __shared__ f32x2 sums_lds[SETS];
  const int row = blockIdx.x, tid = threadIdx.x, piece = tid % PIECES, set = tid / PIECES;
  const int64_t n_rows = p.n_tokens * p.n_heads_q;  // (fits 32 bits)
  // rows of no request are left as they were, and those of no prefix have no shares of one
  const int token = row / p.n_heads_q, head = row % p.n_heads_q;
  if ((token < first_token(p, 0)) | (token >= first_token(p, p.batch))) return;
  int first = 0, end = 0x7fffffff;
  if (params.cu_groups != nullptr) {
    PagedAttnParams of_prefix = p;
    of_prefix.cu_groups = params.cu_groups;
    first = first_token(of_prefix, 0);
    end = first_token(of_prefix, params.n_prefixes);
  }
  // (& on purpose: of two conditions joined by && or || here, this compiler, clang 22, left the second one out)
  const int n_shares = ((token >= first) & (token < end)) ? params.n_shares : params.n_own;
  // the pieces of a unit that was cut come first, in the place of the own share
  int n_cut = 0, wg = 0, slot = 0, slot_row = 0;
  const int slot_rows = params.few.heads * params.rows;
  if (params.few.cuts != nullptr) {
    const int2 at = params.few.cuts[row];
    wg = at.x;
    n_cut = at.y & 0xfffff;
    slot_row = at.y >> 20 & 0xff;
    slot = at.y >> 28;
    if (n_cut == 1) n_cut = 0;
    if ((n_cut == 0) & (p.direct != 0)) return;  // done where it was computed
  }
  const int n_parts = n_cut > 0 ? n_cut + n_shares - 1 : n_shares;
  // where part i is
  auto part = [&](int i, const f32x2*& sums) -> const float* {
    if (i < n_cut) {
      const int64_t at = ((int64_t)(wg + i) * 2 + (i == 0 ? slot : 0)) * slot_rows + slot_row;
      sums = params.few.slot_sums + at;
      return params.few.slot_out + at * D;
    }
    const int64_t at = (i - n_cut + (n_cut > 0)) * n_rows + row;
    sums = p.partial_sums + at;
    return p.partial_out + at * D;
  };
  float m = -INFINITY, l = 0.0f;
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  constexpr int AT_ONCE = 4;
  for (int i0 = set; i0 < n_parts; i0 += SETS * AT_ONCE) {
    f32x2 ml[AT_ONCE];
    f32x4 o4[AT_ONCE];
#pragma unroll
    for (int x = 0; x < AT_ONCE; ++x) {
      const int i = min(i0 + x * SETS, n_parts - 1);
      const f32x2* sums;
      const float* from = part(i, sums);
      ml[x] = *sums;
      o4[x] = *reinterpret_cast<const f32x4*>(from + 4 * piece);
    }
    float m_new = m;
#pragma unroll
    for (int x = 0; x < AT_ONCE; ++x) {
      if (i0 + x * SETS >= n_parts) ml[x] = f32x2{-INFINITY, 0.0f};
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
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += weight > 0.0f ? weight * o4[x][e] : 0.0f;  // (nothing is written of a share without weights)
    }
    m = m_new;
  }
  acc_lds[set][piece] = acc;
  if (piece == 0) sums_lds[set] = f32x2{m, l};
  __syncthreads();
  if (tid >= PIECES) return;
  m = -INFINITY;
#pragma unroll
  for (int x = 0; x < SETS; ++x) m = fmaxf(m, sums_lds[x][0]);
  const float m_use = m == -INFINITY ? 0.0f : m;
  l = 0.0f;
  acc = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int x = 0; x < SETS; ++x) {
    const float weight = fast_exp2(sums_lds[x][0] - m_use);
    l += weight * sums_lds[x][1];
    const f32x4 o4 = acc_lds[x][tid];
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] += weight * o4[e];
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  *reinterpret_cast<u32x2*>(reinterpret_cast<uint16_t*>(p.out) + token * p.out_token + head * p.out_head + 4 * tid) =
      u32x2{pack2<DTYPE>(acc[0] * inv, acc[1] * inv), pack2<DTYPE>(acc[2] * inv, acc[3] * inv)};
  if (tid == 0) p.lse[(int64_t)head * p.n_tokens + token] = l == 0.0f ? INFINITY : (m + log2f(l)) * kLn2;
}

// ---- host ---------------------------------------------------------------------------

struct PagedShape {
  int n_tokens, batch, n_heads_q, n_heads_kv, head_dim;
};
// Row tiles of one kv head: every request may have a partial one.
static int64_t row_tiles(const PagedShape& s) {
  return (int64_t)s.n_tokens * (s.n_heads_q / s.n_heads_kv) / kRowsBM + s.batch;
}
// Shares of a tile's keys: enough for two rounds of the device's workgroups.
// Keys that the queries of a request see, of all of them.
static int64_t seen_keys(int64_t max_q, int64_t max_keys, int window, int n_starting) {
  return window > 0 ? std::min(max_keys, max_q + window + n_starting) : max_keys;
}
static int row_shares(const PagedShape& s, int64_t max_keys) {
  const int64_t items = std::max<int64_t>(row_tiles(s) * s.n_heads_kv, 1);
  const int64_t wanted = (4 * (int64_t)device_cu_count() + items - 1) / items;
  const int64_t most = std::max<int64_t>((max_keys + kRowsBN * kMinTilesPerShare - 1) / (kRowsBN * kMinTilesPerShare), 1);
  return (int)std::min<int64_t>({wanted, most, 256});
}
static size_t shares_bytes(const PagedShape& s, int n_shares) {
  return (size_t)n_shares * s.n_tokens * s.n_heads_q * (s.head_dim + 2) * sizeof(float);
}

static int launch_rows(const PagedAttnParams& p, int head_dim, int dtype, void* stream) {
  const int64_t n_wg = (int64_t)p.n_tiles * p.n_heads_kv * p.n_splits;
  DCP_REQUIRE(n_wg < ((int64_t)1 << 31), "paged_attn: too many work items");
  KernelTimer timer("paged_rows_kernel", stream);
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)n_wg), dim3(kRowsThreads), 0, (hipStream_t)stream, p); };
  if (dtype == DCP_DTYPE_BF16) {
    if (head_dim == 128) launch(paged_rows_kernel<DCP_DTYPE_BF16, 128>);
    else launch(paged_rows_kernel<DCP_DTYPE_BF16, 64>);
  } else {
    if (head_dim == 128) launch(paged_rows_kernel<DCP_DTYPE_FP16, 128>);
    else launch(paged_rows_kernel<DCP_DTYPE_FP16, 64>);
  }
  return check_launch("paged_rows_kernel");
}

// How a call is laid out: which kernel takes the requests' own keys, and what of the workspace is whose.
struct PagedPlan {
  int rows = 0;      // of a chunk of the kernel of few rows; 0: the kernel of rows takes them
  int n_wg = 0, heads = 1;  // of the kernel of few rows; kv heads of a workgroup
  int n_own = 1, n_prefix = 0;  // shares
  size_t cuts = 0, slots = 0, shares = 0;  // bytes
  size_t bytes() const { return cuts + slots + shares; }
};
static size_t up16(size_t n) { return (n + 15) / 16 * 16; }
static PagedPlan plan_paged(const PagedShape& s, int64_t max_q, int64_t max_keys, int n_prefixes, int64_t max_prefix) {
  PagedPlan plan;
  const int64_t rows = max_q * (s.n_heads_q / s.n_heads_kv);
  if (rows <= 32 && s.batch <= kFewMaxBatch) {
    plan.rows = rows <= 16 ? 16 : 32;
    plan.n_wg = 2 * device_cu_count();
    const int64_t tiles = (int64_t)s.batch * s.n_heads_kv * ((max_keys + kFewBN - 1) / kFewBN) / plan.n_wg;
    plan.heads = tiles < (getenv("X_T") ? atoi(getenv("X_T")) : 64) ? 1 : s.n_heads_kv % 4 == 0 ? 4 : s.n_heads_kv % 2 == 0 ? 2 : 1;
    if (getenv("X_HEADS")) plan.heads = std::min(plan.heads, atoi(getenv("X_HEADS")));
    plan.cuts = up16((size_t)s.n_tokens * s.n_heads_q * sizeof(int2));
    plan.slots = (size_t)plan.n_wg * 2 * plan.heads * plan.rows * (s.head_dim + 2) * sizeof(float);
  } else {
    plan.n_own = row_shares(s, max_keys);
  }
  if (n_prefixes > 0) {
    const PagedShape of_prefix = {s.n_tokens, n_prefixes, s.n_heads_q, s.n_heads_kv, s.head_dim};
    plan.n_prefix = row_shares(of_prefix, max_prefix);
  }
  if (plan.n_own + plan.n_prefix > 1) plan.shares = shares_bytes(s, plan.n_own + plan.n_prefix);
  return plan;
}

template <int RT>
static void launch_few_rows(const PagedFewParams& f, const PagedPlan& plan, int head_dim, int dtype, void* stream) {
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)plan.n_wg), dim3(kFewThreads), 0, (hipStream_t)stream, f); };
  if (dtype == DCP_DTYPE_BF16) {
    if (head_dim == 128) launch(paged_few_kernel<DCP_DTYPE_BF16, 128, RT>);
    else launch(paged_few_kernel<DCP_DTYPE_BF16, 64, RT>);
  } else {
    if (head_dim == 128) launch(paged_few_kernel<DCP_DTYPE_FP16, 128, RT>);
    else launch(paged_few_kernel<DCP_DTYPE_FP16, 64, RT>);
  }
}

// The requests' own keys, and the merge where there is something to join.
static int launch_own(PagedAttnParams p, const PagedPlan& plan, const int32_t* cu_groups, int n_prefixes, int head_dim, int dtype, void* workspace,
                      void* stream) {
  PagedFewParams f = {};
  if (plan.rows > 0) {
    f.cuts = reinterpret_cast<int2*>(workspace);
    f.slot_out = reinterpret_cast<float*>(reinterpret_cast<char*>(workspace) + plan.cuts);
    f.slot_sums = reinterpret_cast<f32x2*>(f.slot_out + (size_t)plan.n_wg * 2 * plan.heads * plan.rows * head_dim);
    f.a = p;
    f.heads = plan.heads;
    KernelTimer timer("paged_few_kernel", stream);
    if (plan.rows == 16) launch_few_rows<1>(f, plan, head_dim, dtype, stream);
    else launch_few_rows<2>(f, plan, head_dim, dtype, stream);
    if (const int status = check_launch("paged_few_kernel")) return status;
  } else {
    if (const int status = launch_rows(p, head_dim, dtype, stream)) return status;
    if (p.direct) return DCP_OK;
    f.a = p;
  }
  const PagedMergeParams m = {f, cu_groups, n_prefixes, plan.n_own, plan.n_own + plan.n_prefix, plan.rows};
  KernelTimer timer("paged_merge_kernel", stream);
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)(p.n_tokens * p.n_heads_q)), dim3(kPagedMergeThreads), 0, (hipStream_t)stream, m);
  };
  if (dtype == DCP_DTYPE_BF16) {
    if (head_dim == 128) launch(paged_merge_kernel<DCP_DTYPE_BF16, 128>);
    else launch(paged_merge_kernel<DCP_DTYPE_BF16, 64>);
  } else {
    if (head_dim == 128) launch(paged_merge_kernel<DCP_DTYPE_FP16, 128>);
    else launch(paged_merge_kernel<DCP_DTYPE_FP16, 64>);
  }
  return check_launch("paged_merge_kernel");
}

static void place_shares(PagedAttnParams& p, const PagedPlan& plan, void* workspace, int head_dim) {
  p.partial_out = reinterpret_cast<float*>(reinterpret_cast<char*>(workspace) + plan.cuts + plan.slots);
  p.partial_sums = reinterpret_cast<f32x2*>(p.partial_out + (size_t)(plan.n_own + plan.n_prefix) * p.n_tokens * p.n_heads_q * head_dim);
}

}  // namespace dcp

using namespace dcp;

namespace {

PagedShape shape_of(const dcp_paged_attn_args& x) { return {x.n_tokens, x.batch, x.n_heads_q, x.n_heads_kv, x.head_dim}; }

PagedPlan plan_of(const dcp_paged_attn_args& x) {
  return plan_paged(shape_of(x), x.max_seqlen_q, seen_keys(x.max_seqlen_q, x.max_seqlen_k, x.window, x.n_starting), x.n_prefixes, x.max_prefix_len);
}

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
  DCP_REQUIRE(std::max((int64_t)x.table_width, (int64_t)(x.n_prefixes ? x.prefix_width : 0)) * x.page_size < 0x7fffff00, "paged_attn: too many keys a request");
  DCP_REQUIRE(x.page_stride % 8 == 0 && x.token_stride % 8 == 0 && x.head_stride % 8 == 0 && x.q_token_stride % 8 == 0 && x.q_head_stride % 8 == 0 &&
                  x.out_token_stride % 4 == 0 && x.out_head_stride % 4 == 0, "paged_attn: q, k, v strides must be multiples of 8 elements (out: 4)");
  DCP_REQUIRE(x.page_stride >= 0 && x.token_stride >= 0 && x.head_stride >= 0 && x.q_token_stride >= 0 && x.q_head_stride >= 0 &&
                  x.out_token_stride > 0 && x.out_head_stride > 0, "paged_attn: negative stride");
  DCP_REQUIRE(((reinterpret_cast<uintptr_t>(x.q) | reinterpret_cast<uintptr_t>(x.k_cache) | reinterpret_cast<uintptr_t>(x.v_cache) |
                reinterpret_cast<uintptr_t>(x.out)) & 15) == 0, "paged_attn: q, k, v and out must be 16-byte aligned");
  DCP_REQUIRE((int64_t)x.n_tokens * x.n_heads_q < ((int64_t)1 << 31), "paged_attn: too many queries");
  DCP_REQUIRE(x.cu_seqlens_q != nullptr || x.n_tokens == x.batch, "paged_attn: without cu_seqlens_q every request has one token, got %d for %d",
              x.n_tokens, x.batch);
  if (x.n_tokens == 0 || x.batch == 0) return DCP_OK;
  DCP_REQUIRE(x.q && x.out && x.lse && x.block_table && x.seq_lens && (x.n_pages == 0 || (x.k_cache && x.v_cache)) &&
                  (x.n_prefixes == 0 || (x.prefix_table && x.prefix_lens && x.cu_groups)), "paged_attn: null argument");
  DCP_REQUIRE(x.max_seqlen_q > 0 && x.max_seqlen_k > 0 && (x.n_prefixes == 0 || x.max_prefix_len > 0), "paged_attn: the longest lengths must be positive");
  DCP_REQUIRE(row_tiles(shape_of(x)) < ((int64_t)1 << 31) - x.n_prefixes, "paged_attn: too many rows");
  return DCP_OK;
}

int paged_attn(const dcp_paged_attn_args& x, void* workspace, size_t workspace_bytes, void* stream) {
  DCP_RECORDED(paged_attn(x, workspace, workspace_bytes, stream));
  if (const int status = check_paged(x)) return status;
  if (x.n_tokens == 0 || x.batch == 0) return DCP_OK;
  const PagedPlan plan = plan_of(x);
  const size_t needed = plan.bytes();
  DCP_REQUIRE(needed == 0 || (workspace && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0 && workspace_bytes >= needed),
              "paged_attn: workspace of %zu bytes is missing, not 16-byte aligned or smaller than the %zu needed", workspace_bytes, needed);
  PagedAttnParams p = {};
  p.q = x.q; p.k = x.k_cache; p.v = x.v_cache; p.out = x.out; p.lse = x.lse;
  p.block_table = x.block_table; p.key_lens = x.seq_lens; p.cu_seqlens_q = x.cu_seqlens_q;
  p.table_stride = x.table_stride;
  p.q_token = x.q_token_stride; p.q_head = x.q_head_stride; p.out_token = x.out_token_stride; p.out_head = x.out_head_stride;
  p.page_stride = x.page_stride; p.token_stride = x.token_stride; p.head_stride = x.head_stride;
  p.table_width = x.table_width; p.n_pages = x.n_pages; p.page_size = x.page_size;
  p.batch = p.n_requests = x.batch; p.n_tokens = x.n_tokens;
  p.n_heads_q = x.n_heads_q; p.n_heads_kv = x.n_heads_kv; p.group = x.n_heads_q / x.n_heads_kv;
  p.window = x.window; p.n_starting = x.n_starting;
  p.scale_log2 = x.softmax_scale * kLog2e;
  p.n_splits = plan.n_own;
  p.n_tiles = (int)row_tiles(shape_of(x));
  p.direct = plan.n_own + plan.n_prefix == 1;
  if (!p.direct) place_shares(p, plan, workspace, x.head_dim);
  if (x.n_prefixes > 0) {
    PagedAttnParams pre = p;
    pre.block_table = x.prefix_table; pre.key_lens = x.prefix_lens; pre.cu_groups = x.cu_groups;
    pre.table_stride = x.prefix_stride; pre.table_width = x.prefix_width;
    pre.batch = x.n_prefixes;
    pre.n_splits = plan.n_prefix;
    pre.n_tiles = (int)row_tiles({x.n_tokens, x.n_prefixes, x.n_heads_q, x.n_heads_kv, x.head_dim});
    pre.first_share = plan.n_own;
    if (const int status = launch_rows(pre, x.head_dim, x.dtype, stream)) return status;
  }
  return launch_own(p, plan, x.n_prefixes > 0 ? x.cu_groups : nullptr, x.n_prefixes, x.head_dim, x.dtype, workspace, stream);
}

}  // namespace

extern "C" size_t dcp_paged_attn_workspace_bytes(const dcp_paged_attn_args* args) {
  if (args == nullptr || check_paged(*args) != DCP_OK || args->n_tokens == 0 || args->batch == 0) return 0;
  return plan_of(*args).bytes();
}

extern "C" int dcp_paged_attn(const dcp_paged_attn_args* args, void* workspace, size_t workspace_bytes, void* stream) {
  DCP_REQUIRE(args != nullptr, "paged_attn: null argument");
  return paged_attn(*args, workspace, workspace_bytes, stream);
}
