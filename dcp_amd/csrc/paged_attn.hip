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
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    const int64_t token = out_row[rt] / p.n_heads_q, head = out_row[rt] % p.n_heads_q;
    uint16_t* to = reinterpret_cast<uint16_t*>(p.out) + token * p.out_token + head * p.out_head + 4 * g;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      *reinterpret_cast<u32x2*>(to + 16 * dt) = u32x2{pack2<DTYPE>(o[rt][dt][0] * inv, o[rt][dt][1] * inv),
                                                      pack2<DTYPE>(o[rt][dt][2] * inv, o[rt][dt][3] * inv)};
    if (g == 0) p.lse[head * p.n_tokens + token] = l > 0.0f ? (m_run[rt] + log2f(l)) * kLn2 : INFINITY;
  }
}

// Adds up a row's shares: out = sum_i 2^(m_i - m) O_i / sum_i 2^(m_i - m) l_i, rounded once.  A wave takes a row.
struct PagedMergeParams {
  const float* partial_out;
  const f32x2* partial_sums;
  void* out;
  float* lse;
  const int32_t* cu_seqlens_q;
  const int32_t* cu_groups;
  int64_t out_token, out_head;
  int n_tokens, n_heads_q, batch, n_prefixes;
  int n_own, n_shares;  // shares of the requests' own keys; with those of the prefixes, which come behind them
};
constexpr int kPagedMergeThreads = 256;
template <int DTYPE, int D>
__global__ __launch_bounds__(kPagedMergeThreads) void paged_merge_kernel(const PagedMergeParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t n_rows = p.n_tokens * p.n_heads_q;  // (fits 32 bits)
  // (a wave has one row: said so, what follows from it is scalar, the branches too)
  const int row = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * (kPagedMergeThreads / 64) + (threadIdx.x >> 6)));
  if (row >= n_rows) return;
  constexpr int PER = D / 64;
  // rows of no request are left as they were, and those of no prefix have no shares of one
  const int token = row / p.n_heads_q, head = row % p.n_heads_q;
  auto first_token = [&](int r) { return p.cu_seqlens_q != nullptr ? p.cu_seqlens_q[min(max(r, 0), p.batch)] : r; };
  if (token < first_token(0) || token >= first_token(p.batch)) return;
  int first = 0, end = 0x7fffffff;
  if (p.cu_groups != nullptr) {
    first = first_token(p.cu_groups[0]);
    end = first_token(p.cu_groups[p.n_prefixes]);
  }
  // (& on purpose: of the two conditions joined by && or ||, this compiler, clang 22, leaves the second one out)
  const int n_shares = ((token >= first) & (token < end)) ? p.n_shares : p.n_own;
  float m = -INFINITY;
  for (int i = lane; i < n_shares; i += 64) m = fmaxf(m, p.partial_sums[i * n_rows + row][0]);
#pragma unroll
  for (int off = 32; off > 0; off /= 2) m = fmaxf(m, __shfl_xor(m, off));
  const float m_use = m == -INFINITY ? 0.0f : m;
  float acc[PER] = {}, l = 0.0f;
  for (int i = 0; i < n_shares; ++i) {
    const f32x2 ml = p.partial_sums[i * n_rows + row];
    if (!(ml[1] != 0.0f)) continue;  // (no visible key, and nothing written)
    const float weight = fast_exp2(ml[0] - m_use);
    l += weight * ml[1];
    const float* from = p.partial_out + (i * n_rows + row) * D + PER * lane;
#pragma unroll
    for (int e = 0; e < PER; ++e) acc[e] += weight * from[e];
  }
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
  uint16_t* to = reinterpret_cast<uint16_t*>(p.out) + token * p.out_token + head * p.out_head + PER * lane;
#pragma unroll
  for (int e = 0; e < PER; ++e) to[e] = Elem<DTYPE>::store(acc[e] * inv);
  if (lane == 0) p.lse[(int64_t)head * p.n_tokens + token] = l > 0.0f ? (m + log2f(l)) * kLn2 : INFINITY;
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
static int row_shares(const PagedShape& s, int64_t max_keys) {
  const int64_t items = std::max<int64_t>(row_tiles(s) * s.n_heads_kv, 1);
  const int64_t wanted = (4 * (int64_t)device_cu_count() + items - 1) / items;
  const int64_t most = std::max<int64_t>((max_keys + kRowsBN * kMinTilesPerShare - 1) / (kRowsBN * kMinTilesPerShare), 1);
  return (int)std::min<int64_t>({wanted, most, 256});
}
static size_t shares_bytes(const PagedShape& s, int n_shares) {
  return (size_t)n_shares * s.n_tokens * s.n_heads_q * (s.head_dim + 2) * sizeof(float);
}

static int check_paged(const char* what, const PagedShape& s, const PagedAttnParams& p, float softmax_scale, int dtype) {
  if (dtype != DCP_DTYPE_BF16 && dtype != DCP_DTYPE_FP16)
    return fail(DCP_ERR_UNSUPPORTED, "%s: dtype %d unsupported (bf16 and fp16 only)", what, dtype);
  if (s.head_dim != 64 && s.head_dim != 128) return fail(DCP_ERR_UNSUPPORTED, "%s: head_dim %d unsupported (64 or 128)", what, s.head_dim);
  DCP_REQUIRE(s.n_tokens >= 0 && s.batch >= 0 && p.n_pages >= 0, "%s: negative size", what);
  DCP_REQUIRE(s.n_heads_q > 0 && s.n_heads_kv > 0 && s.n_heads_q % s.n_heads_kv == 0, "%s: n_heads_q %d must be a multiple of n_heads_kv %d",
              what, s.n_heads_q, s.n_heads_kv);
  DCP_REQUIRE(softmax_scale > 0.0f, "%s: softmax_scale must be positive", what);
  DCP_REQUIRE(p.window >= 0 && p.n_starting >= 0, "%s: negative window or number of first tokens", what);
  DCP_REQUIRE(p.page_size > 0 && p.page_size % 16 == 0, "%s: page_size %d must be a positive multiple of 16", what, p.page_size);
  DCP_REQUIRE(p.table_width > 0 && p.table_stride >= 0, "%s: empty block tables", what);
  DCP_REQUIRE((int64_t)p.table_width * p.page_size < 0x7fffff00, "%s: too many keys a request", what);
  DCP_REQUIRE(p.page_stride % 8 == 0 && p.token_stride % 8 == 0 && p.head_stride % 8 == 0 && p.q_token % 8 == 0 && p.q_head % 8 == 0 &&
                  p.out_token % 4 == 0 && p.out_head % 4 == 0, "%s: q, k, v strides must be multiples of 8 elements (out: 4)", what);
  DCP_REQUIRE(p.page_stride >= 0 && p.token_stride >= 0 && p.head_stride >= 0 && p.q_token >= 0 && p.q_head >= 0 && p.out_token > 0 &&
                  p.out_head > 0, "%s: negative stride", what);
  DCP_REQUIRE(((reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v) |
                reinterpret_cast<uintptr_t>(p.out)) & 15) == 0, "%s: q, k, v and out must be 16-byte aligned", what);
  DCP_REQUIRE((int64_t)s.n_tokens * s.n_heads_q < ((int64_t)1 << 31), "%s: too many queries", what);
  return DCP_OK;
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

static int launch_merge(const PagedAttnParams& p, const int32_t* cu_groups, int n_prefixes, int n_shares, int head_dim, int dtype, void* stream) {
  const PagedMergeParams m = {p.partial_out, p.partial_sums, p.out, p.lse, p.cu_seqlens_q, cu_groups, p.out_token, p.out_head,
                              p.n_tokens, p.n_heads_q, p.batch, n_prefixes, p.n_splits, n_shares};
  const int64_t n_wg = ((int64_t)p.n_tokens * p.n_heads_q + kPagedMergeThreads / 64 - 1) / (kPagedMergeThreads / 64);
  KernelTimer timer("paged_merge_kernel", stream);
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)n_wg), dim3(kPagedMergeThreads), 0, (hipStream_t)stream, m); };
  if (dtype == DCP_DTYPE_BF16) {
    if (head_dim == 128) launch(paged_merge_kernel<DCP_DTYPE_BF16, 128>);
    else launch(paged_merge_kernel<DCP_DTYPE_BF16, 64>);
  } else {
    if (head_dim == 128) launch(paged_merge_kernel<DCP_DTYPE_FP16, 128>);
    else launch(paged_merge_kernel<DCP_DTYPE_FP16, 64>);
  }
  return check_launch("paged_merge_kernel");
}

static void place_shares(PagedAttnParams& p, void* workspace, int n_shares, int head_dim) {
  p.partial_out = reinterpret_cast<float*>(workspace);
  p.partial_sums = reinterpret_cast<f32x2*>(p.partial_out + (size_t)n_shares * p.n_tokens * p.n_heads_q * head_dim);
}

}  // namespace dcp

using namespace dcp;

extern "C" size_t dcp_paged_attn_workspace_bytes(int n_tokens, int batch, int n_heads_q, int n_heads_kv, int head_dim, int max_seqlen_q,
                                                 int max_seqlen_k) {
  if (n_tokens <= 0 || batch <= 0 || n_heads_q <= 0 || n_heads_kv <= 0 || n_heads_q % n_heads_kv != 0) return 0;
  const PagedShape s = {n_tokens, batch, n_heads_q, n_heads_kv, head_dim};
  const int n = row_shares(s, max_seqlen_k);
  return n > 1 ? shares_bytes(s, n) : 0;
}

extern "C" int dcp_paged_attn(const void* q, const void* k_cache, const void* v_cache, void* out, float* lse, const int32_t* block_table,
                              const int32_t* seq_lens, const int32_t* cu_seqlens_q, int n_tokens, int batch, int n_heads_q, int n_heads_kv,
                              int head_dim, int64_t q_token_stride, int64_t q_head_stride, int64_t out_token_stride, int64_t out_head_stride,
                              int n_pages, int page_size, int64_t page_stride, int64_t token_stride, int64_t head_stride, int table_width,
                              int64_t table_stride, int max_seqlen_q, int max_seqlen_k, int window, int n_starting, float softmax_scale,
                              int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  DCP_RECORDED(dcp_paged_attn(q, k_cache, v_cache, out, lse, block_table, seq_lens, cu_seqlens_q, n_tokens, batch, n_heads_q, n_heads_kv,
      head_dim, q_token_stride, q_head_stride, out_token_stride, out_head_stride, n_pages, page_size, page_stride, token_stride, head_stride,
      table_width, table_stride, max_seqlen_q, max_seqlen_k, window, n_starting, softmax_scale, dtype, workspace, workspace_bytes, stream));
  const PagedShape s = {n_tokens, batch, n_heads_q, n_heads_kv, head_dim};
  PagedAttnParams p = {};
  p.q = q; p.k = k_cache; p.v = v_cache; p.out = out; p.lse = lse;
  p.block_table = block_table; p.key_lens = seq_lens; p.cu_seqlens_q = cu_seqlens_q;
  p.table_stride = table_stride;
  p.q_token = q_token_stride; p.q_head = q_head_stride; p.out_token = out_token_stride; p.out_head = out_head_stride;
  p.page_stride = page_stride; p.token_stride = token_stride; p.head_stride = head_stride;
  p.table_width = table_width; p.n_pages = n_pages; p.page_size = page_size;
  p.batch = p.n_requests = batch; p.n_tokens = n_tokens;
  p.n_heads_q = n_heads_q; p.n_heads_kv = n_heads_kv;
  p.window = window; p.n_starting = n_starting;
  p.scale_log2 = softmax_scale * kLog2e;
  if (const int status = check_paged("paged_attn", s, p, softmax_scale, dtype)) return status;
  p.group = n_heads_q / n_heads_kv;
  DCP_REQUIRE(cu_seqlens_q != nullptr || n_tokens == batch, "paged_attn: without cu_seqlens_q every request has one token, got %d for %d",
              n_tokens, batch);
  if (n_tokens == 0 || batch == 0) return DCP_OK;
  DCP_REQUIRE(q && out && lse && block_table && seq_lens && (n_pages == 0 || (k_cache && v_cache)), "paged_attn: null argument");
  DCP_REQUIRE(max_seqlen_q > 0 && max_seqlen_k > 0, "paged_attn: the longest lengths must be positive");
  p.n_splits = row_shares(s, max_seqlen_k);
  const int64_t tiles = row_tiles(s);
  DCP_REQUIRE(tiles < ((int64_t)1 << 31), "paged_attn: too many rows");
  p.n_tiles = (int)tiles;
  p.direct = p.n_splits == 1;
  const size_t needed = p.direct ? 0 : shares_bytes(s, p.n_splits);
  DCP_REQUIRE(needed == 0 || (workspace && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0 && workspace_bytes >= needed),
              "paged_attn: workspace of %zu bytes is missing, not 16-byte aligned or smaller than the %zu needed", workspace_bytes, needed);
  if (!p.direct) place_shares(p, workspace, p.n_splits, head_dim);
  if (const int status = launch_rows(p, head_dim, dtype, stream)) return status;
  return p.direct ? DCP_OK : launch_merge(p, nullptr, 0, p.n_splits, head_dim, dtype, stream);
}

extern "C" size_t dcp_shared_prefix_attn_workspace_bytes(int n_tokens, int batch, int n_prefixes, int n_heads_q, int n_heads_kv, int head_dim,
                                                         int max_seqlen_q, int max_seqlen_k, int max_prefix_len) {
  if (n_tokens <= 0 || batch <= 0 || n_prefixes <= 0 || n_heads_q <= 0 || n_heads_kv <= 0 || n_heads_q % n_heads_kv != 0) return 0;
  const PagedShape s = {n_tokens, batch, n_heads_q, n_heads_kv, head_dim}, of_prefix = {n_tokens, n_prefixes, n_heads_q, n_heads_kv, head_dim};
  return shares_bytes(s, row_shares(s, max_seqlen_k) + row_shares(of_prefix, max_prefix_len));
}

extern "C" int dcp_shared_prefix_attn(const void* q, const void* k_cache, const void* v_cache, void* out, float* lse,
                                      const int32_t* prefix_table, const int32_t* prefix_lens, const int32_t* cu_groups,
                                      const int32_t* block_table, const int32_t* seq_lens, const int32_t* cu_seqlens_q, int n_tokens, int batch,
                                      int n_prefixes, int n_heads_q, int n_heads_kv, int head_dim, int64_t q_token_stride,
                                      int64_t q_head_stride, int64_t out_token_stride, int64_t out_head_stride, int n_pages, int page_size,
                                      int64_t page_stride, int64_t token_stride, int64_t head_stride, int prefix_width, int64_t prefix_stride,
                                      int table_width, int64_t table_stride, int max_seqlen_q, int max_seqlen_k, int max_prefix_len,
                                      float softmax_scale, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  DCP_RECORDED(dcp_shared_prefix_attn(q, k_cache, v_cache, out, lse, prefix_table, prefix_lens, cu_groups, block_table, seq_lens,
      cu_seqlens_q, n_tokens, batch, n_prefixes, n_heads_q, n_heads_kv, head_dim, q_token_stride, q_head_stride, out_token_stride,
      out_head_stride, n_pages, page_size, page_stride, token_stride, head_stride, prefix_width, prefix_stride, table_width, table_stride,
      max_seqlen_q, max_seqlen_k, max_prefix_len, softmax_scale, dtype, workspace, workspace_bytes, stream));
  const PagedShape s = {n_tokens, batch, n_heads_q, n_heads_kv, head_dim}, of_prefix = {n_tokens, n_prefixes, n_heads_q, n_heads_kv, head_dim};
  PagedAttnParams p = {};
  p.q = q; p.k = k_cache; p.v = v_cache; p.out = out; p.lse = lse;
  p.block_table = block_table; p.key_lens = seq_lens; p.cu_seqlens_q = cu_seqlens_q;
  p.table_stride = table_stride;
  p.q_token = q_token_stride; p.q_head = q_head_stride; p.out_token = out_token_stride; p.out_head = out_head_stride;
  p.page_stride = page_stride; p.token_stride = token_stride; p.head_stride = head_stride;
  p.table_width = table_width; p.n_pages = n_pages; p.page_size = page_size;
  p.batch = p.n_requests = batch; p.n_tokens = n_tokens;
  p.n_heads_q = n_heads_q; p.n_heads_kv = n_heads_kv;
  p.scale_log2 = softmax_scale * kLog2e;
  PagedAttnParams pre = p;
  pre.block_table = prefix_table; pre.key_lens = prefix_lens; pre.cu_groups = cu_groups;
  pre.table_stride = prefix_stride; pre.table_width = prefix_width; pre.batch = n_prefixes;
  if (const int status = check_paged("shared_prefix_attn", s, p, softmax_scale, dtype)) return status;
  if (const int status = check_paged("shared_prefix_attn", of_prefix, pre, softmax_scale, dtype)) return status;
  p.group = pre.group = n_heads_q / n_heads_kv;
  DCP_REQUIRE(cu_seqlens_q != nullptr || n_tokens == batch,
              "shared_prefix_attn: without cu_seqlens_q every request has one token, got %d for %d", n_tokens, batch);
  DCP_REQUIRE(n_prefixes > 0 || batch == 0, "shared_prefix_attn: no prefixes");
  if (n_tokens == 0 || batch == 0) return DCP_OK;
  DCP_REQUIRE(q && out && lse && prefix_table && prefix_lens && cu_groups && block_table && seq_lens && (n_pages == 0 || (k_cache && v_cache)),
              "shared_prefix_attn: null argument");
  DCP_REQUIRE(max_seqlen_q > 0 && max_seqlen_k > 0 && max_prefix_len > 0, "shared_prefix_attn: the longest lengths must be positive");
  p.n_splits = row_shares(s, max_seqlen_k);
  pre.n_splits = row_shares(of_prefix, max_prefix_len);
  const int64_t tiles = row_tiles(s);
  DCP_REQUIRE(tiles < ((int64_t)1 << 31) - n_prefixes, "shared_prefix_attn: too many rows");
  p.n_tiles = (int)tiles;
  pre.n_tiles = (int)row_tiles(of_prefix);
  const int n_shares = p.n_splits + pre.n_splits;
  const size_t needed = shares_bytes(s, n_shares);
  DCP_REQUIRE(workspace && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0 && workspace_bytes >= needed,
              "shared_prefix_attn: workspace of %zu bytes is missing, not 16-byte aligned or smaller than the %zu needed", workspace_bytes, needed);
  place_shares(p, workspace, n_shares, head_dim);
  place_shares(pre, workspace, n_shares, head_dim);
  pre.first_share = p.n_splits;
  if (const int status = launch_rows(pre, head_dim, dtype, stream)) return status;
  if (const int status = launch_rows(p, head_dim, dtype, stream)) return status;
  return launch_merge(p, cu_groups, n_prefixes, n_shares, head_dim, dtype, stream);
}
