// What the kernels that answer over a paged cache have in common: a call's arguments, a request's tokens and the 16-key groups that they
// see, how few rows' work is cut between workgroups and joined, and how many rows' tiles are found.
#pragma once

#include <math.h>

#include "attn_common.h"

namespace dcp {

// Whole numbers from 0 up to 2^31 divided by one that the host knows: 2 n mul / 2^(32 + shift) with mul = floor(2^(31 + shift) / d) + 1 and d
// at most 2^shift is n / d and less than 1 / d more.  (Three instructions; a division by any number is some twenty-five.)
struct Divider {
  uint32_t mul, shift;
  static Divider of(int d) {
    uint32_t shift = 0;
    while (((int64_t)1 << shift) < d) ++shift;
    return {(uint32_t)(((uint64_t)1 << (31 + shift)) / (uint64_t)d) + 1, shift};
  }
};
__device__ __forceinline__ int divide(int n, KernArgs<Divider>& by) { return (int)(__umulhi(2u * (uint32_t)n, by.mul) >> by.shift); }

// Keys that rows look at: the requests' own, or prefixes that requests share.
struct PagedSource {
  const int32_t* block_table;
  const int32_t* key_lens;
  const int32_t* cu_groups;  // prefixes: their requests; null for the requests' own keys
  int64_t table_stride;
  int table_width, batch;    // of prefixes or requests
  int first_share, n_shares; // see PagedParams::partial_out
  int n_tiles, xcd_group;    // row tiles of a kv head (kernel of rows); as many neighbouring work items are on one XCD
  int by_few;                // pieces of rows may be in slots (own keys: where the kernel of few rows takes them, or in 4 bits that of rows cuts them)
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
  // The kernel of few rows (in 4 bits that of rows as well): pieces of the units that are cut between workgroups, and where a row's pieces
  // are (cut_of).
  int2* cuts;        // [token][q head]
  float* slot_out;   // [workgroup][2][head of the workgroup][rows][D]
  f32x2* slot_sums;  // [workgroup][2][head of the workgroup][rows]
  int few_rows, few_heads_log2;  // rows of a unit; kv heads a workgroup takes at once: 1, 2 or 4
  int few_whole;                 // a workgroup takes a unit
  int n_few, few_first;     // workgroups; of paged_both_kernel those before the ones of rows
  int merge_sets;           // of lanes that share a row in the merge, a power of two
  Divider by_page, by_group, by_heads;  // page_size / 16, group, n_heads_kv (in 4 bits)
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

// The result of a row's 4 elements, from the sum of the weights.
template <int DTYPE>
__device__ __forceinline__ void store_row_piece(PagedArgs& p, int64_t token, int64_t head, int d, f32x4 o, float m, float l) {
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  *reinterpret_cast<u32x2*>(reinterpret_cast<uint16_t*>(p.out) + token * p.out_token + head * p.out_head + d) =
      u32x2{pack2<DTYPE>(o[0] * inv, o[1] * inv), pack2<DTYPE>(o[2] * inv, o[3] * inv)};
  if (d == 0) p.lse[head * p.n_tokens + token] = l == 0.0f ? INFINITY : (m + log2f(l)) * kLn2;
}

constexpr int kRowsThreads = 256, kRowsBM = 128, kRowsBN = 64;
constexpr int kMinTilesPerShare = 2;

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
template <int BM = kRowsBM>
__device__ __forceinline__ RowTile find_row_tile(PagedArgs& p, SourceArgs& src, int place) {
  const int lane = threadIdx.x & 63;
  // Up to 64 requests are counted.  Of more, request b's tiles begin at number floor(first_row / BM) + b: that leaves room for its last,
  // partial one, and needs no sum over the requests before it, but its places without a tile lie among the others, and CUs with two tiles
  // beside CUs with none (24 requests of 128 rows on 1024 keys, nearly half of the places empty: 40 us, counted 35; 64 of 64 rows on 4096 267
  // and 213).
  auto start = [&](int first, int b) { return (int)((int64_t)first * p.group / BM) + b; };
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
  const int n_keys = keys_of(p, src, b), n_tiles = (tokens.n * p.group + BM - 1) / BM;
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

// What a workgroup of few rows takes next: tiles [t_begin, t_end) of a request's unit (some of its rows and kv heads), in turns.
struct FewUnit {
  FewRequest request;
  int b, unit, t_begin, t_end;
  int taken, turns;  // turns that it takes, of those that the unit has
};

// A workgroup's share of all tiles (the host has checked that their number fits 32 bits), or its unit: a workgroup's waves go through it
// together, unit by unit.  Shares are counted in turns of the waves at a head's tiles: a cut inside one would cost both of its sides a whole
// one.  (One context of 1500 keys, 8 heads, which 47 tiles a head then fit no better: counted in tiles 14.4 us, in turns 11.4.)
// `chunk_sums`: LDS, an int for every 64 requests.
// WHOLE: it is known to be a unit.  START: turns that the start of a unit is counted as, so that a workgroup of many short units has fewer.
template <int ROWS, int NW, bool WHOLE = false, int START = 0>
struct FewWalk {
  int lane, wg, n_chunks, turns_log2, per, begin, end, at;
  int before = 0, chunk = 0, work, scan, index;
  bool whole_units;
  FewRequest requests;  // of the chunk: a lane's

  __device__ __forceinline__ FewRequest requests_of(int chunk, int& work) const {
    PagedArgs& p = fresh_kernel_args<PagedParams>();
    const int b = chunk * 64 + lane, turns = 1 << turns_log2;
    FewRequest r;
    r.first_tok = r.n_tok = r.n_keys = 0;
    r.n_tiles = 1;
    work = 0;
    if (b < p.own.batch) {
      r = FewRequest(p, b);
      work = r.units(p, ROWS) * (WHOLE || whole_units ? 1 : START + ((r.n_tiles + turns - 1) >> turns_log2));
    }
    return r;
  }
  __device__ __forceinline__ FewWalk(int wg_, int* chunk_sums) {
    PagedArgs& p0 = fresh_kernel_args<PagedParams>();
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    lane = threadIdx.x & 63;
    wg = wg_;
    n_chunks = (p0.own.batch + 63) / 64;
    whole_units = WHOLE || p0.few_whole != 0;
    turns_log2 = (NW == 8 ? 3 : 2) - p0.few_heads_log2;
    int total = 0;
    requests = requests_of(0, work);
    scan = wave_scan(work);  // the chunk's tiles (or units) up to and with the lane's request
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
    per = whole_units ? 1 : (total - 1) / p0.n_few + 1;
    begin = (int)min((int64_t)wg * per, (int64_t)total);
    end = (int)min((int64_t)begin + per, (int64_t)total);
    at = begin;
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
    index = __builtin_amdgcn_readfirstlane(min(__popcll(__ballot(before + scan <= begin)), 63));  // in the chunk
  }
  // The next piece of the share, if there is one.
  __device__ __forceinline__ bool next(FewUnit& u) {
    while (at < end) {
      if (index == 64) {
        before += __builtin_amdgcn_readlane(scan, 63);
        if (++chunk >= n_chunks) return false;
        requests = requests_of(chunk, work);
        scan = wave_scan(work);
        index = 0;
      }
      const int unit_end = before + __builtin_amdgcn_readlane(scan, index);
      if (at >= unit_end) {  // (no rows, or done)
        ++index;
        continue;
      }
      u.request = requests.of_lane(index);
      u.b = chunk * 64 + index;
      const int in_request = at - (unit_end - __builtin_amdgcn_readlane(work, index)), turns = 1 << turns_log2;
      if (in_request < 0) return false;  // (tables whose tokens are many times those there are: their sums wrap)
      u.turns = whole_units ? 1 : (u.request.n_tiles + turns - 1) >> turns_log2;
      u.unit = __builtin_amdgcn_readfirstlane(in_request / (u.turns + START));
      int first_turn = in_request - u.unit * (u.turns + START) - START;
      if (START > 0 && first_turn < 0) {
        at -= first_turn;
        first_turn = 0;
        if (at >= end) return false;
      }
      u.taken = min(u.turns - first_turn, end - at);
      u.t_begin = whole_units ? 0 : first_turn * turns;
      u.t_end = whole_units ? u.request.n_tiles : min(u.request.n_tiles, u.t_begin + u.taken * turns);
      at += u.taken;
      return true;
    }
    return false;
  }
  // (after next) where the piece is kept if its unit is cut: slot 0 if the share begins in the unit, and over how many
  // workgroups a unit that begins here is cut
  __device__ __forceinline__ int slot(const FewUnit& u) const { return at - u.taken == begin ? 0 : 1; }
  __device__ __forceinline__ int n_cut(const FewUnit& u) const { return (at - u.taken + u.turns - 1) / per - wg + 1; }
};

// The waves' results of a unit's piece joined and stored; `slot` and `n_cut` as FewWalk has them of it.  Wave x has row r's O, relative to its maximum, at lds + x * WAVE as
// float [row][D + 4], the maximum and the sum of the weights in sums[x][row]; it is of the workgroup's kv head x % heads.
// `token_of(p, r)`: r / group.  ONE_HEAD: the workgroup has one kv head.
template <int DTYPE, int D, int ROWS, int NW, int WAVE, bool ONE_HEAD = false, typename Walk, typename TokenOf>
__device__ __forceinline__ void join_few(const Walk& walk, const FewUnit& u, int slot, int n_cut, const char* lds, const float (*sums)[ROWS][2],
                                         int kv_head0, int row0, TokenOf token_of) {
  PagedArgs& p = fresh_kernel_args<PagedParams>();
  const int heads = ONE_HEAD ? 1 : 1 << p.few_heads_log2, n_rows = u.request.n_tok * p.group, group = p.group;
  const bool cut = u.taken < u.turns;
  constexpr int PIECES = D / 4;  // of a row
  for (int i = threadIdx.x; i < heads * ROWS * PIECES; i += NW * 64) {
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
      const f32x4 o4 = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds + x * WAVE) + row * (D + 4) + 4 * piece);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += weight * o4[e];
    }
    const int tok = token_of(p, r);
    const int64_t token = u.request.first_tok + tok, head = (kv_head0 + of) * group + (r - tok * group);
    if ((piece == 0) & (u.t_begin == 0) & !walk.whole_units) p.cuts[token * p.n_heads_q + head] = cut_of(walk.wg, n_cut, slot, of * ROWS + row);
    if (cut) {
      const int64_t to = (((int64_t)walk.wg * 2 + slot) * heads + of) * ROWS + row;
      *reinterpret_cast<f32x4*>(p.slot_out + to * D + 4 * piece) = acc;
      if (piece == 0) p.slot_sums[to] = f32x2{m, l};
    } else if (!p.direct) {
      const int64_t to = ((int64_t)p.own.first_share * p.n_tokens + token) * p.n_heads_q + head;
      *reinterpret_cast<f32x4*>(p.partial_out + to * D + 4 * piece) = acc;
      if (piece == 0) p.partial_sums[to] = f32x2{m, l};
    } else {
      store_row_piece<DTYPE>(p, token, head, 4 * piece, acc, m, l);
    }
  }
}

// The launch of the kernel that joins rows' parts (paged_attn.hip); `parts`: about how many a row has at most.
int launch_paged_merge(PagedParams& p, int dtype, int head_dim, int64_t parts, void* stream);

}  // namespace dcp
