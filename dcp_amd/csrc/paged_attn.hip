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
#include <algorithm>

#include "paged_rows.h"
#include "record.h"

namespace dcp {

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
  typedef FewLds<D, RT, NW> Lds;
  constexpr int KS = D / 32, DT = D / 16, ROWS = Lds::ROWS, LOADS = Lds::LOADS;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  float(*sums)[ROWS][2] = reinterpret_cast<float(*)[ROWS][2]>(lds + Lds::SUMS);
  int* chunk_sums = reinterpret_cast<int*>(lds + Lds::CHUNKS);

  FewWalk<ROWS, NW> walk(wg, chunk_sums);
  FewUnit u;
  char* my_lds = lds + w * Lds::WAVE;  // K of a tile and V of a tile
  const uint32_t k_at = lds_address(lds) + w * Lds::WAVE, v_at = k_at + Lds::STAGE;
  while (walk.next(u)) {
    PagedArgs& p = fresh_kernel_args<PagedParams>();
    // the workgroup's kv heads at once, the waves that take turns at a head's tiles, and which of each the wave is
    const int heads = 1 << p.few_heads_log2, head_groups = p.n_heads_kv >> p.few_heads_log2, turns = NW >> p.few_heads_log2;
    const int my_head = w & (heads - 1), my_turn = w >> p.few_heads_log2;
    const FewRequest& request = u.request;
    const int b = u.b, unit = u.unit, t_begin = u.t_begin, t_end = u.t_end;
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
    join_few<DTYPE, D, ROWS, NW, Lds::WAVE>(walk, u, walk.slot(u), walk.n_cut(u), lds, sums, kv_head0, row0,
                                            [](PagedArgs& p, int r) { return r / p.group; });
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

int launch_paged_merge(PagedParams& p, int dtype, int head_dim, int64_t parts, void* stream) {
  const struct { int dtype, head_dim; } x = {dtype, head_dim};
  // eight parts a set of lanes, as far as the longest lengths tell how many there are
  const int sets = kPagedMergeThreads / (head_dim / 4);
  p.merge_sets = 1;
  while (p.merge_sets < sets && parts > 8 * p.merge_sets) p.merge_sets *= 2;
  const int64_t n_wg = ((int64_t)p.n_tokens * p.n_heads_q * p.merge_sets + sets - 1) / sets;
  if (n_wg >= (int64_t)1 << 31) return fail(DCP_ERR_ARG, "paged_attn: too many work items");
  KernelTimer timer("paged_merge_kernel", stream);
  hipLaunchKernelGGL((DCP_PAGED_KERNEL(paged_merge_kernel)), dim3((unsigned)n_wg), dim3(kPagedMergeThreads), 0, (hipStream_t)stream, p);
  return check_launch("paged_merge_kernel");
}

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
  p.few_rows = plan.rows; p.few_heads_log2 = plan.heads / 2; p.few_whole = plan.whole; p.n_few = plan.n_few; p.few_first = plan.few_first;

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
    const int64_t units = std::max<int64_t>((int64_t)x.batch * x.n_heads_kv / plan.heads, 1);
    if (status == DCP_OK)
      status = launch_paged_merge(p, x.dtype, x.head_dim, (plan.few && !plan.whole ? plan.n_few / units + 2 : plan.n_own) + plan.n_prefix, stream);
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
