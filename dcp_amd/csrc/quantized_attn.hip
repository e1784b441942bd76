// Attention over a paged K/V cache held in 4 bits (quantized_cache.h has the layout): causal or with a sliding window and first
// tokens that stay visible, for any number of new tokens a request.
//
//   out = softmax(scale q K^T) V over the visible keys, lse = log sum exp, K and V what the cache stands for
//
// Products are formed transposed, as over a cache of 16 bits, with 16x16x32 products of q's type:
//
//   S^T[key, row] = K Q^T      A = rows of K, B = Q in registers
//   O^T[d,   row] = V^T P^T    A = columns of V, B = P^T straight from the S^T accumulators
//
// A lane reads the codes of its own operands, 16 bytes of 16 keys at head size 128, and converts them: K two elements an
// instruction; V as well, and two pairs of keys are then put side by side.  What 4 bits hold times a power of two, 16 bits hold exactly.
// (The device multiplies 4 bits by 8 bits as they are, q in two or three parts.  Its sums of 128 such products were off by 4e-6 to 6e-6 of the sum of
// their sizes, by up to 5e-5 where q's parts are spread over their type; scores here by 2e-7.)
#include <algorithm>

#include "paged_rows.h"
#include "record.h"

namespace dcp {

// LDS of the kernel of few rows.  A wave has STAGES tiles of 32 keys under way: of both groups of 16 their codes as they lie in the cache (K's pieces
// in the order of the lanes that take them), then their exponents.  Its result takes the place of its tiles, of EARLY_ROWS and
// fewer that of the second alone.
template <int D, int RT, int NW>
struct QuantFewLds {
  static constexpr int ROWS = 16 * RT, STAGES = 2, GROUP = 16 * D, EXPS = 2 * GROUP, GROUP_EXPS = 256, STAGE = EXPS + 2 * GROUP_EXPS;
  static constexpr int RESULT = ROWS * (D + 4) * 4;  // float [row][D + 4]
  static constexpr int EARLY_ROWS = 8;
  static_assert(EARLY_ROWS * (D + 4) * 4 <= STAGE, "");
  static constexpr int WAVE = STAGES * STAGE > RESULT ? STAGES * STAGE : RESULT;
  static constexpr int SUMS = NW * WAVE;                   // float [wave][row][2]
  static constexpr int BYTES = SUMS + NW * ROWS * 2 * 4;
  static_assert(kFewMaxBatch / 64 * 4 <= SUMS, "");        // (FewWalk's sums, before there are tiles)
};

// The operands of V for two groups of 16 keys: those of elements n D / 16 + 2 U and the one after it.
template <int DTYPE, int D, int U>
__device__ __forceinline__ void two_columns_of_v(const QuantGroup<D> (&x)[2], const float (&scale)[2][4], u32x4& even, u32x4& odd) {
#pragma unroll
  for (int kt = 0; kt < 2; ++kt) {
    uint32_t pair[4];  // of each of the lane's four tokens, the two elements
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (D == 128) pair[j] = two_of_codes<DTYPE, U>(x[kt].v[j], scale[kt][j]);
      else pair[j] = j % 2 ? two_of_codes<DTYPE, 2 + U>(x[kt].v[j / 2], scale[kt][j]) : two_of_codes<DTYPE, U>(x[kt].v[j / 2], scale[kt][j]);
    }
#pragma unroll
    for (int jj = 0; jj < 2; ++jj) {
      even[2 * kt + jj] = __builtin_amdgcn_perm(pair[2 * jj + 1], pair[2 * jj], 0x05040100u);
      odd[2 * kt + jj] = __builtin_amdgcn_perm(pair[2 * jj + 1], pair[2 * jj], 0x07060302u);
    }
  }
}
// O^T += V^T P^T over them.
template <int DTYPE, int D, int RT, int U = 0>
__device__ __forceinline__ void multiply_v(const QuantGroup<D> (&x)[2], const float (&scale)[2][4], const u32x4 (&pb)[RT], f32x4 (&o)[RT][D / 16]) {
  if constexpr (U < D / 32) {
    u32x4 even, odd;
    two_columns_of_v<DTYPE, D, U>(x, scale, even, odd);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      o[rt][2 * U] = mfma_16x16x32<DTYPE>(even, pb[rt], o[rt][2 * U]);
      o[rt][2 * U + 1] = mfma_16x16x32<DTYPE>(odd, pb[rt], o[rt][2 * U + 1]);
    }
    multiply_v<DTYPE, D, RT, U + 1>(x, scale, pb, o);
  }
}

// The kernel of few rows: the waves of a workgroup share no tile.  Each takes tiles of 32 keys of its own and waits for nobody until its
// share of the keys is done; work is cut as over a cache of 16 bits (FewWalk), or whole units where they are short (WHOLE).
//
// What bounds it is the number of instructions: at 7 TB/s the memory would leave a SIMD 335 slots of 4 cycles a tile, and a tile takes 333 with its
// share of starts and joins (64 contexts of up to 8192 keys, 8 kv heads of 128: 38 us, 5.2 TB/s, a slot taken in 73 % of them).  64 conversions
// and 32 of their results put in order are what the tile cannot do without; whether it has to be masked is asked once for 32 of them, and
// weights are taken against a reference maximum that the tile's own is only looked for where the weights' sum says so.  What is done once a
// piece is bound by the fetch of its instructions (some 15 ns each the first time they are met), so each step stands once in the
// code, whichever piece it is of, tiles are not unrolled over their places in LDS, and there is no division by a number known on the host.
//
// The start of a piece counts as kStartTurns turns of its tiles.  us at 0, 2, 3, 4 and 6: 24 requests of up to 4000 keys and 5 tokens 25.7, 22.3, 20.4,
// 20.4, 20.9; 64 of up to 8192 43.6, 40.5, 40.0, 40.7, 42.5; 100 of up to 5000, 4 kv heads of 64, 24.3, 21.9, 21.3, 20.7, 21.7.
constexpr int kStartTurns = 3;
template <int DTYPE, int D, int RT, int NW, bool WHOLE>
__global__ __launch_bounds__(NW * 64, NW == 4 && (RT == 1 || D == 64) ? (RT == 1 && D == 64 ? 4 : 3) : 2) void quantized_few_kernel(const PagedParams) {
  typedef QuantFewLds<D, RT, NW> Lds;
  typedef QuantTile<D> Tile;
  __shared__ __attribute__((aligned(16))) char lds[Lds::BYTES];
  constexpr int KS = D / 32, DT = D / 16, ROWS = Lds::ROWS;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  float(*sums)[ROWS][2] = reinterpret_cast<float(*)[ROWS][2]>(lds + Lds::SUMS);

  FewWalk<ROWS, NW, WHOLE, WHOLE ? 0 : kStartTurns> walk(blockIdx.x, reinterpret_cast<int*>(lds));
  if (walk.n_chunks > 1) __syncthreads();
  // ---- the piece at work -------------------------------------------------------------------
  FewUnit u;
  int kv_head = 0, row0 = 0, n_groups = 0, n_steps = 0;
  const char* head = nullptr;
  int all_last = 0, all_first = 0;  // every row sees the keys up to the one and, of those behind the first tokens, from the other on
  int last_key[RT];                 // of the lane's rows (past the last one: the last one again, not written)
  u32x4 q[RT][KS];                  // slots of product ks: D / 4 elements from g D / 4 on, eight at a time
  // Of 32 of the wave's tiles of it lane 2 i + j holds the 16-key group j of the i-th: where it is, and its first key.  Tiles are asked for two
  // steps ahead, so the keys of the next 32 are known before the last two of these are done.
  int lane_page, lane_tile, lane_key, lane_key_ahead;
  int64_t lane_off;
  uint64_t full = 0, full_ahead;  // bit 2 i + j: every row sees all of that group
  auto ask = [&](int step) {
    PagedArgs& p = fresh_kernel_args<PagedParams>();
    const int group = 2 * (u.t_begin + w + NW * (step + (lane >> 1))) + (lane & 1);
    lane_key_ahead = kNoKey;
    lane_page = -1;
    lane_tile = 0;
    if (group < n_groups && group < 2 * u.t_end) {
      const int at = u.request.groups(p).at(group), entry = divide(at, p.by_page);
      lane_key_ahead = at * 16;
      lane_tile = at - entry * (p.page_size / 16);
      lane_page = p.own.block_table[u.b * p.own.table_stride + entry];
    }
  };
  auto told = [&]() {
    PagedArgs& p = fresh_kernel_args<PagedParams>();
    const bool there = (unsigned)lane_page < (unsigned)p.n_pages;
    lane_off = there ? lane_page * p.page_stride + (int64_t)lane_tile * Tile::BYTES : 0;
    const int key = lane_key_ahead = there ? lane_key_ahead : kNoKey;
    full_ahead = __ballot((key + 15 <= all_last) & ((key >= all_first) | (key + 15 < p.n_starting)));
  };

  // ---- a tile goes from memory straight into LDS, into the place of the one two before it, which the wave has read by then ---------
  char* my_lds = lds + w * Lds::WAVE;
  const uint32_t my_at = lds_address(lds) + w * Lds::WAVE;
  const uint32_t k_from = D == 128 ? Tile::k_of(lane) : 16 * lane, v_from = Tile::v_of(lane), exps_from = Tile::K_EXP + lane % (D / 4) * 4;
  constexpr int LOADS = D == 128 ? 6 : 4;
  auto issue = [&](int step) {
    const uint32_t to = my_at + (step & 1) * Lds::STAGE;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the last reads of what is there are done
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const uint64_t at = (uint64_t)(head + lane_value(lane_off, 2 * (step % 32) + kt));
      KvTile<D>::load_group_at_streaming(to + kt * Lds::GROUP, at, k_from);  // (at head size 64 with V)
      if constexpr (D == 128) KvTile<D>::load_group_at_streaming(to + kt * Lds::GROUP + Tile::V, at, v_from);
      load_async_dword(to + Lds::EXPS + kt * Lds::GROUP_EXPS, exps_from, reinterpret_cast<const void*>(at));
    }
  };
  const char* k_read = my_lds + (D == 128 ? 16 * lane : Tile::k_of(lane));
  const char* v_read = my_lds + Tile::v_of(lane);
  const char* k_exp_read = my_lds + Lds::EXPS - Tile::K_EXP + Tile::k_exp_of(lane);
  const char* v_exp_read = my_lds + Lds::EXPS - Tile::K_EXP + Tile::v_exp_of(lane);

  f32x4 o[RT][DT];
  float m_run[RT], l_run[RT], l_rounded[RT];  // (of the rounded weights)
  int have = 0;  // results to be joined
  asm("" : "+s"(have));  // (not known to be none: the compiler would write the first turn out on its own)
  FewUnit done = {};
  int slot = 0, n_cut = 0, done_head = 0, done_row0 = 0;
  while (true) {
    // ---- the next piece's pages and rows are asked for, the waves' results of the last one are joined ----------------------
    const bool more = walk.next(u) & (!WHOLE | !have);
    if (!more && !have) return;
    if (more) {
      PagedArgs& p = fresh_kernel_args<PagedParams>();
      const int chunk = divide(u.unit, p.by_heads);
      kv_head = u.unit - chunk * p.n_heads_kv;
      row0 = chunk * ROWS;
      n_groups = u.request.n_keys > 0 ? u.request.groups(p).count() : 0;
      n_steps = max((min(u.t_end, n_groups) - u.t_begin - w + NW - 1) / NW, 0);  // (a tile or more has a group)
      head = reinterpret_cast<const char*>(p.k) + kv_head * p.head_stride;
      ask(0);
    }
    // Results of few rows lie in the second tile's place, so that the first tile of the next piece need not wait for them to be read.
    const bool early = done.request.n_tok * fresh_kernel_args<PagedParams>().group - done_row0 <= Lds::EARLY_ROWS;
    if (have) {  // element (4 g + e) D / 16 + dt is o[dt][e]
      float* result = reinterpret_cast<float*>(my_lds + (early ? Lds::STAGE : 0));
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        // O is divided by the sum of the rounded weights, so that rounding one that outweighs the others cancels: its maximum is given as
        // that much larger.  (The reference is a row's maximum of some tile, so the largest weight need not be 1.  rms error against 64 bits
        // in bf16, of which 0.0017 is the result's own rounding: 0.0023 -> 0.0019, for 1 % of the time.)
        const float l = rows_sum(l_run[rt]), rounded = rows_sum(l_rounded[rt]);
        if (g == 0) {
          sums[w][rt * 16 + n][0] = l == 0.0f ? -INFINITY : rounded == 0.0f ? m_run[rt] : m_run[rt] + __builtin_amdgcn_logf(l / rounded);
          sums[w][rt * 16 + n][1] = rounded == 0.0f ? l : rounded;
        }
        if (!early | (rt * 16 + n < Lds::EARLY_ROWS)) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int dt = 0; dt < DT; dt += 4)
              *reinterpret_cast<f32x4*>(result + (rt * 16 + n) * (D + 4) + (4 * g + e) * DT + dt) =
                  f32x4{o[rt][dt][e], o[rt][dt + 1][e], o[rt][dt + 2][e], o[rt][dt + 3][e]};
        }
      }
    }
    if (more) {
      PagedArgs& p = fresh_kernel_args<PagedParams>();
      const int at0 = u.request.n_keys - u.request.n_tok, last_row = u.request.n_tok * p.group - 1;
      all_last = at0 + divide(row0, p.by_group);
      all_first = p.window > 0 ? max(at0 + divide(min(row0 + ROWS - 1, last_row), p.by_group) - p.window + 1, 0) : 0;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const int r = min(row0 + rt * 16 + n, last_row), tok = divide(r, p.by_group), q_head = kv_head * p.group + r - tok * p.group;
        const uint16_t* from = reinterpret_cast<const uint16_t*>(p.q) + (u.request.first_tok + tok) * p.q_token + q_head * p.q_head + g * (D / 4);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) q[rt][ks] = *reinterpret_cast<const u32x4*>(from + 8 * ks);
        last_key[rt] = at0 + tok;
      }
    }
    if (have) phase_barrier();
    wait_loads();  // of pages and rows: no product is to wait for rows that may be under way, and with them for tiles that are
    told();
    const bool issued = more & early & (n_steps > 0) & (have != 0);
    if (issued) issue(0);
    if (have) {
      join_few<DTYPE, D, ROWS, NW, Lds::WAVE, true>(walk, done, slot, n_cut, lds + (early ? Lds::STAGE : 0), sums, done_head, done_row0,
                                              [](PagedArgs& p, int r) { return divide(r, p.by_group); });
      if (!more) return;
      phase_barrier();  // nobody's part of LDS is filled again before all have read it
    }
    for (int i = issued ? 1 : 0; i < min(n_steps, 2); ++i) issue(i);

    const float scale_log2 = fresh_kernel_args<PagedParams>().scale_log2;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      m_run[rt] = kNoMax;
      l_run[rt] = l_rounded[rt] = 0.0f;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[rt][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    bool anchored = false;  // every row has a reference maximum
    for (int step = 0; step < n_steps; ++step) {
      if (step % 32 == 0) {
        lane_key = lane_key_ahead;
        full = full_ahead;
      }
      const int left = n_steps - step;
      if (left > 1) __builtin_amdgcn_s_waitcnt(0x0F70 | LOADS);  // all loads but those of the tile behind it
      else wait_loads();
      asm volatile("" ::: "memory");
      typedef typename Tile::Codes Codes;
      QuantGroup<D> x[2];
      const int stage = (step & 1) * Lds::STAGE;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        x[kt].k = *reinterpret_cast<const Codes*>(k_read + (stage + kt * Lds::GROUP));
        x[kt].v = *reinterpret_cast<const Codes*>(v_read + (stage + kt * Lds::GROUP));
        x[kt].k_exp = *reinterpret_cast<const uint8_t*>(k_exp_read + (stage + kt * Lds::GROUP_EXPS));
        x[kt].v_exp = *reinterpret_cast<const uint32_t*>(v_exp_read + (stage + kt * Lds::GROUP_EXPS));
      }
      const int from = 2 * (step % 32);
      const bool is_full = (full >> from & 3) == 3;
      int tile_key[2] = {0, 0};
      if (!is_full) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) tile_key[kt] = __builtin_amdgcn_readlane(lane_key, from + kt);
      }
      if (left > 2) {
        if ((step + 2) % 32 == 0) {
          ask(step + 2);
          told();
        }
        issue(step + 2);
      }
      f32x4 s[RT][2];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        const float scale = exponent_scale(x[kt].k_exp, 0);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) s[rt][kt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const u32x4 a = eight_of_codes<DTYPE>(x[kt].k[ks], scale);
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) s[rt][kt] = mfma_16x16x32<DTYPE>(a, q[rt][ks], s[rt][kt]);
        }
      }
      if (__builtin_expect(!is_full, 0)) {
        PagedArgs& p = fresh_kernel_args<PagedParams>();
        const KeyGroups groups = u.request.groups(p);
        const int reach = p.window > 0 ? p.window : 0x7fffffff;  // a query sees the keys less than this before its last
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = tile_key[kt] + 4 * g + e;
            if (!((tile_key[kt] != kNoKey) & groups.sees(key))) x[kt].clear_v(e);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
              const bool visible = (key <= last_key[rt]) & ((key < p.n_starting) | (last_key[rt] - key < reach)) & (tile_key[kt] != kNoKey);
              s[rt][kt][e] = visible ? s[rt][kt][e] : -INFINITY;
            }
            __builtin_amdgcn_sched_barrier(0);  // (all conditions at once need more scalar registers than there are)
          }
      }
      u32x4 pb[RT];
      float sum[RT];
      for (bool raise = !anchored;; raise = true) {
        if (__builtin_expect(raise, 0)) {  // the reference to the tile's maximum, what was summed before taken relative to it
          bool without = false, summed = false;
          float alpha[RT];
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            float mx = s[rt][0][0];
#pragma unroll
            for (int e = 1; e < 8; ++e) mx = fmaxf(mx, s[rt][e / 4][e % 4]);
            const float m_new = fmaxf(m_run[rt], rows_max(mx * scale_log2));
            alpha[rt] = fast_exp2(m_run[rt] - m_new);
            m_run[rt] = m_new;
            without |= m_new == kNoMax;
            summed |= l_run[rt] != 0.0f;
          }
          anchored = !__any(without);
          if (__any(summed)) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
              l_run[rt] *= alpha[rt];
              l_rounded[rt] *= alpha[rt];
#pragma unroll
              for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[rt][dt][e] *= alpha[rt];
            }
          }
        }
        bool again = false;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          float y[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = fast_exp2(fmaf(s[rt][e / 4][e % 4], scale_log2, -m_run[rt]));
          sum[rt] = ((y[0] + y[1]) + (y[2] + y[3])) + ((y[4] + y[5]) + (y[6] + y[7]));
          again |= !(sum[rt] < kMaxTileSum);
          // Rounded for the product, to half a step of q's type, summed unrounded.
#pragma unroll
          for (int i = 0; i < 4; ++i) pb[rt][i] = pack2<DTYPE>(y[2 * i], y[2 * i + 1]);
        }
        if (__builtin_expect(raise || !__any(again), 1)) break;
      }
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        l_run[rt] += sum[rt];
#pragma unroll
        for (int i = 0; i < 4; ++i) l_rounded[rt] = add_pair<DTYPE>(pb[rt][i], l_rounded[rt]);
      }
      float scale[2][4];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int j = 0; j < 4; ++j) scale[kt][j] = exponent_scale(x[kt].v_exp, j);
      multiply_v<DTYPE, D, RT>(x, scale, pb, o);
    }
    have = 1;
    done = u;
    done_head = kv_head;
    done_row0 = row0;
    if constexpr (!WHOLE) {
      slot = walk.slot(u);
      n_cut = walk.n_cut(u);
    }
  }
}

// Prompts.  Bound as over a cache of 16 bits by the matrix pipe and the issue of instructions, of which the conversions, once for a workgroup's 128
// rows, make a slot taken in 90 % of the cycles instead of 83 %: two prompts of 2048 with a window of 4096 256 us (1.09 PFLOP/s; over 16 bits 251-263),
// one of 8192 from its start 492 (481).
template <int DTYPE, int D, int RT>
__global__ __launch_bounds__(kRowsThreads, 2) void quantized_rows_kernel(const PagedParams) {
  __shared__ __attribute__((aligned(16))) char lds[RowsLds<D>::BYTES];
  PagedArgs& p = fresh_kernel_args<PagedParams>();
  paged_rows<DTYPE, D, false, true, RT>(p, p.own, blockIdx.x, lds);
}

// ---- host ---------------------------------------------------------------------------

// How a call is laid out, and what of the workspace is whose.
struct QuantPlan {
  bool few = false;    // the kernel of few rows
  bool whole = false;  // a workgroup takes a unit of it; otherwise an equal share of all tiles
  int waves = 4;       // of a workgroup of it
  bool cut = false;    // units may be cut into pieces, by either kernel
  int rows = 16, n_few = 0;  // of a unit, and of a piece's slot; workgroups that may have pieces
  int64_t parts = 1;   // of a row at most, as far as the host knows
  int n_shares = 1;    // of a row's keys, by the kernel of rows
  size_t cuts = 0, slots = 0, shares = 0;  // bytes
  size_t bytes() const { return cuts + slots + shares; }
  QuantPlan& with_slots(const dcp_quantized_attn_args& x) {
    if (cut) {
      cuts = ((size_t)x.n_tokens * x.n_heads_q * sizeof(int2) + 15) / 16 * 16;
      slots = (size_t)n_few * 2 * rows * (x.head_dim + 2) * sizeof(float);
    }
    return *this;
  }
};

// Keys that a request's queries see, of the longest there are.
static int64_t seen_keys(const dcp_quantized_attn_args& x) {
  return x.window > 0 ? std::min<int64_t>(x.max_seqlen_k, (int64_t)x.max_seqlen_q + x.window + x.n_starting) : x.max_seqlen_k;
}

static QuantPlan plan_quantized(const dcp_quantized_attn_args& x) {
  QuantPlan plan;
  const int group = x.n_heads_q / x.n_heads_kv;
  // The kernel of few rows: of requests with up to kQuantFewRows.  Its sums of tiles, the starts of units among them, have to fit 32 bits whatever the lengths are.
  const int64_t own_rows = (int64_t)x.max_seqlen_q * group, all_rows = (int64_t)x.n_tokens * group;
  plan.rows = own_rows <= 16 ? 16 : 32;
  const int64_t most_units = (all_rows + (int64_t)x.batch * (plan.rows - 1)) / plan.rows * x.n_heads_kv;
  plan.few = own_rows <= kQuantFewRows && x.batch <= kFewMaxBatch && (double)most_units * ((double)x.table_width * x.page_size / kFewBN + 2 + kStartTurns) < 2e9;
  if (plan.few) {
    // Whole units where they are short: a unit's chain of tiles, by eight waves where every unit has a CU to itself, against what cutting costs,
    // a second kernel and more starts, which grows with the bytes there are (at 7 TB/s, if all were as long as the longest).  us, whole and cut,
    // 8 kv heads of 128: 1 request of 100 keys 6.0 and 9.0, of 1000 9.1 and 10.4, of 1500 11.1 and 10.4; 16 of 2000 12.7 and 15.6; 32 of 2000
    // 15.5 and 20, of 4000 25 and 30, of up to 4000 19.6 and 19.5; 64 of 500 9.8 and 12.4, of up to 2000 16.5 and 19.3, of up to 4000 28 and 27,
    // of up to 8192 51 and 40; 128 of up to 300 10.5 and 19.4.  Head size 64: 1 of 1000 7.8 and 10.5, of 2000 10.5 and 10.6; windows of 1016 keys
    // of 32 8.4 and 13.7.  32 rows: 4 of 1000 12.4 and 14.7, of 4000 26 and 18; 24 of up to 1000 12.4 and 14.9, of up to 4000 26 and 22.
    const int64_t keys = seen_keys(x), units = std::max<int64_t>(x.batch, all_rows / plan.rows) * x.n_heads_kv;
    plan.waves = units <= device_cu_count() ? 8 : 4;
    const double chain_us = keys * (plan.waves == 8 ? 0.0032 : 0.0045) * (x.head_dim == 128 ? 1.0 : 0.6) * (plan.rows == 16 ? 1.0 : 1.6);
    const double bytes_us = (double)units * keys * x.head_dim * 17 / 16 / 7e6;
    plan.whole = chain_us < (plan.rows == 16 ? 4.5 : 6.5) + std::min(0.45 * bytes_us, 12.0);
    if (!plan.whole) plan.waves = 4;
    // Two workgroups a CU are enough for the memory, of head size 64 (half of the bytes under way) four, of 32 rows three, as many as there are
    // registers for.  us, one, two, three and four: four contexts of 131072 keys 93-96, 96, 96-99, 98; 64 of up to 8192 48, 40, 42, 42; at head
    // size 64 40, 29.5, 29, 28.  32 rows of size 64, two, three and four: 4 tokens of 40 heads of 40 requests of up to 9000 keys 31.1, 31.1, 34.5, of
    // 100 requests 63, 58, 64.
    plan.n_few = plan.whole ? (int)most_units : (x.head_dim == 128 ? 2 : plan.rows == 32 ? 3 : 4) * device_cu_count();
    plan.cut = !plan.whole;
    plan.parts = plan.n_few / units + 2;
    return plan.with_slots(x);
  }
  // The kernel of rows, with tiles of 64 rows where no request has more.  us, of 128 and of 64: 16 requests of 16 tokens behind 4000 keys, 8 kv heads
  // of 128, 46.5 and 39.7, 3 of 300 13.8 and 11.8; 22 of 8 tokens of 40 heads behind up to 9178, head size 64, 39.0 and 31.7.
  plan.rows = own_rows <= 64 ? 64 : kRowsBM;
  const double tiles = (double)((seen_keys(x) + kRowsBN - 1) / kRowsBN);
  if (x.batch <= 64) {
    // find_ranked_tile cuts by the lengths that there are.  That they may be is decided by the longest ones: where the time that cutting takes off
    // them if all are as long is more than what a second kernel and the pieces take, or little less: lengths that differ gain more.  us, whole
    // and cut, 8 kv heads of 128 in tiles of 128 rows, 13 or 30 tokens a request: 3 of 300 keys 13.8 and 16.5, of 700 21.8 and 17.3; 16 of 1000 30
    // and 33, of up to 1000 30 and 23; 32 of 1500 43 and 48, of up to 1500 41 and 27; 48 of 2000 69 and 75, of up to 4000 96 and 63; a prompt of
    // 1024 31 and 41.  (Tiles of 64 rows of size 64 are done faster by four workgroups a CU than by two: 64 requests of 12 tokens behind up to
    // 2000 keys 24.7 and 32.9, 8 of 9 behind up to 26124 32.7 and 35.5.)
    const int64_t units = std::max<int64_t>((all_rows + plan.rows - 1) / plan.rows, x.batch) * x.n_heads_kv;
    const int64_t places = (plan.rows == 64 && x.head_dim == 64 ? 4 : 2) * device_cu_count();
    plan.n_few = (int)(places / x.n_heads_kv * x.n_heads_kv);
    plan.cut = units < places && tiles * (1.0 - (double)units / places) > 10.0;
    plan.parts = std::min<int64_t>(plan.n_few / units + 2, (int64_t)tiles / kMinTilesPerPiece + 1);
  } else {
    plan.n_shares = row_shares(x, x.batch, seen_keys(x), false, plan.rows).n;
    plan.parts = plan.n_shares;
    if (plan.n_shares > 1) plan.shares = (size_t)plan.n_shares * x.n_tokens * x.n_heads_q * (x.head_dim + 2) * sizeof(float);
  }
  return plan.with_slots(x);
}

namespace {

#define DCP_QUANT_KERNEL(kernel, ...)                                                                   \
  (x.dtype == DCP_DTYPE_BF16 ? (x.head_dim == 128 ? kernel<DCP_DTYPE_BF16, 128, ##__VA_ARGS__>          \
                                                  : kernel<DCP_DTYPE_BF16, 64, ##__VA_ARGS__>)          \
                             : (x.head_dim == 128 ? kernel<DCP_DTYPE_FP16, 128, ##__VA_ARGS__>          \
                                                  : kernel<DCP_DTYPE_FP16, 64, ##__VA_ARGS__>))

// What a caller may have wrong, before anything is launched.
int check_quantized(const dcp_quantized_attn_args& x) {
  if (x.dtype != DCP_DTYPE_BF16 && x.dtype != DCP_DTYPE_FP16) return fail(DCP_ERR_UNSUPPORTED, "quantized_attn: dtype %d unsupported (bf16 and fp16 only)", x.dtype);
  if (x.head_dim != 64 && x.head_dim != 128) return fail(DCP_ERR_UNSUPPORTED, "quantized_attn: head_dim %d unsupported (64 or 128)", x.head_dim);
  DCP_REQUIRE(x.n_tokens >= 0 && x.batch >= 0 && x.n_pages >= 0, "quantized_attn: negative size");
  DCP_REQUIRE(x.n_heads_q > 0 && x.n_heads_kv > 0 && x.n_heads_q % x.n_heads_kv == 0, "quantized_attn: n_heads_q %d must be a multiple of n_heads_kv %d",
              x.n_heads_q, x.n_heads_kv);
  DCP_REQUIRE(x.softmax_scale > 0.0f, "quantized_attn: softmax_scale must be positive");
  DCP_REQUIRE(x.window >= 0 && x.n_starting >= 0, "quantized_attn: negative window or number of first tokens");
  DCP_REQUIRE(x.page_size > 0 && x.page_size % kQuantTokens == 0, "quantized_attn: page_size %d must be a positive multiple of 16", x.page_size);
  DCP_REQUIRE(x.table_width > 0 && x.table_stride >= 0, "quantized_attn: empty block table");
  DCP_REQUIRE((int64_t)x.table_width * x.page_size < kNoKey - 64, "quantized_attn: too many keys a request");
  DCP_REQUIRE(x.page_stride % 16 == 0 && x.head_stride % 16 == 0 && x.q_token_stride % 8 == 0 && x.q_head_stride % 8 == 0 && x.out_token_stride % 4 == 0 &&
                  x.out_head_stride % 4 == 0, "quantized_attn: strides of q must be multiples of 8 elements (out: 4), of the cache of 16 bytes");
  DCP_REQUIRE(x.page_stride >= 0 && x.head_stride >= 0 && x.q_token_stride >= 0 && x.q_head_stride >= 0 && x.out_token_stride > 0 && x.out_head_stride > 0,
              "quantized_attn: negative stride");
  DCP_REQUIRE(((reinterpret_cast<uintptr_t>(x.q) | reinterpret_cast<uintptr_t>(x.cache) | reinterpret_cast<uintptr_t>(x.out)) & 15) == 0,
              "quantized_attn: q, the cache and out must be 16-byte aligned");
  DCP_REQUIRE((int64_t)x.n_tokens * x.n_heads_q < ((int64_t)1 << 31) - 256, "quantized_attn: too many queries");
  DCP_REQUIRE(x.cu_seqlens_q != nullptr || x.n_tokens == x.batch, "quantized_attn: without cu_seqlens_q every request has one token, got %d for %d",
              x.n_tokens, x.batch);
  if (x.n_tokens == 0 || x.batch == 0) return DCP_OK;
  DCP_REQUIRE(x.q && x.out && x.lse && x.block_table && x.seq_lens && (x.n_pages == 0 || x.cache), "quantized_attn: null argument");
  DCP_REQUIRE(x.max_seqlen_q > 0 && x.max_seqlen_k > 0, "quantized_attn: the longest lengths must be positive");
  // (every kernel's work items: at most 64 shares of a row tile)
  DCP_REQUIRE(row_tiles(x, x.batch, 64) * x.n_heads_kv < ((int64_t)1 << 31) - (1 << 20), "quantized_attn: too many rows");
  return DCP_OK;
}

int quantized_attn(const dcp_quantized_attn_args& x, void* workspace, size_t workspace_bytes, void* stream) {
  DCP_RECORDED(quantized_attn(x, workspace, workspace_bytes, stream));
  if (const int status = check_quantized(x)) return status;
  if (x.n_tokens == 0 || x.batch == 0) return DCP_OK;
  const QuantPlan plan = plan_quantized(x);
  const size_t needed = plan.bytes();
  DCP_REQUIRE(needed == 0 || (workspace && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0 && workspace_bytes >= needed),
              "quantized_attn: workspace of %zu bytes is missing, not 16-byte aligned or smaller than the %zu needed", workspace_bytes, needed);
  PagedParams p = {};
  p.q = x.q; p.k = x.cache; p.out = x.out; p.lse = x.lse;
  p.cu_seqlens_q = x.cu_seqlens_q;
  p.q_token = x.q_token_stride; p.q_head = x.q_head_stride; p.out_token = x.out_token_stride; p.out_head = x.out_head_stride;
  p.page_stride = x.page_stride; p.head_stride = x.head_stride;
  p.own = {x.block_table, x.seq_lens, nullptr, x.table_stride, x.table_width, x.batch, 0, plan.n_shares, plan.few ? 0 : (int)row_tiles(x, x.batch, plan.rows), plan.few ? 1 : row_group(x, x.batch, plan.rows), plan.cut};
  p.n_pages = x.n_pages; p.page_size = x.page_size;
  p.n_requests = x.batch; p.n_tokens = x.n_tokens;
  p.n_heads_q = x.n_heads_q; p.n_heads_kv = x.n_heads_kv; p.group = x.n_heads_q / x.n_heads_kv;
  p.window = x.window; p.n_starting = x.n_starting;
  p.scale_log2 = x.softmax_scale * kLog2e;
  p.direct = plan.n_shares == 1;
  char* at = reinterpret_cast<char*>(workspace);
  p.cuts = reinterpret_cast<int2*>(at);
  p.slot_out = reinterpret_cast<float*>(at + plan.cuts);
  p.slot_sums = reinterpret_cast<f32x2*>(p.slot_out + (size_t)plan.n_few * 2 * plan.rows * x.head_dim);
  p.partial_out = reinterpret_cast<float*>(at + plan.cuts + plan.slots);
  p.partial_sums = reinterpret_cast<f32x2*>(p.partial_out + (size_t)plan.n_shares * x.n_tokens * x.n_heads_q * x.head_dim);
  p.by_page = Divider::of(x.page_size / kQuantTokens); p.by_group = Divider::of(p.group); p.by_heads = Divider::of(x.n_heads_kv);
  p.few_rows = plan.rows; p.few_whole = plan.whole; p.n_few = plan.n_few;
  const auto launch = [&](auto kernel, const char* name, int64_t n_wg, int threads) {
    if (n_wg * threads >= (int64_t)1 << 32) return fail(DCP_ERR_ARG, "quantized_attn: too many work items");  // (what a launch can have)
    KernelTimer timer(name, stream);
    hipLaunchKernelGGL(kernel, dim3((unsigned)n_wg), dim3(threads), 0, (hipStream_t)stream, p);
    return check_launch(name);
  };
  int status;
  if (!plan.few) {
    const int64_t n_wg = x.batch <= 64 ? std::max<int64_t>((int64_t)p.own.n_tiles * x.n_heads_kv, plan.cut ? plan.n_few : 0)
                                       : row_workgroups(p.own.n_tiles, p.own.xcd_group, x.n_heads_kv, plan.n_shares);
    status = plan.rows == 64 ? launch(DCP_QUANT_KERNEL(quantized_rows_kernel, 1), "quantized_rows_kernel", n_wg, kRowsThreads)
                             : launch(DCP_QUANT_KERNEL(quantized_rows_kernel, 2), "quantized_rows_kernel", n_wg, kRowsThreads);
  } else if (plan.whole && plan.waves == 8)
    status = plan.rows == 16 ? launch(DCP_QUANT_KERNEL(quantized_few_kernel, 1, 8, true), "quantized_few_kernel", p.n_few, 512)
                             : launch(DCP_QUANT_KERNEL(quantized_few_kernel, 2, 8, true), "quantized_few_kernel", p.n_few, 512);
  else if (plan.whole)
    status = plan.rows == 16 ? launch(DCP_QUANT_KERNEL(quantized_few_kernel, 1, 4, true), "quantized_few_kernel", p.n_few, 256)
                             : launch(DCP_QUANT_KERNEL(quantized_few_kernel, 2, 4, true), "quantized_few_kernel", p.n_few, 256);
  else
    status = plan.rows == 16 ? launch(DCP_QUANT_KERNEL(quantized_few_kernel, 1, 4, false), "quantized_few_kernel", p.n_few, 256)
                             : launch(DCP_QUANT_KERNEL(quantized_few_kernel, 2, 4, false), "quantized_few_kernel", p.n_few, 256);
  if (status == DCP_OK && (p.own.by_few || !p.direct))
    status = launch_paged_merge(p, x.dtype, x.head_dim, plan.parts, stream);
  return status;
}

}  // namespace
}  // namespace dcp

using namespace dcp;

extern "C" size_t dcp_quantized_attn_workspace_bytes(const dcp_quantized_attn_args* args) {
  if (args == nullptr || check_quantized(*args) != DCP_OK || args->n_tokens == 0 || args->batch == 0) return 0;
  return plan_quantized(*args).bytes();
}

extern "C" int dcp_quantized_attn(const dcp_quantized_attn_args* args, void* workspace, size_t workspace_bytes, void* stream) {
  DCP_REQUIRE(args != nullptr, "quantized_attn: null argument");
  return quantized_attn(*args, workspace, workspace_bytes, stream);
}
