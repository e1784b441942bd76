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
// (The device multiplies 4 bits by 8 bits as they are, q in two or three parts.  It adds the 128 products of a step to no
// more than 14 bits of the largest: scores were off by 5e-6 of the sum of their products' sizes, here by 1e-7.)
#include <algorithm>

#include "paged_rows.h"
#include "record.h"

namespace dcp {

template <int D, int RT, int NW>
struct QuantFewLds {
  static constexpr int ROWS = 16 * RT, WAVE = ROWS * (D + 4) * 4;  // a wave's result: float [row][D + 4]
  static constexpr int SUMS = NW * WAVE;                           // float [wave][row][2]
  static constexpr int CHUNKS = SUMS + NW * ROWS * 2 * 4;          // int [batch / 64]
  static constexpr int BYTES = CHUNKS + kFewMaxBatch / 64 * 4;
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
// share of the keys is done; work is cut as over a cache of 16 bits (FewWalk).
template <int DTYPE, int D, int RT, int NW>
__global__ __launch_bounds__(NW * 64, RT == 1 ? 3 : 2) void quantized_few_kernel(const PagedParams) {
  typedef QuantFewLds<D, RT, NW> Lds;
  typedef QuantTile<D> Tile;
  __shared__ __attribute__((aligned(16))) char lds[Lds::BYTES];
  constexpr int KS = D / 32, DT = D / 16, ROWS = Lds::ROWS;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  float(*sums)[ROWS][2] = reinterpret_cast<float(*)[ROWS][2]>(lds + Lds::SUMS);

  FewWalk<ROWS, NW> walk(blockIdx.x, reinterpret_cast<int*>(lds + Lds::CHUNKS));
  FewUnit u;
  while (walk.next(u)) {
    PagedArgs& p = fresh_kernel_args<PagedParams>();
    const FewRequest& request = u.request;
    const int kv_head = u.unit % p.n_heads_kv, row0 = u.unit / p.n_heads_kv * ROWS, n_rows = request.n_tok * p.group;
    const KeyGroups groups = request.groups(p);
    const int n_groups = request.n_keys > 0 ? groups.count() : 0;

    // ---- where the wave's next 32 tiles are: lane 2 i + j holds the 16-key group j of the i-th of them ------------
    int64_t lane_off = 0;
    int lane_key = kNoKey;
    auto look_up = [&](int step) {
      PagedArgs& p = fresh_kernel_args<PagedParams>();
      const int group = 2 * (u.t_begin + w + NW * (step + (lane >> 1))) + (lane & 1);
      lane_off = 0;
      lane_key = kNoKey;
      if (group < n_groups && group < 2 * u.t_end) {
        const int key = groups.at(group) * 16, entry = key / p.page_size;
        const int page = p.own.block_table[u.b * p.own.table_stride + entry];
        if ((unsigned)page < (unsigned)p.n_pages) {
          lane_key = key;
          lane_off = page * p.page_stride + (int64_t)((key - entry * p.page_size) / 16) * Tile::BYTES;
        }
      }
    };
    const char* head = reinterpret_cast<const char*>(p.k) + kv_head * p.head_stride;
    const int n_steps = n_groups > 0 && u.t_begin + w < u.t_end ? (u.t_end - u.t_begin - w + NW - 1) / NW : 0;
    QuantGroup<D> next[2];
    int next_key[2];
    auto load = [&](int step) {
      if (step % 32 == 0) look_up(step);
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        const int from = 2 * (step % 32) + kt;
        const char* at = head + lane_value(lane_off, from);
        next_key[kt] = __builtin_amdgcn_readlane(lane_key, from);
        typedef typename Tile::Codes Codes;
        next[kt].k = __builtin_nontemporal_load(reinterpret_cast<const Codes*>(at + Tile::k_of(lane)));
        next[kt].k_exp = *reinterpret_cast<const uint8_t*>(at + Tile::k_exp_of(lane));
        next[kt].v = __builtin_nontemporal_load(reinterpret_cast<const Codes*>(at + Tile::v_of(lane)));
        next[kt].v_exp = *reinterpret_cast<const uint32_t*>(at + Tile::v_exp_of(lane));
      }
    };
    if (n_steps > 0) load(0);

    // ---- this lane's rows --------------------------------------------------------------
    int last_key[RT], first_key[RT];
    int w_last = 0x7fffffff, w_first = 0;
    u32x4 q[RT][KS];  // slots of product ks: D / 4 elements from g D / 4 on, eight at a time
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int r = row0 + rt * 16 + n, tok = r / p.group, q_head = kv_head * p.group + r % p.group;
      const bool live = r < n_rows;
      const uint16_t* from = reinterpret_cast<const uint16_t*>(p.q) + (request.first_tok + tok) * p.q_token + q_head * p.q_head + g * (D / 4);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        q[rt][ks] = u32x4{0, 0, 0, 0};
        if (live) q[rt][ks] = *reinterpret_cast<const u32x4*>(from + 8 * ks);
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

    for (int step = 0; step < n_steps; ++step) {
      QuantGroup<D> x[2] = {next[0], next[1]};
      const int tile_key[2] = {next_key[0], next_key[1]};
      if (step + 1 < n_steps) load(step + 1);
      bool whole = true, full = true;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        whole = whole & groups.sees_all_of_16(tile_key[kt]);
        full = full & (tile_key[kt] + 15 <= w_last) & ((tile_key[kt] >= w_first) | (tile_key[kt] + 15 < p.n_starting));
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
      if (!(whole & full)) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = tile_key[kt] + 4 * g + e;
            if (!((tile_key[kt] != kNoKey) & groups.sees(key))) x[kt].clear_v(e);
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
          float y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            y[e] = fast_exp2(fmaf(s[rt][kt][e], p.scale_log2, -m_use));
            l_run[rt] += y[e];
          }
          // Rounded for the product, to half a step of q's type, summed unrounded: the largest weight is 1, which is exact.
          pb[rt][2 * kt] = pack2<DTYPE>(y[0], y[1]);
          pb[rt][2 * kt + 1] = pack2<DTYPE>(y[2], y[3]);
        }
      }
      float scale[2][4];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int j = 0; j < 4; ++j) scale[kt][j] = exponent_scale(x[kt].v_exp, j);
      multiply_v<DTYPE, D, RT>(x, scale, pb, o);
    }

    // ---- the waves' results joined: element (4 g + e) D / 16 + dt is o[dt][e] --------------------------------
    float* mine = reinterpret_cast<float*>(lds + w * Lds::WAVE);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const float l = rows_sum(l_run[rt]);
      if (g == 0) {
        sums[w][rt * 16 + n][0] = m_run[rt];
        sums[w][rt * 16 + n][1] = l;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int dt = 0; dt < DT; dt += 4)
          *reinterpret_cast<f32x4*>(mine + (rt * 16 + n) * (D + 4) + (4 * g + e) * DT + dt) =
              f32x4{o[rt][dt][e], o[rt][dt + 1][e], o[rt][dt + 2][e], o[rt][dt + 3][e]};
    }
    __syncthreads();
    join_few<DTYPE, D, ROWS, NW, Lds::WAVE>(walk, u, lds, sums, kv_head, row0);
    __syncthreads();  // nobody's part of LDS is filled again before all have read it
  }
}

template <int DTYPE, int D>
__global__ __launch_bounds__(kRowsThreads, 2) void quantized_rows_kernel(const PagedParams) {
  __shared__ __attribute__((aligned(16))) char lds[RowsLds<D>::BYTES];
  PagedArgs& p = fresh_kernel_args<PagedParams>();
  paged_rows<DTYPE, D, false, true>(p, p.own, blockIdx.x, lds);
}

// ---- host ---------------------------------------------------------------------------

// How a call is laid out, and what of the workspace is whose.
struct QuantPlan {
  bool few = false;    // the kernel of few rows
  bool whole = false;  // a workgroup takes a unit of it; otherwise an equal share of all tiles
  int rows = 16, n_few = 0;
  int n_shares = 1;    // of a row's keys, by the kernel of rows
  size_t cuts = 0, slots = 0, shares = 0;  // bytes
  size_t bytes() const { return cuts + slots + shares; }
};

// Keys that a request's queries see, of the longest there are.
static int64_t seen_keys(const dcp_quantized_attn_args& x) {
  return x.window > 0 ? std::min<int64_t>(x.max_seqlen_k, (int64_t)x.max_seqlen_q + x.window + x.n_starting) : x.max_seqlen_k;
}

static QuantPlan plan_quantized(const dcp_quantized_attn_args& x) {
  QuantPlan plan;
  const int group = x.n_heads_q / x.n_heads_kv;
  // The kernel of few rows: of requests with up to 32.  Its sums of tiles have to fit 32 bits whatever the lengths are.
  const int64_t own_rows = (int64_t)x.max_seqlen_q * group, all_rows = (int64_t)x.n_tokens * group;
  plan.rows = own_rows <= 16 ? 16 : 32;
  const int64_t most_units = (all_rows + (int64_t)x.batch * (plan.rows - 1)) / plan.rows * x.n_heads_kv;
  plan.few = own_rows <= 32 && x.batch <= kFewMaxBatch && (double)most_units * ((double)x.table_width * x.page_size / kFewBN + 2) < 2e9;
  if (plan.few) {
    plan.n_few = (plan.rows == 16 ? 3 : 2) * device_cu_count();
    plan.cuts = ((size_t)x.n_tokens * x.n_heads_q * sizeof(int2) + 15) / 16 * 16;
    plan.slots = (size_t)plan.n_few * 2 * plan.rows * (x.head_dim + 2) * sizeof(float);
  } else {
    plan.n_shares = row_shares(x, x.batch, seen_keys(x), false).n;
    if (plan.n_shares > 1) plan.shares = (size_t)plan.n_shares * x.n_tokens * x.n_heads_q * (x.head_dim + 2) * sizeof(float);
  }
  return plan;
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
  DCP_REQUIRE(row_tiles(x, x.batch) * x.n_heads_kv < ((int64_t)1 << 31) - (1 << 20), "quantized_attn: too many rows");
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
  p.own = {x.block_table, x.seq_lens, nullptr, x.table_stride, x.table_width, x.batch, 0, plan.n_shares, (int)row_tiles(x, x.batch), row_group(x, x.batch), plan.few && !plan.whole};
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
  p.few_rows = plan.rows; p.few_whole = plan.whole; p.n_few = plan.n_few;
  const auto launch = [&](auto kernel, const char* name, int64_t n_wg) {
    if (n_wg >= (int64_t)1 << 31) return fail(DCP_ERR_ARG, "quantized_attn: too many work items");
    KernelTimer timer(name, stream);
    hipLaunchKernelGGL(kernel, dim3((unsigned)n_wg), dim3(256), 0, (hipStream_t)stream, p);
    return check_launch(name);
  };
  int status;
  if (!plan.few)
    status = launch(DCP_QUANT_KERNEL(quantized_rows_kernel), "quantized_rows_kernel", row_workgroups(p.own.n_tiles, p.own.xcd_group, x.n_heads_kv, plan.n_shares));
  else if (plan.rows == 16) status = launch(DCP_QUANT_KERNEL(quantized_few_kernel, 1, 4), "quantized_few_kernel", p.n_few);
  else status = launch(DCP_QUANT_KERNEL(quantized_few_kernel, 2, 4), "quantized_few_kernel", p.n_few);
  if (status == DCP_OK && (p.own.by_few || !p.direct)) {
    const int64_t units = std::max<int64_t>((int64_t)x.batch * x.n_heads_kv, 1);
    status = launch_paged_merge(p, x.dtype, x.head_dim, plan.few ? plan.n_few / units + 2 : plan.n_shares, stream);
  }
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
