// Writes into a paged K/V cache held in 4 bits, and its rows taken back to 16 bits (quantized_cache.h has the layout).
//
// Both are bound by HBM where there is enough to do, by a launch and two trips to memory where there is not.  A lane takes 8 elements
// of a token's row, 16 bytes of the 16-bit side and 4 of the other, for several heads one after the other; the lanes of a wave
// are 4 tokens (8 at head size 64) with all of their pieces, so that of neighbouring slots both K and V are 256 bytes in a row: lanes of one
// token and four heads touched four times that of V (write and read of 16384 tokens of 8 heads of 128 43.5 us, so 28.9).  By themselves these are
// 15.0 and 14.4 us, 5.7 and 5.9 TB/s; the read of 131072 tokens takes 127, 5.4 TB/s (a copy of 2 GiB by torch: 4.95).
#include <algorithm>

#include "quantized_cache.h"
#include "record.h"

namespace dcp {

struct QuantRowsParams {
  char* k;  // rows in 16 bits, read or written
  char* v;
  const int64_t* slots;
  char* cache;
  int64_t k_token, k_head, v_token, v_head;  // strides of the rows in bytes
  int64_t page_stride, head_stride;          // of the cache in bytes
  int64_t n_slots;
  int n_tokens, page_size, n_heads;
  int head_groups;  // of kQuantHeads heads
};

// Which rows a thread has: token `token`, piece `piece` of heads [head, head_end).
constexpr int kQuantThreads = 256, kQuantHeads = 4;
template <int D>
struct QuantRows {
  static constexpr int PIECES = D / 8, TOKENS = kQuantThreads / PIECES;  // of a row, of a workgroup
  int token, piece, head, head_end;
  __device__ __forceinline__ QuantRows(const QuantRowsParams& p) {
    const int wg = blockIdx.x / p.head_groups;
    token = (int)min((int64_t)wg * TOKENS + threadIdx.x / PIECES, (int64_t)0x7fffffff);
    piece = threadIdx.x % PIECES;
    head = (blockIdx.x - wg * p.head_groups) * kQuantHeads;
    head_end = min(head + kQuantHeads, p.n_heads);
  }
};
// Where the 17 D bytes of head 0 begin that hold a slot's token, and its number j among the 16.
template <int D>
__device__ __forceinline__ char* tile_of_slot(const QuantRowsParams& p, int64_t slot, int& j) {
  const int64_t page = p.n_slots < 0x7fffffff ? (uint32_t)slot / (uint32_t)p.page_size : slot / p.page_size;
  const int offset = (int)(slot - page * p.page_size);
  j = offset % kQuantTokens;
  return p.cache + page * p.page_stride + (int64_t)(offset / kQuantTokens) * QuantTile<D>::BYTES;
}

// Eight elements, of which four lanes have a block, in 4 bits; `byte`: the block's exponent.
template <int DTYPE>
__device__ __forceinline__ uint32_t to_codes(u32x4 x, uint32_t& byte) {
  float f[8];
  uint32_t top = 0;  // bits of the largest size: as whole numbers sizes are in their own order, and what is no number is above them
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    f[e] = Elem<DTYPE>::load((uint16_t)(x[e / 2] >> (16 * (e % 2))));
    top = max(top, __float_as_uint(f[e]) & 0x7fffffffu);
  }
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xf, 0xf, true));  // quad_perm 1 0 3 2
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xf, 0xf, true));  // quad_perm 2 3 0 1
  // e + 127, the smallest with top <= 7 2^e: two less than top's own exponent, one more where its mantissa is past 1.75.  (Below the
  // type's normal numbers 0, which holds all of them.)
  byte = top >= 0x7f800000u ? 255u : (uint32_t)max((int)((top + 0x1fffffu) >> 23) - 2, 0);
  const float scale = __uint_as_float(byte << 23);
  // The conversion takes the nearest, ties to the even code, and 6 for what is past 5.  Where a block has the type's largest numbers 4 2^e is
  // past the type's end: sizes past 3 2^e are 3 2^e there.
  constexpr uint32_t LAST = DTYPE == DCP_DTYPE_BF16 ? 126 + 127 : 14 + 127;
  if (__builtin_expect(byte == LAST, 0)) {
    const float most = 3.0f * scale;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = fminf(fmaxf(f[e], -most), most);
  }
  uint32_t codes = 0;
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[0], f[1], scale, 0);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[2], f[3], scale, 1);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[4], f[5], scale, 2);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[6], f[7], scale, 3);
  return codes;
}

template <int DTYPE, int D>
__global__ __launch_bounds__(kQuantThreads) void quantized_write_kernel(const QuantRowsParams p) {
  typedef QuantTile<D> Tile;
  const QuantRows<D> rows(p);
  if (rows.token >= p.n_tokens) return;  // (a block's four lanes are of one token)
  const int64_t slot = p.slots[rows.token];
  const char* k_from = p.k + (rows.token * p.k_token + rows.piece * 16);
  const char* v_from = p.v + (rows.token * p.v_token + rows.piece * 16);
  u32x4 x[kQuantHeads][2];
#pragma unroll
  for (int h = 0; h < kQuantHeads; ++h) {
    if (rows.head + h >= rows.head_end) break;
    x[h][0] = *reinterpret_cast<const u32x4*>(k_from + (rows.head + h) * p.k_head);
    x[h][1] = *reinterpret_cast<const u32x4*>(v_from + (rows.head + h) * p.v_head);
  }
  if ((slot < 0) | (slot >= p.n_slots)) return;
  int j;
  char* tile = tile_of_slot<D>(p, slot, j) + rows.head * p.head_stride;
#pragma unroll
  for (int h = 0; h < kQuantHeads; ++h, tile += p.head_stride) {
    if (rows.head + h >= rows.head_end) break;
    uint32_t k_exp, v_exp;
    const uint32_t k = to_codes<DTYPE>(x[h][0], k_exp), v = to_codes<DTYPE>(x[h][1], v_exp);
    *reinterpret_cast<uint32_t*>(tile + j * (D / 2) + rows.piece * 4) = k;
    char* to = tile + Tile::V + j / 4 * (2 * D) + j % 4 * Tile::V_PIECE + rows.piece * 16;  // a sixteenth of a row: 4 V_PIECE bytes further each
    if constexpr (D == 128) {
      *reinterpret_cast<uint32_t*>(to) = v;
    } else {
      *reinterpret_cast<uint16_t*>(to) = (uint16_t)v;
      *reinterpret_cast<uint16_t*>(to + 8) = (uint16_t)(v >> 16);
    }
    if (rows.piece % 4 == 0) {
      tile[Tile::K_EXP + j * Tile::BLOCKS + rows.piece / 4] = (char)k_exp;
      tile[Tile::V_EXP + (j / 4 * Tile::BLOCKS + rows.piece / 4) * 4 + j % 4] = (char)v_exp;
    }
  }
}

template <int DTYPE, int D>
__global__ __launch_bounds__(kQuantThreads) void quantized_read_kernel(const QuantRowsParams p) {
  typedef QuantTile<D> Tile;
  const QuantRows<D> rows(p);
  if (rows.token >= p.n_tokens) return;
  const int64_t slot = p.slots[rows.token];
  char* k_to = p.k + (rows.token * p.k_token + rows.piece * 16);
  char* v_to = p.v + (rows.token * p.v_token + rows.piece * 16);
  const bool there = (slot >= 0) & (slot < p.n_slots);
  uint32_t codes[kQuantHeads][2], exps[kQuantHeads][2];
  if (there) {
    int j;
    const char* tile = tile_of_slot<D>(p, slot, j) + rows.head * p.head_stride;
#pragma unroll
    for (int h = 0; h < kQuantHeads; ++h, tile += p.head_stride) {
      if (rows.head + h >= rows.head_end) break;
      codes[h][0] = *reinterpret_cast<const uint32_t*>(tile + j * (D / 2) + rows.piece * 4);
      const char* from = tile + Tile::V + j / 4 * (2 * D) + j % 4 * Tile::V_PIECE + rows.piece * 16;
      if constexpr (D == 128) codes[h][1] = *reinterpret_cast<const uint32_t*>(from);
      else codes[h][1] = *reinterpret_cast<const uint16_t*>(from) | (uint32_t)*reinterpret_cast<const uint16_t*>(from + 8) << 16;
      exps[h][0] = (uint8_t)tile[Tile::K_EXP + j * Tile::BLOCKS + rows.piece / 4];
      exps[h][1] = (uint8_t)tile[Tile::V_EXP + (j / 4 * Tile::BLOCKS + rows.piece / 4) * 4 + j % 4];
    }
  }
#pragma unroll
  for (int h = 0; h < kQuantHeads; ++h) {
    if (rows.head + h >= rows.head_end) break;
#pragma unroll
    for (int of = 0; of < 2; ++of) {
      u32x4 x = {0, 0, 0, 0};
      if (there) x = eight_of_codes<DTYPE>(codes[h][of], exponent_scale(exps[h][of], 0));
      __builtin_nontemporal_store(x, reinterpret_cast<u32x4*>(of ? v_to + (rows.head + h) * p.v_head : k_to + (rows.head + h) * p.k_head));
    }
  }
}

namespace {

int64_t row_workgroups(const QuantRowsParams& p, int head_dim) {
  const int64_t tokens = kQuantThreads / (head_dim / 8);  // of a workgroup
  return (p.n_tokens + tokens - 1) / tokens * p.head_groups;
}

// Strides of an axis, in elements; of an axis of one they say nothing.
struct RowStrides {
  int64_t token, head;
  RowStrides of(int n_tokens, int n_heads) const { return {n_tokens == 1 ? 0 : token, n_heads == 1 ? 0 : head}; }
  bool good() const { return token >= 0 && head >= 0 && token % 8 == 0 && head % 8 == 0; }
};

// What the calls have in common: their arguments, checked, as the kernels take them.
int quantized_rows(const char* what, QuantRowsParams& p, const void* k, const void* v, const int64_t* slot_mapping, const void* cache, int n_tokens,
                   int n_heads_kv, int head_dim, int dtype, RowStrides k_strides, RowStrides v_strides, int64_t n_pages, int page_size,
                   int64_t cache_page_stride, int64_t cache_head_stride) {
  if (dtype != DCP_DTYPE_BF16 && dtype != DCP_DTYPE_FP16) return fail(DCP_ERR_UNSUPPORTED, "%s: dtype %d unsupported (bf16 and fp16 only)", what, dtype);
  if (head_dim != 64 && head_dim != 128) return fail(DCP_ERR_UNSUPPORTED, "%s: head_dim %d unsupported (64 or 128)", what, head_dim);
  DCP_REQUIRE(n_tokens >= 0 && n_pages >= 0 && n_heads_kv > 0, "%s: sizes must be positive", what);
  DCP_REQUIRE(page_size > 0 && page_size % kQuantTokens == 0, "%s: page_size %d must be a positive multiple of 16", what, page_size);
  k_strides = k_strides.of(n_tokens, n_heads_kv);
  v_strides = v_strides.of(n_tokens, n_heads_kv);
  DCP_REQUIRE(k_strides.good() && v_strides.good(), "%s: strides of k and v must be multiples of 8 elements, not negative", what);
  DCP_REQUIRE(cache_page_stride >= 0 && cache_head_stride >= 0 && cache_page_stride % 16 == 0 && cache_head_stride % 16 == 0,
              "%s: strides of the cache must be multiples of 16 bytes, not negative", what);
  DCP_REQUIRE(n_heads_kv <= 1 << 20, "%s: too many heads", what);
  DCP_REQUIRE(n_pages <= ((int64_t)1 << 62) / page_size, "%s: too many pages", what);
  if (n_tokens == 0) return DCP_OK;
  DCP_REQUIRE(k && v && slot_mapping && (n_pages == 0 || cache), "%s: null argument", what);
  DCP_REQUIRE((((uintptr_t)k | (uintptr_t)v | (uintptr_t)cache) & 15) == 0, "%s: k, v and the cache must be 16-byte aligned", what);
  p = {(char*)k, (char*)v, slot_mapping, (char*)cache, k_strides.token * 2, k_strides.head * 2, v_strides.token * 2, v_strides.head * 2,
       cache_page_stride, cache_head_stride, n_pages * page_size, n_tokens, page_size, n_heads_kv, (n_heads_kv + kQuantHeads - 1) / kQuantHeads};
  DCP_REQUIRE(row_workgroups(p, head_dim) < (int64_t)1 << 31, "%s: too many rows", what);
  return DCP_OK;
}

template <typename Kernel>
int launch_rows(Kernel kernel, const char* name, const QuantRowsParams& p, int head_dim, void* stream) {
  KernelTimer timer(name, stream);
  hipLaunchKernelGGL(kernel, dim3((unsigned)row_workgroups(p, head_dim)), dim3(kQuantThreads), 0, (hipStream_t)stream, p);
  return check_launch(name);
}

}  // namespace
}  // namespace dcp

using namespace dcp;

#define DCP_QUANT_KERNEL(kernel)                                                                        \
  (dtype == DCP_DTYPE_BF16 ? (head_dim == 128 ? kernel<DCP_DTYPE_BF16, 128> : kernel<DCP_DTYPE_BF16, 64>) \
                           : (head_dim == 128 ? kernel<DCP_DTYPE_FP16, 128> : kernel<DCP_DTYPE_FP16, 64>))

extern "C" int dcp_quantized_cache_write_strided(const void* k, const void* v, const int64_t* slot_mapping, void* cache, int n_tokens, int n_heads_kv,
                                                 int head_dim, int dtype, int64_t k_token_stride, int64_t k_head_stride, int64_t v_token_stride,
                                                 int64_t v_head_stride, int64_t n_pages, int page_size, int64_t cache_page_stride,
                                                 int64_t cache_head_stride, void* stream) {
  DCP_RECORDED(dcp_quantized_cache_write_strided(k, v, slot_mapping, cache, n_tokens, n_heads_kv, head_dim, dtype, k_token_stride, k_head_stride,
      v_token_stride, v_head_stride, n_pages, page_size, cache_page_stride, cache_head_stride, stream));
  QuantRowsParams p;
  if (const int status = quantized_rows("quantized_cache_write", p, k, v, slot_mapping, cache, n_tokens, n_heads_kv, head_dim, dtype,
                                        {k_token_stride, k_head_stride}, {v_token_stride, v_head_stride}, n_pages, page_size, cache_page_stride,
                                        cache_head_stride))
    return status;
  if (n_tokens == 0 || n_pages == 0) return DCP_OK;
  return launch_rows(DCP_QUANT_KERNEL(quantized_write_kernel), "quantized_write_kernel", p, head_dim, stream);
}

extern "C" int dcp_quantized_cache_write(const void* k, const void* v, const int64_t* slot_mapping, void* cache, int n_tokens, int n_heads_kv,
                                         int head_dim, int dtype, int64_t token_stride, int64_t head_stride, int64_t n_pages, int page_size,
                                         int64_t cache_page_stride, int64_t cache_head_stride, void* stream) {
  return dcp_quantized_cache_write_strided(k, v, slot_mapping, cache, n_tokens, n_heads_kv, head_dim, dtype, token_stride, head_stride, token_stride,
                                           head_stride, n_pages, page_size, cache_page_stride, cache_head_stride, stream);
}

extern "C" int dcp_quantized_cache_read_strided(const void* cache, const int64_t* slot_mapping, void* k, void* v, int n_tokens, int n_heads_kv,
                                                int head_dim, int dtype, int64_t k_token_stride, int64_t k_head_stride, int64_t v_token_stride,
                                                int64_t v_head_stride, int64_t n_pages, int page_size, int64_t cache_page_stride,
                                                int64_t cache_head_stride, void* stream) {
  DCP_RECORDED(dcp_quantized_cache_read_strided(cache, slot_mapping, k, v, n_tokens, n_heads_kv, head_dim, dtype, k_token_stride, k_head_stride,
      v_token_stride, v_head_stride, n_pages, page_size, cache_page_stride, cache_head_stride, stream));
  QuantRowsParams p;
  if (const int status = quantized_rows("quantized_cache_read", p, k, v, slot_mapping, cache, n_tokens, n_heads_kv, head_dim, dtype,
                                        {k_token_stride, k_head_stride}, {v_token_stride, v_head_stride}, n_pages, page_size, cache_page_stride,
                                        cache_head_stride))
    return status;
  if (n_tokens == 0) return DCP_OK;
  return launch_rows(DCP_QUANT_KERNEL(quantized_read_kernel), "quantized_read_kernel", p, head_dim, stream);
}

extern "C" int dcp_quantized_cache_read(const void* cache, const int64_t* slot_mapping, void* k, void* v, int n_tokens, int n_heads_kv, int head_dim,
                                        int dtype, int64_t token_stride, int64_t head_stride, int64_t n_pages, int page_size,
                                        int64_t cache_page_stride, int64_t cache_head_stride, void* stream) {
  return dcp_quantized_cache_read_strided(cache, slot_mapping, k, v, n_tokens, n_heads_kv, head_dim, dtype, token_stride, head_stride, token_stride,
                                          head_stride, n_pages, page_size, cache_page_stride, cache_head_stride, stream);
}
