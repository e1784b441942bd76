// Writes into a paged K/V cache held in 4 bits, and its rows taken back to 16 bits (quantized_cache.h has the layout).
//
// Both are bound by HBM where there is enough to do, by a launch and one or two trips to memory where there is not.  A lane has 8
// elements of a token's row, the 16 bytes that it moves of the 16-bit side at once; four lanes are a block, whose largest element
// they find together.
#include <algorithm>

#include "quantized_cache.h"
#include "record.h"

namespace dcp {

struct QuantRowsParams {
  char* k;  // rows in 16 bits, read or written
  char* v;
  const int64_t* slots;
  char* cache;
  int64_t token, head;             // strides of the rows in bytes
  int64_t page_stride, head_stride;  // of the cache in bytes
  int64_t n_slots;
  int n_tokens, page_size, n_heads;
  int token_pieces;  // 8-element pieces of a token's K and V
};

// Where a token's 17 D bytes begin, and its number among the 16.
template <int D>
__device__ __forceinline__ char* tile_of_slot(const QuantRowsParams& p, int64_t slot, int head, int& j) {
  const int64_t page = p.n_slots < 0x7fffffff ? (uint32_t)slot / (uint32_t)p.page_size : slot / p.page_size;
  const int offset = (int)(slot - page * p.page_size);
  j = offset % kQuantTokens;
  return p.cache + page * p.page_stride + head * p.head_stride + (int64_t)(offset / kQuantTokens) * QuantTile<D>::BYTES;
}

constexpr int kQuantThreads = 256;

template <int DTYPE, int D>
__global__ __launch_bounds__(kQuantThreads) void quantized_write_kernel(const QuantRowsParams p) {
  typedef QuantTile<D> Tile;
  constexpr int ROW = D / 8;  // pieces of a row
  const int64_t i = (int64_t)blockIdx.x * kQuantThreads + threadIdx.x;
  const int64_t token = i / p.token_pieces;
  if (token >= p.n_tokens) return;  // (a block's four lanes are of one token)
  const int in_token = (int)(i - token * p.token_pieces), half = p.token_pieces / 2;
  const bool is_v = in_token >= half;
  const int at = is_v ? in_token - half : in_token, head = at / ROW, piece = at % ROW;
  const u32x4 x = *reinterpret_cast<const u32x4*>((is_v ? p.v : p.k) + token * p.token + head * p.head + piece * 16);
  const int64_t slot = p.slots[token];
  float f[8];
  uint32_t top = 0;  // bits of the largest size: as whole numbers sizes are in their own order, and what is no number is above them
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    f[e] = Elem<DTYPE>::load((uint16_t)(x[e / 2] >> (16 * (e % 2))));
    top = max(top, __float_as_uint(f[e]) & 0x7fffffffu);
  }
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xf, 0xf, true));  // quad_perm 1 0 3 2
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xf, 0xf, true));  // quad_perm 2 3 0 1
  if ((slot < 0) | (slot >= p.n_slots)) return;
  // e + 127, the smallest with top <= 7 2^e: two less than top's own exponent, one more where its mantissa is past 1.75.  (Below the
  // type's normal numbers 0, which holds all of them.)
  const uint32_t byte = top >= 0x7f800000u ? 255u : (uint32_t)max((int)(top + 0x1fffffu >> 23) - 2, 0);
  const float scale = __uint_as_float(byte << 23);
  // The conversion takes the nearest, ties to the even code, and 6 for what is past 5.  Where a block has the type's largest number 4 2^e is
  // past the type's end: sizes past 3 2^e are 3 2^e there.
  constexpr uint32_t LAST = DTYPE == DCP_DTYPE_BF16 ? 126 + 127 : 14 + 127;
  if (byte == LAST) {
    const float most = 3.0f * scale;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = fminf(fmaxf(f[e], -most), most);
  }
  uint32_t codes = 0;
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[0], f[1], scale, 0);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[2], f[3], scale, 1);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[4], f[5], scale, 2);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[6], f[7], scale, 3);
  int j;
  char* tile = tile_of_slot<D>(p, slot, head, j);
  if (!is_v) {
    *reinterpret_cast<uint32_t*>(tile + j * (D / 2) + piece * 4) = codes;
    if (piece % 4 == 0) tile[Tile::K_EXP + j * Tile::BLOCKS + piece / 4] = (char)byte;
    return;
  }
  char* to = tile + Tile::V + j / 4 * (2 * D) + j % 4 * Tile::V_PIECE;  // sixteenth n: 4 V_PIECE bytes further each
  if constexpr (D == 128) {
    *reinterpret_cast<uint32_t*>(to + piece * 16) = codes;
  } else {
    *reinterpret_cast<uint16_t*>(to + piece * 16) = (uint16_t)codes;
    *reinterpret_cast<uint16_t*>(to + piece * 16 + 8) = (uint16_t)(codes >> 16);
  }
  if (piece % 4 == 0) tile[Tile::V_EXP + (j / 4 * Tile::BLOCKS + piece / 4) * 4 + j % 4] = (char)byte;
}

template <int DTYPE, int D>
__global__ __launch_bounds__(kQuantThreads) void quantized_read_kernel(const QuantRowsParams p) {
  typedef QuantTile<D> Tile;
  constexpr int ROW = D / 8;
  const int64_t i = (int64_t)blockIdx.x * kQuantThreads + threadIdx.x;
  const int64_t token = i / p.token_pieces;
  if (token >= p.n_tokens) return;
  const int in_token = (int)(i - token * p.token_pieces), half = p.token_pieces / 2;
  const bool is_v = in_token >= half;
  const int at = is_v ? in_token - half : in_token, head = at / ROW, piece = at % ROW;
  const int64_t slot = p.slots[token];
  u32x4 x = {0, 0, 0, 0};
  if ((slot >= 0) & (slot < p.n_slots)) {
    int j;
    const char* tile = tile_of_slot<D>(p, slot, head, j);
    uint32_t codes, byte;
    if (!is_v) {
      codes = *reinterpret_cast<const uint32_t*>(tile + j * (D / 2) + piece * 4);
      byte = (uint8_t)tile[Tile::K_EXP + j * Tile::BLOCKS + piece / 4];
    } else {
      const char* from = tile + Tile::V + j / 4 * (2 * D) + j % 4 * Tile::V_PIECE + piece * 16;
      if constexpr (D == 128) codes = *reinterpret_cast<const uint32_t*>(from);
      else codes = *reinterpret_cast<const uint16_t*>(from) | (uint32_t)*reinterpret_cast<const uint16_t*>(from + 8) << 16;
      byte = (uint8_t)tile[Tile::V_EXP + (j / 4 * Tile::BLOCKS + piece / 4) * 4 + j % 4];
    }
    x = eight_of_codes<DTYPE>(codes, exponent_scale(byte, 0));
  }
  *reinterpret_cast<u32x4*>((is_v ? p.v : p.k) + token * p.token + head * p.head + piece * 16) = x;
}

namespace {

// What the two calls have in common: their arguments, checked, as the kernels take them.
int quantized_rows(const char* what, QuantRowsParams& p, const void* k, const void* v, const int64_t* slot_mapping, const void* cache, int n_tokens,
                   int n_heads_kv, int head_dim, int dtype, int64_t token_stride, int64_t head_stride, int64_t n_pages, int page_size,
                   int64_t cache_page_stride, int64_t cache_head_stride) {
  if (dtype != DCP_DTYPE_BF16 && dtype != DCP_DTYPE_FP16) return fail(DCP_ERR_UNSUPPORTED, "%s: dtype %d unsupported (bf16 and fp16 only)", what, dtype);
  if (head_dim != 64 && head_dim != 128) return fail(DCP_ERR_UNSUPPORTED, "%s: head_dim %d unsupported (64 or 128)", what, head_dim);
  DCP_REQUIRE(n_tokens >= 0 && n_pages >= 0 && n_heads_kv > 0, "%s: sizes must be positive", what);
  DCP_REQUIRE(page_size > 0 && page_size % kQuantTokens == 0, "%s: page_size %d must be a positive multiple of 16", what, page_size);
  DCP_REQUIRE(token_stride >= 0 && head_stride >= 0 && token_stride % 8 == 0 && head_stride % 8 == 0,
              "%s: strides of k and v must be multiples of 8 elements, not negative", what);
  DCP_REQUIRE(cache_page_stride >= 0 && cache_head_stride >= 0 && cache_page_stride % 16 == 0 && cache_head_stride % 16 == 0,
              "%s: strides of the cache must be multiples of 16 bytes, not negative", what);
  DCP_REQUIRE(n_heads_kv <= 1 << 20, "%s: too many heads", what);
  DCP_REQUIRE(n_pages <= ((int64_t)1 << 62) / page_size, "%s: too many pages", what);
  if (n_tokens == 0) return DCP_OK;
  DCP_REQUIRE(k && v && slot_mapping && (n_pages == 0 || cache), "%s: null argument", what);
  DCP_REQUIRE((((uintptr_t)k | (uintptr_t)v | (uintptr_t)cache) & 15) == 0, "%s: k, v and the cache must be 16-byte aligned", what);
  p = {(char*)k, (char*)v, slot_mapping, (char*)cache, token_stride * 2, head_stride * 2, cache_page_stride, cache_head_stride, n_pages * page_size,
       n_tokens, page_size, n_heads_kv, 2 * n_heads_kv * (head_dim / 8)};
  const int64_t n_wg = ((int64_t)n_tokens * p.token_pieces + kQuantThreads - 1) / kQuantThreads;
  DCP_REQUIRE(n_wg < (int64_t)1 << 31, "%s: too many rows", what);
  return DCP_OK;
}

template <typename Kernel>
int launch_rows(Kernel kernel, const char* name, const QuantRowsParams& p, void* stream) {
  const int64_t n_wg = ((int64_t)p.n_tokens * p.token_pieces + kQuantThreads - 1) / kQuantThreads;
  KernelTimer timer(name, stream);
  hipLaunchKernelGGL(kernel, dim3((unsigned)n_wg), dim3(kQuantThreads), 0, (hipStream_t)stream, p);
  return check_launch(name);
}

}  // namespace
}  // namespace dcp

using namespace dcp;

#define DCP_QUANT_KERNEL(kernel)                                                                        \
  (dtype == DCP_DTYPE_BF16 ? (head_dim == 128 ? kernel<DCP_DTYPE_BF16, 128> : kernel<DCP_DTYPE_BF16, 64>) \
                           : (head_dim == 128 ? kernel<DCP_DTYPE_FP16, 128> : kernel<DCP_DTYPE_FP16, 64>))

extern "C" int dcp_quantized_cache_write(const void* k, const void* v, const int64_t* slot_mapping, void* cache, int n_tokens, int n_heads_kv,
                                         int head_dim, int dtype, int64_t token_stride, int64_t head_stride, int64_t n_pages, int page_size,
                                         int64_t cache_page_stride, int64_t cache_head_stride, void* stream) {
  DCP_RECORDED(dcp_quantized_cache_write(k, v, slot_mapping, cache, n_tokens, n_heads_kv, head_dim, dtype, token_stride, head_stride, n_pages,
      page_size, cache_page_stride, cache_head_stride, stream));
  QuantRowsParams p;
  if (const int status = quantized_rows("quantized_cache_write", p, k, v, slot_mapping, cache, n_tokens, n_heads_kv, head_dim, dtype, token_stride,
                                        head_stride, n_pages, page_size, cache_page_stride, cache_head_stride))
    return status;
  if (n_tokens == 0 || n_pages == 0) return DCP_OK;
  return launch_rows(DCP_QUANT_KERNEL(quantized_write_kernel), "quantized_write_kernel", p, stream);
}

extern "C" int dcp_quantized_cache_read(const void* cache, const int64_t* slot_mapping, void* k, void* v, int n_tokens, int n_heads_kv, int head_dim,
                                        int dtype, int64_t token_stride, int64_t head_stride, int64_t n_pages, int page_size,
                                        int64_t cache_page_stride, int64_t cache_head_stride, void* stream) {
  DCP_RECORDED(dcp_quantized_cache_read(cache, slot_mapping, k, v, n_tokens, n_heads_kv, head_dim, dtype, token_stride, head_stride, n_pages,
      page_size, cache_page_stride, cache_head_stride, stream));
  QuantRowsParams p;
  if (const int status = quantized_rows("quantized_cache_read", p, k, v, slot_mapping, cache, n_tokens, n_heads_kv, head_dim, dtype, token_stride,
                                        head_stride, n_pages, page_size, cache_page_stride, cache_head_stride))
    return status;
  if (n_tokens == 0) return DCP_OK;
  return launch_rows(DCP_QUANT_KERNEL(quantized_read_kernel), "quantized_read_kernel", p, stream);
}
