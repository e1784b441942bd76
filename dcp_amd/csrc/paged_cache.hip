// The tables of a paged K/V cache and the writes through them: what a step of answering needs beside attention.
//
// paged_cache_tables_kernel turns the requests' lengths into the step's tables: pages of the free list appended to the
// requests' rows, and for every new token its position and its slot (page * page_size + offset).  Two sums over the
// requests decide everything, the pages taken and the tokens added before each of them.  Every workgroup takes both for
// itself (8 bytes a request out of the L2) and then serves its share of tokens and pages, so the step needs one launch and
// no workspace.  A launch and three dependent trips to memory bound it up to some 10^5 tokens.
//
// paged_cache_write_kernel moves the new tokens' rows of K and V into the cache.  HBM-bound.
#include <algorithm>
#include <utility>

#include "common.h"
#include "record.h"

namespace dcp {


struct CacheTablesParams {
  const int32_t* cached_lens;
  const int32_t* new_lens;
  int32_t* block_table;
  int64_t table_stride;
  const int32_t* free_pages;
  int64_t* slot_mapping;
  int32_t* positions;
  int32_t* cu_seqlens;
  int32_t* seq_lens;
  int32_t* pages_taken;
  int batch, table_width, n_free, page_size, n_tokens;
};

// What a request's lengths say.  (Lengths below zero count as zero; the sum of two fits 32 bits unsigned.)
struct RequestStep {
  uint32_t cached, total;
  int have, taken;  // pages in its row, pages that it takes
  __device__ __forceinline__ RequestStep(const CacheTablesParams& p, int b) {
    const uint32_t size = (uint32_t)p.page_size;
    cached = (uint32_t)max(p.cached_lens[b], 0);
    total = cached + (uint32_t)max(p.new_lens[b], 0);
    have = (int)min(cached / size + (cached % size != 0), (uint32_t)p.table_width);
    taken = (int)min(total / size + (total % size != 0), (uint32_t)p.table_width) - have;
  }
  __device__ __forceinline__ uint32_t added() const { return total - cached; }
};

// The sums are 64-bit ones: whatever the lengths are, they do not wrap, and the searches below stay inside the batch.
struct StepSums {
  int64_t tokens, pages;
};

template <int THREADS>
__global__ __launch_bounds__(THREADS) void paged_cache_tables_kernel(const CacheTablesParams p) {
  __shared__ StepSums ends[THREADS];  // sums up to and with each thread's requests
  const int tid = threadIdx.x;
  const int per_thread = (p.batch + THREADS - 1) / THREADS;
  const int b0 = min(tid * per_thread, p.batch), b1 = min(b0 + per_thread, p.batch);
  StepSums sum = {0, 0};
  for (int b = b0; b < b1; ++b) {
    const RequestStep r(p, b);
    sum.tokens += r.added();
    sum.pages += r.taken;
  }
  ends[tid] = sum;
  __syncthreads();
  for (int step = 1; step < THREADS; step *= 2) {
    StepSums before = {0, 0};
    if (tid >= step) before = ends[tid - step];
    __syncthreads();
    ends[tid].tokens += before.tokens;
    ends[tid].pages += before.pages;
    __syncthreads();
  }
  const StepSums all = ends[THREADS - 1];
  const int first = blockIdx.x * THREADS + tid, stride = gridDim.x * THREADS;

  // the request that holds the `index`-th of the tokens or pages, and the sums before it
  auto find = [&](int64_t index, auto of, StepSums& before) -> int {
    int lo = 0, hi = THREADS - 1;  // the first thread whose sum passes it
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (of(ends[mid]) > index) hi = mid;
      else lo = mid + 1;
    }
    before = lo > 0 ? ends[lo - 1] : StepSums{0, 0};
    int b = lo * per_thread;
    for (; b < p.batch - 1; ++b) {
      const RequestStep r(p, b);
      const StepSums after = {before.tokens + r.added(), before.pages + r.taken};
      if (of(after) > index) break;
      before = after;
    }
    return b;
  };
  auto free_page = [&](int64_t index) -> int { return index < p.n_free ? p.free_pages[index] : -1; };

  for (int64_t t = first; t < p.n_tokens; t += stride) {
    int64_t slot = -1;
    uint32_t position = 0;
    if (t < all.tokens) {
      StepSums before;
      const int b = find(t, [](const StepSums& s) { return s.tokens; }, before);
      const RequestStep r(p, b);
      position = r.cached + (uint32_t)(t - before.tokens);
      const uint32_t index = position / (uint32_t)p.page_size;
      if (index < (uint32_t)p.table_width) {
        const int page = (int)index < r.have ? p.block_table[b * p.table_stride + index] : free_page(before.pages + (int)index - r.have);
        if (page >= 0) slot = (int64_t)page * p.page_size + position % (uint32_t)p.page_size;
      }
    }
    p.slot_mapping[t] = slot;
    p.positions[t] = (int32_t)position;
  }
  for (int64_t i = first; i < all.pages; i += stride) {
    StepSums before;
    const int b = find(i, [](const StepSums& s) { return s.pages; }, before);
    const RequestStep r(p, b);
    p.block_table[b * p.table_stride + r.have + (i - before.pages)] = free_page(i);
  }
  if (blockIdx.x == 0) {
    int64_t at = tid > 0 ? ends[tid - 1].tokens : 0;
    const int64_t most = 0x7fffffff;
    for (int b = b0; b < b1; ++b) {
      const RequestStep r(p, b);
      p.cu_seqlens[b] = (int32_t)min(at, most);
      at += r.added();
      p.seq_lens[b] = (int32_t)min((int64_t)r.total, most);
    }
    if (tid == 0) {
      p.cu_seqlens[p.batch] = (int32_t)min(all.tokens, most);
      *p.pages_taken = (int32_t)min(all.pages, most);
    }
  }
}

struct CacheWriteParams {
  const char* k;
  const char* v;
  const int64_t* slots;
  char* k_cache;
  char* v_cache;
  int64_t in_token, in_head, page, token, head;  // strides in bytes
  int64_t n_slots;
  int n_tokens, page_size, head_pieces, token_pieces;  // pieces of a head's row; of a token's K and V
  int wg_tokens;
};

// A workgroup takes one token, or as many short ones as give a thread kWriteAtOnce pieces.  Piece: what a lane moves at once, 16 bytes
// wherever addresses and strides allow.  What is read does not depend on the slots, so it comes at the same time as they do, for tokens
// without a slot too.  16384 tokens of 8 heads of 128, 134 MB: 21.6 us, 6.2 TB/s.  First the slots and then four tokens' rows a
// workgroup 30.4; both at once 27.9; one token a workgroup 25.9; its stores past the caches 21.6, its loads past them as well 23.6.
constexpr int kWriteThreads = 256, kWriteAtOnce = 2;
template <typename Piece>
__global__ __launch_bounds__(kWriteThreads) void paged_cache_write_kernel(const CacheWriteParams p) {
  const int64_t t0 = (int64_t)blockIdx.x * p.wg_tokens;
  const int n = (int)min((int64_t)p.wg_tokens, p.n_tokens - t0) * p.token_pieces, half = p.token_pieces / 2;
  for (int i0 = threadIdx.x; i0 < n; i0 += kWriteThreads * kWriteAtOnce) {
    Piece x[kWriteAtOnce];
    int64_t slot[kWriteAtOnce];
    char* into[kWriteAtOnce];
#pragma unroll
    for (int j = 0; j < kWriteAtOnce; ++j) {
      const int i = i0 + j * kWriteThreads, token = i / p.token_pieces, in_token = i - token * p.token_pieces;
      const bool is_v = in_token >= half;
      const int at = is_v ? in_token - half : in_token, head = at / p.head_pieces, piece = at - head * p.head_pieces;
      slot[j] = -1;
      if (i < n) {
        slot[j] = p.slots[t0 + token];
        x[j] = *reinterpret_cast<const Piece*>((is_v ? p.v : p.k) + (t0 + token) * p.in_token + head * p.in_head + (int64_t)piece * sizeof(Piece));
      }
      into[j] = (is_v ? p.v_cache : p.k_cache) + head * p.head + (int64_t)piece * sizeof(Piece);
    }
#pragma unroll
    for (int j = 0; j < kWriteAtOnce; ++j) {
      if ((slot[j] < 0) | (slot[j] >= p.n_slots)) continue;
      const int64_t page = p.n_slots < 0x7fffffff ? (uint32_t)slot[j] / (uint32_t)p.page_size : slot[j] / p.page_size;
      __builtin_nontemporal_store(x[j], reinterpret_cast<Piece*>(into[j] + page * p.page + (slot[j] - page * p.page_size) * p.token));
    }
  }
}

}  // namespace dcp

using namespace dcp;

extern "C" int dcp_paged_cache_tables(const int32_t* cached_lens, const int32_t* new_lens, int32_t* block_table, int64_t table_stride,
                                      const int32_t* free_pages, int64_t* slot_mapping, int32_t* positions, int32_t* cu_seqlens,
                                      int32_t* seq_lens, int32_t* pages_taken, int batch, int table_width, int n_free, int page_size,
                                      int n_tokens, void* stream) {
  DCP_RECORDED(dcp_paged_cache_tables(cached_lens, new_lens, block_table, table_stride, free_pages, slot_mapping, positions,
      cu_seqlens, seq_lens, pages_taken, batch, table_width, n_free, page_size, n_tokens, stream));
  DCP_REQUIRE(batch >= 0 && n_tokens >= 0 && n_free >= 0, "paged_cache_tables: negative size");
  DCP_REQUIRE(page_size > 0, "paged_cache_tables: page_size must be positive, got %d", page_size);
  DCP_REQUIRE(table_width > 0 && table_stride >= table_width, "paged_cache_tables: rows of %d entries every %lld do not make a table",
              table_width, (long long)table_stride);
  DCP_REQUIRE(cu_seqlens && pages_taken && (batch == 0 || (cached_lens && new_lens && block_table && seq_lens)) &&
                  (n_free == 0 || free_pages) && (n_tokens == 0 || (slot_mapping && positions)),
              "paged_cache_tables: null argument");
  // (workgroups read the lengths and the free list while others write: the last step's seq_lens, say, are not both)
  const auto overlap = [](const void* a, int64_t n, const void* b, int64_t m) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return x < y + (uintptr_t)m && y < x + (uintptr_t)n;
  };
  const int64_t n = 4 * (int64_t)batch, tokens = n_tokens;
  const std::pair<const void*, int64_t> read[] = {{cached_lens, n}, {new_lens, n}, {free_pages, 4 * (int64_t)n_free}};
  const std::pair<const void*, int64_t> written[] = {{seq_lens, n}, {cu_seqlens, n + 4}, {pages_taken, 4}, {positions, 4 * tokens}, {slot_mapping, 8 * tokens},
                                                     {block_table, 4 * (std::max<int64_t>(batch - 1, 0) * table_stride + table_width)}};
  for (const auto& w : written)
    for (const auto& r : read)
      DCP_REQUIRE(batch == 0 || r.second == 0 || w.second == 0 || !overlap(w.first, w.second, r.first, r.second), "paged_cache_tables: an input is also written to");
  CacheTablesParams p = {cached_lens, new_lens, block_table, table_stride, free_pages, slot_mapping, positions, cu_seqlens,
                         seq_lens, pages_taken, batch, table_width, n_free, page_size, n_tokens};
  const int64_t most = std::max(n_tokens, 1);
  KernelTimer timer("paged_cache_tables_kernel", stream);
  const auto launch = [&](auto kernel, int threads) {
    const int n_wg = (int)std::min<int64_t>((most + threads - 1) / threads, 2 * device_cu_count());
    hipLaunchKernelGGL(kernel, dim3(n_wg), dim3(threads), 0, (hipStream_t)stream, p);
  };
  // A thread takes the lengths of batch / threads requests one after the other, and as many again for a token or page.
  // us, of 256 and of 1024 threads: 4090 requests 18.5 and 12.2, 1024 7.9 and 8.0.
  if (batch <= 1024) launch(paged_cache_tables_kernel<256>, 256);
  else launch(paged_cache_tables_kernel<1024>, 1024);
  return check_launch("paged_cache_tables_kernel");
}

extern "C" int dcp_paged_cache_write(const void* k, const void* v, const int64_t* slot_mapping, void* k_cache, void* v_cache,
                                     int n_tokens, int n_heads_kv, int head_dim, int elem_size, int64_t token_stride,
                                     int64_t head_stride, int64_t n_pages, int page_size, int64_t cache_page_stride,
                                     int64_t cache_token_stride, int64_t cache_head_stride, void* stream) {
  DCP_RECORDED(dcp_paged_cache_write(k, v, slot_mapping, k_cache, v_cache, n_tokens, n_heads_kv, head_dim, elem_size, token_stride,
      head_stride, n_pages, page_size, cache_page_stride, cache_token_stride, cache_head_stride, stream));
  DCP_REQUIRE(elem_size == 1 || elem_size == 2 || elem_size == 4, "paged_cache_write: unsupported element size %d", elem_size);
  DCP_REQUIRE(n_tokens >= 0 && n_pages >= 0 && n_heads_kv > 0 && head_dim > 0 && page_size > 0, "paged_cache_write: sizes must be positive");
  DCP_REQUIRE(token_stride >= 0 && head_stride >= 0 && cache_page_stride >= 0 && cache_token_stride >= 0 && cache_head_stride >= 0,
              "paged_cache_write: negative stride");
  if (n_tokens == 0 || n_pages == 0) return DCP_OK;
  DCP_REQUIRE(k && v && slot_mapping && k_cache && v_cache, "paged_cache_write: null argument");
  const int64_t size = elem_size, row = head_dim * size;
  CacheWriteParams p = {(const char*)k, (const char*)v, slot_mapping, (char*)k_cache, (char*)v_cache, token_stride * size,
                        head_stride * size, cache_page_stride * size, cache_token_stride * size, cache_head_stride * size,
                        n_pages * page_size, n_tokens, page_size, 0, 0, 0};
  const uint64_t all = (uint64_t)(uintptr_t)k | (uintptr_t)v | (uintptr_t)k_cache | (uintptr_t)v_cache | p.in_token | p.in_head |
                       p.page | p.token | p.head | row;
  const int piece = all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : all % 2 == 0 ? 2 : 1;
  DCP_REQUIRE(2 * (int64_t)n_heads_kv * (row / piece) < ((int64_t)1 << 30), "paged_cache_write: rows too long");
  p.head_pieces = (int)(row / piece);
  p.token_pieces = 2 * n_heads_kv * p.head_pieces;
  p.wg_tokens = std::max(kWriteThreads * kWriteAtOnce / p.token_pieces, 1);
  const int64_t n_wg = ((int64_t)n_tokens + p.wg_tokens - 1) / p.wg_tokens;
  KernelTimer timer("paged_cache_write_kernel", stream);
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)n_wg), dim3(kWriteThreads), 0, (hipStream_t)stream, p); };
  if (piece == 16) launch(paged_cache_write_kernel<u32x4>);
  else if (piece == 4) launch(paged_cache_write_kernel<uint32_t>);
  else if (piece == 2) launch(paged_cache_write_kernel<uint16_t>);
  else launch(paged_cache_write_kernel<uint8_t>);
  return check_launch("paged_cache_write_kernel");
}
