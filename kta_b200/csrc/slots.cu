// Block tables and slot maps of a paged KV cache from request lengths, sm_100a.
//
//   held_b = ceil(ctx_b / S), need_b = ceil((ctx_b + new_b) / S)    (S tokens to a block)
//   taken_b = sum_{a < b} (need_a - held_a),  table[b, j] = free[taken_b + j - held_b],
//                                             held_b <= j < need_b
//   token i of request b, at row offset_b + i: position p = ctx_b + i,
//                                              slot = table[b, p / S] * S + p % S
//
// A step's bookkeeping in one launch, so that no length has to travel to the host and back. The
// bytes are few (12 per token written, 8 per request read); what bounds it is the chain launch ->
// lengths -> scan -> table entry -> store: 2.5 us for 8 single tokens, 3.1 us for 256 requests of drafts,
// 4.8 us for 64 prompts (128k tokens, 1.6 MB), in a graph. So every CTA scans all lengths by itself (at most
// 2048, one round of loads, no second kernel and no flag between CTAs) and then writes its own
// part of the tokens and of the new table entries. A token in a block taken by this very call
// reads its id from the free list instead of the table, so no CTA waits for another's stores;
// entries below held_b are read and never written, those from held_b on written and never read.
#include <algorithm>

#include "kta_common.cuh"
#include "kta_host.h"

namespace kta {
namespace slots {

constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int MAX_BATCH = 2048;  // the decode entries' limit; three int tables in shared memory

enum : unsigned int {
  SITE_LENGTH = 0x801,  // a length below zero or past the table
  SITE_TOKENS = 0x802,  // more new tokens than rows
  SITE_BLOCKS = 0x803,  // more new blocks than the free list holds
};

struct Params {
  const int32_t* ctx;    // [B] tokens already in the cache
  const int32_t* fresh;  // [B] new tokens
  int32_t* tables;       // [B, max_blocks], row stride table_stride
  const int32_t* pool;   // [pool_size] free block ids, taken from the front
  int64_t* slots;        // [rows]
  int32_t* positions;    // [rows]
  int32_t* offsets;      // [B + 1]
  int32_t* used;         // [1]
  long long table_stride;
  int batch, max_blocks, pool_size, block, rows;
  int token_ctas;  // the others write table entries
  unsigned int* status;
};

// tokens < 2^31 and block <= 2^20: the sum stays in 32 bits
__device__ __forceinline__ int blocks_of(int tokens, int block) {
  return static_cast<int>((static_cast<unsigned>(tokens) + static_cast<unsigned>(block) - 1u) /
                          static_cast<unsigned>(block));
}

// The last b of [0, n) with first[b] <= x, for ascending first[0..n] with first[0] <= x < first[n];
// requests without an element (first[b] == first[b + 1]) are never it.
__device__ __forceinline__ int owner_of(const int* first, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (first[mid + 1] > x) {
      hi = mid;
    } else {
      lo = mid + 1;
    }
  }
  return lo;
}

__global__ void __launch_bounds__(THREADS) slots_kernel(const Params p) {
  extern __shared__ int tab[];
  int* row0 = tab;                        // [B + 1] first row of each request
  int* blk0 = row0 + p.batch + 1;         // [B + 1] first new block of each request
  int* held_tokens = blk0 + p.batch + 1;  // [B] ctx
  __shared__ long long warp_rows[WARPS], warp_blks[WARPS];
  pdl_launch_dependents();
  pdl_wait();  // the previous grid's writes (this launch's inputs) are visible from here on

  // ---- exclusive scan of (new tokens, new blocks): each thread a run of requests ----
  const int per = (p.batch + THREADS - 1) / THREADS;
  const int b0 = min(threadIdx.x * per, p.batch), b1 = min(b0 + per, p.batch);
  const long long room = static_cast<long long>(p.max_blocks) * p.block;
  long long rows = 0, blks = 0;
  for (int b = b0; b < b1; ++b) {
    const long long c = p.ctx[b], n = p.fresh[b];
    const bool bad = c < 0 || n < 0 || c + n > room;  // counted as a request without new tokens
    if (bad && blockIdx.x == 0) record_status(p.status, KTA_ERR_DEVICE_BOUNDS, SITE_LENGTH);
    held_tokens[b] = bad ? 0 : static_cast<int>(c);
    row0[b] = bad ? 0 : static_cast<int>(n);
    rows += bad ? 0 : n;
    if (!bad) {
      blks += blocks_of(static_cast<int>(c + n), p.block) - blocks_of(static_cast<int>(c), p.block);
    }
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long in_rows = rows, in_blks = blks;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long r = __shfl_up_sync(0xffffffffu, in_rows, o);
    const long long k = __shfl_up_sync(0xffffffffu, in_blks, o);
    if (lane >= o) {
      in_rows += r;
      in_blks += k;
    }
  }
  if (lane == 31) {
    warp_rows[warp] = in_rows;
    warp_blks[warp] = in_blks;
  }
  __syncthreads();
  long long before_rows = in_rows - rows, before_blks = in_blks - blks;
  long long all_rows = 0, all_blks = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) {
      before_rows += warp_rows[w];
      before_blks += warp_blks[w];
    }
    all_rows += warp_rows[w];
    all_blks += warp_blks[w];
  }
  // The tables hold 32 bits: rows past the last and blocks past the pool are cut off there
  // (64-bit sums above, so a cut is seen and recorded, never wrapped).
  const long long max_blk = 0x7fffffffLL;
  for (int b = b0; b < b1; ++b) {
    const int c = held_tokens[b], n = row0[b];
    row0[b] = static_cast<int>(min(before_rows, static_cast<long long>(p.rows)));
    blk0[b] = static_cast<int>(min(before_blks, max_blk));
    before_rows += n;
    before_blks += blocks_of(c + n, p.block) - blocks_of(c, p.block);
  }
  const int total = static_cast<int>(min(all_rows, static_cast<long long>(p.rows)));
  const int total_blks = static_cast<int>(min(all_blks, max_blk));
  if (threadIdx.x == 0) {
    row0[p.batch] = total;
    blk0[p.batch] = total_blks;
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    for (int b = threadIdx.x; b <= p.batch; b += THREADS) p.offsets[b] = row0[b];
    if (threadIdx.x == 0) {
      *p.used = min(total_blks, p.pool_size);
      if (all_rows > p.rows) record_status(p.status, KTA_ERR_DEVICE_BOUNDS, SITE_TOKENS);
      if (all_blks > p.pool_size) record_status(p.status, KTA_ERR_DEVICE_BOUNDS, SITE_BLOCKS);
    }
  }

  if (static_cast<int>(blockIdx.x) < p.token_ctas) {
    // ---- the token map ----
    const int step = p.token_ctas * THREADS;
    for (int row = blockIdx.x * THREADS + threadIdx.x; row < p.rows; row += step) {
      int pos = 0, id = -1;
      if (row < total) {
        const int b = owner_of(row0, p.batch, row);
        const int c = held_tokens[b];
        pos = c + (row - row0[b]);
        const int j = static_cast<int>(static_cast<unsigned>(pos) / static_cast<unsigned>(p.block));
        const int held = blocks_of(c, p.block);
        if (j < held) {
          id = p.tables[b * p.table_stride + j];
        } else {
          const long long k = static_cast<long long>(blk0[b]) + (j - held);
          if (k < p.pool_size) id = p.pool[k];
        }
      }
      p.slots[row] = id < 0 ? -1 : static_cast<long long>(id) * p.block + pos % p.block;
      p.positions[row] = pos;
    }
  } else {
    // ---- the new table entries ----
    const int step = (static_cast<int>(gridDim.x) - p.token_ctas) * THREADS;
    for (long long k = (blockIdx.x - p.token_ctas) * THREADS + threadIdx.x; k < total_blks; k += step) {
      const int b = owner_of(blk0, p.batch, static_cast<int>(k));
      const long long j = blocks_of(held_tokens[b], p.block) + (k - blk0[b]);
      p.tables[b * p.table_stride + j] = k < p.pool_size ? p.pool[k] : -1;
    }
  }
}

int launch(const void* ctx, const void* fresh, void* tables, const void* pool, void* slots_out,
           void* positions, void* offsets, void* used, int64_t B, int64_t max_blocks,
           int64_t table_stride, int64_t pool_size, int64_t block, int64_t rows,
           cudaStream_t stream) {
  if (!ctx || !fresh || !tables || !slots_out || !positions || !offsets || !used) {
    return KTA_ERR_INVALID_ARG;
  }
  if (B <= 0 || max_blocks <= 0 || block <= 0 || rows <= 0 || pool_size < 0) {
    return KTA_ERR_INVALID_ARG;
  }
  if (pool == nullptr && pool_size > 0) return KTA_ERR_INVALID_ARG;
  if (B > 1 && table_stride < max_blocks) return KTA_ERR_INVALID_ARG;
  // positions are 32-bit; row and block counts leave room for a grid stride
  if (B > MAX_BATCH || block > (1 << 20) || max_blocks > (1LL << 31) - 1 ||
      max_blocks * block > (1LL << 31) - 1 || rows > (1LL << 30) || pool_size > (1LL << 31) - 1) {
    return KTA_ERR_UNSUPPORTED;
  }
  for (const void* q : {ctx, fresh, static_cast<const void*>(tables), pool,
                        static_cast<const void*>(positions), static_cast<const void*>(offsets),
                        static_cast<const void*>(used)}) {
    if (reinterpret_cast<uintptr_t>(q) & 3) return KTA_ERR_ALIGN;
  }
  if (reinterpret_cast<uintptr_t>(slots_out) & 7) return KTA_ERR_ALIGN;
  int s = require_sm100();
  if (s != KTA_OK) return s;
  Params prm;
  prm.ctx = static_cast<const int32_t*>(ctx);
  prm.fresh = static_cast<const int32_t*>(fresh);
  prm.tables = static_cast<int32_t*>(tables);
  prm.pool = static_cast<const int32_t*>(pool);
  prm.slots = static_cast<int64_t*>(slots_out);
  prm.positions = static_cast<int32_t*>(positions);
  prm.offsets = static_cast<int32_t*>(offsets);
  prm.used = static_cast<int32_t*>(used);
  prm.table_stride = table_stride;
  prm.batch = static_cast<int>(B);
  prm.max_blocks = static_cast<int>(max_blocks);
  prm.pool_size = static_cast<int>(pool_size);
  prm.block = static_cast<int>(block);
  prm.rows = static_cast<int>(rows);
  prm.status = device_status_ptr();
  // a token or an entry for a thread, at most eight CTAs on each SM
  const auto ctas = [](long long n) {
    return static_cast<int>(std::max(1LL, std::min((n + THREADS - 1) / THREADS, 4LL * current_sm_count())));
  };
  prm.token_ctas = ctas(rows);
  const int grid = prm.token_ctas + ctas(rows / block + B);
  const size_t smem = (3 * static_cast<size_t>(B) + 2) * sizeof(int);
  return launch_ex(slots_kernel, dim3(grid), dim3(THREADS), smem, stream, 1, prm);
}

}  // namespace slots
}  // namespace kta

extern "C" int kta_cache_slots(const void* context_lens, const void* new_lens, void* block_tables,
                               const void* free_blocks, void* slots, void* positions, void* offsets,
                               void* used, int64_t B, int64_t max_blocks, int64_t table_stride,
                               int64_t num_free, int64_t block_size, int64_t max_tokens,
                               void* stream) {
  return kta::slots::launch(context_lens, new_lens, block_tables, free_blocks, slots, positions,
                            offsets, used, B, max_blocks, table_stride, num_free, block_size,
                            max_tokens, static_cast<cudaStream_t>(stream));
}
