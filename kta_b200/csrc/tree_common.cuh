// What the two tree-attention kernels (tree.cu: many query rows, tree_narrow.cu: up to 64) share:
// the work list of a launch, the walk of a CTA over its range, the TMA producers, and the clean-up
// of V tiles that end inside a page. The operator is described in tree.cu.
#pragma once

#include "kta_common.cuh"
#include "kta_host.h"

namespace kta {
namespace tree {

constexpr int BM = 128;               // query rows of a row tile
constexpr int BN = 128;               // keys of a tile
constexpr int NUM_THREADS = 384;      // twelve warps, three to a scheduler
constexpr int MMA_WARP = 8;           // warps 0-7 differ between the kernels
constexpr int K_WARP = 9;             // TMA producers
constexpr int V_WARP = 10;
constexpr int Q_WARP = 11;
constexpr int MAX_DRAFT = 64;         // bits of a row of the tree
constexpr int MAX_GROUP = 16;
constexpr int MAX_BATCH = 1 << 16;
constexpr int MAX_CTAS = 256;         // the workspace is sized for this many
constexpr int NARROW_ROWS = 64;       // up to so many rows of a request: tree_narrow.cu
constexpr float RESCALE_THRESHOLD = 8.0f;  // log2 units: the maximum moves when it grew > 2^8

enum : unsigned int {
  SITE_PROD_KV = 0x901,
  SITE_PROD_Q = 0x902,
  SITE_MMA_Q = 0x903,
  SITE_MMA_K = 0x904,
  SITE_MMA_V = 0x90C,
  SITE_MMA_P = 0x905,
  SITE_MMA_OFREE = 0x906,
  SITE_SM_S = 0x907,
  SITE_SM_V = 0x908,
  SITE_SM_ML = 0x909,
  SITE_SM_O = 0x90A,
  SITE_SM_PV = 0x90B,
  SITE_SMEM = 0x910,     // shared memory not aligned as declared
  SITE_REQUEST = 0x911,  // lengths or offsets out of range
  SITE_BLOCK = 0x912,    // a block id out of range
};

// What the join kernel needs of a unit that starts in a CTA's range and ends in a later one.
struct Desc {
  int count;    // ranges that hold a part of it; 0: none
  int slot;     // the first part's slot
  int next;     // CTA of the second part; the others follow row_tiles apart, each in slot 0
  int row;      // first query token
  int tokens;
  int kvh;
  int pad[2];
};

struct Params {
  const int32_t* ctx;      // [B]
  const int32_t* offsets;  // [B + 1]
  const int64_t* tree;     // [rows] or nullptr: a chain
  const int32_t* tables;   // [B, max_blocks]
  void* out;               // [rows, Hq, D]
  float* lse;              // [rows, Hq]
  const void* v;           // the V cache, for drafted rows that are not finite
  Desc* desc;              // [CTAs]
  float2* part_ml;         // [2 CTAs][row_cap] (maximum, sum), log2 units
  float* part_o;           // [2 CTAs][row_cap][D], not normalised
  long long table_stride;
  int batch, rows, hq, hkv, group, max_new, max_blocks, num_blocks;
  int page_log2;           // tokens of a block
  int box_log2;            // tokens of a TMA box: min(block, 128)
  int tok_tile;            // drafted tokens of a row tile: 128 / group
  int box_tokens;          // tokens of the Q box: min(tok_tile, max_new)
  int row_tiles;           // CTAs that share a range
  int row_cap;             // rows of a partial
  float scale_log2;        // softmax scale * log2(e)
  unsigned int* status;
};

__device__ __forceinline__ void tma_load_5d(const CUtensorMap* map, uint64_t* bar, void* dst, int32_t x,
                                            int32_t y, int32_t z, int32_t w, int32_t v) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(v)
      : "memory");
}

struct Request {
  int row, tokens, ctx, len;  // first row, drafted tokens, cached tokens, both
  bool bad;
};

__device__ __forceinline__ Request request_of(const Params& p, int b) {
  const int a = p.offsets[b], z = p.offsets[b + 1], c = p.ctx[b];
  Request r;
  const long long room = static_cast<long long>(p.max_blocks) << p.page_log2;
  const long long t = static_cast<long long>(z) - a;
  r.bad = a < 0 || t < 0 || z > p.rows || t > p.max_new || c < 0 || c + t > room;
  r.row = a;
  r.tokens = r.bad ? 0 : static_cast<int>(t);
  r.ctx = c;
  r.len = r.bad ? 0 : c + r.tokens;
  return r;
}

// Tiles of keys of a request: none without a query row.
__device__ __forceinline__ int tiles_of(const Request& r) {
  return r.tokens > 0 ? (r.len + BN - 1) / BN : 0;
}

// Row tiles of a request.
__device__ __forceinline__ int row_tiles_of(const Params& p, int tokens) {
  return (tokens + p.tok_tile - 1) / p.tok_tile;
}

// The work list: tile i of KV head h of request b, b-major, each counted once for every row tile
// of its request (the CTAs of a range share those). Range k of n is [total k / n, total (k + 1) / n)
// rounded down to whole tiles; n <= total / row_tiles, so that none is empty.
struct Ranges {
  int total, n;
  __device__ __forceinline__ Ranges(const Params& p, int total_) : total(total_) {
    n = total == 0 ? 0 : max(1, min(static_cast<int>(gridDim.x) / p.row_tiles, total / p.row_tiles));
  }
  __device__ __forceinline__ int start(int k) const {
    return static_cast<int>(static_cast<long long>(total) * k / n);
  }
  // the range of the last tile before position `end`, the end of a unit
  __device__ __forceinline__ int owner_before(int end) const {
    return static_cast<int>((static_cast<long long>(end) * n - 1) / total);
  }
};

// A range's walk over its segments: runs of count() tiles from i0 on of one (request, KV head).
// Few fields, since the softmax warps keep it beside a row of S.
struct Walk {
  int row, tokens, ctx;  // of the request
  int b, kvh, i0;
  int left;              // of the range from here on, in the work list's count
  int turn;              // the CTA of the range's that takes the segment's first row tile

  __device__ __forceinline__ void set(const Request& r) {
    row = r.row;
    tokens = r.tokens;
    ctx = r.ctx;
  }
  __device__ __forceinline__ int len() const { return ctx + tokens; }
  __device__ __forceinline__ int tiles() const { return (len() + BN - 1) / BN; }
  __device__ __forceinline__ int count(const Params& p) const {
    return min(tiles() - i0, left / row_tiles_of(p, tokens));
  }
  __device__ __forceinline__ void next(const Params& p) {
    const int k = row_tiles_of(p, tokens);
    left -= count(p) * k;
    if (left <= 0) return;
    turn = (turn + k) % p.row_tiles;
    i0 = 0;
    if (++kvh == p.hkv) {
      kvh = 0;
      Request r;
      do {  // tiles are left in the range, so a request with some follows
        r = request_of(p, ++b);
      } while (tiles_of(r) == 0);
      set(r);
    }
  }
  // The row tile of the request that falls to CTA `member` of the range's. Requests have between
  // one and row_tiles of them: the CTAs take turns, so that each has its share over some segments.
  __device__ __forceinline__ int row_tile(const Params& p, int member) const {
    const int k = member - turn;
    return k < 0 ? k + p.row_tiles : k;
  }
  // Drafted tokens of row tile rt in the request: 0 where it has fewer.
  __device__ __forceinline__ int rows(const Params& p, int rt) const {
    return max(0, min(tokens - rt * p.tok_tile, p.tok_tile));
  }
  // To the next segment, this one included, in which CTA `member` has rows.
  __device__ __forceinline__ void settle(const Params& p, int member) {
    while (left > 0 && rows(p, row_tile(p, member)) == 0) next(p);
  }
};

// Bits lo .. lo + 31 of a row's view of the keys, lo = first key of the word less ctx: cached
// keys (negative) are all seen, drafted ones by the row's bits.
__device__ __forceinline__ uint32_t view_word(uint64_t bits, int lo) {
  if (lo <= -32) return 0xffffffffu;
  if (lo < 0) return (0xffffffffu >> (32 + lo)) | static_cast<uint32_t>(bits << -lo);
  return lo < 64 ? static_cast<uint32_t>(bits >> lo) : 0u;
}

// 16-bit elements of a word whose exponent is all ones (infinities and NaN), as a mask of them.
template <bool BF16>
__device__ __forceinline__ uint32_t nonfinite(uint32_t w) {
  constexpr uint32_t E = BF16 ? 0x7F80u : 0x7C00u;
  return ((w & E) == E ? 0xffffu : 0u) | ((w >> 16 & E) == E ? 0xffff0000u : 0u);
}

// Rows [from, from + count) of a V tile (shared memory, [8 tokens][half][8][128 B] groups) of which
// [first, valid) are drafted tokens: rows past `valid` become zero (0 * NaN from a page's unwritten
// rows would reach every query row through the matrix product), and so do drafted elements that
// are not finite, whose tokens are recorded in bad[0..1] (token = row + token0) for the epilogue.
// By 128 threads.
template <bool BF16, int D>
__device__ __forceinline__ void clean_v(uint8_t* tile, int from, int count, int first, int valid, int token0,
                                        int tid, unsigned int* bad) {
  constexpr int CHUNKS = D / 8;  // 16-byte pieces of a row
  for (int i = tid + max(first, from) * CHUNKS; i < (from + count) * CHUNKS; i += 128) {
    const int row = i / CHUNKS, ch = i % CHUNKS;
    uint4* at = reinterpret_cast<uint4*>(tile + (row >> 3) * (D / 64 * 1024) + (ch >> 3) * 1024 +
                                         (row & 7) * 128 + (ch & 7) * 16);
    if (row >= valid) {
      *at = make_uint4(0u, 0u, 0u, 0u);
      continue;
    }
    const uint4 u = *at;
    const uint4 n = make_uint4(nonfinite<BF16>(u.x), nonfinite<BF16>(u.y), nonfinite<BF16>(u.z),
                               nonfinite<BF16>(u.w));
    if ((n.x | n.y | n.z | n.w) != 0u) {
      *at = make_uint4(u.x & ~n.x, u.y & ~n.y, u.z & ~n.z, u.w & ~n.w);
      const int token = row + token0;
      atomicOr(bad + (token >> 5), 1u << (token & 31));
    }
  }
}

template <bool BF16>
__device__ __forceinline__ float load16(const void* base, long long i) {
  if constexpr (BF16) {
    return __bfloat162float(static_cast<const __nv_bfloat16*>(base)[i]);
  } else {
    return __half2float(static_cast<const __half*>(base)[i]);
  }
}

// The bits of drafted token t (in its request of `tokens`): the drafted tokens that it sees.
__device__ __forceinline__ uint64_t bits_of(const Params& p, int row, int t, int tokens) {
  const uint64_t bits = p.tree != nullptr ? static_cast<uint64_t>(p.tree[row + t])
                                          : (2ull << t) - 1ull;  // a chain; t = 63: all ones
  return tokens < 64 ? bits & ((1ull << tokens) - 1ull) : bits;
}

// The start of every CTA, after griddepcontrol.wait and with the barriers initialised: finds its
// range's first segment and end, by all threads. plan[0..8] and warp_sum[12] are shared memory;
// rejected requests' rows are zeroed on the way. Synchronises the CTA twice.
template <int D>
__device__ __forceinline__ Walk plan_range(const Params& p, int member, volatile int* plan, int* warp_sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per = (p.batch + NUM_THREADS - 1) / NUM_THREADS;  // requests of a thread
  const int b0 = min(static_cast<int>(threadIdx.x) * per, p.batch), b1 = min(b0 + per, p.batch);
  auto work_of = [&](const Request& r) { return tiles_of(r) * p.hkv * row_tiles_of(p, r.tokens); };
  // a thread's first request is kept: with up to 384 of them nothing is loaded twice
  Request mine_first = {};
  int mine = 0;
  bool bad = false;
  for (int b = b0; b < b1; ++b) {
    const Request r = request_of(p, b);
    if (b == b0) mine_first = r;
    mine += work_of(r);
    bad |= r.bad;
  }
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) warp_sum[warp] = incl;
  __syncthreads();
  int before = incl - mine, total = 0;
#pragma unroll
  for (int w = 0; w < NUM_THREADS / 32; ++w) {
    if (w < warp) before += warp_sum[w];
    total += warp_sum[w];
  }
  const Ranges rg(p, total);
  const int range = blockIdx.x / p.row_tiles;
  const bool busy = range < rg.n;
  if (busy) {
    // the range's two ends, by the threads whose requests they fall into
    const int from = rg.start(range), to = rg.start(range + 1);
    for (int e = 0; e < 2; ++e) {
      const int at = e == 0 ? from : to;
      if (at < before || at >= before + mine) continue;
      int t = before;
      for (int b = b0; b < b1; ++b) {
        const Request r = b == b0 ? mine_first : request_of(p, b);
        const int n = work_of(r);
        if (at >= t + n) {
          t += n;
          continue;
        }
        const int k = row_tiles_of(p, r.tokens), pair = tiles_of(r) * k;
        const int kvh = (at - t) / pair, off = at - t - kvh * pair;
        if (e == 0) {
          plan[0] = b;
          plan[1] = kvh;
          plan[2] = off / k;
          plan[6] = r.row;
          plan[7] = r.tokens;
          plan[8] = r.ctx;
        }
        plan[3 + e] = at - off % k;
        break;
      }
    }
    if (threadIdx.x == 0) {
      if (to == total) plan[4] = total;
      plan[5] = total;
    }
  }
  if (__syncthreads_or(bad ? 1 : 0)) {
    // requests that are out of range: their rows that exist become zero
    for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
      if (!request_of(p, b).bad) continue;
      if (threadIdx.x == 0) record_status(p.status, KTA_ERR_DEVICE_BOUNDS, SITE_REQUEST);
      const long long a = max(p.offsets[b], 0), z = min(p.offsets[b + 1], p.rows);
      const long long words = (z - a) * p.hq * (D / 2);
      uint32_t* o = static_cast<uint32_t*>(p.out) + a * p.hq * (D / 2);
      for (long long i = threadIdx.x; i < words; i += NUM_THREADS) o[i] = 0u;
      for (long long i = threadIdx.x; i < (z - a) * p.hq; i += NUM_THREADS) p.lse[a * p.hq + i] = -INFINITY;
    }
  }
  Walk w;
  w.left = 0;
  if (busy) {
    w.b = plan[0];
    w.kvh = plan[1];
    w.i0 = plan[2];
    w.left = plan[4] - plan[3];
    w.turn = 0;
    w.row = plan[6];
    w.tokens = plan[7];
    w.ctx = plan[8];
    w.settle(p, member);
  }
  return w;
}

// What the join kernel needs, when a unit starts in the segment `w` and goes on behind the range.
__device__ __forceinline__ Desc describe(const Params& p, const Walk& w, int rt, int tokens, int slot,
                                         volatile int* plan) {
  const Ranges r(p, plan[5]);
  const int range = blockIdx.x / p.row_tiles;
  const int end = plan[4] - w.left + w.tiles() * row_tiles_of(p, w.tokens);  // of the unit
  Desc d = {};
  d.count = r.owner_before(end) - range + 1;
  d.slot = slot;
  d.next = (range + 1) * p.row_tiles + rt;  // a range's first segment is row tile = member
  d.row = w.row + rt * p.tok_tile;
  d.tokens = tokens;
  d.kvh = w.kvh;
  return d;
}

// Producer warp of K or V: the range's tiles into a ring of STAGES, lane i loading page i.
template <int D, int STAGES>
__device__ __forceinline__ void produce_kv(const Params& p, Walk w, int member, const CUtensorMap* map,
                                           uint8_t* ring, uint64_t* full, uint64_t* empty,
                                           volatile int* abort_flag) {
  constexpr int GROUP = D / 64 * 1024, TILE = BN / 8 * GROUP;
  const int lane = threadIdx.x & 31;
  const int box = 1 << p.box_log2;
  const int pages = BN >> p.box_log2;          // boxes of a tile
  const int split = p.page_log2 - p.box_log2;  // log2 of boxes in a block
  const int group_box = box / 8;
  uint32_t n = 0;  // tiles so far
  bool ok = true;
  // this lane's block of tile i; only used a tile or two later, so that it stays in flight
  auto block_of = [&](int i) -> int {
    const int at = i * pages + lane;
    if (lane >= pages || at << p.box_log2 >= w.len()) return 0;
    return p.tables[w.b * p.table_stride + (at >> split)];
  };
  for (; w.left > 0 && ok; w.next(p), w.settle(p, member)) {
    const int end = w.i0 + w.count(p);
    int id = block_of(w.i0), id1 = w.i0 + 1 < end ? block_of(w.i0 + 1) : 0;
    for (int i = w.i0; i < end; ++i, ++n) {
      const int id2 = i + 2 < end ? block_of(i + 2) : 0;
      const int st = static_cast<int>(n % STAGES);
      if (!mbar_wait(&empty[st], ((n / STAGES) & 1u) ^ 1u, abort_flag, p.status, SITE_PROD_KV)) {
        ok = false;
        break;
      }
      const int held = min(pages, (w.len() - i * BN + box - 1) >> p.box_log2);
      if (lane == 0) mbar_arrive_expect_tx(&full[st], static_cast<uint32_t>(held * group_box * GROUP));
      __syncwarp();
      if (lane < held) {
        // the block's first (token, head) row; past the tensor, which reads as zeros, for no block
        int first = p.num_blocks * p.hkv << p.page_log2;
        if (id >= 0 && id < p.num_blocks) {
          first = (id * p.hkv << p.page_log2) + w.kvh;
        } else {
          record_status(p.status, KTA_ERR_DEVICE_BOUNDS, SITE_BLOCK);
        }
        tma_load_5d(map, &full[st], ring + st * TILE + lane * group_box * GROUP, 0, 0, 0,
                    ((i * pages + lane) & ((1 << split) - 1)) * group_box, first);
      }
      __syncwarp();
      id = id1;
      id1 = id2;
    }
  }
  if (*abort_flag != 0 && lane == 0) {
    // a role gave up: no copy may be in flight when the block ends (bounded like every wait)
    int none = 0;
    for (uint32_t k = n > STAGES ? n - STAGES : 0; k < n; ++k) {
      mbar_wait(&full[k % STAGES], (k / STAGES) & 1u, &none, p.status, SITE_PROD_KV);
    }
  }
}

// Producer warp of Q: each segment's query rows, [half][rows][128 B], into one of BUFS buffers.
template <int D, int BUFS>
__device__ __forceinline__ void produce_q(const Params& p, Walk w, int member, const CUtensorMap* map,
                                          uint8_t* base, int buf_bytes, int half_bytes, uint64_t* full,
                                          uint64_t* empty, volatile int* abort_flag) {
  if ((threadIdx.x & 31) == 0) {
    uint32_t n = 0;  // segments so far
    for (; w.left > 0; w.next(p), w.settle(p, member), ++n) {
      const uint32_t buf = n % BUFS;
      if (!mbar_wait(&empty[buf], ((n / BUFS) & 1u) ^ 1u, abort_flag, p.status, SITE_PROD_Q)) break;
      mbar_arrive_expect_tx(&full[buf], static_cast<uint32_t>(p.box_tokens * p.group * D * 2));
#pragma unroll
      for (int h = 0; h < D / 64; ++h) {
        tma_load_3d(map, &full[buf], base + buf * buf_bytes + h * half_bytes, h * 64, w.kvh * p.group,
                    w.row + w.row_tile(p, member) * p.tok_tile);
      }
    }
    if (*abort_flag != 0) {
      int none = 0;
      for (uint32_t k = n > BUFS ? n - BUFS : 0; k < n; ++k) {
        mbar_wait(&full[k % BUFS], (k / BUFS) & 1u, &none, p.status, SITE_PROD_Q);
      }
    }
  }
  __syncwarp();
}

// tree_narrow.cu; the tensor maps are encoded by the caller.
template <bool BF16, int D>
int launch_narrow(const Params& p, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                  int grid, cudaStream_t stream);

}  // namespace tree
}  // namespace kta
