// What the two tree-attention kernels (tree.cu: many query rows, tree_narrow.cu: up to 32) share:
// the work list of a launch, the walk of a CTA over its share, the TMA producers, and the clean-up
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
constexpr int MAX_BATCH = 2048;       // the decode entries' limit
constexpr int MAX_CTAS = 160;         // the workspace is sized for this many
constexpr int NARROW_ROWS = 32;       // up to so many rows of a request: tree_narrow.cu
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
  SITE_SM_TURN = 0x90D,
  SITE_SMEM = 0x910,     // shared memory not aligned as declared
  SITE_REQUEST = 0x911,  // lengths or offsets out of range
  SITE_BLOCK = 0x912,    // a block id out of range
};

// mbar_wait() with all behind the first try in one place: the roles' code, inlined many times, has to
// pass through the SM's instruction caches for every segment (148 single tokens over 100 keys 28.4 us
// with it inlined, 25.0 so).
static __device__ __noinline__ bool wait_on(uint64_t* bar, uint32_t parity, volatile int* abort,
                                     unsigned int* status, unsigned int site) {
  return mbar_wait(bar, parity, abort, status, site);
}
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, volatile int* abort,
                                         unsigned int* status, unsigned int site) {
  return mbar_try_wait(smem_u32(bar), parity) || wait_on(bar, parity, abort, status, site);
}

// What the join kernel needs of a unit (a row tile's tiles of one (request, KV head)) that starts in a
// share and ends in a later one.
struct Desc {
  int span;    // shares that hold a part of it; 0: none
  int row;     // first query token
  int tokens;
  int kvh;
};

struct Params {
  const int32_t* ctx;      // [B]
  const int32_t* offsets;  // [B + 1]
  const int64_t* tree;     // [rows] or nullptr: a chain
  const int32_t* tables;   // [B, max_blocks]
  void* out;               // [rows, Hq, D]
  float* lse;              // [rows, Hq]
  const void* v;           // the V cache, for drafted rows that are not finite
  Desc* desc;              // [MAX_CTAS] by share and row tile
  float2* part_ml;         // [2 MAX_CTAS][row_cap] (maximum, sum), log2 units
  float* part_o;           // [2 MAX_CTAS][row_cap][D] or [D / 4][row_cap][4], not normalised
  long long table_stride;
  int batch, rows, hq, hkv, group, max_new, max_blocks, num_blocks;
  int page_log2;           // tokens of a block
  int box_log2;            // tokens of a TMA box: min(block, 128)
  int tok_tile;            // drafted tokens of a row tile: 128 / group
  int box_tokens;          // tokens of the Q box: min(tok_tile, max_new)
  int row_tiles;           // members of a share
  int groups;              // shares: one for as many CTAs
  int row_cap;             // rows of a partial
  float scale_log2;        // softmax scale * log2(e)
  unsigned int* status;
};

__device__ __forceinline__ void tma_load_5d_hint(const CUtensorMap* map, uint64_t* bar, void* dst, int32_t x,
                                                 int32_t y, int32_t z, int32_t w, int32_t v,
                                                 uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4, %5, %6, %7}], [%2], %8;" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(v),
      "l"(policy)
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

// The work list: the 128-key tiles of every (request, KV head), b-major, each counted once for every
// row tile of its request, in equal shares for `row_tiles` CTAs each (a share's members). A segment's
// start and end cost a CTA about as much as SWITCH tiles (with equal numbers of tiles, shares of 3
// segments had their keys at 183 us and shares of 10 at 215), so every unit counts so many more, ahead
// of its first tile: 64 requests of 8 tokens, 8 KV heads, over 1024 to 8192 keys 196.4 us, 198.4 with
// equal numbers of tiles; 64 single tokens over 64 to 512 keys 25.6 and 26.6; 16 trees of 33 to 64 tokens
// of 8 heads over 500 to 2000 keys 66 and 74; but 32 single tokens over 256 to 1024 keys 24.3 and 23.3.
// Not where a share has less than a tile (one request of 4 tokens over 1024 keys 15.0 us, 16.3 with
// them counted, when a segment's start cost more than it does now).
//
// Shares that are taken as they are finished (the first 78 to 88 % to each CTA, the rest in one to
// three rounds from a counter) measured 218 to 246 us where these take 202: what a cut unit costs is
// more than the even end gives.
constexpr int SWITCH = 3;

struct Shares {
  int total, n, extra;  // extra: what a unit counts beyond its tiles
  int length, longer;   // of a share, before it is rounded down to tiles; the first `longer` have one more
  __device__ __forceinline__ Shares(const Params& p, int tiles, int units) {
    extra = tiles >= p.row_tiles * p.groups ? SWITCH : 0;  // a tile to a share, and more
    total = tiles + extra * units;
    // a share is at least (1 + extra) row_tiles long, so that it has a tile wherever it starts
    const int least = (1 + extra) * p.row_tiles;
    n = total >= p.groups * least ? p.groups : total == 0 ? 0 : max(1, total / least);
    length = n == 0 ? 0 : static_cast<int>(static_cast<unsigned>(total) / static_cast<unsigned>(n));
    longer = total - length * n;
  }
  // Where share r starts, before it is rounded down to a tile.
  __device__ __forceinline__ int start(int r) const { return r >= n ? total : length * r + min(r, longer); }
  // the last share that starts before position x > 0
  __device__ __forceinline__ int before(int x) const {
    const int y = x - longer * (length + 1);  // into the shorter ones
    return y <= 0 ? (x - 1) / (length + 1) : min(n - 1, longer + (y - 1) / length);
  }
};

// The request that holds a position of the list.
struct Holder {
  int b, start;  // start: its own position
  int unit;      // what one of its (request, KV head) takes of the list
  int row, tokens, ctx;
};
constexpr int PLAN_BYTES = 128 + 2 * static_cast<int>(sizeof(Holder));  // shared memory of plan()

// A CTA's walk over the segments of its share: runs of count() tiles from i0 on of one (request, KV
// head). Every warp walks by itself, beside its work: what a request's tiles are is kept, no division
// is left where there is one row tile (ONE: always), and few fields, since the softmax warps keep them
// beside a row of S. With two or three divisions to a step each role spent 2000 to 4000 cycles on it:
// 148 single tokens over 100 keys, eight one-tile segments to a CTA, took 39 us.
template <bool ONE>
struct Walk {
  int row, tokens, ctx;  // of the request
  int b, kvh, i0;
  int left;              // of the share from here on, in the list's count
  int extra;             // what a unit counts beyond its tiles
  int n, k;              // tiles of the request, and row tiles
  int member, turn;      // this CTA in its share; the member with the segment's first row tile

  __device__ __forceinline__ void enter(const Params& p, int row_, int tokens_, int ctx_) {
    row = row_;
    tokens = tokens_;
    ctx = ctx_;
    n = (ctx + tokens + BN - 1) / BN;
    k = ONE ? 1 : row_tiles_of(p, tokens);
  }
  __device__ __forceinline__ int len() const { return ctx + tokens; }
  __device__ __forceinline__ int tiles() const { return n; }
  __device__ __forceinline__ int count() const {
    return min(n - i0, (ONE || k == 1 ? left : left / k) - (i0 == 0 ? extra : 0));
  }
  // The row tile of the request that falls to this member. Requests have between one and row_tiles
  // of them: the members take turns, so that each has its share over some segments.
  __device__ __forceinline__ int row_tile(const Params& p) const {
    if (ONE) return 0;
    const int t = member - turn;
    return t < 0 ? t + p.row_tiles : t;
  }
  // Drafted tokens of this member's row tile: 0 where the request has fewer.
  __device__ __forceinline__ int rows(const Params& p) const {
    return ONE ? tokens : max(0, min(tokens - row_tile(p) * p.tok_tile, p.tok_tile));
  }
  // To the next segment with rows for this member, this one included; left is 0 where there is none.
  __device__ __forceinline__ void settle(const Params& p) {
    while (!ONE && left > 0 && rows(p) == 0) step(p);
  }
  __device__ __forceinline__ void next(const Params& p) {
    step(p);
    settle(p);
  }

 private:
  __device__ __forceinline__ void step(const Params& p) {
    const int some = count() + (i0 == 0 ? extra : 0);
    left -= ONE ? some : some * k;
    if (left <= 0) return;
    if (!ONE) {
      turn += k;
      turn = turn >= p.row_tiles ? turn - p.row_tiles : turn;
    }
    i0 = 0;
    if (++kvh == p.hkv) {
      kvh = 0;
      Request r;
      do {  // tiles are left in the share, so a request with some follows
        r = request_of(p, ++b);
      } while (tiles_of(r) == 0);
      enter(p, r.row, r.tokens, r.ctx);
    }
  }
};

// The start of every CTA, after griddepcontrol.wait: places its share and returns the walk over it
// (left is 0 where it has none); member 0 describes the unit that the share's end cuts. By all
// threads; `scratch` is PLAN_BYTES of shared memory for this alone, so that each warp goes on by
// itself from the last barrier. Rows of requests that are out of range become zero.
template <int D, bool ONE>
__device__ __forceinline__ Walk<ONE> plan(const Params& p, uint8_t* scratch) {
  int2* warp_sum = reinterpret_cast<int2*>(scratch);
  volatile Holder* holders = reinterpret_cast<volatile Holder*>(scratch + 128);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per = (p.batch + NUM_THREADS - 1) / NUM_THREADS;  // requests of a thread
  const int b0 = min(static_cast<int>(threadIdx.x) * per, p.batch), b1 = min(b0 + per, p.batch);
  // a thread's first request is kept: with up to 384 of them nothing is loaded twice
  Request kept = {};
  if (b0 < b1) kept = request_of(p, b0);
  // The block tables into L2, a line for a thread: a producer that misses it waits behind the
  // stream's own reads.
  const unsigned lines = (static_cast<unsigned>(p.max_blocks) + 31u) / 32u;  // of a request
  const unsigned line = threadIdx.x * gridDim.x + blockIdx.x;
  if (line < static_cast<unsigned long long>(lines) * p.batch) {
    const unsigned b = line / lines;
    const int32_t* at = p.tables + b * p.table_stride + (line - b * lines) * 32u;
    asm volatile("prefetch.global.L2 [%0];" ::"l"(at));
  }
  int2 mine = make_int2(0, 0);  // tiles and units of the thread's requests, for each row tile
  bool bad = false;
  for (int b = b0; b < b1; ++b) {
    const Request r = b == b0 ? kept : request_of(p, b);
    const int k = p.hkv * (ONE ? 1 : row_tiles_of(p, r.tokens)), n = tiles_of(r);
    mine.x += n * k;
    mine.y += n > 0 ? k : 0;
    bad |= r.bad;
  }
  int2 incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, incl.x, o), y = __shfl_up_sync(0xffffffffu, incl.y, o);
    if (lane >= o) incl = make_int2(incl.x + x, incl.y + y);
  }
  if (lane == 31) warp_sum[warp] = incl;
  const int any_bad = __syncthreads_or(bad ? 1 : 0);
  int2 ahead = make_int2(incl.x - mine.x, incl.y - mine.y), all = make_int2(0, 0);
#pragma unroll
  for (int w = 0; w < NUM_THREADS / 32; ++w) {
    const int2 v = warp_sum[w];
    if (w < warp) ahead = make_int2(ahead.x + v.x, ahead.y + v.y);
    all = make_int2(all.x + v.x, all.y + v.y);
  }
  const Shares sh(p, all.x, all.y);
  const int share = ONE ? blockIdx.x : static_cast<int>(blockIdx.x) / p.row_tiles;
  const int member = ONE ? 0 : static_cast<int>(blockIdx.x) - share * p.row_tiles;
  const int at0 = sh.start(share), at1 = sh.start(share + 1);
  if (share < sh.n) {
    // the requests with the starts of the share and of the next one, by the threads that have them
    const int before = ahead.x + sh.extra * ahead.y, end = before + mine.x + sh.extra * mine.y;
    const bool has0 = at0 >= before && at0 < end, has1 = at1 >= before && at1 < end;
    if (has0 || has1) {
      int t = before;
      for (int b = b0; b < b1; ++b) {
        const Request r = b == b0 ? kept : request_of(p, b);
        const int k = ONE ? 1 : row_tiles_of(p, r.tokens);
        const int unit = tiles_of(r) > 0 ? (tiles_of(r) + sh.extra) * k : 0;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int at = q == 0 ? at0 : at1;
          if (at < t || at >= t + unit * p.hkv) continue;
          volatile Holder* z = holders + q;
          z->b = b;
          z->start = t;
          z->unit = unit;
          z->row = r.row;
          z->tokens = r.tokens;
          z->ctx = r.ctx;
        }
        t += unit * p.hkv;
      }
    }
  }
  if (any_bad) {
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
  __syncthreads();
  Walk<ONE> w = {};
  w.extra = sh.extra;
  w.member = member;
  Desc cut = {};  // of the unit that starts in this share and ends in a later one
  if (share < sh.n) {
    // Of position `at` of the list: the tile that holds it, the tile's own position, its unit's.
    struct Place {
      int kvh, tile, at, unit, unit_end;
    };
    auto place = [&](volatile Holder& h, int at, int k) -> Place {
      Place z;
      const int length = h.unit;
      z.kvh = (at - h.start) / length;
      z.unit = h.start + z.kvh * length;
      z.unit_end = z.unit + length;
      const int in = at - z.unit;
      z.tile = max((ONE || k == 1 ? in : in / k) - sh.extra, 0);
      z.at = z.unit + (z.tile > 0 ? z.tile + sh.extra : 0) * k;
      return z;
    };
    w.enter(p, holders[0].row, holders[0].tokens, holders[0].ctx);
    const Place from = place(holders[0], at0, w.k);
    int end = sh.total;
    if (share + 1 < sh.n) {
      const int k = ONE ? 1 : row_tiles_of(p, holders[1].tokens);
      const Place to = place(holders[1], at1, k);
      end = to.at;
      const int rt = threadIdx.x;
      // the next share starts inside a unit, and that unit starts in this one
      if (rt < p.row_tiles && rt < k && end > to.unit && to.unit >= from.at) {
        cut.span = sh.before(to.unit_end) - share + 1;
        cut.row = holders[1].row + rt * p.tok_tile;
        cut.tokens = min(holders[1].tokens - rt * p.tok_tile, p.tok_tile);
        cut.kvh = to.kvh;
      }
    }
    w.b = holders[0].b;
    w.kvh = from.kvh;
    w.i0 = from.tile;
    w.left = end - from.at;
    w.settle(p);
  }
  if (member == 0 && threadIdx.x < p.row_tiles) p.desc[blockIdx.x + threadIdx.x] = cut;
  return w;
}

// The slot of a part of a unit that a share holds: one for a unit from an earlier share, one for a
// unit that goes on in the next.
__device__ __forceinline__ long long slot_of(const Params& p, int share, int rt, bool from_before) {
  return 2LL * (share * p.row_tiles + rt) + (from_before ? 0 : 1);
}

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
  const int ch = tid % CHUNKS;
  uint8_t* piece = tile + (ch >> 3) * 1024 + (ch & 7) * 16;
#pragma unroll 1
  for (int row = max(first, from) + tid / CHUNKS; row < from + count; row += 128 / CHUNKS) {
    uint4* at = reinterpret_cast<uint4*>(piece + (row >> 3) * (D / 64 * 1024) + (row & 7) * 128);
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

// Two elements of O. A weighted mean is never beyond its values, but the rounding of the weights (up to
// 2^-11) can carry a mean of f16's largest numbers past 65520, which would become infinite: what is
// finite stays so. (A bf16 mean would be infinite in fp32 already.)
template <bool BF16>
__device__ __forceinline__ uint32_t pack_o(float a, float b) {
  if constexpr (!BF16) {
    const auto within = [](float x) {
      return fabsf(x) < INFINITY ? fminf(fmaxf(x, -65504.f), 65504.f) : x;
    };
    a = within(a);
    b = within(b);
  }
  return pack2<BF16>(a, b);
}

// The bits of drafted token t (in its request of `tokens`): the drafted tokens that it sees.
__device__ __forceinline__ uint64_t bits_of(const Params& p, int row, int t, int tokens) {
  const uint64_t bits = p.tree != nullptr ? static_cast<uint64_t>(p.tree[row + t])
                                          : (2ull << t) - 1ull;  // a chain; t = 63: all ones
  return tokens < 64 ? bits & ((1ull << tokens) - 1ull) : bits;
}

// One K or V producer's loads, into a ring of STAGES: lane i loads page i of a tile.
template <int D, int STAGES>
struct Loader {
  static constexpr int GROUP = D / 64 * 1024, TILE = BN / 8 * GROUP;
  const CUtensorMap* map;
  uint8_t* ring;
  uint64_t* full;
  uint64_t* empty;
  volatile int* abort;
  uint64_t policy;
  uint32_t n;   // tiles so far
  int id, id1;  // this lane's blocks of the segment's next two tiles, in flight

  // this lane's block of tile i
  template <typename W>
  __device__ __forceinline__ int block_of(const Params& p, const W& w, int i) const {
    const int at = i * (BN >> p.box_log2) + static_cast<int>(threadIdx.x & 31);
    if (static_cast<int>(threadIdx.x & 31) >= BN >> p.box_log2 || at << p.box_log2 >= w.len()) return 0;
    return p.tables[w.b * p.table_stride + (at >> (p.page_log2 - p.box_log2))];
  }
  template <typename W>
  __device__ __forceinline__ void start(const Params& p, const W& w, int end) {
    id = block_of(p, w, w.i0);
    id1 = w.i0 + 1 < end ? block_of(p, w, w.i0 + 1) : 0;
  }
  // Tile i of the segment that ends before tile `end`.
  template <typename W>
  __device__ __forceinline__ bool load(const Params& p, const W& w, int i, int end) {
    const int lane = threadIdx.x & 31;
    const int box = 1 << p.box_log2, pages = BN >> p.box_log2, group_box = box / 8;
    const int id2 = i + 2 < end ? block_of(p, w, i + 2) : 0;
    const int st = static_cast<int>(n % STAGES);
    if (!wait_for(&empty[st], ((n / STAGES) & 1u) ^ 1u, abort, p.status, SITE_PROD_KV)) return false;
    ++n;
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
      const int boxes = 1 << (p.page_log2 - p.box_log2);  // of a block
      tma_load_5d_hint(map, &full[st], ring + st * TILE + lane * group_box * GROUP, 0, 0, 0,
                       ((i * pages + lane) & (boxes - 1)) * group_box, first, policy);
    }
    __syncwarp();
    id = id1;
    id1 = id2;
    return true;
  }
  // After another role gave up: no copy may be in flight when the block ends (bounded like every
  // wait).
  __device__ __forceinline__ void drain(const Params& p) {
    if (*abort == 0 || (threadIdx.x & 31) != 0) return;
    int none = 0;
    for (uint32_t k = n > STAGES ? n - STAGES : 0; k < n; ++k) {
      wait_for(&full[k % STAGES], (k / STAGES) & 1u, &none, p.status, SITE_PROD_KV);
    }
  }
};

// K or V producer warp.
template <int D, int STAGES, typename W>
__device__ __forceinline__ void produce_kv(const Params& p, W w, Loader<D, STAGES> ld) {
  bool ok = true;
  for (; w.left > 0 && ok; w.next(p)) {
    const int end = w.i0 + w.count();
    ld.start(p, w, end);
    for (int i = w.i0; i < end && ok; ++i) ok = ld.load(p, w, i, end);
    if (!ok) break;
  }
  ld.drain(p);
}

// Producer warp of Q: each segment's query rows, [half][rows][128 B], into one of BUFS buffers.
template <int D, int BUFS, typename W>
__device__ __forceinline__ void produce_q(const Params& p, W w, const CUtensorMap* map, uint8_t* base,
                                          int buf_bytes, int half_bytes, uint64_t* full, uint64_t* empty,
                                          volatile int* abort_flag) {
  if ((threadIdx.x & 31) == 0) {
    uint32_t n = 0;  // segments so far
    for (; w.left > 0; w.next(p)) {
      const uint32_t buf = n % BUFS;
      if (!wait_for(&empty[buf], ((n / BUFS) & 1u) ^ 1u, abort_flag, p.status, SITE_PROD_Q)) break;
      ++n;
      mbar_arrive_expect_tx(&full[buf], static_cast<uint32_t>(p.box_tokens * p.group * D * 2));
#pragma unroll
      for (int h = 0; h < D / 64; ++h) {
        tma_load_3d(map, &full[buf], base + buf * buf_bytes + h * half_bytes, h * 64, w.kvh * p.group,
                    w.row + w.row_tile(p) * p.tok_tile);
      }
    }
    if (*abort_flag != 0) {
      int none = 0;
      for (uint32_t k = n > BUFS ? n - BUFS : 0; k < n; ++k) {
        wait_for(&full[k % BUFS], (k / BUFS) & 1u, &none, p.status, SITE_PROD_Q);
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
