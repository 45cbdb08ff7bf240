// What the two tree-attention kernels (tree.cu: many query rows, tree_narrow.cu: up to 64) share:
// the work list of a launch, the walk of a CTA over its range, the TMA producers, and the clean-up
// of V tiles that end inside a page. The operator is described in tree.cu.
#pragma once

#include <cstddef>

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
constexpr int ROUNDS = 4;             // ranges of a CTA, about
constexpr int MAX_ITEMS = ROUNDS * MAX_CTAS;
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
  SITE_NEXT = 0x913,     // the next range's entry
  SITE_NEXT_FREE = 0x914,
  SITE_JOIN = 0x915,     // the warps that join a unit, among themselves
};

// The work list is the 128-key tiles of every (request, KV head), cut into ranges (plan_kernel).
// An item is a range for one of its row_tiles members.
struct Range {
  int b, kvh, i0;        // the first tile
  int left;              // its length in the work list's count, 0: no more ranges
  int row, tokens, ctx;  // of request b
  int home;              // i0 > 0: the range in which the first tile's unit starts
  int span;              // ranges that hold a part of the unit that starts here and ends later; 0: none
  int id, member;        // filled in where the item is taken
  int pad;
};
constexpr int RANGE_WORDS = sizeof(Range) / 4;

// Ranges stand in the order of the list, `cuts` of a share one after the other. Items are taken in
// the order (cut, share, member).
struct Plan {
  int shares, cuts;
  unsigned int next;  // items taken beyond the first gridDim.x
};

struct Params {
  const int32_t* ctx;      // [B]
  const int32_t* offsets;  // [B + 1]
  const int64_t* tree;     // [rows] or nullptr: a chain
  const int32_t* tables;   // [B, max_blocks]
  void* out;               // [rows, Hq, D]
  float* lse;              // [rows, Hq]
  const void* v;           // the V cache, for drafted rows that are not finite
  Plan* plan;
  Range* ranges;           // [MAX_ITEMS]
  unsigned int* arrived;   // [MAX_ITEMS] parts of the unit that starts in a range, for a row tile
  float2* part_ml;         // [2 MAX_ITEMS][row_cap] (maximum, sum), log2 units
  float* part_o;           // [2 MAX_ITEMS][row_cap][D], not normalised
  long long table_stride;
  int batch, rows, hq, hkv, group, max_new, max_blocks, num_blocks;
  int page_log2;           // tokens of a block
  int box_log2;            // tokens of a TMA box: min(block, 128)
  int tok_tile;            // drafted tokens of a row tile: 128 / group
  int box_tokens;          // tokens of the Q box: min(tok_tile, max_new)
  int row_tiles;           // members of a range, a row tile each
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

// A CTA's walk over the segments of its ranges: runs of count() tiles from i0 on of one (request,
// KV head). Few fields, since the softmax warps keep it beside a row of S. Every warp walks by
// itself; from the second range on it reads them from a two-entry ring in shared memory that the K
// producer fills.
struct Feed {
  Range* ring;  // [2]
  uint64_t* full;
  uint64_t* empty;
  volatile int* abort;
};

struct Walk {
  int row, tokens, ctx;  // of the request
  int b, kvh, i0;
  int left;              // of the range from here on, in the work list's count
  int turn;              // the member that takes the segment's first row tile
  int id, member;        // of the item
  uint32_t taken;        // entries of the ring so far

  __device__ __forceinline__ int len() const { return ctx + tokens; }
  __device__ __forceinline__ int tiles() const { return (len() + BN - 1) / BN; }
  __device__ __forceinline__ int count(const Params& p) const {
    return min(tiles() - i0, left / row_tiles_of(p, tokens));
  }
  // The row tile of the request that falls to this member. Requests have between one and row_tiles
  // of them: the members take turns, so that each has its share over some segments.
  __device__ __forceinline__ int row_tile(const Params& p) const {
    const int k = member - turn;
    return k < 0 ? k + p.row_tiles : k;
  }
  // Drafted tokens of this member's row tile: 0 where the request has fewer.
  __device__ __forceinline__ int rows(const Params& p) const {
    return max(0, min(tokens - row_tile(p) * p.tok_tile, p.tok_tile));
  }
  __device__ __forceinline__ void set(const Range& r) {
    b = r.b;
    kvh = r.kvh;
    i0 = r.i0;
    left = r.left;
    row = r.row;
    tokens = r.tokens;
    ctx = r.ctx;
    id = r.id;
    member = r.member;
    turn = 0;
  }
  // Past this segment, inside the range.
  __device__ __forceinline__ void step(const Params& p) {
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
      row = r.row;
      tokens = r.tokens;
      ctx = r.ctx;
    }
  }
  // To the range's next segment, this one included, in which the member has rows; left is 0 where
  // there is none.
  __device__ __forceinline__ void settle(const Params& p) {
    while (left > 0 && rows(p) == 0) step(p);
  }
  // The CTA's first item; left is 0 where it has none.
  __device__ __forceinline__ void open(const Params& p) {
    taken = 0;
    left = 0;
    const int share = static_cast<int>(blockIdx.x) / p.row_tiles;
    if (share >= p.plan->shares) return;
    const int range = share * p.plan->cuts;
    Range r = p.ranges[range];
    r.id = range;
    r.member = static_cast<int>(blockIdx.x) - share * p.row_tiles;
    set(r);
  }
  // The next range from the ring, by a warp (or by its lane 0 alone); left is 0 at the end.
  __device__ __forceinline__ void take(const Params& p, const Feed& f, bool alone) {
    left = 0;
    const uint32_t at = taken & 1u;
    if (!mbar_wait(&f.full[at], (taken >> 1) & 1u, f.abort, p.status, SITE_NEXT)) return;
    set(f.ring[at]);
    ++taken;
    if (!alone) __syncwarp();
    if (alone || (threadIdx.x & 31) == 0) mbar_arrive(&f.empty[at]);
  }
  // A first segment with rows, from the first item or a later one.
  __device__ __forceinline__ void begin(const Params& p, const Feed& f, bool alone = false) {
    open(p);
    if (left <= 0) return;
    settle(p);
    while (left <= 0) {
      take(p, f, alone);
      if (left <= 0) return;
      settle(p);
    }
  }
  // The next segment with rows, in this range or the next ones.
  __device__ __forceinline__ void next(const Params& p, const Feed& f, bool alone = false) {
    step(p);
    if (left > 0) settle(p);
    while (left <= 0) {
      take(p, f, alone);
      if (left <= 0) return;
      settle(p);
    }
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

// One K or V producer's loads, into a ring of STAGES: lane i loads page i of a tile.
template <int D, int STAGES>
struct Loader {
  static constexpr int GROUP = D / 64 * 1024, TILE = BN / 8 * GROUP;
  const CUtensorMap* map;
  uint8_t* ring;
  uint64_t* full;
  uint64_t* empty;
  volatile int* abort;
  uint32_t n;   // tiles so far
  int id, id1;  // this lane's blocks of the segment's next two tiles, in flight

  // this lane's block of tile i
  __device__ __forceinline__ int block_of(const Params& p, const Walk& w, int i) const {
    const int at = i * (BN >> p.box_log2) + static_cast<int>(threadIdx.x & 31);
    if (static_cast<int>(threadIdx.x & 31) >= BN >> p.box_log2 || at << p.box_log2 >= w.len()) return 0;
    return p.tables[w.b * p.table_stride + (at >> (p.page_log2 - p.box_log2))];
  }
  __device__ __forceinline__ void start(const Params& p, const Walk& w, int end) {
    id = block_of(p, w, w.i0);
    id1 = w.i0 + 1 < end ? block_of(p, w, w.i0 + 1) : 0;
  }
  // Tile i of the segment that ends before tile `end`.
  __device__ __forceinline__ bool load(const Params& p, const Walk& w, int i, int end) {
    const int lane = threadIdx.x & 31;
    const int box = 1 << p.box_log2, pages = BN >> p.box_log2, group_box = box / 8;
    const int id2 = i + 2 < end ? block_of(p, w, i + 2) : 0;
    const int st = static_cast<int>(n % STAGES);
    if (!mbar_wait(&empty[st], ((n / STAGES) & 1u) ^ 1u, abort, p.status, SITE_PROD_KV)) return false;
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
      tma_load_5d(map, &full[st], ring + st * TILE + lane * group_box * GROUP, 0, 0, 0,
                  ((i * pages + lane) & (boxes - 1)) * group_box, first);
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
      mbar_wait(&full[k % STAGES], (k / STAGES) & 1u, &none, p.status, SITE_PROD_KV);
    }
  }
};

// V producer warp.
template <int D, int STAGES>
__device__ __forceinline__ void produce_v(const Params& p, const Feed& feed, Loader<D, STAGES> ld) {
  Walk w;
  bool ok = true;
  for (w.begin(p, feed); w.left > 0 && ok; w.next(p, feed)) {
    const int end = w.i0 + w.count(p);
    ld.start(p, w, end);
    for (int i = w.i0; i < end && ok; ++i) ok = ld.load(p, w, i, end);
    if (!ok) break;
  }
  ld.drain(p);
}

// K producer warp, which also takes the CTA's items: the first gridDim.x are the CTAs' own, the
// others go to whoever comes first. It asks for the next one (an atomic, then a load) some tiles
// before the range ends, so late that a CTA that is behind leaves it to others and early enough
// that no tile waits for the answer.
constexpr int ASK_AHEAD = 6, READ_AHEAD = 3;

template <int D, int STAGES>
__device__ __forceinline__ void produce_k(const Params& p, const Feed& feed, Loader<D, STAGES> ld) {
  const int lane = threadIdx.x & 31;
  const int shares = p.plan->shares, cuts = p.plan->cuts;
  // the first round's items are the CTAs' own; where there are fewer shares, nothing else is taken
  const int items = cuts > 1 ? shares * cuts * p.row_tiles : 0;
  Walk w;
  w.open(p);
  uint32_t pushed = 0;
  bool ok = true;
  while (w.left > 0 && ok) {
    int state = 0;  // of the next item: 1 asked for, 2 read
    int item = 0, word = 0;
    auto ask = [&]() {
      item = lane == 0 ? static_cast<int>(gridDim.x + atomicAdd(&p.plan->next, 1u)) : 0;
      state = 1;
    };
    auto read = [&]() {  // lane i gets word i of the entry
      item = __shfl_sync(0xffffffffu, item, 0);
      word = 0;
      if (item >= 0 && item < items) {
        const int at = item / p.row_tiles, cut = at / shares;
        const int range = (at - cut * shares) * cuts + cut;
        if (lane < RANGE_WORDS) word = reinterpret_cast<const int*>(p.ranges + range)[lane];
        if (lane == offsetof(Range, id) / 4) word = range;
        if (lane == offsetof(Range, member) / 4) word = item - at * p.row_tiles;
      }
      state = 2;
    };
    w.settle(p);
    while (w.left > 0 && ok) {
      const int tiles = w.count(p), end = w.i0 + tiles;
      // tiles of the range from here on, as far as this segment tells
      const bool last = w.left - tiles * row_tiles_of(p, w.tokens) <= 0;
      ld.start(p, w, end);
      for (int i = w.i0; i < end && ok; ++i) {
        if (last && state == 0 && end - i <= ASK_AHEAD) ask();
        if (last && state == 1 && end - i <= READ_AHEAD) read();
        ok = ld.load(p, w, i, end);
      }
      if (!ok) break;
      w.step(p);
      w.settle(p);
    }
    if (!ok) break;
    const uint32_t at = pushed & 1u;
    if (!mbar_wait(&feed.empty[at], ((pushed >> 1) & 1u) ^ 1u, feed.abort, p.status, SITE_NEXT_FREE)) break;
    // An item without rows for its member is passed over here: the MMA warp looks one segment ahead
    // before it issues a segment's last product, and two such items would have it wait for an entry
    // whose place in the ring the softmax warps only free behind that product.
    do {
      if (state == 0) ask();
      if (state == 1) read();
      if (lane < RANGE_WORDS) reinterpret_cast<volatile int*>(feed.ring + at)[lane] = word;
      __syncwarp();
      w.set(feed.ring[at]);
      __syncwarp();
      state = 0;
      if (w.left <= 0) break;  // no more
      Walk first = w;
      first.settle(p);
      if (first.left > 0) break;
    } while (true);
    if (lane == 0) mbar_arrive(&feed.full[at]);
    ++pushed;
  }
  ld.drain(p);
}

// Producer warp of Q: each segment's query rows, [half][rows][128 B], into one of BUFS buffers.
template <int D, int BUFS>
__device__ __forceinline__ void produce_q(const Params& p, const Feed& feed, const CUtensorMap* map,
                                          uint8_t* base, int buf_bytes, int half_bytes, uint64_t* full,
                                          uint64_t* empty) {
  if ((threadIdx.x & 31) == 0) {
    Walk w;
    uint32_t n = 0;  // segments so far
    for (w.begin(p, feed, true); w.left > 0; w.next(p, feed, true)) {
      const uint32_t buf = n % BUFS;
      if (!mbar_wait(&empty[buf], ((n / BUFS) & 1u) ^ 1u, feed.abort, p.status, SITE_PROD_Q)) break;
      ++n;
      mbar_arrive_expect_tx(&full[buf], static_cast<uint32_t>(p.box_tokens * p.group * D * 2));
#pragma unroll
      for (int h = 0; h < D / 64; ++h) {
        tma_load_3d(map, &full[buf], base + buf * buf_bytes + h * half_bytes, h * 64, w.kvh * p.group,
                    w.row + w.row_tile(p) * p.tok_tile);
      }
    }
    if (*feed.abort != 0) {
      int none = 0;
      for (uint32_t k = n > BUFS ? n - BUFS : 0; k < n; ++k) {
        mbar_wait(&full[k % BUFS], (k / BUFS) & 1u, &none, p.status, SITE_PROD_Q);
      }
    }
  }
  __syncwarp();
}

// The slot of a part of a unit (a row tile's tiles of one (request, KV head)) that range `id` holds:
// one for a unit from an earlier range, one for a unit that goes on in the next.
__device__ __forceinline__ long long slot_of(const Params& p, int id, int rt, bool from_before) {
  return 2LL * (static_cast<long long>(id) * p.row_tiles + rt) + (from_before ? 0 : 1);
}

// The WARPS warps that hold a segment's result, among themselves: sync() orders their earlier
// writes (shared and global) before their later accesses, with the library's bounded wait.
template <int WARPS>
struct Team {
  uint64_t* bar;  // count WARPS
  volatile int* abort;
  volatile int* flag;
  unsigned int* status;
  int warp;  // 0 .. WARPS - 1
  uint32_t phase;
  __device__ __forceinline__ bool sync() {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
    const bool ok = mbar_wait(bar, phase, abort, status, SITE_JOIN);
    phase ^= 1u;
    return ok;
  }
};

// After a part's stores: counts it, and where it is the unit's last, joins the parts: M = max m,
// O = sum 2^(m - M) O_part / sum 2^(m - M) l, in the order of the ranges whoever comes last. A warp
// takes a row at a time (a lane four dimensions), the loads of four rows and parts together.
template <bool BF16, int D, int WARPS>
__device__ __forceinline__ bool join(const Params& p, Team<WARPS>& team, const Walk& w, int rt, int tokens) {
  const Range* mine = p.ranges + w.id;
  const int home = w.i0 > 0 ? mine->home : w.id;
  const int span = p.ranges[home].span;
  if (!team.sync()) return false;
  if (team.warp == 0 && (threadIdx.x & 31) == 0) {
    __threadfence();  // cumulative: the team's stores before this arrival
    const unsigned int before = atomicAdd(p.arrived + home * p.row_tiles + rt, 1u);
    __threadfence();
    *team.flag = before + 1u == static_cast<unsigned int>(span) ? 1 : 0;
  }
  if (!team.sync()) return false;
  if (*team.flag == 0) return true;
  constexpr int U = 4, PARTS = 4;
  const int rows = tokens * p.group, lane = threadIdx.x & 31;
  for (int r0 = team.warp; r0 < rows; r0 += WARPS * U) {
    float m[U], l[U];
    float4 o[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      m[u] = -INFINITY;
      l[u] = 0.f;
      o[u] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (int c0 = 0; c0 < span; c0 += PARTS) {
      float2 ml[PARTS][U];
      float4 part[PARTS][U];
#pragma unroll
      for (int c = 0; c < PARTS; ++c) {
        const long long slot = slot_of(p, home + c0 + c, rt, c0 + c > 0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int r = r0 + u * WARPS;
          ml[c][u] = make_float2(-INFINITY, 0.f);
          part[c][u] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (r < rows && lane < D / 4 && c0 + c < span) {
            ml[c][u] = __ldcg(p.part_ml + slot * p.row_cap + r);
            part[c][u] = __ldcg(reinterpret_cast<const float4*>(p.part_o + (slot * p.row_cap + r) * D) + lane);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float top = m[u];
#pragma unroll
        for (int c = 0; c < PARTS; ++c) top = fmaxf(top, ml[c][u].x);
        const float base = top == -INFINITY ? 0.f : top, a = ex2(m[u] - base);
        m[u] = top;
        l[u] *= a;
        o[u] = make_float4(o[u].x * a, o[u].y * a, o[u].z * a, o[u].w * a);
#pragma unroll
        for (int c = 0; c < PARTS; ++c) {
          const float b = ex2(ml[c][u].x - base);
          l[u] = fmaf(ml[c][u].y, b, l[u]);
          o[u].x = fmaf(part[c][u].x, b, o[u].x);
          o[u].y = fmaf(part[c][u].y, b, o[u].y);
          o[u].z = fmaf(part[c][u].z, b, o[u].z);
          o[u].w = fmaf(part[c][u].w, b, o[u].w);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = r0 + u * WARPS;
      if (r >= rows || lane >= D / 4) continue;
      const float inv = l[u] == 0.f ? 0.f : 1.f / l[u];  // a row that sees nothing: O = 0
      const int tok = r / p.group;
      const long long at = static_cast<long long>(w.row + rt * p.tok_tile + tok) * p.hq + w.kvh * p.group +
                           (r - tok * p.group);
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at * D + lane * 4) =
          make_uint2(pack2<BF16>(o[u].x * inv, o[u].y * inv), pack2<BF16>(o[u].z * inv, o[u].w * inv));
      if (lane == 0) p.lse[at] = l[u] == 0.f ? -INFINITY : (m[u] + log2f(l[u])) * 0.6931471805599453f;
    }
  }
  return true;
}

// tree_narrow.cu; the tensor maps are encoded by the caller.
template <bool BF16, int D>
int launch_narrow(const Params& p, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                  int grid, cudaStream_t stream);

}  // namespace tree
}  // namespace kta
