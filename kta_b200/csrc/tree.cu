// Attention of a tree of drafted tokens over a paged KV cache, sm_100a.
//
//   For request b with c = ctx[b] tokens in the cache and t drafted ones behind them (rows
//   offsets[b] .. offsets[b + 1] of Q, keys c .. c + t - 1 of the cache, t <= 64):
//   row i sees key p iff p < c, or bit p - c of tree[i] is set (p - c < t);
//   O = softmax(scale Q K^T over the seen keys) V,  LSE = log of the sum, natural.
//
// One drafted token is the decode step of a paged cache; a chain is the tree 1, 11, 111, ...
//
//   * A KV head's query rows of one request (tokens x heads of the group, up to 128 in a row
//     tile) share its K and V, so they are the rows of one tcgen05 tile: S = Q K^T is 128 x 128
//     per 128 keys however few of them are real. At 128 rows the tensor core needs ~1000 cycles
//     for a tile of keys, the softmax ~1500 and the HBM stream ~2800 (64 KB at an SM's share), so
//     the padding of few rows is free and one kernel serves from 1 to 128 rows at HBM speed.
//   * Work is the list of 128-key tiles of every (request, KV head), in contiguous ranges of
//     equal length, one range per CTA (or per `row_tiles` CTAs with a row tile each, which then
//     read the same K and V at about the same time: the second reader finds them in L2). Ragged
//     lengths balance to a tile; what a range cuts is joined by a second small kernel from fp32
//     partials (O, maximum, sum) in the workspace: no counters to keep at zero between calls.
//   * Six roles in 192 threads: warps 0-3 softmax (thread = query row = TMEM lane), warp 4 TMA
//     producer, warp 5 TMEM owner and MMA issuer. K and V tiles share a ring of six slots in the
//     order the tensor core takes them, K(0) K(1) V(0) K(2) V(1) ...: S of the next tile is
//     computed while the softmax works, in the other of two S buffers.
//   * Pages: a box of the tensor map is one page (up to 128 tokens) of one head, with the token
//     index split as (8, page / 8): shared memory gets 8-token groups of both 64-wide halves of
//     the head, [group][half][8 tokens][128 B], which for every page size is one uniform stride
//     for the matrix descriptors and one TMA per page. Lane i of the producer loads page i.
//   * The last tile of a request ends inside a page: K's leftover columns are masked by
//     selection, and V's leftover rows are set to zero in shared memory, since 0 * NaN from a
//     page's unwritten rows would reach every row through the matrix product. Likewise a drafted
//     V row that is not finite is zeroed and handed to the rows that see it alone.
//   * Out-of-range lengths, offsets and block ids become status KTA_ERR_DEVICE_BOUNDS: such a
//     request's rows are zero (LSE -inf), such a block reads as zeros. Every wait is bounded.
#include <algorithm>
#include <cmath>

#include "kta_common.cuh"
#include "kta_host.h"

namespace kta {
namespace tree {

constexpr int BM = 128;               // query rows of a row tile: TMEM lanes
constexpr int BN = 128;               // keys of a tile
constexpr int RING = 3;               // K tiles in flight, and V tiles
constexpr int HK = BN / 2;            // keys of a tile that a softmax warpgroup takes
constexpr int SOFTMAX_WARPS = 8;      // two warpgroups
constexpr int MMA_WARP = 8;
constexpr int K_WARP = 9;             // TMA producers
constexpr int V_WARP = 10;
constexpr int Q_WARP = 11;
constexpr int NUM_THREADS = 384;
constexpr int MAX_DRAFT = 64;         // bits of a row of the tree
constexpr int MAX_GROUP = 16;
constexpr int MAX_BATCH = 1 << 16;
constexpr int MAX_CTAS = 256;         // the workspace is sized for this many
constexpr float RESCALE_THRESHOLD = 8.0f;  // log2 units: the maximum moves when it grew > 2^8
constexpr uint32_t COL_O = 256;       // TMEM: S buffer i at i * 128, O of warpgroup w at 256 + w * 128

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

template <int D>
struct Layout {
  static constexpr int HALVES = D / 64;
  static constexpr int GROUP = HALVES * 1024;      // 8 tokens: [half][8][128 B]
  static constexpr int TILE = BN / 8 * GROUP;      // a K or V tile
  static constexpr int Q_HALF = BM * 128;          // [128 rows][64 d]
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_K = OFF_Q + HALVES * Q_HALF;
  static constexpr int OFF_V = OFF_K + RING * TILE;
  static constexpr int OFF_ML = OFF_V + RING * TILE;  // [warpgroup][128 rows] (maximum, sum)
  static constexpr int OFF_BAR = OFF_ML + 2 * BM * 8;
  // k_full[R], k_empty[R], v_full[R], v_empty[R], q_full[2], q_empty[2], s_full[2], p_full[2][2],
  // pv_done[2], ml_full, o_done, o_free
  static constexpr int NUM_BARS = 4 * RING + 15;
  static constexpr int OFF_MISC = OFF_BAR + NUM_BARS * 8;
  // misc: tmem base, abort, non-finite drafts, the range's first segment and end
  static constexpr int TOTAL = OFF_MISC + 64;
  static_assert(TOTAL <= 232448, "shared memory budget of one sm_100 CTA");
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
  float4* part_o;          // [2 CTAs][D / 4][row_cap], not normalised
  long long table_stride;
  int batch, rows, hq, hkv, group, max_new, max_blocks, num_blocks;
  int page_log2;           // tokens of a block
  int box_log2;            // tokens of a TMA box: min(block, 128)
  int tok_tile;            // drafted tokens of a row tile: 128 / group
  int box_tokens;          // tokens of the Q box: min(tok_tile, max_new)
  int row_tiles;           // CTAs that share a range
  int q_bufs, q_shift;     // Q tiles in shared memory, bytes from one to the next
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

// Half an S tile of one query row (64 keys; this thread's TMEM lane): P = 2^(S sl - m) over the
// first 32 columns, the running maximum m (log2 units) and the row sum l of this half. m moves only
// when the true maximum grew by more than 2^8, so O is rescaled rarely; that waits for the PV
// before. pv_done is at most one phase behind: S of this tile was issued behind the PV before that.
template <bool MASKED, bool BF16, int D>
__device__ __forceinline__ bool softmax_step(uint32_t t_s, uint32_t t_o, const uint32_t (&view)[2],
                                             float sl, float& m_used, float& lsum, uint64_t* pv_done,
                                             uint32_t pv_parity, volatile int* abort,
                                             unsigned int* status) {
  uint32_t r[HK];
#pragma unroll
  for (int q = 0; q < HK / 32; ++q) {
    tmem_ld_32x32b_x32(t_s + q * 32, *reinterpret_cast<uint32_t(*)[32]>(r + q * 32));
  }
  tmem_ld_wait();
  reg_fence(r);
  if (MASKED) {
#pragma unroll
    for (int c = 0; c < HK; ++c) {
      if (!((view[c / 32] >> (c % 32)) & 1u)) r[c] = __float_as_uint(-INFINITY);
    }
  }
  float mx[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) mx[i] = -INFINITY;
#pragma unroll
  for (int i = 0; i < HK / 2; ++i) {
    mx[i & 3] = max3(mx[i & 3], __uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
  }
  const float rmax = max3(mx[0], mx[1], fmaxf(mx[2], mx[3])) * sl;
  float factor = 1.f;
  bool rescale = false;
  if (rmax > m_used + RESCALE_THRESHOLD) {
    factor = ex2(m_used - rmax);  // 0 where nothing was seen so far
    rescale = m_used != -INFINITY;
    m_used = rmax;
  }
  lsum *= factor;
  if (__any_sync(0xffffffffu, rescale)) {
    if (!mbar_wait(pv_done, pv_parity, abort, status, SITE_SM_PV)) return false;
    tc_fence_after();
    const float f = rescale ? factor : 1.f;
#pragma unroll 1
    for (int c = 0; c < D; c += 16) {
      uint32_t o[16];
      tmem_ld_32x32b_x16(t_o + c, o);
      tmem_ld_wait();
      reg_fence(o);
#pragma unroll
      for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
      tmem_st_32x32b_x16(t_o + c, o);
    }
  }
  // a row that has seen nothing keeps m = -inf: subtract 0 there, every exponential is 2^-inf
  const float m = m_used == -INFINITY ? 0.f : m_used;
  const uint64_t sl2 = f2(sl, sl);
  const uint64_t neg2 = f2(-m, -m);
  uint64_t sum2[4] = {0ull, 0ull, 0ull, 0ull};
  uint32_t pk[HK / 2];
#pragma unroll
  for (int i = 0; i < HK / 2; ++i) {
    const uint64_t x = fma2(f2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), sl2, neg2);
    float x0, x1;
    f2_split(x, x0, x1);
    const float e0 = ex2(x0), e1 = ex2(x1);
    sum2[i & 3] = add2(sum2[i & 3], f2(e0, e1));
    pk[i] = pack2<BF16>(e0, e1);
  }
  tmem_st_32x32b_x32(t_s, pk);
  tmem_st_wait();
  const uint64_t s01 = add2(add2(sum2[0], sum2[1]), add2(sum2[2], sum2[3]));
  float s0, s1;
  f2_split(s01, s0, s1);
  lsum += s0 + s1;
  return true;
}

// 16-bit elements of a word whose exponent is all ones (infinities and NaN), as a mask of them.
template <bool BF16>
__device__ __forceinline__ uint32_t nonfinite(uint32_t w) {
  constexpr uint32_t E = BF16 ? 0x7F80u : 0x7C00u;
  return ((w & E) == E ? 0xffffu : 0u) | ((w >> 16 & E) == E ? 0xffff0000u : 0u);
}

// Rows [from, from + 64) of a V tile (shared memory) of which [first, valid) are drafted tokens:
// rows past `valid` become zero, and so do drafted elements that are not finite, whose tokens are
// recorded in bad[0..1] (token = row + token0). By the 128 threads of a warpgroup.
template <bool BF16, int D>
__device__ __forceinline__ void clean_v(uint8_t* tile, int from, int first, int valid, int token0, int tid,
                                        unsigned int* bad) {
  constexpr int CHUNKS = D / 8;  // 16-byte pieces of a row
  for (int i = tid + max(first, from) * CHUNKS; i < (from + HK) * CHUNKS; i += BM) {
    const int row = i / CHUNKS, ch = i % CHUNKS;
    uint4* at = reinterpret_cast<uint4*>(tile + (row >> 3) * Layout<D>::GROUP + (ch >> 3) * 1024 +
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

template <bool BF16, int D>
__global__ void __launch_bounds__(NUM_THREADS, 1)
    tree_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                const __grid_constant__ CUtensorMap tmV, const Params p) {
  using L = Layout<D>;
  // Asked for at 1024 bytes (the 128-byte swizzle's period): there is no room to round up in.
  extern __shared__ __align__(1024) uint8_t smem[];
  if ((smem_u32(smem) & 1023u) != 0) {
    pdl_wait();
    if (threadIdx.x == 0) {
      record_status(p.status, KTA_ERR_LAUNCH, SITE_SMEM);
      p.desc[blockIdx.x] = Desc{};
    }
    return;
  }
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint64_t* k_empty = k_full + RING;
  uint64_t* v_full = k_empty + RING;
  uint64_t* v_empty = v_full + RING;
  uint64_t* q_full = v_empty + RING;  // [Q buffer]
  uint64_t* q_empty = q_full + 2;     // [Q buffer]: the segment's last S has read Q
  uint64_t* s_full = q_empty + 2;    // [S buffer]
  uint64_t* p_full = s_full + 2;     // [buffer][warpgroup]: its half of P written, of V cleaned
  uint64_t* pv_done = p_full + 4;    // [warpgroup]: one phase for each PV into its O
  uint64_t* ml_full = pv_done + 2;   // both warpgroups' maxima and sums are in shared memory
  uint64_t* o_done = ml_full + 1;    // the segment's last PV
  uint64_t* o_free = o_done + 1;     // the epilogue has read both O
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + L::OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::OFF_MISC + 4);
  unsigned int* bad = reinterpret_cast<unsigned int*>(smem + L::OFF_MISC + 8);   // [2]
  // the range's first segment (request, KV head, tile), its place in the work list, the range's end,
  // and the list's total
  volatile int* plan = reinterpret_cast<volatile int*>(smem + L::OFF_MISC + 16);  // [6]
  float2* ml = reinterpret_cast<float2*>(smem + L::OFF_ML);
  int* warp_sum = reinterpret_cast<int*>(smem + L::OFF_K);  // before the ring is used

  const int warp = warp_id();
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < RING; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[2 * i], SOFTMAX_WARPS / 2);
      mbar_init(&p_full[2 * i + 1], SOFTMAX_WARPS / 2);
      mbar_init(&pv_done[i], 1);
    }
    mbar_init(ml_full, SOFTMAX_WARPS);
    mbar_init(o_done, 1);
    mbar_init(o_free, SOFTMAX_WARPS);
    *abort_flag = 0;
    bad[0] = bad[1] = 0u;
    fence_barrier_init();
  }
  if (warp == K_WARP && lane == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == MMA_WARP) {
    tmem_alloc(tmem_holder, 512);
    tmem_relinquish();
  }
  pdl_wait();  // the previous grid's writes (this launch's inputs) are visible from here on
  // after the wait: the join kernel may be scheduled now, and waits for this grid itself
  pdl_launch_dependents();

  // ---- the work list: thread i sums a run of requests ----
  const int per = (p.batch + NUM_THREADS - 1) / NUM_THREADS;
  const int b0 = min(static_cast<int>(threadIdx.x) * per, p.batch), b1 = min(b0 + per, p.batch);
  auto work_of = [&](const Request& r) { return tiles_of(r) * p.hkv * row_tiles_of(p, r.tokens); };
  int mine = 0;
  for (int b = b0; b < b1; ++b) mine += work_of(request_of(p, b));
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) warp_sum[warp] = incl;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  int before = incl - mine, total = 0;
#pragma unroll
  for (int w = 0; w < NUM_THREADS / 32; ++w) {
    if (w < warp) before += warp_sum[w];
    total += warp_sum[w];
  }
  const Ranges rg(p, total);
  const int range = blockIdx.x / p.row_tiles, member = blockIdx.x % p.row_tiles;
  const bool busy = range < rg.n;
  if (busy) {
    // the range's two ends, by the threads whose requests they fall into
    const int from = rg.start(range), to = rg.start(range + 1);
    for (int e = 0; e < 2; ++e) {
      const int at = e == 0 ? from : to;
      if (at < before || at >= before + mine) continue;
      int t = before;
      for (int b = b0; b < b1; ++b) {
        const Request r = request_of(p, b);
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
  fence_proxy_async_smem();  // the scan's use of the ring's memory comes before its TMA writes
  __syncthreads();
  Walk w;
  w.left = 0;
  if (busy) {
    w.b = plan[0];
    w.kvh = plan[1];
    w.i0 = plan[2];
    w.left = plan[4] - plan[3];
    w.turn = 0;
    w.set(request_of(p, w.b));
    w.settle(p, member);
  }

  if (warp == K_WARP || warp == V_WARP) {
    // ------------------------------ K and V producers ------------------------------
    const bool is_k = warp == K_WARP;
    uint64_t* full = is_k ? k_full : v_full;
    uint64_t* empty = is_k ? k_empty : v_empty;
    uint8_t* ring = smem + (is_k ? L::OFF_K : L::OFF_V);
    const CUtensorMap* map = is_k ? &tmK : &tmV;
    const int box = 1 << p.box_log2;
    const int pages = BN >> p.box_log2;          // boxes of a tile: lane i loads box i
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
        const int st = static_cast<int>(n % RING);
        if (!mbar_wait(&empty[st], ((n / RING) & 1u) ^ 1u, abort_flag, p.status, SITE_PROD_KV)) {
          ok = false;
          break;
        }
        const int held = min(pages, (w.len() - i * BN + box - 1) >> p.box_log2);
        if (lane == 0) {
          mbar_arrive_expect_tx(&full[st], static_cast<uint32_t>(held * group_box * L::GROUP));
        }
        __syncwarp();
        if (lane < held) {
          // the block's first (token, head) row; past the tensor, which reads as zeros, for no block
          int first = p.num_blocks * p.hkv << p.page_log2;
          if (id >= 0 && id < p.num_blocks) {
            first = (id * p.hkv << p.page_log2) + w.kvh;
          } else {
            record_status(p.status, KTA_ERR_DEVICE_BOUNDS, SITE_BLOCK);
          }
          tma_load_5d(map, &full[st], ring + st * L::TILE + lane * group_box * L::GROUP, 0, 0, 0,
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
      for (uint32_t k = n > RING ? n - RING : 0; k < n; ++k) {
        mbar_wait(&full[k % RING], (k / RING) & 1u, &none, p.status, SITE_PROD_KV);
      }
    }
  } else if (warp == Q_WARP) {
    // ------------------------------ Q producer ------------------------------
    if (lane == 0) {
      uint32_t n = 0;  // segments so far: buffer n % q_bufs
      for (; w.left > 0; w.next(p), w.settle(p, member), ++n) {
        const uint32_t buf = n % p.q_bufs, phase = (n / p.q_bufs) & 1u;
        if (!mbar_wait(&q_empty[buf], phase ^ 1u, abort_flag, p.status, SITE_PROD_Q)) break;
        mbar_arrive_expect_tx(&q_full[buf], static_cast<uint32_t>(p.box_tokens * p.group * D * 2));
#pragma unroll
        for (int h = 0; h < L::HALVES; ++h) {
          tma_load_3d(&tmQ, &q_full[buf], smem + L::OFF_Q + h * L::Q_HALF + buf * p.q_shift, h * 64,
                      w.kvh * p.group, w.row + w.row_tile(p, member) * p.tok_tile);
        }
      }
      if (*abort_flag != 0) {
        int none = 0;
        for (uint32_t k = n > static_cast<uint32_t>(p.q_bufs) ? n - p.q_bufs : 0; k < n; ++k) {
          mbar_wait(&q_full[k % p.q_bufs], (k / p.q_bufs) & 1u, &none, p.status, SITE_PROD_Q);
        }
      }
    }
    __syncwarp();
  } else if (warp == MMA_WARP) {
    // ------------------------------ MMA issuer ------------------------------
    constexpr uint32_t FMT = BF16 ? 1u : 0u;
    constexpr uint32_t idesc_s = make_idesc(BM, BN, FMT, FMT, 0u, 0u);  // Q K^T, both K-major
    constexpr uint32_t idesc_o = make_idesc(BM, D, FMT, FMT, 0u, 1u);   // P (TMEM) V (MN-major)
    // w and j run one tile ahead of the PVs, into the next segment: its first S is ready when the
    // softmax warps come from this one's epilogue.
    int j = 0, tiles = w.left > 0 ? w.count(p) : 0;
    uint32_t segment = 0, o_phase = 0;
    bool first_segment = true;
    // S of tile t into buffer t & 1, which holds P of tile t - 2 until its PV has read it: that was
    // issued before and ends before this begins.
    auto issue_s = [&](uint32_t t) -> bool {
      const uint32_t buf = segment % p.q_bufs;
      if (j == 0 && !mbar_wait(&q_full[buf], (segment / p.q_bufs) & 1u, abort_flag, p.status, SITE_MMA_Q)) {
        return false;
      }
      const int st = static_cast<int>(t % RING);
      if (!mbar_wait(&k_full[st], (t / RING) & 1u, abort_flag, p.status, SITE_MMA_K)) return false;
      tc_fence_after();
      const uint64_t qdesc = sdesc_sw128(smem_u32(smem + L::OFF_Q + buf * p.q_shift), 16, 1024);
      const uint64_t kdesc = sdesc_sw128(smem_u32(smem + L::OFF_K + st * L::TILE), 16, L::GROUP);
      if (elect_one_sync()) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t qo = ((kk >> 2) * L::Q_HALF + (kk & 3) * 32) >> 4;
          const uint32_t ko = ((kk >> 2) * 1024 + (kk & 3) * 32) >> 4;
          umma_f16(tmem + (t & 1u) * BN, qdesc + qo, kdesc + ko, idesc_s, kk > 0 ? 1u : 0u);
        }
        umma_commit(&s_full[t & 1u]);
        umma_commit(&k_empty[st]);
        if (j + 1 == tiles) umma_commit(&q_empty[buf]);
      }
      __syncwarp();
      return true;
    };
    bool more = w.left > 0;
    if (more && !issue_s(0)) more = false;
    for (uint32_t g = 0; more; ++g) {  // tile g: S buffer g & 1, its phase (g >> 1) & 1
      const bool first = j == 0, last = j + 1 == tiles;
      if (last) {
        w.next(p);
        w.settle(p, member);
        j = 0;
        tiles = w.left > 0 ? w.count(p) : 0;
        ++segment;
      } else {
        ++j;
      }
      more = w.left > 0;
      if (more && !issue_s(g + 1)) break;
      const int st = static_cast<int>(g % RING);
      if (!mbar_wait(&v_full[st], (g / RING) & 1u, abort_flag, p.status, SITE_MMA_V)) break;
      const uint64_t vdesc = sdesc_sw128(smem_u32(smem + L::OFF_V + st * L::TILE), 1024, L::GROUP);
      bool ok = true;
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // the warpgroups' halves of the keys, into their own O
        ok = ok && mbar_wait(&p_full[2 * (g & 1u) + h], (g >> 1) & 1u, abort_flag, p.status, SITE_MMA_P);
        if (first && h == 0 && !first_segment) {  // the last segment's O has been read
          ok = ok && mbar_wait(o_free, o_phase, abort_flag, p.status, SITE_MMA_OFREE);
          o_phase ^= 1u;
        }
        if (!ok) break;
        tc_fence_after();
        if (elect_one_sync()) {
#pragma unroll
          for (int kk = 0; kk < HK / 16; ++kk) {
            umma_f16_tmem_a(tmem + COL_O + h * BN, tmem + (g & 1u) * BN + h * HK + kk * 8,
                            vdesc + static_cast<uint64_t>((h * HK / 16 + kk) * 2 * L::GROUP / 16),
                            idesc_o, (!first || kk > 0) ? 1u : 0u);
          }
          umma_commit(&pv_done[h]);
          if (h == 1) umma_commit(&v_empty[st]);
          if (h == 1 && last) umma_commit(o_done);
        }
        __syncwarp();
      }
      if (!ok) break;
      if (last) first_segment = false;
    }
  } else {
    // ------------- softmax, O correction and epilogue (thread = query row) -------------
    const int wg = warp >> 2, quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t t_s = tmem + lane_base + wg * HK;  // this half of S buffer 0
    const uint32_t t_o = tmem + lane_base + COL_O;    // O of warpgroup 0; the other's is BN columns on
    const float sl = p.scale_log2;
    uint32_t g = 0;  // tiles of keys so far
    uint32_t o_phase = 0;
    bool ok = true;
    if (threadIdx.x == 0) p.desc[blockIdx.x] = Desc{};  // no unit to join so far
    for (bool first_part = true; w.left > 0 && ok; w.next(p), w.settle(p, member), first_part = false) {
      const int rt = w.row_tile(p, member);
      const int tokens = w.rows(p, rt);
      const int rows = tokens * p.group;
      const bool live = row < rows;
      const bool warp_on = quarter * 32 < rows;
      uint64_t bits = 0;
      if (live) {
        const int t = rt * p.tok_tile + row / p.group;
        bits = p.tree != nullptr ? static_cast<uint64_t>(p.tree[w.row + t])
                                 : (2ull << t) - 1ull;  // t = 63: all ones
        if (w.tokens < 64) bits &= (1ull << w.tokens) - 1ull;
      }
      const int tiles = w.count(p);
      float m_used = -INFINITY, lsum = 0.f;
      for (int j = 0; j < tiles; ++j, ++g) {
        const int k0 = (w.i0 + j) * BN;
        const bool masked = k0 + BN > w.ctx;
        if (masked) {
          const int st = static_cast<int>(g % RING);
          if (!mbar_wait(&v_full[st], (g / RING) & 1u, abort_flag, p.status, SITE_SM_V)) {
            ok = false;
            break;
          }
          clean_v<BF16, D>(smem + L::OFF_V + st * L::TILE, wg * HK, w.ctx - k0, w.len() - k0, k0 - w.ctx,
                           row, bad);
          fence_proxy_async_smem();
        }
        if (!mbar_wait(&s_full[g & 1u], (g >> 1) & 1u, abort_flag, p.status, SITE_SM_S)) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (warp_on) {
          const uint32_t at = t_s + (g & 1u) * BN;
          uint32_t view[2];
          if (masked) {
            view[0] = view_word(bits, k0 + wg * HK - w.ctx);
            view[1] = view_word(bits, k0 + wg * HK + 32 - w.ctx);
            ok = softmax_step<true, BF16, D>(at, t_o + wg * BN, view, sl, m_used, lsum, &pv_done[wg],
                                             (g - 1) & 1u, abort_flag, p.status);
          } else {
            ok = softmax_step<false, BF16, D>(at, t_o + wg * BN, view, sl, m_used, lsum, &pv_done[wg],
                                              (g - 1) & 1u, abort_flag, p.status);
          }
          if (!ok) break;
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[2 * (g & 1u) + wg]);
      }
      if (!ok) break;
      // ---- epilogue: the two warpgroups' states become one, each for half of D ----
      ml[wg * BM + row] = make_float2(m_used, lsum);
      __syncwarp();
      if (lane == 0) mbar_arrive(ml_full);
      if (!mbar_wait(ml_full, o_phase, abort_flag, p.status, SITE_SM_ML)) break;
      if (!mbar_wait(o_done, o_phase, abort_flag, p.status, SITE_SM_O)) break;
      o_phase ^= 1u;
      tc_fence_after();
      const bool whole = w.i0 == 0 && tiles == w.tiles();
      const int slot = 2 * static_cast<int>(blockIdx.x) + (first_part ? 0 : 1);
      const int tok = row / p.group, head = row - tok * p.group;
      const int token = w.row + rt * p.tok_tile + tok;
      const int q_head = w.kvh * p.group + head;
      const uint64_t lost = bits & (static_cast<uint64_t>(bad[1]) << 32 | bad[0]);
      if (warp_on) {
        const float2 a = ml[row], b = ml[BM + row];
        const float m = fmaxf(a.x, b.x);
        const float base = m == -INFINITY ? 0.f : m;
        float wa = ex2(a.x - base), wb = ex2(b.x - base);
        const float l = fmaf(wa, a.y, wb * b.y);
        if (whole) {  // a row that sees nothing: O = 0
          const float inv = l == 0.f ? 0.f : 1.f / l;
          wa *= inv;
          wb *= inv;
        }
#pragma unroll 1
        for (int c = wg * (D / 2); c < (wg + 1) * (D / 2); c += 32) {
          uint32_t o[32], o1[32];
          tmem_ld_32x32b_x32(t_o + c, o);
          tmem_ld_32x32b_x32(t_o + BN + c, o1);
          tmem_ld_wait();
          reg_fence(o);
          reg_fence(o1);
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            o[i] = __float_as_uint(fmaf(__uint_as_float(o[i]), wa, __uint_as_float(o1[i]) * wb));
          }
          if (live && lost != 0) {
            // drafted V elements that are not finite, for the rows that see them
            for (uint64_t left = lost; left != 0; left &= left - 1) {
              const int key = w.ctx + __ffsll(static_cast<long long>(left)) - 1;
              if (key < w.i0 * BN || key >= (w.i0 + tiles) * BN) continue;
              const int id = p.tables[w.b * p.table_stride + (key >> p.page_log2)];
              if (id < 0 || id >= p.num_blocks) continue;
              const long long at =
                  (((static_cast<long long>(id) << p.page_log2) + (key & ((1 << p.page_log2) - 1))) *
                       p.hkv + w.kvh) * D + c;
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                const float v = load16<BF16>(p.v, at + i);
                if (!isfinite(v)) o[i] = __float_as_uint(__uint_as_float(o[i]) + v);
              }
            }
          }
          if (live && whole) {
            uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) +
                                                  (static_cast<long long>(token) * p.hq + q_head) * D + c);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t pk[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                pk[e] = pack2<BF16>(__uint_as_float(o[8 * i + 2 * e]), __uint_as_float(o[8 * i + 2 * e + 1]));
              }
              dst[i] = make_uint4(pk[0], pk[1], pk[2], pk[3]);
            }
          } else if (live) {
            float4* dst = p.part_o + (static_cast<long long>(slot) * (D / 4) + c / 4) * p.row_cap + row;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              dst[i * p.row_cap] =
                  make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]),
                              __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3]));
            }
          }
        }
        if (wg == 0 && live && whole) {
          p.lse[static_cast<long long>(token) * p.hq + q_head] =
              l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
        } else if (wg == 0 && live) {
          p.part_ml[static_cast<long long>(slot) * p.row_cap + row] = make_float2(m, l);
        }
      }
      if (threadIdx.x == 0 && !whole && w.i0 == 0) {  // the unit starts here: this CTA describes it
        const Ranges r(p, plan[5]);
        const int end = plan[4] - w.left + w.tiles() * row_tiles_of(p, w.tokens);  // of the unit
        Desc d = {};
        d.count = r.owner_before(end) - range + 1;
        d.slot = slot;
        d.next = (range + 1) * p.row_tiles + rt;  // a range's first segment is row tile = member
        d.row = w.row + rt * p.tok_tile;
        d.tokens = tokens;
        d.kvh = w.kvh;
        p.desc[blockIdx.x] = d;
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(o_free);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == MMA_WARP) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the parts of a unit that several ranges hold: M = max m, O = sum 2^(m - M) O_part /
// sum 2^(m - M) l. Block (x, y): the unit that starts in CTA x, part y of its elements; a thread
// takes four elements of a row, rows of a warp back to back, eight parts' loads at a time.
constexpr int JOIN_THREADS = 128;
constexpr int JOIN_PARTS = 8;

template <bool BF16, int D>
__global__ void __launch_bounds__(JOIN_THREADS) join_kernel(const Params p) {
  pdl_launch_dependents();
  pdl_wait();
  const Desc d = p.desc[blockIdx.x];
  if (d.count == 0) return;
  const int rows = d.tokens * p.group;
  const int items = rows * (D / 4);
  for (int item = blockIdx.y * JOIN_THREADS + threadIdx.x; item < items;
       item += gridDim.y * JOIN_THREADS) {
    const int d4 = item / rows, row = item - d4 * rows;
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c0 = 0; c0 < d.count; c0 += JOIN_PARTS) {
      float2 ml[JOIN_PARTS];
      float4 part[JOIN_PARTS];
#pragma unroll
      for (int i = 0; i < JOIN_PARTS; ++i) {
        const int c = c0 + i;
        ml[i] = make_float2(-INFINITY, 0.f);
        part[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (c < d.count) {
          const long long slot = c == 0 ? d.slot : 2LL * (d.next + (c - 1) * p.row_tiles);
          ml[i] = __ldcg(p.part_ml + slot * p.row_cap + row);
          part[i] = __ldcg(p.part_o + (slot * (D / 4) + d4) * p.row_cap + row);
        }
      }
      float top = m;
#pragma unroll
      for (int i = 0; i < JOIN_PARTS; ++i) top = fmaxf(top, ml[i].x);
      const float base = top == -INFINITY ? 0.f : top;
      const float keep = exp2f(m - base);
      l *= keep;
      o.x *= keep;
      o.y *= keep;
      o.z *= keep;
      o.w *= keep;
#pragma unroll
      for (int i = 0; i < JOIN_PARTS; ++i) {
        if (c0 + i >= d.count) continue;
        const float wt = exp2f(ml[i].x - base);
        l = fmaf(wt, ml[i].y, l);
        o.x = fmaf(wt, part[i].x, o.x);
        o.y = fmaf(wt, part[i].y, o.y);
        o.z = fmaf(wt, part[i].z, o.z);
        o.w = fmaf(wt, part[i].w, o.w);
      }
      m = top;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int tok = row / p.group;
    const long long at =
        static_cast<long long>(d.row + tok) * p.hq + d.kvh * p.group + (row - tok * p.group);
    uint2* dst = reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at * D + d4 * 4);
    *dst = make_uint2(pack2<BF16>(o.x * inv, o.y * inv), pack2<BF16>(o.z * inv, o.w * inv));
    if (d4 == 0) p.lse[at] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
  }
}

// Workspace: descriptors, (maximum, sum) and O of two partial units of every CTA.
struct Workspace {
  size_t off_ml, off_o, total;
  int row_cap;
  Workspace(long long max_new, long long group, long long D) {
    const long long tile = BM / group;
    row_cap = static_cast<int>((std::min(tile, max_new) * group + 7) / 8 * 8);
    off_ml = sizeof(Desc) * MAX_CTAS;
    off_o = off_ml + sizeof(float2) * 2 * MAX_CTAS * row_cap;
    total = off_o + sizeof(float) * 2 * MAX_CTAS * static_cast<size_t>(row_cap) * D;
  }
};

bool sizes_ok(int64_t max_new, int64_t Hq, int64_t Hkv, int64_t D) {
  return max_new > 0 && max_new <= MAX_DRAFT && Hq > 0 && Hkv > 0 && Hq % Hkv == 0 &&
         Hq / Hkv <= MAX_GROUP && (D == 64 || D == 128);
}

template <bool BF16, int D>
int go(Params& p, const void* Q, const void* Kc, const void* Vc, int64_t q_token, cudaStream_t stream) {
  using L = Layout<D>;
  const CUtensorMapDataType type = BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  CUtensorMap tq, tk, tv;
  {
    const uint64_t dims[3] = {D, static_cast<uint64_t>(p.hq), static_cast<uint64_t>(p.rows)};
    const uint64_t strides[2] = {D * 2, static_cast<uint64_t>(q_token) * 2};
    const uint32_t box[3] = {64, static_cast<uint32_t>(p.group), static_cast<uint32_t>(p.box_tokens)};
    const int s = encode_tmap(&tq, type, 3, Q, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
    if (s != KTA_OK) return s;
  }
  // A block of a head: (64 d, 8 tokens, half, group of 8 tokens), and the (token, head) row at
  // which it starts.
  const uint64_t page = uint64_t{1} << p.page_log2, token = static_cast<uint64_t>(p.hkv) * D * 2;
  const uint64_t dims[5] = {64, 8, L::HALVES, page / 8, static_cast<uint64_t>(p.num_blocks) * page * p.hkv};
  const uint64_t strides[4] = {token, 128, 8 * token, D * 2};
  const uint32_t box[5] = {64, 8, L::HALVES, (1u << p.box_log2) / 8, 1};
  int s = encode_tmap(&tk, type, 5, Kc, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  if (s != KTA_OK) return s;
  s = encode_tmap(&tv, type, 5, Vc, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  if (s != KTA_OK) return s;
  auto kernel = tree_kernel<BF16, D>;
  s = set_kernel_smem(reinterpret_cast<const void*>(kernel), L::TOTAL);
  if (s != KTA_OK) return s;
  const int sms = std::min(current_sm_count(), MAX_CTAS);
  if (sms < p.row_tiles) return KTA_ERR_UNSUPPORTED;
  const int grid = sms / p.row_tiles * p.row_tiles;
  s = launch_ex(kernel, dim3(grid), dim3(NUM_THREADS), L::TOTAL, stream, 1, tq, tk, tv, p);
  if (s != KTA_OK) return s;
  // four elements a thread and at most four passes
  const int parts = std::max(1, std::min(8, p.row_cap * (D / 4) / (2 * JOIN_THREADS)));
  return launch_ex(join_kernel<BF16, D>, dim3(grid, parts), dim3(JOIN_THREADS), 0, stream, 1, p);
}

template <bool BF16>
int launch(const void* Q, const void* Kc, const void* Vc, const void* tables, const void* ctx,
           const void* offsets, const void* tree, void* O, void* LSE, int64_t tokens, int64_t B,
           int64_t Hq, int64_t Hkv, int64_t D, int64_t q_token, int64_t num_blocks, int64_t block,
           int64_t max_blocks, int64_t table_stride, int64_t max_new, float scale, void* workspace,
           size_t ws_bytes, cudaStream_t stream) {
  if (!Q || !Kc || !Vc || !tables || !ctx || !offsets || !O || !LSE) return KTA_ERR_INVALID_ARG;
  if (tokens <= 0 || B <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0 || num_blocks <= 0 || block <= 0 ||
      max_blocks <= 0 || max_new <= 0) {
    return KTA_ERR_INVALID_ARG;
  }
  if (!(scale > 0.f) || !std::isfinite(scale)) return KTA_ERR_INVALID_ARG;
  if (B > 1 && table_stride < max_blocks) return KTA_ERR_INVALID_ARG;
  if (!sizes_ok(max_new, Hq, Hkv, D) || B > MAX_BATCH) return KTA_ERR_UNSUPPORTED;
  if (block < 8 || block > 256 || (block & (block - 1)) != 0) return KTA_ERR_UNSUPPORTED;
  // key positions, rows and (token, head) rows of the cache stay in int32
  if (max_blocks > (1LL << 30) / block || tokens > (1LL << 30) || Hq > 65536 ||
      num_blocks > ((1LL << 31) - 1) / (block * Hkv)) {
    return KTA_ERR_UNSUPPORTED;
  }
  // and so does the work list: every request's tiles of keys, for each KV head and row tile
  const long long row_tiles = (max_new + BM / (Hq / Hkv) - 1) / (BM / (Hq / Hkv));
  if (B * Hkv * row_tiles * ((max_blocks * block + BN - 1) / BN) > (1LL << 31) - 1) {
    return KTA_ERR_UNSUPPORTED;
  }
  if (q_token < Hq * D) return KTA_ERR_INVALID_ARG;
  if (q_token % 8 != 0 || !aligned16(Q) || !aligned16(Kc) || !aligned16(Vc) || !aligned16(O)) {
    return KTA_ERR_ALIGN;
  }
  for (const void* q : {tables, ctx, offsets, static_cast<const void*>(LSE)}) {
    if (reinterpret_cast<uintptr_t>(q) & 3) return KTA_ERR_ALIGN;
  }
  if (reinterpret_cast<uintptr_t>(tree) & 7) return KTA_ERR_ALIGN;
  const long long group = Hq / Hkv;
  const Workspace ws(max_new, group, D);
  if (workspace == nullptr || ws_bytes < ws.total || !aligned16(workspace)) return KTA_ERR_WORKSPACE;
  int s = require_sm100();
  if (s != KTA_OK) return s;
  Params p = {};
  p.ctx = static_cast<const int32_t*>(ctx);
  p.offsets = static_cast<const int32_t*>(offsets);
  p.tree = static_cast<const int64_t*>(tree);
  p.tables = static_cast<const int32_t*>(tables);
  p.out = O;
  p.lse = static_cast<float*>(LSE);
  p.v = Vc;
  uint8_t* base = static_cast<uint8_t*>(workspace);
  p.desc = reinterpret_cast<Desc*>(base);
  p.part_ml = reinterpret_cast<float2*>(base + ws.off_ml);
  p.part_o = reinterpret_cast<float4*>(base + ws.off_o);
  p.table_stride = table_stride;
  p.batch = static_cast<int>(B);
  p.rows = static_cast<int>(tokens);
  p.hq = static_cast<int>(Hq);
  p.hkv = static_cast<int>(Hkv);
  p.group = static_cast<int>(group);
  p.max_new = static_cast<int>(max_new);
  p.max_blocks = static_cast<int>(max_blocks);
  p.num_blocks = static_cast<int>(num_blocks);
  while ((int64_t{1} << p.page_log2) < block) ++p.page_log2;
  p.box_log2 = std::min(p.page_log2, 7);
  p.tok_tile = BM / p.group;
  p.box_tokens = std::min(p.tok_tile, p.max_new);
  p.row_tiles = static_cast<int>(row_tiles);
  // two Q tiles where they fit (64 rows): the next segment's Q then comes while this one runs
  const int q_rows = (p.box_tokens * p.group + 7) / 8 * 8;
  p.q_bufs = q_rows <= BM / 2 ? 2 : 1;
  p.q_shift = BM / 2 * 128;
  p.row_cap = ws.row_cap;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.status = device_status_ptr();
  if (D == 64) return go<BF16, 64>(p, Q, Kc, Vc, q_token, stream);
  return go<BF16, 128>(p, Q, Kc, Vc, q_token, stream);
}

}  // namespace tree
}  // namespace kta

extern "C" size_t kta_tree_attn_workspace_bytes(int64_t max_new, int64_t Hq, int64_t Hkv, int64_t D) {
  if (!kta::tree::sizes_ok(max_new, Hq, Hkv, D)) return 0;
  return kta::tree::Workspace(max_new, Hq / Hkv, D).total;
}

#define KTA_TREE_ENTRY(NAME, BF16)                                                                  \
  extern "C" int kta_tree_attn_##NAME(                                                              \
      const void* Q, const void* Kc, const void* Vc, const void* block_tables,                      \
      const void* context_lens, const void* offsets, const void* tree, void* O, void* LSE,          \
      int64_t tokens, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t q_token,               \
      int64_t num_blocks, int64_t block_size, int64_t max_blocks, int64_t table_stride,             \
      int64_t max_new, float scale, void* workspace, size_t ws_bytes, void* stream) {               \
    return kta::tree::launch<BF16>(Q, Kc, Vc, block_tables, context_lens, offsets, tree, O, LSE,    \
                                   tokens, B, Hq, Hkv, D, q_token, num_blocks, block_size,          \
                                   max_blocks, table_stride, max_new, scale, workspace, ws_bytes,   \
                                   static_cast<cudaStream_t>(stream));                              \
  }

KTA_TREE_ENTRY(f16, false)
KTA_TREE_ENTRY(bf16, true)
