// Attention of a tree of drafted tokens over a paged KV cache, sm_100a.
//
//   For request b with c = ctx[b] tokens in the cache and t drafted ones behind them (rows
//   offsets[b] .. offsets[b + 1] of Q, keys c .. c + t - 1 of the cache, t <= 64):
//   row i sees key p iff p < c, or bit p - c of tree[i] is set (p - c < t);
//   O = softmax(scale Q K^T over the seen keys) V,  LSE = log of the sum, natural.
//
// One drafted token is the decode step of a paged cache; a chain is the tree 1, 11, 111, ...
//
// Two kernels compute it, by the query rows of a KV head that a request can have (drafted tokens x
// heads of the group): up to 32 of them are the narrow side of the products (tree_narrow.cu), more are
// row tiles of 128 (wide_kernel here). Common to both:
//
//   * Work is the list of 128-key tiles of every (request, KV head), in equal shares, one for a CTA
//     (or for `row_tiles` CTAs, which take the row tiles of the share's units in turn and find each
//     other's K and V in L2). What a share cuts is joined by a second small kernel from fp32 partials
//     (O, maximum, sum) in the workspace: no counters to keep at zero between calls, no order of
//     arrival in the result. Every CTA finds its share by itself from the lengths (a separate plan
//     kernel: 9 to 13 us more; the last arriver joining instead of a kernel: 22 us where one request
//     of 8 tokens over 1003 keys takes 11.2).
//   * Pages: a box of the tensor map is one page (up to 128 tokens) of one head, with the token
//     index split as (8, page / 8): shared memory gets 8-token groups of both 64-wide halves of
//     the head, [group][half][8 tokens][128 B], which for every page size is one uniform stride
//     for the matrix descriptors and one TMA per page. Lane i of the producer loads page i.
//   * The last tile of a request ends inside a page: K's leftover columns are masked by
//     selection, and V's leftover rows are set to zero in shared memory, since 0 * NaN from a
//     page's unwritten rows would reach every row through the matrix product. Likewise a drafted
//     V row that is not finite is zeroed and handed to the rows that see it alone.
//   * The weights are rounded to the storage type for the product with V (the sums are taken before):
//     O is off by 0.0023 of its norm in bf16 and 0.00029 in f16, where its own rounding alone gives
//     0.0017 and 0.00021. With what the rounding leaves as a second operand O has the smaller error,
//     but wide_kernel, whose tensor pipe is under the power cap, takes 506 us for 403 (32 trees of 33 to
//     64 tokens), and in tree_narrow.cu, with both in one product of twice the columns, long requests
//     of heads of 128 cost nothing, but one request of 8 tokens 5 %, 148 over 100 keys 8 to 15 %, and 32
//     rows of heads of 64 13 % (193 us, 218). Not taken: attn.cu and decode.cu round them as well.
//   * Out-of-range lengths, offsets and block ids become status KTA_ERR_DEVICE_BOUNDS: such a
//     request's rows are zero (LSE -inf), such a block reads as zeros. Every wait is bounded.
//
// wide_kernel, tensor- and power-bound. 32 trees of 33 to 64 tokens with 8 heads to a KV head, over
// 2048 to 8192 keys: 404 us in a long run of calls (690 TFLOP/s of the rows that exist, 14 % more with
// their padding), 344 to 375 in short ones, the SMs at 1.54 to 1.6 GHz under the 1000 W cap and ~1930
// cycles to a 128 x 128 tile.
//
//   * Warps 0-3 and 4-7 are two softmax warpgroups: each takes 64 keys of every tile (thread = query
//     row = TMEM lane) and has its own O, maximum and sum, so that neither waits for the other before
//     the segment's end, where the states are joined through shared memory. A row of 64 in registers
//     leaves room for P and two S buffers: S of the next tile is computed beside the softmax.
//   * The two warps of a scheduler take turns with their exponentials (`turn`): the one's loads, maxima
//     and stores run beside the other's MUFU work (402 us sustained, 412 in step).
//   * Warp 8 issues the MMAs (S = Q K^T from shared memory, O += P V with P in the S columns of
//     TMEM), warps 9-11 produce K, V and Q. K and V have rings of three tiles each.
//   * Measured and not kept: two row tiles to a CTA over shared K and V, a warpgroup each (355
//     against 349 us in one run, 417 against 384 at 64 tokens to a tree); S issued for 64 keys at a
//     time (407 to 418 against 395); a part of the exponentials on the FMA pipe, whose power costs
//     more clock than the wait for the MUFU pipe (437 against 423 sustained).
#include <algorithm>
#include <cmath>

#include "tree_common.cuh"

namespace kta {
namespace tree {

constexpr int RING = 3;               // K tiles in flight, and V tiles
constexpr int HK = BN / 2;            // keys of a tile that a softmax warpgroup takes
constexpr int SOFTMAX_WARPS = 8;      // two warpgroups
constexpr uint32_t COL_O = 256;       // TMEM: S buffer i at i * 128, O of warpgroup w at 256 + w * 128

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
  // k_full[R], k_empty[R], v_full[R], v_empty[R], q_full, q_empty, s_full[2], p_full[2][2],
  // pv_done[2], ml_full, ml_empty, o_done, o_free, turn[8]
  static constexpr int NUM_BARS = 4 * RING + 22;
  static constexpr int OFF_MISC = OFF_BAR + NUM_BARS * 8;
  static constexpr int OFF_PLAN = OFF_MISC + 16;  // after tmem base, abort, non-finite drafts [2]
  static constexpr int TOTAL = OFF_PLAN + PLAN_BYTES;
  static_assert(TOTAL <= 232448, "shared memory budget of one sm_100 CTA");
};

// Half an S tile of one query row (64 keys; this thread's TMEM lane): P = 2^(S sl - m) over the
// first 32 columns, the running maximum m (log2 units) and the row sum l of this half. m moves only
// when the true maximum grew by more than 2^8, so O is rescaled rarely; that waits for the PV
// before. The exponentials start with this warp's turn and then hand it to `other`'s.
// pv_done is at most one phase behind: S of this tile was issued behind the PV before that.
template <bool MASKED, bool BF16, int D>
__device__ __forceinline__ bool softmax_step(uint32_t t_s, uint32_t t_o, const uint32_t (&view)[2],
                                             float sl, float& m_used, float& lsum, uint64_t* pv_done,
                                             uint32_t pv_parity, uint64_t* turn, uint64_t* other,
                                             uint32_t turn_parity, volatile int* abort,
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
    if (!wait_for(pv_done, pv_parity, abort, status, SITE_SM_PV)) return false;
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
  if (!wait_for(turn, turn_parity, abort, status, SITE_SM_TURN)) return false;
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
    pk[i] = pack2<BF16>(e0, e1);  // rounded as the head of this file explains; the sum is of e
  }
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(other);
  tmem_st_32x32b_x32(t_s, pk);
  tmem_st_wait();
  const uint64_t s01 = add2(add2(sum2[0], sum2[1]), add2(sum2[2], sum2[3]));
  float s0, s1;
  f2_split(s01, s0, s1);
  lsum += s0 + s1;
  return true;
}

// 32 bytes, 32-byte aligned
__device__ __forceinline__ void st_global_v8(void* dst, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(v[0]), "r"(v[1]),
               "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

template <bool BF16, int D>
__global__ void __launch_bounds__(NUM_THREADS, 1)
    wide_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
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
  uint64_t* q_full = v_empty + RING;
  uint64_t* q_empty = q_full + 1;    // the segment's last S has read Q
  uint64_t* s_full = q_empty + 1;    // [S buffer]
  uint64_t* p_full = s_full + 2;     // [buffer][warpgroup]: its half of P written, of V cleaned
  uint64_t* pv_done = p_full + 4;    // [warpgroup]: one phase for each PV into its O
  uint64_t* ml_full = pv_done + 2;   // both warpgroups' maxima and sums are in shared memory
  uint64_t* ml_empty = ml_full + 1;  // ... and read
  uint64_t* o_done = ml_empty + 1;   // the segment's last PV
  uint64_t* o_free = o_done + 1;     // the epilogue has read both O
  uint64_t* turn = o_free + 1;       // [softmax warp]: the exponentials of a tile are its own
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + L::OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::OFF_MISC + 4);
  unsigned int* bad = reinterpret_cast<unsigned int*>(smem + L::OFF_MISC + 8);   // [2]
  float2* ml = reinterpret_cast<float2*>(smem + L::OFF_ML);

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
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[2 * i], SOFTMAX_WARPS / 2);
      mbar_init(&p_full[2 * i + 1], SOFTMAX_WARPS / 2);
      mbar_init(&pv_done[i], 1);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    mbar_init(ml_full, SOFTMAX_WARPS);
    mbar_init(ml_empty, SOFTMAX_WARPS);
    mbar_init(o_done, 1);
    mbar_init(o_free, SOFTMAX_WARPS);
    for (int i = 0; i < SOFTMAX_WARPS; ++i) mbar_init(&turn[i], 1);
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
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  pdl_wait();  // the previous grid's writes (this launch's inputs) are visible from here on
  // after the wait: the join kernel may be scheduled now, and waits for this grid itself
  pdl_launch_dependents();
  Walk<false> w = plan<D, false>(p, smem + L::OFF_PLAN);
  // K and V that one row tile reads once leave L2 first (64 requests of 8 tokens, 8 heads to a KV head,
  // 1024 to 8192 keys: 197 us, 205 without); members of a share find them there.
  const uint64_t policy = p.row_tiles > 1 ? l2_policy_evict_normal() : l2_policy_evict_first();

  if (warp == K_WARP) {
    produce_kv(p, w, Loader<D, RING>{&tmK, smem + L::OFF_K, k_full, k_empty, abort_flag,
                                     policy, 0u, 0, 0});
  } else if (warp == V_WARP) {
    produce_kv(p, w, Loader<D, RING>{&tmV, smem + L::OFF_V, v_full, v_empty, abort_flag,
                                     policy, 0u, 0, 0});
  } else if (warp == Q_WARP) {
    produce_q<D, 1>(p, w, &tmQ, smem + L::OFF_Q, 0, L::Q_HALF, q_full, q_empty, abort_flag);
  } else if (warp == MMA_WARP) {
    // ------------------------------ MMA issuer ------------------------------
    constexpr uint32_t FMT = BF16 ? 1u : 0u;
    constexpr uint32_t idesc_s = make_idesc(BM, BN, FMT, FMT, 0u, 0u);  // Q K^T, both K-major
    constexpr uint32_t idesc_o = make_idesc(BM, D, FMT, FMT, 0u, 1u);   // P (TMEM) V (MN-major)
    // w and j run one tile ahead of the PVs, into the next segment: its first S is ready when the
    // softmax warps come from this one's epilogue.
    const uint64_t qdesc = sdesc_sw128(smem_u32(smem + L::OFF_Q), 16, 1024);
    int j = 0, tiles = w.left > 0 ? w.count() : 0;
    uint32_t segment = 0, o_phase = 0;
    bool first_segment = true;
    // S of tile t into buffer t & 1, which holds P of tile t - 2 until its PV has read it: that was
    // issued before and ends before this begins.
    auto issue_s = [&](uint32_t t) -> bool {
      if (j == 0 && !wait_for(q_full, segment & 1u, abort_flag, p.status, SITE_MMA_Q)) return false;
      const int st = static_cast<int>(t % RING);
      if (!wait_for(&k_full[st], (t / RING) & 1u, abort_flag, p.status, SITE_MMA_K)) return false;
      tc_fence_after();
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
        if (j + 1 == tiles) umma_commit(q_empty);
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
        j = 0;
        tiles = w.left > 0 ? w.count() : 0;
        ++segment;
      } else {
        ++j;
      }
      more = w.left > 0;
      if (more && !issue_s(g + 1)) break;
      const int st = static_cast<int>(g % RING);
      if (!wait_for(&v_full[st], (g / RING) & 1u, abort_flag, p.status, SITE_MMA_V)) break;
      const uint64_t vdesc = sdesc_sw128(smem_u32(smem + L::OFF_V + st * L::TILE), 1024, L::GROUP);
      bool ok = true;
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // the warpgroups' halves of the keys, into their own O
        ok = ok && wait_for(&p_full[2 * (g & 1u) + h], (g >> 1) & 1u, abort_flag, p.status, SITE_MMA_P);
        if (first && h == 0 && !first_segment) {  // the last segment's O has been read
          ok = ok && wait_for(o_free, o_phase, abort_flag, p.status, SITE_MMA_OFREE);
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
    const int tok = row / p.group, head = row - tok * p.group;
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t t_s = tmem + lane_base + wg * HK;  // this half of S buffer 0
    const uint32_t t_o = tmem + lane_base + COL_O;    // O of warpgroup 0; the other's is BN columns on
    const float sl = p.scale_log2;
    uint32_t g = 0;  // tiles of keys so far
    uint32_t turns = 0;
    uint32_t o_phase = 0;
    bool ok = true;
    // what this thread's row of a segment sees
    auto bits_at = [&](const Walk<false>& v) -> uint64_t {
      if (v.left <= 0 || row >= v.rows(p) * p.group) return 0ull;
      return bits_of(p, v.row, v.row_tile(p) * p.tok_tile + tok, v.tokens);
    };
    uint64_t bits = bits_at(w);
    while (w.left > 0 && ok) {
      const int rt = w.row_tile(p);
      const int tokens = w.rows(p);
      const int rows = tokens * p.group;
      const bool live = row < rows;
      const bool warp_on = quarter * 32 < rows;
      const int tiles = w.count();
      float m_used = -INFINITY, lsum = 0.f;
      for (int j = 0; j < tiles; ++j, ++g) {
        const int k0 = (w.i0 + j) * BN;
        const bool masked = k0 + BN > w.ctx;
        if (!wait_for(&s_full[g & 1u], (g >> 1) & 1u, abort_flag, p.status, SITE_SM_S)) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (masked) {
          // behind S of this tile: the V tile before in this place has been waited for by then, so that
          // the phase is the right one
          const int st = static_cast<int>(g % RING);
          if (!wait_for(&v_full[st], (g / RING) & 1u, abort_flag, p.status, SITE_SM_V)) {
            ok = false;
            break;
          }
          clean_v<BF16, D>(smem + L::OFF_V + st * L::TILE, wg * HK, HK, w.ctx - k0, w.len() - k0, k0 - w.ctx,
                           row, bad);
          fence_proxy_async_smem();
        }
        if (warp_on) {
          const uint32_t at = t_s + (g & 1u) * BN;
          uint32_t view[2];
          if (masked) {
            view[0] = view_word(bits, k0 + wg * HK - w.ctx);
            view[1] = view_word(bits, k0 + wg * HK + 32 - w.ctx);
            ok = softmax_step<true, BF16, D>(at, t_o + wg * BN, view, sl, m_used, lsum, &pv_done[wg],
                                             (g - 1) & 1u, &turn[warp], &turn[warp ^ 4],
                                              (turns + wg + 1) & 1u, abort_flag, p.status);
          } else {
            ok = softmax_step<false, BF16, D>(at, t_o + wg * BN, view, sl, m_used, lsum, &pv_done[wg],
                                              (g - 1) & 1u, &turn[warp], &turn[warp ^ 4],
                                              (turns + wg + 1) & 1u, abort_flag, p.status);
          }
          ++turns;
          if (!ok) break;
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[2 * (g & 1u) + wg]);
      }
      if (!ok) break;
      // ---- epilogue: the two warpgroups' states become one, each for half of D ----
      Walk<false> following = w;  // its loads come behind the last products
      following.next(p);
      const uint64_t following_bits = bits_at(following);
      if (!wait_for(ml_empty, o_phase ^ 1u, abort_flag, p.status, SITE_SM_ML)) break;
      ml[wg * BM + row] = make_float2(m_used, lsum);
      __syncwarp();
      if (lane == 0) mbar_arrive(ml_full);
      if (!wait_for(ml_full, o_phase, abort_flag, p.status, SITE_SM_ML)) break;
      const float2 ml_a = ml[row], ml_b = ml[BM + row];
      __syncwarp();
      if (lane == 0) mbar_arrive(ml_empty);
      if (!wait_for(o_done, o_phase, abort_flag, p.status, SITE_SM_O)) break;
      o_phase ^= 1u;
      tc_fence_after();
      const bool whole = w.i0 == 0 && tiles == w.tiles();
      const long long slot = slot_of(p, static_cast<int>(blockIdx.x) / p.row_tiles, rt, w.i0 > 0);
      const int token = w.row + rt * p.tok_tile + tok;
      const int q_head = w.kvh * p.group + head;
      const uint64_t lost = bits & (static_cast<uint64_t>(bad[1]) << 32 | bad[0]);
      if (warp_on) {
        const float m = fmaxf(ml_a.x, ml_b.x);
        const float base = m == -INFINITY ? 0.f : m;
        float wa = ex2(ml_a.x - base), wb = ex2(ml_b.x - base);
        const float l = fmaf(wa, ml_a.y, wb * ml_b.y);
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
            uint16_t* dst = static_cast<uint16_t*>(p.out) +
                            (static_cast<long long>(token) * p.hq + q_head) * D + c;
#pragma unroll
            for (int i = 0; i < 2; ++i) {  // a sector at a time
              uint32_t pk[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                pk[e] = pack_o<BF16>(__uint_as_float(o[16 * i + 2 * e]), __uint_as_float(o[16 * i + 2 * e + 1]));
              }
              st_global_v8(dst + 16 * i, pk);
            }
          } else if (live) {
            float4* dst = reinterpret_cast<float4*>(p.part_o) +
                          (slot * (D / 4) + c / 4) * p.row_cap + row;  // a warp's rows back to back
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
          p.part_ml[slot * p.row_cap + row] = make_float2(m, l);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(o_free);
      w = following;
      bits = following_bits;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == MMA_WARP) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the parts of a unit that several shares hold: M = max m, O = sum 2^(m - M) O_part /
// sum 2^(m - M) l, in the shares' order. Block (x, y): the unit that starts in share and row tile x,
// part y of its elements; a thread takes four elements of a row, eight parts' loads at a time.
constexpr int JOIN_THREADS = 128;
constexpr int JOIN_PARTS = 8;

template <bool BF16, int D, bool WIDE>
__global__ void __launch_bounds__(JOIN_THREADS) join_kernel(const Params p) {
  pdl_launch_dependents();
  pdl_wait();
  const Desc d = p.desc[blockIdx.x];
  if (d.span == 0) return;
  const int share = static_cast<int>(blockIdx.x) / p.row_tiles;
  const int rt = static_cast<int>(blockIdx.x) - share * p.row_tiles;
  const int rows = d.tokens * p.group, items = rows * (D / 4);
  for (int item = blockIdx.y * JOIN_THREADS + threadIdx.x; item < items;
       item += gridDim.y * JOIN_THREADS) {
    // in the order that the part's kernel wrote, [d / 4][row] or [row][d / 4]
    const int row = WIDE ? item % rows : item / (D / 4), d4 = WIDE ? item / rows : item % (D / 4);
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c0 = 0; c0 < d.span; c0 += JOIN_PARTS) {
      float2 ml[JOIN_PARTS];
      float4 part[JOIN_PARTS];
#pragma unroll
      for (int i = 0; i < JOIN_PARTS; ++i) {
        const int c = c0 + i;
        ml[i] = make_float2(-INFINITY, 0.f);
        part[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (c < d.span) {
          const long long slot = slot_of(p, share + c, rt, c > 0);
          ml[i] = __ldcg(p.part_ml + slot * p.row_cap + row);
          part[i] = __ldcg(reinterpret_cast<const float4*>(p.part_o) +
                           (WIDE ? (slot * (D / 4) + d4) * p.row_cap + row
                                 : (slot * p.row_cap + row) * (D / 4) + d4));
        }
      }
      float top = m;
#pragma unroll
      for (int i = 0; i < JOIN_PARTS; ++i) top = fmaxf(top, ml[i].x);
      const float base = top == -INFINITY ? 0.f : top;
      const float keep = ex2(m - base);
      l *= keep;
      o = make_float4(o.x * keep, o.y * keep, o.z * keep, o.w * keep);
#pragma unroll
      for (int i = 0; i < JOIN_PARTS; ++i) {
        const float wt = ex2(ml[i].x - base);
        l = fmaf(wt, ml[i].y, l);
        o.x = fmaf(wt, part[i].x, o.x);
        o.y = fmaf(wt, part[i].y, o.y);
        o.z = fmaf(wt, part[i].z, o.z);
        o.w = fmaf(wt, part[i].w, o.w);
      }
      m = top;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;  // a row that sees nothing: O = 0
    const int tok = row / p.group;
    const long long at =
        static_cast<long long>(d.row + tok) * p.hq + d.kvh * p.group + (row - tok * p.group);
    uint2* dst = reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at * D + d4 * 4);
    *dst = make_uint2(pack_o<BF16>(o.x * inv, o.y * inv), pack_o<BF16>(o.z * inv, o.w * inv));
    if (d4 == 0) p.lse[at] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
  }
}

// Workspace: descriptors, and (maximum, sum) and O of two partial units of every share and row tile.
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
  // A token's row of a head is 128 or 256 bytes: promoted to more, L2 would fetch the next head's too
  // (64 x 8000 keys, 8 KV heads of 64: 185 us, 237 with 256 bytes; rings of six tiles there 190; 2 KV
  // heads of 64 over 30000 keys 168 and 217). With one KV head the next row is the next token's: 167 us
  // either way for 64 x 60000 keys. Heads of 128: 325 either way, 64 requests of 8 tokens 196.7 with 256
  // bytes and 197.4 with 128.
  const auto promotion = D == 64 ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B : CU_TENSOR_MAP_L2_PROMOTION_L2_256B;
  int s = encode_tmap(&tk, type, 5, Kc, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, promotion);
  if (s != KTA_OK) return s;
  s = encode_tmap(&tv, type, 5, Vc, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, promotion);
  if (s != KTA_OK) return s;
  const int sms = std::min(current_sm_count(), MAX_CTAS);
  if (sms < p.row_tiles) return KTA_ERR_UNSUPPORTED;
  p.groups = sms / p.row_tiles;
  const int grid = p.groups * p.row_tiles;
  // One tcgen05 tile has 128 rows in wide_kernel however few are real, and 16 or 32 in the other.
  const bool narrow = p.box_tokens * p.group <= NARROW_ROWS;
  if (narrow) {
    s = launch_narrow<BF16, D>(p, tq, tk, tv, grid, stream);
  } else {
    auto kernel = wide_kernel<BF16, D>;
    s = set_kernel_smem(reinterpret_cast<const void*>(kernel), L::TOTAL);
    if (s != KTA_OK) return s;
    s = launch_ex(kernel, dim3(grid), dim3(NUM_THREADS), L::TOTAL, stream, 1, tq, tk, tv, p);
  }
  if (s != KTA_OK) return s;
  // a float4 for a thread, in at most two passes
  const int parts = std::max(1, std::min(16, p.row_cap * (D / 4) / JOIN_THREADS));
  auto join = narrow ? join_kernel<BF16, D, false> : join_kernel<BF16, D, true>;
  return launch_ex(join, dim3(grid, parts), dim3(JOIN_THREADS), 0, stream, 1, p);
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
  const float scale_log2 = scale * 1.4426950408889634f;
  if (!(scale > 0.f) || !std::isfinite(scale_log2)) return KTA_ERR_INVALID_ARG;
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
  if (B * Hkv * row_tiles * ((max_blocks * block + BN - 1) / BN + SWITCH) > (1LL << 31) - 1) {
    return KTA_ERR_UNSUPPORTED;
  }
  if (q_token < Hq * D) return KTA_ERR_INVALID_ARG;
  if (q_token % 8 != 0 || !aligned16(Q) || !aligned16(Kc) || !aligned16(Vc) ||
      (reinterpret_cast<uintptr_t>(O) & 31) != 0) {  // O is written a sector at a time
    return KTA_ERR_ALIGN;
  }
  for (const void* q : {tables, ctx, offsets, static_cast<const void*>(LSE)}) {
    if (reinterpret_cast<uintptr_t>(q) & 3) return KTA_ERR_ALIGN;
  }
  if (reinterpret_cast<uintptr_t>(tree) & 7) return KTA_ERR_ALIGN;
  // a CTA may still read rows of Q where another has written O
  const uintptr_t q0 = reinterpret_cast<uintptr_t>(Q), o0 = reinterpret_cast<uintptr_t>(O);
  const uintptr_t q1 = q0 + 2 * static_cast<uintptr_t>((tokens - 1) * q_token + Hq * D);
  if (o0 < q1 && q0 < o0 + 2 * static_cast<uintptr_t>(tokens * Hq * D)) return KTA_ERR_INVALID_ARG;
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
  p.part_o = reinterpret_cast<float*>(base + ws.off_o);
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
  p.row_cap = ws.row_cap;
  p.scale_log2 = scale_log2;
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
