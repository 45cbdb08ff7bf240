// Tree attention over pages for up to 32 query rows of a KV head (drafted tokens x heads of the
// group): decode steps and small trees, HBM-bound on K and V. The operator, its work list and its
// join are described in tree.cu.
//
// The query rows are the narrow side of both products (N = 16 or 32 instead of 128 lanes that
// are mostly padding), so keys and head dimensions are the 128 lanes:
//
//   S^T [128 keys, N] = K Q^T          (A = K tile, B = Q, both K-major in shared memory)
//   O^T [D, N]       += V^T P^T        (A = V tile, MN-major; B = P, K-major in shared memory)
//
// The tensor work of a key tile falls with N: with 128 rows of padding the SMs run into the 1000 W
// cap at 1260 MHz, and the stream with them. From 33 rows on wide_kernel is faster all the same, since
// the softmax here does a column at a time (64 rows: 235 us with N = 64, 197 there; 32 rows: 196 here,
// 201 there; one request of 32 rows over 1000 keys 15.0 and 16.3).
//
// Measured: 4 x 131071 keys, 8 KV heads, one token of 4 heads: 330 us, 6500 GB/s (396 at 128 rows,
// sustained). 64 requests of 8 tokens x 4 heads over 1k-8k keys, 8 KV heads: 197 us, 6180 GB/s. One
// request of 8 tokens over 1000 keys: 11.2 us with its join, of which the launches and the plan are 5,
// the loads' latency 2, one tile's chain of products and softmax 2, the join 2. 148 single tokens over
// 100 keys: 25 us; a segment is a chain of ~3000 cycles there, a third of it walk and clean-up.
//
//   * Warps 0-3 softmax: warp w has keys 32 w .. 32 w + 31 of every tile, 16 keys at a time in the
//     accumulator layout of 16x256b loads (a thread holds keys lane / 4 + 8 i and neighbouring
//     columns). A column's maximum is only compared, not reduced, while no score exceeds the
//     running one by 2^8; sums stay in the thread's own keys until the segment ends. P goes to
//     shared memory with transposing 8 x 8 stores.
//   * Each softmax warp has its own O accumulator, so no warp waits for another's maximum. Warps
//     4-7 (a quarter of the head dimensions each) scale an accumulator when its warp asks for it,
//     which is rare, and write the segment's result: the four states joined, as the final output
//     or as a partial.
//   * Warp 8 issues the MMAs, warps 9-11 produce K, V and Q by TMA.
#include "tree_common.cuh"

namespace kta {
namespace tree {

constexpr int SOFTMAX_WARPS = 4;
constexpr int OUT_WARPS = 4;  // correction and epilogue

enum : unsigned int {
  SITE_N_MMA_CORR = 0x921,
  SITE_N_SM_P = 0x922,
  SITE_N_SM_ML = 0x923,
  SITE_N_OUT_P = 0x924,
  SITE_N_OUT_PV = 0x925,
  SITE_N_OUT_O = 0x926,
  SITE_N_OUT_ML = 0x927,
};

template <int D, int N>
struct Narrow {
  static constexpr int HALVES = D / 64;
  static constexpr int GROUP = HALVES * 1024;
  static constexpr int TILE = BN / 8 * GROUP;
  static constexpr int RING = 3, Q_BUFS = 2;
  static constexpr int Q_HALF = N * 128;
  static constexpr int Q_BUF = HALVES * Q_HALF;
  static constexpr int P_BUF = 2 * N * 128;  // [64 keys of a half][N rows][128 B]
  static constexpr int OFF_K = 0;
  static constexpr int OFF_V = OFF_K + RING * TILE;
  static constexpr int OFF_Q = OFF_V + RING * TILE;
  static constexpr int OFF_P = OFF_Q + Q_BUFS * Q_BUF;
  static constexpr int OFF_ML = OFF_P + 2 * P_BUF;                   // [warp][N] (maximum, sum)
  static constexpr int OFF_FACTOR = OFF_ML + SOFTMAX_WARPS * N * 8;  // [buffer][warp][N]
  static constexpr int OFF_WEIGHT = OFF_FACTOR + 2 * SOFTMAX_WARPS * N * 4;  // [N][warp]
  static constexpr int OFF_BAR = OFF_WEIGHT + SOFTMAX_WARPS * N * 4;
  // k_full, k_empty, v_full, v_empty, q_full, q_empty, s_full[2], p_full[2], p_empty[2], pv_done,
  // corrected, ml_full, ml_empty, o_full, o_free
  static constexpr int NUM_BARS = 4 * RING + 2 * Q_BUFS + 12;
  static constexpr int OFF_MISC = OFF_BAR + NUM_BARS * 8;
  // misc: tmem base, abort, non-finite drafts [2], correction requests [2][4]
  static constexpr int OFF_PLAN = OFF_MISC + 48;
  static constexpr int TOTAL = OFF_PLAN + PLAN_BYTES;
  static_assert(TOTAL <= 232448, "shared memory budget of one sm_100 CTA");
  // TMEM: S^T of buffer i at i N, O^T of warp w at (2 + w) N
  static constexpr uint32_t COL_O = 2 * N;
  static constexpr uint32_t TMEM_COLS = N == 16 ? 128 : 256;
};

// 16 lanes (from taddr's) x N columns: register 4 c + e is lane (lane / 4) + 8 (e / 2), column
// 8 c + 2 (lane % 4) + e % 2.
template <int N>
__device__ __forceinline__ void tmem_ld_16x256b(uint32_t taddr, uint32_t* r) {
  if constexpr (N == 16) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
                   "=r"(r[7])
                 : "r"(taddr));
  } else {
    static_assert(N == 32);
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32"
        " {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
          "=r"(r[15])
        : "r"(taddr));
  }
}

// Four 8 x 8 blocks of 16-bit elements, each transposed: lane l gives the address of row l % 8 of
// block l / 8 in memory and holds (row lane / 4, columns 2 (lane % 4), + 1) of every block.
__device__ __forceinline__ void stmatrix_x4_trans(uint32_t addr, uint32_t a, uint32_t b, uint32_t c,
                                                  uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr),
               "r"(a), "r"(b), "r"(c), "r"(d)
               : "memory");
}

// A column that has seen no key yet: below every score, and finite, so that a masked score (-inf)
// less it stays -inf.
constexpr float UNSEEN = -3.402823466e38f;

template <bool BF16, int D, int N>
__global__ void __launch_bounds__(NUM_THREADS, 1)
    narrow_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                  const __grid_constant__ CUtensorMap tmV, const Params p) {
  using L = Narrow<D, N>;
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
  uint64_t* k_empty = k_full + L::RING;
  uint64_t* v_full = k_empty + L::RING;
  uint64_t* v_empty = v_full + L::RING;
  uint64_t* q_full = v_empty + L::RING;       // [Q buffer]
  uint64_t* q_empty = q_full + L::Q_BUFS;     // [Q buffer]: the segment's last S has read Q
  uint64_t* s_full = q_empty + L::Q_BUFS;     // [buffer]
  uint64_t* p_full = s_full + 2;              // [buffer]: P, and a V tile's clean-up, are written
  uint64_t* p_empty = p_full + 2;             // [buffer]: the PV has read P, warps 4-7 its requests
  uint64_t* pv_done = p_empty + 2;            // one phase for each PV
  uint64_t* corrected = pv_done + 1;          // the scaling that a tile asked for is done
  uint64_t* ml_full = corrected + 1;          // the segment's maxima and sums are written
  uint64_t* ml_empty = ml_full + 1;           // ... and read, and the weights made of them
  uint64_t* o_full = ml_empty + 1;            // the segment's last PV
  uint64_t* o_free = o_full + 1;              // the epilogue has read O
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + L::OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::OFF_MISC + 4);
  unsigned int* bad = reinterpret_cast<unsigned int*>(smem + L::OFF_MISC + 8);    // [2]
  volatile int* ask = reinterpret_cast<volatile int*>(smem + L::OFF_MISC + 16);   // [buffer][warp]
  float2* ml = reinterpret_cast<float2*>(smem + L::OFF_ML);
  float4* weights = reinterpret_cast<float4*>(smem + L::OFF_WEIGHT);  // [N] of the four warps
  volatile float* factors = reinterpret_cast<volatile float*>(smem + L::OFF_FACTOR);

  const int warp = warp_id();
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < L::RING; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int s = 0; s < L::Q_BUFS; ++s) {
      mbar_init(&q_full[s], 1);
      mbar_init(&q_empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], SOFTMAX_WARPS);
      mbar_init(&p_empty[i], 1 + OUT_WARPS);
    }
    mbar_init(pv_done, 1);
    mbar_init(corrected, OUT_WARPS);
    mbar_init(ml_full, SOFTMAX_WARPS);
    mbar_init(ml_empty, OUT_WARPS);
    mbar_init(o_full, 1);
    mbar_init(o_free, OUT_WARPS);
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
    tmem_alloc(tmem_holder, L::TMEM_COLS);
    tmem_relinquish();
  }
  // query rows that no load writes are columns of zeros
  for (int i = threadIdx.x; i < L::Q_BUFS * L::Q_BUF / 16; i += NUM_THREADS) {
    *reinterpret_cast<uint4*>(smem + L::OFF_Q + i * 16) = make_uint4(0u, 0u, 0u, 0u);
  }
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  pdl_wait();  // the previous grid's writes (this launch's inputs) are visible from here on
  // after the wait: the join kernel may be scheduled now, and waits for this grid itself
  pdl_launch_dependents();
  Walk<true> w = plan<D, true>(p, smem + L::OFF_PLAN);

  // K and V are read once: evict first, and the tables, partials and code stay in L2
  if (warp == K_WARP) {
    produce_kv(p, w, Loader<D, L::RING>{&tmK, smem + L::OFF_K, k_full, k_empty, abort_flag,
                                        l2_policy_evict_first(), 0u, 0, 0});
  } else if (warp == V_WARP) {
    produce_kv(p, w, Loader<D, L::RING>{&tmV, smem + L::OFF_V, v_full, v_empty, abort_flag,
                                        l2_policy_evict_first(), 0u, 0, 0});
  } else if (warp == Q_WARP) {
    produce_q<D, L::Q_BUFS>(p, w, &tmQ, smem + L::OFF_Q, L::Q_BUF, L::Q_HALF, q_full, q_empty, abort_flag);
  } else if (warp == MMA_WARP) {
    // ------------------------------ MMA issuer ------------------------------
    constexpr uint32_t FMT = BF16 ? 1u : 0u;
    constexpr uint32_t idesc_s = make_idesc(BN, N, FMT, FMT, 0u, 0u);  // K Q^T, both K-major
    constexpr uint32_t idesc_o = make_idesc(128, N, FMT, FMT, 1u, 0u);  // V^T (MN-major) P^T
    // 64 dimensions are one MN block: with a block stride of zero the lanes from 64 on repeat it
    constexpr uint32_t V_BLOCK = D == 128 ? 1024u : 0u;
    // w and j run one tile ahead of the PVs, into the next segment
    int j = 0, tiles = w.left > 0 ? w.count() : 0;
    uint32_t segment = 0, o_phase = 0, corrections = 0;
    bool first_segment = true;
    // S^T of tile t into buffer t & 1: the softmax has read tile t - 2 from it, since that tile's P
    // was waited for.
    auto issue_s = [&](uint32_t t) -> bool {
      const uint32_t buf = segment % L::Q_BUFS;
      if (j == 0 &&
          !wait_for(&q_full[buf], (segment / L::Q_BUFS) & 1u, abort_flag, p.status, SITE_MMA_Q)) {
        return false;
      }
      const int st = static_cast<int>(t % L::RING);
      if (!wait_for(&k_full[st], (t / L::RING) & 1u, abort_flag, p.status, SITE_MMA_K)) return false;
      tc_fence_after();
      const uint64_t kdesc = sdesc_sw128(smem_u32(smem + L::OFF_K + st * L::TILE), 16, L::GROUP);
      const uint64_t qdesc = sdesc_sw128(smem_u32(smem + L::OFF_Q + buf * L::Q_BUF), 16, 1024);
      if (elect_one_sync()) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t ko = ((kk >> 2) * 1024 + (kk & 3) * 32) >> 4;
          const uint32_t qo = ((kk >> 2) * L::Q_HALF + (kk & 3) * 32) >> 4;
          umma_f16(tmem + (t & 1u) * N, kdesc + ko, qdesc + qo, idesc_s, kk > 0 ? 1u : 0u);
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
    for (uint32_t g = 0; more; ++g) {  // tile g: S and P buffer g & 1, their phase (g >> 1) & 1
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
      const uint32_t buf = g & 1u;
      const int st = static_cast<int>(g % L::RING);
      if (!wait_for(&v_full[st], (g / L::RING) & 1u, abort_flag, p.status, SITE_MMA_V)) break;
      if (!wait_for(&p_full[buf], (g >> 1) & 1u, abort_flag, p.status, SITE_MMA_P)) break;
      if (first && !first_segment) {  // the last segment's O has been read
        if (!wait_for(o_free, o_phase, abort_flag, p.status, SITE_MMA_OFREE)) break;
        o_phase ^= 1u;
      }
      if (ask[buf * 4] | ask[buf * 4 + 1] | ask[buf * 4 + 2] | ask[buf * 4 + 3]) {
        if (!wait_for(corrected, corrections & 1u, abort_flag, p.status, SITE_N_MMA_CORR)) break;
        ++corrections;
      }
      tc_fence_after();
      const uint64_t vdesc = sdesc_sw128(smem_u32(smem + L::OFF_V + st * L::TILE), V_BLOCK, L::GROUP);
      const uint64_t pdesc = sdesc_sw128(smem_u32(smem + L::OFF_P + buf * L::P_BUF), 16, 1024);
      if (elect_one_sync()) {
#pragma unroll
        for (int h = 0; h < SOFTMAX_WARPS; ++h) {  // warp h's 32 keys into its own O
#pragma unroll
          for (int kk = 0; kk < 2; ++kk) {
            umma_f16(tmem + L::COL_O + h * N, vdesc + static_cast<uint64_t>((2 * h + kk) * 2 * L::GROUP / 16),
                     pdesc + static_cast<uint64_t>(((h >> 1) * N * 128 + (h & 1) * 64 + kk * 32) / 16),
                     idesc_o, (!first || kk > 0) ? 1u : 0u);
          }
        }
        umma_commit(pv_done);
        umma_commit(&p_empty[buf]);
        umma_commit(&v_empty[st]);
        if (last) umma_commit(o_full);
      }
      __syncwarp();
      if (last) first_segment = false;
    }
  } else if (warp < SOFTMAX_WARPS) {
    // ------------------------------ softmax ------------------------------
    constexpr int C8 = N / 8;  // blocks of eight columns (query rows)
    const float sl = p.scale_log2;
    const uint64_t sl2 = f2(sl, sl);
    const int col0 = 2 * (lane & 3);  // this thread's columns: 8 c + col0, + 1
    const uint32_t t_s = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    // this lane's row of the transposing stores: column lane % 8 of a block, keys 8 (lane / 8) ...
    const uint32_t p_row = smem_u32(smem + L::OFF_P) + (warp >> 1) * (N * 128) + (lane & 7) * 128 +
                           ((((warp & 1) * 4 + (lane >> 3)) ^ (lane & 7)) << 4);
    uint32_t g = 0, segment = 0;
    bool ok = true;
    Walk<true> following;
    // lane r: what row r of a segment sees
    const int tok = lane / p.group;
    auto bits_at = [&](const Walk<true>& v) -> uint64_t {
      return v.left > 0 && tok < v.tokens ? bits_of(p, v.row, tok, v.tokens) : 0ull;
    };
    uint64_t bits = bits_at(w), following_bits = 0;
    for (; w.left > 0 && ok; w = following, bits = following_bits, ++segment) {
      const int tiles = w.count();
      float m[C8][2];
      uint64_t sum[C8];
#pragma unroll
      for (int c = 0; c < C8; ++c) {
        m[c][0] = m[c][1] = UNSEEN;
        sum[c] = 0ull;
      }
      for (int j = 0; j < tiles; ++j, ++g) {
        const int k0 = (w.i0 + j) * BN;
        const uint32_t buf = g & 1u;
        const bool masked = k0 + BN > w.ctx;
        if (j + 1 == tiles) {  // the next segment's request, while this one's last tile comes
          following = w;
          following.next(p);
          following_bits = bits_at(following);
        }
        if (!wait_for(&s_full[buf], (g >> 1) & 1u, abort_flag, p.status, SITE_SM_S)) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (masked) {
          // behind S of this tile: the V tile before in this place has been waited for by then, so that
          // the phase is the right one
          const int st = static_cast<int>(g % L::RING);
          if (!wait_for(&v_full[st], (g / L::RING) & 1u, abort_flag, p.status, SITE_SM_V)) {
            ok = false;
            break;
          }
          clean_v<BF16, D>(smem + L::OFF_V + st * L::TILE, 0, BN, w.ctx - k0, w.len() - k0, k0 - w.ctx,
                           threadIdx.x, bad);
        }
        uint32_t s[2][N / 2];  // [16 keys][4 c + e]
        tmem_ld_16x256b<N>(t_s + buf * N, s[0]);
        tmem_ld_16x256b<N>(t_s + buf * N + (16u << 16), s[1]);
        tmem_ld_wait();
        reg_fence(s[0]);
        reg_fence(s[1]);
        if (masked) {
          const int key = k0 - w.ctx + warp * 32 + (lane >> 2);  // of the first, drafted from 0 on
#pragma unroll
          for (int c = 0; c < C8; ++c) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t view = view_word(__shfl_sync(0xffffffffu, bits, 8 * c + col0 + e), key);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                if (!((view >> (8 * i)) & 1u)) s[i >> 1][4 * c + 2 * (i & 1) + e] = __float_as_uint(-INFINITY);
              }
            }
          }
        }
        // s sl - m of the thread's i-th key, columns 8 c + col0 and its neighbour
        auto shifted = [&](int c, int i) -> uint64_t {
          return fma2(f2(__uint_as_float(s[i >> 1][4 * c + 2 * (i & 1)]),
                         __uint_as_float(s[i >> 1][4 * c + 2 * (i & 1) + 1])),
                      sl2, f2(-m[c][0], -m[c][1]));
        };
        float top = -INFINITY;
#pragma unroll
        for (int c = 0; c < C8; ++c) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float x0, x1;
            f2_split(shifted(c, i), x0, x1);
            top = max3(top, x0, x1);
          }
        }
        // the buffer of P and of the factors: the PV two tiles ago has read the one, warps 4-7 the other
        if (!wait_for(&p_empty[buf], ((g >> 1) & 1u) ^ 1u, abort_flag, p.status, SITE_N_SM_P)) {
          ok = false;
          break;
        }
        int scale_o = 0;
        if (__any_sync(0xffffffffu, top > RESCALE_THRESHOLD)) {
          // some column's maximum moves: take the columns' maxima over the warp's 32 keys
          bool scale = false;
          volatile float* out = factors + (buf * SOFTMAX_WARPS + warp) * N;
#pragma unroll
          for (int c = 0; c < C8; ++c) {
            float f[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float mx = -INFINITY;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                mx = fmaxf(mx, __uint_as_float(s[i >> 1][4 * c + 2 * (i & 1) + e]));
              }
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
              mx *= sl;
              f[e] = 1.f;
              if (mx > m[c][e] + RESCALE_THRESHOLD) {
                f[e] = ex2(m[c][e] - mx);  // 0 where nothing was seen so far
                scale |= m[c][e] != UNSEEN;
                m[c][e] = mx;
              }
              if (lane < 4) out[8 * c + col0 + e] = f[e];
            }
            float s0, s1;
            f2_split(sum[c], s0, s1);
            sum[c] = f2(s0 * f[0], s1 * f[1]);
          }
          scale_o = __any_sync(0xffffffffu, scale) ? 1 : 0;
        }
#pragma unroll
        for (int c = 0; c < C8; ++c) {
          uint32_t pk[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float x0, x1;
            f2_split(shifted(c, i), x0, x1);
            const float e0 = ex2(x0), e1 = ex2(x1);
            sum[c] = add2(sum[c], f2(e0, e1));
            pk[i] = pack2<BF16>(e0, e1);  // rounded as tree.cu explains; the sum is of e
          }
          stmatrix_x4_trans(p_row + buf * L::P_BUF + c * 1024, pk[0], pk[1], pk[2], pk[3]);
        }
        if (lane == 0) ask[buf * 4 + warp] = scale_o;
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[buf]);
      }
      if (!ok) break;
      // ---- the segment's maxima and sums ----
      if (!wait_for(ml_empty, (segment & 1u) ^ 1u, abort_flag, p.status, SITE_N_SM_ML)) break;
#pragma unroll
      for (int c = 0; c < C8; ++c) {
        float l[2];
        f2_split(sum[c], l[0], l[1]);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          l[e] += __shfl_xor_sync(0xffffffffu, l[e], 4);
          l[e] += __shfl_xor_sync(0xffffffffu, l[e], 8);
          l[e] += __shfl_xor_sync(0xffffffffu, l[e], 16);
          if (lane < 4) {
            ml[warp * N + 8 * c + col0 + e] = make_float2(m[c][e] == UNSEEN ? -INFINITY : m[c][e], l[e]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(ml_full);
    }
  } else {
    // --------------- correction and epilogue (thread = head dimension) ---------------
    const int quarter = warp & 3;
    const int d = quarter * 32 + lane;
    const int tok_r = lane / p.group;  // of row `lane`
    const uint32_t t_o = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + L::COL_O;
    uint32_t g = 0, segment = 0;
    bool ok = true;
    for (; w.left > 0 && ok; w.next(p), ++segment) {
      const int tiles = w.count();
      for (int j = 0; j < tiles; ++j, ++g) {
        const uint32_t buf = g & 1u;
        if (!wait_for(&p_full[buf], (g >> 1) & 1u, abort_flag, p.status, SITE_N_OUT_P)) {
          ok = false;
          break;
        }
        bool any = false;
        for (int h = 0; h < SOFTMAX_WARPS; ++h) any |= ask[buf * 4 + h] != 0;
        if (!any) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_empty[buf]);
          continue;
        }
        // the PV before; the one before that is complete, since this tile's S came behind it
        if (!wait_for(pv_done, (g - 1) & 1u, abort_flag, p.status, SITE_N_OUT_PV)) {
          ok = false;
          break;
        }
        tc_fence_after();
        for (int h = 0; h < SOFTMAX_WARPS; ++h) {
          if (ask[buf * 4 + h] == 0) continue;
          volatile float* f = factors + (buf * SOFTMAX_WARPS + h) * N;
#pragma unroll 1
          for (int c = 0; c < N; c += 16) {
            uint32_t o[16];
            tmem_ld_32x32b_x16(t_o + h * N + c, o);
            tmem_ld_wait();
            reg_fence(o);
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f[c + i]);
            tmem_st_32x32b_x16(t_o + h * N + c, o);
          }
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(corrected);
          mbar_arrive(&p_empty[buf]);
        }
      }
      if (!ok) break;
      if (!wait_for(ml_full, segment & 1u, abort_flag, p.status, SITE_N_OUT_ML)) break;
      const bool whole = w.i0 == 0 && tiles == w.tiles();
      const int rows = w.tokens * p.group;
      const long long slot = slot_of(p, blockIdx.x, 0, w.i0 > 0);
      // Lane r: the weights of row r's four states. The four warps write the same values; none gets
      // to the next segment's while another reads these (ml_empty).
      if (lane < N) {
        const int r = lane;
        float wt[SOFTMAX_WARPS];
        float top = -INFINITY, l = 0.f;
#pragma unroll
        for (int h = 0; h < SOFTMAX_WARPS; ++h) top = fmaxf(top, ml[h * N + r].x);
        const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int h = 0; h < SOFTMAX_WARPS; ++h) {
          const float2 v = ml[h * N + r];
          wt[h] = ex2(v.x - base);
          l = fmaf(wt[h], v.y, l);
        }
        if (r < rows && quarter == 0) {
          if (whole) {
            p.lse[static_cast<long long>(w.row + tok_r) * p.hq + w.kvh * p.group + (r - tok_r * p.group)] =
                l == 0.f ? -INFINITY : (top + log2f(l)) * 0.6931471805599453f;
          } else {
            p.part_ml[slot * p.row_cap + r] = make_float2(top, l);
          }
        }
        // a row that sees nothing: O = 0; a partial stays as it is, for the join to divide
        const float inv = !whole ? 1.f : l == 0.f ? 0.f : 1.f / l;
        weights[r] = make_float4(wt[0] * inv, wt[1] * inv, wt[2] * inv, wt[3] * inv);
      }
      __syncwarp();
      if (!wait_for(o_full, segment & 1u, abort_flag, p.status, SITE_N_OUT_O)) break;
      tc_fence_after();
      uint16_t* out = static_cast<uint16_t*>(p.out) +
                      (static_cast<long long>(w.row) * p.hq + w.kvh * p.group) * D + d;
      float* part = p.part_o + slot * p.row_cap * D + d;
      const int gap = (p.hq - p.group) * D;  // from a token's last head to the next token's first
      long long at = 0;
      int head = 0;
#pragma unroll 1
      for (int c = 0; c < rows; c += 8) {
        uint32_t o[SOFTMAX_WARPS][8];
#pragma unroll
        for (int h = 0; h < SOFTMAX_WARPS; ++h) tmem_ld_32x32b_x8(t_o + h * N + c, o[h]);
        tmem_ld_wait();
#pragma unroll
        for (int h = 0; h < SOFTMAX_WARPS; ++h) reg_fence(o[h]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float4 wt = weights[c + i];
          float v = __uint_as_float(o[0][i]) * wt.x;
          v = fmaf(__uint_as_float(o[1][i]), wt.y, v);
          v = fmaf(__uint_as_float(o[2][i]), wt.z, v);
          v = fmaf(__uint_as_float(o[3][i]), wt.w, v);
          if (c + i < rows && d < D) {
            if (whole) {
              out[at] = static_cast<uint16_t>(pack_o<BF16>(v, 0.f) & 0xffffu);
            } else {
              part[(c + i) * D] = v;
            }
          }
          at += D;
          if (++head == p.group) {
            head = 0;
            at += gap;
          }
        }
      }
      if ((bad[0] | bad[1]) != 0u && d < D) {
        // drafted V elements that are not finite, for the rows that see them
        const uint64_t marked = static_cast<uint64_t>(bad[1]) << 32 | bad[0];
        for (int r = 0; r < rows; ++r) {
          const int tok = r / p.group;
          for (uint64_t left = marked & bits_of(p, w.row, tok, w.tokens); left != 0; left &= left - 1) {
            const int key = w.ctx + __ffsll(static_cast<long long>(left)) - 1;
            if (key < w.i0 * BN || key >= (w.i0 + tiles) * BN) continue;
            const int id = p.tables[w.b * p.table_stride + (key >> p.page_log2)];
            if (id < 0 || id >= p.num_blocks) continue;
            const float v = load16<BF16>(
                p.v, (((static_cast<long long>(id) << p.page_log2) + (key & ((1 << p.page_log2) - 1))) *
                          p.hkv + w.kvh) * D + d);
            if (isfinite(v)) continue;
            if (whole) {
              uint16_t* o = out + (static_cast<long long>(tok) * p.hq + (r - tok * p.group)) * D;
              *o = static_cast<uint16_t>(pack2<BF16>(load16<BF16>(o, 0) + v, 0.f) & 0xffffu);
            } else {
              part[r * D] += v;
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(ml_empty);
        mbar_arrive(o_free);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == MMA_WARP) {
    tc_fence_after();
    tmem_dealloc(tmem, L::TMEM_COLS);
  }
}

template <bool BF16, int D>
int launch_narrow(const Params& p, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                  int grid, cudaStream_t stream) {
  auto go = [&](auto kernel, int smem) -> int {
    const int s = set_kernel_smem(reinterpret_cast<const void*>(kernel), smem);
    if (s != KTA_OK) return s;
    return launch_ex(kernel, dim3(grid), dim3(NUM_THREADS), smem, stream, 1, tq, tk, tv, p);
  };
  const int rows = p.box_tokens * p.group;
  static_assert(NARROW_ROWS == 32, "the most query rows of a kernel below");
  return rows <= 16 ? go(narrow_kernel<BF16, D, 16>, Narrow<D, 16>::TOTAL)
                    : go(narrow_kernel<BF16, D, 32>, Narrow<D, 32>::TOTAL);
}

template int launch_narrow<false, 64>(const Params&, const CUtensorMap&, const CUtensorMap&,
                                      const CUtensorMap&, int, cudaStream_t);
template int launch_narrow<true, 64>(const Params&, const CUtensorMap&, const CUtensorMap&,
                                     const CUtensorMap&, int, cudaStream_t);
template int launch_narrow<false, 128>(const Params&, const CUtensorMap&, const CUtensorMap&,
                                       const CUtensorMap&, int, cudaStream_t);
template int launch_narrow<true, 128>(const Params&, const CUtensorMap&, const CUtensorMap&,
                                      const CUtensorMap&, int, cudaStream_t);

}  // namespace tree
}  // namespace kta
