// Rotary positions, sm_100a: alone (forward and gradient), and fused with the write of K and V
// into a paged cache.
//
//   pair i of a row, (a, b) = (x_i, x_{i + rot/2}) (half layout) or (x_2i, x_{2i+1}) (interleaved):
//   (a, b) -> scale (a cos t - b sin t, b cos t + a sin t),   t = position * freq_i
//   dimensions from rot on are copied; the gradient is the same map with -t (its transpose).
//
// The angle is kept in turns as a 64-bit fraction: f = frac(freq / 2 pi) 2^64 is an integer, off by
// at most one, and position * f mod 2^64 drops whole turns exactly. So an angle is off by |position|
// 2^-64 turns (4e-7 rad at 2^40; a 32-bit product would be off by 0.06 rad at a million) and by the
// one 32-bit rounding, that of the reduced angle (2^-25 of a half turn). Rotation in fp32, one
// rounding to the storage type.
//
// HBM-bound: 4 bytes per element (read once, written once). A CTA takes a few tokens: its threads
// first put their loads in flight, then compute the tokens' cos and sin once into shared memory
// for all heads (64 pairs against 32 or more heads), then rotate. A work item is two 16-byte
// vectors half a region apart (rotated region or rest), which is the pair of the half layout and
// in every layout keeps a warp's loads and stores contiguous.
//
// Figures of replayed graphs. Small CTAs with two items to a thread in flight, and streaming loads and
// stores: 32768 x 32 heads take 89.3 us (6010 GB/s; a plain copy of as many bytes 82.5) against 97.6
// with 256 threads and four items, 101 to 127 with 512 threads or without the streaming hints. Few
// tokens are latency: there a thread has one item, and a token's heads are spread over several CTAs
// (512 tokens of 48 heads: 4.3 us with one item to a thread, 5.6 with 256 threads and four; 64 tokens
// 1.8 us). With few heads the angles are the work: a thread keeps its pair where it can, and its
// frequency's fraction (32768 tokens of one head 13.6 us without, 10.1 so with more tokens to a CTA).
// With the cache write, 16384 tokens of 48 heads: 64.3 us, 6260 GB/s. Single calls on changing inputs,
// one after the other: 96.1 us (5590 GB/s) and 66.9 (6020).
#include <algorithm>
#include <cmath>

#include "kta_common.cuh"
#include "kta_host.h"

namespace kta {
namespace rope {

constexpr int THREADS = 128;
constexpr int MAX_D = 1024;
constexpr int MAX_TOKENS = 32;   // tokens of a CTA
constexpr int VEC = 8;           // 16-byte vectors of 16-bit elements

enum : unsigned int { SITE_SLOT = 0x811 };

struct View {  // rows of D elements of one head each
  const void* in;
  void* out;
  long long in_token, in_head, out_token, out_head;  // strides in elements
};

struct Params {
  View q, k, v;            // k and v: only with a cache, out = the cache
  const void* positions;   // [tokens] int32 or int64
  const int64_t* slots;    // [tokens], or nullptr without a cache
  const double* freqs;     // [rot / 2] radians per position
  long long num_slots;
  int tokens, hq, hkv, rows;  // rows of a token: hq (+ 2 hkv)
  int pos64, rot, items, rot_items;  // items of a row, those of them that rotate
  int rest;                // vectors between an item's two in the region that is copied
  int per_cta;             // tokens of a CTA
  int half_log2;           // of rot / 2 where that divides THREADS, else -1
  float scale, sign;
  unsigned int* status;
};

template <typename T>
__device__ __forceinline__ float2 unpack(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <>
__device__ __forceinline__ float2 unpack<__nv_bfloat16>(uint32_t w) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
}
template <typename T>
__device__ __forceinline__ uint32_t pack(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack<__half>(float a, float b) { return pack_f16x2(a, b); }
template <>
__device__ __forceinline__ uint32_t pack<__nv_bfloat16>(float a, float b) { return pack_bf16x2(a, b); }

// frac(freq / 2 pi) as a 64-bit fraction of a turn, within 2^-64 for |freq| < 2^40. 1 / (2 pi) in two
// parts, and the first product's rounding error by fma (Dekker's exact product): one product in 64
// bits would be off by 2^-53 of the frequency, which a position of 2^40 makes 7e-5 rad. The rest is
// small enough to become an integer by an addition.
__device__ __forceinline__ uint64_t turn_fraction(double freq) {
  constexpr double HI = 0x1.45f306dc9c883p-3, LO = -0x1.6b01ec5417056p-57;
  constexpr double ONES = 0x1.8p52;  // doubles around it are the whole numbers
  const double turns = freq * HI, rest = fma(freq, LO, fma(freq, HI, -turns));
  const long long whole = __double2ll_rn((turns - rint(turns)) * 0x1p64);  // of [-1/2, 1/2] turns
  const long long more = __double_as_longlong(fma(rest, 0x1p64, ONES)) - __double_as_longlong(ONES);
  return static_cast<uint64_t>(whole + (fabs(freq) < 0x1p40 ? more : 0));
}

// An item's place: source, destination and first vector's two element offsets, its token in the
// CTA and its first pair (-1: copied). dst == nullptr: nothing to do.
template <typename T>
struct Item {
  const T* src;
  T* dst;
  int second;  // elements from the first vector to the second
  int token, pair;
};

template <typename T, bool CACHE>
__device__ __forceinline__ Item<T> item_at(const Params& p, int token0, int token, int row, int piece,
                                           const long long* slot) {
  Item<T> it;
  it.token = token;
  const long long n = token0 + token;
  const View* v = &p.q;
  int head = row;
  long long out_row = n;
  bool on = true, turns = piece < p.rot_items;
  if (CACHE && row >= p.hq) {
    head -= p.hq;
    v = &p.k;
    if (head >= p.hkv) {
      head -= p.hkv;
      v = &p.v;
      turns = false;
    }
    out_row = slot[token];
    on = out_row >= 0;
  }
  int first;
  if (piece < p.rot_items) {
    first = piece * VEC;
    it.second = p.rot_items * VEC;
  } else {
    first = p.rot + (piece - p.rot_items) * VEC;
    it.second = p.rest * VEC;
  }
  it.pair = turns ? piece : -1;
  it.src = static_cast<const T*>(v->in) + n * v->in_token + head * v->in_head + first;
  it.dst = on ? static_cast<T*>(v->out) + out_row * v->out_token + head * v->out_head + first : nullptr;
  return it;
}

// UNROLL: items of a thread whose loads are in flight together. SPREAD: a token's items over
// gridDim.y CTAs, one for a thread; twelve of them to an SM (with 48 registers, and so ten, 64 tokens of
// 32 heads take 2.8 us, not 2.4). Nine otherwise (with 64 registers, and so eight, 32768 tokens of 32
// heads take 95 us, not 92).
template <typename T, bool INTER, bool CACHE, int UNROLL, bool SPREAD>
__global__ void __launch_bounds__(THREADS, SPREAD ? 12 : 9) rope_kernel(const Params p) {
  extern __shared__ float2 turn[];  // [tokens of the CTA][rot / 2] scale * (cos, sin)
  __shared__ long long slot[MAX_TOKENS];
  pdl_launch_dependents();
  pdl_wait();  // the previous grid's writes (this launch's inputs) are visible from here on
  const int token0 = blockIdx.x * p.per_cta;
  const int tokens = min(p.per_cta, p.tokens - token0);
  if constexpr (CACHE) {
    if (threadIdx.x < tokens) {
      long long s = p.slots[token0 + threadIdx.x];
      if (s >= p.num_slots) {
        record_status(p.status, KTA_ERR_DEVICE_BOUNDS, SITE_SLOT);
        s = -1;
      }
      slot[threadIdx.x] = s;
    }
    __syncthreads();
  }
  const int half = p.rot >> 1;
  // The thread's first item, and how far the next one lies (in items, rows and tokens): steps
  // with a carry instead of two divisions for each item.
  const int d_piece = THREADS % p.items, d_row = THREADS / p.items;
  const int first = (SPREAD ? blockIdx.y * THREADS : 0) + threadIdx.x;
  int piece = first % p.items;
  int row = first / p.items;
  int token = row / p.rows;
  row -= token * p.rows;
  bool table = false;
  while (true) {
    Item<T> it[UNROLL];
    uint4 lo[UNROLL], hi[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      it[u].dst = nullptr;
      if (token < tokens) {
        it[u] = item_at<T, CACHE>(p, token0, token, row, piece, slot);
        if (it[u].dst != nullptr) {
          lo[u] = __ldcs(reinterpret_cast<const uint4*>(it[u].src));
          hi[u] = __ldcs(reinterpret_cast<const uint4*>(it[u].src + it[u].second));
        }
      }
      piece += d_piece;
      row += d_row;
      if (piece >= p.items) {
        piece -= p.items;
        ++row;
      }
      while (row >= p.rows) {
        row -= p.rows;
        ++token;
      }
    }
    if (!table) {  // once, behind the first loads
      table = true;
      auto angle = [&](int t, int f, uint64_t fraction) {
        const long long pos = p.pos64 ? static_cast<const int64_t*>(p.positions)[token0 + t]
                                      : static_cast<const int32_t*>(p.positions)[token0 + t];
        const uint64_t phase = static_cast<uint64_t>(pos) * fraction;
        // half turns in [-1, 1)
        const float x = static_cast<float>(static_cast<int32_t>(phase >> 32)) * 4.656612873077393e-10f;
        float s, c;
        sincospif(x, &s, &c);
        turn[t * half + f] = make_float2(c * p.scale, s * p.scale * p.sign);
      };
      if (!SPREAD && p.half_log2 >= 0) {  // a thread keeps its pair
        const int f = threadIdx.x & (half - 1);
        const uint64_t fraction = turn_fraction(p.freqs[f]);
        for (int t = threadIdx.x >> p.half_log2; t < tokens; t += THREADS >> p.half_log2) angle(t, f, fraction);
      } else {
        for (int i = threadIdx.x; i < tokens * half; i += THREADS) {
          const int t = i / half, f = i - t * half;
          angle(t, f, turn_fraction(p.freqs[f]));
        }
      }
      __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      if (it[u].dst == nullptr) continue;
      uint4 a = lo[u], b = hi[u];
      if (it[u].pair >= 0) {
        uint32_t* aw = reinterpret_cast<uint32_t*>(&a);
        uint32_t* bw = reinterpret_cast<uint32_t*>(&b);
        if constexpr (INTER) {
          // each vector holds four pairs of neighbours
          const float2* ta = turn + it[u].token * half + it[u].pair * (VEC / 2);
          const float2* tb = ta + p.rot_items * (VEC / 2);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 x = unpack<T>(aw[i]), y = unpack<T>(bw[i]);
            const float2 c = ta[i], d = tb[i];
            aw[i] = pack<T>(x.x * c.x - x.y * c.y, x.y * c.x + x.x * c.y);
            bw[i] = pack<T>(y.x * d.x - y.y * d.y, y.y * d.x + y.x * d.y);
          }
        } else {
          // element j of the first vector pairs with element j of the second
          const float2* t = turn + it[u].token * half + it[u].pair * VEC;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 x = unpack<T>(aw[i]), y = unpack<T>(bw[i]);
            const float2 c = t[2 * i], d = t[2 * i + 1];
            aw[i] = pack<T>(x.x * c.x - y.x * c.y, x.y * d.x - y.y * d.y);
            bw[i] = pack<T>(y.x * c.x + x.x * c.y, y.y * d.x + x.y * d.y);
          }
        }
      }
      __stcs(reinterpret_cast<uint4*>(it[u].dst), a);
      __stcs(reinterpret_cast<uint4*>(it[u].dst + it[u].second), b);
    }
    if (SPREAD || token >= tokens) break;
  }
}

bool view_ok(const void* in, const void* out, long long heads, const long long* st) {
  return in != nullptr && out != nullptr && heads > 0 && st[0] >= 0 && st[1] >= 0;
}

// Strides in elements: rows start on 16-byte boundaries, and no two rows of an output overlap.
int strides_status(const long long* in, const long long* out, long long tokens, long long heads,
                   long long D) {
  for (int i = 0; i < 2; ++i) {
    if (in[i] < 0 || out[i] < 0) return KTA_ERR_INVALID_ARG;
    if (in[i] % VEC != 0 || out[i] % VEC != 0) return KTA_ERR_ALIGN;
  }
  if ((tokens > 1 && out[0] < D) || (heads > 1 && out[1] < D)) return KTA_ERR_INVALID_ARG;
  // token-major or head-major: the rows of the inner dimension end before the outer one's next
  if (tokens > 1 && heads > 1 && out[0] < out[1] * (heads - 1) + D && out[1] < out[0] * (tokens - 1) + D) {
    return KTA_ERR_INVALID_ARG;
  }
  return KTA_OK;
}

int sizes_status(int64_t tokens, int64_t D, int64_t rot, float scale, int64_t pos_bytes) {
  if (tokens <= 0 || D <= 0 || rot <= 0 || rot > D) return KTA_ERR_INVALID_ARG;
  if (!std::isfinite(scale) || (pos_bytes != 4 && pos_bytes != 8)) return KTA_ERR_INVALID_ARG;
  if (D > MAX_D || tokens > (1LL << 30)) return KTA_ERR_UNSUPPORTED;
  if (D % (2 * VEC) != 0 || rot % (2 * VEC) != 0) return KTA_ERR_ALIGN;
  return KTA_OK;
}

int pointers_status(const void* positions, int64_t pos_bytes, const void* freqs) {
  if (positions == nullptr || freqs == nullptr) return KTA_ERR_INVALID_ARG;
  if (reinterpret_cast<uintptr_t>(positions) % static_cast<uintptr_t>(pos_bytes) != 0 ||
      reinterpret_cast<uintptr_t>(freqs) % 8 != 0) {
    return KTA_ERR_ALIGN;
  }
  return KTA_OK;
}

template <typename T, bool CACHE, int UNROLL, bool SPREAD>
int start(const Params& p, dim3 grid, bool interleaved, cudaStream_t stream) {
  const size_t smem = static_cast<size_t>(p.per_cta) * (p.rot / 2) * sizeof(float2);
  auto kernel = interleaved ? rope_kernel<T, true, CACHE, UNROLL, SPREAD>
                            : rope_kernel<T, false, CACHE, UNROLL, SPREAD>;
  return launch_ex(kernel, grid, dim3(THREADS), smem, stream, 1, p);
}

template <typename T, bool CACHE>
int go(Params& p, int64_t D, bool interleaved, cudaStream_t stream) {
  int s = require_sm100();
  if (s != KTA_OK) return s;
  p.rot_items = p.rot / (2 * VEC);
  p.items = static_cast<int>(D) / (2 * VEC);
  p.rest = p.items - p.rot_items;
  // in place, what is not rotated stays where it is
  if (!CACHE && p.q.in == p.q.out && p.q.in_token == p.q.out_token && p.q.in_head == p.q.out_head) {
    p.items = p.rot_items;
  }
  p.status = device_status_ptr();
  p.half_log2 = -1;
  for (int i = 0; 1 << i <= THREADS; ++i) {
    if (p.rot == 2 << i) p.half_log2 = i;
  }
  const long long per_token = static_cast<long long>(p.rows) * p.items;
  const int sms = current_sm_count();
  // One item to a thread while they are little more than the SMs hold at once (1536 threads each; the
  // limit of 2048 is 1184 tokens of 32 heads of 128 at 148 SMs), if a token fills a CTA. 1024 tokens of 32 heads take 5.4 us so and 5.7
  // the other way; 2400, past the limit, would take 9.6 us so and take 9.4 the other way. 9400 tokens of
  // 4 heads, which do not fill a CTA, 11.2 and 6.5.
  if (per_token >= THREADS && p.tokens * per_token <= 2048LL * sms) {
    p.per_cta = 1;
    const dim3 grid(p.tokens, static_cast<unsigned>((per_token + THREADS - 1) / THREADS));
    return start<T, CACHE, 1, true>(p, grid, interleaved, stream);
  }
  // Tokens of a CTA: four items for a thread, but never fewer CTAs than fill the SMs, nor more than
  // eight tokens where they give every thread an item (32768 tokens of one head: 10.3 us with 16
  // tokens, 12.3 with 8; of four heads 15.8 with 8, 18.3 with 16).
  int per = 1;
  const int most = std::max(1, std::min(MAX_TOKENS, 4096 / p.rot));  // and 16 KB of cos and sin
  while (per < most && per * per_token < (per < 8 ? 4 : 1) * THREADS && p.tokens / (2 * per) >= 8 * sms) per *= 2;
  p.per_cta = per;
  return start<T, CACHE, 2, false>(p, dim3((p.tokens + per - 1) / per), interleaved, stream);
}

template <typename T>
int launch(const void* X, const void* positions, int64_t pos_bytes, const void* freqs, void* Y,
           int64_t tokens, int64_t heads, int64_t D, int64_t rot, int64_t x_token, int64_t x_head,
           int64_t y_token, int64_t y_head, int interleaved, int inverse, float scale,
           cudaStream_t stream) {
  const long long in[2] = {x_token, x_head}, out[2] = {y_token, y_head};
  int s = sizes_status(tokens, D, rot, scale, pos_bytes);
  if (s != KTA_OK) return s;
  if (!view_ok(X, Y, heads, in)) return KTA_ERR_INVALID_ARG;
  if (heads > (1 << 20)) return KTA_ERR_UNSUPPORTED;
  s = pointers_status(positions, pos_bytes, freqs);
  if (s != KTA_OK) return s;
  s = strides_status(in, out, tokens, heads, D);
  if (s != KTA_OK) return s;
  if (!aligned16(X) || !aligned16(Y)) return KTA_ERR_ALIGN;
  Params p = {};
  p.q = View{X, Y, x_token, x_head, y_token, y_head};
  p.positions = positions;
  p.pos64 = pos_bytes == 8;
  p.freqs = static_cast<const double*>(freqs);
  p.tokens = static_cast<int>(tokens);
  p.hq = p.rows = static_cast<int>(heads);
  p.rot = static_cast<int>(rot);
  p.scale = scale;
  p.sign = inverse ? -1.f : 1.f;
  return go<T, false>(p, D, interleaved != 0, stream);
}

template <typename T>
int launch_cache(const void* Q, const void* K, const void* V, const void* positions,
                 int64_t pos_bytes, const void* slots, const void* freqs, void* Qo, void* Kc,
                 void* Vc, int64_t tokens, int64_t Hq, int64_t Hkv, int64_t D, int64_t rot,
                 const int64_t* strides, int64_t num_slots, int interleaved, float scale,
                 cudaStream_t stream) {
  int s = sizes_status(tokens, D, rot, scale, pos_bytes);
  if (s != KTA_OK) return s;
  if (strides == nullptr || slots == nullptr || num_slots <= 0) return KTA_ERR_INVALID_ARG;
  const long long q_in[2] = {strides[0], strides[1]}, k_in[2] = {strides[2], strides[3]};
  const long long v_in[2] = {strides[4], strides[5]}, q_out[2] = {strides[6], strides[7]};
  const long long cache[2] = {Hkv * D, D};
  if (!view_ok(Q, Qo, Hq, q_in) || !view_ok(K, Kc, Hkv, k_in) || !view_ok(V, Vc, Hkv, v_in)) {
    return KTA_ERR_INVALID_ARG;
  }
  if (Hq > (1 << 20) || Hkv > (1 << 20)) return KTA_ERR_UNSUPPORTED;
  s = pointers_status(positions, pos_bytes, freqs);
  if (s != KTA_OK) return s;
  if ((s = strides_status(q_in, q_out, tokens, Hq, D)) != KTA_OK) return s;
  if ((s = strides_status(k_in, cache, tokens, Hkv, D)) != KTA_OK) return s;
  if ((s = strides_status(v_in, cache, tokens, Hkv, D)) != KTA_OK) return s;
  for (const void* q : {Q, K, V, static_cast<const void*>(Qo), static_cast<const void*>(Kc),
                        static_cast<const void*>(Vc)}) {
    if (!aligned16(q)) return KTA_ERR_ALIGN;
  }
  if (reinterpret_cast<uintptr_t>(slots) & 7) return KTA_ERR_ALIGN;
  Params p = {};
  p.q = View{Q, Qo, q_in[0], q_in[1], q_out[0], q_out[1]};
  p.k = View{K, Kc, k_in[0], k_in[1], cache[0], cache[1]};
  p.v = View{V, Vc, v_in[0], v_in[1], cache[0], cache[1]};
  p.positions = positions;
  p.pos64 = pos_bytes == 8;
  p.slots = static_cast<const int64_t*>(slots);
  p.freqs = static_cast<const double*>(freqs);
  p.num_slots = num_slots;
  p.tokens = static_cast<int>(tokens);
  p.hq = static_cast<int>(Hq);
  p.hkv = static_cast<int>(Hkv);
  p.rows = static_cast<int>(Hq + 2 * Hkv);
  p.rot = static_cast<int>(rot);
  p.scale = scale;
  p.sign = 1.f;
  return go<T, true>(p, D, interleaved != 0, stream);
}

}  // namespace rope
}  // namespace kta

#define KTA_ROPE_ENTRIES(NAME, TYPE)                                                               \
  extern "C" int kta_rope_##NAME(const void* X, const void* positions, int64_t pos_bytes,          \
                                 const void* freqs, void* Y, int64_t tokens, int64_t heads,        \
                                 int64_t D, int64_t rot, int64_t x_token, int64_t x_head,          \
                                 int64_t y_token, int64_t y_head, int interleaved, int inverse,    \
                                 float scale, void* stream) {                                      \
    return kta::rope::launch<TYPE>(X, positions, pos_bytes, freqs, Y, tokens, heads, D, rot,       \
                                   x_token, x_head, y_token, y_head, interleaved, inverse, scale,  \
                                   static_cast<cudaStream_t>(stream));                             \
  }                                                                                                \
  extern "C" int kta_rope_cache_##NAME(                                                            \
      const void* Q, const void* K, const void* V, const void* positions, int64_t pos_bytes,       \
      const void* slots, const void* freqs, void* Qo, void* Kc, void* Vc, int64_t tokens,          \
      int64_t Hq, int64_t Hkv, int64_t D, int64_t rot, const int64_t* strides, int64_t num_slots,  \
      int interleaved, float scale, void* stream) {                                                \
    return kta::rope::launch_cache<TYPE>(Q, K, V, positions, pos_bytes, slots, freqs, Qo, Kc, Vc,  \
                                         tokens, Hq, Hkv, D, rot, strides, num_slots, interleaved, \
                                         scale, static_cast<cudaStream_t>(stream));                \
  }

KTA_ROPE_ENTRIES(f16, __half)
KTA_ROPE_ENTRIES(bf16, __nv_bfloat16)
