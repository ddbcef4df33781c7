// Attention of attention_span.cuh on the fifth-generation tensor cores: sequences with more than 16 packed rows (query row x head of a key
// head), that is draft trees and chunks of prompts.
//
// One CTA owns up to 256 packed rows of one sequence and key head and walks the tokens that they see between them, 128 at a time; a split of
// the walk leaves partial sums for span_merge_kernel. S = Q K^T and O += P V are tcgen05.mma with their accumulators in tensor memory
// (two of S, two of O: all 512 columns). Two softmax groups of four warps, a thread to a row, work on two items at a time, so that one's
// exponentials run under the other's products:
//
//   more than 128 rows   items are (token tile, row tile): both row tiles read the same K and V
//   up to 128 rows       items are token tiles: the groups take them in turn, for the same rows, and join (m, l, O) at the end
//
//   warps 0 - 7   softmax        warp 9   issuer
//   bf16 cache    warps 8, 10 ask for K by TMA, warp 11 for V; it also looks through V where not every row sees the whole tile
//   e4m3 cache    K is an operand as it is, with queries in two e4m3 pieces; V travels as f16: warp 8 asks for both, warps 10 - 15 widen V
//   4-bit cache   warps 10 - 15 widen K and V (kv4.cuh) to f16, which warp 8 asks for tile by tile, in a unit of the tile or of each row; queries are f16
//
// What bounds it (times from captured graphs): two tiles of 128 x 128 scores take the softmax groups some 3200 clocks, the tensor pipe 2048 at heads of 128; and a CTA's way in (lengths,
// table, queries, keys, first products: 9000 clocks) and out (4000), which nothing on its SM runs under. 2 x 2048 rows behind 4096 tokens without a window, 32
// query and 8 key heads of 128: 1097 TFLOP/s, e4m3 1007; under a window of 1024 with 64 first tokens 735, of the products that the window leaves. (CTAs
// that stay and take item after item hid the way in, but missed the instruction cache 7000 times an SM for 2800: 146 us for 115 at that
// window then; 126 for 197 with 16 trees of equal lengths.) Over a 4-bit cache 2 x 2048 rows behind 2500 and 6143 tokens take
// 515 us, 697 TFLOP/s (bf16 327, e4m3 395): widening a tile of K and one of V takes three warps each about as long as the groups' softmax, they share its
// SM's issue slots, and every one of the 32 CTAs of a key head widens the same tiles. (471 us without rows of their own units, whose code, not taken there,
// costs a third more misses of the instruction cache, and a look at the smallest row in front of each tile.)
//
// What a row sees of a tile is four words of bits, from its bounds and its mask; tiles that all rows of a warp see whole have code
// without them. Values of places that some row does not see may be infinite or NaN: they are taken out of the tile there, and rows that
// do see them get them in the end from the cache (slow, and never taken otherwise). Every wait is bounded (ptx.cuh).
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <limits.h>

#include <algorithm>
#include <type_traits>

#include "attention_span.cuh"
#include "attention_util.cuh"
#include "kv4.cuh"
#include "tma_host.h"

namespace fllm {
namespace {
constexpr int kTcRows = 256, kWideners = 6;       // packed rows of a CTA; warps that widen V of an e4m3 cache
constexpr int kBf16 = 0, kE4m3 = 1;        // kinds of caches, and kKv4
template <int KV> constexpr int tc_threads() { return KV == kBf16 ? 384 : 512; }
template <int KV> constexpr int kQThreads = KV == kE4m3 ? 384 : 256;      // that load queries
constexpr float kTcLift = 6.f;             // f16 weights: their reference lies so far below the row's (their largest is 2^14 then)
constexpr int kTilePages = kTile / kPage;
template <int N> using Int = std::integral_constant<int, N>;
template <bool B> using Bool = std::integral_constant<bool, B>;

constexpr int kRawTokens = 64;             // of a piece of an e4m3 tile
constexpr int kKv4Slots = 3;               // of tiles of 4-bit rows
constexpr int kKv4Team = 3;                // warps that widen K, and V
constexpr int kKv4Top = -6;                // their largest magnitude is below 2 to this as f16 (kv4_widen_f16)
// A tile of 4-bit rows is widened in one unit (a power of two) where the largest magnitude of every row is 2^-13 or more in it: its values are then off by 2^-11
// of that at most. In other tiles each row is lifted by a power of two of its own, which its scores, in fp32, or its weights give back: a row keeps its bits
// beside rows of any size, be they seen or not. (Weights are below 2^15 and fall by the lift before they go to the product: 2^-25 of a unit in which the largest
// is 2^6 or more, so an output loses 2^-28 of the largest value so far for a token at most.) A text whose tiles are all such takes longer: 2 x 2048 rows behind
// 2500 and 6143 tokens 1026 us, 795 with only its keys so, 827 with its values (515 with neither).
constexpr int kKv4Even = 127 - 13, kKv4MostLift = 20;
constexpr int kTcFlags = 400;              // bytes of barriers and flags
constexpr int kAtVReady = 12, kAtPHalf = 16, kAtFlags = 38;      // of the barriers, in that order: 2, 2, and what follows them

// Shared memory: two tiles of Q, two stages of K and of V, 16-bit values in rows of 128 bytes. e4m3: Q in two e4m3 pieces, four stages of K as it
// is, V in 16 bits behind four slots of raw halves of tiles (eight where there is one tile of Q). 4 bits: three slots of raw tiles of K or V.
template <int D, int KV>
struct TcSmem {
  static constexpr int kT = tile_bytes<D>();           // a 128-row tile of 16-bit values
  static constexpr int kStages = KV == kE4m3 ? 4 : 2, kK = KV == kE4m3 ? kTile * D : kT;      // of K
  static constexpr int kRaw = KV == kE4m3 ? kRawTokens * D : KV == kKv4 ? kTile * kKv4Row<D> : 0;
  static constexpr int kTiles = 6 * kT + (KV == kKv4 ? kKv4Slots : 4) * kRaw;
  static constexpr int kLifts = KV == kKv4 ? 2 * 4 * kTile : 0;      // of the rows of K, then of V, by tile
  static constexpr int kTotal = kTiles + kTcFlags + kTcRows * 4 + kLifts + 1024;
};

__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
template <bool F16>
__device__ __forceinline__ uint32_t pack_16(float lo, float hi) {
  if constexpr (F16) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    return pack_bf16x2(lo, hi);
  }
}
__device__ __forceinline__ float pow2_of(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
// bits [lo, hi) of 32
__device__ __forceinline__ uint32_t bits_between(int lo, int hi) {
  lo = max(lo, 0);
  hi = min(hi, 32);
  return hi <= lo ? 0u : (0xFFFFFFFFu >> (32 - (hi - lo))) << lo;
}

// What a row sees of the walk's 128 tokens from tok0 on (base and beg in the walk's places): its context, and (trees, out of line: few tiles hold nodes, and what a mask needs would be held in
// registers beside the scores of those that do not) the nodes that row `qi` of the sequence sees.
__device__ __forceinline__ uint4 context_bits(const SpanParams& p, int base, int beg, int tok0) {
  uint32_t vis[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int t = tok0 + 32 * c;
    vis[c] = bits_between(beg - t, base - t) | bits_between(0, min(p.first, base) - t);
  }
  return make_uint4(vis[0], vis[1], vis[2], vis[3]);
}
__device__ __noinline__ uint4 tree_bits(const SpanParams& p, int q0, int qn, int kv_len, int gap, int qi, int tok0) {
  unsigned long long b[kSpanWords + 1] = {0, 0, 0, 0, 0};
  SpanRow row = span_row(p, q0, qn, kv_len + gap, qi, b);
  row.base -= gap;
  row.beg -= gap;
  const uint4 context = context_bits(p, row.base, row.beg, tok0);
  uint32_t vis[4] = {context.x, context.y, context.z, context.w};
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int n = tok0 + 32 * c - row.base;            // node of the word's first token
    if (n < 0) vis[c] |= n > -32 ? (uint32_t)(b[0] << -n) : 0u;
    else if (n < 64 * kSpanWords) vis[c] |= (uint32_t)((b[n >> 6] >> (n & 63)) | ((n & 63) ? b[(n >> 6) + 1] << (64 - (n & 63)) : 0ull));
  }
  return make_uint4(vis[0], vis[1], vis[2], vis[3]);
}
__device__ __forceinline__ uint4 row_bits(const SpanParams& p, int q0, int qn, int kv_len, int gap, int qi, int tok0) {
  if (qi < 0) return make_uint4(0, 0, 0, 0);
  if (p.tree_mask) return tree_bits(p, q0, qn, kv_len, gap, qi, tok0);
  const int base = max(kv_len - qn + qi + 1, 0);
  return context_bits(p, base, p.window > 0 ? max(0, base - p.window) : 0, tok0);
}

// tanh of the scaled scores of a tile in place, for a soft-cap.
__device__ __noinline__ void cap_scores(uint32_t t_s, float cap_in) {
#pragma unroll 1
  for (int c = 0; c < 8; ++c) {
    uint32_t s[16];
    tmem_ld_32x16(t_s + 16 * c, s);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = __float_as_uint(tanhf(__uint_as_float(s[i]) * cap_in));
    tmem_st_32x16(t_s + 16 * c, s);
  }
  tmem_st_wait();
}

__device__ __forceinline__ int4 lds_int4(const volatile int* at) {
  int4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(smem_u32(const_cast<const int*>(at))) : "memory");
  return v;
}
// Exponent field of a 4-bit row's largest magnitude, and how far the row is lifted beside a tile's unit of 2^up.
__device__ __forceinline__ int kv4_top_field(const Kv4Scale& k) {
  return (int)(__float_as_uint(fmaxf(fabsf(k.low), fabsf(fmaf(15.f, k.step, k.low)))) >> 23);
}
__device__ __forceinline__ int kv4_lift(int field, int up) { return min(max(126 + kKv4Top - field - up, 0), kKv4MostLift); }
__device__ __forceinline__ float kv4_lowered(uint32_t lifts, int byte) { return pow2_of(-(int)(lifts >> 8 * byte & 0xFF)); }

// A tile of rows that are lifted, widened (kv4_widen_f16) by kKv4Team warps, `at` of their lanes this one. Values that nobody sees, of places outside [beg, end) and
// behind `first`, are 0, and rows of values that read as NaN where `odd_met` is to know of them.
template <int D>
__device__ __noinline__ void widen_lifted(const uint8_t* src, uint8_t* to, int up, int at, int line_of_page, int line_of_half, bool is_v, int beg, int end, int first,
                                          int* odd_met, uint8_t* lifts) {
  constexpr int kEach = 4, kPieces = D / 8 / kEach;      // words of a row that a lane takes
#pragma unroll 1
  for (int i = at; i < kTile * kPieces; i += 32 * kKv4Team) {
    const int tok = i / kPieces, c0 = i % kPieces * kEach;
    const uint8_t* row = src + tok * kKv4Row<D>;
    uint32_t codes[kEach];
#pragma unroll
    for (int w = 0; w < kEach; ++w) codes[w] = *reinterpret_cast<const uint32_t*>(row + (c0 + w) * 4);
    const Kv4Scale k = kv4_scale_of(*reinterpret_cast<const uint32_t*>(row + D / 2));
    const bool there = tok < end && (tok >= beg || tok < first), nan = !(fabsf(k.step) < INFINITY);
    const int lift = kv4_lift(kv4_top_field(k), up);
    if (c0 == 0) lifts[tok] = (uint8_t)lift;
    uint32_t even = 0, odd = 0, low2 = 0;
    if (!is_v || (there && !(odd_met && nan))) {
      const int to_unit = up + lift;
      const float f1 = pow2_of(to_unit >> 1), f2 = pow2_of(to_unit - (to_unit >> 1)), step = k.step * f1 * f2, low = k.low * f1 * f2;
      even = pack_16<true>(step * 16777216.f, step * 16777216.f);
      odd = pack_16<true>(step * 1048576.f, step * 1048576.f);
      low2 = pack_16<true>(low, low);
    }
    if (is_v && odd_met && there && nan) *reinterpret_cast<volatile int*>(odd_met) = 1;
    uint8_t* line = to + (tok >> 4) * line_of_page + (tok & 15) * 128;
#pragma unroll
    for (int w = 0; w < kEach; ++w) {
      const int c = c0 + w;
      *reinterpret_cast<uint4*>(line + (c >> 3) * line_of_half + (((c & 7) ^ (tok & 7)) << 4)) = kv4_widen_f16(codes[w], even, odd, low2);
    }
  }
}

// Scores of a tile whose keys were lifted (`lifts`), or under a soft-cap (`cap_in`), in place.
__device__ __noinline__ void change_scores(uint32_t t_s, const uint8_t* lifts, float cap_in) {
#pragma unroll 1
  for (int c = 0; c < 8; ++c) {
    uint32_t s[16];
    tmem_ld_32x16(t_s + 16 * c, s);
    tmem_ld_wait();
    if (lifts) {
      const uint4 w = *reinterpret_cast<const uint4*>(lifts + 16 * c);
      const uint32_t of[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = __float_as_uint(__uint_as_float(s[i]) * kv4_lowered(of[i >> 2], i & 3));
    }
    if (cap_in > 0.f) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = __float_as_uint(tanhf(__uint_as_float(s[i]) * cap_in));
    }
    tmem_st_32x16(t_s + 16 * c, s);
  }
  tmem_st_wait();
}
// Weights of a tile whose values were lifted, in place (two to a word), and handed over, when the values are there, which write down by how much.
template <int D>
__device__ __noinline__ void lower_weights(uint32_t t_p, uint8_t* smem, int t, int group) {
  using S = TcSmem<D, kKv4>;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kTiles);
  mbar_wait(bars + kAtVReady + (t & 1), (t >> 1) & 1, reinterpret_cast<volatile int*>(bars + kAtFlags) + 1);
  const uint8_t* lifts = smem + S::kTiles + kTcFlags + kTcRows * 4 + (4 + (t & 3)) * kTile;
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {
    uint32_t w[16];
    tmem_ld_32x16(t_p + 16 * c, w);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint32_t of = *reinterpret_cast<const uint16_t*>(lifts + 32 * c + 2 * i);
      const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      w[i] = pack_16<true>(x.x * kv4_lowered(of, 0), x.y * kv4_lowered(of, 1));
    }
    tmem_st_32x16(t_p + 16 * c, w);
  }
  tmem_st_wait();
  tc_fence_before_sync();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bars + kAtPHalf + group);
}

// A row's softmax over one tile of 128 tokens: scores in registers, weights as 16-bit values over the scores' first columns, the first 64 of them
// handed over (p_half) before the others are computed; O of the warp is rescaled when a row's maximum has moved by more than 2^8, or its unit by `shrink`. Scores that the row
// does not see become -inf first, 32 columns at a time where some row of the warp does not see them all.
template <int D, bool F16>
__device__ __forceinline__ void softmax_tile(uint32_t t_s, uint32_t t_o, bool whole, const uint4& visible, float scale, bool have_o, uint64_t* p_half,
                                             float& m_used, float& l, float shrink = 1.f) {
  uint32_t s[4][32];
#pragma unroll
  for (int c = 0; c < 4; ++c) tmem_ld_32x32(t_s + 32 * c, s[c]);
  tmem_ld_wait();
  if (!whole) {
    const uint32_t vis[4] = {visible.x, visible.y, visible.z, visible.w};
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      if (__all_sync(0xffffffffu, vis[c] == 0xffffffffu)) continue;
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (!(vis[c] & (1u << j))) s[c][j] = 0xFF800000u;
    }
  }
  float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int i = 0; i < 128; i += 2)
    mx[(i >> 1) & 3] = fmaxf(fmaxf(mx[(i >> 1) & 3], __uint_as_float(s[i >> 5][i & 31])), __uint_as_float(s[i >> 5][(i & 31) + 1]));
  // the scale is positive, so it commutes with the maximum
  const float m = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale;
  const bool grow = m > m_used + kLazyRescale || (m_used == -INFINITY && m > -INFINITY);
  if (__any_sync(0xffffffffu, grow || shrink != 1.f)) {
    const float m_new = fmaxf(m_used, m);
    const float corr = m_new == -INFINITY ? 1.f : ex2(m_used - m_new);
    m_used = m_new;
    l *= corr;
    if (have_o) {
#pragma unroll 1
      for (int c = 0; c < D / 16; ++c) {
        uint32_t o[16];
        tmem_ld_32x16(t_o + 16 * c, o);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * (corr * shrink));
        tmem_st_32x16(t_o + 16 * c, o);
      }
    }
  }
  const float m_ref = m_used == -INFINITY ? 0.f : m_used - (F16 ? kTcLift : 0.f);
  uint64_t sum[2] = {0, 0};
  const uint64_t scale2 = pack2(scale, scale), ref2 = pack2(-m_ref, -m_ref);
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint32_t w[16];
#pragma unroll
    for (int j = 0; j < 32; j += 2) {
      const uint64_t x = fma2(pack2(__uint_as_float(s[c][j]), __uint_as_float(s[c][j + 1])), scale2, ref2);
      float2 e = unpack2(x);
      e.x = ex2(e.x); e.y = ex2(e.y);
      sum[j >> 1 & 1] = add2(sum[j >> 1 & 1], pack2(e.x, e.y));
      w[j >> 1] = pack_16<F16>(e.x, e.y);
    }
    tmem_st_32x16(t_s + 16 * c, w);
    if (c == 1) {
      tmem_st_wait();
      tc_fence_before_sync();
      __syncwarp();
      if ((threadIdx.x & 31) == 0) mbar_arrive(p_half);
    }
  }
  const float2 l0 = unpack2(sum[0]), l1 = unpack2(sum[1]);
  l += (l0.x + l0.y) + (l1.x + l1.y);
  tmem_st_wait();
}

// Rows of a tile that a thread goes through at a fixed distance, as (query row, head) pairs without a division for each.
struct RowWalk {
  int q, h, step_q, step_h, G;
  __device__ __forceinline__ RowWalk(int row, int step, int group) : G(group) {
    q = row / G; h = row - q * G;
    step_q = step / G; step_h = step - step_q * G;
  }
  __device__ __forceinline__ void next() {
    q += step_q; h += step_h;
    if (h >= G) { h -= G; ++q; }
  }
};

// K-major operand of 128 rows: 16-bit values in 128-byte swizzled rows, or rows of D bytes (128 or 64), swizzled over their length.
template <int D, bool BYTES>
__device__ __forceinline__ uint64_t desc_k_major(uint32_t saddr) {
  if constexpr (BYTES && D == 64)
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (uint64_t)1 << 16 | (uint64_t)(512 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)4 << 61;
  else
    return make_smem_desc_sw128(saddr);
}

// Queries of rows [0, tiles x 128) to shared memory in swizzled rows, by THREADS threads, `tid` of them this one. Beside an e4m3 cache: two e4m3
// pieces, of the value times a power of two per row (its largest magnitude is between 2^7 and 2^8 then) and of what that leaves, four bits each of
// a bf16's eight. Exact down to 2^-9 of the row's largest value, within 2^-17 of that value below. 4 bits: f16, times a power of two per row (between 2^14 and
// 2^15; within 2^-38 of the largest), dims in the order of kv4_widen_f16. bf16: asynchronous copies.
template <int D, int KV, int THREADS>
__device__ __forceinline__ void load_q(const SpanParams& p, int tid, uint8_t* sq, float* factors, int tiles, int q0, int row0, int n_rows, int kvh) {
  constexpr int C = D / 8, kStep = THREADS / C;        // rows between those of a thread
  const int c = tid % C, r0 = tid / C;
  RowWalk at(row0 + r0, kStep, p.group);
  const bf16* head = static_cast<const bf16*>(p.q) + (size_t)q0 * p.ldq + (size_t)kvh * p.group * D + c * 8;
  if constexpr (KV == kBf16) {
#pragma unroll 2
    for (int r = r0; r < tiles * kRows; r += kStep, at.next()) {
      const bool valid = r < n_rows;
      const bf16* src = valid ? head + (size_t)at.q * p.ldq + (size_t)at.h * D : static_cast<const bf16*>(p.q);
      uint8_t* dst = sq + (r >> 7) * tile_bytes<D>() + (c >> 3) * kHalf + (r & (kRows - 1)) * 128 + (((c & 7) ^ (r & 7)) << 4);
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(valid ? 16 : 0) : "memory");
      if (c == 0) factors[r] = p.scale_log2;
    }
  } else {
    constexpr int kBatch = 4;                          // loads on their way at once
#pragma unroll 1
    for (int i0 = 0; i0 * kStep < tiles * kRows; i0 += kBatch) {
      uint4 v[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i, at.next()) {
        const int r = r0 + (i0 + i) * kStep;
        v[i] = r < n_rows ? __ldg(reinterpret_cast<const uint4*>(head + (size_t)at.q * p.ldq + (size_t)at.h * D)) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int r = r0 + (i0 + i) * kStep, rr = r & (kRows - 1);
        const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
        uint32_t most = __vmaxu2(__vmaxu2(w[0] & 0x7FFF7FFFu, w[1] & 0x7FFF7FFFu), __vmaxu2(w[2] & 0x7FFF7FFFu, w[3] & 0x7FFF7FFFu));
#pragma unroll
        for (int o = C / 2; o > 0; o >>= 1) most = __vmaxu2(most, __shfl_xor_sync(0xffffffffu, most, o));
        const int top = (int)(max(most & 0xFFFFu, most >> 16) >> 7);      // largest exponent field of the row
        const bool odd = top == 0xFF;                  // an infinity or a NaN: no score of the row is a number (a soft-cap would make 1 of an infinite one: NaN here)
        const int up = odd ? 0 : min(127 + (KV == kKv4 ? 14 : 7) - top, 126);
        const float f = odd ? __int_as_float(0x7FC00000) : __uint_as_float((uint32_t)(127 + up) << 23);
        if constexpr (KV == kKv4) {
          if (r >= tiles * kRows) continue;
          uint32_t h[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 x = unpack_bf16x2(w[e]);
            h[e] = pack_16<true>(x.x * f, x.y * f);
          }
          *reinterpret_cast<uint4*>(sq + (r >> 7) * tile_bytes<D>() + (c >> 3) * kHalf + rr * 128 + (((c & 7) ^ (rr & 7)) << 4)) =
              make_uint4(__byte_perm(h[0], h[2], 0x5410), __byte_perm(h[0], h[2], 0x7632), __byte_perm(h[1], h[3], 0x5410), __byte_perm(h[1], h[3], 0x7632));
          if (c == 0) factors[r] = span_factor(p.scale_log2, up);
          continue;
        }
        uint32_t high[2] = {0, 0}, low[2] = {0, 0};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float2 x = unpack_bf16x2(w[e]);
          x.x *= f; x.y *= f;
          const uint32_t a = __nv_cvt_float2_to_fp8x2(x, __NV_SATFINITE, __NV_E4M3);
          const uint2 h = e4m3x4_to_f16(a);
          const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&h.x));
          const uint32_t b = __nv_cvt_float2_to_fp8x2(make_float2(x.x - y.x, x.y - y.y), __NV_SATFINITE, __NV_E4M3);
          high[e >> 1] |= a << (16 * (e & 1));
          low[e >> 1] |= b << (16 * (e & 1));
        }
        if (r >= tiles * kRows) continue;
        uint8_t* at8 = sq + (r >> 7) * tile_bytes<D>() + rr * D + (((c >> 1) ^ (D == 128 ? rr & 7 : (rr >> 1) & 3)) << 4) + (c & 1) * 8;
        *reinterpret_cast<uint2*>(at8) = make_uint2(high[0], high[1]);
        *reinterpret_cast<uint2*>(at8 + kRows * D) = make_uint2(low[0], low[1]);
        if (c == 0) factors[r] = span_factor(p.scale_log2, up);
      }
    }
  }
}
__device__ __forceinline__ void q_loaded() {
  asm volatile("cp.async.wait_all;" ::: "memory");
  fence_proxy_async_smem();
}

// `bytes` (a multiple of 16) that lie in a row, to shared memory; both on 16-byte boundaries.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes),
               "r"(smem_u32(bar)) : "memory");
}

// First pool row of a page of a tile, or `none` (behind the pool: TMA fills it with zeros) for pages that nobody sees and pages that are not there.
struct PageRows {
  const SpanParams& p;
  const int* table;
  int kvh, head, gap, count, none;         // of the walk's `count` pages those from `head` on lie `gap` further in the text
  __device__ __forceinline__ int page_of(int i) const { return i < head ? i : i + gap; }
  __device__ __forceinline__ int operator()(int i, bool& bad) const {
    if (i >= count) return none;
    const int page = page_of(i), b = span_block(p, table, page);
    bad |= b < 0;
    return b < 0 ? none : (int)span_pool_row(p, b, kvh, page);
  }
};

// The same for the tiles of a walk, by a whole warp: a lane looks up one page, so that of four tiles at a time, one round ahead. (Page after page by
// all lanes, in front of every tile, the producers took longer than the products.)
struct PagesAhead {
  const PageRows& rows;
  int t0, n_tiles, now, next;
  bool bad;
  __device__ __forceinline__ PagesAhead(const PageRows& r, int first, int n) : rows(r), t0(first), n_tiles(n), now(0), next(0), bad(false) {
    next = look(0);
  }
  __device__ __forceinline__ int look(int it) {
    const int at = it + ((threadIdx.x & 31) >> 3);
    return at < n_tiles ? rows((t0 + at) * kTilePages + (threadIdx.x & 7), bad) : rows.none;
  }
  __device__ __forceinline__ void to(int it) {         // tile after tile
    if ((it & 3) == 0) { now = next; next = look(it + 4); }
  }
  __device__ __forceinline__ int row(int it, int page) const { return __shfl_sync(0xffffffffu, now, (it & 3) * 8 + page); }
};

// Sum of 0 x value over 16-bit values, a NaN once there was an infinity or a NaN among them.
template <bool F16>
__device__ __forceinline__ void odd_sum(uint32_t& sum, uint32_t w) {
  if constexpr (F16) asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(sum) : "r"(w), "r"(0u));
  else asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(sum) : "r"(w), "r"(0u));
}
// Infinities and NaN of 16-bit values set to zero.
__device__ __forceinline__ uint32_t without_odd_bf16(uint32_t w) {
  return ((w & 0x7F80u) == 0x7F80u ? 0u : w & 0xFFFFu) | ((w & 0x7F800000u) == 0x7F800000u ? 0u : w & 0xFFFF0000u);
}
__device__ __forceinline__ uint32_t without_odd_f16(uint32_t w) {
  return ((w & 0x7C00u) == 0x7C00u ? 0u : w & 0xFFFFu) | ((w & 0x7C000000u) == 0x7C000000u ? 0u : w & 0xFFFF0000u);
}

// Into how many pieces the walk of an item is cut. An item's share of all the work, counted in tiles of 128 rows from the lengths, times the number of
// SMs is the number of SMs that it could keep; a piece costs a start, partial sums and their way through memory, so that is rounded down, but for
// items that would hold two SMs almost. us of 32 query and 8 key heads of 128: 16 trees of 64 nodes behind 6000 tokens: 107 in one piece each,
// 137 in two, 161 in four; 4 of 32: 67 in one, 36 in four, 49 in six; 16 of 64 behind 1000 to 12,000: 182 in one each, 201 in pieces of up to 13 tiles,
// 157 by this rule, 172 where two pieces begin at 1.35 SMs (from captured graphs, before the last steps: 152 by the rule since).
__device__ __forceinline__ int tiles_of(const SpanParams& p, int qn, int kv_len) {
  const int tiles = max((kv_len + kTile - 1) / kTile, 1);
  return p.window > 0 ? (int)min((long long)tiles, ((long long)p.window + p.first + min(qn, kTcRows / p.group + 2) + 2 * kPage) / kTile + 1) : tiles;
}
__device__ __forceinline__ float weight_of_rows(int rows) { return rows > kRows ? 2.f : 1.f; }
__device__ __forceinline__ int pieces_of(const SpanParams& p, int n_rows, int tiles) {
  float total = 0.f;
  for (int s0 = 0; s0 < p.num_seqs; s0 += 32) {
    const int s = s0 + (threadIdx.x & 31);
    float mine = 0.f;
    if (s < p.num_seqs) {
      int q0, qn, kv_len;
      span_lengths(p, s, false, q0, qn, kv_len);
      const int rows = qn * p.group, whole = rows / kTcRows;
      if (rows > p.rows_from) mine = (2.f * whole + (rows > whole * kTcRows ? weight_of_rows(rows - whole * kTcRows) : 0.f)) * tiles_of(p, qn, kv_len);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    total += mine;
  }
  const float sms = weight_of_rows(n_rows) * tiles * p.sms / (total * p.hkv);
  return max(1, min(min(sms < 2.f ? (sms >= 1.7f ? 2 : 1) : (int)sms, p.splits), tiles));
}

// What the rows of a tile see between them and what all of them see, by a warp for itself: the end of the context that all see, where windows begin
// first and last, the end of what any sees.
struct TileSees {
  int min_base, min_beg, max_beg, end;
};
__device__ __forceinline__ TileSees tile_sees(const SpanParams& p, int q0, int qn, int kv_len, int row0, int n_rows) {
  TileSees t;
  const int first = row0 / p.group, last = (row0 + n_rows - 1) / p.group;      // query rows
  if (p.tree_mask) {
    int a = INT_MAX, b = INT_MAX, d = 0;
    for (int qi = first + (threadIdx.x & 31); qi <= last; qi += 32) {
      unsigned long long bits[kSpanWords];
      const SpanRow r = span_row(p, q0, qn, kv_len, qi, bits);
      a = min(a, r.base); b = min(b, r.beg); d = max(d, r.beg);
    }
    t.min_base = __reduce_min_sync(0xffffffffu, a);
    t.min_beg = __reduce_min_sync(0xffffffffu, b);
    t.max_beg = __reduce_max_sync(0xffffffffu, d);
    t.end = kv_len;
  } else {
    t.min_base = max(kv_len - qn + first + 1, 0);
    t.end = max(kv_len - qn + last + 1, 0);
    t.min_beg = p.window > 0 ? max(t.min_base - p.window, 0) : 0;
    t.max_beg = p.window > 0 ? max(t.end - p.window, 0) : 0;
  }
  return t;
}

template <int D, int KV, bool SEARCH>
__global__ void __launch_bounds__(tc_threads<KV>(), 1)
span_tc_kernel(const __grid_constant__ CUtensorMap tma_k, const __grid_constant__ CUtensorMap tma_v, const __grid_constant__ SpanParams p, int row_tiles, int halved) {
  using S = TcSmem<D, KV>;
  constexpr int TB = S::kT;
  constexpr bool KV8 = KV == kE4m3, KV4 = KV == kKv4;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *sq = smem, *sk = smem + 2 * TB, *sv = smem + 4 * TB;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kTiles);
  constexpr int KS = S::kStages;
  uint64_t *k_full = bars, *k_empty = bars + 4;                                               // [KS] by stage
  uint64_t *v_full = bars + 8, *v_empty = bars + 10, *v_ready = bars + kAtVReady;                    // [2] by stage; ready: looked through, or widened
  uint64_t *s_full = bars + 14, *p_half = bars + kAtPHalf, *p_ready = bars + 18;                    // [2] by softmax group
  uint64_t *o_done = bars + 20, *q_full = bars + 21;
  uint64_t *raw_full = bars + 22, *raw_empty = bars + 30;                                     // [8] by slot
  // A 4-bit cache has three raw slots, and units that softmax has to know, by stage of V [2]; and a barrier that nobody waits for
  uint64_t *v_unit = raw_full + 4, *nobody = raw_full + 7;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kAtFlags);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* odd_met = reinterpret_cast<int*>(tmem_slot + 2);     // values were taken out of tiles of V
  // [4] by tile of a 4-bit cache: keys and values are times 2 to x and y, rows are lifted where z and w are not 0
  volatile int* units = reinterpret_cast<volatile int*>(bars + 40);
  float* factors = reinterpret_cast<float*>(smem + S::kTiles + kTcFlags);
  uint8_t *k_lifts = smem + S::kTiles + kTcFlags + kTcRows * 4, *v_lifts = k_lifts + 4 * kTile;      // [4][kTile]
  static_assert(40 * 8 + 16 * 4 <= kTcFlags && kTcFlags % 16 == 0, "barriers and flags");

  const int warp = uniform_warp(), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&v_full[i], 1); mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1); mbar_init(&p_half[i], 4); mbar_init(&p_ready[i], 4); mbar_init(&v_ready[i], KV4 ? kKv4Team : KV8 ? kWideners : 1);
    }
    for (int i = 0; i < KS; ++i) { mbar_init(&k_full[i], KV8 ? 1 : KV4 ? kKv4Team : D / 64); mbar_init(&k_empty[i], 1); }
    for (int i = 0; i < 8; ++i) { mbar_init(&raw_full[i], 1); mbar_init(&raw_empty[i], KV4 ? kKv4Team : kWideners); }
    mbar_init(o_done, 1); mbar_init(q_full, kQThreads<KV> / 32);
    *abort_flag = 0;
    *odd_met = 0;
    fence_barrier_init();
  }
  if (!KV4 && warp == 8 && lane == 0) { tma_prefetch_desc(&tma_k); if (!KV8) tma_prefetch_desc(&tma_v); }
  pdl_wait();
  const int split = blockIdx.y;
  // Whole tiles of the longest sequence come first, those that see the most before others; then what is left of the rows. The last `halved` of the whole
  // ones are two CTAs of half the rows each.
  int rest = blockIdx.x, half = -1;
  const int from_halves = SEARCH ? INT_MAX / 2 : row_tiles * p.num_seqs * p.hkv - halved;
  if (rest >= from_halves + 2 * halved) {
    rest -= halved;
  } else if (rest >= from_halves) {
    half = (rest - from_halves) & 1;
    rest = from_halves + ((rest - from_halves) >> 1);
  }
  const int kvh = rest % p.hkv;
  rest /= p.hkv;
  const int at_tile = rest / p.num_seqs;
  int seq = rest % p.num_seqs, tile = at_tile < row_tiles ? row_tiles - 1 - at_tile : at_tile;
  if constexpr (SEARCH) {
    if (!span_find(p, kTcRows, p.rows_from, INT_MAX, rest, blockIdx.x == gridDim.x - 1 && split == 0, seq, tile)) return;
  }
  int q0, qn, kv_len;
  if (!span_lengths(p, seq, threadIdx.x == 0, q0, qn, kv_len)) return;
  const int G = p.group, all_rows = qn * G, row0 = tile * kTcRows + (half > 0 ? kRows : 0);
  if (all_rows <= p.rows_from || row0 >= all_rows) return;
  const int n_rows = min(half < 0 ? kTcRows : kRows, all_rows - row0);
  const int walk = tiles_of(p, qn, kv_len), pieces = p.splits > 1 ? pieces_of(p, n_rows, walk) : 1;
  if (split >= pieces) return;
  const bool two = n_rows > kRows;                     // two row tiles that share K and V, or two groups that share a row tile
  if (warp == 9) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  pdl_launch_dependents();                             // not before the allocation
  // Queries: the softmax groups, and beside an e4m3 cache, where there is more to it than to copy them, four of the warps that wait for V. (Whoever
  // asks for K and V is not among them.)
  const bool q_too = KV8 && warp >= 12;
  if (warp < 8 || q_too) load_q<D, KV, kQThreads<KV>>(p, warp < 8 ? (int)threadIdx.x : (int)threadIdx.x - 128, sq, factors, two ? 2 : 1, q0, row0, n_rows, kvh);

  const int group = warp >> 2;                         // of softmax warps
  const int r_first = (two ? group * kRows : 0) + (warp & 3) * 32, r = r_first + lane;
  const int qi = warp < 8 && r < n_rows ? (row0 + r) / G : -1;
  const TileSees sees = tile_sees(p, q0, qn, kv_len, row0, n_rows);
  // The walk goes over the first tokens' pages and those from the window on as if they lay one behind the other: from here on places are the walk's,
  // in which context, windows and lengths are what they are in a text without the `gap`. (A text with a gap has its context behind it, so no first
  // token lies elsewhere. Tiles of 128 tokens of the text each, 3 x 777 rows under a window of 512 with 16 first tokens, 64 query and 8 key heads of 64,
  // e4m3: 90 us; so: 81.)
  const SpanRange range = span_range(p, kPage, sees.min_beg, sees.end);
  const int gap = (range.lo - range.head) * kPage, min_base = sees.min_base - gap, max_beg = sees.max_beg - gap;
  kv_len -= gap;
  const int any_beg = sees.min_beg - gap, any_end = sees.end - gap;      // tokens that some row sees, the first ones aside
  const int per_piece = (walk + pieces - 1) / pieces;      // (the last one goes on to the end, should that be further)
  const int n_all = (range.count + kTilePages - 1) / kTilePages, t0 = min(split * per_piece, n_all), n_tiles = split == pieces - 1 ? n_all - t0 : min(per_piece, n_all - t0);
  const int shift = two ? 1 : 0, n_items = n_tiles << shift;
  // not every row of the CTA sees the whole tile
  auto partial = [&](int tok0) { return !(tok0 + kTile <= min_base && (tok0 >= max_beg || tok0 + kTile <= p.first)); };
  const PageRows page_rows{p, p.block_tables + (size_t)seq * p.max_blocks, kvh, range.head, range.lo - range.head, range.count,
                           (int)(p.num_blocks * p.hkv * p.block_pages * kPage)};

  // The block was launched with 168 registers a thread (e4m3 and 4 bits: 128): 256 x 208 + 128 x 88 = 384 x 168, 256 x 192 + 256 x 64 = 512 x 128,
  // or 256 x 176 + 256 x 80 (4 bits, 2 x 2048 rows behind 2500 and 6143 tokens: 512 us; with 64, 72 and 88 for those that widen 576, 534 and 526).
  if (warp >= 8) {
    if constexpr (KV4) asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    else if constexpr (KV8) asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    bool bad = false;
    if (q_too) {
      q_loaded();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
      asm volatile("bar.arrive 2, 384;" ::: "memory");
    }
    if (warp == 9) {
      constexpr int fmt = KV == kBf16 ? 1 : 0;
      constexpr uint32_t idesc_s = make_idesc(128, 128, fmt, fmt);      // (e4m3 x e4m3 has the same bits as f16 x f16)
      constexpr uint32_t idesc_pv = make_idesc(128, D, fmt, fmt) | (1u << 16);     // B is MN-major
      const uint64_t dq = desc_k_major<D, KV8>(smem_u32(sq)), dk = desc_k_major<D, KV8>(smem_u32(sk));
      // V: [page][D / 64][16][64]; at D = 128 the second 64-wide atom of a row lies half a page further
      const uint64_t dv = (uint64_t)((smem_u32(sv) & 0x3FFFFu) >> 4) | (uint64_t)((D == 128 ? 2048 : 1024) >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 |
                          (uint64_t)1 << 46 | (uint64_t)2 << 61;
      // The group of an item is known at compile time, and whether there are two row tiles: addresses and descriptors stay in uniform registers.
      auto issue_s = [&](auto two_tiles, auto g, int n) {
        constexpr bool kTwo = decltype(two_tiles)::value;
        constexpr int kG = decltype(g)::value;
        const int t = kTwo ? n >> 1 : n, b = kTwo || KV8 ? t & (KS - 1) : kG;
        const uint64_t a0 = dq + (uint64_t)(kTwo ? kG * (TB >> 4) : 0), b0 = dk + (uint64_t)(b * (S::kK >> 4));
        if constexpr (KV8) {
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {           // both pieces of Q on the same K
            const int piece = k / (D / 32), off = (k % (D / 32)) * 2;
            tc_mma_f8f6f4(tmem_base + 128 * kG, a0 + (uint64_t)(piece * (kRows * D >> 4) + off), b0 + (uint64_t)off, idesc_s, k > 0);
          }
        } else {
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t off = ((k >> 2) * kHalf + (k & 3) * 32) >> 4;
            tc_mma_bf16(tmem_base + 128 * kG, a0 + off, b0 + off, idesc_s, k > 0);
          }
        }
        tc_commit(&s_full[kG]);
        if (!kTwo || kG) tc_commit(&k_empty[b]);
      };
      auto issue_pv = [&](auto g, int b, bool first, auto part) {            // over tokens [64 part, 64 part + 64)
        constexpr int kG = decltype(g)::value, kPart = decltype(part)::value;
        const uint32_t t_p = tmem_base + 128 * kG, t_o = tmem_base + 256 + 128 * kG;
#pragma unroll
        for (int k = 4 * kPart; k < 4 * kPart + 4; ++k)
          tc_mma_bf16_ts(t_o, t_p + 8 * k, dv + (uint64_t)(b * (TB >> 4)) + k * (D / 64) * (2048 >> 4), idesc_pv, (!first || k > 0) ? 1u : 0u);
      };
      auto step = [&](auto two_tiles, auto g, int n) {      // PV of item n, S of item n + 2
        constexpr bool kTwo = decltype(two_tiles)::value;
        constexpr int kG = decltype(g)::value;
        const int t = kTwo ? n >> 1 : n, b = kTwo ? t & 1 : kG, k = n >> 1;
        if (!mbar_wait(&v_ready[b], (t >> 1) & 1, abort_flag) || !mbar_wait(&p_half[kG], k & 1, abort_flag)) return false;
        tc_fence_after_sync();
        issue_pv(g, b, k == 0, Int<0>{});
        if (!mbar_wait(&p_ready[kG], k & 1, abort_flag)) return false;
        tc_fence_after_sync();
        issue_pv(g, b, k == 0, Int<1>{});
        if (!kTwo || kG) tc_commit(&v_empty[b]);
        if (n + 2 < n_items) {
          const int t2 = kTwo ? t + 1 : t + 2;
          if (!mbar_wait(&k_full[kTwo || KV8 ? t2 & (KS - 1) : kG], (t2 / KS) & 1, abort_flag)) return false;
          tc_fence_after_sync();
          issue_s(two_tiles, g, n + 2);
        }
        return true;
      };
      auto walk = [&](auto two_tiles) {
        constexpr bool kTwo = decltype(two_tiles)::value;
        if (!mbar_wait(q_full, 0, abort_flag) || !mbar_wait(&k_full[0], 0, abort_flag)) return;
        tc_fence_after_sync();
        issue_s(two_tiles, Int<0>{}, 0);
        if (n_items > 1) {
          if (!kTwo && !mbar_wait(&k_full[1], 0, abort_flag)) return;
          tc_fence_after_sync();
          issue_s(two_tiles, Int<1>{}, 1);
        }
        for (int n = 0; n < n_items; n += 2) {
          if (!step(two_tiles, Int<0>{}, n)) return;
          if (n + 1 < n_items && !step(two_tiles, Int<1>{}, n + 1)) return;
        }
        tc_commit(o_done);
      };
      if (n_items > 0 && elect_one()) {
        if (two) walk(Bool<true>{});
        else walk(Bool<false>{});
      }
      __syncwarp();
    } else if constexpr (KV4) {
      // Warp 8 asks for tiles, K0, V0, K1, V1, ..., through a ring of slots. Three warps widen those of K, three those of V, each a part of every one. (All six
      // one tile after the other, each with its waits and its search for a unit: 600 us where so 534, 2 x 2048 rows behind 2500 and 6143 tokens.)
      const int part = (warp - 10) % kKv4Team, pieces = 2 * n_tiles;
      PagesAhead pages_k(page_rows, t0, warp == 8 ? n_tiles : 0), pages_v(page_rows, t0, warp == 8 ? n_tiles : 0);
      constexpr int kPageBytes = kPage * kKv4Row<D>;
      bool ok = true;
      for (int x = 0; ok && warp == 8 && x < pieces; ++x) {
        const int it = x >> 1, slot = x % kKv4Slots;
        const bool is_v = x & 1;
        if (is_v) pages_v.to(it);
        else pages_k.to(it);
        if (x >= kKv4Slots && !mbar_wait_warp(&raw_empty[slot], (x / kKv4Slots - 1) & 1, abort_flag)) { ok = false; break; }
        const int now = is_v ? pages_v.now : pages_k.now;
        uint8_t* at = smem + 6 * TB + slot * S::kRaw;
        // A page is 16 rows in one piece: the lanes that looked the tile's pages up ask for one each. One that nobody sees, or that is not there, is zeros.
        const int pg = lane - (it & 3) * kTilePages;
        const bool mine = pg >= 0 && pg < kTilePages && now != page_rows.none;
        const uint32_t asked = __ballot_sync(0xffffffffu, mine) >> ((it & 3) * kTilePages);
        if (asked != (1u << kTilePages) - 1) {
          for (int i = lane; i < S::kRaw / 16; i += 32)
            if (!(asked >> (i / (kPageBytes / 16)) & 1)) *reinterpret_cast<uint4*>(at + i * 16) = make_uint4(0, 0, 0, 0);
          fence_proxy_async_smem();                    // (a later tile comes by a bulk copy)
          __syncwarp();
        }
        if (lane == 0) mbar_expect_tx(&raw_full[slot], __popc(asked) * kPageBytes);
        __syncwarp();
        if (mine) bulk_load(at + pg * kPageBytes, static_cast<const uint8_t*>(is_v ? p.v_cache : p.k_cache) + (size_t)now * kKv4Row<D>, kPageBytes, &raw_full[slot]);
        __syncwarp();
      }
      // A lane takes two words of a row, half a row apart. Steps and lowest values of the warp's rows are made ready a lane to a row.
      constexpr int kWords = D / 16, kTurnRows = 32 / kWords, kTurns = kTile / kTurnRows, kMost = (kTurns + kKv4Team - 1) / kKv4Team;
      constexpr int kBatch = 32 / kTurnRows;           // turns whose rows 32 lanes have
      const int word = lane % kWords, sub = lane / kWords;
      const bool is_v = warp >= 10 + kKv4Team;
      int up_v = 127;                                  // values are times 2^up_v
      for (int it = 0; ok && warp >= 10 && it < n_tiles; ++it) {
        const int x = 2 * it + is_v, slot = x % kKv4Slots, b = it & 1, tile0 = (t0 + it) * kTile;
        const bool look = partial(tile0);
        if (!mbar_wait_warp(&raw_full[slot], x / kKv4Slots & 1, abort_flag)) { ok = false; break; }
        const uint8_t* src = smem + 6 * TB + slot * S::kRaw;
        auto seen = [&](int tok) { return tok < any_end && (tok >= any_beg || tok < p.first); };
        // The largest magnitude of the tile that some row sees, by every warp for itself, a lane to four rows. It goes below 2^kKv4Top; that of values, whose
        // sums go over all tiles, only where it is above that of those before, with room for four times as much. (By warp 8 for all of them, in turn with its
        // copies: 670 us for the 2 x 2048 rows.)
        uint32_t ends = 0;                             // the largest field, and 255 less the least (rows of zeros, and of values that are no numbers, aside)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t field = kv4_top_field(kv4_scale_of(*reinterpret_cast<const uint32_t*>(src + (32 * i + lane) * kKv4Row<D> + D / 2)));
          if ((!look || seen(tile0 + 32 * i + lane)) && field - 1 < 254) ends = __vmaxu2(ends, 0x00FF0000u - 0xFFFFu * field);
        }
        const uint32_t most = __reduce_max_sync(0xffffffffu, ends & 0xFFFFu);
        int up = 126 + kKv4Top - (int)most;
        if (is_v) up = up_v = up < up_v ? up - 2 : up_v;
        up = min(up, 120);
        const bool lifted = __any_sync(0xffffffffu, 255 - (int)(ends >> 16) + up < kKv4Even);
        const float f1 = pow2_of(up >> 1), f2 = pow2_of(up - (up >> 1));
        if (it >= 2 && !mbar_wait_warp(is_v ? &v_empty[b] : &k_empty[b], ((it >> 1) - 1) & 1, abort_flag)) { ok = false; break; }
        if (part == 0 && lane == 0) {
          units[4 * (it & 3) + is_v] = up;
          units[4 * (it & 3) + 2 + is_v] = lifted;
          if (is_v) mbar_arrive(&v_unit[b]);
        }
        uint8_t* const to = is_v ? sv + b * TB : sk + b * TB;
        // of row tok: V: [page][half][16][64]
        const int line_of_page = is_v ? (D / 64) * 2048 : 16 * 128, line_of_half = is_v ? 2048 : kHalf;
        if (lifted) {
          widen_lifted<D>(src, to, up, part * 32 + lane, line_of_page, line_of_half, is_v, look ? any_beg - tile0 : 0, look ? any_end - tile0 : kTile, p.first - tile0,
                          look ? odd_met : nullptr, (is_v ? v_lifts : k_lifts) + (it & 3) * kTile);
        } else
#pragma unroll
        for (int u0 = 0; u0 < kMost; u0 += kBatch) {
          uint32_t even = 0, odd = 0, low2 = 0;        // of a row of values that reads as NaN, or that nobody sees: 0
          const int mine = (part + kKv4Team * (u0 + lane / kTurnRows)) * kTurnRows + lane % kTurnRows;
          if (mine < kTile) {
            const Kv4Scale k = kv4_scale_of(*reinterpret_cast<const uint32_t*>(src + mine * kKv4Row<D> + D / 2));
            const bool there = !look || seen(tile0 + mine), nan = !(fabsf(k.step) < INFINITY);
            if (!is_v || (there && !(look && nan))) {
              const float step = k.step * f1 * f2, low = k.low * f1 * f2;
              even = pack_16<true>(step * 16777216.f, step * 16777216.f);
              odd = pack_16<true>(step * 1048576.f, step * 1048576.f);
              low2 = pack_16<true>(low, low);
            }
            if (is_v && look && there && nan) *reinterpret_cast<volatile int*>(odd_met) = 1;
          }
          constexpr int kHere = kBatch;
          uint32_t w[kHere][2];
          const uint8_t* from = src + ((part + kKv4Team * u0) * kTurnRows + sub) * kKv4Row<D> + word * 4;
#pragma unroll
          for (int u = 0; u < kHere; ++u)
            if (u0 + u < kMost && part + kKv4Team * (u0 + u) < kTurns) {
              w[u][0] = *reinterpret_cast<const uint32_t*>(from + u * kKv4Team * kTurnRows * kKv4Row<D>);
              w[u][1] = *reinterpret_cast<const uint32_t*>(from + u * kKv4Team * kTurnRows * kKv4Row<D> + kWords * 4);
            }
#pragma unroll
          for (int u = 0; u < kHere; ++u) {
            if (u0 + u >= kMost) continue;
            const uint32_t e = __shfl_sync(0xffffffffu, even, u * kTurnRows + sub), o = __shfl_sync(0xffffffffu, odd, u * kTurnRows + sub);
            const uint32_t l = __shfl_sync(0xffffffffu, low2, u * kTurnRows + sub);
            if (part + kKv4Team * (u0 + u) >= kTurns) continue;
            const int tok = (part + kKv4Team * (u0 + u)) * kTurnRows + sub;
            uint8_t* line = to + (tok >> 4) * line_of_page + (tok & 15) * 128;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int c = word + h * kWords;
              *reinterpret_cast<uint4*>(line + (c >> 3) * line_of_half + (((c & 7) ^ (tok & 7)) << 4)) = kv4_widen_f16(w[u][h], e, o, l);
            }
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&raw_empty[slot]);
          mbar_arrive(is_v ? &v_ready[b] : &k_full[b]);
        }
        __syncwarp();
      }
      bad = pages_k.bad;
    } else if constexpr (!KV8) {
      const bool is_v = warp == 11;
      const int half = warp == 10 ? 1 : 0;
      PagesAhead pages(page_rows, t0, n_tiles);
      auto ask = [&](int it) {                         // all lanes; false: gave up
        const int b = it & 1;
        int rows[kTilePages];
        pages.to(it);
#pragma unroll
        for (int pg = 0; pg < kTilePages; ++pg) rows[pg] = pages.row(it, pg);
        if (it >= 2 && !mbar_wait_warp(is_v ? &v_empty[b] : &k_empty[b], ((it >> 1) - 1) & 1, abort_flag)) return false;
        if (elect_one()) {
          if (is_v) {
            mbar_expect_tx(&v_full[b], TB);
#pragma unroll
            for (int pg = 0; pg < kTilePages; ++pg) tma_load_3d(sv + b * TB + pg * (D / 64) * 2048, &tma_v, &v_full[b], 0, rows[pg], 0);
          } else {
            mbar_expect_tx(&k_full[b], kHalf);
#pragma unroll
            for (int pg = 0; pg < kTilePages; ++pg) tma_load_2d(sk + b * TB + half * kHalf + pg * 2048, &tma_k, &k_full[b], 64 * half, rows[pg]);
          }
        }
        __syncwarp();
        return true;
      };
      if (!is_v) {
        for (int it = 0; it < n_tiles && (half == 0 || D == 128); ++it)
          if (!ask(it)) break;
      } else if (n_tiles > 0) {
        bool ok = ask(0);
        for (int it = 0; ok && it < n_tiles; ++it) {
          if (it == 0 && n_tiles > 1) ok = ask(1);
          const int b = it & 1;
          ok = ok && mbar_wait_warp(&v_full[b], (it >> 1) & 1, abort_flag);
          if (!ok) break;
          if (partial((t0 + it) * kTile)) {
            uint4* v = reinterpret_cast<uint4*>(sv + b * TB);
            uint32_t sum[4] = {0, 0, 0, 0};
#pragma unroll 8
            for (int i = lane; i < TB / 16; i += 32) {
              const uint4 w = v[i];
              odd_sum<false>(sum[0], w.x); odd_sum<false>(sum[1], w.y); odd_sum<false>(sum[2], w.z); odd_sum<false>(sum[3], w.w);
            }
            if (__any_sync(0xffffffffu, odd_bf16x2(sum[0]) || odd_bf16x2(sum[1]) || odd_bf16x2(sum[2]) || odd_bf16x2(sum[3]))) {
              for (int i = lane; i < TB / 16; i += 32) {
                uint4 w = v[i];
                w.x = without_odd_bf16(w.x); w.y = without_odd_bf16(w.y); w.z = without_odd_bf16(w.z); w.w = without_odd_bf16(w.w);
                v[i] = w;
              }
              fence_proxy_async_smem();
              if (lane == 0) atomicOr(odd_met, 1);
              __syncwarp();
            }
          }
          if (lane == 0) mbar_arrive(&v_ready[b]);
          if (it >= 1 && it + 1 < n_tiles) ok = ask(it + 1);
        }
      }
      bad = pages.bad;
    } else {
      // Warp 8 asks for tiles of K, and for V in raw halves of tiles through a ring of slots; each of the other six warps widens a part of every half.
      const int part = warp - 10;
      const int slots = two ? 4 : 8, turn = two ? 2 : 3, pieces = 2 * n_tiles;
      auto slot_at = [&](int s) { return s < 4 ? smem + 6 * TB + s * S::kRaw : sq + TB + (s - 4) * S::kRaw; };      // the unused tile of Q
      PagesAhead pages(page_rows, t0, warp == 8 ? n_tiles : 0);
      auto ask_k = [&](int it) {                       // warp 8
        const int b = it & (KS - 1);
        int rows[kTilePages];
        pages.to(it);
#pragma unroll
        for (int pg = 0; pg < kTilePages; ++pg) rows[pg] = pages.row(it, pg);
        if (it >= KS && !mbar_wait_warp(&k_empty[b], (it / KS - 1) & 1, abort_flag)) return false;
        if (elect_one()) {
          mbar_expect_tx(&k_full[b], S::kK);
#pragma unroll
          for (int pg = 0; pg < kTilePages; ++pg) tma_load_2d(sk + b * S::kK + pg * kPage * D, &tma_k, &k_full[b], 0, rows[pg]);
        }
        __syncwarp();
        return true;
      };
      auto ask = [&](int j) {                          // warp 8
        const int it = j >> 1, s = j & (slots - 1);
        if (j >= slots && !mbar_wait_warp(&raw_empty[s], ((j >> turn) - 1) & 1, abort_flag)) return false;
        // A page is 16 D bytes in a row: the four lanes that looked the piece's pages up ask for one each. One that nobody sees, or that is not
        // there, is zeros.
        const int pg = lane - (it & 3) * kTilePages - (j & 1) * (kTilePages / 2);
        const bool mine = pg >= 0 && pg < kTilePages / 2 && pages.now != page_rows.none;
        const uint32_t asked = __ballot_sync(0xffffffffu, mine) >> ((it & 3) * kTilePages + (j & 1) * (kTilePages / 2));
        if (asked != 15u) {
          for (int i = lane; i < S::kRaw / 16; i += 32)
            if (!(asked >> (i / D) & 1)) *reinterpret_cast<uint4*>(slot_at(s) + i * 16) = make_uint4(0, 0, 0, 0);
          __syncwarp();
        }
        if (lane == 0) mbar_expect_tx(&raw_full[s], __popc(asked) * kPage * D);
        __syncwarp();
        if (mine) bulk_load(slot_at(s) + pg * kPage * D, static_cast<const uint8_t*>(p.v_cache) + (size_t)pages.now * D, kPage * D, &raw_full[s]);
        __syncwarp();
        return true;
      };
      bool ok = true;
      if (warp == 8)
        for (int j = 0; ok && j < pieces; ++j) ok = ((j & 1) || ask_k(j >> 1)) && ask(j);
      for (int j = 0; ok && warp != 8 && j < pieces; ++j) {
        const int it = j >> 1, b = it & 1, s = j & (slots - 1);
        ok = ok && mbar_wait_warp(&raw_full[s], (j >> turn) & 1, abort_flag) &&
             (it < 2 || (j & 1) || mbar_wait_warp(&v_empty[b], ((it >> 1) - 1) & 1, abort_flag));
        if (!ok) break;
        const uint8_t* src = slot_at(s) + lane * 16;
        // A turn of the warp covers kTurnRows rows. The two 16-byte pieces that a lane makes of one lie in one half of the row; at D = 128
        // neighbouring lanes of different halves store them in opposite order, so that eight lanes meet 32 banks.
        constexpr int CPR = D / 16, kTurnRows = 32 / CPR, kTurns = kRawTokens / kTurnRows, kMost = (kTurns + kWideners - 1) / kWideners;
        const int rr = lane / CPR, c = 2 * (lane % CPR), flip = D == 128 ? (c >> 3) & 1 : 0;
        uint8_t* dst = sv + b * TB + (j & 1) * (kRawTokens / kPage) * (D / 64) * 2048 + (c >> 3) * 2048;      // V: [page][half][16][64]
        uint4 raw[kMost];
#pragma unroll
        for (int u = 0; u < kMost; ++u)
          if (part + kWideners * u < kTurns) raw[u] = *reinterpret_cast<const uint4*>(src + (part + kWideners * u) * 512);
        const bool look = partial((t0 + it) * kTile);
        uint32_t sum[2] = {0, 0};
#pragma unroll
        for (int u = 0; u < kMost; ++u) {
          if (part + kWideners * u >= kTurns) continue;
          const uint2 h0 = e4m3x4_to_f16(flip ? raw[u].z : raw[u].x), h1 = e4m3x4_to_f16(flip ? raw[u].w : raw[u].y);
          const uint2 h2 = e4m3x4_to_f16(flip ? raw[u].x : raw[u].z), h3 = e4m3x4_to_f16(flip ? raw[u].y : raw[u].w);
          uint4 x = make_uint4(h0.x, h0.y, h1.x, h1.y), z = make_uint4(h2.x, h2.y, h3.x, h3.y);
          if (look) {
            odd_sum<true>(sum[0], x.x); odd_sum<true>(sum[1], x.y); odd_sum<true>(sum[0], x.z); odd_sum<true>(sum[1], x.w);
            odd_sum<true>(sum[0], z.x); odd_sum<true>(sum[1], z.y); odd_sum<true>(sum[0], z.z); odd_sum<true>(sum[1], z.w);
            x.x = without_odd_f16(x.x); x.y = without_odd_f16(x.y); x.z = without_odd_f16(x.z); x.w = without_odd_f16(x.w);
            z.x = without_odd_f16(z.x); z.y = without_odd_f16(z.y); z.z = without_odd_f16(z.z); z.w = without_odd_f16(z.w);
          }
          const int row = (part + kWideners * u) * kTurnRows + rr;
          uint8_t* line = dst + (row >> 4) * (D / 64) * 2048 + (row & 15) * 128;
          *reinterpret_cast<uint4*>(line + ((((c & 7) + flip) ^ (row & 7)) << 4)) = x;
          *reinterpret_cast<uint4*>(line + ((((c & 7) + 1 - flip) ^ (row & 7)) << 4)) = z;
        }
        if (odd_f16x2(sum[0]) || odd_f16x2(sum[1])) atomicOr(odd_met, 1);
        if (j & 1) fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&raw_empty[s]);
          if (j & 1) mbar_arrive(&v_ready[b]);
        }
        __syncwarp();
      }
      bad = pages.bad;
    }
    if (bad && p.status) atomicCAS(p.status, FLLM_OK, FLLM_ERR_BAD_ARGS);
  } else {
    if constexpr (KV4) asm volatile("setmaxnreg.inc.sync.aligned.u32 176;");
    else if constexpr (KV8) asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    else asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    q_loaded();
    __syncwarp();
    if (lane == 0) mbar_arrive(q_full);
    if constexpr (KV8) asm volatile("bar.sync 2, 384;" ::: "memory");
    else asm volatile("bar.sync 1, 256;" ::: "memory");
    float factor = factors[r], scale = p.softcap > 0.f ? p.softcap * kLog2e : factor;
    const float row_factor = factor;
    int up_v = 0;                                      // O is in units of 2^-up_v
    const uint32_t t_s = tmem_base + 128 * group + lane_off, t_o = tmem_base + 256 + 128 * group + lane_off;
    // tokens [w_beg, w_base) are seen by all rows of this warp
    int w_base = min_base, w_beg = max_beg;
    if (!p.tree_mask) {
      const int ctx = kv_len - qn + 1;
      w_base = max(ctx + (row0 + r_first) / G, 0);
      w_beg = p.window > 0 ? max(ctx + (row0 + min(r_first + 31, n_rows - 1)) / G - p.window, 0) : 0;
    }
    float m_used = -INFINITY, l = 0.f;
    bool ok = true;
    for (int n = group; n < n_items; n += 2) {
      const int k = n >> 1, tok0 = (t0 + (n >> shift)) * kTile;
      if (!mbar_wait(&s_full[group], k & 1, abort_flag)) { ok = false; break; }
      tc_fence_after_sync();
      float shrink = 1.f;
      const int t = n >> shift;
      int4 unit = make_int4(0, 0, 0, 0);
      if constexpr (KV4) {
        if (!mbar_wait(&v_unit[t & 1], (t >> 1) & 1, abort_flag)) { ok = false; break; }
        unit = lds_int4(units + 4 * (t & 3));
        const int up = unit.x, now = unit.y;
        // Not 0, nor infinite, as factors of rows are not (span_factor): a score of 0 in an unseen place beside one, or a 0 beside the other, would be a NaN.
        factor = fminf(fmaxf(row_factor * pow2_of(-(up >> 1)) * pow2_of((up >> 1) - up), FLT_MIN), FLT_MAX);
        if (p.softcap <= 0.f) scale = factor;
        if (k > 0 && now != up_v) shrink = pow2_of(max(now - up_v, -126));
        up_v = now;
      }
      const bool whole = tok0 + kTile <= w_base && (tok0 >= w_beg || tok0 + kTile <= p.first);
      uint4 vis = make_uint4(0, 0, 0, 0);
      if (!whole) vis = row_bits(p, q0, qn, kv_len, gap, qi, tok0);
      if constexpr (KV4) {
        if (unit.z || p.softcap > 0.f)
          change_scores(t_s, unit.z ? k_lifts + (t & 3) * kTile : nullptr, p.softcap > 0.f ? fminf(factor / (p.softcap * kLog2e), FLT_MAX) : 0.f);
      } else {
        if (p.softcap > 0.f) cap_scores(t_s, factor / (p.softcap * kLog2e));
      }
      softmax_tile<D, KV != kBf16>(t_s, t_o, whole, vis, scale, k > 0, unit.w ? nobody : &p_half[group], m_used, l, shrink);
      if constexpr (KV4) {
        if (unit.w) lower_weights<D>(t_s, smem, t, group);
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_ready[group]);
    }
    if (KV != kBf16) m_used -= kTcLift;
    const bool splits = pieces > 1;
    const int G_row = qi >= 0 ? kvh * G + (row0 + r) - qi * G : 0;
    const float sink = p.sinks && qi >= 0 ? p.sinks[G_row] * kLog2e : -INFINITY;
    uint8_t* dst = splits ? reinterpret_cast<uint8_t*>(p.ws_o + (((size_t)(q0 + max(qi, 0)) * p.hq + G_row) * p.splits + split) * D)
                          : reinterpret_cast<uint8_t*>(static_cast<bf16*>(p.out) + (size_t)(q0 + max(qi, 0)) * p.ldo + (size_t)G_row * D);
    ok = ok && n_items > 0 && mbar_wait(o_done, 0, abort_flag);       // (a group without items too: what follows reuses K and V)
    const bool have = ok && n_items > group;
    tc_fence_after_sync();
    float c_mine = 1.f, c_other = 0.f;
    bool other = false;
    const int at = (warp & 3) * 32 + lane;
    float* swap = reinterpret_cast<float*>(sk);        // O of the second group, [column][row]; then its maxima and sums
    if (!two) {
      float2* swap_ml = reinterpret_cast<float2*>(sv);
      if (group == 1) {
        if (have) {
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            tmem_ld_32x32(t_o + 32 * c, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              float v = __uint_as_float(o[i]);
              if constexpr (KV4) v = v * pow2_of(-(up_v >> 1)) * pow2_of((up_v >> 1) - up_v);
              swap[(32 * c + i) * kRows + at] = v;
            }
          }
        }
        swap_ml[at] = make_float2(have ? m_used : -INFINITY, have ? l : 0.f);
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (group == 0) {
        other = n_items > 1;
        const float2 ml = swap_ml[at];
        const float mm = fmaxf(m_used, ml.x);
        if (other) {
          c_mine = m_used == -INFINITY ? (mm == -INFINITY ? 1.f : 0.f) : ex2(m_used - mm);
          c_other = ml.x == -INFINITY ? (mm == -INFINITY ? 1.f : 0.f) : ex2(ml.x - mm);
          l = l * c_mine + ml.y * c_other;
          m_used = mm;
        }
      }
    }
    if (two || group == 0) {
      // (m, l, O) of the rows: to the workspace, or normalised with the head's sink to the output. A lane puts its row, kPass bytes of it at a time, into
      // shared memory of the warp's own (Q and K have been read) and asks for it to be copied.
      if (!splits) {
        float ll = l, less = 1.f;
        if (p.sinks && qi >= 0 && (m_used != -INFINITY || l != 0.f)) {       // (a row that saw nothing stays 0, whatever the sink)
          const float mn = fmaxf(m_used, sink);
          less = m_used == -INFINITY ? 0.f : ex2(m_used - mn);
          ll = ll * less + ex2(sink - mn);
        }
        const float norm = ll == 0.f || !have ? 0.f : less / ll;
        c_mine *= norm;
        c_other *= norm;
      }
      if (p.splits > 1 && qi >= 0) {                   // what span_merge_kernel reads: the row's maxima and sums, or that it is done
        float2* ml = reinterpret_cast<float2*>(p.ws_ml) + ((size_t)(q0 + qi) * p.hq + G_row) * p.splits;
        ml[split] = !splits ? make_float2(0.f, -1.f) : have ? make_float2(m_used, l) : make_float2(-INFINITY, 0.f);
        if (splits && split == 0)
          for (int i = pieces; i < p.splits; ++i) ml[i] = make_float2(-INFINITY, 0.f);
      }
      constexpr int kPass = D == 128 ? 256 : 128, kPitch = kPass + 16;
      static_assert(4 * 32 * kPitch <= 2 * TB && 8 * 32 * kPitch <= 4 * TB, "room of the rows");
      uint8_t* stage = sq + (size_t)(warp * 32 + lane) * kPitch;
      const int cols = splits ? kPass / 4 : kPass / 2;
#pragma unroll 1
      for (int c0 = 0; c0 < D; c0 += cols) {
        if (c0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
#pragma unroll 1
        for (int h = 0; h < cols; h += 32) {
          uint32_t o[32];
          if (have) {
            tmem_ld_32x32(t_o + c0 + h, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              float v = __uint_as_float(o[i]) * c_mine;
              if constexpr (KV4) v = v * pow2_of(-(up_v >> 1)) * pow2_of((up_v >> 1) - up_v);
              o[i] = __float_as_uint(v);
            }
            if (other) {
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) + swap[(c0 + h + i) * kRows + at] * c_other);
            }
            if constexpr (KV4) {                       // of eight columns the dims (kv4_widen_f16)
#pragma unroll
              for (int i = 0; i < 32; i += 8) {
                const uint32_t d[8] = {o[i], o[i + 2], o[i + 4], o[i + 6], o[i + 1], o[i + 3], o[i + 5], o[i + 7]};
#pragma unroll
                for (int e = 0; e < 8; ++e) o[i + e] = d[e];
              }
            }
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0;
          }
          if (splits) {
#pragma unroll
            for (int i = 0; i < 32; i += 4) *reinterpret_cast<uint4*>(stage + (h + i) * 4) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          } else {
#pragma unroll
            for (int i = 0; i < 32; i += 8)
              *reinterpret_cast<uint4*>(stage + (h + i) * 2) =
                  make_uint4(pack_bf16x2(__uint_as_float(o[i]), __uint_as_float(o[i + 1])), pack_bf16x2(__uint_as_float(o[i + 2]), __uint_as_float(o[i + 3])),
                             pack_bf16x2(__uint_as_float(o[i + 4]), __uint_as_float(o[i + 5])), pack_bf16x2(__uint_as_float(o[i + 6]), __uint_as_float(o[i + 7])));
          }
        }
        fence_proxy_async_smem();
        if (qi >= 0)
          asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst + (size_t)c0 * (splits ? 4 : 2)), "r"(smem_u32(stage)), "r"(kPass) : "memory");
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      }
      if (*odd_met && qi >= 0) {
        asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        // infinities and NaN that were taken out of tiles, added to the rows that see them
        for (int it = 0; it < n_tiles; ++it) {
          const int tok0 = (t0 + it) * kTile;
          if (!partial(tok0)) continue;
          const uint4 visible = row_bits(p, q0, qn, kv_len, gap, qi, tok0);
          const uint32_t vis[4] = {visible.x, visible.y, visible.z, visible.w};
          for (int i = 0; i < kTile; ++i) {
            if (!(vis[i >> 5] >> (i & 31) & 1)) continue;
            const int page = page_rows.page_of((tok0 + i) / kPage), b = span_block(p, page_rows.table, page);
            if (b < 0) continue;
            const size_t at = (size_t)(span_pool_row(p, b, kvh, page) + (i & 15)) * (KV4 ? kKv4Row<D> : D);
            if constexpr (KV4) {                       // a row is NaN as a whole, or a number
              if ((static_cast<const uint16_t*>(p.v_cache)[(at + D / 2) / 2] & 0x7F80u) != 0x7F80u) continue;
            }
            for (int d = 0; d < D; ++d) {
              float x;
              if constexpr (KV4) {
                x = __int_as_float(0x7FC00000);
              } else if constexpr (KV8) {
                x = (static_cast<const uint8_t*>(p.v_cache)[at + d] & 0x7F) == 0x7F ? __int_as_float(0x7FC00000) : 0.f;
              } else {
                x = __bfloat162float(static_cast<const bf16*>(p.v_cache)[at + d]);
              }
              if (isfinite(x)) continue;
              if (splits) reinterpret_cast<float*>(dst)[d] += x;
              else reinterpret_cast<bf16*>(dst)[d] = __float2bfloat16(__bfloat162float(reinterpret_cast<bf16*>(dst)[d]) + x);
            }
          }
        }
      }
    }
  }
  asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 9) { tc_fence_after_sync(); tmem_dealloc(tmem_base, 512); }
  if (threadIdx.x == 0 && *abort_flag && p.status) atomicCAS(p.status, FLLM_OK, FLLM_ERR_MBAR_TIMEOUT);
}

template <int D, int KV>
void launch_tc(SpanParams p, cudaStream_t s) {
  static bool configured[kMaxDevices] = {};
  constexpr int smem = TcSmem<D, KV>::kTotal;
  static_assert(smem <= 227 * 1024, "shared memory");
  if (first_call_on_device(configured)) {
    cuda_check(cudaFuncSetAttribute(span_tc_kernel<D, KV, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), "span_tc smem");
    cuda_check(cudaFuncSetAttribute(span_tc_kernel<D, KV, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), "span_tc smem");
  }
  const uint64_t rows = (uint64_t)p.num_blocks * p.hkv * p.block_pages * kPage;
  // encoded for every call: they cost less than looking up by an address what another tensor may since have
  CUtensorMap mk{}, mv{};
  if (KV == kE4m3) {
    mk = make_tmap_bytes(p.k_cache, rows, D, kPage);
  } else if (KV == kBf16) {
    mk = make_tmap_2d(p.k_cache, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, rows, D, D * 2, kPage, 64, true);
    mv = make_tmap_parts(p.v_cache, rows, D, kPage, D / 64);
  }
  // (What is left of the longest sequence's rows is a whole tile from 129 rows on.)
  const long long most = (long long)p.max_q_len * p.group, row_tiles = (most + kRows - 1) / kTcRows, whole = row_tiles * p.num_seqs * p.hkv;
  // Where the last round of whole tiles, and what is left of rows behind it, would leave half of the SMs or more without work, two SMs share each of its
  // tiles by rows. (2 x 2048 rows under a window of 1024, 32 query and 8 key heads of 128, three rounds and 68 tiles: 99 us, 105 without.)
  const long long left = most > row_tiles * kTcRows ? (long long)p.num_seqs * p.hkv : 0;
  const long long tiles = span_tiles(p, most, kTcRows, p.search);
  const int last = (int)(whole % p.sms), halved = p.splits == 1 && !p.search && 2 * last + left <= p.sms ? last : 0;
  const long long ctas = tiles * p.hkv + halved;
  if (ctas > INT_MAX) throw std::runtime_error("attention_span: too many query rows");
  auto go = [&](auto kernel) { launch_pdl(kernel, dim3((unsigned)ctas, p.splits), dim3(tc_threads<KV>()), smem, s, mk, mv, p, (int)row_tiles, halved); };
  if (p.search) go(span_tc_kernel<D, KV, true>);
  else go(span_tc_kernel<D, KV, false>);
}
}  // namespace

bool attention_span_tc_supported(const SpanParams& p) {
  return (p.head_dim == 64 || p.head_dim == 128) && p.num_blocks * p.hkv * p.block_pages * kPage <= INT_MAX - kTile;
}
void attention_span_tc(const SpanParams& p, cudaStream_t s) {
  if (p.kv4) p.head_dim == 64 ? launch_tc<64, kKv4>(p, s) : launch_tc<128, kKv4>(p, s);
  else if (p.head_dim == 64) p.kv_fp8 ? launch_tc<64, kE4m3>(p, s) : launch_tc<64, kBf16>(p, s);
  else p.kv_fp8 ? launch_tc<128, kE4m3>(p, s) : launch_tc<128, kBf16>(p, s);
}
}  // namespace fllm
