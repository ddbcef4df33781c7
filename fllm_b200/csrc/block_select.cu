// Which blocks of the cache a query row reads: bounds of the keys of every full block, scores of the blocks from them, and the best of a row's.
//
// Bounds of a block and key head are two int8 codes a channel and an exponent: hi[d] = ceil(max_t k[t, d] / 2^e), lo[d] = floor(min_t k[t, d] / 2^e), e the
// smallest with |k| <= 127 x 2^e (at least -120). For the heads h of a key head's group
//
//   sum_h q_h . k <= sum_d (u[d] max k[d] - w[d] min k[d]),   u = sum_h max(q_h, 0),  w = sum_h max(-q_h, 0)
//
// so with u and w in 7 bits (a common power of two for each row and key head, nearest, ties to even) a block's score is 2^e (u . hi - w . lo): a product of
// whole numbers below 2^23, exact in 32 bits in any order, times a power of two. Equal inputs have equal scores, whatever they are computed beside, and
// ties go to the lower block.
//
// A row whose text has more than `count` blocks reads the first `lead`, the last `tail` (its own among them, which may not be full) and the best of those
// between; one of fewer blocks reads all. A block with a value that is not finite (or 2^107 and above) scores infinity: it is read, so that it shows.
// Values of a query that are not finite count as 0.
//
// The scores of a step go through memory; scores are products of 16 blocks and 8 rows on mma.sync of int8 (a block's codes are read once for a tile of rows, in
// pieces of 16 bytes), the choice is a search for the last key that is taken, digit by digit.
//
// What bounds them (us from captured graphs, scores and choice together): reading the codes, where there are many (64 decode rows of 4000 to 32,000 tokens, 8 key heads
// of 128, 139 MB: 61, some 45 of them for the scores, 3.1 TB/s: a warp waits for table and codes with 16 blocks on their way); trips to memory one behind the other and
// the barriers of a choice where there are few (one row of 30,000 tokens: 18); the choices of prompts, one CTA for each row and head (602 rows of 3000 to 6300
// tokens: 64, some 40 for them). Bounds: 1 to 4.
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <limits.h>

#include <algorithm>
#include <stdexcept>
#include <type_traits>

#include "attention_span.cuh"
#include "kv4.cuh"
#include "tma_host.h"

namespace fllm {
namespace {
using bf16 = __nv_bfloat16;
constexpr int kTail = 16;                   // bytes of a block's bounds behind the codes: the exponent, and zeros
constexpr int kNotFinite = 127;             // exponent of a block with a value that is not finite
constexpr int kLeastExp = -120, kMostExp = 100;

__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
// The smallest e with top <= 127 x 2^e, top > 0 (kLeastExp at least).
__device__ __forceinline__ int unit_of(float top) {
  const int e = max((int)(__float_as_uint(top) >> 23) - 127 - 6, kLeastExp);
  return top > 127.f * pow2(min(e, 120)) ? e + 1 : e;
}

// ---------------------------------------------------------------------------- bounds
// CH neighbouring channels of a row of the cache, the lane-th such piece.
template <int D, int KIND>
__device__ __forceinline__ void load_channels(const uint8_t* row, int lane, float (&v)[D / 32]) {
  constexpr int CH = D / 32;
  if constexpr (KIND == 0) {
    const uint32_t* src = reinterpret_cast<const uint32_t*>(row) + lane * (CH / 2);
#pragma unroll
    for (int i = 0; i < CH / 2; ++i) {
      const float2 f = unpack_bf16x2(src[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  } else if constexpr (KIND == 1) {
    const uint16_t* src = reinterpret_cast<const uint16_t*>(row) + lane * (CH / 2);
#pragma unroll
    for (int i = 0; i < CH / 2; ++i) {
      const float2 f = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(src[i], __NV_E4M3)));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  } else {
    const Kv4Scale s = kv4_scale_of(*reinterpret_cast<const uint32_t*>(row + D / 2));
    using Codes = std::conditional_t<CH == 2, uint8_t, std::conditional_t<CH == 4, uint16_t, uint32_t>>;
    const uint32_t codes = reinterpret_cast<const Codes*>(row)[lane];
#pragma unroll
    for (int i = 0; i < CH; ++i) v[i] = kv4_value(codes >> 4 * i & 15, s);
  }
}

// A warp per (row of the step, key head): where the row's slot is the last of its block, the block is full, and its bounds are found.
template <int D, int KIND>
__global__ void __launch_bounds__(128) kv_bounds_kernel(const __grid_constant__ BoundsParams p) {
  constexpr int CH = D / 32, RB = KIND == 0 ? 2 * D : KIND == 1 ? D : kKv4Row<D>;
  pdl_launch_dependents();
  pdl_wait();
  const int item = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int row = item / p.hkv, head = item - row * p.hkv;
  if (row >= p.rows) return;
  const int slot = p.slots[row];
  if (slot < 0 || slot % p.block_size != p.block_size - 1) return;
  const int block = slot / p.block_size;
  if (block >= p.num_blocks) {
    if (lane == 0 && p.status) atomicCAS(p.status, FLLM_OK, FLLM_ERR_BAD_ARGS);
    return;
  }
  const uint8_t* src = static_cast<const uint8_t*>(p.k_cache) + ((size_t)block * p.hkv + head) * p.block_size * RB;
  float hi[CH], lo[CH], odd = 0.f;
#pragma unroll
  for (int i = 0; i < CH; ++i) { hi[i] = -INFINITY; lo[i] = INFINITY; }
#pragma unroll 16
  for (int r = 0; r < p.block_size; ++r) {
    float v[CH];
    load_channels<D, KIND>(src + (size_t)r * RB, lane, v);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      hi[i] = fmaxf(hi[i], v[i]);
      lo[i] = fminf(lo[i], v[i]);
      odd = fmaf(v[i], 0.f, odd);
    }
  }
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < CH; ++i) top = fmaxf(top, fmaxf(fabsf(hi[i]), fabsf(lo[i])));
  top = warp_max(top);
  int e = top > 0.f ? unit_of(top) : kLeastExp;
  const bool bad = __any_sync(0xffffffffu, odd != 0.f) || e > kMostExp;
  if (bad) e = kNotFinite;
  const float f = bad ? 0.f : pow2(-e);
  int8_t* dst = p.bounds + ((size_t)block * p.hkv + head) * (2 * D + kTail);
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    dst[lane * CH + i] = bad ? 0 : (int8_t)__float2int_ru(hi[i] * f);
    dst[D + lane * CH + i] = bad ? 0 : (int8_t)__float2int_rd(lo[i] * f);
  }
  if (lane < kTail) dst[2 * D + lane] = lane == 0 ? (int8_t)e : 0;
}

// ---------------------------------------------------------------------------- scores
__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

constexpr int kScoreBlocks = 16;            // of a warp's step

// One CTA per (tile of 8 x NQ rows of a sequence, key head, piece of the text).
template <int D, int NQ, bool SEARCH>
__global__ void __launch_bounds__(128) block_score_kernel(const __grid_constant__ SelectParams p) {
  constexpr int kTileRows = 8 * NQ, kPitch = 2 * D + 16;      // of a row's codes: a piece of 16 bytes more, so that eight rows meet other banks
  __shared__ __align__(16) uint8_t codes[kTileRows * kPitch];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const SpanParams& s = p.rows;
  int work = blockIdx.x / p.pieces;
  const int piece = blockIdx.x - work * p.pieces;
  const int kvh = work % s.hkv;
  work /= s.hkv;
  pdl_launch_dependents();
  pdl_wait();
  int seq = work % s.num_seqs, tile = work / s.num_seqs, q0, qn, kv_len;
  if constexpr (SEARCH) {
    if (!span_find(s, kTileRows, 0, INT_MAX, work, blockIdx.x == gridDim.x - 1, seq, tile)) return;
  }
  if (!span_lengths(s, seq, threadIdx.x == 0, q0, qn, kv_len)) return;
  const int row0 = tile * kTileRows;
  if (row0 >= qn) return;
  const int n_rows = min(kTileRows, qn - row0);
  if (q0 + row0 >= p.row_to || q0 + row0 + n_rows <= p.row_from) return;
  // blocks that the tile's last row chooses among
  const int last = max(kv_len - qn + row0 + n_rows, 0);       // its tokens
  const int most = (last + p.block_size - 1) / p.block_size;
  if (most <= p.count) return;
  const int end = most - p.tail;
  const int steps = (end - p.lead + 4 * kScoreBlocks - 1) / (4 * kScoreBlocks), each = (steps + p.pieces - 1) / p.pieces;
  const int first = p.lead + piece * each * 4 * kScoreBlocks, stop = min(end, first + each * 4 * kScoreBlocks);
  if (first >= stop) return;

  const int* table = s.block_tables + (size_t)seq * s.max_blocks;
  constexpr int J = 2 * D / 64;             // pieces of 16 bytes of a lane
  // The block of lane & 15 of a step is looked up two steps ahead of its use.
  bool missing = false;
  auto look = [&](int b0) {
    const int at = b0 + (lane & 15);
    const int id = at < stop && at < s.max_blocks ? table[at] : 0;
    const bool there = (unsigned)id < (unsigned)s.num_blocks;
    missing |= !there;
    return there ? id : -1;
  };
  constexpr int kStep = 4 * kScoreBlocks;
  const int mine0 = first + warp * kScoreBlocks;
  int id = mine0 < stop ? look(mine0) : 0, id1 = mine0 + kStep < stop ? look(mine0 + kStep) : 0;
  // u and -w of the rows: a warp to a row (what the products have of rows that are not there goes nowhere)
  for (int r = warp; r < n_rows; r += 4) {
    constexpr int CH = D / 32;
    float u[CH], w[CH];
#pragma unroll
    for (int i = 0; i < CH; ++i) u[i] = w[i] = 0.f;
    const uint32_t* src = reinterpret_cast<const uint32_t*>(static_cast<const bf16*>(s.q) + (size_t)(q0 + row0 + r) * s.ldq + (size_t)kvh * p.group * D) + lane * (CH / 2);
    for (int h0 = 0; h0 < p.group; h0 += 4) {           // heads in their order, four on their way at once
      uint32_t q4[4][CH / 2];
#pragma unroll
      for (int h = 0; h < 4; ++h)
#pragma unroll
        for (int i = 0; i < CH / 2; ++i) q4[h][i] = h0 + h < p.group ? src[(h0 + h) * (D / 2) + i] : 0u;
#pragma unroll
      for (int h = 0; h < 4; ++h)
#pragma unroll
        for (int i = 0; i < CH / 2; ++i) {
          const float2 f = unpack_bf16x2(q4[h][i]);
          const float x[2] = {isfinite(f.x) ? f.x : 0.f, isfinite(f.y) ? f.y : 0.f};
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            u[2 * i + k] = fminf(u[2 * i + k] + fmaxf(x[k], 0.f), FLT_MAX);
            w[2 * i + k] = fminf(w[2 * i + k] + fmaxf(-x[k], 0.f), FLT_MAX);
          }
        }
    }
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < CH; ++i) top = fmaxf(top, fmaxf(u[i], w[i]));
    top = warp_max(top);
    const int e = top > 0.f ? unit_of(top) : 0;
    const float f = pow2(-min(e, 126)) ;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      codes[r * kPitch + lane * CH + i] = (uint8_t)__float2int_rn(u[i] * f);
      codes[r * kPitch + D + lane * CH + i] = (uint8_t)-__float2int_rn(w[i] * f);
    }
  }
  __syncthreads();

  for (int b0 = mine0; b0 < stop; b0 += kStep) {
    const int id2 = b0 + 2 * kStep < stop ? look(b0 + 2 * kStep) : 0;
    const int e_at = id >= 0 ? (int)p.bounds[((size_t)id * s.hkv + kvh) * (2 * D + kTail) + 2 * D] : -128;
    uint4 a[2][J];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int other = __shfl_sync(0xffffffffu, max(id, 0), g + 8 * h);
      const int8_t* of = p.bounds + ((size_t)other * s.hkv + kvh) * (2 * D + kTail) + 16 * t;
#pragma unroll
      for (int j = 0; j < J; ++j) a[h][j] = *reinterpret_cast<const uint4*>(of + 64 * j);
    }
    id = id1;
    id1 = id2;
    const int e0 = __shfl_sync(0xffffffffu, e_at, g), e1 = __shfl_sync(0xffffffffu, e_at, g + 8);
#pragma unroll 1
    for (int n = 0; n < NQ; ++n) {
      if (8 * n >= n_rows) break;
      int c[4] = {0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const uint4 b = *reinterpret_cast<const uint4*>(codes + (8 * n + g) * kPitch + 64 * j + 16 * t);
        mma_s8(c, a[0][j].x, a[1][j].x, a[0][j].y, a[1][j].y, b.x, b.y);
        mma_s8(c, a[0][j].z, a[1][j].z, a[0][j].w, a[1][j].w, b.z, b.w);
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int r = 8 * n + 2 * t + (x & 1), b = b0 + g + 8 * (x >> 1), e = x >> 1 ? e1 : e0;
        const float score = e == kNotFinite ? INFINITY : e == -128 ? -INFINITY : (float)c[x] * pow2(e);
        const int at = q0 + row0 + r;
        if (r < n_rows && b < stop && at >= p.row_from && at < p.row_to) p.scores[((size_t)(at - p.row_from) * s.hkv + kvh) * p.stride + b] = score;
      }
    }
  }
  if (missing && s.status) atomicCAS(s.status, FLLM_OK, FLLM_ERR_BAD_ARGS);
}

// ---------------------------------------------------------------------------- the best
constexpr int kSelectThreads = 256, kBins = 2048;

__device__ __forceinline__ uint32_t key_of(float f) {
  const uint32_t b = __float_as_uint(f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
// Exclusive sum over the threads. `sums` is free again behind the next barrier.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* sums) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t upto = v;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const uint32_t x = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += x;
  }
  if (lane == 31) sums[warp] = upto;
  __syncthreads();
  uint32_t before = 0;
#pragma unroll
  for (int w = 0; w < kSelectThreads / 32; ++w)
    if (w < warp) before += sums[w];
  return before + upto - v;
}

// One CTA per (row, key head): the key of the last block that is taken digit by digit, from the largest, then what is above it, and of what equals it as many
// as are left, from the lowest block on.
__global__ void __launch_bounds__(kSelectThreads) block_choose_kernel(const __grid_constant__ SelectParams p) {
  extern __shared__ uint32_t keys_s[];
  __shared__ uint32_t hist[kBins];
  __shared__ unsigned long long sums[kSelectThreads / 32];
  __shared__ uint32_t parts[kSelectThreads / 32];
  __shared__ uint32_t found[2];
  const SpanParams& s = p.rows;
  const int local = blockIdx.x / s.hkv, kvh = blockIdx.x - local * s.hkv, row = p.row_from + local, tid = threadIdx.x;
  pdl_launch_dependents();
  pdl_wait();
  int* out = p.out + ((size_t)row * s.hkv + kvh) * p.count;
  int seq, q0, qn, kv_len, tokens = 0;
  if (span_seq_of(s, row, seq) && span_lengths(s, seq, false, q0, qn, kv_len) && row - q0 < qn) tokens = max(kv_len - qn + row - q0 + 1, 0);
  const int most = (tokens + p.block_size - 1) / p.block_size;
  if (most <= p.count) {                    // all of them
    for (int i = tid; i < p.count; i += kSelectThreads) out[i] = i < most ? i : -1;
    return;
  }
  for (int i = tid; i < p.lead; i += kSelectThreads) out[i] = i;
  for (int i = tid; i < p.tail; i += kSelectThreads) out[p.count - p.tail + i] = most - p.tail + i;
  int want = p.count - p.lead - p.tail;
  if (want == 0) return;
  const int n = most - p.lead - p.tail;
  const float* scores = p.scores + ((size_t)local * s.hkv + kvh) * p.stride + p.lead;
  uint32_t least = 0xFFFFFFFFu, most_key = 0;
#pragma unroll 8
  for (int i = tid; i < n; i += kSelectThreads) {
    const uint32_t k = key_of(scores[i]);
    keys_s[i] = k;
    least = min(least, k);
    most_key = max(most_key, k);
  }
  least = __reduce_min_sync(0xffffffffu, least);
  most_key = __reduce_max_sync(0xffffffffu, most_key);
  if ((tid & 31) == 0) sums[tid >> 5] = (unsigned long long)most_key << 32 | least;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSelectThreads / 32; ++w) {
    least = min(least, (uint32_t)sums[w]);
    most_key = max(most_key, (uint32_t)(sums[w] >> 32));
  }
  // Digits are of what a key is above the least, from its 11 highest bits down, so that scores of one magnitude do not all meet in one counter.
  uint32_t prefix = 0, mask = 0;
  int upper = 32 - __clz(most_key - least);            // bits that are still open
#pragma unroll 1
  while (true) {
    const int bits = 11, shift = max(upper - bits, 0);
    for (int i = tid; i < kBins; i += kSelectThreads) hist[i] = 0;
    __syncthreads();
#pragma unroll 8
    for (int i = tid; i < n; i += kSelectThreads) {
      const uint32_t k = keys_s[i] - least;
      if ((k & mask) == prefix) atomicAdd(&hist[(k & ~mask) >> shift], 1u);
    }
    __syncthreads();
    // from the largest digit down: a thread has kBins / 256 of them
    constexpr int kEach = kBins / kSelectThreads;
    const int from = kBins - 1 - tid * kEach;
    uint32_t mine[kEach];
    uint32_t sum = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      mine[i] = hist[from - i];
      sum += mine[i];
    }
    uint32_t above = block_scan(sum, parts);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if (above < (uint32_t)want && (uint32_t)want <= above + mine[i]) { found[0] = (uint32_t)(from - i); found[1] = above; }
      above += mine[i];
    }
    __syncthreads();
    prefix |= found[0] << shift;
    mask = 0xFFFFFFFFu << shift;
    want -= (int)found[1];                  // of those with this digit
    upper = shift;
    if (!shift) break;
    __syncthreads();
  }
  prefix += least;
  // A warp has neighbouring blocks, 32 at a time: the place of one among the others' is a sum over the warps in front of it, and a count of lanes.
  const int warp = tid >> 5, lane = tid & 31, each = ((n + kSelectThreads - 1) / kSelectThreads) * 32;
  const int from = min(warp * each, n), to = min(from + each, n);
  int over = 0, equal = 0;
#pragma unroll 4
  for (int i0 = from; i0 < to; i0 += 32) {
    const uint32_t k = i0 + lane < to ? keys_s[i0 + lane] : 0;
    over += __popc(__ballot_sync(0xffffffffu, i0 + lane < to && k > prefix));
    equal += __popc(__ballot_sync(0xffffffffu, i0 + lane < to && k == prefix));
  }
  if (lane == 0) sums[warp] = (unsigned long long)over << 32 | (uint32_t)equal;
  __syncthreads();
  over = equal = 0;
#pragma unroll
  for (int w = 0; w < kSelectThreads / 32; ++w)
    if (w < warp) {
      over += (int)(sums[w] >> 32);
      equal += (int)(uint32_t)sums[w];
    }
  const unsigned below = (1u << lane) - 1;
#pragma unroll 4
  for (int i0 = from; i0 < to; i0 += 32) {
    const uint32_t k = i0 + lane < to ? keys_s[i0 + lane] : 0;
    const bool is_over = i0 + lane < to && k > prefix, is_equal = i0 + lane < to && k == prefix;
    const unsigned o = __ballot_sync(0xffffffffu, is_over), e = __ballot_sync(0xffffffffu, is_equal);
    const int my_over = over + __popc(o & below), my_equal = equal + __popc(e & below);
    if (is_over || (is_equal && my_equal < want)) out[p.lead + my_over + min(my_equal, want)] = p.lead + i0 + lane;
    over += __popc(o);
    equal += __popc(e);
  }
}

template <int D>
void launch_bounds(const BoundsParams& p, int kind, cudaStream_t s) {
  const long long ctas = ((long long)p.rows * p.hkv + 3) / 4;
  if (ctas > INT_MAX / 4) throw std::runtime_error("kv_bounds: too many rows");
  auto go = [&](auto kernel) { launch_pdl(kernel, dim3((unsigned)ctas), dim3(128), 0, s, p); };
  if (kind == 0) go(kv_bounds_kernel<D, 0>);
  else if (kind == 1) go(kv_bounds_kernel<D, 1>);
  else go(kv_bounds_kernel<D, kKv4>);
}

template <int D, int NQ>
void launch_scores(SelectParams p, cudaStream_t s) {
  const long long tiles = span_tiles(p.rows, p.rows.max_q_len, 8 * NQ, p.rows.search) * p.rows.hkv;
  // Pieces of the text for two rounds of CTAs, so that long texts do not hold their SMs alone in the end (64 decode rows of 4000 to 32,000 tokens, 8 key heads of
  // 128, the scores' kernel in one run: 48 us with half as many, 34 so, 37 with twice, 42 with four times as many), a step of each warp at least.
  const long long steps = (std::max(p.stride - p.lead - p.tail, 1) + 4 * kScoreBlocks - 1) / (4 * kScoreBlocks);
  p.pieces = (int)std::max<long long>(1, std::min<long long>(16LL * sm_count() / tiles, steps));
  if (tiles * p.pieces > INT_MAX) throw std::runtime_error("select_blocks: too many query rows");
  if (p.rows.search) launch_pdl(block_score_kernel<D, NQ, true>, dim3((unsigned)(tiles * p.pieces)), dim3(128), 0, s, p);
  else launch_pdl(block_score_kernel<D, NQ, false>, dim3((unsigned)(tiles * p.pieces)), dim3(128), 0, s, p);
}
}  // namespace

void kv_bounds(const BoundsParams& p, int kind, cudaStream_t s) {
  if (p.rows <= 0) return;
  switch (p.head_dim) {
    case 64: launch_bounds<64>(p, kind, s); break;
    case 128: launch_bounds<128>(p, kind, s); break;
    default: launch_bounds<256>(p, kind, s); break;
  }
  cuda_check(cudaGetLastError(), "kv_bounds launch");
}

int select_blocks(SelectParams p, cudaStream_t s) {
  int n = 0;
  static bool configured[kMaxDevices] = {};
  if (first_call_on_device(configured))
    cuda_check(cudaFuncSetAttribute(block_choose_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSelectBlocks * 4), "block_choose smem");
  if (p.stride > p.count) {                 // some row may have to choose
    const bool few = p.rows.max_q_len <= 8;
    switch (p.rows.head_dim) {
      case 64: few ? launch_scores<64, 1>(p, s) : launch_scores<64, 8>(p, s); break;
      case 128: few ? launch_scores<128, 1>(p, s) : launch_scores<128, 8>(p, s); break;
      default: few ? launch_scores<256, 1>(p, s) : launch_scores<256, 4>(p, s); break;
    }
    ++n;
  }
  launch_pdl(block_choose_kernel, dim3((unsigned)((long long)(p.row_to - p.row_from) * p.rows.hkv)), dim3(kSelectThreads), (size_t)(p.stride > p.count ? p.stride * 4 : 0), s, p);
  cuda_check(cudaGetLastError(), "select_blocks launch");
  return n + 1;
}
}  // namespace fllm
