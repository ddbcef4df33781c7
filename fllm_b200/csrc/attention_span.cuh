// What a query row sees of a paged cache when a sliding window leaves the first tokens visible, and when rows are the nodes of a draft
// tree; shared by the kernels of attention_span.cu and attention_span_tc.cu.
//
// Row r of a sequence stands at place P in its text and sees token j of the context (j < base) if j > P - window or j < first, and node n
// of the tree (stored at base + n) if its bit is set in the row's mask (its ancestors and itself) and the same holds for the node's
// place. Plain rows have base = P + 1 and no mask; tree rows P = base + (bits set) - 1, and the k-th bit set stands at base + k. So a
// mask is trimmed once and every token is then two comparisons or one bit.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

#include "fllm_ops.h"
#include "ptx.cuh"

namespace fllm {
namespace {
constexpr int kSpanWords = 4;              // 64-bit words of a tree mask: at most 256 nodes

struct SpanRow {
  int base;                                // context tokens are those in front of it
  int beg;                                 // where the window begins, its end at most
};

// Row `qi` of the qn rows of a sequence; `bits` (trees): its mask, trimmed, p.words of them.
__device__ __forceinline__ SpanRow span_row(const SpanParams& p, int q0, int qn, int kv_len, int qi, unsigned long long* bits) {
  SpanRow r;
  int count = 0;
  if (p.tree_mask) {
    r.base = min(max(p.tree_base[q0 + qi], 0), kv_len);
    const int nodes = kv_len - r.base;
    for (int w = 0; w < p.words; ++w) {
      unsigned long long m = p.tree_mask[(size_t)(q0 + qi) * p.words + w];
      const int left = nodes - 64 * w;     // nodes that are stored
      if (left < 64) m = left <= 0 ? 0ull : m & ((1ull << left) - 1);
      bits[w] = m;
      count += __popcll(m);
    }
  } else {
    r.base = max(kv_len - qn + qi + 1, 0);
  }
  const int place = r.base + count - 1;
  r.beg = p.window > 0 ? max(0, place - p.window + 1) : 0;
  if (count && r.beg > r.base) {           // ancestors behind the window, those among the first tokens excepted
    int k = 0;
    for (int w = 0; w < p.words; ++w) {
      unsigned long long m = bits[w], keep = 0;
      while (m) {
        const unsigned long long bit = m & (~m + 1);
        if (r.base + k >= r.beg || r.base + k < p.first) keep |= bit;
        m ^= bit;
        ++k;
      }
      bits[w] = keep;
    }
    r.beg = r.base;                        // no context is left in the window, and nodes that stay may lie anywhere behind it
  }
  return r;
}

__device__ __forceinline__ bool span_sees(const SpanParams& p, int tok, int base, int beg, const unsigned long long* bits) {
  if (tok < base) return tok >= beg || tok < p.first;
  const int n = tok - base;
  return n < 64 * p.words && (bits[n >> 6] >> (n & 63) & 1);
}

// Tokens that the rows of a tile see between them, in pieces of `unit` tokens: the first `head` pieces of the text, then those from `lo` on.
struct SpanRange {
  int head, lo, count;
  __device__ __forceinline__ int piece(int i) const { return i < head ? i : i - head + lo; }
};
__device__ __forceinline__ SpanRange span_range(const SpanParams& p, int unit, int min_beg, int end) {
  SpanRange s;
  s.lo = min_beg / unit;
  s.head = p.first > 0 ? min((min(p.first, end) + unit - 1) / unit, s.lo) : 0;
  s.count = end > 0 ? s.head + max((end + unit - 1) / unit - s.lo, 0) : 0;
  return s;
}

// Query rows of a sequence and its length, no longer than its row of the table reaches (a walk is then bounded by the table, whatever the lengths on
// the device say); false where they are none to compute with, which is reported, as is a length out of reach.
__device__ __forceinline__ bool span_lengths(const SpanParams& p, int seq, bool report, int& q0, int& qn, int& kv_len) {
  q0 = p.q_starts[seq];
  const int end = p.q_starts[seq + 1], len = p.kv_lens[seq];
  const bool good = q0 >= 0 && end >= q0 && end <= p.tokens && end - q0 <= p.max_q_len;
  qn = good ? end - q0 : 0;
  kv_len = min(max(len, 0), p.reach);
  if ((!good || (qn > 0 && len > p.reach)) && report && p.status) atomicCAS(p.status, FLLM_OK, FLLM_ERR_BAD_ARGS);
  return qn > 0;
}

// The factor of a row's scores whose queries were multiplied by 2^up, -126 <= up <= 126. Never 0, which an infinity would make a NaN: scores whose
// factor is below the smallest normal number are below 2^-100, whatever it is.
__device__ __forceinline__ float span_factor(float scale, int up) { return fmaxf(scale * __uint_as_float((uint32_t)(127 - up) << 23), FLT_MIN); }

// Which sequence's which tile of `unit` rows is the item-th one, sequences of `from` < packed rows <= `to` counted, a sequence's last tile first; by a warp.
// `report`: lengths that are none to compute with are reported, of all sequences.
__device__ __forceinline__ bool span_find(const SpanParams& p, int unit, int from, int to, int item, bool report, int& seq, int& tile) {
  constexpr int kEach = 4;                 // sequences of a lane at a time
  const int lane = threadIdx.x & 31;
  bool found = false;
  for (int s0 = 0; s0 < p.num_seqs && (report || !found); s0 += 32 * kEach) {
    int mine[kEach], sum = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int s = s0 + lane * kEach + i;
      int q0, qn = 0, kv_len;
      if (s < p.num_seqs) span_lengths(p, s, report, q0, qn, kv_len);
      const int rows = qn * p.group;
      mine[i] = rows > from && rows <= to ? (rows + unit - 1) / unit : 0;
      sum += mine[i];
    }
    int upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    const unsigned behind = __ballot_sync(0xffffffffu, item < upto);
    if (!found && behind) {
      found = true;
      int left = item - (upto - sum), at = -1;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        if (at < 0 && left < mine[i]) {
          at = i;
          left = mine[i] - 1 - left;
        } else if (at < 0) {
          left -= mine[i];
        }
      }
      const int who = __ffs(behind) - 1;
      seq = s0 + who * kEach + __shfl_sync(0xffffffffu, at, who);
      tile = __shfl_sync(0xffffffffu, left, who);
    }
    item -= __shfl_sync(0xffffffffu, upto, 31);
  }
  return found;
}

// Block id of the 16 tokens from 16 * page on, or -1 where the table does not reach or the entry names no block of the pool.
__device__ __forceinline__ int span_block(const SpanParams& p, const int* table, int page) {
  const int at = page / p.block_pages;
  const int b = at < p.max_blocks ? table[at] : -1;
  return (unsigned)b < (unsigned)p.num_blocks ? b : -1;
}
// First row of a page of a key head in the pool seen as rows of head_dim values.
__device__ __forceinline__ long long span_pool_row(const SpanParams& p, int block, int kvh, int page) {
  return ((long long)block * p.hkv + kvh) * (16 * p.block_pages) + 16 * (page % p.block_pages);
}

// Four e4m3 bytes as f16, which holds all of their values.
__device__ __forceinline__ uint2 e4m3x4_to_f16(uint32_t w) {
  uint2 h;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\tcvt.rn.f16x2.e4m3x2 %1, hi;\n\t}" : "=r"(h.x), "=r"(h.y) : "r"(w));
  return h;
}

// bit 7 of each byte that is a NaN
__device__ __forceinline__ uint32_t e4m3_nan(uint32_t w) { return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u; }

__device__ __forceinline__ bool odd_bf16x2(uint32_t w) { return (w & 0x7F80u) == 0x7F80u || (w & 0x7F800000u) == 0x7F800000u; }
__device__ __forceinline__ bool odd_f16x2(uint32_t w) { return (w & 0x7C00u) == 0x7C00u || (w & 0x7C000000u) == 0x7C000000u; }
}  // namespace
}  // namespace fllm
