// Attention over a paged cache under a window behind which the first tokens stay visible, and for the nodes of draft trees: the kernel of
// sequences with few packed rows (query row x head of a key head), the merge of split sequences, and the choice between the kernels.
//
//   o_r = sum_j e^(s_rj - m_r) v_j / (sum_j e^(s_rj - m_r) [+ e^(sink - m_r)]),  s_rj = scale q_r . k_j,  j over what row r sees
//
// (attention_span.cuh says what that is; a row that sees nothing is 0.) One CTA per (sequence, 16 packed rows, key head, split). Its four
// warps take the 16-token pages that the rows see between them in turn: the first tokens' pages and the window's, nothing in between. Each
// streams its pages through a private cp.async ring, so the main loop has no barrier; (m, l, O) of the warps are joined in shared memory,
// those of up to eight splits in that of their cluster, of more by span_merge_kernel. Sequences with more than 16 packed rows go to attention_span_tc.cu
// where that has a kernel, and enough to do.
//
// What bounds it (times of passes in a captured graph, where the host is not waited for; a single call of a few us is some 4 us longer): memory, where there
// is enough to read (one row of 64 sequences under a window of 4096, 32 query and 8 key heads of 128: 169 us, 6.4 TB/s);
// a CTA's way in and out, some 5 us, where there is little (one sequence, a window of 256: 6.3 us); in between the latency of each warp's chain of
// products, maxima and exponentials, of which ten warps an SM hide less than half (48 sequences of an e4m3 cache under 1000 with 130 first tokens, 64 query
// and 8 key heads of 64: 22.6 us, 2.5 TB/s). Rows that read selected blocks are a CTA each (p.picks): 64 that read 128 blocks of 8 key heads of 128 take 104 us,
// 5.2 TB/s; 602 prompt rows that read 64 each 397, 6.4 TB/s of what L2 holds.
//
// Scores and sums are fp32. Weights are rounded to the operands' 16 bits for the product with the values (bf16, at most 2^-8 of each and of
// either sign; f16 beside an e4m3 cache). An e4m3 cache is widened to f16, which holds all of its values; queries are f16 there as well, times a
// power of two per row that puts the row's largest magnitude between 2^14 and 2^15: what a bf16 value loses is below 2^-38 of that magnitude.
//
// Values in places that a row does not see may be anything: a weight of zero times a NaN would be a NaN, so in pages that not every row
// sees whole, infinities and NaN of V are taken out of the tile in front of the product and added to the rows that see them. Those that a row sees show
// in its output even where their weight is 0 in 32 bits, whichever part of the walk they are in.
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <limits.h>

#include <algorithm>

#include "attention_span_rows.cuh"
#include "attention_util.cuh"
#include "tma_host.h"

namespace fllm {
namespace {
// Weights in f16 are taken to a reference 2^12 below the row's maximum: below 2^-14 of their unit they would lose bits.
constexpr float kF16Lift = 12.f;

__device__ __forceinline__ void cp_async16_or_zero(void* smem, const void* gmem, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(smem)), "l"(gmem), "r"(there ? 16 : 0) : "memory");
}

// An e4m3 page stays as it is in shared memory and becomes operands in registers, which needs no order of columns that memory does not have: a lane
// takes 16 bytes of a key row for four k-steps (queries lie in the same order), and 16 bytes of each of four value rows, two tokens of a dim to a
// register. So of column block i of O, column n is dim i of the n-th piece of 16 (or 8, at D = 64) values. (Through f16 tiles in shared memory, ldmatrix
// behind them, 48 sequences under a window of 1000 with 130 first tokens, 64 query and 8 key heads of 64, took 42 us, 31 so, both with all 16 rows.)
template <int D>
__device__ __forceinline__ int dim_of(int i, int n) {
  if constexpr (D == 64) return 8 * n + i;
  return (i >> 4) * 128 + 16 * n + (i & 15);
}
// Pieces of 16 bytes of row r lie at piece ^ this: rows next to each other (keys), every second row (values) meet other banks.
template <int D> __device__ __forceinline__ int turn_k(int r) { return D == 64 ? 0 : (r & 1) << 2; }
template <int D> __device__ __forceinline__ int turn_v(int r) { return D == 64 ? (r >> 1) & 3 : r & 6; }

template <int D, bool KV8>
struct RowsSmem {
  static constexpr int kPages = KV8 && D <= 128 ? 2 : 1;                 // of a turn of a warp
  static constexpr int kStages = KV8 ? (D == 64 ? 6 : 4) : D == 256 ? 2 : 3;
  static constexpr int kPageElems = kPage * D;
  static constexpr int kPageBytes = kPageElems * (KV8 ? 1 : 2);          // a K or V page
  static constexpr int kWarpRing = kStages * 2 * kPageBytes;
  static constexpr int kRing = 4 * kWarpRing;
  static constexpr int kMerge = 4 * kSpanRows * (D + 2) * 4, kPart = kSpanRows * (D + 4) * 4;
  static constexpr int kQPitch = D + (KV8 ? 8 : 0);
  static constexpr int kQ = kSpanRows * kQPitch * 2;
  static constexpr int kInfo = kSpanRows * (8 * kSpanWords + 4 * 3);
  static constexpr int kTotal = kQ + kInfo + kRing + 128;
  static_assert(kMerge + kPart <= kRing && kQ % 16 == 0 && kInfo % 16 == 0, "shared memory");
};

// CTAs of an SM, by registers and shared memory.
template <int D, bool KV8> constexpr int rows_resident() { return D == 256 ? 1 : D == 64 ? 4 : KV8 ? 3 : 2; }

// NARROW: up to 8 packed rows, for which scores and sums are transposed, S^T = K Q^T and O^T = V^T P^T: the products' 16 rows are tokens and dims, their
// 8 columns the rows, and nothing is computed for rows 8 to 15. A lane's operands are the same registers in another order; it holds scores of rows 2t and
// 2t + 1 and tokens g and g + 8 (otherwise rows g and g + 8 and tokens 2t, 2t + 1 of each half). us of decode rows, so and with 16 rows: 48 sequences of an
// e4m3 cache under 1000 with 130 first tokens, 64 query and 8 key heads of 64: 22.6, 28.8; one under 256, 32 and 8 of 128: 6.3, 6.8; 64 under 4096: 166 both.
// MODE: whose rows a CTA's are, as its place says, looked up (p.search; its code in all calls cost the smallest 3 %), or one row's, which reads selected
// blocks (p.picks; up to 16 heads at a time).
template <int D, bool KV8, bool NARROW, int MODE>
__global__ void __launch_bounds__(128, rows_resident<D, KV8>()) span_rows_kernel(const __grid_constant__ SpanParams p) {
  using S = RowsSmem<D, KV8>;
  extern __shared__ __align__(128) uint8_t smem[];
  bf16* qtile = reinterpret_cast<bf16*>(smem);
  unsigned long long* bits = reinterpret_cast<unsigned long long*>(smem + S::kQ);      // [16][4]
  int* bases = reinterpret_cast<int*>(bits + kSpanRows * kSpanWords);
  int* begs = bases + kSpanRows;
  float* factors = reinterpret_cast<float*>(begs + kSpanRows);                         // of a row's scores, to base 2
  uint8_t* ring = smem + S::kQ + S::kInfo;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int G = p.group;
  int work = blockIdx.x / p.splits;
  const int split = blockIdx.x - work * p.splits;
  const int kvh = work % p.hkv;
  work /= p.hkv;
  pdl_launch_dependents();
  pdl_wait();
  int seq, row0, n_rows, q0, qn, kv_len;
  if (!span_rows_of_cta<MODE>(p, work, split, seq, row0, n_rows, q0, qn, kv_len)) return;

  // Every warp finds out what the rows see for itself (a lane to a row), so that its pages are on their way before the queries are.
  int min_base = INT_MAX, max_base = 0, min_beg = INT_MAX, max_beg = 0;      // what they see between them, and what all of them see
  if (lane < kSpanRows) {
    SpanRow r{0, 0};
    unsigned long long mine[kSpanWords] = {0, 0, 0, 0};
    if (lane < n_rows) {
      r = span_row(p, q0, qn, kv_len, (row0 + lane) / G, mine);
      min_base = max_base = r.base;
      min_beg = max_beg = r.beg;
    }
    if (warp == 0) {
      bases[lane] = r.base;
      begs[lane] = r.beg;
#pragma unroll
      for (int w = 0; w < kSpanWords; ++w) bits[lane * kSpanWords + w] = mine[w];
    }
  }
  min_base = __reduce_min_sync(0xffffffffu, min_base);
  max_base = __reduce_max_sync(0xffffffffu, max_base);
  min_beg = __reduce_min_sync(0xffffffffu, min_beg);
  max_beg = __reduce_max_sync(0xffffffffu, max_beg);
  const SpanWalk<MODE> range = span_walk<MODE>(p, q0, row0, kvh, min_beg, max_base, kv_len, warp == 0 && split == 0);
  const int per_split = max(p.min_pages, (range.count + p.splits - 1) / p.splits);
  const int pg0 = min(split * per_split, range.count), pg1 = min(pg0 + per_split, range.count);

  uint8_t* my_ring = ring + (size_t)warp * S::kWarpRing;
  const int* table = p.block_tables + (size_t)seq * p.max_blocks;
  bool bad = false;
  // Blocks of this warp's pages, one to a lane, 32 at a time and those ahead of their use: a table entry looked up where it is needed held every page
  // back by a trip to memory.
  auto look = [&](int it) {
    const int pg = pg0 + warp + 4 * (it + lane);
    const int block = pg < pg1 ? span_block(p, table, range.piece(pg)) : 0;
    bad |= block < 0;
    return block;
  };
  int blocks = 0, blocks_next = look(0);
  auto issue = [&](int it) {
    const int pg = pg0 + warp + 4 * it;
    if ((it & 31) == 0) { blocks = blocks_next; blocks_next = look(it + 32); }
    if (pg < pg1) {
      const int page = range.piece(pg);
      const int block = __shfl_sync(0xffffffffu, blocks, it & 31);
      const long long off = block < 0 ? 0 : span_pool_row(p, block, kvh, page) * D;
      uint8_t* st = my_ring + (size_t)(it % S::kStages) * 2 * S::kPageBytes;
      if constexpr (KV8) {
        const uint8_t *kg = static_cast<const uint8_t*>(p.k_cache) + off, *vg = static_cast<const uint8_t*>(p.v_cache) + off;
#pragma unroll
        for (int i = lane; i < S::kPageBytes / 16; i += 32) {
          const int r = i / (D / 16), c = i - r * (D / 16);
          cp_async16_or_zero(st + r * D + ((c ^ turn_k<D>(r)) << 4), kg + i * 16, block >= 0);
          cp_async16_or_zero(st + S::kPageBytes + r * D + ((c ^ turn_v<D>(r)) << 4), vg + i * 16, block >= 0);
        }
      } else {
        const bf16 *kg = static_cast<const bf16*>(p.k_cache) + off, *vg = static_cast<const bf16*>(p.v_cache) + off;
        bf16* ks = reinterpret_cast<bf16*>(st);
#pragma unroll 8
        for (int i = lane; i < kPage * (D / 8); i += 32) {
          const int r = i / (D / 8), c = i - r * (D / 8);
          cp_async16_or_zero(tile_ptr<D>(ks, r, c), kg + i * 8, block >= 0);
          cp_async16_or_zero(tile_ptr<D>(ks + S::kPageElems, r, c), vg + i * 8, block >= 0);
        }
      }
    }
    cp_async_commit();
  };
  const int my_pages = pg1 > pg0 + warp ? (pg1 - pg0 - warp + 3) / 4 : 0;
  constexpr int kPages = S::kPages;
#pragma unroll
  for (int s = 0; s < S::kStages - kPages; ++s) issue(s);
  // queries; a row's 16-byte pieces lie with D / 8 neighbouring threads
#pragma unroll
  for (int i = threadIdx.x; i < kSpanRows * (D / 8); i += 128) {
    const int r = i / (D / 8), c = i - r * (D / 8);
    uint4 v = make_uint4(0, 0, 0, 0);
    if (r < n_rows) {
      const int qi = (row0 + r) / G, hg = (row0 + r) - qi * G;
      v = *reinterpret_cast<const uint4*>(static_cast<const bf16*>(p.q) + (size_t)(q0 + qi) * p.ldq + (size_t)(kvh * G + hg) * D + c * 8);
    }
    float factor = p.scale_log2;
    if constexpr (KV8) {
      uint32_t* w = reinterpret_cast<uint32_t*>(&v);
      uint32_t top = 0;                    // largest exponent field of the row, infinities and NaN aside
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t a = w[e] >> 7 & 0xFF, b = w[e] >> 23 & 0xFF;
        if (a != 0xFF) top = max(top, a);
        if (b != 0xFF) top = max(top, b);
      }
#pragma unroll
      for (int o = (D / 8 < 32 ? D / 8 : 32) / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      const int up = min(127 + 14 - (int)top, 126);
      const float f = __uint_as_float((uint32_t)(127 + up) << 23);
      factor = span_factor(factor, up);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 x = unpack_bf16x2(w[e]);
        w[e] = pack_16<true>(x.x * f, x.y * f);
      }
      *reinterpret_cast<uint4*>(qtile + r * S::kQPitch + c * 8) = v;
    } else {
      *reinterpret_cast<uint4*>(tile_ptr<D>(qtile, r, c)) = v;
    }
    if (c == 0) factors[r] = factor;
  }
  __syncthreads();
  uint32_t qf[D / 16][4];
  if constexpr (KV8) {
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {     // k-step k % 4 of 64 dims: a lane's two pairs of columns are its four bytes of that step
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint2 v = *reinterpret_cast<const uint2*>(qtile + (g + 8 * h) * S::kQPitch + (k >> 2) * 64 + 16 * t + 4 * (k & 3));
        qf[k][h] = v.x;
        qf[k][2 + h] = v.y;
      }
    }
  } else {
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) ldsm_x4(qf[kk], tile_ptr<D>(qtile, lane & 15, 2 * kk + (lane >> 4)));
  }

  const int row_a = NARROW ? 2 * t : g, row_b = NARROW ? 2 * t + 1 : g + 8;           // a lane's rows
  const int base0 = bases[row_a], base1 = bases[row_b], beg0 = begs[row_a], beg1 = begs[row_b];
  const float f0 = factors[row_a], f1 = factors[row_b];
  const unsigned long long *bits0 = bits + row_a * kSpanWords, *bits1 = bits + row_b * kSpanWords;

  constexpr int kO = NARROW ? D / 16 : D / 8, kS = NARROW ? kPages : 2 * kPages;      // accumulators of O and of S
  // value `x` of a lane (0 to 3) in an accumulator: which of its rows, which of the two places (tokens, column blocks) along the other side
  constexpr auto second_row = [](int x) { return NARROW ? x & 1 : x >> 1; };
  float o[kO][4];
#pragma unroll
  for (int i = 0; i < kO; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

  // kPages pages at a time: with two there are two chains of products and one maximum for both. (One that is not there any more has no token that
  // a row sees.)
  for (int it = 0; it < my_pages; it += kPages) {
#pragma unroll
    for (int h = 0; h < kPages; ++h) issue(it + h + S::kStages - kPages);
    cp_async_wait<S::kStages - kPages>();
    __syncwarp();
    const uint8_t* page_at[kPages];
    int tok0[kPages];
    bool full[kPages];
#pragma unroll
    for (int h = 0; h < kPages; ++h) {
      page_at[h] = my_ring + (size_t)((it + h) % S::kStages) * 2 * S::kPageBytes;
      const bool there = h == 0 || it + h < my_pages;
      tok0[h] = there ? range.piece(pg0 + warp + 4 * (it + h)) * kPage : INT_MAX / 2;
      full[h] = tok0[h] + kPage <= min_base && (tok0[h] >= max_beg || tok0[h] + kPage <= p.first);
    }
    float s[kS][4];
#pragma unroll
    for (int i = 0; i < kS; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
    const int j = lane >> 3;
    if constexpr (KV8) {
#pragma unroll
      for (int grp = 0; grp < D / 64; ++grp) {
#pragma unroll
        for (int h = 0; h < kPages; ++h) {
          uint32_t w[2][4];                // tokens g and g + 8
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int r = 8 * half + g;
            const uint4 raw = *reinterpret_cast<const uint4*>(page_at[h] + r * D + (((4 * grp + t) ^ turn_k<D>(r)) << 4));
            w[half][0] = raw.x; w[half][1] = raw.y; w[half][2] = raw.z; w[half][3] = raw.w;
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint2 x = e4m3x4_to_f16(w[0][k]), y = e4m3x4_to_f16(w[1][k]);
            const uint32_t(&q)[4] = qf[4 * grp + k];
            if constexpr (NARROW) {
              const uint32_t a[4] = {x.x, y.x, x.y, y.y};
              mma_f16(s[h], a, q[0], q[2]);
            } else {
              mma_f16(s[2 * h], q, x.x, x.y);
              mma_f16(s[2 * h + 1], q, y.x, y.y);
            }
          }
        }
      }
    } else {
      bf16* ks = reinterpret_cast<bf16*>(const_cast<uint8_t*>(page_at[0]));
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        uint32_t b[4];
        ldsm_x4(b, tile_ptr<D>(ks, (j >> 1) * 8 + (lane & 7), 2 * kk + (j & 1)));
        if constexpr (NARROW) {
          const uint32_t a[4] = {b[0], b[2], b[1], b[3]};
          mma_bf16(s[0], a, qf[kk][0], qf[kk][2]);
        } else {
          mma_bf16(s[0], qf[kk], b[0], b[1]);
          mma_bf16(s[1], qf[kk], b[2], b[3]);
        }
      }
    }
    float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
    for (int i = 0; i < kS; ++i) {
      const int h = NARROW ? i : i >> 1;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float v = s[i][e] * (second_row(e) ? f1 : f0);
        if (p.softcap > 0.f) v = p.softcap * tanhf(v / (p.softcap * kLog2e)) * kLog2e;
        if (!full[h]) {
          const int tok = tok0[h] + (NARROW ? g + 8 * (e >> 1) : (i & 1) * 8 + 2 * t + (e & 1));
          if (!(second_row(e) ? span_sees(p, tok, base1, beg1, bits1) : span_sees(p, tok, base0, beg0, bits0))) v = -INFINITY;
        }
        s[i][e] = v;
        if (second_row(e)) mx1 = fmaxf(mx1, v);
        else mx0 = fmaxf(mx0, v);
      }
    }
    constexpr int kNext = NARROW ? 4 : 1, kLast = NARROW ? 16 : 2;       // a row's lanes
#pragma unroll
    for (int x = kNext; x <= kLast; x *= 2) {
      mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, x));
      mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, x));
    }
    const float mn0 = fmaxf(m[0], mx0), mn1 = fmaxf(m[1], mx1);
    constexpr float lift = KV8 ? kF16Lift : 0.f;
    const float r0 = mn0 == -INFINITY ? 0.f : mn0 - lift, r1 = mn1 == -INFINITY ? 0.f : mn1 - lift;
    if (__any_sync(0xffffffffu, mn0 != m[0] || mn1 != m[1])) {
      const float c0 = mn0 == -INFINITY ? 1.f : ex2(m[0] - mn0), c1 = mn1 == -INFINITY ? 1.f : ex2(m[1] - mn1);
      l[0] *= c0;
      l[1] *= c1;
#pragma unroll
      for (int i = 0; i < kO; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[i][x] *= second_row(x) ? c1 : c0;
      m[0] = mn0;
      m[1] = mn1;
    }
    uint32_t pf[kPages][NARROW ? 2 : 4];               // narrow: of tokens g and g + 8, both rows
#pragma unroll
    for (int i = 0; i < kS; ++i) {
      float e[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) e[x] = ex2(s[i][x] - (second_row(x) ? r1 : r0));
      l[0] += e[0] + e[NARROW ? 2 : 1];
      l[1] += e[NARROW ? 1 : 2] + e[3];
      uint32_t* w = NARROW ? pf[i] : pf[i >> 1] + 2 * (i & 1);
      w[0] = pack_16<KV8>(e[0], e[1]);
      w[1] = pack_16<KV8>(e[2], e[3]);
    }
    // infinities and NaN of V in a page that not every row sees whole: value(token, column block, column of it)
    auto add_odd = [&](int h, auto value) {
      for (int tk = 0; tk < kPage; ++tk) {
        float w0, w1;
        if constexpr (NARROW) {
          const float2 a = unpack_16<KV8>(__shfl_sync(0xffffffffu, tk < 8 ? pf[h][0] : pf[h][1], (tk & 7) << 2 | t));
          w0 = a.x; w1 = a.y;
        } else {
          const int src = (lane & ~3) | (tk & 7) >> 1;
          const float2 a = unpack_16<KV8>(__shfl_sync(0xffffffffu, tk < 8 ? pf[h][0] : pf[h][2], src));
          const float2 b = unpack_16<KV8>(__shfl_sync(0xffffffffu, tk < 8 ? pf[h][1] : pf[h][3], src));
          w0 = tk & 1 ? a.y : a.x; w1 = tk & 1 ? b.y : b.x;
        }
        const bool sees0 = span_sees(p, tok0[h] + tk, base0, beg0, bits0), sees1 = span_sees(p, tok0[h] + tk, base1, beg1, bits1);
#pragma unroll
        for (int i = 0; i < kO; ++i) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float v = NARROW ? value(tk, 2 * i + e, g) : value(tk, i, 2 * t + e);
            if (isfinite(v)) continue;
            if (sees0) o[i][NARROW ? 2 * e : e] += w0 * v;
            if (sees1) o[i][NARROW ? 2 * e + 1 : 2 + e] += w1 * v;
          }
        }
      }
      __syncwarp();
    };
    uint32_t pt[kPages][2];
    if constexpr (NARROW) {
#pragma unroll
      for (int h = 0; h < kPages; ++h) { pt[h][0] = transposed(pf[h][0]); pt[h][1] = transposed(pf[h][1]); }
    }
    if constexpr (KV8) {
      constexpr int kWords = D == 64 ? 2 : 4, kParts = D == 256 ? 2 : 1;
#pragma unroll
      for (int h = 0; h < kPages; ++h) {
        const uint8_t* v8 = page_at[h] + S::kPageBytes;
        uint32_t nan = 0;
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
          uint32_t w[4][kWords];           // rows 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = 2 * t + (i & 1) + 8 * (i >> 1);
            if constexpr (D == 64) {
              const uint2 x = *reinterpret_cast<const uint2*>(v8 + r * D + (((g >> 1) ^ turn_v<D>(r)) << 4) + (g & 1) * 8);
              w[i][0] = x.x; w[i][1] = x.y;
            } else {
              const uint4 x = *reinterpret_cast<const uint4*>(v8 + r * D + (((8 * part + g) ^ turn_v<D>(r)) << 4));
              w[i][0] = x.x; w[i][1] = x.y; w[i][2] = x.z; w[i][3] = x.w;
            }
          }
          if (tok0[h] == INT_MAX / 2) {    // what lies there is of another page
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int k = 0; k < kWords; ++k) w[i][k] = 0;
          } else if (!full[h]) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int k = 0; k < kWords; ++k) {
                const uint32_t n = e4m3_nan(w[i][k]);
                nan |= n;
                w[i][k] &= ~((n >> 7) * 0xFFu);
              }
            if (__any_sync(0xffffffffu, nan) && part == kParts - 1)
              add_odd(h, [&](int tk, int db, int col) {
                const int d = dim_of<D>(db, col);
                const uint8_t x = v8[tk * D + (((d >> 4) ^ turn_v<D>(tk)) << 4) + (d & 15)];
                return (x & 0x7F) == 0x7F ? __int_as_float(0x7FC00000) : 0.f;
              });
          }
#pragma unroll
          for (int k = 0; k < kWords; ++k) {
            const uint2 a = e4m3x4_to_f16(__byte_perm(w[0][k], w[1][k], 0x5140)), b = e4m3x4_to_f16(__byte_perm(w[0][k], w[1][k], 0x7362));
            const uint2 c = e4m3x4_to_f16(__byte_perm(w[2][k], w[3][k], 0x5140)), d = e4m3x4_to_f16(__byte_perm(w[2][k], w[3][k], 0x7362));
            if constexpr (NARROW) {
              const uint32_t v0[4] = {a.x, a.y, c.x, c.y}, v1[4] = {b.x, b.y, d.x, d.y};
              mma_f16(o[8 * part + 2 * k], v0, pt[h][0], pt[h][1]);
              mma_f16(o[8 * part + 2 * k + 1], v1, pt[h][0], pt[h][1]);
            } else {
              mma_f16(o[16 * part + 4 * k], pf[h], a.x, c.x);
              mma_f16(o[16 * part + 4 * k + 1], pf[h], a.y, c.y);
              mma_f16(o[16 * part + 4 * k + 2], pf[h], b.x, d.x);
              mma_f16(o[16 * part + 4 * k + 3], pf[h], b.y, d.y);
            }
          }
        }
      }
    } else {
      bf16* vs = reinterpret_cast<bf16*>(const_cast<uint8_t*>(page_at[0])) + S::kPageElems;
      if (!full[0]) {
        uint32_t* vw = reinterpret_cast<uint32_t*>(vs);
        bool odd = false;
#pragma unroll 4
        for (int i = lane; i < kPage * D / 2; i += 32) odd |= odd_bf16x2(vw[i]);
        if (__any_sync(0xffffffffu, odd)) {
          add_odd(0, [&](int tk, int db, int col) { return __bfloat162float(tile_ptr<D>(vs, tk, db)[col]); });
          for (int i = lane; i < kPage * D / 2; i += 32) {
            const uint32_t w = vw[i];
            if (odd_bf16x2(w)) vw[i] = (odd_bf16x2(w & 0xFFFFu) ? 0u : w & 0xFFFFu) | (odd_bf16x2(w & 0xFFFF0000u) ? 0u : w & 0xFFFF0000u);
          }
          __syncwarp();
        }
      }
#pragma unroll
      for (int db = 0; db < D / 8; db += 2) {
        uint32_t b[4];
        ldsm_x4_t(b, tile_ptr<D>(vs, (j & 1) * 8 + (lane & 7), db + (j >> 1)));
        if constexpr (NARROW) {
          const uint32_t a[4] = {b[0], b[2], b[1], b[3]};
          mma_bf16(o[db / 2], a, pt[0][0], pt[0][1]);
        } else {
          mma_bf16(o[db], pf[0], b[0], b[1]);
          mma_bf16(o[db + 1], pf[0], b[2], b[3]);
        }
      }
    }
    __syncwarp();
  }
  cp_async_wait<0>();
  if (bad && p.status) atomicCAS(p.status, FLLM_OK, FLLM_ERR_BAD_ARGS);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
#pragma unroll
    for (int x = NARROW ? 4 : 1; x <= (NARROW ? 16 : 2); x *= 2) l[i] += __shfl_xor_sync(0xffffffffu, l[i], x);
  }
  if constexpr (KV8) { m[0] -= kF16Lift; m[1] -= kF16Lift; }

  __syncthreads();                                     // the ring is free
  float* mo = reinterpret_cast<float*>(ring);          // [4][16][D]
  float* mml = mo + 4 * kSpanRows * D;                 // [4][16][2]
  float* part_o = mml + 4 * kSpanRows * 2;             // [16][D]: the CTA's
  float4* part_ml = reinterpret_cast<float4*>(part_o + kSpanRows * D);      // [16]
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = h ? row_b : row_a;
    float* row = mo + ((size_t)warp * 16 + r) * D;
    if constexpr (NARROW && KV8) {
#pragma unroll
      for (int i = 0; i < kO; i += 2) *reinterpret_cast<float4*>(row + dim_of<D>(2 * i, g)) = make_float4(o[i][h], o[i][2 + h], o[i + 1][h], o[i + 1][2 + h]);
    } else if constexpr (NARROW) {
#pragma unroll
      for (int i = 0; i < kO; ++i) { row[16 * i + g] = o[i][h]; row[16 * i + 8 + g] = o[i][2 + h]; }
    } else if constexpr (KV8) {                        // a lane has four neighbouring dims in four neighbouring column blocks
#pragma unroll
      for (int db = 0; db < D / 8; db += 4)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          *reinterpret_cast<float4*>(row + dim_of<D>(db, 2 * t + e)) = make_float4(o[db][2 * h + e], o[db + 1][2 * h + e], o[db + 2][2 * h + e], o[db + 3][2 * h + e]);
    } else {
#pragma unroll
      for (int db = 0; db < D / 8; ++db) *reinterpret_cast<float2*>(row + db * 8 + 2 * t) = make_float2(o[db][2 * h], o[db][2 * h + 1]);
    }
    if ((NARROW ? g : t) == 0) *reinterpret_cast<float2*>(mml + (warp * 16 + r) * 2) = make_float2(m[h], l[h]);
  }
  span_join<D>(p, mo, mml, part_o, part_ml, q0, row0, n_rows, kvh, split);
}

// Joins the splits of a row: one warp per (token, head). `some`: sequences of at most p.rows_from packed rows were another kernel's.
template <int D>
__global__ void __launch_bounds__(128) span_merge_kernel(const __grid_constant__ SpanParams p, int some) {
  pdl_launch_dependents();
  pdl_wait();
  const int pair = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (pair >= p.tokens * p.hq) return;
  const int tok = pair / p.hq, head = pair - tok * p.hq;
  if (tok < p.q_starts[0] || tok >= p.q_starts[p.num_seqs]) return;      // rows of no sequence stay as they are
  if (some) {
    int lo = 0, hi = p.num_seqs;                       // the last sequence that begins at or before tok
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (p.q_starts[mid] <= tok) lo = mid;
      else hi = mid;
    }
    const int rows = (p.q_starts[lo + 1] - p.q_starts[lo]) * p.group;
    if (rows <= p.rows_from) return;
  }
  const float2* ml = reinterpret_cast<const float2*>(p.ws_ml) + (size_t)pair * p.splits;
  const float* part = p.ws_o + (size_t)pair * p.splits * D + lane;
  float2 mine = lane < p.splits ? __ldcg(ml + lane) : make_float2(-INFINITY, 0.f);
  if (__shfl_sync(0xffffffffu, mine.y, 0) < 0.f) return;      // the row was not split
  const float sk = p.sinks ? p.sinks[head] * kLog2e : -INFINITY;
  float mm = mine.x;
  for (int s = lane + 32; s < p.splits; s += 32) mm = fmaxf(mm, __ldcg(ml + s).x);
  const float top = warp_max(mm);
  mm = fmaxf(top, sk);
  float ll = 0.f, a[D / 32];
#pragma unroll
  for (int e = 0; e < D / 32; ++e) a[e] = 0.f;
  for (int s0 = 0; s0 < p.splits; s0 += 32) {
    if (s0) mine = s0 + lane < p.splits ? __ldcg(ml + s0 + lane) : make_float2(-INFINITY, 0.f);
    const float w = mine.x == -INFINITY ? (mm == -INFINITY && mine.y != 0.f ? 1.f : 0.f) : ex2(mine.x - mm);
    ll += mine.y * w;
    // A part that saw nothing has no row to read. One whose factor is 0 has: an infinity or a NaN of its values shows as it does within a part.
    unsigned live = __ballot_sync(0xffffffffu, mine.x != -INFINITY || mine.y != 0.f);
    while (live) {
      int at[4];
      float x[4][D / 32];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        at[k] = live ? __ffs(live) - 1 : -1;
        live &= live - 1;
#pragma unroll
        for (int e = 0; e < D / 32; ++e) x[k][e] = at[k] >= 0 ? __ldcg(part + (size_t)(s0 + at[k]) * D + 32 * e) : 0.f;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float wk = __shfl_sync(0xffffffffu, w, at[k] & 31);
        if (at[k] >= 0) {
#pragma unroll
          for (int e = 0; e < D / 32; ++e) a[e] += x[k][e] * wk;
        }
      }
    }
  }
  ll = warp_sum(ll);
  if (p.sinks && (top != -INFINITY || ll != 0.f)) ll += ex2(sk - mm);        // (see store_row)
  const float inv = ll == 0.f ? 0.f : 1.f / ll;
  bf16* dst = static_cast<bf16*>(p.out) + (size_t)tok * p.ldo + (size_t)head * D + lane;
#pragma unroll
  for (int e = 0; e < D / 32; ++e) dst[32 * e] = __float2bfloat16(a[e] * inv);
}

long long most_rows(const SpanParams& p) { return p.picks ? p.group : std::min<long long>((long long)p.max_q_len * p.group, p.rows_to); }
template <int D, bool KV8, bool NARROW>
void launch_rows(SpanParams p, cudaStream_t s) {
  constexpr int smem = RowsSmem<D, KV8>::kTotal;
  static bool configured[kMaxDevices] = {};
  if (first_call_on_device(configured)) {
    cuda_check(cudaFuncSetAttribute(span_rows_kernel<D, KV8, NARROW, kAsked>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), "span_rows smem");
    cuda_check(cudaFuncSetAttribute(span_rows_kernel<D, KV8, NARROW, kSearch>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), "span_rows smem");
    cuda_check(cudaFuncSetAttribute(span_rows_kernel<D, KV8, NARROW, kPicked>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), "span_rows smem");
  }
  const long long ctas = span_rows_ctas(p) * p.splits;
  if (ctas > INT_MAX) throw std::runtime_error("attention_span: too many query rows");
  auto go = [&](auto kernel) {
    if (p.in_cluster) launch_cluster(true, kernel, dim3((unsigned)ctas), dim3(128), smem, s, (unsigned)p.splits, p);
    else launch_pdl(kernel, dim3((unsigned)ctas), dim3(128), smem, s, p);
  };
  if (p.picks) go(span_rows_kernel<D, KV8, NARROW, kPicked>);
  else if (p.search) go(span_rows_kernel<D, KV8, NARROW, kSearch>);
  else go(span_rows_kernel<D, KV8, NARROW, kAsked>);
}
template <int D>
void launch_rows_of(const SpanParams& p, cudaStream_t s) {
  if (most_rows(p) <= 8) p.kv_fp8 ? launch_rows<D, true, true>(p, s) : launch_rows<D, false, true>(p, s);
  else p.kv_fp8 ? launch_rows<D, true, false>(p, s) : launch_rows<D, false, false>(p, s);
}
template <int D>
void launch_merge(const SpanParams& p, bool some, cudaStream_t s) {
  launch_pdl(span_merge_kernel<D>, dim3((unsigned)(((long long)p.tokens * p.hq + 3) / 4)), dim3(128), 0, s, p, some ? 1 : 0);
}
void merge(const SpanParams& p, bool some, cudaStream_t s) {
  if (p.head_dim == 64) launch_merge<64>(p, some, s);
  else if (p.head_dim == 128) launch_merge<128>(p, some, s);
  else launch_merge<256>(p, some, s);
}
size_t partial_floats(const SpanParams& p, int splits) { return splits > 1 ? (size_t)p.tokens * p.hq * splits * (p.head_dim + 2) : 0; }
}  // namespace

long long span_rows_ctas(SpanParams& p) {
  if (p.picks) {
    p.search = false;
    return (long long)p.tokens * p.hkv * ((p.group + kSpanRows - 1) / kSpanRows);
  }
  return span_tiles(p, most_rows(p), kSpanRows, p.search) * p.hkv;
}

SpanPlan attention_span_plan(const SpanParams& p) {
  SpanPlan plan{};
  const long long most = (long long)p.max_q_len * p.group;
  const long long reach = p.picks ? (long long)p.pick_count * kPage * p.block_pages : p.window > 0 ? (long long)p.window + p.first + p.max_q_len : p.max_kv_len;
  const long long span = std::min<long long>(reach, p.max_kv_len);
  // Sequences of more than 16 packed rows go to the tensor-memory kernel, unless all there is to do is less than 28 pages of 16 rows for each SM: its way
  // in and out is longer (one tree of 8, 12, 32 and 64 nodes behind 900 tokens, 32 query and 8 key heads of 128: 10.6, 11.0, 13.9, 20.4 us here, 15.5, 15.6,
  // 16.1, 18.6 there; 12 nodes behind 4000: 19.2 and 18.6).
  bool search;
  const long long all_tiles = span_tiles(p, most, kSpanRows, search) * p.hkv;
  const bool tc = !p.picks && attention_span_tc_supported(p) && all_tiles * ((span + kPage - 1) / kPage) > 28LL * sm_count();
  if (!tc || (long long)p.min_q_len * p.group <= kSpanRows) {
    SpanParams rows = p;
    rows.rows_to = tc ? kSpanRows : INT_MAX;
    const long long ctas = span_rows_ctas(rows);
    const long long pages = (span + kPage - 1) / kPage;
    // As many splits as leave all CTAs on the SMs at once, four pages at least, one for each of a CTA's warps (over a 4-bit cache a warp takes up to four at a
    // time: in pieces of fewer than 16 some warps have none): a CTA's way in and out is some 5 us (64 sequences
    // under a window of 4096, 8 key heads of 128: 170 us whole, 182 in two, 202 in four; 16 under one of 1024: 24, 17, 24). Up to eight are a
    // cluster and join in it; more, where few sequences are long, leave their rows to a kernel behind.
    const int resident = p.kv4 ? attention_kv4_resident(rows) : p.head_dim == 256 ? 1 : p.head_dim == 64 ? rows_resident<64, false>() : p.kv_fp8 ? rows_resident<128, true>() : rows_resident<128, false>();
    plan.min_pages = 4;
    long long splits = std::min<long long>((long long)resident * sm_count() / ctas, (pages + plan.min_pages - 1) / plan.min_pages);
    // Over a 4-bit cache more than a wave of CTAs of at most 512 pages: sequences are of different lengths, and with one piece each the longest hold their SMs
    // alone in the end (64 of 4000 to 32,000 tokens: 417 us in one piece, 291 in four, 340 in eight; all of 16,000: 266 in one, 229 in two).
    if (p.kv4) splits = std::max(splits, std::min<long long>(8, (pages + 511) / 512));
    if (splits > 8 && (pages < 8 * 64 || (tc && most > kSpanRows))) splits = 8;      // (their workspace would have room for the other kernel's rows, too)
    plan.rows_splits = (int)std::max<long long>(1, std::min<long long>(splits, 128));
    plan.in_cluster = plan.rows_splits > 1 && plan.rows_splits <= 8;
  }
  if (tc && most > kSpanRows) {
    // at most four places for a piece to each SM: those that the kernel finds no work for cost a start all the same
    const long long ctas = span_tiles(p, most, 256, search) * p.hkv, tiles = (span + 127) / 128 + 2;
    plan.tile_splits = (int)std::max<long long>(1, std::min<long long>(std::min<long long>(4LL * sm_count() / ctas, tiles), 32));
  }
  plan.bytes = (partial_floats(p, plan.in_cluster ? 1 : plan.rows_splits) + partial_floats(p, plan.tile_splits)) * sizeof(float);
  return plan;
}

int attention_span(SpanParams p, const SpanPlan& plan, void* workspace, cudaStream_t s) {
  int n = 0;
  p.min_pages = plan.min_pages;
  p.sms = sm_count();
  auto take = [&](int splits) {
    p.splits = splits;
    p.ws_o = static_cast<float*>(workspace);
    p.ws_ml = p.ws_o + (size_t)p.tokens * p.hq * splits * p.head_dim;
    workspace = p.ws_o + partial_floats(p, splits);
  };
  if (plan.tile_splits > 0) {
    take(plan.tile_splits);
    p.rows_from = plan.rows_splits > 0 ? kSpanRows : 0;
    p.rows_to = INT_MAX;
    attention_span_tc(p, s);
    ++n;
    if (p.splits > 1) { merge(p, plan.rows_splits > 0, s); ++n; }
  }
  if (plan.rows_splits > 0) {
    take(plan.rows_splits);
    p.in_cluster = plan.in_cluster;
    p.rows_from = 0;
    p.rows_to = plan.tile_splits > 0 ? kSpanRows : INT_MAX;
    if (p.kv4) attention_kv4_rows(p, s);
    else switch (p.head_dim) {
      case 64: launch_rows_of<64>(p, s); break;
      case 128: launch_rows_of<128>(p, s); break;
      default: launch_rows_of<256>(p, s); break;
    }
    ++n;
    if (p.splits > 1 && !p.in_cluster) { merge(p, false, s); ++n; }      // (the only kernel then)
  }
  cuda_check(cudaGetLastError(), "attention_span launch");
  return n;
}
}  // namespace fllm
