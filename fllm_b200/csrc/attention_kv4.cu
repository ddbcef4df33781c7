// Attention over a cache held in 4 bits (kv4.cuh): sequences with few packed rows (query row x head of a key head), and rows that read selected blocks.
// What a row sees, the splits of a walk and their join are those of attention_span.cu.
//
// A key is z + s c with codes c of 0 to 15, so q . k = s (q . c) + z sum(q): the product is one of queries with codes, step and lowest value come to a
// score once for each token. In the same way o = sum_t (p_t s_t) (c_t - 8) + sum_t p_t (z_t + 8 s_t): the step goes into the weight, the second sum is one
// number a row. So codes are never widened to values: a code is a 16-bit operand as it lies in a word. The bits of c are those of the f16 number c 2^-24 (a
// denormal, which the tensor cores multiply exactly), those of c << 4 are c 2^-20. A word's eight codes are four registers of two, by a mask each and a
// shift for the last two; registers of odd codes hold 16 times as much, which queries (times 1/16 there) or the sums of odd dims make up for. (e4m3 operands,
// of which a byte with a code in it is one as it is, took a quarter longer.) Codes of values are counted from the middle of their range, in that 8 times
// the sum of the weights, a product with ones, is taken off the sums every eighth turn: sums of c alone grow with the text where those of values do
// not, and what the tensor cores cut off of each (it is not rounded) grew to 7e-4 of the outputs over 18,000 tokens.
//
// Scores are transposed, S^T = K Q^T and O^T = V^T P^T: the products' 16 rows are tokens and dims, their 8 columns packed rows, so that nothing is computed
// for rows that are not there (NB: 8 or 16 of them). Of O^T the contraction runs over tokens: two tokens' words of the same dims make the pairs.
//
// Queries are f16 times a power of two for each row (the largest magnitude between 2^14 and 2^15): what a bf16 value loses is below 2^-38 of that
// magnitude, 2^-34 in odd dims. Weights times steps are f16 too, in units of 2^U, U above the exponents of the steps that the warp has met, and of 2^-6:
// a row's reference is moved where a score is more than 8 above it (to base 2), so they stay below 2^15, and those of less than 2^-20 of the reference,
// at steps of the largest size, lose bits: 2^-31 of it at most. All sums are fp32.
//
// Places that a row does not see may hold any step and lowest value, a NaN among them: their weights are set to 0, not multiplied. Codes are always numbers.
//
// One CTA per (sequence, tile of rows, key head, split), or (query row, key head, split) where blocks are selected; its four warps take the walk's pages in
// turn, kPages at a time, each through a private ring of bulk copies (a page of a head is 16 rows in one piece), so the main loop has no barrier.
//
// What bounds it (us from captured graphs): 64 decode rows of 4000 to 32,000 tokens, 32 query and 8 key heads of 128 (1.25 GB): 287, 4.4 TB/s, two thirds of
// what memory gives; all of 16,000: 229, 4.9 TB/s. Masks and shifts run at half the rate of other instructions and take 55 % of their pipe there, and twelve warps
// an SM hide their latency in part (products 27 %, shared memory 33 %). One row of 900 tokens: 8, a CTA's way in and out. 40 rows that read 96 blocks each: 25.
#include <limits.h>

#include <algorithm>
#include <type_traits>

#include "attention_span_rows.cuh"
#include "kv4.cuh"
#include "tma_host.h"

namespace fllm {
namespace {
constexpr int kNowhere = INT_MAX / 2;                    // token of a page that is not there
constexpr float kRefSlack = 8.f;                         // scores above their row's reference, to base 2
constexpr int kWeightLift = 6;                           // weights are below 2^(kRefSlack + 1), f16 holds 2^15

template <int D, int NB>
struct Kv4Smem {
  static constexpr int kRow = kKv4Row<D>, kPageBytes = kPage * kRow;
  // Pages of a turn of a warp. More of them share its maxima, votes and barriers and leave more to do while a result is waited for, fewer leave registers for
  // more CTAs (64 sequences of 4000 to 32,000 tokens, 8 key heads of 128: 4 and three CTAs an SM 291 us, 2 and four 302, 2 and three 323, 1 and four 355).
  static constexpr int kPages = D == 256 ? 1 : NB == 1 ? 4 : 2;
  static constexpr int kStages = D == 256 ? 3 : NB == 1 && D == 128 ? 2 : 3;
  static constexpr int kStage = 2 * kPages * kPageBytes; // K and V
  static constexpr int kRing = 4 * kStages * kStage;
  static constexpr int kMerge = 4 * kSpanRows * (D + 2) * 4 + kSpanRows * (D + 4) * 4;
  static constexpr int kQPitch = D * 2 + 16;             // bytes of a row of queries
  static constexpr int kQ = 8 * NB * kQPitch;
  static constexpr int kInfo = kSpanRows * (8 * kSpanWords + 4 * 4);
  static constexpr int kBars = 4 * kStages * 8 + 4 * kStages * kPages * 4 + 16;
  static constexpr int kBody = kQ + kRing > kMerge ? kQ + kRing : kMerge;     // the join takes the queries' and the ring's place
  static constexpr int kTotal = kInfo + (kBars + 15) / 16 * 16 + kBody + 128;
  static_assert(kPageBytes % 16 == 0 && kQ % 16 == 0 && kInfo % 16 == 0, "shared memory");
};
template <int D, int NB> constexpr int kv4_resident() { return D == 256 || NB == 2 ? 2 : 3; }

__device__ __forceinline__ float pow2_field(int field) { return __uint_as_float((uint32_t)field << 23); }
__device__ __forceinline__ uint32_t lds32(const uint8_t* p) { return *reinterpret_cast<const uint32_t*>(p); }
__device__ __forceinline__ void bulk_in(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes),
               "r"(smem_u32(bar)) : "memory");
}
// As mma_f16, free to be moved by the compiler; and the first product of a sum.
__device__ __forceinline__ void mma_add(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
// Which token of a page is row i of the products (0 to 7, and 8 more: + 4). Rows of a page lie 4 bytes next to a multiple of 32, so neighbouring rows share
// banks; in this order two of 32 lanes meet at most, for keys (a lane's rows i = lane / 4) and for values (i = 2 (lane % 4)).
__device__ __forceinline__ int token_of(int i) { return ((i >> 1) & 1) * 8 + (i >> 2) + (i & 1) * 2; }

template <int D, int NB, int MODE>
__global__ void __launch_bounds__(128, kv4_resident<D, NB>()) kv4_rows_kernel(const __grid_constant__ SpanParams p) {
  using S = Kv4Smem<D, NB>;
  constexpr int kPages = S::kPages, kStages = S::kStages, RB = S::kRow, W = D / 32;       // W: words of a key row that a lane takes
  constexpr uint32_t kLow = 0x000F000Fu, kHigh = 0x00F000F0u, kOnes = 0x3C003C00u;
  extern __shared__ __align__(128) uint8_t smem[];
  unsigned long long* bits = reinterpret_cast<unsigned long long*>(smem);                 // [16][4]
  int* bases = reinterpret_cast<int*>(bits + kSpanRows * kSpanWords);
  int* begs = bases + kSpanRows;
  float* factors = reinterpret_cast<float*>(begs + kSpanRows);                            // of a row's scores, to base 2
  float* qsums = factors + kSpanRows;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kInfo);                          // [4][kStages]
  int* page_tok = reinterpret_cast<int*>(bars + 4 * kStages);                             // [4][kStages][kPages] first token of a page that is on its way
  volatile int* abort_flag = reinterpret_cast<volatile int*>(page_tok + 4 * kStages * kPages);
  uint8_t* body = smem + S::kInfo + (S::kBars + 15) / 16 * 16;
  uint8_t *qtile = body, *ring = body + S::kQ;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int G = p.group;
  int work = blockIdx.x / p.splits;
  const int split = blockIdx.x - work * p.splits;
  const int kvh = work % p.hkv;
  work /= p.hkv;
  if (threadIdx.x < 4 * kStages) {
    mbar_init(bars + threadIdx.x, 1);
    fence_barrier_init();
  }
  if (threadIdx.x == 0) *abort_flag = 0;
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

  uint8_t* my_ring = ring + (size_t)warp * kStages * S::kStage;
  uint64_t* my_bars = bars + warp * kStages;
  int* my_tok = page_tok + warp * kStages * kPages;
  const int* table = p.block_tables + (size_t)seq * p.max_blocks;
  bool bad = false;
  // A warp's pages are kPages neighbours at a time. Their blocks are looked up 32 pages at a time, a lane to a page, ahead of their use.
  constexpr int kTurns = 32 / kPages;
  auto look = [&](int it, int& tok) {                    // first row in the pool, first token; -1 and kNowhere of a page that is not there
    const int pg = pg0 + (warp + 4 * (it + lane / kPages)) * kPages + lane % kPages;
    tok = kNowhere;
    if (pg >= pg1) return -1LL;
    const int page = range.piece(pg), block = span_block(p, table, page);
    bad |= block < 0;
    if (block < 0) return -1LL;
    tok = page * kPage;
    return span_pool_row(p, block, kvh, page) * RB;
  };
  int toks_now, toks_next;
  long long at_now, at_next = look(0, toks_next);
  const int my_turns = pg1 > pg0 + warp * kPages ? (pg1 - pg0 - warp * kPages + 4 * kPages - 1) / (4 * kPages) : 0;
  __syncthreads();                                       // the barriers are there
  int to = 0;                                            // stage of the next turn that is asked for
  auto issue = [&](int it) {
    if (it >= my_turns) return;
    if (it % kTurns == 0) { at_now = at_next; toks_now = toks_next; at_next = look(it + kTurns, toks_next); }
    const int h = lane - it % kTurns * kPages;
    const bool mine = (unsigned)h < (unsigned)kPages, there = mine && at_now >= 0;
    const unsigned asked = __ballot_sync(0xffffffffu, there);
    if (mine) my_tok[to * kPages + h] = toks_now;
    if (lane == 0) mbar_expect_tx(my_bars + to, __popc(asked) * 2 * S::kPageBytes);
    __syncwarp();
    if (there) {
      uint8_t* st = my_ring + to * S::kStage + h * 2 * S::kPageBytes;
      bulk_in(st, static_cast<const uint8_t*>(p.k_cache) + at_now, S::kPageBytes, my_bars + to);
      bulk_in(st + S::kPageBytes, static_cast<const uint8_t*>(p.v_cache) + at_now, S::kPageBytes, my_bars + to);
    }
    to = to + 1 == kStages ? 0 : to + 1;
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) issue(s);
  // Queries, 8 values to a thread, a row with D / 8 neighbouring threads. Of eight dims the pairs (0, 4), (1, 5), (2, 6), (3, 7) are a register each, as
  // the codes of a word are.
#pragma unroll
  for (int i = threadIdx.x; i < NB * 8 * (D / 8); i += 128) {
    const int r = i / (D / 8), c = i - r * (D / 8);
    uint4 v = make_uint4(0, 0, 0, 0);
    if (r < n_rows) {
      const int qi = (row0 + r) / G, hg = (row0 + r) - qi * G;
      v = *reinterpret_cast<const uint4*>(static_cast<const bf16*>(p.q) + (size_t)(q0 + qi) * p.ldq + (size_t)(kvh * G + hg) * D + c * 8);
    }
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t top = 0;                      // largest exponent field of the row, infinities and NaN aside
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t a = w[e] >> 7 & 0xFF, b = w[e] >> 23 & 0xFF;
      if (a != 0xFF) top = max(top, a);
      if (b != 0xFF) top = max(top, b);
    }
#pragma unroll
    for (int o = D / 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    const int up = min(127 + 14 - (int)top, 126);
    const float f = __uint_as_float((uint32_t)(127 + up) << 23);
    float x[8], sum = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 y = unpack_bf16x2(w[e]);
      x[2 * e] = y.x * f;
      x[2 * e + 1] = y.y * f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += x[e];
#pragma unroll
    for (int o = D / 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    *reinterpret_cast<uint4*>(qtile + r * S::kQPitch + c * 16) =
        make_uint4(pack_16<true>(x[0], x[4]), pack_16<true>(x[1] * 0.0625f, x[5] * 0.0625f), pack_16<true>(x[2], x[6]), pack_16<true>(x[3] * 0.0625f, x[7] * 0.0625f));
    if (c == 0) {
      factors[r] = fminf(span_factor(p.scale_log2, up) * 16777216.f, FLT_MAX);      // products are with c 2^-24; an infinity would make a NaN of a score of 0
      qsums[r] = sum * (1.f / 16777216.f);
    }
  }
  __syncthreads();
  uint32_t qf[NB][W][4];                   // columns g of the products; a lane's dims are those of its words of a key row, t + 4 i
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const uint4 v = *reinterpret_cast<const uint4*>(qtile + (8 * n + g) * S::kQPitch + (t + 4 * i) * 16);
      qf[n][i][0] = v.x; qf[n][i][1] = v.y; qf[n][i][2] = v.z; qf[n][i][3] = v.w;
    }
  // A lane's rows are 2t and 2t + 1 of each eight, its tokens rows g and g + 8 of the products.
  float fac[NB][2], qs[NB][2];
  int base[NB][2], beg[NB][2];
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = 8 * n + 2 * t + h;
      const bool in = r < n_rows;
      fac[n][h] = in ? factors[r] : 1.f; qs[n][h] = in ? qsums[r] : 0.f;
      base[n][h] = bases[r]; beg[n][h] = begs[r];
    }
  const int k_at = token_of(g) * RB, v_at = token_of(2 * t) * RB;

  float o[NB][D / 16][4], sum[NB][4];      // sum: of the operands of a row's weights, since it was taken off o
  float m[NB][2], ref[NB][2], l[NB][2], zs[NB][2];       // reference (0 as long as there is none), sum of weights, sum of weights times the middles of ranges
  int unit = 8;                            // U: exponent field that all steps are below, with some room
  float step_limit = pow2_field(unit + 1), of_step = pow2_field(2 * 127 + kWeightLift - unit);
#pragma unroll
  for (int n = 0; n < NB; ++n) {
#pragma unroll
    for (int i = 0; i < D / 16; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
    sum[n][0] = sum[n][1] = sum[n][2] = sum[n][3] = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) { m[n][h] = -INFINITY; ref[n][h] = l[n][h] = zs[n][h] = 0.f; }
  }
  // One turn: the pages at `st`. FULL: all rows see all of it, and there is no soft-cap.
  auto turn = [&](const uint8_t* st, const int* toks, auto full_turn) {
    constexpr bool FULL = decltype(full_turn)::value;
    float x[NB][kPages][4];
#pragma unroll
    for (int i = 0; i < W; ++i)
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int h = 0; h < kPages; ++h) {
          const uint8_t* row = st + h * 2 * S::kPageBytes + k_at + (t + 4 * i) * 4;
          const uint32_t a = lds32(row) >> 8 * k, b = lds32(row + 4 * RB) >> 8 * k;
          const uint32_t op[4] = {a & kLow, b & kLow, a & kHigh, b & kHigh};
#pragma unroll
          for (int n = 0; n < NB; ++n) {
            if (i == 0 && k == 0) mma_first(x[n][h], op, qf[n][0][0], qf[n][0][1]);
            else mma_add(x[n][h], op, qf[n][i][2 * k], qf[n][i][2 * k + 1]);
          }
        }
    Kv4Scale vs[kPages][2];                // of values, the middle of the range instead of its lowest value
#pragma unroll
    for (int h = 0; h < kPages; ++h) {
      const uint8_t* tail = st + h * 2 * S::kPageBytes + k_at + D / 2;
#pragma unroll
      for (int tk = 0; tk < 2; ++tk) {
        const Kv4Scale ks = kv4_scale_of(lds32(tail + 4 * tk * RB));
        vs[h][tk] = kv4_scale_of(lds32(tail + S::kPageBytes + 4 * tk * RB));
        vs[h][tk].low = fmaf(8.f, vs[h][tk].step, vs[h][tk].low);
        bool any = false;
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float v = fmaf(x[n][h][2 * tk + r], ks.step, ks.low * qs[n][r]) * fac[n][r];
            if constexpr (!FULL) {
              if (p.softcap > 0.f) v = p.softcap * tanhf(v / (p.softcap * kLog2e)) * kLog2e;
              const int tok = toks[h] + token_of(g) + 4 * tk;
              const bool sees = span_sees(p, tok, base[n][r], beg[n][r], bits + (8 * n + 2 * t + r) * kSpanWords);
              if (!sees) v = -INFINITY;
              any |= sees;
            }
            x[n][h][2 * tk + r] = v;
          }
        if constexpr (!FULL) {
          if (!any) vs[h][tk] = {0.f, 0.f};              // of a place that none of the lane's rows sees
        }
      }
    }
    float top[NB][2], steepest = fmaxf(fmaxf(0.f, vs[0][0].step), vs[0][1].step);      // largest scores and steps of a lane (a NaN is none)
#pragma unroll
    for (int h = 1; h < kPages; ++h) steepest = fmaxf(fmaxf(steepest, vs[h][0].step), vs[h][1].step);
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        top[n][r] = fmaxf(x[n][0][r], x[n][0][2 + r]);
#pragma unroll
        for (int h = 1; h < kPages; ++h) top[n][r] = fmaxf(fmaxf(top[n][r], x[n][h][r]), x[n][h][2 + r]);
      }
    bool more = steepest >= step_limit;    // a score or a step is out of reach of its reference
#pragma unroll
    for (int n = 0; n < NB; ++n) more |= top[n][0] > m[n][0] + kRefSlack || top[n][1] > m[n][1] + kRefSlack;
    if (__any_sync(0xffffffffu, more)) {
      const int field = __reduce_max_sync(0xffffffffu, (int)(__float_as_uint(steepest) >> 23)), was = unit;
      if (field > unit) unit = min(field + 2, 254);
      const float shrink = unit == was ? 1.f : pow2_field(max(127 + was - unit, 0));
      step_limit = unit == 254 ? INFINITY : pow2_field(unit + 1);
      of_step = pow2_field(2 * 127 + kWeightLift - unit);
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float mx = top[n][r];
#pragma unroll
          for (int d = 4; d <= 16; d *= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
          const float mn = fmaxf(m[n][r], mx);
          const float c = mn == -INFINITY ? 1.f : ex2(m[n][r] - mn);
          m[n][r] = mn;
          ref[n][r] = mn == -INFINITY ? 0.f : mn;
          l[n][r] *= c;
          zs[n][r] *= c;
#pragma unroll
          for (int i = 0; i < D / 16; ++i) { o[n][i][r] *= c * shrink; o[n][i][2 + r] *= c * shrink; }
          sum[n][r] *= c * shrink;
        }
    }
    uint32_t pt[NB][kPages][2];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
#pragma unroll
      for (int h = 0; h < kPages; ++h)
#pragma unroll
        for (int tk = 0; tk < 2; ++tk) {
          float w[2];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float v = x[n][h][2 * tk + r], e = ex2(v - ref[n][r]);
            l[n][r] += e;
            w[r] = e * (vs[h][tk].step * of_step);
            if constexpr (FULL) {
              zs[n][r] = fmaf(e, vs[h][tk].low, zs[n][r]);
            } else {
              if (v == -INFINITY) w[r] = 0.f;
              else zs[n][r] = fmaf(e, vs[h][tk].low, zs[n][r]);
            }
          }
          pt[n][h][tk] = transposed(pack_16<true>(w[0], w[1]));
        }
    }
#pragma unroll
    for (int h = 0; h < kPages; ++h)
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        const uint32_t ones[4] = {kOnes, kOnes, kOnes, kOnes};
        mma_add(sum[n], ones, pt[n][h][0], pt[n][h][1]);
      }
#pragma unroll
    for (int h = 0; h < kPages; ++h)
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        const uint8_t* row = st + h * 2 * S::kPageBytes + S::kPageBytes + v_at + (g + 8 * i) * 4;
        const uint32_t w0 = lds32(row), w1 = lds32(row + 2 * RB), w2 = lds32(row + 4 * RB), w3 = lds32(row + 6 * RB);
        uint32_t a = __byte_perm(w0, w1, 0x5410), b = __byte_perm(w0, w1, 0x7632), c = __byte_perm(w2, w3, 0x5410), d = __byte_perm(w2, w3, 0x7632);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t even[4] = {a & kLow, b & kLow, c & kLow, d & kLow}, odd[4] = {a & kHigh, b & kHigh, c & kHigh, d & kHigh};
#pragma unroll
          for (int n = 0; n < NB; ++n) {
            mma_add(o[n][4 * i + 2 * k], even, pt[n][h][0], pt[n][h][1]);
            mma_add(o[n][4 * i + 2 * k + 1], odd, pt[n][h][0], pt[n][h][1]);
          }
          a >>= 8; b >>= 8; c >>= 8; d >>= 8;
        }
      }
  };
  // Sums of codes become sums of codes from the middle of their range.
  auto centre = [&] {
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          const float unit8 = 8.f / (i & 1 ? 1 << 20 : 1 << 24);
          o[n][i][r] = fmaf(sum[n][r], -unit8, o[n][i][r]);
          o[n][i][2 + r] = fmaf(sum[n][r], -unit8, o[n][i][2 + r]);
        }
        sum[n][r] = 0.f;
      }
  };
  bool ok = true;
  int it = 0, from = 0, phase = 0;
  for (; it < my_turns; ++it) {
    issue(it + kStages - 1);
    if (!mbar_wait_warp(my_bars + from, phase, abort_flag)) { ok = false; break; }
    const uint8_t* st = my_ring + from * S::kStage;
    int toks[kPages];
    bool full = p.softcap <= 0.f;
#pragma unroll
    for (int h = 0; h < kPages; ++h) {
      toks[h] = my_tok[from * kPages + h];
      full = full && toks[h] + kPage <= min_base && (toks[h] >= max_beg || toks[h] + kPage <= p.first);
    }
    if (full) turn(st, toks, std::true_type{});
    else turn(st, toks, std::false_type{});
    if ((it & 7) == 7) centre();
    __syncwarp();                          // the stage is free
    if (++from == kStages) { from = 0; phase ^= 1; }
  }
  centre();
  if (!ok) {                               // copies that are on their way land before the memory is another CTA's
    for (int k = 1; k < kStages; ++k)
      if (it + k < my_turns) {
        int none = 0;
        mbar_wait_warp(my_bars + (it + k) % kStages, ((it + k) / kStages) & 1, &none);
      }
    if (lane == 0 && p.status) atomicCAS(p.status, FLLM_OK, FLLM_ERR_MBAR_TIMEOUT);
  }
  if (bad && p.status) atomicCAS(p.status, FLLM_OK, FLLM_ERR_BAD_ARGS);

  __syncthreads();                         // queries and ring are free
  float* mo = reinterpret_cast<float*>(body);            // [4][16][D]
  float* mml = mo + 4 * kSpanRows * D;                   // [4][16][2]
  float* part_o = mml + 4 * kSpanRows * 2;               // [16][D]: the CTA's
  float4* part_ml = reinterpret_cast<float4*>(part_o + kSpanRows * D);      // [16]
  // of a row's dims a lane has 8 (g + 8 i) + 0 to 7; products were with c 2^-24 (2^-20 of odd dims), weights times 2^(kWeightLift + 127 - unit)
  const float back = pow2_field(unit), even = (float)(1 << (24 - kWeightLift)), odd = even * 0.0625f;
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
#pragma unroll
      for (int d = 4; d <= 16; d *= 2) {
        l[n][r] += __shfl_xor_sync(0xffffffffu, l[n][r], d);
        zs[n][r] += __shfl_xor_sync(0xffffffffu, zs[n][r], d);
      }
      const int at = warp * kSpanRows + 8 * n + 2 * t + r;
      float* row = mo + (size_t)at * D;
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[j] = fmaf(o[n][4 * i + j][r] * (j & 1 ? odd : even), back, zs[n][r]);
          v[4 + j] = fmaf(o[n][4 * i + j][2 + r] * (j & 1 ? odd : even), back, zs[n][r]);
        }
        *reinterpret_cast<float4*>(row + 8 * (g + 8 * i)) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(row + 8 * (g + 8 * i) + 4) = make_float4(v[4], v[5], v[6], v[7]);
      }
      if (g == 0) *reinterpret_cast<float2*>(mml + at * 2) = make_float2(m[n][r], l[n][r]);
    }
  span_join<D>(p, mo, mml, part_o, part_ml, q0, row0, n_rows, kvh, split);
}

bool kv4_few(const SpanParams& p) { return p.picks ? p.group <= 8 : std::min<long long>((long long)p.max_q_len * p.group, p.rows_to) <= 8; }
template <int D, int NB>
void launch_rows(SpanParams p, cudaStream_t s) {
  constexpr int smem = Kv4Smem<D, NB>::kTotal;
  static_assert((smem + 1024) * kv4_resident<D, NB>() <= 228 * 1024, "shared memory");
  static bool configured[kMaxDevices] = {};
  if (first_call_on_device(configured)) {
    cuda_check(cudaFuncSetAttribute(kv4_rows_kernel<D, NB, kAsked>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), "kv4_rows smem");
    cuda_check(cudaFuncSetAttribute(kv4_rows_kernel<D, NB, kSearch>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), "kv4_rows smem");
    cuda_check(cudaFuncSetAttribute(kv4_rows_kernel<D, NB, kPicked>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), "kv4_rows smem");
  }
  const long long ctas = span_rows_ctas(p) * p.splits;
  if (ctas > INT_MAX) throw std::runtime_error("attention: too many query rows");
  auto go = [&](auto kernel) {
    if (p.in_cluster) launch_cluster(true, kernel, dim3((unsigned)ctas), dim3(128), smem, s, (unsigned)p.splits, p);
    else launch_pdl(kernel, dim3((unsigned)ctas), dim3(128), smem, s, p);
  };
  if (p.picks) go(kv4_rows_kernel<D, NB, kPicked>);
  else if (p.search) go(kv4_rows_kernel<D, NB, kSearch>);
  else go(kv4_rows_kernel<D, NB, kAsked>);
}
}  // namespace

int attention_kv4_resident(const SpanParams& p) {
  if (p.head_dim == 256) return kv4_resident<256, 1>();
  return kv4_few(p) ? kv4_resident<128, 1>() : kv4_resident<128, 2>();
}
void attention_kv4_rows(const SpanParams& p, cudaStream_t s) {
  const bool few = kv4_few(p);
  switch (p.head_dim) {
    case 64: few ? launch_rows<64, 1>(p, s) : launch_rows<64, 2>(p, s); break;
    case 128: few ? launch_rows<128, 1>(p, s) : launch_rows<128, 2>(p, s); break;
    default: few ? launch_rows<256, 1>(p, s) : launch_rows<256, 2>(p, s); break;
  }
}
}  // namespace fllm
