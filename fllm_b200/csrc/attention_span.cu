// Attention over a paged cache under a window behind which the first tokens stay visible, and for the nodes of draft trees: the kernel of
// sequences with few packed rows (query row x head of a key head), the merge of split sequences, and the choice between the kernels.
//
//   o_r = sum_j e^(s_rj - m_r) v_j / (sum_j e^(s_rj - m_r) [+ e^(sink - m_r)]),  s_rj = scale q_r . k_j,  j over what row r sees
//
// (attention_span.cuh says what that is; a row that sees nothing is 0.) One CTA per (sequence, 16 packed rows, key head, split). Its four
// warps take the 16-token pages that the rows see between them in turn: the first tokens' pages and the window's, nothing in between. Each
// streams its pages through a private cp.async ring, so the main loop has no barrier; (m, l, O) of the warps are joined in shared memory,
// those of the splits by span_merge_kernel. Sequences with more than 16 packed rows go to attention_span_tc.cu where that has a kernel.
//
// Scores and sums are fp32. Weights are rounded to the operands' 16 bits for the product with the values (bf16, at most 2^-9 each and of
// either sign; f16 beside an e4m3 cache). An e4m3 cache is widened to f16, which holds all of its values; queries are f16 there as well, times a
// power of two per row that puts the row's largest magnitude between 2^14 and 2^15: what a bf16 value loses is below 2^-38 of that magnitude.
//
// Values in places that a row does not see may be anything: a weight of zero times a NaN would be a NaN, so in pages that not every row
// sees whole, infinities and NaN of V are taken out of the tile in front of the product and added to the rows that see them.
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <limits.h>

#include <algorithm>

#include "attention_span.cuh"
#include "attention_util.cuh"
#include "tma_host.h"

namespace fllm {
namespace {
constexpr int kSpanRows = 16;
// Weights in f16 are taken to a reference 2^12 below the row's maximum: below 2^-14 of their unit they would lose bits.
constexpr float kF16Lift = 12.f;

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool F16>
__device__ __forceinline__ void mma_16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (F16) mma_f16(d, a, b0, b1);
  else mma_bf16(d, a, b0, b1);
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
template <bool F16>
__device__ __forceinline__ float2 unpack_16(uint32_t w) {
  if constexpr (F16) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  else return unpack_bf16x2(w);
}
template <bool F16>
__device__ __forceinline__ bool odd_16x2(uint32_t w) {
  if constexpr (F16) return odd_f16x2(w);
  else return odd_bf16x2(w);
}
__device__ __forceinline__ void cp_async16_or_zero(void* smem, const void* gmem, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(smem)), "l"(gmem), "r"(there ? 16 : 0) : "memory");
}

template <int D, bool KV8>
struct RowsSmem {
  static constexpr int kStages = D == 256 && !KV8 ? 2 : 3;
  static constexpr int kPageElems = kPage * D;
  static constexpr int kPageBytes = kPageElems * (KV8 ? 1 : 2);          // a K or V page as it arrives
  static constexpr int kWarpRing = kStages * 2 * kPageBytes;
  static constexpr int kWarpTiles = KV8 ? 2 * kPageElems * 2 : 0;        // widened pages
  static constexpr int kRing = 4 * (kWarpRing + kWarpTiles);
  static constexpr int kMerge = 4 * kSpanRows * (D + 2) * 4;
  static constexpr int kQ = kSpanRows * D * 2;
  static constexpr int kInfo = kSpanRows * (8 * kSpanWords + 4 * 3);
  static constexpr int kTotal = kQ + kInfo + (kRing > kMerge ? kRing : kMerge) + 128;
};

template <int D, bool KV8>
__global__ void __launch_bounds__(128) span_rows_kernel(const __grid_constant__ SpanParams p) {
  using S = RowsSmem<D, KV8>;
  extern __shared__ __align__(128) uint8_t smem[];
  bf16* qtile = reinterpret_cast<bf16*>(smem);
  unsigned long long* bits = reinterpret_cast<unsigned long long*>(smem + S::kQ);      // [16][4]
  int* bases = reinterpret_cast<int*>(bits + kSpanRows * kSpanWords);
  int* begs = bases + kSpanRows;
  float* factors = reinterpret_cast<float*>(begs + kSpanRows);                         // of a row's scores, to base 2
  uint8_t* ring = smem + S::kQ + S::kInfo;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = p.group, split = blockIdx.y;
  const int work = blockIdx.x / p.hkv, kvh = blockIdx.x - work * p.hkv;
  const int seq = work % p.num_seqs, tile = work / p.num_seqs;
  pdl_launch_dependents();
  pdl_wait();
  const int q0 = p.q_starts[seq], qn = p.q_starts[seq + 1] - q0;
  const int all_rows = qn * G, row0 = tile * kSpanRows;
  if (qn <= 0 || all_rows <= p.rows_from || all_rows > p.rows_to || row0 >= all_rows) return;
  if (q0 < 0 || q0 + qn > p.tokens) {
    if (threadIdx.x == 0 && p.status) atomicCAS(p.status, FLLM_OK, FLLM_ERR_BAD_ARGS);
    return;
  }
  const int n_rows = min(kSpanRows, all_rows - row0);
  const int kv_len = max(p.kv_lens[seq], 0);

  if (threadIdx.x < kSpanRows) {
    SpanRow r{0, 0};
    unsigned long long* mine = bits + threadIdx.x * kSpanWords;
    for (int w = 0; w < kSpanWords; ++w) mine[w] = 0;
    if (threadIdx.x < n_rows) r = span_row(p, q0, qn, kv_len, (row0 + threadIdx.x) / G, mine);
    bases[threadIdx.x] = r.base;
    begs[threadIdx.x] = r.beg;
  }
  // queries; a row's 16-byte pieces lie with D / 8 neighbouring threads
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
      const int up = top ? min(max(127 + 14 - (int)top, -100), 100) : 0;
      const float f = __uint_as_float((uint32_t)(127 + up) << 23);
      factor *= __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 x = unpack_bf16x2(w[e]);
        w[e] = pack_16<true>(x.x * f, x.y * f);
      }
    }
    if (c == 0) factors[r] = factor;
    *reinterpret_cast<uint4*>(tile_ptr<D>(qtile, r, c)) = v;
  }
  __syncthreads();
  uint32_t qf[D / 16][4];
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) ldsm_x4(qf[kk], tile_ptr<D>(qtile, lane & 15, 2 * kk + (lane >> 4)));

  // what the tile's rows see between them, and what all of them see
  int min_base = INT_MAX, max_base = 0, min_beg = INT_MAX, max_beg = 0;
  if (lane < n_rows) { min_base = max_base = bases[lane]; min_beg = max_beg = begs[lane]; }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) {
    min_base = min(min_base, __shfl_xor_sync(0xffffffffu, min_base, o));
    max_base = max(max_base, __shfl_xor_sync(0xffffffffu, max_base, o));
    min_beg = min(min_beg, __shfl_xor_sync(0xffffffffu, min_beg, o));
    max_beg = max(max_beg, __shfl_xor_sync(0xffffffffu, max_beg, o));
  }
  min_base = __shfl_sync(0xffffffffu, min_base, 0);
  max_base = __shfl_sync(0xffffffffu, max_base, 0);
  min_beg = __shfl_sync(0xffffffffu, min_beg, 0);
  max_beg = __shfl_sync(0xffffffffu, max_beg, 0);
  const SpanRange range = span_range(p, kPage, min_beg, p.tree_mask ? kv_len : max_base);
  const int per_split = max(p.min_pages, (range.count + p.splits - 1) / p.splits);
  const int pg0 = min(split * per_split, range.count), pg1 = min(pg0 + per_split, range.count);

  const int g = lane >> 2;
  const int base0 = bases[g], base1 = bases[g + 8], beg0 = begs[g], beg1 = begs[g + 8];
  const float f0 = factors[g], f1 = factors[g + 8];
  const unsigned long long *bits0 = bits + g * kSpanWords, *bits1 = bits + (g + 8) * kSpanWords;

  float o[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

  uint8_t* my_ring = ring + (size_t)warp * (S::kWarpRing + S::kWarpTiles);
  bf16* my_tiles = reinterpret_cast<bf16*>(my_ring + S::kWarpRing);
  const int* table = p.block_tables + (size_t)seq * p.max_blocks;
  bool bad = false;
  auto issue = [&](int it) {
    const int pg = pg0 + warp + 4 * it;
    if (pg < pg1) {
      const int page = range.piece(pg);
      const int block = span_block(p, table, page);
      bad |= block < 0;
      const long long off = block < 0 ? 0 : span_pool_row(p, block, kvh, page) * D;
      uint8_t* st = my_ring + (size_t)(it % S::kStages) * 2 * S::kPageBytes;
      if constexpr (KV8) {
        const uint8_t *kg = static_cast<const uint8_t*>(p.k_cache) + off, *vg = static_cast<const uint8_t*>(p.v_cache) + off;
        for (int i = lane; i < S::kPageBytes / 16; i += 32) {
          cp_async16_or_zero(st + i * 16, kg + i * 16, block >= 0);
          cp_async16_or_zero(st + S::kPageBytes + i * 16, vg + i * 16, block >= 0);
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
#pragma unroll
  for (int s = 0; s < S::kStages - 1; ++s) issue(s);
  for (int it = 0; it < my_pages; ++it) {
    issue(it + S::kStages - 1);
    cp_async_wait<S::kStages - 1>();
    __syncwarp();
    uint8_t* st = my_ring + (size_t)(it % S::kStages) * 2 * S::kPageBytes;
    bf16 *ks = reinterpret_cast<bf16*>(st), *vs = ks + S::kPageElems;
    if constexpr (KV8) {
      ks = my_tiles;
      vs = my_tiles + S::kPageElems;
      constexpr int CPR = D / 16;
      for (int i = lane; i < 2 * kPage * CPR; i += 32) {
        const int which = i / (kPage * CPR), c16 = i - which * (kPage * CPR);
        const int r = c16 / CPR, cc = c16 - r * CPR;
        const uint4 raw = *reinterpret_cast<const uint4*>(st + which * S::kPageBytes + r * D + cc * 16);
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
        uint32_t h[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const __half2_raw lo = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[e] & 0xFFFFu), __NV_E4M3);
          const __half2_raw hi = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[e] >> 16), __NV_E4M3);
          h[2 * e] = (uint32_t)lo.x | ((uint32_t)lo.y << 16);
          h[2 * e + 1] = (uint32_t)hi.x | ((uint32_t)hi.y << 16);
        }
        bf16* t = which ? vs : ks;
        *reinterpret_cast<uint4*>(tile_ptr<D>(t, r, 2 * cc)) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4*>(tile_ptr<D>(t, r, 2 * cc + 1)) = make_uint4(h[4], h[5], h[6], h[7]);
      }
      __syncwarp();
    }
    const int tok0 = range.piece(pg0 + warp + 4 * it) * kPage;
    const bool full = tok0 + kPage <= min_base && (tok0 >= max_beg || tok0 + kPage <= p.first);
    float s[2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
    const int j = lane >> 3, t = lane & 3;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      uint32_t b[4];
      ldsm_x4(b, tile_ptr<D>(ks, (j >> 1) * 8 + (lane & 7), 2 * kk + (j & 1)));
      mma_16<KV8>(s[0], qf[kk], b[0], b[1]);
      mma_16<KV8>(s[1], qf[kk], b[2], b[3]);
    }
    float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
    for (int nb = 0; nb < 2; ++nb) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float v = s[nb][e] * (e >= 2 ? f1 : f0);
        if (p.softcap > 0.f) v = p.softcap * tanhf(v / (p.softcap * kLog2e)) * kLog2e;
        if (!full) {
          const int tok = tok0 + nb * 8 + 2 * t + (e & 1);
          if (!(e >= 2 ? span_sees(p, tok, base1, beg1, bits1) : span_sees(p, tok, base0, beg0, bits0))) v = -INFINITY;
        }
        s[nb][e] = v;
        if (e >= 2) mx1 = fmaxf(mx1, v);
        else mx0 = fmaxf(mx0, v);
      }
    }
    mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1));
    mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
    mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1));
    mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
    const float mn0 = fmaxf(m[0], mx0), mn1 = fmaxf(m[1], mx1);
    const float c0 = mn0 == -INFINITY ? 1.f : ex2(m[0] - mn0), c1 = mn1 == -INFINITY ? 1.f : ex2(m[1] - mn1);
    constexpr float lift = KV8 ? kF16Lift : 0.f;
    const float r0 = mn0 == -INFINITY ? 0.f : mn0 - lift, r1 = mn1 == -INFINITY ? 0.f : mn1 - lift;
    uint32_t pf[4];
    float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
    for (int nb = 0; nb < 2; ++nb) {
      const float p0 = ex2(s[nb][0] - r0), p1 = ex2(s[nb][1] - r0), p2 = ex2(s[nb][2] - r1), p3 = ex2(s[nb][3] - r1);
      sum0 += p0 + p1;
      sum1 += p2 + p3;
      pf[2 * nb] = pack_16<KV8>(p0, p1);
      pf[2 * nb + 1] = pack_16<KV8>(p2, p3);
    }
    l[0] = l[0] * c0 + sum0;
    l[1] = l[1] * c1 + sum1;
    m[0] = mn0;
    m[1] = mn1;
#pragma unroll
    for (int db = 0; db < D / 8; ++db) {
      o[db][0] *= c0; o[db][1] *= c0;
      o[db][2] *= c1; o[db][3] *= c1;
    }
    if (!full) {
      uint32_t* vw = reinterpret_cast<uint32_t*>(vs);
      bool odd = false;
#pragma unroll 4
      for (int i = lane; i < kPage * D / 2; i += 32) odd |= odd_16x2<KV8>(vw[i]);
      if (__any_sync(0xffffffffu, odd)) {
        for (int tk = 0; tk < kPage; ++tk) {
          const int src = (lane & ~3) | (tk & 7) >> 1;
          const float2 a = unpack_16<KV8>(__shfl_sync(0xffffffffu, tk < 8 ? pf[0] : pf[2], src));
          const float2 b = unpack_16<KV8>(__shfl_sync(0xffffffffu, tk < 8 ? pf[1] : pf[3], src));
          const float w0 = tk & 1 ? a.y : a.x, w1 = tk & 1 ? b.y : b.x;
          const bool sees0 = span_sees(p, tok0 + tk, base0, beg0, bits0), sees1 = span_sees(p, tok0 + tk, base1, beg1, bits1);
#pragma unroll
          for (int db = 0; db < D / 8; ++db) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(tile_ptr<D>(vs, tk, db) + 2 * t);
            if (odd_16x2<KV8>(w)) {
              const float2 v = unpack_16<KV8>(w);
              if (!isfinite(v.x)) { if (sees0) o[db][0] += w0 * v.x; if (sees1) o[db][2] += w1 * v.x; }
              if (!isfinite(v.y)) { if (sees0) o[db][1] += w0 * v.y; if (sees1) o[db][3] += w1 * v.y; }
            }
          }
        }
        __syncwarp();
        for (int i = lane; i < kPage * D / 2; i += 32) {
          const uint32_t w = vw[i];
          if (odd_16x2<KV8>(w)) vw[i] = (odd_16x2<KV8>(w & 0xFFFFu) ? 0u : w & 0xFFFFu) | (odd_16x2<KV8>(w & 0xFFFF0000u) ? 0u : w & 0xFFFF0000u);
        }
        __syncwarp();
      }
    }
#pragma unroll
    for (int db = 0; db < D / 8; db += 2) {
      uint32_t b[4];
      ldsm_x4_t(b, tile_ptr<D>(vs, (j & 1) * 8 + (lane & 7), db + (j >> 1)));
      mma_16<KV8>(o[db], pf, b[0], b[1]);
      mma_16<KV8>(o[db + 1], pf, b[2], b[3]);
    }
    __syncwarp();
  }
  cp_async_wait<0>();
  if (bad && p.status) atomicCAS(p.status, FLLM_OK, FLLM_ERR_BAD_ARGS);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
  }

  if constexpr (KV8) { m[0] -= kF16Lift; m[1] -= kF16Lift; }

  __syncthreads();                                     // the ring is free
  float* mo = reinterpret_cast<float*>(ring);          // [4][16][D]
  float* mml = mo + 4 * kSpanRows * D;                 // [4][16][2]
  const int t4 = lane & 3;
#pragma unroll
  for (int db = 0; db < D / 8; ++db) {
    *reinterpret_cast<float2*>(mo + ((size_t)warp * 16 + g) * D + db * 8 + 2 * t4) = make_float2(o[db][0], o[db][1]);
    *reinterpret_cast<float2*>(mo + ((size_t)warp * 16 + g + 8) * D + db * 8 + 2 * t4) = make_float2(o[db][2], o[db][3]);
  }
  if (t4 == 0) {
    *reinterpret_cast<float2*>(mml + (warp * 16 + g) * 2) = make_float2(m[0], l[0]);
    *reinterpret_cast<float2*>(mml + (warp * 16 + g + 8) * 2) = make_float2(m[1], l[1]);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n_rows * (D / 2); i += 128) {
    const int r = i / (D / 2), d2 = (i - r * (D / 2)) * 2;
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) mm = fmaxf(mm, mml[(w * 16 + r) * 2]);
    float ll = 0.f, a0 = 0.f, a1 = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float mw = mml[(w * 16 + r) * 2];
      const float c = mw == -INFINITY ? (mm == -INFINITY ? 1.f : 0.f) : ex2(mw - mm);
      const float2 v = *reinterpret_cast<const float2*>(mo + ((size_t)w * 16 + r) * D + d2);
      ll += mml[(w * 16 + r) * 2 + 1] * c;
      if (c != 0.f) { a0 += v.x * c; a1 += v.y * c; }
    }
    const int qi = (row0 + r) / G, head = kvh * G + (row0 + r) - qi * G;
    const size_t tok = (size_t)(q0 + qi);
    if (p.splits == 1) {
      if (p.sinks) {
        const float sk = p.sinks[head] * kLog2e;
        const float mn = fmaxf(mm, sk);
        const float c = mm == -INFINITY ? 0.f : ex2(mm - mn);
        ll = ll * c + ex2(sk - mn);
        a0 *= c;
        a1 *= c;
      }
      const float inv = ll == 0.f ? 0.f : 1.f / ll;
      *reinterpret_cast<uint32_t*>(static_cast<bf16*>(p.out) + tok * p.ldo + (size_t)head * D + d2) = pack_bf16x2(a0 * inv, a1 * inv);
    } else {
      const size_t at = (tok * p.hq + head) * p.splits + split;
      *reinterpret_cast<float2*>(p.ws_o + at * D + d2) = make_float2(a0, a1);
      if (d2 == 0) *reinterpret_cast<float2*>(p.ws_ml + at * 2) = make_float2(mm, ll);
    }
  }
}

// Joins the splits of a row: one warp per (token, head). `some`: only sequences of p.rows_from < packed rows <= p.rows_to were split.
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
    if (rows <= p.rows_from || rows > p.rows_to) return;
  }
  const float2* ml = reinterpret_cast<const float2*>(p.ws_ml) + (size_t)pair * p.splits;
  const float* part = p.ws_o + (size_t)pair * p.splits * D + lane;
  float2 mine = lane < p.splits ? __ldcg(ml + lane) : make_float2(-INFINITY, 0.f);
  if (__shfl_sync(0xffffffffu, mine.y, 0) < 0.f) return;      // the row was not split
  const float sk = p.sinks ? p.sinks[head] * kLog2e : -INFINITY;
  float mm = mine.x;
  for (int s = lane + 32; s < p.splits; s += 32) mm = fmaxf(mm, __ldcg(ml + s).x);
  mm = fmaxf(warp_max(mm), sk);
  float ll = 0.f, a[D / 32];
#pragma unroll
  for (int e = 0; e < D / 32; ++e) a[e] = 0.f;
  for (int s0 = 0; s0 < p.splits; s0 += 32) {
    if (s0) mine = s0 + lane < p.splits ? __ldcg(ml + s0 + lane) : make_float2(-INFINITY, 0.f);
    const float w = mine.x == -INFINITY ? (mm == -INFINITY && mine.y != 0.f ? 1.f : 0.f) : ex2(mine.x - mm);
    ll += mine.y * w;
    unsigned live = __ballot_sync(0xffffffffu, w != 0.f);     // (of the others there are no rows)
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
  ll = warp_sum(ll) + (p.sinks ? ex2(sk - mm) : 0.f);
  const float inv = ll == 0.f ? 0.f : 1.f / ll;
  bf16* dst = static_cast<bf16*>(p.out) + (size_t)tok * p.ldo + (size_t)head * D + lane;
#pragma unroll
  for (int e = 0; e < D / 32; ++e) dst[32 * e] = __float2bfloat16(a[e] * inv);
}

template <int D, bool KV8>
void launch_rows(const SpanParams& p, cudaStream_t s) {
  static bool configured[kMaxDevices] = {};
  if (first_call_on_device(configured))
    cuda_check(cudaFuncSetAttribute(span_rows_kernel<D, KV8>, cudaFuncAttributeMaxDynamicSharedMemorySize, RowsSmem<D, KV8>::kTotal), "span_rows smem");
  const long long most = (long long)p.max_q_len * p.group < p.rows_to ? (long long)p.max_q_len * p.group : p.rows_to;
  const long long tiles = (most + kSpanRows - 1) / kSpanRows;
  const long long ctas = tiles * p.num_seqs * p.hkv;
  if (ctas > INT_MAX) throw std::runtime_error("attention_span: too many query rows");
  launch_pdl(span_rows_kernel<D, KV8>, dim3((unsigned)ctas, p.splits), dim3(128), RowsSmem<D, KV8>::kTotal, s, p);
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

SpanPlan attention_span_plan(const SpanParams& p) {
  SpanPlan plan{};
  const bool tc = attention_span_tc_supported(p);
  const long long most = (long long)p.max_q_len * p.group;
  const long long span = std::min<long long>(p.window > 0 ? (long long)p.window + p.first + p.max_q_len : p.max_kv_len, p.max_kv_len);
  if (!tc || (long long)p.min_q_len * p.group <= kSpanRows) {
    const long long ctas = ((tc ? std::min<long long>(most, kSpanRows) : most) + kSpanRows - 1) / kSpanRows * p.num_seqs * p.hkv;
    const long long pages = (span + kPage - 1) / kPage;
    plan.min_pages = 8;
    long long splits = 1;
    if (ctas < 4 * sm_count()) splits = std::min<long long>((4LL * sm_count() + ctas - 1) / ctas, (pages + plan.min_pages - 1) / plan.min_pages);
    plan.rows_splits = (int)std::max<long long>(1, std::min<long long>(splits, 128));
  }
  if (tc && most > kSpanRows) {
    // at most four places for a piece to each SM: those that the kernel finds no work for cost a start all the same
    const long long ctas = (most + 255) / 256 * p.num_seqs * p.hkv, tiles = (span + 127) / 128 + 2;
    plan.tile_splits = (int)std::max<long long>(1, std::min<long long>(std::min<long long>(4LL * sm_count() / ctas, tiles), 32));
  }
  plan.bytes = (partial_floats(p, plan.rows_splits) + partial_floats(p, plan.tile_splits)) * sizeof(float);
  return plan;
}

int attention_span(SpanParams p, const SpanPlan& plan, void* workspace, cudaStream_t s) {
  int n = 0;
  const bool both = plan.rows_splits > 0 && plan.tile_splits > 0;
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
    p.rows_from = kSpanRows;
    p.rows_to = INT_MAX;
    attention_span_tc(p, s);
    ++n;
    if (p.splits > 1) { merge(p, both, s); ++n; }
  }
  if (plan.rows_splits > 0) {
    take(plan.rows_splits);
    p.rows_from = 0;
    p.rows_to = attention_span_tc_supported(p) ? kSpanRows : INT_MAX;
    switch (p.head_dim) {
      case 64: p.kv_fp8 ? launch_rows<64, true>(p, s) : launch_rows<64, false>(p, s); break;
      case 128: p.kv_fp8 ? launch_rows<128, true>(p, s) : launch_rows<128, false>(p, s); break;
      default: p.kv_fp8 ? launch_rows<256, true>(p, s) : launch_rows<256, false>(p, s); break;
    }
    ++n;
    if (p.splits > 1) { merge(p, both, s); ++n; }
  }
  cuda_check(cudaGetLastError(), "attention_span launch");
  return n;
}
}  // namespace fllm
