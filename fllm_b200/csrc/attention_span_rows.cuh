// What the kernels of sequences with few packed rows (attention_span.cu, attention_kv4.cu) share: products of f16 operands, the transposition of
// weights, the join of a CTA's four warps and of the splits that are a cluster.
#pragma once
#include <cuda_fp16.h>

#include "attention_span.cuh"
#include "attention_util.cuh"

namespace fllm {
namespace {
constexpr int kSpanRows = 16;              // packed rows of a CTA
constexpr int kAsked = 0, kSearch = 1, kPicked = 2;      // whose rows a CTA's are: as its place says, looked up, one row's that reads selected blocks

// Rows [row0, row0 + n_rows) of the qn x group packed rows of sequence `seq` are this CTA's; false: none are. The same for all splits, which are a cluster where
// they join in one: all of them leave, or none.
template <int MODE>
__device__ __forceinline__ bool span_rows_of_cta(const SpanParams& p, int work, int split, int& seq, int& row0, int& n_rows, int& q0, int& qn, int& kv_len) {
  const int G = p.group;
  if constexpr (MODE == kPicked) {
    const int tiles = (G + kSpanRows - 1) / kSpanRows, row = work / tiles, tile = work - row * tiles;
    if (!span_seq_of(p, row, seq) || !span_lengths(p, seq, threadIdx.x == 0, q0, qn, kv_len) || row - q0 >= qn) return false;
    row0 = (row - q0) * G + tile * kSpanRows;
    n_rows = min(kSpanRows, G - tile * kSpanRows);
    return true;
  }
  seq = work % p.num_seqs;
  int tile = work / p.num_seqs;
  if constexpr (MODE == kSearch) {
    if (!span_find(p, kSpanRows, 0, p.rows_to, work, blockIdx.x == gridDim.x - 1, seq, tile)) return false;
  }
  if (!span_lengths(p, seq, threadIdx.x == 0, q0, qn, kv_len)) return false;
  const int all_rows = qn * G;
  row0 = tile * kSpanRows;
  if (all_rows > p.rows_to || row0 >= all_rows) return false;
  n_rows = min(kSpanRows, all_rows - row0);
  return true;
}

// The pages that a CTA's rows see between them, in the order of the walk: all that the range names, or those of selected blocks.
template <int MODE>
struct SpanWalk : SpanRange {};
template <>
struct SpanWalk<kPicked> {
  const int* picks;
  int block_pages, count;
  __device__ __forceinline__ int piece(int i) const { return picks[i / block_pages] * block_pages + i % block_pages; }
};
template <int MODE>
__device__ __forceinline__ SpanWalk<MODE> span_walk(const SpanParams& p, int q0, int row0, int kvh, int min_beg, int max_base, int kv_len, bool report) {
  SpanWalk<MODE> w;
  if constexpr (MODE == kPicked) {
    const int block = kPage * p.block_pages;
    w.picks = p.picks + ((size_t)(q0 + row0 / p.group) * p.hkv + kvh) * p.pick_count;
    w.block_pages = p.block_pages;
    w.count = span_count_picks(p, w.picks, (max_base + block - 1) / block, report) * p.block_pages;
  } else {
    static_cast<SpanRange&>(w) = span_range(p, kPage, min_beg, p.tree_mask ? kv_len : max_base);
  }
  return w;
}

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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
// A lane's two 16-bit values of an 8 x 8 matrix, row lane / 4 and columns 2 (lane % 4), for those of the transposed one.
__device__ __forceinline__ uint32_t transposed(uint32_t w) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(w));
  return d;
}
// Four values of a row, normalised with the head's sink. (A row that saw nothing has m = -inf and l = 0, not NaN as one of NaN scores: no sink is added to
// it, where e^(sink - m) of a sink of -inf would be a NaN.)
template <int D>
__device__ __forceinline__ void store_row(const SpanParams& p, int q0, int row, int kvh, int d, float4 a, float mm, float ll) {
  const int qi = row / p.group, head = kvh * p.group + row - qi * p.group;
  float c = 1.f;
  if (p.sinks && (mm != -INFINITY || ll != 0.f)) {
    const float sk = p.sinks[head] * kLog2e, mn = fmaxf(mm, sk);
    c = mm == -INFINITY ? 0.f : ex2(mm - mn);
    ll = ll * c + ex2(sk - mn);
  }
  const float inv = ll == 0.f ? 0.f : c / ll;
  *reinterpret_cast<uint2*>(static_cast<bf16*>(p.out) + (size_t)(q0 + qi) * p.ldo + (size_t)head * D + d) =
      make_uint2(pack_bf16x2(a.x * inv, a.y * inv), pack_bf16x2(a.z * inv, a.w * inv));
}

// (m, l, O) of a CTA's four warps, mo [4][16][D] and mml [4][16][2], to the output, to the workspace, or (part_o [16][D], part_ml [16]) to the CTAs of its
// cluster. By 128 threads.
template <int D>
__device__ __forceinline__ void span_join(const SpanParams& p, const float* mo, const float* mml, float* part_o, float4* part_ml, int q0, int row0, int n_rows,
                                          int kvh, int split) {
  const int G = p.group;
  __syncthreads();
  for (int i = threadIdx.x; i < n_rows * (D / 4); i += 128) {
    const int r = i / (D / 4), d = (i - r * (D / 4)) * 4;
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) mm = fmaxf(mm, mml[(w * 16 + r) * 2]);
    float ll = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float2 ml = *reinterpret_cast<const float2*>(mml + (w * 16 + r) * 2);
      const float c = ml.x == -INFINITY ? (mm == -INFINITY ? 1.f : 0.f) : ex2(ml.x - mm);
      const float4 v = *reinterpret_cast<const float4*>(mo + ((size_t)w * 16 + r) * D + d);
      ll += ml.y * c;
      a.x += v.x * c; a.y += v.y * c; a.z += v.z * c; a.w += v.w * c;      // (a factor of 0 too: 0 x NaN is what one warp would have made of it)
    }
    if (p.splits == 1) {
      store_row<D>(p, q0, row0 + r, kvh, d, a, mm, ll);
    } else if (p.in_cluster) {
      *reinterpret_cast<float4*>(part_o + r * D + d) = a;
      if (d == 0) part_ml[r] = make_float4(mm, ll, 0.f, 0.f);
    } else {
      const int qi = (row0 + r) / G, head = kvh * G + (row0 + r) - qi * G;
      const size_t at = ((size_t)(q0 + qi) * p.hq + head) * p.splits + split;
      *reinterpret_cast<float4*>(p.ws_o + at * D + d) = a;
      if (d == 0) *reinterpret_cast<float2*>(p.ws_ml + at * 2) = make_float2(mm, ll);
    }
  }
  if (p.in_cluster) {
    // the splits are a cluster: each CTA takes a share of the row's values from all of them
    cluster_sync();
    for (int i = split * 128 + threadIdx.x; i < n_rows * (D / 4); i += 128 * p.splits) {
      const int r = i / (D / 4), d = (i - r * (D / 4)) * 4;
      float mm = -INFINITY, ll = 0.f;
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int c = 0; c < p.splits; ++c) {
        const float4 ml = ld_dsmem_f4(smem_u32(part_ml + r), c), v = ld_dsmem_f4(smem_u32(part_o + r * D + d), c);
        if (ml.x == -INFINITY && ml.y == 0.f) continue;
        const float mn = fmaxf(mm, ml.x);
        const float w0 = mm == -INFINITY ? (mn == -INFINITY ? 1.f : 0.f) : ex2(mm - mn), w1 = ml.x == -INFINITY ? (mn == -INFINITY ? 1.f : 0.f) : ex2(ml.x - mn);
        mm = mn;
        ll = ll * w0 + ml.y * w1;
        a.x = a.x * w0 + v.x * w1; a.y = a.y * w0 + v.y * w1; a.z = a.z * w0 + v.z * w1; a.w = a.w * w0 + v.w * w1;
      }
      store_row<D>(p, q0, row0 + r, kvh, d, a, mm, ll);
    }
    cluster_sync();                                    // no CTA leaves while another reads its rows
  }
}
}  // namespace
}  // namespace fllm
