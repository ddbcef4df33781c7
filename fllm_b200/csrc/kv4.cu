// Rows written to a cache held in 4 bits (kv4.cuh), and read back. D / 8 lanes share a row, eight values of 16 bytes each.
//
// Memory bounds both where there is much to move: 2 x 8192 x 8 rows of 128 (34 MB read, 9 MB written, and back as 67 MB of fp32).
#include <stdexcept>

#include "fllm_ops.h"
#include "kv4.cuh"
#include "tma_host.h"

namespace fllm {
namespace {
constexpr int kThreads = 256;

// Row of a slot in the pool: first byte, or null where there is none (reported unless the slot is negative).
__device__ __forceinline__ uint8_t* row_of(uint8_t* pool, const Kv4Rows& p, int slot, int head, int row_bytes) {
  if (slot < 0) return nullptr;
  const int block = slot / p.block_size;
  if (block >= p.num_blocks) {
    if (p.status) atomicCAS(p.status, FLLM_OK, FLLM_ERR_BAD_ARGS);
    return nullptr;
  }
  return pool + (((size_t)block * p.hkv + head) * p.block_size + (slot - block * p.block_size)) * row_bytes;
}

template <int D>
__global__ void __launch_bounds__(kThreads) kv4_write_kernel(const __grid_constant__ Kv4Rows p) {
  constexpr int LANES = D / 8;
  pdl_launch_dependents();
  pdl_wait();
  const long long item = ((long long)blockIdx.x * kThreads + threadIdx.x) / LANES;      // (row, keys or values, head)
  const int sub = threadIdx.x % LANES;
  const bool in = item < (long long)p.rows * 2 * p.hkv;
  const int row = in ? (int)(item / (2 * p.hkv)) : 0, of = in ? (int)(item - (long long)row * 2 * p.hkv) : 0;
  const bool is_v = of >= p.hkv;
  const int head = is_v ? of - p.hkv : of;
  const int slot = in ? p.slots[row] : -1;
  float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (slot >= 0) {
    const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(is_v ? p.v : p.k) + (size_t)row * (is_v ? p.ldv : p.ldk) + (size_t)head * D + sub * 8;
    const uint4 w = __ldg(reinterpret_cast<const uint4*>(src));
    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack_bf16x2(ws[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
  const Kv4Scale s = kv4_scale<8, LANES>(v);
  uint8_t* dst = row_of(is_v ? p.v_cache : p.k_cache, p, slot, head, kKv4Row<D>);
  if (!dst) return;
  uint32_t codes = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) codes |= kv4_code(v[i], s) << (4 * i);
  *reinterpret_cast<uint32_t*>(dst + sub * 4) = codes;
  if (sub == 0) *reinterpret_cast<uint32_t*>(dst + D / 2) = s.packed();
}

template <int D>
__global__ void __launch_bounds__(kThreads) kv4_read_kernel(const __grid_constant__ Kv4Rows p, float* out) {
  constexpr int LANES = D / 8;
  pdl_launch_dependents();
  pdl_wait();
  const long long item = ((long long)blockIdx.x * kThreads + threadIdx.x) / LANES;      // (row, head)
  const int sub = threadIdx.x % LANES;
  if (item >= (long long)p.rows * p.hkv) return;
  const int row = (int)(item / p.hkv), head = (int)(item - (long long)row * p.hkv);
  const uint8_t* src = row_of(p.k_cache, p, p.slots[row], head, kKv4Row<D>);
  float4 lo = make_float4(0.f, 0.f, 0.f, 0.f), hi = lo;
  if (src) {
    const uint32_t codes = *reinterpret_cast<const uint32_t*>(src + sub * 4);
    const Kv4Scale s = kv4_scale_of(*reinterpret_cast<const uint32_t*>(src + D / 2));
    lo = make_float4(kv4_value(codes & 15, s), kv4_value(codes >> 4 & 15, s), kv4_value(codes >> 8 & 15, s), kv4_value(codes >> 12 & 15, s));
    hi = make_float4(kv4_value(codes >> 16 & 15, s), kv4_value(codes >> 20 & 15, s), kv4_value(codes >> 24 & 15, s), kv4_value(codes >> 28, s));
  }
  float4* dst = reinterpret_cast<float4*>(out + (size_t)item * D + sub * 8);
  dst[0] = lo;
  dst[1] = hi;
}

template <int D>
unsigned grid_of(long long items) {
  const long long ctas = (items * (D / 8) + kThreads - 1) / kThreads;
  if (ctas > 0x7fffffffLL) throw std::runtime_error("4-bit cache: too many rows");
  return (unsigned)ctas;
}
template <class Go>
void by_width(int head_dim, Go&& go) {
  switch (head_dim) {
    case 64: go(std::integral_constant<int, 64>{}); break;
    case 128: go(std::integral_constant<int, 128>{}); break;
    case 256: go(std::integral_constant<int, 256>{}); break;
    default: throw std::runtime_error("4-bit cache: head_dim must be 64, 128 or 256");
  }
}
}  // namespace

void kv4_write(const Kv4Rows& p, cudaStream_t s) {
  if (p.rows <= 0) return;
  by_width(p.head_dim, [&](auto d) { launch_pdl(kv4_write_kernel<decltype(d)::value>, dim3(grid_of<decltype(d)::value>((long long)p.rows * 2 * p.hkv)), dim3(kThreads), 0, s, p); });
  cuda_check(cudaGetLastError(), "kv4_write launch");
}
void kv4_read(const Kv4Rows& p, float* out, cudaStream_t s) {
  if (p.rows <= 0) return;
  by_width(p.head_dim, [&](auto d) { launch_pdl(kv4_read_kernel<decltype(d)::value>, dim3(grid_of<decltype(d)::value>((long long)p.rows * p.hkv)), dim3(kThreads), 0, s, p, out); });
  cuda_check(cudaGetLastError(), "kv4_read launch");
}
}  // namespace fllm
