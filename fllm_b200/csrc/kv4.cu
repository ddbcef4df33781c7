// Rows written to a cache held in 4 bits (kv4.cuh), and read back. D / 8 lanes share a row, eight values of 16 bytes each; rows next to each other go to the same
// head, whose rows of a block lie one behind the other.
//
// 8192 rows of 8 heads of 128, keys and values (34 MB read, 9 MB written): 22 us, 1.9 TB/s, what the codes cost to compute (34 with a division for each value and
// for every place, of which the quotient's nearest integer now comes from a product and an exact remainder); read back (4.5 MB, 34 MB as fp32): 9 us, 4.2 TB/s.
// One row: 1 to 2 us, the launch.
#include <stdexcept>

#include "fllm_ops.h"
#include "kv4.cuh"
#include "tma_host.h"

namespace fllm {
namespace {
constexpr int kThreads = 256;
constexpr uint32_t kSigns = 0x80008000u;

__device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// Row of a slot in the pool: first byte, or null where there is none (reported unless the slot is negative).
__device__ __forceinline__ uint8_t* row_of(uint8_t* pool, const Kv4Rows& p, int slot, int head, int row_bytes) {
  if (slot < 0) return nullptr;
  const int block = p.block_shift >= 0 ? slot >> p.block_shift : slot / p.block_size;
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
  const int row = blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES, of = blockIdx.y;      // of: a head of the keys, then of the values
  const int sub = threadIdx.x % LANES;
  const bool in = row < p.rows;
  const bool is_v = of >= p.hkv;
  const int head = is_v ? of - p.hkv : of;
  const int slot = in ? p.slots[row] : -1;
  uint32_t ws[4] = {0, 0, 0, 0};
  if (slot >= 0) {
    const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(is_v ? p.v : p.k) + (size_t)row * (is_v ? p.ldv : p.ldk) + (size_t)head * D + sub * 8;
    const uint4 w = *reinterpret_cast<const uint4*>(src);
    ws[0] = w.x; ws[1] = w.y; ws[2] = w.z; ws[3] = w.w;
  }
  // The lowest value and the lowest of the negated ones, a NaN where there is one, side by side in a word.
  uint32_t ends;
  {
    const uint32_t lo = min2(min2(ws[0], ws[1]), min2(ws[2], ws[3])), hi = min2(min2(ws[0] ^ kSigns, ws[1] ^ kSigns), min2(ws[2] ^ kSigns, ws[3] ^ kSigns));
    ends = min2(__byte_perm(lo, hi, 0x5410), __byte_perm(lo, hi, 0x7632));
  }
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) ends = min2(ends, __shfl_xor_sync(0xffffffffu, ends, o));
  const float2 end = unpack_bf16x2(ends);
  const Kv4Scale s = kv4_scale_between(end.x, -end.y);
  uint8_t* dst = row_of(is_v ? p.v_cache : p.k_cache, p, slot, head, kKv4Row<D>);
  if (!dst) return;
  uint32_t codes = 0;
  const bool plain = s.step > 0x1p-100f && s.step < 0x1p100f;
  const float inv = __fdividef(1.f, plain ? s.step : 1.f);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack_bf16x2(ws[i]);
    if (plain) codes |= kv4_code_by(f.x, s, inv) << 8 * i | kv4_code_by(f.y, s, inv) << (8 * i + 4);
    else codes |= kv4_code(f.x, s) << 8 * i | kv4_code(f.y, s) << (8 * i + 4);
  }
  *reinterpret_cast<uint32_t*>(dst + sub * 4) = codes;
  if (sub == 0) *reinterpret_cast<uint32_t*>(dst + D / 2) = s.packed();
}

template <int D>
__global__ void __launch_bounds__(kThreads) kv4_read_kernel(const __grid_constant__ Kv4Rows p, float* out) {
  constexpr int LANES = D / 8;
  pdl_launch_dependents();
  pdl_wait();
  const int row = blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES, head = blockIdx.y;
  const int sub = threadIdx.x % LANES;
  if (row >= p.rows) return;
  const uint8_t* src = row_of(p.k_cache, p, p.slots[row], head, kKv4Row<D>);
  float4 lo = make_float4(0.f, 0.f, 0.f, 0.f), hi = lo;
  if (src) {
    const uint32_t codes = *reinterpret_cast<const uint32_t*>(src + sub * 4);
    const Kv4Scale s = kv4_scale_of(*reinterpret_cast<const uint32_t*>(src + D / 2));
    lo = make_float4(kv4_value(codes & 15, s), kv4_value(codes >> 4 & 15, s), kv4_value(codes >> 8 & 15, s), kv4_value(codes >> 12 & 15, s));
    hi = make_float4(kv4_value(codes >> 16 & 15, s), kv4_value(codes >> 20 & 15, s), kv4_value(codes >> 24 & 15, s), kv4_value(codes >> 28, s));
  }
  float4* dst = reinterpret_cast<float4*>(out + ((size_t)row * p.hkv + head) * D + sub * 8);
  dst[0] = lo;
  dst[1] = hi;
}

template <int D>
dim3 grid_of(int rows, int heads) {
  constexpr int kRows = kThreads / (D / 8);
  if (heads > 65535) throw std::runtime_error("4-bit cache: too many heads");
  return dim3((unsigned)((rows + kRows - 1) / kRows), (unsigned)heads);
}
Kv4Rows with_shift(Kv4Rows p) {
  p.block_shift = (p.block_size & (p.block_size - 1)) == 0 ? __builtin_ctz(p.block_size) : -1;
  return p;
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
  by_width(p.head_dim, [&](auto d) { launch_pdl(kv4_write_kernel<decltype(d)::value>, grid_of<decltype(d)::value>(p.rows, 2 * p.hkv), dim3(kThreads), 0, s, with_shift(p)); });
  cuda_check(cudaGetLastError(), "kv4_write launch");
}
void kv4_read(const Kv4Rows& p, float* out, cudaStream_t s) {
  if (p.rows <= 0) return;
  by_width(p.head_dim, [&](auto d) { launch_pdl(kv4_read_kernel<decltype(d)::value>, grid_of<decltype(d)::value>(p.rows, p.hkv), dim3(kThreads), 0, s, with_shift(p), out); });
  cuda_check(cudaGetLastError(), "kv4_read launch");
}
}  // namespace fllm
