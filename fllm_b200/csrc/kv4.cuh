// Rows of a cache held in 4 bits. The row of a token and key head is D / 2 bytes of codes (dims 2i and 2i + 1 in the low and the high half of byte i)
// and two bf16: a step s and a lowest value z; code c stands for z + s c, in fp32. For values x, which are bf16 themselves,
//
//   z = min x,  s = (max x - z) / 15 rounded up to bf16,  c = (x - z) / s rounded to nearest (ties to even)
//
// so the largest value is within reach of code 15 and no value is further than s / 2 from what its code stands for. (x - z is what fp32 makes of it.
// kv4_code rounds its quotient by s, kv4_code_by, of kv4_write, a product that it mends by what is left of x - z; both see a tie as one and write the same bytes.) A row whose values are all alike has s = 0 and is exact. One with an infinity or a NaN, or whose range fp32 does not
// hold, has s = NaN: all of it reads as NaN.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "ptx.cuh"

namespace fllm {
namespace {
template <int D> constexpr int kKv4Row = D / 2 + 4;      // bytes

struct Kv4Scale {
  float step, low;
  __device__ __forceinline__ uint32_t packed() const { return __float_as_uint(step) >> 16 | (__float_as_uint(low) & 0xFFFF0000u); }
};
__device__ __forceinline__ Kv4Scale kv4_scale_of(uint32_t packed) { return {__uint_as_float(packed << 16), __uint_as_float(packed & 0xFFFF0000u)}; }

// Step and lowest value of N values a lane of LANES neighbouring lanes (bf16 values in fp32).
template <int N, int LANES>
__device__ __forceinline__ Kv4Scale kv4_scale(const float (&v)[N]) {
  float lo = v[0], hi = v[0], odd = 0.f;                 // odd: a NaN once a value was not finite
#pragma unroll
  for (int i = 0; i < N; ++i) { lo = fminf(lo, v[i]); hi = fmaxf(hi, v[i]); odd = fmaf(v[i], 0.f, odd); }
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    odd += __shfl_xor_sync(0xffffffffu, odd, o);
  }
  const float range = hi - lo;
  Kv4Scale s;
  const bool fine = odd == 0.f && range < INFINITY;
  s.low = fine ? lo : 0.f;
  s.step = fine ? __uint_as_float((__float_as_uint(__fdiv_rn(range, 15.f)) + 0xFFFFu) & 0xFFFF0000u) : __int_as_float(0x7FC00000);
  return s;
}
// Step and lowest value of a row from its lowest and largest one (infinite or NaN where some value is).
__device__ __forceinline__ Kv4Scale kv4_scale_between(float lo, float hi) {
  const float range = hi - lo;
  const bool fine = fabsf(lo) < INFINITY && fabsf(hi) < INFINITY && range < INFINITY;
  Kv4Scale s;
  s.low = fine ? lo : 0.f;
  s.step = fine ? __uint_as_float((__float_as_uint(__fdiv_rn(range, 15.f)) + 0xFFFFu) & 0xFFFF0000u) : __int_as_float(0x7FC00000);
  return s;
}
__device__ __forceinline__ uint32_t kv4_code(float x, const Kv4Scale& s) {
  if (!(s.step > 0.f)) return 0;
  return (uint32_t)fminf(rintf(__fdiv_rn(x - s.low, s.step)), 15.f);
}
// The same without a division, `inv` 1 / step or near it, for steps of 2^-100 to 2^100: what c leaves of x - z is exact, and says whether c is the nearest
// (of two as near, the even one).
__device__ __forceinline__ uint32_t kv4_code_by(float x, const Kv4Scale& s, float inv) {
  const float d = x - s.low, t = fmaf(d, inv, 8388608.f);       // 2^23: a sum's last bit is that of ones
  float c = t - 8388608.f;
  const float r = fmaf(-c, s.step, d), off = fabsf(r) - 0.5f * s.step;
  if (off > 0.f || (off == 0.f && (__float_as_uint(t) & 1))) c += r > 0.f ? 1.f : -1.f;
  return (uint32_t)fminf(c, 15.f);
}
__device__ __forceinline__ float kv4_value(uint32_t code, const Kv4Scale& s) { return fmaf((float)code, s.step, s.low); }

// Eight codes, of dims 0 to 7, as f16 values z + s c, rounded once, dims in the order 0, 4, 1, 5, 2, 6, 3, 7. The bits of c are those of the f16 number
// c 2^-24, those of c << 4 are c 2^-20: `even` is s 2^24, `odd` s 2^20, `low` z, in both halves of a word (so values are below 2^-6, where s 2^24 is a number).
__device__ __forceinline__ uint4 kv4_widen_f16(uint32_t codes, uint32_t even, uint32_t odd, uint32_t low) {
  uint4 v;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(v.x) : "r"(codes & 0x000F000Fu), "r"(even), "r"(low));
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(v.y) : "r"(codes & 0x00F000F0u), "r"(odd), "r"(low));
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(v.z) : "r"(codes >> 8 & 0x000F000Fu), "r"(even), "r"(low));
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(v.w) : "r"(codes >> 8 & 0x00F000F0u), "r"(odd), "r"(low));
  return v;
}

// A warp's row of D values, EPL to a lane (bf16 values in fp32): PAIRS: v[2i], v[2i + 1] are dims 2 (lane + 32 i) and the next; otherwise v[i] is dim
// lane + 32 i. All lanes take part.
template <int D, bool PAIRS>
__device__ __forceinline__ void kv4_store_row(const float (&v)[D / 32], uint8_t* row, int lane) {
  const Kv4Scale s = kv4_scale<D / 32, 32>(v);
  if constexpr (PAIRS) {
#pragma unroll
    for (int j = 0; j < D / 32; j += 2) row[lane + 16 * j] = (uint8_t)(kv4_code(v[j], s) | kv4_code(v[j + 1], s) << 4);
  } else {
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      const uint32_t mine = kv4_code(v[j], s), next = __shfl_down_sync(0xffffffffu, mine, 1);
      if (!(lane & 1)) row[(lane + 32 * j) >> 1] = (uint8_t)(mine | next << 4);
    }
  }
  if (lane == 0) *reinterpret_cast<uint32_t*>(row + D / 2) = s.packed();
}
}  // namespace
}  // namespace fllm
