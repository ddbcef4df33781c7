// Rows and blocks of the cache pools that change places: copies of whole blocks (a fork that writes into a shared one) and the move of a
// draft tree's accepted rows to the places behind the context that they would have had without the tree. Bytes are bytes here: the element
// type only decides how wide an access may be.
//
// Both read and write what they move once and compute nothing; HBM bounds them where there is much to move (160 blocks of 36 layers, 8 heads of 128, bf16:
// 116 us, 6.5 TB/s) and the launch where there is little (one block: 1.7 us, two rows: 2.5, from captured graphs). Every pool and layer goes in one
// launch. The 56 rows that move of 64 accepted paths there, 16.5 MB, take 9.0 us, 1.8 TB/s: one CTA for each of 72 planes and 64 sequences, four rounds of
// them, and in each four trips to memory one behind the other (count, path, table, rows).
#include <stdexcept>

#include "fllm_ops.h"
#include "ptx.cuh"
#include "tma_host.h"

namespace fllm {
namespace {
template <int V> struct Wide;
template <> struct Wide<16> { using type = uint4; };
template <> struct Wide<4> { using type = uint32_t; };
template <> struct Wide<1> { using type = uint8_t; };

// What a kernel is given of the pools: few of them, the usual case, make a launch cheaper (3.4 us of the host's time with room for all 96).
template <int N>
struct SomePools {
  KvPool pool[N];
  int block_size;
  long long blocks;
  explicit SomePools(const KvPools& p) : block_size(p.block_size), blocks(p.blocks) {
    for (int i = 0; i < p.count; ++i) pool[i] = p.pool[i];
  }
};
constexpr int kFewPools = 4;

// Pairs (source, destination) in memory of the device, or in the launch itself: what the host lists needs no memory that has to outlive the call, no copy
// that the host waits for, and a captured graph keeps it. (One listed pair, us a call: 6.4; through a tensor made of the list 19.9, and behind 100 ms of
// other work as long as that; a copy by PyTorch 8.2.)
struct PairsAt {
  const int* at;
  __device__ __forceinline__ int2 operator()(int i) const { return make_int2(at[2 * i], at[2 * i + 1]); }
};
struct PairsListed {
  int2 pair[kListedPairs];
  __device__ __forceinline__ int2 operator()(int i) const { return pair[i]; }
};

template <int N>
__device__ __forceinline__ const KvPool& pool_of_plane(const SomePools<N>& p, int& plane) {
  int i = 0;
  while (plane >= p.pool[i].planes) plane -= p.pool[i++].planes;
  return p.pool[i];
}

constexpr int kCopyThreads = 256, kCopyEach = 4;       // accesses of a thread, all on their way at once

template <int V, int N, class Pairs>
__global__ void __launch_bounds__(kCopyThreads) kv_copy_blocks_kernel(const __grid_constant__ SomePools<N> p, const __grid_constant__ Pairs pairs, int n, int chunks, int* status) {
  using T = typename Wide<V>::type;
  int plane = blockIdx.x / chunks;
  const int chunk = blockIdx.x - plane * chunks;
  const KvPool& pool = pool_of_plane(p, plane);
  const long long width = (long long)pool.heads * p.block_size * pool.row_bytes / V;       // of a block
  pdl_launch_dependents();
  pdl_wait();
  for (int i = blockIdx.y; i < n; i += gridDim.y) {
    const int2 pair = pairs(i);
    const int src = pair.x, dst = pair.y;
    if (src < 0 || dst < 0 || src >= p.blocks || dst >= p.blocks) {
      if (threadIdx.x == 0 && status) atomicCAS(status, FLLM_OK, FLLM_ERR_BAD_ARGS);
      continue;
    }
    T* base = reinterpret_cast<T*>(static_cast<uint8_t*>(pool.base) + plane * pool.plane_stride);
    const T* from = base + src * width;
    T* to = base + dst * width;
    T v[kCopyEach];
    const long long at = (long long)chunk * (kCopyThreads * kCopyEach) + threadIdx.x;
#pragma unroll
    for (int k = 0; k < kCopyEach; ++k)
      if (at + k * kCopyThreads < width) v[k] = from[at + k * kCopyThreads];
#pragma unroll
    for (int k = 0; k < kCopyEach; ++k)
      if (at + k * kCopyThreads < width) to[at + k * kCopyThreads] = v[k];
  }
}

// A thread owns the same V bytes of every row of a sequence in one plane and head, and goes through the accepted path in its order: path[i] >= i
// and rising, so no row is written before it has been read, whatever the rows of one path overwrite of each other.
constexpr int kMoveThreads = 128, kMoveBatch = 8, kMoveSteps = 64;
template <int V, int N>
__global__ void __launch_bounds__(kMoveThreads) kv_compact_kernel(const __grid_constant__ SomePools<N> p, const int* tables, int max_blocks, const int* base,
                                                                  const int* path, int depth, const int* counts, int chunks, int* status) {
  using T = typename Wide<V>::type;
  __shared__ long long from[kMoveSteps], to[kMoveSteps];       // rows of one head in front of the step's; to < 0: nothing moves
  const int seq = blockIdx.y;
  int plane = blockIdx.x / chunks;
  const int chunk = blockIdx.x - plane * chunks;
  const KvPool& pool = pool_of_plane(p, plane);
  const int cols = pool.row_bytes / V;
  const int at = chunk * kMoveThreads + threadIdx.x;           // (head, column)
  const int head = at / cols, col = at - head * cols;
  const bool mine = head < pool.heads;
  T* rows = reinterpret_cast<T*>(static_cast<uint8_t*>(pool.base) + plane * pool.plane_stride);
  pdl_launch_dependents();
  pdl_wait();
  const int count = min(counts[seq], depth), b0 = base[seq];
  const int* table = tables + (size_t)seq * max_blocks;
  auto place = [&](long long tok, long long& row) {            // block and offset of a token; false: there is no such page
    const long long page = tok / p.block_size;
    if (tok < 0 || page >= max_blocks) return false;
    const int block = table[page];
    if (block < 0 || block >= p.blocks) return false;
    row = (long long)block * pool.heads * p.block_size + tok - page * p.block_size;
    return true;
  };
  for (int s0 = 0; s0 < count; s0 += kMoveSteps) {
    const int steps = min(kMoveSteps, count - s0);
    if (threadIdx.x < steps) {
      const int i = s0 + threadIdx.x, n = path[(size_t)seq * depth + i];
      long long f = 0, t = -1;
      if (n != i) {
        if (n < i || b0 < 0 || !place((long long)b0 + n, f) || !place((long long)b0 + i, t)) {
          t = -1;
          if (status) atomicCAS(status, FLLM_OK, FLLM_ERR_BAD_ARGS);
        }
      }
      from[threadIdx.x] = f;
      to[threadIdx.x] = t;
    }
    __syncthreads();
    if (mine) {
      const long long shift = (long long)head * p.block_size;
      for (int i0 = 0; i0 < steps; i0 += kMoveBatch) {
        T v[kMoveBatch];
#pragma unroll
        for (int k = 0; k < kMoveBatch; ++k)
          if (i0 + k < steps && to[i0 + k] >= 0) v[k] = rows[(from[i0 + k] + shift) * cols + col];
#pragma unroll
        for (int k = 0; k < kMoveBatch; ++k)
          if (i0 + k < steps && to[i0 + k] >= 0) rows[(to[i0 + k] + shift) * cols + col] = v[k];
      }
    }
    __syncthreads();
  }
}

// widest access that all pools allow to whole blocks, or to rows
int access_width(const KvPools& p, bool blocks) {
  int v = 16;
  for (int i = 0; i < p.count; ++i) {
    const KvPool& q = p.pool[i];
    const unsigned long long all = reinterpret_cast<uintptr_t>(q.base) | (unsigned long long)q.plane_stride |
                                   (unsigned long long)q.row_bytes * (blocks ? q.heads * p.block_size : 1);
    while (all & (v - 1)) v = v == 16 ? 4 : 1;
  }
  return v;
}

template <class Pairs>
int copy_blocks(const KvPools& p, const Pairs& pairs, int n, int* status, cudaStream_t s) {
  if (n <= 0 || p.planes <= 0) return 0;
  const int v = access_width(p, true);
  long long most = 0;
  for (int i = 0; i < p.count; ++i) most = max(most, (long long)p.pool[i].heads * p.block_size * p.pool[i].row_bytes / v);
  const long long chunks = (most + kCopyThreads * kCopyEach - 1) / (kCopyThreads * kCopyEach);
  if (chunks * p.planes > 0x7fffffffLL) throw std::runtime_error("kv_copy_blocks: pools too large");
  const dim3 grid((unsigned)(chunks * p.planes), (unsigned)min(n, 65535));
  auto go = [&](auto kernel, auto pools) { launch_pdl(kernel, grid, dim3(kCopyThreads), 0, s, pools, pairs, n, (int)chunks, status); };
  if (v == 16 && p.count <= kFewPools) go(kv_copy_blocks_kernel<16, kFewPools, Pairs>, SomePools<kFewPools>(p));
  else if (v == 16) go(kv_copy_blocks_kernel<16, kMaxKvPools, Pairs>, SomePools<kMaxKvPools>(p));
  else if (v == 4) go(kv_copy_blocks_kernel<4, kMaxKvPools, Pairs>, SomePools<kMaxKvPools>(p));
  else go(kv_copy_blocks_kernel<1, kMaxKvPools, Pairs>, SomePools<kMaxKvPools>(p));
  cuda_check(cudaGetLastError(), "kv_copy_blocks launch");
  return 1;
}
static_assert(sizeof(SomePools<kMaxKvPools>) + sizeof(PairsListed) + 32 <= 4096, "a kernel's parameters");
}  // namespace

int kv_copy_blocks(const KvPools& p, const int* pairs, int n, int* status, cudaStream_t s) { return copy_blocks(p, PairsAt{pairs}, n, status, s); }

int kv_copy_listed(const KvPools& p, const int* pairs, int n, int* status, cudaStream_t s) {
  int launches = 0;
  for (int i = 0; i < n; i += kListedPairs) {
    PairsListed some{};
    const int here = min(n - i, kListedPairs);
    for (int k = 0; k < here; ++k) some.pair[k] = make_int2(pairs[2 * (i + k)], pairs[2 * (i + k) + 1]);
    launches += copy_blocks(p, some, here, status, s);
  }
  return launches;
}

int kv_compact(const KvPools& p, const int* block_tables, int max_blocks, const int* base, const int* path, int depth, const int* counts,
               int seqs, int* status, cudaStream_t s) {
  if (seqs <= 0 || depth <= 0 || p.planes <= 0) return 0;
  if (seqs > 65535) throw std::runtime_error("kv_compact: more than 65535 sequences");
  const int v = access_width(p, false);
  long long most = 0;
  for (int i = 0; i < p.count; ++i) most = max(most, (long long)p.pool[i].heads * (p.pool[i].row_bytes / v));
  const long long chunks = (most + kMoveThreads - 1) / kMoveThreads;
  if (chunks * p.planes > 0x7fffffffLL || most > 0x3fffffffLL) throw std::runtime_error("kv_compact: pools too large");
  const dim3 grid((unsigned)(chunks * p.planes), (unsigned)seqs);
  auto go = [&](auto kernel, auto pools) {
    launch_pdl(kernel, grid, dim3(kMoveThreads), 0, s, pools, block_tables, max_blocks, base, path, depth, counts, (int)chunks, status);
  };
  if (v == 16 && p.count <= kFewPools) go(kv_compact_kernel<16, kFewPools>, SomePools<kFewPools>(p));
  else if (v == 16) go(kv_compact_kernel<16, kMaxKvPools>, SomePools<kMaxKvPools>(p));
  else if (v == 4) go(kv_compact_kernel<4, kMaxKvPools>, SomePools<kMaxKvPools>(p));
  else go(kv_compact_kernel<1, kMaxKvPools>, SomePools<kMaxKvPools>(p));
  cuda_check(cudaGetLastError(), "kv_compact launch");
  return 1;
}
}  // namespace fllm
