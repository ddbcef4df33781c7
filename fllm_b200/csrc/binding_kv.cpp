// torch.ops.fllm_b200 bindings of the moves inside the cache pools.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include "fllm_ops.h"

namespace {
using at::Tensor;
using c10::optional;

inline cudaStream_t cur_stream() { return c10::cuda::getCurrentCUDAStream().stream(); }

inline void check_ints(const Tensor& t, const Tensor& like, int64_t at_least, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device() && t.scalar_type() == at::kInt && t.is_contiguous() && t.numel() >= at_least, name,
              " must be a contiguous int32 tensor of at least ", at_least, " values on the device of the others");
}

// Pools [planes, blocks, heads, block_size, width], a block's values contiguous; up to kMaxKvPools of them from `from` on
fllm::KvPools make_pools(const std::vector<Tensor>& pools, size_t from) {
  fllm::KvPools p;
  p.count = p.planes = 0;
  for (size_t i = from; i < pools.size() && p.count < fllm::kMaxKvPools; ++i) {
    const Tensor& t = pools[i];
    fllm::KvPool& q = p.pool[p.count++];
    const int64_t elem = t.element_size();
    q.base = t.data_ptr();
    q.planes = (int)t.size(0);
    q.plane_stride = t.size(0) > 1 ? t.stride(0) * elem : 0;
    q.heads = (int)t.size(2);
    q.row_bytes = (int)(t.size(4) * elem);
    p.planes += q.planes;
  }
  p.block_size = (int)pools[0].size(3);
  p.blocks = pools[0].size(1);
  return p;
}
void check_pools(const std::vector<Tensor>& pools) {
  TORCH_CHECK(!pools.empty(), "no cache pools");
  for (const Tensor& t : pools) {
    TORCH_CHECK(t.is_cuda() && t.device() == pools[0].device() && t.dim() == 5 && t.numel() > 0, "cache pools must be CUDA tensors [planes, blocks, heads, block_size, width] of one device");
    TORCH_CHECK(t.size(1) == pools[0].size(1) && t.size(3) == pools[0].size(3) && t.size(1) < INT32_MAX, "cache pools must agree in blocks and block size");
    TORCH_CHECK(t.stride(4) == 1 && t.stride(3) == t.size(4) && t.stride(2) == t.size(3) * t.size(4) && t.stride(1) == t.size(2) * t.stride(2) && t.size(4) * (int64_t)t.element_size() < (1 << 24) && t.size(0) < (1 << 24), "the blocks of a cache pool must be contiguous");
  }
}

int64_t kv_copy_blocks(const std::vector<Tensor>& pools, const Tensor& pairs, const optional<Tensor>& status) {
  check_pools(pools);
  TORCH_CHECK(pairs.dim() == 2 && pairs.size(1) == 2 && pairs.size(0) < INT32_MAX / 2, "pairs must be int32 [n, 2]");
  check_ints(pairs, pools[0], 0, "pairs");
  int* st = nullptr;
  if (status.has_value() && status->defined()) { check_ints(*status, pools[0], 1, "status"); st = status->data_ptr<int>(); }
  c10::cuda::CUDAGuard guard(pools[0].device());
  int64_t n = 0;
  for (size_t i = 0; i < pools.size(); i += fllm::kMaxKvPools)
    n += fllm::kv_copy_blocks(make_pools(pools, i), pairs.data_ptr<int>(), (int)pairs.size(0), st, cur_stream());
  return n;
}

// Pairs that the host lists, one behind the other: source, destination, source, ...
int64_t kv_copy_listed(const std::vector<Tensor>& pools, const std::vector<int64_t>& pairs, const optional<Tensor>& status) {
  check_pools(pools);
  TORCH_CHECK(pairs.size() % 2 == 0 && pairs.size() < INT32_MAX, "pairs must be sources and destinations");
  std::vector<int> of32;
  of32.reserve(pairs.size());
  for (const int64_t b : pairs) {
    TORCH_CHECK(b >= 0 && b < pools[0].size(1), "copy of block ", b, ": the pool has ", pools[0].size(1));
    of32.push_back((int)b);
  }
  int* st = nullptr;
  if (status.has_value() && status->defined()) { check_ints(*status, pools[0], 1, "status"); st = status->data_ptr<int>(); }
  c10::cuda::CUDAGuard guard(pools[0].device());
  int64_t n = 0;
  for (size_t i = 0; i < pools.size(); i += fllm::kMaxKvPools)
    n += fllm::kv_copy_listed(make_pools(pools, i), of32.data(), (int)(of32.size() / 2), st, cur_stream());
  return n;
}

int64_t kv_compact(const std::vector<Tensor>& pools, const Tensor& block_tables, const Tensor& base, const Tensor& path, const Tensor& counts,
                   const optional<Tensor>& status) {
  check_pools(pools);
  TORCH_CHECK(path.dim() == 2 && block_tables.dim() == 2, "block_tables [seqs, blocks] and path [seqs, depth] must be matrices");
  const int64_t B = path.size(0);
  TORCH_CHECK(block_tables.size(0) >= B && path.size(1) < INT32_MAX && B < 65536, "kv_compact: block_tables for every path, at most 65535 of them");
  check_ints(block_tables, pools[0], 0, "block_tables");
  check_ints(path, pools[0], 0, "path");
  check_ints(base, pools[0], B, "base");
  check_ints(counts, pools[0], B, "counts");
  int* st = nullptr;
  if (status.has_value() && status->defined()) { check_ints(*status, pools[0], 1, "status"); st = status->data_ptr<int>(); }
  c10::cuda::CUDAGuard guard(pools[0].device());
  // rows of whole 16-byte pieces and others (the factors of keys are 4 bytes to a row) go in launches of their own
  std::vector<Tensor> kinds[2];
  for (const Tensor& t : pools) kinds[t.size(4) * (int64_t)t.element_size() % 16 ? 1 : 0].push_back(t);
  int64_t n = 0;
  for (const auto& some : kinds)
    for (size_t i = 0; i < some.size(); i += fllm::kMaxKvPools)
      n += fllm::kv_compact(make_pools(some, i), block_tables.data_ptr<int>(), (int)block_tables.size(1), base.data_ptr<int>(), path.data_ptr<int>(),
                            (int)path.size(1), counts.data_ptr<int>(), (int)B, st, cur_stream());
  return n;
}
}  // namespace

TORCH_LIBRARY_FRAGMENT(fllm_b200, m) {
  m.def("kv_copy_blocks(Tensor(a!)[] pools, Tensor pairs, Tensor? status=None) -> int", &kv_copy_blocks);
  m.def("kv_copy_listed(Tensor(a!)[] pools, int[] pairs, Tensor? status=None) -> int", &kv_copy_listed);
  m.def("kv_compact(Tensor(a!)[] pools, Tensor block_tables, Tensor base, Tensor path, Tensor counts, Tensor? status=None) -> int", &kv_compact);
}
