// torch.ops.fllm_b200 bindings of caches held in 4 bits and of the choice of blocks that a query row reads.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include <algorithm>

#include "fllm_ops.h"

namespace {
using at::Tensor;
using c10::optional;

inline cudaStream_t cur_stream() { return c10::cuda::getCurrentCUDAStream().stream(); }

inline void check_ints(const Tensor& t, const Tensor& like, int64_t at_least, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device() && t.scalar_type() == at::kInt && t.is_contiguous() && t.numel() >= at_least, name,
              " must be a contiguous int32 tensor of at least ", at_least, " values on the device of the others");
}
inline int* status_of(const optional<Tensor>& status, const Tensor& like) {
  if (!status.has_value() || !status->defined()) return nullptr;
  check_ints(*status, like, 1, "status");
  return status->data_ptr<int>();
}
inline bool aligned(const Tensor& t, int bytes) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & (bytes - 1)) == 0; }
inline void check_head_dim(int64_t d) { TORCH_CHECK(d == 64 || d == 128 || d == 256, "head_dim must be 64, 128 or 256"); }

// A pool of 4-bit rows; fills in what it says of the sizes
void take_pool(fllm::Kv4Rows& p, const Tensor& cache, const char* name) {
  TORCH_CHECK(cache.is_cuda() && cache.scalar_type() == at::kByte && cache.dim() == 4 && cache.is_contiguous() && cache.numel() > 0 && aligned(cache, 16), name,
              " must be a contiguous uint8 pool [blocks, hkv, block_size, head_dim / 2 + 4] on a 16-byte boundary");
  p.head_dim = (int)(cache.size(3) - 4) * 2;
  check_head_dim(p.head_dim);
  TORCH_CHECK(cache.size(3) == p.head_dim / 2 + 4 && cache.size(0) * cache.size(2) < INT32_MAX && cache.size(1) < (1 << 20), name, ": sizes out of range");
  p.num_blocks = (int)cache.size(0);
  p.hkv = (int)cache.size(1);
  p.block_size = (int)cache.size(2);
}

void kv4_write(const Tensor& k, const Tensor& v, const Tensor& slots, Tensor k_cache, Tensor v_cache, const optional<Tensor>& status) {
  fllm::Kv4Rows p{};
  take_pool(p, k_cache, "k_cache");
  TORCH_CHECK(v_cache.sizes() == k_cache.sizes() && v_cache.device() == k_cache.device(), "k_cache and v_cache must be alike");
  take_pool(p, v_cache, "v_cache");
  for (const Tensor* t : {&k, &v})
    TORCH_CHECK(t->is_cuda() && t->device() == k_cache.device() && t->scalar_type() == at::kBFloat16 && t->dim() == 2 && t->size(1) == (int64_t)p.hkv * p.head_dim &&
                    t->size(0) == k.size(0) && (t->size(0) == 0 || (t->stride(1) == 1 && t->stride(0) % 8 == 0 && aligned(*t, 16))),
                "k and v must be bf16 [rows, hkv * head_dim], rows on 16-byte boundaries");
  TORCH_CHECK(k.size(0) < INT32_MAX / 64, "kv4_write: too many rows");
  check_ints(slots, k_cache, k.size(0), "slots");
  p.status = status_of(status, k_cache);
  p.k = k.data_ptr(); p.ldk = k.stride(0);
  p.v = v.data_ptr(); p.ldv = v.stride(0);
  p.slots = slots.data_ptr<int>();
  p.k_cache = k_cache.data_ptr<uint8_t>();
  p.v_cache = v_cache.data_ptr<uint8_t>();
  p.rows = (int)k.size(0);
  c10::cuda::CUDAGuard guard(k_cache.device());
  fllm::kv4_write(p, cur_stream());
}

Tensor kv4_read(const Tensor& cache, const Tensor& slots, const optional<Tensor>& status) {
  fllm::Kv4Rows p{};
  take_pool(p, cache, "cache");
  TORCH_CHECK(slots.dim() == 1 && slots.numel() < INT32_MAX / 64, "slots must be int32 [rows]");
  check_ints(slots, cache, 0, "slots");
  p.status = status_of(status, cache);
  p.slots = slots.data_ptr<int>();
  p.k_cache = static_cast<uint8_t*>(cache.data_ptr());
  p.rows = (int)slots.numel();
  c10::cuda::CUDAGuard guard(cache.device());
  Tensor out = at::empty({slots.numel(), (int64_t)p.hkv * p.head_dim}, cache.options().dtype(at::kFloat));
  fllm::kv4_read(p, out.data_ptr<float>(), cur_stream());
  return out;
}

// [blocks, hkv, 2 * head_dim + 16] int8 -> head_dim
int64_t check_bounds(const Tensor& bounds, int64_t hkv) {
  TORCH_CHECK(bounds.is_cuda() && bounds.scalar_type() == at::kChar && bounds.dim() == 3 && bounds.is_contiguous() && bounds.numel() > 0 && aligned(bounds, 16) &&
                  bounds.size(1) == hkv && bounds.size(0) < INT32_MAX,
              "bounds must be contiguous int8 [blocks, hkv, 2 * head_dim + 16] on a 16-byte boundary");
  const int64_t d = (bounds.size(2) - 16) / 2;
  check_head_dim(d);
  TORCH_CHECK(bounds.size(2) == 2 * d + 16, "bounds must be [blocks, hkv, 2 * head_dim + 16]");
  return d;
}

void kv_bounds(const Tensor& k_cache, Tensor bounds, const Tensor& slots, const optional<Tensor>& status) {
  TORCH_CHECK(k_cache.is_cuda() && k_cache.dim() == 4 && k_cache.is_contiguous() && aligned(k_cache, 16) && k_cache.device() == bounds.device(),
              "k_cache must be a contiguous pool [blocks, hkv, block_size, row] on the device of the bounds");
  fllm::BoundsParams p{};
  p.head_dim = (int)check_bounds(bounds, k_cache.size(1));
  TORCH_CHECK(bounds.size(0) == k_cache.size(0), "bounds for every block of the pool");
  const auto type = k_cache.scalar_type();
  const int64_t row = k_cache.size(3);
  int kind = -1;
  if (type == at::kBFloat16 && row == p.head_dim) kind = 0;
  else if ((type == at::kFloat8_e4m3fn || type == at::kByte) && row == p.head_dim) kind = 1;
  else if (type == at::kByte && row == p.head_dim / 2 + 4) kind = fllm::kKv4;
  TORCH_CHECK(kind >= 0, "kv_bounds: k_cache must hold bf16, e4m3 or 4-bit rows of the bounds' head_dim");
  TORCH_CHECK(k_cache.size(0) * k_cache.size(2) < INT32_MAX && k_cache.size(1) < (1 << 20) && slots.dim() == 1 && slots.numel() < INT32_MAX / 64, "kv_bounds: sizes out of range");
  check_ints(slots, k_cache, 0, "slots");
  p.status = status_of(status, k_cache);
  p.k_cache = k_cache.data_ptr();
  p.bounds = bounds.data_ptr<int8_t>();
  p.slots = slots.data_ptr<int>();
  p.rows = (int)slots.numel();
  p.hkv = (int)k_cache.size(1);
  p.block_size = (int)k_cache.size(2);
  p.num_blocks = (int)k_cache.size(0);
  c10::cuda::CUDAGuard guard(k_cache.device());
  fllm::kv_bounds(p, kind, cur_stream());
}

// -> (blocks [rows, hkv, count], kernels launched)
std::tuple<Tensor, int64_t> select_blocks(const Tensor& q, const Tensor& bounds, const Tensor& block_tables, const Tensor& q_starts, const Tensor& kv_lens, int64_t num_seqs,
                                          int64_t max_q_len, int64_t max_kv_len, int64_t hq, int64_t hkv, int64_t head_dim, int64_t block_size, int64_t count,
                                          int64_t lead, int64_t tail, const optional<Tensor>& status, int64_t scores_bytes) {
  TORCH_CHECK(hq > 0 && hkv > 0 && hq % hkv == 0 && hq <= 65536, "select_blocks: query heads must be a multiple of the key heads");
  TORCH_CHECK(check_bounds(bounds, hkv) == head_dim, "select_blocks: bounds of another head_dim");
  TORCH_CHECK(q.is_cuda() && q.device() == bounds.device() && q.scalar_type() == at::kBFloat16 && q.dim() == 2 && q.size(1) == hq * head_dim &&
                  (q.size(0) == 0 || (q.stride(1) == 1 && q.stride(0) % 8 == 0 && aligned(q, 16))),
              "q must be bf16 rows of hq * head_dim values on 16-byte boundaries");
  TORCH_CHECK(block_size > 0 && block_size < (1 << 20) && lead >= 0 && tail >= 1 && lead < (1 << 20) && tail < (1 << 20) && count >= lead + tail && count <= fllm::kMostSelectBlocks,
              "select_blocks: count must have room for the first and the last blocks, one of the last at least");
  TORCH_CHECK(num_seqs >= 0 && max_q_len >= 0 && max_kv_len >= 0 && num_seqs < INT32_MAX && q.size(0) < INT32_MAX / 2, "select_blocks: lengths out of range");
  TORCH_CHECK(block_tables.dim() == 2 && block_tables.size(0) >= num_seqs && block_tables.size(1) < (1 << 26), "select_blocks: block_tables [num_seqs, blocks]");
  check_ints(block_tables, q, 0, "block_tables");
  check_ints(q_starts, q, num_seqs + 1, "q_starts");
  check_ints(kv_lens, q, num_seqs, "kv_lens");
  fllm::SelectParams p{};
  fllm::SpanParams& s = p.rows;
  s.q = q.data_ptr(); s.ldq = q.size(0) ? q.stride(0) : 0;
  s.block_tables = block_tables.data_ptr<int>(); s.max_blocks = (int)block_tables.size(1);
  s.num_blocks = bounds.size(0);
  s.q_starts = q_starts.data_ptr<int>(); s.kv_lens = kv_lens.data_ptr<int>();
  s.tokens = (int)q.size(0); s.num_seqs = (int)num_seqs;
  s.hq = (int)hq; s.hkv = (int)hkv; s.group = 1; s.head_dim = (int)head_dim;
  s.max_q_len = (int)std::max<int64_t>(1, std::min<int64_t>(max_q_len, q.size(0)));
  // No text is taken for longer than the tables reach, or than it was said to be: one that is gets reported.
  const int64_t blocks = std::min<int64_t>((std::min<int64_t>(max_kv_len, INT32_MAX / 4) + block_size - 1) / block_size, block_tables.size(1));
  s.reach = (int)std::min<int64_t>(blocks * block_size, INT32_MAX / 2 - 4096);
  s.status = status_of(status, q);
  p.bounds = bounds.data_ptr<int8_t>();
  p.group = (int)(hq / hkv); p.block_size = (int)block_size;
  p.count = (int)count; p.lead = (int)lead; p.tail = (int)tail;
  p.stride = (int)blocks;
  TORCH_CHECK(blocks <= fllm::kMostSelectBlocks || blocks <= count, "select_blocks: texts of at most ", fllm::kMostSelectBlocks, " blocks");
  TORCH_CHECK(q.size(0) * hkv < INT32_MAX, "select_blocks: too many rows");
  c10::cuda::CUDAGuard guard(q.device());
  Tensor out = at::empty({q.size(0), hkv, count}, q.options().dtype(at::kInt));
  if (q.size(0) == 0) return {out, 0};
  if (num_seqs == 0) return {out.fill_(-1), 0};
  p.out = out.data_ptr<int>();
  // Scores are of this call alone: two streams or two captured graphs do not share them. Rows of long prompts beside long texts take their turns in them.
  const int64_t rows = p.stride > p.count ? std::min<int64_t>(q.size(0), std::max<int64_t>(64, scores_bytes / (4 * hkv * p.stride))) : q.size(0);
  Tensor scores;
  if (p.stride > p.count) {
    scores = at::empty({rows * hkv * p.stride}, q.options().dtype(at::kFloat));
    p.scores = scores.data_ptr<float>();
  }
  int64_t n = 0;
  for (int64_t from = 0; from < q.size(0); from += rows) {
    p.row_from = (int)from;
    p.row_to = (int)std::min<int64_t>(from + rows, q.size(0));
    n += fllm::select_blocks(p, cur_stream());
  }
  return {out, n};
}
}  // namespace

TORCH_LIBRARY_FRAGMENT(fllm_b200, m) {
  m.def("kv4_write(Tensor k, Tensor v, Tensor slots, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor? status=None) -> ()", &kv4_write);
  m.def("kv4_read(Tensor cache, Tensor slots, Tensor? status=None) -> Tensor", &kv4_read);
  m.def("kv_bounds(Tensor k_cache, Tensor(a!) bounds, Tensor slots, Tensor? status=None) -> ()", &kv_bounds);
  m.def("select_blocks(Tensor q, Tensor bounds, Tensor block_tables, Tensor q_starts, Tensor kv_lens, int num_seqs, int max_q_len, int max_kv_len, int hq, int hkv, "
        "int head_dim, int block_size, int count, int lead, int tail, Tensor? status=None, int scores_bytes=268435456) -> (Tensor, int)", &select_blocks);
}
