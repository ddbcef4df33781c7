// torch.ops.fllm_b200 bindings of attention over what a window and the first tokens leave visible and of draft trees.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include <cmath>

#include "fllm_ops.h"

namespace {
using at::Tensor;
using c10::optional;

inline cudaStream_t cur_stream() { return c10::cuda::getCurrentCUDAStream().stream(); }

inline void check_ints(const Tensor& t, const Tensor& like, int64_t at_least, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device() && t.scalar_type() == at::kInt && t.is_contiguous() && t.numel() >= at_least, name,
              " must be a contiguous int32 tensor of at least ", at_least, " values on the device of the others");
}
inline bool is_e4m3(const Tensor& t) { return t.scalar_type() == at::kFloat8_e4m3fn || t.scalar_type() == at::kByte; }

// -> (output rows, kernels launched)
std::tuple<Tensor, int64_t> attention_span(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& block_tables, const Tensor& q_starts,
                       const Tensor& kv_lens, int64_t num_seqs, int64_t max_q_len, int64_t min_q_len, int64_t max_kv_len, int64_t hq,
                       int64_t hkv, int64_t head_dim, double scale, int64_t window, int64_t first, const optional<Tensor>& sinks, double softcap,
                       const optional<Tensor>& tree_mask, const optional<Tensor>& tree_base, const optional<Tensor>& status, const optional<Tensor>& picks) {
  fllm::SpanParams p{};
  TORCH_CHECK(hq > 0 && hkv > 0 && hq % hkv == 0 && hq <= 65536, "attention: query heads must be a multiple of the key heads");
  TORCH_CHECK(head_dim == 64 || head_dim == 128 || head_dim == 256, "attention: head_dim must be 64, 128 or 256");
  TORCH_CHECK(q.is_cuda() && q.scalar_type() == at::kBFloat16 && q.dim() == 2 && q.stride(1) == 1 && q.size(1) == hq * head_dim && q.stride(0) % 8 == 0 &&
                  (reinterpret_cast<uintptr_t>(q.data_ptr()) & 15) == 0,
              "q must be bf16 rows of hq * head_dim values on 16-byte boundaries");
  p.kv4 = k_cache.scalar_type() == at::kByte && k_cache.dim() == 4 && k_cache.size(3) == head_dim / 2 + 4;
  auto pool = [&](const Tensor& t, const char* name) {
    TORCH_CHECK(t.is_cuda() && t.device() == q.device() && t.dim() == 4 && t.is_contiguous() && t.sizes() == k_cache.sizes() &&
                    t.scalar_type() == k_cache.scalar_type() && (t.scalar_type() == at::kBFloat16 || is_e4m3(t)) && t.size(1) == hkv &&
                    t.size(2) % 16 == 0 && t.size(2) > 0 && (p.kv4 || t.size(3) == head_dim) && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0,
                name, " must be a contiguous bf16 or e4m3 pool [blocks, hkv, block_size, head_dim] or one of 4-bit rows (uint8, head_dim / 2 + 4 of them), block_size a "
                "multiple of 16");
  };
  pool(k_cache, "k_cache");
  pool(v_cache, "v_cache");
  TORCH_CHECK(num_seqs >= 0 && max_q_len >= 0 && min_q_len >= 0 && min_q_len <= max_q_len && max_kv_len >= 0 && num_seqs < INT32_MAX &&
                  max_q_len < INT32_MAX && max_kv_len < INT32_MAX && q.size(0) < INT32_MAX / 2, "attention: lengths out of range");
  TORCH_CHECK(block_tables.dim() == 2 && block_tables.size(0) >= num_seqs && block_tables.size(1) < (1 << 26), "attention: block_tables [num_seqs, blocks]");
  check_ints(block_tables, q, 0, "block_tables");
  check_ints(q_starts, q, num_seqs + 1, "q_starts");
  check_ints(kv_lens, q, num_seqs, "kv_lens");
  TORCH_CHECK(std::isfinite((float)scale) && scale >= 2e-38 && std::isfinite(softcap) && softcap >= 0, "attention: scale must be positive, softcap not negative");
  TORCH_CHECK(window >= 0 && first >= 0 && window < INT32_MAX && first < INT32_MAX, "attention: window and first must not be negative");
  if (sinks.has_value() && sinks->defined()) {
    TORCH_CHECK(sinks->is_cuda() && sinks->device() == q.device() && sinks->scalar_type() == at::kFloat && sinks->is_contiguous() && sinks->numel() == hq,
                "sinks must be fp32 [hq]");
    p.sinks = sinks->data_ptr<float>();
  }
  if (tree_mask.has_value() && tree_mask->defined()) {
    TORCH_CHECK(tree_base.has_value() && tree_base->defined(), "attention_tree: tree_mask needs tree_base");
    TORCH_CHECK(tree_mask->is_cuda() && tree_mask->device() == q.device() && tree_mask->scalar_type() == at::kLong && tree_mask->is_contiguous() &&
                    (tree_mask->dim() == 1 || tree_mask->dim() == 2) && tree_mask->size(0) == q.size(0),
                "tree_mask must be contiguous int64 [rows] or [rows, words]");
    p.words = tree_mask->dim() == 1 ? 1 : (int)tree_mask->size(1);
    TORCH_CHECK(p.words >= 1 && p.words <= 4, "tree_mask: at most 256 nodes, 64 to a word");
    check_ints(*tree_base, q, q.size(0), "tree_base");
    p.tree_mask = reinterpret_cast<const unsigned long long*>(tree_mask->data_ptr<int64_t>());
    p.tree_base = tree_base->data_ptr<int>();
  }
  if (status.has_value() && status->defined()) {
    check_ints(*status, q, 1, "status");
    p.status = status->data_ptr<int>();
  }
  if (picks.has_value() && picks->defined()) {
    TORCH_CHECK(!p.tree_mask && window == 0, "attention_blocks: selected blocks have no window and no tree");
    TORCH_CHECK(picks->dim() == 3 && picks->size(0) == q.size(0) && picks->size(1) == hkv && picks->size(2) > 0 && picks->size(2) < (1 << 24),
                "attention_blocks: blocks must be int32 [rows, hkv, count]");
    check_ints(*picks, q, 0, "blocks");
    p.picks = picks->data_ptr<int>();
    p.pick_count = (int)picks->size(2);
  }
  p.q = q.data_ptr(); p.ldq = q.stride(0);
  p.k_cache = k_cache.data_ptr(); p.v_cache = v_cache.data_ptr();
  p.block_tables = block_tables.data_ptr<int>(); p.max_blocks = (int)block_tables.size(1);
  p.block_pages = (int)(k_cache.size(2) / 16); p.num_blocks = k_cache.size(0);
  p.q_starts = q_starts.data_ptr<int>(); p.kv_lens = kv_lens.data_ptr<int>();
  p.tokens = (int)q.size(0); p.num_seqs = (int)num_seqs;
  p.hq = (int)hq; p.hkv = (int)hkv; p.group = (int)(hq / hkv); p.head_dim = (int)head_dim;
  p.kv_fp8 = is_e4m3(k_cache) && !p.kv4;
  // No sequence has more rows than there are, and none may be said to have none: one that has more than announced is reported by a kernel.
  p.max_q_len = (int)std::max<int64_t>(1, std::min<int64_t>(max_q_len, q.size(0)));
  p.min_q_len = (int)std::min<int64_t>(min_q_len, p.max_q_len); p.max_kv_len = (int)max_kv_len;
  p.reach = (int)std::min<int64_t>(block_tables.size(1) * k_cache.size(2), INT32_MAX / 2 - 4096);
  p.window = (int)window; p.first = window > 0 ? (int)first : 0;
  p.scale_log2 = (float)(scale * 1.4426950408889634); p.softcap = (float)softcap;
  c10::cuda::CUDAGuard guard(q.device());
  Tensor out = at::empty({q.size(0), q.size(1)}, q.options());
  if (p.tokens == 0 || num_seqs == 0) return {out, 0};
  p.out = out.data_ptr(); p.ldo = out.stride(0);
  const fllm::SpanPlan plan = fllm::attention_span_plan(p);
  TORCH_CHECK(plan.rows_splits > 0 || plan.tile_splits > 0, "attention: no kernel was planned for the rows");
  Tensor ws;                                  // of this call alone: two streams or two captured graphs do not share it
  if (plan.bytes) ws = at::empty({(int64_t)plan.bytes}, q.options().dtype(at::kByte));
  const int n = fllm::attention_span(p, plan, plan.bytes ? ws.data_ptr() : nullptr, cur_stream());
  return {out, n};
}
}  // namespace

TORCH_LIBRARY_FRAGMENT(fllm_b200, m) {
  m.def("attention_span(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_tables, Tensor q_starts, Tensor kv_lens, int num_seqs, "
        "int max_q_len, int min_q_len, int max_kv_len, int hq, int hkv, int head_dim, float scale, int window, int first, Tensor? sinks, float softcap, "
        "Tensor? tree_mask=None, Tensor? tree_base=None, Tensor? status=None, Tensor? picks=None) -> (Tensor, int)", &attention_span);
}
