// torch_ops.cpp -- the `mas_b200::*` PyTorch operators, implemented in C++ over the C ABI.
//
// Each operator unpacks its tensors into the plain pointers, sizes and strides of the matching
// include/mas_b200.h entry point and launches on the tensor's device and current stream. Doing this in
// C++ keeps a call at dispatcher cost (a few microseconds): the serving loop issues several of these
// ops per layer, and a Python-level operator body would make short steps CPU-bound. The fake (meta)
// kernels that torch.compile traces with are registered from Python (ops.py); the argument checks
// that must raise flashinfer's Python exception types stay in the Python wrappers, and the checks
// here are the last line (TORCH_CHECK -> RuntimeError).
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include <cmath>
#include <optional>
#include <string>
#include <tuple>

#include "../../include/mas_b200.h"

namespace {

int act_code(const at::Tensor& t) {
  if (t.scalar_type() == at::kBFloat16) return MAS_DTYPE_BF16;
  if (t.scalar_type() == at::kHalf) return MAS_DTYPE_FP16;
  TORCH_CHECK(false, "mas_b200: unsupported dtype ", t.scalar_type(), "; expected bfloat16 or float16");
}

int id_code(const at::Tensor& t) {
  if (t.scalar_type() == at::kInt) return MAS_DTYPE_INT32;
  if (t.scalar_type() == at::kLong) return MAS_DTYPE_INT64;
  TORCH_CHECK(false, "mas_b200: indices must be int32 or int64, got ", t.scalar_type());
}

// Numbers go into messages as std::to_string: streaming an integer from this library crashed on a machine whose process
// had a second C++ runtime's locale facets loaded.
void check(int rc, const char* fn) {
  TORCH_CHECK(rc == MAS_OK, fn, " failed with status ", std::to_string(rc), ": ", mas_status_string(rc));
}

// [rows, cols] view of a tensor whose last dimension is contiguous and whose leading dimensions
// collapse into one: returns (rows, row stride in elements).
struct Rows {
  int64_t rows;
  int64_t cols;
  int64_t stride;
};

Rows rows_of(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.dim() >= 1, "mas_b200: ", name, " must have at least one dimension");
  const int64_t cols = t.size(-1);
  TORCH_CHECK(t.stride(-1) == 1 || cols <= 1, "mas_b200: ", name, " must be contiguous in its last dimension");
  if (t.dim() == 1) return {1, cols, cols};
  int64_t rows = 1;
  for (int64_t d = 0; d < t.dim() - 1; ++d) rows *= t.size(d);
  const int64_t stride = t.stride(-2);
  for (int64_t d = 0; d + 2 < t.dim(); ++d) {
    TORCH_CHECK(t.size(d + 1) == 1 || t.stride(d) == t.stride(d + 1) * t.size(d + 1),
                "mas_b200: ", name, "'s leading dimensions must be collapsible into one");
  }
  return {rows, cols, rows > 1 ? stride : cols};
}

void* stream_of(const at::Tensor& t) {
  return static_cast<void*>(c10::cuda::getCurrentCUDAStream(t.device().index()).stream());
}

// The weight is read as `cols` contiguous elements of the activation dtype.
void check_norm_operands(const at::Tensor& input, const at::Tensor& residual, const at::Tensor& weight,
                         int64_t cols) {
  TORCH_CHECK(residual.scalar_type() == input.scalar_type() && weight.scalar_type() == input.scalar_type(),
              "mas_b200: input, residual and weight must share one dtype");
  TORCH_CHECK(weight.dim() == 1 && weight.numel() == cols && weight.is_contiguous(),
              "mas_b200: weight must be a contiguous (hidden_size,) vector");
}

void fused_add_rmsnorm(at::Tensor input, at::Tensor residual, at::Tensor weight, double eps, bool enable_pdl) {
  const c10::cuda::CUDAGuard guard(input.device());
  const Rows x = rows_of(input, "input"), r = rows_of(residual, "residual");
  TORCH_CHECK(x.rows == r.rows && x.cols == r.cols, "mas_b200: input and residual shapes differ");
  check_norm_operands(input, residual, weight, x.cols);
  check(mas_fused_add_rmsnorm(input.data_ptr(), residual.data_ptr(), weight.data_ptr(), x.rows, x.cols, x.stride,
                              r.stride, static_cast<float>(eps), act_code(input), enable_pdl, stream_of(input)),
        "mas_fused_add_rmsnorm");
}

void fused_add_rmsnorm_quant(at::Tensor out, at::Tensor input, at::Tensor residual, at::Tensor weight,
                             at::Tensor scale, double eps, bool enable_pdl) {
  const c10::cuda::CUDAGuard guard(input.device());
  const Rows o = rows_of(out, "out"), x = rows_of(input, "input"), r = rows_of(residual, "residual");
  TORCH_CHECK(o.rows == x.rows && x.rows == r.rows && o.cols == x.cols && x.cols == r.cols,
              "mas_b200: out, input and residual shapes differ");
  TORCH_CHECK(out.scalar_type() == at::kFloat8_e4m3fn, "mas_b200: out must be float8_e4m3fn");
  TORCH_CHECK(scale.scalar_type() == at::kFloat && scale.numel() == 1, "mas_b200: scale must be one fp32 value");
  check_norm_operands(input, residual, weight, x.cols);
  check(mas_fused_add_rmsnorm_quant(out.data_ptr(), input.data_ptr(), residual.data_ptr(), weight.data_ptr(),
                                    scale.data_ptr<float>(), x.rows, x.cols, o.stride, x.stride, r.stride,
                                    static_cast<float>(eps), act_code(input), MAS_DTYPE_FP8_E4M3, enable_pdl,
                                    stream_of(input)),
        "mas_fused_add_rmsnorm_quant");
}

void silu_and_mul(at::Tensor out, at::Tensor input, bool enable_pdl) {
  const c10::cuda::CUDAGuard guard(input.device());
  const Rows o = rows_of(out, "out"), x = rows_of(input, "input");
  TORCH_CHECK(o.rows == x.rows && x.cols == 2 * o.cols, "mas_b200: out must be input[..., :d]-shaped");
  check(mas_silu_and_mul(out.data_ptr(), input.data_ptr(), x.rows, o.cols, o.stride, x.stride, act_code(input),
                         enable_pdl, stream_of(input)),
        "mas_silu_and_mul");
}

void silu_and_mul_quant(at::Tensor out, at::Tensor input, at::Tensor scale, bool enable_pdl) {
  const c10::cuda::CUDAGuard guard(input.device());
  const Rows o = rows_of(out, "out"), x = rows_of(input, "input");
  TORCH_CHECK(o.rows == x.rows && x.cols == 2 * o.cols, "mas_b200: out must be input[..., :d]-shaped");
  TORCH_CHECK(out.scalar_type() == at::kFloat8_e4m3fn, "mas_b200: out must be float8_e4m3fn");
  TORCH_CHECK(scale.scalar_type() == at::kFloat && scale.numel() == 1, "mas_b200: scale must be one fp32 value");
  check(mas_silu_and_mul_quant(out.data_ptr(), input.data_ptr(), scale.data_ptr<float>(), x.rows, o.cols, o.stride,
                               x.stride, act_code(input), MAS_DTYPE_FP8_E4M3, enable_pdl, stream_of(input)),
        "mas_silu_and_mul_quant");
}

// q and k as (tokens, heads, head_size) views, contiguous within a head; one contiguous position per
// token; an fp32 cache. The kernels read positions[0 .. tokens) with unit stride.
void check_rope_operands(const at::Tensor& q, const at::Tensor& k, const at::Tensor& cos_sin_cache,
                         const at::Tensor& pos_ids) {
  TORCH_CHECK(q.dim() == 3 && k.dim() == 3, "mas_b200: q and k must be (tokens, heads, head_size) views");
  TORCH_CHECK(q.size(0) == k.size(0) && q.size(2) == k.size(2), "mas_b200: q and k token counts or head sizes differ");
  TORCH_CHECK(q.stride(2) == 1 && k.stride(2) == 1, "mas_b200: q and k must be contiguous within a head");
  TORCH_CHECK(q.scalar_type() == k.scalar_type(), "mas_b200: q and k must share one dtype");
  TORCH_CHECK(cos_sin_cache.dim() == 2 && cos_sin_cache.is_contiguous() && cos_sin_cache.scalar_type() == at::kFloat,
              "mas_b200: cos_sin_cache must be a contiguous fp32 (max_positions, rotary_dim) tensor");
  TORCH_CHECK(pos_ids.is_contiguous() && pos_ids.numel() == q.size(0),
              "mas_b200: positions must be contiguous with one entry per token");
}

void apply_rope_pos_ids_cos_sin_cache(at::Tensor q, at::Tensor k, at::Tensor cos_sin_cache, at::Tensor pos_ids,
                                      bool interleave, bool enable_pdl) {
  const c10::cuda::CUDAGuard guard(q.device());
  check_rope_operands(q, k, cos_sin_cache, pos_ids);
  check(mas_rope_cos_sin_cache_inplace(pos_ids.data_ptr(), id_code(pos_ids), q.data_ptr(), k.data_ptr(),
                                       cos_sin_cache.data_ptr<float>(), q.size(0), q.size(1), k.size(1), q.size(2),
                                       cos_sin_cache.size(1), cos_sin_cache.size(0), q.stride(0), q.stride(1),
                                       k.stride(0), k.stride(1), interleave ? 0 : 1, act_code(q), nullptr, enable_pdl,
                                       stream_of(q)),
        "mas_rope_cos_sin_cache_inplace");
}

void apply_rope_q_scale(at::Tensor q, at::Tensor k, at::Tensor cos_sin_cache, at::Tensor pos_ids, bool interleave,
                        double beta, int64_t original_max, bool enable_pdl) {
  const c10::cuda::CUDAGuard guard(q.device());
  check_rope_operands(q, k, cos_sin_cache, pos_ids);
  check(mas_rope_cos_sin_cache_q_scale_inplace(
            pos_ids.data_ptr(), id_code(pos_ids), q.data_ptr(), k.data_ptr(), cos_sin_cache.data_ptr<float>(),
            q.size(0), q.size(1), k.size(1), q.size(2), cos_sin_cache.size(1), cos_sin_cache.size(0), q.stride(0),
            q.stride(1), k.stride(0), k.stride(1), interleave ? 0 : 1, static_cast<float>(beta), original_max,
            act_code(q), nullptr, enable_pdl, stream_of(q)),
        "mas_rope_cos_sin_cache_q_scale_inplace");
}

// One layer's paged cache as the C ABI describes it: 4-D k/v caches with identical strides, NHD
// ([pages, page_size, heads, head_size]) or HND ([pages, heads, page_size, head_size]).
MasPagedKVCache paged_cache(const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& kv_indices,
                            const at::Tensor& kv_indptr, bool hnd) {
  TORCH_CHECK(k_cache.dim() == 4 && v_cache.dim() == 4, "mas_b200: k_cache and v_cache must be 4-D");
  TORCH_CHECK(k_cache.sizes() == v_cache.sizes() && k_cache.strides() == v_cache.strides(),
              "mas_b200: k/v cache shapes and strides must be identical");
  TORCH_CHECK(k_cache.stride(3) == 1, "mas_b200: the cache's last dimension must be contiguous");
  TORCH_CHECK(kv_indices.scalar_type() == at::kInt && kv_indptr.scalar_type() == at::kInt &&
                  kv_indices.is_contiguous() && kv_indptr.is_contiguous() && kv_indptr.dim() == 1 &&
                  kv_indptr.numel() >= 1,
              "mas_b200: kv_indices and kv_indptr must be contiguous int32 vectors");
  MasPagedKVCache c = {};
  c.k_cache = k_cache.data_ptr();
  c.v_cache = v_cache.data_ptr();
  c.num_pages = k_cache.size(0);
  c.page_size = hnd ? k_cache.size(2) : k_cache.size(1);
  c.stride_page = k_cache.stride(0);
  c.stride_entry = hnd ? k_cache.stride(2) : k_cache.stride(1);
  c.stride_head = hnd ? k_cache.stride(1) : k_cache.stride(2);
  c.kv_indices = kv_indices.data_ptr<int32_t>();
  c.num_indices = kv_indices.numel();
  c.kv_indptr = kv_indptr.data_ptr<int32_t>();
  c.batch_size = kv_indptr.numel() - 1;
  return c;
}

void append_paged_kv_cache(at::Tensor k, at::Tensor v, at::Tensor batch_indices, at::Tensor positions,
                           at::Tensor k_cache, at::Tensor v_cache, at::Tensor kv_indices, at::Tensor kv_indptr,
                           bool hnd, bool enable_pdl) {
  const c10::cuda::CUDAGuard guard(k.device());
  TORCH_CHECK(k.dim() == 3 && v.dim() == 3 && k.sizes() == v.sizes(), "mas_b200: k and v must be (tokens, heads, head_size)");
  TORCH_CHECK(k.stride(2) == 1 && v.stride(2) == 1, "mas_b200: k and v must be contiguous in head_size");
  TORCH_CHECK(batch_indices.scalar_type() == at::kInt && batch_indices.is_contiguous() &&
                  batch_indices.numel() == k.size(0) && positions.is_contiguous() && positions.numel() == k.size(0),
              "mas_b200: batch_indices (int32) and positions must be contiguous, one per token");
  TORCH_CHECK(k_cache.scalar_type() == k.scalar_type() && v.scalar_type() == k.scalar_type(),
              "mas_b200: k, v and the caches must share one dtype");
  const MasPagedKVCache c = paged_cache(k_cache, v_cache, kv_indices, kv_indptr, hnd);
  TORCH_CHECK((hnd ? k_cache.size(1) : k_cache.size(2)) == k.size(1) && k_cache.size(3) == k.size(2),
              "mas_b200: the cache's heads/head_size differ from k's");
  check(mas_append_paged_kv_cache(k.data_ptr(), v.data_ptr(), batch_indices.data_ptr<int32_t>(), positions.data_ptr(),
                                  id_code(positions), &c, k.size(0), k.size(1), k.size(2), k.stride(0), k.stride(1),
                                  v.stride(0), v.stride(1), act_code(k), nullptr, enable_pdl, stream_of(k)),
        "mas_append_paged_kv_cache");
}

void rope_append_paged_kv_cache(at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor cos_sin_cache,
                                at::Tensor pos_ids, at::Tensor batch_indices, at::Tensor k_cache, at::Tensor v_cache,
                                at::Tensor kv_indices, at::Tensor kv_indptr, bool interleave, bool hnd, double beta,
                                int64_t original_max, bool enable_pdl) {
  const c10::cuda::CUDAGuard guard(q.device());
  TORCH_CHECK(q.dim() == 3 && k.dim() == 3 && v.dim() == 3, "mas_b200: q, k and v must be (tokens, heads, head_size) views");
  TORCH_CHECK(k.sizes() == v.sizes() && q.size(2) == k.size(2) && q.size(0) == k.size(0),
              "mas_b200: q, k and v shapes disagree");
  TORCH_CHECK(cos_sin_cache.dim() == 2 && cos_sin_cache.is_contiguous(), "mas_b200: cos_sin_cache must be contiguous");
  TORCH_CHECK(batch_indices.scalar_type() == at::kInt && batch_indices.is_contiguous() &&
                  batch_indices.numel() == q.size(0) && pos_ids.is_contiguous() && pos_ids.numel() == q.size(0),
              "mas_b200: batch_indices (int32) and positions must be contiguous, one per token");
  TORCH_CHECK(k_cache.scalar_type() == k.scalar_type() && v.scalar_type() == k.scalar_type() &&
                  q.scalar_type() == k.scalar_type(),
              "mas_b200: q, k, v and the caches must share one dtype");
  const MasPagedKVCache c = paged_cache(k_cache, v_cache, kv_indices, kv_indptr, hnd);
  TORCH_CHECK((hnd ? k_cache.size(1) : k_cache.size(2)) == k.size(1) && k_cache.size(3) == k.size(2),
              "mas_b200: the cache's heads/head_size differ from k's");
  check(mas_rope_append_paged_kv_cache(
            pos_ids.data_ptr(), id_code(pos_ids), q.data_ptr(), k.data_ptr(), v.data_ptr(),
            cos_sin_cache.data_ptr<float>(), batch_indices.data_ptr<int32_t>(), &c, q.size(0), q.size(1), k.size(1),
            q.size(2), cos_sin_cache.size(1), cos_sin_cache.size(0), q.stride(0), q.stride(1), k.stride(0), k.stride(1),
            v.stride(0), v.stride(1), interleave ? 0 : 1, static_cast<float>(beta), original_max, act_code(q), nullptr,
            enable_pdl, stream_of(q)),
        "mas_rope_append_paged_kv_cache");
}

void gather(at::Tensor& out, const at::Tensor& ids, const at::Tensor& weight, bool enable_pdl) {
  TORCH_CHECK(weight.dim() == 2 && weight.stride(1) == 1, "mas_b200: weight must be (num_embeddings, dim)");
  TORCH_CHECK(ids.is_contiguous(), "mas_b200: input_ids must be contiguous");
  TORCH_CHECK(out.is_contiguous(), "mas_b200: out must be contiguous");
  check(mas_embedding_gather(out.data_ptr(), weight.data_ptr(), ids.data_ptr(), id_code(ids), ids.numel(),
                             weight.size(1), weight.size(0), weight.size(1), weight.stride(0),
                             static_cast<int>(weight.element_size()), nullptr, enable_pdl, stream_of(weight)),
        "mas_embedding_gather");
}

at::Tensor embedding(at::Tensor input_ids, at::Tensor weight, bool enable_pdl) {
  const c10::cuda::CUDAGuard guard(weight.device());
  std::vector<int64_t> shape(input_ids.sizes().begin(), input_ids.sizes().end());
  shape.push_back(weight.size(1));
  at::Tensor out = at::empty(shape, weight.options());
  gather(out, input_ids.contiguous(), weight, enable_pdl);
  return out;
}

at::Tensor embedding_fill(at::Tensor input_ids, at::Tensor weight, at::Tensor last_tokens, bool enable_pdl) {
  const c10::cuda::CUDAGuard guard(weight.device());
  TORCH_CHECK(weight.dim() == 2 && weight.stride(1) == 1, "mas_b200: weight must be (num_embeddings, dim)");
  TORCH_CHECK(input_ids.is_contiguous(), "mas_b200: input_ids must be contiguous (it is updated in place)");
  TORCH_CHECK(last_tokens.is_contiguous(), "mas_b200: last_tokens must be contiguous");
  std::vector<int64_t> shape(input_ids.sizes().begin(), input_ids.sizes().end());
  shape.push_back(weight.size(1));
  at::Tensor out = at::empty(shape, weight.options());
  check(mas_embedding_gather_fill_placeholders(
            out.data_ptr(), weight.data_ptr(), input_ids.data_ptr(), id_code(input_ids), last_tokens.data_ptr(),
            id_code(last_tokens), last_tokens.numel(), input_ids.numel(), weight.size(1), weight.size(0),
            weight.size(1), weight.stride(0), static_cast<int>(weight.element_size()), nullptr, enable_pdl,
            stream_of(weight)),
        "mas_embedding_gather_fill_placeholders");
  return out;
}

void embedding_out(at::Tensor out, at::Tensor input_ids, at::Tensor weight, bool enable_pdl) {
  const c10::cuda::CUDAGuard guard(weight.device());
  gather(out, input_ids, weight, enable_pdl);
}

// ------------------------------------------------------------------------------------------------
// The 4-bit paged cache. These operators check their arguments here (ValueError, as the Python layer's checks
// elsewhere) and allocate what they return: a decode step calls several of them a layer, and a dozen attribute
// reads and allocations from Python cost more than the kernels of a small step.
// ------------------------------------------------------------------------------------------------
void same_device(const at::Tensor& ref, std::initializer_list<const at::Tensor*> others) {
  for (const at::Tensor* t : others)
    TORCH_CHECK(t->device() == ref.device(), "Expected all tensors to be on the same device, but found ", t->device(),
                " beside ", ref.device());
}

void check_int32(const at::Tensor& t, const char* name, int64_t entries = -1) {
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt && t.is_contiguous() && t.dim() == 1,
                    name, " must be a contiguous int32 vector");
  TORCH_CHECK_VALUE(entries < 0 || t.numel() == entries, name, " must have ", std::to_string(entries), " entries, got ",
                    std::to_string(t.numel()));
}

// Index vectors of either integer type, as the kernels read them.
at::Tensor as_int32(const at::Tensor& t, const char* name) {
  if (t.scalar_type() == at::kInt && t.is_contiguous()) return t;
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, name, " must be int32 or int64");
  // What int32 does not hold becomes its nearest value, which the kernels refuse; a plain cast could name a token or a length.
  return (t.scalar_type() == at::kLong ? t.clamp(INT32_MIN, INT32_MAX) : t).to(at::kInt).contiguous();
}

// A dimension of one entry may carry any stride: it is never stepped over.
int64_t step_of(const at::Tensor& t, int64_t dim, int64_t otherwise) {
  return t.size(dim) > 1 ? t.stride(dim) : otherwise;
}

MasInt4KVCache int4_cache(const at::Tensor& k_codes, const at::Tensor& v_codes, const at::Tensor& pairs, bool hnd) {
  TORCH_CHECK_VALUE(k_codes.dim() == 4 && pairs.dim() == 4 && k_codes.sizes() == v_codes.sizes(),
                    "k/v codes must be 4-D with identical shapes, pairs 4-D");
  TORCH_CHECK_VALUE(k_codes.scalar_type() == at::kByte && v_codes.scalar_type() == at::kByte &&
                        pairs.scalar_type() == at::kBFloat16,
                    "k/v codes must be uint8 and pairs bfloat16");
  same_device(k_codes, {&v_codes, &pairs});
  const int64_t entries = hnd ? 2 : 1, heads = hnd ? 1 : 2, row = k_codes.size(3);
  TORCH_CHECK_VALUE(row == 32 || row == 64, "head_dim must be 64 or 128, got ", std::to_string(2 * row));
  MasInt4KVCache c = {};
  c.k_codes = k_codes.data_ptr();
  c.v_codes = v_codes.data_ptr();
  c.pairs = pairs.data_ptr();
  c.num_pages = k_codes.size(0);
  c.page_size = k_codes.size(entries);
  TORCH_CHECK_VALUE(c.page_size > 0 && k_codes.size(heads) > 0, "page_size and the number of heads must be positive");
  TORCH_CHECK_VALUE(pairs.size(0) == c.num_pages && pairs.size(1) == k_codes.size(heads) &&
                        pairs.size(2) == c.page_size && pairs.size(3) == 4,
                    "pairs must be (pages, heads, page_size, 4)");
  const int64_t inner = c.page_size * 4, page = k_codes.size(heads) * inner;
  TORCH_CHECK_VALUE(pairs.stride(3) == 1 && step_of(pairs, 2, 4) == 4 && step_of(pairs, 1, inner) == inner,
                    "pairs must be contiguous within a page");
  c.pair_stride_page = step_of(pairs, 0, page);
  TORCH_CHECK_VALUE(c.pair_stride_page % 4 == 0 && c.pair_stride_page >= page,
                    "pairs' pages must not overlap and lie a multiple of 4 elements apart");
  c.stride_page = step_of(k_codes, 0, row);
  c.stride_entry = step_of(k_codes, entries, row);
  c.stride_head = step_of(k_codes, heads, row);
  TORCH_CHECK_VALUE(k_codes.stride(3) == 1 && v_codes.stride(3) == 1 && c.stride_page % 16 == 0 &&
                        c.stride_entry % 16 == 0 && c.stride_head % 16 == 0,
                    "k/v codes must be contiguous in the last dimension, the others' strides multiples of 16");
  TORCH_CHECK_VALUE(c.stride_page == step_of(v_codes, 0, row) && c.stride_entry == step_of(v_codes, entries, row) &&
                        c.stride_head == step_of(v_codes, heads, row),
                    "k/v codes must have identical strides");
  TORCH_CHECK_VALUE(reinterpret_cast<uintptr_t>(c.k_codes) % 16 == 0 && reinterpret_cast<uintptr_t>(c.v_codes) % 16 == 0 &&
                        reinterpret_cast<uintptr_t>(c.pairs) % 8 == 0,
                    "k/v codes must be 16-byte aligned, pairs 8-byte aligned");
  return c;
}

// block_tables' row stride; seq_lens and the tables checked against each other.
int64_t check_tables(const at::Tensor& block_tables, const at::Tensor& seq_lens) {
  check_int32(seq_lens, "seq_lens");
  TORCH_CHECK_VALUE(block_tables.dim() == 2 && block_tables.scalar_type() == at::kInt &&
                        block_tables.size(0) == seq_lens.numel() && step_of(block_tables, 1, 1) == 1,
                    "block_tables must be an int32 (batch_size, max_blocks) tensor, contiguous within a row");
  const int64_t stride = step_of(block_tables, 0, block_tables.size(1));
  TORCH_CHECK_VALUE(stride >= block_tables.size(1), "block_tables' rows must not overlap");
  return stride;
}

int64_t check_pages(const at::Tensor& lens, const char* name, const at::Tensor& seq_lens, const at::Tensor& block_tables,
                    const at::Tensor& free_pages, const at::Tensor& num_free, int64_t page_size) {
  const int64_t stride = check_tables(block_tables, seq_lens);
  check_int32(free_pages, "free_pages");
  check_int32(num_free, "num_free", 1);
  TORCH_CHECK_VALUE(lens.dim() == 1 && lens.numel() == seq_lens.numel(), name, " must be (batch_size,)");
  TORCH_CHECK_VALUE(page_size > 0, "page_size must be positive");
  TORCH_CHECK_VALUE(seq_lens.numel() <= 8192, "at most 8192 requests a call, got ", std::to_string(seq_lens.numel()));
  same_device(seq_lens, {&lens, &block_tables, &free_pages, &num_free});
  return stride;
}

void allocate_paged_kv_out(at::Tensor append_lens, at::Tensor seq_lens, at::Tensor block_tables, at::Tensor free_pages,
                           at::Tensor num_free, at::Tensor cum_lens, at::Tensor batch_indices, at::Tensor positions,
                           at::Tensor last_page_len, int64_t page_size, int64_t max_tokens, bool enable_pdl) {
  const c10::cuda::CUDAGuard guard(seq_lens.device());
  const int64_t stride = check_pages(append_lens, "append_lens", seq_lens, block_tables, free_pages, num_free, page_size);
  const int64_t batch = seq_lens.numel();
  TORCH_CHECK_VALUE(max_tokens >= 0, "max_tokens must not be negative");
  check_int32(cum_lens, "cum_append_lens", batch + 1);
  check_int32(batch_indices, "batch_indices", max_tokens);
  check_int32(positions, "positions", max_tokens);
  check_int32(last_page_len, "kv_last_page_len", batch);
  same_device(seq_lens, {&cum_lens, &batch_indices, &positions, &last_page_len});
  const at::Tensor lens = as_int32(append_lens, "append_lens");
  check(mas_allocate_paged_kv(lens.data_ptr<int32_t>(), seq_lens.data_ptr<int32_t>(), block_tables.data_ptr<int32_t>(),
                              free_pages.data_ptr<int32_t>(), num_free.data_ptr<int32_t>(),
                              cum_lens.data_ptr<int32_t>(), batch_indices.data_ptr<int32_t>(),
                              positions.data_ptr<int32_t>(), last_page_len.data_ptr<int32_t>(), batch,
                              block_tables.size(1), stride, page_size, max_tokens, free_pages.numel(), nullptr,
                              enable_pdl, stream_of(seq_lens)),
        "mas_allocate_paged_kv");
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> allocate_paged_kv(
    at::Tensor append_lens, at::Tensor seq_lens, at::Tensor block_tables, at::Tensor free_pages, at::Tensor num_free,
    int64_t page_size, int64_t max_tokens, bool enable_pdl) {
  const c10::cuda::CUDAGuard guard(seq_lens.device());
  TORCH_CHECK_VALUE(max_tokens >= 0, "max_tokens must not be negative");
  const auto options = seq_lens.options().dtype(at::kInt);
  at::Tensor cum = at::empty({seq_lens.numel() + 1}, options), bi = at::empty({max_tokens}, options);
  at::Tensor pos = at::empty({max_tokens}, options), last = at::empty({seq_lens.numel()}, options);
  allocate_paged_kv_out(append_lens, seq_lens, block_tables, free_pages, num_free, cum, bi, pos, last, page_size,
                        max_tokens, enable_pdl);
  return {cum, bi, pos, last};
}

void release_paged_kv(at::Tensor keep_lens, at::Tensor seq_lens, at::Tensor block_tables, at::Tensor free_pages,
                      at::Tensor num_free, int64_t page_size, bool enable_pdl) {
  const c10::cuda::CUDAGuard guard(seq_lens.device());
  const int64_t stride = check_pages(keep_lens, "keep_lens", seq_lens, block_tables, free_pages, num_free, page_size);
  const at::Tensor lens = as_int32(keep_lens, "keep_lens");
  check(mas_release_paged_kv(lens.data_ptr<int32_t>(), seq_lens.data_ptr<int32_t>(), block_tables.data_ptr<int32_t>(),
                             free_pages.data_ptr<int32_t>(), num_free.data_ptr<int32_t>(), seq_lens.numel(),
                             block_tables.size(1), stride, page_size, free_pages.numel(), nullptr, enable_pdl,
                             stream_of(seq_lens)),
        "mas_release_paged_kv");
}

// The rows of an append or a read, and the tokens they belong to.
struct Int4Rows {
  at::Tensor batch_indices, positions, kv_indices, kv_indptr;
};

Int4Rows int4_rows(const at::Tensor& k, const at::Tensor& v, const at::Tensor& batch_indices, const at::Tensor& positions,
                   const at::Tensor& k_codes, const at::Tensor& kv_indices, const at::Tensor& kv_indptr, bool hnd) {
  TORCH_CHECK_VALUE(k.dim() == 3 && v.sizes() == k.sizes() && k.scalar_type() == v.scalar_type(),
                    "k and v must be (tokens, heads, head_dim), equal in shape and dtype");
  TORCH_CHECK_VALUE(k.scalar_type() == at::kBFloat16 || k.scalar_type() == at::kHalf, "unsupported dtype ",
                    k.scalar_type(), "; expected bfloat16 or float16");
  TORCH_CHECK_VALUE(k.stride(2) == 1 && v.stride(2) == 1, "k and v must be contiguous in head_dim");
  TORCH_CHECK_VALUE(k_codes.size(hnd ? 1 : 2) == k.size(1) && 2 * k_codes.size(3) == k.size(2),
                    "cache heads/head_dim differ from k's");
  TORCH_CHECK_VALUE(batch_indices.dim() == 1 && positions.dim() == 1 && batch_indices.numel() == k.size(0) &&
                        positions.numel() == k.size(0),
                    "batch_indices and positions must have one entry per token");
  TORCH_CHECK_VALUE(kv_indptr.dim() == 1 && kv_indptr.numel() >= 1, "kv_indptr must have batch_size + 1 entries");
  same_device(k, {&v, &batch_indices, &positions, &k_codes, &kv_indices, &kv_indptr});
  TORCH_CHECK_VALUE(positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong,
                    "positions must be int32 or int64");
  return {as_int32(batch_indices, "batch_indices"), positions.contiguous(), as_int32(kv_indices, "kv_indices"),
          as_int32(kv_indptr, "kv_indptr")};
}

void append_paged_kv_cache_int4(at::Tensor k, at::Tensor v, at::Tensor batch_indices, at::Tensor positions,
                                at::Tensor k_codes, at::Tensor v_codes, at::Tensor pairs, at::Tensor kv_indices,
                                at::Tensor kv_indptr, bool hnd, bool enable_pdl) {
  const c10::cuda::CUDAGuard guard(k.device());
  const MasInt4KVCache c = int4_cache(k_codes, v_codes, pairs, hnd);
  const Int4Rows r = int4_rows(k, v, batch_indices, positions, k_codes, kv_indices, kv_indptr, hnd);
  check(mas_append_paged_kv_cache_int4(k.data_ptr(), v.data_ptr(), r.batch_indices.data_ptr<int32_t>(),
                                       r.positions.data_ptr(), id_code(r.positions), &c,
                                       r.kv_indices.data_ptr<int32_t>(), r.kv_indices.numel(),
                                       r.kv_indptr.data_ptr<int32_t>(), r.kv_indptr.numel() - 1, k.size(0), k.size(1),
                                       k.size(2), k.stride(0), k.stride(1), v.stride(0), v.stride(1), act_code(k),
                                       nullptr, enable_pdl, stream_of(k)),
        "mas_append_paged_kv_cache_int4");
}

void read_paged_kv_cache_int4_out(at::Tensor k, at::Tensor v, at::Tensor batch_indices, at::Tensor positions,
                                  at::Tensor k_codes, at::Tensor v_codes, at::Tensor pairs, at::Tensor kv_indices,
                                  at::Tensor kv_indptr, bool hnd, bool enable_pdl) {
  const c10::cuda::CUDAGuard guard(k_codes.device());
  const MasInt4KVCache c = int4_cache(k_codes, v_codes, pairs, hnd);
  const Int4Rows r = int4_rows(k, v, batch_indices, positions, k_codes, kv_indices, kv_indptr, hnd);
  check(mas_read_paged_kv_cache_int4(k.data_ptr(), v.data_ptr(), r.batch_indices.data_ptr<int32_t>(),
                                     r.positions.data_ptr(), id_code(r.positions), &c,
                                     r.kv_indices.data_ptr<int32_t>(), r.kv_indices.numel(),
                                     r.kv_indptr.data_ptr<int32_t>(), r.kv_indptr.numel() - 1, k.size(0), k.size(1),
                                     k.size(2), k.stride(0), k.stride(1), v.stride(0), v.stride(1), act_code(k), nullptr,
                                     enable_pdl, stream_of(k)),
        "mas_read_paged_kv_cache_int4");
}

std::tuple<at::Tensor, at::Tensor> read_paged_kv_cache_int4(at::Tensor batch_indices, at::Tensor positions,
                                                            at::Tensor k_codes, at::Tensor v_codes, at::Tensor pairs,
                                                            at::Tensor kv_indices, at::Tensor kv_indptr,
                                                            at::ScalarType dtype, bool hnd, bool enable_pdl) {
  const c10::cuda::CUDAGuard guard(k_codes.device());
  TORCH_CHECK_VALUE(k_codes.dim() == 4, "k/v codes must be 4-D");
  const auto options = k_codes.options().dtype(dtype);
  const int64_t tokens = batch_indices.numel(), heads = k_codes.size(hnd ? 1 : 2), dim = 2 * k_codes.size(3);
  at::Tensor k = at::empty({tokens, heads, dim}, options), v = at::empty({tokens, heads, dim}, options);
  read_paged_kv_cache_int4_out(k, v, batch_indices, positions, k_codes, v_codes, pairs, kv_indices, kv_indptr, hnd,
                               enable_pdl);
  return {k, v};
}

// (tokens, heads, head_dim) or (tokens, heads * head_dim) as heads and strides.
struct HeadRows {
  int64_t tokens, heads, stride_token, stride_head;
};

HeadRows head_rows(const at::Tensor& t, int64_t dim, const char* name) {
  TORCH_CHECK_VALUE((t.dim() == 3 && t.size(2) == dim) || (t.dim() == 2 && t.size(1) % dim == 0), name,
                    " must be (tokens, heads * head_dim) or (tokens, heads, head_dim) with the cache's head_dim ", std::to_string(dim));
  TORCH_CHECK_VALUE(t.stride(-1) == 1, name, " must be contiguous in head_dim");
  if (t.dim() == 2) return {t.size(0), t.size(1) / dim, t.stride(0), dim};
  return {t.size(0), t.size(1), t.stride(0), t.stride(1)};
}

void paged_attention_int4_out(at::Tensor out, std::optional<at::Tensor> lse, at::Tensor query, at::Tensor k_codes,
                              at::Tensor v_codes, at::Tensor pairs, at::Tensor block_tables, at::Tensor seq_lens,
                              std::optional<at::Tensor> cum_seq_lens_q, std::optional<double> sm_scale, bool causal,
                              bool hnd, bool enable_pdl) {
  const c10::cuda::CUDAGuard guard(query.device());
  const MasInt4KVCache c = int4_cache(k_codes, v_codes, pairs, hnd);
  const int64_t dim = 2 * k_codes.size(3), kv_heads = k_codes.size(hnd ? 1 : 2), batch = seq_lens.numel();
  TORCH_CHECK_VALUE(query.scalar_type() == at::kBFloat16 || query.scalar_type() == at::kHalf, "unsupported dtype ",
                    query.scalar_type(), "; expected bfloat16 or float16");
  const HeadRows q = head_rows(query, dim, "query");
  TORCH_CHECK_VALUE(q.heads > 0 && q.heads % kv_heads == 0, "query heads ", std::to_string(q.heads), " do not go with the cache's ",
                    std::to_string(kv_heads));
  TORCH_CHECK_VALUE(out.sizes() == query.sizes() && out.scalar_type() == query.scalar_type(),
                    "out must have the shape and dtype of query");
  const HeadRows o = head_rows(out, dim, "out");
  const int64_t table_stride = check_tables(block_tables, seq_lens);
  same_device(query, {&out, &k_codes, &block_tables, &seq_lens});
  const int32_t* cum = nullptr;
  if (cum_seq_lens_q.has_value()) {
    check_int32(*cum_seq_lens_q, "cum_seq_lens_q", batch + 1);
    same_device(query, {&*cum_seq_lens_q});
    cum = cum_seq_lens_q->data_ptr<int32_t>();
  } else {
    TORCH_CHECK_VALUE(q.tokens == batch, "without cum_seq_lens_q, query must have one row a request");
  }
  TORCH_CHECK_VALUE(q.tokens <= INT32_MAX / q.heads, "query has more than 2^31 rows of heads");
  float* lse_ptr = nullptr;
  if (lse.has_value()) {
    TORCH_CHECK_VALUE(lse->scalar_type() == at::kFloat && lse->is_contiguous() && lse->numel() == q.tokens * q.heads,
                      "lse must be contiguous fp32 (tokens, heads)");
    same_device(query, {&*lse});
    lse_ptr = lse->data_ptr<float>();
  }
  if (batch == 0 || q.tokens == 0) return;
  // Scratch of this call alone: from the caching allocator, so a captured call keeps its own in the graph's pool.
  int64_t bytes = 0;
  check(mas_paged_attention_int4_workspace(dim, &bytes), "mas_paged_attention_int4_workspace");
  at::Tensor work = at::empty({bytes}, query.options().dtype(at::kByte));
  check(mas_paged_attention_int4(query.data_ptr(), out.data_ptr(), lse_ptr, &c, block_tables.data_ptr<int32_t>(),
                                 table_stride, block_tables.size(1), seq_lens.data_ptr<int32_t>(), cum, batch, q.tokens,
                                 q.heads, kv_heads, dim, q.stride_token, q.stride_head, o.stride_token, o.stride_head,
                                 static_cast<float>(sm_scale.has_value() ? *sm_scale : 1.0 / std::sqrt((double)dim)),
                                 causal, act_code(query), work.data_ptr(), bytes, nullptr, enable_pdl, stream_of(query)),
        "mas_paged_attention_int4");
}

std::tuple<at::Tensor, at::Tensor> paged_attention_int4(at::Tensor query, at::Tensor k_codes, at::Tensor v_codes,
                                                        at::Tensor pairs, at::Tensor block_tables, at::Tensor seq_lens,
                                                        std::optional<at::Tensor> cum_seq_lens_q,
                                                        std::optional<double> sm_scale, bool causal, bool hnd,
                                                        bool return_lse, bool enable_pdl) {
  const c10::cuda::CUDAGuard guard(query.device());
  TORCH_CHECK_VALUE(query.dim() == 2 || query.dim() == 3, "query must be 2-D or 3-D");
  TORCH_CHECK_VALUE(k_codes.dim() == 4 && k_codes.size(3) > 0, "k/v codes must be 4-D");
  at::Tensor out = at::empty(query.sizes(), query.options());
  std::optional<at::Tensor> lse;
  const int64_t heads = query.dim() == 3 ? query.size(1) : query.size(1) / (2 * k_codes.size(3));
  at::Tensor held = at::empty({return_lse ? query.size(0) : 0, heads}, query.options().dtype(at::kFloat));
  if (return_lse) lse = held;
  paged_attention_int4_out(out, lse, query, k_codes, v_codes, pairs, block_tables, seq_lens, cum_seq_lens_q, sm_scale,
                           causal, hnd, enable_pdl);
  return {out, held};
}

}  // namespace

TORCH_LIBRARY(mas_b200, m) {
  m.def("fused_add_rmsnorm(Tensor(a!) input, Tensor(b!) residual, Tensor weight, float eps, bool enable_pdl) -> ()");
  m.def("fused_add_rmsnorm_quant(Tensor(a!) out, Tensor input, Tensor(b!) residual, Tensor weight, Tensor scale, "
        "float eps, bool enable_pdl) -> ()");
  m.def("silu_and_mul(Tensor(a!) out, Tensor input, bool enable_pdl) -> ()");
  m.def("silu_and_mul_quant(Tensor(a!) out, Tensor input, Tensor scale, bool enable_pdl) -> ()");
  m.def("apply_rope_pos_ids_cos_sin_cache(Tensor(a!) q, Tensor(b!) k, Tensor cos_sin_cache, Tensor pos_ids, "
        "bool interleave, bool enable_pdl) -> ()");
  m.def("apply_rope_q_scale(Tensor(a!) q, Tensor(b!) k, Tensor cos_sin_cache, Tensor pos_ids, bool interleave, "
        "float beta, int original_max, bool enable_pdl) -> ()");
  m.def("append_paged_kv_cache(Tensor k, Tensor v, Tensor batch_indices, Tensor positions, Tensor(a!) k_cache, "
        "Tensor(b!) v_cache, Tensor kv_indices, Tensor kv_indptr, bool hnd, bool enable_pdl) -> ()");
  m.def("rope_append_paged_kv_cache(Tensor(a!) q, Tensor(b!) k, Tensor v, Tensor cos_sin_cache, Tensor pos_ids, "
        "Tensor batch_indices, Tensor(c!) k_cache, Tensor(d!) v_cache, Tensor kv_indices, Tensor kv_indptr, "
        "bool interleave, bool hnd, float beta, int original_max, bool enable_pdl) -> ()");
  m.def("embedding(Tensor input_ids, Tensor weight, bool enable_pdl) -> Tensor");
  m.def("embedding_out(Tensor(a!) out, Tensor input_ids, Tensor weight, bool enable_pdl) -> ()");
  m.def("embedding_fill(Tensor(a!) input_ids, Tensor weight, Tensor last_tokens, bool enable_pdl) -> Tensor");
  m.def("allocate_paged_kv(Tensor append_lens, Tensor(a!) seq_lens, Tensor(b!) block_tables, Tensor free_pages, "
        "Tensor(c!) num_free, int page_size, int max_tokens, bool enable_pdl) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("allocate_paged_kv_out(Tensor append_lens, Tensor(a!) seq_lens, Tensor(b!) block_tables, Tensor free_pages, "
        "Tensor(c!) num_free, Tensor(d!) cum_append_lens, Tensor(e!) batch_indices, Tensor(f!) positions, "
        "Tensor(g!) kv_last_page_len, int page_size, int max_tokens, bool enable_pdl) -> ()");
  m.def("release_paged_kv(Tensor keep_lens, Tensor(a!) seq_lens, Tensor block_tables, Tensor(b!) free_pages, "
        "Tensor(c!) num_free, int page_size, bool enable_pdl) -> ()");
  m.def("append_paged_kv_cache_int4(Tensor k, Tensor v, Tensor batch_indices, Tensor positions, "
        "Tensor(a!) k_codes, Tensor(b!) v_codes, Tensor(c!) pairs, Tensor kv_indices, Tensor kv_indptr, bool hnd, "
        "bool enable_pdl) -> ()");
  m.def("read_paged_kv_cache_int4(Tensor batch_indices, Tensor positions, Tensor k_codes, Tensor v_codes, "
        "Tensor pairs, Tensor kv_indices, Tensor kv_indptr, ScalarType dtype, bool hnd, bool enable_pdl) -> "
        "(Tensor, Tensor)");
  m.def("read_paged_kv_cache_int4_out(Tensor(a!) k, Tensor(b!) v, Tensor batch_indices, Tensor positions, "
        "Tensor k_codes, Tensor v_codes, Tensor pairs, Tensor kv_indices, Tensor kv_indptr, bool hnd, "
        "bool enable_pdl) -> ()");
  m.def("paged_attention_int4(Tensor query, Tensor k_codes, Tensor v_codes, Tensor pairs, Tensor block_tables, "
        "Tensor seq_lens, Tensor? cum_seq_lens_q, float? sm_scale, bool causal, bool hnd, bool return_lse, "
        "bool enable_pdl) -> (Tensor, Tensor)");
  m.def("paged_attention_int4_out(Tensor(a!) out, Tensor(b!)? lse, Tensor query, Tensor k_codes, Tensor v_codes, "
        "Tensor pairs, Tensor block_tables, Tensor seq_lens, Tensor? cum_seq_lens_q, float? sm_scale, bool causal, "
        "bool hnd, bool enable_pdl) -> ()");
}

TORCH_LIBRARY_IMPL(mas_b200, CUDA, m) {
  m.impl("fused_add_rmsnorm", &fused_add_rmsnorm);
  m.impl("fused_add_rmsnorm_quant", &fused_add_rmsnorm_quant);
  m.impl("silu_and_mul", &silu_and_mul);
  m.impl("silu_and_mul_quant", &silu_and_mul_quant);
  m.impl("apply_rope_pos_ids_cos_sin_cache", &apply_rope_pos_ids_cos_sin_cache);
  m.impl("apply_rope_q_scale", &apply_rope_q_scale);
  m.impl("append_paged_kv_cache", &append_paged_kv_cache);
  m.impl("rope_append_paged_kv_cache", &rope_append_paged_kv_cache);
  m.impl("embedding", &embedding);
  m.impl("embedding_out", &embedding_out);
  m.impl("embedding_fill", &embedding_fill);
  m.impl("allocate_paged_kv", &allocate_paged_kv);
  m.impl("allocate_paged_kv_out", &allocate_paged_kv_out);
  m.impl("release_paged_kv", &release_paged_kv);
  m.impl("append_paged_kv_cache_int4", &append_paged_kv_cache_int4);
  m.impl("read_paged_kv_cache_int4", &read_paged_kv_cache_int4);
  m.impl("read_paged_kv_cache_int4_out", &read_paged_kv_cache_int4_out);
  m.impl("paged_attention_int4", &paged_attention_int4);
  m.impl("paged_attention_int4_out", &paged_attention_int4_out);
}
