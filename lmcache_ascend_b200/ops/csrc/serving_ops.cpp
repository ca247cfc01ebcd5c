// Host side of the serving operators: argument checks, outputs and launches.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>
#include <cmath>
#include <limits>

#include "serving_ops.h"

namespace lmc {
namespace {

// Devices go into messages as strings: printing one through libc10's stream
// operator crosses two copies of the C++ library when this one is linked in.

// `t` is on `dev`, has `dtype` and is dense in memory.
void check_dense(const at::Tensor &t, const char *op, const char *name,
                        const c10::Device &dev, at::ScalarType dtype) {
  TORCH_CHECK(t.device() == dev, op, ": ", name, " is on ", t.device().str(), ", expected ", dev.str());
  TORCH_CHECK(t.scalar_type() == dtype, op, ": ", name, " must be ", dtype, ", got ",
              t.scalar_type());
  TORCH_CHECK(t.is_contiguous(), op, ": ", name, " must be contiguous");
}

DeviceStatus *checked_status(const c10::optional<at::Tensor> &status, const char *op,
                                    const c10::Device &dev) {
  if (!status.has_value()) return nullptr;
  TORCH_CHECK(status->device() == dev && status->is_contiguous() &&
                  status->nbytes() >= kDeviceStatusBytes,
              op, ": status must be a contiguous tensor of >= 24 bytes on ", dev.str());
  return reinterpret_cast<DeviceStatus *>(status->data_ptr());
}

// A dense tensor on the device (without the dispatcher: a decode step's call
// is mostly such overhead).
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType dtype, const c10::Device &dev) {
  return at::detail::empty_cuda(sizes, dtype, dev, c10::nullopt);
}

// The operators are forward only: an input that asks for gradients, or carries a
// tangent of forward differentiation, would lose them without a word.  (An operand
// that is not given is null.)
void check_no_grad(const char *op, std::initializer_list<const at::Tensor *> operands) {
  const bool backward = at::GradMode::is_enabled();
  const bool forward = c10::AutogradState::get_tls_state().get_fw_grad_mode();
  for (const at::Tensor *t : operands) {
    if (t == nullptr) continue;
    TORCH_CHECK(!backward || !t->requires_grad(), op,
                ": forward only, and an operand requires grad");
    TORCH_CHECK(!forward || !t->_fw_grad(/*level=*/0).defined(), op,
                ": forward only, and an operand carries a tangent");
  }
}

const at::Tensor *given(const c10::optional<at::Tensor> &t) { return t.has_value() ? &*t : nullptr; }

// `n` elements of `base` from `first` on, as a tensor of their own (a view without
// the dispatcher).
at::Tensor part_of(const at::Tensor &base, int64_t first, int64_t n) {
  auto t = at::detail::make_tensor<c10::TensorImpl>(
      c10::TensorImpl::VIEW, c10::Storage(base.storage()), base.key_set(), base.dtype());
  t.unsafeGetTensorImpl()->set_storage_offset(first);
  t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
  return t;
}

RowType row_type(at::ScalarType t) {
  return t == at::kFloat ? RowType::kFloat
         : t == at::kBFloat16 ? RowType::kBFloat16 : RowType::kHalf;
}

// A [T, heads * D] or [T, heads, D] tensor as rows: heads adjacent, any row stride.
void check_rows(const at::Tensor &x, const char *op, const char *name, const c10::Device &dev,
                at::ScalarType dtype, int64_t T, int64_t D) {
  TORCH_CHECK(x.device() == dev, op, ": ", name, " is on ", x.device().str(), ", expected ", dev.str());
  TORCH_CHECK(x.scalar_type() == dtype, op, ": ", name, " must be ", dtype, ", got ",
              x.scalar_type());
  TORCH_CHECK((x.dim() == 2 || x.dim() == 3) && x.size(0) == T, op, ": ", name,
              " must be [T, heads * D] or [T, heads, D] with T = ", T);
  if (x.dim() == 2) {
    TORCH_CHECK(x.size(1) % D == 0 && (x.size(1) <= 1 || x.stride(1) == 1), op, ": ", name,
                " rows must be contiguous and a multiple of head_size ", D);
  } else {
    TORCH_CHECK(x.size(2) == D && (D <= 1 || x.stride(2) == 1) &&
                    (x.size(1) <= 1 || x.stride(1) == D),
                op, ": ", name, " rows must be contiguous with heads of ", D);
  }
}

int64_t heads_of(const at::Tensor &x, int64_t D) {
  return x.dim() == 2 ? x.size(1) / D : x.size(1);
}

bool rows_aligned(const at::Tensor &x) {
  const int64_t es = x.element_size();
  return reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0 &&
         (x.size(0) <= 1 || x.stride(0) * es % 16 == 0);
}

bool cache_aligned(const at::Tensor &x) {
  const int64_t es = x.element_size();
  bool ok = reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0;
  for (int d = 0; d < 3; ++d) ok = ok && (x.size(d) <= 1 || x.stride(d) * es % 16 == 0);
  return ok;
}

// Rows that 16-byte vectors and TMA boxes can read: elements adjacent, every
// other stride and the base on 16 bytes.
bool vector_rows(const at::Tensor &x) {
  const int64_t es = x.element_size(), last = x.dim() - 1;
  bool ok = reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0 && x.stride(last) == 1;
  for (int64_t d = 0; d < last; ++d)
    ok = ok && (x.size(d) <= 1 || (x.stride(d) > 0 && x.stride(d) * es % 16 == 0));
  return ok;
}

// `x` itself when vectors can read its rows, else a dense copy (a dense tensor
// that starts off 16 bytes is copied too: new storage is aligned).
at::Tensor with_vector_rows(const at::Tensor &x) {
  return vector_rows(x) ? x : x.clone(at::MemoryFormat::Contiguous);
}

void check_scores(const char *op, double scale, double softcap,
                  const c10::optional<at::Tensor> &slopes, int64_t heads,
                  const c10::Device &dev) {
  // the kernels hold both in fp32, times log2 e and (the cap's argument) 2 scale / cap
  const float f = static_cast<float>(scale), cap = static_cast<float>(softcap);
  constexpr float kLeast = std::numeric_limits<float>::min(), kMost = 1e38f;
  TORCH_CHECK(f >= kLeast && f <= kMost, op, ": scale must be positive and finite (in fp32)");
  TORCH_CHECK(softcap == 0 || (cap >= kLeast && cap <= kMost), op,
              ": softcap must be >= 0 and finite (0: none)");
  TORCH_CHECK(softcap == 0 || scale / softcap <= 1e37, op, ": softcap too small for the scale");
  if (slopes.has_value()) {
    check_dense(*slopes, op, "alibi_slopes", dev, at::kFloat);
    TORCH_CHECK(slopes->dim() == 1 && slopes->numel() == heads, op,
                ": alibi_slopes must be [heads]");
  }
}

void check_heads(const char *op, const at::Tensor &q, int64_t heads, int64_t kv_heads, int64_t D) {
  TORCH_CHECK(q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf, op,
              ": bfloat16 or float16 on the device, got ", q.scalar_type());
  TORCH_CHECK(D == 64 || D == 128, op, ": head_dim 64 or 128 on the device, got ", D);
  TORCH_CHECK(kv_heads >= 1 && heads >= 1 && heads % kv_heads == 0, op, ": ", heads,
              " query heads over ", kv_heads, " KV heads");
}

}  // namespace

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor>
build_slot_mapping(const at::Tensor &context_lens, const at::Tensor &new_lens,
                   at::Tensor &block_tables, int64_t block_size, int64_t num_tokens,
                   const c10::optional<at::Tensor> &free_blocks, int64_t num_blocks,
                   bool long_slots, const c10::optional<at::Tensor> &status) {
  const char *op = "build_slot_mapping";
  TORCH_CHECK(block_size >= 1 && block_size <= (1 << 20), op, ": bad block_size ", block_size);
  TORCH_CHECK(block_tables.is_cuda(), op, ": block_tables must be on the device");
  const c10::Device dev = block_tables.device();
  const auto lt = context_lens.scalar_type();
  TORCH_CHECK(lt == at::kInt || lt == at::kLong, op, ": lengths must be int32 or int64");
  check_dense(context_lens, op, "context_lens", dev, lt);
  check_dense(new_lens, op, "new_lens", dev, lt);
  const int64_t B = context_lens.numel();
  TORCH_CHECK(context_lens.dim() == 1 && new_lens.dim() == 1 && new_lens.numel() == B, op,
              ": context_lens and new_lens must be [batch]");
  TORCH_CHECK(block_tables.scalar_type() == at::kInt && block_tables.dim() == 2 &&
                  block_tables.size(0) >= B &&
                  (block_tables.size(1) <= 1 || block_tables.stride(1) == 1),
              op, ": block_tables must be int32 [>= batch, width] with contiguous rows");
  TORCH_CHECK(num_tokens >= 0 && num_tokens <= 0x7fffffff, op, ": bad num_tokens ", num_tokens);
  TORCH_CHECK(num_blocks >= 0 && num_blocks <= 0x7fffffff, op, ": bad num_blocks ", num_blocks);
  TORCH_CHECK(long_slots || num_blocks * block_size <= 0x7fffffff, op,
              ": slots of ", num_blocks, " blocks of ", block_size, " do not fit in int32");
  TORCH_CHECK(B <= (1 << 24) && block_tables.size(1) <= 0x7fffffff, op, ": too many requests");
  if (free_blocks.has_value()) {
    check_dense(*free_blocks, op, "free_blocks", dev, at::kInt);
    TORCH_CHECK(free_blocks->dim() == 1, op, ": free_blocks must be [free]");
  }
  const c10::cuda::CUDAGuard guard(dev);
  const auto slot_type = long_slots ? at::kLong : at::kInt;
  // six results in two allocations, each on 128 bytes
  auto even = [](int64_t n) { return (n + 31) / 32 * 32; };
  const auto wide = fresh({2 * even(num_tokens)}, slot_type, dev);
  const auto slots = part_of(wide, 0, num_tokens);
  const auto positions = part_of(wide, even(num_tokens), num_tokens);
  const auto narrow = fresh({even(num_tokens) + 3 * even(B + 1)}, at::kInt, dev);
  const auto request_ids = part_of(narrow, 0, num_tokens);
  const auto start = part_of(narrow, even(num_tokens), B + 1);
  const auto seq_lens = part_of(narrow, even(num_tokens) + even(B + 1), B);
  const auto taken = part_of(narrow, even(num_tokens) + 2 * even(B + 1), B + 1);
  SlotArgs a;
  a.ctx = context_lens.data_ptr();
  a.fresh = new_lens.data_ptr();
  a.tables = block_tables.data_ptr<int>();
  a.grow = free_blocks.has_value();
  a.free_blocks = a.grow ? free_blocks->data_ptr<int>() : nullptr;
  a.table_stride = block_tables.stride(0);
  a.num_free = free_blocks.has_value() ? free_blocks->numel() : 0;
  a.num_blocks = num_blocks;
  a.batch = static_cast<int>(B);
  a.width = static_cast<int>(block_tables.size(1));
  a.block_size = static_cast<int>(block_size);
  a.block_shift = -1;
  for (int i = 0; i < 21; ++i)
    if (block_size == (1ll << i)) a.block_shift = i;
  a.num_tokens = num_tokens;
  a.slots = slots.data_ptr();
  a.positions = positions.data_ptr();
  a.request_ids = request_ids.data_ptr<int>();
  a.start = start.data_ptr<int>();
  a.seq_lens = B ? seq_lens.data_ptr<int>() : nullptr;
  a.taken = taken.data_ptr<int>();
  a.status = checked_status(status, op, dev);
  C10_CUDA_CHECK(launch_slot_mapping(a, lt == at::kLong, long_slots,
                                     at::cuda::getCurrentCUDAStream().stream()));
  return {slots, positions, request_ids, start, seq_lens, taken};
}

// Returns q rotated and, when asked for, k rotated, in the given tensors or new
// ones; with caches and a slot map k and v go to their pages.
std::tuple<at::Tensor, c10::optional<at::Tensor>> rotary_embedding_and_cache(
    const at::Tensor &positions, const at::Tensor &query, const c10::optional<at::Tensor> &key,
    const c10::optional<at::Tensor> &value, const c10::optional<at::Tensor> &key_cache,
    const c10::optional<at::Tensor> &value_cache, const c10::optional<at::Tensor> &slot_mapping,
    int64_t head_size, const at::Tensor &cos_sin_cache, bool is_neox,
    const c10::optional<at::Tensor> &given_query_out,
    const c10::optional<at::Tensor> &given_key_out, bool new_key_out,
    const c10::optional<at::Tensor> &status) {
  const char *op = "rotary_embedding";
  TORCH_CHECK(query.is_cuda(), op, ": query must be on the device");
  const c10::Device dev = query.device();
  const auto dt = query.scalar_type();
  check_no_grad(op, {&query, given(key), given(value), given(key_cache), given(value_cache),
                     &cos_sin_cache, given(given_query_out), given(given_key_out)});
  const c10::cuda::CUDAGuard guard(dev);
  const at::Tensor query_out =
      given_query_out.has_value() ? *given_query_out : fresh(query.sizes(), dt, dev);
  c10::optional<at::Tensor> key_out = given_key_out;
  if (!key_out.has_value() && new_key_out && key.has_value())
    key_out = fresh(key->sizes(), dt, dev);
  const int64_t D = head_size;
  TORCH_CHECK(D >= 1 && D <= 65536, op, ": bad head_size ", D);
  TORCH_CHECK(dt == at::kBFloat16 || dt == at::kHalf || dt == at::kFloat, op,
              ": rows must be bfloat16, float16 or float32, got ", dt);
  TORCH_CHECK(positions.dim() == 1 && (positions.scalar_type() == at::kLong ||
                                       positions.scalar_type() == at::kInt),
              op, ": positions must be int32 or int64 [T]");
  check_dense(positions, op, "positions", dev, positions.scalar_type());
  const int64_t T = positions.numel();
  check_rows(query, op, "query", dev, dt, T, D);
  check_rows(query_out, op, "query_out", dev, dt, T, D);
  TORCH_CHECK(heads_of(query_out, D) == heads_of(query, D), op, ": query_out has other heads");
  TORCH_CHECK(cos_sin_cache.dim() == 2 && (cos_sin_cache.scalar_type() == at::kFloat ||
                                           cos_sin_cache.scalar_type() == at::kBFloat16 ||
                                           cos_sin_cache.scalar_type() == at::kHalf),
              op, ": cos_sin_cache must be a float32, bfloat16 or float16 [positions, rot] table");
  check_dense(cos_sin_cache, op, "cos_sin_cache", dev, cos_sin_cache.scalar_type());
  const int64_t rot = cos_sin_cache.size(1);
  TORCH_CHECK(rot >= 2 && rot % 2 == 0 && rot <= D, op, ": rotated part ", rot,
              " must be even and within the head of ", D);
  RopeArgs a = {};
  a.positions = positions.data_ptr();
  a.long_pos = positions.scalar_type() == at::kLong;
  a.q = query.data_ptr();
  a.q_stride = query.stride(0);
  a.q_out = query_out.data_ptr();
  a.q_out_stride = query_out.stride(0);
  a.heads = static_cast<int>(heads_of(query, D));
  bool vec = rows_aligned(query) && rows_aligned(query_out);
  if (key.has_value()) {
    check_rows(*key, op, "key", dev, dt, T, D);
    a.kv_heads = static_cast<int>(heads_of(*key, D));
    a.k = key->data_ptr();
    a.k_stride = key->stride(0);
    vec = vec && rows_aligned(*key);
    if (key_out.has_value()) {
      check_rows(*key_out, op, "key_out", dev, dt, T, D);
      TORCH_CHECK(heads_of(*key_out, D) == a.kv_heads, op, ": key_out has other heads");
      a.k_out = key_out->data_ptr();
      a.k_out_stride = key_out->stride(0);
      vec = vec && rows_aligned(*key_out);
    }
  } else {
    TORCH_CHECK(!key_out.has_value(), op, ": key_out without key");
  }
  const bool cached = slot_mapping.has_value();
  TORCH_CHECK(cached == key_cache.has_value() && cached == value_cache.has_value() &&
                  cached == value.has_value() && (!cached || key.has_value()),
              op, ": key, value, key_cache, value_cache and slot_mapping go together");
  if (cached) {
    check_rows(*value, op, "value", dev, dt, T, D);
    TORCH_CHECK(heads_of(*value, D) == a.kv_heads, op, ": key and value differ in heads");
    a.v = value->data_ptr();
    a.v_stride = value->stride(0);
    const at::Tensor &kc = *key_cache, &vc = *value_cache;
    for (const at::Tensor *c : {&kc, &vc})
      TORCH_CHECK(c->device() == dev && c->scalar_type() == dt && c->dim() == 4 &&
                      c->size(2) == a.kv_heads && c->size(3) == D &&
                      (D <= 1 || c->stride(3) == 1) && c->sizes() == kc.sizes(),
                  op, ": caches must be ", dt, " [blocks, block size, ", a.kv_heads, ", ", D,
                  "] with contiguous heads on ", dev.str());
    TORCH_CHECK(slot_mapping->dim() == 1 && slot_mapping->numel() == T &&
                    (slot_mapping->scalar_type() == at::kLong ||
                     slot_mapping->scalar_type() == at::kInt),
                op, ": slot_mapping must be int32 or int64 [T]");
    check_dense(*slot_mapping, op, "slot_mapping", dev, slot_mapping->scalar_type());
    TORCH_CHECK(kc.size(0) * kc.size(1) <= (1ll << 40) && kc.size(0) <= 0x7fffffff &&
                    kc.size(1) >= 1 && kc.size(1) <= 0x7fffffff,
                op, ": bad cache size");
    a.slots = slot_mapping->data_ptr();
    a.long_slots = slot_mapping->scalar_type() == at::kLong;
    a.k_cache = kc.data_ptr();
    a.v_cache = vc.data_ptr();
    a.k_block = kc.stride(0), a.k_slot = kc.stride(1), a.k_head = kc.stride(2);
    a.v_block = vc.stride(0), a.v_slot = vc.stride(1), a.v_head = vc.stride(2);
    a.block_size = static_cast<int>(kc.size(1));
    a.num_slots = kc.size(0) * kc.size(1);
    vec = vec && rows_aligned(*value) && cache_aligned(kc) && cache_aligned(vc);
  }
  a.table = cos_sin_cache.data_ptr();
  a.max_pos = cos_sin_cache.size(0);
  a.num_tokens = T;
  a.dim = static_cast<int>(D);
  a.rot = static_cast<int>(rot);
  a.neox = is_neox;
  a.status = checked_status(status, op, dev);
  if (T == 0 || a.heads + a.kv_heads == 0) return {query_out, key_out};
  const int64_t es = query.element_size(), cs = cos_sin_cache.element_size();
  // 16-byte units: whole pairs of vectors in the head and in its rotated part,
  // and table rows whose halves start on 16 bytes
  vec = vec && D * es % 32 == 0 && D * es <= 32 * 256 && rot * es % 32 == 0 && rot / 2 * cs % 16 == 0 &&
        16 / es * cs % 16 == 0 && reinterpret_cast<uintptr_t>(a.table) % 16 == 0;
  C10_CUDA_CHECK(launch_rope_cache(a, row_type(dt), row_type(cos_sin_cache.scalar_type()), vec,
                                   at::cuda::getCurrentCUDAStream().stream()));
  return {query_out, key_out};
}

std::tuple<at::Tensor, c10::optional<at::Tensor>> shared_prefix_attention(
    const at::Tensor &query, const at::Tensor &key_cache, const at::Tensor &value_cache,
    const at::Tensor &prefix_blocks, int64_t prefix_len, const at::Tensor &block_tables,
    const at::Tensor &own_lens, double scale, double softcap,
    const c10::optional<at::Tensor> &alibi_slopes, bool return_lse,
    const c10::optional<at::Tensor> &status) {
  const char *op = "shared_prefix_attention";
  TORCH_CHECK(query.is_cuda(), op, ": query must be on the device");
  const c10::Device dev = query.device();
  const auto dt = query.scalar_type();
  check_no_grad(op, {&query, &key_cache, &value_cache, given(alibi_slopes)});
  TORCH_CHECK(query.dim() == 3 || query.dim() == 4, op,
              ": query must be [B, H, D] or [B, q_len, H, D]");
  const at::Tensor q4 = query.dim() == 3 ? query.unsqueeze(1) : query;
  const int64_t B = q4.size(0), Tq = q4.size(1), H = q4.size(2), D = q4.size(3);
  TORCH_CHECK(key_cache.dim() == 4 && key_cache.sizes() == value_cache.sizes() &&
                  key_cache.size(3) == D && key_cache.device() == dev &&
                  value_cache.device() == dev && key_cache.scalar_type() == dt &&
                  value_cache.scalar_type() == dt,
              op, ": caches must be ", dt, " [blocks, block size, KV heads, ", D, "] on ", dev.str());
  const int64_t NB = key_cache.size(0), BS = key_cache.size(1), KH = key_cache.size(2);
  check_heads(op, query, H, KH, D);
  check_scores(op, scale, softcap, alibi_slopes, H, dev);
  TORCH_CHECK(vector_rows(key_cache) && vector_rows(value_cache), op,
              ": cache rows must be contiguous and 16-byte aligned");
  TORCH_CHECK(Tq >= 1 && Tq <= 1024, op, ": q_len must be 1 to 1024, got ", Tq);
  TORCH_CHECK(BS >= 1 && BS <= (1 << 20) && NB >= 1 && NB < 0x7fffffff, op,
              ": bad cache size");
  check_dense(prefix_blocks, op, "prefix_blocks", dev, at::kInt);
  check_dense(own_lens, op, "seq_lens", dev, at::kInt);
  TORCH_CHECK(block_tables.device() == dev && block_tables.scalar_type() == at::kInt &&
                  block_tables.dim() == 2 && block_tables.size(0) >= B &&
                  (block_tables.size(1) <= 1 || block_tables.stride(1) == 1),
              op, ": block_tables must be int32 [>= batch, width] with contiguous rows");
  TORCH_CHECK(own_lens.dim() == 1 && own_lens.numel() == B, op, ": seq_lens must be [batch]");
  TORCH_CHECK(prefix_len >= 0 && prefix_len <= (1ll << 29) &&
                  prefix_blocks.numel() * BS >= prefix_len,
              op, ": prefix of ", prefix_len, " tokens needs more than ", prefix_blocks.numel(),
              " blocks of ", BS);
  TORCH_CHECK(block_tables.size(1) <= (1ll << 29) / BS, op, ": block_tables too wide");
  TORCH_CHECK(B * Tq * H <= 0x7fffffff, op, ": too many rows");
  const c10::cuda::CUDAGuard guard(dev);
  const at::Tensor q = with_vector_rows(q4);
  auto out = fresh(query.sizes(), dt, dev);
  c10::optional<at::Tensor> lse;
  if (return_lse)
    lse = fresh(query.sizes().slice(0, query.dim() - 1), at::kFloat, dev);
  if (B * H == 0) return {out, lse};
  PagedArgs a = {};
  a.q = q.data_ptr(), a.k = key_cache.data_ptr(), a.v = value_cache.data_ptr();
  a.out = out.data_ptr();
  a.lse = return_lse ? lse->data_ptr<float>() : nullptr;
  a.prefix_blocks = prefix_blocks.data_ptr<int>();
  a.tables = block_tables.data_ptr<int>();
  a.own_lens = own_lens.data_ptr<int>();
  a.slopes = alibi_slopes.has_value() ? alibi_slopes->data_ptr<float>() : nullptr;
  a.q_batch = q.stride(0), a.q_token = q.stride(1), a.q_head = q.stride(2);
  a.k_block = key_cache.stride(0), a.k_slot = key_cache.stride(1), a.k_head = key_cache.stride(2);
  a.v_block = value_cache.stride(0), a.v_slot = value_cache.stride(1);
  a.v_head = value_cache.stride(2);
  a.table_stride = block_tables.stride(0);
  a.prefix_len = prefix_len;
  a.batch = static_cast<int>(B), a.q_len = static_cast<int>(Tq);
  a.heads = static_cast<int>(H), a.kv_heads = static_cast<int>(KH);
  a.block_size = static_cast<int>(BS), a.num_blocks = static_cast<int>(NB);
  a.width = static_cast<int>(block_tables.size(1));
  a.scale = static_cast<float>(scale), a.softcap = static_cast<float>(softcap);
  a.status = checked_status(status, op, dev);
  const auto workspace =
      fresh({shared_prefix_attention_workspace(a, static_cast<int>(D))}, at::kByte, dev);
  C10_CUDA_CHECK(launch_shared_prefix_attention(a, row_type(dt), static_cast<int>(D),
                                                workspace.data_ptr(),
                                                at::cuda::getCurrentCUDAStream().stream()));
  return {out, lse};
}

std::tuple<at::Tensor, c10::optional<at::Tensor>> position_attention(
    const at::Tensor &query, const at::Tensor &key, const at::Tensor &value,
    const at::Tensor &q_positions, const c10::optional<at::Tensor> &k_positions, double scale,
    double softcap, const c10::optional<at::Tensor> &alibi_slopes,
    const c10::optional<at::Tensor> &q_documents, const c10::optional<at::Tensor> &k_documents,
    const c10::optional<at::Tensor> &q_prefix_lens, bool causal, bool return_lse) {
  const char *op = "position_attention";
  TORCH_CHECK(query.is_cuda(), op, ": query must be on the device");
  const c10::Device dev = query.device();
  const auto dt = query.scalar_type();
  check_no_grad(op, {&query, &key, &value, given(alibi_slopes)});
  TORCH_CHECK(query.dim() == 3, op, ": query must be [Tq, H, D]");
  const int64_t Tq = query.size(0), H = query.size(1), D = query.size(2);
  TORCH_CHECK(key.dim() == 3 && key.sizes() == value.sizes() && key.size(2) == D &&
                  key.device() == dev && value.device() == dev && key.scalar_type() == dt &&
                  value.scalar_type() == dt,
              op, ": key and value must be ", dt, " [Tk, KV heads, ", D, "] on ", dev.str());
  const int64_t Tk = key.size(0), KH = key.size(1);
  check_heads(op, query, H, KH, D);
  check_scores(op, scale, softcap, alibi_slopes, H, dev);
  TORCH_CHECK(Tk <= (1ll << 30) && Tq * H <= 0x7fffffff, op, ": too many rows");
  auto check_pos = [&](const at::Tensor &p, const char *name, int64_t n) {
    TORCH_CHECK(p.scalar_type() == at::kInt || p.scalar_type() == at::kLong, op, ": ", name,
                " must be int32 or int64");
    check_dense(p, op, name, dev, p.scalar_type());
    TORCH_CHECK(p.dim() == 1 && p.numel() == n, op, ": ", name, " must have ", n, " entries");
  };
  check_pos(q_positions, "q_positions", Tq);
  if (k_positions.has_value()) check_pos(*k_positions, "k_positions", Tk);
  TORCH_CHECK(q_documents.has_value() == k_documents.has_value(), op,
              ": q_documents and k_documents go together");
  auto check_int = [&](const c10::optional<at::Tensor> &p, const char *name, int64_t n) {
    if (!p.has_value()) return;
    check_dense(*p, op, name, dev, at::kInt);
    TORCH_CHECK(p->dim() == 1 && p->numel() == n, op, ": ", name, " must have ", n, " entries");
  };
  check_int(q_documents, "q_documents", Tq);
  check_int(k_documents, "k_documents", Tk);
  check_int(q_prefix_lens, "q_prefix_lens", Tq);
  const c10::cuda::CUDAGuard guard(dev);
  const at::Tensor q = with_vector_rows(query);
  const at::Tensor k = with_vector_rows(key);
  const at::Tensor v = with_vector_rows(value);
  auto out = fresh({Tq, H, D}, dt, dev);
  c10::optional<at::Tensor> lse;
  if (return_lse) lse = fresh({Tq, H}, at::kFloat, dev);
  if (Tq == 0) return {out, lse};
  if (Tk == 0) {
    out.zero_();
    if (return_lse) lse->fill_(-std::numeric_limits<float>::infinity());
    return {out, lse};
  }
  PositionArgs a = {};
  a.q = q.data_ptr(), a.k = k.data_ptr(), a.v = v.data_ptr();
  a.out = out.data_ptr();
  a.lse = return_lse ? lse->data_ptr<float>() : nullptr;
  a.q_pos = q_positions.data_ptr();
  a.k_pos = k_positions.has_value() && Tk ? k_positions->data_ptr() : nullptr;
  a.long_q_pos = q_positions.scalar_type() == at::kLong;
  a.long_k_pos = k_positions.has_value() && k_positions->scalar_type() == at::kLong;
  a.q_doc = q_documents.has_value() ? q_documents->data_ptr<int>() : nullptr;
  a.k_doc = k_documents.has_value() ? k_documents->data_ptr<int>() : nullptr;
  a.q_prefix = q_prefix_lens.has_value() ? q_prefix_lens->data_ptr<int>() : nullptr;
  a.slopes = alibi_slopes.has_value() ? alibi_slopes->data_ptr<float>() : nullptr;
  a.q_token = q.stride(0), a.q_head = q.stride(1);
  a.k_token = k.stride(0), a.k_head = k.stride(1);
  a.v_token = v.stride(0), a.v_head = v.stride(1);
  a.q_tokens = static_cast<int>(Tq), a.k_tokens = static_cast<int>(Tk);
  a.heads = static_cast<int>(H), a.kv_heads = static_cast<int>(KH);
  a.causal = causal;
  a.scale = static_cast<float>(scale), a.softcap = static_cast<float>(softcap);
  const auto workspace =
      fresh({position_attention_workspace(a, static_cast<int>(D))}, at::kByte, dev);
  C10_CUDA_CHECK(launch_position_attention(a, row_type(dt), static_cast<int>(D),
                                           workspace.data_ptr(),
                                           at::cuda::getCurrentCUDAStream().stream()));
  return {out, lse};
}

// The passes of a call of these sizes (for tests: which kernel a shape reaches).
std::tuple<int, int, int> shared_prefix_attention_passes(int64_t batch, int64_t q_len,
                                                         int64_t heads, int64_t kv_heads,
                                                         int64_t block_size, int64_t prefix_len,
                                                         int64_t width) {
  PagedArgs a = {};
  a.batch = static_cast<int>(batch), a.q_len = static_cast<int>(q_len);
  a.heads = static_cast<int>(heads), a.kv_heads = static_cast<int>(kv_heads);
  a.block_size = static_cast<int>(block_size), a.width = static_cast<int>(width);
  a.prefix_len = prefix_len;
  const PrefixPasses p = prefix_passes(a);
  return {p.tensor_core, p.split_prefix, p.own};
}

std::tuple<int, int> position_attention_passes(int64_t q_tokens, int64_t k_tokens, int64_t heads,
                                               int64_t kv_heads) {
  PositionArgs a = {};
  a.q_tokens = static_cast<int>(q_tokens), a.k_tokens = static_cast<int>(k_tokens);
  a.heads = static_cast<int>(heads), a.kv_heads = static_cast<int>(kv_heads);
  const PositionPasses p = position_passes(a);
  return {p.tensor_core, p.split};
}

}  // namespace lmc
