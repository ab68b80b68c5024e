// host.cpp -- Python module slm_turbo_b200._host: the host side of the
// serving-step entry points (kv_page_plan, kv_rotary, kv_rotary_store,
// kv_dequantize_load, kv_prompt_attention).
//
// Checks of arguments, output allocation, the current stream and the call of
// the C entry.  These calls run once per layer or step and their kernels take
// a few microseconds for small batches, less than the same host work took in
// Python: a rotary call of 777 tokens was 16.7 us, 6 of them on the GPU.
#include <ATen/core/grad_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>

#include <array>
#include <cmath>
#include <initializer_list>
#include <optional>
#include <sstream>
#include <string>
#include <tuple>

#include "slm_turbo_b200.h"

namespace py = pybind11;
using at::Tensor;
using Opt = std::optional<Tensor>;

namespace {

template <typename... T>
[[noreturn]] void refuse(const T&... parts) {
  std::ostringstream s;
  (s << ... << parts);
  throw std::runtime_error(s.str());
}

// ------------------------------------------------------------ device state --
py::object g_error_word;               // device index -> address of its error word
std::array<int32_t*, 64> g_error_words{};

int32_t* error_word(int index) {
  if (index < (int)g_error_words.size() && g_error_words[index]) return g_error_words[index];
  auto* p = reinterpret_cast<int32_t*>(g_error_word(index).cast<uintptr_t>());
  if (index < (int)g_error_words.size()) g_error_words[index] = p;
  return p;
}

void check(int status, const char* what) {
  if (status != SLMT_OK) refuse(what, ": ", slmt_status_string(status), " (status ", status, ")");
}

// ------------------------------------------------------------------ checks --
bool half_type(const Tensor& t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; }

const char* type_name(const Tensor& t) { return c10::toString(t.scalar_type()); }

int tag(at::ScalarType t) {
  switch (t) {
    case at::kHalf: return SLMT_DTYPE_F16;
    case at::kBFloat16: return SLMT_DTYPE_BF16;
    case at::kFloat: return SLMT_DTYPE_F32;
    case at::kInt: return SLMT_DTYPE_I32;
    case at::kLong: return SLMT_DTYPE_I64;
    default: return -1;
  }
}

void need_half_cuda(const Tensor& t, const char* what, const char* name) {
  if (!t.is_cuda()) refuse(what, ": ", name, " must be a CUDA tensor");
  if (!half_type(t)) refuse(what, ": ", name, " must be float16/bfloat16, got ", type_name(t));
}

void same_device(const char* what, int index, std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors)
    if (t && (!t->is_cuda() || t->get_device() != index))
      refuse(what, ": tensors on ", t->device(), " and cuda:", index);
}

// Neither direction of autograd passes: gradients that would be lost while it
// records, and tangents of dual tensors, which no_grad does not switch off.
void no_autograd(const char* what, std::initializer_list<const Tensor*> tensors) {
  const bool records = at::GradMode::is_enabled();
  for (const Tensor* t : tensors) {
    if (!t) continue;
    if (records && t->requires_grad())
      refuse(what, ": has no backward pass; call it under torch.no_grad() or on detached tensors");
    if (t->_fw_grad(0).defined())
      refuse(what, ": has no forward-mode or backward pass; call it on the primal of the dual tensor");
  }
}

const Tensor* get(const Opt& t) { return t ? &*t : nullptr; }

// An output of the call: torch.empty without the dispatcher's part (a page plan
// has three: 8.1 us with it, 7.0 without).
Tensor fresh(at::IntArrayRef shape, at::ScalarType type, const Tensor& beside) {
  return Tensor(at::detail::empty_cuda(shape, type, beside.device(), std::nullopt));
}

Tensor int32_of(const Tensor& t) {
  return t.scalar_type() == at::kInt && t.is_contiguous() ? t : t.to(at::kInt).contiguous();
}

template <typename T>
T* data(const Tensor& t) {
  return reinterpret_cast<T*>(t.data_ptr());
}

Tensor unit_rows(const Tensor& t) { return t.stride(2) == 1 ? t : t.contiguous(); }

// --------------------------------------------------------------- page plan --
std::tuple<Tensor, Tensor, Tensor> page_plan(const Tensor& query_start_loc, const Tensor& seq_lens,
                                             const Tensor& block_tables, int64_t block_size, int64_t num_tokens,
                                             const Opt& free_blocks, const Opt& free_cursor, const Opt& slot_mapping,
                                             const Opt& positions) {
  constexpr const char* W = "page plan";
  if (!block_tables.is_cuda()) refuse(W, ": block_tables must be a CUDA tensor");
  if (block_tables.scalar_type() != at::kInt)
    refuse(W, ": block_tables must be int32, got ", type_name(block_tables));
  const int index = block_tables.get_device();
  const int64_t R = seq_lens.numel();
  if (block_tables.dim() != 2 || block_tables.size(0) < R || (block_tables.size(1) > 1 && block_tables.stride(1) != 1))
    refuse(W, ": block_tables must be [", R, ", max_blocks] with unit column stride");
  if (query_start_loc.numel() < R + 1)
    refuse(W, ": query_start_loc needs ", R + 1, " entries, has ", query_start_loc.numel());
  if (num_tokens < 0) refuse(W, ": num_tokens must not be negative, got ", num_tokens);
  if (free_blocks && (free_blocks->scalar_type() != at::kInt || !free_blocks->is_contiguous()))
    refuse(W, ": free_blocks must be contiguous int32");
  if (free_cursor && (free_cursor->scalar_type() != at::kInt || free_cursor->numel() != 1))
    refuse(W, ": free_cursor must be one int32");
  for (const Tensor* t : {get(slot_mapping), get(positions)})
    if (t && (t->scalar_type() != at::kLong || !t->is_contiguous() || t->numel() != num_tokens))
      refuse(W, ": slot_mapping and positions must be contiguous int64 of length ", num_tokens);
  same_device(W, index, {&query_start_loc, &seq_lens, get(free_blocks), get(free_cursor), get(slot_mapping),
                         get(positions)});
  const c10::cuda::OptionalCUDAGuard guard(block_tables.device());
  const Tensor qsl = int32_of(query_start_loc), sl = int32_of(seq_lens);
  Tensor slots = slot_mapping ? *slot_mapping : fresh({num_tokens}, at::kLong, block_tables);
  Tensor pos = positions ? *positions : fresh({num_tokens}, at::kLong, block_tables);
  Tensor cursor = fresh({1}, at::kInt, block_tables);
  // an empty free list is a list all the same (its tensor has no address)
  const int32_t* list = nullptr;
  if (free_blocks) list = free_blocks->numel() ? data<int32_t>(*free_blocks) : data<int32_t>(cursor);
  check(slmt_page_plan(data<int32_t>(qsl), data<int32_t>(sl), R, data<int32_t>(block_tables), block_tables.stride(0),
                       block_tables.size(1), block_size, list, free_blocks ? free_blocks->numel() : 0, free_cursor ? data<int32_t>(*free_cursor) : nullptr,
                       num_tokens, data<int64_t>(slots), data<int64_t>(pos), data<int32_t>(cursor), error_word(index),
                       c10::cuda::getCurrentCUDAStream(index).stream()),
        W);
  return {slots, pos, cursor};
}

// ------------------------------------------------------------------ rotary --
void rotary_checks(const char* what, const Tensor& query, const Tensor& key, const Tensor& positions,
                   const Tensor& inv_freq, const Opt& query_out, const Opt& key_out) {
  need_half_cuda(query, what, "query");
  need_half_cuda(key, what, "key");
  if (query.scalar_type() != key.scalar_type()) refuse(what, ": query/key dtypes differ");
  if (query.dim() != 3 || key.dim() != 3 || query.size(0) != key.size(0) || query.size(2) != key.size(2))
    refuse(what, ": query/key must be [N, H, D] and [N, KV, D], got ", query.sizes(), " and ", key.sizes());
  if ((positions.scalar_type() != at::kInt && positions.scalar_type() != at::kLong) || positions.dim() != 1 ||
      positions.size(0) != query.size(0))
    refuse(what, ": positions must be int32/int64 of length ", query.size(0));
  if (inv_freq.scalar_type() != at::kFloat || inv_freq.dim() != 1 || 2 * inv_freq.numel() > query.size(2))
    refuse(what, ": inv_freq must be float32 with at most head_dim/2 entries");
  if (query_out && (query_out->sizes() != query.sizes() || query_out->scalar_type() != query.scalar_type() ||
                    query_out->stride(2) != 1))
    refuse(what, ": query_out must be ", query.sizes(), " ", type_name(query), " with unit head-dim stride");
  if (key_out &&
      (key_out->sizes() != key.sizes() || key_out->scalar_type() != key.scalar_type() || key_out->stride(2) != 1))
    refuse(what, ": key_out must be ", key.sizes(), " ", type_name(key), " with unit head-dim stride");
  same_device(what, query.get_device(), {&key, &positions, &inv_freq, get(query_out), get(key_out)});
  no_autograd(what, {&query, &key, &inv_freq, get(query_out), get(key_out)});
}

std::tuple<Tensor, Tensor> rotary(const Tensor& query, const Tensor& key, const Tensor& positions,
                                  const Tensor& inv_freq, bool interleaved, double scaling, const Opt& query_out,
                                  const Opt& key_out) {
  constexpr const char* W = "rotary";
  rotary_checks(W, query, key, positions, inv_freq, query_out, key_out);
  const c10::cuda::OptionalCUDAGuard guard(query.device());
  // an in-place call reads the caller's own rows, whatever their strides
  const Tensor q = unit_rows(query), k = unit_rows(key), pos = positions.contiguous(), freq = inv_freq.contiguous();
  Tensor qo = query_out ? *query_out : fresh(q.sizes(), q.scalar_type(), q);
  Tensor ko = key_out ? *key_out : fresh(k.sizes(), k.scalar_type(), k);
  check(slmt_rotary(q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1),
                    tag(q.scalar_type()), pos.data_ptr(), tag(pos.scalar_type()), data<float>(freq), 2 * freq.numel(),
                    interleaved, (float)scaling, q.size(0), q.size(1), k.size(1), q.size(2), qo.data_ptr(),
                    qo.stride(0), qo.stride(1), ko.data_ptr(), ko.stride(0), ko.stride(1),
                    c10::cuda::getCurrentCUDAStream(q.get_device()).stream()),
        W);
  return {qo, ko};
}

std::tuple<Tensor, Opt> rotary_store(const Tensor& query, const Tensor& key, const Tensor& value,
                                     const Tensor& positions, const Tensor& inv_freq, const Tensor& kv_cache,
                                     const Tensor& slot_mapping, bool interleaved, double scaling,
                                     const Opt& query_out, const Opt& key_out, bool return_key) {
  constexpr const char* W = "rotary store";
  rotary_checks(W, query, key, positions, inv_freq, query_out, key_out);
  need_half_cuda(value, W, "value");
  const int64_t N = key.size(0), KV = key.size(1), D = key.size(2);
  if (value.scalar_type() != key.scalar_type() || value.sizes() != key.sizes())
    refuse(W, ": value must be ", key.sizes(), " ", type_name(key));
  if (kv_cache.scalar_type() != at::kByte || !kv_cache.is_contiguous() || kv_cache.dim() != 4)
    refuse(W, ": kv_cache must be contiguous uint8 [num_blocks, block_size, KV, D+8]");
  if (kv_cache.size(2) != KV || kv_cache.size(3) != D + 8)
    refuse(W, ": cache rows are [", kv_cache.size(2), ", ", kv_cache.size(3), "], expected [", KV, ", ", D + 8, "]");
  if (slot_mapping.scalar_type() != at::kLong || slot_mapping.numel() != N)
    refuse(W, ": slot_mapping must be int64 of length ", N);
  if (key_out && !return_key) refuse(W, ": key_out is given but return_key is False");
  const int index = query.get_device();
  same_device(W, index, {&value, &kv_cache, &slot_mapping});
  no_autograd(W, {&value});
  const c10::cuda::OptionalCUDAGuard guard(query.device());
  const Tensor q = unit_rows(query), k = unit_rows(key), v = unit_rows(value);
  const Tensor pos = positions.contiguous(), freq = inv_freq.contiguous(), slots = slot_mapping.contiguous();
  Tensor qo = query_out ? *query_out : fresh(q.sizes(), q.scalar_type(), q);
  Opt ko = key_out;
  if (!ko && return_key) ko = fresh(k.sizes(), k.scalar_type(), k);
  check(slmt_rotary_store(q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1),
                          v.data_ptr(), v.stride(0), v.stride(1), tag(q.scalar_type()), pos.data_ptr(),
                          tag(pos.scalar_type()), data<float>(freq), 2 * freq.numel(), interleaved, (float)scaling, N,
                          q.size(1), KV, D, qo.data_ptr(), qo.stride(0), qo.stride(1), ko ? ko->data_ptr() : nullptr,
                          ko ? ko->stride(0) : 0, ko ? ko->stride(1) : 0, data<uint8_t>(kv_cache), kv_cache.size(0),
                          kv_cache.size(1), data<int64_t>(slots), error_word(index),
                          c10::cuda::getCurrentCUDAStream(index).stream()),
        W);
  return {qo, ko};
}

// -------------------------------------------------------------------- load --
std::tuple<Tensor, Tensor> dequantize_load(const Tensor& kv_cache, const Tensor& slot_mapping, at::ScalarType dtype,
                                           const Opt& key_out, const Opt& value_out) {
  constexpr const char* W = "load";
  if (!kv_cache.is_cuda()) refuse(W, ": kv_cache must be a CUDA tensor");
  if (kv_cache.scalar_type() != at::kByte) refuse(W, ": kv_cache must be uint8, got ", type_name(kv_cache));
  if (kv_cache.dim() != 4 || !kv_cache.is_contiguous())
    refuse(W, ": kv_cache must be contiguous [num_blocks, block_size, KV, D+8]");
  if (slot_mapping.scalar_type() != at::kLong || slot_mapping.dim() != 1)
    refuse(W, ": slot_mapping must be int64 [N]");
  if (dtype != at::kHalf && dtype != at::kBFloat16 && dtype != at::kFloat)
    refuse(W, ": dtype must be float16/bfloat16/float32, got ", c10::toString(dtype));
  const int64_t N = slot_mapping.numel(), KV = kv_cache.size(2), D = kv_cache.size(3) - 8;
  const std::array<int64_t, 3> shape{N, KV, D};
  for (const Tensor* t : {get(key_out), get(value_out)})
    if (t && (t->sizes() != at::IntArrayRef(shape) || t->scalar_type() != dtype || !t->is_contiguous()))
      refuse(W, ": key_out and value_out must be contiguous ", at::IntArrayRef(shape), " ", c10::toString(dtype));
  if (D <= 0) refuse(W, ": head_dim must be 64/80/128");
  const int index = kv_cache.get_device();
  same_device(W, index, {&slot_mapping, get(key_out), get(value_out)});
  no_autograd(W, {get(key_out), get(value_out)});
  const c10::cuda::OptionalCUDAGuard guard(kv_cache.device());
  const Tensor slots = slot_mapping.contiguous();
  Tensor k = key_out ? *key_out : fresh(shape, dtype, kv_cache);
  Tensor v = value_out ? *value_out : fresh(shape, dtype, kv_cache);
  check(slmt_kv_dequantize_load(data<uint8_t>(kv_cache), kv_cache.size(0), kv_cache.size(1), KV, D,
                                data<int64_t>(slots), N, k.data_ptr(), v.data_ptr(), tag(dtype), error_word(index),
                                c10::cuda::getCurrentCUDAStream(index).stream()),
        W);
  return {k, v};
}

// -------------------------------------------------------- prompt attention --
// `t` itself where 16-byte rows can be copied from it, else a dense copy.
Tensor tile_ready(const Tensor& t) {
  const int64_t token = t.stride(0), head = t.stride(1);
  if (t.stride(2) == 1 && token > 0 && head > 0 && (token | head) % 8 == 0 &&
      reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0)
    return t;
  return t.clone(at::MemoryFormat::Contiguous);
}

Tensor prompt_attention(const Tensor& query, const Tensor& key, const Tensor& value, const Tensor& query_start_loc,
                        int64_t max_query_len, const Opt& seq_lens, const Opt& given_out,
                        std::optional<double> sm_scale) {
  constexpr const char* W = "prompt attention";
  need_half_cuda(query, W, "query");
  if (query.dim() != 3 || key.dim() != 3 || key.sizes() != value.sizes() || key.size(0) != query.size(0) ||
      key.size(2) != query.size(2))
    refuse(W, ": query [N, Hq, D] and key/value [N, KV, D] expected, got ", query.sizes(), ", ", key.sizes(), ", ",
           value.sizes());
  if (key.scalar_type() != query.scalar_type() || value.scalar_type() != query.scalar_type())
    refuse(W, ": query/key/value dtypes differ");
  const int64_t N = query.size(0), H = query.size(1), D = query.size(2), KV = key.size(1);
  if (KV == 0 || H % KV) refuse(W, ": ", H, " query heads do not divide over ", KV, " kv heads");
  const int64_t R = query_start_loc.numel() - 1;
  if (R < 0 || (seq_lens && seq_lens->numel() != R))
    refuse(W, ": query_start_loc must have one entry more than there are requests");
  if (given_out && (given_out->sizes() != query.sizes() || (N > 0 && given_out->stride(2) != 1)))
    refuse(W, ": out must be ", query.sizes(), " with unit head-dim stride");
  const int index = query.get_device();
  same_device(W, index, {&key, &value, &query_start_loc, get(seq_lens), get(given_out)});
  no_autograd(W, {&query, &key, &value, get(given_out)});
  const c10::cuda::OptionalCUDAGuard guard(query.device());
  Tensor out = given_out ? *given_out : fresh(query.sizes(), at::kFloat, query);
  if (N == 0) return out;
  const Tensor q = tile_ready(query), k = tile_ready(key), v = tile_ready(value);
  const Tensor qsl = int32_of(query_start_loc);
  const Opt sl = seq_lens ? Opt(int32_of(*seq_lens)) : Opt();
  check(slmt_prompt_attention(q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1),
                              v.data_ptr(), v.stride(0), v.stride(1), tag(q.scalar_type()), data<int32_t>(qsl),
                              sl ? data<int32_t>(*sl) : nullptr, R, max_query_len, N, H, KV, D,
                              (float)(sm_scale ? *sm_scale : 1.0 / std::sqrt((double)D)), out.data_ptr(),
                              tag(out.scalar_type()), out.stride(0), out.stride(1), error_word(index),
                              c10::cuda::getCurrentCUDAStream(index).stream()),
        W);
  return out;
}

}  // namespace

PYBIND11_MODULE(_host, m) {
  m.def("set_error_words", [](py::object f) {
    g_error_word = std::move(f);
    g_error_words.fill(nullptr);
  });
  m.def("page_plan", &page_plan);
  m.def("rotary", &rotary);
  m.def("rotary_store", &rotary_store);
  m.def("dequantize_load", &dequantize_load);
  m.def("prompt_attention", &prompt_attention);
  // the function object must not outlive the interpreter
  py::module_::import("atexit").attr("register")(py::cpp_function([] { g_error_word = py::object(); }));
}
