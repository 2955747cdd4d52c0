// memopt_C_packed.cpp — the packed-batch operators of the Python module:
// device page tables, rotary positions fused with the cache write, attention
// over packed prompts (additions; no reference counterpart).  Like
// memopt_C.cpp, a thin wrapper that checks tensors, allocates outputs and
// calls the C-ABI on the current stream; nothing here synchronises, so every
// call can be captured into a CUDA graph.
#include "torch_common.h"

#include <vector>

namespace {

using memopt_torch::aligned_contig;
using memopt_torch::aligned16;
using memopt_torch::check;
using memopt_torch::cur_stream;

void int32_cuda(const torch::Tensor& t, const char* who, const char* name, int64_t dim, const torch::Device& dev) {
  TORCH_CHECK(t.dim() == dim && t.scalar_type() == torch::kInt32, who, ": ", name, " must be int32 with ", dim,
              " dimension(s)");
  TORCH_CHECK(t.device() == dev, who, ": ", name, " must be on ", dev);
}

// Tensors that a call updates in place.
void int32_inplace(const torch::Tensor& t, const char* who, const char* name, int64_t dim, const torch::Device& dev) {
  int32_cuda(t, who, name, dim, dev);
  TORCH_CHECK(t.is_contiguous(), who, ": ", name, " is updated in place and must be contiguous");
}

// The bytes that a tensor spans, and whether two such spans meet.
struct Span {
  const char *begin = nullptr, *end = nullptr;
  Span() = default;
  explicit Span(const torch::Tensor& t) {
    const auto sizes = t.sizes(), strides = t.strides();
    int64_t last = 0;
    for (size_t d = 0; d < sizes.size(); ++d) {
      if (sizes[d] == 0) return;
      last += (sizes[d] - 1) * strides[d];
    }
    begin = static_cast<const char*>(t.data_ptr());
    end = begin + (last + 1) * t.element_size();
  }
  bool meets(const Span& o) const { return begin && o.begin && begin < o.end && o.begin < end; }
};
bool overlap(const torch::Tensor& a, const torch::Tensor& b) { return Span(a).meets(Span(b)); }

// A contiguous tensor inside a buffer: several outputs behind one allocation.
torch::Tensor part_of(const torch::Tensor& buf, int64_t at, at::IntArrayRef sizes) {
  auto t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(buf.storage()), buf.key_set(), buf.dtype());
  t.unsafeGetTensorImpl()->set_storage_offset(at);
  t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
  return t;
}

int to_int(int64_t v, const char* who, const char* name) {
  TORCH_CHECK(v >= 0 && v <= 0x7fffffff, who, ": ", name, " out of range");
  return static_cast<int>(v);
}

void no_grad_input(const torch::Tensor& t, const char* who) {
  TORCH_CHECK(!(at::GradMode::is_enabled() && t.requires_grad()), who,
              ": the operator has no gradient; detach its inputs or call it under torch.no_grad()");
}

int dtype_of(const torch::Tensor& t, const char* who) {
  TORCH_CHECK(t.scalar_type() == torch::kFloat16 || t.scalar_type() == torch::kBFloat16, who,
              ": tensors must be float16 or bfloat16");
  return t.scalar_type() == torch::kFloat16 ? MEMOPT_DTYPE_F16 : MEMOPT_DTYPE_BF16;
}

// Packed rows [T, heads, D]: any token stride that is a multiple of 8 elements
// (a slice of a fused projection), everything else is copied.
torch::Tensor packed_rows(const torch::Tensor& t) {
  const int64_t h = t.size(1), d = t.size(2);
  const bool ok = (t.stride(2) == 1 || d == 1) && (t.stride(1) == d || h == 1) &&
                  (t.size(0) <= 1 || (t.stride(0) % 8 == 0 && t.stride(0) >= h * d)) && aligned16(t);
  return ok ? t : aligned_contig(t);
}
int64_t row_stride(const torch::Tensor& t) { return t.size(0) <= 1 ? t.size(1) * t.size(2) : t.stride(0); }

void packed_check(const torch::Tensor& t, const char* who, const char* name, const torch::Tensor& like) {
  TORCH_CHECK(t.is_cuda(), who, ": ", name, " must be a CUDA tensor");
  TORCH_CHECK(t.device() == like.device(), who, ": ", name, " must be on ", like.device());
  TORCH_CHECK(t.dim() == 3, who, ": ", name, " must be 3-D [num_tokens, heads, head_dim]");
  TORCH_CHECK(t.scalar_type() == like.scalar_type(), who, ": ", name, " must have the query's dtype");
  TORCH_CHECK(t.size(0) == like.size(0), who, ": ", name, " token count mismatch");
  TORCH_CHECK(t.size(2) == like.size(2), who, ": ", name, " head_dim mismatch");
  no_grad_input(t, who);
}

struct PageTensors {
  int R, MB, NB, B;
};
// What a call updates meets nothing else that it takes: lens are the new or kept
// lengths, offsets the position offsets (null: none).
PageTensors page_checks(const char* who, const torch::Tensor& block_tables, const torch::Tensor& context_lens,
                        const torch::Tensor* offsets, const torch::Tensor& free_pages, const torch::Tensor& pool_state,
                        const torch::Tensor& rows, const torch::Tensor* lens, int block_size) {
  TORCH_CHECK(block_tables.is_cuda(), who, ": block_tables must be a CUDA tensor");
  const auto dev = block_tables.device();
  int32_inplace(block_tables, who, "block_tables", 2, dev);
  int32_inplace(context_lens, who, "context_lens", 1, dev);
  int32_inplace(free_pages, who, "free_pages", 1, dev);
  int32_inplace(pool_state, who, "pool_state", 1, dev);
  int32_cuda(rows, who, "rows", 1, dev);
  TORCH_CHECK(context_lens.size(0) == block_tables.size(0), who, ": context_lens length != block_tables rows");
  TORCH_CHECK(pool_state.size(0) == 4, who, ": pool_state must hold 4 values (head, count, status, ticket)");
  TORCH_CHECK(block_size > 0, who, ": block_size must be > 0");
  if (offsets) {
    int32_inplace(*offsets, who, "position_offsets", 1, dev);
    TORCH_CHECK(offsets->size(0) == block_tables.size(0), who, ": position_offsets length != block_tables rows");
  }
  TORCH_CHECK(!lens || lens->size(0) == rows.size(0), who, ": new_lens / keep_lens length != rows length");
  const Span none;
  const Span all[] = {Span(block_tables), Span(context_lens), Span(free_pages), Span(pool_state),
                      offsets ? Span(*offsets) : none, Span(rows), lens ? Span(*lens) : none};
  constexpr int kUpdated = 5, kAll = 7;
  for (int i = 0; i < kUpdated; ++i)
    for (int j = i + 1; j < kAll; ++j)
      TORCH_CHECK(!all[i].meets(all[j]), who, ": tensors that the call updates must not overlap the others");
  return {to_int(block_tables.size(0), who, "table rows"), to_int(block_tables.size(1), who, "table width"),
          to_int(free_pages.size(0), who, "number of pages"), to_int(rows.size(0), who, "batch")};
}

}  // namespace

namespace {

std::vector<torch::Tensor> reserve(const char* who, torch::Tensor block_tables, torch::Tensor context_lens,
                                   const torch::Tensor* position_offsets, torch::Tensor free_pages,
                                   torch::Tensor pool_state, torch::Tensor rows, torch::Tensor new_lens, int block_size,
                                   int64_t max_tokens, bool replace) {
  int32_cuda(new_lens, who, "new_lens", 1, block_tables.device());
  const PageTensors n = page_checks(who, block_tables, context_lens, position_offsets, free_pages, pool_state, rows,
                                    &new_lens, block_size);
  TORCH_CHECK(max_tokens >= 0 && max_tokens <= 0x7fffffff, who, ": max_tokens out of range");
  rows = rows.contiguous();
  new_lens = new_lens.contiguous();
  const at::cuda::CUDAGuard g(block_tables.device());
  // One allocation behind the outputs (an allocation each costs the host
  // more than the launch), every one 16-byte aligned.
  auto up4 = [](int64_t v) { return (v + 3) & ~int64_t(3); };
  const int64_t at_pos = up4(max_tokens), at_tables = at_pos + up4(max_tokens);
  const int64_t at_cu = at_tables + up4(static_cast<int64_t>(n.B) * n.MB), at_lens = at_cu + up4(n.B + 1);
  const int64_t at_attend = at_lens + up4(n.B);
  const auto buf = torch::empty({position_offsets ? at_attend + n.B : at_lens + n.B}, block_tables.options());
  auto slots = part_of(buf, 0, {max_tokens}), positions = part_of(buf, at_pos, {max_tokens});
  auto tables = part_of(buf, at_tables, {n.B, n.MB}), cu = part_of(buf, at_cu, {n.B + 1});
  auto lens = part_of(buf, at_lens, {n.B});
  auto p = [](const torch::Tensor& t) { return t.data_ptr<int32_t>(); };
  if (!position_offsets) {
    check(memopt_reserve_slots(p(block_tables), p(context_lens), n.R, n.MB, p(free_pages), n.NB, p(pool_state),
                               p(rows), p(new_lens), n.B, block_size, max_tokens, p(cu), p(slots), p(positions),
                               p(tables), p(lens), cur_stream()),
          who);
    return {cu, slots, positions, tables, lens};
  }
  auto attend = part_of(buf, at_attend, {n.B});
  check(memopt_reserve_rows(p(block_tables), p(context_lens), p(*position_offsets), n.R, n.MB, p(free_pages), n.NB,
                            p(pool_state), p(rows), p(new_lens), n.B, block_size, max_tokens, replace ? 1 : 0, p(cu),
                            p(slots), p(positions), p(tables), p(lens), p(attend), cur_stream()),
        who);
  return {cu, slots, positions, tables, lens, attend};
}

}  // namespace

std::vector<torch::Tensor> reserve_slots(torch::Tensor block_tables, torch::Tensor context_lens,
                                         torch::Tensor free_pages, torch::Tensor pool_state, torch::Tensor rows,
                                         torch::Tensor new_lens, int block_size, int64_t max_tokens) {
  return reserve("reserve_slots", block_tables, context_lens, nullptr, free_pages, pool_state, rows, new_lens,
                 block_size, max_tokens, false);
}

std::vector<torch::Tensor> reserve_rows(torch::Tensor block_tables, torch::Tensor context_lens,
                                        torch::Tensor position_offsets, torch::Tensor free_pages,
                                        torch::Tensor pool_state, torch::Tensor rows, torch::Tensor new_lens,
                                        int block_size, int64_t max_tokens, bool replace) {
  return reserve("reserve_rows", block_tables, context_lens, &position_offsets, free_pages, pool_state, rows, new_lens,
                 block_size, max_tokens, replace);
}

void truncate_rows(torch::Tensor block_tables, torch::Tensor context_lens, torch::Tensor free_pages,
                   torch::Tensor pool_state, torch::Tensor rows, c10::optional<torch::Tensor> keep_lens,
                   int block_size) {
  const char* who = "truncate_rows";
  if (keep_lens.has_value()) int32_cuda(*keep_lens, who, "keep_lens", 1, block_tables.device());
  const PageTensors n = page_checks(who, block_tables, context_lens, nullptr, free_pages, pool_state, rows,
                                    keep_lens.has_value() ? &*keep_lens : nullptr, block_size);
  torch::Tensor keep;
  if (keep_lens.has_value()) keep = keep_lens->contiguous();
  rows = rows.contiguous();
  const at::cuda::CUDAGuard g(block_tables.device());
  check(memopt_truncate_rows(block_tables.data_ptr<int32_t>(), context_lens.data_ptr<int32_t>(), n.R, n.MB,
                             free_pages.data_ptr<int32_t>(), n.NB, pool_state.data_ptr<int32_t>(),
                             rows.data_ptr<int32_t>(), keep.defined() ? keep.data_ptr<int32_t>() : nullptr, n.B,
                             block_size, cur_stream()),
        who);
}

namespace {

std::vector<torch::Tensor> rotary(const char* who, torch::Tensor query, torch::Tensor keys,
                                  const torch::Tensor* values, torch::Tensor positions, torch::Tensor inv_freq,
                                  const std::vector<int64_t>& sections, const torch::Tensor* slot_mapping,
                                  const torch::Tensor* key_cache, const torch::Tensor* value_cache,
                                  bool interleaved) {
  TORCH_CHECK(query.is_cuda(), who, ": query must be a CUDA tensor");
  TORCH_CHECK(query.dim() == 3, who, ": query must be 3-D [num_tokens, num_heads, head_dim]");
  const int dtype = dtype_of(query, who);
  no_grad_input(query, who);
  packed_check(keys, who, "keys", query);
  const int64_t T = query.size(0), A = static_cast<int64_t>(sections.size());
  const int H = to_int(query.size(1), who, "num_heads"), KVH = to_int(keys.size(1), who, "num_kv_heads");
  const int D = to_int(query.size(2), who, "head_dim");
  TORCH_CHECK(A >= 1 && A <= 4, who, ": sections must name 1 to 4 axes");
  TORCH_CHECK(positions.scalar_type() == torch::kInt32, who, ": positions must be int32");
  TORCH_CHECK(positions.device() == query.device(), who, ": positions must be on ", query.device());
  TORCH_CHECK((positions.dim() == 2 && positions.size(0) == A && positions.size(1) == T) ||
                  (positions.dim() == 1 && A == 1 && positions.size(0) == T),
              who, ": positions must be [num_axes, num_tokens] (or [num_tokens] for one axis)");
  TORCH_CHECK(inv_freq.dim() == 1 && inv_freq.scalar_type() == torch::kFloat64, who,
              ": inv_freq must be float64 [num_pairs]");
  TORCH_CHECK(inv_freq.device() == query.device(), who, ": inv_freq must be on ", query.device());
  std::vector<int32_t> sec;
  for (int64_t s : sections) sec.push_back(to_int(s, who, "a section"));
  const int P = to_int(inv_freq.size(0), who, "num_pairs");
  int64_t NB = 0;
  int BS = 1;
  torch::Tensor v, slots;
  if (slot_mapping) {
    packed_check(*values, who, "values", query);
    TORCH_CHECK(values->size(1) == KVH, who, ": keys/values num_heads mismatch");
    int32_cuda(*slot_mapping, who, "slot_mapping", 1, query.device());
    TORCH_CHECK(slot_mapping->size(0) == T, who, ": slot_mapping length != num_tokens");
    for (const auto* c : {key_cache, value_cache}) {
      TORCH_CHECK(c->is_cuda() && c->device() == query.device() && c->dim() == 4 &&
                      c->scalar_type() == torch::kFloat16 && c->is_contiguous() && aligned16(*c),
                  who, ": caches must be contiguous fp16 [num_blocks, block_size, num_kv_heads, head_dim] on the "
                       "query's device");
      TORCH_CHECK(c->size(2) == KVH && c->size(3) == D, who, ": cache heads or head_dim do not match the keys");
    }
    TORCH_CHECK(key_cache->sizes() == value_cache->sizes(), who, ": key_cache and value_cache shapes differ");
    const Span kc(*key_cache), vc(*value_cache), in[] = {Span(query), Span(keys), Span(*values)};
    TORCH_CHECK(!kc.meets(vc), who, ": key_cache and value_cache overlap");
    for (const Span& x : in)
      TORCH_CHECK(!x.meets(kc) && !x.meets(vc), who, ": the caches must not overlap the inputs");
    NB = key_cache->size(0);
    BS = to_int(key_cache->size(1), who, "block_size");
    slots = slot_mapping->contiguous();
    v = packed_rows(*values);
  }
  const at::cuda::CUDAGuard g(query.device());
  // Decode steps wait for the host: one allocation behind both outputs (32 tokens of
  // 32/8 heads: 6.9 -> 6.2 us a call).  Larger ones stay apart, so that either can be
  // freed without the other.
  torch::Tensor q_out, k_out;
  if (query.numel() + keys.numel() <= (1 << 19) && query.numel() % 8 == 0) {
    const auto buf = torch::empty({query.numel() + keys.numel()}, query.options());
    q_out = part_of(buf, 0, query.sizes());
    k_out = part_of(buf, query.numel(), keys.sizes());
  } else {
    q_out = torch::empty(query.sizes(), query.options());
    k_out = torch::empty(keys.sizes(), keys.options());
  }
  if (T == 0 || H + KVH == 0) return {q_out, k_out};
  auto q = packed_rows(query), k = packed_rows(keys);
  positions = positions.contiguous();
  inv_freq = inv_freq.contiguous();
  check(memopt_rotary_write_cache(
            q.data_ptr(), row_stride(q), k.data_ptr(), row_stride(k), v.defined() ? v.data_ptr() : nullptr,
            v.defined() ? row_stride(v) : 0, dtype, T, H, KVH, D, positions.data_ptr<int32_t>(), static_cast<int>(A),
            sec.data(), inv_freq.data_ptr<double>(), P, interleaved ? 1 : 0, q_out.data_ptr(), k_out.data_ptr(),
            slots.defined() ? slots.data_ptr<int32_t>() : nullptr, slots.defined() ? key_cache->data_ptr() : nullptr,
            slots.defined() ? value_cache->data_ptr() : nullptr, NB, BS, cur_stream()),
        who);
  return {q_out, k_out};
}

}  // namespace

std::vector<torch::Tensor> apply_rotary(torch::Tensor query, torch::Tensor keys, torch::Tensor positions,
                                        torch::Tensor inv_freq, std::vector<int64_t> sections, bool interleaved) {
  return rotary("apply_rotary", query, keys, nullptr, positions, inv_freq, sections, nullptr, nullptr, nullptr,
                interleaved);
}

std::vector<torch::Tensor> rotary_write_cache(torch::Tensor query, torch::Tensor keys, torch::Tensor values,
                                              torch::Tensor positions, torch::Tensor inv_freq,
                                              std::vector<int64_t> sections, torch::Tensor slot_mapping,
                                              torch::Tensor key_cache, torch::Tensor value_cache, bool interleaved) {
  return rotary("rotary_write_cache", query, keys, &values, positions, inv_freq, sections, &slot_mapping, &key_cache,
                &value_cache, interleaved);
}

torch::Tensor packed_attention(torch::Tensor query, torch::Tensor keys, torch::Tensor values,
                               torch::Tensor cu_seqlens, int64_t max_seqlen, int64_t window_size, bool causal,
                               c10::optional<torch::Tensor> out_, bool zero_rest) {
  const char* who = "packed_attention";
  TORCH_CHECK(query.is_cuda(), who, ": query must be a CUDA tensor");
  TORCH_CHECK(query.dim() == 3, who, ": query must be 3-D [num_tokens, num_heads, head_dim]");
  const int dtype = dtype_of(query, who);
  no_grad_input(query, who);
  packed_check(keys, who, "keys", query);
  packed_check(values, who, "values", query);
  int32_cuda(cu_seqlens, who, "cu_seqlens", 1, query.device());
  TORCH_CHECK(cu_seqlens.size(0) >= 1, who, ": cu_seqlens must hold num_seqs + 1 values");
  const int64_t T = query.size(0);
  const int S = to_int(cu_seqlens.size(0) - 1, who, "num_seqs");
  const int H = to_int(query.size(1), who, "num_heads"), KVH = to_int(keys.size(1), who, "num_kv_heads");
  const int D = to_int(query.size(2), who, "head_dim");
  TORCH_CHECK(values.size(1) == KVH, who, ": keys/values num_heads mismatch");
  TORCH_CHECK(KVH > 0 && H > 0 && H % KVH == 0, who, ": keys num_heads ", KVH, " does not divide query num_heads ", H);
  TORCH_CHECK(max_seqlen >= 0 && max_seqlen <= 0x7fffffff, who, ": max_seqlen out of range");
  const at::cuda::CUDAGuard g(query.device());
  torch::Tensor out;
  if (out_.has_value()) {
    out = *out_;
    TORCH_CHECK(out.sizes() == query.sizes() && out.scalar_type() == query.scalar_type() &&
                    out.device() == query.device() && out.is_contiguous() && (out.numel() == 0 || aligned16(out)),
                who, ": out must be a contiguous 16-byte aligned tensor of the query's shape, dtype and device");
    TORCH_CHECK(!overlap(out, query) && !overlap(out, keys) && !overlap(out, values), who,
                ": out must not overlap the inputs");
  } else {
    out = torch::empty(query.sizes(), query.options());
  }
  if (T == 0 || (S == 0 && !zero_rest)) return out;
  auto q = packed_rows(query), k = packed_rows(keys), v = packed_rows(values);
  cu_seqlens = cu_seqlens.contiguous();
  const int window = window_size <= 0 || window_size > 0x7fffffff ? 0 : static_cast<int>(window_size);
  const size_t ws_bytes = memopt_packed_attention_workspace_size(S, T, static_cast<int>(max_seqlen), H, KVH, D, window,
                                                                 causal ? 1 : 0);
  torch::Tensor ws;
  if (ws_bytes > 0) ws = torch::empty({static_cast<int64_t>(ws_bytes)}, query.options().dtype(torch::kUInt8));
  check(memopt_packed_attention_ex(q.data_ptr(), row_stride(q), k.data_ptr(), row_stride(k), v.data_ptr(),
                                   row_stride(v), dtype, cu_seqlens.data_ptr<int32_t>(), S, T,
                                   static_cast<int>(max_seqlen), H, KVH, D, window, causal ? 1 : 0, zero_rest ? 1 : 0,
                                   out.data_ptr(), ws_bytes ? ws.data_ptr() : nullptr, ws_bytes, cur_stream()),
        who);
  return out;
}

void bind_packed(pybind11::module_& m) {
  namespace py = pybind11;
  m.def("reserve_slots", &reserve_slots,
        "Reserve new_lens[b] tokens for table row rows[b]: pages from the free ring, and the batch's cu_seqlens, "
        "slot_mapping, positions, block tables and context lengths",
        py::arg("block_tables"), py::arg("context_lens"), py::arg("free_pages"), py::arg("pool_state"),
        py::arg("rows"), py::arg("new_lens"), py::arg("block_size"), py::arg("max_tokens"));
  m.def("reserve_rows", &reserve_rows,
        "reserve_slots over rows that may have been evicted from: positions are index + position_offsets[row]; with "
        "replace the rows begin anew, unless the call is refused; also returns the lengths to attend over, 0 if refused",
        py::arg("block_tables"), py::arg("context_lens"), py::arg("position_offsets"), py::arg("free_pages"),
        py::arg("pool_state"), py::arg("rows"), py::arg("new_lens"), py::arg("block_size"), py::arg("max_tokens"),
        py::arg("replace") = false);
  m.def("truncate_rows", &truncate_rows,
        "Cut table row rows[b] to its first keep_lens[b] tokens (None: to nothing) and return the pages to the ring",
        py::arg("block_tables"), py::arg("context_lens"), py::arg("free_pages"), py::arg("pool_state"),
        py::arg("rows"), py::arg("keep_lens"), py::arg("block_size"));
  m.def("apply_rotary", &apply_rotary, "Rotary positions with 1 to 4 axes; returns (query, keys) rotated",
        py::arg("query"), py::arg("keys"), py::arg("positions"), py::arg("inv_freq"), py::arg("sections"),
        py::arg("interleaved") = false);
  m.def("rotary_write_cache", &rotary_write_cache,
        "apply_rotary fused with the write of the rotated keys and the values into an fp16 pool via slot_mapping",
        py::arg("query"), py::arg("keys"), py::arg("values"), py::arg("positions"), py::arg("inv_freq"),
        py::arg("sections"), py::arg("slot_mapping"), py::arg("key_cache"), py::arg("value_cache"),
        py::arg("interleaved") = false);
  m.def("packed_attention", &packed_attention,
        "Attention inside each sequence of a packed batch, grouped heads; rows outside every sequence are left as they "
        "are, or with zero_rest those from cu_seqlens[-1] on become 0",
        py::arg("query"), py::arg("keys"), py::arg("values"), py::arg("cu_seqlens"), py::arg("max_seqlen"),
        py::arg("window_size") = -1, py::arg("causal") = true, py::arg("out") = py::none(),
        py::arg("zero_rest") = false);
}
