// The operators of the paged cache (kv_append_, paged_attention, select_pages): checks, outputs, launches.  Part of
// torch_ops.cpp, inside its namespace.  Nothing turns to Python: these have no second form.
#pragma once

int as_int(int64_t x, const char* op) {
  TORCH_CHECK(x <= std::numeric_limits<int>::max(), op, ": a dimension of ", x, " is too large");
  return (int)x;
}

void check_tensor(const Tensor& t, const Tensor& with, int64_t dim, const char* op, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.layout() == at::kStrided, name, " must be a dense tensor");
  TORCH_CHECK(t.device() == with.device(), op, ": ", name, " must be on the device of the other operands");
  TORCH_CHECK(t.dim() == dim, op, ": ", name, " must have ", dim, " dimensions");
}

void check_ints(const Tensor& t, const Tensor& with, int64_t dim, const char* op, const char* name) {
  check_tensor(t, with, dim, op, name);
  TORCH_CHECK(t.scalar_type() == at::kInt, name, " must be int32");
  TORCH_CHECK(dim == 1 ? t.is_contiguous() : t.size(-1) <= 1 || t.stride(-1) == 1, name, " must have contiguous rows");
}

// Nothing here has a gradient: tokens are generated with it.
void check_no_gradient(const Tensor& t, const char* op) {
  TORCH_CHECK(!at::GradMode::is_enabled() || !t.requires_grad(), op, " has no gradient: call it under torch.no_grad()");
}

struct Strides {
  long long of[3];
  // (of a single token or head none is used)
  explicit Strides(const Tensor& t) : of{t.size(0) == 1 ? 0 : t.stride(0), t.size(1) == 1 ? 0 : t.stride(1), t.stride(2)} {}
};

// The cache as the C entry points take it; q is (rows, heads, head_dim).  keys / values undefined: bounds only.
iex_paged_cache paged_cache(const char* op, const Tensor& q, const Tensor& keys, const Tensor& values, const Tensor& table, const Tensor& lengths,
                            const std::optional<Tensor>& bounds, const std::optional<Tensor>& key_exponents, const std::optional<Tensor>& value_exponents) {
  iex_paged_cache c{};
  c.dtype = dtype_code(q.scalar_type());
  TORCH_CHECK(c.dtype == IEX_F16 || c.dtype == IEX_BF16, op, ": fp16 or bf16");
  check_ints(table, q, 2, op, "page_table");
  check_ints(lengths, q, 1, op, "lengths");
  TORCH_CHECK(lengths.size(0) == table.size(0), op, ": a length for every row of page_table (", lengths.size(0), ", ", table.size(0), ")");
  c.table = table.const_data_ptr<int>(), c.lengths = lengths.const_data_ptr<int>();
  c.seqs = as_int(table.size(0), op), c.table_width = as_int(table.size(1), op), c.table_stride = table.stride(0);
  if (keys.defined()) {
    check_tensor(keys, q, 4, op, "keys");
    check_tensor(values, q, 4, op, "values");
    TORCH_CHECK(values.sizes() == keys.sizes() && values.scalar_type() == keys.scalar_type(), op, ": keys and values must be alike");
    TORCH_CHECK(keys.size(3) == q.size(2), op, ": heads of ", q.size(2), " over a cache of heads of ", keys.size(3));
    for (const Tensor* t : {&keys, &values}) {
      check_no_gradient(*t, op);
      TORCH_CHECK(t->numel() == 0 || t->select(0, 0).is_contiguous(), op, ": a page of keys or values must be contiguous");
    }
    c.pages = as_int(keys.size(0), op), c.kv_heads = as_int(keys.size(1), op), c.page_size = as_int(keys.size(2), op), c.head_dim = as_int(keys.size(3), op);
    c.key_page_stride = keys.stride(0), c.value_page_stride = values.stride(0);
    c.keys = const_cast<void*>(keys.const_data_ptr()), c.values = const_cast<void*>(values.const_data_ptr());
    c.eight_bits = keys.scalar_type() == at::kFloat8_e4m3fn;
    TORCH_CHECK(c.eight_bits || keys.scalar_type() == q.scalar_type(), op, ": the cache must hold the operands' type or float8_e4m3fn");
    TORCH_CHECK(key_exponents.has_value() == (bool)c.eight_bits && value_exponents.has_value() == (bool)c.eight_bits, op,
                ": a float8_e4m3fn cache has exponents of keys and of values, another none");
    if (c.eight_bits) {
      for (const Tensor* t : {&*key_exponents, &*value_exponents}) {
        check_tensor(*t, q, 3, op, "exponents");
        TORCH_CHECK(t->scalar_type() == at::kByte && t->is_contiguous() && t->sizes() == keys.sizes().slice(0, 3), op,
                    ": exponents must be contiguous uint8 (pages, kv_heads, page_size)");
      }
      c.key_exponents = const_cast<uint8_t*>(key_exponents->const_data_ptr<uint8_t>());
      c.value_exponents = const_cast<uint8_t*>(value_exponents->const_data_ptr<uint8_t>());
    }
  }
  if (bounds) {
    check_tensor(*bounds, q, 4, op, "bounds");
    check_no_gradient(*bounds, op);
    if (!keys.defined()) c.pages = as_int(bounds->size(0), op), c.kv_heads = as_int(bounds->size(1), op), c.head_dim = as_int(bounds->size(3), op);
    TORCH_CHECK(bounds->scalar_type() == q.scalar_type() && bounds->is_contiguous() && bounds->size(0) == c.pages && bounds->size(1) == c.kv_heads &&
                    bounds->size(2) == 2 && bounds->size(3) == c.head_dim && c.head_dim == q.size(2),
                op, ": bounds must be contiguous (pages, kv_heads, 2, head_dim) of the operands' type");
    c.bounds = const_cast<void*>(bounds->const_data_ptr());
  }
  return c;
}

void changed(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

Tensor kv_append(const Tensor& k, const Tensor& v, const Tensor& keys, const Tensor& values, const Tensor& page_table, const Tensor& lengths,
                 const std::optional<Tensor>& offsets, const std::optional<Tensor>& q, const std::optional<Tensor>& rotation, bool interleaved,
                 const std::optional<Tensor>& bounds, const std::optional<Tensor>& key_exponents, const std::optional<Tensor>& value_exponents) {
  constexpr const char* op = "kv_append_";
  check_tensor(k, k, 3, op, "k");
  check_tensor(v, k, 3, op, "v");
  TORCH_CHECK(v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type(), op, ": k and v must be alike");
  const iex_paged_cache c = paged_cache(op, k, keys, values, page_table, lengths, bounds, key_exponents, value_exponents);
  TORCH_CHECK(k.size(1) == c.kv_heads, op, ": ", k.size(1), " heads over a cache of ", c.kv_heads);
  for (const Tensor* t : {&k, &v}) check_no_gradient(*t, op);
  if (offsets) {
    check_ints(*offsets, k, 1, op, "offsets");
    TORCH_CHECK(offsets->size(0) == (int64_t)c.seqs + 1, op, ": offsets must have an entry more than there are sequences");
  } else {
    TORCH_CHECK(k.size(0) == c.seqs, op, ": one token per sequence without offsets (", k.size(0), " tokens, ", c.seqs, " sequences)");
  }
  if (q) {
    check_tensor(*q, k, 3, op, "q");
    check_no_gradient(*q, op);
    TORCH_CHECK(q->scalar_type() == k.scalar_type() && q->size(0) == k.size(0) && q->size(2) == k.size(2), op, ": q must be (tokens, heads, head_dim) like k");
  }
  int rotary = 0, positions = 0;
  if (rotation) {
    check_tensor(*rotation, k, 2, op, "rotation");
    check_no_gradient(*rotation, op);
    TORCH_CHECK(rotation->scalar_type() == at::kFloat && rotation->is_contiguous(), op, ": rotation must be contiguous float32 (positions, rotated features)");
    positions = as_int(rotation->size(0), op), rotary = as_int(rotation->size(1), op);
  }
  const c10::DeviceGuard guard(k.device());
  const Tensor out = q ? at::empty_like(*q) : Tensor();
  const Strides ks(k), vs(v), qs(q ? *q : k), os(q ? out : k);
  check(iex_kv_append(&c, as_int(k.size(0), op), offsets ? offsets->const_data_ptr<int>() : nullptr, q ? as_int(q->size(1), op) : 0, k.const_data_ptr(), ks.of,
                      v.const_data_ptr(), vs.of, q ? q->const_data_ptr() : nullptr, qs.of, q ? out.data_ptr() : nullptr, os.of,
                      rotation ? rotation->const_data_ptr<float>() : nullptr, positions, rotary, interleaved, stream_of(k)),
        op);
  for (const Tensor* t : {&keys, &values}) changed(*t);
  for (const std::optional<Tensor>* t : {&bounds, &key_exponents, &value_exponents})
    if (*t) changed(**t);
  return out;
}

Tensor paged_attention(const Tensor& q, const Tensor& keys, const Tensor& values, const Tensor& page_table, const Tensor& lengths, std::optional<double> scale,
                       const std::optional<Tensor>& pages, const std::optional<Tensor>& key_exponents, const std::optional<Tensor>& value_exponents) {
  constexpr const char* op = "paged_attention";
  check_tensor(q, q, 3, op, "q");
  check_no_gradient(q, op);
  const iex_paged_cache c = paged_cache(op, q, keys, values, page_table, lengths, {}, key_exponents, value_exponents);
  TORCH_CHECK(q.size(0) == c.seqs, op, ": one token per sequence (", q.size(0), ", ", c.seqs, ")");
  int count = 0;
  if (pages) {
    check_ints(*pages, q, 3, op, "pages");
    TORCH_CHECK(pages->is_contiguous() && pages->size(0) == c.seqs && pages->size(1) == c.kv_heads, op, ": pages must be contiguous (sequences, kv_heads, count)");
    count = as_int(pages->size(2), op);
  }
  const c10::DeviceGuard guard(q.device());
  if ((pages && count == 0) || c.pages == 0) return at::zeros_like(q);   // nothing to attend to
  const Tensor out = at::empty_like(q);
  const int heads = as_int(q.size(1), op);
  const Strides qs(q), os(out);
  const size_t bytes = iex_paged_attention_workspace_bytes(&c, heads, count);
  const Tensor ws = workspace(bytes, q);
  check(iex_paged_attention(&c, heads, q.const_data_ptr(), qs.of, (float)scale.value_or(1.0 / std::sqrt((double)q.size(2))), pages ? pages->const_data_ptr<int>() : nullptr,
                            count, out.data_ptr(), os.of, ws.defined() ? ws.data_ptr() : nullptr, bytes, stream_of(q)),
        op);
  return out;
}

Tensor select_pages(const Tensor& q, const Tensor& bounds, const Tensor& page_table, const Tensor& lengths, int64_t page_size, int64_t count, int64_t first,
                    int64_t last) {
  constexpr const char* op = "select_pages";
  check_tensor(q, q, 3, op, "q");
  check_no_gradient(q, op);
  iex_paged_cache c = paged_cache(op, q, Tensor(), Tensor(), page_table, lengths, bounds, {}, {});
  c.page_size = as_int(page_size, op);
  TORCH_CHECK(q.size(0) == c.seqs, op, ": one token per sequence (", q.size(0), ", ", c.seqs, ")");
  const c10::DeviceGuard guard(q.device());
  TORCH_CHECK(count > 0, op, ": at least one page");
  const Tensor out = at::empty({q.size(0), c.kv_heads, count}, page_table.options());
  const size_t bytes = iex_select_pages_workspace_bytes(&c);
  const Tensor ws = workspace(bytes, q);
  const Strides qs(q);
  check(iex_select_pages(&c, as_int(q.size(1), op), q.const_data_ptr(), qs.of, as_int(count, op), as_int(first, op), as_int(last, op), out.data_ptr<int>(),
                         ws.defined() ? ws.data_ptr() : nullptr, bytes, stream_of(q)),
        op);
  return out;
}
