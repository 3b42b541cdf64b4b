// mxq_py.cpp -- the serving calls' Python side: the checks of the arguments, the
// outputs' allocation and the call into libmxq.so (include/mxq.h), without a
// detour over ctypes.  These calls take the GPU 3 to 10 microseconds where a
// step is small, and the same work in Python took 17 to 22.  All arithmetic is the
// library's; errors are raised as cpu_model_b200._lib.check raises them.
#include <torch/extension.h>

#include <c10/cuda/CUDAStream.h>

#include "mxq.h"

namespace {

using at::Tensor;
using c10::optional;

[[noreturn]] void refuse(const std::string& what) { throw py::value_error(what); }

const char* type_name(at::ScalarType t) { return c10::toString(t); }

void want(const Tensor& t, at::ScalarType type, const char* name) {
  if (!t.defined() || !t.is_cuda()) refuse(std::string(name) + " must be a CUDA tensor");
  if (t.scalar_type() != type)
    refuse(std::string(name) + " must be " + type_name(type) + ", got " + type_name(t.scalar_type()));
  if (!t.is_contiguous()) refuse(std::string(name) + " must be contiguous");
}

int row_type(const Tensor& t, const char* name) {
  if (!t.defined() || !t.is_cuda()) refuse(std::string(name) + " must be a CUDA tensor");
  switch (t.scalar_type()) {
    case at::kFloat: return MXQ_DT_F32;
    case at::kBFloat16: return MXQ_DT_BF16;
    case at::kHalf: return MXQ_DT_F16;
    default:
      refuse(std::string(name) + " must be float32, bfloat16 or float16, got " + type_name(t.scalar_type()));
  }
}

// Elements from one row to the next; the dimensions of a row lie side by side.
int64_t row_stride(const Tensor& t, const char* name) {
  int64_t inner = 1;
  for (int64_t d = t.dim() - 1; d > 0; --d) {
    if (t.size(d) != 1 && t.stride(d) != inner) refuse(std::string(name) + ": only rows may have a stride");
    inner *= t.size(d);
  }
  return t.size(0) > 1 ? t.stride(0) : std::max(inner, t.stride(0));
}

void same_device(const Tensor& first, std::initializer_list<const Tensor*> others) {
  for (const Tensor* t : others)
    if (t && t->defined() && t->get_device() != first.get_device()) refuse("tensors lie on different devices");
}

// The outputs and their views are made below autograd: nothing here is recorded.
using Below = at::AutoDispatchBelowADInplaceOrView;

// Tensors that a call has written into: a graph that saved one is told.
void written(std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

// The context, bound to the current stream of the tensors' device.
mxq_ctx bind(uintptr_t ctx, const Tensor& on) {
  mxq_ctx c = reinterpret_cast<mxq_ctx>(ctx);
  mxq_set_stream(c, c10::cuda::getCurrentCUDAStream(on.get_device()).stream());
  return c;
}

void check(int rc, uintptr_t ctx) {
  if (rc == MXQ_OK) return;
  py::object vp = py::module_::import("ctypes").attr("c_void_p")(ctx);
  py::module_::import("cpu_model_b200._lib").attr("check")(rc, vp);
}

template <typename T>
T* ptr(const Tensor& t) {
  return static_cast<T*>(t.data_ptr());
}
template <typename T>
T* ptr(const optional<Tensor>& t) {
  return t ? static_cast<T*>(t->data_ptr()) : nullptr;
}
const Tensor* ref(const optional<Tensor>& t) { return t ? &*t : nullptr; }

constexpr int64_t kBlock = MXQ_KV_BLOCK;

struct KVCache {
  Tensor k, v, k_scale, v_scale;
  mxq_kv_cache c;
  KVCache(const Tensor& k_, const Tensor& v_, const Tensor& ks, const Tensor& vs) : k(k_), v(v_), k_scale(ks), v_scale(vs) {
    want(k, at::kChar, "k");
    want(v, at::kChar, "v");
    want(k_scale, at::kByte, "k_scale");
    want(v_scale, at::kByte, "v_scale");
    if (k.dim() != 5 || k.size(3) != kBlock) refuse("k must be [n_pages][heads][blocks][32][head_dim]");
    const int64_t n = k.size(0), h = k.size(1), nb = k.size(2), d = k.size(4);
    if (k.numel() == 0) refuse("kv cache: no pages, heads, blocks or dimensions");
    if (v.sizes() != at::IntArrayRef({n, h, nb, d / 2, 4, 2, 8}))
      refuse("v must be [n_pages][heads][blocks][head_dim / 2][4][2][8]");
    if (k_scale.sizes() != at::IntArrayRef({n, h, nb}) || v_scale.sizes() != at::IntArrayRef({n, h, nb}))
      refuse("k_scale and v_scale must be [n_pages][heads][blocks]");
    same_device(k, {&v, &k_scale, &v_scale});
    if (n > INT32_MAX || h > INT32_MAX || nb > INT32_MAX / kBlock || d > INT32_MAX) refuse("kv cache: too large");
    c = mxq_kv_cache{nullptr, nullptr, nullptr, nullptr, (int)n, (int)(nb * kBlock), (int)h, (int)d};
  }
  // Where the tensors' memory is now: they are the caller's, who may have given them another.
  mxq_kv_cache now() const {
    const int64_t blocks = (int64_t)c.n_pages * c.n_kv_heads * (c.page_size / kBlock), values = blocks * kBlock * c.head_dim;
    const std::pair<const Tensor*, int64_t> all[] = {{&k, values}, {&v, values}, {&k_scale, blocks}, {&v_scale, blocks}};
    for (const auto& [t, n] : all)
      if (t->numel() != n || !t->is_cuda() || !t->is_contiguous() || t->element_size() != 1)
        refuse("kv cache: a tensor is not what the cache was made of");
    mxq_kv_cache at = c;
    at.k = k.data_ptr();
    at.v = v.data_ptr();
    at.k_scale = ptr<uint8_t>(k_scale);
    at.v_scale = ptr<uint8_t>(v_scale);
    return at;
  }
};

void want_table(const Tensor& table, int64_t rows) {
  want(table, at::kInt, "table");
  if (table.dim() != 2 || table.size(0) != rows) refuse("table must be [n_requests][max_pages]");
}

py::tuple kv_plan(uintptr_t ctx, const Tensor& past, const Tensor& add, int64_t page_size, const Tensor& table,
                  const Tensor& free_pages, const Tensor& free_count, int64_t n, bool in_place) {
  const Below below;
  want(past, at::kInt, "past");
  want(add, at::kInt, "new");
  want(free_pages, at::kInt, "free_pages");
  want(free_count, at::kInt, "free_count");
  const int64_t r = past.numel();
  if (add.numel() != r || free_count.numel() != 1)
    refuse("kv_plan: past and new must hold one length a request, free_count one number");
  want_table(table, r);
  if (n < 0) refuse("kv_plan: n_tokens is negative");
  if (page_size < 0) refuse("kv_plan: bad page size");
  same_device(past, {&add, &table, &free_pages, &free_count});
  // one allocation for the maps and the two numbers
  const int64_t rest = 3 * n + r + 1;
  const Tensor buf = at::empty({rest + (in_place ? 1 : 2 + r)}, past.options());
  int32_t* at = ptr<int32_t>(buf);
  const Tensor left = in_place ? free_count : buf.narrow(0, rest + 1, 1);
  const Tensor len = in_place ? past : buf.narrow(0, rest + 2, r);
  check(mxq_kv_plan(bind(ctx, past), ptr<int32_t>(past), ptr<int32_t>(add), r, page_size, ptr<int32_t>(table),
                    table.size(1), ptr<int32_t>(free_pages), free_pages.numel(), ptr<int32_t>(free_count),
                    in_place ? ptr<int32_t>(past) : at + rest + 2, at + 3 * n, at, at + n, at + 2 * n, n,
                    in_place ? ptr<int32_t>(free_count) : at + rest + 1, at + rest),
        ctx);
  written({&table});
  if (in_place) written({&past, &free_count});
  return py::make_tuple(len, buf.narrow(0, 3 * n, r + 1), buf.narrow(0, 0, n), buf.narrow(0, n, n), buf.narrow(0, 2 * n, n),
                        left, buf.narrow(0, rest, 1));
}

void kv_release(uintptr_t ctx, const Tensor& done, const Tensor& lengths, int64_t page_size, const Tensor& table,
                const Tensor& free_pages, const Tensor& free_count) {
  if (done.scalar_type() != at::kBool) want(done, at::kByte, "done");
  else want(done, at::kBool, "done");
  want(lengths, at::kInt, "lengths");
  want(free_pages, at::kInt, "free_pages");
  want(free_count, at::kInt, "free_count");
  const int64_t r = lengths.numel();
  if (done.numel() != r || free_count.numel() != 1)
    refuse("kv_release: done and lengths must hold one value a request, free_count one number");
  want_table(table, r);
  if (page_size < 0) refuse("kv_release: bad page size");
  same_device(lengths, {&done, &table, &free_pages, &free_count});
  check(mxq_kv_release(bind(ctx, lengths), ptr<uint8_t>(done), ptr<int32_t>(lengths), r, page_size, ptr<int32_t>(table),
                       table.size(1), ptr<int32_t>(free_pages), free_pages.numel(), ptr<int32_t>(free_count)),
        ctx);
  written({&lengths, &table, &free_pages, &free_count});
}

void kv_append(uintptr_t ctx, const KVCache& cache, const Tensor& k, const Tensor& v, const Tensor& slots) {
  const int dt = row_type(k, "k");
  want(slots, at::kInt, "slots");
  if (v.scalar_type() != k.scalar_type() || v.sizes() != k.sizes() || !v.is_cuda())
    refuse("kv_append: k and v must have one type and shape");
  const int64_t n = slots.numel();
  if (k.sizes() != at::IntArrayRef({n, cache.c.n_kv_heads, cache.c.head_dim}))
    refuse("kv_append: k and v must be [n][heads][head_dim] of the cache with one slot a row");
  same_device(cache.k, {&cache.v, &cache.k_scale, &cache.v_scale, &k, &v, &slots});
  const mxq_kv_cache c = cache.now();
  check(mxq_kv_append_strided(bind(ctx, k), &c, dt, k.data_ptr(), row_stride(k, "k"), v.data_ptr(), row_stride(v, "v"),
                              ptr<int32_t>(slots), n),
        ctx);
  written({&cache.k, &cache.v, &cache.k_scale, &cache.v_scale});
}

py::tuple kv_read(uintptr_t ctx, const KVCache& cache, const Tensor& slots, at::ScalarType type) {
  const Below below;
  want(slots, at::kInt, "slots");
  if (type != at::kFloat && type != at::kBFloat16 && type != at::kHalf)
    refuse(std::string("kv_read: float32, bfloat16 or float16, got ") + type_name(type));
  same_device(cache.k, {&cache.v, &cache.k_scale, &cache.v_scale, &slots});
  const mxq_kv_cache c = cache.now();
  const int64_t n = slots.numel();
  const Tensor k = at::empty({n, cache.c.n_kv_heads, cache.c.head_dim}, slots.options().dtype(type));
  const Tensor v = at::empty_like(k);
  check(mxq_kv_read(bind(ctx, slots), &c, ptr<int32_t>(slots), n, row_type(k, "k"), k.data_ptr(), v.data_ptr()), ctx);
  return py::make_tuple(k, v);
}

py::tuple kv_attention(uintptr_t ctx, const Tensor& q, const KVCache& cache, const Tensor& table, const Tensor& ctx_len,
                       const Tensor& cu, optional<double> scale, optional<int64_t> max_new, bool want_lse) {
  const Below below;
  const int dt = row_type(q, "q");
  want(ctx_len, at::kInt, "ctx_len");
  want(cu, at::kInt, "cu");
  const int64_t r = ctx_len.numel();
  want_table(table, r);
  const int64_t d = cache.c.head_dim;
  if (q.dim() != 3 || q.size(2) != d || q.size(1) % cache.c.n_kv_heads)
    refuse("kv_attention: q must be [n][heads][head_dim] with heads a multiple of the cache's");
  if (cu.numel() != r + 1) refuse("kv_attention: cu must hold n_requests + 1 offsets");
  if (max_new && *max_new < 1) refuse("kv_attention: max_new must be positive");
  same_device(cache.k, {&cache.v, &cache.k_scale, &cache.v_scale, &q, &table, &ctx_len, &cu});
  const mxq_kv_cache c = cache.now();
  const int64_t n = q.size(0), hq = q.size(1);
  const Tensor out = at::empty({n, hq, d}, q.options());
  optional<Tensor> lse;
  if (want_lse) lse = at::empty({n, hq}, q.options().dtype(at::kFloat));
  check(mxq_kv_attention(bind(ctx, q), &c, dt, q.data_ptr(), row_stride(q, "q"), n, hq, ptr<int32_t>(table),
                         table.size(1), ptr<int32_t>(ctx_len), ptr<int32_t>(cu), r,
                         max_new ? *max_new : std::max<int64_t>(n, 1),
                         (float)(scale ? *scale : 1.0 / std::sqrt((double)d)), out.data_ptr(), ptr<float>(lse)),
        ctx);
  return py::make_tuple(out, lse);
}

int logits_rows(const Tensor& logits, const Tensor& targets) {
  const int dt = row_type(logits, "logits");
  want(targets, at::kInt, "targets");
  if (logits.dim() != 2 || targets.numel() != logits.size(0))
    refuse("logits must be [rows][vocab] with one target a row");
  return dt;
}

py::tuple token_logprobs(uintptr_t ctx, const Tensor& logits, const Tensor& targets, int64_t top_k) {
  const Below below;
  const int dt = logits_rows(logits, targets);
  const int64_t n = logits.size(0), v = logits.size(1);
  if (top_k < 0 || top_k > std::min<int64_t>(v, MXQ_TOPK_MAX))
    refuse("token_logprobs: top_k must be in [0, min(32, vocab)]");
  same_device(logits, {&targets});
  const auto f32 = logits.options().dtype(at::kFloat);
  const Tensor logp = at::empty({n}, f32), entropy = at::empty({n}, f32), lse = at::empty({n}, f32);
  optional<Tensor> top, ids;
  if (top_k) {
    top = at::empty({n, top_k}, f32);
    ids = at::empty({n, top_k}, targets.options());
  }
  check(mxq_token_logprobs(bind(ctx, logits), dt, logits.data_ptr(), row_stride(logits, "logits"), n, v,
                           ptr<int32_t>(targets), top_k, ptr<float>(logp), ptr<float>(entropy), ptr<float>(lse),
                           ptr<float>(top), ptr<int32_t>(ids)),
        ctx);
  return py::make_tuple(logp, entropy, lse, top, ids);
}

Tensor token_logprobs_grad(uintptr_t ctx, const Tensor& logits, const Tensor& targets, const Tensor& lse,
                           const optional<Tensor>& entropy, const optional<Tensor>& dlogp, const optional<Tensor>& dentropy,
                           const optional<Tensor>& out) {
  const Below below;
  const int dt = logits_rows(logits, targets);
  const int64_t n = logits.size(0), v = logits.size(1);
  auto a_row = [&](const Tensor& t, const char* name) {
    want(t, at::kFloat, name);
    if (t.numel() != n) refuse(std::string("token_logprobs_grad: ") + name + " must hold one value a row");
  };
  a_row(lse, "lse");
  if (entropy) a_row(*entropy, "entropy");
  if (dlogp) a_row(*dlogp, "dlogp");
  if (dentropy) a_row(*dentropy, "dentropy");
  if (dentropy && !entropy) refuse("token_logprobs_grad: dentropy needs the entropy");
  if (out && (out->scalar_type() != logits.scalar_type() || out->sizes() != logits.sizes() || !out->is_cuda()))
    refuse("token_logprobs_grad: out must have the logits' type and shape");
  const Tensor g = out ? *out : at::empty({n, v}, logits.options());
  same_device(logits, {&targets, &lse, ref(entropy), ref(dlogp), ref(dentropy), &g});
  check(mxq_token_logprobs_grad(bind(ctx, logits), dt, logits.data_ptr(), row_stride(logits, "logits"), n, v,
                                ptr<int32_t>(targets), ptr<float>(lse), ptr<float>(entropy), ptr<float>(dlogp),
                                ptr<float>(dentropy), g.data_ptr(), row_stride(g, "out")),
        ctx);
  if (out) written({&g});
  return g;
}

}  // namespace

PYBIND11_MODULE(_serve, m) {
  m.doc() = "The serving calls of libmxq.so over torch tensors (see cpu_model_b200.mx).";
  py::class_<KVCache>(m, "KVCache",
                      "A paged 8-bit K/V cache (mxq_kv_cache): int8 values, one E8M0 scale for each block of 32 tokens and "
                      "head.  The four tensors are the caller's: k int8 [n_pages][H][page/32][32][D], v int8 "
                      "[n_pages][H][page/32][D/2][4][2][8], k_scale and v_scale uint8 [n_pages][H][page/32].")
      .def(py::init<const Tensor&, const Tensor&, const Tensor&, const Tensor&>(), py::arg("k"), py::arg("v"),
           py::arg("k_scale"), py::arg("v_scale"))
      .def_readonly("k", &KVCache::k)
      .def_readonly("v", &KVCache::v)
      .def_readonly("k_scale", &KVCache::k_scale)
      .def_readonly("v_scale", &KVCache::v_scale)
      .def_property_readonly("n_pages", [](const KVCache& c) { return c.c.n_pages; })
      .def_property_readonly("page_size", [](const KVCache& c) { return c.c.page_size; })
      .def_property_readonly("n_kv_heads", [](const KVCache& c) { return c.c.n_kv_heads; })
      .def_property_readonly("head_dim", [](const KVCache& c) { return c.c.head_dim; });
  m.def("kv_plan", &kv_plan);
  m.def("kv_release", &kv_release);
  m.def("kv_append", &kv_append);
  m.def("kv_read", &kv_read);
  m.def("kv_attention", &kv_attention);
  m.def("token_logprobs", &token_logprobs);
  m.def("token_logprobs_grad", &token_logprobs_grad);
}
