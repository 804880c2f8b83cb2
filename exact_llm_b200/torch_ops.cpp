// torch.ops.exact.* for drafted trees: schemas, argument checks and calls of the C ABI.
//
// The operators are small (a compaction runs 5 us), so what stands between a Python call and the launch is
// kept in C++: these take about a third of the time of the same checks in Python.  The entry points come from
// the library that exact_llm_b200._lib loaded (exb_torch_bind), and its errors are raised as its ExbError.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/extension.h>
#include <torch/library.h>

#include "exactb200.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

struct Entries {
  decltype(&exb_last_error) last_error = nullptr;
  decltype(&exb_tree_attention_workspace_bytes) workspace = nullptr;
  decltype(&exb_tree_attention) attention = nullptr;
  decltype(&exb_tree_verify) verify = nullptr;
  decltype(&exb_kv_compact) compact = nullptr;
  decltype(&exb_kv_copy_pages) copy = nullptr;
} lib;

constexpr int64_t EXP_LEN = 256 * 40 + 2;

void check(int rc) {
  if (rc == 0) return;
  const std::string msg = "exb error " + std::to_string(rc) + ": " + lib.last_error();
  py::gil_scoped_acquire gil;
  py::object cls = py::module_::import("exact_llm_b200._lib").attr("ExbError");
  PyErr_SetString(cls.ptr(), msg.c_str());
  python_error err;
  err.persist();
  throw err;
}

// dtype, shape (-1: any size) and contiguity of an argument
void want(const char* name, const Tensor& t, at::ScalarType type, at::IntArrayRef shape) {
  TORCH_CHECK_TYPE(t.scalar_type() == type, name, " must be ", type, ", not ", t.scalar_type());
  bool ok = t.dim() == (int64_t)shape.size();
  for (size_t i = 0; ok && i < shape.size(); ++i) ok = shape[i] < 0 || t.size(i) == shape[i];
  TORCH_CHECK_VALUE(ok, name, " has shape ", t.sizes(), ", not ", shape, " (-1: any)");
  TORCH_CHECK_VALUE(t.is_contiguous(), name, " must be contiguous");
}

void one_device(const Tensor& first, std::initializer_list<const Tensor*> rest, const OptTensor& status) {
  for (const Tensor* t : rest)
    TORCH_CHECK_VALUE(t->device() == first.device(), "tensors on ", first.device(), " and ", t->device(),
                      ": exact:: operators run on one CUDA device");
  if (status) {
    TORCH_CHECK_VALUE(status->device() == first.device(), "status is on ", status->device());
    want("status", *status, at::kInt, {1});
  }
}

exb_kv_view view(const char* op, const Tensor& k, const Tensor& ks, const Tensor& v, bool layered) {
  TORCH_CHECK_TYPE(k.scalar_type() == at::kShort && ks.scalar_type() == at::kChar && v.scalar_type() == at::kInt, op,
                   ": k int16, ks int8, v int32");
  const int64_t n = layered ? 5 : 4;
  TORCH_CHECK_VALUE(k.dim() == n && v.sizes() == k.sizes() && ks.sizes() == k.sizes().slice(0, n - 1), op,
                    ": cache shapes k ", k.sizes(), ", ks ", ks.sizes(), ", v ", v.sizes(), "; want ", n,
                    "-dimensional k and v of one shape and ks without the last dimension");
  TORCH_CHECK_VALUE(k.stride(n - 1) == 1 && v.stride(n - 1) == 1, op, ": the values of a cache row must lie together");
  for (int64_t d = 0; d < n; ++d) TORCH_CHECK_VALUE(k.size(d) <= INT32_MAX, op, ": cache dimension above 2^31");
  const int64_t l = layered ? 1 : 0;
  exb_kv_view x = {};
  x.k = k.data_ptr<int16_t>();
  x.ks = ks.data_ptr<int8_t>();
  x.v = v.data_ptr<int32_t>();
  x.layers = layered ? (int)k.size(0) : 1;
  x.pages = (int)k.size(l);
  x.KV = (int)k.size(l + 1);
  x.page = (int)k.size(l + 2);
  x.hd = (int)k.size(l + 3);
  if (layered) {
    x.k_layer = k.stride(0);
    x.s_layer = ks.stride(0);
    x.v_layer = v.stride(0);
  }
  x.k_page = k.stride(l); x.k_head = k.stride(l + 1); x.k_pos = k.stride(l + 2);
  x.s_page = ks.stride(l); x.s_head = ks.stride(l + 1); x.s_pos = ks.stride(l + 2);
  x.v_page = v.stride(l); x.v_head = v.stride(l + 1); x.v_pos = v.stride(l + 2);
  return x;
}

int32_t* status_of(const OptTensor& s) { return s ? s->data_ptr<int32_t>() : nullptr; }
void* stream_of(const Tensor& t) { return at::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// ------------------------------------------------------------------ tree attention
int64_t check_attention(const Tensor& q, const Tensor& qs, const Tensor& k, const Tensor& table, const Tensor& ctx,
                        const Tensor& row_start, const Tensor& mask, const Tensor& exp_t) {
  TORCH_CHECK_VALUE(q.scalar_type() == at::kShort && q.dim() == 3 && q.is_contiguous(),
                    "exact::tree_attention: q must be contiguous int16 (R, H, hd)");
  TORCH_CHECK_VALUE(k.dim() == 4 && k.size(3) == q.size(2) && k.size(1) > 0 && q.size(1) % k.size(1) == 0 &&
                        q.size(0) <= INT32_MAX && q.size(1) <= INT32_MAX,
                    "exact::tree_attention: q ", q.sizes(), " does not fit the cache ", k.sizes());
  const int64_t B = ctx.dim() == 1 ? ctx.size(0) : -2;
  want("qs", qs, at::kInt, {q.size(0), q.size(1)});
  want("ctx", ctx, at::kInt, {B});
  want("table", table, at::kInt, {B, -1});
  want("row_start", row_start, at::kInt, {B + 1});
  want("mask", mask, at::kLong, {q.size(0), -1});
  want("exp_t", exp_t, at::kInt, {EXP_LEN});
  TORCH_CHECK_VALUE(B < INT32_MAX && table.size(1) <= INT32_MAX && mask.size(1) <= INT32_MAX, "exact::tree_attention: size above 2^31");
  return B;
}

Tensor tree_attention(const Tensor& q, const Tensor& qs, const Tensor& k, const Tensor& ks, const Tensor& v,
                      const Tensor& table, const Tensor& ctx, const Tensor& row_start, const Tensor& mask,
                      const Tensor& exp_t, const OptTensor& status) {
  const int64_t B = check_attention(q, qs, k, table, ctx, row_start, mask, exp_t);
  const exb_kv_view kv = view("exact::tree_attention", k, ks, v, false);
  one_device(q, {&qs, &k, &ks, &v, &table, &ctx, &row_start, &mask, &exp_t}, status);
  c10::cuda::CUDAGuard guard(q.device());
  Tensor out = at::empty(q.sizes(), q.options().dtype(at::kLong));
  const int R = (int)q.size(0), H = (int)q.size(1);
  if (R == 0) return out;
  const size_t nb = lib.workspace(R, H, (int)B);
  Tensor ws = at::empty({(int64_t)nb}, q.options().dtype(at::kByte));
  check(lib.attention(&kv, q.data_ptr<int16_t>(), qs.data_ptr<int32_t>(), R, H, table.data_ptr<int32_t>(), (int)B,
                      (int)table.size(1), ctx.data_ptr<int32_t>(), row_start.data_ptr<int32_t>(),
                      reinterpret_cast<const uint64_t*>(mask.data_ptr<int64_t>()), (int)mask.size(1),
                      exp_t.data_ptr<int32_t>(), out.data_ptr<int64_t>(), ws.data_ptr(), nb, status_of(status),
                      stream_of(q)));
  return out;
}

Tensor tree_attention_meta(const Tensor& q, const Tensor& qs, const Tensor& k, const Tensor&, const Tensor&,
                           const Tensor& table, const Tensor& ctx, const Tensor& row_start, const Tensor& mask,
                           const Tensor& exp_t, const OptTensor&) {
  check_attention(q, qs, k, table, ctx, row_start, mask, exp_t);
  return at::empty(q.sizes(), q.options().dtype(at::kLong));
}

// ------------------------------------------------------------------ verification
using Four = std::tuple<Tensor, Tensor, Tensor, Tensor>;

int64_t check_verify(const Tensor& logits, const Tensor& u20, const Tensor& tokens, const Tensor& parent,
                     const Tensor& row_start, const Tensor& exp_t, int64_t max_len) {
  TORCH_CHECK_VALUE(logits.scalar_type() == at::kLong && logits.dim() == 2 && (logits.size(1) <= 1 || logits.stride(1) == 1),
                    "exact::tree_verify: logits must be int64 (R, V) with rows in one piece");
  TORCH_CHECK_VALUE(logits.size(1) >= 1 && logits.size(1) <= INT32_MAX && logits.size(0) <= INT32_MAX && max_len >= 1 &&
                        max_len <= INT32_MAX,
                    "exact::tree_verify: V >= 1 and max_len >= 1");
  TORCH_CHECK_VALUE(row_start.dim() == 1 && row_start.size(0) >= 1 && row_start.size(0) <= INT32_MAX,
                    "exact::tree_verify: row_start (B + 1)");
  const int64_t R = logits.size(0);
  want("u20", u20, at::kInt, {R});
  want("tokens", tokens, at::kInt, {R});
  want("parent", parent, at::kInt, {R});
  want("row_start", row_start, at::kInt, {-1});
  want("exp_t", exp_t, at::kInt, {EXP_LEN});
  return row_start.size(0) - 1;
}

Four verify_outputs(const Tensor& logits, int64_t B, int64_t max_len) {
  const auto o = logits.options().dtype(at::kInt);
  return {at::empty({logits.size(0)}, o), at::empty({B}, o), at::empty({B, max_len}, o), at::empty({B, max_len}, o)};
}

Four tree_verify(const Tensor& logits, const Tensor& u20, const Tensor& tokens, const Tensor& parent,
                 const Tensor& row_start, const Tensor& exp_t, int64_t tnum, int64_t max_len) {
  const int64_t B = check_verify(logits, u20, tokens, parent, row_start, exp_t, max_len);
  one_device(logits, {&u20, &tokens, &parent, &row_start, &exp_t}, {});
  c10::cuda::CUDAGuard guard(logits.device());
  Four out = verify_outputs(logits, B, max_len);
  const int R = (int)logits.size(0), V = (int)logits.size(1);
  check(lib.verify(logits.data_ptr<int64_t>(), R > 1 ? logits.stride(0) : V, R, V, u20.data_ptr<int32_t>(), tnum,
                   tokens.data_ptr<int32_t>(), parent.data_ptr<int32_t>(), row_start.data_ptr<int32_t>(), (int)B,
                   (int)max_len, exp_t.data_ptr<int32_t>(), std::get<0>(out).data_ptr<int32_t>(),
                   std::get<1>(out).data_ptr<int32_t>(), std::get<2>(out).data_ptr<int32_t>(),
                   std::get<3>(out).data_ptr<int32_t>(), stream_of(logits)));
  return out;
}

Four tree_verify_meta(const Tensor& logits, const Tensor& u20, const Tensor& tokens, const Tensor& parent,
                      const Tensor& row_start, const Tensor& exp_t, int64_t, int64_t max_len) {
  return verify_outputs(logits, check_verify(logits, u20, tokens, parent, row_start, exp_t, max_len), max_len);
}

// ------------------------------------------------------------------ cache rows
int64_t check_compact(const Tensor& table, const Tensor& ctx, const Tensor& path, const Tensor& n) {
  const int64_t B = ctx.dim() == 1 ? ctx.size(0) : -2;
  want("ctx", ctx, at::kInt, {B});
  want("table", table, at::kInt, {B, -1});
  want("path", path, at::kInt, {B, -1});
  want("n", n, at::kInt, {B});
  TORCH_CHECK_VALUE(B <= INT32_MAX && table.size(1) <= INT32_MAX && path.size(1) <= INT32_MAX, "exact::kv_compact_: size above 2^31");
  return B;
}

Tensor kv_compact(const Tensor& k, const Tensor& ks, const Tensor& v, const Tensor& table, const Tensor& ctx,
                  const Tensor& path, const Tensor& n, const OptTensor& status) {
  const int64_t B = check_compact(table, ctx, path, n);
  const exb_kv_view kv = view("exact::kv_compact_", k, ks, v, true);
  one_device(k, {&ks, &v, &table, &ctx, &path, &n}, status);
  c10::cuda::CUDAGuard guard(k.device());
  Tensor out = at::empty({B}, ctx.options());
  if (B)
    check(lib.compact(&kv, table.data_ptr<int32_t>(), (int)B, (int)table.size(1), ctx.data_ptr<int32_t>(),
                      path.data_ptr<int32_t>(), (int)path.size(1), n.data_ptr<int32_t>(), out.data_ptr<int32_t>(),
                      status_of(status), stream_of(k)));
  return out;
}

Tensor kv_compact_meta(const Tensor&, const Tensor&, const Tensor&, const Tensor& table, const Tensor& ctx,
                       const Tensor& path, const Tensor& n, const OptTensor&) {
  return at::empty({check_compact(table, ctx, path, n)}, ctx.options());
}

void kv_copy_pages(const Tensor& k, const Tensor& ks, const Tensor& v, const Tensor& src, const Tensor& dst,
                   const Tensor& rows, const OptTensor& status) {
  const exb_kv_view kv = view("exact::kv_copy_pages_", k, ks, v, true);
  want("src", src, at::kInt, {-1});
  want("dst", dst, at::kInt, {src.size(0)});
  want("rows", rows, at::kInt, {src.size(0)});
  TORCH_CHECK_VALUE(src.size(0) <= INT32_MAX, "exact::kv_copy_pages_: size above 2^31");
  one_device(k, {&ks, &v, &src, &dst, &rows}, status);
  c10::cuda::CUDAGuard guard(k.device());
  if (src.size(0))
    check(lib.copy(&kv, src.data_ptr<int32_t>(), dst.data_ptr<int32_t>(), rows.data_ptr<int32_t>(), (int)src.size(0),
                   status_of(status), stream_of(k)));
}

void kv_copy_pages_meta(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                        const OptTensor&) {}

}  // namespace

TORCH_LIBRARY_FRAGMENT(exact, m) {
  m.def("tree_attention(Tensor q, Tensor qs, Tensor k, Tensor ks, Tensor v, Tensor table, Tensor ctx, "
        "Tensor row_start, Tensor mask, Tensor exp_t, Tensor(a!)? status=None) -> Tensor");
  m.def("tree_verify(Tensor logits, Tensor u20, Tensor tokens, Tensor parent, Tensor row_start, Tensor exp_t, "
        "int tnum, int max_len) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("kv_compact_(Tensor(a!) k, Tensor(b!) ks, Tensor(c!) v, Tensor table, Tensor ctx, Tensor path, Tensor n, "
        "Tensor(d!)? status=None) -> Tensor");
  m.def("kv_copy_pages_(Tensor(a!) k, Tensor(b!) ks, Tensor(c!) v, Tensor src, Tensor dst, Tensor rows, "
        "Tensor(d!)? status=None) -> ()");
}
TORCH_LIBRARY_IMPL(exact, CUDA, m) {
  m.impl("tree_attention", tree_attention);
  m.impl("tree_verify", tree_verify);
  m.impl("kv_compact_", kv_compact);
  m.impl("kv_copy_pages_", kv_copy_pages);
}
TORCH_LIBRARY_IMPL(exact, Meta, m) {
  m.impl("tree_attention", tree_attention_meta);
  m.impl("tree_verify", tree_verify_meta);
  m.impl("kv_compact_", kv_compact_meta);
  m.impl("kv_copy_pages_", kv_copy_pages_meta);
}

// the entry points of the loaded library, in the order of Entries
extern "C" void exb_torch_bind(void* const* p) {
  lib.last_error = reinterpret_cast<decltype(lib.last_error)>(p[0]);
  lib.workspace = reinterpret_cast<decltype(lib.workspace)>(p[1]);
  lib.attention = reinterpret_cast<decltype(lib.attention)>(p[2]);
  lib.verify = reinterpret_cast<decltype(lib.verify)>(p[3]);
  lib.compact = reinterpret_cast<decltype(lib.compact)>(p[4]);
  lib.copy = reinterpret_cast<decltype(lib.copy)>(p[5]);
}
