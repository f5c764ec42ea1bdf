// Torch-facing wrappers of the paged KV cache (csrc/paged_kernels.h).  What a call looks at on the host is checked before the
// device, so that a refused call is refused anywhere.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <pybind11/pybind11.h>
#include <torch/extension.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <utility>
#include <vector>

#include "paged_kernels.h"
#include "paged_plan.h"

namespace py = pybind11;
using namespace penny;

namespace {
using OptTensor = c10::optional<at::Tensor>;

cudaStream_t cur() { return at::cuda::getCurrentCUDAStream().stream(); }
void need(bool ok, const char* msg) { TORCH_CHECK(ok, "penny: ", msg); }
void ck(cudaError_t rc, const char* what) { TORCH_CHECK(rc == cudaSuccess, "penny: ", what, ": ", cudaGetErrorString(rc)); }
bool aligned(const at::Tensor& t) { return ((uintptr_t)t.data_ptr() & 15) == 0; }
bool ints(const at::Tensor& t, int64_t n) { return t.scalar_type() == at::kInt && t.is_contiguous() && t.dim() == 1 && t.numel() == n; }
bool no_grad(const at::Tensor& t) { return !t.requires_grad() || !at::GradMode::is_enabled(); }

PagedType type_of(const at::Tensor& t, const char* msg) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return PAGED_BF16;
    case at::kHalf: return PAGED_FP16;
    case at::kFloat8_e4m3fn: return PAGED_E4M3;
    default: need(false, msg); return PAGED_BF16;
  }
}

// k and v as a pool, with the scales that its type needs.
PagedPool pool_of(const at::Tensor& k, const at::Tensor& v, PagedType type, PagedType cache, const OptTensor& k_scale, const OptTensor& v_scale) {
  // (the stride of a dimension of one says nothing)
  bool alike = k.dim() == 4 && v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type();
  for (int i = 0; alike && i < 4; ++i) alike = k.size(i) <= 1 || k.stride(i) == v.stride(i);
  need(alike, "paged caches: k and v [pages, page_size, kv_heads, dim] of one type, shape and strides");
  need(k.size(0) >= 1 && k.size(1) >= 1 && k.size(2) >= 1 && k.size(0) < (1ll << 31) && k.size(1) < (1ll << 31), "paged caches: pages and heads");
  need(cache == PAGED_E4M3 || cache == type, "paged caches: of the projection's type or e4m3");
  need(k.stride(3) == 1 && aligned(k) && aligned(v), "paged caches: contiguous in dim, 16-byte aligned");
  need(no_grad(k) && no_grad(v), "paged caches: no gradients");
  const int64_t size = k.element_size();
  for (int i = 0; i < 3; ++i)
    need(k.size(i) == 1 || (k.stride(i) * size % 16 == 0 && k.stride(i) >= 0), "paged caches: strides of whole 16 bytes");
  need(k_scale.has_value() == (cache == PAGED_E4M3) && v_scale.has_value() == (cache == PAGED_E4M3), "k_scale and v_scale: beside e4m3 caches, and only there");
  auto stride = [&](int i) -> long long { return k.size(i) == 1 ? 0 : k.stride(i); };
  PagedPool p = {k.data_ptr(), v.data_ptr(), stride(0), stride(1), stride(2), nullptr, nullptr,
                 (int)k.size(0), (int)k.size(1), (int)k.size(2), (int)k.size(3)};
  if (cache == PAGED_E4M3) {
    for (const at::Tensor* s : {&*k_scale, &*v_scale})
      need(s->scalar_type() == at::kFloat && s->is_contiguous() && s->dim() == 1 && s->numel() == k.size(2), "k_scale and v_scale: [kv_heads] fp32");
    need(no_grad(*k_scale) && no_grad(*v_scale), "paged caches: no gradients");
    p.k_scale = k_scale->data_ptr<float>();
    p.v_scale = v_scale->data_ptr<float>();
  }
  return p;
}
void on_device(const at::Tensor& first, std::initializer_list<const at::Tensor*> rest, const char* msg) {
  bool ok = first.is_cuda();
  for (const at::Tensor* t : rest) ok = ok && t->device() == first.device();
  need(ok, msg);
}
int sms_of(int device) {
  int sms = 0;
  ck(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device), "device");
  return sms;
}

// Where a tensor's elements lie: runs of `len` bytes at `n` by `step`, the largest step first; dimensions of one are left out.
struct Runs {
  uintptr_t at;
  std::vector<std::pair<int64_t, int64_t>> dims;  // (n, step in bytes)
  int64_t len;
  explicit Runs(const at::Tensor& t) : at((uintptr_t)t.data_ptr()), len(t.element_size()) {
    for (int i = 0; i < t.dim(); ++i)
      if (t.size(i) > 1 && (i + 1 < t.dim() || t.stride(i) != 1)) dims.push_back({t.size(i), t.stride(i) * t.element_size()});
    if (t.dim() > 0 && (t.size(-1) <= 1 || t.stride(-1) == 1)) len *= t.size(-1);
    std::stable_sort(dims.begin(), dims.end(), [](auto& a, auto& b) { return a.second > b.second; });
  }
};
// From a tensor's first byte to behind its last.
std::pair<uintptr_t, uintptr_t> bounds(const at::Tensor& t) {
  const auto sizes = t.sizes(), strides = t.strides();
  int64_t n = 1;
  for (size_t i = 0; i < sizes.size(); ++i) n += (sizes[i] - 1) * strides[i];
  const uintptr_t at = (uintptr_t)t.data_ptr();
  return {at, at + n * t.element_size()};
}
// Do runs of a and runs of b, both laid out by dims[i...], meet if b's are `off` bytes further?
bool meet_at(const Runs& a, const Runs& b, size_t i, int64_t off) {
  if (i == a.dims.size()) return off < a.len && -off < b.len;
  const auto [n, step] = a.dims[i];
  if (step == 0) return meet_at(a, b, i + 1, off);
  int64_t wa = a.len, wb = b.len;  // of what is inside a step
  for (size_t j = i + 1; j < a.dims.size(); ++j) wa += (a.dims[j].first - 1) * a.dims[j].second, wb += (a.dims[j].first - 1) * a.dims[j].second;
  // off + d step in (-wb, wa): one or two d, unless steps overlap
  auto floor_div = [](int64_t x, int64_t y) { return x >= 0 ? x / y : -((-x + y - 1) / y); };
  for (int64_t d = std::max(1 - n, floor_div(-wb - off, step)); d < n && off + d * step < wa; ++d)
    if (off + d * step > -wb && meet_at(a, b, i + 1, off + d * step)) return true;
  return false;
}
bool overlap(const at::Tensor& ta, const at::Tensor& tb) {
  if (ta.numel() == 0 || tb.numel() == 0) return false;
  const auto in_a = bounds(ta), in_b = bounds(tb);
  if (in_a.second <= in_b.first || in_b.second <= in_a.first) return false;
  const Runs a(ta), b(tb);
  if (a.dims == b.dims) return meet_at(a, b, 0, (int64_t)(b.at - a.at));
  // laid out in two ways, within each other's bounds: all runs in order
  int64_t count = 0;
  for (const Runs* r : {&a, &b}) {
    int64_t n = 1;
    for (auto& d : r->dims) n *= d.first;
    count += n;
  }
  if (count > 1 << 22) return true;
  std::vector<std::pair<uintptr_t, const Runs*>> runs;
  for (const Runs* r : {&a, &b}) {
    std::vector<uintptr_t> at = {r->at};
    for (auto& d : r->dims) {
      const size_t n = at.size();
      for (int64_t i = 1; i < d.first; ++i)
        for (size_t j = 0; j < n; ++j) at.push_back(at[j] + i * d.second);
    }
    for (uintptr_t x : at) runs.push_back({x, r});
  }
  std::sort(runs.begin(), runs.end());
  uintptr_t end_a = 0, end_b = 0;
  for (auto& [x, r] : runs) {
    if (x < (r == &a ? end_b : end_a)) return true;
    (r == &a ? end_a : end_b) = x + r->len;  // (runs of one tensor have one length: the last begun is the last to end)
  }
  return false;
}
// Every element of b where a has the one of the same indices (the last dimension may be shorter)
bool same_place(const at::Tensor& a, const at::Tensor& b) {
  bool same = a.data_ptr() == b.data_ptr();
  for (int i = 0; same && i + 1 < a.dim(); ++i) same = a.size(i) <= 1 || a.stride(i) == b.stride(i);
  return same;
}
}  // namespace

void bind_paged(py::module_& m) {
  m.attr("PAGED_MAX_ROWS") = kPagedMaxRows;
  // Tokens come (news[r] > 0) and leave (news[r] < 0, the last ones): table, lengths, free and free_count in place; returns or
  // fills (slots [tokens] int64, positions [tokens] int32, offsets [rows + 1] int32, granted [rows] bool).
  m.def("page_tables", [](at::Tensor table, at::Tensor lengths, at::Tensor free, at::Tensor free_count, at::Tensor news, int64_t page_size,
                          int64_t tokens, c10::optional<std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor>> out,
                          c10::optional<int64_t> max_len) {
    need(table.scalar_type() == at::kInt && table.dim() == 2 && table.size(0) >= 1 && table.size(1) >= 1, "page_tables: table [rows, pages of a row] int32");
    const int64_t R = table.size(0), W = table.size(1);
    need(R <= kPagedMaxRows, "page_tables: more than PAGED_MAX_ROWS rows");
    need((W == 1 || table.stride(1) == 1) && (R == 1 || table.stride(0) >= W), "page_tables: a table with contiguous rows that do not overlap");
    need(ints(lengths, R) && ints(news, R), "page_tables: lengths and new tokens [rows] int32");
    need(free.dim() == 1 && free.numel() >= 1 && free.numel() < (1ll << 31) && ints(free, free.numel()) && ints(free_count, 1),
         "page_tables: free [pages] and free_count [1] int32");
    need(page_size >= 1 && page_size < (1ll << 30) && W < (1ll << 31), "page_tables: page size");
    need(tokens >= 0 && tokens < (1ll << 31) - 8, "page_tables: tokens");
    need(!max_len.has_value() || *max_len >= 0, "page_tables: max_len");
    if (out.has_value()) {
      const auto& [slots, positions, offsets, granted] = *out;
      need(slots.scalar_type() == at::kLong && slots.is_contiguous() && slots.dim() == 1 && slots.numel() == tokens && ints(positions, tokens) &&
               ints(offsets, R + 1) && granted.scalar_type() == at::kBool && granted.is_contiguous() && granted.dim() == 1 && granted.numel() == R,
           "page_tables: out is (slots [tokens] int64, positions [tokens] int32, offsets [rows + 1] int32, granted [rows] bool)");
      need(aligned(slots) && aligned(positions), "page_tables: 16-byte aligned slots and positions");
    }
    {  // (the state is read and written by different CTAs, new by some after others have written)
      const at::Tensor* all[9] = {&table, &lengths, &free, &free_count, &news};
      int n = 5;
      if (out.has_value())
        for (const at::Tensor* t : {&std::get<0>(*out), &std::get<1>(*out), &std::get<2>(*out), &std::get<3>(*out)}) all[n++] = t;
      std::pair<uintptr_t, uintptr_t> in[9];
      for (int i = 0; i < n; ++i) {
        in[i] = bounds(*all[i]);
        for (int j = 0; j < i; ++j)
          need(all[i]->numel() == 0 || all[j]->numel() == 0 || in[i].second <= in[j].first || in[j].second <= in[i].first,
               "page_tables: table, lengths, free, free_count, new tokens and out in memory of their own");
      }
    }
    on_device(table, {&lengths, &free, &free_count, &news}, "page_tables expects tensors on one CUDA device");
    const at::cuda::OptionalCUDAGuard guard(table.device());
    if (!out.has_value()) {
      // one allocation for the four (of a call of 6.7 us on the host, four took 3)
      const int64_t at1 = (tokens * 8 + 15) / 16 * 16, at2 = at1 + (tokens * 4 + 15) / 16 * 16, at3 = at2 + (R + 1) * 4;
      const at::Tensor all = at::detail::empty_cuda({at3 + R}, at::kByte, table.device(), c10::nullopt);
      auto part = [&](int64_t from, int64_t n, at::ScalarType type) {
        at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(), c10::scalarTypeToTypeMeta(type));
        t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
        t.unsafeGetTensorImpl()->set_storage_offset(from / (int64_t)c10::elementSize(type));
        return t;
      };
      out = std::make_tuple(part(0, tokens, at::kLong), part(at1, tokens, at::kInt), part(at2, R + 1, at::kInt), part(at3, R, at::kBool));
    }
    const auto& [slots, positions, offsets, granted] = *out;
    on_device(table, {&slots, &positions, &offsets, &granted}, "page_tables expects tensors on one CUDA device");
    const PageTables a = {table.data_ptr<int>(), table.stride(0), lengths.data_ptr<int>(), free.data_ptr<int>(), free_count.data_ptr<int>(),
                          news.data_ptr<int>(), (long long*)slots.data_ptr<int64_t>(), positions.data_ptr<int>(), offsets.data_ptr<int>(),
                          granted.data_ptr<bool>(), (int)R, (int)W, (int)free.numel(), (int)page_size, (int)tokens,
                          (int)std::min<int64_t>(max_len.value_or(INT_MAX), INT_MAX)};
    ck(launch_page_tables(a, cur()), "page_tables");
    return *out;
  }, py::arg("table"), py::arg("lengths"), py::arg("free"), py::arg("free_count"), py::arg("new"), py::arg("page_size"), py::arg("tokens"),
     py::arg("out") = py::none(), py::arg("max_len") = py::none());
  // qkv [tokens, (heads + 2 kv_heads) dim]: q and k rotated in place or into out [tokens, (heads + kv_heads) dim], k and v to their slots.
  m.def("paged_append", [](at::Tensor qkv, at::Tensor k, at::Tensor v, at::Tensor slots, at::Tensor positions, int64_t heads, double theta,
                           OptTensor out, OptTensor k_scale, OptTensor v_scale, bool early) {
    const PagedType type = type_of(qkv, "paged_append: bf16 or fp16 qkv"), cache = type_of(k, "paged_append: bf16, fp16 or e4m3 caches");
    need(type != PAGED_E4M3, "paged_append: bf16 or fp16 qkv");
    const PagedPool pool = pool_of(k, v, type, cache, k_scale, v_scale);
    const int64_t D = pool.dim, T = qkv.size(0);
    for (int i = 0; i < 3; ++i) need(k.size(i) == 1 || k.stride(i) > 0, "paged_append: caches whose rows do not overlap");
    need(D % 16 == 0 && D >= 16 && D <= 256, "paged_append: dim a multiple of 16, up to 256");
    need(heads >= 0 && heads < (1 << 20) && qkv.dim() == 2 && qkv.size(1) == (heads + 2 * pool.heads) * D && T < (1ll << 31),
         "paged_append: qkv must be [tokens, (heads + 2 kv_heads) dim]");
    need(qkv.stride(1) == 1 && (T <= 1 || (qkv.stride(0) >= qkv.size(1) && qkv.stride(0) % 8 == 0)) && aligned(qkv),
         "paged_append: rows of qkv contiguous, 16-byte aligned");
    need(slots.scalar_type() == at::kLong && slots.is_contiguous() && slots.dim() == 1 && slots.numel() == T && ints(positions, T),
         "paged_append: slots [tokens] int64, positions [tokens] int32");
    need(theta > 0 && std::isfinite(theta), "paged_append: theta above zero");
    need(no_grad(qkv) && (!out.has_value() || no_grad(*out)), "paged_append: no gradients");
    if (out.has_value())
      need(out->scalar_type() == qkv.scalar_type() && out->dim() == 2 && out->size(0) == T && out->size(1) == (heads + pool.heads) * D &&
               out->stride(1) == 1 && (T <= 1 || (out->stride(0) >= out->size(1) && out->stride(0) % 8 == 0)) && aligned(*out),
           "paged_append: out must be [tokens, (heads + kv_heads) dim], like qkv");
    if (out.has_value()) need(!overlap(*out, qkv) || same_place(*out, qkv), "paged_append: out is the start of qkv's rows, or apart from them");
    need(!overlap(k, v), "paged_append: k apart from v");
    on_device(qkv, {&k, &v, &slots, &positions}, "paged_append expects tensors on one CUDA device");
    if (out.has_value()) on_device(qkv, {&*out}, "paged_append expects tensors on one CUDA device");
    if (k_scale.has_value()) on_device(qkv, {&*k_scale, &*v_scale}, "paged_append expects tensors on one CUDA device");
    const at::cuda::OptionalCUDAGuard guard(qkv.device());
    ck(launch_paged_append(qkv.data_ptr(), qkv.stride(0), out.has_value() ? out->data_ptr() : nullptr, out.has_value() ? out->stride(0) : 0, type, pool,
                           cache, (const long long*)slots.data_ptr<int64_t>(), positions.data_ptr<int>(), (int)T, (int)heads, theta, early, cur()),
       "paged_append");
  }, py::arg("qkv"), py::arg("k"), py::arg("v"), py::arg("slots"), py::arg("positions"), py::arg("heads"), py::arg("theta"),
     py::arg("out") = py::none(), py::arg("k_scale") = py::none(), py::arg("v_scale") = py::none(), py::arg("early") = false);
  m.def("paged_attention_workspace_bytes", [](int64_t rows, int64_t heads, int64_t kv_heads, int64_t dim, int64_t max_len, int64_t window) {
    need(rows >= 1 && kv_heads >= 1 && heads >= kv_heads && heads % kv_heads == 0 && dim >= 1 && max_len >= 1 && window >= 0,
         "paged_attention_workspace_bytes: rows, heads and lengths");
    need(rows < (1 << 24) && heads < (1 << 20) && dim <= 256, "paged_attention_workspace_bytes: rows, heads and dim");
    return (int64_t)paged_attention_workspace_bytes((int)rows, (int)heads, (int)kv_heads, (int)dim, (int)std::min<int64_t>(max_len, paged::kMaxLen),
                                                    (int)std::min<int64_t>(window, 1ll << 30),
                                                    sms_of(at::cuda::current_device()));
  }, py::arg("rows"), py::arg("heads"), py::arg("kv_heads"), py::arg("dim"), py::arg("max_len"), py::arg("window") = 0);
  // q [rows, heads, dim], one token of every row, attends to the row's last `window` positions (0: all of them).
  m.def("paged_attention", [](at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor table, at::Tensor lengths, OptTensor out, OptTensor lse,
                              c10::optional<double> scale, int64_t window, OptTensor k_scale, OptTensor v_scale, OptTensor workspace, bool early) {
    const PagedType type = type_of(q, "paged_attention: bf16 or fp16 q"), cache = type_of(k, "paged_attention: bf16, fp16 or e4m3 caches");
    need(type != PAGED_E4M3, "paged_attention: bf16 or fp16 q");
    const PagedPool pool = pool_of(k, v, type, cache, k_scale, v_scale);
    need(q.dim() == 3 && q.size(2) == pool.dim, "paged_attention: q must be [rows, heads, dim]");
    const int64_t B = q.size(0), H = q.size(1);
    need(B < (1 << 24) && H < (1 << 20) && H >= 1 && H % pool.heads == 0, "paged_attention: heads a multiple of the caches'");
    need(pool.dim == 64 || pool.dim == 128 || pool.dim == 256, "paged_attention: dim 64, 128 or 256");
    need(paged::steps_of(pool.pages, pool.page_size, pool.page_stride, pool.pos_stride, (int)k.element_size()).bytes > 0,
         "paged_attention: caches that reach over 2^32 times what divides their strides");
    need(pool.page_size == 1 || pool.pos_stride * k.element_size() <= 1 << 26, "paged_attention: positions of a page at most 64 MB apart");
    auto rows_ok = [&](const at::Tensor& t) {
      return t.stride(2) == 1 && (B <= 1 || t.stride(0) % 8 == 0) && (H == 1 || t.stride(1) % 8 == 0) && aligned(t);
    };
    // rows and heads that do not overlap: one of the two outside the other
    auto apart = [&](const at::Tensor& t) {
      const int64_t D = pool.dim, b = B > 1 ? t.stride(0) : INT64_MAX, h = H > 1 ? t.stride(1) : INT64_MAX;
      if (B <= 1 || H <= 1) return b >= D && h >= D;
      return (h >= D && b / H >= h) || (b >= D && h / B >= b);
    };
    need(rows_ok(q), "paged_attention: heads of q contiguous, 16-byte aligned");
    need(table.scalar_type() == at::kInt && table.dim() == 2 && table.size(0) == B && table.size(1) >= 1 && table.size(1) < (1ll << 31) &&
             (table.size(1) == 1 || table.stride(1) == 1),
         "paged_attention: table [rows, pages of a row] int32 with contiguous rows");
    need(ints(lengths, B), "paged_attention: lengths [rows] int32");
    need(window >= 0, "paged_attention: a window of no or some positions");
    need(!scale.has_value() || std::isfinite((float)*scale), "paged_attention: a finite scale");
    need(no_grad(q) && (!out.has_value() || no_grad(*out)) && (!lse.has_value() || no_grad(*lse)), "paged_attention: no gradients");
    if (out.has_value())
      need(out->scalar_type() == q.scalar_type() && out->sizes() == q.sizes() && rows_ok(*out) && apart(*out), "paged_attention: out like q, its rows apart");
    if (out.has_value()) need(!overlap(*out, q) || same_place(*out, q), "paged_attention: out is q, or apart from it");
    if (lse.has_value())
      need(lse->scalar_type() == at::kFloat && lse->is_contiguous() && lse->dim() == 2 && lse->size(0) == B && lse->size(1) == H, "paged_attention: lse [rows, heads] fp32");
    if (workspace.has_value()) need(workspace->is_contiguous() && aligned(*workspace), "paged_attention: 16-byte aligned contiguous workspace");
    on_device(q, {&k, &v, &table, &lengths}, "paged_attention expects tensors on one CUDA device");
    for (const OptTensor* t : {&out, &lse, &k_scale, &v_scale, &workspace})
      if (t->has_value()) on_device(q, {&**t}, "paged_attention expects tensors on one CUDA device");
    const at::cuda::OptionalCUDAGuard guard(q.device());
    if (!out.has_value()) out = at::detail::empty_cuda({B, H, pool.dim}, q.scalar_type(), q.device(), c10::nullopt);
    if (B == 0) return *out;
    const int sms = sms_of(q.get_device());
    const int win = (int)std::min<int64_t>(window, 1ll << 30);
    const int max_len = (int)std::min<int64_t>(table.size(1) * pool.page_size, paged::kMaxLen);
    need(B * (int64_t)paged::units_of(win > 0 && win < max_len ? win : max_len, 16) <= paged::kMaxUnits, "paged_attention: a table for over 2^34 positions");
    const size_t bytes = paged_attention_workspace_bytes((int)B, (int)H, pool.heads, pool.dim, max_len, win, sms);
    if (workspace.has_value()) need(workspace->nbytes() >= bytes, "workspace too small (paged_attention_workspace_bytes)");
    else if (bytes > 0) workspace = at::detail::empty_cuda({(int64_t)bytes}, at::kByte, q.device(), c10::nullopt);
    const PagedAttention a = {q.data_ptr(), q.stride(0), q.stride(1), out->data_ptr(), out->stride(0), out->stride(1),
                              lse.has_value() ? lse->data_ptr<float>() : nullptr, table.data_ptr<int>(), table.stride(0), lengths.data_ptr<int>(),
                              (int)B, (int)H, (int)table.size(1), win, scale.has_value() ? (float)*scale : 1.0f / std::sqrt((float)pool.dim), early};
    ck(launch_paged_attention(a, type, pool, cache, workspace.has_value() ? workspace->data_ptr() : nullptr, sms, cur()), "paged_attention");
    return *out;
  }, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("table"), py::arg("lengths"), py::arg("out") = py::none(), py::arg("lse") = py::none(),
     py::arg("scale") = py::none(), py::arg("window") = 0, py::arg("k_scale") = py::none(), py::arg("v_scale") = py::none(),
     py::arg("workspace") = py::none(), py::arg("early") = false);
}
