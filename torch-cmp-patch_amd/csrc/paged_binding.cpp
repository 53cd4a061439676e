// cmpext3._native -- torch binding of the paged key-value cache's operators
// (include/cmpext3_paged.h), in the manner of the attention's: unsupported
// input raises RuntimeError, work goes to the caller's current stream, and
// nothing waits for the device.
#include <cmath>

#include "binding.h"

#include "../../include/cmpext3_paged.h"

using namespace cmpext3_binding;

namespace {

using Optional = c10::optional<torch::Tensor>;

struct Str {
  int64_t s[3];
  explicit Str(const torch::Tensor& t) : s{t.stride(0), t.stride(1), t.stride(2)} {}
};

bool given(const Optional& t) { return t.has_value() && t->defined(); }

// An [_, _, _, D] tensor of the call's dtype and device.
void check_data(const char* name, const torch::Tensor& t, const torch::Tensor& like) {
  TORCH_CHECK(t.dim() == 4, "cmpext3 paged: ", name, " must be 4D");
  TORCH_CHECK(t.device() == like.device(), "cmpext3 paged: ", name, " on another device");
  TORCH_CHECK(t.scalar_type() == like.scalar_type(), "cmpext3 paged: ", name, " of another dtype");
  TORCH_CHECK(t.size(3) == like.size(3), "cmpext3 paged: ", name, " of another head dim");
}

int check_first(const char* name, const torch::Tensor& t) {
  TORCH_CHECK(t.dim() == 4, "cmpext3 paged: ", name, " must be 4D");
  TORCH_CHECK(t.is_cuda(), "cmpext3 paged: tensors must be on the GPU");
  const int dtype = dtype_code(t.scalar_type());
  TORCH_CHECK(dtype >= 0, "cmpext3 paged: unsupported dtype ", t.scalar_type());
  for (int i = 0; i < 4; ++i)
    TORCH_CHECK(t.size(i) <= INT32_MAX, "cmpext3 paged: ", name, " has a dim past 32 bits");
  return dtype;
}

// The operators have no backward: a call whose gradient would be lost is refused.
void check_grad(std::initializer_list<const torch::Tensor*> tensors) {
  if (!at::GradMode::is_enabled()) return;
  for (const torch::Tensor* t : tensors)
    TORCH_CHECK(!t->defined() || !t->requires_grad(),
                "cmpext3 paged: no backward here (call under torch.no_grad(), or detach)");
}

// Pages: [num_pages, H_kv, page_size, D], read and written in place.
void check_pages(const char* name, const torch::Tensor& t, const torch::Tensor& like, int64_t Hkv) {
  check_data(name, t, like);
  TORCH_CHECK(t.size(1) == Hkv, "cmpext3 paged: ", name, " must hold ", Hkv, " heads");
  TORCH_CHECK(t.size(0) >= 1 && t.size(2) >= 1 && t.size(0) <= INT32_MAX && t.size(2) <= INT32_MAX,
              "cmpext3 paged: ", name, " has no pages or no slots");
  TORCH_CHECK(t.stride(3) == 1, "cmpext3 paged: ", name, " needs a contiguous last dim");
}

void check_ints(const char* name, const torch::Tensor& t, const torch::Tensor& like, at::IntArrayRef sizes) {
  TORCH_CHECK(t.device() == like.device(), "cmpext3 paged: ", name, " on another device");
  TORCH_CHECK(t.scalar_type() == at::kInt, "cmpext3 paged: ", name, " must be int32");
  TORCH_CHECK(t.sizes() == sizes, "cmpext3 paged: ", name, " must have shape ", sizes, ", not ", t.sizes());
}

// page_table [B, width] and the per-sequence lengths [B]
struct Map {
  torch::Tensor table, lens, fresh;
  int width;
  int64_t stride;
  Map(const torch::Tensor& page_table, const torch::Tensor& seq_lens, const Optional& new_lens,
      const torch::Tensor& like) {
    const int64_t B = like.size(0);
    TORCH_CHECK(page_table.dim() == 2 && page_table.size(1) <= INT32_MAX,
                "cmpext3 paged: page_table must be [batch, pages of a sequence]");
    check_ints("page_table", page_table, like, {B, page_table.size(1)});
    check_ints("seq_lens", seq_lens, like, {B});
    table = page_table.size(1) > 1 && page_table.stride(1) != 1 ? page_table.contiguous() : page_table;
    lens = seq_lens.contiguous();
    if (given(new_lens)) {
      check_ints("new_lens", *new_lens, like, {B});
      fresh = new_lens->contiguous();
    }
    width = (int)table.size(1);
    stride = table.stride(0);
  }
  const int32_t* pages() const { return table.numel() ? table.data_ptr<int32_t>() : nullptr; }
  const int32_t* news() const { return fresh.defined() ? fresh.data_ptr<int32_t>() : nullptr; }
};

// Rows in whole 16-byte chunks at 16-byte aligned addresses: the tensor itself
// where it is laid out so, else a contiguous copy.
torch::Tensor chunk_rows(const torch::Tensor& t) {
  const int64_t es = t.element_size();
  bool ok = t.stride(3) == 1 && ((uintptr_t)t.data_ptr() & 15u) == 0;
  for (int i = 0; i < 3; ++i) ok = ok && (t.size(i) <= 1 || (t.stride(i) >= 0 && t.stride(i) * es % 16 == 0));
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

// The output of a call, in the query's own memory order where that is [B,S,H,D].
torch::Tensor like_query(const torch::Tensor& q) {
  const int64_t B = q.size(0), H = q.size(1), S = q.size(2), D = q.size(3);
  const bool bshd = H > 1 && S > 1 && q.stride(1) == D && q.stride(2) == H * D;
  return bshd ? torch::empty({B, S, H, D}, q.options()).transpose(1, 2) : torch::empty({B, H, S, D}, q.options());
}

void wrote(const torch::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

void check_rc(int rc, const char* what) {
  TORCH_CHECK(rc == CMPEXT3_OK, "cmpext3 ", what, ": ", cmpext3_attn_strerror(rc));
}

hipStream_t stream_of(const torch::Tensor& t) {
  return at::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

}  // namespace

static c10::optional<torch::Tensor> paged_append(
    torch::Tensor key, torch::Tensor value, torch::Tensor key_pages, torch::Tensor value_pages,
    torch::Tensor page_table, torch::Tensor seq_lens, Optional query, Optional cos, Optional sin, Optional positions,
    Optional new_lens, bool interleaved, Optional key_bounds) {
  const int dtype = check_first("key", key);
  const int64_t B = key.size(0), Hkv = key.size(1), S = key.size(2), D = key.size(3);
  check_data("value", value, key);
  TORCH_CHECK(value.sizes() == key.sizes(), "cmpext3 paged: value must have key's shape");
  check_pages("key_pages", key_pages, key, Hkv);
  check_pages("value_pages", value_pages, key, Hkv);
  TORCH_CHECK(value_pages.sizes() == key_pages.sizes(), "cmpext3 paged: value_pages must have key_pages' shape");
  const int64_t P = key_pages.size(0), page = key_pages.size(2);
  TORCH_CHECK(given(cos) == given(sin), "cmpext3 paged: cos and sin come together");
  TORCH_CHECK(!given(query) || given(cos), "cmpext3 paged: query is there to be rotated: cos and sin are missing");
  TORCH_CHECK(!given(positions) || given(cos), "cmpext3 paged: positions name rows of cos and sin, which are missing");
  const torch::Tensor none;
  check_grad({&key, &value, &key_pages, &value_pages, given(query) ? &*query : &none, given(cos) ? &*cos : &none,
              given(sin) ? &*sin : &none, given(key_bounds) ? &*key_bounds : &none});
  torch::Tensor c, s, at_rows, q, out;
  int rows = 0, rot = 0;
  int64_t row_stride = 0;
  if (given(cos)) {
    TORCH_CHECK(cos->dim() == 2 && cos->sizes() == sin->sizes() && cos->scalar_type() == at::kFloat &&
                    sin->scalar_type() == at::kFloat && cos->device() == key.device() && sin->device() == key.device(),
                "cmpext3 paged: cos and sin must be fp32 [rows, rotated dims / 2] on key's device");
    TORCH_CHECK(cos->size(0) >= 1 && cos->size(0) <= INT32_MAX && cos->size(1) >= 1 && 2 * cos->size(1) <= D,
                "cmpext3 paged: cos and sin rotate ", 2 * cos->size(1), " of ", D, " dims");
    // rows of wider tables (half of [cos, cos], say) are read where they lie
    const bool as_is = cos->stride(0) == sin->stride(0) &&
                       (cos->size(1) == 1 || (cos->stride(1) == 1 && sin->stride(1) == 1));
    c = as_is ? *cos : cos->contiguous();
    s = as_is ? *sin : sin->contiguous();
    rows = (int)c.size(0);
    rot = 2 * (int)c.size(1);
    row_stride = rows > 1 ? c.stride(0) : 0;
  }
  if (given(positions)) {
    check_ints("positions", *positions, key, {B, S});
    at_rows = positions->contiguous();
  }
  int64_t H = Hkv;
  if (given(query)) {
    check_data("query", *query, key);
    H = query->size(1);
    TORCH_CHECK(query->size(0) == B && query->size(2) == S && Hkv >= 1 && H >= 1 && H % Hkv == 0,
                "cmpext3 paged: query must be [batch, a multiple of key's heads, columns, head dim]");
  }
  if (given(key_bounds)) {
    check_data("key_bounds", *key_bounds, key);
    TORCH_CHECK(key_bounds->size(0) == P && key_bounds->size(1) == Hkv && key_bounds->size(2) == 2 &&
                    key_bounds->stride(3) == 1,
                "cmpext3 paged: key_bounds must be [pages, heads, 2, head dim]");
  }
  const Map map(page_table, seq_lens, new_lens, key);
  const at::hip::HIPGuardMasqueradingAsCUDA guard(key.device());
  if (given(query)) out = like_query(*query);
  if (B * S == 0) return given(query) ? c10::optional<torch::Tensor>(out) : c10::nullopt;
  TORCH_CHECK(D * key.element_size() % 16 == 0 && D <= 256,
              "cmpext3 paged: head dim ", D, " is not whole 16-byte chunks up to 256");
  const torch::Tensor k = chunk_rows(key), v = chunk_rows(value);
  if (given(query)) q = chunk_rows(*query);
  const Str ks(k), vs(v), qs(given(query) ? q : k), os(given(query) ? out : k), kps(key_pages), vps(value_pages),
      kbs(given(key_bounds) ? *key_bounds : k);
  check_rc(cmpext3_paged_append(
               k.data_ptr(), v.data_ptr(), given(query) ? q.data_ptr() : nullptr,
               given(query) ? out.data_ptr() : nullptr, key_pages.data_ptr(), value_pages.data_ptr(),
               given(key_bounds) ? key_bounds->data_ptr() : nullptr, dtype, (int)B, (int)H, (int)Hkv, (int)S, (int)D,
               (int)P, (int)page, ks.s, vs.s, qs.s, os.s, kps.s, vps.s, kbs.s, map.pages(), map.width, map.stride,
               map.lens.data_ptr<int32_t>(), map.news(),
               at_rows.defined() ? at_rows.data_ptr<int32_t>() : nullptr, rot ? c.data_ptr<float>() : nullptr,
               rot ? s.data_ptr<float>() : nullptr, rows, rot, row_stride, interleaved ? 1 : 0, stream_of(key)),
           "paged_append");
  wrote(key_pages);
  wrote(value_pages);
  if (given(key_bounds)) wrote(*key_bounds);
  return given(query) ? c10::optional<torch::Tensor>(out) : c10::nullopt;
}

static torch::Tensor paged_attention(torch::Tensor query, torch::Tensor key_pages, torch::Tensor value_pages,
                                     torch::Tensor page_table, torch::Tensor seq_lens,
                                     c10::optional<double> scale_arg, Optional new_lens, Optional selected) {
  const int dtype = check_first("query", query);
  const int64_t B = query.size(0), H = query.size(1), S = query.size(2), D = query.size(3);
  TORCH_CHECK(key_pages.dim() == 4, "cmpext3 paged: key_pages must be 4D");
  const int64_t Hkv = key_pages.size(1);
  TORCH_CHECK(Hkv >= 1 && H >= 1 && H % Hkv == 0, "cmpext3 paged: ", H, " query heads over ", Hkv, " key heads");
  check_pages("key_pages", key_pages, query, Hkv);
  check_pages("value_pages", value_pages, query, Hkv);
  TORCH_CHECK(value_pages.sizes() == key_pages.sizes(), "cmpext3 paged: value_pages must have key_pages' shape");
  TORCH_CHECK(S <= 16, "cmpext3 paged: at most 16 query columns (a prompt goes through scaled_dot_product_attention)");
  check_grad({&query, &key_pages, &value_pages});
  const Map map(page_table, seq_lens, new_lens, query);
  torch::Tensor sel;
  if (given(selected)) {
    TORCH_CHECK(selected->dim() == 3 && selected->size(2) >= 1 && selected->size(2) <= INT32_MAX,
                "cmpext3 paged: selected must be [batch, key heads, pages], with a page at least");
    check_ints("selected", *selected, query, {B, Hkv, selected->size(2)});
    sel = selected->contiguous();
  }
  const float scale = scale_arg.has_value() ? (float)scale_arg.value() : 1.0f / std::sqrt((float)D);
  TORCH_CHECK(std::isfinite(scale), "cmpext3 paged: non-finite scale");
  const at::hip::HIPGuardMasqueradingAsCUDA guard(query.device());
  hipStream_t stream = stream_of(query);
  torch::Tensor out = like_query(query);
  if (out.numel() == 0) return out;
  TORCH_CHECK(D * query.element_size() % 16 == 0 && D <= 256,
              "cmpext3 paged: head dim ", D, " is not whole 16-byte chunks up to 256");
  const torch::Tensor q = chunk_rows(query);
  const int page = (int)key_pages.size(2), K = sel.defined() ? (int)sel.size(2) : 0;
  const size_t need = cmpext3_paged_attn_workspace_size(dtype, (int)B, (int)H, (int)Hkv, (int)S, (int)D, page,
                                                        map.width, K);
  // A captured call's workspace is the graph's own (its counters are cleared
  // at every replay): replays beside eager calls on the stream, or of another
  // graph, share nothing with it.
  Workspace ws;
  torch::Tensor own;
  if (need > 0 && capturing(stream)) {
    own = torch::empty({(int64_t)need}, query.options().dtype(at::kByte));
    own.narrow(0, 0, CMPEXT3_WORKSPACE_COUNTER_BYTES).zero_();
    ws.ptr = own.data_ptr();
    ws.bytes = need;
  } else {
    ws = workspace_for(query, stream, need);
  }
  const Str qs(q), kps(key_pages), vps(value_pages), os(out);
  check_rc(cmpext3_paged_attn(q.data_ptr(), key_pages.data_ptr(), value_pages.data_ptr(), out.data_ptr(), dtype, (int)B,
                              (int)H, (int)Hkv, (int)S, (int)D, (int)key_pages.size(0), page, qs.s, kps.s, vps.s, os.s,
                              map.pages(), map.width, map.stride, map.lens.data_ptr<int32_t>(), map.news(),
                              sel.defined() ? sel.data_ptr<int32_t>() : nullptr, K, scale, ws.ptr, ws.bytes, stream),
           "paged_attention");
  return out;
}

static torch::Tensor paged_select(torch::Tensor query, torch::Tensor key_bounds, torch::Tensor page_table,
                                  torch::Tensor seq_lens, int64_t page_size, int64_t n_selected) {
  const int dtype = check_first("query", query);
  const int64_t B = query.size(0), H = query.size(1), D = query.size(3);
  TORCH_CHECK(query.size(2) == 1, "cmpext3 paged: pages are selected for one query column");
  check_data("key_bounds", key_bounds, query);
  const int64_t Hkv = key_bounds.size(1);
  TORCH_CHECK(Hkv >= 1 && H >= 1 && H % Hkv == 0, "cmpext3 paged: ", H, " query heads over ", Hkv, " key heads");
  TORCH_CHECK(key_bounds.size(0) >= 1 && key_bounds.size(0) <= INT32_MAX && key_bounds.size(2) == 2 &&
                  key_bounds.stride(3) == 1,
              "cmpext3 paged: key_bounds must be [pages, heads, 2, head dim]");
  TORCH_CHECK(page_size >= 1 && page_size <= INT32_MAX, "cmpext3 paged: page_size ", page_size);
  TORCH_CHECK(n_selected >= 1 && n_selected <= INT32_MAX, "cmpext3 paged: n_selected ", n_selected);
  const Map map(page_table, seq_lens, c10::nullopt, query);
  const at::hip::HIPGuardMasqueradingAsCUDA guard(query.device());
  torch::Tensor out = torch::empty({B, Hkv, n_selected}, query.options().dtype(at::kInt));
  if (out.numel() == 0) return out;
  TORCH_CHECK(D * query.element_size() % 16 == 0 && D >= 1 && D <= 256,
              "cmpext3 paged: head dim ", D, " is not whole 16-byte chunks up to 256");
  const torch::Tensor q = chunk_rows(query);
  const size_t need = cmpext3_paged_select_workspace_size((int)B, (int)Hkv, map.width);
  torch::Tensor ws;
  if (need > 0) ws = torch::empty({(int64_t)need}, query.options().dtype(at::kByte));
  const Str qs(q), kbs(key_bounds);
  check_rc(cmpext3_paged_select(q.data_ptr(), key_bounds.data_ptr(), out.data_ptr<int32_t>(), dtype, (int)B, (int)H,
                                (int)Hkv, (int)D, (int)key_bounds.size(0), (int)page_size, qs.s, kbs.s, map.pages(),
                                map.width, map.stride, map.lens.data_ptr<int32_t>(), (int)n_selected,
                                need > 0 ? ws.data_ptr() : nullptr, need, stream_of(query)),
           "paged_select");
  return out;
}

namespace cmpext3_binding {

void register_paged(pybind11::module_& m) {
  m.def("paged_append", &paged_append,
        "Keys and values of new tokens into their pages, rotated on the way; returns the rotated queries",
        py::arg("key"), py::arg("value"), py::arg("key_pages"), py::arg("value_pages"), py::arg("page_table"),
        py::arg("seq_lens"), py::arg("query") = py::none(), py::arg("cos") = py::none(), py::arg("sin") = py::none(),
        py::arg("positions") = py::none(), py::arg("new_lens") = py::none(), py::arg("interleaved") = false,
        py::arg("key_bounds") = py::none());
  m.def("paged_attention", &paged_attention, "Attention of new tokens over the pages of their sequences",
        py::arg("query"), py::arg("key_pages"), py::arg("value_pages"), py::arg("page_table"), py::arg("seq_lens"),
        py::arg("scale") = py::none(), py::arg("new_lens") = py::none(), py::arg("selected") = py::none());
  m.def("paged_select", &paged_select, "The pages of each sequence its new token attends to, by key bounds",
        py::arg("query"), py::arg("key_bounds"), py::arg("page_table"), py::arg("seq_lens"), py::arg("page_size"),
        py::arg("n_selected"));
}

}  // namespace cmpext3_binding
