// The binding's functions of the decode step: rotary positions, the paged cache and the
// attention over it. Included by native.cpp only. Each operator has a validating function
// (*_fwd), which takes its outputs and raises the errors, and the call of the Python API,
// which does the ordinary case in one native call (native_calls.hpp).
#pragma once

namespace {

// [..., heads, head_dim], with head_dim contiguous: a contiguous tensor, or [tokens, heads,
// head_dim] with any token and head strides.
struct HeadsView {
  View v;
  int64_t tokens = 0, heads = 0, dim = 0, token_stride = 0, head_stride = 0;
};

HeadsView validate_heads(const char* name, const py::handle& obj) {
  const std::string device_type =
      THPVariable_Check(obj.ptr())
          ? std::string(c10::DeviceTypeName(THPVariable_Unpack(obj.ptr()).device().type(), /*lower_case=*/true))
          : std::string(py::str(obj.attr("device").attr("type")));
  HeadsView h;
  if (device_type != "cuda" || obj.attr("is_contiguous")().cast<bool>()) {
    h.v = validate_tensor(name, obj);  // raises if it is not on a GPU
  } else {
    const std::string type = py::str(obj.attr("dtype"));
    const auto tag = tag_from_dtype_str(type);
    if (!tag) unsupported_dtype(type);
    h.v = View{obj.attr("data_ptr")().cast<uintptr_t>(), *tag, obj.attr("device").attr("index").cast<int64_t>(), {}};
    for (py::handle d : obj.attr("shape")) h.v.shape.push_back(d.cast<int64_t>());
  }
  if (h.v.dtype != F32 && h.v.dtype != F16 && h.v.dtype != BF16) {
    unsupported_dtype(std::string(name) + " is " + tag_debug(h.v.dtype));
  }
  const std::vector<int64_t>& s = h.v.shape;
  if (s.size() < 3) shape_mismatch(std::string(name) + " must be [..., heads, head_dim], got " + shape_str(s));
  h.heads = s[s.size() - 2];
  h.dim = s.back();
  h.tokens = product(s, 0, s.size() - 2);
  h.token_stride = h.heads * h.dim;
  h.head_stride = h.dim;
  if (!obj.attr("is_contiguous")().cast<bool>()) {
    std::vector<int64_t> strides;
    for (py::handle d : obj.attr("stride")()) strides.push_back(d.cast<int64_t>());
    if (s.size() != 3 || strides.size() != 3 || (strides[2] != 1 && h.dim > 1)) {
      value_error(std::string("argument '") + name +
                  "' must be contiguous, or [tokens, heads, head_dim] with a contiguous last dimension");
    }
    h.token_stride = strides[0];
    h.head_stride = strides[1];
  }
  return h;
}

// Whether no two elements share memory, as far as the strides of tokens and heads tell.
bool apart(int64_t tokens, int64_t heads, int64_t dim, int64_t token_stride, int64_t head_stride) {
  if (tokens * heads * dim == 0) return true;
  int64_t n0 = tokens, s0 = token_stride, n1 = heads, s1 = head_stride;
  if (s0 < s1) std::swap(n0, n1), std::swap(s0, s1);
  if (n1 > 1 && s1 < dim) return false;
  return n0 <= 1 || s0 >= (n1 - 1) * (n1 > 1 ? s1 : 0) + dim;
}
bool apart(const HeadsView& h) { return apart(h.tokens, h.heads, h.dim, h.token_stride, h.head_stride); }

// Where heads lie, in bytes.
struct Region {
  int64_t at, tokens, heads, length, token_stride, head_stride;
  Region(uintptr_t ptr, int64_t size, int64_t tokens, int64_t heads, int64_t dim, int64_t token_stride, int64_t head_stride)
      : at((int64_t)ptr), tokens(tokens), heads(heads), length(dim * size), token_stride(tokens > 1 ? token_stride * size : 0),
        head_stride(heads > 1 ? head_stride * size : 0) {}
  // A contiguous tensor.
  Region(uintptr_t ptr, int64_t bytes) : Region(ptr, 1, 1, 1, bytes, 0, 0) {}
  bool empty() const { return tokens * heads * length == 0; }
  int64_t extent() const { return (heads - 1) * head_stride + length; }  // of a token
  int64_t end() const { return at + (tokens - 1) * token_stride + extent(); }
};

// Whether two tensors of heads have memory in common. Exact, but that those of one range with different strides
// of their tokens, and with more than 2^20 pairs of heads at different strides, count as such.
bool share(const Region& a, const Region& b) {
  if (a.empty() || b.empty() || a.end() <= b.at || b.end() <= a.at) return false;
  if (a.tokens > 1 && b.tokens > 1 && a.token_stride != b.token_stride) return true;
  const int64_t period = a.tokens > 1 ? a.token_stride : b.token_stride, apart = b.at - a.at;
  if (period > 0) {  // slices of a row side by side
    const int64_t after = (apart % period + period) % period;
    if (after >= a.extent() && after + b.extent() <= period) return false;
  }
  // x: from a head of a's to one of b's, of the same token; b's of another one are whole periods on.
  const auto meet = [&](int64_t x) {
    const auto by = [&](int64_t t) {
      return t > -a.tokens && t < b.tokens && x + t * period < a.length && x + t * period > -b.length;
    };
    if (period <= 0) return by(0);
    const int64_t t = std::clamp(-x / period, 1 - a.tokens, b.tokens - 1);
    return by(t - 1) || by(t) || by(t + 1);
  };
  const bool even = a.heads == 1 || b.heads == 1 || a.head_stride == b.head_stride;
  if (even) {
    const int64_t stride = a.heads > 1 ? a.head_stride : b.head_stride;
    for (int64_t d = 1 - a.heads; d < b.heads; ++d) {
      if (meet(apart + d * stride)) return true;
    }
    return false;
  }
  if (a.heads > (int64_t(1) << 20) / b.heads) return true;
  for (int64_t i = 0; i < a.heads; ++i) {
    for (int64_t j = 0; j < b.heads; ++j) {
      if (meet(apart + j * b.head_stride - i * a.head_stride)) return true;
    }
  }
  return false;
}
Region region(const HeadsView& h) {
  return {h.v.ptr, h.v.dtype == F32 ? 4 : 2, h.tokens, h.heads, h.dim, h.token_stride, h.head_stride};
}
Region region(const View& v) {
  const int64_t size = v.dtype == F32 ? 4 : v.dtype == F16 || v.dtype == BF16 ? 2 : 1;
  return {v.ptr, size * product(v.shape, 0, v.shape.size())};
}
// An output that is not the input itself.
template <class A, class B>
void check_apart(const char* out, const A& a, const char* other, const B& b) {
  if (share(region(a), region(b))) {
    value_error(std::string("arguments '") + out + "' and '" + other + "' are the same memory, or share some of it");
  }
}

constexpr int64_t kMaxRopeDim = 2048;

// Frequencies float64 [half] of heads of `dim`: half.
int64_t check_frequencies(const RawView& f, int64_t dim, int64_t device) {
  if (f.dtype_str != "torch.float64") unsupported_dtype("frequencies must be float64, got " + f.dtype_str);
  if (f.shape.size() != 1 || 2 * f.shape[0] > dim) {
    shape_mismatch("frequencies must be 1-D with at most head_dim / 2 = " + std::to_string(dim / 2) +
                   " elements, got " + shape_str(f.shape));
  }
  if (f.device_index != device) value_error("device mismatch: 'frequencies' is not on q's device");
  return f.shape[0];
}

bool parse_layout(const std::string& layout) {
  if (layout == "half") return false;
  if (layout == "interleaved") return true;
  value_error("layout must be 'half' or 'interleaved', got \"" + layout + "\"");
}

void check_tokens(const char* name, const View& v, const HeadsView& q) {
  const std::vector<int64_t> want(q.v.shape.begin(), q.v.shape.end() - 2);
  if (v.shape != want) {
    shape_mismatch(std::string(name) + " shape " + shape_str(v.shape) + " must be q's without its heads, " +
                   shape_str(want));
  }
}

void check_like_q(const char* name, const HeadsView& h, const HeadsView& q) {
  check_dtype_matches(name, h.v, q.v, "q");
  check_same_device(name, h.v, q.v, "q");
  const bool leading = h.v.shape.size() == q.v.shape.size() &&
                       std::equal(h.v.shape.begin(), h.v.shape.end() - 2, q.v.shape.begin());
  if (!leading || h.dim != q.dim) {
    shape_mismatch(std::string(name) + " must have q's tokens and head_dim; got q=" + shape_str(q.v.shape) + ", " +
                   name + "=" + shape_str(h.v.shape));
  }
}

void check_rope_sizes(const HeadsView& q, const HeadsView& k) {
  if (q.dim > kMaxRopeDim) shape_mismatch("head_dim (" + std::to_string(q.dim) + ") must be at most 2048");
  if (q.heads + 2 * k.heads > (int64_t(1) << 20) / (q.dim > 0 ? q.dim : 1)) {
    shape_mismatch("a token of more than 2^20 elements");
  }
}

// An output of the same heads as `from`, or `from` itself.
void check_out(const char* name, const HeadsView& out, const HeadsView& from, const char* of) {
  check_dtype_matches(name, out.v, from.v, of);
  check_same_device(name, out.v, from.v, of);
  if (out.v.shape != from.v.shape) shape_mismatch(std::string(name) + " must match " + of + "'s shape");
  if (!apart(out)) value_error(std::string("argument '") + name + "' has elements that share memory: not an output");
  if (out.v.ptr == from.v.ptr && (out.token_stride != from.token_stride || out.head_stride != from.head_stride)) {
    value_error(std::string("argument '") + name + "' overlaps '" + of + "' with other strides");
  }
}

void rope_at_fwd(py::handle q, py::handle k, py::handle positions, py::handle frequencies, py::handle q_out,
                 py::handle k_out, const std::string& layout, double scale, bool inverse) {
  const bool interleaved = parse_layout(layout);
  const HeadsView qv = validate_heads("q", q), kv = validate_heads("k", k);
  const View pv = validate_int64_tensor("positions", positions);
  const RawView fv = validate_and_extract("frequencies", frequencies);
  const HeadsView qo = validate_heads("q_out", q_out), ko = validate_heads("k_out", k_out);
  check_like_q("k", kv, qv);
  check_tokens("positions", pv, qv);
  check_same_device("positions", pv, qv.v, "q");
  const int64_t half = check_frequencies(fv, qv.dim, qv.v.device_index);
  check_rope_sizes(qv, kv);
  check_out("q_out", qo, qv, "q");
  check_out("k_out", ko, kv, "k");
  check_apart("q_out", qo, "k_out", ko);
  check_apart("q_out", qo, "k", kv);
  check_apart("k_out", ko, "q", qv);
  if (qo.v.ptr != qv.v.ptr) check_apart("q_out", qo, "q", qv);
  if (ko.v.ptr != kv.v.ptr) check_apart("k_out", ko, "k", kv);
  const int64_t strides[8] = {qv.token_stride, qv.head_stride, kv.token_stride, kv.head_stride,
                              qo.token_stride, qo.head_stride, ko.token_stride, ko.head_stride};
  const Launch launch(qv.v.device_index);
  check_launch("launch_rope_at_fwd",
               launch_rope_at_fwd((const void*)qv.v.ptr, (const void*)kv.v.ptr, (void*)qo.v.ptr, (void*)ko.v.ptr,
                                  (const int64_t*)pv.ptr, (const void*)fv.ptr, strides, qv.tokens, qv.heads, kv.heads,
                                  qv.dim, half, interleaved, inverse, (float)scale, qv.v.dtype, launch.st));
}

// A cache [pages, page_size, kv_heads, head_dim] of `like`'s type or FP8.
View validate_cache(const char* name, const py::handle& obj, const HeadsView& like, int64_t kv_heads) {
  View c = validate_tensor(name, obj);
  if (c.dtype != like.v.dtype && c.dtype != F8E4M3 && c.dtype != F8E5M2) {
    value_error(std::string("dtype mismatch: '") + name + "' is " + tag_debug(c.dtype) + " but expected " +
                tag_debug(like.v.dtype) + " (as 'q') or FP8");
  }
  check_same_device(name, c, like.v, "q");
  if (c.shape.size() != 4 || c.shape[2] != kv_heads || c.shape[3] != like.dim || c.shape[1] < 1) {
    shape_mismatch(std::string(name) + " must be [pages, page_size, " + std::to_string(kv_heads) + ", " +
                   std::to_string(like.dim) + "] with a page_size of 1 or more, got " + shape_str(c.shape));
  }
  return c;
}

void check_cache_pair(const View& keys, const View& values) {
  check_dtype_matches("value_cache", values, keys, "key_cache");
  if (keys.shape != values.shape) {
    shape_mismatch("key_cache and value_cache must share the same shape; got " + shape_str(keys.shape) + " and " +
                   shape_str(values.shape));
  }
}

bool is_fp8(int32_t tag) { return tag == F8E4M3 || tag == F8E5M2; }

// Scales of an FP8 cache; one of q's type has none.
bool cache_scale_ok(double scale, bool fp8) { return fp8 ? scale >= 1e-30 && scale <= 1e30 : scale == 1.0; }
void check_cache_scales(double key_scale, double value_scale, int32_t cache) {
  if (!cache_scale_ok(key_scale, is_fp8(cache)) || !cache_scale_ok(value_scale, is_fp8(cache))) {
    value_error(is_fp8(cache) ? "key_scale and value_scale must be in [1e-30, 1e30]"
                              : "key_scale and value_scale belong to an FP8 cache: 1 for one of q's type");
  }
}

void rope_to_cache_fwd(py::handle q, py::handle k, py::handle v, py::handle key_cache, py::handle value_cache,
                       py::handle slots, py::handle positions, py::handle frequencies, py::handle q_out,
                       const std::string& layout, double scale, double key_scale, double value_scale) {
  const bool interleaved = parse_layout(layout);
  const HeadsView qv = validate_heads("q", q), kv = validate_heads("k", k), vv = validate_heads("v", v);
  check_like_q("k", kv, qv);
  check_like_q("v", vv, qv);
  if (vv.heads != kv.heads) {
    shape_mismatch("k and v must share the same shape; got k=" + shape_str(kv.v.shape) + ", v=" +
                   shape_str(vv.v.shape));
  }
  const View kc = validate_cache("key_cache", key_cache, qv, kv.heads);
  const View vc = validate_cache("value_cache", value_cache, qv, kv.heads);
  check_cache_pair(kc, vc);
  check_cache_scales(key_scale, value_scale, kc.dtype);
  const View sv = validate_int64_tensor("slots", slots), pv = validate_int64_tensor("positions", positions);
  const RawView fv = validate_and_extract("frequencies", frequencies);
  const HeadsView qo = validate_heads("q_out", q_out);
  check_tokens("slots", sv, qv);
  check_tokens("positions", pv, qv);
  check_same_device("slots", sv, qv.v, "q");
  check_same_device("positions", pv, qv.v, "q");
  const int64_t half = check_frequencies(fv, qv.dim, qv.v.device_index);
  check_rope_sizes(qv, kv);
  check_out("q_out", qo, qv, "q");
  check_apart("q_out", qo, "k", kv);
  check_apart("q_out", qo, "v", vv);
  if (qo.v.ptr != qv.v.ptr) check_apart("q_out", qo, "q", qv);
  check_apart("key_cache", kc, "value_cache", vc);
  const auto check_cache_apart = [&](const char* name, const View& cache) {
    check_apart(name, cache, "q_out", qo);
    check_apart(name, cache, "q", qv);
    check_apart(name, cache, "k", kv);
    check_apart(name, cache, "v", vv);
  };
  check_cache_apart("key_cache", kc);
  check_cache_apart("value_cache", vc);
  const int64_t strides[8] = {qv.token_stride, qv.head_stride, kv.token_stride, kv.head_stride,
                              vv.token_stride, vv.head_stride, qo.token_stride, qo.head_stride};
  const Launch launch(qv.v.device_index);
  check_launch("launch_rope_to_cache_fwd",
               launch_rope_to_cache_fwd((const void*)qv.v.ptr, (const void*)kv.v.ptr, (const void*)vv.v.ptr,
                                        (void*)qo.v.ptr, (void*)kc.ptr, (void*)vc.ptr, (const int64_t*)sv.ptr,
                                        (const int64_t*)pv.ptr, (const void*)fv.ptr, strides, qv.tokens, qv.heads,
                                        kv.heads, qv.dim, half, kc.shape[0] * kc.shape[1], interleaved, (float)scale,
                                        (float)key_scale, (float)value_scale, qv.v.dtype, kc.dtype, launch.st));
}

constexpr int64_t kMaxPositions = int64_t(1) << 30;

// Limits of the attention's launcher that no shape check covers; nullptr if they hold.
const char* attention_limits(int64_t sequences, int64_t heads, int64_t kv_heads, int64_t dim, int64_t pages,
                             int64_t page, int64_t table_width) {
  if (kv_heads < 1 || heads < kv_heads || heads % kv_heads != 0) return "q's heads must be a multiple of the caches'";
  if (dim < 16 || dim > 256 || dim % 16 != 0) return "head_dim must be a multiple of 16, at most 256";
  if (pages > INT32_MAX / page) return "a cache of 2^31 positions or more";
  if (table_width > kMaxPositions / page) return "page_table holds more than 2^30 positions a sequence";
  if (heads > 65536 || sequences > (int64_t(1) << 23) / heads) return "more than 2^23 query heads";
  return nullptr;
}

// 0 for what paged_attention_fwd refuses.
int64_t paged_attention_workspace(py::handle q, py::handle key_cache, py::handle page_table) {
  const HeadsView qv = validate_heads("q", q);
  const RawView kv = validate_and_extract("key_cache", key_cache), tv = validate_and_extract("page_table", page_table);
  const auto tag = tag_from_dtype_str(kv.dtype_str);
  if (qv.v.shape.size() != 3 || kv.shape.size() != 4 || tv.shape.size() != 2 || !tag) return 0;
  return cck_paged_attention_workspace(qv.tokens, qv.heads, kv.shape[2], qv.dim, kv.shape[1], tv.shape[1], *tag);
}

void paged_attention_fwd(py::handle q, py::handle key_cache, py::handle value_cache, py::handle page_table,
                         py::handle lengths, py::handle out, py::handle lse, py::handle workspace, double scale,
                         int64_t window, double key_scale, double value_scale) {
  const HeadsView qv = validate_heads("q", q);
  if (qv.v.shape.size() != 3) shape_mismatch("q must be 3-D [sequences, heads, head_dim], got " + shape_str(qv.v.shape));
  const RawView shape = validate_and_extract("key_cache", key_cache);
  const int64_t kv_heads = shape.shape.size() == 4 ? shape.shape[2] : 0;
  const View kc = validate_cache("key_cache", key_cache, qv, kv_heads);
  const View vc = validate_cache("value_cache", value_cache, qv, kv_heads);
  check_cache_pair(kc, vc);
  check_cache_scales(key_scale, value_scale, kc.dtype);
  const View tv = validate_int64_tensor("page_table", page_table), lv = validate_int64_tensor("lengths", lengths);
  check_same_device("page_table", tv, qv.v, "q");
  check_same_device("lengths", lv, qv.v, "q");
  if (tv.shape.size() != 2 || tv.shape[0] != qv.tokens) {
    shape_mismatch("page_table must be [" + std::to_string(qv.tokens) + " sequences, pages of each], got " +
                   shape_str(tv.shape));
  }
  if (lv.shape != std::vector<int64_t>{qv.tokens}) {
    shape_mismatch("lengths shape " + shape_str(lv.shape) + " must be [" + std::to_string(qv.tokens) + "]");
  }
  if (window < 0) value_error("window must be 0 (none) or more, got " + std::to_string(window));
  if (const char* wrong = attention_limits(qv.tokens, qv.heads, kv_heads, qv.dim, kc.shape[0], kc.shape[1],
                                          tv.shape[1])) {
    shape_mismatch(std::string(wrong) + "; got q=" + shape_str(qv.v.shape) + ", key_cache=" + shape_str(kc.shape) +
                   ", page_table=" + shape_str(tv.shape));
  }
  const View ov = validate_tensor("out", out);
  check_dtype_matches("out", ov, qv.v, "q");
  check_same_device("out", ov, qv.v, "q");
  if (ov.shape != qv.v.shape) shape_mismatch("out must match q's shape");
  std::optional<View> ev, wv;
  if (!lse.is_none()) {
    ev = validate_tensor("lse", lse);
    require_f32("lse", *ev);
    check_same_device("lse", *ev, qv.v, "q");
    if (ev->shape != std::vector<int64_t>{qv.tokens, qv.heads}) shape_mismatch("lse must be [sequences, heads]");
  }
  const int64_t bytes =
      cck_paged_attention_workspace(qv.tokens, qv.heads, kv_heads, qv.dim, kc.shape[1], tv.shape[1], kc.dtype);
  if (!workspace.is_none()) {
    wv = validate_tensor("workspace", workspace);
    require_f32("workspace", *wv);
    check_same_device("workspace", *wv, qv.v, "q");
  }
  if ((wv ? product(wv->shape, 0, wv->shape.size()) * 4 : 0) < bytes) {
    shape_mismatch("workspace must have " + std::to_string(bytes / 4) + " elements or more");
  }
  const Launch launch(qv.v.device_index);
  check_launch("launch_paged_attention_fwd",
               launch_paged_attention_fwd((const void*)qv.v.ptr, (const void*)kc.ptr, (const void*)vc.ptr,
                                          (const int64_t*)tv.ptr, (const int64_t*)lv.ptr, (void*)ov.ptr,
                                          ev ? (float*)ev->ptr : nullptr, wv ? (void*)wv->ptr : nullptr,
                                          qv.token_stride, qv.head_stride, qv.tokens, qv.heads, kv_heads, qv.dim,
                                          kc.shape[0], kc.shape[1], tv.shape[1], window, (float)scale,
                                          (float)key_scale, (float)value_scale, qv.v.dtype, kc.dtype, launch.st));
}

}  // namespace
