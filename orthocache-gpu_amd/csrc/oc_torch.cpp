// The entry points of orthocache_gpu.rotary, .paged_cache and .changed_scores
// for torch tensors: argument checks, outputs and workspaces from torch's
// allocator, and one call of the C ABI (include/orthocache_paged.h) on torch's
// current stream.  These calls take a few microseconds on the GPU at a decode
// step's sizes, and the same checks in Python took 14 to 20; here they take 3
// to 5.  Host code only: the kernels are liborthocache_hip's.
#include <torch/csrc/utils/pybind.h>

#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <cmath>
#include <limits>
#include <optional>
#include <string>

#include "orthocache_hip.h"
#include "orthocache_paged.h"

namespace py = pybind11;

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

template <typename... A>
[[noreturn]] void raise(PyObject* type, const A&... a) {
  PyErr_SetString(type, std::string(c10::str(a...)).c_str());
  throw py::error_already_set();
}

template <typename... A>
void need(bool ok, const A&... a) {
  if (!ok) raise(PyExc_ValueError, a...);
}

// a status of the library as the package's OrthoCacheHIPError
void check(const char* name, int rc) {
  if (rc) py::module_::import("orthocache_gpu._native").attr("check")(name, rc);
}

int32_t i32(int64_t v, const char* what) {
  need(v >= std::numeric_limits<int32_t>::min() && v <= std::numeric_limits<int32_t>::max(), what, " ", v,
       " does not fit 32 bits");
  return (int32_t)v;
}

int dtype_code(at::ScalarType t, const char* what, bool fp8 = true) {
  switch (t) {
    case at::kFloat: return OC_F32;
    case at::kHalf: return OC_F16;
    case at::kBFloat16: return OC_BF16;
    case at::kFloat8_e4m3fn:
      if (fp8) return OC_FP8_E4M3FN;
      [[fallthrough]];
    default: raise(PyExc_TypeError, "orthocache_gpu: unsupported ", what, " dtype ", t);
  }
}

// Collects the device of a call's tensors.
struct OnGpu {
  c10::Device dev{c10::kCPU};
  void operator()(const Tensor& t) {
    if (!t.is_cuda())
      raise(PyExc_RuntimeError, "orthocache_gpu runs on an AMD GPU only: got a tensor on '", t.device().str(),
            "'. Move the inputs to the GPU (there is no CPU fallback).");
    if (dev.is_cpu()) dev = t.device();
    else if (t.device() != dev)
      raise(PyExc_RuntimeError, "orthocache_gpu: tensors on different devices (", dev.str(), " vs ", t.device().str(), ")");
  }
  void operator()(const OptTensor& t) {
    if (t) (*this)(*t);
  }
};

// These operators record no gradient: an input that wants one is refused
// rather than cut off silently.
void no_grad_needed(const char* what, const Tensor& t) {
  if (t.requires_grad() && at::GradMode::is_enabled())
    raise(PyExc_RuntimeError, what, " records no gradient: call it under torch.no_grad(), or detach its inputs");
}
void no_grad_needed(const char* what, const OptTensor& t) {
  if (t) no_grad_needed(what, *t);
}

// whether elements of t may share memory (an expanded view, say)
bool overlaps(const Tensor& t) {
  if (t.is_contiguous()) return false;
  std::vector<std::pair<int64_t, int64_t>> d;
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.size(i) > 1) d.emplace_back(std::abs(t.stride(i)), t.size(i));
  std::sort(d.begin(), d.end());
  int64_t reach = 0;  // of the elements along the dimensions of smaller strides
  for (auto& [st, n] : d) {
    if (st <= reach) return true;
    reach += st * (n - 1);
  }
  return false;
}

// t, or a copy of it, with a contiguous last dimension
Tensor rows_ready(const Tensor& t) { return t.stride(-1) == 1 || t.size(-1) <= 1 ? t : t.contiguous(); }

// t, or a copy of its own, with a contiguous last dimension, 16-byte aligned
// rows, and (tokens >= 0) rows along that dimension that share no memory
Tensor ready16(const Tensor& t, int64_t tokens = -1) {
  const int64_t es = t.element_size(), last = t.dim() - 1;
  bool ok = t.stride(last) == 1 && (uintptr_t)t.data_ptr() % 16 == 0 && (tokens < 0 || t.stride(tokens) >= t.size(last));
  for (int64_t i = 0; i < last && ok; ++i) ok = t.stride(i) * es % 16 == 0;
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

// an int32 tensor of the shape (-1: any size) with a contiguous last dimension
Tensor index_tensor(const Tensor& t, std::initializer_list<int64_t> shape, const char* what) {
  if (t.scalar_type() != at::kInt) raise(PyExc_TypeError, what, " must be int32, got ", t.scalar_type());
  bool ok = t.dim() == (int64_t)shape.size();
  int64_t i = 0;
  for (int64_t n : shape) {
    ok = ok && (n < 0 || t.size(i) == n);
    ++i;
  }
  need(ok, what, " must be ", at::IntArrayRef(shape), ", got ", t.sizes());
  return rows_ready(t);
}

Tensor tile_flags(const Tensor& m, int64_t batch, int64_t heads) {
  if (m.scalar_type() != at::kBool && m.scalar_type() != at::kByte)
    raise(PyExc_TypeError, "evict_mask must be bool or uint8, got ", m.scalar_type());
  need(m.dim() == 3 && m.size(0) == batch && (heads >= 0 ? m.size(1) == heads : m.size(1) >= 1), "evict_mask must be (",
       batch, ", ", heads >= 0 ? std::to_string(heads) : "heads", ", tiles), got ", m.sizes());
  return rows_ready(m);
}

void check_caches(const Tensor& k, const Tensor& v, bool layers) {
  need((k.dim() == 4 || (layers && k.dim() == 5)) && k.sizes() == v.sizes(), "k_cache and v_cache must be ",
       layers ? "4-D or 5-D" : "4-D", " of one shape, got ", k.sizes(), " and ", v.sizes());
  if (k.scalar_type() != v.scalar_type())
    raise(PyExc_TypeError, "k_cache and v_cache must share a dtype (", k.scalar_type(), ", ", v.scalar_type(), ")");
  const int64_t bs = k.size(-2);
  need(bs >= 1 && !(bs & (bs - 1)), "block_size (", bs, ") must be a power of 2");
  need(k.size(-1) <= 1 || (k.stride(-1) == 1 && v.stride(-1) == 1), "cache rows must be contiguous along head_dim");
}

// whether two tensors are known to share memory (interleaved views are not)
bool share(const Tensor& a, const Tensor& b, bool same_counts = true) {
  const at::MemOverlapStatus s = at::get_overlap_status(a, b);
  return s == at::MemOverlapStatus::Partial || (same_counts && s == at::MemOverlapStatus::Full);
}

void written_caches(const Tensor& k, const Tensor& v) {
  no_grad_needed("a written cache", k), no_grad_needed("a written cache", v);
  need(!share(k, v), "k_cache and v_cache must be different memory");
  need(!overlaps(k) && !overlaps(v), "elements of a cache that is written may not share memory");
}

void cache_scales(const Tensor& cache, double ks, double vs) {
  for (double s : {ks, vs}) {
    need(s > 0 && std::isfinite((float)s) && (float)s > 0, "scales must be positive and finite, got ", s);
    need(s == 1.0 || cache.scalar_type() == at::kFloat8_e4m3fn, "k_scale and v_scale are for float8_e4m3fn caches, not ",
         cache.scalar_type());
  }
}

// the columns that a table turns (0 without one)
int32_t check_table(const OptTensor& f, int64_t d, const std::string& layout) {
  need(layout == "half" || layout == "interleaved", "layout must be one of ('half', 'interleaved'), got '", layout, "'");
  if (!f) return 0;
  need(f->scalar_type() == at::kDouble && f->dim() == 1 && f->is_contiguous(), "inv_freq must be a contiguous float64 vector");
  need(2 * f->size(0) <= d, "the table turns ", 2 * f->size(0), " columns, head_dim is ", d);
  return (int32_t)(2 * f->size(0));
}

Tensor check_positions(const Tensor& p) {
  if (p.scalar_type() != at::kInt && p.scalar_type() != at::kLong)
    raise(PyExc_TypeError, "positions must be int32 or int64, got ", p.scalar_type());
  return rows_ready(p);
}

void* stream_of(c10::Device d) { return (void*)c10::hip::getCurrentHIPStream(d.index()).stream(); }

Tensor bytes(size_t n, c10::Device d) { return at::empty({(int64_t)n}, at::TensorOptions().dtype(at::kByte).device(d)); }

Tensor int_zero(c10::Device d) { return at::zeros({1}, at::TensorOptions().dtype(at::kInt).device(d)); }

template <typename T>
T* ptr(const OptTensor& t) {
  return t ? (T*)t->data_ptr() : nullptr;
}

// ------------------------------------------------------------ rotary

py::object apply_rotary(const Tensor& q_in, const OptTensor& k_in, const Tensor& positions_in, const Tensor& inv_freq,
                        double scale, const std::string& layout, bool backward, bool inplace) {
  no_grad_needed("apply_rotary", q_in);
  no_grad_needed("apply_rotary", k_in);
  OnGpu on;
  on(q_in), on(k_in), on(positions_in), on(inv_freq);
  const bool flat = q_in.dim() == 3;
  need(flat || q_in.dim() == 4, "q must be (tokens, heads, d) or (batch, heads, tokens, d), got ", q_in.sizes());
  oc_rotary_params p{};
  p.dtype = dtype_code(q_in.scalar_type(), "q", false);
  const int64_t d = q_in.size(-1);
  p.rotary_dim = check_table(inv_freq, d, layout);
  if (k_in) {
    bool ok = k_in->dim() == q_in.dim();
    for (int64_t i = 0; ok && i < q_in.dim(); ++i) ok = i == 1 || k_in->size(i) == q_in.size(i);
    need(ok, "k ", k_in->sizes(), " does not match q ", q_in.sizes());
    if (k_in->scalar_type() != q_in.scalar_type())
      raise(PyExc_TypeError, "q and k must share a dtype (", q_in.scalar_type(), ", ", k_in->scalar_type(), ")");
  }
  const int64_t tokens = flat ? q_in.size(0) : q_in.size(2), batch = flat ? 1 : q_in.size(0);
  const Tensor positions = check_positions(positions_in);
  need((positions.dim() == 1 && positions.size(0) == tokens) ||
           (positions.dim() == 2 && positions.size(0) == batch && positions.size(1) == tokens),
       "positions must be (", tokens, ",) or (", batch, ", ", tokens, "), got ", positions.sizes());
  const c10::DeviceGuard guard(on.dev);
  Tensor x[2] = {q_in, k_in ? *k_in : Tensor()}, y[2];
  for (int i = 0; i < (k_in ? 2 : 1); ++i) {
    if (inplace) {
      need((x[i].stride(-1) == 1 || d <= 1) && !overlaps(x[i]),
           "in place, the last dimension must be contiguous and no elements may share memory");
      y[i] = x[i];
    } else {
      x[i] = rows_ready(x[i]);
      y[i] = at::empty_like(x[i]);
      if (y[i].stride(-1) != 1) y[i] = at::empty(x[i].sizes(), x[i].options());
    }
    const int64_t b = flat ? -1 : 0, h = 1, s = flat ? 0 : 2;
    p.x[i] = x[i].data_ptr(), p.y[i] = y[i].data_ptr();
    p.x_stride_b[i] = b < 0 ? 0 : x[i].stride(0), p.x_stride_h[i] = x[i].stride(h), p.x_stride_s[i] = x[i].stride(s);
    p.y_stride_b[i] = b < 0 ? 0 : y[i].stride(0), p.y_stride_h[i] = y[i].stride(h), p.y_stride_s[i] = y[i].stride(s);
    p.heads[i] = i32(x[i].size(1), "heads");
  }
  need(!inplace || !k_in || ((x[0].data_ptr() != x[1].data_ptr() || !x[0].numel() || !x[1].numel()) && !share(x[0], x[1])),
       "in place, q and k must be different tensors");
  p.batch = i32(batch, "batch"), p.tokens = i32(tokens, "tokens"), p.head_dim = i32(d, "head_dim");
  p.interleaved = layout == "interleaved", p.backward = backward;
  p.positions = positions.data_ptr(), p.positions_64 = positions.scalar_type() == at::kLong;
  p.positions_stride_b = positions.dim() == 2 && batch > 1 ? positions.stride(0) : 0;
  p.inv_freq = (const double*)inv_freq.data_ptr(), p.scale = (float)scale;
  check("oc_apply_rotary", oc_apply_rotary(&p, stream_of(on.dev)));
  return k_in ? py::object(py::make_tuple(y[0], y[1])) : py::cast(y[0]);
}

// ------------------------------------------------------------ append

OptTensor append_paged(const Tensor& k_in, const Tensor& v_in, const Tensor& kc, const Tensor& vc, const Tensor& tables_in,
                       const Tensor& lens_in, const OptTensor& q_in, const OptTensor& cu_in, const OptTensor& pos_in,
                       const OptTensor& inv_freq, double scale, const std::string& layout, double k_scale, double v_scale,
                       bool sync) {
  no_grad_needed("append_paged", k_in), no_grad_needed("append_paged", v_in), no_grad_needed("append_paged", q_in);
  OnGpu on;
  on(k_in), on(v_in), on(kc), on(vc), on(tables_in), on(lens_in), on(q_in), on(cu_in), on(pos_in), on(inv_freq);
  check_caches(kc, vc, false);
  written_caches(kc, vc);
  const int64_t hkv = kc.size(1), d = kc.size(3);
  need(k_in.dim() == 3 && k_in.size(1) == hkv && k_in.size(2) == d && v_in.sizes() == k_in.sizes(),
       "k and v must be (tokens, ", hkv, ", ", d, "), got ", k_in.sizes(), " and ", v_in.sizes());
  const int64_t tokens = k_in.size(0);
  need(!q_in || (q_in->dim() == 3 && q_in->size(0) == tokens && q_in->size(2) == d), "q must be (", tokens, ", heads, ", d,
       "), got ", q_in ? q_in->sizes() : at::IntArrayRef());
  if (v_in.scalar_type() != k_in.scalar_type() || (q_in && q_in->scalar_type() != k_in.scalar_type()))
    raise(PyExc_TypeError, "q, k and v must share a dtype");
  cache_scales(kc, k_scale, v_scale);
  oc_append_params p{};
  const Tensor lens = index_tensor(lens_in, {-1}, "context_lens");
  const int64_t n = lens.size(0);
  const Tensor tables = index_tensor(tables_in, {n, -1}, "block_tables");
  OptTensor cu, pos;
  if (cu_in) cu = index_tensor(*cu_in, {n + 1}, "cu_seqlens");
  else need(tokens == n, tokens, " tokens for ", n, " sequences need cu_seqlens");
  p.rotary_dim = check_table(inv_freq, d, layout);
  p.dtype = dtype_code(k_in.scalar_type(), "k", false), p.cache_dtype = dtype_code(kc.scalar_type(), "cache");
  if (pos_in) {
    need(pos_in->dim() == 1 && pos_in->size(0) == tokens, "positions must be (", tokens, ",), got ", pos_in->sizes());
    pos = check_positions(*pos_in);
    p.positions = pos->data_ptr(), p.positions_64 = pos->scalar_type() == at::kLong;
  }
  const c10::DeviceGuard guard(on.dev);
  const Tensor k = rows_ready(k_in), v = rows_ready(v_in);
  OptTensor q, out, flag;
  if (q_in) {
    q = rows_ready(*q_in);
    out = at::empty(q->sizes(), q->options());
    if (n == 0) out->zero_();
    p.q = q->data_ptr(), p.q_stride_s = q->stride(0), p.q_stride_h = q->stride(1), p.num_q_heads = i32(q->size(1), "heads");
    p.q_out = out->data_ptr(), p.q_out_stride_s = out->stride(0), p.q_out_stride_h = out->stride(1);
  }
  if (sync) flag = int_zero(on.dev);
  p.k = k.data_ptr(), p.k_stride_s = k.stride(0), p.k_stride_h = k.stride(1);
  p.v = v.data_ptr(), p.v_stride_s = v.stride(0), p.v_stride_h = v.stride(1);
  p.k_cache = kc.data_ptr(), p.v_cache = vc.data_ptr();
  p.k_cache_stride_b = kc.stride(0), p.k_cache_stride_h = kc.stride(1), p.k_cache_stride_s = kc.stride(2);
  p.v_cache_stride_b = vc.stride(0), p.v_cache_stride_h = vc.stride(1), p.v_cache_stride_s = vc.stride(2);
  p.tokens = i32(tokens, "tokens"), p.num_seqs = i32(n, "sequences"), p.num_kv_heads = i32(hkv, "heads");
  p.head_dim = i32(d, "head_dim"), p.block_size = i32(kc.size(2), "block_size"), p.num_blocks = kc.size(0);
  p.max_blocks = i32(tables.size(1), "max_blocks"), p.block_tables = (const int32_t*)tables.data_ptr();
  p.bt_stride = tables.stride(0), p.context_lens = (const int32_t*)lens.data_ptr(), p.cu_seqlens = ptr<const int32_t>(cu);
  p.interleaved = layout == "interleaved", p.inv_freq = ptr<const double>(inv_freq), p.scale = (float)scale;
  p.k_scale = (float)k_scale, p.v_scale = (float)v_scale, p.error_flag = ptr<int32_t>(flag);
  check("oc_append_paged", oc_append_paged(&p, stream_of(on.dev)));
  need(!sync || flag->item<int>() == 0, "block_tables holds no block in [0, num_blocks) for some of the tokens");
  return out;
}

// ------------------------------------------------------------ attention

// the score changes, and the tensors that the block points to
struct Mods {
  oc_score_mods m{};
  OptTensor slopes, prefix, evict;
};

Mods score_mods(std::optional<double> scale, double softcap, const OptTensor& slopes, int64_t window, const OptTensor& prefix,
                const OptTensor& evict, int64_t batch, int64_t hq, int64_t hkv, int64_t d) {
  Mods r;
  const double s = scale ? *scale : 1.0 / std::sqrt((double)d);
  need(std::isfinite((float)s), "scale ", s, " must be finite");
  need(softcap >= 0 && std::isfinite((float)softcap) && (softcap == 0 || (float)softcap > 0), "softcap ", softcap,
       " must be 0 (none) or positive");
  need(window >= 0, "window ", window, " must be 0 (none) or positive");
  r.m.scale = (float)s, r.m.softcap = (float)softcap;
  r.m.window = (int32_t)std::min<int64_t>(window, std::numeric_limits<int32_t>::max());
  if (slopes) {
    need(slopes->scalar_type() == at::kFloat && slopes->dim() == 1 && slopes->size(0) == hq, "alibi_slopes must be float32 (",
         hq, ",)");
    r.slopes = slopes->contiguous();
    r.m.slopes = (const float*)r.slopes->data_ptr();
  }
  if (prefix) {
    r.prefix = index_tensor(*prefix, {batch}, "prefix_lens");
    r.m.prefix_lens = (const int32_t*)r.prefix->data_ptr();
  }
  if (evict) {
    r.evict = tile_flags(*evict, batch, hkv);
    r.m.evict = (const uint8_t*)r.evict->data_ptr();
    r.m.evict_stride_b = r.evict->stride(0), r.m.evict_stride_h = r.evict->stride(1);
    r.m.evict_cols = i32(r.evict->size(2), "tiles");
  }
  return r;
}

Tensor attend_paged(const Tensor& q_in, const Tensor& kc, const Tensor& vc, const Tensor& tables_in, const Tensor& lens_in,
                    std::optional<double> scale, double softcap, const OptTensor& slopes, int64_t window,
                    const OptTensor& prefix, double k_scale, double v_scale, const OptTensor& evict,
                    std::optional<int64_t> num_splits, bool sync, const OptTensor& out_in, bool portable) {
  for (const Tensor* t : {&q_in, &kc, &vc}) no_grad_needed("attend_paged", *t);
  no_grad_needed("attend_paged", slopes);
  OnGpu on;
  on(q_in), on(kc), on(vc), on(tables_in), on(lens_in), on(slopes), on(prefix), on(evict);
  check_caches(kc, vc, false);
  const int64_t hkv = kc.size(1), d = kc.size(3);
  need(q_in.dim() == 3 && q_in.size(2) == d, "q must be (num_seqs, heads, ", d, "), got ", q_in.sizes());
  const int64_t n = q_in.size(0), hq = q_in.size(1);
  need(hkv > 0 && hq % hkv == 0, hq, " query heads on ", hkv, " kv heads");
  oc_attend_paged_params p{};
  p.dtype = dtype_code(q_in.scalar_type(), "q", false);
  if (kc.scalar_type() != q_in.scalar_type() && kc.scalar_type() != at::kFloat8_e4m3fn)
    raise(PyExc_TypeError, "the cache must have q's dtype (", q_in.scalar_type(), ") or float8_e4m3fn, got ", kc.scalar_type());
  p.cache_dtype = dtype_code(kc.scalar_type(), "cache");
  cache_scales(kc, k_scale, v_scale);
  const Tensor tables = index_tensor(tables_in, {n, -1}, "block_tables");
  const Tensor lens = index_tensor(lens_in, {n}, "context_lens");
  need(!num_splits || *num_splits >= 1, "num_splits (", num_splits.value_or(1), ") must be positive");
  const c10::DeviceGuard guard(on.dev);
  Tensor out;
  if (out_in) {
    out = *out_in;
    need(out.dim() == 3 && out.sizes() == q_in.sizes() && out.scalar_type() == q_in.scalar_type() && out.device() == on.dev &&
             (d <= 1 || out.stride(2) == 1) && !overlaps(out),
         "out must be a (", n, ", ", hq, ", ", d, ") ", q_in.scalar_type(), " tensor on ", on.dev.str(),
         " with a contiguous last dim and no elements that share memory");
    no_grad_needed("attend_paged", out);
    need(!share(out, q_in, false) && !share(out, kc) && !share(out, vc), "out may be q, but share no other memory with the inputs");
  } else {
    out = at::empty(q_in.sizes(), q_in.options().memory_format(at::MemoryFormat::Contiguous));
  }
  const Tensor q = ready16(q_in);
  const Mods mods = score_mods(scale, softcap, slopes, window, prefix, evict, n, hq, hkv, d);
  OptTensor flag, ws;
  if (sync) flag = int_zero(on.dev);
  p.q = q.data_ptr(), p.q_stride_b = q.stride(0), p.q_stride_h = q.stride(1);
  p.k = kc.data_ptr(), p.v = vc.data_ptr();
  p.k_stride_b = kc.stride(0), p.k_stride_h = kc.stride(1), p.k_stride_s = kc.stride(2);
  p.v_stride_b = vc.stride(0), p.v_stride_h = vc.stride(1), p.v_stride_s = vc.stride(2);
  p.block_tables = (const int32_t*)tables.data_ptr(), p.bt_stride = tables.stride(0), p.num_blocks = kc.size(0);
  p.context_lens = (const int32_t*)lens.data_ptr(), p.max_blocks = i32(tables.size(1), "max_blocks");
  p.block_size = i32(kc.size(2), "block_size");
  p.num_seqs = i32(n, "sequences"), p.num_q_heads = i32(hq, "heads"), p.num_kv_heads = i32(hkv, "heads");
  p.head_dim = i32(d, "head_dim"), p.k_scale = (float)k_scale, p.v_scale = (float)v_scale, p.mods = mods.m;
  p.num_splits = i32(num_splits.value_or(0), "num_splits"), p.portable = portable;
  p.out = out.data_ptr(), p.out_stride_b = out.stride(0), p.out_stride_h = out.stride(1), p.error_flag = ptr<int32_t>(flag);
  if (const size_t size = oc_attend_paged_workspace_size(&p)) {
    ws = bytes(size, on.dev);  // of the call's own: two captured graphs replayed at once share nothing
    p.workspace = ws->data_ptr(), p.workspace_bytes = size;
  }
  check("oc_attend_paged", oc_attend_paged(&p, stream_of(on.dev)));
  need(!sync || flag->item<int>() == 0, "block_tables holds a block id outside [0, num_blocks)");
  return out;
}

Tensor attend_prompt(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, std::optional<double> scale, double softcap,
                     const OptTensor& slopes, int64_t window, const OptTensor& prefix, const OptTensor& docs_in,
                     const OptTensor& evict) {
  for (const Tensor* t : {&q_in, &k_in, &v_in}) no_grad_needed("attend_prompt", *t);
  no_grad_needed("attend_prompt", slopes);
  OnGpu on;
  on(q_in), on(k_in), on(v_in), on(slopes), on(prefix), on(docs_in), on(evict);
  need(q_in.dim() == 4 && k_in.dim() == 4 && v_in.sizes() == k_in.sizes(), "q (B, Hq, Sq, d) and k, v (B, Hkv, Skv, d) expected, got ",
       q_in.sizes(), ", ", k_in.sizes(), ", ", v_in.sizes());
  const int64_t B = q_in.size(0), hq = q_in.size(1), sq = q_in.size(2), d = q_in.size(3), hkv = k_in.size(1), skv = k_in.size(2);
  need(k_in.size(0) == B && k_in.size(3) == d && hkv > 0 && hq % hkv == 0, "k ", k_in.sizes(), " does not match q ", q_in.sizes());
  if (k_in.scalar_type() != q_in.scalar_type() || v_in.scalar_type() != q_in.scalar_type())
    raise(PyExc_TypeError, "q, k and v must share a dtype (", q_in.scalar_type(), ", ", k_in.scalar_type(), ", ", v_in.scalar_type(), ")");
  oc_attend_prompt_params p{};
  p.dtype = dtype_code(q_in.scalar_type(), "q", false);
  if (d != 64 && d != 128) raise(PyExc_NotImplementedError, "head_dim ", d, " is not supported (64 or 128)");
  const Mods mods = score_mods(scale, softcap, slopes, window, prefix, evict, B, hq, hkv, d);
  const c10::DeviceGuard guard(on.dev);
  OptTensor docs, ws;
  if (docs_in) {
    docs = index_tensor(docs_in->dim() == 1 ? docs_in->unsqueeze(0).expand({B, -1}) : *docs_in, {B, skv}, "documents");
    p.documents = (const int32_t*)docs->data_ptr(), p.documents_stride_b = docs->stride(0);
  }
  const Tensor q = ready16(q_in), k = ready16(k_in, 2), v = ready16(v_in, 2);
  Tensor out = at::empty({B, hq, sq, d}, q_in.options().memory_format(at::MemoryFormat::Contiguous));
  p.q = q.data_ptr(), p.q_stride_b = q.stride(0), p.q_stride_h = q.stride(1), p.q_stride_s = q.stride(2);
  p.k = k.data_ptr(), p.k_stride_b = k.stride(0), p.k_stride_h = k.stride(1), p.k_stride_s = k.stride(2);
  p.v = v.data_ptr(), p.v_stride_b = v.stride(0), p.v_stride_h = v.stride(1), p.v_stride_s = v.stride(2);
  p.out = out.data_ptr(), p.out_stride_b = out.stride(0), p.out_stride_h = out.stride(1), p.out_stride_s = out.stride(2);
  p.batch = i32(B, "batch"), p.num_q_heads = i32(hq, "heads"), p.num_kv_heads = i32(hkv, "heads");
  p.q_len = i32(sq, "q_len"), p.kv_len = i32(skv, "kv_len"), p.head_dim = i32(d, "head_dim"), p.mods = mods.m;
  if (const size_t size = oc_attend_prompt_workspace_size(&p)) {
    ws = bytes(size, on.dev);
    p.workspace = ws->data_ptr(), p.workspace_bytes = size;
  }
  check("oc_attend_prompt", oc_attend_prompt(&p, stream_of(on.dev)));
  return out;
}

// ------------------------------------------------------------ pages

constexpr int64_t kMaxSeqs = 4096;

struct Tables {
  Tensor t, l, r, s;
};
using OutTables = std::optional<std::tuple<Tensor, Tensor, Tensor, Tensor>>;

Tables out_tables(const OutTables& out, int64_t rows, int64_t cols, int64_t blocks, c10::Device dev,
                  std::initializer_list<const Tensor*> inputs) {
  if (!out) {
    // one allocation: the tables, the lengths, the counts and the status
    const Tensor flat = at::empty({rows * cols + rows + blocks + 1}, at::TensorOptions().dtype(at::kInt).device(dev));
    const int64_t a = rows * cols, b = a + rows, c = b + blocks;
    return {flat.as_strided({rows, cols}, {cols, 1}, 0), flat.as_strided({rows}, {1}, a), flat.as_strided({blocks}, {1}, b),
            flat.as_strided({1}, {1}, c)};
  }
  const auto& [t, l, r, s] = *out;
  auto fits = [&](const Tensor& x, at::IntArrayRef shape, const char* what) {
    need(x.scalar_type() == at::kInt && x.sizes() == shape && x.device() == dev && x.is_contiguous(), "out.", what,
         " must be a contiguous int32 ", shape, " tensor on ", dev.str());
    const char *lo = (const char*)x.data_ptr(), *hi = lo + 4 * x.numel();
    for (const Tensor* i : inputs) {
      if (!i->defined() || !i->numel() || !x.numel()) continue;
      int64_t reach = 1;
      for (int64_t e = 0; e < i->dim(); ++e) reach += (i->size(e) - 1) * i->stride(e);
      const char* b = (const char*)i->data_ptr();
      need(!(b < hi && lo < b + reach * i->element_size()), "out.", what, " overlaps an input: the old tables must stay");
    }
  };
  const Tensor* parts[] = {&t, &l, &r, &s};
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < i; ++j) need(!share(*parts[i], *parts[j]), "two tensors of out share memory");
  fits(t, {rows, cols}, "block_tables"), fits(l, {rows}, "context_lens"), fits(r, {blocks}, "ref_counts"), fits(s, {1}, "status");
  return {t, l, r, s};
}

py::tuple fork_pages(Tensor kc, Tensor vc, const Tensor& tables_in, const Tensor& lens_in, const Tensor& refs_in,
                     const OptTensor& parents_in, const OptTensor& fresh_in, int64_t fresh_all, std::optional<int64_t> max_blocks,
                     const OutTables& out) {
  OnGpu on;
  on(kc), on(vc), on(tables_in), on(lens_in), on(refs_in), on(parents_in), on(fresh_in);
  check_caches(kc, vc, true);
  written_caches(kc, vc);
  if (kc.dim() == 4) kc = kc.unsqueeze(0), vc = vc.unsqueeze(0);
  const int64_t nb = kc.size(1);
  const Tensor lens = index_tensor(lens_in, {-1}, "context_lens");
  const int64_t n = lens.size(0);
  const Tensor tables = index_tensor(tables_in, {n, -1}, "block_tables"), refs = index_tensor(refs_in, {nb}, "ref_counts");
  const c10::DeviceGuard guard(on.dev);
  Tensor parents, fresh;
  int64_t children = n;
  if (parents_in) {
    parents = index_tensor(*parents_in, {-1}, "parents");
    children = parents.size(0);
  }
  if (n > kMaxSeqs || children > kMaxSeqs)
    raise(PyExc_NotImplementedError, "at most ", kMaxSeqs, " sequences and children, got ", n, " and ", children);
  if (fresh_in) {
    fresh = index_tensor(*fresh_in, {children}, "new_tokens");
  } else {
    need(fresh_all >= 0, "new_tokens ", fresh_all, " is negative");
    if (fresh_all) fresh = at::full({children}, i32(fresh_all, "new_tokens"), at::TensorOptions().dtype(at::kInt).device(on.dev));
  }
  const int64_t cols = max_blocks.value_or(tables.size(1));
  need(cols >= 0, "max_blocks ", cols, " is negative");
  const Tables o = out_tables(out, children, cols, nb, on.dev, {&tables, &lens, &refs, &parents, &fresh});
  oc_fork_params p{};
  p.k_cache = kc.data_ptr(), p.v_cache = vc.data_ptr();
  p.k_stride_l = kc.stride(0), p.k_stride_b = kc.stride(1), p.k_stride_h = kc.stride(2), p.k_stride_s = kc.stride(3);
  p.v_stride_l = vc.stride(0), p.v_stride_b = vc.stride(1), p.v_stride_h = vc.stride(2), p.v_stride_s = vc.stride(3);
  p.cache_dtype = dtype_code(kc.scalar_type(), "cache"), p.layers = nb ? i32(kc.size(0), "layers") : 0;
  p.num_kv_heads = i32(kc.size(2), "heads"), p.head_dim = i32(kc.size(4), "head_dim"), p.block_size = i32(kc.size(3), "block_size");
  p.num_seqs = (int32_t)n, p.num_children = (int32_t)children, p.max_blocks = i32(tables.size(1), "max_blocks");
  p.out_max_blocks = i32(cols, "max_blocks"), p.num_blocks = nb;
  p.block_tables = (const int32_t*)tables.data_ptr(), p.bt_stride = tables.stride(0);
  p.context_lens = (const int32_t*)lens.data_ptr(), p.ref_counts = (const int32_t*)refs.data_ptr();
  p.parents = parents.defined() ? (const int32_t*)parents.data_ptr() : nullptr;
  p.new_tokens = fresh.defined() ? (const int32_t*)fresh.data_ptr() : nullptr;
  p.out_block_tables = (int32_t*)o.t.data_ptr(), p.out_bt_stride = cols, p.out_context_lens = (int32_t*)o.l.data_ptr();
  p.out_ref_counts = (int32_t*)o.r.data_ptr(), p.status = (int32_t*)o.s.data_ptr();
  const size_t size = oc_fork_pages_workspace_size(&p);
  const Tensor ws = bytes(std::max<size_t>(size, 1), on.dev);
  p.workspace = ws.data_ptr(), p.workspace_bytes = size;
  check("oc_fork_pages", oc_fork_pages(&p, stream_of(on.dev)));
  return py::make_tuple(o.t, o.l, o.r, o.s);
}

py::tuple evict_pages(const Tensor& tables_in, const Tensor& lens_in, const Tensor& refs_in, const Tensor& mask_in,
                      int64_t block_size, const OutTables& out) {
  OnGpu on;
  on(tables_in), on(lens_in), on(refs_in), on(mask_in);
  const Tensor lens = index_tensor(lens_in, {-1}, "context_lens");
  const int64_t n = lens.size(0);
  const Tensor tables = index_tensor(tables_in, {n, -1}, "block_tables"), refs = index_tensor(refs_in, {-1}, "ref_counts");
  need(block_size >= 1 && 64 % block_size == 0, "block_size (", block_size, ") must divide a tile of 64 tokens");
  const c10::DeviceGuard guard(on.dev);
  const Tensor mask = tile_flags(mask_in.dim() == 2 ? mask_in.unsqueeze(1) : mask_in, n, -1);
  const int64_t cols = tables.size(1), nb = refs.size(0), tiles = (cols * block_size + 63) / 64;
  const Tables o = out_tables(out, n, cols, nb, on.dev, {&tables, &lens, &refs, &mask});
  Tensor map = at::empty({n, tiles}, at::TensorOptions().dtype(at::kInt).device(on.dev));
  oc_evict_params p{};
  p.num_seqs = i32(n, "sequences"), p.num_kv_heads = i32(mask.size(1), "heads"), p.block_size = (int32_t)block_size;
  p.max_blocks = i32(cols, "max_blocks"), p.num_blocks = nb;
  p.block_tables = (const int32_t*)tables.data_ptr(), p.bt_stride = tables.stride(0);
  p.context_lens = (const int32_t*)lens.data_ptr(), p.ref_counts = (const int32_t*)refs.data_ptr();
  p.evict = (const uint8_t*)mask.data_ptr(), p.evict_stride_b = mask.stride(0), p.evict_stride_h = mask.stride(1);
  p.evict_cols = i32(mask.size(2), "tiles"), p.tile_map_cols = i32(tiles, "tiles");
  p.out_block_tables = (int32_t*)o.t.data_ptr(), p.out_bt_stride = cols, p.out_context_lens = (int32_t*)o.l.data_ptr();
  p.out_ref_counts = (int32_t*)o.r.data_ptr(), p.tile_map = (int32_t*)map.data_ptr(), p.status = (int32_t*)o.s.data_ptr();
  check("oc_evict_pages", oc_evict_pages(&p, stream_of(on.dev)));
  return py::make_tuple(o.t, o.l, o.r, o.s, map);
}

}  // namespace

PYBIND11_MODULE(_oc_torch, m) {
  m.def("overlaps", &overlaps);
  m.def("apply_rotary", &apply_rotary);
  m.def("append_paged", &append_paged);
  m.def("attend_paged", &attend_paged);
  m.def("attend_prompt", &attend_prompt);
  m.def("fork_pages", &fork_pages);
  m.def("evict_pages", &evict_pages);
}
