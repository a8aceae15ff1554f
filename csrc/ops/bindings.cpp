// bindings.cpp -- tilelang._tl_ops: the serving operators on torch tensors.
//
// Checks every argument (type, device, shape, strides) before anything is launched, allocates outputs and
// workspaces from torch's allocator on the current stream (so a call can be captured into a graph, and two calls
// share no scratch memory) and hands plain argument blocks to the gfx950 kernels, or to their host forms for CPU
// tensors.  Tensors of any device may be passed, whatever device is current.
#include <ATen/EmptyTensor.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/hip/HIPStream.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>
#include <sstream>
#include <string>
#include <vector>

#include "ops.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = c10::optional<Tensor>;

namespace {

template <typename... A>
std::string text(const A&... a) {
  std::ostringstream os;
  (os << ... << a);
  return os.str();
}

// The message is put together only where the check fails.
#define NEED_AS(error, ok, ...) \
  do {                          \
    if (!(ok)) throw error(text(__VA_ARGS__)); \
  } while (0)
#define NEED(ok, ...) NEED_AS(py::value_error, ok, __VA_ARGS__)

// One call's tensors: all on the first one's device, none asking for a gradient or carrying a tangent.
struct Call {
  const char* name;
  c10::optional<c10::Device> device;

  void on(const Tensor& t, const char* arg) {
    NEED(t.defined(), name, ": argument '", arg, "' is an undefined tensor");
    if (!device) {
      NEED(t.is_cpu() || t.is_cuda(), name, ": argument '", arg, "' must be a CPU or a ROCm (cuda) tensor, got ",
           t.device().str());
      device = t.device();
    }
    NEED(t.device() == *device, name, ": argument '", arg, "' is on ", t.device().str(), ", expected ",
         device->str());
    data(t, arg);
    NEED(!t.is_neg(), name, ": argument '", arg, "' is a view whose memory holds the negative, pass its resolve_neg()");
    if (t.unsafeGetTensorImpl()->autograd_meta() == nullptr) return;
    if (t.requires_grad() && at::GradMode::is_enabled())
      throw std::runtime_error(text(name, ": argument '", arg, "' requires a gradient, and the operator has none"));
    if (c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined())
      throw std::runtime_error(text(name, ": argument '", arg, "' has a tangent, and the operator has no derivative"));
  }
  // The tensor's memory.  Fake and functional tensors, lazy zeros, wrappers and sparse ones have none.
  void* data(const Tensor& t, const char* arg) const {
    if (t.defined() && t.layout() == c10::kStrided && t.has_storage() && t.storage().device() == t.device()) {
      void* const p = t.data_ptr();
      if (p != nullptr || t.numel() == 0) return p;
    }
    throw py::value_error(text(name, ": argument '", arg, "' has a null data pointer"));
  }
  void dims(const Tensor& t, const char* arg, int64_t n) const {
    NEED(t.dim() == n, name, ": argument '", arg, "' has ", t.dim(), " dims, expected ", n);
  }
  void size(const Tensor& t, const char* arg, int d, int64_t n) const {
    NEED(t.size(d) == n, name, ": argument '", arg, "' dim ", d, " is ", t.size(d), ", expected ", n);
  }
  void dtype(const Tensor& t, const char* arg, c10::ScalarType s) const {
    NEED_AS(py::type_error, t.scalar_type() == s, name, ": argument '", arg, "' has dtype ",
            c10::toString(t.scalar_type()), ", expected ", c10::toString(s));
  }
  void contiguous(const Tensor& t, const char* arg) const {
    NEED(t.is_contiguous(), name, ": argument '", arg, "' must be contiguous");
  }
  tl_ops::Type type(const Tensor& t, const char* arg, bool f32) const {
    switch (t.scalar_type()) {
      case c10::ScalarType::BFloat16: return tl_ops::kBF16;
      case c10::ScalarType::Half: return tl_ops::kF16;
      case c10::ScalarType::Float:
        if (f32) return tl_ops::kF32;
        [[fallthrough]];
      default:
        throw py::type_error(text(name, ": argument '", arg, "' has dtype ", c10::toString(t.scalar_type()),
                                  ", expected BFloat16", f32 ? ", Half or Float" : " or Half"));
    }
  }
  // `t` is about to be written: autograd has to see that what it saved of it is stale.
  void writes(const Tensor& t) const {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  }
  bool cpu() const { return device->is_cpu(); }
  // Memory of the current stream, straight from the device's allocator.
  Tensor fresh(c10::IntArrayRef sizes, c10::ScalarType s) const {
    if (cpu()) return at::detail::empty_cpu(sizes, s);
    return at::detail::empty_cuda(sizes, s, *device, c10::nullopt);
  }
  tl_ops::Stream stream() const { return c10::hip::getCurrentHIPStream(device->index()).stream(); }
};

Tensor last_dense(const Tensor& t) { return t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous(); }

// The memory from a tensor's first byte to its last one.
struct Range {
  uintptr_t begin, end;
  bool meets(const Range& r) const { return begin < r.end && r.begin < end; }
};
Range range_of(const Tensor& t) {
  const auto begin = reinterpret_cast<uintptr_t>(t.data_ptr());
  if (t.numel() == 0) return {begin, 0};  // meets nothing
  const auto sizes = t.sizes(), strides = t.strides();
  int64_t last = 0;
  for (size_t d = 0; d < sizes.size(); ++d) last += (sizes[d] - 1) * strides[d];
  return {begin, begin + uintptr_t((last + 1) * int64_t(t.element_size()))};
}

// [..., n] as [rows, n] with dense rows
Tensor rows_of(const Tensor& t, int64_t n) {
  return last_dense(t.dim() == 2 ? t : t.reshape({t.numel() / n, n}));
}

// ------------------------------------------------------------------------------------------- norm

py::tuple add_rms_norm_quant(const Tensor& x, const Tensor& weight, const OptTensor& residual, double eps,
                             int64_t group, bool pow2, bool return_norm) {
  Call c{"add_rms_norm_quant", {}};
  c.on(x, "x");
  c.on(weight, "weight");
  if (residual) c.on(*residual, "residual");
  NEED(x.dim() >= 1, c.name, ": argument 'x' has 0 dims, expected 1 or more");
  const int64_t n = x.size(-1);
  tl_ops::NormQuantArgs a{};
  a.type = c.type(x, "x", true);
  NEED(n >= 1 && n <= tl_ops::kNormMaxWidth, c.name, ": rows of ", n, " elements, expected 1 to ",
       tl_ops::kNormMaxWidth);
  c.dims(weight, "weight", 1);
  c.size(weight, "weight", 0, n);
  c.dtype(weight, "weight", x.scalar_type());
  if (residual) {
    c.dtype(*residual, "residual", x.scalar_type());
    NEED(residual->sizes() == x.sizes(), c.name, ": residual ", residual->sizes(), " does not match x ", x.sizes());
  }
  NEED(group == 0 || (group >= 16 && group <= 512 && (group & (group - 1)) == 0), c.name, ": group is ", group,
       ", expected 0 (one scale for each row) or a power of two from 16 to 512");
  NEED(group == 0 || n % group == 0, c.name, ": rows of ", n, " elements do not split into groups of ", group);

  c10::DeviceGuard guard(*c.device);
  const Tensor x2 = rows_of(x, n), w = weight.contiguous(), r2 = residual ? rows_of(*residual, n) : Tensor();
  a.rows = x2.size(0);
  NEED(a.rows <= INT32_MAX, c.name, ": ", a.rows, " rows, expected fewer than 2^31");
  a.width = int(n);
  a.group = int(group ? group : n);
  a.eps = float(eps);
  a.pow2 = pow2;
  std::vector<int64_t> scales(x.sizes().begin(), x.sizes().end());
  scales.back() = n / a.group;
  const Tensor q = c.fresh(x.sizes(), c10::ScalarType::Float8_e4m3fn);
  const Tensor s = c.fresh(scales, c10::ScalarType::Float);
  const Tensor h = residual ? c.fresh(x.sizes(), x.scalar_type()) : Tensor();
  const Tensor y = return_norm ? c.fresh(x.sizes(), x.scalar_type()) : Tensor();
  a.x = c.data(x2, "x");
  a.x_stride = x2.stride(0);
  a.weight = c.data(w, "weight");
  if (residual) a.residual = c.data(r2, "residual"), a.residual_stride = r2.stride(0), a.h = h.data_ptr();
  if (return_norm) a.y = y.data_ptr();
  a.q = static_cast<uint8_t*>(q.data_ptr());
  a.scale = static_cast<float*>(s.data_ptr());
  if (c.cpu())
    tl_ops::norm_quant_cpu(a);
  else
    tl_ops::norm_quant_hip(a, c.stream());
  const auto or_none = [](const Tensor& t) -> py::object { return t.defined() ? py::cast(t) : py::none(); };
  return py::make_tuple(q, s, or_none(h), or_none(y));
}

// ------------------------------------------------------------------------------------------- cache

tl_ops::Cache cache_of(Call& c, const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs, int64_t dim,
                       const Tensor& table, const Tensor& lengths, int64_t batch, Range (&pools)[4]) {
  const std::pair<const Tensor*, const char*> all[] = {{&k, "cache.k"},             {&v, "cache.v"},
                                                       {&ks, "cache.k_scale"},      {&vs, "cache.v_scale"},
                                                       {&table, "block_table"},     {&lengths, "lengths"}};
  for (const auto& t : all) c.on(*t.first, t.second);
  c.dtype(k, "cache.k", c10::ScalarType::Float8_e4m3fn);
  c.dtype(v, "cache.v", c10::ScalarType::Float8_e4m3fn);
  c.dims(k, "cache.k", 4);
  c.dims(v, "cache.v", 4);
  const int64_t pages = k.size(0), heads = k.size(1), page = k.size(2), wide = k.size(3);
  NEED(pages >= 1 && heads >= 1 && heads <= 65535 && pages * heads <= INT32_MAX, c.name, ": a cache of ", pages,
       " pages and ", heads, " heads");
  NEED(page >= 16 && page <= 1024 && (page & (page - 1)) == 0, c.name, ": pages of ", page,
       " tokens, expected a power of two from 16 to 1024");
  NEED(wide >= 64 && wide <= 256 && wide % 64 == 0, c.name, ": cache.k is ", wide,
       " wide, expected a multiple of 64 up to 256");
  NEED(dim >= 1 && dim <= wide && dim > wide - 64, c.name, ": heads of ", dim, " in a cache that is ", wide, " wide");
  for (int d = 0; d < 4; ++d) c.size(v, "cache.v", d, k.size(d < 2 ? d : 5 - d));
  const std::pair<const Tensor*, const char*> scales[] = {{&ks, "cache.k_scale"}, {&vs, "cache.v_scale"}};
  for (const auto& t : scales) {
    c.dtype(*t.first, t.second, c10::ScalarType::Float);
    c.dims(*t.first, t.second, 2);
    c.size(*t.first, t.second, 0, pages);
    c.size(*t.first, t.second, 1, heads);
  }
  for (int i = 0; i < 4; ++i) c.contiguous(*all[i].first, all[i].second);
  NEED(reinterpret_cast<uintptr_t>(k.data_ptr()) % 16 == 0 && reinterpret_cast<uintptr_t>(v.data_ptr()) % 16 == 0,
       c.name, ": the cache must begin on a 16-byte boundary");
  c.dtype(table, "block_table", c10::ScalarType::Int);
  c.dims(table, "block_table", 2);
  c.size(table, "block_table", 0, batch);
  NEED(table.size(1) <= 1 || table.stride(1) == 1, c.name, ": block_table's rows must be dense");
  NEED(table.size(1) * page <= (int64_t(1) << 30), c.name, ": block_table holds ", table.size(1), " pages of ", page,
       " tokens, expected at most 2^30 tokens");
  c.dtype(lengths, "lengths", c10::ScalarType::Int);
  c.dims(lengths, "lengths", 1);
  c.size(lengths, "lengths", 0, batch);
  c.contiguous(lengths, "lengths");
  for (int i = 0; i < 4; ++i) {
    pools[i] = range_of(*all[i].first);
    for (int j = 0; j < i; ++j)
      NEED(!pools[i].meets(pools[j]), c.name, ": ", all[j].second, " and ", all[i].second, " share memory");
  }
  tl_ops::Cache r{};
  r.k = static_cast<uint8_t*>(k.data_ptr());
  r.v = static_cast<uint8_t*>(v.data_ptr());
  r.k_scale = static_cast<float*>(ks.data_ptr());
  r.v_scale = static_cast<float*>(vs.data_ptr());
  r.table = static_cast<const int*>(table.data_ptr());
  r.lengths = static_cast<const int*>(lengths.data_ptr());
  r.pages = pages;
  r.table_stride = table.stride(0);
  r.table_width = int(table.size(1));
  r.heads = int(heads);
  r.dim = int(dim);
  r.wide = int(wide);
  while ((1 << r.page_shift) < page) ++r.page_shift;
  return r;
}

void kv_cache_append(const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs, int64_t dim,
                     const Tensor& new_k, const Tensor& new_v, const Tensor& table, const Tensor& lengths) {
  Call c{"kv_cache_append", {}};
  c.on(new_k, "k");
  c.on(new_v, "v");
  c.dims(new_k, "k", 4);
  tl_ops::AppendArgs a{};
  a.type = c.type(new_k, "k", true);
  c.dtype(new_v, "v", new_k.scalar_type());
  NEED(new_v.sizes() == new_k.sizes(), c.name, ": v ", new_v.sizes(), " does not match k ", new_k.sizes());
  Range pools[4];
  a.cache = cache_of(c, k, v, ks, vs, dim, table, lengths, new_k.size(0), pools);
  c.size(new_k, "k", 2, a.cache.heads);
  c.size(new_k, "k", 3, dim);
  NEED(new_k.size(0) <= 32767, c.name, ": ", new_k.size(0), " sequences, expected at most 32767");
  NEED(new_k.size(1) <= (int64_t(1) << 19), c.name, ": ", new_k.size(1), " new tokens, expected at most 2^19");
  a.batch = int(new_k.size(0));
  a.new_tokens = int(new_k.size(1));
  // what the workgroups write must be nothing that others read
  const std::pair<const Tensor*, const char*> read[] = {
      {&new_k, "k"}, {&new_v, "v"}, {&table, "block_table"}, {&lengths, "lengths"}};
  const std::pair<const Tensor*, const char*> written[] = {
      {&k, "cache.k"}, {&v, "cache.v"}, {&ks, "cache.k_scale"}, {&vs, "cache.v_scale"}};
  for (const auto& r : read) {
    const Range range = range_of(*r.first);
    for (int i = 0; i < 4; ++i)
      NEED(!range.meets(pools[i]), c.name, ": ", r.second, " and ", written[i].second, " share memory");
  }
  for (const auto& w : written) c.writes(*w.first);
  c10::DeviceGuard guard(*c.device);
  const Tensor x[2] = {last_dense(new_k), last_dense(new_v)};
  for (int i = 0; i < 2; ++i) {
    a.x[i] = c.data(x[i], i ? "v" : "k");
    a.stride_b[i] = x[i].stride(0);
    a.stride_t[i] = x[i].stride(1);
    a.stride_h[i] = x[i].stride(2);
  }
  if (c.cpu())
    tl_ops::kv_append_cpu(a);
  else
    tl_ops::kv_append_hip(a, c.stream());
}

py::object kv_cache_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs,
                              int64_t dim, const Tensor& table, const Tensor& lengths,
                              const c10::optional<double>& scale, bool return_lse) {
  Call c{"kv_cache_attention", {}};
  c.on(q, "q");
  c.dims(q, "q", 4);
  tl_ops::AttentionArgs a{};
  a.type = c.type(q, "q", false);
  Range pools[4];
  a.cache = cache_of(c, k, v, ks, vs, dim, table, lengths, q.size(0), pools);
  c.size(q, "q", 3, dim);
  const int64_t batch = q.size(0), tokens = q.size(1), heads = q.size(2);
  NEED(heads >= 1 && heads % a.cache.heads == 0, c.name, ": ", heads, " query heads do not share ", a.cache.heads,
       " key heads");
  NEED(batch <= 65535, c.name, ": ", batch, " sequences, expected at most 65535");
  NEED(tokens * heads <= (int64_t(1) << 27) && batch * tokens * heads <= INT32_MAX, c.name, ": ", batch, " x ", tokens,
       " x ", heads, " query rows are too many for one call");
  a.batch = int(batch);
  a.new_tokens = int(tokens);
  a.heads = int(heads);
  a.scale = scale ? float(*scale) : 1.0f / std::sqrt(float(dim));
  NEED(std::isfinite(a.scale), c.name, ": sm_scale is ", *scale, ", expected a finite float32");
  c10::DeviceGuard guard(*c.device);
  const Tensor q2 = last_dense(q), out = c.fresh(q.sizes(), q.scalar_type());
  const Tensor lse = return_lse ? c.fresh({batch, tokens, heads}, c10::ScalarType::Float) : Tensor();
  a.q = c.data(q2, "q");
  a.stride_b = q2.stride(0);
  a.stride_t = q2.stride(1);
  a.stride_h = q2.stride(2);
  a.out = out.data_ptr();
  if (return_lse) a.lse = static_cast<float*>(lse.data_ptr());
  if (c.cpu()) {
    tl_ops::kv_attention_cpu(a);
  } else if (out.numel()) {
    tl_ops::kv_attention_plan(a, int64_t(a.cache.table_width) << a.cache.page_shift);
    Tensor parts;  // freed on return: torch's allocator hands it out again behind this stream's work only
    if (a.splits > 1) {
      const int64_t n = batch * tokens * heads * a.splits;
      parts = c.fresh({n * (dim + 2)}, c10::ScalarType::Float);
      a.part_o = static_cast<float*>(parts.data_ptr());
      a.part_ml = a.part_o + n * dim;
    }
    tl_ops::kv_attention_hip(a, c.stream());
  }
  if (!return_lse) return py::cast(out);
  return py::make_tuple(out, lse);
}

// ------------------------------------------------------------------------------------------- beams

py::tuple beam_select(const Tensor& logits, const Tensor& scores, int64_t take, const OptTensor& finished,
                      int64_t eos) {
  Call c{"beam_select", {}};
  c.on(logits, "logits");
  c.on(scores, "scores");
  if (finished) c.on(*finished, "finished");
  c.dims(scores, "scores", 2);
  c.dtype(scores, "scores", c10::ScalarType::Float);
  const int64_t batch = scores.size(0), beams = scores.size(1);
  NEED(logits.dim() == 2 || logits.dim() == 3, c.name, ": argument 'logits' has ", logits.dim(),
       " dims, expected 2 or 3");
  tl_ops::BeamArgs a{};
  a.type = c.type(logits, "logits", true);
  if (logits.dim() == 3) {
    c.size(logits, "logits", 0, batch);
    c.size(logits, "logits", 1, beams);
  } else {
    c.size(logits, "logits", 0, batch * beams);
  }
  const int64_t vocab = logits.size(-1);
  NEED(vocab >= 1 && vocab <= tl_ops::kBeamMaxVocab && beams >= 1 && beams <= tl_ops::kBeamMaxBeams, c.name, ": ",
       beams, " beams over ", vocab, " tokens, expected 1 to ", tl_ops::kBeamMaxBeams, " beams over 1 to ",
       tl_ops::kBeamMaxVocab, " tokens");
  NEED(take >= 1 && take <= tl_ops::kBeamMaxTake && take <= beams * vocab, c.name, ": take is ", take,
       ", expected 1 to ", std::min<int64_t>(tl_ops::kBeamMaxTake, beams * vocab));
  NEED(batch * beams <= 65535, c.name, ": ", batch * beams, " rows, expected at most 65535");
  if (finished) {
    c.dtype(*finished, "finished", c10::ScalarType::Bool);
    NEED(finished->sizes() == scores.sizes(), c.name, ": finished ", finished->sizes(), " does not match scores ",
         scores.sizes());
    NEED(eos >= 0 && eos < vocab, c.name, ": eos_id is ", eos, ", expected one of the ", vocab, " tokens");
  }
  c10::DeviceGuard guard(*c.device);
  const Tensor x = rows_of(logits, vocab), sc = scores.contiguous(), fin = finished ? finished->contiguous() : Tensor();
  const Tensor out_scores = c.fresh({batch, take}, c10::ScalarType::Float),
               out_parents = c.fresh({batch, take}, c10::ScalarType::Long),
               out_tokens = c.fresh({batch, take}, c10::ScalarType::Long);
  a.logits = c.data(x, "logits");
  a.stride = x.stride(0);
  a.scores = static_cast<const float*>(c.data(sc, "scores"));
  if (finished) a.finished = static_cast<const uint8_t*>(c.data(fin, "finished"));
  a.eos = eos;
  a.out_scores = static_cast<float*>(out_scores.data_ptr());
  a.out_parents = static_cast<int64_t*>(out_parents.data_ptr());
  a.out_tokens = static_cast<int64_t*>(out_tokens.data_ptr());
  a.batch = batch;
  a.beams = int(beams);
  a.take = int(take);
  a.vocab = int(vocab);
  if (c.cpu()) {
    tl_ops::beam_select_cpu(a);
  } else if (batch) {
    a.chunks = tl_ops::beam_select_chunks(a.vocab);
    const Tensor parts = c.fresh({tl_ops::beam_select_scratch(batch * beams, a.chunks, a.take)},
                                 c10::ScalarType::Long);
    tl_ops::beam_select_hip(a, static_cast<uint64_t*>(parts.data_ptr()), c.stream());
  }
  return py::make_tuple(out_scores, out_parents, out_tokens);
}

void reorder_states(const std::vector<Tensor>& states, const Tensor& parents, const c10::optional<int64_t>& length) {
  Call c{"reorder_states", {}};
  c.on(parents, "parents");
  c.dtype(parents, "parents", c10::ScalarType::Long);
  c.dims(parents, "parents", 2);
  c.contiguous(parents, "parents");
  const int64_t batch = parents.size(0), beams = parents.size(1), rows = batch * beams;
  NEED(beams >= 1 && beams <= tl_ops::kReorderMaxBeams, c.name, ": ", beams, " beams, expected 1 to ",
       tl_ops::kReorderMaxBeams);
  NEED(batch <= 65535, c.name, ": ", batch, " sequences, expected at most 65535");
  NEED(!length || *length >= 0, c.name, ": length is ", length.value_or(0), ", expected 0 or more");
  std::vector<tl_ops::ReorderState> moved;
  for (const Tensor& t : states) {
    c.on(t, "states");
    NEED(t.dim() >= (length ? 2 : 1), c.name, ": a state has ", t.dim(), " dims, expected ", length ? 2 : 1,
         " or more");
    NEED(t.size(0) == rows, c.name, ": a state has ", t.size(0), " rows, expected ", batch, " x ", beams);
    NEED(!length || *length <= t.size(1), c.name, ": length is ", length.value_or(0), ", and a state has ", t.size(1));
    if (t.numel() == 0) continue;
    // what moves of a row: its elements, dense from the row's beginning
    int64_t moves = 1;
    for (int64_t d = t.dim() - 1; d >= 1; --d) {
      const int64_t n = d == 1 && length ? *length : t.size(d);
      NEED(n <= 1 || t.stride(d) == moves, c.name, ": what moves of a state's row must be contiguous");
      moves *= n;
    }
    const int64_t bytes = moves * int64_t(t.element_size()), stride = t.stride(0) * int64_t(t.element_size());
    if (bytes == 0) continue;
    NEED(rows == 1 || stride >= bytes, c.name, ": a state's rows overlap");
    NEED(bytes <= tl_ops::kReorderMaxBytes, c.name, ": ", bytes, " bytes of a state's row, expected at most ",
         tl_ops::kReorderMaxBytes);
    moved.push_back({static_cast<uint8_t*>(t.data_ptr()), stride, bytes, 0});
  }
  // No byte may be moved twice.  In the order of their addresses, two states that share a range must be columns of
  // one buffer: rows equally far apart, the second's bytes behind the first's and before its next row.
  std::vector<tl_ops::ReorderState> sorted = moved;
  std::sort(sorted.begin(), sorted.end(), [](const auto& p, const auto& q) { return p.data < q.data; });
  const auto end = [&](const tl_ops::ReorderState& s) { return s.data + (rows - 1) * s.stride + s.bytes; };
  const auto* own = static_cast<const uint8_t*>(parents.data_ptr());
  for (const auto& t : sorted)
    NEED(end(t) <= own || own + parents.nbytes() <= t.data, c.name, ": parents and a state share memory");
  for (size_t i = 0; i < sorted.size(); ++i)
    for (size_t j = i + 1; j < sorted.size() && sorted[j].data < end(sorted[i]); ++j) {
      const int64_t off = (sorted[j].data - sorted[i].data) % std::max<int64_t>(sorted[i].stride, 1);
      NEED(rows > 1 && sorted[i].stride == sorted[j].stride && off >= sorted[i].bytes &&
               off + sorted[j].bytes <= sorted[i].stride,
           c.name, ": two states share memory");
    }
  for (const Tensor& t : states) c.writes(t);
  c10::DeviceGuard guard(*c.device);
  tl_ops::ReorderArgs a{};
  a.parents = static_cast<const int64_t*>(parents.data_ptr());
  a.batch = batch;
  a.beams = int(beams);
  for (size_t i = 0; i < moved.size(); i += tl_ops::kReorderStates) {
    a.states = int(std::min<size_t>(moved.size() - i, tl_ops::kReorderStates));
    std::copy_n(moved.begin() + i, a.states, a.state);
    if (c.cpu())
      tl_ops::reorder_cpu(a);
    else
      tl_ops::reorder_hip(a, c.stream());
  }
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("add_rms_norm_quant", &add_rms_norm_quant);
  m.def("kv_cache_append", &kv_cache_append);
  m.def("kv_cache_attention", &kv_cache_attention);
  m.def("beam_select", &beam_select);
  m.def("reorder_states", &reorder_states);
}
