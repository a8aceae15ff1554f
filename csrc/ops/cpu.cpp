// cpu.cpp -- the serving operators on host tensors: their definitions, element by element in float32 (the beam
// search's values and the attention's sums in float64), with the bounds checks of the device kernels.  For the models'
// CPU runs and tests.
#include <c10/util/BFloat16.h>
#include <c10/util/Float8_e4m3fn.h>
#include <c10/util/Half.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <limits>
#include <vector>

#include "ops.h"

namespace tl_ops {
namespace {

constexpr float kFp8Max = 448.0f, kAmaxFloor = 1e-4f;
constexpr float kInf = std::numeric_limits<float>::infinity();

float load(const void* p, int64_t i, Type t) {
  if (t == kF32) return static_cast<const float*>(p)[i];
  if (t == kF16) return static_cast<const c10::Half*>(p)[i];
  return static_cast<const c10::BFloat16*>(p)[i];
}

void store(void* p, int64_t i, Type t, float v) {
  if (t == kF32)
    static_cast<float*>(p)[i] = v;
  else if (t == kF16)
    static_cast<c10::Half*>(p)[i] = v;
  else
    static_cast<c10::BFloat16*>(p)[i] = v;
}

uint8_t to_fp8(float v) { return c10::Float8_e4m3fn(v).x; }
float from_fp8(uint8_t c) { return c10::Float8_e4m3fn(c, c10::Float8_e4m3fn::from_bits()); }

float pow2_scale(float amax) {
  if (amax == kInf) return 0x1p120f;  // that of the largest value, as the kernels take it from the bits
  int e;
  const float m = std::frexp(amax / kFp8Max, &e);
  return std::ldexp(1.0f, m == 0.5f ? e - 1 : e);
}

// The pool's page that holds position `at` of sequence b, or -1.
int64_t page_of(const Cache& c, int b, int64_t at) {
  const int64_t nth = at >> c.page_shift;
  if (at < 0 || nth >= c.table_width) return -1;
  const int id = c.table[b * c.table_stride + nth];
  return id >= 0 && id < c.pages ? id : -1;
}

}  // namespace

void norm_quant_cpu(const NormQuantArgs& a) {
  std::vector<float> y(a.width);
  for (int64_t row = 0; row < a.rows; ++row) {
    double ss = 0.0;
    for (int j = 0; j < a.width; ++j) {
      float h = load(a.x, row * a.x_stride + j, a.type);
      if (a.residual) h += load(a.residual, row * a.residual_stride + j, a.type);
      if (a.h) store(a.h, row * a.width + j, a.type, h);
      ss += double(h) * h;
      y[j] = h;
    }
    const float r = 1.0f / std::sqrt(float(ss / a.width) + a.eps);
    for (int j = 0; j < a.width; ++j) {
      y[j] *= r * load(a.weight, j, a.type);
      if (a.y) store(a.y, row * a.width + j, a.type, y[j]);
    }
    for (int g = 0; g < a.width / a.group; ++g) {
      float m = kAmaxFloor;
      for (int j = 0; j < a.group; ++j) m = std::fmax(m, std::fabs(y[g * a.group + j]));
      const float s = a.pow2 ? pow2_scale(m) : m / kFp8Max;
      a.scale[row * (a.width / a.group) + g] = s;
      for (int j = 0; j < a.group; ++j) a.q[row * a.width + g * a.group + j] = to_fp8(y[g * a.group + j] / s);
    }
  }
}

void kv_append_cpu(const AppendArgs& a) {
  const Cache& c = a.cache;
  const int page = 1 << c.page_shift;
  for (int b = 0; b < a.batch; ++b) {
    const int64_t end = std::min<int64_t>(c.lengths[b], int64_t(c.table_width) * page);
    const int64_t begin = int64_t(c.lengths[b]) - a.new_tokens;
    for (int64_t lo = std::max<int64_t>(begin, 0); lo < end;) {
      const int64_t hi = std::min<int64_t>(end, (lo / page + 1) * page), id = page_of(c, b, lo);
      for (int w = 0; id >= 0 && w < 2; ++w)
        for (int h = 0; h < c.heads; ++h) {
          const auto x = [&](int64_t at, int d) {
            return load(a.x[w], b * a.stride_b[w] + (at - begin) * a.stride_t[w] + h * a.stride_h[w] + d, a.type);
          };
          uint8_t* pool = (w ? c.v : c.k) + (id * c.heads + h) * int64_t(page) * c.wide;
          const auto code = [&](int64_t slot, int d) -> uint8_t& {
            return pool[w ? d * page + slot : slot * c.wide + d];
          };
          float amax = kAmaxFloor;
          for (int64_t at = lo; at < hi; ++at)
            for (int d = 0; d < c.dim; ++d) {
              const float v = std::fabs(x(at, d));
              if (v < kInf) amax = std::fmax(amax, v);
            }
          float& scale = (w ? c.v_scale : c.k_scale)[id * c.heads + h];
          const float before = lo % page ? scale : 0.0f, after = std::fmax(pow2_scale(amax), before);
          scale = after;
          if (after > before)
            for (int64_t slot = 0; slot < lo % page; ++slot)
              for (int d = 0; d < c.wide; ++d) code(slot, d) = to_fp8(from_fp8(code(slot, d)) * (before / after));
          for (int64_t at = lo; at < hi; ++at)
            for (int d = 0; d < c.wide; ++d) {
              const float v = d < c.dim ? x(at, d) / after : 0.0f;
              code(at % page, d) = to_fp8(v > kFp8Max ? kFp8Max : v < -kFp8Max ? -kFp8Max : v);
            }
        }
      lo = hi;
    }
  }
}

void kv_attention_cpu(const AttentionArgs& a) {
  const Cache& c = a.cache;
  const int page = 1 << c.page_shift, per = a.heads / c.heads;
  std::vector<float> q(c.dim), s;
  std::vector<double> o(c.dim);  // sums of values up to float32's largest
  std::vector<int64_t> where;
  for (int b = 0; b < a.batch; ++b) {
    const int64_t len = c.lengths[b], most = int64_t(c.table_width) * page;
    for (int i = 0; i < a.new_tokens; ++i)
      for (int h = 0; h < a.heads; ++h) {
        const int64_t keys = std::min(std::max<int64_t>(len - a.new_tokens + i + 1, 0), most);
        for (int d = 0; d < c.dim; ++d)
          q[d] = load(a.q, b * a.stride_b + i * a.stride_t + h * a.stride_h + d, a.type);
        s.clear();
        where.clear();
        float top = -kInf;
        for (int64_t at = 0; at < keys; ++at) {
          const int64_t id = page_of(c, b, at);
          if (id < 0) continue;
          const int64_t ph = id * c.heads + h / per;
          const uint8_t* k = c.k + (ph * page + at % page) * c.wide;
          float x = 0.0f;
          for (int d = 0; d < c.dim; ++d) x += q[d] * from_fp8(k[d]);
          s.push_back(x * c.k_scale[ph] * a.scale);
          where.push_back(at);
          top = std::fmax(top, s.back());
        }
        double sum = 0.0;
        std::fill(o.begin(), o.end(), 0.0);
        for (size_t j = 0; j < s.size(); ++j) {
          const float p = std::exp(s[j] - (top == -kInf ? 0.0f : top));
          const int64_t ph = page_of(c, b, where[j]) * c.heads + h / per;
          const uint8_t* v = c.v + ph * page * c.wide + where[j] % page;
          sum += p;
          for (int d = 0; d < c.dim; ++d) o[d] += double(p) * c.v_scale[ph] * from_fp8(v[d * page]);
        }
        const int64_t at = (int64_t(b) * a.new_tokens + i) * a.heads + h;
        for (int d = 0; d < c.dim; ++d) store(a.out, at * c.dim + d, a.type, sum == 0.0 ? 0.0f : float(o[d] / sum));
        if (a.lse) a.lse[at] = sum == 0.0 ? -kInf : float(top + std::log(sum));
      }
  }
}

void beam_select_cpu(const BeamArgs& a) {
  const double inf = kInf;
  const int64_t all = int64_t(a.beams) * a.vocab;
  std::vector<double> value(all);
  std::vector<int64_t> order(all);
  for (int64_t b = 0; b < a.batch; ++b) {
    for (int k = 0; k < a.beams; ++k) {
      const int64_t row = b * a.beams + k;
      double* v = value.data() + int64_t(k) * a.vocab;
      const double score = a.scores[row];
      if (!std::isfinite(score) || (a.finished && a.finished[row])) {
        std::fill(v, v + a.vocab, -inf);
        if (std::isfinite(score)) v[a.eos] = score;
        continue;
      }
      double top = -inf, sum = 0.0;
      for (int t = 0; t < a.vocab; ++t) {
        v[t] = load(a.logits, row * a.stride + t, a.type);
        top = std::fmax(top, v[t]);
      }
      for (int t = 0; t < a.vocab; ++t) sum += std::exp(v[t] - top);
      const double lse = top + std::log(sum);
      for (int t = 0; t < a.vocab; ++t) v[t] = std::isfinite(lse) ? score + (v[t] - lse) : -inf;
    }
    for (int64_t i = 0; i < all; ++i) order[i] = i;
    std::partial_sort(order.begin(), order.begin() + a.take, order.end(), [&](int64_t i, int64_t j) {
      return value[i] > value[j] || (value[i] == value[j] && i < j);
    });
    for (int n = 0; n < a.take; ++n) {
      a.out_scores[b * a.take + n] = float(value[order[n]]);
      a.out_parents[b * a.take + n] = order[n] / a.vocab;
      a.out_tokens[b * a.take + n] = order[n] % a.vocab;
    }
  }
}

void reorder_cpu(const ReorderArgs& a) {
  std::vector<uint8_t> before;
  for (int i = 0; i < a.states; ++i) {
    const ReorderState& st = a.state[i];
    before.resize(size_t(a.beams) * st.bytes);
    for (int64_t b = 0; b < a.batch; ++b) {
      uint8_t* base = st.data + b * a.beams * st.stride;
      for (int k = 0; k < a.beams; ++k) std::memcpy(before.data() + k * st.bytes, base + k * st.stride, st.bytes);
      for (int k = 0; k < a.beams; ++k) {
        const int64_t p = a.parents[b * a.beams + k];
        if (p >= 0 && p < a.beams) std::memcpy(base + k * st.stride, before.data() + p * st.bytes, st.bytes);
      }
    }
  }
}

}  // namespace tl_ops
