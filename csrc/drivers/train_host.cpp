#include "drivers/train_host.h"

#include <unistd.h>

#include <algorithm>
#include <cmath>
#include <functional>
#include <limits>
#include <mutex>
#include <numeric>
#include <thread>
#include <vector>

#include "kernels/philox.h"
#include "runtime/common.h"
#include "runtime/thread_pool.h"

namespace oap {

namespace {

constexpr double kInf = std::numeric_limits<double>::infinity();

// One pool for the process; a pool runs one loop at a time.  The child of a fork has none of the
// pool's threads and runs alone.  The pool is never taken down: a child that ends normally would
// join threads that it does not have.
void parallel(int64_t n, const std::function<void(int64_t, int64_t)>& f) {
  static const pid_t owner = getpid();
  if (getpid() != owner) {
    if (n > 0) f(0, n);
    return;
  }
  static std::mutex mu;
  static ThreadPool& pool = *new ThreadPool(
      int(std::min<unsigned>(std::max(1u, std::thread::hardware_concurrency()), 16)));
  std::lock_guard<std::mutex> lock(mu);
  pool.parallel_for(n, [&](int, int64_t b, int64_t e) { f(b, e); });
}

// A logit of the gate as it counts: NaN is an expert that is left out, +inf the largest finite
// number (its score is the limit's, not inf / inf).
double gate_logit(float v) {
  return v == v ? double(std::min(v, std::numeric_limits<float>::max())) : -kInf;
}

double sigmoid(double z) { return 1.0 / (1.0 + std::exp(-z)); }

}  // namespace

void dropout_host(const kern::DropoutArgs& a) {
  const uint64_t key = a.seed_ptr ? uint64_t(*a.seed_ptr) : a.seed;
  const float* x = static_cast<const float*>(a.x);
  const float* res = static_cast<const float*>(a.residual);
  float* y = static_cast<float*>(a.y);
  parallel(a.n, [&](int64_t b, int64_t e) {
    uint64_t block = ~uint64_t(0);
    kern::Philox4 r = {};
    for (int64_t i = b; i < e; ++i) {
      const uint64_t g = a.offset + uint64_t(i);
      if (g >> 2 != block) {
        block = g >> 2;
        r = kern::philox4x32_10(block, key);
      }
      const float v = kern::dropout_keeps(r.w[g & 3], a.threshold) ? x[i] * a.scale : 0.f;
      y[i] = res ? v + res[i] : v;
    }
  });
}

void route_host(const kern::RouteArgs& a) {
  const float* logits = static_cast<const float*>(a.logits);
  const int E = a.experts, per = E / a.groups;
  const bool grouped = a.top_groups < a.groups;
  parallel(a.tokens, [&](int64_t b, int64_t end) {
    std::vector<double> z(E), s(E), c(E), gv(a.groups), w(a.k);
    std::vector<int> order(E), gorder(a.groups);
    for (int64_t t = b; t < end; ++t) {
      double zmax = -kInf, sum = 0.0;
      for (int e = 0; e < E; ++e) {
        z[e] = gate_logit(logits[t * a.ld + e]);
        zmax = std::max(zmax, z[e]);
      }
      for (int e = 0; e < E; ++e) {
        s[e] = a.sigmoid ? sigmoid(z[e]) : z[e] > -kInf ? std::exp(z[e] - zmax) : 0.0;
        sum += s[e];
      }
      for (int e = 0; e < E; ++e) {
        if (!a.sigmoid) s[e] /= sum;
        c[e] = s[e] + (a.bias ? double(a.bias[e]) : 0.0);
        if (!(z[e] > -kInf) || c[e] != c[e]) c[e] = -kInf;
      }
      if (grouped) {
        for (int g = 0; g < a.groups; ++g) {
          double b0 = -kInf, b1 = -kInf;
          for (int e = g * per; e < (g + 1) * per; ++e) {
            b1 = std::max(b1, std::min(b0, c[e]));
            b0 = std::max(b0, c[e]);
          }
          gv[g] = b1 > -kInf ? b0 + b1 : b0;
        }
        std::iota(gorder.begin(), gorder.end(), 0);
        std::stable_sort(gorder.begin(), gorder.end(), [&](int p, int q) { return gv[p] > gv[q]; });
        for (int r = a.top_groups; r < a.groups; ++r)
          std::fill_n(c.begin() + gorder[r] * per, per, -kInf);
      }
      const std::vector<double>& by = a.bias ? c : z;
      std::iota(order.begin(), order.end(), 0);
      std::stable_sort(order.begin(), order.end(), [&](int p, int q) {
        const double vp = c[p] > -kInf ? by[p] : -kInf, vq = c[q] > -kInf ? by[q] : -kInf;
        return vp > vq;
      });
      double zref = -kInf, norm = 0.0;
      for (int r = 0; r < a.k; ++r)
        if (c[order[r]] > -kInf) zref = std::max(zref, z[order[r]]);
      if (a.sigmoid) zref = std::min(zref, 0.0);
      for (int r = 0; r < a.k; ++r) {
        const int e = order[r];
        const bool some = c[e] > -kInf;
        a.indices[t * a.k + r] = some ? e : -1;
        if (!a.renormalize)
          w[r] = s[e];
        else if (a.sigmoid)
          w[r] = z[e] > 0 ? sigmoid(z[e]) : std::exp(z[e] - zref) / (1.0 + std::exp(z[e]));
        else
          w[r] = std::exp(z[e] - zref);
        if (!some) w[r] = 0.0;
        norm += w[r];
      }
      for (int r = 0; r < a.k; ++r) {
        const double v = a.renormalize ? w[r] / norm : w[r];
        a.weights[t * a.k + r] = a.indices[t * a.k + r] >= 0 ? float(v * a.scale) : 0.f;
      }
    }
  });
  std::fill_n(a.counts, E, 0);
  for (int64_t i = 0; i < a.tokens * a.k; ++i)
    if (a.indices[i] >= 0) ++a.counts[a.indices[i]];
}

void route_grad_host(const kern::RouteGradArgs& a) {
  const float* logits = static_cast<const float*>(a.logits);
  float* out = static_cast<float*>(a.grad_logits);
  const int E = a.experts;
  const bool all = !a.sigmoid && !a.renormalize;
  parallel(a.tokens, [&](int64_t b, int64_t end) {
    std::vector<double> d(E);
    for (int64_t t = b; t < end; ++t) {
      std::fill(d.begin(), d.end(), 0.0);
      double dot = 0.0;
      for (int r = 0; r < a.k; ++r)
        if (a.indices[t * a.k + r] >= 0)
          dot += double(a.grad[t * a.k + r]) * a.weights[t * a.k + r];
      const double mean = a.renormalize ? dot / a.scale : 0.0;
      for (int r = 0; r < a.k; ++r) {
        const int e = a.indices[t * a.k + r];
        if (e < 0) continue;
        double v = double(a.weights[t * a.k + r]) * (a.grad[t * a.k + r] - mean);
        if (a.sigmoid) v *= 1.0 / (1.0 + std::exp(double(logits[t * a.ld + e])));
        d[e] = v;
      }
      if (all) {
        double zmax = -kInf, sum = 0.0;
        for (int e = 0; e < E; ++e) {
          zmax = std::max(zmax, gate_logit(logits[t * a.ld + e]));
        }
        for (int e = 0; e < E; ++e) {
          const double v = gate_logit(logits[t * a.ld + e]);
          if (v > -kInf) sum += std::exp(v - zmax);
        }
        for (int e = 0; e < E; ++e) {
          const double v = gate_logit(logits[t * a.ld + e]);
          if (v > -kInf) d[e] -= std::exp(v - zmax) / sum * dot;
        }
      }
      for (int e = 0; e < E; ++e) out[t * E + e] = float(d[e]);
    }
  });
}

namespace {

double ce_logit(const kern::CeArgs& a, int64_t i, int64_t j) {
  if (a.bias && a.bias[j] == -std::numeric_limits<float>::infinity()) return -kInf;
  const float* x = static_cast<const float*>(a.x) + i * a.ldx;
  const float* w = static_cast<const float*>(a.w) + j * a.ldw;
  double z = a.bias ? double(a.bias[j]) : 0.0;
  for (int k = 0; k < a.dim; ++k) z += double(x[k]) * w[k];
  // (a sum refers to the maximum as it is kept, in fp32: their difference stays in range)
  return std::fabs(z) > 0x1p28 ? double(float(z)) : z;
}

bool has_loss(const kern::CeArgs& a, int64_t i) {
  return a.target[i] != a.ignore && a.target[i] >= 0 && a.target[i] < a.classes;
}

// (rows without a loss, or whose loss nobody asks the gradient of, take no part)
bool has_gradient(const kern::CeArgs& a, const float* grad, bool per_row, int64_t i) {
  return has_loss(a, i) && !(per_row && grad[i] == 0.f);
}

}  // namespace

void ce_forward_host(const kern::CeArgs& a, float* loss, float2* stat, float* total, bool mean) {
  parallel(a.n, [&](int64_t b, int64_t end) {
    std::vector<double> z(a.classes);
    for (int64_t i = b; i < end; ++i) {
      double m = -kInf, s = 0.0;
      for (int64_t j = 0; j < a.classes; ++j) {
        z[j] = ce_logit(a, i, j);
        m = std::max(m, z[j]);
      }
      // (the sum refers to the maximum as it is kept)
      const double ref = m > -kInf ? double(float(m)) : 0.0;
      for (int64_t j = 0; j < a.classes; ++j) s += std::exp(z[j] - ref);
      stat[i] = make_float2(float(m), float(s));
      if (a.target[i] == a.ignore)
        loss[i] = 0.f;
      else if (!has_loss(a, i))
        loss[i] = std::numeric_limits<float>::quiet_NaN();
      else
        loss[i] = float(z[a.target[i]] == -kInf ? kInf : std::log(s) + (ref - z[a.target[i]]));
    }
  });
  if (!total) return;
  double s = 0.0;
  int64_t k = 0;
  for (int64_t i = 0; i < a.n; ++i)
    if (a.target[i] != a.ignore) {
      s += loss[i];
      ++k;
    }
  *total = float(mean ? s / double(std::max<int64_t>(k, 1)) : s);
}

void ce_backward_host(const kern::CeArgs& a, const float2* stat, const float* grad, bool per_row,
                      bool mean, float* dx, float* dw, float* db) {
  int64_t k = 0;
  for (int64_t i = 0; i < a.n; ++i) k += a.target[i] != a.ignore;
  const double share = mean ? 1.0 / double(std::max<int64_t>(k, 1)) : 1.0;
  const float* x = static_cast<const float*>(a.x);
  const float* w = static_cast<const float*>(a.w);
  auto dz = [&](int64_t i, int64_t j) {
    const double z = ce_logit(a, i, j);
    if (z == -kInf) return 0.0;
    const double p = std::exp(z - double(stat[i].x)) / double(stat[i].y) -
                     (a.target[i] == j ? 1.0 : 0.0);
    return p * (per_row ? double(grad[i]) : double(grad[0]) * share);
  };
  if (dx)
    parallel(a.n, [&](int64_t b, int64_t end) {
      std::vector<double> acc(a.dim);
      for (int64_t i = b; i < end; ++i) {
        std::fill(acc.begin(), acc.end(), 0.0);
        for (int64_t j = 0; has_gradient(a, grad, per_row, i) && j < a.classes; ++j) {
          const double d = dz(i, j);
          if (d != 0.0)
            for (int c = 0; c < a.dim; ++c) acc[c] += d * w[j * a.ldw + c];
        }
        for (int c = 0; c < a.dim; ++c) dx[i * a.dim + c] = float(acc[c]);
      }
    });
  if (dw || db)
    parallel(a.classes, [&](int64_t b, int64_t end) {
      std::vector<double> acc(a.dim);
      for (int64_t j = b; j < end; ++j) {
        std::fill(acc.begin(), acc.end(), 0.0);
        double bias = 0.0;
        for (int64_t i = 0; i < a.n; ++i) {
          if (!has_gradient(a, grad, per_row, i)) continue;
          const double d = dz(i, j);
          bias += d;
          if (d != 0.0)
            for (int c = 0; c < a.dim; ++c) acc[c] += d * x[i * a.ldx + c];
        }
        if (db) db[j] = float(bias);
        if (dw)
          for (int c = 0; c < a.dim; ++c) dw[j * a.dim + c] = float(acc[c]);
      }
    });
}

}  // namespace oap
