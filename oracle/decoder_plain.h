// TEST INFRASTRUCTURE: float64 restatement of a transformer layer with decayed
// linear attention and rotary positions on several axes, used only as the oracle of
// the encrypted layer in tests. Parity unpinned by the reference, which has no
// transformer code; stated in natural units from the definitions, with the exact or
// the Chebyshev form of the remaining non-linear functions (transformer_plain.h).
// Pinned on the CPU against NumPy (tests/test_plain_decoder_cpu.py).
#pragma once
#include "transformer_plain.h"

namespace plain_decoder {

using plain_transformer::Ranges;
using plain_transformer::Spec;
using plain_transformer::Weights;

// pairs_of_axis[a] pairs of features of a head follow axis a, one axis after the
// other; positions[a][t]: token t on axis a
struct Positions {
  std::vector<int> pairs_of_axis;
  std::vector<std::vector<double>> positions;
  double base = 10000.0;
  bool halves = false;
};

// x: [tokens][heads * dim], turned in place
inline void Turn(std::vector<double> &x, const Positions &p, int tokens, int heads, int dim) {
  const int pairs = dim / 2;
  for (int t = 0; t < tokens; t++)
    for (int h = 0; h < heads; h++) {
      double *f = &x[((size_t)t * heads + h) * dim];
      int pair = 0;
      for (size_t axis = 0; axis < p.pairs_of_axis.size(); axis++)
        for (int i = 0; i < p.pairs_of_axis[axis]; i++, pair++) {
          const double angle = p.positions[axis][t] * std::pow(p.base, -(double)i / p.pairs_of_axis[axis]);
          double &u = f[p.halves ? pair : 2 * pair], &v = f[p.halves ? pair + pairs : 2 * pair + 1];
          const double a = u * std::cos(angle) - v * std::sin(angle), b = u * std::sin(angle) + v * std::cos(angle);
          u = a;
          v = b;
        }
    }
}

// o[t] = sum_{u <= t} decay^(t - u) (q_t . k_u) / sqrt(dim) v_u for every head
inline std::vector<double> Attention(const std::vector<double> &q, const std::vector<double> &k,
                                     const std::vector<double> &v, const std::vector<double> &decay, int tokens,
                                     int dim) {
  const int heads = decay.size();
  std::vector<double> o((size_t)tokens * heads * dim, 0.0);
  for (int t = 0; t < tokens; t++)
    for (int h = 0; h < heads; h++)
      for (int u = 0; u <= t; u++) {
        const size_t a = ((size_t)t * heads + h) * dim, b = ((size_t)u * heads + h) * dim;
        double s = 0;
        for (int d = 0; d < dim; d++) s += q[a + d] * k[b + d];
        s *= std::pow(decay[h], t - u) / std::sqrt((double)dim);
        for (int d = 0; d < dim; d++) o[a + d] += s * v[b + d];
      }
  return o;
}

inline void Layer(std::vector<double> &out, const std::vector<double> &x, const Spec &s, const Weights &w,
                  const std::vector<double> &decay, const Positions &p, Ranges *ranges = nullptr) {
  using plain_transformer::Linear;
  const int T = s.seq_len, H = s.hidden;
  Ranges local;
  Ranges &rg = ranges ? *ranges : local;
  std::vector<double> q, k, v, h1, a, h2;
  Linear(q, x, w.wq, w.bq, T, H, H);
  Linear(k, x, w.wk, w.bk, T, H, H);
  Linear(v, x, w.wv, w.bv, T, H, H);
  Turn(q, p, T, s.heads, s.head_dim);
  Turn(k, p, T, s.heads, s.head_dim);
  Linear(h1, Attention(q, k, v, decay, T, s.head_dim), w.wo, w.bo, T, H, H);
  for (size_t i = 0; i < h1.size(); i++) h1[i] += x[i];
  plain_transformer::LayerNorm(h1, s, w.gamma1, w.beta1, &rg.var_min, &rg.var_max);
  Linear(a, h1, w.w1, w.b1, T, H, s.ffn);
  for (auto &v1 : a) {
    rg.pre_abs = std::fmax(rg.pre_abs, std::fabs(v1));
    v1 = s.exact ? 0.5 * v1 * (1.0 + std::erf(v1 / std::sqrt(2.0)))
                 : s.gelu_range * plain_transformer::Clenshaw(s.gelu_c, v1 / s.gelu_range);
  }
  Linear(h2, a, w.w2, w.b2, T, s.ffn, H);
  for (size_t i = 0; i < h2.size(); i++) h2[i] += h1[i];
  plain_transformer::LayerNorm(h2, s, w.gamma2, w.beta2, &rg.var_min, &rg.var_max);
  for (double v2 : h2) rg.out_abs = std::fmax(rg.out_abs, std::fabs(v2));
  out = std::move(h2);
}

}  // namespace plain_decoder
