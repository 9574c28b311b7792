// Runs the float64 layer of oracle/decoder_plain.h (exact functions) on data from a
// file, so that a Python test can compare it with an independent implementation
// (host only, no GPU).
//
//   plain_decoder <in.bin> <out.bin>
// in.bin: int32 seq_len, hidden, heads, ffn, axes, halves; int32 pairs[axes];
//         float64 ln_eps, base, decay[heads], positions[axes][seq_len], wq wk wv wo w1 w2
//         bq bk bv bo b1 b2 gamma1 beta1 gamma2 beta2, x[seq_len][hidden].
// out.bin: float64 out[seq_len][hidden].
#include <cstdint>
#include <fstream>

#include "../../oracle/decoder_plain.h"

int main(int argc, char **argv) {
  if (argc < 3) return 2;
  std::ifstream in(argv[1], std::ios::binary);
  int32_t head[6];
  in.read(reinterpret_cast<char *>(head), sizeof(head));
  const int T = head[0], H = head[1], heads = head[2], F = head[3];
  plain_decoder::Positions p;
  std::vector<int32_t> pairs(head[4]);
  in.read(reinterpret_cast<char *>(pairs.data()), (std::streamsize)(pairs.size() * sizeof(int32_t)));
  p.pairs_of_axis.assign(pairs.begin(), pairs.end());
  p.halves = head[5] != 0;
  auto vec = [&](size_t n) {
    std::vector<double> v(n);
    in.read(reinterpret_cast<char *>(v.data()), (std::streamsize)(n * sizeof(double)));
    return v;
  };
  plain_transformer::Spec s{};
  s.seq_len = T, s.hidden = H, s.heads = heads, s.head_dim = H / heads, s.ffn = F, s.exact = true;
  const auto par = vec(2), decay = vec(heads);
  s.ln_eps = par[0];
  p.base = par[1];
  for (int a = 0; a < head[4]; a++) p.positions.push_back(vec(T));
  const auto wq = vec((size_t)H * H), wk = vec((size_t)H * H), wv = vec((size_t)H * H), wo = vec((size_t)H * H);
  const auto w1 = vec((size_t)H * F), w2 = vec((size_t)F * H);
  const auto bq = vec(H), bk = vec(H), bv = vec(H), bo = vec(H), b1 = vec(F), b2 = vec(H);
  const auto g1 = vec(H), e1 = vec(H), g2 = vec(H), e2 = vec(H), x = vec((size_t)T * H);
  if (!in) return 1;
  const plain_transformer::Weights w{wq.data(), wk.data(), wv.data(), wo.data(), w1.data(), w2.data(),
                                     bq.data(), bk.data(), bv.data(), bo.data(), b1.data(), b2.data(),
                                     g1.data(), e1.data(), g2.data(), e2.data()};
  std::vector<double> out;
  plain_decoder::Layer(out, x, s, w, decay, p);
  std::ofstream(argv[2], std::ios::binary)
      .write(reinterpret_cast<const char *>(out.data()), (std::streamsize)(out.size() * sizeof(double)));
  return 0;
}
