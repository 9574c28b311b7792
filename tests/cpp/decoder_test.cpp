// Encrypted linear attention with a decay for each head and rotary positions on two
// axes, against float64 (oracle/decoder_plain.h). Parity unpinned by the reference,
// which has no transformer code.
//
//   decoder_test <parameter.json> tokens          token by token over kept keys and values
//   decoder_test <parameter.json> layer [halves]  one layer over a prompt of 16 tokens
#include <cstring>
#include <iomanip>

#include "../../oracle/decoder_plain.h"
#include "cheddar/Transformer.h"

using namespace cheddar;
using word = uint32_t;

static double Verdict(double err, double bar, const char *what) {
  std::cout << what << ": max error " << std::scientific << err << ", allowed " << bar << std::fixed << "\n";
  std::cout << "precision_bits " << -std::log2(err) << "\n";
  if (!(err < bar)) Fail(std::string("FAIL: ") + what);
  return err;
}

// Five tokens of four features, every slot another sequence, uniform in [-1, 1].
// A fresh ciphertext's slots are off by at most e = 2^-20 (error polynomials of
// deviation 3.2 times a ternary secret: 820 on a coefficient, 2^17.7 on a slot, 4.5
// deviations over all slots, on a scale of 2^40), and as much again comes with a
// rescale or a key switch. Turned by a position: 3 e. A score of four products:
// 4 * 2 * 3 e and two rescales, 26 e, below 4 in magnitude. The sum over five
// tokens: 5 (26 e + 4 * 2 e) = 170 e, below 2^-12.
static void Tokens(std::shared_ptr<BootContext<word>> ctx, UserInterface<word> &ui, const Parameter<word> &param) {
  const int T = 5, D = 4, slots = param.degree_ / 2, level = 8;
  const double decay = 0.8, base = 100.0;
  const std::vector<int> axes = {1, 1};
  std::vector<std::vector<double>> positions(2, std::vector<double>(T));
  for (int t = 0; t < T; t++) positions[0][t] = t / 2, positions[1][t] = t % 2 + 3;
  const auto angles = RotaryAngles(axes, positions, base, D / 2, T);
  std::mt19937_64 gen(5);
  std::uniform_real_distribution<double> uni(-1.0, 1.0);
  std::vector<std::vector<double>> val[3];  // q, k, v: [token * D + feature][slot]
  for (auto &x : val) x.assign(T * D, std::vector<double>(slots));
  for (auto &x : val)
    for (auto &row : x)
      for (auto &v : row) v = uni(gen);
  ConstContextPtr<word> base_ctx = ctx;
  DecayedTokens<word> kept(base_ctx, D, decay);
  double worst = 0;
  for (int t = 0; t < T; t++) {
    std::vector<Ciphertext<word>> in[3];
    for (int part = 0; part < 3; part++)
      for (int d = 0; d < D; d++) {
        std::vector<Complex> msg(slots);
        for (int i = 0; i < slots; i++) msg[i] = Complex(val[part][t * D + d][i], 0.0);
        Plaintext<word> pt;
        ctx->encoder().Encode(pt, level, param.GetScale(level), msg, 0);
        in[part].emplace_back();
        ui.Encrypt(in[part].back(), pt);
      }
    // queries and keys turned together: two rows of D features
    std::vector<Constant<word>> c(D / 2), s(D / 2);
    const double scale = param.GetScale(level - 1) * param.GetRescalePrimeProd(level) / in[0][0].GetScale();
    for (int i = 0; i < D / 2; i++) {
      ctx->encoder().EncodeConstant(c[i], level, scale, std::cos(angles[i][t]));
      ctx->encoder().EncodeConstant(s[i], level, scale, std::sin(angles[i][t]));
    }
    std::vector<const Ciphertext<word> *> rows, v;
    for (int part = 0; part < 2; part++)
      for (int d = 0; d < D; d++) rows.push_back(&in[part][d]);
    std::vector<Ciphertext<word>> turned, q(D), k(D), low(D), o;
    ctx->Rotary(turned, rows, D / 2, false, c, s);
    std::vector<const Ciphertext<word> *> qp;
    for (int d = 0; d < D; d++) {
      ctx->Rescale(q[d], turned[d]);
      ctx->Rescale(k[d], turned[D + d]);
      ctx->LevelDown(low[d], in[2][d], level - 1);
      qp.push_back(&q[d]);
      v.push_back(&low[d]);
    }
    kept.Append(std::move(k), v);
    kept.Attend(o, qp, ui.GetMultiplicationKey(), 1.0);
    AssertTrue(param.NPToLevel(o[0].GetNP()) == level - 4, "decoder_test: wrong level");
    std::vector<std::vector<Complex>> got(D);
    for (int d = 0; d < D; d++) {
      Plaintext<word> pt;
      ui.Decrypt(pt, o[d]);
      ctx->encoder().Decode(got[d], pt);
    }
    for (int i = 0; i < slots; i++) {
      std::vector<double> x[3];
      for (int part = 0; part < 3; part++)
        for (int u = 0; u <= t; u++)
          for (int d = 0; d < D; d++) x[part].push_back(val[part][u * D + d][i]);
      plain_decoder::Positions p{axes, positions, base, false};
      plain_decoder::Turn(x[0], p, t + 1, 1, D);
      plain_decoder::Turn(x[1], p, t + 1, 1, D);
      const auto want = plain_decoder::Attention(x[0], x[1], x[2], {decay}, t + 1, D);
      for (int d = 0; d < D; d++)  // without the oracle's 1 / sqrt(D)
        worst = std::max(worst, std::abs(got[d][i].real() - 2.0 * want[(size_t)t * D + d]));
    }
  }
  Verdict(worst, std::ldexp(1.0, -12), "token by token");
}

int main(int argc, char **argv) {
  if (argc < 3) {
    std::cerr << "usage: decoder_test <parameter.json> tokens | layer [halves]\n";
    return 2;
  }
  const bool layer_mode = !strcmp(argv[2], "layer"), halves = argc > 3 && !strcmp(argv[3], "halves");
  Random::Seed(0xDEC0);
  ParameterJson json = LoadParameterJson(argv[1]);
  auto param = MakeParameter<word>(json);
  BootParameter boot_param(param->max_level_, json.num_cts_levels, json.num_stc_levels);
  auto ctx = BootContext<word>::Create(*param, boot_param);
  UserInterface<word> ui(ctx);
  ui.UseDeviceSampling(true);
  if (!layer_mode) {
    Tokens(ctx, ui, *param);
    std::cout << "PASS\n";
    return 0;
  }
  const int slots = param->degree_ / 2;
  ctx->PrepareEvalMod();
  ctx->PrepareEvalSpecialFFT(slots);
  TransformerConfig cfg = TransformerConfig::Small();
  cfg.decay = {0.9, 0.75};
  cfg.rotary_pairs = {3, 2};  // of a head's eight pairs: three stay
  cfg.rotary_halves = halves;
  cfg.rotary_base = 100.0;
  cfg.rotary_positions.assign(2, std::vector<double>(cfg.seq_len));
  for (int t = 0; t < cfg.seq_len; t++) cfg.rotary_positions[0][t] = t / 4, cfg.rotary_positions[1][t] = t % 4;
  TransformerWeights w = TransformerWeights::Random(cfg, 11, 0.08);
  EncryptedTransformerLayer<word> layer(ctx, cfg, w);
  EvkRequest req;
  ctx->AddRequiredRotations(req, slots);
  layer.AddRequiredRotations(req);
  ui.PrepareRotationKey(req);
  const int T = cfg.seq_len, H = cfg.hidden, B = layer.BatchSize();
  std::vector<double> x((size_t)B * T * H);
  std::mt19937_64 gen(3);
  std::normal_distribution<double> nd(0.0, 1.0);
  for (auto &v : x) v = nd(gen);
  const int level = boot_param.GetEndLevel() - (cfg.pair_boot ? 1 : 0);
  std::vector<Ciphertext<word>> in(H), out;
  for (int j = 0; j < H; j++) {
    std::vector<Complex> msg(slots);
    for (int t = 0; t < T; t++)
      for (int b = 0; b < B; b++) msg[(size_t)t * B + b] = Complex(x[((size_t)b * T + t) * H + j] / cfg.act_div, 0.0);
    Plaintext<word> pt;
    ctx->encoder().Encode(pt, level, param->GetScale(level), msg, 0);
    ui.Encrypt(in[j], pt);
  }
  layer.Forward(out, in, ui.GetEvkMap());
  std::cout << "stages:";
  for (auto &[name, s] : layer.StageSeconds()) std::cout << " [" << name << " " << std::fixed << std::setprecision(3) << s << " s]";
  std::cout << "\n";
  plain_transformer::Spec spec{T, H, cfg.heads, cfg.head_dim, cfg.ffn, cfg.score_range, cfg.sum_lo, cfg.sum_hi,
                               cfg.var_lo, cfg.var_hi, cfg.gelu_range, cfg.ln_eps, layer.polys().exp_c,
                               layer.polys().inv_c, layer.polys().rsqrt_c, layer.polys().gelu_c, false};
  plain_transformer::Weights pw{w.wq.data(), w.wk.data(), w.wv.data(), w.wo.data(), w.w1.data(), w.w2.data(),
                                w.bq.data(), w.bk.data(), w.bv.data(), w.bo.data(), w.b1.data(), w.b2.data(),
                                w.gamma1.data(), w.beta1.data(), w.gamma2.data(), w.beta2.data()};
  const plain_decoder::Positions pos{cfg.rotary_pairs, cfg.rotary_positions, cfg.rotary_base, halves};
  std::vector<double> got((size_t)B * T * H);
  for (int j = 0; j < H; j++) {
    Plaintext<word> dec;
    std::vector<Complex> msg;
    ui.Decrypt(dec, out[j]);
    ctx->encoder().Decode(msg, dec);
    for (int t = 0; t < T; t++)
      for (int b = 0; b < B; b++) got[((size_t)b * T + t) * H + j] = msg[(size_t)t * B + b].real() * cfg.act_div;
  }
  plain_transformer::Ranges rg;
  double worst = 0;
  for (int b = 0; b < B; b++) {
    const std::vector<double> xb(x.begin() + (size_t)b * T * H, x.begin() + (size_t)(b + 1) * T * H);
    std::vector<double> want;
    plain_decoder::Layer(want, xb, spec, pw, cfg.decay, pos, &rg);
    for (size_t i = 0; i < want.size(); i++) worst = std::max(worst, std::abs(got[(size_t)b * T * H + i] - want[i]));
  }
  std::cout << "ranges: variance [" << rg.var_min << ", " << rg.var_max << "], |pre-activation| " << rg.pre_abs
            << ", |output| " << rg.out_abs << "\n";
  AssertTrue(rg.var_min > cfg.var_lo && rg.var_max < cfg.var_hi && rg.pre_abs < cfg.gelu_range && rg.out_abs < cfg.act_div,
             "FAIL: an input left the interval its series was fitted on");
  // the bar of the softmax layer's test: two bootstraps of 2^-19 on values scaled to
  // [-1, 1], multiplied by up to 1 / sqrt(var_lo) and act_div on the way out
  Verdict(worst, std::ldexp(1.0, -12), "layer");
  std::cout << "PASS\n";
  return 0;
}
