// Forms of the encrypted transformer layer that have to leave the same words as one
// another, and softmax attention with rotary positions against float64. Parity unpinned
// by the reference, which has no transformer code.
//
//   layer_forms_test <parameter.json> blocks softmax|linear  attention's products in blocks of any size
//   layer_forms_test <parameter.json> ranks softmax|linear   two ranks against one
//   layer_forms_test <parameter.json> again                  linear attention's kept weights, called again
//   layer_forms_test <parameter.json> rotary                 softmax attention with rotary positions
//
// The two ranks are threads of this process, each with contexts of its own, on one GPU.
// What they exchange is copied between two meetings on the host, with each one's stream
// idle, so that no kernel waits for another rank's.
#include <condition_variable>
#include <cstring>
#include <iomanip>
#include <mutex>
#include <thread>

#include "../../oracle/decoder_plain.h"
#include "cheddar/Transformer.h"

using namespace cheddar;
using word = uint32_t;

struct Meeting {
  std::mutex mu;
  std::condition_variable cv;
  int world, arrived = 0;
  long long turn = 0;
  void *from = nullptr;  // the root's buffer
  void Meet() {
    std::unique_lock<std::mutex> lock(mu);
    const long long mine = turn;
    if (++arrived == world) {
      arrived = 0;
      turn++;
      cv.notify_all();
    } else if (!cv.wait_for(lock, std::chrono::seconds(120), [&] { return turn != mine; })) {
      Fail("a rank did not come");
    }
  }
};
class ThreadGroup : public RankGroup {
 public:
  ThreadGroup(int rank, std::shared_ptr<Meeting> m) : m_(std::move(m)) {
    rank_ = rank;
    world_ = m_->world;
  }
  void Broadcast(void *buf, size_t bytes, int root, void *) override {
    cfhe_context *h = detail::CurrentHandle();
    CheckAbi(cfhe_synchronize(h));
    if (root == rank_) m_->from = buf;
    m_->Meet();
    if (root != rank_) {
      CheckAbi(cfhe_copy_d2d(h, buf, m_->from, bytes));
      CheckAbi(cfhe_synchronize(h));
    }
    m_->Meet();
  }

 private:
  std::shared_ptr<Meeting> m_;
};

struct Setup {
  ParameterJson json;
  std::shared_ptr<Parameter<word>> param;
  std::unique_ptr<BootParameter> boot;
  std::shared_ptr<BootContext<word>> ctx;
  std::unique_ptr<UserInterface<word>> ui;
  TransformerConfig cfg = TransformerConfig::Small();
  TransformerWeights w;
  std::vector<double> x;  // [sequence][token][feature]
  std::vector<Ciphertext<word>> in;

  std::shared_ptr<BootContext<word>> NewContext() const {
    auto c = BootContext<word>::Create(*param, *boot);
    c->PrepareEvalMod();
    c->PrepareEvalSpecialFFT(param->degree_ / 2);
    return c;
  }
  Setup(const char *file, bool linear, bool turned) {
    Random::Seed(0xF0E5);
    json = LoadParameterJson(file);
    param = MakeParameter<word>(json);
    boot = std::make_unique<BootParameter>(param->max_level_, json.num_cts_levels, json.num_stc_levels);
    ctx = NewContext();
    ui = std::make_unique<UserInterface<word>>(ctx);
    ui->UseDeviceSampling(true);
    if (linear) cfg.decay = {0.9, 0.75};
    if (turned) {
      cfg.rotary_pairs = {3, 2};  // of a head's eight pairs: three stay
      cfg.rotary_base = 100.0;
      cfg.rotary_positions.assign(2, std::vector<double>(cfg.seq_len));
      for (int t = 0; t < cfg.seq_len; t++) cfg.rotary_positions[0][t] = t / 4, cfg.rotary_positions[1][t] = t % 4;
    }
    w = TransformerWeights::Random(cfg, 11, 0.08);
    EvkRequest req;
    const int slots = param->degree_ / 2, T = cfg.seq_len, H = cfg.hidden, B = slots / T;
    ctx->AddRequiredRotations(req, slots);
    EncryptedTransformerLayer<word>(ctx, cfg, w).AddRequiredRotations(req);
    ui->PrepareRotationKey(req);
    x.resize((size_t)B * T * H);
    std::mt19937_64 gen(3);
    std::normal_distribution<double> nd(0.0, 1.0);
    for (auto &v : x) v = nd(gen);
    const int level = boot->GetEndLevel() - (cfg.pair_boot ? 1 : 0);
    in.resize(H);
    for (int j = 0; j < H; j++) {
      std::vector<Complex> msg(slots);
      for (int t = 0; t < T; t++)
        for (int b = 0; b < B; b++) msg[(size_t)t * B + b] = Complex(x[((size_t)b * T + t) * H + j] / cfg.act_div, 0.0);
      Plaintext<word> pt;
      ctx->encoder().Encode(pt, level, param->GetScale(level), msg, 0);
      ui->Encrypt(in[j], pt);
    }
    ctx->Synchronize();
  }
};

using Words = std::vector<std::vector<word>>;
static Words WordsOf(const std::vector<Ciphertext<word>> &out) {
  Words words;
  for (const auto &c : out)
    for (const auto *poly : {&c.bx_, &c.ax_}) {
      words.emplace_back();
      CopyDeviceToHost(words.back(), *poly);
      CheckAbi(cfhe_synchronize(detail::CurrentHandle()));
    }
  return words;
}
static Words Run(Setup &s, const TransformerConfig &cfg) {
  EncryptedTransformerLayer<word> layer(s.ctx, cfg, s.w);
  std::vector<Ciphertext<word>> out;
  layer.Forward(out, s.in, s.ui->GetEvkMap());
  return WordsOf(out);
}

// A head's 4 x 4 scores and 4 x 16 weighted values at once, then in blocks that divide
// neither: the same words.
static void Blocks(Setup &s) {
  const Words whole = Run(s, s.cfg);
  for (int products : {1, 3, 10}) {
    TransformerConfig cfg = s.cfg;
    cfg.products = products;
    AssertTrue(Run(s, cfg) == whole, "FAIL: other words with " + std::to_string(products) + " products at a time");
  }
}

// One head and 16 residual ciphertexts a rank.
static void Ranks(Setup &s) {
  const Words one = Run(s, s.cfg);
  auto meeting = std::make_shared<Meeting>();
  meeting->world = 2;
  struct Rank {
    std::shared_ptr<BootContext<word>> ctx;
    std::unique_ptr<EncryptedTransformerLayer<word>> layer;
    std::vector<Ciphertext<word>> out;
    Words words;
    std::string error;
  } ranks[2];
  for (int r = 0; r < 2; r++) {
    ranks[r].ctx = s.NewContext();
    ranks[r].layer = std::make_unique<EncryptedTransformerLayer<word>>(ranks[r].ctx, s.cfg, s.w,
                                                                       std::make_shared<ThreadGroup>(r, meeting));
  }
  std::vector<std::thread> threads;
  for (int r = 0; r < 2; r++)
    threads.emplace_back([&, r] {
      ScopedCurrentHandle scope(ranks[r].ctx->h_);
      try {
        ranks[r].layer->Forward(ranks[r].out, s.in, s.ui->GetEvkMap());
        ranks[r].words = WordsOf(ranks[r].out);
      } catch (const std::exception &e) {
        ranks[r].error = e.what();
      }
    });
  for (auto &t : threads) t.join();
  for (const Rank &r : ranks) {
    AssertTrue(r.error.empty(), "FAIL: " + r.error);
    AssertTrue(r.words == one, "FAIL: a rank's words are not those of one GPU");
  }
}

// Inputs whose scale differs in the last place (what a stack of layers hands on) find
// the kept weights, and the same inputs leave the same words.
static void Again(Setup &s) {
  EncryptedTransformerLayer<word> layer(s.ctx, s.cfg, s.w);
  std::vector<Ciphertext<word>> out;
  layer.Forward(out, s.in, s.ui->GetEvkMap());
  const Words first = WordsOf(out);
  const int kept = layer.KeptPlaintexts();
  AssertTrue(kept == 2 * s.cfg.seq_len + s.cfg.head_dim, "FAIL: weights of two decays, and a cosine and sine per pair");
  const double scale = s.in[0].GetScale();
  for (int ulps = -2; ulps <= 2; ulps++) {
    for (auto &c : s.in) c.SetScale(scale * (1.0 + ulps * std::ldexp(1.0, -52)));
    layer.Forward(out, s.in, s.ui->GetEvkMap());
    AssertTrue(layer.KeptPlaintexts() == kept, "FAIL: " + std::to_string(layer.KeptPlaintexts()) + " plaintexts are kept");
    if (ulps == 0) AssertTrue(WordsOf(out) == first, "FAIL: other words from the same inputs");
  }
}

// The textbook layer with rotary positions before softmax; `zero` leaves them out
static std::vector<double> Plain(const std::vector<double> &x, const plain_transformer::Spec &s,
                                 const plain_transformer::Weights &w, const plain_decoder::Positions &p, bool zero,
                                 plain_transformer::Ranges &rg) {
  using namespace plain_transformer;
  const int T = s.seq_len, H = s.hidden, D = s.head_dim;
  std::vector<double> q, k, v, o((size_t)T * H, 0.0), h1, a, h2;
  Linear(q, x, w.wq, w.bq, T, H, H);
  Linear(k, x, w.wk, w.bk, T, H, H);
  Linear(v, x, w.wv, w.bv, T, H, H);
  if (!zero) {
    plain_decoder::Turn(q, p, T, s.heads, D);
    plain_decoder::Turn(k, p, T, s.heads, D);
  }
  for (int h = 0; h < s.heads; h++)
    for (int t = 0; t < T; t++) {
      std::vector<double> e(T);
      double sum = 0;
      for (int u = 0; u < T; u++) {
        double score = 0;
        for (int d = 0; d < D; d++) score += q[(size_t)t * H + h * D + d] * k[(size_t)u * H + h * D + d];
        score /= std::sqrt((double)D);
        rg.score_abs = std::fmax(rg.score_abs, std::fabs(score));
        sum += e[u] = Clenshaw(s.exp_c, score / s.score_range);
      }
      rg.sum_min = std::fmin(rg.sum_min, sum / T);
      rg.sum_max = std::fmax(rg.sum_max, sum / T);
      const double inv = Clenshaw(s.inv_c, (2.0 * sum / T - (s.sum_hi + s.sum_lo)) / (s.sum_hi - s.sum_lo));
      for (int u = 0; u < T; u++)
        for (int d = 0; d < D; d++) o[(size_t)t * H + h * D + d] += e[u] * inv * v[(size_t)u * H + h * D + d];
    }
  Linear(h1, o, w.wo, w.bo, T, H, H);
  for (size_t i = 0; i < h1.size(); i++) h1[i] += x[i];
  LayerNorm(h1, s, w.gamma1, w.beta1, &rg.var_min, &rg.var_max);
  Linear(a, h1, w.w1, w.b1, T, H, s.ffn);
  for (auto &z : a) {
    rg.pre_abs = std::fmax(rg.pre_abs, std::fabs(z));
    z = s.gelu_range * Clenshaw(s.gelu_c, z / s.gelu_range);
  }
  Linear(h2, a, w.w2, w.b2, T, s.ffn, H);
  for (size_t i = 0; i < h2.size(); i++) h2[i] += h1[i];
  LayerNorm(h2, s, w.gamma2, w.beta2, &rg.var_min, &rg.var_max);
  return h2;
}

static void Rotary(Setup &s) {
  const TransformerConfig &cfg = s.cfg;
  EncryptedTransformerLayer<word> layer(s.ctx, cfg, s.w);
  const auto &w = s.w;
  const int T = cfg.seq_len, H = cfg.hidden, B = layer.BatchSize();
  const plain_transformer::Spec spec{T, H, cfg.heads, cfg.head_dim, cfg.ffn, cfg.score_range, cfg.sum_lo, cfg.sum_hi,
                                     cfg.var_lo, cfg.var_hi, cfg.gelu_range, cfg.ln_eps, layer.polys().exp_c,
                                     layer.polys().inv_c, layer.polys().rsqrt_c, layer.polys().gelu_c, false};
  const plain_transformer::Weights pw{w.wq.data(), w.wk.data(), w.wv.data(), w.wo.data(), w.w1.data(), w.w2.data(),
                                      w.bq.data(), w.bk.data(), w.bv.data(), w.bo.data(), w.b1.data(), w.b2.data(),
                                      w.gamma1.data(), w.beta1.data(), w.gamma2.data(), w.beta2.data()};
  const plain_decoder::Positions pos{cfg.rotary_pairs, cfg.rotary_positions, cfg.rotary_base, cfg.rotary_halves};
  plain_transformer::Ranges rg, unused;
  {
    // the statement above against the oracle's, without positions: sums of at most 64
    // terms of about one in another order
    const std::vector<double> x0(s.x.begin(), s.x.begin() + (size_t)T * H);
    std::vector<double> same;
    plain_transformer::Layer(same, x0, spec, pw);
    const auto mine = Plain(x0, spec, pw, pos, true, unused);
    for (size_t i = 0; i < same.size(); i++)
      AssertTrue(std::abs(same[i] - mine[i]) < 1e-9, "FAIL: the float64 layers differ");
  }
  std::vector<Ciphertext<word>> out;
  layer.Forward(out, s.in, s.ui->GetEvkMap());
  std::vector<double> got((size_t)B * T * H);
  for (int j = 0; j < H; j++) {
    Plaintext<word> dec;
    std::vector<Complex> msg;
    s.ui->Decrypt(dec, out[j]);
    s.ctx->encoder().Decode(msg, dec);
    for (int t = 0; t < T; t++)
      for (int b = 0; b < B; b++) got[((size_t)b * T + t) * H + j] = msg[(size_t)t * B + b].real() * cfg.act_div;
  }
  double worst = 0;
  for (int b = 0; b < B; b++) {
    const std::vector<double> xb(s.x.begin() + (size_t)b * T * H, s.x.begin() + (size_t)(b + 1) * T * H);
    const auto want = Plain(xb, spec, pw, pos, false, rg);
    for (size_t i = 0; i < want.size(); i++) worst = std::max(worst, std::abs(got[(size_t)b * T * H + i] - want[i]));
  }
  std::cout << "ranges: score " << rg.score_abs << ", sum [" << rg.sum_min << ", " << rg.sum_max << "], variance ["
            << rg.var_min << ", " << rg.var_max << "], |pre-activation| " << rg.pre_abs << "\n";
  AssertTrue(rg.score_abs < cfg.score_range && rg.sum_min > cfg.sum_lo && rg.sum_max < cfg.sum_hi &&
                 rg.var_min > cfg.var_lo && rg.var_max < cfg.var_hi && rg.pre_abs < cfg.gelu_range,
             "FAIL: an input left the interval its series was fitted on");
  // the bar of the softmax layer's test; a turn of unit length adds one rescale's error
  std::cout << "max error " << std::scientific << worst << ", precision_bits " << std::fixed << -std::log2(worst) << "\n";
  AssertTrue(worst < std::ldexp(1.0, -12), "FAIL: softmax attention with rotary positions");
}

int main(int argc, char **argv) {
  if (argc < 3) {
    std::cerr << "usage: layer_forms_test <parameter.json> blocks|ranks softmax|linear | again | rotary\n";
    return 2;
  }
  const std::string mode = argv[2];
  const bool linear = mode == "again" || (argc > 3 && !strcmp(argv[3], "linear"));
  Setup s(argv[1], linear, linear || mode == "rotary");
  if (mode == "blocks")
    Blocks(s);
  else if (mode == "ranks")
    Ranks(s);
  else if (mode == "again")
    Again(s);
  else
    Rotary(s);
  std::cout << "PASS\n";
  return 0;
}
