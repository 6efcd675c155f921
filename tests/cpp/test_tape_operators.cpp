// test_tape_operators.cpp -- the long-history operators on the device tape (tape.hpp), run together as a policy over
// histories uses them: LayerNorm -> q | k | v -> grouped_attention with a relative position bias and each sample's own
// length -> output projection and residual -> LayerNorm -> logits -> policy_loss. The same graph is written out here in
// f64 on the host, and every gradient of the tape's backward() is compared with central differences of its loss. Exit
// status 0 when every check passes.
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <string>
#include <vector>

#include "../../talos-xii_amd/host/tape.hpp"

using namespace talos::tape;
using Vec = std::vector<double>;

static int g_fail = 0, g_pass = 0;
static void check(bool ok, const std::string& name) {
  if (ok) ++g_pass;
  else { ++g_fail; std::printf("FAIL %s\n", name.c_str()); }
}

static uint64_t g_seed = 17;
static double uniform() {
  g_seed = g_seed * 6364136223846793005ULL + 1442695040888963407ULL;
  return (g_seed >> 11) / 9007199254740992.0;
}
static Vec draws(size_t n, double lo, double hi) {
  Vec v(n);
  for (double& x : v) x = (double)(float)(lo + (hi - lo) * uniform());
  return v;
}

// sizes: samples, tokens, width, heads on key heads, head width, actions, buckets up to a distance
constexpr int B = 2, S = 11, D = 12, H = 4, KV = 2, HD = 6, V = 7, NB = 6, FAR = 5, N = 2 * FAR + 1, ROWS = B * S;
constexpr double EPS = 1e-5, LOW = 0.2, HIGH = 0.3, KL = 0.05;
static const int LENS[B] = {11, 7};

struct Params {
  Vec x, g1, b1, wq, wk, wv, wo, table, g2, b2, wl;
};
static const char* kNames[] = {"x", "g1", "b1", "wq", "wk", "wv", "wo", "table", "g2", "b2", "wl"};
static Vec* field(Params& p, int i) {
  Vec* f[] = {&p.x, &p.g1, &p.b1, &p.wq, &p.wk, &p.wv, &p.wo, &p.table, &p.g2, &p.b2, &p.wl};
  return f[i];
}
static PolicyBatch g_batch;

static Vec norm(const Vec& x, const Vec& g, const Vec& b) {
  Vec y(x.size());
  for (int r = 0; r < ROWS; ++r) {
    double m = 0, v = 0;
    for (int c = 0; c < D; ++c) m += x[r * D + c] / D;
    for (int c = 0; c < D; ++c) v += (x[r * D + c] - m) * (x[r * D + c] - m) / D;
    for (int c = 0; c < D; ++c) y[r * D + c] = (x[r * D + c] - m) / std::sqrt(v + EPS) * g[c] + b[c];
  }
  return y;
}
static Vec mul(const Vec& a, const Vec& w, int in, int out) {
  Vec y((size_t)ROWS * out, 0.0);
  for (int r = 0; r < ROWS; ++r)
    for (int i = 0; i < in; ++i)
      for (int o = 0; o < out; ++o) y[r * out + o] += a[r * in + i] * w[i * out + o];
  return y;
}
static int bucket(int d) {  // one direction
  const int n = d < 0 ? -d : 0, few = NB / 2;
  if (n < few) return n;
  if (n >= FAR) return NB - 1;
  return std::min(NB - 1, few + (int)std::floor(std::log((double)n / few) / std::log((double)FAR / few) * (NB - few) + 1e-9));
}
static double loss_of(const Params& p) {
  const Vec a = norm(p.x, p.g1, p.b1);
  const Vec q = mul(a, p.wq, D, H * HD), k = mul(a, p.wk, D, KV * HD), v = mul(a, p.wv, D, KV * HD);
  Vec o((size_t)ROWS * H * HD, 0.0);
  for (int b = 0; b < B; ++b)
    for (int h = 0; h < H; ++h)
      for (int i = 0; i < LENS[b]; ++i) {
        Vec s(i + 1);
        double top = -1e300, z = 0;
        for (int j = 0; j <= i; ++j) {
          double x = 0;
          for (int d = 0; d < HD; ++d) x += q[((b * S + i) * H + h) * HD + d] * k[((b * S + j) * KV + h / (H / KV)) * HD + d];
          s[j] = x / std::sqrt((double)HD) + p.table[bucket(std::max(j - i, -FAR)) * H + h];
          top = std::max(top, s[j]);
        }
        for (double& x : s) z += x = std::exp(x - top);
        for (int j = 0; j <= i; ++j)
          for (int d = 0; d < HD; ++d)
            o[((b * S + i) * H + h) * HD + d] += s[j] / z * v[((b * S + j) * KV + h / (H / KV)) * HD + d];
      }
  Vec y = mul(o, p.wo, H * HD, D);
  for (size_t i = 0; i < y.size(); ++i) y[i] += p.x[i];
  const Vec logits = mul(norm(y, p.g2, p.b2), p.wl, D, V);
  double loss = 0;
  for (int r = 0; r < ROWS; ++r) {
    const double w = g_batch.weight[r], adv = g_batch.adv[r];
    if (w == 0) continue;
    double z = 0;
    for (int c = 0; c < V; ++c) z += std::exp(logits[r * V + c]);
    const double lp = logits[r * V + g_batch.actions[r]] - std::log(z), ratio = std::exp(lp - g_batch.old_logp[r]);
    const double held = std::min(std::max(ratio, 1 - LOW), 1 + HIGH), gap = g_batch.ref_logp[r] - lp;
    loss += w * (KL * (std::exp(gap) - gap - 1) - std::min(ratio * adv, held * adv));
  }
  return loss;
}

int main() {
  std::setvbuf(stdout, nullptr, _IONBF, 0);
  try {
    Params p{draws(ROWS * D, -1, 1),       draws(D, 0.8, 1.2),           draws(D, -0.2, 0.2),
             draws(D * H * HD, -0.5, 0.5), draws(D * KV * HD, -0.5, 0.5), draws(D * KV * HD, -0.5, 0.5),
             draws(H * HD * D, -0.3, 0.3), draws(NB * H, -0.5, 0.5),     draws(D, 0.8, 1.2),
             draws(D, -0.2, 0.2),          draws(D * V, -0.6, 0.6)};
    for (int r = 0; r < ROWS; ++r) {
      const bool pad = r % S >= LENS[r / S];
      g_batch.actions.push_back((int32_t)(uniform() * V));
      g_batch.adv.push_back((double)(float)(uniform() * 2 - 1));
      // far enough from the clip's borders that a difference of 1e-5 crosses none
      g_batch.old_logp.push_back((double)(float)(-1.9 + 0.3 * (r % 4)));
      g_batch.ref_logp.push_back((double)(float)(-2.2 + 0.2 * (r % 3)));
      g_batch.weight.push_back(pad ? 0.0 : 1.0 / 32);
    }
    const std::vector<int32_t> lens(LENS, LENS + B);
    LayerNorm n1(D, EPS), n2(D, EPS);
    n1.weight.set_data(p.g1);
    n1.bias.set_data(p.b1);
    n2.weight.set_data(p.g2);
    n2.bias.set_data(p.b2);
    Tensor x = Tensor::from_vec(p.x, {(size_t)ROWS, (size_t)D});
    Tensor wq = Tensor::from_vec(p.wq, {D, H * HD}), wk = Tensor::from_vec(p.wk, {D, KV * HD});
    Tensor wv = Tensor::from_vec(p.wv, {D, KV * HD}), wo = Tensor::from_vec(p.wo, {H * HD, D});
    Tensor table = Tensor::from_vec(p.table, {NB, H}), wl = Tensor::from_vec(p.wl, {D, V});
    auto graph = [&] {
      Tensor a = n1.forward(x);
      Tensor bias = relative_position_bias(table, FAR, false);
      Tensor o = grouped_attention(a.matmul(wq).reshape({B, S, H, HD}), a.matmul(wk).reshape({B, S, KV, HD}),
                                   a.matmul(wv).reshape({B, S, KV, HD}), true, &bias, lens, lens);
      Tensor y = x + o.reshape({ROWS, H * HD}).matmul(wo);
      return policy_loss(n2.forward(y).matmul(wl), g_batch, LOW, HIGH, KL);
    };
    Tensor loss = graph();
    const double want = loss_of(p);
    check(std::fabs(loss.item() - want) <= 1e-5 * (1 + std::fabs(want)), "loss");
    loss.backward();
    const Tensor* leaves[] = {&x, &n1.weight, &n1.bias, &wq, &wk, &wv, &wo, &table, &n2.weight, &n2.bias, &wl};
    std::vector<Vec> once;
    for (int f = 0; f < 11; ++f) {
      const Vec got = leaves[f]->grad();
      once.push_back(got);
      Vec* v = field(p, f);
      double worst = 0;
      for (size_t i = 0; i < v->size(); ++i) {
        const double keep = (*v)[i], h = 1e-5;
        (*v)[i] = keep + h;
        const double up = loss_of(p);
        (*v)[i] = keep - h;
        const double down = loss_of(p);
        (*v)[i] = keep;
        worst = std::max(worst, std::fabs((up - down) / (2 * h) - got[i]));
      }
      // fp32 gradients of order 0.1 through some 40 roundings each, and differences good to 1e-9
      if (worst > 2e-6) std::printf("  d %s off by %.3g\n", kNames[f], worst);
      check(worst <= 2e-6, std::string("gradient of ") + kNames[f]);
    }
    // gradients add up, and a scaled loss scales them
    Tensor again = graph().scale(0.5);
    again.backward();
    for (int f = 0; f < 11; ++f) {
      const Vec got = leaves[f]->grad();
      double worst = 0;
      for (size_t i = 0; i < got.size(); ++i) worst = std::max(worst, std::fabs(got[i] - 1.5 * once[f][i]));
      check(worst <= 1e-6, std::string("accumulated gradient of ") + kNames[f]);
    }
    auto panics = [](auto&& fn) {
      try {
        fn();
      } catch (const Panic&) {
        return true;
      }
      return false;
    };
    check(panics([&] { LayerNorm(5).forward(x); }), "LayerNorm panics on another width");
    check(panics([&] { relative_position_bias(table, 2, false); }), "a distance within the exact buckets panics");
    check(panics([&] { grouped_attention(x, x, x, true); }), "attention panics on the rank");
    check(panics([&] { policy_loss(x, PolicyBatch{}, LOW, HIGH, KL); }), "the loss panics without its rows");
  } catch (const std::exception& e) {
    check(false, std::string("exception ") + e.what());
  }
  std::printf("%d passed, %d failed\n", g_pass, g_fail);
  return g_fail ? 1 : 0;
}
