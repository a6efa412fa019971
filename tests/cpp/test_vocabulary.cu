// The C++ entry points of the vocabulary operators on a context: embedding
// lookup, its gradient (written and accumulated), distillation with gradient,
// and sampling, against host loops in double precision.
// Built by __graft_entry__.build(). Prints one line per check and "ALL PASSED"
// / "FAILED <n>".
#include <moderngpu/kernel_embedding.hxx>
#include <moderngpu/kernel_distill.hxx>
#include <moderngpu/kernel_sample.hxx>
#include <cmath>
#include <random>

using namespace mgpu;

static int failures = 0;
static void report(const char* name, bool ok) {
  printf("%-52s %s\n", name, ok ? "ok" : "FAIL");
  if(!ok) ++failures;
}

int main() {
  standard_context_t context(false);
  std::mt19937 rng(5);
  std::normal_distribution<float> normal;
  const int rows = 300, width = 72, count = 2000;
  std::vector<float> table(rows * width), grad(count * width);
  for(float& v : table) v = normal(rng);
  for(float& v : grad) v = normal(rng);
  std::vector<int> tokens(count);
  for(int& t : tokens) t = (int)(rng() % (rows + 3)) - 1;   // some are none
  mem_t<float> table_d = to_mem(table, context);
  mem_t<float> grad_d = to_mem(grad, context);
  mem_t<int> tokens_d = to_mem(tokens, context);

  mem_t<float> out_d(count * width, context);
  embedding_lookup(table_d.data(), rows, width, (int64_t)width, tokens_d.data(),
    count, 0.5f, out_d.data(), context);
  context.synchronize();
  std::vector<float> out = from_mem(out_d);
  bool ok = true;
  for(int i = 0; i < count; ++i)
    for(int c = 0; c < width; ++c) {
      int t = tokens[i];
      float want = t >= 0 && t < rows ? 0.5f * table[t * width + c] : 0.0f;
      ok = ok && out[i * width + c] == want;
    }
  report("embedding_lookup", ok);

  // 2,000 terms at the most: 2,001 roundings of 2^-24 of their sizes.
  std::vector<double> want(rows * width), size(rows * width);
  for(int i = 0; i < count; ++i)
    if(tokens[i] >= 0 && tokens[i] < rows)
      for(int c = 0; c < width; ++c) {
        want[tokens[i] * width + c] += grad[i * width + c];
        size[tokens[i] * width + c] += std::fabs(grad[i * width + c]);
      }
  mem_t<float> sums_d(rows * width, context);
  for(int pass = 1; pass <= 2; ++pass) {
    embedding_gradient(grad_d.data(), (int64_t)width, width, tokens_d.data(),
      count, rows, 1.0f, pass > 1, sums_d.data(), context);
    context.synchronize();
    std::vector<float> sums = from_mem(sums_d);
    ok = true;
    for(size_t i = 0; i < sums.size(); ++i)
      ok = ok && std::fabs(sums[i] - pass * want[i]) <=
        pass * size[i] * 2003 * std::ldexp(1.0, -24);
    report(pass > 1 ? "embedding_gradient, accumulated" :
      "embedding_gradient", ok);
  }

  const int n = 7, vocabulary = 5003, entries = 9;
  std::vector<float> logits(n * vocabulary), teacher(n * entries);
  std::vector<int64_t> at(n * entries);
  for(float& v : logits) v = 3 * normal(rng);
  for(float& v : teacher) v = normal(rng);
  for(int64_t& j : at) j = (int64_t)(rng() % vocabulary);
  at[0] = -1;
  at[2 * entries + 1] = at[2 * entries];
  mem_t<float> logits_d = to_mem(logits, context);
  mem_t<float> teacher_d = to_mem(teacher, context);
  mem_t<int64_t> at_d = to_mem(at, context);
  mem_t<float> losses_d(n, context), slopes_d(n * vocabulary, context);
  mem_t<float> plain_d(n, context);
  distill_loss_gradient(logits_d.data(), (int64_t)vocabulary, n, vocabulary,
    at_d.data(), teacher_d.data(), entries, 2.0f, (const float*)nullptr,
    losses_d.data(), slopes_d.data(), (int64_t)vocabulary, context);
  distill_loss(logits_d.data(), (int64_t)vocabulary, n, vocabulary,
    at_d.data(), teacher_d.data(), entries, 2.0f, plain_d.data(), context);
  context.synchronize();
  std::vector<float> losses = from_mem(losses_d), slopes = from_mem(slopes_d);
  ok = losses == from_mem(plain_d);
  for(int i = 0; i < n; ++i) {
    const float* x = &logits[i * vocabulary];
    double mass = 0, taught = 0, loss = 0;
    for(int v = 0; v < vocabulary; ++v) mass += std::exp(x[v] / 2.0);
    std::vector<double> slope(vocabulary);
    for(int v = 0; v < vocabulary; ++v)
      slope[v] = 2 * std::exp(x[v] / 2.0) / mass;
    for(int k = 0; k < entries; ++k)
      if(at[i * entries + k] >= 0) taught += std::exp(teacher[i * entries + k] /
        2.0);
    for(int k = 0; k < entries; ++k) {
      int64_t j = at[i * entries + k];
      if(j < 0) continue;
      double p = std::exp(teacher[i * entries + k] / 2.0) / taught;
      loss += 4 * p * (std::log(p) - x[j] / 2.0 + std::log(mass));
      slope[j] -= 2 * p;
    }
    // Weights to 2^-18, of sums and of differences of order 10.
    ok = ok && std::fabs(losses[i] - loss) <= 1e-4;
    for(int v = 0; v < vocabulary; ++v)
      ok = ok && std::fabs(slopes[i * vocabulary + v] - slope[v]) <= 1e-5;
  }
  report("distill_loss and distill_loss_gradient", ok);

  std::vector<float> uniforms(n);
  for(float& u : uniforms) u = (rng() >> 8) * std::ldexp(1.0f, -24);
  mem_t<float> uniforms_d = to_mem(uniforms, context);
  mem_t<int> drawn_d(n, context);
  sampling_t settings;
  settings.temperature = 1.5f;
  settings.top_k = 40;
  sample_tokens(logits_d.data(), (int64_t)vocabulary, n, vocabulary,
    uniforms_d.data(), settings, drawn_d.data(), context);
  context.synchronize();
  std::vector<int> drawn = from_mem(drawn_d);
  ok = true;
  for(int i = 0; i < n; ++i) {
    const float* x = &logits[i * vocabulary];
    std::vector<int> order(vocabulary);
    for(int v = 0; v < vocabulary; ++v) order[v] = v;
    std::stable_sort(order.begin(), order.end(),
      [&](int a, int b) { return x[a] > x[b]; });
    order.resize(40);
    std::sort(order.begin(), order.end());
    float peak = *std::max_element(x, x + vocabulary);
    double mass = 0, sum = 0;
    for(int v : order) mass += std::exp(((double)x[v] - peak) / 1.5);
    int token = -1;
    for(int v : order) {
      sum += std::exp(((double)x[v] - peak) / 1.5);
      if(token < 0 && sum > uniforms[i] * mass) token = v;
    }
    ok = ok && drawn[i] == token;
  }
  report("sample_tokens", ok);

  if(failures) printf("FAILED %d\n", failures);
  else printf("ALL PASSED\n");
  return failures ? 1 : 0;
}
