// test_decode_step.cpp -- the decode step of the C++ mirror
// (ocelotl_amd/host/kernel_backend.hpp: qk_norm_rope_d, paged_attention_d,
// logits_process_d) as a program chains them, on values whose results are
// known in closed form, and the lengths that it refuses.  Needs an MI355X.
#include <cmath>
#include <cstdio>
#include <string>
#include <vector>

#include "kernel_backend.hpp"
#include "okq.h"

using namespace ocelotl;

namespace {

struct Failure {
  std::string what;
};
#define CHECK(cond, msg)                                                                     \
  do {                                                                                       \
    if (!(cond)) throw Failure{std::string(msg) + "  [" #cond "] line " + std::to_string(__LINE__)}; \
  } while (0)

template <class T>
T ok(Result<T> r, const char *what) {
  if (r.is_err()) throw Failure{std::string(what) + ": " + r.error().to_string()};
  return std::move(r.value());
}
void ok(Result<void> r, const char *what) {
  if (r.is_err()) throw Failure{std::string(what) + ": " + r.error().to_string()};
}

template <class T>
T *to_device(const std::vector<T> &v) {
  void *p = nullptr;
  CHECK(okq_alloc(&p, v.size() * sizeof(T)) == OKQ_OK, "alloc");
  CHECK(okq_memcpy_h2d(p, v.data(), v.size() * sizeof(T), nullptr) == OKQ_OK, "copy");
  return static_cast<T *>(p);
}
template <class T>
std::vector<T> to_host(const T *p, size_t n) {
  std::vector<T> v(n);
  CHECK(okq_sync(nullptr) == OKQ_OK && okq_memcpy_d2h(v.data(), p, n * sizeof(T), nullptr) == OKQ_OK, "copy back");
  CHECK(okq_sync(nullptr) == OKQ_OK, "sync");
  return v;
}

// Two sequences of one and two tokens: keys of zero weigh every token alike,
// so attention gives the mean of the values, which the cache got through
// qk_norm_rope_d; its queries are turned by known angles.
void run() {
  HipKernelBackend be = ok(HipKernelBackend::create(0), "create");
  const size_t d = 64, q_heads = 4, kv_heads = 2, page = 16, n_pages = 3, tokens = 3;
  const size_t row = d * sizeof(float), bytes = n_pages * kv_heads * page * row;
  float *pages = to_device(std::vector<float>(2 * bytes / sizeof(float), NAN));
  okq_kv_pages cache{OKQ_TYPE_F32, (int64_t)n_pages, (int64_t)page, (int64_t)kv_heads, (int64_t)d,
                     (int64_t)(kv_heads * page * row), (int64_t)(page * row), (int64_t)row, pages,
                     pages + bytes / sizeof(float)};
  std::vector<float> q(tokens * q_heads * d, 1.0f), k(tokens * kv_heads * d, 0.0f), v(tokens * kv_heads * d);
  for (size_t t = 0; t < tokens; ++t)
    for (size_t i = 0; i < kv_heads * d; ++i) v[t * kv_heads * d + i] = (float)(t + 1) * (1.0f + (float)(i % 7));
  const std::vector<float> freq(d / 2, 0.5f);
  DeviceTensor qd = ok(be.upload(q.data(), q.size()), "q"), kd = ok(be.upload(k.data(), k.size()), "k"),
               vd = ok(be.upload(v.data(), v.size()), "v"), fd = ok(be.upload(freq.data(), freq.size()), "freq"),
               qo = ok(be.alloc(q.size()), "q_out");
  // token 0 is sequence 0's; tokens 1 and 2 are sequence 1's, on page 2
  const int32_t *pos = to_device(std::vector<int32_t>{0, 0, 3});
  const int64_t *slots = to_device(std::vector<int64_t>{5 * 0 + 0, 32, 33});
  ok(be.qk_norm_rope_d(qd, kd, vd, tokens, q_heads, nullptr, nullptr, 1e-6f, pos, fd, false, qo, cache, slots), "rope");
  const std::vector<float> turned = ok(qo.to_host_owned(), "q_out host");
  for (size_t i = 0; i < q_heads * d; ++i) CHECK(turned[i] == 1.0f, "position 0 turns nothing");
  const float lo = (float)(std::cos(1.5) - std::sin(1.5)), hi = (float)(std::cos(1.5) + std::sin(1.5));
  for (size_t i = 0; i < q_heads * d; ++i)
    CHECK(std::fabs(turned[2 * q_heads * d + i] - (i % d < d / 2 ? lo : hi)) < 1e-6f, "position 3 turns by 1.5");

  DeviceTensor q2 = ok(be.upload(turned.data(), 2 * q_heads * d), "q of the two sequences"),
               out = ok(be.alloc(2 * q_heads * d), "out"), lse = ok(be.alloc(2 * q_heads), "lse");
  const int32_t *table = to_device(std::vector<int32_t>{0, 2}), *lengths = to_device(std::vector<int32_t>{1, 2});
  ok(be.paged_attention_d(q2, 2, q_heads, cache, table, 1, lengths, 2, 0.125f, 0.0f, 0, out, &lse), "attention");
  const std::vector<float> o = ok(out.to_host_owned(), "out host"), ls = ok(lse.to_host_owned(), "lse host");
  for (size_t h = 0; h < q_heads; ++h) {
    CHECK(std::fabs(ls[h]) < 1e-6f && std::fabs(ls[q_heads + h] - std::log(2.0f)) < 1e-6f, "lse of zero scores");
    for (size_t i = 0; i < d; ++i) {
      const float one = 1.0f + (float)((h / 2 * d + i) % 7);
      CHECK(std::fabs(o[h * d + i] - one) < 1e-5f, "one token: its value");
      CHECK(std::fabs(o[(q_heads + h) * d + i] - 2.5f * one) < 1e-5f, "two tokens: their mean");
    }
  }

  std::vector<float> logits = {1, 5, 4, 2, /**/ 3, 3, 3, 3};
  DeviceTensor ld = ok(be.upload(logits.data(), 8), "logits"), lo2 = ok(be.alloc(8), "processed");
  const std::vector<float> rep = {2.0f, 1.0f};
  DeviceTensor rd = ok(be.upload(rep.data(), 2), "rep");
  int32_t *best = to_device(std::vector<int32_t>{-9, -9});
  LogitsOptions opt;
  opt.history = to_device(std::vector<int32_t>{1, 0});
  opt.history_len = to_device(std::vector<int32_t>{1, 0});
  opt.history_stride = 1;
  opt.repetition = &rd;
  opt.mask = to_device(std::vector<uint32_t>{15, 12});
  opt.mask_stride = 1;
  ok(be.logits_process_d(ld, 2, 4, opt, lo2, best), "logits");
  CHECK(ok(lo2.to_host_owned(), "processed host") ==
            (std::vector<float>{1, 2.5f, 4, 2, -INFINITY, -INFINITY, 3, 3}),
        "processed logits");
  CHECK(to_host(best, 2) == (std::vector<int32_t>{2, 2}), "greedy tokens");

  // lengths are checked before anything is launched
  auto e = be.paged_attention_d(q2, 3, q_heads, cache, table, 1, lengths, 2, 0.125f, 0.0f, 0, out, nullptr);
  CHECK(e.is_err() && e.error().as_kernel()->message.find("q length") != std::string::npos, "q length");
  e = be.logits_process_d(ld, 2, 5, opt, lo2, best);
  CHECK(e.is_err() && e.error().as_kernel()->message.find("logits length") != std::string::npos, "logits length");
  cache.type = OKQ_TYPE_Q4_K;
  e = be.qk_norm_rope_d(qd, kd, vd, tokens, q_heads, nullptr, nullptr, 1e-6f, pos, fd, false, qo, cache, slots);
  CHECK(e.is_err() && e.error().as_unsupported()->feature == "kv_cache_type", "cache type");
}

}  // namespace

int main() {
  try {
    run();
  } catch (const Failure &f) {
    std::printf("FAILED: %s\n", f.what.c_str());
    return 1;
  }
  std::printf("decode step: ok\n");
  return 0;
}
