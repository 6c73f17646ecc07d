// test_expert_layer.cpp -- a sparse layer of the C++ mirror
// (ocelotl_amd/host/kernel_backend.hpp: residual_norm_d, moe_route_d,
// moe_mlp_d) as a program chains them, on values whose results are known in
// closed form, and the lengths that it refuses.  Needs an MI355X.
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

// Q8_0 rows whose first value is `scale` (a power of two's f16 bits), the others zero.
std::vector<uint8_t> first_only(size_t rows, size_t cols, uint16_t scale) {
  std::vector<uint8_t> b(rows * cols / 32 * 34, 0);
  for (size_t r = 0; r < rows; ++r) {
    uint8_t *p = b.data() + r * cols / 32 * 34;
    p[0] = (uint8_t)(scale & 255);
    p[1] = (uint8_t)(scale >> 8);
    p[2] = 1;
  }
  return b;
}
std::vector<uint8_t> joined(std::vector<uint8_t> a, const std::vector<uint8_t> &b) {
  a.insert(a.end(), b.begin(), b.end());
  return a;
}

// Three rows of 32 values: x = 1, branch = 2 + row.  Expert 0 multiplies by 1,
// expert 1 by 2 (gate, up), both sum their first inner value (down).
void run() {
  HipKernelBackend be = ok(HipKernelBackend::create(0), "create");
  const size_t rows = 3, hidden = 32, inner = 64, experts = 2, top_k = 2;
  std::vector<float> x(rows * hidden, 1.0f), branch(rows * hidden), one(hidden, 1.0f), half(hidden, 0.5f);
  for (size_t i = 0; i < branch.size(); ++i) branch[i] = 2.0f + (float)(i / hidden);
  DeviceTensor xd = ok(be.upload(x.data(), x.size()), "x"), bd = ok(be.upload(branch.data(), branch.size()), "branch"),
               od = ok(be.upload(one.data(), hidden), "ones"), gd = ok(be.upload(half.data(), hidden), "gate"),
               sum = ok(be.alloc(rows * hidden), "sum"), normed = ok(be.alloc(rows * hidden), "normed");
  // without a norm: sum = 3 x + 2 * 0.5 * branch; its rows are constant, so their norm is 1
  ok(be.residual_norm_d(xd, bd, rows, hidden, nullptr, &gd, 2.0f, 3.0f, &od, 0.0f, &sum, &normed), "residual norm");
  const std::vector<float> s = ok(sum.to_host_owned(), "sum host"), n = ok(normed.to_host_owned(), "normed host");
  for (size_t i = 0; i < s.size(); ++i) {
    CHECK(s[i] == 5.0f + (float)(i / hidden), "sum");
    CHECK(std::fabs(n[i] - 1.0f) < 1e-6f, "normed");
  }

  // logits 0 and ln 3: probabilities 1/4 and 3/4
  std::vector<float> w(experts * hidden, 0.0f);
  w[hidden] = std::log(3.0f);
  DeviceTensor wd = ok(be.upload(w.data(), w.size()), "router"), weights = ok(be.alloc(rows * top_k), "weights");
  void *ids = nullptr;
  CHECK(okq_alloc(&ids, rows * top_k * sizeof(int32_t)) == OKQ_OK, "alloc");
  RouteOptions opt;
  opt.top_k = top_k;
  ok(be.moe_route_d(normed, rows, hidden, wd, experts, opt, (int32_t *)ids, weights, nullptr), "route");
  const std::vector<float> p = ok(weights.to_host_owned(), "weights host");
  std::vector<int32_t> chosen(rows * top_k);
  CHECK(okq_sync(nullptr) == OKQ_OK && okq_memcpy_d2h(chosen.data(), ids, chosen.size() * 4, nullptr) == OKQ_OK &&
            okq_sync(nullptr) == OKQ_OK, "ids back");
  for (size_t r = 0; r < rows; ++r) {
    CHECK(chosen[2 * r] == 1 && chosen[2 * r + 1] == 0, "the larger score first");
    CHECK(std::fabs(p[2 * r] - 0.75f) < 1e-6f && std::fabs(p[2 * r + 1] - 0.25f) < 1e-6f, "weights");
  }

  auto stack = [&](size_t ne0, size_t ne1, uint16_t a, uint16_t b) {
    const std::vector<uint8_t> bytes = joined(first_only(ne1, ne0, a), first_only(ne1, ne0, b));
    return ok(be.upload_quantized(GgmlTensorType::Q8_0, ne0, ne1 * experts, bytes.data(), bytes.size()), "weights");
  };
  const QuantizedWeight gate = stack(hidden, inner, 0x3c00, 0x4000), up = stack(hidden, inner, 0x3c00, 0x4000),
                        down = stack(inner, hidden, 0x3c00, 0x3c00);
  DeviceTensor out = ok(be.alloc(rows * hidden), "out");
  ok(be.moe_mlp_d(normed, rows, hidden, inner, experts, top_k, (const int32_t *)ids, weights, gate, up, down, out), "experts");
  const std::vector<float> o = ok(out.to_host_owned(), "out host");
  auto gated = [](double g) { return g / (1.0 + std::exp(-g)) * g; };
  const float want = (float)(0.75 * gated(2.0) + 0.25 * gated(1.0));
  for (float v : o) CHECK(std::fabs(v - want) < 1e-5f, "experts' sum");

  // lengths are checked before anything is launched
  auto e = be.residual_norm_d(xd, bd, rows + 1, hidden, nullptr, nullptr, 1.0f, 1.0f, &od, 0.0f, &sum, &normed);
  CHECK(e.is_err() && e.error().as_kernel()->message.find("x length") != std::string::npos, "x length");
  e = be.moe_route_d(normed, rows, hidden, wd, experts + 1, opt, (int32_t *)ids, weights, nullptr);
  CHECK(e.is_err() && e.error().as_kernel()->message.find("weight length") != std::string::npos, "weight length");
  e = be.moe_mlp_d(normed, rows, hidden, inner, experts + 1, top_k, (const int32_t *)ids, weights, gate, up, down, out);
  CHECK(e.is_err() && e.error().as_kernel()->message.find("shape does not match") != std::string::npos, "stack shape");
  CHECK(okq_free(ids) == OKQ_OK, "free");
}

}  // namespace

int main() {
  try {
    run();
  } catch (const Failure &f) {
    std::printf("FAILED: %s\n", f.what.c_str());
    return 1;
  }
  std::printf("expert layer: ok\n");
  return 0;
}
