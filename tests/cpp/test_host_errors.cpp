// test_host_errors.cpp -- what the C-ABI's host side does where the HIP runtime
// refuses something, on the CPU: the runtime's entry points that libokq.so
// calls are defined here and fail on request, so nothing reaches a device.
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <map>
#include <string>
#include <utility>

#include <hip/hip_runtime_api.h>

#include "okq.h"

namespace {

int g_launches = 0;       // kernels launched
int g_refuse_launch = 0;  // as many launches, from the next one on, are refused
bool g_capturing = false;
bool g_no_memory = false;
hipError_t g_error = hipSuccess;

hipError_t left(hipError_t e) {
  if (e != hipSuccess) g_error = e;
  return e;
}

}  // namespace

extern "C" {

hipError_t hipGetDevice(int *d) {
  *d = 0;
  return hipSuccess;
}
hipError_t hipGetDevicePropertiesR0600(hipDeviceProp_tR0600 *p, int) {
  std::memset(p, 0, sizeof *p);
  std::strcpy(p->gcnArchName, "gfx950");
  p->multiProcessorCount = 256;
  return hipSuccess;
}
hipError_t hipMalloc(void **p, size_t n) {
  if (g_no_memory) return left(hipErrorOutOfMemory);
  *p = std::malloc(n);
  return hipSuccess;
}
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus *s) {
  *s = g_capturing ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone;
  return hipSuccess;
}
// what a launch's <<<...>>> goes through before hipLaunchKernel
hipError_t __hipPushCallConfiguration(dim3, dim3, size_t, hipStream_t) { return hipSuccess; }
hipError_t __hipPopCallConfiguration(dim3 *, dim3 *, size_t *, hipStream_t *) { return hipSuccess; }
hipError_t hipLaunchKernel(const void *, dim3, dim3, void **, size_t, hipStream_t) {
  if (g_refuse_launch > 0) {
    --g_refuse_launch;
    return left(hipErrorLaunchFailure);
  }
  ++g_launches;
  return hipSuccess;
}
hipError_t hipGetLastError() {
  const hipError_t e = g_error;
  g_error = hipSuccess;
  return e;
}

}  // extern "C"

namespace {

struct Failure {
  std::string what;
};
#define CHECK(cond, msg)                                                                     \
  do {                                                                                       \
    if (!(cond)) throw Failure{std::string(msg) + "  [" #cond "] line " + std::to_string(__LINE__)}; \
  } while (0)

void *const P = reinterpret_cast<void *>(4096);  // an aligned address that is never read

void *stream(int i) { return reinterpret_cast<void *>((size_t)(0x1000 * (i + 1))); }

std::string error() {
  char buf[512];
  okq_last_error(buf, sizeof buf);
  return buf;
}

okq_status logits(void *s) {
  return okq_logits_process((const float *)P, 1000, 2, 1000, nullptr, 0, nullptr, nullptr, nullptr, nullptr, nullptr,
                            nullptr, nullptr, 0, nullptr, nullptr, 0, (float *)P, 1000, (int32_t *)P, s);
}

// One sequence of up to 4000 tokens, which is split; or a batch that is not.
okq_status attention(void *s, int64_t seqs = 1, int64_t max_length = 4000) {
  const okq_kv_pages c{OKQ_TYPE_BF16, 4000, 16, 2, 64, 2 * 16 * 128, 16 * 128, 128, P, P};
  return okq_paged_attention((const float *)P, 4 * 64, seqs, 4, &c, (const int32_t *)P, 250, (const int32_t *)P,
                             max_length, 0.125f, 0.0f, 0, (float *)P, 4 * 64, nullptr, s);
}

int launches(okq_status (*call)(void *), void *s, okq_status want) {
  const int before = g_launches;
  const okq_status st = call(s);
  CHECK(st == want, "status " + std::to_string(st) + " (" + error() + ")");
  return g_launches - before;
}
okq_status split_attention(void *s) { return attention(s); }

// Counters that a kernel expects to be zero are filled by the first call on a
// stream; where that fill is refused, the next call fills them.
void refused_fills() {
  int i = 0;
  for (okq_status (*call)(void *) : {logits, split_attention}) {
    void *s = stream(i++);
    g_refuse_launch = 1;
    CHECK(launches(call, s, OKQ_E_LAUNCH) == 0, "a refused fill is an error");
    CHECK(launches(call, s, OKQ_OK) == 2, "the next call fills and computes");
    CHECK(launches(call, s, OKQ_OK) == 1, "later calls compute only");
  }
  // a fill that would be recorded instead of run fills nothing yet
  for (okq_status (*call)(void *) : {logits, split_attention}) {
    void *s = stream(i++);
    g_refuse_launch = 1;
    CHECK(launches(call, s, OKQ_E_LAUNCH) == 0, "a refused fill is an error");
    g_capturing = true;
    CHECK(launches(call, s, OKQ_E_ALLOC) == 0, "nothing is recorded");
    g_capturing = false;
    CHECK(launches(call, s, OKQ_OK) == 2, "the next call fills and computes");
  }
}

// A workspace that cannot be had is the call's own.
void missing_workspaces() {
  const std::pair<okq_status (*)(void *), const char *> calls[] = {{logits, "logits_process workspace"},
                                                                   {split_attention, "paged_attention workspace"}};
  int i = 0;
  for (const auto &[call, words] : calls) {
    g_capturing = true;
    CHECK(launches(call, stream(i++), OKQ_E_ALLOC) == 0, "not during a capture");
    CHECK(error().find(words) != std::string::npos && error().find("capture") != std::string::npos, error());
    g_capturing = false;
    g_no_memory = true;
    CHECK(launches(call, stream(i++), OKQ_E_ALLOC) == 0, "not without memory");
    CHECK(error().find(words) != std::string::npos && error().find("hipMalloc") != std::string::npos, error());
    g_no_memory = false;
  }
  g_no_memory = true;
  CHECK(attention(stream(i), 700, 16) == OKQ_OK, "a call that splits nothing goes on without");
  g_no_memory = false;
}

}  // namespace

int main(int argc, char **argv) {
  const std::map<std::string, void (*)()> cases = {{"refused_fills", refused_fills},
                                                   {"missing_workspaces", missing_workspaces}};
  const auto it = cases.find(argc > 1 ? argv[1] : "");
  if (it == cases.end()) {
    std::printf("no such case\n");
    return 2;
  }
  try {
    it->second();
  } catch (const Failure &f) {
    std::printf("FAILED: %s\n", f.what.c_str());
    return 1;
  }
  std::printf("%s: ok\n", argv[1]);
  return 0;
}
