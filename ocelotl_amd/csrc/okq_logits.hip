// okq_logits.hip -- what happens to the output head's logits before a token is
// chosen: penalties for repeated tokens, biases, a grammar mask, and the
// index of the largest result.  Every operation is rounded on its own (this
// file is compiled without contraction), so that equal definitions choose the
// same token.
#include "okq_device.h"
#include "okq_internal.h"

namespace okq {

namespace {

constexpr int kSlice = 4096;  // vocabulary entries of a workgroup
constexpr uint32_t kSeen = 0x80000000u;

// A result's place in the order of results: larger values first, then lower
// indexes, NaN before everything.  Zeros of both signs are one value.
__device__ __forceinline__ uint64_t key_of(float v, int i) {
  const uint32_t u = as_u32(v + 0.0f);
  const uint32_t o = v != v ? 0xffffffffu : (u & 0x80000000u) ? ~u : u | 0x80000000u;
  return ((uint64_t)o << 32) | (0xffffffffu - (uint32_t)i);
}
__device__ __forceinline__ int32_t best_of(uint64_t key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return o == 0xffffffffu || o <= 0x007fffffu ? -1 : (int32_t)(0xffffffffu - (uint32_t)key);
}
__device__ __forceinline__ uint64_t wave_max(uint64_t k) {
  for (int d = 1; d < 64; d *= 2) {
    const uint64_t o = __shfl_xor(k, d);
    k = o > k ? o : k;
  }
  return k;
}

}  // namespace

// A workgroup per row and slice of the vocabulary.  The row's history and
// biases that fall into the slice are gathered into LDS (integer counts, whose
// order does not matter; bias sums by one wave in list order), then the slice
// streams through.
__global__ __launch_bounds__(256) void logits_kernel(LogitsArgs a, int slices, uint64_t *keys) {
  __shared__ uint32_t cnt[kSlice];
  __shared__ float bsum[kSlice];
  __shared__ uint64_t red[4];
  const int row = (int)(blockIdx.x / (unsigned)slices), slice = (int)(blockIdx.x % (unsigned)slices);
  const int base = slice * kSlice, tid = (int)threadIdx.x;
  const int n = a.vocab - base < kSlice ? a.vocab - base : kSlice;
  for (int i = tid; i < kSlice; i += 256) {
    cnt[i] = 0;
    bsum[i] = 0.0f;
  }
  __syncthreads();
  if (a.bias_ids && tid < 64) {
    const int64_t len = a.bias_len[row] < a.bias_stride ? a.bias_len[row] : a.bias_stride;
    const int32_t *ids = a.bias_ids + row * a.bias_stride;
    const float *b = a.bias + row * a.bias_stride;
    for (int64_t j = 0; j < len; j += 64) {
      const int64_t i = j + tid;
      const uint32_t at = i < len ? (uint32_t)ids[i] - (uint32_t)base : 0xffffffffu;
      const bool in = at < (uint32_t)n;
      const float v = in ? b[i] : 0.0f;
      // entries of one token follow each other in list order, whatever lanes hold them
      uint64_t left = __ballot(in);
      while (left) {
        const int first = __builtin_ctzll(left);
        if (tid == first) bsum[at] += v;
        wave_sync();
        left &= left - 1;
      }
    }
  }
  if (a.hist) {
    const int64_t len = a.hist_len[row] < a.hist_stride ? a.hist_len[row] : a.hist_stride;
    const int64_t start = a.hist_start ? a.hist_start[row] : 0;
    const int32_t *ids = a.hist + row * a.hist_stride;
    for (int64_t i = tid; i < len; i += 256) {
      const uint32_t at = (uint32_t)ids[i] - (uint32_t)base;
      if (at >= (uint32_t)n) continue;
      atomicOr(&cnt[at], kSeen);
      if (i >= start) atomicAdd(&cnt[at], 1u);
    }
  }
  __syncthreads();
  const float rep = a.rep ? a.rep[row] : 1.0f, freq = a.freq ? a.freq[row] : 0.0f, pres = a.pres ? a.pres[row] : 0.0f;
  const float *x = a.x + row * a.x_stride + base;
  float *out = a.out + row * a.out_stride + base;
  const uint32_t *mask = a.mask ? a.mask + row * a.mask_stride + base / 32 : nullptr;
  uint64_t best = 0;
  for (int i = tid; i < n; i += 256) {
    float v = x[i];
    const uint32_t c = cnt[i];
    if (c) {
      v = v > 0.0f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
      const uint32_t k = c & ~kSeen;
      if (k) v = __fsub_rn(__fsub_rn(v, __fmul_rn(freq, (float)k)), pres);
    }
    if (a.bias_ids) v = __fadd_rn(v, bsum[i]);
    if (mask && !(mask[i >> 5] >> (i & 31) & 1u)) v = -INFINITY;
    out[i] = v;
    const uint64_t key = key_of(v, base + i);
    best = key > best ? key : best;
  }
  if (!keys) return;
  best = wave_max(best);
  if ((tid & 63) == 0) red[tid >> 6] = best;
  __syncthreads();
  if (tid == 0) {
    uint64_t k = red[0];
    for (int w = 1; w < 4; ++w) k = red[w] > k ? red[w] : k;
    keys[(int64_t)row * slices + slice] = k;
  }
}

__global__ __launch_bounds__(64) void logits_best_kernel(const uint64_t *keys, int slices, int32_t *best) {
  const uint64_t *k = keys + (int64_t)blockIdx.x * slices;
  uint64_t b = 0;
  for (int i = (int)threadIdx.x; i < slices; i += 64) b = k[i] > b ? k[i] : b;
  b = wave_max(b);
  if (threadIdx.x == 0) best[blockIdx.x] = best_of(b);
}

size_t logits_workspace(int64_t rows, int64_t vocab) { return (size_t)rows * ((size_t)vocab + kSlice - 1) / kSlice * 8 + 8 * rows; }

hipError_t launch_logits(const LogitsArgs &a, void *workspace, hipStream_t s) {
  const int slices = (a.vocab + kSlice - 1) / kSlice;
  uint64_t *keys = a.best ? static_cast<uint64_t *>(workspace) : nullptr;
  launch_timed(logits_kernel, dim3((unsigned)((int64_t)a.rows * slices)), dim3(256), 0u, s, a, slices, keys);
  if (a.best) hipLaunchKernelGGL(logits_best_kernel, dim3((unsigned)a.rows), dim3(64), 0, s, keys, slices, a.best);
  return hipGetLastError();
}

}  // namespace okq
