// okq_logits.hip -- what happens to the output head's logits before a token is
// chosen: penalties for repeated tokens, biases, a grammar mask, and the
// index of the largest result.  Every operation is rounded on its own (this
// file is compiled without contraction), so that equal definitions choose the
// same token.
#include "okq_device.h"
#include "okq_internal.h"

namespace okq {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

namespace {

constexpr int kThreads = 512;
constexpr int kAhead = 8;  // history entries that a thread requests before it needs them
// A token's word: its count in the answer so far, or kPrompt where only the
// prompt holds it; kBiased where a bias is listed.
constexpr uint32_t kBiased = 0x80000000u, kPrompt = 0x40000000u, kCount = 0x3fffffffu;

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
template <class T>
__device__ __forceinline__ T load_any(const void *p) {  // any alignment
  T v;
  __builtin_memcpy(&v, p, sizeof v);
  return v;
}
template <class T>
__device__ __forceinline__ void store_any(void *p, T v) {
  __builtin_memcpy(p, &v, sizeof v);
}
__device__ __forceinline__ uint64_t wave_max(uint64_t k) {
  for (int d = 1; d < 64; d *= 2) {
    const uint64_t o = __shfl_xor(k, d);
    k = o > k ? o : k;
  }
  return k;
}

}  // namespace

// A workgroup per row and slice of 2048 V entries of the vocabulary, four
// consecutive ones a thread and step.  The slice's logits are requested first;
// while they come, the row's whole history and bias list are read (they stay
// in the caches for the row's other slices) and what falls into the slice is
// gathered in LDS: counts, whose order does not matter, by integer atomics;
// biases by the thread that holds a token's first entry, in list order.  The
// workgroup that ends last on a row turns the largest key into the token.
// Memory bounds it: the logits are read and written once.
template <int V, bool kMarks>  // kMarks: there is a history or biases
__global__ __launch_bounds__(kThreads) void logits_kernel(LogitsArgs a, int slices, uint64_t *keys, uint32_t *arrived) {
  constexpr int kSlice = 4 * kThreads * V, kWaves = kThreads / 64;
  __shared__ uint32_t marks[kMarks ? kSlice : 1];
  __shared__ float bsum[kMarks ? kSlice : 1];
  __shared__ uint64_t red[kWaves];
  __shared__ int list_at[kMarks ? kThreads : 1];
  __shared__ float list_value[kMarks ? kThreads : 1];
  __shared__ int wave_count[kWaves];
  const int row = (int)(blockIdx.x / (unsigned)slices), slice = (int)(blockIdx.x - (unsigned)row * (unsigned)slices);
  const int base = slice * kSlice, tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n = a.vocab - base < kSlice ? a.vocab - base : kSlice;
  const float *x = a.x + row * a.x_stride + base;
  float *out = a.out + row * a.out_stride + base;
  const uint32_t *mask = a.mask ? a.mask + row * a.mask_stride + base / 32 : nullptr;
  f32x4 v[V];
  uint32_t allowed[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int i = 4 * (tid + j * kThreads);
    allowed[j] = 0xffffffffu;
    if (i + 4 <= n) {
      v[j] = load_any<f32x4>(x + i);
    } else {
      v[j] = f32x4{0, 0, 0, 0};
      for (int e = 0; e < 4; ++e)
        if (i + e < n) v[j][e] = x[i + e];
    }
    if (mask && i < n) allowed[j] = mask[i >> 5] >> (i & 31);
  }
  float rep = 1.0f, freq = 0.0f, pres = 0.0f;
  if (kMarks) {
    const int32_t *hist = a.hist ? a.hist + row * a.hist_stride : nullptr;
    int ids[kAhead], len = 0, start = 0;
    if (hist) {
      len = a.hist_len[row] < a.hist_stride ? a.hist_len[row] : (int)a.hist_stride;
      start = a.hist_start ? a.hist_start[row] : 0;
#pragma unroll
      for (int j = 0; j < kAhead; ++j) ids[j] = tid + j * kThreads < a.hist_stride ? hist[tid + j * kThreads] : -1;
      rep = a.rep ? a.rep[row] : 1.0f;
      freq = a.freq ? a.freq[row] : 0.0f;
      pres = a.pres ? a.pres[row] : 0.0f;
    }
    for (int i = tid; i < kSlice / 4; i += kThreads) reinterpret_cast<u32x4 *>(marks)[i] = u32x4{0, 0, 0, 0};
    __syncthreads();
    if (hist) {
      auto count = [&](int i, int id) {
        const uint32_t at = (uint32_t)id - (uint32_t)base;
        if (i >= len || at >= (uint32_t)n) return;
        if (i >= start) atomicAdd(&marks[at], 1u);
        else atomicOr(&marks[at], kPrompt);
      };
#pragma unroll
      for (int j = 0; j < kAhead; ++j) count(tid + j * kThreads, ids[j]);
      for (int i = tid + kAhead * kThreads; i < len; i += kThreads) count(i, hist[i]);
    }
    if (a.bias_ids) {
      const int blen = a.bias_len[row] < a.bias_stride ? a.bias_len[row] : (int)a.bias_stride;
      const int32_t *bid = a.bias_ids + row * a.bias_stride;
      const float *b = a.bias + row * a.bias_stride;
      for (int i0 = 0; i0 < blen; i0 += kThreads) {
        // the slice's entries among the next kThreads, in list order
        const int i = i0 + tid;
        const uint32_t at = i < blen ? (uint32_t)bid[i] - (uint32_t)base : 0xffffffffu;
        const bool in = at < (uint32_t)n;
        const float value = in ? b[i] : 0.0f;
        const uint64_t who = __ballot(in);
        if (lane == 0) wave_count[wave] = __builtin_popcountll(who);
        __syncthreads();
        int place = 0, entries = 0;
        for (int w = 0; w < kWaves; ++w) {
          place += w < wave ? wave_count[w] : 0;
          entries += wave_count[w];
        }
        place += __builtin_popcountll(who & ((1ull << lane) - 1));
        if (in) {
          list_at[place] = (int)at;
          list_value[place] = value;
        }
        __syncthreads();
        if (in) {
          bool first = true;
          for (int e = 0; e < place; ++e) first = first && list_at[e] != (int)at;
          if (first) {
            const bool old = marks[at] & kBiased;
            float sum = old ? __fadd_rn(bsum[at], value) : value;
            for (int e = place + 1; e < entries; ++e)
              if (list_at[e] == (int)at) sum = __fadd_rn(sum, list_value[e]);
            bsum[at] = sum;
            if (!old) atomicOr(&marks[at], kBiased);
          }
        }
        __syncthreads();
      }
    }
    __syncthreads();
  }
  uint64_t best = 0;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int i = 4 * (tid + j * kThreads);
    if (kMarks) {
      const u32x4 c = reinterpret_cast<const u32x4 *>(marks)[i / 4];
      if (c[0] | c[1] | c[2] | c[3]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t k = c[e] & kCount;
          if (c[e] & ~kBiased) v[j][e] = v[j][e] > 0.0f ? __fdiv_rn(v[j][e], rep) : __fmul_rn(v[j][e], rep);
          if (k) v[j][e] = __fsub_rn(__fsub_rn(v[j][e], __fmul_rn(freq, (float)k)), pres);
          if (c[e] & kBiased) v[j][e] = __fadd_rn(v[j][e], bsum[i + e]);
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (!(allowed[j] >> e & 1u)) v[j][e] = -INFINITY;
      if (i + e < n) {
        const uint64_t key = key_of(v[j][e], base + i + e);
        best = key > best ? key : best;
      }
    }
    if (i + 4 <= n) {
      store_any(out + i, v[j]);
    } else {
      for (int e = 0; e < 4; ++e)
        if (i + e < n) out[i + e] = v[j][e];
    }
  }
  if (!a.best) return;
  best = wave_max(best);
  if (lane == 0) red[wave] = best;
  __syncthreads();
  if (tid != 0) return;
  for (int w = 1; w < kWaves; ++w) best = red[w] > best ? red[w] : best;
  if (slices == 1) {
    a.best[row] = best_of(best);
    return;
  }
  // Atomics of agent scope; the wait between them is the order that the last
  // workgroup relies on.  Both words are zero again afterwards.
  __hip_atomic_fetch_max(&keys[row], best, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  if (__hip_atomic_fetch_add(&arrived[row], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != (uint32_t)slices - 1) return;
  a.best[row] = best_of(__hip_atomic_exchange(&keys[row], (uint64_t)0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
  __hip_atomic_store(&arrived[row], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

size_t logits_workspace(int64_t rows) { return (size_t)rows * (sizeof(uint64_t) + sizeof(uint32_t)); }

hipError_t launch_logits(const LogitsArgs &a, void *workspace, int cu_count, hipStream_t s) {
  uint64_t *keys = static_cast<uint64_t *>(workspace);
  uint32_t *arrived = reinterpret_cast<uint32_t *>(keys + a.rows);
  auto run = [&](auto kernel, int slice) {
    const int slices = (int)(((int64_t)a.vocab + slice - 1) / slice);
    launch_timed(kernel, dim3((unsigned)((int64_t)a.rows * slices)), dim3(kThreads), 0u, s, a, slices, keys, arrived);
  };
  const bool marks = a.hist || a.bias_ids;
  // small slices until there is a workgroup for every CU: a call of few rows is
  // a wait for memory, which more CUs share
  if ((int64_t)a.rows * a.vocab <= (int64_t)cu_count * 8192) {
    if (marks) run(logits_kernel<1, true>, 4 * kThreads);
    else run(logits_kernel<1, false>, 4 * kThreads);
  } else {
    if (marks) run(logits_kernel<2, true>, 8 * kThreads);
    else run(logits_kernel<4, false>, 16 * kThreads);
  }
  return hipGetLastError();
}

}  // namespace okq
