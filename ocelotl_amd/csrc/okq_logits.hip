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
constexpr int kVB = 4, kVH = 4;
constexpr int kAhead = 8;  // history entries that a thread requests before it needs them
// A token's word: its count in the answer so far, or kPrompt where only the
// prompt holds it; kBiased where a bias is listed.
constexpr uint32_t kBiased = 0x80000000u, kPrompt = 0x40000000u, kCount = 0x3fffffffu;

// A result's place in the order of results: larger values first, then lower
// indexes; all ones is for NaN, before everything.  Zeros of both signs are
// one value.
__device__ __forceinline__ uint64_t key_of(float v, int i) {
  const uint32_t u = as_u32(v + 0.0f);
  const uint32_t o = (u & 0x80000000u) ? ~u : u | 0x80000000u;
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
// Any alignment, and past the caches, which the logits of the rows to come fill.
__device__ __forceinline__ void store_past(float *p, f32x4 v) {
  typedef f32x4 f32x4_4 __attribute__((aligned(4)));
  __builtin_nontemporal_store(v, reinterpret_cast<f32x4_4 *>(p));
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
template <int V, bool kMarks, bool kBias>  // a history; biases (with marks)
__global__ __launch_bounds__(kThreads) void logits_kernel(LogitsArgs a, int slices, uint64_t *keys, uint32_t *arrived) {
  constexpr int kSlice = 4 * kThreads * V, kWaves = kThreads / 64;
  __shared__ uint32_t marks[kMarks ? kSlice : 1];
  __shared__ float bsum[kBias ? kSlice : 1];
  __shared__ int list_at[kBias ? kThreads : 1];
  __shared__ float list_value[kBias ? kThreads : 1];
  __shared__ int wave_count[kWaves];
  __shared__ uint64_t red[kWaves];
  const int row = (int)(blockIdx.x / (unsigned)slices), slice = (int)(blockIdx.x - (unsigned)row * (unsigned)slices);
  const int base = slice * kSlice, tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n = a.vocab - base < kSlice ? a.vocab - base : kSlice;
  const float *x = a.x + row * a.x_stride + base;
  float *out = a.out + row * a.out_stride + base;
  f32x4 v[V];
  uint32_t allowed[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int i = 4 * (tid + j * kThreads);
    if (i + 4 <= n) {
      v[j] = load_any<f32x4>(x + i);
    } else {
      v[j] = f32x4{0, 0, 0, 0};
      for (int e = 0; e < 4; ++e)
        if (i + e < n) v[j][e] = x[i + e];
    }
  }
  // Everything else that the row needs is requested at once, within its
  // buffers whatever the lengths are, and looked at later: read one after the
  // other, lengths first, these are six waits for memory.
  const float *some = x;  // stands in for an absent parameter
  float rep = *(a.rep ? a.rep + row : some), freq = *(a.freq ? a.freq + row : some), pres = *(a.pres ? a.pres + row : some);
  const int32_t *none = reinterpret_cast<const int32_t *>(some);
  const bool hist = kMarks && a.hist, biased = kBias && a.bias_ids;
  int len = *(hist ? a.hist_len + row : none), start = *(hist && a.hist_start ? a.hist_start + row : none);
  int blen = *(biased ? a.bias_len + row : none);
  const int32_t *ids = a.hist + row * a.hist_stride, *bids = a.bias_ids + row * a.bias_stride;
  const float *bias = a.bias + row * a.bias_stride;
  int id[kMarks ? kAhead : 1], bid = -1;
  float bvalue = 0.0f;
  if (hist) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j) id[j] = tid + j * kThreads < a.hist_stride ? ids[tid + j * kThreads] : -1;
  }
  if (biased && tid < a.bias_stride) {
    bid = bids[tid];
    bvalue = bias[tid];
  }
  if (a.mask) {
    const uint32_t *mask = a.mask + row * a.mask_stride + base / 32;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int i = 4 * (tid + j * kThreads);
      allowed[j] = i < n ? mask[i >> 5] >> (i & 31) : 0;
    }
  }
  rep = a.rep ? rep : 1.0f;
  freq = a.freq ? freq : 0.0f;
  pres = a.pres ? pres : 0.0f;
  len = !hist ? 0 : len < a.hist_stride ? len : (int)a.hist_stride;
  start = hist && a.hist_start ? start : 0;
  blen = !biased ? 0 : blen < a.bias_stride ? blen : (int)a.bias_stride;
  if constexpr (kMarks) {
    for (int i = tid; i < kSlice / 4; i += kThreads) reinterpret_cast<u32x4 *>(marks)[i] = u32x4{0, 0, 0, 0};
    __syncthreads();
    auto count = [&](int i, int token) {
      const uint32_t at = (uint32_t)token - (uint32_t)base;
      if (i >= len || at >= (uint32_t)n) return;
      if (i >= start) atomicAdd(&marks[at], 1u);
      else atomicOr(&marks[at], kPrompt);
    };
    if (hist) {
#pragma unroll
      for (int j = 0; j < kAhead; ++j) count(tid + j * kThreads, id[j]);
      for (int i = tid + kAhead * kThreads; i < len; i += kThreads) count(i, ids[i]);
    }
    if constexpr (kBias) {
      for (int i0 = 0; i0 < blen; i0 += kThreads) {
        // the slice's entries among the next kThreads, in list order
        const int i = i0 + tid;
        if (i0 > 0 && i < blen) {
          bid = bids[i];
          bvalue = bias[i];
        }
        const uint32_t at = (uint32_t)bid - (uint32_t)base;
        const bool in = i < blen && at < (uint32_t)n;
        const uint64_t who = __ballot(in);
        if (lane == 0) wave_count[wave] = __builtin_popcountll(who);
        __syncthreads();
        int place = 0, entries = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
          const int c = wave_count[w];
          place += w < wave ? c : 0;
          entries += c;
        }
        place += __builtin_popcountll(who & ((1ull << lane) - 1));
        if (in) {
          list_at[place] = (int)at;
          list_value[place] = bvalue;
        }
        __syncthreads();
        if (in) {
          bool first = true;
          for (int e = 0; e < place; ++e) first = first && list_at[e] != (int)at;
          if (first) {
            const bool old = marks[at] & kBiased;
            float sum = old ? __fadd_rn(bsum[at], bvalue) : bvalue;
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
  float top = -INFINITY;  // the thread's largest, its lowest place, and whether one is NaN
  int where = 0;
  bool nan = false;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int i = 4 * (tid + j * kThreads);
    if constexpr (kMarks) {
      const u32x4 c = reinterpret_cast<const u32x4 *>(marks)[i / 4];
      if (c[0] | c[1] | c[2] | c[3]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t k = c[e] & kCount;
          if (c[e] & ~kBiased) v[j][e] = v[j][e] > 0.0f ? __fdiv_rn(v[j][e], rep) : __fmul_rn(v[j][e], rep);
          if (k) v[j][e] = __fsub_rn(__fsub_rn(v[j][e], __fmul_rn(freq, (float)k)), pres);
          if constexpr (kBias)
            if (c[e] & kBiased) v[j][e] = __fadd_rn(v[j][e], bsum[i + e]);
        }
      }
    }
    if (a.mask) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[j][e] = allowed[j] >> e & 1u ? v[j][e] : -INFINITY;
    }
    if (i + 4 <= n) {
      store_past(out + i, v[j]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        nan = nan || v[j][e] != v[j][e];
        where = v[j][e] > top ? i + e : where;
        top = v[j][e] > top ? v[j][e] : top;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < n) {
          out[i + e] = v[j][e];
          nan = nan || v[j][e] != v[j][e];
          where = v[j][e] > top ? i + e : where;
          top = v[j][e] > top ? v[j][e] : top;
        }
    }
  }
  uint64_t best = nan ? ~0ull : key_of(top, base + where);
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
  // small slices until there is a workgroup for every CU: a call of few rows is
  // a wait for memory, which more CUs share
  const bool few = (int64_t)a.rows * a.vocab <= (int64_t)cu_count * 8192;
  if (a.bias_ids) {
    if (few) run(logits_kernel<1, true, true>, 4 * kThreads);
    else run(logits_kernel<kVB, true, true>, 4 * kVB * kThreads);
  } else if (a.hist) {
    if (few) run(logits_kernel<1, true, false>, 4 * kThreads);
    else run(logits_kernel<kVH, true, false>, 4 * kVH * kThreads);
  } else {
    if (few) run(logits_kernel<1, false, false>, 4 * kThreads);
    else run(logits_kernel<4, false, false>, 16 * kThreads);
  }
  return hipGetLastError();
}

}  // namespace okq
