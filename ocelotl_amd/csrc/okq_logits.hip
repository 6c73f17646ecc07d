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

constexpr int kThreads = 1024;
constexpr int kAhead = 4;  // history entries that a thread requests before it needs them
// A token's word: how often the answer so far holds it, kPrompt if the prompt
// does, kBiased if a bias is listed, and (for lists of at most kThreads) the
// bias's place in its list, which leaves the count kShortBits bits.
constexpr uint32_t kBiased = 0x80000000u, kPrompt = 0x40000000u;
constexpr int kShortBits = 20;
static_assert(kThreads <= 1 << (30 - kShortBits), "a place fits beside the count");

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
// Any alignment; past the caches, where nothing of a row is read twice.
typedef f32x4 f32x4_4 __attribute__((aligned(4)));
__device__ __forceinline__ f32x4 load_past(const float *p) {
  return __builtin_nontemporal_load(reinterpret_cast<const f32x4_4 *>(p));
}
__device__ __forceinline__ void store_past(float *p, f32x4 v) {
  __builtin_nontemporal_store(v, reinterpret_cast<f32x4_4 *>(p));
}
__device__ __forceinline__ uint64_t wave_max(uint64_t k) {
  for (int d = 1; d < 64; d *= 2) {
    const uint64_t o = __shfl_xor(k, d);
    k = o > k ? o : k;
  }
  return k;
}

// Where the slices of a row meet.  Each row has a line of its own: rows that
// share one wait for each other's atomics (8 rows of 128256: 9.1 us).
struct alignas(128) Meeting {
  uint64_t key;
  uint32_t arrived;
};

// A slice's best key joins its row's; the last slice's workgroup names the
// token.  Atomics of agent scope; the wait between them is the order that the
// last one relies on.  Both words are zero again afterwards.
__device__ __forceinline__ void choose(const LogitsArgs &a, int row, int slices, uint64_t best, Meeting *meet) {
  if (slices > 1) {
    __hip_atomic_fetch_max(&meet[row].key, best, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (__hip_atomic_fetch_add(&meet[row].arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != (uint32_t)slices - 1)
      return;
    best = __hip_atomic_exchange(&meet[row].key, (uint64_t)0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(&meet[row].arrived, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  a.best[row] = best_of(best);
}

}  // namespace

// A workgroup per row and slice of 4096 V entries of the vocabulary, four
// consecutive ones a thread and step.  The slice's logits are requested first;
// while they come, the row's whole history and bias list are read (they stay
// in the caches for the row's other slices) and what falls into the slice is
// gathered in LDS: counts, whose order does not matter, by integer atomics;
// biases by the thread that holds a token's first entry, in list order.  The
// workgroup that ends last on a row turns the largest key into the token.
// Memory bounds it: the logits are read and written once (200 rows of 262144
// with a mask, 426 MB: 85 us, 5.0 TB/s); a single row the chain logits or lists
// -> LDS -> result -> meeting place (128256 entries, 1 MB: 5.7 us).  Bias lists
// of more than kThreads entries go through LDS kThreads at a time, with two
// waits each and a search for a token's first entry (128256 entries: 6.2 us with
// 1024 biases, 12.2 with 1025, 17.2 with 2000; 64 rows 14.4, 50 and 76): request
// biases are tens, so that is left as it is.
template <int V, bool kMarks, int kBias>  // a history; biases (with marks): 1 a list of kThreads at most, 2 a longer one
__global__ __launch_bounds__(kThreads) void logits_kernel(LogitsArgs a, int slices, Meeting *meet) {
  constexpr int kSlice = 4 * kThreads * V, kWaves = kThreads / 64;
  constexpr uint32_t kCount = kBias == 1 ? (1u << kShortBits) - 1 : 0x3fffffffu;
  __shared__ uint32_t marks[kMarks ? kSlice : 1];
  __shared__ float bsum[kBias == 2 ? kSlice : 1];
  __shared__ int list_at[kBias ? kThreads : 1];
  __shared__ float list_value[kBias ? kThreads : 1];
  __shared__ int wave_count[kWaves];
  __shared__ int twice;  // a token is listed twice
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
      v[j] = load_past(x + i);
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
  int entries = 0;  // of the list in LDS
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
    // the slice's entries of the list's next kThreads, in list order: where
    // each goes, then the entry itself
    uint32_t at = 0;
    uint64_t who = 0;
    auto find = [&](int i) {
      at = (uint32_t)bid - (uint32_t)base;
      who = __ballot(i < blen && at < (uint32_t)n);
      if (lane == 0) wave_count[wave] = __builtin_popcountll(who);
    };
    auto list = [&](int &place) {  // false: not this slice's
      entries = 0;
      place = __builtin_popcountll(who & ((1ull << lane) - 1));
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const int c = wave_count[w];
        place += w < wave ? c : 0;
        entries += c;
      }
      if (!(who >> lane & 1)) return false;
      list_at[place] = (int)at;
      list_value[place] = bvalue;
      return true;
    };
    if (kBias == 2 && biased) find(tid);
    if (kBias == 1 && tid == 0) twice = 0;
    __syncthreads();
    auto count = [&](int i, int token) {
      const uint32_t where = (uint32_t)token - (uint32_t)base;
      if (i >= len || where >= (uint32_t)n) return;
      if (i >= start) atomicAdd(&marks[where], 1u);
      else atomicOr(&marks[where], kPrompt);
    };
    if (hist) {
#pragma unroll
      for (int j = 0; j < kAhead; ++j) count(tid + j * kThreads, id[j]);
      for (int i = tid + kAhead * kThreads; i < len; i += kThreads) count(i, ids[i]);
    }
    if constexpr (kBias == 1) {
      at = (uint32_t)bid - (uint32_t)base;
      const bool in = tid < blen && at < (uint32_t)n;
      list_at[tid] = in ? (int)at : -1;
      list_value[tid] = bvalue;
      if (in && (atomicOr(&marks[at], kBiased | (uint32_t)tid << kShortBits) & kBiased)) twice = 1;
    }
    if constexpr (kBias == 2) {
      for (int i0 = 0; i0 < blen; i0 += kThreads) {
        if (i0 > 0) {
          if (i0 + tid < blen) {
            bid = bids[i0 + tid];
            bvalue = bias[i0 + tid];
          }
          find(i0 + tid);
          __syncthreads();
        }
        int place;
        const bool in = list(place);
        __syncthreads();
        bool first = in;
        for (int e = 0; e < place && first; ++e) first = list_at[e] != (int)at;
        if (first) {  // a token's first entry here adds them all
          const bool old = marks[at] & kBiased;
          float sum = old ? __fadd_rn(bsum[at], bvalue) : bvalue;
          for (int e = place + 1; e < entries; ++e)
            if (list_at[e] == (int)at) sum = __fadd_rn(sum, list_value[e]);
          bsum[at] = sum;
          if (!old) atomicOr(&marks[at], kBiased);
        }
        __syncthreads();
      }
    }
    __syncthreads();
  }
  float top = -INFINITY;  // the thread's largest, its lowest place, and whether one is NaN
  int where = 0;
  bool nan = false;
  auto rank = [&](float value, int i) {
    nan = nan || value != value;
    where = value > top ? i : where;
    top = value > top ? value : top;
  };
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int i = 4 * (tid + j * kThreads);
    if constexpr (kMarks) {
      const u32x4 c = reinterpret_cast<const u32x4 *>(marks)[i / 4];
      if (c[0] | c[1] | c[2] | c[3]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t k = c[e] & kCount;
          if (c[e] & (kPrompt | kCount)) v[j][e] = v[j][e] > 0.0f ? __fdiv_rn(v[j][e], rep) : __fmul_rn(v[j][e], rep);
          if (k) v[j][e] = __fsub_rn(__fsub_rn(v[j][e], __fmul_rn(freq, (float)k)), pres);
          if constexpr (kBias == 2)
            if (c[e] & kBiased) v[j][e] = __fadd_rn(v[j][e], bsum[i + e]);
          if constexpr (kBias == 1)
            if (c[e] & kBiased) {
              float sum = list_value[c[e] >> kShortBits & (kThreads - 1)];
              if (twice) {  // some token is: the places of a word may be mixed
                bool any = false;
                for (int b = 0; b < blen; ++b)
                  if (list_at[b] == i + e) {
                    sum = any ? __fadd_rn(sum, list_value[b]) : list_value[b];
                    any = true;
                  }
              }
              v[j][e] = __fadd_rn(v[j][e], sum);
            }
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
      for (int e = 0; e < 4; ++e) rank(v[j][e], i + e);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < n) {
          out[i + e] = v[j][e];
          rank(v[j][e], i + e);
        }
    }
  }
  if (a.best) {
    uint64_t best = wave_max(nan ? ~0ull : key_of(top, base + where));
    if (lane == 0) red[wave] = best;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < kWaves; ++w) best = red[w] > best ? red[w] : best;
      choose(a, row, slices, best, meet);
    }
  }
}

size_t logits_workspace(int64_t rows) { return (size_t)rows * sizeof(Meeting); }

hipError_t launch_logits(const LogitsArgs &a, void *workspace, int cu_count, hipStream_t s) {
  Meeting *meet = static_cast<Meeting *>(workspace);
  auto run = [&](auto kernel, int slice) {
    const int slices = (int)(((int64_t)a.vocab + slice - 1) / slice);
    launch_timed(kernel, dim3((unsigned)((int64_t)a.rows * slices)), dim3(kThreads), 0u, s, a, slices, meet);
  };
  // small slices until there is a workgroup for every CU: a call of few rows is
  // a wait for memory, which more CUs share
  // (16 rows of 128256: 7.9 us in small slices, 9.3 in large; 32 rows: 12.5 and 9.9)
  const bool few = (int64_t)a.rows * a.vocab <= (int64_t)cu_count * 8192;
  if (a.bias_ids && (a.bias_stride > kThreads || a.hist_stride >= 1 << kShortBits)) {
    if (few) run(logits_kernel<1, true, 2>, 4 * kThreads);
    else run(logits_kernel<2, true, 2>, 8 * kThreads);
  } else if (a.bias_ids) {
    if (few) run(logits_kernel<1, true, 1>, 4 * kThreads);
    else run(logits_kernel<4, true, 1>, 16 * kThreads);
  } else if (a.hist) {
    if (few) run(logits_kernel<1, true, 0>, 4 * kThreads);
    else run(logits_kernel<4, true, 0>, 16 * kThreads);
  } else {
    if (few) run(logits_kernel<1, false, 0>, 4 * kThreads);
    else run(logits_kernel<4, false, 0>, 16 * kThreads);
  }
  return hipGetLastError();
}

}  // namespace okq
