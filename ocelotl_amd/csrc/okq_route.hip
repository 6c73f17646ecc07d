// okq_route.hip -- routing to experts: the router's product, its scores, and
// the choice of every token's experts with their weights.
//
//   z = x W^T + bias,  p = softmax(z) or 1 / (1 + exp(-z)),  c = p + choice_bias
//   groups: the top_groups of largest sum of their group_best largest c stay
//   ids: the top_k experts of largest c, ties to the lowest; weights: their p,
//   divided by their sum if renormalised, times scale
//
// Everything up to the weights is in 64 bits.  The choice is a comparison of
// values that may lie next to each other: in 32 bits the order of a sum would
// decide it, and a token's experts would change with the batch that it came
// in.  In 64 the products of f32 values are exact and a sum of thousands is
// off by some 1e-15, so a split or tile shows in the ids only where two experts
// are that near each other (equal rows of W give equal sums, whatever the split).
#include <algorithm>

#include "okq_device.h"
#include "okq_internal.h"

namespace okq {

namespace {

typedef double f64x4 __attribute__((ext_vector_type(4)));

constexpr int kF32 = 0, kF16 = 1, kBF16 = 30;
constexpr int kRows = 16;  // token rows of a tile
// waves of a workgroup of NT expert tiles: a row each for the choice where a
// tile's registers leave room
constexpr int waves_of(int NT) { return NT == 1 ? 16 : 8; }
constexpr int kMostSlices = 4;

template <int kType>
struct WType {
  typedef float type;
};
template <>
struct WType<kF16> {
  typedef _Float16 type;
};
template <>
struct WType<kBF16> {
  typedef __bf16 type;
};

// Values k .. k + 3 of a row, one load each, or one for all four.
template <class T, bool kWide>
__device__ __forceinline__ void get4(const T *row, int k, T v[4]) {
  if constexpr (kWide) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    const T4 t = *reinterpret_cast<const T4 *>(row + k);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = t[e];
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = row[k + e];
  }
}

// A double's order as an unsigned integer's; NaN does not come here.
__device__ __forceinline__ uint64_t order_of(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v + 0.0);  // -0 as 0
  return u >> 63 ? ~u : u | (1ull << 63);
}
constexpr uint64_t kOrderNone = 0x000FFFFFFFFFFFFFull;  // order_of(-infinity)

__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
// the largest v of the wave's lanes
__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
  v = umax(v, dpp_row_u<0xB1>(v));
  v = umax(v, dpp_row_u<0x4E>(v));
  v = umax(v, dpp_row_u<0x141>(v));
  v = umax(v, dpp_row_u<0x140>(v));
  const uint32_t a = umax((uint32_t)__builtin_amdgcn_readlane((int)v, 0), (uint32_t)__builtin_amdgcn_readlane((int)v, 16));
  const uint32_t b = umax((uint32_t)__builtin_amdgcn_readlane((int)v, 32), (uint32_t)__builtin_amdgcn_readlane((int)v, 48));
  return umax(a, b);
}
// The index (below 2^31) of the largest key, the lowest among equals.
__device__ __forceinline__ int wave_best(uint64_t key, int index, uint64_t &best) {
  const uint32_t hi = (uint32_t)(key >> 32), top = wave_umax(hi);
  const uint32_t lo = hi == top ? (uint32_t)key : 0u, low = wave_umax(lo);
  best = (uint64_t)top << 32 | low;
  return 0x7fffffff - (int)wave_umax(key == best ? 0x7fffffffu - (uint32_t)index : 0u);
}
__device__ __forceinline__ double wave_fold(double v, bool sum) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const double o = __shfl_xor(v, d);
    v = sum ? v + o : __builtin_fmax(v, o);
  }
  return v;
}

__device__ __forceinline__ double lane_of(double v, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  return __builtin_bit_cast(double, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(u >> 32), lane) << 32 |
                                        (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, lane));
}

// The choice for one row by one wave: experts lane, lane + 64, ... of up to 64 N
// in registers.  z: its logits in LDS, left as what groups are chosen by.
template <int N>
__device__ __forceinline__ void choose(const RouteArgs &a, int row, double *z, int lane) {
  const int E = a.experts;
  double p[N], c[N], top = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int e = lane + 64 * i;
    p[i] = e < E ? z[e] : -INFINITY;
    if (a.logits && e < E) a.logits[(int64_t)row * E + e] = (float)p[i];
    nan = nan || __builtin_isnan(p[i]);
    top = __builtin_fmax(top, p[i]);
  }
  if (a.sigmoid) {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = 1.0 / (1.0 + exp(-p[i]));
  } else {
    top = wave_fold(top, false);
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      p[i] = exp(p[i] - top);
      sum += lane + 64 * i < E ? p[i] : 0.0;
    }
    sum = wave_fold(sum, true);
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] /= sum;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int e = lane + 64 * i;
    c[i] = p[i] + (a.choice_bias && e < E ? (double)a.choice_bias[e] : 0.0);
    nan = nan || (e < E && __builtin_isnan(c[i]));
    if (e >= E) c[i] = -INFINITY;
  }
  const int64_t at = (int64_t)row * a.top_k;
  if (__builtin_amdgcn_ballot_w64(nan) != 0) {
    if (lane < a.top_k) {
      a.ids[at + lane] = -1;
      a.weights[at + lane] = __builtin_nanf("");
    }
    return;
  }
  if (a.groups > 1) {
    // 2^share lanes a group, each with its best one or two of every so many;
    // they meet, then the group's place among the groups
    const int size = E / a.groups, share = 31 - __builtin_clz(64 / a.groups);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (lane + 64 * i < E) z[lane + 64 * i] = c[i];
    wave_sync();
    const int group = lane >> share;
    double one = -INFINITY, two = -INFINITY;
    if (group < a.groups)
      for (int i = lane & ((1 << share) - 1); i < size; i += 1 << share) {
        const double v = z[group * size + i];
        two = __builtin_fmax(two, __builtin_fmin(one, v));
        one = __builtin_fmax(one, v);
      }
    for (int d = 1; d < 1 << share; d *= 2) {
      const double o = __shfl_xor(one, d), t = __shfl_xor(two, d);
      two = __builtin_fmax(__builtin_fmin(one, o), __builtin_fmax(two, t));
      one = __builtin_fmax(one, o);
    }
    const double mine = a.group_best == 2 && size > 1 ? one + two : one;
    int place = 0;
    for (int g = 0; g < a.groups; ++g) {
      const double o = lane_of(mine, g << share);
      place += o > mine || (o == mine && g < group) ? 1 : 0;
    }
    const uint64_t stay = __builtin_amdgcn_ballot_w64(group < a.groups && place < a.top_groups);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (!((stay >> ((((lane + 64 * i) / size) << share) & 63)) & 1)) c[i] = -INFINITY;
  }
  // one expert after the other; lane j keeps the j-th
  uint64_t key[N];
#pragma unroll
  for (int i = 0; i < N; ++i) key[i] = order_of(c[i]);
  double sum = 0.0, kept = 0.0;
  int id = -1;
  for (int j = 0; j < a.top_k; ++j) {
    uint64_t best = kOrderNone;
    double score = 0.0;
    int index = 0x7ffffffe;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (key[i] > best) best = key[i], score = p[i], index = lane + 64 * i;
    uint64_t all;
    const int e = wave_best(best, index, all);
    if (all == kOrderNone) break;  // nothing left but -infinity
    const double chosen = lane_of(score, e & 63);
    sum += chosen;
    if (lane == j) kept = chosen, id = e;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (e == lane + 64 * i) key[i] = kOrderNone;
  }
  if (lane < a.top_k) {
    if (a.renormalise) kept = sum > 0.0 ? kept / sum : 0.0;
    a.ids[at + lane] = id;
    a.weights[at + lane] = (float)(kept * (double)a.scale);
  }
}

}  // namespace

// A tile's products go through v_mfma_f64_16x16x4: lane l holds the row l % 16
// of the tokens and of the experts, and of each 16 values of K the four from
// 4 (l / 16) on, one load of each for four products.  (The order of K inside
// a step is the same on both sides, so it does not matter which value is
// which.)  The f64 pipe takes 64 cycles a product, which bounds long batches.
//
// A workgroup's waves split K between them, and each takes NT expert tiles at
// once: every value is read and widened once a workgroup.  (A tile a wave, all
// waves over the same tokens' rows, read those from the L2 eight times: 4096 x
// 2048 with 128 experts 75 us, now 64 (BF16) and 56 (F32).)  They meet in LDS in pairs.
//
// What is left beside the products (65.5K of 138K cycles of that call): 19 us
// for launch, join, scores and choice, a row a wave at a time.  One row (of
// 2048, 128 experts): 11.7 us, the trip to memory, the join, the choice, one
// behind the other; 61 rows of 2560, 256 experts in groups: 22.
//
// whole: the workgroup has all experts of its 16 rows.  Otherwise it has NT
// tiles and one slice of K, and the rows' last workgroup adds the slices up in
// their order.
template <int kType, bool kWide, int NT>
__global__ __launch_bounds__(waves_of(NT) * 64) void route_kernel(RouteArgs a, RoutePlan plan, double *part,
                                                                  uint32_t *arrived) {
  typedef typename WType<kType>::type T;
  constexpr int kWaves = waves_of(NT);
  constexpr int kAhead = NT == 1 ? 4 : 8 / NT < 2 ? 2 : 8 / NT;  // chunks of 16 values in flight
  extern __shared__ __align__(16) double lds[];
  __shared__ f64x4 meet[kWaves / 2][NT][64];
  __shared__ int last;
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int E = a.experts, tiles = (E + 15) / 16, K = a.hidden;
  const int row0 = (int)blockIdx.x * kRows, rows = std::min(kRows, a.rows - row0);
  double *z = lds;  // [16][E]

  const int k_lo = plan.whole ? 0 : (int)blockIdx.z * plan.span, k_hi = plan.whole ? K : std::min(K, k_lo + plan.span);
  const int chunks = (k_hi - k_lo + 15) / 16;
  const int c_lo = chunks * wave / kWaves, c_hi = chunks * (wave + 1) / kWaves, c_full = std::min(c_hi, (k_hi - k_lo) / 16);
  const float *xr = a.x + (int64_t)std::min(row0 + n, a.rows - 1) * a.x_stride;
  for (int t0 = plan.whole ? 0 : (int)blockIdx.y * NT; t0 < (plan.whole ? tiles : (int)blockIdx.y * NT + 1); t0 += NT) {
    f64x4 acc[NT] = {};
    const T *wr[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) wr[t] = static_cast<const T *>(a.w) + (int64_t)std::min(16 * (t0 + t) + n, E - 1) * K;
    // past the last whole chunk it is loaded again, and dropped
    float xv[kAhead][4];
    T wv[kAhead][NT][4];
    auto load = [&](int i, int ch) {
      const int k = k_lo + 16 * std::min(ch, c_full - 1) + 4 * g;
      get4<float, kWide>(xr, k, xv[i]);
#pragma unroll
      for (int t = 0; t < NT; ++t) get4<T, kWide>(wr[t], k, wv[i][t]);
    };
    auto times = [&](int i) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int t = 0; t < NT; ++t)
          acc[t] = __builtin_amdgcn_mfma_f64_16x16x4f64((double)xv[i][e], (double)(float)wv[i][t][e], acc[t], 0, 0, 0);
    };
    if (c_lo < c_full) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) load(i, c_lo + i);
      int ch = c_lo;
      for (; ch + kAhead <= c_full; ch += kAhead) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          times(i);
          __builtin_amdgcn_sched_barrier(0);
          load(i, ch + i + kAhead);
        }
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (ch + i < c_full) times(i);
    }
    if (c_full < c_hi) {  // the last chunk of the row, zeros behind its end
      const int k = k_lo + 16 * c_full + 4 * g;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int at = std::min(k + e, K - 1);
        const float x = xr[at];
        xv[0][e] = k + e < K ? x : 0.0f;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const T w = wr[t][at];
          wv[0][t][e] = k + e < K ? w : (T)0.0f;
        }
      }
      times(0);
    }
    for (int half = kWaves / 2; half > 0; half /= 2) {
      if (wave >= half && wave < 2 * half)
#pragma unroll
        for (int t = 0; t < NT; ++t) meet[wave - half][t][lane] = acc[t];
      __syncthreads();
      if (wave < half)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t] += meet[wave][t][lane];
      __syncthreads();
    }
    if (wave == 0) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int e = 16 * (t0 + t) + n;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 4 * i + g;  // element i of lane l in D: row 4 i + l / 16, column l % 16
          if (r >= rows || e >= E) continue;
          if (plan.whole) {
            z[r * E + e] = acc[t][i] + (a.bias ? (double)a.bias[e] : 0.0);
          } else {
            double *to = part + (((int64_t)blockIdx.x * plan.slices + blockIdx.z) * kRows + r) * E + e;
            __hip_atomic_store(to, acc[t][i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          }
        }
      }
    }
  }
  if (!plan.whole) {
    // agent-scope stores, waited for before the count, as the loads behind it
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    const uint32_t all = gridDim.y * gridDim.z;
    uint32_t *mine = arrived + 32 * blockIdx.x;
    if (tid == 0) last = __hip_atomic_fetch_add(mine, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == all - 1;
    __syncthreads();
    if (!last) return;
    if (tid == 0) __hip_atomic_store(mine, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const double *from = part + (int64_t)blockIdx.x * plan.slices * kRows * E;
    for (int i = tid; i < rows * E; i += kWaves * 64) {
      double v[kMostSlices];  // requested together
#pragma unroll
      for (int o = 0; o < kMostSlices; ++o)
        v[o] = o < plan.slices ? __hip_atomic_load(from + (int64_t)o * kRows * E + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.0;
#pragma unroll
      for (int o = 1; o < kMostSlices; ++o) v[0] += v[o];
      z[i] = v[0] + (a.bias ? (double)a.bias[i % E] : 0.0);
    }
  }
  __syncthreads();
  for (int r = wave; r < rows; r += kWaves) {
    if (E <= 128) choose<2>(a, row0 + r, z + r * E, lane);
    else if (E <= 256) choose<4>(a, row0 + r, z + r * E, lane);
    else choose<8>(a, row0 + r, z + r * E, lane);
  }
}

RoutePlan route_plan(const RouteArgs &a, int cu_count) {
  RoutePlan p{};
  p.tiles = (a.rows + kRows - 1) / kRows;
  p.lds = (size_t)kRows * a.experts * sizeof(double);
  const int et = (a.experts + 15) / 16;
  // a workgroup per tile of rows once those fill half the card
  p.whole = p.tiles >= cu_count / 2;
  if (!p.whole) {
    // an expert tile a workgroup, slices of at least 1024 values (64 a wave),
    // about a workgroup a CU
    const int want = std::max(1, std::min(cu_count / (p.tiles * et), cu_count / 2 / p.tiles));
    const int most = std::max(1, a.hidden / 1024);
    const int s = std::min({want, most, kMostSlices});
    p.span = ((a.hidden + s - 1) / s + 15) / 16 * 16;
    p.slices = (a.hidden + p.span - 1) / p.span;
  }
  // the same for every call (tiles * slices is at most half of cu_count, or
  // cu_count / et), so that any first call makes room for a captured one
  p.part_bytes = (size_t)cu_count * kRows * kMaxExperts / 2 * sizeof(double);
  p.arrived_bytes = (size_t)cu_count / 2 * 128;
  return p;
}

template <int kType, bool kWide>
static void launch_route(const RouteArgs &a, const RoutePlan &p, double *part, uint32_t *arrived, hipStream_t s) {
  const int et = (a.experts + 15) / 16;
  const dim3 grid((unsigned)p.tiles, p.whole ? 1u : (unsigned)et, p.whole ? 1u : (unsigned)p.slices);
  const unsigned lds = (unsigned)p.lds;
  // a tile a workgroup of 1024 threads, unless the launch would have 2^32 of them (the last 16 of 2^26 rows)
  const bool one = !p.whole || (et == 1 && (uint64_t)p.tiles * (waves_of(1) * 64) <= UINT32_MAX);
  if (one) launch_timed(route_kernel<kType, kWide, 1>, grid, dim3(waves_of(1) * 64), lds, s, a, p, part, arrived);
  else if (et <= 4) launch_timed(route_kernel<kType, kWide, 4>, grid, dim3(waves_of(4) * 64), lds, s, a, p, part, arrived);
  else launch_timed(route_kernel<kType, kWide, 8>, grid, dim3(waves_of(8) * 64), lds, s, a, p, part, arrived);
}

hipError_t launch_route(const RouteArgs &a, const RoutePlan &p, void *part, void *arrived, hipStream_t s) {
  const bool wide = a.hidden % 4 == 0 && a.x_stride % 4 == 0 && reinterpret_cast<uintptr_t>(a.x) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(a.w) % 16 == 0;
  double *pt = static_cast<double *>(part);
  uint32_t *ar = static_cast<uint32_t *>(arrived);
#define OKQ_ROUTE(T_) wide ? launch_route<T_, true>(a, p, pt, ar, s) : launch_route<T_, false>(a, p, pt, ar, s)
  if (a.w_type == kF16) OKQ_ROUTE(kF16);
  else if (a.w_type == kBF16) OKQ_ROUTE(kBF16);
  else OKQ_ROUTE(kF32);
#undef OKQ_ROUTE
  return hipGetLastError();
}

}  // namespace okq
