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
// off by some 1e-15, so no split or tile shows in the ids.
#include <algorithm>

#include "okq_device.h"
#include "okq_internal.h"

namespace okq {

namespace {

typedef double f64x4 __attribute__((ext_vector_type(4)));

constexpr int kF32 = 0, kF16 = 1, kBF16 = 30;
constexpr int kWaves = 8, kRows = 16;  // of a workgroup; token rows of a tile

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

// Values k .. k + 3 of a row of n (none past its end), one load each, or one
// for all four.
template <class T, bool kWide>
__device__ __forceinline__ void get4(const T *row, int k, int n, float v[4]) {
  if constexpr (kWide) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    T4 t = {};
    if (k < n) t = *reinterpret_cast<const T4 *>(row + k);  // n a multiple of 4
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (float)t[e];
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = k + e < n ? (float)row[k + e] : 0.0f;
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

// The choice for one row by one wave.  z: its logits in LDS, E of them, left
// as scores; c: as many values of scratch.
__device__ __forceinline__ void choose(const RouteArgs &a, int row, double *z, double *c, int lane) {
  const int E = a.experts;
  double top = -INFINITY;
  bool nan = false;
  for (int e = lane; e < E; e += 64) {
    if (a.logits) a.logits[(int64_t)row * E + e] = (float)z[e];
    nan = nan || __builtin_isnan(z[e]);
    top = __builtin_fmax(top, z[e]);
  }
  if (a.sigmoid) {
    for (int e = lane; e < E; e += 64) z[e] = 1.0 / (1.0 + exp(-z[e]));
  } else {
    top = wave_fold(top, false);
    double sum = 0.0;
    for (int e = lane; e < E; e += 64) {
      z[e] = exp(z[e] - top);
      sum += z[e];
    }
    sum = wave_fold(sum, true);
    for (int e = lane; e < E; e += 64) z[e] /= sum;
  }
  for (int e = lane; e < E; e += 64) {
    const double v = a.choice_bias ? z[e] + (double)a.choice_bias[e] : z[e];
    nan = nan || __builtin_isnan(v);
    c[e] = v;
  }
  const int64_t at = (int64_t)row * a.top_k;
  if (__builtin_amdgcn_ballot_w64(nan) != 0) {
    if (lane < a.top_k) {
      a.ids[at + lane] = -1;
      a.weights[at + lane] = __builtin_nanf("");
    }
    return;
  }
  wave_sync();
  if (a.groups > 1) {
    // lane g: group g's best one or two, then its place among the groups
    const int size = E / a.groups;
    double one = -INFINITY, two = -INFINITY;
    if (lane < a.groups)
      for (int i = 0; i < size; ++i) {
        const double v = c[lane * size + i];
        two = __builtin_fmax(two, __builtin_fmin(one, v));
        one = __builtin_fmax(one, v);
      }
    const uint64_t mine = order_of(a.group_best == 2 && size > 1 ? one + two : one);
    int place = 0;
    for (int g = 0; g < a.groups; ++g) {
      const uint64_t o = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(mine >> 32), g) << 32 |
                         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)mine, g);
      place += o > mine || (o == mine && g < lane) ? 1 : 0;
    }
    const uint64_t stay = __builtin_amdgcn_ballot_w64(lane < a.groups && place < a.top_groups);
    wave_sync();
    for (int e = lane; e < E; e += 64)
      if (!((stay >> (e / size)) & 1)) c[e] = -INFINITY;
    wave_sync();
  }
  // one expert after the other; lane j keeps the j-th
  double sum = 0.0, kept = 0.0;
  int id = -1;
  for (int j = 0; j < a.top_k; ++j) {
    uint64_t key = kOrderNone;
    int index = 0x7ffffffe;
    for (int e = lane; e < E; e += 64) {
      const uint64_t k = order_of(c[e]);
      if (k > key) key = k, index = e;
    }
    uint64_t best;
    const int e = wave_best(key, index, best);
    if (best == kOrderNone) break;  // nothing left but -infinity
    const double p = z[e];
    sum += p;
    if (lane == j) kept = p, id = e;
    if (lane == (e & 63)) c[e] = -INFINITY;
    wave_sync();
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
// which.)  The f64 pipe takes 64 cycles a product, which bounds long batches:
// 2048 flops a conversion of two values, so nothing is staged.
//
// whole: the workgroup has all experts of its 16 rows, wt waves side by side
// over the expert tiles and kWaves / wt over K.  Otherwise it has one expert
// tile and one slice of K, its waves split that, and the tile's last
// workgroup adds the slices up in their order.
template <int kType, bool kWide>
__global__ __launch_bounds__(kWaves * 64) void route_kernel(RouteArgs a, RoutePlan plan, double *part, uint32_t *arrived) {
  typedef typename WType<kType>::type T;
  extern __shared__ __align__(16) double lds[];
  __shared__ double meet[kWaves][256];
  __shared__ int last;
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int E = a.experts, tiles = (E + 15) / 16, K = a.hidden;
  const int row0 = (int)blockIdx.x * kRows;
  double *z = lds, *c = lds + kRows * E;  // [16][E]

  const int wt = plan.whole ? (tiles >= 8 ? 8 : tiles > 2 ? 4 : tiles) : 1, wk = kWaves / wt;
  const int ks = wave / wt;  // this wave's share of K
  const int k_lo = plan.whole ? 0 : (int)blockIdx.z * plan.span, k_hi = plan.whole ? K : std::min(K, k_lo + plan.span);
  const int chunks = (k_hi - k_lo + 15) / 16;
  const int c_lo = chunks * ks / wk, c_hi = chunks * (ks + 1) / wk;
  const float *xr = a.x + (int64_t)std::min(row0 + n, a.rows - 1) * a.x_stride;
  // element i of lane l in D: row 4 i + l / 16, column l % 16
  for (int t0 = plan.whole ? 0 : (int)blockIdx.y; t0 < (plan.whole ? tiles : (int)blockIdx.y + 1); t0 += wt) {
    const int t = t0 + wave % wt;
    const T *wr = static_cast<const T *>(a.w) + (int64_t)std::min(16 * t + n, E - 1) * K;
    f64x4 acc = {0.0, 0.0, 0.0, 0.0};
    if (t < tiles) {
#pragma unroll 4
      for (int ch = c_lo; ch < c_hi; ++ch) {
        float xv[4], wv[4];
        const int k = k_lo + 16 * ch + 4 * g;
        get4<float, kWide>(xr, k, k_hi, xv);
        get4<T, kWide>(wr, k, k_hi, wv);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)xv[e], (double)wv[e], acc, 0, 0, 0);
      }
    }
    if (wk > 1) {  // the waves of one expert tile meet, in their order
#pragma unroll
      for (int i = 0; i < 4; ++i) meet[wave][64 * i + lane] = acc[i];
      __syncthreads();
      if (ks == 0)
        for (int o = 1; o < wk; ++o)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[i] += meet[wave + o * wt][64 * i + lane];
      __syncthreads();
    }
    if (ks == 0 && 16 * t + n < E) {
      const int e = 16 * t + n;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 4 * i + g;
        if (plan.whole) {
          z[r * E + e] = acc[i] + (a.bias ? (double)a.bias[e] : 0.0);
        } else {
          double *to = part + (((int64_t)blockIdx.x * plan.slices + blockIdx.z) * kRows + r) * E + e;
          __hip_atomic_store(to, acc[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
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
    for (int i = tid; i < kRows * E; i += kWaves * 64) {
      double v = a.bias ? (double)a.bias[i % E] : 0.0;
      double s = 0.0;
      for (int o = 0; o < plan.slices; ++o)
        s += __hip_atomic_load(from + (int64_t)o * kRows * E + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      z[i] = s + v;
    }
  }
  __syncthreads();
  for (int r = wave; r < kRows && row0 + r < a.rows; r += kWaves) choose(a, row0 + r, z + r * E, c + r * E, lane);
}

RoutePlan route_plan(const RouteArgs &a, int cu_count) {
  RoutePlan p{};
  p.tiles = (a.rows + kRows - 1) / kRows;
  p.lds = (size_t)2 * kRows * a.experts * sizeof(double);
  const int et = (a.experts + 15) / 16;
  // a workgroup per tile of rows once those fill half the card
  p.whole = p.tiles >= cu_count / 2;
  if (!p.whole) {
    // slices of at least 512 values (64 a wave), about two workgroups a CU
    const int want = std::max(1, 2 * cu_count / (p.tiles * et));
    const int most = std::max(1, a.hidden / 512);
    const int s = std::min({want, most, 16});
    p.span = ((a.hidden + s - 1) / s + 15) / 16 * 16;
    p.slices = (a.hidden + p.span - 1) / p.span;
    p.part_bytes = (size_t)p.tiles * p.slices * kRows * a.experts * sizeof(double);
    p.arrived_bytes = (size_t)p.tiles * 128;
  }
  return p;
}

hipError_t launch_route(const RouteArgs &a, const RoutePlan &p, void *part, void *arrived, hipStream_t s) {
  const int et = (a.experts + 15) / 16;
  const dim3 grid((unsigned)p.tiles, p.whole ? 1u : (unsigned)et, p.whole ? 1u : (unsigned)p.slices);
  const bool wide = a.hidden % 4 == 0 && a.x_stride % 4 == 0 && reinterpret_cast<uintptr_t>(a.x) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(a.w) % 16 == 0;
  double *pt = static_cast<double *>(part);
  uint32_t *ar = static_cast<uint32_t *>(arrived);
#define OKQ_ROUTE(T_)                                                                                          \
  {                                                                                                            \
    if (wide) launch_timed(route_kernel<T_, true>, grid, dim3(kWaves * 64), (unsigned)p.lds, s, a, p, pt, ar);  \
    else launch_timed(route_kernel<T_, false>, grid, dim3(kWaves * 64), (unsigned)p.lds, s, a, p, pt, ar);      \
  }
  if (a.w_type == kF16) OKQ_ROUTE(kF16)
  else if (a.w_type == kBF16) OKQ_ROUTE(kBF16)
  else OKQ_ROUTE(kF32)
#undef OKQ_ROUTE
  return hipGetLastError();
}

}  // namespace okq
