// okq_residual.hip -- from one block of a layer to the next, in one pass over
// the rows: the norm behind the block, its gate and scale, the residual sum,
// and the norm ahead of the next block.
//
//   b = post ? branch * (1 / sqrt(sum branch^2 / hidden + eps)) * post : branch
//   y = residual_scale * x + branch_scale * gate * b
//   n = y * (1 / sqrt(sum y^2 / hidden + eps)) * pre
#include <algorithm>

#include "okq_device.h"
#include "okq_internal.h"

namespace okq {

namespace {

constexpr int kF16 = 1, kBF16 = 30;

// The workgroup's sum of v, the same in every thread: waves by DPP, then the
// waves' sums in every 16-lane row, in one fixed order.
__device__ __forceinline__ float block_sum(float v, float *red, int tid, int waves) {
  v = wave_sum(v);
  if (waves == 1) return v;
  if ((tid & 63) == 0) red[tid >> 6] = v;
  __syncthreads();
  const int i16 = tid & 15;
  float t = i16 < waves ? red[i16] : 0.0f;
  t += dpp_row_f<0xB1>(t);
  t += dpp_row_f<0x4E>(t);
  t += dpp_row_f<0x141>(t);
  t += dpp_row_f<0x140>(t);
  return t;
}

template <class T, int N>
struct Vec {
  typedef T type __attribute__((ext_vector_type(N)));
};
template <class T>
struct Vec<T, 1> {
  typedef T type;
};

// N values rounded to nearest even once, in the type of the next projections' rows
template <int N>
__device__ __forceinline__ void put(void *base, int type, int64_t at, const float *v) {
  if (type == kBF16 || type == kF16) {
    uint16_t h[N];
#pragma unroll
    for (int e = 0; e < N; ++e)
      h[e] = type == kBF16 ? __builtin_bit_cast(uint16_t, (__bf16)v[e]) : __builtin_bit_cast(uint16_t, (_Float16)v[e]);
    typename Vec<uint16_t, N>::type o;
    __builtin_memcpy(&o, h, sizeof o);
    *reinterpret_cast<typename Vec<uint16_t, N>::type *>(static_cast<uint16_t *>(base) + at) = o;
  } else {
    typename Vec<float, N>::type o;
    __builtin_memcpy(&o, v, sizeof o);
    *reinterpret_cast<typename Vec<float, N>::type *>(static_cast<float *>(base) + at) = o;
  }
}
template <int N>
__device__ __forceinline__ void get(const float *p, float *v) {
  typename Vec<float, N>::type o = *reinterpret_cast<const typename Vec<float, N>::type *>(p);
  __builtin_memcpy(v, &o, sizeof o);
}

}  // namespace

// A row stays in its workgroup's registers from the first load to the last
// store, V groups of N values a thread, and everything it needs is requested
// at once: one wait for memory, two joins in LDS.  Bounded by memory for many
// rows (4096 x 4096: 268 MB in 51 us called with new rows each time, 5.2 TB/s,
// the rate of a large copy; 39 us on the same ones), by that wait for few
// (1 x 4096: 2.9 us, 48 x 2560: 3.9).  Where rows are not 16-byte aligned a
// value a load: 1531 x 1111, gated, 8.3 us, 3.7 TB/s.
template <int N, int V>
__global__ __launch_bounds__(1024) void residual_norm_kernel(ResidualArgs a) {
  __shared__ float red[2][16];
  const int tid = (int)threadIdx.x, nt = (int)blockDim.x, waves = nt >> 6;
  const int64_t row = (int64_t)blockIdx.x;
  const int groups = (int)(a.hidden / N);
  const float *xr = a.x + row * a.x_stride, *br = a.branch + row * a.branch_stride;
  const float *gr = a.gate ? a.gate + row * a.gate_stride : nullptr;
  float x[V][N], b[V][N], g[V][N], w[V][N], p[V][N];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int i = tid + j * nt;
#pragma unroll
    for (int e = 0; e < N; ++e) x[j][e] = b[j][e] = w[j][e] = 0.0f, g[j][e] = p[j][e] = 1.0f;
    if (i < groups) {
      get<N>(br + (int64_t)i * N, b[j]);
      get<N>(xr + (int64_t)i * N, x[j]);
      if (a.post) get<N>(a.post + (int64_t)i * N, p[j]);
      if (gr) get<N>(gr + (int64_t)i * N, g[j]);
      if (a.pre) get<N>(a.pre + (int64_t)i * N, w[j]);
    }
  }
  float inv = 1.0f;
  if (a.post) {
    float ss = 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int e = 0; e < N; ++e) ss += b[j][e] * b[j][e];
    inv = 1.0f / sqrtf(block_sum(ss, red[0], tid, waves) / (float)a.hidden + a.eps);
  }
  float ss = 0.0f;
#pragma unroll
  for (int j = 0; j < V; ++j)
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float t = b[j][e] * inv * p[j][e];  // without a norm: times 1 twice, exactly
      const float y = a.residual_scale * x[j][e] + a.branch_scale * (g[j][e] * t);
      x[j][e] = y;
      // (past the row's end: zeros)
      ss += y * y;
    }
  if (a.sum) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int i = tid + j * nt;
      if (i < groups) put<N>(a.sum, 0, row * a.sum_stride + (int64_t)i * N, x[j]);
    }
  }
  if (!a.normed) return;
  inv = 1.0f / sqrtf(block_sum(ss, red[1], tid, waves) / (float)a.hidden + a.eps);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int i = tid + j * nt;
    float o[N];
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] = x[j][e] * inv * w[j][e];
    if (i < groups) put<N>(a.normed, a.normed_type, row * a.normed_stride + (int64_t)i * N, o);
  }
}

// Rows too long for registers: the branch is read twice, the sum formed twice
// (or read back where it was stored).
__global__ __launch_bounds__(1024) void residual_norm_long_kernel(ResidualArgs a) {
  __shared__ float red[2][16];
  const int tid = (int)threadIdx.x, nt = (int)blockDim.x, waves = nt >> 6;
  const int64_t row = (int64_t)blockIdx.x;
  const float *xr = a.x + row * a.x_stride, *br = a.branch + row * a.branch_stride;
  const float *gr = a.gate ? a.gate + row * a.gate_stride : nullptr;
  float unit = 1.0f;
  if (a.post) {
    float ss = 0.0f;
    for (int64_t i = tid; i < a.hidden; i += nt) ss += br[i] * br[i];
    unit = 1.0f / sqrtf(block_sum(ss, red[0], tid, waves) / (float)a.hidden + a.eps);
  }
  auto at = [&](int64_t i) {
    const float t = br[i] * unit * (a.post ? a.post[i] : 1.0f);
    return a.residual_scale * xr[i] + a.branch_scale * ((gr ? gr[i] : 1.0f) * t);
  };
  float ss = 0.0f;
  for (int64_t i = tid; i < a.hidden; i += nt) {
    const float y = at(i);
    ss += y * y;
    if (a.sum) a.sum[row * a.sum_stride + i] = y;
  }
  if (!a.normed) return;
  const float inv = 1.0f / sqrtf(block_sum(ss, red[1], tid, waves) / (float)a.hidden + a.eps);
  // a stored sum may have taken x's or branch's place; each thread reads its own stores
  for (int64_t i = tid; i < a.hidden; i += nt) {
    const float o = (a.sum ? a.sum[row * a.sum_stride + i] : at(i)) * inv * a.pre[i];
    put<1>(a.normed, a.normed_type, row * a.normed_stride + i, &o);
  }
}

hipError_t launch_residual_norm(const ResidualArgs &a, hipStream_t s) {
  if (a.rows <= 0) return hipSuccess;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.branch) |
                         reinterpret_cast<uintptr_t>(a.post) | reinterpret_cast<uintptr_t>(a.gate) |
                         reinterpret_cast<uintptr_t>(a.pre) | reinterpret_cast<uintptr_t>(a.sum) |
                         (reinterpret_cast<uintptr_t>(a.normed) << (a.normed_type ? 1 : 0));
  const int64_t strides = a.hidden | a.x_stride | a.branch_stride | a.gate_stride | (a.sum ? a.sum_stride : 0) |
                          (a.normed ? a.normed_stride : 0);
  const dim3 grid((unsigned)a.rows);
  const bool wide = bits % 16 == 0 && strides % 4 == 0 && a.hidden <= 4 * 4 * 1024;
  const int64_t groups = wide ? a.hidden / 4 : a.hidden;
  const unsigned nt = (unsigned)(std::min<int64_t>(groups, 1024) + 63) / 64 * 64;
  const int64_t per = (groups + nt - 1) / nt;
#define OKQ_NORM(N_, V_) launch_timed(residual_norm_kernel<N_, V_>, grid, dim3(nt), 0u, s, a)
  if (wide) {
    if (per == 1) OKQ_NORM(4, 1);
    else if (per == 2) OKQ_NORM(4, 2);
    else OKQ_NORM(4, 4);
  } else if (per <= 8) {
    if (per <= 2) OKQ_NORM(1, 2);
    else OKQ_NORM(1, 8);
  } else {
    launch_timed(residual_norm_long_kernel, grid, dim3(1024), 0u, s, a);
  }
#undef OKQ_NORM
  return hipGetLastError();
}

}  // namespace okq
