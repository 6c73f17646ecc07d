// okq_attention.hip -- attention of one new token of each sequence over a
// paged key-value cache:
//   out = sum_t p_t V[t] / sum_t p_t,  p_t = exp(s_t - max s),
//   s_t = scale * q . K[t]  (softcap * tanh(s_t / softcap) where capped),
// over the visible tokens, in one pass with the running maximum and sum.
#include "okq_device.h"
#include "okq_internal.h"

namespace okq {

namespace {

constexpr int kF32 = 0, kF16 = 1;

// Value i of a cached row.
__device__ __forceinline__ float cached(int type, const uint8_t *row, int i) {
  if (type == kF32) return reinterpret_cast<const float *>(row)[i];
  if (type == kQ8_0) return deq_elem(kQ8_0, row, (uint32_t)i);
  const uint16_t b = reinterpret_cast<const uint16_t *>(row)[i];
  return type == kF16 ? f16_bits_hw(b) : as_f32((uint32_t)b << 16);
}

}  // namespace

// One workgroup per sequence and query head; its four waves take the tokens
// in turn, a wave's lanes the row's values.  Any head_dim up to kMaxHeadDim,
// any alignment, every cache type.
__global__ __launch_bounds__(256) void attention_rows_kernel(AttnArgs a) {
  constexpr int kV = kMaxHeadDim / 64;
  __shared__ float lds[4][kMaxHeadDim + 2];
  const int wave = (int)threadIdx.x >> 6, lane = (int)threadIdx.x & 63;
  const int D = a.cache.head_dim, pt = a.cache.page_tokens;
  const int seq = (int)(blockIdx.x / (unsigned)a.q_heads), h = (int)(blockIdx.x % (unsigned)a.q_heads);
  const int64_t kv_at = (int64_t)(h / a.group) * a.cache.head_stride;
  float q[kV], o[kV];
  for (int j = 0; j < kV; ++j) {
    const int i = lane + 64 * j;
    q[j] = i < D ? a.q[seq * a.q_stride + (int64_t)h * D + i] : 0.0f;
    o[j] = 0.0f;
  }
  int len = a.lengths[seq];
  len = len < a.max_len ? len : a.max_len;
  const int lo = a.window && len > a.window ? len - a.window : 0;
  float m = -INFINITY, l = 0.0f;
  for (int t = lo + wave; t < len; t += 4) {
    const int page = a.table[(int64_t)seq * a.table_width + t / pt];
    if ((unsigned)page >= (unsigned)a.cache.n_pages) continue;
    const int64_t at = page * a.cache.page_stride + kv_at + t % pt * a.cache.token_stride;
    float dot = 0.0f;
    for (int j = 0; j < kV; ++j) {
      const int i = lane + 64 * j;
      if (i < D) dot += q[j] * cached(a.cache.type, a.cache.k + at, i);
    }
    float s = wave_sum(dot) * a.scale;
    if (a.softcap > 0.0f) s = a.softcap * tanhf(s / a.softcap);
    const float top = fmaxf(m, s), base = top == -INFINITY ? 0.0f : top;
    const float keep = expf(m - base), p = expf(s - base);
    m = top;
    l = l * keep + p;
    for (int j = 0; j < kV; ++j) {
      const int i = lane + 64 * j;
      if (i < D) o[j] = o[j] * keep + p * cached(a.cache.type, a.cache.v + at, i);
    }
  }
  for (int j = 0; j < kV; ++j)
    if (lane + 64 * j < D) lds[wave][lane + 64 * j] = o[j];
  if (lane == 0) {
    lds[wave][kMaxHeadDim] = m;
    lds[wave][kMaxHeadDim + 1] = l;
  }
  __syncthreads();
  float top = -INFINITY, sum = 0.0f;
  for (int w = 0; w < 4; ++w) top = fmaxf(top, lds[w][kMaxHeadDim]);
  const float base = top == -INFINITY ? 0.0f : top;
  for (int w = 0; w < 4; ++w) sum += lds[w][kMaxHeadDim + 1] * expf(lds[w][kMaxHeadDim] - base);
  for (int i = (int)threadIdx.x; i < D; i += 256) {
    float v = 0.0f;
    for (int w = 0; w < 4; ++w) v += lds[w][i] * expf(lds[w][kMaxHeadDim] - base);
    a.out[seq * a.out_stride + (int64_t)h * D + i] = sum == 0.0f ? 0.0f : v / sum;
  }
  if (a.lse && threadIdx.x == 0) a.lse[(int64_t)seq * a.q_heads + h] = top == INFINITY ? top : base + logf(sum);
}

hipError_t launch_attention(const AttnArgs &a, hipStream_t s) {
  launch_timed(attention_rows_kernel, dim3((unsigned)(a.seqs * a.q_heads)), dim3(256), 0u, s, a);
  return hipGetLastError();
}

}  // namespace okq
