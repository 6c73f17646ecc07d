// okq_rope.hip -- RMS norm of query and key heads, the position rotation, and
// the store of keys and values into a paged cache, in one pass.
//
//   y = x * (1 / sqrt(sum x^2 / D + eps)) * w           (per head, optional)
//   (y[a], y[b]) -> (y[a] cos t - y[b] sin t, y[b] cos t + y[a] sin t),
//   t = position * inv_freq[i], (a, b) = (2i, 2i+1) or (i, i + rotary/2)
#include "okq_device.h"
#include "okq_internal.h"

namespace okq {

namespace {

constexpr int kF32 = 0, kF16 = 1, kBF16 = 30;

// cos and sin of pos * freq.  The angle and its remainder by pi/2 are formed
// in 64 bits (in 32 a position of 10^5 would lose the angle's last 17 bits);
// what is left, at most pi/4, is rounded to f32 once, and Taylor's series to
// a^9 (sine) and a^10 (cosine) are off by less than 2e-9 there.
__device__ __forceinline__ void angle_cs(int pos, float freq, float &c, float &s) {
  const double t = (double)pos * (double)freq;
  const double n = __builtin_rint(t * 0.63661977236758134308);
  // pi/2 in two parts: n of up to 2^33 leaves the remainder exact to 2^-40
  const double r = __builtin_fma(-n, 6.123233995736766036e-17, __builtin_fma(-n, 1.5707963267948965580, t));
  const int quad = (int)(n - 4.0 * __builtin_floor(n * 0.25));
  const float a = (float)r, a2 = a * a;
  float p = __builtin_fmaf(a2, 2.7557319e-06f, -1.9841270e-04f);
  p = __builtin_fmaf(a2, p, 8.3333333e-03f);
  p = __builtin_fmaf(a2, p, -1.6666667e-01f);
  const float sn = __builtin_fmaf(a * a2, p, a);
  p = __builtin_fmaf(a2, -2.7557319e-07f, 2.4801587e-05f);
  p = __builtin_fmaf(a2, p, -1.3888889e-03f);
  p = __builtin_fmaf(a2, p, 4.1666667e-02f);
  p = __builtin_fmaf(a2, p, -0.5f);
  const float cs = __builtin_fmaf(a2, p, 1.0f);
  const float x = quad & 1 ? sn : cs, y = quad & 1 ? cs : sn;
  c = quad == 1 || quad == 2 ? -x : x;
  s = quad >= 2 ? -y : y;
}

__device__ __forceinline__ uint16_t bf16_bits(float f) { return __builtin_bit_cast(uint16_t, (__bf16)f); }
__device__ __forceinline__ uint16_t f16_bits(float f) { return __builtin_bit_cast(uint16_t, (_Float16)f); }

}  // namespace

// One wave per row (a head of a token): the row passes through LDS, any
// head_dim up to kMaxHeadDim, any alignment, every cache type.
__global__ __launch_bounds__(256) void rope_rows_kernel(RopeArgs a) {
  __shared__ float lds[4][kMaxHeadDim];
  const int wave = (int)threadIdx.x >> 6, lane = (int)threadIdx.x & 63;
  const int D = a.head_dim, hkv = a.kv_heads;
  const int per_token = a.q_heads + hkv * (a.cache.k ? 2 : 1);
  const int64_t row = (int64_t)blockIdx.x * 4 + wave;
  if (row >= (int64_t)a.tokens * per_token) return;  // a wave's LDS is its own: no barrier below
  float *y = lds[wave];
  const int64_t tok = row / per_token;
  const int h = (int)(row % per_token);
  const int kind = h < a.q_heads ? 0 : h < a.q_heads + hkv ? 1 : 2;
  const int head = kind == 0 ? h : kind == 1 ? h - a.q_heads : h - a.q_heads - hkv;
  const float *x = (kind == 0 ? a.q + tok * a.q_stride : kind == 1 ? a.k + tok * a.k_stride : a.v + tok * a.v_stride) +
                   (int64_t)head * D;
  const float *w = kind == 0 ? a.q_norm : kind == 1 ? a.k_norm : nullptr;
  float ss = 0.0f;
  for (int i = lane; i < D; i += 64) {
    const float v = x[i];
    y[i] = v;
    ss += v * v;
  }
  wave_sync();
  if (w) {
    const float inv = 1.0f / sqrtf(wave_sum(ss) / (float)D + a.eps);
    for (int i = lane; i < D; i += 64) y[i] = y[i] * inv * w[i];
    wave_sync();
  }
  if (kind < 2) {
    const int half = a.rotary / 2;
    const int pos = a.rotary ? a.positions[tok] : 0;
    for (int i = lane; i < half; i += 64) {
      float c, s;
      angle_cs(pos, a.inv_freq[i], c, s);
      const int ia = a.interleaved ? 2 * i : i, ib = a.interleaved ? 2 * i + 1 : i + half;
      const float u = y[ia], v = y[ib];
      y[ia] = u * c - v * s;
      y[ib] = v * c + u * s;
    }
    wave_sync();
  }
  float *dense = kind == 0   ? a.q_out + tok * a.q_out_stride + (int64_t)head * D
                 : kind == 1 && a.k_out ? a.k_out + tok * a.k_out_stride + (int64_t)head * D
                                        : nullptr;
  if (dense)
    for (int i = lane; i < D; i += 64) dense[i] = y[i];
  if (kind == 0 || !a.cache.k) return;
  const int64_t slot = a.slots[tok];
  const int pt = a.cache.page_tokens;
  if (slot < 0 || slot >= (int64_t)a.cache.n_pages * pt) return;
  uint8_t *dst = (kind == 1 ? a.cache.k : a.cache.v) + slot / pt * a.cache.page_stride +
                 (int64_t)head * a.cache.head_stride + slot % pt * a.cache.token_stride;
  if (a.cache.type == kF32) {
    for (int i = lane; i < D; i += 64) reinterpret_cast<float *>(dst)[i] = y[i];
  } else if (a.cache.type == kQ8_0) {
    // okq_quantize's rounding: d = max / 127 kept as f16, codes from 1 / d in f32
    for (int b = lane; b < D / 32; b += 64) {
      float m = 0.0f;
      for (int j = 0; j < 32; ++j) m = fabsf(y[32 * b + j]) > m ? fabsf(y[32 * b + j]) : m;
      const float d = __fdiv_rn(m, 127.0f), id = d != 0.0f ? __fdiv_rn(1.0f, d) : 0.0f;
      uint8_t *blk = dst + b * kQ8Bytes;
      *reinterpret_cast<uint16_t *>(blk) = f16_bits(d);
      for (int j = 0; j < 32; ++j) {
        const int c = (int)__builtin_rintf(__fmul_rn(y[32 * b + j], id));
        blk[2 + j] = (uint8_t)(int8_t)(c < -127 ? -127 : c > 127 ? 127 : c);
      }
    }
  } else {
    for (int i = lane; i < D; i += 64)
      reinterpret_cast<uint16_t *>(dst)[i] = a.cache.type == kF16 ? f16_bits(y[i]) : bf16_bits(y[i]);
  }
}

hipError_t launch_rope(const RopeArgs &a, int, hipStream_t s) {
  const int64_t rows = (int64_t)a.tokens * (a.q_heads + a.kv_heads * (a.cache.k ? 2 : 1));
  launch_timed(rope_rows_kernel, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0u, s, a);
  return hipGetLastError();
}

}  // namespace okq
