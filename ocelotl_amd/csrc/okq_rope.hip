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

// Rows that rope_kernel's lanes do not divide (head_dim or rotary no multiple
// of eight, Q8_0 blocks across the halves of a rotation): one wave a row, which
// passes through LDS.  Up to some dozens of tokens it is as fast as the host's
// call (48 tokens: 4.7 us; into Q8_0 6.2); a prompt it takes four to six times
// its bytes' time for, as a row's angles are formed for it alone and a Q8_0
// block is one lane's (4096 tokens of 32 + 8 heads: head_dim 100, BF16 112 us,
// 144 MB; 96 into Q8_0 137 us, 133 MB; rope_kernel takes 28 for 96 into BF16).
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


// ---- eight values a lane --------------------------------------------------------
//
// A head's row in registers: a lane holds four rotation pairs (or eight values
// past the rotation), so every pair and its cosine and sine are one lane's,
// kLanes lanes (a power of two, at least head_dim / 8) a row, 64 / kLanes
// heads of one token a pass of the wave.  The angles, 64-bit arithmetic, are
// formed once for all of a wave's passes.  What bounds it is memory: a row is
// read and written once, in 16-byte pieces, kAhead passes requested at a time
// (4096 tokens of 32 + 8 heads of 128, 184 MB: 35 us, 5.3 TB/s, with two;
// four, and outputs through the caches, 46).  Into Q8_0, 177 MB, the same rows
// take 34.6 us turned by halves, 37.2 in neighbouring pairs.

typedef float f32x4 __attribute__((ext_vector_type(4)));

namespace {

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

// Sum over the kLanes lanes of a row, in every one of them, in one fixed order.
template <int kLanes>
__device__ __forceinline__ float row_sum(float v) {
  v += dpp_row_f<0xB1>(v);
  v += dpp_row_f<0x4E>(v);
  if (kLanes >= 8) v += dpp_row_f<0x141>(v);
  if (kLanes >= 16) v += dpp_row_f<0x140>(v);
  if (kLanes >= 32) {
    const auto a = __builtin_amdgcn_permlane16_swap(as_u32(v), as_u32(v), false, false);
    v = as_f32(a[0]) + as_f32(a[1]);
  }
  if (kLanes >= 64) {
    const auto a = __builtin_amdgcn_permlane32_swap(as_u32(v), as_u32(v), false, false);
    v = as_f32(a[0]) + as_f32(a[1]);
  }
  return v;
}

__device__ __forceinline__ float abs_max(f32x4 v) {
  return fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
}
// Four codes of a block whose largest value is m, and the block's scale.
__device__ __forceinline__ uint32_t codes_q8(f32x4 v, float m, float &d) {
  d = __fdiv_rn(m, 127.0f);
  const float id = d != 0.0f ? __fdiv_rn(1.0f, d) : 0.0f;
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int c = (int)__builtin_rintf(__fmul_rn(v[e], id));
    w |= (uint32_t)((c < -127 ? -127 : c > 127 ? 127 : c) & 0xff) << (8 * e);
  }
  return w;
}

// Stored past the caches, which the rows to come fill.
__device__ __forceinline__ void store_past(float *p, f32x4 v) {
  typedef f32x4 f32x4_4 __attribute__((aligned(4)));
  __builtin_nontemporal_store(v, reinterpret_cast<f32x4_4 *>(p));
}

constexpr int kAhead = 2;

}  // namespace

template <int kLanes>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs a, int shares, int passes) {
  constexpr int kHeads = 64 / kLanes;
  const int wave = (int)(blockIdx.x * 4 + (threadIdx.x >> 6)), lane = (int)threadIdx.x & 63;
  if (wave >= a.tokens * shares) return;
  const int tok = __builtin_amdgcn_readfirstlane(wave / shares), share = wave - tok * shares;
  const int D = a.head_dim, total = a.q_heads + a.kv_heads * (a.cache.k ? 2 : 1);
  const int u = lane & (kLanes - 1), hp = lane / kLanes;
  const bool live = 8 * u < D, turns = 8 * u < a.rotary, split = turns && !a.interleaved;
  const int p0 = split ? 4 * u : 8 * u, p1 = split ? a.rotary / 2 + 4 * u : 8 * u + 4;

  // requested together: the first rows, the norms' weights, the position
  const int h0 = share * passes * kHeads + hp, h_end = min(total, (share + 1) * passes * kHeads);
  f32x4 lo[kAhead], hi[kAhead];
  auto request = [&](int h, f32x4 &x, f32x4 &y) {
    x = y = f32x4{0, 0, 0, 0};
    if (h >= h_end || !live) return;
    const float *row = h < a.q_heads                ? a.q + tok * a.q_stride + (int64_t)h * D
                       : h < a.q_heads + a.kv_heads ? a.k + tok * a.k_stride + (int64_t)(h - a.q_heads) * D
                                                    : a.v + tok * a.v_stride + (int64_t)(h - a.q_heads - a.kv_heads) * D;
    x = load_any<f32x4>(row + p0);
    y = load_any<f32x4>(row + p1);
  };
#pragma unroll
  for (int j = 0; j < kAhead; ++j) request(h0 + j * kHeads, lo[j], hi[j]);
  const int pos = a.rotary ? a.positions[tok] : 0;
  f32x4 freq = {0, 0, 0, 0}, qw0 = {1, 1, 1, 1}, qw1 = qw0, kw0 = qw0, kw1 = qw0;
  if (turns) freq = load_any<f32x4>(a.inv_freq + 4 * u);
  if (a.q_norm && live) qw0 = load_any<f32x4>(a.q_norm + p0), qw1 = load_any<f32x4>(a.q_norm + p1);
  if (a.k_norm && live) kw0 = load_any<f32x4>(a.k_norm + p0), kw1 = load_any<f32x4>(a.k_norm + p1);
  uint8_t *krow = nullptr, *vrow = nullptr;  // the token's rows of head 0
  if (a.cache.k) {
    const int64_t slot = a.slots[tok];
    const int pt = a.cache.page_tokens;
    if (slot >= 0 && slot < (int64_t)a.cache.n_pages * pt) {
      const int64_t page = slot <= INT32_MAX ? (int64_t)((uint32_t)slot / (uint32_t)pt) : slot / pt;
      const int64_t at = page * a.cache.page_stride + (slot - page * pt) * a.cache.token_stride;
      krow = a.cache.k + at;
      vrow = a.cache.v + at;
    }
  }
  float cs[4], sn[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) angle_cs(pos, freq[e], cs[e], sn[e]);

  for (int h1 = h0; h1 - hp < h_end; h1 += kAhead * kHeads) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int h = h1 + j * kHeads;
      if (h - hp >= h_end) break;
      f32x4 x = lo[j], y = hi[j];
      request(h + kAhead * kHeads, lo[j], hi[j]);
      const bool is_q = h < a.q_heads, is_v = h >= a.q_heads + a.kv_heads;
      const bool norm = (is_q ? a.q_norm : a.k_norm) && !is_v;
      if (a.q_norm || a.k_norm) {
        const float ss = row_sum<kLanes>((x[0] * x[0] + x[1] * x[1]) + (x[2] * x[2] + x[3] * x[3]) +
                                         ((y[0] * y[0] + y[1] * y[1]) + (y[2] * y[2] + y[3] * y[3])));
        const float inv = 1.0f / sqrtf(ss / (float)D + a.eps);
        if (norm) {
          x = x * inv * (is_q ? qw0 : kw0);
          y = y * inv * (is_q ? qw1 : kw1);
        }
      }
      if (turns && !is_v) {
        if (split) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float s = x[e], t = y[e];
            x[e] = s * cs[e] - t * sn[e];
            y[e] = t * cs[e] + s * sn[e];
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            float s = x[e], t = x[e + 1];
            x[e] = s * cs[e / 2] - t * sn[e / 2];
            x[e + 1] = t * cs[e / 2] + s * sn[e / 2];
            s = y[e], t = y[e + 1];
            y[e] = s * cs[2 + e / 2] - t * sn[2 + e / 2];
            y[e + 1] = t * cs[2 + e / 2] + s * sn[2 + e / 2];
          }
        }
      }
      const int kv = is_q ? 0 : is_v ? h - a.q_heads - a.kv_heads : h - a.q_heads;
      if (a.cache.type == kQ8_0 && a.cache.k) {
        // a block's 32 values are four lanes' eight, or, turned by halves
        // (rotary / 2 is a multiple of 32 here), eight lanes' four
        float m0 = abs_max(x), m1 = abs_max(y);
        const float both = fmaxf(m0, m1);
        float four = fmaxf(both, dpp_row_f<0xB1>(both));
        four = fmaxf(four, dpp_row_f<0x4E>(four));
        m0 = fmaxf(m0, dpp_row_f<0xB1>(m0));
        m0 = fmaxf(m0, dpp_row_f<0x4E>(m0));
        m0 = fmaxf(m0, dpp_row_f<0x141>(m0));
        m1 = fmaxf(m1, dpp_row_f<0xB1>(m1));
        m1 = fmaxf(m1, dpp_row_f<0x4E>(m1));
        m1 = fmaxf(m1, dpp_row_f<0x141>(m1));
        uint8_t *dst = is_v ? vrow : krow;
        if (h < h_end && live && !is_q && dst) {
          dst += (int64_t)kv * a.cache.head_stride;
          float d0, d1;
          const uint32_t c0 = codes_q8(x, split ? m0 : four, d0), c1 = codes_q8(y, split ? m1 : four, d1);
          uint8_t *b0 = dst + p0 / 32 * kQ8Bytes, *b1 = dst + p1 / 32 * kQ8Bytes;
          store_any(b0 + 2 + p0 % 32, c0);
          store_any(b1 + 2 + p1 % 32, c1);
          if (p0 % 32 == 0) store_any(b0, f16_bits(d0));
          if (split && p1 % 32 == 0) store_any(b1, f16_bits(d1));
        }
      }
      if (h >= h_end || !live) continue;
      float *dense = is_q                ? a.q_out + tok * a.q_out_stride + (int64_t)h * D
                     : a.k_out && !is_v ? a.k_out + tok * a.k_out_stride + (int64_t)kv * D
                                        : nullptr;
      if (dense) {
        store_past(dense + p0, x);
        store_past(dense + p1, y);
      }
      uint8_t *dst = is_v ? vrow : krow;
      if (is_q || !dst || a.cache.type == kQ8_0) continue;
      dst += (int64_t)kv * a.cache.head_stride;
      if (a.cache.type == kF32) {
        store_any(dst + 4 * p0, x);
        store_any(dst + 4 * p1, y);
      } else {
        typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
        auto pack = [&](float s, float t) {
          return a.cache.type == kF16 ? (uint32_t)f16_bits(s) | (uint32_t)f16_bits(t) << 16
                                      : (uint32_t)bf16_bits(s) | (uint32_t)bf16_bits(t) << 16;
        };
        store_any(dst + 2 * p0, u32x2{pack(x[0], x[1]), pack(x[2], x[3])});
        store_any(dst + 2 * p1, u32x2{pack(y[0], y[1]), pack(y[2], y[3])});
      }
    }
  }
}

hipError_t launch_rope(const RopeArgs &a, int cu_count, hipStream_t s) {
  const int heads = a.q_heads + a.kv_heads * (a.cache.k ? 2 : 1), D = a.head_dim;
  // whole lanes of eight values; Q8_0 blocks that lanes share evenly
  if (D % 8 == 0 && a.rotary % 8 == 0 && (!a.cache.k || a.cache.type != kQ8_0 || a.interleaved || a.rotary % 64 == 0)) {
    const int lanes = D <= 64 ? 8 : D <= 128 ? 16 : D <= 256 ? 32 : 64, at_once = 64 / lanes;
    const int all = (heads + at_once - 1) / at_once;  // a token's passes
    // A wave takes several passes of a token, sharing its angles, once there
    // are waves enough: 32 a CU, rounded down (2048 tokens of 32 + 8 heads of
    // 128: 16.8 us so, 18.4 with 64; 2598 of 28 + 7 of 96: 17.3, 19.2)
    const int64_t some = 32 * (int64_t)cu_count, want = ((int64_t)a.tokens * all + some - 1) / some;
    const int passes = (int)(want < 1 ? 1 : want > all ? all : want), shares = (all + passes - 1) / passes;
    const dim3 grid((unsigned)(((int64_t)a.tokens * shares + 3) / 4));
    if (lanes == 8) launch_timed(rope_kernel<8>, grid, dim3(256), 0u, s, a, shares, passes);
    else if (lanes == 16) launch_timed(rope_kernel<16>, grid, dim3(256), 0u, s, a, shares, passes);
    else if (lanes == 32) launch_timed(rope_kernel<32>, grid, dim3(256), 0u, s, a, shares, passes);
    else launch_timed(rope_kernel<64>, grid, dim3(256), 0u, s, a, shares, passes);
    return hipGetLastError();
  }
  const int64_t rows = (int64_t)a.tokens * heads;
  launch_timed(rope_rows_kernel, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0u, s, a);
  return hipGetLastError();
}

}  // namespace okq
