// okq_moe.hip -- the gated MLP of every token's experts over stacked GGUF
// tensors [experts][rows][blocks], and the weighted sum of their results:
//
//   out[t] = sum_j weight[t, j] * down_e(silu(gate_e(x[t])) * up_e(x[t])),  e = ids[t, j]
//
// A pair is a token and one of its experts, t * top_k + j.  Two products over
// the pairs, expert by expert, and a sum over each token's: gate and up
// together, whose waves hold both sums of a column and leave silu(gate) * up;
// down, which leaves every pair's weighted row; the sum in the order of j.
//
// Numerics.  A row's activations are scaled by a power of two (for every 256 of
// them, in tiles for the row) and split into two fp16 planes, x = hi + lo to
// 2^-22; the weights' integer parts are exact in fp16 (okq_mfma.h), so every
// product is exact and only f32 sums round.  A row that holds an infinity or a
// NaN gets a NaN scale.
#include <algorithm>

#include "okq_device.h"
#include "okq_internal.h"
#include "okq_mfma.h"

namespace okq {

namespace {

constexpr int kWaves = 8;
constexpr int kPassPairs = 65536;  // at most, of a pass: they count in 16 bits
constexpr int kFewPairs = 64;      // not sorted: a lane each
constexpr int kBatch = 4;          // column tiles whose waves meet in LDS together

// ---- a lane's share of 16 columns x 256 values of K --------------------------------
// v_mfma_f32_16x16x32_f16: lane l holds row / column l % 16 and, at step t,
// eight of the values of lane group g = l / 16: those from at(t, g) on.

__device__ __forceinline__ h8 join8(h2 a, h2 b, h2 c, h2 d) { return h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]}; }

struct ExpQ4K {
  static constexpr int kType = kQ4_K;
  static constexpr bool kMins = true, kLow = false;
  // nibble plane t & 1 of bytes 8 (t / 2) .. of qs chunk g
  __device__ static int at(int t, int g) { return 64 * g + 32 * (t & 1) + 8 * (t >> 1); }
  struct Item {
    u32x4 hd, q0, q1;
  };
  __device__ static void load(Item &it, Rsrc rs, uint32_t blk, int g) {
    it.hd = bload4(rs, blk);
    it.q0 = bload4(rs, blk + 16u + 32u * (uint32_t)g);
    it.q1 = bload4(rs, blk + 32u + 32u * (uint32_t)g);
  }
  // scales of the chunk's two sub-blocks as (multiplier, offset) of 1024 + q
  // and of 1024 + 16 q; their mins
  struct Cur {
    h2 sc[2], off[2];
    h8 m;
    float d, dmin;
  };
  __device__ static Cur header(const u32x4 &hd, int g) {
    Cur c;
    const uint32_t k = 2u * ((uint32_t)g & 1u);
    // (masks: a choice between the two became a branch)
    const uint32_t early = g < 2 ? 0xFFFFFFFFu : 0u;
    auto pick = [&](uint32_t a, uint32_t b) { return (a & early) | (b & ~early); };
    const uint32_t sc4 = pick(hd.y & 0x3F3F3F3Fu, (hd.w & 0x0F0F0F0Fu) | ((hd.y >> 2) & 0x30303030u));
    const uint32_t m4 = pick(hd.z & 0x3F3F3F3Fu, ((hd.w >> 4) & 0x0F0F0F0Fu) | ((hd.z >> 2) & 0x30303030u));
    const h2 s0 = byte_pair(sc4, k), s1 = byte_pair(sc4, k + 1u), m0 = byte_pair(m4, k), m1 = byte_pair(m4, k + 1u);
    auto by = [](h2 v, float f) { return v * h2{(_Float16)f, (_Float16)f}; };
    c.sc[0] = s0;
    c.off[0] = by(s0, -1024.0f);
    c.sc[1] = by(s1, 0.0625f);
    c.off[1] = by(s1, -64.0f);
    const h2 z = {(_Float16)0.0f, (_Float16)0.0f};
    c.m = join8(m0, m1, z, z);
    c.d = f16_bits_hw(hd.x & 0xffffu);
    c.dmin = f16_bits_hw(hd.x >> 16);
    return c;
  }
  __device__ static Cur begin(const Item &it, int g, int, int) { return header(it.hd, g); }
  __device__ static void frag(const Item &it, const Cur &c, int t, int, h8 &b1, h8 &) {
    const int nib = t & 1, p8 = t >> 1;
    const u32x4 pc = (p8 >> 1) ? it.q1 : it.q0;
    const uint32_t d0 = (p8 & 1) ? pc.z : pc.x, d1 = (p8 & 1) ? pc.w : pc.y;
    const uint32_t mask = nib ? 0xF0F0F0F0u : 0x0F0F0F0Fu;
    h2 p0, p1, p2, p3;
    nib4(d0 & mask, c.sc[nib], c.off[nib], p0, p1);
    nib4(d1 & mask, c.sc[nib], c.off[nib], p2, p3);
    b1 = join8(p0, p1, p2, p3);
  }
};

// Q4_K with the fifth bit from qh: bit 2 g + nibble plane of qh[l] for byte l.
struct ExpQ5K {
  static constexpr int kType = kQ5_K;
  static constexpr bool kMins = true, kLow = false;
  __device__ static int at(int t, int g) { return ExpQ4K::at(t, g); }
  struct Item {
    u32x4 hd, h0, h1, q0, q1;
  };
  using Cur = ExpQ4K::Cur;
  __device__ static void load(Item &it, Rsrc rs, uint32_t blk, int g) {
    it.hd = bload4(rs, blk);
    it.h0 = bload4(rs, blk + 16u);
    it.h1 = bload4(rs, blk + 32u);
    it.q0 = bload4(rs, blk + 48u + 32u * (uint32_t)g);
    it.q1 = bload4(rs, blk + 64u + 32u * (uint32_t)g);
  }
  __device__ static Cur begin(const Item &it, int g, int, int) { return ExpQ4K::header(it.hd, g); }
  __device__ static void frag(const Item &it, const Cur &c, int t, int g, h8 &b1, h8 &) {
    const int nib = t & 1, p8 = t >> 1;
    const u32x4 pc = (p8 >> 1) ? it.q1 : it.q0, hc = (p8 >> 1) ? it.h1 : it.h0;
    const uint32_t d0 = (p8 & 1) ? pc.z : pc.x, d1 = (p8 & 1) ? pc.w : pc.y;
    const uint32_t e0 = (p8 & 1) ? hc.z : hc.x, e1 = (p8 & 1) ? hc.w : hc.y;
    // bit 4 of the byte on the low plane (1024 + q5), the exponent byte
    // 0x64 | h on the high one (1024 + 256 h + 16 q4)
    const uint32_t sh = 2u * (uint32_t)g + (uint32_t)nib;
    const uint32_t f0 = (e0 >> sh) & 0x01010101u, f1 = (e1 >> sh) & 0x01010101u;
    const uint32_t n0 = nib ? d0 & 0xF0F0F0F0u : (d0 & 0x0F0F0F0Fu) | (f0 << 4);
    const uint32_t n1 = nib ? d1 & 0xF0F0F0F0u : (d1 & 0x0F0F0F0Fu) | (f1 << 4);
    const uint32_t x0 = nib ? f0 | 0x64646464u : 0x64646464u, x1 = nib ? f1 | 0x64646464u : 0x64646464u;
    const uint32_t lo = nib ? 0x05010400u : 0x04010400u, hi = nib ? 0x07030602u : 0x04030402u;
    b1 = join8(nib_pair(__builtin_amdgcn_perm(x0, n0, lo), c.sc[nib], c.off[nib]),
               nib_pair(__builtin_amdgcn_perm(x0, n0, hi), c.sc[nib], c.off[nib]),
               nib_pair(__builtin_amdgcn_perm(x1, n1, lo), c.sc[nib], c.off[nib]),
               nib_pair(__builtin_amdgcn_perm(x1, n1, hi), c.sc[nib], c.off[nib]));
  }
};

// Blocks of 210 bytes: every 8-byte field is a window of three dwords from the
// one below it, realigned.  The window of d ends at most 2 bytes past the
// block, in a dword that holds d.
struct ExpQ6K {
  static constexpr int kType = kQ6_K;
  static constexpr bool kMins = false, kLow = true;
  // half t / 4, quarter t % 4
  __device__ static int at(int t, int g) { return 128 * (t >> 2) + 32 * (t & 3) + 8 * g; }
  struct Item {
    u32x3 ql[4], qh[2];  // ql: (half, quarter & 1)
    u32x4 sc4;
    uint32_t sc1, r;
  };
  struct Cur {
    uint32_t L[4][2], H[2][2], S[4];
    float d;
  };
  __device__ static void load(Item &it, Rsrc rs, uint32_t blk, int g) {
    const uint32_t r = blk & 3u, a = blk - r;
#pragma unroll
    for (int p = 0; p < 4; ++p)
      it.ql[p] = __builtin_amdgcn_raw_buffer_load_b96(rs, a + 64u * (uint32_t)(p >> 1) + 32u * (uint32_t)(p & 1) + 8u * (uint32_t)g, 0, 0);
#pragma unroll
    for (int h = 0; h < 2; ++h)
      it.qh[h] = __builtin_amdgcn_raw_buffer_load_b96(rs, a + 128u + 32u * (uint32_t)h + 8u * (uint32_t)g, 0, 0);
    it.sc4 = bload4(rs, a + 192u);
    it.sc1 = __builtin_amdgcn_raw_buffer_load_b32(rs, a + 208u, 0, 0);
    it.r = r;
  }
  __device__ static Cur begin(const Item &it, int, int, int) {
    Cur c;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      c.L[p][0] = realign(it.ql[p].y, it.ql[p].x, it.r);
      c.L[p][1] = realign(it.ql[p].z, it.ql[p].y, it.r);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      c.H[h][0] = realign(it.qh[h].y, it.qh[h].x, it.r);
      c.H[h][1] = realign(it.qh[h].z, it.qh[h].y, it.r);
    }
    c.S[0] = realign(it.sc4.y, it.sc4.x, it.r);
    c.S[1] = realign(it.sc4.z, it.sc4.y, it.r);
    c.S[2] = realign(it.sc4.w, it.sc4.z, it.r);
    c.S[3] = realign(it.sc1, it.sc4.w, it.r);
    c.d = f16_bits_hw((it.sc1 >> (8u * it.r)) & 0xffffu);
    return c;
  }
  __device__ static void frag(const Item &, const Cur &c, int t, int g, h8 &b1, h8 &b2) {
    const int hh = t >> 2, qq = t & 3;
    const uint32_t *lq = c.L[2 * hh + (qq & 1)], *hq = c.H[hh];
    const int sh4 = 4 * (qq >> 1), sh2 = 2 * qq;
    const uint32_t q0 = ((lq[0] >> sh4) & 0x0F0F0F0Fu) | (((hq[0] >> sh2) & 0x03030303u) << 4);
    const uint32_t q1 = ((lq[1] >> sh4) & 0x0F0F0F0Fu) | (((hq[1] >> sh2) & 0x03030303u) << 4);
    const int sc = __builtin_amdgcn_sbfe((int)c.S[2 * hh + (qq >> 1)], 8u * (2u * (uint32_t)(qq & 1) + ((uint32_t)g >> 1)), 8u);
    const _Float16 sf = (_Float16)(float)sc;
    const h2 sc2 = {sf, sf};
    h2 p0, p1, p2, p3, l0, l1, l2, l3;
    q6_4(q0, sc2, p0, p1, l0, l1);
    q6_4(q1, sc2, p2, p3, l2, l3);
    b1 = join8(p0, p1, p2, p3);
    b2 = join8(l0, l1, l2, l3);
  }
};

// Eight blocks of 34 bytes, 2 g and 2 g + 1 the lane group's.  d goes into the
// two exact planes of d * q; where that could pass fp16 (|d| >= 256, which no
// weights of ordinary size have), a tile's item goes in two parts.  A row of K not a multiple of 256 ends inside an
// item: what follows it (the next row's blocks, or nothing) gets a d of zero and
// meets zeros (both: a scale that is no number, or a product past fp16, times
// zero would be NaN).
struct ExpQ80 {
  static constexpr int kType = kQ8_0;
  static constexpr bool kMins = false, kLow = true;
  __device__ static int at(int t, int g) { return 64 * g + 8 * t; }
  struct Item {
    u32x4 w0, w1, w2, w3;
    u32x2 w4;
    uint32_t r;
  };
  struct Cur {
    uint32_t w[17];
    h2 d0, d1;
    float d;
  };
  __device__ static void load(Item &it, Rsrc rs, uint32_t blk, int g) {
    const uint32_t at = blk + 68u * (uint32_t)g, r = at & 3u, a = at - r;
    it.w0 = bload4(rs, a);
    it.w1 = bload4(rs, a + 16u);
    it.w2 = bload4(rs, a + 32u);
    it.w3 = bload4(rs, a + 48u);
    it.w4 = __builtin_amdgcn_raw_buffer_load_b64(rs, a + 64u, 0, 0);
    it.r = r;
  }
  // the scales' bits, zeros behind the row's last block
  __device__ static void scales(const Item &it, int g, int left, uint32_t &e0, uint32_t &e1) {
    const uint32_t w0 = realign(it.w0.y, it.w0.x, it.r), w8 = realign(it.w2.y, it.w2.x, it.r);
    e0 = 64 * g < left ? w0 & 0xffffu : 0u;
    e1 = 64 * g + 32 < left ? w8 >> 16 : 0u;
  }
  // |d| from 256 on (infinities and NaN among them): d * q may pass fp16
  __device__ static bool large(uint32_t e) { return (e & 0x7fffu) >= 0x5c00u; }
  __device__ static bool any_large(const Item &it, int g, int left) {
    uint32_t e0, e1;
    scales(it, g, left, e0, e1);
    return __builtin_amdgcn_ballot_w64(large(e0) || large(e1)) != 0;
  }
  // part 0: the blocks of ordinary scales; part 1: the large ones, d / 256 (an
  // exact fp16) in the planes and 256 in front of their sum
  __device__ static Cur begin(const Item &it, int g, int left, int part) {
    const uint32_t raw[18] = {it.w0.x, it.w0.y, it.w0.z, it.w0.w, it.w1.x, it.w1.y, it.w1.z, it.w1.w, it.w2.x,
                              it.w2.y, it.w2.z, it.w2.w, it.w3.x, it.w3.y, it.w3.z, it.w3.w, it.w4.x, it.w4.y};
    Cur c;
#pragma unroll
    for (int i = 0; i < 17; ++i) c.w[i] = realign(raw[i + 1], raw[i], it.r);
    uint32_t e0, e1;
    scales(it, g, left, e0, e1);
    c.d = 1.0f;
    if (part >= 0) {
      e0 = large(e0) == (part == 1) ? e0 : 0u;
      e1 = large(e1) == (part == 1) ? e1 : 0u;
    }
    _Float16 d0 = __builtin_bit_cast(_Float16, (uint16_t)e0), d1 = __builtin_bit_cast(_Float16, (uint16_t)e1);
    if (part == 1) {
      d0 *= (_Float16)0.00390625f;
      d1 *= (_Float16)0.00390625f;
      c.d = 256.0f;
    }
    c.d0 = h2{d0, d0};
    c.d1 = h2{d1, d1};
    return c;
  }
  __device__ static void frag(const Item &, const Cur &c, int t, int, h8 &b1, h8 &b2) {
    const int blk = t >> 2, o = 2 * (t & 3);
    const uint32_t qa = blk ? c.w[9 + o] : realign(c.w[o + 1], c.w[o], 2u);
    const uint32_t qb = blk ? c.w[10 + o] : realign(c.w[o + 2], c.w[o + 1], 2u);
    h2 p0, p1, p2, p3, l0, l1, l2, l3;
    q8_4(qa, blk ? c.d1 : c.d0, p0, p1, l0, l1);
    q8_4(qb, blk ? c.d1 : c.d0, p2, p3, l2, l3);
    b1 = join8(p0, p1, p2, p3);
    b2 = join8(l0, l1, l2, l3);
  }
};

// A lane's row of activations for one item: both planes' fragments, the sums
// of its two sub-blocks of 32 as (hi, lo) pairs (Q4_K, Q5_K), and the scale.
struct ActA {
  h8 hi[8], lo[8], sums;
  float scale;
};

template <class F>
__device__ __forceinline__ void load_row(float4 raw[16], const float *row, int k0, int K, int g) {
#pragma unroll
  for (int t = 0; t < 8; ++t) {
    const int k = k0 + F::at(t, g);
    const bool in = F::kType != kQ8_0 || k < K;  // other formats' rows are whole items
    const float4 *p = reinterpret_cast<const float4 *>(row + (in ? k : 0));
    raw[2 * t] = p[0];
    raw[2 * t + 1] = p[1];
    if (!in) raw[2 * t] = raw[2 * t + 1] = float4{0.0f, 0.0f, 0.0f, 0.0f};
  }
}

// The lane groups of a row share their scale 2^s: the largest |x| of its 256
// lies in [512, 1024).
template <class F>
__device__ __forceinline__ void convert(ActA &A, const float4 raw[16]) {
  // the largest magnitude as a bit pattern (NaN above infinity above every
  // finite value): the largest of the positive ones in signed order, of the
  // negative ones in unsigned order
  int pos = 0;
  uint32_t neg = 0;
  auto value = [&](int t, int e) {
    const float4 v = raw[2 * t + (e >> 2)];
    return (e & 3) == 0 ? v.x : (e & 3) == 1 ? v.y : (e & 3) == 2 ? v.z : v.w;
  };
#pragma unroll
  for (int t = 0; t < 8; ++t)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t b = as_u32(value(t, e));
      pos = pos > (int)b ? pos : (int)b;
      neg = neg > b ? neg : b;
    }
  neg &= 0x7fffffffu;  // without a negative value: the positives' largest once more
  uint32_t top = neg > (uint32_t)pos ? neg : (uint32_t)pos;
  uint32_t o = (uint32_t)__shfl_xor((int)top, 16);
  top = top > o ? top : o;
  o = (uint32_t)__shfl_xor((int)top, 32);
  top = top > o ? top : o;
  const bool odd = top >= 0x7f800000u;
  const int s = top > 0 && !odd ? __builtin_amdgcn_frexp_expf(as_f32(top)) - 10 : 0;
  A.scale = odd ? __builtin_nanf("") : ldexpf(1.0f, s);
  float sum[2] = {0.0f, 0.0f};
  const h2 one = {(_Float16)1.0f, (_Float16)1.0f};
  auto put = [&](int t, auto &&plane, auto &&rest) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const h2 h = {(_Float16)plane(value(t, e)), (_Float16)plane(value(t, e + 1))};
      const h2 l = {(_Float16)rest(value(t, e), h[0]), (_Float16)rest(value(t, e + 1), h[1])};
      A.hi[t][e] = h[0];
      A.hi[t][e + 1] = h[1];
      A.lo[t][e] = l[0];
      A.lo[t][e + 1] = l[1];
      // sums of what the planes hold
      if (F::kMins) sum[t & 1] = __builtin_amdgcn_fdot2(l, one, __builtin_amdgcn_fdot2(h, one, sum[t & 1], false), false);
    }
    __builtin_amdgcn_sched_barrier(0);  // planes take the raw values' registers, piece by piece
  };
  // 2^-s a normal f32 (every row of the wave): one mixed multiply-add a plane
  if (__builtin_amdgcn_ballot_w64(s < -100 || s > 100) == 0) {
    const float f = ldexpf(1.0f, -s);
#pragma unroll
    for (int t = 0; t < 8; ++t)
      put(t, [&](float v) { return __builtin_fmaf(v, f, 0.0f); },
          [&](float v, _Float16 h) { return __builtin_fmaf(v, f, -(float)h); });
  } else {
#pragma unroll
    for (int t = 0; t < 8; ++t)
      put(t, [&](float v) { return ldexpf(v, -s); }, [&](float v, _Float16 h) { return ldexpf(v, -s) - (float)h; });
  }
  if (F::kMins) {
    const _Float16 h0 = (_Float16)sum[0], h1 = (_Float16)sum[1];
    const _Float16 z = (_Float16)0.0f;
    A.sums = h8{h0, (_Float16)(sum[0] - (float)h0), h1, (_Float16)(sum[1] - (float)h1), z, z, z, z};
  }
}

// acc (rows 4 g .. 4 g + 3 of the lane's column) += the item's products; rs:
// the rows' scales; left: the values of the row from the item on; part: of
// Q8_0's blocks, one of the two or all (-1).
template <class F>
__device__ __forceinline__ void contract(f4 &acc, const typename F::Item &it, const ActA &A, const f4 &rs, int g,
                                         int left, int part = -1) {
  const f4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
  const typename F::Cur c = F::begin(it, g, left, part);
  f4 s = zero, low = zero;  // two chains: a product waits for the one before it in its own
#pragma unroll
  for (int t = 0; t < 8; ++t) {
    h8 b1, b2;
    F::frag(it, c, t, g, b1, b2);
    s = __builtin_amdgcn_mfma_f32_16x16x32_f16(A.hi[t], b1, s, 0, 0, 0);
    low = __builtin_amdgcn_mfma_f32_16x16x32_f16(A.lo[t], b1, low, 0, 0, 0);
    // (lo * b2 is below 2^-22 of the product)
    if constexpr (F::kLow) low = __builtin_amdgcn_mfma_f32_16x16x32_f16(A.hi[t], b2, low, 0, 0, 0);
  }
  s += low;
  if constexpr (F::kMins) {
    const f4 m = __builtin_amdgcn_mfma_f32_16x16x32_f16(A.sums, c.m, zero, 0, 0, 0);
#pragma unroll
    for (int v = 0; v < 4; ++v) acc[v] = fmaf(rs[v], fmaf(-c.dmin, m[v], c.d * s[v]), acc[v]);
  } else {
#pragma unroll
    for (int v = 0; v < 4; ++v) acc[v] = fmaf(c.d * rs[v], s[v], acc[v]);
  }
}

// One product over the pairs: y[p] = act(W_e x_p), p's expert e.
struct MoeProduct {
  const float *x;       // rows of K: of tokens (top_k pairs share one), or of pairs (share 1)
  int64_t x_stride;
  int share;
  const uint8_t *w[2];  // stacked tensors of the pass: gate and up, or down
  uint64_t w_bytes;     // of each
  uint64_t expert_bytes;
  const int32_t *ids;
  const float *weights;  // down: a pair's factor
  const int *order, *count;  // sorted pairs and the number of jobs (null: few pairs, not sorted)
  const ExpertTile *jobs;    // up to 16 rows of an expert each
  float *y;              // [pairs][N]
  int pairs, experts, K, N, nsb, row_bytes;
  int slices;            // of K, each with a part of y [slices][NM][pairs][N]; 1: the product itself
  int slots, steps;      // column tiles side by side in a workgroup; steps over all columns
  int rounds;            // few pairs: steps of a workgroup
};

}  // namespace

// A workgroup has one slice of K of at most kWaves items, and passes over steps
// of `slots` column tiles of up to 16 rows of one expert (a job).  A wave keeps
// its item's activations in registers (16 rows, both planes: 64 of them) while
// the weights of one tile after the other come through a ring of D, so that
// each weight is read once and nothing but weights is read in the loop; the
// waves of a slice meet in LDS, kBatch tiles at a time in one of two buffers,
// one barrier a batch.
//
// Sorted pairs: the workgroups of a slice share out all jobs' steps evenly,
// whatever the experts' shares of the rows are.  With one workgroup an expert's
// columns, unused experts left CUs idle and one of 17 rows took twice the time
// of the others: 96 rows of 8 of 256 experts, gate and up 169 -> 87 us.
//
// What bounds it: for many experts memory (48 rows of 8 of 128, 2048 x 768 in
// Q4_K: gate and up 47 us, down 33, for 208 and 104 MB: 4.4 and 3.2 TB/s with
// 9 us of launch, sort, rows and their planes ahead of the stream; 13 rows of 2
// of 8, 4096 x 14336: 528 MB in 121 us, Q6_K down 385 MB in 112); for one row
// the chain ids, rows, weights, join: 10.7 and 8.0 us.  A tile costs a wave
// some 170 VALU instructions an item, which with 8 waves a CU take 40-50% of
// the cycles.
//
// A few pairs (kFewPairs at most) whose experts mostly differ are not sorted (a
// launch of 5 us): every workgroup has a pair's expert and lists its pairs by
// itself, going on if no earlier pair has the same, `rounds` steps and as many
// turns as it has 16 rows.
template <class F, int NM, int D>
__global__ __launch_bounds__(kWaves * 64) void moe_stream_kernel(MoeProduct a) {
  __shared__ f4 red[2][kBatch][kWaves][NM][64];
  __shared__ uint8_t lists[kWaves][kFewPairs];
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int waves = (int)blockDim.x >> 6, z = (int)blockIdx.z;
  const int s0 = z * a.nsb / a.slices, kw = (z + 1) * a.nsb / a.slices - s0;  // the slice's items
  const int slot = __builtin_amdgcn_readfirstlane(wave / kw), ks = wave - slot * kw, item = s0 + ks;
  const bool idle = slot >= a.slots;  // a slice with fewer items than its launch has waves for
  const uint32_t sb = (uint32_t)(F::kType == kQ8_0 ? 8 * kQ8Bytes : sb_bytes_of(F::kType));

  // the steps [u, end) of this workgroup, job * steps + step (sorted pairs), or
  // of its expert's turns
  int u, end, expert = 0, m = 0;
  if (a.order) {
    const int64_t all = (int64_t)a.count[0] * a.steps;
    u = (int)(all * blockIdx.x / gridDim.x);
    end = (int)(all * (blockIdx.x + 1) / gridDim.x);
  } else {
    const int id = a.ids[std::min(lane, a.pairs - 1)], job = (int)blockIdx.y;
    expert = __builtin_amdgcn_readlane(id, job);
    const uint64_t all = __builtin_amdgcn_ballot_w64(lane < a.pairs && id == expert);
    if ((uint32_t)expert >= (uint32_t)a.experts || __builtin_ctzll(all) != job) return;
    m = __builtin_popcountll(all);
    if (all >> lane & 1) lists[wave][__builtin_popcountll(all & ((1ull << lane) - 1))] = (uint8_t)lane;
    wave_sync();
    u = 0;
    end = (m + 15) / 16;
  }
  int parity = 0;
  while (u < end) {
    // (opaque, so that a job's addresses are not formed ahead of the loop, where
    // they would take the registers that the loads need)
    int l = lane;
    asm volatile("" : "+v"(l));
    const int n = l & 15, g = l >> 4;
    int step0, steps, rows, pair;
    if (a.order) {
      const int job = u / a.steps;
      const ExpertTile t = a.jobs[job];
      expert = t.expert;
      rows = t.rows;
      step0 = u - job * a.steps;
      steps = std::min(a.steps - step0, end - u);
      u += steps;
      pair = a.order[t.row0 + std::min(n, rows - 1)];
    } else {
      rows = std::min(16, m - 16 * u);
      step0 = (int)blockIdx.x * a.rounds;
      steps = std::min(a.steps - step0, a.rounds);
      pair = lists[wave][16 * u + std::min(n, rows - 1)];
      u += 1;
    }
    // the expert's weights from the dword at or below its first byte, to the
    // last dword that holds a byte of the stack
    Rsrc rs[NM];
    uint32_t skew[NM];
#pragma unroll
    for (int i = 0; i < NM; ++i) {
      const uint64_t from = (uint64_t)expert * a.expert_bytes;
      const uint8_t *base = a.w[i] + from;
      skew[i] = (uint32_t)(reinterpret_cast<uintptr_t>(base) & 3u);
      const uint64_t left = (a.w_bytes - from + skew[i] + 3u) & ~3ull;
      rs[i] = make_rsrc(base - skew[i], (uint32_t)std::min<uint64_t>(left, 0xFFFFFFFCull));
    }
    typename F::Item S[D][NM];
    // the weights of the wave's i-th tile (past the steps, or columns past the
    // last: past the stack, nothing)
    auto load_one = [&](typename F::Item &it, int i, int k) {
      const int col = ((step0 + i) * a.slots + slot) * 16 + n;
      const bool in = !idle && i < steps && col < a.N;
      const uint32_t at = (uint32_t)col * (uint32_t)a.row_bytes + (uint32_t)item * sb;
      F::load(it, rs[k], in ? at + skew[k] : 0xFFFFF000u, g);
    };
    auto load_tile = [&](typename F::Item *it, int i) {
#pragma unroll
      for (int k = 0; k < NM; ++k) load_one(it[k], i, k);
    };
    ActA A;
    f4 scales, factor = {};  // of the four rows whose sums the lane holds
    int mine[4];             // their pairs
#pragma unroll
    for (int v = 0; v < 4; ++v) mine[v] = __shfl(pair, 4 * g + v);
    {
      float4 raw[16];
      load_row<F>(raw, a.x + (int64_t)(pair / a.share) * a.x_stride, item * 256, a.K, g);
      __builtin_amdgcn_sched_barrier(0);  // the activations ahead of the weights: loads return in order
#pragma unroll
      for (int d = 0; d < D; ++d) load_tile(S[d], d);
      if constexpr (NM == 1)
#pragma unroll
        for (int v = 0; v < 4; ++v) factor[v] = a.weights[mine[v]];
      __builtin_amdgcn_sched_barrier(0);
      convert<F>(A, raw);
#pragma unroll
      for (int v = 0; v < 4; ++v) scales[v] = __shfl(A.scale, 4 * g + v);
    }
    for (int i0 = 0; i0 < steps; i0 += D) {
#pragma unroll
      for (int d = 0; d < D; ++d) {
        const int i = i0 + d;  // (may be one past the last: zeros, not stored)
#pragma unroll
        for (int k = 0; k < NM; ++k) {
          f4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
          const int left = a.K - 256 * item;
          bool whole = true;
          if constexpr (F::kType == kQ8_0) whole = !F::any_large(S[d][k], g, left);
          if (whole) {
            contract<F>(acc, S[d][k], A, scales, g, left);
          } else {
            // in two, the item loaded anew (kept, it would cost every other one registers)
#pragma unroll 1
            for (int part = 0; part < 2; ++part) {
              typename F::Item it;
              load_one(it, i, k);
              contract<F>(acc, it, A, scales, g, left, part);
            }
          }
          red[parity][i % kBatch][wave][k][l] = acc;
        }
        // into the registers that this tile's weights have left (issued any
        // earlier, they took others, and moving them waited for every load)
        __builtin_amdgcn_sched_barrier(0);
        load_tile(S[d], i + D);
      }
      const int done = std::min(i0 + D, steps);
      if (done % kBatch != 0 && done < steps) continue;
      lds_barrier();  // the weights stay in flight
      // the batch's tiles, a wave each, over their items in order; the next
      // batch goes to the other buffer, and other waves first
      const int from = (done - 1) / kBatch * kBatch, n_tiles = (done - from) * a.slots;
      for (int j = parity ? waves - 1 - wave : wave; j < n_tiles; j += waves) {
        const int b = j / a.slots, sl = j - b * a.slots;
        f4 sum[NM];
#pragma unroll
        for (int k = 0; k < NM; ++k) {
          f4 v[kWaves];
#pragma unroll
          for (int w = 0; w < kWaves; ++w)
            v[w] = w < kw ? red[parity][b][sl * kw + w][k][l] : f4{0.0f, 0.0f, 0.0f, 0.0f};
          sum[k] = v[0];
#pragma unroll
          for (int w = 1; w < kWaves; ++w) sum[k] += v[w];
        }
        const int col = ((step0 + from + b) * a.slots + sl) * 16 + n;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const int64_t q = mine[v];
          if (4 * g + v >= rows || col >= a.N) continue;
          if (NM == 2 && a.slices > 1) {
            float *y = a.y + ((int64_t)z * NM * a.pairs + q) * a.N + col;
            y[0] = sum[0][v];
            y[(int64_t)a.pairs * a.N] = sum[NM - 1][v];
          } else if (NM == 2) {
            a.y[q * a.N + col] = (sum[0][v] * (1.0f / (1.0f + expf(-sum[0][v])))) * sum[NM - 1][v];
          } else {
            a.y[((int64_t)z * a.pairs + q) * a.N + col] = sum[0][v] * factor[v];
          }
        }
      }
      parity ^= 1;
    }
  }
}

// silu(gate) * up from the slices' parts [slices][2][n].
__global__ __launch_bounds__(256) void moe_gate_kernel(const float4 *__restrict__ part, int slices, int64_t n4,
                                                       float4 *__restrict__ y) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n4) return;
  float4 g = part[i], u = part[n4 + i];
  for (int z = 1; z < slices; ++z) {
    const float4 a = part[2 * z * n4 + i], b = part[(2 * z + 1) * n4 + i];
    g = float4{g.x + a.x, g.y + a.y, g.z + a.z, g.w + a.w};
    u = float4{u.x + b.x, u.y + b.y, u.z + b.z, u.w + b.w};
  }
  auto f = [](float v, float w) { return (v * (1.0f / (1.0f + expf(-v)))) * w; };
  y[i] = float4{f(g.x, u.x), f(g.y, u.y), f(g.z, u.z), f(g.w, u.w)};
}

// ---- many rows: the pairs sorted by expert ------------------------------------------

// order: the pairs by expert; place: each pair's place in it (-1: no such
// expert); count: tiles of up to `height` rows, and pairs with an expert; the
// tiles.  One workgroup: the ids of 4096 tokens are 128 KB, and their counts
// meet in LDS (32768 pairs 28 us, 384 5).  (Pairs of an expert come in any
// order: a row's result does not depend on its place.)
__global__ __launch_bounds__(1024) void moe_sort_kernel(const int32_t *__restrict__ ids, int pairs, int experts,
                                                        int height, int *__restrict__ order, int *__restrict__ place,
                                                        int *__restrict__ count, ExpertTile *__restrict__ tiles) {
  constexpr int kPer = kMoeMaxExperts / 1024, kHeld = 16;
  __shared__ int next[kMoeMaxExperts];
  __shared__ int2 waves[16];
  __shared__ uint16_t sorted[kPassPairs];  // stored in order: scattered from one CU, 32768 words took 8 us more
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int e = tid; e < kMoeMaxExperts; e += 1024) next[e] = 0;
  __syncthreads();
  // kHeld ids of a thread are requested at once; the first of them stay for the
  // second pass
  int held[kHeld];
  auto get = [&](int p0) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int p = p0 + 1024 * i + tid;
      const int e = ids[p < pairs ? p : 0];
      held[i] = p < pairs && (uint32_t)e < (uint32_t)experts ? e : -1;
    }
  };
  const int last = (pairs - 1) / (1024 * kHeld) * (1024 * kHeld);
  for (int p0 = last; p0 >= 0; p0 -= 1024 * kHeld) {
    get(p0);
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (held[i] >= 0) atomicAdd(&next[held[i]], 1);
  }
  __syncthreads();
  // rows and tiles ahead of each expert: kPer experts a thread
  int m[kPer], rows = 0, mine = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    m[i] = next[kPer * tid + i];
    rows += m[i];
    mine += (m[i] + height - 1) / height;
  }
  int r = rows, t = mine;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int ro = __shfl_up(r, d), to = __shfl_up(t, d);
    r += lane >= d ? ro : 0;
    t += lane >= d ? to : 0;
  }
  if (lane == 63) waves[wave] = int2{r, t};
  __syncthreads();
  r -= rows;
  t -= mine;
  for (int w = 0; w < wave; ++w) {
    r += waves[w].x;
    t += waves[w].y;
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    next[kPer * tid + i] = r;
    for (int at = 0; at < m[i]; at += height) {
      const int n = m[i] - at < height ? m[i] - at : height;
      tiles[t++] = ExpertTile{kPer * tid + i, r + at, n, (n + 31) / 32};
    }
    r += m[i];
  }
  __syncthreads();  // (the waves' sums are read)
  if (tid == 1023) {
    count[0] = t;
    count[1] = r;
    waves[0].x = r;
  }
  for (int p0 = 0; p0 <= last; p0 += 1024 * kHeld) {
    if (p0) get(p0);
    int at[kHeld];
#pragma unroll
    for (int i = 0; i < kHeld; ++i) at[i] = held[i] >= 0 ? atomicAdd(&next[held[i]], 1) : -1;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int p = p0 + 1024 * i + tid;
      if (p < pairs) place[p] = at[i];
      if (at[i] >= 0) sorted[at[i]] = (uint16_t)p;
    }
  }
  __syncthreads();
  const int n = waves[0].x;  // pairs with an expert
#pragma unroll 4
  for (int i = tid; i < n; i += 1024) order[i] = sorted[i];
}

// Rows of K values as two fp16 planes of rows of Kp (zeros behind K), their
// per-32 sums and scales: a wave a row, CH chunks of 8 values a lane (0: as
// many as the row has, read twice).  count: rows that there are, where only
// the device knows.
template <int CH>
__global__ __launch_bounds__(256) void moe_planes_kernel(const float *__restrict__ x, int64_t x_stride, int rows,
                                                         const int *__restrict__ count, int K, int Kp,
                                                         _Float16 *__restrict__ hi, _Float16 *__restrict__ lo,
                                                         h2 *__restrict__ sums, float *__restrict__ rscale) {
  const int lane = (int)threadIdx.x & 63, row = (int)blockIdx.x * 4 + ((int)threadIdx.x >> 6);
  if (row >= (count ? count[1] : rows)) return;
  const float *from = x + (int64_t)row * x_stride;
  const int chunks = Kp / 8, full = K / 8;
  auto get = [&](int c, float v[8]) {
    const float4 *p = reinterpret_cast<const float4 *>(from + 8 * (c < full ? c : 0));
    const float4 a = p[0], b = p[1];
    const float w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c < full ? w[e] : 0.0f;
  };
  auto top_of = [](uint32_t top, const float v[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t b = as_u32(v[e]) & 0x7fffffffu;
      top = top > b ? top : b;
    }
    return top;
  };
  float v[CH ? CH : 1][8];
  uint32_t top = 0;
  if constexpr (CH > 0) {
#pragma unroll
    for (int i = 0; i < CH; ++i) get(lane + 64 * i, v[i]);
#pragma unroll
    for (int i = 0; i < CH; ++i) top = top_of(top, v[i]);
  } else {
    for (int c = lane; c < full; c += 64) {
      get(c, v[0]);
      top = top_of(top, v[0]);
    }
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint32_t o = (uint32_t)__shfl_xor((int)top, d);
    top = top > o ? top : o;
  }
  const bool odd = top >= 0x7f800000u;
  const int s = top > 0 && !odd ? __builtin_amdgcn_frexp_expf(as_f32(top)) - 10 : 0;
  if (lane == 0) rscale[row] = odd ? __builtin_nanf("") : ldexpf(1.0f, s);
  auto put = [&](int c, const float w[8]) {
    h8 h, l;
    float t = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float y = ldexpf(w[e], -s);
      h[e] = (_Float16)y;
      l[e] = (_Float16)(y - (float)h[e]);
      t += (float)h[e] + (float)l[e];  // what the planes hold
    }
    t += dpp_row_f<0xB1>(t);
    t += dpp_row_f<0x4E>(t);
    if (c < chunks) {
      const int64_t at = (int64_t)row * Kp + 8 * c;
      *reinterpret_cast<h8 *>(hi + at) = h;
      *reinterpret_cast<h8 *>(lo + at) = l;
      if ((c & 3) == 0) sums[at / 32] = h2{(_Float16)t, (_Float16)(t - (float)(_Float16)t)};
    }
  };
  if constexpr (CH > 0) {
#pragma unroll
    for (int i = 0; i < CH; ++i) put(lane + 64 * i, v[i]);
  } else {
    for (int c0 = 0; c0 < chunks; c0 += 64) {
      get(c0 + lane, v[0]);
      put(c0 + lane, v[0]);
    }
  }
}

// out[t] = the sum of its pairs' rows, in their order; zeros for none.  place:
// where a pair's row is; without it, its own place if it has an expert.  Rows
// may come in slices to add up.
template <int N>
__global__ __launch_bounds__(256) void moe_sum_kernel(const float *__restrict__ y, const int32_t *__restrict__ ids,
                                                      const int *__restrict__ place, int top_k, int experts, int hidden,
                                                      int slices, int64_t slice, float *__restrict__ out,
                                                      int64_t out_stride) {
  typedef float fN __attribute__((ext_vector_type(N)));
  const int64_t t = blockIdx.x;
  const int c = ((int)blockIdx.y * 256 + (int)threadIdx.x) * N;
  if (c >= hidden) return;
  fN sum = {};
  for (int j = 0; j < top_k; ++j) {
    const int64_t p = t * top_k + j;
    const int64_t at = place ? place[p] : (uint32_t)ids[p] < (uint32_t)experts ? p : -1;
    if (at >= 0)
      for (int z = 0; z < slices; ++z) sum += *reinterpret_cast<const fN *>(y + z * slice + at * hidden + c);
  }
  *reinterpret_cast<fN *>(out + t * out_stride + c) = sum;
}

static size_t up256(size_t v) { return (v + 255) & ~(size_t)255; }
static int whole(int k) { return (k + 255) / 256 * 256; }

// Planes of `rows` rows of K values at a place of the workspace.
struct Planes {
  size_t hi, lo, sums, rscale, end;
  Planes(size_t at, int64_t rows, int K) {
    const size_t n = (size_t)rows * (size_t)whole(K);
    hi = at;
    lo = hi + up256(n * 2);
    sums = lo + up256(n * 2);
    rscale = sums + up256(n / 8);
    end = rscale + up256((size_t)rows * 4);
  }
};

// Slices of K of at most kWaves items.
static int k_slices(int K) { return ((K + 255) / 256 + kWaves - 1) / kWaves; }

static MoePlan plan_of(const MoeArgs &a, bool tiled) {
  MoePlan p{};
  p.tiled = tiled;
  const size_t gs = p.tiled ? 1 : k_slices(a.hidden), ds = p.tiled ? 1 : k_slices(a.inner);
  // a pass keeps to about 1 GiB of results, and to what its kernels count in
  // 32 bits
  const int64_t one = 4 * ((int64_t)a.inner * (gs > 1 ? 1 + 2 * gs : 2) + (int64_t)a.hidden * ds);
  const int64_t most = std::min<int64_t>({kPassPairs, (1 << 30) / one, (UINT32_MAX - (1 << 20)) / (2 * (int64_t)whole(std::max(a.inner, a.hidden)))});
  p.pass_rows = std::max<int64_t>(1, std::min<int64_t>(a.rows, most / a.top_k));
  const size_t pairs = (size_t)p.pass_rows * a.top_k;
  p.off_inner = 0;
  p.off_pair = up256(pairs * a.inner * sizeof(float));
  p.off_order = p.off_pair + up256(pairs * a.hidden * ds * sizeof(float));
  p.off_x = p.off_order + 2 * up256(pairs * sizeof(int)) + 256 +
            up256(expert_tiles(pairs, a.experts, p.tiled ? 128 : 16) * sizeof(ExpertTile));
  if (p.tiled)
    p.workspace = Planes(Planes(p.off_x, p.pass_rows, a.hidden).end, pairs, a.inner).end;
  else
    p.workspace = p.off_x + (gs > 1 ? up256(2 * gs * pairs * a.inner * sizeof(float)) : 0);
  return p;
}

MoePlan moe_plan(const MoeArgs &a) {
  // Sorted tiles from 28 rows an expert on average, where they begin to be the
  // faster ones: at 24 and 32, us streamed / tiled, 2048 x 768 Q4_K and Q6_K with
  // 128 experts 237 / 248 and 298 / 275, 2048 x 1536 Q5_K and Q8_0 with 32 150 /
  // 157 and 173 / 168, 4096 x 4096 Q6_K with 8 199 / 215 and 251 / 239.
  // The average is the call's: every pass over it goes the same way, also where
  // a pass has fewer rows an expert (of more than 2340 experts, or the last one).
  const int64_t least = 28 * (int64_t)a.experts;  // pairs
  const bool tiled = (int64_t)a.rows * a.top_k >= least;
  MoePlan p = plan_of(a, tiled);
  p.reserve = p.workspace;
  if (tiled) {
    MoeArgs streamed = a;
    streamed.rows = (int)((least + a.top_k - 1) / a.top_k);
    p.reserve = std::max(p.reserve, plan_of(streamed, false).workspace);
  }
  return p;
}

// The sorted pairs' places in the workspace.
struct Sorted {
  int *order, *place, *count;
  ExpertTile *tiles;
  Sorted(uint8_t *ws, const MoePlan &p, int top_k) {
    const size_t n = up256((size_t)p.pass_rows * top_k * sizeof(int)) / sizeof(int);
    order = reinterpret_cast<int *>(ws + p.off_order);
    place = order + n;
    count = place + n;
    tiles = reinterpret_cast<ExpertTile *>(count + 64);
  }
};

static hipError_t launch_planes(const float *x, int64_t x_stride, int64_t rows, const int *count, int K, uint8_t *ws,
                                const Planes &p, hipStream_t s) {
  const int Kp = whole(K), ch = (Kp / 8 + 63) / 64;
  const dim3 grid((unsigned)((rows + 3) / 4));
  _Float16 *hi = reinterpret_cast<_Float16 *>(ws + p.hi), *lo = reinterpret_cast<_Float16 *>(ws + p.lo);
  h2 *sums = reinterpret_cast<h2 *>(ws + p.sums);
  float *rscale = reinterpret_cast<float *>(ws + p.rscale);
#define OKQ_PLANES(CH_) \
  launch_timed(moe_planes_kernel<CH_>, grid, dim3(256), 0u, s, x, x_stride, (int)rows, count, K, Kp, hi, lo, sums, rscale)
  if (ch == 1) OKQ_PLANES(1);
  else if (ch == 2) OKQ_PLANES(2);
  else if (ch <= 4) OKQ_PLANES(4);
  else if (ch <= 8) OKQ_PLANES(8);
  else OKQ_PLANES(0);
#undef OKQ_PLANES
  return hipGetLastError();
}

static hipError_t launch_sum(const MoeArgs &a, const float *y, const int32_t *ids, const int *place, int64_t rows,
                             int slices, float *out, hipStream_t s) {
  const int64_t slice = rows * a.top_k * a.hidden;
  const bool wide = (reinterpret_cast<uintptr_t>(out) & 15u) == 0 && a.out_stride % 4 == 0;
  const dim3 grid((unsigned)rows, (unsigned)((a.hidden / (wide ? 4 : 1) + 255) / 256));
  if (wide) launch_timed(moe_sum_kernel<4>, grid, dim3(256), 0u, s, y, ids, place, a.top_k, a.experts, a.hidden,
                         slices, slice, out, a.out_stride);
  else launch_timed(moe_sum_kernel<1>, grid, dim3(256), 0u, s, y, ids, place, a.top_k, a.experts, a.hidden,
                         slices, slice, out, a.out_stride);
  return hipGetLastError();
}

template <class F, int NM>
static hipError_t launch_product(MoeProduct a, int cu_count, hipStream_t s) {
  const int kw = (a.nsb + a.slices - 1) / a.slices;  // items of the longest slice
  a.slots = kWaves / kw;
  a.steps = ((a.N + 15) / 16 + a.slots - 1) / a.slots;
  const dim3 block(64 * kw * a.slots);
  // one workgroup a CU (its registers fill it), each with an even share of the steps
  const int groups = std::max(1, cu_count / a.slices);
  dim3 grid(groups, 1, a.slices);
  if (!a.order) {
    a.rounds = (int)((a.pairs * (int64_t)a.steps + groups - 1) / groups);
    grid = dim3((a.steps + a.rounds - 1) / a.rounds, a.pairs, a.slices);
  }
  // Two tiles in flight a wave where a workgroup has more than two.  us a call
  // with two / with one: 48 rows, 8 of 128, 2048 x 768 Q4_K 92 / 97, Q5_K 116 /
  // 120, Q6_K 146 / 148 and 2048 x 1440 Q8_0 234 / 243, though the latter two's
  // down spills 17 and 10 registers for it (their gate and up would spill 63 and
  // 33).  Two steps in all, one row, 8 of 128, 2048 x 768: 25.3 / 22.6
  // in Q4_K and Q6_K, 28.7 / 26.7 in Q8_0.
  if ((a.order || a.rounds > 2) && (NM == 1 || !F::kLow))
    launch_timed(moe_stream_kernel<F, NM, NM == 1 || !F::kLow ? 2 : 1>, grid, block, 0u, s, a);
  else
    launch_timed(moe_stream_kernel<F, NM, 1>, grid, block, 0u, s, a);
  return hipGetLastError();
}

template <int NM>
static hipError_t launch_product(int type, const MoeProduct &a, int cu_count, hipStream_t s) {
  if (type == kQ4_K) return launch_product<ExpQ4K, NM>(a, cu_count, s);
  if (type == kQ5_K) return launch_product<ExpQ5K, NM>(a, cu_count, s);
  if (type == kQ6_K) return launch_product<ExpQ6K, NM>(a, cu_count, s);
  return launch_product<ExpQ80, NM>(a, cu_count, s);
}

static MoeProduct product(int type, int K, int N, int experts) {
  MoeProduct p{};
  p.K = K;
  p.N = N;
  p.experts = experts;
  p.nsb = (K + 255) / 256;
  p.slices = k_slices(K);
  p.row_bytes = type == kQ8_0 ? K / 32 * kQ8Bytes : K / 256 * sb_bytes_of(type);
  p.expert_bytes = (uint64_t)N * (uint64_t)p.row_bytes;
  p.w_bytes = p.expert_bytes * (uint64_t)experts;
  return p;
}

// A pass over `rows` rows from t0 on, the pairs sorted.
static hipError_t tiled_pass(const MoeArgs &a, const MoePlan &plan, uint8_t *ws, int64_t t0, int64_t rows, hipStream_t s) {
  const int64_t pairs = rows * a.top_k, room = plan.pass_rows * a.top_k;
  float *inner = reinterpret_cast<float *>(ws + plan.off_inner), *pair = reinterpret_cast<float *>(ws + plan.off_pair);
  const Sorted so(ws, plan, a.top_k);
  const Planes px(plan.off_x, plan.pass_rows, a.hidden), ph(px.end, room, a.inner);
  const int32_t *ids = a.ids + t0 * a.top_k;
  launch_timed(moe_sort_kernel, dim3(1), dim3(1024), 0u, s, ids, (int)pairs, a.experts, 128, so.order, so.place,
               so.count, so.tiles);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess) e = launch_planes(a.x + t0 * a.x_stride, a.x_stride, rows, nullptr, a.hidden, ws, px, s);
  if (e != hipSuccess) return e;
  auto run = [&](int type, bool gate_up, const MoeProduct &m, const Planes &p, int64_t n, float *y) {
    ExpertMat mat{};
    mat.w[0] = m.w[0];
    mat.w[1] = m.w[1];
    mat.w_bytes = m.w_bytes;
    mat.expert_bytes = m.expert_bytes;
    mat.order = so.order;
    mat.weights = a.weights + t0 * a.top_k;
    mat.y = y;
    mat.n = m.N;
    mat.row_bytes = m.row_bytes;
    mat.top_k = a.top_k;
    return launch_experts(type, gate_up, reinterpret_cast<_Float16 *>(ws + p.hi), reinterpret_cast<_Float16 *>(ws + p.lo),
                          ws + p.sums, reinterpret_cast<float *>(ws + p.rscale), (int)n, whole(m.K), mat, so.count, so.tiles,
                          expert_tiles(pairs, a.experts, 128), s);
  };
  MoeProduct g = product(a.gate_up_type, a.hidden, a.inner, a.experts);
  g.w[0] = a.gate;
  g.w[1] = a.up;
  e = run(a.gate_up_type, true, g, px, rows, inner);
  if (e == hipSuccess) e = launch_planes(inner, a.inner, pairs, so.count, a.inner, ws, ph, s);
  if (e != hipSuccess) return e;
  MoeProduct d = product(a.down_type, a.inner, a.hidden, a.experts);
  d.w[0] = a.down;
  e = run(a.down_type, false, d, ph, pairs, pair);
  if (e != hipSuccess) return e;
  return launch_sum(a, pair, ids, so.place, rows, 1, a.out + t0 * a.out_stride, s);
}

// The same with each expert's weights streamed past its rows.
static hipError_t stream_pass(const MoeArgs &a, const MoePlan &plan, uint8_t *ws, int64_t t0, int64_t rows, int cu_count,
                              hipStream_t s) {
  float *inner = reinterpret_cast<float *>(ws + plan.off_inner), *pair = reinterpret_cast<float *>(ws + plan.off_pair);
  MoeProduct g = product(a.gate_up_type, a.hidden, a.inner, a.experts);
  g.x = a.x + t0 * a.x_stride;
  g.x_stride = a.x_stride;
  g.share = a.top_k;
  g.w[0] = a.gate;
  g.w[1] = a.up;
  g.ids = a.ids + t0 * a.top_k;
  g.y = g.slices > 1 ? reinterpret_cast<float *>(ws + plan.off_x) : inner;
  g.pairs = (int)(rows * a.top_k);
  // One row's experts differ; of more rows', half of the experts' number still
  // mostly do (26 pairs of 8 experts, 4096 x 14336, unsorted: 590 us, most
  // workgroups having found an earlier pair of their expert; sorted: 300).  Where
  // they do not, the same happens: 64 pairs of one expert, 2048 x 768 of 128 in
  // Q4_K, 166 us, as many of different ones 51; 65 pairs, sorted, 35.
  if (g.pairs > kFewPairs || (rows > 1 && 2 * g.pairs > a.experts)) {
    const Sorted so(ws, plan, a.top_k);
    launch_timed(moe_sort_kernel, dim3(1), dim3(1024), 0u, s, g.ids, g.pairs, a.experts, 16, so.order, so.place, so.count,
                 so.tiles);
    const hipError_t sorted = hipGetLastError();
    if (sorted != hipSuccess) return sorted;
    g.order = so.order;
    g.count = so.count;
    g.jobs = so.tiles;
  }
  hipError_t e = launch_product<2>(a.gate_up_type, g, cu_count, s);
  if (e == hipSuccess && g.slices > 1) {  // (a pair without an expert: whatever lies there, which nothing reads)
    const int64_t n4 = (int64_t)g.pairs * a.inner / 4;
    launch_timed(moe_gate_kernel, dim3((unsigned)((n4 + 255) / 256)), dim3(256), 0u, s,
                 reinterpret_cast<const float4 *>(g.y), g.slices, n4, reinterpret_cast<float4 *>(inner));
    e = hipGetLastError();
  }
  if (e != hipSuccess) return e;
  MoeProduct d = product(a.down_type, a.inner, a.hidden, a.experts);
  d.x = inner;
  d.x_stride = a.inner;
  d.share = 1;
  d.w[0] = a.down;
  d.ids = g.ids;
  d.weights = a.weights + t0 * a.top_k;
  d.y = pair;
  d.pairs = g.pairs;
  d.order = g.order;
  d.count = g.count;
  d.jobs = g.jobs;
  e = launch_product<1>(a.down_type, d, cu_count, s);
  if (e != hipSuccess) return e;
  return launch_sum(a, pair, g.ids, nullptr, rows, d.slices, a.out + t0 * a.out_stride, s);
}

hipError_t launch_moe(const MoeArgs &a, const MoePlan &plan, void *workspace, int cu_count, hipStream_t s) {
  uint8_t *ws = static_cast<uint8_t *>(workspace);
  for (int64_t t0 = 0; t0 < a.rows; t0 += plan.pass_rows) {
    const int64_t rows = std::min<int64_t>(plan.pass_rows, a.rows - t0);
    const hipError_t e = plan.tiled ? tiled_pass(a, plan, ws, t0, rows, s) : stream_pass(a, plan, ws, t0, rows, cu_count, s);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace okq
