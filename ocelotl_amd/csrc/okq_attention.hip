// okq_attention.hip -- attention of one new token of each sequence over a
// paged key-value cache:
//   out = sum_t p_t V[t] / sum_t p_t,  p_t = exp(s_t - max s),
//   s_t = scale * q . K[t]  (softcap * tanh(s_t / softcap) where capped),
// over the visible tokens, in one pass with the running maximum and sum.
//
// attention_tiles_kernel: matrix instructions over tiles of cached rows, a
// long cache split over workgroups and joined by the last of them.
// attention_rows_kernel: rows that the tiles' vector loads do not reach
// (head_dim or addresses that are no multiple of 16 bytes, head_dim above
// 256), one value at a time; a split sequence is joined by a launch of its own.
#include <algorithm>
#include <type_traits>

#include "okq_device.h"
#include "okq_internal.h"

namespace okq {

namespace {

constexpr int kF32 = 0, kF16 = 1, kBF16 = 30;

// A score without its infinities: NaN in their place.  The products of an
// infinite key with a query's limbs are infinite or NaN, whichever the bits of
// the query make them, so the one rule for all caches is NaN.
__device__ __forceinline__ float finite_or_nan(float s) { return __builtin_fmaf(s, 0.0f, s); }

// Value i of a cached row.
template <int kType>
__device__ __forceinline__ float cached(const uint8_t *row, int i) {
  if constexpr (kType == kF32) return reinterpret_cast<const float *>(row)[i];
  if constexpr (kType == kQ8_0) return deq_elem(kQ8_0, row, (uint32_t)i);
  const uint16_t b = reinterpret_cast<const uint16_t *>(row)[i];
  return kType == kF16 ? f16_bits_hw(b) : as_f32((uint32_t)b << 16);
}

constexpr int kRowHeads = 4, kRowTokens = 4;
// As many waves as the registers of a row allow: one workgroup has all tokens.
constexpr int row_waves(int kV) { return kV <= 4 ? 16 : 8; }
// Where a chunk's results for a head begin: outputs, maximum, sum.
__device__ __forceinline__ int64_t row_part(unsigned block, int chunks, unsigned chunk, int h, int D) {
  return (((int64_t)block * chunks + chunk) * kRowHeads + h) * (D + 2);
}

}  // namespace

// A workgroup per sequence, kRowHeads query heads of a key/value head, which
// share its rows, and chunk of the sequence; its waves take kRowTokens tokens
// each in turn, a wave's lanes the row's values.  Any head_dim up to 64 kV, any
// alignment.  The waits for pages and rows bound it, so a wave asks for all its
// tokens' rows at once, and sequences are split, each into the same number of
// equal chunks, until there are two workgroups a CU (16 sequences of 2000
// tokens, 32 heads over 8, bf16: head_dim 512 170 us, 100 109; unsplit 282 and
// 170; token by token, a workgroup of four waves a head, 3986 and 928).  A
// chunk's outputs, maxima and sums go to `part`.
template <int kType, int kV>
__global__ __launch_bounds__(64 * row_waves(kV)) void attention_rows_kernel(AttnArgs a, int sets, float *part) {
  constexpr int kRowWaves = row_waves(kV);
  __shared__ float lds[kRowWaves][kRowHeads][64 * kV + 2];
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = (int)threadIdx.x & 63;
  const int D = a.cache.head_dim, pt = a.cache.page_tokens;
  const int set = (int)(blockIdx.x % (unsigned)sets), pair = (int)(blockIdx.x / (unsigned)sets);
  const int seq = pair / a.cache.kv_heads, kvh = pair - seq * a.cache.kv_heads;
  const int heads = a.group - set * kRowHeads < kRowHeads ? a.group - set * kRowHeads : kRowHeads;
  const int64_t h0 = (int64_t)kvh * a.group + set * kRowHeads;
  const uint8_t *kb = a.cache.k + (int64_t)kvh * a.cache.head_stride, *vb = a.cache.v + (int64_t)kvh * a.cache.head_stride;
  const int32_t *table = a.table + (int64_t)seq * a.table_width;
  float q[kRowHeads][kV], o[kRowHeads][kV], m[kRowHeads], l[kRowHeads];
#pragma unroll
  for (int h = 0; h < kRowHeads; ++h) {
#pragma unroll
    for (int j = 0; j < kV; ++j) {
      const int i = lane + 64 * j;
      q[h][j] = h < heads && i < D ? a.q[seq * a.q_stride + (h0 + h) * D + i] : 0.0f;
      o[h][j] = 0.0f;
    }
    m[h] = -INFINITY;
    l[h] = 0.0f;
  }
  int len = a.lengths[seq];
  len = len < a.max_len ? len : a.max_len;
  int lo = a.window && len > a.window ? len - a.window : 0;
  const int chunks = (int)gridDim.y;
  if (len > lo) {
    constexpr int kTurn = kRowWaves * kRowTokens;
    const int per = ((len - lo + kTurn - 1) / kTurn + chunks - 1) / chunks * kTurn;
    lo += per * (int)blockIdx.y;
    len = len - lo < per ? len : lo + per;  // may leave nothing
  }
  for (int t0 = lo + wave * kRowTokens; t0 < len; t0 += kRowWaves * kRowTokens) {
    bool seen[kRowTokens];
    float k[kRowTokens][kV], v[kRowTokens][kV];
    int64_t at[kRowTokens];
#pragma unroll
    for (int u = 0; u < kRowTokens; ++u) {  // tokens that are not seen read the cache's first row
      const int t = t0 + u < len ? t0 + u : len - 1, page = table[t / pt];
      seen[u] = t0 + u < len && (unsigned)page < (unsigned)a.cache.n_pages;
      at[u] = seen[u] ? page * a.cache.page_stride + t % pt * a.cache.token_stride : 0;
    }
#pragma unroll
    for (int u = 0; u < kRowTokens; ++u)
#pragma unroll
      for (int j = 0; j < kV; ++j) {
        const int i = lane + 64 * j;
        const float kx = cached<kType>(kb + at[u], i < D ? i : 0), vx = cached<kType>(vb + at[u], i < D ? i : 0);
        k[u][j] = i < D ? kx : 0.0f;
        v[u][j] = i < D && seen[u] ? vx : 0.0f;
      }
#pragma unroll
    for (int h = 0; h < kRowHeads; ++h) {
      float s[kRowTokens], top = m[h];
#pragma unroll
      for (int u = 0; u < kRowTokens; ++u) {
        float dot = 0.0f;
#pragma unroll
        for (int j = 0; j < kV; ++j) dot += q[h][j] * k[u][j];
        s[u] = finite_or_nan(wave_sum(dot)) * a.scale;
        if (a.softcap > 0.0f) s[u] = a.softcap * tanhf(s[u] / a.softcap);
        s[u] = seen[u] ? s[u] : -INFINITY;
        top = fmaxf(top, s[u]);
      }
      const float base = top == -INFINITY ? 0.0f : top, keep = expf(m[h] - base);
      m[h] = top;
      l[h] *= keep;
#pragma unroll
      for (int j = 0; j < kV; ++j) o[h][j] *= keep;
#pragma unroll
      for (int u = 0; u < kRowTokens; ++u) {
        const float p = expf(s[u] - base);
        l[h] += p;
#pragma unroll
        for (int j = 0; j < kV; ++j) o[h][j] += p * v[u][j];
      }
    }
  }
#pragma unroll
  for (int h = 0; h < kRowHeads; ++h) {
#pragma unroll
    for (int j = 0; j < kV; ++j) lds[wave][h][lane + 64 * j] = o[h][j];
    if (lane == 0) {
      lds[wave][h][64 * kV] = m[h];
      lds[wave][h][64 * kV + 1] = l[h];
    }
  }
  __syncthreads();
  for (int h = 0; h < heads; ++h) {
    float top = -INFINITY, sum = 0.0f, weight[kRowWaves];
#pragma unroll
    for (int w = 0; w < kRowWaves; ++w) top = fmaxf(top, lds[w][h][64 * kV]);
    const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int w = 0; w < kRowWaves; ++w) {
      weight[w] = expf(lds[w][h][64 * kV] - base);
      sum += lds[w][h][64 * kV + 1] * weight[w];
    }
    for (int i = (int)threadIdx.x; i < D; i += 64 * kRowWaves) {
      float x = 0.0f;
#pragma unroll
      for (int w = 0; w < kRowWaves; ++w) x += lds[w][h][i] * weight[w];
      if (chunks == 1) a.out[seq * a.out_stride + (h0 + h) * D + i] = sum == 0.0f ? 0.0f : x / sum;
      else part[row_part(blockIdx.x, chunks, blockIdx.y, h, D) + i] = x;
    }
    if (threadIdx.x == 0) {
      if (chunks > 1) {
        part[row_part(blockIdx.x, chunks, blockIdx.y, h, D) + D] = top;
        part[row_part(blockIdx.x, chunks, blockIdx.y, h, D) + D + 1] = sum;
      } else if (a.lse) {
        a.lse[(int64_t)seq * a.q_heads + h0 + h] = top == INFINITY ? top : base + logf(sum);
      }
    }
  }
}

// The chunks' results into one, in their order: a workgroup per first kernel's
// workgroup of a sequence and head.
__global__ __launch_bounds__(256) void attention_rows_join_kernel(AttnArgs a, int sets, int chunks, const float *part) {
  const int set = (int)(blockIdx.x % (unsigned)sets), pair = (int)(blockIdx.x / (unsigned)sets), h = (int)blockIdx.y;
  const int seq = pair / a.cache.kv_heads, kvh = pair - seq * a.cache.kv_heads, D = a.cache.head_dim;
  if (set * kRowHeads + h >= a.group) return;
  const int64_t head = (int64_t)kvh * a.group + set * kRowHeads + h;
  part += row_part(blockIdx.x, chunks, 0, h, D);
  const int64_t step = (int64_t)kRowHeads * (D + 2);
  float top = -INFINITY, sum = 0.0f, x[kMaxHeadDim / 256] = {};
  for (int c = 0; c < chunks; ++c) top = fmaxf(top, part[c * step + D]);
  const float base = top == -INFINITY ? 0.0f : top;
  for (int c = 0; c < chunks; ++c) {
    const float weight = expf(part[c * step + D] - base);
    sum += part[c * step + D + 1] * weight;
#pragma unroll
    for (int j = 0; j < kMaxHeadDim / 256; ++j) {
      const int i = (int)threadIdx.x + 256 * j;
      if (i < D) x[j] += part[c * step + i] * weight;
    }
  }
#pragma unroll
  for (int j = 0; j < kMaxHeadDim / 256; ++j) {
    const int i = (int)threadIdx.x + 256 * j;
    if (i < D) a.out[seq * a.out_stride + head * D + i] = sum == 0.0f ? 0.0f : x[j] / sum;
  }
  if (a.lse && threadIdx.x == 0) a.lse[(int64_t)seq * a.q_heads + head] = top == INFINITY ? top : base + logf(sum);
}


// ---- tiles ---------------------------------------------------------------------
//
// A wave takes tiles of 32 cached tokens (16 of f32) of one key/value head and
// the up to 16 query heads that read it, which share every cached byte.
//
//   S[token][head] = K Q^T        A = K: lane (token = l & 15, 8 dims from 8 (l >> 4))
//   O[dim][head]  += V^T P        B = P: lane (head = l & 15, 8 tokens of l >> 4)
//
// S leaves the matrix unit with lane (head = l & 15) holding tokens
// 4 (l >> 4) + 0..3 of each 16, which is what the second product wants as its
// B operand if tokens {4g..4g+3, 16+4g..16+4g+3} are called its k-slots
// 8g..8g+7: the probabilities never leave their lane.  Maxima, sums and the
// rescaling of O are per head, so per lane too.  V comes in rows (a lane takes
// 8 dims of its 8 tokens, 16 lanes a row's 128) and is turned by v_perm.
//
// The queries and probabilities are f32, the matrix instructions' operands 16
// bits: each is split into limbs whose sum is the f32 value -- three bf16
// (exactly; BF16 and Q8_0 caches), two f16 (to 2^-23, scaled by a power of two
// into f16's range; F16 caches) -- and each limb gets its product.  Over F16
// caches the second limb has a scale of its own, so do the weights of a tile
// and head, and those too small for it go in by themselves: a weight keeps its
// precision however far it lies below the largest (a token whose value is near
// zero may have that one).  The price is a sum per limb, added to O in f32: 24
// sequences, window 1024, head_dim 256, 14.6 us (13.8 with limbs of one scale),
// 517 tokens 8.3 (7.8), 131072 tokens 99.2 (98.6).  The cached values are exact
// operands as they are.  A tile's 48 products of bf16 take 768 cycles of the
// matrix unit against the 16 KB that a SIMD's share of the memory takes 7400
// cycles for.
//
// Q8_0 codes become bf16 exactly; a block's scale goes with its partial scores
// (they leave the matrix unit per block) and, for V, with P before the limbs:
// bf16 limbs have f32's range, so neither weights nor scales far below others
// lose bits.
//
// What bounds it: memory, once the cache is long (131072 tokens of 8 key/value
// heads of 128, bf16, 537 MB: 97 us, 5.5 TB/s; 64 ragged sequences of at most
// 8192, 268 MB: 54 us, 5.0 TB/s); Q8_0 what two waves a SIMD have in flight, as
// its rows come in pieces of 2 and 8 bytes, beside the instructions that decode
// them and split the weights block by block (131072 tokens, 285 MB: 75 us, 3.8
// TB/s; 68 with two f16 limbs, which lose small weights); a short cache the
// chain length -> page -> row -> result -> count -> join, each a trip to memory
// (517 tokens, 2 MB: 7.9 us).

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

namespace {

constexpr int kHeads = 16;            // query heads of a tile
constexpr int kWaves = 4;             // of a workgroup
constexpr int kThreads = 64 * kWaves;
constexpr int kPages = 512;           // pages that a workgroup holds the places of
constexpr float kGrowth = 8.0f;       // how far (in powers of two) weights may exceed 1 before O is rescaled
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

struct TileArgs {
  AttnArgs a;
  uint32_t page_mul, page_shift;  // token / page_tokens = umulhi(2 token, mul) >> shift
  uint32_t token_stride;
  int head_tiles;                 // tiles of kHeads query heads in a group
  float inv_units;
  int units;                      // chunks of all sequences together that the split aims at
  int min_tiles;                  // of a chunk
  int segment;                    // tokens, a multiple of the waves' tiles, of at most kPages pages
  uint32_t part_bytes;
  float *part;                    // a slot for each chunk of a split sequence and head tile: O, maxima, sums
  uint32_t *arrived;              // at a sequence's first slot: chunks that are done; zero between calls
};

constexpr int kGridY = 32768;

// ceil(a / b) with 1 / b at hand.  Exact while a < 2^22 or the quotient is
// below 2^20; past both it is off by less than 2^-22 of itself, which leaves a
// split uneven by that much, and the last chunk still ends with its sequence.
__device__ __forceinline__ int ceil_div(int a, int b, float inv_b) {
  int q = (int)(((float)a + (float)b - 0.5f) * inv_b);
  q += (int64_t)q * b < a ? 1 : 0;
  q -= (int64_t)(q - 1) * b >= a ? 1 : 0;
  return q;
}

// Inclusive sum over the lanes: within 16 lanes by shifts, then each row's last
// lane added to the rows after it.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast31 into rows 2 and 3
  return v;
}
__device__ __forceinline__ float cross_max(float v) {  // over the four 16-lane rows
  auto a = __builtin_amdgcn_permlane32_swap(as_u32(v), as_u32(v), false, false);
  v = fmaxf(as_f32(a[0]), as_f32(a[1]));
  a = __builtin_amdgcn_permlane16_swap(as_u32(v), as_u32(v), false, false);
  return fmaxf(as_f32(a[0]), as_f32(a[1]));
}
__device__ __forceinline__ float cross_sum(float v) {
  auto a = __builtin_amdgcn_permlane32_swap(as_u32(v), as_u32(v), false, false);
  v = as_f32(a[0]) + as_f32(a[1]);
  a = __builtin_amdgcn_permlane16_swap(as_u32(v), as_u32(v), false, false);
  return as_f32(a[0]) + as_f32(a[1]);
}
// Lane `kLane` of the own 16-lane row.
template <int kLane>
__device__ __forceinline__ float row_lane(float v) {
  return as_f32((uint32_t)__builtin_amdgcn_update_dpp(0, (int)as_u32(v), 0x150 + kLane, 0xf, 0xf, true));
}
__device__ __forceinline__ uint32_t hi16s(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }
__device__ __forceinline__ uint32_t lo16s(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }

// Eight f32 values as three bf16 limbs (cut off, so their sum is exact).
__device__ __forceinline__ void limbs_bf16(const float (&x)[8], u32x4 (&limb)[3]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float a = x[2 * j], b = x[2 * j + 1];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      limb[k][j] = hi16s(as_u32(a), as_u32(b));
      a -= as_f32(as_u32(a) & 0xffff0000u);
      b -= as_f32(as_u32(b) & 0xffff0000u);
    }
  }
}
// Eight f32 values below 2^14 as two f16 limbs, the second 2^11 times its
// worth, so that it has a range of its own: off by at most 2^-23 of the value
// from kLeast on, by 2^-36 below.  (A query's largest element is 2^13 to 2^14
// here: what is 2^26 times smaller is off by 2^-49 of the largest.)
constexpr float kApart = 2048.0f, kLeast = 0x1p-13f;
__device__ __forceinline__ void limbs_f16(const float (&x)[8], u32x4 (&limb)[2]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    f16x2 hi = {(_Float16)x[2 * j], (_Float16)x[2 * j + 1]};
    asm("" : "+v"(hi));  // one rounding for both uses
    const f16x2 lo = {(_Float16)((x[2 * j] - (float)hi[0]) * kApart), (_Float16)((x[2 * j + 1] - (float)hi[1]) * kApart)};
    limb[0][j] = __builtin_bit_cast(uint32_t, hi);
    limb[1][j] = __builtin_bit_cast(uint32_t, lo);
  }
}
// Two codes (byte kByte of each register) as bf16, which holds them exactly.
template <int kByte>
__device__ __forceinline__ uint32_t codes_bf16(uint32_t a, uint32_t b) {
  return hi16s(as_u32((float)(int8_t)(a >> (8 * kByte))), as_u32((float)(int8_t)(b >> (8 * kByte))));
}
template <int kFrom>  // of one register, bytes kFrom and kFrom + 1
__device__ __forceinline__ uint32_t pair_bf16(uint32_t v) {
  return hi16s(as_u32((float)(int8_t)(v >> (8 * kFrom))), as_u32((float)(int8_t)(v >> (8 * kFrom + 8))));
}
// A register whose upper half nothing reads (so that nothing clears it).
__device__ __forceinline__ uint32_t low_half(uint16_t v) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  const u16x2 w = {v, 0};
  return __builtin_bit_cast(uint32_t, __builtin_shufflevector(w, w, 0, -1));
}
// x[j] = p[j] * (lane j, or 8 + j, of the own row's d): a block's scales of the
// lane's eight token slots.
__device__ __forceinline__ void scale_slots(const float (&p)[8], float d, int upper, float (&x)[8]) {
  if (!upper) {
    x[0] = p[0] * row_lane<0>(d), x[1] = p[1] * row_lane<1>(d), x[2] = p[2] * row_lane<2>(d);
    x[3] = p[3] * row_lane<3>(d), x[4] = p[4] * row_lane<4>(d), x[5] = p[5] * row_lane<5>(d);
    x[6] = p[6] * row_lane<6>(d), x[7] = p[7] * row_lane<7>(d);
  } else {
    x[0] = p[0] * row_lane<8>(d), x[1] = p[1] * row_lane<9>(d), x[2] = p[2] * row_lane<10>(d);
    x[3] = p[3] * row_lane<11>(d), x[4] = p[4] * row_lane<12>(d), x[5] = p[5] * row_lane<13>(d);
    x[6] = p[6] * row_lane<14>(d), x[7] = p[7] * row_lane<15>(d);
  }
}
template <int kType>
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (kType != kF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma4(float a, float b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}
template <class T>
__device__ __forceinline__ T load_any(const void *p) {  // any alignment
  T v;
  __builtin_memcpy(&v, p, sizeof v);
  return v;
}

// tanh of a lane's values, off by at most 3 steps of 2^-24: below 0.625 an odd
// polynomial (towards the least largest relative error by Lawson's reweighted
// least squares; 8.2e-9 with its coefficients in f32), beyond 1 - 2 / (exp(2 |x|) + 1), which loses nothing there.  Scores are
// mostly far below their cap, and a wave without larger ones skips that half.
// (The library's tanhf, with branches a value, took 5 us of a 20 us call.)
template <int kN>
__device__ __forceinline__ void tanh_all(float (&x)[kN]) {
  float big = 0.0f;
#pragma unroll
  for (int j = 0; j < kN; ++j) big = __builtin_fmaxf(big, __builtin_fabsf(x[j]));
  const bool beyond = __ballot(!(big < 0.625f)) != 0;
#pragma unroll
  for (int j = 0; j < kN; ++j) {
    const float z = x[j] * x[j];
    float p = __builtin_fmaf(z, -5.7050843e-03f, 2.0639173e-02f);
    p = __builtin_fmaf(z, p, -5.3739741e-02f);
    p = __builtin_fmaf(z, p, 1.3331442e-01f);
    p = __builtin_fmaf(z, p, -3.3333282e-01f);
    float y = __builtin_fmaf(x[j] * z, p, x[j]);
    if (beyond) {
      const float a = __builtin_fabsf(x[j]);
      const float e = __builtin_amdgcn_exp2f(a * (2.0f * kLog2e));
      const float far = __builtin_copysignf(__builtin_fmaf(-2.0f, __builtin_amdgcn_rcpf(e + 1.0f), 1.0f), x[j]);
      y = a < 0.625f ? y : far;
    }
    x[j] = y;
  }
}

// Chunks' results go between workgroups past the XCDs' own L2 caches, by stores
// and loads of agent scope (kAgent); the writer waits for its stores
// (results_stored) before it counts itself done.  A release fence in their
// place writes the XCD's whole L2 back, for every wave: 303 us instead of 64 on
// a ragged batch of 64 sequences, 177 instead of 98 on one of 131072 tokens.
constexpr int kAgent = 16;  // sc1
__device__ __forceinline__ void results_stored() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

}  // namespace

template <int kType, int NC, bool kFull>  // head_dim <= 32 NC; kFull: equal
__global__ __launch_bounds__(kThreads, NC <= 4 ? 2 : 1) void attention_tiles_kernel(TileArgs ta) {
  constexpr bool kF = kType == kF32, kQ = kType == kQ8_0;
  constexpr int kL = kF ? 1 : kType == kF16 ? 2 : 3;             // limbs
  constexpr int kSub = kF ? 1 : 2;                                  // 16-token products of a tile
  constexpr int kTile = 16 * kSub, kSlots = 4 * kSub;               // tokens of a tile, of a lane
  constexpr int kStep = kWaves * kTile;
  constexpr int kQC = kF ? 2 * NC : NC, kPer = kF ? 4 : 8;          // chunks of 16 (f32) or 32 dims, a lane's dims of one
  // dims of a lane's load of V; Q8_0: two, so that a product's 16 rows (one
  // dim of each lane) lie in one block and its scales can go with P
  constexpr int kVD = kQ ? 2 : kF || NC <= 2 ? 4 : 8;
  constexpr int kVG = (32 * NC + 16 * kVD - 1) / (16 * kVD);        // such groups
  // Wide Q8_0 rows: loads of four dims, a 16-lane row's upper eight lanes those
  // of the next block, so a register holds two blocks: half the loads and
  // registers (4 sequences of 14563, 4 heads of 256: 47.4 us, in loads of two
  // dims 47.7).  At head_dim 128 loads of two dims are the faster ones, as most
  // of the four-byte loads lie across two words (131072 tokens: 74.7 us, 77.7).
  constexpr bool kPaired = kQ && NC > 4;
  constexpr int kVL = kPaired ? (NC + 1) / 2 : kVG;                 // a token's loads of V
  constexpr int kSB = (NC + 1) / 2;                                 // registers of Q8_0 scales
  constexpr bool kRegQ = NC <= (kQ ? 3 : 4);  // the queries' limbs in registers, every wave its own; else one copy in LDS
  constexpr int kQuads = NC <= 2 ? 16 : NC <= 4 ? 32 : 64;          // threads of a row of outputs, four values each
  __shared__ u32x4 q_lds[kRegQ ? 1 : kQC * kL * 64];
  constexpr int kMergeFloats = NC <= 4 ? 4096 : 8192;  // LDS for the waves' outputs
  __shared__ float merge[kMergeFloats];
  __shared__ int64_t offs[kWaves][2][kTile];
  __shared__ int64_t page_at[kPages];
  __shared__ float m_lds[kWaves][kHeads], l_lds[kWaves][kHeads];
  __shared__ int last;

  const AttnArgs &a = ta.a;
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int D = kFull ? 32 * NC : a.cache.head_dim, heads_kv = a.cache.kv_heads * ta.head_tiles;

  // ---- which chunk: all tiles in order, a sequence's shared out evenly over
  // its chunks; every wave counts them by itself
  const int head_at = (int)blockIdx.x, unit = (int)(blockIdx.z * (unsigned)kGridY + blockIdx.y);
  int tokens = 0, first = 0, tiles = 0;  // of sequence s0 + lane
  auto look = [&](int s0) {
    int len = s0 + lane < a.seqs ? a.lengths[s0 + lane] : 0;
    len = len < a.max_len ? len : a.max_len;
    len = len > 0 ? len : 0;
    first = a.window && len > a.window ? len - a.window : 0;
    tokens = len - first;
    tiles = (tokens + kTile - 1) / kTile;
  };
  int total = 0;
  for (int s0 = 0; s0 < a.seqs; s0 += 64) {
    look(s0);
    total += __builtin_amdgcn_readlane(wave_scan(tiles), 63);
  }
  int chunk = ceil_div(total, ta.units, ta.inv_units);
  chunk = (chunk + kWaves - 1) / kWaves * kWaves;  // a tile more for one wave costs what it costs for all
  chunk = chunk < ta.min_tiles ? ta.min_tiles : chunk;
  int seq = -1, at = 0, chunks = 0, slot = 0, lo = 0, hi = 0, before = 0, alone = 0;
  for (int s0 = 0; s0 < a.seqs; s0 += 64) {
    if (a.seqs > 64) look(s0);
    // A sequence's own chunks are not below half the root of its tiles: what
    // fewer tiles save each of them, the join of more chunks takes back (60000
    // tokens of one head: 17.6 us in 117 chunks, 32.6 in 469).
    int own = (int)(0.5f * __builtin_amdgcn_sqrtf((float)tiles));
    own = own > chunk ? (own + kWaves - 1) / kWaves * kWaves : chunk;
    const int c = s0 + lane >= a.seqs ? 0 : tiles > own ? ceil_div(tiles, own, __builtin_amdgcn_rcpf((float)own)) : 1;
    const int sum = wave_scan(c);
    const uint64_t who = __ballot(unit >= before + sum - c && unit < before + sum), ones = __ballot(c == 1);
    if (who) {
      const int w = __builtin_ctzll(who);
      seq = s0 + w;
      chunks = __builtin_amdgcn_readlane(c, w);
      slot = before + __builtin_amdgcn_readlane(sum - c, w);
      at = unit - slot;
      slot -= alone + __builtin_popcountll(ones & ((1ull << w) - 1));  // sequences of one chunk need no slot
      const int per = ceil_div(__builtin_amdgcn_readlane(tiles, w), chunks, __builtin_amdgcn_rcpf((float)chunks));
      const int begin = __builtin_amdgcn_readlane(first, w), end = begin + __builtin_amdgcn_readlane(tokens, w);
      lo = begin + at * per * kTile;
      hi = at == chunks - 1 || lo + per * kTile > end ? end : lo + per * kTile;
      break;
    }
    before += __builtin_amdgcn_readlane(sum, 63);
    alone += __builtin_popcountll(ones);
  }
  if (seq < 0) return;  // the split needs fewer workgroups than it may
  const int kvh = ta.head_tiles == 1 ? head_at : head_at / ta.head_tiles, ht = head_at - kvh * ta.head_tiles;
  const int heads = a.group - ht * kHeads < kHeads ? a.group - ht * kHeads : kHeads;
  const int h0 = kvh * a.group + ht * kHeads;

  // ---- loads of a tile: its rows' offsets (lane i the i-th token's) through
  // LDS; K in the A operand's order, V in rows.  Dims past head_dim repeat dim
  // 0 (their queries are zero, their outputs dropped).  A tile's K is requested
  // when the products of the tile before have read theirs, its V likewise: each
  // wait hides behind the other half.
  const int32_t *table = a.table + (int64_t)seq * a.table_width;
  const uint8_t *kb = a.cache.k + (int64_t)kvh * a.cache.head_stride, *vb = a.cache.v + (int64_t)kvh * a.cache.head_stride;
  const int pt = a.cache.page_tokens, mine = lane & (kTile - 1);
  auto page_of = [&](int t) { return (int)(__umulhi(2u * (uint32_t)t, ta.page_mul) >> ta.page_shift); };
  auto place = [&](int t0, int end, int page0, int buf) {  // the tile's offsets; a bit for each token that is not seen
    const int t = t0 + mine, page = page_of(t);
    const int64_t base = t < end ? page_at[page - page0] : -1;
    const bool in = base >= 0;
    const uint32_t within = (uint32_t)(t - page * pt) * ta.token_stride;
    if (lane < kTile) offs[wave][buf][lane] = in ? base + within : 0;
    wave_sync();
    return (uint32_t)__ballot(!in);  // lanes past kTile repeat
  };
  u32x4 kr[kSub][kQC], vr[kSlots][kVL];
  float dk[kSB], dv[kSB];  // Q8_0: scale of token slot n & 7, block 2 i + (n >> 3)
  auto scales = [&](const uint8_t *base, int buf, float (&d)[kSB]) {
    const uint8_t *row = base + offs[wave][buf][16 * ((n & 7) >> 2) + 4 * g + (n & 3)];
#pragma unroll
    for (int i = 0; i < kSB; ++i) {
      const bool there = kFull ? 2 * i + 1 < NC || n < 8 : 32 * (2 * i + (n >> 3)) < D;
      d[i] = f16_bits_hw(load_any<uint16_t>(row + (there ? kQ8Bytes * (2 * i + (n >> 3)) : 0)));
    }
  };
  auto load_k = [&](int buf) {
    if constexpr (kQ) scales(kb, buf, dk);
#pragma unroll
    for (int s = 0; s < kSub; ++s) {
      const uint8_t *row = kb + offs[wave][buf][16 * s + n];
      if constexpr (kQ) row += 2 + 8 * g;
#pragma unroll
      for (int c = 0; c < kQC; ++c) {
        if constexpr (kQ) {
          const u32x2 v = load_any<u32x2>(row + (kFull || 32 * c < D ? kQ8Bytes * c : 0));
          kr[s][c] = u32x4{v[0], v[1], 0, 0};
        } else {
          const int i = 4 * kPer * c + kPer * g;
          kr[s][c] = *reinterpret_cast<const u32x4 *>(row + (kFull || i < D ? i * (kF ? 4 : 2) : 0));
        }
      }
    }
  };
  auto load_v = [&](int buf) {
    if constexpr (kQ) scales(vb, buf, dv);
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      const uint8_t *row = vb + offs[wave][buf][16 * (j >> 2) + 4 * g + (j & 3)];
      if constexpr (kQ) row += 2 + (kPaired ? 4 * (n & 7) : 2 * n);
#pragma unroll
      for (int v = 0; v < kVL; ++v) {
        const int i = 16 * kVD * v + kVD * n, ii = (kFull && 32 * NC % (16 * kVD) == 0) || i < D ? i : 0;
        if constexpr (kQ && !kPaired) {
          vr[j][v] = u32x4{low_half(load_any<uint16_t>(row + (kFull || 32 * v < D ? kQ8Bytes * v : 0))), 0, 0, 0};
        } else if constexpr (kPaired) {
          const bool there = kFull ? 2 * v + 1 < NC || n < 8 : 32 * (2 * v + (n >> 3)) < D;
          vr[j][v] = u32x4{load_any<uint32_t>(row + (there ? kQ8Bytes * (2 * v + (n >> 3)) : 0)), 0, 0, 0};
        } else if constexpr (kF || kVD == 8) {
          vr[j][v] = *reinterpret_cast<const u32x4 *>(row + ii * (kF ? 4 : 2));
        } else {
          const u32x2 w = *reinterpret_cast<const u32x2 *>(row + ii * 2);
          vr[j][v] = u32x4{w[0], w[1], 0, 0};
        }
      }
    }
  };

  // ---- queries, requested before the first rows: the product's B operand,
  // lane (head n, dims kPer g on of every chunk)
  constexpr int kMy = kRegQ ? kQC : (kQC + kWaves - 1) / kWaves;  // a wave's chunks
  const float *q = a.q + (int64_t)seq * a.q_stride + (int64_t)h0 * D;
  float x[kMy][kPer];
#pragma unroll
  for (int u = 0; u < kMy; ++u)
#pragma unroll
    for (int j = 0; j < kPer; j += 4) {
      const int i = 4 * kPer * (kRegQ ? u : wave + u * kWaves) + kPer * g + j;
      // heads and dims that are not there read others, and become zero below
      const f32x4 v = load_any<f32x4>(q + (int64_t)(n < heads ? n : 0) * D + (i < D ? i : 0));
#pragma unroll
      for (int e = 0; e < 4; ++e) x[u][j + e] = v[e];
    }
  u32x4 ql[kRegQ ? kQC : 1][kL];
  auto query = [&](int c, int k) { return kRegQ ? ql[c][k] : q_lds[(c * kL + k) * 64 + lane]; };
  // of this lane's head: scores times this are powers of two, or a share of the cap
  float to_log2 = a.softcap > 0.0f ? a.scale / a.softcap : a.scale * kLog2e;
  const float cap = a.softcap * kLog2e;

  f32x4 o[kVG * kVD];
#pragma unroll
  for (int t = 0; t < kVG * kVD; ++t) o[t] = f32x4{0, 0, 0, 0};
  float m = -INFINITY, l = 0.0f;
  for (int seg = lo; seg < hi; seg += ta.segment) {
    const int end = hi - seg < ta.segment ? hi : seg + ta.segment;
    const int page0 = page_of(seg), pages = page_of(end - 1) - page0 + 1;
    if (seg > lo) __syncthreads();
    for (int i = tid; i < pages; i += kThreads) {
      const int page = table[page0 + i];
      page_at[i] = (unsigned)page < (unsigned)a.cache.n_pages ? page * a.cache.page_stride : -1;
    }
    __syncthreads();
    int t0 = seg + wave * kTile, buf = 0;
    uint32_t hidden = 0;
    // the queries are here (they were asked for before the pages): said so
    // that their use after the next loads waits for nothing
    auto settled = [&]() {
#pragma unroll
      for (int u = 0; u < kMy; ++u)
#pragma unroll
        for (int j = 0; j < kPer; ++j) asm volatile("" : "+v"(x[u][j]));
    };
    settled();
    if (t0 < end) {
      hidden = place(t0, end, page0, 0);
      load_k(0);
      load_v(0);
    }
    if (seg == lo) {
      settled();  // and not used before the first rows are requested
#pragma unroll
      for (int u = 0; u < kMy; ++u)
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          const bool there = n < heads && (kFull || 4 * kPer * (kRegQ ? u : wave + u * kWaves) + kPer * g + j < D);
          x[u][j] = there ? x[u][j] : 0.0f;
        }
      if constexpr (kType == kF16) {  // f16 limbs: every head's largest value just below 2^14
        float mx = 0.0f;
#pragma unroll
        for (int u = 0; u < kMy; ++u)
#pragma unroll
          for (int j = 0; j < kPer; ++j) mx = __builtin_fmaxf(mx, __builtin_fabsf(x[u][j]));
        mx = cross_max(mx);
        if constexpr (!kRegQ) {
          if (g == 0) m_lds[wave][n] = mx;
          __syncthreads();
#pragma unroll
          for (int w = 0; w < kWaves; ++w) mx = __builtin_fmaxf(mx, m_lds[w][n]);
        }
        const int e = mx > 0.0f && mx < INFINITY ? 14 - __builtin_amdgcn_frexp_expf(mx) : 0;
        to_log2 = ldexpf(to_log2, -e);
#pragma unroll
        for (int u = 0; u < kMy; ++u)
#pragma unroll
          for (int j = 0; j < kPer; ++j) x[u][j] = ldexpf(x[u][j], e);
      }
#pragma unroll
      for (int u = 0; u < kMy; ++u) {
        u32x4 limb[kL];
        if constexpr (kF) limb[0] = u32x4{as_u32(x[u][0]), as_u32(x[u][1]), as_u32(x[u][2]), as_u32(x[u][3])};
        else if constexpr (kType == kF16) limbs_f16(x[u], limb);
        else limbs_bf16(x[u], limb);
#pragma unroll
        for (int k = 0; k < kL; ++k) {
          if constexpr (kRegQ) ql[u][k] = limb[k];
          else if (wave + u * kWaves < kQC) q_lds[((wave + u * kWaves) * kL + k) * 64 + lane] = limb[k];
        }
      }
      if constexpr (!kRegQ) __syncthreads();
    }
    while (t0 < end) {
      const bool more = t0 + kStep < end;
      uint32_t hidden_next = 0;
      if (more) hidden_next = place(t0 + kStep, end, page0, buf ^ 1);
      // scores
      float p[kSlots];
      if constexpr (kQ) {  // a block's products, times its keys' scales
#pragma unroll
        for (int j = 0; j < kSlots; ++j) p[j] = 0.0f;
        // A block's products are folded in behind the next block's.  pinned()
        // keeps the folding there: left to itself it moves behind all blocks,
        // whose products and scales then need more registers than there are.
        float b[2][8];
        auto fold = [&](int c) {
          float y[8];
          scale_slots(b[c & 1], dk[c >> 1], c & 1, y);
#pragma unroll
          for (int j = 0; j < kSlots; ++j) p[j] += y[j];
        };
#pragma unroll
        for (int c = 0; c < kQC; ++c) {
#pragma unroll
          for (int s = 0; s < kSub; ++s) {
            u32x4 op;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              op[2 * w] = pair_bf16<0>(kr[s][c][w]);
              op[2 * w + 1] = pair_bf16<2>(kr[s][c][w]);
            }
            f32x4 t = {0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < kL; ++k) t = mfma<kType>(op, query(c, k), t);
#pragma unroll
            for (int i = 0; i < 4; ++i) b[c & 1][4 * s + i] = t[i];
          }
          if (c > 0) fold(c - 1);
#pragma unroll
          for (int j = 0; j < kSlots; ++j) asm volatile("" : "+v"(p[j]));
          __builtin_amdgcn_sched_barrier(0);  // a block at a time: all at once spill
        }
        fold(kQC - 1);
      } else {
        constexpr int kAcc = kF ? 4 : kL;  // one sum a limb, or a quarter of the dims: products that do not wait for each other
        f32x4 part[kSub][kAcc];
#pragma unroll
        for (int s = 0; s < kSub; ++s)
#pragma unroll
          for (int k = 0; k < kAcc; ++k) part[s][k] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < kQC; ++c)
#pragma unroll
          for (int k = 0; k < kL; ++k) {
            const u32x4 qq = query(c, k);
#pragma unroll
            for (int s = 0; s < kSub; ++s) {
              if constexpr (kF) {
#pragma unroll
                for (int e = 0; e < 4; ++e) part[s][e] = mfma4(as_f32(kr[s][c][e]), as_f32(qq[e]), part[s][e]);
              } else {
                part[s][k] = mfma<kType>(kr[s][c], qq, part[s][k]);
              }
            }
          }
#pragma unroll
        for (int s = 0; s < kSub; ++s) {
          f32x4 acc = part[s][kAcc - 1];
#pragma unroll
          for (int k = kAcc - 2; k >= 0; --k) acc = kType == kF16 ? acc * (1.0f / kApart) + part[s][k] : acc + part[s][k];
#pragma unroll
          for (int i = 0; i < 4; ++i) p[4 * s + i] = acc[i];
        }
      }
      if (more) load_k(buf ^ 1);
#pragma unroll
      for (int j = 0; j < kSlots; ++j) p[j] = finite_or_nan(p[j]) * to_log2;
      if (a.softcap > 0.0f) {
        tanh_all(p);
#pragma unroll
        for (int j = 0; j < kSlots; ++j) p[j] *= cap;
      }
      if (hidden) {  // no weight, and values that are zero whatever the memory holds
        const uint32_t own = hidden >> (4 * g);
#pragma unroll
        for (int j = 0; j < kSlots; ++j) {
          const bool out = own >> (16 * (j >> 2) + (j & 3)) & 1u;
          p[j] = out ? -INFINITY : p[j];
#pragma unroll
          for (int v = 0; v < kVL; ++v)
            if constexpr (!kQ) vr[j][v] = out ? u32x4{0, 0, 0, 0} : vr[j][v];
        }
        if constexpr (kQ) {
          const bool out = own >> (16 * ((n & 7) >> 2) + (n & 3)) & 1u;
#pragma unroll
          for (int i = 0; i < kSB; ++i) dv[i] = out ? 0.0f : dv[i];
        }
      }
      float top = p[0];
#pragma unroll
      for (int j = 1; j < kSlots; ++j) top = __builtin_fmaxf(top, p[j]);
      top = cross_max(top);
      const float tile_top = top;
      if (__ballot(top > m + kGrowth) != 0) {
        top = __builtin_fmaxf(m, top);
        const float f = __builtin_amdgcn_exp2f(m - (top == -INFINITY ? 0.0f : top));
        m = top;
        l *= f;
#pragma unroll
        for (int t = 0; t < kVG * kVD; ++t) o[t] *= f;
      }
      const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
      for (int j = 0; j < kSlots; ++j) {
        p[j] = __builtin_amdgcn_exp2f(p[j] - base);
        l += p[j];
      }
      // outputs
      if constexpr (kF) {
#pragma unroll
        for (int v = 0; v < kVG; ++v)
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[4 * v + e] = mfma4(as_f32(vr[j][v][e]), p[j], o[4 * v + e]);
      } else if constexpr (kQ) {
        // of a pair of blocks, lanes below 8 keep the lower two dims, those above
        // the upper: the rest is swapped between them
        const uint32_t halves = n < 8 ? 0x05040100u : 0x03020706u;
        uint32_t codes[kSlots];  // two dims' codes of block v in bytes 0 and 1, of a pair's second in bytes 2 and 3
#pragma unroll
        for (int v = 0; v < kVG; ++v) {  // block v
#pragma unroll
          for (int j = 0; j < kSlots; ++j) {
            if constexpr (!kPaired) {
              codes[j] = vr[j][v][0];
            } else if (v % 2 == 0) {
              const uint32_t x = vr[j][v / 2][0];
              codes[j] = __builtin_amdgcn_perm((uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x128, 0xf, 0xf, true), x, halves);
            }
          }
          float y[8];
          scale_slots(p, dv[v >> 1], v & 1, y);
          u32x4 limb[kL];
          limbs_bf16(y, limb);
          u32x4 op[2];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const bool second = kPaired && v % 2 != 0;
            op[0][j] = second ? codes_bf16<2>(codes[2 * j], codes[2 * j + 1]) : codes_bf16<0>(codes[2 * j], codes[2 * j + 1]);
            op[1][j] = second ? codes_bf16<3>(codes[2 * j], codes[2 * j + 1]) : codes_bf16<1>(codes[2 * j], codes[2 * j + 1]);
          }
#pragma unroll
          for (int k = 0; k < kL; ++k)
#pragma unroll
            for (int d = 0; d < 2; ++d) o[2 * v + d] = mfma<kType>(op[d], limb[k], o[2 * v + d]);
          __builtin_amdgcn_sched_barrier(0);
        }
      } else {
        // Two f16 limbs hold a weight that is at least kLeast, so F16's weights
        // go in scaled by a power of two, their tile's and head's own (the
        // largest is 2^13 to 2^14), and what is still smaller, 26 powers of two
        // below its tile's largest, waits for another turn: a weight is off by
        // 2^-23 of itself, however far below the largest it is.
        float x[kSlots], down = 1.0f;
#pragma unroll
        for (int j = 0; j < kSlots; ++j) x[j] = p[j];
        if constexpr (kType == kF16) {
          const int e = 13 - (int)__builtin_floorf(__builtin_fmaxf(tile_top - base, -100.0f));
          const float up = ldexpf(1.0f, e);
          down = ldexpf(1.0f, -e);
#pragma unroll
          for (int j = 0; j < kSlots; ++j) x[j] *= up;
        }
        for (;;) {
          float later[kSlots];
          bool again = false;
          if constexpr (kType == kF16) {
            uint32_t least = ~0u;  // zeros and NaN do not count
#pragma unroll
            for (int j = 0; j < kSlots; ++j) least = min(least, as_u32(x[j]) - 1u);
            again = __ballot(least < as_u32(kLeast) - 1u) != 0;
            if (again) {
#pragma unroll
              for (int j = 0; j < kSlots; ++j) {
                const bool small = x[j] < kLeast;
                later[j] = small ? x[j] * 0x1p26f : 0.0f;
                x[j] = small ? 0.0f : x[j];
              }
            }
          }
          u32x4 limb[kL];
          if constexpr (kType == kBF16) limbs_bf16(x, limb);
          else limbs_f16(x, limb);
#pragma unroll
          for (int v = 0; v < kVG; ++v)
#pragma unroll
            for (int d0 = 0; d0 < kVD; d0 += 4) {
              // not turned for all turns at once, before the loop: too many registers
              if constexpr (kType == kF16) {
#pragma unroll
                for (int j = 0; j < kSlots; ++j) {
                  asm volatile("" : "+v"(vr[j][v][d0 / 2]));
                  asm volatile("" : "+v"(vr[j][v][d0 / 2 + 1]));
                }
              }
              u32x4 op[4];
#pragma unroll
              for (int d = 0; d < 4; ++d)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  const uint32_t lower = vr[2 * j][v][(d0 + d) / 2], upper = vr[2 * j + 1][v][(d0 + d) / 2];
                  op[d][j] = d & 1 ? hi16s(lower, upper) : lo16s(lower, upper);
                }
              f32x4 *acc = o + v * kVD + d0;
              if constexpr (kType == kBF16) {
#pragma unroll
                for (int k = 0; k < kL; ++k)
#pragma unroll
                  for (int d = 0; d < 4; ++d) acc[d] = mfma<kType>(op[d], limb[k], acc[d]);
              } else {
                f32x4 t[kL][4];
#pragma unroll
                for (int k = 0; k < kL; ++k)
#pragma unroll
                  for (int d = 0; d < 4; ++d) t[k][d] = mfma<kType>(op[d], limb[k], f32x4{0, 0, 0, 0});
#pragma unroll
                for (int d = 0; d < 4; ++d)
#pragma unroll
                  for (int i = 0; i < 4; ++i)
                    acc[d][i] = __builtin_fmaf(t[0][d][i], down, __builtin_fmaf(t[1][d][i], down * (1.0f / kApart), acc[d][i]));
              }
            }
          if (!again) break;
#pragma unroll
          for (int j = 0; j < kSlots; ++j) x[j] = later[j];
          down *= 0x1p-26f;
        }
      }
      if (!more) break;
      buf ^= 1;
      load_v(buf);
      hidden = hidden_next;
      t0 += kStep;
    }
  }

  // ---- the waves' results into one
  l = cross_sum(l);
  if (g == 0) {
    m_lds[wave][n] = m;
    l_lds[wave][n] = l;
  }
  const int DS = D + 4, fit = kMergeFloats / (kWaves * DS);  // heads that fit at once
  const int slot_floats = ((a.group < kHeads ? a.group : kHeads) * (D + 2) + 3) / 4 * 4;
  const auto part = __builtin_amdgcn_make_buffer_rsrc(ta.part, 0, (int)ta.part_bytes, 0x00020000);
  const uint32_t origin = 4u * ((uint32_t)slot * heads_kv + head_at) * slot_floats, step = 4u * heads_kv * slot_floats;
  float *out = a.out + (int64_t)seq * a.out_stride + (int64_t)h0 * D;
  float *lse = a.lse ? a.lse + (int64_t)seq * a.q_heads + h0 : nullptr;
  constexpr int kRows = kThreads / kQuads;  // rows of outputs that the threads hold at once
  const int row = tid / kQuads, quad = tid % kQuads;
  auto finish = [&](int h, f32x4 v, float top, float sum) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = sum == 0.0f ? 0.0f : v[i] / sum;
    __builtin_memcpy(out + h * D + 4 * quad, &v, sizeof v);
    if (lse && quad == 0) lse[h] = sum == 0.0f ? -INFINITY : ((top == -INFINITY ? 0.0f : top) + __builtin_amdgcn_logf(sum)) * kLn2;
  };
  for (int p0 = 0; p0 < heads; p0 += fit) {
    const int count = heads - p0 < fit ? heads - p0 : fit;
    if (p0 > 0) __syncthreads();
    if (n >= p0 && n < p0 + count) {
      float *to = merge + (wave * fit + n - p0) * DS;
#pragma unroll
      for (int v = 0; v < kVG; ++v)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 4 * g + i, dim = 16 * kVD * v + (kPaired ? 4 * (r & 7) + 2 * (r >> 3) : kVD * r);
          if constexpr (kQ) {
            if (!kFull && dim >= D) continue;
            to[dim] = o[v * kVD][i];
            to[dim + 1] = o[v * kVD + 1][i];
          } else {
#pragma unroll
            for (int d = 0; d < kVD; d += 4)
              if ((kFull && 32 * NC % (16 * kVD) == 0) || dim + d < D)
                *reinterpret_cast<f32x4 *>(to + dim + d) = f32x4{o[v * kVD + d][i], o[v * kVD + d + 1][i],
                                                                 o[v * kVD + d + 2][i], o[v * kVD + d + 3][i]};
          }
        }
    }
    __syncthreads();
    for (int h = p0 + row; h < p0 + count; h += kRows) {
      if (4 * quad >= D) break;
      float top = m_lds[0][h], sum = 0.0f;
#pragma unroll
      for (int w = 1; w < kWaves; ++w) top = __builtin_fmaxf(top, m_lds[w][h]);
      const float base = top == -INFINITY ? 0.0f : top;
      f32x4 v = {0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float weight = __builtin_amdgcn_exp2f(m_lds[w][h] - base);
        sum += weight * l_lds[w][h];
        v += weight * *reinterpret_cast<const f32x4 *>(merge + (w * fit + h - p0) * DS + 4 * quad);
      }
      if (chunks == 1) {
        finish(h, v, top, sum);
      } else {
        const uint32_t mine_at = origin + (uint32_t)at * step;
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), part, mine_at + 4 * (h * D + 4 * quad), 0, kAgent);
        if (quad == 0) {
          __builtin_amdgcn_raw_buffer_store_b32(as_u32(top), part, mine_at + 4 * (heads * D + h), 0, kAgent);
          __builtin_amdgcn_raw_buffer_store_b32(as_u32(sum), part, mine_at + 4 * (heads * D + heads + h), 0, kAgent);
        }
      }
    }
  }
  if (chunks == 1) return;

  // ---- the chunks' results into one, by the workgroup that finishes last, in
  // the chunks' order
  results_stored();
  __syncthreads();
  uint32_t *arrived = ta.arrived + (int64_t)slot * heads_kv + head_at;
  if (tid == 0)
    last = __hip_atomic_fetch_add(arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)chunks - 1;
  __syncthreads();
  if (!last) return;
  if (tid == 0) __hip_atomic_store(arrived, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  // Where the rows are fewer than the threads hold, teams of rows take every
  // teams-th chunk, with a running maximum and sum of their own, and meet in LDS.
  const int teams = heads >= kRows ? 1 : kRows / heads, team = heads >= kRows ? 0 : row * (256 / heads + 1) >> 8;
  for (int h = row - team * heads; h < heads; h += kRows) {
    f32x4 v = {0, 0, 0, 0};
    float top = -INFINITY, sum = 0.0f;
    // n chunks requested together: with four a wait each, a join of 123 takes
    // 8 us more than with sixteen, one of five 0.5 us less
    auto gather = [&](auto count, int i0) {
      constexpr int kN = decltype(count)::value;
      float mi[kN], li[kN];
      f32x4 vi[kN];
#pragma unroll
      for (int u = 0; u < kN; ++u) {
        int i = i0 + u * teams;
        mi[u] = -INFINITY, li[u] = 0.0f, vi[u] = f32x4{0, 0, 0, 0};
        if (kN > 4 && i >= chunks) continue;
        i = i < chunks ? i : i0;
        const uint32_t from = origin + (uint32_t)i * step;
        mi[u] = as_f32(__builtin_amdgcn_raw_buffer_load_b32(part, from + 4 * (heads * D + h), 0, kAgent));
        li[u] = as_f32(__builtin_amdgcn_raw_buffer_load_b32(part, from + 4 * (heads * D + heads + h), 0, kAgent));
        vi[u] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(part, from + 4 * (h * D + 4 * quad), 0, kAgent));
      }
      float most = top;
#pragma unroll
      for (int u = 0; u < kN; ++u) {
        if (kN <= 4 && i0 + u * teams >= chunks) mi[u] = -INFINITY, li[u] = 0.0f, vi[u] = f32x4{0, 0, 0, 0};
        most = __builtin_fmaxf(most, mi[u]);
      }
      const float base = most == -INFINITY ? 0.0f : most, keep = __builtin_amdgcn_exp2f(top - base);
      v *= keep;
      sum *= keep;
      top = most;
#pragma unroll
      for (int u = 0; u < kN; ++u) {
        const float w = __builtin_amdgcn_exp2f(mi[u] - base);
        sum += w * li[u];
        v += w * vi[u];
      }
    };
    if (team < teams && 4 * quad < D) {
      if (chunks <= 4 * teams) {
        if (team < chunks) gather(std::integral_constant<int, 4>{}, team);
      } else {
        for (int i0 = team; i0 < chunks; i0 += 16 * teams) gather(std::integral_constant<int, 16>{}, i0);
      }
    }
    if (teams > 1) {  // every row here once
      f32x4 *joined = reinterpret_cast<f32x4 *>(merge);
      joined[tid] = v;
      merge[4 * kThreads + 2 * tid] = top;
      merge[4 * kThreads + 2 * tid + 1] = sum;
      __syncthreads();
      if (team > 0) return;
      float most = top;
      for (int t = 1; t < teams; ++t) most = __builtin_fmaxf(most, merge[4 * kThreads + 2 * (tid + t * heads * kQuads)]);
      const float base = most == -INFINITY ? 0.0f : most, keep = __builtin_amdgcn_exp2f(top - base);
      v *= keep;
      sum *= keep;
      for (int t = 1; t < teams; ++t) {
        const int from = tid + t * heads * kQuads;
        const float w = __builtin_amdgcn_exp2f(merge[4 * kThreads + 2 * from] - base);
        sum += w * merge[4 * kThreads + 2 * from + 1];
        v += w * joined[from];
      }
      top = most;
    }
    if (team == 0 && 4 * quad < D) finish(h, v, top, sum);
  }
}

namespace {

template <int kType, int NC>
void launch_tiles(const TileArgs &ta, dim3 grid, hipStream_t s) {
  if (ta.a.cache.head_dim == 32 * NC) launch_timed(attention_tiles_kernel<kType, NC, true>, grid, dim3(kThreads), 0u, s, ta);
  else launch_timed(attention_tiles_kernel<kType, NC, false>, grid, dim3(kThreads), 0u, s, ta);
}
template <int kType>
void launch_tiles(const TileArgs &ta, dim3 grid, hipStream_t s) {
  const int D = ta.a.cache.head_dim;
  if (D <= 64) launch_tiles<kType, 2>(ta, grid, s);
  else if (D <= 96) launch_tiles<kType, 3>(ta, grid, s);
  else if (D <= 128) launch_tiles<kType, 4>(ta, grid, s);
  else launch_tiles<kType, 8>(ta, grid, s);
}

template <int kType>
void launch_rows(const AttnArgs &a, int chunks, float *part, hipStream_t s) {
  const int sets = (a.group + kRowHeads - 1) / kRowHeads;
  const unsigned pairs = (unsigned)(a.seqs * a.cache.kv_heads * sets);
  auto run = [&](auto kernel, int waves) {
    launch_timed(kernel, dim3(pairs, (unsigned)chunks), dim3(64 * waves), 0u, s, a, sets, part);
  };
  if (a.cache.head_dim <= 128) run(attention_rows_kernel<kType, 2>, row_waves(2));
  else if (a.cache.head_dim <= 256) run(attention_rows_kernel<kType, 4>, row_waves(4));
  else run(attention_rows_kernel<kType, 8>, row_waves(8));
  if (chunks > 1) launch_timed(attention_rows_join_kernel, dim3(pairs, kRowHeads), dim3(256), 0u, s, a, sets, chunks, (const float *)part);
}

}  // namespace

AttnPlan attention_plan(const AttnArgs &a, int cu_count) {
  AttnPlan p{};
  const KvPages &c = a.cache;
  const uint64_t strides = (uint64_t)(c.page_stride | c.head_stride | c.token_stride);
  const bool aligned = ((reinterpret_cast<uintptr_t>(c.k) | reinterpret_cast<uintptr_t>(c.v) | strides) & 15u) == 0;
  const uint64_t page = (uint64_t)c.token_stride * (uint64_t)c.page_tokens;  // 32-bit offsets within a page
  p.tiles = c.head_dim <= 256 && c.token_stride < (1ll << 32) && page < (1ull << 32) &&
            (c.type == kQ8_0 || (aligned && c.head_dim % (c.type == kF32 ? 4 : 8) == 0));
  if (!p.tiles) {
    // chunks of four turns of a workgroup's waves at least
    const int64_t pairs = (int64_t)a.seqs * c.kv_heads * ((a.group + kRowHeads - 1) / kRowHeads), most = 2 * (int64_t)cu_count;
    const int64_t turn = row_waves(c.head_dim <= 256 ? 4 : 8) * kRowTokens;
    p.units = (int)std::max<int64_t>(1, std::min(most / pairs, a.max_len / (4 * turn)));
    p.splits = p.units > 1;
    p.part_bytes = (size_t)(most * kRowHeads * (c.head_dim + 2)) * sizeof(float);
    return p;
  }
  const int tile = c.type == kF32 ? 16 : 32, head_tiles = (a.group + kHeads - 1) / kHeads;
  const int64_t pairs = (int64_t)c.kv_heads * head_tiles, most = ((int64_t)a.max_len + tile - 1) / tile;
  // workgroups that run at once: above head_dim 128 a wave takes more than half
  // of a SIMD's registers (held to half, 4 sequences of 14563 tokens of Q8_0 and
  // 4 heads of 256 take 77.4 us for 47.7)
  const int64_t aim = (c.head_dim <= 128 ? 2 : 1) * (int64_t)cu_count;
  // All chunks (units + seqs a head at most) at once where the sequences leave
  // room for that.  Where they do not, the card is full without a split, which
  // then only evens its end: twice as many units, but none of fewer than four
  // tiles a wave (64 sequences of 500 tokens: 27.4 us whole, 34.7 in halves).
  const int64_t units = aim / pairs;
  const bool room = a.seqs <= units / 2;
  p.units = (int)std::max<int64_t>(1, room ? units - a.seqs : 2 * units);
  p.min_tiles = room ? kWaves : 4 * kWaves;
  const int64_t chunks = std::max<int64_t>(1, (most + p.min_tiles - 1) / p.min_tiles);
  p.splits = chunks > 1 && p.units > 1;  // one unit: every sequence is one chunk
  p.grid = p.splits ? std::min<int64_t>(a.seqs + p.units + 1, a.seqs * chunks) : a.seqs;
  if (units >= 1) {  // the same for every call of these heads: slots for the most units
    const size_t slots = (size_t)(2 * (2 * units + 1) * pairs);
    p.arrived_bytes = slots * sizeof(uint32_t);
    p.part_bytes = slots * (size_t)((std::min(a.group, kHeads) * (c.head_dim + 2) + 3) / 4 * 4) * sizeof(float);
  }
  return p;
}

hipError_t launch_attention(const AttnArgs &a, const AttnPlan &p, void *part, void *arrived, hipStream_t s) {
  if (!p.tiles) {
    float *rows = static_cast<float *>(part);
    if (a.cache.type == kF32) launch_rows<kF32>(a, p.units, rows, s);
    else if (a.cache.type == kF16) launch_rows<kF16>(a, p.units, rows, s);
    else if (a.cache.type == kBF16) launch_rows<kBF16>(a, p.units, rows, s);
    else launch_rows<kQ8_0>(a, p.units, rows, s);
    return hipGetLastError();
  }
  // token / page_tokens for tokens below 2^31: floor(2^(31 + n) / d) + 1 with
  // 2^n >= d, times the token, loses nothing above bit 31 + n
  const uint32_t d = (uint32_t)a.cache.page_tokens;
  uint32_t n = 0;
  while (((uint64_t)1 << n) < d) ++n;
  const int tile = a.cache.type == kF32 ? 16 : 32, step = kWaves * tile;
  TileArgs ta{};
  ta.a = a;
  ta.page_mul = (uint32_t)(((uint64_t)1 << (31 + n)) / d + 1);
  ta.page_shift = n;
  ta.token_stride = (uint32_t)a.cache.token_stride;
  ta.head_tiles = (a.group + kHeads - 1) / kHeads;
  ta.units = p.units;
  ta.inv_units = 1.0f / (float)p.units;
  ta.min_tiles = p.min_tiles;
  ta.segment = (int)(std::min<int64_t>((int64_t)(kPages - 2) * d, 1 << 30) / step * step);
  ta.part_bytes = (uint32_t)p.part_bytes;
  ta.part = static_cast<float *>(part);
  ta.arrived = static_cast<uint32_t *>(arrived);
  const unsigned y = (unsigned)std::min<int64_t>(p.grid, kGridY);
  const dim3 grid((unsigned)(a.cache.kv_heads * ta.head_tiles), y, (unsigned)((p.grid + y - 1) / y));
  if (a.cache.type == kF32) launch_tiles<kF32>(ta, grid, s);
  else if (a.cache.type == kF16) launch_tiles<kF16>(ta, grid, s);
  else if (a.cache.type == kBF16) launch_tiles<kBF16>(ta, grid, s);
  else launch_tiles<kQ8_0>(ta, grid, s);
  return hipGetLastError();
}

}  // namespace okq
