// okq_gemm_f32.hip -- prefill dequant-GEMM for f32 activations with the
// weights dequantised in registers: Y[M,N] = X[M,K] W[N,K]^T (+bias), Q4_K,
// Q5_K, Q6_K and Q8_0, one or several matrices that read the same X.  bf16
// activations (one fp16 plane: kTwo false) take it where their own kernels
// do not pay: Q6_K grids too small for gemm_wide_q6k_kernel's tiles (us per
// call, against weights staged through LDS: 64 x 4096 -> 14336 80 -> 34, 300 x
// 4096 -> 14336 185 -> 100, 128 x 14336 -> 4096 61 -> 48, 33 x 4096 -> 4096 24
// -> 22), and Q4_K / Q5_K tensors within 256 rows of 4 GiB (elsewhere the
// kernels of okq_gemm_wide.hip and okq_gemm_pair.hip are faster: 128 x 4096 ->
// 1024 15.6 against 19.4).
//
// Numerics.  A = the pre-pass's row-scaled activations as two fp16 planes,
// x = hi + lo to 2^-22; B = the integer part of the weight, exact in fp16
// (Q4_K / Q5_K: sc * q; Q8_0: q; Q6_K: sc * (q - 32) as B1 = its fp16
// rounding and the exact remainder B2 in {-1, 0, 1}).  Both planes are
// contracted with B (Q6_K: hi with B1 and B2, lo with B1: lo * B2 is below
// 2^-22 of the product), so every product is exact and only f32 sums round;
// d is applied in f32 per super-block (Q8_0: per block of 32), with the
// Q4_K / Q5_K min term dmin * sum_j m_j xsum_j from one more MFMA.
//
// Per call, against a kernel that staged dequantised weights in LDS
// (us): 512 x 4096 -> 14336 Q4_K 219 -> 123, Q5_K 244 -> 136, Q6_K 306 -> 168,
// Q8_0 219 -> 152; 2048 x 14336 -> 4096 Q4_K 767 -> 450, Q6_K 1007 -> 602;
// 64 x 14336 -> 4096 Q4_K 58 -> 34; 33 x 4096 -> 4096 Q4_K 24 -> 20.
//
// What bounds it: the MFMAs, two per weight fragment and row block (Q6_K
// three) where bf16 activations need one, at the rate that the power budget
// leaves them.  So a weight is dequantised once for both planes, by the one
// wave that owns its column, and only the activations pass through LDS.
//
// Layout: one 8-wave workgroup per CU on a 128 x 256 tile; wave w owns
// columns 32w .. 32w+31 for all 128 rows (four 32x32x16 MFMA blocks).  A
// stage is half a super-block (128 K): 64 KB of activations (both planes) and
// 2 KB of per-32 sums, double-buffered in LDS by buffer-to-LDS copies one
// stage ahead; a super-block per stage would not fit twice.  The 16-byte
// chunk c of row r sits at chunk c ^ (r & 15).  A step (8 per stage, 16 K)
// contracts the hi fragments while the lo ones are read, then the lo
// fragments while the next step's hi ones are read and its weights
// dequantised: as many fragment registers as for one plane.
//   * K order inside a stage: MFMA step s, lane group g = lane / 32.
//     Q4_K / Q5_K: k = 64 g + 8 s + [0, 8) (lane group g reads the 32 qs bytes
//     of one chunk, low nibbles at steps 0-3).  Q6_K / Q8_0: k = 32 (s / 2) +
//     16 g + 8 (s & 1) + [0, 8) (a step stays inside one Q8_0 block and one
//     Q6_K scale).
#include "okq_gemm_f32.h"

namespace okq {

// Tiles of 32 kNB rows (a row's result does not depend on the height).
template <int kType, int kNB, bool kTwo>
__global__ __launch_bounds__(512) void gemm_f32_kernel(const _Float16 *__restrict__ xhi, const _Float16 *__restrict__ xlo,
                                                       const h2 *__restrict__ xsum, const float *__restrict__ rscale,
                                                       int M, int K, PrefillMats mats) {
  f32_body<kType, kNB, kTwo>(xhi, xlo, xsum, rscale, M, K, mats);
}

// Tile height in 32-row blocks: a stage of 2, 3 or 4 blocks takes about 0.6,
// 0.8 and 1 of the full tile's time (what does not scale is the weights'
// dequantisation and the loads), so the height of least total.
static int tile_blocks(int64_t M) {
  const int64_t c4 = 10 * ((M + 127) / 128), c3 = 8 * ((M + 95) / 96), c2 = 6 * ((M + 63) / 64);
  return c4 <= c3 && c4 <= c2 ? 4 : c3 <= c2 ? 3 : 2;
}
static int tile_rows(int64_t M) { return 32 * tile_blocks(M); }
int gemm_f32_blocks(int64_t M) { return tile_blocks(M); }
int gemm_f32_tiles(int64_t M, int64_t N) { return (int)(((M + tile_rows(M) - 1) / tile_rows(M)) * ((N + kFN - 1) / kFN)); }

hipError_t launch_gemm_f32(int type, const _Float16 *xhi, const _Float16 *xlo, const void *xsum, const float *rscale,
                           int64_t M, int64_t K, PrefillMats &mats, int count, hipStream_t s) {
  if (K % 256 != 0 || count < 1 || count > kPrefillMats) return hipErrorInvalidValue;
  int px = 0;
  for (int i = 0; i < kPrefillMats; ++i) {
    PrefillMat &m = mats.mat[i];
    if (i >= count) {
      m.px0 = INT32_MAX;
      continue;
    }
    if (m.ksplit < 1 || m.ksplit > K / 256) return hipErrorInvalidValue;
    m.tiles = gemm_f32_tiles(M, m.n);
    m.px0 = px;
    m.pxn = (m.tiles * m.ksplit + 7) / 8;
    px += m.pxn;
  }
  const dim3 grid((unsigned)(px * 8)), block(512);
  const h2 *sums = static_cast<const h2 *>(xsum);
  const int nb = tile_blocks(M);
#define OKQ_F32_NB(TYPE_, TWO_)                                                                                         \
  if (nb == 2)                                                                                                          \
    launch_timed(gemm_f32_kernel<TYPE_, 2, TWO_>, grid, block, 0u, s, xhi, xlo, sums, rscale, (int)M, (int)K, mats);     \
  else if (nb == 3)                                                                                                     \
    launch_timed(gemm_f32_kernel<TYPE_, 3, TWO_>, grid, block, 0u, s, xhi, xlo, sums, rscale, (int)M, (int)K, mats);     \
  else                                                                                                                  \
    launch_timed(gemm_f32_kernel<TYPE_, 4, TWO_>, grid, block, 0u, s, xhi, xlo, sums, rscale, (int)M, (int)K, mats)
#define OKQ_F32(TYPE_)          \
  if (xlo) {                    \
    OKQ_F32_NB(TYPE_, true);    \
  } else {                      \
    OKQ_F32_NB(TYPE_, false);   \
  }
  if (type == kQ4_K) {
    OKQ_F32(kQ4_K)
  } else if (type == kQ5_K) {
    OKQ_F32(kQ5_K)
  } else if (type == kQ6_K) {
    OKQ_F32(kQ6_K)
  } else if (xlo) {  // bf16 Q8_0: okq_gemm_q8.hip
    OKQ_F32_NB(kQ8_0, true);
  } else {
    return hipErrorInvalidValue;
  }
#undef OKQ_F32_NB
#undef OKQ_F32
  return hipGetLastError();
}

}  // namespace okq
