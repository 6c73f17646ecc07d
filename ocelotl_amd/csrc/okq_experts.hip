// okq_experts.hip -- a layer's experts over many rows: every expert's rows,
// sorted together, in tiles of up to 128 through the f32 prefill GEMM's body
// (okq_gemm_f32.h).
//
// What bounds it: the MFMAs, two per weight fragment and row block (Q6_K
// three): 4096 tokens, 8 of 128 experts, 2048 x 768: gate and up in Q4_K 521-549
// us, 750-790 TFLOP/s of them (49% of the cycles), down in Q6_K 361-384, 810-860.
// (The dense kernel does 980 and 1070 on 512 x 4096 -> 14336.  A workgroup here
// has 16 or 6 stages, and nothing runs beside its first loads and its
// epilogue.)  Tiles of 64 rows wait for their weights, requested one stage
// ahead: 333 tokens, 6 of 31, 2560 x 1440 in Q8_0: 168 and 92 us.
// A tile's height is its expert's own: full ones of 128
// rows, and one of 32, 64, 96 or 128 for the rest, chosen per workgroup.
#include "okq_gemm_f32.h"

namespace okq {

// Workgroup b runs on XCD b % 8.  Tiles in eight contiguous ranges, all columns
// of a tile behind one another: an expert's weights and a tile's activations
// are each read by one XCD, close in time.
template <int kType, int kExperts>
__global__ __launch_bounds__(512) void experts_kernel(const _Float16 *__restrict__ xhi, const _Float16 *__restrict__ xlo,
                                                      const h2 *__restrict__ xsum, const float *__restrict__ rscale,
                                                      int M, int K, ExpertMat mat, const int *__restrict__ count,
                                                      const ExpertTile *__restrict__ tiles, int columns) {
  const int n = count[0], per = (n + 7) / 8;
  const int b = (int)blockIdx.x, i = b / 8 / columns;
  const int t = b % 8 * per + i;
  if (i >= per || t >= n) return;
  const ExpertTile et = tiles[t];
  const int column = b / 8 - i * columns;
  const PrefillMats none{};
  switch (et.blocks) {
  case 1: return f32_body<kType, 1, true, kExperts>(xhi, xlo, xsum, rscale, M, K, none, mat, et, column);
  case 2: return f32_body<kType, 2, true, kExperts>(xhi, xlo, xsum, rscale, M, K, none, mat, et, column);
  case 3: return f32_body<kType, 3, true, kExperts>(xhi, xlo, xsum, rscale, M, K, none, mat, et, column);
  default: return f32_body<kType, 4, true, kExperts>(xhi, xlo, xsum, rscale, M, K, none, mat, et, column);
  }
}

hipError_t launch_experts(int type, bool gate_up, const _Float16 *xhi, const _Float16 *xlo, const void *xsum,
                          const float *rscale, int M, int K, const ExpertMat &mat, const int *count,
                          const ExpertTile *tiles, int64_t most_tiles, hipStream_t s) {
  const int width = gate_up ? kFN / 2 : kFN, columns = (mat.n + width - 1) / width;
  const int64_t blocks = (most_tiles + 7) / 8 * 8 * columns;
  if (blocks >= 1 << 23) return hipErrorInvalidValue;
  const dim3 grid((unsigned)blocks), block(512);
  const h2 *sums = static_cast<const h2 *>(xsum);
#define OKQ_EXPERTS(T_)                                                                                                \
  {                                                                                                                    \
    if (gate_up)                                                                                                       \
      launch_timed(experts_kernel<T_, 1>, grid, block, 0u, s, xhi, xlo, sums, rscale, M, K, mat, count, tiles, columns); \
    else                                                                                                               \
      launch_timed(experts_kernel<T_, 2>, grid, block, 0u, s, xhi, xlo, sums, rscale, M, K, mat, count, tiles, columns); \
  }
  if (type == kQ4_K) OKQ_EXPERTS(kQ4_K)
  else if (type == kQ5_K) OKQ_EXPERTS(kQ5_K)
  else if (type == kQ6_K) OKQ_EXPERTS(kQ6_K)
  else OKQ_EXPERTS(kQ8_0)
#undef OKQ_EXPERTS
  return hipGetLastError();
}

}  // namespace okq
