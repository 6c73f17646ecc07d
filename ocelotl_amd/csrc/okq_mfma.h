// okq_mfma.h -- vector types, buffer descriptors and the dequantisation of
// GGUF weights into MFMA B fragments, shared by the kernels that contract them
// through v_mfma_f32_16x16x32_f16 (decode batches, a layer's experts).
#pragma once
#include "okq_device.h"

namespace okq {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f16x __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x3 __attribute__((ext_vector_type(3)));
typedef __amdgpu_buffer_rsrc_t Rsrc;

// Buffer descriptor over [base, base + bytes), bytes < 2^32.  Loads past the
// end return zeros: rows beyond M or N stage as zeros without branches.
__device__ __forceinline__ Rsrc make_rsrc(const void *base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), (short)0, (int)bytes, 0x00020000);
}
__device__ __forceinline__ u32x4 bload4(Rsrc r, uint32_t off) { return __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0); }

typedef float f4 __attribute__((ext_vector_type(4)));

// ---- weights as exact fp16 B fragments ------------------------------------------
// 0x6400 | q is the fp16 value 1024 + q; (1024+q)*sc - 1024*sc = sc*q is one
// fused fp16 FMA whose exact result (an integer <= 945) is representable.
__device__ __forceinline__ h2 nib_pair(uint32_t spread, h2 sc2, h2 off2) {
  return __builtin_elementwise_fma(__builtin_bit_cast(h2, spread), sc2, off2);
}
// Four nibbles (one per byte of n4) -> two fp16 pairs of sc*q, in byte order.
// v_perm_b32 interleaves the bytes with the 0x64 exponent byte of 1024.
__device__ __forceinline__ void nib4(uint32_t n4, h2 sc2, h2 off2, h2 &p0, h2 &p1) {
  p0 = nib_pair(__builtin_amdgcn_perm(0x64646464u, n4, 0x04010400u), sc2, off2);
  p1 = nib_pair(__builtin_amdgcn_perm(0x64646464u, n4, 0x04030402u), sc2, off2);
}

// v = sc * (q - 32) for the four 6-bit values in the bytes of q4, as two
// exact fp16 planes v = hi + lo: 0x64|q is the fp16 1024 + q, minus 1056
// gives q - 32 exactly; hi = fp16(v) is exact while |v| <= 2048 and rounds to
// an even integer above (|v| <= 4096), and lo = fma(q - 32, sc, -hi) is the
// exact remainder (-1, 0 or 1).
__device__ __forceinline__ void q6_4(uint32_t q4, h2 sc2, h2 &p0, h2 &p1, h2 &l0, h2 &l1) {
  const h2 off = {(_Float16)-1056.0f, (_Float16)-1056.0f};
  const h2 a = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, q4, 0x04010400u)) + off;
  const h2 b = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, q4, 0x04030402u)) + off;
  p0 = a * sc2;
  p1 = b * sc2;
  l0 = __builtin_elementwise_fma(a, sc2, -p0);
  l1 = __builtin_elementwise_fma(b, sc2, -p1);
}

// d * q for the four int8 quants in the bytes of q4, as two exact fp16 planes
// d * q = hi + lo: (q ^ 0x80) | 0x6400 is the fp16 1152 + q, minus 1152 gives
// q exactly; hi = fp16(d * q) (one rounding) and lo = fma(q, d, -hi) is the
// exact remainder.  Exact because d * q has at most 19 significant bits whose
// lowest is at least 2^-24 (d is an fp16), so the remainder fits an fp16, for
// every block with |d * q| below 65520 (|d| < 511.9, any block quantised from
// fp16-representable weights).
__device__ __forceinline__ void q8_4(uint32_t q4, h2 d2, h2 &p0, h2 &p1, h2 &l0, h2 &l1) {
  const h2 off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
  const uint32_t b = q4 ^ 0x80808080u;
  const h2 a = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u)) + off;
  const h2 c = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u)) + off;
  p0 = a * d2;
  p1 = c * d2;
  l0 = __builtin_elementwise_fma(a, d2, -p0);
  l1 = __builtin_elementwise_fma(c, d2, -p1);
}

// The Q4_K / Q5_K header of an item, unpacked four bytes at a time: the 6-bit
// scales (and mins) of sub-blocks 0-3 are the low bits of bytes 0-3 (4-7),
// those of 4-7 a nibble of bytes 8-11 and the two top bits of bytes 0-3
// (4-7), so one dword of four scales is one AND, or two shifts and three
// bit operations; v_perm_b32 then puts a byte under the 0x64 exponent (1024 +
// sc) twice, and a packed add leaves the fp16 pair (sc, sc).  Field by field
// (shifts and masks per sub-block, a conversion each) the header cost as many
// VALU instructions as the weights' nibbles.  5 rows x 4096 -> 14336 in Q5_K
// 18.6 -> 18.1 us per call, 32-row gate + up in Q4_K 30.8 -> 30.0 us, 8 rows
// unchanged: the items wait for memory more than for issue slots.
__device__ __forceinline__ h2 byte_pair(uint32_t four, uint32_t j) {
  return __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, four, 0x04000400u + 0x00010001u * j)) +
         h2{(_Float16)-1024.0f, (_Float16)-1024.0f};
}

// Workgroup barrier for LDS only: waits for this wave's LDS operations, not
// for its vector-memory loads (loads issued ahead stay in flight across it).
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_s_waitcnt(0xC07F);  // gfx9 encoding: lgkmcnt(0), vmcnt and expcnt unconstrained
  __builtin_amdgcn_s_barrier();
}

}  // namespace okq
