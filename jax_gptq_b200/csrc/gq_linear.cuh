// Shared by the two forms of the packed-weight product (gq_linear.cu: a few
// tokens; gq_linear_tc.cu: many): the laid-out weights and their decoding.
#pragma once

#include "gq_common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

namespace gq {
namespace lin {

constexpr int KC = 128;      // positions per block
constexpr int ROWS = 16;     // rows per block

// Place of 16-byte piece `i` in row r of a block (its own inverse): the row's 4
// (8) pieces are exchanged so that pieces i of 8 consecutive rows cover 128
// different bytes modulo 128.
template <int WIDTH>
__host__ __device__ __forceinline__ int piece_at(int i, int r) {
  return WIDTH == 4 ? i ^ ((r >> 1) & 3) : i ^ (r & 7);
}

template <bool BF16>
__device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
  uint32_t d;
  if constexpr (BF16)
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  else
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// {a, b} rounded to 16 bits, a in the low half (exact for the values used here).
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  uint32_t d;
  if constexpr (BF16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(b), "f"(a));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(b), "f"(a));
  return d;
}

// What a granule's offset becomes before its codes are decoded: the bit
// pattern that sub2 takes off, or for 8-bit codes in bf16 a float.
template <int WIDTH, bool BF16>
__device__ __forceinline__ uint32_t offset_operand(float o) {
  if constexpr (WIDTH == 4) return pack2<BF16>(16.f + o, 16.f + o);
  else if constexpr (BF16) return __float_as_uint(8388608.f + o);
  else return pack2<false>(1024.f + o, 1024.f + o);
}

// (x & mask) | bits as the one instruction it is: left to the compiler it took
// two, and a one-token product of 28672 x 8192 36.2 us in place of 33.8.
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t bits) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(d) : "r"(x), "r"(mask), "r"(bits));
  return d;
}

// The four pairs (code - offset) of 8 positions.  4-bit fields are moved into
// the mantissa of 16.0, where they count in ones: bits 3-6 of a bf16, bits 6-9
// of an fp16; 8-bit fields into the mantissa of 2^23 (float) or 1024 (fp16).
// Field i of a 4-bit word begins at bit 3 + 4 (i / 2) + 16 (i % 2), wrapping, so
// that the first pair is in place for bf16 and a rotation brings the others.
template <int WIDTH, bool BF16>
__device__ __forceinline__ void decode8(const uint32_t* w, uint32_t off, uint32_t (&v)[4]) {
  if constexpr (WIDTH == 4) {
    const uint32_t x = w[0];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      if constexpr (BF16)
        v[p] = and_or(__funnelshift_r(x, x, 4 * p), 0x00780078u, 0x41804180u);
      else
        v[p] = and_or(__funnelshift_r(x, x, (4 * p + 29) & 31), 0x03c003c0u, 0x4c004c00u);
    }
#pragma unroll
    for (int p = 0; p < 4; ++p) v[p] = sub2<BF16>(v[p], off);
  } else if constexpr (BF16) {
    const float o = __uint_as_float(off);
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const uint32_t x = w[p >> 1];
      const float a = __uint_as_float(__byte_perm(x, 0x4b000000u, (p & 1) ? 0x7442 : 0x7440));
      const float b = __uint_as_float(__byte_perm(x, 0x4b000000u, (p & 1) ? 0x7443 : 0x7441));
      v[p] = pack2<true>(a - o, b - o);
    }
  } else {
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const uint32_t x = w[p >> 1];
      v[p] = sub2<false>(__byte_perm(x, 0x64646464u, (p & 1) ? 0x4342 : 0x4140), off);
    }
  }
}

__device__ __forceinline__ void store_out(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store_out(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store_out(float* p, float v) { *p = v; }

// The many-token form (gq_linear_tc.cu).  x: [cols, ldx] 16-bit values in
// position order, 16-byte aligned, ldx a multiple of 8; for float32 (dtype 0)
// three columns per token.
int run_many(const uint32_t* qw, const float* params, int64_t m, int64_t k, int bits, int granule,
             const uint16_t* x, int64_t ldx, int dtype, int64_t tokens, void* y, int64_t ldy,
             cudaStream_t st);
// Its choice on a device of `sms` SMs: columns of an MMA, MMAs side by side, CTAs along K,
// tiles, and the slots and barriers of its three rings (copied codes, decoded blocks,
// accumulators).
void many_form(int64_t m, int64_t k, int bits, int granule, int dtype, int64_t tokens, int sms,
               int64_t* form);

}  // namespace lin
}  // namespace gq
