// Shared by the kernels of the decoder losses (vocab.hip, vocab8.hip).
#pragma once
#include "common.h"
#include "kernels.h"

namespace {

constexpr int BK = 64;               // K tile
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
#if CLIP_OPERAND_F16
constexpr float G_SCALE = 32768.f;
#else
constexpr float G_SCALE = 1.f;       // bf16 has fp32's range
#endif
constexpr double FIX = 274877906944.0;   // 2^38: fixed-point unit of the target sums, |sum| <= 2^24 rows
constexpr int FIX_COPIES = 8;            // copies of their table
constexpr int ROW_FIX = 8;               // large entries of a row of G that dh is corrected for
typedef __attribute__((ext_vector_type(4))) unsigned int u32x4_t;
typedef __attribute__((ext_vector_type(2))) unsigned int u32x2_t;

// ---- buffer descriptor of [p, p + bytes): loads past the end return zero, which is how ragged vocabulary tails are read
__device__ __forceinline__ u32x4_t make_rsrc(const void* p, int64_t bytes) {
  const uint64_t a = (uint64_t)p;
  const int64_t b = bytes < 0 ? 0 : (bytes > 0xffffffffll ? 0xffffffffll : bytes);
  u32x4_t r;
  r[0] = __builtin_amdgcn_readfirstlane((uint32_t)a);
  r[1] = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32) & 0xffffu);
  r[2] = __builtin_amdgcn_readfirstlane((uint32_t)b);
  r[3] = 0x00020000u;
  return r;
}
// one wave's 1-KiB LDS-DMA piece: lane l's 16 bytes at r + voff land at lds + 16 l
__device__ __forceinline__ void dma16(const u32x4_t& r, uint32_t voff, uint32_t lds) {
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
  asm volatile("s_mov_b32 m0, %2\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voff), "s"(r), "s"(lds) : "memory", "m0");
#pragma clang diagnostic pop
}

// sum / max over the 16 lanes fr = lane & 15, and over the 4 lanes fq = lane >> 4
__device__ __forceinline__ float fr_sum(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
__device__ __forceinline__ float fq_sum(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}
__device__ __forceinline__ float fq_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, 64));
  return fmaxf(v, __shfl_xor(v, 32, 64));
}

// 32-byte slot swizzle of an R-major K tile image [64 k][2 R bytes]
template <int R>
__device__ __forceinline__ int tr_swz(int k) {
  static_assert(R >= 128, "rows of eight slots and more");
  return (k & 3) | ((k >> 3) & 1) << 2;
}

// 16 bytes of dW, written once and not read again here; rows of a caller's own stride may start on 8 bytes only
__device__ __forceinline__ void store_dw(bf16_t* o, const u32x4_t& v, bool wide) {
  if (wide) {
    __builtin_nontemporal_store(v, reinterpret_cast<u32x4_t*>(o));
  } else {
    __builtin_nontemporal_store((u32x2_t){v[0], v[1]}, reinterpret_cast<u32x2_t*>(o));
    __builtin_nontemporal_store((u32x2_t){v[2], v[3]}, reinterpret_cast<u32x2_t*>(o) + 1);
  }
}

// Row and column within its 256 x 256 tile of the q-th group of 4 partials that vocab8_kernel stores of a dh tile
__device__ __forceinline__ void dh_partial_at(int q, int& row, int& col) {
  const int lane = q & 63, i = q >> 6 & 1, nh = q >> 7 & 1, m = q >> 8 & 3, mh = q >> 10 & 1, w = q >> 11;
  row = mh * 128 + (w >> 2) * 64 + m * 16 + (lane & 15);
  col = (w & 3) * 64 + nh * 32 + i * 16 + (lane >> 4) * 4;
}

// What the product kernels compute; A [M, K] and B [N, K], "R-major" = stored [K, R]
//   V_STATS  rows x vocabulary: every row's (max, sum of exp2) over 64 columns at a time       A = live rows, B = W
//   V_GRAD   the same product once more -> G and the column sums of G before rounding
//   V_DH     rows x hidden over a range of the vocabulary piece -> fp32 partial                A = G, B = W (R-major)
//   V_DW     vocabulary x hidden over the rows -> 16-bit dW                                    A = G, B = live rows (both R-major)
//   V_PROD   both, sharing one launch (vocab8.hip)
enum { V_STATS = 0, V_GRAD = 1, V_DH = 2, V_DW = 3, V_PROD = 4 };

}  // namespace
