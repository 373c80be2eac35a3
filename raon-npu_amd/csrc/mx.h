// Microscaled 4-bit rows (MXFP4): blocks of 32 columns that share a power of two.
//
//   s    = clamp(floor(log2 max|x|) - 2, -127, 127), -127 for a block of zeros; held as the byte s + 127;
//   code = the e2m1 value nearest to x 2^-s, ties to the even code, magnitudes above 6 to 6, with x's sign:
//          bit 3 the sign, bits 0..2 an index into 0, 0.5, 1, 1.5, 2, 3, 4, 6.
// A block that holds NaN or an infinity has scale byte 255, which stands for NaN, and codes 0.  A row of K
// columns has P = K rounded up to 32 of them, zeros past K: P / 2 bytes of codes (the even column in the low
// half of its byte) and P / 32 scale bytes.
#pragma once

#include "../../include/raon_moe.h"
#include "rmoe_internal.h"

namespace rmoe {

constexpr int kMxBlock = 32;

// One element of a row type as fp32, and fp32 rounded to it (RTNE, by the conversion instructions).
template <int DT>
struct RowElem;
template <>
struct RowElem<RMOE_DT_BF16> {
  typedef uint16_t T;
  static __device__ __forceinline__ float get(T v) { return bf16_to_f32(v); }
  static __device__ __forceinline__ T put(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }
};
template <>
struct RowElem<RMOE_DT_F16> {
  typedef uint16_t T;
  static __device__ __forceinline__ float get(T v) { return (float)__builtin_bit_cast(_Float16, v); }
  // The fp32 value is formed first: the compiler makes one instruction with a single rounding of some
  // products with their conversion to fp16.
  static __device__ __forceinline__ T put(float v) {
    asm("" : "+v"(v));
    return __builtin_bit_cast(uint16_t, (_Float16)v);
  }
};
template <>
struct RowElem<RMOE_DT_F32> {
  typedef float T;
  static __device__ __forceinline__ float get(T v) { return v; }
  static __device__ __forceinline__ T put(float v) { return v; }
};

// Eight consecutive columns of a row.
template <int DT>
struct alignas(16) Chunk {
  typename RowElem<DT>::T v[8];
};
// Loads and stores of the columns c..c+7 of a row `width` wide: by 16 bytes, or (kWide false: rows that are not
// aligned to 16 bytes or end inside a chunk) one by one, with zeros past the end.  kOnce: read past the caches' order of
// use, for rows of kOnceBytes and more that are not read again.
template <int DT, bool kWide, bool kOnce = false>
__device__ __forceinline__ Chunk<DT> load_chunk(const void* row, int c, int width) {
  const auto* p = static_cast<const typename RowElem<DT>::T*>(row) + c;
  Chunk<DT> r;
  if constexpr (kWide) {
    const uint4* q = reinterpret_cast<const uint4*>(p);
    uint4* o = reinterpret_cast<uint4*>(r.v);
#pragma unroll
    for (int i = 0; i < (int)(sizeof(r) / 16); ++i) o[i] = kOnce ? load_stream16(reinterpret_cast<const uint8_t*>(q + i)) : q[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = c + i < width ? p[i] : (typename RowElem<DT>::T)0;
  }
  return r;
}
template <int DT, bool kWide>
__device__ __forceinline__ void store_chunk(void* row, int c, int width, const Chunk<DT>& r) {
  auto* p = static_cast<typename RowElem<DT>::T*>(row) + c;
  if constexpr (kWide) {
    uint4* q = reinterpret_cast<uint4*>(p);
    const uint4* o = reinterpret_cast<const uint4*>(r.v);
#pragma unroll
    for (int i = 0; i < (int)(sizeof(r) / 16); ++i) q[i] = o[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < width) p[i] = r.v[i];
  }
}

// A block of 32 columns, eight in each lane of a quad, to its scale byte and the lane's eight codes (column i in
// bits 4i..4i+3).
__device__ __forceinline__ uint32_t mx_quantize8(const float (&x)[8], uint32_t& scale_byte) {
  uint32_t top = 0;  // magnitude bits: ordered as the magnitudes, infinities and NaN above all
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xF, 0xF, false));
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xF, 0xF, false));
  // floor(log2) of a normal value is its exponent field - 127; below 2^-125 the scale is 2^-127 whatever it is.
  const uint32_t e = top >> 23;
  const bool bad = e == 0xffu;
  const uint32_t b = e > 2 ? e - 2 : 0u;
  scale_byte = bad ? 0xffu : b;
  // The scale as fp32: 2^-127 is subnormal.
  const float s = __uint_as_float(b ? b << 23 : 0x00400000u);
  uint32_t q = 0;
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, x[0], x[1], s, 0);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, x[2], x[3], s, 1);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, x[4], x[5], s, 2);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, x[6], x[7], s, 3);
  return bad ? 0u : q;
}
// The value code i (0..7) of q stands for, fp32 (exact).
__device__ __forceinline__ float mx_value(uint32_t q, int i, uint32_t scale_byte) {
  const uint32_t n = q >> (4 * i);
  const uint32_t m = n & 7u;
  // 0.5 in magnitude 1, else 1 or 1.5 times 2^(m / 2 - 1).
  const uint32_t mag = m < 2 ? m * 0x3f000000u : ((m >> 1) + 126u) << 23 | (m & 1u) << 22;
  const float v = __builtin_amdgcn_ldexpf(__uint_as_float(mag | (n & 8u) << 28), (int)scale_byte - 127);
  return scale_byte == 0xffu ? __uint_as_float(0x7fc00000u) : v;
}

}  // namespace rmoe
