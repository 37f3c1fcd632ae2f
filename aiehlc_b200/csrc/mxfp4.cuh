// Microscaled 4-bit floating point: what a block is, how a quantised matrix lies in memory, and the
// conversions every kernel of this format shares.
//
// A block is 32 consecutive elements of a row.  It shares one power of two and holds e2m1 numbers
// (sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6), as the OCP Microscaling specification defines MXFP4:
//     e     = floor(log2(max |x|)) - 2, at least -127      (2 = exponent of the largest e2m1 number, 6)
//     x_hat = 2^e * round_half_even_e2m1(x * 2^-e), at most 6 * 2^e in magnitude
// A block with an infinity or a NaN in it is NaN as a whole (scale byte 255, codes 0).
//
// codes : uint8 [rows][16 * blocks], element 2i in the low half of byte i, zeros past the last column
// scales: e + 127, in tiles of 128 rows x 4 blocks = 512 bytes, the order the tensor cores read them in
//         (one 16-byte line per TMEM lane), zeros for rows and blocks that do not exist
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace aiehlc {

constexpr int kMxBlock = 32;           // elements that share a scale
constexpr int kMxScaleTile = 512;      // bytes of scales for 128 rows x 4 blocks
constexpr int kMxNan = 255;            // scale byte of a block that is NaN

__host__ __device__ __forceinline__ long long mx_blocks(long long cols) { return (cols + kMxBlock - 1) / kMxBlock; }
__host__ __device__ __forceinline__ long long mx_pitch(long long cols) { return mx_blocks(cols) * (kMxBlock / 2); }
__host__ __device__ __forceinline__ long long mx_words(long long cols) { return (mx_blocks(cols) + 3) / 4; }
__host__ __device__ __forceinline__ long long mx_scale_bytes(long long rows, long long cols) {
  return (rows + 127) / 128 * mx_words(cols) * kMxScaleTile;
}
// Where the four scales of row `r` (of its tile's 128) lie in a scale tile.
__host__ __device__ __forceinline__ int mx_scale_word(int r) { return (r & 31) * 16 + ((r >> 5) & 3) * 4; }

// Scale byte of a block from the largest |x| as float bits (an infinity or NaN in the block shows as the
// exponent 255): floor(log2) is the exponent field, subnormal maxima end at the smallest scale.
__device__ __forceinline__ int mx_scale_of(uint32_t max_bits) {
  const int e = static_cast<int>(max_bits >> 23);
  return e == 255 ? kMxNan : (e > 2 ? e - 2 : 0);
}
// 2^-e for scale byte s: exact, and normal for every finite scale mx_scale_of gives (s <= 252).
__device__ __forceinline__ float mx_inverse(int s) { return __uint_as_float(static_cast<uint32_t>(254 - s) << 23); }
// 2^e for scale byte s (2^-127 is subnormal); NaN for 255.
__device__ __forceinline__ float mx_scale_value(int s) {
  return __uint_as_float(s == kMxNan ? 0x7FC00000u : s == 0 ? 0x00400000u : static_cast<uint32_t>(s) << 23);
}
// Eight values, already divided by the scale, to eight codes, v[0] in the low four bits.  The conversion rounds to
// nearest, ties to even, and saturates at 6.  (A block that is NaN has its codes replaced by zeros.)
__device__ __forceinline__ uint32_t mx_codes8(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}
// Eight codes to eight halves (exact).
__device__ __forceinline__ void mx_decode8(uint32_t codes, __half2 (&h)[4]) {
  uint32_t r0, r1, r2, r3;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(codes));
  h[0] = *reinterpret_cast<__half2*>(&r0);
  h[1] = *reinterpret_cast<__half2*>(&r1);
  h[2] = *reinterpret_cast<__half2*>(&r2);
  h[3] = *reinterpret_cast<__half2*>(&r3);
}

// One element of each type the entry points take (AIEHLC_TYPE_*), rounded to nearest even.
template <typename T> __device__ __forceinline__ T mx_from_float(float v);
template <> __device__ __forceinline__ float mx_from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 mx_from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half mx_from_float<__half>(float v) { return __float2half_rn(v); }

}  // namespace aiehlc
