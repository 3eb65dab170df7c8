// sym_b200 -- microscaled values: blocks of 32 values of a row share one
// power-of-two scale 2^s, stored as the byte s + 127 (255: the block held an
// infinity or a NaN and stands for NaN).
//
//   mxfp4   s = max(floor(log2 amax) - 2, -127); codes are the 4-bit floats
//           0, .5, 1, 1.5, 2, 3, 4, 6 with a sign, two per byte (the lower
//           index in the lower half). amax 2^-s lies in [4, 8): values above 6
//           saturate, ties go to the even code.
//   mxint8  s = max(floor(log2 amax), -120); codes are k = rne(x 2^(6-s)),
//           |k| <= 127. -120 keeps 2^(s-6) a normal 32-bit number.
//
// Every product below is exact (a power of two in range), so the only
// rounding is the one to the code: the codes are those of the definition in
// real arithmetic, whatever the order of the work.
//
// Layouts. Codes are row-major, rows padded to whole blocks with zero codes.
// mxint8 scales are row-major [rows, blocks]. mxfp4 scales lie in tiles of
// 128 rows x 4 blocks (512 bytes, tiles of one 128-row group consecutive),
// byte 16 (r mod 32) + 4 (r / 32) + b of a tile: the order in which one
// tcgen05.cp brings a tile to the tensor cores' scale columns.
#pragma once

#include "sb_cuda.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace mx {

constexpr int kBlock = 32;

__host__ __device__ __forceinline__ int64_t blocks_of(int64_t cols) { return (cols + kBlock - 1) / kBlock; }
/// Scale tiles (4 blocks) along a row.
__host__ __device__ __forceinline__ int64_t quads_of(int64_t cols) { return (cols + 127) / 128; }
/// Byte offset of the 4-byte scale word of row r, tile column q.
__host__ __device__ __forceinline__ int64_t scale_word(int64_t r, int64_t q, int64_t quads) {
  return ((r >> 7) * quads + q) * 512 + (r & 31) * 16 + ((r >> 5) & 3) * 4;
}

// Value types of x, y and the expanded matrices.
template <int DT> struct Value;
template <> struct Value<SBC_F32> {
  using T = float;
  static __device__ __forceinline__ float up(T v) { return v; }
  static __device__ __forceinline__ T down(float v) { return v; }
};
template <> struct Value<SBC_F16> {
  using T = __half;
  static __device__ __forceinline__ float up(T v) { return __half2float(v); }
  static __device__ __forceinline__ T down(float v) { return __float2half_rn(v); }
};
template <> struct Value<SBC_BF16> {
  using T = __nv_bfloat16;
  static __device__ __forceinline__ float up(T v) { return __bfloat162float(v); }
  static __device__ __forceinline__ T down(float v) { return __float2bfloat16_rn(v); }
};

/// Eight consecutive values at p; `have` of them exist (the rest read as
/// zero). VEC: p is 16-byte aligned.
template <int DT, bool VEC>
__device__ __forceinline__ void load8(float (&v)[8], const typename Value<DT>::T *p, int have) {
  using T = typename Value<DT>::T;
  if (VEC && have >= 8) {
    T raw[8];
    const uint4 *s = reinterpret_cast<const uint4 *>(p);
    uint4 *d = reinterpret_cast<uint4 *>(raw);
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof raw / 16); ++i)
      d[i] = __ldg(s + i);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      v[i] = Value<DT>::up(raw[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      v[i] = i < have ? Value<DT>::up(p[i]) : 0.f;
  }
}

template <int DT, bool VEC>
__device__ __forceinline__ void store8(typename Value<DT>::T *p, const float (&v)[8], int have) {
  using T = typename Value<DT>::T;
  if (VEC && have >= 8) {
    T raw[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      raw[i] = Value<DT>::down(v[i]);
    const uint4 *s = reinterpret_cast<const uint4 *>(raw);
    uint4 *d = reinterpret_cast<uint4 *>(p);
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof raw / 16); ++i)
      __stcs(d + i, s[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < have)
        p[i] = Value<DT>::down(v[i]);
  }
}

/// max(a, |b|) that keeps a NaN.
__device__ __forceinline__ float abs_max(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(fabsf(b)));
  return r;
}

/// Scale byte of a block whose largest magnitude is amax. The exponent field
/// of a 32-bit number is its floor(log2) + 127 (0 for subnormals and zero,
/// which the clamps cover).
template <int FMT> __device__ __forceinline__ uint32_t scale_byte(float amax) {
  const uint32_t f = __float_as_uint(amax) >> 23;
  if (f == 255)
    return 255;
  return FMT == SBC_MXFP4 ? (f > 2 ? f - 2 : 0) : (f > 7 ? f : 7);
}

/// 2^-s (mxfp4) or 2^(6-s) (mxint8): a normal number for every byte below 255
/// that scale_byte gives. The codes of a block with byte 255 are 0, which the
/// callers set: a NaN would convert to the largest code.
template <int FMT> __device__ __forceinline__ float inverse_scale(uint32_t byte) {
  return __uint_as_float((FMT == SBC_MXFP4 ? 254 - byte : 260 - byte) << 23);
}

/// 2^(field - 127) for any field, subnormal results included.
__device__ __forceinline__ float power(int field) {
  return __uint_as_float(field >= 1 ? static_cast<uint32_t>(field) << 23
                                    : (field > -23 ? 0x00400000u >> -field : 0u));
}

/// 2^s of an mxfp4 block, 2^(s-6) of an mxint8 block; NaN for byte 255.
template <int FMT> __device__ __forceinline__ float scale_value(uint32_t byte) {
  if (byte == 255)
    return __uint_as_float(0x7fffffffu);
  return power(FMT == SBC_MXFP4 ? static_cast<int>(byte) : static_cast<int>(byte) - 6);
}

/// Eight 4-bit codes of v[0..7] (already divided by the scale).
__device__ __forceinline__ uint32_t codes4(const float (&v)[8]) {
  uint32_t r;
  asm("{\n .reg .b8 a, b, c, d;\n"
      " cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
      " cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n"
      " mov.b32 %0, {a, b, c, d};\n}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

/// One 8-bit code: rne(v) clamped to +-127.
__device__ __forceinline__ uint32_t code8(float v) {
  return static_cast<uint32_t>(__float2int_rn(fminf(fmaxf(v, -127.f), 127.f))) & 255u;
}
__device__ __forceinline__ uint32_t codes8x4(float a, float b, float c, float d) {
  return code8(a) | (code8(b) << 8) | (code8(c) << 16) | (code8(d) << 24);
}

/// The values (before the scale) of eight 4-bit codes.
__device__ __forceinline__ void values4(float (&v)[8], uint32_t codes) {
  uint32_t h[4];
  asm("{\n .reg .b8 a, b, c, d;\n mov.b32 {a, b, c, d}, %4;\n"
      " cvt.rn.f16x2.e2m1x2 %0, a;\n cvt.rn.f16x2.e2m1x2 %1, b;\n"
      " cvt.rn.f16x2.e2m1x2 %2, c;\n cvt.rn.f16x2.e2m1x2 %3, d;\n}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(codes));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

/// The values (before the scale) of four 8-bit codes.
__device__ __forceinline__ void values8x4(float *v, uint32_t w) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    v[i] = static_cast<float>(static_cast<int8_t>(w >> (8 * i)));
}

} // namespace mx
