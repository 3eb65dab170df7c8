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
#include <type_traits>

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

/// A pair of 16-bit values in 32 bits each.
template <int DT> __device__ __forceinline__ float2 unpack2(uint32_t w) {
  if (DT == SBC_F16)
    return __half22float2(*reinterpret_cast<const __half2 *>(&w));
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
/// Two values rounded to 16 bits, the first in the lower half.
template <int DT> __device__ __forceinline__ uint32_t pack2(float a, float b) {
  uint32_t r;
  if (DT == SBC_F16)
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  else
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}

/// Eight consecutive values as they lie in memory. Loading and converting are
/// apart so that a thread's loads can all be on their way before the first is
/// waited for.
template <int DT> struct Raw8 {
  uint4 q[DT == SBC_F32 ? 2 : 1];

  /// The values at p, of which `have` exist; the rest are zero. VEC: p is
  /// 16-byte aligned.
  template <bool VEC> __device__ __forceinline__ void load(const typename Value<DT>::T *p, int have) {
    if (VEC && have >= 8) {
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof q / 16); ++i)
        q[i] = __ldg(reinterpret_cast<const uint4 *>(p) + i);
    } else {
      using U = typename std::conditional<DT == SBC_F32, uint32_t, uint16_t>::type;
      const U *u = reinterpret_cast<const U *>(p);
      U v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        v[i] = i < have ? __ldg(u + i) : U(0);
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof q / 4); ++i) {
        uint32_t w;
        if (DT == SBC_F32)
          w = v[i];
        else
          w = v[2 * i & 7] | static_cast<uint32_t>(v[2 * i + 1 & 7]) << 16;
        reinterpret_cast<uint32_t *>(q)[i] = w;
      }
    }
  }

  /// The values as four pairs in 32 bits.
  __device__ __forceinline__ void values(float2 (&v)[4]) const {
    const uint32_t *w = reinterpret_cast<const uint32_t *>(q);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (DT == SBC_F32)
        v[i] = make_float2(__uint_as_float(w[2 * i & 7]), __uint_as_float(w[2 * i + 1 & 7]));
      else
        v[i] = unpack2<DT>(w[i]);
    }
  }

  /// The largest magnitude, a NaN above all. Magnitudes order like their bits,
  /// so 16-bit values are compared two at a time as whole numbers.
  __device__ __forceinline__ float top() const {
    const uint32_t *w = reinterpret_cast<const uint32_t *>(q);
    if (DT == SBC_F32) {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        m = max(m, w[i & 7] & 0x7fffffffu);
      return __uint_as_float(m);
    }
    uint32_t m = w[0] & 0x7fff7fffu;
#pragma unroll
    for (int i = 1; i < 4; ++i)
      m = __vmaxu2(m, w[i] & 0x7fff7fffu);
    m = max(m & 0xffffu, m >> 16);
    return unpack2<DT>(m).x;
  }
};

/// The largest magnitude over the 2^n lanes of a block's quarters; magnitudes
/// and NaN order like their bits.
template <int N> __device__ __forceinline__ float top_of_lanes(float m) {
  uint32_t u = __float_as_uint(m);
#pragma unroll
  for (int i = 1; i < 1 << N; i *= 2)
    u = max(u, __shfl_xor_sync(~0u, u, i));
  return __uint_as_float(u);
}

/// Eight values to p, of which `have` exist; VEC: p is 16-byte aligned.
template <int DT, bool VEC>
__device__ __forceinline__ void store8(typename Value<DT>::T *p, const float2 (&v)[4], int have) {
  uint4 q[DT == SBC_F32 ? 2 : 1];
  uint32_t *w = reinterpret_cast<uint32_t *>(q);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (DT == SBC_F32) {
      w[2 * i & 7] = __float_as_uint(v[i].x);
      w[2 * i + 1 & 7] = __float_as_uint(v[i].y);
    } else {
      w[i] = pack2<DT>(v[i].x, v[i].y);
    }
  }
  if (VEC && have >= 8) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof q / 16); ++i)
      __stcs(reinterpret_cast<uint4 *>(p) + i, q[i]);
  } else {
    using U = typename std::conditional<DT == SBC_F32, uint32_t, uint16_t>::type;
    U *u = reinterpret_cast<U *>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < have)
        u[i] = DT == SBC_F32 ? static_cast<U>(w[i & 7]) : static_cast<U>(w[i >> 1] >> (i & 1) * 16);
  }
}

/// V values of a row, V = 8 or (16-bit types) 16: a thread's share of a block,
/// so that a block's own work is shared by 32 / V lanes. Sixteen lie in one
/// 32-byte sector, taken by one instruction where it is aligned to that.
template <int DT> struct Part {
  static constexpr int kValues = DT == SBC_F32 ? 8 : 16;
  static constexpr int kLanes = 128 / kValues; // per 128 columns
  Raw8<DT> raw[kValues / 8];

  template <bool VEC> __device__ __forceinline__ void load(const typename Value<DT>::T *p, int have) {
    if (VEC && have >= kValues && reinterpret_cast<uintptr_t>(p) % 32 == 0) {
      uint32_t *w = reinterpret_cast<uint32_t *>(raw);
      asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                   : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                   : "l"(p));
    } else {
#pragma unroll
      for (int i = 0; i < kValues / 8; ++i)
        raw[i].template load<VEC>(p + 8 * i, have - 8 * i);
    }
  }

  /// Largest magnitude of the block, from the lanes that share it.
  __device__ __forceinline__ float block_top() const {
    float top = raw[0].top();
    if (kValues == 16)
      top = __uint_as_float(max(__float_as_uint(top), __float_as_uint(raw[kValues / 8 - 1].top())));
    return top_of_lanes<kValues == 8 ? 2 : 1>(top);
  }
};

/// The eight values v in their type, as words.
template <int DT> __device__ __forceinline__ void to_words(uint4 *words, const float2 (&v)[4]) {
  uint32_t *w = reinterpret_cast<uint32_t *>(words);
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (DT == SBC_F32) {
      w[2 * k] = __float_as_uint(v[k].x);
      w[2 * k + 1] = __float_as_uint(v[k].y);
    } else {
      w[k] = pack2<DT>(v[k].x, v[k].y);
    }
}

/// Stores a part's values (32 bytes), of which `have` exist; p is 16-byte
/// aligned.
template <int DT>
__device__ __forceinline__ void store_part(typename Value<DT>::T *p, const uint4 (&q)[2], int have) {
  constexpr int V = Part<DT>::kValues;
  const uint32_t *w = reinterpret_cast<const uint32_t *>(q);
  if (have >= V && reinterpret_cast<uintptr_t>(p) % 32 == 0) {
    asm volatile("st.global.cs.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                 "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
  } else if (have >= V) {
    __stcs(reinterpret_cast<uint4 *>(p), q[0]);
    __stcs(reinterpret_cast<uint4 *>(p) + 1, q[1]);
  } else {
    using U = typename std::conditional<DT == SBC_F32, uint32_t, uint16_t>::type;
    U *u = reinterpret_cast<U *>(p);
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < have)
        u[i] = DT == SBC_F32 ? static_cast<U>(w[i & 7]) : static_cast<U>(w[i / 2 & 7] >> (i & 1) * 16);
  }
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

/// v times one factor.
__device__ __forceinline__ void times(float2 (&v)[4], float f) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    v[i] = __fmul2_rn(v[i], make_float2(f, f));
}

/// Eight 4-bit codes of v (already divided by the scale).
__device__ __forceinline__ uint32_t codes4(const float2 (&v)[4]) {
  uint32_t r;
  asm("{\n .reg .b8 a, b, c, d;\n"
      " cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
      " cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n"
      " mov.b32 %0, {a, b, c, d};\n}"
      : "=r"(r)
      : "f"(v[0].x), "f"(v[0].y), "f"(v[1].x), "f"(v[1].y), "f"(v[2].x), "f"(v[2].y), "f"(v[3].x), "f"(v[3].y));
  return r;
}

/// Eight 8-bit codes rne(v inv) clamped to +-127. Adding 1.5 2^23 in the same
/// step rounds the exact product to a whole number (ties to even) and leaves
/// its two's complement in the low byte: no conversion instruction, whose unit
/// the exponentials need.
__device__ __forceinline__ uint2 codes8(const float2 (&v)[4], float inv) {
  constexpr float kWhole = 12582912.f;
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = __ffma2_rn(v[i], make_float2(inv, inv), make_float2(kWhole, kWhole));
    w[2 * i] = __float_as_uint(fminf(fmaxf(t.x, kWhole - 127.f), kWhole + 127.f));
    w[2 * i + 1] = __float_as_uint(fminf(fmaxf(t.y, kWhole - 127.f), kWhole + 127.f));
  }
  return make_uint2(__byte_perm(__byte_perm(w[0], w[1], 0x0040), __byte_perm(w[2], w[3], 0x0040), 0x5410),
                    __byte_perm(__byte_perm(w[4], w[5], 0x0040), __byte_perm(w[6], w[7], 0x0040), 0x5410));
}

/// The values (before the scale) of eight 4-bit codes, as pairs of 16-bit floats.
/// All four pairs are to be used: with this compiler (12.9) the conversions gave
/// zeros where the upper pairs were not and the upper codes known to be zero.
__device__ __forceinline__ void pairs4(uint32_t (&h)[4], uint32_t codes) {
  asm("{\n .reg .b8 a, b, c, d;\n mov.b32 {a, b, c, d}, %4;\n"
      " cvt.rn.f16x2.e2m1x2 %0, a;\n cvt.rn.f16x2.e2m1x2 %1, b;\n"
      " cvt.rn.f16x2.e2m1x2 %2, c;\n cvt.rn.f16x2.e2m1x2 %3, d;\n}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(codes));
}

/// The same in 32 bits.
__device__ __forceinline__ void values4(float2 (&v)[4], uint32_t codes) {
  uint32_t h[4];
  pairs4(h, codes);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    v[i] = unpack2<SBC_F16>(h[i]);
}

/// The values of eight 8-bit codes with their scale: code + 128 in the last
/// bits of 2^23 + 128 + code, again without a conversion instruction. The
/// product and the difference are exact (a NaN scale gives NaN; an infinite
/// offset cannot arise, 2^(s-6) being at most 2^121).
__device__ __forceinline__ void values8(float2 (&v)[4], uint2 codes, float scale) {
  const uint32_t w[2] = {codes.x ^ 0x80808080u, codes.y ^ 0x80808080u};
  const float offset = -8388736.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 b = make_float2(__uint_as_float(__byte_perm(w[i / 2], 0x4b000000u, 0x7440 + (2 * i & 3))),
                                 __uint_as_float(__byte_perm(w[i / 2], 0x4b000000u, 0x7440 + (2 * i + 1 & 3))));
    v[i] = __fmul2_rn(__fadd2_rn(b, make_float2(offset, offset)), make_float2(scale, scale));
  }
}

// Rows that do not start on 16-byte boundaries. A warp's lanes then take
// neighbouring elements, 32 at a time, and exchange them with the owners of the
// parts through shared memory; each lane loading or storing its own part
// element by element would touch 32 sectors per instruction (five times slower
// for 16-bit values, measured). A warp holds 32 V / 128 rows of 128 elements.

constexpr int kScratch = 1024; // bytes per warp

/// The elements of a warp's rows on their way: fetch() issues the loads,
/// place() hands each lane the V elements of its part.
template <typename U, int V> struct Ragged {
  static constexpr int kRows = V / 4;
  U e[kRows][4];

  /// `rows` of the warp's rows exist, with `n` elements each from p on.
  __device__ __forceinline__ void fetch(const U *p, int64_t stride, int rows, int n) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        e[r][j] = r < rows && lane + 32 * j < n ? __ldg(p + r * stride + lane + 32 * j) : U(0);
  }
  __device__ __forceinline__ void place(uint4 *part, uint8_t *scratch) const {
    const int lane = threadIdx.x & 31;
    U *s = reinterpret_cast<U *>(scratch);
    __syncwarp(); // the last use of the scratch is over
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        s[r * 128 + lane + 32 * j] = e[r][j];
    __syncwarp();
    constexpr int kVec = V * static_cast<int>(sizeof(U)) / 16;
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      part[i] = reinterpret_cast<const uint4 *>(scratch)[lane * kVec + i];
  }
};

/// Stores the lanes' parts (V elements each, as words) to a warp's rows.
template <typename U, int V>
__device__ __forceinline__ void ragged_store(const uint4 *part, uint8_t *scratch, U *p, int64_t stride, int rows, int n) {
  constexpr int kRows = V / 4, kVec = V * static_cast<int>(sizeof(U)) / 16;
  const int lane = threadIdx.x & 31;
  __syncwarp();
#pragma unroll
  for (int i = 0; i < kVec; ++i)
    reinterpret_cast<uint4 *>(scratch)[lane * kVec + i] = part[i];
  __syncwarp();
  const U *s = reinterpret_cast<const U *>(scratch);
#pragma unroll
  for (int r = 0; r < kRows; ++r)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (r < rows && lane + 32 * j < n)
        p[r * stride + lane + 32 * j] = s[r * 128 + lane + 32 * j];
}

/// A type's bits.
template <int DT> using Bits = typename std::conditional<DT == SBC_F32, uint32_t, uint16_t>::type;

} // namespace mx
