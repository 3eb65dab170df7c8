// sym_b200 -- microscaled quantisation and its inverse (formats: mx_values.h).
//
// One block of threads takes a tile of 128 rows x 128 columns, which is one
// 512-byte scale tile in either direction. All kernels are bound by memory:
// they read each value once and write each code once.
#include "barriers.h"
#include "mx_values.h"

namespace {

using namespace mx;

constexpr int kTile = 128;
constexpr int kThreads = 256;

struct QuantizeArgs {
  const void *x;
  int64_t rows, cols, row_stride;
  uint8_t *codes, *scales;     // blocks along the columns, or NULL
  uint8_t *codes_t, *scales_t; // blocks along the rows: the codes of x^T, or NULL
  uint32_t *clear;             // words set to zero, or NULL
  int64_t clear_words;
  uint32_t tiles_c;
};

/// Blocks along the columns. Thread unit: 8 values of one row; four lanes
/// share a block (two shuffles for its largest magnitude), sixteen a scale
/// word. `u` counts the tile's units, 16 per row.
template <int FMT>
__device__ __forceinline__ void row_unit(const QuantizeArgs &a, const float (&v)[8], int64_t r, int64_t c) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    m = abs_max(m, v[i]);
  m = abs_max(m, __shfl_xor_sync(~0u, m, 1));
  m = abs_max(m, __shfl_xor_sync(~0u, m, 2));
  const uint32_t byte = scale_byte<FMT>(m);
  const float inv = inverse_scale<FMT>(byte);
  float s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    s[i] = v[i] * inv;
  const int64_t blocks = blocks_of(a.cols);
  const bool in = r < a.rows && c < blocks * kBlock;
  const int lane = threadIdx.x & 31;
  if (FMT == SBC_MXFP4) {
    const uint32_t w = byte == 255 ? 0 : codes4(s);
    if (in)
      *reinterpret_cast<uint32_t *>(a.codes + r * blocks * 16 + c / 2) = w;
    // the word of the tile's four blocks; those past the row's end are 0
    uint32_t word = (c < blocks * kBlock ? byte : 0) << ((lane >> 2 & 3) * 8);
    word |= __shfl_xor_sync(~0u, word, 4);
    word |= __shfl_xor_sync(~0u, word, 8);
    if ((lane & 15) == 0 && r < a.rows)
      *reinterpret_cast<uint32_t *>(a.scales + scale_word(r, c >> 7, quads_of(a.cols))) = word;
  } else {
    uint2 w = make_uint2(codes8x4(s[0], s[1], s[2], s[3]), codes8x4(s[4], s[5], s[6], s[7]));
    if (byte == 255)
      w = make_uint2(0, 0);
    if (in) {
      *reinterpret_cast<uint2 *>(a.codes + r * blocks * 32 + c) = w;
      if ((lane & 3) == 0)
        a.scales[r * blocks + c / 32] = static_cast<uint8_t>(byte);
    }
  }
}

template <int DT, int FMT, bool ROWS, bool ACROSS, bool VEC>
__global__ void __launch_bounds__(kThreads) k_mx_quantize(const __grid_constant__ QuantizeArgs a) {
  using T = typename Value<DT>::T;
  // A kernel launched to overlap this one's end may begin its own set-up; it
  // waits for this grid's completion before it reads what is written here.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int t = threadIdx.x;
  for (int64_t i = blockIdx.x * static_cast<int64_t>(kThreads) + t; i < a.clear_words;
       i += static_cast<int64_t>(gridDim.x) * kThreads)
    a.clear[i] = 0;
  const uint32_t tr = blockIdx.x / a.tiles_c, tc = blockIdx.x - tr * a.tiles_c;
  const int64_t r0 = static_cast<int64_t>(tr) * kTile, c0 = static_cast<int64_t>(tc) * kTile;
  const T *x = static_cast<const T *>(a.x);
  const int c8 = (t & 15) * 8;
  const int64_t c = c0 + c8;
  const int have = static_cast<int>(a.cols - c < 0 ? 0 : a.cols - c < 8 ? a.cols - c : 8);
  const int here = static_cast<int>(a.rows - r0 < kTile ? a.rows - r0 : kTile);

  if constexpr (!ACROSS) {
#pragma unroll 4
    for (int i = 0; i < 8; ++i) {
      const int row = (t >> 4) + 16 * i;
      if ((row & ~1) >= here) // the warp's two rows
        break;
      float v[8];
      load8<DT, VEC>(v, x + (r0 + row) * a.row_stride + c, row < here ? have : 0);
      row_unit<FMT>(a, v, r0 + row, c);
    }
  } else {
    extern __shared__ uint4 smem[];
    T *tile = reinterpret_cast<T *>(smem);                           // [128][128]
    uint4 *codes = smem + kTile * kTile * sizeof(T) / 16;            // [128 columns][4]
    uint8_t *scales = reinterpret_cast<uint8_t *>(codes + kTile * 4); // [512]
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int row = (t >> 4) + 16 * i;
      float v[8];
      load8<DT, VEC>(v, x + (r0 + row) * a.row_stride + c, row < here ? have : 0);
      T *d = tile + row * kTile + c8;
      T raw[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        raw[k] = Value<DT>::down(v[k]);
#pragma unroll
      for (int k = 0; k < static_cast<int>(sizeof raw / 16); ++k)
        reinterpret_cast<uint4 *>(d)[k] = reinterpret_cast<const uint4 *>(raw)[k];
      if (ROWS && (row & ~1) < here)
        row_unit<FMT>(a, v, r0 + row, c);
    }
    __syncthreads();
    // Blocks along the rows: a thread takes 32 rows of one column. The lanes
    // of a warp read neighbouring columns, so no bank is hit twice.
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int col = t & 127, rb = (t >> 7) + 2 * i;
      float v[32];
      float m = 0.f;
#pragma unroll
      for (int k = 0; k < 32; ++k) {
        v[k] = Value<DT>::up(tile[(rb * 32 + k) * kTile + col]);
        m = abs_max(m, v[k]);
      }
      const uint32_t byte = scale_byte<SBC_MXFP4>(m);
      const float inv = inverse_scale<SBC_MXFP4>(byte);
      uint32_t w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float s[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
          s[j] = v[8 * k + j] * inv;
        w[k] = byte == 255 ? 0 : codes4(s);
      }
      codes[col * 4 + (rb ^ (col >> 1 & 3))] = make_uint4(w[0], w[1], w[2], w[3]);
      scales[(col & 31) * 16 + (col >> 5) * 4 + rb] = static_cast<uint8_t>(r0 + rb * 32 < a.rows ? byte : 0);
    }
    __syncthreads();
    const int64_t blocks = blocks_of(a.rows), quads = quads_of(a.rows);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int col = (t >> 2) + 64 * i, rb = t & 3;
      if (c0 + col < a.cols && r0 / 32 + rb < blocks)
        *reinterpret_cast<uint4 *>(a.codes_t + (c0 + col) * blocks * 16 + (r0 / 32 + rb) * 16) =
            codes[col * 4 + (rb ^ (col >> 1 & 3))];
    }
    if (t < 128) { // rows of the scale tile past the last column stay as they were
      const int col = (t >> 2) + 32 * (t & 3);
      if (c0 + col < a.cols)
        *reinterpret_cast<uint32_t *>(a.scales_t + scale_word(c0 + col, tr, quads)) =
            reinterpret_cast<const uint32_t *>(scales)[t];
    }
  }
}

struct DequantizeArgs {
  const uint8_t *codes, *scales;
  void *out;
  int64_t rows, cols;
  uint32_t tiles_c;
};

/// Codes to values, in the layout of the codes: [rows, cols]. Thread unit as
/// in k_mx_quantize.
template <int DT, int FMT, bool VEC>
__global__ void __launch_bounds__(kThreads) k_mx_dequantize(const __grid_constant__ DequantizeArgs a) {
  using T = typename Value<DT>::T;
  const uint32_t tr = blockIdx.x / a.tiles_c, tc = blockIdx.x - tr * a.tiles_c;
  const int64_t r0 = static_cast<int64_t>(tr) * kTile;
  const int t = threadIdx.x;
  const int64_t c = static_cast<int64_t>(tc) * kTile + (t & 15) * 8;
  const int have = static_cast<int>(a.cols - c < 8 ? a.cols - c : 8);
  const int64_t blocks = blocks_of(a.cols), quads = quads_of(a.cols);
  if (have <= 0)
    return;
#pragma unroll 4
  for (int i = 0; i < 8; ++i) {
    const int64_t r = r0 + (t >> 4) + 16 * i;
    if (r >= a.rows)
      return;
    float v[8], s;
    if (FMT == SBC_MXFP4) {
      values4(v, __ldg(reinterpret_cast<const uint32_t *>(a.codes + r * blocks * 16 + c / 2)));
      s = scale_value<FMT>(__ldg(a.scales + scale_word(r, c >> 7, quads) + (c >> 5 & 3)));
    } else {
      const uint2 w = __ldg(reinterpret_cast<const uint2 *>(a.codes + r * blocks * 32 + c));
      values8x4(v, w.x);
      values8x4(v + 4, w.y);
      s = scale_value<FMT>(__ldg(a.scales + r * blocks + c / 32));
    }
#pragma unroll
    for (int k = 0; k < 8; ++k)
      v[k] *= s;
    store8<DT, VEC>(static_cast<T *>(a.out) + r * a.cols + c, v, have);
  }
}

/// mxfp4 codes [rows, cols] to values [cols, rows]. The tile's codes go to
/// shared memory, row r at slot 16 (r mod 8) + r / 8 of 18 words: a thread
/// reads one word (8 columns) of each of 8 consecutive rows, the lanes of a
/// warp 16 row groups x 2 words on 32 distinct banks, and writes 8 values of
/// each column as one run (128 values of a column per half-warp).
template <int DT, bool VEC>
__global__ void __launch_bounds__(kThreads) k_mx_dequantize_t(const __grid_constant__ DequantizeArgs a) {
  using T = typename Value<DT>::T;
  constexpr int kPitch = 18;
  __shared__ uint32_t codes[kTile * kPitch];
  __shared__ uint32_t scales[kTile];
  const uint32_t tr = blockIdx.x / a.tiles_c, tc = blockIdx.x - tr * a.tiles_c;
  const int64_t r0 = static_cast<int64_t>(tr) * kTile, c0 = static_cast<int64_t>(tc) * kTile;
  const int64_t blocks = blocks_of(a.cols), quads = quads_of(a.cols);
  const int t = threadIdx.x;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = (t >> 2) + 64 * i, q = t & 3;
    if (r0 + row < a.rows && c0 / 32 + q < blocks) {
      const uint4 w = __ldg(reinterpret_cast<const uint4 *>(a.codes + (r0 + row) * blocks * 16 + (c0 / 32 + q) * 16));
      uint32_t *d = codes + (16 * (row & 7) + row / 8) * kPitch + 4 * q;
      reinterpret_cast<uint2 *>(d)[0] = make_uint2(w.x, w.y);
      reinterpret_cast<uint2 *>(d)[1] = make_uint2(w.z, w.w);
    }
  }
  if (t < kTile && r0 + t < a.rows)
    scales[t] = __ldg(reinterpret_cast<const uint32_t *>(a.scales + scale_word(r0 + t, tc, quads)));
  __syncthreads();
  const int ag = t & 15, c = t >> 4; // rows 8 ag + i, columns 8 c + j
  const int64_t r = r0 + 8 * ag;
  const int have = static_cast<int>(a.rows - r < 8 ? a.rows - r : 8);
  if (have <= 0 || c0 + 8 * c >= a.cols)
    return;
  float v[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (i >= have) { // rows past the end: nothing was staged
#pragma unroll
      for (int j = 0; j < 8; ++j)
        v[i][j] = 0.f;
      continue;
    }
    values4(v[i], codes[(16 * i + ag) * kPitch + c]);
    const float s = scale_value<SBC_MXFP4>(scales[8 * ag + i] >> (c >> 2) * 8 & 255);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      v[i][j] *= s;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (c0 + 8 * c + j >= a.cols)
      return;
    const float col[8] = {v[0][j], v[1][j], v[2][j], v[3][j], v[4][j], v[5][j], v[6][j], v[7][j]};
    store8<DT, VEC>(static_cast<T *>(a.out) + (c0 + 8 * c + j) * a.rows + r, col, have);
  }
}

int width(int dt) { return dt == SBC_F32 ? 4 : 2; }

bool grid_of(int64_t rows, int64_t cols, uint32_t *tiles_c, uint32_t *grid) {
  const int64_t tc = (cols + kTile - 1) / kTile, n = ((rows + kTile - 1) / kTile) * tc;
  if (n > INT32_MAX)
    return false;
  *tiles_c = static_cast<uint32_t>(tc);
  *grid = static_cast<uint32_t>(n);
  return true;
}

template <int DT, bool VEC> int launch_quantize(const QuantizeArgs &a, int fmt, uint32_t grid, cudaStream_t s) {
  if (!a.codes_t) {
    if (fmt == SBC_MXFP4)
      k_mx_quantize<DT, SBC_MXFP4, true, false, VEC><<<grid, kThreads, 0, s>>>(a);
    else
      k_mx_quantize<DT, SBC_MXINT8, true, false, VEC><<<grid, kThreads, 0, s>>>(a);
  } else {
    const int bytes = kTile * kTile * static_cast<int>(sizeof(typename Value<DT>::T)) + kTile * 64 + 512;
    auto k = a.codes ? k_mx_quantize<DT, SBC_MXFP4, true, true, VEC> : k_mx_quantize<DT, SBC_MXFP4, false, true, VEC>;
    const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess)
      return e;
    k<<<grid, kThreads, bytes, s>>>(a);
  }
  sbc::count_launch();
  return cudaGetLastError();
}

template <int DT, bool VEC>
int launch_dequantize(const DequantizeArgs &a, int fmt, int transpose, uint32_t grid, cudaStream_t s) {
  if (transpose)
    k_mx_dequantize_t<DT, VEC><<<grid, kThreads, 0, s>>>(a);
  else if (fmt == SBC_MXFP4)
    k_mx_dequantize<DT, SBC_MXFP4, VEC><<<grid, kThreads, 0, s>>>(a);
  else
    k_mx_dequantize<DT, SBC_MXINT8, VEC><<<grid, kThreads, 0, s>>>(a);
  sbc::count_launch();
  return cudaGetLastError();
}

} // namespace

extern "C" {

int sbc_mx_quantize(const void *x, int32_t dtype, int64_t rows, int64_t cols, int64_t row_stride, const sbc_mx *along,
                    const sbc_mx *across, uint32_t *clear, int64_t clear_words, void *stream) {
  QuantizeArgs a{};
  uint32_t grid = 0;
  if (!x || rows <= 0 || cols <= 0 || (!along && !across) || (across && across->format != SBC_MXFP4) ||
      (along && across && along->format != SBC_MXFP4) || dtype < SBC_F32 || dtype > SBC_BF16 ||
      !grid_of(rows, cols, &a.tiles_c, &grid))
    return SBC_EINVAL;
  a.x = x;
  a.rows = rows;
  a.cols = cols;
  a.row_stride = row_stride;
  a.codes = along ? static_cast<uint8_t *>(along->codes) : nullptr;
  a.scales = along ? static_cast<uint8_t *>(along->scales) : nullptr;
  a.codes_t = across ? static_cast<uint8_t *>(across->codes) : nullptr;
  a.scales_t = across ? static_cast<uint8_t *>(across->scales) : nullptr;
  a.clear = clear;
  a.clear_words = clear ? clear_words : 0;
  const int fmt = along ? along->format : static_cast<int>(SBC_MXFP4);
  const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && row_stride * width(dtype) % 16 == 0;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
  case SBC_F32:
    return vec ? launch_quantize<SBC_F32, true>(a, fmt, grid, s) : launch_quantize<SBC_F32, false>(a, fmt, grid, s);
  case SBC_F16:
    return vec ? launch_quantize<SBC_F16, true>(a, fmt, grid, s) : launch_quantize<SBC_F16, false>(a, fmt, grid, s);
  default:
    return vec ? launch_quantize<SBC_BF16, true>(a, fmt, grid, s) : launch_quantize<SBC_BF16, false>(a, fmt, grid, s);
  }
}

int sbc_mx_dequantize(const sbc_mx *q, void *out, int32_t dtype, int32_t transpose, void *stream) {
  DequantizeArgs a{};
  uint32_t grid = 0;
  if (!q || !out || q->rows <= 0 || q->cols <= 0 || (transpose && q->format != SBC_MXFP4) || dtype < SBC_F32 ||
      dtype > SBC_BF16 || !grid_of(q->rows, q->cols, &a.tiles_c, &grid))
    return SBC_EINVAL;
  a.codes = static_cast<const uint8_t *>(q->codes);
  a.scales = static_cast<const uint8_t *>(q->scales);
  a.out = out;
  a.rows = q->rows;
  a.cols = q->cols;
  const int64_t run = transpose ? q->rows : q->cols;
  const bool vec = reinterpret_cast<uintptr_t>(out) % 16 == 0 && run * width(dtype) % 16 == 0;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
  case SBC_F32:
    return vec ? launch_dequantize<SBC_F32, true>(a, q->format, transpose, grid, s)
               : launch_dequantize<SBC_F32, false>(a, q->format, transpose, grid, s);
  case SBC_F16:
    return vec ? launch_dequantize<SBC_F16, true>(a, q->format, transpose, grid, s)
               : launch_dequantize<SBC_F16, false>(a, q->format, transpose, grid, s);
  default:
    return vec ? launch_dequantize<SBC_BF16, true>(a, q->format, transpose, grid, s)
               : launch_dequantize<SBC_BF16, false>(a, q->format, transpose, grid, s);
  }
}

} // extern "C"
