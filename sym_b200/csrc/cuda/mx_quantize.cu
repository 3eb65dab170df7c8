// sym_b200 -- microscaled quantisation and its inverse (formats: mx_values.h).
//
// One block of threads takes a tile of 128 columns, 64 or 128 rows: with 128
// rows one 512-byte scale tile in either direction. All kernels are bound by
// memory: they read each value once and write each code once. What it takes
// to get there: loads of all of a thread's parts before the first use, 32
// bytes per thread (one sector), magnitudes compared as packed whole numbers,
// scaling in packed 32-bit pairs, no 64-bit division per part.
//
// Measured (8192 x 8192, captured back to back; bytes of the task over time):
//   rows, f16 26.2 us = 6.5 TB/s, f32 45.3 us = 6.7; both directions in one
//   read, f16 39.1 us = 5.3, f32 64.7 us = 5.3 (the issue of the second
//   direction's instructions, 66 % busy); across alone, f16 34.6 us = 4.9;
//   back to values, f16 26.3 us = 6.5, f32 47.7 us = 6.4, transposed f16
//   30.2 us = 5.6, f32 56 us = 5.4. [28672, 8192] to [in, out]: f16 111 us = 5.4,
//   f32 184 us = 5.8.
//   Rows of 8191 columns (through shared memory per warp): f16 39.9, 61 and,
//   back, 36.7 us; each lane by itself 53, 80 and 196.
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
  uint32_t tiles_c;
};

/// Codes and scale of a thread's part of a block. codes and scales point at
/// this thread's place in the row; `exists`: its block does.
template <int DT, int FMT, int V>
__device__ __forceinline__ void quantize_part(const Raw8<DT> (&in)[V / 8], float top, uint8_t *codes, uint8_t *scales,
                                              bool exists, bool row_exists) {
  const uint32_t byte = scale_byte<FMT>(top);
  const float inv = inverse_scale<FMT>(byte);
  uint32_t w[FMT == SBC_MXFP4 ? V / 8 : V / 4];
#pragma unroll
  for (int i = 0; i < V / 8; ++i) {
    float2 v[4];
    in[i].values(v);
    if (FMT == SBC_MXFP4) {
      times(v, inv);
      w[i] = codes4(v);
    } else {
      const uint2 c = codes8(v, inv);
      w[2 * i] = c.x;
      w[2 * i + 1] = c.y;
    }
  }
  constexpr int kWords = sizeof w / 4;
#pragma unroll
  for (int i = 0; i < kWords; ++i)
    if (byte == 255)
      w[i] = 0;
  if (exists) {
    if constexpr (kWords == 1)
      *reinterpret_cast<uint32_t *>(codes) = w[0];
    else if constexpr (kWords == 2)
      *reinterpret_cast<uint2 *>(codes) = make_uint2(w[0], w[1]);
    else
      *reinterpret_cast<uint4 *>(codes) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  // mxfp4: the bytes of a scale tile's blocks past the row's end are 0
  if ((threadIdx.x & (32 / V - 1)) == 0 && (FMT == SBC_MXFP4 ? row_exists : exists))
    *scales = static_cast<uint8_t>(exists ? byte : 0);
}

/// The words of a scale tile's rows past the matrix's last are 0: no product
/// stores what they scale, but the same values have the same bytes. Thread t
/// < 128 of the block that has the matrix's last row in this tile column. Where
/// the call stands decides what the compiler keeps in registers. Both directions,
/// rows off 16-byte boundaries: first (8192 x 8191 f16 61 us; last 73, with
/// spills); aligned rows: last (8192 x 8192 f32 64.7 us; first 70.2). One
/// direction: last (8192 x 8192 f16 26.2 us; first 26.7).
__device__ __forceinline__ void clear_absent_rows(uint8_t *scales, int64_t rows, int64_t tc, int64_t quads) {
  const int64_t r = ((rows - 1) & ~int64_t{127}) + threadIdx.x;
  if (threadIdx.x < 128 && r >= rows)
    *reinterpret_cast<uint32_t *>(scales + scale_word(r, tc, quads)) = 0;
}

/// The parts of a block's rows from r0 on, whose starts have no alignment.
template <int DT, int UNITS>
__device__ __forceinline__ void load_ragged(Part<DT> (&in)[UNITS], const QuantizeArgs &a, int64_t r0, int64_t c0) {
  __shared__ uint4 scratch[kThreads / 32][kScratch / 16];
  using R = Ragged<Bits<DT>, Part<DT>::kValues>;
  constexpr int kStride = kThreads / Part<DT>::kLanes;
  const int warp = threadIdx.x >> 5;
  const int64_t r = r0 + warp * R::kRows, left = a.cols - c0;
  const Bits<DT> *x = static_cast<const Bits<DT> *>(a.x) + r * a.row_stride + c0;
  R ragged[UNITS];
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
    const int64_t rows = a.rows - r - i * kStride;
    ragged[i].fetch(x + i * kStride * a.row_stride, a.row_stride, rows < R::kRows ? static_cast<int>(rows) : R::kRows,
                    left < kTile ? static_cast<int>(left) : kTile);
  }
#pragma unroll
  for (int i = 0; i < UNITS; ++i)
    ragged[i].place(reinterpret_cast<uint4 *>(&in[i]), reinterpret_cast<uint8_t *>(scratch[warp]));
}

/// Blocks along the columns only: 64 rows (FEW: as many as one unit a thread
/// covers) x 128 columns per block of threads, the loads of all units before
/// the first use.
template <int DT, int FMT, bool FEW, bool VEC>
__global__ void __launch_bounds__(kThreads) k_mx_quantize(const __grid_constant__ QuantizeArgs a) {
  using T = typename Value<DT>::T;
  constexpr int V = Part<DT>::kValues, kLanes = Part<DT>::kLanes, kStride = kThreads / kLanes; // rows between units
  constexpr int kUnits = FEW ? 1 : 64 / kStride;
  // A kernel launched to overlap this one's end may begin its own set-up; it
  // waits for this grid's completion before it reads what is written here.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tr = blockIdx.x / a.tiles_c, tc = blockIdx.x - tr * a.tiles_c;
  const int row = threadIdx.x / kLanes, c8 = threadIdx.x % kLanes * V;
  const int64_t r0 = static_cast<int64_t>(tr) * (kUnits * kStride) + row;
  const int64_t c = static_cast<int64_t>(tc) * kTile + c8, left = a.cols - c;
  const int have = static_cast<int>(left < 0 ? 0 : left < V ? left : V);
  const T *x = static_cast<const T *>(a.x) + r0 * a.row_stride + c;
  const int rows = static_cast<int>(a.rows - r0 < 64 ? a.rows - r0 : 64); // from r0 on
  Part<DT> in[kUnits];
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < kUnits; ++i)
      in[i].template load<true>(x + i * kStride * a.row_stride, i * kStride < rows ? have : 0);
  } else {
    load_ragged<DT, kUnits>(in, a, static_cast<int64_t>(tr) * (kUnits * kStride), static_cast<int64_t>(tc) * kTile);
  }
  const int64_t blocks = blocks_of(a.cols);
  const bool exists = c < blocks * kBlock;
  constexpr int kBytes = FMT == SBC_MXFP4 ? 16 : 32; // of codes per block
  uint8_t *codes = a.codes + r0 * blocks * kBytes + c * kBytes / 32;
  const int64_t code_step = blocks * (kBytes * kStride);
  uint8_t *scales = a.scales + (FMT == SBC_MXFP4 ? scale_word(r0, tc, quads_of(a.cols)) + c8 / 32 : r0 * blocks + c / 32);
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    // mxfp4, 64 rows from a multiple of 64: within a scale tile 32 rows are 4
    // bytes and one row 16
    const int64_t scale_step = FMT == SBC_MXFP4 ? (i * kStride / 32) * 4 + (i * kStride % 32) * 16 : i * kStride * blocks;
    const bool row_exists = i * kStride < rows;
    quantize_part<DT, FMT, V>(in[i].raw, in[i].block_top(), codes + i * code_step, scales + scale_step,
                              row_exists && exists, row_exists);
  }
  if (FMT == SBC_MXFP4 && static_cast<int64_t>(tr + 1) * (kUnits * kStride) >= a.rows)
    clear_absent_rows(a.scales, a.rows, tc, quads_of(a.cols));
}

/// Blocks along the rows, and with ROWS along the columns too, from one read:
/// a tile of 128 x 128 values. 16-bit values: four blocks an SM (64 registers;
/// across alone 34.6 us against 40.6 for 8192 x 8192). 32-bit values: as many
/// registers as hold all of a thread's loads (124, two blocks an SM; three
/// blocks took 79 us for both directions, two 65).
template <int DT, bool ROWS, bool VEC>
__global__ void __launch_bounds__(kThreads, DT == SBC_F32 ? 1 : VEC ? 4 : 3) k_mx_quantize_across(const __grid_constant__ QuantizeArgs a) {
  using T = typename Value<DT>::T;
  const int t = threadIdx.x;
  const uint32_t tr = blockIdx.x / a.tiles_c, tc = blockIdx.x - tr * a.tiles_c;
  const int64_t r0 = static_cast<int64_t>(tr) * kTile, c0 = static_cast<int64_t>(tc) * kTile;
  constexpr int V = Part<DT>::kValues, kLanes = Part<DT>::kLanes, kStride = kThreads / kLanes, kUnits = kTile / kStride;
  const int row0 = t / kLanes, c8 = t % kLanes * V;
  const int64_t c = c0 + c8, left = a.cols - c;
  const int have = static_cast<int>(left < 0 ? 0 : left < V ? left : V);
  const int here = static_cast<int>(a.rows - r0 < kTile ? a.rows - r0 : kTile);
  const T *x = static_cast<const T *>(a.x) + (r0 + row0) * a.row_stride + c;
  extern __shared__ uint4 smem[];
  T *tile = reinterpret_cast<T *>(smem);                           // [128][128]
  uint4 *codes = smem + kTile * kTile * sizeof(T) / 16;            // [128 columns][4]
  uint8_t *scales = reinterpret_cast<uint8_t *>(codes + kTile * 4); // [512]
  const int64_t row_blocks = blocks_of(a.cols);
  if (!VEC && ROWS && here < kTile)
    clear_absent_rows(a.scales, a.rows, tc, quads_of(a.cols));
  uint8_t *row_codes = a.codes + (r0 + row0) * row_blocks * 16 + c / 2;
  uint8_t *row_scales = a.scales + scale_word(r0 + row0, tc, quads_of(a.cols)) + c8 / 32;
  Part<DT> in[kUnits];
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < kUnits; ++i)
      in[i].template load<true>(x + i * kStride * a.row_stride, row0 + i * kStride < here ? have : 0);
  } else {
    load_ragged<DT, kUnits>(in, a, r0, c0);
  }
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    const int row = row0 + i * kStride;
#pragma unroll
    for (int j = 0; j < V / 8; ++j)
      *reinterpret_cast<Raw8<DT> *>(tile + row * kTile + c8 + 8 * j) = in[i].raw[j];
    if (ROWS)
      quantize_part<DT, SBC_MXFP4, V>(in[i].raw, in[i].block_top(), row_codes + i * (kStride * 16) * row_blocks,
                                      row_scales + (i * kStride / 32) * 4 + (i * kStride % 32) * 16,
                                      row < here && c < row_blocks * kBlock, row < here);
  }
  __syncthreads();
  // Blocks along the rows: a thread takes 32 rows of two neighbouring 16-bit
  // columns, or of two 32-bit columns 64 apart, so that the lanes of a warp
  // read neighbouring words and no bank is hit twice.
  const int rb = t >> 6, word = t & 63;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    if (DT != SBC_F32 && half)
      break;
    constexpr int kCols = DT == SBC_F32 ? 1 : 2;
    const int col = DT == SBC_F32 ? word + 64 * half : 2 * word;
    uint32_t w[32], m = 0; // m: the largest magnitudes, as bits
#pragma unroll
    for (int k = 0; k < 32; ++k) {
      w[k] = *reinterpret_cast<const uint32_t *>(tile + (rb * 32 + k) * kTile + col);
      m = DT == SBC_F32 ? max(m, w[k] & 0x7fffffffu) : __vmaxu2(m, w[k] & 0x7fff7fffu);
    }
#pragma unroll
    for (int j = 0; j < kCols; ++j) {
      float2 top = make_float2(__uint_as_float(m), 0.f);
      if (DT != SBC_F32)
        top = unpack2<DT>(m);
      const uint32_t byte = scale_byte<SBC_MXFP4>(j ? top.y : top.x);
      const float inv = inverse_scale<SBC_MXFP4>(byte);
      uint32_t out[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float2 s[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t x0 = w[8 * k + 2 * i], x1 = w[8 * k + 2 * i + 1];
          if (DT == SBC_F32)
            s[i] = make_float2(__uint_as_float(x0), __uint_as_float(x1));
          else // column j of both rows
            s[i] = unpack2<DT>(__byte_perm(x0, x1, j ? 0x7632 : 0x5410));
        }
        times(s, inv);
        out[k] = byte == 255 ? 0 : codes4(s);
      }
      codes[(col + j) * 4 + (rb ^ (col >> 1 & 3))] = make_uint4(out[0], out[1], out[2], out[3]);
      scales[(col + j & 31) * 16 + (col + j >> 5) * 4 + rb] = static_cast<uint8_t>(r0 + rb * 32 < a.rows ? byte : 0);
    }
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
  if (t < 128) { // 0 for the scale tile's rows past the last column
    const int col = (t >> 2) + 32 * (t & 3);
    *reinterpret_cast<uint32_t *>(a.scales_t + scale_word(c0 + col, tr, quads)) =
        c0 + col < a.cols ? reinterpret_cast<const uint32_t *>(scales)[t] : 0;
  }
  if (VEC && ROWS && here < kTile)
    clear_absent_rows(a.scales, a.rows, tc, quads_of(a.cols));
}

struct DequantizeArgs {
  const uint8_t *codes, *scales;
  void *out;
  int64_t rows, cols;
  uint32_t tiles_c, tiles;
};

/// Codes to values, in the layout of the codes: [rows, cols]. A thread takes 8
/// values of a row (4 of 32 bits, so that a warp's stores are contiguous) in
/// each of its units, whose loads all come first.
template <int DT, int FMT, bool FEW, bool VEC>
__global__ void __launch_bounds__(kThreads) k_mx_dequantize(const __grid_constant__ DequantizeArgs a) {
  using T = typename Value<DT>::T;
  constexpr int V = DT == SBC_F32 ? 4 : 8, kLanes = kTile / V, kStride = kThreads / kLanes;
  constexpr int kUnits = FEW ? 1 : 64 / kStride;
  constexpr int kBytes = FMT == SBC_MXFP4 ? 16 : 32; // of codes per block
  using C = typename std::conditional<V * kBytes / 32 == 8, uint2, uint32_t>::type;
  const uint32_t tr = blockIdx.x / a.tiles_c, tc = blockIdx.x - tr * a.tiles_c;
  const int c8 = threadIdx.x % kLanes * V;
  const int64_t r0 = static_cast<int64_t>(tr) * (kUnits * kStride) + threadIdx.x / kLanes;
  const int64_t c = static_cast<int64_t>(tc) * kTile + c8, left = a.cols - c;
  const int have = static_cast<int>(left < V ? left : V);
  const int rows = static_cast<int>(a.rows - r0 < 64 ? a.rows - r0 : 64); // from r0 on
  if (VEC && (have <= 0 || rows <= 0))
    return;
  const int64_t blocks = blocks_of(a.cols);
  const bool exists = c < blocks * kBlock;
  // four 4-bit codes are half a word, which two lanes read
  const uint8_t *codes_at = a.codes + r0 * blocks * kBytes + (c * kBytes / 32 & ~int64_t{3});
  const bool upper = V * kBytes / 32 == 2 && (c & 4);
  const uint8_t *scales = a.scales + (FMT == SBC_MXFP4 ? scale_word(r0, tc, quads_of(a.cols)) + c8 / 32 : r0 * blocks + c / 32);
  C codes[kUnits];
  uint32_t scale[kUnits];
#pragma unroll
  for (int i = 0; i < kUnits; ++i)
    if (i * kStride < rows && (VEC || exists)) {
      const int64_t step = FMT == SBC_MXFP4 ? (i * kStride / 32) * 4 + (i * kStride % 32) * 16 : i * kStride * blocks;
      codes[i] = __ldg(reinterpret_cast<const C *>(codes_at + i * (kStride * kBytes) * blocks));
      scale[i] = __ldg(scales + step);
    }
  T *out = static_cast<T *>(a.out) + r0 * a.cols + c;
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    if (VEC && i * kStride >= rows)
      return;
    float2 v[4];
    const float s = scale_value<FMT>(scale[i]);
    if constexpr (FMT == SBC_MXFP4) {
      values4(v, codes[i]); // the whole word, of which four values are this lane's
      if (V == 4 && upper) {
        v[0] = v[2];
        v[1] = v[3];
      }
      times(v, s);
    } else {
      uint2 w = make_uint2(0, 0);
      if constexpr (V == 8)
        w = codes[i];
      else
        w.x = codes[i];
      values8(v, w, s);
    }
    T *p = out + i * kStride * a.cols;
    if constexpr (!VEC) { // the warp's rows together: kWarpRows, from its first on
      __shared__ uint4 scratch[kThreads / 32][kScratch / 16];
      constexpr int kWarpRows = V / 4;
      uint4 words[2];
      to_words<DT>(words, v);
      const int64_t first = r0 - (threadIdx.x & 31) / kLanes + i * kStride, c0 = static_cast<int64_t>(tc) * kTile;
      const int64_t there = a.rows - first, n = a.cols - c0;
      ragged_store<Bits<DT>, V>(words, reinterpret_cast<uint8_t *>(scratch[threadIdx.x >> 5]),
                                static_cast<Bits<DT> *>(a.out) + first * a.cols + c0, a.cols,
                                there < kWarpRows ? static_cast<int>(there) : kWarpRows,
                                n < kTile ? static_cast<int>(n) : kTile);
    } else if constexpr (V == 8) {
      store8<DT, true>(p, v, have);
    } else if (have >= 4) {
      __stcs(reinterpret_cast<float4 *>(p), make_float4(v[0].x, v[0].y, v[1].x, v[1].y));
    } else {
      const float e[4] = {v[0].x, v[0].y, v[1].x, v[1].y};
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (k < have)
          p[k] = Value<DT>::down(e[k]);
    }
  }
}

/// mxfp4 codes [rows, cols] to values [cols, rows]. The tile's codes go to
/// shared memory, row r at slot 16 (r mod 8) + r / 8 of 18 words: a thread
/// reads one word (8 columns) of each of 8 consecutive rows, the lanes of a
/// warp 16 row groups x 2 words on 32 distinct banks, and writes 8 values of
/// each column as one run (128 values of a column per half-warp).
/// A block takes every gridDim-th tile (16-bit values; one tile with 32-bit
/// ones); the next tile's codes and scales are on their way to registers while
/// this one's values are stored. A lane's eight 32-bit values are stored as one
/// sector: as two halves, [28672, 8192] took 213 us instead of 184.
template <int DT, bool VEC>
__global__ void __launch_bounds__(kThreads, DT == SBC_F32 ? 3 : 4) k_mx_dequantize_t(const __grid_constant__ DequantizeArgs a) {
  using T = typename Value<DT>::T;
  constexpr int kPitch = 18;
  __shared__ uint32_t codes[2][kTile * kPitch];
  __shared__ uint32_t scales[2][kTile];
  const int64_t blocks = blocks_of(a.cols), quads = quads_of(a.cols);
  const int t = threadIdx.x;
  uint4 next[2];
  uint32_t next_scale = 0;
  const auto fetch = [&](uint32_t tile) {
    const uint32_t tr = tile / a.tiles_c, tc = tile - tr * a.tiles_c;
    const int64_t r0 = static_cast<int64_t>(tr) * kTile, block = static_cast<int64_t>(tc) * 4 + (t & 3);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t r = r0 + (t >> 2) + 64 * i;
      if (r < a.rows && block < blocks)
        next[i] = __ldg(reinterpret_cast<const uint4 *>(a.codes + (r * blocks + block) * 16));
    }
    if (t < kTile && r0 + t < a.rows)
      next_scale = __ldg(reinterpret_cast<const uint32_t *>(a.scales + scale_word(r0 + t, tc, quads)));
  };
  if (blockIdx.x < a.tiles)
    fetch(blockIdx.x);
  int buf = 0;
  for (uint32_t tile = blockIdx.x; tile < a.tiles; tile += gridDim.x, buf ^= 1) {
    const uint32_t tr = tile / a.tiles_c, tc = tile - tr * a.tiles_c;
    const int64_t r0 = static_cast<int64_t>(tr) * kTile, c0 = static_cast<int64_t>(tc) * kTile;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = (t >> 2) + 64 * i;
      uint2 *d = reinterpret_cast<uint2 *>(codes[buf] + (16 * (row & 7) + row / 8) * kPitch + 4 * (t & 3));
      d[0] = make_uint2(next[i].x, next[i].y);
      d[1] = make_uint2(next[i].z, next[i].w);
    }
    if (t < kTile)
      scales[buf][t] = next_scale;
    __syncthreads(); // the other buffer's readers are past it: they wrote this one before
    if (tile + gridDim.x < a.tiles)
      fetch(tile + gridDim.x);
    const int ag = t & 15, c = t >> 4; // rows 8 ag + i, columns 8 c + j
    const int64_t r = r0 + 8 * ag;
    const int have = static_cast<int>(a.rows - r < 8 ? a.rows - r : 8);
    if (VEC && (have <= 0 || c0 + 8 * c >= a.cols))
      continue;
    // Two columns at a time from the codes' 16-bit values, which keeps the
    // registers of four blocks to an SM (16-bit values: 64, at the price of 44
    // bytes of spills). What was staged for rows past the end
    // is never stored.
    uint32_t h[8][4];
    float scale[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      pairs4(h[i], codes[buf][(16 * i + ag) * kPitch + c]);
      scale[i] = scale_value<SBC_MXFP4>(scales[buf][8 * ag + i] >> (c >> 2) * 8 & 255);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float2 two[8]; // columns 2 j and 2 j + 1 of eight rows
#pragma unroll
      for (int i = 0; i < 8; ++i)
        two[i] = __fmul2_rn(unpack2<SBC_F16>(h[i][j]), make_float2(scale[i], scale[i]));
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (VEC && c0 + 8 * c + 2 * j + k >= a.cols)
          break;
        float2 col[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          col[i] = k ? make_float2(two[2 * i].y, two[2 * i + 1].y) : make_float2(two[2 * i].x, two[2 * i + 1].x);
        if constexpr (VEC && DT == SBC_F32) {
          uint4 words[2];
          to_words<DT>(words, col);
          store_part<DT>(static_cast<T *>(a.out) + (c0 + 8 * c + 2 * j + k) * a.rows + r, words, have);
        } else if constexpr (VEC) {
          store8<DT, true>(static_cast<T *>(a.out) + (c0 + 8 * c + 2 * j + k) * a.rows + r, col, have);
        } else { // the warp's two columns, 8 apart, together
          __shared__ uint4 scratch[kThreads / 32][kScratch / 16];
          uint4 words[2];
          to_words<DT>(words, col);
          const int64_t first = c0 + 8 * (c & ~1) + 2 * j + k, n = a.rows - r0;
          ragged_store<Bits<DT>, 8>(words, reinterpret_cast<uint8_t *>(scratch[t >> 5]),
                                    static_cast<Bits<DT> *>(a.out) + first * a.rows + r0, 8 * a.rows,
                                    (first < a.cols) + (first + 8 < a.cols), n < kTile ? static_cast<int>(n) : kTile);
        }
      }
    }
  }
}

int width(int dt) { return dt == SBC_F32 ? 4 : 2; }

bool grid_of(int64_t rows, int64_t cols, int tile_rows, uint32_t *tiles_c, uint32_t *grid) {
  const int64_t tc = (cols + kTile - 1) / kTile, n = ((rows + tile_rows - 1) / tile_rows) * tc;
  if (n > INT32_MAX)
    return false;
  *tiles_c = static_cast<uint32_t>(tc);
  *grid = static_cast<uint32_t>(n);
  return true;
}

template <int DT, bool VEC> int launch_quantize(const QuantizeArgs &a, int fmt, bool few, uint32_t grid, cudaStream_t s) {
  if (!a.codes_t) {
    auto k = few ? (fmt == SBC_MXFP4 ? k_mx_quantize<DT, SBC_MXFP4, true, VEC> : k_mx_quantize<DT, SBC_MXINT8, true, VEC>)
                 : (fmt == SBC_MXFP4 ? k_mx_quantize<DT, SBC_MXFP4, false, VEC> : k_mx_quantize<DT, SBC_MXINT8, false, VEC>);
    k<<<grid, kThreads, 0, s>>>(a);
  } else {
    const int bytes = kTile * kTile * static_cast<int>(sizeof(typename Value<DT>::T)) + kTile * 64 + 512;
    const cudaError_t e = a.codes ? sbc::allow_shared<k_mx_quantize_across<DT, true, VEC>>(bytes)
                                  : sbc::allow_shared<k_mx_quantize_across<DT, false, VEC>>(bytes);
    if (e != cudaSuccess)
      return e;
    auto k = a.codes ? k_mx_quantize_across<DT, true, VEC> : k_mx_quantize_across<DT, false, VEC>;
    k<<<grid, kThreads, bytes, s>>>(a);
  }
  sbc::count_launch();
  return cudaGetLastError();
}

template <int DT, bool VEC>
int launch_dequantize(const DequantizeArgs &a, int fmt, int transpose, bool few, uint32_t grid, cudaStream_t s) {
  if (transpose) {
    k_mx_dequantize_t<DT, VEC><<<grid, kThreads, 0, s>>>(a);
  } else {
    auto k =
        few ? (fmt == SBC_MXFP4 ? k_mx_dequantize<DT, SBC_MXFP4, true, VEC> : k_mx_dequantize<DT, SBC_MXINT8, true, VEC>)
            : (fmt == SBC_MXFP4 ? k_mx_dequantize<DT, SBC_MXFP4, false, VEC> : k_mx_dequantize<DT, SBC_MXINT8, false, VEC>);
    k<<<grid, kThreads, 0, s>>>(a);
  }
  sbc::count_launch();
  return cudaGetLastError();
}

/// Whether the row-by-row kernels take one unit a thread: while that fills the
/// SMs at most twice over, a few tokens wait for one load's latency (and more
/// blocks share it) instead of four loads' issue.
bool few_of(int64_t rows, int64_t cols) { return rows * ((cols + kTile - 1) / kTile) <= 16 * 2048; }

} // namespace

extern "C" {

int sbc_mx_quantize(const void *x, int32_t dtype, int64_t rows, int64_t cols, int64_t row_stride, const sbc_mx *along,
                    const sbc_mx *across, void *stream) {
  QuantizeArgs a{};
  uint32_t grid = 0;
  const bool few = few_of(rows, cols);
  if (!x || rows <= 0 || cols <= 0 || (!along && !across) || (across && across->format != SBC_MXFP4) ||
      (along && across && along->format != SBC_MXFP4) || dtype < SBC_F32 || dtype > SBC_BF16 ||
      !grid_of(rows, cols, across ? kTile : few ? (dtype == SBC_F32 ? 16 : 32) : 64, &a.tiles_c, &grid))
    return SBC_EINVAL;
  a.x = x;
  a.rows = rows;
  a.cols = cols;
  a.row_stride = row_stride;
  a.codes = along ? static_cast<uint8_t *>(along->codes) : nullptr;
  a.scales = along ? static_cast<uint8_t *>(along->scales) : nullptr;
  a.codes_t = across ? static_cast<uint8_t *>(across->codes) : nullptr;
  a.scales_t = across ? static_cast<uint8_t *>(across->scales) : nullptr;
  const int fmt = along ? along->format : static_cast<int>(SBC_MXFP4);
  const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && row_stride * width(dtype) % 16 == 0;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
  case SBC_F32:
    return vec ? launch_quantize<SBC_F32, true>(a, fmt, few, grid, s) : launch_quantize<SBC_F32, false>(a, fmt, few, grid, s);
  case SBC_F16:
    return vec ? launch_quantize<SBC_F16, true>(a, fmt, few, grid, s) : launch_quantize<SBC_F16, false>(a, fmt, few, grid, s);
  default:
    return vec ? launch_quantize<SBC_BF16, true>(a, fmt, few, grid, s) : launch_quantize<SBC_BF16, false>(a, fmt, few, grid, s);
  }
}

int sbc_mx_dequantize(const sbc_mx *q, void *out, int32_t dtype, int32_t transpose, void *stream) {
  DequantizeArgs a{};
  uint32_t grid = 0;
  const bool few = q && few_of(q->rows, q->cols);
  if (!q || !out || q->rows <= 0 || q->cols <= 0 || (transpose && q->format != SBC_MXFP4) || dtype < SBC_F32 ||
      dtype > SBC_BF16 || !grid_of(q->rows, q->cols, transpose ? kTile : few ? (dtype == SBC_F32 ? 8 : 16) : 64, &a.tiles_c, &grid))
    return SBC_EINVAL;
  a.tiles = grid;
  // Transposed 16-bit values: the blocks that stay on the SMs, each with the next
  // tile's codes on their way ([28672, 8192] 111 us, one block per tile 120).
  // 32-bit values: one block per tile (184 us, four staying blocks an SM 222).
  if (transpose && dtype != SBC_F32) {
    int device = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e == cudaSuccess)
      e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
    if (e != cudaSuccess)
      return e;
    const uint32_t stay = static_cast<uint32_t>(sms) * 4;
    grid = grid < stay ? grid : stay;
  }
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
    return vec ? launch_dequantize<SBC_F32, true>(a, q->format, transpose, few, grid, s)
               : launch_dequantize<SBC_F32, false>(a, q->format, transpose, few, grid, s);
  case SBC_F16:
    return vec ? launch_dequantize<SBC_F16, true>(a, q->format, transpose, few, grid, s)
               : launch_dequantize<SBC_F16, false>(a, q->format, transpose, few, grid, s);
  default:
    return vec ? launch_dequantize<SBC_BF16, true>(a, q->format, transpose, few, grid, s)
               : launch_dequantize<SBC_BF16, false>(a, q->format, transpose, few, grid, s);
  }
}

} // extern "C"
