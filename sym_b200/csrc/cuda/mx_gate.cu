// sym_b200 -- the gated SiLU of a feed-forward layer, h = silu(g) u with
// silu(g) = g / (1 + exp(-g)), whose inputs are kept for the backward pass in
// 8 bits (mxint8: mx_values.h):
//   dg = dh u s (1 + g (1 - s)),  du = dh g s,  s = 1 / (1 + exp(-g))
// with g and u as their 8-bit copies stand for them. The forward pass uses the
// inputs themselves, so h does not depend on the copies.
//
// Bound by memory: for 16-bit values the forward pass reads 4 bytes per
// element and writes 2 + 2.06, the backward pass the same the other way
// round. A block of threads takes 32 rows x 128 columns, a thread 16 values of
// a row (8 of 32 bits, of two rows), two (four) lanes a block of 32.
// Measured, forward and backward over 8192 x 8192: f16 184.5 us = 5.9 TB/s,
// f32 300 us = 6.3; over 8192 x 11008 bf16 250 us of launches = 5.8. What holds the
// f16 forward pass below a copy is its issue (57 to 64 % busy: exponential,
// reciprocal, two sets of codes per value) beside the loads in flight: four
// blocks an SM (64 registers), three took 197 us for both passes.
#include "barriers.h"
#include "mx_values.h"

namespace {

using namespace mx;

constexpr int kThreads = 256;
constexpr int kTile = 128;
constexpr int kRows = 32;
constexpr uint32_t kMaxY = 32768; // row tiles along the grid's y

struct GateArgs {
  const void *gate, *up; // forward: inputs; backward: `gate` is dh
  void *h, *dup;         // forward: h; backward: dgate (h) and dup
  int64_t gate_stride, up_stride, h_stride, dup_stride;
  uint8_t *gate_codes, *gate_scales, *up_codes, *up_scales;
  int64_t rows, cols, blocks;
};

/// 1 / (1 + exp(-g)) from exp(-|g|), which cannot overflow: far below zero the
/// result is exp(g), down to the subnormals. For results in 16 bits the
/// exponential is 2^(-|g| log2 e), log2 e as a sum of two 32-bit numbers so
/// that one rounding of the exponent is left (|g| 2^-24 of the value), and the
/// reciprocal of 1 .. 2 the hardware's (one unit in the last place): both
/// thousands of times below a 16-bit step. 32-bit results take expf and an exact
/// division.
template <int DT> __device__ __forceinline__ float sigmoid(float g) {
  const float a = -fabsf(g);
  if (DT == SBC_F32) {
    const float e = expf(a);
    return (g < 0.f ? e : 1.f) / (1.f + e);
  }
  const float e = exp2f(fmaf(a, 1.44269502f, a * 1.92596303e-8f));
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e)); // of a normal number
  return (g < 0.f ? e : 1.f) * r;
}

template <int DT> __device__ __forceinline__ float2 sigmoid2(float2 g) {
  return make_float2(sigmoid<DT>(g.x), sigmoid<DT>(g.y));
}

/// Keep a part's values in 8 bits.
template <int DT>
__device__ __forceinline__ void keep(uint8_t *codes, uint8_t *scales, const Part<DT> &in, int64_t block, int at,
                                     bool exists) {
  constexpr int N = Part<DT>::kValues / 8;
  const uint32_t byte = scale_byte<SBC_MXINT8>(in.block_top());
  const float inv = inverse_scale<SBC_MXINT8>(byte);
  uint2 w[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float2 v[4];
    in.raw[i].values(v);
    w[i] = codes8(v, inv);
    if (byte == 255)
      w[i] = make_uint2(0, 0);
  }
  if (exists) {
    if (N == 2)
      __stcs(reinterpret_cast<uint4 *>(codes + block * 32 + at), make_uint4(w[0].x, w[0].y, w[N - 1].x, w[N - 1].y));
    else
      __stcs(reinterpret_cast<uint2 *>(codes + block * 32 + at), w[0]);
    if (at == 0)
      scales[block] = static_cast<uint8_t>(byte);
  }
}

/// Where a thread works: row r0 (and kStride on), column c, `cols` of its values
/// existing.
template <int DT> struct Place {
  static constexpr int kStride = kThreads / Part<DT>::kLanes, kUnits = kRows / kStride;
  int64_t r0, c;
  int cols, in_block;
  __device__ __forceinline__ explicit Place(const GateArgs &a) {
    r0 = (static_cast<int64_t>(blockIdx.z) * kMaxY + blockIdx.y) * kRows + threadIdx.x / Part<DT>::kLanes;
    c = static_cast<int64_t>(blockIdx.x) * kTile + threadIdx.x % Part<DT>::kLanes * Part<DT>::kValues;
    const int64_t left = a.cols - c;
    cols = static_cast<int>(left < 0 ? 0 : left < Part<DT>::kValues ? left : Part<DT>::kValues);
    in_block = static_cast<int>(c % kBlock);
  }
};

/// One matrix's parts of a thread block's rows, and their stores, when rows have
/// no alignment.
template <int DT> struct RaggedRows {
  using U = Bits<DT>;
  using R = Ragged<U, Part<DT>::kValues>;
  static constexpr int kStride = Place<DT>::kStride;
  int64_t r, c0;
  int n;
  uint8_t *scratch;
  __device__ __forceinline__ RaggedRows(const GateArgs &a, uint4 (*shared)[kScratch / 16]) {
    r = (static_cast<int64_t>(blockIdx.z) * kMaxY + blockIdx.y) * kRows + (threadIdx.x >> 5) * R::kRows;
    c0 = static_cast<int64_t>(blockIdx.x) * kTile;
    const int64_t left = a.cols - c0;
    n = static_cast<int>(left < kTile ? left : kTile);
    scratch = reinterpret_cast<uint8_t *>(shared[threadIdx.x >> 5]);
  }
  __device__ __forceinline__ int rows(const GateArgs &a, int unit) const {
    const int64_t there = a.rows - r - unit * kStride;
    return static_cast<int>(there < R::kRows ? there : R::kRows);
  }
  __device__ __forceinline__ void fetch(R &ragged, const GateArgs &a, const void *x, int64_t stride, int unit) const {
    ragged.fetch(static_cast<const U *>(x) + (r + unit * kStride) * stride + c0, stride, rows(a, unit), n);
  }
  __device__ __forceinline__ void store(const GateArgs &a, void *x, int64_t stride, int unit,
                                        const uint4 (&words)[2]) const {
    ragged_store<U, Part<DT>::kValues>(words, scratch, static_cast<U *>(x) + (r + unit * kStride) * stride + c0, stride,
                                       rows(a, unit), n);
  }
};

template <int DT, bool KEEP, bool VEC>
__global__ void __launch_bounds__(kThreads, 4) k_silu_mul(const __grid_constant__ GateArgs a) {
  using T = typename Value<DT>::T;
  using P = Place<DT>;
  constexpr int N = Part<DT>::kValues / 8;
  const P p(a);
  const T *gate_at = static_cast<const T *>(a.gate) + p.r0 * a.gate_stride + p.c;
  const T *up_at = static_cast<const T *>(a.up) + p.r0 * a.up_stride + p.c;
  T *h_at = static_cast<T *>(a.h) + p.r0 * a.cols + p.c;
  const int64_t block = p.r0 * a.blocks + p.c / kBlock;
  Part<DT> gate[P::kUnits], up[P::kUnits];
  __shared__ uint4 scratch[VEC ? 1 : kThreads / 32][kScratch / 16];
  const RaggedRows<DT> ragged(a, scratch);
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < P::kUnits; ++i) {
      const int have = p.r0 + P::kStride * i < a.rows ? p.cols : 0;
      gate[i].template load<true>(gate_at + P::kStride * i * a.gate_stride, have);
      up[i].template load<true>(up_at + P::kStride * i * a.up_stride, have);
    }
  } else {
    typename RaggedRows<DT>::R in[P::kUnits][2];
#pragma unroll
    for (int i = 0; i < P::kUnits; ++i) {
      ragged.fetch(in[i][0], a, a.gate, a.gate_stride, i);
      ragged.fetch(in[i][1], a, a.up, a.up_stride, i);
    }
#pragma unroll
    for (int i = 0; i < P::kUnits; ++i) {
      in[i][0].place(reinterpret_cast<uint4 *>(&gate[i]), ragged.scratch);
      in[i][1].place(reinterpret_cast<uint4 *>(&up[i]), ragged.scratch);
    }
  }
#pragma unroll
  for (int i = 0; i < P::kUnits; ++i) {
    const bool row_exists = p.r0 + P::kStride * i < a.rows;
    if (KEEP) {
      const bool exists = row_exists && p.c < a.blocks * kBlock;
      const int64_t at = block + P::kStride * i * a.blocks;
      keep<DT>(a.gate_codes, a.gate_scales, gate[i], at, p.in_block, exists);
      keep<DT>(a.up_codes, a.up_scales, up[i], at, p.in_block, exists);
    }
    uint4 h[2];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      float2 g[4], u[4], v[4];
      gate[i].raw[j].values(g);
      up[i].raw[j].values(u);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        v[k] = __fmul2_rn(__fmul2_rn(g[k], sigmoid2<DT>(g[k])), u[k]);
      to_words<DT>(h + j, v);
    }
    if constexpr (!VEC)
      ragged.store(a, a.h, a.cols, i, h);
    else if (row_exists)
      store_part<DT>(h_at + P::kStride * i * a.cols, h, p.cols);
  }
}

template <int DT, bool VEC>
__global__ void __launch_bounds__(kThreads) k_silu_mul_backward(const __grid_constant__ GateArgs a) {
  using T = typename Value<DT>::T;
  using P = Place<DT>;
  constexpr int N = Part<DT>::kValues / 8;
  const P p(a);
  if (VEC && p.cols <= 0)
    return;
  __shared__ uint4 scratch[VEC ? 1 : kThreads / 32][kScratch / 16];
  const RaggedRows<DT> ragged(a, scratch);
  typename RaggedRows<DT>::R elements[VEC ? 1 : P::kUnits];
  Part<DT> in[P::kUnits];
  uint2 gate[P::kUnits][N], up[P::kUnits][N];
  uint32_t gate_scale[P::kUnits], up_scale[P::kUnits];
  const T *dh_at = static_cast<const T *>(a.gate) + p.r0 * a.gate_stride + p.c;
  const int64_t block0 = p.r0 * a.blocks + p.c / kBlock;
  const auto codes = [](uint2 (&w)[N], const uint8_t *at) {
    if (N == 2) {
      const uint4 q = __ldg(reinterpret_cast<const uint4 *>(at));
      w[0] = make_uint2(q.x, q.y);
      w[N - 1] = make_uint2(q.z, q.w);
    } else {
      w[0] = __ldg(reinterpret_cast<const uint2 *>(at));
    }
  };
#pragma unroll
  for (int i = 0; i < P::kUnits; ++i) {
    if constexpr (!VEC)
      ragged.fetch(elements[i], a, a.gate, a.gate_stride, i);
    if (p.r0 + P::kStride * i < a.rows && (VEC || p.c < a.blocks * kBlock)) {
      const int64_t block = block0 + P::kStride * i * a.blocks;
      if constexpr (VEC)
        in[i].template load<true>(dh_at + P::kStride * i * a.gate_stride, p.cols);
      codes(gate[i], a.gate_codes + block * 32 + p.in_block);
      codes(up[i], a.up_codes + block * 32 + p.in_block);
      gate_scale[i] = __ldg(a.gate_scales + block);
      up_scale[i] = __ldg(a.up_scales + block);
    }
  }
  T *dgate_at = static_cast<T *>(a.h) + p.r0 * a.h_stride + p.c;
  T *dup_at = static_cast<T *>(a.dup) + p.r0 * a.dup_stride + p.c;
#pragma unroll
  for (int i = 0; i < P::kUnits; ++i) {
    if (VEC && p.r0 + P::kStride * i >= a.rows)
      return;
    if constexpr (!VEC)
      elements[i].place(reinterpret_cast<uint4 *>(&in[i]), ragged.scratch);
    const float gs = scale_value<SBC_MXINT8>(gate_scale[i]), us = scale_value<SBC_MXINT8>(up_scale[i]);
    const float2 one = make_float2(1.f, 1.f);
    uint4 dgate[2], dup[2];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      float2 dh[4], g[4], u[4], dg[4], du[4];
      in[i].raw[j].values(dh);
      values8(g, gate[i][j], gs);
      values8(u, up[i][j], us);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 s = sigmoid2<DT>(g[k]);
        const float2 rest = __fadd2_rn(one, make_float2(-s.x, -s.y));
        dg[k] = __fmul2_rn(__fmul2_rn(dh[k], u[k]), __fmul2_rn(s, __ffma2_rn(g[k], rest, one)));
        du[k] = __fmul2_rn(dh[k], __fmul2_rn(g[k], s));
      }
      to_words<DT>(dgate + j, dg);
      to_words<DT>(dup + j, du);
    }
    if constexpr (VEC) {
      store_part<DT>(dgate_at + P::kStride * i * a.h_stride, dgate, p.cols);
      store_part<DT>(dup_at + P::kStride * i * a.dup_stride, dup, p.cols);
    } else {
      ragged.store(a, a.h, a.h_stride, i, dgate);
      ragged.store(a, a.dup, a.dup_stride, i, dup);
    }
  }
}

bool aligned(const void *p, int64_t stride, int width) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * width % 16 == 0;
}

bool shape(GateArgs &a, int64_t rows, int64_t cols, dim3 *grid) {
  if (rows <= 0 || cols <= 0)
    return false;
  a.rows = rows;
  a.cols = cols;
  a.blocks = blocks_of(cols);
  const int64_t tc = (cols + kTile - 1) / kTile, tr = (rows + kRows - 1) / kRows, z = (tr + kMaxY - 1) / kMaxY;
  if (tc > INT32_MAX || z > 65535)
    return false;
  *grid = dim3(static_cast<unsigned>(tc), static_cast<unsigned>(tr < kMaxY ? tr : kMaxY), static_cast<unsigned>(z));
  return true;
}

template <int DT> int launch_forward(const GateArgs &a, bool vec, dim3 grid, cudaStream_t s) {
  const bool keep = a.gate_codes != nullptr;
  auto k = keep ? (vec ? k_silu_mul<DT, true, true> : k_silu_mul<DT, true, false>)
                : (vec ? k_silu_mul<DT, false, true> : k_silu_mul<DT, false, false>);
  k<<<grid, kThreads, 0, s>>>(a);
  sbc::count_launch();
  return cudaGetLastError();
}

template <int DT> int launch_backward(const GateArgs &a, bool vec, dim3 grid, cudaStream_t s) {
  auto k = vec ? k_silu_mul_backward<DT, true> : k_silu_mul_backward<DT, false>;
  k<<<grid, kThreads, 0, s>>>(a);
  sbc::count_launch();
  return cudaGetLastError();
}

} // namespace

extern "C" {

int sbc_silu_mul(const void *gate, int64_t gate_stride, const void *up, int64_t up_stride, int32_t dtype, int64_t rows,
                 int64_t cols, void *h, const sbc_mx *gate_q, const sbc_mx *up_q, void *stream) {
  GateArgs a{};
  dim3 grid;
  if (!gate || !up || !h || !gate_q != !up_q || dtype < SBC_F32 || dtype > SBC_BF16 || !shape(a, rows, cols, &grid))
    return SBC_EINVAL;
  a.gate = gate;
  a.gate_stride = gate_stride;
  a.up = up;
  a.up_stride = up_stride;
  a.h = h;
  if (gate_q) {
    if (gate_q->format != SBC_MXINT8 || up_q->format != SBC_MXINT8 || gate_q->rows != rows || up_q->rows != rows ||
        gate_q->cols != cols || up_q->cols != cols)
      return SBC_EINVAL;
    a.gate_codes = static_cast<uint8_t *>(gate_q->codes);
    a.gate_scales = static_cast<uint8_t *>(gate_q->scales);
    a.up_codes = static_cast<uint8_t *>(up_q->codes);
    a.up_scales = static_cast<uint8_t *>(up_q->scales);
  }
  const int w = dtype == SBC_F32 ? 4 : 2;
  const bool vec = aligned(gate, gate_stride, w) && aligned(up, up_stride, w) && aligned(h, cols, w);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == SBC_F32   ? launch_forward<SBC_F32>(a, vec, grid, s)
         : dtype == SBC_F16 ? launch_forward<SBC_F16>(a, vec, grid, s)
                            : launch_forward<SBC_BF16>(a, vec, grid, s);
}

int sbc_silu_mul_backward(const void *dh, int64_t dh_stride, int32_t dtype, const sbc_mx *gate_q, const sbc_mx *up_q,
                          void *dgate, int64_t dgate_stride, void *dup, int64_t dup_stride, void *stream) {
  GateArgs a{};
  dim3 grid;
  if (!dh || !gate_q || !up_q || !dgate || !dup || dtype < SBC_F32 || dtype > SBC_BF16 ||
      gate_q->format != SBC_MXINT8 || up_q->format != SBC_MXINT8 || gate_q->rows != up_q->rows ||
      gate_q->cols != up_q->cols || !shape(a, gate_q->rows, gate_q->cols, &grid))
    return SBC_EINVAL;
  a.gate = dh;
  a.gate_stride = dh_stride;
  a.h = dgate;
  a.h_stride = dgate_stride;
  a.dup = dup;
  a.dup_stride = dup_stride;
  a.gate_codes = static_cast<uint8_t *>(gate_q->codes);
  a.gate_scales = static_cast<uint8_t *>(gate_q->scales);
  a.up_codes = static_cast<uint8_t *>(up_q->codes);
  a.up_scales = static_cast<uint8_t *>(up_q->scales);
  const int w = dtype == SBC_F32 ? 4 : 2;
  const bool vec = aligned(dh, dh_stride, w) && aligned(dgate, dgate_stride, w) && aligned(dup, dup_stride, w);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == SBC_F32   ? launch_backward<SBC_F32>(a, vec, grid, s)
         : dtype == SBC_F16 ? launch_backward<SBC_F16>(a, vec, grid, s)
                            : launch_backward<SBC_BF16>(a, vec, grid, s);
}

} // extern "C"
