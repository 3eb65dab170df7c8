// sym_b200 -- the gated SiLU of a feed-forward layer, h = silu(g) u with
// silu(g) = g / (1 + exp(-g)), whose inputs are kept for the backward pass in
// 8 bits (mxint8: mx_values.h):
//   dg = dh u s (1 + g (1 - s)),  du = dh g s,  s = 1 / (1 + exp(-g))
// with g and u as their 8-bit copies stand for them. The forward pass uses the
// inputs themselves, so h does not depend on the copies.
//
// Bound by memory: for 16-bit values the forward pass reads 4 bytes per
// element and writes 2 + 2.06, the backward pass the same the other way
// round. A thread takes 8 elements of one row, four lanes a block.
#include "barriers.h"
#include "mx_values.h"

namespace {

using namespace mx;

constexpr int kThreads = 256;
constexpr int kUnits = 2; // units of 8 elements per thread

struct GateArgs {
  const void *gate, *up; // forward: inputs; backward: `gate` is dh
  void *h, *dup;         // forward: h; backward: dgate (h) and dup
  int64_t gate_stride, up_stride, h_stride, dup_stride;
  uint8_t *gate_codes, *gate_scales, *up_codes, *up_scales;
  int64_t rows, cols;
  uint32_t row_units; // units of 8 per row, a multiple of 4
  int64_t units;
};

/// 1 / (1 + exp(-g)) from exp(-|g|), which cannot overflow: far below zero the
/// result is exp(g), down to the subnormals.
__device__ __forceinline__ float sigmoid(float g) {
  const float e = expf(-fabsf(g));
  return (g < 0.f ? e : 1.f) / (1.f + e);
}

/// Keep eight values of one block quarter in 8 bits.
__device__ __forceinline__ void keep8(uint8_t *codes, uint8_t *scales, const float (&v)[8], int64_t block, int quarter,
                                      bool in) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    m = abs_max(m, v[i]);
  m = abs_max(m, __shfl_xor_sync(~0u, m, 1));
  m = abs_max(m, __shfl_xor_sync(~0u, m, 2));
  const uint32_t byte = scale_byte<SBC_MXINT8>(m);
  const float inv = inverse_scale<SBC_MXINT8>(byte);
  uint2 w = make_uint2(codes8x4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv),
                       codes8x4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv));
  if (byte == 255)
    w = make_uint2(0, 0);
  if (in) {
    *reinterpret_cast<uint2 *>(codes + block * 32 + quarter * 8) = w;
    if (quarter == 0)
      scales[block] = static_cast<uint8_t>(byte);
  }
}

template <int DT, bool KEEP, bool VEC>
__global__ void __launch_bounds__(kThreads) k_silu_mul(const __grid_constant__ GateArgs a) {
  using T = typename Value<DT>::T;
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    const int64_t unit = (static_cast<int64_t>(blockIdx.x) * kUnits + i) * kThreads + threadIdx.x;
    const bool in = unit < a.units;
    const int64_t r = in ? unit / a.row_units : 0, u8 = in ? unit - r * a.row_units : 0, c = u8 * 8;
    const int have = !in ? 0 : static_cast<int>(a.cols - c < 0 ? 0 : a.cols - c < 8 ? a.cols - c : 8);
    float g[8], u[8], h[8];
    load8<DT, VEC>(g, static_cast<const T *>(a.gate) + r * a.gate_stride + c, have);
    load8<DT, VEC>(u, static_cast<const T *>(a.up) + r * a.up_stride + c, have);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      h[k] = g[k] * sigmoid(g[k]) * u[k];
    store8<DT, VEC>(static_cast<T *>(a.h) + r * a.cols + c, h, have);
    if (KEEP) {
      const int64_t block = r * (a.row_units / 4) + u8 / 4;
      keep8(a.gate_codes, a.gate_scales, g, block, u8 & 3, in);
      keep8(a.up_codes, a.up_scales, u, block, u8 & 3, in);
    }
  }
}

template <int DT, bool VEC>
__global__ void __launch_bounds__(kThreads) k_silu_mul_backward(const __grid_constant__ GateArgs a) {
  using T = typename Value<DT>::T;
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    const int64_t unit = (static_cast<int64_t>(blockIdx.x) * kUnits + i) * kThreads + threadIdx.x;
    if (unit >= a.units)
      return;
    const int64_t r = unit / a.row_units, u8 = unit - r * a.row_units, c = u8 * 8;
    const int have = static_cast<int>(a.cols - c < 0 ? 0 : a.cols - c < 8 ? a.cols - c : 8);
    const int64_t block = r * (a.row_units / 4) + u8 / 4;
    float dh[8], g[8], u[8], dg[8], du[8];
    load8<DT, VEC>(dh, static_cast<const T *>(a.gate) + r * a.gate_stride + c, have);
    const uint2 gw = __ldg(reinterpret_cast<const uint2 *>(a.gate_codes + block * 32 + (u8 & 3) * 8));
    const uint2 uw = __ldg(reinterpret_cast<const uint2 *>(a.up_codes + block * 32 + (u8 & 3) * 8));
    const float gs = scale_value<SBC_MXINT8>(__ldg(a.gate_scales + block));
    const float us = scale_value<SBC_MXINT8>(__ldg(a.up_scales + block));
    values8x4(g, gw.x);
    values8x4(g + 4, gw.y);
    values8x4(u, uw.x);
    values8x4(u + 4, uw.y);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float gv = g[k] * gs, uv = u[k] * us, s = sigmoid(gv);
      dg[k] = dh[k] * uv * (s * (1.f + gv * (1.f - s)));
      du[k] = dh[k] * (gv * s);
    }
    store8<DT, VEC>(static_cast<T *>(a.h) + r * a.h_stride + c, dg, have);
    store8<DT, VEC>(static_cast<T *>(a.dup) + r * a.dup_stride + c, du, have);
  }
}

bool aligned(const void *p, int64_t stride, int width) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * width % 16 == 0;
}

bool shape(GateArgs &a, int64_t rows, int64_t cols, unsigned *grid) {
  if (rows <= 0 || cols <= 0 || blocks_of(cols) > INT32_MAX / 4)
    return false;
  a.rows = rows;
  a.cols = cols;
  a.row_units = static_cast<uint32_t>(blocks_of(cols) * 4);
  a.units = rows * a.row_units;
  const int64_t n = (a.units + kThreads * kUnits - 1) / (kThreads * kUnits);
  if (n > INT32_MAX)
    return false;
  *grid = static_cast<unsigned>(n);
  return true;
}

template <int DT> int launch_forward(const GateArgs &a, bool vec, unsigned grid, cudaStream_t s) {
  const bool keep = a.gate_codes != nullptr;
  auto k = keep ? (vec ? k_silu_mul<DT, true, true> : k_silu_mul<DT, true, false>)
                : (vec ? k_silu_mul<DT, false, true> : k_silu_mul<DT, false, false>);
  k<<<grid, kThreads, 0, s>>>(a);
  sbc::count_launch();
  return cudaGetLastError();
}

template <int DT> int launch_backward(const GateArgs &a, bool vec, unsigned grid, cudaStream_t s) {
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
  unsigned grid = 0;
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
  unsigned grid = 0;
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
