// sym_b200 -- the gated SiLU of a feed-forward layer, h = silu(g) u with
// silu(g) = g / (1 + exp(-g)), whose inputs are kept for the backward pass in
// 8 bits (mxint8: mx_values.h):
//   dg = dh u s (1 + g (1 - s)),  du = dh g s,  s = 1 / (1 + exp(-g))
// with g and u as their 8-bit copies stand for them. The forward pass uses the
// inputs themselves, so h does not depend on the copies.
//
// Bound by memory: for 16-bit values the forward pass reads 4 bytes per
// element and writes 2 + 2.06, the backward pass the same the other way
// round. A block of threads takes 16 rows x 128 columns per unit, a thread 8
// elements of a row, four lanes a block of 32.
#include "barriers.h"
#include "mx_values.h"

namespace {

using namespace mx;

constexpr int kThreads = 256;
constexpr int kTile = 128;
constexpr int kUnits = 2; // rows (16 apart) per thread

struct GateArgs {
  const void *gate, *up; // forward: inputs; backward: `gate` is dh
  void *h, *dup;         // forward: h; backward: dgate (h) and dup
  int64_t gate_stride, up_stride, h_stride, dup_stride;
  uint8_t *gate_codes, *gate_scales, *up_codes, *up_scales;
  int64_t rows, cols, blocks;
  uint32_t tiles_c;
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
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return (g < 0.f ? e : 1.f) * r;
}

template <int DT> __device__ __forceinline__ float2 sigmoid2(float2 g) {
  return make_float2(sigmoid<DT>(g.x), sigmoid<DT>(g.y));
}

/// Keep eight values of one block quarter in 8 bits.
template <int DT>
__device__ __forceinline__ void keep8(uint8_t *codes, uint8_t *scales, const Raw8<DT> &raw, const float2 (&v)[4],
                                      int64_t block, int quarter, bool exists) {
  const uint32_t byte = scale_byte<SBC_MXINT8>(top_of_lanes<2>(raw.top()));
  uint2 w = codes8(v, inverse_scale<SBC_MXINT8>(byte));
  if (byte == 255)
    w = make_uint2(0, 0);
  if (exists) {
    __stcs(reinterpret_cast<uint2 *>(codes + block * 32 + quarter * 8), w);
    if (quarter == 0)
      scales[block] = static_cast<uint8_t>(byte);
  }
}

template <int DT, bool KEEP, bool VEC>
__global__ void __launch_bounds__(kThreads) k_silu_mul(const __grid_constant__ GateArgs a) {
  using T = typename Value<DT>::T;
  const uint32_t tr = blockIdx.x / a.tiles_c, tc = blockIdx.x - tr * a.tiles_c;
  const int64_t r0 = static_cast<int64_t>(tr) * (16 * kUnits) + (threadIdx.x >> 4);
  const int64_t c = static_cast<int64_t>(tc) * kTile + (threadIdx.x & 15) * 8;
  const int cols = static_cast<int>(a.cols - c < 0 ? 0 : a.cols - c < 8 ? a.cols - c : 8);
  const T *gate_at = static_cast<const T *>(a.gate) + r0 * a.gate_stride + c;
  const T *up_at = static_cast<const T *>(a.up) + r0 * a.up_stride + c;
  T *h_at = static_cast<T *>(a.h) + r0 * a.cols + c;
  const int64_t block = r0 * a.blocks + c / kBlock;
  Raw8<DT> gate[kUnits], up[kUnits];
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    const int have = r0 + 16 * i < a.rows ? cols : 0;
    gate[i].template load<VEC>(gate_at + 16 * i * a.gate_stride, have);
    up[i].template load<VEC>(up_at + 16 * i * a.up_stride, have);
  }
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    float2 g[4], u[4], h[4];
    gate[i].values(g);
    up[i].values(u);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      h[k] = __fmul2_rn(__fmul2_rn(g[k], sigmoid2<DT>(g[k])), u[k]);
    const bool row_exists = r0 + 16 * i < a.rows;
    if (row_exists)
      store8<DT, VEC>(h_at + 16 * i * a.cols, h, cols);
    if (KEEP) {
      const bool exists = row_exists && c < a.blocks * kBlock;
      keep8(a.gate_codes, a.gate_scales, gate[i], g, block + 16 * i * a.blocks, threadIdx.x & 3, exists);
      keep8(a.up_codes, a.up_scales, up[i], u, block + 16 * i * a.blocks, threadIdx.x & 3, exists);
    }
  }
}

template <int DT, bool VEC>
__global__ void __launch_bounds__(kThreads) k_silu_mul_backward(const __grid_constant__ GateArgs a) {
  using T = typename Value<DT>::T;
  const uint32_t tr = blockIdx.x / a.tiles_c, tc = blockIdx.x - tr * a.tiles_c;
  const int64_t r0 = static_cast<int64_t>(tr) * (16 * kUnits) + (threadIdx.x >> 4);
  const int64_t c = static_cast<int64_t>(tc) * kTile + (threadIdx.x & 15) * 8;
  const int cols = static_cast<int>(a.cols - c < 8 ? a.cols - c : 8);
  if (cols <= 0)
    return;
  Raw8<DT> in[kUnits];
  uint2 gate[kUnits], up[kUnits];
  uint32_t gate_scale[kUnits], up_scale[kUnits];
  const T *dh_at = static_cast<const T *>(a.gate) + r0 * a.gate_stride + c;
  const int64_t block0 = r0 * a.blocks + c / kBlock;
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    const int64_t block = block0 + 16 * i * a.blocks, at = block * 32 + (threadIdx.x & 3) * 8;
    if (r0 + 16 * i < a.rows) {
      in[i].template load<VEC>(dh_at + 16 * i * a.gate_stride, cols);
      gate[i] = __ldg(reinterpret_cast<const uint2 *>(a.gate_codes + at));
      up[i] = __ldg(reinterpret_cast<const uint2 *>(a.up_codes + at));
      gate_scale[i] = __ldg(a.gate_scales + block);
      up_scale[i] = __ldg(a.up_scales + block);
    }
  }
  T *dgate_at = static_cast<T *>(a.h) + r0 * a.h_stride + c, *dup_at = static_cast<T *>(a.dup) + r0 * a.dup_stride + c;
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    if (r0 + 16 * i >= a.rows)
      return;
    float2 dh[4], g[4], u[4], dg[4], du[4];
    in[i].values(dh);
    values8(g, gate[i], scale_value<SBC_MXINT8>(gate_scale[i]));
    values8(u, up[i], scale_value<SBC_MXINT8>(up_scale[i]));
    const float2 one = make_float2(1.f, 1.f);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 s = sigmoid2<DT>(g[k]);
      const float2 rest = __fadd2_rn(one, make_float2(-s.x, -s.y));
      dg[k] = __fmul2_rn(__fmul2_rn(dh[k], u[k]), __fmul2_rn(s, __ffma2_rn(g[k], rest, one)));
      du[k] = __fmul2_rn(dh[k], __fmul2_rn(g[k], s));
    }
    store8<DT, VEC>(dgate_at + 16 * i * a.h_stride, dg, cols);
    store8<DT, VEC>(dup_at + 16 * i * a.dup_stride, du, cols);
  }
}

bool aligned(const void *p, int64_t stride, int width) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * width % 16 == 0;
}

bool shape(GateArgs &a, int64_t rows, int64_t cols, unsigned *grid) {
  if (rows <= 0 || cols <= 0)
    return false;
  a.rows = rows;
  a.cols = cols;
  a.blocks = blocks_of(cols);
  const int64_t tc = (cols + kTile - 1) / kTile, n = (rows + 16 * kUnits - 1) / (16 * kUnits) * tc;
  if (n > INT32_MAX)
    return false;
  a.tiles_c = static_cast<uint32_t>(tc);
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
