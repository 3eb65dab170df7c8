// sym_b200 -- the product of two mxfp4 matrices on the tensor cores:
//   y[m, n] = sum_k A[m, k] B[n, k],   A [M, K] (activations), B [N, K] (weights)
// with both operands as 4-bit codes and their scales (mx_values.h), by
// tcgen05.mma kind::mxf4 with one scale per 32 values, accumulated in 32 bits.
//
// Orientation. B's rows are the MMA's M side (128 lanes of the accumulator),
// A's rows its N side (columns): a step for a single token then streams 128
// weight rows against 8 columns, and a warp's store of one accumulator column
// is 32 consecutive values of a row of y.
//
// Split. A CTA takes one tile of 128 rows of B x NT rows of A, and where there
// are few tiles a cluster of CTAs shares one along K. Each then holds a
// partial sum in 32 bits in its shared memory, and the CTAs of the cluster add
// them, each for its part of the tile, in the order of their ranks: no
// workspace, no atomics, the same result every time.
//
// Few rows of A (FUSED): the CTA quantises its part of A itself, straight into
// the shared-memory layout that the tensor cores read, while its first weight
// boxes are in flight. That saves a launch and a round trip through memory.
//
// What bounds it, few rows: the weights' bytes. [28672, 8192] by 1, 16, 64 rows
// of given codes 21.9, 23.4, 26.5 us = 5.7, 5.3, 4.7 TB/s; with quantisation
// in front 23.0, 24.7, 27.8 (its end overlaps the first weight copies).
// Small weights end in latency: one row x [4096, 4096] 5.8 us in a graph, of
// which its bytes are 1.4.
#include "barriers.h"
#include "mx_values.h"

#include <atomic>
#include <cstring>
#include <mutex>
#include <type_traits>

namespace {

using namespace mx;
using namespace sbc;

constexpr int kRowsB = 128;       // rows of B per tile
constexpr int kStep = 256;        // K per stage: 128 bytes of codes per row
constexpr int kScaleStage = 1024; // two scale tiles (2 x 128 of K) of one 128-row group
constexpr int kThreads = 192;     // warp 0 loads, warp 1 multiplies, warps 2-5 quantise and store
constexpr int kMaxSplit = 8;      // portable cluster size
constexpr int kSmemMax = 227 * 1024;
constexpr int kUnits = 4;         // FUSED: units of 8 values of A in flight per thread
// The wait limit is for one step, whose copies or products are awaited. The
// storing warps await all steps of a tile: they add this for each, five times
// what a step takes with every SM streaming at the memory's rate.
constexpr uint64_t kStepNs = 8000;

struct ProductArgs {
  CUtensorMap map_a, map_b; // codes [rows, bytes], boxes of NT (128) rows x 128 bytes, 128-byte swizzle
  const uint8_t *scales_a, *scales_b;
  const void *x; // FUSED: A's values, rows x_stride elements apart
  int64_t x_stride;
  void *y;
  int32_t *fault;
  uint64_t wait_ns;
  int64_t m, n, k;
  uint32_t split;   // CTAs along K
  uint32_t quads;   // scale tiles along K
  uint32_t steps;   // stages along K
  uint32_t tiles_a; // tiles along A
  uint32_t k64;     // MMA steps along K
  int32_t x_vec;    // FUSED: rows of x start on 16-byte boundaries
  int32_t y_vec;    // N is a multiple of 4 and y starts on a 16-byte boundary
  int32_t after_quantize; // launched to overlap the end of the kernel that writes A and its scales
  int32_t withhold;       // test hook: the first CTA issues no copy of B's codes for its first step
};

// Two CTAs fit an SM (228 KB): 100 to 113 KB of stages, and at most 256 of the
// 512 columns of tensor memory, so that one CTA's set-up and sums overlap the
// other's stream.
template <int NT, bool FUSED> struct Shape {
  static constexpr int kBytesB = kRowsB * 128;
  static constexpr int kBytesA = FUSED ? 0 : NT * 128;
  static constexpr int kScales = kBytesB + kBytesA; // offset in a stage: B's, then A's
  static constexpr int kStage = kScales + (FUSED ? 1 : 2) * kScaleStage;
  static constexpr int kStages = FUSED ? 4 : NT <= 32 ? 5 : NT <= 64 ? 4 : 3;
  // FUSED: A's codes and scales per step, beside the ring. A scale tile's 8-row
  // groups are 128 bytes each; only those of NT rows are kept, and the copy to
  // tensor memory reads the next tiles' bytes for the others, whose columns
  // nobody uses.
  static constexpr int kTileA = NT * 16;
  static constexpr int kStepA = FUSED ? NT * 128 : 0;
  static constexpr int kScaleA = FUSED ? 2 * kTileA : 0;
  static constexpr int kAcc = NT < 32 ? 32 : NT;                    // columns of the accumulator
  static constexpr int kCols = kAcc + 16 * kStages <= 128 ? 128 : 256; // + 8 + 8 scale columns per stage
};

// The loading and the multiplying warp run their loops as a whole, and one
// lane is elected inside each issuing instruction. Every value such an
// instruction takes is then the same in all lanes by construction and stays in
// uniform registers; a loop under "one lane only" moves each operand across for
// every instruction, which alone took 212 cycles per product, against the 64
// to 128 that the product needs.
#define SBC_ELECTED(instruction) "{\n .reg .pred one;\n elect.sync _|one, 0xffffffff;\n @one " instruction "\n}"

/// A bounded wait of the whole warp, with one answer for all lanes: a warp
/// whose lanes each went by their own clock could leave a loop in parts, and
/// the tensor-memory loads, stmatrix and elections behind these waits need
/// every lane. The only wait of these kernels, in every warp.
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, uint64_t limit_ns) {
  return __all_sync(~0u, mbar_wait_often(bar, parity, limit_ns));
}

__device__ __forceinline__ void expect_bytes(uint32_t bar, uint32_t bytes) {
  asm volatile(SBC_ELECTED("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;")::"r"(bar), "r"(bytes) : "memory");
}

__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap *map, int32_t x, int32_t y, uint32_t bar) {
  asm volatile(SBC_ELECTED("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
                           "[%0], [%1, {%2, %3}], [%4];")::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
               : "memory");
}

__device__ __forceinline__ void load_bytes(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
  asm volatile(SBC_ELECTED("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];")::"r"(dst),
               "l"(__cvta_generic_to_global(src)), "r"(bytes), "r"(bar)
               : "memory");
}

/// Shared-memory descriptor of K-major codes with the 128-byte swizzle
/// (groups of 8 rows x 128 bytes, 1024 bytes apart).
__device__ __forceinline__ uint64_t codes_desc(uint32_t addr) {
  return static_cast<uint64_t>((addr & 0x3ffff) >> 4) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
/// Of one scale tile: 32 rows of 16 bytes, no swizzle, groups of 8 rows 128
/// bytes apart.
__device__ __forceinline__ uint64_t scales_desc(uint32_t addr) {
  return static_cast<uint64_t>((addr & 0x3ffff) >> 4) | (1ull << 16) | (8ull << 32) | (1ull << 46);
}

/// One 512-byte scale tile to 4 columns of tensor memory, to all four lane quarters.
__device__ __forceinline__ void copy_scales(uint32_t column, uint32_t smem) {
  asm volatile(SBC_ELECTED("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;")::"r"(column), "l"(scales_desc(smem))
               : "memory");
}

__device__ __forceinline__ void multiply(uint32_t d, uint64_t b, uint64_t a, uint32_t idesc, uint32_t scale_b,
                                         uint32_t scale_a, uint32_t accumulate) {
  asm volatile("{\n .reg .pred p, one;\n setp.ne.u32 p, %6, 0;\n elect.sync _|one, 0xffffffff;\n"
               " @one tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}" ::"r"(d),
               "l"(b), "l"(a), "r"(idesc), "r"(scale_b), "r"(scale_a), "r"(accumulate)
               : "memory");
}

__device__ __forceinline__ void commit(uint64_t *bar) {
  asm volatile(SBC_ELECTED("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];")::"r"(
                   smem_addr(bar))
               : "memory");
}

/// kind::mxf4: both types e2m1 (1), scales of powers of two (bit 23), N / 8 at
/// bit 17, M / 128 at bit 27; the K half of a scale word (bytes 0-1 or 2-3) at
/// bits 4 (second operand) and 29 (first operand).
template <int NT> __device__ __forceinline__ uint32_t instruction(uint32_t half) {
  return (1u << 7) | (1u << 10) | (static_cast<uint32_t>(NT / 8) << 17) | (1u << 23) | (1u << 27) | (half << 5) |
         (half << 30);
}

/// 8 or 32 columns of this warp's 32 lanes: register i of a lane holds column i.
__device__ __forceinline__ void read8(uint32_t (&r)[8], uint32_t addr) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void read32(uint32_t (&r)[32], uint32_t addr) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
               "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                 "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                 "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
                 "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]),
                 "=r"(r[30]), "=r"(r[31])
               : "r"(addr)
               : "memory");
}

/// Four values of the partial sums [cols][128] that a CTA of the cluster holds.
__device__ __forceinline__ float4 peer_values(uint32_t addr, uint32_t rank) {
  uint32_t at;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(at)
               : "memory");
  return v;
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <int DT, int XT, int NT, bool FUSED>
__global__ void __launch_bounds__(kThreads) k_mx_product(const __grid_constant__ ProductArgs a) {
  using S = Shape<NT, FUSED>;
  using T = typename Value<DT>::T;
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t full[S::kStages], empty[S::kStages], ready;
  __shared__ uint32_t tmem_base;
  const uint32_t stage0 = (smem_addr(raw) + 1023) & ~1023u;
  const uint32_t own_a = stage0 + S::kStages * S::kStage; // FUSED: the codes of all steps, then the scales
  const int warp = __shfl_sync(~0u, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  const uint32_t tile = blockIdx.x / a.split, rank = blockIdx.x - tile * a.split;
  const uint32_t tb = tile / a.tiles_a, ta = tile - tb * a.tiles_a;
  const uint32_t ks0 = a.steps * rank / a.split, ks1 = a.steps * (rank + 1) / a.split;
  const int64_t m0 = static_cast<int64_t>(ta) * NT;
  const int cols = static_cast<int>(a.m - m0 < NT ? a.m - m0 : NT);
  const int first = static_cast<int>(ks1 - ks0 < S::kStages ? ks1 - ks0 : S::kStages); // stages of the first round

  const auto scale_bytes = [&](uint32_t ks) { return (a.quads - 2 * ks < 2 ? 1u : 2u) * 512u; };
  const auto load_b = [&](uint32_t ks, int st) {
    const uint32_t at = stage0 + st * S::kStage, bar = smem_addr(&full[st]);
    expect_bytes(bar, S::kBytesB + S::kBytesA + (FUSED ? 1 : 2) * scale_bytes(ks));
    if (!(a.withhold && blockIdx.x == 0 && ks == ks0))
      load_box(at, &a.map_b, ks * 128, tb * kRowsB, bar);
    load_bytes(at + S::kScales, a.scales_b + (static_cast<int64_t>(tb) * a.quads + 2 * static_cast<int64_t>(ks)) * 512,
               scale_bytes(ks), bar);
  };

  // The first weights are on their way before anything else: they wait neither
  // for tensor memory nor for the kernel that quantises A.
  if (warp == 0) {
    if (lane == 0) {
      for (int i = 0; i < S::kStages; ++i) {
        mbar_init(&full[i], 1);
        mbar_init(&empty[i], 1);
      }
      mbar_init(&ready, 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    for (int st = 0; st < first; ++st)
      load_b(ks0 + st, st);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_base)),
                 "n"(S::kCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if constexpr (FUSED) if (warp >= 2) {
    const int t = threadIdx.x - 64;
    // 8 values of one row per unit, four lanes a block, 32 units of a row a
    // step; 1, 2 or 4 rows at a time, so that a part of one or two steps
    // keeps all warps busy. The loads of a group of units come before its
    // first use.
    const typename Value<XT>::T *x = static_cast<const typename Value<XT>::T *>(a.x);
    const int in_row = static_cast<int>(ks1 - ks0) * 32;
    const int lg = in_row <= 32 ? 5 : in_row <= 64 ? 6 : 7;
    const uint32_t scales = own_a + (ks1 - ks0) * S::kStepA;
    for (int row = t >> lg; row < cols; row += 128 >> lg) {
      const typename Value<XT>::T *p = x + (m0 + row) * a.x_stride;
      for (int at0 = t & ((1 << lg) - 1); at0 < in_row; at0 += kUnits << lg) {
        Raw8<XT> in[kUnits];
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
          const int at = at0 + (i << lg);
          const int64_t c = static_cast<int64_t>(ks0) * kStep + at * 8;
          const int have = at >= in_row || c >= a.k ? 0 : static_cast<int>(a.k - c < 8 ? a.k - c : 8);
          if (a.x_vec)
            in[i].template load<true>(p + c, have);
          else
            in[i].template load<false>(p + c, have);
        }
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
          const int at = at0 + (i << lg);
          if (at >= in_row) // whole warps
            break;
          const int step = at >> 5, kk = (at & 31) * 8;
          const uint32_t byte = scale_byte<SBC_MXFP4>(top_of_lanes<2>(in[i].top()));
          float2 v[4];
          in[i].values(v);
          times(v, inverse_scale<SBC_MXFP4>(byte));
          const uint32_t w = byte == 255 ? 0 : codes4(v);
          // the 128-byte swizzle: 16-byte chunk kk / 32 of row r lies at chunk (kk / 32) ^ (r mod 8)
          const uint32_t code_at =
              own_a + step * S::kStepA + row * 128 + (((kk >> 5) ^ (row & 7)) << 4) + (kk >> 1 & 15);
          asm volatile("st.shared.u32 [%0], %1;" ::"r"(code_at), "r"(w) : "memory");
          if ((lane & 3) == 0)
            asm volatile("st.shared.u8 [%0], %1;" ::"r"(scales + step * S::kScaleA + (kk >> 7) * S::kTileA +
                                                        row * 16 + (kk >> 5 & 3)),
                         "r"(byte)
                         : "memory");
        }
      }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = __shfl_sync(~0u, tmem_base, 0);
  if (warp == 0) {
    const uint8_t *sa = FUSED ? nullptr : a.scales_a + m0 / 128 * a.quads * 512;
    const auto load_a = [&](uint32_t ks, int st) {
      if (FUSED)
        return;
      const uint32_t at = stage0 + st * S::kStage, bar = smem_addr(&full[st]);
      load_box(at + S::kBytesB, &a.map_a, ks * 128, static_cast<int32_t>(m0), bar);
      load_bytes(at + S::kScales + kScaleStage, sa + static_cast<int64_t>(ks) * 1024, scale_bytes(ks), bar);
    };
    if (!FUSED && a.after_quantize)
      asm volatile("griddepcontrol.wait;" ::: "memory");
    for (int st = 0; st < first; ++st)
      load_a(ks0 + st, st);
    int st = 0;
    uint32_t phase = 0;
    for (uint32_t ks = ks0 + first; ks < ks1; ++ks) {
      if (!warp_wait(&empty[st], phase, a.wait_ns)) {
        *a.fault = 2;
        break;
      }
      load_b(ks, st);
      load_a(ks, st);
      if (++st == S::kStages) {
        st = 0;
        phase ^= 1;
      }
    }
    // Whatever happens to the other warps, leave only once the last copies
    // into each stage have landed.
    for (int i = 0; i < first; ++i)
      warp_wait(&full[i], i < st ? phase ^ 1 : phase, a.wait_ns);
  } else if (warp == 1) {
    // Scales go to tensor memory one stage ahead of the products that use
    // them, so that no product waits for its own. Each stage has columns of its
    // own: a stage is filled again only once the products that read it are done,
    // so nothing still reads the columns that a copy overwrites.
    int st = 0, next = 0;
    uint32_t phase = 0;
    const auto scales = [&](uint32_t ks) {
      if (!warp_wait(&full[next], phase, a.wait_ns))
        return false;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t at = stage0 + next * S::kStage + S::kScales;
      const uint32_t at_sa =
          FUSED ? own_a + (ks1 - ks0) * S::kStepA + (ks - ks0) * S::kScaleA : at + kScaleStage;
      const uint32_t sb = tmem + S::kAcc + next * 16, sa = sb + 8;
      const uint32_t tiles = a.quads - 2 * ks < 2 ? 1 : 2;
      for (uint32_t q = 0; q < tiles; ++q) {
        copy_scales(sb + 4 * q, at + q * 512);
        copy_scales(sa + 4 * q, at_sa + q * (FUSED ? S::kTileA : 512));
      }
      if (++next == S::kStages) {
        next = 0;
        phase ^= 1;
      }
      return true;
    };
    bool ok = scales(ks0);
    for (uint32_t ks = ks0; ks < ks1 && ok; ++ks) {
      if (ks + 1 < ks1)
        ok = scales(ks + 1);
      const uint32_t left = a.k64 - 4 * ks, mmas = left < 4 ? left : 4;
      const uint32_t at = stage0 + st * S::kStage;
      const uint32_t at_a = FUSED ? own_a + (ks - ks0) * S::kStepA : at + S::kBytesB;
      const uint32_t sb = tmem + S::kAcc + st * 16, sa = sb + 8;
      const uint64_t desc_b = codes_desc(at), desc_a = codes_desc(at_a); // 32 bytes on: + 2
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i)
        if (i < mmas)
          multiply(tmem, desc_b + 2 * i, desc_a + 2 * i, instruction<NT>(i & 1), sb + 4 * (i >> 1), sa + 4 * (i >> 1),
                   (ks - ks0) | i);
      commit(&empty[st]);
      if (++st == S::kStages)
        st = 0;
    }
    commit(&ready);
    if (!ok) { // leave once the products in flight are done
      *a.fault = 2;
      warp_wait(&ready, 0, a.wait_ns);
    }
  } else {
    if (!FUSED && a.after_quantize)
      asm volatile("griddepcontrol.wait;" ::: "memory");
    const int quarter = warp & 3; // the lanes of tensor memory that this warp may read
    const int row = quarter * 32 + lane;
    const uint32_t acc = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    if (!warp_wait(&ready, 0, a.wait_ns + (ks1 - ks0) * kStepNs))
      *a.fault = 2;
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    // The part's sums as [cols][128] in the stages, all of which have been read.
    float *part = reinterpret_cast<float *>(raw + (stage0 - smem_addr(raw))) + row;
    constexpr int kBatch = NT < 32 ? 8 : 32;
    for (int c = 0; c < cols; c += kBatch) {
      uint32_t v[kBatch];
      if constexpr (kBatch == 8)
        read8(v, acc + c);
      else
        read32(v, acc + c);
      asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
        part[(c + i) * 128] = __uint_as_float(v[i]);
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(S::kCols) : "memory");
  if (a.split > 1)
    cluster_sync();
  // This CTA's share of the tile's columns of 128 values, a warp per column,
  // four neighbouring values per lane.
  const int c0 = cols * static_cast<int>(rank) / static_cast<int>(a.split);
  const int c1 = cols * static_cast<int>(rank + 1) / static_cast<int>(a.split);
  const int64_t n = static_cast<int64_t>(tb) * kRowsB + lane * 4;
  for (int c = c0 + warp; c < c1; c += kThreads / 32) {
    const uint32_t at = stage0 + (c * 128 + lane * 4) * 4;
    float4 part[kMaxSplit];
#pragma unroll
    for (int r = 0; r < kMaxSplit; ++r)
      if (r < static_cast<int>(a.split))
        part[r] = peer_values(at, r);
    float v[4] = {part[0].x, part[0].y, part[0].z, part[0].w};
#pragma unroll
    for (int r = 1; r < kMaxSplit; ++r)
      if (r < static_cast<int>(a.split)) {
        v[0] += part[r].x;
        v[1] += part[r].y;
        v[2] += part[r].z;
        v[3] += part[r].w;
      }
    T *y = static_cast<T *>(a.y) + (m0 + c) * a.n + n;
    if (a.y_vec && n < a.n) { // n is a multiple of 4, and so is a.n
      alignas(16) T out[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        out[i] = Value<DT>::down(v[i]);
      using V = typename std::conditional<sizeof(T) == 4, uint4, uint2>::type;
      *reinterpret_cast<V *>(y) = *reinterpret_cast<const V *>(out);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < a.n)
          y[i] = Value<DT>::down(v[i]);
    }
  }
  if (a.split > 1)
    cluster_sync(); // nobody leaves while its memory is read
}

// ---------------------------------------------------------------------------
// Many rows: pairs of SMs on tiles of 256 rows of B x NB rows of A.
//
// The two CTAs of a cluster share each MMA (cta_group::2, 256 x NB x 64): each
// holds 128 rows of B, half of the rows of A and the accumulator of its own
// 128 rows, so an SM loads half as many bytes of A per product as alone. The
// grid is persistent, a cluster per pair of SMs; eight epilogue warps empty a
// finished accumulator into registers and let the next tile's products begin
// before they store. Both CTAs' copies count on the barriers of the first
// CTA, whose warp 1 issues all products.
//
// A step of K (256) takes 570 cycles against the 512 of its four products; a
// tile change 3,000 more (the last products' latency, 128 KB of accumulator
// read at about 80 bytes per cycle, the way back to the issuing warp). Two
// accumulators of 192 columns hide the change, but read a sixth more operand
// bytes per product and are slower where the rounds of tiles do not favour
// them; 384 columns in two products a step measured the same within 2 %.
// Measured with the quantisation of A: 8192 x 28672 x 8192 831 us = 4.6
// PFLOP/s (under the power cap, SM clock near 1.35 GHz: 82 % of four times
// cuBLAS's sustained bf16 rate), 2048 x 11008 x 4096 43.7 us = 4.2. Given codes:
// 8192 x 8192 x 8192 199 us = 5.5, 2048 x 4096 x 11008 35.3 us = 5.2, 2048 x 11008
// x 4096 39.2 us = 4.7.
// ---------------------------------------------------------------------------
constexpr int kPairThreads = 384; // warp 0 loads, warp 1 multiplies, warps 4-11 store

struct PairArgs {
  CUtensorMap map_a, map_b;               // codes, boxes of NB / 2 (128) rows x 128 bytes, 128-byte swizzle
  CUtensorMap map_scales_a, map_scales_b; // scale tiles [tiles, 512 bytes], boxes of 2
  void *y;
  int32_t *fault;
  uint64_t wait_ns;
  int64_t m, n;
  uint32_t quads, steps, k64;
  uint32_t tiles_a, tiles_b;
  int32_t y_vec; // N is a multiple of 8 and y starts on a 16-byte boundary
  int32_t after_quantize;
  int32_t withhold; // test hook, as in ProductArgs
};

template <int NB> struct PairShape {
  static constexpr int kBytesB = kRowsB * 128;
  static constexpr int kBytesA = NB / 2 * 128;
  static constexpr int kGroups = (NB + 127) / 128; // 128-row groups of A's scales, all in both CTAs
  static constexpr int kScales = kBytesB + kBytesA;
  static constexpr int kStage = kScales + (1 + kGroups) * kScaleStage;
  static constexpr int kTurn = 8 * 2048; // per epilogue warp 32 columns x 32 lanes of 16-bit values
  static constexpr int kBufs = NB == 256 ? 1 : 2;            // accumulators of NB columns
  static constexpr int kScaleCol = kBufs * NB;               // then, per stage, the scales' columns
  static constexpr int kScaleCols = 8 + 8 * kGroups;
  static constexpr int kFit = (kSmemMax - kTurn - 2048) / kStage;
  static constexpr int kRoom = (512 - kScaleCol) / kScaleCols;
  static constexpr int kStages = kFit < kRoom ? (kFit < 8 ? kFit : 8) : (kRoom < 8 ? kRoom : 8);
  static constexpr int kSmem = kStages * kStage + kTurn + 1024;
};

/// A box into this CTA's shared memory, counted on a barrier of the pair's first CTA.
__device__ __forceinline__ void load_box_pair(uint32_t dst, const CUtensorMap *map, int32_t x, int32_t y, uint32_t bar) {
  asm volatile(SBC_ELECTED("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 "
                           "[%0], [%1, {%2, %3}], [%4];")::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
               : "memory");
}

__device__ __forceinline__ void copy_scales_pair(uint32_t column, uint32_t smem) {
  asm volatile(SBC_ELECTED("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;")::"r"(column), "l"(scales_desc(smem))
               : "memory");
}

__device__ __forceinline__ void multiply_pair(uint32_t d, uint64_t b, uint64_t a, uint32_t idesc, uint32_t scale_b,
                                              uint32_t scale_a, uint32_t accumulate) {
  asm volatile("{\n .reg .pred p, one;\n setp.ne.u32 p, %6, 0;\n elect.sync _|one, 0xffffffff;\n"
               " @one tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}" ::"r"(d),
               "l"(b), "l"(a), "r"(idesc), "r"(scale_b), "r"(scale_a), "r"(accumulate)
               : "memory");
}

/// One arrival on the barrier at the same place in both CTAs, once the
/// products issued so far are done.
__device__ __forceinline__ void commit_pair(uint64_t *bar) {
  asm volatile("{\n .reg .b16 both;\n .reg .pred one;\n mov.b16 both, 3;\n elect.sync _|one, 0xffffffff;\n"
               " @one tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], both;\n}" ::"r"(
                   smem_addr(bar))
               : "memory");
}

__device__ __forceinline__ uint32_t in_first_cta(const uint64_t *bar) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(at) : "r"(smem_addr(bar)));
  return at;
}

/// 32 columns of 16 lanes: registers 4j .. 4j+3 of lane t hold row t / 4,
/// columns 8j + 2 (t mod 4) and the next, then row t / 4 + 8, the same columns.
__device__ __forceinline__ void read16x32(uint32_t (&r)[16], uint32_t addr) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
               "%15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                 "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(addr)
               : "memory");
}

/// Tile `i` of the order: groups of 8 tiles along B, in which B varies fastest,
/// so that the tiles in flight at once share rows of both operands in L2.
__device__ __forceinline__ void pair_tile(const PairArgs &a, uint32_t i, uint32_t &tb, uint32_t &ta) {
  const uint32_t per = 8 * a.tiles_a, g = i / per, r = i - g * per;
  const uint32_t wide = a.tiles_b - 8 * g < 8 ? a.tiles_b - 8 * g : 8;
  ta = r / wide;
  tb = 8 * g + r - ta * wide;
}

template <int DT, int NB>
__global__ void __launch_bounds__(kPairThreads, 1) k_mx_product_pair(const __grid_constant__ PairArgs a) {
  using S = PairShape<NB>;
  using T = typename Value<DT>::T;
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t full[S::kStages], empty[S::kStages], ready[S::kBufs], drained[S::kBufs];
  __shared__ uint32_t tmem_base;
  const uint32_t stage0 = (smem_addr(raw) + 1023) & ~1023u;
  const int warp = __shfl_sync(~0u, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = blockIdx.x & 1, clusters = gridDim.x >> 1, tiles = a.tiles_a * a.tiles_b;

  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < S::kBufs; ++i) {
      mbar_init(&ready[i], 1);
      mbar_init(&drained[i], 16); // eight warps of each CTA
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&tmem_base))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  cluster_sync(); // the other CTA's barriers and columns are there
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = __shfl_sync(~0u, tmem_base, 0);
  if (a.after_quantize)
    asm volatile("griddepcontrol.wait;" ::: "memory");

  if (warp == 0) {
    const uint32_t first_full = in_first_cta(full);
    int st = 0, armed = 0;
    uint32_t phase = 1; // the first round of stages is free
    bool ok = true;
    for (uint32_t i = blockIdx.x >> 1; i < tiles && ok; i += clusters) {
      uint32_t tb, ta;
      pair_tile(a, i, tb, ta);
      const int32_t row_b = static_cast<int32_t>(tb * 256 + rank * 128);
      const int32_t row_a = static_cast<int32_t>(ta * NB + rank * (NB / 2));
      const int32_t scale_b = static_cast<int32_t>((tb * 2 + rank) * a.quads);
      const int32_t scale_a = static_cast<int32_t>(ta * NB / 128 * a.quads);
      for (uint32_t ks = 0; ks < a.steps; ++ks) {
        ok = warp_wait(&empty[st], phase, a.wait_ns);
        if (!ok) {
          *a.fault = 2;
          break;
        }
        if (rank == 0)
          expect_bytes(smem_addr(&full[st]), 2 * S::kStage);
        const uint32_t at = stage0 + st * S::kStage, bar = first_full + 8 * st;
        if (!(a.withhold && blockIdx.x == 0 && armed == 0))
          load_box_pair(at, &a.map_b, ks * 128, row_b, bar);
        load_box_pair(at + S::kBytesB, &a.map_a, ks * 128, row_a, bar);
        load_box_pair(at + S::kScales, &a.map_scales_b, 0, scale_b + 2 * ks, bar);
#pragma unroll
        for (int g = 0; g < S::kGroups; ++g)
          load_box_pair(at + S::kScales + (1 + g) * kScaleStage, &a.map_scales_a, 0, scale_a + g * a.quads + 2 * ks,
                        bar);
        armed = armed < S::kStages ? armed + 1 : armed;
        if (++st == S::kStages) {
          st = 0;
          phase ^= 1;
        }
      }
    }
    // Leave only once the last copies of both CTAs into each stage have
    // landed; the second CTA is held by the cluster barrier below.
    if (rank == 0)
      for (int i = 0; i < armed; ++i)
        warp_wait(&full[i], i < st ? phase ^ 1 : phase, a.wait_ns);
  } else if (warp == 1 && rank == 0) {
    constexpr uint32_t kInstr = (1u << 7) | (1u << 10) | (static_cast<uint32_t>(NB / 8) << 17) | (1u << 23) | (2u << 27);
    // Scales go to tensor memory one stage ahead of the products that use
    // them, to columns of their stage (see k_mx_product).
    int st = 0, next = 0;
    uint32_t phase = 0, turn = 0;
    bool ok = true;
    const auto scales = [&](uint32_t ks) {
      if (!warp_wait(&full[next], phase, a.wait_ns))
        return false;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t at = stage0 + next * S::kStage + S::kScales;
      const uint32_t sb = tmem + S::kScaleCol + next * S::kScaleCols, sa = sb + 8;
      const uint32_t tiles = a.quads - 2 * ks < 2 ? 1 : 2;
      for (uint32_t q = 0; q < tiles; ++q) {
        copy_scales_pair(sb + 4 * q, at + q * 512);
#pragma unroll
        for (int g = 0; g < S::kGroups; ++g)
          copy_scales_pair(sa + 4 * (q * S::kGroups + g), at + (1 + g) * kScaleStage + q * 512);
      }
      if (++next == S::kStages) {
        next = 0;
        phase ^= 1;
      }
      return true;
    };
    for (uint32_t i = blockIdx.x >> 1; i < tiles && ok; i += clusters, ++turn) {
      const uint32_t buf = turn % S::kBufs, use = turn / S::kBufs;
      const uint32_t acc = tmem + buf * NB;
      // A column of scales holds 32 rows; every other tile of 192 rows starts
      // in the middle of a group of 128.
      uint32_t tb, ta;
      pair_tile(a, i, tb, ta);
      const uint32_t skip = NB == 192 ? (ta & 1) * 2 : 0;
      ok = scales(0) && warp_wait(&drained[buf], (use & 1) ^ 1, a.wait_ns);
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      for (uint32_t ks = 0; ks < a.steps && ok; ++ks) {
        if (ks + 1 < a.steps)
          ok = scales(ks + 1);
        const uint32_t left = a.k64 - 4 * ks, mmas = left < 4 ? left : 4;
        const uint32_t at = stage0 + st * S::kStage;
        const uint32_t sb = tmem + S::kScaleCol + st * S::kScaleCols, sa = sb + 8;
        const uint64_t desc_b = codes_desc(at), desc_a = codes_desc(at + S::kBytesB); // 32 bytes on: + 2
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j)
          if (j < mmas)
            multiply_pair(acc, desc_b + 2 * j, desc_a + 2 * j, kInstr | (j & 1) << 5 | (j & 1) << 30, sb + 4 * (j >> 1),
                          sa + 4 * S::kGroups * (j >> 1) + skip, ks | j);
        commit_pair(&empty[st]);
        if (++st == S::kStages)
          st = 0;
      }
      commit_pair(&ready[buf]);
      if (!ok) { // leave once the products in flight are done
        *a.fault = 2;
        warp_wait(&ready[buf], use & 1, a.wait_ns);
      }
    }
  } else if (warp >= 4) {
    const int quarter = warp & 3, half = warp >> 2 & 1; // lanes and columns of this warp
    uint32_t turn = 0;
    for (uint32_t i = blockIdx.x >> 1; i < tiles; i += clusters, ++turn) {
      const uint32_t buf = turn % S::kBufs, use = turn / S::kBufs;
      uint32_t tb, ta;
      pair_tile(a, i, tb, ta);
      if (!warp_wait(&ready[buf], use & 1, a.wait_ns + a.steps * kStepNs)) {
        *a.fault = 2;
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t acc = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + buf * NB + half * (NB / 2);
      const int64_t n = static_cast<int64_t>(tb) * 256 + rank * 128 + quarter * 32;
      const int64_t m0 = static_cast<int64_t>(ta) * NB + half * (NB / 2);
      const int cols = static_cast<int>(a.m - m0 < NB / 2 ? a.m - m0 : NB / 2);
      const auto release = [&] {
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        if (lane == 0)
          asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(in_first_cta(&drained[buf]))
                       : "memory");
      };
      if constexpr (sizeof(T) == 2) {
        // 16 lanes x 32 columns per read: a lane holds two neighbouring columns
        // of one row (an mma fragment), which packs into 16-bit pairs and is
        // stored transposed by stmatrix: [column][32 rows] in shared memory,
        // 64 bytes per column, 16-byte pieces swapped so that eight columns
        // cover all banks. From there each lane stores 16 bytes of a row of y.
        uint32_t p[NB / 64][2][8];
#pragma unroll
        for (int round = 0; round < 2; ++round) { // half the columns at a time bounds the registers
          constexpr int kC = (NB / 64 + 1) / 2, kAll = NB / 64;
          uint32_t v[kC][2][16];
#pragma unroll
          for (int c = 0; c < kC; ++c)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if (round * kC + c < kAll)
                read16x32(v[c][h], acc + (static_cast<uint32_t>(h * 16) << 16) + (round * kC + c) * 32);
          if (round == 0)
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
          else
            release();
#pragma unroll
          for (int c = 0; c < kC && round * kC + c < kAll; ++c)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int k = 0; k < 8; ++k)
                p[round * kC + c][h][k] = pack2<DT>(__uint_as_float(v[c][h][2 * k]), __uint_as_float(v[c][h][2 * k + 1]));
        }
        const uint32_t turn_at = stage0 + S::kStages * S::kStage + (warp - 4) * 2048;
#pragma unroll
        for (int c = 0; c < NB / 64; ++c) {
          if (c * 32 >= cols)
            break;
          __syncwarp();
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int g = 0; g < 2; ++g) { // 16 columns: matrices (rows 0-7, 8-15) x (columns 0-7, 8-15)
              const int col = g * 16 + (lane >> 4) * 8 + (lane & 7), piece = h * 2 + (lane >> 3 & 1);
              const uint32_t at = turn_at + col * 64 + ((piece ^ (col >> 1 & 3)) << 4);
              asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(at),
                           "r"(p[c][h][4 * g]), "r"(p[c][h][4 * g + 1]), "r"(p[c][h][4 * g + 2]),
                           "r"(p[c][h][4 * g + 3])
                           : "memory");
            }
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int col = k * 8 + (lane >> 2), piece = lane & 3;
            uint4 out;
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(out.x), "=r"(out.y), "=r"(out.z), "=r"(out.w)
                         : "r"(turn_at + col * 64 + ((piece ^ (col >> 1 & 3)) << 4)));
            if (c * 32 + col >= cols)
              continue;
            T *y = static_cast<T *>(a.y) + (m0 + c * 32 + col) * a.n + n + piece * 8;
            if (a.y_vec && n + piece * 8 < a.n) {
              *reinterpret_cast<uint4 *>(y) = out;
            } else {
              const T *e = reinterpret_cast<const T *>(&out);
#pragma unroll
              for (int j = 0; j < 8; ++j)
                if (n + piece * 8 + j < a.n)
                  y[j] = e[j];
            }
          }
        }
      } else {
        uint32_t v[NB / 64][32];
#pragma unroll
        for (int c = 0; c < NB / 64; ++c)
          read32(v[c], acc + c * 32);
        release();
        float *y = static_cast<float *>(a.y) + m0 * a.n + n + lane;
        if (n + lane < a.n) {
#pragma unroll
          for (int c = 0; c < NB / 64; ++c)
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (c * 32 + k < cols)
                y[(c * 32 + k) * a.n] = __uint_as_float(v[c][k]);
        }
      }
      __syncwarp();
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  cluster_sync(); // neither CTA leaves while the other still signals or reads here
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

/// SM count of the current device.
int sm_count() {
  static std::atomic<int> known[64];
  int device = 0, sms = 0;
  if (cudaGetDevice(&device) != cudaSuccess)
    return 0;
  if (device < 64 && (sms = known[device].load(std::memory_order_relaxed)))
    return sms;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess)
    return 0;
  if (device < 64)
    known[device].store(sms, std::memory_order_relaxed);
  return sms;
}

struct Plan {
  bool fused;
  int pair; // rows of A of a pair's tile, 0: no pairs
  int nt;
  int64_t tiles_a, tiles_b, steps;
  int split;
};

/// The kernel, tile and split of a product, by its sizes.
///
/// Up to 128 rows of A, one tile of A: the fewest columns that hold it. Its
/// weights are read once, so what counts is that enough of them are on their
/// way: the CTAs of a tile (split) are as many as give each SM one, or two
/// where one alone would pass its ring more than twice (steps > 8). Measured,
/// us, [4096, 4096] (16 steps, 32 tiles) by split 1 / 2 / 4 / 8: one row 10.5 /
/// 8.0 / 6.4 / 6.1, 64 rows 15.6 / 12.8 / 11.7 / 15.0; [28672, 8192] (224
/// tiles): 26.2 / 31.2 / 37.0 / 50.5 with 16 rows; [11008, 4096] (86 tiles) by
/// split 1 / 2 / 3 / 4: 13.0 / 11.9 / 11.6 / 15.1.
///
/// FUSED, a CTA's part of A at most 8 row steps (two loads per thread): one row
/// x [11008, 4096] 9.5 against 10.7 us in two launches; with 12 row steps 10.6
/// against 10.7, with 24 12.6 against 10.8.
///
/// More rows: pairs of SMs with 256, 192 or 128 rows of A a tile, or the tiles of
/// one CTA with their split. The cost of each is the rounds of tiles that the
/// SMs need times a tile's cycles: its steps, the change to the next tile, and no
/// less than its results take to store. The cycles are fits to measured times;
/// over 48 shapes the choice by them loses 0.2 % against the best of the four.
/// Measured, us, pairs of 256 / 192 / 128 / single CTAs, with given codes: 11008 x
/// 4096 x 2048 51.2 / 48.2 / 56.3 / 109; 2048 x 11008 x 4096 38.5 / 44.0 / 55.0 /
/// 75.6; 1003 x 8192 x 1024 10.8 / 12.0 / 13.0 / 19.9; 1003 x 1024 x 8192 16.0 /
/// 15.4 / 14.9 / 12.3; quantised in the call, 256 x 4096 x 4096 13.0 / 11.9 / 11.3 /
/// 12.2; 256 x 1024 x 8192 23.4 / 21.5 / 17.9 / 12.6.
bool plan_of(int64_t m, int64_t n, int64_t k, int sms, Plan *p) {
  p->nt = m <= 8 ? 8 : m <= 16 ? 16 : m <= 32 ? 32 : m <= 64 ? 64 : 128;
  p->tiles_a = (m + p->nt - 1) / p->nt;
  p->tiles_b = (n + kRowsB - 1) / kRowsB;
  p->steps = (k + kStep - 1) / kStep;
  // coordinates of the copies (rows, bytes along K) are 31-bit
  if (sms <= 1 || m > INT32_MAX - 256 || n > INT32_MAX - 256 || k > INT32_MAX || p->tiles_a > INT32_MAX / 8 / p->tiles_b ||
      (m > n ? m : n) / 128 + 2 > INT32_MAX / quads_of(k))
    return false;
  const int64_t tiles = p->tiles_a * p->tiles_b;
  int64_t split = sms / tiles;
  split = split < 1 ? 1 : split > kMaxSplit ? kMaxSplit : split;
  if (p->steps > 8 * split) {
    split = 2 * sms / tiles;
    split = split < 1 ? 1 : split > kMaxSplit ? kMaxSplit : split;
  }
  split = split < p->steps ? split : p->steps;
  const int64_t each = (p->steps + split - 1) / split;
  p->split = static_cast<int>((p->steps + each - 1) / each);
  p->fused = m <= 8 && m * each <= 8;
  p->pair = 0;
  if (m > 128) {
    const double ctas = static_cast<double>(tiles * p->split) / sms, full = ctas < 1 ? 1 : ctas;
    double best = full * each * 480 + (full < 2 ? 1 : full / 2) * 6000;
    const struct { int rows, step, change, least; } pairs[] = {
        {256, 511, 3350, 4700}, {192, 522, 1350, 4000}, {128, 505, 720, 3240}};
    for (const auto &c : pairs) {
      const int64_t t = (m + c.rows - 1) / c.rows * ((n + 255) / 256), rounds = (t + sms / 2 - 1) / (sms / 2);
      const int64_t tile = p->steps * c.step + c.change;
      const double cost = static_cast<double>(rounds) * (tile < c.least ? c.least : tile);
      if (cost < best) {
        best = cost;
        p->pair = c.rows;
      }
    }
  }
  return true;
}

/// Codes [rows, pitch] as boxes of `box_rows` rows x 128 bytes; what lies past
/// the end reads as zero codes.
bool encode_codes(CUtensorMap *map, const void *base, int64_t rows, int64_t pitch, int box_rows) {
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(pitch), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(pitch)};
  const cuuint32_t box[2] = {128, static_cast<cuuint32_t>(box_rows)};
  return encode_tiled(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int DT, int XT, int NT, bool FUSED> int launch(const ProductArgs &a, const Plan &p, cudaStream_t s) {
  using S = Shape<NT, FUSED>;
  auto k = k_mx_product<DT, XT, NT, FUSED>;
  const int own = FUSED ? static_cast<int>((p.steps + p.split - 1) / p.split) * (S::kStepA + S::kScaleA) + 512 : 0;
  const int bytes = S::kStages * S::kStage + own + 1024; // + the alignment of the first stage
  cudaError_t e = allow_shared<k_mx_product<DT, XT, NT, FUSED>>(kSmemMax - 1024);
  if (e != cudaSuccess)
    return e;
  cudaLaunchAttribute attr[2]{};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(p.split);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(p.tiles_a * p.tiles_b * p.split));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(bytes);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = a.after_quantize ? 2 : 1;
  e = cudaLaunchKernelEx(&cfg, k, a);
  if (e == cudaSuccess) {
    count_launch();
    count_wait_launch();
  }
  return e;
}

/// Scale tiles of a matrix [rows, cols] as rows of 512 bytes, boxes of two; what
/// lies past the end reads as 0.
bool encode_scales(CUtensorMap *map, const void *base, int64_t rows, int64_t quads) {
  const cuuint64_t dims[2] = {128, static_cast<cuuint64_t>((rows + 127) / 128 * quads)};
  const cuuint64_t strides[1] = {512};
  const cuuint32_t box[2] = {128, 2};
  return encode_tiled(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE);
}

template <int DT, int NB> int launch_pair(const ProductArgs &a, const sbc_mx *qa, const sbc_mx *qb, int sms, cudaStream_t s) {
  PairArgs args{};
  const int64_t pitch = blocks_of(a.k) * 16;
  if (!encode_codes(&args.map_a, qa->codes, a.m, pitch, NB / 2) ||
      !encode_codes(&args.map_b, qb->codes, a.n, pitch, kRowsB) ||
      !encode_scales(&args.map_scales_a, qa->scales, a.m, a.quads) ||
      !encode_scales(&args.map_scales_b, qb->scales, a.n, a.quads))
    return SBC_EUNSUPPORTED;
  args.y = a.y;
  args.fault = a.fault;
  args.wait_ns = a.wait_ns;
  args.m = a.m;
  args.n = a.n;
  args.quads = a.quads;
  args.steps = a.steps;
  args.k64 = a.k64;
  args.tiles_a = static_cast<uint32_t>((a.m + NB - 1) / NB);
  args.tiles_b = static_cast<uint32_t>((a.n + 255) / 256);
  args.y_vec = a.n % 8 == 0 && reinterpret_cast<uintptr_t>(a.y) % 16 == 0;
  args.after_quantize = a.after_quantize;
  args.withhold = a.withhold;
  auto k = k_mx_product_pair<DT, NB>;
  cudaError_t e = allow_shared<k_mx_product_pair<DT, NB>>(PairShape<NB>::kSmem);
  if (e != cudaSuccess)
    return e;
  const uint32_t tiles = args.tiles_a * args.tiles_b, pairs = static_cast<uint32_t>(sms / 2);
  cudaLaunchAttribute attr[2]{};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(2 * (tiles < pairs ? tiles : pairs));
  cfg.blockDim = dim3(kPairThreads);
  cfg.dynamicSmemBytes = PairShape<NB>::kSmem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = a.after_quantize ? 2 : 1;
  e = cudaLaunchKernelEx(&cfg, k, args);
  if (e == cudaSuccess) {
    count_launch();
    count_wait_launch();
  }
  return e;
}

template <int DT>
int launch_plan(const ProductArgs &a, const Plan &p, const sbc_mx *qa, const sbc_mx *qb, int x_dtype, cudaStream_t s) {
  if (p.pair == 256)
    return launch_pair<DT, 256>(a, qa, qb, sm_count(), s);
  if (p.pair == 192)
    return launch_pair<DT, 192>(a, qa, qb, sm_count(), s);
  if (p.pair)
    return launch_pair<DT, 128>(a, qa, qb, sm_count(), s);
  if (a.x) {
    return x_dtype == SBC_F32   ? launch<DT, SBC_F32, 8, true>(a, p, s)
           : x_dtype == SBC_F16 ? launch<DT, SBC_F16, 8, true>(a, p, s)
                                : launch<DT, SBC_BF16, 8, true>(a, p, s);
  }
  switch (p.nt) {
  case 8:
    return launch<DT, SBC_F32, 8, false>(a, p, s);
  case 16:
    return launch<DT, SBC_F32, 16, false>(a, p, s);
  case 32:
    return launch<DT, SBC_F32, 32, false>(a, p, s);
  case 64:
    return launch<DT, SBC_F32, 64, false>(a, p, s);
  default:
    return launch<DT, SBC_F32, 128, false>(a, p, s);
  }
}

/// Armed by sbc_test_withhold_mx: the wait limit of the next launch.
std::atomic<uint64_t> g_withhold{0};

/// The words in mapped pinned host memory that kernels set to 2 when a wait
/// runs out, one per device (64 bytes apart; devices from 63 on share the
/// last), so that one device's stall says nothing of another's products.
constexpr int kFaultWords = 64, kFaultPitch = 16;
std::atomic<int32_t *> g_fault_words{nullptr};

int32_t *fault_word_of(int32_t *words, int device) {
  return words + kFaultPitch * (device < kFaultWords ? device : kFaultWords - 1);
}

/// The current device's word; allocated with the first product, NULL where that
/// fails (the next product tries again).
int32_t *fault_word() {
  static std::mutex lock;
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess)
    return nullptr;
  int32_t *words = g_fault_words.load(std::memory_order_acquire);
  if (!words) {
    const std::lock_guard<std::mutex> held(lock);
    words = g_fault_words.load(std::memory_order_relaxed);
    if (!words) {
      // legal while some stream is being captured
      cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
      cudaThreadExchangeStreamCaptureMode(&mode);
      void *p = nullptr;
      const size_t bytes = kFaultWords * kFaultPitch * sizeof(int32_t);
      if (cudaHostAlloc(&p, bytes, cudaHostAllocMapped | cudaHostAllocPortable) == cudaSuccess) {
        words = static_cast<int32_t *>(p);
        std::memset(words, 0, bytes);
        g_fault_words.store(words, std::memory_order_release);
      } else {
        cudaGetLastError();
      }
      cudaThreadExchangeStreamCaptureMode(&mode);
    }
  }
  return words ? fault_word_of(words, device) : nullptr;
}

} // namespace

extern "C" {

void sbc_test_withhold_mx(uint64_t wait_limit_ns) { g_withhold.store(wait_limit_ns, std::memory_order_relaxed); }

int sbc_test_mx_plan(int64_t m, int64_t n, int64_t k, int32_t sms, sbc_mx_choice *out) {
  Plan p;
  if (!out || m <= 0 || n <= 0 || k <= 0 || !plan_of(m, n, k, sms, &p))
    return SBC_EINVAL;
  const int64_t pairs = sms / 2, tiles = p.pair ? (m + p.pair - 1) / p.pair * ((n + 255) / 256) : 1;
  *out = sbc_mx_choice{p.pair, p.nt, p.split, p.fused, static_cast<int32_t>(p.pair ? (tiles + pairs - 1) / pairs : 1)};
  return 0;
}

int sbc_mx_take_fault(int32_t device) {
  int32_t *words = g_fault_words.load(std::memory_order_acquire);
  return words && device >= 0 ? __atomic_exchange_n(fault_word_of(words, device), 0, __ATOMIC_RELAXED) : 0;
}

void sbc_test_mx_fault(int32_t device) {
  if (fault_word() && device >= 0)
    __atomic_store_n(fault_word_of(g_fault_words.load(std::memory_order_acquire), device), 2, __ATOMIC_RELAXED);
}

int sbc_mx_fuses_quantize(int64_t m, int64_t n, int64_t k) {
  Plan p;
  return m > 0 && n > 0 && k > 0 && plan_of(m, n, k, sm_count(), &p) && p.fused;
}

int sbc_mx_product(const sbc_mx *a, const void *x, int32_t x_dtype, int64_t x_stride, const sbc_mx *b, void *y,
                   int32_t dtype, int32_t after_quantize, void *stream) {
  Plan p;
  int32_t *fault = fault_word();
  if (!fault)
    return cudaErrorMemoryAllocation;
  if (!a || !b || !y || a->format != SBC_MXFP4 || b->format != SBC_MXFP4 || a->rows <= 0 || b->rows <= 0 ||
      a->cols <= 0 || a->cols != b->cols || dtype < SBC_F32 || dtype > SBC_BF16 ||
      !plan_of(a->rows, b->rows, a->cols, sm_count(), &p) || (x && !p.fused) || (!x && !a->codes))
    return SBC_EINVAL;
  ProductArgs args{};
  const int64_t pitch = blocks_of(a->cols) * 16;
  if ((!x && !encode_codes(&args.map_a, a->codes, a->rows, pitch, p.nt)) ||
      !encode_codes(&args.map_b, b->codes, b->rows, pitch, kRowsB))
    return SBC_EUNSUPPORTED;
  args.scales_a = static_cast<const uint8_t *>(a->scales);
  args.scales_b = static_cast<const uint8_t *>(b->scales);
  args.x = x;
  args.x_stride = x_stride;
  args.x_vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && x_stride * (x_dtype == SBC_F32 ? 4 : 2) % 16 == 0;
  args.y = y;
  args.y_vec = b->rows % 4 == 0 && reinterpret_cast<uintptr_t>(y) % 16 == 0;
  args.fault = fault;
  args.wait_ns = wait_limit_ns();
  if (const uint64_t limit = g_withhold.exchange(0, std::memory_order_relaxed)) {
    args.withhold = 1;
    args.wait_ns = limit;
  }
  args.m = a->rows;
  args.n = b->rows;
  args.k = a->cols;
  args.split = static_cast<uint32_t>(p.split);
  args.quads = static_cast<uint32_t>(quads_of(a->cols));
  args.steps = static_cast<uint32_t>(p.steps);
  args.tiles_a = static_cast<uint32_t>(p.tiles_a);
  args.k64 = static_cast<uint32_t>((a->cols + 63) / 64);
  args.after_quantize = after_quantize;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
  case SBC_F32:
    return launch_plan<SBC_F32>(args, p, a, b, x_dtype, s);
  case SBC_F16:
    return launch_plan<SBC_F16>(args, p, a, b, x_dtype, s);
  default:
    return launch_plan<SBC_BF16>(args, p, a, b, x_dtype, s);
  }
}

} // extern "C"
