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
// Split. The work is cut into units of (128 rows of B, NT rows of A, 256 of
// K), numbered with K fastest; CTA c of G takes the units
// [c U / G, (c + 1) U / G). Every CTA so streams the same number of bytes
// whatever the sizes, which is what a few tokens need: there the weights' bytes
// are the whole cost. A tile that several CTAs share is summed by the one that
// arrives last, from the others' 32-bit partials in the order of the CTAs, so
// the result does not depend on which one that is. Nobody waits for another
// CTA.
#include "barriers.h"
#include "mx_values.h"

#include <mutex>

namespace {

using namespace mx;
using namespace sbc;

constexpr int kRowsB = 128;          // rows of B per tile
constexpr int kStep = 256;           // K per stage: 128 bytes of codes per row
constexpr int kScaleStage = 1024;    // two scale tiles (2 x 128 of K) of one 128-row group
constexpr int kThreads = 192;        // warp 0 loads, warp 1 multiplies, warps 2-5 store
constexpr int kSmemMax = 227 * 1024;

struct ProductArgs {
  CUtensorMap map_a, map_b; // codes [rows, bytes], boxes of NT (128) rows x 128 bytes, 128-byte swizzle
  const uint8_t *scales_a, *scales_b;
  void *y;
  float *partials;    // [2 G][NT][128]
  uint32_t *arrivals; // per tile, zero at the start
  int32_t *fault;
  uint64_t wait_ns;
  int64_t m, n;
  int64_t units;
  uint32_t quads;   // scale tiles along K
  uint32_t steps;   // stages along K
  uint32_t tiles_a; // tiles along A
  uint32_t k64;     // MMA steps along K
  int32_t after_quantize; // launched to overlap the end of the kernel that writes A, its scales and `arrivals`
};

template <int NT> struct Shape {
  static constexpr int kBytesB = kRowsB * 128;
  static constexpr int kBytesA = NT * 128;
  static constexpr int kStage = kBytesB + kBytesA + 2 * kScaleStage;
  static constexpr int kStages = (kSmemMax - 2048) / kStage < 12 ? (kSmemMax - 2048) / kStage : 12;
  static constexpr int kSmem = kStages * kStage + 1024; // + the alignment of the first stage
  static constexpr int kAcc = NT < 32 ? 32 : NT;        // columns of one accumulator
  static constexpr int kScaleCol = 2 * kAcc;            // then two buffers of 8 + 8 scale columns
  static constexpr int kCols = kScaleCol + 32 <= 128 ? 128 : kScaleCol + 32 <= 256 ? 256 : 512;
};

__device__ __forceinline__ bool elected() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(p));
  return p != 0;
}

__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap *map, int32_t x, int32_t y, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
               "[%4];" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
               : "memory");
}

__device__ __forceinline__ void load_bytes(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
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
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(column), "l"(scales_desc(smem)) : "memory");
}

__device__ __forceinline__ void multiply(uint32_t d, uint64_t b, uint64_t a, uint32_t idesc, uint32_t scale_b,
                                         uint32_t scale_a, uint32_t accumulate) {
  asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %6, 0;\n"
               " tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}" ::"r"(d),
               "l"(b), "l"(a), "r"(idesc), "r"(scale_b), "r"(scale_a), "r"(accumulate)
               : "memory");
}

__device__ __forceinline__ void commit(uint64_t *bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
               : "memory");
}

/// kind::mxf4: both types e2m1 (1), scales of powers of two (bit 23), N / 8 at
/// bit 17, M / 128 at bit 27; the K half of a scale word (bytes 0-1 or 2-3) at
/// bits 4 (second operand) and 29 (first operand).
template <int NT> __device__ __forceinline__ uint32_t instruction(uint32_t half) {
  return (1u << 7) | (1u << 10) | (static_cast<uint32_t>(NT / 8) << 17) | (1u << 23) | (1u << 27) | (half << 5) |
         (half << 30);
}

__device__ __forceinline__ void read8(float (&v)[8], uint32_t addr) {
  uint32_t r[8];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(addr)
               : "memory");
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 8; ++i)
    v[i] = __uint_as_float(r[i]);
}

/// First unit of CTA c.
__device__ __forceinline__ int64_t first_unit(const ProductArgs &a, uint32_t c) {
  return a.units * c / gridDim.x;
}

template <int DT, int NT>
__global__ void __launch_bounds__(kThreads, 1) k_mx_product(const __grid_constant__ ProductArgs a) {
  using S = Shape<NT>;
  using T = typename Value<DT>::T;
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t full[S::kStages], empty[S::kStages], ready[2], drained[2];
  __shared__ uint32_t tmem_base;
  __shared__ uint32_t last;
  const uint32_t stage0 = (smem_addr(raw) + 1023) & ~1023u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ready[i], 1);
      mbar_init(&drained[i], 128);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_base)),
                 "n"(S::kCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = tmem_base;
  const int64_t begin = first_unit(a, blockIdx.x), end = first_unit(a, blockIdx.x + 1);

  if (warp == 0) {
    if (elected()) {
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&a.map_b)) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&a.map_a)) : "memory");
      const auto scale_bytes = [&](uint32_t ks) { return (a.quads - 2 * ks < 2 ? 1u : 2u) * 512u; };
      const auto load_b = [&](int64_t u, int st) {
        const uint32_t tile = static_cast<uint32_t>(u / a.steps), ks = static_cast<uint32_t>(u % a.steps);
        const uint32_t tb = tile / a.tiles_a, at = stage0 + st * S::kStage, bar = smem_addr(&full[st]);
        load_box(at, &a.map_b, ks * 128, tb * kRowsB, bar);
        load_bytes(at + S::kBytesB + S::kBytesA, a.scales_b + (static_cast<int64_t>(tb) * a.quads + 2 * ks) * 512,
                   scale_bytes(ks), bar);
      };
      const auto load_a = [&](int64_t u, int st) {
        const uint32_t tile = static_cast<uint32_t>(u / a.steps), ks = static_cast<uint32_t>(u % a.steps);
        const uint32_t ta = tile % a.tiles_a, at = stage0 + st * S::kStage, bar = smem_addr(&full[st]);
        load_box(at + S::kBytesB, &a.map_a, ks * 128, ta * NT, bar);
        load_bytes(at + S::kBytesB + S::kBytesA + kScaleStage,
                   a.scales_a + (static_cast<int64_t>(ta) * NT / 128 * a.quads + 2 * ks) * 512, scale_bytes(ks), bar);
      };
      const auto arm = [&](int64_t u, int st) {
        mbar_expect_tx(&full[st], S::kBytesB + S::kBytesA + 2 * scale_bytes(static_cast<uint32_t>(u % a.steps)));
      };
      int64_t u = begin;
      // The first round of stages: the weights' loads do not wait for the
      // kernel that quantises A.
      const int first = static_cast<int>(end - begin < S::kStages ? end - begin : S::kStages);
      for (int st = 0; st < first; ++st) {
        arm(begin + st, st);
        load_b(begin + st, st);
      }
      if (a.after_quantize)
        asm volatile("griddepcontrol.wait;" ::: "memory");
      for (int st = 0; st < first; ++st)
        load_a(begin + st, st);
      u += first;
      int st = 0;
      uint32_t phase = 0;
      for (; u < end; ++u) {
        if (!mbar_wait(&empty[st], phase, a.wait_ns)) {
          *a.fault = 2;
          break;
        }
        arm(u, st);
        load_b(u, st);
        load_a(u, st);
        if (++st == S::kStages) {
          st = 0;
          phase ^= 1;
        }
      }
      // Whatever happens to the other warps, leave only once the last copies
      // into each stage have landed.
      for (int i = 0; i < first; ++i)
        mbar_wait(&full[i], i < st ? phase ^ 1 : phase, a.wait_ns);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elected()) {
      int st = 0;
      uint32_t phase = 0;
      uint32_t seg = 0;
      for (int64_t u = begin; u < end; ++seg) {
        const int64_t tile_end = (u / a.steps + 1) * a.steps;
        const int64_t stop = tile_end < end ? tile_end : end;
        const uint32_t buf = seg & 1;
        const uint32_t acc = tmem + buf * S::kAcc;
        if (seg >= 2 && !mbar_wait(&drained[buf], (seg >> 1) + 1 & 1, a.wait_ns)) {
          *a.fault = 2;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        bool ok = true;
        for (uint32_t fresh = 0; u < stop; ++u, fresh = 1) {
          if (!mbar_wait(&full[st], phase, a.wait_ns)) {
            ok = false;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t ks = static_cast<uint32_t>(u % a.steps);
          const uint32_t left = a.k64 - 4 * ks, mmas = left < 4 ? left : 4;
          const uint32_t at = stage0 + st * S::kStage;
          // Two buffers of scale columns in turn; copies and products of one
          // thread run in order.
          const uint32_t sb = tmem + S::kScaleCol + (st & 1) * 16, sa = sb + 8;
          for (uint32_t q = 0; q < (mmas + 1) / 2; ++q) {
            copy_scales(sb + 4 * q, at + S::kBytesB + S::kBytesA + q * 512);
            copy_scales(sa + 4 * q, at + S::kBytesB + S::kBytesA + kScaleStage + q * 512);
          }
          for (uint32_t i = 0; i < mmas; ++i)
            multiply(acc, codes_desc(at + 32 * i), codes_desc(at + S::kBytesB + 32 * i), instruction<NT>(i & 1),
                     sb + 4 * (i >> 1), sa + 4 * (i >> 1), fresh | i);
          commit(&empty[st]);
          if (++st == S::kStages) {
            st = 0;
            phase ^= 1;
          }
        }
        commit(&ready[buf]);
        if (!ok) { // leave once the products in flight are done
          *a.fault = 2;
          mbar_wait(&ready[buf], seg >> 1 & 1, a.wait_ns);
          break;
        }
      }
    }
    __syncwarp();
  } else {
    const int quarter = warp & 3; // the lanes of tensor memory that this warp may read
    const int row = quarter * 32 + lane;
    if (a.after_quantize)
      asm volatile("griddepcontrol.wait;" ::: "memory");
    uint32_t seg = 0;
    bool ok = true;
    for (int64_t u = begin; u < end && ok; ++seg) {
      const int64_t tile = u / a.steps, tile_begin = tile * a.steps, tile_end = tile_begin + a.steps;
      const int64_t stop = tile_end < end ? tile_end : end;
      const uint32_t buf = seg & 1;
      const uint32_t acc = tmem + buf * S::kAcc + (static_cast<uint32_t>(quarter * 32) << 16);
      ok = mbar_wait(&ready[buf], seg >> 1 & 1, a.wait_ns);
      if (!ok) {
        *a.fault = 2;
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const int64_t tb = tile / a.tiles_a, ta = tile % a.tiles_a;
      const int64_t n = tb * kRowsB + row, m0 = ta * NT;
      T *y = static_cast<T *>(a.y) + m0 * a.n + n;
      const bool whole = u == tile_begin && stop == tile_end;
      const int cols = static_cast<int>(a.m - m0 < NT ? a.m - m0 : NT);
      if (whole) {
        for (int c = 0; c < cols; c += 8) {
          float v[8];
          read8(v, acc + c);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (n < a.n && c + i < cols)
              y[(c + i) * a.n] = Value<DT>::down(v[i]);
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        mbar_arrive(&drained[buf]);
      } else {
        float *mine = a.partials + (2 * static_cast<int64_t>(blockIdx.x) + (u != begin)) * NT * 128 + row;
        for (int c = 0; c < cols; c += 8) {
          float v[8];
          read8(v, acc + c);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (c + i < cols)
              __stcg(mine + (c + i) * 128, v[i]);
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        mbar_arrive(&drained[buf]);
        // the CTAs that share the tile: [c0, c1]
        uint32_t c0 = blockIdx.x, c1 = blockIdx.x;
        while (first_unit(a, c0) > tile_begin)
          --c0;
        while (first_unit(a, c1 + 1) < tile_end)
          ++c1;
        __threadfence();
        asm volatile("bar.sync 1, 128;" ::: "memory");
        if (row == 0)
          last = atomicAdd(a.arrivals + tile, 1u) == c1 - c0;
        asm volatile("bar.sync 1, 128;" ::: "memory");
        if (last) {
          __threadfence();
          for (int c = 0; c < cols; c += 8) {
            float v[8] = {};
            for (uint32_t p = c0; p <= c1; ++p) {
              const int64_t pu = first_unit(a, p);
              const float *theirs =
                  a.partials + (2 * static_cast<int64_t>(p) + (pu < tile_begin)) * NT * 128 + row;
#pragma unroll
              for (int i = 0; i < 8; ++i)
                if (c + i < cols)
                  v[i] += __ldcg(theirs + (c + i) * 128);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (n < a.n && c + i < cols)
                y[(c + i) * a.n] = Value<DT>::down(v[i]);
          }
        }
        asm volatile("bar.sync 1, 128;" ::: "memory"); // `last` is read before it is written again
      }
      u = stop;
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(S::kCols) : "memory");
}

int sm_count() {
  int device = 0, sms = 0;
  if (cudaGetDevice(&device) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess)
    return 0;
  return sms;
}

struct Plan {
  int nt;
  int64_t tiles_a, tiles_b, steps, units, grid;
  int64_t arrivals_bytes, partials_bytes;
};

int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }

/// The tile and the split of a product, by its sizes: the fewest columns (rows
/// of A) that hold all of A, at most 128.
bool plan_of(int64_t m, int64_t n, int64_t k, int sms, Plan *p) {
  p->nt = m <= 8 ? 8 : m <= 16 ? 16 : m <= 32 ? 32 : m <= 64 ? 64 : 128;
  p->tiles_a = (m + p->nt - 1) / p->nt;
  p->tiles_b = (n + kRowsB - 1) / kRowsB;
  p->steps = (k + kStep - 1) / kStep;
  if (sms <= 0 || p->tiles_a > INT32_MAX / p->tiles_b)
    return false;
  p->units = p->tiles_a * p->tiles_b * p->steps;
  p->grid = p->units < sms ? p->units : sms;
  p->arrivals_bytes = up256(p->tiles_a * p->tiles_b * 4);
  p->partials_bytes = 2 * p->grid * p->nt * 128 * 4;
  return true;
}

/// Codes [rows, pitch] as boxes of `box_rows` rows x 128 bytes; what lies past
/// the end reads as zero codes.
bool encode_codes(CUtensorMap *map, const void *base, int64_t rows, int64_t pitch, int box_rows) {
  PFN_cuTensorMapEncodeTiled_v12000 enc = tensor_map_encoder();
  if (!enc)
    return false;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(pitch), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(pitch)};
  const cuuint32_t box[2] = {128, static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t estr[2] = {1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DT, int NT> int launch(const ProductArgs &a, int64_t grid, cudaStream_t s) {
  auto k = k_mx_product<DT, NT>;
  cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<NT>::kSmem);
  if (e != cudaSuccess)
    return e;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Shape<NT>::kSmem;
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = a.after_quantize ? 1 : 0;
  e = cudaLaunchKernelEx(&cfg, k, a);
  if (e == cudaSuccess) {
    count_launch();
    count_wait_launch();
  }
  return e;
}

template <int DT> int launch_nt(const ProductArgs &a, const Plan &p, cudaStream_t s) {
  switch (p.nt) {
  case 8:
    return launch<DT, 8>(a, p.grid, s);
  case 16:
    return launch<DT, 16>(a, p.grid, s);
  case 32:
    return launch<DT, 32>(a, p.grid, s);
  case 64:
    return launch<DT, 64>(a, p.grid, s);
  default:
    return launch<DT, 128>(a, p.grid, s);
  }
}

/// The word in mapped pinned host memory that kernels set to 2 when a wait
/// runs out: one for the process, allocated on first use.
int32_t *fault_word() {
  static int32_t *word = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    // legal while some stream is being captured
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    cudaThreadExchangeStreamCaptureMode(&mode);
    void *p = nullptr;
    if (cudaHostAlloc(&p, 64, cudaHostAllocMapped | cudaHostAllocPortable) == cudaSuccess) {
      word = static_cast<int32_t *>(p);
      *word = 0;
    }
    cudaThreadExchangeStreamCaptureMode(&mode);
  });
  return word;
}

} // namespace

extern "C" {

int sbc_mx_take_fault(void) {
  int32_t *w = fault_word();
  if (!w)
    return -1;
  return __atomic_exchange_n(w, 0, __ATOMIC_RELAXED);
}

int sbc_mx_product_workspace(int64_t m, int64_t n, int64_t k, int64_t *bytes) {
  Plan p;
  if (m <= 0 || n <= 0 || k <= 0 || !plan_of(m, n, k, sm_count(), &p))
    return SBC_EINVAL;
  *bytes = p.arrivals_bytes + p.partials_bytes;
  return 0;
}

int sbc_mx_product(const sbc_mx *a, const sbc_mx *b, void *y, int32_t dtype, void *workspace, int32_t after_quantize,
                   void *stream) {
  Plan p;
  int32_t *fault = fault_word();
  if (!a || !b || !y || !workspace || !fault || a->format != SBC_MXFP4 || b->format != SBC_MXFP4 || a->rows <= 0 ||
      b->rows <= 0 || a->cols <= 0 || a->cols != b->cols || dtype < SBC_F32 || dtype > SBC_BF16 ||
      !plan_of(a->rows, b->rows, a->cols, sm_count(), &p))
    return SBC_EINVAL;
  ProductArgs args{};
  const int64_t pitch = blocks_of(a->cols) * 16;
  if (!encode_codes(&args.map_a, a->codes, a->rows, pitch, p.nt) ||
      !encode_codes(&args.map_b, b->codes, b->rows, pitch, kRowsB))
    return SBC_EUNSUPPORTED;
  args.scales_a = static_cast<const uint8_t *>(a->scales);
  args.scales_b = static_cast<const uint8_t *>(b->scales);
  args.y = y;
  args.arrivals = static_cast<uint32_t *>(workspace);
  args.partials = reinterpret_cast<float *>(static_cast<uint8_t *>(workspace) + p.arrivals_bytes);
  args.fault = fault;
  args.wait_ns = wait_limit_ns();
  args.m = a->rows;
  args.n = b->rows;
  args.units = p.units;
  args.quads = static_cast<uint32_t>(quads_of(a->cols));
  args.steps = static_cast<uint32_t>(p.steps);
  args.tiles_a = static_cast<uint32_t>(p.tiles_a);
  args.k64 = static_cast<uint32_t>((a->cols + 63) / 64);
  args.after_quantize = after_quantize;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (!after_quantize) {
    const cudaError_t e = cudaMemsetAsync(workspace, 0, p.arrivals_bytes, s);
    if (e != cudaSuccess)
      return e;
  }
  switch (dtype) {
  case SBC_F32:
    return launch_nt<SBC_F32>(args, p, s);
  case SBC_F16:
    return launch_nt<SBC_F16>(args, p, s);
  default:
    return launch_nt<SBC_BF16>(args, p, s);
  }
}

int64_t sbc_mx_product_clear_words(int64_t m, int64_t n, int64_t k) {
  Plan p;
  return plan_of(m, n, k, sm_count(), &p) ? p.arrivals_bytes / 4 : 0;
}

} // extern "C"
