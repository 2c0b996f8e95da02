// Block-scaled fp8 complex GEMM for sm_100a:
//
//   C[b] = alpha * sum over blocks g of 128 k of  sA[b][g][m] sB[b][g][n] (A_g x B_g^T)[m][n]  + beta * C[b]
//
// with A, B fp8 planes (each e4m3 or e5m2) and one float32 scale per block (1 or 128 rows x 128 k) of
// either operand: the operands quantize.cu writes.
//
// The scales differ from block to block, so a block's product cannot stay in the tensor-memory
// accumulator while the next one is added to it.  Per 128 k the MMA warp fills one of two tensor-memory
// buffers (Re and Im, BN columns each) and eight epilogue warps move the other one into float32
// sums in registers, acc += (d * sA) * sB in packed pairs.  A 128 x 128 block is 16 MMAs of 64 clocks
// = 1024 clocks of tensor pipe; moving it takes 256 packed instructions per scheduler beside 64
// columns of tensor-memory loads, so the sums hide behind the MMAs.  The float32 sums of a 128 x 128
// complex tile are 128 registers in each of 256 threads, which is what bounds the tile: no wider
// tile fits the register file.
//
// Either operand may be the 128-row side of the tile (the product is symmetric in A and B); the
// plan takes the one that wastes fewer rows, so one row of A against many rows of B is a
// 128 x 16 tile that reads B once.  Problems whose tiles do not fill the device evenly are cut into
// equal runs of 128-k blocks instead of whole tiles: a CTA that holds part of a tile's blocks writes
// its sums to the plan's workspace, and the CTA that completes the tile adds the parts in the order
// of k, whoever that is, so results do not depend on timing.
#include <new>

#include "gemm_kernels.cuh"

namespace ccglib_b200 {
namespace {

constexpr int kEpiWarps = 8;
constexpr int kFirstEpiWarp = 4;  // warps 2 and 3 only complete the first warpgroup
constexpr int kScaledThreads = 32 * (kFirstEpiWarp + kEpiWarps);
// Registers: 384 threads start with 168 each (64512 in all); the first warpgroup hands back all but 40,
// the two epilogue warpgroups take 232: 128 * 40 + 256 * 232 = 64512.
constexpr int kRegsFirst = 40, kRegsEpi = 232;
static_assert(128 * kRegsFirst + 32 * kEpiWarps * kRegsEpi <= kScaledThreads * 168, "register split");
constexpr int kBlockK = 128;
constexpr int kAccBuffers = 2;

struct ScaledParams {
  GemmParams g;  // M, N, tiles, layout of C, alpha, beta, waits; row side = tile rows
  const float *row_scale, *col_scale;  // [batch][k_blocks][row_blocks / col_blocks]
  uint32_t row_blocks, col_blocks;
  uint32_t row_shift, col_shift;  // log2 of the rows one scale covers (0 or 7)
  // equal runs of blocks (null: whole tiles)
  float *parts;        // two per CTA: [2][BN][128] sums
  unsigned *counters;  // blocks added so far, one per tile; zero between runs
};

template <int BN> struct ScaledCfg {
  static constexpr int kAPlane = kBlockM * kBlockK;
  static constexpr int kBPlane = BN * kBlockK;
  static constexpr int kABytes = 2 * kAPlane;
  static constexpr int kStageBytes = 2 * kAPlane + 2 * kBPlane;
  static constexpr int kStagingBytes = kEpiWarps * kStagingTile;
  static constexpr int kBarrierBytes = 256;
  static constexpr int kRaw = (kMaxSmem - 1024 - kBarrierBytes - kStagingBytes) / kStageBytes;
  static constexpr int kStages = kRaw > 6 ? 6 : kRaw;
  static constexpr int kSmemBytes = kStages * kStageBytes + kStagingBytes + kBarrierBytes + 1024;
  static constexpr int kHalf = BN / 2;  // columns of one epilogue warp
  static_assert(kStages >= 2, "need at least two stages");
  // Up to 64 columns one MMA multiplies an A plane by both B planes, which lie one behind the other in
  // the stage: columns [Ar.Br | Ar.Bi] and [Ai.Br | Ai.Bi], added up on the way out of tensor
  // memory.  An MMA of 128 rows costs the same for 64 columns as for 128, so this halves the tensor
  // time of narrow tiles; at 128 columns there is no tensor memory for it.
  static constexpr bool kStacked = BN <= 64;
  static constexpr int kAccCols = kStacked ? 4 * BN : 2 * BN;
  static_assert(kAccCols * kAccBuffers <= kTmemCols, "accumulators exceed tensor memory");
  static_assert(BN % 16 == 0 && BN >= 16 && BN <= 128, "tile width");
};

// A run of consecutive blocks of one tile.
struct Segment {
  uint32_t tile, k0, k1;
};

// Block range of CTA c when `units` blocks are dealt to `ctas` CTAs.
__device__ __forceinline__ uint64_t run_start(uint64_t units, uint32_t ctas, uint32_t c) {
  return units * c / ctas;
}
// The CTA whose run holds block u.
__device__ __forceinline__ uint32_t run_owner(uint64_t units, uint32_t ctas, uint64_t u) {
  return static_cast<uint32_t>(((u + 1) * ctas - 1) / units);
}

// The work list of a CTA, walked by every role in the same order.
struct Walk {
  uint64_t at, end;  // equal runs: blocks
  uint32_t tile;     // whole tiles
  bool runs;
  __device__ __forceinline__ Walk(const ScaledParams &p) {
    runs = p.parts != nullptr;
    if (runs) {
      const uint64_t units = static_cast<uint64_t>(p.g.num_tiles) * p.g.k_blocks;
      at = run_start(units, gridDim.x, blockIdx.x);
      end = run_start(units, gridDim.x, blockIdx.x + 1);
    } else {
      at = end = 0;
    }
    tile = blockIdx.x;
  }
  __device__ __forceinline__ bool next(const ScaledParams &p, Segment &s) {
    if (!runs) {
      if (tile >= p.g.num_tiles) return false;
      s.tile = tile;
      s.k0 = 0;
      s.k1 = p.g.k_blocks;
      tile += gridDim.x;
      return true;
    }
    if (at >= end) return false;
    s.tile = static_cast<uint32_t>(at / p.g.k_blocks);
    const uint64_t base = static_cast<uint64_t>(s.tile) * p.g.k_blocks;
    s.k0 = static_cast<uint32_t>(at - base);
    const uint64_t stop = end - base < p.g.k_blocks ? end - base : p.g.k_blocks;
    s.k1 = static_cast<uint32_t>(stop);
    at = base + stop;
    return true;
  }
};

__device__ __forceinline__ void epi_sync() {
  asm volatile("bar.sync 1, %0;" ::"n"(32 * kEpiWarps) : "memory");
}

// Two neighbouring columns as one register pair.
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pair_of(float lo, float hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ f32x2 pair_of(uint32_t lo, uint32_t hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}
__device__ __forceinline__ void split_pair(f32x2 v, float &lo, float &hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
// acc += (d * s) * t.  In this order nothing overflows or vanishes that the scaled sum itself does not:
// s * t alone may leave float32 where d is zero or large.
__device__ __forceinline__ void scale_add(f32x2 &acc, f32x2 d, f32x2 s, f32x2 t) {
  asm("{\n\t.reg .b64 v;\n\tmul.rn.f32x2 v, %1, %2;\n\tfma.rn.f32x2 %0, v, %3, %0;\n\t}"
      : "+l"(acc)
      : "l"(d), "l"(s), "l"(t));
}

__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 sub2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

template <int N> __device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N> __device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

template <int N> __device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, uint32_t *r);
template <> __device__ __forceinline__ void tmem_ld_cols<8>(uint32_t taddr, uint32_t *r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]),
                 "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}
template <> __device__ __forceinline__ void tmem_ld_cols<16>(uint32_t taddr, uint32_t *r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

// Wait for this warp's tensor-memory loads; the values are operands, so nothing that uses them can be
// scheduled ahead of the wait.
template <int N> __device__ __forceinline__ void tmem_wait_cols(uint32_t *r);
template <> __device__ __forceinline__ void tmem_wait_cols<8>(uint32_t *r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                 "+r"(r[6]), "+r"(r[7])
               :
               : "memory");
}
template <> __device__ __forceinline__ void tmem_wait_cols<16>(uint32_t *r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                 "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                 "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}

// alpha and beta on the sums of row m, columns n0 .. n0 + HALF.
template <typename OutT, int HALF>
__device__ __forceinline__ void scale_sums(const GemmParams &p, uint32_t b, uint32_t m, uint32_t n0,
                                           float (&re)[HALF], float (&im)[HALF]) {
  if (p.have_alpha) {
#pragma unroll
    for (int j = 0; j < HALF; ++j) {
      const float r = re[j];
      re[j] = p.alpha_re * r - p.alpha_im * im[j];
      im[j] = p.alpha_im * r + p.alpha_re * im[j];
    }
  }
  if (p.have_beta && m < p.M) {
    const COffsets o = c_offsets(p, b, m, n0);
    const OutT *C = static_cast<const OutT *>(p.c);
#pragma unroll
    for (int j = 0; j < HALF; ++j) {
      if (n0 + j < p.N) {
        const float cr = OutTraits<OutT>::to_acc(C[o.base_re + j * o.stride_j]);
        const float ci = OutTraits<OutT>::to_acc(C[o.base_re + j * o.stride_j + o.off_im]);
        re[j] += p.beta_re * cr - p.beta_im * ci;
        im[j] += p.beta_im * cr + p.beta_re * ci;
      }
    }
  }
}

// Word j (0..31) of tile t of a row as it stands in C: 128 bytes of the row.  Planar tiles are the
// real part's 128-byte pieces, then the imaginary part's; interleaved ones follow one another.
template <typename OutT, int HALF, int T, int J>
__device__ __forceinline__ uint32_t row_word(bool inter, const float (&re)[HALF],
                                             const float (&im)[HALF]) {
  constexpr int kPer = 4 / sizeof(OutT);
  constexpr int kTiles = HALF * 2 / (32 * kPer);
  constexpr int kPlaneTiles = kTiles / 2;
  float v[2];
  if (inter) {
    constexpr int e = (T * 32 + J) * kPer;  // element of the (re, im) sequence
    v[0] = (e & 1) ? im[e / 2] : re[e / 2];
    v[1] = im[e / 2];  // 16-bit: the pair (re, im); unused otherwise
  } else {
    constexpr int c = ((T % kPlaneTiles) * 32 + J) * kPer;
    v[0] = T < kPlaneTiles ? re[c] : im[c];
    v[1] = T < kPlaneTiles ? re[c + kPer - 1] : im[c + kPer - 1];
  }
  return Packer<OutT>::word(v);
}

template <typename OutT, int HALF, int T, int... J>
__device__ __forceinline__ void row_words(bool inter, const float (&re)[HALF],
                                          const float (&im)[HALF], uint32_t (&w)[32]) {
  if constexpr (sizeof...(J) < 32) {
    row_words<OutT, HALF, T, J..., static_cast<int>(sizeof...(J))>(inter, re, im, w);
  } else {
    ((w[J] = row_word<OutT, HALF, T, J>(inter, re, im)), ...);
  }
}

// One tile of 32 rows x 128 bytes through the warp's staging tile and out by a TMA store.
template <typename OutT, int HALF, int T>
__device__ __forceinline__ void store_tile(const GemmParams &p, const CUtensorMap *tm_c,
                                           uint32_t staging, uint32_t lane, uint32_t b, uint32_t m0,
                                           uint32_t n0, const float (&re)[HALF],
                                           const float (&im)[HALF]) {
  constexpr int kPer = 4 / sizeof(OutT);
  constexpr int kTiles = HALF * 2 / (32 * kPer);
  constexpr int kPlaneTiles = kTiles / 2;
  const bool inter = p.c_layout == kInterRow;
  const uint32_t first = inter ? n0 + T * 16 * kPer : n0 + (T % kPlaneTiles) * 32 * kPer;
  if (first >= p.N || m0 >= p.M) return;  // uniform over the warp
  uint32_t w[32];
  row_words<OutT, HALF, T>(inter, re, im, w);
  if (lane == 0) bulk_wait_group_read<0>();
  __syncwarp();
  const uint32_t row = staging + lane * 128;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    st_shared_v4(row + ((j ^ (lane & 7)) << 4), w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
  }
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) {
    const int32_t x = static_cast<int32_t>(first * sizeof(OutT) * (inter ? 2 : 1));
    const int32_t z = static_cast<int32_t>(inter ? b : 2 * b + (T < kPlaneTiles ? 0 : 1));
    tma_store_3d(tm_c, staging, x, static_cast<int32_t>(m0), z);
    bulk_commit_group();
  }
}

template <typename OutT, int HALF, int... T>
__device__ __forceinline__ void store_tiles(const GemmParams &p, const CUtensorMap *tm_c,
                                            uint32_t staging, uint32_t lane, uint32_t b, uint32_t m0,
                                            uint32_t n0, const float (&re)[HALF],
                                            const float (&im)[HALF]) {
  constexpr int kTiles = HALF * 2 * static_cast<int>(sizeof(OutT)) / 128;
  if constexpr (sizeof...(T) < kTiles) {
    store_tiles<OutT, HALF, T..., static_cast<int>(sizeof...(T))>(p, tm_c, staging, lane, b, m0, n0,
                                                                  re, im);
  } else {
    (store_tile<OutT, HALF, T>(p, tm_c, staging, lane, b, m0, n0, re, im), ...);
  }
}

// Row m, HALF columns from n0, straight from registers.
template <typename OutT, int HALF>
__device__ __forceinline__ void store_direct(const GemmParams &p, uint32_t b, uint32_t m, uint32_t n0,
                                             const float (&re)[HALF], const float (&im)[HALF]) {
  if (m >= p.M || n0 >= p.N) return;
  using Tr = OutTraits<OutT>;
  OutT *C = static_cast<OutT *>(p.c);
  const COffsets o = c_offsets(p, b, m, n0);
  const int valid = static_cast<int>(min(static_cast<uint32_t>(HALF), p.N - n0));
  if (p.vec_ok && valid == HALF && p.c_layout == kPlanarRow) {
    store_run<OutT, HALF>(C + o.base_re, re, valid, true);
    store_run<OutT, HALF>(C + o.base_re + o.off_im, im, valid, true);
    return;
  }
  if (p.c_layout == kInterRow || p.c_layout == kInterCol) {
    // one store per complex value
    struct alignas(2 * sizeof(OutT)) Pair {
      OutT re, im;
    };
    if (p.pair_ok) {
#pragma unroll
      for (int j = 0; j < HALF; ++j) {
        if (j < valid) {
          *reinterpret_cast<Pair *>(C + o.base_re + j * o.stride_j) =
              Pair{Tr::to_out(re[j]), Tr::to_out(im[j])};
        }
      }
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < HALF; ++j) {
    if (j < valid) {
      C[o.base_re + j * o.stride_j] = Tr::to_out(re[j]);
      C[o.base_re + j * o.stride_j + o.off_im] = Tr::to_out(im[j]);
    }
  }
}

template <int BN, typename OutT>
__global__ void __launch_bounds__(kScaledThreads, 1)
scaled_gemm_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                   const __grid_constant__ CUtensorMap tm_c, const ScaledParams p) {
  using C = ScaledCfg<BN>;
  constexpr int kStages = C::kStages;
  constexpr int HALF = C::kHalf;

  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023u) & ~static_cast<uintptr_t>(1023u));
  uint64_t *bars =
      reinterpret_cast<uint64_t *>(smem + kStages * C::kStageBytes + C::kStagingBytes);
  const uint32_t bar_full = smem_u32(bars);
  const uint32_t bar_empty = bar_full + 8 * kStages;
  const uint32_t bar_acc_full = bar_empty + 8 * kStages;
  const uint32_t bar_acc_empty = bar_acc_full + 8 * kAccBuffers;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * kStages + 2 * kAccBuffers);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
  volatile unsigned *last_flag = tmem_slot + 2;
  const uint32_t smem_base = smem_u32(smem);
  const uint32_t warp = threadIdx.x >> 5;
  const uint32_t lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (int s = 0; s < kAccBuffers; ++s) {
      mbar_init(bar_acc_full + 8 * s, 1);
      mbar_init(bar_acc_empty + 8 * s, kEpiWarps);
    }
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tensormap(&tm_a);
    prefetch_tensormap(&tm_b);
    if (p.g.epi_tma) prefetch_tensormap(&tm_c);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp < kFirstEpiWarp) {
  regs_dec<kRegsFirst>();
  Walk walk(p);
  Segment seg;
  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    uint32_t stage = 0, phase = 0, issued = 0;
    bool ok = true;
    while (ok && walk.next(p, seg)) {
      const TileCoord t = decode_tile(p.g, seg.tile);
      for (uint32_t kb = seg.k0; kb < seg.k1; ++kb) {
        if (!mbar_wait(bar_empty + 8 * stage, phase ^ 1, abort_flag, p.g.status,
                       kDevTimeoutProducer, p.g.wait_cycles)) {
          ok = false;
          break;
        }
        if (lane == 0) {
          const uint32_t full = bar_full + 8 * stage;
          const uint32_t dst = smem_base + stage * C::kStageBytes;
          const int32_t x = static_cast<int32_t>(kb * kBlockK), z = static_cast<int32_t>(2 * t.b);
          mbar_arrive_expect_tx(full, C::kStageBytes);
          tma_load_3d(dst, &tm_a, x, static_cast<int32_t>(t.mt * kBlockM), z, full);
          tma_load_3d(dst + C::kABytes, &tm_b, x, static_cast<int32_t>(t.nt * BN), z, full);
        }
        __syncwarp();
        issued |= 1u << stage;
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    if (*abort_flag) {
      // our own copies must land before the CTA leaves
      for (int s = 0; s < kStages; ++s) {
        if (!(issued & (1u << s))) continue;
        const uint32_t parity = (static_cast<uint32_t>(s) < stage) ? phase : (phase ^ 1);
        const long long t0 = clock64();
        while (!mbar_try_wait(bar_full + 8 * s, parity)) {
          if (clock64() - t0 > p.g.wait_cycles) {
            atomicOr(p.g.status, kDevTimeoutDrain);
            break;
          }
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0;
    bool ok = true;
    while (ok && walk.next(p, seg)) {
      for (uint32_t kb = seg.k0; kb < seg.k1; ++kb) {
        if (!mbar_wait(bar_acc_empty + 8 * acc, acc_phase ^ 1, abort_flag, p.g.status,
                       kDevTimeoutMma, p.g.wait_cycles) ||
            !mbar_wait(bar_full + 8 * stage, phase, abort_flag, p.g.status, kDevTimeoutMma,
                       p.g.wait_cycles)) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (lane == 0) {
          const uint32_t a_base = smem_base + stage * C::kStageBytes;
          const uint32_t b_base = a_base + C::kABytes;
          const uint32_t d = tmem_base + acc * C::kAccCols;
#pragma unroll
          for (int k = 0; k < kBlockK / 32; ++k) {
            const uint64_t a_re = smem_desc<128>(a_base + k * 32);
            const uint64_t a_im = smem_desc<128>(a_base + C::kAPlane + k * 32);
            const uint64_t b_re = smem_desc<128>(b_base + k * 32);
            if constexpr (C::kStacked) {
              tc_mma<kKindF8F6F4>(d, a_re, b_re, p.g.idesc, k != 0);
              tc_mma<kKindF8F6F4>(d + 2 * BN, a_im, b_re, p.g.idesc, k != 0);
            } else {
              const uint64_t b_im = smem_desc<128>(b_base + C::kBPlane + k * 32);
              tc_mma<kKindF8F6F4>(d, a_re, b_re, p.g.idesc, k != 0);
              tc_mma<kKindF8F6F4>(d + BN, a_re, b_im, p.g.idesc, k != 0);
              tc_mma<kKindF8F6F4>(d + BN, a_im, b_re, p.g.idesc, 1u);
              tc_mma<kKindF8F6F4>(d, a_im, b_im, p.g.idesc_neg_a, 1u);
            }
          }
          tc_commit(bar_empty + 8 * stage);
          tc_commit(bar_acc_full + 8 * acc);
        }
        __syncwarp();
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1;
        }
        if (++acc == kAccBuffers) {
          acc = 0;
          acc_phase ^= 1;
        }
      }
    }
  }
  } else {
    // ------------------------------------------------------------------ epilogue warps
    regs_inc<kRegsEpi>();
    Walk walk(p);
    Segment seg;
    const uint32_t quad = warp & 3;                     // tensor-memory lanes of this warp
    const uint32_t half = (warp - kFirstEpiWarp) >> 2;  // which half of the columns
    const uint32_t staging =
        smem_base + kStages * C::kStageBytes + (warp - kFirstEpiWarp) * kStagingTile;
    // the column scales of the block (two buffers) at the head of the staging tile
    f32x2 *col_buf = reinterpret_cast<f32x2 *>(
        smem + kStages * C::kStageBytes + (warp - kFirstEpiWarp) * kStagingTile);
    uint32_t acc = 0, acc_phase = 0;
    bool ok = true;
    while (walk.next(p, seg)) {
      f32x2 sum[2][HALF / 2];  // Re, Im
      const TileCoord t = decode_tile(p.g, seg.tile);
      const uint32_t m = t.mt * kBlockM + quad * 32 + lane;
      const uint32_t n0 = t.nt * BN + half * HALF;
      // this lane's row scale, and the scales of two of the warp's columns
      const float *rs = p.row_scale + (static_cast<size_t>(t.b) * p.g.k_blocks + seg.k0) * p.row_blocks;
      const float *cs = p.col_scale + (static_cast<size_t>(t.b) * p.g.k_blocks + seg.k0) * p.col_blocks;
      const uint32_t c0 = n0 + 2 * lane, c1 = c0 + 1;
      const bool row_in = m < p.g.M;
      const bool in0 = 2 * lane < HALF && c0 < p.g.N, in1 = 2 * lane < HALF && c1 < p.g.N;
      const uint32_t ri = m >> p.row_shift, i0 = c0 >> p.col_shift, i1 = c1 >> p.col_shift;
      float s_next = row_in ? __ldg(rs + ri) : 0.0f;
      float t0_next = in0 ? __ldg(cs + i0) : 0.0f;
      float t1_next = in1 ? __ldg(cs + i1) : 0.0f;
#pragma unroll
      for (int j = 0; j < HALF / 2; ++j) sum[0][j] = sum[1][j] = 0;
      // the column scales go through the staging tile: its last store must have read it
      if (lane == 0) bulk_wait_group_read<0>();
      __syncwarp();
      for (uint32_t kb = seg.k0; ok && kb < seg.k1; ++kb) {
        const f32x2 s = pair_of(s_next, s_next);
        f32x2 *cols = col_buf + (kb & 1) * (HALF / 2);
        if (2 * lane < HALF) cols[lane] = pair_of(t0_next, t1_next);
        if (kb + 1 < seg.k1) {
          rs += p.row_blocks;
          cs += p.col_blocks;
          s_next = row_in ? __ldg(rs + ri) : 0.0f;
          t0_next = in0 ? __ldg(cs + i0) : 0.0f;
          t1_next = in1 ? __ldg(cs + i1) : 0.0f;
        }
        __syncwarp();  // the column scales are in place
        ok = mbar_wait(bar_acc_full + 8 * acc, acc_phase, abort_flag, p.g.status,
                       kDevTimeoutEpilogue, p.g.wait_cycles);
        ok = __all_sync(0xFFFFFFFFu, ok);
        if (!ok) break;
        tc_fence_after();
        const uint32_t taddr =
            tmem_base + ((quad * 32) << 16) + acc * C::kAccCols + half * HALF;
        // kCols columns of every accumulator at a time, the next ones on their way while these are added
        constexpr int kCols = HALF < 16 || C::kStacked ? 8 : 16;
        constexpr int kAccs = C::kStacked ? 4 : 2;
        uint32_t d[2][kAccs][kCols];
#pragma unroll
        for (int i = 0; i < kAccs; ++i) tmem_ld_cols<kCols>(taddr + i * BN, d[0][i]);
#pragma unroll
        for (int c = 0; c < HALF; c += kCols) {
          const int now = (c / kCols) & 1;
#pragma unroll
          for (int i = 0; i < kAccs; ++i) tmem_wait_cols<kCols>(d[now][i]);
          if (c + kCols < HALF) {
#pragma unroll
            for (int i = 0; i < kAccs; ++i) {
              tmem_ld_cols<kCols>(taddr + i * BN + c + kCols, d[now ^ 1][i]);
            }
          } else {
            // the buffer is read: the MMAs of the block after next may fill it
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_acc_empty + 8 * acc);
          }
#pragma unroll
          for (int j = 0; j < kCols; j += 4) {
            const ulonglong2 t = *reinterpret_cast<const ulonglong2 *>(cols + (c + j) / 2);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int e = j + 2 * h;
              f32x2 v_re = pair_of(d[now][0][e], d[now][0][e + 1]);
              f32x2 v_im = pair_of(d[now][1][e], d[now][1][e + 1]);
              if constexpr (C::kStacked) {
                v_re = sub2(v_re, pair_of(d[now][3][e], d[now][3][e + 1]));
                v_im = add2(v_im, pair_of(d[now][2][e], d[now][2][e + 1]));
              }
              scale_add(sum[0][(c + e) / 2], v_re, s, h == 0 ? t.x : t.y);
              scale_add(sum[1][(c + e) / 2], v_im, s, h == 0 ? t.x : t.y);
            }
          }
        }
        if (++acc == kAccBuffers) {
          acc = 0;
          acc_phase ^= 1;
        }
      }
      float re[HALF], im[HALF];
#pragma unroll
      for (int j = 0; j < HALF / 2; ++j) {
        split_pair(sum[0][j], re[2 * j], re[2 * j + 1]);
        split_pair(sum[1][j], im[2 * j], im[2 * j + 1]);
      }
      bool finish = ok;
      if (seg.k1 - seg.k0 < p.g.k_blocks) {
        // Part of a tile: add it through the workspace.  A CTA's run holds at most one part that
        // begins inside a tile (slot 0) and one that begins a tile without ending it (slot 1).
        // The counter is kept up even after a wait gave up, so that it is zero for the next run.
        constexpr size_t kPart = 2 * BN * kBlockM;
        const uint64_t units = static_cast<uint64_t>(p.g.num_tiles) * p.g.k_blocks;
        const uint64_t base = static_cast<uint64_t>(seg.tile) * p.g.k_blocks;
        const uint32_t at = half * HALF * kBlockM + quad * 32 + lane;
        float *mine = p.parts + (2 * static_cast<size_t>(blockIdx.x) + (seg.k0 == 0 ? 1 : 0)) * kPart + at;
#pragma unroll
        for (int j = 0; j < HALF; ++j) {
          __stcg(mine + j * kBlockM, re[j]);
          __stcg(mine + (BN + j) * kBlockM, im[j]);
        }
        __threadfence();
        epi_sync();
        if (threadIdx.x == 32 * kFirstEpiWarp) {
          const unsigned add = seg.k1 - seg.k0;
          const unsigned before = atomicAdd(p.counters + seg.tile, add);
          const bool last = before + add == p.g.k_blocks;
          if (last) p.counters[seg.tile] = 0;
          __threadfence();
          *last_flag = last ? 1u : 0u;
        }
        epi_sync();
        finish = *last_flag != 0 && ok;
        epi_sync();  // the flag may be written again
        if (finish) {
#pragma unroll
          for (int j = 0; j < HALF; ++j) re[j] = im[j] = 0.0f;
          const uint32_t from = run_owner(units, gridDim.x, base);
          const uint32_t to = run_owner(units, gridDim.x, base + p.g.k_blocks - 1);
          for (uint32_t c = from; c <= to; ++c) {
            const uint32_t slot = run_start(units, gridDim.x, c) > base ? 0 : 1;
            const float *part = p.parts + (2 * static_cast<size_t>(c) + slot) * kPart + at;
#pragma unroll
            for (int j = 0; j < HALF; ++j) {
              re[j] += __ldcg(part + j * kBlockM);
              im[j] += __ldcg(part + (BN + j) * kBlockM);
            }
          }
        }
      }
      if (finish) {
        scale_sums<OutT, HALF>(p.g, t.b, m, n0, re, im);
        bool stored = false;
        if constexpr (HALF * 2 * sizeof(OutT) >= 256) {
          if (p.g.epi_tma) {
            store_tiles<OutT, HALF>(p.g, &tm_c, staging, lane, t.b, t.mt * kBlockM + quad * 32, n0,
                                    re, im);
            stored = true;
          }
        }
        if (!stored) store_direct<OutT, HALF>(p.g, t.b, m, n0, re, im);
      }
    }
    if (p.g.epi_tma && lane == 0) bulk_wait_group<0>();
    __syncwarp();
  }

  // ------------------------------------------------------------------ tear-down
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

using ScaledFn = void (*)(const CUtensorMap, const CUtensorMap, const CUtensorMap,
                          const ScaledParams);

struct ScaledEntry {
  ScaledFn fn;
  int smem;
};

template <typename OutT> ScaledEntry pick_width(int bn) {
  switch (bn) {
  case 128:
    return {scaled_gemm_kernel<128, OutT>, ScaledCfg<128>::kSmemBytes};
  case 64:
    return {scaled_gemm_kernel<64, OutT>, ScaledCfg<64>::kSmemBytes};
  case 32:
    return {scaled_gemm_kernel<32, OutT>, ScaledCfg<32>::kSmemBytes};
  default:
    return {scaled_gemm_kernel<16, OutT>, ScaledCfg<16>::kSmemBytes};
  }
}

bool is_fp8(int t) { return t == CCGLIB_B200_FLOAT8E4M3 || t == CCGLIB_B200_FLOAT8E5M2; }

} // namespace
} // namespace ccglib_b200

using namespace ccglib_b200;

struct ccglib_b200_scaled_gemm_plan {
  ccglib_b200_scaled_gemm_desc desc;
  ScaledEntry kernel;
  int bn;
  bool swapped;  // B is the 128-row side of the tile
  size_t rows, cols, k_blocks, tiles;
  size_t runs;   // > 0: CTAs that share the blocks in equal runs
  size_t out_bytes;
  int device, sms;
  long long wait_cycles;
  unsigned *status;
  float *parts;
  unsigned *counters;
  size_t scratch_bytes;
};

extern "C" int ccglib_b200_scaled_gemm_plan_create(const ccglib_b200_scaled_gemm_desc *desc,
                                                   ccglib_b200_scaled_gemm_plan **out) {
  if (desc == nullptr || out == nullptr) {
    set_last_error("scaled_gemm_plan_create: null argument");
    return CCGLIB_B200_INVALID_ARGUMENT;
  }
  *out = nullptr;
  const ccglib_b200_scaled_gemm_desc &d = *desc;
  if (d.batch == 0 || d.m == 0 || d.n == 0 || d.k == 0) {
    set_last_error("scaled_gemm_plan_create: batch, M, N and K must be positive");
    return CCGLIB_B200_INVALID_ARGUMENT;
  }
  // byte coordinates along K and along a row of C are 32-bit signed in the TMA unit
  if (d.m > 0x0FFFFFFFull || d.n > 0x0FFFFFFFull || d.k > 0x7FFFFF00ull || d.batch > 0x3FFFFFFFull) {
    set_last_error("scaled_gemm_plan_create: dimension too large");
    return CCGLIB_B200_INVALID_ARGUMENT;
  }
  if (!is_fp8(d.type_a) || !is_fp8(d.type_b)) {
    set_last_error("scaled_gemm_plan_create: A and B must be float8e4m3 or float8e5m2 (got %d, %d)",
                   d.type_a, d.type_b);
    return CCGLIB_B200_UNSUPPORTED;
  }
  if (d.type_out != CCGLIB_B200_FLOAT32 && d.type_out != CCGLIB_B200_FLOAT16 &&
      d.type_out != CCGLIB_B200_BFLOAT16) {
    set_last_error("scaled_gemm_plan_create: output must be float32, float16 or bfloat16 (got %d)",
                   d.type_out);
    return CCGLIB_B200_UNSUPPORTED;
  }
  if ((d.a_block_rows != 1 && d.a_block_rows != 128) ||
      (d.b_block_rows != 1 && d.b_block_rows != 128)) {
    set_last_error("scaled_gemm_plan_create: a block has 1 or 128 rows (got %zu, %zu)",
                   d.a_block_rows, d.b_block_rows);
    return CCGLIB_B200_INVALID_ARGUMENT;
  }
  if ((d.c_complex_axis != CCGLIB_B200_PLANAR && d.c_complex_axis != CCGLIB_B200_INTERLEAVED) ||
      (d.c_mem_order != CCGLIB_B200_ROW_MAJOR && d.c_mem_order != CCGLIB_B200_COL_MAJOR)) {
    set_last_error("scaled_gemm_plan_create: unknown complex axis location %d or memory order %d",
                   d.c_complex_axis, d.c_mem_order);
    return CCGLIB_B200_INVALID_ARGUMENT;
  }
  ccglib_b200_scaled_gemm_plan plan{};
  plan.desc = d;
  CCGLIB_CUDA_TRY(cudaGetDevice(&plan.device));
  plan.sms = sm_count();
  if (plan.sms <= 0) return CCGLIB_B200_CUDA_ERROR;
  int cc_major = 0;
  CCGLIB_CUDA_TRY(cudaDeviceGetAttribute(&cc_major, cudaDevAttrComputeCapabilityMajor, plan.device));
  if (cc_major != 10) {
    set_last_error("This architecture is not supported (need compute capability 10.x)");
    return CCGLIB_B200_UNSUPPORTED;
  }
  plan.wait_cycles = wait_limit_cycles();
  plan.k_blocks = ceil_div<size_t>(d.k, kBlockK);

  // ---- which operand is the 128-row side, and how many columns a tile has: an operand of at most
  // 64 rows is the column side, in the narrowest tile that holds it
  plan.swapped = d.m <= 64 && d.m < d.n;
  plan.rows = plan.swapped ? d.n : d.m;
  plan.cols = plan.swapped ? d.m : d.n;
  plan.bn = plan.cols <= 16 ? 16 : plan.cols <= 32 ? 32 : plan.cols <= 64 ? 64 : 128;
  plan.tiles = d.batch * ceil_div<size_t>(plan.rows, kBlockM) * ceil_div<size_t>(plan.cols, plan.bn);
  if (plan.tiles > 0x7FFFFFFFull) {
    set_last_error("scaled_gemm_plan_create: too many tiles");
    return CCGLIB_B200_INVALID_ARGUMENT;
  }
  const size_t sms = static_cast<size_t>(plan.sms);
  const size_t waves = ceil_div(plan.tiles, sms);
  const size_t units = plan.tiles * plan.k_blocks;
  if (waves <= 4 && plan.k_blocks > 1 && plan.tiles * 10 < waves * sms * 9) {
    const size_t ctas = units / 4 < sms ? units / 4 : sms;
    if (ctas > plan.tiles) plan.runs = ctas;
  }
  switch (d.type_out) {
  case CCGLIB_B200_FLOAT32:
    plan.kernel = pick_width<float>(plan.bn);
    plan.out_bytes = 4;
    break;
  case CCGLIB_B200_FLOAT16:
    plan.kernel = pick_width<__half>(plan.bn);
    plan.out_bytes = 2;
    break;
  default:
    plan.kernel = pick_width<__nv_bfloat16>(plan.bn);
    plan.out_bytes = 2;
    break;
  }
  CCGLIB_CUDA_TRY(cudaFuncSetAttribute(reinterpret_cast<const void *>(plan.kernel.fn),
                                       cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       plan.kernel.smem));
  int rc = device_status_address(&plan.status);
  if (rc != CCGLIB_B200_OK) return rc;
  if (plan.runs > 0) {
    const size_t parts = 2 * plan.runs * 2 * plan.bn * kBlockM * sizeof(float);
    plan.scratch_bytes = parts + plan.tiles * sizeof(unsigned);
    if (cudaMalloc(&plan.parts, plan.scratch_bytes) != cudaSuccess) {
      cudaGetLastError();
      set_last_error("scaled_gemm_plan_create: could not allocate %zu bytes of workspace",
                     plan.scratch_bytes);
      return CCGLIB_B200_OUT_OF_MEMORY;
    }
    plan.counters = reinterpret_cast<unsigned *>(reinterpret_cast<char *>(plan.parts) + parts);
    // complete before the plan is used on any stream
    cudaError_t err = cudaMemset(plan.counters, 0, plan.tiles * sizeof(unsigned));
    if (err == cudaSuccess) err = cudaStreamSynchronize(nullptr);
    if (err != cudaSuccess) {
      cudaFree(plan.parts);
      return cuda_fail(err, "clearing the workspace");
    }
  }
  *out = new (std::nothrow) ccglib_b200_scaled_gemm_plan(plan);
  if (*out == nullptr) {
    if (plan.parts != nullptr) cudaFree(plan.parts);
    set_last_error("scaled_gemm_plan_create: out of host memory");
    return CCGLIB_B200_OUT_OF_MEMORY;
  }
  return CCGLIB_B200_OK;
}

extern "C" int ccglib_b200_scaled_gemm_run(ccglib_b200_scaled_gemm_plan *plan, const void *d_a,
                                           const float *d_a_scale, const void *d_b,
                                           const float *d_b_scale, void *d_c, void *stream_v) {
  if (plan == nullptr || d_a == nullptr || d_a_scale == nullptr || d_b == nullptr ||
      d_b_scale == nullptr || d_c == nullptr) {
    set_last_error("scaled_gemm_run: null argument");
    return CCGLIB_B200_INVALID_ARGUMENT;
  }
  if (!aligned16(d_a) || !aligned16(d_b)) {
    set_last_error("scaled_gemm_run: A and B must be 16-byte aligned");
    return CCGLIB_B200_INVALID_ARGUMENT;
  }
  const ccglib_b200_scaled_gemm_desc &d = plan->desc;
  if (((reinterpret_cast<uintptr_t>(d_a_scale) | reinterpret_cast<uintptr_t>(d_b_scale)) & 3u) != 0 ||
      reinterpret_cast<uintptr_t>(d_c) % plan->out_bytes != 0) {
    set_last_error("scaled_gemm_run: scales and C must be aligned to their elements");
    return CCGLIB_B200_INVALID_ARGUMENT;
  }
  int device = -1;
  CCGLIB_CUDA_TRY(cudaGetDevice(&device));
  if (device != plan->device) {
    set_last_error("scaled_gemm_run: the plan belongs to device %d, the current device is %d",
                   plan->device, device);
    return CCGLIB_B200_INVALID_ARGUMENT;
  }
  ScaledParams p{};
  GemmParams &g = p.g;
  g.M = static_cast<uint32_t>(plan->rows);
  g.N = static_cast<uint32_t>(plan->cols);
  g.k_blocks = static_cast<uint32_t>(plan->k_blocks);
  g.tiles_m = static_cast<uint32_t>(ceil_div<size_t>(plan->rows, kBlockM));
  g.tiles_n = static_cast<uint32_t>(ceil_div<size_t>(plan->cols, plan->bn));
  g.group_n = g.tiles_m <= 2 ? 4 : 8;
  g.num_tiles = static_cast<uint32_t>(plan->tiles);
  const int row_type = plan->swapped ? d.type_b : d.type_a;
  const int col_type = plan->swapped ? d.type_a : d.type_b;
  const int mma_n = plan->bn <= 64 ? 2 * plan->bn : plan->bn;
  // instruction descriptor: fp32 accumulator, operand formats (0 e4m3, 1 e5m2), N >> 3, M >> 4
  g.idesc = (1u << 4) | ((row_type == CCGLIB_B200_FLOAT8E5M2 ? 1u : 0u) << 7) |
            ((col_type == CCGLIB_B200_FLOAT8E5M2 ? 1u : 0u) << 10) |
            (static_cast<uint32_t>(mma_n >> 3) << 17) | (static_cast<uint32_t>(kBlockM >> 4) << 24);
  g.idesc_neg_a = g.idesc | (1u << 13);
  g.c = d_c;
  // C^T of the swapped product in one order is C in the other
  const bool row = (d.c_mem_order == CCGLIB_B200_ROW_MAJOR) != plan->swapped;
  const bool planar = d.c_complex_axis == CCGLIB_B200_PLANAR;
  g.c_layout = planar ? (row ? kPlanarRow : kPlanarCol) : (row ? kInterRow : kInterCol);
  g.alpha_re = d.alpha_re;
  g.alpha_im = d.alpha_im;
  g.beta_re = d.beta_re;
  g.beta_im = d.beta_im;
  g.have_alpha = (d.alpha_re != 1.0f || d.alpha_im != 0.0f) ? 1u : 0u;
  g.have_beta = (d.beta_re != 0.0f || d.beta_im != 0.0f) ? 1u : 0u;
  const size_t run_bytes = (planar ? plan->cols : 2 * plan->cols) * plan->out_bytes;
  g.vec_ok = (row && aligned16(d_c) && run_bytes % 16 == 0) ? 1u : 0u;
  g.pair_ok = reinterpret_cast<uintptr_t>(d_c) % (2 * plan->out_bytes) == 0 ? 1u : 0u;
  g.epi_tma = g.vec_ok && plan->bn / 2 * 2 * plan->out_bytes >= 256 ? 1u : 0u;
  g.status = plan->status;
  g.wait_cycles = plan->wait_cycles;
  p.row_scale = plan->swapped ? d_b_scale : d_a_scale;
  p.col_scale = plan->swapped ? d_a_scale : d_b_scale;
  const size_t row_block = plan->swapped ? d.b_block_rows : d.a_block_rows;
  const size_t col_block = plan->swapped ? d.a_block_rows : d.b_block_rows;
  p.row_blocks = static_cast<uint32_t>(ceil_div(plan->rows, row_block));
  p.col_blocks = static_cast<uint32_t>(ceil_div(plan->cols, col_block));
  p.row_shift = row_block == 128 ? 7 : 0;
  p.col_shift = col_block == 128 ? 7 : 0;
  p.parts = plan->parts;
  p.counters = plan->counters;

  const size_t pitch = ceil_div<size_t>(d.k, 16) * 16;
  CUtensorMap tm_a, tm_b, tm_c;
  int rc = make_map(&tm_a, plan->swapped ? d_b : d_a, d.k, plan->rows, 2 * d.batch, pitch,
                    pitch * plan->rows, 128, kBlockM, 2);
  if (rc != CCGLIB_B200_OK) return rc;
  rc = make_map(&tm_b, plan->swapped ? d_a : d_b, d.k, plan->cols, 2 * d.batch, pitch,
                pitch * plan->cols, 128, plan->bn, 2);
  if (rc != CCGLIB_B200_OK) return rc;
  tm_c = tm_a;  // placeholder when the epilogue stores from registers
  if (g.epi_tma) {
    rc = make_map(&tm_c, d_c, run_bytes, plan->rows, planar ? 2 * d.batch : d.batch, run_bytes,
                  plan->rows * run_bytes, 128, 32, 1);
    if (rc != CCGLIB_B200_OK) return rc;
  }
  const size_t ctas = plan->runs > 0 ? plan->runs
                      : plan->tiles < static_cast<size_t>(plan->sms) ? plan->tiles
                                                                     : plan->sms;
  plan->kernel.fn<<<static_cast<unsigned>(ctas), kScaledThreads, plan->kernel.smem,
                    static_cast<cudaStream_t>(stream_v)>>>(tm_a, tm_b, tm_c, p);
  CCGLIB_CUDA_TRY(cudaGetLastError());
  return CCGLIB_B200_OK;
}

extern "C" size_t ccglib_b200_scaled_gemm_plan_scratch_bytes(
    const ccglib_b200_scaled_gemm_plan *plan) {
  return plan != nullptr ? plan->scratch_bytes : 0;
}

extern "C" int ccglib_b200_scaled_gemm_plan_tile(const ccglib_b200_scaled_gemm_plan *plan,
                                                 int tile[3]) {
  if (plan == nullptr || tile == nullptr) {
    set_last_error("scaled_gemm_plan_tile: null argument");
    return CCGLIB_B200_INVALID_ARGUMENT;
  }
  tile[0] = plan->bn;
  tile[1] = plan->swapped ? 1 : 0;
  tile[2] = static_cast<int>(plan->runs);
  return CCGLIB_B200_OK;
}

extern "C" int ccglib_b200_scaled_gemm_plan_destroy(ccglib_b200_scaled_gemm_plan *plan) {
  if (plan == nullptr) return CCGLIB_B200_OK;
  if (plan->parts != nullptr) cudaFree(plan->parts);
  delete plan;
  return CCGLIB_B200_OK;
}
