// Block-scaled fp8 complex GEMM for sm_100a:
//
//   C[b] = alpha * sum over blocks g of 128 k of  sA[b][g][m] sB[b][g][n] (A_g x B_g^T)[m][n]  + beta * C[b]
//
// with A, B fp8 planes (each e4m3 or e5m2) and one float32 scale per block (1 or 128 rows x 128 k) of
// either operand: the operands quantize.cu writes.
//
// The scales differ from block to block, so a block's product cannot stay in the tensor-memory
// accumulator while the next one is added to it.  Per 128 k the MMA warps fill one of two tensor-memory
// buffers (Re and Im, BN columns each) while eight epilogue warps add the other one to float32 sums in
// registers, sum += d * (sA sB).  The sums of a 128 x 128 complex tile are 128 registers in each of 256
// threads, which is what bounds the tile: no wider tile fits the register file.
//
// What bounds it at 4096 x 4096 x 16384, measured in clocks per 128 x 128 x 128 block: the 16 MMAs take
// 1570 (a 128-column MMA reads 8 KiB of operands from shared memory beside the 64 KiB that TMA brings in
// per block; their arithmetic alone is 1024), adding a block to the sums takes 600 of an epilogue
// warp's time and hides behind them.  With normally distributed operands the 1 kW power cap takes the
// clock to 1.25 .. 1.45 GHz: 1.95 to 2.02 PFLOP/s, against 2.31 of the unscaled kernel with the same
// tile and 2.69 with 256 columns.  Tried and dropped: sixteen epilogue warps (2640 clocks), packed
// two-value arithmetic (more register moves than it saves), Re and Im handed over apart (2500).
//
// Either operand may be the 128-row side of the tile (the product is symmetric in A and B): A, unless
// it has at most 64 rows and fewer than B.  So one row of A against many rows of B is a
// 128 x 16 tile that reads B once: memory-bound, 1 x 8192 x 8192 in 31 us (134 MB, 4.3 TB/s; a set-up of
// 3 us and the last exchange of 2 us are in it).  Problems whose tiles do not fill the device evenly may
// be cut into equal runs of 128-k blocks instead of whole tiles: a CTA that holds part of a tile's blocks
// writes its sums to the plan's workspace, and the CTA that completes the tile adds the parts in the
// order of k, whoever that is, so results do not depend on timing.
#include <cmath>
#include <cstdlib>
#include <new>

#include "gemm_kernels.cuh"

namespace ccglib_b200 {
namespace {

constexpr int kBlockK = 128;
constexpr int kAccBuffers = 2;
constexpr int kStoreBytes = 64;                // bytes of a row in one TMA store
constexpr int kStoreTile = 32 * kStoreBytes;  // 32 rows of them
constexpr int kStoreTiles = 2;                 // staging of an epilogue warp: two stores in flight

struct ScaledParams {
  GemmParams g;  // M, N, tiles, layout of C, alpha, beta, waits; row side = tile rows
  const float *row_scale, *col_scale;  // [batch][k_blocks][row_blocks / col_blocks]
  uint32_t row_blocks, col_blocks;
  uint32_t row_shift, col_shift;  // log2 of the rows one scale covers (0 or 7)
  uint32_t lift_limit;  // largest scale in a tile that keeps its sums times 2^64, as float32 bits
  // equal runs of blocks (null: whole tiles)
  float *parts;        // two per CTA: [2][BN][128] sums
  unsigned *counters;  // blocks added so far, one per tile; zero between runs
};

template <int BN> struct ScaledCfg {
  static constexpr int kAPlane = kBlockM * kBlockK;
  static constexpr int kBPlane = BN * kBlockK;
  static constexpr int kABytes = 2 * kAPlane;
  static constexpr int kStageBytes = 2 * kAPlane + 2 * kBPlane;
  // Epilogue warps: four (one per quarter of the lanes) for each half of the columns.
  static constexpr int kCols = BN / 2;
  static constexpr int kEpiWarps = 4 * BN / kCols;
  // 128 sums per thread need a register split: 384 threads start with 168 each (64512 in all); the
  // first warpgroup (one warp of it idle) hands back all but 40, the others take 232: 128 * 40 +
  // 256 * 232 = 64512.
  static constexpr bool kSplitRegs = BN == 128;
  static constexpr int kFirstEpiWarp = kSplitRegs ? 4 : 3;  // 0 loads, 1 and 2 multiply
  static constexpr int kThreads = 32 * (kFirstEpiWarp + kEpiWarps);
  static constexpr int kStagingBytes = kEpiWarps * kStoreTiles * kStoreTile;
  static constexpr int kBarrierBytes = 256;
  static constexpr int kRaw = (kMaxSmem - 1024 - kBarrierBytes - kStagingBytes) / kStageBytes;
  static constexpr int kStages = kRaw > 6 ? 6 : kRaw;
  static constexpr int kSmemBytes = kStages * kStageBytes + kStagingBytes + kBarrierBytes + 1024;
  static_assert(kStages >= 2, "need at least two stages");
  // Up to 64 columns one MMA multiplies an A plane by both B planes, which lie one behind the other in
  // the stage: columns [Ar.Br | Ar.Bi] and [Ai.Br | Ai.Bi], added up on the way out of tensor
  // memory.  An MMA of 128 rows costs the same for 64 columns as for 128, so this halves the tensor
  // time of narrow tiles.  At 128 columns the four products of two buffers would be twice the tensor
  // memory there is.
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
  // Blocks of the whole list.
  __device__ __forceinline__ uint64_t blocks(const ScaledParams &p) const {
    if (runs) return end - at;
    if (tile >= p.g.num_tiles) return 0;
    return static_cast<uint64_t>((p.g.num_tiles - 1 - tile) / gridDim.x + 1) * p.g.k_blocks;
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

// Barrier of the epilogue warps.
template <int THREADS> __device__ __forceinline__ void epi_sync() {
  asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory");
}

// Volatile, so that it stays behind the wait for the tensor-memory load that `a` comes from.  (The packed
// two-value form of it was slower here: moving values in and out of aligned register pairs took more
// instructions than it saved.)
__device__ __forceinline__ void fma_to(float &acc, float a, float b) {
  asm volatile("fma.rn.f32 %0, %1, %2, %0;" : "+f"(acc) : "f"(a), "f"(b));
}

__device__ __forceinline__ void mul_pair(float &a, float &b, float f) {
  asm("{\n"
      ".reg .b64 x, y;\n"
      "mov.b64 x, {%0, %1};\n"
      "mov.b64 y, {%2, %2};\n"
      "mul.rn.f32x2 x, x, y;\n"
      "mov.b64 {%0, %1}, x;\n"
      "}"
      : "+f"(a), "+f"(b)
      : "f"(f));
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

__device__ __forceinline__ void tmem_st_8(uint32_t taddr, const uint32_t *r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr),
               "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

// How a block's sums d are scaled by s (of the row) and t (of the column).  d is a multiple of 2^-32 below
// 2^41, so d s t can be an ordinary float32 where s t is not; and where d is zero the result is zero.
//   s and t in [2^-63, 2^63] or zero: s t is normal or zero, and d * (s t) is what add_block adds.
//   Smaller ones are common (the quantiser gives a silent block 2^-126).  A tile whose first block has
//   such scales keeps its sums times a power of two, 2^64 or, in rows that begin below 2^-63, 2^117, for
//   t from 2^-126 and s 2^p from 2^-9: s 2^p t, at least 2^-135, is below the normal range only where
//   s t < 2^-190 and d s t vanishes, and is not zero, so that an infinite sum stays infinite.  s 2^p
//   up to 2^(l + 64) and t up to 2^l keep the sum of all blocks below 2^127 (2^l is lift_limit).
//   A block with any other scale: scale_block writes d s t over d first.  Where every block needs it that
//   takes 1.1 (one row) to 1.75 times the time, in float64 (a scale above 2^63 or subnormal) 1.4 to 4.2
//   times: 4096 x 4096 x 16384 0.91, 1.59 and 3.87 ms.
// A power of two taken out of d in add_block instead, one multiplication per value, took 3 to 12 % more time
// where one row in 64 is silent; this takes 0 to 4 % more than d * (s t) alone, which was wrong there.
__host__ __device__ constexpr uint32_t exponent_bits(int e) { return static_cast<uint32_t>(127 + e) << 23; }

// |x| is zero or between the float32 with the bits low and that with the bits high.
__device__ __forceinline__ bool zero_or_between(float x, uint32_t low, uint32_t high) {
  const uint32_t u = __float_as_uint(x) & 0x7FFFFFFFu;
  return u == 0 || u - low <= high - low;
}

// s (times the power of two that the row's sums are kept times) and t are in the ranges above.
__device__ __forceinline__ bool in_range(float s, float t0, float t1, bool lifted, uint32_t limit) {
  const uint32_t t_low = lifted ? exponent_bits(-126) : exponent_bits(-63);
  const uint32_t t_high = lifted ? limit : exponent_bits(63);
  return zero_or_between(s, lifted ? exponent_bits(-9) : exponent_bits(-63),
                         lifted ? limit + (64u << 23) : exponent_bits(63)) &&
         zero_or_between(t0, t_low, t_high) && zero_or_between(t1, t_low, t_high);
}

// The accumulators of one block at `taddr` -> d s t in their place, to be added as it is.  SMALL: the
// scales are up to 2^63 and none is subnormal; a power of two moves from d to s then, such that s 2^p t is
// below 2^127 and, as above, not zero.  Else in float64, whose range holds every s t.
template <int BN, bool SMALL>
__device__ __forceinline__ void scale_columns(uint32_t taddr, const float *cols, float s) {
  using C = ScaledCfg<BN>;
  constexpr int kAccs = C::kStacked ? 4 : 2;
  constexpr int kStep = C::kStacked || C::kCols < 16 ? 8 : 16;
  const bool one = fabsf(s) >= 1.0f, middle = fabsf(s) >= 0x1p-63f;
  const float down = one ? 1.0f : middle ? 0x1p-64f : 0x1p-117f;
  const float s_up = s * (one ? 1.0f : middle ? 0x1p64f : 0x1p117f);
#pragma unroll 1
  for (int c = 0; c < C::kCols; c += kStep) {
    uint32_t v[kAccs][kStep];
#pragma unroll
    for (int i = 0; i < kAccs; ++i) tmem_ld_cols<kStep>(taddr + i * BN + c, v[i]);
    tmem_wait_ld();
#pragma unroll
    for (int j = 0; j < kStep; ++j) {
      const float t = cols[c + j];
#pragma unroll
      for (int plane = 0; plane < 2; ++plane) {
        float x = __uint_as_float(v[plane][j]);
        if constexpr (C::kStacked) {
          fma_to(x, __uint_as_float(v[kAccs - 1 - plane][j]), plane == 0 ? -1.0f : 1.0f);
        } else {
          asm volatile("" : "+f"(x));  // volatile like fma_to: not ahead of the wait
        }
        if constexpr (SMALL) {
          x = (x * down) * (s_up * t);
        } else {
          x = static_cast<float>(static_cast<double>(x) * (static_cast<double>(s) * t));
        }
        v[plane][j] = __float_as_uint(x);
      }
      if constexpr (C::kStacked) v[2][j] = v[3][j] = 0;
    }
#pragma unroll
    for (int i = 0; i < kAccs; ++i) {
#pragma unroll
      for (int j = 0; j < kStep; j += 8) tmem_st_8(taddr + i * BN + c + j, v[i] + j);
    }
  }
  tmem_wait_st();
}
// (a call, so that add_block's registers are allotted without it)
template <int BN>
__device__ __noinline__ void scale_block(uint32_t taddr, const float *cols, float s, bool small) {
  if (small) {
    scale_columns<BN, true>(taddr, cols, s);
  } else {
    scale_columns<BN, false>(taddr, cols, s);
  }
}

// The accumulators of one block at `taddr` (this warp's lanes and columns) -> sum += scaled block;
// arrives on `done` when tensor memory is read.  ONE: one scale, `col_scale`, covers the columns; else
// they are at `cols`.
template <int BN, bool ONE>
__device__ __forceinline__ void add_block(uint32_t taddr, uint32_t done, uint32_t lane,
                                          const float *cols, float row_scale, float col_scale,
                                          float (&sum)[2][ScaledCfg<BN>::kCols]) {
  using C = ScaledCfg<BN>;
  const float s = ONE ? row_scale * col_scale : row_scale;
  // Steps of kStep columns of both planes; the next step's loads are on their way while this one's
  // values are added.  Stacked accumulators are [Ar.Br | Ar.Bi | Ai.Br | Ai.Bi].
  constexpr int kAccs = C::kStacked ? 4 : 2;
  constexpr int kStep = C::kStacked || C::kCols < 16 ? 8 : 16;
  uint32_t d[2][kAccs][kStep];
#pragma unroll
  for (int i = 0; i < kAccs; ++i) tmem_ld_cols<kStep>(taddr + i * BN, d[0][i]);
#pragma unroll
  for (int c = 0; c < C::kCols; c += kStep) {
    uint32_t(&v)[kAccs][kStep] = d[(c / kStep) & 1];
    tmem_wait_ld();
    if (c + kStep < C::kCols) {
#pragma unroll
      for (int i = 0; i < kAccs; ++i) {
        tmem_ld_cols<kStep>(taddr + i * BN + c + kStep, d[((c / kStep) & 1) ^ 1][i]);
      }
    } else {
      // the buffer is read: the MMAs of the block after next may fill it
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(done);
    }
#pragma unroll
    for (int j = 0; j < kStep; j += 4) {
      float f[4] = {s, s, s, s};
      if constexpr (!ONE) {
        const float4 t = *reinterpret_cast<const float4 *>(cols + c + j);
        f[0] = t.x; f[1] = t.y; f[2] = t.z; f[3] = t.w;
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] *= s;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
#pragma unroll
        for (int plane = 0; plane < 2; ++plane) {
          float x = __uint_as_float(v[plane][j + e]);
          // Re = Ar.Br - Ai.Bi, Im = Ar.Bi + Ai.Br
          if constexpr (C::kStacked) {
            fma_to(x, __uint_as_float(v[kAccs - 1 - plane][j + e]), plane == 0 ? -1.0f : 1.0f);
          }
          fma_to(sum[plane][c + j + e], x, f[e]);
        }
      }
    }
  }
}

// alpha and beta on the sums of row m, columns n0 .. n0 + COLS.
template <typename OutT, int COLS>
__device__ __forceinline__ void scale_sums(const GemmParams &p, uint32_t b, uint32_t m, uint32_t n0,
                                           float (&re)[COLS], float (&im)[COLS]) {
  if (p.have_alpha) {
#pragma unroll
    for (int j = 0; j < COLS; ++j) {
      const float r = re[j];
      re[j] = p.alpha_re * r - p.alpha_im * im[j];
      im[j] = p.alpha_im * r + p.alpha_re * im[j];
    }
  }
  if (p.have_beta && m < p.M) {
    const COffsets o = c_offsets(p, b, m, n0);
    const OutT *C = static_cast<const OutT *>(p.c);
#pragma unroll
    for (int j = 0; j < COLS; ++j) {
      if (n0 + j < p.N) {
        const float cr = OutTraits<OutT>::to_acc(C[o.base_re + j * o.stride_j]);
        const float ci = OutTraits<OutT>::to_acc(C[o.base_re + j * o.stride_j + o.off_im]);
        re[j] += p.beta_re * cr - p.beta_im * ci;
        im[j] += p.beta_im * cr + p.beta_re * ci;
      }
    }
  }
}

// The rows of a warp's part of C leave in boxes of 32 rows x 64 bytes: the pieces of the real plane,
// then those of the imaginary one; or, interleaved, the pieces of the (re, im) sequence in order.
template <typename OutT, int COLS> struct Boxes {
  static constexpr int kPer = 4 / static_cast<int>(sizeof(OutT));  // values per word
  static constexpr int kPlane = COLS * static_cast<int>(sizeof(OutT)) / kStoreBytes;
  static constexpr int kCount = 2 * kPlane;
};

// Word J of box T of a row.
template <typename OutT, int COLS, int T, int J>
__device__ __forceinline__ uint32_t row_word(bool inter, const float (&re)[COLS],
                                             const float (&im)[COLS]) {
  using B = Boxes<OutT, COLS>;
  float v[2];
  if (inter) {
    constexpr int e = (T * 16 + J) * B::kPer;  // place in the (re, im) sequence
    v[0] = (e & 1) ? im[e / 2] : re[e / 2];
    v[1] = im[e / 2];  // 16-bit words hold a whole (re, im); unused otherwise
  } else {
    constexpr int c = ((T % B::kPlane) * 16 + J) * B::kPer;
    v[0] = T < B::kPlane ? re[c] : im[c];
    v[1] = T < B::kPlane ? re[c + B::kPer - 1] : im[c + B::kPer - 1];
  }
  return Packer<OutT>::word(v);
}

template <typename OutT, int COLS, int T, int... J>
__device__ __forceinline__ void row_words(bool inter, const float (&re)[COLS],
                                          const float (&im)[COLS], uint32_t (&w)[16]) {
  if constexpr (sizeof...(J) < 16) {
    row_words<OutT, COLS, T, J..., static_cast<int>(sizeof...(J))>(inter, re, im, w);
  } else {
    ((w[J] = row_word<OutT, COLS, T, J>(inter, re, im)), ...);
  }
}

// One box through one of the warp's staging tiles (written the way a 64-byte-swizzled TMA store reads it: 16-byte
// piece j of row r at j ^ ((r >> 1) & 3)) and out.
template <typename OutT, int COLS, int T>
__device__ __forceinline__ void store_box(const GemmParams &p, const CUtensorMap *tm_c,
                                          uint32_t staging, uint32_t lane, uint32_t b, uint32_t m0,
                                          uint32_t n0, const float (&re)[COLS],
                                          const float (&im)[COLS]) {
  using B = Boxes<OutT, COLS>;
  const bool inter = p.c_layout == kInterRow;
  const uint32_t first = n0 + (inter ? T * 8 * B::kPer : (T % B::kPlane) * 16 * B::kPer);
  if (first >= p.N || m0 >= p.M) {  // uniform over the warp
    // an empty group keeps the count: a staging tile is free when all but the newest group are done
    if (lane == 0) bulk_commit_group();
    return;
  }
  uint32_t w[16];
  row_words<OutT, COLS, T>(inter, re, im, w);
  if (lane == 0) bulk_wait_group_read<kStoreTiles - 1>();
  __syncwarp();
  const uint32_t tile = staging + (T % kStoreTiles) * kStoreTile;
  const uint32_t row = tile + lane * kStoreBytes;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    st_shared_v4(row + ((j ^ ((lane >> 1) & 3)) << 4), w[4 * j], w[4 * j + 1], w[4 * j + 2],
                 w[4 * j + 3]);
  }
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) {
    const int32_t x = static_cast<int32_t>(first * sizeof(OutT) * (inter ? 2 : 1));
    const int32_t z = static_cast<int32_t>(inter ? b : 2 * b + (T < B::kPlane ? 0 : 1));
    tma_store_3d(tm_c, tile, x, static_cast<int32_t>(m0), z);
    bulk_commit_group();
  }
}

template <typename OutT, int COLS, int... T>
__device__ __forceinline__ void store_boxes(const GemmParams &p, const CUtensorMap *tm_c,
                                            uint32_t staging, uint32_t lane, uint32_t b, uint32_t m0,
                                            uint32_t n0, const float (&re)[COLS],
                                            const float (&im)[COLS]) {
  if constexpr (sizeof...(T) < Boxes<OutT, COLS>::kCount) {
    store_boxes<OutT, COLS, T..., static_cast<int>(sizeof...(T))>(p, tm_c, staging, lane, b, m0, n0,
                                                                  re, im);
  } else {
    (store_box<OutT, COLS, T>(p, tm_c, staging, lane, b, m0, n0, re, im), ...);
  }
}

// Row m (m0 + lane), COLS columns from n0, without the TMA unit.  Row-major rows that start anywhere turn in
// the warp's staging tiles, kTurn columns of one plane at a time, so that lanes store along the row
// (a lane to a row, a store touched 32 rows: 3 x 1000 x 2501 x 1984 took 180 us).
template <typename OutT, int COLS>
__device__ __forceinline__ void store_direct(const GemmParams &p, float *turn, uint32_t lane, uint32_t b,
                                             uint32_t m0, uint32_t n0, const float (&re)[COLS],
                                             const float (&im)[COLS]) {
  if (m0 >= p.M || n0 >= p.N) return;  // uniform over the warp
  using Tr = OutTraits<OutT>;
  OutT *C = static_cast<OutT *>(p.c);
  if (p.c_layout == kPlanarRow || p.c_layout == kInterRow) {
    constexpr int kTurn = COLS < 32 ? COLS : 32;
    static_assert(32 * kTurn * sizeof(float) <= kStoreTiles * kStoreTile, "staging");
    constexpr uint32_t kRows = 32 / kTurn;  // rows stored by one instruction
    const COffsets o = c_offsets(p, b, m0, n0);
    const size_t pitch = (p.c_layout == kInterRow ? 2 : 1) * static_cast<size_t>(p.N);
    const uint32_t rows = min(32u, p.M - m0), col = lane % kTurn, sub = lane / kTurn;
#pragma unroll
    for (int c = 0; c < COLS; c += kTurn) {
#pragma unroll
      for (int plane = 0; plane < 2; ++plane) {
        __syncwarp();
#pragma unroll
        for (int j = 0; j < kTurn; ++j) {
          turn[lane * kTurn + (j ^ (lane & (kTurn - 1)))] = plane == 0 ? re[c + j] : im[c + j];
        }
        __syncwarp();
        OutT *dst = C + o.base_re + (plane == 0 ? 0 : o.off_im) + (c + col) * o.stride_j;
        if (n0 + c + col < p.N) {
          for (uint32_t r = sub; r < rows; r += kRows) {
            dst[r * pitch] = Tr::to_out(turn[r * kTurn + (col ^ (r & (kTurn - 1)))]);
          }
        }
      }
    }
    __syncwarp();
    return;
  }
  // column-major: consecutive lanes hold consecutive rows
  const uint32_t m = m0 + lane;
  if (m >= p.M) return;
  const COffsets o = c_offsets(p, b, m, n0);
  const int valid = static_cast<int>(min(static_cast<uint32_t>(COLS), p.N - n0));
  if (p.c_layout == kInterCol && p.pair_ok) {
    // one store per complex value
    struct alignas(2 * sizeof(OutT)) Pair {
      OutT re, im;
    };
#pragma unroll
    for (int j = 0; j < COLS; ++j) {
      if (j < valid) {
        *reinterpret_cast<Pair *>(C + o.base_re + j * o.stride_j) =
            Pair{Tr::to_out(re[j]), Tr::to_out(im[j])};
      }
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < COLS; ++j) {
    if (j < valid) {
      C[o.base_re + j * o.stride_j] = Tr::to_out(re[j]);
      C[o.base_re + j * o.stride_j + o.off_im] = Tr::to_out(im[j]);
    }
  }
}

template <int BN, typename OutT>
__global__ void __launch_bounds__(ScaledCfg<BN>::kThreads, 1)
scaled_gemm_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                   const __grid_constant__ CUtensorMap tm_c, const ScaledParams p) {
  using C = ScaledCfg<BN>;
  constexpr int kStages = C::kStages;
  constexpr int COLS = C::kCols;

  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023u) & ~static_cast<uintptr_t>(1023u));
  uint64_t *bars =
      reinterpret_cast<uint64_t *>(smem + kStages * C::kStageBytes + C::kStagingBytes);
  const uint32_t bar_full = smem_u32(bars);
  const uint32_t bar_empty = bar_full + 8 * kStages;
  const uint32_t bar_acc_full = bar_empty + 8 * kStages;
  const uint32_t bar_acc_empty = bar_acc_full + 8 * kAccBuffers;
  const uint32_t bar_turn = bar_acc_empty + 8 * kAccBuffers;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * kStages + 2 * kAccBuffers + 2);
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
      mbar_init(bar_acc_empty + 8 * s, C::kEpiWarps);
    }
    mbar_init(bar_turn, 1);
    mbar_init(bar_turn + 8, 1);
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
  let_next_start();

  if (warp < C::kFirstEpiWarp) {
    if constexpr (C::kSplitRegs) regs_dec<40>();
    Walk walk(p);
    Segment seg;
    if (warp == 0) {
      // ------------------------------------------------------------------ TMA producer
      wait_for_previous();
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
    } else if (warp <= 2) {
      // ------------------------------------------------------------------ MMA issuers
      // Two warps take the blocks in turn, each its own accumulator buffer.  Issuing blocks while the tensor
      // core's short queue is full, so one warp alone leaves the tensor core idle while it waits for the
      // barriers of the next block (350 clocks of 1900); the other has done that when its turn comes.
      wait_for_previous();  // its run time is not counted against the limits below
      const uint32_t acc = warp - 1;
      const uint64_t blocks = walk.blocks(p);
      uint32_t stage = acc, phase = 0, turn = 0;
      static_assert(kStages > 2 && kAccBuffers == 2, "a stage and a buffer for either warp");
      for (uint64_t i = acc; i < blocks; i += 2, ++turn) {
        if (!mbar_wait(bar_acc_empty + 8 * acc, (turn & 1) ^ 1, abort_flag, p.g.status, kDevTimeoutMma,
                       p.g.wait_cycles) ||
            !mbar_wait(bar_full + 8 * stage, phase, abort_flag, p.g.status, kDevTimeoutMma,
                       p.g.wait_cycles)) {
          break;
        }
        // the other warp has issued block i - 1
        if (i > 0 && !mbar_wait(bar_turn + 8 * acc, (acc == 0 ? turn - 1 : turn) & 1, abort_flag, p.g.status,
                                kDevTimeoutMma, p.g.wait_cycles)) {
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
          if (i + 1 < blocks) mbar_arrive(bar_turn + 8 * (acc ^ 1));
          tc_commit(bar_empty + 8 * stage);
          tc_commit(bar_acc_full + 8 * acc);
        }
        __syncwarp();
        stage += 2;
        if (stage >= kStages) {
          stage -= kStages;
          phase ^= 1;
        }
      }
    }
  } else {
    // ------------------------------------------------------------------ epilogue warps
    if constexpr (C::kSplitRegs) regs_inc<232>();
    wait_for_previous();
    Walk walk(p);
    Segment seg{};
    const uint32_t quad = warp & 3;                       // tensor-memory lanes of this warp
    const uint32_t first_col = ((warp - C::kFirstEpiWarp) >> 2) * COLS;  // columns of this warp
    const uint32_t staging =
        smem_base + kStages * C::kStageBytes + (warp - C::kFirstEpiWarp) * (kStoreTiles * kStoreTile);
    // the column scales of the block (two buffers) at the head of the staging tile
    float *col_buf = reinterpret_cast<float *>(
        smem + kStages * C::kStageBytes + (warp - C::kFirstEpiWarp) * (kStoreTiles * kStoreTile));
    uint32_t acc = 0, acc_phase = 0;
    bool ok = true;
    // the scales of the next block: this lane's row, and two of the warp's columns
    const float *rs = nullptr, *cs = nullptr;
    float s_next = 0.0f, t0_next = 0.0f, t1_next = 0.0f;
    uint32_t ri = 0, i0 = 0, i1 = 0;
    bool row_in = false, in0 = false, in1 = false;
    auto load_scales = [&]() {
      s_next = row_in ? __ldg(rs + ri) : 0.0f;
      t0_next = in0 ? __ldg(cs + i0) : 0.0f;
      t1_next = in1 ? __ldg(cs + i1) : 0.0f;
    };
    auto first_scales = [&](const Segment &of) {
      const TileCoord t = decode_tile(p.g, of.tile);
      const uint32_t m = t.mt * kBlockM + quad * 32 + lane, c0 = t.nt * BN + first_col + 2 * lane;
      const size_t block = static_cast<size_t>(t.b) * p.g.k_blocks + of.k0;
      rs = p.row_scale + block * p.row_blocks;
      cs = p.col_scale + block * p.col_blocks;
      row_in = m < p.g.M;
      in0 = 2 * lane < COLS && c0 < p.g.N;
      in1 = 2 * lane < COLS && c0 + 1 < p.g.N;
      ri = m >> p.row_shift;
      i0 = c0 >> p.col_shift;
      i1 = (c0 + 1) >> p.col_shift;
      load_scales();
    };
    bool more = walk.next(p, seg);
    if (more) first_scales(seg);
    while (more) {
      float sum[2][COLS];  // Re, Im
      const TileCoord t = decode_tile(p.g, seg.tile);
      const uint32_t m = t.mt * kBlockM + quad * 32 + lane;
      const uint32_t n0 = t.nt * BN + first_col;
#pragma unroll
      for (int j = 0; j < COLS; ++j) sum[0][j] = sum[1][j] = 0.0f;
      // what this row's sums are kept times
      float up = 1.0f;
      bool lifted = false;
      auto lower = [&]() {
        const float down = up == 0x1p64f ? 0x1p-64f : 0x1p-117f;
#pragma unroll
        for (int j = 0; j < COLS; j += 2) {
          mul_pair(sum[0][j], sum[0][j + 1], down);
          mul_pair(sum[1][j], sum[1][j + 1], down);
        }
        up = 1.0f;
        lifted = false;
      };
      for (uint32_t kb = seg.k0; ok && kb < seg.k1; ++kb) {
        const float s = s_next, t0 = t0_next, t1 = t1_next;
        if (kb + 1 < seg.k1) {
          rs += p.row_blocks;
          cs += p.col_blocks;
          load_scales();
        }
        // any column's scale stands for the block's where one covers 128 columns
        const float col = __shfl_sync(0xFFFFFFFFu, t0, 0);
        bool plain = __all_sync(0xFFFFFFFFu, in_range(s * up, t0, t1, lifted, p.lift_limit));
        if (!plain) {
          if (kb == seg.k0) {
            lifted = true;
            up = s != 0.0f && fabsf(s) < 0x1p-63f ? 0x1p117f : 0x1p64f;
            plain = __all_sync(0xFFFFFFFFu, in_range(s * up, t0, t1, true, p.lift_limit));
          }
          if (!plain && lifted) {
            lower();
            plain = __all_sync(0xFFFFFFFFu, in_range(s, t0, t1, false, p.lift_limit));
          }
        }
        const bool one = plain && p.col_shift != 0;
        float *cols = col_buf + (kb & 1) * COLS;
        if (!one) {
          // through the staging tile, once the last stores have read it
          if (lane == 0) bulk_wait_group_read<0>();
          __syncwarp();
          if (2 * lane < COLS) {
            *reinterpret_cast<float2 *>(cols + 2 * lane) = make_float2(t0, t1);
          }
          __syncwarp();
        }
        ok = mbar_wait(bar_acc_full + 8 * acc, acc_phase, abort_flag, p.g.status,
                       kDevTimeoutEpilogue, p.g.wait_cycles);
        ok = __all_sync(0xFFFFFFFFu, ok);
        if (!ok) break;
        tc_fence_after();
        const uint32_t taddr =
            tmem_base + ((quad * 32) << 16) + acc * C::kAccCols + first_col;
        const uint32_t done = bar_acc_empty + 8 * acc;
        if (plain && !one) {
          add_block<BN, false>(taddr, done, lane, cols, s * up, 0.0f, sum);
        } else {
          if (!plain) {
            constexpr uint32_t kLow = exponent_bits(-126), kHigh = exponent_bits(63);
            const bool small = __all_sync(0xFFFFFFFFu, zero_or_between(s, kLow, kHigh) &&
                                                           zero_or_between(t0, kLow, kHigh) &&
                                                           zero_or_between(t1, kLow, kHigh));
            scale_block<BN>(taddr, cols, s, small);
          }
          add_block<BN, true>(taddr, done, lane, cols, plain ? s * up : 1.0f, plain ? col : 1.0f, sum);
        }
        if (++acc == kAccBuffers) {
          acc = 0;
          acc_phase ^= 1;
        }
      }
      if (lifted) lower();
      // the next tile's first scales are on their way while this tile is stored
      Segment next{};
      more = walk.next(p, next);
      if (more) first_scales(next);
      float(&re)[COLS] = sum[0], (&im)[COLS] = sum[1];
      bool finish = ok;
      if (seg.k1 - seg.k0 < p.g.k_blocks) {
        // Part of a tile: add it through the workspace.  A CTA's run holds at most one part that
        // begins inside a tile (slot 0) and one that begins a tile without ending it (slot 1).
        // The counter is kept up even after a wait gave up, so that it is zero for the next run.
        constexpr size_t kPart = 2 * BN * kBlockM;
        const uint64_t units = static_cast<uint64_t>(p.g.num_tiles) * p.g.k_blocks;
        const uint64_t base = static_cast<uint64_t>(seg.tile) * p.g.k_blocks;
        // [plane][column / 4][row][column % 4]: a lane moves four columns of its row at a time
        const uint32_t at = (first_col * kBlockM + (quad * 32 + lane) * 4);
        float *mine = p.parts + (2 * static_cast<size_t>(blockIdx.x) + (seg.k0 == 0 ? 1 : 0)) * kPart + at;
#pragma unroll
        for (int j = 0; j < COLS; j += 4) {
          __stcg(reinterpret_cast<float4 *>(mine + j * kBlockM),
                 make_float4(re[j], re[j + 1], re[j + 2], re[j + 3]));
          __stcg(reinterpret_cast<float4 *>(mine + (BN + j) * kBlockM),
                 make_float4(im[j], im[j + 1], im[j + 2], im[j + 3]));
        }
        __threadfence();
        epi_sync<32 * C::kEpiWarps>();
        if (threadIdx.x == 32 * C::kFirstEpiWarp) {
          const unsigned add = seg.k1 - seg.k0;
          const unsigned before = atomicAdd(p.counters + seg.tile, add);
          const bool last = before + add == p.g.k_blocks;
          if (last) p.counters[seg.tile] = 0;
          __threadfence();
          *last_flag = last ? 1u : 0u;
        }
        epi_sync<32 * C::kEpiWarps>();
        finish = *last_flag != 0 && ok;
        epi_sync<32 * C::kEpiWarps>();  // the flag may be written again
        if (finish) {
#pragma unroll
          for (int j = 0; j < COLS; ++j) re[j] = im[j] = 0.0f;
          const uint32_t from = run_owner(units, gridDim.x, base);
          const uint32_t to = run_owner(units, gridDim.x, base + p.g.k_blocks - 1);
          for (uint32_t c = from; c <= to; ++c) {
            const uint32_t slot = run_start(units, gridDim.x, c) > base ? 0 : 1;
            const float *part = p.parts + (2 * static_cast<size_t>(c) + slot) * kPart + at;
#pragma unroll
            for (int j = 0; j < COLS; j += 4) {
              const float4 x = __ldcg(reinterpret_cast<const float4 *>(part + j * kBlockM));
              const float4 y = __ldcg(reinterpret_cast<const float4 *>(part + (BN + j) * kBlockM));
              re[j] += x.x; re[j + 1] += x.y; re[j + 2] += x.z; re[j + 3] += x.w;
              im[j] += y.x; im[j + 1] += y.y; im[j + 2] += y.z; im[j + 3] += y.w;
            }
          }
        }
      }
      if (finish) {
        scale_sums<OutT, COLS>(p.g, t.b, m, n0, re, im);
        bool stored = false;
        if constexpr (Boxes<OutT, COLS>::kPlane > 0) {
          if (p.g.epi_tma) {
            store_boxes<OutT, COLS>(p.g, &tm_c, staging, lane, t.b, t.mt * kBlockM + quad * 32, n0,
                                    re, im);
            stored = true;
          }
        }
        if (!stored) {
          store_direct<OutT, COLS>(p.g, col_buf, lane, t.b, t.mt * kBlockM + quad * 32, n0, re, im);
        }
      }
      seg = next;
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
  int smem, threads;
  bool boxes;  // a warp's columns fill the boxes of the TMA store
};

template <int BN, typename OutT> ScaledEntry entry() {
  using C = ScaledCfg<BN>;
  return {scaled_gemm_kernel<BN, OutT>, C::kSmemBytes, C::kThreads, Boxes<OutT, C::kCols>::kPlane > 0};
}

template <typename OutT> ScaledEntry pick_width(int bn) {
  return bn == 128  ? entry<128, OutT>()
         : bn == 64 ? entry<64, OutT>()
         : bn == 32 ? entry<32, OutT>()
                    : entry<16, OutT>();
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
  const size_t sms = static_cast<size_t>(plan.sms);
  const int narrowest = plan.cols <= 16 ? 16 : plan.cols <= 32 ? 32 : plan.cols <= 64 ? 64 : 0;
  const char *env = std::getenv("CCGLIB_B200_SCALED_BN");
  const int forced_bn = env != nullptr ? std::atoi(env) : 0;
  env = std::getenv("CCGLIB_B200_SCALED_RUNS");
  const int forced_runs = env != nullptr && *env != '\0' ? std::atoi(env) : -1;
  // Whole tiles, or all blocks in equal runs?  And 128 or 64 columns where there is a choice?  Estimated
  // in clocks; on 16 shapes from 256 x 256 x 256 to 4096 x 4096 x 4096 the choice is within 4 % of the
  // best of the four forms (1024 x 1024 x 1024: 11.0 us, the others 13.6 to 18.8; 256 x 256 x 4096: 17.5,
  // the others 24 to 32; 2048 x 2048 x 2048: 39, the others 52 to 59).
  const size_t col_block = plan.swapped ? d.a_block_rows : d.b_block_rows;
  double least = 0.0;
  for (int bn : {128, 64, 32, 16}) {
    if (narrowest != 0 ? bn != narrowest : bn < 64) continue;
    if (forced_bn != 0 && narrowest == 0 && bn != forced_bn) continue;
    const size_t tiles = d.batch * ceil_div<size_t>(plan.rows, kBlockM) * ceil_div<size_t>(plan.cols, bn);
    const size_t units = tiles * plan.k_blocks;
    // clocks of one block, of storing a tile, and of adding a shared tile's parts, measured
    const bool one = col_block == 1;  // a factor for every column
    const double block = bn == 128 ? (one ? 2200.0 : 1600.0) : bn == 64 ? (one ? 1450.0 : 1150.0) : 800.0;
    const double store = 40.0 * bn, part = 350.0 * bn;
    const double whole = static_cast<double>(ceil_div(tiles, sms)) *
                         (static_cast<double>(plan.k_blocks) * block + store);
    const size_t ctas = units / 4 < sms ? units / 4 : sms;
    const double shared = ctas > 0 ? static_cast<double>(units) / static_cast<double>(ctas) * block +
                                         store + part
                                   : 0.0;
    const bool may_share = plan.k_blocks > 1 && ctas > 1 && ceil_div(tiles, sms) <= 4;
    const bool runs = may_share && (forced_runs >= 0 ? forced_runs != 0 : shared < whole);
    const double cost = runs ? shared : whole;
    if (plan.tiles == 0 || cost < least) {
      least = cost;
      plan.bn = bn;
      plan.tiles = tiles;
      plan.runs = runs ? ctas : 0;
    }
  }
  if (plan.tiles == 0) {
    set_last_error("CCGLIB_B200_SCALED_BN must be 64 or 128");
    return CCGLIB_B200_INVALID_ARGUMENT;
  }
  if (plan.tiles > 0x7FFFFFFFull) {
    set_last_error("scaled_gemm_plan_create: too many tiles");
    return CCGLIB_B200_INVALID_ARGUMENT;
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
  const size_t pitch = ceil_div<size_t>(d.k, 16) * 16;
  const size_t c_bytes = d.batch * 2 * d.m * d.n * plan->out_bytes;
  const size_t scale_bytes = d.batch * plan->k_blocks * sizeof(float);
  if (overlap(d_c, c_bytes, d_a, d.batch * 2 * d.m * pitch) ||
      overlap(d_c, c_bytes, d_b, d.batch * 2 * d.n * pitch) ||
      overlap(d_c, c_bytes, d_a_scale, scale_bytes * ceil_div(d.m, d.a_block_rows)) ||
      overlap(d_c, c_bytes, d_b_scale, scale_bytes * ceil_div(d.n, d.b_block_rows))) {
    set_last_error("scaled_gemm_run: C overlaps an operand");
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
  g.epi_tma = g.vec_ok && plan->kernel.boxes ? 1u : 0u;
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
  // 2^l: largest scales whose blocks, lifted by 2^64, add up to less than 2^127.  A block's sums are at
  // most 256 products of the types' largest values (448 < 2^9, 57344 < 2^16).
  const double most = std::log2(256.0 * static_cast<double>(plan->k_blocks)) +
                      (d.type_a == CCGLIB_B200_FLOAT8E5M2 ? 16.0 : 9.0) +
                      (d.type_b == CCGLIB_B200_FLOAT8E5M2 ? 16.0 : 9.0);
  p.lift_limit = static_cast<uint32_t>(127 + static_cast<int>(std::floor((63.0 - most) / 2))) << 23;

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
                  plan->rows * run_bytes, kStoreBytes, 32, 1);
    if (rc != CCGLIB_B200_OK) return rc;
  }
  const size_t ctas = plan->runs > 0 ? plan->runs
                      : plan->tiles < static_cast<size_t>(plan->sms) ? plan->tiles
                                                                     : plan->sms;
  CCGLIB_CUDA_TRY(launch_programmatic(plan->kernel.fn, static_cast<unsigned>(ctas), plan->kernel.threads,
                                      plan->kernel.smem, 1, static_cast<cudaStream_t>(stream_v), tm_a, tm_b,
                                      tm_c, p));
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
