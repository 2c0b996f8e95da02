// Orthogonalisation of complex matrices by Newton-Schulz products.
//
//   X <- X / ||X||_F;   `steps` times:  S = X X^H,  P = a I + b S + c S S,  X <- P X
//
// (M <= N; for M > N the same on X^T, i.e. S = X^T conj(X) and X <- X P^T).  Every step keeps the
// singular vectors and maps each singular value s to s (a + b s^2 + c s^4).
//
// Three launches per step and nothing else, float32 sums on the tensor cores (kind::f16).  S and P are
// Hermitian: only tiles on and above the diagonal are computed, each stored a second time as its
// mirror image.  X is never transposed: where a product contracts over rows, its operand is read with
// the rows as K (the MN-major form of the shared-memory descriptor).  The Gram product stores S + b/2c I,
// whose square is P but for a factor and a multiple of I; the last update writes the caller's type and
// layout.  The launches are programmatic: a product's CTAs set up while the one before it drains.
//
// X, S and P are states of the iteration and are kept as pairs of float16, the rounded value and what the
// rounding leaves, times powers of two that put their largest possible entries near the top of float16
// (choose_scales): about 20 bits, also in rows fainter than the others by several decades.  A product
// takes its K three times, low x high, high x low and high x high, into the same float32 sums.  What is
// lost in the end is the rounding of the output (relative error 2.1e-4 float16, 1.7e-3 bfloat16).  Single
// float16 iterates take a third of the multiplications, but a step's roundings do not decay, those that
// turn the singular vectors least of all: they ended at 7e-4 after eight steps that converge and at 1.4 to
// 3.8e-3 after 5 to 8 of the steep quintic.  Leaving out one of the low halves (of X in S, of S, of P)
// still ends at 5e-4 to 3e-3 in the steep map.
//
// Measured: 8 x 4096 x 1024, eight steps, 9.8 to 10.1 ms (1.07 PFLOP/s in the three passes over K,
// power-capped); 1024 x 1024, five steps, 344 to 353 us (23 us a product of 1024^3 in three passes: operands
// on their way from L2 into 144 SMs, and two latencies).  Single float16: 3.5 ms and 182 us.
#include <cmath>
#include <cstdlib>
#include <new>

#include "gemm_kernels.cuh"

namespace ccglib_b200 {
namespace {

constexpr int kOrthK = 64;          // float16 values of K per stage: one 128-byte swizzle span
constexpr int kOrthBox = 32 * 64;   // staging box: 32 rows x 32 float16
constexpr int kOrthStaging = 4 * 4 * kOrthBox;  // per epilogue warp: Re, Im and their mirror images

// The products are taken over K three times: low halves of A by high halves of B, high by low, high by high.
// (low by low is below the last bit of either.)
constexpr uint32_t kPasses = 3;

struct OrthParams {
  uint32_t m, n;        // result: m x n per batch item
  uint32_t k_blocks;    // of one pass
  uint32_t tiles_m, tiles_n, group_n;
  uint32_t per_batch, num_tiles;
  uint32_t hermitian;   // compute tiles that touch or lie above the diagonal, store their mirror image
  uint32_t conj_b;      // A x B^H instead of A x B^T
  float alpha, diag;    // result = alpha * sum + diag * I
  uint32_t pair;        // the result is a pair of float16; else float16 or bfloat16
  uint32_t bf16;
  uint32_t boxes;       // the result leaves by TMA; else value by value to `out` [batch][2][m][n_out]
  uint16_t *out;
  uint32_t n_out;
  unsigned int *status;
  long long wait_cycles;
  long long tile_cycles;  // limit of the wait for a tile's sums, all of K
};

template <int BN> struct OrthCfg {
  // 64 columns: one MMA multiplies an A plane by both B planes (see scaled_gemm.cu)
  static constexpr bool kStacked = BN == 64;
  static constexpr int kAccCols = kStacked ? 4 * BN : 2 * BN;
  static constexpr int kAccStages = 2;
  static constexpr int kABytes = 2 * kBlockM * 128;
  static constexpr int kBBytes = 2 * BN * 128;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kStages = (kMaxSmem - 1024 - 256 - kOrthStaging) / kStageBytes;
  static constexpr int kSmemBytes = kStages * kStageBytes + kOrthStaging + 1024 + 256;
  static_assert(kStages >= 3 && kAccCols * kAccStages <= kTmemCols, "tile does not fit");
};

// Shared-memory descriptor of an operand whose rows are K: 128-byte rows of 64 values along M or N,
// groups of eight rows 1024 bytes apart, the next 64 values `atom` bytes on.
__device__ __forceinline__ uint64_t smem_desc_mn(uint32_t saddr, uint32_t atom) {
  return static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(atom >> 4) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

template <int BN>
__device__ __forceinline__ TileCoord orth_tile(const OrthParams &p, uint32_t tile) {
  TileCoord t;
  t.b = tile / p.per_batch;
  uint32_t r = tile - t.b * p.per_batch;
  if (p.hermitian) {
    for (t.mt = 0;; ++t.mt) {
      const uint32_t first = t.mt * kBlockM / BN, width = p.tiles_n - first;
      if (r < width) {
        t.nt = first + r;
        return t;
      }
      r -= width;
    }
  }
  // column panels, as in decode_tile
  const uint32_t panel = p.group_n * p.tiles_m;
  const uint32_t g = r / panel, first_n = g * p.group_n;
  const uint32_t width = min(p.group_n, p.tiles_n - first_n);
  r -= g * panel;
  t.mt = r / width;
  t.nt = first_n + (r - t.mt * width);
  return t;
}

__device__ __forceinline__ uint32_t pack_half(float lo, float hi, bool bf16) {
  if (bf16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
  }
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&v);
}

__device__ __forceinline__ uint16_t round_half(float v, bool bf16) {
  return bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}

__device__ __forceinline__ void st_shared_u16(uint32_t addr, uint16_t v) {
  asm volatile("st.shared.u16 [%0], %1;" ::"r"(addr), "h"(v) : "memory");
}

// 32 rows x 32 columns (one row per lane, from m0; columns from n0) of one batch item: the sums -> the result.
__device__ __forceinline__ void orth_store(const OrthParams &p, const CUtensorMap *tm_c,
                                           uint32_t staging, uint32_t lane, uint32_t b, uint32_t m0,
                                           uint32_t n0, float (&re)[32], float (&im)[32]) {
  const uint32_t m = m0 + lane;
  const bool diagonal = p.hermitian && n0 == m0;
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    re[j] *= p.alpha;
    im[j] *= p.alpha;
    if (diagonal && j == static_cast<int>(lane)) re[j] += p.diag;
  }
  if (!p.boxes) {
    if (m < p.m) {
      const size_t plane = static_cast<size_t>(p.m) * p.n_out;
      uint16_t *dst = p.out + static_cast<size_t>(b) * 2 * plane + static_cast<size_t>(m) * p.n_out + n0;
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        if (n0 + j < p.n_out) {
          dst[j] = round_half(re[j], p.bf16);
          dst[plane + j] = round_half(im[j], p.bf16);
        }
      }
    }
    return;
  }
  const uint32_t halves = p.pair ? 2 : 1;
  const uint32_t row = staging + lane * 64;
#pragma unroll 1
  for (uint32_t half = 0; half < halves; ++half) {
    // 16-byte piece j of row r of a box stands at j ^ ((r >> 1) & 3): the 64-byte swizzle
    if (lane == 0) bulk_wait_group_read<0>();
    __syncwarp();
    uint32_t r[16], i[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      r[j] = pack_half(re[2 * j], re[2 * j + 1], p.bf16);
      i[j] = pack_half(im[2 * j], im[2 * j + 1], p.bf16);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t at = row + ((j ^ ((lane >> 1) & 3)) << 4);
      st_shared_v4(at, r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
      st_shared_v4(at + kOrthBox, i[4 * j], i[4 * j + 1], i[4 * j + 2], i[4 * j + 3]);
    }
    if (p.hermitian) {
      // the mirror image: row n0 + j, this lane's column.  On the diagonal block it goes over the
      // rows just written: below the diagonal, and zero imaginary parts on it.
      const uint32_t mirror = diagonal ? staging : staging + 2 * kOrthBox;
      if (diagonal) __syncwarp();
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        if (!diagonal || j > static_cast<int>(lane)) {
          const uint32_t at = mirror + j * 64 + (((lane >> 3) ^ ((j >> 1) & 3)) << 4) + (lane & 7) * 2;
          const int shift = 16 * (j & 1);
          st_shared_u16(at, static_cast<uint16_t>(r[j / 2] >> shift));
          st_shared_u16(at + kOrthBox, static_cast<uint16_t>((i[j / 2] >> shift) ^ 0x8000u));
        }
      }
      if (diagonal) {
        st_shared_u16(staging + kOrthBox + lane * 64 + (((lane >> 3) ^ ((lane >> 1) & 3)) << 4) +
                          (lane & 7) * 2, 0);
      }
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      const int32_t z = static_cast<int32_t>(2 * (halves * b + half));
      const int32_t x = static_cast<int32_t>(n0 * 2), y = static_cast<int32_t>(m0);
      if (m0 < p.m) {
        tma_store_3d(tm_c, staging, x, y, z);
        tma_store_3d(tm_c, staging + kOrthBox, x, y, z + 1);
        if (p.hermitian && !diagonal && n0 < p.m) {
          const int32_t tx = static_cast<int32_t>(m0 * 2), ty = static_cast<int32_t>(n0);
          tma_store_3d(tm_c, staging + 2 * kOrthBox, tx, ty, z);
          tma_store_3d(tm_c, staging + 3 * kOrthBox, tx, ty, z + 1);
        }
      }
      bulk_commit_group();
    }
    if (half + 1 < halves) {  // what the rounding leaves (pairs are float16)
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float2 hr = __half22float2(*reinterpret_cast<const __half2 *>(&r[j]));
        const float2 hi = __half22float2(*reinterpret_cast<const __half2 *>(&i[j]));
        re[2 * j] -= hr.x;
        re[2 * j + 1] -= hr.y;
        im[2 * j] -= hi.x;
        im[2 * j + 1] -= hi.y;
      }
    }
  }
}

constexpr uint32_t kAtom = 2 * kOrthK * 128;  // 64 values along M or N of both planes, MN-major

// Loads of one stage: block kb (of all passes) of tile t.
template <int BN, bool A_MN, bool B_MN>
__device__ __forceinline__ void load_stage(const OrthParams &p, const CUtensorMap *tm_a,
                                           const CUtensorMap *tm_b, const TileCoord &t, uint32_t kb,
                                           uint32_t dst, uint32_t full) {
  using C = OrthCfg<BN>;
  const uint32_t pass = kb / p.k_blocks;
  const int32_t k = static_cast<int32_t>((kb - pass * p.k_blocks) * kOrthK);
  // the planes of a batch item: high Re, Im, low Re, Im
  const int32_t z_a = static_cast<int32_t>(4 * t.b + (pass == 0 ? 2 : 0));
  const int32_t z_b = static_cast<int32_t>(4 * t.b + (pass == 1 ? 2 : 0));
  const int32_t m0 = static_cast<int32_t>(t.mt * kBlockM), n0 = static_cast<int32_t>(t.nt * BN);
  mbar_arrive_expect_tx(full, C::kStageBytes);
  if constexpr (A_MN) {
#pragma unroll
    for (int i = 0; i < kBlockM / 64; ++i) tma_load_3d(dst + i * kAtom, tm_a, (m0 + 64 * i) * 2, k, z_a, full);
  } else {
    tma_load_3d(dst, tm_a, k * 2, m0, z_a, full);
  }
  if constexpr (B_MN) {
#pragma unroll
    for (int i = 0; i < BN / 64; ++i) {
      tma_load_3d(dst + C::kABytes + i * kAtom, tm_b, (n0 + 64 * i) * 2, k, z_b, full);
    }
  } else {
    tma_load_3d(dst + C::kABytes, tm_b, k * 2, n0, z_b, full);
  }
}

// MMAs of one stage into the accumulators at d; more: add to what is there.
template <int BN, bool A_MN, bool B_MN>
__device__ __forceinline__ void issue_stage(uint32_t a_base, uint32_t d, bool conj_b, bool more) {
  using C = OrthCfg<BN>;
  // descriptor: fp32 sums, f16 operands, bit 13 negates A, bits 15 / 16 say that A / B is MN-major
  constexpr uint32_t kIdesc = (1u << 4) | (A_MN ? 1u << 15 : 0u) | (B_MN ? 1u << 16 : 0u) |
                              (static_cast<uint32_t>((C::kStacked ? 2 * BN : BN) >> 3) << 17) |
                              (static_cast<uint32_t>(kBlockM >> 4) << 24);
  constexpr uint32_t kNegA = kIdesc | (1u << 13);
  // A x B^T: Re = Ar.Br - Ai.Bi, Im = Ar.Bi + Ai.Br; with conj(B): Re = Ar.Br + Ai.Bi, Im = Ai.Br - Ar.Bi
  const uint32_t ar_bi = conj_b ? kNegA : kIdesc, ai_bi = conj_b ? kIdesc : kNegA;
  const uint32_t b_base = a_base + C::kABytes;
#pragma unroll
  for (int k = 0; k < kOrthK / 16; ++k) {
    // plane of 64 x 64 values of an MN-major atom: 8 KiB; 16 rows of K: 2 KiB
    const uint64_t a_re = A_MN ? smem_desc_mn(a_base + k * 2048, kAtom) : smem_desc<128>(a_base + k * 32);
    const uint64_t a_im = A_MN ? smem_desc_mn(a_base + kAtom / 2 + k * 2048, kAtom)
                               : smem_desc<128>(a_base + kBlockM * 128 + k * 32);
    const uint32_t add = more || k != 0 ? 1u : 0u;
    if constexpr (C::kStacked) {
      // both B planes lie one behind the other: [Ar.Br | Ar.Bi], [Ai.Br | Ai.Bi]
      const uint64_t b_both = B_MN ? smem_desc_mn(b_base + k * 2048, kAtom / 2)
                                   : smem_desc<128>(b_base + k * 32);
      tc_mma<kKindF16>(d, a_re, b_both, kIdesc, add);
      tc_mma<kKindF16>(d + 2 * BN, a_im, b_both, kIdesc, add);
    } else {
      const uint64_t b_re = B_MN ? smem_desc_mn(b_base + k * 2048, kAtom) : smem_desc<128>(b_base + k * 32);
      const uint64_t b_im = B_MN ? smem_desc_mn(b_base + kAtom / 2 + k * 2048, kAtom)
                                 : smem_desc<128>(b_base + BN * 128 + k * 32);
      tc_mma<kKindF16>(d, a_re, b_re, kIdesc, add);
      tc_mma<kKindF16>(d + BN, a_re, b_im, ar_bi, add);
      tc_mma<kKindF16>(d + BN, a_im, b_re, kIdesc, 1u);
      tc_mma<kKindF16>(d, a_im, b_im, ai_bi, 1u);
    }
  }
}

// 32 columns of the accumulators at taddr as Re and Im.
template <int BN>
__device__ __forceinline__ void read_chunk(uint32_t taddr, bool conj_b, float (&re)[32], float (&im)[32]) {
  uint32_t r[32], i[32];
  tmem_ld_32x32b_x32(taddr, r);
  tmem_ld_32x32b_x32(taddr + BN, i);
  tmem_wait_ld();
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    re[j] = __uint_as_float(r[j]);
    im[j] = __uint_as_float(i[j]);
  }
  if constexpr (OrthCfg<BN>::kStacked) {
    tmem_ld_32x32b_x32(taddr + 2 * BN, i);  // Ai.Br
    tmem_ld_32x32b_x32(taddr + 3 * BN, r);  // Ai.Bi
    tmem_wait_ld();
    const float sign = conj_b ? -1.0f : 1.0f;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      re[j] -= sign * __uint_as_float(r[j]);
      im[j] = sign * im[j] + __uint_as_float(i[j]);
    }
  }
}

// After an abort: our own copies must land before the CTA leaves (or reuses its stages).
template <int STAGES>
__device__ __forceinline__ void drain_loads(uint32_t bar_full, uint32_t issued, uint32_t stage,
                                            uint32_t phase, const OrthParams &p) {
  for (int s = 0; s < STAGES; ++s) {
    if (!(issued & (1u << s))) continue;
    const uint32_t parity = (static_cast<uint32_t>(s) < stage) ? phase : (phase ^ 1);
    const long long t0 = clock64();
    while (!mbar_try_wait(bar_full + 8 * s, parity)) {
      if (clock64() - t0 > p.wait_cycles) {
        atomicOr(p.status, kDevTimeoutDrain);
        break;
      }
    }
  }
}

// result = alpha * A x op(B)^T + diag * I, tiles of 128 x BN, of operands that are pairs of float16.  An
// operand that is MN-major is stored [K][M or N]; the others are stored [M or N][K].  Roles as in
// cgemm_tcgen05_kernel.
template <int BN, bool A_MN, bool B_MN>
__global__ void __launch_bounds__(kThreads, 1)
orth_product_kernel(const __grid_constant__ CUtensorMap tm_a,
                    const __grid_constant__ CUtensorMap tm_b,
                    const __grid_constant__ CUtensorMap tm_c, const OrthParams p) {
  using C = OrthCfg<BN>;
  constexpr int kStages = C::kStages;

  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023u) & ~static_cast<uintptr_t>(1023u));
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + kStages * C::kStageBytes + kOrthStaging);
  const uint32_t bar_full = smem_u32(bars);
  const uint32_t bar_empty = bar_full + 8 * kStages;
  const uint32_t bar_acc_full = bar_empty + 8 * kStages;
  const uint32_t bar_acc_empty = bar_acc_full + 8 * C::kAccStages;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * kStages + 2 * C::kAccStages);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
  const uint32_t smem_base = smem_u32(smem);
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (int s = 0; s < C::kAccStages; ++s) {
      mbar_init(bar_acc_full + 8 * s, 1);
      mbar_init(bar_acc_empty + 8 * s, 4);
    }
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tensormap(&tm_a);
    prefetch_tensormap(&tm_b);
    prefetch_tensormap(&tm_c);
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

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    wait_for_previous();
    uint32_t stage = 0, phase = 0, issued = 0;
    bool ok = true;
    for (uint32_t tile = blockIdx.x; ok && tile < p.num_tiles; tile += gridDim.x) {
      const TileCoord t = orth_tile<BN>(p, tile);
      for (uint32_t kb = 0; kb < kPasses * p.k_blocks; ++kb) {
        if (!mbar_wait(bar_empty + 8 * stage, phase ^ 1, abort_flag, p.status, kDevTimeoutProducer,
                       p.wait_cycles)) {
          ok = false;
          break;
        }
        if (lane == 0) {
          load_stage<BN, A_MN, B_MN>(p, &tm_a, &tm_b, t, kb, smem_base + stage * C::kStageBytes,
                                     bar_full + 8 * stage);
        }
        __syncwarp();
        issued |= 1u << stage;
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    if (*abort_flag) drain_loads<kStages>(bar_full, issued, stage, phase, p);
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    wait_for_previous();  // its run time is not counted against the limits below
    uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0;
    bool ok = true;
    for (uint32_t tile = blockIdx.x; ok && tile < p.num_tiles; tile += gridDim.x) {
      if (!mbar_wait(bar_acc_empty + 8 * acc, acc_phase ^ 1, abort_flag, p.status, kDevTimeoutMma,
                     p.wait_cycles)) {
        break;
      }
      tc_fence_after();
      const uint32_t d = tmem_base + acc * C::kAccCols;
      for (uint32_t kb = 0; kb < kPasses * p.k_blocks; ++kb) {
        if (!mbar_wait(bar_full + 8 * stage, phase, abort_flag, p.status, kDevTimeoutMma,
                       p.wait_cycles)) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (lane == 0) {
          issue_stage<BN, A_MN, B_MN>(smem_base + stage * C::kStageBytes, d, p.conj_b != 0, kb != 0);
          tc_commit(bar_empty + 8 * stage);
          if (kb + 1 == kPasses * p.k_blocks) tc_commit(bar_acc_full + 8 * acc);
        }
        __syncwarp();
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (++acc == C::kAccStages) {
        acc = 0;
        acc_phase ^= 1;
      }
    }
  } else {
    // ------------------------------------------------------------------ epilogue warps
    wait_for_previous();
    const uint32_t quad = warp & 3;
    const uint32_t staging = smem_base + kStages * C::kStageBytes + quad * (4 * kOrthBox);
    uint32_t acc = 0, acc_phase = 0;
    for (uint32_t tile = blockIdx.x; tile < p.num_tiles; tile += gridDim.x) {
      const TileCoord t = orth_tile<BN>(p, tile);
      const uint32_t m0 = t.mt * kBlockM + quad * 32;
      bool ok = mbar_wait(bar_acc_full + 8 * acc, acc_phase, abort_flag, p.status,
                          kDevTimeoutEpilogue, p.tile_cycles);
      if (!__all_sync(0xFFFFFFFFu, ok)) break;
      tc_fence_after();
      const uint32_t taddr = tmem_base + ((quad * 32) << 16) + acc * C::kAccCols;
#pragma unroll 1
      for (uint32_t c0 = 0; c0 < BN; c0 += 32) {
        const uint32_t n0 = t.nt * BN + c0;
        if (n0 >= p.n) break;
        if (m0 >= p.m || (p.hermitian && n0 < m0)) continue;  // comes from the mirror image
        float re[32], im[32];
        read_chunk<BN>(taddr + c0, p.conj_b != 0, re, im);
        orth_store(p, &tm_c, staging, lane, t.b, m0, n0, re, im);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_acc_empty + 8 * acc);
      if (++acc == C::kAccStages) {
        acc = 0;
        acc_phase ^= 1;
      }
    }
    if (lane == 0) bulk_wait_group<0>();
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

// The same for problems whose tiles leave most SMs idle: a cluster of SPLIT CTAs shares the K of one
// tile and every CTA finishes BN / SPLIT of its columns.  Partial sums travel through distributed shared
// memory into the (by then unused) stages, and are added in the order of the CTAs.  1024 x 1024 on
// 72 CTAs of 128 x 64 spent 15.5 k clocks per product loading 48 KiB per block of K through one SM's port to
// L2; shared, a CTA loads half or a quarter of that.
template <int BN, bool A_MN, bool B_MN, int SPLIT>
__global__ void __launch_bounds__(kThreads, 1)
orth_split_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                  const __grid_constant__ CUtensorMap tm_c, const OrthParams p) {
  using C = OrthCfg<BN>;
  constexpr int kStages = C::kStages;
  constexpr uint32_t kChunks = BN / SPLIT / 32;  // 32-column pieces a CTA finishes
  static_assert(BN % (32 * SPLIT) == 0, "whole pieces");
  static_assert((SPLIT - 1) * 2 * kChunks * 4 * kStagingTile <= kStages * C::kStageBytes,
                "partial sums exceed the stages");

  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023u) & ~static_cast<uintptr_t>(1023u));
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + kStages * C::kStageBytes + kOrthStaging);
  const uint32_t bar_full = smem_u32(bars);
  const uint32_t bar_empty = bar_full + 8 * kStages;
  const uint32_t bar_acc_full = bar_empty + 8 * kStages;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * kStages + 1);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
  const uint32_t smem_base = smem_u32(smem);
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    mbar_init(bar_acc_full, 1);
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tensormap(&tm_a);
    prefetch_tensormap(&tm_b);
    prefetch_tensormap(&tm_c);
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

  const TileCoord t = orth_tile<BN>(p, cluster_id_x());
  const uint32_t kb0 = kPasses * p.k_blocks * rank / SPLIT, kb1 = kPasses * p.k_blocks * (rank + 1) / SPLIT;
  bool done = false;  // epilogue warps: this CTA's sums are complete
  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    wait_for_previous();
    uint32_t stage = 0, phase = 0, issued = 0;
    for (uint32_t kb = kb0; kb < kb1; ++kb) {
      if (!mbar_wait(bar_empty + 8 * stage, phase ^ 1, abort_flag, p.status, kDevTimeoutProducer,
                     p.wait_cycles)) {
        break;
      }
      if (lane == 0) {
        load_stage<BN, A_MN, B_MN>(p, &tm_a, &tm_b, t, kb, smem_base + stage * C::kStageBytes,
                                   bar_full + 8 * stage);
      }
      __syncwarp();
      issued |= 1u << stage;
      if (++stage == kStages) {
        stage = 0;
        phase ^= 1;
      }
    }
    if (*abort_flag) drain_loads<kStages>(bar_full, issued, stage, phase, p);
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    wait_for_previous();  // its run time is not counted against the limits below
    uint32_t stage = 0, phase = 0;
    for (uint32_t kb = kb0; kb < kb1; ++kb) {
      if (!mbar_wait(bar_full + 8 * stage, phase, abort_flag, p.status, kDevTimeoutMma, p.wait_cycles)) {
        break;
      }
      tc_fence_after();
      if (lane == 0) {
        issue_stage<BN, A_MN, B_MN>(smem_base + stage * C::kStageBytes, tmem_base, p.conj_b != 0, kb != kb0);
        tc_commit(bar_empty + 8 * stage);
        if (kb + 1 == kb1) tc_commit(bar_acc_full);
      }
      __syncwarp();
      if (++stage == kStages) {
        stage = 0;
        phase ^= 1;
      }
    }
  } else {
    wait_for_previous();
    done = mbar_wait(bar_acc_full, 0, abort_flag, p.status, kDevTimeoutEpilogue, p.tile_cycles);
    done = __all_sync(0xFFFFFFFFu, done);
  }
  __syncwarp();

  // every CTA of the cluster has read its stages (or given up): they may receive partial sums
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  const uint32_t quad = warp & 3;
  const uint32_t taddr = tmem_base + ((quad * 32) << 16);
  // 4 KiB for 32 rows x 32 columns of one plane from source i (of the SPLIT - 1 others)
  auto recv = [&](uint32_t i, uint32_t plane, uint32_t c) {
    return smem_base + ((((i * 2 + plane) * kChunks + c) * 4 + quad) * kStagingTile) + lane * 128;
  };
  if (warp >= 2 && done) {
    for (uint32_t step = 1; step < SPLIT; ++step) {
      const uint32_t dest = (rank + step) % SPLIT;
      const uint32_t idx = rank - (rank > dest ? 1u : 0u);  // our place among dest's sources
#pragma unroll 1
      for (uint32_t c = 0; c < kChunks; ++c) {
        float re[32], im[32];
        read_chunk<BN>(taddr + (dest * kChunks + c) * 32, p.conj_b != 0, re, im);
        const uint32_t to_re = map_to_cta(recv(idx, 0, c), dest), to_im = map_to_cta(recv(idx, 1, c), dest);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t off = (j ^ (lane & 7)) << 4;  // no bank is hit twice
          st_shared_cluster_v4(to_re + off, __float_as_uint(re[4 * j]), __float_as_uint(re[4 * j + 1]),
                               __float_as_uint(re[4 * j + 2]), __float_as_uint(re[4 * j + 3]));
          st_shared_cluster_v4(to_im + off, __float_as_uint(im[4 * j]), __float_as_uint(im[4 * j + 1]),
                               __float_as_uint(im[4 * j + 2]), __float_as_uint(im[4 * j + 3]));
        }
      }
    }
  }
  __syncwarp();
  cluster_sync();  // all partial sums are in place

  if (warp >= 2 && done && !*abort_flag) {
    const uint32_t staging = smem_base + kStages * C::kStageBytes + quad * (4 * kOrthBox);
    const uint32_t m0 = t.mt * kBlockM + quad * 32;
#pragma unroll 1
    for (uint32_t c = 0; c < kChunks; ++c) {
      const uint32_t col = (rank * kChunks + c) * 32, n0 = t.nt * BN + col;
      if (n0 >= p.n || m0 >= p.m || (p.hermitian && n0 < m0)) continue;
      float re[32], im[32];
      read_chunk<BN>(taddr + col, p.conj_b != 0, re, im);
#pragma unroll 1
      for (uint32_t i = 0; i + 1 < SPLIT; ++i) {
        const uint32_t from_re = recv(i, 0, c), from_im = recv(i, 1, c);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t off = (j ^ (lane & 7)) << 4;
          uint32_t x[4], y[4];
          ld_shared_v4(from_re + off, x[0], x[1], x[2], x[3]);
          ld_shared_v4(from_im + off, y[0], y[1], y[2], y[3]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            re[4 * j + e] += __uint_as_float(x[e]);
            im[4 * j + e] += __uint_as_float(y[e]);
          }
        }
      }
      orth_store(p, &tm_c, staging, lane, t.b, m0, n0, re, im);
    }
    if (lane == 0) bulk_wait_group<0>();
  }
  __syncwarp();

  // ------------------------------------------------------------------ tear-down
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

using OrthFn = void (*)(const CUtensorMap, const CUtensorMap, const CUtensorMap, const OrthParams);

template <int BN, bool A_MN, bool B_MN> OrthFn orth_kernel(int split) {
  if constexpr (BN == 128) {
    if (split == 4) return orth_split_kernel<BN, A_MN, B_MN, 4>;
  }
  return split == 2 ? orth_split_kernel<BN, A_MN, B_MN, 2> : orth_product_kernel<BN, A_MN, B_MN>;
}
template <int BN> OrthFn orth_kernel(int split, bool a_mn, bool b_mn) {
  return a_mn   ? orth_kernel<BN, true, true>(split)
         : b_mn ? orth_kernel<BN, false, true>(split)
                : orth_kernel<BN, false, false>(split);
}
OrthFn orth_kernel(int bn, int split, bool a_mn, bool b_mn) {
  return bn == 128 ? orth_kernel<128>(split, a_mn, b_mn) : orth_kernel<64>(split, a_mn, b_mn);
}
int orth_smem(int bn) { return bn == 128 ? OrthCfg<128>::kSmemBytes : OrthCfg<64>::kSmemBytes; }

// Tiles of one product: the width, and how many CTAs share the K of a tile.
struct ProductShape {
  int bn, split;
  size_t per_batch;
  double clocks;  // estimated
};

// Estimated clocks: a block of K (of three passes) costs what its bytes take through the SM's port to L2
// (64 KiB resp. 48 KiB, 128 resp. 64 columns), a tile its epilogue (of a Hermitian result 100 per column,
// else 60), an exchange of partial sums 60 per column.
ProductShape pick_shape(size_t batch, size_t m, size_t n, size_t k, bool hermitian, size_t sms) {
  ProductShape best{0, 1, 0, 0.0};
  double least = 0.0;
  const size_t k_blocks = kPasses * ceil_div<size_t>(k, kOrthK);
  const char *env = std::getenv("CCGLIB_B200_ORTH_SPLIT");  // 1, 2 or 4: by hand, where it fits
  const int forced = env != nullptr ? std::atoi(env) : 0;
  for (int bn : {128, 64}) {
    const size_t rows = ceil_div<size_t>(m, kBlockM), cols = ceil_div<size_t>(n, bn);
    size_t tiles = 0;
    for (size_t i = 0; i < rows; ++i) tiles += cols - (hermitian ? i * kBlockM / bn : 0);
    for (int split : {1, 2, 4}) {
      const size_t ctas = batch * tiles * split;
      // (clusters of four do not fill the processor groups: at most 32 of them run at once)
      if (split > 1 && (ctas > (split == 4 ? sms * 86 / 100 : sms) || k_blocks < static_cast<size_t>(split) || bn < 32 * split)) continue;
      const double blocks = static_cast<double>(ceil_div<size_t>(k_blocks, split));
      double cost = static_cast<double>(ceil_div(ctas, sms)) *
                        (blocks * (bn == 128 ? 1250.0 : 950.0) + (hermitian ? 100.0 : 60.0) * bn / split) +
                    (split > 1 ? 60.0 * bn : 0.0);
      const double clocks = cost;
      if (forced != 0 && split == forced) cost *= 1e-3;
      if (best.bn == 0 || cost < least) {
        best = {bn, split, tiles, clocks};
        least = cost;
      }
    }
  }
  return best;
}

// ---- norm and first iterate ---------------------------------------------------------------------

template <typename T> __device__ __forceinline__ float as_float(T v);
template <> __device__ __forceinline__ float as_float(float v) { return v; }
template <> __device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// Eight consecutive values from a 16-byte aligned address.
__device__ __forceinline__ void load8(const float *src, float (&v)[8]) {
  const float4 a = reinterpret_cast<const float4 *>(src)[0];
  const float4 b = reinterpret_cast<const float4 *>(src)[1];
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <typename T> __device__ __forceinline__ void load8(const T *src, float (&v)[8]) {
  const uint4 q = *reinterpret_cast<const uint4 *>(src);
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const T *h = reinterpret_cast<const T *>(&w[i]);
    v[2 * i] = as_float(h[0]);
    v[2 * i + 1] = as_float(h[1]);
  }
}

constexpr int kNormThreads = 256;
constexpr size_t kNormChunk = 16384;  // values one CTA adds up

// Sums of squares of kNormChunk values each.  Eight values at a time in float32, where that neither
// overflows nor vanishes (else in float64); these in float64.  Memory-bound: converting every value to
// float64 took four times as long.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kNormThreads)
norm_kernel(const T *in, double *sums, size_t values, size_t chunks, size_t items) {
  __shared__ double part[kNormThreads / 32];
  for (size_t item = blockIdx.x; item < items; item += gridDim.x) {
    const size_t b = item / chunks, c = item - b * chunks;
    const T *src = in + b * values;
    const size_t end = min(values, (c + 1) * kNormChunk);
    double sum = 0.0;
#pragma unroll 4
    for (size_t i = c * kNormChunk + threadIdx.x * 8; i < end; i += kNormThreads * 8) {
      float v[8];
      if constexpr (VEC) {  // `values` is a multiple of eight
        load8(src + i, v);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = i + j < end ? as_float(src[i + j]) : 0.0f;
      }
      float s = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) s = fmaf(v[j], v[j], s);
      if (s > 1e-24f && s < 1e38f) {
        sum += s;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += static_cast<double>(v[j]) * v[j];
      }
    }
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
      double all = 0.0;
      for (int w = 0; w < kNormThreads / 32; ++w) all += part[w];
      sums[item] = all;
    }
    __syncthreads();
  }
}

struct FirstParams {
  const void *in;      // the caller's matrices, rows x cols
  const double *sums;  // [batch][chunks]
  size_t chunks, batch, rows, cols;
  __half *x;           // [batch][high Re, Im, low Re, Im][rows][pitch], zeros behind cols
  size_t pitch;
  float scale;
};

constexpr size_t kFirstChunk = 8192;  // complex values (padded rows) one CTA converts

// x -> its float16 and what the rounding leaves.
__device__ __forceinline__ void split_pair(float v0, float v1, __half2 &high, __half2 &low) {
  high = __floats2half2_rn(v0, v1);
  const float2 h = __half22float2(high);
  low = __floats2half2_rn(v0 - h.x, v1 - h.y);
}

// X0 = scale * input / norm.  VEC: rows need no padding, the planes are converted as they lie.
template <typename T, bool IL, bool VEC>
__global__ void __launch_bounds__(256) first_kernel(const FirstParams p) {
  __shared__ double part[256 / 32];
  const size_t plane = p.rows * p.pitch, per_batch = ceil_div<size_t>(plane, kFirstChunk);
  const size_t items = p.batch * per_batch;
  for (size_t item = blockIdx.x; item < items; item += gridDim.x) {
    const size_t b = item / per_batch;
    double sum = 0.0;
    for (size_t i = threadIdx.x; i < p.chunks; i += 256) sum += p.sums[b * p.chunks + i];
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
    __syncthreads();
    sum = 0.0;
    for (int w = 0; w < 256 / 32; ++w) sum += part[w];
    // A zero matrix stays zero (and one with a NaN becomes NaN).  A factor outside float32's comfortable
    // range is applied in two steps that are inside it: |x| * factor is at most scale.
    const double factor = sum == 0.0 ? 0.0 : static_cast<double>(p.scale) / sqrt(sum);
    const double half = factor < 1e-30 ? 1e-25 : factor > 1e30 ? 1e25 : 1.0;
    const float f0 = static_cast<float>(half), f1 = static_cast<float>(factor / half);
    const T *in = static_cast<const T *>(p.in) + b * 2 * p.rows * p.cols;
    __half *x = p.x + b * 4 * plane;
    const size_t first = (item - b * per_batch) * kFirstChunk;
    const size_t end = min(plane, first + kFirstChunk);
    if constexpr (VEC) {
#pragma unroll 4
      for (size_t i = first + threadIdx.x * 8; i < end; i += 256 * 8) {
        float v[2][8];
        load8(IL ? in + 2 * i : in + i, v[0]);
        load8(IL ? in + 2 * i + 8 : in + i + plane, v[1]);
        __half2 re[4], im[4], re_low[4], im_low[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          // interleaved: pairs 2j, 2j + 1 of the 16 values
          const float r0 = IL ? v[j / 2][(4 * j) & 7] : v[0][2 * j];
          const float i0 = IL ? v[j / 2][(4 * j + 1) & 7] : v[1][2 * j];
          const float r1 = IL ? v[j / 2][(4 * j + 2) & 7] : v[0][2 * j + 1];
          const float i1 = IL ? v[j / 2][(4 * j + 3) & 7] : v[1][2 * j + 1];
          split_pair(r0 * f0 * f1, r1 * f0 * f1, re[j], re_low[j]);
          split_pair(i0 * f0 * f1, i1 * f0 * f1, im[j], im_low[j]);
        }
        *reinterpret_cast<uint4 *>(x + i) = *reinterpret_cast<const uint4 *>(re);
        *reinterpret_cast<uint4 *>(x + i + plane) = *reinterpret_cast<const uint4 *>(im);
        *reinterpret_cast<uint4 *>(x + i + 2 * plane) = *reinterpret_cast<const uint4 *>(re_low);
        *reinterpret_cast<uint4 *>(x + i + 3 * plane) = *reinterpret_cast<const uint4 *>(im_low);
      }
    } else {
#pragma unroll 4
      for (size_t i = first + threadIdx.x; i < end; i += 256) {
        const size_t r = i / p.pitch, c = i - r * p.pitch;
        float re = 0.0f, im = 0.0f;
        if (c < p.cols) {
          const size_t s = r * p.cols + c;
          re = as_float(IL ? in[2 * s] : in[s]);
          im = as_float(IL ? in[2 * s + 1] : in[s + p.rows * p.cols]);
        }
        __half2 high, low;
        split_pair(re * f0 * f1, im * f0 * f1, high, low);
        x[i] = __low2half(high);
        x[i + plane] = __high2half(high);
        x[i + 2 * plane] = __low2half(low);
        x[i + 3 * plane] = __high2half(low);
      }
    }
    __syncthreads();
  }
}

template <typename T>
void launch_first_form(const FirstParams &p, bool il, bool vec, unsigned grid, cudaStream_t stream) {
  if (il) {
    if (vec) {
      first_kernel<T, true, true><<<grid, 256, 0, stream>>>(p);
    } else {
      first_kernel<T, true, false><<<grid, 256, 0, stream>>>(p);
    }
  } else if (vec) {
    first_kernel<T, false, true><<<grid, 256, 0, stream>>>(p);
  } else {
    first_kernel<T, false, false><<<grid, 256, 0, stream>>>(p);
  }
}

// ---- small matrices: the whole iteration in one launch ---------------------------------------------
//
// X, S and P in shared memory, float32 throughout: for matrices whose products are too small for
// 128-row tiles and a launch each.  X is kept transposed, V[l][i]: with S and P Hermitian, every product
// then reads rows of neighbouring values,
//   S_ij = sum_l V[l][i] conj(V[l][j]),  (S S)_ij = sum_k conj(S[k][i]) S[k][j],
//   V'[l][i] = a V[l][i] + sum_j conj(P[j][i]) V[l][j].
// A cluster of up to eight CTAs shares a matrix by rows of V where one CTA cannot hold it or SMs would
// stay idle: each adds up its rows' share of S, the shares go to all through distributed shared memory
// and are added in the order of the CTAs, and P is computed by each for itself.

constexpr int kSmallThreads = 512;
constexpr int kSmallRows = 2;  // rows of V' per thread in the update
constexpr size_t kSmallMaxSide = 64;
constexpr uint32_t kSmallMaxParts = 8;
constexpr int kSmallSmem = kMaxSmem - 2048;  // dynamic; the rest is static

struct SmallParams {
  const void *in;
  void *out;
  size_t batch, m, n;  // as the caller holds them
  uint32_t s, l, sp;   // short and long side, short side rounded up to four
  uint32_t parts;      // CTAs per matrix (the cluster)
  bool tall;
  int type_in, bf16, inter, steps;
  float a, b, c;
};

// V's share, S, P, and the others' shares of S (twice: one set is read while the next may arrive).
size_t small_smem(size_t s, size_t l, size_t parts) {
  const size_t sp = ceil_div<size_t>(s, 4) * 4;
  return (2 * ceil_div(l, parts) * sp + 2 * 2 * sp * sp + 2 * (parts - 1) * 2 * sp * sp) * sizeof(float);
}

// Four rows' worth of complex values.
struct Quad {
  float re[4], im[4];
};
__device__ __forceinline__ Quad load_quad(const float *re, const float *im) {
  const float4 r = *reinterpret_cast<const float4 *>(re), i = *reinterpret_cast<const float4 *>(im);
  return {{r.x, r.y, r.z, r.w}, {i.x, i.y, i.z, i.w}};
}
__device__ __forceinline__ void store_quad(float *re, float *im, const Quad &q) {
  *reinterpret_cast<float4 *>(re) = make_float4(q.re[0], q.re[1], q.re[2], q.re[3]);
  *reinterpret_cast<float4 *>(im) = make_float4(q.im[0], q.im[1], q.im[2], q.im[3]);
}

// H_ij = sum_k conj(v[k][i]) v[k][j] for all i <= j (Hermitian), `rows` rows of sp values; each 2 x 2 block
// on or above the diagonal by `lanes` neighbouring threads that deal out k.  store(i, j, H_ij) for
// i <= j.  (Larger blocks load less, but the unrolled sums of k over lanes made the step as long as its
// code: instructions arrive no faster than a few clocks each when they run once.)
template <typename Store>
__device__ __forceinline__ void gram_blocks(const float *re, const float *im, uint32_t rows, uint32_t sp,
                                            uint32_t lanes, const uint16_t *blocks, Store store) {
  const uint32_t pairs = (sp / 2) * (sp / 2 + 1) / 2;
  const uint32_t sub = threadIdx.x % lanes, per_turn = kSmallThreads / lanes;
  // a warp goes on while any of its groups has a block: the shuffles need all of them
  const uint32_t warp_first = (threadIdx.x & ~31u) / lanes;
#pragma unroll 1
  for (uint32_t turn = 0; turn + warp_first < pairs; turn += per_turn) {
    const uint32_t pair = turn + threadIdx.x / lanes;
    const bool on = pair < pairs;
    const uint32_t block = blocks[on ? pair : 0], bi = block >> 8, bj = block & 255;
    float h[2][2][2] = {};
#pragma unroll 4
    for (uint32_t k = sub; k < rows; k += lanes) {
      const float2 ur = *reinterpret_cast<const float2 *>(re + k * sp + 2 * bi);
      const float2 ui = *reinterpret_cast<const float2 *>(im + k * sp + 2 * bi);
      const float2 vr = *reinterpret_cast<const float2 *>(re + k * sp + 2 * bj);
      const float2 vi = *reinterpret_cast<const float2 *>(im + k * sp + 2 * bj);
      const float u[2][2] = {{ur.x, ui.x}, {ur.y, ui.y}}, v[2][2] = {{vr.x, vi.x}, {vr.y, vi.y}};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          h[i][j][0] = fmaf(u[i][0], v[j][0], fmaf(u[i][1], v[j][1], h[i][j][0]));
          h[i][j][1] = fmaf(u[i][0], v[j][1], fmaf(-u[i][1], v[j][0], h[i][j][1]));
        }
      }
    }
#pragma unroll 1
    for (uint32_t o = lanes / 2; o > 0; o >>= 1) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float &x = (&h[0][0][0])[i];
        x += __shfl_xor_sync(0xFFFFFFFFu, x, o);
      }
    }
    if (on && sub == 0) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (2 * bi + i <= 2 * bj + j) store(2 * bi + i, 2 * bj + j, h[i][j][0], h[i][j][1]);
        }
      }
    }
  }
}

__device__ __forceinline__ float load_value(const void *in, size_t i, int type) {
  return type == CCGLIB_B200_FLOAT32   ? static_cast<const float *>(in)[i]
         : type == CCGLIB_B200_FLOAT16 ? __half2float(static_cast<const __half *>(in)[i])
                                       : __bfloat162float(static_cast<const __nv_bfloat16 *>(in)[i]);
}

// Threads per block: all there are, but at least four k for each.
__device__ __forceinline__ uint32_t lanes_for(uint32_t pairs, uint32_t rows) {
  uint32_t lanes = 1;
  while (lanes < 32 && lanes * 2 * pairs <= kSmallThreads && lanes * 8 <= rows) lanes *= 2;
  return lanes;
}

__device__ __forceinline__ void st_shared_cluster_f64(uint32_t addr_cluster, double v) {
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(addr_cluster), "d"(v) : "memory");
}

__global__ void __launch_bounds__(kSmallThreads) small_kernel(const SmallParams p) {
  extern __shared__ __align__(16) float small_smem_raw[];
  __shared__ double part[kSmallThreads / 32];
  __shared__ double squares[kSmallMaxParts];  // sums of squares of the cluster's CTAs
  // the 2 x 2 blocks on and above the diagonal, row by row: (row << 8) + column
  __shared__ uint16_t blocks[(kSmallMaxSide / 2) * (kSmallMaxSide / 2 + 1) / 2];
  const uint32_t parts = p.parts, rank = parts > 1 ? cluster_ctarank() : 0;
  // this CTA's rows of V
  const uint32_t l_first = static_cast<uint32_t>(static_cast<uint64_t>(p.l) * rank / parts);
  const uint32_t sp = p.sp, l = static_cast<uint32_t>(static_cast<uint64_t>(p.l) * (rank + 1) / parts) - l_first;
  const uint32_t square = sp * sp;
  float *x_re = small_smem_raw, *x_im = x_re + l * sp;
  float *s_re = small_smem_raw + 2 * ceil_div(p.l, parts) * sp, *s_im = s_re + square;
  float *p_re = s_im + square, *p_im = p_re + square;
  float *others = p_im + square;  // [2][parts - 1][2][sp][sp]
  const uint32_t nb = sp / 4, pairs = (sp / 2) * (sp / 2 + 1) / 2;
  const uint32_t lanes_l = lanes_for(pairs, l), lanes_s = lanes_for(pairs, sp);
  for (uint32_t i = threadIdx.x; i < sp / 2; i += kSmallThreads) {
    uint32_t at_block = i * (sp / 2) - i * (i - 1) / 2;
    for (uint32_t j = i; j < sp / 2; ++j) blocks[at_block++] = static_cast<uint16_t>(i << 8 | j);
  }
  // the update deals (row group, column group) pairs to the threads, whole row groups at a time
  const uint32_t groups = kSmallThreads / nb, row_0 = threadIdx.x / nb, i0 = threadIdx.x % nb * 4;
  const size_t plane = p.m * p.n;
  uint32_t turn = 0;  // which set of shares the next exchange uses
  __syncwarp();
  if (parts > 1) cluster_sync();  // the others have started
  for (size_t b = blockIdx.x / parts; b < p.batch; b += gridDim.x / parts) {
    // X and its norm (float64: no input overflows or vanishes in it)
    double sum = 0.0;
    for (uint32_t i = threadIdx.x; i < l * sp; i += kSmallThreads) {
      const uint32_t r = i / sp, col = i - r * sp, row = l_first + r;  // V[row][col]
      float re = 0.0f, im = 0.0f;
      if (col < p.s) {
        const size_t e = p.tall ? static_cast<size_t>(row) * p.n + col : static_cast<size_t>(col) * p.n + row;
        const size_t base = b * 2 * plane;
        re = load_value(p.in, base + (p.inter ? 2 * e : e), p.type_in);
        im = load_value(p.in, base + (p.inter ? 2 * e + 1 : e + plane), p.type_in);
      }
      x_re[i] = re;
      x_im[i] = im;
      sum += static_cast<double>(re) * re + static_cast<double>(im) * im;
    }
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
    __syncthreads();
    sum = 0.0;
    for (int w = 0; w < kSmallThreads / 32; ++w) sum += part[w];
    if (parts > 1) {
      if (threadIdx.x < parts) {
        st_shared_cluster_f64(map_to_cta(smem_u32(&squares[rank]), threadIdx.x), sum);
      }
      __syncwarp();
      cluster_sync();
      sum = 0.0;
      for (uint32_t i = 0; i < parts; ++i) sum += squares[i];
    }
    const double factor = sum == 0.0 ? 0.0 : 1.0 / sqrt(sum);
    for (uint32_t i = threadIdx.x; i < l * sp; i += kSmallThreads) {
      x_re[i] = static_cast<float>(x_re[i] * factor);
      x_im[i] = static_cast<float>(x_im[i] * factor);
    }
    __syncthreads();
    for (int step = 0; step < p.steps; ++step) {
      gram_blocks(x_re, x_im, l, sp, lanes_l, blocks, [&](uint32_t i, uint32_t j, float re, float im) {
        // S_ij = conj(H_ij)
        const uint32_t ij = i * sp + j, ji = j * sp + i;
        im = i == j ? 0.0f : im;
        s_re[ij] = re;
        s_im[ij] = -im;
        s_re[ji] = re;
        s_im[ji] = im;
      });
      __syncthreads();
      if (parts > 1) {
        // A share goes to place `rank` (less one behind the receiver's own) of the set of this turn.  The
        // set is free: whoever read it last turn but one has been at last turn's barrier since.
        float *set = others + static_cast<size_t>(turn) * (parts - 1) * 2 * square;
        for (uint32_t peer = 0; peer < parts; ++peer) {
          if (peer == rank) continue;
          const uint32_t to = map_to_cta(smem_u32(set + (rank - (rank > peer ? 1 : 0)) * 2 * square), peer);
          for (uint32_t i = threadIdx.x * 4; i < 2 * square; i += kSmallThreads * 4) {
            const float4 v = *reinterpret_cast<const float4 *>(s_re + i);
            st_shared_cluster_v4(to + i * 4, __float_as_uint(v.x), __float_as_uint(v.y),
                                 __float_as_uint(v.z), __float_as_uint(v.w));
          }
        }
        __syncwarp();
        cluster_sync();
        for (uint32_t i = threadIdx.x; i < 2 * square; i += kSmallThreads) {
          float all = 0.0f;
          for (uint32_t r = 0; r < parts; ++r) {
            all += r == rank ? s_re[i] : set[(r - (r > rank ? 1 : 0)) * 2 * square + i];
          }
          s_re[i] = all;
        }
        turn ^= 1;
        __syncthreads();
      }
      gram_blocks(s_re, s_im, sp, sp, lanes_s, blocks, [&](uint32_t i, uint32_t j, float re, float im) {
        const uint32_t ij = i * sp + j, ji = j * sp + i;
        re = p.b * s_re[ij] + p.c * re;
        im = i == j ? 0.0f : p.b * s_im[ij] + p.c * im;
        p_re[ij] = re;
        p_im[ij] = im;
        p_re[ji] = re;
        p_im[ji] = -im;
      });
      __syncthreads();
      // kSmallRows rows of V' x four columns per thread; a pass reads its rows before any is written
      const uint32_t lb = ceil_div<uint32_t>(l, kSmallRows);
      for (uint32_t first = 0; first < lb; first += groups) {
        const uint32_t l0 = (first + row_0) * kSmallRows;
        const bool on = row_0 < groups && l0 < l;
        float vr[kSmallRows][4], vi[kSmallRows][4];
        if (on) {
#pragma unroll
          for (int r = 0; r < kSmallRows; ++r) {
            const uint32_t at = min(l0 + r, l - 1) * sp + i0;
            const Quad q = load_quad(x_re + at, x_im + at);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              vr[r][i] = p.a * q.re[i];
              vi[r][i] = p.a * q.im[i];
            }
          }
#pragma unroll 1
          for (uint32_t j = 0; j < sp; j += 4) {
            Quad x[kSmallRows];
#pragma unroll
            for (int r = 0; r < kSmallRows; ++r) {
              const uint32_t from = min(l0 + r, l - 1) * sp + j;
              x[r] = load_quad(x_re + from, x_im + from);
            }
#pragma unroll
            for (int jj = 0; jj < 4; ++jj) {
              const Quad q = load_quad(p_re + (j + jj) * sp + i0, p_im + (j + jj) * sp + i0);
#pragma unroll
              for (int r = 0; r < kSmallRows; ++r) {
                const float cr = x[r].re[jj], ci = x[r].im[jj];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  vr[r][i] = fmaf(q.re[i], cr, fmaf(q.im[i], ci, vr[r][i]));
                  vi[r][i] = fmaf(q.re[i], ci, fmaf(-q.im[i], cr, vi[r][i]));
                }
              }
            }
          }
        }
        __syncthreads();
        if (on) {
#pragma unroll
          for (int r = 0; r < kSmallRows; ++r) {
            if (l0 + r < l) {
              Quad q;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                q.re[i] = vr[r][i];
                q.im[i] = vi[r][i];
              }
              store_quad(x_re + (l0 + r) * sp + i0, x_im + (l0 + r) * sp + i0, q);
            }
          }
        }
      }
      __syncthreads();
    }
    // every CTA of the cluster has read the input: d_out may be d_in
    uint16_t *out = static_cast<uint16_t *>(p.out) + b * 2 * plane;
    for (uint32_t e = threadIdx.x; e < l * p.s; e += kSmallThreads) {
      // along the rows of the output
      const uint32_t row = p.tall ? e / p.s : e % l, col = p.tall ? e - row * p.s : e / l;  // V[row][col]
      const size_t to = p.tall ? static_cast<size_t>(l_first + row) * p.n + col
                               : static_cast<size_t>(col) * p.n + l_first + row;
      out[to] = round_half(x_re[row * sp + col], p.bf16);
      out[to + plane] = round_half(x_im[row * sp + col], p.bf16);
    }
    __syncthreads();
  }
}

} // namespace
} // namespace ccglib_b200

using namespace ccglib_b200;

// How P = a I + b S + c S^2 is computed:
//   kSquare   c (S + h I)^2 + (a - c h^2) I with h = b / 2c, one Hermitian square of what the Gram product
//             stores (h on its diagonal);
//   kLinear   c = 0: the Gram product stores it;
//   kProduct  (c S + b I) S + a I, the Gram product computed twice, for b so much larger than c that the
//             square would cancel: c h^2 more than eight times the largest coefficient.
enum PolyForm { kSquare, kLinear, kProduct };

struct ccglib_b200_orthogonalize_plan {
  ccglib_b200_orthogonalize_desc desc;
  size_t n, l;          // short and long side
  size_t n_p, cols_p;   // row pitches of S and P, and of X: multiples of eight
  bool tall;            // m > n
  PolyForm form;
  float shift;          // kSquare: b / 2c
  float scale, s_scale, t_scale, p_scale;  // powers of two that X, S (+ shift I), T and P are kept times
  ProductShape gram, poly, update;
  uint32_t small;       // > 0: the whole iteration in one launch, so many CTAs per matrix
  size_t chunks;
  int device, sms;
  long long wait_cycles;
  unsigned *status;
  void *scratch;
  size_t scratch_bytes;
  __half *x[2], *s, *t, *p;  // [batch][4][m][cols_p], [batch][4][n][n_p]: high Re, Im, low Re, Im
  double *sums;
  // tensor maps of the workspace: X as either operand of the Gram product and as the operand of the
  // update, T (or S) and S as the operands of their product, P as the operand of the update, and all as results
  CUtensorMap gram_a[2], gram_b[2], update_x[2], x_out[2], poly_a, poly_b, update_p, s_out, t_out, p_out;
};

namespace {

// One operand: planes of `rows` x `cols` (row pitch `pitch` values), contracted over its columns, or over
// its rows (by_rows).
struct Operand {
  const __half *data;
  size_t rows, cols, pitch;
  bool by_rows;
};

struct Product {
  Operand a, b;
  const CUtensorMap *tm_a, *tm_b, *tm_c;
  size_t m, n;  // n: columns written
  ProductShape shape;
  bool hermitian, conj;
  float alpha, diag;
  bool pair;
  // what the last product has of its own
  void *out = nullptr;
  size_t out_pitch = 0;
  bool boxes = true, bf16 = false;
};

// Map of an operand whose tile has `tile` rows of the result's.
int operand_map(CUtensorMap *tm, const Operand &o, size_t batch, int tile) {
  const uint32_t box = o.by_rows ? kOrthK : static_cast<uint32_t>(tile);
  return make_map(tm, o.data, o.cols * 2, o.rows, 4 * batch, o.pitch * 2, o.rows * o.pitch * 2, 128, box, 2);
}

// Map of a result: planes of rows x cols 16-bit values.
int result_map(CUtensorMap *tm, const void *out, size_t planes, size_t rows, size_t cols) {
  return make_map(tm, out, cols * 2, rows, planes, cols * 2, rows * cols * 2, 64, 32, 1);
}

// X as an operand: contracted over the long side in S, over the short side in the update.
Operand x_operand(const ccglib_b200_orthogonalize_plan &plan, int which, bool over_long) {
  return {plan.x[which], plan.desc.m, plan.cols_p, plan.cols_p, plan.tall == over_long};
}
Operand square_operand(const ccglib_b200_orthogonalize_plan &plan, const __half *data) {
  return {data, plan.n, plan.n_p, plan.n_p, false};
}

int make_maps(ccglib_b200_orthogonalize_plan &plan) {
  const size_t batch = plan.desc.batch, planes = 4 * batch;
  const Operand s = square_operand(plan, plan.s), t = square_operand(plan, plan.t),
                p = square_operand(plan, plan.p);
  int rc = operand_map(&plan.poly_a, t, batch, kBlockM);
  if (rc == CCGLIB_B200_OK) rc = operand_map(&plan.poly_b, s, batch, plan.poly.bn);
  if (rc == CCGLIB_B200_OK) rc = operand_map(&plan.update_p, p, batch, plan.tall ? plan.update.bn : kBlockM);
  if (rc == CCGLIB_B200_OK) rc = result_map(&plan.s_out, plan.s, planes, plan.n, plan.n_p);
  if (rc == CCGLIB_B200_OK) rc = result_map(&plan.t_out, plan.t, planes, plan.n, plan.n_p);
  if (rc == CCGLIB_B200_OK) rc = result_map(&plan.p_out, plan.p, planes, plan.n, plan.n_p);
  for (int i = 0; i < 2; ++i) {
    const Operand x_long = x_operand(plan, i, true), x_short = x_operand(plan, i, false);
    if (rc == CCGLIB_B200_OK) rc = operand_map(&plan.gram_a[i], x_long, batch, kBlockM);
    if (rc == CCGLIB_B200_OK) rc = operand_map(&plan.gram_b[i], x_long, batch, plan.gram.bn);
    if (rc == CCGLIB_B200_OK) {
      rc = operand_map(&plan.update_x[i], x_short, batch, plan.tall ? kBlockM : plan.update.bn);
    }
    if (rc == CCGLIB_B200_OK) rc = result_map(&plan.x_out[i], plan.x[i], planes, plan.desc.m, plan.cols_p);
  }
  return rc;
}

int launch_product(const ccglib_b200_orthogonalize_plan &plan, const Product &q, cudaStream_t stream) {
  const size_t batch = plan.desc.batch;
  OrthParams g{};
  g.m = static_cast<uint32_t>(q.m);
  g.n = static_cast<uint32_t>(q.n);
  g.k_blocks = static_cast<uint32_t>(ceil_div<size_t>(q.a.by_rows ? q.a.rows : q.a.cols, kOrthK));
  g.tiles_m = static_cast<uint32_t>(ceil_div<size_t>(q.m, kBlockM));
  g.tiles_n = static_cast<uint32_t>(ceil_div<size_t>(q.n, q.shape.bn));
  g.group_n = g.tiles_m <= 2 ? 4 : 8;
  g.per_batch = static_cast<uint32_t>(q.shape.per_batch);
  g.num_tiles = static_cast<uint32_t>(batch * q.shape.per_batch);
  g.hermitian = q.hermitian ? 1u : 0u;
  g.conj_b = q.conj ? 1u : 0u;
  g.alpha = q.alpha;
  g.diag = q.diag;
  g.pair = q.pair ? 1u : 0u;
  g.bf16 = q.bf16 ? 1u : 0u;
  g.boxes = q.boxes ? 1u : 0u;
  g.out = static_cast<uint16_t *>(q.out);
  g.n_out = static_cast<uint32_t>(q.out_pitch);
  g.status = plan.status;
  g.wait_cycles = plan.wait_cycles;
  // a block takes about a thousand clocks: K of 1e8 values would come near the default limit by itself
  g.tile_cycles = plan.wait_cycles + 8192ll * kPasses * g.k_blocks;
  unsigned grid = g.num_tiles < static_cast<uint32_t>(plan.sms) ? g.num_tiles : plan.sms;
  if (q.shape.split > 1) grid = g.num_tiles * q.shape.split;  // one cluster per tile
  CCGLIB_CUDA_TRY(launch_programmatic(
      orth_kernel(q.shape.bn, q.shape.split, q.a.by_rows, q.b.by_rows), grid, kThreads,
      orth_smem(q.shape.bn), q.shape.split, stream, *q.tm_a, *q.tm_b, *q.tm_c, g));
  return CCGLIB_B200_OK;
}

template <typename T>
int launch_first(const ccglib_b200_orthogonalize_plan &plan, const void *d_in, cudaStream_t stream) {
  const ccglib_b200_orthogonalize_desc &d = plan.desc;
  const size_t cap = static_cast<size_t>(plan.sms) * 8;
  size_t items = d.batch * plan.chunks;
  unsigned grid = static_cast<unsigned>(items < cap ? items : cap);
  const T *in = static_cast<const T *>(d_in);
  if (aligned16(d_in) && 2 * d.m * d.n % 8 == 0) {
    norm_kernel<T, true><<<grid, kNormThreads, 0, stream>>>(in, plan.sums, 2 * d.m * d.n, plan.chunks, items);
  } else {
    norm_kernel<T, false><<<grid, kNormThreads, 0, stream>>>(in, plan.sums, 2 * d.m * d.n, plan.chunks, items);
  }
  CCGLIB_CUDA_TRY(cudaGetLastError());
  FirstParams p{};
  p.in = d_in;
  p.sums = plan.sums;
  p.chunks = plan.chunks;
  p.batch = d.batch;
  p.rows = d.m;
  p.cols = d.n;
  p.x = plan.x[0];
  p.pitch = plan.cols_p;
  p.scale = plan.scale;
  items = d.batch * ceil_div<size_t>(d.m * plan.cols_p, kFirstChunk);
  grid = static_cast<unsigned>(items < cap ? items : cap);
  launch_first_form<T>(p, d.input_complex_axis == CCGLIB_B200_INTERLEAVED,
                       d.n % 8 == 0 && aligned16(d_in), grid, stream);
  CCGLIB_CUDA_TRY(cudaGetLastError());
  return CCGLIB_B200_OK;
}

// 2^e, |e| at most 14, that takes `bound` to 2^13 .. 2^14 (to 2^14 at most where it is large).
float scale_for(double bound) {
  if (!(bound > 0.0)) return 1.0f;
  const double e = std::floor(14.0 - std::log2(bound));
  return static_cast<float>(std::exp2(e > 14.0 ? 14.0 : e < -14.0 ? -14.0 : e));
}

// Powers of two that keep the iterates inside float16 and as far from its smallest values as that allows: no
// entry of a matrix exceeds its largest singular value, and the largest in any step follows from the map
// (1.0001 and 1.1: what the points miss and rounding adds).
void choose_scales(ccglib_b200_orthogonalize_plan &plan) {
  const double a = plan.desc.a, b = plan.desc.b, c = plan.desc.c;
  constexpr int kPoints = 512;
  double top = 1.0, most = 1.0;
  for (int step = 0; step < plan.desc.steps && most < 1e6; ++step) {
    double next = 0.0;
    for (int i = 1; i <= kPoints; ++i) {
      const double v = top * i / kPoints, q = v * v;
      next = std::fmax(next, std::fabs(v * (a + b * q + c * q * q)));
    }
    top = 1.0001 * next;
    most = std::fmax(most, top);
  }
  plan.form = c == 0.0 ? kLinear : kSquare;
  if (plan.form == kSquare) {
    plan.shift = static_cast<float>(b / (2.0 * c));
    const double largest = std::fmax(std::fabs(a), std::fmax(std::fabs(b), std::fabs(c)));
    // (the negation catches an infinite quotient too)
    if (!(std::fabs(c) * plan.shift * plan.shift <= 8.0 * largest)) plan.form = kProduct;
  }
  if (plan.form != kSquare) plan.shift = 0.0f;
  double s = 0.0, t = 0.0, p = 0.0;
  for (int i = 0; i <= kPoints; ++i) {
    const double q = most * most * i / kPoints;
    s = std::fmax(s, std::fabs(q + plan.shift));
    t = std::fmax(t, std::fabs(b + c * q));
    p = std::fmax(p, std::fabs(a + b * q + c * q * q));
  }
  plan.s_scale = scale_for(1.1 * s);
  plan.t_scale = scale_for(1.1 * t);
  plan.p_scale = scale_for(1.1 * p);
  plan.scale = scale_for(1.1 * most);
}

} // namespace

extern "C" int ccglib_b200_orthogonalize_plan_create(const ccglib_b200_orthogonalize_desc *desc,
                                                     ccglib_b200_orthogonalize_plan **out) {
  if (desc == nullptr || out == nullptr) {
    set_last_error("orthogonalize_plan_create: null argument");
    return CCGLIB_B200_INVALID_ARGUMENT;
  }
  *out = nullptr;
  const ccglib_b200_orthogonalize_desc &d = *desc;
  if (d.batch == 0 || d.m == 0 || d.n == 0) {
    set_last_error("orthogonalize_plan_create: batch, M and N must be positive");
    return CCGLIB_B200_INVALID_ARGUMENT;
  }
  if (d.m > 0x0FFFFFFFull || d.n > 0x0FFFFFFFull || d.batch > 0x3FFFFFFFull ||
      d.batch > (size_t{1} << 52) / (d.m * d.n)) {
    set_last_error("orthogonalize_plan_create: dimension too large");
    return CCGLIB_B200_INVALID_ARGUMENT;
  }
  if (d.type_in != CCGLIB_B200_FLOAT16 && d.type_in != CCGLIB_B200_BFLOAT16 &&
      d.type_in != CCGLIB_B200_FLOAT32) {
    set_last_error("orthogonalize_plan_create: input must be float16, bfloat16 or float32 (got %d)",
                   d.type_in);
    return CCGLIB_B200_UNSUPPORTED;
  }
  if (d.type_out != CCGLIB_B200_FLOAT16 && d.type_out != CCGLIB_B200_BFLOAT16) {
    set_last_error("orthogonalize_plan_create: output must be float16 or bfloat16 (got %d)", d.type_out);
    return CCGLIB_B200_UNSUPPORTED;
  }
  if (d.input_complex_axis != CCGLIB_B200_PLANAR &&
      d.input_complex_axis != CCGLIB_B200_INTERLEAVED) {
    set_last_error("orthogonalize_plan_create: unknown complex axis location %d", d.input_complex_axis);
    return CCGLIB_B200_INVALID_ARGUMENT;
  }
  if (d.steps < 1 || d.steps > 1000) {
    set_last_error("orthogonalize_plan_create: steps must be 1 .. 1000 (got %d)", d.steps);
    return CCGLIB_B200_INVALID_ARGUMENT;
  }
  if (!std::isfinite(d.a) || !std::isfinite(d.b) || !std::isfinite(d.c)) {
    set_last_error("orthogonalize_plan_create: coefficients must be finite");
    return CCGLIB_B200_INVALID_ARGUMENT;
  }
  ccglib_b200_orthogonalize_plan plan{};
  plan.desc = d;
  plan.tall = d.m > d.n;
  plan.n = plan.tall ? d.n : d.m;
  plan.l = plan.tall ? d.m : d.n;
  plan.n_p = ceil_div<size_t>(plan.n, 8) * 8;
  plan.cols_p = ceil_div<size_t>(d.n, 8) * 8;
  choose_scales(plan);
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
  int rc = device_status_address(&plan.status);
  if (rc != CCGLIB_B200_OK) return rc;
  plan.gram = pick_shape(d.batch, plan.n, plan.n_p, plan.l, true, plan.sms);
  plan.poly = pick_shape(d.batch, plan.n, plan.n_p, plan.n, true, plan.sms);
  plan.update = pick_shape(d.batch, d.m, plan.cols_p, plan.n, false, plan.sms);
  // One launch (with how many CTAs per matrix), or three launches per step?  Estimates in microseconds
  // per step.  On short sides 1 .. 64, long sides 1 .. 4000 and batches 1, 64 and 1024 the choice is within
  // 26 % of the best form, in nine of ten cases within 6 % (33 x 400 x 64, five steps: 128 us in one launch,
  // 188 in three; 64 x 64: 155 and 136).
  const size_t sms = static_cast<size_t>(plan.sms);
  double least = 3 * 1.5 + (plan.gram.clocks + plan.poly.clocks + plan.update.clocks) / 1900.0;
  // CCGLIB_B200_ORTH_SMALL: 0 for three launches, 1, 2, 4 or 8 for one with so many CTAs (where it fits)
  const char *env = std::getenv("CCGLIB_B200_ORTH_SMALL");
  const int forced = env != nullptr && *env != '\0' ? std::atoi(env) : -1;
  for (uint32_t parts = 1; parts <= kSmallMaxParts && plan.n <= kSmallMaxSide; parts *= 2) {
    if (small_smem(plan.n, plan.l, parts) > static_cast<size_t>(kSmallSmem) || parts > plan.l) continue;
    const double side = static_cast<double>(ceil_div<size_t>(plan.n, 4) * 4);
    const double macs = side * side * (2.0 * static_cast<double>(plan.l) / parts + side);
    // (clusters of four and eight leave some SMs of a processor group over)
    const size_t room = parts >= 4 ? sms * 86 / 100 : sms;
    const double turns = static_cast<double>(ceil_div(d.batch * parts, room));
    const double exchange = parts > 1 ? 0.5 + 0.1 * parts + 5e-4 * (parts - 1) * side * side : 0.0;
    double cost = turns * (1.5 + 4e-5 * macs + exchange);
    if (forced >= 0) cost = static_cast<int>(parts) == forced ? -1.0 : 1e30;
    if (cost < least) {
      least = cost;
      plan.small = parts;
    }
  }
  if (plan.small) {
    CCGLIB_CUDA_TRY(cudaFuncSetAttribute(reinterpret_cast<const void *>(small_kernel),
                                         cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         kSmallSmem));
    *out = new (std::nothrow) ccglib_b200_orthogonalize_plan(plan);
    if (*out == nullptr) {
      set_last_error("orthogonalize_plan_create: out of host memory");
      return CCGLIB_B200_OUT_OF_MEMORY;
    }
    return CCGLIB_B200_OK;
  }
  if (d.batch > 0x1FFFFFFFull) {  // 32-bit signed plane coordinates in the TMA unit
    set_last_error("orthogonalize_plan_create: dimension too large");
    return CCGLIB_B200_INVALID_ARGUMENT;
  }
  if (d.batch * plan.gram.per_batch > 0x7FFFFFFFull ||
      d.batch * plan.poly.per_batch > 0x7FFFFFFFull ||
      d.batch * plan.update.per_batch > 0x7FFFFFFFull) {
    set_last_error("orthogonalize_plan_create: too many tiles");
    return CCGLIB_B200_INVALID_ARGUMENT;
  }
  for (const ProductShape &shape : {plan.gram, plan.poly, plan.update}) {
    for (int form = 0; form < 3; ++form) {
      CCGLIB_CUDA_TRY(cudaFuncSetAttribute(
          reinterpret_cast<const void *>(orth_kernel(shape.bn, shape.split, form == 2, form >= 1)),
          cudaFuncAttributeMaxDynamicSharedMemorySize, orth_smem(shape.bn)));
    }
  }
  plan.chunks = ceil_div<size_t>(2 * d.m * d.n, kNormChunk);
  const size_t x_bytes = ceil_div<size_t>(d.batch * 4 * d.m * plan.cols_p * 2, 256) * 256;
  const size_t s_bytes = ceil_div<size_t>(d.batch * 4 * plan.n * plan.n_p * 2, 256) * 256;
  const size_t squares = plan.form == kSquare ? 2 : plan.form == kLinear ? 1 : 3;
  plan.scratch_bytes = 2 * x_bytes + squares * s_bytes + d.batch * plan.chunks * sizeof(double);
  if (cudaMalloc(&plan.scratch, plan.scratch_bytes) != cudaSuccess) {
    cudaGetLastError();
    set_last_error("orthogonalize_plan_create: could not allocate %zu bytes of workspace",
                   plan.scratch_bytes);
    return CCGLIB_B200_OUT_OF_MEMORY;
  }
  char *at = static_cast<char *>(plan.scratch);
  auto take = [&](size_t bytes) {
    char *here = at;
    at += bytes;
    return here;
  };
  plan.x[0] = reinterpret_cast<__half *>(take(x_bytes));
  plan.x[1] = reinterpret_cast<__half *>(take(x_bytes));
  // (what a form has no use for stands for the array that it is not)
  plan.p = reinterpret_cast<__half *>(take(s_bytes));
  plan.s = plan.form == kLinear ? plan.p : reinterpret_cast<__half *>(take(s_bytes));
  plan.t = plan.form == kProduct ? reinterpret_cast<__half *>(take(s_bytes)) : plan.s;
  plan.sums = reinterpret_cast<double *>(at);
  rc = make_maps(plan);
  if (rc != CCGLIB_B200_OK) {
    cudaFree(plan.scratch);
    return rc;
  }
  *out = new (std::nothrow) ccglib_b200_orthogonalize_plan(plan);
  if (*out == nullptr) {
    cudaFree(plan.scratch);
    set_last_error("orthogonalize_plan_create: out of host memory");
    return CCGLIB_B200_OUT_OF_MEMORY;
  }
  return CCGLIB_B200_OK;
}

extern "C" int ccglib_b200_orthogonalize_run(ccglib_b200_orthogonalize_plan *plan, const void *d_in,
                                             void *d_out, void *stream_v) {
  if (plan == nullptr || d_in == nullptr || d_out == nullptr) {
    set_last_error("orthogonalize_run: null argument");
    return CCGLIB_B200_INVALID_ARGUMENT;
  }
  const ccglib_b200_orthogonalize_desc &d = plan->desc;
  const size_t in_bytes = d.type_in == CCGLIB_B200_FLOAT32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(d_in) % in_bytes != 0 || reinterpret_cast<uintptr_t>(d_out) % 2 != 0) {
    set_last_error("orthogonalize_run: input and output must be aligned to their elements");
    return CCGLIB_B200_INVALID_ARGUMENT;
  }
  // One launch takes the matrices of a batch in any order, each from its input to its output: only the same
  // array in the same layout may be both.
  const size_t values = d.batch * 2 * d.m * d.n;
  const bool same = d_in == d_out && d.type_in == d.type_out && d.input_complex_axis == CCGLIB_B200_PLANAR;
  if (!same && overlap(d_in, values * in_bytes, d_out, values * 2)) {
    set_last_error("orthogonalize_run: input and output overlap (in place needs a planar input of the output's "
                   "type, and the same address)");
    return CCGLIB_B200_INVALID_ARGUMENT;
  }
  int device = -1;
  CCGLIB_CUDA_TRY(cudaGetDevice(&device));
  if (device != plan->device) {
    set_last_error("orthogonalize_run: the plan belongs to device %d, the current device is %d",
                   plan->device, device);
    return CCGLIB_B200_INVALID_ARGUMENT;
  }
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  if (plan->small) {
    SmallParams q{};
    q.in = d_in;
    q.out = d_out;
    q.batch = d.batch;
    q.m = d.m;
    q.n = d.n;
    q.s = static_cast<uint32_t>(plan->n);
    q.l = static_cast<uint32_t>(plan->l);
    q.sp = static_cast<uint32_t>(ceil_div<size_t>(plan->n, 4) * 4);
    q.tall = plan->tall;
    q.type_in = d.type_in;
    q.bf16 = d.type_out == CCGLIB_B200_BFLOAT16;
    q.inter = d.input_complex_axis == CCGLIB_B200_INTERLEAVED;
    q.steps = d.steps;
    q.a = d.a;
    q.b = d.b;
    q.c = d.c;
    q.parts = plan->small;
    const size_t cap = static_cast<size_t>(plan->sms) * 8;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>((d.batch < cap ? d.batch : cap) * plan->small));
    cfg.blockDim = dim3(kSmallThreads);
    cfg.dynamicSmemBytes = small_smem(plan->n, plan->l, plan->small);
    cfg.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = plan->small;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = plan->small > 1 ? 1 : 0;
    CCGLIB_CUDA_TRY(cudaLaunchKernelEx(&cfg, small_kernel, q));
    return CCGLIB_B200_OK;
  }
  int rc = d.type_in == CCGLIB_B200_FLOAT32   ? launch_first<float>(*plan, d_in, stream)
           : d.type_in == CCGLIB_B200_FLOAT16 ? launch_first<__half>(*plan, d_in, stream)
                                              : launch_first<__nv_bfloat16>(*plan, d_in, stream);
  const size_t n = plan->n, n_p = plan->n_p, cols_p = plan->cols_p;
  const bool tall = plan->tall;
  const float s_scale = plan->s_scale, t_scale = plan->t_scale, p_scale = plan->p_scale;
  for (int step = 0; rc == CCGLIB_B200_OK && step < d.steps; ++step) {
    const bool last = step + 1 == d.steps;
    const int now = step & 1;
    const Operand x_long = x_operand(*plan, now, true), x_short = x_operand(*plan, now, false);
    const Operand s = square_operand(*plan, plan->s), t = square_operand(*plan, plan->t),
                  p = square_operand(*plan, plan->p);
    // the Gram product X X^H as alpha S + diag I
    const auto gram = [&](const CUtensorMap *out, float alpha, float diag) {
      return launch_product(*plan, {x_long, x_long, &plan->gram_a[now], &plan->gram_b[now], out, n, n_p, plan->gram,
                                    true, true, alpha / (plan->scale * plan->scale), diag, true}, stream);
    };
    if (plan->form == kLinear) {
      rc = gram(&plan->p_out, p_scale * d.b, p_scale * d.a);
    } else {
      rc = gram(&plan->s_out, s_scale, s_scale * plan->shift);
      float alpha = p_scale / (s_scale * s_scale) * d.c;
      double diag = d.a - static_cast<double>(d.c) * plan->shift * plan->shift;
      if (rc == CCGLIB_B200_OK && plan->form == kProduct) {
        rc = gram(&plan->t_out, t_scale * d.c, t_scale * d.b);
        alpha = p_scale / (s_scale * t_scale);
        diag = d.a;
      }
      if (rc != CCGLIB_B200_OK) break;
      rc = launch_product(*plan, {t, s, &plan->poly_a, &plan->poly_b, &plan->p_out, n, n_p, plan->poly, true, true,
                                  alpha, static_cast<float>(p_scale * diag), true}, stream);
    }
    if (rc != CCGLIB_B200_OK) break;
    // X = P X
    const CUtensorMap *tm_x = &plan->update_x[now], *tm_p = &plan->update_p;
    Product update{tall ? x_short : p, tall ? p : x_short, tall ? tm_x : tm_p, tall ? tm_p : tm_x,
                   &plan->x_out[now ^ 1], d.m, cols_p, plan->update, false, false, 1.0f / p_scale, 0.0f, true};
    CUtensorMap tm_out;
    if (last) {
      update.alpha = 1.0f / (p_scale * plan->scale);
      update.pair = false;
      update.out = d_out;
      update.out_pitch = d.n;
      update.boxes = d.n % 8 == 0 && aligned16(d_out);
      update.bf16 = d.type_out == CCGLIB_B200_BFLOAT16;
      if (update.boxes) {
        rc = result_map(&tm_out, d_out, 2 * d.batch, d.m, d.n);
        if (rc != CCGLIB_B200_OK) break;
        update.tm_c = &tm_out;
      }
    }
    rc = launch_product(*plan, update, stream);
  }
  return rc;
}

extern "C" size_t ccglib_b200_orthogonalize_plan_scratch_bytes(
    const ccglib_b200_orthogonalize_plan *plan) {
  return plan != nullptr ? plan->scratch_bytes : 0;
}

extern "C" int ccglib_b200_orthogonalize_plan_destroy(ccglib_b200_orthogonalize_plan *plan) {
  if (plan == nullptr) return CCGLIB_B200_OK;
  if (plan->scratch != nullptr) cudaFree(plan->scratch);
  delete plan;
  return CCGLIB_B200_OK;
}
