// Block quantiser: float16 / bfloat16 / float32 complex matrices -> fp8 planes with one float32 scale
// per block, the operand form of the scaled GEMM (scaled_gemm.cu).
//
//   amax  = max(|re|, |im|) over the finite entries of the block
//   scale = max(amax / FMAX, 2^-126)         FMAX = 448 (e4m3), 57344 (e5m2)
//   q     = fp8_rne(x * (FMAX / amax))       every step a correctly rounded float32 operation
//
// (x * 2^126 where the scale is at its floor.)  FMAX / amax is one rounding away from the exact factor,
// 1 / scale would be two: with 16-bit input exact ties between two fp8 values are common, and after a second
// rounding they fall to either side.
//
// A block is 128 consecutive k of one row, or 128 x 128 (rows x k); re and im share the scale, so a
// phase survives.  The floor 2^-126 keeps the factor finite; a silent block gets it and quantises to
// zeros.  A NaN stays a NaN and an infinity becomes what the format has for it (e5m2: infinity,
// e4m3: NaN); neither enters amax, so one bad sample does not cost its block the other samples.
//
// Memory-bound: every input byte is read once, every output byte written once, the block lives in
// registers between its maximum and its rounding.  K contiguous, float32 interleaved 4 x 4096 x 16384:
// 445 to 467 us for 2.69 GB, 5.8 to 6.0 TB/s.  Rows contiguous, bfloat16 3 x 5003 x 4001: 111 us for
// 0.36 GB, 3.2 TB/s, bound by issuing and waiting for its loads, which are two bytes wide for planar 16-bit
// input of any size and alignment (a lane reads one row of one k).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <type_traits>

#include "common.cuh"

namespace ccglib_b200 {
namespace {

constexpr int kBlockK = 128;
constexpr float kMinScale = 1.17549435e-38f;  // 2^-126

struct QuantizeParams {
  const void *in;
  uint8_t *out;   // [batch][2][rows][pitch]
  float *scale;   // [batch][blocks_k][blocks_rows]
  size_t batch, rows, k, pitch;
  size_t blocks_k, blocks_rows;
  float im_sign;  // -1: the conjugate is written
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// Two elements held in one 32-bit word.
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t w);
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}

// |x| as bits, 0 for NaN and infinities (bit patterns of non-negative floats order like the values)
__device__ __forceinline__ uint32_t finite_abs_bits(float x) {
  const uint32_t u = __float_as_uint(x) & 0x7FFFFFFFu;
  return u < 0x7F800000u ? u : 0u;
}

template <bool E5M2> __device__ __forceinline__ float block_scale(uint32_t amax_bits) {
  const float s = __fdiv_rn(__uint_as_float(amax_bits), E5M2 ? 57344.0f : 448.0f);
  return fmaxf(s, kMinScale);
}

// What the values of a block with this maximum and scale are multiplied by.
template <bool E5M2> __device__ __forceinline__ float block_factor(uint32_t amax_bits, float scale) {
  return scale > kMinScale ? __fdiv_rn(E5M2 ? 57344.0f : 448.0f, __uint_as_float(amax_bits))
                           : 8.507059e37f;  // 2^126
}

// Four scaled values -> four fp8 bytes, first value in the low byte.  SPECIAL: the values may hold
// infinities, which the conversion would saturate (finite ones never exceed the format here).
template <bool E5M2, bool SPECIAL = false>
__device__ __forceinline__ uint32_t pack4(const float (&v)[4]) {
  constexpr __nv_fp8_interpretation_t kFmt = E5M2 ? __NV_E5M2 : __NV_E4M3;
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[0], v[1]), __NV_SATFINITE, kFmt);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[2], v[3]), __NV_SATFINITE, kFmt);
  uint32_t w = lo | (hi << 16);
  if constexpr (SPECIAL) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (fabsf(v[i]) == __uint_as_float(0x7F800000u)) {
        const uint32_t sign = v[i] < 0.0f ? 0x80u : 0u;
        w = (w & ~(0xFFu << (8 * i))) | ((sign | (E5M2 ? 0x7Cu : 0x7Fu)) << (8 * i));
      }
    }
  }
  return w;
}

// Four consecutive complex samples k0..k0+3 of row r of one batch item (K contiguous).  VEC: K is a
// multiple of four, so a quad is inside the row or outside it as a whole and its words are aligned;
// outside, an address inside stands in and the values are dropped, so that no load waits for a branch.
template <typename T, bool IL, bool VEC>
__device__ __forceinline__ void load_quad(const T *in, size_t rows, size_t k, size_t r, size_t k0,
                                          float (&re)[4], float (&im)[4]) {
  if constexpr (VEC) {
    const bool inside = r < rows && k0 < k;
    const size_t at = min(r, rows - 1) * k + (k0 < k ? k0 : 0);
    if constexpr (IL) {
      const T *src = in + at * 2;
      if constexpr (sizeof(T) == 4) {
        const float4 a = __ldcs(reinterpret_cast<const float4 *>(src));
        const float4 b = __ldcs(reinterpret_cast<const float4 *>(src) + 1);
        re[0] = a.x; im[0] = a.y; re[1] = a.z; im[1] = a.w;
        re[2] = b.x; im[2] = b.y; re[3] = b.z; im[3] = b.w;
      } else {
        const uint4 a = __ldcs(reinterpret_cast<const uint4 *>(src));
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 v = unpack2<T>(w[i]);
          re[i] = v.x;
          im[i] = v.y;
        }
      }
    } else {
      const T *s0 = in + at;
      const T *s1 = s0 + rows * k;
      if constexpr (sizeof(T) == 4) {
        const float4 a = __ldcs(reinterpret_cast<const float4 *>(s0));
        const float4 b = __ldcs(reinterpret_cast<const float4 *>(s1));
        re[0] = a.x; re[1] = a.y; re[2] = a.z; re[3] = a.w;
        im[0] = b.x; im[1] = b.y; im[2] = b.z; im[3] = b.w;
      } else {
        const uint2 a = __ldcs(reinterpret_cast<const uint2 *>(s0));
        const uint2 b = __ldcs(reinterpret_cast<const uint2 *>(s1));
        const float2 a0 = unpack2<T>(a.x), a1 = unpack2<T>(a.y);
        const float2 b0 = unpack2<T>(b.x), b1 = unpack2<T>(b.y);
        re[0] = a0.x; re[1] = a0.y; re[2] = a1.x; re[3] = a1.y;
        im[0] = b0.x; im[1] = b0.y; im[2] = b1.x; im[3] = b1.y;
      }
    }
    if (!inside) {
#pragma unroll
      for (int i = 0; i < 4; ++i) re[i] = im[i] = 0.0f;
    }
  } else {
    const size_t row = min(r, rows - 1) * k;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const size_t s = row + min(k0 + i, k - 1);
      re[i] = to_float(IL ? in[2 * s] : in[s]);
      im[i] = to_float(IL ? in[2 * s + 1] : in[s + rows * k]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (r >= rows || k0 + i >= k) re[i] = im[i] = 0.0f;
    }
  }
}

// K contiguous.  A warp takes 128 k of kRows rows, a lane four consecutive samples of each row: loads
// and stores of a warp are whole 128-byte lines.  kWarps = 1: one scale per row, every warp on its
// own.  kWarps = 16: the block's 128 rows are the 16 warps' 8 rows each and share one scale.
template <typename T, bool IL, bool VEC, bool E5M2, int kRows, int kWarps>
__global__ void __launch_bounds__(kWarps == 1 ? 256 : 32 * kWarps)
quantize_rows_kernel(const QuantizeParams p) {
  constexpr bool kTile = kWarps > 1;
  __shared__ uint32_t warp_max[2][kTile ? kWarps : 1];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const size_t groups = ceil_div<size_t>(p.rows, kRows * kWarps);
  const size_t items = p.batch * groups * p.blocks_k;
  const size_t first = kTile ? blockIdx.x : blockIdx.x * (blockDim.x >> 5) + warp;
  const size_t step = kTile ? gridDim.x : gridDim.x * (blockDim.x >> 5);
  [[maybe_unused]] int turn = 0;
  for (size_t item = first; item < items; item += step) {
    const size_t kb = item % p.blocks_k;
    const size_t rest = item / p.blocks_k;
    const size_t group = rest % groups, b = rest / groups;
    const size_t r0 = group * (kRows * kWarps) + (kTile ? warp * kRows : 0);
    const size_t k0 = kb * kBlockK + lane * 4;
    const T *in = static_cast<const T *>(p.in) + b * 2 * p.rows * p.k;
    float re[kRows][4], im[kRows][4];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      load_quad<T, IL, VEC>(in, p.rows, p.k, r0 + i, k0, re[i], im[i]);
    }
    // Maxima of the bits without the sign: infinities and NaN are behind all finite values and are taken
    // out in a second go where there are any.
    uint32_t top[kRows];
    bool special = false;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      uint32_t t = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        t = max(t, max(__float_as_uint(re[i][j]) & 0x7FFFFFFFu, __float_as_uint(im[i][j]) & 0x7FFFFFFFu));
      }
      top[i] = t;
      special |= t >= 0x7F800000u;
    }
    if (special) {
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        uint32_t t = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          t = max(t, max(finite_abs_bits(re[i][j]), finite_abs_bits(im[i][j])));
        }
        top[i] = t;
      }
    }
    if constexpr (kTile) {
      uint32_t t = top[0];
#pragma unroll
      for (int i = 1; i < kRows; ++i) t = max(t, top[i]);
      t = __reduce_max_sync(0xFFFFFFFFu, t);
      if (lane == 0) warp_max[turn][warp] = t;
      __syncthreads();
      t = __reduce_max_sync(0xFFFFFFFFu, warp_max[turn][lane & (kWarps - 1)]);
      turn ^= 1;  // the other half of warp_max is free: every warp has passed this barrier
#pragma unroll
      for (int i = 0; i < kRows; ++i) top[i] = t;
    } else {
#pragma unroll
      for (int i = 0; i < kRows; ++i) top[i] = __reduce_max_sync(0xFFFFFFFFu, top[i]);
    }
    float *scale_row = p.scale + (b * p.blocks_k + kb) * p.blocks_rows;
    [[maybe_unused]] float mine = 0.0f;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const float s = block_scale<E5M2>(top[i]);
      const float inv = block_factor<E5M2>(top[i], s), inv_im = p.im_sign * inv;
      if constexpr (kTile) {
        if (i == 0 && threadIdx.x == 0) scale_row[group] = s;
      } else {
        if (lane == static_cast<uint32_t>(i)) mine = s;
      }
      const size_t r = r0 + i;
      if (r < p.rows && k0 < p.pitch) {
        float a[4], c[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          a[j] = re[i][j] * inv;
          c[j] = im[i][j] * inv_im;
        }
        uint8_t *dst = p.out + ((b * 2) * p.rows + r) * p.pitch + k0;
        uint32_t w_re = pack4<E5M2>(a), w_im = pack4<E5M2>(c);
        if (special) {
          w_re = pack4<E5M2, true>(a);
          w_im = pack4<E5M2, true>(c);
        }
        *reinterpret_cast<uint32_t *>(dst) = w_re;
        *reinterpret_cast<uint32_t *>(dst + p.rows * p.pitch) = w_im;
      }
    }
    if constexpr (!kTile) {
      if (lane < kRows && r0 + lane < p.rows) scale_row[r0 + lane] = mine;
    }
  }
}

// One complex value as it lies in memory: two 16-bit halves (re low) or two floats.
template <typename T> struct Raw {
  uint32_t w;
  __device__ __forceinline__ float2 value() const { return unpack2<T>(w); }
};
template <> struct Raw<float> {
  float2 v;
  __device__ __forceinline__ float2 value() const { return v; }
};
// N complex values `stride` complex apart, from re (and im, planar).  All loads are under way before the
// first is used.
template <typename T, bool IL, int N>
__device__ __forceinline__ void load_raw(const T *re, const T *im, size_t stride, Raw<T> (&x)[N]) {
  if constexpr (IL) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (sizeof(T) == 4) {
        x[i].v = __ldcs(reinterpret_cast<const float2 *>(re) + i * stride);
      } else {
        x[i].w = __ldcs(reinterpret_cast<const uint32_t *>(re) + i * stride);
      }
    }
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i].v = make_float2(__ldcs(re + i * stride), __ldcs(im + i * stride));
  } else {
    unsigned short lo[N], hi[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      lo[i] = __ldcs(reinterpret_cast<const unsigned short *>(re) + i * stride);
      hi[i] = __ldcs(reinterpret_cast<const unsigned short *>(im) + i * stride);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) x[i].w = lo[i] | (static_cast<uint32_t>(hi[i]) << 16);
  }
}

// Largest finite |re|, |im| of N values, as the bits of a float32; `special` is raised if there are others.
template <typename T, int N>
__device__ __forceinline__ uint32_t top_bits(const Raw<T> (&x)[N], bool &special) {
  // the patterns without the sign order like the values, infinities and NaN behind all others
  uint32_t m = 0;
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < N; ++i) m = __vmaxu2(m, x[i].w & 0x7FFF7FFFu);
    m = max(m & 0xFFFFu, m >> 16);
    if (m < (std::is_same_v<T, __half> ? 0x7C00u : 0x7F80u)) return __float_as_uint(unpack2<T>(m).x);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      m = max(m, max(__float_as_uint(x[i].v.x) & 0x7FFFFFFFu, __float_as_uint(x[i].v.y) & 0x7FFFFFFFu));
    }
    if (m < 0x7F800000u) return m;
  }
  special = true;
  m = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float2 v = x[i].value();
    m = max(m, max(finite_abs_bits(v.x), finite_abs_bits(v.y)));
  }
  return m;
}

// Rows contiguous ([k][rows]): the operand of a product over the matrix's other axis.  A CTA takes
// 128 rows x 128 k; a lane reads one row of every fourth of them, so a warp's loads run along the
// rows; the bytes turn in shared memory (8 k of a row per store) and leave in runs of 128.  TILE: one
// scale for the block, else one per row.  Values wait in registers as they came (16-bit types: one
// register per complex value, so that two CTAs fit an SM and one loads while the other stores).
constexpr int kColWarps = 16;
constexpr int kColK = kBlockK / kColWarps;  // k per warp
constexpr int kColPitch = kBlockK + 8;      // 8-byte accesses down the rows touch every bank once

template <typename T, bool IL, bool E5M2, bool TILE>
__global__ void __launch_bounds__(32 * kColWarps, sizeof(T) == 2 ? 2 : 1)
quantize_cols_kernel(const QuantizeParams p) {
  __shared__ __align__(16) uint8_t bytes[2][128 * kColPitch];
  __shared__ uint32_t row_max[128];
  __shared__ float row_inv[128];
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const size_t groups = ceil_div<size_t>(p.rows, 128);
  const size_t items = p.batch * groups * p.blocks_k;
  for (size_t item = blockIdx.x; item < items; item += gridDim.x) {
    const size_t group = item % groups;
    const size_t rest = item / groups;
    const size_t kb = rest % p.blocks_k, b = rest / p.blocks_k;
    const size_t r0 = group * 128, k0 = kb * kBlockK + warp * kColK;
    const T *in = static_cast<const T *>(p.in) + b * 2 * p.rows * p.k;
    if (tid < 128) row_max[tid] = 0;
    Raw<T> x[4][kColK];
    if (r0 + 128 <= p.rows && (kb + 1) * kBlockK <= p.k) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const T *re = in + (k0 * p.rows + r0 + 32 * j + lane) * (IL ? 2 : 1);
        load_raw<T, IL, kColK>(re, re + p.rows * p.k, p.rows, x[j]);
      }
    } else {
      // at the edges: the last row and k stand in for what lies outside, then zeros
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const size_t r = r0 + 32 * j + lane;
        const T *re = in + (min(k0, p.k - 1) * p.rows + min(r, p.rows - 1)) * (IL ? 2 : 1);
#pragma unroll
        for (int i = 0; i < kColK; ++i) {
          Raw<T> one[1];
          load_raw<T, IL, 1>(re, re + p.rows * p.k, 0, one);
          x[j][i] = r < p.rows && k0 + i < p.k ? one[0] : Raw<T>{};
          if (k0 + i + 1 < p.k) re += p.rows * (IL ? 2 : 1);
        }
      }
    }
    __syncthreads();  // row_max is zero; the previous item's bytes have been read
    bool special = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) atomicMax(&row_max[32 * j + lane], top_bits<T, kColK>(x[j], special));
    __syncthreads();
    float inv_tile = 0.0f;
    if constexpr (TILE) {
      uint32_t t = max(max(row_max[lane], row_max[32 + lane]), max(row_max[64 + lane], row_max[96 + lane]));
      t = __reduce_max_sync(0xFFFFFFFFu, t);
      const float s = block_scale<E5M2>(t);
      inv_tile = block_factor<E5M2>(t, s);
      if (tid == 0) p.scale[(b * p.blocks_k + kb) * p.blocks_rows + group] = s;
    } else {
      if (tid < 128) {
        const float s = block_scale<E5M2>(row_max[tid]);
        row_inv[tid] = block_factor<E5M2>(row_max[tid], s);
        if (r0 + tid < p.rows) p.scale[(b * p.blocks_k + kb) * p.blocks_rows + r0 + tid] = s;
      }
      __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float inv = TILE ? inv_tile : row_inv[32 * j + lane], inv_im = p.im_sign * inv;
      const uint32_t at = (32 * j + lane) * kColPitch + warp * kColK;
      uint32_t w[4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float a[4], c[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 v = x[j][4 * h + i].value();
          a[i] = v.x * inv;
          c[i] = v.y * inv_im;
        }
        w[h] = pack4<E5M2>(a);
        w[2 + h] = pack4<E5M2>(c);
        if (special) {
          w[h] = pack4<E5M2, true>(a);
          w[2 + h] = pack4<E5M2, true>(c);
        }
      }
      *reinterpret_cast<uint2 *>(&bytes[0][at]) = make_uint2(w[0], w[1]);
      *reinterpret_cast<uint2 *>(&bytes[1][at]) = make_uint2(w[2], w[3]);
    }
    __syncthreads();
    // 2 planes x 128 rows x 16 pieces of 8 bytes
#pragma unroll
    for (int i = 0; i < 2 * 128 * 16 / (32 * kColWarps); ++i) {
      const uint32_t piece = i * 32 * kColWarps + tid;
      const uint32_t plane = piece >> 11, r = (piece >> 4) & 127, y = (piece & 15) * 8;
      const size_t k_at = kb * kBlockK + y;
      if (r0 + r < p.rows && k_at < p.pitch) {
        *reinterpret_cast<uint2 *>(p.out + ((b * 2 + plane) * p.rows + r0 + r) * p.pitch + k_at) =
            *reinterpret_cast<const uint2 *>(&bytes[plane][r * kColPitch + y]);
      }
    }
  }
}

unsigned grid_for(size_t ctas, size_t per_sm) {
  const size_t cap = static_cast<size_t>(sm_count()) * per_sm;
  return static_cast<unsigned>(ctas < cap ? ctas : cap);
}

template <typename T, bool IL, bool E5M2>
int launch(const QuantizeParams &p, bool col_major, bool tile, cudaStream_t stream) {
  if (col_major) {
    const unsigned grid = grid_for(p.batch * ceil_div<size_t>(p.rows, 128) * p.blocks_k, 16);
    if (tile) {
      quantize_cols_kernel<T, IL, E5M2, true><<<grid, 32 * kColWarps, 0, stream>>>(p);
    } else {
      quantize_cols_kernel<T, IL, E5M2, false><<<grid, 32 * kColWarps, 0, stream>>>(p);
    }
  } else {
    const bool vec = p.k % 4 == 0;
    if (tile) {
      const unsigned grid = grid_for(p.batch * ceil_div<size_t>(p.rows, 128) * p.blocks_k, 16);
      if (vec) {
        quantize_rows_kernel<T, IL, true, E5M2, 8, 16><<<grid, 512, 0, stream>>>(p);
      } else {
        quantize_rows_kernel<T, IL, false, E5M2, 8, 16><<<grid, 512, 0, stream>>>(p);
      }
    } else {
      const size_t warps = p.batch * ceil_div<size_t>(p.rows, 4) * p.blocks_k;
      const unsigned grid = grid_for(ceil_div<size_t>(warps, 8), 64);
      if (vec) {
        quantize_rows_kernel<T, IL, true, E5M2, 4, 1><<<grid, 256, 0, stream>>>(p);
      } else {
        quantize_rows_kernel<T, IL, false, E5M2, 4, 1><<<grid, 256, 0, stream>>>(p);
      }
    }
  }
  CCGLIB_CUDA_TRY(cudaGetLastError());
  return CCGLIB_B200_OK;
}

template <typename T>
int launch_typed(const QuantizeParams &p, bool il, bool e5m2, bool col_major, bool tile,
                 cudaStream_t stream) {
  if (il) {
    return e5m2 ? launch<T, true, true>(p, col_major, tile, stream)
                : launch<T, true, false>(p, col_major, tile, stream);
  }
  return e5m2 ? launch<T, false, true>(p, col_major, tile, stream)
              : launch<T, false, false>(p, col_major, tile, stream);
}

} // namespace
} // namespace ccglib_b200

using namespace ccglib_b200;

extern "C" int ccglib_b200_quantize_run(const ccglib_b200_quantize_desc *desc, const void *d_in,
                                        void *d_out, float *d_scale, void *stream_v) {
  if (desc == nullptr || d_in == nullptr || d_out == nullptr || d_scale == nullptr) {
    set_last_error("quantize_run: null argument");
    return CCGLIB_B200_INVALID_ARGUMENT;
  }
  const ccglib_b200_quantize_desc &d = *desc;
  if (d.batch == 0 || d.rows == 0 || d.k == 0) {
    set_last_error("quantize_run: batch, rows and K must be positive");
    return CCGLIB_B200_INVALID_ARGUMENT;
  }
  // (the last test keeps the byte counts below inside 64 bits)
  if (d.rows > 0x7FFFFFFFull || d.k > 0x7FFFFFFFull || d.batch > 0x3FFFFFFFull ||
      d.batch > (size_t{1} << 58) / (d.rows * d.k)) {
    set_last_error("quantize_run: dimension too large");
    return CCGLIB_B200_INVALID_ARGUMENT;
  }
  if (d.type_in != CCGLIB_B200_FLOAT16 && d.type_in != CCGLIB_B200_BFLOAT16 &&
      d.type_in != CCGLIB_B200_FLOAT32) {
    set_last_error("quantize_run: input must be float16, bfloat16 or float32 (got %d)", d.type_in);
    return CCGLIB_B200_UNSUPPORTED;
  }
  if (d.type_out != CCGLIB_B200_FLOAT8E4M3 && d.type_out != CCGLIB_B200_FLOAT8E5M2) {
    set_last_error("quantize_run: output must be float8e4m3 or float8e5m2 (got %d)", d.type_out);
    return CCGLIB_B200_UNSUPPORTED;
  }
  if (d.block_rows != 1 && d.block_rows != 128) {
    set_last_error("quantize_run: a block has 1 or 128 rows (got %zu)", d.block_rows);
    return CCGLIB_B200_INVALID_ARGUMENT;
  }
  if ((d.input_complex_axis != CCGLIB_B200_PLANAR &&
       d.input_complex_axis != CCGLIB_B200_INTERLEAVED) ||
      (d.input_mem_order != CCGLIB_B200_ROW_MAJOR && d.input_mem_order != CCGLIB_B200_COL_MAJOR)) {
    set_last_error("quantize_run: unknown complex axis location %d or memory order %d",
                   d.input_complex_axis, d.input_mem_order);
    return CCGLIB_B200_INVALID_ARGUMENT;
  }
  if (d.conjugate != 0 && d.conjugate != 1) {
    set_last_error("quantize_run: conjugate must be 0 or 1 (got %d)", d.conjugate);
    return CCGLIB_B200_INVALID_ARGUMENT;
  }
  if (!aligned16(d_in) || !aligned16(d_out) || (reinterpret_cast<uintptr_t>(d_scale) & 3u) != 0) {
    set_last_error("quantize_run: input and output must be 16-byte aligned, scales 4-byte aligned");
    return CCGLIB_B200_INVALID_ARGUMENT;
  }
  QuantizeParams p{};
  p.in = d_in;
  p.out = static_cast<uint8_t *>(d_out);
  p.scale = d_scale;
  p.batch = d.batch;
  p.rows = d.rows;
  p.k = d.k;
  p.pitch = ceil_div<size_t>(d.k, 16) * 16;
  p.blocks_k = ceil_div<size_t>(d.k, kBlockK);
  p.blocks_rows = ceil_div<size_t>(d.rows, d.block_rows);
  p.im_sign = d.conjugate ? -1.0f : 1.0f;
  // blocks are read and written in any order
  const size_t in_bytes = d.batch * 2 * d.rows * d.k * (d.type_in == CCGLIB_B200_FLOAT32 ? 4 : 2);
  const size_t out_bytes = d.batch * 2 * d.rows * p.pitch;
  const size_t scale_bytes = d.batch * p.blocks_k * p.blocks_rows * sizeof(float);
  if (overlap(d_in, in_bytes, d_out, out_bytes) || overlap(d_in, in_bytes, d_scale, scale_bytes) ||
      overlap(d_out, out_bytes, d_scale, scale_bytes)) {
    set_last_error("quantize_run: input, output and scales must not overlap");
    return CCGLIB_B200_INVALID_ARGUMENT;
  }
  if (sm_count() <= 0) return CCGLIB_B200_CUDA_ERROR;
  const bool il = d.input_complex_axis == CCGLIB_B200_INTERLEAVED;
  const bool e5m2 = d.type_out == CCGLIB_B200_FLOAT8E5M2;
  const bool col = d.input_mem_order == CCGLIB_B200_COL_MAJOR;
  const bool tile = d.block_rows == 128;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  switch (d.type_in) {
  case CCGLIB_B200_FLOAT16:
    return launch_typed<__half>(p, il, e5m2, col, tile, stream);
  case CCGLIB_B200_BFLOAT16:
    return launch_typed<__nv_bfloat16>(p, il, e5m2, col, tile, stream);
  default:
    return launch_typed<float>(p, il, e5m2, col, tile, stream);
  }
}
