// Orthogonalisation of complex matrices by Newton-Schulz products.
//
//   X <- X / ||X||_F;   `steps` times:  S = X X^H,  P = b S + c S S,  X <- a X + P X
//
// (on the shorter side: a matrix with more rows than columns is iterated as its transpose).  Every step
// keeps the singular vectors and maps each singular value s to s (a + b s^2 + c s^4).
//
// The three products of a step run on the tensor cores, kind::f16 with float32 sums, through
// cgemm_tcgen05_kernel with an epilogue of its own: the conjugate of B comes from the negate bit of
// the other cross product, S and P are computed on and above the diagonal and mirrored on the way
// out, b S and a X are added from the operand that is there already, and the update stores X and its
// transpose (the next step contracts over the one, then the other), so a step is three launches and
// nothing else.  The last update writes the caller's type and layout.
//
// Between products X, S and P are float16.  All three are bounded (a singular value is at most about
// one), X is kept times a power of two near sqrt(long side) so that its entries are near one, and float16
// keeps eleven bits where bfloat16, the other 16-bit choice, keeps eight: rms error 1 to 2.5e-3 of the
// result after 5 to 8 steps, about that of rounding it to bfloat16.  Sums and the norm
// are float32 and float64.
#include <cmath>
#include <new>

#include "gemm_kernels.cuh"

namespace ccglib_b200 {
namespace {

using OrthFn = void (*)(const CUtensorMap, const CUtensorMap, const CUtensorMap, const GemmParams);

OrthFn orth_kernel(int bn) {
  return bn == 256   ? cgemm_tcgen05_kernel<kKindF16, 256, 128, 2, OrthHalf, 0>
         : bn == 128 ? cgemm_tcgen05_kernel<kKindF16, 128, 128, 2, OrthHalf, 0>
                     : cgemm_tcgen05_kernel<kKindF16, 64, 128, 2, OrthHalf, 0>;
}

int orth_smem(int bn) {
  return bn == 256   ? Cfg<256, 128, 2, 0>::kSmemBytes
         : bn == 128 ? Cfg<128, 128, 2, 0>::kSmemBytes
                     : Cfg<64, 128, 2, 0>::kSmemBytes;
}

// Tiles of one product and the width that finishes soonest: waves x time per tile relative to a 128-wide
// tile (a 64-wide one takes as long on the tensor pipe, a 256-wide one 5 % less per column).
struct ProductShape {
  int bn;
  size_t per_batch;
};

size_t upper_tiles(size_t n, size_t bn) {
  const size_t rows = ceil_div<size_t>(n, kBlockM), cols = ceil_div<size_t>(n, bn);
  size_t tiles = 0;
  for (size_t i = 0; i < rows; ++i) tiles += cols - i * kBlockM / bn;
  return tiles;
}

ProductShape pick_shape(size_t batch, size_t m, size_t n, bool hermitian, size_t sms) {
  ProductShape best{0, 0};
  double least = 0.0;
  for (int bn : {128, 256, 64}) {
    const size_t tiles = hermitian ? upper_tiles(m, bn)
                                   : ceil_div<size_t>(m, kBlockM) * ceil_div<size_t>(n, bn);
    const double cost = static_cast<double>(ceil_div(batch * tiles, sms)) *
                        (bn == 256 ? 1.9 : bn == 128 ? 1.0 : 0.95);
    if (best.bn == 0 || cost < least) {
      best = {bn, tiles};
      least = cost;
    }
  }
  return best;
}

// ---- norm and first iterate ---------------------------------------------------------------------

template <typename T> __device__ __forceinline__ float as_float(T v);
template <> __device__ __forceinline__ float as_float(float v) { return v; }
template <> __device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }

constexpr int kNormThreads = 256;
constexpr size_t kNormChunk = 16384;  // values one CTA adds up

// Sums of squares of kNormChunk values each, in float64 (no input overflows or vanishes in it).
template <typename T>
__global__ void __launch_bounds__(kNormThreads)
norm_kernel(const T *in, double *sums, size_t values, size_t chunks, size_t items) {
  __shared__ double part[kNormThreads / 32];
  for (size_t item = blockIdx.x; item < items; item += gridDim.x) {
    const size_t b = item / chunks, c = item - b * chunks;
    const T *src = in + b * values;
    const size_t end = min(values, (c + 1) * kNormChunk);
    double sum = 0.0;
    for (size_t i = c * kNormChunk + threadIdx.x; i < end; i += kNormThreads) {
      const double v = static_cast<double>(as_float(src[i]));
      sum += v * v;
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
  __half *x, *x_t;       // x: [batch][2][short_p][long_p], x_t: [batch][2][long_p][short_p]
  size_t rows_p, cols_p;  // rows and cols rounded up to eight
  bool tall;              // rows is the long side: x is the transpose of the input
  float scale;
};

constexpr int kFirstTile = 64;

// X0 = scale * input / norm and its transpose, zero padded.  A CTA turns one 64 x 64 tile of a plane
// pair in shared memory, so that both copies are written along their rows.
template <typename T, bool IL>
__global__ void __launch_bounds__(256) first_kernel(const FirstParams p) {
  __shared__ __half tile[2][kFirstTile][kFirstTile + 2];
  __shared__ double part[256 / 32];
  const size_t tr = ceil_div<size_t>(p.rows_p, kFirstTile), tc = ceil_div<size_t>(p.cols_p, kFirstTile);
  const size_t items = p.batch * tr * tc;
  // input rows x cols planes: `straight` has its layout, `turned` the transposed one
  __half *straight = p.tall ? p.x_t : p.x, *turned = p.tall ? p.x : p.x_t;
  const size_t plane_p = p.rows_p * p.cols_p;
  for (size_t item = blockIdx.x; item < items; item += gridDim.x) {
    const size_t b = item / (tr * tc), rest = item - b * (tr * tc);
    const size_t r0 = rest / tc * kFirstTile, c0 = rest % tc * kFirstTile;
    double sum = 0.0;
    for (size_t i = threadIdx.x; i < p.chunks; i += 256) sum += p.sums[b * p.chunks + i];
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
    __syncthreads();
    sum = 0.0;
    for (int w = 0; w < 256 / 32; ++w) sum += part[w];
    // a zero matrix stays zero (and one with a NaN becomes NaN)
    const double factor = sum == 0.0 ? 0.0 : static_cast<double>(p.scale) / sqrt(sum);
    const T *in = static_cast<const T *>(p.in) + b * 2 * p.rows * p.cols;
    for (int i = threadIdx.x; i < kFirstTile * kFirstTile; i += 256) {
      const size_t r = r0 + i / kFirstTile, c = c0 + i % kFirstTile;
      float re = 0.0f, im = 0.0f;
      if (r < p.rows && c < p.cols) {
        const size_t s = r * p.cols + c;
        re = as_float(IL ? in[2 * s] : in[s]);
        im = as_float(IL ? in[2 * s + 1] : in[s + p.rows * p.cols]);
      }
      const __half hr = __float2half_rn(static_cast<float>(re * factor));
      const __half hi = __float2half_rn(static_cast<float>(im * factor));
      if (r < p.rows_p && c < p.cols_p) {
        __half *dst = straight + b * 2 * plane_p + r * p.cols_p + c;
        dst[0] = hr;
        dst[plane_p] = hi;
      }
      tile[0][i / kFirstTile][i % kFirstTile] = hr;
      tile[1][i / kFirstTile][i % kFirstTile] = hi;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kFirstTile * kFirstTile; i += 256) {
      const int y = i / kFirstTile, x = i % kFirstTile;
      const size_t c = c0 + y, r = r0 + x;
      if (r < p.rows_p && c < p.cols_p) {
        __half *dst = turned + b * 2 * plane_p + c * p.rows_p + r;
        dst[0] = tile[0][x][y];
        dst[plane_p] = tile[1][x][y];
      }
    }
    __syncthreads();
  }
}

} // namespace
} // namespace ccglib_b200

using namespace ccglib_b200;

struct ccglib_b200_orthogonalize_plan {
  ccglib_b200_orthogonalize_desc desc;
  size_t n, l, n_p, l_p;  // short and long side, and both rounded up to eight
  bool tall;              // m > n: iterate on the transpose
  float scale;            // power of two near sqrt(long side)
  ProductShape gram, update;
  size_t chunks;
  int device, sms;
  long long wait_cycles;
  unsigned *status;
  void *scratch;
  size_t scratch_bytes;
  __half *x, *x_t[2], *s, *p;
  double *sums;
};

namespace {

struct Product {
  const __half *a, *b;  // planes of m x k and n x k
  size_t m, n, k;
  ProductShape shape;
  bool hermitian, conj;
  float alpha, beta;
  const __half *c0;
  void *c;
  __half *c_t;
  bool last;
};

int launch_product(const ccglib_b200_orthogonalize_plan &plan, const Product &q, cudaStream_t stream) {
  const size_t batch = plan.desc.batch;
  GemmParams g{};
  g.M = static_cast<uint32_t>(q.m);
  g.N = static_cast<uint32_t>(q.n);
  g.k_blocks = static_cast<uint32_t>(ceil_div<size_t>(q.k * 2, 128));
  g.tiles_m = static_cast<uint32_t>(ceil_div<size_t>(q.m, kBlockM));
  g.tiles_n = static_cast<uint32_t>(ceil_div<size_t>(q.n, q.shape.bn));
  g.group_n = (q.shape.bn == 256 || g.tiles_m <= 2) ? 4 : 8;
  g.num_tiles = static_cast<uint32_t>(batch * q.shape.per_batch);
  g.idesc = (1u << 4) | (static_cast<uint32_t>(q.shape.bn >> 3) << 17) |
            (static_cast<uint32_t>(kBlockM >> 4) << 24);  // fp32 sums, f16 operands
  g.idesc_neg_a = g.idesc | (1u << 13);
  g.c = q.c;
  g.c_layout = kPlanarRow;
  g.alpha_re = q.alpha;
  g.beta_re = q.beta;
  g.have_beta = q.c0 != nullptr ? 1u : 0u;
  g.c_in = q.c0;
  g.c_t = q.c_t;
  g.conj_b = q.conj ? 1u : 0u;
  g.hermitian = q.hermitian ? static_cast<uint32_t>(q.shape.per_batch) : 0u;
  if (q.last) {
    g.final_type = static_cast<uint32_t>(plan.desc.type_out);
    g.final_trans = plan.tall ? 1u : 0u;
    g.final_m = static_cast<uint32_t>(plan.n);
    g.final_n = static_cast<uint32_t>(plan.l);
    g.beta_im = 1.0f / plan.scale;
    g.vec_ok = (!plan.tall && plan.l % 8 == 0 && aligned16(q.c)) ? 1u : 0u;
  }
  g.status = plan.status;
  g.wait_cycles = plan.wait_cycles;
  CUtensorMap tm_a, tm_b;
  int rc = make_map(&tm_a, q.a, q.k * 2, q.m, 2 * batch, q.k * 2, q.m * q.k * 2, 128, kBlockM, 2);
  if (rc != CCGLIB_B200_OK) return rc;
  rc = make_map(&tm_b, q.b, q.k * 2, q.n, 2 * batch, q.k * 2, q.n * q.k * 2, 128, q.shape.bn, 2);
  if (rc != CCGLIB_B200_OK) return rc;
  const unsigned grid = g.num_tiles < static_cast<uint32_t>(plan.sms) ? g.num_tiles : plan.sms;
  orth_kernel(q.shape.bn)<<<grid, kThreads, orth_smem(q.shape.bn), stream>>>(tm_a, tm_b, tm_a, g);
  CCGLIB_CUDA_TRY(cudaGetLastError());
  return CCGLIB_B200_OK;
}

template <typename T>
int launch_first(const ccglib_b200_orthogonalize_plan &plan, const void *d_in, cudaStream_t stream) {
  const ccglib_b200_orthogonalize_desc &d = plan.desc;
  const size_t items = d.batch * plan.chunks;
  const size_t cap = static_cast<size_t>(plan.sms) * 8;
  norm_kernel<T><<<static_cast<unsigned>(items < cap ? items : cap), kNormThreads, 0, stream>>>(
      static_cast<const T *>(d_in), plan.sums, 2 * d.m * d.n, plan.chunks, items);
  CCGLIB_CUDA_TRY(cudaGetLastError());
  FirstParams p{};
  p.in = d_in;
  p.sums = plan.sums;
  p.chunks = plan.chunks;
  p.batch = d.batch;
  p.rows = d.m;
  p.cols = d.n;
  p.x = plan.x;
  p.x_t = plan.x_t[0];
  p.rows_p = plan.tall ? plan.l_p : plan.n_p;
  p.cols_p = plan.tall ? plan.n_p : plan.l_p;
  p.tall = plan.tall;
  p.scale = plan.scale;
  const size_t tiles = d.batch * ceil_div<size_t>(p.rows_p, kFirstTile) * ceil_div<size_t>(p.cols_p, kFirstTile);
  const unsigned grid = static_cast<unsigned>(tiles < cap ? tiles : cap);
  if (d.input_complex_axis == CCGLIB_B200_INTERLEAVED) {
    first_kernel<T, true><<<grid, 256, 0, stream>>>(p);
  } else {
    first_kernel<T, false><<<grid, 256, 0, stream>>>(p);
  }
  CCGLIB_CUDA_TRY(cudaGetLastError());
  return CCGLIB_B200_OK;
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
  plan.l_p = ceil_div<size_t>(plan.l, 8) * 8;
  plan.scale = std::exp2(std::rint(0.5f * std::log2(static_cast<float>(plan.l))));
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
  plan.gram = pick_shape(d.batch, plan.n_p, plan.n_p, true, plan.sms);
  plan.update = pick_shape(d.batch, plan.n_p, plan.l_p, false, plan.sms);
  if (d.batch * plan.gram.per_batch > 0x7FFFFFFFull ||
      d.batch * plan.update.per_batch > 0x7FFFFFFFull) {
    set_last_error("orthogonalize_plan_create: too many tiles");
    return CCGLIB_B200_INVALID_ARGUMENT;
  }
  for (int bn : {64, 128, 256}) {
    CCGLIB_CUDA_TRY(cudaFuncSetAttribute(reinterpret_cast<const void *>(orth_kernel(bn)),
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, orth_smem(bn)));
  }
  plan.chunks = ceil_div<size_t>(2 * d.m * d.n, kNormChunk);
  const size_t x_bytes = ceil_div<size_t>(d.batch * 2 * plan.n_p * plan.l_p * 2, 256) * 256;
  const size_t s_bytes = ceil_div<size_t>(d.batch * 2 * plan.n_p * plan.n_p * 2, 256) * 256;
  plan.scratch_bytes = 3 * x_bytes + 2 * s_bytes + d.batch * plan.chunks * sizeof(double);
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
  plan.x = reinterpret_cast<__half *>(take(x_bytes));
  plan.x_t[0] = reinterpret_cast<__half *>(take(x_bytes));
  plan.x_t[1] = reinterpret_cast<__half *>(take(x_bytes));
  plan.s = reinterpret_cast<__half *>(take(s_bytes));
  plan.p = reinterpret_cast<__half *>(take(s_bytes));
  plan.sums = reinterpret_cast<double *>(at);
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
  int device = -1;
  CCGLIB_CUDA_TRY(cudaGetDevice(&device));
  if (device != plan->device) {
    set_last_error("orthogonalize_run: the plan belongs to device %d, the current device is %d",
                   plan->device, device);
    return CCGLIB_B200_INVALID_ARGUMENT;
  }
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  int rc = d.type_in == CCGLIB_B200_FLOAT32   ? launch_first<float>(*plan, d_in, stream)
           : d.type_in == CCGLIB_B200_FLOAT16 ? launch_first<__half>(*plan, d_in, stream)
                                              : launch_first<__nv_bfloat16>(*plan, d_in, stream);
  const size_t n = plan->n_p, l = plan->l_p;
  const float unscale = 1.0f / (plan->scale * plan->scale);
  for (int step = 0; rc == CCGLIB_B200_OK && step < d.steps; ++step) {
    const bool last = step + 1 == d.steps;
    __half *now = plan->x_t[step & 1], *next = plan->x_t[(step & 1) ^ 1];
    const Product gram{plan->x, plan->x, n, n, l, plan->gram, true, true, unscale, 0.0f,
                       nullptr, plan->s, plan->s, false};
    rc = launch_product(*plan, gram, stream);
    if (rc != CCGLIB_B200_OK) break;
    const Product poly{plan->s, plan->s, n, n, n, plan->gram, true, true, d.c, d.b,
                       plan->s, plan->p, plan->p, false};
    rc = launch_product(*plan, poly, stream);
    if (rc != CCGLIB_B200_OK) break;
    // (X is read as C0 and written by the same thread; the operand is its transpose)
    const Product update{plan->p, now, n, l, n, plan->update, false, false, 1.0f, d.a,
                         plan->x, last ? d_out : plan->x, last ? nullptr : next, last};
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
