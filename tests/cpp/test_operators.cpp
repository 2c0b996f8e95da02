// Self-checking program for ccglib::quantize::Quantize, ccglib::mma::ScaledGEMM and
// ccglib::orthogonalize::Orthogonalize with raw CUDA handles and cu:: objects.  Prints one line per case;
// exit code = failures.
#include <cmath>
#include <complex>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <functional>
#include <random>
#include <stdexcept>
#include <string>
#include <vector>

#include <cuda.h>
#include <cuda_fp16.h>

#include <cudawrappers/cu.hpp>

#include <ccglib/gemm/scaled.h>
#include <ccglib/orthogonalize/orthogonalize.h>
#include <ccglib/quantize/quantize.h>

namespace {

int failures = 0;

void run_case(const char *name, const std::function<bool()> &body) {
  bool ok = false;
  std::string detail;
  try {
    ok = body();
  } catch (const std::exception &e) {
    detail = std::string("exception: ") + e.what();
  }
  std::printf("%s %s %s\n", ok ? "PASS" : "FAIL", name, detail.c_str());
  if (!ok) ++failures;
}

bool throws_with(const std::function<void()> &body, const char *needle) {
  try {
    body();
  } catch (const std::exception &e) {
    return std::strstr(e.what(), needle) != nullptr;
  }
  return false;
}

struct Buffer {
  CUdeviceptr p{};
  explicit Buffer(size_t bytes) { cu::checkCudaCall(cuMemAlloc(&p, bytes)); }
  ~Buffer() { cuMemFree(p); }
};

// Small integers quantise exactly when every block's largest value is 448 (scale 1), so the product is
// an exact integer: all of it fits float32.
bool quantize_and_multiply(CUdevice device, CUstream stream) {
  const size_t B = 2, M = 5, N = 130, K = 200;
  std::mt19937 rng(1);
  std::uniform_int_distribution<int> small(-4, 4);
  std::vector<float> a(B * 2 * M * K), b(B * 2 * N * K);
  for (auto *v : {&a, &b}) {
    for (size_t i = 0; i < v->size(); ++i) (*v)[i] = static_cast<float>(small(rng));
    for (size_t row = 0; row < v->size() / K; ++row) {
      (*v)[row * K] = 448.0f;
      (*v)[row * K + 128] = -448.0f;
    }
  }
  using ccglib::ValueType;
  ccglib::quantize::Quantize qa(B, M, K, device, stream, ValueType::float32, ValueType::float8e4m3);
  ccglib::quantize::Quantize qb(B, N, K, device, stream, ValueType::float32, ValueType::float8e4m3, 128);
  ccglib::mma::ScaledGEMM gemm(B, M, N, K, device, stream, ValueType::float8e4m3,
                               ValueType::float8e4m3);
  if (qa.OutputBytes() != B * 2 * M * 208 || qa.ScaleBytes() != B * 2 * M * 4 ||
      qb.ScaleBytes() != B * 2 * 2 * 4 || gemm.stream() != stream) {
    return false;
  }
  Buffer da(a.size() * 4), db(b.size() * 4), fa(qa.OutputBytes()), fb(qb.OutputBytes()),
      sa(qa.ScaleBytes()), sb(qb.ScaleBytes()), dc(B * 2 * M * N * 4);
  cu::checkCudaCall(cuMemcpyHtoD(da.p, a.data(), a.size() * 4));
  cu::checkCudaCall(cuMemcpyHtoD(db.p, b.data(), b.size() * 4));
  qa.Run(da.p, fa.p, sa.p);
  qb.Run(db.p, fb.p, sb.p);
  gemm.Run(fa.p, sa.p, fb.p, sb.p, dc.p);
  cu::checkCudaCall(cuStreamSynchronize(stream));
  std::vector<float> c(B * 2 * M * N);
  cu::checkCudaCall(cuMemcpyDtoH(c.data(), dc.p, c.size() * 4));
  for (size_t i = 0; i < B; ++i) {
    for (size_t m = 0; m < M; ++m) {
      for (size_t n = 0; n < N; ++n) {
        double re = 0, im = 0;
        for (size_t k = 0; k < K; ++k) {
          const double ar = a[((i * 2) * M + m) * K + k], ai = a[((i * 2 + 1) * M + m) * K + k];
          const double br = b[((i * 2) * N + n) * K + k], bi = b[((i * 2 + 1) * N + n) * K + k];
          re += ar * br - ai * bi;
          im += ar * bi + ai * br;
        }
        if (c[((i * 2) * M + m) * N + n] != re || c[((i * 2 + 1) * M + m) * N + n] != im) return false;
      }
    }
  }
  return true;
}

// Rows of the result are orthonormal.
bool orthogonalize_rows(cu::Device &device, cu::Stream &stream) {
  const size_t M = 12, N = 90;
  std::mt19937 rng(2);
  std::normal_distribution<float> normal;
  std::vector<float> x(2 * M * N);
  for (float &v : x) v = normal(rng);
  ccglib::orthogonalize::Orthogonalize ortho(1, M, N, device, stream, ccglib::ValueType::float32,
                                             ccglib::ValueType::float16, 12,
                                             ccglib::orthogonalize::convergent);
  Buffer in(x.size() * 4), out(x.size() * 2);
  cu::checkCudaCall(cuMemcpyHtoD(in.p, x.data(), x.size() * 4));
  ortho.Run(in.p, out.p);
  cu::checkCudaCall(cuStreamSynchronize(ortho.stream()));
  std::vector<half> y(x.size());
  cu::checkCudaCall(cuMemcpyDtoH(y.data(), out.p, y.size() * 2));
  for (size_t i = 0; i < M; ++i) {
    for (size_t j = 0; j < M; ++j) {
      std::complex<double> dot = 0;
      for (size_t k = 0; k < N; ++k) {
        dot += std::complex<double>(__half2float(y[i * N + k]), __half2float(y[(M + i) * N + k])) *
               std::conj(std::complex<double>(__half2float(y[j * N + k]),
                                              __half2float(y[(M + j) * N + k])));
      }
      // rounding to float16 moves either row by at most 2^-11 of its length
      if (std::abs(dot - (i == j ? 1.0 : 0.0)) > 4.0 / 2048) return false;
    }
  }
  return true;
}

bool error_cases(CUdevice device, CUstream stream) {
  using ccglib::ValueType;
  return throws_with([&] { ccglib::quantize::Quantize(1, 1, 1, device, stream, ValueType::float32,
                                                      ValueType::float8e4m3, 64); },
                     "1 or 128 rows") &&
         throws_with([&] { ccglib::mma::ScaledGEMM(1, 8, 8, 8, device, stream, ValueType::float16,
                                                   ValueType::float8e4m3); },
                     "float8e4m3 or float8e5m2") &&
         throws_with([&] { ccglib::orthogonalize::Orthogonalize(1, 8, 8, device, stream,
                                                                ValueType::float32,
                                                                ValueType::float32); },
                     "output must be float16 or bfloat16");
}

} // namespace

int main() {
  cu::checkCudaCall(cuInit(0));
  CUdevice device{};
  CUcontext context{};
  CUstream stream{};
  cu::checkCudaCall(cuDeviceGet(&device, 0));
  cu::checkCudaCall(cuDevicePrimaryCtxRetain(&context, device));
  cu::checkCudaCall(cuCtxSetCurrent(context));
  cu::checkCudaCall(cuStreamCreate(&stream, CU_STREAM_NON_BLOCKING));
  run_case("quantize_and_scaled_gemm", [&] { return quantize_and_multiply(device, stream); });
  run_case("orthogonalize_cu_objects", [] {
    cu::Device device(0);
    cu::Stream stream(CU_STREAM_NON_BLOCKING);
    return orthogonalize_rows(device, stream);
  });
  run_case("error_cases", [&] { return error_cases(device, stream); });
  unsigned word = 0;
  ccglib_b200_device_status(&word);
  std::printf("%s device_status_clean\n", word == 0 ? "PASS" : "FAIL");
  failures += word != 0;
  std::printf("%d failure(s)\n", failures);
  return failures;
}
