// The sum of a K split's partials with the linear's epilogue, where the GEMM's own blocks do not join them: rows whose
// length is no multiple of four in the decode GEMV. One pass over S M N floats of at most 16 rows: a launch bounds it.
#include "epi.h"
#include "host.h"
#include "kernels.h"

namespace ifd {

__global__ __launch_bounds__(256) void k_splitk_epi(const float* __restrict__ part, int S, int M, int N, Epi e, void* C,
                                                    int ldc) {
  const size_t mn = (size_t)M * N, i = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= mn) return;
  const int m = (int)(i / N), n = (int)(i % N);
  float v[1] = {0.f};
  for (int z = 0; z < S; z++) v[0] += part[z * mn + i];
  epi_store(e, C, (size_t)m * ldc + n, m, n, 1, v);
}

int launch_splitk_epi(const float* part, int S, int M, int N, const Epi& e, void* C, int ldc, hipStream_t st) {
  const size_t n = (size_t)M * N;
  if (n == 0) return IFD_OK;
  hipLaunchKernelGGL(k_splitk_epi, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, part, S, M, N, e, C, ldc);
  return check_launch("split-K epilogue");
}

}  // namespace ifd
