// The sum of a K split's partials with the linear's epilogue, where the decode GEMV's own blocks do not join them: calls
// without counters, or of more column tiles than there are (N past 128 K). One pass over S M N floats, 16 bytes per load.
#include "epi.h"
#include "host.h"
#include "kernels.h"

namespace ifd {

__global__ __launch_bounds__(256) void k_splitk_epi(const float* __restrict__ part, int S, int M, int N, Epi e, void* C,
                                                    int ldc) {
  const int pn = epi_part_row(N);
  const size_t mn = (size_t)M * pn, i = 4 * ((size_t)blockIdx.x * 256 + threadIdx.x);
  if (i >= mn) return;
  const int m = (int)(i / pn), n = (int)(i % pn);
  float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int z = 0; z < S; z++) {
    const float4 x = *(const float4*)(part + z * mn + i);
    v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w;
  }
  epi_store(e, C, (size_t)m * ldc + n, m, n, N - n, v);
}

int launch_splitk_epi(const float* part, int S, int M, int N, const Epi& e, void* C, int ldc, hipStream_t st) {
  const size_t n = (size_t)M * epi_part_row(N) / 4;
  if (n == 0) return IFD_OK;
  hipLaunchKernelGGL(k_splitk_epi, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, part, S, M, N, e, C, ldc);
  return check_launch("split-K epilogue");
}

}  // namespace ifd
