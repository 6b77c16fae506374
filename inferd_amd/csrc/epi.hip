// The epilogue of a linear as a pass of its own over the fp32 product in the workspace.
#include "epi.h"
#include "host.h"
#include "kernels.h"

namespace ifd {

__global__ __launch_bounds__(256) void k_epi(const float* __restrict__ y, int M, int N, Epi e, void* C, int ldc,
                                             int out_f32) {
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (size_t)M * N) return;
  const int m = (int)(i / N), n = (int)(i % N);
  float v = y[i];
  if (e.bias) v += bf2f(e.bias[n]);
  v = epi_act(v, e.act);
  if (e.res) v += bf2f(e.res[(size_t)m * e.ldr + n]);
  store_mode(C, (size_t)m * ldc + n, v, out_f32 ? 2 : 0);
}

int launch_epi(const float* y, int M, int N, const Epi& e, void* C, int ldc, int out_f32, hipStream_t st) {
  const size_t n = (size_t)M * N;
  if (n == 0) return IFD_OK;
  if ((n + 255) / 256 > 0x7fffffffu) return fail(IFD_ERR_UNSUPPORTED, "epilogue: %d x %d is too large", M, N);
  hipLaunchKernelGGL(k_epi, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, y, M, N, e, C, ldc, out_f32);
  return check_launch("epilogue");
}

}  // namespace ifd
