// Rows of activations as e4m3 codes with a power-of-two scale per 128 elements: codes [rows][KB * 128] (zeros past K), scales [KB][rows].
//
// Bound: memory.  A warp takes a block of a row, a lane four elements of it; the largest magnitude is a maximum of bit patterns over the warp.
#include "act.cuh"
#include "common.cuh"
#include "fp8.cuh"
#include "host_util.h"

namespace mx {

template <typename T>
__global__ void __launch_bounds__(256) fp8_rows_kernel(const T* __restrict__ x, long long ldx, const int* __restrict__ index, int x_rows, int rows, int K, int kb,
                                                       uint8_t* __restrict__ codes, float* __restrict__ scale) {
  pdl_prologue();
  const int lane = threadIdx.x & 31;
  const long long unit = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (unit >= (long long)rows * kb) return;
  const int r = (int)(unit / kb), b = (int)(unit - (long long)r * kb);
  const int src = index ? index[r] : r;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  if (src >= 0 && src < x_rows) {
    const T* p = x + src * ldx + b * FP8_BLOCK;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (b * FP8_BLOCK + 4 * lane + i < K) v[i] = to_f32<T>(p[4 * lane + i]);
  }
  uint32_t m = max(max(fp8_mag(v[0]), fp8_mag(v[1])), max(fp8_mag(v[2]), fp8_mag(v[3])));
  m = __reduce_max_sync(0xffffffffu, m);
  if (src >= x_rows) m = 0x7fc00000u;
  float inv;
  const float s = fp8_scale(__uint_as_float(m), &inv);
  const uint32_t word = m >= 0x7f800000u ? 0u : fp8_pack4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
  *reinterpret_cast<uint32_t*>(codes + ((size_t)r * kb + b) * FP8_BLOCK + 4 * lane) = word;
  if (lane == 0) scale[(size_t)b * rows + r] = s;
}

}  // namespace mx

using namespace mx;

// x: bf16 (f32 = 0) or fp32 rows, `ldx` elements apart, K of them used; index: row r of the result is row index[r] of x (negative: zeros; past the end: NaN).
MX_HOST_API int mx_fp8_rows(const void* x, int f32, long long ldx, const int* index, int x_rows, int rows, int K, void* codes, float* scale, cudaStream_t st) {
  if (rows <= 0) return 0;
  if (K < 1 || x_rows < 0) return -101;
  if (((uintptr_t)codes) & 15) return -114;
  const int kb = (K + FP8_BLOCK - 1) / FP8_BLOCK;
  const long long ctas = ((long long)rows * kb + 7) / 8;
  if (ctas > 0x7fffffffll) return -106;
  if (f32) launch_pdl(fp8_rows_kernel<float>, dim3((unsigned)ctas), dim3(256), 0, st, (const float*)x, ldx, index, x_rows, rows, K, kb, (uint8_t*)codes, scale);
  else launch_pdl(fp8_rows_kernel<__nv_bfloat16>, dim3((unsigned)ctas), dim3(256), 0, st, (const __nv_bfloat16*)x, ldx, index, x_rows, rows, K, kb, (uint8_t*)codes, scale);
  return (int)cudaGetLastError();
}
