// Rows of activations as e4m3 codes with a power-of-two scale per 128 elements: codes [rows][KB * 128] (zeros past K), scales [KB][rows].
//
// Bound: memory; 4096 x 14336 bf16 in 32 us, 5.6 TB/s of the 6.5 that a copy reaches (27 us).  Sixteen lanes take a block, eight elements each: 16-byte loads, a maximum of bit patterns over the half-warp, 8-byte stores.  A warp has IT
// such pairs of blocks of a row under way, and eight CTAs share an SM.  The warps of eight neighbouring rows lie side by side, so that their scales, four bytes each, share a sector.
#include "act.cuh"
#include "common.cuh"
#include "fp8.cuh"
#include "host_util.h"

namespace mx {

struct Fp8RowsParams {
  const void* x;
  long long ldx;
  const int* index;
  int x_rows, rows, K, kb, chunks;       // chunks: runs of 2 IT blocks in a row
  uint8_t* codes;
  float* scale;
};

// VEC: rows start on 16 bytes
template <typename T, int IT, bool VEC>
__global__ void __launch_bounds__(256, VEC && sizeof(T) == 2 ? 8 : 4) fp8_rows_kernel(const Fp8RowsParams p) {
  pdl_prologue();
  const int lane = threadIdx.x & 31, half = lane >> 4, sub = lane & 15;
  const int unit = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int g = unit / (8 * p.chunks), i = unit - g * 8 * p.chunks, n = min(8, p.rows - g * 8);
  if (n <= 0) return;
  const int chunk = i / n, r = g * 8 + i - chunk * n;
  if (chunk >= p.chunks) return;
  const int src = p.index ? p.index[r] : r;
  const bool some = src >= 0 && src < p.x_rows;
  const T* row = (const T*)p.x + (some ? src : 0) * p.ldx;
  const int b0 = chunk * 2 * IT + half, at0 = b0 * FP8_BLOCK + 8 * sub;
  Row8<T> v[IT];
  if (VEC) {
#pragma unroll
    for (int t = 0; t < IT; ++t) v[t].load(row + (at0 + t * 2 * FP8_BLOCK + 8 <= p.K ? at0 + t * 2 * FP8_BLOCK : 0));      // (K is 8 at least)
  }
  if (!VEC || !some || (chunk + 1) * 2 * IT * FP8_BLOCK > p.K) {                // the row's last run, or no row
#pragma unroll
    for (int t = 0; t < IT; ++t) {
      const int at = at0 + t * 2 * FP8_BLOCK;
      if (VEC && some && at + 8 <= p.K) continue;
      v[t].zero();
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (some && at + j < p.K) v[t].put(j, row[at + j]);
    }
  }
  uint32_t m[IT];
#pragma unroll
  for (int t = 0; t < IT; ++t) m[t] = v[t].top();
  half_warp_max<IT>(m, T());
#pragma unroll
  for (int t = 0; t < IT; ++t) {
    const int b = b0 + 2 * t;
    if (src >= p.x_rows) m[t] = 0x7fc00000u;               // no such row: NaN
    float inv;
    const float s = fp8_scale(__uint_as_float(m[t]), &inv);
    const uint2 w = m[t] < 0x7f800000u ? v[t].codes(inv) : make_uint2(0, 0);
    if (b < p.kb) {
      *reinterpret_cast<uint2*>(p.codes + ((size_t)r * p.kb + b) * FP8_BLOCK + 8 * sub) = w;
      if (sub == 0) p.scale[(size_t)b * p.rows + r] = s;
    }
  }
}

template <typename T> static int launch_rows(Fp8RowsParams p, cudaStream_t st) {
  const bool vec = p.x_rows > 0 && p.K >= 8 && p.ldx * (long long)sizeof(T) % 16 == 0 && ((uintptr_t)p.x & 15) == 0;
  // pairs of blocks per warp: four where that leaves the SMs eight warps each, one for the few rows of a decode step
  const bool many = (long long)p.rows * p.kb >= 8ll * 8 * sm_count();
  const int per = many ? 8 : 2;
  p.chunks = (p.kb + per - 1) / per;
  const long long ctas = ((long long)p.rows * p.chunks + 7) / 8;
  if (ctas >= 1ll << 28) return -106;
  const dim3 grid((unsigned)ctas);
  if (many) { if (vec) launch_pdl(fp8_rows_kernel<T, 4, true>, grid, dim3(256), 0, st, p); else launch_pdl(fp8_rows_kernel<T, 4, false>, grid, dim3(256), 0, st, p); }
  else { if (vec) launch_pdl(fp8_rows_kernel<T, 1, true>, grid, dim3(256), 0, st, p); else launch_pdl(fp8_rows_kernel<T, 1, false>, grid, dim3(256), 0, st, p); }
  return (int)cudaGetLastError();
}

// x: bf16 (f32 = 0) or fp32 rows, `ldx` elements apart, K of them used; index: row r of the result is row index[r] of x (negative: zeros; past the end: NaN).
int fp8_rows_launch(const void* x, int f32, long long ldx, const int* index, int x_rows, int rows, int K, void* codes, float* scale, cudaStream_t st) {
  if (rows <= 0) return 0;
  if (K < 1 || x_rows < 0) return -101;
  if (((uintptr_t)codes) & 15) return -114;
  Fp8RowsParams p{x, ldx, index, x_rows, rows, K, (K + FP8_BLOCK - 1) / FP8_BLOCK, 0, (uint8_t*)codes, scale};
  return f32 ? launch_rows<float>(p, st) : launch_rows<__nv_bfloat16>(p, st);
}

}  // namespace mx

MX_HOST_API int mx_fp8_rows(const void* x, int f32, long long ldx, const int* index, int x_rows, int rows, int K, void* codes, float* scale, cudaStream_t st) {
  return mx::fp8_rows_launch(x, f32, ldx, index, x_rows, rows, K, codes, scale, st);
}
