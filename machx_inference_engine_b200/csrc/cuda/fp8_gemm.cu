// Products of e4m3 rows with e4m3 weights, both with scales per 128 elements of K:
//   y[m, n] = act(sum_b sx[b][m] sw[n / 16][b] sum_{k in b} x8[m][k] w8[n][k] + bias[n])
// for dense layers, rows sorted by expert, and slots of one row and one expert.
//
// The plainest form: tiles of 32 x 32 outputs, fp32 multiplications of decoded codes, a block of K at a time.
#include "act.cuh"
#include "common.cuh"
#include "fp8.cuh"
#include "host_util.h"

namespace mx {

struct Fp8Params {
  const uint8_t* x;          // [rows][kb * 128]
  const float* sx;           // [kb][x_rows]
  const uint8_t* w;          // [E][N][kb * 128]
  const float* sw;           // [E][ceil(N / 16)][kb]
  void* C;
  long long ldc;
  int out_f32, M, N, kb, x_rows, E;
  const float* bias;         // [N] or [E][N]
  const float* row_scale;    // [M]
  int act;
  float act_alpha, act_limit;
  const int* seg;            // experts: first packed row of expert e_lo + i, and how many
  const int* counts;
  const int* slot;           // slots: expert of output row m, whose input is row m / x_div
  int x_div, e_lo;
};

__global__ void __launch_bounds__(256) fp8_gemm_kernel(const Fp8Params p) {
  __shared__ float sa[32][FP8_BLOCK + 1], sb[32][FP8_BLOCK + 1], so[32][33];
  __shared__ int s_tile[3];
  pdl_prologue();
  const int tid = threadIdx.x, n0 = blockIdx.x * 32;
  if (tid == 0) {
    int e = 0, row0 = blockIdx.y * 32, rows = min(32, p.M - row0);
    if (p.slot) {
      row0 = blockIdx.y; rows = 1;
      e = p.slot[row0] - p.e_lo;
    } else if (p.seg) {
      int t = blockIdx.y;
      rows = 0;
      for (e = 0; e < p.E; ++e) {
        const int c = p.counts[e], tiles = (c + 31) / 32;
        if (t < tiles) { row0 = p.seg[e] + t * 32; rows = min(32, c - t * 32); break; }
        t -= tiles;
      }
      rows = min(rows, p.M - row0);
    }
    s_tile[0] = e; s_tile[1] = row0; s_tile[2] = rows;
  }
  __syncthreads();
  const int e = s_tile[0], row0 = s_tile[1], rows = s_tile[2];
  if (rows <= 0) return;
  const bool owned = e >= 0 && e < p.E;
  const int r = tid >> 3, c = tid & 7, groups = (p.N + FP8_ROWS - 1) / FP8_ROWS;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  auto in_row = [&](int i) { return p.slot ? (row0 + i) / p.x_div : row0 + i; };
  for (int b = 0; b < p.kb && owned; ++b) {
    __syncthreads();
    for (int i = tid; i < 32 * FP8_BLOCK; i += 256) {
      const int rr = i >> 7, k = i & 127;
      __nv_fp8_e4m3 v;
      v.__x = rr < rows ? p.x[(size_t)in_row(rr) * p.kb * FP8_BLOCK + b * FP8_BLOCK + k] : 0;
      sa[rr][k] = float(v);
      v.__x = n0 + rr < p.N ? p.w[((size_t)e * p.N + n0 + rr) * p.kb * FP8_BLOCK + b * FP8_BLOCK + k] : 0;
      sb[rr][k] = float(v);
    }
    __syncthreads();
    if (r < rows) {
      const float sx = p.sx[(size_t)b * p.x_rows + in_row(r)];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = n0 + c + 8 * j;
        if (n >= p.N) continue;
        float d = 0.f;
        for (int k = 0; k < FP8_BLOCK; ++k) d = fmaf(sa[r][k], sb[c + 8 * j][k], d);
        acc[j] = fmaf(d, sx * p.sw[((size_t)e * groups + n / FP8_ROWS) * p.kb + b], acc[j]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int n = n0 + c + 8 * j;
    so[r][c + 8 * j] = acc[j] + (p.bias && owned && n < p.N ? p.bias[(size_t)e * p.N + n] : 0.f);
  }
  __syncthreads();
  if (r >= rows) return;
  const bool gated = act_gated(p.act);
  const float rs = owned ? (p.row_scale ? p.row_scale[row0 + r] : 1.f) : 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int i = c + 8 * j;
    float v = so[r][i];
    int o = n0 + i, on = p.N;
    if (gated) {
      if (i >= 16) continue;
      v = glu_apply(p.act, v, so[r][16 + i], p.act_alpha, p.act_limit);
      o = n0 / 2 + i; on = p.N / 2;
    } else {
      v = act_unary<false>(p.act, v, p.act_alpha, p.act_limit);
    }
    if (o >= on) continue;
    v = owned ? v * rs : 0.f;
    if (p.out_f32) ((float*)p.C)[(row0 + r) * p.ldc + o] = v;
    else ((__nv_bfloat16*)p.C)[(row0 + r) * p.ldc + o] = __float2bfloat16(v);
  }
}

}  // namespace mx

using namespace mx;

// M rows of output (dense: rows of x; experts: rows of the packing; slots: slots).  counts / seg: those of the bank's first expert on.
MX_HOST_API int mx_fp8_gemm(const void* x, const float* sx, int x_rows, const void* w, const float* sw, int E, void* c, long long ldc, int out_f32, const float* bias,
                            const float* row_scale, int act, float act_alpha, float act_limit, int M, int N, int kb, const int* counts, const int* seg, const int* slot,
                            int x_div, int e_lo, cudaStream_t st) {
  if (M <= 0 || N <= 0) return 0;
  if (kb < 1 || x_div < 1 || E < 1) return -101;
  if (act_gated(act) && N % 32) return -104;
  Fp8Params p{(const uint8_t*)x, sx, (const uint8_t*)w, sw, c, ldc, out_f32, M, N, kb, x_rows, E, bias, row_scale, act, act_alpha, act_limit, seg, counts, slot, x_div, e_lo};
  const int tiles = slot ? M : (M + 31) / 32 + (seg ? (E < M ? E : M) : 0);
  if (tiles > 65535) return -106;
  launch_pdl(fp8_gemm_kernel, dim3((N + 31) / 32, tiles), dim3(256), 0, st, p);
  return (int)cudaGetLastError();
}
