// Products of up to eight rows with e4m3 weights of a size where the latency of the launch counts more than reading them: a decode step's smaller layers, and the slots of a token.
//   y[m, n] = act(sum_b sx[b][m] sw[n / 16][b] sum_{k in b} x8[m][k] w8[n][k] + bias[n])
//
// Bound: latency, of the launch, of the rows and of one or two rounds of loads.  So nothing is set up: no boxes, barriers or accumulators outside of registers, and no sums that wait
// for another CTA in global memory.  A CTA takes 32 weight rows (16 gate and 16 up rows of a gated layer), its four warps every fourth block of K, and where that leaves SMs idle a
// cluster of 2, 4 or 8 CTAs shares the blocks: the first of them adds the sums, in their order.  1024 x 8192 takes 14.5 us without clusters and 5.0 with.  The weights go from
// global memory to registers in the layout of mma.m16n8k32: a lane's 16 bytes are four consecutive k of four steps, the rows' codes in shared memory are read the same way, and the
// order of k within a block is free.  (On B200 these products take a tenth of the time: tcgen05 has them faster, but its accumulators come back through two more waits.)  Every
// CTA rounds the blocks of the rows that it needs itself.  The first weights are on their way to L2 before the launch before has ended.
// Measured in a graph of calls over more weights than L2 holds, us, with the streaming kernel in brackets: 1 x 512 x 2048 3.3 (5.3), 1 x 1024 x 8192 5.4 (7.9), 1 x 5120 x 2880 6.7 (9.1), 1 x 12288 x 2048 8.6
// (9.6); gated slots, 10 of 512 of 1024 x 2048, 7.9 (9.0).  One layer again and again, its weights in L2: 3.2 (5.5), 4.7 (7.7), 5.9 (8.7), 6.3 (9.0) and 7.4 (8.3).
#include "act.cuh"
#include "cluster.cuh"
#include "common.cuh"
#include "fp8.cuh"
#include "host_util.h"

namespace mx {

constexpr int FV_WARPS = 4, FV_THREADS = FV_WARPS * 32, FV_CTAS = 4, FV_ROWS = 8;     // a CTA's warps, CTAs of an SM, most rows of x
constexpr int FV_BLOCKS = 64;                    // rounded blocks of rows that a CTA keeps, at most
constexpr int FV_MAX_CUTS = 8;

__host__ __device__ inline int fv_pitch(int blocks) { return blocks * FP8_BLOCK + 64; }      // (eight lanes read two rows: different banks)

__device__ __forceinline__ void mma_e4m3(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

constexpr int MT = 2;                            // runs of 16 weight rows of a CTA: gate and up rows, or neighbours
__global__ void __launch_bounds__(FV_THREADS, FV_CTAS) fp8_gemv_kernel(const Fp8Params p) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  __shared__ __align__(16) float s_red[FV_WARPS][MT * 16][FV_ROWS];
  __shared__ float s_join[FV_MAX_CUTS - 1][MT][FV_THREADS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  const int cuts = p.cuts, cut = cuts > 1 ? (int)cluster_rank() : 0, it = cuts > 1 ? blockIdx.x / cuts : blockIdx.x;
  const int first = (int)((long long)p.kb * cut / cuts), end = (int)((long long)p.kb * (cut + 1) / cuts), blocks = end - first;
  const int rows = p.slot ? 1 : p.M, pitch = fv_pitch((p.kb + cuts - 1) / cuts), groups = (p.N + 16 * MT - 1) / (16 * MT), sw_groups = (p.N + FP8_ROWS - 1) / FP8_ROWS;
  uint8_t* const codes = smem_raw;
  float* const s_sx = reinterpret_cast<float*>(smem_raw + rows * pitch);         // [blocks][FV_ROWS]
  const int s = it / groups, n0 = (it - s * groups) * 16 * MT;                   // (dense: s = 0)
  const size_t row_bytes = (size_t)p.kb * FP8_BLOCK;
  if (cuts > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;");         // (memory of the first CTA is written once it runs)
  if (!p.slot) {                                                                 // (which experts are read the launch before may say)
    const int lines = min(16 * MT, p.N - n0) * blocks;
    const uint8_t* at = p.w + n0 * row_bytes + first * FP8_BLOCK;
    for (int i = tid; i < lines; i += FV_THREADS) {
      const int r = i / blocks;
      asm volatile("prefetch.global.L2 [%0];" ::"l"(at + r * row_bytes + (i - r * blocks) * FP8_BLOCK));
    }
  }
  pdl_wait();
  const int e = p.slot ? p.slot[s] - p.e_lo : 0, x0 = p.slot ? s / p.x_div : 0;
  const bool owned = e >= 0 && e < p.E;
  const int ee = min(max(e, 0), p.E - 1);

  // ---- this CTA's blocks of the rows, as codes
  if (p.xb) {
    constexpr int RB = 2;                                                        // pairs of blocks of a warp that are loaded together
    const int half = lane >> 4, sub = lane & 15, pairs = (blocks + 1) / 2 * rows;
    for (int j0 = warp * RB; j0 < pairs; j0 += FV_WARPS * RB) {
      Row8<__nv_bfloat16> v[RB];
      uint32_t m[RB];
      int b[RB], r[RB];
#pragma unroll
      for (int j = 0; j < RB; ++j) {
        const int i = min(j0 + j, pairs - 1), pair = i / rows;
        r[j] = i - pair * rows;
        b[j] = 2 * pair + half;
        const int at = (first + b[j]) * FP8_BLOCK + 8 * sub;
        const __nv_bfloat16* row = p.xb + (long long)(x0 + r[j]) * p.ldx;
        v[j].load(row + (at + 8 <= p.K ? at : 0));                               // (K is 8 at least)
        if (at + 8 > p.K) {
          v[j].zero();
#pragma unroll
          for (int c = 0; c < 8; ++c)
            if (at + c < p.K) v[j].put(c, row[at + c]);
        }
      }
#pragma unroll
      for (int j = 0; j < RB; ++j) m[j] = v[j].top();
      half_warp_max<RB>(m, __nv_bfloat16());
#pragma unroll
      for (int j = 0; j < RB; ++j) {
        if (j0 + j >= pairs || b[j] >= blocks) continue;
        float inv;
        const float sc = fp8_scale(__uint_as_float(m[j]), &inv);
        *reinterpret_cast<uint2*>(codes + r[j] * pitch + b[j] * FP8_BLOCK + 8 * sub) = m[j] < 0x7f800000u ? v[j].codes(inv) : make_uint2(0, 0);
        if (sub == 0) s_sx[b[j] * FV_ROWS + r[j]] = sc;
      }
    }
  } else {                                                                       // rounded before
    const int runs = blocks * (FP8_BLOCK / 16);
    for (int i = tid; i < runs * rows; i += FV_THREADS) {
      const int r = i / runs, c = i - r * runs;
      *reinterpret_cast<uint4*>(codes + r * pitch + c * 16) = __ldg(reinterpret_cast<const uint4*>(p.xc + (size_t)(x0 + r) * row_bytes + first * FP8_BLOCK) + c);
    }
    for (int i = tid; i < blocks * rows; i += FV_THREADS) {
      const int b = i / rows, r = i - b * rows;
      s_sx[b * FV_ROWS + r] = p.sx[(size_t)(first + b) * p.x_rows + x0 + r];
    }
  }
  __syncthreads();

  // ---- the products: rows g and g + 8 of each run, columns 2 t4 and 2 t4 + 1 of x's rows
  float tot[MT][4];
  const uint8_t* wr[MT][2];
  const float* swp[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
    for (int i = 0; i < 4; ++i) tot[mt][i] = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) wr[mt][h] = p.w + ((size_t)ee * p.N + min(n0 + mt * 16 + h * 8 + g, p.N - 1)) * row_bytes + first * FP8_BLOCK + t4 * 16;
    swp[mt] = p.sw + ((size_t)ee * sw_groups + min(n0 / 16 + mt, sw_groups - 1)) * p.kb + first;
  }
  const uint8_t* xr = codes + min(g, rows - 1) * pitch + t4 * 16;                // (columns past the rows repeat the last one)
  for (int b = warp; b < blocks; b += FV_WARPS) {
    uint4 a[MT][2][2];                                                           // half of the rows, half of the block
    float sw[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int k = 0; k < 2; ++k) a[mt][h][k] = __ldcs(reinterpret_cast<const uint4*>(wr[mt][h] + (size_t)b * FP8_BLOCK + k * 64));
      sw[mt] = __ldg(swp[mt] + b);
    }
    const uint4 x0v = *reinterpret_cast<const uint4*>(xr + b * FP8_BLOCK), x1v = *reinterpret_cast<const uint4*>(xr + b * FP8_BLOCK + 64);
    const float2 sx = *reinterpret_cast<const float2*>(s_sx + b * FV_ROWS + 2 * t4);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float d[4] = {0.f, 0.f, 0.f, 0.f};
      const uint4(&w)[2][2] = a[mt];
      mma_e4m3(d, w[0][0].x, w[1][0].x, w[0][0].y, w[1][0].y, x0v.x, x0v.y);
      mma_e4m3(d, w[0][0].z, w[1][0].z, w[0][0].w, w[1][0].w, x0v.z, x0v.w);
      mma_e4m3(d, w[0][1].x, w[1][1].x, w[0][1].y, w[1][1].y, x1v.x, x1v.y);
      mma_e4m3(d, w[0][1].z, w[1][1].z, w[0][1].w, w[1][1].w, x1v.z, x1v.w);
      const float s0 = sw[mt] * sx.x, s1 = sw[mt] * sx.y;
      tot[mt][0] = fmaf(d[0], s0, tot[mt][0]); tot[mt][1] = fmaf(d[1], s1, tot[mt][1]);
      tot[mt][2] = fmaf(d[2], s0, tot[mt][2]); tot[mt][3] = fmaf(d[3], s1, tot[mt][3]);
    }
  }

  pdl_launch_dependents();                                                       // (earlier, the next layers' CTAs wait where this one's loads are wanted)

  // ---- the warps' sums, joined in their order, then those of the cluster's CTAs in theirs, and the epilogue: a thread has row r of each run and row m of x
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int h = 0; h < 2; ++h) *reinterpret_cast<float2*>(&s_red[warp][mt * 16 + h * 8 + g][2 * t4]) = make_float2(tot[mt][2 * h], tot[mt][2 * h + 1]);
  __syncthreads();
  const int r = tid & 15, m = tid >> 4;
  float v[2] = {0.f, 0.f};
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int w = 0; w < FV_WARPS; ++w) v[mt] += s_red[w][mt * 16 + r][m];
  if (cuts > 1) {
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (cut) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) cluster_st(smem_u32(&s_join[cut - 1][mt][tid]), 0, v[mt]);
    }
    cluster_sync_all();
    if (cut) return;
    for (int c = 0; c < cuts - 1; ++c)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) v[mt] += s_join[c][mt][tid];
  }
  if (m >= rows) return;
  const int out_row = p.slot ? s : m;
  const bool gated = act_gated(p.act);
  if (p.bias) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
      if (n0 + mt * 16 + r < p.N) v[mt] += p.bias[(size_t)ee * p.N + n0 + mt * 16 + r];
  }
  if (gated) glu_run<1>(p.act, v, p.act_alpha, p.act_limit);
  const float scale = p.row_scale ? p.row_scale[out_row] : 1.f;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    if (gated && mt) break;
    float y = v[mt];
    if (!gated && p.act) y = act_unary<false, true>(p.act, y, p.act_alpha, p.act_limit);
    if (p.row_scale) y *= scale;
    if (!owned) y = 0.f;
    const int o = (gated ? n0 / 2 : n0 + mt * 16) + r;
    if (o >= (gated ? p.N / 2 : p.N)) continue;
    if (p.out_f32) ((float*)p.C)[out_row * p.ldc + o] = y;
    else ((__nv_bfloat16*)p.C)[out_row * p.ldc + o] = __float2bfloat16(y);
  }
}

// Pieces along K and bytes of rounded rows; no cuts: left to the streaming kernel, which has the memory busier once it runs.  In a model's chain of launches that kernel fills its
// rings with weights under the launch before, so long rows want a smaller limit than calls in a loop show.  Decode of one token, ms with the streaming kernel -> with these
// limits: Qwen3-MoE-30B's shape 3.64 -> 3.12, Qwen3-Next's 4.75 -> 3.98, gpt-oss-20b's 2.71 -> 2.58; Llama-3-8B's (K = 4096, layers of 4096 blocks and up) 2.95 -> 3.21 if it
// took them, so it does not.  The border between the limits lies at 24 blocks of K.  It was looked for in 24 layers of a llama of hidden size H (K of the layers but the last of
// each, whose rows are 3.5 H long), ms a token with the small limit for every K -> the large one: H of 20 blocks 1.56 -> 1.50, 26 2.27 -> 2.22, 28 1.93 -> 1.94 to 2.19, 30 2.11 ->
// 2.33, 32 2.15 -> 2.37.
// With more rows the rounding that every CTA does again counts, us: 4 x 5120 x 2880 10.3 -> 7.8, 8 x 1024 x 8192 9.8 -> 7.5, but 4 x 6144 x 4096 9.9 -> 11.2, 4 x 2048 x 14336
// 10.3 -> 11.5.  CTAs past a wave: slots, 10 x 2048 x 512 (640 CTAs, 592 at a time) 8.2 -> 6.8, 16 x 2048 x 768 (1024) 6.5 -> 9.5.  Pieces are powers of two and leave an eighth
// of the SMs' room: clusters of three that would have filled it (576 CTAs) waited for a place and took twice the time.
struct GemvPlan { int cuts, smem; long long items; };
static GemvPlan gemv_plan(const Fp8Call& c) {
  GemvPlan g{};
  if (c.nt != 16 || c.counts || c.index || (!c.slot && c.M > FV_ROWS)) return g;
  const int kb = (c.K + FP8_BLOCK - 1) / FP8_BLOCK, rows = c.slot ? 1 : c.M;
  const long long wave = (long long)FV_CTAS * sm_count();
  g.items = (c.slot ? (long long)c.M : 1) * ((c.N + 16 * MT - 1) / (16 * MT));
  const long long most = c.slot || kb <= 24 ? 8192 : 3000;
  if (g.items * kb > most || rows * g.items * kb > 2 * 8192 || 4 * g.items > 5 * wave) return g;
  int cuts = 1;
  while (cuts < FV_MAX_CUTS && 16 * cuts * g.items <= 7 * wave && 2 * cuts * FV_WARPS <= kb) cuts *= 2;
  const int blocks = (kb + cuts - 1) / cuts;
  if (rows * blocks > FV_BLOCKS) return g;
  g.smem = rows * fv_pitch(blocks) + blocks * FV_ROWS * 4;
  g.cuts = cuts;
  return g;
}
bool fp8_gemv_takes(const Fp8Call& c) { return gemv_plan(c).cuts > 0; }
// whether the kernel rounds bf16 rows itself: 16-byte runs of at least eight
bool fp8_gemv_rounds(const Fp8Call& c) { return c.xb && c.K >= 8 && c.ldx % 8 == 0 && ((uintptr_t)c.xb & 15) == 0; }

int fp8_gemv_launch(const Fp8Call& c, bool round, cudaStream_t st) {
  const GemvPlan g = gemv_plan(c);
  Fp8Params p = fp8_params(c);
  if (((uintptr_t)c.w | (uintptr_t)c.codes) & 15) return -114;
  if (round) { p.xb = (const __nv_bfloat16*)c.xb; p.ldx = c.ldx; }
  p.xc = (const uint8_t*)c.codes;
  p.w = (const uint8_t*)c.w;
  p.cuts = g.cuts;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(g.items * g.cuts)); cfg.blockDim = dim3(FV_THREADS); cfg.dynamicSmemBytes = g.smem; cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = g.cuts; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr; cfg.numAttrs = g.cuts > 1 ? 2 : 1;
  return (int)cudaLaunchKernelEx(&cfg, fp8_gemv_kernel, p);
}

}  // namespace mx
