// Products of many e4m3 rows with e4m3 weights, scales per 128 elements of K on both sides, on the tensor cores:
//   y[m, n] = act(sum_b sx[b][m] sw[n / 16][b] sum_{k in b} x8[m][k] w8[n][k] + bias[n])
// for dense layers and for rows sorted by expert.
//
// A block of K is one stage: 128 rows of x and BN of w, 128 bytes each, and four tcgen05.mma of K = 32.  Its sums have a scale of their own, so they cannot
// stay in TMEM: sixteen warps read each block's 128 x BN sums and add s_x s_w times them to fp32 sums in registers, BN / 4 columns of a row per thread, while the
// tensor cores fill the next accumulator.
//   warp 0      TMA loads into a ring of NST stages
//   warp 1      tcgen05.mma from one thread into a ring of 512 / BN accumulators
//   warps 2, 3  asynchronous copies of the block's scales (128 of the rows, BN / 16 of the weights) into a ring.  Loads into registers would be waited for one block
//               ahead at most, whatever the distance: they share the counters by which a warp waits
//   warps 4-19  sums (warp & 3: rows, warp / 4 - 1: quarter of the columns); a finished tile goes through shared memory, so that rows are written in runs of 64 or 128 bytes
// A dense product with fewer tiles than SMs is cut along K: the pieces of a tile leave fp32 sums, and the warp that arrives last adds them in the order of the pieces.
//
// What bounds it is the way from L2 to shared memory, about 60 bytes a cycle and SM, and for long prompts the power cap.  A block of a 128 x 256 tile is 48 KB for 512 cycles of
// products and takes 860; of 128 x 128, 32 KB for 256 cycles, 630.  Without the products a block takes no less; without the loads it takes 540 (256 columns).  Tiles of 256 x
// 256 on pairs of SMs load a third less and were built: with room for two blocks' sums the signals between the CTAs took what was saved (423 to 500 ns a block, this
// kernel 455), and under the power cap 4096 x 28672 x 4096 took 574 us, this kernel 544.
// Measured, of rows that were rounded before: 4096 x 28672 x 4096 gated 494 us after a pause (1.95 PFLOP/s, 1.16 of the measured bf16 burst), 538 back to back under the power cap;
// 512 x 4096 x 14336 44 us back to back (1.38 PFLOP/s).  With the rounding 503, 560 and 52.
// Every mbarrier wait is bounded.
#include "act.cuh"
#include "common.cuh"
#include "fp8.cuh"
#include "host_util.h"

namespace mx {

constexpr int FG_BM = 128, FG_SUMS = 16, FG_THREADS = 128 + 32 * FG_SUMS, FG_MAX_E = 1024, FG_MAX_PIECES = 256;      // FG_SUMS: warps that hold sums
// m-tiles that are walked together under each column of tiles: as many as leave a band of x of 32 MB, which stays in L2 while w streams past it once per band.
// 4096 x 28672 x 4096 under the power cap: groups of 4, 8, 16 and all 32 m-tiles 643, 595, 586 and 572 us
__host__ __device__ inline int fg_group(int kb) { return kb >= 256 ? 8 : 2048 / kb; }

template <int BN, bool F32> struct Fp8GemmShape {
  static constexpr int A = FG_BM * FP8_BLOCK, B = BN * FP8_BLOCK, STAGE = A + B;
  static constexpr int ROW = BN == 128 && !F32 ? 64 : 128; // bytes of a staged row of a warp's outputs
  static constexpr int OUT = FG_SUMS * 32 * ROW;
  static constexpr int NST = BN == 256 ? 3 : F32 ? 4 : 5;
  static constexpr int ACC = 512 / BN;
  // A slot of scales is free again when the products of the block NST before are done, since they waited for the sums of the block ACC before them.
  static constexpr int RING = NST + ACC, SC = FG_BM + BN / FP8_ROWS;
  struct Small {                                           // what is not tiles, behind them
    alignas(16) float scale[RING][SC];
    uint64_t bar[2 * NST + 2 * ACC];
    int sum[FG_THREADS / 32];
    uint32_t tmem;
    int abort;
    uint16_t pre[FG_MAX_E + 1];                            // experts: m-tiles before expert i
  };
  static constexpr int SMEM = NST * STAGE + OUT + (int)sizeof(Small);
  static_assert(SMEM <= 227 * 1024, "shared memory of a block");
};

// KIND: 0 no activation, 1 gated, 2 element-wise.  The tile's end runs once per tile and is bound by fetching its instructions, so each instance has what it needs only.
template <int BN, int KIND, bool F32>
__global__ void __launch_bounds__(FG_THREADS, 1)
fp8_gemm_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w, const Fp8Params p) {
  using S = Fp8GemmShape<BN, F32>;
  constexpr int NST = S::NST, ACC = S::ACC;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  auto& small = *reinterpret_cast<typename S::Small*>(smem_raw + NST * S::STAGE + S::OUT);
  auto& s_bar = small.bar;
  auto& s_pre = small.pre;
  auto& s_sum = small.sum;
  uint32_t& s_tmem = small.tmem;
  int& s_abort = small.abort;
  const uint32_t base = smem_u32(smem_raw);
  if (base & 1023) {                                       // (swizzled tiles start on 1 KiB; no static shared memory lies before them)
    if (threadIdx.x == 0) atomicCAS(p.status, 0, ERR_BAD_ARGUMENT);
    return;
  }
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t bar_full = smem_u32(s_bar), bar_empty = bar_full + 8 * NST, bar_tfull = bar_empty + 8 * NST, bar_tempty = bar_tfull + 8 * ACC;
  volatile int* abort_flag = &s_abort;
  if (tid == 0) {
    for (int s = 0; s < NST; ++s) { mbar_init(bar_full + 8 * s, 1 + 64); mbar_init(bar_empty + 8 * s, 1); }
    for (int a = 0; a < ACC; ++a) { mbar_init(bar_tfull + 8 * a, 2); mbar_init(bar_tempty + 8 * a, FG_SUMS); }
    s_abort = 0;
    fence_mbar_init();
  }
  // tensor memory is taken when the launch before has ended: it may still want some, and would wait for a CTA that waits for it
  pdl_wait();
  if (warp == 1) { tmem_alloc(smem_u32(&s_tmem), 512); tmem_relinquish(); pdl_launch_dependents(); }

  // ---- tiles: dense in bands of m-tiles; experts one after the other, their m-tiles under each column of tiles
  const bool banked = p.counts != nullptr;
  const int n_tiles = (p.N + BN - 1) / BN;
  int m_tiles = (p.M + FG_BM - 1) / FG_BM;
  if (banked) {
    int run = 0;
    for (int e0 = 0; e0 < p.E; e0 += FG_THREADS) {
      const int e = e0 + tid;
      int incl = e < p.E ? (p.counts[e] + FG_BM - 1) / FG_BM : 0;
      const int mine = incl;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += u;
      }
      if (lane == 31) s_sum[warp] = incl;
      __syncthreads();
      int before = run;
#pragma unroll
      for (int w = 0; w < FG_THREADS / 32; ++w) {
        if (w < warp) before += s_sum[w];
        run += s_sum[w];
      }
      if (e < p.E) s_pre[e] = (uint16_t)(before + incl - mine);
      __syncthreads();
    }
    m_tiles = run;
    if (tid == 0) s_pre[p.E] = (uint16_t)run;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  const int cuts = p.cuts, tiles = m_tiles * n_tiles * cuts, sw_groups = (p.N + FP8_ROWS - 1) / FP8_ROWS;
  struct Tile { int e, row0, rows, nt, k0, k1; };        // and its blocks of K
  auto tile = [&](int t) {
    Tile r;
    const int piece = cuts > 1 ? t % cuts : 0;
    if (cuts > 1) t /= cuts;
    r.k0 = (int)((long long)p.kb * piece / cuts);
    r.k1 = (int)((long long)p.kb * (piece + 1) / cuts);
    if (banked) {
      int lo = 0, hi = p.E - 1;                            // the expert with s_pre * n_tiles <= t < the next one's
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (s_pre[mid] * n_tiles <= t) lo = mid; else hi = mid - 1;
      }
      const int i = t - s_pre[lo] * n_tiles, mt = s_pre[lo + 1] - s_pre[lo];
      r.e = lo;
      r.nt = i / mt;
      const int m = i - r.nt * mt;
      r.row0 = p.seg[lo] + m * FG_BM;
      r.rows = r.row0 < 0 ? 0 : min(min(FG_BM, p.counts[lo] - m * FG_BM), p.M - r.row0);
    } else {
      const int band = min(fg_group(p.kb), m_tiles), full = band * n_tiles, g = t / full, i = t - g * full, gm = min(band, m_tiles - g * band);
      r.e = 0;
      r.nt = i / gm;
      r.row0 = (g * band + i - r.nt * gm) * FG_BM;
      r.rows = min(FG_BM, p.M - r.row0);
    }
    return r;
  };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 32;");
    if (warp == 0 && lane == 0) {
      prefetch_tmap(&tm_x); prefetch_tmap(&tm_w);
      uint32_t s = 0, ph = 1;
      bool ok = true;
      for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
        const Tile at = tile(t);
        for (int k = at.k0; k < at.k1; ++k) {
          if (!(ok = mbar_wait(bar_empty + 8 * s, ph, p.status, ERR_MBAR_TIMEOUT_PRODUCER, abort_flag))) break;
          const uint32_t dst = base + s * S::STAGE;
          mbar_expect_tx(bar_full + 8 * s, S::STAGE);
          tma_load_2d(dst, &tm_x, bar_full + 8 * s, k * (FP8_BLOCK / 2), at.row0);
          tma_load_3d(dst + S::A, &tm_w, bar_full + 8 * s, k * (FP8_BLOCK / 2), at.nt * BN, at.e);
          if (++s == NST) { s = 0; ph ^= 1; }
        }
      }
    } else if (warp == 1) {
      const uint32_t leader = elect_one();
      constexpr uint32_t idesc = umma_idesc_e4m3(FG_BM, BN);
      uint32_t s = 0, ph = 0, a = 0, aph = 1;
      bool ok = true, data = false, room = false;
      for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
        const int piece = cuts > 1 ? t % cuts : 0, n = (int)((long long)p.kb * (piece + 1) / cuts) - (int)((long long)p.kb * piece / cuts);
        for (int k = 0; k < n; ++k) {
          if (!room && !(ok = mbar_wait(bar_tempty + 8 * a, aph, p.status, ERR_MBAR_TIMEOUT_MMA, abort_flag))) break;
          if (!data && !(ok = mbar_wait(bar_full + 8 * s, ph, p.status, ERR_MBAR_TIMEOUT_MMA, abort_flag))) break;
          __syncwarp();                                    // (no lane may miss a phase)
          tc_fence_after();
          const uint64_t dx = umma_desc_k_sw128(base + s * S::STAGE), dw = umma_desc_k_sw128(base + s * S::STAGE + S::A);
          const uint32_t d = tmem + a * BN, empty = bar_empty + 8 * s, tfull = bar_tfull + 8 * a;
          if (++s == NST) { s = 0; ph ^= 1; }
          if (++a == ACC) { a = 0; aph ^= 1; }
          data = mbar_peek(bar_full + 8 * s, ph);
          room = mbar_peek(bar_tempty + 8 * a, aph);
#pragma unroll
          for (int kk = 0; kk < FP8_BLOCK / 32; ++kk) umma_e4m3(leader, d, dx + 2 * kk, dw + 2 * kk, idesc, kk != 0);
          umma_commit_if(leader, empty);
          mbar_arrive_if(leader, tfull);                   // (what this thread has seen arrive, the scales among it, is seen by who waits here)
          umma_commit_if(leader, tfull);
        }
      }
    } else if (warp >= 2) {
      uint32_t s = 0, ph = 1, r = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
        const Tile at = tile(t);
        // warp 2: rows lane, lane + 32, ..; warp 3: runs of 16 weight rows.  What lies past the matrix has a neighbour's scale
        const float* from[4];
        if (warp == 2) {
#pragma unroll
          for (int i = 0; i < 4; ++i) from[i] = p.sx + min(max(at.row0, 0) + lane + 32 * i, p.x_rows - 1);
        } else {
          from[0] = p.sw + ((size_t)at.e * sw_groups + min(at.nt * (BN / FP8_ROWS) + lane, sw_groups - 1)) * p.kb;
        }
        for (int k = at.k0; k < at.k1; ++k) {
          if (!(ok = mbar_wait(bar_empty + 8 * s, ph, p.status, ERR_MBAR_TIMEOUT_PRODUCER, abort_flag))) break;
          const uint32_t to = smem_u32(small.scale[r]) + 4 * lane;
          if (warp == 2) {
#pragma unroll
            for (int i = 0; i < 4; ++i) copy4(to + 128 * i, from[i] + (size_t)k * p.x_rows);
          } else if (lane < BN / FP8_ROWS) {
            copy4(to + 4 * FG_BM, from[0] + k);
          }
          arrive_copies(bar_full + 8 * s);
          if (++s == NST) { s = 0; ph ^= 1; }
          if (++r == S::RING) r = 0;
        }
      }
    }
    __syncwarp();
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 112;");
    constexpr int HC = BN * 4 / FG_SUMS, G = HC / FP8_ROWS;          // columns of a thread, and the scales that they have
    const int q = warp & 3, part = (warp - 4) >> 2;
    constexpr int ESZ = F32 ? 4 : 2, PIECE = KIND == 1 ? 8 : 16;        // outputs of 16 sums
    constexpr int ROW_BYTES = HC * PIECE / 16 * ESZ;       // of a thread's outputs
    constexpr int PASSES = ROW_BYTES > S::ROW ? ROW_BYTES / S::ROW : 1, RB = ROW_BYTES / PASSES, CPR = RB / 16;
    static_assert(HC / 32 >= PASSES, "a pass has whole runs of 32 sums");
    uint8_t* const stage = smem_raw + NST * S::STAGE + (warp - 4) * (32 * S::ROW);
    // chunks of a staged row are turned so that those of eight rows lie in different banks
    static_assert(S::ROW == 128 || S::ROW == 64, "staged rows");
    auto turn = [](int r) { return S::ROW == 128 ? r & 7 : r >> 1 & 3; };
    const int on = KIND == 1 ? p.N >> 1 : p.N;
    const bool wide = (((uintptr_t)p.C) & 15) == 0 && (p.ldc * ESZ) % 16 == 0;
    uint32_t a = 0, aph = 0, ring = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
      const Tile at = tile(t);
      const int mine = q * 32 + lane, col0 = at.nt * BN + part * HC;
      float2 acc[HC / 2];
#pragma unroll
      for (int j = 0; j < HC / 2; ++j) acc[j] = make_float2(0.f, 0.f);
      for (int k = at.k0; k < at.k1; ++k) {
        if (!(ok = mbar_wait(bar_tfull + 8 * a, aph, p.status, ERR_MBAR_TIMEOUT_EPILOGUE, abort_flag))) break;
        tc_fence_after();
        const float sx = small.scale[ring][mine];
        const float* swp = &small.scale[ring][FG_BM + part * G];
        const uint32_t from = tmem + ((uint32_t)(q * 32) << 16) + a * BN + part * HC;
#pragma unroll
        for (int g = 0; g < G; g += 2) {
          uint32_t r[32];
          tmem_ld_cols<32>(from + 16 * g, r);
          const float2 sw = *reinterpret_cast<const float2*>(swp + g);
          const float s0 = sx * sw.x, s1 = sx * sw.y;
          tmem_ld_wait();
          if (g + 2 == G) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_tempty + 8 * a);
          }
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float sc = j < 8 ? s0 : s1;
            acc[8 * g + j] = fma2(make_float2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1])), make_float2(sc, sc), acc[8 * g + j]);
          }
        }
        if (++a == ACC) { a = 0; aph ^= 1; }
        if (++ring == S::RING) ring = 0;
      }
      if (!ok) break;

      if (cuts > 1) {
        const int w = warp - 4, own = t / cuts;
        auto slab = [&](int piece) { return reinterpret_cast<float4*>(p.part) + ((size_t)(own * cuts + piece) * FG_SUMS + w) * (HC / 4 * 32) + lane; };
        float4* to = slab(t - own * cuts);
#pragma unroll
        for (int j = 0; j < HC / 4; ++j) to[j * 32] = make_float4(acc[2 * j].x, acc[2 * j].y, acc[2 * j + 1].x, acc[2 * j + 1].y);
        if (!warp_arrives_last(p.tickets + own * FG_SUMS + w, cuts)) continue;
        const float4* from = slab(0);
#pragma unroll
        for (int j = 0; j < HC / 4; ++j) {
          const float4 v = __ldcg(from + j * 32);
          acc[2 * j] = make_float2(v.x, v.y); acc[2 * j + 1] = make_float2(v.z, v.w);
        }
        for (int piece = 1; piece < cuts; ++piece) {
          from = slab(piece);
#pragma unroll
          for (int j = 0; j < HC / 4; ++j) {
            const float4 v = __ldcg(from + j * 32);
            acc[2 * j].x += v.x; acc[2 * j].y += v.y; acc[2 * j + 1].x += v.z; acc[2 * j + 1].y += v.w;
          }
        }
      }

      // ---- the tile: bias, activation, scale; a row's outputs meet in shared memory and are written as lines
      const float rs = p.row_scale && mine < at.rows ? p.row_scale[at.row0 + mine] : 1.f;
      const float* bias = p.bias ? p.bias + (size_t)at.e * p.N : nullptr;
      const int live = min(32, at.rows - q * 32);
#pragma unroll
      for (int pass = 0; pass < PASSES; ++pass) {
#pragma unroll
        for (int g = 0; g < HC / 32 / PASSES; ++g) {
          const int c0 = (pass * (HC / 32 / PASSES) + g) * 32;
          float v[32];
#pragma unroll
          for (int j = 0; j < 16; ++j) { v[2 * j] = acc[c0 / 2 + j].x; v[2 * j + 1] = acc[c0 / 2 + j].y; }
          if (bias) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] += __ldg(bias + min(col0 + c0 + j, p.N - 1));
          }
          if constexpr (KIND == 1) glu_run<16>(p.act, v, p.act_alpha, p.act_limit);
          if constexpr (KIND == 2) act_unary_run<false, true>(p.act, v, p.act_alpha, p.act_limit);
          constexpr int n = 2 * PIECE;
#pragma unroll
          for (int j = 0; j < n; j += 16 / ESZ) {
            uint8_t* to = stage + lane * S::ROW + ((((g * n + j) * ESZ / 16) ^ turn(lane)) << 4);
            if constexpr (F32) *reinterpret_cast<float4*>(to) = make_float4(v[j] * rs, v[j + 1] * rs, v[j + 2] * rs, v[j + 3] * rs);
            else *reinterpret_cast<uint4*>(to) = make_uint4(pack_bf16(v[j] * rs, v[j + 1] * rs), pack_bf16(v[j + 2] * rs, v[j + 3] * rs),
                                                            pack_bf16(v[j + 4] * rs, v[j + 5] * rs), pack_bf16(v[j + 6] * rs, v[j + 7] * rs));
          }
        }
        __syncwarp();
        const int ch = lane % CPR, out0 = (KIND == 1 ? col0 >> 1 : col0) + pass * (RB / ESZ) + ch * (16 / ESZ), inside = min(16 / ESZ, on - out0);
        uint8_t* to = (uint8_t*)p.C + ((size_t)(at.row0 + q * 32 + lane / CPR) * p.ldc + out0) * ESZ;
        const size_t step = (size_t)(32 / CPR) * p.ldc * ESZ;
#pragma unroll 4
        for (int r = lane / CPR; r < live; r += 32 / CPR, to += step) {
          const uint4 x = *reinterpret_cast<const uint4*>(stage + r * S::ROW + ((ch ^ turn(r)) << 4));
          if (wide && inside == 16 / ESZ) {
            *reinterpret_cast<uint4*>(to) = x;
          } else {
            const uint32_t word[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int j = 0; j < 16 / ESZ; ++j)
              if (j < inside) {
                if constexpr (F32) reinterpret_cast<uint32_t*>(to)[j] = word[j];
                else reinterpret_cast<uint16_t*>(to)[j] = (uint16_t)(word[j / 2] >> (16 * (j & 1)));
              }
          }
        }
        __syncwarp();
      }
    }
  }
  if (*abort_flag)                                         // a wait ran out: copies still in flight land before shared memory is released
    for (int i = 0; i < 200; ++i) __nanosleep(1000);
  tc_fence_before();
  __syncthreads();
  if (warp == 1) { tc_fence_after(); tmem_dealloc(tmem, 512); }
}

template <int BN, int KIND, bool F32> static int launch_gemm(const CUtensorMap& tx, const CUtensorMap& tw, const Fp8Params& p, long long tiles, cudaStream_t st) {
  using S = Fp8GemmShape<BN, F32>;
  auto kern = fp8_gemm_kernel<BN, KIND, F32>;
  static DeviceOnce configured;
  if (configured.pending()) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
    if (e != cudaSuccess) return (int)e;
    configured.mark();
  }
  launch_pdl(kern, dim3(tiles < sm_count() ? (unsigned)tiles : sm_count()), dim3(FG_THREADS), S::SMEM, st, tx, tw, p);
  return (int)cudaGetLastError();
}

// bytes of the sums of `pieces` pieces of tiles of bn columns
static long long tile_scratch(long long pieces, int bn) { return 4 * pieces * FG_BM * bn; }

// Dense (M rows) or experts (counts / seg: from the bank's first expert on; M rows of the packing), tiles of bn = 128 or 256 columns; dense ones in `cuts` pieces along K.
int fp8_gemm_launch(const Fp8Call& c, cudaStream_t st) {
  Fp8Params p = fp8_params(c);
  p.cuts = c.cuts > 1 ? c.cuts : 1;
  const int bn = c.bn;
  if (c.E > FG_MAX_E || c.slot || (bn != 128 && bn != 256) || (c.counts && (c.M + FG_BM - 1) / FG_BM + c.E > 65535)) return -106;
  if (((uintptr_t)c.codes | (uintptr_t)c.w) & 15) return -114;
  const long long tiles = ((c.M + FG_BM - 1) / FG_BM + (c.counts ? (c.E < c.M ? c.E : c.M) : 0)) * (long long)((c.N + bn - 1) / bn);
  if (tiles >= 1ll << 31) return -106;
  if (p.cuts > 1 && (c.counts || p.cuts > p.kb || tiles * FG_SUMS > CUT_TICKETS || tiles * p.cuts > FG_MAX_PIECES || ((uintptr_t)c.scratch & 15))) return -106;
  if (p.cuts > 1 && (!c.scratch || !c.tickets || c.scratch_bytes < tile_scratch(tiles * p.cuts, bn))) return -131;
  CUtensorMap tx, tw;
  int r = fp8_tmap(&tx, c.codes, p.kb, c.rows, 0, FG_BM);
  if (!r) r = fp8_tmap(&tw, c.w, p.kb, p.N, c.E, bn);
  if (r) return r;
  const int kind = p.act == 0 ? 0 : act_gated(p.act) ? 1 : 2;
#define MX_FG(BN_, KIND_) if (bn == BN_ && kind == KIND_) return p.out_f32 ? launch_gemm<BN_, KIND_, true>(tx, tw, p, tiles * p.cuts, st) : launch_gemm<BN_, KIND_, false>(tx, tw, p, tiles * p.cuts, st)
  MX_FG(256, 0); MX_FG(256, 1); MX_FG(256, 2);
  MX_FG(128, 0); MX_FG(128, 1); MX_FG(128, 2);
#undef MX_FG
  return -106;
}

}  // namespace mx

using namespace mx;

// Bytes of scratch (16-byte aligned) that `pieces` pieces of tiles of bn columns want.
MX_HOST_API long long mx_fp8_tile_scratch(int pieces, int bn) { return tile_scratch(pieces, bn); }

MX_HOST_API int mx_fp8_call_bytes() { return (int)sizeof(Fp8Call); }

// A product (see Fp8Call): rows that are bf16 still are rounded, then the streaming kernel (nt) or the tiled one (bn) runs.
// -130: bf16 rows that have to be rounded first, and no room for codes; nothing was launched.  -131: too little room for partial sums.
MX_HOST_API int mx_fp8_product(const Fp8Call* call, cudaStream_t st) {
  const Fp8Call& c = *call;
  if (c.M <= 0 || c.N <= 0) return 0;
  if (c.K < 1 || c.x_div < 1 || c.E < 1 || c.rows < 1) return -101;
  if (act_gated(c.act) && c.N % 32) return -104;
  const bool gemv = fp8_gemv_takes(c), round = gemv ? fp8_gemv_rounds(c) : fp8_stream_rounds(c);
  if (c.xb && !round) {
    if (!c.codes) return -130;
    const int r = fp8_rows_launch(c.xb, 0, c.ldx, c.index, c.xb_rows, c.rows, c.K, c.codes, c.scale, st);
    if (r) return r;
  }
  if (gemv) return fp8_gemv_launch(c, round, st);
  return c.nt ? fp8_stream_launch(c, round, st) : fp8_gemm_launch(c, st);
}
