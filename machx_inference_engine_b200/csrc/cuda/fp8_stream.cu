// Products of a few e4m3 rows (up to 64 together) with e4m3 weights, bound by reading the weights: a dense layer of a decode batch, an expert's few rows, a slot's one row.
//   y[m, n] = act(sum_b sx[b][m] sw[n / 16][b] sum_{k in b} x8[m][k] w8[n][k] + bias[n])
//
// The weights are the M side of tcgen05.mma (128 weight rows x 128 bytes: one block of K, one TMA box) and the rows its N side, padded to NT = 16, 32 or 64
// columns; the tensor cores need a small part of the time that the box takes to arrive, whatever NT.  Every block has scales of its own, so its sums go from
// TMEM to registers, where a thread owns a weight row and adds s_x s_w times them to NT sums in fp32.
//   warp 0      TMA boxes of weights and of rows into a ring of NST stages, and asynchronous copies of their scales into a ring of their own
//   warp 1      tcgen05.mma from one thread into a ring of ACC accumulators
//   warps 2-5   32 weight rows each: scale and add, epilogue
//   warps 6, 7  (ROUND) bf16 rows to codes: for up to eight rows every CTA rounds the blocks that it needs itself, once, into shared memory, so that a decode step is
//               one launch (smaller layers: fp8_gemv.cu)
// The work is the list of (group of rows, 128 weight rows, block of K) laid end to end, of which every CTA takes an equal run.  A tile that is cut leaves fp32
// partials (at most two per CTA); the warp that arrives last adds them in the order of the CTAs, so results do not depend on timing.
// Bound: memory, and for a token the latencies of one launch.  Two CTAs share an SM: with one and 80 KB of weights under way 8 x 28672 x 4096 took 32 us.
// Measured in a graph of calls over more weights than L2 holds: 8 x 28672 x 4096 gated 25.1 us (4.7 TB/s), 1 x 6144 x 4096 9.6 us, 1 x 28672 x 4096 23.4 us, 1 x 4096 x 14336 14.3 us (about five from launch
// to the first sums), experts of 64 tokens, 8 of 128 of 1536 x 2048, 63.7 us (6.2 TB/s, 0.95 of a copy's rate), slots of four tokens, 4 of 32 of 2880 x 2880, 23.6 us.  One layer again and again, its weights in
// L2: 1 x 6144 x 4096 8.3 us, 1 x 4096 x 14336 10.9.
// Every mbarrier wait is bounded.
#include "act.cuh"
#include "common.cuh"
#include "fp8.cuh"
#include "host_util.h"

namespace mx {

constexpr int FS_TILE = 128;             // weight rows per tile
constexpr int FS_W = FS_TILE * FP8_BLOCK;
constexpr int FS_MAX_E = 1024;
constexpr int FS_MAX_GRID = CUT_TICKETS / 4;

template <int NT, bool ROUND> struct Fp8StreamShape {
  static_assert(!ROUND || NT == 16, "rows that are rounded here");
  static constexpr int X = NT * FP8_BLOCK;
  static constexpr int STAGE = FS_W + (ROUND ? 0 : X);
  static constexpr int BLOCKS = ROUND ? 26 : 0;        // blocks of rounded rows that a CTA keeps
  static constexpr int CTAS = 2;                       // per SM
  static constexpr int OUT = 4 * 8 * 32 * 4;           // eight columns of a warp's sums, on their way out
  static constexpr int ROOM = 104 * 1024 - OUT;      // for stages and rounded rows
  static constexpr int SMEM = ROOM + OUT + 1024;
  static constexpr int NST = ROUND ? 5 : ROOM / STAGE; // at most; fewer where a run needs more rounded rows
  static constexpr int ACC = 4;
  static constexpr int TMEM = NT * ACC;                // 64, 128, 256 columns: two CTAs have 512
  // Scales of a unit: 8 of the weights, NT of the rows.  A slot is free again when the products of the unit NST before are done, since they waited for the sums
  // of the unit ACC before them.
  static constexpr int RING = NST + ACC, SC = 8 + (ROUND ? 0 : NT);
  static constexpr int THREADS = ROUND ? 256 : 192;
};

// A run of `per` units for every CTA; shorter runs would cost more in partial sums than they gain.
__host__ __device__ inline int fp8_run(int total, int grid) {
  const int per = (total - 1) / grid + 1;
  return per < 2 ? 2 : per;
}

template <int NT, bool ROUND>
__global__ void __launch_bounds__(Fp8StreamShape<NT, ROUND>::THREADS, Fp8StreamShape<NT, ROUND>::CTAS)
fp8_stream_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, const Fp8Params p) {
  using S = Fp8StreamShape<NT, ROUND>;
  constexpr int MST = S::NST, ACC = S::ACC, FS_THREADS = S::THREADS;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t s_bar[2 * MST + 2 * ACC + S::BLOCKS];
  __shared__ __align__(16) float s_scale[S::RING][S::SC];
  __shared__ __align__(16) float s_rows[ROUND ? S::BLOCKS : 1][NT];
  __shared__ uint16_t s_pre[FS_MAX_E + 1];
  __shared__ int s_sum[FS_THREADS / 32];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t bar_full = smem_u32(s_bar), bar_empty = bar_full + 8 * MST, bar_tfull = bar_empty + 8 * MST, bar_tempty = bar_tfull + 8 * ACC, bar_x = bar_tempty + 8 * ACC;
  volatile int* abort_flag = &s_abort;
  if (tid == 0) {
    for (int s = 0; s < MST; ++s) { mbar_init(bar_full + 8 * s, 1 + 32); mbar_init(bar_empty + 8 * s, 1); }      // (the boxes, and every lane's copies)
    for (int a = 0; a < ACC; ++a) { mbar_init(bar_tfull + 8 * a, 2); mbar_init(bar_tempty + 8 * a, 4); }
    for (int b = 0; b < S::BLOCKS; ++b) mbar_init(bar_x + 8 * b, p.slot ? 1 : p.M);
    s_abort = 0;
    fence_mbar_init();
  }

  // ---- the list of work
  const bool banked = p.counts != nullptr;
  const int n_tiles = (p.N + FS_TILE - 1) / FS_TILE;
  int groups = p.slot ? p.M : 1;
  if (banked) {
    pdl_wait();
    int run = 0;
    for (int e0 = 0; e0 < p.E; e0 += FS_THREADS) {
      const int e = e0 + tid;
      int incl = e < p.E ? (p.counts[e] + NT - 1) / NT : 0;
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
      for (int w = 0; w < FS_THREADS / 32; ++w) {
        if (w < warp) before += s_sum[w];
        run += s_sum[w];
      }
      if (e < p.E) s_pre[e] = (uint16_t)(before + incl - mine);
      __syncthreads();
    }
    groups = run;
    if (tid == 0) s_pre[p.E] = (uint16_t)run;
  }
  __syncthreads();
  const int total = groups * n_tiles * p.kb;
  const int per = fp8_run(total, (int)gridDim.x);
  const int my0 = min((long long)total, (long long)blockIdx.x * per), my1 = min(total, my0 + per);

  // a unit of the list: group (expert e, output rows row0 .. row0 + rows - 1), tile nt, block k
  struct Place { int g, e, row0, rows, nt, k; };
  auto group = [&](Place& r) {                         // what r.g is
    if (p.slot) {
      r.row0 = r.g; r.rows = 1;
      r.e = p.slot[r.g] - p.e_lo;
    } else if (banked) {
      int lo = 0, hi = p.E - 1;                        // the expert with s_pre <= g < the next one's
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (s_pre[mid] <= r.g) lo = mid; else hi = mid - 1;
      }
      const int c = r.g - s_pre[lo];
      r.e = lo;
      r.row0 = p.seg[lo] + c * NT;
      r.rows = r.row0 < 0 ? 0 : min(min(NT, p.counts[lo] - c * NT), p.M - r.row0);
    } else {
      r.e = 0; r.row0 = 0; r.rows = p.M;
    }
  };
  auto place = [&](int pos) {
    Place r;
    const int t = pos / p.kb;
    r.k = pos - t * p.kb;
    r.g = t / n_tiles;
    r.nt = t - r.g * n_tiles;
    group(r);
    return r;
  };
  auto next_tile = [&](Place& r, bool any) {           // (any: there is one)
    r.k = 0;
    if (++r.nt == n_tiles) {
      r.nt = 0; ++r.g;
      if (any) group(r);
    }
  };
  const int blocks = p.slot ? per : min(p.kb, per);    // (ROUND) that a run needs; a dense layer's come again in every tile
  const int NST = ROUND ? min(MST, (S::ROOM - blocks * S::X) / S::STAGE) : MST;
  const uint32_t rows_at = base + NST * S::STAGE, out_at = base + S::ROOM;
  const bool early = !banked && !p.slot;               // which weights are read does not depend on the launch before
  const int sw_groups = (p.N + FP8_ROWS - 1) / FP8_ROWS;

  if (warp == 0) {
    // ------------------------------------------------ TMA, scales
    if (my0 < my1) {
      if (lane == 0) { prefetch_tmap(&tm_w); if (!ROUND) prefetch_tmap(&tm_x); }
      if (!early && !banked) pdl_wait();
      auto load_w = [&](int s, const Place& at) {
        mbar_expect_tx(bar_full + 8 * s, S::STAGE);
        tma_load_3d(base + s * S::STAGE, &tm_w, bar_full + 8 * s, at.k * (FP8_BLOCK / 2), at.nt * FS_TILE, min(max(at.e, 0), p.E - 1));
      };
      auto next = [&](Place& r, int i) {
        if (++r.k == p.kb) next_tile(r, i + 1 < my1);
      };
      Place at = place(my0), w = at;
      int ahead = 0;
      if (early) {
        for (; ahead < NST && my0 + ahead < my1; ++ahead) {
          if (lane == 0) load_w(ahead, w);
          next(w, my0 + ahead);
        }
        pdl_wait();
      }
      uint32_t s = 0, ph = 1, r = 0;
      for (int pos = my0; pos < my1; ++pos) {
        if (pos - my0 >= ahead) {
          if (!mbar_wait(bar_empty + 8 * s, ph, p.status, ERR_MBAR_TIMEOUT_PRODUCER, abort_flag)) break;
          if (lane == 0) load_w(s, at);
        }
        const uint32_t to = smem_u32(s_scale[r]) + 4 * lane;
        if (lane < 8) copy4(to, p.sw + ((size_t)min(max(at.e, 0), p.E - 1) * sw_groups + min(at.nt * (FS_TILE / FP8_ROWS) + lane, sw_groups - 1)) * p.kb + at.k);
        if constexpr (!ROUND) {
          const int row = p.slot ? at.row0 / p.x_div : at.row0;
          if (lane == 0) tma_load_2d(base + s * S::STAGE + FS_W, &tm_x, bar_full + 8 * s, at.k * (FP8_BLOCK / 2), row);
          const float* from = p.sx + (size_t)at.k * p.x_rows + row + lane;
#pragma unroll
          for (int c = 0; c < NT; c += 32)
            if (c + lane < at.rows) copy4(to + 32 + 4 * c, from + c);
        }
        arrive_copies(bar_full + 8 * s);
        if (++s == NST) { s = 0; ph ^= 1; }
        if (++r == S::RING) r = 0;
        next(at, pos);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------ products
    // Tensor memory is taken when the launch before has ended: it may still want some, and would wait for a CTA that waits for it.  For the same reason the next
    // launch's CTAs may come only now.
    if (!banked) pdl_wait();
    tmem_alloc(smem_u32(&s_tmem), S::TMEM);
    tmem_relinquish();
    pdl_launch_dependents();
    tc_fence_before();
    asm volatile("bar.sync 1, 160;" ::: "memory");
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    {
      const uint32_t leader = elect_one();
      constexpr uint32_t idesc = umma_idesc_e4m3(FS_TILE, NT);
      uint32_t s = 0, ph = 0, a = 0, aph = 1;
      int x = 0;                                       // block of rounded rows
      for (int pos = my0; pos < my1; ++pos) {
        if (!mbar_wait(bar_tempty + 8 * a, aph, p.status, ERR_MBAR_TIMEOUT_MMA, abort_flag)) break;
        if (!mbar_wait(bar_full + 8 * s, ph, p.status, ERR_MBAR_TIMEOUT_MMA, abort_flag)) break;
        if (ROUND && !mbar_wait(bar_x + 8 * x, 0, p.status, ERR_MBAR_TIMEOUT_DEQUANT, abort_flag)) break;
        __syncwarp();                                  // (no lane may miss a phase)
        tc_fence_after();
        const uint64_t dw = umma_desc_k_sw128(base + s * S::STAGE);
        const uint64_t dx = umma_desc_k_sw128(ROUND ? rows_at + x * S::X : base + s * S::STAGE + FS_W);
#pragma unroll
        for (int kk = 0; kk < FP8_BLOCK / 32; ++kk) umma_e4m3(leader, tmem + a * NT, dw + 2 * kk, dx + 2 * kk, idesc, kk != 0);
        umma_commit_if(leader, bar_empty + 8 * s);
        mbar_arrive_if(leader, bar_tfull + 8 * a);                // (what this thread has seen arrive, the scales among it, is seen by who waits here)
        umma_commit_if(leader, bar_tfull + 8 * a);
        if (++s == NST) { s = 0; ph ^= 1; }
        if (++a == ACC) { a = 0; aph ^= 1; }
        if (ROUND && ++x == blocks) x = 0;
      }
    }
  } else if (warp < 6) {
    // ------------------------------------------------ scales, sums, epilogue: a thread owns weight row `n`
    const int q = warp & 3;
    asm volatile("bar.sync 1, 160;" ::: "memory");
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    if (!banked) pdl_wait();
    uint32_t a = 0, aph = 0, ring = 0;
    int x = 0;
    bool ok = true;
    Place at;
    if (my0 < my1) at = place(my0);
    for (int pos = my0; ok && pos < my1;) {
      const int first = at.k, n_units = min(my1 - pos, p.kb - at.k);
      const int n = at.nt * FS_TILE + q * 32 + lane;
      const int e = min(max(at.e, 0), p.E - 1);
      float2 acc[NT / 2];
#pragma unroll
      for (int j = 0; j < NT / 2; ++j) acc[j] = make_float2(0.f, 0.f);
      for (int i = 0; i < n_units; ++i) {
        if (!(ok = mbar_wait(bar_tfull + 8 * a, aph, p.status, ERR_MBAR_TIMEOUT_EPILOGUE, abort_flag))) break;
        tc_fence_after();
        const float4* sx = reinterpret_cast<const float4*>(ROUND ? s_rows[x] : s_scale[ring] + 8);
        const float sw = s_scale[ring][2 * q + (lane >> 4)];
        constexpr int C = NT < 32 ? NT : 32;
#pragma unroll
        for (int c0 = 0; c0 < NT; c0 += C) {
          uint32_t r[C];
          tmem_ld_cols<C>(tmem + ((uint32_t)(q * 32) << 16) + a * NT + c0, r);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < C; j += 4) {
            const float4 t = sx[(c0 + j) / 4];
            float2& u = acc[(c0 + j) / 2];
            float2& v = acc[(c0 + j) / 2 + 1];
            u = fma2(make_float2(__uint_as_float(r[j]), __uint_as_float(r[j + 1])), mul2(make_float2(t.x, t.y), make_float2(sw, sw)), u);
            v = fma2(make_float2(__uint_as_float(r[j + 2]), __uint_as_float(r[j + 3])), mul2(make_float2(t.z, t.w), make_float2(sw, sw)), v);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_tempty + 8 * a);
        if (++ring == S::RING) ring = 0;
        if (ROUND && ++x == blocks) x = 0;
        if (++a == ACC) { a = 0; aph ^= 1; }
      }
      if (!ok) break;

      // ---- a cut tile: partials, and the last warp to arrive adds them up
      bool mine_to_finish = true;
      if (n_units < p.kb) {
        const int t0 = pos - first, c0 = t0 / per, c1 = (t0 + p.kb - 1) / per;
        float4* part = reinterpret_cast<float4*>(p.part);
        auto slab = [&](int c) { return part + (((size_t)c * 2 + (c == c0 ? 1 : 0)) * 4 + q) * (NT / 4 * 32) + lane; };
        float4* mine = slab(blockIdx.x);
#pragma unroll
        for (int j = 0; j < NT / 4; ++j)
          if (4 * j < at.rows) mine[j * 32] = make_float4(acc[2 * j].x, acc[2 * j].y, acc[2 * j + 1].x, acc[2 * j + 1].y);
        mine_to_finish = warp_arrives_last(p.tickets + c0 * 4 + q, c1 - c0 + 1);
        if (mine_to_finish) {
#pragma unroll
          for (int j = 0; j < NT / 2; ++j) acc[j] = make_float2(0.f, 0.f);
          // P parts of 4 J columns at a time are under way; they are added in order (eight for four of up to eight rows: 8 x 4096 x 14336 17.3 -> 16.9 us, 1 x 4096 x 4096 7.55 -> 7.25; twelve 16.5, 7.5)
          constexpr int LIVE = ROUND ? 2 : NT / 4, J = LIVE < 4 ? LIVE : 4, P = ROUND ? 8 : 4;
#pragma unroll
          for (int j0 = 0; j0 < LIVE; j0 += J) {
            if (4 * j0 < at.rows) {
              for (int c = c0; c <= c1; c += P) {
                float4 v[P][J];
#pragma unroll
                for (int i = 0; i < P; ++i)
#pragma unroll
                  for (int j = 0; j < J; ++j)
                    v[i][j] = c + i <= c1 && 4 * (j0 + j) < at.rows ? __ldcg(slab(c + i) + (j0 + j) * 32) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int i = 0; i < P; ++i)
#pragma unroll
                  for (int j = 0; j < J; ++j) {
                    float2& u = acc[2 * (j0 + j)];
                    float2& w = acc[2 * (j0 + j) + 1];
                    u.x += v[i][j].x; u.y += v[i][j].y; w.x += v[i][j].z; w.y += v[i][j].w;
                  }
              }
            }
          }
        }
      }
      if (mine_to_finish) {
        // ---- epilogue: gate rows are lanes 0-15, their up rows lanes 16-31.  Eight columns at a time go through shared memory, so that the code that follows exists
        // once: unrolled over the columns it is fetched from L2 instruction by instruction (20 rows: 14000 cycles)
        const bool gated = act_gated(p.act), owned = at.e >= 0 && at.e < p.E;
        const float bias = p.bias && n < p.N ? p.bias[(size_t)e * p.N + n] : 0.f;
        const int on = gated ? p.N >> 1 : p.N, o = gated ? at.nt * (FS_TILE / 2) + q * 16 + (lane & 15) : n;
        const bool write = o < on && (!gated || lane < 16);
        float* const col = reinterpret_cast<float*>(smem_raw + (out_at - smem_u32(smem_raw))) + q * 256 + lane;
#pragma unroll 1
        for (int j0 = 0; j0 < at.rows; j0 += 8) {
#pragma unroll
          for (int g = 0; g < NT / 8; ++g)
            if (8 * g == j0) {
#pragma unroll
              for (int j = 0; j < 4; ++j) { col[64 * j] = acc[4 * g + j].x; col[64 * j + 32] = acc[4 * g + j].y; }
            }
          const int live = min(8, at.rows - j0);
          float v[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = col[32 * j] + bias;             // (a lane reads what it has written; columns past the live ones hold anything)
          if (gated) {
            float pair[16];
#pragma unroll
            for (int j = 0; j < 8; ++j) { pair[j] = v[j]; pair[8 + j] = __shfl_down_sync(0xffffffffu, v[j], 16); }
            glu_run<8>(p.act, pair, p.act_alpha, p.act_limit);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = pair[j];
          } else if (p.act) {
            act_unary_run<false, true>(p.act, v, p.act_alpha, p.act_limit);
          }
          if (p.row_scale) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] *= p.row_scale[at.row0 + min(j0 + j, at.rows - 1)];
          }
          if (!owned) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = 0.f;
          }
          const size_t first = (size_t)(at.row0 + j0) * p.ldc + o;
          if (write) {
            if (p.out_f32) {
#pragma unroll
              for (int j = 0; j < 8; ++j)
                if (j < live) ((float*)p.C)[first + j * p.ldc] = v[j];
            } else {
#pragma unroll
              for (int j = 0; j < 8; ++j)
                if (j < live) ((__nv_bfloat16*)p.C)[first + j * p.ldc] = __float2bfloat16(v[j]);
            }
          }
        }
      }
      pos += n_units;
      next_tile(at, pos < my1);
    }
  } else if constexpr (ROUND) {
    // ------------------------------------------------ rows to codes: half a warp a block of a row, four pairs of blocks at a time; the blocks in the order of their use
    pdl_wait();
    const int half = lane >> 4, sub = lane & 15, rows = p.slot ? 1 : p.M, need = min(blocks, my1 - my0), items = (need + 1) / 2 * rows;
    uint8_t* const xs = smem_raw + (rows_at - smem_u32(smem_raw));
    for (int i0 = (warp - 6) * 4; i0 < items; i0 += 8) {
      Row8<__nv_bfloat16> v[4];
      int b[4], r[4];
      uint32_t m[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int i = min(i0 + t, items - 1), pair = i / rows;
        r[t] = i - pair * rows;
        b[t] = 2 * pair + half;
        const int unit = my0 + min(b[t], need - 1), tile = unit / p.kb, at = (unit - tile * p.kb) * FP8_BLOCK + 8 * sub;
        const __nv_bfloat16* row = p.xb + (long long)(p.slot ? tile / n_tiles / p.x_div : r[t]) * p.ldx;
        v[t].load(row + (at + 8 <= p.K ? at : 0));             // (K is 8 at least)
        if (at + 8 > p.K) {
          v[t].zero();
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (at + j < p.K) v[t].put(j, row[at + j]);
        }
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) m[t] = v[t].top();
      half_warp_max<4>(m, __nv_bfloat16());
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        if (i0 + t >= items || b[t] >= need) continue;
        float inv;
        const float sc = fp8_scale(__uint_as_float(m[t]), &inv);
        const uint2 w = m[t] < 0x7f800000u ? v[t].codes(inv) : make_uint2(0, 0);
        *reinterpret_cast<uint2*>(xs + b[t] * S::X + sw128_offset(r[t], sub >> 1) + (sub & 1) * 8) = w;
        if (sub == 0) s_rows[b[t]][r[t]] = sc;
      }
      fence_proxy_async();
      __syncwarp();
      if (sub == 0) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
          if (i0 + t < items && b[t] < need) mbar_arrive(bar_x + 8 * b[t]);
      }
    }
  }
  if (*abort_flag)                                         // a wait ran out: copies still in flight land before shared memory is released
    for (int i = 0; i < 200; ++i) __nanosleep(1000);
  tc_fence_before();
  __syncthreads();
  if (warp == 1) { tc_fence_after(); tmem_dealloc(s_tmem, S::TMEM); }
}

// bytes of partial sums of a launch with groups of nt rows, whatever its grid
static long long stream_scratch(int nt) { return 4ll * FS_MAX_GRID * 2 * FS_TILE * nt; }
static int stream_grid(int ctas) { return ctas * sm_count() < FS_MAX_GRID ? ctas * sm_count() : FS_MAX_GRID; }

template <int NT, bool ROUND> static int launch_stream(const CUtensorMap& tw, const CUtensorMap& tx, const Fp8Params& p, cudaStream_t st) {
  using S = Fp8StreamShape<NT, ROUND>;
  auto kern = fp8_stream_kernel<NT, ROUND>;
  static DeviceOnce configured;
  if (configured.pending()) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
    if (e != cudaSuccess) return (int)e;
    configured.mark();
  }
  launch_pdl(kern, dim3(stream_grid(S::CTAS)), dim3(S::THREADS), S::SMEM, st, tw, tx, p);
  return (int)cudaGetLastError();
}

// Whether the streaming kernel rounds a launch's rows itself: up to eight (slots: one each), of which a CTA's share of the blocks fits its shared memory.  us, two launches -> one: 4 rows x
// 6144 x 4096 11.6 -> 10.5, 4096 x 14336 17.6 -> 15.7, 28672 x 4096 28.2 -> 24.9, and a launch less on the host (5 us of 15); 8 rows even; 16 rows 12.3 -> 15.7, 27.7 -> 44.3.
bool fp8_stream_rounds(const Fp8Call& c) {
  using S = Fp8StreamShape<16, true>;
  if (!c.xb || c.nt != 16 || c.counts || (!c.slot && c.M > 8) || c.K < 8 || c.ldx % 8 || ((uintptr_t)c.xb & 15)) return false;
  const int kb = (c.K + FP8_BLOCK - 1) / FP8_BLOCK, n_tiles = (c.N + FS_TILE - 1) / FS_TILE;
  const long long total = (c.slot ? (long long)c.M : 1) * n_tiles * kb;
  if (total >= 1ll << 30) return false;
  const int per = fp8_run((int)total, stream_grid(S::CTAS));
  return (c.slot ? per : per < kb ? per : kb) <= S::BLOCKS;
}

// Dense (M <= nt), experts (counts / seg) or slots (slot), in groups of nt = 16, 32 or 64 rows.
int fp8_stream_launch(const Fp8Call& c, bool round, cudaStream_t st) {
  Fp8Params p = fp8_params(c);
  const int nt = c.nt;
  const long long groups = c.slot ? c.M : c.counts ? (long long)c.M / nt + (c.E < c.M ? c.E : c.M) + 1 : 1;
  if ((c.counts && c.E > FS_MAX_E) || groups >= 65536 || groups * ((p.N + FS_TILE - 1) / FS_TILE) * p.kb >= 1ll << 30 || (!c.slot && !c.counts && c.M > nt)) return -106;      // (units are counted in 32 bits)
  if (((uintptr_t)c.codes | (uintptr_t)c.w | (uintptr_t)c.scratch) & 15) return -114;
  if (!c.scratch || !c.tickets || c.scratch_bytes < stream_scratch(nt)) return -131;
  CUtensorMap tw, tx;
  int r = fp8_tmap(&tw, c.w, p.kb, p.N, c.E, FS_TILE);
  if (r) return r;
  if (round) {
    p.xb = (const __nv_bfloat16*)c.xb;
    p.ldx = c.ldx;
    return launch_stream<16, true>(tw, tw, p, st);
  }
  r = fp8_tmap(&tx, c.codes, p.kb, c.rows, 0, nt);
  if (r) return r;
  switch (nt) {
    case 16: return launch_stream<16, false>(tw, tx, p, st);
    case 32: return launch_stream<32, false>(tw, tx, p, st);
    case 64: return launch_stream<64, false>(tw, tx, p, st);
    default: return -106;
  }
}

}  // namespace mx

// Bytes of scratch (16-byte aligned) that a launch with groups of up to `nt` rows wants.
MX_HOST_API long long mx_fp8_stream_scratch(int nt) { return mx::stream_scratch(nt); }
