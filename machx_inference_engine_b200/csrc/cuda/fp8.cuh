// Rounding of activations to e4m3 with a power-of-two scale per 128 elements, shared by the quantiser and the products that round their rows themselves.
#pragma once
#include "common.cuh"
#include "host_util.h"
#include <cuda_fp8.h>

namespace mx {

constexpr int FP8_BLOCK = 128;   // elements of K per scale
constexpr int FP8_ROWS = 16;     // weight rows per scale

// Scale of a block with largest magnitude `amax`: the smallest power of two, 2^-100 at least, with amax <= 448 scale; 1 for zeros, NaN for infinities and NaN
// (the caller then writes zero codes).  *inv = 1 / scale, a power of two as well: x * inv is exact, so the codes are those of a division.
__device__ __forceinline__ float fp8_scale(float amax, float* inv) {
  const uint32_t bits = __float_as_uint(amax);
  *inv = 1.f;
  if (bits >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  if (bits == 0) return 1.f;
  int e = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u);      // biased: 448 = 1.75 * 2^8
  e = max(e, 27);
  *inv = __uint_as_float((uint32_t)(254 - e) << 23);
  return __uint_as_float((uint32_t)e << 23);
}
// max |v| as bits, NaN above infinity (magnitudes of floats order like their bits)
__device__ __forceinline__ uint32_t fp8_mag(float v) { return __float_as_uint(v) & 0x7fffffffu; }

__device__ __forceinline__ uint32_t fp8_pack4(float a, float b, float c, float d) {
  const __nv_fp8x2_storage_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const __nv_fp8x2_storage_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return (uint32_t)lo | ((uint32_t)hi << 16);
}

// Eight elements as they were loaded, and the bits of their largest magnitude: 16 for bf16, which are the high half of an fp32's.
template <typename T> struct Row8;
template <> struct Row8<__nv_bfloat16> {
  uint32_t w[4];
  __device__ __forceinline__ void load(const __nv_bfloat16* p) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  }
  __device__ __forceinline__ void zero() { w[0] = w[1] = w[2] = w[3] = 0; }
  __device__ __forceinline__ void put(int j, __nv_bfloat16 v) { w[j >> 1] |= (uint32_t)__bfloat16_as_ushort(v) << (16 * (j & 1)); }
  __device__ __forceinline__ uint32_t top() const {
    const uint32_t k = 0x7fff7fffu, m = __vmaxu2(__vmaxu2(w[0] & k, w[1] & k), __vmaxu2(w[2] & k, w[3] & k));
    return max(m & 0xffffu, m >> 16);
  }
  __device__ __forceinline__ uint2 codes(float inv) const {
    return make_uint2(fp8_pack4(bf16_lo(w[0]) * inv, bf16_hi(w[0]) * inv, bf16_lo(w[1]) * inv, bf16_hi(w[1]) * inv),
                      fp8_pack4(bf16_lo(w[2]) * inv, bf16_hi(w[2]) * inv, bf16_lo(w[3]) * inv, bf16_hi(w[3]) * inv));
  }
};
template <> struct Row8<float> {
  float f[8];
  __device__ __forceinline__ void load(const float* p) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = 0.f;
  }
  __device__ __forceinline__ void put(int j, float v) { f[j] = v; }
  __device__ __forceinline__ uint32_t top() const {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, fp8_mag(f[j]));
    return m;
  }
  __device__ __forceinline__ uint2 codes(float inv) const {
    return make_uint2(fp8_pack4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv), fp8_pack4(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv));
  }
};
// the largest over the sixteen lanes of a block, for IT blocks: bf16 magnitudes of two blocks share a register on the way
template <int IT> __device__ __forceinline__ void half_warp_max(uint32_t (&m)[IT], __nv_bfloat16) {
  constexpr int W = (IT + 1) / 2;
  uint32_t w[W];
#pragma unroll
  for (int t = 0; t < W; ++t) w[t] = m[2 * t] | (2 * t + 1 < IT ? m[2 * t + 1 < IT ? 2 * t + 1 : 0] << 16 : 0u);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1)
#pragma unroll
    for (int t = 0; t < W; ++t) w[t] = __vmaxu2(w[t], __shfl_xor_sync(0xffffffffu, w[t], o));
#pragma unroll
  for (int t = 0; t < IT; ++t) m[t] = t & 1 ? w[t / 2] & 0xffff0000u : w[t / 2] << 16;
}
template <int IT> __device__ __forceinline__ void half_warp_max(uint32_t (&m)[IT], float) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1)
#pragma unroll
    for (int t = 0; t < IT; ++t) m[t] = max(m[t], __shfl_xor_sync(0xffffffffu, m[t], o));
}

// D[tmem] (+)= A[smem] * B[smem], e4m3 inputs (K = 32 a step), fp32 accumulate.  A whole warp comes here and `leader` (elect_one) issues: in a branch of one
// thread the descriptors have to be moved to uniform registers before every instruction (four products and two commits: 470 cycles, 94 this way).
__device__ __forceinline__ void umma_e4m3(uint32_t leader, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void umma_commit_if(uint32_t leader, uint32_t bar) {
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n"
               ::"r"(bar), "r"(leader) : "memory");
}
__device__ __forceinline__ void mbar_arrive_if(uint32_t leader, uint32_t bar) {
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t@q mbarrier.arrive.shared::cta.b64 _, [%0];\n\t}\n" ::"r"(bar), "r"(leader) : "memory");
}
// whether a phase has completed, without waiting: asked ahead of the work that it is asked before, the answer costs nothing
__device__ __forceinline__ bool mbar_peek(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
// kind::f8f6f4 instruction descriptor: e4m3 x e4m3 -> fp32, M x N tile, both operands K-major.
__host__ __device__ constexpr uint32_t umma_idesc_e4m3(int M, int N) { return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24); }

// two fp32 numbers in one register pair: d = a * b + c and a * b, each rounded once
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}" : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
template <int N> __device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, uint32_t (&r)[N]) {      // N columns of 32 lanes
  static_assert(N == 16 || N == 32, "columns of one load");
  if constexpr (N == 32) {
    tmem_ld_32x32(taddr, r);
  } else {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
          "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
  }
}

// 4 bytes from global to shared memory, asynchronously; `arrive_copies`: the barrier is arrived at when this thread's copies so far have landed.
__device__ __forceinline__ void copy4(uint32_t dst, const void* src) { asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void arrive_copies(uint32_t bar) { asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory"); }

// What a product multiplies and writes.
struct Fp8Params {
  const __nv_bfloat16* xb;   // rows that a kernel rounds itself, `ldx` elements apart, of K
  long long ldx;
  int K;
  const uint8_t* xc;         // rounded rows, and [E][N][kb * 128] of weights, of the kernel that reads them without boxes
  const uint8_t* w;
  const float* sx;           // [kb][x_rows]
  int x_rows;
  const float* sw;           // [E][ceil(N / 16)][kb]
  void* C;
  long long ldc;
  int out_f32, M, N, kb, E;
  const float* bias;         // [N] or [E][N]
  const float* row_scale;    // [M]
  int act;
  float act_alpha, act_limit;
  const int* counts;         // experts: rows of expert i of the bank, and the first of them
  const int* seg;
  const int* slot;           // slots: expert of output row m, whose input is row m / x_div
  int x_div, e_lo, cuts;     // cuts: pieces of a tile along K
  float* part;               // partial sums of cut tiles
  int* tickets;
  int* status;
};

// A product as the caller describes it (ops/cuda.py packs the fields in this order).
struct Fp8Call {
  const void* xb;            // bf16 rows, rounded into codes and scale first; null: these hold the rounded rows
  long long ldx;
  const int* index;          // row of xb that rounded row r is; null: r
  void* codes;               // [rows][kb * 128]
  float* scale;              // [kb][rows]
  const void* w;
  const float* sw;
  void* c;
  long long ldc;
  const float* bias;         // the rest as in Fp8Params
  const float* row_scale;
  const int* counts;
  const int* seg;
  const int* slot;
  float* scratch;            // partial sums, `scratch_bytes` of room, and the counters of cut work (host_util.h)
  int* tickets;
  long long scratch_bytes;
  int xb_rows, rows;         // rows of xb, and rounded rows
  int M, N, K, E, out_f32, act, x_div, e_lo;
  int nt, bn, cuts;          // rows of a group of the streaming kernel, or 0 and the columns of a tile and its pieces along K of the tiled one
  float act_alpha, act_limit;
  int unused;
};
int fp8_rows_launch(const void* x, int f32, long long ldx, const int* index, int x_rows, int rows, int K, void* codes, float* scale, cudaStream_t st);
bool fp8_gemv_takes(const Fp8Call& c);
bool fp8_gemv_rounds(const Fp8Call& c);
int fp8_gemv_launch(const Fp8Call& c, bool round, cudaStream_t st);
bool fp8_stream_rounds(const Fp8Call& c);
int fp8_stream_launch(const Fp8Call& c, bool round, cudaStream_t st);
int fp8_gemm_launch(const Fp8Call& c, cudaStream_t st);
inline Fp8Params fp8_params(const Fp8Call& c) {
  Fp8Params p{};
  p.sx = c.scale; p.x_rows = c.rows; p.sw = c.sw; p.C = c.c; p.ldc = c.ldc; p.out_f32 = c.out_f32; p.M = c.M; p.N = c.N; p.K = c.K; p.kb = (c.K + FP8_BLOCK - 1) / FP8_BLOCK; p.E = c.E;
  p.bias = c.bias; p.row_scale = c.row_scale; p.act = c.act; p.act_alpha = c.act_alpha; p.act_limit = c.act_limit; p.counts = c.counts; p.seg = c.seg; p.slot = c.slot;
  p.x_div = c.x_div; p.e_lo = c.e_lo; p.part = c.scratch; p.tickets = c.tickets; p.status = status_word();
  return p;
}

// A warp's arrival at a counter that the `pieces` of cut work share; true for the last, which leaves the counter at zero and may read what all of them have written.  The fence
// is the atomic's own, of one lane (__threadfence() by every lane costs a sequentially consistent one each), so both sides go through a barrier of the warp: the lanes' writes come
// before that lane's release, and their reads after its acquire.  The shuffle in between orders nothing.
__device__ __forceinline__ bool warp_arrives_last(int* counter, int pieces) {
  int before = 0;
  __syncwarp();
  if ((threadIdx.x & 31) == 0) {
    asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
    if (before == pieces - 1) *counter = 0;
  }
  before = __shfl_sync(0xffffffffu, before, 0);
  __syncwarp();
  return before == pieces - 1;
}

// Boxes of `rows` rows by one block of codes [E][n][kb * 128] (E = 0: [n][kb * 128]).  Codes travel as two-byte elements: the tile is bytes either way.
inline int fp8_tmap(CUtensorMap* out, const void* codes, int kb, int n, int E, int rows) {
  const uint64_t row = (uint64_t)kb * FP8_BLOCK;
  uint64_t dims[3] = {row / 2, (uint64_t)n, (uint64_t)E}, strides[2] = {row, row * (uint64_t)n};
  uint32_t box[3] = {FP8_BLOCK / 2, (uint32_t)rows, 1};
  return make_tmap_bf16(out, codes, E ? 3 : 2, dims, strides, box, 1);
}

}  // namespace mx
