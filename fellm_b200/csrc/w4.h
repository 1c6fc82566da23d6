// A matrix [N, K] in four bits, as every kernel that reads one finds it.
//
// w[n, k] = q[n, k] s[n, k / G]: levels q of -8..7, a scale for every G (32, 64 or 128) consecutive elements of a row.  A
// scale has at most five significant bits, a level at most four of which -8 needs one: their product has at most eight, so
// it is a bfloat16 number EXACTLY, and the matrix means the same numbers to a kernel that scales its sums of x q group by
// group and to one that feeds bfloat16 weights to the tensor cores.
//
// Levels: slabs of 16 rows x chunks of 64 k, 512 bytes each, slab after slab and in it chunk after chunk; a warp reads a
// chunk in one load of 16 bytes a lane.  Lane 4 g + c has rows g and g + 8, and of the chunk's two halves the elements
// 8 c .. 8 c + 7: word j is half j / 2, elements 4 (j % 2) .. + 3 of those eight.  In a word, turned left by three bits, four
// bits each, q + 8:
//   bits  0 row g element 0,   4 row g+8 element 0,   8 row g element 2,  12 row g+8 element 2,
//   bits 16 row g element 1,  20 row g+8 element 1,  24 row g element 3,  28 row g+8 element 3,
// so that the word turned right by 4 r and masked with 0x00780078 has at the top of bfloat16's mantissa what the r-th operand
// register of an mma.m16n8k16 wants, whose k slots {2c, 2c+1, 2c+8, 2c+9} are taken for elements {0, 1, 2, 3} (a sum does not
// ask in which order): or-ed with 0x41804180 it is the pair of 16 + (q + 8).
// Scales: bfloat16 pairs (row g, row g + 8), eight of them for each slab and group.
// Rows behind N are levels 0 under scales 0, elements behind K levels 0.  Behind the last slab there are W4_READ_AHEAD chunks (and
// as many chunks' scales at groups of 32) of memory of no meaning: a kernel that fetches ahead need not ask where a row ends.
#pragma once
#include "common.cuh"

#define W4_SLAB 16
#define W4_CHUNK 64
#define W4_READ_AHEAD 32

// (the caller keeps one of these with the matrix and hands its address to the launchers)
struct W4Ref {
  const uint4* q;            // [slabs][chunks][32]
  const unsigned* s;         // [slabs][groups][8]
  int N, K, chunks, groups;  // groups: as many as cover chunks * 64 elements
  int gshift;                // log2 of the group: 5, 6 or 7
};

// An RMSNorm handed on between two products.  The one that adds into the rows leaves, beside out += .., next_x[m, n] =
// bfloat16(out[m, n] next_w[n]) and next_ssq[m * (N / P) + n / P] = the sums of out[m, n]^2 over P columns (a slab's 16 up to 16 rows, a
// warp's 32 beyond); the one behind the norm reads such rows as x and multiplies its sums of row m by
// 1 / sqrt(sum of ssq[m * parts ..] / K + eps) before the bias.  A product does one of the two.
struct W4Norm {
  const float* next_w; bf16* next_x; float* next_ssq;
  const float* ssq; int parts; float eps;
};

// The r-th pair of a word as 2^-DOWN (16 + q + 8).  (One three-input operation: written as an and with a constant and an or with another it
// becomes two.)
template <int DOWN> __device__ __forceinline__ unsigned w4_pair_biased(unsigned word, int r) {
  unsigned v;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;\n" : "=r"(v) : "r"(__funnelshift_r(word, word, 4 * r)), "r"(0x00780078u), "r"(0x41804180u - DOWN * 0x00800080u));
  return v;
}
// minus 24 of it: 2^-DOWN times the levels themselves, exactly.
#define W4_MINUS_24 0xc1c0c1c0u
template <int DOWN> __device__ __forceinline__ unsigned w4_pair(unsigned word, int r) {
  const unsigned b = w4_pair_biased<DOWN>(word, r), off = W4_MINUS_24 - DOWN * 0x00800080u;
  __nv_bfloat162 v = __hadd2(*(const __nv_bfloat162*)&b, *(const __nv_bfloat162*)&off);
  return *(unsigned*)&v;
}
// The r-th pair of a word times its scale (s2: in both halves; off2: times -24 of it): (16 + q + 8) s - 24 s in one fused operation, exact,
// since 24 s and the result are bfloat16 numbers.
__device__ __forceinline__ unsigned w4_value(unsigned word, int r, unsigned s2, unsigned off2) {
  const unsigned b = w4_pair_biased<0>(word, r);
  __nv_bfloat162 v = __hfma2(*(const __nv_bfloat162*)&b, *(const __nv_bfloat162*)&s2, *(const __nv_bfloat162*)&off2);
  return *(unsigned*)&v;
}
__device__ __forceinline__ unsigned times_minus_24(unsigned s2) {
  const unsigned c = W4_MINUS_24;
  __nv_bfloat162 v = __hmul2(*(const __nv_bfloat162*)&s2, *(const __nv_bfloat162*)&c);
  return *(unsigned*)&v;
}
__device__ __forceinline__ float w4_scale_lo(unsigned s) { return __uint_as_float(s << 16); }
__device__ __forceinline__ float w4_scale_hi(unsigned s) { return __uint_as_float(s & 0xffff0000u); }
// A float32 number as three bfloat16 ones (in the upper halves), a + b + c = v exactly: 8 bits of its mantissa each (as far
// down as bfloat16 reaches, 2^-133).  An infinity or NaN is the first piece alone.
__device__ __forceinline__ void w4_split3(float v, unsigned& a, unsigned& b, unsigned& c) {
  const unsigned u = __float_as_uint(v);
  a = u & 0xffff0000u;
  const float r = (u & 0x7f800000u) == 0x7f800000u ? 0.f : v - __uint_as_float(a);
  b = __float_as_uint(r) & 0xffff0000u;
  c = __float_as_uint(r - __uint_as_float(b)) & 0xffff0000u;
  if ((u & 0x7f800000u) == 0x7f800000u && (u & 0x7fffffu)) a |= 0x400000u;                 // a NaN whose high bits are those of an infinity
}

static inline int w4_check(const W4Ref* w) {
  if (!w || !w->q || !w->s) return FELLM_ERR_ARG;
  if (w->N < 1 || w->K < 1 || w->gshift < 5 || w->gshift > 7 || w->chunks != ceil_div(w->K, W4_CHUNK)) return FELLM_ERR_SIZE;
  return w->groups == (int)(((long long)w->chunks * W4_CHUNK + (1 << w->gshift) - 1) >> w->gshift) ? 0 : FELLM_ERR_SIZE;
}

// What a product does with its sums, and the types beside it, as the launchers are told.
enum { W4_STORE = 0, W4_ACC = 1, W4_SWIGLU = 2, W4_RELU2 = 6, W4_EPI = 0xff, W4_X_BF16 = 0x100, W4_OUT_BF16 = 0x200 };
static inline int w4_check_epi(int flags, int N) {
  const int epi = flags & W4_EPI;
  if (epi != W4_STORE && epi != W4_ACC && epi != W4_SWIGLU && epi != W4_RELU2) return FELLM_ERR_ARG;
  return epi == W4_SWIGLU && N % W4_SLAB ? FELLM_ERR_SIZE : 0;
}

// SiLU(g) * u with t = exp(-|g|), which is finite and whose denominator is between 1 and 2 for every g: g / (1 + exp(-g)) is 0 from g = -88.7 on, where
// exp(-g) is no float32 number, the function down to -103 is not.
__device__ __forceinline__ float w4_silu_mul(float g, float u) {
  const float t = expf(-fabsf(g));
  return (g < 0.f ? g * t : g) / (1.0f + t) * u;
}
// The same for a bfloat16 result, by the approximate exponential and reciprocal: 2^-24 (1 + exp(-g)), with the exponential as a square, is finite and has
// a reciprocal down to g = -104, where the function goes below all numbers.  Both are good to 2^-22 and the exponential's argument adds 2^-24 of itself: 2^-20
// for small gates, 2^-18 at -16, 2^-16 at -88 beside half a step of 2^-9 or more (a gate counts down to 2^-126).  Two operations more than
// g / (1 + exp(-g)) by the same means, which is 0 from g = -87.3 on; a fifth of w4_silu_mul's (2,048 rows, 16,384 x 2,048: with that the epilogue takes longer
// than the MMAs of a tile).
__device__ __forceinline__ float w4_silu_mul_fast(float g, float u) {
  const float unit = 5.9604644775390625e-8f;                // 2^-24
  float h, r;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(h) : "f"(g * -0.72134752044448170f));
  asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(fmaf(h * unit, h, unit)));
  return g * unit * r * u;
}

// Rows of x as a product wants them where it cannot read them as they are: bfloat16 rows on no 16-byte boundary or of a K that is no
// multiple of 8 (copied, zeros up to whole chunks), and float32 rows, every 64 elements of which become three times 64 bfloat16 whose sum
// they are, the smallest first.
static __global__ void __launch_bounds__(256) w4_rows_kernel(const void* x, int x_bf16, long long ldx, unsigned short* out, int M, int K, int chunks) {
  pdl_launch_dependents();
  pdl_wait();
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  const int width = chunks * W4_CHUNK;
  const int m = (int)(i / width), k = (int)(i % width);
  if (m >= M) return;
  if (x_bf16) {
    out[i] = k < K ? ((const unsigned short*)x)[(size_t)m * ldx + k] : (unsigned short)0;
    return;
  }
  unsigned a, b, c;
  w4_split3(k < K ? ((const float*)x)[(size_t)m * ldx + k] : 0.f, a, b, c);
  unsigned short* o = out + (size_t)m * 3 * width + (size_t)(k / W4_CHUNK) * 3 * W4_CHUNK + k % W4_CHUNK;
  o[0] = (unsigned short)(c >> 16); o[W4_CHUNK] = (unsigned short)(b >> 16); o[2 * W4_CHUNK] = (unsigned short)(a >> 16);
}
static inline int w4_copy_rows(const void* x, int x_bf16, long long ldx, void* out, int M, int K, int chunks, cudaStream_t stream) {
  if ((uintptr_t)out & 15) return FELLM_ERR_ARG;
  const long long blocks = ((long long)M * chunks * W4_CHUNK + 255) / 256;
  if (blocks >= (1ll << 31)) return FELLM_ERR_SIZE;
  return launch_k_class(launch_class_for_rows(M, 0), w4_rows_kernel, dim3((unsigned)blocks, 1, 1), dim3(256, 1, 1), 0, stream, 1, x, x_bf16, ldx,
                        (unsigned short*)out, M, K, chunks);
}
