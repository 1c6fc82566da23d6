// y = x W^T of a matrix in four bits (w4.h) for a handful of rows, x bfloat16 or float32, float32 sums.
//
// mma.m16n8k16 with the weights as the 16 rows and up to eight rows of x as the columns.  A warp walks over its share of a
// slab's chunks: 16 bytes a lane are the operands of four MMAs (three shifts, four and-ors, four subtractions for 8 weights),
// the columns' operands come straight from x (a lane's eight consecutive elements feed two MMAs).  Every group's sum is
// made by itself and joins the total times its scale, in float32.  The shares of a slab's warps are added in shared memory,
// in one order.
//
// float32 rows of x are cut into three bfloat16 numbers each, x = x1 + x2 + x3 exactly (8 bits of the mantissa a piece, so
// nothing is rounded), which meet the same weights in three MMAs.
#include "w4.h"

#define GW_WARPS 8
#define GW_THREADS (32 * GW_WARPS)

enum { EPI_STORE = 0, EPI_ACC = 1, EPI_SWIGLU = 2, EPI_F32 = 3, EPI_RELU2 = 6 };      // 6: max(v, 0)^2
enum { X_BF16 = 0, X_BF16_ANY = 1, X_F32 = 2 };       // rows on 16 bytes and K a multiple of 8; any bfloat16; float32

struct GwArgs {
  W4Ref w;
  const void* x; const float* bias; void* out;
  long long ldx, ldo;
  int M, epi, out_bf16;
};

__device__ __forceinline__ void mma_bf16(float* d, const unsigned* a, unsigned b0, unsigned b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Eight elements of a row of x from k on as operand registers [part][4].
template <int XT> struct XParts { static constexpr int N = XT == X_F32 ? 3 : 1; };
template <int XT>
__device__ __forceinline__ void load_x8(const GwArgs& a, int m, int k, unsigned (*b)[4]) {
  constexpr int P = XParts<XT>::N;
#pragma unroll
  for (int p = 0; p < P; ++p)
#pragma unroll
    for (int i = 0; i < 4; ++i) b[p][i] = 0u;
  if (m >= a.M) return;
  if (XT == X_BF16) {
    if (k < a.w.K) { const uint4 v = *(const uint4*)((const bf16*)a.x + (size_t)m * a.ldx + k); b[0][0] = v.x; b[0][1] = v.y; b[0][2] = v.z; b[0][3] = v.w; }
  } else if (XT == X_BF16_ANY) {
    const unsigned short* p = (const unsigned short*)a.x + (size_t)m * a.ldx + k;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned lo = k + 2 * i < a.w.K ? p[2 * i] : 0, hi = k + 2 * i + 1 < a.w.K ? p[2 * i + 1] : 0;
      b[0][i] = lo | hi << 16;
    }
  } else {
    const float* p = (const float*)a.x + (size_t)m * a.ldx + k;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      unsigned lo[3], hi[3];
      w4_split3(k + 2 * i < a.w.K ? p[2 * i] : 0.f, lo[0], lo[1], lo[2]);
      w4_split3(k + 2 * i + 1 < a.w.K ? p[2 * i + 1] : 0.f, hi[0], hi[1], hi[2]);
#pragma unroll
      for (int q = 0; q < P; ++q) b[q][i] = lo[q] >> 16 | hi[q];
    }
  }
}

// One value of the result (two of the gated form's sums give one).
__device__ __forceinline__ void put(const GwArgs& a, int m, int n, float v) {
  const size_t o = (size_t)m * a.ldo + n;
  if (a.epi == EPI_ACC) ((float*)a.out)[o] += v;
  else {
    if (a.epi == EPI_RELU2) { v = fmaxf(v, 0.f); v *= v; }
    if (a.out_bf16) ((bf16*)a.out)[o] = __float2bfloat16_rn(v);
    else ((float*)a.out)[o] = v;
  }
}

template <int XT>
__global__ void __launch_bounds__(GW_THREADS) gemm_w4_rows_kernel(GwArgs a) {
  constexpr int P = XParts<XT>::N;
  __shared__ float red[GW_WARPS][8][W4_SLAB + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int slab = blockIdx.x, m0 = blockIdx.y * 8;
  pdl_launch_dependents();
  pdl_wait();
  // whole groups a warp
  const int per = a.w.gshift == 7 ? 2 : 1, units = (a.w.chunks + per - 1) / per;
  const int lo = (int)((long long)units * warp / GW_WARPS) * per, hi = min((int)((long long)units * (warp + 1) / GW_WARPS) * per, a.w.chunks);
  const uint4* q = a.w.q + (size_t)slab * a.w.chunks * 32 + lane;
  const unsigned* s = a.w.s + (size_t)slab * a.w.groups * 8 + g;
  float total[4] = {0.f, 0.f, 0.f, 0.f}, part[4] = {0.f, 0.f, 0.f, 0.f};
  for (int ch = lo; ch < hi; ++ch) {
    const uint4 qv = q[(size_t)ch * 32];
    const unsigned word[4] = {qv.x, qv.y, qv.z, qv.w};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      unsigned b[P][4];
      load_x8<XT>(a, m0 + g, ch * W4_CHUNK + h * 32 + c * 8, b);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        unsigned w[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) w[r] = w4_pair(word[2 * h + j], r);
#pragma unroll
        for (int p = P - 1; p >= 0; --p) mma_bf16(part, w, b[p][2 * j], b[p][2 * j + 1]);
      }
      const int k_end = ch * W4_CHUNK + (h + 1) * 32;
      if ((k_end & ((1 << a.w.gshift) - 1)) == 0 || (ch == hi - 1 && h == 1)) {
        const unsigned sv = s[(size_t)((k_end - 1) >> a.w.gshift) * 8];
        const float s0 = w4_scale_lo(sv), s1 = w4_scale_hi(sv);
        total[0] = fmaf(s0, part[0], total[0]); total[1] = fmaf(s0, part[1], total[1]);
        total[2] = fmaf(s1, part[2], total[2]); total[3] = fmaf(s1, part[3], total[3]);
        part[0] = part[1] = part[2] = part[3] = 0.f;
      }
    }
  }
  red[warp][2 * c][g] = total[0]; red[warp][2 * c + 1][g] = total[1];
  red[warp][2 * c][g + 8] = total[2]; red[warp][2 * c + 1][g + 8] = total[3];
  __syncthreads();
  const int t = threadIdx.x / W4_SLAB, r = threadIdx.x % W4_SLAB, m = m0 + t, n = slab * W4_SLAB + r;
  if (t >= 8) return;
  float v = 0.f;
#pragma unroll
  for (int w = 0; w < GW_WARPS; ++w) v += red[w][t][r];
  if (a.bias && n < a.w.N) v += a.bias[n];
  if (a.epi == EPI_SWIGLU) {
    const float up = __shfl_down_sync(0xffffffffu, v, 8);
    if (r < 8 && m < a.M && n < a.w.N) put(a, m, slab * 8 + r, glu_act(v, up, 0.f, 1.f));
  } else if (m < a.M && n < a.w.N) put(a, m, n, v);
}

// x [M, K] (x_bf16: bfloat16, else float32), out [M, N] ([M, N/2] for the gated form, whose rows are 8 gate, 8 up, ...).
FELLM_API int fellm_gemm_w4(const void* x, int x_bf16, long long ldx, const void* q, const void* s, const float* bias, void* out, int out_bf16,
                            long long ldo, int epi, int M, int N, int K, int chunks, int groups, int gshift, cudaStream_t stream) {
  if (M <= 0) return 0;
  if (!x || !q || !s || !out) return FELLM_ERR_ARG;
  if (N < 1 || K < 1 || gshift < 5 || gshift > 7 || chunks != ceil_div(K, W4_CHUNK)) return FELLM_ERR_SIZE;
  if (groups != (int)(((long long)chunks * W4_CHUNK + (1 << gshift) - 1) >> gshift)) return FELLM_ERR_SIZE;
  if (epi != EPI_STORE && epi != EPI_ACC && epi != EPI_SWIGLU && epi != EPI_F32 && epi != EPI_RELU2) return FELLM_ERR_ARG;
  if (epi == EPI_SWIGLU && N % W4_SLAB) return FELLM_ERR_SIZE;
  const GwArgs a = {{(const uint4*)q, (const unsigned*)s, N, K, chunks, groups, gshift}, x, bias, out, ldx, ldo, M, epi, out_bf16};
  const dim3 grid(ceil_div(N, W4_SLAB), ceil_div(M, 8), 1), block(GW_THREADS, 1, 1);
  if (grid.y > 65535) return FELLM_ERR_SIZE;
  if (!x_bf16) return launch_k_class(1, gemm_w4_rows_kernel<X_F32>, grid, block, 0, stream, 1, a);
  if (K % 8 == 0 && ldx % 8 == 0 && ((uintptr_t)x & 15) == 0) return launch_k_class(1, gemm_w4_rows_kernel<X_BF16>, grid, block, 0, stream, 1, a);
  return launch_k_class(1, gemm_w4_rows_kernel<X_BF16_ANY>, grid, block, 0, stream, 1, a);
}
