// y = x W^T of a matrix in four bits (w4.h) for a handful of rows, x bfloat16 or float32, float32 sums.
//
// mma.m16n8k16 with the weights as the 16 rows and up to eight rows of x as the columns.  Some warps share a slab's K; one walks
// over its share in units of four chunks.  16 bytes a lane are the operands of four MMAs (three turns, four and-ors and
// four subtractions for 8 weights, w4.h), the columns' operands come straight from x (a
// lane's eight consecutive elements feed two MMAs; the first level of cache holds them for the next slab).  Every group's sum
// is made by itself and joins the total times its scale, in float32.  The shares of a slab's warps are added in shared memory,
// in one order.
//
// Bound by the matrix's bytes where enough of them are on their way and by the instructions that unpack them: an SM's four
// schedulers have some 86 cycles each for a chunk that memory delivers.  So every warp keeps two units (4 KB) in flight through
// a ring of its own in shared memory (cp.async: no registers are held, and the ring runs on over the end of a slab), and what
// is not unpacking is shared out over four chunks.
//
// float32 rows of x are cut into three bfloat16 numbers each, x = x1 + x2 + x3 exactly (8 bits of the mantissa a piece, so
// nothing is rounded), which meet the same weights in three MMAs.
#include "w4.h"

#define GW_UNIT 4                      // chunks
#define GW_DEPTH 3                     // units of a warp's ring: one is used, the others are on their way
#define GW_SLOT (GW_UNIT * (512 + 64)) // a unit's levels, its groups' scales (eight at groups of 32)

enum { EPI_STORE = 0, EPI_ACC = 1, EPI_SWIGLU = 2, EPI_F32 = 3, EPI_RELU2 = 6 };      // 6: max(v, 0)^2
enum { X_BF16 = 0, X_BF16_ANY = 1, X_F32 = 2 };       // rows on 16 bytes and K a multiple of 8; any bfloat16; float32

struct GwArgs {
  W4Ref w;
  const void* x; const float* bias; void* out;
  long long ldx, ldo;
  int M, epi, out_bf16;
  int share;                 // warps that share a slab: a power of two, all of a block's warps in such groups
};

__device__ __forceinline__ void mma_bf16(float* d, const unsigned* a, unsigned b0, unsigned b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Eight elements of a row of x from k on as operand registers [part][4].
template <int XT> struct XParts { static constexpr int N = XT == X_F32 ? 3 : 1; };
// `row` points to the row's element 0.  FULL: all eight are there.
template <int XT, bool FULL>
__device__ __forceinline__ void load_x8(const void* row, int k, int K, unsigned (*b)[4]) {
  constexpr int P = XParts<XT>::N;
  if (XT == X_BF16) {
    const uint4 v = FULL || k < K ? *(const uint4*)((const bf16*)row + k) : make_uint4(0u, 0u, 0u, 0u);
    b[0][0] = v.x; b[0][1] = v.y; b[0][2] = v.z; b[0][3] = v.w;
  } else if (XT == X_BF16_ANY) {
    const unsigned short* p = (const unsigned short*)row + k;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned lo = FULL || k + 2 * i < K ? p[2 * i] : 0, hi = FULL || k + 2 * i + 1 < K ? p[2 * i + 1] : 0;
      b[0][i] = lo | hi << 16;
    }
  } else {
    const float* p = (const float*)row + k;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      unsigned lo[3], hi[3];
      w4_split3(FULL || k + 2 * i < K ? p[2 * i] : 0.f, lo[0], lo[1], lo[2]);
      w4_split3(FULL || k + 2 * i + 1 < K ? p[2 * i + 1] : 0.f, hi[0], hi[1], hi[2]);
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

struct TrueType { static constexpr bool value = true; };
struct FalseType { static constexpr bool value = false; };
__device__ __forceinline__ void cp_async16(unsigned dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory"); }

// XT: what x is.  NT: tiles of eight rows of x.  GS: log2 of the group.
template <int XT, int NT, int GS>
__global__ void __launch_bounds__(512) gemm_w4_rows_kernel(GwArgs a) {
  constexpr int P = XParts<XT>::N, COLS = 8 * NT;
  extern __shared__ __align__(16) unsigned char smem[];
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int slabs = (a.w.N + W4_SLAB - 1) / W4_SLAB, m0 = blockIdx.y * COLS, cols = min(a.M - m0, COLS);
  const int group = warp / a.share, sub = warp % a.share, groups = warps / a.share;
  const int first = blockIdx.x * groups + group, step = gridDim.x * groups;
  const unsigned char* ring = smem + (size_t)warp * GW_DEPTH * GW_SLOT;
  const unsigned ring_at = (unsigned)__cvta_generic_to_shared(ring);
  float* red = reinterpret_cast<float*>(smem + (size_t)warps * GW_DEPTH * GW_SLOT);      // [2][warps][COLS][17]
  // this warp's units of every slab
  const int units = (a.w.chunks + GW_UNIT - 1) / GW_UNIT, lo = units * sub / a.share, hi = units * (sub + 1) / a.share;
  constexpr int SCALES = 256 >> GS;                         // groups a unit
  int f_slab = first, f_unit = lo;
  unsigned f_at = ring_at;
  const uint4* fq = a.w.q + ((size_t)f_slab * a.w.chunks + lo * GW_UNIT) * 32 + lane;
  const unsigned* fs = a.w.s + ((size_t)f_slab * a.w.groups + lo * SCALES) * 8 + 4 * lane;
  // (a unit that ends behind the slab's last chunk takes what lies behind it along)
  auto fetch = [&]() {
    if (f_slab < slabs && lo < hi) {
#pragma unroll
      for (int i = 0; i < GW_UNIT; ++i) cp_async16(f_at + i * 512 + lane * 16, fq + i * 32);
      if (lane < 2 * SCALES) cp_async16(f_at + GW_UNIT * 512 + lane * 16, fs);
      fq += GW_UNIT * 32; fs += SCALES * 8;
      if (++f_unit == hi) {
        f_unit = lo; f_slab += step;
        fq = a.w.q + ((size_t)f_slab * a.w.chunks + lo * GW_UNIT) * 32 + lane;
        fs = a.w.s + ((size_t)f_slab * a.w.groups + lo * SCALES) * 8 + 4 * lane;
      }
    }
    cp_commit();
    f_at = f_at == ring_at + (GW_DEPTH - 1) * GW_SLOT ? ring_at : f_at + GW_SLOT;
  };
#pragma unroll
  for (int i = 0; i < GW_DEPTH - 1; ++i) fetch();          // (weights: nothing in front of this kernel writes them)
  pdl_launch_dependents();
  pdl_wait();
  const unsigned char* xrow[NT];                            // (columns behind the last row repeat it: nobody reads their sums)
#pragma unroll
  for (int t = 0; t < NT; ++t) xrow[t] = (const unsigned char*)a.x + (size_t)(m0 + min(8 * t + g, cols - 1)) * a.ldx * (XT == X_F32 ? 4 : 2);
  const unsigned char* at = ring;
  int turn = 0;
  for (int slab = first; slab < slabs; slab += step, turn ^= 1) {
    float total[NT][4], part[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) total[t][i] = part[t][i] = 0.f;
    auto chunk = [&](int i, int ch, auto full) {
      unsigned b[2][NT][P][4];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int t = 0; t < NT; ++t) load_x8<XT, decltype(full)::value>(xrow[t], ch * W4_CHUNK + h * 32 + c * 8, a.w.K, b[h][t]);
      const uint4 qv = *(const uint4*)(at + i * 512 + lane * 16);
      const unsigned word[4] = {qv.x, qv.y, qv.z, qv.w};
      const unsigned* sc = (const unsigned*)(at + GW_UNIT * 512) + g;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          unsigned w[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) w[r] = w4_pair(word[2 * h + j], r);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
#pragma unroll
            for (int p = P - 1; p >= 0; --p) mma_bf16(part[t], w, b[h][t][p][2 * j], b[h][t][p][2 * j + 1]);
          }
        }
        if (GS == 5 || (h == 1 && (GS == 6 || (i & 1) || ch == a.w.chunks - 1))) {
          const unsigned sv = sc[(GS == 5 ? 2 * i + h : GS == 6 ? i : i >> 1) * 8];
          const float s0 = w4_scale_lo(sv), s1 = w4_scale_hi(sv);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            total[t][0] = fmaf(s0, part[t][0], total[t][0]); total[t][1] = fmaf(s0, part[t][1], total[t][1]);
            total[t][2] = fmaf(s1, part[t][2], total[t][2]); total[t][3] = fmaf(s1, part[t][3], total[t][3]);
            part[t][0] = part[t][1] = part[t][2] = part[t][3] = 0.f;
          }
        }
      }
    };
    for (int u = lo; u < hi; ++u) {
      cp_wait<GW_DEPTH - 2>();
      __syncwarp();                                          // every lane's copies have come, and every lane has read the unit before
      fetch();                                               // over that one
      if ((u + 1) * GW_UNIT * W4_CHUNK <= a.w.K) {
#pragma unroll
        for (int i = 0; i < GW_UNIT; ++i) chunk(i, u * GW_UNIT + i, TrueType());
      } else {
#pragma unroll
        for (int i = 0; i < GW_UNIT; ++i) if (u * GW_UNIT + i < a.w.chunks) chunk(i, u * GW_UNIT + i, FalseType());
      }
      at = at == ring + (GW_DEPTH - 1) * GW_SLOT ? ring : at + GW_SLOT;
    }
    // the warps' shares together: two buffers in turn, so that one barrier a slab is enough
    float* mine = red + ((size_t)(turn * warps + warp) * COLS) * 17;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float* p = mine + (8 * t + 2 * c) * 17 + g;
      if (8 * t + 2 * c < cols) { p[0] = total[t][0]; p[8] = total[t][2]; }
      if (8 * t + 2 * c + 1 < cols) { p[17] = total[t][1]; p[25] = total[t][3]; }
    }
    if (a.share == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;\n" ::"r"(1 + group), "r"(32 * a.share) : "memory");
    for (int i = 32 * sub + lane; i < ((cols + 1) & ~1) * W4_SLAB; i += 32 * a.share) {         // (a warp takes two rows of x)
      const int t = i / W4_SLAB, r = i % W4_SLAB, m = m0 + t, n = slab * W4_SLAB + r;
      const float* p = red + ((size_t)(turn * warps + group * a.share) * COLS + t) * 17 + r;
      float v = 0.f;
      for (int w = 0; w < a.share; ++w) v += p[w * COLS * 17];
      if (a.bias && n < a.w.N) v += a.bias[n];
      if (a.epi == EPI_SWIGLU) {
        const float up = __shfl_down_sync(0xffffffffu, v, 8);
        if (r < 8 && t < cols && n < a.w.N) put(a, m, slab * 8 + r, glu_act(v, up, 0.f, 1.f));
      } else if (t < cols && n < a.w.N) put(a, m, n, v);
    }
  }
}

template <int XT, int NT, int GS>
static int launch_rows(GwArgs a, cudaStream_t stream) {
  const int slabs = ceil_div(a.w.N, W4_SLAB), units = ceil_div(a.w.chunks, GW_UNIT), n_sm = fellm_sm_count(), tiles = ceil_div(a.M, 8 * NT);
  auto kern = gemm_w4_rows_kernel<XT, NT, GS>;
  auto bytes = [](int warps) { return (size_t)warps * (GW_DEPTH * GW_SLOT + 2 * 8 * NT * 17 * 4); };
  static int resident = 0;                              // blocks of eight warps an SM holds, asked once
  if (!resident) {
    int n = 0;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes(16));
    if (e != cudaSuccess) return (int)e;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, 256, bytes(8)) != cudaSuccess || n < 1) n = 1;
    resident = n;
  }
  // how many warps share a slab: the time of the busiest warp, in units and some three quarters of one for the end of a slab
  const int most = resident * 8 * n_sm;
  int best = 1;
  double best_t = 1e30;
  for (int share = 1; share <= 16 && share <= units; share *= 2) {
    const double t = (double)ceil_div(slabs, most / share < 1 ? 1 : most / share) * (ceil_div(units, share) + 0.75);
    if (t < best_t) { best_t = t; best = share; }
  }
  a.share = best;
  const int warps = best == 16 ? 16 : slabs <= n_sm * (8 / best) ? best : 8;       // (few slabs: a block each)
  const int groups = warps / best, want = ceil_div(slabs, groups), fit = resident * 8 / warps * n_sm;
  const dim3 grid(want < fit ? want : (fit > 0 ? fit : n_sm), tiles, 1);
  if (grid.y > 65535) return FELLM_ERR_SIZE;
  return launch_k_class(1, kern, grid, dim3(warps * 32, 1, 1), bytes(warps), stream, 1, a);
}
template <int XT, int NT>
static int launch_rows_group(const GwArgs& a, cudaStream_t stream) {
  return a.w.gshift == 5 ? launch_rows<XT, NT, 5>(a, stream) : a.w.gshift == 6 ? launch_rows<XT, NT, 6>(a, stream) : launch_rows<XT, NT, 7>(a, stream);
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
  const GwArgs a = {{(const uint4*)q, (const unsigned*)s, N, K, chunks, groups, gshift}, x, bias, out, ldx, ldo, M, epi, out_bf16, 1};
  if (!x_bf16) return launch_rows_group<X_F32, 1>(a, stream);
  if (K % 8 || ldx % 8 || ((uintptr_t)x & 15)) return launch_rows_group<X_BF16_ANY, 1>(a, stream);
  return M <= 8 ? launch_rows_group<X_BF16, 1>(a, stream) : M <= 16 ? launch_rows_group<X_BF16, 2>(a, stream) : launch_rows_group<X_BF16, 4>(a, stream);
}
