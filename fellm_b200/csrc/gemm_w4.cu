// y = x W^T of a matrix in four bits (w4.h) for a handful of rows, x bfloat16 or float32, float32 sums.
//
// mma.m16n8k16 with the weights as the 16 rows and up to eight rows of x as the columns.  Some warps share a slab's K; one walks
// over its share in units of four chunks.  16 bytes a lane are the operands of four MMAs (three turns, four and-ors and
// four subtractions for 8 weights, w4.h), the columns' operands come straight from x (a
// lane's eight consecutive elements feed two MMAs; the first level of cache holds them for the next slab).  Every group's sum
// is made by itself and joins the total times its scale, in float32.  The shares of a slab's warps are added in shared memory,
// in one order.
//
// A group's G products of x with levels can be 8 G times as large as x, which may be no float32 number although the result, with the scales in it,
// is one.  So the levels are unpacked as q / (8 G), exact and at no cost (the constants have other exponents): no group's sum is above the largest x,
// and none too small to be kept (x is a multiple of 2^-133, the products of 2^-143).  The total is in the same unit and leaves it at
// the end: what it loses by that lies below 2^-140.
//
// No unit is full (8 rows of 8,192 x 8,192: memory 28%, issue slots 33%, ALU 29% of the launch): a warp waits for its columns' operands, 16 bytes of x
// for every 8 of weights, of which the first level of cache has 44%, and for its own unpacking, and sixteen warps an SM do not cover both.  That product takes
// 10.7 us, with operands of x that are constants 8.8, without the unpacking 9.8, without either 6.4; one row of 65,536 x 2,048 17.0, 15.7, 14.1 and 12.0.  Every
// warp keeps three units (6.8 KB) of weights in flight through
// a ring of its own in shared memory (cp.async: no registers are held, and the ring runs on over the end of a slab), and what
// is not unpacking is shared out over four chunks.
//
// float32 rows of x are cut into three bfloat16 numbers each, x = x1 + x2 + x3 exactly (8 bits of the mantissa a piece, so
// nothing is rounded), which meet the same weights in three MMAs.  Cut by every warp for itself, that is more work than unpacking the
// weights (five rows, 8,192 x 8,192: 37 us): a large matrix has them cut once, by a launch in front.
#include "w4.h"

#define GW_DEPTH 4                     // units of a warp's ring: one is used, the others are on their way
#define GW_SLOT (4 * (512 + 64))       // a unit: four chunks' levels, their groups' scales (eight at groups of 32)
#define GW_BUFFERS 2                   // for the warps' shares, in turn, so that one barrier a segment is enough

enum { X_BF16 = 0, X_BF16_ANY = 1, X_F32 = 2, X_CUT = 3 };       // rows on 16 bytes and K a multiple of 8; any bfloat16; float32; float32 cut by w4_rows_kernel

struct GwArgs {
  W4Ref w;
  const void* x; const float* bias; void* out;
  long long ldx, ldo;
  int M, epi, out_bf16;
  int per_block, over;       // slabs a block, and how many blocks have one more
  W4Norm norm;
};

__device__ __forceinline__ void mma_bf16(float* d, const unsigned* a, unsigned b0, unsigned b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Eight elements of a row of x from k on as operand registers [part][4].
template <int XT> struct XParts { static constexpr int N = XT == X_F32 || XT == X_CUT ? 3 : 1; };
// Eight elements from p on, of which `left` are the row's.  FULL: all eight.
template <int XT, bool FULL>
__device__ __forceinline__ void load_x8(const void* at, int left, unsigned (*b)[4]) {
  constexpr int P = XParts<XT>::N;
  if (XT == X_CUT) {
#pragma unroll
    for (int q = 0; q < P; ++q) {
      const uint4 v = *(const uint4*)((const unsigned char*)at + (2 - q) * W4_CHUNK * 2);
      b[q][0] = v.x; b[q][1] = v.y; b[q][2] = v.z; b[q][3] = v.w;
    }
  } else if (XT == X_BF16) {
    const uint4 v = FULL || left > 0 ? *(const uint4*)at : make_uint4(0u, 0u, 0u, 0u);
    b[0][0] = v.x; b[0][1] = v.y; b[0][2] = v.z; b[0][3] = v.w;
  } else if (XT == X_BF16_ANY) {
    const unsigned short* p = (const unsigned short*)at;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned lo = FULL || 2 * i < left ? p[2 * i] : 0, hi = FULL || 2 * i + 1 < left ? p[2 * i + 1] : 0;
      b[0][i] = lo | hi << 16;
    }
  } else {
    const float* p = (const float*)at;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      unsigned lo[3], hi[3];
      w4_split3(FULL || 2 * i < left ? p[2 * i] : 0.f, lo[0], lo[1], lo[2]);
      w4_split3(FULL || 2 * i + 1 < left ? p[2 * i + 1] : 0.f, hi[0], hi[1], hi[2]);
#pragma unroll
      for (int q = 0; q < P; ++q) b[q][i] = lo[q] >> 16 | hi[q];
    }
  }
}

__device__ __forceinline__ void mma_bf16_first(float* d, const unsigned* a, unsigned b0, unsigned b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

// One value of the result (two of the gated form's sums give one).
__device__ __forceinline__ void put(const GwArgs& a, int m, int n, float v) {
  const size_t o = (size_t)m * a.ldo + n;
  if (a.epi == W4_ACC) ((float*)a.out)[o] += v;
  else {
    if (a.epi == W4_RELU2) { v = fmaxf(v, 0.f); v *= v; }
    if (a.out_bf16) ((bf16*)a.out)[o] = __float2bfloat16_rn(v);
    else ((float*)a.out)[o] = v;
  }
}

struct TrueType { static constexpr bool value = true; };
struct FalseType { static constexpr bool value = false; };
// (offsets as immediates: an addition for every copy and load is an instruction in thirty)
template <int DST, int SRC> __device__ __forceinline__ void cp_async16(unsigned dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0 + %2], [%1 + %3], 16;\n" ::"r"(dst), "l"(src), "n"(DST), "n"(SRC) : "memory");
}
template <int OFF> __device__ __forceinline__ uint4 lds128(unsigned at) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4 + %5];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at), "n"(OFF));
  return v;
}
template <int OFF> __device__ __forceinline__ unsigned lds32(unsigned at) {
  unsigned v;
  asm volatile("ld.shared.b32 %0, [%1 + %2];\n" : "=r"(v) : "r"(at), "n"(OFF));
  return v;
}
template <int I> struct Int { static constexpr int value = I; };
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory"); }

// What a block's warps do next with the slabs that are left of its range: t slabs side by side, `share` = warps / t warps each, t a power
// of two: whole rounds of a slab a warp (nothing to be put together), and the rest of the range by all warps too.
struct Segment {
  int slab, lo, hi;          // this warp's slab and its units of it
  int t, share;
};
__device__ __forceinline__ Segment next_segment(int slab, int left, int warp, int warps, int units) {
  Segment s;
  const int log_w = 31 - __clz(warps), log_t = min(log_w, 31 - __clz(left)), log_share = log_w - log_t;        // (left >= 1)
  s.t = 1 << log_t;
  s.share = 1 << log_share;
  const int sub = warp & (s.share - 1);
  s.slab = slab + (warp >> log_share);
  s.lo = (units * sub) >> log_share; s.hi = (units * (sub + 1)) >> log_share;
  return s;
}

// XT: what x is.  NT: tiles of eight rows of x.  GS: log2 of the group.  R: neighbouring slabs a warp takes together (a "slab" below is
// R of them, a unit 4 / R chunks of each): the same columns' operands for both.  HANDED: a norm is handed on to it or by it (a kernel of its
// own: carried by every product, its code cost 4% where it does not run).
template <int XT, int NT, int GS, int R, bool HANDED>
__maxnreg__(128) __global__ void gemm_w4_rows_kernel(GwArgs a) {
  constexpr int UNIT = 4 / R, ROWS = R * W4_SLAB, P = XParts<XT>::N, COLS = 8 * NT, XB = XT == X_F32 ? 4 : 2, XC = W4_CHUNK * XB * (XT == X_CUT ? 3 : 1);      // bytes of an element and of a chunk of x
  extern __shared__ __align__(16) unsigned char smem[];
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int all_slabs = (a.w.N + W4_SLAB - 1) / W4_SLAB, slabs = (all_slabs + R - 1) / R, m0 = blockIdx.y * COLS, cols = min(a.M - m0, COLS);
  const int first = (int)blockIdx.x * a.per_block + min((int)blockIdx.x, a.over), end = first + a.per_block + ((int)blockIdx.x < a.over ? 1 : 0);
  const unsigned ring = (unsigned)__cvta_generic_to_shared(smem) + warp * GW_DEPTH * GW_SLOT;
  float* red = reinterpret_cast<float*>(smem + (size_t)warps * GW_DEPTH * GW_SLOT);      // [GW_BUFFERS][warps][COLS][ROWS + 1]
  const int units = (a.w.chunks + UNIT - 1) / UNIT;
  constexpr int SCALES = (UNIT * W4_CHUNK) >> GS;           // groups a unit
  // what is fetched next: of which segment, how many units are left of it (a unit that ends behind the slab's last chunk takes what lies
  // behind it along)
  int f_slab = first, f_left = 0;
  unsigned f_at = ring + lane * 16;
  const uint4* fq = a.w.q;
  const unsigned* fs = a.w.s;
  size_t q2 = 0, s2 = 0;                                    // to the second slab
  auto fetch = [&]() {
    while (f_left == 0 && f_slab < end) {
      const Segment n = next_segment(f_slab, end - f_slab, warp, warps, units);
      f_slab += n.t;
      f_left = n.hi - n.lo;
      fq = a.w.q + ((size_t)(R * n.slab) * a.w.chunks + n.lo * UNIT) * 32 + lane;
      fs = a.w.s + ((size_t)(R * n.slab) * a.w.groups + n.lo * SCALES) * 8 + 4 * lane;
      if (R == 2 && 2 * n.slab + 1 < all_slabs) { q2 = (size_t)a.w.chunks * 32; s2 = (size_t)a.w.groups * 8; }
      else q2 = s2 = 0;                                      // (an odd slab's neighbour is itself)
    }
    if (f_left > 0) {
      cp_async16<0, 0>(f_at, fq); cp_async16<512, 512>(f_at, fq);
      if (R == 1) { cp_async16<1024, 1024>(f_at, fq); cp_async16<1536, 1536>(f_at, fq); }
      else { cp_async16<1024, 0>(f_at, fq + q2); cp_async16<1536, 512>(f_at, fq + q2); }
      if (lane < 2 * SCALES) {
        cp_async16<2048, 0>(f_at, fs);
        if (R == 2) cp_async16<2048 + 128, 0>(f_at, fs + s2);
      }
      fq += UNIT * 32; fs += SCALES * 8;
      --f_left;
    }
    cp_commit();
    f_at = f_at == ring + lane * 16 + (GW_DEPTH - 1) * GW_SLOT ? ring + lane * 16 : f_at + GW_SLOT;
  };
#pragma unroll 1
  for (int i = 0; i < GW_DEPTH - 1; ++i) fetch();          // (weights: nothing in front of this kernel writes them)
  pdl_launch_dependents();
  pdl_wait();
  // the rows' norm factors: row by row a warp asks for the parts now and sums them behind its first segment
  constexpr int RS_ROWS = NT == 2 ? 2 : 1;                  // rows a warp (of eight at least; 16 rows at most)
  __shared__ float row_factor[16];
  float parts[RS_ROWS][4];
  if (HANDED && a.norm.ssq) {
#pragma unroll
    for (int k = 0; k < RS_ROWS; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int m = warp + 8 * k, p = lane + 32 * i;
        parts[k][i] = warp < 8 && m < a.M && p < a.norm.parts ? a.norm.ssq[(size_t)m * a.norm.parts + p] : 0.f;
      }
  }
  const unsigned char* xrow[NT];                            // (columns behind the last row repeat it: nobody reads their sums)
#pragma unroll
  for (int t = 0; t < NT; ++t) xrow[t] = (const unsigned char*)a.x + (size_t)(m0 + min(8 * t + g, cols - 1)) * a.ldx * XB + c * 8 * XB;
  unsigned at = ring;
  int turn = 0;
  for (int next = first; next < end; turn ^= 1) {
    const Segment seg = next_segment(next, end - next, warp, warps, units);
    next += seg.t;
    float total[R][NT][4], part[R][NT][4];
#pragma unroll
    for (int k = 0; k < R; ++k)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) total[k][t][i] = 0.f;
    // chunk i of unit u, whose elements of x lie from `xu` on
    auto chunk = [&](auto idx, int u, const unsigned char* const* xu, auto full) {
      constexpr int i = decltype(idx)::value;
      unsigned b[2][NT][P][4];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int t = 0; t < NT; ++t)
          load_x8<XT, decltype(full)::value>(xu[t] + i * XC + h * 32 * XB, a.w.K - (u * UNIT + i) * W4_CHUNK - h * 32 - c * 8, b[h][t]);
#pragma unroll
      for (int k = 0; k < R; ++k) {
        const uint4 qv = k ? lds128<i * 512 + 1024>(at + lane * 16) : lds128<i * 512>(at + lane * 16);
        const unsigned word[4] = {qv.x, qv.y, qv.z, qv.w};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            unsigned w[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) w[r] = w4_pair<GS + 3>(word[2 * h + j], r);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
#pragma unroll
              for (int p = P - 1; p >= 0; --p) {
                if (j == 0 && p == P - 1 && (GS == 5 || (h == 0 && (GS == 6 || !(i & 1))))) mma_bf16_first(part[k][t], w, b[h][t][p][0], b[h][t][p][1]);
                else mma_bf16(part[k][t], w, b[h][t][p][2 * j], b[h][t][p][2 * j + 1]);
              }
            }
          }
          if (GS == 5 || (h == 1 && (GS == 6 || (i & 1) || (!decltype(full)::value && u * UNIT + i == a.w.chunks - 1)))) {
            constexpr int S0 = 2048 + (GS == 5 ? 2 * i : GS == 6 ? i : i >> 1) * 32;
            const unsigned sa = at + g * 4 + (k ? 128u : 0u), sv = GS == 5 && h ? lds32<S0 + 32>(sa) : lds32<S0>(sa);
            const float s0 = w4_scale_lo(sv), s1 = w4_scale_hi(sv);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              float* to = total[k][t];
              const float* from = part[k][t];
              to[0] = fmaf(s0, from[0], to[0]); to[1] = fmaf(s0, from[1], to[1]);
              to[2] = fmaf(s1, from[2], to[2]); to[3] = fmaf(s1, from[3], to[3]);
            }
          }
        }
      }
    };
    for (int u = seg.lo; u < seg.hi; ++u) {
      cp_wait<GW_DEPTH - 2>();
      __syncwarp();                                          // every lane's copies have come, and every lane has read the unit before
      fetch();                                               // over that one
      const unsigned char* xu[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) xu[t] = xrow[t] + (size_t)u * (UNIT * XC);
      if ((u + 1) * UNIT * W4_CHUNK <= a.w.K) {
        chunk(Int<0>(), u, xu, TrueType()); chunk(Int<1>(), u, xu, TrueType());
        if (R == 1) { chunk(Int<2 / R>(), u, xu, TrueType()); chunk(Int<3 / R>(), u, xu, TrueType()); }
      } else {
        chunk(Int<0>(), u, xu, FalseType());
        if (u * UNIT + 1 < a.w.chunks) chunk(Int<1>(), u, xu, FalseType());
        if (R == 1 && u * UNIT + 2 < a.w.chunks) chunk(Int<2 / R>(), u, xu, FalseType());
        if (R == 1 && u * UNIT + 3 < a.w.chunks) chunk(Int<3 / R>(), u, xu, FalseType());
      }
      at = at == ring + (GW_DEPTH - 1) * GW_SLOT ? ring : at + GW_SLOT;
    }
    // the warps' shares together
    float* mine = red + ((size_t)(turn * warps + warp) * COLS) * (ROWS + 1);
#pragma unroll
    for (int k = 0; k < R; ++k)
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float* p = mine + (8 * t + 2 * c) * (ROWS + 1) + k * W4_SLAB + g;
        if (8 * t + 2 * c < cols) { p[0] = total[k][t][0]; p[8] = total[k][t][2]; }
        if (8 * t + 2 * c + 1 < cols) { p[ROWS + 1] = total[k][t][1]; p[ROWS + 9] = total[k][t][3]; }
      }
    const bool factors = HANDED && a.norm.ssq && next == first + seg.t;                     // (this was the first segment)
    if (factors) {
#pragma unroll
      for (int k = 0; k < RS_ROWS; ++k) {
        float sum = (parts[k][0] + parts[k][1]) + (parts[k][2] + parts[k][3]);
        sum = warp_sum(sum);
        if (warp < 8 && lane == 0 && warp + 8 * k < 16) row_factor[warp + 8 * k] = 1.0f / sqrtf(sum / (float)a.w.K + a.norm.eps);
      }
    }
    if (seg.share == 1 && !factors) __syncwarp();
    else __syncthreads();
    const int sub = warp & (seg.share - 1);
    for (int i = 32 * sub + lane; i < (R == 2 ? cols : (cols + 1) & ~1) * ROWS; i += 32 * seg.share) {      // (whole warps: one row of x or two)
      const int t = i / ROWS, r = i % W4_SLAB, m = m0 + t, slab = R * seg.slab + (R == 2 ? (i / W4_SLAB) & 1 : 0), n = slab * W4_SLAB + r;
      const float* p = red + ((size_t)(turn * warps + warp - sub) * COLS + t) * (ROWS + 1) + i % ROWS;
      float v = 0.f;
      for (int w = 0; w < seg.share; ++w) v += p[w * COLS * (ROWS + 1)];
      v *= (float)(1 << (GS + 3));
      if (HANDED && a.norm.ssq) v *= row_factor[t];
      if (a.bias && n < a.w.N) v += a.bias[n];
      if (HANDED && a.norm.next_x) {                                   // (out += ..; N is a multiple of 16: a half warp is a row's slab)
        const bool in = t < cols && n < a.w.N;               // (the second slab of a pair may be nobody's)
        float sum = 0.f;
        if (in) {
          const size_t o = (size_t)m * a.ldo + n;
          v += ((const float*)a.out)[o];
          ((float*)a.out)[o] = v;
          a.norm.next_x[(size_t)m * a.w.N + n] = __float2bfloat16_rn(v * a.norm.next_w[n]);
          sum = v * v;
        }
#pragma unroll
        for (int x = 8; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
        if (in && r == 0) a.norm.next_ssq[(size_t)m * (a.w.N / W4_SLAB) + slab] = sum;
        continue;
      }
      if (a.epi == W4_SWIGLU) {
        const float up = __shfl_down_sync(0xffffffffu, v, 8);
        if (r < 8 && t < cols && n < a.w.N) put(a, m, slab * 8 + r, w4_silu_mul(v, up));
      } else if (t < cols && n < a.w.N) put(a, m, n, v);
    }
  }
}

template <int XT, int NT, int GS, int R, bool HANDED>
static int launch_rows(GwArgs a, cudaStream_t stream) {
  const int slabs = ceil_div(ceil_div(a.w.N, W4_SLAB), R), units = ceil_div(a.w.chunks, 4 / R), n_sm = fellm_sm_count(), tiles = ceil_div(a.M, 8 * NT);
  auto kern = gemm_w4_rows_kernel<XT, NT, GS, R, HANDED>;
  auto bytes = [](int warps) { return (size_t)warps * (GW_DEPTH * GW_SLOT + GW_BUFFERS * 8 * NT * (R * W4_SLAB + 1) * 4); };
  static int asked[64];                                 // blocks of eight warps an SM holds, asked once a device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return FELLM_ERR_ARG;
  int& resident = asked[dev];
  if (!resident) {
    int n = 0;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes(16));
    if (e != cudaSuccess) return (int)e;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, 256, bytes(8)) != cudaSuccess || n < 1) n = 1;
    resident = n;
  }
  // Two blocks of eight warps an SM (what their rings leave room for), each a range of neighbouring slabs: every slot is filled before a block
  // gets a second slab, since blocks are not spread over SMs evenly otherwise.  Few slabs: a block each, of sixteen warps where K is long
  const int warps = slabs <= n_sm && units >= 16 ? 16 : 8, per = warps == 16 ? 1 : resident;
  const dim3 grid(slabs < n_sm * per ? slabs : n_sm * per, tiles, 1);
  if (grid.y > 65535) return FELLM_ERR_SIZE;
  a.per_block = slabs / (int)grid.x; a.over = slabs % (int)grid.x;
  return launch_k_class(1, kern, grid, dim3(warps * 32, 1, 1), bytes(warps), stream, 1, a);
}
template <int XT, int NT, int R, bool HANDED = false>
static int launch_rows_group(const GwArgs& a, cudaStream_t stream) {
  return a.w.gshift == 5   ? launch_rows<XT, NT, 5, R, HANDED>(a, stream)
         : a.w.gshift == 6 ? launch_rows<XT, NT, 6, R, HANDED>(a, stream) : launch_rows<XT, NT, 7, R, HANDED>(a, stream);
}
template <bool HANDED>
static int launch_bf16_rows(const GwArgs& a, cudaStream_t stream) {
  if (a.M <= 8) return launch_rows_group<X_BF16, 1, 1, HANDED>(a, stream);
  // (9 to 16 rows: pairs of slabs where every SM gets one, 9,216 x 1,024 4.2 -> 3.8 us; else each for itself, 4,096 x 1,024 3.4 -> 2.8)
  return a.w.N <= 2 * W4_SLAB * fellm_sm_count() ? launch_rows_group<X_BF16, 2, 1, HANDED>(a, stream) : launch_rows_group<X_BF16, 2, 2, HANDED>(a, stream);
}

// x [M, K] (x_bf16: bfloat16, else float32), out [M, N] ([M, N/2] for the gated form, whose rows are 8 gate, 8 up, ...).
// scratch: null, or room for float32 rows cut in three, M x chunks x 192 numbers of bfloat16.
FELLM_API int fellm_gemm_w4(const void* x, long long ldx, const W4Ref* w, const float* bias, void* out, long long ldo, int flags, int M, void* scratch,
                            const W4Norm* norm, cudaStream_t stream) {
  if (M <= 0) return 0;
  if (!x || !out) return FELLM_ERR_ARG;
  if (int e = w4_check(w)) return e;
  if (int e = w4_check_epi(flags, w->N)) return e;
  if (norm) {
    if (M > 16 || !(flags & W4_X_BF16)) return FELLM_ERR_SIZE;
    if (norm->next_x && norm->ssq) return FELLM_ERR_ARG;
    if (norm->next_x && (!norm->next_w || !norm->next_ssq || (flags & W4_EPI) != W4_ACC || w->N % W4_SLAB || ldo < w->N)) return FELLM_ERR_ARG;
    if (norm->ssq && (norm->parts < 1 || norm->parts > 128)) return FELLM_ERR_ARG;
  }
  const int x_bf16 = flags & W4_X_BF16, K = w->K;
  GwArgs a = {*w, x, bias, out, ldx, ldo, M, flags & W4_EPI, (flags & W4_OUT_BF16) != 0, 0, 0, norm ? *norm : W4Norm{}};
  if (!x_bf16 && scratch) {
    if (int e = w4_copy_rows(x, 0, ldx, scratch, M, K, w->chunks, stream)) return e;
    a.x = scratch; a.ldx = 3ll * w->chunks * W4_CHUNK;
    return launch_rows_group<X_CUT, 1, 1>(a, stream);
  }
  if (!x_bf16) return launch_rows_group<X_F32, 1, 1>(a, stream);
  if (K % 8 || ldx % 8 || ((uintptr_t)x & 15)) return norm ? FELLM_ERR_SIZE : launch_rows_group<X_BF16_ANY, 1, 1>(a, stream);
  return norm ? launch_bf16_rows<true>(a, stream) : launch_bf16_rows<false>(a, stream);
}
