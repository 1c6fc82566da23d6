// y = x W^T of a matrix in four bits (w4.h) for more than a handful of rows, on tcgen05: D[n, t] = sum_k W[n, k] x[t, k], the
// MMA's 128 rows are weight rows, its 16 to 256 columns are rows of x.
//
// The weights become bfloat16 on their way to the MMA: level * scale is a bfloat16 number exactly (w4.h), so this
// rounds nothing, and K may be summed whatever the groups.  (16 + level + 8) is a shift and an and-or away (the
// four bits at the top of bfloat16's mantissa at exponent 4), and one fused multiply-add makes (that) * s - 24 s: both 24 s and the
// result are bfloat16 numbers.  Sixteen warps do this, eight a stage, the next stage's eight at the same time.
//
// Tiles of up to 128 rows of x (KB 2: two chunks of K a stage) have their weights in TENSOR memory, a lane a row: the levels come through a
// ring of each warp's own (cp.async) and leave by tcgen05.st.  In shared memory, writing them and the MMA's reading them take 256 of the
// some 340 cycles a chunk, whatever the width (32 rows, 8,192 x 8,192: 17.4 us, in tensor memory 15.8; 128 rows: 23.3 and 21.6).
// Wider tiles (KB 1) need tensor memory for their sums and are bound by the MMAs: there the weights go to shared memory in the 128-byte
// swizzle, a warp a slab of 16 rows, 16 bytes a lane from memory, several chunks ahead in registers.
// x comes by TMA, one thread issues the MMAs, four warps store what is finished: lane = weight row, so a row of the result
// leaves in pieces of 32 neighbouring columns.
//
// Persistent over tiles with two accumulators in tensor memory; where there are too few tiles for the SMs, the K range of a
// tile is shared out over a cluster of 2, 4 or 8 CTAs, whose sums are put together through distributed shared memory, in
// rank order, each rank finishing its share of the columns, four at a time.  A decode step's products are a few microseconds, a good part
// of it code that runs once: a short loop over four columns beats straight code for sixteen, and every long division in front of
// the first load shows (32 requests of a 16-layer model of width 1,024: 0.553 -> 0.495 ms a step by these).
//
// Measured, a few one after another from a graph: 64 rows, 8,192 x 8,192 17.4 us (floor 5.8: unpacking bounds it, some 280 cycles a chunk, and
// 7 us of launch, first loads, exchange and stores); 2,048 rows, gated 16,384 x 2,048 104 us, 1,320 TFLOP/s; 4,096 rows, 8,192 x 8,192
// 408 us, 1,350 TFLOP/s.  Repeated for a second the GPU runs at its power's clock: the gated product 121 us, 1,135 TFLOP/s at 1,410 MHz.
//
// Roles in a CTA: warp 0 TMA of x (one lane), warp 1 MMA issuer (one lane) and owner of tensor memory, then two sets of
// eight warps for weights, the last four warps epilogue (tensor memory lanes 32 (warp % 4) ..).  Every wait on an mbarrier is bounded: after a
// second a role records itself in `status` (141 x, 142 MMA, 143 weights, 144 epilogue, 145 accumulator) and all roles run
// through to the common exit, where tensor memory is freed.
#include <cuda.h>
#include "w4.h"

#define SETS 2                         // sets of eight warps that make weights, each every other stage (three took registers from one another)
#define W4U_THREADS (32 * (2 + 8 * SETS + 4))
#define W4U_SPIN_LIMIT (1u << 26)
#define W4U_A_BYTES (128 * 128)        // 128 weight rows x 64 k

__device__ __forceinline__ unsigned smem_u32(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(unsigned bar, unsigned count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(bar), "r"(count)); }
__device__ __forceinline__ void mbar_expect_tx(unsigned bar, unsigned bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(unsigned bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(bar) : "memory"); }
__device__ __forceinline__ bool mbar_try(unsigned bar, unsigned parity) {
  unsigned ok;
  asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
// Bounded wait: after some 2^31 cycles, a second (by the SM's own clock: reading the global timer takes longer than most waits
// here), it records `code` and sets `dead`, and from then on no wait of this CTA waits: all roles run through to the common exit,
// the same way as ever (so that no role's loop has to carry a verdict; what they store is of no use, and the status word says so).
__device__ __forceinline__ void wait_slow(unsigned bar, unsigned parity, int* status, int code, volatile int* dead, unsigned nap) {
  pdl_wait();                                               // (what the kernel in front takes is not counted)
  const long long t0 = clock64();
  for (unsigned i = 0; i < W4U_SPIN_LIMIT; ++i) {
    if (mbar_try(bar, parity) || *dead) return;
    if (nap) __nanosleep(nap);
    if ((i & 63) == 63 && clock64() - t0 > (1ll << 31)) break;
  }
  *dead = 1;
  if (status) atomicExch(status, code);
}
#define W4U_WAIT(bar, parity, code) \
  do { if (!mbar_try(bar, parity)) wait_slow(bar, parity, a.status, code, &dead, 0); } while (0)
// The epilogue's wait for a finished accumulator, most of a tile's time: one warp asks, now and then (four that ask all the time
// took a third of the issue slots), the others sleep at a barrier.
#define W4U_WAIT_EPILOGUE(bar, parity) \
  do { \
    if (warp == 2 + 8 * SETS && !mbar_try(bar, parity)) wait_slow(bar, parity, a.status, 144, &dead, 64); \
    asm volatile("bar.sync 1, 128;\n" ::: "memory"); \
  } while (0)
__device__ __forceinline__ void tma_load_2d(unsigned dst, const CUtensorMap* map, int c0, int c1, unsigned bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n"
               ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1) : "memory");
}
// K-major operand tile, rows of 128 bytes, 128-byte swizzle, 8-row groups 1024 bytes apart: the descriptor's upper word, and its
// lower one from the address (a further piece of 32 bytes of K is 2 more).
#define W4U_DESC_HI ((1024u >> 4) | 1u << 14 | 2u << 29)
__device__ __forceinline__ unsigned umma_desc_lo(unsigned smem_addr) { return (smem_addr & 0x3FFFF) >> 4; }
// kind::f16: D float32, A and B bfloat16, both K-major.
__device__ __forceinline__ unsigned umma_idesc(int m, int n) { return 1u << 4 | 1u << 7 | 1u << 10 | (unsigned)(n >> 3) << 17 | (unsigned)(m >> 4) << 24; }
// The four MMAs of a stage's 64 k.
__device__ __forceinline__ void umma_stage(unsigned d, unsigned a_lo, unsigned b_lo, unsigned idesc, unsigned accumulate) {
#pragma unroll
  for (int k = 0; k < 4; ++k)
    asm volatile("{\n.reg .pred p;\n.reg .b64 da, db;\nsetp.ne.b32 p, %4, 0;\nmov.b64 da, {%1, %5};\nmov.b64 db, {%2, %5};\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n}\n"
                 ::"r"(d), "r"(a_lo + 2 * k), "r"(b_lo + 2 * k), "r"(idesc), "r"(k ? 1u : accumulate), "r"(W4U_DESC_HI) : "memory");
}
// The same with the weights in tensor memory (a lane a row, two k a column): 8 columns an MMA.
__device__ __forceinline__ void umma_stage_tmem(unsigned d, unsigned a, unsigned b_lo, unsigned idesc, unsigned accumulate) {
#pragma unroll
  for (int k = 0; k < 4; ++k)
    asm volatile("{\n.reg .pred p;\n.reg .b64 db;\nsetp.ne.b32 p, %4, 0;\nmov.b64 db, {%2, %5};\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n}\n"
                 ::"r"(d), "r"(a + 8 * k), "r"(b_lo + 2 * k), "r"(idesc), "r"(k ? 1u : accumulate), "r"(W4U_DESC_HI) : "memory");
}
// One lane of a converged warp, the same one every time.  (A role's loop runs in the whole warp, so that its counters and
// descriptors are uniform; a loop inside `if (lane == 0)` took some 800 cycles a stage for its scalar arithmetic.)
__device__ __forceinline__ bool elect_one() {
  unsigned p;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ void umma_commit(unsigned bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_ld16(unsigned taddr, float* v) {
  unsigned* r = reinterpret_cast<unsigned*>(v);
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
                 "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(taddr) : "memory");
  asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
}
__device__ __forceinline__ void tmem_ld4(unsigned taddr, float* v) {
  unsigned* r = reinterpret_cast<unsigned*>(v);
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(taddr) : "memory");
  asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
}
// 16 columns += 16 others (one wait for both; tmem_st_wait() behind the last of them).
__device__ __forceinline__ void tmem_add16(unsigned to, unsigned from) {
  unsigned r[16], f[16];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%32];\n"
               "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%33];\n"
               "tcgen05.wait::ld.sync.aligned;\n"
               : "=&r"(r[0]), "=&r"(r[1]), "=&r"(r[2]), "=&r"(r[3]), "=&r"(r[4]), "=&r"(r[5]), "=&r"(r[6]), "=&r"(r[7]), "=&r"(r[8]), "=&r"(r[9]), "=&r"(r[10]),
                 "=&r"(r[11]), "=&r"(r[12]), "=&r"(r[13]), "=&r"(r[14]), "=&r"(r[15]), "=&r"(f[0]), "=&r"(f[1]), "=&r"(f[2]), "=&r"(f[3]), "=&r"(f[4]), "=&r"(f[5]),
                 "=&r"(f[6]), "=&r"(f[7]), "=&r"(f[8]), "=&r"(f[9]), "=&r"(f[10]), "=&r"(f[11]), "=&r"(f[12]), "=&r"(f[13]), "=&r"(f[14]), "=&r"(f[15])
               : "r"(to), "r"(from) : "memory");
#pragma unroll
  for (int j = 0; j < 16; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) + __uint_as_float(f[j]));
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};\n"
               ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
                 "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(to) : "memory");
}
__device__ __forceinline__ void tmem_st32(unsigned taddr, const unsigned* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,"
               "%27,%28,%29,%30,%31};\n"
               ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
                 "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
                 "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }
template <int N> __device__ __forceinline__ void tmem_ld(unsigned at, float* v) {
  if (N == 16) tmem_ld16(at, v);
  else tmem_ld4(at, v);
}
// N columns of a tile's sums: of an accumulator and the one `before` columns from it (0: of one run), each the sums of two that lie `lo` columns
// apart (0: of one).
template <int N> __device__ __forceinline__ void tmem_sums(unsigned at, unsigned lo, unsigned before, float* v) {
  float more[N];
  tmem_ld<N>(at, v);
  if (before) {
    tmem_ld<N>(at + before, more);
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] += more[j];
  }
  if (!lo) return;
  tmem_ld<N>(at + lo, more);
  if (before) {
    float last[N];
    tmem_ld<N>(at + before + lo, last);
#pragma unroll
    for (int j = 0; j < N; ++j) more[j] += last[j];
  }
#pragma unroll
  for (int j = 0; j < N; ++j) v[j] += more[j];
}
__device__ __forceinline__ unsigned cluster_rank() { unsigned r; asm("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r)); return r; }
__device__ __forceinline__ unsigned mapa(unsigned addr, unsigned rank) {
  unsigned r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void st_cluster_v4(unsigned addr, float a, float b, float c, float d) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};\n" ::"r"(addr), "f"(a), "f"(b), "f"(c), "f"(d) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}

// PARTS 1: x as it is; 3: every 64 columns of x are three times 64, whose sum they are.
struct W4uArgs {
  W4Ref w;
  const float* bias; void* out; int* status;
  long long ldo;
  int M;
  int bn;                    // rows of x a tile, a multiple of 16, <= 256
  int m_tiles, total;        // tiles along x, and all of them
  int stages, splits, log_splits, tmem_cols;
  int run;                   // blocks of K that are summed in one accumulator
  int raw_at, w_col;         // KB 2: where the warps' rings lie, from the stages on; the first column of tensor memory of the weights
  int buffers, acc_cols;     // accumulators (used in turn), columns of tensor memory from one to the next
  int share;                 // columns of a tile that a rank of a cluster finishes, a multiple of 4
  int recv_apart;            // what other ranks send lies behind the stages, not over them
  W4Norm norm;
};
// The tensor cores cut a sum's last bits off where they add to it, always towards zero: float32 results of bfloat16 rows were off by 8e-8 of
// themselves over 512 k, 1.8e-7 over 1,024, 4.1e-7 over 2,048, 1.0e-6 over 4,096, 2.4e-6 over 8,192, and those of float32 rows by as much again
// for each of their small pieces' products.  So K is summed in runs of up to 48 chunks, which float32
// additions put together, and the two small pieces of float32 rows have an accumulator of their own.  bfloat16 results too, though half a
// step of theirs is 2e-3 or more: what is cut off has a direction, goes with the largest of the sums on the way (sums over
// 2^20 k that come back to a thirtieth of it: 3% of the result) and rounds the wrong way (1,029 x [2,056 x 8,192]: 0.14% of the results, in
// runs 0.05%; 40.4 -> 42.3 us, 2,048 x [8,192 x 8,192] 204 -> 207).  A short K is one run and takes what it took.
#define W4U_RUN 48
#define W4U_RAW 4                     // units of a warp's ring of levels (KB 2): two slabs' chunk, their scales
#define W4U_RAW_SLOT 1152
#define W4U_NORM_ROWS 128             // rows of a product that a norm is handed on to or by: one tile's

__device__ __forceinline__ void st_shared_v4(unsigned addr, unsigned a, unsigned b, unsigned c, unsigned d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

__device__ __forceinline__ unsigned ld_shared(unsigned addr) {
  unsigned v;
  asm volatile("ld.shared.b32 %0, [%1];\n" : "=r"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint4 ld_shared_v4(unsigned addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ void copy16(unsigned dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src) : "memory"); }

// Neighbouring lanes, features n and n + 1, hold columns x and y each: the even one stores both features of x, the odd one of y.
template <bool BF16> __device__ __forceinline__ void store_pair(unsigned char* p, float x, float y, int hi, bool in) {
  if (BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
    const unsigned own = *(const unsigned*)&v, other = __shfl_xor_sync(0xffffffffu, own, 1);
    if (in) *(unsigned*)p = __byte_perm(own, other, hi ? 0x3276 : 0x5410);
  } else {
    const float other = __shfl_xor_sync(0xffffffffu, hi ? x : y, 1);
    if (in) *(float2*)p = hi ? make_float2(other, y) : make_float2(x, other);
  }
}
template <bool BF16> __device__ __forceinline__ void store1(unsigned char* p, float x) {
  if (BF16) *(bf16*)p = __float2bfloat16_rn(x);
  else *(float*)p = x;
}

// COLS finished columns (rows of x from m on, `rows` of them count) of weight row n, a warp's lanes neighbouring weight rows.  The
// result leaves in pairs of features where they lie on a pair's boundary: neighbouring lanes give each other one of two columns
// (bfloat16, 2,048 rows, 16,384 x 2,048: 122 us a feature at a time, 104 in pairs).
template <int EPI, bool BF16, int COLS>
__device__ __forceinline__ void finish_some(const W4uArgs& a, float* v, int m, int rows, int n, float bias, bool pairs) {
  constexpr int SIZE = BF16 ? 2 : 4;
  const int lane = threadIdx.x & 31, hi = lane & 1;
  const bool in = n < a.w.N;
  const size_t row = (size_t)a.ldo * SIZE;
#pragma unroll
  for (int j = 0; j < COLS; ++j) v[j] += bias;
  if (EPI == W4_SWIGLU) {
    // lanes 8..15 and 24..31 hold what the eight before them are multiplied with: those take the even columns, these the odd
    const bool gate = !(lane & 8);
    const int f = ((n & ~15) >> 1) + (lane & 7), odd = gate ? 0 : 1;
    float z[COLS / 2];
#pragma unroll
    for (int j = 0; j < COLS; j += 2) {
      const float other = __shfl_xor_sync(0xffffffffu, gate ? v[j + 1] : v[j], 8), g = gate ? v[j] : other, u = gate ? other : v[j + 1];
      z[j >> 1] = BF16 ? w4_silu_mul_fast(g, u) : w4_silu_mul(g, u);
    }
    if (pairs) {
      const int first = odd + 2 * hi;                        // this lane's column of the first four
      unsigned char* p = (unsigned char*)a.out + ((size_t)(m + first) * a.ldo + (f & ~1)) * SIZE;
#pragma unroll
      for (int j = 0; j < COLS / 2; j += 2, p += 4 * row) {
        store_pair<BF16>(p, z[j], z[j + 1], hi, in && 2 * j + first < rows);
      }
    } else if (in) {
      unsigned char* p = (unsigned char*)a.out + ((size_t)(m + odd) * a.ldo + f) * SIZE;
#pragma unroll
      for (int j = 0; j < COLS / 2; ++j, p += 2 * row) if (2 * j + odd < rows) store1<BF16>(p, z[j]);
    }
    return;
  }
  if (EPI == W4_RELU2) {
#pragma unroll
    for (int j = 0; j < COLS; ++j) { v[j] = fmaxf(v[j], 0.f); v[j] *= v[j]; }
  }
  if (pairs) {
    unsigned char* p = (unsigned char*)a.out + ((size_t)(m + hi) * a.ldo + (n & ~1)) * SIZE;
#pragma unroll
    for (int j = 0; j < COLS; j += 2, p += 2 * row) store_pair<BF16>(p, v[j], v[j + 1], hi, in && j + hi < rows);
  } else if (in) {
    unsigned char* p = (unsigned char*)a.out + ((size_t)m * a.ldo + n) * SIZE;
    float old[COLS];
    if (EPI == W4_ACC) {
      const unsigned char* from = p;
#pragma unroll
      for (int j = 0; j < COLS; ++j, from += row) if (j < rows) old[j] = *(const float*)from;
    }
#pragma unroll
    for (int j = 0; j < COLS; ++j, p += row) if (j < rows) store1<BF16>(p, EPI == W4_ACC ? v[j] + old[j] : v[j]);
  }
}
// What out += .. adds to in COLS columns from m on, as store_pair will write it.
template <int COLS> __device__ __forceinline__ void load_old(const W4uArgs& a, float2* old, int m, int rows, int n) {
  const int hi = threadIdx.x & 1;
  const float* p = (const float*)a.out + (size_t)(m + hi) * a.ldo + (n & ~1);
#pragma unroll
  for (int j = 0; j < COLS / 2; ++j, p += 2 * a.ldo) old[j] = n < a.w.N && 2 * j + hi < rows ? *(const float2*)p : make_float2(0.f, 0.f);
}
// What the neighbouring lane will store of this lane's feature belongs to its own sum.
template <int COLS> __device__ __forceinline__ void add_old(float* v, const float2* old) {
  const bool hi = threadIdx.x & 1;
#pragma unroll
  for (int j = 0; j < COLS; j += 2) {
    const float mine = hi ? old[j / 2].y : old[j / 2].x, others = hi ? old[j / 2].x : old[j / 2].y;
    const float got = __shfl_xor_sync(0xffffffffu, others, 1);
    v[j] += hi ? got : mine; v[j + 1] += hi ? mine : got;
  }
}
// COLS finished columns of out += .. (rows of x from m on) as the norm behind them wants them: their squares' sums over the warp's 32
// features (a lane keeps half of its columns and gives away the other half, until it has one) and the weighted rows.
template <int COLS> __device__ __forceinline__ void hand_on(const W4uArgs& a, const float* v, int m, int rows, int n, float weight) {
  const int lane = threadIdx.x & 31, hi = lane & 1, column = (lane >> 1) & (COLS - 1);
  const bool in = n < a.w.N;
  float s[COLS];
#pragma unroll
  for (int j = 0; j < COLS; ++j) s[j] = v[j] * v[j];
#pragma unroll
  for (int half = COLS / 2; half > 0; half >>= 1) {
    const bool upper = lane & (2 * half);
#pragma unroll
    for (int j = 0; j < half; ++j) {
      const float give = upper ? s[j] : s[j + half], keep = upper ? s[j + half] : s[j];
      s[j] = keep + __shfl_xor_sync(0xffffffffu, give, 2 * half);
    }
  }
  float sum = s[0] + __shfl_xor_sync(0xffffffffu, s[0], 1);
#pragma unroll
  for (int bit = 2 * COLS; bit < 32; bit *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, bit);
  if (in && lane == 2 * column && column < rows) a.norm.next_ssq[(size_t)(m + column) * (a.w.N / 32) + n / 32] = sum;
  unsigned char* p = (unsigned char*)(a.norm.next_x + (size_t)(m + hi) * a.w.N + (n & ~1));
#pragma unroll
  for (int j = 0; j < COLS; j += 2, p += 4 * (size_t)a.w.N) store_pair<true>(p, v[j] * weight, v[j + 1] * weight, hi, in && j + hi < rows);
}
// A row's factor by a thread: its parts are a few lines of the second level of cache, all on their way at once.
__device__ __forceinline__ float row_factor_of(const W4uArgs& a, int m) {
  const float* p = a.norm.ssq + (size_t)m * a.norm.parts;
  float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
  if (a.norm.parts % 4 == 0) {
#pragma unroll 8
    for (int i = 0; i < a.norm.parts; i += 4) {
      const float4 v = *(const float4*)(p + i);
      s0 += v.x; s1 += v.y; s2 += v.z; s3 += v.w;
    }
  } else {
#pragma unroll 4
    for (int i = 0; i < a.norm.parts; ++i) s0 += p[i];
  }
  return 1.0f / sqrtf(((s0 + s1) + (s2 + s3)) / (float)a.w.K + a.norm.eps);
}
// Columns c_from .. c_to of a tile (rows of x from m0 + c_from on): ready() waits for the accumulator, take(c, v) fetches COLS of its columns.
// What is added to is asked for ahead, the first of it under the MMAs.
// HANDED: `factors` are the rows' (a.norm.ssq), or a norm is handed on behind out += ..
template <int EPI, bool BF16, bool HANDED, int COLS, class Ready, class Take>
__device__ __forceinline__ void finish_columns(const W4uArgs& a, const float* factors, Ready ready, Take take, int c_from, int c_to, int m0, int n) {
  const bool handing = HANDED && EPI == W4_ACC && a.norm.next_x;
  const float weight = handing && n < a.w.N ? a.norm.next_w[n] : 0.f;
  const float bias = a.bias && n < a.w.N ? a.bias[n] : 0.f;
  const int features = EPI == W4_SWIGLU ? a.w.N / 2 : a.w.N;
  const bool pairs = !((features | (int)a.ldo) & 1) && ((uintptr_t)a.out & (BF16 ? 3 : 7)) == 0, ahead = EPI == W4_ACC && pairs;
  c_to = min(c_to, a.M - m0);
  float2 old[EPI == W4_ACC ? COLS / 2 : 1];
  if (ahead && c_from < c_to) load_old<COLS>(a, old, m0 + c_from, a.M - m0 - c_from, n);
  ready();
  for (int c = c_from; c < c_to; c += COLS) {
    float v[COLS];
    take(c, v);
    if (HANDED && a.norm.ssq) {
#pragma unroll
      for (int j = 0; j < COLS; ++j) v[j] *= factors[m0 + c + j];
    }
    if (ahead) {
      add_old<COLS>(v, old);
      if (c + COLS < c_to) load_old<COLS>(a, old, m0 + c + COLS, a.M - m0 - c - COLS, n);
    }
    finish_some<EPI, BF16, COLS>(a, v, m0 + c, a.M - m0 - c, n, bias, pairs);
    if (handing) hand_on<COLS>(a, v, m0 + c, a.M - m0 - c, n, weight);           // (v is what has been stored: pairs, so the old values are in it)
  }
}
// A role's place in the ring of stages, and how often it has been round (its parity).  A role that fills stages waits for the
// parity before its own: of a new barrier that is complete.
struct Ring {
  unsigned stage = 0, parity = 0;
  __device__ __forceinline__ void add(unsigned n, unsigned stages) { stage += n; if (stage >= stages) { stage -= stages; parity ^= 1u; } }        // n <= stages
  __device__ __forceinline__ void add_many(unsigned n, unsigned stages) { stage += n; parity ^= (stage / stages) & 1u; stage %= stages; }
};

// KB: chunks of K a stage.  Two where a tile is narrow (up to 128 columns), whose weights go to tensor memory: one handshake and one commit cost the
// issuing warp as much as three MMAs of 64 columns.
// EPI, BF16: what becomes of the sums, and whether the result is bfloat16 (kernels of their own: with all of them in one, the registers that
// one wants are spilled by the others, 2,048 rows of a gated 16,384 x 2,048 106 -> 114 us).
// HANDED: a norm is handed on to it or by it.  RUNS: K is more than one run (code that runs once is cold: a product of a short K that
// carries it takes 3% longer, 32 rows, gated 9,216 x 1,024, 4.22 -> 4.35 us).
template <bool SPLIT, int PARTS, int KB, int EPI, bool BF16, bool HANDED, bool RUNS>
__global__ void __launch_bounds__(W4U_THREADS, 1) gemm_w4_umma_kernel(const __grid_constant__ CUtensorMap map_x, W4uArgs a) {
  constexpr int AHEAD = 4;               // stages (KB 1) whose chunk a warp holds in registers ahead of the one it unpacks
  constexpr bool TMEM = KB == 2;         // weights in tensor memory
  constexpr unsigned A_BYTES = TMEM ? 0u : W4U_A_BYTES;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  __shared__ __align__(8) unsigned long long bars[2 * 8 + 4];           // full[8], empty[8], acc_full[2], acc_empty[2]
  __shared__ unsigned tmem_base_s;
  __shared__ int dead;                   // a wait gave up
  __shared__ float row_factor[HANDED ? W4U_NORM_ROWS : 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned tiles = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const unsigned x_bytes = (unsigned)a.bn * 128u, stage_bytes = A_BYTES + KB * x_bytes;
  const unsigned full0 = smem_u32(&bars[0]), empty0 = smem_u32(&bars[8]), accfull0 = smem_u32(&bars[16]), accempty0 = smem_u32(&bars[18]);
  const int m_tiles = a.m_tiles, total = a.total;
  const int rank = SPLIT ? (int)cluster_rank() : 0;
  const int first = (int)blockIdx.x >> (SPLIT ? a.log_splits : 0), step = SPLIT ? total : (int)gridDim.x;
  // this CTA's chunks of K
  const int k_stages = (a.w.chunks + KB - 1) / KB;
  const int c_lo = SPLIT ? ((k_stages * rank) >> a.log_splits) * KB : 0, c_hi = SPLIT ? ((k_stages * (rank + 1)) >> a.log_splits) * KB : k_stages * KB;
  const int blocks = (c_hi - c_lo) / KB * PARTS;

  // Barriers and tensor memory are made while the weights' warps ask for their first chunks.  (Tensor memory before the next kernel may start:
  // one that took it first, and waited for this one, would never see its end.  Nor is this one beside another that takes tensor memory: 704
  // threads of 80 registers leave 9,216.)
  auto set_up = [&]() {
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
    pdl_launch_dependents();
    if (SPLIT) asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");        // (waited for where another rank's memory is written)
  };
  if (warp == 0 && lane == 0) {
    dead = 0;
    for (int s = 0; s < a.stages; ++s) { mbar_init(full0 + 8 * s, 1 + 8); mbar_init(empty0 + 8 * s, 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(accfull0 + 8 * b, 1); mbar_init(accempty0 + 8 * b, 4); }
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  __syncwarp();
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&tmem_base_s)), "r"(a.tmem_cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  if (warp < 2 || warp >= 2 + 8 * SETS) set_up();
  const unsigned acc_cols = a.acc_cols, lo_cols = PARTS == 3 ? acc_cols / 2 : 0u;

  if (warp == 0) {
    pdl_wait();                                              // x is the output of the kernel before this one
    Ring ring;
    for (int t = first; t < total; t += step) {
      const int m0 = (t % m_tiles) * a.bn;
      for (int b = 0; b < blocks; ++b) {
        const unsigned full = full0 + 8 * ring.stage;
        W4U_WAIT(empty0 + 8 * ring.stage, ring.parity ^ 1u, 141);
        __syncwarp();
        if (elect_one()) {
          mbar_expect_tx(full, KB * x_bytes);
#pragma unroll
          for (int i = 0; i < KB; ++i)                       // (behind the end of K: zeros)
            tma_load_2d(tiles + ring.stage * stage_bytes + A_BYTES + i * x_bytes, &map_x, (c_lo * PARTS + b * KB + i) * W4_CHUNK, m0, full);
        }
        ring.add(1, a.stages);
      }
    }
  } else if (warp == 1) {
    const unsigned idesc = umma_idesc(128, a.bn), a_lo = umma_desc_lo(tiles), tmem_base = tmem_base_s, w_base = tmem_base + a.w_col;
    unsigned use = 0;
    Ring ring;
    for (int t = first; t < total; t += step) {
      for (int b0 = 0; b0 < blocks; b0 += a.run, ++use) {
        const unsigned acc = a.buffers == 2 ? use & 1 : 0u, round = a.buffers == 2 ? use >> 1 : use, d = tmem_base + acc * acc_cols;
        if (round) W4U_WAIT(accempty0 + 8 * acc, (round - 1) & 1, 145);
        const int run = min(blocks - b0, a.run);
        int part = 0;
        for (int b = 0; b < run; ++b) {
          const unsigned lo = a_lo + ring.stage * (stage_bytes >> 4), empty = empty0 + 8 * ring.stage, to = PARTS == 3 && part < 2 ? d + lo_cols : d;
          W4U_WAIT(full0 + 8 * ring.stage, ring.parity, 142);
          __syncwarp();
          asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
          if (elect_one()) {
#pragma unroll
            for (int i = 0; i < KB; ++i)
              if (TMEM) umma_stage_tmem(to, w_base + ring.stage * (KB * 32) + i * 32, lo + i * (x_bytes >> 4), idesc, (b | i) ? 1u : 0u);
              else umma_stage(to, lo, lo + (A_BYTES >> 4), idesc, b && !(PARTS == 3 && b == 2) ? 1u : 0u);
            umma_commit(empty);
            if (b == run - 1) umma_commit(accfull0 + 8 * acc);
          }
          if (PARTS == 3) part = part == 2 ? 0 : part + 1;
          ring.add(1, a.stages);
        }
      }
    }
  } else if (TMEM && warp < 2 + 8 * SETS) {
    // Weights into tensor memory: a warp has 32 rows (its quarter of the lanes) of every set's stage's one or other chunk.  A lane is a row:
    // its 64 weights lie with those of the row 8 further on in four lanes' 16 bytes of the layout, which come through a ring of the warp's
    // own in shared memory, in an order in which neither the copies nor the reads meet a bank twice.
    const int quarter = warp & 3, set = (warp - 2) >> 3, sub = ((warp - 2) >> 2) & 1, g = lane & 7, slabs = (a.w.N + W4_SLAB - 1) / W4_SLAB;
    const unsigned raw = tiles + a.raw_at + (warp - 2) * W4U_RAW * W4U_RAW_SLOT;
    const unsigned copy_at = (unsigned)((lane >> 2) * 4 + ((lane & 3) ^ ((lane >> 3) & 3))) * 16u;
    const unsigned read_at = (unsigned)(lane >> 4) * 512u + (unsigned)g * 64u, turn = (unsigned)((g >> 1) & 3) * 16u, scale_at = 1024u + (unsigned)(lane >> 4) * 64u + (unsigned)g * 4u;
    const int high = (lane >> 3) & 1;
    const bool two_scales = a.w.gshift == 5;
    Ring base;
    for (int t = first; t < total; t += step) {
      const int slab = (t / m_tiles) * 8 + quarter * 2, mine = slab + (lane >> 4);
      // (a slab that is not there: the first one, times 0)
      const int s_slab = slab + ((lane >> 2) & 1), c_first = c_lo + set * KB + sub;
      const uint4* q0 = a.w.q + ((size_t)(slab < slabs ? slab : 0) * a.w.chunks + c_first) * 32 + lane;
      const long long q1 = ((long long)(slab + 1 < slabs ? slab + 1 : 0) - (slab < slabs ? slab : 0)) * a.w.chunks * 32;
      const unsigned* sc = a.w.s + ((size_t)(s_slab < slabs ? s_slab : 0) * a.w.groups + (two_scales ? (lane >> 1) & 1 : 0)) * 8 + (lane & 1) * 4;
      int left = (blocks - set + SETS - 1) / SETS;            // of this set's blocks, to be fetched
      unsigned k = (unsigned)c_first * W4_CHUNK, write_at = raw, at = raw;
      auto fetch = [&]() {
        if (--left >= 0) {
          copy16(write_at + copy_at, q0);
          copy16(write_at + 512u + copy_at, q0 + q1);
          if (lane < 8) copy16(write_at + 1024u + lane * 16u, sc + (k >> a.w.gshift) * 8u);
          q0 += SETS * KB * 32;
          k += SETS * KB * W4_CHUNK;
        }
        asm volatile("cp.async.commit_group;\n" ::: "memory");
        write_at = write_at == raw + (W4U_RAW - 1) * W4U_RAW_SLOT ? raw : write_at + W4U_RAW_SLOT;
      };
      Ring ring = base;
      ring.add(set, a.stages);
#pragma unroll 1
      for (int u = 0; u < W4U_RAW - 1; ++u) fetch();
      if (t == first) set_up();
      const unsigned to = tmem_base_s + a.w_col + ((unsigned)(quarter * 32) << 16) + sub * 32;
      for (int b = set; b < blocks; b += SETS) {
        asm volatile("cp.async.wait_group %0;\n" ::"n"(W4U_RAW - 2) : "memory");
        __syncwarp();                                        // every lane's copies have come, and every lane has read the unit before
        fetch();                                             // over that one
        const bool in = mine < slabs && c_lo + b * KB + sub < a.w.chunks;
        const unsigned sa = in ? ld_shared(at + scale_at) : 0u, sb = two_scales ? (in ? ld_shared(at + scale_at + 32u) : 0u) : sa;
        unsigned v[32];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint4 x = ld_shared_v4(at + read_at + (((unsigned)c * 16u) ^ turn));
          const unsigned w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const unsigned s2 = __byte_perm(h ? sb : sa, 0, high ? 0x3232 : 0x1010), off = times_minus_24(s2);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              v[16 * h + 4 * c + 2 * j] = w4_value(w[2 * h + j], high, s2, off);
              v[16 * h + 4 * c + 2 * j + 1] = w4_value(w[2 * h + j], high + 2, s2, off);
            }
          }
        }
        at = at == raw + (W4U_RAW - 1) * W4U_RAW_SLOT ? raw : at + W4U_RAW_SLOT;
        W4U_WAIT(empty0 + 8 * ring.stage, ring.parity ^ 1u, 143);
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
        __syncwarp();
        tmem_st32(to + ring.stage * (KB * 32), v);
        tmem_st_wait();
        asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(full0 + 8 * ring.stage);
        ring.add(SETS, a.stages);
      }
      __syncwarp();
      base.add_many(blocks, a.stages);
    }
  } else if (!TMEM && warp < 2 + 8 * SETS) {
    // weights: nothing in front of this kernel writes them, so they need not wait for it
    const int sl = (warp - 2) & 7, set = (warp - 2) >> 3, g = lane >> 2, c = lane & 3, slabs = (a.w.N + W4_SLAB - 1) / W4_SLAB;
    Ring base;
    // where the lane's pieces lie in the tile: row 16 sl + g (and + 8: the same swizzle), pieces c and 4 + c of its eight.  Odd rows
    // are written the far piece first, so that eight lanes of a store meet every bank once.
    const bool flip = g & 1, two_scales = a.w.gshift == 5;
    const unsigned row = tiles + (unsigned)(16 * sl + g) * 128u, near = (unsigned)(c ^ g) * 16u, far = (unsigned)((c + 4) ^ g) * 16u;
    const unsigned p0 = row + (flip ? far : near), p1 = row + (flip ? near : far);
    for (int t = first; t < total; t += step) {
      const int slab = (t / m_tiles) * 8 + sl;
      const bool have = slab < slabs;
      const uint4* q = a.w.q + ((size_t)(have ? slab : 0) * a.w.chunks + c_lo) * 32 + lane;
      const unsigned* sc = a.w.s + (size_t)(have ? slab : 0) * a.w.groups * 8 + g;
      uint4 qv[AHEAD];
      unsigned sv[AHEAD][2];
      // This set's blocks of the tile: set, set + SETS, ...; `ahead`: the next one to be fetched.  Behind the last one loads go on
      // (into the next slab or the room behind the matrix): a load that may not happen would have to be waited for at once.
      unsigned ahead = set;
      auto fetch = [&](int u) {
        const unsigned ch = PARTS == 1 ? ahead : ahead / 3;
        qv[u] = __ldg(q + ch * 32u);
        const unsigned* at = sc + ((((unsigned)c_lo + ch) * W4_CHUNK) >> a.w.gshift) * 8u;
        sv[u][0] = __ldg(at);
        sv[u][1] = __ldg(at + (two_scales ? 8 : 0));
        ahead += SETS;
      };
      Ring ring = base;
      ring.add(set, a.stages);
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) fetch(u);
      if (t == first) set_up();
      for (int b0 = set; b0 < blocks; b0 += SETS * AHEAD) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
          if (b0 + u * SETS >= blocks) break;
          const unsigned at = ring.stage * stage_bytes;
          const uint4 x = qv[u];
          const unsigned sa = have ? sv[u][0] : 0u, sb = have ? sv[u][1] : 0u, s_first = flip ? sb : sa, s_second = flip ? sa : sb;
          const unsigned w[4] = {flip ? x.z : x.x, flip ? x.w : x.y, flip ? x.x : x.z, flip ? x.y : x.w};
          unsigned v[2][2][4];                              // [row g, g + 8][piece][..]
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const unsigned s2 = __byte_perm(h ? s_second : s_first, 0, r ? 0x3232 : 0x1010), off = times_minus_24(s2);
              v[r][h][0] = w4_value(w[2 * h], r, s2, off); v[r][h][1] = w4_value(w[2 * h], r + 2, s2, off);
              v[r][h][2] = w4_value(w[2 * h + 1], r, s2, off); v[r][h][3] = w4_value(w[2 * h + 1], r + 2, s2, off);
            }
          fetch(u);
          W4U_WAIT(empty0 + 8 * ring.stage, ring.parity ^ 1u, 143);
#pragma unroll
          for (int r = 0; r < 2; ++r) {                     // (row g + 8: eight rows of 128 bytes further on)
            st_shared_v4(at + p0 + r * 1024u, v[r][0][0], v[r][0][1], v[r][0][2], v[r][0][3]);
            st_shared_v4(at + p1 + r * 1024u, v[r][1][0], v[r][1][1], v[r][1][2], v[r][1][3]);
          }
          asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
          __syncwarp();
          if (lane == 0) mbar_arrive(full0 + 8 * ring.stage);
          ring.add(SETS, a.stages);
        }
      }
      base.add_many(blocks, a.stages);
    }
  }
  __syncwarp();
  // The epilogue: the last four warps, a tile behind the MMAs; the CTA's last tile (a cluster's only one) by the sixteen warps that have made
  // all weights too, a fifth of the columns each four.
  const bool epi_warp = warp >= 2 + 8 * SETS;
  const int quarter = warp & 3, row = quarter * 32 + lane, fifth = epi_warp ? 4 : (warp - 2) >> 2;
  const unsigned tmem_base = tmem_base_s, quarter_base = tmem_base + ((unsigned)(quarter * 32) << 16);
  const int last = SPLIT ? 0 : (total - 1 - first) / step;  // this CTA's last tile
  const int runs = !RUNS || blocks <= a.run ? 1 : (blocks + a.run - 1) / a.run;             // accumulators a tile goes through
  if (HANDED && a.norm.ssq && epi_warp) {                    // (while the others are at work; they see it behind a barrier below)
    pdl_wait();
    const int m = threadIdx.x - 32 * (2 + 8 * SETS);
    row_factor[m] = m < a.M ? row_factor_of(a, m) : 0.f;
  }
  auto where = [&](int use) { return quarter_base + (a.buffers == 2 ? (unsigned)(use & 1) * acc_cols : 0u); };
  auto release = [&](int use) {
    if (lane == 0) mbar_arrive(accempty0 + (a.buffers == 2 ? 8 * (use & 1) : 0));
  };
  // A tile's sums: the epilogue's warps wait for each of its runs and add the one before to it, whose accumulator is free then; of the CTA's last
  // tile the last two stay apart, and whoever finishes a column adds them.  The other
  // warps go on when those have seen the last run (they are not there for every phase of its barrier).
  auto before = [&](int tile) { return !RUNS || runs == 1 || tile < last ? 0u : where(tile * runs + runs - 2) - where(tile * runs + runs - 1); };
  auto tile_ready = [&](int tile, bool everyone) {
    if (epi_warp) {
      for (int r = 0; r < runs; ++r) {
        const int use = tile * runs + r;
        W4U_WAIT_EPILOGUE(accfull0 + (a.buffers == 2 ? 8 * (use & 1) : 0), (a.buffers == 2 ? use >> 1 : use) & 1);
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
        __syncwarp();
        if (RUNS && r > 0 && !(everyone && r == runs - 1)) {
          for (int c = 0; c < a.bn; c += 16) {
            tmem_add16(where(use) + c, where(use - 1) + c);
            if (PARTS == 3) tmem_add16(where(use) + lo_cols + c, where(use - 1) + lo_cols + c);
          }
          tmem_st_wait();
          asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
          __syncwarp();
          release(use - 1);
        }
      }
      if (everyone) {
        asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
        asm volatile("bar.arrive 2, %0;\n" ::"n"(32 * (8 * SETS + 4)) : "memory");
      }
    } else asm volatile("bar.sync 2, %0;\n" ::"n"(32 * (8 * SETS + 4)) : "memory");
    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
    __syncwarp();
  };
  if (!SPLIT && warp >= 2) {
    pdl_wait();
    for (int tile = epi_warp ? 0 : last; tile <= last; ++tile) {
      const int t = first + tile * step, use = tile * runs + runs - 1, groups = a.bn / 16;
      const int m0 = (t % m_tiles) * a.bn, n = (t / m_tiles) * 128 + row;
      const unsigned from = where(use), also = before(tile);
      finish_columns<EPI, BF16, HANDED, 16>(a, row_factor, [&]() { tile_ready(tile, tile == last); }, [&](int c, float* v) { tmem_sums<16>(from + c, lo_cols, also, v); },
                                            tile < last ? 0 : groups * fifth / 5 * 16, tile < last ? a.bn : groups * (fifth + 1) / 5 * 16, m0, n);
      if (tile < last) {
        asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
        __syncwarp();
        release(use);
      }
    }
  }
  if (SPLIT) {
    // Every rank sends the other ranks' columns of its sums to them: [sending rank, without the owner][its groups of four columns][128 rows][4], so that a
    // warp's store is 512 bytes in a row (16 bytes here and there took ten times as long: they travel one by one).
    const int t = first, m0 = (t % m_tiles) * a.bn, n = (t / m_tiles) * 128 + row;
    const int share = a.share, groups = share / 4, c0 = rank * share;
    const unsigned from = where(runs - 1), also = before(0);
    const unsigned recv = a.recv_apart ? tiles + (unsigned)a.stages * stage_bytes : tiles;
    asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");         // every rank has started: its memory is there
    if (warp < 2) {
      __syncwarp();
      if (!a.recv_apart) cluster_sync();
      cluster_sync();
    } else {
      const float4* mine = reinterpret_cast<const float4*>(smem_raw + (recv - smem_u32(smem_raw))) + row;
      pdl_wait();
      finish_columns<EPI, BF16, HANDED, 4>(a, row_factor, [&]() {
        tile_ready(0, true);
        if (!a.recv_apart) cluster_sync();                                        // every rank's MMAs have read their stages
        for (int c = fifth * 16; c < a.bn && m0 + c < a.M; c += 5 * 16) {
          float v[16];
          tmem_sums<16>(from + c, lo_cols, also, v);
          int owner = (c >> 2) / groups, group = (c >> 2) - owner * groups;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (owner != rank && m0 + c + 4 * j < a.M)
              st_cluster_v4(mapa(recv + (unsigned)((((rank < owner ? rank : rank - 1) * groups + group) * 128 + row) * 16), (unsigned)owner), v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
            if (++group == groups) { group = 0; ++owner; }
          }
        }
        __syncwarp();
        cluster_sync();
      }, [&](int c, float* v) {
        float own[4];
        tmem_sums<4>(from + c, lo_cols, also, own);
        const float4* part = mine + (c - c0) / 4 * 128;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int r = 0; r < a.splits; ++r) {                 // (in the ranks' order)
          const float4 x = r == rank ? make_float4(own[0], own[1], own[2], own[3]) : *part;
          if (r != rank) part += groups * 128;
          sum.x += x.x; sum.y += x.y; sum.z += x.z; sum.w += x.w;
        }
        v[0] = sum.x; v[1] = sum.y; v[2] = sum.z; v[3] = sum.w;
      }, c0 + groups * fifth / 5 * 4, min(a.bn, c0 + groups * (fifth + 1) / 5 * 4), m0, n);
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
  __syncthreads();
  if (dead) for (int i = 0; i < 64; ++i) __nanosleep(100000);        // (some milliseconds: what is on its way into this memory has come)
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem_base), "r"(a.tmem_cols) : "memory");
  }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                  CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  if (!fn) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess) fn = (EncodeTiledFn)p;
  }
  return fn;
}

// Clusters of `splits` CTAs, each an SM's all, that the device holds at once: the CTAs of one sit in one GPC, so this is less than SMs /
// splits (a product whose clusters of 8 do not fit takes twice as long).  Asked once a device and size.
static int clusters_at_once(int splits) {
  static int cache[64][9];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 0;
  if (!cache[dev][splits]) {
    const size_t smem = 221 * 1024;
    auto kern = gemm_w4_umma_kernel<true, 1, 1, W4_STORE, true, false, false>;
    int n = 0;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) == cudaSuccess) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(splits * 64, 1, 1); cfg.blockDim = dim3(W4U_THREADS, 1, 1); cfg.dynamicSmemBytes = smem;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = splits; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr; cfg.numAttrs = 1;
      if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) { n = 0; cudaGetLastError(); }
    }
    cache[dev][splits] = n > 0 ? n : 1;
  }
  return cache[dev][splits];
}

template <int EPI, bool BF16, int PARTS, int KB, bool HANDED, bool RUNS>
static int launch_tiles_of(const CUtensorMap& map, const W4uArgs& a, int grid, size_t smem, cudaStream_t stream) {
  auto kern = a.splits > 1 ? gemm_w4_umma_kernel<true, PARTS, KB, EPI, BF16, HANDED, RUNS> : gemm_w4_umma_kernel<false, PARTS, KB, EPI, BF16, HANDED, RUNS>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return (int)e;
  return launch_k_class(1, kern, dim3(grid, 1, 1), dim3(W4U_THREADS, 1, 1), smem, stream, a.splits, map, a);
}
template <int EPI, bool BF16, bool RUNS>
static int launch_tiles(const CUtensorMap& map, const W4uArgs& a, int parts, int kb, int grid, size_t smem, cudaStream_t stream) {
  if (parts == 3) return BF16 ? FELLM_ERR_ARG : launch_tiles_of<EPI, false, 3, 1, false, RUNS>(map, a, grid, smem, stream);      // (float32 rows make float32 results)
  if (a.norm.next_x || a.norm.ssq) return launch_tiles_of<EPI, BF16, 1, 2, true, RUNS>(map, a, grid, smem, stream);      // (up to 128 rows)
  return kb == 2 ? launch_tiles_of<EPI, BF16, 1, 2, false, RUNS>(map, a, grid, smem, stream) : launch_tiles_of<EPI, BF16, 1, 1, false, RUNS>(map, a, grid, smem, stream);
}
template <int EPI, bool BF16>
static int launch_runs(int runs, const CUtensorMap& map, const W4uArgs& a, int parts, int kb, int grid, size_t smem, cudaStream_t stream) {
  return runs > 1 ? launch_tiles<EPI, BF16, true>(map, a, parts, kb, grid, smem, stream) : launch_tiles<EPI, BF16, false>(map, a, parts, kb, grid, smem, stream);
}

// x that TMA cannot read as it is (float32, or rows that are not on 16 bytes) is copied into `scratch` first: M x chunks x 64 numbers of
// bfloat16, three times as many for float32; scratch null: x is read itself.
FELLM_API int fellm_gemm_w4_umma(const void* x, long long ldx, const W4Ref* w, const float* bias, void* out, long long ldo, int flags, int M, void* scratch,
                                 const W4Norm* norm, int* status, cudaStream_t stream) {
  if (M <= 0) return 0;
  if (!x || !out || !status) return FELLM_ERR_ARG;
  if (int e = w4_check(w)) return e;
  if (int e = w4_check_epi(flags, w->N)) return e;
  const int x_bf16 = (flags & W4_X_BF16) != 0, N = w->N, K = w->K, chunks = w->chunks;
  const bool copied = scratch != nullptr;
  if (!copied && (!x_bf16 || K % 8 || (M > 1 && (ldx % 8 || ldx < K)) || ((uintptr_t)x & 15))) return FELLM_ERR_ARG;
  const int parts = x_bf16 ? 1 : 3;
  if (norm) {
    if (copied || M > W4U_NORM_ROWS || (norm->next_x && norm->ssq)) return FELLM_ERR_SIZE;
    if (norm->next_x && (!norm->next_w || !norm->next_ssq || (flags & W4_EPI) != W4_ACC || N % 32 || ldo < N || ldo % 2 || ((uintptr_t)out & 7))) return FELLM_ERR_ARG;
    if (norm->ssq && (norm->parts < 1 || norm->parts > 128 || ((uintptr_t)norm->ssq & 15))) return FELLM_ERR_ARG;
  }
  if (copied) {
    if (int e = w4_copy_rows(x, x_bf16, ldx, scratch, M, K, chunks, stream)) return e;
    x = scratch; ldx = (long long)parts * chunks * W4_CHUNK;
  }
  W4uArgs a = {*w, bias, out, status, ldo, M};
  a.norm = norm ? *norm : W4Norm{};
  const int n_sm = fellm_sm_count(), n_tiles = ceil_div(N, 128);
  const bool to_bf16 = (flags & W4_OUT_BF16) != 0;
  const int most = parts == 3 && chunks > W4U_RUN ? 128 : 256;          // (columns of a tile: tensor memory holds what its sums need)
  // Columns of a tile and CTAs that share its K, by the time of the busiest SM.  A chunk counts 0.21 us up to 64 columns and 0.29 at 128
  // (weights in tensor memory take 0.15 to 0.17 in a long K, but few have one: with that, steps of 64 and 128 requests got 8 to 12% slower),
  // 0.37 at 256, where the MMAs bound it; a cluster's exchange 0.9 us and what its sums take at some 22 GB/s an SM.
  // A product that takes nearly all SMs costs its neighbours a microsecond: nothing of the next one starts under it (32 rows, gated
  // 9,216 x 1,024, one after another: 6.6 us in clusters of two on 144 SMs, 5.0 on 72 by themselves).
  double least = 1e30;
  int total = 1;
  a.bn = 16; a.splits = 1; a.log_splits = 0;
  for (int m_tiles = ceil_div(M, most), i = 0; i < 8 && m_tiles <= ceil_div(M, 16); ++m_tiles, ++i) {
    const int bn = ceil_div(ceil_div(M, m_tiles), 16) * 16, tiles = n_tiles * ceil_div(M, bn);
    if (i > 0 && bn < 112) break;                       // (every tile makes its weights again)
    const double chunk_us = bn <= 64 ? 0.21 : bn <= 128 ? 0.13 + 0.00122 * bn : 0.2 + 0.00066 * bn;
    for (int ls = 0; ls <= 3; ++ls) {
      const int s = 1 << ls;
      if (s > 1 && (chunks < 4 * s || tiles > clusters_at_once(s))) break;
      const double t = ceil_div(tiles * s, n_sm) * (double)ceil_div(chunks, s) * parts * chunk_us + (4 * tiles * s > 3 * n_sm ? 1.0 : 0.0) + (s > 1 ? 0.9 + bn * 0.0234 * (s - 1) / s : 0.0);
      if (t < least) { least = t; a.bn = bn; a.splits = s; a.log_splits = ls; total = tiles; }
    }
  }
  a.m_tiles = ceil_div(M, a.bn); a.total = total;
  const int kb = parts == 1 && a.bn <= 128 ? 2 : 1, stage = kb * a.bn * 128 + (kb == 2 ? 0 : W4U_A_BYTES), raw = kb == 2 ? 8 * SETS * W4U_RAW * W4U_RAW_SLOT : 0;
  a.share = ceil_div(a.bn / 4, a.splits) * 4;
  const int room = 220 * 1024 - raw, recv = (a.splits - 1) * a.share * 512;
  const int blocks = ceil_div(ceil_div(chunks, kb), a.splits) * parts;
  const int runs = ceil_div(blocks, W4U_RUN / kb * parts);
  a.run = ceil_div(blocks / parts, runs) * parts;
  a.acc_cols = 16;
  while (a.acc_cols < a.bn) a.acc_cols *= 2;
  if (parts == 3) a.acc_cols *= 2;
  a.buffers = (a.splits == 1 || runs > 1) && 2 * a.acc_cols <= 512 ? 2 : 1;
  if (runs > 1 && a.buffers < 2) return FELLM_ERR_SIZE;
  a.tmem_cols = kb == 2 ? 512 : a.buffers * a.acc_cols < 32 ? 32 : a.buffers * a.acc_cols;
  a.stages = room / stage < 8 ? room / stage : 8;
  a.w_col = ceil_div(a.buffers * a.acc_cols, 64) * 64;
  if (kb == 2 && (512 - a.w_col) / 64 < a.stages) a.stages = (512 - a.w_col) / 64;
  a.recv_apart = (room - recv) / stage >= 3;
  if (a.recv_apart && (room - recv) / stage < a.stages) a.stages = (room - recv) / stage;
  if (!a.recv_apart && recv > a.stages * stage) return FELLM_ERR_SIZE;
  a.raw_at = a.stages * stage + (a.recv_apart ? recv : 0);
  EncodeTiledFn fn = encode_fn();
  if (!fn) return FELLM_ERR_ARG;
  CUtensorMap map;
  cuuint64_t dims[2] = {copied ? (cuuint64_t)parts * chunks * W4_CHUNK : (cuuint64_t)K, (cuuint64_t)M};
  cuuint64_t strides[1] = {(cuuint64_t)(M == 1 && !copied ? (long long)ceil_div(K, 8) * 8 : ldx) * 2};
  cuuint32_t box[2] = {W4_CHUNK, (cuuint32_t)a.bn}, estr[2] = {1, 1};
  const CUresult r = fn(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(x), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return 1000 + (int)r;
  const size_t smem = (size_t)a.raw_at + raw + 1024;
  const int grid = a.splits > 1 ? total * a.splits : (total < n_sm ? total : n_sm);
  switch (flags & W4_EPI) {
    case W4_ACC: return to_bf16 ? FELLM_ERR_ARG : launch_runs<W4_ACC, false>(runs, map, a, parts, kb, grid, smem, stream);
    case W4_SWIGLU: return to_bf16 ? launch_runs<W4_SWIGLU, true>(runs, map, a, parts, kb, grid, smem, stream) : launch_runs<W4_SWIGLU, false>(runs, map, a, parts, kb, grid, smem, stream);
    case W4_RELU2: return to_bf16 ? launch_runs<W4_RELU2, true>(runs, map, a, parts, kb, grid, smem, stream) : launch_runs<W4_RELU2, false>(runs, map, a, parts, kb, grid, smem, stream);
    default: return to_bf16 ? launch_runs<W4_STORE, true>(runs, map, a, parts, kb, grid, smem, stream) : launch_runs<W4_STORE, false>(runs, map, a, parts, kb, grid, smem, stream);
  }
}
