// Matrices in four bits (w4.h): into the form, out of it, and rows of it as token embeddings.
#include "w4.h"

#define W4_THREADS 256

// Rounds a positive finite float to five significant bits, to nearest, ties to even.
__device__ __forceinline__ float round5(float a) {
  unsigned u = __float_as_uint(a);
  u += 0x3ffffu + ((u >> 19) & 1u);
  return __uint_as_float(u & 0xfff80000u);
}

// A group's scale from its largest and smallest element: an eighth of the largest magnitude, in five significant bits (taken before the
// division, which is exact: behind it a number below the normal ones would have fewer), negative where that magnitude is a positive element's
// (so that the extreme is level -8, not the missing +8).  Below the
// normal numbers: 0, the group is zeros.  Not above 31 * 2^118: 24 s has to stay
// finite, with which the weights are made bfloat16 numbers.  NaN where an element is not finite.
__device__ __forceinline__ float group_scale(float hi, float lo, bool finite) {
  if (!finite) return __uint_as_float(0x7fc00000u);
  float s = fminf(round5(fmaxf(hi, -lo)) * 0.125f, __uint_as_float(0x7cf80000u));
  if (s < 1.1754943508222875e-38f) s = 0.f;
  return hi > -lo ? -s : s;
}
// The level of w under scale s (inv: 1 / s rounded, 0 for scale 0), 0..15 = level + 8: w / s to the nearest whole number, ties to even,
// EXACTLY.  x = w inv, corrected once by its remainder, is the quotient rounded to float32 (Markstein: a correctly rounded reciprocal
// and one fused correction give the correctly rounded quotient).  A bfloat16 w over five bits cannot lie so near a half that this
// rounding reaches it (both are fractions of small numbers: 2^-10 away at least, or on it).  A float32 w can: there the remainder
// w - q s, exact in one fused operation (q s has at most nine bits, what is left of w is below s), says on which side it lies.
template <bool NARROW>
__device__ __forceinline__ unsigned level_of(float w, float s, float inv) {
  float x = w * inv;
  x = fmaf(fmaf(-x, s, w), inv, x);
  x = fminf(fmaxf(x, -8.f), 7.f);
  const float up = x + 12582920.f;                          // 1.5 * 2^23 + 8: the sum's last place is a whole number's
  unsigned level = __float_as_uint(up) & 15u;
  if (!NARROW) {
    const float left = fmaf(-(up - 12582920.f), s, w), half = 0.5f * fabsf(s);
    if (fabsf(left) > half) {
      if ((left > 0.f) == (s > 0.f)) { if (level < 15u) ++level; }
      else if (level > 0u) --level;
    }
  }
  return level;
}

// What lane (g, c) keeps of two chunks: rows g, g + 8 x quarters of 32 elements x its eight.
__device__ __forceinline__ void load8(const float* row, bool row_ok, int k, int K, bool vec, float* v) {
  if (!row_ok) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.f;
    return;
  }
  if (vec && k + 8 <= K) {
    const float4 x = *(const float4*)(row + k), y = *(const float4*)(row + k + 4);
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w; v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = k + i < K ? row[k + i] : 0.f;
}
// Two rows' eight levels (0..15 each) of a half chunk -> the two words of w4.h.
__device__ __forceinline__ unsigned pack_word(const unsigned* a, const unsigned* b) {
  const unsigned w = a[0] | b[0] << 4 | a[2] << 8 | b[2] << 12 | a[1] << 16 | b[1] << 20 | a[3] << 24 | b[3] << 28;
  return __funnelshift_l(w, w, 3);
}

struct W4Out { uint4* q; unsigned* s; int N, K, chunks, groups, gshift; };

// A warp's slab x 128 elements in levels: lane (g, c) has rows g, g + 8, four quarters of 32 elements, eight of each.
// element(r, h, i) gives them as float32, s and inv the scale and its reciprocal of every row and quarter.
template <bool NARROW, class Element>
__device__ __forceinline__ void put_levels(const W4Out& o, int slab, int pair, int lane, Element element, const float (*s)[4], const float (*inv)[4]) {
#pragma unroll
  for (int ch = 0; ch < 2; ++ch) {
    if (2 * pair + ch >= o.chunks) break;
    unsigned word[4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int q = 2 * ch + h;
      unsigned a[8], b[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) { a[i] = level_of<NARROW>(element(0, q, i), s[0][q], inv[0][q]); b[i] = level_of<NARROW>(element(1, q, i), s[1][q], inv[1][q]); }
      word[2 * h] = pack_word(a, b); word[2 * h + 1] = pack_word(a + 4, b + 4);
    }
    o.q[((size_t)slab * o.chunks + 2 * pair + ch) * 32 + lane] = make_uint4(word[0], word[1], word[2], word[3]);
  }
  // quarter c's scales by lane c (a group's first quarter only)
  const int g = lane >> 2, c = lane & 3;
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    if (c != h || ((h << 5) & ((1 << o.gshift) - 1))) continue;
    const int grp = (pair * 128 + h * 32) >> o.gshift;
    if (grp < o.groups) o.s[((size_t)slab * o.groups + grp) * 8 + g] = __float_as_uint(s[0][h]) >> 16 | (__float_as_uint(s[1][h]) & 0xffff0000u);
  }
}

// A warp a slab x 128 elements.  Every element is read once, by loads of 16 bytes of which four neighbouring lanes take 64 consecutive bytes of a row
// (128 of a float32 one).  Bound by instructions (issue slots 74% of a bfloat16 launch, 60% of a float32 one, whose 121 registers a thread leave sixteen warps
// an SM): 65,536 x 2,048 takes 82 us from bfloat16, 52 at memory's rate, and 173 from float32, 93 at memory's rate.
__global__ void __launch_bounds__(W4_THREADS) quantize_w4_f32_kernel(const float* w, long long ldw, int vec, W4Out o) {
  const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int pairs = (o.chunks + 1) / 2;
  const long long unit = (long long)blockIdx.x * (W4_THREADS / 32) + (threadIdx.x >> 5);
  const int slab = (int)(unit / pairs), pair = (int)(unit % pairs);
  if (slab * W4_SLAB >= o.N) return;
  float v[2][4][8];
  float hi[2][4], lo[2][4];
  bool fin[2][4];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int n = slab * W4_SLAB + g + 8 * r;
    const float* row = w + (size_t)n * ldw;
#pragma unroll
    for (int h = 0; h < 4; ++h) load8(row, n < o.N, pair * 128 + h * 32 + c * 8, o.K, vec != 0, v[r][h]);
  }
#pragma unroll
  for (int r = 0; r < 2; ++r)
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      float a = v[r][h][0], b = a, zero = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) { a = fmaxf(a, v[r][h][i]); b = fminf(b, v[r][h][i]); zero = fmaf(v[r][h][i], 0.f, zero); }
      bool ok = zero == 0.f;                                // (0 times an infinity or NaN is none)
#pragma unroll
      for (int x = 1; x < 4; x <<= 1) {
        a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, x));
        b = fminf(b, __shfl_xor_sync(0xffffffffu, b, x));
        ok = __shfl_xor_sync(0xffffffffu, (int)ok, x) && ok;
      }
      hi[r][h] = a; lo[r][h] = b; fin[r][h] = ok;
    }
  // groups of 64 and 128: the quarters' extremes put together
#pragma unroll
  for (int r = 0; r < 2; ++r)
#pragma unroll
    for (int step = 1; step <= 2; step <<= 1) {
      if ((32 * step) >> o.gshift) continue;               // (this distance is between groups already)
#pragma unroll
      for (int h = 0; h < 4; ++h) if (!(h & step)) {
        const float a = fmaxf(hi[r][h], hi[r][h | step]), b = fminf(lo[r][h], lo[r][h | step]);
        const bool ok = fin[r][h] && fin[r][h | step];
        hi[r][h] = hi[r][h | step] = a; lo[r][h] = lo[r][h | step] = b; fin[r][h] = fin[r][h | step] = ok;
      }
    }
  float s[2][4], inv[2][4];
#pragma unroll
  for (int r = 0; r < 2; ++r)
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      s[r][h] = group_scale(hi[r][h], lo[r][h], fin[r][h]);
      inv[r][h] = s[r][h] != 0.f ? 1.f / s[r][h] : 0.f;
    }
  put_levels<false>(o, slab, pair, lane, [&](int r, int h, int i) { return v[r][h][i]; }, s, inv);
}

// bfloat16: the elements stay as they came (two in a register), their extremes are taken two at a time.  A group's largest element and the
// negative of its smallest travel as one pair; an element that is none makes them none, an infinity is one of them.
__device__ __forceinline__ unsigned max2_nan(unsigned a, unsigned b) {
  __nv_bfloat162 v = __hmax2_nan(*(const __nv_bfloat162*)&a, *(const __nv_bfloat162*)&b);
  return *(unsigned*)&v;
}
__global__ void __launch_bounds__(W4_THREADS) quantize_w4_bf16_kernel(const bf16* w, long long ldw, int vec, W4Out o) {
  const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int pairs = (o.chunks + 1) / 2;
  const long long unit = (long long)blockIdx.x * (W4_THREADS / 32) + (threadIdx.x >> 5);
  const int slab = (int)(unit / pairs), pair = (int)(unit % pairs);
  if (slab * W4_SLAB >= o.N) return;
  uint4 raw[2][4];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int n = slab * W4_SLAB + g + 8 * r;
    const unsigned short* row = (const unsigned short*)w + (size_t)n * ldw;
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const int k = pair * 128 + h * 32 + c * 8;
      if (n < o.N && vec && k + 8 <= o.K) raw[r][h] = *(const uint4*)(row + k);
      else {
        unsigned x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const unsigned lo = n < o.N && k + 2 * i < o.K ? row[k + 2 * i] : 0, hi = n < o.N && k + 2 * i + 1 < o.K ? row[k + 2 * i + 1] : 0;
          x[i] = lo | hi << 16;
        }
        raw[r][h] = make_uint4(x[0], x[1], x[2], x[3]);
      }
    }
  }
  unsigned m[2][4];                                          // (largest, minus the smallest)
#pragma unroll
  for (int r = 0; r < 2; ++r)
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const unsigned x[4] = {raw[r][h].x, raw[r][h].y, raw[r][h].z, raw[r][h].w}, sign = 0x80008000u;
      const unsigned up = max2_nan(max2_nan(x[0], x[1]), max2_nan(x[2], x[3]));
      const unsigned down = max2_nan(max2_nan(x[0] ^ sign, x[1] ^ sign), max2_nan(x[2] ^ sign, x[3] ^ sign));
      m[r][h] = max2_nan(__byte_perm(up, down, 0x5410), __byte_perm(up, down, 0x7632));
    }
  float s[2][4], inv[2][4];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    if (o.gshift >= 6) { m[r][0] = m[r][1] = max2_nan(m[r][0], m[r][1]); m[r][2] = m[r][3] = max2_nan(m[r][2], m[r][3]); }
    if (o.gshift == 7) m[r][0] = m[r][1] = m[r][2] = m[r][3] = max2_nan(m[r][0], m[r][2]);
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      if ((h << 5) & ((1 << o.gshift) - 1)) { s[r][h] = s[r][h - 1]; inv[r][h] = inv[r][h - 1]; continue; }
      unsigned x = m[r][h];
      x = max2_nan(x, __shfl_xor_sync(0xffffffffu, x, 1));
      x = max2_nan(x, __shfl_xor_sync(0xffffffffu, x, 2));
      const float hi = __uint_as_float(x << 16), lo = -__uint_as_float(x & 0xffff0000u);
      s[r][h] = group_scale(hi, lo, fabsf(hi) <= 3.4028234663852886e38f && fabsf(lo) <= 3.4028234663852886e38f);
      inv[r][h] = s[r][h] != 0.f ? 1.f / s[r][h] : 0.f;
    }
  }
  put_levels<true>(o, slab, pair, lane, [&](int r, int h, int i) {
    const unsigned x[4] = {raw[r][h].x, raw[r][h].y, raw[r][h].z, raw[r][h].w};
    return i & 1 ? __uint_as_float(x[i >> 1] & 0xffff0000u) : __uint_as_float(x[i >> 1] << 16);
  }, s, inv);
}

// Levels and scales that exist already -> the layout.  bad: 1 a level outside -8..7, 2 a scale that is not finite, has more
// than five significant bits or is above 31 * 2^118 or not a normal number.
__global__ void __launch_bounds__(W4_THREADS) pack_w4_kernel(const signed char* lv, long long ldl, const bf16* sc, long long lds, W4Out o, int groups_in, int* bad) {
  const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const long long unit = (long long)blockIdx.x * (W4_THREADS / 32) + (threadIdx.x >> 5);
  const int slab = (int)(unit / o.chunks), chunk = (int)(unit % o.chunks);
  if (slab * W4_SLAB >= o.N) return;
  unsigned word[4];
  bool wrong = false;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    unsigned u[2][8];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int n = slab * W4_SLAB + g + 8 * r, k = chunk * W4_CHUNK + h * 32 + c * 8;
      const signed char* p = lv + (size_t)n * ldl + k;
      signed char b[8];
      const bool row_ok = n < o.N;
      if (row_ok && k + 8 <= o.K && ((uintptr_t)p & 7) == 0) *(uint2*)b = *(const uint2*)p;
      else {
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] = row_ok && k + i < o.K ? p[i] : (signed char)0;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) { wrong = wrong || b[i] < -8 || b[i] > 7; u[r][i] = (unsigned)(b[i] + 8) & 15u; }
    }
    word[2 * h] = pack_word(u[0], u[1]); word[2 * h + 1] = pack_word(u[0] + 4, u[1] + 4);
  }
  if (wrong) atomicOr(bad, 1);
  o.q[((size_t)slab * o.chunks + chunk) * 32 + lane] = make_uint4(word[0], word[1], word[2], word[3]);
  // the groups that start in this chunk: lane c the c-th (a chunk starts two of 32, one of 64, every other one of 128)
  const int first = (chunk * W4_CHUNK + (1 << o.gshift) - 1) >> o.gshift, end = ((chunk + 1) * W4_CHUNK + (1 << o.gshift) - 1) >> o.gshift;
  const int grp = first + c;
  if (grp < end && grp < o.groups) {
    unsigned half[2];
    bool odd = false;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int n = slab * W4_SLAB + g + 8 * r;
      half[r] = n < o.N && grp < groups_in ? (unsigned)*(const unsigned short*)(sc + (size_t)n * lds + grp) : 0u;
      const unsigned mag = half[r] & 0x7fffu;
      odd = odd || (half[r] & 7u) || mag > 0x7cf8u || (mag && mag < 0x80u);
    }
    if (odd) atomicOr(bad, 2);
    o.s[((size_t)slab * o.groups + grp) * 8 + g] = half[0] | half[1] << 16;
  }
}

// The eight elements of row `row` from k on (k a multiple of 8, in the padded width).
__device__ __forceinline__ void row8(const W4Ref& m, int row, int k, float* v) {
  const int slab = row / W4_SLAB, r = row % W4_SLAB, g = r & 7, chunk = k / W4_CHUNK, h = (k / 32) & 1, c = (k / 8) & 3;
  const uint2 w = *((const uint2*)(m.q + ((size_t)slab * m.chunks + chunk) * 32 + 4 * g + c) + h);
  const unsigned sw = m.s[((size_t)slab * m.groups + (k >> m.gshift)) * 8 + g];
  const float s = r < 8 ? w4_scale_lo(sw) : w4_scale_hi(sw);
  const int sh = r < 8 ? 0 : 4;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const unsigned x = i ? w.y : w.x, u = __funnelshift_r(x, x, 3) >> sh;
    v[4 * i + 0] = s * (float)((int)(u & 15u) - 8);
    v[4 * i + 1] = s * (float)((int)(u >> 16 & 15u) - 8);
    v[4 * i + 2] = s * (float)((int)(u >> 8 & 15u) - 8);
    v[4 * i + 3] = s * (float)((int)(u >> 24 & 15u) - 8);
  }
}
// (whole pieces of bfloat16 do not come here: dequantize_w4_kernel has them as they are)
template <typename T>
__device__ __forceinline__ void store8(T* p, const float* v, int left, bool vec) {
  if (sizeof(T) == 4 && vec && left >= 8) {
    *(float4*)p = make_float4(v[0], v[1], v[2], v[3]);
    *(float4*)((float*)p + 4) = make_float4(v[4], v[5], v[6], v[7]);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) if (i < left) p[i] = from_f<T>(v[i]);
}

// The matrix's values (exact in either type).  A warp a slab x chunk: 16 bytes a lane in, a lane's pieces of 8 elements of its two rows out,
// or, where rows are not on 16 bytes, through shared memory and out row by row (1,003 x 1,357: 12 us element by element).
template <typename T>
__global__ void __launch_bounds__(W4_THREADS) dequantize_w4_kernel(W4Ref m, T* out, long long ldo, int vec) {
  const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const long long unit = (long long)blockIdx.x * (W4_THREADS / 32) + (threadIdx.x >> 5);
  const int slab = (int)(unit / m.chunks), chunk = (int)(unit % m.chunks);
  if (slab * W4_SLAB >= m.N) return;
  __shared__ T rows[W4_THREADS / 32][W4_SLAB][W4_CHUNK + 4 / sizeof(T)];
  T (*mine)[W4_CHUNK + 4 / sizeof(T)] = rows[threadIdx.x >> 5];
  const uint4 q = m.q[(size_t)unit * 32 + lane];
  const unsigned w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int k = chunk * W4_CHUNK + h * 32 + c * 8;
    const unsigned s = m.s[((size_t)slab * m.groups + ((chunk * W4_CHUNK + h * 32) >> m.gshift)) * 8 + g];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int n = slab * W4_SLAB + g + 8 * r;
      const unsigned s2 = __byte_perm(s, 0, r ? 0x3232 : 0x1010), off = times_minus_24(s2);
      const unsigned v[4] = {w4_value(w[2 * h], r, s2, off), w4_value(w[2 * h], r + 2, s2, off), w4_value(w[2 * h + 1], r, s2, off), w4_value(w[2 * h + 1], r + 2, s2, off)};
      T* p = out + (size_t)n * ldo + k;
      if (sizeof(T) == 2 && vec && k + 8 <= m.K) {
        if (n < m.N) *(uint4*)p = make_uint4(v[0], v[1], v[2], v[3]);
        continue;
      }
      float f[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(v[i] << 16); f[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u); }
      if (vec) {
        if (n < m.N) store8(p, f, m.K - k, true);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) mine[g + 8 * r][h * 32 + c * 8 + i] = from_f<T>(f[i]);
      }
    }
  }
  if (vec) return;
  __syncwarp();
  const int left = m.K - chunk * W4_CHUNK;
  for (int r = 0; r < W4_SLAB && slab * W4_SLAB + r < m.N; ++r) {
    T* p = out + (size_t)(slab * W4_SLAB + r) * ldo + chunk * W4_CHUNK;
    if (lane < left) p[lane] = mine[r][lane];
    if (lane + 32 < left) p[lane + 32] = mine[r][lane + 32];
  }
}

// A thread eight elements of a token's row, times `scale`.  A token outside the table: zeros and *status = 1.
__global__ void __launch_bounds__(W4_THREADS) embed_rows_w4_kernel(const int* tokens, W4Ref m, float* out, int T, int vec, int* status, float scale) {
  pdl_launch_dependents();
  pdl_wait();
  const int pieces = (m.K + 7) / 8;
  const long long i = (long long)blockIdx.x * W4_THREADS + threadIdx.x;
  const long long t = i / pieces;
  const int k = (int)(i % pieces) * 8;
  if (t >= T) return;
  const int tok = tokens[t];
  float v[8];
  if (tok < 0 || tok >= m.N) {
    if (status && k == 0) atomicExch(status, 1);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.f;
  } else {
    row8(m, tok, k, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= scale;
  }
  store8(out + (size_t)t * m.K + k, v, m.K - k, vec != 0);
}

static bool grid_ok(long long blocks) { return blocks > 0 && blocks < (1ll << 31); }

// Returns when the matrix is laid out: a product reads it ahead of the kernel in front, on whatever stream.
FELLM_API int fellm_quantize_w4(const void* w, int w_bf16, long long ldw, const W4Ref* m, cudaStream_t stream) {
  if (!w) return FELLM_ERR_ARG;
  if (int e = w4_check(m)) return e;
  const W4Out o = {(uint4*)m->q, (unsigned*)m->s, m->N, m->K, m->chunks, m->groups, m->gshift};
  const long long units = (long long)ceil_div(m->N, W4_SLAB) * ((m->chunks + 1) / 2), blocks = (units + W4_THREADS / 32 - 1) / (W4_THREADS / 32);
  if (!grid_ok(blocks)) return FELLM_ERR_SIZE;
  if (w_bf16) quantize_w4_bf16_kernel<<<(unsigned)blocks, W4_THREADS, 0, stream>>>((const bf16*)w, ldw, ldw % 8 == 0 && ((uintptr_t)w & 15) == 0, o);
  else quantize_w4_f32_kernel<<<(unsigned)blocks, W4_THREADS, 0, stream>>>((const float*)w, ldw, ldw % 4 == 0 && ((uintptr_t)w & 15) == 0, o);
  const int e = launch_status();
  return e ? e : (int)cudaStreamSynchronize(stream);
}
FELLM_API int fellm_pack_w4(const void* levels, long long ldl, const void* scales, long long lds, int groups_in, const W4Ref* m, int* bad, cudaStream_t stream) {
  if (!levels || !scales || !bad) return FELLM_ERR_ARG;
  if (int e = w4_check(m)) return e;
  const W4Out o = {(uint4*)m->q, (unsigned*)m->s, m->N, m->K, m->chunks, m->groups, m->gshift};
  const long long units = (long long)ceil_div(m->N, W4_SLAB) * m->chunks, blocks = (units + W4_THREADS / 32 - 1) / (W4_THREADS / 32);
  if (!grid_ok(blocks)) return FELLM_ERR_SIZE;
  pack_w4_kernel<<<(unsigned)blocks, W4_THREADS, 0, stream>>>((const signed char*)levels, ldl, (const bf16*)scales, lds, o, groups_in, bad);
  return launch_status();
}
FELLM_API int fellm_dequantize_w4(const W4Ref* m, void* out, int out_bf16, long long ldo, cudaStream_t stream) {
  if (!out) return FELLM_ERR_ARG;
  if (int e = w4_check(m)) return e;
  const long long blocks = ((long long)ceil_div(m->N, W4_SLAB) * m->chunks + W4_THREADS / 32 - 1) / (W4_THREADS / 32);
  if (!grid_ok(blocks)) return FELLM_ERR_SIZE;
  const int vec = ldo % (out_bf16 ? 8 : 4) == 0 && ((uintptr_t)out & 15) == 0;
  if (out_bf16) dequantize_w4_kernel<bf16><<<(unsigned)blocks, W4_THREADS, 0, stream>>>(*m, (bf16*)out, ldo, vec);
  else dequantize_w4_kernel<float><<<(unsigned)blocks, W4_THREADS, 0, stream>>>(*m, (float*)out, ldo, vec);
  return launch_status();
}
FELLM_API int fellm_embed_rows_w4(const int* tokens, const W4Ref* m, void* out, int T, int* status, float scale, cudaStream_t stream) {
  if (T <= 0) return 0;
  if (!tokens || !out) return FELLM_ERR_ARG;
  if (int e = w4_check(m)) return e;
  const long long blocks = ((long long)T * ceil_div(m->K, 8) + W4_THREADS - 1) / W4_THREADS;
  if (!grid_ok(blocks)) return FELLM_ERR_SIZE;
  return launch_k_class(launch_class_for_rows(T, 2), embed_rows_w4_kernel, dim3((unsigned)blocks, 1, 1), dim3(W4_THREADS, 1, 1), 0, stream, 1,
                        tokens, *m, (float*)out, T, (int)(m->K % 4 == 0 && ((uintptr_t)out & 15) == 0), status, scale);
}
