// Activation checkpoints in 8 bits: microscaled blocks of 32 consecutive elements (memory order), int8 codes and one E8M0
// exponent byte a block, and the backward passes that read the codes where they would read the saved activation.
//
//   m = max |x_i| of the block; e = floor(log2 m) - 6, one more when m * 2^-e >= 127.5, clamped to [-127, 121]
//   q_i = rint(x_i * 2^-e) (ties to even), scale byte e + 127; value = q_i * 2^e
//
// e is the smallest exponent for which nothing rounds past 127, so every element is off by at most half a step (2^(e-1), at most
// m / 127.5); x * 2^-e is exact, which leaves ONE rounding.  The cap keeps 127 * 2^e finite: only above 127.5 * 2^121 =
// 3.39e38 does an element saturate (off by less than one step).  A block with a NaN or an infinity stores scale byte 255 and reads back
// as NaN: a diverged run stays non-finite.  What is rounded to zero loses its sign, and with it the mask of a ReLU or LeakyReLU that is read off the
// checkpoint: IPRGAN_MX8_SIGNS keeps it (mx8_code), at the price of an error below one step instead of half a step for those elements.
// Why int8 and a power of two: at 1.03 bytes an element the noise is 43 dB under a
// normally distributed signal (an 8-bit float's 3-bit mantissa: 31 dB), and the scale costs no multiplication error.
#include "common.h"

#include <float.h>

namespace iprgan {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 nbf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 nbf16x8 __attribute__((ext_vector_type(8)));

// ---- V consecutive elements (V = 4 or 8) of a tensor of storage kind ST (IPRGAN_ST_*): 16-byte accesses per plane where possible
template <int V>
__device__ __forceinline__ void ldbf(const __bf16* b, float* v) {
  if constexpr (V == 8) {
    const nbf16x8 h = *(const nbf16x8*)b;
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = (float)h[k];
  } else {
    const nbf16x4 h = *(const nbf16x4*)b;
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = (float)h[k];
  }
}
template <int V>
__device__ __forceinline__ void stbf(__bf16* b, const float* v) {
  if constexpr (V == 8) {
    nbf16x8 h;
#pragma unroll
    for (int k = 0; k < 8; ++k) h[k] = (__bf16)v[k];
    *(nbf16x8*)b = h;
  } else {
    nbf16x4 h;
#pragma unroll
    for (int k = 0; k < 4; ++k) h[k] = (__bf16)v[k];
    *(nbf16x4*)b = h;
  }
}
template <int ST, int V>
__device__ __forceinline__ void ldv(const void* base, size_t e, size_t ps, float* v) {
  if constexpr (ST == IPRGAN_ST_F32) {
#pragma unroll
    for (int k = 0; k < V; k += 4) {
      const f32x4 a = *(const f32x4*)((const float*)base + e + k);
      v[k] = a.x; v[k + 1] = a.y; v[k + 2] = a.z; v[k + 3] = a.w;
    }
  } else if constexpr (ST == IPRGAN_ST_BF16) {
    ldbf<V>((const __bf16*)base + e, v);
  } else {                                     // three planes: x = h + (m + l), exact
    float m[V], l[V];
    ldbf<V>((const __bf16*)base + e, v);
    ldbf<V>((const __bf16*)base + ps + e, m);
    ldbf<V>((const __bf16*)base + 2 * ps + e, l);
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] += m[k] + l[k];
  }
}
template <int ST, int V>
__device__ __forceinline__ void stv(void* base, size_t e, size_t ps, const float* v) {
#pragma clang fp contract(off)      // v is the fp32 value every storage kind holds: no v - h fused into the product that formed v
  if constexpr (ST == IPRGAN_ST_F32) {
#pragma unroll
    for (int k = 0; k < V; k += 4) {
      const f32x4 a = {v[k], v[k + 1], v[k + 2], v[k + 3]};
      *(f32x4*)((float*)base + e + k) = a;
    }
  } else if constexpr (ST == IPRGAN_ST_BF16) {
    stbf<V>((__bf16*)base + e, v);
  } else {
    float r[V], q[V];
#pragma unroll
    for (int k = 0; k < V; ++k) r[k] = v[k] - (float)(__bf16)v[k];
#pragma unroll
    for (int k = 0; k < V; ++k) q[k] = r[k] - (float)(__bf16)r[k];
    stbf<V>((__bf16*)base + e, v);
    stbf<V>((__bf16*)base + ps + e, r);
    stbf<V>((__bf16*)base + 2 * ps + e, q);
  }
}
// one element (the last, incomplete group of a tensor)
template <int ST>
__device__ __forceinline__ float ld1(const void* base, size_t e, size_t ps) {
  if constexpr (ST == IPRGAN_ST_F32) return ((const float*)base)[e];
  const __bf16* b = (const __bf16*)base + e;
  return ST == IPRGAN_ST_BF16 ? (float)b[0] : (float)b[0] + ((float)b[ps] + (float)b[2 * ps]);
}
template <int ST>
__device__ __forceinline__ void st1(void* base, size_t e, size_t ps, float v) {
#pragma clang fp contract(off)
  if constexpr (ST == IPRGAN_ST_F32) { ((float*)base)[e] = v; return; }
  __bf16* b = (__bf16*)base + e;
  const __bf16 h = (__bf16)v;
  b[0] = h;
  if constexpr (ST == IPRGAN_ST_X3) {
    const float r = v - (float)h;
    const __bf16 m = (__bf16)r;
    b[ps] = m;
    b[2 * ps] = (__bf16)(r - (float)m);
  }
}

// ---- the format
// scale byte of a block from the bit pattern of its largest magnitude (NaN and inf patterns are the largest of all)
__device__ __forceinline__ unsigned mx8_scale(unsigned amax) {
  if (amax >= 0x7f800000u) return 255u;
  int s = (int)(amax >> 23) - 6 + ((amax & 0x7fffffu) >= 0x7f0000u ? 1 : 0);      // e + 127 (subnormal amax: below the clamp)
  return (unsigned)(s < 0 ? 0 : s > 248 ? 248 : s);
}
// 2^-e and 2^e of a scale byte; 255 decodes to NaN, 0 to the subnormal 2^-127
__device__ __forceinline__ float mx8_inv(unsigned s) { return __uint_as_float((254u - s) << 23); }
__device__ __forceinline__ float mx8_step(unsigned s) {
  return __uint_as_float(s == 0 ? 0x00400000u : s == 255u ? 0x7fc00000u : s << 23);
}
// int8 code in the low byte: adding 1.5 * 2^23 rounds to an integer, ties to even; the clamp acts above 127.5 * 2^121 only
// SIGNS: a positive value is never stored as zero but as one step at least - what reads x > 0 off the codes reads it off x.  (A negative one may
// still be stored as zero: neither is positive.)
template <bool SIGNS>
__device__ __forceinline__ unsigned mx8_code(float x, float inv) {
  float t = fminf(fmaxf(x * inv, -127.f), 127.f);
  if (SIGNS) t = x > 0.f ? fmaxf(t, 1.f) : t;
  return __float_as_uint(t + 12582912.f) & 0xffu;
}
template <bool SIGNS>
__device__ __forceinline__ unsigned pack4(const float* v, float inv) {
  return mx8_code<SIGNS>(v[0], inv) | mx8_code<SIGNS>(v[1], inv) << 8 | mx8_code<SIGNS>(v[2], inv) << 16 | mx8_code<SIGNS>(v[3], inv) << 24;
}
template <int V>
__device__ __forceinline__ void ldcodes(const int8_t* q, size_t e, float* v) {          // codes as floats, not yet scaled
  unsigned w[V / 4];
  if constexpr (V == 8) {
    const uint2 a = *(const uint2*)(q + e);
    w[0] = a.x; w[1] = a.y;
  } else {
    w[0] = *(const unsigned*)(q + e);
  }
#pragma unroll
  for (int k = 0; k < V; ++k) v[k] = (float)(int)(int8_t)(w[k / 4] >> 8 * (k & 3));
}

// Quantise: a thread owns V consecutive elements, 32 / V neighbouring lanes share a block and its maximum.  n is the element count;
// lanes past the end contribute zeros.  Bound by HBM (reads sizeof(x), writes 1 + 1/32 bytes an element): 256x128x128x64 bf16 156 to 169 us =
// 4.8 to 5.2 TB/s, the rate of a copy; two or four pieces in flight a thread are slower (173, 179 us).
template <int ST, int V, bool SIGNS>
__global__ __launch_bounds__(256) void mx8_quant_kernel(const void* __restrict__ x, int8_t* __restrict__ q,
                                                        uint8_t* __restrict__ scales, size_t n, size_t ps) {
  constexpr int L = 32 / V;                     // lanes of a block
  const size_t stride = (size_t)gridDim.x * 256 * V;
  // whole waves walk together: a wave's first element decides, so no lane of a block leaves the shuffle early
  for (size_t e = ((size_t)blockIdx.x * 256 + threadIdx.x) * V; e - (size_t)(threadIdx.x & 63) * V < n; e += stride) {
    float v[V];
    const bool full = e + V <= n;
    if (full) {
      ldv<ST, V>(x, e, ps, v);
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] = e + k < n ? ld1<ST>(x, e + k, ps) : 0.f;
    }
    unsigned m = 0;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const unsigned b = __float_as_uint(v[k]) & 0x7fffffffu;
      m = b > m ? b : m;
    }
#pragma unroll
    for (int o = 1; o < L; o <<= 1) {
      const unsigned b = __shfl_xor(m, o, 64);
      m = b > m ? b : m;
    }
    const unsigned s = mx8_scale(m);
    if (s == 255u) {
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] = 0.f;
    }
    const float inv = s == 255u ? 1.f : mx8_inv(s);
    if (full) {
      if constexpr (V == 8) {
        *(uint2*)(q + e) = make_uint2(pack4<SIGNS>(v, inv), pack4<SIGNS>(v + 4, inv));
      } else {
        *(unsigned*)(q + e) = pack4<SIGNS>(v, inv);
      }
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k)
        if (e + k < n) q[e + k] = (int8_t)mx8_code<SIGNS>(v[k], inv);
    }
    if ((threadIdx.x & (L - 1)) == 0 && e < n) scales[e >> 5] = (uint8_t)s;
  }
}

// The border of a norm layer's mask, v > 0  <=>  sgn * x > thr: in 64 bits, and rounded towards the side that keeps the comparison exact for every
// fp32 x.
__device__ __forceinline__ void mask_threshold(float mean, float invstd, float gamma, float beta, float& thr, float& sgn) {
  const double k = (double)gamma * (double)invstd;
  sgn = k < 0.0 ? -1.f : 1.f;
  double t;
  if (k == 0.0) {
    t = beta > 0.f ? -HUGE_VAL : HUGE_VAL;                                           // v = beta everywhere
  } else {
    t = (double)mean - (double)beta / k;
    if (k < 0.0) t = -t;
  }
  thr = __double2float_rd(t);
}
// ... as ONE number for both directions: x > border. With a negative factor the mask is x < -thr, its other side x >= -thr: x > the fp32 number below -thr.
__global__ __launch_bounds__(256) void mx8_border_kernel(const float* __restrict__ gamma, const float* __restrict__ beta,
                                                         const float* __restrict__ mean, const float* __restrict__ invstd,
                                                         float* __restrict__ border, int G, int C) {
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (size_t)G * C) return;
  const int c = (int)(i % C);
  float t, s;
  mask_threshold(mean[i], invstd[i], gamma ? gamma[c] : 1.f, beta ? beta[c] : 0.f, t, s);
  border[i] = s > 0.f ? t : nextafterf(-t, -HUGE_VALF);
}

struct Walk {
  size_t group, sg, sp;                // elements of a group; a stride in groups and elements
  FastDiv d_group, d_row;
  int C, sc;                           // a stride in channels, modulo C
};
// Quantise a norm layer's input with its mask kept: an element above its channel's border b gets the code f + 1 at least, one that is not f at most,
// f = floor(b 2^-e).  Rounding moves an element by half a step at most, so where this acts it is off by less than one.  (A code would have to be 128:
// it stays 127.)  Neighbours in a row are neighbouring channels; a thread follows its place in the group and its channel from stride to stride
// without a division.  256x64x64x128 bf16 90 us, fp32 144, three planes 193 with the borders' launch (77, 130, 193 without borders): half again as many vector
// instructions, which 2-byte elements no longer hide behind HBM.
template <int ST, int V>
__global__ __launch_bounds__(256) void mx8_quant_norm_kernel(const void* __restrict__ x, int8_t* __restrict__ q, uint8_t* __restrict__ scales,
                                                             const float* __restrict__ border, size_t n, size_t ps, Walk wk) {
  constexpr int L = 32 / V;
  const size_t stride = (size_t)gridDim.x * 256 * V;
  const unsigned e0 = (blockIdx.x * 256 + threadIdx.x) * V;                            // (at most 8192 blocks)
  size_t g = fdiv(e0, wk.d_group), p = e0 - g * wk.group;      // (behind the tensor's end: not used)
  int c = (int)(e0 - fdiv(e0, wk.d_row) * wk.C);
  for (size_t e = e0; e - (size_t)(threadIdx.x & 63) * V < n; e += stride) {
    float v[V], b[V];
    const bool in = e < n;                               // (C % V = 0: all of V or none)
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = b[k] = 0.f;
    if (in) {
      ldv<ST, V>(x, e, ps, v);
      ldv<IPRGAN_ST_F32, V>(border, g * wk.C + c, 0, b);
    }
    unsigned m = 0;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const unsigned a = __float_as_uint(v[k]) & 0x7fffffffu;
      m = a > m ? a : m;
    }
#pragma unroll
    for (int o = 1; o < L; o <<= 1) {
      const unsigned a = __shfl_xor(m, o, 64);
      m = a > m ? a : m;
    }
    const unsigned s = mx8_scale(m);
    const float inv = s == 255u ? 1.f : mx8_inv(s);
    unsigned w[V / 4];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float r = rintf(fminf(fmaxf(v[k] * inv, -127.f), 127.f)), f = floorf(b[k] * inv);
      const bool above = v[k] > b[k];
      const float t = __builtin_amdgcn_fmed3f(r, above ? f + 1.f : -127.f, above ? 127.f : f);
      const unsigned code = __float_as_uint(t + 12582912.f) & 0xffu;
      w[k / 4] = k % 4 ? w[k / 4] | code << 8 * (k % 4) : code;
    }
#pragma unroll
    for (int k = 0; k < V / 4; ++k) w[k] = s == 255u ? 0u : w[k];
    if (in) {
      if constexpr (V == 8) *(uint2*)(q + e) = make_uint2(w[0], w[1]);
      else *(unsigned*)(q + e) = w[0];
      if ((threadIdx.x & (L - 1)) == 0) scales[e >> 5] = (uint8_t)s;
    }
    g += wk.sg;
    p += wk.sp;
    if (p >= wk.group) { p -= wk.group; ++g; }
    c += wk.sc;
    if (c >= wk.C) c -= wk.C;
  }
}

// Restore: the same bytes the other way, 146 us at the same size (5.6 TB/s); half as many elements in fp32 174 (3.9 TB/s).  Small tensors are bound by
// the launch (27 540 elements: 2.4 us).
template <int ST, int V>
__global__ __launch_bounds__(256) void mx8_dequant_kernel(const int8_t* __restrict__ q, const uint8_t* __restrict__ scales,
                                                          void* __restrict__ y, size_t n, size_t ps) {
  const size_t stride = (size_t)gridDim.x * 256 * V;
  for (size_t e = ((size_t)blockIdx.x * 256 + threadIdx.x) * V; e < n; e += stride) {
    const float step = mx8_step(scales[e >> 5]);
    if (e + V <= n) {
      float v[V];
      ldcodes<V>(q, e, v);
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] *= step;
      stv<ST, V>(y, e, ps, v);
    } else {
      for (int k = 0; k < V; ++k)
        if (e + k < n) st1<ST>(y, e + k, ps, (float)q[e + k] * step);
    }
  }
}

// dz = dy * act'(out), out read from its checkpoint: one pass, HBM (sizeof(dy) twice and 1 + 1/32 bytes an element)
template <int ST, int V>
__global__ __launch_bounds__(256) void mx8_act_bwd_kernel(const void* __restrict__ dy, const int8_t* __restrict__ q,
                                                          const uint8_t* __restrict__ scales, void* __restrict__ dz, size_t n,
                                                          int act, float slope) {
  const size_t stride = (size_t)gridDim.x * 256 * V;
  for (size_t e = ((size_t)blockIdx.x * 256 + threadIdx.x) * V; e < n; e += stride) {
    const float step = mx8_step(scales[e >> 5]);
    if (e + V <= n) {
      float v[V], g[V];
      ldcodes<V>(q, e, v);
      ldv<ST, V>(dy, e, 0, g);
#pragma unroll
      for (int k = 0; k < V; ++k) g[k] *= act_grad_from_out(v[k] * step, act, slope);
      stv<ST, V>(dz, e, 0, g);
    } else {
      for (int k = 0; k < V; ++k)
        if (e + k < n) st1<ST>(dz, e + k, 0, ld1<ST>(dy, e + k, 0) * act_grad_from_out((float)q[e + k] * step, act, slope));
    }
  }
}

// ---- norm backward from the checkpoint of the layer's input ---------------------------------------------------------------------
//   t = (x - mean) * invstd;  v = t * gamma + beta;  dz = dy * act'(v);  s1 = sum dz, s2 = sum dz * t over the M rows of a group
//   dx = gamma * invstd * (dz - s1 / M - t * s2 / M);  dgamma = s2, dbeta = s1 (summed over groups);  PReLU: dslope = sum dy min(v, 0)
// The activation's mask v > 0 is ONE comparison against a per-channel threshold, x > mean - beta / (gamma * invstd) (the other
// way round for a negative factor; mask_threshold): no rounding of v can flip an element next to zero - and it costs less than forming v.
// x is the checkpoint's value: mx8_quant_norm_kernel keeps it on x's own side of the threshold, mx8_quant_kernel may carry it over by half a step.
// Layout: a block is TC channel groups of V channels x TR = 256 / TC row lanes; blockIdx.y walks channel chunks, blockIdx.z
// groups.  Every thread keeps its channels, so the constants are loaded once for any channel count (TC need not divide 256:
// TC = 9 for 36 channels leaves 4 of 256 threads idle).
// Rows go to the blocks in chunks of 4 * TR, chunk by chunk round the grid: all blocks together sweep the tensor.  (One contiguous
// run of rows a block puts the blocks a power of two apart and on the same memory channels: 208 us instead of 89 for the reduction
// over 256x64x64x128 bf16.)
// Bound by HBM: the statistics need all of dy and the codes before the first dx, so both are read twice - 16.1 + 24.0 us for 128x32x32x128 fp32
// (5.2 and 6.3 TB/s: the second pass walks backwards and finds part of them cached), 93 + 111 us for 256x64x64x128 bf16, three planes 189 + 316.
struct NormGeom {
  int TC, TR, gy, NB;
};
static NormGeom norm_geom(int G, int M, int C, int V) {
  NormGeom g;
  const int cq = cdiv(C, V);
  g.gy = cdiv(cq, 64);
  g.TC = cdiv(cq, g.gy);
  g.TR = 256 / g.TC;
  int nb = cdiv(M, g.TR * 4);
  const int cap = (int)cdivz(1024, (size_t)g.gy * G);         // four blocks a CU in all
  g.NB = nb < cap ? nb : cap;
  return g;
}

// int row numbers, and the grid's limits: 65535 groups, as many chunks of 64 V channels
static bool norm_sizes_ok(long long G, long long M, long long C) {
  return G > 0 && G <= 65535 && M > 0 && M <= (1 << 30) && C >= 4 && C <= 65535 * 512;
}

template <int V>
__device__ __forceinline__ void ldf(const float* p, int c, float dflt, float* v) {
#pragma unroll
  for (int k = 0; k < V; k += 4) {
    f32x4 a = {dflt, dflt, dflt, dflt};
    if (p) a = *(const f32x4*)(p + c + k);
    v[k] = a.x; v[k + 1] = a.y; v[k + 2] = a.z; v[k + 3] = a.w;
  }
}

struct NormArgs {
  const int8_t* q;
  const uint8_t* scales;
  const void* dy;
  void* dx;
  const float *gamma, *beta, *mean, *invstd, *slope_ptr;
  float *part, *sums, *dgamma, *dbeta, *dslope, *colpart;
  size_t dyps, dxps;
  int G, M, C, TC, TR, nsum;          // nsum: partial sums a channel (2, or 3 with a slope gradient)
  int RL;                                  // row lanes of the sums in the apply pass; 0: they are in `sums`
  float slope;
};

// A thread's sums over the rows it walks are fp32 for 64 chunks (256 rows) at a time, then added to a 64-bit sum in its own place in LDS: a
// chain of rounded additions has 256 links however long the tensor (an InstanceNorm of many groups leaves a group to one block: thousands of
// rows a thread).  In registers the wide sums cost the loop its fourth block a CU: 104 us for the reduction over 256x64x64x128 bf16 instead of 92.
constexpr int FOLD = 64;
template <int V>
__device__ __forceinline__ void fold(double* mine, float* s, bool first) {
  asm volatile("" ::: "memory");       // (left to itself the compiler keeps them in registers over the loop)
#pragma unroll
  for (int k = 0; k < V; ++k) {
    mine[k] = first ? (double)s[k] : mine[k] + (double)s[k];
    s[k] = 0.f;
  }
}

// ACT: 0 none, 1 mask with a slope (ReLU: slope 0), 2 the same plus the slope gradient (PReLU)
template <int SG, int V, int ACT>
__global__ __launch_bounds__(256) void mx8_norm_reduce_kernel(const NormArgs a) {
  const float slope = a.slope_ptr ? *a.slope_ptr : a.slope;
  const int grp = blockIdx.z, C = a.C, TC = a.TC, TR = a.TR;
  const int tr = threadIdx.x / TC, tc = threadIdx.x - tr * TC;
  const int c = (blockIdx.y * TC + tc) * V;
  const bool ok = c < C && tr < TR;
  const size_t gofs = (size_t)grp * a.M * C;
  __shared__ double sh[2][256][V + 1];
  float s1[V], s2[V];
  double s3 = 0.;                                        // the slope's gradient is ONE sum over the whole tensor, often much smaller than its
                                                         // terms: two fused multiply-adds an element in 64 bits, free beside the loads
#pragma unroll
  for (int k = 0; k < V; ++k) s1[k] = s2[k] = 0.f;
  if (ok) {
    float m[V], is[V], ga[V], be[V], thr[V], sgn[V];
    ldf<V>(a.mean + (size_t)grp * C, c, 0.f, m);
    ldf<V>(a.invstd + (size_t)grp * C, c, 1.f, is);
    ldf<V>(a.gamma, c, 1.f, ga);
    ldf<V>(a.beta, c, 0.f, be);
    if (ACT) {
#pragma unroll
      for (int k = 0; k < V; ++k) mask_threshold(m[k], is[k], ga[k], be[k], thr[k], sgn[k]);
    }
    double va[ACT == 2 ? V : 1], vb[ACT == 2 ? V : 1];  // the activation's input v = x va + vb
    if (ACT == 2) {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        va[k] = (double)is[k] * (double)ga[k];
        vb[k] = (double)be[k] - (double)m[k] * va[k];
      }
    }
    auto accumulate = [&](const float* x, float step, const float* g) {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float xv = x[k] * step, t = (xv - m[k]) * is[k];
        float dz = g[k];
        if (ACT) {
          const bool pos = sgn[k] * xv > thr[k];
          if (ACT == 2) s3 = fma((double)(pos ? 0.f : g[k]), fma((double)xv, va[k], vb[k]), s3);
          dz = pos ? dz : dz * slope;
        }
        s1[k] += dz;
        s2[k] += dz * t;
      }
    };
    const int start = blockIdx.x * 4 * TR, step = gridDim.x * 4 * TR;      // (every block has a chunk)
#pragma unroll 1
    for (int lo = start; lo < a.M; lo += FOLD * step) {
      for (int r0 = lo; r0 < min(a.M, lo + FOLD * step); r0 += step) {
        const int r = r0 + tr;
        if (r0 + 4 * TR <= a.M) {                          // four rows in flight
          float x[4][V], g[4][V], st[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const size_t e = gofs + (size_t)(r + u * TR) * C + c;
            ldcodes<V>(a.q, e, x[u]);
            st[u] = mx8_step(a.scales[e >> 5]);
            ldv<SG, V>(a.dy, e, a.dyps, g[u]);
          }
#pragma unroll
          for (int u = 0; u < 4; ++u) accumulate(x[u], st[u], g[u]);
        } else {
          for (int q = r; q < a.M; q += TR) {
            float x[V], g[V];
            const size_t e = gofs + (size_t)q * C + c;
            ldcodes<V>(a.q, e, x);
            ldv<SG, V>(a.dy, e, a.dyps, g);
            accumulate(x, mx8_step(a.scales[e >> 5]), g);
          }
        }
      }
      fold<V>(sh[0][threadIdx.x], s1, lo == start);
      fold<V>(sh[1][threadIdx.x], s2, lo == start);
    }
  }
  __shared__ double sh3[4];
  if (ACT == 2) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s3 += __shfl_xor(s3, o, 64);
    if ((threadIdx.x & 63) == 0) sh3[threadIdx.x >> 6] = s3;
  }
  __syncthreads();
  // fixed order: deterministic.  Thread j sums channel j % (TC * V) of sum j / (TC * V)
  const int W = TC * V;
  float* p = a.part + ((size_t)grp * gridDim.x + blockIdx.x) * a.nsum * C;
  for (int j = threadIdx.x; j < a.nsum * W; j += 256) {
    const int which = j / W, ch = j - which * W, col = ch / V, k = ch - col * V;
    const int cc = blockIdx.y * W + ch;
    if (cc >= C) continue;
    double s = 0.;                                       // (up to 256 row lanes in a row: in 64 bits)
    if (which < 2) {
      for (int i = 0; i < TR; ++i) s += sh[which][i * TC + col][k];
    } else if (ch < 2) {                                 // the block's one sum, in two parts, in the chunk's first two places; zero in the rest
      for (int i = 0; i < 4; ++i) s += sh3[i];
      if (ch) s -= (double)(float)s;
    }
    p[(size_t)which * C + cc] = (float)s;
  }
}

// part [G][NB][W] -> sums [G][W], W = nsum * C: 16 columns x 64 row lanes a block, added in fixed order
__global__ __launch_bounds__(1024) void mx8_norm_final_kernel(const float* __restrict__ part, int NB, int W, float* __restrict__ sums) {
  __shared__ double sh[64][17];
  const int cl = threadIdx.x & 15, rl = threadIdx.x >> 4, w = blockIdx.x * 16 + cl;
  part += (size_t)blockIdx.y * NB * W;
  double s = 0.;
  if (w < W) {
#pragma unroll 4
    for (int r = rl; r < NB; r += 64) s += part[(size_t)r * W + w];
  }
  sh[rl][cl] = s;
  __syncthreads();
  if (threadIdx.x < 64) {                               // 4 lanes a column, then their four sums
    double t = 0.;
#pragma unroll
    for (int i = 0; i < 16; ++i) t += sh[rl * 16 + i][cl];
    t += __shfl_xor(t, 16, 64);
    t += __shfl_xor(t, 32, 64);
    if (rl == 0 && w < W) sums[(size_t)blockIdx.y * W + w] = (float)t;
  }
}

// Few partial rows (G NB <= 24 RL): the apply pass adds them itself, every block those of its own channels, RL row lanes x W / 2 quads of the two
// sums - one launch less.  64x32x32x8 fp32: 13.5 -> 10.6 us, wall 25.2 -> 22.4; 16x24x24x64 PReLU: 12.0 both, wall 27.8 -> 25.1.  Past that the
// row of loads in every block costs more than the launch.  tot [2][W]: the sums of rows first .. first + rows.
__device__ __forceinline__ void chunk_sums(const NormArgs& a, int W, int first, int rows, double (*red)[4], float* tot) {
  const int Q = W / 2, rl = threadIdx.x / Q, q = threadIdx.x - rl * Q, which = q >= W / 4, col = blockIdx.y * W + (q - which * (W / 4)) * 4;
  if (rl < a.RL) {
    double d[4] = {0., 0., 0., 0.};
    if (col < a.C) {
      const float* p = a.part + ((size_t)first * a.nsum + which) * a.C + col;
#pragma unroll 4
      for (int r = rl; r < rows; r += a.RL) {
        const f32x4 v = *(const f32x4*)(p + (size_t)r * a.nsum * a.C);
#pragma unroll
        for (int k = 0; k < 4; ++k) d[k] += v[k];
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) red[threadIdx.x][k] = d[k];
  }
  __syncthreads();
  for (int j = threadIdx.x; j < 2 * W; j += 256) {
    double d = 0.;
    for (int l = 0; l < a.RL; ++l) d += red[l * Q + j / 4][j & 3];
    tot[j] = (float)d;
  }
  __syncthreads();
}

template <int SG, int SD, int V, int ACT>
__global__ __launch_bounds__(256) void mx8_norm_apply_kernel(const NormArgs a) {
  const float slope = a.slope_ptr ? *a.slope_ptr : a.slope;
  const int grp = blockIdx.z, C = a.C, TC = a.TC, TR = a.TR;
  const int tr = threadIdx.x / TC, tc = threadIdx.x - tr * TC;
  const int c = (blockIdx.y * TC + tc) * V;
  const bool ok = c < C && tr < TR;
  const size_t gofs = (size_t)grp * a.M * C;
  // the reduction ends at the tensor's end: walking backwards finds its last rows still in the cache
  const int chunks = (a.M + 4 * TR - 1) / (4 * TR);
  __shared__ union {
    double cs[256][V + 1];
    float g[2][256][V + 1];
  } sh;
  __shared__ double red[256][4];
  __shared__ float tot[2 * 64 * V];
  const int W = TC * V;
  if (a.RL) chunk_sums(a, W, grp * gridDim.x, gridDim.x, red, tot);
  float cs[V];
#pragma unroll
  for (int k = 0; k < V; ++k) cs[k] = 0.f;
  if (ok) {
    float m[V], is[V], ga[V], be[V], thr[V], sgn[V], s1[V], s2[V];
    const float* su = a.sums + (size_t)grp * a.nsum * C;
    ldf<V>(a.mean + (size_t)grp * C, c, 0.f, m);
    ldf<V>(a.invstd + (size_t)grp * C, c, 1.f, is);
    ldf<V>(a.gamma, c, 1.f, ga);
    ldf<V>(a.beta, c, 0.f, be);
    if (a.RL) {
#pragma unroll
      for (int k = 0; k < V; ++k) { s1[k] = tot[tc * V + k]; s2[k] = tot[W + tc * V + k]; }
    } else {
      ldf<V>(su, c, 0.f, s1);
      ldf<V>(su + C, c, 0.f, s2);
    }
    if (ACT) {
#pragma unroll
      for (int k = 0; k < V; ++k) mask_threshold(m[k], is[k], ga[k], be[k], thr[k], sgn[k]);
    }
    const float invM = 1.f / (float)a.M;
#pragma unroll
    for (int k = 0; k < V; ++k) { ga[k] *= is[k]; s1[k] *= invM; s2[k] *= invM; }
    auto body = [&](size_t e, const float* x, float step, const float* g) {
      float o[V];
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float xv = x[k] * step, t = (xv - m[k]) * is[k];
        float dz = g[k];
        if (ACT) dz = sgn[k] * xv > thr[k] ? dz : dz * slope;
        o[k] = ga[k] * (dz - s1[k] - t * s2[k]);
        cs[k] += o[k];
      }
      stv<SD, V>(a.dx, e, a.dxps, o);
    };
    const int start = chunks - 1 - (int)blockIdx.x, nb = (int)gridDim.x;
#pragma unroll 1
    for (int hi = start; hi >= 0; hi -= FOLD * nb) {
      for (int q = hi; q >= 0 && q > hi - FOLD * nb; q -= nb) {
        const int r0 = q * 4 * TR, r = r0 + tr;
        if (r0 + 4 * TR <= a.M) {
          float x[4][V], g[4][V], st[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const size_t e = gofs + (size_t)(r + u * TR) * C + c;
            ldcodes<V>(a.q, e, x[u]);
            st[u] = mx8_step(a.scales[e >> 5]);
            ldv<SG, V>(a.dy, e, a.dyps, g[u]);
          }
#pragma unroll
          for (int u = 0; u < 4; ++u) body(gofs + (size_t)(r + u * TR) * C + c, x[u], st[u], g[u]);
        } else {
          for (int z = r; z < a.M; z += TR) {
            float x[V], g[V];
            const size_t e = gofs + (size_t)z * C + c;
            ldcodes<V>(a.q, e, x);
            ldv<SG, V>(a.dy, e, a.dyps, g);
            body(e, x, mx8_step(a.scales[e >> 5]), g);
          }
        }
      }
      if (a.colpart) fold<V>(sh.cs[threadIdx.x], cs, hi == start);
    }
  }
  if (a.colpart) {                                     // column sums of dx: [row of blocks][2][C], as iprgan_colsum_partials reads them
    __syncthreads();
    for (int ch = threadIdx.x; ch < W; ch += 256) {
      const int col = ch / V, k = ch - col * V;
      if (blockIdx.y * W + ch >= C) continue;
      double s = 0.;
      for (int i = 0; i < TR; ++i) s += sh.cs[i * TC + col][k];
      a.colpart[((size_t)grp * gridDim.x + blockIdx.x) * 2 * C + blockIdx.y * W + ch] = (float)s;
    }
    __syncthreads();
  }
  if (blockIdx.x != 0 || grp != 0) return;             // (uniform) one block of each channel chunk sums the groups' parameter gradients
  if (a.dgamma && a.RL) {
    if (a.G > 1) {
      __syncthreads();
      chunk_sums(a, W, 0, a.G * gridDim.x, red, tot);
    }
    for (int ch = threadIdx.x; ch < W; ch += 256) {
      const int cc = blockIdx.y * W + ch;
      if (cc >= C) continue;
      a.dgamma[cc] = tot[W + ch];
      a.dbeta[cc] = tot[ch];
    }
  } else if (a.dgamma) {
    double d1[V], d2[V];
#pragma unroll
    for (int k = 0; k < V; ++k) d1[k] = d2[k] = 0.;
    if (ok) {
      for (int g = tr; g < a.G; g += TR) {
        float t1[V], t2[V];
        ldf<V>(a.sums + (size_t)g * a.nsum * C, c, 0.f, t1);
        ldf<V>(a.sums + (size_t)g * a.nsum * C + C, c, 0.f, t2);
#pragma unroll
        for (int k = 0; k < V; ++k) { d1[k] += t1[k]; d2[k] += t2[k]; }
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < V; ++k) { sh.g[0][threadIdx.x][k] = (float)d1[k]; sh.g[1][threadIdx.x][k] = (float)d2[k]; }
    __syncthreads();
    for (int ch = threadIdx.x; ch < W; ch += 256) {
      const int col = ch / V, k = ch - col * V, cc = blockIdx.y * W + ch;
      if (cc >= C) continue;
      double b = 0., g = 0.;
      for (int i = 0; i < TR; ++i) { b += sh.g[0][i * TC + col][k]; g += sh.g[1][i * TC + col][k]; }
      a.dgamma[cc] = (float)g;
      a.dbeta[cc] = (float)b;
    }
  }
  if (a.dslope && blockIdx.y == 0) {
    double d = 0.;
    if (a.RL) {
      for (int j = threadIdx.x; j < (int)(gridDim.x * gridDim.y) * 2; j += 256) {
        const int r = j / 2 / (int)gridDim.y, y = j / 2 - r * (int)gridDim.y;
        d += (double)a.part[((size_t)r * a.nsum + 2) * C + y * W + (j & 1)];
      }
    } else {
      for (int j = threadIdx.x; j < C; j += 256) d += (double)a.sums[2 * (size_t)C + j];
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) d += __shfl_xor(d, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6][0] = d;
    __syncthreads();
    if (threadIdx.x == 0) *a.dslope = (float)((red[0][0] + red[1][0]) + (red[2][0] + red[3][0]));
  }
}

template <int SG, int SD, int V>
static int norm_bwd_go(NormArgs a, const NormGeom& g, int act, hipStream_t st) {
  const dim3 grid(g.NB, g.gy, a.G), blk(256);
  auto red = act == 0 ? mx8_norm_reduce_kernel<SG, V, 0> : act == 1 ? mx8_norm_reduce_kernel<SG, V, 1> : mx8_norm_reduce_kernel<SG, V, 2>;
  hipLaunchKernelGGL(red, grid, blk, 0, st, a);
  IPR_LAUNCH_CHECK();
  if (!a.RL) {
    hipLaunchKernelGGL(mx8_norm_final_kernel, dim3(cdiv(a.nsum * a.C, 16), a.G), dim3(1024), 0, st, a.part, g.NB, a.nsum * a.C, a.sums);
    IPR_LAUNCH_CHECK();
  }
  auto app = act == 0 ? mx8_norm_apply_kernel<SG, SD, V, 0> : mx8_norm_apply_kernel<SG, SD, V, 1>;
  hipLaunchKernelGGL(app, grid, blk, 0, st, a);
  IPR_LAUNCH_CHECK();
  return 0;
}

static inline bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }
static inline bool al8(const void* p) { return ((uintptr_t)p & 7) == 0; }
static inline unsigned flat_grid(size_t n, int V) {
  const size_t b = cdivz(n, (size_t)256 * V);
  return (unsigned)(b < 8192 ? b : 8192);
}

}  // namespace iprgan

using namespace iprgan;

extern "C" {

int iprgan_mx8_quant(const void* x, void* codes, void* scales, size_t n, int kind, size_t pstride, void* stream) {
  IPR_CHECK(n > 0, "mx8_quant: empty input");
  IPR_CHECK(x && codes && scales, "mx8_quant: null operand");
  const bool signs = kind & IPRGAN_MX8_SIGNS;
  kind &= ~IPRGAN_MX8_SIGNS;
  IPR_CHECK(kind >= IPRGAN_ST_F32 && kind <= IPRGAN_ST_X3, "mx8_quant: storage kind %d", kind);
  IPR_CHECK((kind == IPRGAN_ST_F32 ? al16(x) : al8(x)) && al16(codes), "mx8_quant: operands must be 16-byte aligned (8: bf16 and three planes)");
  if (kind == IPRGAN_ST_X3 && !pstride) pstride = n;
  IPR_CHECK(kind != IPRGAN_ST_X3 || pstride >= n, "mx8_quant: plane stride %zu below %zu elements", pstride, n);
  hipStream_t st = (hipStream_t)stream;
  const bool wide = kind != IPRGAN_ST_F32 && al16(x) && (kind != IPRGAN_ST_X3 || pstride % 8 == 0);
  IPR_CHECK(kind != IPRGAN_ST_X3 || pstride % 4 == 0, "mx8_quant: plane stride %zu is not a multiple of 4", pstride);
#define QUANT(ST, V) (signs ? mx8_quant_kernel<ST, V, true> : mx8_quant_kernel<ST, V, false>)
  auto k = kind == IPRGAN_ST_F32 ? QUANT(0, 4) : kind == IPRGAN_ST_BF16 ? (wide ? QUANT(1, 8) : QUANT(1, 4)) : wide ? QUANT(2, 8) : QUANT(2, 4);
#undef QUANT
  hipLaunchKernelGGL(k, dim3(flat_grid(n, wide ? 8 : 4)), dim3(256), 0, st, x, (int8_t*)codes, (uint8_t*)scales, n, pstride);
  IPR_LAUNCH_CHECK();
  return 0;
}

int iprgan_mx8_quant_norm(const void* x, void* codes, void* scales, const float* gamma, const float* beta, const float* save_mean,
                          const float* save_invstd, float* ws, long long G, long long M, long long C, int kind, size_t pstride, void* stream) {
  IPR_CHECK(G > 0 && M > 0 && C > 0, "mx8_quant_norm: empty input (%lld groups of %lld rows, %lld channels)", G, M, C);
  IPR_CHECK(C % 4 == 0, "mx8_quant_norm: C=%lld must be a multiple of 4", C);
  IPR_CHECK(norm_sizes_ok(G, M, C), "mx8_quant_norm: %lld groups of %lld rows, %lld channels (at most 65535, 2^30, 65535 * 512)", G, M, C);
  IPR_CHECK(x && codes && scales && save_mean && save_invstd && ws, "mx8_quant_norm: null operand");
  IPR_CHECK(!gamma == !beta, "mx8_quant_norm: gamma and beta are both needed (or both absent)");
  IPR_CHECK(kind >= IPRGAN_ST_F32 && kind <= IPRGAN_ST_X3, "mx8_quant_norm: storage kind %d", kind);
  const size_t n = (size_t)G * M * C, tab = (size_t)G * C;
  if (kind == IPRGAN_ST_X3 && !pstride) pstride = n;
  IPR_CHECK(kind != IPRGAN_ST_X3 || (pstride >= n && pstride % 4 == 0), "mx8_quant_norm: plane stride %zu for %zu elements", pstride, n);
  IPR_CHECK((kind == IPRGAN_ST_F32 ? al16(x) : al8(x)) && al16(codes) && al16(ws), "mx8_quant_norm: operands must be 16-byte aligned (8: bf16 and three planes)");
  IPR_CHECK(cdivz(tab, 256) * 256 <= 0xffffffffull, "mx8_quant_norm: %lld groups of %lld channels are too many borders", G, C);
  hipStream_t st = (hipStream_t)stream;
  hipLaunchKernelGGL(mx8_border_kernel, dim3((unsigned)cdivz(tab, 256)), dim3(256), 0, st, gamma, beta, save_mean, save_invstd, ws, (int)G, (int)C);
  IPR_LAUNCH_CHECK();
  const bool wide = kind != IPRGAN_ST_F32 && C % 8 == 0 && al16(x) && (kind != IPRGAN_ST_X3 || pstride % 8 == 0);
  auto k = kind == IPRGAN_ST_F32 ? mx8_quant_norm_kernel<0, 4> : kind == IPRGAN_ST_BF16 ? (wide ? mx8_quant_norm_kernel<1, 8> : mx8_quant_norm_kernel<1, 4>)
           : wide ? mx8_quant_norm_kernel<2, 8> : mx8_quant_norm_kernel<2, 4>;
  const unsigned blocks = flat_grid(n, wide ? 8 : 4);
  const size_t stride = (size_t)blocks * 256 * (wide ? 8 : 4);
  Walk w;
  w.group = (size_t)M * C;
  w.sg = stride / w.group;
  w.sp = stride % w.group;
  w.C = (int)C;
  w.sc = (int)(stride % (size_t)C);
  w.d_group = make_fastdiv((uint32_t)(w.group < 0x7fffffff ? w.group : 0x7fffffff));      // (a thread's first element is below 2^25)
  w.d_row = make_fastdiv((uint32_t)C);
  hipLaunchKernelGGL(k, dim3(blocks), dim3(256), 0, st, x, (int8_t*)codes, (uint8_t*)scales, ws, n, pstride, w);
  IPR_LAUNCH_CHECK();
  return 0;
}

int iprgan_mx8_dequant(const void* codes, const void* scales, void* y, size_t n, int kind, size_t pstride, void* stream) {
  IPR_CHECK(n > 0, "mx8_dequant: empty input");
  IPR_CHECK(y && codes && scales, "mx8_dequant: null operand");
  IPR_CHECK(kind >= IPRGAN_ST_F32 && kind <= IPRGAN_ST_X3, "mx8_dequant: storage kind %d", kind);
  IPR_CHECK((kind == IPRGAN_ST_F32 ? al16(y) : al8(y)) && al16(codes), "mx8_dequant: operands must be 16-byte aligned (8: bf16 and three planes)");
  if (kind == IPRGAN_ST_X3 && !pstride) pstride = n;
  IPR_CHECK(kind != IPRGAN_ST_X3 || (pstride >= n && pstride % 4 == 0), "mx8_dequant: plane stride %zu for %zu elements", pstride, n);
  hipStream_t st = (hipStream_t)stream;
  const bool wide = kind != IPRGAN_ST_F32 && al16(y) && (kind != IPRGAN_ST_X3 || pstride % 8 == 0);
  auto k = kind == IPRGAN_ST_F32 ? mx8_dequant_kernel<0, 4> : kind == IPRGAN_ST_BF16 ? (wide ? mx8_dequant_kernel<1, 8> : mx8_dequant_kernel<1, 4>)
           : wide ? mx8_dequant_kernel<2, 8> : mx8_dequant_kernel<2, 4>;
  hipLaunchKernelGGL(k, dim3(flat_grid(n, wide ? 8 : 4)), dim3(256), 0, st, (const int8_t*)codes, (const uint8_t*)scales, y, n, pstride);
  IPR_LAUNCH_CHECK();
  return 0;
}

int iprgan_mx8_act_bwd(const void* dy, const void* codes, const void* scales, void* dz, size_t n, int act, float slope, int kind,
                       void* stream) {
  IPR_CHECK(n > 0, "mx8_act_bwd: empty input");
  IPR_CHECK(dy && dz && codes && scales, "mx8_act_bwd: null operand");
  IPR_CHECK(kind == IPRGAN_ST_F32 || kind == IPRGAN_ST_BF16, "mx8_act_bwd: storage kind %d (fp32 or bf16)", kind);
  IPR_CHECK(act >= IPRGAN_ACT_NONE && act <= IPRGAN_ACT_SIGMOID_PM1, "mx8_act_bwd: activation %d", act);
  IPR_CHECK((kind == IPRGAN_ST_F32 ? al16(dy) && al16(dz) : al8(dy) && al8(dz)) && al16(codes),
            "mx8_act_bwd: operands must be 16-byte aligned (8: bf16)");
  const bool wide = kind == IPRGAN_ST_BF16 && al16(dy) && al16(dz);
  auto k = kind == IPRGAN_ST_F32 ? mx8_act_bwd_kernel<0, 4> : wide ? mx8_act_bwd_kernel<1, 8> : mx8_act_bwd_kernel<1, 4>;
  hipLaunchKernelGGL(k, dim3(flat_grid(n, wide ? 8 : 4)), dim3(256), 0, (hipStream_t)stream, dy, (const int8_t*)codes,
                     (const uint8_t*)scales, dz, n, act, slope);
  IPR_LAUNCH_CHECK();
  return 0;
}

// the most partial rows either vector width asks for
size_t iprgan_mx8_norm_bwd_ws_floats(long long G, long long M, long long C) {
  if (!norm_sizes_ok(G, M, C)) return 0;
  const NormGeom a = norm_geom((int)G, (int)M, (int)C, 4), b = norm_geom((int)G, (int)M, (int)C, 8);
  const size_t nb = (size_t)G * (a.NB > b.NB ? a.NB : b.NB);
  return nb * 3 * C + (size_t)G * 3 * C + (nb + 64) * 2 * C;         // partials, sums, column sums of dx and their compacted rows
}

int iprgan_mx8_norm_bwd(const void* codes, const void* scales, const void* dy, const float* gamma, const float* beta,
                        const float* save_mean, const float* save_invstd, const float* slope_dev, void* dx, float* dgamma,
                        float* dbeta, float* dslope, float* ws, long long groups, long long rows, long long channels, int act, float slope,
                        float* dbias_prev, long long dbias_n, float dbias_beta, int dy_kind, size_t dy_pstride, int dx_kind,
                        size_t dx_pstride, void* stream) {
  IPR_CHECK(groups > 0 && rows > 0 && channels > 0, "mx8_norm_bwd: empty input (%lld groups of %lld rows, %lld channels)", groups, rows, channels);
  IPR_CHECK(channels % 4 == 0, "mx8_norm_bwd: C=%lld must be a multiple of 4", channels);
  IPR_CHECK(norm_sizes_ok(groups, rows, channels), "mx8_norm_bwd: %lld groups of %lld rows, %lld channels (at most 65535, 2^30, 65535 * 512)", groups, rows, channels);
  const int G = (int)groups, M = (int)rows, C = (int)channels;
  IPR_CHECK(codes && scales && dy && dx && save_mean && save_invstd && ws, "mx8_norm_bwd: null operand");
  IPR_CHECK(act == IPRGAN_ACT_NONE || !gamma == !beta, "mx8_norm_bwd: the mask is recomputed from x: gamma and beta are both needed (or both absent)");
  IPR_CHECK(!beta || gamma, "mx8_norm_bwd: beta without gamma");
  IPR_CHECK(!dgamma == !dbeta, "mx8_norm_bwd: dgamma and dbeta are both needed (or both absent)");
  IPR_CHECK(act == IPRGAN_ACT_NONE || act == IPRGAN_ACT_RELU || act == IPRGAN_ACT_LRELU,
            "mx8_norm_bwd: activation %d (none, ReLU and LeakyReLU / PReLU can be recomputed from the input)", act);
  IPR_CHECK(!dslope || (slope_dev && G == 1), "mx8_norm_bwd: a slope gradient needs the slope on the device and one group");
  IPR_CHECK(!slope_dev || act == IPRGAN_ACT_LRELU, "mx8_norm_bwd: a device slope belongs to IPRGAN_ACT_LRELU");
  IPR_CHECK(dy_kind >= IPRGAN_ST_F32 && dy_kind <= IPRGAN_ST_X3, "mx8_norm_bwd: dy kind %d", dy_kind);
  IPR_CHECK(dx_kind == dy_kind || (dy_kind == IPRGAN_ST_F32 && dx_kind == IPRGAN_ST_X3), "mx8_norm_bwd: dx kind %d from dy kind %d", dx_kind, dy_kind);
  IPR_CHECK(!dbias_prev || (dbias_n > 0 && dbias_n <= C), "mx8_norm_bwd: %lld bias gradients for %d channels", dbias_n, C);
  const size_t n = (size_t)G * M * C;
  if (!dy_pstride) dy_pstride = n;
  if (!dx_pstride) dx_pstride = n;
  IPR_CHECK(dy_kind != IPRGAN_ST_X3 || (dy_pstride >= n && dy_pstride % 4 == 0), "mx8_norm_bwd: dy plane stride %zu", dy_pstride);
  IPR_CHECK(dx_kind != IPRGAN_ST_X3 || (dx_pstride >= n && dx_pstride % 4 == 0), "mx8_norm_bwd: dx plane stride %zu", dx_pstride);
  IPR_CHECK((dy_kind == IPRGAN_ST_F32 ? al16(dy) : al8(dy)) && (dx_kind == IPRGAN_ST_F32 ? al16(dx) : al8(dx)) && al16(codes) && al16(save_mean) && al16(save_invstd) && al16(ws) && (!gamma || al16(gamma)) && (!beta || al16(beta)),
            "mx8_norm_bwd: operands must be 16-byte aligned (8: bf16 and three planes)");
  hipStream_t st = (hipStream_t)stream;
  const bool wide = dy_kind != IPRGAN_ST_F32 && C % 8 == 0 && al16(dy) && al16(dx) && (dy_kind != IPRGAN_ST_X3 || (dy_pstride % 8 == 0 && dx_pstride % 8 == 0));
  const NormGeom g = norm_geom(G, M, C, wide ? 8 : 4);
  IPR_CHECK(g.gy <= 65535, "mx8_norm_bwd: %d channels in chunks of %d", C, g.TC * (wide ? 8 : 4));
  NormArgs a;
  memset(&a, 0, sizeof(a));
  a.q = (const int8_t*)codes; a.scales = (const uint8_t*)scales; a.dy = dy; a.dx = dx;
  a.gamma = gamma; a.beta = beta; a.mean = save_mean; a.invstd = save_invstd; a.slope_ptr = slope_dev;
  a.dgamma = dgamma; a.dbeta = dbeta; a.dslope = dslope; a.dyps = dy_pstride; a.dxps = dx_pstride;
  a.G = G; a.M = M; a.C = C; a.TC = g.TC; a.TR = g.TR; a.slope = act == IPRGAN_ACT_RELU ? 0.f : slope;
  a.nsum = dslope ? 3 : 2;
  const int quads = g.TC * (wide ? 8 : 4) / 2, lanes = 256 / quads < 16 ? 256 / quads : 16;
  a.RL = (long long)G * g.NB <= 24 * lanes ? lanes : 0;
  a.part = ws;
  a.sums = ws + (size_t)G * g.NB * a.nsum * C;
  float* colpart = a.sums + (size_t)G * a.nsum * C;
  a.colpart = dbias_prev ? colpart : nullptr;
  const int am = act == IPRGAN_ACT_NONE ? 0 : dslope ? 2 : 1;
  int rc;
  if (dy_kind == IPRGAN_ST_F32) {
    rc = dx_kind == IPRGAN_ST_F32 ? norm_bwd_go<0, 0, 4>(a, g, am, st) : norm_bwd_go<0, 2, 4>(a, g, am, st);
  } else if (dy_kind == IPRGAN_ST_BF16) {
    rc = wide ? norm_bwd_go<1, 1, 8>(a, g, am, st) : norm_bwd_go<1, 1, 4>(a, g, am, st);
  } else {
    rc = wide ? norm_bwd_go<2, 2, 8>(a, g, am, st) : norm_bwd_go<2, 2, 4>(a, g, am, st);
  }
  if (rc) return rc;
  if (dbias_prev) return iprgan_colsum_partials(colpart, G * g.NB, C, (int)dbias_n, dbias_prev, dbias_beta, stream);
  return 0;
}

}  // extern "C"
