// Microscaled 4-bit floating point: quantisation, reading back, the product y = act(x W^T + b) with 4-bit weights, and the
// product's gradient with respect to x.
//
// Format: blocks of 32 elements along a row, one E8M0 exponent byte a block, elements E2M1 (sign, 2 exponent bits, 1 mantissa
// bit: 0, .5, 1, 1.5, 2, 3, 4, 6).  Rows are padded with zero codes to whole groups of 128 elements, so a row is KB = 4 *
// ceil(cols / 128) blocks: KB * 16 bytes of codes (element 2i in the low half of byte i) and KB scale bytes - every block is 16 aligned
// bytes, every 128 elements' scales one aligned word, and no kernel has a tail along K on its 4-bit operands.
//   e = floor(log2 max|x|) - 2, one more when max|x| * 2^-e >= 7, clamped to [-127, 125]; round to nearest, ties to the even code
// e is the smallest exponent for which nothing rounds past 6: an element is off by at most half the distance of its neighbours.
// x * 2^-e is exact, so this is ONE rounding.  A block with a NaN or an infinity stores scale byte 255 and reads back as NaN.
//
// Sizes in the comments below are M x N x K (x [M][K], W [N][K]) throughout, times the device's.
#include "common.h"

#include <atomic>

namespace iprgan {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// Rows of odd lengths start on any element: vector accesses that promise no more than the element's own alignment (the memory system takes
// them at any address).  1281 x 2085 x 3237 fp32: 203 us element by element, 79 like this; nothing changes where rows are aligned.
typedef f32x4 f32x4u __attribute__((aligned(4)));
typedef bf16x4 bf16x4u __attribute__((aligned(2)));
typedef bf16x8 bf16x8u __attribute__((aligned(2)));
typedef bf16x8 bf16x8w __attribute__((aligned(4)));

// scale byte from the bit pattern of the largest magnitude; see mx8.hip for the same rule with 8-bit codes
__device__ __forceinline__ unsigned mx4_scale(unsigned amax) {
  if (amax >= 0x7f800000u) return 255u;
  const int s = (int)(amax >> 23) - 2 + ((amax & 0x7fffffu) >= 0x600000u ? 1 : 0);
  return (unsigned)(s < 0 ? 0 : s > 252 ? 252 : s);
}
__device__ __forceinline__ float mx4_inv(unsigned s) { return __uint_as_float((254u - s) << 23); }
__device__ __forceinline__ float mx4_step(unsigned s) {
  return __uint_as_float(s == 0 ? 0x00400000u : s == 255u ? 0x7fc00000u : s << 23);
}

// 8 consecutive elements of row `r` from column c on; zero behind the row's end
template <bool BF>
__device__ __forceinline__ void ld8(const void* base, size_t r, int ld, int c, float* v) {
  if (c + 8 <= ld) {
    if constexpr (BF) {
      const bf16x8 h = *(const bf16x8u*)((const __bf16*)base + r * ld + c);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = (float)h[k];
    } else {
      const float* p = (const float*)base + r * ld + c;
      const f32x4 a = *(const f32x4u*)p, b = *(const f32x4u*)(p + 4);
#pragma unroll
      for (int k = 0; k < 4; ++k) { v[k] = a[k]; v[k + 4] = b[k]; }
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    v[k] = 0.f;
    if (c + k < ld) v[k] = BF ? (float)((const __bf16*)base)[r * ld + c + k] : ((const float*)base)[r * ld + c + k];
  }
}

// A thread owns 8 consecutive elements (4 bytes of codes); 4 neighbouring lanes share a block.  HBM-bound: 1024 x 18432 fp32 13.5 us (6.3 TB/s, part
// of it from the cache), 8192 x 8192 bf16 33 us (5.1 TB/s); reading back 16.4 us at the first size.
template <bool BF>
__global__ __launch_bounds__(256) void mx4_quant_kernel(const void* __restrict__ x, unsigned* __restrict__ codes,
                                                        uint8_t* __restrict__ scales, unsigned groups, int cols, FastDiv d_row) {
  const unsigned stride = gridDim.x * 256;
  for (unsigned i = blockIdx.x * 256 + threadIdx.x; i < groups; i += stride) {       // groups % 16 == 0: a block's lanes stay together
    const unsigned r = fdiv(i, d_row), c = (i - r * d_row.d) * 8;
    float v[8];
    ld8<BF>(x, r, cols, (int)c, v);
    unsigned m = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const unsigned b = __float_as_uint(v[k]) & 0x7fffffffu;
      m = b > m ? b : m;
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      const unsigned b = __shfl_xor(m, o, 64);
      m = b > m ? b : m;
    }
    const unsigned s = mx4_scale(m);
    unsigned w = 0;
    if (s != 255u) {
      const float inv = mx4_inv(s);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = fminf(fmaxf(v[k] * inv, -6.f), 6.f);       // (the clamp acts at the exponent cap only)
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], 1.f, 0);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], 1.f, 1);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], 1.f, 2);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], 1.f, 3);
    }
    codes[i] = w;
    if ((i & 3) == 0) scales[i >> 2] = (uint8_t)s;
  }
}

template <bool BF>
__global__ __launch_bounds__(256) void mx4_dequant_kernel(const unsigned* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                          void* __restrict__ y, unsigned groups, int cols, FastDiv d_row) {
  const unsigned stride = gridDim.x * 256;
  for (unsigned i = blockIdx.x * 256 + threadIdx.x; i < groups; i += stride) {
    const unsigned r = fdiv(i, d_row), c = (i - r * d_row.d) * 8;
    if ((int)c >= cols) continue;
    const unsigned w = codes[i];
    const float step = mx4_step(scales[i >> 2]);
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 1),
                p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 2), q = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 3);
    const float v[8] = {a.x * step, a.y * step, b.x * step, b.y * step, p.x * step, p.y * step, q.x * step, q.y * step};
    if ((int)c + 8 <= cols) {
      if (BF) {
        bf16x8 h;
#pragma unroll
        for (int k = 0; k < 8; ++k) h[k] = (__bf16)v[k];
        *(bf16x8u*)((__bf16*)y + (size_t)r * cols + c) = h;
      } else {
        float* o = (float*)y + (size_t)r * cols + c;
        const f32x4 lo = {v[0], v[1], v[2], v[3]}, hi = {v[4], v[5], v[6], v[7]};
        *(f32x4u*)o = lo;
        *(f32x4u*)(o + 4) = hi;
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if ((int)c + k >= cols) break;
        if (BF) ((__bf16*)y)[(size_t)r * cols + c + k] = (__bf16)v[k];
        else ((float*)y)[(size_t)r * cols + c + k] = v[k];
      }
    }
  }
}

// ---- the product ---------------------------------------------------------------------------------------------------------------
// Both forms compute the TRANSPOSED tile: the weights are the matrix instruction's first operand (its rows = output columns n), x is the
// second (its columns = output rows m), so a lane's four results are four consecutive n of one row m: 16-byte fp32 or 8-byte bf16 stores.
struct LinArgs {
  const void* x;                 // [M][K] fp32 / bf16, or 4-bit codes
  const uint8_t* xs;             // scales of a 4-bit x
  const uint8_t *w, *ws;         // weights' codes [N][KB * 16] and scales [N][KB]
  const float* bias;
  void* y;
  float* slab;                   // [splits][M][N] when the K axis is split
  int M, N, K, KB, steps_per_split;      // a step is 128 elements of K
  int act, y_bf16, vec8;                 // vec8: 8 bf16 columns at once
  float slope;
};

// none, ReLU, LeakyReLU (none: slope 1).  tanh and the sigmoid go through the slab pass: their code, once an accumulator, would make the
// product kernels' epilogues several times their loops.
__device__ __forceinline__ float lin_act(float v, int act, float slope) {
  return v > 0.f ? v : act == IPRGAN_ACT_RELU ? 0.f : v * slope;
}
__device__ __forceinline__ void store4(const LinArgs& a, int z, int m, int n, f32x4 v) {
  if (m >= a.M || n >= a.N) return;
  const size_t o = ((size_t)(a.slab ? z : 0) * a.M + m) * a.N + n;
  if (n + 4 <= a.N) {
    if (!a.slab) {
      f32x4 b = {0.f, 0.f, 0.f, 0.f};
      if (a.bias) b = *(const f32x4u*)(a.bias + n);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = lin_act(v[k] + b[k], a.act, a.slope);
      if (a.y_bf16) {
        const bf16x4 h = {(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
        *(bf16x4u*)((__bf16*)a.y + o) = h;
        return;
      }
    }
    *(f32x4u*)((a.slab ? a.slab : (float*)a.y) + o) = v;
    return;
  }
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    if (n + k >= a.N) continue;
    if (a.slab) {
      a.slab[o + k] = v[k];
      continue;
    }
    const float r = lin_act(v[k] + (a.bias ? a.bias[n + k] : 0.f), a.act, a.slope);
    if (a.y_bf16) ((__bf16*)a.y)[o + k] = (__bf16)r;
    else ((float*)a.y)[o + k] = r;
  }
}

// 8 consecutive elements of a row as loaded: 8 floats, or 8 bf16
template <bool BF>
struct Raw8 {
  f32x4 a, b;
};
template <>
struct Raw8<true> {
  bf16x8 h;
};
// ... from column c on; zero behind the row's end, which only the LAST step along the row can meet (`tail`, uniform).  Elsewhere there is no
// branch: the first version branched on every load, and every branch waited for its own load (4096^3 bf16: 287 us instead of 183).
template <bool BF>
__device__ __forceinline__ Raw8<BF> row8(const uint8_t* row, int c, int cols, bool tail) {
  Raw8<BF> r;
  auto get = [&](int at) {
    if constexpr (BF) {
      r.h = *(const bf16x8u*)(row + (size_t)at * 2);
    } else {
      r.a = *(const f32x4u*)(row + (size_t)at * 4);
      r.b = *(const f32x4u*)(row + (size_t)at * 4 + 16);
    }
  };
  if (!tail) {
    get(c);
    return r;
  }
  const bool full = c + 8 <= cols;
  if (cols >= 8) get(full ? c : 0);
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    if constexpr (BF) {
      if (!full) r.h[k] = c + k < cols ? ((const __bf16*)row)[c + k] : (__bf16)0.f;
    } else {
      if (full) continue;
      const float v = c + k < cols ? ((const float*)row)[c + k] : 0.f;
      if (k < 4) r.a[k & 3] = v;
      else r.b[k & 3] = v;
    }
  }
  return r;
}

// 8 fp4 elements (one word) of a block -> bf16, exact (a 4-bit value times a power of two)
__device__ __forceinline__ bf16x8 widen_fp4(unsigned w, float scale) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1),
               c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3);
  const bf16x8 r = {a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
  return r;
}
// x in PL bf16 planes: one (bf16 input) or three (fp32 input: x = h + m + l exactly, so the products with the exactly widened weights
// are exact and only the fp32 accumulation rounds)
template <int PL>
__device__ __forceinline__ void split_planes(const float* v, bf16x8* p) {
#pragma unroll
  for (int k = 0; k < 8; ++k) p[0][k] = (__bf16)v[k];
  if (PL == 3) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float r = v[k] - (float)p[0][k];
      p[1][k] = (__bf16)r;
      p[2][k] = (__bf16)(r - (float)p[1][k]);
    }
  }
}

template <int PL, class R>
__device__ __forceinline__ void split_raw(const R& r, bf16x8* p) {
  if constexpr (PL == 1) {
    p[0] = r.h;
  } else {
    const float v[8] = {r.a[0], r.a[1], r.a[2], r.a[3], r.b[0], r.b[1], r.b[2], r.b[3]};
    split_planes<3>(v, p);
  }
}

// Which tile and K split a block takes.  The XCDs get contiguous runs of (split, tile) pairs - each has its own L2 - and inside a split the
// tiles go 4 along n, then down m: blocks that share a K range of x, or rows of W, sit on one XCD (4096^3 fp32: 389 -> 381 us).
struct Place {
  int n, m, z;
};
__device__ __forceinline__ Place place(int tn, int tm) {
  const unsigned all = gridDim.x, per = all / 8, rem = all % 8, xcd = blockIdx.x % 8;
  const unsigned id = xcd * per + min(xcd, rem) + blockIdx.x / 8, tiles = (unsigned)tn * tm;
  const unsigned z = id / tiles, t = id - z * tiles, grp = t / (4u * tm), in = t - grp * 4u * tm, gw = min(4u, tn - grp * 4u);
  return Place{(int)(grp * 4 + in % gw), (int)(in / gw), (int)z};
}

// Few rows (1 x 16384 x 8192 with 4-bit x 13.9 us, 5.1 TB/s of weights; 1 x 4096 x 4096 bf16 4.7 us): 8 waves, WK along K x 8 / WK along n (16 *
// NF columns each); both operands straight from memory to registers, no barrier before the end, where the WK partial tiles are added in LDS in fixed order - one launch where a split over blocks takes two.  XT: 0 = 4-bit x
// (the scaled instruction), 1 = bf16, 3 = fp32 (planes).  Bound by latency, or by the split of fp32 x into planes (176 vector instructions a
// step and 16 rows, repeated by every wave: why more rows go through LDS below).
template <int MF, int NF, int XT>
__global__ __launch_bounds__(512, NF == 1 && XT != 3 ? 4 : 2) void mx4_direct_kernel(const LinArgs a, int tn, int tm, int wk) {
  constexpr int PL = XT == 3 ? 3 : 1;
  __shared__ f32x4 red[8][NF * MF][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
  const Place pl = place(tn, tm);
  const int kw = wave % wk, nw = wave / wk;
  const int n0 = (pl.n * (8 / wk) + nw) * 16 * NF, m0 = pl.m * 16 * MF;
  const int s0 = pl.z * a.steps_per_split + kw, s1 = min(a.KB / 4, (pl.z + 1) * a.steps_per_split);
  f32x4 acc[NF][MF];
#pragma unroll
  for (int n = 0; n < NF; ++n)
#pragma unroll
    for (int m = 0; m < MF; ++m) acc[n][m] = f32x4{0.f, 0.f, 0.f, 0.f};
  const i32x4 *wp[NF], *xp[MF];
  // (the four scale bytes of a row and step by one lane each, handed round: byte loads by all lanes cost as many cache accesses as the codes)
  const unsigned* wsp = (const unsigned*)(a.ws + (size_t)min(n0 + (lane & (16 * NF - 1)), a.N - 1) * a.KB);
  const unsigned* xsp = (const unsigned*)(a.xs + (size_t)min(m0 + (lane & (16 * MF - 1)), a.M - 1) * a.KB);
#pragma unroll
  for (int n = 0; n < NF; ++n) {
    const size_t r = min(n0 + n * 16 + i, a.N - 1);         // rows past the end repeat the last one; their results are not stored
    wp[n] = (const i32x4*)(a.w + r * a.KB * 16) + g;
  }
  constexpr unsigned ESZ = XT == 1 ? 2 : 4;
  const uint8_t* xrow[MF];
#pragma unroll
  for (int m = 0; m < MF; ++m) {
    const size_t r = min(m0 + m * 16 + i, a.M - 1);
    xp[m] = (const i32x4*)((const uint8_t*)a.x + r * a.KB * 16) + g;
    xrow[m] = (const uint8_t*)a.x + r * a.K * ESZ;
  }
  i32x4 wq[2][NF], xq[2][MF];
  int wsn[2], xsn[2];
  Raw8<XT == 1> xv[2][XT ? MF : 1][4];
  auto load = [&](int s, int b) {
#pragma unroll
    for (int n = 0; n < NF; ++n) wq[b][n] = wp[n][s * 4];
    if (lane < 16 * NF) wsn[b] = (int)wsp[s];
    if (XT == 0 && (MF == 4 || lane < 16 * MF)) xsn[b] = (int)xsp[s];
#pragma unroll
    for (int m = 0; m < MF; ++m) {
      if constexpr (XT == 0) {
        xq[b][m] = xp[m][s * 4];
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) xv[b][m][j] = row8<XT == 1>(xrow[m], s * 128 + g * 32 + j * 8, a.K, s * 128 + 128 > a.K);
      }
    }
  };
  auto mul = [&](int b) {
    int wsc[NF], xsc[MF];
#pragma unroll
    for (int n = 0; n < NF; ++n) wsc[n] = __builtin_amdgcn_ds_bpermute((n * 16 + i) * 4, wsn[b]) >> (g * 8) & 255;
#pragma unroll
    for (int m = 0; m < MF; ++m) xsc[m] = XT == 0 ? __builtin_amdgcn_ds_bpermute((m * 16 + i) * 4, xsn[b]) >> (g * 8) & 255 : 0;
    if constexpr (XT == 0) {
#pragma unroll
      for (int n = 0; n < NF; ++n)
#pragma unroll
        for (int m = 0; m < MF; ++m) {
          const i32x4 p = wq[b][n], q = xq[b][m];
          const i32x8 w8 = {p[0], p[1], p[2], p[3], 0, 0, 0, 0}, x8 = {q[0], q[1], q[2], q[3], 0, 0, 0, 0};
          acc[n][m] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w8, x8, acc[n][m], 4, 4, 0, wsc[n], 0, xsc[m]);
        }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        bf16x8 wf[NF];
#pragma unroll
        for (int n = 0; n < NF; ++n) wf[n] = widen_fp4((unsigned)wq[b][n][j], mx4_step((unsigned)wsc[n]));
#pragma unroll
        for (int m = 0; m < MF; ++m) {
          bf16x8 p[PL];
          split_raw<PL>(xv[b][m][j], p);
#pragma unroll
          for (int q = PL - 1; q >= 0; --q)
#pragma unroll
            for (int n = 0; n < NF; ++n) acc[n][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf[n], p[q], acc[n][m], 0, 0, 0);
        }
      }
    }
  };
  if (s0 < s1) load(s0, 0);
#pragma unroll 1
  for (int s = s0; s < s1; s += 2 * wk) {
    if (s + wk < s1) load(s + wk, 1);
    __builtin_amdgcn_sched_barrier(0);                      // the next step's loads leave before this one is multiplied
    mul(0);
    if (s + wk >= s1) break;
    if (s + 2 * wk < s1) load(s + 2 * wk, 0);
    __builtin_amdgcn_sched_barrier(0);
    mul(1);
  }
  if (wk > 1) {
    if (kw) {
#pragma unroll
      for (int n = 0; n < NF; ++n)
#pragma unroll
        for (int m = 0; m < MF; ++m) red[wave][n * MF + m][lane] = acc[n][m];
    }
    __syncthreads();
    if (kw) return;
    for (int k = 1; k < wk; ++k)
#pragma unroll
      for (int n = 0; n < NF; ++n)
#pragma unroll
        for (int m = 0; m < MF; ++m) acc[n][m] += red[wave + k][n * MF + m][lane];
  }
#pragma unroll
  for (int n = 0; n < NF; ++n)
#pragma unroll
    for (int m = 0; m < MF; ++m) store4(a, pl.z, m0 + m * 16 + i, n0 + n * 16 + g * 4, acc[n][m]);
}

typedef __attribute__((address_space(3))) void lds_void;
template <int BYTES>
__device__ __forceinline__ void lds_dma(__amdgpu_buffer_rsrc_t rs, unsigned lds, unsigned voff, unsigned soff) {
#if defined(__HIP_DEVICE_COMPILE__)      // (an error that the host pass defers silently, dropping the kernel's stub)
  if constexpr (BYTES == 16) __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void*)(uintptr_t)lds, 16, voff, soff, 0, 0);
  else __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void*)(uintptr_t)lds, 4, voff, soff, 0, 0);
#endif
}
// (the barrier alone is no fence to the compiler)
__device__ __forceinline__ void block_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// More rows of fp32 / bf16 x.  A block is 4 waves: each owns 16 * NF output columns (their weights come through a part of LDS that is the wave's
// own: a lane holds whole 16-byte blocks, lane group g block g of the step, and the step's four instructions take 8 elements of each block -
// the order of K is free as long as both operands agree); the 16 * MF rows of x are shared through LDS, split into planes on the way in.
// What bounds it at 4096^3: bf16 136 us, 1010 TFLOP/s - two blocks a CU, whose loads, LDS traffic and multiplications overlap to about 45 % of
// the matrix pipe; fp32 309 to 318 us, three products each.
// (a barrier for LDS alone: __syncthreads would also wait for the loads in flight)
__device__ __forceinline__ void lds_sync() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  block_barrier();
}
// Where a row keeps its 16-byte pieces: piece c at c ^ swz(row).  A 16-byte LDS read serves 16 lanes at a time, lanes 0-3, 12-15, 20-23 and
// 24-27 the first: rows 0-3 and 12-15 of lane group 0, rows 4-11 of group 1.  This order of the rows (0-15) gives the halves disjoint banks.
__device__ __forceinline__ int swz(int row) { return (row & 3) | ((row >> 2 & 1) * 2 ^ (row >> 3) * 3) << 2; }
template <int MF, int NF, int PL>
__global__ __launch_bounds__(256, NF < 4 ? 2 : 1) void mx4_linear_kernel(const LinArgs a, int tn, int tm) {
  constexpr int AHEAD = (PL == 1 ? NF < 4 : MF <= 2) ? 2 : 1;      // (three: 1 to 15 % slower; two elsewhere: no gain)
  constexpr bool DMA = !(MF == 4 && NF == 2 && PL == 3);
  __shared__ u32x4 ws[DMA ? AHEAD : 1][4][DMA ? NF * 64 : 1];
  constexpr int XB = PL == 1 ? 2 : 1;                       // planes of x: two buffers of bf16 (one barrier a step: 4096^3 143 -> 137 us), one of
                                                            // fp32, 48 KB at most, where blocks beside it hide the barriers
  __shared__ bf16x8 xs[XB][PL][MF * 16][16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, g = lane >> 4;
  const Place pl = place(tn, tm);
  const int n0 = pl.n * 64 * NF + wave * 16 * NF, m0 = pl.m * 16 * MF;
  const int s0 = pl.z * a.steps_per_split, s1 = min(a.KB / 4, s0 + a.steps_per_split);
  const int xr = threadIdx.x >> 4, xc = (threadIdx.x & 15) * 8;
  f32x4 acc[NF][MF];
#pragma unroll
  for (int n = 0; n < NF; ++n)
#pragma unroll
    for (int m = 0; m < MF; ++m) acc[n][m] = f32x4{0.f, 0.f, 0.f, 0.f};
  // W goes through LDS by DMA: four neighbouring lanes fetch a row's 64 bytes, where the fragments' own order (neighbours in different rows) takes
  // an access a lane (4096^3: bf16 149 -> 140 us, fp32 328 -> 318).  Piece c of row r at c ^ ((r >> 1) & 3): no conflicts.  Not for fp32 in 64 x
  // 128 tiles, where the 8 KB more leave two blocks a CU instead of three (64 x 16384 x 8192, either way round: 67 -> 73).  Columns past N repeat the last row;
  // their results are not stored.
  const __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc((void*)(a.w + (size_t)min(n0, a.N - 1) * a.KB * 16), 0, -1, 0x00020000);
  unsigned wo[NF];
#pragma unroll
  for (int n = 0; n < NF; ++n) {
    const int row = DMA ? lane >> 2 : i, piece = DMA ? (lane & 3) ^ ((lane >> 3) & 3) : g;
    wo[n] = (unsigned)max(min(n * 16 + row, a.N - 1 - n0), 0) * a.KB * 16 + piece * 16;
  }
  const unsigned wbase = (unsigned)(uintptr_t)(lds_void*)&ws[0][wave][0];
  const int fr = i * 4 + (g ^ ((i >> 1) & 3));
  // a step's four scale bytes of one column a lane: 64 cache accesses an instruction, where a byte a lane and fragment takes 64 for each
  const unsigned* sp = (const unsigned*)(a.ws + (size_t)min(n0 + (lane & (16 * NF - 1)), a.N - 1) * a.KB);
  const uint8_t* xrow[MF];
#pragma unroll
  for (int t = 0; t < MF; ++t) xrow[t] = (const uint8_t*)a.x + (size_t)min(m0 + xr + t * 16, a.M - 1) * a.K * (PL == 1 ? 2 : 4);
  u32x4 wq[NF], wn[DMA ? 1 : NF];
  unsigned sq[NF], sn[AHEAD];
  Raw8<PL == 1> xv[AHEAD][MF];
  auto load = [&](int s, int b) {
#pragma unroll
    for (int n = 0; n < NF; ++n) {
      if constexpr (DMA) lds_dma<16>(rw, wbase + b * (4 * NF * 1024) + n * 1024, wo[n], s * 64);
      else wn[n] = __builtin_amdgcn_raw_buffer_load_b128(rw, wo[n], s * 64, 0);
    }
    asm volatile("" ::: "memory");                            // (x is loaded after W: once x is there, W is)
    if (NF == 4 || lane < 16 * NF) sn[b] = sp[s];
#pragma unroll
    for (int t = 0; t < MF; ++t) xv[b][t] = row8<PL == 1>(xrow[t], s * 128 + xc, a.K, s * 128 + 128 > a.K);
  };
#pragma unroll
  for (int b = 0; b < AHEAD; ++b)
    if (s0 + b < s1) load(s0 + b, b);
  auto step = [&](int s, int b) {
#pragma unroll
    for (int t = 0; t < MF; ++t) {
      if constexpr (PL == 1) asm volatile("" ::"v"(xv[b][t].h) : "memory");
      else asm volatile("" ::"v"(xv[b][t].a), "v"(xv[b][t].b) : "memory");
    }
    if (XB == 1 && s > s0) lds_sync();                      // every wave has read the last step's planes
    bf16x8(*xb)[MF * 16][16] = xs[XB == 2 ? (s - s0) & 1 : 0];
#pragma unroll
    for (int t = 0; t < MF; ++t) {
      bf16x8 p[PL];
      split_raw<PL>(xv[b][t], p);
#pragma unroll
      for (int q = 0; q < PL; ++q) xb[q][xr + t * 16][(threadIdx.x & 15) ^ swz(xr)] = p[q];
    }
#pragma unroll
    for (int n = 0; n < NF; ++n) {
      if constexpr (DMA) wq[n] = ws[b][wave][n * 64 + fr];
      else wq[n] = wn[n];
      sq[n] = (unsigned)__builtin_amdgcn_ds_bpermute((n * 16 + i) * 4, (int)sn[b]) >> (g * 8) & 255u;
    }
    lds_sync();
    if (s + AHEAD < s1) load(s + AHEAD, b);                 // in flight while AHEAD steps are multiplied
    // (8 elements j, plane q) pairs in turn, the smallest plane first; x fragments are read D pairs ahead of their use - left to itself the
    // compiler waits for every read (2048 x 4096 x 4096 fp32: 225 -> 206 us)
    constexpr int P = 4 * PL, D = PL == 1 ? 3 : 2;
    bf16x8 xf[D + 1][MF], wf[NF];
    auto read = [&](int p) {
#pragma unroll
      for (int m = 0; m < MF; ++m) xf[p % (D + 1)][m] = xb[PL - 1 - p % PL][m * 16 + i][(g * 4 + p / PL) ^ swz(i)];
    };
#pragma unroll
    for (int p = 0; p < D; ++p) read(p);
#pragma unroll
    for (int p = 0; p < P; ++p) {
      if (p + D < P) read(p + D);
      if (p % PL == 0) {
#pragma unroll
        for (int n = 0; n < NF; ++n) wf[n] = widen_fp4(wq[n][p / PL], mx4_step(sq[n]));
      }
#pragma unroll
      for (int m = 0; m < MF; ++m)
#pragma unroll
        for (int n = 0; n < NF; ++n) acc[n][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf[n], xf[p % (D + 1)][m], acc[n][m], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
#pragma unroll 1
  for (int s = s0; s < s1; s += AHEAD) {
#pragma unroll
    for (int b = 0; b < AHEAD; ++b)
      if (s + b < s1) step(s + b, b);
  }
#pragma unroll
  for (int n = 0; n < NF; ++n)
#pragma unroll
    for (int m = 0; m < MF; ++m) store4(a, pl.z, m0 + m * 16 + i, n0 + n * 16 + g * 4, acc[n][m]);
}

// ---- many rows of 4-bit x -----------------------------------------------------------------------------------------------------------
// The scaled matrix instruction multiplies 128 elements of K at once: a lane holds one 16-byte block of its row (i = lane & 15, block
// g = lane >> 4 of the step) and that block's scale byte, for each operand.
// Many rows: TN x TM tiles, WN x WM waves, codes and scales of both operands through two LDS slots filled by LDS-DMA, a stage of 256
// elements of K (two steps of the instruction) in each; the first half of the waves loads W, the second half x.
//   * A row is 128 bytes a stage, a whole cache line: 25 M L2 requests at 8192^3, where stages of 128 elements made 42 M of half a line
//     each (2048 x 4096 x 4096: 38 -> 35 us; 8192^3 300 -> 290).
//   * The stages of ALL tiles a block computes form one stream (a block walks tiles blockIdx.x, + gridDim.x, ..), and the fragments of the
//     next step are read while the last D of this one are multiplied, so the matrix pipe does not wait at a step's or a tile's start.
//     Where a stage ends, a wave waits for its share of the next, then ONE barrier - every wave's share has landed, and every wave is
//     done with this stage's slot, which is refilled.
//   * Piece c (16 bytes) of row r sits at position c ^ ((r >> 1) & 7): the 16 lanes that an LDS read serves together then touch all
//     banks.  A DMA lane's place in LDS is fixed, so the swizzle is in its address.
//   * S16 (rows of whole 512-element groups): the scales of two stages travel as one 16-byte piece a row; 4-byte pieces, two a row and
//     stage, cost the intake as much as a third of the codes (64 cache lines an instruction).
//   * Tile order: the XCDs take contiguous runs (each has its own L2), and a run walks 4 tiles along n, then down m.
// What bounds it, 256 x 256 at 8192^3, 281 to 302 us: the multiplications alone take 160 to 196 at the clock the chip sustains under them (it falls from 2.4 to
// 1.9 GHz), the loop without its DMA 226: LDS serves the fragments and the DMA's writes for 60 % of the time, in the matrix pipe's way.
template <int TN, int TM, int WN, int WM, bool S16>
__global__ __launch_bounds__(WN* WM * 64, 2) void mx4_gemm4_kernel(const LinArgs a, int tn, int tm) {
  constexpr int WAVES = WN * WM, NT = TN / WN / 16, MT = TM / WM / 16, D = 3;       // D: W fragments read ahead
  constexpr int PC = (TN + TM) / 8 / WAVES, PS = (TN + TM) / 64 / WAVES, L = PC + (S16 ? 0 : 2 * PS);      // DMA pieces a wave and stage
  constexpr int XC = TN * 128, WS = XC + TM * 128, XS = WS + (S16 ? 0 : TN * 8), STAGE = XS + (S16 ? 0 : TM * 8);
  constexpr int RING = 2 * STAGE, SSLOT = (TN + TM) * 16, SR = S16 ? 16 : 4;                   // SR: scale bytes of a row in LDS
  static_assert(TN == TM && WAVES % 2 == 0 && PS >= 1 && NT % (D + 1) == 0 && MT == 4, "each half of the waves loads one operand");
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  const unsigned ring = (unsigned)(uintptr_t)(lds_void*)smem;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, g = lane >> 4;
  const int s0 = blockIdx.z * a.steps_per_split, steps = min(a.KB / 4, s0 + a.steps_per_split) - s0;
  const unsigned total = (unsigned)tn * tm, per = total / 8, rem = total % 8;
  auto tile_at = [&](unsigned b, int& n0, int& m0) {
    const unsigned xcd = b % 8, id = xcd * per + min(xcd, rem) + b / 8;
    const unsigned grp = id / (4u * tm), in = id - grp * 4u * tm, gw = min(4u, tn - grp * 4u);
    n0 = (int)(grp * 4 + in % gw) * TN;
    m0 = (int)(in / gw) * TM;
  };
  const int tiles = (int)((total - blockIdx.x + gridDim.x - 1) / gridDim.x);            // blockIdx.x < total
  const int turns = (steps + 1) / 2, stages = tiles * turns;                            // the last stage of an odd number of steps holds one

  // the loading side: cursor (it, is) = tile and stage of the next piece, the tile's addresses
  const bool mine_w = wave < WAVES / 2;
  const int sub = mine_w ? wave : wave - WAVES / 2;
  __amdgpu_buffer_rsrc_t rc, rs;
  unsigned vc[PC], vs[PS];
  const unsigned piece = (lane & 7) ^ (lane >> 4);                                       // of even p; p odd: ^ 4
  int it = 0, is = 0;
  auto aim = [&](int k) {
    int n0, m0;
    tile_at(blockIdx.x + k * gridDim.x, n0, m0);
    const int base = mine_w ? n0 : m0, last = (mine_w ? a.N : a.M) - 1 - base;              // rows past the end repeat the last one
    rc = __builtin_amdgcn_make_buffer_rsrc((void*)((mine_w ? a.w : (const uint8_t*)a.x) + (size_t)base * a.KB * 16), 0, -1, 0x00020000);
    rs = __builtin_amdgcn_make_buffer_rsrc((void*)((mine_w ? a.ws : a.xs) + (size_t)base * a.KB), 0, -1, 0x00020000);
#pragma unroll
    for (int p = 0; p < PC; ++p) vc[p] = (unsigned)min((sub * PC + p) * 8 + (lane >> 3), last) * a.KB * 16 + (piece ^ (p & 1) * 4) * 16;
#pragma unroll
    for (int p = 0; p < PS; ++p) vs[p] = (unsigned)min((sub * PS + p) * 64 + lane, last) * a.KB;
  };
  const unsigned lc = ring + (mine_w ? 0 : XC) + sub * PC * 1024;
  const unsigned ls = S16 ? ring + RING + (mine_w ? 0 : TN * 16) + sub * PS * 1024 : ring + (mine_w ? WS : XS) + sub * PS * 256;
  auto issue = [&](int d) {                             // stage d of the stream (S16: every tile has a multiple of 2 stages)
    const unsigned slot = (unsigned)(d & 1) * STAGE, s = s0 + is * 2;
    const bool one = is * 2 + 1 == steps;               // the second half would lie behind the rows: the first again, not read from LDS
    if constexpr (S16) {
      if ((d & 1) == 0) {
#pragma unroll
        for (int p = 0; p < PS; ++p) lds_dma<16>(rs, ls + ((d >> 1) & 1) * SSLOT + p * 1024, vs[p], s * 4);
      }
    }
#pragma unroll
    for (int p = 0; p < PC; ++p) lds_dma<16>(rc, lc + slot + p * 1024, one && (piece ^ (p & 1) * 4) >= 4 ? vc[p] - 64 : vc[p], s * 64);
    if constexpr (!S16) {
#pragma unroll
      for (int p = 0; p < PS; ++p) {
        lds_dma<4>(rs, ls + slot + p * 256, vs[p], s * 4);
        lds_dma<4>(rs, ls + slot + (mine_w ? TN : TM) * 4 + p * 256, vs[p], one ? s * 4 : s * 4 + 4);
      }
    }
    if (++is == turns) {
      is = 0;
      if (++it < tiles) aim(it);
    }
  };
  const int wn = wave % WN, wm = wave / WN;
  i32x4 xf[2][MT], wf[D + 1];
  int xsc[2][MT], wsc[D + 1];
  const uint8_t *wl, *xl, *wsl, *xsl;                   // where this lane reads the fragments and scales of a step
  auto look = [&](int d, int u) {
    const uint8_t* st = smem + (d & 1) * STAGE;
    const int f = i * 128 + ((u * 4 + g) ^ (i >> 1)) * 16;
    wl = st + wn * (NT * 2048) + f;
    xl = st + XC + wm * (MT * 2048) + f;
    const uint8_t* sc = S16 ? smem + RING + ((d >> 1) & 1) * SSLOT + ((d & 1) * 2 + u) * 4 + g : st + WS + u * (TN * 4) + g;
    wsl = sc + (wn * NT * 16 + i) * SR;
    xsl = sc + TN * (S16 ? 16 : 8) + (wm * MT * 16 + i) * SR;
  };
  auto read_w = [&](int n, int f) { wf[f] = *(const i32x4*)(wl + n * 2048); wsc[f] = wsl[n * 16 * SR]; };
  auto read_x = [&](int u, int m) { xf[u][m] = *(const i32x4*)(xl + m * 2048); xsc[u][m] = xsl[m * 16 * SR]; };
  aim(0);
  issue(0);
  if (stages > 1) {
    issue(1);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(L) : "memory");
  } else {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }
  block_barrier();
  look(0, 0);
#pragma unroll
  for (int m = 0; m < MT; ++m) read_x(0, m);
#pragma unroll
  for (int n = 0; n < D; ++n) read_w(n, n);
  int d = 0;
#pragma unroll 1
  for (int k = 0; k < tiles; ++k) {
    f32x4 acc[NT][MT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int m = 0; m < MT; ++m) acc[n][m] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int t = 0; t < turns; ++t, ++d) {
      const bool one = t * 2 + 1 == steps;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (u && one) {                                 // the next stage's x went to xf[1]
#pragma unroll
          for (int m = 0; m < MT; ++m) { xf[0][m] = xf[1][m]; xsc[0][m] = xsc[1][m]; }
          break;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if (n == NT - D) {                            // everything of this step has been read
            if (u || one) {
              if (d + 1 < stages) {
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
                block_barrier();
                if (d + 2 < stages) issue(d + 2);
              }
              look(d + 1, 0);                           // (behind the last stage: read, not used)
            } else {
              look(d, 1);
            }
          }
          read_w((n + D) % NT, (n + D) % (D + 1));
          if (n == NT - 3) { read_x(u ^ 1, 0); read_x(u ^ 1, 1); }
          if (n == NT - 2) read_x(u ^ 1, 2);
          if (n == NT - 1) read_x(u ^ 1, 3);
          const i32x4 wq = wf[n % (D + 1)];
          const i32x8 w8 = {wq[0], wq[1], wq[2], wq[3], 0, 0, 0, 0};
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            const i32x8 x8 = {xf[u][m][0], xf[u][m][1], xf[u][m][2], xf[u][m][3], 0, 0, 0, 0};
            acc[n][m] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w8, x8, acc[n][m], 4, 4, 0, wsc[n % (D + 1)], 0, xsc[u][m]);
          }
          // (an empty read of each result: left to itself the compiler moves the multiplications behind the branches, past all reads)
#pragma unroll
          for (int m = 0; m < MT; ++m) asm volatile("" : "+v"(acc[n][m]));
          __builtin_amdgcn_sched_barrier(0);            // the reads stay D fragments ahead of the multiplications
        }
      }
    }
    int n0, m0;
    tile_at(blockIdx.x + k * gridDim.x, n0, m0);
    n0 += wn * NT * 16;
    m0 += wm * MT * 16 + i;
    if (a.vec8 && !a.slab) {
      // bf16, 16 bytes a lane: lane groups g and g ^ 1 trade halves of two neighbouring fragments, so that a lane holds 8 columns
#pragma unroll
      for (int n = 0; n < NT; n += 2) {
        const int col = n0 + (n + (g & 1)) * 16 + (g >> 1) * 8;
        float b0[4], b1[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int ca = n0 + n * 16 + g * 4 + c;
          b0[c] = a.bias && ca < a.N ? a.bias[ca] : 0.f;
          b1[c] = a.bias && ca + 16 < a.N ? a.bias[ca + 16] : 0.f;
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          bf16x2 p[4];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            p[c] = bf16x2{(__bf16)lin_act(acc[n][m][2 * c] + b0[2 * c], a.act, a.slope), (__bf16)lin_act(acc[n][m][2 * c + 1] + b0[2 * c + 1], a.act, a.slope)};
            p[2 + c] = bf16x2{(__bf16)lin_act(acc[n + 1][m][2 * c] + b1[2 * c], a.act, a.slope),
                              (__bf16)lin_act(acc[n + 1][m][2 * c + 1] + b1[2 * c + 1], a.act, a.slope)};
          }
          const auto lo = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, p[0]), __builtin_bit_cast(unsigned, p[2]), false, false);
          const auto hi = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, p[1]), __builtin_bit_cast(unsigned, p[3]), false, false);
          const u32x4 o = {lo[0], hi[0], lo[1], hi[1]};
          if (m0 + m * 16 < a.M && col < a.N) *(u32x4*)((__bf16*)a.y + (size_t)(m0 + m * 16) * a.N + col) = o;
        }
      }
    } else {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) store4(a, blockIdx.z, m0 + m * 16, n0 + n * 16 + g * 4, acc[n][m]);
    }
  }
}

// out[m][n] = act(sum over the splits + bias[n]).  A block covers 256 / LZ groups of V elements; LZ lanes of each group add every
// LZ-th split and are then added in lane order: a fixed order whatever the launch, and the loads of 64 splits are not one chain.
template <int V, int LZ>
__global__ __launch_bounds__(256) void mx4_slab_reduce_kernel(const float* __restrict__ slab, int splits, size_t total, int N,
                                                              const float* __restrict__ bias, void* __restrict__ out, int act,
                                                              float slope, int out_bf16) {
  constexpr int GR = 256 / LZ;
  __shared__ float sh[LZ][GR][V + (V > 1)];
  const int gr = threadIdx.x % GR, lz = threadIdx.x / GR;
  const size_t e = ((size_t)blockIdx.x * GR + gr) * V;
  float s[V];
#pragma unroll
  for (int k = 0; k < V; ++k) s[k] = 0.f;
  if (e < total) {
#pragma unroll 4
    for (int z = lz; z < splits; z += LZ) {
      const float* p = slab + (size_t)z * total + e;
      if constexpr (V == 4) {
        const f32x4 q = *(const f32x4*)p;
#pragma unroll
        for (int k = 0; k < 4; ++k) s[k] += q[k];
      } else {
        s[0] += p[0];
      }
    }
  }
#pragma unroll
  for (int k = 0; k < V; ++k) sh[lz][gr][k] = s[k];
  __syncthreads();
  if (lz || e >= total) return;
  const int n = (int)(e % (size_t)N);
#pragma unroll
  for (int k = 0; k < V; ++k) {
    float v = 0.f;
#pragma unroll
    for (int z = 0; z < LZ; ++z) v += sh[z][gr][k];
    s[k] = act_apply(v + (bias ? bias[n + k] : 0.f), act, slope);
  }
  if constexpr (V == 4) {
    if (out_bf16) {
      const bf16x4 h = {(__bf16)s[0], (__bf16)s[1], (__bf16)s[2], (__bf16)s[3]};
      *(bf16x4*)((__bf16*)out + e) = h;
    } else {
      const f32x4 q = {s[0], s[1], s[2], s[3]};
      *(f32x4*)((float*)out + e) = q;
    }
  } else {
    if (out_bf16) ((__bf16*)out)[e] = (__bf16)s[0];
    else ((float*)out)[e] = s[0];
  }
}

// ---- gradient with respect to x: dx[m][k] = sum_n dy[m][n] W[n][k] -----------------------------------------------------------------
// The reduction runs along the rows of W, so a lane needs 8 rows' values of one k.  It reads KW words (8 KW elements of one block) of each of
// its 8 rows, widens them with the rows' scales and interleaves row pairs: the eight vectors it then holds per word are its operands for EIGHT
// instructions j = 0..7, whose row i stands for k = 8 KW i + j - the 8 x 8 transposition costs 32 permutes a word and no LDS.  A wave
// covers 128 KW k; the block's 4 waves split the rows n and add their tiles through LDS.  The lane's results over j are 8 consecutive k.
// Few rows of dy stream the weights: 4 x 8192 x 16384 bf16 18.6 us, 3.8 TB/s.  Many are bound by the vector instructions that widen W and split dy
// beside the multiplications: 1024 x 8192 x 4096 bf16 93 us, 740 TFLOP/s, fp32 183 us, 1 130 over its three planes.
struct BwdArgs {
  const void* dy;
  const uint8_t *w, *ws;
  void* dx;
  float* slab;                 // [splits][M][K] when the rows n are split over blocks
  int M, N, K, KB, steps_per_wave, dx_bf16;       // a step is 32 rows of W
};
template <int KW>
struct Words {
  typedef unsigned type __attribute__((ext_vector_type(KW)));
};
template <int MF, int KW, int PL, bool ODD>
__global__ __launch_bounds__(256, 2) void mx4_linear_bwd_kernel(const BwdArgs a, int tk, int tm) {
  typedef typename Words<KW>::type words;
  constexpr int RB = PL == 1 ? 64 : 128;                    // bytes of a dy row in a step
  constexpr bool DMA = MF > 1 && !ODD;
  __shared__ union {
    float tile[4][16][132];
    u32x4 dy[4][DMA ? MF * RB : 1];                                   // [wave]: MF * 16 rows of RB / 16 pieces
  } sh;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, g = lane >> 4;
  const Place pl = place(tk, tm);
  const int k0 = pl.n * 128 * KW, m0 = pl.m * 16 * MF;
  const int blk = min(k0 / 32 + i * KW / 4, a.KB - 1);      // (k past the padded row repeat the last block; their results are not stored)
  const uint8_t* wp = a.w + (size_t)blk * 16 + i * KW % 4 * 4;
  // the scales of a step: lane l holds four of row l % 32 (KW = 2: lanes from 32 on the next four), handed round
  const uint8_t* sp = a.ws + min(k0 / 32 + (lane >> 5) * 4, a.KB - 4);
  const int sl = ((KW == 2 ? (i >> 3) * 32 : 0) + g * 8) * 4, sb = (i * KW / 4 & 3) * 8;
  const uint8_t* drow[MF];
#pragma unroll
  for (int m = 0; m < MF; ++m) drow[m] = (const uint8_t*)a.dy + (size_t)min(m0 + m * 16 + i, a.M - 1) * a.N * (PL == 1 ? 2 : 4);
  const int steps = (a.N + 31) / 32;
  const int s0 = (pl.z * 4 + wave) * a.steps_per_wave, s1 = min(steps, s0 + a.steps_per_wave);         // (a wave may be left without a step)
  // Several fragments of dy go through LDS by DMA, a wave's own rows: neighbouring lanes fetch a row's bytes, where the fragments' order takes an
  // access a lane (512 x 4096 x 4096: bf16 42 -> 36 us, fp32 67 -> 62; one fragment is not worth its waits, 32 rows by 8192 and 16384 33 -> 36).
  // Piece c of row r at c ^ swz_dy(r): no bank conflicts.  Row ends are met by the last step alone, which loads to registers; so do rows of
  // odd length.
  constexpr int PR = RB / 16, DP = DMA ? MF * 16 * RB / 1024 : 1;     // pieces a row; DMA instructions a step
  auto swz_dy = [](int r) { return PR == 4 ? r >> 1 & 3 : (r >> 1 & 1) | ((r >> 2 & 1) * 2 ^ (r >> 3 & 1) * 3) << 1; };
  unsigned dofs[DP];
  const __amdgpu_buffer_rsrc_t rd = __builtin_amdgcn_make_buffer_rsrc((void*)((const uint8_t*)a.dy + (size_t)m0 * a.N * (RB / 32)), 0, -1, 0x00020000);
#pragma unroll
  for (int p = 0; p < DP; ++p) {
    const int r = p * (64 / PR) + lane / PR;
    dofs[p] = (unsigned)min(r, a.M - 1 - m0) * (unsigned)a.N * (RB / 32) + ((lane % PR) ^ swz_dy(r)) * 16;
  }
  const unsigned dbase = (unsigned)(uintptr_t)(lds_void*)&sh.dy[wave][0];
  f32x4 acc[KW][8][MF];
#pragma unroll
  for (int w = 0; w < KW; ++w)
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int m = 0; m < MF; ++m) acc[w][j][m] = f32x4{0.f, 0.f, 0.f, 0.f};
  words wn[8];
  unsigned sn = 0;
  Raw8<PL == 1> xn[MF];
  // ODD: bf16 rows of odd length.  Every second one starts in the middle of a 4-byte word, where a vector load takes twice as long, so its elements
  // are taken from the five words that hold them: 512 x 8193 x 6208 226 -> 151 us (106 with N = 8192).  An instance of its own, for the form of
  // 64 rows only: the shifts would cost the others more than they give (4 rows: 14.7 -> 15.6 us).
  unsigned xw[MF], whole = 0;                               // the fifth word; ~0 but for the last step, whose loads look for the row's end
  auto load = [&](int s) {
    const int nb = s * 32 + g * 8;
    const bool tail = s * 32 + 32 > a.N;
    if (DMA && !tail) {
#pragma unroll
      for (int p = 0; p < DP; ++p) lds_dma<16>(rd, dbase + p * 1024, dofs[p], s * RB);
    }
    if (DMA) asm volatile("" ::: "memory");                 // (W is loaded after dy: once W is there, dy is)
    if (KW == 2 || lane < 32) sn = *(const unsigned*)(sp + (size_t)min(s * 32 + (lane & 31), a.N - 1) * a.KB);
#pragma unroll
    for (int r = 0; r < 8; ++r) wn[r] = *(const words*)(wp + (size_t)min(nb + r, a.N - 1) * a.KB * 16);      // rows past N meet a zero of dy
    if (!DMA || tail) {
#pragma unroll
      for (int m = 0; m < MF; ++m) {
        if constexpr (ODD) {
          xw[m] = 0;
          if (!tail) {
            const unsigned half = (unsigned)(uintptr_t)drow[m] & 2;
            const uint8_t* p = drow[m] + (size_t)nb * 2 - half;
            xn[m].h = *(const bf16x8w*)p;
            xw[m] = *(const unsigned*)(p + 12 + half * 2);  // (never past the word of the last element)
            continue;
          }
        }
        xn[m] = row8<PL == 1>(drow[m], nb, a.N, tail);
      }
    }
    whole = tail ? 0u : ~0u;
  };
  if (s0 < s1) load(s0);
#pragma unroll 1
  for (int s = s0; s < s1; ++s) {
    words wq[8];
    float sc[8];
    bf16x8 xf[MF][PL];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      if constexpr (DMA && KW == 1) asm volatile("" ::"v"(wn[r][0]) : "memory");
      if constexpr (DMA && KW > 1) asm volatile("" ::"v"(wn[r]) : "memory");
      wq[r] = wn[r];
      sc[r] = mx4_step((unsigned)__builtin_amdgcn_ds_bpermute(sl + r * 4, (int)sn) >> sb & 255u);
    }
    if (DMA && whole) {
#pragma unroll
      for (int m = 0; m < MF; ++m) {
        const u32x4* d = &sh.dy[wave][(m * 16 + i) * PR];
        if constexpr (PL == 1) {
          xn[m].h = __builtin_bit_cast(bf16x8, d[g ^ swz_dy(i)]);
        } else {
          xn[m].a = __builtin_bit_cast(f32x4, d[(2 * g) ^ swz_dy(i)]);
          xn[m].b = __builtin_bit_cast(f32x4, d[(2 * g + 1) ^ swz_dy(i)]);
        }
      }
    }
#pragma unroll
    for (int m = 0; m < MF; ++m) {
      split_raw<PL>(xn[m], xf[m]);
      if constexpr (ODD) {
        const unsigned sh = ((unsigned)(uintptr_t)drow[m] & 2) * 8 & whole;
        u32x4 d = __builtin_bit_cast(u32x4, xf[m][0]);
#pragma unroll
        for (int q = 0; q < 4; ++q) d[q] = __builtin_amdgcn_alignbit(q < 3 ? d[q + 1] : xw[m], d[q], sh);
        xf[m][0] = __builtin_bit_cast(bf16x8, d);
      }
    }
    if (DMA) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");        // dy has been read
    if (s + 1 < s1) load(s + 1);
    __builtin_amdgcn_sched_barrier(0);                      // the next step's loads leave before this one is multiplied
#pragma unroll
    for (int w = 0; w < KW; ++w)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        unsigned p[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          bf16x2 t;
          switch (b) {                                      // (the byte number is an immediate)
            case 0: t = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(wq[r][w], sc[r], 0); break;
            case 1: t = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(wq[r][w], sc[r], 1); break;
            case 2: t = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(wq[r][w], sc[r], 2); break;
            default: t = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(wq[r][w], sc[r], 3); break;
          }
          p[r] = __builtin_bit_cast(unsigned, t);
        }
        u32x4 lo, hi;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          lo[r] = __builtin_amdgcn_perm(p[2 * r + 1], p[2 * r], 0x05040100u);
          hi[r] = __builtin_amdgcn_perm(p[2 * r + 1], p[2 * r], 0x07060302u);
        }
        const bf16x8 wl = __builtin_bit_cast(bf16x8, lo), wh = __builtin_bit_cast(bf16x8, hi);
#pragma unroll
        for (int q = PL - 1; q >= 0; --q)
#pragma unroll
          for (int m = 0; m < MF; ++m) {
            acc[w][2 * b][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wl, xf[m][q], acc[w][2 * b][m], 0, 0, 0);
            acc[w][2 * b + 1][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wh, xf[m][q], acc[w][2 * b + 1][m], 0, 0, 0);
          }
      }
  }
#pragma unroll
  for (int m = 0; m < MF; ++m)
#pragma unroll
    for (int w = 0; w < KW; ++w) {
      __syncthreads();                                      // (before the first: the tiles lie where dy lay)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const f32x4 lo = {acc[w][0][m][r], acc[w][1][m][r], acc[w][2][m][r], acc[w][3][m][r]},
                    hi = {acc[w][4][m][r], acc[w][5][m][r], acc[w][6][m][r], acc[w][7][m][r]};
        *(f32x4*)&sh.tile[wave][i][8 * (g * 4 + r)] = lo;
        *(f32x4*)&sh.tile[wave][i][8 * (g * 4 + r) + 4] = hi;
      }
      __syncthreads();
      const int mm = threadIdx.x >> 4, kk = threadIdx.x & 15, row = m0 + m * 16 + mm, k = k0 + (kk * KW + w) * 8;
      if (row >= a.M || k >= a.K) continue;
      float v[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] = (sh.tile[0][mm][kk * 8 + q] + sh.tile[1][mm][kk * 8 + q]) + (sh.tile[2][mm][kk * 8 + q] + sh.tile[3][mm][kk * 8 + q]);
      const size_t o = ((size_t)(a.slab ? pl.z : 0) * a.M + row) * a.K + k;
      if (a.slab || !a.dx_bf16) {
        float* d = a.slab ? a.slab : (float*)a.dx;
        if (k + 8 <= a.K) {
          const f32x4 lo = {v[0], v[1], v[2], v[3]}, hi = {v[4], v[5], v[6], v[7]};
          *(f32x4u*)(d + o) = lo;
          *(f32x4u*)(d + o + 4) = hi;
        } else {
          for (int q = 0; q < 8 && k + q < a.K; ++q) d[o + q] = v[q];
        }
      } else {
        bf16x8 h;
#pragma unroll
        for (int q = 0; q < 8; ++q) h[q] = (__bf16)v[q];
        if (k + 8 <= a.K) {
          *(bf16x8u*)((__bf16*)a.dx + o) = h;
        } else {
          for (int q = 0; q < 8 && k + q < a.K; ++q) ((__bf16*)a.dx)[o + q] = h[q];
        }
      }
    }
}

static inline bool aligned(const void* p, unsigned a) { return ((uintptr_t)p & (a - 1)) == 0; }
static inline int kb_of(int cols) { return 4 * cdiv(cols, 128); }
constexpr long long MAX_COLS = 0x7fffff80;      // of a row: its padded length is an int

// a launch has fewer than 2^32 threads along x
static inline bool grid_ok(size_t blocks, unsigned threads) { return blocks * threads <= 0xffffffffull; }

struct SlabGrid {
  bool vec, deep;                // 4 outputs a group; 8 lanes a group, which pay for themselves from 8 splits on
  size_t blocks;
};
static SlabGrid slab_grid(int splits, int M, int N, const void* out, int out_bf16) {
  SlabGrid g;
  g.vec = N % 4 == 0 && aligned(out, out_bf16 ? 8 : 16);
  g.deep = splits >= 8;
  g.blocks = cdivz((size_t)M * N, (g.vec ? 4 : 1) * (g.deep ? 32 : 256));
  return g;
}
static int slab_reduce(const float* slab, int splits, int M, int N, const float* bias, void* out, int act, float slope, int out_bf16,
                       hipStream_t st) {
  const size_t total = (size_t)M * N;
  const SlabGrid g = slab_grid(splits, M, N, out, out_bf16);      // (grid_ok: the entry points look before they launch the product)
  const bool vec = g.vec, deep = g.deep;
  auto k = vec ? (deep ? mx4_slab_reduce_kernel<4, 8> : mx4_slab_reduce_kernel<4, 1>) : (deep ? mx4_slab_reduce_kernel<1, 8> : mx4_slab_reduce_kernel<1, 1>);
  hipLaunchKernelGGL(k, dim3((unsigned)g.blocks), dim3(256), 0, st, slab, splits, total, N, bias, out, act, slope, out_bf16);
  IPR_LAUNCH_CHECK();
  return 0;
}

template <int TN, int TM, int WN, int WM, bool S16>
static int gemm4_go(const LinArgs& a, int tn, int tm, int splits, hipStream_t st) {
  constexpr int LDS = (TN + TM) * (S16 ? 2 * 128 + 2 * 16 : 2 * 136);
  auto k = mx4_gemm4_kernel<TN, TM, WN, WM, S16>;
  static std::atomic<unsigned long long> ready{0};           // one bit a device: more than 64 KB of dynamic LDS has to be allowed once
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e == hipSuccess && (dev >= 64 || !(ready.load() >> dev & 1))) {
    e = hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
    if (e == hipSuccess && dev < 64) ready.fetch_or(1ull << dev);
  }
  IPR_CHECK(e == hipSuccess, "mx4_linear: %d bytes of LDS: %s", LDS, hipGetErrorString(e));
  const unsigned total = (unsigned)tn * tm, resident = TN == 256 ? 256 : 512;       // blocks the chip holds at once
  hipLaunchKernelGGL(k, dim3(total < resident ? total : resident, 1, splits), dim3(WN * WM * 64), LDS, st, a, tn, tm);
  IPR_LAUNCH_CHECK();
  return 0;
}

// How the products are cut.  A form of a kernel is a tile and what a step along the reduction costs: `step` us for one block a CU (by x: fp32,
// bf16), `more` of that for each further block beside it, of at most `resident`.  Every form is tried with every split of the reduction: the
// steps in a row, overlapped with the weights at 4 TB/s, read `again` times for each further row of tiles, plus a second launch and the slabs'
// traffic (8 bytes a partial result at 4 TB/s) where it is split.  Fitted to sweeps of 140 sizes over all forms and 1 to 48 splits: within 10 % of the fastest
// in nine of ten, at worst 25 % (few blocks on an idle chip step faster than the estimate knows).  The largest form only where it fills the
// chip twice: one block of it alone on a CU waits for its own loads.
struct Form {
  int mf, nf;                    // 16-row fragments of x, fragments (kernels above) or words (gradient) of the weights
  int resident[2];
  double step[2], more[2];
};
struct Cut {
  int form, tm, tn, splits, steps_per_split;
  double us;
};
static Cut cut(const Form* forms, int count, int kind, int rows_f, int cols_f, int M, int N, int steps, int unit, double weights, double again) {
  Cut best;
  memset(&best, 0, sizeof(best));
  best.us = 1e30;
  for (int f = 0; f < count; ++f) {
    const Form& q = forms[f];
    const int tm = cdiv(M, rows_f * q.mf), tn = cdiv(N, cols_f * q.nf), R = q.resident[kind];
    const double read = weights * (1 + again * (tm - 1)) / 4e6;
    if (q.mf > 1 && rows_f * q.mf >= 2 * M) continue;       // half the tile's rows or more would be empty
    for (int want = 1; want <= 64 && want <= steps; want = want < 8 ? want + 1 : want + want / 4) {
      const int per = rup(cdiv(steps, want), unit), splits = cdiv(steps, per);
      const double blocks = (double)tm * tn * splits;
      if (q.mf * q.nf == 16 && blocks < 512.) continue;
      if (want > 1 && blocks > 256. * 3 * R) break;         // the chip is full three times over: no further split shortens anything
      const double b = (double)((long long)((blocks + 255) / 256)), full = (double)((long long)(b / R)), rem = b - full * R;
      const double row = full * (1 + q.more[kind] * (R - 1)) + (rem > 0 ? 1 + q.more[kind] * (rem - 1) : 0.);
      double us = per * q.step[kind] * row;
      us = sqrt(us * us + read * read);
      if (splits > 1) us += 5. + splits * (double)M * N * 2e-6;
      if (us < best.us) best = Cut{f, tm, tn, splits, per, us};
    }
  }
  return best;
}

//   LDS    : 16 * mf rows x 64 * nf columns a block.  Four fragments a wave halve the LDS reads a multiplication (4096^3 fp32: 450 -> 400 us)
//   direct : 16 * mf rows x 16 * nf * (8 / wk) columns a block, wk waves along K.  For 4-bit x of up to 64 rows; else for up to 16, where the LDS form
//            would be split or leaves half the chip idle and the estimate is 2 us lower, K <= 4096 and not too many columns.  Against LDS, device
//            time, M x N x K: 8 x 1024 x 1024 fp32 4.3 : 6.4 us, bf16 3.4 : 4.2; 1 x 4096 x 4096 bf16 4.8 : 6.7, fp32 8.7 : 7.9 (one launch less
//            for the host); outside the rule 4 x 2000 x 300 fp32 6.6 : 4.4, 16 x 1024 x 18432 bf16 23.5 : 8.1 (18 steps in a row),
//            4 x 65536 x 1024 bf16 16.5 : 8.1, 8 x 16384 x 4096 fp32 23.2 : 21.5 (every wave splits x again).  Two fragments of bf16 x: no size.
//   tile   : 4-bit x of more rows: square tiles, 256 where they fill three quarters of the chip, else 128
struct LinPlan {
  int mf, nf, wk, tile, s16, tm, tn, splits, steps_per_split;
};
static LinPlan lin_plan(int M, int N, int K, int x_kind) {
  static const Form lds[4] = {{1, 1, {8, 8}, {0.46, 0.28}, {0.65, 0.4}}, {2, 2, {4, 4}, {1.1, 0.5}, {0.65, 0.6}}, {4, 2, {3, 3}, {2.1, 0.75}, {0.45, 0.55}}, {4, 4, {2, 2}, {3.6, 1.5}, {0.35, 0.3}}};
  static const Form direct = {1, 1, {2, 2}, {0.6, 0.35}, {0.2, 0.2}}, tile = {1, 1, {1, 2}, {1.1, 0.4}, {0., 0.2}};      // (tile: by size, 256 or 128)
  LinPlan p;
  memset(&p, 0, sizeof(p));
  const int steps = kb_of(K) / 4, kind = x_kind != IPRGAN_X_F32;
  const double weights = (double)N * K * 0.53;
  Cut c, d;
  bool dir = x_kind == IPRGAN_X_MX4 && M <= 64;
  if (M <= 64) {
    p.wk = 1;
    while (p.wk < 8 && p.wk * 2 <= steps) p.wk *= 2;
    p.mf = M <= 16 ? 1 : M <= 32 ? 2 : 4;
    p.nf = N >= 256 * 32 * (8 / p.wk) ? 2 : 1;              // two fragments a wave once that leaves a block for every CU
    Form f = direct;
    f.step[kind] /= p.wk;
    d = cut(&f, 1, kind, 16 * p.mf, 16 * p.nf * (8 / p.wk), M, N, steps, p.wk, weights, 1.);
  }
  if (x_kind != IPRGAN_X_MX4) {
    c = cut(lds, 4, kind, 16, 64, M, N, steps, 1, weights, 1.);
    dir = M <= 16 && (kind == 0 || p.nf == 1) && (c.splits > 1 || c.tn < 128) && d.us + 2. < c.us && steps <= 32 && (long long)steps * N <= (kind ? 600000 : 200000);
  }
  if (dir) {
    c = d;
  } else if (x_kind != IPRGAN_X_MX4) {
    p.wk = 0;
    p.mf = lds[c.form].mf;
    p.nf = lds[c.form].nf;
  } else {
    p.wk = 0;
    p.tile = (long long)cdiv(M, 256) * cdiv(N, 256) >= 192 ? 256 : 128;
    p.s16 = steps % 4 == 0;                                 // the form that moves the scales of four stages at once
    c = cut(&tile, 1, p.tile == 128, p.tile, p.tile, M, N, steps, p.s16 ? 4 : 2, weights, 1.);
  }
  p.tm = c.tm;
  p.tn = c.tn;
  p.splits = c.splits;
  p.steps_per_split = c.steps_per_split;
  return p;
}

// The gradient's reduction runs along N, 4 waves a block, a step is 32 rows of W a wave.  More words a lane make wider reads of W and share the
// planes of dy; more rows of dy share the widened W.  1024 x 4096 x 4096: fp32 137 us with (2, 1), 99 with (2, 2); bf16 81, and 57 with (4, 1).
struct BwdPlan {
  int form, tm, tk, splits, steps_per_split;
};
static const Form* bwd_forms(int dy_bf16) {
  static const Form f32[3] = {{1, 1, {4, 4}, {0.82, 0.82}, {0.75, 0.75}}, {1, 2, {2, 2}, {1.03, 1.03}, {0.85, 0.85}}, {2, 2, {2, 2}, {1.75, 1.75}, {0.5, 0.5}}};
  static const Form b16[3] = {{1, 1, {4, 4}, {0.68, 0.72}, {0.75, 0.75}}, {1, 2, {3, 3}, {0.72, 0.8}, {0.85, 0.85}}, {4, 1, {2, 2}, {1.08, 1.75}, {0.33, 0.33}}};
  return dy_bf16 ? b16 : f32;
}
static BwdPlan bwd_plan(int M, int N, int K, int dy_bf16) {
  const Cut c = cut(bwd_forms(dy_bf16), 3, dy_bf16 ? N & 1 : 0, 16, 128, M, K, cdiv(cdiv(N, 32), 4), 1, (double)N * K * 0.53, 0.4);      // (bf16: rows of even, odd length)
  return BwdPlan{c.form, c.tm, c.tn, c.splits, c.steps_per_split};
}

}  // namespace iprgan

using namespace iprgan;

extern "C" {

int iprgan_mx4_pitch(long long cols) { return cols > 0 && cols <= MAX_COLS ? kb_of((int)cols) : 0; }

static int mx4_rows_check(const char* who, long long rows, long long cols, unsigned* groups) {
  IPR_CHECK(rows > 0 && cols > 0, "%s: empty input (%lld rows of %lld)", who, rows, cols);
  const size_t g = rows < 0x7fff0000ll && cols <= MAX_COLS ? (size_t)rows * cdivz((size_t)cols, 128) * 16 : ~(size_t)0;
  IPR_CHECK(g < 0x7fff0000ull, "%s: %lld rows of %lld are too many elements", who, rows, cols);
  *groups = (unsigned)g;
  return 0;
}

int iprgan_mx4_quant(const void* x, void* codes, void* scales, long long rows, long long cols, int x_bf16, void* stream) {
  unsigned groups;
  if (mx4_rows_check("mx4_quant", rows, cols, &groups)) return 1;
  IPR_CHECK(x && codes && scales, "mx4_quant: null operand");
  IPR_CHECK(x_bf16 == 0 || x_bf16 == 1, "mx4_quant: storage kind %d (fp32 or bf16)", x_bf16);
  IPR_CHECK(aligned(codes, 16) && aligned(scales, 4) && aligned(x, x_bf16 ? 2 : 4), "mx4_quant: codes must be 16-byte, scales 4-byte aligned");
  auto k = x_bf16 ? mx4_quant_kernel<true> : mx4_quant_kernel<false>;
  const unsigned blocks = (groups + 255) / 256;
  hipLaunchKernelGGL(k, dim3(blocks < 8192 ? blocks : 8192), dim3(256), 0, (hipStream_t)stream, x, (unsigned*)codes, (uint8_t*)scales,
                     groups, (int)cols, make_fastdiv((uint32_t)kb_of((int)cols) * 4));
  IPR_LAUNCH_CHECK();
  return 0;
}

int iprgan_mx4_dequant(const void* codes, const void* scales, void* y, long long rows, long long cols, int y_bf16, void* stream) {
  unsigned groups;
  if (mx4_rows_check("mx4_dequant", rows, cols, &groups)) return 1;
  IPR_CHECK(y && codes && scales, "mx4_dequant: null operand");
  IPR_CHECK(y_bf16 == 0 || y_bf16 == 1, "mx4_dequant: storage kind %d (fp32 or bf16)", y_bf16);
  IPR_CHECK(aligned(codes, 16) && aligned(scales, 4) && aligned(y, y_bf16 ? 2 : 4), "mx4_dequant: codes must be 16-byte, scales 4-byte aligned");
  auto k = y_bf16 ? mx4_dequant_kernel<true> : mx4_dequant_kernel<false>;
  const unsigned blocks = (groups + 255) / 256;
  hipLaunchKernelGGL(k, dim3(blocks < 8192 ? blocks : 8192), dim3(256), 0, (hipStream_t)stream, (const unsigned*)codes,
                     (const uint8_t*)scales, y, groups, (int)cols, make_fastdiv((uint32_t)kb_of((int)cols) * 4));
  IPR_LAUNCH_CHECK();
  return 0;
}

static bool lin_sizes_ok(long long M, long long N, long long K) {
  return M > 0 && N > 0 && K > 0 && M < (1 << 30) && N < (1 << 24) && K < (1 << 24);      // M: 2 M and every tile's rows are ints
}
static int lin_check(const char* who, long long M, long long N, long long K) {
  IPR_CHECK(M > 0 && N > 0 && K > 0, "%s: empty product (M=%lld, N=%lld, K=%lld)", who, M, N, K);
  IPR_CHECK(lin_sizes_ok(M, N, K), "%s: M=%lld, N=%lld, K=%lld (M below 2^30, N and K below 2^24)", who, M, N, K);
  return 0;
}

// tanh and the sigmoid are applied by the pass that adds the slabs, also where there is only one
static bool lin_slab(const LinPlan& p, int act) { return p.splits > 1 || act > IPRGAN_ACT_LRELU; }

size_t iprgan_mx4_linear_ws_floats(long long M, long long N, long long K, int x_kind, int act) {
  if (!lin_sizes_ok(M, N, K)) return 0;
  const LinPlan p = lin_plan((int)M, (int)N, (int)K, x_kind);
  return lin_slab(p, act) ? (size_t)p.splits * M * N : 0;
}

int iprgan_mx4_linear(const void* x, const void* x_scales, const void* w_codes, const void* w_scales, const float* bias, void* y,
                      float* ws, long long rows, long long outs, long long ins, int x_kind, int act, float slope, int y_bf16, void* stream) {
  if (lin_check("mx4_linear", rows, outs, ins)) return 1;
  const int M = (int)rows, N = (int)outs, K = (int)ins;
  IPR_CHECK(x_kind == IPRGAN_X_F32 || x_kind == IPRGAN_X_BF16 || x_kind == IPRGAN_X_MX4, "mx4_linear: kind %d of x", x_kind);
  IPR_CHECK(x && w_codes && w_scales && y && (x_kind != IPRGAN_X_MX4 || x_scales), "mx4_linear: null operand");
  IPR_CHECK(y_bf16 == 0 || y_bf16 == 1, "mx4_linear: storage kind %d of y (fp32 or bf16)", y_bf16);
  IPR_CHECK(act >= IPRGAN_ACT_NONE && act <= IPRGAN_ACT_SIGMOID_PM1, "mx4_linear: activation %d", act);
  IPR_CHECK(aligned(w_codes, 16) && aligned(w_scales, 4) && aligned(x, x_kind == IPRGAN_X_MX4 ? 16 : x_kind == IPRGAN_X_BF16 ? 2 : 4) &&
                (x_kind != IPRGAN_X_MX4 || aligned(x_scales, 4)) && aligned(y, y_bf16 ? 2 : 4),
            "mx4_linear: codes must be 16-byte, scales 4-byte aligned");
  const LinPlan p = lin_plan(M, N, K, x_kind);
  const bool slab = lin_slab(p, act);
  IPR_CHECK(p.tile || grid_ok((size_t)p.tm * p.tn * p.splits, p.wk ? 512 : 256), "mx4_linear: M=%d, N=%d are too many tiles for a launch", M, N);
  IPR_CHECK((long long)p.tm * p.tn < 0x7fffffffll && (!slab || grid_ok(slab_grid(p.splits, M, N, y, y_bf16).blocks, 256)),
            "mx4_linear: M=%d, N=%d are too many results", M, N);
  IPR_CHECK(!slab || (ws && aligned(ws, 16)), "mx4_linear: the workspace of iprgan_mx4_linear_ws_floats is missing");
  hipStream_t st = (hipStream_t)stream;
  LinArgs a;
  a.x = x; a.xs = (const uint8_t*)x_scales; a.w = (const uint8_t*)w_codes; a.ws = (const uint8_t*)w_scales; a.bias = bias; a.y = y;
  a.slab = slab ? ws : nullptr;
  a.M = M; a.N = N; a.K = K; a.KB = kb_of(K); a.steps_per_split = p.steps_per_split;
  a.act = act; a.slope = act == IPRGAN_ACT_LRELU ? slope : 1.f; a.y_bf16 = y_bf16;
  a.vec8 = y_bf16 && N % 8 == 0 && aligned(y, 16);
  const dim3 grid((unsigned)p.tn * p.tm * p.splits);
  if (p.tile) {
    const int rc = p.tile == 256 ? (p.s16 ? gemm4_go<256, 256, 2, 4, true>(a, p.tn, p.tm, p.splits, st) : gemm4_go<256, 256, 2, 4, false>(a, p.tn, p.tm, p.splits, st))
                                 : (p.s16 ? gemm4_go<128, 128, 2, 2, true>(a, p.tn, p.tm, p.splits, st) : gemm4_go<128, 128, 2, 2, false>(a, p.tn, p.tm, p.splits, st));
    if (rc) return rc;
  } else if (p.wk) {
#define DIRECT(MF, XT) (p.nf == 2 ? mx4_direct_kernel<MF, 2, XT> : mx4_direct_kernel<MF, 1, XT>)
    auto k = x_kind == IPRGAN_X_F32 ? DIRECT(1, 3) : x_kind == IPRGAN_X_BF16 ? mx4_direct_kernel<1, 1, 1> : p.mf == 1 ? DIRECT(1, 0) : p.mf == 2 ? DIRECT(2, 0) : DIRECT(4, 0);
#undef DIRECT
    hipLaunchKernelGGL(k, grid, dim3(512), 0, st, a, p.tn, p.tm, p.wk);
  } else {
#define LDSX(PL) (p.mf == 1 ? mx4_linear_kernel<1, 1, PL> : p.mf == 2 ? mx4_linear_kernel<2, 2, PL> : p.nf == 2 ? mx4_linear_kernel<4, 2, PL> : mx4_linear_kernel<4, 4, PL>)
    auto k = x_kind == IPRGAN_X_BF16 ? LDSX(1) : LDSX(3);
#undef LDSX
    hipLaunchKernelGGL(k, grid, dim3(256), 0, st, a, p.tn, p.tm);
  }
  IPR_LAUNCH_CHECK();
  return slab ? slab_reduce(ws, p.splits, M, N, bias, y, act, slope, y_bf16, st) : 0;
}

int iprgan_mx4_form(long long M, long long N, long long K, int x_kind, int gradient, int* form) {
  if (lin_check("mx4_form", M, N, K)) return 1;
  IPR_CHECK(form && x_kind >= IPRGAN_X_F32 && x_kind <= (gradient ? IPRGAN_X_BF16 : IPRGAN_X_MX4), "mx4_form: kind %d", x_kind);
  if (gradient) {
    const BwdPlan p = bwd_plan((int)M, (int)N, (int)K, x_kind);
    const Form& f = bwd_forms(x_kind)[p.form];
    const int v[5] = {3, 16 * f.mf, 128 * f.nf, x_kind && f.mf == 4 && (N & 1), p.splits};
    memcpy(form, v, sizeof(v));
  } else {
    const LinPlan p = lin_plan((int)M, (int)N, (int)K, x_kind);
    const int v[5] = {p.tile ? 2 : p.wk ? 1 : 0, p.tile ? p.tile : 16 * p.mf, p.tile ? p.tile : 16 * p.nf * (p.wk ? 8 / p.wk : 4), p.tile ? p.s16 : p.wk, p.splits};
    memcpy(form, v, sizeof(v));
  }
  return 0;
}

size_t iprgan_mx4_linear_bwd_ws_floats(long long M, long long N, long long K, int dy_bf16) {
  if (!lin_sizes_ok(M, N, K)) return 0;
  const BwdPlan p = bwd_plan((int)M, (int)N, (int)K, dy_bf16);
  return p.splits > 1 ? (size_t)p.splits * M * K : 0;
}

int iprgan_mx4_linear_bwd(const void* dy, const void* w_codes, const void* w_scales, void* dx, float* ws, long long rows, long long outs,
                          long long ins, int dy_bf16, int dx_bf16, void* stream) {
  if (lin_check("mx4_linear_bwd", rows, outs, ins)) return 1;
  const int M = (int)rows, N = (int)outs, K = (int)ins;
  IPR_CHECK(dy && w_codes && w_scales && dx, "mx4_linear_bwd: null operand");
  IPR_CHECK((dy_bf16 == 0 || dy_bf16 == 1) && (dx_bf16 == 0 || dx_bf16 == 1), "mx4_linear_bwd: storage kinds %d, %d (fp32 or bf16)", dy_bf16, dx_bf16);
  IPR_CHECK(aligned(w_codes, 16) && aligned(w_scales, 4) && aligned(dy, dy_bf16 ? 2 : 4) && aligned(dx, dx_bf16 ? 2 : 4),
            "mx4_linear_bwd: codes must be 16-byte, scales 4-byte aligned");
  const BwdPlan p = bwd_plan(M, N, K, dy_bf16);
  IPR_CHECK(grid_ok((size_t)p.tm * p.tk * p.splits, 256) && (p.splits == 1 || grid_ok(slab_grid(p.splits, M, K, dx, dx_bf16).blocks, 256)),
            "mx4_linear_bwd: M=%d, K=%d are too many tiles for a launch", M, K);
  IPR_CHECK(p.splits == 1 || (ws && aligned(ws, 16)), "mx4_linear_bwd: the workspace of iprgan_mx4_linear_bwd_ws_floats is missing");
  hipStream_t st = (hipStream_t)stream;
  BwdArgs a;
  a.dy = dy; a.w = (const uint8_t*)w_codes; a.ws = (const uint8_t*)w_scales; a.dx = dx;
  a.slab = p.splits > 1 ? ws : nullptr;
  a.M = M; a.N = N; a.K = K; a.KB = kb_of(K); a.steps_per_wave = p.steps_per_split; a.dx_bf16 = dx_bf16;
  const dim3 grid((unsigned)p.tk * p.tm * p.splits), blk(256);
  const bool odd = ((unsigned)(uintptr_t)dy | (unsigned)N * 2) & 2;
  auto k = !dy_bf16 ? (p.form == 0 ? mx4_linear_bwd_kernel<1, 1, 3, false> : p.form == 1 ? mx4_linear_bwd_kernel<1, 2, 3, false> : mx4_linear_bwd_kernel<2, 2, 3, false>)
                    : (p.form == 0 ? mx4_linear_bwd_kernel<1, 1, 1, false> : p.form == 1 ? mx4_linear_bwd_kernel<1, 2, 1, false>
                       : odd ? mx4_linear_bwd_kernel<4, 1, 1, true> : mx4_linear_bwd_kernel<4, 1, 1, false>);
  hipLaunchKernelGGL(k, grid, blk, 0, st, a, p.tk, p.tm);
  IPR_LAUNCH_CHECK();
  return p.splits > 1 ? slab_reduce(ws, p.splits, M, K, nullptr, dx, IPRGAN_ACT_NONE, 0.f, dx_bf16, st) : 0;
}

}  // extern "C"
