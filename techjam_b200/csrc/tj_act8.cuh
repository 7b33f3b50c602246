// 8-bit activations: e4m3 codes with one power-of-two scale (e8m0) for each
// run of 128 columns, and the memory-bound kernels on them (pack, restore,
// weight pack, GELU's gradient).
//
// Of a block's finite values let a be the largest magnitude.  The scale is
// the smallest 2^e, e >= -127, with a <= 448 * 2^e (448: e4m3's largest
// value), 2^0 for a block of zeros, and code = e4m3(x * 2^-e), rounded to
// nearest even.  The product x * 2^-e is exact (or far below half of e4m3's
// smallest step), so a code depends on its block alone and is the same bit
// for bit wherever the packing runs.  Infinities and NaN become the NaN code
// and leave their neighbours' scale alone.  A power of two also keeps
// code * 2^e exact in 32 bits and in bf16, and is what the tensor cores'
// block-scaled products take.
//
// All kernels here move bytes once and are bound by HBM; a 128-column block
// belongs to 8 lanes, so its maximum takes three shuffles, and the lanes'
// 4-element pieces interleave so that every load and store of a warp covers
// whole 32-byte sectors.
#pragma once
#include <cuda_bf16.h>

#include <type_traits>

#include "tj_common.cuh"

namespace tj {

constexpr int kBlk = 128;  // columns (and, for weights, rows) that share a scale

enum Dtype : int { kF32 = 0, kF16 = 1, kBF16 = 2, kE4M3 = 3 };

TJ_DEV int n_blocks(int cols) { return (cols + kBlk - 1) / kBlk; }

// Biased exponent byte of the block scale for largest finite magnitude amax.
// amax = 1.m * 2^(E-127); 448 = 1.75 * 2^8.
TJ_DEV uint32_t scale_byte(float amax) {
  const uint32_t u = __float_as_uint(amax);
  if (u == 0u) return 127u;
  const int b = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return (uint32_t)max(b, 0);
}
// 2^(127 - byte) for a byte that scale_byte gives (0..247): always normal.
TJ_DEV float scale_inv(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }
// 2^(byte - 127); 255 is NaN.
TJ_DEV float scale_value(uint32_t byte) {
  return __uint_as_float(byte == 0u ? 0x400000u : (byte == 255u ? 0x7fffffffu : byte << 23));
}
TJ_DEV float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : 0.f;
}
// Codes of (a, b), a in the low byte.  The conversion saturates an infinity;
// CAREFUL makes it the NaN code (x * 0 is NaN then).
template <bool CAREFUL>
TJ_DEV uint32_t e4m3x2(float a, float b, float inv) {
  uint16_t r;
  const float ya = CAREFUL ? fmaf(a, inv, a * 0.f) : a * inv, yb = CAREFUL ? fmaf(b, inv, b * 0.f) : b * inv;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(yb), "f"(ya));
  return r;
}
// Codes of four values that are no infinities, in one word.
TJ_DEV uint32_t e4m3_word(float a, float b, float c, float d) {
  uint32_t r;
  asm("{\n\t.reg .b16 l, h;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n\t"
      "mov.b32 %0, {l, h};\n\t}"
      : "=r"(r)
      : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}
template <bool CAREFUL>
TJ_DEV uint32_t e4m3x4(const float (&v)[4], float inv) {
  if constexpr (CAREFUL) return e4m3x2<true>(v[0], v[1], inv) | (e4m3x2<true>(v[2], v[3], inv) << 16);
  return e4m3_word(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
}
TJ_DEV void e4m3x4_value(uint32_t codes, float scale, float (&v)[4]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t f16;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(f16) : "h"((uint16_t)(codes >> (16 * h))));
    const float2 f = __half22float2(*reinterpret_cast<__half2*>(&f16));
    v[2 * h] = f.x * scale;
    v[2 * h + 1] = f.y * scale;
  }
}

// A lane's share of a 128-column block at column c0: four pieces of four
// elements.  VEC: piece j is columns 4 (sub + 8 j)..+3, one load (rows
// aligned, widths a multiple of 4).  Otherwise element e of piece j is column
// sub + 8 (4 j + e), so that the lanes' single-element accesses still lie
// side by side.  Elements past cols read as zero and are not written.
template <bool VEC>
TJ_DEV int piece_col(int c0, int sub, int j, int e) {
  return VEC ? c0 + 4 * (sub + 8 * j) + e : c0 + sub + 8 * (4 * j + e);
}
template <typename T>
TJ_DEV float to_f32(T v);
template <>
TJ_DEV float to_f32<float>(float v) { return v; }
template <>
TJ_DEV float to_f32<__half>(__half v) { return __half2float(v); }
template <>
TJ_DEV float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

// Rounded to nearest even.
template <typename T>
TJ_DEV T from_f32(float v);
template <>
TJ_DEV float from_f32<float>(float v) { return v; }
template <>
TJ_DEV __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
TJ_DEV __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
// A restored value: no infinity has a code, and one beyond T's range (a
// rounded-up maximum: 65504 becomes 65536 in 8 bits) is T's largest.
template <typename T>
TJ_DEV T from_f32_restored(float v) {
  constexpr float kMax = std::is_same_v<T, __half> ? 65504.f : (sizeof(T) == 2 ? 3.3895313892515355e38f : 3.402823466e38f);
  if (fabsf(v) > kMax) v = copysignf(kMax, v);
  return from_f32<T>(v);
}

template <typename T, bool VEC>
TJ_DEV void load4(const T* row, int c0, int sub, int j, int cols, float (&v)[4]) {
  if constexpr (VEC) {
    const int c = piece_col<true>(c0, sub, j, 0);
    if (c < cols) {
      if constexpr (sizeof(T) == 4) {
        const float4 f = *reinterpret_cast<const float4*>(row + c);
        v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
      } else {
        const uint2 u = *reinterpret_cast<const uint2*>(row + c);
        const T* t = reinterpret_cast<const T*>(&u);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = to_f32<T>(t[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = 0.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = piece_col<false>(c0, sub, j, i);
      v[i] = c < cols ? to_f32<T>(row[c]) : 0.f;
    }
  }
}
template <typename T, bool VEC>
TJ_DEV void store4(T* row, int c0, int sub, int j, int cols, const T (&v)[4]) {
  if constexpr (VEC) {
    const int c = piece_col<true>(c0, sub, j, 0);
    if (c < cols) {
      if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(row + c) = make_float4(v[0], v[1], v[2], v[3]);
      } else {
        uint2 u;
        T* t = reinterpret_cast<T*>(&u);
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i] = v[i];
        *reinterpret_cast<uint2*>(row + c) = u;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = piece_col<false>(c0, sub, j, i);
      if (c < cols) row[c] = v[i];
    }
  }
}
template <bool VEC>
TJ_DEV uint32_t load_codes4(const uint8_t* row, int c0, int sub, int j, int cols) {
  if constexpr (VEC) {
    const int c = piece_col<true>(c0, sub, j, 0);
    return c < cols ? *reinterpret_cast<const uint32_t*>(row + c) : 0u;
  }
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = piece_col<false>(c0, sub, j, i);
    if (c < cols) w |= (uint32_t)row[c] << (8 * i);
  }
  return w;
}
template <bool VEC>
TJ_DEV void store_codes4(uint8_t* row, int c0, int sub, int j, int cols, uint32_t w) {
  if constexpr (VEC) {
    const int c = piece_col<true>(c0, sub, j, 0);
    if (c < cols) *reinterpret_cast<uint32_t*>(row + c) = w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = piece_col<false>(c0, sub, j, i);
      if (c < cols) row[c] = (uint8_t)(w >> (8 * i));
    }
  }
}

TJ_DEV float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Largest over the 8 lanes that share a block.
TJ_DEV float max8(float v) {
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// The 16 values of this lane (its share of the block at column c0) into codes, and the block's scale.  Called by whole warps.
// The maximum drops a NaN but not an infinity: only a warp that meets one
// takes the finite values' maximum and the careful conversion.
template <bool VEC>
TJ_DEV void pack_block(const float (&v)[4][4], int c0, int cols, uint8_t* codes_row, uint8_t* scale, int sub,
                       bool live) {
  float amax = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    amax = max3f(amax, fmaxf(fabsf(v[j][0]), fabsf(v[j][1])), fmaxf(fabsf(v[j][2]), fabsf(v[j][3])));
  amax = max8(amax);
  const bool careful = __any_sync(0xffffffffu, amax > 3.402823466e38f);
  if (careful) {
    amax = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) amax = fmaxf(amax, finite_abs(v[j][i]));
    amax = max8(amax);
  }
  const uint32_t byte = scale_byte(amax);
  if (!live) return;
  const float inv = scale_inv(byte);
  if (careful) {
#pragma unroll
    for (int j = 0; j < 4; ++j) store_codes4<VEC>(codes_row, c0, sub, j, cols, e4m3x4<true>(v[j], inv));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) store_codes4<VEC>(codes_row, c0, sub, j, cols, e4m3x4<false>(v[j], inv));
  }
  if (sub == 0) *scale = (uint8_t)byte;
}

// Block of this group of 8 lanes: four neighbouring blocks to a warp.
struct BlockAt {
  long long row;
  int blk, c0;
  bool live;
};
TJ_DEV BlockAt block_at(long long rows, int cols) {
  const int nb = n_blocks(cols);
  const long long g = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 3;
  BlockAt b;
  b.live = g < rows * nb;
  b.row = b.live ? g / nb : 0;
  b.blk = b.live ? (int)(g - b.row * nb) : 0;
  b.c0 = b.blk * kBlk;
  return b;
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) act8_pack_kernel(const T* __restrict__ x, long long rows, int cols,
                                                        const uint8_t* __restrict__ mask,
                                                        uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  const BlockAt b = block_at(rows, cols);
  const int sub = threadIdx.x & 7;
  const bool valid = b.live && (mask == nullptr || mask[b.row] != 0);
  float v[4][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) load4<T, VEC>(x + b.row * cols, b.c0, sub, j, valid ? cols : 0, v[j]);
  pack_block<VEC>(v, b.c0, cols, codes + b.row * cols, scales + b.row * n_blocks(cols) + b.blk, sub, b.live);
}

// (Pieces of 8 or 16 codes a lane, for wider stores, and two or four blocks a
// lane measured the same or slower, 20-23 us for 33.5M codes to bf16: two
// thirds of the traffic are writes.)
template <typename T, bool VEC>
TJ_DEV void act8_unpack(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, long long rows, int cols,
                        const uint8_t* __restrict__ mask, T* __restrict__ out) {
  const BlockAt b = block_at(rows, cols);
  const int sub = threadIdx.x & 7;
  if (!b.live) return;
  const bool valid = mask == nullptr || mask[b.row] != 0;
  const float s = valid ? scale_value(scales[b.row * n_blocks(cols) + b.blk]) : 0.f;
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = load_codes4<VEC>(codes + b.row * cols, b.c0, sub, j, valid ? cols : 0);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float v[4];
    e4m3x4_value(w[j], s, v);
    T o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = from_f32_restored<T>(v[i]);
    store4<T, VEC>(out + b.row * cols, b.c0, sub, j, cols, o);
  }
}
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) act8_unpack_kernel(const uint8_t* __restrict__ codes,
                                                          const uint8_t* __restrict__ scales, long long rows,
                                                          int cols, T* __restrict__ out) {
  act8_unpack<T, VEC>(codes, scales, rows, cols, nullptr, out);
}

// One CTA per 128 x 128 block of a weight [n, k]: codes [n, k] (or [k, n]
// when TR) and one scale per block; the transposed copy goes through shared
// memory.  A model that serves packs once, one that trains packs both orders
// every step.  Two passes over the block in single elements, the second from
// L1 and L2: 18 us for 4096 x 1024 fp32, 22 transposed, where its 21 MB take 3.
template <typename T, bool TR>
__global__ void __launch_bounds__(256) weight8_pack_kernel(const T* __restrict__ w, int n, int k,
                                                           uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  __shared__ float s_max[8];
  __shared__ uint8_t s_codes[TR ? 128 * 129 : 1];
  const int kb = blockIdx.x, nb = blockIdx.y;
  const int col = kb * kBlk + (threadIdx.x & 127);
  const int r0 = nb * kBlk + (threadIdx.x >> 7);
  float amax = 0.f;
  if (col < k)
    for (int r = r0; r < min(n, (nb + 1) * kBlk); r += 2) amax = fmaxf(amax, finite_abs(to_f32<T>(w[(long long)r * k + col])));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = amax;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = fmaxf(amax, s_max[i]);
  const uint32_t byte = scale_byte(amax);
  const float inv = scale_inv(byte);
  if (threadIdx.x == 0) {
    if constexpr (TR) scales[(long long)kb * n_blocks(n) + nb] = (uint8_t)byte;
    else scales[(long long)nb * n_blocks(k) + kb] = (uint8_t)byte;
  }
  if (col < k)
    for (int r = r0; r < min(n, (nb + 1) * kBlk); r += 2) {
      const float v = to_f32<T>(w[(long long)r * k + col]);
      const uint8_t c = (uint8_t)e4m3x2<true>(v, 0.f, inv);
      if constexpr (TR) s_codes[(threadIdx.x & 127) * 129 + (r - nb * kBlk)] = c;
      else codes[(long long)r * k + col] = c;
    }
  if constexpr (TR) {
    __syncthreads();
    const int row = nb * kBlk + (threadIdx.x & 127);
    if (row < n)
      for (int c = threadIdx.x >> 7; c < min(kBlk, k - kb * kBlk); c += 2)
        codes[(long long)(kb * kBlk + c) * n + row] = s_codes[c * 129 + (threadIdx.x & 127)];
  }
}

// erfc(a / sqrt 2) exp(a^2 / 2) / 2 for a >= 0 is a polynomial in
// t = 1 / (1 + 0.475 a) without a constant term: fitted here (iterated weighted
// least squares over 0 <= a <= 13.2, past which exp(-a^2 / 2) is below 32 bits'
// normal range) and rounded to 32 bits so that it stays within 6.7e-8 relative,
// 3.4e-8 absolute.  Evaluated in 32 bits it is off by 3e-7 at most, 8e-8 rms.
// (Eight terms in 1 / (1 + 0.225 a): 1.9e-7, 4.5e-7 and 1.2e-7, which changed
// 1.4 times as many 8-bit codes of gelu as a plain 32-bit evaluation does.)
constexpr float kTailStep = 0.475f;
constexpr int kTailTerms = 9;
#define TJ_TAIL_COEFS                                                                                             \
  {0.18952046f, 0.18885313f, 0.15437007f, 0.01159445f, 0.1560375f, -0.5561017f, 0.5773829f, -0.2728236f, \
   0.051166784f}

// d gelu(h) / dh = Phi(h) + h phi(h), Phi the normal distribution and phi its
// density, for the exact (erf) GELU; two values at a time.  With a = |h|,
// u = exp(-a^2 / 2) and v = u (a / sqrt(2 pi) - erfc(a / sqrt 2) exp(a^2 / 2) / 2)
// it is 1 + v for h >= 0 and -v for h < 0 (formed as 1/2 - (1/2 + v) it loses
// the tail, all of it at h = -7), and one exponential serves both terms of v.
// What 32 bits keep: 2e-7 for h > -1, and below it 6e-7 of the value to -3,
// 1.4e-6 to -5, 3.4e-6 to -9 (a plain evaluation: 6e-7, 7e-7, 2.1e-6), from
// the roundings of a^2 / 2.  min.NaN keeps a NaN and makes an infinity finite,
// so that a u is 0 and not NaN.
TJ_DEV float2 gelu_slope_x2(float h0, float h1) {
  float a0, a1;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(a0) : "f"(fabsf(h0)), "f"(1e18f));
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(a1) : "f"(fabsf(h1)), "f"(1e18f));
  constexpr float kC[kTailTerms] = TJ_TAIL_COEFS;
  const uint64_t a = f32x2(a0, a1);
  const float2 den = f32x2_split(ffma_x2(a, f32x2(kTailStep, kTailStep), f32x2(1.f, 1.f)));
  const float2 aa = f32x2_split(fmul_x2(fmul_x2(a, f32x2(0.72134752044448170f, 0.72134752044448170f)), a));  // log2(e) / 2
  // a reciprocal each: one of the product for both costs three products and
  // keeping a NaN from its neighbour (143 us for 137 at 32768 x 4096 bf16)
  float t0, t1;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t0) : "f"(den.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t1) : "f"(den.y));
  const uint64_t t = f32x2(t0, t1), u = f32x2(fast_exp2(-aa.x), fast_exp2(-aa.y));
  uint64_t q = f32x2(kC[kTailTerms - 1], kC[kTailTerms - 1]);
#pragma unroll
  for (int i = kTailTerms - 2; i >= 0; --i) q = ffma_x2(t, q, f32x2(kC[i], kC[i]));
  // -v; the 1 is then added under a predicate (a select after both sums: 141 us for 137)
  float2 m = f32x2_split(fmul_x2(u, ffma_x2(a, f32x2(-0.39894228040143268f, -0.39894228040143268f), fmul_x2(t, q))));
  asm("{.reg .pred p; setp.ge.f32 p, %1, 0f00000000; @p sub.f32 %0, 0f3F800000, %0;}" : "+f"(m.x) : "f"(h0));
  asm("{.reg .pred p; setp.ge.f32 p, %1, 0f00000000; @p sub.f32 %0, 0f3F800000, %0;}" : "+f"(m.y) : "f"(h1));
  return m;
}

// CTAs per SM of the packing forms of 16-bit gradients, left to the compiler
// otherwise (16384 x 4096, 8-bit h: 96 us bf16 and 94 fp16 for 102 and 102; h
// in 16 bits: 94 and 102 for 113 and 109, 6 CTAs 109 and 143).
template <typename T, bool H8, bool PACK>
constexpr int gelu_bwd_ctas() { return sizeof(T) == 2 && PACK ? (H8 ? 6 : 5) : 0; }

// dh = dy * gelu'(h), rounded to T; PACK: also the 8-bit form of the rounded
// dh, so that the packed copy is the one that packing dh would give.
// h: 8-bit copy (H8) or a tensor of type T.
template <typename T, bool H8, bool PACK, bool VEC>
__global__ void __launch_bounds__(256, gelu_bwd_ctas<T, H8, PACK>()) gelu_bwd_kernel(const T* __restrict__ dy, const void* __restrict__ h,
                                                       const uint8_t* __restrict__ h_scales, long long rows, int cols,
                                                       const uint8_t* __restrict__ mask, T* __restrict__ dh,
                                                       uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  const BlockAt b = block_at(rows, cols);
  const int sub = threadIdx.x & 7;
  if (!PACK && !b.live) return;
  const bool valid = b.live && (mask == nullptr || mask[b.row] != 0);
  const int lim = valid ? cols : 0;
  const long long base = b.row * cols;
  float g[4][4], hv[4][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) load4<T, VEC>(dy + base, b.c0, sub, j, lim, g[j]);
  if constexpr (H8) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      w[j] = load_codes4<VEC>(static_cast<const uint8_t*>(h) + base, b.c0, sub, j, lim);
    const float s = valid ? scale_value(h_scales[b.row * n_blocks(cols) + b.blk]) : 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) e4m3x4_value(w[j], s, hv[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) load4<T, VEC>(static_cast<const T*>(h) + base, b.c0, sub, j, lim, hv[j]);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    T o[4];
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      const float2 sl = gelu_slope_x2(hv[j][i], hv[j][i + 1]);
      o[i] = from_f32<T>(g[j][i] * sl.x);  // masked rows: 0 * slope(0)
      o[i + 1] = from_f32<T>(g[j][i + 1] * sl.y);
      if constexpr (PACK) {
        g[j][i] = to_f32<T>(o[i]);
        g[j][i + 1] = to_f32<T>(o[i + 1]);
      }
    }
    if (b.live) store4<T, VEC>(dh + base, b.c0, sub, j, cols, o);
  }
  if constexpr (PACK)
    pack_block<VEC>(g, b.c0, cols, codes + base, scales + b.row * n_blocks(cols) + b.blk, sub, b.live);
}

// Column sums of in[n, cols], into out0 for c < split and out1 after it: a CTA
// has 8 columns (a 32-byte sector of a row), its 128 groups of 8 lanes every
// 128th row each; joined in a fixed order.  (32 columns to a CTA: 7.6 us for
// 592 x 2048, too few CTAs.)
TJ_DEV void column_sum(const float* __restrict__ in, int n, int cols, float* __restrict__ out0,
                       float* __restrict__ out1, int split, unsigned block) {
  __shared__ float s[128][9];
  const int col = threadIdx.x & 7, grp = threadIdx.x >> 3;
  const int c = block * 8 + col;
  float a = 0.f;
  if (c < cols) {
    for (int r0 = grp; r0 < n; r0 += 128 * 8) {
      float b[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) b[q] = r0 + 128 * q < n ? in[(size_t)(r0 + 128 * q) * cols + c] : 0.f;
#pragma unroll
      for (int q = 0; q < 8; ++q) a += b[q];
    }
  }
  s[grp][col] = a;
  __syncthreads();
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (w < 8) {
    const float t = warp_sum((s[lane][w] + s[lane + 32][w]) + (s[lane + 64][w] + s[lane + 96][w]));
    const int cc = block * 8 + w;
    if (lane == 0 && cc < cols) {
      if (cc < split) out0[cc] = t;
      else out1[cc - split] = t;
    }
  }
}

static __global__ void __launch_bounds__(1024) column_sum_kernel(const float* __restrict__ in, int n, int cols,
                                                                 float* __restrict__ out0, float* __restrict__ out1,
                                                                 int split) {
  column_sum(in, n, cols, out0, out1, split, blockIdx.x);
}

}  // namespace tj
