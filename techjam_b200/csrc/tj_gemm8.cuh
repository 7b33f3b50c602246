// Products of 8-bit activations and weights (tj_act8.cuh) on the tensor cores:
//
//   out[M, N] = sum over K blocks kb of 2^(ea[m, kb] + ew[n/128, kb]) * (codes A . codes W)  + bias [+ resid]
//
// tcgen05.mma kind::mxf8f6f4 multiplies by one e8m0 scale per 32 elements of K
// as it accumulates; a block of 128 is four of its steps with the same scale,
// so the scaling costs nothing and the sum stays in the FP32 accumulator.
// The scales are read from TMEM: 128 rows take four columns (row r in lane
// r % 32 of column r / 32, the same in all four lane quarters), and the four
// bytes of a column's word, picked by the instruction's scale id, hold four
// consecutive K blocks.  One word per row thus serves 512 of K.
//
// Persistent and warp-specialised, one CTA per SM:
//   warp 0      TMA loads of A and W tiles (128 bytes of K) into a ring
//   warp 1      issues the MMAs into one of two accumulators
//   warp 2      allocates TMEM
//   warps 4-7   write the scales to a ring of TMEM slots
//   warps 8..   epilogue: TMEM -> registers (thread = row) -> swizzled shared
//               memory -> TMA stores, which also clip the ragged edges
//
// The tensor core truncates when it adds to the accumulator; over 32 steps
// (1024 of K) that is about 6e-7 of the sum and grows with K.  A 32-bit result
// and the GELU kind, whose codes would more often fall on the wrong side of a
// boundary, therefore start a new accumulator after each 1024 of K, and the
// epilogue adds them up in registers, rounded to nearest.
#pragma once
#include "tj_act8.cuh"
#include "tj_gemm.cuh"

namespace tj {

enum Gemm8Kind : int { kG8F16 = 0, kG8BF16 = 1, kG8F32 = 2, kG8Gelu = 3 };

struct Gemm8Params {
  int M, N, K;
  int kblocks;  // 128-element blocks of K
  const uint8_t* a_scales;  // [M, kblocks]
  const uint8_t* w_scales;  // [ceil(N / 128), kblocks]
  const float* bias;        // [N] or null
  const uint8_t* mask;      // [M] or null: rows with 0 leave zeros
  int a_words, w_words;     // scale rows may be read as 32-bit words
  int has_resid;            // kG8F32: resid through its tensor map
  uint8_t* g_scales;        // kG8Gelu: [M, ceil(N / 128)]
  uint8_t* h_scales;
  int* err;
};

constexpr int kG8BM = 128;
constexpr int kG8Chunk = 8;  // kG8F32, kG8Gelu: K blocks per accumulator

template <int BN, int KIND>
struct Gemm8Cfg {
  static constexpr int kStageBytes = (kG8BM + BN) * 128;
  static constexpr int kCW = KIND == kG8Gelu ? 128 : 64;  // columns per epilogue warp
  static constexpr int kEpiWarps = 4 * BN / kCW;
  static constexpr int kBufs = KIND == kG8F32 || KIND == kG8Gelu ? 4 : 2;  // 4 KB staging buffers per epilogue warp
  static constexpr int kStagingBytes = kEpiWarps * kBufs * 4096;
  static constexpr int kStages = (224 * 1024 - kStagingBytes) / kStageBytes;
  static constexpr int kSfSlots = 4;
  static constexpr int kSfCols = 4 + BN / 32;
  static constexpr int kSfCol0 = 2 * BN;
  static constexpr int kTmemCols = 2 * BN + kSfSlots * kSfCols <= 256 ? 256 : 512;
  static constexpr int kThreads = 256 + 32 * kEpiWarps;
  static constexpr int kSmemBytes = 1024 + kStages * kStageBytes + kStagingBytes + 512;
  static_assert(kSmemBytes <= 232448, "shared memory");
  static_assert(2 * BN + kSfSlots * kSfCols <= 512, "TMEM");
};

// kind::mxf8f6f4, e4m3 x e4m3, e8m0 scales: the scale ids of B and A are added per K block.
__host__ __device__ constexpr uint32_t idesc_mx8(int M, int N) {
  return ((uint32_t)(N >> 3) << 17) | (1u << 23) | ((uint32_t)(M >> 7) << 27);
}
TJ_DEV uint32_t idesc_mx8_ids(uint32_t id) { return (id << 4) | (id << 29); }

TJ_DEV void umma_mx8_elect(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa,
                           uint32_t sfb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred e, p;\n\t.reg .b32 r;\n\t"
      "elect.sync r|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(
          d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}

template <int N>
TJ_DEV void tmem_st_words(uint32_t taddr, const uint32_t (&r)[N]) {
  static_assert(N == 2 || N == 4 || N == 8, "columns");
  if constexpr (N == 2)
    asm volatile("tcgen05.st.sync.aligned.32x32b.x2.b32 [%0], {%1,%2};" ::"r"(taddr), "r"(r[0]), "r"(r[1]) : "memory");
  if constexpr (N == 4)
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3])
                 : "memory");
  if constexpr (N == 8)
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}

TJ_DEV void tma_store_2d(const CUtensorMap* map, const void* src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map),
               "r"(smem_u32(src)), "r"(x), "r"(y)
               : "memory");
}
TJ_DEV void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// At most N of this thread's bulk stores may still read their shared memory.
template <int N>
TJ_DEV void bulk_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
TJ_DEV void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

TJ_DEV void mbar_arrive_cluster_release(uint32_t cluster_addr) {  // one lane of a converged warp
  asm volatile(
      "{\n\t.reg .pred e;\n\t.reg .b32 r;\n\t"
      "elect.sync r|e, 0xffffffff;\n\t"
      "@e mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];\n\t}" ::"r"(cluster_addr)
      : "memory");
}
// Plain remote arrive (as mbar_arrive_cluster), by one lane of a converged warp.
TJ_DEV void mbar_arrive_cluster_elect(uint32_t cluster_addr) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t.reg .b32 r;\n\t"
      "elect.sync r|e, 0xffffffff;\n\t"
      "@e mbarrier.arrive.shared::cluster.b64 _, [%0];\n\t}" ::"r"(cluster_addr)
      : "memory");
}
// Bounded wait that also acquires what the other CTA of the pair released.
TJ_DEV bool mbar_wait_cluster_warp(uint64_t* bar, uint32_t parity, int* err, int site) {
  auto try_wait = [&] {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
  };
  if (__all_sync(0xffffffffu, try_wait())) return true;
  if (!mbar_wait_warp<true>(bar, parity, err, site)) return false;
  return __all_sync(0xffffffffu, try_wait());  // complete: returns at once, with the acquire
}

// Four bytes of a scale row from block b0 on; past the end 2^0.  words: the
// rows start at multiples of 4 and are multiples of 4 long.
TJ_DEV uint32_t scale_word(const uint8_t* row, int b0, int blocks, bool words) {
  if (words) return __ldg(reinterpret_cast<const uint32_t*>(row + b0));
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) w |= (uint32_t)(b0 + i < blocks ? __ldg(row + b0 + i) : 127) << (8 * i);
  return w;
}

// Whether any of the tile's 128 rows is valid (whole warp).
TJ_DEV bool tile_has_rows(const uint8_t* mask, int row0, int M, int lane) {
  if (mask == nullptr) return true;
  int any = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = row0 + lane + 32 * i;
    if (r < M) any |= __ldg(mask + r);
  }
  return __any_sync(0xffffffffu, any != 0);
}

TJ_DEV uint32_t pack_bf162(float a, float b) {
  __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}

// 16-byte piece j of this lane's 128-byte row in a 32-row staging buffer (the
// 128-byte TMA swizzle; conflict-free for one piece per lane).
TJ_DEV uint8_t* staged(uint8_t* buf, int lane, int j) { return buf + lane * 128 + ((j ^ (lane & 7)) << 4); }

// gelu(x) = max(x, 0) - |x| T(|x|) exp(-x^2 / 2) for two values, where
// T(a) = erfc(a / sqrt 2) exp(a^2 / 2) / 2 is the polynomial of tj_act8.cuh.
// Nothing cancels for x < 0.  exp(-x^2 / 2) = 2^-((x log2(e) / 2) x): rounded
// twice where the square of x sqrt(log2(e) / 2) counts its rounding twice.  A
// reciprocal for each value keeps a value's result its own; one of the product
// for both took as long (16384 x 2048 x 512: 55 us a call) and cost bits.  For
// |x| near the largest float t flushes to zero and the exponential is zero.
TJ_DEV uint64_t gelu8_x2(uint64_t x) {
  const float2 v = f32x2_split(x);
  float t0, t1;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t0) : "f"(fmaf(fabsf(v.x), kTailStep, 1.f)));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t1) : "f"(fmaf(fabsf(v.y), kTailStep, 1.f)));
  const uint64_t t = f32x2(t0, t1);
  constexpr float kC[kTailTerms] = TJ_TAIL_COEFS;
  uint64_t q = f32x2(kC[kTailTerms - 1], kC[kTailTerms - 1]);
#pragma unroll
  for (int i = kTailTerms - 2; i >= 0; --i) q = ffma_x2(t, q, f32x2(kC[i], kC[i]));
  const float2 yy = f32x2_split(fmul_x2(fmul_x2(x, f32x2(0.72134752044448170f, 0.72134752044448170f)), x));  // log2(e) / 2
  const float2 tail = f32x2_split(fmul_x2(fmul_x2(t, q), f32x2(fast_exp2(-yy.x), fast_exp2(-yy.y))));
  return f32x2(fmaf(-fabsf(v.x), tail.x, fmaxf(v.x, 0.f)), fmaf(-fabsf(v.y), tail.y, fmaxf(v.y, 0.f)));
}
// Codes of four values that are no infinities, times inv (twice the same).
TJ_DEV uint32_t e4m3_pairs(uint64_t x, uint64_t y, uint64_t inv) {
  const float2 a = f32x2_split(fmul_x2(x, inv)), b = f32x2_split(fmul_x2(y, inv));
  return e4m3_word(a.x, a.y, b.x, b.y);
}

// GELU epilogue of N columns (a block of 128, or half of one) of one row: h in
// 32 bits, two to a word -> staged codes of g = gelu(h) and of h from 16-byte
// piece `piece0` on, and the block's scale bytes (rows that are not valid:
// zeros).  join(a, b) takes the maxima with the other half's.
// gelu grows with h > 0 and its dip for h < 0 is 0.17 deep, which gelu(0.3)
// exceeds: above that the largest |g| is gelu of the largest h (as computed
// too: no smaller h comes out on the other side of any scale's border), and
// only a warp with a smaller one looks at every g.  Called by whole warps.
template <int N, typename Join>
TJ_DEV void gelu_pack_row(uint64_t (&h)[N / 2], bool valid, uint8_t* bufg, uint8_t* bufh, int piece0, int lane,
                          uint32_t& gbyte, uint32_t& hbyte, Join&& join) {
  float hmax = 0.f, hpos = 0.f;
  auto maxima = [&] {
    float m[4] = {0.f, 0.f, 0.f, 0.f}, q[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const float2 v = f32x2_split(h[i]);
      m[i & 3] = max3f(m[i & 3], fabsf(v.x), fabsf(v.y));
      q[i & 3] = max3f(q[i & 3], v.x, v.y);
    }
    hmax = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
    hpos = fmaxf(fmaxf(q[0], q[1]), fmaxf(q[2], q[3]));
  };
  maxima();
  if (__any_sync(0xffffffffu, hmax > 3.402823466e38f)) {  // infinities become NaN, which the maxima drop
    const float nan = __int_as_float(0x7fffffff);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const float2 v = f32x2_split(h[i]);
      h[i] = f32x2(fabsf(v.x) > 3.402823466e38f ? nan : v.x, fabsf(v.y) > 3.402823466e38f ? nan : v.y);
    }
    maxima();
  }
  join(hmax, hpos);
  float gmax = f32x2_split(gelu8_x2(f32x2(hpos, 0.f))).x;
  if (__any_sync(0xffffffffu, hpos < 0.3f)) {  // the same in both halves' warps
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const float2 g = f32x2_split(gelu8_x2(h[i]));
      gmax = max3f(gmax, fabsf(g.x), fabsf(g.y));
    }
    float same = gmax;
    join(gmax, same);
  }
  gbyte = valid ? scale_byte(gmax) : 127u;
  hbyte = valid ? scale_byte(hmax) : 127u;
  const uint64_t ginv = f32x2(scale_inv(gbyte), scale_inv(gbyte)), hinv = f32x2(scale_inv(hbyte), scale_inv(hbyte));
#pragma unroll
  for (int j = 0; j < N / 16; ++j) {
    uint32_t gw[4], hw[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint64_t v0 = h[8 * j + 2 * i], v1 = h[8 * j + 2 * i + 1];
      gw[i] = e4m3_pairs(gelu8_x2(v0), gelu8_x2(v1), ginv);
      hw[i] = e4m3_pairs(v0, v1, hinv);
    }
    *reinterpret_cast<uint4*>(staged(bufg, lane, piece0 + j)) = make_uint4(gw[0], gw[1], gw[2], gw[3]);
    *reinterpret_cast<uint4*>(staged(bufh, lane, piece0 + j)) = make_uint4(hw[0], hw[1], hw[2], hw[3]);
  }
  if (!valid) {
#pragma unroll
    for (int j = 0; j < N / 16; ++j) {
      *reinterpret_cast<uint4*>(staged(bufg, lane, piece0 + j)) = make_uint4(0, 0, 0, 0);
      *reinterpret_cast<uint4*>(staged(bufh, lane, piece0 + j)) = make_uint4(0, 0, 0, 0);
    }
  }
}
// h = the bias of columns col0.. (zeros past n), and h += 32 accumulator columns.
template <int N>
TJ_DEV void bias_pairs(uint64_t (&h)[N / 2], const float* bias, int col0, int n) {
#pragma unroll
  for (int j = 0; j < N / 4; ++j) {
    float4 b = make_float4(0.f, 0.f, 0.f, 0.f);
    if (bias != nullptr && col0 + 4 * j < n) b = __ldg(reinterpret_cast<const float4*>(bias + col0) + j);
    h[2 * j] = f32x2(b.x, b.y);
    h[2 * j + 1] = f32x2(b.z, b.w);
  }
}
TJ_DEV void add_pairs(uint64_t* h, const uint32_t (&r)[32]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) h[i] = fadd_x2(h[i], f32x2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])));
}

// Adds the bias of columns col0.. (zeros past n) to 32 values.
TJ_DEV void add_bias32(float* v, const float* bias, int col0, int n) {
  if (bias == nullptr) return;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (col0 + 4 * j < n) {
      const float4 b = __ldg(reinterpret_cast<const float4*>(bias + col0) + j);
      v[4 * j] += b.x; v[4 * j + 1] += b.y; v[4 * j + 2] += b.z; v[4 * j + 3] += b.w;
    }
}

template <int BN, int KIND>
__global__ void __launch_bounds__(Gemm8Cfg<BN, KIND>::kThreads, 1)
    gemm8_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW,
                 const __grid_constant__ CUtensorMap tmOut, const __grid_constant__ CUtensorMap tmAux,
                 const Gemm8Params p) {
  using Cfg = Gemm8Cfg<BN, KIND>;
  constexpr int S = Cfg::kStages, SF = Cfg::kSfSlots;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* staging = smem + S * Cfg::kStageBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(staging + Cfg::kStagingBytes);
  uint64_t* empty = full + S;
  uint64_t* acc_full = empty + S;       // [2]
  uint64_t* acc_empty = acc_full + 2;   // [2]
  uint64_t* sf_full = acc_empty + 2;    // [SF]
  uint64_t* sf_empty = sf_full + SF;    // [SF]
  uint64_t* res_full = sf_empty + SF;   // [epilogue warps][bufs], kG8F32
  uint64_t* drained = res_full + (KIND == kG8F32 ? Cfg::kEpiWarps * Cfg::kBufs : 0);  // every MMA is complete
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
  static_assert((2 * S + 5 + 2 * SF + 32) * 8 + 4 <= 512, "barrier space");

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) { mbar_init(full + i, 1); mbar_init(empty + i, 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(acc_full + i, 1); mbar_init(acc_empty + i, Cfg::kEpiWarps); }
    for (int i = 0; i < SF; ++i) { mbar_init(sf_full + i, 4); mbar_init(sf_empty + i, 1); }
    if constexpr (KIND == kG8F32)
      for (int i = 0; i < Cfg::kEpiWarps * Cfg::kBufs; ++i) mbar_init(res_full + i, 1);
    mbar_init(drained, 1);
    fence_mbar_init();
  }
  if (warp == 2) {
    tmem_alloc(tmem_slot, Cfg::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  const int n_tiles = (p.N + BN - 1) / BN;
  const int m_tiles = (p.M + kG8BM - 1) / kG8BM;
  const long long total = (long long)m_tiles * n_tiles;
  const int kblocks = p.kblocks;
  constexpr int kChunk = KIND == kG8F32 || KIND == kG8Gelu ? kG8Chunk : 1 << 30;  // K blocks per accumulator

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0) { tma_prefetch_desc(&tmA); tma_prefetch_desc(&tmW); }
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (long long t = blockIdx.x; t < total && ok; t += gridDim.x) {
      const int mt = (int)(t / n_tiles), nt = (int)(t % n_tiles);
      if (!tile_has_rows(p.mask, mt * kG8BM, p.M, lane)) continue;
      for (int kb = 0; kb < kblocks; ++kb) {
        if (!mbar_wait_warp<true>(empty + stage, phase ^ 1u, p.err, kErrGemm8Producer)) { ok = false; break; }
        if (lane == 0) {
          uint8_t* sa = smem + stage * Cfg::kStageBytes;
          mbar_expect_tx(full + stage, Cfg::kStageBytes);
          tma_load_2d(sa, &tmA, full + stage, kb * 128, mt * kG8BM);
          tma_load_2d(sa + kG8BM * 128, &tmW, full + stage, kb * 128, nt * BN);
        }
        __syncwarp();
        if (++stage == S) { stage = 0; phase ^= 1u; }
      }
    }
    if (lane == 0) Drain().ring(full, S, stage, phase);
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    int stage = 0, abuf = 0, slot = 0;
    uint32_t phase = 0, aphase = 0, sphase = 0;
    bool ok = true;
    for (long long t = blockIdx.x; t < total && ok; t += gridDim.x) {
      const int mt = (int)(t / n_tiles);
      if (!tile_has_rows(p.mask, mt * kG8BM, p.M, lane)) continue;
      for (int kb = 0; kb < kblocks; ++kb) {
        const bool first = kb % kChunk == 0;
        if (first) {
          if (!mbar_wait_warp<true>(acc_empty + abuf, aphase ^ 1u, p.err, kErrGemm8Mma)) { ok = false; break; }
        }
        if ((kb & 3) == 0) {
          if (!mbar_wait_warp<true>(sf_full + slot, sphase, p.err, kErrGemm8Mma)) { ok = false; break; }
        }
        if (!mbar_wait_warp<true>(full + stage, phase, p.err, kErrGemm8Mma)) { ok = false; break; }
        tc_fence_after();
        const uint32_t sa = smem_u32(smem + stage * Cfg::kStageBytes);
        const uint32_t sb = sa + kG8BM * 128;
        const uint32_t sfa = tmem_base + Cfg::kSfCol0 + slot * Cfg::kSfCols;
        const uint32_t idesc = idesc_mx8(kG8BM, BN) | idesc_mx8_ids(kb & 3);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
          umma_mx8_elect(tmem_base + abuf * BN, smem_desc(sa + ks * 32, 16, 1024, 128),
                         smem_desc(sb + ks * 32, 16, 1024, 128), idesc, sfa, sfa + 4, !(first && ks == 0));
        umma_commit_elect(empty + stage);
        if (++stage == S) { stage = 0; phase ^= 1u; }
        if ((kb & 3) == 3 || kb + 1 == kblocks) {
          umma_commit_elect(sf_empty + slot);
          if (++slot == SF) { slot = 0; sphase ^= 1u; }
        }
        if (kb % kChunk == kChunk - 1 || kb + 1 == kblocks) {
          umma_commit_elect(acc_full + abuf);
          if (++abuf == 2) { abuf = 0; aphase ^= 1u; }
        }
      }
    }
    umma_commit_elect(drained);
    Drain().wait(drained, 0);
    __syncwarp();
  } else if (warp >= 4 && warp < 8) {
    // ------------------------------------------------------------ scales -> TMEM
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    int slot = 0;
    uint32_t sphase = 0;
    bool ok = true;
    for (long long t = blockIdx.x; t < total && ok; t += gridDim.x) {
      const int mt = (int)(t / n_tiles), nt = (int)(t % n_tiles);
      if (!tile_has_rows(p.mask, mt * kG8BM, p.M, lane)) continue;
      const uint8_t* wrow = p.w_scales + (long long)(nt * BN / kBlk) * kblocks;
      uint32_t a[4], b[BN / 32];
      auto fetch = [&](int kb) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int row = mt * kG8BM + 32 * c + lane;
          a[c] = row < p.M ? scale_word(p.a_scales + (long long)row * kblocks, kb, kblocks, p.a_words) : 0x7f7f7f7fu;
        }
        b[0] = scale_word(wrow, kb, kblocks, p.w_words);
#pragma unroll
        for (int c = 1; c < BN / 32; ++c) b[c] = b[0];
      };
      for (int kb = 0; kb < kblocks; kb += 4) {
        fetch(kb);
        if (!mbar_wait_warp<true>(sf_empty + slot, sphase ^ 1u, p.err, kErrGemm8Scales)) { ok = false; break; }
        tc_fence_after();
        const uint32_t at = tmem_base + lanes + Cfg::kSfCol0 + slot * Cfg::kSfCols;
        tmem_st_words<4>(at, a);
        tmem_st_words<BN / 32>(at + 4, b);
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive_elect(sf_full + slot);
        if (++slot == SF) { slot = 0; sphase ^= 1u; }
      }
    }
  } else if (warp >= 8) {
    // ------------------------------------------------------------ epilogue
    const int ew = warp - 8;
    const int quarter = warp & 3;
    const int cg = ew >> 2;  // column group of this warp
    uint8_t* bufs = staging + ew * Cfg::kBufs * 4096;
    int abuf = 0;
    uint32_t aphase = 0;
    bool ok = true;
    // staging buffers are used in turn; each use ends in one bulk store of lane 0
    uint32_t used = 0;
    uint32_t rphase = 0;  // kG8F32: bit b: parity of buffer b's next residual load
    for (long long t = blockIdx.x; t < total && ok; t += gridDim.x) {
      const int mt = (int)(t / n_tiles), nt = (int)(t % n_tiles);
      const bool live = tile_has_rows(p.mask, mt * kG8BM, p.M, lane);
      const int row0 = mt * kG8BM + quarter * 32;
      const int col0 = nt * BN + cg * Cfg::kCW;
      const int row = row0 + lane;
      const bool valid = row < p.M && (p.mask == nullptr || __ldg(p.mask + row) != 0);
      const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + cg * Cfg::kCW;
      auto wait_acc = [&] {
        ok = mbar_wait_warp<true>(acc_full + abuf, aphase, p.err, kErrGemm8Epilogue);
        tc_fence_after();
        return ok;
      };
      auto free_acc = [&] {
        tc_fence_before();
        mbar_arrive_elect(acc_empty + abuf);
        if (++abuf == 2) { abuf = 0; aphase ^= 1u; }
      };
      if constexpr (KIND == kG8F32) {
        // 64 columns as two 32-column (128-byte) pieces; the residual is
        // fetched into the staging buffers while the MMAs run
        const int pieces = row0 < p.M ? min(2, (p.N - col0 + 31) / 32) : 0;  // may be negative: none
        const bool fetch = p.has_resid && live;
        if (fetch && lane == 0) {
          for (int c = 0; c < pieces; ++c) {
            const uint32_t b = (used + c) % Cfg::kBufs;
            bulk_wait_read<2>();  // the store that used this buffer last is four or three back
            mbar_expect_tx(res_full + ew * Cfg::kBufs + b, 4096);
            tma_load_2d(bufs + b * 4096, &tmAux, res_full + ew * Cfg::kBufs + b, col0 + 32 * c, row0);
          }
        }
        __syncwarp();
        float acc[64];
#pragma unroll
        for (int i = 0; i < 64; ++i) acc[i] = 0.f;
        if (live) {
          for (int kb = 0; kb < kblocks; kb += kChunk) {
            if (!wait_acc()) break;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              uint32_t r[32];
              tmem_ld32(taddr + abuf * BN + 32 * c, r);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) acc[32 * c + i] += __uint_as_float(r[i]);
            }
            free_acc();
          }
          // after an expired wait the loop still goes on to the residual's
          // own waits, so that no load is in flight when the block ends
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (c < pieces) {
            const int col = col0 + 32 * c;
            const uint32_t b = used % Cfg::kBufs;
            uint8_t* buf = bufs + b * 4096;
            if (fetch) {
              uint64_t* bar = res_full + ew * Cfg::kBufs + b;
              if (!mbar_wait_warp<true>(bar, (rphase >> b) & 1u, p.err, kErrGemm8Epilogue)) {
                ok = false;
                Drain().wait(bar, (rphase >> b) & 1u);
                __syncwarp();
              }
              rphase ^= 1u << b;
            } else {
              if (lane == 0) bulk_wait_read<2>();
              __syncwarp();
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              float4* dst = reinterpret_cast<float4*>(staged(buf, lane, j));
              float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
              if (valid) {
                o = make_float4(acc[32 * c + 4 * j], acc[32 * c + 4 * j + 1], acc[32 * c + 4 * j + 2],
                                acc[32 * c + 4 * j + 3]);
                if (p.bias != nullptr && col + 4 * j < p.N) {
                  const float4 bb = __ldg(reinterpret_cast<const float4*>(p.bias + col) + j);
                  o.x += bb.x; o.y += bb.y; o.z += bb.z; o.w += bb.w;
                }
                if (p.has_resid) {
                  const float4 rr = *dst;
                  o.x += rr.x; o.y += rr.y; o.z += rr.z; o.w += rr.w;
                }
              }
              *dst = o;
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_2d(&tmOut, buf, col, row0);
              bulk_commit();
            }
            ++used;
          }
        }
      } else if constexpr (KIND == kG8F16 || KIND == kG8BF16) {
        uint32_t w[32];
        if (live) {
          if (!wait_acc()) break;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t r[32];
            tmem_ld32(taddr + abuf * BN + 32 * c, r);
            tmem_ld_wait();
            if (c == 1) free_acc();
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              float4 o = make_float4(__uint_as_float(r[4 * j]), __uint_as_float(r[4 * j + 1]),
                                     __uint_as_float(r[4 * j + 2]), __uint_as_float(r[4 * j + 3]));
              if (p.bias != nullptr && col0 + 32 * c + 4 * j < p.N) {
                const float4 bb = __ldg(reinterpret_cast<const float4*>(p.bias + col0 + 32 * c) + j);
                o.x += bb.x; o.y += bb.y; o.z += bb.z; o.w += bb.w;
              }
              if constexpr (KIND == kG8F16) {
                w[16 * c + 2 * j] = pack_half2(o.x, o.y);
                w[16 * c + 2 * j + 1] = pack_half2(o.z, o.w);
              } else {
                w[16 * c + 2 * j] = pack_bf162(o.x, o.y);
                w[16 * c + 2 * j + 1] = pack_bf162(o.z, o.w);
              }
            }
          }
        }
        if (row0 < p.M && col0 < p.N) {
          uint8_t* buf = bufs + (used % Cfg::kBufs) * 4096;
          if (lane == 0) bulk_wait_read<Cfg::kBufs - 1>();
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 8; ++j)
            *reinterpret_cast<uint4*>(staged(buf, lane, j)) =
                valid ? make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]) : make_uint4(0, 0, 0, 0);
          fence_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&tmOut, buf, col0, row0);
            bulk_commit();
          }
          ++used;
        }
      } else {
        // GELU: this warp's 128 columns are one block of g and of h, and a
        // thread holds a whole row of it
        const bool store = row0 < p.M && col0 < p.N;
        uint32_t gbyte = 127u, hbyte = 127u;
        uint8_t* bufg = bufs + (used % Cfg::kBufs) * 4096;
        uint8_t* bufh = bufs + ((used + 1) % Cfg::kBufs) * 4096;
        uint64_t h[64];
        bias_pairs<128>(h, p.bias, col0, p.N);
        if (live) {
          for (int kb = 0; kb < kblocks; kb += kChunk) {
            if (!wait_acc()) break;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint32_t r[32];
              tmem_ld32(taddr + abuf * BN + 32 * c, r);
              tmem_ld_wait();
              add_pairs(h + 16 * c, r);
            }
            free_acc();
          }
          if (!ok) break;
        }
        if (store) {
          if (lane == 0) bulk_wait_read<2>();
          __syncwarp();
          gelu_pack_row<128>(h, valid, bufg, bufh, 0, lane, gbyte, hbyte, [](float&, float&) {});
          fence_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&tmOut, bufg, col0, row0);
            bulk_commit();
            tma_store_2d(&tmAux, bufh, col0, row0);
            bulk_commit();
          }
          used += 2;
          if (row < p.M) {
            const long long s = (long long)row * n_blocks(p.N) + col0 / kBlk;
            p.g_scales[s] = (uint8_t)gbyte;
            p.h_scales[s] = (uint8_t)hbyte;
          }
        }
      }
    }
    if (lane == 0) bulk_wait_all();
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 2) tmem_dealloc(tmem_base, Cfg::kTmemCols);
}

// ------------------------------------------------------------------ CTA pairs
// A pair computes 256 x 256 tiles with cta_group::2: each CTA stages 128 rows
// of A and 128 of the 256 W rows, 32 KB for 512 cycles of MMA (a 128 x 128
// tile of one CTA needs 32 KB for 256, twice what an SM gets from L2).
//
// TMEM holds two 256-column accumulators and the scales only because the
// accumulators overlap by 32 columns: buffer 0 has columns 0-255, buffer 1
// columns 224-479.  The epilogue of a tile therefore reads the shared columns
// first and announces them (`shared_free`), and the next tile's MMAs wait for
// that besides their buffer.  Meanwhile the operand ring fills, so that the
// loads, which bound the kernel, do not pause.
template <int KIND>
struct Gemm8PairCfg {
  static constexpr int kBN = 256;
  static constexpr int kStageBytes = 2 * 128 * 128;
  // kG8Gelu: 16 epilogue warps of 64 columns, each two sharing a block and its
  // staging (with 8 of 128 columns the SFU and FMA latencies showed: 64 us
  // for 16384 x 2048 x 512); else 8 warps of 128 columns
  static constexpr int kEpiWarps = KIND == kG8Gelu ? 16 : 8;
  static constexpr int kStagingBytes = 64 * 1024;
  static constexpr int kStages = 5;
  static constexpr int kAcc1 = 224;   // first column of buffer 1
  static constexpr int kSfCol0 = 480;
  static constexpr int kSfSlots = 2;
  static constexpr int kSfCols = 12;  // 4 for A's 128 rows, 8 for W's 256
  static constexpr int kThreads = 256 + 32 * kEpiWarps;
  // kG8Gelu: warpgroups with 24 + 40 + 4 * 104 (96 spilled more and took a sixth longer); kG8F32: 56 + 56 + 2 * 200
  static constexpr int kRegLaunch = KIND == kG8Gelu ? 80 : 128;
  static constexpr int kSmemBytes = 1024 + kStages * kStageBytes + kStagingBytes + 512;
  static_assert(kSmemBytes <= 232448, "shared memory");
};

TJ_DEV void umma_mx8_pair_elect(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa,
                                uint32_t sfb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred e, p;\n\t.reg .b32 r;\n\t"
      "elect.sync r|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "@e tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(
          d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}

template <int KIND>
__global__ void __launch_bounds__(Gemm8PairCfg<KIND>::kThreads, 1)
    gemm8_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW,
                      const __grid_constant__ CUtensorMap tmOut, const __grid_constant__ CUtensorMap tmAux,
                      const Gemm8Params p) {
  using Cfg = Gemm8PairCfg<KIND>;
  constexpr int S = Cfg::kStages, SF = Cfg::kSfSlots;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* staging = smem + S * Cfg::kStageBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(staging + Cfg::kStagingBytes);  // [S] (even CTA's copy)
  uint64_t* empty = full + S;             // [S]
  uint64_t* acc_full = empty + S;         // [2]
  uint64_t* acc_empty = acc_full + 2;     // [2] (even CTA's copy)
  uint64_t* shared_free = acc_empty + 2;  // the shared columns are read (even CTA's copy)
  uint64_t* sf_full = shared_free + 1;    // [SF] (even CTA's copy)
  uint64_t* sf_empty = sf_full + SF;      // [SF]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sf_empty + SF);
  volatile uint8_t* agreed = reinterpret_cast<volatile uint8_t*>(tmem_slot + 1);  // kG8Gelu: [2][16], an epilogue warp's wait succeeded
  uint64_t* res_full = full + 32;  // kG8F32: [8 epilogue warps][2]
  uint64_t* drained = full + 48;   // every MMA is complete (even CTA's copy)
  static_assert((2 * S + 5 + 2 * SF) * 8 + 4 + 32 <= 256, "barrier space");

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;
  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) { mbar_init(full + i, 1); mbar_init(empty + i, 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(acc_full + i, 1); mbar_init(acc_empty + i, 2 * Cfg::kEpiWarps); }
    mbar_init(shared_free, 8);
    for (int i = 0; i < SF; ++i) { mbar_init(sf_full + i, 8); mbar_init(sf_empty + i, 1); }
    if constexpr (KIND == kG8F32)
      for (int i = 0; i < 16; ++i) mbar_init(res_full + i, 1);
    mbar_init(drained, 1);
    fence_mbar_init();
  }
  if (warp == 2) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  const int n_tiles = (p.N + 255) / 256;
  const int m_tiles = (p.M + 255) / 256;
  const long long total = (long long)m_tiles * n_tiles;
  const int kblocks = p.kblocks;
  constexpr int kChunk = KIND == kG8F32 || KIND == kG8Gelu ? kG8Chunk : 1 << 30;
  // both CTAs take or leave a tile together
  auto pair_has_rows = [&](int mt) {
    return tile_has_rows(p.mask, mt * 256, p.M, lane) || tile_has_rows(p.mask, mt * 256 + 128, p.M, lane);
  };

  if (warp < 4) {
    if constexpr (KIND == kG8Gelu) reg_dealloc<24>();
    if constexpr (KIND == kG8F32) reg_dealloc<56>();
    if (warp == 0) {
      // ---------------------------------------------------------- TMA producer
      if (lane == 0) { tma_prefetch_desc(&tmA); tma_prefetch_desc(&tmW); }
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (long long t = pair; t < total && ok; t += n_pairs) {
        const int mt = (int)(t / n_tiles), nt = (int)(t % n_tiles);
        if (!pair_has_rows(mt)) continue;
        if (lane == 0) {
          for (int kb = 0; kb < kblocks; ++kb) {
            if (!mbar_wait<true>(empty + stage, phase ^ 1u, p.err, kErrGemm8Producer)) { ok = false; break; }
            uint8_t* sa = smem + stage * Cfg::kStageBytes;
            const uint32_t lb = pair_leader_bar(full + stage);
            if (rank == 0) mbar_expect_tx(full + stage, 2 * Cfg::kStageBytes);
            tma_load_2d_pair(sa, &tmA, lb, kb * 128, mt * 256 + (int)rank * 128);
            tma_load_2d_pair(sa + 16384, &tmW, lb, kb * 128, nt * 256 + (int)rank * 128);
            if (++stage == S) { stage = 0; phase ^= 1u; }
          }
        }
        ok = __all_sync(0xffffffffu, ok);
      }
      // the loads signal the even CTA, but both learn when the MMAs have used them
      if (lane == 0) Drain().ring(empty, S, stage, phase);
      __syncwarp();
    } else if (warp == 1 && rank == 0) {
      // ---------------------------------------------------------- MMA issuer
      int stage = 0, abuf = 0, slot = 0;
      uint32_t phase = 0, aphase = 0, sphase = 0, shphase = 0;
      bool ok = true, any = false;
      for (long long t = pair; t < total && ok; t += n_pairs) {
        if (!pair_has_rows((int)(t / n_tiles))) continue;
        for (int kb = 0; kb < kblocks; ++kb) {
          const bool first = kb % kChunk == 0;
          if (first) {
            if (!mbar_wait_warp<true>(acc_empty + abuf, aphase ^ 1u, p.err, kErrGemm8Mma)) { ok = false; break; }
            if (any) {  // the accumulator before this one has given up the shared columns
              if (!mbar_wait_warp<true>(shared_free, shphase, p.err, kErrGemm8Mma)) { ok = false; break; }
              shphase ^= 1u;
            }
            any = true;
          }
          if ((kb & 3) == 0) {
            if (!mbar_wait_warp<true>(sf_full + slot, sphase, p.err, kErrGemm8Mma)) { ok = false; break; }
          }
          if (!mbar_wait_warp<true>(full + stage, phase, p.err, kErrGemm8Mma)) { ok = false; break; }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * Cfg::kStageBytes);
          const uint32_t sfa = tmem_base + Cfg::kSfCol0 + slot * Cfg::kSfCols;
          const uint32_t idesc = idesc_mx8(256, 256) | idesc_mx8_ids(kb & 3);
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            umma_mx8_pair_elect(tmem_base + abuf * Cfg::kAcc1, smem_desc(sa + ks * 32, 16, 1024, 128),
                                smem_desc(sa + 16384 + ks * 32, 16, 1024, 128), idesc, sfa, sfa + 4,
                                !(first && ks == 0));
          umma_commit_pair_both_elect(empty + stage);
          if (++stage == S) { stage = 0; phase ^= 1u; }
          if ((kb & 3) == 3 || kb + 1 == kblocks) {
            umma_commit_pair_both_elect(sf_empty + slot);
            if (++slot == SF) { slot = 0; sphase ^= 1u; }
          }
          if (kb % kChunk == kChunk - 1 || kb + 1 == kblocks) {
            umma_commit_pair_both_elect(acc_full + abuf);
            if (++abuf == 2) { abuf = 0; aphase ^= 1u; }
          }
        }
      }
      umma_commit_pair_elect(drained);
      Drain().wait(drained, 0);
      __syncwarp();
    }
  } else if (warp < 8) {
    // ------------------------------------------------------------ scales -> TMEM
    if constexpr (KIND == kG8Gelu) reg_dealloc<40>();
    if constexpr (KIND == kG8F32) reg_dealloc<56>();
    // The words of a group of four K blocks are on their way a group ahead,
    // across tiles, so that no slot waits for global memory.
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t sf_full0 = map_to_rank(sf_full, 0);
    uint32_t a[4], b0, b4;
    auto next_tile = [&](long long t) {
      while (t < total && !pair_has_rows((int)(t / n_tiles))) t += n_pairs;
      return t;
    };
    auto fetch = [&](long long t, int kb) {
      if (t >= total) return;
      const int mt = (int)(t / n_tiles), nt = (int)(t % n_tiles);
      const uint8_t* wrow = p.w_scales + (long long)(2 * nt) * kblocks;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int row = mt * 256 + (int)rank * 128 + 32 * c + lane;
        a[c] = row < p.M ? scale_word(p.a_scales + (long long)row * kblocks, kb, kblocks, p.a_words) : 0x7f7f7f7fu;
      }
      b0 = scale_word(wrow, kb, kblocks, p.w_words);
      b4 = nt * 256 + 128 < p.N ? scale_word(wrow + kblocks, kb, kblocks, p.w_words) : 0x7f7f7f7fu;
    };
    int slot = 0;
    uint32_t sphase = 0;
    bool ok = true;
    long long t = next_tile(pair);
    fetch(t, 0);
    while (t < total && ok) {
      const long long after = next_tile(t + n_pairs);
      for (int kb = 0; kb < kblocks; kb += 4) {
        const uint32_t wa[4] = {a[0], a[1], a[2], a[3]};
        const uint32_t wb[8] = {b0, b0, b0, b0, b4, b4, b4, b4};
        if (kb + 4 < kblocks) fetch(t, kb + 4);
        else fetch(after, 0);
        if (!mbar_wait_warp<true>(sf_empty + slot, sphase ^ 1u, p.err, kErrGemm8Scales)) { ok = false; break; }
        tc_fence_after();
        const uint32_t at = tmem_base + lanes + Cfg::kSfCol0 + slot * Cfg::kSfCols;
        tmem_st_words<4>(at, wa);
        tmem_st_words<8>(at + 4, wb);
        tmem_st_wait();
        // TMEM alone is handed over, which the tcgen05 fences order; a release
        // at cluster scope would wait for the loads above (22 us of 158)
        tc_fence_before();
        mbar_arrive_cluster_elect(sf_full0 + (uint32_t)(slot * sizeof(uint64_t)));
        if (++slot == SF) { slot = 0; sphase ^= 1u; }
      }
      t = after;
    }
  } else {
    // ------------------------------------------------------------ epilogue
    if constexpr (KIND == kG8Gelu) reg_alloc<104>();
    if constexpr (KIND == kG8F32) reg_alloc<200>();
    const int ew = warp - 8, quarter = warp & 3;
    constexpr int kGroups = Cfg::kEpiWarps / 4, kCW = 256 / kGroups;
    const int cg = ew >> 2;  // column group
    // two 4 KB buffers a warp, or a pair of warps
    uint8_t* bufs = staging + (KIND == kG8Gelu ? 4 * (cg >> 1) + quarter : ew) * 8192;
    const uint32_t acc_empty0 = map_to_rank(acc_empty, 0), shared_free0 = map_to_rank(shared_free, 0);
    uint32_t used = 0;  // staging buffers used so far
    int turn = 0;       // kG8Gelu: set of flags of this tile
    uint32_t rphase = 0;  // kG8F32: bit b: parity of buffer b's next residual load
    int abuf = 0;
    uint32_t aphase = 0;
    bool ok = true;
    for (long long t = pair; t < total && ok; t += n_pairs) {
      const int mt = (int)(t / n_tiles), nt = (int)(t % n_tiles);
      const bool live = pair_has_rows(mt);
      const int row0 = mt * 256 + (int)rank * 128 + quarter * 32;
      const int col0 = nt * 256 + cg * kCW;
      const int row = row0 + lane;
      const bool valid = row < p.M && (p.mask == nullptr || __ldg(p.mask + row) != 0);
      auto wait_acc = [&] {
        ok = mbar_wait_warp<true>(acc_full + abuf, aphase, p.err, kErrGemm8Epilogue);
        tc_fence_after();
        return ok;
      };
      auto acc_addr = [&] { return tmem_base + ((uint32_t)(quarter * 32) << 16) + abuf * Cfg::kAcc1 + cg * kCW; };
      auto free_shared = [&] {
        tc_fence_before();
        mbar_arrive_cluster_elect(shared_free0);
      };
      auto free_acc = [&] {
        tc_fence_before();
        mbar_arrive_cluster_elect(acc_empty0 + (uint32_t)(abuf * sizeof(uint64_t)));
        if (++abuf == 2) { abuf = 0; aphase ^= 1u; }
      };
      if constexpr (KIND == kG8Gelu) {
        uint64_t h[32];
        bias_pairs<64>(h, p.bias, col0, p.N);
        if (live) {
          for (int kb = 0; kb < kblocks; kb += kChunk) {
            if (!wait_acc()) break;
            const uint32_t taddr = acc_addr();
            // buffer 0 shares its last 32 columns (group 3's second piece),
            // buffer 1 its first (group 0's first)
            const bool swap = abuf == 0 && cg == 3;
            const bool mine = swap || (abuf == 1 && cg == 0);
            uint32_t r[32];
            tmem_ld32(taddr + (swap ? 32 : 0), r);
            tmem_ld_wait();
            if (mine) free_shared();
            if (swap) add_pairs(h + 16, r); else add_pairs(h, r);
            tmem_ld32(taddr + (swap ? 0 : 32), r);
            tmem_ld_wait();
            free_acc();
            if (swap) add_pairs(h, r); else add_pairs(h + 16, r);
          }
        }
        // the two warps of a block meet at a barrier of their own, and
        // exchange their maxima in the staging before the codes fill it.
        // Neither leaves alone, which would keep the other waiting for good:
        // they agree first that both their waits succeeded.
        float2* other = reinterpret_cast<float2*>(bufs);
        const int bar_id = 1 + (cg >> 1) * 4 + quarter;
        auto meet = [&] { asm volatile("bar.sync %0, 64;" ::"r"(bar_id) : "memory"); };
        volatile uint8_t* flags = agreed + 16 * turn;
        turn ^= 1;
        if (lane == 0) flags[ew] = ok ? 1 : 0;
        meet();
        ok = flags[ew] != 0 && flags[ew ^ 4] != 0;
        if (!ok) break;
        const int cb = nt * 256 + (cg >> 1) * 128;  // the block's first column
        if (row0 < p.M && cb < p.N) {
          uint32_t gbyte, hbyte;
          if ((cg & 1) == 0 && lane == 0) bulk_wait_read<0>();  // before the first meeting: the staging is free
          gelu_pack_row<64>(h, valid, bufs, bufs + 4096, 4 * (cg & 1), lane, gbyte, hbyte, [&](float& a, float& b) {
            meet();
            other[32 * (cg & 1) + lane] = make_float2(a, b);
            meet();
            const float2 o = other[32 * ((cg & 1) ^ 1) + lane];
            meet();
            a = fmaxf(a, o.x);
            b = fmaxf(b, o.y);
          });
          fence_async_smem();
          meet();
          if ((cg & 1) == 0) {
            if (lane == 0) {
              tma_store_2d(&tmOut, bufs, cb, row0);
              tma_store_2d(&tmAux, bufs + 4096, cb, row0);
              bulk_commit();
            }
            if (row < p.M) {
              const long long s = (long long)row * n_blocks(p.N) + cb / kBlk;
              p.g_scales[s] = (uint8_t)gbyte;
              p.h_scales[s] = (uint8_t)hbyte;
            }
          }
        }
      } else if constexpr (KIND == kG8F32) {
        // 128 columns as four 32-column (128-byte) pieces; the residual comes
        // into the staging buffers two pieces ahead of its use
        const int pieces = row0 < p.M ? max(0, min(4, (p.N - col0 + 31) / 32)) : 0;
        const bool fetch = p.has_resid && live;
        auto load_resid = [&](int c) {  // lane 0; its buffer's store has been read
          const uint32_t b = (used + c) & 1;
          mbar_expect_tx(res_full + 2 * ew + b, 4096);
          tma_load_2d(bufs + b * 4096, &tmAux, res_full + 2 * ew + b, col0 + 32 * c, row0);
        };
        if (fetch && lane == 0) {
          bulk_wait_read<0>();
          for (int c = 0; c < min(2, pieces); ++c) load_resid(c);
        }
        __syncwarp();
        float acc[128];
#pragma unroll
        for (int i = 0; i < 128; ++i) acc[i] = 0.f;
        if (live) {
          for (int kb = 0; kb < kblocks; kb += kChunk) {
            if (!wait_acc()) break;  // on to the residual's own waits, so that no load is in flight at the end
            const uint32_t taddr = acc_addr();
            uint32_t r[32];
            // buffer 0 shares its last 32 columns (group 1's last piece), buffer 1 its first
            const bool swap = abuf == 0 && cg == 1;
            const bool mine = swap || (abuf == 1 && cg == 0);
            auto add = [&](float* a) {
#pragma unroll
              for (int i = 0; i < 32; ++i) a[i] += __uint_as_float(r[i]);
            };
            if (swap) {
              tmem_ld32(taddr + 96, r);
              tmem_ld_wait();
              free_shared();
              add(acc + 96);
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              if (c == 3 && swap) continue;  // warp-uniform
              tmem_ld32(taddr + 32 * c, r);
              tmem_ld_wait();
              if (c == 0 && mine && !swap) free_shared();
              add(acc + 32 * c);
            }
            free_acc();
          }
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if (c < pieces) {
            const int col = col0 + 32 * c;
            const uint32_t b = (used + c) & 1;
            uint8_t* buf = bufs + b * 4096;
            if (fetch) {
              uint64_t* bar = res_full + 2 * ew + b;
              if (!mbar_wait_warp<true>(bar, (rphase >> b) & 1u, p.err, kErrGemm8Epilogue)) {
                ok = false;
                Drain().wait(bar, (rphase >> b) & 1u);
                __syncwarp();
              }
              rphase ^= 1u << b;
            } else {
              if (lane == 0) bulk_wait_read<1>();
              __syncwarp();
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              float4* dst = reinterpret_cast<float4*>(staged(buf, lane, j));
              float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
              if (valid) {
                o = make_float4(acc[32 * c + 4 * j], acc[32 * c + 4 * j + 1], acc[32 * c + 4 * j + 2],
                                acc[32 * c + 4 * j + 3]);
                if (p.bias != nullptr && col + 4 * j < p.N) {
                  const float4 bb = __ldg(reinterpret_cast<const float4*>(p.bias + col) + j);
                  o.x += bb.x; o.y += bb.y; o.z += bb.z; o.w += bb.w;
                }
                if (p.has_resid) {
                  const float4 rr = *dst;
                  o.x += rr.x; o.y += rr.y; o.z += rr.z; o.w += rr.w;
                }
              }
              *dst = o;
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_2d(&tmOut, buf, col, row0);
              bulk_commit();
              if (fetch && c + 2 < pieces) {
                bulk_wait_read<0>();
                load_resid(c + 2);
              }
            }
            __syncwarp();
          }
        }
        used += pieces;
      } else {
        if (live && !wait_acc()) break;
        const int cur = abuf;
        const uint32_t taddr = acc_addr();
        const bool mine = cg == (cur ^ 1);
        // two 64-column pieces, the one with the shared columns first
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int piece = cur == 0 && cg == 1 ? 1 - q : q;
          const int col = col0 + 64 * piece;
          uint32_t r[2][32];
          if (live) {
            tmem_ld32(taddr + 64 * piece, r[0]);
            tmem_ld32(taddr + 64 * piece + 32, r[1]);
            tmem_ld_wait();
            if (q == 0 && mine) free_shared();
            if (q == 1) free_acc();
          }
          if (row0 >= p.M || col >= p.N) continue;
          uint32_t w[32];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float* v = reinterpret_cast<float*>(r[c]);
            if (live) add_bias32(v, p.bias, col + 32 * c, p.N);
#pragma unroll
            for (int j = 0; j < 16; ++j)
              w[16 * c + j] = KIND == kG8F16 ? pack_half2(v[2 * j], v[2 * j + 1]) : pack_bf162(v[2 * j], v[2 * j + 1]);
          }
          uint8_t* buf = bufs + (used++ & 1) * 4096;
          if (lane == 0) bulk_wait_read<1>();  // the store of this buffer is the one before last
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 8; ++j)
            *reinterpret_cast<uint4*>(staged(buf, lane, j)) =
                valid ? make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]) : make_uint4(0, 0, 0, 0);
          fence_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&tmOut, buf, col, row0);
            bulk_commit();
          }
        }
      }
    }
    if (lane == 0) bulk_wait_all();
    __syncwarp();
  }
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  if (warp == 2) tmem_dealloc_pair(tmem_base, 512);
}

}  // namespace tj
