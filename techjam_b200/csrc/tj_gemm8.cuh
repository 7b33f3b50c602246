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
// therefore starts a new accumulator after each 1024 of K, and the epilogue
// adds them up in registers, rounded to nearest.
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
  int has_resid;            // kG8F32: resid through its tensor map
  uint8_t* g_scales;        // kG8Gelu: [M, ceil(N / 128)]
  uint8_t* h_scales;
  int* err;
};

constexpr int kG8BM = 128;
constexpr int kG8Chunk = 8;  // kG8F32: K blocks per accumulator

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

// Four bytes of a scale row from block b0 on (byte loads: rows start anywhere); past the end 2^0.
TJ_DEV uint32_t scale_word(const uint8_t* row, int b0, int blocks) {
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
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(res_full + (KIND == kG8F32 ? Cfg::kEpiWarps * Cfg::kBufs : 0));
  static_assert((2 * S + 4 + 2 * SF + 32) * 8 + 4 <= 512, "barrier space");

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) { mbar_init(full + i, 1); mbar_init(empty + i, 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(acc_full + i, 1); mbar_init(acc_empty + i, Cfg::kEpiWarps); }
    for (int i = 0; i < SF; ++i) { mbar_init(sf_full + i, 4); mbar_init(sf_empty + i, 1); }
    if constexpr (KIND == kG8F32)
      for (int i = 0; i < Cfg::kEpiWarps * Cfg::kBufs; ++i) mbar_init(res_full + i, 1);
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
  constexpr int kChunk = KIND == kG8F32 ? kG8Chunk : 1 << 30;  // K blocks per accumulator

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
        if (!mbar_wait_warp(empty + stage, phase ^ 1u, p.err, kErrGemm8Producer)) { ok = false; break; }
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
    if (!ok && lane == 0) mbar_drain(full, S, stage, phase);
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
          if (!mbar_wait_warp(acc_empty + abuf, aphase ^ 1u, p.err, kErrGemm8Mma)) { ok = false; break; }
        }
        if ((kb & 3) == 0) {
          if (!mbar_wait_warp(sf_full + slot, sphase, p.err, kErrGemm8Mma)) { ok = false; break; }
        }
        if (!mbar_wait_warp(full + stage, phase, p.err, kErrGemm8Mma)) { ok = false; break; }
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
      for (int kb = 0; kb < kblocks; kb += 4) {
        uint32_t a[4], b[BN / 32];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int row = mt * kG8BM + 32 * c + lane;
          a[c] = row < p.M ? scale_word(p.a_scales + (long long)row * kblocks, kb, kblocks) : 0x7f7f7f7fu;
        }
        b[0] = scale_word(wrow, kb, kblocks);
#pragma unroll
        for (int c = 1; c < BN / 32; ++c) b[c] = b[0];
        if (!mbar_wait_warp(sf_empty + slot, sphase ^ 1u, p.err, kErrGemm8Scales)) { ok = false; break; }
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
        ok = mbar_wait_warp(acc_full + abuf, aphase, p.err, kErrGemm8Epilogue);
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
              if (!mbar_wait_warp(bar, (rphase >> b) & 1u, p.err, kErrGemm8Epilogue)) {
                ok = false;
                mbar_drain(bar, 1, 1, (rphase >> b) & 1u);
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
        // GELU: this warp's 128 columns are one block of g = gelu(h) and of
        // h = acc + bias, and a thread holds a whole row of it.  First pass
        // over the accumulator: the two maxima.  Second: the codes.
        float hmax = 0.f, hpos = 0.f, gmax = 0.f;
        const bool store = row0 < p.M && col0 < p.N;
        uint8_t* bufg = bufs + (used % Cfg::kBufs) * 4096;
        uint8_t* bufh = bufs + ((used + 1) % Cfg::kBufs) * 4096;
        auto load_h = [&](int c, float (&h)[32]) {
          uint32_t r[32];
          tmem_ld32(taddr + abuf * BN + 32 * c, r);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            float4 bb = make_float4(0.f, 0.f, 0.f, 0.f);
            if (p.bias != nullptr && col0 + 32 * c + 4 * j < p.N)
              bb = __ldg(reinterpret_cast<const float4*>(p.bias + col0 + 32 * c) + j);
            h[4 * j] = __uint_as_float(r[4 * j]) + bb.x;
            h[4 * j + 1] = __uint_as_float(r[4 * j + 1]) + bb.y;
            h[4 * j + 2] = __uint_as_float(r[4 * j + 2]) + bb.z;
            h[4 * j + 3] = __uint_as_float(r[4 * j + 3]) + bb.w;
          }
        };
        uint32_t gbyte = 127u, hbyte = 127u;
        if (live) {
          if (!wait_acc()) break;
          for (int c = 0; c < 4; ++c) {
            float h[32];
            load_h(c, h);
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const float a = finite_abs(h[i]);
              hmax = fmaxf(hmax, a);
              if (h[i] > 0.f) hpos = fmaxf(hpos, a);
            }
          }
          // gelu grows with h > 0 and its dip for h < 0 is 0.17 deep, which
          // gelu(0.3) exceeds: above that the largest |g| is gelu(hpos)
          gmax = gelu_erf_x2(hpos, 0.f).x;
          if (__any_sync(0xffffffffu, hpos < 0.3f)) {
            for (int c = 0; c < 4; ++c) {
              float h[32];
              load_h(c, h);
#pragma unroll
              for (int i = 0; i < 32; i += 2) {
                const float2 g = gelu_erf_x2(h[i], h[i + 1]);
                gmax = fmaxf(gmax, fmaxf(finite_abs(g.x), finite_abs(g.y)));
              }
            }
          }
          gbyte = valid ? scale_byte(gmax) : 127u;
          hbyte = valid ? scale_byte(hmax) : 127u;
        }
        if (store) {
          if (lane == 0) bulk_wait_read<2>();
          __syncwarp();
        }
        const float ginv = scale_inv(gbyte), hinv = scale_inv(hbyte);
        for (int c = 0; c < 4; ++c) {
          uint32_t gw[8], hw[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) gw[i] = hw[i] = 0u;
          if (live) {
            float h[32];
            load_h(c, h);
            if (c == 3) free_acc();
            if (valid) {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const float2 g0 = gelu_erf_x2(h[4 * i], h[4 * i + 1]), g1 = gelu_erf_x2(h[4 * i + 2], h[4 * i + 3]);
                gw[i] = e4m3x2<true>(g0.x, g0.y, ginv) | (e4m3x2<true>(g1.x, g1.y, ginv) << 16);
                hw[i] = e4m3x2<true>(h[4 * i], h[4 * i + 1], hinv) | (e4m3x2<true>(h[4 * i + 2], h[4 * i + 3], hinv) << 16);
              }
            }
          }
          if (store) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              *reinterpret_cast<uint4*>(staged(bufg, lane, 2 * c + j)) =
                  make_uint4(gw[4 * j], gw[4 * j + 1], gw[4 * j + 2], gw[4 * j + 3]);
              *reinterpret_cast<uint4*>(staged(bufh, lane, 2 * c + j)) =
                  make_uint4(hw[4 * j], hw[4 * j + 1], hw[4 * j + 2], hw[4 * j + 3]);
            }
          }
        }
        if (store) {
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
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 2) tmem_dealloc(tmem_base, Cfg::kTmemCols);
}

}  // namespace tj
