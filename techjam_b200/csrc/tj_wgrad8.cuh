// Weight and bias gradients of a linear layer from an 8-bit copy of its input:
//
//   dW[n, k] = sum over tokens t of dY[t, n] * X[t, k],   db[n] = sum over t of dY[t, n]
//
// dY is fp16 or bf16, X e4m3 codes with a scale per token and 128 columns.
// The scale runs along the summed dimension, so it cannot stay outside the
// product: X is restored to dY's type first (exact in bf16), by the unpacking
// kernel into the workspace.  Restoring it on the way into shared memory was
// built and measured too: each CTA then converts every code of its tile again
// for each 256 columns of dY, 20 pipe cycles for four bf16 values, and at
// 4096 x 1024 over 24.6k tokens that kernel took 276 us against 21 + 188.
// Both operands are token-major in memory, i.e. MN-major for the tensor core.
//
// A CTA pair computes a 256 x 256 tile (tcgen05.mma kind::f16, cta_group::2,
// FP32 accumulation): each CTA stages 128 columns of dY and of X by TMA, 32 KB
// for 512 cycles of MMA.  Tokens are split over CTA pairs when the tiles do
// not fill the GPU, and the parts summed in a fixed order.
//
// The tensor core truncates when it adds to the accumulator, about 6e-7 of
// the sum over 512 tokens and growing with their number, so each 512 tokens
// start a new accumulator, and the epilogue adds those up in registers.
//
//   warp 0       TMA loads                 warp 1   MMA issuer (even CTA)
//   warp 2       TMEM; clears masked tokens
//   warps 4-7    db, from global memory (L2: the tiles pass through it anyway)
//   warps 8-15   accumulators -> registers -> dW
//
// Masked tokens take no part whatever their dY and X hold: 64-token stages
// without a valid token are left out of the stage list; X was restored with
// zeros in masked rows, and in stages that have some warp 2 of each CTA clears
// their rows of dY's tile before the MMAs.  Only those stages go through
// threads: the others' loads signal the even CTA's barrier themselves.  (With
// every stage announced by a thread of the odd CTA, whose release at cluster
// scope waits for its SM's memory traffic, the kernel took 247 us instead of
// the 188 that it takes now.)
#pragma once
#include "tj_act8.cuh"
#include "tj_gemm8.cuh"

namespace tj {

constexpr int kWgTok = 64;     // tokens per stage
constexpr int kWgChunk = 8;    // stages per accumulator
constexpr int kWgStages = 7;
constexpr int kWgStageBytes = 2 * 64 * 128 * 2;  // 128 columns of dY and of X, 64 tokens, 16 bits
constexpr int kWgThreads = 512;
constexpr int kWgRegLaunch = 128;  // warpgroups with 48 + 112 + 2 * 176
constexpr int kWgSmemBytes = 1024 + kWgStages * kWgStageBytes + 512;

struct Wgrad8Params {
  long long T;  // tokens
  int N, K;
  const void* dy;         // [T, N]
  const uint8_t* mask;    // [T] or null
  const int* list;        // live stages: index, bit 31 set when some of its tokens are masked; null: all
  const int* n_list;
  int splits;
  float* dw;  // [splits][N, K]
  float* db;  // [splits * k_tiles][4][N] partial sums
  int* err;
};

// Stages of 64 tokens that hold a valid one, in order (256 threads).
TJ_DEV void wgrad8_list(const uint8_t* __restrict__ mask, long long T, int* __restrict__ list,
                        int* __restrict__ n_list) {
  __shared__ int s_warp[8];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int stages = (int)((T + kWgTok - 1) / kWgTok);
  int before = 0;
  for (int s0 = 0; s0 < stages; s0 += 256) {
    const int s = s0 + (int)threadIdx.x;
    int n = 0, full = 0;
    if (s < stages) {
      const long long t0 = (long long)s * kWgTok;
      full = (int)min((long long)kWgTok, T - t0);
      if (full == kWgTok && (reinterpret_cast<uintptr_t>(mask) & 15) == 0) {
        const uint4* m = reinterpret_cast<const uint4*>(mask + t0);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint4 v = m[q];
          n += (__popc(__vcmpne4(v.x, 0u)) + __popc(__vcmpne4(v.y, 0u)) + __popc(__vcmpne4(v.z, 0u)) +
                __popc(__vcmpne4(v.w, 0u))) >> 3;
        }
      } else {
#pragma unroll 8
        for (int i = 0; i < full; ++i) n += mask[t0 + i] != 0;
      }
    }
    const int live = n > 0 ? 1 : 0;
    const uint32_t vote = __ballot_sync(0xffffffffu, live);
    if (lane == 0) s_warp[w] = __popc(vote);
    __syncthreads();
    int at = before + __popc(vote & ((1u << lane) - 1u));
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const int c = s_warp[q];
      if (q < w) at += c;
      before += c;
    }
    if (live) list[at] = s | (n < full ? (int)0x80000000 : 0);
    __syncthreads();
  }
  if (threadIdx.x == 0) *n_list = before;
}

// Before the product: X restored to T (zeros in masked rows), and in one block
// more the stage list.  One launch for both: a launch is 3 us of a small call.
template <typename T>
__global__ void __launch_bounds__(256) wgrad8_prep_kernel(const uint8_t* __restrict__ codes,
                                                          const uint8_t* __restrict__ scales, long long rows, int cols,
                                                          const uint8_t* __restrict__ mask, T* __restrict__ out,
                                                          unsigned unpack_blocks, int* __restrict__ list,
                                                          int* __restrict__ n_list) {
  if (blockIdx.x == unpack_blocks) {
    wgrad8_list(mask, rows, list, n_list);
    return;
  }
  act8_unpack<T, true>(codes, scales, rows, cols, mask, out);
}

// After it: the first blocks add up the parts of dW (n values, a multiple of
// 4; out[i] = sum over s of in[s][i], in order), the others db's columns.
__global__ void __launch_bounds__(1024) wgrad8_finish_kernel(const float* __restrict__ in, int splits, long long n,
                                                             float* __restrict__ out, unsigned join_blocks,
                                                             const float* __restrict__ db_in, int db_rows, int db_n,
                                                             float* __restrict__ db) {
  if (blockIdx.x >= join_blocks) {
    column_sum(db_in, db_rows, db_n, db, db, db_n, blockIdx.x - join_blocks);
    return;
  }
  const long long i = 4 * ((long long)blockIdx.x * blockDim.x + threadIdx.x);
  if (i >= n) return;
  float4 a = *reinterpret_cast<const float4*>(in + i);
#pragma unroll 4
  for (int s = 1; s < splits; ++s) {
    const float4 b = *reinterpret_cast<const float4*>(in + (long long)s * n + i);
    a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
  }
  *reinterpret_cast<float4*>(out + i) = a;
}

template <typename T>
__global__ void __launch_bounds__(kWgThreads, 1)
    wgrad8_kernel(const __grid_constant__ CUtensorMap tmY, const __grid_constant__ CUtensorMap tmX,
                  const Wgrad8Params p) {
  constexpr int S = kWgStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S * kWgStageBytes);  // [S] both CTAs' tiles (even CTA's copy)
  uint64_t* a_full = full + S;      // [S] this CTA's tiles of a stage with masked tokens
  uint64_t* cleared = a_full + S;   // [S] and both CTAs have cleared them (even CTA's copy)
  uint64_t* empty = cleared + S;    // [S]
  uint64_t* acc_full = empty + S;     // [2]
  uint64_t* acc_empty = acc_full + 2; // [2] (even CTA's copy is the live one)
  uint64_t* drained = acc_empty + 2;  // every MMA is complete (even CTA's copy)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(full + i, 1);
      mbar_init(a_full + i, 1);
      mbar_init(cleared + i, 2);
      mbar_init(empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) { mbar_init(acc_full + i, 1); mbar_init(acc_empty + i, 16); }
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

  const int k_tiles = (p.K + 255) / 256;
  const int tiles = ((p.N + 255) / 256) * k_tiles;
  const int items = tiles * p.splits;
  const int n_live = p.list != nullptr ? *p.n_list : (int)((p.T + kWgTok - 1) / kWgTok);
  struct Item { int n0, k0, kt, split, s0, s1; };
  auto item_at = [&](int it) {
    Item r;
    r.split = it / tiles;
    const int tile = it - r.split * tiles;
    r.kt = tile % k_tiles;
    r.n0 = (tile / k_tiles) * 256 + (int)rank * 128;
    r.k0 = r.kt * 256;
    r.s0 = (int)((long long)n_live * r.split / p.splits);
    r.s1 = (int)((long long)n_live * (r.split + 1) / p.splits);
    return r;
  };

  if (warp < 4) {
    reg_dealloc<48>();
    if (warp == 0 && lane == 0) {
      // ---------------------------------------------------------- TMA producer
      tma_prefetch_desc(&tmY);
      tma_prefetch_desc(&tmX);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int it = pair; it < items && ok; it += n_pairs) {
        const Item im = item_at(it);
        for (int s = im.s0; s < im.s1; ++s) {
          const int entry = p.list != nullptr ? p.list[s] : s;
          const int t0 = (entry & 0x7fffffff) * kWgTok;
          if (!mbar_wait<true>(empty + stage, phase ^ 1u, p.err, kErrWgradProducer)) { ok = false; break; }
          uint8_t* sa = smem + stage * kWgStageBytes;
          const int k0 = im.k0 + (int)rank * 128;
          if (entry < 0) {
            mbar_expect_tx(a_full + stage, kWgStageBytes);
            tma_load_2d(sa, &tmY, a_full + stage, im.n0, t0);
            tma_load_2d(sa + 8192, &tmY, a_full + stage, im.n0 + 64, t0);
            tma_load_2d(sa + 16384, &tmX, a_full + stage, k0, t0);
            tma_load_2d(sa + 24576, &tmX, a_full + stage, k0 + 64, t0);
          } else {
            const uint32_t lb = pair_leader_bar(full + stage);
            if (rank == 0) mbar_expect_tx(full + stage, 2 * kWgStageBytes);
            tma_load_2d_pair(sa, &tmY, lb, im.n0, t0);
            tma_load_2d_pair(sa + 8192, &tmY, lb, im.n0 + 64, t0);
            tma_load_2d_pair(sa + 16384, &tmX, lb, k0, t0);
            tma_load_2d_pair(sa + 24576, &tmX, lb, k0 + 64, t0);
          }
          if (++stage == S) { stage = 0; phase ^= 1u; }
        }
      }
      // the loads signal the even CTA, but both learn when the MMAs have used them
      Drain().ring(empty, S, stage, phase);
    } else if (warp == 1 && rank == 0) {
      // ---------------------------------------------------------- MMA issuer
      constexpr uint32_t idesc =
          idesc_f16_f32(256, 256, true, true) | (std::is_same_v<T, __half> ? 0u : (1u << 7) | (1u << 10));
      int stage = 0, abuf = 0;
      uint32_t aphase = 0;
      uint32_t fbits = 0, cbits = 0;  // bit i: parity of the next use of full / cleared i
      bool ok = true;
      for (int it = pair; it < items && ok; it += n_pairs) {
        const Item im = item_at(it);
        int entry = p.list != nullptr && im.s0 < im.s1 ? p.list[im.s0] : 0;
        for (int s = im.s0; s < im.s1; ++s) {
          const bool first = (s - im.s0) % kWgChunk == 0;
          const int next = p.list != nullptr && s + 1 < im.s1 ? p.list[s + 1] : 0;
          if (first && !mbar_wait_warp<true>(acc_empty + abuf, aphase ^ 1u, p.err, kErrWgradMma)) { ok = false; break; }
          if (entry < 0) {
            if (!mbar_wait_cluster_warp(cleared + stage, (cbits >> stage) & 1u, p.err, kErrWgradMma)) { ok = false; break; }
            cbits ^= 1u << stage;
          } else {
            if (!mbar_wait_warp<true>(full + stage, (fbits >> stage) & 1u, p.err, kErrWgradMma)) { ok = false; break; }
            fbits ^= 1u << stage;
          }
          entry = next;
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * kWgStageBytes);
#pragma unroll
          for (int ks = 0; ks < kWgTok / 16; ++ks)
            umma_f16_ss_pair_elect(tmem_base + abuf * 256, smem_desc(sa + ks * 2048, 8192, 1024, 128),
                                   smem_desc(sa + 16384 + ks * 2048, 8192, 1024, 128), idesc, !(first && ks == 0));
          umma_commit_pair_both_elect(empty + stage);
          if (++stage == S) stage = 0;
          if ((s - im.s0) % kWgChunk == kWgChunk - 1 || s + 1 == im.s1) {
            umma_commit_pair_both_elect(acc_full + abuf);
            if (++abuf == 2) { abuf = 0; aphase ^= 1u; }
          }
        }
      }
      umma_commit_pair_elect(drained);
      Drain().wait(drained, 0);
      __syncwarp();
    } else if (warp == 2 && p.list != nullptr) {
      // ---------------------------------------------------------- masked tokens of dY's tile
      const uint32_t cleared0 = map_to_rank(cleared, 0);
      int stage = 0;
      uint32_t abits = 0;
      bool ok = true;
      for (int it = pair; it < items && ok; it += n_pairs) {
        const Item im = item_at(it);
        for (int s = im.s0; s < im.s1; ++s) {
          const int entry = p.list[s];
          if (entry < 0) {
            // the mask before the wait: the tile is then cleared as it lands,
            // stages before its MMAs
            const long long t0 = (long long)(entry & 0x7fffffff) * kWgTok;
            uint32_t out[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const long long t = t0 + 32 * h + lane;
              out[h] = __ballot_sync(0xffffffffu, t < p.T && __ldg(p.mask + t) == 0);
            }
            if (!mbar_wait_warp<true>(a_full + stage, (abits >> stage) & 1u, p.err, kErrWgradEdge)) { ok = false; break; }
            abits ^= 1u << stage;
            uint8_t* sa = smem + stage * kWgStageBytes;
#pragma unroll
            for (int h = 0; h < 2; ++h)
              for (uint32_t left = out[h]; left != 0; left &= left - 1) {  // 16 lanes clear a token's 256 bytes
                const int tok = 32 * h + __ffs(left) - 1;
                if (lane < 16) *reinterpret_cast<uint4*>(sa + (lane >> 3) * 8192 + tok * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
              }
            fence_async_smem();
            __syncwarp();
            mbar_arrive_cluster_release(cleared0 + (uint32_t)(stage * sizeof(uint64_t)));
          }
          if (++stage == S) stage = 0;
        }
      }
    }
  } else if (warp < 8) {
    // ------------------------------------------------------------ db
    // The tiles of one n share its sum: k tile kt takes the kt-th of every
    // k_tiles stages.  A thread has 8 columns of every eighth token.
    reg_dealloc<112>();
    const int c8 = threadIdx.x & 15, r8 = (threadIdx.x & 127) >> 4;
    for (int it = pair; it < items; it += n_pairs) {
      const Item im = item_at(it);
      const int n = im.n0 + 8 * c8;
      float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (n < p.N) {
        for (int s = im.s0 + im.kt; s < im.s1; s += k_tiles) {
          const int entry = p.list != nullptr ? p.list[s] : s;
          const long long t0 = (long long)(entry & 0x7fffffff) * kWgTok + r8;
          uint4 v[8];
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            const long long t = t0 + 8 * q;
            bool use = t < p.T;
            if (use && entry < 0) use = __ldg(p.mask + t) != 0;
            v[q] = use ? __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p.dy) + t * p.N + n)) : make_uint4(0, 0, 0, 0);
          }
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            const T* e = reinterpret_cast<const T*>(&v[q]);
#pragma unroll
            for (int j = 0; j < 8; ++j) sum[j] += to_f32<T>(e[j]);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 16);
      if (lane < 16 && n < p.N) {
        float* out = p.db + ((long long)(im.split * k_tiles + im.kt) * 4 + (warp - 4)) * p.N + n;
        *reinterpret_cast<float4*>(out) = make_float4(sum[0], sum[1], sum[2], sum[3]);
        *reinterpret_cast<float4*>(out + 4) = make_float4(sum[4], sum[5], sum[6], sum[7]);
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue
    reg_alloc<176>();
    const int ew = warp - 8, quarter = warp & 3, half = ew >> 2;
    const uint32_t acc_empty0 = map_to_rank(acc_empty, 0);
    int abuf = 0;
    uint32_t aphase = 0;
    bool ok = true;
    for (int it = pair; it < items && ok; it += n_pairs) {
      const Item im = item_at(it);
      float acc[128];
#pragma unroll
      for (int q = 0; q < 128; ++q) acc[q] = 0.f;
      for (int s = im.s0; s < im.s1; s += kWgChunk) {
        if (!mbar_wait_warp<true>(acc_full + abuf, aphase, p.err, kErrWgradEpilogue)) { ok = false; break; }
        tc_fence_after();
        const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + abuf * 256 + half * 128;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t r[32];
          tmem_ld32(taddr + 32 * c, r);
          tmem_ld_wait();
#pragma unroll
          for (int q = 0; q < 32; ++q) acc[32 * c + q] += __uint_as_float(r[q]);
        }
        tc_fence_before();
        mbar_arrive_cluster_elect(acc_empty0 + (uint32_t)(abuf * sizeof(uint64_t)));
        if (++abuf == 2) { abuf = 0; aphase ^= 1u; }
      }
      if (!ok) break;
      const int n = im.n0 + quarter * 32 + lane;
      const int c0 = im.k0 + half * 128;
      if (n < p.N) {
        float* row = p.dw + ((long long)im.split * p.N + n) * p.K;
#pragma unroll
        for (int q = 0; q < 32; ++q)
          if (c0 + 4 * q < p.K)
            *reinterpret_cast<float4*>(row + c0 + 4 * q) = make_float4(acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]);
      }
    }
  }
  __syncwarp();  // the loading thread's warp too is whole again at the aligned barrier
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  if (warp == 2) tmem_dealloc_pair(tmem_base, 512);
}

}  // namespace tj
