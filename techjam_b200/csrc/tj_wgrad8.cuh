// Weight and bias gradients of a linear layer from an 8-bit copy of its input:
//
//   dW[n, k] = sum over tokens t of dY[t, n] * X[t, k],   db[n] = sum over t of dY[t, n]
//
// dY is fp16 or bf16, X e4m3 codes with a scale per token and 128 columns.
// The scale runs along the summed dimension, so it cannot stay outside the
// product: X is restored to dY's type on the way into shared memory (exact in
// bf16) and multiplied by tcgen05.mma kind::f16 with FP32 accumulation.  Both
// operands are token-major in memory, i.e. MN-major for the tensor core.
//
// A CTA pair computes a 256 x 256 tile (cta_group::2): each CTA stages 128
// columns of dY (TMA) and restores 128 columns of X (one scale block), so a
// 64-token stage costs its shared memory 32 KB of writes and 32 KB of operand
// reads for 512 cycles of MMA; a single CTA's 128 x 256 tile would need 1.5
// times that and be bound by shared memory.  Tokens are split over CTA pairs
// when the tiles do not fill the GPU, and the parts summed in a fixed order.
//
// The tensor core truncates when it adds to the accumulator, about 6e-7 of
// the sum over 512 tokens and growing with their number, so each 512 tokens
// start a new accumulator, and the epilogue adds those up in registers.
//
//   warp 0       TMA loads of dY and codes     warp 1   MMA issuer (even CTA)
//   warps 4-11   X codes -> operand tile; db.  Two groups of four take the
//                stages in turn.  One scheduler has two of these warps, so what
//                they cost is instructions: the codes come by TMA (no addresses,
//                no edges), only the scale bytes by loads, two stages ahead
//   warps 1-3 of the odd CTA   tell the even CTA that a stage's operands are
//                ready.  That takes a release at cluster scope, which waits
//                for all of a warp's loads (about 1700 cycles): three warps
//                in turn that have none keep up, warps 4-11 would not
//   warp 2       TMEM                      warps 12-19  accumulators -> registers -> dW
//
// Masked tokens take no part whatever their dY and X hold: 64-token stages
// without a valid token are left out of the stage list, and in stages with
// some, warps 4-7 clear the masked tokens' rows of both operands.
#pragma once
#include "tj_act8.cuh"
#include "tj_gemm8.cuh"

namespace tj {

constexpr int kWgTok = 64;     // tokens per stage
constexpr int kWgChunk = 8;    // stages per accumulator
constexpr int kWgStages = 5;
constexpr int kWgStageBytes = 2 * 64 * 128 * 2 + 64 * 128;  // 128 columns of dY and of X in 16 bits, X's codes, 64 tokens
constexpr int kWgThreads = 640;
constexpr int kWgRegLaunch = 96;
constexpr int kWgSmemBytes = 1024 + kWgStages * kWgStageBytes + 512;

struct Wgrad8Params {
  long long T;  // tokens
  int N, K;
  const uint8_t* scales;  // [T, ceil(K / 128)]
  const uint8_t* mask;    // [T] or null
  const int* list;        // live stages: index, bit 31 set when some of its tokens are masked; null: all
  const int* n_list;
  int splits;
  float* dw;  // [splits][N, K]
  float* db;  // [splits * k_tiles][4][N] partial sums
  int* err;
};

// Stages of 64 tokens that hold a valid one, in order.  One block.
__global__ void __launch_bounds__(1024) wgrad8_list_kernel(const uint8_t* __restrict__ mask, long long T,
                                                           int* __restrict__ list, int* __restrict__ n_list) {
  __shared__ int s_warp[32];
  __shared__ int s_base;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  if (threadIdx.x == 0) s_base = 0;
  __syncthreads();
  const int stages = (int)((T + kWgTok - 1) / kWgTok);
  for (int s0 = 0; s0 < stages; s0 += blockDim.x) {
    const int s = s0 + threadIdx.x;
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
        for (int i = 0; i < full; ++i) n += mask[t0 + i] != 0;
      }
    }
    const int live = n > 0 ? 1 : 0;
    int incl = live;
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += u;
    }
    if (lane == 31) s_warp[w] = incl;
    __syncthreads();
    if (w == 0) {
      int v = s_warp[lane];
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      s_warp[lane] = v;
    }
    __syncthreads();
    const int at = s_base + incl - live + (w > 0 ? s_warp[w - 1] : 0);
    if (live) list[at] = s | (n < full ? (int)0x80000000 : 0);
    __syncthreads();
    if (threadIdx.x == blockDim.x - 1) s_base = at + live;
    __syncthreads();
  }
  if (threadIdx.x == 0) *n_list = s_base;
}

// out[i] = sum over s of in[s][i] for i < n (n a multiple of 4), in order.
__global__ void __launch_bounds__(256) wgrad8_join_kernel(const float* __restrict__ in, int splits, long long n,
                                                          float* __restrict__ out) {
  const long long i = 4 * ((long long)blockIdx.x * blockDim.x + threadIdx.x);
  if (i >= n) return;
  float4 a = *reinterpret_cast<const float4*>(in + i);
  for (int s = 1; s < splits; ++s) {
    const float4 b = *reinterpret_cast<const float4*>(in + (long long)s * n + i);
    a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
  }
  *reinterpret_cast<float4*>(out + i) = a;
}

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
  if (!mbar_wait_warp(bar, parity, err, site)) return false;
  return __all_sync(0xffffffffu, try_wait());  // complete: returns at once, with the acquire
}

// tcgen05.ld of 16 columns.
TJ_DEV void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

// 16 codes times 2^(byte-127) as 16 values of type T, two to a word.
//
// A code s eeee mmm is moved bit by bit into T's fields (bf16: exponent
// 0000eeee, fp16: 0eeee), which is its value times 2^-120 or 2^-8, subnormal
// codes included, and one multiplication by 2^(byte-127) times that constant
// gives the restored value: exact wherever T holds it.  Scales for which the
// factor is no normal number of T, and the NaN code, go through fp32.
// Measured in this kernel's place (8192 codes a stage): the conversions
// e4m3 -> f16 -> f32 -> T took 2000 cycles a stage with four warps.
template <typename T>
TJ_DEV void restore16(const uint4& c, uint32_t byte, uint32_t (&w)[8]) {
  constexpr bool kHalf = std::is_same_v<T, __half>;
  const uint32_t in[4] = {c.x, c.y, c.z, c.w};
  uint32_t nan = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) nan |= (in[i] & 0x7f7f7f7fu) + 0x01010101u;
  if ((nan & 0x80808080u) == 0u && byte <= 134u && (!kHalf || byte >= 105u)) {
    const uint32_t f = kHalf ? (byte - 104u) << 10 : (byte + 120u) << 7;
    const uint32_t f2 = f | (f << 16);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t t = __byte_perm(in[i >> 1], 0u, (i & 1) ? 0x3424 : 0x1404);  // codes in the high bytes
      const uint32_t v = (kHalf ? (t >> 1) & 0x3f803f80u : (t >> 4) & 0x07f007f0u) | (t & 0x80008000u);
      if constexpr (kHalf) asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(w[i]) : "r"(v), "r"(f2));
      else asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(w[i]) : "r"(v), "r"(f2));
    }
    return;
  }
  const float s = scale_value(byte);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float v[4];
    e4m3x4_value(in[i], s, v);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = to_f32<T>(from_f32_restored<T>(v[j]));
    w[2 * i] = kHalf ? pack_half2(v[0], v[1]) : pack_bf162(v[0], v[1]);
    w[2 * i + 1] = kHalf ? pack_half2(v[2], v[3]) : pack_bf162(v[2], v[3]);
  }
}

template <typename T>
__global__ void __launch_bounds__(kWgThreads, 1)
    wgrad8_kernel(const __grid_constant__ CUtensorMap tmY, const __grid_constant__ CUtensorMap tmX,
                  const Wgrad8Params p) {
  constexpr int S = kWgStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* a_full = reinterpret_cast<uint64_t*>(smem + S * kWgStageBytes);  // [S] this CTA's dY tile and codes landed
  uint64_t* full = a_full + S;        // [S] both CTAs' operands ready (in the even CTA: its four warps and the odd CTA's relay)
  uint64_t* b_full = full + S;        // [S] the odd CTA's operands ready
  uint64_t* empty = b_full + S;       // [S]
  uint64_t* acc_full = empty + S;     // [2]
  uint64_t* acc_empty = acc_full + 2; // [2] (even CTA's copy is the live one)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) { mbar_init(a_full + i, 1); mbar_init(full + i, 5); mbar_init(b_full + i, 4); mbar_init(empty + i, 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(acc_full + i, 1); mbar_init(acc_empty + i, 16); }
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
    reg_dealloc<32>();
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
          const int idx = p.list != nullptr ? (p.list[s] & 0x7fffffff) : s;
          if (!mbar_wait(empty + stage, phase ^ 1u, p.err, kErrWgradProducer)) { ok = false; break; }
          uint8_t* sa = smem + stage * kWgStageBytes;
          mbar_expect_tx(a_full + stage, 64 * 128 * 3);
          tma_load_2d(sa + 32768, &tmX, a_full + stage, im.k0 + (int)rank * kBlk, idx * kWgTok);
          tma_load_2d(sa, &tmY, a_full + stage, im.n0, idx * kWgTok);
          tma_load_2d(sa + 8192, &tmY, a_full + stage, im.n0 + 64, idx * kWgTok);
          if (++stage == S) { stage = 0; phase ^= 1u; }
        }
      }
      if (!ok) mbar_drain(a_full, S, stage, phase);
    } else if (warp == 1 && rank == 0) {
      // ---------------------------------------------------------- MMA issuer
      constexpr uint32_t idesc =
          idesc_f16_f32(256, 256, true, true) | (std::is_same_v<T, __half> ? 0u : (1u << 7) | (1u << 10));
      int stage = 0, abuf = 0;
      uint32_t phase = 0, aphase = 0;
      bool ok = true;
      for (int it = pair; it < items && ok; it += n_pairs) {
        const Item im = item_at(it);
        for (int s = im.s0; s < im.s1; ++s) {
          const bool first = (s - im.s0) % kWgChunk == 0;
          if (first && !mbar_wait_warp(acc_empty + abuf, aphase ^ 1u, p.err, kErrWgradMma)) { ok = false; break; }
          if (!mbar_wait_cluster_warp(full + stage, phase, p.err, kErrWgradMma)) { ok = false; break; }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * kWgStageBytes);
#pragma unroll
          for (int ks = 0; ks < kWgTok / 16; ++ks)
            umma_f16_ss_pair_elect(tmem_base + abuf * 256, smem_desc(sa + ks * 2048, 8192, 1024, 128),
                                   smem_desc(sa + 16384 + ks * 2048, 8192, 1024, 128), idesc, !(first && ks == 0));
          umma_commit_pair_both_elect(empty + stage);
          if (++stage == S) { stage = 0; phase ^= 1u; }
          if ((s - im.s0) % kWgChunk == kWgChunk - 1 || s + 1 == im.s1) {
            umma_commit_pair_both_elect(acc_full + abuf);
            if (++abuf == 2) { abuf = 0; aphase ^= 1u; }
          }
        }
      }
    }
    if (rank == 1 && warp >= 1) {
      // ---------------------------------------------------------- odd CTA's operands ready
      const uint32_t full0 = map_to_rank(full, 0);
      int stage = 0, turn = 1;
      uint32_t phase = 0;
      bool ok = true;
      for (int it = pair; it < items && ok; it += n_pairs) {
        const Item im = item_at(it);
        for (int s = im.s0; s < im.s1; ++s) {
          if (turn == warp) {
            if (!mbar_wait_warp(b_full + stage, phase, p.err, kErrWgradRestore)) { ok = false; break; }
            mbar_arrive_cluster_release(full0 + (uint32_t)(stage * sizeof(uint64_t)));
          }
          if (++turn == 4) turn = 1;
          if (++stage == S) { stage = 0; phase ^= 1u; }
        }
      }
    }
  } else if (warp < 12) {
    // ------------------------------------------------------------ X codes -> operand tile, db
    reg_dealloc<64>();
    const int grp = (warp - 4) >> 2;
    const int i = threadIdx.x & 127;
    const int kblocks = n_blocks(p.K);
    // pass j: token 16 j + tok0, codes 16 c16.. of the 64-column atom.  The 8
    // lanes of a shared-memory phase have tokens t and t ^ 5 with four pieces
    // each: bit 2 sends them to different halves of the codes' (swizzled) 128
    // bytes, bit 0 to even and odd pieces of the operand rows
    const int tok0 = (2 * (i >> 4)) ^ ((i & 4) ? 5 : 0);
    const int atom = (i >> 3) & 1;
    const int c16 = i & 3;
    const int sw = tok0 & 7;  // the same in every pass
    const uint32_t src = 32768 + tok0 * 128 + (((4 * atom + c16) ^ sw) << 4);
    const uint32_t dst0 = 16384 + atom * 8192 + tok0 * 128 + (((2 * c16) ^ sw) << 4);
    const uint32_t dst1 = 16384 + atom * 8192 + tok0 * 128 + (((2 * c16 + 1) ^ sw) << 4);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    int turn = 0;  // group of the next stage
    for (int it = pair; it < items && ok; it += n_pairs) {
      const Item im = item_at(it);
      const int blk = min(im.k0 / kBlk + (int)rank, kblocks - 1);  // past K the codes are zeros under any scale
      // db of columns 2 (i % 64) and the next over tokens 32 (i / 64)..+31 of
      // this group's stages that fall to this k tile: the tiles of one n share the sum
      float sum0 = 0.f, sum1 = 0.f;
      int mine = 0;  // stages of this group so far
      auto entry_at = [&](int s) { return s < im.s1 ? (p.list != nullptr ? p.list[s] : s) : 0; };
      // scale bytes of the four tokens of this thread (clamped past T, where the codes are zeros)
      auto scales_of = [&](int entry) {
        const int t0 = (entry & 0x7fffffff) * kWgTok + tok0, last = (int)p.T - 1;
        uint32_t w = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          w |= (uint32_t)__ldg(p.scales + (long long)min(t0 + 16 * j, last) * kblocks + blk) << (8 * j);
        return w;
      };
      int s = im.s0;
      if (turn != grp) {  // the other group takes the item's first stage
        ++s;
        if (++stage == S) { stage = 0; phase ^= 1u; }
      }
      int entry = entry_at(s), next = entry_at(s + 2);
      uint32_t bytes = scales_of(entry);
      for (; s < im.s1; s += 2) {
        uint8_t* sa = smem + stage * kWgStageBytes;
        const uint32_t bytes_next = scales_of(next);
        const int after = entry_at(s + 4);
        // the codes landed; their loads were issued when `empty` had completed
        if (!mbar_wait_warp(a_full + stage, phase, p.err, kErrWgradRestore)) { ok = false; break; }
        uint4 c[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) c[j] = *reinterpret_cast<const uint4*>(sa + src + 2048 * j);
        if (entry < 0) {
          // some tokens are masked: clear their codes and their rows of the dY tile
          const long long t0 = (long long)(entry & 0x7fffffff) * kWgTok;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const long long t = t0 + 16 * j + tok0;
            if (t >= p.T || __ldg(p.mask + t) == 0) c[j] = make_uint4(0, 0, 0, 0);
          }
          const int tok = i >> 1;
          if (t0 + tok < p.T && __ldg(p.mask + t0 + tok) == 0) {
            uint4* row = reinterpret_cast<uint4*>(sa + (i & 1) * 8192 + tok * 128);
#pragma unroll
            for (int q = 0; q < 8; ++q) row[q] = make_uint4(0, 0, 0, 0);
          }
          asm volatile("bar.sync %0, 128;" ::"r"(1 + grp) : "memory");
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t w[8];
          restore16<T>(c[j], (bytes >> (8 * j)) & 255u, w);
          *reinterpret_cast<uint4*>(sa + dst0 + 2048 * j) = make_uint4(w[0], w[1], w[2], w[3]);
          *reinterpret_cast<uint4*>(sa + dst1 + 2048 * j) = make_uint4(w[4], w[5], w[6], w[7]);
        }
        fence_async_smem();
        if (mine % k_tiles == im.kt) {  // this k tile's share of db
          const uint8_t* at = sa + ((i >> 5) & 1) * 8192 + (i & 3) * 4;
#pragma unroll 8
          for (int q = 0; q < 32; ++q) {
            const int tok = 32 * (i >> 6) + q;
            const uint32_t u = *reinterpret_cast<const uint32_t*>(at + tok * 128 + ((((i & 31) >> 2) ^ (tok & 7)) << 4));
            const T* v = reinterpret_cast<const T*>(&u);
            sum0 += to_f32<T>(v[0]);
            sum1 += to_f32<T>(v[1]);
          }
        }
        ++mine;
        __syncwarp();
        mbar_arrive_elect((rank == 0 ? full : b_full) + stage);
        entry = next;
        next = after;
        bytes = bytes_next;
        stage += 2;
        if (stage >= S) { stage -= S; phase ^= 1u; }
      }
      if (!ok) break;
      // leave stage, phase and turn where the next item starts: s is s1 or s1 + 1
      if (s > im.s1) {
        if (--stage < 0) { stage = S - 1; phase ^= 1u; }
      }
      turn ^= (im.s1 - im.s0) & 1;
      const int n = im.n0 + 2 * (i & 63);
      if (n < p.N)
        *reinterpret_cast<float2*>(p.db + ((long long)(im.split * k_tiles + im.kt) * 4 + grp * 2 + (i >> 6)) * p.N + n) =
            make_float2(sum0, sum1);
    }
  } else {
    // ------------------------------------------------------------ epilogue
    reg_alloc<160>();
    const int ew = warp - 12, quarter = warp & 3, half = ew >> 2;
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
        if (!mbar_wait_warp(acc_full + abuf, aphase, p.err, kErrWgradEpilogue)) { ok = false; break; }
        tc_fence_after();
        const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + abuf * 256 + half * 128;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          uint32_t r[16];
          tmem_ld16(taddr + 16 * c, r);
          tmem_ld_wait();
#pragma unroll
          for (int q = 0; q < 16; ++q) acc[16 * c + q] += __uint_as_float(r[q]);
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
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  if (warp == 2) tmem_dealloc_pair(tmem_base, 512);
}

}  // namespace tj
