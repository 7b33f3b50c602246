// C ABI of the 8-bit activation operators: packing and restoring, GELU's
// gradient (tj_act8.cuh), the block-scaled product (tj_gemm8.cuh) and the
// weight gradient (tj_wgrad8.cuh).
#include <algorithm>
#include <mutex>
#include <type_traits>

#include "tj.h"
#include "tj_host.h"
#include "tj_wgrad8.cuh"

namespace tj_host {
int set_train_wait_limit(unsigned long long ns) {
  TJH_CUDA(cudaMemcpyToSymbol(tj::g_tj_wait_ns, &ns, sizeof(ns)));
  return TJ_OK;
}
}  // namespace tj_host

namespace {

using tj_host::fail;

bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
bool plain(int dtype) { return dtype == TJ_F32 || dtype == TJ_F16 || dtype == TJ_BF16; }
size_t vec_bytes(int dtype) { return dtype == TJ_F32 ? 16 : 8; }
int blocks_of(int cols) { return (cols + tj::kBlk - 1) / tj::kBlk; }
constexpr int kMaxSize = 0x7fffff00;  // sizes up to here can be rounded up to a tile in an int

// CTAs for 8 lanes per 128-column block, 256 threads each.
int block_grid(long long rows, int cols, unsigned* grid) {
  if (rows < 0 || cols <= 0) return fail(TJ_ERR_INVALID, "rows %lld, columns %d", rows, cols);
  if (cols > kMaxSize || rows > 0x7fffffffLL * 32 / blocks_of(cols)) return fail(TJ_ERR_UNSUPPORTED, "too many blocks");
  *grid = (unsigned)((rows * blocks_of(cols) + 31) / 32);
  return TJ_OK;
}

template <typename T>
int pack_t(const void* x, long long rows, int cols, const uint8_t* mask, uint8_t* codes, uint8_t* scales, bool vec,
           unsigned grid, cudaStream_t st) {
  if (vec) tj::act8_pack_kernel<T, true><<<grid, 256, 0, st>>>(static_cast<const T*>(x), rows, cols, mask, codes, scales);
  else tj::act8_pack_kernel<T, false><<<grid, 256, 0, st>>>(static_cast<const T*>(x), rows, cols, mask, codes, scales);
  TJH_CUDA(cudaGetLastError());
  return TJ_OK;
}
template <typename T>
int unpack_t(const uint8_t* codes, const uint8_t* scales, long long rows, int cols, void* out, bool vec,
             unsigned grid, cudaStream_t st) {
  if (vec) tj::act8_unpack_kernel<T, true><<<grid, 256, 0, st>>>(codes, scales, rows, cols, static_cast<T*>(out));
  else tj::act8_unpack_kernel<T, false><<<grid, 256, 0, st>>>(codes, scales, rows, cols, static_cast<T*>(out));
  TJH_CUDA(cudaGetLastError());
  return TJ_OK;
}

struct GeluArgs {
  const void* dy;
  const void* h;
  const uint8_t* h_scales;
  long long rows;
  int cols;
  const uint8_t* mask;
  void* dh;
  uint8_t* codes;
  uint8_t* scales;
};
template <typename T, bool H8, bool PACK, bool VEC>
void gelu_launch(const GeluArgs& a, unsigned grid, cudaStream_t st) {
  tj::gelu_bwd_kernel<T, H8, PACK, VEC><<<grid, 256, 0, st>>>(static_cast<const T*>(a.dy), a.h, a.h_scales, a.rows, a.cols,
                                                              a.mask, static_cast<T*>(a.dh), a.codes, a.scales);
}
template <typename T>
int gelu_t(const GeluArgs& a, bool vec, unsigned grid, cudaStream_t st) {
  const bool h8 = a.h_scales != nullptr, pack = a.codes != nullptr;
  if (vec) {
    if (h8) { if (pack) gelu_launch<T, true, true, true>(a, grid, st); else gelu_launch<T, true, false, true>(a, grid, st); }
    else { if (pack) gelu_launch<T, false, true, true>(a, grid, st); else gelu_launch<T, false, false, true>(a, grid, st); }
  } else {
    if (h8) { if (pack) gelu_launch<T, true, true, false>(a, grid, st); else gelu_launch<T, true, false, false>(a, grid, st); }
    else { if (pack) gelu_launch<T, false, true, false>(a, grid, st); else gelu_launch<T, false, false, false>(a, grid, st); }
  }
  TJH_CUDA(cudaGetLastError());
  return TJ_OK;
}

// Opts a kernel in to its dynamic shared memory, once per device.
template <typename K>
int allow_smem(K kern, int bytes, int dev, bool (&done)[64], std::mutex& mu) {
  std::lock_guard<std::mutex> lock(mu);
  if (dev < 0 || dev >= 64) return fail(TJ_ERR_NO_DEVICE, "device index %d out of range", dev);
  if (!done[dev]) {
    TJH_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done[dev] = true;
  }
  return TJ_OK;
}

struct Gemm8Args {
  const void* a;
  const void* w;
  void* out;
  const void* aux_in;  // residual
  void* aux_out;       // GELU: codes of the input
};

template <int BN, int KIND>
int launch_gemm8(const Gemm8Args& g, const tj::Gemm8Params& p, int dev, int sms, cudaStream_t st) {
  using Cfg = tj::Gemm8Cfg<BN, KIND>;
  auto kern = tj::gemm8_kernel<BN, KIND>;
  static std::mutex mu;
  static bool done[64] = {};
  TJH_CHECK(allow_smem(kern, Cfg::kSmemBytes, dev, done, mu));
  CUtensorMap ta, tw, to, tx;
  TJH_CHECK(tj_host::make_map(&ta, g.a, 1, p.M, p.K, tj::kG8BM, 128));
  TJH_CHECK(tj_host::make_map(&tw, g.w, 1, p.N, p.K, BN, 128));
  constexpr int elt = KIND == tj::kG8Gelu ? 1 : (KIND == tj::kG8F32 ? 4 : 2);
  TJH_CHECK(tj_host::make_map(&to, g.out, elt, p.M, p.N, 32, 128 / elt));
  tx = to;
  if (KIND == tj::kG8Gelu) TJH_CHECK(tj_host::make_map(&tx, g.aux_out, 1, p.M, p.N, 32, 128));
  else if (g.aux_in != nullptr) TJH_CHECK(tj_host::make_map(&tx, g.aux_in, 4, p.M, p.N, 32, 32));
  const long long tiles = (long long)((p.M + tj::kG8BM - 1) / tj::kG8BM) * ((p.N + BN - 1) / BN);
  kern<<<(unsigned)std::min<long long>(tiles, sms), Cfg::kThreads, Cfg::kSmemBytes, st>>>(ta, tw, to, tx, p);
  TJH_CUDA(cudaGetLastError());
  return TJ_OK;
}

// CTA pairs that run at once, and the kernel's attributes, once per device.
template <typename K>
int cluster_pairs(K kern, cudaLaunchConfig_t cfg, int regs, int dev, int (&max_pairs)[64], std::mutex& mu, int* pairs) {
  std::lock_guard<std::mutex> lock(mu);
  if (dev < 0 || dev >= 64) return fail(TJ_ERR_NO_DEVICE, "device index %d out of range", dev);
  if (max_pairs[dev] == 0) {
    // The warpgroups' register budgets add up to what the launch gives; with
    // any other count an increase would wait for registers that nobody frees,
    // so refuse to launch.
    cudaFuncAttributes fa;
    TJH_CUDA(cudaFuncGetAttributes(&fa, kern));
    if (regs != 0 && fa.numRegs != regs)
      return fail(TJ_ERR_UNSUPPORTED, "kernel built with %d registers per thread, needs %d", fa.numRegs, regs);
    TJH_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)cfg.dynamicSmemBytes));
    cfg.gridDim = dim3(2);
    int n = 0;
    TJH_CUDA(cudaOccupancyMaxActiveClusters(&n, kern, &cfg));
    max_pairs[dev] = n > 0 ? n : 1;
  }
  *pairs = max_pairs[dev];
  return TJ_OK;
}
struct PairLaunch {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  PairLaunch(int threads, int smem, cudaStream_t st) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
};

template <int KIND>
int launch_gemm8_pair(const Gemm8Args& g, const tj::Gemm8Params& p, int dev, cudaStream_t st) {
  using Cfg = tj::Gemm8PairCfg<KIND>;
  auto kern = tj::gemm8_pair_kernel<KIND>;
  static std::mutex mu;
  static int max_pairs[64] = {};
  PairLaunch l(Cfg::kThreads, Cfg::kSmemBytes, st);
  int pairs = 0;
  TJH_CHECK(cluster_pairs(kern, l.cfg, KIND == tj::kG8Gelu || KIND == tj::kG8F32 ? Cfg::kRegLaunch : 0, dev, max_pairs, mu, &pairs));
  CUtensorMap ta, tw, to, tx;
  TJH_CHECK(tj_host::make_map(&ta, g.a, 1, p.M, p.K, 128, 128));
  TJH_CHECK(tj_host::make_map(&tw, g.w, 1, p.N, p.K, 128, 128));
  constexpr int elt = KIND == tj::kG8Gelu ? 1 : (KIND == tj::kG8F32 ? 4 : 2);
  TJH_CHECK(tj_host::make_map(&to, g.out, elt, p.M, p.N, 32, 128 / elt));
  tx = to;
  if (KIND == tj::kG8Gelu) TJH_CHECK(tj_host::make_map(&tx, g.aux_out, 1, p.M, p.N, 32, 128));
  else if (g.aux_in != nullptr) TJH_CHECK(tj_host::make_map(&tx, g.aux_in, 4, p.M, p.N, 32, 32));
  const long long tiles = (long long)((p.M + 255) / 256) * ((p.N + 255) / 256);
  l.cfg.gridDim = dim3(2 * (unsigned)std::min<long long>(tiles, pairs));
  TJH_CUDA(cudaLaunchKernelEx(&l.cfg, kern, ta, tw, to, tx, p));
  return TJ_OK;
}

int gemm8_params(tj::Gemm8Params* p, const void* a, const uint8_t* as, const void* w, const uint8_t* ws,
                 const float* bias, int m, int n, int k, const uint8_t* mask, int* err) {
  if (m < 0 || n <= 0 || k <= 0) return fail(TJ_ERR_INVALID, "product of [%d, %d] and [%d, %d]", m, k, n, k);
  if (m > kMaxSize || n > kMaxSize || k > kMaxSize) return fail(TJ_ERR_UNSUPPORTED, "product too large");
  if (!w || !ws || !err || (m > 0 && (!a || !as))) return fail(TJ_ERR_INVALID, "null argument");
  if (k % 16) return fail(TJ_ERR_UNSUPPORTED, "need k %% 16 == 0");
  if (bias != nullptr && !aligned(bias, 16)) return fail(TJ_ERR_INVALID, "bias not 16-byte aligned");
  p->M = m; p->N = n; p->K = k;
  p->kblocks = blocks_of(k);
  p->a_words = p->kblocks % 4 == 0 && aligned(as, 4);
  p->w_words = p->kblocks % 4 == 0 && aligned(ws, 4);
  p->a_scales = as; p->w_scales = ws; p->bias = bias; p->mask = mask; p->err = err;
  return TJ_OK;
}

template <int KIND>
int gemm8_kind(const Gemm8Args& g, const tj::Gemm8Params& p, int dev, int sms, cudaStream_t st) {
  // 256 x 256 tiles of CTA pairs once they fill the GPU.  A 32-bit result with
  // a short sum is bound by its bytes, and the single CTAs' deeper staging
  // moves them better (32768 x 4096 x 1024, residual: 261 us for 266; but
  // 32768 x 1024 x 4096: 184 for 158, and 16384 x 2048 x 2048: 108 for 103).
  const long long pair_tiles = (long long)((p.M + 255) / 256) * ((p.N + 255) / 256);
  if (2 * pair_tiles >= sms && (KIND != tj::kG8F32 || p.kblocks >= 16)) return launch_gemm8_pair<KIND>(g, p, dev, st);
  if constexpr (KIND != tj::kG8Gelu) {
    // few tiles: half as wide, so that twice as many SMs share the weight's bytes
    const long long tiles = (long long)((p.M + 127) / 128) * ((p.N + 127) / 128);
    if (2 * tiles <= sms) return launch_gemm8<64, KIND>(g, p, dev, sms, st);
  }
  return launch_gemm8<128, KIND>(g, p, dev, sms, st);
}

struct WgradPlan {
  int splits, k_tiles;
  size_t list, db, x, dw, bytes;  // offsets of the stage list, the db parts, the restored input and the dW parts
};
int wgrad_plan(long long rows, int n, int k, int sms, WgradPlan* w) {
  if (rows < 0 || n <= 0 || k <= 0) return fail(TJ_ERR_INVALID, "weight gradient of [%lld, %d] and [%lld, %d]", rows, n, rows, k);
  if (n % 8 || k % 16) return fail(TJ_ERR_UNSUPPORTED, "need n %% 8 == 0 and k %% 16 == 0");
  if (rows > 0x7fffffffLL || n > kMaxSize || k > kMaxSize) return fail(TJ_ERR_UNSUPPORTED, "weight gradient too large");
  const long long stages = (rows + tj::kWgTok - 1) / tj::kWgTok;
  w->k_tiles = (k + 255) / 256;
  const long long tiles = (long long)((n + 255) / 256) * w->k_tiles;
  const long long pairs = sms / 2;
  // parts of at least two stages, as many as still run at once (633 tokens,
  // 12 tiles: 15.7 us in 5 parts, 20.3 in 2)
  w->splits = (int)std::max<long long>(1, std::min((stages + 1) / 2, pairs / std::max<long long>(1, tiles)));
  auto up = [](size_t v) { return (v + 255) / 256 * 256; };
  w->list = 0;
  w->db = up(sizeof(int) * (size_t)(stages + 1));
  w->x = w->db + up(sizeof(float) * 4 * (size_t)n * w->splits * w->k_tiles);
  w->dw = w->x + up(2 * (size_t)rows * (size_t)k);
  w->bytes = w->dw + (w->splits > 1 ? sizeof(float) * (size_t)n * k * w->splits : 0);
  return TJ_OK;
}

template <typename T>
int launch_wgrad8(const void* dy, const void* x, const tj::Wgrad8Params& p, int dev, int sms, cudaStream_t st) {
  auto kern = tj::wgrad8_kernel<T>;
  static std::mutex mu;
  static int max_pairs[64] = {};
  PairLaunch l(tj::kWgThreads, tj::kWgSmemBytes, st);
  int pairs = 0;
  TJH_CHECK(cluster_pairs(kern, l.cfg, tj::kWgRegLaunch, dev, max_pairs, mu, &pairs));
  CUtensorMap ty, tx;
  TJH_CHECK(tj_host::make_map(&ty, dy, 2, p.T, p.N, tj::kWgTok, 64));
  TJH_CHECK(tj_host::make_map(&tx, x, 2, p.T, p.K, tj::kWgTok, 64));
  const long long items = (long long)((p.N + 255) / 256) * ((p.K + 255) / 256) * p.splits;
  l.cfg.gridDim = dim3(2 * (unsigned)std::min<long long>(items, pairs));
  TJH_CUDA(cudaLaunchKernelEx(&l.cfg, kern, ty, tx, p));
  return TJ_OK;
}

}  // namespace

extern "C" {

int tj_act8_pack(const void* x, int dtype, long long rows, int cols, const uint8_t* mask, void* codes,
                 uint8_t* scales, void* stream) {
  unsigned grid;
  TJH_CHECK(block_grid(rows, cols, &grid));
  if (!plain(dtype)) return fail(TJ_ERR_INVALID, "unknown dtype %d", dtype);
  if (rows == 0) return TJ_OK;
  if (!x || !codes || !scales) return fail(TJ_ERR_INVALID, "null argument");
  const bool vec = cols % 4 == 0 && aligned(x, vec_bytes(dtype)) && aligned(codes, 4);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* c = static_cast<uint8_t*>(codes);
  switch (dtype) {
    case TJ_F32: return pack_t<float>(x, rows, cols, mask, c, scales, vec, grid, st);
    case TJ_F16: return pack_t<__half>(x, rows, cols, mask, c, scales, vec, grid, st);
    default: return pack_t<__nv_bfloat16>(x, rows, cols, mask, c, scales, vec, grid, st);
  }
}

int tj_act8_unpack(const void* codes, const uint8_t* scales, long long rows, int cols, void* out, int dtype,
                   void* stream) {
  unsigned grid;
  TJH_CHECK(block_grid(rows, cols, &grid));
  if (!plain(dtype)) return fail(TJ_ERR_INVALID, "unknown dtype %d", dtype);
  if (rows == 0) return TJ_OK;
  if (!out || !codes || !scales) return fail(TJ_ERR_INVALID, "null argument");
  const bool vec = cols % 4 == 0 && aligned(out, vec_bytes(dtype)) && aligned(codes, 4);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const uint8_t* c = static_cast<const uint8_t*>(codes);
  switch (dtype) {
    case TJ_F32: return unpack_t<float>(c, scales, rows, cols, out, vec, grid, st);
    case TJ_F16: return unpack_t<__half>(c, scales, rows, cols, out, vec, grid, st);
    default: return unpack_t<__nv_bfloat16>(c, scales, rows, cols, out, vec, grid, st);
  }
}

int tj_weight8_pack(const void* w, int dtype, int n, int k, int transpose, void* codes, uint8_t* scales,
                    void* stream) {
  if (n <= 0 || k <= 0) return fail(TJ_ERR_INVALID, "weight [%d, %d]", n, k);
  if (!plain(dtype)) return fail(TJ_ERR_INVALID, "unknown dtype %d", dtype);
  if (!w || !codes || !scales) return fail(TJ_ERR_INVALID, "null argument");
  if (k > kMaxSize || n > 65535 * tj::kBlk) return fail(TJ_ERR_UNSUPPORTED, "weight [%d, %d] too large", n, k);
  const dim3 grid(blocks_of(k), blocks_of(n));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* c = static_cast<uint8_t*>(codes);
#define TJ_WPACK(T)                                                                                                  \
  if (transpose) tj::weight8_pack_kernel<T, true><<<grid, 256, 0, st>>>(static_cast<const T*>(w), n, k, c, scales); \
  else tj::weight8_pack_kernel<T, false><<<grid, 256, 0, st>>>(static_cast<const T*>(w), n, k, c, scales);
  switch (dtype) {
    case TJ_F32: TJ_WPACK(float) break;
    case TJ_F16: TJ_WPACK(__half) break;
    default: TJ_WPACK(__nv_bfloat16) break;
  }
#undef TJ_WPACK
  TJH_CUDA(cudaGetLastError());
  return TJ_OK;
}

int tj_gelu_backward(const void* dy, int dtype, const void* h, const uint8_t* h8_scales, long long rows, int cols,
                     const uint8_t* mask, void* dh, void* dh8_codes, uint8_t* dh8_scales, void* stream) {
  unsigned grid;
  TJH_CHECK(block_grid(rows, cols, &grid));
  if (!plain(dtype)) return fail(TJ_ERR_INVALID, "unknown dtype %d", dtype);
  if ((dh8_codes == nullptr) != (dh8_scales == nullptr)) return fail(TJ_ERR_INVALID, "an 8-bit tensor needs its codes and its scales");
  if (rows == 0) return TJ_OK;
  if (!dy || !h || !dh) return fail(TJ_ERR_INVALID, "null argument");
  const bool vec = cols % 4 == 0 && aligned(dy, vec_bytes(dtype)) && aligned(dh, vec_bytes(dtype)) &&
                   aligned(h, h8_scales ? 4 : vec_bytes(dtype)) && aligned(dh8_codes, 4);
  const GeluArgs a{dy, h, h8_scales, rows, cols, mask, dh, static_cast<uint8_t*>(dh8_codes), dh8_scales};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case TJ_F32: return gelu_t<float>(a, vec, grid, st);
    case TJ_F16: return gelu_t<__half>(a, vec, grid, st);
    default: return gelu_t<__nv_bfloat16>(a, vec, grid, st);
  }
}

int tj_gemm8(const void* a, const uint8_t* a_scales, const void* w, const uint8_t* w_scales, const float* bias, int m,
             int n, int k, const uint8_t* mask, const float* resid, void* out, int out_dtype, int* err, void* stream) {
  tj::Gemm8Params p{};
  TJH_CHECK(gemm8_params(&p, a, a_scales, w, w_scales, bias, m, n, k, mask, err));
  if (!plain(out_dtype)) return fail(TJ_ERR_INVALID, "unknown dtype %d", out_dtype);
  if (resid != nullptr && out_dtype != TJ_F32) return fail(TJ_ERR_UNSUPPORTED, "a residual needs a 32-bit result");
  if (n % 8) return fail(TJ_ERR_UNSUPPORTED, "need n %% 8 == 0");
  if (m == 0) return TJ_OK;
  if (!out) return fail(TJ_ERR_INVALID, "null argument");
  int dev, sms;
  TJH_CHECK(tj_host::device(&dev, &sms));
  p.has_resid = resid != nullptr;
  const Gemm8Args g{a, w, out, resid, nullptr};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (out_dtype) {
    case TJ_F32: return gemm8_kind<tj::kG8F32>(g, p, dev, sms, st);
    case TJ_F16: return gemm8_kind<tj::kG8F16>(g, p, dev, sms, st);
    default: return gemm8_kind<tj::kG8BF16>(g, p, dev, sms, st);
  }
}

int tj_gemm8_gelu(const void* a, const uint8_t* a_scales, const void* w, const uint8_t* w_scales, const float* bias,
                  int m, int n, int k, const uint8_t* mask, void* g_codes, uint8_t* g_scales, void* h_codes,
                  uint8_t* h_scales, int* err, void* stream) {
  tj::Gemm8Params p{};
  TJH_CHECK(gemm8_params(&p, a, a_scales, w, w_scales, bias, m, n, k, mask, err));
  if (n % 16) return fail(TJ_ERR_UNSUPPORTED, "need n %% 16 == 0");
  if (m == 0) return TJ_OK;
  if (!g_codes || !g_scales || !h_codes || !h_scales) return fail(TJ_ERR_INVALID, "null argument");
  int dev, sms;
  TJH_CHECK(tj_host::device(&dev, &sms));
  p.g_scales = g_scales;
  p.h_scales = h_scales;
  const Gemm8Args g{a, w, g_codes, nullptr, h_codes};
  return gemm8_kind<tj::kG8Gelu>(g, p, dev, sms, static_cast<cudaStream_t>(stream));
}

int tj_wgrad8_workspace_bytes(long long rows, int n, int k, size_t* bytes) {
  if (!bytes) return fail(TJ_ERR_INVALID, "null argument");
  int dev, sms;
  TJH_CHECK(tj_host::device(&dev, &sms));
  WgradPlan w;
  TJH_CHECK(wgrad_plan(rows, n, k, sms, &w));
  *bytes = w.bytes;
  return TJ_OK;
}

int tj_wgrad8(const void* dy, int dtype, const void* x8_codes, const uint8_t* x8_scales, long long rows, int n, int k,
              const uint8_t* mask, float* dw, float* db, void* workspace, size_t workspace_bytes, int* err,
              void* stream) {
  if (dtype != TJ_F16 && dtype != TJ_BF16) return fail(TJ_ERR_UNSUPPORTED, "dy must be fp16 or bf16");
  int dev, sms;
  TJH_CHECK(tj_host::device(&dev, &sms));
  WgradPlan w;
  TJH_CHECK(wgrad_plan(rows, n, k, sms, &w));
  if (!dw || !db || !err || (rows > 0 && (!dy || !x8_codes || !x8_scales))) return fail(TJ_ERR_INVALID, "null argument");
  if (!aligned(x8_codes, 16) || !aligned(dw, 16)) return fail(TJ_ERR_INVALID, "tensor not 16-byte aligned");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (rows == 0) {
    TJH_CUDA(cudaMemsetAsync(dw, 0, sizeof(float) * (size_t)n * k, st));
    TJH_CUDA(cudaMemsetAsync(db, 0, sizeof(float) * (size_t)n, st));
    return TJ_OK;
  }
  if (!workspace || workspace_bytes < w.bytes || !aligned(workspace, 16))
    return fail(TJ_ERR_INVALID, "workspace of %zu bytes, needs %zu (16-byte aligned)", workspace_bytes, w.bytes);
  uint8_t* base = static_cast<uint8_t*>(workspace);
  tj::Wgrad8Params p{};
  p.T = rows; p.N = n; p.K = k;
  p.dy = dy;
  p.mask = mask;
  p.splits = w.splits;
  p.dw = w.splits > 1 ? reinterpret_cast<float*>(base + w.dw) : dw;
  p.db = reinterpret_cast<float*>(base + w.db);
  p.err = err;
  int* list = mask != nullptr ? reinterpret_cast<int*>(base + w.list) : nullptr;
  if (list != nullptr) {
    p.list = list + 1;
    p.n_list = list;
  }
  unsigned grid;
  TJH_CHECK(block_grid(rows, k, &grid));
  const unsigned blocks = grid + (list != nullptr ? 1u : 0u);
  const uint8_t* codes = static_cast<const uint8_t*>(x8_codes);
  if (dtype == TJ_F16) {
    tj::wgrad8_prep_kernel<__half><<<blocks, 256, 0, st>>>(codes, x8_scales, rows, k, mask, reinterpret_cast<__half*>(base + w.x),
                                                           grid, list ? list + 1 : nullptr, list);
    TJH_CUDA(cudaGetLastError());
    TJH_CHECK(launch_wgrad8<__half>(dy, base + w.x, p, dev, sms, st));
  } else {
    tj::wgrad8_prep_kernel<__nv_bfloat16><<<blocks, 256, 0, st>>>(
        codes, x8_scales, rows, k, mask, reinterpret_cast<__nv_bfloat16*>(base + w.x), grid, list ? list + 1 : nullptr, list);
    TJH_CUDA(cudaGetLastError());
    TJH_CHECK(launch_wgrad8<__nv_bfloat16>(dy, base + w.x, p, dev, sms, st));
  }
  const long long total = (long long)n * k;
  const unsigned join = w.splits > 1 ? (unsigned)((total / 4 + 1023) / 1024) : 0u;
  tj::wgrad8_finish_kernel<<<join + (n + 7) / 8, 1024, 0, st>>>(p.dw, w.splits, total, dw, join, p.db,
                                                                4 * w.splits * w.k_tiles, n, db);
  TJH_CUDA(cudaGetLastError());
  return TJ_OK;
}

}  // extern "C"
