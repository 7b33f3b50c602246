// Layer norm for training: the forward pass that keeps its statistics (and,
// on request, an 8-bit copy of its input or output), and the backward pass
// with the reduction of the weight's and bias's gradients.
//
//   y  = xhat * gamma + beta,        xhat = (x - mean) * rstd
//   g  = dy * gamma
//   dx = rstd * (g - sum(g)/d - xhat * sum(g xhat)/d)  [+ resid]
//   dgamma = sum over rows of dy * xhat,  dbeta = sum over rows of dy
//
// Bound by HBM: every row is read once and written once, and held in
// registers in between.  WR warps share a row: each has 1024 of its columns
// forward, and 512 backward, where x, dy, the residual's gradient and the
// lane's share of dgamma and dbeta take five registers a column (1024 a warp
// spilled at 168 registers; see norm_bwd_kernel).  Columns are laid out as in tj_act8.cuh: a
// 128-column block belongs to 8 lanes.  Rows whose mask byte is 0 are not
// read: they leave zeros in every output and nothing in the sums.
#pragma once
#include "tj_act8.cuh"

namespace tj {

// First column of this lane's block in step i of the warp's 1024 columns.
TJ_DEV int norm_blk(int lane, int i) { return 512 * i + 128 * (lane >> 3); }
// Column of element e of its piece j there.
template <bool VEC>
TJ_DEV int norm_col(int lane, int i, int j, int e) { return piece_col<VEC>(norm_blk(lane, i), lane & 7, j, e); }

// Sum of N values over the WR warps of a row, WARPS warps in the CTA, whose
// rows run in step when WR > 1.  Every warp gets the same bits.  smem holds two
// sets, used in turn (`turn` flips): with one barrier between, a set is
// written again only after every warp has read it.
template <int WARPS, int WR, int N>
TJ_DEV void row_sum(float (&v)[N], float (*smem)[WARPS * N], int& turn, int warp, int lane) {
#pragma unroll
  for (int n = 0; n < N; ++n) v[n] = warp_sum(v[n]);
  if constexpr (WR > 1) {
    float* set = smem[turn];
    turn ^= 1;
    if (lane == 0)
#pragma unroll
      for (int n = 0; n < N; ++n) set[warp * N + n] = v[n];
    __syncthreads();
    const int w0 = warp - warp % WR;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < WR; ++w) s += set[(w0 + w) * N + n];
      v[n] = s;
    }
  }
}

constexpr int kNormWarps = 4;    // warps per CTA forward, and backward up to 2048 columns
// Warps per CTA and CTAs per SM backward: 16 warps of up to 128 registers.
constexpr int norm_bwd_warps(int wr) { return wr > kNormWarps ? wr : kNormWarps; }
constexpr int norm_bwd_ctas(int wr) { return 16 / norm_bwd_warps(wr); }

struct NormFwdParams {
  const void* x;
  const float* gamma;
  const float* beta;
  const uint8_t* mask;
  void* y;
  uint8_t* y_scales;  // y in 8 bits
  float* mean;
  float* rstd;
  uint8_t* x_codes;  // 8-bit copy of x, or null
  uint8_t* x_scales;
  long long rows;
  int d;
  float eps;
};

// CTAs per SM forward.  What hides the loads is rows in flight: 32768 x 1024
// fp32 to fp16, padded, took 41, 35 and 32 us with 4, 6 and 8; packing and the
// scalar loads need the registers of 6 (48 us to 8 bits with a copy of x, 49
// with 8).  To 8 bits with a copy of x the ALU pipe, which takes packing's
// maxima and conversions, is busy 64% of the time and 69% of the issue slots
// are taken, at 3.3 TB/s.
template <typename Y>
constexpr int norm_fwd_ctas(bool vec) { return std::is_same_v<Y, uint8_t> || !vec ? 6 : 8; }

// NI: 512-column steps per warp (1 or 2).
template <typename T, typename Y, int WR, int NI, bool VEC>
__global__ void __launch_bounds__(32 * kNormWarps, norm_fwd_ctas<Y>(VEC)) norm_fwd_kernel(const NormFwdParams p) {
  __shared__ float s_red[2][kNormWarps];
  int red = 0;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * (kNormWarps / WR) + warp / WR;
  const int base = (warp % WR) * 1024;
  const bool in = row < p.rows;
  const bool valid = in && (p.mask == nullptr || p.mask[row] != 0);
  const int d = p.d, lim = valid ? d : 0;
  const long long at = in ? row * d : 0;
  float v[NI][4][4];
  float sum[1] = {0.f};
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      load4<T, VEC>(static_cast<const T*>(p.x) + at, base + norm_blk(lane, i), lane & 7, j, lim, v[i][j]);
      sum[0] += (v[i][j][0] + v[i][j][1]) + (v[i][j][2] + v[i][j][3]);
    }
  row_sum<kNormWarps, WR, 1>(sum, s_red, red, warp, lane);
  const float mean = sum[0] / d;
  float sq[1] = {0.f};
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float c = v[i][j][e] - mean;
        if (base + norm_col<VEC>(lane, i, j, e) < lim) sq[0] += c * c;
      }
  row_sum<kNormWarps, WR, 1>(sq, s_red, red, warp, lane);
  const float rstd = valid ? rsqrtf(sq[0] / d + p.eps) : 0.f;
  if (in && warp % WR == 0 && lane == 0) {
    p.mean[row] = mean;
    p.rstd[row] = rstd;
  }
  const int nb = n_blocks(d);
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int c0 = base + norm_blk(lane, i), sub = lane & 7;
    const bool live = in && c0 < d;
    if (p.x_codes != nullptr)
      pack_block<VEC>(v[i], c0, d, p.x_codes + at, p.x_scales + (in ? row * nb : 0) + c0 / kBlk, lane & 7, live);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float g[4], bt[4];
      load4<float, VEC>(p.gamma, c0, sub, j, lim, g);
      load4<float, VEC>(p.beta, c0, sub, j, lim, bt);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[i][j][e] = piece_col<VEC>(c0, sub, j, e) < lim ? (v[i][j][e] - mean) * rstd * g[e] + bt[e] : 0.f;
      if constexpr (!std::is_same_v<Y, uint8_t>) {
        Y o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = from_f32<Y>(v[i][j][e]);
        if (in) store4<Y, VEC>(static_cast<Y*>(p.y) + at, c0, sub, j, d, o);
      }
    }
    if constexpr (std::is_same_v<Y, uint8_t>)
      pack_block<VEC>(v[i], c0, d, static_cast<uint8_t*>(p.y) + at, p.y_scales + (in ? row * nb : 0) + c0 / kBlk,
                      lane & 7, live);
  }
}

struct NormBwdParams {
  const void* dy;
  const void* x;            // tensor of dx's type, or 8-bit codes
  const uint8_t* x_scales;  // with 8-bit codes
  const float* gamma;
  const float* mean;
  const float* rstd;
  const uint8_t* mask;
  const void* resid;  // gradient of the residual branch, dx's type, or null
  void* dx;
  float* dgamma;
  float* dbeta;
  float* partial;  // [gridDim.x][2][d] sums of dy * xhat and of dy; not used by a grid of one CTA
  long long rows;
  int d;
};

// DY: type of dy; X: type of dx (and of x unless X8).  A CTA walks rows with
// a stride; each lane keeps the sums of its own columns, joined over the
// CTA's row groups at the end and over the CTAs by column_sum_kernel, always
// in the same order.  What bounds it is the latency of a row's loads with 16
// warps an SM: with an 8-bit x 7 of the 10.8 cycles between a warp's
// instructions wait for global memory, at 4.5 TB/s (32768 x 1024, 76 us).
template <typename DY, typename X, bool X8, int WR, bool VEC>
__global__ void __launch_bounds__(32 * norm_bwd_warps(WR), norm_bwd_ctas(WR)) norm_bwd_kernel(const NormBwdParams p) {
  constexpr int kWarps = norm_bwd_warps(WR);
  constexpr int kGroups = kWarps / WR;  // rows in flight per CTA
  __shared__ float s_red[2][kWarps * 2];
  int red = 0;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // the lane's block: of the warp's 512 columns, and of the row
  const int blk = norm_blk(lane, 0), c0 = (warp % WR) * 512 + blk, sub = lane & 7;
  const int d = p.d, nb = n_blocks(d);
  const float inv_d = 1.f / d;
  float acc_w[4][4], acc_b[4][4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc_w[j][e] = acc_b[j][e] = 0.f;

  const long long step = (long long)gridDim.x * kGroups;
  auto valid_at = [&](long long row) { return row < p.rows && (p.mask == nullptr || p.mask[row] != 0); };
  bool valid = valid_at((long long)blockIdx.x * kGroups + warp / WR);
  // the CTA's row groups run the same number of iterations: row_sum meets at barriers
  for (long long r0 = (long long)blockIdx.x * kGroups; r0 < p.rows; r0 += step) {
    const long long row = r0 + warp / WR;
    const bool in = row < p.rows;
    const int lim = valid ? d : 0;
    const long long at = in ? row * d : 0;
    // everything that the row needs is on its way before anything waits
    const float mean = valid ? p.mean[row] : 0.f, rstd = valid ? p.rstd[row] : 0.f;
    float g[4][4], xh[4][4], r[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) load4<DY, VEC>(static_cast<const DY*>(p.dy) + at, c0, sub, j, lim, g[j]);
    if constexpr (X8) {
      const float s = c0 < lim ? scale_value(p.x_scales[row * nb + c0 / kBlk]) : 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        e4m3x4_value(load_codes4<VEC>(static_cast<const uint8_t*>(p.x) + at, c0, sub, j, lim), s, xh[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) load4<X, VEC>(static_cast<const X*>(p.x) + at, c0, sub, j, lim, xh[j]);
    }
    if (p.resid != nullptr) {
#pragma unroll
      for (int j = 0; j < 4; ++j) load4<X, VEC>(static_cast<const X*>(p.resid) + at, c0, sub, j, lim, r[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) r[j][e] = 0.f;
    }
    const bool valid_next = valid_at(row + step);
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float gm[4];
      load4<float, VEC>(p.gamma, c0, sub, j, d, gm);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float xv = valid ? (xh[j][e] - mean) * rstd : 0.f;
        const float dyv = g[j][e];  // 0 past the row's end and for masked rows
        acc_w[j][e] += dyv * xv;
        acc_b[j][e] += dyv;
        const float gv = dyv * gm[e];
        s[0] += gv;
        s[1] += gv * xv;
        xh[j][e] = xv;
        g[j][e] = gv;
      }
    }
    row_sum<kWarps, WR, 2>(s, s_red, red, warp, lane);
    const float m0 = s[0] * inv_d, m1 = s[1] * inv_d;
    if (in) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        X o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          o[e] = from_f32<X>(valid ? rstd * (g[j][e] - m0 - xh[j][e] * m1) + r[j][e] : 0.f);
        store4<X, VEC>(static_cast<X*>(p.dx) + at, c0, sub, j, d, o);
      }
    }
    valid = valid_next;
  }

  // sums over the CTA's row groups, in group order
  __shared__ float s_acc[kGroups > 1 ? 512 : 1];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    auto& acc = q == 0 ? acc_w : acc_b;
    float* out = gridDim.x > 1 ? p.partial + ((size_t)blockIdx.x * 2 + q) * d : (q == 0 ? p.dgamma : p.dbeta);
    if constexpr (kGroups > 1) {
      static_assert(kGroups == 1 || WR <= 2, "row groups");
#pragma unroll
      for (int w = 1; w < kGroups; ++w) {
#pragma unroll
        for (int half = 0; half < WR; ++half) {
          __syncthreads();
          if (warp / WR == w && warp % WR == half)
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) s_acc[piece_col<VEC>(blk, sub, j, e)] = acc[j][e];
          __syncthreads();
          if (warp / WR == 0 && warp % WR == half)
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[j][e] += s_acc[piece_col<VEC>(blk, sub, j, e)];
        }
      }
    }
    if (warp / WR == 0)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int c = piece_col<VEC>(c0, sub, j, e);
          if (c < d) out[c] = acc[j][e];
        }
  }
}

}  // namespace tj
