// layer_grad.hip — what surrounds the experts' gradients in a layer's backward
// pass, for gfx950.
//
//   permute backward       rows sorted by expert back to their tokens: the k
//                          copies of a token's row that the plan made
//                          (MoELayer.swift:752-792) add their gradients
//   add + RMSNorm backward gradient of add_rmsnorm_kernel (Ops.swift:676-730)
//                          with respect to its rows and its weight
#include <algorithm>

#include "moe_common.hpp"
#include "moe_internal.hpp"

namespace moe {

// dx[t] = round(dx_in[t] + sum_s dX[inv[t*k + s]]), eight columns per thread,
// the chunks of all tokens side by side so that narrow rows fill blocks too.
// Up to kRankBatch rows in flight; the ranks are added in order.
constexpr int kRankBatch = 8;

template <typename XT>
__global__ __launch_bounds__(256) void permute_backward_kernel(const XT* __restrict__ dX,
                                                               const uint32_t* __restrict__ inv, int T,
                                                               int H, int k, const XT* dx_in, XT* dx) {
  const uint32_t M = (uint32_t)T * (uint32_t)k, chunks = (uint32_t)H / 8;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t t = i / chunks;
  if (t >= T) return;
  const int h = (int)(i - t * chunks) * 8;
  float acc[8] = {};
  if (dx_in) Vec8<XT>::load(dx_in + t * H + h, acc);
  for (int s0 = 0; s0 < k; s0 += kRankBatch) {
    uint32_t p[kRankBatch];
#pragma unroll
    for (int q = 0; q < kRankBatch; q++) p[q] = s0 + q < k ? inv[t * k + s0 + q] : 0xFFFFFFFFu;
    float v[kRankBatch][8];
#pragma unroll
    for (int q = 0; q < kRankBatch; q++)
      if (p[q] < M) Vec8<XT>::load(dX + (size_t)p[q] * H + h, v[q]);
#pragma unroll
    for (int q = 0; q < kRankBatch; q++)
      if (p[q] < M)
#pragma unroll
        for (int j = 0; j < 8; j++) acc[j] += v[q][j];
  }
  Vec8<XT>::store(dx + t * H + h, acc);
}

hipError_t launch_permute_backward(const void* dX, const uint32_t* inv, int T, int H, int k,
                                   const void* dx_in, void* dx, int dt, hipStream_t st) {
  const dim3 grid((unsigned)(((int64_t)T * (H / 8) + 255) / 256));
#define MOE_PB(XT)                                                                               \
  hipLaunchKernelGGL((permute_backward_kernel<XT>), grid, dim3(256), 0, st, (const XT*)dX, inv, T, \
                     H, k, (const XT*)dx_in, (XT*)dx)
  if (dt == DT_BF16) MOE_PB(bf16_t);
  else if (dt == DT_F16) MOE_PB(f16_t);
  else MOE_PB(float);
#undef MOE_PB
  return hipGetLastError();
}

// With s = 1 / sqrt(mean(r^2) + eps) and n = r s of a row:
//   d_in = d_res + s (dn w - n mean(dn w n)),   dw = sum over rows of dn n
// A block's rows go through its threads one after another; a thread owns
// the same columns of each and keeps their share of dw in registers.
struct NormBackward {
  const void *r, *w, *dn, *dr;
  void* din;
  float* dw;  // [blocks, H] partial sums, or the result where there is one block
  float eps;
  int T, H;
};
constexpr int kNormMax = 4;  // chunks of 8 per thread: rows up to 8192 values

template <typename XT>
__global__ __launch_bounds__(256) void norm_backward_kernel(const NormBackward a) {
  __shared__ float part[2][4][2];
  const int H = a.H, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float dw[kNormMax][8] = {};
  int turn = 0;
  for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x, turn ^= 1) {
    float r[kNormMax][8], g[kNormMax][8];
    float ss = 0.0f, sg = 0.0f;
#pragma unroll
    for (int c = 0; c < kNormMax; c++) {
      const int h = (threadIdx.x + c * 256) * 8;
      if (h < H) {
        float w[8];
        Vec8<XT>::load((const XT*)a.r + t * H + h, r[c]);
        Vec8<XT>::load((const XT*)a.dn + t * H + h, g[c]);
        Vec8<XT>::load((const XT*)a.w + h, w);
#pragma unroll
        for (int j = 0; j < 8; j++) {
          ss = __builtin_fmaf(r[c][j], r[c][j], ss);
          sg = __builtin_fmaf(g[c][j] * w[j], r[c][j], sg);
        }
      }
    }
    ss = group_sum(ss, 6);
    sg = group_sum(sg, 6);
    if (lane == 63) {
      part[turn][wave][0] = ss;
      part[turn][wave][1] = sg;
    }
    __syncthreads();
    ss = (part[turn][0][0] + part[turn][1][0]) + (part[turn][2][0] + part[turn][3][0]);
    sg = (part[turn][0][1] + part[turn][1][1]) + (part[turn][2][1] + part[turn][3][1]);
    const float s = 1.0f / sqrtf(ss / (float)H + a.eps);
    const float m = s * sg / (float)H;  // mean(dn w n)
#pragma unroll
    for (int c = 0; c < kNormMax; c++) {
      const int h = (threadIdx.x + c * 256) * 8;
      if (h < H) {
        float w[8], d[8] = {};
        Vec8<XT>::load((const XT*)a.w + h, w);
        if (a.dr) Vec8<XT>::load((const XT*)a.dr + t * H + h, d);
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const float n = r[c][j] * s;
          d[j] += s * (g[c][j] * w[j] - n * m);
          dw[c][j] = __builtin_fmaf(g[c][j], n, dw[c][j]);
        }
        Vec8<XT>::store((XT*)a.din + t * H + h, d);
      }
    }
  }
#pragma unroll
  for (int c = 0; c < kNormMax; c++) {
    const int h = (threadIdx.x + c * 256) * 8;
    if (h < H) Vec8<float>::store(a.dw + (size_t)blockIdx.x * H + h, dw[c]);
  }
}

// Adds the blocks' partial sums in order.
__global__ __launch_bounds__(256) void norm_weight_kernel(const float* __restrict__ part, int blocks, int H,
                                                          float* __restrict__ dw) {
  const int h = blockIdx.x * 256 + threadIdx.x;
  if (h >= H) return;
  float s = 0.0f;
  for (int b = 0; b < blocks; b++) s += part[(size_t)b * H + h];
  dw[h] = s;
}

static int norm_blocks(int T) { return std::min(T, 512); }

size_t norm_backward_ws_bytes(int T, int H) {
  const int blocks = norm_blocks(T);
  return blocks > 1 ? (size_t)blocks * H * 4 : 0;
}

hipError_t launch_norm_backward(const void* r, const void* w, const void* dn, const void* dr, float eps,
                                int T, int H, int dt, void* din, float* dw, void* ws, hipStream_t st) {
  const int blocks = norm_blocks(T);
  const NormBackward a{r, w, dn, dr, din, blocks > 1 ? (float*)ws : dw, eps, T, H};
  if (dt == DT_BF16) hipLaunchKernelGGL((norm_backward_kernel<bf16_t>), dim3(blocks), dim3(256), 0, st, a);
  else if (dt == DT_F16) hipLaunchKernelGGL((norm_backward_kernel<f16_t>), dim3(blocks), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((norm_backward_kernel<float>), dim3(blocks), dim3(256), 0, st, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || blocks == 1) return e;
  hipLaunchKernelGGL(norm_weight_kernel, dim3((H + 255) / 256), dim3(256), 0, st, (const float*)ws, blocks, H, dw);
  return hipGetLastError();
}

}  // namespace moe
