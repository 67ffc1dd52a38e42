// combine.hip — weighted combine back to token order, shared-expert add,
// elementwise activation and standalone affine dequantisation for gfx950.
//
//   unpermute      Ops.moeUnpermute (Sources/FFAI/Ops/Ops.swift:5030-5110) with
//                  the combine weights rounded to the activation dtype first
//                  (Sources/FFAI/Models/MoELayer.swift:921-935)
//   unpermute backward   its gradient: expert rows and combine weights (the
//                  reference only runs forward)
//   shared add     MoELayer.swift:620-624 (unconditional add) and
//                  Ops.sigmoidScalarFMA (Ops.swift:6256-6317; Qwen3xText.swift:
//                  1054-1103): y = round(routed + sigmoid(g) * shared)
//   activation     Ops.swiglu (Ops.swift:6411-6460) / GPT-OSS clamped swish
//   dequantize     QuantizedOps.dequantizeAffine (QuantizedOps.swift:62-221)
//   add + RMSNorm  Ops.addAndRmsNorm (Ops.swift:676-730), the decoder step
//                  before the MoE block (Qwen3xText.swift:2650-2660)
//   residual       the decoder step after it folded into the final store:
//                  Ops.sigmoidScalarFMAResidual (OpsFused.swift:699-753),
//                  y = round(residual + routed + sigmoid(g) * shared), or
//                  y = round(residual + routed) without a shared expert
#include <algorithm>

#include "moe_common.hpp"
#include "moe_internal.hpp"

namespace moe {

// shared_mode: 0 none, 1 unconditional add, 2 sigmoid-gated add.
template <typename XT>
__device__ __forceinline__ float shared_gate(int mode, const XT* logit, int t) {
  if (mode == 2) return 1.0f / (1.0f + __expf(-to_f<XT>(logit[t])));
  return 1.0f;
}

constexpr int kCombineBatch = 8;  // expert ranks whose rows load together

// One block per token; threads stride over hidden 8 values at a time.
// res (nullable): the decoder residual added before the final rounding.
template <typename XT>
__global__ __launch_bounds__(256) void unpermute_kernel(const XT* __restrict__ Y,
                                                        const uint32_t* __restrict__ inv,
                                                        const float* __restrict__ w, int T, int H,
                                                        int k, XT* __restrict__ out,
                                                        const XT* __restrict__ sout,
                                                        const XT* __restrict__ slogit, int smode,
                                                        const XT* __restrict__ res) {
  const int t = blockIdx.x;
  const uint32_t M = (uint32_t)T * (uint32_t)k;
  const float g = smode ? shared_gate<XT>(smode, slogit, t) : 0.f;
  for (int h = threadIdx.x * 8; h < H; h += blockDim.x * 8) {
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    // ranks in batches of kCombineBatch: every position, then every row of a
    // batch in flight before its fused multiply-adds (in rank order, as the
    // loop over the ranks one at a time contracted them); a position past M
    // reads row 0 and leaves the sum unchanged
    for (int s0 = 0; s0 < k; s0 += kCombineBatch) {
      uint32_t p[kCombineBatch];
      float ws[kCombineBatch];
#pragma unroll
      for (int q = 0; q < kCombineBatch; q++) {
        const int s = min(s0 + q, k - 1);
        p[q] = inv[(size_t)t * k + s];
        ws[q] = round_to<XT>(w[(size_t)t * k + s]);
      }
      float y[kCombineBatch][8];
#pragma unroll
      for (int q = 0; q < kCombineBatch; q++)
        Vec8<XT>::load(Y + (size_t)(p[q] < M ? p[q] : 0u) * H + h, y[q]);
#pragma unroll
      for (int q = 0; q < kCombineBatch; q++) {
        const bool valid = s0 + q < k && p[q] < M;
#pragma unroll
        for (int j = 0; j < 8; j++) acc[j] = valid ? __builtin_fmaf(ws[q], y[q][j], acc[j]) : acc[j];
      }
    }
#pragma unroll
    for (int j = 0; j < 8; j++) acc[j] = round_to<XT>(acc[j]);
    if (res) {
      float rv[8];
      Vec8<XT>::load(res + (size_t)t * H + h, rv);
#pragma unroll
      for (int j = 0; j < 8; j++) acc[j] = rv[j] + acc[j];
    }
    if (smode) {
      float sv[8];
      Vec8<XT>::load(sout + (size_t)t * H + h, sv);
#pragma unroll
      for (int j = 0; j < 8; j++) acc[j] = acc[j] + g * sv[j];
    }
    Vec8<XT>::store(out + (size_t)t * H + h, acc);
  }
}

// Gradient of the combine out[t] = sum_s round(w[t,s]) Y[p(t,s)]:
//   dY[p(t,s)] = round(w[t,s]) g[t],   dw[t,s] = <g[t], Y[p(t,s)]>
// One block per token. The ranks go in batches of kCombineBatch, whose rows
// are all in flight together; a thread keeps its share of the batch's dot
// products over its chunks of the row, and the block adds them along a fixed
// tree. The gradient row is read once per batch (from cache after the first).
// Y and dY may be one buffer: a thread reads its values before it stores them
// and every position belongs to one block. A position past M has a zero dw
// and no row.
template <typename XT>
__global__ __launch_bounds__(256) void unpermute_backward_kernel(const XT* __restrict__ g,
                                                                 const XT* Y,
                                                                 const uint32_t* __restrict__ inv,
                                                                 const float* __restrict__ w,
                                                                 int T, int H, int k, XT* dY,
                                                                 float* __restrict__ dw) {
  __shared__ float part[4][kCombineBatch];
  const int t = blockIdx.x;
  const uint32_t M = (uint32_t)T * (uint32_t)k;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int s0 = 0; s0 < k; s0 += kCombineBatch) {
    uint32_t p[kCombineBatch];
    float ws[kCombineBatch], dot[kCombineBatch];
#pragma unroll
    for (int q = 0; q < kCombineBatch; q++) {
      const int s = min(s0 + q, k - 1);
      p[q] = s0 + q < k ? inv[(size_t)t * k + s] : 0xFFFFFFFFu;
      ws[q] = round_to<XT>(w[(size_t)t * k + s]);
      dot[q] = 0.f;
    }
    for (int h = threadIdx.x * 8; h < H; h += 256 * 8) {
      float gv[8], y[kCombineBatch][8];
      Vec8<XT>::load(g + (size_t)t * H + h, gv);
#pragma unroll
      for (int q = 0; q < kCombineBatch; q++)
        if (p[q] < M) Vec8<XT>::load(Y + (size_t)p[q] * H + h, y[q]);
#pragma unroll
      for (int q = 0; q < kCombineBatch; q++) {
        if (p[q] < M) {
          float o[8];
#pragma unroll
          for (int j = 0; j < 8; j++) {
            dot[q] = __builtin_fmaf(gv[j], y[q][j], dot[q]);
            o[j] = ws[q] * gv[j];
          }
          if (dY) Vec8<XT>::store(dY + (size_t)p[q] * H + h, o);
        }
      }
    }
#pragma unroll
    for (int q = 0; q < kCombineBatch; q++) {
      const float d = group_sum(dot[q], 6);
      if (lane == 63) part[wave][q] = d;
    }
    __syncthreads();
    if (threadIdx.x < kCombineBatch && s0 + (int)threadIdx.x < k)
      dw[(size_t)t * k + s0 + threadIdx.x] = (part[0][threadIdx.x] + part[1][threadIdx.x]) +
                                             (part[2][threadIdx.x] + part[3][threadIdx.x]);
    __syncthreads();
  }
}

template <typename XT>
__global__ __launch_bounds__(256) void add_shared_kernel(XT* __restrict__ y,
                                                         const XT* __restrict__ sout,
                                                         const XT* __restrict__ slogit, int smode,
                                                         int H, const XT* __restrict__ res) {
  const int t = blockIdx.x;
  const float g = shared_gate<XT>(smode, slogit, t);
  for (int h = threadIdx.x * 8; h < H; h += blockDim.x * 8) {
    float a[8], b[8];
    Vec8<XT>::load(y + (size_t)t * H + h, a);
    Vec8<XT>::load(sout + (size_t)t * H + h, b);
    if (res) {
      float rv[8];
      Vec8<XT>::load(res + (size_t)t * H + h, rv);
#pragma unroll
      for (int j = 0; j < 8; j++) a[j] = rv[j] + a[j];
    }
#pragma unroll
    for (int j = 0; j < 8; j++) a[j] = a[j] + g * b[j];
    Vec8<XT>::store(y + (size_t)t * H + h, a);
  }
}

template <typename XT>
__global__ __launch_bounds__(256) void activation_kernel(const XT* __restrict__ g,
                                                         const XT* __restrict__ u,
                                                         XT* __restrict__ out, int64_t n, int act,
                                                         float alpha, float limit) {
  // squared ReLU reads the up projection only; g may be null for it
  const bool gated = act != ACT_RELU2;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n;
       i += (int64_t)gridDim.x * blockDim.x) {
    const float gv = gated ? to_f<XT>(g[i]) : 0.0f;
    out[i] = from_f<XT>(apply_act<XT>(gv, to_f<XT>(u[i]), act, alpha, limit));
  }
}

// bf16 rows -> the f16 A operand of the grouped GEMM (bf16x8_to_a16), 8
// values per thread and step.
__global__ __launch_bounds__(256) void to_a16_kernel(const uint4* __restrict__ x,
                                                     uint4* __restrict__ y, int64_t n8) {
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n8;
       i += (int64_t)gridDim.x * blockDim.x)
    y[i] = bf16x8_to_a16<kA16Shift>(x[i]);
}

hipError_t launch_to_a16(const void* x, void* y, int64_t n, hipStream_t st) {
  if (n % 8 != 0) return hipErrorInvalidValue;
  const int64_t n8 = n / 8;
  const int grid = (int)std::min<int64_t>((n8 + 255) / 256, 4096);
  hipLaunchKernelGGL(to_a16_kernel, dim3(grid), dim3(256), 0, st,
                     reinterpret_cast<const uint4*>(x), reinterpret_cast<uint4*>(y), n8);
  return hipGetLastError();
}

// One block per row: s = round(a + b) stored to res, then
// xn = round(s / sqrt(mean(s^2) + eps) * w) stored to xn. A thread keeps its
// (up to kNormChunks) 8-value chunks in registers between the two halves.
constexpr int kNormChunks = 4;  // rows up to 256 * 8 * 4 = 8192 values

template <typename XT>
__global__ __launch_bounds__(256) void add_rmsnorm_kernel(const XT* __restrict__ a,
                                                          const XT* __restrict__ b,
                                                          const XT* __restrict__ w, float eps,
                                                          int H, XT* __restrict__ res,
                                                          XT* __restrict__ xn) {
  __shared__ float part[4];
  const size_t row = (size_t)blockIdx.x * H;
  float sv[kNormChunks][8];
  float ssq = 0.f;
#pragma unroll
  for (int c = 0; c < kNormChunks; c++) {
    const int h = (threadIdx.x + c * 256) * 8;
    if (h < H) {
      float av[8], bv[8];
      Vec8<XT>::load(a + row + h, av);
      Vec8<XT>::load(b + row + h, bv);
#pragma unroll
      for (int j = 0; j < 8; j++) {
        sv[c][j] = round_to<XT>(av[j] + bv[j]);
        ssq = __builtin_fmaf(sv[c][j], sv[c][j], ssq);
      }
      Vec8<XT>::store(res + row + h, sv[c]);
    }
  }
  ssq = group_sum(ssq, 6);
  if ((threadIdx.x & 63) == 63) part[threadIdx.x >> 6] = ssq;
  __syncthreads();
  const float tot = (part[0] + part[1]) + (part[2] + part[3]);
  const float rms = sqrtf(tot / (float)H + eps);
#pragma unroll
  for (int c = 0; c < kNormChunks; c++) {
    const int h = (threadIdx.x + c * 256) * 8;
    if (h < H) {
      float wv[8], o[8];
      Vec8<XT>::load(w + h, wv);
#pragma unroll
      for (int j = 0; j < 8; j++) o[j] = sv[c][j] / rms * wv[j];
      Vec8<XT>::store(xn + row + h, o);
    }
  }
}

template <typename ST, typename OT>
__global__ __launch_bounds__(256) void dequantize_kernel(const uint32_t* __restrict__ w,
                                                         const ST* __restrict__ s,
                                                         const ST* __restrict__ b, int bits,
                                                         int gs, int64_t numel,
                                                         OT* __restrict__ out) {
#pragma clang fp contract(off)
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < numel;
       i += (int64_t)gridDim.x * blockDim.x) {
    const uint64_t bit = (uint64_t)i * (uint64_t)bits;
    const uint64_t word = bit >> 5;
    const uint32_t sh = (uint32_t)(bit & 31u);
    uint64_t win = w[word];
    if (sh + (uint32_t)bits > 32u) win |= (uint64_t)w[word + 1] << 32;
    const float q = (float)((uint32_t)(win >> sh) & ((1u << bits) - 1u));
    const int64_t g = i / gs;
    const float sq = to_f<ST>(s[g]) * q;
    out[i] = from_f<OT>(sq + to_f<ST>(b[g]));
  }
}

#define MOE_BY_DT(dt, MACRO)          \
  if ((dt) == DT_BF16) { MACRO(bf16_t) } \
  if ((dt) == DT_F16) { MACRO(f16_t) }   \
  if ((dt) == DT_F32) { MACRO(float) }

hipError_t launch_unpermute(const void* Y, const uint32_t* inv, const float* w, int T, int H,
                            int k, void* out, int dt, const void* shared_out,
                            const void* shared_logit, int shared_mode, hipStream_t st,
                            const void* res) {
#define MOE_UP(XT)                                                                            \
  hipLaunchKernelGGL((unpermute_kernel<XT>), dim3(T), dim3(256), 0, st, (const XT*)Y, inv, w, \
                     T, H, k, (XT*)out, (const XT*)shared_out, (const XT*)shared_logit,       \
                     shared_mode, (const XT*)res);                                            \
  return hipGetLastError();
  MOE_BY_DT(dt, MOE_UP)
#undef MOE_UP
  return hipErrorInvalidValue;
}

hipError_t launch_unpermute_backward(const void* g, const void* Y, const uint32_t* inv,
                                     const float* w, int T, int H, int k, void* dY, float* dw,
                                     int dt, hipStream_t st) {
#define MOE_UB(XT)                                                                            \
  hipLaunchKernelGGL((unpermute_backward_kernel<XT>), dim3(T), dim3(256), 0, st, (const XT*)g, \
                     (const XT*)Y, inv, w, T, H, k, (XT*)dY, dw);                             \
  return hipGetLastError();
  MOE_BY_DT(dt, MOE_UB)
#undef MOE_UB
  return hipErrorInvalidValue;
}

hipError_t launch_add_shared(void* y, const void* shared_out, const void* shared_logit,
                             int shared_mode, int T, int H, int dt, hipStream_t st,
                             const void* res) {
#define MOE_AS(XT)                                                                        \
  hipLaunchKernelGGL((add_shared_kernel<XT>), dim3(T), dim3(256), 0, st, (XT*)y,          \
                     (const XT*)shared_out, (const XT*)shared_logit, shared_mode, H,       \
                     (const XT*)res);                                                      \
  return hipGetLastError();
  MOE_BY_DT(dt, MOE_AS)
#undef MOE_AS
  return hipErrorInvalidValue;
}

hipError_t launch_add_rmsnorm(const void* a, const void* b, const void* w, float eps, int T,
                              int H, int dt, void* res, void* xn, hipStream_t st) {
  if (H % 8 != 0 || H > 256 * 8 * kNormChunks) return hipErrorInvalidValue;
#define MOE_AN(XT)                                                                          \
  hipLaunchKernelGGL((add_rmsnorm_kernel<XT>), dim3(T), dim3(256), 0, st, (const XT*)a,     \
                     (const XT*)b, (const XT*)w, eps, H, (XT*)res, (XT*)xn);                \
  return hipGetLastError();
  MOE_BY_DT(dt, MOE_AN)
#undef MOE_AN
  return hipErrorInvalidValue;
}

hipError_t launch_activation(const void* g, const void* u, void* out, int64_t n, int dt, int act,
                             float alpha, float limit, hipStream_t st) {
  const int64_t blocks64 = (n + 255) / 256;
  const int grid = (int)(blocks64 < 65536 ? blocks64 : 65536);
#define MOE_ACT(XT)                                                                          \
  hipLaunchKernelGGL((activation_kernel<XT>), dim3(grid), dim3(256), 0, st, (const XT*)g,   \
                     (const XT*)u, (XT*)out, n, act, alpha, limit);                         \
  return hipGetLastError();
  MOE_BY_DT(dt, MOE_ACT)
#undef MOE_ACT
  return hipErrorInvalidValue;
}

hipError_t launch_dequantize(const uint32_t* w, const void* s, const void* b, int sbdt, int bits,
                             int gs, int64_t numel, void* out, int odt, hipStream_t st) {
  const int64_t blocks64 = (numel + 255) / 256;
  const int grid = (int)(blocks64 < 65536 ? blocks64 : 65536);
#define MOE_DQ2(ST, OT)                                                                     \
  hipLaunchKernelGGL((dequantize_kernel<ST, OT>), dim3(grid), dim3(256), 0, st, w,         \
                     (const ST*)s, (const ST*)b, bits, gs, numel, (OT*)out);               \
  return hipGetLastError();
#define MOE_DQ(ST)                              \
  if (odt == DT_BF16) { MOE_DQ2(ST, bf16_t) }   \
  if (odt == DT_F16) { MOE_DQ2(ST, f16_t) }     \
  if (odt == DT_F32) { MOE_DQ2(ST, float) }
  MOE_BY_DT(sbdt, MOE_DQ)
#undef MOE_DQ
#undef MOE_DQ2
  return hipErrorInvalidValue;
}

}  // namespace moe
