// ckpt8.hip — the gated activation with its inputs kept in 8 bits, and its
// gradient from what was kept, for gfx950.
//
//   activation save      h = act(g, u) as moe_activation_apply, g and u as
//                        microscaled int8 (blocks of 32, a power of two each)
//   restore              the kept values
//   activation backward  d_gate, d_up, the routing weight's gradient, h again
//
// The reference only runs forward (Ops.swift:6400-6460 and the activations of
// moe_common.hpp); these are the two halves of the step that differentiates it.
#include <algorithm>

#include "moe_common.hpp"
#include "moe_internal.hpp"

namespace moe {

constexpr int kKeepBlock = 32;  // values that share an exponent byte

// Exponent byte of a block whose largest magnitude has the bits `top`: the
// least e with |v| < 127.5 * 2^(e - 133) for all of its values, so that every
// code is rounded by at most half a step and none saturates. (The mantissa of
// 127.5 / 64 is 0x7F0000: adding 0x10000 carries from there on.) 255 marks a
// block with an infinity, a NaN or a value of 255/256 * 2^128 or more.
__device__ __forceinline__ uint32_t keep_exponent(uint32_t top) {
  return min((top + 0x10000u) >> 23, 255u);
}

// Eight values of a block as codes; top: the block's largest magnitude's bits.
__device__ __forceinline__ uint2 keep_codes(const float (&v)[8], uint32_t e) {
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const int c = (int)__builtin_rintf(__builtin_ldexpf(v[j], 133 - (int)e));
    w[j >> 2] |= ((uint32_t)c & 0xFFu) << (8 * (j & 3));
  }
  return e == 255u ? make_uint2(0u, 0u) : make_uint2(w[0], w[1]);
}

// (A code times a power of two is exact, below the smallest normal value too.)
__device__ __forceinline__ void kept_values(uint2 c, uint32_t e, float (&v)[8]) {
  const float step = e == 255u ? __builtin_nanf("") : __builtin_ldexpf(1.0f, (int)e - 133);
  const uint32_t w[2] = {c.x, c.y};
#pragma unroll
  for (int j = 0; j < 8; j++) v[j] = (float)(int)(int8_t)(w[j >> 2] >> (8 * (j & 3))) * step;
}

__device__ __forceinline__ uint32_t top_bits(const float (&v)[8]) {
  uint32_t t = 0;
#pragma unroll
  for (int j = 0; j < 8; j++) t = max(t, __float_as_uint(v[j]) & 0x7FFFFFFFu);
  return t;
}

// Largest over the four lanes of a block.
__device__ __forceinline__ uint32_t quad_max(uint32_t t) {
  t = max(t, (uint32_t)__builtin_amdgcn_mov_dpp((int)t, 0xB1, 0xF, 0xF, false));
  return max(t, (uint32_t)__builtin_amdgcn_mov_dpp((int)t, 0x4E, 0xF, 0xF, false));
}

// A value rounded to fp32 here: keeps the compiler from rounding a product
// straight to f16 (v_fma_mixlo_f16), where moe_activation_apply rounds to fp32
// first, so that both give the same bits.
__device__ __forceinline__ float settled(float v) {
  asm("" : "+v"(v));
  return v;
}

// Rows that a call works on: all M, or the count a plan left on the device.
__device__ __forceinline__ int64_t used_rows(const uint32_t* n_rows, int M) {
  return n_rows ? (int64_t)min(*n_rows, (uint32_t)M) : (int64_t)M;
}

// Eight values per thread, four threads per block of 32; rows are whole
// blocks, so the arrays are walked flat. Bound by memory: 32768 rows of 768 in
// bf16 take 36 us (203 MB, 5.6 TB/s where a large copy reaches 5.2: a part may come
// from the caches).
template <typename XT, int ACT>
__global__ __launch_bounds__(256) void activation_save_kernel(
    const XT* gate, const XT* up, int M, int n, float alpha, float limit,
    const uint32_t* __restrict__ n_rows, XT* out, int8_t* __restrict__ codes,
    uint8_t* __restrict__ scales) {
  const int64_t all = (int64_t)M * n, end = used_rows(n_rows, M) * n;
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8; i < end; i += (int64_t)gridDim.x * 2048) {
    float g[8] = {}, u[8], h[8];
    if constexpr (ACT != ACT_RELU2) Vec8<XT>::load(gate + i, g);
    Vec8<XT>::load(up + i, u);
#pragma unroll
    for (int j = 0; j < 8; j++) h[j] = settled(apply_act<XT>(g[j], u[j], ACT, alpha, limit));
    if (out) Vec8<XT>::store(out + i, h);
    auto keep = [&](const float (&v)[8], int64_t at) {
      const uint32_t e = keep_exponent(quad_max(top_bits(v)));
      *reinterpret_cast<uint2*>(codes + at) = keep_codes(v, e);
      if ((threadIdx.x & 3) == 0) scales[at / kKeepBlock] = (uint8_t)e;
    };
    if constexpr (ACT != ACT_RELU2) keep(g, i);
    keep(u, ACT != ACT_RELU2 ? all + i : i);
  }
}

// Bound by memory: 2 x 32768 x 768 values in bf16 take 23 us (153 MB; part in the caches).
template <typename XT>
__global__ __launch_bounds__(256) void restore_kernel(const int8_t* __restrict__ codes,
                                                      const uint8_t* __restrict__ scales,
                                                      int64_t numel, XT* __restrict__ out) {
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8; i < numel; i += (int64_t)gridDim.x * 2048) {
    float v[8];
    kept_values(*reinterpret_cast<const uint2*>(codes + i), scales[i / kKeepBlock], v);
    if constexpr (__is_same(XT, f16_t)) {  // (65024 to 65504 are kept as 64 steps of 1024, which f16 has not)
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] = __builtin_fabsf(v[j]) == 65536.0f ? __builtin_copysignf(65504.0f, v[j]) : v[j];
    }
    Vec8<XT>::store(out + i, v);
  }
}

// e^x to a few roundings wherever it is normal: 2^h for the product h of x and log2 e as
// rounded, times 2^l for what that left (one product alone is off by |x| 2^-24 of the
// result). Past 128 infinity and 0, which the result is in fp32; NaN stays.
__device__ __forceinline__ float near_exp(float x) {
  constexpr float kLog2e = 1.44269502f, kRest = 1.92596303e-8f;  // log2 e and what fp32 leaves of it
  x = x > 128.0f ? 128.0f : (x < -128.0f ? -128.0f : x);
  const float h = x * kLog2e;
  const float l = __builtin_fmaf(x, kRest, __builtin_fmaf(x, kLog2e, -h));
  return __builtin_amdgcn_exp2f(h) * __builtin_fmaf(l, 0.69314718f, 1.0f);
}

// Value and slopes of the activation at (g, u); NaN in either gives NaN in all
// that depends on it (apply_act's clamps would drop it).
template <typename XT, int ACT>
__device__ __forceinline__ void act_slopes(float g, float u, float alpha, float limit, float& h,
                                           float& hg, float& hu) {
  if constexpr (ACT == ACT_RELU2) {
    const float r = u < 0.0f ? 0.0f : u;
    h = r * r;
    hg = 0.0f;
    hu = 2.0f * r;
  } else if constexpr (ACT == ACT_GPTOSS) {
    const float gc = g > limit ? limit : g;
    const float uc = u > limit ? limit : (u < -limit ? -limit : u);
    const float s = __builtin_amdgcn_rcpf(1.0f + near_exp(-alpha * gc));
    const float a = gc * s;
    h = a * (uc + 1.0f);
    hg = g > limit ? 0.0f : (s + alpha * a * (1.0f - s)) * (uc + 1.0f);
    hu = uc == u ? a : uc - uc;  // past the limit 0, a NaN's own
  } else if constexpr (ACT == ACT_GEGLU) {
    const float y = 0.7978845608f * (g + 0.044715f * g * g * g);
    const float l = __builtin_amdgcn_rcpf(1.0f + near_exp(-2.0f * y));
    const float t = l * (1.0f - l);  // 0 where g * g may be infinite
    const float d = t > 0.0f ? l + t * g * (1.5957691216f * (1.0f + 0.134145f * g * g)) : l;
    const float a = round_to<XT>(g * l);
    h = a * u;
    hg = d * u;
    hu = a;
  } else {
    const float s = __builtin_amdgcn_rcpf(1.0f + near_exp(-g));
    const float a = g * s;
    h = a * u;
    hg = (s + a * (1.0f - s)) * u;
    hu = a;
  }
}

struct ActBackward {
  const int8_t* codes;
  const uint8_t* scales;
  const void* dh;
  const float* weight;
  const uint32_t *perm, *n_rows;
  void *dg, *du, *h;
  float* dw;
  int M, n, lg;
  float alpha, limit;
};

// A team takes a row, eight columns a lane and step: 2^lg lanes of a wave, or
// (BLOCK) a block's four waves, whose shares of the dot product meet in LDS. Bound by
// memory: 32768 rows of 768, bf16, take 36.5 us (203 MB, 5.6 TB/s).
template <typename XT, int ACT, bool BLOCK>
__global__ __launch_bounds__(256) void activation_backward_kernel(const ActBackward a) {
  __shared__ float part[4];
  const int lanes = BLOCK ? 256 : 1 << a.lg, lane = threadIdx.x & (lanes - 1);
  const int64_t row = BLOCK ? (int64_t)blockIdx.x : ((int64_t)blockIdx.x * 256 + threadIdx.x) >> a.lg;
  const bool on = row < used_rows(a.n_rows, a.M);
  const int64_t at = row * a.n, all = (int64_t)a.M * a.n;
  const int n = on ? a.n : 0;
  uint32_t pick = 0;
  float w = 1.0f;
  if (on) {
    pick = a.perm ? a.perm[row] : (uint32_t)row;
    if (a.weight) w = pick < (uint32_t)a.M ? round_to<XT>(a.weight[pick]) : 0.0f;
  }
  float dot = 0.0f;
#pragma unroll 2
  for (int c = lane * 8; c < n; c += lanes * 8) {
    const int64_t i = at + c;
    float g[8] = {}, u[8], d[8], dg[8], du[8], h[8];
    constexpr bool GATED = ACT != ACT_RELU2;
    const int64_t iu = GATED ? all + i : i;
    if constexpr (GATED)
      kept_values(*reinterpret_cast<const uint2*>(a.codes + i), a.scales[i / kKeepBlock], g);
    kept_values(*reinterpret_cast<const uint2*>(a.codes + iu), a.scales[iu / kKeepBlock], u);
    Vec8<XT>::load((const XT*)a.dh + i, d);
#pragma unroll
    for (int j = 0; j < 8; j++) {
      float hg, hu;
      act_slopes<XT, ACT>(g[j], u[j], a.alpha, a.limit, h[j], hg, hu);
      dot = __builtin_fmaf(d[j], h[j], dot);
      dg[j] = w * d[j] * hg;
      du[j] = w * d[j] * hu;
    }
    if constexpr (GATED) Vec8<XT>::store((XT*)a.dg + i, dg);
    Vec8<XT>::store((XT*)a.du + i, du);
    if (a.h) Vec8<XT>::store((XT*)a.h + i, h);
  }
  if (!a.dw) return;
  dot = group_sum(dot, BLOCK ? 6 : a.lg);
  if constexpr (BLOCK) {
    if ((threadIdx.x & 63) == 63) part[threadIdx.x >> 6] = dot;
    __syncthreads();
    dot = (part[0] + part[1]) + (part[2] + part[3]);
  }
  if (on && lane == lanes - 1 && pick < (uint32_t)a.M) a.dw[pick] = dot;
}

namespace {

int flat_grid(int64_t numel) { return (int)std::min<int64_t>((numel + 2047) / 2048, 1 << 16); }

template <typename XT>
hipError_t save_t(const void* g, const void* u, int M, int n, int act, float alpha, float limit,
                  const uint32_t* n_rows, void* out, int8_t* codes, uint8_t* scales, hipStream_t st) {
#define MOE_SAVE(ACT)                                                                              \
  case ACT:                                                                                        \
    hipLaunchKernelGGL((activation_save_kernel<XT, ACT>), dim3(flat_grid((int64_t)M * n)), dim3(256), \
                       0, st, (const XT*)g, (const XT*)u, M, n, alpha, limit, n_rows, (XT*)out,    \
                       codes, scales);                                                             \
    return hipGetLastError();
  switch (act) {
    MOE_SAVE(ACT_SWIGLU)
    MOE_SAVE(ACT_GPTOSS)
    MOE_SAVE(ACT_GEGLU)
    MOE_SAVE(ACT_RELU2)
  }
#undef MOE_SAVE
  return hipErrorInvalidValue;
}

// lg 8: a block per row.
template <typename XT>
hipError_t backward_t(const ActBackward& a, int act, hipStream_t st) {
  const dim3 grid((unsigned)((((int64_t)a.M << a.lg) + 255) / 256));
#define MOE_BACK(ACT)                                                                                \
  case ACT:                                                                                          \
    if (a.lg == 8)                                                                                   \
      hipLaunchKernelGGL((activation_backward_kernel<XT, ACT, true>), grid, dim3(256), 0, st, a);    \
    else                                                                                             \
      hipLaunchKernelGGL((activation_backward_kernel<XT, ACT, false>), grid, dim3(256), 0, st, a);   \
    return hipGetLastError();
  switch (act) {
    MOE_BACK(ACT_SWIGLU)
    MOE_BACK(ACT_GPTOSS)
    MOE_BACK(ACT_GEGLU)
    MOE_BACK(ACT_RELU2)
  }
#undef MOE_BACK
  return hipErrorInvalidValue;
}

// log2 of the lanes per row. A block for long rows, and for few rows of more than 512
// columns; else the most lanes of a wave that a row keeps 7/8 busy, or the least
// that hold it in one step. us, bf16: 148 rows of 2880 with 8 lanes 36, a block 12 (the
// call's host work); 8192 rows of 2880 with a wave 39.9, a block 33.0; 10000 rows of
// 768 with 32 lanes 13.2, a block 17.4; 32768 of 768 with 32 lanes 36.5 (5.6 TB/s), a
// wave (3/4 busy) 47.3.
int row_lanes(int M, int n) {
  const int chunks = n / 8;
  if (chunks > 192 || (M < 4096 && chunks > 64)) return 8;
  for (int lg = 6; lg > 3; lg--) {
    const int lanes = 1 << lg, steps = (chunks + lanes - 1) / lanes;
    if (chunks > lanes / 2 && (steps == 1 || 8 * chunks >= 7 * steps * lanes)) return lg;
  }
  return 3;
}

}  // namespace

hipError_t launch_activation_save(const void* g, const void* u, int M, int n, int dt, int act,
                                  float alpha, float limit, const uint32_t* n_rows, void* out,
                                  int8_t* codes, uint8_t* scales, hipStream_t st) {
  if (dt == DT_BF16) return save_t<bf16_t>(g, u, M, n, act, alpha, limit, n_rows, out, codes, scales, st);
  if (dt == DT_F16) return save_t<f16_t>(g, u, M, n, act, alpha, limit, n_rows, out, codes, scales, st);
  return save_t<float>(g, u, M, n, act, alpha, limit, n_rows, out, codes, scales, st);
}

hipError_t launch_restore(const int8_t* codes, const uint8_t* scales, int64_t numel, void* out, int dt,
                          hipStream_t st) {
#define MOE_RESTORE(XT)                                                                            \
  hipLaunchKernelGGL((restore_kernel<XT>), dim3(flat_grid(numel)), dim3(256), 0, st, codes, scales, \
                     numel, (XT*)out)
  if (dt == DT_BF16) MOE_RESTORE(bf16_t);
  else if (dt == DT_F16) MOE_RESTORE(f16_t);
  else MOE_RESTORE(float);
#undef MOE_RESTORE
  return hipGetLastError();
}

hipError_t launch_activation_backward(const int8_t* codes, const uint8_t* scales, const void* dh, int M,
                                      int n, int dt, int act, float alpha, float limit,
                                      const float* weight, const uint32_t* perm, const uint32_t* n_rows,
                                      void* dg, void* du, float* dw, void* h, hipStream_t st) {
  const int lg = row_lanes(M, n);
  const ActBackward a{codes, scales, dh, weight, perm, n_rows, dg, du, h, dw, M, n, lg, alpha, limit};
  if (dt == DT_BF16) return backward_t<bf16_t>(a, act, st);
  if (dt == DT_F16) return backward_t<f16_t>(a, act, st);
  return backward_t<float>(a, act, st);
}

}  // namespace moe
