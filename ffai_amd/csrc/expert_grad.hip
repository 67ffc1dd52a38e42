// expert_grad.hip — gradient of the grouped dequantising product
// (moe_expert_matmul) with respect to its rows, for gfx950:
//
//   dx[p, j] = round(dx_in[p, j] + sum_i dy[row(p), i] W[e(p)][i, j]
//                                [ + sum_i dy2[row(p), i] W2[e(p)][i, j] ])
//
// W = scale * q + bias as stored for the forward ([n, k], packed along k): the
// sum runs along W's rows and the packed axis is the output's. The reference
// only runs forward (Ops.swift:4553-5201).
#include <algorithm>

#include "moe_common.hpp"
#include "moe_internal.hpp"

#ifndef MOE_BITS
#define MOE_BITS 4
#endif

namespace moe {

typedef float f32x16_t __attribute__((ext_vector_type(16)));

// Row tile number `tile` of the plan, tiles of R rows, experts ascending:
// its expert, first sorted position and end. Every lane of a wave calls it;
// false past the last tile. total: all tiles of the plan.
struct GradTile {
  uint32_t e, m0, pend;
};
__device__ __forceinline__ uint32_t grad_tiles(const uint32_t* offsets, int E, uint32_t R) {
  const int lane = threadIdx.x & 63;
  uint32_t sum = 0;
  for (int e0 = 0; e0 < E; e0 += 64) {
    const int e = e0 + lane;
    if (e < E) sum += (offsets[e + 1] - offsets[e] + R - 1) / R;
  }
  return (uint32_t)__builtin_amdgcn_readlane((int)wave_scan_u32(sum), 63);
}
__device__ __forceinline__ bool grad_tile(const uint32_t* offsets, int E, uint32_t R, uint32_t tile, GradTile* t) {
  const int lane = threadIdx.x & 63;
  uint32_t before = 0;
  for (int e0 = 0; e0 < E; e0 += 64) {
    const int e = e0 + lane;
    const uint32_t lo = e < E ? offsets[e] : 0u, hi = e < E ? offsets[e + 1] : 0u;
    const uint32_t own = (hi - lo + R - 1) / R, upto = before + wave_scan_u32(own);
    const uint64_t past = __ballot(upto > tile);
    if (past) {
      const int at = __ffsll((unsigned long long)past) - 1;
      const uint32_t first = (uint32_t)__builtin_amdgcn_readlane((int)(upto - own), at);
      const uint32_t l = (uint32_t)__builtin_amdgcn_readlane((int)lo, at);
      t->e = (uint32_t)(e0 + at);
      t->m0 = l + (tile - first) * R;
      t->pend = min((uint32_t)__builtin_amdgcn_readlane((int)hi, at), t->m0 + R);
      return true;
    }
    before = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
  }
  return false;
}

// ------------------------------------------------------------ fp32 products --
// A block takes 64 rows and 64 columns, a wave a 32 x 32 quarter; 32 values of
// the sum at a time go through LDS in fp32 (the gradient's rows as they are,
// the weights dequantised, which keeps the packed axis across the lanes).
constexpr int kFR = 64, kFC = 64, kFK = 32;

template <int BITS, typename XT, typename ST>
__global__ __launch_bounds__(256) void expert_grad_f32_kernel(const ExpertGradArgs a) {
  __shared__ float As[kFR][kFK + 1], Bs[kFK][kFC];
  const uint32_t nb = (uint32_t)((a.K + kFC - 1) / kFC);
  GradTile t;
  if (!grad_tile(a.offsets, a.E, kFR, blockIdx.x / nb, &t)) return;
  const int j0 = (int)(blockIdx.x % nb) * kFC, tid = threadIdx.x;
  const int lane = tid & 63, wave = tid >> 6, wm = wave >> 1, wn = wave & 1;
  const int col = lane & 31, half = lane >> 5;
  const int words = a.K / 32 * BITS, groups = a.K / 32 >> a.gsh;
  f32x16_t acc = {};
  for (int part = 0; part < (a.dy2 ? 2 : 1); part++) {
    const GemvProj& p = part ? a.p1 : a.p0;
    const XT* dy = (const XT*)(part ? a.dy2 : a.dy);
    const uint32_t* W = p.w + (size_t)t.e * a.N * words;
    const ST* S = (const ST*)p.s + (size_t)t.e * a.N * groups;
    const ST* B = (const ST*)p.b + (size_t)t.e * a.N * groups;
    // thread: a quarter of a gradient row's chunk, eight columns of a weight row
    const uint32_t pos = min(t.m0 + (uint32_t)(tid >> 2), t.pend - 1);
    const size_t arow = a.perm ? a.perm[pos] / (uint32_t)a.topk : pos;
    const int ac = (tid & 3) * 8, bi = tid >> 3, bj = j0 + (tid & 7) * 8;
    for (int i0 = 0; i0 < a.N; i0 += kFK) {
      float av[8] = {}, bv[8] = {};
      if (i0 + ac < a.N) Vec8<XT>::load(dy + arow * a.N + i0 + ac, av);
      const int i = i0 + bi;
      if (i < a.N && bj < a.K) {
        const uint32_t* row = W + (size_t)i * words;
        const size_t g = (size_t)i * groups + (bj / 32 >> a.gsh);
        const float s = to_f<ST>(S[g]), b = to_f<ST>(B[g]);
#pragma unroll
        for (int v = 0; v < 8; v++) {
          const uint32_t bit = (uint32_t)(bj + v) * BITS, lo = bit >> 5, sh = bit & 31;
          uint32_t q = row[lo] >> sh;
          if (sh + BITS > 32) q |= row[lo + 1] << (32 - sh);
          bv[v] = __builtin_fmaf(s, (float)(q & ((1u << BITS) - 1u)), b);
        }
      }
      __syncthreads();
#pragma unroll
      for (int v = 0; v < 8; v++) {
        As[tid >> 2][ac + v] = av[v];
        Bs[bi][(tid & 7) * 8 + v] = bv[v];
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < kFK; k += 2)
        acc = __builtin_amdgcn_mfma_f32_32x32x2f32(As[32 * wm + col][k + half], Bs[k + half][32 * wn + col], acc, 0, 0, 0);
    }
  }
  const int j = j0 + 32 * wn + col;
#pragma unroll
  for (int r = 0; r < 16; r++) {
    const uint32_t pos = t.m0 + (uint32_t)(32 * wm + 8 * (r >> 2) + 4 * half + (r & 3));
    if (pos < t.pend && j < a.K) {
      const size_t at = (size_t)pos * a.K + j;
      const float base = a.dx_in ? to_f<XT>(((const XT*)a.dx_in)[at]) : 0.0f;
      ((XT*)a.dx)[at] = from_f<XT>(base + acc[r]);
    }
  }
}

template <int BITS, typename XT, typename ST>
static hipError_t launch_f32(const ExpertGradArgs& a, hipStream_t st) {
  const int64_t tiles = a.M / kFR + std::min(a.E, a.M), nb = (a.K + kFC - 1) / kFC;
  hipLaunchKernelGGL((expert_grad_f32_kernel<BITS, XT, ST>), dim3((unsigned)(tiles * nb)), dim3(256), 0, st, a);
  return hipGetLastError();
}

#define MOE_CAT2(a, b) a##b
#define MOE_CAT(a, b) MOE_CAT2(a, b)

hipError_t MOE_CAT(launch_expert_grad_b, MOE_BITS)(int xdt, int sbdt, const ExpertGradArgs& a, hipStream_t st) {
  if (xdt == DT_F32) return launch_f32<MOE_BITS, float, float>(a, st);
  if (xdt == DT_BF16)
    return sbdt == DT_BF16 ? launch_f32<MOE_BITS, bf16_t, bf16_t>(a, st) : launch_f32<MOE_BITS, bf16_t, f16_t>(a, st);
  return sbdt == DT_BF16 ? launch_f32<MOE_BITS, f16_t, bf16_t>(a, st) : launch_f32<MOE_BITS, f16_t, f16_t>(a, st);
}

}  // namespace moe
