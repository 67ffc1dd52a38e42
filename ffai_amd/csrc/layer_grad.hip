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

// Eight values as they lie in memory.
template <typename XT>
struct Raw8 {
  uint4 v[sizeof(XT) / 2];
  __device__ __forceinline__ void load(const XT* p) {
#pragma unroll
    for (size_t i = 0; i < sizeof(XT) / 2; i++) v[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void stream(const XT* p) {  // keeps no place in the caches
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (size_t i = 0; i < sizeof(XT) / 2; i++) v[i] = __builtin_bit_cast(uint4, __builtin_nontemporal_load(reinterpret_cast<const u4*>(p) + i));
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(v);
#pragma unroll
    for (int j = 0; j < 8; j++) {
      if constexpr (sizeof(XT) == 4)
        f[j] = __uint_as_float(w[j]);
      else
        f[j] = to_f<XT>(__builtin_bit_cast(XT, (uint16_t)(w[j >> 1] >> (16 * (j & 1)))));
    }
  }
};

// dx[t] = round(dx_in[t] + sum_s dX[inv[t*k + s]]), eight columns per thread,
// the chunks of all tokens side by side so that narrow rows fill blocks too.
// Up to kRankBatch rows in flight, as they lie in memory until all are there; the ranks
// are added in order. Each row is read once, so its loads leave the caches to others.
// Bound by memory: 4096 tokens of 8 rows of 2048, bf16, added to a gradient take 29 us
// (5.8 TB/s where a large copy reaches 5.2); with ordinary loads 32, with each row
// converted where it is loaded 36.
constexpr int kRankBatch = 8;

template <typename XT>
__global__ __launch_bounds__(256) void permute_backward_kernel(const XT* __restrict__ dX,
                                                               const uint32_t* __restrict__ inv, int T,
                                                               int H, int k, const XT* dx_in, XT* dx) {
  const uint32_t M = (uint32_t)T * (uint32_t)k, chunks = (uint32_t)H / 8;
  const int64_t all = (int64_t)T * chunks;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const int64_t t = all < (int64_t)1 << 32 ? (int64_t)((uint32_t)i / chunks) : i / chunks;
    const int h = (int)(i - t * chunks) * 8;
    float acc[8] = {};
    if (dx_in) Vec8<XT>::load(dx_in + t * H + h, acc);
    for (int s0 = 0; s0 < k; s0 += kRankBatch) {
      uint32_t p[kRankBatch];
#pragma unroll
      for (int q = 0; q < kRankBatch; q++) p[q] = s0 + q < k ? inv[t * k + s0 + q] : 0xFFFFFFFFu;
      Raw8<XT> v[kRankBatch];
#pragma unroll
      for (int q = 0; q < kRankBatch; q++)
        if (p[q] < M) v[q].stream(dX + (size_t)p[q] * H + h);
#pragma unroll
      for (int q = 0; q < kRankBatch; q++)
        if (p[q] < M) {
          float f[8];
          v[q].get(f);
#pragma unroll
          for (int j = 0; j < 8; j++) acc[j] += f[j];
        }
    }
    Vec8<XT>::store(dx + t * H + h, acc);
  }
}

hipError_t launch_permute_backward(const void* dX, const uint32_t* inv, int T, int H, int k,
                                   const void* dx_in, void* dx, int dt, hipStream_t st) {
  const dim3 grid((unsigned)std::min<int64_t>(((int64_t)T * (H / 8) + 255) / 256, 1 << 22));
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
// Both row sums come from one pass over the row, which stays in registers: a team
// of W waves takes a row, each lane up to C pieces of 8 columns, and keeps its
// columns' share of dw over all its rows. A 16-bit row is loaded while the one
// before is worked on. The blocks' shares of dw meet in a second launch, in a
// fixed order; few rows are one block's. Bound by memory: 8192 rows of 2048, bf16,
// with a residual's gradient take 24.5 + 4 us (134 MB, 5.5 TB/s in the first launch).
struct NormBackward {
  const void *r, *w, *dn, *dr;
  void* din;
  float* dw;  // [blocks, H] partial sums, or the result where there is one block
  float eps;
  int T, H;
};

template <typename XT, int C, int W>
__global__ __launch_bounds__(256) void norm_backward_kernel(const NormBackward a) {
  constexpr int TEAMS = 4 / W, COLS = 512 * W;  // columns of a piece across a team
  constexpr bool AHEAD = sizeof(XT) == 2;
  __shared__ float part[2][4][2];
  __shared__ __align__(16) float sums[TEAMS > 1 ? TEAMS : 1][TEAMS > 1 ? C * COLS : 4];
  const int H = a.H, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, team = wave / W;
  const int h0 = (threadIdx.x % (64 * W)) * 8;
  Raw8<XT> w[C], r[C], g[C], d[C];
#pragma unroll
  for (int c = 0; c < C; c++)
    if (h0 + c * COLS < H) w[c].load((const XT*)a.w + h0 + c * COLS);
  auto load = [&](int64_t t) {
    if (t >= a.T) return;
#pragma unroll
    for (int c = 0; c < C; c++) {
      const int h = h0 + c * COLS;
      if (h < H) {
        r[c].load((const XT*)a.r + t * H + h);
        g[c].load((const XT*)a.dn + t * H + h);
        if (a.dr) d[c].load((const XT*)a.dr + t * H + h);
      }
    }
  };
  float dw[C][8] = {};
  int turn = 0;
  const int64_t step = (int64_t)gridDim.x * TEAMS;
  if (AHEAD) load((int64_t)blockIdx.x * TEAMS + team);
  for (int64_t base = (int64_t)blockIdx.x * TEAMS; base < a.T; base += step, turn ^= 1) {
    const int64_t t = base + team;
    if (!AHEAD) load(t);
    const bool on = t < a.T;
    float ss = 0.0f, sg = 0.0f;
    Raw8<XT> rc[C], gc[C], dc[C];
#pragma unroll
    for (int c = 0; c < C; c++) {
      if (on && h0 + c * COLS < H) {
        rc[c] = r[c];
        gc[c] = g[c];
        dc[c] = d[c];
        float rv[8], gv[8], wv[8];
        rc[c].get(rv);
        gc[c].get(gv);
        w[c].get(wv);
#pragma unroll
        for (int j = 0; j < 8; j++) {
          ss = __builtin_fmaf(rv[j], rv[j], ss);
          sg = __builtin_fmaf(gv[j] * wv[j], rv[j], sg);
        }
      }
    }
    if (AHEAD) load(t + step);
    ss = group_sum(ss, 6);
    sg = group_sum(sg, 6);
    if constexpr (W == 1) {
      ss = lane_f32(ss, 63);
      sg = lane_f32(sg, 63);
    } else {
      if (lane == 63) {
        part[turn][wave][0] = ss;
        part[turn][wave][1] = sg;
      }
      lds_barrier();
      ss = sg = 0.0f;
#pragma unroll
      for (int i = 0; i < W; i++) {
        ss += part[turn][team * W + i][0];
        sg += part[turn][team * W + i][1];
      }
    }
    const float s = 1.0f / sqrtf(ss / (float)H + a.eps);
    const float m = s * sg / (float)H;  // mean(dn w n)
#pragma unroll
    for (int c = 0; c < C; c++) {
      const int h = h0 + c * COLS;
      if (on && h < H) {
        float rv[8], gv[8], wv[8], o[8] = {};
        rc[c].get(rv);
        gc[c].get(gv);
        w[c].get(wv);
        if (a.dr) dc[c].get(o);
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const float n = rv[j] * s;
          o[j] += s * (gv[j] * wv[j] - n * m);
          dw[c][j] = __builtin_fmaf(gv[j], n, dw[c][j]);
        }
        Vec8<XT>::store((XT*)a.din + t * H + h, o);
      }
    }
  }
  float* out = a.dw + (size_t)blockIdx.x * H;
  if constexpr (TEAMS == 1) {
#pragma unroll
    for (int c = 0; c < C; c++)
      if (h0 + c * COLS < H) Vec8<float>::store(out + h0 + c * COLS, dw[c]);
  } else {
#pragma unroll
    for (int c = 0; c < C; c++) Vec8<float>::store(&sums[team][h0 + c * COLS], dw[c]);
    __syncthreads();
    for (int h = threadIdx.x * 4; h < H; h += 1024) {
      float4 v = *reinterpret_cast<const float4*>(&sums[0][h]);
#pragma unroll
      for (int i = 1; i < TEAMS; i++) {
        const float4 u = *reinterpret_cast<const float4*>(&sums[i][h]);
        v = make_float4(v.x + u.x, v.y + u.y, v.z + u.z, v.w + u.w);
      }
      *reinterpret_cast<float4*>(out + h) = v;
    }
  }
}

// Adds the blocks' shares: 32 columns a block, 32 runs of blocks in order, then
// the runs along a tree.
__global__ __launch_bounds__(1024) void norm_weight_kernel(const float* __restrict__ part, int blocks, int H,
                                                           float* __restrict__ dw) {
  __shared__ float sums[32][33];
  const int col = threadIdx.x & 31, run = threadIdx.x >> 5, h = blockIdx.x * 32 + col;
  const int per = (blocks + 31) / 32, b0 = run * per, b1 = min(b0 + per, blocks);
  float s = 0.0f;
  if (h < H)
#pragma unroll 8
    for (int b = b0; b < b1; b++) s += part[(size_t)b * H + h];
  sums[run][col] = s;
  __syncthreads();
  float v = sums[col][run];  // thread (run, col) now holds run col of column run
#pragma unroll
  for (int off = 16; off; off >>= 1) v += __shfl_xor(v, off, 32);
  if (col == 0 && blockIdx.x * 32 + run < H) dw[blockIdx.x * 32 + run] = v;
}

namespace {

// Waves per row: a lane holds up to three pieces (four above 6144 columns), two of
// fp32 with four waves a SIMD. 4096 rows of 2880, bf16: two waves 20.1 us, four (a third
// of whose lanes have nothing to do) 24.2; of 4096 two waves 25.5, four 26.2, fp32 60.0
// and 50.4. One / two / four waves at 8192 rows of 2048, fp32:
// 57.2 / 49.2 / 47.5 us, bf16 27.8 / 27.4 / 27.7; at 16384 rows of 512 bf16 15.2 / - / 28.9.
int norm_waves(int H) { return H <= 1024 ? 1 : (H <= 3 * 1024 ? 2 : 4); }
// Two blocks a CU (four a CU 29.5 us where two take 27.4, one a CU 37 where two take
// 29). Up to six rows a team one block alone takes less than a second launch: 8 rows
// of 2048 8.6 us for 13.3, 32 rows 19.9 for 13.1.
constexpr int kNormBlocks = 512, kNormAlone = 6;

int norm_blocks(int T, int H) {
  const int teams = 4 / norm_waves(H);
  return T <= kNormAlone * teams ? 1 : std::min((T + teams - 1) / teams, kNormBlocks);
}

template <typename XT>
hipError_t norm_t(const NormBackward& a, int blocks, hipStream_t st) {
  const int W = norm_waves(a.H), C = (a.H + 512 * W - 1) / (512 * W);
#define MOE_NB(CC, WW)                                                                       \
  if (C == CC && W == WW) {                                                                  \
    hipLaunchKernelGGL((norm_backward_kernel<XT, CC, WW>), dim3(blocks), dim3(256), 0, st, a); \
    return hipGetLastError();                                                                \
  }
  MOE_NB(1, 1)
  MOE_NB(2, 1)
  MOE_NB(2, 2)
  MOE_NB(3, 2)
  MOE_NB(2, 4)
  MOE_NB(3, 4)
  MOE_NB(4, 4)
#undef MOE_NB
  return hipErrorInvalidValue;
}

}  // namespace

size_t norm_backward_ws_bytes(int T, int H) {
  const int blocks = norm_blocks(T, H);
  return blocks > 1 ? (size_t)blocks * H * 4 : 0;
}

hipError_t launch_norm_backward(const void* r, const void* w, const void* dn, const void* dr, float eps,
                                int T, int H, int dt, void* din, float* dw, void* ws, hipStream_t st) {
  const int blocks = norm_blocks(T, H);
  const NormBackward a{r, w, dn, dr, din, blocks > 1 ? (float*)ws : dw, eps, T, H};
  const hipError_t e = dt == DT_BF16  ? norm_t<bf16_t>(a, blocks, st)
                       : dt == DT_F16 ? norm_t<f16_t>(a, blocks, st)
                                      : norm_t<float>(a, blocks, st);
  if (e != hipSuccess || blocks == 1) return e;
  hipLaunchKernelGGL(norm_weight_kernel, dim3((H + 31) / 32), dim3(1024), 0, st, (const float*)ws, blocks, H, dw);
  return hipGetLastError();
}

}  // namespace moe
