// lora.hip — low-rank adapters of many requests beside a shared projection,
// forward and backward, for gfx950.
//
//   forward    y_t  = y_t + scale_g B_g (A_g x_t),  g = adapter[t]
//   backward   u_t  = scale_g B_g^T dy_t
//              dx_t = dx_t + A_g^T u_t
//              dA_g = sum_t u_t x_t^T,  dB_g = sum_t dy_t (scale_g A_g x_t)^T
//
// A row whose id is not in [0, n_adapters) has no adapter: its y and dx stay
// as they are, it adds to no gradient. No counterpart in the reference, whose
// adapters are merged into the weights before loading.
//
// Everything is small products along K or N against R (8 .. 128) columns: two
// operations per loaded value and rank, far below the matrix cores' ratio, so
// the kernels are made to read x, y and the adapters once, in whole lines, and
// to spread few rows over the chip.
#include <algorithm>

#include "moe_common.hpp"
#include "moe_internal.hpp"

namespace moe {

namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

constexpr uint32_t kOut = 0x7FFFFFF0u;  // past the end of every view: reads 0
constexpr int kTile = 16;               // rows per matrix tile

// D += A B^T over 16 x 16 tiles: lane (c, q) = (lane % 16, lane / 16) holds
// 16 bytes of row c of either operand (8 values of a 16-bit type, k = 8 q ..,
// one instruction; 4 floats, k = 4 q .., four instructions) and D[4 q + i][c].
template <typename XT>
__device__ __forceinline__ f32x4_t mma(u32x4_t a, u32x4_t b, f32x4_t c) {
  if constexpr (__is_same(XT, bf16_t)) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                   __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  } else if constexpr (__is_same(XT, f16_t)) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a),
                                                  __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
    return c;
  }
}

// The adapter of tile row c (rows past the tile's end and ids out of range:
// -1), the same in all four lane groups.
__device__ __forceinline__ int tile_adapter(const int32_t* __restrict__ adapter, int t0, int rows,
                                            int c, int G) {
  const int a = c < rows ? adapter[t0 + c] : -1;
  return (uint32_t)a < (uint32_t)G ? a : -1;
}

}  // namespace

// ---------------------------------------------------------------- shrink --
// s[z][t][r] = sum over the z-th share of K of x[t][k] a[g][r][k]. One block
// per tile of 16 rows, share of K and share of the tile's distinct adapters
// (blockIdx.y-th, + gridDim.y, ...): a tile whose rows belong to one request
// is one pass, a decode tile of 16 requests is spread over 16 blocks that
// each read one adapter. The four waves take units of 128 bytes per row in
// turn and meet in LDS.
struct ShrinkArgs {
  const void* x;           // [T, K]
  const void* a;           // [G, R, K]
  const int32_t* adapter;  // [T]
  float* s;                // [gridDim.z, T, R]
  int T, K, R, G;
};

template <typename XT, int RT>
__global__ __launch_bounds__(256) void lora_shrink_kernel(ShrinkArgs p) {
  constexpr int V = 16 / sizeof(XT);   // values per load
  constexpr int UNIT = 8 * V;          // values per unit: two loads of four lane groups
  constexpr int LD = RT * 16 + 4;
  __shared__ __attribute__((aligned(16))) float red[4][kTile * LD];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, q = lane >> 4;
  const int t0 = blockIdx.x * kTile, rows = min(kTile, p.T - t0);
  const int ad = tile_adapter(p.adapter, t0, rows, c, p.G);
  const int K = p.K, R = p.R;
  const rsrc_t xr = make_rsrc((const XT*)p.x + (size_t)t0 * K, (uint32_t)((size_t)rows * K * sizeof(XT)));
  const int units = (K + UNIT - 1) / UNIT;
  uint32_t rem = (uint32_t)__ballot(ad >= 0) & 0xFFFFu;
  for (int d = 0; rem; d++) {
    const int lead = __builtin_ctz(rem);
    const int g = __builtin_amdgcn_readlane(ad, lead);
    const uint32_t same = (uint32_t)__ballot(ad == g) & 0xFFFFu;
    rem &= ~same;
    if (d % (int)gridDim.y != (int)blockIdx.y) continue;
    const rsrc_t ar = make_rsrc((const XT*)p.a + (size_t)g * R * K, (uint32_t)((size_t)R * K * sizeof(XT)));
    f32x4_t acc[RT] = {};
    for (int u = blockIdx.z * 4 + wave; u < units; u += 4 * gridDim.z) {
      u32x4_t xv[2], av[2][RT];
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int k = u * UNIT + h * 4 * V + q * V;
        const bool in = k < K;
        xv[h] = bload128(xr, in ? (uint32_t)(c * K + k) * (uint32_t)sizeof(XT) : kOut);
#pragma unroll
        for (int i = 0; i < RT; i++) {
          const int r = i * 16 + c;
          av[h][i] = bload128(ar, in && r < R ? (uint32_t)(r * K + k) * (uint32_t)sizeof(XT) : kOut);
        }
      }
#pragma unroll
      for (int h = 0; h < 2; h++)
#pragma unroll
        for (int i = 0; i < RT; i++) acc[i] = mma<XT>(av[h][i], xv[h], acc[i]);
    }
#pragma unroll
    for (int i = 0; i < RT; i++)
      *reinterpret_cast<f32x4_t*>(&red[wave][c * LD + i * 16 + 4 * q]) = acc[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < RT; i++) {
      const int e = i * 256 + tid, t = e / (RT * 16), r = e % (RT * 16);
      const int at = t * LD + r;
      const float v = (red[0][at] + red[1][at]) + (red[2][at] + red[3][at]);
      if (r < R && ((same >> t) & 1u))
        p.s[((size_t)blockIdx.z * p.T + t0 + t) * R + r] = v;
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------- expand --
// y[t][n] = round(y_in[t][n] + sum_r scale_g s[t][r] b[g][n][r]), s summed
// over its shares of K. A wave takes 16 rows x 64 columns: the b rows are the
// matrix operand whose row m of the j-th product is column 16 (m / 4) + 4 j +
// m % 4, so that lane (c, q) ends with 16 neighbouring columns (q) of row c.
//
// For 16-bit adapters s enters the product as two 16-bit parts, hi = round(s)
// and lo = round(s - hi), laid side by side along the product's 32-value
// inner axis (against the same b values), which keeps 16 (f16: 22) bits of
// it: for rank 16 one instruction holds both. f16 rows are first scaled by a
// power of two to a maximum in [2^14, 2^15), so that neither part over- or
// underflows, and the sum back afterwards.
struct ExpandArgs {
  const float* s;          // [S, T, R]
  const void* b;           // [G, N, R]
  const float* scale;      // nullable [G]
  const int32_t* adapter;  // [T]
  const void* yin;         // nullable [T, N], may be y
  void* y;                 // [T, N]
  int T, N, R, G, S;
};

template <typename XT, int RT>
__global__ __launch_bounds__(256) void lora_expand_kernel(ExpandArgs p) {
  constexpr bool F32 = sizeof(XT) == 4;
  constexpr int V = 16 / sizeof(XT);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, q = lane >> 4;
  const int t0 = blockIdx.x * kTile, rows = min(kTile, p.T - t0);
  const int ad = tile_adapter(p.adapter, t0, rows, c, p.G);
  const int N = p.N, R = p.R;
  const int nb = (blockIdx.z * 4 + wave) * 64;
  if (nb >= N) return;
  const XT* yin = (const XT*)p.yin;
  XT* y = (XT*)p.y;
  const int c8 = R / V;  // 16-byte chunks of an adapter row
  uint32_t rem = (1u << rows) - 1u;
  for (int d = 0; rem; d++) {
    const int lead = __builtin_ctz(rem);
    const int g = __builtin_amdgcn_readlane(ad, lead);
    const uint32_t same = (uint32_t)__ballot(ad == g) & rem;
    rem &= ~same;
    if (d % (int)gridDim.y != (int)blockIdx.y) continue;
    if (g < 0 && p.yin == p.y) continue;  // rows without an adapter, in place
    f32x4_t acc[4] = {};
    float back = 1.f;
    if (g >= 0) {
      const float sc = p.scale ? p.scale[g] : 1.f;
      // this lane's chunks of s (row c): values 8 cc .. (16-bit), 4 cc ..
      u32x4_t sv[RT];
      float v[RT][8];
#pragma unroll
      for (int i = 0; i < RT; i++) {
        const int ci = 4 * i + q;
        const int cc = F32 || ci < c8 ? ci : ci - c8;
        const bool in = cc < c8 && c < rows;
#pragma unroll
        for (int j = 0; j < 8; j++) v[i][j] = 0.f;
        if (in) {
          for (int z = 0; z < p.S; z++) {
            const float* at = p.s + ((size_t)z * p.T + t0 + c) * R + cc * V;
#pragma unroll
            for (int j = 0; j < V; j += 4) {
              const float4 f = *reinterpret_cast<const float4*>(at + j);
              v[i][j] += f.x; v[i][j + 1] += f.y; v[i][j + 2] += f.z; v[i][j + 3] += f.w;
            }
          }
        }
#pragma unroll
        for (int j = 0; j < V; j++) v[i][j] *= sc;
      }
      // rows of other adapters hold no sums of this one (or none at all):
      // they take zeros, and are not stored
      const bool mine = (same >> c) & 1u;
      if constexpr (__is_same(XT, f16_t)) {
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < RT; i++)
#pragma unroll
          for (int j = 0; j < V; j++) m = fmaxf(m, fabsf(v[i][j]));
        m = fmaxf(m, __shfl_xor(m, 16, kWave));
        m = fmaxf(m, __shfl_xor(m, 32, kWave));
        const int eb = (int)((__float_as_uint(m) >> 23) & 255u);
        const int sh = eb == 255 ? 0 : min(14 - (eb - 127), 100);
        back = __builtin_ldexpf(1.f, -sh);
        const float fw = __builtin_ldexpf(1.f, sh);
#pragma unroll
        for (int i = 0; i < RT; i++)
#pragma unroll
          for (int j = 0; j < V; j++) v[i][j] *= fw;
      }
#pragma unroll
      for (int i = 0; i < RT; i++) {
        if constexpr (F32) {
#pragma unroll
          for (int j = 0; j < 4; j++) sv[i][j] = mine ? __float_as_uint(v[i][j]) : 0u;
        } else {
          const bool lo = 4 * i + q >= c8;
          uint32_t h[8];
#pragma unroll
          for (int j = 0; j < 8; j++) {
            const float hi = round_to<XT>(v[i][j]);
            const float rest = __builtin_isfinite(hi) ? v[i][j] - hi : 0.f;
            h[j] = mine ? (uint32_t)__builtin_bit_cast(uint16_t, from_f<XT>(lo ? rest : hi)) : 0u;
          }
#pragma unroll
          for (int j = 0; j < 4; j++) sv[i][j] = h[2 * j] | (h[2 * j + 1] << 16);
        }
      }
      const rsrc_t br = make_rsrc((const XT*)p.b + (size_t)g * N * R, (uint32_t)((size_t)N * R * sizeof(XT)));
#pragma unroll
      for (int i = 0; i < RT; i++) {
        const int ci = 4 * i + q;
        const int cc = F32 || ci < c8 ? ci : ci - c8;
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int n = nb + 16 * (c >> 2) + 4 * j + (c & 3);
          const u32x4_t bv = bload128(br, cc < c8 && n < N ? (uint32_t)(n * R + cc * V) * (uint32_t)sizeof(XT) : kOut);
          acc[j] = mma<XT>(bv, sv[i], acc[j]);
        }
      }
    }
    if ((same >> c) & 1u) {
      const size_t row = (size_t)(t0 + c) * N;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int n = nb + 16 * q + 8 * h;
        if (n < N) {
          float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
          if (yin) Vec8<XT>::load(yin + row + n, o);
#pragma unroll
          for (int j = 0; j < 8; j++)
            o[j] = g < 0 ? o[j] : __builtin_fmaf(acc[2 * h + (j >> 2)][j & 3], back, o[j]);
          Vec8<XT>::store(y + row + n, o);
        }
      }
    }
  }
}

// ------------------------------------------------------------- transpose --
// [G, P, Q] -> [G, Q, P] by tiles of 32 x 32 through LDS: the backward's
// products run along the other axis of A and B.
template <typename E>
__global__ __launch_bounds__(256) void lora_transpose_kernel(const E* __restrict__ in,
                                                             E* __restrict__ out, int P, int Q) {
  __shared__ E tile[32][33];
  const size_t base = (size_t)blockIdx.z * P * Q;
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int p0 = blockIdx.y * 32, q0 = blockIdx.x * 32;
#pragma unroll
  for (int i = y; i < 32; i += 8)
    if (p0 + i < P && q0 + x < Q) tile[i][x] = in[base + (size_t)(p0 + i) * Q + q0 + x];
  __syncthreads();
#pragma unroll
  for (int i = y; i < 32; i += 8)
    if (q0 + i < Q && p0 + x < P) out[base + (size_t)(q0 + i) * P + p0 + x] = tile[x][i];
}

// ----------------------------------------------------- adapter gradients --
// dA_g[r][k] = sum_t u[t][r] x[t][k] and dB_g[n][r] = sum_t s[t][r] dy[t][n]
// over the rows of adapter g, which a dispatch plan lists (perm, offsets).
// fp32 matrix products of 4 rows a step: a lane reads 8 neighbouring columns
// of one row, each of which is one product's operand, so the wide rows go
// from memory to the operand registers as they lie. A block takes 4 x 128
// columns, up to two rank tiles and a share of the adapter's rows; with more
// than one share the fp32 partials are added by lora_sum_kernel.
struct OuterSide {
  const void* wide;    // [T, cols]: x or dy
  const float* small;  // [S, T, R]: u or s before scale
  void* out;           // the gradient, or its fp32 partials [shares, G, ...]
  int cols, S;
  int rank_major;      // out [R, cols] (dA) or [cols, R] (dB)
};
struct OuterArgs {
  OuterSide side[2];
  const uint32_t* perm;
  const uint32_t* offsets;
  const float* scale;
  int T, R, G, sides, shares;
};

template <typename XT, typename OT, int RB>
__global__ __launch_bounds__(256) void lora_outer_kernel(OuterArgs p) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, q = lane >> 4;
  const int g = (int)blockIdx.z / p.sides;
  const OuterSide& sd = p.side[(int)blockIdx.z % p.sides];
  const int share = (int)blockIdx.y % p.shares, r0 = (int)blockIdx.y / p.shares * (RB * 16);
  const int R = p.R, cols = sd.cols;
  const int cb = (blockIdx.x * 4 + wave) * 128;
  if (cb >= cols) return;
  const int col = cb + 8 * c;
  const uint32_t o0 = p.offsets[g], o1 = p.offsets[g + 1];
  const uint32_t len = (o1 - o0 + p.shares - 1) / p.shares;
  const uint32_t b0 = min(o1, o0 + share * len), b1 = min(o1, b0 + len);
  const float sc = p.scale ? p.scale[g] : 1.f;
  f32x4_t acc[RB][8] = {};
  for (uint32_t at = b0; at < b1; at += 4) {
    const bool in = at + q < b1;
    const uint32_t t = in ? p.perm[at + q] : 0u;
    float w[8], s[RB];
#pragma unroll
    for (int j = 0; j < 8; j++) w[j] = 0.f;
    if (in && col < cols) Vec8<XT>::load((const XT*)sd.wide + (size_t)t * cols + col, w);
#pragma unroll
    for (int i = 0; i < RB; i++) {
      const int r = r0 + i * 16 + c;
      s[i] = 0.f;
      if (in && r < R) {
        for (int z = 0; z < sd.S; z++) s[i] += sd.small[((size_t)z * p.T + t) * R + r];
        s[i] *= sc;
      }
    }
#pragma unroll
    for (int i = 0; i < RB; i++)
#pragma unroll
      for (int j = 0; j < 8; j++)
        acc[i][j] = sd.rank_major ? __builtin_amdgcn_mfma_f32_16x16x4f32(s[i], w[j], acc[i][j], 0, 0, 0)
                                  : __builtin_amdgcn_mfma_f32_16x16x4f32(w[j], s[i], acc[i][j], 0, 0, 0);
  }
  OT* out = (OT*)sd.out + ((size_t)share * p.G + g) * R * cols;
#pragma unroll
  for (int i = 0; i < RB; i++) {
#pragma unroll
    for (int h = 0; h < 4; h++) {
      if (sd.rank_major) {
        const int r = r0 + i * 16 + 4 * q + h;
        if (r < R && col < cols) {
          float o[8];
#pragma unroll
          for (int j = 0; j < 8; j++) o[j] = acc[i][j][h];
          Vec8<OT>::store(out + (size_t)r * cols + col, o);
        }
      } else {
        const int r = r0 + i * 16 + c;
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const int n = cb + 8 * (4 * q + h) + j;
          if (r < R && n < cols) out[(size_t)n * R + r] = from_f<OT>(acc[i][j][h]);
        }
      }
    }
  }
}

// out[i] = sum over the shares of their fp32 partials, 8 values a thread.
template <typename XT>
__global__ __launch_bounds__(256) void lora_sum_kernel(const float* __restrict__ part,
                                                       XT* __restrict__ out, int64_t n, int shares) {
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8; i < n; i += (int64_t)gridDim.x * 2048) {
    float a[8];
    Vec8<float>::load(part + i, a);
    for (int z = 1; z < shares; z++) {
      float b[8];
      Vec8<float>::load(part + (size_t)z * n + i, b);
#pragma unroll
      for (int j = 0; j < 8; j++) a[j] += b[j];
    }
    Vec8<XT>::store(out + i, a);
  }
}

// ------------------------------------------------------------------ host --
namespace {

int tiles_of(int T) { return (T + kTile - 1) / kTile; }

// Blocks that share a tile's distinct adapters: as many as a tile can hold
// while the launch is small, one where the tiles alone fill the chip.
int leaders(int T, int G, bool none) {
  const int most = std::min(std::min(kTile, T), G + (none ? 1 : 0));
  return std::max(1, std::min(most, 1024 / tiles_of(T)));
}

template <typename XT>
hipError_t shrink_typed(const ShrinkArgs& a, int S, hipStream_t st) {
  const dim3 grid(tiles_of(a.T), leaders(a.T, a.G, false), S);
#define MOE_SH(RT) hipLaunchKernelGGL((lora_shrink_kernel<XT, RT>), grid, dim3(256), 0, st, a)
  if (a.R <= 16) MOE_SH(1);
  else if (a.R <= 32) MOE_SH(2);
  else if (a.R <= 64) MOE_SH(4);
  else MOE_SH(8);
#undef MOE_SH
  return hipGetLastError();
}

template <typename XT>
hipError_t expand_typed(const ExpandArgs& a, hipStream_t st) {
  const dim3 grid(tiles_of(a.T), leaders(a.T, a.G, true), (a.N + 255) / 256);
#define MOE_EX(RT) hipLaunchKernelGGL((lora_expand_kernel<XT, RT>), grid, dim3(256), 0, st, a)
  if (a.R <= 16) MOE_EX(1);
  else if (a.R <= 32) MOE_EX(2);
  else if (a.R <= 64) MOE_EX(4);
  else MOE_EX(8);
#undef MOE_EX
  return hipGetLastError();
}

// Rows of a shrink launch's output over all its shares, at most, for up to T
// rows (lora_shares keeps shares x blocks within 512), so that a workspace
// sized for many rows also serves a call of few.
size_t partial_rows(int T, int G) {
  return std::max((size_t)T, std::min((size_t)T * 16, (size_t)512 * kTile / std::min(kTile, G)));
}

size_t up256(size_t v) { return (v + 255) / 256 * 256; }

// Shares of the adapters' rows in the outer products.
int outer_shares(const LoraDims& d) {
  const int es = d.dt == DT_F32 ? 4 : 2;
  (void)es;
  const long blocks = (long)d.G * 2 * ((std::max(d.K, d.N) + 511) / 512) * ((d.R + 31) / 32);
  return (int)std::max(1L, std::min({512 / blocks, (long)(d.T + 63) / 64, 16L}));
}

struct BackwardLayout {
  size_t s, u, at, bt, counts, offsets, perm, inv, used, scratch, scratch_bytes, part, total;
};
BackwardLayout backward_layout(const LoraDims& d) {
  BackwardLayout l{};
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += up256(bytes);
    return o;
  };
  const size_t es = d.dt == DT_F32 ? 4 : 2, T = d.T, R = d.R, G = d.G, K = d.K, N = d.N;
  l.s = take(partial_rows(d.T, d.G) * R * 4);
  l.u = take(partial_rows(d.T, d.G) * R * 4);
  l.at = take(G * K * R * es);
  l.bt = take(G * N * R * es);
  l.counts = take(G * 4);
  l.offsets = take((G + 1) * 4);
  l.perm = take(T * 4);
  l.inv = take(T * 4);
  l.used = take((G + 1) * 4);
  l.scratch_bytes = dispatch_scratch_bytes(d.T, 1, d.G);
  l.scratch = take(l.scratch_bytes);
  const size_t sh = outer_shares(d);
  l.part = take(sh > 1 ? sh * G * R * (K + N) * 4 : 0);
  l.total = at;
  return l;
}

template <typename XT>
hipError_t backward_typed(const LoraDims& d, const LoraBackward& a, hipStream_t st) {
  const BackwardLayout l = backward_layout(d);
  char* ws = reinterpret_cast<char*>(a.ws);
  float* s = reinterpret_cast<float*>(ws + l.s);
  float* u = reinterpret_cast<float*>(ws + l.u);
  XT* at = reinterpret_cast<XT*>(ws + l.at);
  XT* bt = reinterpret_cast<XT*>(ws + l.bt);
  const bool grads = a.da || a.db;
  hipError_t e;
#define MOE_OKAY(expr) \
  if ((e = (expr)) != hipSuccess) return e
  const int Ss = lora_shares(d.T, d.G, d.K, d.dt), Su = lora_shares(d.T, d.G, d.N, d.dt);
  if (a.dx || a.da) {
    hipLaunchKernelGGL((lora_transpose_kernel<XT>), dim3((d.R + 31) / 32, (d.N + 31) / 32, d.G),
                       dim3(256), 0, st, (const XT*)a.b, bt, d.N, d.R);
    MOE_OKAY(hipGetLastError());
    const ShrinkArgs sh{a.dy, bt, a.adapter, u, d.T, d.N, d.R, d.G};
    MOE_OKAY(shrink_typed<XT>(sh, Su, st));
  }
  if (a.dx) {
    hipLaunchKernelGGL((lora_transpose_kernel<XT>), dim3((d.K + 31) / 32, (d.R + 31) / 32, d.G),
                       dim3(256), 0, st, (const XT*)a.a, at, d.R, d.K);
    MOE_OKAY(hipGetLastError());
    const ExpandArgs ex{u, at, a.scale, a.adapter, a.dx_in, a.dx, d.T, d.K, d.R, d.G, Su};
    MOE_OKAY(expand_typed<XT>(ex, st));
  }
  if (!grads) return hipSuccess;
  if (a.db) {
    const ShrinkArgs sh{a.x, a.a, a.adapter, s, d.T, d.K, d.R, d.G};
    MOE_OKAY(shrink_typed<XT>(sh, Ss, st));
  }
  uint32_t* offsets = reinterpret_cast<uint32_t*>(ws + l.offsets);
  uint32_t* perm = reinterpret_cast<uint32_t*>(ws + l.perm);
  MOE_OKAY(launch_dispatch_plan(reinterpret_cast<const uint32_t*>(a.adapter), d.T, 1, d.G,
                                reinterpret_cast<uint32_t*>(ws + l.counts), offsets, perm,
                                reinterpret_cast<uint32_t*>(ws + l.inv),
                                reinterpret_cast<uint32_t*>(ws + l.used), ws + l.scratch,
                                l.scratch_bytes, st));
  OuterArgs o{};
  o.perm = perm;
  o.offsets = offsets;
  o.scale = a.scale;
  o.T = d.T;
  o.R = d.R;
  o.G = d.G;
  o.shares = outer_shares(d);
  const size_t na = (size_t)d.G * d.R * d.K, nb = (size_t)d.G * d.R * d.N;
  float* pa = reinterpret_cast<float*>(ws + l.part);
  float* pb = pa + (size_t)o.shares * na;
  int cols = 0;
  if (a.da) {
    o.side[o.sides++] = {a.x, u, o.shares > 1 ? (void*)pa : a.da, d.K, Su, 1};
    cols = std::max(cols, d.K);
  }
  if (a.db) {
    o.side[o.sides++] = {a.dy, s, o.shares > 1 ? (void*)pb : a.db, d.N, Ss, 0};
    cols = std::max(cols, d.N);
  }
  const int RB = d.R <= 16 ? 1 : 2;
  const dim3 grid((cols + 511) / 512, o.shares * ((d.R + RB * 16 - 1) / (RB * 16)), d.G * o.sides);
#define MOE_OU(OT, RB) hipLaunchKernelGGL((lora_outer_kernel<XT, OT, RB>), grid, dim3(256), 0, st, o)
  if (o.shares > 1) {
    if (RB == 1) MOE_OU(float, 1);
    else MOE_OU(float, 2);
  } else {
    if (RB == 1) MOE_OU(XT, 1);
    else MOE_OU(XT, 2);
  }
#undef MOE_OU
  MOE_OKAY(hipGetLastError());
  if (o.shares > 1) {
    auto add = [&](const float* part, void* out, size_t n) {
      const int gr = (int)std::min<size_t>((n + 2047) / 2048, 2048);
      hipLaunchKernelGGL((lora_sum_kernel<XT>), dim3(gr), dim3(256), 0, st, part, (XT*)out, (int64_t)n, o.shares);
      return hipGetLastError();
    };
    if (a.da) MOE_OKAY(add(pa, a.da, na));
    if (a.db) MOE_OKAY(add(pb, a.db, nb));
  }
#undef MOE_OKAY
  return hipSuccess;
}

}  // namespace

// Shares of the inner axis in a shrink launch: enough for two blocks per CU
// when there are few rows, at least one unit for each of a block's waves.
int lora_shares(int T, int G, int K, int dt) {
  const int unit = dt == DT_F32 ? 32 : 64;
  const int units = (K + unit - 1) / unit;
  const int blocks = tiles_of(T) * std::min(std::min(kTile, T), G);
  return std::max(1, std::min({512 / blocks, units / 4, 16}));
}

size_t lora_ws_bytes(const LoraDims& d) {
  return up256(partial_rows(d.T, d.G) * d.R * 4);
}
size_t lora_backward_ws_bytes(const LoraDims& d) { return backward_layout(d).total; }

hipError_t launch_lora(const LoraDims& d, const void* x, const void* a, const void* b,
                       const float* scale, const int32_t* adapter, const void* yin, void* y,
                       void* ws, hipStream_t st) {
  const int S = lora_shares(d.T, d.G, d.K, d.dt);
  float* s = reinterpret_cast<float*>(ws);
  const ShrinkArgs sh{x, a, adapter, s, d.T, d.K, d.R, d.G};
  const ExpandArgs ex{s, b, scale, adapter, yin, y, d.T, d.N, d.R, d.G, S};
#define MOE_LO(XT)                                   \
  {                                                  \
    const hipError_t e = shrink_typed<XT>(sh, S, st); \
    return e != hipSuccess ? e : expand_typed<XT>(ex, st); \
  }
  if (d.dt == DT_BF16) MOE_LO(bf16_t)
  if (d.dt == DT_F16) MOE_LO(f16_t)
  MOE_LO(float)
#undef MOE_LO
}

hipError_t launch_lora_backward(const LoraDims& d, const LoraBackward& a, hipStream_t st) {
  if (d.dt == DT_BF16) return backward_typed<bf16_t>(d, a, st);
  if (d.dt == DT_F16) return backward_typed<f16_t>(d, a, st);
  return backward_typed<float>(d, a, st);
}

}  // namespace moe
