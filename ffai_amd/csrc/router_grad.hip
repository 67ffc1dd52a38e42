// router_grad.hip — the router's losses and the gradient of its logits for
// gfx950.
//
//   balance loss  per-expert counts c_e of the picks, P_e = sum_t p_te over
//                 the counted rows, balance = E sum_e c_e / (k N) P_e / N and
//                 z = sum_t lse(s_t)^2 / N, s = logit_scale * logits
//   backward      d logits of both losses and of the routing weights, every
//                 element written once
//
// No counterpart in the reference, which only runs forward; the rules that
// are differentiated are MoERouter.route's (MoELayer.swift:140-205) and the
// NemotronH sigmoid router's (NemotronHText.swift:838-868).
//
// Both kernels read a row's logits once: a lane holds 8 neighbouring experts
// (16 bytes of a 16-bit row), 2^lg = ceil(E / 8) lanes hold a row and a wave
// 64 / 2^lg rows, so that the row's maximum and sums take lg steps for all of
// a wave's rows together. Sums stay in fp32 along a fixed tree; only integer
// atomics are used on shared counts, so results do not depend on the order
// of blocks or waves.
#include <algorithm>

#include "moe_common.hpp"
#include "moe_internal.hpp"

namespace moe {

namespace {

constexpr int kCols = 8;  // experts per lane

// Eight logits of a row as fp32, `pad` past E. vec: E % 8 == 0 and 16-byte
// aligned rows.
template <typename XT>
__device__ __forceinline__ void load_cols(const XT* __restrict__ row, int c0, int E, bool vec,
                                          float pad, float (&v)[kCols]) {
  if (vec) {
#pragma unroll
    for (int j = 0; j < kCols; j++) v[j] = pad;
    if (c0 < E) Vec8<XT>::load(row + c0, v);
  } else {
#pragma unroll
    for (int j = 0; j < kCols; j++) {
      const float x = to_f<XT>(row[min(c0 + j, E - 1)]);
      v[j] = c0 + j < E ? x : pad;
    }
  }
}

template <typename XT>
__device__ __forceinline__ void store_cols(XT* __restrict__ row, int c0, int E, bool vec,
                                           const float (&v)[kCols]) {
  if (vec) {
    if (c0 < E) Vec8<XT>::store(row + c0, v);
  } else {
#pragma unroll
    for (int j = 0; j < kCols; j++)
      if (c0 + j < E) row[c0 + j] = from_f<XT>(v[j]);
  }
}

// v and the v of the lane 16 (32) away, in either order: v_permlane16_swap
// exchanges the odd rows of 16 lanes of one register with the even rows of the
// other (permlane32: halves of 32), both holding v.
struct Halves {
  float a, b;
};
__device__ __forceinline__ Halves swap16(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return {__uint_as_float(r[0]), __uint_as_float(r[1])};
}
__device__ __forceinline__ Halves swap32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return {__uint_as_float(r[0]), __uint_as_float(r[1])};
}

// Sum / maximum over each aligned group of 2^LG lanes, in every lane of it.
template <int LG> __device__ __forceinline__ float row_sum(float v) {
  if constexpr (LG >= 1) v += dpp_f32<0xB1, 0xF>(0.f, v);
  if constexpr (LG >= 2) v += dpp_f32<0x4E, 0xF>(0.f, v);
  if constexpr (LG >= 3) v += dpp_f32<0x141, 0xF>(0.f, v);
  if constexpr (LG >= 4) v += dpp_f32<0x140, 0xF>(0.f, v);
  if constexpr (LG >= 5) {
    const Halves h = swap16(v);
    v = h.a + h.b;
  }
  if constexpr (LG >= 6) {
    const Halves h = swap32(v);
    v = h.a + h.b;
  }
  return v;
}
template <int LG> __device__ __forceinline__ float row_max(float v) {
  if constexpr (LG >= 1) v = fmaxf(v, dpp_f32<0xB1, 0xF>(v, v));
  if constexpr (LG >= 2) v = fmaxf(v, dpp_f32<0x4E, 0xF>(v, v));
  if constexpr (LG >= 3) v = fmaxf(v, dpp_f32<0x141, 0xF>(v, v));
  if constexpr (LG >= 4) v = fmaxf(v, dpp_f32<0x140, 0xF>(v, v));
  if constexpr (LG >= 5) {
    const Halves h = swap16(v);
    v = fmaxf(h.a, h.b);
  }
  if constexpr (LG >= 6) {
    const Halves h = swap32(v);
    v = fmaxf(h.a, h.b);
  }
  return v;
}

constexpr float kLog2e = 1.44269504088896341f;

// exp(s - m), m the row's maximum, as 2^((s - m) log2(e)): the difference first, so
// that a row far from zero, down to one of the type's lowest value, is as good as
// any (m log2(e) taken off by an fma is one instruction less, at the same time, but
// rounds by up to 2^-24 of itself, a power of its own from |m| of about 2^26 on, and
// overflows). The two roundings, 2^-24 of the exponent each, weigh little where
// the power is large. -inf gives 0 (m finite), NaN stays.
__device__ __forceinline__ float exp_off(float s, float m) {
  return __builtin_amdgcn_exp2f((s - m) * kLog2e);
}

// Row statistics of 2^LG lanes: e_j = exp(s_j - m), 1 / sum e and lse. A row
// of -inf only has e = 0, inv = 0 and lse = 0 (no probability, no loss);
// NaN or +inf in a row makes all of it NaN.
struct RowStat {
  float m, inv, lse;
};
template <int LG>
__device__ __forceinline__ RowStat row_softmax(const float (&s)[kCols], float (&e)[kCols]) {
  float m = s[0];
#pragma unroll
  for (int j = 1; j < kCols; j++) m = fmaxf(m, s[j]);
  m = row_max<LG>(m);
  if (m == -__builtin_huge_valf()) m = 0.f;
  RowStat r;
  r.m = m;
#pragma unroll
  for (int j = 0; j < kCols; j++) e[j] = exp_off(s[j], m);
  float z = 0.f;
#pragma unroll
  for (int j = 0; j < kCols; j++) z += e[j];
  z = row_sum<LG>(z);
  r.inv = z == 0.f ? 0.f : 1.0f / z;
  r.lse = z == 0.f ? 0.f : m + logf(z);
  return r;
}

// exp(-s); the exponent's rounding is put back as a first-order factor (2^d = 1 +
// d ln 2) where the power is finite, since here it does not cancel.
__device__ __forceinline__ float exp_neg_acc(float s) {
  const float t = -s * kLog2e;
  const float e = __builtin_amdgcn_exp2f(t);
  const float d = __builtin_fmaf(-s, kLog2e, -t);
  return __builtin_fabsf(t) < 126.f ? __builtin_fmaf(e, d * 0.69314718f, e) : e;
}

// 1 / (1 + exp(-s)).
__device__ __forceinline__ float sigmoid_acc(float s) { return 1.0f / (1.0f + exp_neg_acc(s)); }

// The sigmoid v and its complement 1 - v = exp(-s) v, which a subtraction from v
// near 1 would round away (at s = 12 to 1 %, from 17 on to 0); 1, which the minimum
// also makes of inf x 0, where the power is past fp32. A NaN is left to v.
struct Sigmoid {
  float v, rest;
};
__device__ __forceinline__ Sigmoid sigmoid_pair(float s) {
  const float e = exp_neg_acc(s), v = 1.0f / (1.0f + e);
  return {v, fminf(e * v, 1.0f)};
}

}  // namespace

// ---------------------------------------------------------- balance loss --
constexpr int kBalWaves = 16;

// The losses from sum_e c_e P_e, sum lse^2 and the counted rows.
__device__ __forceinline__ void store_losses(double dot, double zsum, uint32_t n, int E, int k,
                                             float* losses) {
  const double dn = n ? (double)n : 1.0;
  losses[0] = (float)(dot * (double)E / (dn * dn * (double)k));
  losses[1] = (float)(zsum / dn);
}

// Sum over the wave in its last lane, by DPP (group_sum's steps).
template <int CTRL, int ROW_MASK> __device__ __forceinline__ double dpp_f64(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = (uint32_t)dpp_i32<CTRL, ROW_MASK>(0, (int)(uint32_t)b);
  const uint32_t hi = (uint32_t)dpp_i32<CTRL, ROW_MASK>(0, (int)(uint32_t)(b >> 32));
  return __builtin_bit_cast(double, (uint64_t)lo | ((uint64_t)hi << 32));
}
__device__ __forceinline__ double wave_sum_f64(double v) {
  v += dpp_f64<0xB1, 0xF>(v);
  v += dpp_f64<0x4E, 0xF>(v);
  v += dpp_f64<0x141, 0xF>(v);
  v += dpp_f64<0x140, 0xF>(v);
  v += dpp_f64<0x142, 0xA>(v);
  v += dpp_f64<0x143, 0xC>(v);
  return v;
}

// Partials of block b: P [E4] fp32 and picks [E4] u32 (E4 = E rounded up to
// 4, the rest zeros), then z and the counted rows; then what the second
// launch's blocks leave for the last of them.
constexpr int kBalMaxBlocks = 256, kFinalCols = 32, kFinalBlocks = kTopkMaxE / kFinalCols;
struct BalancePart {
  float* P;
  uint32_t* cnt;
  float* z;
  uint32_t* n;
  double* dot;       // [kFinalBlocks]
  uint32_t* ticket;  // blocks that are done
};
__host__ __device__ inline BalancePart balance_part(void* ws, int nb, int E4) {
  BalancePart p;
  p.P = reinterpret_cast<float*>(ws);
  p.cnt = reinterpret_cast<uint32_t*>(p.P + (size_t)nb * E4);
  p.z = reinterpret_cast<float*>(p.cnt + (size_t)nb * E4);
  p.n = reinterpret_cast<uint32_t*>(p.z + nb);
  p.dot = reinterpret_cast<double*>(p.n + nb);
  p.ticket = reinterpret_cast<uint32_t*>(p.dot + kFinalBlocks);
  return p;
}

struct BalanceArgs {
  const void* logits;
  const uint32_t* idx;
  const uint8_t* mask;  // nullable
  void* ws;
  uint32_t* counts;
  float* prob_sum;
  float* losses;
  int T, E, k, rpb, sigmoid, vec;
  float ls;
};

// Block b takes rows [b rpb, (b + 1) rpb). A lane keeps the probability sums
// of its 8 experts in registers over its rows, the next row's logits in flight;
// the waves' rows and the picks' counts meet in LDS. FULL: rows are 16-byte
// aligned and of exactly 8 * 2^LG experts.
template <typename XT, int LG, bool FULL>
__global__ __launch_bounds__(64 * kBalWaves) void balance_rows_kernel(BalanceArgs a) {
  __shared__ float sP[kBalWaves][kCols << LG];
  __shared__ uint32_t sCnt[kCols << LG];
  __shared__ float sZ[kBalWaves];
  __shared__ uint32_t sN[kBalWaves];
  __shared__ double sDot[kBalWaves];
  constexpr int LPR = 1 << LG, RPW = kWave >> LG, NT = 64 * kBalWaves;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int c0 = (lane & (LPR - 1)) * kCols;
  const int E = FULL ? kCols << LG : a.E, k = a.k;
  const uint8_t* __restrict__ mask = a.mask;
  for (int e = tid; e < (kCols << LG); e += NT) sCnt[e] = 0u;
  __syncthreads();
  const int r0 = blockIdx.x * a.rpb, r1 = min(a.T, r0 + a.rpb);
  const float NEG = -__builtin_huge_valf();
  const XT* __restrict__ logits = reinterpret_cast<const XT*>(a.logits);
  auto load = [&](int r, float (&s)[kCols], bool& on) {
    const int rr = min(r, r1 - 1);
    on = r < r1 && (mask == nullptr || mask[rr] != 0);
    load_cols<XT>(logits + (size_t)rr * E, c0, E, FULL || a.vec, NEG, s);
  };
  float sn[kCols];
  bool on_next;
  const int rw = r0 + wave * RPW + (lane >> LG);
  load(rw, sn, on_next);
  // picks of the block's rows
  {
    const size_t i0 = (size_t)r0 * k;
    const int ne = (r1 - r0) * k;
    for (int i = tid; i < ne; i += NT) {
      const uint32_t e = a.idx[i0 + i];
      const bool on = mask == nullptr || mask[r0 + i / k] != 0;
      if (on && e < (uint32_t)E) atomicAdd(&sCnt[e], 1u);
    }
  }
  float P[kCols];
#pragma unroll
  for (int j = 0; j < kCols; j++) P[j] = 0.f;
  float zs = 0.f;
  uint32_t n = 0;
  for (int rb = rw; __any(rb < r1); rb += kBalWaves * RPW) {
    float s[kCols], e[kCols];
    const bool on = on_next;
#pragma unroll
    for (int j = 0; j < kCols; j++) s[j] = FULL || c0 + j < E ? sn[j] * a.ls : NEG;
    load(rb + kBalWaves * RPW, sn, on_next);
    const RowStat st = row_softmax<LG>(s, e);
    float inv = st.inv;
    if (a.sigmoid) {
      float z = 0.f;
#pragma unroll
      for (int j = 0; j < kCols; j++) {
        e[j] = sigmoid_acc(s[j]);
        z += e[j];
      }
      z = row_sum<LG>(z);
      inv = z == 0.f ? 0.f : 1.0f / z;
    }
    if (on) {
#pragma unroll
      for (int j = 0; j < kCols; j++) P[j] = __builtin_fmaf(e[j], inv, P[j]);
      zs = __builtin_fmaf(st.lse, st.lse, zs);
      n++;
    }
  }
  // rows of the wave (z and n are the same in all lanes of a row), then the
  // block's waves
#pragma unroll
  for (int off = LPR; off < kWave; off <<= 1) {
#pragma unroll
    for (int j = 0; j < kCols; j++) P[j] += __shfl_xor(P[j], off, kWave);
    zs += __shfl_xor(zs, off, kWave);
    n += (uint32_t)__shfl_xor((int)n, off, kWave);
  }
  if (lane < LPR) {
#pragma unroll
    for (int j = 0; j < kCols; j += 4)
      *reinterpret_cast<float4*>(&sP[wave][c0 + j]) = make_float4(P[j], P[j + 1], P[j + 2], P[j + 3]);
  }
  if (lane == 0) {
    sZ[wave] = zs;
    sN[wave] = n;
  }
  __syncthreads();
  const int E4 = (E + 3) & ~3;
  float p = 0.f;  // thread e: expert e's sum over the block
  if (tid < E4) {
#pragma unroll
    for (int w = 0; w < kBalWaves; w += 2) p += sP[w][tid] + sP[w + 1][tid];
    p = tid < E ? p : 0.f;
  }
  float z = 0.f;
  uint32_t nn = 0;
#pragma unroll
  for (int w = 0; w < kBalWaves; w++) {
    z += sZ[w];
    nn += sN[w];
  }
  if (gridDim.x == 1) {
    // the only block has everything: the losses without a second launch
    double dot = 0.0;
    if (tid < E) {
      a.prob_sum[tid] = p;
      a.counts[tid] = sCnt[tid];
      dot = (double)p * (double)sCnt[tid];
    }
    dot = wave_sum_f64(dot);
    if (lane == 63) sDot[wave] = dot;
    __syncthreads();
    if (tid == 0) {
      double all = 0.0;
      const int waves = (E + 63) / 64;
      for (int w = 0; w < waves; w++) all += sDot[w];
      a.counts[E] = nn;
      store_losses(all, (double)z, nn, E, k, a.losses);
    }
    return;
  }
  const BalancePart bp = balance_part(a.ws, gridDim.x, E4);
  if (tid < E4) {
    bp.P[(size_t)blockIdx.x * E4 + tid] = p;
    bp.cnt[(size_t)blockIdx.x * E4 + tid] = tid < E ? sCnt[tid] : 0u;
  }
  if (tid == 0) {
    bp.z[blockIdx.x] = z;
    bp.n[blockIdx.x] = nn;
    if (blockIdx.x == 0) *bp.ticket = 0u;
  }
}

// Adds the blocks' partials: a block per 32 experts (a CU reads about 100
// bytes a nanosecond, 256 x 256 partials are 512 KB: one block took 6.9 us), four
// experts a thread (16-byte loads), 128 threads across the partials. The last
// block to finish, by a ticket that the launch before set to 0, adds the
// blocks' parts of sum_e c_e P_e in their order and forms the losses.
__global__ __launch_bounds__(1024) void balance_final_kernel(void* ws, int nb, int E, int k,
                                                             uint32_t* __restrict__ counts,
                                                             float* __restrict__ prob_sum,
                                                             float* __restrict__ losses) {
  __shared__ float sP[16][kFinalCols];
  __shared__ uint32_t sC[16][kFinalCols];
  __shared__ double sZ[4];
  __shared__ uint32_t sN[4];
  const int E4 = (E + 3) & ~3;
  const BalancePart bp = balance_part(ws, nb, E4);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int c0 = blockIdx.x * kFinalCols, e0 = c0 + (tid & 7) * 4;
  const float zb = tid < nb ? bp.z[tid] : 0.f;
  const uint32_t nbk = tid < nb ? bp.n[tid] : 0u;
  float p[4] = {0.f, 0.f, 0.f, 0.f};
  uint32_t c[4] = {0u, 0u, 0u, 0u};
  if (e0 < E4) {
    float4 v[2];
    uint4 w[2];
#pragma unroll
    for (int i = 0; i < kBalMaxBlocks / 128; i++) {
      const int b = (tid >> 3) + i * 128;
      v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      w[i] = make_uint4(0u, 0u, 0u, 0u);
      if (b < nb) {
        v[i] = *reinterpret_cast<const float4*>(bp.P + (size_t)b * E4 + e0);
        w[i] = *reinterpret_cast<const uint4*>(bp.cnt + (size_t)b * E4 + e0);
      }
    }
    p[0] = v[0].x + v[1].x; p[1] = v[0].y + v[1].y; p[2] = v[0].z + v[1].z; p[3] = v[0].w + v[1].w;
    c[0] = w[0].x + w[1].x; c[1] = w[0].y + w[1].y; c[2] = w[0].z + w[1].z; c[3] = w[0].w + w[1].w;
  }
  // the wave's eight threads per four experts, then the waves
#pragma unroll
  for (int j = 0; j < 4; j++) {
    p[j] += dpp_f32<0x128, 0xF>(0.f, p[j]);  // row_ror:8
    c[j] += (uint32_t)dpp_i32<0x128, 0xF>(0, (int)c[j]);
    Halves h = swap16(p[j]);
    p[j] = h.a + h.b;
    h = swap32(p[j]);
    p[j] = h.a + h.b;
    c[j] += (uint32_t)__shfl_xor((int)c[j], 16, kWave);
    c[j] += (uint32_t)__shfl_xor((int)c[j], 32, kWave);
  }
  if (lane < 8) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
      sP[wave][lane * 4 + j] = p[j];
      sC[wave][lane * 4 + j] = c[j];
    }
  }
  if (wave < 4) {  // up to 256 blocks
    const double z = wave_sum_f64((double)zb);
    const uint32_t n = wave_scan_u32(nbk);
    if (lane == 63) {
      sZ[wave] = z;
      sN[wave] = n;
    }
  }
  __syncthreads();
  if (wave != 0) return;
  double dot = 0.0;
  if (lane < kFinalCols && c0 + lane < E) {
    double pe = 0.0;
    uint32_t ce = 0;
#pragma unroll
    for (int w = 0; w < 16; w += 2) {
      pe += (double)(sP[w][lane] + sP[w + 1][lane]);
      ce += sC[w][lane] + sC[w + 1][lane];
    }
    prob_sum[c0 + lane] = (float)pe;
    counts[c0 + lane] = ce;
    dot = pe * (double)ce;
  }
  dot = wave_sum_f64(dot);
  if (lane != 63) return;
  if (gridDim.x > 1) {
    __hip_atomic_store(&bp.dot[blockIdx.x], dot, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const uint32_t done = __hip_atomic_fetch_add(bp.ticket, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
    if (done + 1 != gridDim.x) return;
    dot = 0.0;
    for (uint32_t b = 0; b < gridDim.x; b++)
      dot += __hip_atomic_load(&bp.dot[b], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  const uint32_t n = (sN[0] + sN[1]) + (sN[2] + sN[3]);
  counts[E] = n;
  store_losses(dot, (sZ[0] + sZ[1]) + (sZ[2] + sZ[3]), n, E, k, losses);
}

namespace {

int lanes_lg(int E) {
  int lg = 0;
  while ((kCols << lg) < E) lg++;
  return lg;
}

// Blocks of a balance pass: one, which needs no second launch, for up to five
// rounds of its waves (four rounds take 6.7 us in a graph and 8.7 us called one
// by one, two launches 8.5 and 12.7; eight rounds 10.4 and 10.0), otherwise up
// to 256, one per CU, of at least a row per wave slot.
int balance_blocks(int T, int E) {
  const int rows = kBalWaves * (kWave >> lanes_lg(E));  // a block's rows in flight
  if (T <= 5 * rows) return 1;
  return (int)std::min<long>(kBalMaxBlocks, (T + rows - 1) / rows);
}

}  // namespace

size_t balance_ws_bytes(int T, int E) {
  const int nb = balance_blocks(T, E);
  return nb == 1 ? 0 : (size_t)nb * (((E + 3) & ~3) + 1) * 8 + kFinalBlocks * 8 + 8;
}

#define MOE_LG(lg, MACRO) \
  switch (lg) {           \
    case 0: MACRO(0)      \
    case 1: MACRO(1)      \
    case 2: MACRO(2)      \
    case 3: MACRO(3)      \
    case 4: MACRO(4)      \
    case 5: MACRO(5)      \
    case 6: MACRO(6)      \
  }

template <typename XT>
static hipError_t balance_typed(const void* logits, int T, int E, int k, bool sigmoid, float ls,
                                const uint32_t* idx, const uint8_t* mask, uint32_t* counts,
                                float* prob_sum, float* losses, void* ws, hipStream_t st) {
  int nb = balance_blocks(T, E);
  const int rpb = (T + nb - 1) / nb;
  nb = (T + rpb - 1) / rpb;
  const int vec = E % kCols == 0 && (reinterpret_cast<uintptr_t>(logits) & 15) == 0;
  const int lg = lanes_lg(E);
  const bool full = vec && E == kCols << lg;
  const BalanceArgs a{logits, idx, mask, ws, counts, prob_sum, losses, T, E, k, rpb, (int)sigmoid, vec, ls};
#define MOE_BL(LG)                                                                                      \
  if (full) hipLaunchKernelGGL((balance_rows_kernel<XT, LG, true>), dim3(nb), dim3(64 * kBalWaves), 0, st, a); \
  else hipLaunchKernelGGL((balance_rows_kernel<XT, LG, false>), dim3(nb), dim3(64 * kBalWaves), 0, st, a);     \
  break;
  MOE_LG(lg, MOE_BL)
#undef MOE_BL
  if (nb > 1)
    hipLaunchKernelGGL(balance_final_kernel, dim3((E + kFinalCols - 1) / kFinalCols), dim3(1024), 0, st,
                       ws, nb, E, k, counts, prob_sum, losses);
  return hipGetLastError();
}

hipError_t launch_balance_loss(const void* logits, int dt, int T, int E, int k, bool sigmoid,
                               float ls, const uint32_t* idx, const uint8_t* mask,
                               uint32_t* counts, float* prob_sum, float* losses, void* ws,
                               hipStream_t st) {
  if (E > kTopkMaxE) return hipErrorInvalidValue;
  if (dt == DT_BF16)
    return balance_typed<bf16_t>(logits, T, E, k, sigmoid, ls, idx, mask, counts, prob_sum, losses, ws, st);
  if (dt == DT_F16)
    return balance_typed<f16_t>(logits, T, E, k, sigmoid, ls, idx, mask, counts, prob_sum, losses, ws, st);
  return balance_typed<float>(logits, T, E, k, sigmoid, ls, idx, mask, counts, prob_sum, losses, ws, st);
}

// -------------------------------------------------------------- backward --
// d logits, with s = ls * logits, p / q the row's softmax / normalised
// sigmoids, f_e = balance_coef E c_e / (k N^2):
//   balance, softmax    p_j (f_j - sum f p)
//   balance, sigmoid    q_j (1 - sigmoid(s_j)) (f_j - sum f q)
//   z                   z_coef 2 / N lse p_j
//   weights             g_r = d_weight_r routed_scale escale[e_r] of the picks:
//     softmax over the picks  w_r (g_r - sum g w)
//     full softmax (+ bias)   d p_r = g_r, or (g_r - sum g v / S) / S of the
//                             renormalised v_r = p_r + ebias, S = sum v; then
//                             p_j (dp_j - sum dp p)
//     sigmoid                 (the same with v = sigmoid, S = sum v + 1e-20)
//                             times v (1 - v)
// all times ls. The picks' values are added into a row image in LDS, from
// which every lane takes its 8 experts (an id that appears twice adds twice).
// Rows whose mask is 0 get zeros whatever they hold.
enum { kPickSoftmax = 0, kFullSoftmax = 1, kSigmoid = 2 };

struct RouterGradArgs {
  const void* logits;
  const uint32_t* idx;
  const float* dw;         // nullable [T, k]
  const uint32_t* counts;  // nullable [E + 1]
  const uint8_t* mask;     // nullable [T]
  const float* ebias;      // nullable [E]
  const float* escale;     // nullable [E]
  void* out;
  int T, E, k, mode, sigmoid, norm, vec;
  float ls, rs, bal, z;
};

// NP: picks per lane, 1 where k fits a row's lanes, else 8 (k <= E <= 8 lanes).
template <typename XT, int LG, bool FULL, int NP>
__global__ __launch_bounds__(256) void router_backward_kernel(RouterGradArgs a) {
  constexpr int LPR = 1 << LG, RPW = kWave >> LG;
  __shared__ __attribute__((aligned(16))) float img[4][kWave * kCols];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int rl = lane & (LPR - 1), c0 = rl * kCols, E = FULL ? kCols << LG : a.E, k = a.k;
  float* im = &img[wave][(lane >> LG) * (LPR * kCols)];  // this row's image
  const float NEG = -__builtin_huge_valf();
  float f[kCols];
  float zc = 0.f;
#pragma unroll
  for (int j = 0; j < kCols; j++) f[j] = 0.f;
  if (a.counts) {
    const uint32_t n = a.counts[E];
    const float fn = n ? (float)n : 1.0f;
    const float fs = a.bal * (float)E / ((float)k * fn) / fn;
    zc = a.z * 2.0f / fn;
#pragma unroll
    for (int j = 0; j < kCols; j++)
      if (FULL || c0 + j < E) f[j] = fs * (float)a.counts[c0 + j];
  }
  const XT* __restrict__ logits = reinterpret_cast<const XT*>(a.logits);
  XT* __restrict__ out = reinterpret_cast<XT*>(a.out);
  for (long rb = ((long)blockIdx.x * 4 + wave) * RPW; rb < a.T; rb += (long)gridDim.x * 4 * RPW) {
    const long r = rb + (lane >> LG);
    const bool in = r < a.T;
    const size_t rr = (size_t)(in ? r : a.T - 1);
    const XT* __restrict__ row = logits + rr * E;
    // everything the row needs is asked for at once: its mask, picks rl, rl +
    // LPR, ... with their gradients, its logits, then the picks' own logits
    const uint32_t mk = a.mask ? a.mask[rr] : 1u;
    float v[NP], g[NP];
    uint32_t pe[NP];
    if (a.dw) {
#pragma unroll
      for (int i = 0; i < NP; i++) {
        const int q = rl + i * LPR;
        const size_t at = rr * k + min(q, k - 1);
        pe[i] = a.idx[at];
        g[i] = a.dw[at];
        if (q >= k) pe[i] = 0xFFFFFFFFu;
      }
    }
    float s[kCols], p[kCols];
    load_cols<XT>(row, c0, E, FULL || a.vec, NEG, s);
    if (a.dw) {
#pragma unroll
      for (int i = 0; i < NP; i++) {
        const bool ok = pe[i] < (uint32_t)E;
        const uint32_t e = ok ? pe[i] : 0u;
        v[i] = to_f<XT>(row[e]);
        g[i] *= a.rs * (a.escale ? a.escale[e] : 1.0f);
        v[i] = ok ? v[i] * a.ls : NEG;
        g[i] = ok ? g[i] : 0.f;
        pe[i] = ok ? pe[i] : 0xFFFFFFFFu;
      }
    }
    const bool on = in && mk != 0;
#pragma unroll
    for (int j = 0; j < kCols; j++) s[j] = FULL || c0 + j < E ? s[j] * a.ls : NEG;
    const RowStat st = row_softmax<LG>(s, p);
#pragma unroll
    for (int j = 0; j < kCols; j++) p[j] *= st.inv;
    // the losses: d_j and the row sum it is centred by. What is not asked for is
    // left out, not multiplied by 0: an infinite logit makes p NaN, but not the
    // sigmoids, nor the weights of picks beside it
    float d[kCols];
    const float zl = zc * st.lse;
    if (a.sigmoid) {
      float q[kCols], rest[kCols], S = 0.f;
#pragma unroll
      for (int j = 0; j < kCols; j++) {
        const Sigmoid sg = sigmoid_pair(s[j]);
        q[j] = sg.v;
        rest[j] = sg.rest;
        S += sg.v;
      }
      S = row_sum<LG>(S);
      const float inv = S == 0.f ? 0.f : 1.0f / S;
      float c = 0.f;
#pragma unroll
      for (int j = 0; j < kCols; j++) {
        q[j] *= inv;
        c = __builtin_fmaf(q[j], f[j], c);
      }
      c = row_sum<LG>(c);
#pragma unroll
      for (int j = 0; j < kCols; j++) d[j] = q[j] * rest[j] * (f[j] - c);
      if (a.z != 0.f) {
#pragma unroll
        for (int j = 0; j < kCols; j++) d[j] = __builtin_fmaf(zl, p[j], d[j]);
      }
    } else {
      float c = 0.f;
#pragma unroll
      for (int j = 0; j < kCols; j++) c = __builtin_fmaf(p[j], f[j], c);
      c = row_sum<LG>(c);
#pragma unroll
      for (int j = 0; j < kCols; j++) d[j] = p[j] * (f[j] - c + zl);
    }
    if (!a.counts) {
#pragma unroll
      for (int j = 0; j < kCols; j++) d[j] = 0.f;
    }
    if (a.dw) {
      // zero image
#pragma unroll
      for (int j = 0; j < kCols; j += 4)
        *reinterpret_cast<float4*>(im + c0 + j) = make_float4(0.f, 0.f, 0.f, 0.f);
      wave_sync();
      float mx = NEG;
#pragma unroll
      for (int i = 0; i < NP; i++) mx = fmaxf(mx, v[i]);
      float S = 0.f, G = 0.f;  // sum of the weights before renormalising, sum g v
      if (a.mode == kPickSoftmax) {
        mx = row_max<LG>(mx);
        mx = mx == NEG ? 0.f : mx;
#pragma unroll
        for (int i = 0; i < NP; i++)
          if ((NP == 1 || i * LPR < k)) {
            v[i] = exp_off(v[i], mx);
            S += v[i];
            G = __builtin_fmaf(g[i], v[i], G);
          }
        S = row_sum<LG>(S);
        G = row_sum<LG>(G);
        const float inv = S == 0.f ? 0.f : 1.0f / S;
        G *= inv;
#pragma unroll
        for (int i = 0; i < NP; i++)
          if ((NP == 1 || i * LPR < k)) g[i] = v[i] * inv * (g[i] - G);
      } else {
        float pv[NP];  // p of the pick (full softmax) or sigmoid' (sigmoid)
#pragma unroll
        for (int i = 0; i < NP; i++) {
          pv[i] = 0.f;
          if ((NP == 1 || i * LPR < k)) {
            if (a.mode == kSigmoid) {
              const Sigmoid sg = sigmoid_pair(v[i]);
              v[i] = sg.v;
              pv[i] = sg.v * sg.rest;
            } else {
              v[i] = exp_off(v[i], st.m) * st.inv;
              pv[i] = v[i];
              if (a.ebias && pe[i] != 0xFFFFFFFFu) v[i] += a.ebias[pe[i]];
            }
            S += v[i];
            G = __builtin_fmaf(g[i], v[i], G);
          }
        }
        S = row_sum<LG>(S);
        G = row_sum<LG>(G);
        const bool renorm = a.norm && (a.mode == kSigmoid ? k > 1 : S > 0.f);
        const float inv = renorm ? 1.0f / (a.mode == kSigmoid ? S + 1e-20f : S) : 1.0f;
        const float Gn = renorm ? G * inv : 0.f;
        float c = 0.f;
#pragma unroll
        for (int i = 0; i < NP; i++)
          if ((NP == 1 || i * LPR < k)) {
            g[i] = (g[i] - Gn) * inv;
            if (a.mode == kSigmoid) g[i] *= pv[i];
            else c = __builtin_fmaf(g[i], pv[i], c);
          }
        if (a.mode == kFullSoftmax) {
          c = row_sum<LG>(c);
#pragma unroll
          for (int j = 0; j < kCols; j++) d[j] = __builtin_fmaf(-p[j], c, d[j]);
#pragma unroll
          for (int i = 0; i < NP; i++) g[i] *= pv[i];
        }
      }
#pragma unroll
      for (int i = 0; i < NP; i++)
        if ((NP == 1 || i * LPR < k) && pe[i] != 0xFFFFFFFFu) unsafeAtomicAdd(im + pe[i], g[i]);
      wave_sync();
#pragma unroll
      for (int j = 0; j < kCols; j += 4) {
        const float4 t = *reinterpret_cast<const float4*>(im + c0 + j);
        d[j] += t.x; d[j + 1] += t.y; d[j + 2] += t.z; d[j + 3] += t.w;
      }
      wave_sync();
    }
#pragma unroll
    for (int j = 0; j < kCols; j++) d[j] = on ? d[j] * a.ls : 0.f;
    if (in) store_cols<XT>(out + rr * E, c0, E, FULL || a.vec, d);
  }
}

hipError_t launch_router_backward(const void* logits, int dt, int T, int E, int k,
                                  const RouteOpts& ro, const uint32_t* idx, const float* dw,
                                  const uint32_t* counts, float bal, float z, const uint8_t* mask,
                                  void* out, hipStream_t st) {
  if (E > kTopkMaxE) return hipErrorInvalidValue;
  RouterGradArgs a{};
  a.logits = logits;
  a.idx = idx;
  a.dw = dw;
  a.counts = counts;
  a.mask = mask;
  a.ebias = ro.ebias;
  a.escale = ro.escale;
  a.out = out;
  a.T = T;
  a.E = E;
  a.k = k;
  a.sigmoid = ro.gating == 2;
  a.norm = ro.norm;
  // as wave_topk forms the weights: softmax over the picks for top-k then
  // softmax and for a renormalised softmax without a bias
  a.mode = ro.gating == 2 ? kSigmoid
           : (ro.gating == 1 || (ro.norm && ro.ebias == nullptr)) ? kPickSoftmax : kFullSoftmax;
  a.vec = E % kCols == 0 &&
          ((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  a.ls = ro.logit_scale;
  a.rs = ro.routed_scale;
  a.bal = bal;
  a.z = z;
  const int lg = lanes_lg(E);
  const int rows = 4 * (kWave >> lg);
  const int grid = (int)std::min<long>(2048, ((long)T + rows - 1) / rows);
  const bool full = a.vec && E == kCols << lg, one = k <= 1 << lg;
#define MOE_RB3(XT, LG, FULL, NP) \
  hipLaunchKernelGGL((router_backward_kernel<XT, LG, FULL, NP>), dim3(grid), dim3(256), 0, st, a)
#define MOE_RB2(XT, LG)                  \
  if (full && one) MOE_RB3(XT, LG, true, 1);  \
  else if (full) MOE_RB3(XT, LG, true, 8);    \
  else if (one) MOE_RB3(XT, LG, false, 1);    \
  else MOE_RB3(XT, LG, false, 8);             \
  break;
#define MOE_RB_B(LG) MOE_RB2(bf16_t, LG)
#define MOE_RB_H(LG) MOE_RB2(f16_t, LG)
#define MOE_RB_F(LG) MOE_RB2(float, LG)
  if (dt == DT_BF16) { MOE_LG(lg, MOE_RB_B) }
  else if (dt == DT_F16) { MOE_LG(lg, MOE_RB_H) }
  else { MOE_LG(lg, MOE_RB_F) }
#undef MOE_RB_B
#undef MOE_RB_H
#undef MOE_RB_F
#undef MOE_RB2
#undef MOE_RB3
  return hipGetLastError();
}

}  // namespace moe
