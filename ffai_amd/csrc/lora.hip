// lora.hip — low-rank adapters of many requests beside a shared projection,
// forward and backward, for gfx950.
//
//   forward    y_t  = y_t + scale_g B_g (A_g x_t),  g = adapter[t]
//   backward   u_t  = scale_g B_g^T dy_t
//              dx_t = dx_t + A_g^T u_t
//              dA_g = sum_t u_t x_t^T,  dB_g = sum_t dy_t (scale_g A_g x_t)^T
//
// A row whose id is not in [0, n_adapters) has no adapter: its y and dx stay
// as they are, it adds to no gradient. No counterpart in the reference.
//
// Everything is small products along K or N against R (8 .. 128) columns: two
// operations per loaded value and rank, far below the matrix cores' ratio, so
// the kernels are made to read x, y and the adapters once, in whole lines, and
// to spread few rows over the chip.
#include <algorithm>
#include <utility>

#include "moe_common.hpp"
#include "moe_internal.hpp"

namespace moe {

namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

constexpr uint32_t kOut = 0x7FFFFFF0u;  // past the end of every view: reads 0
// A lane offset with this in it lies past every view (views hold at most 2^29
// bytes: 2^20 columns of 128 ranks of 4 bytes), also with another one added.
constexpr uint32_t kFar = 0x40000000u;
constexpr int kTile = 16;  // rows per matrix tile

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
// y[t][n] = round(y_in[t][n] + sum_r scale_g s[t][r] b[g][n][r]), with s either
// computed by the same block (FUSED: eight waves share K for a tile of 16
// rows, meet in LDS, and then share N, so that a call is one launch) or added
// up from a shrink launch's shares of K (few rows with large adapters).
//
// For 16-bit adapters s enters the product as two 16-bit parts, hi = round(s)
// and lo = round(s - hi), laid side by side along the product's 32-value
// inner axis (against the same b values), which keeps 16 (f16: 22) bits of
// it: for rank 16 one instruction holds both. f16 rows are first scaled by a
// power of two to a maximum in [2^14, 2^15), so that neither part over- or
// underflows, and the sum back afterwards. Infinities do not survive that: lo x
// inf has a sign of its own, and 0 x inf (a lo of 0, a chunk of the product that
// is not used) is NaN. So a group of columns with a sum that is not finite is
// computed again from the fp32 sums, by products of 4 ranks (16x16x4).
struct ExpandArgs {
  const void* x;           // [T, K]
  const void* a;           // [G, R, K]
  const void* b;           // [G, N, R]
  const float* scale;      // nullable [G]
  const int32_t* adapter;  // [T]
  const void* yin;         // nullable [T, N], may be y
  void* y;                 // nullable [T, N]
  float* s;                // nullable [T, R], receives scale * s
  const float* part;       // not FUSED: [S, T, R]
  int T, K, N, R, G, S;
};

// The backward's form (TURNED) has up to three rows of blocks, which run side by
// side: the list of every adapter's rows (offsets not null), u and dx, and s. u
// and dx meet b and a where the forward has a and b, along their other axis. A
// lane turns neighbouring rows of them in registers on the way to LDS, whose
// layout stays: 4096 rows of 8 adapters 2048 -> 2048 take 16.9 us, as from turned
// copies, which took a launch of 5.1 us more and all adapters' bytes twice. Also
// for few rows of large adapters, which the forward splits (one row 4096 -> 4096
// at rank 128 the whole backward 52 us, split 49; at rank 64 with 64 adapters 45
// and 87).
struct ExpandJobs {
  ExpandArgs job[2];
  uint32_t* offsets;  // nullable [G + 1]
  uint32_t* perm;     // [T]
  int turned;         // jobs from the first one whose a and b lie turned
  int team;    // blocks of a tile
  int shares;  // of an adapter's columns, at most
  int run;     // tiles of an XCD, 0 for few
};

constexpr int kFusedWaves = 8;

// scale * s of tile row c (c8 chunks of 16 bytes' worth of values in LDS, four
// floats i at row[i ^ turn]) as the matrix operand of expand (see there), a step at
// a time; back: what the products have to be multiplied by.
template <typename XT, int RT>
__device__ __forceinline__ void expand_operand(const float4* row, int turn, int c8, int q, bool mine,
                                               u32x4_t (&sv)[RT], float& back) {
  constexpr bool F32 = sizeof(XT) == 4;
  constexpr int V = 16 / sizeof(XT);
  auto chunk = [&](int i, float (&v)[V]) {
    const int ci = 4 * i + q, cc = F32 || ci < c8 ? ci : ci - c8;
    const bool in = mine && cc < c8;
#pragma unroll
    for (int j = 0; j < V; j += 4) {
      const float4 f = row[((min(cc, c8 - 1) * V + j) >> 2) ^ turn];
      v[j] = in ? f.x : 0.f; v[j + 1] = in ? f.y : 0.f;
      v[j + 2] = in ? f.z : 0.f; v[j + 3] = in ? f.w : 0.f;
    }
  };
  back = 1.f;
  float fw = 1.f;
  if constexpr (__is_same(XT, f16_t)) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < RT; i++) {
      float v[V];
      chunk(i, v);
#pragma unroll
      for (int j = 0; j < V; j++) m = fmaxf(m, fabsf(v[j]));
    }
    m = fmaxf(m, __shfl_xor(m, 16, kWave));
    m = fmaxf(m, __shfl_xor(m, 32, kWave));
    const int eb = (int)((__float_as_uint(m) >> 23) & 255u);
    const int sh = eb == 255 ? 0 : min(14 - (eb - 127), 100);
    back = __builtin_ldexpf(1.f, -sh);
    fw = __builtin_ldexpf(1.f, sh);
  }
#pragma unroll
  for (int i = 0; i < RT; i++) {
    float v[V];
    chunk(i, v);
    if constexpr (F32) {
#pragma unroll
      for (int j = 0; j < 4; j++) sv[i][j] = __float_as_uint(v[j]);
    } else {
      const bool lo = 4 * i + q >= c8;
      uint32_t h[8];
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const float f = v[j] * fw, hi = round_to<XT>(f);
        const float rest = __builtin_isfinite(hi) ? f - hi : 0.f;
        h[j] = (uint32_t)__builtin_bit_cast(uint16_t, from_f<XT>(lo ? rest : hi));
      }
#pragma unroll
      for (int j = 0; j < 4; j++) sv[i][j] = h[2 * j] | (h[2 * j + 1] << 16);
    }
    if (RT == 8) __builtin_amdgcn_sched_barrier(0);  // registers: one step's values at a time
  }
}

template <typename F, int... I>
__device__ __forceinline__ void static_for(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I + 1>{}), ...);
}
template <typename F> __device__ __forceinline__ void static_for_15(F&& f) {
  static_for(f, std::make_integer_sequence<int, 15>{});
}

// Orders this wave's LDS accesses of different lanes; loads from global memory
// stay in flight across it.
__device__ __forceinline__ void wave_lds_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Value e of each of a lane's N pieces, one after the other.
template <typename XT, int N>
__device__ __forceinline__ void turn(const u32x4_t (&v)[N], int e, uint32_t (&w)[N * sizeof(XT) / 4]) {
#pragma unroll
  for (int i = 0; i < N * (int)sizeof(XT) / 4; i++) {
    if constexpr (sizeof(XT) == 4) w[i] = v[i][e];
    else w[i] = __builtin_amdgcn_perm(v[2 * i + 1][e >> 1], v[2 * i][e >> 1], e & 1 ? 0x07060302u : 0x05040100u);
  }
}

// The rows of adapter g by a block of W waves: offsets[g] (and the last one),
// and perm from there in ascending order, the layout of moe_dispatch_plan. A
// thread counts ids below and equal to g in a run of 16-byte groups of rows; its
// rows follow those of the threads before it. meet: 2 W values in LDS, free
// for the next call.
template <int W>
__device__ __forceinline__ void list_rows(const int32_t* __restrict__ adapter, int T, int G, int g,
                                          uint32_t* __restrict__ offsets, uint32_t* __restrict__ perm,
                                          uint32_t* meet) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int groups = (T + 3) / 4, per = (groups + 64 * W - 1) / (64 * W);
  const int q0 = min(groups, tid * per), q1 = min(groups, q0 + per);
  const bool vec = (reinterpret_cast<uintptr_t>(adapter) & 15) == 0;
  auto ids = [&](int q, int32_t (&v)[4]) {
    if (vec && q * 4 + 4 <= T) {
      const int4 w = *reinterpret_cast<const int4*>(adapter + q * 4);
      v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++) v[j] = q * 4 + j < T ? adapter[q * 4 + j] : -1;
    }
  };
  uint32_t lt = 0, eq = 0;
  for (int q = q0; q < q1; q++) {
    int32_t v[4];
    ids(q, v);
#pragma unroll
    for (int j = 0; j < 4; j++) {
      lt += v[j] >= 0 && v[j] < g;
      eq += v[j] == g;
    }
  }
  const uint32_t clt = wave_scan_u32(lt), ceq = wave_scan_u32(eq);
  if (lane == 63) {
    meet[wave] = clt;
    meet[W + wave] = ceq;
  }
  __syncthreads();
  uint32_t base = 0, before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < W; w++) {
    base += meet[w];
    all += meet[W + w];
    before += w < wave ? meet[W + w] : 0u;
  }
  __syncthreads();
  if (tid == 0) {
    offsets[g] = base;
    if (g == G - 1) offsets[G] = base + all;
  }
  if (eq == 0) return;
  uint32_t at = base + before + ceq - eq;
  for (int q = q0; q < q1; q++) {
    int32_t v[4];
    ids(q, v);
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (v[j] == g) perm[at++] = (uint32_t)(q * 4 + j);
  }
}

// Waves per SIMD: two blocks on a CU where LDS has room for them, so that a few
// blocks more than CUs (requests that end inside a tile) cost no second round.
constexpr int expand_waves(int rt) { return rt <= 4 ? 4 : 2; }

template <typename XT, int RT, bool FUSED, bool TURNED>
__global__ __launch_bounds__(64 * kFusedWaves, expand_waves(RT)) void lora_expand_kernel(ExpandJobs jobs) {
  constexpr bool F32 = sizeof(XT) == 4;
  constexpr uint32_t ES = sizeof(XT);
  constexpr int V = 16 / sizeof(XT), LD = RT * 16 + 4, W = kFusedWaves;
  constexpr int UNIT = 8 * V;                      // a unit of K: 128 bytes of a row
  // neighbouring columns of a lane: as many as leave LDS for two blocks up to
  // rank 64 (fp32, 7454 rows 264 -> 96 backward at rank 40: 26.2 us with two columns,
  // 31.8 with four; 4096 rows 2048 -> 2048 at rank 64 54.8 and 64.6)
  constexpr int J = F32 && RT >= 4 ? 2 : 4;
  constexpr int NC = 16 * J;                       // columns of a group
  constexpr int C8 = RT * 16 / V;                  // 16-byte chunks of the widest adapter row
  constexpr int BL = NC * C8 / 64;                 // loads of a column group's b rows
  constexpr int AREA = (1 + RT) * 128 > NC * (C8 | 1) ? (1 + RT) * 128 : NC * (C8 | 1);  // 16-byte slots
  static_assert(AREA * 4 >= 2 * kTile * LD, "the sums of a wave and of the block fit an area");
  constexpr int KEPT = AREA - 64;
  static_assert(F32 || (KEPT >= NC * (C8 | 1) && 64 * 4 >= 2 * RT * 16 && kTile == 2 * W), "room for the kept sums");
  // a wave's area holds in turn its units, its sums and its column groups. The
  // block's sums: fp32 in the first one's second half, until its column groups
  // overwrite them; 16-bit types behind the column groups, where they stay, rows 2 w
  // and 2 w + 1 in area w, in an order that puts a chunk's 16 rows on different banks
  __shared__ u32x4_t area[W][AREA];
  auto sums_of = [&](int t) {
    return F32 ? reinterpret_cast<float*>(area[0]) + kTile * LD + t * LD
               : reinterpret_cast<float*>(area[t >> 1] + KEPT) + (t & 1) * RT * 16;
  };
  auto sums_turn = [](int t) { return F32 ? 0 : RT <= 2 ? (t >> 1) & (4 * RT - 1) : t; };
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // all arguments at once (opaque: else each is loaded where it is first used,
  // and waited for there)
  bool turned = false;  // the job's a is [G, K, R], its b [G, R, N]
  int job = 0;
  if constexpr (TURNED) {
    job = (int)blockIdx.y - (jobs.offsets != nullptr);
    if (job < 0) {
      for (int g = blockIdx.x; g < jobs.job[0].G; g += gridDim.x)
        list_rows<W>(jobs.job[0].adapter, jobs.job[0].T, jobs.job[0].G, g, jobs.offsets, jobs.perm,
                     reinterpret_cast<uint32_t*>(area[0]));
      return;
    }
    turned = job < jobs.turned;
  }
  ExpandArgs p = jobs.job[job];
  int team = jobs.team, most = jobs.shares, run = jobs.run;
  asm volatile("" : "+s"(p.x), "+s"(p.a), "+s"(p.b), "+s"(p.scale), "+s"(p.adapter), "+s"(p.yin), "+s"(p.y), "+s"(p.s));
  asm volatile("" : "+s"(p.T), "+s"(p.K), "+s"(p.N), "+s"(p.R), "+s"(p.G), "+s"(team), "+s"(most), "+s"(run));
  // Consecutive blocks go to the eight XCDs in turn. Many tiles: each XCD takes a
  // run of neighbours, whose rows share adapters in its L2, all first blocks of
  // a tile before the second ones. Few: the tiles' first blocks are spread, then
  // the second ones.
  int member, tile;  // one of jobs.team blocks of a tile
  if (run > 0) {
    const int i = (int)(blockIdx.x >> 3);
    member = i / run;
    tile = (int)(blockIdx.x & 7u) * run + i % run;
  } else {
    const uint32_t tiles = (uint32_t)(p.T + kTile - 1) / kTile;
    member = (int)(blockIdx.x / tiles);
    tile = (int)(blockIdx.x % tiles);
  }
  if (tile * (long)kTile >= p.T) return;
  const int t0 = tile * kTile, rows = min(kTile, p.T - t0);
  const int ad = tile_adapter(p.adapter, t0, rows, tid & 15, p.G);
  const int K = p.K, N = p.N, R = p.R, c8 = R / V;
  const rsrc_t xr = make_rsrc((const XT*)p.x + (size_t)t0 * K, (uint32_t)rows * (uint32_t)K * ES);
  const rsrc_t yr = make_rsrc((const XT*)p.yin + (p.yin ? (size_t)t0 * N : 0),
                              p.yin ? (uint32_t)rows * (uint32_t)N * ES : 0u);
  const rsrc_t wr = make_rsrc((XT*)p.y + (p.y ? (size_t)t0 * N : 0), p.y ? (uint32_t)rows * (uint32_t)N * ES : 0u);
  u32x4_t* const mem = area[wave];
  // The team's members take the tile's adapters in turn; where there are fewer
  // adapters than members, several share the columns of one (each repeating
  // its sums).
  uint32_t todo = (1u << rows) - 1u;  // rows with something to do
  if (p.y == nullptr || p.yin == p.y) todo &= (uint32_t)__ballot(ad >= 0);
  // the first row of each of their distinct adapters: rows whose id no row
  // before them has
  bool again = false;
  static_for_15([&](auto i) { again |= dpp_i32<0x110 + decltype(i)::value, 0xF>(-2, ad) == ad; });
  uint32_t heads = (uint32_t)__ballot(!again) & todo;
  const int D = __builtin_popcount(heads);
  int first = member, share = 0, shares = 1;
  if (D == 0) return;
  if (D < team) {
    first = member % D;
    share = member / D;
    shares = min(p.y ? most : 1, (team - first + D - 1) / D);
    if (share >= shares) return;
  }
  // a wave's units of K and groups of columns are neighbours, the waves' shares
  // apart: rows are often a multiple of the 4 KB that the memory channels
  // repeat after, so that all rows of a tile ask one channel for the same k
  const int units = (K + UNIT - 1) / UNIT, uper = (units + W - 1) / W;
  const int u0 = wave * uper, u1 = min(units, u0 + uper);
  const int cw = share * W + wave, cws = shares * W;
  const int groups = (N + NC - 1) / NC, gper = (groups + cws - 1) / cws;
  const int g0 = cw * gper, g1 = min(groups, g0 + gper);
  for (int d = 0; heads; d++) {
    const int lead = __builtin_ctz(heads);
    heads &= heads - 1u;
    if (d < first || (d - first) % team != 0) continue;
    const int g = __builtin_amdgcn_readlane(ad, lead);
    const uint32_t same = (uint32_t)__ballot(ad == g) & todo;
    // (opaque: else what follows from the lane alone, some hundred addresses,
    // is computed ahead of the loop and spilled)
    int lane = tid & 63;
    asm volatile("" : "+v"(lane));
    const int c = lane & 15, q = lane >> 4;
    if (g < 0) {  // rows without an adapter: y = y_in
      for (int n = (cw * 8 + (lane & 7)) * V; n < N; n += 8 * cws * V) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const int r = 8 * h + (lane >> 3);
          const uint32_t off = (same >> r) & 1u ? ((uint32_t)r * N + n) * ES : kFar;
          bstore128(wr, off, bload128(yr, off));
        }
      }
      continue;
    }
    const rsrc_t ar = make_rsrc((const XT*)p.a + (size_t)g * R * K, (uint32_t)R * (uint32_t)K * ES);
    const rsrc_t br = make_rsrc((const XT*)p.b + (size_t)g * N * R, (uint32_t)N * (uint32_t)R * ES);
    const float sc = p.scale ? p.scale[g] : 1.f;
    // ---- loads of b and y
    const uint32_t pieces = (uint32_t)NC * c8;  // a multiple of 64
    uint32_t yo[4];
#pragma unroll
    for (int i = 0; i < 4; i++)
      yo[i] = ((same >> (4 * q + i)) & 1u ? (uint32_t)(4 * q + i) * N * ES : kFar) + (uint32_t)(J * c) * ES;
    u32x4_t bv[BL];
    uint32_t yv[4][J * ES / 4], yn[4][J * ES / 4];
    auto load_y = [&](int grp, uint32_t (&yb)[4][J * ES / 4]) {
      const uint32_t no = grp < g1 && grp * NC + J * c < N ? (uint32_t)grp * NC * ES : kFar;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if constexpr (J * ES == 16) {
          const u32x4_t v = bload128(yr, yo[i] + no);
#pragma unroll
          for (int j = 0; j < 4; j++) yb[i][j] = v[j];
        } else {
          const u32x2_t v = bload64(yr, yo[i] + no);
          yb[i][0] = v[0];
          yb[i][1] = v[1];
        }
      }
    };
    // turned: a lane takes BL neighbouring ranks of V columns
    constexpr int PC = NC / V;
    auto load_b = [&](int grp) {
      if constexpr (TURNED) {
        int l = lane;
        asm volatile("" : "+v"(l));  // (opaque: as above)
        const int bj = l % PC, br0 = l / PC * BL;
        const uint32_t go = grp < g1 ? (uint32_t)grp * NC * ES + (uint32_t)br0 * N * ES + 16u * bj : kFar;
#pragma unroll
        for (int i = 0; i < BL; i++) bv[i] = bload128(br, br0 + i < R ? go + (uint32_t)i * N * ES : kFar);
        return;
      }
      const uint32_t go = grp < g1 ? (uint32_t)grp * NC * R * ES + 16u * lane : kFar;
#pragma unroll
      for (int i = 0; i < BL; i++) bv[i] = bload128(br, 64u * i < pieces ? go + 1024u * i : kFar);
    };
    // ---- shrink. Eight lanes load a row's 128 bytes (lane l: piece l % 8 of
    // row l / 8): the load unit takes 64 neighbouring bytes a clock but only 16
    // when neighbouring lanes are in different rows, as the matrix operands
    // have them. So the pieces change lanes through LDS, piece j of row r in slot
    // 8 r + (j ^ r % 8).
    f32x4_t acc[RT] = {};
    if constexpr (FUSED) {
      const int pr = lane >> 3, pj = lane & 7;
      // turned: rows of a are k's of R ranks. A lane takes NR neighbouring k's of V
      // ranks and turns them in registers into the same order.
      constexpr int NR = 2 * RT, NP = 64 * NR / UNIT;
      const int tc = lane % NP, tn = lane / NP * NR;
      const uint32_t astep = TURNED && turned ? (uint32_t)UNIT * R * ES : 128u;
      const uint32_t arow = TURNED && turned ? (uint32_t)R * ES : 8u * K * ES;  // between a lane's rows of a
      const uint32_t ao = !(TURNED && turned) ? (uint32_t)pr * K * ES + 16u * pj
                          : tc < c8           ? (uint32_t)tn * R * ES + 16u * tc
                                              : kFar;
      uint32_t xo[2];
#pragma unroll
      for (int h = 0; h < 2; h++)
        xo[h] = ((same >> (h * 8 + pr)) & 1u ? (uint32_t)(h * 8 + pr) * K * ES : kFar) + 16u * pj;
      u32x4_t xv[2], av[2 * RT];
      auto load = [&](int u) {
        const uint32_t ko = u < u1 && u * UNIT + pj * V < K ? (uint32_t)u * 128u : kFar;
        const uint32_t ka = !(TURNED && turned) ? ko : u < u1 ? (uint32_t)u * astep : kFar;
#pragma unroll
        for (int h = 0; h < 2; h++) xv[h] = bload128(xr, xo[h] + ko);
#pragma unroll
        for (int i = 0; i < 2 * RT; i++)
          av[i] = bload128(ar, ao + ka + ((TURNED && turned) || i * 8 < R ? i * arow : kFar));
      };
      u32x4_t* const put = mem + pr * 8 + (pj ^ pr);
      const u32x4_t* const get = mem + c * 8;
      load(u0);
      for (int u = u0; u < u1; u++) {
#pragma unroll
        for (int h = 0; h < 2; h++) put[h * 64] = xv[h];
        if (TURNED && turned) {
          char* const to = reinterpret_cast<char*>(mem + 128 + tc * V * 8) + tn * ES % 16;
#pragma unroll
          for (int e = 0; e < V; e++) {
            uint32_t w[NR * ES / 4];
            turn<XT, NR>(av, e, w);
            const int rx = ((tc * V + e) ^ (tc * V >> 3)) & 7;
            if constexpr (NR * ES >= 16) {
#pragma unroll
              for (int z = 0; z < (int)(NR * ES / 16); z++)
                *reinterpret_cast<u32x4_t*>(to + 16 * (8 * e + ((tn / V + z) ^ rx))) =
                    u32x4_t{w[4 * z], w[4 * z + 1], w[4 * z + 2], w[4 * z + 3]};
            } else {
#pragma unroll
              for (int z = 0; z < (int)(NR * ES / 4); z++)
                *reinterpret_cast<uint32_t*>(to + 16 * (8 * e + ((tn / V) ^ rx)) + 4 * z) = w[z];
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < 2 * RT; i++) mem[128 + i * 64 + pr * 8 + (pj ^ pr ^ (TURNED ? i & 7 : 0))] = av[i];
        }
        wave_lds_sync();
        load(u + 1);
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const int at = (4 * h + q) ^ (c & 7);
          const u32x4_t xf = get[at];
#pragma unroll
          for (int i = 0; i < RT; i++) acc[i] = mma<XT>(get[128 + i * 128 + (TURNED ? at ^ (c >> 3) ^ (2 * i & 7) : at)], xf, acc[i]);
          if (RT == 8) __builtin_amdgcn_sched_barrier(0);
        }
        wave_lds_sync();
      }
    }
    uint32_t slot[BL];
    if constexpr (!TURNED) {
      int n = lane / c8, cc = lane % c8;
      const int dn = 64 / c8, dc = 64 % c8;
#pragma unroll
      for (int i = 0; i < BL; i++) {  // piece 64 i + lane: chunk cc of column n
        slot[i] = (uint32_t)((n % J) * 16 + n / J) * (c8 | 1) + cc;
        n += dn;
        cc += dc;
        if (cc >= c8) {
          cc -= c8;
          n++;
        }
      }
    }
    // ---- the waves' sums meet
    float* const red = reinterpret_cast<float*>(mem);
    if constexpr (FUSED) {
#pragma unroll
      for (int i = 0; i < RT; i++) *reinterpret_cast<f32x4_t*>(red + c * LD + i * 16 + 4 * q) = acc[i];
      lds_barrier();
    }
    for (int e = tid; e < RT * 256; e += 64 * W) {
      const int t = e / (RT * 16), r = e % (RT * 16), at = t * LD + r;
      float v = 0.f;
      if constexpr (FUSED) {
#pragma unroll
        for (int w = 0; w < W; w += 2)
          v += reinterpret_cast<float*>(area[w])[at] + reinterpret_cast<float*>(area[w + 1])[at];
      } else if (r < R && ((same >> t) & 1u)) {
        const float* ps = p.part + (size_t)(t0 + t) * R + r;
#pragma unroll 8
        for (int z = 0; z < p.S; z++) v += ps[(size_t)z * p.T * R];
      }
      v *= sc;
      sums_of(t)[r ^ (sums_turn(t) << 2)] = v;
      if (p.s && share == 0 && r < R && ((same >> t) & 1u)) p.s[(size_t)(t0 + t) * R + r] = v;
    }
    lds_barrier();
    if (p.y) {
      // ---- expand: rows of s against the column group's b rows; lane (c, q)
      // gets columns J c .. of rows 4 q .., so that 16 lanes read and write 128
      // neighbouring bytes of y
      u32x4_t sv[RT];
      float back, bk[4] = {1.f, 1.f, 1.f, 1.f};
      expand_operand<XT, RT>(reinterpret_cast<const float4*>(sums_of(c)), sums_turn(c), c8, q, (same >> c) & 1u, sv, back);
      if constexpr (F32) lds_barrier();  // the first wave's column groups overwrite the sums
      if constexpr (__is_same(XT, f16_t)) {
#pragma unroll
        for (int i = 0; i < 4; i++) bk[i] = __shfl(back, 4 * q + i, kWave);
      }
      __builtin_amdgcn_sched_barrier(0);
      load_b(g0);
      load_y(g0, yn);
      uint32_t at[RT];
#pragma unroll
      for (int i = 0; i < RT; i++) {
        const int ci = 4 * i + q, cc = F32 || ci < c8 ? ci : ci - c8;
        at[i] = (uint32_t)c * (c8 | 1) + min(cc, F32 ? c8 : c8 - 1);
      }
      // fp32: chunks past the rank meet the columns' spare slots (c8 is even), which
      // hold zeros, since 0 x inf is not 0
      if (F32 && c8 < C8 && lane < NC) mem[lane * (c8 | 1) + c8] = u32x4_t{0u, 0u, 0u, 0u};
      for (int grp = g0; grp < g1; grp++) {
        if constexpr (TURNED) {
          int l = lane;
          asm volatile("" : "+v"(l));
          const int bj = l % PC, br0 = l / PC * BL, bto = bj * (V / J) * (c8 | 1) * 16 + br0 * ES;
#pragma unroll
          for (int e = 0; e < V; e++) {
            uint32_t w[BL * ES / 4];
            turn<XT, BL>(bv, e, w);
            char* const to = reinterpret_cast<char*>(mem + ((e % J) * 16 + e / J) * (c8 | 1)) + bto;
            if constexpr (BL * ES >= 16) {
#pragma unroll
              for (int z = 0; z < (int)(BL * ES / 16); z++)
                if (br0 + z * V < R)
                  *reinterpret_cast<u32x4_t*>(to + 16 * z) = u32x4_t{w[4 * z], w[4 * z + 1], w[4 * z + 2], w[4 * z + 3]};
            } else if (br0 < R) {
#pragma unroll
              for (int z = 0; z < (int)(BL * ES / 4); z++) *reinterpret_cast<uint32_t*>(to + 4 * z) = w[z];
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < BL; i++)
            if (64u * i < pieces) mem[slot[i]] = bv[i];
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
          for (int j = 0; j < (int)(J * ES / 4); j++) yv[i][j] = yn[i][j];
        wave_lds_sync();
        load_b(grp + 1);
        load_y(grp + 1, yn);
        f32x4_t o[J] = {};
        if (!F32 && RT > 1 && c8 == C8) {
          // chunks fill whole products: hi and lo meet the same b operand
#pragma unroll
          for (int i = 0; i < RT / 2; i++) {
#pragma unroll
            for (int j = 0; j < J; j++) {
              const u32x4_t bf = mem[(uint32_t)j * 16 * (c8 | 1) + at[i]];
              o[j] = mma<XT>(sv[i], bf, o[j]);
              o[j] = mma<XT>(sv[i + RT / 2], bf, o[j]);
            }
            if (BL >= 16) __builtin_amdgcn_sched_barrier(0);  // registers: no operands further ahead
          }
        } else {
#pragma unroll
          for (int i = 0; i < RT; i++) {
#pragma unroll
            for (int j = 0; j < J; j++) o[j] = mma<XT>(sv[i], mem[(uint32_t)j * 16 * (c8 | 1) + at[i]], o[j]);
            if (BL >= 16) __builtin_amdgcn_sched_barrier(0);
          }
        }
        bool redo = false;  // the same in all lanes
        if constexpr (!F32) {
          float top = 0.f;
#pragma unroll
          for (int j = 0; j < J; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) top = __builtin_elementwise_maximum(top, __builtin_fabsf(o[j][i]));  // NaN stays
          redo = __builtin_expect(__any(!(top < __builtin_huge_valf())), 0);
          if (redo) {
            int l = tid & 63;
            asm volatile("" : "+v"(l));  // (opaque: as above)
            const int row = l & 15, k = l >> 4, turn = sums_turn(row) << 2;
            const float* const sum = sums_of(row) + k;
            const XT* const bcol = reinterpret_cast<const XT*>(mem + row * (c8 | 1)) + k;
#pragma unroll
            for (int j = 0; j < J; j++) o[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
            for (int r = 0; r < R; r += 4) {
#pragma unroll
              for (int j = 0; j < J; j++)
                o[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(sum[r ^ turn], to_f<XT>(bcol[j * 16 * (c8 | 1) * V + r]), o[j], 0, 0, 0);
            }
          }
        }
        wave_lds_sync();
        const uint32_t no = grp < g1 && grp * NC + J * c < N ? (uint32_t)grp * NC * ES : kFar;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          uint32_t w[J * ES / 4];
          if constexpr (F32) {
#pragma unroll
            for (int j = 0; j < J; j++) w[j] = __float_as_uint(__uint_as_float(yv[i][j]) + o[j][i]);
          } else {
#pragma unroll
            for (int j = 0; j < J / 2; j++) {
              const uint32_t y2 = yv[i][j];
              const float m = redo ? 1.f : bk[i];
              const float lo = __builtin_fmaf(o[2 * j][i], m, to_f<XT>(__builtin_bit_cast(XT, (uint16_t)(y2 & 0xFFFFu))));
              const float hi = __builtin_fmaf(o[2 * j + 1][i], m, to_f<XT>(__builtin_bit_cast(XT, (uint16_t)(y2 >> 16))));
              w[j] = (uint32_t)__builtin_bit_cast(uint16_t, from_f<XT>(lo)) |
                     ((uint32_t)__builtin_bit_cast(uint16_t, from_f<XT>(hi)) << 16);
            }
          }
          if constexpr (J * ES == 16) bstore128(wr, yo[i] + no, u32x4_t{w[0], w[1], w[2], w[3]});
          else __builtin_amdgcn_raw_buffer_store_b64(u32x2_t{w[0], w[1]}, wr, yo[i] + no, 0, 0);
        }
      }
    }
    lds_barrier();  // before the areas' and the sums' next adapter
  }
}

// ----------------------------------------------------- adapter gradients --
// dA_g[r][k] = sum_t u[t][r] x[t][k] and dB_g[n][r] = sum_t s[t][r] dy[t][n]
// over the rows of adapter g, which the plan lists (perm, offsets); u and s
// with their scale. A lane reads 8 neighbouring columns of a row. fp32 rows, and
// one rank tile of any: each column is an operand of an fp32 product of 4 rows
// (16x16x4), as it lies. More rank tiles of 16-bit rows: a lane reads 8 rows of
// its columns and turns them in registers into the 8 columns' operands of one
// product of 32 rows (16x16x32, eight times the rate), which u and s enter as
// two 16-bit parts as in expand; a wave with a sum that is not finite adds its rows
// again in fp32 products of 4, as there. 4096 rows of 8 adapters 2048 -> 2048: rank 16
// 13.3 us with products of 4 rows, 15.0 with those of 32 (whose steps the
// adapters' chunks fill less); rank 64 42.8 and 27.6.
//
// A block takes 128 columns (or several times that, see outer_span), up to two
// (fp32: four) rank tiles and a chunk of one adapter's rows (an adapter of n rows
// has ceil(n / chunk) equal ones, numbered through over the adapters, so that the
// work is even however the rows spread). Its eight waves share the chunk and
// meet in LDS; where it has fewer rows than their steps they share columns too.
// The gradient of an adapter with one chunk is stored at once, the chunks of the
// others as fp32, which lora_sum_kernel adds. Steps are loaded one
// ahead, the list of rows two ahead. SPAN: the form for several column blocks,
// whose loop takes the plain one's 11.8 us to 13.0.
struct OuterSide {
  const void* wide;    // [T, cols]: x or dy
  const float* small;  // [T, R]: u or s
  void* out;           // [G, R, cols] (rank_major: dA) or [G, cols, R] (dB)
  float* part;         // [chunks of adapters with several, ...] fp32
  int cols;
  int rank_major;
};
struct OuterArgs {
  OuterSide side[2];
  const uint32_t* perm;
  const uint32_t* offsets;
  int R, G, sides;
  uint32_t chunk;  // rows of a chunk, at most
  int span;        // column blocks of a block: 1, 2, 4 or 8
};
constexpr int kOuterWaves = 8, kOuterCols = 128;

// The adapter g whose chunks include number y (or, with of >= 0, adapter
// `of`), its rows [o0, o1) in the plan, its first chunk and how many it has, and
// the place of that first one among the chunks of adapters with several: only those
// have partial gradients. Uniform over the wave; g = G where y is past the last chunk.
struct Chunks {
  int g;
  uint32_t o0, o1, first, n, part;
};
__device__ __forceinline__ Chunks find_chunks(const uint32_t* __restrict__ offsets, int G,
                                              uint32_t chunk, uint32_t y, int of) {
  const int lane = threadIdx.x & 63;
  Chunks r{G, 0, 0, 0, 0, 0};
  uint32_t before = 0, alone = 0;  // chunks of the adapters before, and those that are their adapter's only one
  for (int i = 0; i < G; i += 64) {
    const bool in = i + lane < G;
    const uint32_t a = in ? offsets[i + lane] : 0u, b = in ? offsets[i + lane + 1] : 0u;
    const uint32_t n = (b - a + chunk - 1) / chunk, last = wave_scan_u32(n) + before;
    const int k = of >= 0 ? of - i : __popcll(__ballot(in && last <= y));
    const uint64_t one = __ballot(n == 1);
    if (k < min(64, G - i)) {
      r.g = i + k;
      r.o0 = (uint32_t)__builtin_amdgcn_readlane((int)a, k);
      r.o1 = (uint32_t)__builtin_amdgcn_readlane((int)b, k);
      r.n = (uint32_t)__builtin_amdgcn_readlane((int)n, k);
      r.first = (uint32_t)__builtin_amdgcn_readlane((int)last, k) - r.n;
      r.part = r.first - alone - (uint32_t)__popcll(one & ((1ull << k) - 1ull));
      break;
    }
    alone += (uint32_t)__popcll(one);
    before = (uint32_t)__builtin_amdgcn_readlane((int)last, 63);
  }
  return r;
}

// One adapter's part of the gradient: D[r = 16 k + 4 q + h][column 8 c + j].
template <typename OT, int RB>
__device__ __forceinline__ void outer_store(const f32x4_t (&acc)[RB][8], OT* out, bool rank_major,
                                            int R, int cols, int r0, int cb, int c, int q) {
  const int col = cb + 8 * c;
  if (col >= cols) return;
#pragma unroll
  for (int k = 0; k < RB; k++) {
    const int r = r0 + k * 16 + 4 * q;
    if (r >= R) continue;  // R is a multiple of 8: the four ranks go together
    if (rank_major) {
#pragma unroll
      for (int h = 0; h < 4; h++) {
        float o[8];
#pragma unroll
        for (int j = 0; j < 8; j++) o[j] = acc[k][j][h];
        Vec8<OT>::store(out + (size_t)(r + h) * cols + col, o);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) {
        OT* at = out + (size_t)(col + j) * R + r;
        if constexpr (sizeof(OT) == 4) {
          *reinterpret_cast<f32x4_t*>(at) = acc[k][j];
        } else {
          uint32_t w[2];
#pragma unroll
          for (int h = 0; h < 2; h++)
            w[h] = (uint32_t)__builtin_bit_cast(uint16_t, from_f<OT>(acc[k][j][2 * h])) |
                   ((uint32_t)__builtin_bit_cast(uint16_t, from_f<OT>(acc[k][j][2 * h + 1])) << 16);
          *reinterpret_cast<uint2*>(at) = make_uint2(w[0], w[1]);
        }
      }
    }
  }
}

template <typename XT, int RB, bool SPAN>
__global__ __launch_bounds__(64 * kOuterWaves) void lora_outer_kernel(OuterArgs p) {
  constexpr bool FOUR = sizeof(XT) == 4 || RB == 1;  // products of four rows
  constexpr int XW = sizeof(XT) / 2;                 // 16-byte loads of 8 columns
  constexpr int U = FOUR ? 2 : 8;                    // rows of a lane and step, 4 U of the wave
  __shared__ f32x4_t red[kOuterWaves / 2][RB * 8 * 64];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool second = p.sides == 2 && (blockIdx.z & 1u);
  const OuterSide sd = second ? p.side[1] : p.side[0];
  const int r0 = (int)(p.sides == 2 ? blockIdx.z >> 1 : blockIdx.z) * (RB * 16);
  const int R = p.R, cols = sd.cols;
  const int span = SPAN ? p.span : 1;
  if ((int)blockIdx.x * span * kOuterCols >= cols) return;
  const Chunks ck = find_chunks(p.offsets, p.G, p.chunk, blockIdx.y, -1);
  if (ck.g >= p.G) return;
  const uint32_t rows = (ck.o1 - ck.o0 + ck.n - 1) / ck.n;  // of an equal chunk
  const uint32_t s0 = min(ck.o1, ck.o0 + (blockIdx.y - ck.first) * rows), s1 = min(ck.o1, s0 + rows);
  const int few = rows <= 4 * U ? 8 : rows <= 8 * U ? 4 : rows <= 16 * U ? 2 : 1;
  const int across = min(few, span);  // waves across columns, the others across rows
  const size_t per = (size_t)R * cols;
  for (int it = 0; it < span; it += across) {
    int lane = tid & 63;
    if constexpr (SPAN) asm volatile("" : "+v"(lane));  // (opaque: else its addresses are kept over the loop)
    const int c = lane & 15, q = lane >> 4;
    const float* const small = sd.small + r0 + c;
    const int cb = ((int)blockIdx.x * span + it + (wave & (across - 1))) * kOuterCols, col = cb + 8 * c;
    const XT* const wide = (const XT*)sd.wide + col;
    const uint32_t parts = kOuterWaves / across, len = ((s1 - s0 + parts - 1) / parts + 3u) & ~3u;
    const uint32_t b0 = min(s1, s0 + (uint32_t)(wave / across) * len), b1 = min(s1, b0 + len);
    f32x4_t acc[RB][8] = {};
    if (b0 < b1) {
      // row i of a lane in a step: 4 i + q where every product takes four rows,
      // 8 q + i where one takes all 32
      auto row_of = [&](int i) { return FOUR ? 4 * i + q : 8 * q + i; };
      u32x4_t wv[U][XW];
      float sv[U][RB];
      auto rows_at = [&](uint32_t at) { return p.perm[min(at + (lane & 31), b1 - 1)]; };
      auto load = [&](uint32_t at, uint32_t pv) {
#pragma unroll
        for (int i = 0; i < U; i++) {
          const uint32_t t = (uint32_t)__shfl((int)pv, row_of(i), kWave);
          const bool in = at + row_of(i) < b1;
#pragma unroll
          for (int h = 0; h < XW; h++) wv[i][h] = u32x4_t{0u, 0u, 0u, 0u};
          if (in && col < cols) {
#pragma unroll
            for (int h = 0; h < XW; h++)
              wv[i][h] = *reinterpret_cast<const u32x4_t*>(wide + (size_t)t * cols + h * 4);
          }
#pragma unroll
          for (int j = 0; j < RB; j++) {
            sv[i][j] = 0.f;
            if (in && r0 + j * 16 + c < R) sv[i][j] = small[(size_t)t * R + j * 16];
          }
        }
      };
      uint32_t pv = rows_at(b0), pn = rows_at(b0 + 4 * U);
      load(b0, pv);
      for (uint32_t at = b0; at < b1; at += 4 * U) {
        u32x4_t w0[U][XW];
#pragma unroll
        for (int i = 0; i < U; i++)
#pragma unroll
          for (int h = 0; h < XW; h++) w0[i][h] = wv[i][h];
        if constexpr (FOUR) {
          float s[U][RB];
#pragma unroll
          for (int i = 0; i < U; i++)
#pragma unroll
            for (int j = 0; j < RB; j++) s[i][j] = sv[i][j];
          pv = pn;
          pn = rows_at(at + 8 * U);
          load(at + 4 * U, pv);
#pragma unroll
          for (int i = 0; i < U; i++) {
            if (at + 4 * i >= b1) continue;
            float w[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
              if constexpr (XW == 2) w[j] = __uint_as_float(w0[i][j >> 2][j & 3]);
              else w[j] = to_f<XT>(__builtin_bit_cast(XT, (uint16_t)(w0[i][0][j >> 1] >> (16 * (j & 1)))));
            }
#pragma unroll
            for (int k = 0; k < RB; k++)
#pragma unroll
              for (int j = 0; j < 8; j++)
                acc[k][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(s[i][k], w[j], acc[k][j], 0, 0, 0);
          }
        } else {
          // s as two 16-bit parts; f16 scaled by a power of two so that the
          // step's largest value lies in [2^14, 2^15)
          u32x4_t hi[RB], lo[RB];
          float fw = 1.f, back = 1.f;
          if constexpr (__is_same(XT, f16_t)) {
            float m = 0.f;
#pragma unroll
            for (int i = 0; i < U; i++)
#pragma unroll
              for (int k = 0; k < RB; k++) m = fmaxf(m, fabsf(sv[i][k]));
            m = wave_max_f32(m);
            const int eb = (int)((__float_as_uint(m) >> 23) & 255u);
            const int sh = eb == 255 ? 0 : min(14 - (eb - 127), 100);
            fw = __builtin_ldexpf(1.f, sh);
            back = __builtin_ldexpf(1.f, -sh);
          }
#pragma unroll
          for (int k = 0; k < RB; k++) {
            uint32_t h[8], l[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
              const float f = sv[i][k] * fw, fh = round_to<XT>(f);
              h[i] = (uint32_t)__builtin_bit_cast(uint16_t, from_f<XT>(f));
              l[i] = (uint32_t)__builtin_bit_cast(uint16_t, from_f<XT>(__builtin_isfinite(fh) ? f - fh : 0.f));
            }
#pragma unroll
            for (int m = 0; m < 4; m++) {
              hi[k][m] = h[2 * m] | (h[2 * m + 1] << 16);
              lo[k][m] = l[2 * m] | (l[2 * m + 1] << 16);
            }
          }
          pv = pn;
          pn = rows_at(at + 8 * U);
          load(at + 4 * U, pv);
#pragma unroll
          for (int j = 0; j < 8; j++) {
            // column j of the lane's 8 rows
            u32x4_t x;
#pragma unroll
            for (int m = 0; m < 4; m++)
              x[m] = __builtin_amdgcn_perm(w0[2 * m + 1][0][j >> 1], w0[2 * m][0][j >> 1],
                                           j & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
            for (int k = 0; k < RB; k++) {
              if constexpr (__is_same(XT, f16_t)) {
                const f32x4_t o = mma<XT>(lo[k], x, mma<XT>(hi[k], x, f32x4_t{0.f, 0.f, 0.f, 0.f}));
#pragma unroll
                for (int h = 0; h < 4; h++) acc[k][j][h] = __builtin_fmaf(o[h], back, acc[k][j][h]);
              } else {
                acc[k][j] = mma<XT>(lo[k], x, mma<XT>(hi[k], x, acc[k][j]));
              }
            }
          }
        }
      }
      if constexpr (!FOUR) {
        float nan[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < RB; k++)
#pragma unroll
          for (int j = 0; j < 8; j++)
#pragma unroll
            for (int h = 0; h < 4; h++) nan[h] = __builtin_fmaf(acc[k][j][h], 0.f, nan[h]);
        const float any = (nan[0] + nan[1]) + (nan[2] + nan[3]);
        if (__builtin_expect(__any(any != any), 0)) {
#pragma unroll
          for (int k = 0; k < RB; k++)
#pragma unroll
            for (int j = 0; j < 8; j++) acc[k][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
          for (uint32_t at = b0; at < b1; at += 4) {
            const bool in = at + q < b1;
            const uint32_t t = p.perm[min(at + q, b1 - 1)];
            u32x4_t x{0u, 0u, 0u, 0u};
            if (in && col < cols) x = *reinterpret_cast<const u32x4_t*>(wide + (size_t)t * cols);
#pragma unroll
            for (int k = 0; k < RB; k++) {
              const float s = in && r0 + k * 16 + c < R ? small[(size_t)t * R + k * 16] : 0.f;
#pragma unroll
              for (int j = 0; j < 8; j++)
                acc[k][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                    s, to_f<XT>(__builtin_bit_cast(XT, (uint16_t)(x[j >> 1] >> (16 * (j & 1))))), acc[k][j], 0, 0, 0);
            }
          }
        }
      }
    }
    // the upper half of the waves hands its sums to the lower, down to one
#pragma unroll
    for (int half = kOuterWaves / 2; half >= 1; half >>= 1) {
      if (half < across) break;
      if (wave >= half && wave < 2 * half) {
#pragma unroll
        for (int k = 0; k < RB; k++)
#pragma unroll
          for (int j = 0; j < 8; j++) red[wave - half][(k * 8 + j) * 64 + lane] = acc[k][j];
      }
      lds_barrier();
      if (wave < half) {
#pragma unroll
        for (int k = 0; k < RB; k++)
#pragma unroll
          for (int j = 0; j < 8; j++) acc[k][j] += red[wave][(k * 8 + j) * 64 + lane];
      }
      lds_barrier();
    }
    if (wave < across) {
      if (ck.n == 1) outer_store<XT, RB>(acc, (XT*)sd.out + ck.g * per, sd.rank_major, R, cols, r0, cb, c, q);
      else outer_store<float, RB>(acc, sd.part + (ck.part + blockIdx.y - ck.first) * per, sd.rank_major, R, cols, r0, cb, c, q);
    }
  }
}

// Adds the chunks of the adapters that have several, and writes zeros for
// those without rows; the others are there already. A lane adds 8 neighbouring
// values. Up to eight chunks one wave adds them all in order; more are shared by
// the block's waves, a run of them each, whose sums meet in LDS in the waves' order
// (7454 rows of one adapter 264 -> 96 at rank 40, 117 chunks: 5.8 us, by one wave 14).
constexpr int kSumWaves = 4;
template <typename XT>
__global__ __launch_bounds__(64 * kSumWaves) void lora_sum_kernel(OuterArgs p) {
  __shared__ float meet[kSumWaves - 1][8][64];
  const OuterSide sd = p.side[blockIdx.z];
  const int g = blockIdx.y, lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Chunks ck = find_chunks(p.offsets, p.G, p.chunk, 0, g);
  if (ck.n == 1) return;
  const size_t per = (size_t)p.R * sd.cols;
  auto add = [&](size_t i, uint32_t c0, uint32_t c1, float (&a)[8]) {
#pragma unroll
    for (int j = 0; j < 8; j++) a[j] = 0.f;
    if (i >= per) return;
#pragma unroll 4
    for (uint32_t c = c0; c < c1; c++) {
      float b[8];
      Vec8<float>::load(sd.part + (ck.part + c) * per + i, b);
#pragma unroll
      for (int j = 0; j < 8; j++) a[j] += b[j];
    }
  };
  float a[8];
  if (ck.n <= 8) {
    for (size_t i = ((size_t)blockIdx.x * 64 * kSumWaves + threadIdx.x) * 8; i < per;
         i += (size_t)gridDim.x * 512 * kSumWaves) {
      add(i, 0, ck.n, a);
      Vec8<XT>::store((XT*)sd.out + g * per + i, a);
    }
    return;
  }
  const uint32_t share = (ck.n + kSumWaves - 1) / kSumWaves;
  for (size_t b = (size_t)blockIdx.x * 512; b < per; b += (size_t)gridDim.x * 512) {
    const size_t i = b + lane * 8;
    add(i, min(ck.n, wave * share), min(ck.n, (wave + 1) * share), a);
    if (wave) {
#pragma unroll
      for (int j = 0; j < 8; j++) meet[wave - 1][j][lane] = a[j];
    }
    lds_barrier();
    if (wave == 0 && i < per) {
#pragma unroll
      for (int w = 0; w < kSumWaves - 1; w++)
#pragma unroll
        for (int j = 0; j < 8; j++) a[j] += meet[w][j][lane];
      Vec8<XT>::store((XT*)sd.out + g * per + i, a);
    }
    lds_barrier();
  }
}

// ------------------------------------------------------------------ host --
namespace {

int tiles_of(int T) { return (T + kTile - 1) / kTile; }

// Blocks of the shrink launch that share a tile's distinct adapters.
int leaders(int T, int G) {
  return std::max(1, std::min(std::min(std::min(kTile, T), G), 256 / tiles_of(T)));
}

template <typename XT>
hipError_t shrink_typed(const ShrinkArgs& a, int S, hipStream_t st) {
  const dim3 grid(tiles_of(a.T), leaders(a.T, a.G), S);
#define MOE_SH(RT) hipLaunchKernelGGL((lora_shrink_kernel<XT, RT>), grid, dim3(256), 0, st, a)
  if (a.R <= 16) MOE_SH(1);
  else if (a.R <= 32) MOE_SH(2);
  else if (a.R <= 64) MOE_SH(4);
  else MOE_SH(8);
#undef MOE_SH
  return hipGetLastError();
}

// The team of a tile: together about one block per CU, which share its adapters
// or the columns of one (64 rows of 64 adapters 2048 -> 2048 at rank 16 take
// 9.2 us with a block per adapter and 7.5 with four; 1000 rows 2880 -> 2880 at
// rank 24 12.5 with 252 blocks, 14.2 with 126 and 15.1 with 315), and two where the tiles
// fill the chip, for the tiles in which one request ends and the next begins:
// there a member without an adapter returns, since repeating the sums would cost
// more (4096 rows at rank 64: 30 us instead of 24).
constexpr int kTeamBlocks = 256, kRunTiles = 64;

// S > 0: the sums come from a shrink launch's S shares at a.part.
template <typename XT>
hipError_t expand_typed(const ExpandArgs& a, hipStream_t st, const ExpandJobs* backward = nullptr, int rows = 1) {
  ExpandJobs j{};
  if (backward) j = *backward;
  j.job[0] = a;
  const int tiles = tiles_of(a.T);
  // at least one group of 64 columns per wave; apart all of those
  const int most = a.y ? (a.N + 64 * kFusedWaves - 1) / (64 * kFusedWaves) : 1;
  j.shares = a.S ? most : std::max(1, std::min(most, kTeamBlocks / tiles));
  const int adapters = std::min(std::min(kTile, a.T), a.G + 1);
  j.team = std::min(adapters * j.shares, std::max(2, a.S ? kTile * j.shares : kTeamBlocks / tiles));
  j.run = tiles >= kRunTiles ? (tiles + 7) / 8 : 0;
  const uint32_t blocks = (uint32_t)(j.run ? 8 * j.run : tiles) * (uint32_t)j.team;
#define MOE_EX2(RT, FUSED, TURNED)                                                                   \
  hipLaunchKernelGGL((lora_expand_kernel<XT, RT, FUSED, TURNED>), dim3(blocks, rows), dim3(64 * kFusedWaves), 0, st, j)
#define MOE_EX(RT)                       \
  if (backward) MOE_EX2(RT, true, true); \
  else if (a.S) MOE_EX2(RT, false, false); \
  else MOE_EX2(RT, true, false);
  if (a.R <= 16) { MOE_EX(1) }
  else if (a.R <= 32) { MOE_EX(2) }
  else if (a.R <= 64) { MOE_EX(4) }
  else { MOE_EX(8) }
#undef MOE_EX
#undef MOE_EX2
  return hipGetLastError();
}

// Shares of the inner axis in a shrink launch: enough for two blocks per CU
// when there are few rows, at least one unit for each of a block's waves.
int lora_shares(int T, int G, int K, int dt) {
  const int unit = dt == DT_F32 ? 32 : 64;
  const int units = (K + unit - 1) / unit;
  const int blocks = tiles_of(T) * std::min(std::min(kTile, T), G);
  return std::max(1, std::min({512 / blocks, units / 4, 16}));
}

size_t adapter_bytes(const LoraDims& d) {
  return (size_t)d.R * (d.K + d.N) * (d.dt == DT_F32 ? 4 : 2);
}

// One launch, unless few blocks would each read a large adapter alone. Kernel
// times in one launch and in two: one row of 2048 -> 2048 at rank 16 5.7 us and 2.9 +
// 4.2, at rank 128 17.5 and 5.0 + 10.1 (of 4096 -> 4096 23.0 and 5.0 + 13.6); 64 rows of
// 64 adapters of 4096 -> 4096 at rank 64 19.4 and 9.9 + 13.2.
constexpr size_t kFusedBytes = 256u << 10;
constexpr int kSplitBlocks = 32;
bool lora_fused(const LoraDims& d) {
  return adapter_bytes(d) < kFusedBytes || tiles_of(d.T) * std::min(std::min(kTile, d.T), d.G) > kSplitBlocks;
}

// Bytes of a shrink launch's output over all its shares, at most, for up to T
// rows (lora_shares keeps shares at 16 and shares x blocks at 512), so that a
// workspace sized for many rows also serves a call of few.
size_t partial_bytes(const LoraDims& d) {
  if (adapter_bytes(d) < kFusedBytes) return 0;
  return std::min((size_t)d.T * 16, (size_t)512 * kTile / std::min(kTile, d.G)) * d.R * 4;
}

constexpr int kListRows = 16384;  // rows the backward's first launch lists; more take a plan of their own

size_t up256(size_t v) { return (v + 255) / 256 * 256; }

// Rank tiles of a block of the outer products, so that the wide rows are read
// once or twice: as many as leave the registers for a step ahead.
int outer_ranks(const LoraDims& d) { return d.R <= 16 ? 1 : d.R <= 32 || d.dt != DT_F32 ? 2 : 4; }

// Rows of a chunk in the outer products: about two blocks per CU with the
// adapters' last, smaller chunks, at least 64.
long outer_target(const LoraDims& d) {
  const int rt = outer_ranks(d) * 16;
  const long blocks = (long)((d.K + kOuterCols - 1) / kOuterCols + (d.N + kOuterCols - 1) / kOuterCols) *
                      ((d.R + rt - 1) / rt);
  const long n = 512 / blocks;
  return std::max({4L, n / 2, n - d.G / 2});
}
uint32_t outer_chunk(const LoraDims& d) {
  const long n = outer_target(d);
  return (uint32_t)std::max(64L, (d.T + n - 1) / n);
}
// Chunks of all adapters, at most.
long outer_chunks(const LoraDims& d) {
  return std::min<long>(d.T, std::min(outer_target(d), (long)(d.T + 63) / 64) + d.G);
}

// Chunks of the adapters that have several, at most, whose gradients are kept in
// parts: T rows hold at most T / chunk whole ones, and such an adapter at most one
// more. A chunk has T / target rows and 64 at least. (512 rows of 512 adapters 4096
// -> 4096 at rank 64: 8 parts, 17 MB; 516 chunks, 1.1 GB.)
long outer_parts(const LoraDims& d) {
  const long whole = d.T > 64 ? std::min<long>(outer_target(d), d.T / 64) : 0;
  return whole + std::min<long>(d.G, whole);
}

// Column blocks of a block: more than one where adapters have few rows on
// average, so that its waves have a step of rows each and the chip is not busy
// with blocks of one working wave (2048 rows of 64 adapters 4096 -> 4096 at rank 64
// 52 us instead of 195, 64 rows of 64 adapters 23 instead of 110; where one of
// the 64 has all 2048 rows 61 and 36), as long as 512 blocks remain (512 rows of one
// of 64 adapters 2048 -> 2048 at rank 16 13.3 us, with 256 blocks 22.6).
int outer_span(const LoraDims& d, long blocks) {
  const int step = d.dt == DT_F32 || d.R <= 16 ? 8 : 32, rows = (d.T + d.G - 1) / d.G;
  int span = rows <= step ? 8 : rows <= 2 * step ? 4 : rows <= 4 * step ? 2 : 1;
  while (span > 1 && blocks / span < 512) span /= 2;
  return span;
}

struct BackwardLayout {
  size_t s, u, counts, offsets, perm, inv, used, scratch, scratch_bytes, part, total;
};
BackwardLayout backward_layout(const LoraDims& d) {
  BackwardLayout l{};
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += up256(bytes);
    return o;
  };
  const size_t T = d.T, R = d.R, G = d.G, K = d.K, N = d.N;
  l.s = take(T * R * 4);
  l.u = take(T * R * 4);
  l.counts = take(G * 4);
  l.offsets = take((G + 1) * 4);
  l.perm = take(T * 4);
  l.inv = take(T * 4);
  l.used = take((G + 1) * 4);
  l.scratch_bytes = dispatch_scratch_bytes(d.T, 1, d.G);
  l.scratch = take(l.scratch_bytes);
  l.part = take((size_t)outer_parts(d) * R * (K + N) * 4);
  l.total = at;
  return l;
}

template <typename XT>
hipError_t backward_typed(const LoraDims& d, const LoraBackward& a, hipStream_t st) {
  const BackwardLayout l = backward_layout(d);
  char* ws = reinterpret_cast<char*>(a.ws);
  float* s = reinterpret_cast<float*>(ws + l.s);
  float* u = reinterpret_cast<float*>(ws + l.u);
  uint32_t* offsets = reinterpret_cast<uint32_t*>(ws + l.offsets);
  uint32_t* perm = reinterpret_cast<uint32_t*>(ws + l.perm);
  hipError_t e;
#define MOE_OKAY(expr) \
  if ((e = (expr)) != hipSuccess) return e
  const bool grads = a.da || a.db, need_u = a.dx || a.da, list = grads && d.T <= kListRows;
  if (grads && !list)
    MOE_OKAY(launch_dispatch_plan(reinterpret_cast<const uint32_t*>(a.adapter), d.T, 1, d.G,
                                  reinterpret_cast<uint32_t*>(ws + l.counts), offsets, perm,
                                  reinterpret_cast<uint32_t*>(ws + l.inv),
                                  reinterpret_cast<uint32_t*>(ws + l.used), ws + l.scratch,
                                  l.scratch_bytes, st));
  // u and dx: the forward's kernel with B^T and A^T in the place of A and B (u is
  // the same with and without dx); s: its first half
  const ExpandArgs eu{a.dy, a.b, a.a, a.scale, a.adapter, a.dx_in, a.dx, a.da ? u : nullptr, nullptr,
                      d.T, d.N, d.K, d.R, d.G, 0};
  const ExpandArgs es{a.x, a.a, a.b, a.scale, a.adapter, nullptr, nullptr, s, nullptr,
                      d.T, d.K, d.N, d.R, d.G, 0};
  ExpandJobs jobs{};
  jobs.job[1] = es;  // where both are asked for
  jobs.turned = need_u;
  if (list) {
    jobs.offsets = offsets;
    jobs.perm = perm;
  }
  MOE_OKAY(expand_typed<XT>(need_u ? eu : es, st, &jobs, (int)list + (int)need_u + (a.db != nullptr)));
  if (!grads) return hipSuccess;
  OuterArgs o{};
  o.perm = perm;
  o.offsets = offsets;
  o.R = d.R;
  o.G = d.G;
  o.chunk = outer_chunk(d);
  const long chunks = outer_chunks(d);
  float* const part = reinterpret_cast<float*>(ws + l.part);
  int cols = 0;
  if (a.da) {
    o.side[o.sides++] = {a.x, u, a.da, part, d.K, 1};
    cols = std::max(cols, d.K);
  }
  if (a.db) {
    o.side[o.sides++] = {a.dy, s, a.db, part + (size_t)outer_parts(d) * d.R * d.K, d.N, 0};
    cols = std::max(cols, d.N);
  }
  const int RB = outer_ranks(d);
  const int cblocks = (cols + kOuterCols - 1) / kOuterCols, ranks = o.sides * ((d.R + RB * 16 - 1) / (RB * 16));
  o.span = outer_span(d, cblocks * chunks * ranks);
  const dim3 grid((cblocks + o.span - 1) / o.span, (uint32_t)chunks, ranks);
#define MOE_OU(RB)                                                                             \
  if (o.span > 1) hipLaunchKernelGGL((lora_outer_kernel<XT, RB, true>), grid, dim3(64 * kOuterWaves), 0, st, o); \
  else hipLaunchKernelGGL((lora_outer_kernel<XT, RB, false>), grid, dim3(64 * kOuterWaves), 0, st, o);
  if (RB == 1) { MOE_OU(1) }
  else if (RB == 2) { MOE_OU(2) }
  else if constexpr (sizeof(XT) == 4) { MOE_OU(4) }
#undef MOE_OU
  MOE_OKAY(hipGetLastError());
  const size_t per = (size_t)d.R * cols;
  hipLaunchKernelGGL((lora_sum_kernel<XT>), dim3((uint32_t)std::min<size_t>((per + 511) / 512, 512), d.G, o.sides),
                     dim3(64 * kSumWaves), 0, st, o);
  MOE_OKAY(hipGetLastError());
#undef MOE_OKAY
  return hipSuccess;
}

}  // namespace

size_t lora_ws_bytes(const LoraDims& d) {
  return up256(partial_bytes(d));
}
size_t lora_backward_ws_bytes(const LoraDims& d) { return backward_layout(d).total; }

hipError_t launch_lora(const LoraDims& d, const void* x, const void* a, const void* b,
                       const float* scale, const int32_t* adapter, const void* yin, void* y,
                       void* ws, hipStream_t st) {
  const int S = lora_fused(d) ? 0 : lora_shares(d.T, d.G, d.K, d.dt);
  float* s = reinterpret_cast<float*>(ws);
  const ShrinkArgs sh{x, a, adapter, s, d.T, d.K, d.R, d.G};
  const ExpandArgs ex{x, a, b, scale, adapter, yin, y, nullptr, s, d.T, d.K, d.N, d.R, d.G, S};
#define MOE_LO(XT)                                          \
  {                                                         \
    if (S) {                                                \
      const hipError_t e = shrink_typed<XT>(sh, S, st);     \
      if (e != hipSuccess) return e;                        \
    }                                                       \
    return expand_typed<XT>(ex, st);                        \
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
