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
#include <utility>

#include "gemm_units.hpp"

#ifndef MOE_BITS
#define MOE_BITS 4
#endif

namespace moe {

typedef float f32x16_t __attribute__((ext_vector_type(16)));

// A block's part of the work: a tile of up to R sorted rows of one expert and a
// block of columns. Every wave finds it from the offsets by itself: one round of
// loads, then sums across the lanes. No offset leads past M.
//
// Tiles run through the experts, a tile's column blocks together, the whole list
// in eight contiguous ranges, one per XCD (blocks b, b + 8, ... share an XCD), whose
// L2 then keeps a tile's rows and an expert's weights. Whole tiles first and the
// shortest last, each tile on one XCD, came to the same or more: 128 experts of unequal
// popularity, 64 rows on average, 232 us for 231, 96 267 for 262, 32 of 128 rows, 2880 x
// 2880, 208 for 191, 60 of 150 rows, 1408 x 2048, 269 for 278.
struct GradTile {
  uint32_t e, m0, pend;  // expert, first sorted position, end
  int block;             // of columns
};
constexpr int kGradMaxE = 1024;
template <uint32_t R>
__device__ __forceinline__ bool grad_tile(const ExpertGradArgs& a, GradTile* t) {
  constexpr int P = kGradMaxE / 64;
  const int E = a.E, lane = threadIdx.x & 63;
  const uint32_t nb = (uint32_t)a.nb;
  uint32_t lo[P], hi[P];
#pragma unroll
  for (int i = 0; i < P; i++) {
    lo[i] = hi[i] = 0;
    if (i * 64 < E) {
      lo[i] = min(a.offsets[min(i * 64 + lane, E)], (uint32_t)a.M);
      hi[i] = max(min(a.offsets[min(i * 64 + lane + 1, E)], (uint32_t)a.M), lo[i]);
    }
  }
  uint32_t upto[P], tiles = 0;  // up to and with an expert's
#pragma unroll
  for (int i = 0; i < P; i++) {
    upto[i] = 0;
    if (i * 64 < E) {
      upto[i] = tiles + wave_scan_u32((hi[i] - lo[i] + R - 1) / R);
      tiles = (uint32_t)__builtin_amdgcn_readlane((int)upto[i], 63);
    }
  }
  const uint32_t k = blockIdx.x >> 3, per = (tiles * nb + 7u) >> 3, w = (blockIdx.x & 7u) * per + k, tile = w / nb;
  if (k >= per || tile >= tiles) return false;
  t->block = a.first + (int)(w - tile * nb);
  bool found = false;
#pragma unroll
  for (int i = 0; i < P; i++)
    if (i * 64 < E && !found) {
      const uint64_t past = __ballot(upto[i] > tile);
      if (past) {
        const int at = __ffsll((unsigned long long)past) - 1;
        const uint32_t l = (uint32_t)__builtin_amdgcn_readlane((int)lo[i], at);
        const uint32_t h = (uint32_t)__builtin_amdgcn_readlane((int)hi[i], at);
        const uint32_t first = (uint32_t)__builtin_amdgcn_readlane((int)upto[i], at) - (h - l + R - 1) / R;
        t->e = (uint32_t)(i * 64 + at);
        t->m0 = l + (tile - first) * R;
        t->pend = min(h, t->m0 + R);
        found = true;
      }
    }
  return found;
}
// Row of dy that sorted position pos takes.
__device__ __forceinline__ uint32_t grad_row(const ExpertGradArgs& a, uint32_t pos) {
  return min(a.perm[pos], (uint32_t)a.M - 1u) / (uint32_t)a.topk;
}

// Launches `kernel` on blocks for the most tiles of R rows that a.M rows of a.E
// experts can make, in two launches (left and right columns) where one cannot hold
// them (2^32 threads); hipErrorInvalidConfiguration past two.
static hipError_t launch_grad(void (*kernel)(const ExpertGradArgs), ExpertGradArgs a, int R, int C, int threads, hipStream_t st) {
  const int64_t tiles = (a.M / R + std::min(a.E, a.M) + 7) / 8 * 8, all = (a.K + C - 1) / C;
  const int64_t most = 0xFFFFFFFFll / threads / tiles;  // column blocks of a launch
  if (all > 2 * most) return hipErrorInvalidConfiguration;
  for (int64_t first = 0; first < all; first += most) {
    a.first = (int)first;
    a.nb = (int)std::min(most, all - first);
    hipLaunchKernelGGL(kernel, dim3((unsigned)(tiles * a.nb)), dim3(threads), 0, st, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

// ------------------------------------------------------------ fp32 products --
// fp32 rows: a block takes 64 rows and 64 columns, a wave a 32 x 32 quarter on
// v_mfma_f32_32x32x2; 32 values of the sum at a time go through two LDS buffers
// (the gradient's rows as they are, the weights dequantised, which keeps the
// packed axis across the lanes), loaded while the chunk before is multiplied. A chunk is
// summed by itself and then added, so that a sum of n values goes through 32 + n / 32
// roundings one after another, not n.
// Bound by the matrix cores where there are blocks enough: 64 rows of each of 128
// experts, two 768 x 2048 products at 4 bits, 477 us, 108 TFLOP/s (a large fp32
// product of the library 134). Small layers by the latency of their few chunks:
// 50 rows of each of 8, 512 x 1024, 18.5 us.
constexpr int kFR = 64, kFC = 64, kFK = 32;

template <int BITS>
__global__ __launch_bounds__(256) void expert_grad_f32_kernel(const ExpertGradArgs a) {
  __shared__ float As[2][kFR][kFK + 1], Bs[2][kFK][kFC];
  GradTile t;
  if (!grad_tile<kFR>(a, &t)) return;
  const int j0 = t.block * kFC, tid = threadIdx.x;
  const int lane = tid & 63, wave = tid >> 6, wm = wave >> 1, wn = wave & 1;
  const int col = lane & 31, half = lane >> 5;
  const int words = a.K / 32 * BITS, groups = a.K / 32 >> a.gsh;
  const int parts = (a.N + kFK - 1) / kFK, nchunks = a.dy2 ? 2 * parts : parts;
  // thread: a quarter of a gradient row's chunk, eight columns of a weight row (they
  // lie in two words, from bit `sh` of the first)
  const uint32_t pos = min(t.m0 + (uint32_t)(tid >> 2), t.pend - 1);
  const size_t arow = (size_t)(a.perm ? grad_row(a, pos) : pos) * a.N;
  const int ac = (tid & 3) * 8, bi = tid >> 3, bj = min(j0 + (tid & 7) * 8, a.K - 8);
  const uint32_t bit = (uint32_t)bj * BITS, lo = bit >> 5, sh = bit & 31;
  struct Part {
    float d[8], s, b;
    uint32_t w0, w1;
  };
  auto load = [&](int c, Part& u) {
    const bool second = c >= parts;
    const GemvProj& p = second ? a.p1 : a.p0;
    const int i0 = (second ? c - parts : c) * kFK, i = i0 + bi;
#pragma unroll
    for (int v = 0; v < 8; v++) u.d[v] = 0.0f;
    if (i0 + ac < a.N) Vec8<float>::load((const float*)(second ? a.dy2 : a.dy) + arow + i0 + ac, u.d);
    u.s = u.b = 0.0f;
    u.w0 = u.w1 = 0u;
    if (i < a.N) {
      const uint32_t* row = p.w + ((size_t)t.e * a.N + i) * words;
      const size_t g = ((size_t)t.e * a.N + i) * groups + (bj / 32 >> a.gsh);
      u.w0 = row[lo];
      u.w1 = row[min(lo + 1, (uint32_t)words - 1)];
      u.s = ((const float*)p.s)[g];
      u.b = ((const float*)p.b)[g];
    }
  };
  f32x16_t acc = {};
  Part u;
  load(0, u);
  for (int c = 0; c < nchunks; c++) {
    const int buf = c & 1;
    const uint64_t field = ((uint64_t)u.w1 << 32 | u.w0) >> sh;
    float wv[8];
#pragma unroll
    for (int v = 0; v < 8; v++) {
      As[buf][tid >> 2][ac + v] = u.d[v];
      wv[v] = __builtin_fmaf(u.s, (float)((uint32_t)(field >> (BITS * v)) & ((1u << BITS) - 1u)), u.b);
    }
    Vec8<float>::store(&Bs[buf][bi][(tid & 7) * 8], wv);
    if (c + 1 < nchunks) load(c + 1, u);
    lds_barrier();
    f32x16_t part = {};
#pragma unroll
    for (int k = 0; k < kFK; k += 2)
      part = __builtin_amdgcn_mfma_f32_32x32x2f32(As[buf][32 * wm + col][k + half], Bs[buf][k + half][32 * wn + col], part, 0, 0, 0);
    acc += part;
  }
  const int j = j0 + 32 * wn + col;
#pragma unroll
  for (int r = 0; r < 16; r++) {
    const uint32_t p = t.m0 + (uint32_t)(32 * wm + 8 * (r >> 2) + 4 * half + (r & 3));
    if (p < t.pend && j < a.K) {
      const size_t at = (size_t)p * a.K + j;
      ((float*)a.dx)[at] = (a.dx_in ? ((const float*)a.dx_in)[at] : 0.0f) + acc[r];
    }
  }
}

// ----------------------------------------------------------- 16-bit products --
// Rows in a 16-bit type take v_mfma_f32_32x32x16. A weight, dequantised in fp32, enters
// as two values of the rows' type: itself rounded (hi), and what that left, rounded (lo).
// Together they are within 2^-17 of it in bf16, 2^-23 in f16 (there 2^-25 where that is
// more, half the type's last bit), so that of 16 bits only the result's own rounding
// shows; hi alone, for half the matrix instructions, is off by 2^-8 and 2^-11. bf16
// gradients keep their range. The two are summed apart: a row or a weight that is not
// finite leaves the lo parts' sum NaN or infinite, and hi's alone is the result.
//
// The weights' packed axis is the output's, and the matrix operands want
// neighbours along the sum. The transposition costs nothing: a thread
// dequantises 16 columns of one weight row, with one scale and bias,
// into LDS as they lie ([sum][column]), and ds_read_tr16_b64 hands each lane
// its column's four values of the sum.
//
// A block of eight waves takes a row tile and 128 columns, the waves 2 x 4 with
// 128 rows x 32 columns (hi and lo: 64 columns of LDS) each, other tiles below: four
// waves of twice the columns read less from LDS but leave one wave a SIMD, whose vector
// work then stops the matrix cores. The weights are the products' first operand, so
// that a lane ends with four neighbouring columns of a row of dx.
//
// Per chunk of 64 values the block holds the tile's gradient rows (copied from
// memory straight into a ring of three LDS stages, two chunks ahead) and its
// weights (loaded three chunks ahead into registers, dequantised into two LDS
// buffers between the matrix steps of the chunk before). One barrier a chunk.
//
// 1024 rows of each of 32 experts, 2880 x 2880 at 4 bits, bf16: 966 us, 563 TFLOP/s of
// the product, twice that of the matrix cores; 256 of each of 128, two 768 x 2048
// products: 465 us (8 bits 421; f16 at 4 bits 445). A large bf16 product of the library
// reaches 1276, a loop of nothing but these matrix instructions on random operands
// 1543, with four vector instructions to each 1359: the chip lowers its clock as both
// kinds run, and a block's start and end are hidden by no other at one block a CU.
constexpr int kGK = 64;  // values of the sum per chunk

template <int MI_, int WN_>
struct GradShape {  // 32-row tiles a wave, waves along columns (32 each); two waves along rows
  static constexpr int MI = MI_, WM = 2, WN = WN_;
  static constexpr int NT = 64 * WM * WN, MR = 32 * MI * WM, NC = 32 * WN;
  static constexpr int UN = 2 * WN;               // units of 32 hi or lo parts in a weight row's LDS
  static constexpr int AI = MR * 8 / NT;          // 16-byte copies per thread and chunk
  static constexpr int ABYTES = MR * 128, BBYTES = kGK * UN * 64;
  static_assert(kGK * (NC / 16) == NT, "16 columns of a weight row per thread and chunk");
};

struct GradLds {
  unsigned char *a0, *a1, *a2, *b;
};

typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

template <typename XT>
__device__ __forceinline__ f32x16_t mma16(u32x4_t a, u32x4_t b, f32x16_t c) {
  if constexpr (__is_same(XT, bf16_t))
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                   __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a),
                                                  __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

// Slot of 16-byte piece c of gradient row r in its 128 bytes of LDS: rows lie
// two to a turn of the banks, so 16 rows reading one piece meet every bank once.
__device__ __forceinline__ int grad_swz(int r) { return (r >> 1) & 7; }
// Byte of piece s (8 columns) of unit u of weight row n: four rows that a
// transposing read takes together differ in the unit's slot, the rows and units
// that 16 lanes store together in the piece's.
template <int UN>
__device__ __forceinline__ uint32_t wt_off(int n, int u, int s) {
  const int f = (u ^ (u >> 2)) & 3;
  return (uint32_t)(n * UN * 64 + ((u ^ (n & 3)) << 6) + ((s ^ f) << 4));
}

// Codes 8 q ... 8 q + 7 of a unit, two to a register: code v in half half[v] of
// pr[reg[v]], from bit bit[v] on, and nothing else in that half. As f16 such a half is
// the subnormal code * 2^(bit - 24), exactly (its ten bits hold bit + BITS), so one
// mixed fma with the scale * 2^(24 - bit) gives scale * code + bias in fp32 without
// a shift or a conversion. Codes that would pass bit 10 are shifted down first.
template <int BITS> struct Codes;
template <> struct Codes<2> {
  static constexpr int reg[8] = {0, 1, 2, 3, 0, 1, 2, 3}, half[8] = {0, 0, 0, 0, 1, 1, 1, 1}, bit[8] = {0, 2, 4, 6, 0, 2, 4, 6};
};
template <> struct Codes<3> {
  static constexpr int reg[8] = {0, 1, 2, 3, 0, 1, 2, 3}, half[8] = {0, 0, 0, 0, 1, 1, 1, 1}, bit[8] = {0, 3, 6, 0, 0, 3, 6, 0};
};
template <> struct Codes<4> {
  static constexpr int reg[8] = {0, 1, 2, 3, 0, 1, 2, 3}, half[8] = {0, 0, 0, 0, 1, 1, 1, 1}, bit[8] = {0, 4, 0, 4, 0, 4, 0, 4};
};
template <> struct Codes<5> {
  static constexpr int reg[8] = {0, 0, 1, 3, 1, 2, 3, 2}, half[8] = {0, 1, 0, 0, 1, 0, 1, 1}, bit[8] = {0, 5, 2, 0, 4, 1, 0, 3};
};
template <> struct Codes<6> {
  static constexpr int reg[8] = {0, 3, 0, 1, 1, 3, 2, 2}, half[8] = {0, 0, 1, 0, 1, 1, 0, 1}, bit[8] = {0, 0, 4, 2, 0, 0, 4, 2};
};
template <> struct Codes<8> {
  static constexpr int reg[8] = {0, 0, 1, 1, 2, 2, 3, 3}, half[8] = {0, 1, 0, 1, 0, 1, 0, 1}, bit[8] = {};
};
template <int BITS, int NW>
__device__ __forceinline__ void code_pairs(const uint32_t (&w)[NW], int q, uint32_t (&pr)[4]) {
  constexpr uint32_t kOne = (1u << BITS) - 1u, kPair = kOne * 0x10001u;
  if constexpr (BITS == 4) {
    const uint32_t x = w[q], y = x >> 8;
    pr[0] = x & kPair;
    pr[1] = x & (kPair << 4);
    pr[2] = y & kPair;
    pr[3] = y & (kPair << 4);
  } else if constexpr (BITS == 8) {
#pragma unroll
    for (int p = 0; p < 4; p++) {
      const uint32_t lo = 2 * (p & 1);
      pr[p] = __builtin_amdgcn_perm(0u, w[2 * q + (p >> 1)], lo | 0x0C00u | ((lo + 1) << 16) | 0x0C000000u);
    }
  } else if constexpr (BITS == 2) {  // the quarter's two bytes, one to a half
    const uint32_t lo = 2 * (q & 1);
    const uint32_t x = __builtin_amdgcn_perm(0u, w[q >> 1], lo | 0x0C00u | ((lo + 1) << 16) | 0x0C000000u);
#pragma unroll
    for (int p = 0; p < 4; p++) pr[p] = x & (kPair << (2 * p));
  } else if constexpr (BITS == 3) {  // four codes (12 bits) to a half
    const int lo = 24 * q >> 5, sh = 24 * q & 31;
    const uint32_t f = sh == 8 || sh == 0 ? w[lo] >> sh : __builtin_amdgcn_alignbit(w[lo + 1 < NW ? lo + 1 : lo], w[lo], (uint32_t)sh);
    const uint32_t x = (f & 0xFFFFu) | ((f << 4) & 0xFFFF0000u);
    pr[0] = x & kPair;
    pr[1] = x & (kPair << 3);
    pr[2] = x & (kPair << 6);
    pr[3] = (x >> 9) & kPair;
  } else {  // 5 and 6 bits: each half takes the two bytes from the one that a code starts in
    typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
    const int at = BITS * q, wi = at >> 2, ob = at & 3;
#pragma unroll
    for (int r = 0; r < 4; r++) {
      uint32_t sel = 0, mask = 0;
      int down[2] = {0, 0};
#pragma unroll
      for (int v = 0; v < 8; v++)
        if (Codes<BITS>::reg[v] == r) {
          const int byte = ob + (BITS * v >> 3), o = BITS * v & 7, h = Codes<BITS>::half[v];
          const uint32_t two = (uint32_t)byte | (o + BITS > 8 ? (uint32_t)(byte + 1) << 8 : 0x0C00u);
          sel |= two << (16 * h);
          mask |= (kOne << Codes<BITS>::bit[v]) << (16 * h);
          down[h] = o - Codes<BITS>::bit[v];
        }
      const uint32_t z = __builtin_amdgcn_perm(w[wi + 1], w[wi], sel);
      if (down[0] || down[1]) {
        const u16x2_t t = __builtin_bit_cast(u16x2_t, z) >> u16x2_t{(unsigned short)down[0], (unsigned short)down[1]};
        pr[r] = __builtin_bit_cast(uint32_t, t) & mask;
      } else {
        pr[r] = z & mask;
      }
    }
  }
}

// Columns 8 q ... 8 q + 7 of a unit as weights: rounded to XT, and what that left.
template <int BITS, typename XT, int NW>
__device__ __forceinline__ void weights8(const uint32_t (&w)[NW], int q, float s, float b, u32x4_t& hi, u32x4_t& lo) {
  uint32_t pr[4];
  code_pairs<BITS>(w, q, pr);
  typedef XT x2_t __attribute__((ext_vector_type(2)));
  auto weight = [&](int v) {
    const float code = (float)__builtin_bit_cast(h2_t, pr[Codes<BITS>::reg[v]])[Codes<BITS>::half[v]];
    return __builtin_fmaf(code, s * (float)(1 << (24 - Codes<BITS>::bit[v])), b);
  };
#pragma unroll
  for (int p = 0; p < 4; p++) {
    const float w0 = weight(2 * p), w1 = weight(2 * p + 1);
    uint32_t pair = __builtin_bit_cast(uint32_t, x2_t{(XT)w0, (XT)w1});
    asm("" : "+v"(pair));  // (one conversion of both, not another of each)
    const x2_t h = __builtin_bit_cast(x2_t, pair);
    hi[p] = pair;
    lo[p] = __builtin_bit_cast(uint32_t, x2_t{(XT)(w0 - (float)h[0]), (XT)(w1 - (float)h[1])});
  }
}
// The sum of the products with the hi parts and of those with the lo parts.
__device__ __forceinline__ float joined(float hi, float lo) {
  return __builtin_fabsf(lo) < __builtin_huge_valf() ? hi + lo : hi;
}

// The 16 columns of a unit's half, as the first bits of kHalfWords words: loaded
// from the word that they begin in, `sh` bits (0 or 16) before them.
template <int BITS>
constexpr int kHalfWords = (BITS + 1) / 2;
template <int BITS>
__device__ __forceinline__ void bload_half(rsrc_t r, uint32_t off, uint32_t (&w)[kHalfWords<BITS>]) {
  if constexpr (kHalfWords<BITS> == 1) {
    w[0] = bload32(r, off);
  } else if constexpr (kHalfWords<BITS> == 2) {
    const u32x2_t v = bload64(r, off);
    w[0] = v[0], w[1] = v[1];
  } else if constexpr (kHalfWords<BITS> == 3) {
    const u32x3_t v = bload96(r, off);
    w[0] = v[0], w[1] = v[1], w[2] = v[2];
  } else {
    const u32x4_t v = bload128(r, off);
    w[0] = v[0], w[1] = v[1], w[2] = v[2], w[3] = v[3];
  }
}
template <int BITS>
__device__ __forceinline__ void shift_half(uint32_t (&w)[kHalfWords<BITS>], uint32_t sh) {
  if constexpr (BITS & 1) {
    constexpr int L = kHalfWords<BITS> - 1;
#pragma unroll
    for (int i = 0; i < L; i++) w[i] = __builtin_amdgcn_alignbit(w[i + 1], w[i], sh);
    w[L] >>= sh;
  }
}

// Keeps the compiler from moving a wave's LDS accesses across each other where lanes
// read what other lanes store. (The hardware serves them in order.)
__device__ __forceinline__ void wave_lds_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}

// f(0), f(1), ... with the numbers as types.
template <typename F, int... I>
__device__ __forceinline__ void each(F& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}

template <typename S, bool FAR, int BITS, typename XT>
__device__ __forceinline__ void grad_tile_mma(const ExpertGradArgs& a, const GradLds L, const GradTile& t, int j0) {
  constexpr int MI = S::MI, UN = S::UN, AI = S::AI, NT = S::NT, HW = kHalfWords<BITS>;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / S::WN, wn = wave % S::WN, col = lane & 31, h = lane >> 5;
  const int N = a.N, K = a.K, CU = K >> 5, groups = CU >> a.gsh, row_words = CU * BITS;
  const int per = (N + kGK - 1) / kGK, nchunks = a.dy2 ? 2 * per : per;
  const bool sb_bf16 = a.sb_bf16 != 0;
  auto stage = [&](auto st) -> unsigned char* {
    constexpr int ST = decltype(st)::value;
    return ST == 0 ? L.a0 : (ST == 1 ? L.a1 : L.a2);
  };

  // ---- gradient rows: thread tid copies, for i < AI, the piece that belongs in
  // slot tid % 8 of LDS row tid / 8 + NT / 8 * i (a wave's 64 lanes write one KB)
  // 32-bit offsets from a uniform base (FAR: gathered rows past 4 GB, 64-bit ones).
  // Behind the end of a row its last piece comes again, and zeros take its place when it
  // has arrived (end_rows): an infinity there must not meet the zero weights.
  const int ac = (tid & 7) ^ grad_swz(tid >> 3);
  uint32_t row[AI];
  const uint64_t first = a.perm ? 0 : (uint64_t)t.m0 * (uint64_t)N * 2u;
#pragma unroll
  for (int i = 0; i < AI; i++) {
    const uint32_t pos = min(t.m0 + (uint32_t)((tid >> 3) + NT / 8 * i), t.pend - 1);
    row[i] = a.perm ? grad_row(a, pos) : pos - t.m0;
    if constexpr (!FAR) row[i] *= (uint32_t)N * 2u;
  }
  // (every row of a thread is a multiple of 16 apart from its first: one slot)
  static_assert(NT / 8 % 16 == 0, "slots");
  auto copy_rows = [&](int chunk, auto st) {
    const bool second = chunk >= per;
    const uint32_t c0 = (uint32_t)(second ? chunk - per : chunk) * (kGK * 2);
    const unsigned char* base = reinterpret_cast<const unsigned char*>(second ? a.dy2 : a.dy) + first;
    const uint32_t x = min(c0 + (uint32_t)(16 * ac), (uint32_t)N * 2u - 16u);
#pragma unroll
    for (int i = 0; i < AI; i++) {
      const unsigned char* at = FAR ? base + (uint64_t)row[i] * ((uint64_t)N * 2u) + x : base + (row[i] + x);
      unsigned char* dst = stage(st) + (NT / 8 * i + 8 * wave) * 128;
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)at,
                                       (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
    }
  };
  auto end_rows = [&](int chunk, auto st) {
    const int c0 = (chunk >= per ? chunk - per : chunk) * kGK;
    if (chunk < nchunks && c0 + kGK > N && c0 + 8 * ac >= N)
#pragma unroll
      for (int i = 0; i < AI; i++)
        *reinterpret_cast<u32x4_t*>(stage(st) + NT / 8 * i * 128 + tid * 16) = u32x4_t{0u, 0u, 0u, 0u};
  };

  // ---- weights: thread tid dequantises half tid % 2 of unit tid / 2 % WN of row tid /
  // UN of the chunk. Columns past the end repeat the last unit (never stored), rows past
  // it read as zeros from the views.
  const int bh = tid & 1, bu = (tid >> 1) % S::WN, ju = min((j0 >> 5) + bu, CU - 1), bn = tid / UN;
  struct Units {
    uint32_t w[HW], s, b;
  };
  const uint32_t row_bytes = (uint32_t)row_words * 4u, group_bytes = (uint32_t)groups * 2u;
  const uint32_t bsh = BITS & 1 ? 16u * bh : 0u;
  const uint32_t woffs = (uint32_t)bn * row_bytes + (uint32_t)(ju * BITS + bh * (BITS / 2)) * 4u;
  const uint32_t goffs = (uint32_t)bn * group_bytes + (uint32_t)(ju >> a.gsh) * 2u;
  auto load_units = [&](int chunk, Units& u) {
    const bool second = chunk >= per;
    const GemvProj& p = second ? a.p1 : a.p0;
    const size_t at = (size_t)t.e * (size_t)N;
    const rsrc_t wv = make_rsrc(reinterpret_cast<const unsigned char*>(p.w) + at * row_bytes, (uint32_t)N * row_bytes);
    const rsrc_t sv = make_rsrc(reinterpret_cast<const unsigned char*>(p.s) + at * group_bytes, (uint32_t)N * group_bytes);
    const rsrc_t bv = make_rsrc(reinterpret_cast<const unsigned char*>(p.b) + at * group_bytes, (uint32_t)N * group_bytes);
    const uint32_t n0 = (uint32_t)((second ? chunk - per : chunk) * kGK);
    u.s = bload16(sv, goffs + n0 * group_bytes);
    u.b = bload16(bv, goffs + n0 * group_bytes);
    bload_half<BITS>(wv, woffs + n0 * row_bytes, u.w);
  };
  auto sb_value = [&](uint32_t raw) -> float {
    const float f = (float)__builtin_bit_cast(_Float16, (uint16_t)raw);
    return sb_bf16 ? __uint_as_float(raw << 16) : f;
  };
  // a half's values [8 q, 8 q + 8), hi and lo, into buffer buf
  auto store_quarter = [&](const uint32_t (&w)[HW], float s, float b, int q, int buf) {
    u32x4_t hi, lo;
    weights8<BITS, XT>(w, q, s, b, hi, lo);
    unsigned char* at = L.b + buf * S::BBYTES;
    *reinterpret_cast<u32x4_t*>(at + wt_off<UN>(bn, 2 * bu, 2 * bh + q)) = hi;
    *reinterpret_cast<u32x4_t*>(at + wt_off<UN>(bn, 2 * bu + 1, 2 * bh + q)) = lo;
  };
  auto unit_values = [&](const Units& u, uint32_t (&w)[HW], float& s, float& b) {
    s = sb_value(u.s);
    b = sb_value(u.b);
#pragma unroll
    for (int i = 0; i < HW; i++) w[i] = u.w[i];
    shift_half<BITS>(w, bsh);
  };

  f32x16_t acc[MI][2];  // of the hi parts, of the lo parts
#pragma unroll
  for (int i = 0; i < MI; i++) acc[i][0] = acc[i][1] = f32x16_t{};

  // operands of one 16-value step: gradient rows 32 (MI wm + i) + col, and for hi
  // and lo two transposing reads, of weight rows 16 s + 8 h + 4 q + (lane %
  // 16) / 4 (q < 2): their low two bits are the lane's, so one offset serves all
  struct Frags {
    u32x4_t w[2], d[MI];
  };
  const uint32_t doff = (uint32_t)(32 * MI * wm + col) * 128u;
  const int tr = (lane & 15) >> 2;  // row of four of a transposing read
  uint32_t woff[2];
#pragma unroll
  for (int j = 0; j < 2; j++)
    woff[j] = wt_off<UN>(8 * h + tr, 2 * wn + j, 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) + (uint32_t)(lane & 1) * 8u;
  auto read_frags = [&](auto st, int buf, int s, Frags& f) {
    const unsigned char* Ab = stage(st);
    const unsigned char* Bb = L.b + buf * S::BBYTES + s * (16 * UN * 64);
#pragma unroll
    for (int j = 0; j < 2; j++) {
      typedef __attribute__((address_space(3))) s16x4_t lds_t;
      const u32x2_t lo = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t*)(Bb + woff[j])));
      const u32x2_t hi = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t*)(Bb + woff[j] + 4 * UN * 64)));
      f.w[j] = u32x4_t{lo[0], lo[1], hi[0], hi[1]};
    }
    const uint32_t sw = (uint32_t)(((2 * s + h) ^ grad_swz(col)) << 4);
#pragma unroll
    for (int i = 0; i < MI; i++) f.d[i] = *reinterpret_cast<const u32x4_t*>(Ab + doff + 32 * 128 * i + sw);
  };
  auto mma_step = [&](const Frags& f) {
#pragma unroll
    for (int i = 0; i < MI; i++)
#pragma unroll
      for (int j = 0; j < 2; j++) acc[i][j] = mma16<XT>(f.w[j], f.d[i], acc[i][j]);
  };

  // Order of a chunk's main part: after each matrix instruction its share of the
  // vector work (kSetup for the scales, kQuarter per quarter of a unit), which
  // the matrix cores hide; a quarter's stores follow when its values are there.
  constexpr int kSetup = 10, kQuarter = 46, kWork = kSetup + 2 * kQuarter, kSteps = 6 * MI;
  auto weave = [&](auto seq) {
    auto one = [&](auto ic) {
      constexpr int i = decltype(ic)::value;
      constexpr int done = kWork * i / kSteps, next = kWork * (i + 1) / kSteps;
      constexpr int stored = done < kSetup ? 0 : (done - kSetup) / kQuarter, store = next < kSetup ? 0 : (next - kSetup) / kQuarter;
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      if constexpr (i % (2 * MI) < MI)  // (the next step's operands, early in this one)
        __builtin_amdgcn_sched_group_barrier(0x100, (4 + MI + MI - 1) / MI, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, next - done, 0);
      if constexpr (store > stored) __builtin_amdgcn_sched_group_barrier(0x200, 2 * (store - stored), 0);
    };
    each(one, seq);
  };
  constexpr int kUnitSet = 3;  // vector-memory instructions of a chunk's units per thread
  // Chunk c: rows in stage ST = c % 3, weights in buffer c % 2. Its first
  // operands are read behind the barrier while the previous chunk's last matrix
  // step (operands in registers) runs; chunk c + 2's rows go to the stage that
  // chunk c - 1 left, chunk c + 3's units to the registers that chunk c used,
  // and chunk c + 1's weights are dequantised between the matrix steps. Loads
  // past the end repeat the last chunk, in bounds and unused. At the end the
  // rows of chunk c + 1 have to be there: what was issued after them is chunk
  // c + 2's units, this step's AI copies and chunk c + 3's units; waiting until
  // no more than the last two are out covers them whatever the compiler merged.
  auto chunk_step = [&](auto first, auto st, int c, Units& cu, const Units& nu, Frags& last) {
    constexpr int ST = decltype(st)::value;
    const int buf = c & 1;
    Frags f0, f1;
    read_frags(st, buf, 0, f0);
    if constexpr (!decltype(first)::value) mma_step(last);
    copy_rows(min(c + 2, nchunks - 1), std::integral_constant<int, (ST + 2) % 3>{});
    __builtin_amdgcn_sched_barrier(0);
    load_units(min(c + 3, nchunks - 1), cu);
    __builtin_amdgcn_sched_barrier(0);
    uint32_t w[HW];
    float s, b;
    unit_values(nu, w, s, b);
    read_frags(st, buf, 1, f1);
    mma_step(f0);
    store_quarter(w, s, b, 0, buf ^ 1);
    read_frags(st, buf, 2, f0);
    mma_step(f1);
    read_frags(st, buf, 3, last);
    mma_step(f0);
    store_quarter(w, s, b, 1, buf ^ 1);
    weave(std::make_integer_sequence<int, 6 * MI>{});
    __builtin_amdgcn_sched_barrier(0);
    vmcnt_wait<AI + kUnitSet>();
    end_rows(c + 1, std::integral_constant<int, (ST + 1) % 3>{});
    lds_barrier_copies_in_flight();
  };

  using S0 = std::integral_constant<int, 0>;
  using S1 = std::integral_constant<int, 1>;
  using S2 = std::integral_constant<int, 2>;
  Units u0, u1, u2;
  load_units(0, u0);
  load_units(min(1, nchunks - 1), u1);
  load_units(min(2, nchunks - 1), u2);
  __builtin_amdgcn_sched_barrier(0);
  copy_rows(0, S0{});
  copy_rows(min(1, nchunks - 1), S1{});
  __builtin_amdgcn_sched_barrier(0);
  {
    uint32_t w[HW];
    float s, b;
    unit_values(u0, w, s, b);
    store_quarter(w, s, b, 0, 0);
    store_quarter(w, s, b, 1, 0);
  }
  vmcnt_wait<0>();
  end_rows(0, S0{});
  lds_barrier_copies_in_flight();
  Frags last;
  chunk_step(std::true_type{}, S0{}, 0, u0, u1, last);
  int c = 1;
  for (; c + 3 <= nchunks; c += 3) {
    chunk_step(std::false_type{}, S1{}, c, u1, u2, last);
    chunk_step(std::false_type{}, S2{}, c + 1, u2, u0, last);
    chunk_step(std::false_type{}, S0{}, c + 2, u0, u1, last);
  }
  if (c < nchunks) chunk_step(std::false_type{}, S1{}, c, u1, u2, last);
  if (c + 1 < nchunks) chunk_step(std::false_type{}, S2{}, c + 1, u2, u0, last);
  mma_step(last);
  vmcnt_wait<0>();  // the copies past the end
  __syncthreads();

  // ---- results: lane holds row col of each 32-row tile and columns 8 (r / 4) +
  // 4 h + r % 4; through LDS, so that a lane stores 16 bytes of a row and its
  // neighbours the bytes beside them
  uint16_t* out = reinterpret_cast<uint16_t*>(a.dx);
  const uint16_t* base = reinterpret_cast<const uint16_t*>(a.dx_in);
  constexpr int LINE = 144;  // bytes of a staged row
  static_assert(S::WM * S::WN * 32 * LINE <= 2 * S::BBYTES, "staging");
  unsigned char* mine = L.b + wave * (32 * LINE);
  const int jw = j0 + 32 * wn;
  if (!base) {
#pragma unroll
    for (int i = 0; i < MI; i++) {
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        typedef XT x4_t __attribute__((ext_vector_type(4)));
        x4_t v;
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = (XT)joined(acc[i][0][r + k], acc[i][1][r + k]);
        *reinterpret_cast<u32x2_t*>(mine + col * LINE + r * 4 + h * 8) = __builtin_bit_cast(u32x2_t, v);
      }
      wave_lds_order();
#pragma unroll
      for (int q = 0; q < 2; q++) {
        const int row = 16 * q + (lane >> 2), c8 = lane & 3;
        const u32x4_t v = *reinterpret_cast<const u32x4_t*>(mine + row * LINE + c8 * 16);
        const uint32_t pos = t.m0 + (uint32_t)(32 * (MI * wm + i) + row);
        if (pos < t.pend && jw + 8 * c8 < K)
          *reinterpret_cast<u32x4_t*>(out + (size_t)pos * K + jw + 8 * c8) = v;
      }
      wave_lds_order();
    }
  } else {  // added to dx_in in fp32
#pragma unroll
    for (int i = 0; i < MI; i++) {
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        typedef float f32x4_t __attribute__((ext_vector_type(4)));
        f32x4_t v;
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = joined(acc[i][0][r + k], acc[i][1][r + k]);
        *reinterpret_cast<f32x4_t*>(mine + col * LINE + r * 8 + h * 16) = v;
      }
      wave_lds_order();
#pragma unroll
      for (int q = 0; q < 2; q++) {
        const int row = 16 * q + (lane >> 2), c8 = lane & 3;
        float v[8], o[8];
        Vec8<float>::load(reinterpret_cast<const float*>(mine + row * LINE + c8 * 32), v);
        const uint32_t pos = t.m0 + (uint32_t)(32 * (MI * wm + i) + row);
        const int jc = jw + 8 * c8;
        if (pos < t.pend && jc < K) {
          const size_t at = (size_t)pos * K + jc;
          Vec8<XT>::load(reinterpret_cast<const XT*>(base) + at, o);
#pragma unroll
          for (int k = 0; k < 8; k++) o[k] += v[k];
          Vec8<XT>::store(reinterpret_cast<XT*>(out) + at, o);
        }
      }
      wave_lds_order();
    }
  }
}

typedef GradShape<4, 4> GradTall;     // 256 rows x 128 columns
typedef GradShape<3, 4> GradMost;     // 192 rows
typedef GradShape<2, 4> GradHalf;     // 128 rows
typedef GradShape<1, 4> GradQuarter;  // 64 rows

template <bool FAR, int BITS, typename XT>
__global__ __launch_bounds__(GradTall::NT) void expert_grad_tall_kernel(const ExpertGradArgs a) {
  __shared__ __align__(16) unsigned char a0[GradTall::ABYTES], a1[GradTall::ABYTES], a2[GradTall::ABYTES];
  __shared__ __align__(16) unsigned char b[2 * GradTall::BBYTES];
  GradTile t;
  if (!grad_tile<GradTall::MR>(a, &t)) return;
  const int j0 = t.block * GradTall::NC;
  const GradLds L{a0, a1, a2, b};
  const uint32_t rows = t.pend - t.m0;
  if (rows > 192) grad_tile_mma<GradTall, FAR, BITS, XT>(a, L, t, j0);
  else if (rows > 128) grad_tile_mma<GradMost, FAR, BITS, XT>(a, L, t, j0);
  else if (rows > 64) grad_tile_mma<GradHalf, FAR, BITS, XT>(a, L, t, j0);
  else grad_tile_mma<GradQuarter, FAR, BITS, XT>(a, L, t, j0);
}

// ------------------------------------------------ 16-bit products, few rows --
// Experts with few rows are bound by how fast their weights arrive and are dequantised.
// A block takes up to 32 rows and 128 WN columns; four waves, WN side by side along the
// columns, share the sum (chunks of 32 values in turn) and meet at the end. A wave
// dequantises into LDS of its own, 16 weight rows at a time, so the loop has no barrier:
// LDS serves a wave's stores and reads in order.
//
// 8 rows of each of 128 experts, two 768 x 2048 products at 4 bits, bf16: 100 us, 2.3
// TB/s of experts and rows; 6 rows of each of 32, 2880 x 2880: 69 us, 2.2 TB/s, where a
// large copy reaches 5.2. Bound by instructions: the vector units are busy 59% of a SIMD's
// time and the matrix cores 21%. Of a chunk's 330 vector instructions a wave, a third make
// the lo parts. Three waves a SIMD for two (8 bits: two, they need 207 registers): 75 us for
// 87.
//
// The hi and lo parts are summed together (128 registers of sums would leave two waves a
// SIMD): where a sum is not finite, the block sums the hi parts alone again for the
// elements that were not.
constexpr int kFewRows = 32;
constexpr int kFewLine = 64 * 4 + 16;  // a staged row of 64 fp32 columns

template <int WN, int BITS, typename XT>
__global__ __launch_bounds__(256, BITS == 8 ? 2 : 3) void expert_grad_few_kernel(const ExpertGradArgs a) {
  constexpr int NJ = 4, FK = 32, FC = 128 * WN, STEPS = FK / 16, WK = 4 / WN;
  constexpr int kPart = 16 * 256;  // hi parts of 16 weight rows; the lo parts behind them
  constexpr int kWave = kFewRows * kFewLine;
  static_assert(kWave >= 2 * kPart, "staging");
  __shared__ __align__(16) unsigned char lds[4 * kWave];
  GradTile t;
  if (!grad_tile<kFewRows>(a, &t)) return;
  const int j0 = t.block * FC, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wn = wave % WN, col = lane & 31, h = lane >> 5;
  const int N = a.N, K = a.K, CU = K >> 5, groups = CU >> a.gsh, row_words = CU * BITS;
  const int parts = (N + FK - 1) / FK, nchunks = a.dy2 ? 2 * parts : parts;
  const bool sb_bf16 = a.sb_bf16 != 0;

  const uint32_t pos = min(t.m0 + (uint32_t)col, t.pend - 1);
  const size_t arow = (size_t)(a.perm ? grad_row(a, pos) : pos) * N;
  // lane: unit lane % 4 of weight rows lane / 4 and 16 + lane / 4 of a chunk
  const int bu = lane % NJ, ju = min((j0 >> 5) + NJ * wn + bu, CU - 1), bn = lane / NJ;
  struct Chunk {
    uint32_t w[STEPS][BITS], s[STEPS], b[STEPS];
    u32x4_t d[STEPS];
  };
  auto load = [&](int c, Chunk& u) {
    const bool second = c >= parts;
    const GemvProj& p = second ? a.p1 : a.p0;
    const size_t rows = (size_t)t.e * (size_t)N;
    const rsrc_t wv = make_rsrc(p.w + rows * row_words, (uint32_t)N * (uint32_t)row_words * 4u);
    const rsrc_t sv = make_rsrc(reinterpret_cast<const uint16_t*>(p.s) + rows * groups, (uint32_t)N * (uint32_t)groups * 2u);
    const rsrc_t bv = make_rsrc(reinterpret_cast<const uint16_t*>(p.b) + rows * groups, (uint32_t)N * (uint32_t)groups * 2u);
    const int n0 = (second ? c - parts : c) * FK;
#pragma unroll
    for (int i = 0; i < STEPS; i++) {
      const uint32_t n = (uint32_t)(n0 + bn + 16 * i), g = (n * (uint32_t)groups + (uint32_t)(ju >> a.gsh)) * 2u;
      bload_unit<BITS>(wv, (n * (uint32_t)row_words + (uint32_t)(ju * BITS)) * 4u, u.w[i]);
      u.s[i] = bload16(sv, g);
      u.b[i] = bload16(bv, g);
    }
    const uint16_t* dy = reinterpret_cast<const uint16_t*>(second ? a.dy2 : a.dy) + arow;
#pragma unroll
    for (int s = 0; s < STEPS; s++)
      u.d[s] = *reinterpret_cast<const u32x4_t*>(dy + min(n0 + 16 * s + 8 * h, N - 8));
  };
  auto sb_value = [&](uint32_t raw) -> float {
    const float f = (float)__builtin_bit_cast(_Float16, (uint16_t)raw);
    return sb_bf16 ? __uint_as_float(raw << 16) : f;
  };
  unsigned char* mine = lds + wave * kWave;
  const int tr = (lane & 15) >> 2;
  uint32_t woff[NJ];
#pragma unroll
  for (int j = 0; j < NJ; j++)
    woff[j] = wt_off<NJ>(8 * h + tr, j, 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) + (uint32_t)(lane & 1) * 8u;
  f32x16_t acc[NJ];
  auto products = [&](auto both, int c, const Chunk& u) {
    constexpr int PARTS = decltype(both)::value ? 2 : 1;
    const int n0 = (c >= parts ? c - parts : c) * FK;
#pragma unroll
    for (int s = 0; s < STEPS; s++) {
      const float sc = sb_value(u.s[s]), bi = sb_value(u.b[s]);
#pragma unroll
      for (int q = 0; q < 4; q++) {
        u32x4_t hi, lo;
        weights8<BITS, XT>(u.w[s], q, sc, bi, hi, lo);
        unsigned char* at = mine + wt_off<NJ>(bn, bu, q);
        *reinterpret_cast<u32x4_t*>(at) = hi;
        if constexpr (PARTS == 2) *reinterpret_cast<u32x4_t*>(at + kPart) = lo;
      }
      wave_lds_order();
      // (values past the end of the row met zero weights; an infinity there must not)
      const u32x4_t d = n0 + 16 * s + 8 * h < N ? u.d[s] : u32x4_t{0u, 0u, 0u, 0u};
#pragma unroll
      for (int part = 0; part < PARTS; part++)
#pragma unroll
        for (int j = 0; j < NJ; j++) {
          typedef __attribute__((address_space(3))) s16x4_t lds_t;
          const unsigned char* at = mine + part * kPart + woff[j];
          const u32x2_t x = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t*)at));
          const u32x2_t y = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t*)(at + 4 * 256)));
          acc[j] = mma16<XT>(u32x4_t{x[0], x[1], y[0], y[1]}, d, acc[j]);
        }
      wave_lds_order();
    }
  };
  auto sums = [&](auto both) {
#pragma unroll
    for (int j = 0; j < NJ; j++) acc[j] = f32x16_t{};
    Chunk u0, u1;
    int c = wave / WN;  // chunks c, c + WK, ...; loads past the end repeat the last chunk, unused
    auto ahead = [&](int at, Chunk& u) {
      __builtin_amdgcn_sched_barrier(0);  // (loads sink to their uses otherwise)
      load(min(at, nchunks - 1), u);
      __builtin_amdgcn_sched_barrier(0);
    };
    ahead(c, u0);
    ahead(c + WK, u1);
    for (; c + WK < nchunks; c += 2 * WK) {
      products(both, c, u0);
      ahead(c + 2 * WK, u0);
      products(both, c + WK, u1);
      ahead(c + 3 * WK, u1);
    }
    if (c < nchunks) products(both, c, u0);
  };
  // The waves' sums, 64 columns of each at a time: lane holds row col and columns 8 (r /
  // 4) + 4 h + r % 4 of each 32; thread tid then adds row tid / 8, columns 8 (tid % 8) on.
  // Bit q of `left`'s byte (part WN + g): an element that is left, since it is not finite.
  uint32_t left = 0;
  auto results = [&](auto both) {
#pragma unroll
    for (int part = 0; part < NJ / 2; part++) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 2; j++)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
          const f32x16_t& v = acc[2 * part + j];
          *reinterpret_cast<float4*>(lds + (wave * kFewRows + col) * kFewLine + j * 128 + r * 8 + h * 16) =
              make_float4(v[r], v[r + 1], v[r + 2], v[r + 3]);
        }
      __syncthreads();
      const int row = tid >> 3;
      const uint32_t p = t.m0 + (uint32_t)row;
#pragma unroll
      for (int g = 0; g < WN; g++) {
        const int jc = j0 + 128 * g + 64 * part + 8 * (tid & 7), byte = 8 * (part * WN + g);
        if (p < t.pend && jc < K) {
          float v[WK][8], o[8] = {};
#pragma unroll
          for (int w = 0; w < WK; w++)
            Vec8<float>::load(reinterpret_cast<const float*>(lds + ((w * WN + g) * kFewRows + row) * kFewLine + (tid & 7) * 32), v[w]);
          const size_t at = (size_t)p * K + jc;
          if (a.dx_in) Vec8<XT>::load(reinterpret_cast<const XT*>(a.dx_in) + at, o);
          uint32_t odd = 0;
#pragma unroll
          for (int q = 0; q < 8; q++) {
            float sum = v[0][q] + v[1][q];
            if constexpr (WK == 4) sum += v[2][q] + v[3][q];
            if (!(__builtin_fabsf(sum) < __builtin_huge_valf())) odd |= 1u << q;
            o[q] += sum;
          }
          XT* out = reinterpret_cast<XT*>(a.dx) + at;
          if (decltype(both)::value && !odd) {
            Vec8<XT>::store(out, o);
          } else {
            const uint32_t now = decltype(both)::value ? ~odd : left >> byte;
#pragma unroll
            for (int q = 0; q < 8; q++)
              if (now >> q & 1u) out[q] = (XT)o[q];
            if constexpr (decltype(both)::value) left |= odd << byte;
          }
        }
      }
    }
  };
  sums(std::true_type{});
  results(std::true_type{});
  if (!__syncthreads_or(left != 0)) return;
  sums(std::false_type{});
  results(std::false_type{});
}

typedef GradShape<2, 2> GradMid;  // 128 rows x 64 columns
typedef GradShape<1, 2> GradMidHalf;

template <bool FAR, int BITS, typename XT>
__global__ __launch_bounds__(GradMid::NT, 2) void expert_grad_mid_kernel(const ExpertGradArgs a) {
  __shared__ __align__(16) unsigned char a0[GradMid::ABYTES], a1[GradMid::ABYTES], a2[GradMid::ABYTES];
  __shared__ __align__(16) unsigned char b[2 * GradMid::BBYTES];
  GradTile t;
  if (!grad_tile<GradMid::MR>(a, &t)) return;
  const int j0 = t.block * GradMid::NC;
  const GradLds L{a0, a1, a2, b};
  const uint32_t rows = t.pend - t.m0;
  if (rows > 64) grad_tile_mma<GradMid, FAR, BITS, XT>(a, L, t, j0);
  else grad_tile_mma<GradMidHalf, FAR, BITS, XT>(a, L, t, j0);
}

// Which kernel. Up to 44 rows an expert on average the few-row kernel, its blocks wide
// from 20 rows on where that leaves enough for most of the chip (320); else the tall
// kernel, unless its blocks would not fill the chip (160), then the ordinary one.
// us per call of gate and up 768 x 2048 at 4 bits, bf16, experts of unequal popularity,
// few / wide / ordinary / tall: 128 experts of 16 rows 110 / 118 / 180 / 178, of 24 122 /
// 119 / 185 / 180, of 32 143 / 140 / 192 / 189, of 48 196 / 188 / 204 / 193, of 64 238 /
// 228 / 218 / 219, of 128 426 / 389 / 340 / 284. Other formats: 32 rows of 2 bits 139 / 132
// / 186 / 190, 5 bits 166 / 158 / 205 / 202, 6 bits 168 / 157 / 210 / 197, 8 bits 183 / 167
// / 211 / 203; 48 rows of 2 bits 188 / 178 / 191 / 191, 5 bits 224 / 208 / 213 / 211, 6 bits
// 224 / 211 / 215 / 204, 8 bits 246 / 223 / 218 / 207; f16, 3 bits, 256 experts 512 x 2048 of
// 24 rows 192 / 184 / 280 / 298, of 48 322 / 288 / 311 / 314.
// Few blocks: few and ordinary, 8 experts of 16 rows 21 / 19, one of one row 20 / 19, 4 of
// one row, 2880 x 2880, 34 / 41; few and wide, 32 experts of 32 rows (256 wide ones) 33 / 38, 20 of
// 20 rows, 5120 x 5120 (400) 164 / 160; ordinary and tall, 8 of 256 rows (128 tall ones) 34 /
// 39, 4 of 512, 2880 x 2880 (184) 85 / 70, one of 4096 (256) 67 / 49.
template <int BITS, typename XT>
static hipError_t launch_mma(const ExpertGradArgs& a, hipStream_t st) {
  const int64_t used = std::min(a.E, a.M);
  if ((int64_t)a.M <= 44 * (int64_t)a.E) {
    if ((int64_t)a.M >= 20 * (int64_t)a.E && used * ((a.K + 255) / 256) >= 320)
      return launch_grad(expert_grad_few_kernel<2, BITS, XT>, a, kFewRows, 256, 256, st);
    return launch_grad(expert_grad_few_kernel<1, BITS, XT>, a, kFewRows, 128, 256, st);
  }
  const bool far = a.perm && (int64_t)a.rows * a.N * 2 > 0xFFFFFFFFll;
  if (std::max<int64_t>(used, a.M / GradTall::MR) * ((a.K + GradTall::NC - 1) / GradTall::NC) < 160)
    return launch_grad(far ? expert_grad_mid_kernel<true, BITS, XT> : expert_grad_mid_kernel<false, BITS, XT>, a, GradMid::MR,
                       GradMid::NC, GradMid::NT, st);
  return launch_grad(far ? expert_grad_tall_kernel<true, BITS, XT> : expert_grad_tall_kernel<false, BITS, XT>, a, GradTall::MR,
                     GradTall::NC, GradTall::NT, st);
}

#define MOE_CAT2(a, b) a##b
#define MOE_CAT(a, b) MOE_CAT2(a, b)

hipError_t MOE_CAT(launch_expert_grad_b, MOE_BITS)(int xdt, int sbdt, const ExpertGradArgs& a0, hipStream_t st) {
  if (xdt == DT_F32) return launch_grad(expert_grad_f32_kernel<MOE_BITS>, a0, kFR, kFC, 256, st);
  ExpertGradArgs a = a0;
  a.sb_bf16 = sbdt == DT_BF16;
  return xdt == DT_BF16 ? launch_mma<MOE_BITS, bf16_t>(a, st) : launch_mma<MOE_BITS, f16_t>(a, st);
}

}  // namespace moe
