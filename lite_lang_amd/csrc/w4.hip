// Products with weights of 4 bits and a scale for each group of inputs (gfx950):
//   y[m, n] = sum_k x[m, k] (c[n, k] - z[n, k / group]) s[n, k / group] + bias[n]
// with c in 0 .. 15, z the zero point (8 where a weight has none) and s in x's
// type.
//
// A weight is laid out once (ll_w4_pack) as the operand of a 16x16x32 MFMA: a
// tile is 16 rows of 128 inputs, 1 KB, in which lane l holds 16 bytes: row
// l % 16, and in dword j the inputs 32 j + 8 (l / 16) + 0 .. 7. Nibble i of a
// dword is input 2 i and nibble i + 4 input 2 i + 1, so that a shift, an `and`
// and an `or` make two 16-bit floats at once: 128 + c (times a power of two) in
// bf16, 0x6400 | c, 1024 + c, in fp16. For bf16 the 128 stays in and leaves with
// the zero point: a group's sum is
//   sum x (128 + c) - (128 + z) sum x,
// the second sum taken by the same instruction from a tile of ones (it loses
// 128 / 15 times fp32's rounding, 2^-20 of the result's terms). In fp16 1024 is
// subtracted, which is exact.
#include <algorithm>
#include <mutex>
#include <type_traits>

#include "ll_common.h"

namespace {

constexpr int kTileK = 128;
constexpr int kWavesW4 = 4;

struct PackedW4 {  // the parts of a packed weight, in this order, each 256-aligned
  int64_t codes, scale, zero, total;
};

int64_t align256w(int64_t v) { return (v + 255) & ~(int64_t)255; }

PackedW4 layout_w4(int64_t N, int64_t K, int64_t group, bool zero) {
  const int64_t nt = (N + 15) / 16, kt = (K + kTileK - 1) / kTileK;
  PackedW4 p;
  p.codes = 0;
  p.scale = align256w(nt * kt * 1024);
  p.zero = p.scale + align256w(nt * kt * (kTileK / group) * 16 * 2);
  p.total = p.zero + (zero ? align256w(nt * kt * (kTileK / group) * 16) : 0);
  return p;
}

// One thread per dword of codes; the first ones also lay out scales and zeros.
__global__ __launch_bounds__(256) void w4_pack_kernel(
    const uint8_t* __restrict__ codes, int64_t ldc, const uint16_t* __restrict__ scale, int64_t lds,
    const uint8_t* __restrict__ zero, int64_t ldz, int64_t N, int64_t K, int group, uint8_t* out,
    PackedW4 p) {
  const int64_t nt = (N + 15) / 16, kt = (K + kTileK - 1) / kTileK;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < nt * kt * 256) {
    const int64_t tile = i / 256;
    const int l = (int)(i % 256) / 4, j = (int)(i % 4);
    const int64_t n = tile / kt * 16 + l % 16, k = tile % kt * kTileK + j * 32 + l / 16 * 8;
    uint32_t w = 0;
    if (n < N && k < K) {  // (K is a multiple of 32)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const uint32_t c = codes[n * ldc + k / 2 + b];
        w |= (c & 15u) << (4 * b) | (c >> 4) << (4 * b + 16);
      }
    }
    ((uint32_t*)(out + p.codes))[i] = w;
  }
  const int gpt = kTileK / group;
  if (i < nt * kt * gpt * 16) {
    const int64_t g = i / 16 % (kt * gpt), n = i / 16 / (kt * gpt) * 16 + i % 16;
    const bool in = n < N && g * group < K;
    ((uint16_t*)(out + p.scale))[i] = in ? scale[n * lds + g] : (uint16_t)0;
    if (zero) (out + p.zero)[i] = in ? zero[n * ldz + g] & 15 : (uint8_t)8;
  }
}

struct W4Args {
  const void* x; int64_t ldx;
  const uint8_t* codes; const uint16_t* scale; const uint8_t* zero;
  const void* bias;
  void* y; int64_t ldy;
  int64_t M, N, K, kt;
  float* part; int span, splits;  // sums of `splits` splits of `span` stretches
};

// Two constants of the conversion, kept from the compiler so that they stay in
// registers: an `and` and an `or` of two literals are two instructions, of a
// scalar and a vector register one.
struct W4Bits {
  uint32_t mask, base;
};

template <typename T> struct W4Type;
template <> struct W4Type<__bf16> {
  typedef bf16x8 V;
  typedef __bf16 V2 __attribute__((ext_vector_type(2)));
  // 128 + c and the ones of the sums of x are held small by powers of two, so that
  // no sum passes fp32's range where the result does not: 0x3b00 | c is 2^-16 (128 +
  // c), and the sums are 2^-8 of themselves.
  static constexpr uint32_t base = 0x3b003b00u, one = 0x3b803b80u;
  static constexpr float back = 0x1p16f;  // an accumulator is the result by 1 / back
  // what a converted code is more than the weight, of zero point z, by 2^-8
  static __device__ __forceinline__ float off(float z) {
    return __builtin_fmaf(z, 0x1p-8f, 0.5f);
  }
  static constexpr bool summed(bool) { return true; }  // whether it takes sums of x
  static __device__ __forceinline__ uint32_t pair(uint32_t w, W4Bits b, bool) {
    return (w & b.mask) | b.base;
  }
  static __device__ __forceinline__ f32x4 mfma(V a, V b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float add2(uint32_t x, float c) {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(V2, x), __builtin_bit_cast(V2, one),
                                           c, false);
  }
};
template <> struct W4Type<_Float16> {
  typedef f16x8 V;
  typedef _Float16 V2 __attribute__((ext_vector_type(2)));
  static constexpr uint32_t base = 0x64006400u, one = 0x3c003c00u;
  static constexpr float back = 1.f;
  static __device__ __forceinline__ float off(float z) { return z; }
  static constexpr bool summed(bool zero) { return zero; }  // (without, 8 is taken off in pair())
  static __device__ __forceinline__ uint32_t pair(uint32_t w, W4Bits b, bool zero) {
    const _Float16 o = zero ? (_Float16)1024.f : (_Float16)1032.f;
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(V2, (w & b.mask) | b.base) - (V2){o, o});
  }
  static __device__ __forceinline__ f32x4 mfma(V a, V b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float add2(uint32_t x, float c) {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(V2, x), __builtin_bit_cast(V2, one), c, false);
  }
};

template <typename T> __device__ __forceinline__ W4Bits w4_bits() {
  W4Bits b = {0x000f000fu, W4Type<T>::base};
  asm("" : "+s"(b.mask), "+v"(b.base));
  return b;
}

// What a wave loads of R weight tiles for one stretch of 128 inputs.
template <int GROUP, bool ZERO, int R> struct Stretch {
  static constexpr int kGpt = kTileK / GROUP;
  u32x4 w[R];
  uint2 s[R][kGpt];
  uint32_t z[R][ZERO ? kGpt : 1];
};

template <int GROUP, bool ZERO, int R>
__device__ __forceinline__ void fetch_w(Stretch<GROUP, ZERO, R>& f, const W4Args& a, int nt0,
                                        int last, int kt, int lane) {
  constexpr int kGpt = kTileK / GROUP;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t tile = (int64_t)min(nt0 + r, last) * a.kt + kt;
    f.w[r] = ((const u32x4*)a.codes)[tile * 64 + lane];
#pragma unroll
    for (int gi = 0; gi < kGpt; ++gi) {
      const int64_t at = (tile * kGpt + gi) * 16 + (lane >> 4) * 4;
      f.s[r][gi] = *(const uint2*)(a.scale + at);
      if constexpr (ZERO) f.z[r][gi] = *(const uint32_t*)(a.zero + at);
    }
  }
}

// acc += the products of one stretch. x(j, mb): the operand of chunk j of 32
// inputs; sum(gi, mb): the sum of a lane's own row of x over group gi.
template <typename T, int GROUP, bool ZERO, int R, int MB, typename X, typename S>
__device__ __forceinline__ void multiply(const Stretch<GROUP, ZERO, R>& f, W4Bits bits, X x, S sum,
                                         f32x4 (&acc)[R][MB]) {
  typedef W4Type<T> W;
  typedef typename W::V V;
  constexpr int kCpg = GROUP / 32;  // chunks of 32 inputs per group
#pragma unroll
  for (int gi = 0; gi < kTileK / GROUP; ++gi) {
    f32x4 part[R][MB] = {};
#pragma unroll
    for (int jj = 0; jj < kCpg; ++jj) {
      const int j = gi * kCpg + jj;
      V xf[MB];
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) xf[mb] = x(j, mb);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        u32x4 p;
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = W::pair(f.w[r][j] >> (4 * i), bits, ZERO);
        const V wf = __builtin_bit_cast(V, p);
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) part[r][mb] = W::mfma(wf, xf[mb], part[r][mb]);
      }
    }
    float xsum[MB];
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) xsum[mb] = W::summed(ZERO) ? sum(gi, mb) : 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint16_t sb = (uint16_t)((e < 2 ? f.s[r][gi].x : f.s[r][gi].y) >> (16 * (e & 1)));
        const float s = ll_to_f32(__builtin_bit_cast(T, sb));
        const float z = W::off(ZERO ? (float)((f.z[r][gi] >> (8 * e)) & 255u) : 8.f);
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
          float v = part[r][mb][e];
          if constexpr (W::summed(ZERO)) v = __builtin_fmaf(-z, xsum[mb], v);
          acc[r][mb][e] = __builtin_fmaf(s, v, acc[r][mb][e]);
        }
      }
  }
}

// The sum of a row's inputs in one group, from the operand of 16 rows: by the
// same instruction from a tile of ones.
template <typename T, int GROUP, typename X> __device__ __forceinline__ float sum_of(int gi, X x) {
  typedef W4Type<T> W;
  typedef typename W::V V;
  const u32x4 o = {W::one, W::one, W::one, W::one};
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int jj = 0; jj < GROUP / 32; ++jj)
    s = W::mfma(__builtin_bit_cast(V, o), x(gi * (GROUP / 32) + jj), s);
  return s[0];
}

// R tiles of 16 weight rows by MB tiles of 16 rows of x per workgroup; its waves
// take every WAVES-th stretch of inputs, the loads of AHEAD stretches in flight
// (under no condition, so that a wait counts what came after its load), and add
// up through LDS. What bounds it is the weight's way from memory (151,936 x 1536, 5
// rows: 35 us, 3.6 TB/s), for small weights the chain of loads and the reduction
// (2048 x 11,008, one row: 6.5 us for 11.7 MB); x comes from the L2, which R weight
// tiles share.
template <typename T, int GROUP, bool ZERO, int R, int MB, int WAVES, int AHEAD>
__global__ __launch_bounds__(WAVES * 64) void w4_stream_kernel(W4Args a) {
  typedef typename W4Type<T>::V V;
  __shared__ f32x4 red[WAVES][R * MB][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c16 = lane & 15, g = lane >> 4;
  const int nt0 = blockIdx.x * R, m0 = blockIdx.y * MB * 16, kts = (int)a.kt;
  const int last = (int)((a.N + 15) / 16) - 1;
  const T* xrow[MB];
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
    xrow[mb] = (const T*)a.x + (int64_t)min(m0 + mb * 16 + c16, (int)a.M - 1) * a.ldx;
  const W4Bits bits = w4_bits<T>();
  Stretch<GROUP, ZERO, R> f[AHEAD];
  u32x4 xv[AHEAD][4][MB];
  const auto fetch = [&](int i, int kt0) {
    const int kt = min(kt0, kts - 1);
    fetch_w<GROUP, ZERO, R>(f[i], a, nt0, last, kt, lane);
    // (inputs behind K meet scales of 0: the row's last ones do)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int k = min(kt * kTileK + j * 32 + g * 8, (int)a.K - 8);
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) xv[i][j][mb] = *(const u32x4*)(xrow[mb] + k);
    }
  };
  f32x4 acc[R][MB] = {};
#pragma unroll
  for (int i = 0; i < AHEAD - 1; ++i) fetch(i, wave + i * WAVES);
  for (int kt = wave; kt < kts;) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      fetch((i + AHEAD - 1) % AHEAD, kt + (AHEAD - 1) * WAVES);
      const auto x = [&](int j, int mb) { return __builtin_bit_cast(V, xv[i][j][mb]); };
      const auto sum = [&](int gi, int mb) {
        return sum_of<T, GROUP>(gi, [&](int j) { return x(j, mb); });
      };
      multiply<T, GROUP, ZERO, R, MB>(f[i], bits, x, sum, acc);
      kt += WAVES;
      if (kt >= kts) break;
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) red[wave][r * MB + mb][lane] = acc[r][mb];
  __syncthreads();
  for (int i = wave; i < R * MB; i += WAVES) {
    f32x4 y = red[0][i][lane];
#pragma unroll
    for (int v = 1; v < WAVES; ++v) y += red[v][i][lane];
    y *= W4Type<T>::back;
    const int m = m0 + i % MB * 16 + c16, n = (nt0 + i / MB) * 16 + g * 4;
    if (m >= a.M) continue;
    T* o = (T*)a.y + (int64_t)m * a.ldy + n;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < a.N) {
        if (a.bias) y[e] += ll_to_f32(((const T*)a.bias)[n + e]);
        o[e] = ll_from_f32<T>(y[e]);
      }
  }
}

// Rows of x at any address: one weight tile and 16 rows of x, element by element.
template <typename T, int GROUP, bool ZERO>
__global__ __launch_bounds__(kWavesW4 * 64) void w4_any_kernel(W4Args a) {
  typedef typename W4Type<T>::V V;
  __shared__ f32x4 red[kWavesW4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c16 = lane & 15, g = lane >> 4;
  const int nt = blockIdx.x, m0 = blockIdx.y * 16, kts = (int)a.kt;
  const T* xrow = (const T*)a.x + (int64_t)min(m0 + c16, (int)a.M - 1) * a.ldx;
  f32x4 acc[1][1] = {};
  for (int kt = wave; kt < kts; kt += kWavesW4) {
    Stretch<GROUP, ZERO, 1> f;
    fetch_w<GROUP, ZERO, 1>(f, a, nt, nt, kt, lane);
    u32x4 xv[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int k = min(kt * kTileK + j * 32 + g * 8, (int)a.K - 8);
      T* e = (T*)&xv[j];
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = xrow[k + i];
    }
    const auto x = [&](int j, int) { return __builtin_bit_cast(V, xv[j]); };
    const auto sum = [&](int gi, int) {
      return sum_of<T, GROUP>(gi, [&](int j) { return x(j, 0); });
    };
    multiply<T, GROUP, ZERO, 1, 1>(f, w4_bits<T>(), x, sum, acc);
  }
  red[wave][lane] = acc[0][0];
  __syncthreads();
  if (wave > 0) return;
  f32x4 y = red[0][lane];
#pragma unroll
  for (int v = 1; v < kWavesW4; ++v) y += red[v][lane];
  y *= W4Type<T>::back;
  const int m = m0 + c16;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int n = nt * 16 + g * 4 + e;
    if (m < a.M && n < a.N) {
      if (a.bias) y[e] += ll_to_f32(((const T*)a.bias)[n]);
      ((T*)a.y)[(int64_t)m * a.ldy + n] = ll_from_f32<T>(y[e]);
    }
  }
}

// a lane's value plus those of the 2, 4, 8 or 16 lanes that share its group of a
// row (16 lanes of 8 inputs each)
template <int LANES> __device__ __forceinline__ float sum_lanes(float v) {
  const auto add = [&](auto ctrl) {
    const int i = __builtin_bit_cast(int, v);
    v += __builtin_bit_cast(
        float, __builtin_amdgcn_mov_dpp(i, decltype(ctrl)::value, 0xf, 0xf, true));
  };
  add(std::integral_constant<int, 0xb1>());                          // lane ^ 1
  add(std::integral_constant<int, 0x4e>());                          // lane ^ 2
  if constexpr (LANES >= 8) add(std::integral_constant<int, 0x141>());   // mirrored in 8
  if constexpr (LANES >= 16) add(std::integral_constant<int, 0x140>());  // mirrored in 16
  return v;
}

// More rows of x: its tiles of 16 rows and 128 inputs go through LDS, where four
// waves of R weight tiles each read them, with each row's sum over every group;
// the next stretch is on its way while one is multiplied. A row's 16 pieces of 8
// inputs lie at piece ^ (row % 16), so that the 16 rows of an operand come from
// all banks. A workgroup may take its stretches in KG parts of four waves, added
// up through LDS; blockIdx.z is a split of them, and with more than one the sums
// go to `part` [split][M][N] and w4_finish_kernel adds them up. Nothing bounds it
// alone: conversion, scales and sums fill the VALU for 29% of the time, the accesses
// to x in LDS (8 cycles each) theirs for 38% and the MFMAs the matrix pipes for 11%,
// and they overlap only between workgroups (22,016 x 2048, 40 rows: 14.8 us; 17,920
// x 1536, 333 rows: 35%, 28%, 17%, 45 us, 411 TFLOP/s; 24,000 rows: 2.1 ms, 625).
template <typename T, int GROUP, bool ZERO, int R, int MB, int KG>
__global__ __launch_bounds__(kWavesW4 * 64 * KG, 2) void w4_tile_kernel(W4Args a) {
  typedef typename W4Type<T>::V V;
  constexpr int kGpt = kTileK / GROUP, kDeep = 2;
  constexpr bool kSum = W4Type<T>::summed(ZERO);
  const W4Bits bits = w4_bits<T>();
  constexpr int kRows = MB * 256;
  __shared__ u32x4 s_x[KG * 2 * kRows];
  __shared__ float s_sum[KG][2][kGpt][MB * 16];
  const int tid = threadIdx.x % (kWavesW4 * 64), lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int part = __builtin_amdgcn_readfirstlane(threadIdx.x / (kWavesW4 * 64));
  u32x4* xs = s_x + part * 2 * kRows;
  auto& xsum = s_sum[part];
  const int c16 = lane & 15, g = lane >> 4;
  const int nt0 = (blockIdx.x * kWavesW4 + wave) * R, m0 = blockIdx.y * MB * 16;
  const int last = (int)((a.N + 15) / 16) - 1;
  // this part's stretches; all parts take as many turns, since they share barriers
  const int turns = (min(a.span, (int)a.kt - (int)blockIdx.z * a.span) + KG - 1) / KG;
  const int k0 = blockIdx.z * a.span + part * turns;
  const int k1 = min(min(k0 + turns, (int)(blockIdx.z + 1) * a.span), (int)a.kt);
  const int kmax = min(k1, (int)a.kt) - 1;
  const auto within = [&](int kt) { return max(min(kt, kmax), 0); };
  // a thread's pieces of x: piece tid % 16 of rows tid / 16 + 16 i
  const int piece = tid & 15, row = tid >> 4;
  const T* xrow[MB];
#pragma unroll
  for (int i = 0; i < MB; ++i)
    xrow[i] = (const T*)a.x + (int64_t)min(m0 + i * 16 + row, (int)a.M - 1) * a.ldx;
  u32x4 xr[MB];
  const auto fetch_x = [&](int kt) {
    // (inputs behind K meet scales of 0: the row's last ones do)
    const int k = min(within(kt) * kTileK + piece * 8, (int)a.K - 8);
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) xr[mb] = *(const u32x4*)(xrow[mb] + k);
  };
  const auto put_x = [&](int buf) {
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
      const u32x4 v = xr[mb];
      xs[buf * kRows + (mb * 16 + row) * 16 + (piece ^ row)] = v;
      if constexpr (kSum) {
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) s = W4Type<T>::add2(v[e], s);
        s = sum_lanes<GROUP / 8>(s);
        if (piece % (GROUP / 8) == 0) xsum[buf][piece / (GROUP / 8)][mb * 16 + row] = s;
      }
    }
  };
  const auto wait = [] {  // for every wave's LDS accesses, not for loads from memory
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
  };
  f32x4 acc[R][MB] = {};
  Stretch<GROUP, ZERO, R> f[kDeep];
  fetch_x(k0);
#pragma unroll
  for (int i = 0; i < kDeep - 1; ++i)
    fetch_w<GROUP, ZERO, R>(f[i], a, nt0, last, within(k0 + i), lane);
  put_x(0);
  fetch_x(k0 + 1);
  wait();
  for (int kt = k0; kt < k0 + turns;) {
#pragma unroll
    for (int i = 0; i < kDeep; ++i) {
      const int cur = i & 1, nxt = cur ^ 1;
      fetch_w<GROUP, ZERO, R>(f[(i + kDeep - 1) % kDeep], a, nt0, last, within(kt + kDeep - 1),
                              lane);
      put_x(nxt);
      fetch_x(kt + 2);
      if (kt < k1)
        multiply<T, GROUP, ZERO, R, MB>(
            f[i], bits,
            [&](int j, int mb) {
              return __builtin_bit_cast(
                  V, xs[cur * kRows + (mb * 16 + c16) * 16 + ((j * 4 + g) ^ c16)]);
            },
            [&](int gi, int mb) { return xsum[cur][gi][mb * 16 + c16]; }, acc);
      wait();
      if (++kt >= k0 + turns) break;
    }
  }
  if constexpr (KG > 1) {  // the parts' sums, where x was (no one reads it any more)
    static_assert((KG - 1) * kWavesW4 * R * MB * 64 <= KG * 2 * kRows, "the sums fit");
    f32x4* red = (f32x4*)s_x;
    if (part > 0) {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
          red[(((part - 1) * kWavesW4 + wave) * R * MB + r * MB + mb) * 64 + lane] = acc[r][mb];
    }
    wait();
    if (part > 0) return;
#pragma unroll
    for (int q = 0; q < KG - 1; ++q)
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
          acc[r][mb] += red[((q * kWavesW4 + wave) * R * MB + r * MB + mb) * 64 + lane];
  }
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    const int m = m0 + mb * 16 + c16;
    if (m >= a.M) continue;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int n = (nt0 + r) * 16 + g * 4;
      f32x4 y = acc[r][mb];
      if (a.part) {
        float* o = a.part + ((int64_t)blockIdx.z * a.M + m) * a.N + n;
        if (a.N % 4 == 0 && n < a.N) {
          *(f32x4*)o = y;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n + e < a.N) o[e] = y[e];
        }
        continue;
      }
      y *= W4Type<T>::back;
      T* o = (T*)a.y + (int64_t)m * a.ldy + n;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < a.N) {
          if (a.bias) y[e] += ll_to_f32(((const T*)a.bias)[n + e]);
          o[e] = ll_from_f32<T>(y[e]);
        }
    }
  }
}

// y[m, n] = T(sum over the splits + bias), split after split
template <typename T>
__global__ __launch_bounds__(256) void w4_finish_kernel(W4Args a) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, quads = (a.N + 3) / 4;
  const int64_t m = i / quads, n = i % quads * 4;
  if (m >= a.M) return;
  const float* p = a.part + m * a.N + n;
  T* o = (T*)a.y + m * a.ldy + n;
  if (a.N % 4 == 0) {
    f32x4 y = *(const f32x4*)p;
#pragma unroll 4
    for (int s = 1; s < a.splits; ++s) y += *(const f32x4*)(p + s * a.M * a.N);
    y *= W4Type<T>::back;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (a.bias) y[e] += ll_to_f32(((const T*)a.bias)[n + e]);
      o[e] = ll_from_f32<T>(y[e]);
    }
  } else {
    for (int e = 0; e < 4 && n + e < a.N; ++e) {
      float y = p[e];
      for (int s = 1; s < a.splits; ++s) y += p[s * a.M * a.N + e];
      y *= W4Type<T>::back;
      if (a.bias) y += ll_to_f32(((const T*)a.bias)[n + e]);
      o[e] = ll_from_f32<T>(y);
    }
  }
}

// How a product of more than 16 rows runs. Two weight tiles to a wave halve the
// reads of x in LDS where there are workgroups enough for that (18,000 x 1536, 333
// rows: 47 us against 49 with one; 151,936 x 2048, 40 rows: 59 against 67); one
// tile with the stretches in two parts where there are not (22,016 x 2048, 40
// rows: 16.1 us, 17.9 in one part, 19.3 in four). What then leaves CUs idle is
// split over workgroups and added up by a second launch (2048 x 11,008, 40 rows:
// 12.5 us in eight splits, 13.9 in sixteen; 200 rows: 26.6 in four, 28.5 in two).
struct PlanW4 {
  int mb, r;         // tiles of x per workgroup, weight tiles per wave
  int splits, span;  // of the stretches
  int64_t bytes;     // workspace
};

constexpr int kTwoTiles = 4096;  // weight tiles times blocks of x from which on a wave takes two

PlanW4 plan_w4(int64_t M, int64_t N, int64_t K) {
  PlanW4 p;
  const int64_t nt = (N + 15) / 16, kt = (K + kTileK - 1) / kTileK;
  p.mb = M <= 32 ? 2 : M <= 48 ? 3 : 4;
  const int64_t blocks = (M + p.mb * 16 - 1) / (p.mb * 16);
  p.r = nt * blocks >= kTwoTiles ? 2 : 1;
  const int64_t wgs = (nt + kWavesW4 * p.r - 1) / (kWavesW4 * p.r) * blocks;
  const int64_t s = std::max<int64_t>(1, std::min<int64_t>((M > 64 ? 512 : 256) / wgs, kt / 4));
  p.span = (int)((kt + s - 1) / s);
  p.splits = (int)((kt + p.span - 1) / p.span);
  p.bytes = M > 16 && p.splits > 1 ? p.splits * M * N * 4 : 0;
  return p;
}

template <typename T, int GROUP, bool ZERO, int R, int MB, int WAVES, int AHEAD>
int launch_stream(const W4Args& a, hipStream_t stream) {
  const dim3 grid((unsigned)(((a.N + 15) / 16 + R - 1) / R),
                  (unsigned)((a.M + MB * 16 - 1) / (MB * 16)));
  hipLaunchKernelGGL((w4_stream_kernel<T, GROUP, ZERO, R, MB, WAVES, AHEAD>), grid,
                     dim3(WAVES * 64), 0, stream, a);
  LL_RETURN_LAUNCH();
}

template <typename T, int GROUP, bool ZERO, int R, int MB, int KG>
int launch_tiles(W4Args a, const PlanW4& p, hipStream_t stream) {
  const int64_t nt = (a.N + 15) / 16;
  const dim3 grid((unsigned)((nt + kWavesW4 * R - 1) / (kWavesW4 * R)),
                  (unsigned)((a.M + MB * 16 - 1) / (MB * 16)), (unsigned)p.splits);
  a.span = p.span;
  a.splits = p.splits;
  hipLaunchKernelGGL((w4_tile_kernel<T, GROUP, ZERO, R, MB, KG>), grid, dim3(kWavesW4 * 64 * KG), 0,
                     stream, a);
  if (p.splits > 1) {
    const int64_t items = a.M * ((a.N + 3) / 4);
    hipLaunchKernelGGL((w4_finish_kernel<T>), dim3((unsigned)((items + 255) / 256)), dim3(256), 0,
                       stream, a);
  }
  LL_RETURN_LAUNCH();
}

template <typename T, int GROUP, bool ZERO>
int launch_w4(const W4Args& a, bool vec, const PlanW4& p, hipStream_t stream) {
  if (!vec) {
    const dim3 grid((unsigned)((a.N + 15) / 16), (unsigned)((a.M + 15) / 16));
    hipLaunchKernelGGL((w4_any_kernel<T, GROUP, ZERO>), grid, dim3(kWavesW4 * 64), 0, stream, a);
    LL_RETURN_LAUNCH();
  }
  if (a.M <= 16) {
    // Few weight tiles: a workgroup of 16 waves for each (2048 x 11,008, one row:
    // 6.9 us, 8.1 with 8 waves, 14 with 4). More: two or four tiles share x, of
    // which every workgroup reads all (22,016 x 2048, 8 rows: 8.9 us with two
    // tiles, 11.8 with one; 151,936 x 1536, 5 rows: 37 with four and the next
    // stretch's loads ahead, 42 without; 151,936 x 2048, one row, which leaves
    // registers for more waves: 34 without, 39 with).
    const int64_t nt = (a.N + 15) / 16;
    if (nt <= 512) return launch_stream<T, GROUP, ZERO, 1, 1, 16, 1>(a, stream);
    if (nt <= 2048) return launch_stream<T, GROUP, ZERO, 2, 1, 4, 1>(a, stream);
    return launch_stream<T, GROUP, ZERO, 4, 1, 4, GROUP == 128 && !ZERO ? 1 : 2>(a, stream);
  }
  if (p.r == 1) {
    if (p.mb == 2) return launch_tiles<T, GROUP, ZERO, 1, 2, 2>(a, p, stream);
    if (p.mb == 3) return launch_tiles<T, GROUP, ZERO, 1, 3, 2>(a, p, stream);
    return launch_tiles<T, GROUP, ZERO, 1, 4, 2>(a, p, stream);
  }
  if (p.mb == 2) return launch_tiles<T, GROUP, ZERO, 2, 2, 1>(a, p, stream);
  if (p.mb == 3) return launch_tiles<T, GROUP, ZERO, 2, 3, 1>(a, p, stream);
  return launch_tiles<T, GROUP, ZERO, 2, 4, 1>(a, p, stream);
}

bool w4_shape(int64_t N, int64_t K, int64_t group) {
  return N > 0 && K > 0 && (group == 32 || group == 64 || group == 128) && K % group == 0 &&
         N <= INT32_MAX / 16 && K <= INT32_MAX / 16;
}

}  // namespace

extern "C" int64_t ll_w4_packed_bytes(int64_t N, int64_t K, int64_t group, int has_zero) {
  return w4_shape(N, K, group) ? layout_w4(N, K, group, has_zero != 0).total : 0;
}

extern "C" int ll_w4_pack(const uint8_t* codes, int64_t ldc, const void* scale, int64_t ld_scale,
                          const uint8_t* zero, int64_t ld_zero, int64_t N, int64_t K, int64_t group,
                          void* packed, int64_t packed_bytes, hipStream_t stream) {
  const char* fn = "ll_w4_pack";
  LL_CHECK_ARG(codes && scale && packed, "%s: null pointer", fn);
  LL_CHECK_ARG(w4_shape(N, K, group), "%s: N=%lld K=%lld group=%lld (K a multiple of a group of "
               "32, 64 or 128)", fn, (long long)N, (long long)K, (long long)group);
  const PackedW4 p = layout_w4(N, K, group, zero != nullptr);
  LL_CHECK_ARG(packed_bytes >= p.total && (uintptr_t)packed % 16 == 0,
               "%s: packed holds %lld bytes, needs %lld, 16 B aligned", fn, (long long)packed_bytes,
               (long long)p.total);
  const int64_t items = p.scale / 4;  // (no fewer than the scales')
  LL_CHECK_ARG((items + 255) / 256 <= INT32_MAX / 256, "%s: N=%lld K=%lld is too large", fn,
               (long long)N, (long long)K);
  hipLaunchKernelGGL(w4_pack_kernel, dim3((unsigned)((items + 255) / 256)), dim3(256), 0, stream,
                     codes, ldc, (const uint16_t*)scale, ld_scale, zero, ld_zero, N, K, (int)group,
                     (uint8_t*)packed, p);
  LL_RETURN_LAUNCH();
}

extern "C" int64_t ll_linear_w4_workspace_size(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || M > 1 << 19 || N <= 0 || N > INT32_MAX / 16 || K <= 0 || K > INT32_MAX / 16)
    return 0;
  return plan_w4(M, N, K).bytes;
}

extern "C" int ll_linear_w4(const void* x, int64_t ldx, const void* packed, int has_zero,
                            int64_t group, const void* bias, void* y, int64_t ldy, int64_t M,
                            int64_t N, int64_t K, int dtype, void* workspace,
                            int64_t workspace_bytes, hipStream_t stream) {
  const char* fn = "ll_linear_w4";
  if (M == 0) return LL_OK;
  LL_CHECK_ARG(x && packed && y, "%s: null pointer", fn);
  LL_CHECK_ARG(w4_shape(N, K, group), "%s: N=%lld K=%lld group=%lld (K a multiple of a group of "
               "32, 64 or 128)", fn, (long long)N, (long long)K, (long long)group);
  LL_CHECK_ARG(M > 0 && M <= 1 << 19, "%s: %lld rows (max 2^19)", fn, (long long)M);
  LL_CHECK_ARG(dtype == LL_BF16 || dtype == LL_F16, "%s: bf16 and fp16 only", fn);
  LL_CHECK_ARG((uintptr_t)packed % 16 == 0, "%s: the packed weight is not 16 B aligned", fn);
  LL_CHECK_ARG(ldx >= 0 && (ldy >= N || M == 1), "%s: row strides %lld, %lld", fn, (long long)ldx,
               (long long)ldy);
  const PackedW4 l = layout_w4(N, K, group, has_zero != 0);
  const PlanW4 p = plan_w4(M, N, K);
  LL_CHECK_ARG((M + 15) / 16 <= 65535 && (N + 15) / 16 <= (1 << 22) &&
                   (p.bytes == 0 || M * ((N + 3) / 4) < (int64_t)1 << 31),
               "%s: %lld rows of %lld outputs are more than a launch holds", fn, (long long)M,
               (long long)N);
  W4Args a = {};
  a.x = x; a.ldx = ldx;
  a.codes = (const uint8_t*)packed + l.codes;
  a.scale = (const uint16_t*)((const uint8_t*)packed + l.scale);
  a.zero = has_zero ? (const uint8_t*)packed + l.zero : nullptr;
  a.bias = bias; a.y = y; a.ldy = ldy;
  a.M = M; a.N = N; a.K = K; a.kt = (K + kTileK - 1) / kTileK;
  const bool vec = (uintptr_t)x % 16 == 0 && ldx % 8 == 0;
  std::unique_lock<std::mutex> lock;
  if (vec && p.bytes > 0) {
    LL_CHECK_ARG(workspace && workspace_bytes >= p.bytes && (uintptr_t)workspace % 16 == 0,
                 "%s: the workspace needs %lld bytes, 16 B aligned, got %lld", fn,
                 (long long)p.bytes, (long long)workspace_bytes);
    a.part = (float*)workspace;
    // no other thread's call on this workspace between the two launches
    lock = std::unique_lock<std::mutex>(ll_workspace_mutex(workspace));
  }
  const auto go = [&](auto t) -> int {
    typedef decltype(t) T;
    const auto with = [&](auto z) -> int {
      constexpr bool ZERO = decltype(z)::value;
      if (group == 32) return launch_w4<T, 32, ZERO>(a, vec, p, stream);
      if (group == 64) return launch_w4<T, 64, ZERO>(a, vec, p, stream);
      return launch_w4<T, 128, ZERO>(a, vec, p, stream);
    };
    return has_zero ? with(std::true_type()) : with(std::false_type());
  };
  return dtype == LL_BF16 ? go(__bf16()) : go(_Float16());
}
