// Products with weights of 4 bits and a scale for each group of inputs (gfx950):
//   y[m, n] = sum_k x[m, k] (c[n, k] - z[n, k / group]) s[n, k / group] + bias[n]
// with c in 0 .. 15, z the zero point (8 where a weight has none) and s in x's
// type.
//
// A weight is laid out once (ll_w4_pack) as the operand of a 16x16x32 MFMA: a
// tile is 16 rows of 128 inputs, 1 KB, in which lane l holds 16 bytes: row
// l % 16, and in dword j the inputs 32 j + 8 (l / 16) + 0 .. 7. Nibble i of a
// dword is input 2 i and nibble i + 4 input 2 i + 1, so that a shift, an `and`
// and an `or` make two 16-bit floats at once: 0x4300 | c is 128 + c in bf16,
// 0x6400 | c is 1024 + c in fp16. For bf16 the 128 stays in and leaves with the
// zero point: a group's sum is
//   sum x (128 + c) - (128 + z) sum x,
// the second sum taken by the same instruction from a tile of ones (it loses
// 128 / 15 times fp32's rounding, 2^-20 of the result's terms). In fp16 1024 is
// subtracted, which is exact.
#include <algorithm>

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
__global__ __launch_bounds__(256) void w4_pack_kernel(const uint8_t* __restrict__ codes, int64_t ldc,
                                                      const uint16_t* __restrict__ scale, int64_t lds,
                                                      const uint8_t* __restrict__ zero, int64_t ldz,
                                                      int64_t N, int64_t K, int group, uint8_t* out,
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
};

template <typename T> struct W4Type;
template <> struct W4Type<__bf16> {
  typedef bf16x8 V;
  static constexpr float off = 128.f;
  static constexpr uint32_t one = 0x3f803f80u;
  static __device__ __forceinline__ uint32_t pair(uint32_t w) {
    return (w & 0x000f000fu) | 0x43004300u;
  }
  static __device__ __forceinline__ f32x4 mfma(V a, V b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct W4Type<_Float16> {
  typedef f16x8 V;
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  static constexpr float off = 0.f;
  static constexpr uint32_t one = 0x3c003c00u;
  static __device__ __forceinline__ uint32_t pair(uint32_t w) {
    const h2 b = {(_Float16)1024.f, (_Float16)1024.f};
    return __builtin_bit_cast(uint32_t,
                              __builtin_bit_cast(h2, (w & 0x000f000fu) | 0x64006400u) - b);
  }
  static __device__ __forceinline__ f32x4 mfma(V a, V b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

// R tiles of 16 weight rows by MB tiles of 16 rows of x per workgroup; its waves
// take every fourth stretch of 128 inputs and add up through LDS.
template <typename T, int GROUP, int R, int MB, bool VEC>
__global__ __launch_bounds__(kWavesW4 * 64) void w4_kernel(W4Args a) {
  typedef W4Type<T> W;
  typedef typename W::V V;
  __shared__ f32x4 red[kWavesW4 - 1][R * MB][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c16 = lane & 15, g = lane >> 4;
  constexpr int kGpt = kTileK / GROUP, kCpg = GROUP / 32;  // groups per tile, chunks per group
  const int64_t nt0 = (int64_t)blockIdx.x * R, m0 = (int64_t)blockIdx.y * MB * 16;
  const int64_t ntiles = (a.N + 15) / 16;
  f32x4 acc[R][MB] = {};
  const T* xrow[MB];
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
    xrow[mb] = (const T*)a.x + std::min<int64_t>(m0 + mb * 16 + c16, a.M - 1) * a.ldx;
  V ones;
  {
    u32x4 o = {W::one, W::one, W::one, W::one};
    ones = __builtin_bit_cast(V, o);
  }
  for (int64_t kt = wave; kt < a.kt; kt += kWavesW4) {
    u32x4 w[R];
#pragma unroll
    for (int r = 0; r < R; ++r)
      w[r] = ((const u32x4*)a.codes)[(std::min(nt0 + r, ntiles - 1) * a.kt + kt) * 64 + lane];
    u32x4 xv[4][MB];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        const int64_t k = kt * kTileK + j * 32 + g * 8;
        xv[j][mb] = (u32x4){0, 0, 0, 0};
        if (k < a.K) {
          if constexpr (VEC) {
            xv[j][mb] = *(const u32x4*)(xrow[mb] + k);
          } else {
            T* e = (T*)&xv[j][mb];
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = xrow[mb][k + i];
          }
        }
      }
#pragma unroll
    for (int gi = 0; gi < kGpt; ++gi) {
      f32x4 part[R][MB] = {}, sum[MB] = {};
#pragma unroll
      for (int jj = 0; jj < kCpg; ++jj) {
        const int j = gi * kCpg + jj;
        V xf[MB];
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
          xf[mb] = __builtin_bit_cast(V, xv[j][mb]);
          sum[mb] = W::mfma(ones, xf[mb], sum[mb]);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
          u32x4 p;
#pragma unroll
          for (int i = 0; i < 4; ++i) p[i] = W::pair(w[r][j] >> (4 * i));
          const V wf = __builtin_bit_cast(V, p);
#pragma unroll
          for (int mb = 0; mb < MB; ++mb) part[r][mb] = W::mfma(wf, xf[mb], part[r][mb]);
        }
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int64_t at =
            ((std::min(nt0 + r, ntiles - 1) * a.kt + kt) * kGpt + gi) * 16 + g * 4;
        const uint2 sv = *(const uint2*)(a.scale + at);
        const uint32_t zv = a.zero ? *(const uint32_t*)(a.zero + at) : 0x08080808u;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint16_t bits = (uint16_t)((e < 2 ? sv.x : sv.y) >> (16 * (e & 1)));
          const float s = ll_to_f32(__builtin_bit_cast(T, bits));
          const float z = W::off + (float)((zv >> (8 * e)) & 255u);
#pragma unroll
          for (int mb = 0; mb < MB; ++mb)
            acc[r][mb][e] =
                __builtin_fmaf(s, __builtin_fmaf(-z, sum[mb][e], part[r][mb][e]), acc[r][mb][e]);
        }
      }
    }
  }
  if (wave > 0) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) red[wave - 1][r * MB + mb][lane] = acc[r][mb];
  }
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
      f32x4 y = acc[r][mb];
#pragma unroll
      for (int w = 0; w < kWavesW4 - 1; ++w) y += red[w][r * MB + mb][lane];
      const int64_t m = m0 + mb * 16 + c16;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t n = (nt0 + r) * 16 + g * 4 + e;
        if (m < a.M && n < a.N) {
          float v = y[e];
          if (a.bias) v += ll_to_f32(((const T*)a.bias)[n]);
          ((T*)a.y)[m * a.ldy + n] = ll_from_f32<T>(v);
        }
      }
    }
}

template <typename T, int GROUP>
int launch_w4(const W4Args& a, bool vec, hipStream_t stream) {
  const int64_t nt = (a.N + 15) / 16;
  if (!vec || a.M <= 16) {
    const dim3 grid((unsigned)nt, (unsigned)((a.M + 15) / 16));
    if (vec) hipLaunchKernelGGL((w4_kernel<T, GROUP, 1, 1, true>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((w4_kernel<T, GROUP, 1, 1, false>), grid, dim3(256), 0, stream, a);
  } else {
    const dim3 grid((unsigned)((nt + 1) / 2), (unsigned)((a.M + 63) / 64));
    hipLaunchKernelGGL((w4_kernel<T, GROUP, 2, 4, true>), grid, dim3(256), 0, stream, a);
  }
  LL_RETURN_LAUNCH();
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

extern "C" int ll_linear_w4(const void* x, int64_t ldx, const void* packed, int has_zero,
                            int64_t group, const void* bias, void* y, int64_t ldy, int64_t M,
                            int64_t N, int64_t K, int dtype, hipStream_t stream) {
  const char* fn = "ll_linear_w4";
  if (M == 0) return LL_OK;
  LL_CHECK_ARG(x && packed && y, "%s: null pointer", fn);
  LL_CHECK_ARG(w4_shape(N, K, group), "%s: N=%lld K=%lld group=%lld (K a multiple of a group of "
               "32, 64 or 128)", fn, (long long)N, (long long)K, (long long)group);
  LL_CHECK_ARG(M > 0 && M <= 1 << 19, "%s: %lld rows (max 2^19)", fn, (long long)M);
  LL_CHECK_ARG(dtype == LL_BF16 || dtype == LL_F16, "%s: bf16 and fp16 only", fn);
  LL_CHECK_ARG(ldx >= 0 && (ldy >= N || M == 1), "%s: row strides %lld, %lld", fn, (long long)ldx,
               (long long)ldy);
  const PackedW4 p = layout_w4(N, K, group, has_zero != 0);
  W4Args a;
  a.x = x; a.ldx = ldx;
  a.codes = (const uint8_t*)packed + p.codes;
  a.scale = (const uint16_t*)((const uint8_t*)packed + p.scale);
  a.zero = has_zero ? (const uint8_t*)packed + p.zero : nullptr;
  a.bias = bias; a.y = y; a.ldy = ldy;
  a.M = M; a.N = N; a.K = K; a.kt = (K + kTileK - 1) / kTileK;
  const bool vec = (uintptr_t)x % 16 == 0 && ldx % 8 == 0;
  const auto go = [&](auto t) -> int {
    typedef decltype(t) T;
    if (group == 32) return launch_w4<T, 32>(a, vec, stream);
    if (group == 64) return launch_w4<T, 64>(a, vec, stream);
    return launch_w4<T, 128>(a, vec, stream);
  };
  return dtype == LL_BF16 ? go(__bf16()) : go(_Float16());
}
