// Rotary positions from the frequencies, alone and behind per-head norms, for
// gfx950.
//
// A head's first R = rotary_dim elements are R / 2 pairs; pair i of a token at
// position p turns by the angle p * inv_freq[i] and is scaled by `factor`:
//   y0 = x0 c - x1 s,  y1 = x0 s + x1 c,  c, s = factor * (cos, sin)(p f_i).
// Pair i is (i, i + R/2) (half layout) or (2i, 2i + 1) (interleaved); the
// elements behind R stay as they are. With norms, x is first
// x / sqrt(mean(x^2) + eps) * gamma over the whole head. Everything is fp32
// with one rounding at the store.
//
// No cos/sin table: a table over the context length is rounded where it is
// stored and ends where it ends, while the angle of a far position needs more
// than fp32 (p f_i has 24 + 31 bits). The angle is taken in turns in fp64,
// p * (f_i / 2 pi), whose whole part is dropped exactly; what is left of it
// fits fp32. For frequencies up to 1 and any int32 position the angle is off by
// less than 2^-23 of a turn: of at most 2^28.35 turns, the constant's and the
// frequency's rounding 1.56 x 2^-53 each, 0.99 x 2^-24; the product's 2^-25; and
// 2^-26 for the fraction in fp32. (The largest seen is 1.35 x 2^-24.)
#include <algorithm>

#include "ll_common.h"

namespace {

// Heads of one token: `na` heads at `a`, then `nb` at `b`. The first `nrot`
// of all are rotated (and normalised, where gammas are given: ga for the heads
// at a, gb for those at b); the others are copied.
struct RotArgs {
  const void* a; int64_t a_st, a_sh; void* ao; int64_t ao_st, ao_sh;
  const void* b; int64_t b_st, b_sh; void* bo; int64_t bo_st, bo_sh;
  int na, nb, nrot, D, R;
  const void* ga; const void* gb;
  float eps, factor;
  const void* pos; int pos64;
  const float* inv_freq;
  // rows of `bo` (cache slots); null: row = token. A slot outside [0, nslots)
  // is not stored to (a padded token)
  const int32_t* slots; int64_t nslots;
  int64_t ntok;
};

__device__ __forceinline__ void rot_angle(int64_t pos, float inv_freq, float factor, float& c,
                                          float& s) {
  const double turns = (double)pos * ((double)inv_freq * 0.15915494309189535);
  sincospif(2.0f * (float)(turns - __builtin_rint(turns)), &s, &c);
  c *= factor;
  s *= factor;
}

// Any head_dim, rotary_dim and alignment, for the shapes and strides that the
// 16-byte form below does not take (24,000 tokens of 28/4 heads of 128: 247 us
// against its 68): one wave per (token, head), a lane per pair.
template <typename T, bool INTER>
__global__ __launch_bounds__(64) void rotary_kernel(RotArgs a) {
  const int64_t t = blockIdx.x;
  const int h = blockIdx.y, lane = threadIdx.x;
  const bool isa = h < a.na;
  const int hb = h - a.na;
  const T* x = isa ? (const T*)a.a + t * a.a_st + (int64_t)h * a.a_sh
                   : (const T*)a.b + t * a.b_st + (int64_t)hb * a.b_sh;
  int64_t row = t;
  bool store = true;
  if (!isa && a.slots != nullptr) {
    row = a.slots[t];
    store = row >= 0 && row < a.nslots;
  }
  T* y = isa ? (T*)a.ao + row * a.ao_st + (int64_t)h * a.ao_sh
             : (T*)a.bo + row * a.bo_st + (int64_t)hb * a.bo_sh;
  if (!store) return;
  const bool rot = h < a.nrot;
  const T* g = rot ? (const T*)(isa ? a.ga : a.gb) : nullptr;
  float r = 1.f;
  if (g != nullptr) {
    float ss = 0.f;
    for (int d = lane; d < a.D; d += 64) {
      const float v = ll_to_f32(x[d]);
      ss += v * v;
    }
    r = 1.0f / sqrtf(ll_wave_sum(ss) / (float)a.D + a.eps);
  }
  auto value = [&](int d) {
    const float v = ll_to_f32(x[d]);
    return g != nullptr ? v * r * ll_to_f32(g[d]) : v;
  };
  const int half = rot ? a.R / 2 : 0;
  const int64_t p = half > 0 ? ll_load_idx(a.pos, t, a.pos64) : 0;  // (null where R is 0)
  for (int i = lane; i < half; i += 64) {
    const int d0 = INTER ? 2 * i : i, d1 = INTER ? 2 * i + 1 : i + half;
    float c, s;
    rot_angle(p, a.inv_freq[i], a.factor, c, s);
    const float u = value(d0), w = value(d1);
    y[d0] = ll_from_f32<T>(u * c - w * s);
    y[d1] = ll_from_f32<T>(u * s + w * c);
  }
  for (int d = 2 * half + lane; d < a.D; d += 64)
    y[d] = g != nullptr ? ll_from_f32<T>(value(d)) : x[d];
}

// 16-byte form: a group of LPH lanes per head, 16 elements per lane (one "unit",
// two chunks of 8 that hold its 8 pairs), D / 16 <= LPH units.
// HBM-bound (a token's heads are read and written once), so what counts is
// that nothing else shows: the angles, 60-odd instructions each in fp64 and
// sincospif, are computed once per token and pair into LDS and shared by its
// heads, while the first heads' loads are in flight; a workgroup takes TB
// tokens so that there are enough heads to cover that. The norm's sum stays in
// the LPH lanes of its head; the gammas are read for every head again (from the
// L1; in registers they cost a fifth of the waves: 4000 tokens of 16/2 heads of
// 128 10.4 -> 13.0 us).
template <typename T> struct alignas(16) Chunk { T v[8]; };

// Stores go out non-temporally: nothing of this call reads them, and the lines
// they would leave in the L2 have to be written back at its end anyway (24,000
// tokens of 28/4 heads 81 -> 68 us, 2000 of 32/8 heads of 64 10.6 -> 7.9;
// non-temporal loads gained 3-6% at 24,000 tokens and lost up to 30% at 4000,
// whose rows the projection has just left on the memory side's cache).
template <typename T> __device__ __forceinline__ void store_chunk(T* p, const Chunk<T>& c) {
  constexpr int N = sizeof(c) / 16;
  struct Words { u32x4 w[N]; };
  const Words v = __builtin_bit_cast(Words, c);
#pragma unroll
  for (int i = 0; i < N; ++i) __builtin_nontemporal_store(v.w[i], (u32x4*)p + i);
}

constexpr int kRotThreads = 256;

// What the 16-byte form's addresses are made of. A workgroup's tokens and their
// heads are small numbers and strides are below 2^24 units of 16 bytes, so that
// an address is two 24-bit multiplies and a shifted add to a scalar base: the
// same in 64 bits, at a quarter of the vector unit's rate, cost as much as the
// rotation (16/2 heads of 128 with norms, 2000 tokens 7.4 -> 5.6 us, 24,000 55.6
// -> 51.7; those now 47.1, 5.2 TB/s).
struct RotVec {
  uint32_t a_st, a_sh, ao_st, ao_sh, b_st, b_sh, bo_st, bo_sh;
  uint32_t row_st;  // of a cache slot, to 2^32
  uint32_t nslots;
  int tb;                                         // tokens per workgroup
  int heads_mul, heads_shift, half_mul, half_shift;  // division by heads and pairs
  float inv_d;
};

template <typename T, int LPH, bool INTER, bool NORM>
__global__ __launch_bounds__(kRotThreads) void rotary_vec_kernel(RotArgs a, RotVec v) {
  extern __shared__ __attribute__((aligned(16))) float sh[];  // [TB][R/2] cos, then sin
  typedef Chunk<T> C;
  constexpr int kGroups = kRotThreads / LPH;
  const int half = a.R / 2, heads = a.na + a.nb;
  const int64_t t0 = (int64_t)blockIdx.x * v.tb;
  const int nt = (int)min((int64_t)v.tb, a.ntok - t0);
  const int items = nt * heads;
  const int u = threadIdx.x % LPH;
  const int units = a.D / 16, runits = a.R / 16;
  const bool live = u < units;  // (the others read the head's first chunk and store nothing)
  // The chunks of unit u, such that neighbouring lanes read neighbouring
  // chunks. Half layout: u and u + R / 16 hold pairs 8u .. 8u + 7, and the
  // units behind R share its chunks out likewise; interleaved: u and u + D / 16,
  // chunk c with pairs 4c .. 4c + 3.
  const bool rot0 = INTER ? u < 2 * runits : u < runits;
  const bool rot1 = INTER ? u + units < 2 * runits : rot0;
  const int c0 = !live ? 0 : INTER || rot0 ? u : runits + u;
  const int c1 = !live ? 0 : INTER ? u + units : rot0 ? u + runits : units + u;
  const int p0 = INTER ? 4 * u : 8 * u, p1 = INTER ? 4 * (u + units) : 8 * u + 4;
  const char* const xa = (const char*)a.a + (uint64_t)t0 * v.a_st * 16;
  const char* const xb = (const char*)a.b + (uint64_t)t0 * v.b_st * 16;
  char* const ya = (char*)a.ao + (uint64_t)t0 * v.ao_st * 16;
  char* const yb = (char*)a.bo + (uint64_t)t0 * v.bo_st * 16;

  struct Item {
    C x0, x1;
    T* y;       // null: not stored
    int tok, kind;  // kind: 0 copied, 1 rotated head of a, 2 of b
  };
  auto load = [&](int i) {
    Item it;
    // i / heads by multiplication (exact for the items of a workgroup)
    it.tok = (int)(__umul24(i, v.heads_mul) >> v.heads_shift);
    const int h = i - __umul24(it.tok, heads);
    const bool isa = h < a.na;
    const int hb = isa ? h : h - a.na;
    const uint32_t x_at = __umul24(it.tok, isa ? v.a_st : v.b_st) + __umul24(hb, isa ? v.a_sh : v.b_sh);
    const uint32_t y_at =
        __umul24(it.tok, isa ? v.ao_st : v.bo_st) + __umul24(hb, isa ? v.ao_sh : v.bo_sh);
    const T* x = (const T*)((isa ? xa : xb) + 16 * (uint64_t)x_at);
    char* y = (isa ? ya : yb) + 16 * (uint64_t)y_at;
    if (!isa && a.slots != nullptr) {
      const uint32_t row = (uint32_t)a.slots[t0 + it.tok];
      y = row < v.nslots ? y + 16 * ((uint64_t)row * v.row_st) : nullptr;
    }
    it.y = live ? (T*)y : nullptr;
    it.kind = h < a.nrot ? (isa ? 1 : 2) : 0;
    it.x0 = *(const C*)(x + 8 * c0);
    it.x1 = *(const C*)(x + 8 * c1);
    return it;
  };
  int i = threadIdx.x / LPH;
  Item cur;
  if (i < items) cur = load(i);
  float* s_cos = sh;
  float* s_sin = sh + v.tb * half;
  for (int j = threadIdx.x; j < nt * half; j += kRotThreads) {
    const int tok = (int)(__umul24(j, v.half_mul) >> v.half_shift);
    float c, s;
    rot_angle(ll_load_idx(a.pos, t0 + tok, a.pos64), a.inv_freq[j - __umul24(tok, half)], a.factor,
              c, s);
    s_cos[j] = c;
    s_sin[j] = s;
  }
  __syncthreads();
  // (the groups of a wave leave the loop together or one pass apart; a norm's
  // shuffles stay inside a group)
  for (; i < items; i += kGroups) {
    Item next;
    const bool more = i + kGroups < items;
    if (more) next = load(i + kGroups);
    if (cur.kind == 0) {
      if (cur.y != nullptr) {
        store_chunk(cur.y + 8 * c0, cur.x0);
        store_chunk(cur.y + 8 * c1, cur.x1);
      }
    } else {
      float x[16];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = ll_to_f32(cur.x0.v[e]);
        x[8 + e] = ll_to_f32(cur.x1.v[e]);
      }
      if constexpr (NORM) {
        const bool of_a = cur.kind == 1;
        if ((of_a ? a.ga : a.gb) != nullptr) {
          const T* g = (const T*)(of_a ? a.ga : a.gb);
          const C g0 = *(const C*)(g + 8 * c0), g1 = *(const C*)(g + 8 * c1);
          float ss = 0.f;
#pragma unroll
          for (int e = 0; e < 16; ++e) ss += x[e] * x[e];
          if (!live) ss = 0.f;
#pragma unroll
          for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);
          const float var = ss * v.inv_d + a.eps;
          // (v_rsq_f32, 1 ulp, takes normal numbers)
          const float r = var >= 1e-37f ? __builtin_amdgcn_rsqf(var) : 1.0f / sqrtf(var);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            x[e] = x[e] * r * ll_to_f32(g0.v[e]);
            x[8 + e] = x[8 + e] * r * ll_to_f32(g1.v[e]);
          }
        }
      }
      if (cur.y != nullptr) {
        float y[16];
        const int at = cur.tok * half;
        if constexpr (INTER) {
          auto turn = [&](const float* z, float* w, bool rot, int p) {
            if (rot) {
              const f32x4 c = *(const f32x4*)(s_cos + at + p), s = *(const f32x4*)(s_sin + at + p);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                w[2 * e] = z[2 * e] * c[e] - z[2 * e + 1] * s[e];
                w[2 * e + 1] = z[2 * e] * s[e] + z[2 * e + 1] * c[e];
              }
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e) w[e] = z[e];
            }
          };
          turn(x, y, rot0, p0);
          turn(x + 8, y + 8, rot1, p1);
        } else if (rot0) {
          const f32x4 c4[2] = {*(const f32x4*)(s_cos + at + p0), *(const f32x4*)(s_cos + at + p1)};
          const f32x4 s4[2] = {*(const f32x4*)(s_sin + at + p0), *(const f32x4*)(s_sin + at + p1)};
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float c = c4[e >> 2][e & 3], s = s4[e >> 2][e & 3];
            y[e] = x[e] * c - x[8 + e] * s;
            y[8 + e] = x[e] * s + x[8 + e] * c;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) y[e] = x[e];
        }
        C o0, o1;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          o0.v[e] = ll_from_f32<T>(y[e]);
          o1.v[e] = ll_from_f32<T>(y[8 + e]);
        }
        store_chunk(cur.y + 8 * c0, o0);
        store_chunk(cur.y + 8 * c1, o1);
      }
    }
    if (more) cur = next;
  }
}

template <typename T, int LPH>
void launch_rotary_vec(const RotArgs& a, int interleaved, hipStream_t stream) {
  const int heads = a.na + a.nb;
  // tokens per workgroup: one until the grid fills the CUs eight times over,
  // then as many as fill its lanes twice, at most 8 (1, 2, 4, 8 of them at 24,000
  // tokens: 16/2 heads of 128 46.8, 41.0, 41.2, 42.7 us, with norms 52.9, 47.2,
  // 47.7, 51.8; 12/2 35.9, 32.3, 29.2, 33.2; 8/2 heads of 64 22.1, 15.6, 14.2,
  // 12.8); where one token's heads do, two while what the call moves stays in the
  // memory side's 256 MB (28/4 heads of 128, 8000 tokens: 1 23.3, 2 21.3), else
  // one (24,000: 67.8, 70.5; 64/8, 8000: 53.8, 57.0). LDS 32 KB at most
  const int lanes = heads * LPH;
  int tb = lanes >= kRotThreads
               ? (2 * a.ntok * heads * a.D * (int64_t)sizeof(T) > (int64_t)256 << 20 ? 1 : 2)
               : 2 * kRotThreads / lanes >= 8 ? 8 : 2 * kRotThreads / lanes >= 4 ? 4 : 2;
  tb = (int)std::min<int64_t>(tb, std::max<int64_t>(1, a.ntok / 2048));
  while (tb > 1 && tb * a.R * 4 > 32768) tb /= 2;
  // (a grid has fewer than 2^32 threads: 2^24 tokens, the most, go two by two)
  if (a.ntok >= ((int64_t)1 << 32) / kRotThreads) tb = std::max(tb, 2);
  // i / n = (i * mul) >> shift for i < tb * n: with mul = ceil(2^shift / n), exact
  // while i * n < 2^shift; i and mul have 24 bits and their product 32
  auto divide = [tb](int n, int& mul, int& shift) {
    shift = 0;
    while (((int64_t)1 << shift) < (int64_t)tb * n * n) ++shift;
    mul = n ? (int)((((int64_t)1 << shift) + n - 1) / n) : 0;
  };
  const int64_t es = sizeof(T);
  auto units = [es](int64_t stride) { return (uint32_t)(stride * es / 16); };
  RotVec v = {};
  v.a_st = units(a.a_st); v.a_sh = units(a.a_sh); v.ao_st = units(a.ao_st); v.ao_sh = units(a.ao_sh);
  v.b_st = units(a.b_st); v.b_sh = units(a.b_sh); v.bo_sh = units(a.bo_sh);
  if (a.slots != nullptr) v.row_st = units(a.bo_st);
  else v.bo_st = units(a.bo_st);
  v.nslots = (uint32_t)std::min<int64_t>(a.nslots, (int64_t)1 << 31);  // (a negative slot is above it)
  v.tb = tb;
  divide(heads, v.heads_mul, v.heads_shift);
  divide(a.R / 2, v.half_mul, v.half_shift);
  v.inv_d = 1.0f / (float)a.D;
  const unsigned grid = (unsigned)((a.ntok + tb - 1) / tb);
  const size_t lds = (size_t)tb * a.R * 4;
  const bool norm = a.ga != nullptr || a.gb != nullptr;
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(kRotThreads), lds, stream, a, v);
  };
  if (norm) {
    if (interleaved) go(rotary_vec_kernel<T, LPH, true, true>);
    else go(rotary_vec_kernel<T, LPH, false, true>);
  } else {
    if (interleaved) go(rotary_vec_kernel<T, LPH, true, false>);
    else go(rotary_vec_kernel<T, LPH, false, false>);
  }
}

// Whether every head of the call can be read and written in 16-byte chunks, at
// addresses of the 24-bit kind.
bool rotary_vec_ok(const RotArgs& a, int64_t es) {
  if (a.D % 16 != 0 || a.D > 256 || a.R % 16 != 0) return false;
  const int64_t heads = a.na + a.nb;
  if (8 * heads * heads >= (int64_t)1 << 24) return false;
  // (the heads that there are none of have no strides)
  int64_t st[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  uintptr_t at = (uintptr_t)a.ga | (uintptr_t)a.gb;
  if (a.na) {
    st[0] = a.a_st; st[1] = a.a_sh; st[2] = a.ao_st; st[3] = a.ao_sh;
    at |= (uintptr_t)a.a | (uintptr_t)a.ao;
  }
  if (a.nb) {
    st[4] = a.b_st; st[5] = a.b_sh; st[6] = a.bo_st; st[7] = a.bo_sh;
    at |= (uintptr_t)a.b | (uintptr_t)a.bo;
  }
  for (int i = 0; i < 8; ++i) {
    const int64_t most = i == 6 && a.slots != nullptr ? (int64_t)1 << 32 : (int64_t)1 << 24;
    if (st[i] * es % 16 != 0 || st[i] < 0 || st[i] * es / 16 >= most) return false;
    if (i % 2 == 1 && st[i] * es / 16 * heads >= (int64_t)1 << 31) return false;
  }
  return at % 16 == 0;
}

int launch_rotary(const char* fn, const RotArgs& a, int interleaved, int dtype,
                  hipStream_t stream) {
  LL_CHECK_ARG(a.D > 0 && a.D <= 1024 && a.R >= 0 && a.R <= a.D && a.R % 2 == 0,
               "%s: head_dim %d, rotary_dim %d unsupported", fn, a.D, a.R);
  LL_CHECK_ARG(a.R == 0 || (a.pos && a.inv_freq), "%s: null pointer", fn);
  if (a.na + a.nb == 0) return LL_OK;
  // (a grid holds fewer than 2^32 threads, up to 256 for each token)
  LL_CHECK_ARG(a.ntok <= (int64_t)1 << 24 && a.na + a.nb <= 65535,
               "%s: %lld tokens of %d heads unsupported", fn, (long long)a.ntok, a.na + a.nb);
  // heads or tokens on one address would be rotated over one another
  LL_CHECK_ARG((a.na == 0 || ((a.ao_st != 0 || a.ntok == 1) && (a.ao_sh != 0 || a.na == 1))) &&
                   (a.nb == 0 || ((a.bo_st != 0 || (a.slots ? a.nslots <= 1 : a.ntok == 1)) &&
                                  (a.bo_sh != 0 || a.nb == 1))),
               "%s: an output of stride 0", fn);
  const bool vec = rotary_vec_ok(a, dtype == LL_F32 ? 4 : 2);
  return LL_DISPATCH_DTYPE(dtype, T, [&]() -> int {
    if (vec) {
      const int units = a.D / 16;
      if (units <= 4) launch_rotary_vec<T, 4>(a, interleaved, stream);
      else if (units <= 8) launch_rotary_vec<T, 8>(a, interleaved, stream);
      else launch_rotary_vec<T, 16>(a, interleaved, stream);
      LL_RETURN_LAUNCH();
    }
    const dim3 grid((unsigned)a.ntok, (unsigned)(a.na + a.nb));
    if (interleaved)
      hipLaunchKernelGGL((rotary_kernel<T, true>), grid, dim3(64), 0, stream, a);
    else
      hipLaunchKernelGGL((rotary_kernel<T, false>), grid, dim3(64), 0, stream, a);
    LL_RETURN_LAUNCH();
  });
}

}  // namespace

extern "C" int ll_rope_positions(const void* q, int64_t q_stride_tok, int64_t q_stride_h,
                                 void* q_out, int64_t q_out_stride_tok, int64_t q_out_stride_h,
                                 int64_t q_heads, const void* k, int64_t k_stride_tok,
                                 int64_t k_stride_h, void* k_out, int64_t k_out_stride_tok,
                                 int64_t k_out_stride_h, int64_t k_heads, const void* positions,
                                 int positions_i64, const float* inv_freq, int64_t rotary_dim,
                                 int interleaved, float factor, int64_t ntok, int64_t head_dim,
                                 int dtype, hipStream_t stream) {
  const char* fn = "ll_rope_positions";
  LL_CHECK_ARG(q_heads >= 0 && k_heads >= 0 && q_heads + k_heads <= 65535 && ntok >= 0 &&
                   rotary_dim >= 0 && rotary_dim <= head_dim && head_dim <= 1024,
               "%s: %lld + %lld heads of %lld (%lld rotated), %lld tokens", fn, (long long)q_heads,
               (long long)k_heads, (long long)head_dim, (long long)rotary_dim, (long long)ntok);
  if (ntok == 0) return LL_OK;  // (an empty tensor has no address)
  LL_CHECK_ARG((q_heads == 0 || (q && q_out)) && (k_heads == 0 || (k && k_out)), "%s: null pointer",
               fn);
  RotArgs a = {};
  a.a = q; a.a_st = q_stride_tok; a.a_sh = q_stride_h;
  a.ao = q_out; a.ao_st = q_out_stride_tok; a.ao_sh = q_out_stride_h;
  a.b = k; a.b_st = k_stride_tok; a.b_sh = k_stride_h;
  a.bo = k_out; a.bo_st = k_out_stride_tok; a.bo_sh = k_out_stride_h;
  a.na = (int)q_heads; a.nb = (int)k_heads; a.nrot = a.na + a.nb;
  a.D = (int)head_dim; a.R = (int)rotary_dim;
  a.factor = factor;
  a.pos = positions; a.pos64 = positions_i64; a.inv_freq = inv_freq;
  a.ntok = ntok;
  return launch_rotary(fn, a, interleaved, dtype, stream);
}

extern "C" int ll_qk_norm_rope_kv_scatter(
    const void* qkv, int64_t qkv_row_stride, int64_t ntok, int64_t q_heads, int64_t kv_heads,
    int64_t head_dim, void* q_out, int64_t q_out_stride_tok, int64_t q_out_stride_h,
    const void* q_gamma, const void* k_gamma, float eps, const void* positions, int positions_i64,
    const float* inv_freq, int64_t rotary_dim, int interleaved, float factor, const int32_t* slots,
    void* pool_layer, int64_t pool_slot_stride, int64_t pool_head_stride, int64_t pool_slots,
    int dtype, hipStream_t stream) {
  const char* fn = "ll_qk_norm_rope_kv_scatter";
  LL_CHECK_ARG(q_heads > 0 && kv_heads > 0 && q_heads + 2 * kv_heads <= 65535 && ntok >= 0 &&
                   rotary_dim >= 0 && rotary_dim <= head_dim && head_dim <= 1024 && pool_slots >= 0,
               "%s: %lld + 2 x %lld heads of %lld (%lld rotated), %lld tokens, %lld slots", fn,
               (long long)q_heads, (long long)kv_heads, (long long)head_dim,
               (long long)rotary_dim, (long long)ntok, (long long)pool_slots);
  if (ntok == 0) return LL_OK;
  LL_CHECK_ARG(qkv && q_out && slots && (pool_layer || pool_slots == 0), "%s: null pointer", fn);
  const int64_t es = dtype == LL_F32 ? 4 : 2;
  RotArgs a = {};
  a.a = qkv; a.a_st = qkv_row_stride; a.a_sh = head_dim;
  a.ao = q_out; a.ao_st = q_out_stride_tok; a.ao_sh = q_out_stride_h;
  a.b = (const char*)qkv + q_heads * head_dim * es; a.b_st = qkv_row_stride; a.b_sh = head_dim;
  a.bo = pool_layer; a.bo_st = pool_slot_stride; a.bo_sh = pool_head_stride;
  a.na = (int)q_heads; a.nb = (int)(2 * kv_heads); a.nrot = (int)(q_heads + kv_heads);
  a.D = (int)head_dim; a.R = (int)rotary_dim;
  a.ga = q_gamma; a.gb = k_gamma; a.eps = eps; a.factor = factor;
  a.pos = positions; a.pos64 = positions_i64; a.inv_freq = inv_freq;
  a.slots = slots; a.nslots = pool_slots;
  a.ntok = ntok;
  return launch_rotary(fn, a, interleaved, dtype, stream);
}
