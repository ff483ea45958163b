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
// fits fp32 (below 2^-24 of a turn at any int32 position).
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

// Any head_dim, rotary_dim and alignment: one wave per (token, head), a lane
// per pair.
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
  const int64_t p = rot ? ll_load_idx(a.pos, t, a.pos64) : 0;
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

int launch_rotary(const char* fn, const RotArgs& a, int interleaved, int dtype,
                  hipStream_t stream) {
  LL_CHECK_ARG(a.D > 0 && a.D <= 1024 && a.R >= 0 && a.R <= a.D && a.R % 2 == 0,
               "%s: head_dim %d, rotary_dim %d unsupported", fn, a.D, a.R);
  LL_CHECK_ARG(a.R == 0 || (a.pos && a.inv_freq), "%s: null pointer", fn);
  if (a.na + a.nb == 0) return LL_OK;
  LL_CHECK_ARG(a.ntok < ((int64_t)1 << 31) && a.na + a.nb <= 65535,
               "%s: %lld tokens of %d heads unsupported", fn, (long long)a.ntok, a.na + a.nb);
  return LL_DISPATCH_DTYPE(dtype, T, [&]() -> int {
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
