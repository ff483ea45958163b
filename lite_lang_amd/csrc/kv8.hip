// A KV cache held in 8 bits (gfx950): K and V quantised as they are written,
// read back, and attention of one query token per request over them.
//
// A code is an int8 number or an e4m3 float; a block is `block` consecutive
// slots (a power of two, the page size or a part of it), and every block holds
// an fp32 scale for each K head and each V head:
//   value = code * scale[slot / block, head].
// Tokens of a call that follow each other in one block (padded ones among them
// aside) are a run. With top the
// largest code (127, 448), a run alone asks for the scale
//   s = max(fl32(max |x| / top), 2^-80)
// (the floor keeps every quotient below and its residual normal numbers). A run
// that starts at a block's first slot begins the block anew: whatever a former
// owner of the page left there is forgotten. Any other run continues the block:
// its scale is the larger one of the block's and the run's, and where it grew
// the codes in front of the run are rounded again, to
//   code' = round(code * s_old / s_new).
// Codes are the nearest ones to the quotient itself, ties to even: no code
// depends on how a division rounds.
#include <algorithm>
#include <mutex>

#include "ll_common.h"

namespace {

enum { KV8_INT8 = LL_KV8_INT8, KV8_E4M3 = LL_KV8_E4M3 };

constexpr float kScaleFloor = 0x1p-80f;

template <int CODE> struct CodeOf;
template <> struct CodeOf<KV8_INT8> {
  static constexpr float top = 127.f;
  // the code of q, rounded: adding 1.5 2^23 leaves it in the lowest byte
  static __device__ __forceinline__ uint32_t encode(float q) {
    return __builtin_bit_cast(uint32_t, q + 0x1.8p23f) & 0xffu;
  }
  static __device__ __forceinline__ uint32_t low4(float a, float b, float c, float d) {
    const uint32_t w0 = __builtin_bit_cast(uint32_t, a), w1 = __builtin_bit_cast(uint32_t, b);
    const uint32_t w2 = __builtin_bit_cast(uint32_t, c), w3 = __builtin_bit_cast(uint32_t, d);
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(w3, w2, 0x0c0c0400u),
                                 __builtin_amdgcn_perm(w1, w0, 0x0c0c0400u), 0x05040100u);
  }
  static __device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
    return low4(a + 0x1.8p23f, b + 0x1.8p23f, c + 0x1.8p23f, d + 0x1.8p23f);
  }
  // byte i of w as a number
  static __device__ __forceinline__ float decode(uint32_t w, int i) {
    return (float)(int8_t)(uint8_t)(w >> (8 * i));
  }
};
template <> struct CodeOf<KV8_E4M3> {
  static constexpr float top = 448.f;
  static __device__ __forceinline__ uint32_t encode(float q) {
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q, q, 0, false) & 0xffu;
  }
  static __device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(
        c, d, __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false), true);
  }
  static __device__ __forceinline__ float decode(uint32_t w, int i) {
    switch (i) {
      case 0: return __builtin_amdgcn_cvt_f32_fp8((int)w, 0);
      case 1: return __builtin_amdgcn_cvt_f32_fp8((int)w, 1);
      case 2: return __builtin_amdgcn_cvt_f32_fp8((int)w, 2);
      default: return __builtin_amdgcn_cvt_f32_fp8((int)w, 3);
    }
  }
};

// x / s rounded toward zero, its last bit set where that was inexact (rounding
// to odd): rounding the result once more to 16 bits or fewer gives what rounding
// the quotient itself gives. r is 1 / s. The first two lines are within an ulp
// of the quotient; the residual x - q s then has the quotient's error's sign
// (the scale's floor keeps it from underflowing where a code depends on it).
__device__ __forceinline__ float quotient_to_odd(float x, float s, float r) {
  float q = x * r;
  q = __builtin_fmaf(__builtin_fmaf(-q, s, x), r, q);
  const float e = __builtin_fmaf(-q, s, x);
  uint32_t b = __builtin_bit_cast(uint32_t, q);
  const bool over = (__builtin_bit_cast(uint32_t, e) ^ b) >> 31;  // |q| is too large
  const bool off = e != 0.f;
  b -= (off && over) ? 1u : 0u;
  b |= off ? 1u : 0u;
  return __builtin_bit_cast(float, b);
}

// A code times s_old / s_new, rounded to a code again.
template <int CODE>
__device__ __forceinline__ uint32_t recode(float c, float s_old, float s_new) {
  const double q = (double)c * (double)s_old / (double)s_new;
  float f = (float)q;
  uint32_t b = __builtin_bit_cast(uint32_t, f);
  if ((double)f != q) {
    if (fabs((double)f) > fabs(q)) b -= 1u;
    b |= 1u;
  }
  return CodeOf<CODE>::encode(__builtin_bit_cast(float, b));
}

struct StoreArgs {
  const void* x[2]; int64_t x_st[2], x_sh[2];  // K, V: [ntok, heads, D]
  const int32_t* slots;
  uint8_t* c[2]; int64_t c_st[2], c_sh[2];
  float* s[2]; int64_t s_sb[2], s_sh[2];
  int64_t T, nslots;
  int KVH, D, shift, per;  // block = 1 << shift; tokens per wave
};

constexpr int kStoreWaves = 4;
constexpr int kStoreFill = 8192;  // waves that the card holds
constexpr int kTeamBlock = 32;

// 8 elements of a row as they lie in memory; those at D and behind are 0
template <typename T> struct Raw8 { u32x4 w[sizeof(T) / 2]; };
template <typename T, bool VEC>
__device__ __forceinline__ Raw8<T> load8(const T* p, int d, int D) {
  Raw8<T> r = {};
  if constexpr (VEC) {
    if (d < D)
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i)
        r.w[i] = __builtin_nontemporal_load((const u32x4*)(p + d) + i);
  } else {
    T* e = (T*)r.w;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (d + i < D) e[i] = p[d + i];
  }
  return r;
}
template <typename T> __device__ __forceinline__ float get(const Raw8<T>& r, int i) {
  return ll_to_f32(((const T*)r.w)[i]);
}

// Magnitudes as integers: ordered like the numbers, infinities and NaN on top.
// 16-bit types two at a time.
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
template <typename T> __device__ __forceinline__ uint32_t widen(uint32_t m, const Raw8<T>& r) {
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      m = __builtin_bit_cast(
          uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, m),
                                              __builtin_bit_cast(u16x2, r.w[0][i] & 0x7fff7fffu)));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, r.w[i >> 2][i & 3] & 0x7fffffffu);
  }
  return m;
}
// the number of the larger magnitude held in m; infinite for NaN too
template <typename T> __device__ __forceinline__ float widest(uint32_t m) {
  if constexpr (sizeof(T) == 2) {
    const uint16_t b = (uint16_t)max(m & 0xffffu, m >> 16);
    const float v = ll_to_f32(__builtin_bit_cast(T, b));
    return v < INFINITY ? v : INFINITY;
  } else {
    const float v = __builtin_bit_cast(float, m);
    return v < INFINITY ? v : INFINITY;
  }
}

// The codes of 8 elements. Rounding x * (1 / s) gives the right one but where the
// quotient is next to a border between two codes. For int8 the residual x - c s,
// which is exact, tells: no more than s / 2 beside the border, s / 2 on it. For
// e4m3 the product's bits below the code's last: within 4 steps of half of it
// (the product is off by 1.5); 2^-6 added gives subnormal quotients the steps of
// their codes. A wave with such an element takes the exact quotients.
template <typename T, int CODE>
__device__ __forceinline__ void codes_of(const Raw8<T>& r, float s, float inv, uint32_t& w0,
                                         uint32_t& w1) {
  float v[8], q[8];
  bool near;
  if constexpr (CODE == KV8_INT8) {
    float off = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = get(r, e);
      q[e] = __builtin_fmaf(v[e], inv, 0x1.8p23f);
      off = fmaxf(off, fabsf(__builtin_fmaf(0x1.8p23f - q[e], s, v[e])));
    }
    near = !(off < 0.5f * s);
    w0 = CodeOf<CODE>::low4(q[0], q[1], q[2], q[3]);
    w1 = CodeOf<CODE>::low4(q[4], q[5], q[6], q[7]);
  } else {
    uint32_t gap = 0xffffffffu;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = get(r, e);
      q[e] = v[e] * inv;
      const float z = fabsf(q[e]) < 0x1p-6f ? fabsf(q[e]) + 0x1p-6f : q[e];
      gap = min(gap, (__builtin_bit_cast(uint32_t, z) + 0x80004u) & 0xfffffu);
    }
    near = gap <= 8u;
    w0 = CodeOf<CODE>::encode4(q[0], q[1], q[2], q[3]);
    w1 = CodeOf<CODE>::encode4(q[4], q[5], q[6], q[7]);
  }
  if (__ballot(near)) {
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = quotient_to_odd(v[e], s, inv);
    w0 = CodeOf<CODE>::encode4(q[0], q[1], q[2], q[3]);
    w1 = CodeOf<CODE>::encode4(q[4], q[5], q[6], q[7]);
  }
  if (!(s < INFINITY)) w0 = w1 = 0;
}

template <typename T, int CODE, bool VEC>
__device__ __forceinline__ void store8(uint8_t* p, int d, int D, const Raw8<T>& r, float s,
                                       float inv) {
  uint32_t w0, w1;
  codes_of<T, CODE>(r, s, inv, w0, w1);
  if constexpr (VEC) {
    if (d < D) *(uint2*)(p + d) = make_uint2(w0, w1);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (d + i < D) p[d + i] = (uint8_t)((i < 4 ? w0 : w1) >> (8 * (i & 3)));
  }
}

// The scale that elements of largest magnitude `top` ask for (infinite: NaN).
template <int CODE> __device__ __forceinline__ float scale_of(float top) {
  return top < INFINITY ? fmaxf(top / CodeOf<CODE>::top, kScaleFloor) : __builtin_nanf("");
}

// Lanes that hold a row of D elements, 8 each (a power of two).
__device__ __forceinline__ int lanes_of(int D) {
  int n = 1;
  while (n * 8 < D && n < 64) n *= 2;
  return n;
}

// Blocks of one slot: every row has a scale of its own. A row's elements stay in
// the registers of its lanes between the maximum and the codes. Bound by that one
// chain (slot, row, maximum, codes), with nothing of a next row in flight: 24,000
// tokens of 2 x 128 in 15.2 us (2.4 TB/s, half of a copy's rate).
template <typename T, int CODE, bool VEC>
__global__ __launch_bounds__(kStoreWaves * 64) void store_rows_kernel(StoreArgs a) {
  constexpr int kHold = 2;  // D up to 1024
  const int lane = threadIdx.x & 63, lpr = lanes_of(a.D), units = 2 * a.KVH;
  const int i = (blockIdx.x * kStoreWaves + (threadIdx.x >> 6)) * (64 / lpr) + lane / lpr;
  const int t = min(i / units, (int)a.T - 1);
  const int unit = i % units, d0 = lane % lpr * 8;
  const int kv = unit >= a.KVH, head = unit - kv * a.KVH;
  const int32_t slot = a.slots[t];
  const T* x = (const T*)(kv ? a.x[1] : a.x[0]) + t * (kv ? a.x_st[1] : a.x_st[0]) +
               head * (kv ? a.x_sh[1] : a.x_sh[0]);
  Raw8<T> r[kHold];
  uint32_t m = 0;
#pragma unroll
  for (int k = 0; k < kHold; ++k) {
    r[k] = load8<T, VEC>(x, d0 + k * 512, a.D);
    m = widen(m, r[k]);
  }
  float top = widest<T>(m);
  for (int o = 1; o < lpr; o *= 2) top = fmaxf(top, __shfl_xor(top, o, 64));
  if (i >= (int)a.T * units || slot < 0 || slot >= a.nslots) return;
  const float s = scale_of<CODE>(top), inv = 1.f / s;
  uint8_t* c = (kv ? a.c[1] : a.c[0]) + slot * (kv ? a.c_st[1] : a.c_st[0]) +
               head * (kv ? a.c_sh[1] : a.c_sh[0]);
#pragma unroll
  for (int k = 0; k < kHold; ++k) store8<T, CODE, VEC>(c, d0 + k * 512, a.D, r[k], s, inv);
  if (d0 == 0)
    (kv ? a.s[1] : a.s[0])[slot * (kv ? a.s_sb[1] : a.s_sb[0]) +
                           head * (kv ? a.s_sh[1] : a.s_sh[0])] = s;
}

// A team of waves: the runs that start among `per` tokens, of one head's K or V.
// A row takes as many lanes as it has groups of 8 elements, and the team as many
// rows at a time as fit. The first kHold such groups of rows stay in registers
// between the run's largest element and its codes; the others are read again.
// (Every wave of a team sees the same runs, so the barriers are for all.)
// A run is a chain of round trips (slots, rows, codes), so what counts is how many
// run at a time: registers for 4 groups of rows leave 28 waves per CU (8 groups: 20
// waves, 24,000 tokens of 2 x 128 in blocks of 16 16.6 us, now 12.6: 2.9 TB/s),
// and a run of 64 rows is quicker in four waves (blocks of 64, 5,055 new tokens of
// 4 x 128 behind prefixes: 26 us in one wave, 18.5; 672 of the 5,056 teams have a
// run there, the others read slots and end). Rows are read past the L2 (-2). Blocks
// that grow are rounded again code by code: 40 single tokens of 2 x 128, blocks of
// 16 of random numbers, 10.9 us, and 4.1 where no scale grows.
template <typename T, int CODE, bool VEC, int TEAM>
__global__ __launch_bounds__(kStoreWaves * 64) void store_kernel(StoreArgs a) {
  constexpr int kHold = 4;
  __shared__ float s_top[2][TEAM];
  const int lane = threadIdx.x & 63, me = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int team = (blockIdx.x * kStoreWaves + me) / TEAM, units = 2 * a.KVH, unit = team % units;
  const int64_t t0 = (int64_t)(team / units) * a.per;
  int turn = 0;
  if (t0 >= a.T) return;
  const int kv = unit >= a.KVH, head = unit - kv * a.KVH;
  const T* x = (const T*)a.x[kv] + head * a.x_sh[kv];
  uint8_t* c = a.c[kv] + head * a.c_sh[kv];
  float* sc = a.s[kv] + head * a.s_sh[kv];
  const int64_t xs = a.x_st[kv], cs = a.c_st[kv];
  const int D = a.D, lpr = lanes_of(D), rows = 64 / lpr * TEAM, d0 = lane % lpr * 8;
  const int row = me % TEAM * (64 / lpr) + lane / lpr;
  const auto valid = [&](int32_t s) { return s >= 0 && s < a.nslots; };

  const int64_t t1 = min(t0 + (int64_t)a.per, a.T);
  // the slots of the 64 tokens from t0 on (no run of this wave's starts behind them),
  // and of the 64 before
  const int32_t sl = a.slots[min(t0 + lane, a.T - 1)];
  const int32_t back = a.slots[max(t0 - 1 - lane, (int64_t)0)];
  bool ours = false;  // whether the next token stored begins a run (known behind the first run)
  for (int64_t t = t0; t < t1;) {
    const int32_t first = __builtin_amdgcn_readlane(sl, (int)(t - t0));
    if (!valid(first)) {
      ++t;
      continue;
    }
    const int32_t blk = first >> a.shift;
    // the run's end (the first token of another block; padded ones among the
    // run's belong to no block) and its last token
    int64_t end = -1, last = t + 1;
    int32_t here = sl;
    for (int64_t base = t0; end < 0; base += 64) {
      const bool in = base + lane < a.T, its = valid(here) && here >> a.shift == blk;
      uint64_t other = __ballot(!in || (valid(here) && !its)), same = __ballot(in && its);
      if (base <= t) {  // (the tokens up to t are behind)
        const uint64_t ahead = t - base == 63 ? 0 : ~(uint64_t)0 << (t - base + 1);
        other &= ahead;
        same &= ahead;
      }
      if (other) {
        const int cut = __builtin_ctzll(other);
        same &= ((uint64_t)1 << cut) - 1;
        end = base + cut;
      } else {
        here = a.slots[min(base + 64 + lane, a.T - 1)];
      }
      if (same) last = base + 64 - __builtin_clzll(same);
    }
    if (!ours) {  // a run that began before this wave's tokens is another wave's
      bool theirs = false;
      int32_t s = back;
      for (int64_t base = t0 - 1; base >= 0; base -= 64) {
        const bool is = base - lane >= 0 && valid(s);
        const uint64_t m = __ballot(is), same = __ballot(is && s >> a.shift == blk);
        if (m) {
          theirs = same >> __builtin_ctzll(m) & 1;
          break;
        }
        if (base >= 64) s = a.slots[max(base - 64 - lane, (int64_t)0)];
      }
      ours = true;
      if (theirs) {
        t = end;
        continue;
      }
    }
    const int off = first & ((1 << a.shift) - 1);
    float* sp = sc + blk * a.s_sb[kv];
    const float old = *sp;
    Raw8<T> r[kHold];
    int32_t slot[kHold];
#pragma unroll
    for (int k = 0; k < kHold; ++k) {
      const int64_t i = t + row + k * rows;
      slot[k] = -1;
      r[k] = {};
      if (i < last) {
        slot[k] = a.slots[i];
        r[k] = load8<T, VEC>(x + i * xs, d0, D);
      }
    }
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < kHold; ++k)
      if (valid(slot[k])) m = widen(m, r[k]);
    // what is not held: more rows, and elements from 512 on
    const auto others = [&](auto f) {
      for (int64_t i = t + row; i < last; i += rows) {
        const bool held = i < t + row + kHold * rows;
        const int32_t s = a.slots[i];
        if (!valid(s)) continue;
        for (int d = held ? d0 + 512 : d0; d < D; d += 512)
          f(load8<T, VEC>(x + i * xs, d, D), s, d);
      }
    };
    const bool more = last - t > kHold * rows || D > 512;
    if (more) others([&](const Raw8<T>& v, int32_t, int) { m = widen(m, v); });
    float top = ll_wave_max(widest<T>(m));
    if constexpr (TEAM > 1) {
      if (lane == 0) s_top[turn][me] = top;
      __syncthreads();
#pragma unroll
      for (int k = 0; k < TEAM; ++k) top = fmaxf(top, s_top[turn][k]);
      turn ^= 1;  // (the other half is read no more)
    }
    float s = scale_of<CODE>(top);
    if (off > 0) {
      if (!(s <= old)) {  // it grew, or either is NaN (which stays)
        if (!(s > old)) s = __builtin_nanf("");
        else
          for (int j = row; j < off; j += rows)
            for (int d = d0; d < D; d += 512) {
              uint8_t* p = c + (((int64_t)blk << a.shift) + j) * cs + d;
              for (int e = 0; e < min(8, D - d); ++e)
                p[e] = (uint8_t)recode<CODE>(CodeOf<CODE>::decode(p[e], 0), old, s);
            }
      } else {
        s = old;
      }
    }
    const float inv = 1.f / s;
#pragma unroll
    for (int k = 0; k < kHold; ++k)
      if (valid(slot[k])) store8<T, CODE, VEC>(c + slot[k] * cs, d0, D, r[k], s, inv);
    if (more)
      others([&](const Raw8<T>& v, int32_t to, int d) {
        store8<T, CODE, VEC>(c + to * cs, d, D, v, s, inv);
      });
    if (lane == 0 && me % TEAM == 0) *sp = s;
    t = end;
  }
}

struct LoadArgs {
  const uint8_t* c[2]; int64_t c_st[2], c_sh[2];
  const float* s[2]; int64_t s_sb[2], s_sh[2];
  const int32_t* r2t; int64_t r2t_s, r2t_rows;
  const void* req; int req64;
  const void* start; int start64;
  const void* len; int len64;
  void* o[2]; int64_t o_st[2], o_sh[2];
  int64_t nslots, orows;
  int KVH, D, shift, max_len, pieces;  // pieces: of a head's row
};

constexpr int kLoadThreads = 256, kLoadTokens = 2;
constexpr int kLoadFill = 4096;  // workgroups at most, the batch's requests aside

// A thread has one place in a token's rows, 16 codes (VEC) or one, and takes it
// of every token that is its own, two at a time (four: 10.8 us for 24,000 tokens
// of 2 x 128, two: 10.4, 3.6 TB/s). Bound by memory; the outputs are stored past
// the L2, 2 us quicker.
template <typename T, int CODE, bool VEC>
__global__ __launch_bounds__(kLoadThreads) void load_kernel(LoadArgs a) {
  const int b = blockIdx.y;
  const int64_t row = ll_load_idx(a.req, b, a.req64), len = ll_load_idx(a.len, b, a.len64);
  const int64_t base = ll_load_idx(a.start, b, a.start64);
  if (row < 0 || row >= a.r2t_rows || len <= 0) return;
  const int n = (int)min(len, (int64_t)a.max_len);
  const int32_t* table = a.r2t + row * a.r2t_s;
  const int places = 2 * a.KVH * a.pieces;
  const int here = min(places, kLoadThreads), tokens = kLoadThreads / here;  // of the workgroup
  const int mine = threadIdx.x / here;
  if (mine >= tokens) return;
  const int step = gridDim.x * tokens;
  for (int place = threadIdx.x % here; place < places; place += kLoadThreads) {
    const int piece = place % a.pieces, kh = place / a.pieces;
    const int kv = kh >= a.KVH, head = kh - kv * a.KVH;
    const float* sc = (kv ? a.s[1] : a.s[0]) + head * (kv ? a.s_sh[1] : a.s_sh[0]);
    const uint8_t* c = (kv ? a.c[1] : a.c[0]) + head * (kv ? a.c_sh[1] : a.c_sh[0]);
    T* o = (T*)(kv ? a.o[1] : a.o[0]) + head * (kv ? a.o_sh[1] : a.o_sh[0]);
    const int64_t ssb = kv ? a.s_sb[1] : a.s_sb[0], cst = kv ? a.c_st[1] : a.c_st[0],
                  ost = kv ? a.o_st[1] : a.o_st[0];
    for (int64_t t0 = blockIdx.x * tokens + mine; t0 < n; t0 += (int64_t)step * kLoadTokens) {
      int32_t slot[kLoadTokens];
      float s[kLoadTokens];
      u32x4 w[kLoadTokens];
#pragma unroll
      for (int k = 0; k < kLoadTokens; ++k) {
        const int64_t t = t0 + (int64_t)k * step;
        slot[k] = t < n ? table[t] : -1;
      }
#pragma unroll
      for (int k = 0; k < kLoadTokens; ++k) {
        const bool is = slot[k] >= 0 && slot[k] < a.nslots;
        s[k] = 0.f;
        w[k] = (u32x4){0, 0, 0, 0};
        if (is) {
          s[k] = sc[(slot[k] >> a.shift) * ssb];
          if constexpr (VEC) w[k] = *(const u32x4*)(c + slot[k] * cst + piece * 16);
          else w[k][0] = c[slot[k] * cst + piece];
        }
      }
#pragma unroll
      for (int k = 0; k < kLoadTokens; ++k) {
        const int64_t t = t0 + (int64_t)k * step, to = base + t;
        if (t >= n || to < 0 || to >= a.orows) continue;
        if constexpr (VEC) {
          u32x4 y[sizeof(T)];
          T* e = (T*)y;
#pragma unroll
          for (int j = 0; j < 16; ++j)
            e[j] = ll_from_f32<T>(CodeOf<CODE>::decode(w[k][j >> 2], j & 3) * s[k]);
#pragma unroll
          for (int j = 0; j < (int)sizeof(T); ++j)
            __builtin_nontemporal_store(y[j], (u32x4*)(o + to * ost + piece * 16) + j);
        } else {
          o[to * ost + piece] = ll_from_f32<T>(CodeOf<CODE>::decode(w[k][0], 0) * s[k]);
        }
      }
    }
  }
}

struct DecodeArgs8 {
  const void* q; int64_t q_sb, q_sh;
  const uint8_t* c[2]; int64_t c_st[2], c_sh[2];
  const float* s[2]; int64_t s_sb[2], s_sh[2];
  const int32_t* r2t; int64_t r2t_s, r2t_rows;
  const void* req; int req64;
  const void* len; int len64;
  void* out; int64_t o_sb, o_sh;
  int64_t nslots;
  int B, H, KVH, G, D, shift, max_len;
  int hb, W, whole;  // blocks of 16 query heads, workgroups of each, a request for each
  int qvec, ovec;    // 16-byte loads of q, stores of out
  float scale_log2;
  float* part; float2* part_ml;  // [W + B, H, D], [W + B, H]
  int2* meta;                    // [B]: a request's first part, how many it has
};

__device__ __forceinline__ int decode_len(const DecodeArgs8& a, int b, int64_t* row) {
  *row = ll_load_idx(a.req, b, a.req64);
  const int64_t n = ll_load_idx(a.len, b, a.len64);
  if (*row < 0 || *row >= a.r2t_rows || n <= 0) return 0;
  return (int)std::min<int64_t>(n, a.max_len);
}

constexpr int kAnyMaxD = 512;

// Any head dim and alignment: a wave per request and query head, 64 tokens at a
// time: a lane's own token's score, then every lane's own elements of the sum. Its
// bytes come one by one: 57 ms for 131,072 tokens of 12/2 x 128.
template <typename T, int CODE>
__global__ __launch_bounds__(64) void decode_any_kernel(DecodeArgs8 a) {
  __shared__ float sq[kAnyMaxD], sp[64];
  __shared__ int32_t ss[64];
  const int h = blockIdx.x % a.H, b = blockIdx.x / a.H, lane = threadIdx.x, kvh = h / a.G;
  int64_t row;
  const int n = decode_len(a, b, &row);
  const T* q = (const T*)a.q + b * a.q_sb + h * a.q_sh;
  float top = 0.f;
  for (int d = lane; d < a.D; d += 64) {
    sq[d] = ll_to_f32(q[d]);
    top = fmaxf(top, fabsf(sq[d]));
  }
  // (queries beyond 2^50 as in the matrix form)
  const int e = max(__builtin_amdgcn_frexp_expf(ll_wave_max(top)) - 50, 0);
  const float more = __builtin_ldexpf(1.f, e);
  for (int d = lane; d < a.D; d += 64) sq[d] = __builtin_ldexpf(sq[d], -e);
  __syncthreads();
  const int32_t* table = a.r2t + (n > 0 ? row : 0) * a.r2t_s;
  float m = -INFINITY, l = 0.f, acc[kAnyMaxD / 64] = {};
  for (int t0 = 0; t0 < n; t0 += 64) {
    const int t = t0 + lane;
    const int32_t slot = t < n ? table[t] : -1;
    const bool see = slot >= 0 && slot < a.nslots;
    float x = -INFINITY;
    if (see) {
      const uint8_t* k = a.c[0] + slot * a.c_st[0] + kvh * a.c_sh[0];
      float dot = 0.f;
      for (int d = 0; d < a.D; ++d) dot = __builtin_fmaf(sq[d], CodeOf<CODE>::decode(k[d], 0), dot);
      x = dot * a.s[0][(slot >> a.shift) * a.s_sb[0] + kvh * a.s_sh[0]] * a.scale_log2 * more;
    }
    const float mt = fmaxf(m, ll_wave_max(x));
    const float ms = mt == -INFINITY ? 0.f : mt;
    const float alpha = exp2f(m - ms);
    const float p = see ? exp2f(x - ms) : 0.f;
    l = l * alpha + ll_wave_sum(p);
    m = mt;
    sp[lane] = see ? p * a.s[1][(slot >> a.shift) * a.s_sb[1] + kvh * a.s_sh[1]] : 0.f;
    ss[lane] = see ? slot : -1;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kAnyMaxD / 64; ++j) {
      const int d = lane + 64 * j;
      if (d < a.D) {
        float y = acc[j] * alpha;
        for (int i = 0; i < min(64, n - t0); ++i)
          if (ss[i] >= 0)
            y = __builtin_fmaf(
                sp[i], CodeOf<CODE>::decode(a.c[1][ss[i] * a.c_st[1] + kvh * a.c_sh[1] + d], 0), y);
        acc[j] = y;
      }
    }
    __syncthreads();
  }
  T* o = (T*)a.out + b * a.o_sb + h * a.o_sh;
#pragma unroll
  for (int j = 0; j < kAnyMaxD / 64; ++j) {
    const int d = lane + 64 * j;
    if (d < a.D) o[d] = ll_from_f32<T>(l == 0.f ? 0.f : acc[j] / l);
  }
}

// ------------------------------------------------------------------ matrix form
// A workgroup takes a block of up to 16 query heads that share a KV head, and
// its share of the batch's tokens (below); its waves take every fourth tile of 32.
//   S [16 tokens x 16 heads] = K Q^T,  O^T [16 dims x 16 heads] += V^T P^T
// by 16x16x32 MFMAs, whose k index may run in any order that both operands
// agree on. So a lane's K operand is 16 bytes of its own token's row, and the
// scores that a lane gets, tokens 4 g .. 4 g + 3 and 16 + 4 g .. (g = lane / 16)
// of head lane % 16, are its P operand as they are; its V operand are those
// tokens' bytes of the dims that it owns, each byte put straight into its place.
// No data passes through LDS but the addresses and scales of the tile, and the
// next tile's loads are in flight while one is computed.
//
// q is split into as many bf16 numbers as hold it (fp16 two, fp32 three), a
// probability times its V scale likewise into two (2^-16 of itself; three for
// fp32), so that 8-bit codes are all that is lost. e4m3 codes are bf16 numbers.
// An int8 code c becomes one without arithmetic: the byte u = c + 128 in the low
// half of a bf16 number is u 2^-133 (a subnormal below 128, and the next
// exponent goes on in the same steps), which the MFMA takes as it is. q and P
// are scaled by powers of two to make up for it, and the 128 leaves as the same
// sum of a constant operand: of q once per call, of P with every tile. Its cost
// is a few more roundings of fp32 sums (2^-24 of 128 |sum q|); fp32 calls, where
// that would show, convert the codes instead. The maximum moves only when a tile
// has a larger one.
template <typename T>
constexpr int kQParts = __is_same(T, float) ? 3 : __is_same(T, __bf16) ? 1 : 2;
template <typename T> constexpr int kPParts = __is_same(T, float) ? 3 : 2;

// the upper halves of two floats: their bf16 values, where those are exact
__device__ __forceinline__ uint32_t pack_exact(float lo, float hi) {
  return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, hi), __builtin_bit_cast(uint32_t, lo),
                               0x07060302u);
}
// the lower or upper two e4m3 codes of w as bf16
template <bool HIGH> __device__ __forceinline__ uint32_t fp8_pair(uint32_t w) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, HIGH));
}

// 8 codes of one row (two dwords; with BIAS their bytes are c + 128)
template <int CODE, bool BIAS> __device__ __forceinline__ bf16x8 codes8(uint32_t a, uint32_t b) {
  u32x4 w;
  if constexpr (BIAS) {
    w[0] = __builtin_amdgcn_perm(0u, a, 0x0c010c00u);
    w[1] = __builtin_amdgcn_perm(0u, a, 0x0c030c02u);
    w[2] = __builtin_amdgcn_perm(0u, b, 0x0c010c00u);
    w[3] = __builtin_amdgcn_perm(0u, b, 0x0c030c02u);
  } else if constexpr (CODE == KV8_INT8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t v = i < 2 ? a : b;
      w[i] = pack_exact(CodeOf<CODE>::decode(v, 2 * (i & 1)),
                        CodeOf<CODE>::decode(v, 2 * (i & 1) + 1));
    }
  } else {
    w[0] = fp8_pair<false>(a);
    w[1] = fp8_pair<true>(a);
    w[2] = fp8_pair<false>(b);
    w[3] = fp8_pair<true>(b);
  }
  return __builtin_bit_cast(bf16x8, w);
}

// bytes 2 I and 2 I + 1 of 8 rows
template <int CODE, bool BIAS, int I>
__device__ __forceinline__ void codes_of_rows(const uint32_t (&v)[8], bf16x8& lo, bf16x8& hi) {
  u32x4 w0, w1;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t a = v[2 * e], b = v[2 * e + 1];
    if constexpr (BIAS) {
      w0[e] = __builtin_amdgcn_perm(b, a, 0x0c000c00u | (2u * I) | (4u + 2 * I) << 16);
      w1[e] = __builtin_amdgcn_perm(b, a, 0x0c000c00u | (2u * I + 1) | (5u + 2 * I) << 16);
    } else if constexpr (CODE == KV8_INT8) {
      w0[e] = pack_exact(CodeOf<CODE>::decode(a, 2 * I), CodeOf<CODE>::decode(b, 2 * I));
      w1[e] = pack_exact(CodeOf<CODE>::decode(a, 2 * I + 1), CodeOf<CODE>::decode(b, 2 * I + 1));
    } else {  // the four bytes in their order, then two at a time
      const uint32_t s = __builtin_amdgcn_perm(
          b, a, (2u * I) | (4u + 2 * I) << 8 | (2u * I + 1) << 16 | (5u + 2 * I) << 24);
      w0[e] = fp8_pair<false>(s);
      w1[e] = fp8_pair<true>(s);
    }
  }
  lo = __builtin_bit_cast(bf16x8, w0);
  hi = __builtin_bit_cast(bf16x8, w1);
}

// parts[i]: what is left of x behind parts 0 .. i - 1, in bf16
template <int N> __device__ __forceinline__ void split8(const float (&x)[8], bf16x8 (&parts)[N]) {
  float left[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) left[e] = x[e];
#pragma unroll
  for (int i = 0; i < N; ++i) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      parts[i][e] = (__bf16)left[e];
      left[e] -= (float)parts[i][e];
    }
  }
}

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

template <int N> struct BytesOf;
template <> struct BytesOf<4> { typedef uint32_t V; };
template <> struct BytesOf<8> { typedef uint2 V; };
template <> struct BytesOf<16> { typedef uint4 V; };

constexpr int kTile8 = 32, kWaves8 = 4;
// biased codes: a value of binary exponent e goes to about 2^kUp, and a sum of
// its products, at 2^(kUp - 133), comes back by 2^(133 - kUp + e)
constexpr int kUp = 60;

// a tile's loads: K rows, V bytes, the scale of a lane's own token
template <int D> struct Tile8 {
  u32x4 kw[2][D / 64];
  uint32_t vw[D / 64][8];
  float scale;
  uint32_t see;  // a bit per token that is one
};

// The batch's tokens are dealt out evenly whatever the lengths are: request after
// request in steps of 128 tokens (a tile per wave), workgroup w of a head block
// takes steps w * per .. of the list, per = ceil(steps / W). A request that lies
// in one workgroup's share is finished there; of the others every workgroup
// leaves its part (rows w + b of the workspace: along the list w or b grows from
// part to part, so no two share one) to the merge.
//
// Bound by memory: 40 requests of up to 16,384 tokens, 16/2 x 128, 229 MB in 50 us
// (4.6 TB/s; 70 with a fixed number of splits per request and loads under
// conditions). Two workgroups per CU: a third spills registers (62 us). Short
// shares are bound by their chain (length, slots, rows): one context of 131,072
// tokens, 4 steps to a workgroup, takes 20 us for 68 MB.
constexpr int kStep8 = kWaves8 * kTile8;

__device__ __forceinline__ int steps_of(int n) { return (n + kStep8 - 1) / kStep8; }
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

template <typename T, int CODE, int D>
__global__ __launch_bounds__(kWaves8 * 64, D == 256 || __is_same(T, float) ? 1 : 2)
void decode_mfma_kernel(DecodeArgs8 a) {
  constexpr bool BIAS = CODE == KV8_INT8 && !__is_same(T, float);
  constexpr bool FAR = !__is_same(T, _Float16);  // whether a query may be beyond 2^50
  constexpr int NQ = kQParts<T>, NP = kPParts<T>, NK = D / 64, NV = D / 16;
  typedef typename BytesOf<NV>::V VBytes;
  __shared__ int64_t s_off[kWaves8][2][kTile8];
  __shared__ float s_scale[kWaves8][2][kTile8];
  __shared__ float s_m[kWaves8][16], s_l[kWaves8][16];
  __shared__ f32x4 s_acc[kWaves8 - 1][NV][64];
  __shared__ int s_sum[kWaves8], s_b, s_step, s_n;
  __shared__ int64_t s_row;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int c16 = lane & 15, g = lane >> 4;
  // The heads of one share of tokens read its table, its scales' lines and, with
  // narrow heads, its rows' lines: they sit on one XCD (workgroups go to the 8
  // XCDs in turn).
  const int heads = a.KVH * a.hb, i8 = blockIdx.x / 8, u = i8 % heads;
  const int w = i8 / heads * 8 + blockIdx.x % 8;
  if (w >= a.W) return;
  const int hb = u % a.hb, kvh = u / a.hb;
  const int head = hb * 16 + c16;  // of the KV head's
  const bool live = head < a.G;
  const int h = kvh * a.G + (live ? head : 0);

  int b = w, step = 0, left = INT32_MAX, per = 0;  // where in request b, steps to go
  int64_t row;
  int n;
  if (a.whole) {
    n = decode_len(a, b, &row);
  } else {
    const int each = (a.B + kWaves8 * 64 - 1) / (kWaves8 * 64);
    const int b0 = min((int)threadIdx.x * each, a.B), b1 = min(b0 + each, a.B);
    int mine = 0;
    n = 0;
    for (int i = b0; i < b1; ++i) mine += steps_of(n = decode_len(a, i, &row));
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(upto, o, 64);
      if (lane >= o) upto += v;
    }
    if (lane == 63) s_sum[wave] = upto;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int i = 0; i < kWaves8; ++i) {
      if (i < wave) upto += s_sum[i];
      all += s_sum[i];
    }
    all = uniform(all);
    per = max((int)(((int64_t)all + a.W - 1) / a.W), 1);
    const int64_t from = (int64_t)w * per;
    if (from >= all) return;
    left = (int)min((int64_t)per, all - from);
    if (from >= upto - mine && from < upto) {
      int at = upto - mine, i = b0;
      while (each > 1) {  // (of one, n and row are its own)
        n = decode_len(a, i, &row);
        if (from < at + steps_of(n)) break;
        at += steps_of(n);
        ++i;
      }
      s_b = i;
      s_step = (int)from - at;
      s_n = n;
      s_row = row;
    }
    __syncthreads();
    b = uniform(s_b);
    step = uniform(s_step);
    n = uniform(s_n);
    row = s_row;
  }
  while (true) {
    const int steps = steps_of(n);
    const int take = min(steps - step, left);
    const bool split = step > 0 || take < steps;
    const int t0 = step * kStep8, t1 = (int)min((int64_t)n, ((int64_t)step + take) * kStep8);
    if (!a.whole && step == 0 && u == 0 && threadIdx.x == 0 && n > 0) {
      // what is left of the request lies in the following workgroups, `per` in each
      a.meta[b] = make_int2(w + b, 1 + (steps - take + per - 1) / per);
    }
    left = a.whole ? 0 : left - take;
    if (n == 0) {  // (in a list the merge writes its rows)
      if (a.whole)
        for (int i = threadIdx.x; i < min(16, a.G - hb * 16) * D; i += kWaves8 * 64)
          ((T*)a.out)[b * a.o_sb + (kvh * a.G + hb * 16 + i / D) * a.o_sh + i % D] =
              ll_from_f32<T>(0.f);
    } else {
      const int32_t* table = a.r2t + row * a.r2t_s;
      // a lane's own token of the tile, and whether it looks after its K or its V
      const int tok = lane & 31, kv = lane >> 5;
      const float* sc = a.s[kv] + kvh * a.s_sh[kv];
      const int64_t ssb = a.s_sb[kv], cst = a.c_st[kv];
      const uint8_t* kc = a.c[0] + kvh * a.c_sh[0] + g * 16;
      const uint8_t* vc = a.c[1] + kvh * a.c_sh[1] + c16 * NV;
      constexpr int kStep = kStep8;
      // No load below stands under a condition, so that the waits count how many
      // came after the one they are for: a tile behind the last one fetches row 0.
      const auto entry_of = [&](int t) -> int32_t { return table[min(t + tok, n - 1)]; };
      // (a wave's own LDS, in order: the fences are for the compiler)
      const auto fetch = [&](Tile8<D>& f, int t, int32_t entry) {
        const bool is = t + tok < t1 && entry >= 0 && entry < a.nslots;
        const int64_t s = is ? entry : 0;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        s_off[wave][kv][tok] = s * cst;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        f.scale = sc[(s >> a.shift) * ssb];
        f.see = (uint32_t)__ballot(is);
#pragma unroll
        for (int grp = 0; grp < 2; ++grp) {
          const uint8_t* p = kc + s_off[wave][0][grp * 16 + c16];
#pragma unroll
          for (int i = 0; i < NK; ++i) f.kw[grp][i] = *(const u32x4*)(p + i * 64);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const VBytes v = *(const VBytes*)(vc + s_off[wave][1][(j >> 2) * 16 + g * 4 + (j & 3)]);
          uint32_t w[NK];
          __builtin_memcpy(w, &v, NV);
#pragma unroll
          for (int i = 0; i < NK; ++i) f.vw[i][j] = w[i];
        }
      };

      int t = t0 + wave * kTile8;
      constexpr int kStages = D <= 128 ? 2 : 1;  // tiles held
      Tile8<D> f[kStages];
      int32_t entry[kStages];
#pragma unroll
      for (int s = 0; s < kStages; ++s) entry[s] = entry_of(t + s * kStep);
      u32x4 raw[NK * 2][sizeof(T) / 2];
      {
        const T* q = (const T*)a.q + b * a.q_sb + h * a.q_sh;
#pragma unroll
        for (int i = 0; i < NK * 2; ++i) {
          const int d = (i >> 1) * 64 + g * 16 + (i & 1) * 8;
          if (a.qvec) {
#pragma unroll
            for (int e = 0; e < (int)sizeof(T) / 2; ++e) raw[i][e] = ((const u32x4*)(q + d))[e];
          } else {
            __builtin_memcpy(raw[i], __builtin_assume_aligned(q + d, sizeof(T)), sizeof(raw[i]));
          }
        }
      }
#pragma unroll
      for (int s = 0; s < (kStages > 1 ? kStages - 1 : 1); ++s)
        fetch(f[s], t + s * kStep, entry[s]);
      int32_t next = kStages > 1 ? entry[kStages - 1] : entry_of(t + kStep);
      bf16x8 qf[NK * 2][NQ];
      // of a score's sum; of queries beyond 2^50, which are held smaller so that no sum
      // passes fp32's range before its scales are applied: what takes that back
      float cq = a.scale_log2, more = 1.f;
      bool far = false;
      f32x4 qoff = {0.f, 0.f, 0.f, 0.f};
      {
        float v[NK * 2][8];
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < NK * 2; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
          v[i][e] = live ? ll_to_f32(((const T*)raw[i])[e]) : 0.f;
          top = fmaxf(top, fabsf(v[i][e]));
        }
        float up = 1.f;
        if constexpr (BIAS || FAR) {
          top = fmaxf(top, __shfl_xor(top, 16, 64));
          top = fmaxf(top, __shfl_xor(top, 32, 64));
          const int e = max(__builtin_amdgcn_frexp_expf(top), -50);
          if constexpr (BIAS) {
            up = __builtin_ldexpf(1.f, kUp - e);
            cq *= __builtin_ldexpf(1.f, 133 - kUp + min(e, 50));
          } else {
            up = __builtin_ldexpf(1.f, min(50 - e, 0));
          }
          if constexpr (FAR) {
            more = __builtin_ldexpf(1.f, max(e - 50, 0));
            far = __ballot(e > 50) != 0;
          }
        }
#pragma unroll
        for (int i = 0; i < NK * 2; ++i) {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[i][e] *= up;
          split8<NQ>(v[i], qf[i]);
        }
      }
      bf16x8 c128;  // 128 2^-133
      {
        const u32x4 w = {0x00800080u, 0x00800080u, 0x00800080u, 0x00800080u};
        c128 = __builtin_bit_cast(bf16x8, w);
      }
      if constexpr (BIAS) {
#pragma unroll
        for (int i = 0; i < NK * 2; ++i)
#pragma unroll
          for (int p = 0; p < NQ; ++p) qoff = mfma16(c128, qf[i][p], qoff);
        qoff = -qoff;
      }

      f32x4 acc[NV] = {}, off = {0.f, 0.f, 0.f, 0.f};
      float m = -INFINITY, l = 0.f;
      float up = 1.f, limit = BIAS ? -1.f : INFINITY;  // of V scales; up: their power of two
      int down = 0;                                    // and what takes it back, 2^(73 + down)
      const auto compute = [&](Tile8<D>& f) {
        const float scale = f.see >> tok & 1u ? f.scale : 0.f;
        if constexpr (BIAS) {
          if (__ballot(kv == 1 && scale > limit)) {  // the first tile, or scales 2^40 times larger
            const float top = ll_wave_max(kv == 1 ? scale : 0.f);
            const int e = min(max(__builtin_amdgcn_frexp_expf(top), -60), 100);
            const float nu = __builtin_ldexpf(1.f, kUp - e), r = nu / up;
#pragma unroll
            for (int i = 0; i < NV; ++i) acc[i] *= r;
            off *= r;
            up = nu;
            down = e;
            limit = __builtin_ldexpf(1.f, min(e + 40, 127));
          }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        s_scale[wave][kv][tok] = kv ? scale * up : scale;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        float x[8];
#pragma unroll
        for (int grp = 0; grp < 2; ++grp) {
          f32x4 s = qoff;
#pragma unroll
          for (int i = 0; i < NK * 2; ++i) {
            uint32_t w0 = f.kw[grp][i >> 1][2 * (i & 1)], w1 = f.kw[grp][i >> 1][2 * (i & 1) + 1];
            if constexpr (BIAS) {
              w0 ^= 0x80808080u;
              w1 ^= 0x80808080u;
            }
            const bf16x8 kf = codes8<CODE, BIAS>(w0, w1);
#pragma unroll
            for (int p = 0; p < NQ; ++p) s = mfma16(kf, qf[i][p], s);
          }
          const f32x4 ks = *(const f32x4*)&s_scale[wave][0][grp * 16 + g * 4];
#pragma unroll
          for (int r = 0; r < 4; ++r) x[grp * 4 + r] = s[r] * cq * ks[r];
        }
        // the last tile, slots that are none, or queries that were held smaller
        const bool part = f.see != 0xffffffffu || far;
        if (part) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const bool is = f.see >> ((j >> 2) * 16 + g * 4 + (j & 3)) & 1u;
            x[j] = is ? x[j] * more : -INFINITY;
            if constexpr (CODE == KV8_E4M3) {  // (what is in no token's row may be NaN)
#pragma unroll
              for (int i = 0; i < NK; ++i) f.vw[i][j] = is ? f.vw[i][j] : 0u;
            }
          }
        }
        float mt = x[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) mt = fmaxf(mt, x[j]);
        mt = fmaxf(mt, __shfl_xor(mt, 16, 64));
        mt = fmaxf(mt, __shfl_xor(mt, 32, 64));
        if (__ballot(mt > m)) {
          const float mn = fmaxf(m, mt);
          const float alpha = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
          m = mn;
          l *= alpha;
#pragma unroll
          for (int i = 0; i < NV; ++i) acc[i] *= alpha;
          off *= alpha;
        }
        const float ms = m == -INFINITY ? 0.f : m;
        float pv[8];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const f32x4 vs = *(const f32x4*)&s_scale[wave][1][half * 16 + g * 4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float p = __builtin_amdgcn_exp2f(x[half * 4 + r] - ms);
            l += p;
            pv[half * 4 + r] = p * vs[r];
          }
        }
        bf16x8 pf[NP];
        split8<NP>(pv, pf);
        if constexpr (BIAS) {
#pragma unroll
          for (int p = 0; p < NP; ++p) off = mfma16(c128, pf[p], off);
        }
#pragma unroll
        for (int i = 0; i < NK; ++i) {
          if constexpr (BIAS) {
#pragma unroll
            for (int j = 0; j < 8; ++j) f.vw[i][j] ^= 0x80808080u;
          }
          bf16x8 v0, v1, v2, v3;
          codes_of_rows<CODE, BIAS, 0>(f.vw[i], v0, v1);
          codes_of_rows<CODE, BIAS, 1>(f.vw[i], v2, v3);
#pragma unroll
          for (int p = 0; p < NP; ++p) {
            acc[4 * i + 0] = mfma16(v0, pf[p], acc[4 * i + 0]);
            acc[4 * i + 1] = mfma16(v1, pf[p], acc[4 * i + 1]);
            acc[4 * i + 2] = mfma16(v2, pf[p], acc[4 * i + 2]);
            acc[4 * i + 3] = mfma16(v3, pf[p], acc[4 * i + 3]);
          }
        }
      };

      while (t < t1) {
        if constexpr (kStages > 1) {
#pragma unroll
          for (int s = 0; s < kStages; ++s) {
            fetch(f[(s + kStages - 1) % kStages], t + (kStages - 1) * kStep, next);
            next = entry_of(t + kStages * kStep);
            compute(f[s]);
            t += kStep;
            if (t >= t1) break;
          }
        } else {
          compute(f[0]);
          t += kStep;
          fetch(f[0], t, next);
          next = entry_of(t + kStep);
        }
      }
      if constexpr (BIAS) {
        const float back = __builtin_ldexpf(1.f, 133 - kUp), back2 = __builtin_ldexpf(1.f, down);
#pragma unroll
        for (int i = 0; i < NV; ++i) acc[i] = (acc[i] - off) * back * back2;
      }
      // the waves' sums, by their common maximum
      l += __shfl_xor(l, 16, 64);
      l += __shfl_xor(l, 32, 64);
      if (g == 0) {
        s_m[wave][c16] = m;
        s_l[wave][c16] = l;
      }
      __syncthreads();
      float mm = s_m[0][c16], ll = 0.f;
#pragma unroll
      for (int w = 1; w < kWaves8; ++w) mm = fmaxf(mm, s_m[w][c16]);
      const float mms = mm == -INFINITY ? 0.f : mm;
#pragma unroll
      for (int w = 0; w < kWaves8; ++w)
        ll += s_l[w][c16] * __builtin_amdgcn_exp2f(s_m[w][c16] - mms);
      const float mine = __builtin_amdgcn_exp2f(m - mms);
#pragma unroll
      for (int i = 0; i < NV; ++i) acc[i] *= mine;
      if (wave > 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i) s_acc[wave - 1][i][lane] = acc[i];
      }
      __syncthreads();
      if (wave == 0 && live) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < kWaves8 - 1; ++j) acc[i] += s_acc[j][i][lane];
        if (split) {
          const int64_t at = (int64_t)(w + b) * a.H + h;
          if (g == 0) a.part_ml[at] = make_float2(mm, ll);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            f32x4* o = (f32x4*)(a.part + at * D + (g * 4 + r) * NV);
#pragma unroll
            for (int i = 0; i < NK; ++i)
              o[i] = (f32x4){acc[4 * i][r], acc[4 * i + 1][r], acc[4 * i + 2][r],
                             acc[4 * i + 3][r]};
          }
        } else {
          T* out = (T*)a.out + b * a.o_sb + h * a.o_sh;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            T y[NV];
#pragma unroll
            for (int i = 0; i < NV; ++i) y[i] = ll_from_f32<T>(ll == 0.f ? 0.f : acc[i][r] / ll);
            T* o = out + (g * 4 + r) * NV;
            if (a.ovec) {
              constexpr int kBytes = sizeof(T) * NV;
              __builtin_memcpy(__builtin_assume_aligned(o, kBytes < 16 ? kBytes : 16), y, kBytes);
            } else {
#pragma unroll
              for (int i = 0; i < NV; ++i) o[i] = y[i];
            }
          }
        }
      }
    }
    if (left <= 0 || ++b >= a.B) return;
    step = 0;
    n = decode_len(a, b, &row);
  }
}

// The parts of a request, and the zero rows of an empty one. A workgroup has 4 L
// elements of its heads, L threads every (256 / L)-th part, 8 parts' loads at a
// time: a chain of round trips, 5 us (one request of 256 parts: 5.7 with L = 8, 11
// with 64).
template <typename T, int D, int L>
__global__ __launch_bounds__(256) void merge_kernel(DecodeArgs8 a) {
  constexpr int kRows = 256 / L;
  __shared__ f32x4 s_acc[kRows][L];
  __shared__ float s_m[kRows][L], s_l[kRows][L];
  const int tid = threadIdx.x, lane = tid % L, wave = tid / L;
  const int cols = (a.H * D + 4 * L - 1) / (4 * L);
  const int b = blockIdx.x / cols, at = blockIdx.x % cols * (4 * L) + lane * 4;
  const bool in = at < a.H * D;
  const int h = in ? at / D : 0, d = at % D;
  int64_t row;
  const int n = decode_len(a, b, &row);
  T* o = (T*)a.out + b * a.o_sb + h * a.o_sh + d;
  if (n == 0) {
    if (wave == 0 && in)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = ll_from_f32<T>(0.f);
    return;
  }
  const int2 parts = a.meta[b];
  const int first = uniform(parts.x), ns = uniform(parts.y);
  if (ns == 1) return;
  const float2* ml = a.part_ml + (int64_t)first * a.H + h;
  const float* part = a.part + ((int64_t)first * a.H + h) * D + d;
  float m = -INFINITY, l = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int s = wave; s < ns; s += 8 * kRows) {  // 8 parts at a time
    float2 v[8];
    f32x4 x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t p = min(s + kRows * i, ns - 1);
      v[i] = ml[p * a.H];
      x[i] = *(const f32x4*)(part + p * a.H * D);
    }
    float mn = m;
#pragma unroll
    for (int i = 0; i < 8; ++i) mn = fmaxf(mn, v[i].x);
    const float ms = mn == -INFINITY ? 0.f : mn, alpha = __builtin_amdgcn_exp2f(m - ms);
    m = mn;
    l *= alpha;
    acc *= alpha;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float f = s + kRows * i < ns ? __builtin_amdgcn_exp2f(v[i].x - ms) : 0.f;
      l += s + kRows * i < ns ? v[i].y * f : 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += s + kRows * i < ns ? x[i][e] * f : 0.f;
    }
  }
  s_m[wave][lane] = m;
  s_l[wave][lane] = l;
  s_acc[wave][lane] = acc;
  __syncthreads();
  if (wave > 0 || !in) return;
  float mm = m;
#pragma unroll
  for (int i = 1; i < kRows; ++i) mm = fmaxf(mm, s_m[i][lane]);
  const float ms = mm == -INFINITY ? 0.f : mm, f0 = __builtin_amdgcn_exp2f(m - ms);
  l *= f0;
  acc *= f0;
#pragma unroll
  for (int i = 1; i < kRows; ++i) {
    const float f = __builtin_amdgcn_exp2f(s_m[i][lane] - ms);
    l += s_l[i][lane] * f;
    acc += s_acc[i][lane] * f;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = ll_from_f32<T>(l == 0.f ? 0.f : acc[e] / l);
}

constexpr int64_t kMaxGrid8 = (1 << 24) - 1;  // of 256 threads: fewer than 2^32
constexpr int kPlaces = 512;                  // workgroups that run at a time: two per CU

// Workgroups of a call per head block; bytes: of the parts (0: no request is split)
struct Plan8 {
  int64_t W, heads, bytes;
  bool whole;
};

bool plan8(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t max_len,
           Plan8* p) {
  if (batch <= 0 || batch > 1 << 24 || kv_heads <= 0 || kv_heads > 65535 || q_heads <= 0 ||
      q_heads > 65535 || q_heads % kv_heads != 0 || max_len <= 0 || max_len > 1 << 30 ||
      (head_dim != 64 && head_dim != 128 && head_dim != 256))
    return false;
  p->heads = kv_heads * ((q_heads / kv_heads + 15) / 16);
  const int64_t steps = (max_len + kStep8 - 1) / kStep8;  // of a request at most
  // Short contexts take a workgroup per request and head block, which needs no list,
  // no parts and no second launch (us, so and dealt out: 40 x 600 tokens of 2 KV
  // heads 13.1, 15.8; 1 x 300 9.3, 11.7; 100 x up to 1000 of 4 27.3, 33.1; 128 x up
  // to 2000 of 2 18.6, 21.1), unless longer ones would leave CUs idle (8 x up to
  // 1000 of 2: 14.1, 12.9).
  p->whole = steps <= 6 || (steps <= 16 && batch * p->heads >= 64);
  p->W = batch;
  if (!p->whole)  // (at least one, where the head blocks alone are more than the places)
    p->W = std::min(std::max<int64_t>({kPlaces / p->heads, batch / 4, 1}), batch * steps);
  p->bytes = p->whole ? 0 : (p->W + batch) * q_heads * (head_dim * 4 + 8) + batch * 8;
  return (p->W + 7) / 8 * 8 * p->heads <= kMaxGrid8 && batch * steps <= INT32_MAX &&
         batch * ((q_heads * head_dim + 255) / 256) <= kMaxGrid8;
}

template <typename T, int CODE, int D>
int launch_decode(const DecodeArgs8& a, unsigned grid, hipStream_t stream) {
  hipLaunchKernelGGL((decode_mfma_kernel<T, CODE, D>), dim3(grid), dim3(kWaves8 * 64), 0, stream,
                     a);
  // (no merge of what a launch that failed has not written)
  if (!a.whole && hipPeekAtLastError() == hipSuccess) {
    // few requests have many parts each: more threads along those
    if (a.B <= 8)
      hipLaunchKernelGGL((merge_kernel<T, D, 8>), dim3((unsigned)(a.B * ((a.H * D + 31) / 32))),
                         dim3(256), 0, stream, a);
    else
      hipLaunchKernelGGL((merge_kernel<T, D, 64>), dim3((unsigned)(a.B * ((a.H * D + 255) / 256))),
                         dim3(256), 0, stream, a);
  }
  LL_RETURN_LAUNCH();
}

// log2 of a block size, -1 for others
int block_shift(int64_t block) {
  for (int s = 0; s <= 7; ++s)
    if (block == (int64_t)1 << s) return s;
  return -1;
}

// f with the code kind as a compile-time constant
template <typename F> int dispatch_code(int code, F f) {
  if (code == KV8_INT8) return f(std::integral_constant<int, KV8_INT8>());
  return f(std::integral_constant<int, KV8_E4M3>());
}

#define KV8_CHECK_FORM(fn)                                                                     \
  LL_CHECK_ARG(code == KV8_INT8 || code == KV8_E4M3, "%s: code kind %d", fn, code);           \
  LL_CHECK_ARG(block_shift(block) >= 0, "%s: block %lld is no power of two up to 128", fn,    \
               (long long)block);                                                             \
  LL_CHECK_ARG(slots_n >= 0 && slots_n <= INT32_MAX, "%s: %lld slots", fn, (long long)slots_n); \
  LL_CHECK_ARG(kv_heads > 0 && kv_heads <= 65535, "%s: %lld KV heads", fn, (long long)kv_heads)

// whether n rows this far apart are rows of their own
bool apart(int64_t stride, int64_t n) { return n < 2 || stride != 0; }

bool aligned(int64_t bytes, std::initializer_list<int64_t> vs) {
  for (int64_t v : vs)
    if (v % bytes != 0) return false;
  return true;
}

}  // namespace

extern "C" int ll_kv8_store(const void* k, int64_t k_stride_tok, int64_t k_stride_h, const void* v,
                            int64_t v_stride_tok, int64_t v_stride_h, const int32_t* slots,
                            int64_t ntok, int64_t kv_heads, int64_t head_dim, void* k_codes,
                            int64_t kc_stride_tok, int64_t kc_stride_h, void* v_codes,
                            int64_t vc_stride_tok, int64_t vc_stride_h, float* k_scale,
                            int64_t ks_stride_block, int64_t ks_stride_h, float* v_scale,
                            int64_t vs_stride_block, int64_t vs_stride_h, int64_t slots_n,
                            int64_t block, int code, int dtype, hipStream_t stream) {
  const char* fn = "ll_kv8_store";
  if (ntok == 0) return LL_OK;
  LL_CHECK_ARG(k && v && slots && k_codes && v_codes && k_scale && v_scale, "%s: null pointer", fn);
  KV8_CHECK_FORM(fn);
  LL_CHECK_ARG(ntok > 0 && ntok <= 1 << 24, "%s: %lld tokens (max 2^24)", fn, (long long)ntok);
  LL_CHECK_ARG(head_dim > 0 && head_dim <= 1024, "%s: head_dim %lld unsupported", fn,
               (long long)head_dim);
  LL_CHECK_ARG(apart(kc_stride_tok, slots_n) && apart(kc_stride_h, kv_heads) &&
                   apart(vc_stride_tok, slots_n) && apart(vc_stride_h, kv_heads) &&
                   apart(ks_stride_block, (slots_n + block - 1) / block) &&
                   apart(ks_stride_h, kv_heads) &&
                   apart(vs_stride_block, (slots_n + block - 1) / block) &&
                   apart(vs_stride_h, kv_heads),
               "%s: rows or heads of the cache share an address (stride 0)", fn);
  StoreArgs a;
  a.x[0] = k; a.x_st[0] = k_stride_tok; a.x_sh[0] = k_stride_h;
  a.x[1] = v; a.x_st[1] = v_stride_tok; a.x_sh[1] = v_stride_h;
  a.slots = slots;
  a.c[0] = (uint8_t*)k_codes; a.c_st[0] = kc_stride_tok; a.c_sh[0] = kc_stride_h;
  a.c[1] = (uint8_t*)v_codes; a.c_st[1] = vc_stride_tok; a.c_sh[1] = vc_stride_h;
  a.s[0] = k_scale; a.s_sb[0] = ks_stride_block; a.s_sh[0] = ks_stride_h;
  a.s[1] = v_scale; a.s_sb[1] = vs_stride_block; a.s_sh[1] = vs_stride_h;
  a.T = ntok; a.nslots = slots_n;
  a.KVH = (int)kv_heads; a.D = (int)head_dim; a.shift = block_shift(block);
  const int64_t units = 2 * kv_heads;
  // Few tokens (a decode step, a run each): a wave for each, so that no run waits
  // for another. Many: up to a block's tokens per wave, since a wave whose tokens
  // start no run still reads their slots.
  a.per = 1;
  while (a.per < block && a.per < 64 && ntok * units / a.per >= kStoreFill) a.per *= 2;
  int lpr = 1;
  while (lpr * 8 < head_dim && lpr < 64) lpr *= 2;
  // (a run of 32 rows and more takes four waves)
  const int team = block >= kTeamBlock ? 4 : 1;
  const int64_t waves = block == 1 ? (ntok * units + 64 / lpr - 1) / (64 / lpr)
                                   : (ntok + a.per - 1) / a.per * units * team;
  LL_CHECK_ARG(waves <= (int64_t)INT32_MAX / 64 && ntok * units <= INT32_MAX - 64,
               "%s: %lld tokens of %lld heads", fn, (long long)ntok, (long long)kv_heads);
  const int es = dtype == LL_F32 ? 4 : 2;
  const bool vec = head_dim % 8 == 0 &&
                   aligned(16, {(int64_t)(uintptr_t)k, (int64_t)(uintptr_t)v, k_stride_tok * es,
                                k_stride_h * es, v_stride_tok * es, v_stride_h * es}) &&
                   aligned(8, {(int64_t)(uintptr_t)k_codes, (int64_t)(uintptr_t)v_codes,
                               kc_stride_tok, kc_stride_h, vc_stride_tok, vc_stride_h});
  const dim3 grid((unsigned)((waves + kStoreWaves - 1) / kStoreWaves));
  return LL_DISPATCH_DTYPE(dtype, T, [&]() -> int {
    return dispatch_code(code, [&](auto C) -> int {
      constexpr int CODE = decltype(C)::value;
      const dim3 threads(kStoreWaves * 64);
      if (block == 1 && vec)
        hipLaunchKernelGGL((store_rows_kernel<T, CODE, true>), grid, threads, 0, stream, a);
      else if (block == 1)
        hipLaunchKernelGGL((store_rows_kernel<T, CODE, false>), grid, threads, 0, stream, a);
      else if (team == 1 && vec)
        hipLaunchKernelGGL((store_kernel<T, CODE, true, 1>), grid, threads, 0, stream, a);
      else if (team == 1)
        hipLaunchKernelGGL((store_kernel<T, CODE, false, 1>), grid, threads, 0, stream, a);
      else if (vec)
        hipLaunchKernelGGL((store_kernel<T, CODE, true, 4>), grid, threads, 0, stream, a);
      else
        hipLaunchKernelGGL((store_kernel<T, CODE, false, 4>), grid, threads, 0, stream, a);
      LL_RETURN_LAUNCH();
    });
  });
}

extern "C" int ll_kv8_load(const void* k_codes, int64_t kc_stride_tok, int64_t kc_stride_h,
                           const void* v_codes, int64_t vc_stride_tok, int64_t vc_stride_h,
                           const float* k_scale, int64_t ks_stride_block, int64_t ks_stride_h,
                           const float* v_scale, int64_t vs_stride_block, int64_t vs_stride_h,
                           int64_t slots_n, int64_t block, int code, const int32_t* req_to_tokens,
                           int64_t req_to_tokens_stride, int64_t req_rows, const void* b_req_idx,
                           int req_idx_i64, const void* b_start_loc, int start_loc_i64,
                           const void* b_seq_len, int seq_len_i64, int64_t batch,
                           int64_t max_len_in_batch, void* k_out, int64_t ko_stride_tok,
                           int64_t ko_stride_h, void* v_out, int64_t vo_stride_tok,
                           int64_t vo_stride_h, int64_t out_rows, int64_t kv_heads,
                           int64_t head_dim, int dtype, hipStream_t stream) {
  const char* fn = "ll_kv8_load";
  if (batch == 0 || max_len_in_batch == 0 || out_rows == 0) return LL_OK;
  LL_CHECK_ARG(k_codes && v_codes && k_scale && v_scale && req_to_tokens && b_req_idx &&
                   b_start_loc && b_seq_len && k_out && v_out,
               "%s: null pointer", fn);
  KV8_CHECK_FORM(fn);
  LL_CHECK_ARG(batch > 0 && batch <= 65535, "%s: %lld requests (max 65535)", fn, (long long)batch);
  LL_CHECK_ARG(max_len_in_batch > 0 && max_len_in_batch <= 1 << 30 && out_rows > 0,
               "%s: max_len_in_batch %lld, %lld output rows", fn, (long long)max_len_in_batch,
               (long long)out_rows);
  LL_CHECK_ARG(head_dim > 0 && head_dim <= 1024, "%s: head_dim %lld unsupported", fn,
               (long long)head_dim);
  LL_CHECK_ARG(apart(ko_stride_tok, out_rows) && apart(ko_stride_h, kv_heads) &&
                   apart(vo_stride_tok, out_rows) && apart(vo_stride_h, kv_heads),
               "%s: rows or heads of the output share an address (stride 0)", fn);
  LoadArgs a;
  a.c[0] = (const uint8_t*)k_codes; a.c_st[0] = kc_stride_tok; a.c_sh[0] = kc_stride_h;
  a.c[1] = (const uint8_t*)v_codes; a.c_st[1] = vc_stride_tok; a.c_sh[1] = vc_stride_h;
  a.s[0] = k_scale; a.s_sb[0] = ks_stride_block; a.s_sh[0] = ks_stride_h;
  a.s[1] = v_scale; a.s_sb[1] = vs_stride_block; a.s_sh[1] = vs_stride_h;
  a.r2t = req_to_tokens; a.r2t_s = req_to_tokens_stride; a.r2t_rows = req_rows;
  a.req = b_req_idx; a.req64 = req_idx_i64;
  a.start = b_start_loc; a.start64 = start_loc_i64;
  a.len = b_seq_len; a.len64 = seq_len_i64;
  a.o[0] = k_out; a.o_st[0] = ko_stride_tok; a.o_sh[0] = ko_stride_h;
  a.o[1] = v_out; a.o_st[1] = vo_stride_tok; a.o_sh[1] = vo_stride_h;
  a.nslots = slots_n; a.orows = out_rows;
  a.KVH = (int)kv_heads; a.D = (int)head_dim; a.shift = block_shift(block);
  a.max_len = (int)max_len_in_batch;
  const int es = dtype == LL_F32 ? 4 : 2;
  const bool vec =
      head_dim % 16 == 0 &&
      aligned(16, {(int64_t)(uintptr_t)k_codes, (int64_t)(uintptr_t)v_codes, kc_stride_tok,
                   kc_stride_h, vc_stride_tok, vc_stride_h, (int64_t)(uintptr_t)k_out,
                   (int64_t)(uintptr_t)v_out, ko_stride_tok * es, ko_stride_h * es,
                   vo_stride_tok * es, vo_stride_h * es});
  a.pieces = vec ? a.D / 16 : a.D;
  const int64_t places = 2 * kv_heads * a.pieces;
  LL_CHECK_ARG(places <= INT32_MAX, "%s: %lld heads of %lld", fn, (long long)kv_heads,
               (long long)head_dim);
  // (tokens of a workgroup's turn)
  const int64_t tokens = std::max<int64_t>(1, kLoadThreads / places) * kLoadTokens;
  const int64_t most = std::max<int64_t>(1, kLoadFill / batch);
  const dim3 grid((unsigned)std::min((max_len_in_batch + tokens - 1) / tokens, most),
                  (unsigned)batch);
  return LL_DISPATCH_DTYPE(dtype, T, [&]() -> int {
    return dispatch_code(code, [&](auto C) -> int {
      constexpr int CODE = decltype(C)::value;
      if (vec)
        hipLaunchKernelGGL((load_kernel<T, CODE, true>), grid, dim3(kLoadThreads), 0, stream, a);
      else
        hipLaunchKernelGGL((load_kernel<T, CODE, false>), grid, dim3(kLoadThreads), 0, stream, a);
      LL_RETURN_LAUNCH();
    });
  });
}

extern "C" int64_t ll_kv8_decode_attention_workspace_size(int64_t batch, int64_t q_heads,
                                                          int64_t kv_heads, int64_t head_dim,
                                                          int64_t max_len_in_batch) {
  Plan8 p;
  return plan8(batch, q_heads, kv_heads, head_dim, max_len_in_batch, &p) ? p.bytes : 0;
}

extern "C" int ll_kv8_decode_attention(
    const void* q, int64_t q_stride_b, int64_t q_stride_h, const void* k_codes,
    int64_t kc_stride_tok, int64_t kc_stride_h, const void* v_codes, int64_t vc_stride_tok,
    int64_t vc_stride_h, const float* k_scale, int64_t ks_stride_block, int64_t ks_stride_h,
    const float* v_scale, int64_t vs_stride_block, int64_t vs_stride_h, int64_t slots_n,
    int64_t block, int code, const int32_t* req_to_tokens, int64_t req_to_tokens_stride,
    int64_t req_rows, const void* b_req_idx, int req_idx_i64, const void* b_seq_len,
    int seq_len_i64, void* out, int64_t out_stride_b, int64_t out_stride_h, int64_t batch,
    int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t max_len_in_batch, float sm_scale,
    int dtype, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  const char* fn = "ll_kv8_decode_attention";
  if (batch == 0) return LL_OK;
  LL_CHECK_ARG(q && k_codes && v_codes && k_scale && v_scale && req_to_tokens && b_req_idx &&
                   b_seq_len && out,
               "%s: null pointer", fn);
  KV8_CHECK_FORM(fn);
  LL_CHECK_ARG(batch > 0 && batch <= 1 << 24 && q_heads > 0 && q_heads <= 65535 &&
                   q_heads % kv_heads == 0,
               "%s: %lld requests of %lld query and %lld KV heads", fn, (long long)batch,
               (long long)q_heads, (long long)kv_heads);
  LL_CHECK_ARG(head_dim > 0 && head_dim <= kAnyMaxD, "%s: head_dim %lld unsupported", fn,
               (long long)head_dim);
  LL_CHECK_ARG(max_len_in_batch >= 0 && max_len_in_batch <= 1 << 30,
               "%s: max_len_in_batch %lld out of range", fn, (long long)max_len_in_batch);
  LL_CHECK_ARG(sm_scale > 0.f && sm_scale < INFINITY, "%s: sm_scale %g must be positive", fn,
               (double)sm_scale);
  LL_CHECK_ARG(apart(out_stride_b, batch) && apart(out_stride_h, q_heads),
               "%s: rows or heads of the output share an address (stride 0)", fn);
  DecodeArgs8 a;
  a.q = q; a.q_sb = q_stride_b; a.q_sh = q_stride_h;
  a.c[0] = (const uint8_t*)k_codes; a.c_st[0] = kc_stride_tok; a.c_sh[0] = kc_stride_h;
  a.c[1] = (const uint8_t*)v_codes; a.c_st[1] = vc_stride_tok; a.c_sh[1] = vc_stride_h;
  a.s[0] = k_scale; a.s_sb[0] = ks_stride_block; a.s_sh[0] = ks_stride_h;
  a.s[1] = v_scale; a.s_sb[1] = vs_stride_block; a.s_sh[1] = vs_stride_h;
  a.r2t = req_to_tokens; a.r2t_s = req_to_tokens_stride; a.r2t_rows = req_rows;
  a.req = b_req_idx; a.req64 = req_idx_i64;
  a.len = b_seq_len; a.len64 = seq_len_i64;
  a.out = out; a.o_sb = out_stride_b; a.o_sh = out_stride_h;
  a.nslots = slots_n;
  a.B = (int)batch; a.H = (int)q_heads; a.KVH = (int)kv_heads; a.G = (int)(q_heads / kv_heads);
  a.D = (int)head_dim; a.shift = block_shift(block); a.max_len = (int)max_len_in_batch;
  a.scale_log2 = sm_scale * 1.4426950408889634f;
  const int es = dtype == LL_F32 ? 4 : 2;
  Plan8 p;
  const bool planned = plan8(batch, q_heads, kv_heads, head_dim, max_len_in_batch, &p);
  // (a cache without slots has no row that a masked token's lanes could read)
  const bool mfma =
      planned && slots_n > 0 &&
      aligned(16, {(int64_t)(uintptr_t)k_codes, (int64_t)(uintptr_t)v_codes, kc_stride_tok,
                   kc_stride_h, vc_stride_tok, vc_stride_h});
  if (mfma) {
    a.hb = (a.G + 15) / 16;
    a.W = (int)p.W; a.whole = p.whole;
    a.qvec = aligned(16, {(int64_t)(uintptr_t)q, q_stride_b * es, q_stride_h * es});
    a.ovec = aligned(16, {(int64_t)(uintptr_t)out, out_stride_b * es, out_stride_h * es});
    std::unique_lock<std::mutex> lock;
    if (p.bytes > 0) {
      LL_CHECK_ARG(workspace && workspace_bytes >= p.bytes && (uintptr_t)workspace % 16 == 0,
                   "%s: the workspace needs %lld bytes, 16 B aligned, got %lld", fn,
                   (long long)p.bytes, (long long)workspace_bytes);
      a.part = (float*)workspace;
      a.part_ml = (float2*)((char*)workspace + (p.W + batch) * q_heads * head_dim * 4);
      a.meta = (int2*)(a.part_ml + (p.W + batch) * q_heads);
      // no other thread's call on this workspace between the two launches
      lock = std::unique_lock<std::mutex>(ll_workspace_mutex(workspace));
    }
    const unsigned grid = (unsigned)((p.W + 7) / 8 * 8 * p.heads);
    return LL_DISPATCH_DTYPE(dtype, T, [&]() -> int {
      return dispatch_code(code, [&](auto C) -> int {
        constexpr int CODE = decltype(C)::value;
        if (head_dim == 64) return launch_decode<T, CODE, 64>(a, grid, stream);
        if (head_dim == 128) return launch_decode<T, CODE, 128>(a, grid, stream);
        return launch_decode<T, CODE, 256>(a, grid, stream);
      });
    });
  }
  LL_CHECK_ARG(batch * q_heads <= INT32_MAX / 64, "%s: %lld requests of %lld heads", fn,
               (long long)batch, (long long)q_heads);
  return LL_DISPATCH_DTYPE(dtype, T, [&]() -> int {
    return dispatch_code(code, [&](auto C) -> int {
      constexpr int CODE = decltype(C)::value;
      hipLaunchKernelGGL((decode_any_kernel<T, CODE>), dim3((unsigned)(batch * q_heads)), dim3(64),
                         0, stream, a);
      LL_RETURN_LAUNCH();
    });
  });
}
