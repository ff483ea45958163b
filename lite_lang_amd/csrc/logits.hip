// Controls on the logits that a token is taken from (gfx950): penalties for
// repeated tokens, biases and a mask of the allowed tokens, in one pass.
//
// For token v of request b, with x its logit:
//   seen:  v is among tokens[0 .. seq_len)          (prompt and answer)
//   count: how often v is among tokens[prompt_len .. seq_len)   (the answer)
//   x = seen ? (x > 0 ? x / repetition : x * repetition) : x
//   x = x - frequency * count - (count > 0 ? presence : 0)
//   x = x + w, w the sum of the biases of v, added up in their order
//   x = -inf where the mask's bit v is 0
// in fp32, each operation rounded, and one rounding to the logits' type.
//
// A workgroup takes a stretch of the vocabulary of one request, counts in LDS
// what of the request's tokens falls into it (integer additions: no order
// changes them), and writes its logits once: bound by memory at 40 requests of
// 151,936 logits (13.5 us, 3.7 TB/s). One request of 131,072 tokens takes 17.6 us:
// every one of its 19 workgroups reads all tokens, 8.8 us (so long with ids that
// fall into none), and counting those of its stretch takes the rest, whether they
// are spread evenly (16.0) or as in a text; 115 where all are one token, whose
// additions to one LDS word follow each other.
#include <algorithm>

#include "ll_common.h"

namespace {

constexpr int kEach = 8;  // logits of a thread
constexpr uint32_t kSeen = 0x80000000u;           // the token is in the prompt
constexpr uint32_t kBiased = 0x40000000u;         // it has a bias
constexpr uint32_t kCount = kBiased - 1;

struct LogitArgs {
  const void* x; int64_t ldx;
  void* y; int64_t ldy;
  int64_t V;
  const int32_t* tok; int64_t tok_s, tok_rows, tok_cols;
  const void* req; int req64;
  const void* plen; int plen64;
  const void* len; int len64;
  const float* rep; const float* freq; const float* pres;
  const int32_t* bias_id; const float* bias; int64_t nb, bias_s, biasv_s;
  const uint32_t* mask; int64_t mask_s;
};

// VEC: rows of 16-byte alignment. The logits are on their way while the tokens
// are counted.
template <typename T, bool VEC, int THREADS>
__global__ __launch_bounds__(THREADS) void logits_kernel(LogitArgs a) {
#pragma clang fp contract(off)
  constexpr int kSpan = THREADS * kEach;  // tokens of the vocabulary per workgroup
  constexpr int kVec = 16 / sizeof(T), kLoads = kEach / kVec;
  __shared__ __align__(16) uint32_t cnt[kSpan];
  __shared__ __align__(16) float bias[kSpan];
  __shared__ int twice;
  const int b = blockIdx.y, tid = threadIdx.x;
  const int64_t v0 = (int64_t)blockIdx.x * kSpan;
  const int n = (int)min((int64_t)kSpan, a.V - v0);
  const T* x = (const T*)a.x + b * a.ldx + v0;
  T* y = (T*)a.y + b * a.ldy + v0;
  // a thread's elements: kVec next to each other in each of kLoads places
  const auto place = [&](int k, int e) { return (k * THREADS + tid) * kVec + e; };
  T in[kLoads][kVec];
#pragma unroll
  for (int k = 0; k < kLoads; ++k) {
    if (VEC && place(k, kVec - 1) < n) {
      *(u32x4*)in[k] = *(const u32x4*)(x + place(k, 0));
    } else {
#pragma unroll
      for (int e = 0; e < kVec; ++e) in[k][e] = place(k, e) < n ? x[place(k, e)] : (T)0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < kEach / 4; ++i) ((u32x4*)cnt)[i * THREADS + tid] = (u32x4){0, 0, 0, 0};
  if (tid == 0) twice = 0;
  __syncthreads();
  if (a.tok) {
    const int64_t row = ll_load_idx(a.req, b, a.req64);
    int64_t len64 = ll_load_idx(a.len, b, a.len64);
    const int64_t p64 = ll_load_idx(a.plen, b, a.plen64);
    if (row < 0 || row >= a.tok_rows || len64 < 0) len64 = 0;
    const int len = (int)min(len64, a.tok_cols), plen = (int)max(min(p64, a.tok_cols), (int64_t)0);
    const int32_t* t = a.tok + (len > 0 ? row : 0) * a.tok_s;
    const auto count = [&](int i, uint32_t at) {
      if (at < (uint32_t)n) {
        if (i < plen) atomicOr(&cnt[at], kSeen);
        else atomicAdd(&cnt[at], 1u);
      }
    };
    // four tokens at a time between the row's 16-byte addresses
    const int head = min(len, (int)((16 - ((uintptr_t)t & 15)) / 4 & 3));
    const int quads = (len - head) / 4;
    const i32x4* tq = (const i32x4*)(t + head);
    const uint32_t low = (uint32_t)v0;
    if (tid < head) count(tid, (uint32_t)t[tid] - low);
    const int rest = head + quads * 4;
    if (tid < len - rest) count(rest + tid, (uint32_t)t[rest + tid] - low);
    for (int q = tid; q < quads; q += 4 * THREADS) {
      i32x4 v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = tq[min(q + k * THREADS, quads - 1)];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t c0 = (uint32_t)v[k][0] - low, c1 = (uint32_t)v[k][1] - low;
        const uint32_t c2 = (uint32_t)v[k][2] - low, c3 = (uint32_t)v[k][3] - low;
        if (q + k * THREADS < quads && min(min(c0, c1), min(c2, c3)) < (uint32_t)n) {
          const int i = head + (q + k * THREADS) * 4;
          count(i, c0);
          count(i + 1, c1);
          count(i + 2, c2);
          count(i + 3, c3);
        }
      }
    }
  }
  const int32_t* ids = a.bias_id + b * a.bias_s;
  const float* vals = a.bias + b * a.biasv_s;
  const int nb = (int)a.nb;
  for (int i = tid; i < nb; i += THREADS) {
    const uint32_t at = (uint32_t)ids[i] - (uint32_t)v0;
    if (at < (uint32_t)n && atomicOr(&cnt[at], kBiased) & kBiased) twice = 1;
  }
  if (nb > 0) {
    __syncthreads();
    if (!twice) {
      for (int i = tid; i < nb; i += THREADS) {
        const uint32_t at = (uint32_t)ids[i] - (uint32_t)v0;
        if (at < (uint32_t)n) bias[at] = vals[i];
      }
    } else {
      // Tokens with several: a wave goes through the list in its order and adds up
      // those of its 64 kEach tokens, so that the time grows with the list alone
      // (2^20 entries for 151,936 tokens: 3.0 ms, all of them for one: 38; 300 for
      // 50 tokens: 26 us).
      const int lane = tid & 63, first = (tid >> 6) * (64 * kEach);
#pragma unroll
      for (int k = 0; k < kEach; ++k) bias[first + k * 64 + lane] = -0.f;  // (-0 + v is v)
      constexpr int kAhead = 4;
      for (int i0 = 0; i0 < nb; i0 += kAhead * 64) {
        uint32_t at[kAhead];
        float v[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          const int i = min(i0 + k * 64 + lane, nb - 1);
          at[k] = (uint32_t)ids[i] - (uint32_t)v0;
          v[k] = vals[i];
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          uint64_t todo = __ballot(i0 + k * 64 + lane < nb && at[k] < (uint32_t)n &&
                                   at[k] - (uint32_t)first < 64u * kEach);
          while (todo) {
            const int one = __builtin_amdgcn_readlane((int)at[k], __builtin_ctzll(todo));
            uint64_t same = __ballot(at[k] == (uint32_t)one) & todo;
            todo &= ~same;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            float s = bias[one];
            for (; same; same &= same - 1)
              s = s + __builtin_bit_cast(
                          float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v[k]),
                                                           __builtin_ctzll(same)));
            if (lane == 0) bias[one] = s;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          }
        }
      }
    }
  }
  __syncthreads();
  const float rep = a.rep ? a.rep[b] : 1.f, freq = a.freq ? a.freq[b] : 0.f,
              pres = a.pres ? a.pres[b] : 0.f;
  const uint32_t* mask = a.mask ? a.mask + b * a.mask_s + v0 / 32 : nullptr;
#pragma unroll
  for (int k = 0; k < kLoads; ++k) {
    const int p = place(k, 0);
    if (p >= n) continue;
    // (the elements of a place lie in one word of the mask)
    const uint32_t allowed = mask ? mask[p >> 5] >> (p & 31) : ~0u;
    uint32_t c[kVec];
#pragma unroll
    for (int e = 0; e < kVec; e += 4) *(u32x4*)(c + e) = *(const u32x4*)&cnt[p + e];
    T out[kVec];
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      float v = ll_to_f32(in[k][e]);
      if (c[e] & (kSeen | kCount)) {
        if (a.rep) v = v > 0.f ? v / rep : v * rep;
        const uint32_t said = c[e] & kCount;
        v = v - freq * (float)said;
        v = v - (said ? pres : 0.f);
      }
      if (c[e] & kBiased) v = v + bias[p + e];
      if (!(allowed >> e & 1u)) v = -INFINITY;
      out[e] = ll_from_f32<T>(v);
    }
    if (VEC && place(k, kVec - 1) < n) {
      __builtin_nontemporal_store(*(const u32x4*)out, (u32x4*)(y + p));
    } else {
#pragma unroll
      for (int e = 0; e < kVec; ++e)
        if (p + e < n) y[p + e] = out[e];
    }
  }
}

template <typename T, int THREADS>
int launch_logits(const LogitArgs& a, int64_t batch, bool vec, hipStream_t stream) {
  const dim3 grid((unsigned)((a.V + THREADS * kEach - 1) / (THREADS * kEach)), (unsigned)batch);
  if (vec) hipLaunchKernelGGL((logits_kernel<T, true, THREADS>), grid, dim3(THREADS), 0, stream, a);
  else hipLaunchKernelGGL((logits_kernel<T, false, THREADS>), grid, dim3(THREADS), 0, stream, a);
  LL_RETURN_LAUNCH();
}

}  // namespace

extern "C" int ll_adjust_logits(const void* logits, int64_t ld_logits, void* out, int64_t ld_out,
                                int64_t batch, int64_t vocab, const int32_t* tokens,
                                int64_t tokens_stride, int64_t tokens_rows, int64_t tokens_cols,
                                const void* b_req_idx, int req_idx_i64, const void* b_prompt_len,
                                int prompt_len_i64, const void* b_seq_len, int seq_len_i64,
                                const float* repetition, const float* frequency,
                                const float* presence, const int32_t* bias_ids,
                                int64_t bias_ids_stride, const float* bias_values,
                                int64_t bias_values_stride, int64_t n_bias, const uint32_t* mask,
                                int64_t mask_stride, int dtype, hipStream_t stream) {
  const char* fn = "ll_adjust_logits";
  if (batch == 0 || vocab == 0) return LL_OK;
  LL_CHECK_ARG(logits && out, "%s: null pointer", fn);
  LL_CHECK_ARG(!tokens || (b_req_idx && b_prompt_len && b_seq_len),
               "%s: tokens need their rows and lengths", fn);
  LL_CHECK_ARG(tokens || !(repetition || frequency || presence), "%s: penalties need tokens", fn);
  LL_CHECK_ARG(n_bias >= 0 && n_bias <= 1 << 20 && (n_bias == 0 || (bias_ids && bias_values)),
               "%s: %lld biases", fn, (long long)n_bias);
  LL_CHECK_ARG(batch > 0 && batch <= 65535 && vocab > 0 && vocab <= INT32_MAX - (1 << 14),
               "%s: %lld requests (max 65535) of %lld logits", fn, (long long)batch,
               (long long)vocab);
  LL_CHECK_ARG(batch < 2 || ld_out >= vocab, "%s: output rows %lld apart overlap", fn,
               (long long)ld_out);
  LL_CHECK_ARG(!tokens || (tokens_rows >= 0 && tokens_cols >= 0 && tokens_cols <= (int64_t)kCount),
               "%s: %lld tokens", fn, (long long)tokens_cols);
  LogitArgs a;
  a.x = logits; a.ldx = ld_logits;
  a.y = out; a.ldy = ld_out;
  a.V = vocab;
  a.tok = tokens; a.tok_s = tokens_stride; a.tok_rows = tokens_rows; a.tok_cols = tokens_cols;
  a.req = b_req_idx; a.req64 = req_idx_i64;
  a.plen = b_prompt_len; a.plen64 = prompt_len_i64;
  a.len = b_seq_len; a.len64 = seq_len_i64;
  a.rep = repetition; a.freq = frequency; a.pres = presence;
  a.bias_id = bias_ids; a.bias = bias_values; a.nb = n_bias;
  a.bias_s = bias_ids_stride; a.biasv_s = bias_values_stride;
  a.mask = mask; a.mask_s = mask_stride;
  const int es = dtype == LL_F32 ? 4 : 2;
  const bool vec = ((uintptr_t)logits | (uintptr_t)out) % 16 == 0 &&
                   (batch == 1 || (ld_logits * es % 16 == 0 && ld_out * es % 16 == 0));
  // Every workgroup looks through all of its request's tokens, so room for many
  // of those and few workgroups ask for large ones (1 x 131,072 tokens: 18 us with
  // 1024 threads, 36 with 256); else small ones start and end sooner (40 x 300
  // tokens, 50,257 logits in rows of no alignment: 8.9 us with 256, 11.9 with 1024).
  const bool wide = tokens && tokens_cols > 8192 && batch * ((vocab + 2047) / 2048) <= 1024;
  return LL_DISPATCH_DTYPE(dtype, T, [&]() -> int {
    return wide ? launch_logits<T, 1024>(a, batch, vec, stream)
                : launch_logits<T, 256>(a, batch, vec, stream);
  });
}
