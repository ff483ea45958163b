// Controls on the logits that a token is taken from (gfx950): penalties for
// repeated tokens, biases and a mask of the allowed tokens, in one pass.
//
// For token v of request b, with x its logit:
//   seen:  v is among tokens[0 .. seq_len)          (prompt and answer)
//   count: how often v is among tokens[prompt_len .. seq_len)   (the answer)
//   x = seen ? (x > 0 ? x / repetition : x * repetition) : x
//   x = x - frequency * count - (count > 0 ? presence : 0)
//   x = x + the biases of v, in their order
//   x = -inf where the mask's bit v is 0
// in fp32, each operation rounded, and one rounding to the logits' type.
//
// A workgroup takes a stretch of the vocabulary of one request, counts in LDS
// what of the request's tokens falls into it (integer additions: no order
// changes them), and writes its logits once.
#include <algorithm>

#include "ll_common.h"

namespace {

constexpr int kSpan = 4096;  // tokens of the vocabulary per workgroup
constexpr int kLogitThreads = 512;
constexpr uint32_t kSeen = 0x80000000u;  // the token is in the prompt

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

template <typename T>
__global__ __launch_bounds__(kLogitThreads) void logits_kernel(LogitArgs a) {
#pragma clang fp contract(off)
  __shared__ uint32_t cnt[kSpan], nbias[kSpan];
  __shared__ float bias[kSpan];
  const int b = blockIdx.y, tid = threadIdx.x;
  const int64_t v0 = (int64_t)blockIdx.x * kSpan;
  const int n = (int)std::min<int64_t>(kSpan, a.V - v0);
  for (int i = tid; i < n; i += kLogitThreads) {
    cnt[i] = 0;
    nbias[i] = 0;
  }
  __syncthreads();
  if (a.tok) {
    const int64_t row = ll_load_idx(a.req, b, a.req64);
    int64_t len = std::min<int64_t>(ll_load_idx(a.len, b, a.len64), a.tok_cols);
    if (row < 0 || row >= a.tok_rows) len = 0;
    const int64_t plen = ll_load_idx(a.plen, b, a.plen64);
    const int32_t* t = a.tok + row * a.tok_s;
    for (int64_t i = tid; i < len; i += kLogitThreads) {
      const int64_t at = t[i] - v0;
      if (at >= 0 && at < n) {
        if (i < plen) atomicOr(&cnt[at], kSeen);
        else atomicAdd(&cnt[at], 1u);
      }
    }
  }
  const int32_t* ids = a.bias_id + b * a.bias_s;
  const float* vals = a.bias + b * a.biasv_s;
  for (int64_t i = tid; i < a.nb; i += kLogitThreads) {
    const int64_t at = ids[i] - v0;
    if (at >= 0 && at < n) atomicAdd(&nbias[at], 1u);
  }
  __syncthreads();
  for (int64_t i = tid; i < a.nb; i += kLogitThreads) {
    const int64_t at = ids[i] - v0;
    if (at < 0 || at >= n) continue;
    float s = vals[i];
    if (nbias[at] > 1) {  // a token with several: the first entry's thread adds them up
      bool first = true;
      for (int64_t j = 0; j < i; ++j) first &= ids[j] != ids[i];
      if (!first) continue;
      for (int64_t j = i + 1; j < a.nb; ++j)
        if (ids[j] == ids[i]) s = s + vals[j];
    }
    bias[at] = s;
  }
  __syncthreads();
  const float rep = a.rep ? a.rep[b] : 1.f, freq = a.freq ? a.freq[b] : 0.f,
              pres = a.pres ? a.pres[b] : 0.f;
  const T* x = (const T*)a.x + b * a.ldx + v0;
  T* y = (T*)a.y + b * a.ldy + v0;
  const uint32_t* mask = a.mask ? a.mask + b * a.mask_s + v0 / 32 : nullptr;
  for (int i = tid; i < n; i += kLogitThreads) {
    float v = ll_to_f32(x[i]);
    const uint32_t c = cnt[i];
    if (c) {
      if (a.rep) v = v > 0.f ? v / rep : v * rep;
      const uint32_t said = c & ~kSeen;
      v = v - freq * (float)said;
      v = v - (said ? pres : 0.f);
    }
    if (nbias[i]) v = v + bias[i];
    if (mask && !((mask[i >> 5] >> (i & 31)) & 1u)) v = -INFINITY;
    y[i] = ll_from_f32<T>(v);
  }
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
  LL_CHECK_ARG(batch > 0 && batch <= 65535 && vocab > 0 && vocab <= INT32_MAX - kSpan,
               "%s: %lld requests (max 65535) of %lld logits", fn, (long long)batch,
               (long long)vocab);
  LL_CHECK_ARG(batch < 2 || ld_out >= vocab, "%s: output rows %lld apart overlap", fn,
               (long long)ld_out);
  LL_CHECK_ARG(!tokens || (tokens_rows >= 0 && tokens_cols >= 0 && tokens_cols <= INT32_MAX),
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
  const dim3 grid((unsigned)((vocab + kSpan - 1) / kSpan), (unsigned)batch);
  return LL_DISPATCH_DTYPE(dtype, T, [&]() -> int {
    hipLaunchKernelGGL((logits_kernel<T>), grid, dim3(kLogitThreads), 0, stream, a);
    LL_RETURN_LAUNCH();
  });
}
