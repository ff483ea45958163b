// Slot maps of a batch, built on the device from its lengths and the free
// list: start offsets, positions, pages popped for the new tokens, their cache
// slots and their entries in the slot table (and the block table), gfx950.
//
// Request b holds cached[b] tokens and gets len[b] - cached[b] new ones. With
// pages of P tokens it owns ceil(cached / P) pages and needs ceil(len / P):
// the difference comes off the free list, in batch order, so that request b's
// first new page is free[sum over a < b of need(a) - have(a)], and
//   slot(p) = page(p / P) * P + p % P.
//
// The whole call is one launch: it is bound by what a launch costs (a decode
// step writes a few hundred bytes; 260,000 new tokens write 3 MB, half a
// microsecond of HBM time), so a second launch for the prefix sums would cost
// more than having every workgroup sum the batch's lengths for itself. It
// checks lengths, rows and room before it writes anything: what is wrong there
// is reported in counts[2] and the tables stay as they were. Page ids are taken
// as they are: every workgroup would have to read all that the call takes.
#include <algorithm>

#include "ll_common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxBatch = 8192;    // requests (two int32 sums each in LDS: 64 KB)
constexpr int kMaxRows = 1 << 18;  // slot-table rows (a bit each in LDS: 32 KB)

struct SlotMapArgs {
  const void* rid; int rid64;
  const void* len; int len64;
  const void* cached; int cached64;
  const int32_t* free; int64_t nfree;
  int32_t* table; int64_t table_stride, table_rows, table_cols;
  int32_t* blocks; int64_t blocks_stride, blocks_cols;  // P > 1
  int32_t* slots; int32_t* positions; int64_t cap;
  int32_t* start; int32_t* last; int32_t* counts;
  int B, page, per;  // per: new tokens per workgroup
};

enum { kBadLength = 1, kBadRow = 2, kNoRoom = 4, kNoPages = 8 };

__global__ __launch_bounds__(kThreads) void slot_maps_kernel(SlotMapArgs a) {
  extern __shared__ int32_t sh[];
  int32_t* s_tok = sh;            // [B] first new token of request b
  int32_t* s_page = sh + a.B;     // [B] pages taken by the requests before b
  uint32_t* s_rows = (uint32_t*)(s_page + a.B);  // rows seen, one bit each
  __shared__ int64_t s_wave[2][kThreads / 64];
  __shared__ int s_err;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int P = a.page;
  const int words = (int)((a.table_rows + 31) / 32);
  for (int i = tid; i < words; i += kThreads) s_rows[i] = 0;
  if (tid == 0) s_err = 0;
  __syncthreads();
  // new tokens and pages of every request (0 for lengths that are refused)
  int err = 0;
  for (int b = tid; b < a.B; b += kThreads) {
    const int64_t n = ll_load_idx(a.len, b, a.len64), c = ll_load_idx(a.cached, b, a.cached64);
    const int64_t row = ll_load_idx(a.rid, b, a.rid64);
    int64_t nt = 0, np = 0;
    if (c < 0 || n < c || n > a.table_cols ||
        (P > 1 && (n + P - 1) / P > a.blocks_cols)) {
      err |= kBadLength;
    } else {
      nt = n - c;
      np = (n + P - 1) / P - (c + P - 1) / P;
      if (nt > 0) {  // (a request without new tokens touches no row)
        if (row < 0 || row >= a.table_rows)
          err |= kBadRow;
        else if (atomicOr(&s_rows[row >> 5], 1u << (row & 31)) >> (row & 31) & 1u)
          err |= kBadRow;  // two requests on one row would write the same entries
      }
    }
    s_tok[b] = (int32_t)nt;
    s_page[b] = (int32_t)np;
  }
  if (err) atomicOr(&s_err, err);
  __syncthreads();
  // exclusive prefix sums: a run of requests per thread, 64-bit totals
  const int per = (a.B + kThreads - 1) / kThreads;
  const int b0 = min(tid * per, a.B), b1 = min(b0 + per, a.B);
  int64_t st = 0, sp = 0;
  for (int b = b0; b < b1; ++b) {
    st += s_tok[b];
    sp += s_page[b];
  }
  int64_t it = st, ip = sp;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t ut = __shfl_up(it, o, 64), up = __shfl_up(ip, o, 64);
    if (lane >= o) {
      it += ut;
      ip += up;
    }
  }
  if (lane == 63) {
    s_wave[0][wave] = it;
    s_wave[1][wave] = ip;
  }
  __syncthreads();
  int64_t total_t = 0, total_p = 0, bt = 0, bp = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    if (w < wave) {
      bt += s_wave[0][w];
      bp += s_wave[1][w];
    }
    total_t += s_wave[0][w];
    total_p += s_wave[1][w];
  }
  err = s_err | (total_t > a.cap ? kNoRoom : 0) | (total_p > a.nfree ? kNoPages : 0);
  if (blockIdx.x == 0 && tid == 0) {
    a.counts[0] = (int32_t)min(total_t, (int64_t)INT32_MAX);
    a.counts[1] = (int32_t)min(total_p, (int64_t)INT32_MAX);
    a.counts[2] = err;
  }
  if (err) return;  // the same in every workgroup
  bt += it - st;
  bp += ip - sp;
  for (int b = b0; b < b1; ++b) {
    const int nt = s_tok[b], np = s_page[b];
    s_tok[b] = (int32_t)bt;
    s_page[b] = (int32_t)bp;
    if (blockIdx.x == 0) {
      a.start[b] = (int32_t)bt;
      a.last[b] = nt > 0 ? (int32_t)(bt + nt - 1) : -1;
    }
    bt += nt;
    bp += np;
  }
  __syncthreads();
  const int64_t end = min(total_t, ((int64_t)blockIdx.x + 1) * a.per);
  for (int64_t i = (int64_t)blockIdx.x * a.per + tid; i < end; i += kThreads) {
    // the last request whose first new token is at or before i (requests
    // without new tokens share the start of the one behind them)
    int lo = 0, hi = a.B - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s_tok[mid] <= (int32_t)i) lo = mid; else hi = mid - 1;
    }
    const int32_t c = (int32_t)ll_load_idx(a.cached, lo, a.cached64);
    const int64_t row = ll_load_idx(a.rid, lo, a.rid64);
    const int32_t p = c + (int32_t)i - s_tok[lo];
    const int32_t at = P == 1 ? p : p / P, off = P == 1 ? 0 : p - at * P;
    const int32_t have = P == 1 ? c : (c + P - 1) / P;
    int32_t page;
    if (at >= have) {
      page = a.free[s_page[lo] + at - have];
      if (P > 1 && off == 0) a.blocks[row * a.blocks_stride + at] = page;
    } else {
      page = a.blocks[row * a.blocks_stride + at];  // the page that c ends inside
    }
    const int32_t slot = page * P + off;
    a.slots[i] = slot;
    a.positions[i] = p;
    a.table[row * a.table_stride + p] = slot;
  }
}

}  // namespace

extern "C" int ll_build_slot_maps(const void* b_req_idx, int req_idx_i64, const void* b_seq_len,
                                  int seq_len_i64, const void* b_cached_len, int cached_len_i64,
                                  int64_t batch, const int32_t* free_pages, int64_t n_free,
                                  int64_t page_size, int32_t* block_table,
                                  int64_t block_table_stride, int64_t block_table_cols,
                                  int32_t* req_to_tokens, int64_t req_to_tokens_stride,
                                  int64_t req_rows, int64_t max_len, int32_t* slots,
                                  int32_t* positions, int64_t max_tokens, int32_t* b_start_loc,
                                  int32_t* last_rows, int32_t* counts, hipStream_t stream) {
  const char* fn = "ll_build_slot_maps";
  LL_CHECK_ARG(counts && req_to_tokens && (n_free == 0 || free_pages) &&
                   (max_tokens == 0 || (slots && positions)) &&
                   (batch == 0 || (b_req_idx && b_seq_len && b_cached_len && b_start_loc && last_rows)),
               "%s: null pointer", fn);
  LL_CHECK_ARG(page_size >= 1 && page_size <= (1 << 20) && (page_size == 1 || block_table),
               "%s: page_size %lld%s", fn, (long long)page_size,
               page_size > 1 ? " needs a block table" : "");
  LL_CHECK_ARG(batch >= 0 && batch <= kMaxBatch && req_rows >= 0 && req_rows <= kMaxRows,
               "%s: %lld requests (max %d), %lld table rows (max %d)", fn, (long long)batch,
               kMaxBatch, (long long)req_rows, kMaxRows);
  LL_CHECK_ARG(n_free >= 0 && n_free <= INT32_MAX && max_tokens >= 0 && max_tokens <= INT32_MAX &&
                   max_len >= 0 && max_len <= INT32_MAX - page_size,
               "%s: %lld free pages, %lld tokens, %lld table columns out of range", fn,
               (long long)n_free, (long long)max_tokens, (long long)max_len);
  SlotMapArgs a;
  a.rid = b_req_idx; a.rid64 = req_idx_i64;
  a.len = b_seq_len; a.len64 = seq_len_i64;
  a.cached = b_cached_len; a.cached64 = cached_len_i64;
  a.free = free_pages; a.nfree = n_free;
  a.table = req_to_tokens; a.table_stride = req_to_tokens_stride;
  a.table_rows = req_rows; a.table_cols = max_len;
  a.blocks = block_table; a.blocks_stride = block_table_stride; a.blocks_cols = block_table_cols;
  a.slots = slots; a.positions = positions; a.cap = max_tokens;
  a.start = b_start_loc; a.last = last_rows; a.counts = counts;
  a.B = (int)batch; a.page = (int)page_size;
  // The new tokens are known on the device only: workgroups for all that fit.
  // A token's loads are a chain (its request's values, its page, the store), so
  // a thread has one token while that gives up to 2048 workgroups, and the
  // fewest tokens that does beyond, since each of those sums the batch for
  // itself (in a graph, 1 / 2 / 4 per thread: 1 x 4096 tokens 4.4 / 4.9 / 6.1
  // us, 128 x up to 4096 in pages of 16 6.6 / 7.0 / 8.2, 1000 x 600 11.5 / 11.1
  // / 12.7, 256 x 8000 21.0 / 16.5 / 14.6).
  int64_t per = kThreads;
  while (max_tokens > 2048 * per) per *= 2;
  a.per = (int)per;
  const unsigned grid = (unsigned)std::max<int64_t>(1, ll_cdiv(max_tokens, per));
  const size_t lds = (size_t)batch * 8 + (size_t)((req_rows + 31) / 32) * 4;
  hipLaunchKernelGGL(slot_maps_kernel, dim3(grid), dim3(kThreads), lds, stream, a);
  LL_RETURN_LAUNCH();
}
