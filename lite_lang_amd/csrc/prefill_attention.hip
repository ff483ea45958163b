// NoPad varlen causal prefill attention over the paged KV pool, gfx950.
//
// For request b with L = b_seq_len[b] keys (slot row req_to_tokens[b_req_idx[b]])
// and S = shared[b] keys already cached from a previous request, the query
// rows q[b_start_loc[b] + m], m in [0, L - S), attend to keys n <= m + S.
// S = 0 is the plain NoPad prefill. Windowed, the query at position p = m + S
// attends to the keys n <= p with n > p - window or n < sinks. Semantics:
//   litelang/kernel/develop_flash_attn/flash_attn_v2.py:392-566 (no prompt cache)
//   litelang/kernel/develop_flash_attn/flash_attn_v2.py:569-762 (prompt cache)
// including the rounding of the probabilities to the KV dtype before P.V, which
// the windowed form shares: each is off by half a step at most (2^-8 of it in
// bf16, 2^-11 in fp16), their sum is taken before. Held as two numbers, as the
// decode holds them, they would bring the error against 64 bits from 0.0020 to
// the output rounding's 0.0016 (bf16; fp16 0.00029 to 0.00021) and double the
// P.V products: 40 x 600 under a window of 256 105 -> 122 us, 5 x 4111 behind
// prefixes 111 -> 146, 1 x 32,768 under 4096 994 -> 1400.
//
// Design: one workgroup = 8 waves of 32 query rows, two per SIMD (so that one
// wave's softmax overlaps the other's MFMAs, with the register budget of two
// waves). WPH waves take query rows row0 .. row0 + 32 WPH - 1 of one head and
// the workgroup takes 8 / WPH heads of one KV head (WPH = 2 when the group
// size is a multiple of 4, else 4; windowed calls also take WPH = 1 and 8, by
// the rule at the launch), so every K/V tile staged in LDS serves 256 query
// rows. The two waves of a SIMD run half a tile apart (one's scores meet the
// other's softmax). Per 64-key tile:
//   * K and V rows are DMA'd through the slot table straight into a 4-stage
//     LDS ring (global_load_lds_dwordx4), two tiles ahead of the one being
//     computed, stored key-major with their 16-byte chunks XOR-swizzled by
//     row so that the MFMA operand reads are bank-conflict free; the slot ids
//     are DMA'd too, by every wave into a ring of its own, two tiles ahead
//     of their K/V copies. The P.V operand V^T is read from the key-major V
//     tile with the gfx950 transposing LDS read (ds_read_b64_tr_b16), so no
//     VALU work transposes V;
//   * each wave computes S^T = K . Q^T (2 key blocks of 32, Q^T fragments in
//     registers, v_mfma_f32_32x32x16), the online softmax in the exp2 domain
//     with fp32 state (a row's running maximum moves only when a tile's
//     maximum passes it by more than 2^8, so that the output rows are
//     rescaled about once per work item), and O^T += V^T . P^T with P
//     rounded to the KV dtype;
//   * one barrier per tile.
// A tile that no mask touches takes 4,000 cycles of a SIMD (MFMA 2,048, VALU
// about 2,300; the rest of the two is not overlapped), a masked one some 600
// more, a change of item (Q in, output rows out, all workgroups at about the
// same time) 5,000 to 7,000. us per call, bf16, 16/2 heads of 128, and
// the share of the 1,230 TFLOP/s that a large library product reaches here:
// 1 x 8192 causal 249 (1,100 TFLOP/s, 90%); 1 x 32,768 under a window of 4096
// 967-980 (1,053-1,067, 86-87%); 40 x 600 under a window of 256 90 to 101 by
// card (400-450, 32-36%: six items of one to five tiles per workgroup).
#include <algorithm>
#include <type_traits>

#include "ll_common.h"

namespace {

constexpr int kBK = 64;   // keys per tile
// s_waitcnt immediate for vmcnt(0) with expcnt and lgkmcnt left free (gfx9
// encoding: vmcnt bits 3:0 and 15:14, expcnt 6:4, lgkmcnt 11:8)
constexpr int kVmcntZero = 0x0F70;

constexpr int kStages = 4;  // LDS ring depth (K/V tiles)
constexpr int kAhead = 2;   // tiles that K/V copies run ahead of the scores (slot ids twice that)
// A row's running maximum (exp2 domain) moves only when a tile's maximum
// passes it by more than this: the probabilities then stay at most 2^8
// (exact range in fp32 and in the 16-bit P fed to P.V)
constexpr float kLazyMax = 8.0f;

// 16 B (4 B) global -> LDS DMA of one lane: lane i of the wave lands at
// lds + 16 i (lds + 4 i).
__device__ __forceinline__ void dma16(const void* g, void* lds) {
  __builtin_amdgcn_global_load_lds(g, lds, 16, 0, 0);
}
__device__ __forceinline__ void dma4(const void* g, void* lds) {
  __builtin_amdgcn_global_load_lds(g, lds, 4, 0, 0);
}

// Wait until at most N of this wave's vector memory operations (LDS DMA
// included) are in flight.
template <int N_> __device__ __forceinline__ void vm_wait() {
  static_assert(N_ >= 0 && N_ < 64, "vmcnt is a 6-bit counter");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N_) : "memory");
}

// Workgroup barrier for LDS data only: __syncthreads() would also wait for
// every outstanding global access, the copies of the tiles ahead included.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// s_waitcnt vmcnt(0) with the Q fragments as operands: their loads are
// issued before it and their values are defined by it
__device__ __forceinline__ void q_wait_tie(bf16x8 (&q)[8]) {
  asm volatile("s_waitcnt vmcnt(0)"
               : "+v"(q[0]), "+v"(q[1]), "+v"(q[2]), "+v"(q[3]), "+v"(q[4]), "+v"(q[5]),
                 "+v"(q[6]), "+v"(q[7])::"memory");
}
__device__ __forceinline__ void q_wait_tie(bf16x8 (&q)[4]) {
  asm volatile("s_waitcnt vmcnt(0)" : "+v"(q[0]), "+v"(q[1]), "+v"(q[2]), "+v"(q[3])::"memory");
}
__device__ __forceinline__ void q_wait_tie(f16x8 (&q)[8]) {
  asm volatile("s_waitcnt vmcnt(0)"
               : "+v"(q[0]), "+v"(q[1]), "+v"(q[2]), "+v"(q[3]), "+v"(q[4]), "+v"(q[5]),
                 "+v"(q[6]), "+v"(q[7])::"memory");
}
__device__ __forceinline__ void q_wait_tie(f16x8 (&q)[4]) {
  asm volatile("s_waitcnt vmcnt(0)" : "+v"(q[0]), "+v"(q[1]), "+v"(q[2]), "+v"(q[3])::"memory");
}

template <typename T> struct Vec8;
template <> struct Vec8<__bf16> { typedef bf16x8 type; };
template <> struct Vec8<_Float16> { typedef f16x8 type; };

__device__ __forceinline__ f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// Wait until at most LEFT of this wave's LDS reads are in flight (they complete
// in order); the values pass through the wait, as in ll_lds_wait_tie.
template <int LEFT> __device__ __forceinline__ void lds_wait_tie(s16x4 (&v)[8]) {
  asm volatile("s_waitcnt lgkmcnt(%8)"
               : "+v"(v[0]), "+v"(v[1]), "+v"(v[2]), "+v"(v[3]), "+v"(v[4]), "+v"(v[5]),
                 "+v"(v[6]), "+v"(v[7])
               : "n"(LEFT)
               : "memory");
}
template <int LEFT> __device__ __forceinline__ void lds_wait_tie(s16x4 (&v)[4]) {
  asm volatile("s_waitcnt lgkmcnt(%4)"
               : "+v"(v[0]), "+v"(v[1]), "+v"(v[2]), "+v"(v[3])
               : "n"(LEFT)
               : "memory");
}
// ll_lds_read_tr16 at a constant offset from an LDS address
template <int OFF> __device__ __forceinline__ s16x4 lds_read_tr16_at(uint32_t at) {
  s16x4 r;
  asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(r) : "v"(at), "n"(OFF) : "memory");
  return r;
}

struct PrefillArgs {
  const void* q; int64_t q_st, q_sh;
  const void* k; int64_t k_st, k_sh;
  const void* v; int64_t v_st, v_sh;
  void* o; int64_t o_st, o_sh;
  const int32_t* r2t; int64_t r2t_s;
  const void* req_idx; int req64;
  const void* start_loc; int start64;
  const void* seq_len; int len64;
  const void* shared; int shared64;
  int H, G;
  int nblk, B, KVH;  // MFMA path: query-row blocks per request, requests, KV heads
  float scale_log2;
  float sm_scale;
  int window, sinks;  // windowed forms: visible keys n > p - window or n < sinks (both <= 2^30)
};

// The keys that any query at positions first .. first + rows - 1 sees, causal
// limit aside: [0, sinks) and [low, ...). Where the two meet they are one
// range from 0, given as (0, 0).
struct WindowRange {
  int sinks, low;
};
__device__ __forceinline__ WindowRange window_range(int64_t first, int window, int sinks) {
  const int64_t low = first - window + 1;
  if (low <= sinks) return {0, 0};
  return {sinks, (int)low};
}

// One step of a prefix operation over the lanes of a wave, by data-parallel
// moves (a shuffle through LDS takes ten times as long): v of the lane that
// CTRL names, `id` where there is none or ROWS leaves the row out.
template <int CTRL, int ROWS> __device__ __forceinline__ int lane_move(int id, int v) {
  return __builtin_amdgcn_update_dpp(id, v, CTRL, ROWS, 0xf, false);
}
// Inclusive prefix op over the 64 lanes: within rows of 16 (row_shr 1, 2, 4, 8),
// then the last lane of a row into the next row, and of the first two rows
// into the others (row_bcast 15 and 31).
template <typename Op> __device__ __forceinline__ int lane_scan(int v, int id, Op op) {
  v = op(v, lane_move<0x111, 0xf>(id, v));
  v = op(v, lane_move<0x112, 0xf>(id, v));
  v = op(v, lane_move<0x114, 0xf>(id, v));
  v = op(v, lane_move<0x118, 0xf>(id, v));
  v = op(v, lane_move<0x142, 0xa>(id, v));
  v = op(v, lane_move<0x143, 0xc>(id, v));
  return v;
}

// Between accesses of one wave's lanes to the LDS words of each other. The
// hardware keeps their order; without it the compiler need not, as it may take
// a lane's store for the value of the lane's next load of that word.
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

template <int D> struct FaGeom {
  static constexpr int ROWB = D * 2;            // bytes of a K or V row
  static constexpr int CH = ROWB / 16;          // 16 B chunks per row
  static constexpr int K_B = kBK * ROWB;        // K tile (V tile the same)
  static constexpr int STAGE_B = 2 * K_B;       // K tile, then V tile
  // LDS chunk position of K chunk c of row r (an involution): the operand
  // reads of 16 lanes (16 rows, one chunk) hit 16 distinct 16 B bank slots
  static __device__ __forceinline__ int kswz(int c, int r) {
    return ROWB == 256 ? (c ^ (r & 15)) : (c ^ ((r >> 1) & 7));
  }
  // LDS chunk position of V chunk c of row (key) r: a transposing read
  // (ds_read_b64_tr_b16) of one P.V fragment touches 8 consecutive keys x 4
  // consecutive chunks; this spreads them over all 16 bank slots of 256 B
  // (each slot twice, the minimum for 512 B)
  static __device__ __forceinline__ int vswz(int c, int r) {
    return ROWB == 256 ? (c ^ ((r & 3) << 2)) : (c ^ (((r >> 1) & 1) << 2));
  }
};


// WPH: waves (of 32 query rows each) per head; the 8 waves of a workgroup
// take 8 / WPH heads of one KV head and 32 * WPH query rows of each
template <int WPH_> struct FaShape {
  static constexpr int WPH = WPH_;
  static constexpr int NW = 8;           // waves per workgroup (two per SIMD)
  static constexpr int HPW = NW / WPH;   // heads per workgroup
  static constexpr int RW = 32;          // query rows per wave
  static constexpr int BQ = WPH * RW;    // query rows of one head per workgroup
};

// Work items: one per (query-row block, request, KV head, head group). Item
// numbers ("virtual blocks") put the head groups of one (row block, request,
// KV head) 8 apart, so that they take workgroups of one XCD (workgroup i runs
// on XCD i mod 8, up to a constant rotation) and read its K/V tiles through
// one L2, and put the longest (last) row blocks first. The grid is
// persistent (P workgroups, P a multiple of 16, at most 64 passes):
// workgroup w takes item jP + w on even passes j and, on odd passes, the
// items of its XCD in reverse slot order, (j + 1)P - 8 (w / 8 + 1) + w mod 8
// (a snake over the slots that keeps item mod 8 = w mod 8, so that the items
// of one (request, KV head) stay on one XCD whenever 8 divides the items per
// row block).
__device__ __forceinline__ int64_t fa_item_of_pass(int j, int P, int w) {
  return (j & 1) ? (int64_t)(j + 1) * P - 8 * ((w >> 3) + 1) + (w & 7) : (int64_t)j * P + w;
}

// The fields of the first loads (lengths, shared prefixes, start offsets,
// request rows and the grid geometry) come as scalar arguments ahead of the
// PrefillArgs block: gfx950 preloads leading scalar kernel arguments into
// SGPRs at dispatch, so those loads do not wait for the argument block's
// load. idx64: bit 0 lengths, 1 shared, 2 starts, 3 request rows are int64.
// nv: virtual blocks (items, valid or not) of the launch.
// WIN: windowed. An item's keys are its sinks and, from the first key that its
// first row sees, its window, taken as one list (a tile of their own for the
// sinks cost 16/2 heads, 40 x 600 under 256 with 4 sinks one tile in six), so
// that no table entry in between is read. In the list's positions the masks
// are those of a window with sinks from key 0 on. A wave leaves out the tiles in
// which none of its rows sees a key, and masks those that some of its rows see
// in part.
template <typename T, int D, int WPH, bool WIN>
__global__ __launch_bounds__(512) void prefill_attn_fa_kernel(
    const void* __restrict__ p_len, const void* __restrict__ p_shared,
    const void* __restrict__ p_start, const void* __restrict__ p_rid, int idx64, int nblk, int B,
    int KVH, int G, int nv, PrefillArgs a) {
  typedef typename Vec8<T>::type V8;
  typedef FaGeom<D> FG;
  typedef FaShape<WPH> SH;
  constexpr int QB = 1;  // 32-row query blocks per wave
  constexpr int DS = D / 16;  // k-steps of S^T = K . Q^T
  constexpr int DB = D / 32;  // 32-row d blocks of O^T
  extern __shared__ __attribute__((aligned(16))) char smem[];

  auto rl = [&](int v, int k) -> int { return __builtin_amdgcn_readlane(v, k); };
  auto shfl64 = [&](int64_t v, int k) -> int64_t {
    const uint32_t lo = (uint32_t)__shfl((int)(uint64_t)v, k, 64);
    const uint32_t hi = (uint32_t)__shfl((int)((uint64_t)v >> 32), k, 64);
    return (int64_t)(((uint64_t)hi << 32) | lo);
  };
  const int HP = (G + SH::HPW - 1) / SH::HPW;  // head groups per KV head
  const int P = (int)gridDim.x, w = (int)blockIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int l32 = lane & 31, hf = lane >> 5;

  // The item table, built by every wave alike in one round trip: lane j
  // holds the workgroup's item of pass j (its request's values, its KV head
  // and head group, its first query row, key count and tile count). An item
  // is valid when its row block starts inside its request's query rows.
  int it_L = 0, it_S = 0, it_blk0 = 0, it_kvend = 1, it_nt = 0, it_kvh = 0, it_hp = 0;
  // WIN: the item's keys are one list, key j below it_sk (sinks apart from its
  // window), else j + it_skip; its lengths and positions are counted in it
  int it_sk = 0, it_skip = 0;
  int it_half = -1;           // WIN: the four waves (0-3, 4-7) that have the item, -1: all
  int64_t it_start = 0, it_rid = 0;
  bool it_ok = false;
  if constexpr (WIN) {
    // The windowed form's items are those that exist, the costly first (a
    // grid over all row blocks up to the longest length deals out the missing
    // blocks of shorter requests and of cached prefixes along with the real
    // ones: 5 x 4111 tokens, 60% cached, 28/4 heads: 70 tiles for the busiest
    // workgroup, 54 so). 64 requests at a time, one per lane: the blocks whose
    // window is whole, all alike in cost, request after request; then those
    // nearer their context's start by level, the multiple of BQ that their
    // first position is at or above, the highest level first.
    struct Requests { int64_t L, S, start, rid; };
    auto requests = [&](int c0) {
      const int b = min(c0 + lane, B - 1);
      return Requests{ll_load_idx(p_len, b, idx64 & 1),
                      p_shared ? ll_load_idx(p_shared, b, (idx64 >> 1) & 1) : 0,
                      ll_load_idx(p_start, b, (idx64 >> 2) & 1),
                      ll_load_idx(p_rid, b, (idx64 >> 3) & 1)};
    };
    auto scan = [&](int v) { return lane_scan(v, 0, [](int x, int y) { return x + y; }); };
    auto blocks = [&](const Requests& q, int nreq) {
      return lane < nreq && q.L > q.S ? min(((int)q.L - (int)q.S + SH::BQ - 1) / SH::BQ, nblk) : 0;
    };
    const Requests head = requests(0);
    int total = rl(scan(blocks(head, min(B, 64))), 63);
    for (int c0 = 64; c0 < B; c0 += 64) total += rl(scan(blocks(requests(c0), min(B - c0, 64))), 63);
    // Items for at most half of the workgroups are dealt out by halves: two
    // workgroups of an XCD take an item, one its waves 0-3, one its waves 4-7,
    // which have a SIMD each (16/2 heads, 1 x 256 tokens 16.9 -> 14.5 us, 1 x 700
    // under a window of 256 21.2 -> 18.5; the last pass of a longer call so: 16 x
    // 300 under 100 24.3 -> 28.0).
    const int nitems = (total * KVH + 7) / 8 * 8 * HP;
    int64_t vb = fa_item_of_pass(lane, P, w);
    if (SH::WPH < SH::NW && 2 * nitems <= P) {
      it_half = (w >> 3) & 1;
      vb = lane == 0 && w < 2 * nitems ? 8 * (w >> 4) + (w & 7) : nv;
    }
    const int ui = vb < nv ? ((int)(vb >> 3) / HP) * 8 + (int)(vb & 7) : 0;
    const int want = vb < nv ? ui / KVH : INT32_MAX;  // the lane's (request, block) in that order
    it_kvh = ui % KVH;
    it_hp = vb < nv ? (int)(vb >> 3) % HP : 0;
    const int lam = (a.window + SH::BQ - 1) / SH::BQ;  // level from which the window is whole
    auto highest = [&](int v) {
      return rl(lane_scan(v, INT32_MIN, [](int x, int y) { return max(x, y); }), 63);
    };
    // the first lane whose prefix sum exceeds v
    auto find = [&](int incl, int v) {
      int at = 0;
#pragma unroll
      for (int o = 32; o > 0; o >>= 1)
        if (__shfl(incl, at + o - 1, 64) <= v) at += o;
      return min(at, 63);
    };
    int base = 0;  // (request, block)s listed so far
    for (int c0 = 0; c0 < B; c0 += 64) {
      const int nreq = min(B - c0, 64);
      const Requests q = c0 == 0 ? head : requests(c0);
      const int L = (int)q.L, S = (int)q.S;
      // its blocks, the levels of the first `ramp` of them, the number of whole ones
      const int nb = blocks(q, nreq);
      const int l0 = S / SH::BQ;
      const int ramp = min(nb, max(0, lam - l0)), full = nb - ramp;
      int src = -1, blk = 0;  // lane's request (as a lane number) and row block
      if (nreq == 1) {  // one request: its blocks from the last
        const int n = rl(nb, 0), rel = want - base;
        if (rel >= 0 && rel < n) {
          src = 0;
          blk = n - 1 - rel;
        }
        base += n;
      } else {
        const int incl = scan(full);
        const int total = rl(incl, 63), rel = want - base;
        base += total;
        if (total > 0) {
          const int at = find(incl, rel);
          const int before = __shfl(incl - full, at, 64), last = __shfl(nb, at, 64) - 1;
          if (rel >= 0 && rel < total) {
            src = at;
            blk = last - (rel - before);
          }
        }
        // levels 64 at a time, level hi - i in lane i: the requests that have
        // it, as the prefix sum of +1 where a request's levels begin and -1
        // behind their end (in the wave's slot ring, not in use yet)
        int* edge = (int*)(smem + kStages * FG::STAGE_B + wave * (kStages * kBK * 4));
        const int top = highest(ramp > 0 ? l0 + ramp - 1 : -1);
        const int bot = -highest(ramp > 0 ? -l0 : -INT32_MAX);
        for (int hi = top; hi >= bot; hi -= 64) {
          const int i0 = hi - (l0 + ramp - 1), i1 = hi - l0 + 1;
          edge[lane] = 0;
          wave_lds_fence();
          if (ramp > 0 && i1 > 0 && i0 < 64) {
            atomicAdd(&edge[max(i0, 0)], 1);
            if (i1 < 64) atomicAdd(&edge[i1], -1);
          }
          wave_lds_fence();
          const int cnt = scan(edge[lane]), lincl = scan(cnt);
          const int ltotal = rl(lincl, 63), lrel = want - base;
          base += ltotal;
          const bool mine = lrel >= 0 && lrel < ltotal;
          uint64_t left = __builtin_amdgcn_ballot_w64(mine);
          if (!left) continue;
          const int at = find(lincl, lrel);
          const int nth = lrel - __shfl(lincl - cnt, at, 64);  // of the requests with that level
          while (left) {  // a workgroup's few items of these levels
            const int i = (int)__builtin_ctzll(left);
            left &= left - 1;
            const int d = hi - rl(at, i) - l0;
            const uint64_t has = __builtin_amdgcn_ballot_w64((unsigned)d < (unsigned)ramp);
            const int rank = __builtin_amdgcn_mbcnt_hi((uint32_t)(has >> 32),
                                                       __builtin_amdgcn_mbcnt_lo((uint32_t)has, 0));
            const uint64_t it = __builtin_amdgcn_ballot_w64((unsigned)d < (unsigned)ramp &&
                                                            rank == rl(nth, i));
            const int r = (int)__builtin_ctzll(it);
            if (lane == i) {
              src = r;
              blk = rl(d, r);
            }
          }
        }
      }
      const int from = max(src, 0);
      const int Lx = __shfl(L, from, 64), Sx = __shfl(S, from, 64);
      const int64_t startx = shfl64(q.start, from), ridx = shfl64(q.rid, from);
      if (src >= 0) {
        it_ok = true;
        it_start = startx;
        it_rid = ridx;
        it_blk0 = blk * SH::BQ;
        const WindowRange r = window_range((int64_t)it_blk0 + Sx, a.window, a.sinks);
        it_sk = r.sinks;
        it_skip = r.low - r.sinks;
        it_L = Lx - it_skip;
        it_S = Sx - it_skip;  // (below 0 from a row block past the window on)
        it_kvend = min(it_L, it_blk0 + SH::BQ + it_S);
        it_nt = (it_kvend + kBK - 1) / kBK;
      }
    }
  } else {
    const int64_t vb = fa_item_of_pass(lane, P, w);  // vb >= nv for every pass past the last
    const int units = nblk * B * KVH;
    if (vb < nv && ((int)(vb >> 3) / HP) * 8 + (int)(vb & 7) < units) {
      const int unit = ((int)(vb >> 3) / HP) * 8 + (int)(vb & 7);
      const int b = (unit / KVH) % B;
      // every per-request value in one round trip
      const int64_t L = ll_load_idx(p_len, b, idx64 & 1);
      const int64_t S = p_shared ? ll_load_idx(p_shared, b, (idx64 >> 1) & 1) : 0;
      it_start = ll_load_idx(p_start, b, (idx64 >> 2) & 1);
      it_rid = ll_load_idx(p_rid, b, (idx64 >> 3) & 1);
      const int64_t blk0 = (int64_t)(nblk - 1 - unit / (KVH * B)) * SH::BQ;
      if (blk0 < L - S) {
        // token indices within a request fit in 32 bits (lengths below 2^31)
        it_ok = true;
        it_L = (int)L;
        it_S = (int)S;
        it_blk0 = (int)blk0;
        it_kvend = (int)min(L, blk0 + SH::BQ + S);  // keys of the item
        it_nt = (it_kvend + kBK - 1) / kBK;
        it_kvh = unit % KVH;
        it_hp = (int)(vb >> 3) % HP;
      }
    }
  }
  const uint64_t items = __builtin_amdgcn_ballot_w64(it_ok);
  if (items == 0) return;  // uniform over the workgroup
  int ntot = it_ok ? it_nt : 0;  // tiles of the workgroup's stream
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) ntot += __shfl_xor(ntot, o, 64);
  ntot = __builtin_amdgcn_readfirstlane(ntot);
  auto next_item = [&](int k) -> int {  // the valid item after pass k (64: none)
    const uint64_t rest = k >= 63 ? 0 : items & (~(uint64_t)0 << (k + 1));
    return rest ? (int)__builtin_ctzll(rest) : 64;
  };
  auto rl64 = [&](int64_t v, int k) -> int64_t {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint64_t)v, k);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)((uint64_t)v >> 32), k);
    return (int64_t)(((uint64_t)hi << 32) | lo);
  };

  // This wave's view of an item: its head, its first query row and whether
  // it has rows there, the keys its rows see, the request's query start.
  struct WaveItem {
    int64_t start;
    int h, row0, qlast, S, Lm1, kv_end;
    bool ok;
  };
  auto wave_item = [&](int k) -> WaveItem {
    WaveItem r;
    const int L = rl(it_L, k), S = rl(it_S, k), blk0 = rl(it_blk0, k);
    const int gh = SH::HPW * rl(it_hp, k) + wave / SH::WPH;  // head within the KV head's group
    r.start = rl64(it_start, k);
    r.h = rl(it_kvh, k) * G + (gh < G ? gh : 0);
    r.row0 = blk0 + SH::RW * (wave % SH::WPH);
    r.qlast = L - S - 1;
    r.ok = gh < G && r.row0 <= r.qlast;
    if constexpr (WIN) {
      const int half = rl(it_half, k);
      r.ok = r.ok && (half < 0 || half == wave / 4);
    }
    r.S = S;
    r.Lm1 = L - 1;
    r.kv_end = (int)min((int64_t)L, (int64_t)r.row0 + SH::RW + S);
    return r;
  };
  // Q^T fragments (B operand: column = query row row0 + l32, clamped into the
  // request; k-slots = d 16 s + 8 hf .. +7), in registers for the whole item
  V8 qreg[DS];
  auto load_q = [&](const WaveItem& it) {
    const int r = min(it.row0 + l32, it.qlast);
    const T* qp = (const T*)a.q + (it.start + r) * a.q_st + (int64_t)it.h * a.q_sh + 8 * hf;
#pragma unroll
    for (int s = 0; s < DS; ++s) qreg[s] = *(const V8*)(qp + 16 * s);
  };

  // The workgroup's items run as one stream of 64-key tiles. K and V tiles
  // go from the pool straight into an NST-stage LDS ring
  // (global_load_lds_dwordx4, no VGPR staging); the slot ids that address
  // them are DMA'd likewise, by every wave into a ring of its own, kAhead
  // tiles before the tile's K/V copies. Per stream tile x every wave issues
  // one group: its K/V copies of tile x + kAhead and its slot ids of tile
  // x + 2 kAhead, so that kAhead tiles are in flight while tile x is
  // computed, across item boundaries too (the next item's first tiles load
  // under the current item's last ones). Past the stream's end the groups
  // repeat the last item's last key into stages nothing reads, so that
  // every iteration has the same copies in flight.
  constexpr int NST = kStages;
  constexpr int RPI = 64 / FG::CH;                     // rows per DMA instruction
  constexpr int IPW = kBK * FG::ROWB / 1024 / SH::NW;  // K (and V) instructions per wave per tile
  constexpr int KVC = 2 * IPW;                         // K and V
  static_assert(IPW >= 1 && IPW * SH::NW * 1024 == kBK * FG::ROWB, "tile rows over the waves");
  char* wslots = smem + NST * FG::STAGE_B + wave * (NST * kBK * 4);
  const int dr = lane / FG::CH, dp = lane % FG::CH;

  // The copy cursors: the item (pass) and tile of the next group's copies,
  // with that item's addresses (refreshed only when a cursor moves to the
  // next item, so that an iteration's scalar work stays small: the scalar
  // unit serves all eight waves of the CU). Past the stream's end each
  // stays on the last item's last tile.
  struct SlotCursor {
    int k, u, nt, last_key;
    int sk, skip;  // WIN
    const int32_t* row;
  };
  struct KvCursor {
    int k, left;  // tiles of the item still to copy, the next one included
    const T* kb;
    const T* vb;
  };
  auto slot_at = [&](SlotCursor& c, int k) {
    c.k = k;
    c.u = 0;
    c.nt = rl(it_nt, k);
    c.last_key = rl(it_kvend, k) - 1;
    if constexpr (WIN) {
      c.sk = rl(it_sk, k);
      c.skip = rl(it_skip, k);
    }
    c.row = a.r2t + rl64(it_rid, k) * a.r2t_s;
  };
  auto kv_at = [&](KvCursor& c, int k) {
    c.k = k;
    c.left = rl(it_nt, k);
    const int kvh = rl(it_kvh, k);
    c.kb = (const T*)a.k + (int64_t)kvh * a.k_sh;
    c.vb = (const T*)a.v + (int64_t)kvh * a.v_sh;
  };
  auto slot_next = [&](SlotCursor& c) {
    if (++c.u == c.nt) {
      const int k2 = next_item(c.k);
      if (k2 < 64) slot_at(c, k2); else c.u = c.nt - 1;
    }
  };
  auto kv_next = [&](KvCursor& c) {
    if (--c.left == 0) {
      const int k2 = next_item(c.k);
      if (k2 < 64) kv_at(c, k2); else c.left = 1;
    }
  };
  const int k_first = (int)__builtin_ctzll(items);
  // slot ids of cursor c's tile (keys 64 u + lane, clamped) -> ring entry x % NST
  auto slot_copy = [&](int x, const SlotCursor& c) {
    int key = min(c.u * kBK + lane, c.last_key);
    if (WIN && key >= c.sk) key += c.skip;
    dma4(c.row + key, wslots + (x % NST) * (kBK * 4));
  };
  // this wave's K and V rows of cursor c's tile (slot ids in ring entry
  // x % NST) -> stage x % NST
  auto kv_copy = [&](int x, const KvCursor& c) {
    char* kl = smem + (x % NST) * FG::STAGE_B;
    char* vl = kl + FG::K_B;
    const int32_t* sl = (const int32_t*)(wslots + (x % NST) * (kBK * 4));
    uint32_t slot[IPW];
#pragma unroll
    for (int i = 0; i < IPW; ++i) slot[i] = (uint32_t)sl[(wave * IPW + i) * RPI + dr];
    // (a slot's row by one 32 x 32 -> 64 bit multiply-add: the launcher checks
    // that a token's stride has 32 bits)
    const uint32_t kst = (uint32_t)a.k_st * sizeof(T), vst = (uint32_t)a.v_st * sizeof(T);
#pragma unroll
    for (int i = 0; i < IPW; ++i) {
      const int ii = wave * IPW + i;
      const int r = ii * RPI + dr;  // the LDS chunk position dp of row r holds chunk swz(dp, r)
      dma16((const char*)c.kb + ((uint64_t)slot[i] * kst + 16 * FG::kswz(dp, r)), kl + ii * 1024);
      dma16((const char*)c.vb + ((uint64_t)slot[i] * vst + 16 * FG::vswz(dp, r)), vl + ii * 1024);
    }
  };

  f32x16 acc[DB][QB];
  // a row's running maximum (the same in its two lanes) and the sum of its
  // probabilities over the keys of this lane's half-wave
  float m_run[QB], l_run[QB];
  auto reset = [&]() {
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) acc[db][qb] = (f32x16){};
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      // WIN: finite, so that a row that sees nothing of its wave's first tiles
      // gets exp2(-inf - m) = 0 from them and a later tile's rescale is 0
      m_run[qb] = WIN ? -3.402823466e38f : -INFINITY;
      l_run[qb] = 0.f;
    }
  };
  reset();

  WaveItem cur = wave_item(k_first);
  load_q(cur);
  // slot ids of stream tiles 0 and 1, then (every load so far landed, Q
  // fragments included: a real s_waitcnt, which the compiler's own wait
  // insertion accounts for) the groups of iterations -2 and -1
  SlotCursor cs;
  slot_at(cs, k_first);
  KvCursor ck;
  kv_at(ck, k_first);
#pragma unroll
  for (int x = 0; x < kAhead; ++x) {
    slot_copy(x, cs);
    slot_next(cs);
  }
  __builtin_amdgcn_s_waitcnt(kVmcntZero);
#pragma unroll
  for (int x = 0; x < kAhead; ++x) {
    kv_copy(x, ck);
    kv_next(ck);
    slot_copy(x + kAhead, cs);
    slot_next(cs);
  }

  // S^T[key 32 kb + 8 g + 4 hf + i][query 32 qb + l32] of the current tile in
  // sacc[kb][qb][4 g + i]; the tile's row maxima (exp2 domain) over this
  // half-wave's keys in m_cand
  f32x16 sacc[2][QB];
  float m_cand[QB];
  // (t0: the tile's first key)
  // (masked false_type: the caller knows that every row sees the whole tile)
  auto scores = [&](auto masked, int t0, int buf) {
    const char* kl = smem + buf * FG::STAGE_B;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) sacc[kb][qb] = (f32x16){};
    // the operands of a k-step are read while the step before it multiplies
    auto k_read = [&](int s, V8 (&k)[2]) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int r = 32 * x + l32;
        k[x] = *(const V8*)(kl + r * FG::ROWB + FG::kswz(2 * s + hf, r) * 16);
      }
    };
    V8 ka[2][2];
    k_read(0, ka[0]);
#pragma unroll
    for (int s = 0; s < DS; ++s) {
      if (s + 1 < DS) k_read(s + 1, ka[(s + 1) & 1]);
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) sacc[kb][qb] = mfma32(ka[s & 1][kb], qreg[s], sacc[kb][qb]);
      __builtin_amdgcn_sched_barrier(0);
    }
    // the causal + length mask only where a key can pass the wave's first
    // row's limit (masked keys -> -inf), then the tile's row maxima in the
    // exp2 domain (finite: key 0 is visible to every row, scale_log2 > 0)
    const int last_row_low = cur.row0 + SH::RW - 1 + cur.S - a.window;  // below its window
    const bool need_mask = t0 + kBK - 1 > min(cur.row0 + cur.S, cur.Lm1) ||
                           (WIN && t0 <= last_row_low && t0 + kBK > a.sinks);
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      if (decltype(masked)::value && need_mask) {
        // last key this row sees, relative to the tile (rows past the
        // request see every key of it)
        const int p = cur.row0 + 32 * qb + l32 + cur.S;
        const int lim = min(p, cur.Lm1) - t0;
        // The visible keys as bits, shifted out from the top in the order of
        // the lane's elements: an add and a select per element where compares
        // of each key with the row's limits take four and scalar logic (a
        // masked tile took 1300 cycles more than another, 40 x 600 under a
        // window of 256 112 us, now 108).
        auto first = [](int n) -> uint32_t {  // bits 0 .. n - 1
          const int m = min(max(n, 0), 32);
          return m == 32 ? ~0u : (1u << m) - 1u;
        };
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          uint32_t see = first(lim + 1 - 32 * kb);
          if constexpr (WIN)
            see &= ~first(p - a.window + 1 - t0 - 32 * kb) | first(a.sinks - t0 - 32 * kb);
          see = __builtin_bitreverse32(see) << (4 * hf);
#pragma unroll
          for (int e = 0; e < 16; ++e) {  // key 32 kb + 8 (e / 4) + 4 hf + e % 4
            uint32_t next;
            const bool is = __builtin_uadd_overflow(see, see, &next);
            sacc[kb][qb][e] = is ? sacc[kb][qb][e] : -INFINITY;
            see = (e & 3) == 3 ? next << 4 : next;
          }
        }
      }
      float tmax = -INFINITY;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) tmax = fmaxf(tmax, sacc[kb][qb][e]);
      m_cand[qb] = tmax * a.scale_log2;  // this half-wave's keys only
    }
  };
  // p = 2^(s * scale_log2 - m_run) rounded to T as the P^T fragments of the 4
  // key steps (step s = keys 16 s + {4hf..4hf+3, 8+4hf..8+4hf+3}: S^T block
  // kb = s / 2, g = 2 (s % 2) and g + 1), the row sums into l_run, then
  // O^T[d 32 db + 8 g + 4 hf + i][query 32 qb + l32] += V^T . P^T
  // V^T fragment of key step s, d block db (A operand: lane -> d = 32 db +
  // l32, k-slots 8 hf .. 8 hf + 7 = keys 16 s + 4 hf + {0..3} and
  // 16 s + 8 + 4 hf + {0..3}, the order of the P^T fragments): two
  // transposing reads, the 16-lane group g = lane / 16 reading keys
  // 16 s + 4 (g / 2) + j / 4 (+ 8), d 32 db + 16 (g % 2) + 4 (j % 4) .. + 3
  const int tg = lane >> 4, tj = lane & 15;
  // the lane's LDS address in a V tile of stage 0 of key step 0's first read for
  // each d block: d bytes 64 db + 32 (g % 2) + 8 (j % 4) of key 4 (g / 2) + j / 4.
  // The other reads are whole rows further, which the swizzle repeats every 4.
  uint32_t vaddr[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) {
    const int key = 4 * (tg >> 1) + (tj >> 2);
    const int dbyte = 64 * db + 32 * (tg & 1) + 8 * (tj & 3);
    vaddr[db] = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)smem + FG::K_B +
                key * FG::ROWB + FG::vswz(dbyte >> 4, key) * 16 + (dbyte & 15);
  }
  // the fragments of key step S, two reads per d block: keys 16 S + 4 (g / 2) + j / 4
  // and 8 keys further
  auto v_reads = [&](auto step, const uint32_t (&at)[DB], s16x4 (&v)[2 * DB]) {
    constexpr int S0 = decltype(step)::value * 16 * FG::ROWB;
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      v[2 * db] = lds_read_tr16_at<S0>(at[db]);
      v[2 * db + 1] = lds_read_tr16_at<S0 + 8 * FG::ROWB>(at[db]);
    }
  };
  auto accumulate = [&](int buf) {
    // V fragments a key step ahead of their MFMAs, the first under the
    // exponentials (the waits of reads and MFMAs in turn were a sixth of a
    // tile's time)
    uint32_t vat[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db) vat[db] = vaddr[db] + buf * FG::STAGE_B;
    s16x4 vr[2][2 * DB];
    v_reads(std::integral_constant<int, 0>{}, vat, vr[0]);
    V8 pf[QB][4];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      float psum = 0.f;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int kb = s >> 1, e0 = 8 * (s & 1);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float p = __builtin_amdgcn_exp2f(
              __builtin_fmaf(sacc[kb][qb][e0 + e], a.scale_log2, -m_run[qb]));
          psum += p;
          pf[qb][s][e] = (T)p;
        }
      }
      l_run[qb] += psum;  // this half-wave's keys; the halves add up at the store
    }
    auto multiply = [&](int s, const s16x4 (&v)[2 * DB]) {
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        const V8 va = __builtin_bit_cast(
            V8, __builtin_shufflevector(v[2 * db], v[2 * db + 1], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) acc[db][qb] = mfma32(va, pf[qb][s], acc[db][qb]);
      }
    };
    v_reads(std::integral_constant<int, 1>{}, vat, vr[1]);
    lds_wait_tie<2 * DB>(vr[0]);
    multiply(0, vr[0]);
    v_reads(std::integral_constant<int, 2>{}, vat, vr[0]);
    lds_wait_tie<2 * DB>(vr[1]);
    multiply(1, vr[1]);
    v_reads(std::integral_constant<int, 3>{}, vat, vr[1]);
    lds_wait_tie<2 * DB>(vr[0]);
    multiply(2, vr[0]);
    lds_wait_tie<0>(vr[1]);
    multiply(3, vr[1]);
  };
  // acc[db][qb][4 g + i] = O^T[d = 32 db + 8 g + 4 hf + i][query row0 + 32 qb + l32].
  // The halves of a row (lanes l and l + 32) swap 4-element groups, so that
  // each stores 8 elements of it at a time: half the store instructions, whose
  // 32 rows each take the memory path about 50 cycles (40 x 600, window 256,
  // 16/2 heads: 122 -> 114 us; the same rows as whole lines through LDS: 118).
  // The rows of `out` may start at any element (global memory takes 16 bytes
  // from any address).
  typedef u32x4 __attribute__((aligned(2))) u32x4_any;
  auto store_rows = [&](const WaveItem& it) {
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      const int r = it.row0 + 32 * qb + l32;
      if (r > it.qlast) continue;  // the same in both halves
      const float inv = 1.0f / (l_run[qb] + __shfl_xor(l_run[qb], 32, 64));
      T* op = (T*)a.o + (it.start + r) * a.o_st + (int64_t)it.h * a.o_sh + 8 * hf;
      typedef T T4 __attribute__((ext_vector_type(4)));
      typedef uint32_t U2 __attribute__((ext_vector_type(2)));
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int g = 0; g < 4; g += 2) {
          T4 y0, y1;  // d = 32 db + 8 g + 4 hf + i, and 8 further
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            y0[i] = ll_from_f32<T>(acc[db][qb][4 * g + i] * inv);
            y1[i] = ll_from_f32<T>(acc[db][qb][4 * g + 4 + i] * inv);
          }
          const U2 u0 = __builtin_bit_cast(U2, y0), u1 = __builtin_bit_cast(U2, y1);
          u32x4 w;  // lower half: d = 32 db + 8 g .. + 7, upper: 8 further
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const auto p = __builtin_amdgcn_permlane32_swap(u0[i], u1[i], false, false);
            w[i] = p[0];
            w[2 + i] = p[1];
          }
          *(u32x4_any*)(op + 32 * db + 8 * g) = w;
        }
    }
  };

  // the next item's Q rows are pulled into L2 ahead of its first tile: one
  // 4-byte DMA per lane into this wave's 256-byte sink (never read), lane i
  // touching 128-byte line i % LPR of row i / LPR of the wave's 32 rows
  char* wsink = smem + NST * FG::STAGE_B + SH::NW * (NST * kBK * 4) + wave * 256;
  auto prefetch_q = [&](const WaveItem& it) {
    constexpr int LPR = FG::ROWB / 128;  // 128-byte lines per Q row
    const int r = min(it.row0 + (lane / LPR) % SH::RW, it.qlast);
    const T* qp = (const T*)a.q + (it.start + r) * a.q_st + (int64_t)it.h * a.q_sh + 64 * (lane % LPR);
    dma4(qp, wsink);
  };

  // running maxima, moved only when a row of the wave meets a tile maximum
  // more than kLazyMax above its own (the first tile always): until then the
  // probabilities exp2(s - m_run) stay below 2^kLazyMax, and the output rows
  // and sums are rescaled about once per item instead of at nearly every tile
  auto rescale = [&]() {
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      if (__builtin_amdgcn_ballot_w64(m_cand[qb] > m_run[qb] + kLazyMax)) {
        // both halves of a row (its two lanes) take the row's maximum
        const float m_new = fmaxf(m_run[qb], fmaxf(m_cand[qb], __shfl_xor(m_cand[qb], 32, 64)));
        const float alpha = __builtin_amdgcn_exp2f(m_run[qb] - m_new);
        m_run[qb] = m_new;
        l_run[qb] *= alpha;
#pragma unroll
        for (int db = 0; db < DB; ++db) acc[db][qb] *= alpha;
      }
    }
  };

  // One barrier per tile, the "event" of tile x: behind it every wave's copies
  // of tile x are in, and stage (x + kAhead) % NST is free. The waves 0-3 meet
  // it ahead of the tile's scores; the waves 4-7 ahead of the P.V of tile
  // x - 1, whose scores they have: on each SIMD one wave's scores and P.V
  // (MFMA) then meet the other's softmax (VALU) instead of its like (long
  // windows, 5 x 4111 behind prefixes: 121 -> 117 us; 8 x 2000, 28/4: 184 ->
  // 180). Every wave issues the copies of tile x + kAhead (and the slot ids of
  // tile x + 2 kAhead) behind its scores of tile x, hence behind the event of
  // tile x: all waves are then done with tile x - 2, which had that stage
  // (waves 4-7 with its P.V before the event). So only the group of iteration
  // x - 1 may be in flight at the event of tile x, besides older output stores
  // and newer Q prefetches: vector memory operations complete in issue order,
  // so both only make the wait longer.
  static_assert(NST == kAhead + 2, "the stages the events free");
  const bool lead = wave < SH::NW / 2;
  // the next events whose copies a full wait (at an item's first tile) already
  // covered: those of iteration x - 1 are in after it
  int covered = 0;
  auto event = [&]() {
    if (covered > 0) --covered; else vm_wait<1 + KVC>();
    lds_barrier();
  };
  int cc_k = k_first, cc_u = 0, cc_nt = rl(it_nt, k_first);  // item (pass) and tile computed
  WaveItem done = cur;  // at an item's first tile: the item whose rows acc holds
  if (!lead) event();
  for (int x = 0; x < ntot; ++x) {
    // A run of tiles that every row of the wave sees whole, that are not their
    // item's last and whose copies stay inside the cursors' items: the same
    // steps without the decisions, whose scalar instructions and branches are
    // on every wave's path (a fifth of a tile's time: 32,768 tokens under a
    // window of 4096 1039 -> 985 us)
    int run = cs.nt - 1 - cs.u;
    if (run > 1 && cc_u > 0 && covered == 0 && cur.ok) {
      const int first = cc_u * kBK;  // key of tile x
      const bool whole = !WIN || (cs.u * kBK >= cs.sk &&
                                  first > cur.row0 + SH::RW - 1 + cur.S - a.window);
      run = min(min(run, ck.left - 1), min(cc_nt - 1 - cc_u,
                                           (min(cur.row0 + cur.S, cur.Lm1) + 1 - first) / kBK));
      if (whole && run > 0) {
        const int32_t* ids = cs.row + (WIN ? cs.skip : 0) + cs.u * kBK + lane;
        cc_u += run;
        ck.left -= run;
        cs.u += run;
        for (; run > 0; --run, ++x, ids += kBK) {
          if (lead) event();
          scores(std::false_type{}, 0, x % NST);
          kv_copy(x + kAhead, ck);
          dma4(ids, wslots + ((x + 2 * kAhead) % NST) * (kBK * 4));
          if (!lead) event();  // (of tile x + 1, which there is)
          rescale();
          accumulate(x % NST);
        }
      }
    }
    if (lead) event();
    if (cc_u == 0 && x > 0) {
      // An item's first tile (the first item's Q came with the prologue):
      // its Q fragments, from L2, and the wait for them, before this
      // iteration's copies (the wait covers the copies in flight, which
      // were issued a tile or more ago). The loads and the wait stay in one
      // branch and the fragments pass through the wait as operands: the
      // compiler then sees nothing pending across the loop's back edge (it
      // would otherwise wait for every copy in flight before each scores).
      load_q(cur);
      q_wait_tie(qreg);
      covered = 1;
      // the previous item's rows, then a fresh softmax state
      if (done.ok) store_rows(done);
      reset();
    }
    const int buf = x % NST;
    const int t0 = cc_u * kBK;
    // not where the causal limit or the wave's first row's window leaves the
    // tile out, but where it holds sinks
    const bool work = cur.ok && t0 < cur.kv_end &&
                      (!WIN || t0 + kBK - 1 > cur.row0 + cur.S - a.window || t0 < a.sinks);
    const bool last = cc_u + 1 == cc_nt;
    if (work) scores(std::true_type{}, t0, buf);
    // (behind the score MFMAs, which run on while the addresses are computed)
    kv_copy(x + kAhead, ck);
    kv_next(ck);
    slot_copy(x + 2 * kAhead, cs);
    slot_next(cs);
    if (last) {
      const int k2 = next_item(cc_k);
      if (k2 < 64) prefetch_q(wave_item(k2));
    }
    if (!lead && x + 1 < ntot) event();
    if (work) {
      rescale();
      accumulate(buf);
    }
    if (!last) {
      ++cc_u;
    } else {
      const int k2 = next_item(cc_k);
      if (k2 < 64) {  // (past the last item's last tile the loop ends)
        done = cur;
        cur = wave_item(k2);
        cc_k = k2;
        cc_u = 0;
        cc_nt = rl(it_nt, k2);
      }
    }
  }
  // no copy may still be writing this workgroup's LDS when it ends
  vm_wait<0>();
  if (cur.ok) store_rows(cur);
}

// Generic path: one wave per (query row, head), keys spread over the lanes; for
// fp32, other head dims and unaligned q, K or V (windowed, 16/2 heads, 4 x 300
// under 256: bf16 heads of 128 19 us on the MFMA path, of 96 214 here, fp32 of
// 128 303; 40 x 600: 91, 4590, 6760).
// WIN: only the keys of the row's window and the sinks, taken as one list
// (index j is key j below the sinks, else j + skip), so that no table entry of
// another key is read.
template <typename T, bool WIN>
__global__ __launch_bounds__(64) void prefill_attn_generic_kernel(PrefillArgs a, int D) {
  const int64_t m_row = blockIdx.x;
  const int h = blockIdx.y;
  const int b = blockIdx.z;
  const int kvh = h / a.G;
  const int lane = threadIdx.x;
  const int64_t L = ll_load_idx(a.seq_len, b, a.len64);
  const int64_t S = a.shared ? ll_load_idx(a.shared, b, a.shared64) : 0;
  if (m_row >= L - S) return;
  const int64_t start = ll_load_idx(a.start_loc, b, a.start64);
  const int64_t rid = ll_load_idx(a.req_idx, b, a.req64);
  extern __shared__ float sh[];
  float* qs = sh;
  float* ps = sh + D;
  int* ss = (int*)(ps + 64);
  const T* qp = (const T*)a.q + (start + m_row) * a.q_st + (int64_t)h * a.q_sh;
  for (int d = lane; d < D; d += 64) qs[d] = ll_to_f32(qp[d]);
  __syncthreads();
  int64_t kv_end = min(L, m_row + S + 1);
  int64_t nsink = 0, skip = 0;
  if constexpr (WIN) {
    const WindowRange r = window_range(m_row + S, a.window, a.sinks);
    nsink = r.sinks;
    skip = r.low - r.sinks;
    kv_end -= skip;
  }
  const int nd = (D + 63) / 64;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  const T* kb = (const T*)a.k + (int64_t)kvh * a.k_sh;
  const T* vb = (const T*)a.v + (int64_t)kvh * a.v_sh;
  for (int64_t t0 = 0; t0 < kv_end; t0 += 64) {
    const int64_t t = t0 + lane;
    float s = -INFINITY;
    int slot = 0;
    if (t < kv_end) {
      slot = a.r2t[rid * a.r2t_s + (WIN && t >= nsink ? t + skip : t)];
      const T* kr = kb + (int64_t)slot * a.k_st;
      float dot = 0.f;
      for (int d = 0; d < D; ++d) dot += qs[d] * ll_to_f32(kr[d]);
      s = dot * a.scale_log2;
    }
    const float mn = fmaxf(m, ll_wave_max(s));
    const float alpha = exp2f(m - mn);
    const float p = (t < kv_end) ? exp2f(s - mn) : 0.f;
    l = l * alpha + ll_wave_sum(p);
    m = mn;
    ps[lane] = ll_to_f32(ll_from_f32<T>(p));  // P rounded to the KV dtype before P.V
    ss[lane] = slot;
    __syncthreads();
    const int cnt = (int)min((int64_t)64, kv_end - t0);
    for (int r = 0; r < nd; ++r) {
      const int d = lane + 64 * r;
      float v = acc[r] * alpha;
      if (d < D)
        for (int u = 0; u < cnt; ++u) v += ps[u] * ll_to_f32(vb[(int64_t)ss[u] * a.v_st + d]);
      acc[r] = v;
    }
    __syncthreads();
  }
  T* op = (T*)a.o + (start + m_row) * a.o_st + (int64_t)h * a.o_sh;
  for (int r = 0; r < nd; ++r) {
    const int d = lane + 64 * r;
    if (d < D) op[d] = ll_from_f32<T>(acc[r] / l);
  }
}

// A grid has fewer than 2^32 threads: workgroups of the generic path (one wave)
// in a row, and work items of the MFMA path (512 threads for up to 64 of them,
// in a multiple of 16 workgroups).
constexpr int64_t kMaxRows = (((int64_t)1 << 32) - 1) / 64;
constexpr int64_t kMaxItems = 64 * (((int64_t)1 << 32) / 512 - 16);

// Both entry points: win false is the whole context (window and sinks unused).
int prefill_attention(const char* fn, const void* q, int64_t q_stride_tok, int64_t q_stride_h,
                      const void* k_cache, int64_t k_stride_tok, int64_t k_stride_head,
                      const void* v_cache, int64_t v_stride_tok, int64_t v_stride_head, void* out,
                      int64_t out_stride_tok, int64_t out_stride_h, const int32_t* req_to_tokens,
                      int64_t req_to_tokens_stride, const void* b_req_idx, int req_idx_i64,
                      const void* b_start_loc, int start_loc_i64, const void* b_seq_len,
                      int seq_len_i64, const void* b_shared_seq_len, int shared_i64, int64_t batch,
                      int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t max_input_len,
                      bool win, int64_t window, int64_t sinks, float sm_scale, int dtype,
                      hipStream_t stream) {
  // (an empty tensor has no address: no requests, or none with query rows)
  if (win && (batch == 0 || (!q && !out))) return LL_OK;
  LL_CHECK_ARG(q && k_cache && v_cache && out && req_to_tokens && b_req_idx && b_start_loc &&
                   b_seq_len,
               "%s: null pointer", fn);
  LL_CHECK_ARG(kv_heads > 0 && q_heads % kv_heads == 0,
               "%s: q_heads %lld not a multiple of kv_heads %lld", fn, (long long)q_heads, (long long)kv_heads);
  LL_CHECK_ARG(!win || (batch >= 0 && batch <= 1 << 24 && q_heads > 0 && q_heads <= 65535),
               "%s: %lld requests of %lld heads", fn, (long long)batch, (long long)q_heads);
  LL_CHECK_ARG(head_dim > 0 && head_dim <= 256 && head_dim % 2 == 0,
               "%s: head_dim %lld unsupported", fn, (long long)head_dim);
  // window 1 sees the query's own token alone: no row is left without a key
  LL_CHECK_ARG(!win || (window >= 1 && sinks >= 0), "%s: window %lld (min 1), sinks %lld (min 0)", fn,
               (long long)window, (long long)sinks);
  LL_CHECK_ARG(!win || (sm_scale > 0.f && sm_scale < INFINITY), "%s: sm_scale %g must be positive",
               fn, (double)sm_scale);
  LL_CHECK_ARG(max_input_len <= (win ? 1 << 30 : INT32_MAX), "%s: max_input_len %lld out of range",
               fn, (long long)max_input_len);
  if (batch == 0 || max_input_len <= 0) return LL_OK;
  PrefillArgs a;
  a.q = q; a.q_st = q_stride_tok; a.q_sh = q_stride_h;
  a.k = k_cache; a.k_st = k_stride_tok; a.k_sh = k_stride_head;
  a.v = v_cache; a.v_st = v_stride_tok; a.v_sh = v_stride_head;
  a.o = out; a.o_st = out_stride_tok; a.o_sh = out_stride_h;
  a.r2t = req_to_tokens; a.r2t_s = req_to_tokens_stride;
  a.req_idx = b_req_idx; a.req64 = req_idx_i64;
  a.start_loc = b_start_loc; a.start64 = start_loc_i64;
  a.seq_len = b_seq_len; a.len64 = seq_len_i64;
  a.shared = b_shared_seq_len; a.shared64 = shared_i64;
  a.H = (int)q_heads; a.G = (int)(q_heads / kv_heads);
  a.sm_scale = sm_scale;
  // (lengths are at most 2^30, so a larger window or count sees as much)
  a.window = (int)std::min<int64_t>(window, 1 << 30);
  a.sinks = (int)std::min<int64_t>(sinks, 1 << 30);
  a.scale_log2 = sm_scale * 1.4426950408889634f;

  const bool mfma_ok = (dtype == LL_BF16 || dtype == LL_F16) && (head_dim == 128 || head_dim == 64) &&
                       (q_stride_tok % 8 == 0) && (q_stride_h % 8 == 0) &&
                       (k_stride_tok % 8 == 0) && (k_stride_head % 8 == 0) &&
                       (v_stride_tok % 8 == 0) && (v_stride_head % 8 == 0) &&
                       k_stride_tok >= 0 && k_stride_tok < ((int64_t)1 << 31) &&
                       v_stride_tok >= 0 && v_stride_tok < ((int64_t)1 << 31) &&
                       (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache) % 16 == 0);
  if (!mfma_ok) {
    LL_CHECK_ARG(q_heads <= 65535 && batch <= 65535 && max_input_len <= kMaxRows,
                 "%s: more than 65535 heads or requests, or %lld rows", fn, (long long)kMaxRows);
    const size_t shm = head_dim * 4 + 64 * 4 + 64 * 4;
    return LL_DISPATCH_DTYPE(dtype, T, [&]() -> int {
      const dim3 grid((unsigned)max_input_len, (unsigned)q_heads, (unsigned)batch);
      if (win)
        hipLaunchKernelGGL((prefill_attn_generic_kernel<T, true>), grid, dim3(64), shm, stream, a,
                           (int)head_dim);
      else
        hipLaunchKernelGGL((prefill_attn_generic_kernel<T, false>), grid, dim3(64), shm, stream, a,
                           (int)head_dim);
      LL_RETURN_LAUNCH();
    });
  }
  // four heads of 64 rows per workgroup when the group size allows, else two
  // heads of 128 rows (fewer idle head slots for G = 6 or 7). Windowed, also
  // * eight heads of 32 rows for a group one short of eight: as few idle slots
  //   as two heads, a shorter stretch of keys per item (28/4 heads, 40 x 600
  //   under a window of 256 181 -> 159 us, under 64 146 -> 122, 64 x 150 74 ->
  //   54; the worst of 14 shapes, 4 x 300, 19.8 -> 21.3);
  //   the same for a multiple of eight where the shorter stretch is a tile less
  //   (16/2 heads with 4 sinks, 40 x 600 under 128 91 -> 80 us, under 256 101 ->
  //   94; where it is not, 1 x 8192 under 64 without sinks 29.3 -> 34.7);
  // * one head of 256 rows for single-head groups (16/16 heads, 40 x 600 under
  //   256 158 -> 136 us; 4 x 300 17.1 -> 18.7);
  // * one head for short calls that fit one pass: the up to four waves with
  //   rows then have a SIMD each, without a second workgroup for the other
  //   half (16/2 heads, 1 x 20 tokens 9.6 -> 8.6 us, 8 x 128 17.1 -> 12.0, by
  //   halves of two heads 9.1 and 14.9; where they do not fit one pass 40 x 100
  //   20.7 -> 26.3).
  auto tiles = [&](int w) {  // of an item whose window is whole
    return ((int64_t)a.window + a.sinks + 32 * w - 1 + kBK - 1) / kBK;
  };
  const bool eight = a.G % 8 == 7 || (a.G % 8 == 0 && tiles(1) < tiles(2));
  int wph = win && a.G == 1 ? 8 : win && eight ? 1 : a.G % 4 == 0 ? 2 : 4;
  auto blocks = [&](int w) { return (max_input_len + 32 * w - 1) / (32 * w); };
  auto items = [&](int w) {
    return (blocks(w) * batch * kv_heads + 7) / 8 * 8 * ll_cdiv(a.G, 8 / w);
  };
  LL_CHECK_ARG(batch <= kMaxItems / kv_heads / blocks(wph) && items(wph) <= kMaxItems,
               "%s: %lld blocks of %d rows, %lld requests, %lld KV heads: more than %lld work items",
               fn, (long long)blocks(wph), 32 * wph, (long long)batch, (long long)kv_heads,
               (long long)kMaxItems);
  int cus = 0;
  if (const int rc = ll_device_cus(&cus)) return rc;
  if (win && max_input_len <= 128 && batch * q_heads <= cus) wph = 8;
  a.nblk = (int)blocks(wph);
  a.B = (int)batch;
  a.KVH = (int)kv_heads;
  const int64_t nv = items(wph);
  // persistent grid: one workgroup per CU (the LDS ring takes the whole CU),
  // a multiple of 16 so that the head groups of a (row block, request, KV
  // head) share an XCD on the reversed passes too; more when the items
  // would need more than 64 passes
  int64_t P = std::max<int64_t>(16, cus / 16 * 16);
  if (ll_cdiv(nv, P) > 64) P = (int64_t)ll_cdiv(ll_cdiv(nv, 64), 16) * 16;
  // (windowed: room for the halves of a call with few items)
  P = std::min(P, win && wph < 8 ? 2 * nv : nv);
  const dim3 grid((unsigned)P);
  const dim3 block(512);
  auto launch = [&](auto tag, auto dtag) {
    typedef decltype(tag) T;
    constexpr int D = decltype(dtag)::value;
    constexpr size_t lds = kStages * FaGeom<D>::STAGE_B + 8 * kStages * kBK * 4 + 8 * 256;
    const int idx64 = (a.len64 ? 1 : 0) | (a.shared64 ? 2 : 0) | (a.start64 ? 4 : 0) |
                      (a.req64 ? 8 : 0);
    auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, grid, block, lds, stream, a.seq_len, a.shared, a.start_loc,
                         a.req_idx, idx64, a.nblk, a.B, a.KVH, a.G, (int)nv, a);
    };
    if (wph == 8) {
      go(prefill_attn_fa_kernel<T, D, 8, true>);
    } else if (wph == 1) {
      go(prefill_attn_fa_kernel<T, D, 1, true>);
    } else if (wph == 2) {
      if (win) go(prefill_attn_fa_kernel<T, D, 2, true>);
      else go(prefill_attn_fa_kernel<T, D, 2, false>);
    } else {
      if (win) go(prefill_attn_fa_kernel<T, D, 4, true>);
      else go(prefill_attn_fa_kernel<T, D, 4, false>);
    }
  };
  typedef std::integral_constant<int, 128> D128;
  typedef std::integral_constant<int, 64> D64;
  if (dtype == LL_BF16) {
    if (head_dim == 128) launch(__bf16{}, D128{}); else launch(__bf16{}, D64{});
  } else {
    if (head_dim == 128) launch(_Float16{}, D128{}); else launch(_Float16{}, D64{});
  }
  LL_RETURN_LAUNCH();
}

}  // namespace

extern "C" int ll_prefill_attention(const void* q, int64_t q_stride_tok, int64_t q_stride_h,
                                    const void* k_cache, int64_t k_stride_tok,
                                    int64_t k_stride_head, const void* v_cache,
                                    int64_t v_stride_tok, int64_t v_stride_head, void* out,
                                    int64_t out_stride_tok, int64_t out_stride_h,
                                    const int32_t* req_to_tokens, int64_t req_to_tokens_stride,
                                    const void* b_req_idx, int req_idx_i64,
                                    const void* b_start_loc, int start_loc_i64,
                                    const void* b_seq_len, int seq_len_i64,
                                    const void* b_shared_seq_len, int shared_i64, int64_t batch,
                                    int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                                    int64_t max_input_len, float sm_scale, int dtype,
                                    hipStream_t stream) {
  return prefill_attention("ll_prefill_attention", q, q_stride_tok, q_stride_h, k_cache,
                           k_stride_tok, k_stride_head, v_cache, v_stride_tok, v_stride_head, out,
                           out_stride_tok, out_stride_h, req_to_tokens, req_to_tokens_stride,
                           b_req_idx, req_idx_i64, b_start_loc, start_loc_i64, b_seq_len,
                           seq_len_i64, b_shared_seq_len, shared_i64, batch, q_heads, kv_heads,
                           head_dim, max_input_len, false, 0, 0, sm_scale, dtype, stream);
}

extern "C" int ll_window_prefill_attention(
    const void* q, int64_t q_stride_tok, int64_t q_stride_h, const void* k_cache,
    int64_t k_stride_tok, int64_t k_stride_head, const void* v_cache, int64_t v_stride_tok,
    int64_t v_stride_head, void* out, int64_t out_stride_tok, int64_t out_stride_h,
    const int32_t* req_to_tokens, int64_t req_to_tokens_stride, const void* b_req_idx,
    int req_idx_i64, const void* b_start_loc, int start_loc_i64, const void* b_seq_len,
    int seq_len_i64, const void* b_shared_seq_len, int shared_i64, int64_t batch, int64_t q_heads,
    int64_t kv_heads, int64_t head_dim, int64_t max_input_len, int64_t window, int64_t sinks,
    float sm_scale, int dtype, hipStream_t stream) {
  return prefill_attention("ll_window_prefill_attention", q, q_stride_tok, q_stride_h, k_cache,
                           k_stride_tok, k_stride_head, v_cache, v_stride_tok, v_stride_head, out,
                           out_stride_tok, out_stride_h, req_to_tokens, req_to_tokens_stride,
                           b_req_idx, req_idx_i64, b_start_loc, start_loc_i64, b_seq_len,
                           seq_len_i64, b_shared_seq_len, shared_i64, batch, q_heads, kv_heads,
                           head_dim, max_input_len, true, window, sinks, sm_scale, dtype, stream);
}
