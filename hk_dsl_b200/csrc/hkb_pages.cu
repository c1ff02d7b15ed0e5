// Page bookkeeping under a decode over selected pages: block tables and slots from request lengths,
// a page's summary, the summaries' scores against a query, the budget's best pages.
#include "hkb_common.cuh"
#include "hkb_cluster.cuh"
#include "hkb_sparse.cuh"

extern thread_local int hkb_tls_cuda_error;

namespace hkb {

// ---------------------------------------------------------------------------------
// Block tables, slot mapping and positions from request lengths.
//
// Request i holds old_i tokens and asks for n_i more (n_i < 0: gives -n_i back). With P tokens a page,
// have_i = ceil(old_i / P) pages become want_i = ceil((old_i + n_i) / P); three prefix sums over the requests
// (tokens, pages taken, pages given) place everything: token t belongs to the request whose range of the first
// sum holds t, a new page comes from position count - 1 - (second sum) of the free stack, a page given back
// goes to position count - taken + (third sum). No request waits for another, so one cluster does it all:
// every CTA scans all requests (a chunk of CHUNK at a time: one trip to memory and one three-fold scan), then takes
// its share of the tokens and pages; the in-place updates -- the stack's top, the lengths, the count -- come after a
// cluster barrier, when every CTA has read what it needs of the old state. Deterministic: no atomics.
// Bound: latency (the scan, then two dependent trips), then the stores of 16 bytes a token. Measured, us a call: 64
// requests decoding 3.3 (one CTA of 256 threads), 2048 requests with 48 prompts of 2731 tokens 11.3 (a cluster of sixteen
// CTAs of 1024 threads; of 512 threads 12.0).
// ---------------------------------------------------------------------------------
constexpr int ADV_BLOCKS = 2;                     // 32-token blocks a warp looks up at once

struct AdvanceArgs {
  int* table;
  int64_t table_stride;
  int max_pages;
  int* seq_lens;
  const int* new_tokens;
  int num_reqs, page;
  uint32_t page_magic;             // pos / page = umulhi(pos, magic) >> shift for pos < 2^31, page > 1:
  int page_shift;                  // magic = floor(2^(31 + l) / page) + 1, shift = l - 1, l = ceil(log2 page)
  int* free_pages;
  int* free_count;
  int64_t free_cap;
  int64_t* slots;
  int64_t* positions;
  int64_t tokens;      // rows of slots and positions
  int* q_start;
  int* status;
};

// Sums are held at 2^31 - 1 (adding without going over is associative): no token, page or start past that is real.
struct Sums { int tokens, need, give; };
__device__ __forceinline__ int clamp31(int64_t x) { return (int)max(min(x, (int64_t)0x7fffffff), (int64_t)0); }
__device__ __forceinline__ int sat_add(int x, int y) { return (int)min((uint32_t)x + (uint32_t)y, 0x7fffffffu); }
__device__ __forceinline__ Sums operator+(const Sums& x, const Sums& y) {
  return {sat_add(x.tokens, y.tokens), sat_add(x.need, y.need), sat_add(x.give, y.give)};
}
__device__ __forceinline__ Sums shfl_up(const Sums& s, int by) {
  return {__shfl_up_sync(0xffffffffu, s.tokens, by), __shfl_up_sync(0xffffffffu, s.need, by), __shfl_up_sync(0xffffffffu, s.give, by)};
}
__device__ __forceinline__ Sums shfl_at(const Sums& s, int lane) {
  return {__shfl_sync(0xffffffffu, s.tokens, lane), __shfl_sync(0xffffffffu, s.need, lane), __shfl_sync(0xffffffffu, s.give, lane)};
}

// What a chunk of requests comes to, in shared memory; sums are inclusive and relative to the chunk's beginning.
template <int WARPS, int EACH>
struct AdvChunk {
  static constexpr int CHUNK = WARPS * 32 * EACH;
  int ends[CHUNK], upto[CHUNK], gives[CHUNK];     // tokens, pages taken, pages given
  int old[CHUNK], have[CHUNK];                    // have < 0: refused (-1 - pages)
  Sums warp[WARPS];
};

struct AdvRequest { int old, grow, have, want, status; };

// ceil(tokens / page) for tokens < 2^31, by the multiplication that divides (a division is forty instructions)
__device__ __forceinline__ int adv_pages(const AdvanceArgs& a, int tokens) {
  if (tokens == 0) return 0;
  return a.page == 1 ? tokens : (int)(__umulhi((uint32_t)tokens - 1u, a.page_magic) >> a.page_shift) + 1;
}

__device__ __forceinline__ AdvRequest adv_request(const AdvanceArgs& a, int r) {
  AdvRequest q = {0, 0, 0, 0, HKB_REQ_OK};
  if (r < a.num_reqs) { q.old = max(a.seq_lens[r], 0); q.grow = a.new_tokens[r]; }
  q.have = min(adv_pages(a, q.old), a.max_pages);
  const int after = (int)((uint32_t)q.old + (uint32_t)q.grow);      // old >= 0: only growing can pass 2^31 - 1, and is then negative
  q.want = adv_pages(a, max(after, 0));
  if (q.grow > 0 && (after < 0 || q.want > a.max_pages)) q.status = HKB_REQ_TABLE_FULL;
  return q;
}

// Inclusive sums of this thread's EACH requests, in request order, and the chunk's totals.
template <int WARPS, int EACH>
__device__ __forceinline__ void adv_scan(AdvChunk<WARPS, EACH>& c, const Sums (&v)[EACH], Sums (&incl)[EACH], Sums& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Sums none = {0, 0, 0};
  incl[0] = v[0];
#pragma unroll
  for (int e = 1; e < EACH; ++e) incl[e] = incl[e - 1] + v[e];
  Sums s = incl[EACH - 1];
#pragma unroll
  for (int x = 1; x < 32; x <<= 1) {
    const Sums y = shfl_up(s, x);
    if (lane >= x) s = s + y;
  }
  __syncthreads();                                // the chunk before is done with
  if (lane == 31) c.warp[warp] = s;
  __syncthreads();
  Sums w = lane < WARPS ? c.warp[lane] : none;    // every warp scans the warps' sums
#pragma unroll
  for (int x = 1; x < WARPS; x <<= 1) {
    const Sums y = shfl_up(w, x);
    if (lane >= x) w = w + y;
  }
  total = shfl_at(w, WARPS - 1);
  const Sums warps = shfl_at(w, max(warp - 1, 0)), lanes = shfl_up(s, 1);
  const Sums before = (warp ? warps : none) + (lane ? lanes : none);
#pragma unroll
  for (int e = 0; e < EACH; ++e) incl[e] = before + incl[e];
}

// A chunk's requests: their sums into shared memory, this thread's own into `q`; `before`: the sums of the chunks before.
template <int WARPS, int EACH>
__device__ __forceinline__ void adv_chunk(const AdvanceArgs& a, AdvChunk<WARPS, EACH>& c, int c0, int64_t count,
                                          const Sums& before, Sums& total, AdvRequest (&q)[EACH]) {
  Sums v[EACH], incl[EACH];
#pragma unroll
  for (int e = 0; e < EACH; ++e) q[e] = adv_request(a, c0 + threadIdx.x * EACH + e);
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    v[e].tokens = max(q[e].grow, 0);
    v[e].need = q[e].grow > 0 && q[e].status == HKB_REQ_OK ? max(q[e].want - q[e].have, 0) : 0;
    v[e].give = q[e].grow < 0 ? max(q[e].have - q[e].want, 0) : 0;
  }
  adv_scan(c, v, incl, total);
  if ((int64_t)before.tokens + total.tokens > a.tokens) {  // some of the rows are missing: those requests take no page either
#pragma unroll
    for (int e = 0; e < EACH; ++e)
      if (q[e].grow > 0 && q[e].status == HKB_REQ_OK && (int64_t)before.tokens + incl[e].tokens > a.tokens) {
        q[e].status = HKB_REQ_NO_ROWS;
        v[e].need = 0;
      }
    adv_scan(c, v, incl, total);
  }
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    if (v[e].need > 0 && (int64_t)before.need + incl[e].need > count) q[e].status = HKB_REQ_NO_PAGES;
    const int i = threadIdx.x * EACH + e;
    c.ends[i] = incl[e].tokens; c.upto[i] = incl[e].need; c.gives[i] = incl[e].give;
    c.old[i] = q[e].old;
    c.have[i] = q[e].status == HKB_REQ_OK ? q[e].have : -1 - q[e].have;
  }
  __syncthreads();
}

// The first of n ascending inclusive sums that is greater than x: the request whose range holds x. lo: none before it is.
__device__ __forceinline__ int range_of(const int* ends, int lo, int n, int x) {
  int hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (ends[mid] > x) hi = mid; else lo = mid + 1;
  }
  return lo;
}
// The same for an x that the warp shares: 32 candidates at once.
__device__ __forceinline__ int range_of_warp(const int* ends, int n, int x, int lane) {
  int lo = 0, hi = n;                             // the answer is in [lo, hi)
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32 | 1, at = lo + (lane + 1) * step - 1;        // odd: 32 different banks
    const int m = __popc(__ballot_sync(0xffffffffu, at < hi - 1 && ends[at] <= x));   // groups that lie before it
    lo = lo + m * step;
    hi = min(hi, lo + step);
  }
  return lo;
}

template <int WARPS, int EACH>
__global__ void __launch_bounds__(WARPS * 32, 1) advance_kernel(const AdvanceArgs a) {
  __shared__ AdvChunk<WARPS, EACH> c;
  after_the_last();
  let_the_next();
  constexpr int THREADS = WARPS * 32, CHUNK = THREADS * EACH;
  const int tid = threadIdx.x, lane = tid & 31;
  const int ctas = cluster_size(), rank = cluster_rank();
  const int64_t count = min((int64_t)max(*a.free_count, 0), a.free_cap);
  const uint32_t P = (uint32_t)a.page;

  Sums before = {0, 0, 0}, total;
  int64_t taken = 0;
  AdvRequest q[EACH];
  for (int c0 = 0; c0 < a.num_reqs; c0 += CHUNK) {
    const int n = min(CHUNK, a.num_reqs - c0);
    adv_chunk(a, c, c0, count, before, total, q);
    if ((c0 / CHUNK) % ctas == rank) {
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        const int i = tid * EACH + e;
        if (i >= n) continue;
        a.q_start[c0 + i + 1] = sat_add(before.tokens, c.ends[i]);
        a.status[c0 + i] = q[e].status;
      }
    }
    // This chunk's tokens, dealt to the warps ADV_BLOCKS blocks of 32 at a time (longer runs leave the tokens of many
    // short requests to a few warps). Where they are all one request's, what they share is looked up once; else every
    // lane looks its request up, block by block. A new page's first position is one of the new tokens', whose lane also
    // writes the page into the table. Once one request gets none, none of those after it that need pages gets any (the
    // sum runs on), so the pages handed out are the sum's first ones, in request order.
    const int rows = clamp31(min((int64_t)total.tokens, a.tokens - before.tokens));     // of the chunk
    const int64_t top = count - 1 - before.need;
    int64_t* const slots = a.slots + before.tokens;
    int64_t* const positions = a.positions + before.tokens;
    // one token of request r: its page is table[lp] or, for a new one, last[-lp]
    auto put = [&](int t, uint32_t pos, int have, int* table, const int* last) {
      const uint32_t lp = P == 1 ? pos : __umulhi(pos, a.page_magic) >> a.page_shift;
      const uint32_t off = pos - lp * P;
      int block = -1;
      if (have >= 0) {
        const bool fresh = (int)lp >= have;
        block = fresh ? last[-(int64_t)lp] : table[lp];
        if (fresh && off == 0) table[lp] = block;
      }
      slots[t] = block >= 0 ? (int64_t)block * P + off : -1;
      positions[t] = pos;
    };
    auto enter = [&](int r, uint32_t& shift_r, int& have_r, int*& table_r, const int*& last_r) {
      shift_r = (uint32_t)c.old[r] - (uint32_t)(r ? c.ends[r - 1] : 0);
      have_r = c.have[r];
      table_r = a.table + (int64_t)(c0 + r) * a.table_stride;
      last_r = a.free_pages + (top - (r ? c.upto[r - 1] : 0) + have_r);
    };
    for (int g0 = (rank * WARPS + (tid >> 5)) * 32 * ADV_BLOCKS; g0 < rows; g0 += ctas * WARPS * 32 * ADV_BLOCKS) {
      uint32_t shift;                             // position less token
      int i = range_of_warp(c.ends, n, g0, lane), have;
      int* table;
      const int* last;
      if (g0 + 32 * ADV_BLOCKS <= min(c.ends[i], rows)) {
        enter(i, shift, have, table, last);
#pragma unroll
        for (int u = 0; u < ADV_BLOCKS; ++u) put(g0 + u * 32 + lane, shift + (uint32_t)(g0 + u * 32 + lane), have, table, last);
        continue;
      }
      for (int t0 = g0; t0 < min(g0 + 32 * ADV_BLOCKS, rows); t0 += 32) {
        const int t = t0 + lane;
        // the lane's request: among the next 32, a candidate a lane, by bisection over the lanes; else further on
        const int mine = c.ends[min(i + lane, n - 1)];
        int r = 0;
#pragma unroll
        for (int step = 16; step > 0; step >>= 1)
          if (__shfl_sync(0xffffffffu, mine, r + step - 1) <= t) r += step;
        r += __shfl_sync(0xffffffffu, mine, r) <= t;
        r = min(i + r, n - 1);
        if (t < rows) {
          if (c.ends[r] <= t) r = range_of(c.ends, r, n, t);
          enter(r, shift, have, table, last);
          put(t, shift + (uint32_t)t, have, table, last);
        }
        i = __shfl_sync(0xffffffffu, r, 31);      // where the next block begins, or before
      }
    }
    const int fresh = clamp31(min((int64_t)total.need, count - before.need));
    if ((int64_t)before.need + total.need <= count) {
      taken += total.need;
    } else if (fresh > 0) {                       // short: up to the last request that fits
      const int i = range_of(c.upto, 0, n, fresh);          // the first one past the stack
      taken += i ? c.upto[i - 1] : 0;
    }
    before = before + total;
    // the next adv_scan waits for every thread before it writes
  }
  for (int64_t t = min((int64_t)before.tokens, a.tokens) + rank * THREADS + tid; t < a.tokens; t += ctas * THREADS) {
    a.slots[t] = -1;
    a.positions[t] = 0;
  }
  if (rank == 0 && tid == 0) a.q_start[0] = 0;
  if (ctas > 1) cluster_sync(); else __syncthreads();

  const bool once = a.num_reqs <= CHUNK;          // the one chunk's sums are still in shared memory, its requests in q
  const int64_t given = before.give;
  if (given > 0) {                                // the same in every CTA
    Sums at = {0, 0, 0};
    for (int c0 = 0; c0 < a.num_reqs; c0 += CHUNK) {
      const int n = min(CHUNK, a.num_reqs - c0);
      if (!once) adv_chunk(a, c, c0, count, at, total, q);
      const int64_t at0 = count - taken + at.give;
      const int pages = clamp31(min((int64_t)total.give, a.free_cap - at0));
      for (int64_t y = rank * THREADS + tid; y < pages; y += ctas * THREADS) {      // `pages` may be 2^31 - 1
        const int x = (int)y, i = range_of(c.gives, 0, n, x);                       // its last pages, gives[i] - x of them from here
        a.free_pages[at0 + x] = a.table[(int64_t)(c0 + i) * a.table_stride + c.have[i] - (c.gives[i] - x)];
      }
      at = at + total;
    }
    if (!once) { if (ctas > 1) cluster_sync(); else __syncthreads(); }   // the lengths are read for the last time
  }
  if (rank == 0 && tid == 0) *a.free_count = (int)min(count - taken + given, a.free_cap);
  for (int ch = rank; ch * CHUNK < a.num_reqs; ch += ctas)
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      const int r = ch * CHUNK + tid * EACH + e;
      if (r >= a.num_reqs) continue;
      if (!once) { q[e] = adv_request(a, r); q[e].status = a.status[r]; }      // which this thread wrote
      a.seq_lens[r] = q[e].status == HKB_REQ_OK ? max(q[e].old + q[e].grow, 0) : q[e].old;
    }
}

// ---------------------------------------------------------------------------------
// A page's summary: the least and the greatest key of every channel, over the page's tokens below the
// sequence's length. Values of the cache's own type, so nothing is rounded. A warp takes a (page, kv head) -- of
// pages of more than 32 tokens the CTA's four warps share it, or a decode step's few large pages would each be one
// warp's chain of trips to memory: its lanes hold 16-byte chunks of a row, 32 / chunks rows at a time, and fold them
// with packed minima and maxima that keep a NaN. Bound: bytes (the keys once, two rows a page out). Measured at head size
// 128, eight kv heads: 4 x 8192 new tokens 12.4 us = 6.1 TB/s; 64 decoding sequences 2.0 us, with pages of 256 tokens
// 6.7 (15.0 with a warp a page). Keys through a cp.async ring as the scores': 14.4 to 16.7.
// ---------------------------------------------------------------------------------
constexpr int BOUNDS_WARPS = 4;

struct BoundsArgs {
  uint8_t* bounds;                 // strides in bytes; low row, then high row, row_bytes each
  int64_t b_stride_block, b_stride_head;
  const uint8_t* k;
  int64_t k_stride_block, k_stride_token, k_stride_head;
  int num_blocks;
  const int* table;
  int64_t table_stride;
  int max_pages;
  const int* seq_lens;
  const int* q_start;              // null: one new token a sequence
  int tokens;                      // the step's rows; a start past them counts as it
  int num_seqs, num_kv_heads, page;
  int items;                       // (sequence, page) pairs the grid covers
  bool many;                       // more than the machine holds at once
};

template <int KIND>
struct Pair;                       // two values of a 16-bit type in 32 bits
template <>
struct Pair<HKB_KV_BF16> {
  static __device__ __forceinline__ uint32_t least(uint32_t x, uint32_t y) {
    uint32_t r; asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y)); return r;
  }
  static __device__ __forceinline__ uint32_t most(uint32_t x, uint32_t y) {
    uint32_t r; asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y)); return r;
  }
};
template <>
struct Pair<HKB_KV_F16> {
  static __device__ __forceinline__ uint32_t least(uint32_t x, uint32_t y) {
    uint32_t r; asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y)); return r;
  }
  static __device__ __forceinline__ uint32_t most(uint32_t x, uint32_t y) {
    uint32_t r; asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y)); return r;
  }
};

__device__ __forceinline__ uint32_t f16x2_to_e4m3x2(uint32_t h2) {   // exact for values that came from e4m3
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(h2));
  return r;
}

// KIND: HKB_KV_*; CPR: 16-byte chunks a row (head_dim x element size / 16); SHARE: a CTA a (page, kv head)
template <int KIND, int CPR, bool SHARE>
__global__ void __launch_bounds__(BOUNDS_WARPS * 32) bounds_kernel(const BoundsArgs a) {
  constexpr bool FP8 = KIND == HKB_KV_FP8_E4M3;
  using Pr = Pair<FP8 ? HKB_KV_F16 : KIND>;       // e4m3 widens to f16 exactly
  constexpr int REGS = FP8 ? 8 : 4;               // pairs a 16-byte chunk holds
  constexpr int RPI = 32 / CPR, UNROLL = 8;
  constexpr int STEP = RPI * UNROLL * (SHARE ? BOUNDS_WARPS : 1);
  after_the_last();
  let_the_next();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t unit = SHARE ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * BOUNDS_WARPS + warp;
  const int item = (int)(unit / a.num_kv_heads), head = (int)(unit % a.num_kv_heads);
  if (item >= a.items) return;

  // which page of which sequence. With query starts, sequence r has the items from start[r] / page + 2 r on:
  // its q new tokens touch at most q / page + 2 pages, and so many items it has. Requests that got no rows leave starts
  // past the step's; held at the rows, everyone's items lie in the grid, two at least.
  int r = item, page;
  int len;
  if (a.q_start) {
    auto start = [&](int i) { return min(max(__ldg(a.q_start + i), 0), a.tokens); };
    int lo = 0, hi = a.num_seqs;                  // the last r whose items begin at or before this one is in [lo, hi)
    while (hi - lo > 1) {                         // 32 candidates at once
      const int step = (hi - lo + 31) / 32, at = lo + lane * step;
      const bool below = at < hi && start(at) / a.page + 2 * at <= item;
      const int m = max(__popc(__ballot_sync(0xffffffffu, below)), 1);
      lo += (m - 1) * step;
      hi = min(hi, lo + step);
    }
    r = lo;
    const int s0 = start(r), q = start(r + 1) - s0;
    len = __ldg(a.seq_lens + r);
    if (len <= 0) return;
    const int64_t k = (int64_t)item - (s0 / a.page + 2 * (int64_t)r);
    const int64_t p = max(len - max(q, 1), 0) / a.page + k;   // no new token: the last page, it may have lost some
    if (k < 0 || p >= a.max_pages) return;
    page = (int)p;
  } else {
    len = __ldg(a.seq_lens + r);
    if (len <= 0) return;
    page = (len - 1) / a.page;
  }
  const int64_t first_tok = (int64_t)page * a.page;
  if (first_tok >= len || page >= a.max_pages) return;
  const int live = min((int64_t)a.page, len - first_tok);
  const int block = __ldg(a.table + (int64_t)r * a.table_stride + page);
  if ((unsigned)block >= (unsigned)a.num_blocks) return;

  const uint8_t* src = a.k + (int64_t)block * a.k_stride_block + (int64_t)head * a.k_stride_head + (lane % CPR) * 16;
  uint32_t low[REGS], high[REGS];
  bool any = false;
  int t0 = SHARE ? warp * RPI * UNROLL : 0;
  do {                                            // at least once: a warp without rows of its own reads the last live one
    uint4 v[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {            // a row past the last live one: the last one again
      const uint8_t* at = src + (int64_t)min(t0 + u * RPI + lane / CPR, live - 1) * a.k_stride_token;
      // Many pages' keys pass through, with no place in L1 (12.4 against 14.8 us for 4 x 8192 tokens); of a decode step's
      // few the plain load is the quicker (2.0 against 2.4 us for 64 sequences).
      if (a.many)
        asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(v[u].x), "=r"(v[u].y), "=r"(v[u].z), "=r"(v[u].w) : "l"(at));
      else
        v[u] = __ldg(reinterpret_cast<const uint4*>(at));
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const uint32_t w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
      for (int i = 0; i < REGS; ++i) {
        const uint32_t x = FP8 ? e4m3x2_to_f16x2(w[(i / 2) & 3] >> (i & 1 ? 16 : 0)) : w[i & 3];
        low[i] = any || u ? Pr::least(low[i], x) : x;
        high[i] = any || u ? Pr::most(high[i], x) : x;
      }
    }
    any = true;
    t0 += STEP;
  } while (t0 < live);
#pragma unroll
  for (int x = CPR; x < 32; x <<= 1)
#pragma unroll
    for (int i = 0; i < REGS; ++i) {
      low[i] = Pr::least(low[i], __shfl_xor_sync(0xffffffffu, low[i], x));
      high[i] = Pr::most(high[i], __shfl_xor_sync(0xffffffffu, high[i], x));
    }
  if constexpr (SHARE) {
    __shared__ uint32_t fold[BOUNDS_WARPS - 1][2 * REGS][CPR];
    if (warp > 0 && lane < CPR)
#pragma unroll
      for (int i = 0; i < REGS; ++i) { fold[warp - 1][i][lane] = low[i]; fold[warp - 1][REGS + i][lane] = high[i]; }
    __syncthreads();
    if (warp > 0 || lane >= CPR) return;
#pragma unroll
    for (int w = 0; w < BOUNDS_WARPS - 1; ++w)
#pragma unroll
      for (int i = 0; i < REGS; ++i) {
        low[i] = Pr::least(low[i], fold[w][i][lane]);
        high[i] = Pr::most(high[i], fold[w][REGS + i][lane]);
      }
  }
  if (lane >= CPR) return;
  uint8_t* dst = a.bounds + (int64_t)block * a.b_stride_block + (int64_t)head * a.b_stride_head + lane * 16;
  uint32_t o[2][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (FP8) {
      o[0][i] = f16x2_to_e4m3x2(low[(2 * i) % REGS]) | f16x2_to_e4m3x2(low[(2 * i + 1) % REGS]) << 16;
      o[1][i] = f16x2_to_e4m3x2(high[(2 * i) % REGS]) | f16x2_to_e4m3x2(high[(2 * i + 1) % REGS]) << 16;
    } else {
      o[0][i] = low[i]; o[1][i] = high[i];
    }
  }
  *reinterpret_cast<uint4*>(dst) = make_uint4(o[0][0], o[0][1], o[0][2], o[0][3]);
  *reinterpret_cast<uint4*>(dst + CPR * 16) = make_uint4(o[1][0], o[1][1], o[1][2], o[1][3]);
}

// ---------------------------------------------------------------------------------
// Page scores. score[row, kv head, page] = scale k_scale max_g sum_d max(q_gd low_d, q_gd high_d): no key of the
// page can have a greater logit with any query head g of the group. With q+ = max(q, 0), q- = min(q, 0) the sum
// is q-.low + q+.high, one product of depth 2 head_dim with the summary as it lies in memory (low, then high):
// mma.sync.m16n8k16, sixteen pages on M, the group's heads on N, as the decode walk multiplies. A warp takes a
// (row, kv head, range of pages) and loads its fragments straight from memory: the contraction runs over dims,
// so lane t of a quad takes eight (fp8: sixteen) consecutive ones and the query's fragments are dealt alike. Since a
// lane then reads nothing that another one fetched, the copies run through a cp.async ring in which every lane has its
// own 16-byte places: asynchronous and deep as a walk's ring, without a barrier or a swizzle.
// Bound: bytes (a summary is 2 rows a page where the attention reads 2 rows a token). Measured: 2 x 8192 pages, eight kv
// heads of eight query heads, 13.2 us = 5.1 TB/s (loads straight into registers, two tiles a warp: 14.7 to 16; rings in
// CTAs of four warps instead of one: 17.0, one chain of products a score: 17.3); four sequences of up to 32 pages 2.0 us.
// ---------------------------------------------------------------------------------
constexpr int SCORE_WARPS = 1;
template <int D, bool FP8>
struct ScoreRing {
  static constexpr int TILE = 16 * 2 * D * (FP8 ? 1 : 2);                       // sixteen pages' summaries
  static constexpr int STAGES = TILE >= 16384 ? 2 : TILE >= 8192 ? 3 : 4;
  static constexpr int BYTES = SCORE_WARPS * STAGES * TILE;
};

struct ScoreArgs {
  float* scores;
  int64_t s_stride_row, s_stride_head;
  int columns;
  const __nv_bfloat16* q;
  int64_t q_stride_row, q_stride_head;
  const uint8_t* bounds;           // strides in bytes
  int64_t b_stride_block, b_stride_head;
  int num_blocks;
  const int* table;
  int64_t table_stride;
  const int* seq_lens;
  int page, group;
  float scale;
  const float* k_scale;
  int tiles_per_warp;
};

__device__ __forceinline__ float max_nan(float x, float y) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}

// A page's best product from the definition, by one warp: max_g sum_d max(q_gd low_d, q_gd high_d) for 16-bit summaries.
// Of an infinite bound only the product that counts is in it. `q`: the group's first head; `low`: the page's summary.
template <int KIND, int D>
__device__ __forceinline__ float score_by_definition(const __nv_bfloat16* q, int64_t q_stride_head, int group, const uint8_t* low, int lane) {
  auto wide = [](uint32_t x) {
    return KIND == HKB_KV_F16 ? __half22float2(*reinterpret_cast<__half2*>(&x)) : make_float2(bf16lo(x), bf16hi(x));
  };
  float best = -INFINITY;
#pragma unroll 1
  for (int h = 0; h < group; ++h) {
    float s = 0.f;
#pragma unroll 1
    for (int d = lane * 2; d < D; d += 64) {
      const float2 x = wide(__ldg(reinterpret_cast<const uint32_t*>(q + (int64_t)h * q_stride_head + d)));
      const float2 a = wide(__ldg(reinterpret_cast<const uint32_t*>(low + d * 2)));
      const float2 b = wide(__ldg(reinterpret_cast<const uint32_t*>(low + (D + d) * 2)));
      s += max_nan(x.x * a.x, x.x * b.x) + max_nan(x.y * a.y, x.y * b.y);
    }
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    best = max_nan(best, s);
  }
  return best;
}

// Whether a NaN is among a group's 16-bit query heads.
template <int KIND, int D>
__device__ __forceinline__ int query_is_broken(const __nv_bfloat16* q, int64_t q_stride_head, int group, int lane) {
  constexpr uint32_t INF = KIND == HKB_KV_F16 ? 0x7c00u : 0x7f80u;
  bool nan = false;
#pragma unroll 1
  for (int x = lane; x < group * (D / 8); x += 32) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(q + (int64_t)(x / (D / 8)) * q_stride_head + x % (D / 8) * 8));
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) nan |= (w[i] & 0x7fffu) > INF || (w[i] >> 16 & 0x7fffu) > INF;
  }
  return __any_sync(0xffffffffu, nan);
}

template <int KIND, int D, int NT>
__global__ void __launch_bounds__(SCORE_WARPS * 32, 8) scores_kernel(const ScoreArgs a) {
  constexpr bool FP8 = KIND == HKB_KV_FP8_E4M3, F16 = KIND != HKB_KV_BF16;   // e4m3 widens to f16 exactly
  using Pr = Pair<F16 ? HKB_KV_F16 : HKB_KV_BF16>;
  constexpr int EPC = FP8 ? 16 : 8;            // elements of a lane's 16-byte chunk
  constexpr int STEPS = D / (4 * EPC);         // chunks a lane reads of one row of D values
  constexpr int MPC = EPC / 4;                 // mma a chunk feeds
  constexpr int CHAINS = NT == 1 ? 4 : 2;
  using Ring = ScoreRing<D, FP8>;
  after_the_last();
  let_the_next();
  extern __shared__ __align__(128) uint8_t hkb_smem[];
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int head = blockIdx.y, row = blockIdx.z;
  const int64_t first64 = ((int64_t)blockIdx.x * SCORE_WARPS + (threadIdx.x >> 5)) * a.tiles_per_warp * 16;
  if (first64 >= a.columns) return;
  const int first = (int)first64, last = (int)min(first64 + (int64_t)a.tiles_per_warp * 16, (int64_t)a.columns);
  const int* table = a.table + (int64_t)row * a.table_stride;
  // a page id a lane, two tiles at once and the next two beside them; columns past the sequence hold any number
  auto look_up = [&](int p0) { return p0 + lane < last ? __ldg(table + p0 + lane) : 0; };
  int ids = look_up(first), ids_next = look_up(first + 32);       // beside the length, not behind it
  const int len = max(__ldg(a.seq_lens + row), 0);
  const int pages = (int)min(((int64_t)len + a.page - 1) / a.page, (int64_t)a.columns);
  float* out = a.scores + (int64_t)row * a.s_stride_row + (int64_t)head * a.s_stride_head;
  for (int p = max(first, pages) + lane; p < last; p += 32) out[p] = -INFINITY;
  const int end = min(last, pages);
  if (first >= end) return;

  const uint8_t* base = a.bounds + (int64_t)head * a.b_stride_head + t * 16;
  const uint32_t ring = smem_u32(hkb_smem) + (threadIdx.x >> 5) * (Ring::STAGES * Ring::TILE) + lane * 16;
  int next = first;                            // the next tile to fetch
  auto fetch = [&](int stage) {
    if (next < end) {
      const uint32_t dst = ring + stage * Ring::TILE;
#pragma unroll
      for (int j = 0; j < 2; ++j) {            // pages g and g + 8; an id is clamped into the pool
        const int id = __shfl_sync(0xffffffffu, ids, ((next - first) & 16) + g + 8 * j);
        const uint8_t* src = base + (int64_t)min(max(id, 0), a.num_blocks - 1) * a.b_stride_block;
#pragma unroll
        for (int x = 0; x < 2 * STEPS; ++x) cp_async16(dst + (x * 2 + j) * 512, src + x * 64);
      }
      next += 16;
      if (!((next - first) & 16)) { ids = ids_next; ids_next = look_up(next + 32); }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int k = 0; k < Ring::STAGES - 1; ++k) fetch(k);

  // the query's fragments: head g of the column tile, the dims of this lane's chunks
  uint32_t qf[NT][STEPS][EPC / 2];
  float unit[NT];                              // the power of two that an fp8 cache's query was scaled by
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int h = nt * 8 + g;
    const __nv_bfloat16* qp = a.q + (int64_t)row * a.q_stride_row + (int64_t)(head * a.group + h) * a.q_stride_head;
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
#pragma unroll
      for (int j = 0; j < EPC / 8; ++j) {
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (h < a.group) v = __ldg(reinterpret_cast<const uint4*>(qp + (s * 4 + t) * EPC + j * 8));
        qf[nt][s][j * 4] = v.x; qf[nt][s][j * 4 + 1] = v.y; qf[nt][s][j * 4 + 2] = v.z; qf[nt][s][j * 4 + 3] = v.w;
      }
    unit[nt] = 1.f;
    if (FP8) {
      float top = 0.f;
#pragma unroll
      for (int s = 0; s < STEPS; ++s)
#pragma unroll
        for (int i = 0; i < EPC / 2; ++i)
          top = fmaxf(top, fmaxf(fabsf(bf16lo(qf[nt][s][i])), fabsf(bf16hi(qf[nt][s][i]))));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const F16Scale f = f16_scale(top);
      unit[nt] = f.up;
#pragma unroll
      for (int s = 0; s < STEPS; ++s)
#pragma unroll
        for (int i = 0; i < EPC / 2; ++i)
          qf[nt][s][i] = pack_f16x2(bf16lo(qf[nt][s][i]) * f.down, bf16hi(qf[nt][s][i]) * f.down);
    }
  }
  const float factor = a.scale * (a.k_scale ? __ldg(a.k_scale) : 1.f);

  int stage = 0, stage_next = Ring::STAGES - 1;
  int broken = -1;                             // whether the query has a NaN: not known
  for (int p0 = first; p0 < end; p0 += 16) {
    cp_async_wait<Ring::STAGES - 2>();         // this lane's own copies: nobody else's are read
    const uint32_t tile = ring + stage * Ring::TILE;
    stage = stage + 1 == Ring::STAGES ? 0 : stage + 1;
    float part[CHAINS][NT][4];                 // several chains of products, so that none waits for the one before it
#pragma unroll
    for (int c = 0; c < CHAINS; ++c)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) part[c][nt][i] = 0.f;
#pragma unroll
    for (int half = 0; half < 2; ++half) {     // low bounds meet the query's negative parts, high bounds the positive
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        const uint4 v0 = lds128(tile + ((half * STEPS + s) * 2) * 512), v1 = lds128(tile + ((half * STEPS + s) * 2 + 1) * 512);
        const uint32_t x[2][4] = {{v0.x, v0.y, v0.z, v0.w}, {v1.x, v1.y, v1.z, v1.w}};
#pragma unroll
        for (int m = 0; m < MPC; ++m) {
          uint32_t f[4];
          if (FP8) {
            f[0] = e4m3x2_to_f16x2(x[0][m]); f[1] = e4m3x2_to_f16x2(x[1][m]);
            f[2] = e4m3x2_to_f16x2(x[0][m] >> 16); f[3] = e4m3x2_to_f16x2(x[1][m] >> 16);
          } else {
            f[0] = x[0][(2 * m) & 3]; f[1] = x[1][(2 * m) & 3]; f[2] = x[0][(2 * m + 1) & 3]; f[3] = x[1][(2 * m + 1) & 3];
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            uint32_t b[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) b[i] = half ? Pr::most(qf[nt][s][2 * m + i], 0u) : Pr::least(qf[nt][s][2 * m + i], 0u);
            mma16<F16>(part[(half * (CHAINS / 2) + m % (CHAINS / 2))][nt], f, b);
          }
        }
      }
    }
    float sc[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        sc[nt][i] = CHAINS == 4 ? (part[0][nt][i] + part[1][nt][i]) + (part[2][nt][i] + part[CHAINS - 1][nt][i]) : part[0][nt][i] + part[1][nt][i];
    fetch(stage_next);                         // over the tile before this one
    stage_next = stage_next + 1 == Ring::STAGES ? 0 : stage_next + 1;
    // the greatest over the group's heads: this lane holds heads 2t, 2t + 1 of pages g and g + 8
    float best[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int h = nt * 8 + 2 * t + c;
        const float u = FP8 ? __shfl_sync(0xffffffffu, unit[nt], (2 * t + c) * 4) : 1.f;   // that head's own power of two
        if (h < a.group) {
          best[0] = max_nan(best[0], sc[nt][c] * u);
          best[1] = max_nan(best[1], sc[nt][c + 2] * u);
        }
      }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      best[j] = max_nan(best[j], __shfl_xor_sync(0xffffffffu, best[j], 1));
      best[j] = max_nan(best[j], __shfl_xor_sync(0xffffffffu, best[j], 2));
    }
    const int p = p0 + g + 8 * (t & 1);
    float mine = t & 1 ? best[1] : best[0];
    if constexpr (!FP8) {
      // The rewritten product meets the half of the wrong sign with a zero, and of an infinite bound that is NaN though
      // max(q low, q high) may be finite: pages without a number are computed again. (e4m3 has no infinities.) Not if the
      // query has none itself, or its row would cost a batch some hundred microseconds.
      unsigned bad = __ballot_sync(0xffffffffu, t < 2 && p < end && mine != mine);
      if (bad && broken < 0)
        broken = query_is_broken<KIND, D>(a.q + (int64_t)row * a.q_stride_row + (int64_t)(head * a.group) * a.q_stride_head, a.q_stride_head, a.group, lane);
      if (broken > 0) bad = 0;
      for (; bad; bad &= bad - 1) {
        const int from = __ffs(bad) - 1;
        const int id = __ldg(table + __shfl_sync(0xffffffffu, p, from));
        const uint8_t* low = a.bounds + (int64_t)min(max(id, 0), a.num_blocks - 1) * a.b_stride_block + (int64_t)head * a.b_stride_head;
        const float again = score_by_definition<KIND, D>(
            a.q + (int64_t)row * a.q_stride_row + (int64_t)(head * a.group) * a.q_stride_head, a.q_stride_head, a.group, low, lane);
        if (lane == from) mine = again;
      }
    }
    if (t < 2 && p < end) out[p] = mine * factor;
  }
  cp_async_wait<0>();
}

// ---------------------------------------------------------------------------------
// The budget's best pages of a (row, kv head): the first `first` and the last `last` pages always, then by score
// downwards, ties to the lowest page; written in ascending order, -1 behind. A score becomes a 32-bit key whose
// order is the scores' (NaN above everything: a broken key shows in the answer instead of being left out).
// Integers throughout: the answer depends on no order of anything. Bound: latency.
//
// Narrow tables (select_warp_kernel): a warp takes a (row, kv head), its lanes hold the keys in registers, every
// 32nd page a lane, and the border is bisected between the least and the greatest key: a step is one comparison a
// key and one warp-wide sum, and it ends as soon as a step leaves exactly the budget above it -- ten-odd steps, no
// barrier, no memory but the one trip for the scores.
//
// Wide ones (select_kernel): a CTA takes it, EACH keys a thread in registers where the table's width lets it, and the
// border is found by digits: the keys, less the least of them and shifted up to the full width, fall into 2048 bins
// of a histogram in shared memory (so shifted, scores that differ little still spread over the bins and their atomics
// over the banks); the bin that the border falls into is cut into 2048 again until all of it is taken or it is one value.
// ---------------------------------------------------------------------------------
constexpr int SELECT_BINS = 2048, SELECT_BITS = 11;

struct SelectArgs {
  int* pages;
  int64_t p_stride_row, p_stride_head;
  int budget;
  const float* scores;
  int64_t s_stride_row, s_stride_head;
  int columns;
  const int* seq_lens;
  int page, first, last;
  int num_kv_heads, items;         // items: rows x kv heads
};

__device__ __forceinline__ uint32_t score_key(float x) {
  x += 0.f;                                      // -0 and 0 are one score
  const uint32_t b = __float_as_uint(x);
  if (x != x) return 0xfffffffeu;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

constexpr int SELECT_WARPS = 4;

template <int EACH>
__global__ void __launch_bounds__(SELECT_WARPS * 32, 1) select_warp_kernel(const SelectArgs a) {
  after_the_last();
  let_the_next();
  const int lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * SELECT_WARPS + (threadIdx.x >> 5);
  if (item >= a.items) return;
  const int64_t row = item / a.num_kv_heads, head = item - row * a.num_kv_heads;
  const int len = max(__ldg(a.seq_lens + row), 0);
  int* out = a.pages + row * a.p_stride_row + head * a.p_stride_head;
  const float* in = a.scores + row * a.s_stride_row + head * a.s_stride_head;
  // every column's key is asked for beside the length, not behind it
  float x[EACH];
#pragma unroll
  for (int e = 0; e < EACH; ++e) x[e] = e * 32 + lane < a.columns ? __ldg(in + e * 32 + lane) : 0.f;
  const int n = (int)min(((int64_t)len + a.page - 1) / a.page, (int64_t)a.columns);
  if (n <= a.budget) {
    for (int i = lane; i < a.budget; i += 32) out[i] = i < n ? i : -1;
    return;
  }
  const int end = n - a.last;
  int want = a.budget - a.first - a.last;         // of the candidates, pages first .. end
  uint32_t key[EACH], least = 0xffffffffu, most = 0u;
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int p = e * 32 + lane;
    key[e] = score_key(x[e]);
    if (p >= a.first && p < end) { least = min(least, key[e]); most = max(most, key[e]); }
  }
  least = __reduce_min_sync(0xffffffffu, least);
  most = __reduce_max_sync(0xffffffffu, most);
  // The greatest `lo` that at least `want` candidates reach; `reach` of them do. Keys that no candidate can have
  // stand for the pages always kept (above all) and those past the sequence (key 0 below all: a score's is at least 2^22).
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int p = e * 32 + lane;
    if (p < a.first || p >= end) key[e] = p < n ? 0xffffffffu : 0u;
  }
  const int kept = a.first + a.last;
  uint32_t lo = want > 0 ? least : 0xffffffffu, hi = most;     // in [lo, hi]
  int reach = want > 0 ? end - a.first : 0;
  while (lo < hi && reach != want) {
    const uint32_t mid = lo + ((hi - lo) >> 1) + 1u;           // lo < mid <= hi
    int c = 0;
#pragma unroll
    for (int e = 0; e < EACH; ++e) c += key[e] >= mid;
    c = __reduce_add_sync(0xffffffffu, c) - kept;
    if (c >= want) { lo = mid; reach = c; } else hi = mid - 1u;
  }
  // Taken: keys above lo, and of those equal to it the first that there is room for.
  const bool all = reach == want;
  int at = 0;
  // ties: how many of the keys equal to lo are taken
  int ties = 0x7fffffff;
  if (!all) {
    int c = 0;
#pragma unroll
    for (int e = 0; e < EACH; ++e) c += key[e] > lo;
    ties = want - (__reduce_add_sync(0xffffffffu, c) - kept);
  }
  const unsigned below = (1u << lane) - 1u;
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const bool tie = !all && key[e] == lo;
    const unsigned t = __ballot_sync(0xffffffffu, tie);
    const bool take = key[e] > lo || (all && key[e] == lo) || (tie && __popc(t & below) < ties);
    const unsigned w = __ballot_sync(0xffffffffu, take);
    if (take) out[at + __popc(w & below)] = e * 32 + lane;
    at += __popc(w);
    ties -= min(ties, __popc(t));
  }
}

// Inclusive sum over the CTA's threads; `sums` is one value a warp, free to be written (a barrier behind its last read).
template <int THREADS, class T>
__device__ __forceinline__ T select_scan(T v, T* sums, T& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int x = 1; x < 32; x <<= 1) {
    const T y = __shfl_up_sync(0xffffffffu, v, x);
    if (lane >= x) v += y;
  }
  if (lane == 31) sums[warp] = v;
  __syncthreads();
  T w = lane < THREADS / 32 ? sums[lane] : 0;
  const T own = w;
#pragma unroll
  for (int x = 1; x < THREADS / 32; x <<= 1) {
    const T y = __shfl_up_sync(0xffffffffu, w, x);
    if (lane >= x) w += y;
  }
  total = __shfl_sync(0xffffffffu, w, THREADS / 32 - 1);
  return v + __shfl_sync(0xffffffffu, w - own, warp);
}

// RESIDENT: THREADS x EACH covers the row; otherwise the keys are read again for every pass, THREADS x EACH at a time.
template <int THREADS, int EACH, bool RESIDENT>
__global__ void __launch_bounds__(THREADS) select_kernel(const SelectArgs a) {
  constexpr int SPAN = THREADS * EACH;
  __shared__ int hist[SELECT_BINS];
  __shared__ uint32_t ends[2][THREADS / 32];
  __shared__ int sums[2][THREADS / 32];
  __shared__ uint64_t places[2][THREADS / 32];
  // of every 32 consecutive pages: which lie above the border, which on it, and how many do before them
  constexpr int WORDS = SPAN / 32;
  __shared__ uint32_t above_bits[WORDS], tie_bits[WORDS];
  __shared__ uint64_t before[WORDS];
  __shared__ int first_of[WORDS];
  __shared__ int s_bin, s_above, s_in;
  constexpr int MINE = SELECT_BINS / THREADS;
  after_the_last();
  let_the_next();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int head = blockIdx.y, row = blockIdx.x;
  int* out = a.pages + (int64_t)row * a.p_stride_row + (int64_t)head * a.p_stride_head;
  const float* in = a.scores + (int64_t)row * a.s_stride_row + (int64_t)head * a.s_stride_head + a.first;
  uint32_t key[EACH];
  auto load = [&](int p0, int end) {              // every THREADS-th page a thread
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      const int p = p0 + e * THREADS + tid;
      key[e] = p < end ? score_key(__ldg(in + p)) : 0u;
    }
  };
  if (RESIDENT) load(0, a.columns - a.first);     // beside the length, not behind it; the columns past it are not used
  const int len = max(__ldg(a.seq_lens + row), 0);
  const int n = (int)min(((int64_t)len + a.page - 1) / a.page, (int64_t)a.columns);
  if (n <= a.budget) {
    for (int i = tid; i < a.budget; i += THREADS) out[i] = i < n ? i : -1;
    return;
  }
  // the pages that are always kept, then the candidates between them
  for (int i = tid; i < a.first; i += THREADS) out[i] = i;
  for (int i = tid; i < a.last; i += THREADS) out[a.budget - a.last + i] = n - a.last + i;
  const int m = n - a.first - a.last;
  int want = a.budget - a.first - a.last;         // of the candidates not yet decided
  if (want == 0) return;
  out += a.first;

#pragma unroll
  for (int i = 0; i < MINE; ++i) hist[tid * MINE + i] = 0;
  // columns past the candidates have key 0, which no score has (the least is 2^22)
  if (RESIDENT)
#pragma unroll
    for (int e = 0; e < EACH; ++e)
      if (e * THREADS + tid >= m) key[e] = 0u;
  uint32_t least = 0xffffffffu, most = 0u;         // `least` one less than it is, so that key 0 does not count
  for (int p0 = 0; p0 < m; p0 += SPAN) {
    if (!RESIDENT) load(p0, m);
#pragma unroll
    for (int e = 0; e < EACH; ++e) { least = min(least, key[e] - 1u); most = max(most, key[e]); }
  }
  least = __reduce_min_sync(0xffffffffu, least);
  most = __reduce_max_sync(0xffffffffu, most);
  if (lane == 0) { ends[0][warp] = least; ends[1][warp] = most; }
  __syncthreads();
  least = __reduce_min_sync(0xffffffffu, lane < THREADS / 32 ? ends[0][lane] : 0xffffffffu) + 1u;
  most = __reduce_max_sync(0xffffffffu, lane < THREADS / 32 ? ends[1][lane] : 0u);

  // Keys from `base` on that are below base + 2^(32 - shift) are undecided; all greater ones are taken.
  uint32_t base = least;
  int shift = __clz(most - least), which = 0;     // 32: they are all one value
  bool whole = false, first_pass = true;          // whole: all undecided keys are taken
  while (shift < 32) {
    for (int p0 = 0; p0 < m; p0 += SPAN) {
      if (!RESIDENT) load(p0, m);
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        const uint32_t x = key[e] - base;         // at first every key lies in the range; then one below base wraps to a great x
        if (first_pass ? key[e] != 0u : key[e] >= base && (x >> (31 - shift)) <= 1u)
          atomicAdd(&hist[(x << shift) >> (32 - SELECT_BITS)], 1);
      }
    }
    first_pass = false;
    __syncthreads();
    // the bin in which the keys, counted from the top, reach `want`; the bins are cleared for the next pass
    int bins[MINE], mine = 0;
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
      bins[i] = hist[SELECT_BINS - 1 - tid * MINE - i];
      hist[SELECT_BINS - 1 - tid * MINE - i] = 0;
      mine += bins[i];
    }
    int total;
    int above = select_scan<THREADS>(mine, sums[which], total) - mine;
    which ^= 1;
    if (above < want && above + mine >= want) {   // one thread
      int i = 0;
#pragma unroll
      for (int j = 0; j < MINE - 1; ++j)
        if (i == j && above + bins[j] < want) { above += bins[j]; ++i; }
      int in_bin = 0;
#pragma unroll
      for (int j = 0; j < MINE; ++j)
        if (i == j) in_bin = bins[j];
      s_bin = SELECT_BINS - 1 - tid * MINE - i; s_above = above; s_in = in_bin;
    }
    __syncthreads();
    want -= s_above;
    base += ((uint32_t)s_bin << (32 - SELECT_BITS)) >> shift;
    if (s_in == want) { whole = true; break; }
    shift += SELECT_BITS;                         // 32 and more: the bin is one value
  }
  // Taken: keys above `base`; of those equal to it the first `want` -- or all from it on, where `whole`.
  const unsigned below = (1u << lane) - 1u;
  static_assert(WORDS <= THREADS, "a word a thread");
  if (whole) {                                    // nearly always: no ties to count
    int done = 0;
    for (int p0 = 0; p0 < m; p0 += SPAN) {
      if (!RESIDENT) load(p0, m);
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        const uint32_t up = __ballot_sync(0xffffffffu, key[e] >= base);
        if (lane == 0) above_bits[e * (THREADS / 32) + warp] = up;
      }
      __syncthreads();
      const int mine = tid < WORDS ? __popc(above_bits[tid]) : 0;
      int total;
      const int incl = done + select_scan<THREADS>(mine, sums[which], total);
      if (tid < WORDS) first_of[tid] = incl - mine;
      __syncthreads();
      which ^= 1;
      done += total;
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        const int w = e * (THREADS / 32) + warp;
        if (key[e] >= base) out[first_of[w] + __popc(above_bits[w] & below)] = a.first + p0 + e * THREADS + tid;
      }
      if (!RESIDENT) __syncthreads();             // the words are written again
    }
    return;
  }
  uint64_t done = 0;                              // keys above in the upper half, ties in the lower
  for (int p0 = 0; p0 < m; p0 += SPAN) {
    if (!RESIDENT) load(p0, m);
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      const uint32_t up = __ballot_sync(0xffffffffu, key[e] > base), tie = __ballot_sync(0xffffffffu, key[e] == base);
      if (lane == 0) { above_bits[e * (THREADS / 32) + warp] = up; tie_bits[e * (THREADS / 32) + warp] = tie; }
    }
    __syncthreads();
    const uint64_t mine = tid < WORDS ? (uint64_t)__popc(above_bits[tid]) << 32 | __popc(tie_bits[tid]) : 0;
    uint64_t total;
    const uint64_t incl = done + select_scan<THREADS>(mine, places[which], total);
    if (tid < WORDS) before[tid] = incl - mine;
    __syncthreads();
    which ^= 1;
    done += total;
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      const int w = e * (THREADS / 32) + warp;
      const uint32_t up = above_bits[w], tie = tie_bits[w];
      const int at = (int)(before[w] >> 32) + __popc(up & below), ties = (int)(uint32_t)before[w] + __popc(tie & below);
      if ((up >> lane & 1) || ((tie >> lane & 1) && ties < want)) out[at + min(ties, want)] = a.first + p0 + e * THREADS + tid;
    }
    if (!RESIDENT) __syncthreads();               // the words are written again
  }
}

// What a kernel's 32-bit counter runs up to, in steps of less than as much again.
constexpr int COUNTER_MAX = 1 << 30;

template <int KIND, int D, int NT>
static int launch_scores(const ScoreArgs& a, dim3 grid, cudaStream_t st) {
  static bool armed[64] = {};
  constexpr int smem = ScoreRing<D, KIND == HKB_KV_FP8_E4M3>::BYTES;
  if (arm(scores_kernel<KIND, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem, armed) != cudaSuccess) return HKB_ERR_CUDA;
  return launch((const void*)scores_kernel<KIND, D, NT>, grid, SCORE_WARPS * 32, 1, smem, &a, st);
}

static int advance_tables(int32_t* block_table, int64_t table_stride, int max_pages, int32_t* seq_lens,
                                  const int32_t* new_tokens, int num_reqs, int block_size, int32_t* free_pages,
                                  int64_t free_capacity, int32_t* free_count, int64_t* slot_mapping, int64_t* positions,
                                  int64_t num_rows, int32_t* q_start, int32_t* status, void* stream) {
  if (num_reqs < 0 || max_pages < 0 || free_capacity < 0 || num_rows < 0 ||
      free_capacity > 0x7fffffff || num_rows > 0x40000000 || num_reqs > 0x40000000) return HKB_ERR_SIZE;
  if (block_size <= 0) return HKB_ERR_BLOCK_SIZE;
  if (!free_count || !q_start) return HKB_ERR_NULL;
  if (num_reqs > 0 && (!seq_lens || !new_tokens || !status)) return HKB_ERR_NULL;
  if (num_reqs > 0 && max_pages > 0 && !block_table) return HKB_ERR_NULL;
  if (free_capacity > 0 && !free_pages) return HKB_ERR_NULL;
  if (num_rows > 0 && (!slot_mapping || !positions)) return HKB_ERR_NULL;
  if (num_reqs > 1 && table_stride < max_pages) return HKB_ERR_STRIDE;
  AdvanceArgs a;
  a.table = block_table; a.table_stride = table_stride; a.max_pages = max_pages;
  a.seq_lens = seq_lens; a.new_tokens = new_tokens; a.num_reqs = num_reqs; a.page = block_size;
  int l = 0;
  while (l < 31 && (1u << l) < (uint32_t)block_size) ++l;
  a.page_magic = l ? (uint32_t)((1ull << (31 + l)) / (uint32_t)block_size + 1) : 0;
  a.page_shift = l ? l - 1 : 0;
  a.free_pages = free_pages; a.free_count = free_count; a.free_cap = free_capacity;
  a.slots = slot_mapping; a.positions = positions; a.tokens = num_rows;
  a.q_start = q_start; a.status = status;
  if (num_rows > 4096 || num_reqs > 512) {
    auto kernel = advance_kernel<32, 2>;
    static bool armed[64] = {};
    if (arm(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1, armed) != cudaSuccess) return HKB_ERR_CUDA;
    return launch((const void*)kernel, dim3(16), 1024, 16, 0, &a, (cudaStream_t)stream);
  }
  return launch((const void*)advance_kernel<8, 2>, dim3(1), 256, 1, 0, &a, (cudaStream_t)stream);
}

static int page_bounds(void* bounds, int64_t bounds_stride_block, int64_t bounds_stride_head, int64_t bounds_blocks,
                               hkb_cache_t kc, const int32_t* block_table, int64_t table_stride, int max_pages,
                               const int32_t* seq_lens, const int32_t* q_start, int num_seqs, int64_t num_tokens,
                               int num_kv_heads, int head_dim, int block_size, int kv_dtype, void* stream) {
  if (num_seqs < 0 || num_kv_heads <= 0 || max_pages < 0 || kc.num_blocks < 0 || bounds_blocks < 0 || num_tokens < 0) return HKB_ERR_SIZE;
  if (num_seqs == 0 || max_pages == 0) return HKB_OK;
  if (!bounds || !kc.ptr || !block_table || !seq_lens) return HKB_ERR_NULL;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return HKB_ERR_HEAD_DIM;
  if (block_size <= 0 || block_size > COUNTER_MAX) return HKB_ERR_BLOCK_SIZE;
  if (kv_dtype != HKB_KV_BF16 && kv_dtype != HKB_KV_FP8_E4M3 && kv_dtype != HKB_KV_F16) return HKB_ERR_DTYPE;
  const int es = kv_dtype == HKB_KV_FP8_E4M3 ? 1 : 2;
  if ((kc.stride_block | kc.stride_token | kc.stride_head | bounds_stride_block | bounds_stride_head) * es % 16) return HKB_ERR_STRIDE;
  if (((uintptr_t)kc.ptr | (uintptr_t)bounds) % 16) return HKB_ERR_ALIGN;
  const int64_t items = q_start ? num_tokens / block_size + 2 * (int64_t)num_seqs : num_seqs;
  const bool share = block_size > 32;
  const int64_t per_cta = share ? 1 : BOUNDS_WARPS, ctas = (items * num_kv_heads + per_cta - 1) / per_cta;
  if (items > 0x3fffffff || ctas > 0x7fffffff) return HKB_ERR_SIZE;
  BoundsArgs a;
  a.bounds = (uint8_t*)bounds; a.b_stride_block = bounds_stride_block * es; a.b_stride_head = bounds_stride_head * es;
  a.k = (const uint8_t*)kc.ptr;
  a.k_stride_block = kc.stride_block * es; a.k_stride_token = kc.stride_token * es; a.k_stride_head = kc.stride_head * es;
  const int64_t nb = kc.num_blocks < bounds_blocks ? kc.num_blocks : bounds_blocks;
  a.num_blocks = nb > 0x7fffffff ? 0x7fffffff : (int)nb;
  a.table = block_table; a.table_stride = table_stride; a.max_pages = max_pages;
  a.seq_lens = seq_lens; a.q_start = q_start; a.tokens = num_tokens > 0x7fffffff ? 0x7fffffff : (int)num_tokens;
  a.num_seqs = num_seqs; a.num_kv_heads = num_kv_heads; a.page = block_size;
  a.items = (int)items;
  // Loads in flight live in L1: what reads much keeps the SM's memory for it (4 x 8192 new tokens 12.4 against 15.6 us,
  // 64 pages of 256 tokens 6.7 against 8.4), a decode step's small launch goes along with the step's other kernels.
  int sms = hkb_sm_count(-1);
  if (sms <= 0) sms = 148;
  a.many = items * num_kv_heads * (((int64_t)block_size + 15) / 16) > 64 * sms;        // of 16 tokens
  const int carveout = a.many || share ? 25 : STEP_CARVEOUT;
#define HKB_BOUNDS(KIND, CPR_) \
  if (kv_dtype == KIND && head_dim * es == CPR_ * 16) { \
    const void* kernel = share ? (const void*)bounds_kernel<KIND, CPR_, true> : (const void*)bounds_kernel<KIND, CPR_, false>; \
    return launch(kernel, dim3((unsigned)ctas), BOUNDS_WARPS * 32, 1, 0, &a, (cudaStream_t)stream, carveout); \
  }
  HKB_BOUNDS(HKB_KV_BF16, 8) HKB_BOUNDS(HKB_KV_BF16, 16) HKB_BOUNDS(HKB_KV_BF16, 32)
  HKB_BOUNDS(HKB_KV_F16, 8) HKB_BOUNDS(HKB_KV_F16, 16) HKB_BOUNDS(HKB_KV_F16, 32)
  HKB_BOUNDS(HKB_KV_FP8_E4M3, 4) HKB_BOUNDS(HKB_KV_FP8_E4M3, 8) HKB_BOUNDS(HKB_KV_FP8_E4M3, 16)
#undef HKB_BOUNDS
  return HKB_ERR_UNSUPPORTED;
}

static int page_scores(float* scores, int64_t scores_stride_row, int64_t scores_stride_head, int num_columns,
                               const void* q, int64_t q_stride_row, int64_t q_stride_head,
                               const void* bounds, int64_t bounds_stride_block, int64_t bounds_stride_head,
                               int64_t bounds_blocks, const int32_t* block_table, int64_t table_stride,
                               const int32_t* seq_lens, int num_rows, int num_q_heads, int num_kv_heads, int head_dim,
                               int block_size, float scale, int kv_dtype, const float* k_scale, void* stream) {
  if (num_rows < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_columns < 0 || num_columns > COUNTER_MAX ||
      num_rows > 65535 || num_kv_heads > 65535) return HKB_ERR_SIZE;
  if (num_rows == 0 || num_columns == 0) return HKB_OK;
  if (!scores || !q || !bounds || !block_table || !seq_lens) return HKB_ERR_NULL;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return HKB_ERR_HEAD_DIM;
  if (block_size <= 0) return HKB_ERR_BLOCK_SIZE;
  if (num_q_heads % num_kv_heads || num_q_heads / num_kv_heads > HKB_MAX_GROUP) return HKB_ERR_GROUP;
  if (kv_dtype != HKB_KV_BF16 && kv_dtype != HKB_KV_FP8_E4M3 && kv_dtype != HKB_KV_F16) return HKB_ERR_DTYPE;
  const bool fp8 = kv_dtype == HKB_KV_FP8_E4M3;
  if ((fp8 && !k_scale) || !positive_scale(scale)) return HKB_ERR_SCALE;
  const int es = fp8 ? 1 : 2;
  if ((bounds_stride_block | bounds_stride_head) * es % 16 || (q_stride_row | q_stride_head) % 8) return HKB_ERR_STRIDE;
  if (((uintptr_t)q | (uintptr_t)bounds) % 16 || (uintptr_t)scores % 4) return HKB_ERR_ALIGN;
  if (bounds_blocks < 1) return HKB_ERR_SIZE;
  ScoreArgs a;
  a.scores = scores; a.s_stride_row = scores_stride_row; a.s_stride_head = scores_stride_head; a.columns = num_columns;
  a.q = (const __nv_bfloat16*)q; a.q_stride_row = q_stride_row; a.q_stride_head = q_stride_head;
  a.bounds = (const uint8_t*)bounds; a.b_stride_block = bounds_stride_block * es; a.b_stride_head = bounds_stride_head * es;
  a.num_blocks = bounds_blocks > 0x7fffffff ? 0x7fffffff : (int)bounds_blocks;
  a.table = block_table; a.table_stride = table_stride; a.seq_lens = seq_lens;
  a.page = block_size; a.group = num_q_heads / num_kv_heads; a.scale = scale; a.k_scale = fp8 ? k_scale : nullptr;
  const int64_t tiles = ((int64_t)num_columns + 15) / 16;
  // about twice the warps that the machine holds at once (eight an SM, each a CTA of its own): equal shares of a table
  // are not equal shares of the work where sequences are shorter than it
  int sms = hkb_sm_count(-1);
  if (sms <= 0) sms = 148;
  const int64_t room = (int64_t)sms * 16, per = (tiles * num_rows * num_kv_heads + room - 1) / room;
  a.tiles_per_warp = (int)(per < tiles ? per : tiles);
  const int64_t warps = (tiles + a.tiles_per_warp - 1) / a.tiles_per_warp;
  const dim3 grid((unsigned)((warps + SCORE_WARPS - 1) / SCORE_WARPS), num_kv_heads, num_rows);
  cudaStream_t st = (cudaStream_t)stream;
  const int nt = a.group > 8 ? 2 : 1;
#define HKB_SCORES(KIND, D_) \
  if (kv_dtype == KIND && head_dim == D_) \
    return nt == 1 ? launch_scores<KIND, D_, 1>(a, grid, st) : launch_scores<KIND, D_, 2>(a, grid, st);
  HKB_SCORES(HKB_KV_BF16, 64) HKB_SCORES(HKB_KV_BF16, 128) HKB_SCORES(HKB_KV_BF16, 256)
  HKB_SCORES(HKB_KV_F16, 64) HKB_SCORES(HKB_KV_F16, 128) HKB_SCORES(HKB_KV_F16, 256)
  HKB_SCORES(HKB_KV_FP8_E4M3, 64) HKB_SCORES(HKB_KV_FP8_E4M3, 128) HKB_SCORES(HKB_KV_FP8_E4M3, 256)
#undef HKB_SCORES
  return HKB_ERR_UNSUPPORTED;
}

static int select_pages(int32_t* pages, int64_t pages_stride_row, int64_t pages_stride_head, int budget,
                                const float* scores, int64_t scores_stride_row, int64_t scores_stride_head, int num_columns,
                                const int32_t* seq_lens, int num_rows, int num_kv_heads, int block_size, int first, int last,
                                void* stream) {
  if (num_rows < 0 || num_kv_heads <= 0 || num_kv_heads > 65535 || num_columns < 0 || num_columns > COUNTER_MAX ||
      budget < 0 || budget > COUNTER_MAX || first < 0 || last < 0 || (int64_t)first + last > budget) return HKB_ERR_SIZE;
  if (num_rows == 0 || budget == 0) return HKB_OK;
  if (block_size <= 0) return HKB_ERR_BLOCK_SIZE;
  if (!pages || !seq_lens || (num_columns > 0 && !scores)) return HKB_ERR_NULL;
  if (((uintptr_t)pages | (uintptr_t)scores) % 4) return HKB_ERR_ALIGN;
  SelectArgs a;
  a.pages = pages; a.p_stride_row = pages_stride_row; a.p_stride_head = pages_stride_head; a.budget = budget;
  a.scores = scores; a.s_stride_row = scores_stride_row; a.s_stride_head = scores_stride_head; a.columns = num_columns;
  a.seq_lens = seq_lens; a.page = block_size; a.first = first; a.last = last;
  const int64_t items = (int64_t)num_rows * num_kv_heads;
  if (items > 0x7fffffff) return HKB_ERR_SIZE;
  a.num_kv_heads = num_kv_heads; a.items = (int)items;
  cudaStream_t st = (cudaStream_t)stream;
  int sms = hkb_sm_count(-1);
  if (sms <= 0) sms = 148;
  const dim3 grid(num_rows, num_kv_heads);
  // A warp's steps cost a comparison a key it holds, a CTA's its barriers. Measured, us, (rows x kv heads) of 1000 columns:
  // 8 of them a warp each 6.5, a CTA each 4.2; 64: 7.2, 4.3; 512: 7.5, 9.7 (256 threads); 4096: 18, 45. Of 500: 4.0, 4.3.
  if (num_columns <= 512 || (num_columns <= 1024 && items > 2 * sms)) {
    const void* kernel = num_columns <= 256 ? (const void*)select_warp_kernel<8>
                         : num_columns <= 512 ? (const void*)select_warp_kernel<16> : (const void*)select_warp_kernel<32>;
    return launch(kernel, dim3((unsigned)((items + SELECT_WARPS - 1) / SELECT_WARPS)), SELECT_WARPS * 32, 1, 0, &a, st);
  }
  // A pass costs a thread its keys and the CTA its barriers and its 2048 bins; us, 8 and 512 (rows x kv heads):
  // 2000 columns 4.7, 9.1 (256 threads of eight keys 6.0, 13.7); 4000: 5.2, 14.1 (of eight keys 6.0, 16.6); 8000: 6.9,
  // 19.5 (512 threads of sixteen 8.3, 20.2).
  if (num_columns <= 1024) return launch((const void*)select_kernel<512, 2, true>, grid, 512, 1, 0, &a, st);
  if (num_columns <= 2048) return launch((const void*)select_kernel<512, 4, true>, grid, 512, 1, 0, &a, st);
  if (num_columns <= 4096) return launch((const void*)select_kernel<1024, 4, true>, grid, 1024, 1, 0, &a, st);
  const void* kernel = num_columns <= 8192 ? (const void*)select_kernel<1024, 8, true>
                       : num_columns <= 16384 ? (const void*)select_kernel<1024, 16, true> : (const void*)select_kernel<1024, 16, false>;
  return launch(kernel, grid, 1024, 1, 0, &a, st);
}

}  // namespace hkb

extern "C" int hkb_advance_tables(const hkb_advance_t* p, void* stream) {
  if (!p) return HKB_ERR_NULL;
  if (!hkb::ints({p->max_pages, p->num_reqs, p->block_size})) return HKB_ERR_SIZE;
  return hkb::advance_tables(p->block_table, p->table_stride, (int)p->max_pages, p->seq_lens, p->new_tokens, (int)p->num_reqs,
                             (int)p->block_size, p->free_pages, p->free_capacity, p->free_count, p->slot_mapping,
                             p->positions, p->num_rows, p->q_start, p->status, stream);
}

extern "C" int hkb_page_bounds(const hkb_page_bounds_t* p, void* stream) {
  if (!p) return HKB_ERR_NULL;
  if (!hkb::ints({p->max_pages, p->num_seqs, p->num_kv_heads, p->head_dim, p->block_size, p->kv_dtype})) return HKB_ERR_SIZE;
  return hkb::page_bounds(p->bounds, p->bounds_stride_block, p->bounds_stride_head, p->bounds_blocks, p->k_cache,
                          p->block_table, p->table_stride, (int)p->max_pages, p->seq_lens, p->q_start, (int)p->num_seqs,
                          p->num_tokens, (int)p->num_kv_heads, (int)p->head_dim, (int)p->block_size, (int)p->kv_dtype, stream);
}

extern "C" int hkb_page_scores(const hkb_page_scores_t* p, void* stream) {
  if (!p) return HKB_ERR_NULL;
  if (!hkb::ints({p->num_columns, p->num_rows, p->num_q_heads, p->num_kv_heads, p->head_dim, p->block_size, p->kv_dtype})) return HKB_ERR_SIZE;
  return hkb::page_scores(p->scores, p->scores_stride_row, p->scores_stride_head, (int)p->num_columns, p->q, p->q_stride_row,
                          p->q_stride_head, p->bounds, p->bounds_stride_block, p->bounds_stride_head, p->bounds_blocks,
                          p->block_table, p->table_stride, p->seq_lens, (int)p->num_rows, (int)p->num_q_heads,
                          (int)p->num_kv_heads, (int)p->head_dim, (int)p->block_size, (float)p->scale, (int)p->kv_dtype,
                          p->k_scale, stream);
}

extern "C" int hkb_select_pages(const hkb_select_pages_t* p, void* stream) {
  if (!p) return HKB_ERR_NULL;
  if (!hkb::ints({p->budget, p->num_columns, p->num_rows, p->num_kv_heads, p->block_size, p->first, p->last})) return HKB_ERR_SIZE;
  return hkb::select_pages(p->pages, p->pages_stride_row, p->pages_stride_head, (int)p->budget, p->scores,
                           p->scores_stride_row, p->scores_stride_head, (int)p->num_columns, p->seq_lens, (int)p->num_rows,
                           (int)p->num_kv_heads, (int)p->block_size, (int)p->first, (int)p->last, stream);
}
