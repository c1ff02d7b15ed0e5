// Page bookkeeping under a decode over selected pages: block tables and slots from request lengths,
// a page's summary, the summaries' scores against a query, the budget's best pages.
#include "hkb_common.cuh"
#include "hkb_cluster.cuh"
#include "hkb_walk_mma.cuh"

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
// every CTA scans all requests (a trip to memory a CHUNK of them), then takes its share of the tokens and
// pages; the in-place updates -- the stack's top, the lengths, the count -- come after a cluster barrier, when
// every CTA has read what it needs of the old state. Deterministic: no atomics.
// Bound: latency (two dependent trips and the scans), then the stores of 16 bytes a token.
// ---------------------------------------------------------------------------------
constexpr int ADV_THREADS = 512;      // requests a chunk, one a thread
constexpr int ADV_WARPS = ADV_THREADS / 32;

struct AdvanceArgs {
  int* table;
  int64_t table_stride;
  int max_pages;
  int* seq_lens;
  const int* new_tokens;
  int num_reqs, page;
  int* free_pages;
  int* free_count;
  int64_t free_cap;
  int64_t* slots;
  int64_t* positions;
  int64_t tokens;      // rows of slots and positions
  int* q_start;
  int* status;
};

// Inclusive sum over the CTA's threads (in thread order); `sums` is one value a warp, reused call by call.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* sums, int64_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int x = 1; x < 32; x <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, v, x);
    if (lane >= x) v += y;
  }
  __syncthreads();                       // `sums` of the call before is read
  if (lane == 31) sums[warp] = v;
  __syncthreads();
  int64_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < ADV_WARPS; ++w) {
    const int64_t s = sums[w];
    if (w < warp) before += s;
    total += s;
  }
  return v + before;
}

// The first of n ascending inclusive sums that is greater than x: the thread whose range holds x.
__device__ __forceinline__ int range_of(const int64_t* ends, int n, int64_t x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (ends[mid] > x) hi = mid; else lo = mid + 1;
  }
  return lo;
}

__global__ void __launch_bounds__(ADV_THREADS) advance_kernel(const AdvanceArgs a) {
  __shared__ int64_t sums[ADV_WARPS];
  __shared__ int64_t s_ends[ADV_THREADS], s_upto[ADV_THREADS];
  __shared__ int s_old[ADV_THREADS], s_have[ADV_THREADS], s_ok[ADV_THREADS], s_need[ADV_THREADS];
  const int tid = threadIdx.x;
  const int ctas = cluster_size(), rank = cluster_rank();
  const int64_t count = min((int64_t)max(*a.free_count, 0), a.free_cap);
  const int P = a.page;

  int64_t tok0 = 0, upto0 = 0, taken = 0, given = 0;      // sums over the chunks before
  for (int c0 = 0; c0 < a.num_reqs; c0 += ADV_THREADS) {
    const int n = min(ADV_THREADS, a.num_reqs - c0), r = c0 + tid;
    int64_t old = 0, grow = 0;
    if (tid < n) { old = max(a.seq_lens[r], 0); grow = a.new_tokens[r]; }
    const int64_t after = max(old + grow, (int64_t)0);
    const int64_t have = min((old + P - 1) / P, (int64_t)a.max_pages), want = (after + P - 1) / P;
    const int64_t q = max(grow, (int64_t)0);
    int64_t tok_total, need_total, give_total;
    const int64_t ends = tok0 + block_scan(q, sums, tok_total);
    int st = HKB_REQ_OK;
    if (q > 0) {
      if (want > a.max_pages || after > 0x7fffffffLL) st = HKB_REQ_TABLE_FULL;
      else if (ends > a.tokens) st = HKB_REQ_NO_ROWS;
    }
    const int64_t need = st == HKB_REQ_OK && q > 0 ? max(want - have, (int64_t)0) : 0;
    const int64_t upto = upto0 + block_scan(need, sums, need_total);
    if (need > 0 && upto > count) st = HKB_REQ_NO_PAGES;
    block_scan(grow < 0 ? max(have - want, (int64_t)0) : 0, sums, give_total);
    s_ends[tid] = ends; s_upto[tid] = upto;
    s_old[tid] = (int)old; s_have[tid] = (int)have; s_ok[tid] = st == HKB_REQ_OK; s_need[tid] = (int)need;
    if (tid < n && (c0 / ADV_THREADS) % ctas == rank) {
      a.q_start[r + 1] = (int)min(ends, (int64_t)0x7fffffff);
      if (r == 0) a.q_start[0] = 0;
      a.status[r] = st;
    }
    __syncthreads();

    // this chunk's tokens, shared out over the cluster
    const int64_t t1 = min(tok0 + tok_total, a.tokens);
    for (int64_t t = tok0 + rank * ADV_THREADS + tid; t < t1; t += ctas * ADV_THREADS) {
      const int i = range_of(s_ends, n, t);
      const int64_t start = i ? s_ends[i - 1] : tok0;
      const int64_t pos = s_old[i] + (t - start);
      const int64_t lp = pos / P;
      int64_t block = -1;
      if (s_ok[i]) {
        if (lp < s_have[i]) block = a.table[(int64_t)(c0 + i) * a.table_stride + lp];
        else block = a.free_pages[count - 1 - (s_upto[i] - s_need[i] + lp - s_have[i])];
      }
      a.slots[t] = block >= 0 ? block * P + (pos - lp * P) : -1;
      a.positions[t] = pos;
    }
    // and its new pages. Once one request gets none, none of those after it that need pages gets any (the sum
    // runs on), so the pages handed out are the sum's first ones, in request order.
    const int64_t p1 = min(upto0 + need_total, count);
    for (int64_t x = upto0 + rank * ADV_THREADS + tid; x < p1; x += ctas * ADV_THREADS) {
      const int i = range_of(s_upto, n, x);
      if (!s_ok[i]) continue;
      const int64_t at = s_have[i] + x - (s_upto[i] - s_need[i]);
      a.table[(int64_t)(c0 + i) * a.table_stride + at] = a.free_pages[count - 1 - x];
    }
    int64_t got;
    block_scan(s_ok[tid] ? need : 0, sums, got);
    taken += got;
    tok0 += tok_total; upto0 += need_total; given += give_total;
    __syncthreads();
  }
  for (int64_t t = min(tok0, a.tokens) + rank * ADV_THREADS + tid; t < a.tokens; t += ctas * ADV_THREADS) {
    a.slots[t] = -1;
    a.positions[t] = 0;
  }
  if (a.num_reqs == 0 && rank == 0 && tid == 0) a.q_start[0] = 0;
  cluster_sync();

  if (given > 0) {       // the same in every CTA
    int64_t at0 = count - taken;
    for (int c0 = 0; c0 < a.num_reqs; c0 += ADV_THREADS) {
      const int n = min(ADV_THREADS, a.num_reqs - c0), r = c0 + tid;
      int64_t old = 0, grow = 0;
      if (tid < n) { old = max(a.seq_lens[r], 0); grow = a.new_tokens[r]; }
      const int64_t have = min((old + P - 1) / P, (int64_t)a.max_pages);
      const int64_t want = (max(old + grow, (int64_t)0) + P - 1) / P;
      const int64_t give = grow < 0 ? max(have - want, (int64_t)0) : 0;
      int64_t total;
      s_upto[tid] = block_scan(give, sums, total);
      s_have[tid] = (int)want; s_need[tid] = (int)give;
      __syncthreads();
      for (int64_t x = rank * ADV_THREADS + tid; x < total; x += ctas * ADV_THREADS) {
        const int i = range_of(s_upto, n, x);
        if (at0 + x < a.free_cap)
          a.free_pages[at0 + x] = a.table[(int64_t)(c0 + i) * a.table_stride + s_have[i] + x - (s_upto[i] - s_need[i])];
      }
      at0 += total;
      __syncthreads();
    }
    cluster_sync();
  }
  for (int c = rank; c * ADV_THREADS < a.num_reqs; c += ctas) {
    const int r = c * ADV_THREADS + tid;
    if (r < a.num_reqs) {
      const int64_t old = max(a.seq_lens[r], 0);
      // status[r] was written by this thread
      a.seq_lens[r] = a.status[r] == HKB_REQ_OK ? (int)max(old + a.new_tokens[r], (int64_t)0) : (int)old;
    }
  }
  if (rank == 0 && tid == 0) *a.free_count = (int)min(count - taken + given, a.free_cap);
}

// ---------------------------------------------------------------------------------
// A page's summary: the least and the greatest key of every channel, over the page's tokens below the
// sequence's length. Values of the cache's own type, so nothing is rounded. A warp takes a (page, kv head): its
// lanes hold 16-byte chunks of a row, 32 / chunks rows at a time, and fold them with packed minima and maxima
// that keep a NaN. Bound: bytes (the keys once, two rows a page out).
// ---------------------------------------------------------------------------------
constexpr int BOUNDS_WARPS = 8;

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
  int num_seqs, num_kv_heads, page;
  int items;                       // (sequence, page) pairs the grid covers
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

// KIND: HKB_KV_*; CPR: 16-byte chunks a row (head_dim x element size / 16)
template <int KIND, int CPR>
__global__ void __launch_bounds__(BOUNDS_WARPS * 32) bounds_kernel(const BoundsArgs a) {
  constexpr bool FP8 = KIND == HKB_KV_FP8_E4M3;
  using Pr = Pair<FP8 ? HKB_KV_F16 : KIND>;       // e4m3 widens to f16 exactly
  constexpr int REGS = FP8 ? 8 : 4;               // pairs a 16-byte chunk holds
  constexpr int RPI = 32 / CPR, UNROLL = 8;
  const int lane = threadIdx.x & 31;
  const int64_t unit = (int64_t)blockIdx.x * BOUNDS_WARPS + (threadIdx.x >> 5);
  const int item = (int)(unit / a.num_kv_heads), head = (int)(unit % a.num_kv_heads);
  if (item >= a.items) return;

  // which page of which sequence. With query starts, sequence r has the items from start[r] / page + 2 r on:
  // its q new tokens touch at most q / page + 2 pages, and so many items it has.
  int r = item, page;
  int len;
  if (a.q_start) {
    int lo = 0, hi = a.num_seqs;                  // the last r whose items begin at or before this one is in [lo, hi)
    while (hi - lo > 1) {                         // 32 candidates at once
      const int step = (hi - lo + 31) / 32, at = lo + lane * step;
      const bool below = at < hi && __ldg(a.q_start + at) / a.page + 2 * at <= item;
      const int m = max(__popc(__ballot_sync(0xffffffffu, below)), 1);
      lo += (m - 1) * step;
      hi = min(hi, lo + step);
    }
    r = lo;
    const int s0 = __ldg(a.q_start + r), q = __ldg(a.q_start + r + 1) - s0;
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
  for (int t0 = 0; t0 < live; t0 += RPI * UNROLL) {
    uint4 v[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {            // a row past the last live one: the last one again
      const int t = min(t0 + u * RPI + lane / CPR, live - 1);
      v[u] = __ldg(reinterpret_cast<const uint4*>(src + (int64_t)t * a.k_stride_token));
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
  }
#pragma unroll
  for (int x = CPR; x < 32; x <<= 1)
#pragma unroll
    for (int i = 0; i < REGS; ++i) {
      low[i] = Pr::least(low[i], __shfl_xor_sync(0xffffffffu, low[i], x));
      high[i] = Pr::most(high[i], __shfl_xor_sync(0xffffffffu, high[i], x));
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
// so lane t of a quad takes eight (fp8: sixteen) consecutive ones and the query's fragments are dealt alike.
// Bound: bytes (a summary is 2 rows a page where the attention reads 2 rows a token).
// ---------------------------------------------------------------------------------
constexpr int SCORE_WARPS = 4;

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

template <int KIND, int D, int NT>
__global__ void __launch_bounds__(SCORE_WARPS * 32) scores_kernel(const ScoreArgs a) {
  constexpr bool FP8 = KIND == HKB_KV_FP8_E4M3, F16 = KIND != HKB_KV_BF16;   // e4m3 widens to f16 exactly
  using Pr = Pair<F16 ? HKB_KV_F16 : HKB_KV_BF16>;
  constexpr int EPC = FP8 ? 16 : 8;            // elements of a lane's 16-byte chunk
  constexpr int STEPS = D / (4 * EPC);         // chunks a lane reads of one row of D values
  constexpr int MPC = EPC / 4;                 // mma a chunk feeds
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int head = blockIdx.y, row = blockIdx.z;
  const int first = (blockIdx.x * SCORE_WARPS + (threadIdx.x >> 5)) * a.tiles_per_warp * 16;
  const int last = min(first + a.tiles_per_warp * 16, a.columns);
  if (first >= last) return;
  const int len = max(__ldg(a.seq_lens + row), 0);
  const int pages = (int)min(((int64_t)len + a.page - 1) / a.page, (int64_t)a.columns);
  float* out = a.scores + (int64_t)row * a.s_stride_row + (int64_t)head * a.s_stride_head;
  for (int p = max(first, pages) + lane; p < last; p += 32) out[p] = -INFINITY;
  const int end = min(last, pages);
  if (first >= end) return;

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
      // bf16 -> f16: the head's values are brought below 2^14 by a power of two (exact), so that none overflows
      // and what falls under f16's range is 2^-38 of the largest
      float top = 0.f;
#pragma unroll
      for (int s = 0; s < STEPS; ++s)
#pragma unroll
        for (int i = 0; i < EPC / 2; ++i)
          top = fmaxf(top, fmaxf(fabsf(bf16lo(qf[nt][s][i])), fabsf(bf16hi(qf[nt][s][i]))));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int e = min(max((int)(__float_as_uint(top) >> 23), 14), 253);   // biased exponent; inf and zero keep a finite factor
      const float down = __uint_as_float((uint32_t)(267 - e) << 23);         // 2^(13 - (e - 127)), at most 2^126
      unit[nt] = __uint_as_float((uint32_t)(e - 13) << 23);
#pragma unroll
      for (int s = 0; s < STEPS; ++s)
#pragma unroll
        for (int i = 0; i < EPC / 2; ++i)
          qf[nt][s][i] = pack_f16x2(bf16lo(qf[nt][s][i]) * down, bf16hi(qf[nt][s][i]) * down);
    }
  }
  const float factor = a.scale * (a.k_scale ? __ldg(a.k_scale) : 1.f);
  const int* table = a.table + (int64_t)row * a.table_stride;
  const uint8_t* base = a.bounds + (int64_t)head * a.b_stride_head + t * 16;

  for (int p0 = first; p0 < end; p0 += 16) {
    const uint8_t* src[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {              // a page past the last one: the last one again
      const int id = __ldg(table + min(p0 + g + 8 * j, end - 1));
      src[j] = base + (int64_t)min(max(id, 0), a.num_blocks - 1) * a.b_stride_block;
    }
    float sc[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) sc[nt][i] = 0.f;
#pragma unroll
    for (int half = 0; half < 2; ++half) {     // low bounds meet the query's negative parts, high bounds the positive
      uint4 v[STEPS][2];
#pragma unroll
      for (int s = 0; s < STEPS; ++s)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          v[s][j] = __ldg(reinterpret_cast<const uint4*>(src[j] + half * (D * (FP8 ? 1 : 2)) + s * 64));
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        const uint32_t x[2][4] = {{v[s][0].x, v[s][0].y, v[s][0].z, v[s][0].w}, {v[s][1].x, v[s][1].y, v[s][1].z, v[s][1].w}};
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
            mma16<F16>(sc[nt], f, b);
          }
        }
      }
    }
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
    if (t < 2 && p < end) out[p] = (t ? best[1] : best[0]) * factor;
  }
}

// ---------------------------------------------------------------------------------
// The budget's best pages of a (row, kv head): the first `first` and the last `last` pages always, then by score
// downwards, ties to the lowest page; written in ascending order, -1 behind. A score becomes a 32-bit key whose
// order is the scores' (NaN above everything but the pages that are always kept: a broken key shows in the
// answer instead of being left out); the budget-th greatest key is found digit by digit, eight bits a pass over
// histograms in shared memory, and one more pass writes the pages that lie above it and as many of those on it
// as there is room for. Integers throughout, so the answer depends on no order of anything.
// ---------------------------------------------------------------------------------
constexpr int SELECT_THREADS = 256;

struct SelectArgs {
  int* pages;
  int64_t p_stride_row, p_stride_head;
  int budget;
  const float* scores;
  int64_t s_stride_row, s_stride_head;
  int columns;
  const int* seq_lens;
  int page, first, last;
};

__device__ __forceinline__ uint32_t score_key(float x) {
  x += 0.f;                                      // -0 and 0 are one score
  const uint32_t b = __float_as_uint(x);
  if (x != x) return 0xfffffffeu;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__global__ void __launch_bounds__(SELECT_THREADS) select_kernel(const SelectArgs a) {
  __shared__ int hist[256];
  __shared__ int warp_sum[SELECT_THREADS / 32][2];
  __shared__ int s_digit, s_above;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int head = blockIdx.y, row = blockIdx.x;
  const int len = max(__ldg(a.seq_lens + row), 0);
  const int n = (int)min(((int64_t)len + a.page - 1) / a.page, (int64_t)a.columns);
  int* out = a.pages + (int64_t)row * a.p_stride_row + (int64_t)head * a.p_stride_head;
  const float* in = a.scores + (int64_t)row * a.s_stride_row + (int64_t)head * a.s_stride_head;
  if (n <= a.budget) {
    for (int i = tid; i < a.budget; i += SELECT_THREADS) out[i] = i < n ? i : -1;
    return;
  }
  auto key = [&](int p) -> uint32_t {
    return p < a.first || p >= n - a.last ? 0xffffffffu : score_key(__ldg(in + p));
  };
  uint32_t prefix = 0;      // the digits found so far
  int want = a.budget;      // how many of the keys that begin with them are to be taken
  for (int shift = 24; shift >= 0; shift -= 8) {
    hist[tid] = 0;
    __syncthreads();
    for (int p = tid; p < n; p += SELECT_THREADS) {
      const uint32_t k = key(p);
      if (shift == 24 || (k >> (shift + 8)) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1);
    }
    __syncthreads();
    // the digit whose keys, with all greater ones, first reach `want`: a scan from the top
    const int mine = hist[255 - tid];
    int incl = mine;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, x);
      if (lane >= x) incl += y;
    }
    if (lane == 31) warp_sum[warp][0] = incl;
    __syncthreads();
    for (int w = 0; w < warp; ++w) incl += warp_sum[w][0];
    if (incl >= want && incl - mine < want) { s_digit = 255 - tid; s_above = incl - mine; }
    __syncthreads();
    prefix = prefix << 8 | (uint32_t)s_digit;
    want -= s_above;
    __syncthreads();
  }
  int taken = 0, ties = 0;  // so far, over the whole CTA
  for (int p0 = 0; p0 < n; p0 += SELECT_THREADS) {
    const int p = p0 + tid;
    const uint32_t k = p < n ? key(p) : 0u;
    const bool tie = p < n && k == prefix, above = p < n && k > prefix;
    const unsigned mt = __ballot_sync(0xffffffffu, tie), ma = __ballot_sync(0xffffffffu, above);
    if (lane == 0) { warp_sum[warp][0] = __popc(ma); warp_sum[warp][1] = __popc(mt); }
    __syncthreads();
    const unsigned below = (1u << lane) - 1;
    int at = taken + __popc(ma & below), tie_at = ties + __popc(mt & below);
#pragma unroll
    for (int w = 0; w < SELECT_THREADS / 32; ++w) {
      if (w < warp) { at += warp_sum[w][0]; tie_at += warp_sum[w][1]; }
      taken += warp_sum[w][0]; ties += warp_sum[w][1];
    }
    if (above || (tie && tie_at < want)) out[at + min(tie_at, want)] = p;
    __syncthreads();
  }
}

template <class F>
static int launched(F&& launch) {
  launch();
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) { hkb_tls_cuda_error = (int)e; return HKB_ERR_CUDA; }
  return HKB_OK;
}

}  // namespace hkb

extern "C" int hkb_advance_tables(int32_t* block_table, int64_t table_stride, int max_pages, int32_t* seq_lens,
                                  const int32_t* new_tokens, int num_reqs, int block_size, int32_t* free_pages,
                                  int64_t free_capacity, int32_t* free_count, int64_t* slot_mapping, int64_t* positions,
                                  int64_t num_rows, int32_t* q_start, int32_t* status, void* stream) {
  using namespace hkb;
  if (num_reqs < 0 || max_pages < 0 || free_capacity < 0 || num_rows < 0 || free_capacity > 0x7fffffff) return HKB_ERR_SIZE;
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
  a.free_pages = free_pages; a.free_count = free_count; a.free_cap = free_capacity;
  a.slots = slot_mapping; a.positions = positions; a.tokens = num_rows;
  a.q_start = q_start; a.status = status;
  const int ctas = num_rows > 4096 ? 8 : 1;
  return launch_cluster((const void*)advance_kernel, dim3(ctas), ADV_THREADS, ctas, 0, &a, (cudaStream_t)stream);
}

extern "C" int hkb_page_bounds(void* bounds, int64_t bounds_stride_block, int64_t bounds_stride_head, int64_t bounds_blocks,
                               hkb_cache_t kc, const int32_t* block_table, int64_t table_stride, int max_pages,
                               const int32_t* seq_lens, const int32_t* q_start, int num_seqs, int64_t num_tokens,
                               int num_kv_heads, int head_dim, int block_size, int kv_dtype, void* stream) {
  using namespace hkb;
  if (num_seqs < 0 || num_kv_heads <= 0 || max_pages < 0 || kc.num_blocks < 0 || bounds_blocks < 0 || num_tokens < 0) return HKB_ERR_SIZE;
  if (num_seqs == 0 || max_pages == 0 || (q_start && num_tokens == 0)) return HKB_OK;
  if (!bounds || !kc.ptr || !block_table || !seq_lens) return HKB_ERR_NULL;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return HKB_ERR_HEAD_DIM;
  if (block_size <= 0) return HKB_ERR_BLOCK_SIZE;
  if (kv_dtype != HKB_KV_BF16 && kv_dtype != HKB_KV_FP8_E4M3 && kv_dtype != HKB_KV_F16) return HKB_ERR_DTYPE;
  const int es = kv_dtype == HKB_KV_FP8_E4M3 ? 1 : 2;
  if ((kc.stride_block | kc.stride_token | kc.stride_head | bounds_stride_block | bounds_stride_head) * es % 16) return HKB_ERR_STRIDE;
  if (((uintptr_t)kc.ptr | (uintptr_t)bounds) % 16) return HKB_ERR_ALIGN;
  const int64_t items = q_start ? num_tokens / block_size + 2 * (int64_t)num_seqs : num_seqs;
  const int64_t ctas = (items * num_kv_heads + BOUNDS_WARPS - 1) / BOUNDS_WARPS;
  if (items > 0x3fffffff || ctas > 0x7fffffff) return HKB_ERR_SIZE;
  BoundsArgs a;
  a.bounds = (uint8_t*)bounds; a.b_stride_block = bounds_stride_block * es; a.b_stride_head = bounds_stride_head * es;
  a.k = (const uint8_t*)kc.ptr;
  a.k_stride_block = kc.stride_block * es; a.k_stride_token = kc.stride_token * es; a.k_stride_head = kc.stride_head * es;
  const int64_t nb = kc.num_blocks < bounds_blocks ? kc.num_blocks : bounds_blocks;
  a.num_blocks = nb > 0x7fffffff ? 0x7fffffff : (int)nb;
  a.table = block_table; a.table_stride = table_stride; a.max_pages = max_pages;
  a.seq_lens = seq_lens; a.q_start = q_start; a.num_seqs = num_seqs; a.num_kv_heads = num_kv_heads; a.page = block_size;
  a.items = (int)items;
  cudaStream_t st = (cudaStream_t)stream;
  return launched([&] {
#define HKB_BOUNDS(KIND, CPR_) \
  if (kv_dtype == KIND && head_dim * es == CPR_ * 16) bounds_kernel<KIND, CPR_><<<(unsigned)ctas, BOUNDS_WARPS * 32, 0, st>>>(a);
    HKB_BOUNDS(HKB_KV_BF16, 8) HKB_BOUNDS(HKB_KV_BF16, 16) HKB_BOUNDS(HKB_KV_BF16, 32)
    HKB_BOUNDS(HKB_KV_F16, 8) HKB_BOUNDS(HKB_KV_F16, 16) HKB_BOUNDS(HKB_KV_F16, 32)
    HKB_BOUNDS(HKB_KV_FP8_E4M3, 4) HKB_BOUNDS(HKB_KV_FP8_E4M3, 8) HKB_BOUNDS(HKB_KV_FP8_E4M3, 16)
#undef HKB_BOUNDS
  });
}

extern "C" int hkb_page_scores(float* scores, int64_t scores_stride_row, int64_t scores_stride_head, int num_columns,
                               const void* q, int64_t q_stride_row, int64_t q_stride_head,
                               const void* bounds, int64_t bounds_stride_block, int64_t bounds_stride_head,
                               int64_t bounds_blocks, const int32_t* block_table, int64_t table_stride,
                               const int32_t* seq_lens, int num_rows, int num_q_heads, int num_kv_heads, int head_dim,
                               int block_size, float scale, int kv_dtype, const float* k_scale, void* stream) {
  using namespace hkb;
  if (num_rows < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_columns < 0 || num_rows > 65535 || num_kv_heads > 65535) return HKB_ERR_SIZE;
  if (num_rows == 0 || num_columns == 0) return HKB_OK;
  if (!scores || !q || !bounds || !block_table || !seq_lens) return HKB_ERR_NULL;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return HKB_ERR_HEAD_DIM;
  if (block_size <= 0) return HKB_ERR_BLOCK_SIZE;
  if (num_q_heads % num_kv_heads || num_q_heads / num_kv_heads > HKB_MAX_GROUP) return HKB_ERR_GROUP;
  if (kv_dtype != HKB_KV_BF16 && kv_dtype != HKB_KV_FP8_E4M3 && kv_dtype != HKB_KV_F16) return HKB_ERR_DTYPE;
  const bool fp8 = kv_dtype == HKB_KV_FP8_E4M3;
  if (fp8 && !k_scale) return HKB_ERR_SCALE;
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
  a.tiles_per_warp = 2;
  const int64_t tiles = ((int64_t)num_columns + 15) / 16;
  const int64_t warps = (tiles + a.tiles_per_warp - 1) / a.tiles_per_warp;
  const dim3 grid((unsigned)((warps + SCORE_WARPS - 1) / SCORE_WARPS), num_kv_heads, num_rows);
  cudaStream_t st = (cudaStream_t)stream;
  const int nt = a.group > 8 ? 2 : 1;
  return launched([&] {
#define HKB_SCORES(KIND, D_) \
  if (kv_dtype == KIND && head_dim == D_) { \
    if (nt == 1) scores_kernel<KIND, D_, 1><<<grid, SCORE_WARPS * 32, 0, st>>>(a); \
    else scores_kernel<KIND, D_, 2><<<grid, SCORE_WARPS * 32, 0, st>>>(a); \
  }
    HKB_SCORES(HKB_KV_BF16, 64) HKB_SCORES(HKB_KV_BF16, 128) HKB_SCORES(HKB_KV_BF16, 256)
    HKB_SCORES(HKB_KV_F16, 64) HKB_SCORES(HKB_KV_F16, 128) HKB_SCORES(HKB_KV_F16, 256)
    HKB_SCORES(HKB_KV_FP8_E4M3, 64) HKB_SCORES(HKB_KV_FP8_E4M3, 128) HKB_SCORES(HKB_KV_FP8_E4M3, 256)
#undef HKB_SCORES
  });
}

extern "C" int hkb_select_pages(int32_t* pages, int64_t pages_stride_row, int64_t pages_stride_head, int budget,
                                const float* scores, int64_t scores_stride_row, int64_t scores_stride_head, int num_columns,
                                const int32_t* seq_lens, int num_rows, int num_kv_heads, int block_size, int first, int last,
                                void* stream) {
  using namespace hkb;
  if (num_rows < 0 || num_kv_heads <= 0 || num_kv_heads > 65535 || num_columns < 0 || budget < 0 || first < 0 || last < 0 ||
      (int64_t)first + last > budget) return HKB_ERR_SIZE;
  if (num_rows == 0 || budget == 0) return HKB_OK;
  if (block_size <= 0) return HKB_ERR_BLOCK_SIZE;
  if (!pages || !seq_lens || (num_columns > 0 && !scores)) return HKB_ERR_NULL;
  if (((uintptr_t)pages | (uintptr_t)scores) % 4) return HKB_ERR_ALIGN;
  SelectArgs a;
  a.pages = pages; a.p_stride_row = pages_stride_row; a.p_stride_head = pages_stride_head; a.budget = budget;
  a.scores = scores; a.s_stride_row = scores_stride_row; a.s_stride_head = scores_stride_head; a.columns = num_columns;
  a.seq_lens = seq_lens; a.page = block_size; a.first = first; a.last = last;
  return launched([&] { select_kernel<<<dim3(num_rows, num_kv_heads), SELECT_THREADS, 0, (cudaStream_t)stream>>>(a); });
}
