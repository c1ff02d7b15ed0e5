// Decode attention of one new token over selected pages.
//
// For a row and a kv head the caller lists pages of the row's sequence (hkb_select_pages); the group's query heads
// attend to the tokens of those pages that lie below the sequence's length:
//   out = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale k_scale q.k_t - max),  lse = max + log sum_t p_t.
//
// Bound: bytes (the selected K and V rows once, 4 to 16 flop a byte). A cluster of `splits` CTAs takes a (row, kv
// head); the 16-token tiles of its pages are dealt to all the cluster's warps in turn, each warp a cp.async ring and
// an online softmax of its own (SparseWorker). The warps' normalised partials stay
// in shared memory, and after one cluster barrier every CTA folds its slice of the outputs out of its peers' memory:
// one launch, no scratch, nothing shared between calls.
#include "hkb_cluster.cuh"
#include "hkb_sparse.cuh"

namespace hkb {

struct SparseArgs {
  DecodeArgs d;                  // q, caches, table, lengths, scales; the split scratch is not used
  const int* pages;              // (row, kv head): `budget` pages of the sequence, a negative entry is none
  int64_t p_stride_row, p_stride_head;
  int budget;
  float* out_lse;                // (rows, q heads) or null
};

// CTAs an SM the registers are dealt out for. The rings decide how many fit where a row is 256 bytes or more; with fp8
// rows of 128 the compiler, told nothing or told one, gave the kernel registers that cost it a CTA or its schedule
// (128 x 8 items of 128 pages 91.8 and 115 us, told seven 91.0; 2 x 8 of 512, four warps a CTA, 17.8 told nothing, 15.8
// told one).
template <class P, int WARPS>
constexpr int sparse_ctas() {
  return P::FP8 && WARPS == 2 ? (P::HEAD_DIM == 256 ? 4 : P::HEADS == 8 ? 7 : 5) : 1;
}

template <class P, int WARPS, bool F16>
__global__ void __launch_bounds__(WARPS * 32, sparse_ctas<P, WARPS>()) sparse_kernel(const SparseArgs a) {
  extern __shared__ __align__(128) uint8_t hkb_smem[];
  constexpr int D = P::HEAD_DIM, HEADS = P::HEADS, NST = P::STAGES;
  static_assert(NST >= 2, "a stage is computed on while the next is fetched");
  static_assert(HEADS * (D + 1) * 4 <= P::RING_SMEM, "a warp's partial lies where its ring was");
  after_the_last();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ctas = cluster_size(), rank = cluster_rank();
  const int kvh = blockIdx.y, row = blockIdx.z;
  const int nh = a.d.group, hq0 = kvh * nh;
  const int seq_len = max(__ldg(a.d.seq_lens + row), 0);

  float qs = a.d.scale * LOG2E, vs = 1.f;
  if (a.d.k_scale) qs *= __ldg(a.d.k_scale);
  if (a.d.v_scale) vs = __ldg(a.d.v_scale);

  typename P::Loader ld;
  ld.kbase = a.d.k + (int64_t)kvh * a.d.k_stride_head;
  ld.vbase = a.d.v + (int64_t)kvh * a.d.v_stride_head;
  ld.ksb = a.d.k_stride_block; ld.kst = a.d.k_stride_token;
  ld.vsb = a.d.v_stride_block; ld.vst = a.d.v_stride_token;
  ld.tiles_per_page = a.d.tiles_per_page; ld.num_blocks = a.d.num_blocks;
  ld.prepare(lane);

  // The warp's tiles: every `workers`-th of the list's budget x tiles_per_page, 32 looked up at a time, a batch ahead.
  const int* list = a.pages + (int64_t)row * a.p_stride_row + (int64_t)kvh * a.p_stride_head;
  const int* table = a.d.block_table + (int64_t)row * a.d.table_stride;
  const int workers = ctas * WARPS, tpp = a.d.tiles_per_page, total = a.budget * tpp;
  auto look_up = [&](int i0, int& id, int& tok) {     // lane l: item i0 + l; tok < 0: no tile
    id = 0; tok = -1;
    const int64_t x = (int64_t)(i0 + lane) * workers + rank * WARPS + warp;
    if (x >= total) return;
    const int e = (int)x / tpp, sub = (int)x - e * tpp;
    const int p = __ldg(list + e);
    if (p < 0 || p >= a.d.max_pages) return;
    id = __ldg(table + p);                            // asked for beside the length, not behind it
    const int64_t t0 = (int64_t)p * a.d.block_size + sub * TILE_TOKENS;
    if (t0 < seq_len) tok = (int)t0;
  };
  int next_item = 64, id, tok, id_n, tok_n;
  look_up(0, id, tok);
  look_up(32, id_n, tok_n);
  unsigned live = __ballot_sync(0xffffffffu, tok >= 0);
  const uint32_t ring = smem_u32(hkb_smem) + warp * P::RING_SMEM;
  // Requests the warp's next tile into a ring stage; its first token, or -1 where none is left.
  auto issue = [&](int stage) -> int {
    int t = -1;
    while (!live && (int64_t)(next_item - 32) * workers < total) {
      id = id_n; tok = tok_n;
      live = __ballot_sync(0xffffffffu, tok >= 0);
      look_up(next_item, id_n, tok_n);
      next_item += 32;
    }
    if (live) {
      const int src = __ffs(live) - 1;
      live &= live - 1;
      t = __shfl_sync(0xffffffffu, tok, src);
      ld.issue(ring + stage * P::STAGE_BYTES, t / TILE_TOKENS, __shfl_sync(0xffffffffu, id, src), lane);
    }
    cp_async_commit();
    return t;
  };
  int queue[NST - 1];            // first tokens of the tiles in flight, oldest first
#pragma unroll
  for (int k = 0; k < NST - 1; ++k) queue[k] = issue(k);

  typename P::State st;
  P::begin(st, a.d, row, hq0, nh, lane, qs);
  int sc = 0, sl = NST - 1;
  while (queue[0] >= 0) {
    cp_async_wait<NST - 2>();
    __syncwarp();
    const int t = issue(sl);     // over the tile before
    P::step(st, ring + sc * P::STAGE_BYTES, queue[0], seq_len, queue[0] > seq_len - TILE_TOKENS, lane);
#pragma unroll
    for (int k = 0; k + 1 < NST - 1; ++k) queue[k] = queue[k + 1];
    queue[NST - 2] = t;
    sc = sc + 1 == NST ? 0 : sc + 1;
    sl = sl + 1 == NST ? 0 : sl + 1;
  }
  // Behind the stream, not in front: the next launch's CTAs, waiting in the places that this one's last ones would have
  // been spread over, cost it more than their head start is worth (fp8, 128 x 8 items of 128 pages: 97 against 85 us).
  let_the_next();
  cp_async_wait<0>();
  __syncwarp();

  // The warp's partial over its ring: [head][D] normalised, then [head] lse.
  float* part = reinterpret_cast<float*>(hkb_smem + warp * P::RING_SMEM);
  P::Walk::end(st, lane, nh, vs, part, part + HEADS * D);
  // a NaN among the scores makes the sum NaN: the partial says so instead of counting as empty
#pragma unroll
  for (int nt = 0; nt < HEADS / 8; ++nt)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const unsigned bad = __ballot_sync(0xffffffffu, st.l[nt][c] != st.l[nt][c]);
      const int h = nt * 8 + 2 * (lane & 3) + c;
      if ((lane >> 2) == 0 && h < nh && (bad & (0x11111111u << (lane & 3)))) part[HEADS * D + h] = NAN;
    }
  if (ctas > 1) cluster_sync(); else __syncthreads();

  // Fold: this CTA's slice of the outputs, four columns a quad; `ways` lanes share a quad and take every ways-th
  // worker, four of them requested at once (lse and values together: one trip to the peers for up to 4 ways workers).
  const uint32_t mem = smem_u32(hkb_smem);
  const int quads = nh * (D / 4), share = (quads + ctas - 1) / ctas, x0 = rank * share, slice = min(quads, x0 + share) - x0;
  int ways = 1;
  while (ways < 32 && ways * 4 < workers && ways * 2 * share <= WARPS * 32) ways *= 2;
  const int sub = threadIdx.x & (ways - 1), rows_at_once = WARPS * 32 / ways;
  for (int y = 0; y < slice; y += rows_at_once) {       // uniform over the CTA
    const int x = x0 + y + threadIdx.x / ways;
    const bool mine = x < x0 + slice;
    const int h = mine ? x / (D / 4) : 0, c = x % (D / 4);
    float mx = -INFINITY, den = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int j0 = sub; j0 < workers; j0 += 4 * ways) {
      float lse[4];
      float4 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int j = j0 + u * ways;
        lse[u] = -INFINITY; v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (mine && j < workers) {
          const uint32_t at = peer_smem(mem + (j % WARPS) * P::RING_SMEM, j / WARPS);
          lse[u] = peer_f1(at + (HEADS * D + h) * 4);
          v[u] = peer_f4(at + (h * D + c * 4) * 4);
        }
      }
      const float top = fmaxf(mx, fmaxf(fmaxf(lse[0], lse[1]), fmaxf(lse[2], lse[3])));
      const float ref = top == -INFINITY ? 0.f : top;
      const float keep = fast_exp2((mx - ref) * LOG2E);  // 0 while nothing has been seen
      den *= keep; acc.x *= keep; acc.y *= keep; acc.z *= keep; acc.w *= keep;
      mx = top;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float wt = fast_exp2((lse[u] - ref) * LOG2E);
        den += wt;
        acc.x = fmaf(wt, v[u].x, acc.x); acc.y = fmaf(wt, v[u].y, acc.y); acc.z = fmaf(wt, v[u].z, acc.z); acc.w = fmaf(wt, v[u].w, acc.w);
      }
    }
    for (int o = 1; o < ways; o <<= 1) {
      const float top = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      const float keep = fast_exp2((mx - (top == -INFINITY ? 0.f : top)) * LOG2E);
      mx = top;
      den *= keep; acc.x *= keep; acc.y *= keep; acc.z *= keep; acc.w *= keep;
      den += __shfl_xor_sync(0xffffffffu, den, o);
      acc.x += __shfl_xor_sync(0xffffffffu, acc.x, o); acc.y += __shfl_xor_sync(0xffffffffu, acc.y, o);
      acc.z += __shfl_xor_sync(0xffffffffu, acc.z, o); acc.w += __shfl_xor_sync(0xffffffffu, acc.w, o);
    }
    if (!mine || sub) continue;
    const float inv = den == 0.f ? 0.f : 1.f / den;
    uint2 o;
    o.x = pack16x2<F16>(acc.x * inv, acc.y * inv);
    o.y = pack16x2<F16>(acc.z * inv, acc.w * inv);
    *reinterpret_cast<uint2*>(a.d.out + (int64_t)row * a.d.out_stride_tok + (int64_t)(hq0 + h) * a.d.out_stride_head + c * 4) = o;
    if (a.out_lse && c == 0)
      a.out_lse[(int64_t)row * a.d.num_q_heads + hq0 + h] = den == 0.f ? -INFINITY : mx + logf(den);
  }
  if (ctas > 1) cluster_sync();  // no CTA leaves while a peer reads its memory
}

// How many CTAs, of how many warps, share a (row, kv head). Two warps a CTA, so that many fit an SM and one's first
// and last trips to memory lie under its neighbours' streams, and as many CTAs as the machine holds at once, up to the
// portable cluster: more only adds waves of them (each costs about 6 us whatever it does), fewer leave a batch of few
// rows to few warps. Where even eight CTAs of two warps leave half the machine's mma pipes idle and each warp has more
// than eight tiles to go, four warps a CTA. Measured at head size 128, 16-token pages, us:
//   bf16, 64 x 8 items of 64 pages: 1 CTA 43.8, 2 46.6, 4 53.4 (two warps); 1 CTA of four 45.3
//   bf16, 16 x 8 items of 256 pages: 1 CTA 69.3, 2 47.3, 4 44.0, 8 47.8; 2 x 8 of 1024: 8 CTAs 37.3, of four warps 27.5
//   fp8, 48 x 8 items of 64 pages (rings half the size, so twice the CTAs fit): 1 CTA 28.2, 2 22.6, 4 27.6
// Short lists do not pay for the wider clusters: fp8, 16 x 8 items of 16 pages: 4 CTAs 6.4, 8 8.0; bf16, 8 x 8 of 32: 4
// CTAs 6.3, 8 7.1; with eight heads they pay for a pair from 2048 channels on: fp8, 64 x 8 items of 8 pages 1 CTA 6.6, 2
// 8.0; of 16 11.7, 11.3; of 32 18.7, 16.3 (sixteen heads, of 16: 18.1, 22.8: registers). Nor for a cluster at all: its
// barriers and peers' memory cost about 1 us, and a tile costs a warp 0.37, 0.48, 0.70 us (bf16, head size 64, 128, 256,
// up to eight heads; fp8 0.30, 0.49, 0.65), which the rule takes for 0.33, 0.44, 0.66. (Sixteen heads cost 0.46, 0.60,
// 1.00; taken for twice the eight, since their registers let two CTAs in instead of three.) So one CTA of four warps,
// where the items are one wave of those and the tiles a warp has more of, tiles (1/4 - 1/2c), cost less:
//   bf16, cluster / four warps: 1 x 8 items of 4 pages 4.3 / 3.5, of 8 4.4 / 4.0, of 32 5.2 / 6.7; 16 x 8 of 8 5.2 / 4.4, of
//   32 8.8 / 9.2, 32 x 8 of 16 8.9 / 8.3; head size 256, 1 x 8 of 8 5.1 / 5.4, 16 x 8 of 8 7.1 / 6.1
// and instead of a CTA of two warps where each of the four has four tiles (fp8, 48 x 8 items of 16 pages 10.0 / 7.5, of 32
// 16.7 / 12.5; head size 64, of 8 5.2 / 5.5). Over 144 shapes the rule takes 1.009 of the best form's time, 1.15 at most
// (fp8, 16 x 8 items of 64 pages 12.4, four CTAs 10.8).
struct SparseShape { int ctas, warps; };
static SparseShape sparse_shape(int rows, int kv_heads, int64_t tiles, int ring_bytes, int head_dim, int heads) {
  int sms = hkb_sm_count(-1);
  if (sms <= 0) sms = 148;
  SparseShape s = {1, 2};
  const int64_t items = (int64_t)rows * kv_heads;
  int fit = (227 << 10) / (2 * ring_bytes + 1024);
  fit = fit > 8 ? 8 : fit;
  const int wide = tiles < 64 && fit > 4 ? 4 : fit, pair = heads > 8 || tiles * head_dim < 2048 ? wide : fit;
  while (s.ctas < 8 && items * s.ctas * 2 <= (int64_t)(s.ctas == 1 ? pair : wide) * sms && tiles > s.ctas * 2) s.ctas *= 2;
  if (s.ctas == 8 && items * 8 > 2 * sms && tiles < 64) s.ctas = 4;
  const int rings = (227 << 10) / (4 * ring_bytes + 1024), regs = heads == 8 ? 3 : 2;
  const bool wave = items <= (int64_t)(rings < regs ? rings : regs) * sms;
  const int cost = (64 + head_dim / 2) * (heads / 8), bear = (items * s.ctas > sms ? 1408 : 704) * s.ctas;
  if (wave && (s.ctas == 1 ? tiles >= 16 : tiles * (s.ctas - 2) * cost <= bear)) s = {1, 4};
  else if (s.ctas == 8 && items * 8 <= 2 * sms && tiles > 128) s.warps = 4;
  return s;
}

template <int D, int KIND, int NT, int NST, int WARPS>
static int launch_sparse(const SparseArgs& a, int rows, int splits, cudaStream_t st) {
  using P = SparseWorker<D, KIND, NT, NST>;
  auto kernel = sparse_kernel<P, WARPS, KIND == HKB_KV_F16>;
  constexpr int smem = WARPS * P::RING_SMEM;
  static bool armed[64] = {};
  if (arm(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem, armed) != cudaSuccess) return HKB_ERR_CUDA;
  return launch((const void*)kernel, dim3(splits, a.d.num_kv_heads, rows), WARPS * 32, splits, smem, &a, st);
}

template <int D, int KIND, int NT>
static int dispatch_sparse(const SparseArgs& a, int rows, cudaStream_t st) {
  // Three stages a ring whatever a tile's size: head size 256, bf16, 64 x 8 items of 32 pages 48.8 us on two CTAs an SM
  // against 55.7 on three of two stages; four stages of fp8 33.6 against 27.6 (16 x 8 items of 16 pages of 256 tokens).
  constexpr int NST = 3;
  using P = SparseWorker<D, KIND, NT, NST>;
  const SparseShape shape = sparse_shape(rows, a.d.num_kv_heads, (int64_t)a.budget * a.d.tiles_per_page, P::RING_SMEM, D, P::HEADS);
  return shape.warps == 2 ? launch_sparse<D, KIND, NT, NST, 2>(a, rows, shape.ctas, st) : launch_sparse<D, KIND, NT, NST, 4>(a, rows, shape.ctas, st);
}
template <int KIND, int NT>
static int dispatch_sparse_dim(const SparseArgs& a, int head_dim, int rows, cudaStream_t st) {
  if (head_dim == 64) return dispatch_sparse<64, KIND, NT>(a, rows, st);
  return head_dim == 128 ? dispatch_sparse<128, KIND, NT>(a, rows, st) : dispatch_sparse<256, KIND, NT>(a, rows, st);
}
template <int KIND>
static int dispatch_sparse_group(const SparseArgs& a, int head_dim, int rows, cudaStream_t st) {
  return a.d.group <= 8 ? dispatch_sparse_dim<KIND, 1>(a, head_dim, rows, st) : dispatch_sparse_dim<KIND, 2>(a, head_dim, rows, st);
}

static int sparse_decode(void* out, int64_t out_stride_tok, int64_t out_stride_head, float* out_lse,
                                       const void* q, int64_t q_stride_tok, int64_t q_stride_head,
                                       hkb_cache_t kc, hkb_cache_t vc, const int32_t* block_table, int64_t table_stride,
                                       int max_pages, const int32_t* seq_lens, const int32_t* pages,
                                       int64_t pages_stride_row, int64_t pages_stride_head, int budget, int num_rows,
                                       int num_q_heads, int num_kv_heads, int head_dim, int block_size, float scale,
                                       int kv_dtype, const float* k_scale, const float* v_scale, void* stream) {
  if (num_rows < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || max_pages < 0 || budget < 0) return HKB_ERR_SIZE;
  if (num_rows == 0) return HKB_OK;
  if (num_rows > 65535 || num_kv_heads > 65535) return HKB_ERR_SIZE;
  if (!out || !q || !kc.ptr || !vc.ptr || !seq_lens) return HKB_ERR_NULL;
  if ((max_pages > 0 && !block_table) || (budget > 0 && !pages)) return HKB_ERR_NULL;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return HKB_ERR_HEAD_DIM;
  if (block_size <= 0 || block_size % TILE_TOKENS) return HKB_ERR_BLOCK_SIZE;
  if (num_q_heads % num_kv_heads || num_q_heads / num_kv_heads > HKB_MAX_GROUP) return HKB_ERR_GROUP;
  if (kv_dtype != HKB_KV_BF16 && kv_dtype != HKB_KV_FP8_E4M3 && kv_dtype != HKB_KV_F16) return HKB_ERR_DTYPE;
  const bool fp8 = kv_dtype == HKB_KV_FP8_E4M3;
  if ((fp8 && (!k_scale || !v_scale)) || !positive_scale(scale)) return HKB_ERR_SCALE;
  if (kc.num_blocks < 1 || vc.num_blocks < 1) return HKB_ERR_SIZE;
  if ((int64_t)budget * (block_size / TILE_TOKENS) > 0x7fffffff) return HKB_ERR_SIZE;
  const int es = fp8 ? 1 : 2;
  if ((kc.stride_block | kc.stride_token | kc.stride_head | vc.stride_block | vc.stride_token | vc.stride_head) * es % 16)
    return HKB_ERR_STRIDE;
  if ((q_stride_tok | q_stride_head) % 8 || (out_stride_tok | out_stride_head) % 4) return HKB_ERR_STRIDE;
  if (((uintptr_t)kc.ptr | (uintptr_t)vc.ptr | (uintptr_t)q) % 16 || (uintptr_t)out % 8 || (uintptr_t)out_lse % 4) return HKB_ERR_ALIGN;
  SparseArgs s = {};
  DecodeArgs& a = s.d;
  a.out = (__nv_bfloat16*)out; a.out_stride_tok = out_stride_tok; a.out_stride_head = out_stride_head;
  a.q = (const __nv_bfloat16*)q; a.q_stride_tok = q_stride_tok; a.q_stride_head = q_stride_head;
  a.k = (const uint8_t*)kc.ptr; a.v = (const uint8_t*)vc.ptr;
  a.k_stride_block = kc.stride_block * es; a.k_stride_token = kc.stride_token * es; a.k_stride_head = kc.stride_head * es;
  a.v_stride_block = vc.stride_block * es; a.v_stride_token = vc.stride_token * es; a.v_stride_head = vc.stride_head * es;
  const int64_t nb = kc.num_blocks < vc.num_blocks ? kc.num_blocks : vc.num_blocks;
  a.num_blocks = nb > 0x7fffffff ? 0x7fffffff : (int)nb;
  a.block_table = block_table; a.table_stride = table_stride; a.max_pages = max_pages;
  a.seq_lens = seq_lens;
  a.num_q_heads = num_q_heads; a.num_kv_heads = num_kv_heads; a.group = num_q_heads / num_kv_heads;
  a.tiles_per_page = block_size / TILE_TOKENS; a.block_size = block_size;
  a.scale = scale; a.k_scale = fp8 ? k_scale : nullptr; a.v_scale = fp8 ? v_scale : nullptr;
  s.pages = pages; s.p_stride_row = pages_stride_row; s.p_stride_head = pages_stride_head; s.budget = budget;
  s.out_lse = out_lse;
  cudaStream_t st = (cudaStream_t)stream;
  if (kv_dtype == HKB_KV_F16) return dispatch_sparse_group<HKB_KV_F16>(s, head_dim, num_rows, st);
  if (fp8) return dispatch_sparse_group<HKB_KV_FP8_E4M3>(s, head_dim, num_rows, st);
  return dispatch_sparse_group<HKB_KV_BF16>(s, head_dim, num_rows, st);
}

}  // namespace hkb

extern "C" int hkb_paged_sparse_decode(const hkb_sparse_decode_t* p, void* stream) {
  if (!p) return HKB_ERR_NULL;
  if (!hkb::ints({p->max_pages, p->budget, p->num_rows, p->num_q_heads, p->num_kv_heads, p->head_dim, p->block_size, p->kv_dtype}))
    return HKB_ERR_SIZE;
  return hkb::sparse_decode(p->out, p->out_stride_tok, p->out_stride_head, p->out_lse, p->q, p->q_stride_tok, p->q_stride_head,
                            p->k_cache, p->v_cache, p->block_table, p->table_stride, (int)p->max_pages, p->seq_lens, p->pages,
                            p->pages_stride_row, p->pages_stride_head, (int)p->budget, (int)p->num_rows, (int)p->num_q_heads,
                            (int)p->num_kv_heads, (int)p->head_dim, (int)p->block_size, (float)p->scale, (int)p->kv_dtype,
                            p->k_scale, p->v_scale, stream);
}
