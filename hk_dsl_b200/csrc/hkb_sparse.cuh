// The worker of the decode over selected pages: the walk's transposed products (hkb_walk_mma.cuh) with a lazier softmax.
//
// A warp of the dense walk is one of eight or twelve on its SM and hides its own latencies behind theirs; a selection is
// short, its batch often small, and then one warp's chain of products, maximum, exponentials and products is what is
// waited for. So a score is added up in two chains of products, and the maximum over a tile is not taken at all where
// it is not needed: a lane compares its own scores with the softmax reference, and only if one of the warp's exceeds it
// by 2^8 (the first tile, and rarely after) are maxima exchanged and the accumulators rescaled. A tile then takes a warp
// alone 0.52 us instead of 0.59; what is left is the issue of its instructions one after another (the tensor pipe is
// 16 % busy at twelve warps an SM). Two tiles a step took 0.48 us each and twice the shared memory: 16 x 8 items of 256
// pages 61 against 67 us on a CTA each, but 64 x 8 of 64 pages 48.3 against 45.4, where the rings are what is short.
#pragma once

#include "hkb_walk_mma.cuh"

namespace hkb {

template <int D, int KIND, int NT, int NST>
struct SparseWorker {
  static constexpr bool FP8 = KIND == HKB_KV_FP8_E4M3, F16 = KIND != HKB_KV_BF16;   // e4m3 is widened to f16
  // queries, accumulators and the partial's layout are the walk's
  using Walk = typename std::conditional<FP8, WalkMMAF8<D, NT, NST, 1>, WalkMMA<D, false, NT, 1, NST, KIND == HKB_KV_F16>>::type;
  using State = typename Walk::State;
  using Loader = typename Walk::Loader;
  static constexpr int HEAD_DIM = D, HEADS = NT * 8, STAGES = NST, KD = D / 16;
  static constexpr int STAGE_BYTES = 2 * Loader::TILE_BYTES;    // K, then V
  static constexpr int RING_SMEM = NST * STAGE_BYTES;
  static constexpr float RESCALE_LOG2 = 8.f;

  // One tile, from its first token `tok`; `tail`: it ends behind the sequence.
  __device__ static __forceinline__ void step(State& st, uint32_t ktile, int tok, int seq_len, bool tail, int lane, float qs) {
    const uint32_t vtile = ktile + Loader::TILE_BYTES;
    if (tail) {     // V rows past the sequence: their weight is 0, but 0 * NaN is NaN
      Walk::scrub_tail(vtile, tok, seq_len, lane);
      __syncwarp();
    }
    float sc[NT][4], sd[NT][4];      // even and odd chunks of the dims
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) sc[nt][i] = sd[nt][i] = 0.f;
    if constexpr (FP8) {
#pragma unroll
      for (int s = 0; s < D / 32; ++s) {
        const uint2 lo = lds64(ktile + st.koff[s]), hi = lds64(ktile + st.koff[s] + 8 * D);
        const uint32_t a0[4] = {e4m3x2_to_f16x2(lo.x), e4m3x2_to_f16x2(hi.x), e4m3x2_to_f16x2(lo.x >> 16), e4m3x2_to_f16x2(hi.x >> 16)};
        const uint32_t a1[4] = {e4m3x2_to_f16x2(lo.y), e4m3x2_to_f16x2(hi.y), e4m3x2_to_f16x2(lo.y >> 16), e4m3x2_to_f16x2(hi.y >> 16)};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mma_f16(sc[nt], a0, st.qb[nt][2 * s]);
          mma_f16(sd[nt], a1, st.qb[nt][2 * s + 1]);
        }
      }
    } else {
      const int r = (lane & 7) + ((lane >> 3) & 1) * 8;
#pragma unroll
      for (int kc = 0; kc < KD; ++kc) {
        uint32_t a[4];
        ldmatrix_x4(a, ktile + tile_off<D * 2>(r, kc * 2 + (lane >> 4)));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma16<F16>(kc & 1 ? sd[nt] : sc[nt], a, st.qb[nt][kc]);
      }
    }
    bool over = false;
    float top[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < 4; ++i) sc[nt][i] += sd[nt][i];
      if (tail) {
        if (tok + (lane >> 2) >= seq_len) sc[nt][0] = sc[nt][1] = -INFINITY;
        if (tok + (lane >> 2) + 8 >= seq_len) sc[nt][2] = sc[nt][3] = -INFINITY;
      }
      top[nt][0] = fmaxf(sc[nt][0], sc[nt][2]);
      top[nt][1] = fmaxf(sc[nt][1], sc[nt][3]);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        top[nt][c] *= qs;                          // qs > 0
        over |= top[nt][c] > st.m[nt][c] + RESCALE_LOG2;
      }
    }
    if (__any_sync(0xffffffffu, over)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float mx = fmaxf(st.m[nt][c], top[nt][c]);
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
          const float alpha = fast_exp2(st.m[nt][c] - (mx == -INFINITY ? 0.f : mx));
          st.l[nt][c] *= alpha;
#pragma unroll
          for (int dt = 0; dt < KD; ++dt) { st.o[nt][dt][c] *= alpha; st.o[nt][dt][c + 2] *= alpha; }
          st.m[nt][c] = mx;
        }
    }
    uint32_t pb[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float mu0 = st.m[nt][0] == -INFINITY ? 0.f : -st.m[nt][0], mu1 = st.m[nt][1] == -INFINITY ? 0.f : -st.m[nt][1];
      const float p0 = fast_exp2(fmaf(sc[nt][0], qs, mu0)), p1 = fast_exp2(fmaf(sc[nt][1], qs, mu1));
      const float p2 = fast_exp2(fmaf(sc[nt][2], qs, mu0)), p3 = fast_exp2(fmaf(sc[nt][3], qs, mu1));
      st.l[nt][0] += p0 + p2;
      st.l[nt][1] += p1 + p3;
      // the weights meet V in 16 bits, as in the dense walk; their sum is kept of the unrounded ones
      pb[nt][0] = movmatrix_trans(pack16x2<F16>(p0, p1));
      pb[nt][1] = movmatrix_trans(pack16x2<F16>(p2, p3));
    }
    if constexpr (FP8) {
#pragma unroll
      for (int jj = 0; jj < D / 32; ++jj) {
        const uint32_t w0 = lds32(vtile + st.voff[jj][0]), w1 = lds32(vtile + st.voff[jj][1]);
        const uint32_t w2 = lds32(vtile + st.voff[jj][0] + 8 * D), w3 = lds32(vtile + st.voff[jj][1] + 8 * D);
        const uint32_t x01 = __byte_perm(w0, w1, 0x5140), y01 = __byte_perm(w0, w1, 0x7362);
        const uint32_t x23 = __byte_perm(w2, w3, 0x5140), y23 = __byte_perm(w2, w3, 0x7362);
        const uint32_t a0[4] = {e4m3x2_to_f16x2(x01), e4m3x2_to_f16x2(x01 >> 16), e4m3x2_to_f16x2(x23), e4m3x2_to_f16x2(x23 >> 16)};
        const uint32_t a1[4] = {e4m3x2_to_f16x2(y01), e4m3x2_to_f16x2(y01 >> 16), e4m3x2_to_f16x2(y23), e4m3x2_to_f16x2(y23 >> 16)};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mma_f16(st.o[nt][2 * jj], a0, pb[nt]);
          mma_f16(st.o[nt][2 * jj + 1], a1, pb[nt]);
        }
      }
    } else {
      const int r = (lane & 7) + (lane >> 4) * 8;
#pragma unroll
      for (int dt = 0; dt < KD; ++dt) {
        uint32_t a[4];
        ldmatrix_x4_trans(a, vtile + tile_off<D * 2>(r, dt * 2 + ((lane >> 3) & 1)));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma16<F16>(st.o[nt][dt], a, pb[nt]);
      }
    }
  }
};

}  // namespace hkb
