// The worker of the decode over selected pages: the walk's transposed products (hkb_walk_mma.cuh) with a lazier softmax, and
// bf16 weights in two terms.
//
// A warp of the dense walk is one of eight or twelve on its SM and hides its own latencies behind theirs; a selection is
// short, its batch often small, and then one warp's chain of products, maximum, exponentials and products is what is
// waited for. So a score is added up in two chains of products (the fp8 walk does that too), and where the dense walks
// exchange every tile's maximum to compare it with the softmax reference, here a lane compares its own scores, and only
// if one of the warp's exceeds the reference by 2^8 (the first tile, and rarely after) are maxima exchanged and the
// accumulators rescaled: 16 x 8 items of 256 pages, a CTA of two warps each and one bf16 term a weight, 67 us instead of
// 77. A tile (bf16, head size 128, two terms) costs a warp 0.48 us where its SM holds no other CTA and 0.51 where all SMs
// are full (0.42 and 0.47 with one); what is left is the issue of its instructions one after another (the tensor pipe is
// 16 % busy at twelve warps an SM). Two tiles a step took 0.48 us each and twice the shared memory: 16 x 8 items of 256
// pages 61 against 67 us on a CTA each, but 64 x 8 of 64 pages 48.3 against 45.4, where the rings are what is short.
#pragma once

#include "hkb_walk_mma.cuh"

namespace hkb {

// A head of a bf16 query as f16, for an fp8 cache's products: its values times the power of two that brings the greatest
// magnitude `top` into [2^13, 2^14). That is exact, none overflows whatever the query's range, and what falls under f16's
// is off by 2^-38 of the greatest at most. `up` undoes it. (top zero, subnormal or infinite: a finite pair all the same.)
struct F16Scale { float down, up; };
__device__ __forceinline__ F16Scale f16_scale(float top) {
  const int e = min(max((int)(__float_as_uint(top) >> 23), 14), 253);   // biased exponent
  return {__uint_as_float((uint32_t)(267 - e) << 23), __uint_as_float((uint32_t)(e - 13) << 23)};
}

template <int D, int KIND, int NT, int NST>
struct SparseWorker {
  static constexpr bool FP8 = KIND == HKB_KV_FP8_E4M3, F16 = KIND != HKB_KV_BF16;   // e4m3 is widened to f16
  // accumulators and the partial's layout are the walk's
  using Walk = typename std::conditional<FP8, WalkMMAF8<D, NT, NST, 1>, WalkMMA<D, false, NT, 1, NST, KIND == HKB_KV_F16>>::type;
  struct State : Walk::State { float qs[NT][2]; };     // and what a column's products are multiplied by: logits in units of ln 2
  using Loader = typename Walk::Loader;
  static constexpr int HEAD_DIM = D, HEADS = NT * 8, STAGES = NST, KD = D / 16;
  static constexpr int STAGE_BYTES = 2 * Loader::TILE_BYTES;    // K, then V
  static constexpr int RING_SMEM = NST * STAGE_BYTES;
  static constexpr float RESCALE_LOG2 = 8.f;

  // The weights meet V in 16 bits; their sum is kept of the unrounded ones. fp16's eleven bits do for fp16 answers and for
  // an fp8 cache's bf16 ones (error against float64 0.00027 of the norm, rounded once 0.00021; 0.0017, 0.0017). bf16's eight
  // do not (0.0023, 0.0017), so a bf16 weight is two terms, its upper half and what is left, multiplied one after the other
  // by the V fragment that is there: 0.0017. Both are positive, or an infinite value would meet 0 or two signs and be NaN.
  static constexpr int TERMS = KIND == HKB_KV_BF16 ? 2 : 1;
  __device__ static __forceinline__ uint32_t upper16x2(float lo, float hi) {
    return __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x7632);
  }
  __device__ static __forceinline__ float rest(float x) { return fmaxf(x - bf16hi(__float_as_uint(x)), 0x1p-126f); }

  // As the walk's, but for an fp8 cache's query, which the walk cuts at f16's range: here each head is scaled into it, and
  // NaN and infinities stay what they are.
  __device__ static __forceinline__ void begin(State& st, const DecodeArgs& a, int row, int hq0, int nh, int lane, float qs) {
    if constexpr (FP8) Walk::clear(st, lane);
    else Walk::begin(st, a, row, hq0, nh, lane, qs);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      st.qs[nt][0] = st.qs[nt][1] = qs;
      if constexpr (FP8) {
        const int h = nt * 8 + (lane >> 2), t = lane & 3;
        const uint4* qp = reinterpret_cast<const uint4*>(a.q + (int64_t)row * a.q_stride_tok + (int64_t)(hq0 + h) * a.q_stride_head);
        uint32_t w[KD][2];                           // dims 32 s + 8 t .. + 7: chunks 2 s and 2 s + 1
        float top = 0.f;
#pragma unroll
        for (int s = 0; s < D / 32; ++s) {
          uint4 v = make_uint4(0u, 0u, 0u, 0u);
          if (h < nh) v = __ldg(qp + s * 4 + t);
          w[2 * s][0] = v.x; w[2 * s][1] = v.y; w[2 * s + 1][0] = v.z; w[2 * s + 1][1] = v.w;
        }
#pragma unroll
        for (int kc = 0; kc < KD; ++kc)
#pragma unroll
          for (int i = 0; i < 2; ++i) top = fmaxf(top, fmaxf(fabsf(bf16lo(w[kc][i])), fabsf(bf16hi(w[kc][i]))));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const F16Scale f = f16_scale(top);
#pragma unroll
        for (int kc = 0; kc < KD; ++kc)
#pragma unroll
          for (int i = 0; i < 2; ++i) st.qb[nt][kc][i] = pack_f16x2(bf16lo(w[kc][i]) * f.down, bf16hi(w[kc][i]) * f.down);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float x = qs * __shfl_sync(0xffffffffu, f.up, (2 * t + c) * 4);
          // neither 0, which makes NaN of a masked -inf, nor infinite, which makes NaN of a product of 0: products are
          // below 2^31, so under 2^-126 the logits are nothing
          if (fabsf(x) < 0x1p-126f) x = 0x1p-126f;
          if (x > 0x1.fffffep127f && qs <= 0x1.fffffep127f) x = 0x1.fffffep127f;
          st.qs[nt][c] = x;
        }
      }
    }
  }

  // One tile, from its first token `tok`; `tail`: it ends behind the sequence.
  __device__ static __forceinline__ void step(State& st, uint32_t ktile, int tok, int seq_len, bool tail, int lane) {
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
        top[nt][c] *= st.qs[nt][c];                // > 0
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
    uint32_t pb[NT][2], pr[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float mu0 = st.m[nt][0] == -INFINITY ? 0.f : -st.m[nt][0], mu1 = st.m[nt][1] == -INFINITY ? 0.f : -st.m[nt][1];
      const float qs0 = st.qs[nt][0], qs1 = st.qs[nt][1];
      const float p0 = fast_exp2(fmaf(sc[nt][0], qs0, mu0)), p1 = fast_exp2(fmaf(sc[nt][1], qs1, mu1));
      const float p2 = fast_exp2(fmaf(sc[nt][2], qs0, mu0)), p3 = fast_exp2(fmaf(sc[nt][3], qs1, mu1));
      st.l[nt][0] += p0 + p2;
      st.l[nt][1] += p1 + p3;
      if constexpr (TERMS == 1) {
        pb[nt][0] = movmatrix_trans(pack16x2<F16>(p0, p1));
        pb[nt][1] = movmatrix_trans(pack16x2<F16>(p2, p3));
      } else {
        pb[nt][0] = movmatrix_trans(upper16x2(p0, p1));
        pb[nt][1] = movmatrix_trans(upper16x2(p2, p3));
        pr[nt][0] = movmatrix_trans(pack_bf16x2(rest(p0), rest(p1)));
        pr[nt][1] = movmatrix_trans(pack_bf16x2(rest(p2), rest(p3)));
      }
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
        for (int nt = 0; nt < NT; ++nt) {
          mma16<F16>(st.o[nt][dt], a, pb[nt]);
          if constexpr (TERMS == 2) mma16<F16>(st.o[nt][dt], a, pr[nt]);
        }
      }
    }
  }
};

}  // namespace hkb
