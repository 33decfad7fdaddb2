// What the GEMM kernels do with a tile of logits that is never written: log-probabilities of given tokens straight
// from the hidden states and the output projection.
//   x[i, v] = scale * sum_k h[i, k] w[v, k]          (scale = 1 / temperature)
//   lse_i = log sum_v exp x[i, v],  out_i = x[i, label_i] - lse_i
//   d x[i, v] = d_out_i scale ([v == label_i] - exp(x[i, v] - lse_i)),  d h = d x W,  d W = d x^T h
// Forward: the columns are cut into strips of 64 and tiles of 256 at absolute positions. A lane of the matrix core's
// output holds 16 consecutive columns of a row (the weight rows are fed in the order that makes it so), four lanes a
// strip: maximum and sum of exponentials over the lane's 16 in ascending order, then over the four lanes, then the
// four strips of a tile in ascending order, then the tiles (vocab_logprob.hip). Every kernel does exactly this, so a
// row's bits depend on its own hidden state only. The logits stay in fp32 from the accumulator on; what the framework
// computes from a [T, V] tensor of logits rounds them to that tensor's type first.
// Backward: the same product again with the derivative as its epilogue, rounded to bf16 once, as the operand of the
// two products that follow (up to half a step, 2^-8 relative, of each entry; their sums are in fp32).
#pragma once
#include "gemm_core.h"

namespace vx {

constexpr float VL_LOG2E = 1.44269504f;

// Columns col0 + 16 g .. + 15 (g = lane / 16) of row `row` (this launch's numbering) in v, unscaled; label: the row's label
// (anything below 0 for a row that does not exist). The strip's statistics go to *dst, in units of log 2: the maximum m
// of c v with c = scale log2 e, and the sum of 2^(c v - m), each term one fused multiply-add (m is rounded: 2^-24 |m| in
// lse) and one exponential; the label's logit goes to its place. All 64 lanes call it.
__device__ __forceinline__ void vocab_strip(const GemmParams& p, float (&v)[16], int row, int64_t label, int col0, float2* dst) {
  const int g = (threadIdx.x & 63) >> 4;
  const int c0 = col0 + 16 * g;
  const float c = p.scale * VL_LOG2E;
  const int64_t at = label - p.vocab_base - c0;  // the label's place among the 16
  if (__ballot(label >= 0 && at >= 0 && at < 16 && c0 + at < p.N)) {  // one strip in some thousand per row
#pragma unroll
    for (int e = 0; e < 16; e++)
      if (label >= 0 && e == at && c0 + e < p.N) p.label_logit[row] = v[e] * c;
  }
  if (col0 + 64 > p.N) {  // wave-uniform: the vocabulary ends inside the strip
#pragma unroll
    for (int e = 0; e < 16; e++)
      if (c0 + e >= p.N) v[e] = -INFINITY;
  }
  float m = v[0];
#pragma unroll
  for (int e = 1; e < 16; e++) m = fmaxf(m, v[e]);
  m = fmaxf(m, __shfl_xor(m, 16, 64));
  m = fmaxf(m, __shfl_xor(m, 32, 64));
  m *= c;
  const float ms = m == -INFINITY ? 0.f : m;  // no column, or nothing but -inf (0) and NaN (NaN)
  float s = 0.f;
#pragma unroll
  for (int e = 0; e < 16; e++) s += __builtin_amdgcn_exp2f(__builtin_fmaf(v[e], c, -ms));
  s += __shfl_xor(s, 16, 64);
  s += __shfl_xor(s, 32, 64);
  if (g == 0) *dst = make_float2(m, s);
}

// (m, s) += (m2, s2), both relative to their own maximum (in units of log 2)
__device__ __forceinline__ void vocab_fold(float& m, float& s, float m2, float s2) {
  const float mn = fmaxf(m, m2);
  const float ms = mn == -INFINITY ? 0.f : mn;
  s = s * __builtin_amdgcn_exp2f(m - ms) + s2 * __builtin_amdgcn_exp2f(m2 - ms);
  m = mn;
}

// the four strips of a 256-column tile, `stride` apart in LDS
__device__ __forceinline__ void vocab_fold_strips(const GemmParams& p, const float2* strips, int stride, int row, int n0) {
  float2 a = strips[0];
#pragma unroll
  for (int j = 1; j < 4; j++) vocab_fold(a.x, a.y, strips[j * stride].x, strips[j * stride].y);
  p.lse_part[(int64_t)((p.vocab_base + n0) >> 8) * p.part_ld + row] = a;
}

// What a row's derivatives need: its factor -d_out scale and lse / log 2; a label outside the vocabulary has no gradient,
// whatever d_out holds.
struct VocabRow {
  int64_t label;  // in this launch's columns
  float d, lse2;
  bool has;
};
__device__ __forceinline__ VocabRow vocab_row(const GemmParams& p, int64_t label, float d_out, float lse) {
  VocabRow r;
  r.has = label >= 0 && label < p.tokens;
  r.label = label - p.vocab_base;
  r.d = r.has ? d_out * p.scale : 0.f;
  r.lse2 = r.has ? lse * VL_LOG2E : 0.f;
  return r;
}
// The same 16 columns: their derivatives, zeros past the last column, to C (rows of p.ldc, whole 64-column strips).
__device__ __forceinline__ void vocab_dlogits(const GemmParams& p, const float (&v)[16], int row, bool live, const VocabRow& r, int col0) {
  const int g = (threadIdx.x & 63) >> 4;
  const int c0 = col0 + 16 * g;
  const float c = p.scale * VL_LOG2E;
  const int64_t at = r.label - c0;
  float o[16];
#pragma unroll
  for (int e = 0; e < 16; e++) o[e] = -r.d * __builtin_amdgcn_exp2f(__builtin_fmaf(v[e], c, -r.lse2));
  if (__ballot(r.has && at >= 0 && at < 16)) {
#pragma unroll
    for (int e = 0; e < 16; e++)
      if (r.has && e == at) o[e] = r.d * (1.f - __builtin_amdgcn_exp2f(__builtin_fmaf(v[e], c, -r.lse2)));
  }
  if (col0 + 64 > p.N || __ballot(!r.has)) {  // the vocabulary ends inside the strip, or a row without a gradient (its
#pragma unroll                                // logits may be NaN or infinite)
    for (int e = 0; e < 16; e++)
      if (!r.has || c0 + e >= p.N) o[e] = 0.f;
  }
  if (!live || c0 >= p.ldc) return;
  uint4* cp = (uint4*)(p.c + (int64_t)row * p.ldc + c0);
#pragma unroll
  for (int h = 0; h < 2; h++)
    cp[h] = make_uint4(pack_bf16x2(o[8 * h], o[8 * h + 1]), pack_bf16x2(o[8 * h + 2], o[8 * h + 3]),
                       pack_bf16x2(o[8 * h + 4], o[8 * h + 5]), pack_bf16x2(o[8 * h + 6], o[8 * h + 7]));
}

}  // namespace vx
