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
// two products that follow (half a step, 2^-9 relative, of each entry; their sums are in fp32).
#pragma once
#include "gemm_core.h"

namespace vx {

constexpr float VL_LOG2E = 1.44269504f;

// Columns col0 + 16 g .. + 15 (g = lane / 16) of row `row` (this launch's numbering) in v: the strip's statistics go to
// *dst, the label's logit to its place. All 64 lanes call it; `live`: the row exists.
__device__ __forceinline__ void vocab_strip(const GemmParams& p, float (&v)[16], int row, bool live, int col0, float2* dst) {
  const int g = (threadIdx.x & 63) >> 4;
  const int c0 = col0 + 16 * g;
  int hit = -1;  // the label's place among the 16
  if (live) {
    const int64_t lab = p.labels[row] - p.vocab_base;
    if (lab >= c0 && lab < c0 + 16 && lab < p.N) hit = (int)(lab - c0);
  }
  float m = -INFINITY;
#pragma unroll
  for (int e = 0; e < 16; e++) {
    v[e] *= p.scale;
    if (e == hit) p.label_logit[row] = v[e];
    if (c0 + e >= p.N) v[e] = -INFINITY;
    m = fmaxf(m, v[e]);
  }
  m = fmaxf(m, __shfl_xor(m, 16, 64));
  m = fmaxf(m, __shfl_xor(m, 32, 64));
  const float ms = m == -INFINITY ? 0.f : m;  // no column, or nothing but -inf (0) and NaN (NaN)
  float s = 0.f;
#pragma unroll
  for (int e = 0; e < 16; e++) s += __builtin_amdgcn_exp2f((v[e] - ms) * VL_LOG2E);
  s += __shfl_xor(s, 16, 64);
  s += __shfl_xor(s, 32, 64);
  if (g == 0) *dst = make_float2(m, s);
}

// (m, s) += (m2, s2), both relative to their own maximum
__device__ __forceinline__ void vocab_fold(float& m, float& s, float m2, float s2) {
  const float mn = fmaxf(m, m2);
  const float ms = mn == -INFINITY ? 0.f : mn;
  s = s * __builtin_amdgcn_exp2f((m - ms) * VL_LOG2E) + s2 * __builtin_amdgcn_exp2f((m2 - ms) * VL_LOG2E);
  m = mn;
}

// the four strips of a 256-column tile, `stride` apart in LDS
__device__ __forceinline__ void vocab_fold_strips(const GemmParams& p, const float2* strips, int stride, int row, int n0) {
  float2 a = strips[0];
#pragma unroll
  for (int j = 1; j < 4; j++) vocab_fold(a.x, a.y, strips[j * stride].x, strips[j * stride].y);
  p.lse_part[(int64_t)((p.vocab_base + n0) >> 8) * p.part_ld + row] = a;
}

// The same 16 columns: their derivatives, zeros past the last column, to C (rows of p.ldc, whole 256-column tiles).
__device__ __forceinline__ void vocab_dlogits(const GemmParams& p, const float (&v)[16], int row, bool live, int col0) {
  if (!live) return;
  const int g = (threadIdx.x & 63) >> 4;
  const int c0 = col0 + 16 * g;
  if (c0 >= p.ldc) return;
  const int64_t label = p.labels[row];
  const int64_t lab = label - p.vocab_base;
  // a label outside the vocabulary has no gradient, whatever d_out holds
  const bool has = label >= 0 && label < p.tokens;
  const float d = has ? p.d_out[row] * p.scale : 0.f;
  const float lse = has ? p.lse[row] : 0.f;
  uint32_t w[8];
#pragma unroll
  for (int h = 0; h < 8; h++) {
    float o[2];
#pragma unroll
    for (int c = 0; c < 2; c++) {
      const int e = 2 * h + c;
      const float prob = __builtin_amdgcn_exp2f((v[e] * p.scale - lse) * VL_LOG2E);
      o[c] = has && c0 + e < p.N ? d * ((lab == c0 + e ? 1.f : 0.f) - prob) : 0.f;
    }
    w[h] = pack_bf16x2(o[0], o[1]);
  }
  uint4* cp = (uint4*)(p.c + (int64_t)row * p.ldc + c0);
  cp[0] = make_uint4(w[0], w[1], w[2], w[3]);
  cp[1] = make_uint4(w[4], w[5], w[6], w[7]);
}

}  // namespace vx
