// Routing to experts from softmax or sigmoid scores with a selection bias and expert groups, forward and backward.
//   s = softmax(x) or sigmoid(x),  c = s + bias
//   a group's score is the sum of its best one or two c; experts outside the topk_groups best groups get c = -inf
//   idx = the k largest c, descending;  w_i = scale s_i (/ sum over the selected s)
// Ties go to the lower index, among groups and among experts; NaN ranks with -inf. Beside vx_router_topk (softmax, no
// bias, no groups; vexact/models/qwen3_moe/modeling_qwen3_moe.py:128-134).
// Which of two close scores is larger must not hang on a rounding (a trainer and a rollout have to route alike, and a
// bias makes near ties common), so scores, biased scores and group scores are held in 64 bits.
// A decode step (64 tokens x 256 experts in 8 groups, 8 of them selected: 8.4 us) is bound by its eight selections, each of
// which needs the one before; a large batch by the issue of vector instructions, not by memory: 16384 tokens take 32 us (0.6
// TB/s) with the vector units at work in 91 % of the busy cycles, their gradient 17 us (2 TB/s) in 81 %. Of a forward call's
// 30 us the scores (64-bit exponential and division) and the row's loads take 11, the group scores 8 to 10 and a selection 1.1
// (k = 1 without groups 12.1 us, k = 8 20.1, k = 8 in 8 groups 29.8; softmax 14.6 / 21.9 / 29.5; no renormalisation 27.0 and
// 28.2 of the last). One wavefront per token keeps a row in registers, so every selection is a few cross-lane maxima and no
// memory is read twice.
#include "common.h"

namespace vx {

constexpr int GR_MAX_E = 512, GR_MAX_K = 64, GR_MAX_GROUPS = 64;

struct RouterParams {
  const void* logits;
  int64_t ld;
  const float* bias;  // optional
  void* weights;
  void* idx;
  int64_t T;
  int E, k, n_groups, topk_groups, group_top;
  int sigmoid, renorm;
  float scale;
};

// a 64-bit key that orders as the value does; above 0 for every value (0 marks an expert already taken)
__device__ __forceinline__ uint64_t order_key(double c) {
  if (!(c == c)) c = -INFINITY;
  const uint64_t b = __builtin_bit_cast(uint64_t, c + 0.0);  // -0 ties with +0
  return (b >> 63) ? ~b : b | 0x8000000000000000ull;
}

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

__device__ __forceinline__ double router_sigmoid(double x) { return 1.0 / (1.0 + exp(-x)); }

// One wavefront per token, lane owns experts lane + 64 i, i < PER.
template <int PER, bool LB, bool WB, bool I64>
__global__ __launch_bounds__(256) void router_grouped_kernel(RouterParams p) {
  __shared__ double cs[4][64 * PER];
  __shared__ double sel[4][GR_MAX_K];
  __shared__ int seli[4][GR_MAX_K];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const int64_t t_ = (int64_t)blockIdx.x * 4 + wv;
  const bool live = t_ < p.T;
  const int64_t t = live ? t_ : p.T - 1;  // a wavefront past the end repeats the last token and stores nothing
  float x[PER];
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const int e = lane + 64 * i;
    x[i] = -INFINITY;
    if (e < p.E) x[i] = LB ? bf16_to_f32(((const bf16_t*)p.logits)[t * p.ld + e]) : ((const float*)p.logits)[t * p.ld + e];
    m = fmaxf(m, x[i]);
  }
  double s[PER];
  if (p.sigmoid) {
#pragma unroll
    for (int i = 0; i < PER; i++) s[i] = router_sigmoid((double)x[i]);
  } else {
    m = wave_max(m);
    double z = 0.0;
#pragma unroll
    for (int i = 0; i < PER; i++) {
      s[i] = lane + 64 * i < p.E ? exp((double)x[i] - (double)m) : 0.0;
      z += s[i];
    }
    z = wave_sum_f64(z);
#pragma unroll
    for (int i = 0; i < PER; i++) s[i] /= z;
  }
  uint64_t key[PER];
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const int e = lane + 64 * i;
    const double c = s[i] + (p.bias && e < p.E ? (double)p.bias[e] : 0.0);
    key[i] = e < p.E ? order_key(c) : 0;
    cs[wv][e] = c == c ? c : -INFINITY;
  }
  if (p.n_groups > 1) {
    __syncthreads();
    // 64 >> gb lanes per group (2^gb >= n_groups) take every such element of it, their best two are merged pairwise: 8
    // groups of 32 take 4 reads and 3 merges where one lane per group took 32 reads (64 tokens: 10.1 -> 8.4 us)
    const int size = p.E / p.n_groups;
    int gb = 0;
    while ((1 << gb) < p.n_groups) gb++;
    const int lpg = 64 >> gb, grp = lane >> (6 - gb), part = lane & (lpg - 1);
    double a = -INFINITY, b = -INFINITY;
    if (grp < p.n_groups)
      for (int j = part; j < size; j += lpg) {
        const double c = cs[wv][grp * size + j];
        b = fmax(b, fmin(a, c));
        a = fmax(a, c);
      }
    for (int o = 1; o < lpg; o <<= 1) {
      const double oa = __shfl_xor(a, o, 64), ob = __shfl_xor(b, o, 64);
      b = fmax(fmin(a, oa), fmax(b, ob));
      a = fmax(a, oa);
    }
    double score = p.group_top == 2 && size > 1 ? a + b : a;
    if (!(score == score)) score = -INFINITY;  // +inf and -inf among the best two
    int before = 0;  // groups that come before this lane's
    for (int h = 0; h < p.n_groups; h++) {
      const uint64_t bits = __builtin_bit_cast(uint64_t, score);
      const double o = __builtin_bit_cast(double, ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(bits >> 32), h * lpg) << 32) |
                                                      (uint32_t)__builtin_amdgcn_readlane((int)bits, h * lpg));
      before += o > score || (o == score && h < grp);
    }
    const uint64_t kept = __ballot(grp < p.n_groups && before < p.topk_groups);  // bits grp * lpg ..
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const int e = lane + 64 * i;
      if (e < p.E && !((kept >> (e / size * lpg)) & 1)) key[i] = order_key(-INFINITY);
    }
  }
  for (int j = 0; j < p.k; j++) {
    uint32_t hi = 0;
#pragma unroll
    for (int i = 0; i < PER; i++) hi = max(hi, (uint32_t)(key[i] >> 32));
    hi = wave_max_u32(hi);
    // almost always one expert holds the largest upper half; only otherwise the lower halves decide
    int holders = 0;
#pragma unroll
    for (int i = 0; i < PER; i++) holders += __popcll(__ballot((uint32_t)(key[i] >> 32) == hi));
    uint32_t lo = 0;
    if (holders > 1) {
#pragma unroll
      for (int i = 0; i < PER; i++) lo = max(lo, (uint32_t)(key[i] >> 32) == hi ? (uint32_t)key[i] : 0u);
      lo = wave_max_u32(lo);
    }
    bool open = true;  // wave-uniform: the lowest index that holds it is the first lane of the first i
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const uint64_t who = open ? __ballot((uint32_t)(key[i] >> 32) == hi && (holders == 1 || (uint32_t)key[i] == lo)) : 0;
      if (who) {
        open = false;
        if (lane == __builtin_ctzll(who)) {
          key[i] = 0;
          sel[wv][j] = s[i];
          seli[wv][j] = lane + 64 * i;
        }
      }
    }
  }
  __syncthreads();
  const double mine = lane < p.k ? sel[wv][lane] : 0.0;
  double w = mine;
  if (p.renorm) {
    const double tot = wave_sum_f64(mine);
    w = tot == 0.0 ? 0.0 : mine / tot;  // sigmoid scores may all have vanished
  }
  if (live && lane < p.k) {
    const float wf = (float)(w * (double)p.scale);
    if constexpr (WB) ((bf16_t*)p.weights)[t * p.k + lane] = f32_to_bf16(wf);
    else ((float*)p.weights)[t * p.k + lane] = wf;
    if constexpr (I64) ((int64_t*)p.idx)[t * p.k + lane] = seli[wv][lane];
    else ((int*)p.idx)[t * p.k + lane] = seli[wv][lane];
  }
}

// Gradient of the weights with respect to the logits; the selection and the bias have none.
//   d_sel_i = scale d_w_i, renormalised: scale (d_w_i - sum_j d_w_j n_j) / S with n = s / S, S = sum of the selected s
//   sigmoid: d_x = d_sel s (1 - s) at the selected experts, 0 elsewhere
//   softmax: d_x_j = s_j (d_sel_j - sum_i d_sel_i s_i)
template <int PER, bool LB, bool WB>
__global__ __launch_bounds__(256) void router_grouped_bwd_kernel(const void* __restrict__ logits, const int64_t* __restrict__ idx,
                                                                 const void* __restrict__ d_w, void* __restrict__ d_logits, int64_t T,
                                                                 int E, int k, int64_t ld, int64_t ldo, int sigmoid, int renorm, float scale) {
  __shared__ double ss[4][64 * PER], ds[4][64 * PER];
  __shared__ int owner[4][64 * PER];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const int64_t t_ = (int64_t)blockIdx.x * 4 + wv;
  const bool live = t_ < T;
  const int64_t t = live ? t_ : T - 1;
  double s[PER];
  float x[PER], m = -INFINITY;
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const int e = lane + 64 * i;
    x[i] = -INFINITY;
    if (e < E) x[i] = LB ? bf16_to_f32(((const bf16_t*)logits)[t * ld + e]) : ((const float*)logits)[t * ld + e];
    m = fmaxf(m, x[i]);
  }
  if (sigmoid) {
#pragma unroll
    for (int i = 0; i < PER; i++) s[i] = router_sigmoid((double)x[i]);
  } else {
    m = wave_max(m);
    double z = 0.0;
#pragma unroll
    for (int i = 0; i < PER; i++) {
      s[i] = lane + 64 * i < E ? exp((double)x[i] - (double)m) : 0.0;
      z += s[i];
    }
    z = wave_sum_f64(z);
#pragma unroll
    for (int i = 0; i < PER; i++) s[i] /= z;
  }
#pragma unroll
  for (int i = 0; i < PER; i++) {
    ss[wv][lane + 64 * i] = s[i];
    ds[wv][lane + 64 * i] = 0.0;
  }
  __syncthreads();
  int at = -1;
  double sel = 0.0, d = 0.0;
  if (lane < k) {
    const int64_t v = idx[t * k + lane];
    if (v >= 0 && v < E) {  // anything else selects nothing
      at = (int)v;
      sel = ss[wv][at];
      d = (double)scale * (WB ? (double)bf16_to_f32(((const bf16_t*)d_w)[t * k + lane]) : (double)((const float*)d_w)[t * k + lane]);
    }
  }
  if (renorm) {
    const double tot = wave_sum_f64(sel);
    const double dot = wave_sum_f64(d * sel);
    d = tot == 0.0 ? 0.0 : (d - dot / tot) / tot;
  }
  const double c = wave_sum_f64(at >= 0 ? d * sel : 0.0);
  if (at >= 0) { ds[wv][at] = d; owner[wv][at] = lane; }
  __syncthreads();
  // an expert that is named twice (never by the forward) has one owner and lanes that lost: then every lane adds up the
  // derivatives of its expert in ascending order
  if (__ballot(at >= 0 && owner[wv][at] != lane)) {
    double sum = 0.0;
    for (int j = 0; j < k; j++) {
      const int other = __shfl(at, j, 64);
      const double dj = __shfl(d, j, 64);
      if (other == at) sum += dj;
    }
    if (at >= 0) ds[wv][at] = sum;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const int e = lane + 64 * i;
    if (e < E && live) {
      const double g = sigmoid ? ds[wv][e] * s[i] * (1.0 - s[i]) : s[i] * (ds[wv][e] - c);
      if constexpr (LB) ((bf16_t*)d_logits)[t * ldo + e] = f32_to_bf16((float)g);
      else ((float*)d_logits)[t * ldo + e] = (float)g;
    }
  }
}

}  // namespace vx

using namespace vx;

extern "C" {

static int router_args(int64_t T, int E, int k, int n_groups, int topk_groups, int group_top) {
  if (T < 0 || E <= 0 || k <= 0 || n_groups <= 0 || topk_groups <= 0) return VX_ERR_ARG;
  if (E % n_groups != 0 || topk_groups > n_groups || (group_top != 1 && group_top != 2)) return VX_ERR_ARG;
  if ((int64_t)topk_groups * (E / n_groups) < k) return VX_ERR_ARG;
  if (E > GR_MAX_E || k > GR_MAX_K || n_groups > GR_MAX_GROUPS || (T + 3) / 4 > 0x7fffffff) return VX_ERR_UNSUPPORTED;
  return VX_OK;
}

#define VX_ROUTER_PER(CALL)            \
  do {                                 \
    if (E <= 64) { CALL(1); }          \
    else if (E <= 128) { CALL(2); }    \
    else if (E <= 256) { CALL(4); }    \
    else { CALL(8); }                  \
  } while (0)

int vx_router_grouped(const void* logits, const float* bias, void* weights, void* idx, int64_t T, int E, int k, int64_t ld,
                      int sigmoid, int n_groups, int topk_groups, int group_top, int renorm, float scale, int logits_bf16,
                      int weights_bf16, int idx_i64, hipStream_t stream) {
  if (!logits || !weights || !idx) return VX_ERR_ARG;
  const int rc = router_args(T, E, k, n_groups, topk_groups, group_top);
  if (rc != VX_OK) return rc;
  if (T == 0) return VX_OK;
  RouterParams p = {logits, ld, bias, weights, idx, T, E, k, n_groups, topk_groups, group_top, sigmoid, renorm, scale};
  const unsigned grid = (unsigned)((T + 3) / 4);
#define VX_GR(PER)                                                                                                     \
  if (logits_bf16 && weights_bf16 && idx_i64) router_grouped_kernel<PER, true, true, true><<<grid, 256, 0, stream>>>(p);    \
  else if (logits_bf16 && weights_bf16) router_grouped_kernel<PER, true, true, false><<<grid, 256, 0, stream>>>(p);         \
  else if (logits_bf16 && idx_i64) router_grouped_kernel<PER, true, false, true><<<grid, 256, 0, stream>>>(p);              \
  else if (logits_bf16) router_grouped_kernel<PER, true, false, false><<<grid, 256, 0, stream>>>(p);                        \
  else if (weights_bf16 && idx_i64) router_grouped_kernel<PER, false, true, true><<<grid, 256, 0, stream>>>(p);             \
  else if (weights_bf16) router_grouped_kernel<PER, false, true, false><<<grid, 256, 0, stream>>>(p);                       \
  else if (idx_i64) router_grouped_kernel<PER, false, false, true><<<grid, 256, 0, stream>>>(p);                            \
  else router_grouped_kernel<PER, false, false, false><<<grid, 256, 0, stream>>>(p)
  VX_ROUTER_PER(VX_GR);
#undef VX_GR
  return launch_status();
}

int vx_router_grouped_bwd(const void* logits, const int64_t* idx, const void* d_weights, void* d_logits, int64_t T, int E, int k,
                          int64_t ld, int64_t ld_out, int sigmoid, int renorm, float scale, int logits_bf16, int weights_bf16,
                          hipStream_t stream) {
  if (!logits || !idx || !d_weights || !d_logits) return VX_ERR_ARG;
  const int rc = router_args(T, E, k, 1, 1, 1);
  if (rc != VX_OK) return rc;
  if (T == 0) return VX_OK;
  const unsigned grid = (unsigned)((T + 3) / 4);
#define VX_GRB(PER, LBV, WBV) \
  router_grouped_bwd_kernel<PER, LBV, WBV><<<grid, 256, 0, stream>>>(logits, idx, d_weights, d_logits, T, E, k, ld, ld_out, sigmoid, renorm, scale)
#define VX_GRC(PER)                                        \
  if (logits_bf16 && weights_bf16) VX_GRB(PER, true, true); \
  else if (logits_bf16) VX_GRB(PER, true, false);           \
  else if (weights_bf16) VX_GRB(PER, false, true);          \
  else VX_GRB(PER, false, false)
  VX_ROUTER_PER(VX_GRC);
#undef VX_GRC
#undef VX_GRB
  return launch_status();
}

}  // extern "C"
