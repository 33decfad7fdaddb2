// Log-probabilities of given tokens straight from the hidden states and the output projection, and their gradients,
// without logits in memory (mathematics and roundings: vocab_logprob.h). Beside vx_logprobs, which wants the
// [T, V] logits (vexact/batch_invariant_ops/standalone_logprobs.py:28-55).
//   forward : GEMM with the row statistics as its epilogue -> one (max, sum) per row and 256 columns -> fold per row
//   backward: per piece of the vocabulary, GEMM with the derivative as its epilogue into a bf16 piece [T, piece], then
//             d W rows of the piece = piece^T h, and fp32 partial sums of d h per segment of 8192 columns, folded in
//             ascending order. The segments are at absolute positions, so the bits do not depend on the piece width.
// Bound by the matrix products from some hundred rows on: 16384 rows x 151936 x 2048 take 7.8 ms (1.31 PFLOP/s, 88 % of a
// library product's rate); 4096 rows with gradients 8.8 ms: forward 1.33, recomputed logits 1.26, d h 1.05, d W 1.08 PFLOP/s
// (the last two read their operands through 8-byte transposing LDS reads). A few rows are bound by reading the weights once
// (7 rows: 114 us, 5.7 TB/s).
#include <algorithm>

#include "gemm_core.h"
#include "gemm_seg.h"
#include "gemm_wide.h"
#include "vocab_logprob.h"

namespace vx {

constexpr int VL_BM = 64, VL_BN = 256, VL_BK = 64;
constexpr int VL_RB = VL_BK * 2 + 16;  // LDS row pitch: 16 bytes on, so that the rows of a fragment read hit distinct banks
constexpr int VL_SEG = 8192;           // columns per partial sum of d h
constexpr int VL_FEW = 64;             // rows up to which the forward streams the weights (gemm_stream_kernel)
constexpr int VL_ROW_EACH = 512;       // rows up to which the final fold has a workgroup for each

// The general kernel: any H that is a multiple of 8, any number of rows. 64 rows x 256 columns per workgroup, one
// 64-column strip per wavefront, operands through registers into one of two LDS buffers.
template <int EPI>
__global__ __launch_bounds__(256) void vocab_gemm_kernel(GemmParams p) {
  __shared__ __attribute__((aligned(16))) uint8_t lx[2][VL_BM * VL_RB];
  __shared__ __attribute__((aligned(16))) uint8_t lw[2][VL_BN * VL_RB];
  __shared__ float2 strips[4][VL_BM];
  const int row0 = blockIdx.y * VL_BM, n0 = blockIdx.x * VL_BN;
  const int rows = min(VL_BM, p.M - row0), K = p.K;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int r16 = lane & 15, g = lane >> 4;

  // piece q = tid + 256 j: row q / 8, 16-byte piece q % 8 (the same for all j)
  const int c8 = tid & 7;
  const bf16_t* xrow[2];
  const bf16_t* wrow[8];
#pragma unroll
  for (int j = 0; j < 2; j++) xrow[j] = p.x + (int64_t)(row0 + min((tid >> 3) + 32 * j, rows - 1)) * p.ldx;
#pragma unroll
  for (int j = 0; j < 8; j++) wrow[j] = p.w + (int64_t)min(n0 + (tid >> 3) + 32 * j, p.N - 1) * p.ldw;
  uint4 gx[2], gw[8];
  auto gload = [&](int k0) {
    const int k = k0 + 8 * c8 < K ? k0 + 8 * c8 : 0;  // a piece past K re-reads the row's first one; zeroed in lstore
#pragma unroll
    for (int j = 0; j < 2; j++) gx[j] = ldg16_raw(xrow[j] + k);
#pragma unroll
    for (int j = 0; j < 8; j++) gw[j] = ldg16_raw(wrow[j] + k);
  };
  auto lstore = [&](int buf, int k0) {
    const bool ok = k0 + 8 * c8 < K;
#pragma unroll
    for (int j = 0; j < 2; j++) *(uint4*)(&lx[buf][((tid >> 3) + 32 * j) * VL_RB + c8 * 16]) = mask16(gx[j], ok);
#pragma unroll
    for (int j = 0; j < 8; j++) *(uint4*)(&lw[buf][((tid >> 3) + 32 * j) * VL_RB + c8 * 16]) = mask16(gw[j], ok);
  };

  f32x4 acc[4][4];  // [row tile][weight fragment]
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int nk = (K + VL_BK - 1) / VL_BK;
  gload(0);
  lstore(0, 0);
  __syncthreads();
  for (int kt = 0; kt < nk; kt++) {
    const int buf = kt & 1;
    if (kt + 1 < nk) gload((kt + 1) * VL_BK);
#pragma unroll
    for (int ks = 0; ks < 2; ks++) {
      uint4 wf[4], xf[4];
      // MFMA row rho of fragment j is weight row 16 (rho / 4) + 4 j + rho % 4 of the strip: a lane then holds 16
      // consecutive columns
#pragma unroll
      for (int j = 0; j < 4; j++)
        wf[j] = *(const uint4*)(&lw[buf][(64 * wave + 16 * (r16 >> 2) + 4 * j + (r16 & 3)) * VL_RB + (32 * ks + 8 * g) * 2]);
#pragma unroll
      for (int i = 0; i < 4; i++) xf[i] = *(const uint4*)(&lx[buf][(16 * i + r16) * VL_RB + (32 * ks + 8 * g) * 2]);
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] = mfma16(wf[j], xf[i], acc[i][j]);
    }
    if (kt + 1 < nk) lstore(buf ^ 1, (kt + 1) * VL_BK);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int m = 16 * i + r16;
    float v[16];
#pragma unroll
    for (int e = 0; e < 16; e++) v[e] = acc[i][e >> 2][e & 3];
    const bool live = m < rows;
    const int64_t label = live ? p.labels[row0 + m] : -1;
    if constexpr (EPI == EPI_LSE) {
      vocab_strip(p, v, row0 + m, label, n0 + 64 * wave, &strips[wave][m]);
    } else {
      const VocabRow r = vocab_row(p, label, live ? p.d_out[row0 + m] : 0.f, live ? p.lse[row0 + m] : 0.f);
      vocab_dlogits(p, v, row0 + m, live, r, n0 + 64 * wave);
    }
  }
  if constexpr (EPI == EPI_LSE) {
    __syncthreads();
    if (tid < rows) vocab_fold_strips(p, &strips[0][tid], VL_BM, row0 + tid, n0);
  }
}

// out = x[label] - lse, lse = M + log S over a row's tile statistics. One wavefront per row, lane r folds the tiles r, r + 64,
// ... in ascending order, then the lanes fold pairwise (r with r ^ 32, then 16, ... 1). STRIPS: the four strips of a tile
// come one by one. Up to 512 rows a workgroup each and ten tiles of a lane on their way at once, since the time is that of
// trips to memory (V = 151936: 16 rows 132 -> 116 us the whole call, 300 rows 4 us less); more rows in workgroups of 16: with
// [tile][row] partials one of its loads then uses whole 128-byte lines (8192 rows x 256: 697 against 737 us).
template <bool STRIPS, int ROWS>
__global__ __launch_bounds__(64 * ROWS) void vocab_final_kernel(const float2* __restrict__ part, int64_t part_ld, int ntiles, int nstrips,
                                                           const float* __restrict__ label_logit, const int64_t* __restrict__ labels,
                                                           float* __restrict__ out, float* __restrict__ lse_out, int64_t T, int64_t V) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * ROWS + (threadIdx.x >> 6);
  if (row >= T) return;
  float m = -INFINITY, sum = 0.f;
  constexpr int U = ROWS == 1 ? 10 : 4, NS = STRIPS ? 4 : 1;
  const int last = (STRIPS ? nstrips : ntiles) - 1;
  for (int t0 = lane; t0 < ntiles; t0 += 64 * U) {
    float2 st[U][NS];
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int j = 0; j < NS; j++) st[u][j] = part[(int64_t)min(NS * (t0 + 64 * u) + j, last) * part_ld + row];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int t = t0 + 64 * u;
      if (t < ntiles) {
        float2 a = st[u][0];
#pragma unroll
        for (int j = 1; j < NS; j++) {
          const bool there = NS * t + j <= last;
          vocab_fold(a.x, a.y, there ? st[u][j].x : -INFINITY, there ? st[u][j].y : 0.f);
        }
        vocab_fold(m, sum, a.x, a.y);
      }
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float m2 = __shfl_xor(m, o, 64), s2 = __shfl_xor(sum, o, 64);
    vocab_fold(m, sum, m2, s2);
  }
  if (lane != 0) return;
  const float ls = __builtin_amdgcn_logf(sum);  // log2, as m
  if (lse_out) lse_out[row] = (m + ls) * 0.693147181f;
  if (out) {
    const int64_t lab = labels[row];
    out[row] = lab >= 0 && lab < V ? ((label_logit[row] - m) - ls) * 0.693147181f : NAN;
  }
}

// d h: acc (+)= the partial sums of a piece's segments, in ascending order; after the last piece rounded to bf16.
// Four columns per thread.
__global__ __launch_bounds__(256) void vocab_dh_kernel(const float* __restrict__ part, int nseg, int64_t stride, float* __restrict__ acc,
                                                       int first, bf16_t* __restrict__ dh, int64_t ld, int64_t T, int H) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= T * H) return;
  f32x4 a = first ? *(const f32x4*)(part + i) : *(const f32x4*)(acc + i);
  for (int s = first ? 1 : 0; s < nseg; s++) a += *(const f32x4*)(part + s * stride + i);
  if (dh) {
    uint2 pk;
    pk.x = pack_bf16x2(a[0], a[1]);
    pk.y = pack_bf16x2(a[2], a[3]);
    *(uint2*)(dh + i / H * ld + i % H) = pk;
  } else {
    *(f32x4*)(acc + i) = a;
  }
}

// The rows that d W multiplies the derivatives with: those without a label as zeros. Their derivatives are zeros, and a
// padded row may hold anything, NaN times 0 among it. Eight elements per thread.
__global__ __launch_bounds__(256) void vocab_rows_kernel(const bf16_t* __restrict__ h, int64_t ldh, const int64_t* __restrict__ labels,
                                                         bf16_t* __restrict__ out, int64_t T, int H, int64_t V) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int per = H / 8;
  const int64_t row = i / per;
  if (row >= T) return;
  const int col = (int)(i - row * per) * 8;
  const int64_t label = labels[row];
  *(uint4*)(out + row * H + col) = ldg16(h + row * ldh + col, label >= 0 && label < V);
}

// Rows of the wide kernel's tiles: those whose rounds of 256 workgroups take least, a tile of 192 or 128 rows counted as
// 0.85 or 0.7 of one of 256.
static int vocab_tile_rows(int64_t M, int64_t N) {
  const int64_t tn = (N + WD_BN - 1) / WD_BN;
  auto cost = [&](int64_t bm, int64_t weight) { return ((M + bm - 1) / bm * tn + 255) / 256 * weight; };
  const int64_t c256 = cost(256, 100), c192 = cost(192, 85), c128 = cost(128, 70);
  return c128 < c192 && c128 < c256 ? 128 : c192 < c256 ? 192 : 256;
}

// Logit products of the columns [0, N) of this launch's weights for all rows; row chunks keep the wide kernel's 32-bit
// offsets in range.
template <int EPI>
static int launch_vocab_gemm(const GemmParams& p_in, int64_t T, hipStream_t stream) {
  const int64_t lim = (int64_t)1 << 32;
  int64_t chunk = T;
  while ((chunk * p_in.ldx + p_in.K) * 2 >= lim || (chunk + 63) / 64 > 65535) chunk = (chunk / 2 + 255) / 256 * 256;
  for (int64_t r0 = 0; r0 < T; r0 += chunk) {
    GemmParams p = p_in;
    p.M = (int)std::min(chunk, T - r0);
    p.x += r0 * p.ldx;
    p.labels += r0;
    if (EPI == EPI_LSE) { p.lse_part += r0; p.label_logit += r0; }
    else { p.lse += r0; p.d_out += r0; p.c += r0 * p.ldc; }
    if (EPI == EPI_LSE && T <= VL_FEW) {
      const unsigned nt = (unsigned)(((int64_t)p.N + 63) / 64);
      if (p.M <= 16) gemm_stream_kernel<1, EPI_LSE, false, 8, 2><<<nt, 256, 0, stream>>>(p);
      else if (p.M <= 32) gemm_stream_kernel<2, EPI_LSE, false, 8, 2><<<nt, 256, 0, stream>>>(p);
      else gemm_stream_kernel<4, EPI_LSE, false><<<nt, 256, 0, stream>>>(p);
      continue;
    }
    if (p.M > 64) {
      bool done;
      switch (vocab_tile_rows(p.M, p.N)) {
        case 128: done = gemm_wide_launch_t<EPI, false, 4>(p, ((int64_t)p.M + 127) / 128, p.M, stream); break;
        case 192: done = gemm_wide_launch_t<EPI, false, 6>(p, ((int64_t)p.M + 191) / 192, p.M, stream); break;
        default: done = gemm_wide_launch_t<EPI, false>(p, ((int64_t)p.M + WD_BM - 1) / WD_BM, p.M, stream);
      }
      if (done) continue;
    }
    const dim3 grid((unsigned)(((int64_t)p.N + VL_BN - 1) / VL_BN), (unsigned)(((int64_t)p.M + VL_BM - 1) / VL_BM));
    vocab_gemm_kernel<EPI><<<grid, 256, 0, stream>>>(p);
  }
  return launch_status();
}

// The kernels address a launch's rows with 32-bit byte offsets: launches of 256 rows or columns, the fewest that these are
// split into, must stay within them.
constexpr int64_t VL_MAX_LD = (int64_t)1 << 22;
static bool vocab_args_ok(const void* h, const void* w, int64_t T, int64_t V, int64_t H, int64_t ldh, int64_t ldw) {
  return V <= 0x7fffff00 && T <= 0x7fffff00 && H <= VL_MAX_LD && ldh >= 0 && ldw >= 0 && ldh <= VL_MAX_LD && ldw <= VL_MAX_LD &&
         gemm_fast_ok(h, w, H, ldh, ldw);
}

// The kernels work with scale log2 e: an infinite one, or one that the hardware flushes to zero, makes NaN of the -inf that
// stands in for columns past the vocabulary; a negative one takes the smallest logit for the largest.
static bool vocab_scale_ok(float scale) { return scale >= 0x1p-126f && scale <= 0x1p127f; }

// columns of one launch: whole 256-column tiles, weight bytes within 32 bits
static int64_t vocab_cols_limit(int64_t V, int64_t H, int64_t ldw) {
  int64_t n = (V + 255) / 256 * 256;
  while ((n * ldw + H) * 2 >= ((int64_t)1 << 32)) n = (n / 2 + 255) / 256 * 256;
  return n;
}

static inline int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }

// The backward's piece: segments per piece so that the piece and its partial sums stay near 768 MB (the whole
// vocabulary at once up to some hundred rows, one segment at a time from some ten thousand) and the piece's weights
// within the kernels' 32-bit offsets. Rows are never split (d W is one chain over them), so from there on the workspace grows
// with them, T (16384 + 10 H) bytes: 1.0 GB at 16384 rows of H 2048, 2.4 GB at 65536.
struct VocabPlan {
  int64_t segs, per, pieces, ld;  // segments of the vocabulary, of a piece; pieces; columns of the piece buffer
  int64_t dlog_bytes, part_bytes, acc_bytes, rows_bytes;
  int64_t bytes() const { return dlog_bytes + part_bytes + acc_bytes + rows_bytes; }
};
static VocabPlan vocab_plan(int64_t T, int64_t V, int64_t H, int64_t ldw) {
  VocabPlan q;
  q.segs = (V + VL_SEG - 1) / VL_SEG;
  const int64_t seg_bytes = T * VL_SEG * 2 + T * H * 4;
  const int64_t reach = ((((int64_t)1 << 32) - 1) / 2 - H) / (VL_SEG * ldw);
  const int64_t most = std::max<int64_t>(1, std::min({q.segs, ((int64_t)768 << 20) / seg_bytes, reach}));
  q.pieces = (q.segs + most - 1) / most;
  q.per = (q.segs + q.pieces - 1) / q.pieces;
  q.pieces = (q.segs + q.per - 1) / q.per;
  q.ld = std::min(q.per * VL_SEG, (V + 63) / 64 * 64);
  q.dlog_bytes = up256(T * q.ld * 2);
  q.part_bytes = up256(q.per * T * H * 4);
  q.acc_bytes = up256(T * H * 4);
  q.rows_bytes = up256(T * H * 2);
  return q;
}

// whether the products over a piece stay within their kernels' 32-bit offsets, and vocab_dh_kernel's grid below 2^32 threads
static bool vocab_plan_fits(const VocabPlan& q, int64_t T, int64_t H, int64_t ldw) {
  const int64_t lim = (int64_t)1 << 32;
  return (T * q.ld + VL_SEG) * 2 < lim && (q.per * VL_SEG * ldw + H) * 2 < lim && T * H / 4 <= 0xffffff00;
}

}  // namespace vx

using namespace vx;

extern "C" {

int64_t vx_vocab_logprobs_workspace_bytes(int64_t T, int64_t V) {
  if (T <= 0 || V <= 0) return 0;
  // per 256 columns, or per 64 for a few rows
  return up256((T <= VL_FEW ? (V + 255) / 256 * 4 : (V + 255) / 256) * T * 8) + up256(T * 4);
}

int vx_vocab_logprobs(const void* hidden, const void* weight, const int64_t* labels, float* out, float* lse, int64_t T, int64_t V,
                      int64_t H, int64_t ldh, int64_t ldw, float scale, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  if (!hidden || !weight || !labels || (!out && !lse) || T < 0 || V <= 0 || H <= 0 || !vocab_scale_ok(scale)) return VX_ERR_ARG;
  if (!vocab_args_ok(hidden, weight, T, V, H, ldh, ldw)) return VX_ERR_UNSUPPORTED;
  if (T == 0) return VX_OK;
  if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < vx_vocab_logprobs_workspace_bytes(T, V)) return VX_ERR_WORKSPACE;
  const int64_t ntiles = (V + 255) / 256, step = vocab_cols_limit(V, H, ldw);
  GemmParams p = {};
  p.x = (const bf16_t*)hidden; p.ldx = ldh;
  p.ldw = ldw; p.K = (int)H;
  p.labels = labels; p.scale = scale; p.tokens = V;
  p.lse_part = (float2*)workspace; p.part_ld = T;
  const bool few = T <= VL_FEW;
  p.label_logit = (float*)((uint8_t*)workspace + up256((few ? 4 * ntiles : ntiles) * T * 8));
  for (int64_t v0 = 0; v0 < V; v0 += step) {
    p.w = (const bf16_t*)weight + v0 * ldw;
    p.N = (int)std::min(step, V - v0);
    p.vocab_base = (int)v0;
    const int rc = launch_vocab_gemm<EPI_LSE>(p, T, stream);
    if (rc != VX_OK) return rc;
  }
  const int nstrips = (int)((V + 63) / 64);
  auto final = [&](auto kernel, int64_t rows) {
    kernel<<<(unsigned)((T + rows - 1) / rows), 64 * rows, 0, stream>>>(p.lse_part, T, (int)ntiles, nstrips, p.label_logit, labels, out, lse, T, V);
  };
  static_assert(VL_FEW <= VL_ROW_EACH);
  if (few) final(vocab_final_kernel<true, 1>, 1);
  else if (T <= VL_ROW_EACH) final(vocab_final_kernel<false, 1>, 1);
  else final(vocab_final_kernel<false, 16>, 16);
  return launch_status();
}

int64_t vx_vocab_logprobs_bwd_workspace_bytes(int64_t T, int64_t V, int64_t H) {
  if (T <= 0 || V <= 0 || H <= 0 || T > 0x7fffff00 || V > 0x7fffff00 || H > VL_MAX_LD) return 0;
  const VocabPlan q = vocab_plan(T, V, H, H);  // a larger row pitch only makes for more, smaller pieces
  return vocab_plan_fits(q, T, H, H) ? q.bytes() : 0;
}

int vx_vocab_logprobs_bwd(const void* hidden, const void* weight, const int64_t* labels, const float* lse, const float* d_out,
                          void* d_hidden, void* d_weight, int64_t T, int64_t V, int64_t H, int64_t ldh, int64_t ldw, int64_t ld_dh,
                          int64_t ld_dw, float scale, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  if (!hidden || !weight || !labels || !lse || !d_out || (!d_hidden && !d_weight) || T <= 0 || V <= 0 || H <= 0 || !vocab_scale_ok(scale))
    return VX_ERR_ARG;
  if (!vocab_args_ok(hidden, weight, T, V, H, ldh, ldw)) return VX_ERR_UNSUPPORTED;
  if ((d_hidden && (ld_dh % 4 || ((uintptr_t)d_hidden & 7))) || (d_weight && (ld_dw % 4 || ((uintptr_t)d_weight & 7)))) return VX_ERR_UNSUPPORTED;
  // rows closer than H, or one for all: as vx_vocab_logprobs_bwd_workspace_bytes plans
  const VocabPlan q = vocab_plan(T, V, H, std::max(ldw, H));
  if (!vocab_plan_fits(q, T, H, std::max(ldw, H))) return VX_ERR_UNSUPPORTED;
  if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < q.bytes()) return VX_ERR_WORKSPACE;
  bf16_t* dlog = (bf16_t*)workspace;
  float* part = (float*)((uint8_t*)workspace + q.dlog_bytes);
  float* acc = (float*)((uint8_t*)part + q.part_bytes);
  bf16_t* rows = (bf16_t*)((uint8_t*)acc + q.acc_bytes);
  if (d_weight)
    vocab_rows_kernel<<<(unsigned)((T * (H / 8) + 255) / 256), 256, 0, stream>>>((const bf16_t*)hidden, ldh, labels, rows, T, (int)H, V);
  for (int64_t i = 0; i < q.pieces; i++) {
    const int64_t v0 = i * q.per * VL_SEG, cols = std::min(q.per * VL_SEG, V - v0);
    const bf16_t* w = (const bf16_t*)weight + v0 * ldw;
    GemmParams p = {};
    p.x = (const bf16_t*)hidden; p.ldx = ldh;
    p.w = w; p.ldw = ldw; p.N = (int)cols; p.K = (int)H;
    p.c = dlog; p.ldc = q.ld;
    p.labels = labels; p.lse = lse; p.d_out = d_out; p.scale = scale; p.vocab_base = (int)v0; p.tokens = V;
    int rc = launch_vocab_gemm<EPI_DLOGITS>(p, T, stream);
    if (rc != VX_OK) return rc;
    if (d_hidden) {
      rc = launch_gemm_nn_segments(dlog, q.ld, w, ldw, part, T, H, cols, VL_SEG, stream);
      if (rc != VX_OK) return rc;
      const bool last = i + 1 == q.pieces;
      vocab_dh_kernel<<<(unsigned)((T * H / 4 + 255) / 256), 256, 0, stream>>>(
          part, (int)((cols + VL_SEG - 1) / VL_SEG), T * H, acc, i == 0, last ? (bf16_t*)d_hidden : nullptr, ld_dh, T, (int)H);
    }
    if (d_weight) {
      rc = launch_gemm_tn_rows(dlog, q.ld, rows, H, (bf16_t*)d_weight + v0 * ld_dw, ld_dw, T,
                               (cols + 63) / 64 * 64, cols, H, stream);
      if (rc != VX_OK) return rc;
    }
  }
  return launch_status();
}

}  // extern "C"
