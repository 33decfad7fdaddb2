// Dense products of the vocabulary-sized backward pass, launched from vocab_logprob.hip on the kernels of moe_bwd.hip.
#pragma once
#include "common.h"

namespace vx {

// out[s][m][n] = sum over the columns c of segment s of a[m, c] w[c, n], fp32, s = 0 .. ceil(cols / seg_cols) - 1:
// each segment is one ascending chain of MFMAs. a [M, lda] bf16, zero from column `cols` to the next multiple of 64;
// w [cols, N] bf16, N contiguous and a multiple of 8; seg_cols a multiple of 64.
int launch_gemm_nn_segments(const bf16_t* a, int64_t lda, const bf16_t* w, int64_t ldw, float* out, int64_t M, int64_t N,
                            int64_t cols, int seg_cols, hipStream_t stream);

// dw[n][k] = sum over the rows r of dy[r][n] x[r][k], bf16, one chain per element; dy holds N columns (a multiple of
// 8), of which the first n_store are output rows.
int launch_gemm_tn_rows(const bf16_t* dy, int64_t lddy, const bf16_t* x, int64_t ldx, bf16_t* dw, int64_t lddw, int64_t rows,
                        int64_t N, int64_t n_store, int64_t K, hipStream_t stream);

}  // namespace vx
