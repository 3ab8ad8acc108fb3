// The matrix products of the gated feed-forward block, as its two kernel families take them (fc_ff_ffma.cu for fp32 and
// for what the tensor cores' copies cannot address, fc_ff_tc.cu for bf16 and fp16).
#pragma once

#include "fc_internal.h"

namespace fc {

enum FfEpilogue {
    FF_STORE = 0,     // C = A B + bias, rounded once; rows below row_split go to c0, the others to c1
    FF_GATE = 1,      // two products at once, with b0 and b1: gate, up; C0 = act(gate + bias0) (up + bias1)
    FF_GATE_BACK = 2  // the product is dh: from the saved gate and up, C0[m][0..n) = dgate, C0[m][n..2n) = dup, C1 = h
};

// C[m][n] = sum_k A(m, k) B(n, k)
struct FfProduct {
    int type, act, kind;
    int m, n, k;
    const void *a;
    int64_t lda;
    bool a_by_k;  // A(m, k) = a[m * lda + k]; else a[k * lda + m]
    const void *b0, *b1;
    int64_t ldb;
    bool b_by_k;  // B(n, k) = b[n * ldb + k]; else b[k * ldb + n]
    int b_split;  // !b_by_k: rows k >= b_split come from b1, at k - b_split.  k where there is one matrix
    void *c0, *c1;
    int64_t ldc;
    int row_split;             // FF_STORE: m where there is one destination.  A null destination is not stored to
    const void *bias0, *bias1; // one value a column, or null
    const void *gate_in, *up_in;  // FF_GATE_BACK: [m][n]
    void *gate_out, *up_out;      // FF_GATE: [m][n], or null
    float *part;               // FF_STORE with splits > 1: [splits][m][n]
    int splits;
};

int launch_ff_ffma(fc_context *ctx, const FfProduct &p);
// shares of the reduction for an FF_STORE product, so that few output tiles still occupy the GPU
int ff_ffma_splits(int m, int n, int k);

}  // namespace fc
