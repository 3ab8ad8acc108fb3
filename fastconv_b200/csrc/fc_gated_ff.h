// The matrix products of the gated feed-forward block, as its kernel families take them: fc_ff_few.cu for a few rows,
// fc_ff_tc.cu (tensor cores) for everything else.
#pragma once

#include "fc_internal.h"

namespace fc {

enum FfEpilogue {
    FF_STORE = 0,     // C = A B + bias, rounded once; rows below row_split go to c0, the others to c1
    FF_GATE = 1,      // two products at once, with b0 and b1: gate, up; C0 = act(gate + bias0) (up + bias1)
    FF_GATE_BACK = 2  // the product is dh: from the saved gate and up, c0 = dgate, c0 + a_skip = dup, c1 = h
};

// C[m][n] = sum_k A(m, k) B(n, k)
struct FfProduct {
    int type, act, kind;
    int planes;  // 1: A and B are of `type`.  3: sums of three bf16 planes (fp32)
    int m, n, k;
    const void *a;
    int64_t lda;
    bool a_by_k;  // A(m, k) = a[m * lda + k]; else a[k * lda + m]
    int64_t a_skip;  // where A has two parts (b_split < k, row_split < m): the second part's distance from the first
    int64_t a_plane, b_plane, c_plane, c1_plane;  // from one plane to the next
    const void *b0, *b1;
    int64_t ldb;
    bool b_by_k;  // B(n, k) = b[n * ldb + k]; else b[k * ldb + n]
    int b_split;  // !b_by_k: rows k >= b_split come from b1, at k - b_split.  k where there is one matrix
    void *c0, *c1;
    int64_t ldc, ldc1;         // of c0 (and c1, but for FF_GATE_BACK)
    int row_split;             // FF_STORE: m where there is one destination.  A null destination is not computed
    const void *bias0, *bias1; // one value a column, or null
    float *gate, *up;          // what stands before the activation: written by FF_GATE (null: not wanted), read by FF_GATE_BACK
    float *part;               // room for the shares of a split reduction: ff_tc_part_floats
};

// Where the saved value of row m, column n lies in the gate's or the up projection's share of `saved`: [rows][n] in fp32, in
// blocks of 32 rows that are ordered [4 columns][row][column], so that a warp whose lanes are rows moves 16 bytes a lane to
// neighbouring addresses.  The last block has fewer rows; plain rows where n is no multiple of 4.
#ifdef __CUDACC__
__host__ __device__
#endif
inline int64_t ff_saved_at(int64_t m, int64_t n, int64_t rows, int64_t cols) {
    if (cols % 4) return m * cols + n;
    const int64_t block = m / 32 * 32, in_block = rows - block < 32 ? rows - block : 32;
    return block * cols + ((n >> 2) * in_block + (m - block)) * 4 + (n & 3);
}

constexpr int FF_FEW_ROWS = 8;
bool ff_few_fits(const FfProduct &p);  // at most FF_FEW_ROWS; FF_GATE's c0 and FF_STORE's a are fp32
int launch_ff_few(fc_context *ctx, const FfProduct &p);

size_t ff_tc_part_floats(const FfProduct &p);  // what p.part has to hold
fc_ff_product_plan ff_tc_cut(const FfProduct &p);
int launch_ff_tc(fc_context *ctx, const FfProduct &p);

}  // namespace fc
