// The gated feed-forward block over the rows (pixels, tokens) of a channels-last map, and its gradient.
//
//   g = x Wg^T + bg,  u = x Wu^T + bu,  h = act(g) u,  y = h Wd^T + bd
//   dh = dy Wd;  dg = dh u act'(g);  du = dh act(g)
//   dx = dg Wg + du Wu;  dWg = dg^T x;  dWu = du^T x;  dWd = dy^T h;  the biases' gradients are column sums
//
// Forward: one kernel for both projections, the activation and the product; one for the way down.  Backward: one product
// whose epilogue turns dh into dg, du and h (dh itself is never stored), then dx over the joined reduction [dg du], both
// input weights' gradients as one product over [dg du]^T, and dWd.  h, dg and du are rounded to the block's type between the kernels, as
// the tensor cores take them; every sum is fp32.
#include <type_traits>

#include "fc_gated_ff.h"
#include "fc_last.cuh"

namespace fc {

namespace {

using namespace last;

constexpr int JOIN_THREADS = 256;

// ---- the shares of a split reduction, added in order --------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(JOIN_THREADS) ff_join_kernel(const float *__restrict__ part, const FfProduct p) {
    pdl_wait();
    const int64_t total = (int64_t)p.m * p.n;
    for (int64_t i = (int64_t)blockIdx.x * JOIN_THREADS + threadIdx.x; i < total; i += (int64_t)gridDim.x * JOIN_THREADS) {
        float v = 0.0f;
        for (int s = 0; s < p.splits; ++s) v += part[s * total + i];
        const int64_t m = i / p.n, n = i - m * p.n;
        const bool second = m >= p.row_split;
        T *c = (T *)(second ? p.c1 : p.c0);
        if (c == nullptr) continue;
        if (p.bias0) v += Elem<T>::load(((const T *)p.bias0)[n]);
        c[(second ? m - p.row_split : m) * p.ldc + n] = Elem<T>::store(v);
    }
}

// ---- column sums: the biases' gradients ---------------------------------------------------------------------------
constexpr int SUM_COLS = 32, SUM_ROWS = 8;

// part[chunk][n]: the sum of the chunk's rows
template <typename T>
__global__ void __launch_bounds__(SUM_COLS *SUM_ROWS) ff_colsum_kernel(const T *__restrict__ a, int64_t lda, int rows, int n,
                                                                      int chunk_rows, float *__restrict__ part) {
    __shared__ float s[SUM_ROWS][SUM_COLS];
    pdl_wait();
    const int tx = threadIdx.x % SUM_COLS, ty = threadIdx.x / SUM_COLS;
    const int64_t c = (int64_t)blockIdx.x * SUM_COLS + tx;
    const int64_t r0 = (int64_t)blockIdx.y * chunk_rows, r1 = min((int64_t)rows, r0 + chunk_rows);
    float v = 0.0f;
    if (c < n)
        for (int64_t r = r0 + ty; r < r1; r += SUM_ROWS) v += Elem<T>::load(a[r * lda + c]);
    s[ty][tx] = v;
    __syncthreads();
    if (ty == 0 && c < n) {
#pragma unroll
        for (int i = 1; i < SUM_ROWS; ++i) v += s[i][tx];
        part[(size_t)blockIdx.y * n + c] = v;
    }
}

template <typename T>
__global__ void __launch_bounds__(JOIN_THREADS) ff_colsum_join_kernel(const float *__restrict__ part, int n, int chunks, int split,
                                                                     T *__restrict__ out0, T *__restrict__ out1) {
    pdl_wait();
    const int64_t c = (int64_t)blockIdx.x * JOIN_THREADS + threadIdx.x;
    if (c >= n) return;
    float v = 0.0f;
    for (int i = 0; i < chunks; ++i) v += part[(size_t)i * n + c];
    T *out = c < split ? out0 : out1;
    if (out) out[c < split ? c : c - split] = Elem<T>::store(v);
}

int colsum_chunks(int rows, int n) {
    const long long cols = ceil_div(n, SUM_COLS);
    long long chunks = ceil_div(148 * 8, cols > 0 ? cols : 1);
    const long long most = ceil_div(rows, 4 * SUM_ROWS);
    if (chunks > most) chunks = most;
    return chunks < 1 ? 1 : (int)chunks;
}

// out0[c] (c < split) and out1[c - split] = sums of a's columns; part: colsum_chunks * n floats
int colsum(fc_context *ctx, int type, const void *a, int64_t lda, int rows, int n, int split, void *out0, void *out1, float *part) {
    const int want = colsum_chunks(rows, n);
    const int chunk_rows = rows > 0 ? (int)ceil_div(rows, want) : 1;
    const int chunks = rows > 0 ? (int)ceil_div(rows, chunk_rows) : 0;
    return with_type(type, [&](auto t) -> int {
        using T = decltype(t);
        if (chunks > 0)
            FC_CHECK_CUDA(launch_pdl(ff_colsum_kernel<T>, dim3((unsigned)ceil_div(n, SUM_COLS), chunks), dim3(SUM_COLS * SUM_ROWS), 0,
                                     ctx->stream, (const T *)a, lda, rows, n, chunk_rows, part));
        FC_CHECK_CUDA(launch_pdl(ff_colsum_join_kernel<T>, dim3((unsigned)ceil_div(n, JOIN_THREADS)), dim3(JOIN_THREADS), 0, ctx->stream,
                                 (const float *)part, n, chunks, split, (T *)out0, (T *)out1));
        return FC_OK;
    });
}

// ---- host ---------------------------------------------------------------------------------------------------------

struct Block {
    int rows, in, hidden, out, type, act;
    int64_t xs, ys;
};

int block_of(const fc_gated_ff_desc *d, Block *b) {
    FC_REQUIRE(d != nullptr, FC_ERR_INVALID_ARG, "descriptor is NULL");
    FC_REQUIRE(d->rows >= 0 && d->in_channels > 0 && d->hidden > 0 && d->out_channels > 0, FC_ERR_INVALID_ARG,
               "rows %d, channels in %d, hidden %d, out %d", d->rows, d->in_channels, d->hidden, d->out_channels);
    FC_REQUIRE(d->hidden < (1 << 30), FC_ERR_UNSUPPORTED, "%d hidden channels", d->hidden);
    FC_REQUIRE(dtype_ok(d->type), FC_ERR_INVALID_ARG, "unknown element type %d", d->type);
    FC_REQUIRE(act_ok(d->act), FC_ERR_INVALID_ARG, "unknown activation %d", d->act);
    const int64_t xs = d->x_stride ? d->x_stride : d->in_channels, ys = d->y_stride ? d->y_stride : d->out_channels;
    FC_REQUIRE(xs >= d->in_channels && ys >= d->out_channels, FC_ERR_INVALID_ARG,
               "row strides %lld, %lld are less than the %d, %d channels", (long long)xs, (long long)ys, d->in_channels,
               d->out_channels);
    *b = Block{d->rows, d->in_channels, d->hidden, d->out_channels, d->type, d->act, xs, ys};
    return FC_OK;
}

FfProduct product(const Block &b, int kind, int m, int n, int k, const void *a, int64_t lda, bool a_by_k, const void *b0,
                  int64_t ldb, bool b_by_k, void *c0, int64_t ldc) {
    FfProduct p = {};
    p.type = b.type; p.act = b.act; p.kind = kind;
    p.m = m; p.n = n; p.k = k;
    p.a = a; p.lda = lda; p.a_by_k = a_by_k;
    p.b0 = b0; p.ldb = ldb; p.b_by_k = b_by_k; p.b_split = k;
    p.c0 = c0; p.ldc = ldc; p.row_split = m;
    p.splits = 1;
    return p;
}

// the block's FF_STORE products
FfProduct down_product(const Block &b, const void *h, const void *w_down, const void *bias, void *y) {
    FfProduct p = product(b, FF_STORE, b.rows, b.out, b.hidden, h, b.hidden, true, w_down, b.hidden, true, y, b.ys);
    p.bias0 = bias;
    return p;
}
FfProduct dx_product(const Block &b, const void *dgu, const void *w_gate, const void *w_up, void *dx) {
    FfProduct p = product(b, FF_STORE, b.rows, b.in, 2 * b.hidden, dgu, 2 * (int64_t)b.hidden, true, w_gate, b.in, false, dx, b.xs);
    p.b1 = w_up;
    p.b_split = b.hidden;
    return p;
}
FfProduct dw_in_product(const Block &b, const void *dgu, const void *x, void *dw_gate, void *dw_up) {
    FfProduct p =
        product(b, FF_STORE, 2 * b.hidden, b.in, b.rows, dgu, 2 * (int64_t)b.hidden, false, x, b.xs, false, dw_gate, b.in);
    p.c1 = dw_up;
    p.row_split = b.hidden;
    return p;
}
FfProduct dw_down_product(const Block &b, const void *dy, const void *h, void *dw_down) {
    return product(b, FF_STORE, b.out, b.hidden, b.rows, dy, b.ys, false, h, b.hidden, false, dw_down, b.hidden);
}

struct Work {
    uint8_t *h, *dgu;
    float *part;
    size_t bytes;
};

Work carve(const Block &b, void *base, bool backward) {
    Carver c = {(uint8_t *)base, 0};
    const size_t e = dtype_size(b.type), rh = (size_t)b.rows * b.hidden;
    Work w = {};
    size_t part = 0;
    auto at_least = [&](size_t n) { if (n > part) part = n; };
    auto shares = [&](const FfProduct &p) {  // of either kernel family: which one runs depends on the call's addresses too
        const int s = ff_ffma_splits(p.m, p.n, p.k);
        if (s > 1) at_least((size_t)s * p.m * p.n);
        if (b.type != FC_DTYPE_F32 && p.k > 0) at_least(ff_tc_part_floats(p));
    };
    w.h = c.take<uint8_t>(rh * e);
    if (!backward) {
        shares(down_product(b, nullptr, nullptr, nullptr, nullptr));
    } else {
        w.dgu = c.take<uint8_t>(2 * rh * e);
        shares(dx_product(b, nullptr, nullptr, nullptr, nullptr));
        shares(dw_in_product(b, nullptr, nullptr, nullptr, nullptr));
        shares(dw_down_product(b, nullptr, nullptr, nullptr));
        at_least((size_t)colsum_chunks(b.rows, 2 * b.hidden) * 2 * b.hidden);
        at_least((size_t)colsum_chunks(b.rows, b.out) * b.out);
    }
    w.part = c.take<float>(part);
    w.bytes = c.used;
    return w;
}

int multiply(fc_context *ctx, FfProduct p, float *part) {
    p.part = part;
    if (p.kind != FF_GATE_BACK && ff_few_fits(p)) return launch_ff_few(ctx, p);
    if (ff_tc_fits(p)) return launch_ff_tc(ctx, p);
    if (p.kind == FF_STORE) p.splits = ff_ffma_splits(p.m, p.n, p.k);
    FC_PROPAGATE(launch_ff_ffma(ctx, p));
    if (p.splits == 1) return FC_OK;
    return with_type(p.type, [&](auto t) -> int {
        long long blocks = (long long)ceil_div((size_t)p.m * p.n, JOIN_THREADS);
        if (blocks > 148 * 8) blocks = 148 * 8;
        FC_CHECK_CUDA(launch_pdl(ff_join_kernel<decltype(t)>, dim3((unsigned)blocks), dim3(JOIN_THREADS), 0, ctx->stream,
                                 (const float *)part, p));
        return FC_OK;
    });
}

int check_pointers(const Block &b, std::initializer_list<const void *> needed, std::initializer_list<const void *> optional) {
    for (const void *p : needed) FC_REQUIRE(p != nullptr, FC_ERR_INVALID_ARG, "NULL operand");
    for (const auto &list : {needed, optional})
        for (const void *p : list)
            FC_REQUIRE((uintptr_t)p % dtype_size(b.type) == 0, FC_ERR_INVALID_ARG,
                       "an operand's address is no multiple of its element size");
    return FC_OK;
}

int check_workspace(const void *ws, size_t bytes, size_t need) {
    FC_REQUIRE(need == 0 || (ws != nullptr && aligned16(ws) && bytes >= need), FC_ERR_INVALID_ARG,
               "workspace of %zu bytes at %p: %zu are needed, on a 16-byte boundary", bytes, ws, need);
    return FC_OK;
}

}  // namespace

}  // namespace fc

using namespace fc;

extern "C" {

int fc_gated_ff_workspace(const fc_gated_ff_desc *desc, size_t *forward_bytes, size_t *backward_bytes) {
    Block b;
    FC_PROPAGATE(block_of(desc, &b));
    if (forward_bytes) *forward_bytes = carve(b, nullptr, false).bytes;
    if (backward_bytes) *backward_bytes = carve(b, nullptr, true).bytes;
    return FC_OK;
}

int fc_gated_ff_forward(fc_context *ctx, const fc_gated_ff_desc *desc, const void *d_x, const void *d_w_gate, const void *d_w_up,
                        const void *d_w_down, const void *d_b_gate, const void *d_b_up, const void *d_b_down, void *d_y,
                        float *d_saved, void *d_workspace, size_t workspace_bytes) {
    FC_REQUIRE(ctx != nullptr, FC_ERR_INVALID_ARG, "context is NULL");
    Block b;
    FC_PROPAGATE(block_of(desc, &b));
    if (b.rows == 0) return FC_OK;
    FC_PROPAGATE(check_pointers(b, {d_x, d_w_gate, d_w_up, d_w_down, d_y}, {d_b_gate, d_b_up, d_b_down}));
    FC_REQUIRE((uintptr_t)d_saved % 4 == 0, FC_ERR_INVALID_ARG, "the saved values' address is no multiple of 4");
    const Work w = carve(b, d_workspace, false);
    FC_PROPAGATE(check_workspace(d_workspace, workspace_bytes, w.bytes));
    DeviceScope dev(ctx->device);
    FC_CHECK_CUDA(dev.status());
    FfProduct p = product(b, FF_GATE, b.rows, b.hidden, b.in, d_x, b.xs, true, d_w_gate, b.in, true, w.h, b.hidden);
    p.b1 = d_w_up;
    p.bias0 = d_b_gate;
    p.bias1 = d_b_up;
    p.gate = d_saved;
    p.up = d_saved ? d_saved + (size_t)b.rows * b.hidden : nullptr;
    FC_PROPAGATE(multiply(ctx, p, nullptr));
    return multiply(ctx, down_product(b, w.h, d_w_down, d_b_down, d_y), w.part);
}

int fc_gated_ff_backward(fc_context *ctx, const fc_gated_ff_desc *desc, const void *d_dy, const void *d_x, const void *d_w_gate,
                         const void *d_w_up, const void *d_w_down, const float *d_saved, void *d_dx, void *d_dw_gate,
                         void *d_dw_up, void *d_dw_down, void *d_db_gate, void *d_db_up, void *d_db_down, void *d_workspace,
                         size_t workspace_bytes) {
    FC_REQUIRE(ctx != nullptr, FC_ERR_INVALID_ARG, "context is NULL");
    Block b;
    FC_PROPAGATE(block_of(desc, &b));
    if (b.rows > 0) FC_PROPAGATE(check_pointers(b, {d_dy, d_x, d_w_gate, d_w_up, d_w_down, d_saved}, {}));
    FC_REQUIRE((uintptr_t)d_saved % 4 == 0, FC_ERR_INVALID_ARG, "the saved values' address is no multiple of 4");
    FC_PROPAGATE(check_pointers(b, {}, {d_dx, d_dw_gate, d_dw_up, d_dw_down, d_db_gate, d_db_up, d_db_down}));
    const Work w = carve(b, d_workspace, true);
    FC_PROPAGATE(check_workspace(d_workspace, workspace_bytes, w.bytes));
    DeviceScope dev(ctx->device);
    FC_CHECK_CUDA(dev.status());
    const int64_t two = 2 * (int64_t)b.hidden;
    if (b.rows > 0) {
        FfProduct p = product(b, FF_GATE_BACK, b.rows, b.hidden, b.out, d_dy, b.ys, true, d_w_down, b.hidden, false, w.dgu, two);
        p.gate = const_cast<float *>(d_saved);
        p.up = p.gate + (size_t)b.rows * b.hidden;
        p.c1 = w.h;
        FC_PROPAGATE(multiply(ctx, p, nullptr));
        if (d_dx) FC_PROPAGATE(multiply(ctx, dx_product(b, w.dgu, d_w_gate, d_w_up, d_dx), w.part));
    }
    if (d_dw_gate || d_dw_up) FC_PROPAGATE(multiply(ctx, dw_in_product(b, w.dgu, d_x, d_dw_gate, d_dw_up), w.part));
    if (d_dw_down) FC_PROPAGATE(multiply(ctx, dw_down_product(b, d_dy, w.h, d_dw_down), w.part));
    if (d_db_gate || d_db_up)
        FC_PROPAGATE(colsum(ctx, b.type, w.dgu, two, b.rows, (int)two, b.hidden, d_db_gate, d_db_up, w.part));
    if (d_db_down) FC_PROPAGATE(colsum(ctx, b.type, d_dy, b.ys, b.rows, b.out, b.out, d_db_down, nullptr, w.part));
    return FC_OK;
}

}  // extern "C"
