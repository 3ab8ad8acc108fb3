// The gated feed-forward block over the rows (pixels, tokens) of a channels-last map, and its gradient.
//
//   g = x Wg^T + bg,  u = x Wu^T + bu,  h = act(g) u,  y = h Wd^T + bd
//   dh = dy Wd;  dg = dh u act'(g);  du = dh act(g)
//   dx = dg Wg + du Wu;  dWg = dg^T x;  dWu = du^T x;  dWd = dy^T h;  the biases' gradients are column sums
//
// Forward: one kernel for both projections, the activation and the product; one for the way down.  Backward: one product
// whose epilogue turns dh into dg, du and h (dh itself is never stored), then dx over the joined reduction [dg du], both
// input weights' gradients as one product over [dg du]^T, and dWd.  h, dg and du are rounded to the block's type between
// the kernels, as the tensor cores take them (fp32: three bf16 parts that hold all its bits); every sum is fp32, and so are the
// saved g and u: rounding them would add a second rounding to dg, du and h.
#include <type_traits>

#include "fc_gated_ff.h"
#include "fc_last.cuh"

namespace fc {

namespace {

using namespace last;

// ---- operands that the tensor cores' copies cannot take as they lie ------------------------------------------------
// fp32, which is split into three bf16 planes, and rows that are no multiples of 16 bytes.  One launch for all of a call's.
struct PackItem {
    const void *src;
    int64_t ld;
    int rows, cols, wide;  // wide: the source can be read in 16-byte vectors
    uint16_t *dst;
    int64_t ldp, plane;
    long long end;  // vectors of 8 of this item and those before it
};
struct PackList {
    PackItem item[5];
    int count;
};

template <typename T>
__global__ void __launch_bounds__(256) ff_pack_kernel(const PackList list) {
    constexpr int VEC = 16 / sizeof(T), PLANES = sizeof(T) == 4 ? 3 : 1;
    pdl_wait();
    pdl_next();
    const long long total = list.item[list.count - 1].end;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        int k = 0;
        while (i >= list.item[k].end) ++k;
        const PackItem &p = list.item[k];
        const long long at = i - (k ? list.item[k - 1].end : 0);
        const int per_row = (int)(p.ldp >> 3);
        const long long row = at / per_row;
        const int c = (int)(at - row * per_row) * 8;
        const T *src = (const T *)p.src + row * p.ld + c;
        float v[8];
        if (p.wide && c + 8 <= p.cols) {
#pragma unroll
            for (int j = 0; j < 8; j += VEC) {
                float f[VEC];
                Vec<T, VEC>::load(src + j).unpack(f);
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[j + e] = f[e];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = c + j < p.cols ? Elem<T>::load(src[j]) : 0.0f;
        }
        uint16_t *dst = p.dst + row * p.ldp + c;
        if constexpr (PLANES == 1) {
            Vec<T, 8> out;
            out.pack(v);
            out.store(dst);
        } else {
#pragma unroll
            for (int z = 0; z < 3; ++z) {
                Vec<__nv_bfloat16, 8> out;
                float part[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    part[j] = z < 2 ? bf16_part(v[j]) : v[j];
                    v[j] = fabsf(part[j]) <= 3.4028234e38f ? v[j] - part[j] : 0.0f;
                }
                out.pack(part);
                out.store(dst + z * p.plane);
            }
        }
    }
}

// ---- column sums: the biases' gradients ---------------------------------------------------------------------------
// One launch for the three of a call where a block can add up all rows of its 32 columns; with more rows shares of them, and a
// second launch that adds the shares in order.
constexpr int SUM_COLS = 32, SUM_ROWS = 32;

struct SumItem {
    const void *a;
    int64_t lda, plane;  // plane > 0: the sum of three bf16 planes
    int n, first;        // columns; the item's first block of columns
    float *part;         // [chunks][n]
    void *out;
};
struct SumList {
    SumItem item[3];
    int count, blocks, rows, chunks, chunk_rows;
};

template <typename T>
__global__ void __launch_bounds__(SUM_COLS *SUM_ROWS) ff_colsum_kernel(const SumList list) {
    __shared__ float s[SUM_ROWS][SUM_COLS + 1];
    pdl_wait();
    pdl_next();
    int k = 0;
    while (k + 1 < list.count && (int)blockIdx.x >= list.item[k + 1].first) ++k;
    const SumItem &p = list.item[k];
    const int tx = threadIdx.x % SUM_COLS, ty = threadIdx.x / SUM_COLS;
    const int64_t c = (int64_t)(blockIdx.x - p.first) * SUM_COLS + tx;
    const int64_t r0 = (int64_t)blockIdx.y * list.chunk_rows, r1 = min((int64_t)list.rows, r0 + list.chunk_rows);
    float v = 0.0f;
    if (c < p.n) {
        if (p.plane > 0) {
            const __nv_bfloat16 *a = (const __nv_bfloat16 *)p.a + c;
#pragma unroll 4
            for (int64_t r = r0 + ty; r < r1; r += SUM_ROWS)
                v += __bfloat162float(a[r * p.lda]) + __bfloat162float(a[p.plane + r * p.lda]) +
                     __bfloat162float(a[2 * p.plane + r * p.lda]);
        } else {
            const T *a = (const T *)p.a + c;
#pragma unroll 8
            for (int64_t r = r0 + ty; r < r1; r += SUM_ROWS) v += Elem<T>::load(a[r * p.lda]);
        }
    }
    s[ty][tx] = v;
    __syncthreads();
    v = s[tx][ty];  // the sums of column ty, one to a lane
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    const int64_t col = (int64_t)(blockIdx.x - p.first) * SUM_COLS + ty;
    if (tx > 0 || col >= p.n) return;
    if (list.chunks > 1)
        p.part[(size_t)blockIdx.y * p.n + col] = v;
    else
        ((T *)p.out)[col] = Elem<T>::store(v);
}

template <typename T>
__global__ void __launch_bounds__(SUM_COLS) ff_colsum_join_kernel(const SumList list) {
    pdl_wait();
    pdl_next();
    int k = 0;
    while (k + 1 < list.count && (int)blockIdx.x >= list.item[k + 1].first) ++k;
    const SumItem &p = list.item[k];
    const int64_t c = (int64_t)(blockIdx.x - p.first) * SUM_COLS + threadIdx.x;
    if (c >= p.n) return;
    float v = 0.0f;
#pragma unroll 8
    for (int i = 0; i < list.chunks; ++i) v += p.part[(size_t)i * p.n + c];
    ((T *)p.out)[c] = Elem<T>::store(v);
}

// shares of the rows: one up to 2048 of them, else enough that blocks reach every SM: of at most 512 rows, but no more than 64
int colsum_chunks(int rows) {
    if (rows <= 2048) return 1;
    const long long c = ceil_div(rows, 512);
    return c > 64 ? 64 : (int)c;
}

struct Sums {
    SumList list;
    void add(const void *a, int64_t lda, int64_t plane, int n, void *out, float *part) {
        if (out == nullptr) return;
        list.item[list.count++] = SumItem{a, lda, plane, n, list.blocks, part, out};
        list.blocks += (int)ceil_div(n, SUM_COLS);
    }
    int run(fc_context *ctx, int type, int rows) {
        if (list.count == 0) return FC_OK;
        list.rows = rows;
        list.chunk_rows = (int)ceil_div(rows, colsum_chunks(rows));
        list.chunks = (int)ceil_div(rows, list.chunk_rows);
        return with_type(type, [&](auto t) -> int {
            using T = decltype(t);
            FC_CHECK_CUDA(launch_early(ff_colsum_kernel<T>, dim3(list.blocks, list.chunks), dim3(SUM_COLS * SUM_ROWS), 0, ctx, list));
            if (list.chunks > 1)
                FC_CHECK_CUDA(launch_early(ff_colsum_join_kernel<T>, dim3(list.blocks), dim3(SUM_COLS), 0, ctx, list));
            return FC_OK;
        });
    }
};

// ---- host ---------------------------------------------------------------------------------------------------------

struct Block {
    int rows, in, hidden, out, type, act;
    int64_t xs, ys;
};

int block_of(const fc_gated_ff_desc *d, Block *b) {
    FC_REQUIRE(d != nullptr, FC_ERR_INVALID_ARG, "descriptor is NULL");
    FC_REQUIRE(d->rows >= 0 && d->in_channels > 0 && d->hidden > 0 && d->out_channels > 0, FC_ERR_INVALID_ARG,
               "rows %d, channels in %d, hidden %d, out %d", d->rows, d->in_channels, d->hidden, d->out_channels);
    FC_REQUIRE(d->in_channels < (1 << 30) && d->hidden < (1 << 30) && d->out_channels < (1 << 30), FC_ERR_UNSUPPORTED,
               "channels in %d, hidden %d, out %d", d->in_channels, d->hidden, d->out_channels);
    FC_REQUIRE(dtype_ok(d->type), FC_ERR_INVALID_ARG, "unknown element type %d", d->type);
    FC_REQUIRE(act_ok(d->act), FC_ERR_INVALID_ARG, "unknown activation %d", d->act);
    const int64_t xs = d->x_stride ? d->x_stride : d->in_channels, ys = d->y_stride ? d->y_stride : d->out_channels;
    FC_REQUIRE(xs >= d->in_channels && ys >= d->out_channels, FC_ERR_INVALID_ARG,
               "row strides %lld, %lld are less than the %d, %d channels", (long long)xs, (long long)ys, d->in_channels,
               d->out_channels);
    *b = Block{d->rows, d->in_channels, d->hidden, d->out_channels, d->type, d->act, xs, ys};
    return FC_OK;
}

// A matrix as a product reads it: 16-bit values in rows of a multiple of 8, one plane or three.
struct Matrix {
    const void *p;
    int64_t ld, plane;
};

FfProduct product(const Block &b, int kind, int m, int n, int k, const Matrix &a, bool a_by_k, const Matrix &b0, bool b_by_k) {
    FfProduct p = {};
    p.type = b.type; p.act = b.act; p.kind = kind;
    p.planes = b.type == FC_DTYPE_F32 ? 3 : 1;
    p.m = m; p.n = n; p.k = k;
    p.a = a.p; p.lda = a.ld; p.a_plane = a.plane; p.a_by_k = a_by_k;
    p.b0 = b0.p; p.ldb = b0.ld; p.b_plane = b0.plane; p.b_by_k = b_by_k;
    p.b_split = k;
    p.row_split = m;
    return p;
}

// the block's products, but for what only a call knows
FfProduct gate_product(const Block &b, const Matrix &x, const Matrix &w_gate, const void *w_up) {
    FfProduct p = product(b, FF_GATE, b.rows, b.hidden, b.in, x, true, w_gate, true);
    p.b1 = w_up;
    return p;
}
FfProduct back_gate_product(const Block &b, const Matrix &dy, const Matrix &w_down) {
    return product(b, FF_GATE_BACK, b.rows, b.hidden, b.out, dy, true, w_down, false);
}
FfProduct down_product(const Block &b, const Matrix &h, const Matrix &w_down, const void *bias, void *y) {
    FfProduct p = product(b, FF_STORE, b.rows, b.out, b.hidden, h, true, w_down, true);
    p.bias0 = bias;
    p.c0 = y; p.ldc = b.ys;
    return p;
}
FfProduct dx_product(const Block &b, const Matrix &dgu, const Matrix &w_gate, const void *w_up, void *dx) {
    FfProduct p = product(b, FF_STORE, b.rows, b.in, 2 * b.hidden, dgu, true, w_gate, false);
    p.a_skip = dgu.ld / 2;
    p.b1 = w_up;
    p.b_split = b.hidden;
    p.c0 = dx; p.ldc = b.xs;
    return p;
}
FfProduct dw_in_product(const Block &b, const Matrix &dgu, const Matrix &x, void *dw_gate, void *dw_up) {
    FfProduct p = product(b, FF_STORE, 2 * b.hidden, b.in, b.rows, dgu, false, x, false);
    p.a_skip = dgu.ld / 2;
    p.row_split = b.hidden;
    p.c0 = dw_gate; p.c1 = dw_up; p.ldc = b.in;
    return p;
}
FfProduct dw_down_product(const Block &b, const Matrix &dy, const Matrix &h, void *dw_down) {
    FfProduct p = product(b, FF_STORE, b.out, b.hidden, b.rows, dy, false, h, false);
    p.c0 = dw_down; p.ldc = b.hidden;
    return p;
}

// The workspace: h, [dg du], packed copies of the operands (whether they are needed depends on the call's addresses too), and
// the shares of split reductions and column sums.
struct Work {
    Matrix h, dgu, x, dy, w_gate, w_up, w_down;
    float *part;
    size_t bytes;
};

Work carve(const Block &b, void *base, bool backward) {
    Carver c = {(uint8_t *)base, 0};
    const int planes = b.type == FC_DTYPE_F32 ? 3 : 1;
    auto matrix = [&](int64_t rows, int64_t ld) {
        const int64_t plane = rows * ld;
        return Matrix{c.take<uint16_t>((size_t)plane * planes), ld, plane};
    };
    const int64_t in = round_up(b.in, 8), hidden = round_up(b.hidden, 8), out = round_up(b.out, 8);
    Work w = {};
    size_t part = 0;
    auto at_least = [&](size_t n) { if (n > part) part = n; };
    w.h = matrix(b.rows, hidden);
    if (!backward && b.rows <= FF_FEW_ROWS) c.take<float>((size_t)b.rows * hidden);  // h is fp32 there, and begins where w.h does
    w.x = matrix(b.rows, in);
    w.w_gate = matrix(b.hidden, in);
    w.w_up = matrix(b.hidden, in);
    w.w_down = matrix(b.out, hidden);
    if (!backward) {
        at_least(ff_tc_part_floats(down_product(b, w.h, w.w_down, nullptr, nullptr)));
    } else {
        w.dy = matrix(b.rows, out);
        w.dgu = matrix(b.rows, 2 * hidden);
        at_least(ff_tc_part_floats(dx_product(b, w.dgu, w.w_gate, nullptr, nullptr)));
        at_least(ff_tc_part_floats(dw_in_product(b, w.dgu, w.x, nullptr, nullptr)));
        at_least(ff_tc_part_floats(dw_down_product(b, w.dy, w.h, nullptr)));
        at_least((size_t)colsum_chunks(b.rows) * (2 * (size_t)b.hidden + b.out));
    }
    w.part = c.take<float>(part);
    w.bytes = c.used;
    return w;
}

// The operands of one call: as they lie where the copies can take them so, else packed.
struct Packer {
    const Block &b;
    PackList list;
    long long total;
    explicit Packer(const Block &block) : b(block), list(), total(0) {}
    static bool lies_well(const Block &b, const void *p, int64_t ld) { return b.type != FC_DTYPE_F32 && ld % 8 == 0 && aligned16(p); }
    Matrix use(const void *p, int64_t ld, int rows, int cols, const Matrix &room, bool as_it_lies) {
        if (as_it_lies) return Matrix{p, ld, 0};
        const int vec = 16 / (int)dtype_size(b.type);
        total += rows * (room.ld / 8);
        list.item[list.count++] = PackItem{p, ld, rows, cols, ld % vec == 0 && aligned16(p), (uint16_t *)room.p, room.ld, room.plane, total};
        return room;
    }
    Matrix use(const void *p, int64_t ld, int rows, int cols, const Matrix &room) {
        return use(p, ld, rows, cols, room, lies_well(b, p, ld));
    }
    int run(fc_context *ctx) {
        if (list.count == 0) return FC_OK;
        return with_type(b.type, [&](auto t) -> int {
            long long blocks = ceil_div((size_t)total, 256);
            if (blocks > 148 * 16) blocks = 148 * 16;
            FC_CHECK_CUDA(launch_early(ff_pack_kernel<decltype(t)>, dim3((unsigned)blocks), dim3(256), 0, ctx, list));
            return FC_OK;
        });
    }
};

int multiply(fc_context *ctx, FfProduct p, float *part) {
    p.part = part;
    return launch_ff_tc(ctx, p);
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

int fc_gated_ff_plan(const fc_gated_ff_desc *desc, int product, fc_ff_product_plan *plan) {
    Block b;
    FC_PROPAGATE(block_of(desc, &b));
    FC_REQUIRE(plan != nullptr, FC_ERR_INVALID_ARG, "plan is NULL");
    FC_REQUIRE(b.rows > 0, FC_ERR_INVALID_ARG, "a block of no rows has no products");
    const Matrix none = {};
    switch (product) {
        case FC_FF_GATE: *plan = ff_tc_cut(gate_product(b, none, none, nullptr)); return FC_OK;
        case FC_FF_DOWN: *plan = ff_tc_cut(down_product(b, none, none, nullptr, nullptr)); return FC_OK;
        case FC_FF_BACK_GATE: *plan = ff_tc_cut(back_gate_product(b, none, none)); return FC_OK;
        case FC_FF_DX: *plan = ff_tc_cut(dx_product(b, none, none, nullptr, nullptr)); return FC_OK;
        case FC_FF_DW_IN: *plan = ff_tc_cut(dw_in_product(b, none, none, nullptr, nullptr)); return FC_OK;
        case FC_FF_DW_DOWN: *plan = ff_tc_cut(dw_down_product(b, none, none, nullptr)); return FC_OK;
    }
    FC_REQUIRE(false, FC_ERR_INVALID_ARG, "unknown product %d", product);
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
    FC_PROPAGATE(check_outputs({d_y, d_saved, d_workspace}, {d_x, d_w_gate, d_w_up, d_w_down, d_b_gate, d_b_up, d_b_down}));
    const Work w = carve(b, d_workspace, false);
    FC_PROPAGATE(check_workspace(d_workspace, workspace_bytes, w.bytes));
    DeviceScope dev(ctx->device);
    FC_CHECK_CUDA(dev.status());
    float *up = d_saved ? d_saved + (size_t)b.rows * b.hidden : nullptr;
    const Matrix x0 = {d_x, b.xs, 0}, wg0 = {d_w_gate, b.in, 0}, wd0 = {d_w_down, b.hidden, 0};
    auto gate = [&](const Matrix &x, const Matrix &w_gate, const void *w_up) {
        FfProduct p = gate_product(b, x, w_gate, w_up);
        p.bias0 = d_b_gate;
        p.bias1 = d_b_up;
        p.gate = d_saved;
        p.up = up;
        p.c0 = const_cast<void *>(w.h.p); p.ldc = w.h.ld; p.c_plane = w.h.plane;
        return p;
    };
    {
        const FfProduct first = gate(x0, wg0, d_w_up), second = down_product(b, w.h, wd0, d_b_down, d_y);
        if (ff_few_fits(first) && ff_few_fits(second)) {
            FC_PROPAGATE(launch_ff_few(ctx, first));
            return launch_ff_few(ctx, second);
        }
    }
    Packer pack(b);
    const bool w_in = Packer::lies_well(b, d_w_gate, b.in) && Packer::lies_well(b, d_w_up, b.in);
    const Matrix x = pack.use(d_x, b.xs, b.rows, b.in, w.x), w_gate = pack.use(d_w_gate, b.in, b.hidden, b.in, w.w_gate, w_in),
                 w_up = pack.use(d_w_up, b.in, b.hidden, b.in, w.w_up, w_in),
                 w_down = pack.use(d_w_down, b.hidden, b.out, b.hidden, w.w_down);
    FC_PROPAGATE(pack.run(ctx));
    FC_PROPAGATE(multiply(ctx, gate(x, w_gate, w_up.p), nullptr));
    return multiply(ctx, down_product(b, w.h, w_down, d_b_down, d_y), w.part);
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
    FC_PROPAGATE(check_outputs({d_dx, d_dw_gate, d_dw_up, d_dw_down, d_db_gate, d_db_up, d_db_down, d_workspace},
                               {d_dy, d_x, d_w_gate, d_w_up, d_w_down, d_saved}));
    const Work w = carve(b, d_workspace, true);
    FC_PROPAGATE(check_workspace(d_workspace, workspace_bytes, w.bytes));
    DeviceScope dev(ctx->device);
    FC_CHECK_CUDA(dev.status());
    const size_t e = dtype_size(b.type);
    if (b.rows == 0) {  // sums of nothing
        const struct { void *p; size_t n; } grads[] = {{d_dw_gate, (size_t)b.hidden * b.in}, {d_dw_up, (size_t)b.hidden * b.in},
                                                       {d_dw_down, (size_t)b.out * b.hidden}, {d_db_gate, (size_t)b.hidden},
                                                       {d_db_up, (size_t)b.hidden}, {d_db_down, (size_t)b.out}};
        for (const auto &g : grads)
            if (g.p) FC_CHECK_CUDA(cudaMemsetAsync(g.p, 0, g.n * e, ctx->stream));
        return FC_OK;
    }
    Packer pack(b);
    const bool w_in = Packer::lies_well(b, d_w_gate, b.in) && Packer::lies_well(b, d_w_up, b.in);
    const Matrix dy = pack.use(d_dy, b.ys, b.rows, b.out, w.dy), w_down = pack.use(d_w_down, b.hidden, b.out, b.hidden, w.w_down);
    Matrix x = {}, w_gate = {}, w_up = {};
    if (d_dw_gate || d_dw_up) x = pack.use(d_x, b.xs, b.rows, b.in, w.x);
    if (d_dx) {
        w_gate = pack.use(d_w_gate, b.in, b.hidden, b.in, w.w_gate, w_in);
        w_up = pack.use(d_w_up, b.in, b.hidden, b.in, w.w_up, w_in);
    }
    FC_PROPAGATE(pack.run(ctx));

    FfProduct p = back_gate_product(b, dy, w_down);
    p.gate = const_cast<float *>(d_saved);
    p.up = p.gate + (size_t)b.rows * b.hidden;
    p.a_skip = w.dgu.ld / 2;
    p.c0 = const_cast<void *>(w.dgu.p); p.ldc = w.dgu.ld; p.c_plane = w.dgu.plane;
    p.c1 = const_cast<void *>(w.h.p); p.ldc1 = w.h.ld; p.c1_plane = w.h.plane;
    FC_PROPAGATE(multiply(ctx, p, nullptr));
    if (d_dx) FC_PROPAGATE(multiply(ctx, dx_product(b, w.dgu, w_gate, w_up.p, d_dx), w.part));
    if (d_dw_gate || d_dw_up) FC_PROPAGATE(multiply(ctx, dw_in_product(b, w.dgu, x, d_dw_gate, d_dw_up), w.part));
    if (d_dw_down) FC_PROPAGATE(multiply(ctx, dw_down_product(b, dy, w.h, d_dw_down), w.part));

    const int64_t plane = b.type == FC_DTYPE_F32 ? w.dgu.plane : 0;
    const uint8_t *dgu = (const uint8_t *)w.dgu.p;
    const size_t chunks = colsum_chunks(b.rows);
    Sums sums = {};
    sums.add(dgu, w.dgu.ld, plane, b.hidden, d_db_gate, w.part);
    sums.add(dgu + w.dgu.ld, w.dgu.ld, plane, b.hidden, d_db_up, w.part + chunks * b.hidden);
    sums.add(d_dy, b.ys, 0, b.out, d_db_down, w.part + 2 * chunks * b.hidden);
    FC_PROPAGATE(sums.run(ctx, b.type, b.rows));
    return FC_OK;
}

}  // extern "C"
