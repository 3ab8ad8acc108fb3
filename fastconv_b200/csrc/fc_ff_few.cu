// The feed-forward block for a few rows (single tokens, single pixels): up to 8 rows, where reading the weights is all the
// work there is.
//
// A warp has four weight rows and a share of the reduction: per step each lane loads 16 bytes of the four (all in flight at
// once) and of every row of A, which the first-level cache holds after the first warp, and multiplies in fp32 pairs.  Shares
// of a reduction meet in shared memory, lanes by shuffles, both in a fixed order.  For FF_GATE the four are two rows of the
// gate's weights and the same two of the up projection's.  h stays in fp32 whatever the type: no tensor core asks for less, and
// it is a few KB beside the weights.  One row 1024->4096->1024 in bf16, 25 MB of weights: 6.8 to 7.1 us
// for both launches, 3.6 TB/s (6.3 us replayed from a graph), where tensor-core tiles of 256 rows took 23.7; 8 rows are where the
// multiplications begin to show beside the loads.
#include <type_traits>

#include "fc_gated_ff.h"
#include "fc_last.cuh"

namespace fc {

namespace {

using namespace last;

constexpr int FEW_THREADS = 256, FEW_WARPS = FEW_THREADS / 32, NW = 4;  // weight rows of a warp

template <typename T, int R, int KIND>
__global__ void __launch_bounds__(FEW_THREADS) ff_few_kernel(const FfProduct p, int log_shares) {
    constexpr int VEC = 16 / sizeof(T), STEP = KIND == FF_GATE ? NW / 2 : NW;  // columns of a warp
    __shared__ float meet[FEW_WARPS][R * NW];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int shares = 1 << log_shares, share = warp & (shares - 1);
    const long long n0 = ((long long)blockIdx.x * (FEW_WARPS >> log_shares) + (warp >> log_shares)) * STEP;
    pdl_wait();
    pdl_next();
    const T *w[NW];
#pragma unroll
    for (int j = 0; j < NW; ++j) {
        const long long n = min(n0 + j % STEP, (long long)p.n - 1);  // past the end: a row that is read and not used
        w[j] = (const T *)(j < STEP ? p.b0 : p.b1) + n * p.ldb;
    }
    Pair acc[R][NW];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int j = 0; j < NW; ++j) acc[r][j] = 0;
    using A = std::conditional_t<KIND == FF_GATE, T, float>;  // x; h
    const A *a = (const A *)p.a;
    const int vectors = p.k / VEC, hop = 32 << log_shares;
#pragma unroll(R > 2 ? 1 : 2)
    for (int i = (share << 5) + lane; i < vectors; i += hop) {
        constexpr int AN = 16 / sizeof(A);  // a vector of T is one or two of A
        Vec<T, VEC> bv[NW];
        Vec<A, AN> av[R][VEC / AN];
#pragma unroll
        for (int j = 0; j < NW; ++j) bv[j] = Vec<T, VEC>::load(w[j] + (size_t)i * VEC);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int h = 0; h < VEC / AN; ++h)
                av[r][h] = Vec<A, AN>::load(a + (r < p.m ? r : 0) * p.lda + (size_t)i * VEC + h * AN);
        Pair b[NW][VEC / 2];
#pragma unroll
        for (int j = 0; j < NW; ++j) unpack_pairs(bv[j], b[j]);
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int h = 0; h < VEC / AN; ++h) {
                Pair c[AN / 2];
                unpack_pairs(av[r][h], c);
#pragma unroll
                for (int j = 0; j < NW; ++j)
#pragma unroll
                    for (int e = 0; e < AN / 2; ++e) acc[r][j] = fma2(c[e], b[j][h * AN / 2 + e], acc[r][j]);
            }
        }
    }
    float mine = 0.0f;  // lane r * NW + j (R * NW <= 32) ends up with that sum
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int j = 0; j < NW; ++j) {
            const float2 h = split(acc[r][j]);
            float v = h.x + h.y;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
            if (lane == r * NW + j) mine = v;
        }
    if (shares > 1) {
        if (lane < R * NW) meet[warp][lane] = mine;
        __syncthreads();
        if (share > 0) return;
        if (lane < R * NW)
            for (int i = 1; i < shares; ++i) mine += meet[warp + i][lane];
    }
    const int r = lane / NW, j = lane % NW;
    if (KIND == FF_GATE) {
        const float up = __shfl_down_sync(0xffffffffu, mine, STEP);
        const long long n = n0 + j;
        if (lane >= R * NW || r >= p.m || j >= STEP || n >= p.n) return;
        float g = mine, u = up, act, slope;
        if (p.bias0) g += Elem<T>::load(((const T *)p.bias0)[n]);
        if (p.bias1) u += Elem<T>::load(((const T *)p.bias1)[n]);
        act_both_rt(p.act, g, act, slope);
        ((float *)p.c0)[r * p.ldc + n] = act * u;
        if (p.gate) {
            const int64_t at = ff_saved_at(r, n, p.m, p.n);
            p.gate[at] = g;
            p.up[at] = u;
        }
    } else {
        const long long n = n0 + j;
        if (lane >= R * NW || r >= p.m || n >= p.n) return;
        if (p.bias0) mine += Elem<T>::load(((const T *)p.bias0)[n]);
        ((T *)p.c0)[r * p.ldc + n] = Elem<T>::store(mine);
    }
}

}  // namespace

// rows of whole, aligned 16-byte vectors along the reduction
bool ff_few_fits(const FfProduct &p) {
    const int vec = 16 / (int)dtype_size(p.type);
    if (p.m < 1 || p.m > FF_FEW_ROWS || !p.a_by_k || !p.b_by_k || p.b_split < p.k || p.row_split < p.m) return false;
    if (p.k % vec || p.lda % vec || p.ldb % vec) return false;
    return aligned16(p.a) && aligned16(p.b0) && aligned16(p.b1);
}

int launch_ff_few(fc_context *ctx, const FfProduct &p) {
    // shares of the reduction: about 24 warps to an SM, but no share of less than two steps
    const int step = p.kind == FF_GATE ? NW / 2 : NW, vec = 16 / (int)dtype_size(p.type);
    const long long warps = ceil_div(p.n, step);
    int log_shares = 0;
    while (log_shares < 3 && (warps << log_shares) < 148 * 24 && p.k / vec >= (128 << log_shares)) ++log_shares;
    const long long blocks = ceil_div(warps << log_shares, FEW_WARPS);
    FC_REQUIRE(blocks < (1ll << 31), FC_ERR_UNSUPPORTED, "product of %lld blocks", blocks);
    return with_type(p.type, [&](auto t) -> int {
        using T = decltype(t);
        auto go = [&](auto kernel) -> int {
            FC_CHECK_CUDA(launch_early(kernel, dim3((unsigned)blocks), dim3(FEW_THREADS), 0, ctx, p, log_shares));
            return FC_OK;
        };
        if (p.kind == FF_GATE)
            return p.m == 1 ? go(ff_few_kernel<T, 1, FF_GATE>) : p.m == 2 ? go(ff_few_kernel<T, 2, FF_GATE>)
                 : p.m <= 4 ? go(ff_few_kernel<T, 4, FF_GATE>) : go(ff_few_kernel<T, 8, FF_GATE>);
        return p.m == 1 ? go(ff_few_kernel<T, 1, FF_STORE>) : p.m == 2 ? go(ff_few_kernel<T, 2, FF_STORE>)
             : p.m <= 4 ? go(ff_few_kernel<T, 4, FF_STORE>) : go(ff_few_kernel<T, 8, FF_STORE>);
    });
}

}  // namespace fc
