// The feed-forward block's matrix products on the FP32 pipe: every type, size, stride and alignment.  One fused
// multiply-add per term and an fp32 accumulator per output element, so fp32 results have fp32's own error; bf16 and fp16
// come here only where a row is no multiple of 16 bytes, which the tensor cores' copies need.
//
// A block computes 128 x 128 outputs with 256 threads of 8 x 8 each (two 4-wide pieces along both axes, so that a warp's
// 128-bit reads of shared memory are conflict-free), 16 reduction steps to a slab, the next slab on its way from memory in
// registers while this one is multiplied.  FMAs go out in pairs (fma.rn.f32x2).  For FF_GATE the 128 columns are 64 of the
// gate and the same 64 of the up projection, so one thread holds both values that its product needs.
#include <type_traits>

#include "fc_gated_ff.h"
#include "fc_last.cuh"

namespace fc {

namespace {

using namespace last;

constexpr int BM = 128, BN = 128, BK = 16, FF_THREADS = 256, PAD = 4;

// eight neighbouring elements of a row from `at` on, zero from `end` on
template <typename T>
__device__ __forceinline__ void load8(const T *row, int64_t at, int64_t end, bool wide, float (&f)[8]) {
    constexpr int VEC = 16 / sizeof(T);
    if (wide && at + 8 <= end) {
#pragma unroll
        for (int i = 0; i < 8; i += VEC) {
            float g[VEC];
            Vec<T, VEC>::load(row + at + i).unpack(g);
#pragma unroll
            for (int j = 0; j < VEC; ++j) f[i + j] = g[j];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = at + i < end ? Elem<T>::load(row[at + i]) : 0.0f;
    }
}

template <typename T, bool A_BY_K, bool B_BY_K, int KIND>
__global__ void __launch_bounds__(FF_THREADS, 2) ff_ffma_kernel(const FfProduct p, int n_tiles, int m_tiles, int k_share, bool a_wide,
                                                               bool b_wide) {
    __shared__ __align__(16) float As[2][BK][BM + PAD], Bs[2][BK][BN + PAD];
    pdl_wait();
    const int tid = threadIdx.x;
    const long long id = blockIdx.x;
    const int nt = (int)(id % n_tiles);
    const long long rest = id / n_tiles;
    const int mt = (int)(rest % m_tiles), part = (int)(rest / m_tiles);
    constexpr int N_STEP = KIND == FF_GATE ? BN / 2 : BN;  // output columns of a tile
    const int64_t m0 = (int64_t)mt * BM, n0 = (int64_t)nt * N_STEP;
    const int64_t k_begin = (int64_t)part * k_share, k_end = min((int64_t)p.k, k_begin + k_share);
    const T *a = (const T *)p.a, *b0 = (const T *)p.b0, *b1 = (const T *)p.b1;

    float ra[8], rb[8];
    auto fetch = [&](int64_t k0) {
        if (A_BY_K) {
            const int64_t m = m0 + (tid & 127);
            load8<T>(a + m * p.lda, k0 + (tid >> 7) * 8, m < p.m ? k_end : 0, a_wide, ra);
        } else {
            const int64_t k = k0 + (tid >> 4);
            load8<T>(a + k * p.lda, m0 + (tid & 15) * 8, k < k_end ? p.m : 0, a_wide, ra);
        }
        if (B_BY_K) {
            const int r = tid & 127;
            const bool second = KIND == FF_GATE && r >= N_STEP;
            const int64_t n = n0 + (second ? r - N_STEP : r);
            load8<T>((second ? b1 : b0) + n * p.ldb, k0 + (tid >> 7) * 8, n < p.n ? k_end : 0, b_wide, rb);
        } else {
            const int64_t k = k0 + (tid >> 4);
            const T *row = k < p.b_split ? b0 + k * p.ldb : b1 + (k - p.b_split) * p.ldb;
            load8<T>(row, n0 + (tid & 15) * 8, k < k_end ? p.n : 0, b_wide, rb);
        }
    };
    auto put = [&](int s) {
        if (A_BY_K) {
#pragma unroll
            for (int i = 0; i < 8; ++i) As[s][(tid >> 7) * 8 + i][tid & 127] = ra[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; i += 4)
                *(float4 *)&As[s][tid >> 4][(tid & 15) * 8 + i] = make_float4(ra[i], ra[i + 1], ra[i + 2], ra[i + 3]);
        }
        if (B_BY_K) {
#pragma unroll
            for (int i = 0; i < 8; ++i) Bs[s][(tid >> 7) * 8 + i][tid & 127] = rb[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; i += 4)
                *(float4 *)&Bs[s][tid >> 4][(tid & 15) * 8 + i] = make_float4(rb[i], rb[i + 1], rb[i + 2], rb[i + 3]);
        }
    };

    const int tx = tid & 15, ty = tid >> 4;
    Pair acc[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = 0;
    fetch(k_begin);
    put(0);
    __syncthreads();
    int s = 0;
    for (int64_t k0 = k_begin; k0 < k_end; k0 += BK, s ^= 1) {
        const bool more = k0 + BK < k_end;
        if (more) fetch(k0 + BK);
#pragma unroll
        for (int k = 0; k < BK; ++k) {
            float av[8];
            *(float4 *)&av[0] = *(const float4 *)&As[s][k][ty * 4];
            *(float4 *)&av[4] = *(const float4 *)&As[s][k][64 + ty * 4];
            ulonglong2 bl = *(const ulonglong2 *)&Bs[s][k][tx * 4], bh = *(const ulonglong2 *)&Bs[s][k][64 + tx * 4];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const Pair v = pair(av[i], av[i]);
                acc[i][0] = fma2(v, bl.x, acc[i][0]);
                acc[i][1] = fma2(v, bl.y, acc[i][1]);
                acc[i][2] = fma2(v, bh.x, acc[i][2]);
                acc[i][3] = fma2(v, bh.y, acc[i][3]);
            }
        }
        if (more) put(s ^ 1);
        __syncthreads();
    }

    const T *bias0 = (const T *)p.bias0, *bias1 = (const T *)p.bias1;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t m = m0 + (i < 4 ? ty * 4 + i : 64 + ty * 4 + i - 4);
        if (m >= p.m) continue;
        float v[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = split(acc[i][j]);
            v[2 * j] = f.x;
            v[2 * j + 1] = f.y;
        }
        if (KIND == FF_GATE) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t n = n0 + tx * 4 + j;
                if (n >= p.n) continue;
                float g = v[j], u = v[4 + j], act, slope;
                if (bias0) g += Elem<T>::load(bias0[n]);
                if (bias1) u += Elem<T>::load(bias1[n]);
                act_both_rt(p.act, g, act, slope);
                ((T *)p.c0)[m * p.ldc + n] = Elem<T>::store(act * u);
                if (p.gate) {
                    const int64_t at = ff_saved_at(m, n, p.m, p.n);
                    p.gate[at] = g;
                    p.up[at] = u;
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int64_t n = n0 + (j < 4 ? tx * 4 + j : 64 + tx * 4 + j - 4);
                if (n >= p.n) continue;
                if (KIND == FF_GATE_BACK) {
                    const int64_t at = ff_saved_at(m, n, p.m, p.n);
                    const float g = p.gate[at], u = p.up[at];
                    float act, slope;
                    act_both_rt(p.act, g, act, slope);
                    ((T *)p.c0)[m * p.ldc + n] = Elem<T>::store(v[j] * u * slope);
                    ((T *)p.c0)[m * p.ldc + p.n + n] = Elem<T>::store(v[j] * act);
                    ((T *)p.c1)[m * p.n + n] = Elem<T>::store(act * u);
                } else if (p.splits > 1) {
                    p.part[((int64_t)part * p.m + m) * p.n + n] = v[j];
                } else {
                    const bool second = m >= p.row_split;
                    T *c = (T *)(second ? p.c1 : p.c0);
                    if (c == nullptr) continue;
                    const float f = bias0 ? v[j] + Elem<T>::load(bias0[n]) : v[j];
                    c[(second ? m - p.row_split : m) * p.ldc + n] = Elem<T>::store(f);
                }
            }
        }
    }
}

}  // namespace

// enough shares for about two blocks on every SM, of at least 128 steps each
int ff_ffma_splits(int m, int n, int k) {
    const long long tiles = (long long)ceil_div(m, BM) * ceil_div(n, BN);
    if (tiles == 0 || tiles >= 148) return 1;
    long long s = 296 / tiles;
    if (s > k / 128) s = k / 128;
    if (s > 32) s = 32;
    return s < 1 ? 1 : (int)s;
}

int launch_ff_ffma(fc_context *ctx, const FfProduct &p) {
    const int step = p.kind == FF_GATE ? BN / 2 : BN;
    const long long n_tiles = ceil_div(p.n, step), m_tiles = ceil_div(p.m, BM);
    const int k_share = (int)ceil_div(ceil_div(p.k, p.splits), BK) * BK;
    const long long blocks = n_tiles * m_tiles * p.splits;
    FC_REQUIRE(blocks < (1ll << 31), FC_ERR_UNSUPPORTED, "product of %lld blocks", blocks);
    if (blocks == 0) return FC_OK;
    return with_type(p.type, [&](auto t) -> int {
        using T = decltype(t);
        const int vec = 16 / sizeof(T);
        const bool a_wide = p.lda % vec == 0 && aligned16(p.a);
        const bool b_wide = p.ldb % vec == 0 && aligned16(p.b0) && aligned16(p.b1);
        auto go = [&](auto kernel) -> int {
            FC_CHECK_CUDA(launch_pdl(kernel, dim3((unsigned)blocks), dim3(FF_THREADS), 0, ctx->stream, p, (int)n_tiles, (int)m_tiles,
                                     k_share, a_wide, b_wide));
            return FC_OK;
        };
        if (p.kind == FF_GATE) return go(ff_ffma_kernel<T, true, true, FF_GATE>);
        if (p.kind == FF_GATE_BACK) return go(ff_ffma_kernel<T, true, false, FF_GATE_BACK>);
        if (!p.a_by_k) return go(ff_ffma_kernel<T, false, false, FF_STORE>);
        return p.b_by_k ? go(ff_ffma_kernel<T, true, true, FF_STORE>) : go(ff_ffma_kernel<T, true, false, FF_STORE>);
    });
}

}  // namespace fc
