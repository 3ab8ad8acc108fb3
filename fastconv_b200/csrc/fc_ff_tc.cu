// The feed-forward block's matrix products on the 5th-generation tensor cores, bf16 and fp16.
//
// A pair of CTAs computes 256 x bn outputs (bn = 64, 128 or 256) with tcgen05.mma.cta_group::2: each CTA stages its own 128
// rows of A and half of B's columns, so an operand byte is fetched into shared memory once for 256 rows or bn columns.
// Persistent; per CTA
//   warp 0      producer: TMA boxes of 64 reduction steps into a ring of 5 stages (16 KB of A, up to 16 KB of B)
//   warp 1      of the pair's first CTA: the matrix instructions, into one of two accumulators in tensor memory
//   warps 2..9  epilogue of the other accumulator: 32 rows x 32 columns at a time, from tensor memory through registers and
//               a swizzled 2 KB piece of shared memory to a TMA store, which also cuts off what lies outside the matrix
// Operands come as they lie in memory: rows along the reduction (K-major) or across it (MN-major, for the products whose
// reduction runs over rows of the map or of a weight matrix); no transposed copy is made.
//
// FF_GATE: the first CTA's half of B are rows of the gate's weights, the second's the same rows of the up projection's, so
// columns j and bn/2 + j of the accumulator are the two values that one output needs.
#include <cstring>
#include <type_traits>

#include "fc_gated_ff.h"
#include "fc_last.cuh"
#include "fc_tc_common.cuh"

namespace fc {

namespace {

using namespace last;
using namespace tc;

constexpr int KB = 64;                        // reduction steps of a stage: 128 bytes, one swizzle span
constexpr int FF_STAGES = 5;
constexpr int HALF_BYTES = 128 * KB * 2;      // one CTA's A, and the most of its B, in a stage
constexpr int EPI_WARPS = 8;
constexpr int PIECE = 32 * 32 * 2;            // 32 rows x 32 columns of 16 bits
constexpr int PIECES = 4;                     // a warp's ring of pieces on their way out
constexpr int FF_TC_THREADS = 64 + 32 * EPI_WARPS;
constexpr int RING_BYTES = FF_STAGES * 2 * HALF_BYTES;
constexpr int OUT_BYTES = EPI_WARPS * PIECES * PIECE;
constexpr int FF_SMEM = 1024 + RING_BYTES + OUT_BYTES + 256;

struct FfMaps {
    CUtensorMap a[2], b[2], c[3];
};

struct FfTc {
    int m, n;                 // rows of one destination, columns
    int m_tiles, dest_tiles;  // row tiles in all, and of one destination
    int live_tiles, skip;     // those that are computed: live_tiles from `skip` on
    int n_tiles, splits;
    int kb_total, kb_first, kb_share;  // k-blocks; those before kb_first come from the first maps; of one share
    int bn, act;
    long long items;
    const void *bias0, *bias1;
    float *gate, *up;  // saved: written (FF_GATE) or read (FF_GATE_BACK)
    float *part;
    int *status;
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t first_cta(uint32_t addr) {  // the same place in the pair's first CTA
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ void arrive_remote(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// into this CTA's shared memory, reported to the first CTA's barrier
__device__ __forceinline__ void pair_load_2d(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
        "l"(map), "r"(bar), "r"(x), "r"(y)
        : "memory");
}
__device__ __forceinline__ void store_2d(const CUtensorMap *map, uint32_t src, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map), "r"(src), "r"(x), "r"(y)
                 : "memory");
}
__device__ __forceinline__ void pair_commit(uint32_t bar) {  // arrives at the barrier of both CTAs
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
        "h"((uint16_t)3)
        : "memory");
}
__device__ __forceinline__ void pair_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,"
        "%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// Operand descriptor of a tile in 128-byte rows with the 128-byte swizzle.  K-major: a row is one matrix row, groups of 8
// rows are 1024 bytes apart.  MN-major: a row is one reduction step of 64 matrix rows; groups of 8 steps are 1024 bytes apart
// (stride offset), blocks of 64 matrix rows KB * 128 bytes (leading offset).
template <bool BY_K>
__device__ __forceinline__ uint64_t operand(uint32_t addr) {
    uint64_t d = (uint64_t)((addr & 0x3FFFF) >> 4);
    d |= (uint64_t)(BY_K ? 1 : (KB * 128) >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}

// Sixteen-bit values of 32 neighbouring columns of this lane's row -> one piece (64-byte swizzle) -> TMA store.
struct Outlet {
    uint32_t base;  // the warp's pieces
    int next;
    __device__ __forceinline__ uint32_t open() {  // a piece that is free again
        asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(PIECES - 1) : "memory");
        __syncwarp();
        const uint32_t p = base + next * PIECE;
        next = (next + 1) % PIECES;
        return p;
    }
    template <typename T>
    __device__ __forceinline__ void put(const CUtensorMap *map, const float (&v)[32], int x, int y, int lane) {
        const uint32_t p = open();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                Vec<T, 2> two;
                const float f[2] = {v[8 * i + 2 * j], v[8 * i + 2 * j + 1]};
                two.pack(f);
                w[j] = *reinterpret_cast<const uint32_t *>(&two);
            }
            const uint32_t at = p + lane * 64 + ((i ^ ((lane >> 1) & 3)) << 4);
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
            store_2d(map, p, x, y);
        }
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");  // one group a piece in every lane, so that all count alike
    }
};

// 32 columns from n on of a 16-byte aligned vector of n_end (a multiple of 8) values, added to v
template <typename T>
__device__ __forceinline__ void add_bias(const void *bias, int n, int n_end, float (&v)[32]) {
    if (bias == nullptr) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (n + 8 * i >= n_end) break;
        float f[8];
        Vec<T, 8>::load((const T *)bias + n + 8 * i).unpack(f);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[8 * i + j] += f[j];
    }
}

template <int ACT>
__device__ __forceinline__ void gate_values(const float (&g)[32], const float (&u)[32], float (&h)[32]) {
#pragma unroll
    for (int j = 0; j < 32; ++j) h[j] = act_value<ACT, false>(g[j]) * u[j];
}
template <int ACT>
__device__ __forceinline__ void gate_back_values(float (&g)[32], float (&u)[32], float (&dh)[32]) {
    // in: g, u, dh; out: dg, du, h
#pragma unroll
    for (int j = 0; j < 32; ++j) {
        float a, d;
        act_both<ACT, false>(g[j], a, d);
        g[j] = dh[j] * u[j] * d;
        const float h = a * u[j];
        u[j] = dh[j] * a;
        dh[j] = h;
    }
}

template <typename T, bool A_BY_K, bool B_BY_K, int KIND>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(FF_TC_THREADS, 1)
    ff_tc_kernel(const __grid_constant__ FfMaps maps, const FfTc P) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem = (smem_u32(smem_raw) + 1023) & ~1023u;
    const uint32_t out_base = smem + RING_BYTES;
    const uint32_t bars = out_base + OUT_BYTES;
    auto bar_full = [&](int s) { return bars + 8 * s; };
    auto bar_empty = [&](int s) { return bars + 8 * (FF_STAGES + s); };
    auto bar_acc_full = [&](int a) { return bars + 8 * (2 * FF_STAGES + a); };
    auto bar_acc_empty = [&](int a) { return bars + 8 * (2 * FF_STAGES + 2 + a); };
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word;
    volatile int *abort_flag = &abort_word;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const long long first = blockIdx.x >> 1, step = gridDim.x >> 1;
    const uint32_t b_bytes = (uint32_t)P.bn / 2 * 128;  // this CTA's share of B in a stage

    if (threadIdx.x == 0) {
        for (int s = 0; s < FF_STAGES; ++s) {
            mbar_init(bar_full(s), 1);
            mbar_init(bar_empty(s), 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(bar_acc_full(a), 1);
            mbar_init(bar_acc_empty(a), 2 * EPI_WARPS);
        }
        abort_word = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(2 * P.bn)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    pdl_wait();

    auto decode = [&](long long item, int &mt, int &nt, int &split) {
        nt = (int)(item % P.n_tiles);
        const long long rest = item / P.n_tiles;
        mt = P.skip + (int)(rest % P.live_tiles);
        split = (int)(rest / P.live_tiles);
    };

    if (warp == 0) {
        if (lane == 0) {
            int g = 0;
            bool ok = true;
            for (long long item = first; item < P.items && ok; item += step) {
                int mt, nt, split;
                decode(item, mt, nt, split);
                const int dest = mt / P.dest_tiles;
                const int m0 = (mt - dest * P.dest_tiles) * 256 + (int)rank * 128;
                const int n0 = KIND == FF_GATE ? nt * (P.bn / 2) : nt * P.bn + (int)rank * (P.bn / 2);
                const int lo = split * P.kb_share, hi = min(P.kb_total, lo + P.kb_share);
                for (int kb = lo; kb < hi; ++kb, ++g) {
                    const int s = g % FF_STAGES;
                    if (!mbar_wait(bar_empty(s), ((g / FF_STAGES) & 1) ^ 1, abort_flag, P.status)) {
                        ok = false;
                        break;
                    }
                    const uint32_t a_at = smem + s * 2 * HALF_BYTES, b_at = a_at + HALF_BYTES;
                    const uint32_t full = first_cta(bar_full(s));
                    if (rank == 0) mbar_expect_tx(bar_full(s), 2 * (HALF_BYTES + b_bytes));
                    const int second = kb >= P.kb_first;
                    const int k0 = (second ? kb - P.kb_first : kb) * KB;
                    const CUtensorMap *am = &maps.a[A_BY_K ? second : dest];
                    const CUtensorMap *bm = &maps.b[KIND == FF_GATE ? (int)rank : second];
                    if (A_BY_K) {
                        pair_load_2d(a_at, am, full, k0, m0);
                    } else {
#pragma unroll
                        for (int i = 0; i < 2; ++i) pair_load_2d(a_at + i * KB * 128, am, full, m0 + 64 * i, k0);
                    }
                    if (B_BY_K) {
                        pair_load_2d(b_at, bm, full, k0, n0);
                    } else {
                        for (int i = 0; i < P.bn / 128; ++i) pair_load_2d(b_at + i * KB * 128, bm, full, n0 + 64 * i, k0);
                    }
                }
            }
            // the other CTA's last releases have arrived here before this one may end
            for (int i = 0; i < FF_STAGES && ok; ++i, ++g)
                ok = mbar_wait(bar_empty(g % FF_STAGES), ((g / FF_STAGES) & 1) ^ 1, abort_flag, P.status);
        }
    } else if (warp == 1) {
        if (rank == 0 && lane == 0) {
            constexpr uint32_t type = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
            const uint32_t idesc = (1u << 4) | (type << 7) | (type << 10) | ((A_BY_K ? 0u : 1u) << 15) | ((B_BY_K ? 0u : 1u) << 16) |
                                   ((uint32_t)(P.bn >> 3) << 17) | ((256u >> 4) << 24);
            int g = 0, t = 0;
            bool ok = true;
            for (long long item = first; item < P.items && ok; item += step, ++t) {
                int mt, nt, split;
                decode(item, mt, nt, split);
                const int lo = split * P.kb_share, hi = min(P.kb_total, lo + P.kb_share);
                const int acc = t & 1;
                if (!mbar_wait(bar_acc_empty(acc), ((t >> 1) & 1) ^ 1, abort_flag, P.status)) break;
                tc_fence_after();
                const uint32_t d = tmem + acc * P.bn;
                for (int kb = lo; kb < hi; ++kb, ++g) {
                    const int s = g % FF_STAGES;
                    if (!mbar_wait(bar_full(s), (g / FF_STAGES) & 1, abort_flag, P.status)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t a_at = smem + s * 2 * HALF_BYTES, b_at = a_at + HALF_BYTES;
#pragma unroll
                    for (int k = 0; k < KB / 16; ++k)  // 16 steps: 32 bytes along a row, or 16 rows
                        pair_mma(d, operand<A_BY_K>(a_at + k * (A_BY_K ? 32 : 2048)), operand<B_BY_K>(b_at + k * (B_BY_K ? 32 : 2048)),
                                 idesc, kb > lo || k > 0);
                    pair_commit(bar_empty(s));
                }
                if (ok) pair_commit(bar_acc_full(acc));
            }
        }
    } else {
        const int quad = warp & 3, half = (warp - 2) >> 2;  // tensor memory lanes of this warp; every second column piece
        Outlet out = {out_base + (uint32_t)(warp - 2) * PIECES * PIECE, 0};
        const int cols = KIND == FF_GATE ? P.bn / 2 : P.bn;  // output columns of a tile
        int t = 0;
        for (long long item = first; item < P.items; item += step, ++t) {
            int mt, nt, split;
            decode(item, mt, nt, split);
            const int dest = mt / P.dest_tiles;
            const int y = (mt - dest * P.dest_tiles) * 256 + (int)rank * 128 + quad * 32;  // the warp's first row
            const int acc = t & 1;
            if (!mbar_wait(bar_acc_full(acc), (t >> 1) & 1, abort_flag, P.status)) break;
            tc_fence_after();
            const uint32_t d = tmem + acc * P.bn + ((uint32_t)(quad * 32) << 16);
            const int row = y + lane, block_rows = min(32, P.m - y);  // of the block of 32 rows in the saved layout
            for (int c = half * 32; c < cols; c += 64) {
                const int x = nt * cols + c;
                if (x >= P.n || y >= P.m) break;
                uint32_t r[32];
                float v[32];
                tmem_ld32(d + c, r);
                if (KIND == FF_GATE) {
                    uint32_t r2[32];
                    float u[32];
                    tmem_ld32(d + cols + c, r2);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]), u[j] = __uint_as_float(r2[j]);
                    add_bias<T>(P.bias0, x, P.n, v);
                    add_bias<T>(P.bias1, x, P.n, u);
                    if (P.gate != nullptr && row < P.m) {
                        float4 *gs = (float4 *)(P.gate + (size_t)y * P.n) + (size_t)(x / 4) * block_rows + lane;
                        float4 *us = (float4 *)(P.up + (size_t)y * P.n) + (size_t)(x / 4) * block_rows + lane;
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            if (x + 4 * j >= P.n) break;
                            gs[(size_t)j * block_rows] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
                            us[(size_t)j * block_rows] = make_float4(u[4 * j], u[4 * j + 1], u[4 * j + 2], u[4 * j + 3]);
                        }
                    }
                    float h[32];
                    switch (P.act) {
                        case FC_ACT_RELU: gate_values<FC_ACT_RELU>(v, u, h); break;
                        case FC_ACT_SILU: gate_values<FC_ACT_SILU>(v, u, h); break;
                        case FC_ACT_GELU: gate_values<FC_ACT_GELU>(v, u, h); break;
                        case FC_ACT_GELU_TANH: gate_values<FC_ACT_GELU_TANH>(v, u, h); break;
                        case FC_ACT_SIGMOID: gate_values<FC_ACT_SIGMOID>(v, u, h); break;
                        default: gate_values<FC_ACT_NONE>(v, u, h);
                    }
                    out.put<T>(&maps.c[0], h, x, y, lane);
                } else if (KIND == FF_GATE_BACK) {
                    float g[32], u[32];
#pragma unroll
                    for (int j = 0; j < 32; ++j) g[j] = u[j] = 0.0f;
                    if (row < P.m) {
                        const float4 *gs = (const float4 *)(P.gate + (size_t)y * P.n) + (size_t)(x / 4) * block_rows + lane;
                        const float4 *us = (const float4 *)(P.up + (size_t)y * P.n) + (size_t)(x / 4) * block_rows + lane;
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            if (x + 4 * j >= P.n) break;
                            const float4 a = __ldg(gs + (size_t)j * block_rows), b = __ldg(us + (size_t)j * block_rows);
                            g[4 * j] = a.x, g[4 * j + 1] = a.y, g[4 * j + 2] = a.z, g[4 * j + 3] = a.w;
                            u[4 * j] = b.x, u[4 * j + 1] = b.y, u[4 * j + 2] = b.z, u[4 * j + 3] = b.w;
                        }
                    }
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
                    switch (P.act) {
                        case FC_ACT_RELU: gate_back_values<FC_ACT_RELU>(g, u, v); break;
                        case FC_ACT_SILU: gate_back_values<FC_ACT_SILU>(g, u, v); break;
                        case FC_ACT_GELU: gate_back_values<FC_ACT_GELU>(g, u, v); break;
                        case FC_ACT_GELU_TANH: gate_back_values<FC_ACT_GELU_TANH>(g, u, v); break;
                        case FC_ACT_SIGMOID: gate_back_values<FC_ACT_SIGMOID>(g, u, v); break;
                        default: gate_back_values<FC_ACT_NONE>(g, u, v);
                    }
                    out.put<T>(&maps.c[0], g, x, y, lane);
                    out.put<T>(&maps.c[1], u, x, y, lane);
                    out.put<T>(&maps.c[2], v, x, y, lane);
                } else {
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
                    if (P.splits > 1) {  // [share][block of 32 rows][4 columns][row]
                        const size_t block = ((size_t)split * P.m_tiles + mt) * 8 + rank * 4 + quad;
                        float4 *ps = (float4 *)P.part + (block * (P.n / 4) + x / 4) * 32 + lane;
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            if (x + 4 * j >= P.n) break;
                            ps[j * 32] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
                        }
                    } else {
                        add_bias<T>(P.bias0, x, P.n, v);
                        out.put<T>(&maps.c[dest], v, x, y, lane);
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) arrive_remote(first_cta(bar_acc_empty(acc)));
        }
        asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }

    __syncthreads();
    if (*abort_flag) {  // let copies that are still in flight land before shared memory is released
        for (int i = 0; i < 64; ++i) __nanosleep(1000);
    }
    tc_fence_before();
    cluster_sync();
    if (warp == 1) {
        __syncwarp();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * P.bn) : "memory");
    }
}

// the shares of a split reduction, added in order; a thread has four columns of one row
template <typename T>
__global__ void __launch_bounds__(256) ff_tc_join_kernel(const FfTc P, T *c0, T *c1, int64_t ldc) {
    pdl_wait();
    const int quads = P.n / 4, col_blocks = (quads + 3) / 4;
    const long long blocks = (long long)P.m_tiles * 8 * col_blocks * 4;  // of 8 rows x 4 quads: a warp each
    for (long long w = ((long long)blockIdx.x * 256 + threadIdx.x) >> 5; w < blocks; w += (long long)gridDim.x * 8) {
        const int lane = threadIdx.x & 31;
        const int r8 = (int)(w & 3);
        const long long rest = w >> 2;
        const int q = (int)(rest % col_blocks) * 4 + (lane >> 3);
        const long long block = rest / col_blocks;
        const int r = r8 * 8 + (lane & 7);
        const int mt = (int)(block >> 3), dest = mt / P.dest_tiles;
        const int row = (mt - dest * P.dest_tiles) * 256 + (int)(block & 7) * 32 + r;
        T *c = dest ? c1 : c0;
        if (q >= quads || row >= P.m || c == nullptr) continue;
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int s = 0; s < P.splits; ++s) {
            const float4 f = __ldg((const float4 *)P.part + (((size_t)s * P.m_tiles * 8 + block) * quads + q) * 32 + r);
            v[0] += f.x, v[1] += f.y, v[2] += f.z, v[3] += f.w;
        }
        if (P.bias0) {
            float b[4];
            Vec<T, 4>::load((const T *)P.bias0 + 4 * q).unpack(b);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] += b[i];
        }
        Vec<T, 4> out;
        out.pack(v);
        out.store(c + (size_t)row * ldc + 4 * q);
    }
}

// ---- host -----------------------------------------------------------------------------------------------------------

// a matrix of 16-bit values, rows `ld` apart; box = box_cols x box_rows
int matrix_map(CUtensorMap *map, int type, const void *base, long long cols, long long rows, int64_t ld, int box_cols, int box_rows) {
    EncodeTiledFn enc;
    FC_PROPAGATE(get_encoder(&enc));
    cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
    cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows};
    cuuint32_t estr[2] = {1, 1};
    const CUresult r = enc(map, type == FC_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
                           const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           box_cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    FC_REQUIRE(r == CUDA_SUCCESS, FC_ERR_CUDA, "cuTensorMapEncodeTiled failed with %d (%lld x %lld, rows %lld apart)", (int)r, rows, cols,
               (long long)ld);
    return FC_OK;
}

}  // namespace

// Tile width and shares of the reduction, by an estimate in SM clocks: a k-block of 256 x bn takes 2 bn clocks of the matrix
// pipe and (16 KB + 64 bn bytes) at about 56 bytes a clock of operand copies; the first tile's latency and a tile's epilogue
// that nothing hides, about 2500; a split result is written and read once more by every share (about 3000 bytes a clock, all SMs),
// and joined by a kernel of its own (about 4000).
FfTcPlan ff_tc_plan(int kind, int dests, int m, int n, int kb_total, bool b_by_k) {
    const int pairs = 74;
    FfTcPlan best = {256, 1};
    double best_cost = 1e300;
    for (int bn = 256; bn >= (b_by_k ? 64 : 128); bn /= 2) {
        const int cols = kind == FF_GATE ? bn / 2 : bn;
        const double tiles = (double)dests * ceil_div(m, 256) * ceil_div(n, cols);
        for (int s = 1; s <= (kind == FF_STORE ? 16 : 1); ++s) {
            if (s > 1 && kb_total / s < 4) break;
            const int share = (int)ceil_div(kb_total, s);
            if (s > 1 && (s - 1) * share >= kb_total) continue;  // the last share would be empty
            const double copies = (16384.0 + 64.0 * bn) / 56.0, mma = 2.0 * bn;
            const double waves = (double)ceil_div((size_t)(tiles * s), pairs);
            double cost = waves * share * (copies > mma ? copies : mma) + 2500.0;
            if (s > 1) cost += 4000.0 + (double)s * dests * m * n * 8.0 / 3000.0;
            if (cost < best_cost * 0.999) {
                best_cost = cost;
                best = {bn, s};
            }
        }
    }
    return best;
}

static void tc_shape(const FfProduct &p, int *dests, int *m, int *kb_first, int *kb_total) {
    *dests = p.row_split < p.m ? 2 : 1;
    *m = p.row_split < p.m ? p.row_split : p.m;
    *kb_first = (int)ceil_div(p.b_split, KB);
    *kb_total = *kb_first + (p.b_split < p.k ? (int)ceil_div(p.k - p.b_split, KB) : 0);
}

size_t ff_tc_part_floats(const FfProduct &p) {
    if (p.kind != FF_STORE) return 0;
    int dests, m, kb_first, kb_total;
    tc_shape(p, &dests, &m, &kb_first, &kb_total);
    const FfTcPlan plan = ff_tc_plan(p.kind, dests, m, p.n, kb_total, p.b_by_k);
    return plan.splits > 1 ? (size_t)plan.splits * dests * ceil_div(m, 256) * 256 * p.n : 0;
}

// what the copies need: rows that are multiples of 16 bytes, on 16-byte boundaries
bool ff_tc_fits(const FfProduct &p) {
    if (p.type == FC_DTYPE_F32 || p.m == 0 || p.k == 0) return false;
    if (p.lda % 8 || p.ldb % 8 || p.ldc % 8 || p.n % 8) return false;
    if (p.b_split < p.k && p.b_split % 8) return false;
    if (p.row_split < p.m && p.row_split % 8) return false;
    const void *all[] = {p.a, p.b0, p.b1, p.c0, p.c1, p.bias0, p.bias1, p.gate, p.up};
    for (const void *q : all)
        if (!aligned16(q)) return false;
    return true;
}

int launch_ff_tc(fc_context *ctx, const FfProduct &p) {
    int dests, m, kb_first, kb_total;
    tc_shape(p, &dests, &m, &kb_first, &kb_total);
    const FfTcPlan plan = ff_tc_plan(p.kind, dests, m, p.n, kb_total, p.b_by_k);
    FfTc P = {};
    P.m = m;
    P.n = p.n;
    P.dest_tiles = (int)ceil_div(m, 256);
    P.m_tiles = dests * P.dest_tiles;
    P.skip = dests == 2 && p.c0 == nullptr ? P.dest_tiles : 0;
    P.live_tiles = dests == 2 && (p.c0 == nullptr || p.c1 == nullptr) ? P.dest_tiles : P.m_tiles;
    P.bn = plan.bn;
    P.n_tiles = (int)ceil_div(p.n, p.kind == FF_GATE ? plan.bn / 2 : plan.bn);
    P.splits = plan.splits;
    P.kb_total = kb_total;
    P.kb_first = kb_first;
    P.kb_share = (int)ceil_div(kb_total, plan.splits);
    P.act = p.act;
    P.items = (long long)P.live_tiles * P.n_tiles * P.splits;
    P.bias0 = p.bias0;
    P.bias1 = p.bias1;
    P.gate = p.gate;
    P.up = p.up;
    P.part = p.part;
    P.status = ctx->d_status;

    FfMaps maps;
    memset(&maps, 0, sizeof maps);
    const uint8_t *a = (const uint8_t *)p.a;
    const int second = dests == 2 || p.b_split < p.k;
    for (int i = 0; i <= second; ++i) {  // A's columns (K-major: the reduction; MN-major: the rows of one destination)
        const int cols = p.a_by_k ? (i ? p.k - p.b_split : p.b_split) : m;
        const int skip = i == 0 ? 0 : p.a_by_k ? p.b_split : m;
        FC_PROPAGATE(matrix_map(&maps.a[i], p.type, a + (size_t)skip * 2, cols, p.a_by_k ? p.m : p.k, p.lda, 64, p.a_by_k ? 128 : KB));
    }
    const void *b[2] = {p.b0, p.b1};
    for (int i = 0; i < 2 && b[i]; ++i) {
        const int k = p.kind == FF_GATE ? p.k : i ? p.k - p.b_split : p.b_split;
        FC_PROPAGATE(p.b_by_k ? matrix_map(&maps.b[i], p.type, b[i], k, p.n, p.ldb, 64, plan.bn / 2)
                              : matrix_map(&maps.b[i], p.type, b[i], p.n, k, p.ldb, 64, KB));
    }
    void *c[3] = {p.c0, p.c1, nullptr};
    if (p.kind == FF_GATE_BACK) {
        c[1] = (uint8_t *)p.c0 + (size_t)p.n * 2;
        c[2] = p.c1;
    }
    if (P.splits == 1)
        for (int i = 0; i < 3; ++i)
            if (c[i]) FC_PROPAGATE(matrix_map(&maps.c[i], p.type, c[i], p.n, m, i == 2 ? p.n : p.ldc, 32, 32));

    long long pairs = ctx->sm_count / 2;
    if (pairs > P.items) pairs = P.items;
    return with_type(p.type, [&](auto t) -> int {
        using T = decltype(t);
        if constexpr (std::is_same<T, float>::value) {
            set_error("fp32 has no tensor-core product");
            return FC_ERR_UNSUPPORTED;
        } else {
            auto go = [&](auto kernel) -> int {
                FC_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, FF_SMEM));
                FC_CHECK_CUDA(launch_pdl(kernel, dim3((unsigned)(2 * pairs)), dim3(FF_TC_THREADS), FF_SMEM, ctx->stream, maps, P));
                return FC_OK;
            };
            if (p.kind == FF_GATE) return go(ff_tc_kernel<T, true, true, FF_GATE>);
            if (p.kind == FF_GATE_BACK) return go(ff_tc_kernel<T, true, false, FF_GATE_BACK>);
            FC_PROPAGATE(!p.a_by_k  ? go(ff_tc_kernel<T, false, false, FF_STORE>)
                         : p.b_by_k ? go(ff_tc_kernel<T, true, true, FF_STORE>)
                                    : go(ff_tc_kernel<T, true, false, FF_STORE>));
            if (P.splits > 1) {
                long long blocks = ceil_div((size_t)P.m_tiles * 8 * 4 * ceil_div(p.n, 16), 8);
                if (blocks > 148 * 8) blocks = 148 * 8;
                FC_CHECK_CUDA(launch_pdl(ff_tc_join_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, ctx->stream, P, (T *)p.c0,
                                         (T *)p.c1, p.ldc));
            }
            return FC_OK;
        }
    });
}

}  // namespace fc
