// The feed-forward block's matrix products on the 5th-generation tensor cores.
//
// A pair of CTAs computes 256 x bn outputs (bn = 64, 128 or 256) with tcgen05.mma.cta_group::2: each CTA stages its own 128
// rows of A and half of B's columns, so an operand byte is fetched into shared memory once for 256 rows or bn columns.
// Persistent; per CTA
//   warp 0      producer: TMA boxes of 64 reduction steps (a k-block) into a ring of stages
//   warp 1      of the pair's first CTA: the matrix instructions, into one of two accumulators in tensor memory
//   warps 2..9  epilogue of the other accumulator: 32 rows x 32 columns at a time, from tensor memory through registers and
//               a swizzled 2 KB piece of shared memory to a TMA store, which also cuts off what lies outside the matrix
// Operands come as they lie in memory: rows along the reduction (K-major) or across it (MN-major, for the products whose
// reduction runs over rows of the map or of a weight matrix); no transposed copy is made.
//
// FF_GATE: the first CTA's half of B are rows of the gate's weights, the second's the same rows of the up projection's, so
// columns j and bn/2 + j of the accumulator are the two values that one output needs.
//
// fp32 (three planes): a value is the sum of three bf16 values exactly, x = h + m + l (8 bits each).  Of the nine products of two
// values the six largest are taken, hh, hm, mh, hl, lh, mm; the others are below 2^-25 of the result.  The tensor cores' fp32
// additions round toward zero, which over a long reduction adds up to a bias of some 2e-8 an instruction: the five small
// products, where that does not matter, have an accumulator of their own, and the sum of hh is taken over into registers,
// rounded to nearest, every 256 steps.  Six times the work of a bf16 product; 107 TFLOP/s at 3137 rows 256->1024->256, where
// products on the FP32 pipe gave 29.
//
// What bounds them, measured on one B200 in bf16: a plain product of 210 GFLOP takes 126 to 144 us by the clock that the power
// cap leaves, the matrix pipe active 0.94 of the time; the gate's of 50176 rows 512->2048 (210 GFLOP) 136 us, 0.91.  With 12544
// rows 1024->4096 the gate that also writes 0.41 GB of saved values takes 177 us, and the backward gate (105 GFLOP) 150 us for
// 0.75 GB, 5 TB/s: memory.  Small products are bound by a tile's way through set-up, first copies and epilogue, 5 us.
#include <cstring>
#include <type_traits>

#include "fc_gated_ff.h"
#include "fc_last.cuh"
#include "fc_tc_common.cuh"

namespace fc {

namespace {

using namespace last;
using namespace tc;

constexpr int KB = 64;                    // reduction steps of a k-block: 128 bytes, one swizzle span
constexpr int HALF_BYTES = 128 * KB * 2;  // one CTA's A in a k-block and plane
constexpr int EPI_WARPS = 8;
constexpr int PIECE = 32 * 32 * 2;        // 32 rows x 32 columns of 16 bits
constexpr int FF_TC_THREADS = 64 + 32 * EPI_WARPS;
constexpr int CHUNK = 4;                  // k-blocks whose sum stays in tensor memory, three planes

// The ring of stages and, for every epilogue warp, of pieces on their way out.  Six stages of bn = 256 (narrower tiles have room
// for more); FF_GATE_BACK, which waits for memory and not for the matrix pipe, gives one for the three pieces that it writes at
// a time.
template <int PLANES, int KIND>
struct Ring {
    static constexpr int kPieces = KIND == FF_GATE_BACK || PLANES == 3 ? 4 : 2;
    static constexpr int kBytes =
        PLANES == 1 ? (KIND == FF_GATE_BACK ? 5 : 6) * 2 * HALF_BYTES : 2 * 3 * (HALF_BYTES + HALF_BYTES / 2);
    static constexpr int kOut = EPI_WARPS * kPieces * PIECE;
    static constexpr int kMost = 10;  // stages
    static constexpr int kSmem = 1024 + kBytes + kOut + 256;
};
// A stage holds one k-block of bn = 256 (512 clocks of the matrix pipe) or of three planes, else two: a stage's round of wait,
// commit and release takes some 430 clocks, which one k-block of a narrower tile does not fill.
__host__ __device__ constexpr int ff_kb_bytes(int planes, int bn) { return planes * (HALF_BYTES + bn * 64); }

struct FfMaps {
    CUtensorMap a[2], b[2], c[3];
};

struct FfTc {
    int m, n;                 // rows of one destination, columns
    int m_tiles, dest_tiles;  // row tiles in all, and of one destination
    int live_tiles, skip;     // those that are computed: live_tiles from `skip` on
    int n_tiles, splits;
    int kb_total, kb_first, kb_share;  // k-blocks; those before kb_first come from the first maps; of one share
    int bn, stages, act;
    int kbs;                  // k-blocks of a stage
    int items;                // tiles times shares
    const void *bias0, *bias1;
    int bias_wide;            // the biases can be read in 16-byte vectors
    float *gate, *up;         // saved: written (FF_GATE) or read (FF_GATE_BACK)
    int saved_wide;           // in float4
    void *c0, *c1;            // FF_STORE: destinations that are stored to without TMA (else null)
    int64_t ldc;
    float *part;
    int *status;
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}
__device__ __forceinline__ uint32_t first_cta(uint32_t addr) {  // the same place in the pair's first CTA
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// Nothing in memory is handed over, and no arrival at a barrier is ordered by it: each CTA has waited for those that the other
// sends to its own barriers before it comes here (the producer for the ring's, the matrix warp for the accumulators').
__device__ __forceinline__ void cluster_leave() {
    asm volatile("barrier.cluster.arrive.relaxed;\n\tbarrier.cluster.wait;" ::: "memory");
}
__device__ __forceinline__ void arrive_remote(uint32_t bar) {
    // relaxed: what it stands for are reads of tensor memory, ordered by the tcgen05 fences; a release would wait for the
    // warp's global stores too
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// into this CTA's shared memory, reported to the first CTA's barrier
__device__ __forceinline__ void pair_load(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
            dst),
        "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}
__device__ __forceinline__ void store_3d(const CUtensorMap *map, uint32_t src, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map), "r"(src), "r"(x), "r"(y),
                 "r"(z)
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
// what was loaded is there after the wait and not before: keeps its uses behind it
template <int N>
__device__ __forceinline__ void tmem_landed(uint32_t (&r)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
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

template <typename T>
__device__ __forceinline__ void pack_row(const float (&v)[32], uint32_t (&w)[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        Vec<T, 2> two;
        const float f[2] = {v[2 * i], v[2 * i + 1]};
        two.pack(f);
        w[i] = *reinterpret_cast<const uint32_t *>(&two);
    }
}

// Sixteen-bit values of 32 neighbouring columns of this lane's row -> one piece (64-byte swizzle) -> TMA store.
template <int PIECES>
struct Outlet {
    uint32_t base;  // the warp's pieces
    int next;
    // N pieces at once: one wait until as many are free, one fence
    template <int N>
    __device__ __forceinline__ void put(const CUtensorMap *map, int map_step, const uint32_t (&w)[N][16], int x, int y, int z, int z_step,
                                        int lane) {
        asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(PIECES - N) : "memory");
        __syncwarp();
        uint32_t at[N];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            at[k] = base + next * PIECE;
            next = (next + 1) & (PIECES - 1);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at[k] + lane * 64 + ((i ^ ((lane >> 1) & 3)) << 4)),
                             "r"(w[k][4 * i]), "r"(w[k][4 * i + 1]), "r"(w[k][4 * i + 2]), "r"(w[k][4 * i + 3])
                             : "memory");
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
#pragma unroll
        for (int k = 0; k < N; ++k) {
            if (lane == 0) store_3d(map + k * map_step, at[k], x, y, z + k * z_step);
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");  // one group a piece in every lane, so that all count alike
        }
    }
    template <typename T>
    __device__ __forceinline__ void put(const CUtensorMap *map, const float (&v)[32], int x, int y, int z, int lane) {
        uint32_t w[1][16];
        pack_row<T>(v, w[0]);
        put<1>(map, 0, w, x, y, z, 0, lane);
    }
};

// the values of the vector's columns from n on, added to v
template <typename T>
__device__ __forceinline__ void add_bias(const void *bias, int wide, int n, int n_end, float (&v)[32]) {
    constexpr int VEC = 16 / sizeof(T);
    if (bias == nullptr) return;
    if (wide && n + 32 <= n_end) {
#pragma unroll
        for (int i = 0; i < 32; i += VEC) {
            float f[VEC];
            Vec<T, VEC>::load((const T *)bias + n + i).unpack(f);
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[i + j] += f[j];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i)
            if (n + i < n_end) v[i] += Elem<T>::load(((const T *)bias)[n + i]);
    }
}

// 32 rows x 32 columns that lie in registers a row a lane -> rows y.. and columns x.. of c, turned in the warp's 4 KB of shared
// memory so that a warp writes a row's neighbouring columns: for destinations that TMA cannot address, and fp32.
template <typename T>
__device__ __forceinline__ void store_block(float *turn, T *c, int64_t ldc, int y, int m, int x, int n, const float (&v)[32], int lane) {
#pragma unroll
    for (int j = 0; j < 32; ++j) turn[lane * 32 + (j ^ lane)] = v[j];
    __syncwarp();
    const int rows = min(32, m - y);
    T *to = c + (size_t)y * ldc + x + lane;
    if (x + lane < n)
#pragma unroll 4
        for (int r = 0; r < rows; ++r, to += ldc) *to = Elem<T>::store(turn[r * 32 + (lane ^ r)]);
    __syncwarp();
}

// 32 saved values of the row y + lane, from column x on (ff_saved_at)
template <bool STORE>
__device__ __forceinline__ void saved_row(const FfTc &P, float *base, int y, int lane, int x, float (&v)[32]) {
    const int block_rows = min(32, P.m - y);
    if (P.saved_wide) {
        float4 *p = (float4 *)(base + (size_t)y * P.n) + (size_t)(x / 4) * block_rows + lane;
        auto move = [&](int j, int at) {
            if (STORE) {
                p[at] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
            } else {
                const float4 f = p[at];
                v[4 * j] = f.x, v[4 * j + 1] = f.y, v[4 * j + 2] = f.z, v[4 * j + 3] = f.w;
            }
        };
        if (x + 32 <= P.n && block_rows == 32) {
#pragma unroll
            for (int j = 0; j < 8; ++j) move(j, j * 32);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (x + 4 * j < P.n) move(j, j * block_rows);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            if (x + j >= P.n) break;
            float *p = base + ff_saved_at(y + lane, x + j, P.m, P.n);
            if (STORE)
                *p = v[j];
            else
                v[j] = *p;
        }
    }
}

// to a matrix that a product will read again: one plane of 16 bits, or the three bf16 parts
template <typename OT, int PLANES, int PIECES>
__device__ __forceinline__ void put_planes(Outlet<PIECES> &out, const CUtensorMap *map, float (&v)[32], int x, int y, int lane) {
    if constexpr (PLANES == 1) {
        out.template put<OT>(map, v, x, y, 0, lane);
    } else {
        float most = 0.0f;
#pragma unroll
        for (int j = 0; j < 32; ++j) most = fmaxf(most, fabsf(v[j]));
        const bool huge = most > 3.38e38f;  // where rounding to bf16 could give infinity, or it is there already
#pragma unroll 1
        for (int z = 0; z < 3; ++z) {  // a loop, as the pieces are: a launch of one tile a CTA waits for the instructions themselves
            uint32_t w[1][16];
            if (!huge) {
#pragma unroll
                for (int j = 0; j < 16; ++j) {  // of the third part: all that is left
                    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[0][j]) : "f"(v[2 * j + 1]), "f"(v[2 * j]));
                    v[2 * j] -= __uint_as_float(w[0][j] << 16);
                    v[2 * j + 1] -= __uint_as_float(w[0][j] & 0xffff0000u);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const float p = bf16_part(v[2 * j]), q = bf16_part(v[2 * j + 1]);
                    w[0][j] = __float_as_uint(p) >> 16 | (__float_as_uint(q) & 0xffff0000u);
                    v[2 * j] = fabsf(p) <= 3.4028234e38f ? v[2 * j] - p : 0.0f;
                    v[2 * j + 1] = fabsf(q) <= 3.4028234e38f ? v[2 * j + 1] - q : 0.0f;
                }
            }
            out.template put<1>(map, 0, w, x, y, z, 0, lane);
        }
    }
}

// fp32: GELU by the library's erfc, in a call for two values at a time (act, act' of both), because 32 copies of it are 50 KB of
// straight code that a tile would wait for.
__device__ __noinline__ float4 exact_gelu(float y, float z) {
    float4 r;
    act_both<FC_ACT_GELU, true>(y, r.x, r.y);
    act_both<FC_ACT_GELU, true>(z, r.z, r.w);
    return r;
}
// The other activations in line: exp(-z) = 2^t (1 + ln 2 * rest) with the rounding of t = -z log2(e) made good, and a
// reciprocal with one Newton step; a few units in the 23rd bit.  z is bounded so that no step overflows: below -87 the result is
// that of -87, 1.6e-38.
__device__ __forceinline__ float fine_sigmoid(float z) {
    z = at_most(at_least(z, -87.0f), 128.0f);
    const float t = z * -1.44269504088896341f;
    const float rest = fmaf(z, -1.44269504088896341f, -t) + z * -1.92596299e-8f;  // log2(e) = 1.44269502162933350 + 1.92596299e-8
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
    const float x = 1.0f + fmaf(e, rest * 0.69314718055994531f, e);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return fmaf(r, fmaf(-x, r, 1.0f), r);
}
template <int ACT>
__device__ __forceinline__ void fine_both(float z, float &a, float &d) {
    if (ACT == FC_ACT_SILU) {
        const float s = fine_sigmoid(z);
        a = at_least(z, -87.0f) * s;
        d = fmaf(a, 1.0f - s, s);
    } else if (ACT == FC_ACT_GELU_TANH) {
        z = at_least(z, -87.0f);
        const float t = fminf(z * z, 1e6f);
        const float s = fine_sigmoid(1.59576912160573071f * z * fmaf(0.044715f, t, 1.0f));
        a = z * s;
        d = fmaf(a * (1.0f - s), 1.59576912160573071f * fmaf(0.134145f, t, 1.0f), s);
    } else if (ACT == FC_ACT_SIGMOID) {
        a = fine_sigmoid(z);
        d = a * (1.0f - a);
    } else {
        act_both<ACT, true>(z, a, d);  // none, ReLU
    }
}
// use(j, act(g[j]), act'(g[j])) for all 32
template <typename F>
__device__ __forceinline__ void exact_acts(int act, const float (&g)[32], F &&use) {
    auto all = [&](auto kind) {
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            float a, d;
            fine_both<decltype(kind)::value>(g[j], a, d);
            use(j, a, d);
        }
    };
    switch (act) {
        case FC_ACT_GELU:
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
                const float4 f = exact_gelu(g[j], g[j + 1]);
                use(j, f.x, f.y);
                use(j + 1, f.z, f.w);
            }
            break;
        case FC_ACT_SILU: all(std::integral_constant<int, FC_ACT_SILU>()); break;
        case FC_ACT_GELU_TANH: all(std::integral_constant<int, FC_ACT_GELU_TANH>()); break;
        case FC_ACT_SIGMOID: all(std::integral_constant<int, FC_ACT_SIGMOID>()); break;
        case FC_ACT_RELU: all(std::integral_constant<int, FC_ACT_RELU>()); break;
        default: all(std::integral_constant<int, FC_ACT_NONE>());
    }
}
__device__ __forceinline__ void gate_values_exact(int act, float (&g)[32], const float (&u)[32]) {
    exact_acts(act, g, [&](int j, float a, float) { g[j] = a * u[j]; });
}
__device__ __forceinline__ void gate_back_values_exact(int act, float (&g)[32], float (&u)[32], float (&dh)[32]) {
    exact_acts(act, g, [&](int j, float a, float d) {
        const float h = a * u[j];
        g[j] = dh[j] * u[j] * d;
        u[j] = dh[j] * a;
        dh[j] = h;
    });
}

template <int ACT>
__device__ __forceinline__ void gate_values(float (&g)[32], const float (&u)[32]) {  // in: g, u; out: h in g
#pragma unroll
    for (int j = 0; j < 32; j += 2) {
        const float2 h = split(mul2(act_value2<ACT, false>(pair(g[j], g[j + 1])), pair(u[j], u[j + 1])));
        g[j] = h.x, g[j + 1] = h.y;
    }
}
template <int ACT>
__device__ __forceinline__ void gate_back_values(float (&g)[32], float (&u)[32], float (&dh)[32]) {
    // in: g, u, dh; out: dg, du, h
#pragma unroll
    for (int j = 0; j < 32; j += 2) {
        Pair a, d;
        act_both2<ACT, false>(pair(g[j], g[j + 1]), a, d);
        const Pair up = pair(u[j], u[j + 1]), e = pair(dh[j], dh[j + 1]);
        const float2 dg = split(mul2(mul2(e, up), d)), du = split(mul2(e, a)), h = split(mul2(a, up));
        g[j] = dg.x, g[j + 1] = dg.y;
        u[j] = du.x, u[j + 1] = du.y;
        dh[j] = h.x, dh[j + 1] = h.y;
    }
}

// OT: type of the operands.  T: of biases and of what FF_STORE stores.
template <typename OT, typename T, int PLANES, bool A_BY_K, bool B_BY_K, int KIND>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(FF_TC_THREADS, 1)
    ff_tc_kernel(const __grid_constant__ FfMaps maps, const FfTc P) {
    using R = Ring<PLANES, KIND>;
    constexpr bool kExact = PLANES == 3;
    constexpr int kMost = R::kMost;
    const int S = P.stages;
    const uint32_t b_bytes = (uint32_t)P.bn * 64;  // this CTA's share of B in a stage and plane
    const uint32_t kb_bytes = PLANES * (HALF_BYTES + b_bytes);
    const int kbs = PLANES == 1 ? P.kbs : 1;
    const uint32_t stage_bytes = kbs * kb_bytes;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem = (smem_u32(smem_raw) + 1023) & ~1023u;
    const uint32_t out_base = smem + R::kBytes;
    const uint32_t bars = out_base + R::kOut;
    auto bar_full = [&](int s) { return bars + 8 * s; };
    auto bar_empty = [&](int s) { return bars + 8 * (kMost + s); };
    auto bar_acc_full = [&](int a) { return bars + 8 * (2 * kMost + a); };
    auto bar_acc_empty = [&](int a) { return bars + 8 * (2 * kMost + 2 + a); };
    auto bar_small_empty = [&](int a) { return bars + 8 * (2 * kMost + 4 + a); };  // three planes: the small products' accumulators
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word;
    volatile int *abort_flag = &abort_word;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const uint32_t first = blockIdx.x >> 1, step = gridDim.x >> 1, items = P.items;
    const uint32_t tmem_cols = PLANES == 1 ? 2 * P.bn : 4 * P.bn;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(bar_full(s), 1);
            mbar_init(bar_empty(s), 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(bar_acc_full(a), 1);
            mbar_init(bar_acc_empty(a), 2 * EPI_WARPS);
            mbar_init(bar_small_empty(a), 2 * EPI_WARPS);
        }
        abort_word = 0;
        for (int i = 0; i < 2; ++i) {  // descriptors on their way before the first copy wants them
            asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.a[i]) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.b[i]) : "memory");
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(tmem_cols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    pdl_wait();
    pdl_next();

    auto decode = [&](uint32_t item, int &mt, int &nt, int &share) {
        const uint32_t rest = item / (uint32_t)P.n_tiles;
        nt = (int)(item - rest * P.n_tiles);
        share = (int)(P.splits > 1 ? rest / (uint32_t)P.live_tiles : 0);
        mt = P.skip + (int)(rest - share * P.live_tiles);
    };

    // Warps 0 and 1 run their loops with all lanes, on values that are the same in all of them, and one elected lane issues:
    // matrix instructions and copies take their operands from uniform registers, and in a branch of one lane each of them
    // costs some 150 clocks of moves.
    if (warp == 0) {
        int s = 0;
        uint32_t phase = 0;  // of the ring's current round
        bool ok = true;
        for (uint32_t item = first; item < items && ok; item += step) {
            int mt, nt, share;
            decode(item, mt, nt, share);
            const int dest = mt >= P.dest_tiles;
            const int m0 = (mt - dest * P.dest_tiles) * 256 + (int)rank * 128;
            const int n0 = KIND == FF_GATE ? nt * (P.bn / 2) : nt * P.bn + (int)rank * (P.bn / 2);
            const int lo = share * P.kb_share, hi = min(P.kb_total, lo + P.kb_share);
            for (int k_lo = lo; k_lo < hi; k_lo += kbs) {
                if (!mbar_wait(bar_empty(s), phase ^ 1, abort_flag, P.status)) {
                    ok = false;
                    break;
                }
                if (elect_one()) {
                    const int k_hi = min(hi, k_lo + kbs);
                    const uint32_t full = first_cta(bar_full(s));
                    if (rank == 0) mbar_expect_tx(bar_full(s), 2 * (k_hi - k_lo) * kb_bytes);
                    uint32_t a_at = smem + s * stage_bytes;
                    for (int kb = k_lo; kb < k_hi; ++kb, a_at += kb_bytes) {
                        const uint32_t b_at = a_at + PLANES * HALF_BYTES;
                        const int second = kb >= P.kb_first;
                        const int k0 = (second ? kb - P.kb_first : kb) * KB;
                        const CUtensorMap *am = &maps.a[A_BY_K ? second : dest];
                        const CUtensorMap *bm = &maps.b[KIND == FF_GATE ? (int)rank : second];
#pragma unroll
                        for (int z = 0; z < PLANES; ++z) {
                            const uint32_t az = a_at + z * HALF_BYTES, bz = b_at + z * b_bytes;
                            if (A_BY_K) {
                                pair_load(az, am, full, k0, m0, z);
                            } else {
#pragma unroll
                                for (int i = 0; i < 2; ++i) pair_load(az + i * KB * 128, am, full, m0 + 64 * i, k0, z);
                            }
                            if (B_BY_K) {
                                pair_load(bz, bm, full, k0, n0, z);
                            } else {
                                pair_load(bz, bm, full, n0, k0, z);
                                if (P.bn > 128) pair_load(bz + KB * 128, bm, full, n0 + 64, k0, z);
                            }
                        }
                    }
                }
                __syncwarp();
                if (++s == S) s = 0, phase ^= 1;
            }
        }
        // the other CTA's last releases have arrived here before this one may end
        for (int i = 0; i < S && ok; ++i) {
            ok = mbar_wait(bar_empty(s), phase ^ 1, abort_flag, P.status);
            if (++s == S) s = 0, phase ^= 1;
        }
    } else if (warp == 1) {
        if (rank == 0) {
            constexpr uint32_t type = std::is_same<OT, __nv_bfloat16>::value ? 1 : 0;
            const uint32_t idesc = (1u << 4) | (type << 7) | (type << 10) | ((A_BY_K ? 0u : 1u) << 15) | ((B_BY_K ? 0u : 1u) << 16) |
                                   ((uint32_t)(P.bn >> 3) << 17) | ((256u >> 4) << 24);
            int s = 0, t = 0, c = 0;  // stage; tiles and accumulators so far
            uint32_t phase = 0;
            bool ok = true;
            for (uint32_t item = first; item < items && ok; item += step, ++t) {
                int mt, nt, share;
                decode(item, mt, nt, share);
                const int lo = share * P.kb_share, hi = min(P.kb_total, lo + P.kb_share);
                const uint32_t small = tmem + (2 + (t & 1)) * P.bn;
                if (PLANES == 3) ok = mbar_wait(bar_small_empty(t & 1), ((t >> 1) & 1) ^ 1, abort_flag, P.status);
                for (int k_lo = lo; k_lo < hi && ok; k_lo += PLANES == 3 ? CHUNK : hi - lo, ++c) {
                    const int k_hi = PLANES == 3 ? min(hi, k_lo + CHUNK) : hi, acc = c & 1;
                    if (!mbar_wait(bar_acc_empty(acc), ((c >> 1) & 1) ^ 1, abort_flag, P.status)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t d = tmem + acc * P.bn;
                    for (int kb = k_lo; kb < k_hi; kb += kbs) {
                        if (!mbar_wait(bar_full(s), phase, abort_flag, P.status)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        if (elect_one()) {
                            uint32_t a_at = smem + s * stage_bytes;
                            const int upto = min(k_hi, kb + kbs);
                            for (int j = kb; j < upto; ++j, a_at += kb_bytes) {
                                const uint32_t b_at = a_at + PLANES * HALF_BYTES;
#pragma unroll
                                for (int k = 0; k < KB / 16; ++k) {  // 16 steps: 32 bytes along a row, or 16 rows
                                    auto a = [&](int z) { return operand<A_BY_K>(a_at + z * HALF_BYTES + k * (A_BY_K ? 32 : 2048)); };
                                    auto b = [&](int z) { return operand<B_BY_K>(b_at + z * b_bytes + k * (B_BY_K ? 32 : 2048)); };
                                    pair_mma(d, a(0), b(0), idesc, j > k_lo || k > 0);
                                    if (PLANES == 3) {
                                        pair_mma(small, a(0), b(1), idesc, j > lo || k > 0);
                                        pair_mma(small, a(1), b(0), idesc, 1);
                                        pair_mma(small, a(0), b(2), idesc, 1);
                                        pair_mma(small, a(2), b(0), idesc, 1);
                                        pair_mma(small, a(1), b(1), idesc, 1);
                                    }
                                }
                            }
                            pair_commit(bar_empty(s));
                            if (kb + kbs >= k_hi) pair_commit(bar_acc_full(acc));
                        }
                        __syncwarp();
                        if (++s == S) s = 0, phase ^= 1;
                    }
                }
            }
            // The last releases of both accumulators have arrived here, the other CTA's too, before this one may end: the waits
            // that a further use of each would begin with.
            for (int i = 0; i < 2 && ok; ++i, ++c, ++t) {
                ok = mbar_wait(bar_acc_empty(c & 1), ((c >> 1) & 1) ^ 1, abort_flag, P.status);
                if (PLANES == 3 && ok) ok = mbar_wait(bar_small_empty(t & 1), ((t >> 1) & 1) ^ 1, abort_flag, P.status);
            }
        }
    } else {
        const int quad = warp & 3, half = (warp - 2) >> 2;  // tensor memory lanes of this warp; every second column piece
        Outlet<R::kPieces> out = {out_base + (uint32_t)(warp - 2) * R::kPieces * PIECE, 0};
        float *turn = reinterpret_cast<float *>(smem_raw + (out.base - smem_u32(smem_raw)));
        const int cols = KIND == FF_GATE ? P.bn / 2 : P.bn;  // output columns of a tile
        int t = 0, c = 0;
        bool ok = true;
        for (uint32_t item = first; item < items && ok; item += step, ++t) {
            int mt, nt, share;
            decode(item, mt, nt, share);
            const int dest = mt >= P.dest_tiles;
            const int y = (mt - dest * P.dest_tiles) * 256 + (int)rank * 128 + quad * 32;  // the warp's first row
            const int row = y + lane;
            const uint32_t lanes = (uint32_t)(quad * 32) << 16;
            auto fetch = [&](uint32_t at, float (&v)[32], bool add) {
                uint32_t r[32];
                tmem_ld32(at + lanes, r);
                tmem_ld_wait();
                tmem_landed(r);
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] = add ? v[j] + __uint_as_float(r[j]) : __uint_as_float(r[j]);
            };
            auto saved = [&](int x, float (&g)[32], float (&u)[32]) {
                if (row >= P.m || x + 32 > P.n) {  // what is past the edge is computed with zeros and not stored
#pragma unroll
                    for (int j = 0; j < 32; ++j) g[j] = u[j] = 0.0f;
                }
                if (row < P.m && x < P.n) {
                    saved_row<false>(P, P.gate, y, lane, x, g);
                    saved_row<false>(P, P.up, y, lane, x, u);
                }
            };
            auto back = [&](float (&g)[32], float (&u)[32], float (&v)[32]) {  // in: g, u, dh; out: dg, du, h
                if constexpr (kExact) {
                    gate_back_values_exact(P.act, g, u, v);
                } else {
                    switch (P.act) {
                        case FC_ACT_RELU: gate_back_values<FC_ACT_RELU>(g, u, v); break;
                        case FC_ACT_SILU: gate_back_values<FC_ACT_SILU>(g, u, v); break;
                        case FC_ACT_GELU: gate_back_values<FC_ACT_GELU>(g, u, v); break;
                        case FC_ACT_GELU_TANH: gate_back_values<FC_ACT_GELU_TANH>(g, u, v); break;
                        case FC_ACT_SIGMOID: gate_back_values<FC_ACT_SIGMOID>(g, u, v); break;
                        default: gate_back_values<FC_ACT_NONE>(g, u, v);
                    }
                }
            };
            // 32 columns from x on: v the product; FF_GATE: v the gate's, u the up projection's
            auto emit = [&](int x, float (&v)[32], float (&u)[32]) {
                if (x >= P.n || y >= P.m) return;
                if (KIND == FF_GATE) {
                    add_bias<T>(P.bias0, P.bias_wide, x, P.n, v);
                    add_bias<T>(P.bias1, P.bias_wide, x, P.n, u);
                    if (P.gate != nullptr && row < P.m) {
                        saved_row<true>(P, P.gate, y, lane, x, v);
                        saved_row<true>(P, P.up, y, lane, x, u);
                    }
                    if constexpr (kExact) {
                        gate_values_exact(P.act, v, u);
                    } else {
                        switch (P.act) {
                            case FC_ACT_RELU: gate_values<FC_ACT_RELU>(v, u); break;
                            case FC_ACT_SILU: gate_values<FC_ACT_SILU>(v, u); break;
                            case FC_ACT_GELU: gate_values<FC_ACT_GELU>(v, u); break;
                            case FC_ACT_GELU_TANH: gate_values<FC_ACT_GELU_TANH>(v, u); break;
                            case FC_ACT_SIGMOID: gate_values<FC_ACT_SIGMOID>(v, u); break;
                            default: gate_values<FC_ACT_NONE>(v, u);
                        }
                    }
                    put_planes<OT, PLANES, R::kPieces>(out, &maps.c[0], v, x, y, lane);
                } else if (KIND == FF_GATE_BACK) {
                    float g[32];
                    saved(x, g, u);
                    back(g, u, v);
                    put_planes<OT, PLANES, R::kPieces>(out, &maps.c[0], g, x, y, lane);
                    put_planes<OT, PLANES, R::kPieces>(out, &maps.c[1], u, x, y, lane);
                    put_planes<OT, PLANES, R::kPieces>(out, &maps.c[2], v, x, y, lane);
                } else if (P.splits > 1) {  // [share][block of 32 rows][4 columns][row]
                    const int quads = (P.n + 3) / 4;
                    const size_t block = ((size_t)share * P.m_tiles + mt) * 8 + rank * 4 + quad;
                    float4 *ps = (float4 *)P.part + (block * quads + x / 4) * 32 + lane;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        if (x + 4 * j >= P.n) break;
                        ps[j * 32] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
                    }
                } else {
                    add_bias<T>(P.bias0, P.bias_wide, x, P.n, v);
                    T *c = (T *)(dest ? P.c1 : P.c0);
                    if (c != nullptr) {
                        store_block(turn, c, P.ldc, y, P.m, x, P.n, v, lane);
                    } else if constexpr (PLANES == 1) {
                        out.template put<OT>(&maps.c[dest], v, x, y, 0, lane);
                    }
                }
            };
            if constexpr (PLANES == 1) {
                const int acc = c & 1;
                float g[32], up[32];  // FF_GATE_BACK: the saved values, requested a piece ahead of their use
                if (KIND == FF_GATE_BACK) saved(nt * cols + half * 32, g, up);
                if (!mbar_wait(bar_acc_full(acc), (c >> 1) & 1, abort_flag, P.status)) break;
                ++c;
                tc_fence_after();
                const uint32_t d = tmem + acc * P.bn;
                for (int j = half * 32; KIND == FF_GATE_BACK && j < cols; j += 64) {
                    const int x = nt * cols + j;
                    if (x >= P.n || y >= P.m) break;
                    float v[32];
                    fetch(d + j, v, false);
                    back(g, up, v);
                    uint32_t w[3][16];
                    pack_row<OT>(g, w[0]);
                    pack_row<OT>(up, w[1]);
                    pack_row<OT>(v, w[2]);
                    if (j + 64 < cols) saved(x + 64, g, up);
                    if constexpr (KIND == FF_GATE_BACK) out.template put<3>(&maps.c[0], 1, w, x, y, 0, 0, lane);
                }
                for (int j = half * 32; KIND != FF_GATE_BACK && j < cols; j += 64) {
                    if (nt * cols + j >= P.n || y >= P.m) break;
                    float v[32], u[32];
                    fetch(d + j, v, false);
                    if (KIND == FF_GATE) fetch(d + cols + j, u, false);
                    emit(nt * cols + j, v, u);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) arrive_remote(first_cta(bar_acc_empty(acc)));
            } else {
                // bn = 128: this warp's two pieces, the gate's and the up projection's, or two neighbours
                const int p0 = KIND == FF_GATE ? half * 32 : half * 64, p1 = KIND == FF_GATE ? 64 + half * 32 : half * 64 + 32;
                const int lo = share * P.kb_share, hi = min(P.kb_total, lo + P.kb_share);
                float v[32], u[32];
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] = u[j] = 0.0f;
                for (int k = lo; k < hi; k += CHUNK, ++c) {
                    const int acc = c & 1;
                    ok = mbar_wait(bar_acc_full(acc), (c >> 1) & 1, abort_flag, P.status);
                    if (!ok) break;
                    tc_fence_after();
                    fetch(tmem + acc * P.bn + p0, v, true);
                    fetch(tmem + acc * P.bn + p1, u, true);
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) arrive_remote(first_cta(bar_acc_empty(acc)));
                }
                if (!ok) break;
                // the last accumulator's barrier stood for the small products too
                tc_fence_after();
                fetch(tmem + (2 + (t & 1)) * P.bn + p0, v, true);
                fetch(tmem + (2 + (t & 1)) * P.bn + p1, u, true);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) arrive_remote(first_cta(bar_small_empty(t & 1)));
                if (KIND == FF_GATE) {
                    emit(nt * cols + p0, v, u);
                } else {
                    float w[32];
#pragma unroll 1
                    for (int i = 0; i < 2; ++i) {
                        emit(nt * cols + (i ? p1 : p0), v, w);
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] = u[j];
                    }
                }
            }
        }
        asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }

    __syncthreads();
    if (*abort_flag) {  // let copies that are still in flight land before shared memory is released
        for (int i = 0; i < 64; ++i) __nanosleep(1000);
    }
    tc_fence_before();
    cluster_leave();
    if (warp == 1) {
        __syncwarp();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(tmem_cols) : "memory");
    }
}

// the shares of a split reduction, added in order; a thread has four columns of one row
template <typename T>
__global__ void __launch_bounds__(256) ff_tc_join_kernel(const FfTc P, T *c0, T *c1, int wide) {
    pdl_wait();
    pdl_next();
    const int quads = (P.n + 3) / 4, col_blocks = (quads + 3) / 4;
    const long long blocks = (long long)P.m_tiles * 8 * col_blocks * 4;  // of 8 rows x 4 quads: a warp each
    for (long long w = ((long long)blockIdx.x * 256 + threadIdx.x) >> 5; w < blocks; w += (long long)gridDim.x * 8) {
        const int lane = threadIdx.x & 31;
        const int r8 = (int)(w & 3);
        const long long rest = w >> 2;
        const int q = (int)(rest % col_blocks) * 4 + (lane >> 3);
        const long long block = rest / col_blocks;
        const int r = r8 * 8 + (lane & 7);
        const int mt = (int)(block >> 3), dest = mt >= P.dest_tiles;
        const int row = (mt - dest * P.dest_tiles) * 256 + (int)(block & 7) * 32 + r;
        T *c = dest ? c1 : c0;
        if (q >= quads || row >= P.m || c == nullptr) continue;
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int s = 0; s < P.splits; ++s) {
            const float4 f = ((const float4 *)P.part)[(((size_t)s * P.m_tiles * 8 + block) * quads + q) * 32 + r];
            v[0] += f.x, v[1] += f.y, v[2] += f.z, v[3] += f.w;
        }
        if (P.bias0)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (4 * q + i < P.n) v[i] += Elem<T>::load(((const T *)P.bias0)[4 * q + i]);
        T *to = c + (size_t)row * P.ldc + 4 * q;
        if (wide && 4 * q + 4 <= P.n) {
            Vec<T, 4> out;
            out.pack(v);
            out.store(to);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (4 * q + i < P.n) to[i] = Elem<T>::store(v[i]);
        }
    }
}

// ---- host -----------------------------------------------------------------------------------------------------------

// matrices of 16-bit values, rows `ld` apart, planes `plane` apart; box = box_cols x box_rows of one plane
int matrix_map(CUtensorMap *map, bool bf16, const void *base, long long cols, long long rows, int64_t ld, int planes, int64_t plane,
               int box_cols, int box_rows) {
    EncodeTiledFn enc;
    FC_PROPAGATE(get_encoder(&enc));
    cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)planes};
    cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)(planes > 1 ? plane : ld) * 2};
    cuuint32_t box[3] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows, 1};
    cuuint32_t estr[3] = {1, 1, 1};
    const CUresult r = enc(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void *>(base),
                           dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           box_cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    FC_REQUIRE(r == CUDA_SUCCESS, FC_ERR_CUDA, "cuTensorMapEncodeTiled failed with %d (%lld x %lld, rows %lld apart)", (int)r, rows, cols,
               (long long)ld);
    return FC_OK;
}

}  // namespace

// Tile width and shares of the reduction, by an estimate in SM clocks.  A k-block of 256 x 256 takes 512 clocks of the matrix pipe
// and is measured at 560, one of 128 columns at 275 and of 64 at 215 (two to a stage; 435 each with one); of three planes, 24
// instructions of 128 columns, at 1600.  Operand copies run at about 60 bytes a clock.  The first tile's latency and a last
// epilogue that nothing hides come to about 5000; a split result is written and read once more by every share (about
// 3000 bytes a clock, all SMs) and joined by a kernel of its own (about 4000).
struct FfTcPlan {
    int bn, splits;
};
static FfTcPlan ff_tc_plan(int planes, int kind, int dests, int m, int n, int kb_total, bool b_by_k) {
    const int pairs = 74;
    FfTcPlan best = {128, 1};
    double best_cost = 1e300;
    for (int bn = planes == 1 ? 256 : 128; bn >= (b_by_k && planes == 1 ? 64 : 128); bn /= 2) {
        const int cols = kind == FF_GATE ? bn / 2 : bn;
        const double tiles = (double)dests * ceil_div(m, 256) * ceil_div(n, cols);
        for (int s = 1; s <= (kind == FF_STORE ? 16 : 1); ++s) {
            if (s > 1 && kb_total / s < 4) break;
            const int share = (int)ceil_div(kb_total, s);
            if (s > 1 && (s - 1) * share >= kb_total) continue;  // the last share would be empty
            const double copies = planes * (16384.0 + 64.0 * bn) / 60.0, mma = planes == 3 ? 1600.0 : bn == 256 ? 560.0 : bn == 128 ? 275.0 : 215.0;
            const double waves = (double)ceil_div((size_t)(tiles * s), pairs);
            double cost = waves * share * (copies > mma ? copies : mma) + 5000.0;
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
    if (p.kind != FF_STORE || p.m == 0 || p.k == 0) return 0;
    int dests, m, kb_first, kb_total;
    tc_shape(p, &dests, &m, &kb_first, &kb_total);
    const FfTcPlan plan = ff_tc_plan(p.planes, p.kind, dests, m, p.n, kb_total, p.b_by_k);
    return plan.splits > 1 ? (size_t)plan.splits * dests * ceil_div(m, 256) * 256 * round_up(p.n, 4) : 0;
}

fc_ff_product_plan ff_tc_cut(const FfProduct &p) {
    int dests, m, kb_first, kb_total;
    tc_shape(p, &dests, &m, &kb_first, &kb_total);
    const FfTcPlan plan = ff_tc_plan(p.planes, p.kind, dests, m, p.n, kb_total, p.b_by_k);
    const int columns = p.kind == FF_GATE ? plan.bn / 2 : plan.bn;
    return fc_ff_product_plan{plan.bn, plan.splits, (int64_t)dests * (int64_t)ceil_div(m, 256) * (int64_t)ceil_div(p.n, columns)};
}

int launch_ff_tc(fc_context *ctx, const FfProduct &p) {
    int dests, m, kb_first, kb_total;
    tc_shape(p, &dests, &m, &kb_first, &kb_total);
    const FfTcPlan plan = ff_tc_plan(p.planes, p.kind, dests, m, p.n, kb_total, p.b_by_k);
    const int vec = 16 / (int)dtype_size(p.type);
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
    const long long items = (long long)P.live_tiles * P.n_tiles * P.splits;
    FC_REQUIRE(items < (1ll << 31) - 4096, FC_ERR_UNSUPPORTED, "product of %lld tiles", items);  // item + step stays in 32 bits
    P.items = (int)items;
    P.bias0 = p.bias0;
    P.bias1 = p.bias1;
    P.bias_wide = aligned16(p.bias0) && aligned16(p.bias1);
    P.gate = p.gate;
    P.up = p.up;
    P.saved_wide = aligned16(p.gate) && p.n % 4 == 0;
    P.ldc = p.ldc;
    P.part = p.part;
    P.status = ctx->d_status;
    // FF_STORE goes through TMA where the destination allows it.  A store is cut off at 16 bytes: where the columns end inside
    // such a piece, zeros would go to what lies behind them.  (In the workspace they may.)
    const bool c_wide = p.ldc % vec == 0 && aligned16(p.c0) && aligned16(p.c1);
    const bool by_copies = p.kind != FF_STORE || (p.planes == 1 && c_wide && p.n % vec == 0);
    if (!by_copies) {
        P.c0 = p.c0;
        P.c1 = p.c1;
    }

    FfMaps maps;
    memset(&maps, 0, sizeof maps);
    const bool bf16 = p.type != FC_DTYPE_F16;
    const uint8_t *a = (const uint8_t *)p.a;
    const int second = dests == 2 || p.b_split < p.k;
    for (int i = 0; i <= second; ++i) {  // A's columns (K-major: the reduction; MN-major: the rows of one destination)
        const int cols = p.a_by_k ? (i ? p.k - p.b_split : p.b_split) : m;
        FC_PROPAGATE(matrix_map(&maps.a[i], bf16, a + (i ? (size_t)p.a_skip * 2 : 0), cols, p.a_by_k ? p.m : p.k, p.lda, p.planes,
                                p.a_plane, 64, p.a_by_k ? 128 : KB));
    }
    const void *b[2] = {p.b0, p.b1};
    for (int i = 0; i < 2 && b[i]; ++i) {
        const int k = p.kind == FF_GATE ? p.k : i ? p.k - p.b_split : p.b_split;
        FC_PROPAGATE(p.b_by_k ? matrix_map(&maps.b[i], bf16, b[i], k, p.n, p.ldb, p.planes, p.b_plane, 64, plan.bn / 2)
                              : matrix_map(&maps.b[i], bf16, b[i], p.n, k, p.ldb, p.planes, p.b_plane, 64, KB));
    }
    if (by_copies && P.splits == 1) {
        const void *c[3] = {p.c0, p.c1, nullptr};
        if (p.kind == FF_GATE_BACK) {
            c[1] = (const uint8_t *)p.c0 + (size_t)p.a_skip * 2;
            c[2] = p.c1;
        }
        for (int i = 0; i < 3; ++i)
            if (c[i])
                FC_PROPAGATE(matrix_map(&maps.c[i], bf16, c[i], p.n, m, i == 2 ? p.ldc1 : p.ldc, p.kind == FF_STORE ? 1 : p.planes,
                                        i == 2 ? p.c1_plane : p.c_plane, 32, 32));
    }

    int pairs = ctx->sm_count / 2;
    if (pairs > P.items) pairs = P.items;
    auto run = [&](auto ot, auto t, auto planes) -> int {
        using OT = decltype(ot);
        using T = decltype(t);
        constexpr int PLANES = decltype(planes)::value;
        auto go = [&](auto kernel, auto ring) -> int {
            using R = decltype(ring);
            constexpr int SMEM = R::kSmem;
            P.kbs = PLANES == 1 && P.bn < 256 ? 2 : 1;
            const int room = R::kBytes / (P.kbs * ff_kb_bytes(PLANES, P.bn));
            P.stages = room < R::kMost ? room : R::kMost;
            FC_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
            FC_CHECK_CUDA(launch_early(kernel, dim3((unsigned)(2 * pairs)), dim3(FF_TC_THREADS), SMEM, ctx, maps, P));
            return FC_OK;
        };
        if (p.kind == FF_GATE) return go(ff_tc_kernel<OT, T, PLANES, true, true, FF_GATE>, Ring<PLANES, FF_GATE>());
        if (p.kind == FF_GATE_BACK) return go(ff_tc_kernel<OT, T, PLANES, true, false, FF_GATE_BACK>, Ring<PLANES, FF_GATE_BACK>());
        const Ring<PLANES, FF_STORE> ring;
        FC_PROPAGATE(!p.a_by_k  ? go(ff_tc_kernel<OT, T, PLANES, false, false, FF_STORE>, ring)
                     : p.b_by_k ? go(ff_tc_kernel<OT, T, PLANES, true, true, FF_STORE>, ring)
                                : go(ff_tc_kernel<OT, T, PLANES, true, false, FF_STORE>, ring));
        if (P.splits > 1) {
            long long blocks = ceil_div((size_t)P.m_tiles * 8 * 4 * ceil_div(p.n, 16), 8);
            if (blocks > 148 * 8) blocks = 148 * 8;
            FC_CHECK_CUDA(launch_early(ff_tc_join_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, ctx, P, (T *)p.c0, (T *)p.c1,
                                     (int)c_wide));
        }
        return FC_OK;
    };
    const std::integral_constant<int, 1> one;
    if (p.planes == 3) return run(__nv_bfloat16(), float(), std::integral_constant<int, 3>());
    return p.type == FC_DTYPE_BF16 ? run(__nv_bfloat16(), __nv_bfloat16(), one) : run(__half(), __half(), one);
}

}  // namespace fc
