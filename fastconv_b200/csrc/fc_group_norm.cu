// Group norm with an activation over channels-last maps, and its gradient.
//
//   mean, var over the pixels and channels of a group; xhat = (x - mean) / sqrt(var + eps); z = gamma xhat + beta
//   y = act(z);   dz = dy act'(z);   dgamma = sum dz xhat, dbeta = sum dz (over images and pixels)
//   dx = rstd (gamma dz - A - xhat B),  A = mean over the group of gamma dz,  B = mean of gamma dz xhat
//
// A thread owns a vector of neighbouring channels and walks over pixels.  Sums are fp32; the variance is taken around a
// value of the channel itself (the first one the thread sees) and joined pairwise by
//   M2 = M2a + M2b + (mean_a - mean_b)^2 na nb / (na + nb),
// so that a level far from zero costs no digits.  No atomics: results are the same from run to run.
//
// One kernel where a cluster's shared memory holds an image's block of channels (then a map is read once); otherwise
// three each way: sums of a chunk of pixels per channel, their join per group, the map itself.  The bound is memory: 64 x
// 28x28x512 fp32 takes 46 us (4.5 TB/s, 0.68 of the measured copy rate; two blocks of 100 KB to an SM leave memory waiting
// between a block's loads and its stores), 64 x 56x56x256 bf16 57 us forward and 124 us backward (3.6 and 2.5 TB/s): half of the
// issue slots are taken and memory is far from full, so a block's way from barrier to barrier is what it waits for.  In three
// kernels, whose joins have one block a group: one 224x224x128 bf16 image in 32 groups 34 us forward and 106 backward (floors
// 4 and 6), one 112x112x256 in 1 group 104 and 60 (2 and 3); element by element 64 x 56x56x256 bf16 at stride 259 176 and 369.
#include <cooperative_groups.h>

#include <numeric>
#include <type_traits>

#include "fc_last.cuh"

namespace fc {

namespace {

using namespace last;

constexpr int NORM_THREADS = 256;

struct NormShape {
    int batch, pixels, channels, groups, cpg;
    int64_t xs, ys;  // elements from one pixel to the next: of x and dx; of y and dy
    float eps;
    int cols, col_tiles;       // vectors of a column tile, column tiles
    int chunks, chunk_pixels;  // shares of an image's pixels
    int params_f32;            // gamma, beta, dgamma, dbeta are fp32; else of x's type
};

template <typename T>
__device__ __forceinline__ float param(const void *p, int c, int f32, float absent) {
    if (p == nullptr) return absent;
    return f32 ? ((const float *)p)[c] : Elem<T>::load(((const T *)p)[c]);
}

// the values of VEC channels from c on; c is a multiple of VEC
template <typename T, int VEC>
__device__ __forceinline__ void params(const void *p, int c, int f32, float absent, float (&v)[VEC]) {
    if (p == nullptr) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = absent;
    } else if (((uintptr_t)p & 15) != 0 || VEC == 1) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = param<T>(p, c + i, f32, absent);
    } else if (f32) {
        constexpr int N = VEC < 4 ? VEC : 4;
#pragma unroll
        for (int i = 0; i < VEC; i += N) {
            float w[N];
            Vec<float, N>::load((const float *)p + c + i).unpack(w);
#pragma unroll
            for (int j = 0; j < N; ++j) v[i + j] = w[j];
        }
    } else {
        Vec<T, VEC>::load((const T *)p + c).unpack(v);
    }
}
__device__ __forceinline__ float quick_inverse(float v) {  // to a unit in the last place
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// a / b for 0 <= a < 2^22, where by = 1 / b to a unit in the last place
__device__ __forceinline__ int quotient(int a, float by) { return (int)(((float)a + 0.5f) * by); }

// which image, share of pixels and columns a block has
struct Place {
    int img, chunk, p0, p1, col, row, rows, c0;
    bool live;
};
template <int VEC>
__device__ __forceinline__ Place place_of(const NormShape &s) {
    Place b;
    const long long id = blockIdx.x;
    const int tile = (int)(id % s.col_tiles);
    const long long rest = id / s.col_tiles;
    b.chunk = (int)(rest % s.chunks);
    b.img = (int)(rest / s.chunks);
    b.p0 = b.chunk * s.chunk_pixels;
    b.p1 = b.p0 + min(s.chunk_pixels, s.pixels - b.p0);
    b.rows = NORM_THREADS / s.cols;
    b.row = threadIdx.x / s.cols;
    b.col = threadIdx.x % s.cols;
    b.c0 = (tile * s.cols + b.col) * VEC;
    b.live = b.row < b.rows && b.c0 < s.channels;
    return b;
}

// use(p, load(p)) for the thread's pixels p, N loads before the first use: plain loads stay behind the stores before them
template <int N, typename L, typename U>
__device__ __forceinline__ void over_pixels(const Place &b, L &&load, U &&use) {
    int p = b.p0 + b.row;
    for (; p + (N - 1) * b.rows < b.p1; p += N * b.rows) {
        decltype(load(0)) v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = load(p + i * b.rows);
#pragma unroll
        for (int i = 0; i < N; ++i) use(p + i * b.rows, v[i]);
    }
    for (; p < b.p1; p += b.rows) use(p, load(p));
}

// joins (nb, mb, qb) into (na, ma, qa): count, mean, sum of squared deviations
__device__ __forceinline__ void join(float &na, float &ma, float &qa, float nb, float mb, float qb) {
    if (nb == 0.0f) return;
    const float n = na + nb, d = mb - ma, share = nb / n;
    qa += qb + d * d * na * share;
    ma += d * share;
    na = n;
}

__device__ __forceinline__ float block_sum(float v, float *scratch) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();  // scratch may still be read from an earlier sum
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    float t = 0.0f;
    for (int i = 0; i < (int)(blockDim.x >> 5); ++i) t += scratch[i];
    return t;
}

// ---- forward ----------------------------------------------------------------------------------------------------

// part[(img * chunks + chunk) * channels + c] = (mean, M2) of the channel over the chunk
template <typename T, int VEC>
__global__ void __launch_bounds__(NORM_THREADS) norm_part_kernel(const T *x, float2 *__restrict__ part,
                                                                const NormShape s) {
    __shared__ float2 stat[NORM_THREADS * VEC];
    pdl_wait();
    pdl_next();
    const Place b = place_of<VEC>(s);
    float k[VEC], sum[VEC], sq[VEC];
    int n = 0;
#pragma unroll
    for (int i = 0; i < VEC; ++i) k[i] = sum[i] = sq[i] = 0.0f;
    if (b.live) {
        const T *src = x + (size_t)b.img * s.pixels * s.xs + b.c0;
        int p = b.p0 + b.row;
        if (p < b.p1) Vec<T, VEC>::load(src + (size_t)p * s.xs).unpack(k);
#pragma unroll 4
        for (; p < b.p1; p += b.rows, ++n) {
            float f[VEC];
            Vec<T, VEC>::load(src + (size_t)p * s.xs).unpack(f);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float d = f[i] - k[i];
                sum[i] += d;
                sq[i] = fmaf(d, d, sq[i]);
            }
        }
    }
    const float inv = n > 0 ? 1.0f / n : 0.0f;
#pragma unroll
    for (int i = 0; i < VEC; ++i)
        stat[threadIdx.x * VEC + i] = make_float2(k[i] + sum[i] * inv, fmaxf(sq[i] - sum[i] * sum[i] * inv, 0.0f));
    __syncthreads();
    const int count = b.p1 - b.p0;
    const int first = b.c0 - b.col * VEC;  // the tile's first channel
    for (int i = threadIdx.x; i < s.cols * VEC && first + i < s.channels; i += NORM_THREADS) {
        float na = 0.0f, ma = 0.0f, qa = 0.0f;
        for (int r = 0; r < b.rows; ++r) {
            const float2 v = stat[r * s.cols * VEC + i];
            const int nr = count > r ? (count - r + b.rows - 1) / b.rows : 0;
            join(na, ma, qa, (float)nr, v.x, v.y);
        }
        part[((size_t)b.img * s.chunks + b.chunk) * s.channels + first + i] = make_float2(ma, qa);
    }
}

// mean and rstd of one group of one image from the chunks' sums
__global__ void __launch_bounds__(NORM_THREADS) norm_join_kernel(const float2 *part, float *__restrict__ mean,
                                                                float *__restrict__ rstd, const NormShape s) {
    __shared__ float scratch[NORM_THREADS / 32];
    pdl_wait();
    pdl_next();
    const int img = blockIdx.x / s.groups, g = blockIdx.x % s.groups;
    const float2 *src = part + (size_t)img * s.chunks * s.channels + g * s.cpg;
    const int items = s.chunks * s.cpg;
    const float inv = 1.0f / ((float)s.pixels * (float)s.cpg);
    const float level = src[0].x;  // means are added as distances from one of them, which costs no digits
    float a = 0.0f;
    for (int i = threadIdx.x; i < items; i += NORM_THREADS) {
        const int chunk = i / s.cpg, n = min(s.chunk_pixels, s.pixels - chunk * s.chunk_pixels);
        a = fmaf(src[(size_t)chunk * s.channels + i % s.cpg].x - level, (float)n, a);
    }
    const float m = fmaf(block_sum(a, scratch), inv, level);
    float q = 0.0f;
    for (int i = threadIdx.x; i < items; i += NORM_THREADS) {
        const int chunk = i / s.cpg, n = min(s.chunk_pixels, s.pixels - chunk * s.chunk_pixels);
        const float2 v = src[(size_t)chunk * s.channels + i % s.cpg];
        const float d = v.x - m;
        q += fmaf(d * d, (float)n, v.y);
    }
    const float var = block_sum(q, scratch) * inv;
    if (threadIdx.x == 0) {
        mean[blockIdx.x] = m;
        rstd[blockIdx.x] = 1.0f / sqrtf(var + s.eps);
    }
}

template <typename T, int VEC, int ACT>
__global__ void __launch_bounds__(NORM_THREADS) norm_apply_kernel(const T *x, const void *gamma,
                                                                 const void *beta, const float *mean,
                                                                 const float *rstd, T *__restrict__ y,
                                                                 const NormShape s) {
    constexpr bool kExact = std::is_same<T, float>::value;
    pdl_wait();
    pdl_next();
    const Place b = place_of<VEC>(s);
    if (!b.live) return;
    float m[VEC], a[VEC], o[VEC];
    params<T, VEC>(gamma, b.c0, s.params_f32, 1.0f, a);
    params<T, VEC>(beta, b.c0, s.params_f32, 0.0f, o);
    int g = b.c0 / s.cpg, j = b.c0 - g * s.cpg;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        m[i] = mean[b.img * s.groups + g];
        a[i] *= rstd[b.img * s.groups + g];
        if (++j == s.cpg) j = 0, ++g;
    }
    const T *src = x + (size_t)b.img * s.pixels * s.xs + b.c0;
    T *dst = y + (size_t)b.img * s.pixels * s.ys + b.c0;
    over_pixels<4>(
        b, [&](int p) { return Vec<T, VEC>::load(src + (size_t)p * s.xs); },
        [&](int p, const Vec<T, VEC> &v) {
            float f[VEC];
            v.unpack(f);
#pragma unroll
            for (int i = 0; i < VEC; ++i) f[i] = act_value<ACT, kExact>(fmaf(f[i] - m[i], a[i], o[i]));
            Vec<T, VEC> out;
            out.pack(f);
            out.store(dst + (size_t)p * s.ys);
        });
}

// ---- backward ---------------------------------------------------------------------------------------------------

// what a thread keeps of its channels in the backward pass
template <typename T, int VEC>
struct BackChannels {
    float m[VEC], r[VEC], g[VEC], o[VEC];
    __device__ __forceinline__ BackChannels(const void *gamma, const void *beta, const float *mean, const float *rstd, int img,
                                            int c0, const NormShape &s) {
        params<T, VEC>(gamma, c0, s.params_f32, 1.0f, g);
        params<T, VEC>(beta, c0, s.params_f32, 0.0f, o);
        int k = c0 / s.cpg, j = c0 - k * s.cpg;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            m[i] = mean[img * s.groups + k];
            r[i] = rstd[img * s.groups + k];
            if (++j == s.cpg) j = 0, ++k;
        }
    }
    // dz and xhat of channel i
    template <int ACT>
    __device__ __forceinline__ void at(int i, float x, float dy, float &dz, float &xhat) const {
        constexpr bool kExact = std::is_same<T, float>::value;
        xhat = (x - m[i]) * r[i];
        float a, d;
        act_both<ACT, kExact>(fmaf(xhat, g[i], o[i]), a, d);
        dz = dy * d;
    }
};

// part[(img * chunks + chunk) * channels + c] = (sum dz, sum dz xhat) of the channel over the chunk
template <typename T, int VEC, int ACT>
__global__ void __launch_bounds__(NORM_THREADS) norm_back_part_kernel(const T *dy, const T *x,
                                                                     const void *gamma,
                                                                     const void *beta,
                                                                     const float *mean,
                                                                     const float *rstd, float2 *__restrict__ part,
                                                                     const NormShape s) {
    __shared__ float2 stat[NORM_THREADS * VEC];
    pdl_wait();
    pdl_next();
    const Place b = place_of<VEC>(s);
    float s1[VEC], s2[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) s1[i] = s2[i] = 0.0f;
    if (b.live) {
        const BackChannels<T, VEC> ch(gamma, beta, mean, rstd, b.img, b.c0, s);
        const T *sx = x + (size_t)b.img * s.pixels * s.xs + b.c0, *sdy = dy + (size_t)b.img * s.pixels * s.ys + b.c0;
#pragma unroll 2
        for (int p = b.p0 + b.row; p < b.p1; p += b.rows) {
            float f[VEC], d[VEC];
            Vec<T, VEC>::load(sx + (size_t)p * s.xs).unpack(f);
            Vec<T, VEC>::load(sdy + (size_t)p * s.ys).unpack(d);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                float dz, xhat;
                ch.template at<ACT>(i, f[i], d[i], dz, xhat);
                s1[i] += dz;
                s2[i] = fmaf(dz, xhat, s2[i]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) stat[threadIdx.x * VEC + i] = make_float2(s1[i], s2[i]);
    __syncthreads();
    const int first = b.c0 - b.col * VEC;
    for (int i = threadIdx.x; i < s.cols * VEC && first + i < s.channels; i += NORM_THREADS) {
        float2 t = make_float2(0.0f, 0.0f);
        for (int r = 0; r < b.rows; ++r) {
            const float2 v = stat[r * s.cols * VEC + i];
            t.x += v.x;
            t.y += v.y;
        }
        part[((size_t)b.img * s.chunks + b.chunk) * s.channels + first + i] = t;
    }
}

// sums[img * channels + c] = the channel's (sum dz, sum dz xhat); ab[img * groups + g] = (A, B)
template <typename T>
__global__ void __launch_bounds__(NORM_THREADS) norm_back_join_kernel(const float2 *part,
                                                                     const void *gamma, float2 *__restrict__ sums,
                                                                     float2 *__restrict__ ab, const NormShape s) {
    __shared__ float scratch[NORM_THREADS / 32];
    pdl_wait();
    pdl_next();
    const int img = blockIdx.x / s.groups, g = blockIdx.x % s.groups;
    float a = 0.0f, q = 0.0f;
    for (int i = threadIdx.x; i < s.cpg; i += NORM_THREADS) {
        const int c = g * s.cpg + i;
        float2 t = make_float2(0.0f, 0.0f);
        const float2 *src = part + (size_t)img * s.chunks * s.channels + c;
        for (int k = 0; k < s.chunks; k += 16) {  // in order, sixteen loads at a time
            float2 v[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = k + j < s.chunks ? src[(size_t)(k + j) * s.channels] : make_float2(0.0f, 0.0f);
#pragma unroll
            for (int j = 0; j < 16; ++j) t.x += v[j].x, t.y += v[j].y;
        }
        sums[(size_t)img * s.channels + c] = t;
        const float w = param<T>(gamma, c, s.params_f32, 1.0f);
        a = fmaf(w, t.x, a);
        q = fmaf(w, t.y, q);
    }
    const float inv = 1.0f / ((float)s.pixels * (float)s.cpg);
    a = block_sum(a, scratch) * inv;
    q = block_sum(q, scratch) * inv;
    if (threadIdx.x == 0) ab[blockIdx.x] = make_float2(a, q);
}

template <typename T, int VEC, int ACT>
__global__ void __launch_bounds__(NORM_THREADS) norm_back_apply_kernel(const T *dy, const T *x,
                                                                      const void *gamma,
                                                                      const void *beta,
                                                                      const float *mean,
                                                                      const float *rstd,
                                                                      const float2 *ab, T *__restrict__ dx,
                                                                      const NormShape s) {
    pdl_wait();
    pdl_next();
    const Place b = place_of<VEC>(s);
    if (!b.live) return;
    const BackChannels<T, VEC> ch(gamma, beta, mean, rstd, b.img, b.c0, s);
    float2 t[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) t[i] = ab[b.img * s.groups + (b.c0 + i) / s.cpg];
    const T *sx = x + (size_t)b.img * s.pixels * s.xs + b.c0, *sdy = dy + (size_t)b.img * s.pixels * s.ys + b.c0;
    T *dst = dx + (size_t)b.img * s.pixels * s.xs + b.c0;
    struct Two {
        Vec<T, VEC> x, dy;
    };
    over_pixels<2>(
        b, [&](int p) { return Two{Vec<T, VEC>::load(sx + (size_t)p * s.xs), Vec<T, VEC>::load(sdy + (size_t)p * s.ys)}; },
        [&](int p, const Two &v) {
            float f[VEC], d[VEC];
            v.x.unpack(f);
            v.dy.unpack(d);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                float dz, xhat;
                ch.template at<ACT>(i, f[i], d[i], dz, xhat);
                f[i] = ch.r[i] * (fmaf(dz, ch.g[i], -t[i].x) - xhat * t[i].y);
            }
            Vec<T, VEC> out;
            out.pack(f);
            out.store(dst + (size_t)p * s.xs);
        });
}

// ---- one kernel: the map stays in shared memory between its statistics and its result ---------------------------------
//
// A cluster of 1 to 8 blocks has one image's block of channels (whole groups, whole vectors), each block a share of the
// pixels, which it copies to shared memory once; sums go through the blocks' shared memory.  A thread reads back only
// what it copied itself.
struct Fused {
    int cb, vectors, rows;  // channels and vectors of a block of channels; threads of one vector column
    int blocks;             // blocks of channels of an image
    int cluster, pc;        // blocks of a cluster; pixels of one block
    int groups, log_tg;     // groups of a block of channels; 2^log_tg threads add one up
    int width, per_row;     // channels of a slot of GroupSums, slots of a group in a row
    int part;               // pixels of one of the COPY_GROUPS parts that copies are waited for in
    float by_vectors, by_cpg;  // 1 / vectors, 1 / channels of a group
    size_t smem;
};
constexpr int FUSED_THREADS = 256, COPY_GROUPS = 4;

struct FusedPlace {
    int rank, cblk, img, np, row, col, c0;
    int g0, j0;  // group of the thread's first channel, counted in the block; that channel's place in it
    bool live;
    int64_t p0;
};
__device__ __forceinline__ FusedPlace fused_place(const NormShape &s, const Fused &f, int vec) {
    FusedPlace b;
    b.rank = blockIdx.x & (f.cluster - 1);  // clusters of 1, 2, 4 or 8
    b.cblk = blockIdx.x >> (f.cluster == 8 ? 3 : f.cluster >> 1);
    b.img = blockIdx.y;
    b.p0 = (int64_t)b.rank * f.pc;
    b.np = (int)max((int64_t)0, min((int64_t)f.pc, s.pixels - b.p0));
    b.row = quotient(threadIdx.x, f.by_vectors);
    b.col = threadIdx.x - b.row * f.vectors;
    b.live = b.row < f.rows;
    b.c0 = b.cblk * f.cb + b.col * vec;
    b.g0 = quotient(b.col * vec, f.by_cpg);
    b.j0 = b.col * vec - b.g0 * s.cpg;
    return b;
}
// use(i, group of the block that the thread's channel i belongs to)
template <int VEC, bool UNI, typename F>
__device__ __forceinline__ void over_groups(const NormShape &s, const FusedPlace &b, F &&use) {
    if (UNI) {  // a vector lies in one group
#pragma unroll
        for (int i = 0; i < VEC; ++i) use(i, b.g0);
        return;
    }
    int g = b.g0, j = b.j0;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        use(i, g);
        if (++j == s.cpg) j = 0, ++g;
    }
}
// The cluster's barrier.  Only threads that wrote what other blocks will read make their writes visible: the fence waits for
// everything that a thread has under way.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync(bool wrote) {
    if (wrote) asm volatile("fence.acq_rel.cluster;" ::: "memory");
    __syncwarp();
    cluster_arrive();
    cluster_wait();
}
__device__ __forceinline__ void copy16(void *to, const void *from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}
template <int N>
__device__ __forceinline__ void copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// f(begin, end) for each of the COPY_GROUPS parts of the block's pixels, once this thread's copies of the part have landed
template <typename F>
__device__ __forceinline__ void as_they_land(int np, int part, F &&f) {
    copies_wait<3>();
    f(0, min(np, part));
    copies_wait<2>();
    f(part, min(np, 2 * part));
    copies_wait<1>();
    f(2 * part, min(np, 3 * part));
    copies_wait<0>();
    f(3 * part, np);
}
template <typename F>
__device__ __forceinline__ void copy_parts(int np, int part, F &&f) {
#pragma unroll
    for (int i = 0; i < COPY_GROUPS; ++i) {
        f(i * part, i + 1 < COPY_GROUPS ? min(np, (i + 1) * part) : np);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
}

// Block-wide sums per group of what the threads hold per channel.  A thread hands in one value a slot, a slot being its whole
// vector where a group's channels are whole vectors, else a channel; a group's slots of all rows lie together, so that
// `tg` neighbouring threads (a power of two) add them without index arithmetic.
struct GroupSums {
    int groups, slots, log_tg;  // groups of the block; slots of a group in all rows; 2^log_tg threads to a group
    float *stat, *scratch, *red;  // [planes][rows * cb], [planes][8], [planes][groups]
    int plane, per_row;
    template <int VEC, bool UNI>
    __device__ __forceinline__ void put(const NormShape &s, const FusedPlace &b, int which, const float (&v)[VEC]) const {
        float *to = stat + which * plane + b.row * per_row;
        if (UNI) {
            float t = 0.0f;
#pragma unroll
            for (int i = 0; i < VEC; ++i) t += v[i];
            to[b.g0 * slots + b.j0 / VEC] = t;
        } else {
            int at = b.g0 * slots + b.j0, j = b.j0;
#pragma unroll
            for (int i = 0; i < VEC; ++i, ++at) {
                to[at] = v[i];
                if (++j == s.cpg) j = 0, at += slots - s.cpg;
            }
        }
    }
    // red[which * groups + g] for `planes` planes, complete and visible to the block on return
    template <int PLANES>
    __device__ __forceinline__ void add() const {
        __syncthreads();
        const int tg = 1 << log_tg, l = threadIdx.x & (tg - 1), lane = threadIdx.x & 31;
        for (int g = threadIdx.x >> log_tg; g < groups || tg > 1; g += FUSED_THREADS >> log_tg) {
            float t[PLANES];
#pragma unroll
            for (int k = 0; k < PLANES; ++k) {
                t[k] = 0.0f;
                if (g < groups)
                    for (int e = l; e < slots; e += tg) t[k] += stat[k * plane + g * slots + e];
                for (int o = min(tg, 32) / 2; o > 0; o >>= 1) t[k] += __shfl_xor_sync(0xffffffffu, t[k], o);
                if (tg > 32) {
                    if (lane == 0) scratch[k * 8 + (threadIdx.x >> 5)] = t[k];
                } else if (l == 0 && g < groups) {
                    red[k * groups + g] = t[k];
                }
            }
            if (tg > 1) break;  // then every group has its threads
        }
        __syncthreads();
        if (tg > 32) {
            if (threadIdx.x < groups) {
#pragma unroll
                for (int k = 0; k < PLANES; ++k) {
                    float t = 0.0f;
                    for (int w = 0; w < tg / 32; ++w) t += scratch[k * 8 + threadIdx.x * (tg / 32) + w];
                    red[k * groups + threadIdx.x] = t;
                }
            }
            __syncthreads();
        }
    }
};

// Squares are taken around one value of the group, its first in the block.  Where that turns out to be more than four standard
// deviations from the mean, they are taken once more around the mean, so the variance never loses more than some four of
// its 24 bits, however far the map is from zero.  The blocks of a cluster are joined by the means' distances.
template <typename T, int ACT, bool UNI>
__global__ void __launch_bounds__(FUSED_THREADS, UNI ? 4 : 2) norm_fused_kernel(const T *x, const void *gamma,
                                                                  const void *beta, T *__restrict__ y,
                                                                  float *__restrict__ mean, float *__restrict__ rstd,
                                                                  const NormShape s, const Fused f) {
    constexpr int VEC = 16 / sizeof(T);
    constexpr int OF_GROUP = UNI ? 1 : VEC / 2;  // pairs of what belongs to a group
    constexpr bool kExact = std::is_same<T, float>::value;
    using V = Vec<T, VEC>;
    namespace cg = cooperative_groups;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float scratch[2 * 8];
    V *data = (V *)smem;  // [pc][vectors]
    GroupSums gs;
    gs.groups = f.groups;
    gs.per_row = f.per_row;
    gs.slots = f.rows * f.per_row;
    gs.log_tg = f.log_tg;
    gs.plane = f.rows * f.cb;
    gs.stat = (float *)(data + (size_t)f.pc * f.vectors);
    gs.scratch = scratch;
    gs.red = gs.stat + 2 * gs.plane;
    float2 *share = (float2 *)(gs.red + 2 * gs.groups);  // [groups]: this block's (mean, M2)
    float2 *total = share + gs.groups;                   // [groups]: (mean, rstd)
    const FusedPlace b = fused_place(s, f, VEC);
    V *mine = data + b.row * f.vectors + b.col;
    const int hop = f.rows * f.vectors;
    pdl_wait();
    pdl_next();
    if (b.live) {
        const T *src = x + ((size_t)b.img * s.pixels + b.p0 + b.row) * s.xs + b.c0;
        const int64_t src_hop = f.rows * s.xs;
        V *to = mine;
        copy_parts(b.np, f.part, [&](int from, int upto) {
            for (int p = from + b.row; p < upto; p += f.rows, to += hop, src += src_hop) copy16(to, src);
        });
    }
    // this thread's group, where a thread sums one up in the end, and its level
    const T *corner = x + ((size_t)b.img * s.pixels + b.p0) * s.xs + b.cblk * f.cb;
    const bool sums = threadIdx.x < gs.groups;
    float level = sums ? Elem<T>::load(corner[threadIdx.x * s.cpg]) : 0.0f;
    float v[VEC], u[VEC];
    over_groups<VEC, UNI>(s, b, [&](int i, int g) { v[i] = b.live ? -Elem<T>::load(corner[g * s.cpg]) : 0.0f; });
    const float n_inv = quick_inverse((float)b.np * (float)s.cpg);
    auto deviations = [&](auto &&passes) {  // from -v; their sums and squares' sums to gs.red
        Pair from[OF_GROUP], sum[VEC / 2], sq[VEC / 2];
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) {
            if (i < OF_GROUP) from[i] = pair(v[2 * i], v[2 * i + 1]);
            sum[i] = sq[i] = 0;
        }
        const V *at = mine;
        passes([&](int begin, int end) {
            if (!b.live) return;
#pragma unroll 2
            for (int p = begin + b.row; p < end; p += f.rows, at += hop) {
                Pair q[VEC / 2];
                unpack_pairs(V::load(at), q);
#pragma unroll
                for (int i = 0; i < VEC / 2; ++i) {
                    const Pair d = add2(q[i], from[UNI ? 0 : i]);
                    sum[i] = add2(sum[i], d);
                    sq[i] = fma2(d, d, sq[i]);
                }
            }
        });
        if (b.live) {
            float a[VEC], c[VEC];
#pragma unroll
            for (int i = 0; i < VEC / 2; ++i) {
                a[2 * i] = split(sum[i]).x, a[2 * i + 1] = split(sum[i]).y;
                c[2 * i] = split(sq[i]).x, c[2 * i + 1] = split(sq[i]).y;
            }
            gs.put<VEC, UNI>(s, b, 0, a);
            gs.put<VEC, UNI>(s, b, 1, c);
        }
        gs.template add<2>();
    };
    deviations([&](auto &&part) { as_they_land(b.np, f.part, part); });
    float d = 0.0f, q = 0.0f;
    if (sums) {
        d = gs.red[threadIdx.x] * n_inv;
        q = fmaf(-d, gs.red[threadIdx.x], gs.red[gs.groups + threadIdx.x]);
        level += d;
        share[threadIdx.x] = make_float2(level, fmaxf(q, 0.0f));
    }
    if (__syncthreads_or(sums && !(gs.red[threadIdx.x] * d <= 16.0f * q) && d != 0.0f)) {
        over_groups<VEC, UNI>(s, b, [&](int i, int g) { v[i] = b.live ? -share[g].x : 0.0f; });
        deviations([&](auto &&part) { part(0, b.np); });
        if (sums) {
            d = gs.red[threadIdx.x] * n_inv;
            q = fmaf(-d, gs.red[threadIdx.x], gs.red[gs.groups + threadIdx.x]);
            share[threadIdx.x] = make_float2(level + d, fmaxf(q, 0.0f));
        }
    }
    if (f.cluster > 1)
        cluster_sync(sums);
    else
        __syncthreads();
    if (sums) {
        const int g = threadIdx.x;
        float2 w[8];
#pragma unroll
        for (int r = 0; r < 8; ++r)
            if (r < f.cluster) w[r] = f.cluster > 1 ? *cg::this_cluster().map_shared_rank(share + g, r) : share[g];
        const float all_inv = quick_inverse((float)s.pixels), m0 = w[0].x;
        float m = 0.0f, sq = 0.0f;
#pragma unroll
        for (int r = 0; r < 8; ++r)
            if (r < f.cluster) m = fmaf((float)min(f.pc, s.pixels - r * f.pc), w[r].x - m0, m);
        m = fmaf(m, all_inv, m0);
#pragma unroll
        for (int r = 0; r < 8; ++r)
            if (r < f.cluster) {
                const float e = w[r].x - m;
                sq = fmaf((float)min(f.pc, s.pixels - r * f.pc) * (float)s.cpg, e * e, sq + w[r].y);
            }
        const float rs = 1.0f / sqrtf(fmaf(sq, all_inv * quick_inverse((float)s.cpg), s.eps));
        total[g] = make_float2(m, rs);
        const int at = b.img * s.groups + b.cblk * gs.groups + g;
        if (b.rank == 0 && mean != nullptr) mean[at] = m;
        if (b.rank == 0 && rstd != nullptr) rstd[at] = rs;
    }
    __syncthreads();
    if (f.cluster > 1) cluster_arrive();
    if (b.live) {
        Pair m[OF_GROUP], a[VEC / 2], o[VEC / 2];
        float w[VEC];
        params<T, VEC>(gamma, b.c0, s.params_f32, 1.0f, u);
        params<T, VEC>(beta, b.c0, s.params_f32, 0.0f, v);
        over_groups<VEC, UNI>(s, b, [&](int i, int g) {
            const float2 t = total[g];
            u[i] *= t.y;
            w[i] = -t.x;
        });
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) {
            if (i < OF_GROUP) m[i] = pair(w[2 * i], w[2 * i + 1]);
            a[i] = pair(u[2 * i], u[2 * i + 1]);
            o[i] = pair(v[2 * i], v[2 * i + 1]);
        }
        T *dst = y + ((size_t)b.img * s.pixels + b.p0 + b.row) * s.ys + b.c0;
        const int64_t dst_hop = f.rows * s.ys;
        const V *at = mine;
#pragma unroll 2
        for (int p = b.row; p < b.np; p += f.rows, at += hop, dst += dst_hop) {
            Pair q[VEC / 2];
            unpack_pairs(V::load(at), q);
#pragma unroll
            for (int i = 0; i < VEC / 2; ++i)
                q[i] = act_value2<ACT, kExact>(fma2(add2(q[i], m[UNI ? 0 : i]), a[i], o[i]));
            V out;
            pack_pairs(out, q);
            out.store(dst);
        }
    }
    if (f.cluster > 1) cluster_wait();  // the others have read this block's sums
}

// sums[img * channels + c]: the image's (sum dz, sum dz xhat)
template <typename T, int ACT, bool UNI>
__global__ void __launch_bounds__(FUSED_THREADS, UNI ? 4 : 2) norm_back_fused_kernel(const T *dy, const T *x,
                                                                       const void *gamma,
                                                                       const void *beta,
                                                                       const float *mean,
                                                                       const float *rstd, T *__restrict__ dx,
                                                                       float2 *__restrict__ sums, const NormShape s, const Fused f) {
    constexpr int VEC = 16 / sizeof(T);
    using V = Vec<T, VEC>;
    namespace cg = cooperative_groups;
    extern __shared__ __align__(16) uint8_t smem[];
    V *xs = (V *)smem, *ds = xs + (size_t)f.pc * f.vectors;    // [pc][vectors] each
    float2 *stat = (float2 *)(ds + (size_t)f.pc * f.vectors);  // [rows][cb]: a thread's sums
    float2 *share = stat + f.rows * f.cb;                      // [cb]: this block's
    float2 *total = share + f.cb;                              // [cb]: the image's
    float2 *ab = total + f.cb;                                 // [groups of the block]
    const FusedPlace b = fused_place(s, f, VEC);
    const int hop = f.rows * f.vectors, start = b.row * f.vectors + b.col;
    pdl_wait();
    pdl_next();
    if (b.live) {
        const T *sx = x + ((size_t)b.img * s.pixels + b.p0 + b.row) * s.xs + b.c0;
        const T *sd = dy + ((size_t)b.img * s.pixels + b.p0 + b.row) * s.ys + b.c0;
        const int64_t x_hop = f.rows * s.xs, d_hop = f.rows * s.ys;
        int at = start;
        copy_parts(b.np, f.part, [&](int from, int upto) {
            for (int p = from + b.row; p < upto; p += f.rows, at += hop, sx += x_hop, sd += d_hop) {
                copy16(xs + at, sx);
                copy16(ds + at, sd);
            }
        });
    }
    constexpr bool kExact = std::is_same<T, float>::value;
    // With xm = x - mean:  z = (gamma rstd) xm + beta,  dx = (gamma rstd) dz - rstd A - xm (rstd^2 B).  What belongs to a group
    // is one pair where a vector lies in one (UNI).
    constexpr int PAIRS = VEC / 2, OF_GROUP = UNI ? 1 : PAIRS;
    Pair m[OF_GROUP], gr[PAIRS], bt[PAIRS];  // -mean, gamma rstd, beta
    if (b.live) {
        float fm[VEC], fg[VEC], fb[VEC];
        params<T, VEC>(gamma, b.c0, s.params_f32, 1.0f, fg);
        params<T, VEC>(beta, b.c0, s.params_f32, 0.0f, fb);
        over_groups<VEC, UNI>(s, b, [&](int i, int g) {
            const int at = b.img * s.groups + b.cblk * f.groups + g;
            fm[i] = -mean[at];
            fg[i] *= rstd[at];
        });
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
            if (i < OF_GROUP) m[i] = pair(fm[2 * i], fm[2 * i + 1]);
            gr[i] = pair(fg[2 * i], fg[2 * i + 1]);
            bt[i] = pair(fb[2 * i], fb[2 * i + 1]);
        }
    }
    // dz and x - mean of a pair of channels
    auto one = [&](int i, Pair v, Pair d, Pair &dz, Pair &xm) {
        xm = add2(v, m[UNI ? 0 : i]);
        Pair a, slope;
        act_both2<ACT, kExact>(fma2(xm, gr[i], bt[i]), a, slope);
        dz = mul2(d, slope);
    };
    {
        Pair s1[VEC / 2], s2[VEC / 2];
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) s1[i] = s2[i] = 0;
        int at = start;
        as_they_land(b.np, f.part, [&](int from, int upto) {
            if (!b.live) return;
#pragma unroll 1
            for (int p = from + b.row; p < upto; p += f.rows, at += hop) {
                Pair v[VEC / 2], d[VEC / 2];
                unpack_pairs(V::load(xs + at), v);
                unpack_pairs(V::load(ds + at), d);
#pragma unroll
                for (int i = 0; i < VEC / 2; ++i) {
                    Pair dz, xm;
                    one(i, v[i], d[i], dz, xm);
                    s1[i] = add2(s1[i], dz);
                    s2[i] = fma2(dz, xm, s2[i]);
                }
            }
        });
        if (b.live) {
            float fr[VEC];
            over_groups<VEC, UNI>(s, b, [&](int i, int g) { fr[i] = rstd[b.img * s.groups + b.cblk * f.groups + g]; });
#pragma unroll
            for (int i = 0; i < VEC / 2; ++i) {
                const float2 p = split(s1[i]), q = split(s2[i]);
                stat[b.row * f.cb + b.col * VEC + 2 * i] = make_float2(p.x, q.x * fr[2 * i]);
                stat[b.row * f.cb + b.col * VEC + 2 * i + 1] = make_float2(p.y, q.y * fr[2 * i + 1]);
            }
        }
    }
    __syncthreads();
    // a channel's rows are added by FUSED_THREADS / cb threads, and those by the first
    const int parts = f.cb >= FUSED_THREADS ? 1 : min(f.rows, FUSED_THREADS / f.cb);
    if (parts > 1) {
        const int c = threadIdx.x % f.cb, part = threadIdx.x / f.cb;
        if (part < parts) {
            float2 t = make_float2(0.0f, 0.0f);
            for (int r = part; r < f.rows; r += parts) {
                const float2 v = stat[r * f.cb + c];
                t.x += v.x;
                t.y += v.y;
            }
            stat[part * f.cb + c] = t;  // nobody else reads row `part` of this channel
        }
        __syncthreads();
    }
    for (int c = threadIdx.x; c < f.cb; c += FUSED_THREADS) {
        float2 t = make_float2(0.0f, 0.0f);
        for (int r = 0; r < (parts > 1 ? parts : f.rows); ++r) {
            const float2 v = stat[r * f.cb + c];
            t.x += v.x;
            t.y += v.y;
        }
        share[c] = t;
    }
    if (f.cluster > 1)
        cluster_sync(threadIdx.x < f.cb);
    else
        __syncthreads();
    for (int c = threadIdx.x; c < f.cb; c += FUSED_THREADS) {
        float2 t = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int r = 0; r < 8; ++r)
            if (r < f.cluster) {
                const float2 v = f.cluster > 1 ? *cg::this_cluster().map_shared_rank(share + c, r) : share[c];
                t.x += v.x;
                t.y += v.y;
            }
        total[c] = t;
        if (b.rank == 0) sums[(size_t)b.img * s.channels + b.cblk * f.cb + c] = t;
    }
    __syncthreads();
    if (f.cluster > 1) cluster_arrive();
    if (dx != nullptr) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, groups = f.cb / s.cpg;
        const float inv = quick_inverse((float)s.pixels * (float)s.cpg);
        for (int g = warp; g < groups; g += FUSED_THREADS / 32) {
            float a = 0.0f, q = 0.0f;
            for (int i = lane; i < s.cpg; i += 32) {
                const int c = g * s.cpg + i;
                const float w = param<T>(gamma, b.cblk * f.cb + c, s.params_f32, 1.0f);
                a = fmaf(w, total[c].x, a);
                q = fmaf(w, total[c].y, q);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                a += __shfl_xor_sync(0xffffffffu, a, o);
                q += __shfl_xor_sync(0xffffffffu, q, o);
            }
            if (lane == 0) {
                const float r = rstd[b.img * s.groups + b.cblk * f.groups + g];
                ab[g] = make_float2(-a * inv * r, -q * inv * r * r);
            }
        }
        __syncthreads();
        if (b.live) {
            float fa[VEC], fb[VEC];
            over_groups<VEC, UNI>(s, b, [&](int i, int g) { fa[i] = ab[g].x, fb[i] = ab[g].y; });
            Pair ta[OF_GROUP], tb[OF_GROUP];
#pragma unroll
            for (int i = 0; i < OF_GROUP; ++i) ta[i] = pair(fa[2 * i], fa[2 * i + 1]), tb[i] = pair(fb[2 * i], fb[2 * i + 1]);
            T *dst = dx + ((size_t)b.img * s.pixels + b.p0 + b.row) * s.xs + b.c0;
            const int64_t dst_hop = f.rows * s.xs;
            int at = start;
#pragma unroll 1
            for (int p = b.row; p < b.np; p += f.rows, at += hop, dst += dst_hop) {
                Pair v[VEC / 2], d[VEC / 2];
                unpack_pairs(V::load(xs + at), v);
                unpack_pairs(V::load(ds + at), d);
#pragma unroll
                for (int i = 0; i < VEC / 2; ++i) {
                    Pair dz, xm;
                    one(i, v[i], d[i], dz, xm);
                    v[i] = fma2(dz, gr[i], fma2(xm, tb[UNI ? 0 : i], ta[UNI ? 0 : i]));
                }
                V out;
                pack_pairs(out, v);
                out.store(dst);
            }
        }
    }
    if (f.cluster > 1) cluster_wait();
}

// dgamma[c], dbeta[c]: the images' sums.  32 channels x 8 shares of the images to a block; the shares are added in order.
template <typename T>
__global__ void __launch_bounds__(NORM_THREADS) norm_back_params_kernel(const float2 *sums, void *dgamma, void *dbeta,
                                                                       const NormShape s) {
    __shared__ float2 shares[8][32];
    pdl_wait();
    pdl_next();
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, c = blockIdx.x * 32 + tx;
    float2 t = make_float2(0.0f, 0.0f);
    if (c < s.channels)
#pragma unroll 4
        for (int n = ty; n < s.batch; n += 8) {
            const float2 v = sums[(size_t)n * s.channels + c];
            t.x += v.x;
            t.y += v.y;
        }
    shares[ty][tx] = t;
    __syncthreads();
    if (ty > 0 || c >= s.channels) return;
#pragma unroll
    for (int i = 1; i < 8; ++i) {
        t.x += shares[i][tx].x;
        t.y += shares[i][tx].y;
    }
    if (s.params_f32) {
        if (dgamma) ((float *)dgamma)[c] = t.y;
        if (dbeta) ((float *)dbeta)[c] = t.x;
    } else {
        if (dgamma) ((T *)dgamma)[c] = Elem<T>::store(t.y);
        if (dbeta) ((T *)dbeta)[c] = Elem<T>::store(t.x);
    }
}

// ---- host -------------------------------------------------------------------------------------------------------

int norm_shape(const fc_group_norm_desc *d, NormShape *s) {
    FC_REQUIRE(d != nullptr, FC_ERR_INVALID_ARG, "descriptor is NULL");
    FC_REQUIRE(d->batch >= 0 && d->pixels > 0 && d->channels > 0 && d->groups > 0, FC_ERR_INVALID_ARG,
               "batch %d, pixels %d, channels %d, groups %d", d->batch, d->pixels, d->channels, d->groups);
    FC_REQUIRE(d->pixels < (1 << 30) && d->channels <= (1 << 20), FC_ERR_UNSUPPORTED, "%d pixels of %d channels", d->pixels, d->channels);
    FC_REQUIRE(d->channels % d->groups == 0, FC_ERR_INVALID_ARG, "%d groups do not divide %d channels", d->groups, d->channels);
    FC_REQUIRE(dtype_ok(d->type), FC_ERR_INVALID_ARG, "unknown element type %d", d->type);
    FC_REQUIRE(d->param_type == FC_DTYPE_F32 || d->param_type == d->type, FC_ERR_INVALID_ARG,
               "parameters are fp32 or of the map's type, not of type %d", d->param_type);
    FC_REQUIRE(act_ok(d->act), FC_ERR_INVALID_ARG, "unknown activation %d", d->act);
    FC_REQUIRE(d->eps >= 0.0f, FC_ERR_INVALID_ARG, "eps is negative or not a number");
    const int64_t xs = d->x_stride ? d->x_stride : d->channels, ys = d->y_stride ? d->y_stride : d->channels;
    FC_REQUIRE(xs >= d->channels && ys >= d->channels, FC_ERR_INVALID_ARG, "pixel strides %lld, %lld are less than the %d channels",
               (long long)xs, (long long)ys, d->channels);
    FC_REQUIRE((long long)d->batch * d->groups < (1ll << 31), FC_ERR_UNSUPPORTED, "%d images of %d groups", d->batch, d->groups);
    *s = NormShape{d->batch, d->pixels, d->channels, d->groups, d->channels / d->groups, xs, ys, d->eps, 0, 0, 0, 0,
                   d->param_type == FC_DTYPE_F32};
    return FC_OK;
}

// Columns and shares of pixels for vectors of `vec` channels: about eight blocks to an SM, at least four pixels to a thread.
void norm_split(NormShape *s, int vec) {
    const int vectors = (s->channels + vec - 1) / vec;
    s->col_tiles = (vectors + NORM_THREADS - 1) / NORM_THREADS;
    s->cols = (vectors + s->col_tiles - 1) / s->col_tiles;
    const int rows = NORM_THREADS / s->cols;
    const long long others = (long long)s->batch * s->col_tiles;
    long long chunks = others > 0 ? (148 * 8 + others - 1) / others : 1;
    const long long most = ((long long)s->pixels + 4 * rows - 1) / (4 * rows);
    if (chunks > most) chunks = most;
    if (chunks < 1) chunks = 1;
    s->chunk_pixels = (int)(((long long)s->pixels + chunks - 1) / chunks);
    s->chunks = (s->pixels + s->chunk_pixels - 1) / s->chunk_pixels;
}

// The one-kernel form for vectors of 16 bytes, or false where an image's smallest block of channels is more than eight
// blocks' shared memory holds.  Chosen by an estimate in nanoseconds: `waves` rounds of blocks of about 2.5 us, in a cluster 350
// ns a block more, which several blocks of an SM overlap; 0.7 us of instructions that a block takes whatever it holds; and
// the bytes at 6500 a nanosecond, less where the runs of a pixel are shorter than the 32 bytes that memory moves or where
// there are fewer blocks than SMs.  64 x 56x56x256 bf16 forward: runs of 64 bytes in clusters of 4 57 us, of 32 in 2 60, of 128 in
// 8 63, of 64 in 8 71, of 32 in one block 79; in three kernels 103 (backward 124 against 187).
bool fused_plan(const NormShape &s, int esize, bool backward, Fused *best) {
    const int vec = 16 / esize, arrays = backward ? 2 : 1;
    if (s.channels % vec || s.batch > 65535) return false;
    const int unit = std::lcm(s.cpg, vec);  // divides channels, as both do
    double best_cost = 1e300;
    const double bytes = (double)s.batch * s.pixels * s.channels * esize * (arrays + 1);
    for (int k = 1; k * unit <= s.channels; ++k) {
        const int cb = k * unit, vectors = cb / vec, run = cb * esize;
        if (vectors > FUSED_THREADS || cb / s.cpg > FUSED_THREADS) break;
        if (s.channels % cb) continue;
        for (int cluster = 1; cluster <= 8; cluster *= 2) {
            Fused f = {cb, vectors, FUSED_THREADS / vectors, s.channels / cb, cluster, (s.pixels + cluster - 1) / cluster, cb / s.cpg};
            f.width = s.cpg % vec ? 1 : vec;
            f.per_row = s.cpg / f.width;
            f.part = (int)ceil_div(ceil_div(f.pc, f.rows), COPY_GROUPS) * f.rows;
            f.by_vectors = 1.0f / vectors;
            f.by_cpg = 1.0f / s.cpg;
            if (cluster > 1 && (long long)f.pc * (cluster - 1) >= s.pixels) break;  // a block would have no pixels
            f.smem = (size_t)f.pc * run * arrays + ((size_t)f.rows * cb + 3 * cb) * sizeof(float2);
            while ((2 << f.log_tg) * f.groups <= FUSED_THREADS) ++f.log_tg;
            if (f.smem > 200 * 1024) continue;
            const double blocks = (double)s.batch * f.blocks * cluster;
            double per_sm = 220.0 * 1024 / (f.smem + 1024.0);
            per_sm = per_sm > 6 ? 6 : (double)(int)per_sm;
            const double waves = (double)(long long)((blocks + 148 * per_sm - 1) / (148 * per_sm));
            const double eff = (run >= 64 ? 1.0 : run >= 32 ? 0.95 : 0.6) * (blocks < 148 ? blocks / 148 : 1.0) *
                               (per_sm < 2 ? 0.75 : 1.0);
            const double cost = waves * (2500.0 + (cluster > 1 ? 350.0 * cluster : 0.0)) / (waves > 1 ? per_sm : 1.0) + blocks / 148 * 700.0 +
                                bytes / (6500.0 * eff);
            if (cost < best_cost) {
                best_cost = cost;
                *best = f;
            }
        }
    }
    return best_cost < 1e300;
}

struct NormWork {
    float2 *part, *sums, *ab;
    float *mean, *rstd;
    size_t bytes;
};

NormWork norm_carve(const NormShape &s, void *base, bool backward) {
    Carver c = {(uint8_t *)base, 0};
    NormWork w = {};
    w.part = c.take<float2>((size_t)s.batch * s.chunks * s.channels);
    if (backward) {
        w.sums = c.take<float2>((size_t)s.batch * s.channels);
        w.ab = c.take<float2>((size_t)s.batch * s.groups);
    } else {
        w.mean = c.take<float>((size_t)s.batch * s.groups);
        w.rstd = c.take<float>((size_t)s.batch * s.groups);
    }
    w.bytes = c.used;
    return w;
}

// vectors of 16 bytes where every address and stride allows them, single elements otherwise
template <typename T>
bool wide_ok(const NormShape &s, std::initializer_list<const void *> maps) {
    const int vec = 16 / sizeof(T);
    if (s.channels % vec || s.xs % vec || s.ys % vec) return false;
    for (const void *p : maps)
        if (!aligned16(p)) return false;
    return true;
}

// f(T(), integral_constant<int, elements of a vector>): 16 bytes, or 1 element where channels, strides or addresses do not fit
template <typename F>
int with_vectors(const NormShape &s, int type, std::initializer_list<const void *> maps, F &&f) {
    return with_type(type, [&](auto t) -> int {
        using T = decltype(t);
        if (wide_ok<T>(s, maps)) return f(t, std::integral_constant<int, 16 / (int)sizeof(T)>());
        return f(t, std::integral_constant<int, 1>());
    });
}

int check_maps(const fc_group_norm_desc *d, std::initializer_list<const void *> maps, std::initializer_list<const void *> params,
               const float *mean, const float *rstd) {
    for (const void *p : maps) {
        FC_REQUIRE(p != nullptr, FC_ERR_INVALID_ARG, "NULL map");
        FC_REQUIRE((uintptr_t)p % dtype_size(d->type) == 0, FC_ERR_INVALID_ARG, "a map's address is no multiple of its element size");
    }
    for (const void *p : params)
        FC_REQUIRE((uintptr_t)p % dtype_size(d->param_type) == 0, FC_ERR_INVALID_ARG,
                   "a parameter's address is no multiple of its element size");
    FC_REQUIRE((uintptr_t)mean % 4 == 0 && (uintptr_t)rstd % 4 == 0, FC_ERR_INVALID_ARG, "an address of mean or rstd is no multiple of 4");
    return FC_OK;
}

}  // namespace

}  // namespace fc

using namespace fc;

extern "C" {

int fc_group_norm_workspace(const fc_group_norm_desc *desc, size_t *forward_bytes, size_t *backward_bytes) {
    NormShape s;
    FC_PROPAGATE(norm_shape(desc, &s));
    size_t most[2] = {0, 0};
    for (int wide = 0; wide < 2; ++wide) {  // either width may be chosen, by the addresses of the call
        norm_split(&s, wide ? 16 / (int)dtype_size(desc->type) : 1);
        for (int b = 0; b < 2; ++b) {
            const size_t n = norm_carve(s, nullptr, b == 1).bytes;
            if (n > most[b]) most[b] = n;
        }
    }
    if (forward_bytes) *forward_bytes = most[0];
    if (backward_bytes) *backward_bytes = most[1];
    return FC_OK;
}

int fc_group_norm_forward(fc_context *ctx, const fc_group_norm_desc *desc, const void *d_x, const void *d_gamma,
                          const void *d_beta, void *d_y, float *d_mean, float *d_rstd, void *d_workspace,
                          size_t workspace_bytes) {
    FC_REQUIRE(ctx != nullptr, FC_ERR_INVALID_ARG, "context is NULL");
    NormShape s;
    FC_PROPAGATE(norm_shape(desc, &s));
    if (s.batch == 0) return FC_OK;
    FC_PROPAGATE(check_maps(desc, {d_x, d_y}, {d_gamma, d_beta}, d_mean, d_rstd));
    FC_PROPAGATE(check_outputs({d_y, d_mean, d_rstd, d_workspace}, {d_x, d_gamma, d_beta}));
    size_t need;
    FC_PROPAGATE(fc_group_norm_workspace(desc, &need, nullptr));
    FC_REQUIRE(d_workspace != nullptr && aligned16(d_workspace) && workspace_bytes >= need, FC_ERR_INVALID_ARG,
               "workspace of %zu bytes at %p: %zu are needed, on a 16-byte boundary", workspace_bytes, d_workspace, need);
    DeviceScope dev(ctx->device);
    FC_CHECK_CUDA(dev.status());
    return with_vectors(s, desc->type, {d_x, d_y}, [&](auto t, auto v) -> int {
        using T = decltype(t);
        constexpr int VEC = decltype(v)::value;
        Fused f;
        if constexpr (VEC > 1) {
            if (fused_plan(s, sizeof(T), false, &f))
                return with_act(desc->act, [&](auto a) -> int {
                    constexpr int A = decltype(a)::value;
                    auto kernel = f.width > 1 ? norm_fused_kernel<T, A, true> : norm_fused_kernel<T, A, false>;
                    FC_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024));
                    FC_CHECK_CUDA(launch_clusters(kernel, dim3(f.blocks * f.cluster, s.batch), FUSED_THREADS, f.cluster, f.smem,
                                                  ctx, (const T *)d_x, d_gamma, d_beta, (T *)d_y, d_mean, d_rstd, s, f));
                    return FC_OK;
                });
        }
        norm_split(&s, VEC);
        const long long blocks = (long long)s.batch * s.chunks * s.col_tiles;
        FC_REQUIRE(blocks < (1ll << 31), FC_ERR_UNSUPPORTED, "%lld blocks", blocks);
        const NormWork w = norm_carve(s, d_workspace, false);
        float *mean = d_mean ? d_mean : w.mean, *rstd = d_rstd ? d_rstd : w.rstd;
        FC_CHECK_CUDA(launch_early(norm_part_kernel<T, VEC>, dim3((unsigned)blocks), dim3(NORM_THREADS), 0, ctx, (const T *)d_x,
                                 w.part, s));
        FC_CHECK_CUDA(launch_early(norm_join_kernel, dim3(s.batch * s.groups), dim3(NORM_THREADS), 0, ctx,
                                 (const float2 *)w.part, mean, rstd, s));
        return with_act(desc->act, [&](auto a) -> int {
            FC_CHECK_CUDA(launch_early(norm_apply_kernel<T, VEC, decltype(a)::value>, dim3((unsigned)blocks), dim3(NORM_THREADS), 0,
                                     ctx, (const T *)d_x, d_gamma, d_beta, (const float *)mean, (const float *)rstd,
                                     (T *)d_y, s));
            return FC_OK;
        });
    });
}

int fc_group_norm_backward(fc_context *ctx, const fc_group_norm_desc *desc, const void *d_dy, const void *d_x,
                           const void *d_gamma, const void *d_beta, const float *d_mean, const float *d_rstd, void *d_dx,
                           void *d_dgamma, void *d_dbeta, void *d_workspace, size_t workspace_bytes) {
    FC_REQUIRE(ctx != nullptr, FC_ERR_INVALID_ARG, "context is NULL");
    NormShape s;
    FC_PROPAGATE(norm_shape(desc, &s));
    if (s.batch > 0) FC_PROPAGATE(check_maps(desc, {d_dy, d_x, d_dx ? d_dx : d_x}, {}, nullptr, nullptr));
    FC_PROPAGATE(check_maps(desc, {}, {d_gamma, d_beta, d_dgamma, d_dbeta}, d_mean, d_rstd));  // of no images they are written too
    FC_PROPAGATE(check_outputs({d_dx, d_dgamma, d_dbeta, d_workspace}, {d_dy, d_x, d_gamma, d_beta, d_mean, d_rstd}));
    FC_REQUIRE(s.batch == 0 || (d_mean != nullptr && d_rstd != nullptr), FC_ERR_INVALID_ARG,
               "the gradient needs the forward pass's mean and rstd");
    size_t need;
    FC_PROPAGATE(fc_group_norm_workspace(desc, nullptr, &need));
    FC_REQUIRE(need == 0 || (d_workspace != nullptr && aligned16(d_workspace) && workspace_bytes >= need), FC_ERR_INVALID_ARG,
               "workspace of %zu bytes at %p: %zu are needed, on a 16-byte boundary", workspace_bytes, d_workspace, need);
    DeviceScope dev(ctx->device);
    FC_CHECK_CUDA(dev.status());
    return with_vectors(s, desc->type, {d_dy, d_x, d_dx}, [&](auto t, auto v) -> int {
        using T = decltype(t);
        constexpr int VEC = decltype(v)::value;
        norm_split(&s, VEC);
        const long long blocks = (long long)s.batch * s.chunks * s.col_tiles;
        FC_REQUIRE(blocks < (1ll << 31), FC_ERR_UNSUPPORTED, "%lld blocks", blocks);
        const NormWork w = norm_carve(s, d_workspace, true);
        Fused f;
        bool fused = false;
        if constexpr (VEC > 1) fused = s.batch > 0 && fused_plan(s, sizeof(T), true, &f);
        if (fused) {
            if constexpr (VEC > 1)
                FC_PROPAGATE(with_act(desc->act, [&](auto a) -> int {
                    constexpr int A = decltype(a)::value;
                    auto kernel = f.width > 1 ? norm_back_fused_kernel<T, A, true> : norm_back_fused_kernel<T, A, false>;
                    FC_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024));
                    FC_CHECK_CUDA(launch_clusters(kernel, dim3(f.blocks * f.cluster, s.batch), FUSED_THREADS, f.cluster, f.smem,
                                                  ctx, (const T *)d_dy, (const T *)d_x, d_gamma, d_beta, d_mean, d_rstd,
                                                  (T *)d_dx, w.sums, s, f));
                    return FC_OK;
                }));
        } else if (s.batch > 0) {
            FC_PROPAGATE(with_act(desc->act, [&](auto a) -> int {
                FC_CHECK_CUDA(launch_early(norm_back_part_kernel<T, VEC, decltype(a)::value>, dim3((unsigned)blocks),
                                         dim3(NORM_THREADS), 0, ctx, (const T *)d_dy, (const T *)d_x, d_gamma, d_beta,
                                         d_mean, d_rstd, w.part, s));
                return FC_OK;
            }));
            FC_CHECK_CUDA(launch_early(norm_back_join_kernel<T>, dim3(s.batch * s.groups), dim3(NORM_THREADS), 0, ctx,
                                     (const float2 *)w.part, d_gamma, w.sums, w.ab, s));
            if (d_dx != nullptr)
                FC_PROPAGATE(with_act(desc->act, [&](auto a) -> int {
                    FC_CHECK_CUDA(launch_early(norm_back_apply_kernel<T, VEC, decltype(a)::value>, dim3((unsigned)blocks),
                                             dim3(NORM_THREADS), 0, ctx, (const T *)d_dy, (const T *)d_x, d_gamma, d_beta,
                                             d_mean, d_rstd, (const float2 *)w.ab, (T *)d_dx, s));
                    return FC_OK;
                }));
        }
        if (d_dgamma != nullptr || d_dbeta != nullptr)
            FC_CHECK_CUDA(launch_early(norm_back_params_kernel<T>, dim3((s.channels + 31) / 32),
                                     dim3(NORM_THREADS), 0, ctx, (const float2 *)w.sums, d_dgamma, d_dbeta, s));
        return FC_OK;
    });
}

}  // extern "C"
