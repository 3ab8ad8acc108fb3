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
// Three kernels each way: sums of a chunk of pixels per channel; their join per group; the map itself.
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
    return f32 ? __ldg((const float *)p + c) : Elem<T>::load(((const T *)p)[c]);
}

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
    b.p1 = min(s.pixels, b.p0 + s.chunk_pixels);
    b.rows = NORM_THREADS / s.cols;
    b.row = threadIdx.x / s.cols;
    b.col = threadIdx.x % s.cols;
    b.c0 = (tile * s.cols + b.col) * VEC;
    b.live = b.row < b.rows && b.c0 < s.channels;
    return b;
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
__global__ void __launch_bounds__(NORM_THREADS) norm_part_kernel(const T *__restrict__ x, float2 *__restrict__ part,
                                                                const NormShape s) {
    __shared__ float2 stat[NORM_THREADS * VEC];
    pdl_wait();
    const Place b = place_of<VEC>(s);
    float k[VEC], sum[VEC], sq[VEC];
    int n = 0;
#pragma unroll
    for (int i = 0; i < VEC; ++i) k[i] = sum[i] = sq[i] = 0.0f;
    if (b.live) {
        const T *src = x + (size_t)b.img * s.pixels * s.xs + b.c0;
        int p = b.p0 + b.row;
        if (p < b.p1) ((const Vec<T, VEC> *)(src + (size_t)p * s.xs))->unpack(k);
#pragma unroll 4
        for (; p < b.p1; p += b.rows, ++n) {
            float f[VEC];
            ((const Vec<T, VEC> *)(src + (size_t)p * s.xs))->unpack(f);
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
__global__ void __launch_bounds__(NORM_THREADS) norm_join_kernel(const float2 *__restrict__ part, float *__restrict__ mean,
                                                                float *__restrict__ rstd, const NormShape s) {
    __shared__ float scratch[NORM_THREADS / 32];
    pdl_wait();
    const int img = blockIdx.x / s.groups, g = blockIdx.x % s.groups;
    const float2 *src = part + (size_t)img * s.chunks * s.channels + g * s.cpg;
    const int items = s.chunks * s.cpg;
    const float inv = 1.0f / ((float)s.pixels * (float)s.cpg);
    float a = 0.0f;
    for (int i = threadIdx.x; i < items; i += NORM_THREADS) {
        const int chunk = i / s.cpg, n = min(s.pixels, (chunk + 1) * s.chunk_pixels) - chunk * s.chunk_pixels;
        a = fmaf(src[(size_t)chunk * s.channels + i % s.cpg].x, (float)n, a);
    }
    const float m = block_sum(a, scratch) * inv;
    float q = 0.0f;
    for (int i = threadIdx.x; i < items; i += NORM_THREADS) {
        const int chunk = i / s.cpg, n = min(s.pixels, (chunk + 1) * s.chunk_pixels) - chunk * s.chunk_pixels;
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
__global__ void __launch_bounds__(NORM_THREADS) norm_apply_kernel(const T *__restrict__ x, const void *__restrict__ gamma,
                                                                 const void *__restrict__ beta, const float *__restrict__ mean,
                                                                 const float *__restrict__ rstd, T *__restrict__ y,
                                                                 const NormShape s) {
    constexpr bool kExact = std::is_same<T, float>::value;
    pdl_wait();
    const Place b = place_of<VEC>(s);
    if (!b.live) return;
    float m[VEC], a[VEC], o[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        const int c = b.c0 + i, at = b.img * s.groups + c / s.cpg;
        m[i] = mean[at];
        a[i] = rstd[at] * param<T>(gamma, c, s.params_f32, 1.0f);
        o[i] = param<T>(beta, c, s.params_f32, 0.0f);
    }
    const T *src = x + (size_t)b.img * s.pixels * s.xs + b.c0;
    T *dst = y + (size_t)b.img * s.pixels * s.ys + b.c0;
#pragma unroll 4
    for (int p = b.p0 + b.row; p < b.p1; p += b.rows) {
        float f[VEC];
        ((const Vec<T, VEC> *)(src + (size_t)p * s.xs))->unpack(f);
#pragma unroll
        for (int i = 0; i < VEC; ++i) f[i] = act_value<ACT, kExact>(fmaf(f[i] - m[i], a[i], o[i]));
        ((Vec<T, VEC> *)(dst + (size_t)p * s.ys))->pack(f);
    }
}

// ---- backward ---------------------------------------------------------------------------------------------------

// what a thread keeps of its channels in the backward pass
template <typename T, int VEC>
struct BackChannels {
    float m[VEC], r[VEC], g[VEC], o[VEC];
    __device__ __forceinline__ BackChannels(const void *gamma, const void *beta, const float *mean, const float *rstd, int img,
                                            int c0, const NormShape &s) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const int c = c0 + i, at = img * s.groups + c / s.cpg;
            m[i] = mean[at];
            r[i] = rstd[at];
            g[i] = param<T>(gamma, c, s.params_f32, 1.0f);
            o[i] = param<T>(beta, c, s.params_f32, 0.0f);
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
__global__ void __launch_bounds__(NORM_THREADS) norm_back_part_kernel(const T *__restrict__ dy, const T *__restrict__ x,
                                                                     const void *__restrict__ gamma,
                                                                     const void *__restrict__ beta,
                                                                     const float *__restrict__ mean,
                                                                     const float *__restrict__ rstd, float2 *__restrict__ part,
                                                                     const NormShape s) {
    __shared__ float2 stat[NORM_THREADS * VEC];
    pdl_wait();
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
            ((const Vec<T, VEC> *)(sx + (size_t)p * s.xs))->unpack(f);
            ((const Vec<T, VEC> *)(sdy + (size_t)p * s.ys))->unpack(d);
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
__global__ void __launch_bounds__(NORM_THREADS) norm_back_join_kernel(const float2 *__restrict__ part,
                                                                     const void *__restrict__ gamma, float2 *__restrict__ sums,
                                                                     float2 *__restrict__ ab, const NormShape s) {
    __shared__ float scratch[NORM_THREADS / 32];
    pdl_wait();
    const int img = blockIdx.x / s.groups, g = blockIdx.x % s.groups;
    float a = 0.0f, q = 0.0f;
    for (int i = threadIdx.x; i < s.cpg; i += NORM_THREADS) {
        const int c = g * s.cpg + i;
        float2 t = make_float2(0.0f, 0.0f);
        for (int k = 0; k < s.chunks; ++k) {
            const float2 v = part[((size_t)img * s.chunks + k) * s.channels + c];
            t.x += v.x;
            t.y += v.y;
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
__global__ void __launch_bounds__(NORM_THREADS) norm_back_apply_kernel(const T *__restrict__ dy, const T *__restrict__ x,
                                                                      const void *__restrict__ gamma,
                                                                      const void *__restrict__ beta,
                                                                      const float *__restrict__ mean,
                                                                      const float *__restrict__ rstd,
                                                                      const float2 *__restrict__ ab, T *__restrict__ dx,
                                                                      const NormShape s) {
    pdl_wait();
    const Place b = place_of<VEC>(s);
    if (!b.live) return;
    const BackChannels<T, VEC> ch(gamma, beta, mean, rstd, b.img, b.c0, s);
    float2 t[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) t[i] = ab[b.img * s.groups + (b.c0 + i) / s.cpg];
    const T *sx = x + (size_t)b.img * s.pixels * s.xs + b.c0, *sdy = dy + (size_t)b.img * s.pixels * s.ys + b.c0;
    T *dst = dx + (size_t)b.img * s.pixels * s.xs + b.c0;
#pragma unroll 2
    for (int p = b.p0 + b.row; p < b.p1; p += b.rows) {
        float f[VEC], d[VEC];
        ((const Vec<T, VEC> *)(sx + (size_t)p * s.xs))->unpack(f);
        ((const Vec<T, VEC> *)(sdy + (size_t)p * s.ys))->unpack(d);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            float dz, xhat;
            ch.template at<ACT>(i, f[i], d[i], dz, xhat);
            f[i] = ch.r[i] * (fmaf(dz, ch.g[i], -t[i].x) - xhat * t[i].y);
        }
        ((Vec<T, VEC> *)(dst + (size_t)p * s.xs))->pack(f);
    }
}

// dgamma[c], dbeta[c]: the images' sums, added in order
template <typename T>
__global__ void __launch_bounds__(NORM_THREADS) norm_back_params_kernel(const float2 *__restrict__ sums, void *dgamma, void *dbeta,
                                                                       const NormShape s) {
    pdl_wait();
    const int c = blockIdx.x * NORM_THREADS + threadIdx.x;
    if (c >= s.channels) return;
    float2 t = make_float2(0.0f, 0.0f);
    for (int n = 0; n < s.batch; ++n) {
        const float2 v = sums[(size_t)n * s.channels + c];
        t.x += v.x;
        t.y += v.y;
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

// f(T(), integral_constant<int, elements of a vector>) for the widest vector that fits
template <typename F>
int with_vectors(const NormShape &s, int type, std::initializer_list<const void *> maps, F &&f) {
    return with_type(type, [&](auto t) -> int {
        using T = decltype(t);
        if (wide_ok<T>(s, maps)) return f(t, std::integral_constant<int, 16 / (int)sizeof(T)>());
        return f(t, std::integral_constant<int, 1>());
    });
}

int check_maps(const fc_group_norm_desc *d, std::initializer_list<const void *> maps, std::initializer_list<const void *> params) {
    for (const void *p : maps) {
        FC_REQUIRE(p != nullptr, FC_ERR_INVALID_ARG, "NULL map");
        FC_REQUIRE((uintptr_t)p % dtype_size(d->type) == 0, FC_ERR_INVALID_ARG, "a map's address is no multiple of its element size");
    }
    for (const void *p : params)
        FC_REQUIRE((uintptr_t)p % dtype_size(d->param_type) == 0, FC_ERR_INVALID_ARG,
                   "a parameter's address is no multiple of its element size");
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
    FC_PROPAGATE(check_maps(desc, {d_x, d_y}, {d_gamma, d_beta}));
    size_t need;
    FC_PROPAGATE(fc_group_norm_workspace(desc, &need, nullptr));
    FC_REQUIRE(d_workspace != nullptr && aligned16(d_workspace) && workspace_bytes >= need, FC_ERR_INVALID_ARG,
               "workspace of %zu bytes at %p: %zu are needed, on a 16-byte boundary", workspace_bytes, d_workspace, need);
    DeviceScope dev(ctx->device);
    FC_CHECK_CUDA(dev.status());
    return with_vectors(s, desc->type, {d_x, d_y}, [&](auto t, auto v) -> int {
        using T = decltype(t);
        constexpr int VEC = decltype(v)::value;
        norm_split(&s, VEC);
        const long long blocks = (long long)s.batch * s.chunks * s.col_tiles;
        FC_REQUIRE(blocks < (1ll << 31), FC_ERR_UNSUPPORTED, "%lld blocks", blocks);
        const NormWork w = norm_carve(s, d_workspace, false);
        float *mean = d_mean ? d_mean : w.mean, *rstd = d_rstd ? d_rstd : w.rstd;
        FC_CHECK_CUDA(launch_pdl(norm_part_kernel<T, VEC>, dim3((unsigned)blocks), dim3(NORM_THREADS), 0, ctx->stream, (const T *)d_x,
                                 w.part, s));
        FC_CHECK_CUDA(launch_pdl(norm_join_kernel, dim3(s.batch * s.groups), dim3(NORM_THREADS), 0, ctx->stream,
                                 (const float2 *)w.part, mean, rstd, s));
        return with_act(desc->act, [&](auto a) -> int {
            FC_CHECK_CUDA(launch_pdl(norm_apply_kernel<T, VEC, decltype(a)::value>, dim3((unsigned)blocks), dim3(NORM_THREADS), 0,
                                     ctx->stream, (const T *)d_x, d_gamma, d_beta, (const float *)mean, (const float *)rstd,
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
    if (s.batch > 0) FC_PROPAGATE(check_maps(desc, {d_dy, d_x, d_dx ? d_dx : d_x}, {d_gamma, d_beta, d_dgamma, d_dbeta}));
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
        if (s.batch > 0) {
            FC_PROPAGATE(with_act(desc->act, [&](auto a) -> int {
                FC_CHECK_CUDA(launch_pdl(norm_back_part_kernel<T, VEC, decltype(a)::value>, dim3((unsigned)blocks),
                                         dim3(NORM_THREADS), 0, ctx->stream, (const T *)d_dy, (const T *)d_x, d_gamma, d_beta,
                                         d_mean, d_rstd, w.part, s));
                return FC_OK;
            }));
            FC_CHECK_CUDA(launch_pdl(norm_back_join_kernel<T>, dim3(s.batch * s.groups), dim3(NORM_THREADS), 0, ctx->stream,
                                     (const float2 *)w.part, d_gamma, w.sums, w.ab, s));
            if (d_dx != nullptr)
                FC_PROPAGATE(with_act(desc->act, [&](auto a) -> int {
                    FC_CHECK_CUDA(launch_pdl(norm_back_apply_kernel<T, VEC, decltype(a)::value>, dim3((unsigned)blocks),
                                             dim3(NORM_THREADS), 0, ctx->stream, (const T *)d_dy, (const T *)d_x, d_gamma, d_beta,
                                             d_mean, d_rstd, (const float2 *)w.ab, (T *)d_dx, s));
                    return FC_OK;
                }));
        }
        if (d_dgamma != nullptr || d_dbeta != nullptr)
            FC_CHECK_CUDA(launch_pdl(norm_back_params_kernel<T>, dim3((s.channels + NORM_THREADS - 1) / NORM_THREADS),
                                     dim3(NORM_THREADS), 0, ctx->stream, (const float2 *)w.sums, d_dgamma, d_dbeta, s));
        return FC_OK;
    });
}

}  // extern "C"
