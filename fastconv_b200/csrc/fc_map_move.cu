// Moves between the convolution layers' maps (fp32, [n][c][pixels]) and channels-last ones ([n][pixels][c] in fp32, bf16
// or fp16, rounded to nearest on the way in).  Each direction is the other's gradient.
//
// One read and one write per element, nothing to compute: the bound is HBM.  A block moves a tile of 64 channels x 64
// pixels through shared memory so that both sides see runs of at least 128 bytes.
#include <type_traits>

#include "fc_last.cuh"

namespace fc {

namespace {

using namespace last;

constexpr int TILE = 64, MOVE_THREADS = 256;

struct MoveShape {
    int batch, channels, pixels;
    int64_t stride;  // elements from one pixel of the channels-last map to the next
    int ctiles, ptiles;
};

// kPairs: two neighbouring channels of the channels-last map move as one word (16-bit types, even stride, 4-byte aligned).
template <typename T, bool kToLast, bool kPairs>
__global__ void __launch_bounds__(MOVE_THREADS) map_move_kernel(float *__restrict__ planes, T *__restrict__ last_map,
                                                               const MoveShape s) {
    __shared__ float tile[TILE][TILE + 1];  // [channel][pixel]
    const uint32_t rest = blockIdx.x / (uint32_t)s.ctiles, ct = blockIdx.x - rest * s.ctiles;
    const uint32_t img = rest / (uint32_t)s.ptiles, pt = rest - img * s.ptiles;
    const int c0 = (int)ct * TILE, p0 = (int)pt * TILE;
    const int nc = min(TILE, s.channels - c0), np = min(TILE, s.pixels - p0);
    float *plane = planes + ((size_t)img * s.channels + c0) * s.pixels + p0;
    T *row = last_map + ((size_t)img * s.pixels + p0) * s.stride + c0;
    const bool whole = nc == TILE && np == TILE;
    // one side walks over pixels with 64 threads, a channel a step; the other over channels, a pixel a step
    const int px = threadIdx.x & (TILE - 1), cy = threadIdx.x / TILE;
    constexpr int C_LANES = kPairs ? TILE / 2 : TILE, P_STEP = MOVE_THREADS / C_LANES, C_STEP = MOVE_THREADS / TILE;
    const int cx = threadIdx.x % C_LANES, py = threadIdx.x / C_LANES;
    auto plane_side = [&](auto &&one) {
        if (whole) {
#pragma unroll
            for (int i = 0; i < TILE / C_STEP; ++i) one(cy + i * C_STEP);
        } else if (px < np) {
            for (int c = cy; c < nc; c += C_STEP) one(c);
        }
    };
    auto last_side = [&](auto &&one) {
        if (whole) {
#pragma unroll
            for (int i = 0; i < TILE / P_STEP; ++i) one(py + i * P_STEP);
        } else {
            for (int p = py; p < np; p += P_STEP) one(p);
        }
    };
    pdl_wait();
    pdl_next();
    if (kToLast) {
        plane_side([&](int c) { tile[c][px] = __ldg(plane + (size_t)c * s.pixels + px); });
        __syncthreads();
        last_side([&](int p) {
            T *to = row + (size_t)p * s.stride;
            if constexpr (kPairs) {
                if (2 * cx + 1 < nc)
                    Elem<T>::store2(to + 2 * cx, tile[2 * cx][p], tile[2 * cx + 1][p]);
                else if (2 * cx < nc)
                    to[2 * cx] = Elem<T>::store(tile[2 * cx][p]);
            } else if (cx < nc) {
                to[cx] = Elem<T>::store(tile[cx][p]);
            }
        });
    } else {
        last_side([&](int p) {
            const T *from = row + (size_t)p * s.stride;
            if constexpr (kPairs) {
                if (2 * cx + 1 < nc)
                    Elem<T>::load2(from + 2 * cx, tile[2 * cx][p], tile[2 * cx + 1][p]);
                else if (2 * cx < nc)
                    tile[2 * cx][p] = Elem<T>::load(from[2 * cx]);
            } else if (cx < nc) {
                tile[cx][p] = Elem<T>::load(from[cx]);
            }
        });
        __syncthreads();
        plane_side([&](int c) { plane[(size_t)c * s.pixels + px] = tile[c][px]; });
    }
}

int move(fc_context *ctx, float *planes, void *last_map, int batch, int channels, int pixels, int64_t stride, int type,
         bool to_last) {
    FC_REQUIRE(ctx != nullptr, FC_ERR_INVALID_ARG, "context is NULL");
    FC_REQUIRE(batch >= 0 && channels > 0 && pixels > 0, FC_ERR_INVALID_ARG, "batch %d, channels %d, pixels %d", batch,
               channels, pixels);
    FC_REQUIRE(channels < (1 << 30) && pixels < (1 << 30), FC_ERR_UNSUPPORTED, "%d channels, %d pixels", channels, pixels);
    FC_REQUIRE(dtype_ok(type), FC_ERR_INVALID_ARG, "unknown element type %d", type);
    if (stride == 0) stride = channels;
    FC_REQUIRE(stride >= channels, FC_ERR_INVALID_ARG, "pixel stride %lld is less than the %d channels", (long long)stride,
               channels);
    if (batch == 0) return FC_OK;
    FC_REQUIRE(planes != nullptr && last_map != nullptr, FC_ERR_INVALID_ARG, "NULL map");
    FC_REQUIRE((uintptr_t)planes % 4 == 0 && (uintptr_t)last_map % dtype_size(type) == 0, FC_ERR_INVALID_ARG,
               "a map's address is no multiple of its element size");
    MoveShape s = {batch, channels, pixels, stride, (channels + TILE - 1) / TILE, (pixels + TILE - 1) / TILE};
    const long long blocks = (long long)batch * s.ctiles * s.ptiles;
    FC_REQUIRE(blocks < (1ll << 31), FC_ERR_UNSUPPORTED, "map of %lld tiles", blocks);
    DeviceScope dev(ctx->device);
    FC_CHECK_CUDA(dev.status());
    return with_type(type, [&](auto t) -> int {
        using T = decltype(t);
        auto go = [&](auto kernel) -> int {
            FC_CHECK_CUDA(launch_pdl(kernel, dim3((unsigned)blocks), dim3(MOVE_THREADS), 0, ctx->stream, planes, (T *)last_map, s));
            return FC_OK;
        };
        if constexpr (sizeof(T) == 2)
            if (stride % 2 == 0 && (uintptr_t)last_map % 4 == 0)
                return to_last ? go(map_move_kernel<T, true, true>) : go(map_move_kernel<T, false, true>);
        return to_last ? go(map_move_kernel<T, true, false>) : go(map_move_kernel<T, false, false>);
    });
}

}  // namespace

}  // namespace fc

using namespace fc;

extern "C" {

int fc_map_to_channels_last(fc_context *ctx, const float *d_planes, void *d_last, int batch, int channels, int pixels,
                            int64_t last_stride, int type) {
    return move(ctx, const_cast<float *>(d_planes), d_last, batch, channels, pixels, last_stride, type, true);
}

int fc_map_from_channels_last(fc_context *ctx, const void *d_last, float *d_planes, int batch, int channels, int pixels,
                              int64_t last_stride, int type) {
    return move(ctx, d_planes, const_cast<void *>(d_last), batch, channels, pixels, last_stride, type, false);
}

}  // extern "C"
