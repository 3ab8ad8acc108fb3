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

template <typename T, bool kToLast>
__global__ void __launch_bounds__(MOVE_THREADS) map_move_kernel(float *__restrict__ planes, T *__restrict__ last_map,
                                                               const MoveShape s) {
    __shared__ float tile[TILE][TILE + 1];  // [channel][pixel]
    pdl_wait();
    pdl_next();
    const long long id = blockIdx.x;
    const int ct = (int)(id % s.ctiles);
    const long long rest = id / s.ctiles;
    const int pt = (int)(rest % s.ptiles), img = (int)(rest / s.ptiles);
    const int c0 = ct * TILE, p0 = pt * TILE;
    const int tx = threadIdx.x & (TILE - 1), ty = threadIdx.x / TILE;
    float *plane = planes + ((size_t)img * s.channels + c0) * s.pixels + p0;
    T *row = last_map + ((size_t)img * s.pixels + p0) * s.stride + c0;
    const int nc = min(TILE, s.channels - c0), np = min(TILE, s.pixels - p0);
    if (kToLast) {
        if (tx < np)
            for (int c = ty; c < nc; c += MOVE_THREADS / TILE) tile[c][tx] = plane[(size_t)c * s.pixels + tx];
        __syncthreads();
        if (tx < nc)
            for (int p = ty; p < np; p += MOVE_THREADS / TILE) row[(size_t)p * s.stride + tx] = Elem<T>::store(tile[tx][p]);
    } else {
        if (tx < nc)
            for (int p = ty; p < np; p += MOVE_THREADS / TILE) tile[tx][p] = Elem<T>::load(row[(size_t)p * s.stride + tx]);
        __syncthreads();
        if (tx < np)
            for (int c = ty; c < nc; c += MOVE_THREADS / TILE) plane[(size_t)c * s.pixels + tx] = tile[c][tx];
    }
}

int move(fc_context *ctx, float *planes, void *last_map, int batch, int channels, int pixels, int64_t stride, int type,
         bool to_last) {
    FC_REQUIRE(ctx != nullptr, FC_ERR_INVALID_ARG, "context is NULL");
    FC_REQUIRE(batch >= 0 && channels > 0 && pixels > 0, FC_ERR_INVALID_ARG, "batch %d, channels %d, pixels %d", batch,
               channels, pixels);
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
        FC_CHECK_CUDA(launch_pdl(to_last ? map_move_kernel<T, true> : map_move_kernel<T, false>, dim3((unsigned)blocks),
                                 dim3(MOVE_THREADS), 0, ctx->stream, planes, (T *)last_map, s));
        return FC_OK;
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
