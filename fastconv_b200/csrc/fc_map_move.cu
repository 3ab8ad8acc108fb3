// Moves between the convolution layers' maps (fp32, [n][c][pixels]) and channels-last ones ([n][pixels][c] in fp32, bf16
// or fp16, rounded to nearest on the way in).  Each direction is the other's gradient.
//
// One read and one write per element, nothing to compute: the bound is HBM.  A block turns a tile of 4096 elements in shared
// memory, 64 channels x 64 pixels or, for maps of few channels, 32 x 128, 16 x 256 or 8 x 512, so that both sides see runs of
// at least 128 bytes (of all its channels, where a pixel has fewer bytes); all loads of a thread are in flight at once.
// 64 x 56x56x256 to bf16, 308 MB: 53 to 56 us, 5.5 to 5.8 TB/s, 0.84 to 0.89 of the measured copy rate; element by element in a loop 62 us.
#include <type_traits>

#include "fc_last.cuh"

namespace fc {

namespace {

using namespace last;

constexpr int TILE = 4096, MOVE_THREADS = 256;

struct MoveShape {
    int channels, pixels;
    int64_t stride;  // elements from one pixel of the channels-last map to the next
    int ctiles, ptiles;
};

// kPairs: two neighbouring channels of the channels-last map move as one word (16-bit types, even stride, 4-byte aligned).
template <typename T, bool kToLast, bool kPairs, int TC>
__global__ void __launch_bounds__(MOVE_THREADS, 8) map_move_kernel(float *planes, T *last_map, const MoveShape s) {
    constexpr int TP = TILE / TC, PAD = TC < 32 ? 32 / TC : 1;  // the pad keeps a warp's columns in different banks
    __shared__ float tile[TC][TP + PAD];                        // [channel][pixel]
    const uint32_t rest = blockIdx.x / (uint32_t)s.ctiles, ct = blockIdx.x - rest * s.ctiles;
    const uint32_t img = rest / (uint32_t)s.ptiles, pt = rest - img * s.ptiles;
    const int c0 = (int)ct * TC, p0 = (int)pt * TP;
    const int nc = min(TC, s.channels - c0), np = min(TP, s.pixels - p0);
    float *plane = planes + ((size_t)img * s.channels + c0) * s.pixels + p0;
    T *row = last_map + ((size_t)img * s.pixels + p0) * s.stride + c0;
    constexpr int STEP = kPairs ? 2 : 1, LANES = TC / STEP;  // channels of an access; accesses of a pixel
    pdl_wait();
    pdl_next();
    constexpr int P_ITEMS = TILE / MOVE_THREADS, L_ITEMS = P_ITEMS / STEP;  // of a thread, on either side
    // use(i, channel, pixel, whether that is inside the map); inside is known where the whole tile is
    auto plane_side = [&](auto whole, auto &&use) {
#pragma unroll
        for (int i = 0; i < P_ITEMS; ++i) {
            const int at = i * MOVE_THREADS + threadIdx.x, c = at / TP, px = at % TP;
            use(i, c, px, decltype(whole)::value || (c < nc && px < np));
        }
    };
    auto last_side = [&](auto whole, auto &&use) {
#pragma unroll
        for (int i = 0; i < L_ITEMS; ++i) {
            const int at = i * MOVE_THREADS + threadIdx.x, c = at % LANES * STEP, p = at / LANES;
            use(i, c, p, decltype(whole)::value || (c < nc && p < np));
        }
    };
    auto turn = [&](auto whole) {
        constexpr bool W = decltype(whole)::value;
        if (kToLast) {
            float v[P_ITEMS];  // all loads before the first use
            plane_side(whole, [&](int i, int c, int px, bool in) { v[i] = in ? plane[(size_t)c * s.pixels + px] : 0.0f; });
            plane_side(whole, [&](int i, int c, int px, bool) { tile[c][px] = v[i]; });
            __syncthreads();
            last_side(whole, [&](int, int c, int p, bool in) {
                if (!in) return;
                T *to = row + (size_t)p * s.stride + c;
                if (kPairs && (W || c + 1 < nc)) {
                    if constexpr (kPairs) Elem<T>::store2(to, tile[c][p], tile[c + 1][p]);
                } else {
                    *to = Elem<T>::store(tile[c][p]);
                }
            });
        } else {
            float v[L_ITEMS][STEP];
            last_side(whole, [&](int i, int c, int p, bool in) {
                const T *from = row + (size_t)p * s.stride + c;
#pragma unroll
                for (int j = 0; j < STEP; ++j) v[i][j] = 0.0f;
                if (kPairs && in && (W || c + 1 < nc)) {
                    if constexpr (kPairs) Elem<T>::load2(from, v[i][0], v[i][1]);
                } else if (in) {
                    v[i][0] = Elem<T>::load(*from);
                }
            });
            last_side(whole, [&](int i, int c, int p, bool) {
#pragma unroll
                for (int j = 0; j < STEP; ++j) tile[c + j][p] = v[i][j];
            });
            __syncthreads();
            plane_side(whole, [&](int, int c, int px, bool in) {
                if (in) plane[(size_t)c * s.pixels + px] = tile[c][px];
            });
        }
    };
    if (nc == TC && np == TP)
        turn(std::true_type());
    else
        turn(std::false_type());
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
    FC_PROPAGATE(check_outputs({to_last ? last_map : planes}, {to_last ? planes : last_map}));
    const int tc = channels > 32 ? 64 : channels > 16 ? 32 : channels > 8 ? 16 : 8;
    MoveShape s = {channels, pixels, stride, (channels + tc - 1) / tc, (int)ceil_div(pixels, TILE / tc)};
    const long long blocks = (long long)batch * s.ctiles * s.ptiles;
    FC_REQUIRE(blocks < (1ll << 31), FC_ERR_UNSUPPORTED, "map of %lld tiles", blocks);
    DeviceScope dev(ctx->device);
    FC_CHECK_CUDA(dev.status());
    return with_type(type, [&](auto t) -> int {
        using T = decltype(t);
        auto go = [&](auto pairs, auto width) -> int {
            constexpr bool P = decltype(pairs)::value;
            constexpr int TC = decltype(width)::value;
            FC_CHECK_CUDA(launch_early(to_last ? map_move_kernel<T, true, P, TC> : map_move_kernel<T, false, P, TC>, dim3((unsigned)blocks),
                                     dim3(MOVE_THREADS), 0, ctx, planes, (T *)last_map, s));
            return FC_OK;
        };
        auto by_width = [&](auto pairs) -> int {
            switch (tc) {
                case 8: return go(pairs, std::integral_constant<int, 8>());
                case 16: return go(pairs, std::integral_constant<int, 16>());
                case 32: return go(pairs, std::integral_constant<int, 32>());
                default: return go(pairs, std::integral_constant<int, 64>());
            }
        };
        if constexpr (sizeof(T) == 2)
            if (stride % 2 == 0 && (uintptr_t)last_map % 4 == 0) return by_width(std::true_type());
        return by_width(std::false_type());
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
