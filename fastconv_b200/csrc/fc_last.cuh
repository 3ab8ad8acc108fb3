// Shared pieces of the channels-last operators (fc_map_move.cu, fc_group_norm.cu, fc_gated_ff*.cu): element types,
// vectors of them, activations with their derivatives, and the host-side checks.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "fc_internal.h"

namespace fc {
namespace last {

// ---- element types ----------------------------------------------------------------------------------------------
// Everything is computed in fp32; a value is rounded once, to nearest, where it is stored.
template <typename T>
struct Elem;
template <>
struct Elem<float> {
    static constexpr int kType = FC_DTYPE_F32;
    static __device__ __forceinline__ float load(float v) { return v; }
    static __device__ __forceinline__ float store(float v) { return v; }
};
template <>
struct Elem<__nv_bfloat16> {
    static constexpr int kType = FC_DTYPE_BF16;
    static __device__ __forceinline__ float load(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 store(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Elem<__half> {
    static constexpr int kType = FC_DTYPE_F16;
    static __device__ __forceinline__ float load(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half store(float v) { return __float2half_rn(v); }
};

// N neighbouring elements, moved with one access (N * sizeof(T) is 2, 4, 8 or 16 bytes and the address a multiple of it)
template <typename T, int N>
struct alignas(N * sizeof(T)) Vec {
    T v[N];
    __device__ __forceinline__ void unpack(float (&f)[N]) const {
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = Elem<T>::load(v[i]);
    }
    __device__ __forceinline__ void pack(const float (&f)[N]) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = Elem<T>::store(f[i]);
    }
};

inline size_t dtype_size(int type) { return type == FC_DTYPE_F32 ? 4 : 2; }
inline bool dtype_ok(int type) { return type >= FC_DTYPE_F32 && type <= FC_DTYPE_F16; }
inline bool act_ok(int act) { return act >= FC_ACT_NONE && act <= FC_ACT_SIGMOID; }
inline bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

// ---- activations ------------------------------------------------------------------------------------------------
// kExact: the correctly scaled library functions, for results that are kept in fp32.  Otherwise the hardware's
// exponential and division (a few units in the 23rd bit), for results that are rounded to 8 or 11 bits anyway.
template <bool kExact>
__device__ __forceinline__ float sigmoid(float z) {
    // exp(-z) = inf for very negative z: the quotient is then 0, as it should be
    return kExact ? 1.0f / (1.0f + expf(-z)) : __fdividef(1.0f, 1.0f + __expf(-z));
}

// act(z); kAct is an fc_activation.  A NaN stays one in every activation.
template <int kAct, bool kExact>
__device__ __forceinline__ float act_value(float z) {
    if (kAct == FC_ACT_RELU) return z < 0.0f ? 0.0f : z;
    if (kAct == FC_ACT_SILU) return z * sigmoid<kExact>(z);
    if (kAct == FC_ACT_GELU) return 0.5f * z * erfcf(-0.70710678118654752f * z);  // erfc keeps the digits of the tail
    if (kAct == FC_ACT_GELU_TANH) {
        // 0.5 (1 + tanh v) = sigmoid(2 v); the square is bounded so that huge z give 0 or z and no inf * 0
        const float t = fminf(z * z, 1e6f);
        return z * sigmoid<kExact>(1.59576912160573071f * z * (1.0f + 0.044715f * t));
    }
    if (kAct == FC_ACT_SIGMOID) return sigmoid<kExact>(z);
    return z;
}

// act(z) and act'(z)
template <int kAct, bool kExact>
__device__ __forceinline__ void act_both(float z, float &a, float &d) {
    if (kAct == FC_ACT_RELU) {
        a = z < 0.0f ? 0.0f : z;
        d = z > 0.0f ? 1.0f : 0.0f;
    } else if (kAct == FC_ACT_SILU) {
        const float s = sigmoid<kExact>(z);
        a = z * s;
        d = s + a * (1.0f - s);
    } else if (kAct == FC_ACT_GELU) {
        const float cdf = 0.5f * erfcf(-0.70710678118654752f * z);
        a = z * cdf;
        d = cdf + 0.39894228040143268f * z * (kExact ? expf(-0.5f * z * z) : __expf(-0.5f * z * z));
    } else if (kAct == FC_ACT_GELU_TANH) {
        const float t = fminf(z * z, 1e6f);
        const float s = sigmoid<kExact>(1.59576912160573071f * z * (1.0f + 0.044715f * t));
        a = z * s;
        d = s + a * (1.0f - s) * 1.59576912160573071f * (1.0f + 0.134145f * t);
    } else if (kAct == FC_ACT_SIGMOID) {
        a = sigmoid<kExact>(z);
        d = a * (1.0f - a);
    } else {
        a = z;
        d = 1.0f;
    }
}

// Calls f(std::integral_constant<int, act>) for a run-time activation.
template <typename F>
int with_act(int act, F &&f) {
    switch (act) {
        case FC_ACT_NONE: return f(std::integral_constant<int, FC_ACT_NONE>());
        case FC_ACT_RELU: return f(std::integral_constant<int, FC_ACT_RELU>());
        case FC_ACT_SILU: return f(std::integral_constant<int, FC_ACT_SILU>());
        case FC_ACT_GELU: return f(std::integral_constant<int, FC_ACT_GELU>());
        case FC_ACT_GELU_TANH: return f(std::integral_constant<int, FC_ACT_GELU_TANH>());
        default: return f(std::integral_constant<int, FC_ACT_SIGMOID>());
    }
}

// Calls f(T()) for a run-time element type.
template <typename F>
int with_type(int type, F &&f) {
    switch (type) {
        case FC_DTYPE_BF16: return f(__nv_bfloat16());
        case FC_DTYPE_F16: return f(__half());
        default: return f(float());
    }
}

// Makes the context's device current for one call and puts the caller's back.
class DeviceScope {
   public:
    explicit DeviceScope(int device) : before_(-1) {
        if (cudaGetDevice(&before_) != cudaSuccess) before_ = -1;
        status_ = before_ == device ? cudaSuccess : cudaSetDevice(device);
        if (before_ == device) before_ = -1;
    }
    ~DeviceScope() {
        if (before_ >= 0) cudaSetDevice(before_);
    }
    cudaError_t status() const { return status_; }

   private:
    int before_;
    cudaError_t status_;
};

// A bump allocator over the workspace that the caller passed; with a null base it only counts.
struct Carver {
    uint8_t *base;
    size_t used;
    template <typename T>
    T *take(size_t elems) {
        const size_t at = used;
        used += (elems * sizeof(T) + 255) & ~(size_t)255;
        return base ? reinterpret_cast<T *>(base + at) : nullptr;
    }
};

}  // namespace last
}  // namespace fc
