// Shared pieces of the channels-last operators (fc_map_move.cu, fc_group_norm.cu, fc_gated_ff*.cu): element types,
// vectors of them, activations with their derivatives, and the host-side checks.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <initializer_list>

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
    static __device__ __forceinline__ void load2(const __nv_bfloat16 *from, float &a, float &b) {
        const uint32_t w = *reinterpret_cast<const uint32_t *>(from);  // a bf16 is the upper half of its fp32
        a = __uint_as_float(w << 16);
        b = __uint_as_float(w & 0xffff0000u);
    }
    static __device__ __forceinline__ void store2(__nv_bfloat16 *to, float a, float b) {
        *reinterpret_cast<__nv_bfloat162 *>(to) = __floats2bfloat162_rn(a, b);
    }
};
template <>
struct Elem<__half> {
    static constexpr int kType = FC_DTYPE_F16;
    static __device__ __forceinline__ float load(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half store(float v) { return __float2half_rn(v); }
    static __device__ __forceinline__ void load2(const __half *from, float &a, float &b) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(from));
        a = f.x;
        b = f.y;
    }
    static __device__ __forceinline__ void store2(__half *to, float a, float b) {
        *reinterpret_cast<__half2 *>(to) = __floats2half2_rn(a, b);
    }
};

// N neighbouring elements, moved with one access (N * sizeof(T) is 2, 4, 8 or 16 bytes and the address a multiple of it)
template <int BYTES>
struct Word;
template <>
struct Word<16> { typedef uint4 type; };
template <>
struct Word<8> { typedef uint2 type; };
template <>
struct Word<4> { typedef uint32_t type; };
template <>
struct Word<2> { typedef uint16_t type; };

template <typename T, int N>
struct alignas(N * sizeof(T)) Vec {
    T v[N];
    typedef typename Word<N * sizeof(T)>::type W;
    static __device__ __forceinline__ Vec load(const void *p) {
        Vec r;
        *reinterpret_cast<W *>(&r) = *reinterpret_cast<const W *>(p);
        return r;
    }
    __device__ __forceinline__ void store(void *p) const { *reinterpret_cast<W *>(p) = *reinterpret_cast<const W *>(this); }
    __device__ __forceinline__ void unpack(float (&f)[N]) const {
        if constexpr (sizeof(T) == 2 && N % 2 == 0) {
#pragma unroll
            for (int i = 0; i < N; i += 2) Elem<T>::load2(v + i, f[i], f[i + 1]);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) f[i] = Elem<T>::load(v[i]);
        }
    }
    __device__ __forceinline__ void pack(const float (&f)[N]) {
        if constexpr (sizeof(T) == 2 && N % 2 == 0) {
#pragma unroll
            for (int i = 0; i < N; i += 2) Elem<T>::store2(v + i, f[i], f[i + 1]);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = Elem<T>::store(f[i]);
        }
    }
};

inline size_t dtype_size(int type) { return type == FC_DTYPE_F32 ? 4 : 2; }
inline bool dtype_ok(int type) { return type >= FC_DTYPE_F32 && type <= FC_DTYPE_F16; }
inline bool act_ok(int act) { return act >= FC_ACT_NONE && act <= FC_ACT_SIGMOID; }
inline bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

// The upper part of a value that is to be the sum of bf16 values: to nearest, but never up to infinity.
__device__ __forceinline__ float bf16_part(float v) {
    const float p = __bfloat162float(__float2bfloat16_rn(v));
    return fabsf(v) <= 3.4028234e38f && !(fabsf(p) <= 3.4028234e38f) ? __uint_as_float(__float_as_uint(v) & 0xffff0000u) : p;
}

// ---- activations ------------------------------------------------------------------------------------------------
// kExact: the library's functions, for results that are kept in fp32.  Otherwise the hardware's power of two and
// reciprocal (a few units in the 23rd bit, 1 + |z| times as many where exp's argument is large; GELU 1.4e-6 and z^2 2^-22; subnormals
// as zero), for results that are rounded to 8 or 11 bits anyway: two instructions of the special-function unit instead of
// some twenty.
__device__ __forceinline__ float fast_exp(float z) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(z * 1.44269504088896341f));
    return r;
}
// the larger and the smaller of two; a NaN stays one
__device__ __forceinline__ float at_least(float z, float low) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(z), "f"(low));
    return r;
}
__device__ __forceinline__ float at_most(float z, float high) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(z), "f"(high));
    return r;
}
template <bool kExact>
__device__ __forceinline__ float sigmoid(float z) {
    // exp(-z) = inf for very negative z: the quotient is then 0, as it should be
    if (kExact) return 1.0f / (1.0f + expf(-z));
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + fast_exp(-z)));
    return r;
}

// erfc(x) exp(x^2) for 0 <= x <= 9.2 (GELU down to z = -13, where it leaves the type's range) to 1.4e-6 of its value, so that
// GELU's tail is right relative to itself: t P(t) with t = 1 / (1 + 0.38 x), the seven coefficients fitted for the smallest relative
// error by weighted least squares whose weights follow the error (Lawson's iteration).  With five a fit reaches 4e-5, with
// eight 4e-7.
__device__ __forceinline__ float erfc_scaled(float x) {
    float t;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(fmaf(0.38f, x, 1.0f)));
    float p = fmaf(-0.124917876f, t, 0.334109922f);
    p = fmaf(p, t, -0.066917909f);
    p = fmaf(p, t, 0.245439537f);
    p = fmaf(p, t, 0.181628259f);
    p = fmaf(p, t, 0.216349916f);
    p = fmaf(p, t, 0.214307148f);
    return p * t;
}
// the normal distribution's function at z, and its density
template <bool kExact>
__device__ __forceinline__ void normal(float z, float &cdf, float &density) {
    if (kExact) {
        cdf = 0.5f * erfcf(-0.70710678118654752f * z);  // erfc keeps the digits of the tail
        density = 0.39894228040143268f * expf(-0.5f * z * z);
    } else {
        const float e = fast_exp(-0.5f * z * z);
        const float tail = 0.5f * e * erfc_scaled(0.70710678118654752f * fabsf(z));
        cdf = z < 0.0f ? tail : 1.0f - tail;
        density = 0.39894228040143268f * e;
    }
}

// act(z); kAct is an fc_activation.  A NaN stays one in every activation.
template <int kAct, bool kExact>
__device__ __forceinline__ float act_value(float z) {
    if (kAct == FC_ACT_RELU) return z < 0.0f ? 0.0f : z;
    if (kAct == FC_ACT_SILU) return z * sigmoid<kExact>(z);
    if (kAct == FC_ACT_GELU) {
        float cdf, density;
        normal<kExact>(z, cdf, density);
        return z * cdf;
    }
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
        float cdf, density;
        normal<kExact>(z, cdf, density);
        a = z * cdf;
        d = fmaf(z, density, cdf);
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

// the same for an activation that is known at run time only
__device__ __forceinline__ void act_both_rt(int act, float z, float &a, float &d) {
    switch (act) {
        case FC_ACT_RELU: return act_both<FC_ACT_RELU, true>(z, a, d);
        case FC_ACT_SILU: return act_both<FC_ACT_SILU, true>(z, a, d);
        case FC_ACT_GELU: return act_both<FC_ACT_GELU, true>(z, a, d);
        case FC_ACT_GELU_TANH: return act_both<FC_ACT_GELU_TANH, true>(z, a, d);
        case FC_ACT_SIGMOID: return act_both<FC_ACT_SIGMOID, true>(z, a, d);
        default: return act_both<FC_ACT_NONE, true>(z, a, d);
    }
}

// ---- pairs ------------------------------------------------------------------------------------------------------
// Two fp32 values in one 64-bit register: one instruction adds, multiplies or multiplies and adds both, each half rounded
// like the scalar instruction.
typedef uint64_t Pair;
__device__ __forceinline__ Pair pair(float a, float b) {
    Pair r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 split(Pair p) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p));
    return f;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
    Pair r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
    Pair r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
template <typename T, int N>
__device__ __forceinline__ void unpack_pairs(const Vec<T, N> &v, Pair (&p)[N / 2]) {
    float f[N];
    v.unpack(f);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) p[i] = pair(f[2 * i], f[2 * i + 1]);
}
template <typename T, int N>
__device__ __forceinline__ void pack_pairs(Vec<T, N> &v, const Pair (&p)[N / 2]) {
    float f[N];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        const float2 h = split(p[i]);
        f[2 * i] = h.x;
        f[2 * i + 1] = h.y;
    }
    v.pack(f);
}
// Two sigmoids with one reciprocal: 1/a = b/(ab), 1/b = a/(ab).  The exponentials are bounded by 2^60 so that the product is
// finite (and a NaN stays in its half: z itself is multiplied in later); a sigmoid below 2^-60 comes out as 2^-60, and what is
// multiplied by it is bounded from below (low_bounded) so that the product stays at nothing for any z.  The
// special-function unit, which gives four results a clock to a quarter of an SM, is what the activations wait for.
__device__ __forceinline__ Pair sigmoid_fast2(Pair z) {
    const float2 t = split(mul2(z, pair(-1.44269504088896341f, -1.44269504088896341f)));
    float a, b, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(a) : "f"(fminf(t.x, 60.0f)));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(b) : "f"(fminf(t.y, 60.0f)));
    const float2 u = split(add2(pair(a, b), pair(1.0f, 1.0f)));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(u.x * u.y));
    return mul2(pair(r, r), pair(u.y, u.x));
}
__device__ __forceinline__ Pair low_bounded(Pair z) {
    const float2 f = split(z);
    return pair(at_least(f.x, -64.0f), at_least(f.y, -64.0f));
}
__device__ __forceinline__ Pair gelu_tanh_argument(Pair z) {  // sqrt(8 / pi) (z + 0.044715 z^3), |z| bounded in the cube
    const float2 q = split(mul2(z, z));
    const Pair t = pair(fminf(q.x, 1e6f), fminf(q.y, 1e6f));
    const Pair k = pair(0.044715f * 1.59576912160573071f, 0.044715f * 1.59576912160573071f);
    return mul2(z, fma2(t, k, pair(1.59576912160573071f, 1.59576912160573071f)));
}
template <int kAct, bool kExact>
__device__ __forceinline__ Pair act_value2(Pair z) {
    if (kAct == FC_ACT_NONE) return z;
    if (kAct == FC_ACT_SILU && !kExact) return mul2(low_bounded(z), sigmoid_fast2(z));
    if (kAct == FC_ACT_GELU_TANH && !kExact) return mul2(low_bounded(z), sigmoid_fast2(gelu_tanh_argument(z)));
    const float2 f = split(z);
    return pair(act_value<kAct, kExact>(f.x), act_value<kAct, kExact>(f.y));
}
template <int kAct, bool kExact>
__device__ __forceinline__ void act_both2(Pair z, Pair &a, Pair &d) {
    if (kAct == FC_ACT_SILU && !kExact) {
        const Pair s = sigmoid_fast2(z), one = pair(1.0f, 1.0f), minus = pair(-1.0f, -1.0f);
        a = mul2(low_bounded(z), s);
        d = fma2(a, fma2(s, minus, one), s);
        return;
    }
    const float2 f = split(z);
    float a0, a1, d0, d1;
    act_both<kAct, kExact>(f.x, a0, d0);
    act_both<kAct, kExact>(f.y, a1, d1);
    a = pair(a0, a1);
    d = pair(d0, d1);
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

// Refuses an output that begins where an input or another output does (NULL: absent).  Maps may lie in one another's gaps, so
// ranges are not compared.
inline int check_outputs(std::initializer_list<const void *> outputs, std::initializer_list<const void *> inputs) {
    for (const void *const *o = outputs.begin(); o != outputs.end(); ++o) {
        if (*o == nullptr) continue;
        for (const void *i : inputs) FC_REQUIRE(*o != i, FC_ERR_INVALID_ARG, "an output is an input");
        for (const void *const *p = outputs.begin(); p != o; ++p)
            FC_REQUIRE(*o != *p, FC_ERR_INVALID_ARG, "two outputs are one");
    }
    return FC_OK;
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

// Lets the next kernel of the stream begin its set-up (barriers, tensor memory, descriptors) on SMs that this one leaves
// free or has left; it touches nothing of this one's before its own pdl_wait().  Every block says so after its own wait, which
// keeps the chain: a kernel ends only after the one before it.  What another kernel may have written is read by plain loads, not
// through the read-only path (ld.global.nc, which __ldg and pointers to const that are __restrict__ turn into): it has to stand
// still from a kernel's start on, not from its wait on.
__device__ __forceinline__ void pdl_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Launches of kernels that call pdl_next(), in stream order like every other (programmatic dependent launch); the context
// remembers that it has had one.
template <typename... KArgs, typename... Args>
inline cudaError_t launch_early(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, fc_context *ctx, Args &&...args) {
    ctx->signals_early = true;
    return launch_programmatic(pdl_enabled(), kernel, grid, block, smem, ctx->stream, static_cast<Args &&>(args)...);
}
// in clusters of `cluster` blocks
template <typename... KArgs, typename... Args>
inline cudaError_t launch_clusters(void (*kernel)(KArgs...), dim3 grid, unsigned threads, unsigned cluster, size_t smem,
                                   fc_context *ctx, Args &&...args) {
    ctx->signals_early = true;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, KArgs(args)...);
}

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
