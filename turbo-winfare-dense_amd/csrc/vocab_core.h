// What the kernels of the vocabulary matrix share: vector types, the floating types of rows, the softcap, buffer
// resources and loads into LDS.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

namespace twd {

namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

// fp32 -> bf16 bits, round to nearest even (NaN stays NaN)
__device__ __forceinline__ uint32_t bf16_bits(float v) {
    const uint32_t u = __float_as_uint(v);
    if (v != v) return (u >> 16) | 0x40u;
    return (u + 0x7FFFu + ((u >> 16) & 1u)) >> 16;
}

// Two floats as bf16 in a word, each rounded to nearest even (NaN stays NaN), in one instruction.
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
    typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, bf16x2_t{static_cast<__bf16>(lo), static_cast<__bf16>(hi)});
}

// f(0) .. f(N - 1), the numbers known to the compiler: for sums in registers, which have no index.
template <int N, typename F>
__device__ __forceinline__ void each(F&& f) {
    if constexpr (N > 0) {
        each<N - 1>(f);
        f(std::integral_constant<int, N - 1>{});
    }
}

template <typename T>
struct Eight;
template <>
struct Eight<float> {
    static constexpr uint32_t kBytes = 32;
    __device__ static void load(const float* p, bool wide, float* v) {
        if (wide) {
            const f32x4_t a = reinterpret_cast<const f32x4_t*>(p)[0], b = reinterpret_cast<const f32x4_t*>(p)[1];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = p[i];
        }
    }
};
struct Bf16 {
    uint16_t u;
};
struct Fp16 {
    _Float16 h;
};
template <typename T>
__device__ __forceinline__ float half_to_f32(uint32_t bits);
template <>
__device__ __forceinline__ float half_to_f32<Bf16>(uint32_t bits) { return __uint_as_float(bits << 16); }
template <>
__device__ __forceinline__ float half_to_f32<Fp16>(uint32_t bits) {
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(bits)));
}
template <typename T>
__device__ __forceinline__ uint32_t f32_to_half(float v);
template <>
__device__ __forceinline__ uint32_t f32_to_half<Bf16>(float v) { return bf16_bits(v); }
template <>
__device__ __forceinline__ uint32_t f32_to_half<Fp16>(float v) {
    return __builtin_bit_cast(uint16_t, static_cast<_Float16>(v));
}
template <typename T>
struct Eight {
    static constexpr uint32_t kBytes = 16;
    __device__ static void load(const T* p, bool wide, float* v) {
        if (wide) {
            const u32x4_t a = *reinterpret_cast<const u32x4_t*>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[2 * i] = half_to_f32<T>(a[i] & 0xFFFFu), v[2 * i + 1] = half_to_f32<T>(a[i] >> 16);
        } else {
            const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = half_to_f32<T>(q[i]);
        }
    }
};

// A softcap's reciprocal and its multiples stay normal numbers.
constexpr float kMinSoftCap = 1e-30f, kMaxSoftCap = 1e30f;

struct SoftCap {
    float cap, inv, twice;  // cap (0: none), 1 / cap, 2 log2(e) / cap
};

inline SoftCap soft_cap(float cap) {
    const double c = cap > 0.0f ? cap : 1.0;
    return SoftCap{cap, static_cast<float>(1.0 / c), static_cast<float>(2.8853900817779268 / c)};
}

// cap * tanh(v / cap) of N logits. Below the cap it is v + v t^2 r(t^2) with t = v / cap, r the polynomial
// through (tanh(t)/t - 1)/t^2 at nine Chebyshev nodes of t^2 in 0..1: v itself enters the last sum exactly,
// so the roundings of t count for less than half (at most 3 * 2^-24 of the result in all, 1.8 seen). Past
// the cap it is cap - 2 cap / (exp(2 |t|) + 1), where the subtracted part is at most 0.31 of the result
// (3.6 * 2^-24). A wave takes the second way only if one of its logits needs it. tanhf(v / cap) spent 36
// instructions on every logit, as much time as the products of a tile of 2,048 columns.
template <int N>
__device__ __forceinline__ void cap_logits(float (&y)[N], const SoftCap& c) {
    if (!(c.cap > 0.0f)) return;
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) top = fmaxf(top, fabsf(y[i]));
    const bool past = __builtin_amdgcn_ballot_w64(top > c.cap) != 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float v = y[i], t = v * c.inv, t2 = t * t;
        float p = -4.8467110900674015e-05f;
        p = fmaf(p, t2, 0.000337689823936671f);
        p = fmaf(p, t2, -0.0012421574375301295f);
        p = fmaf(p, t2, 0.00347838643938303f);
        p = fmaf(p, t2, -0.008826250210404396f);
        p = fmaf(p, t2, 0.0218625757843256f);
        p = fmaf(p, t2, -0.05396759510040283f);
        p = fmaf(p, t2, 0.13333331048488617f);
        p = fmaf(p, t2, -0.3333333432674408f);
        float z = fmaf(v * t2, p, v);
        if (past) {
            const float e = __builtin_amdgcn_exp2f(fabsf(v) * c.twice);  // past 2^128: 1 / inf is 0
            const float w = fmaf(-2.0f * c.cap, __builtin_amdgcn_rcpf(e + 1.0f), c.cap);
            z = fabsf(v) > c.cap ? copysignf(w, v) : z;  // a NaN stays one by the first way
        }
        y[i] = z;
    }
}

__device__ __forceinline__ void store_logit(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_logit(uint16_t* p, float v) { *p = static_cast<uint16_t>(bf16_bits(v)); }

template <typename Out>
struct Sixteen {
    Out e[16 / sizeof(Out)];
};

// 16 bytes of logits at any alignment, n of them at most; they are not read here again.
template <typename Out>
__device__ __forceinline__ void store_logits(Out* p, u32x4_t v, uint32_t n) {
    constexpr uint32_t kEach = 16 / sizeof(Out);
    typedef u32x4_t __attribute__((aligned(2))) any_place_t;
    if (n >= kEach) {
        __builtin_nontemporal_store(v, reinterpret_cast<any_place_t*>(p));
    } else {
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i)
            if (i < n) p[i] = __builtin_bit_cast(Sixteen<Out>, v).e[i];
    }
}

// A barrier that waits for the wave's LDS accesses only: loads on their way into registers stay in flight.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

constexpr int kStreamed = 2;  // a buffer access that is not read again: non-temporal
// What the cache on the memory's side holds: weights up to this size are found there by the next call, and streaming them
// would lose that.
constexpr uint64_t kMemoryCache = 256ull << 20;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const void* p, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, static_cast<int>(bytes), 0x00027000);
}

// The target of a load straight into LDS.
typedef __attribute__((address_space(3))) void lds_void;

constexpr int kVmcnt0 = 0x0F70;  // s_waitcnt vmcnt(0), no other counter

}  // namespace

}  // namespace twd
