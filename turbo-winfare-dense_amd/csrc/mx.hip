// Microscaled 4-bit floating point: rows quantised to the format and back, and the LM head's product
// with weights held in it.
//
// The format (OCP Microscaling, MXFP4): a block is 32 consecutive columns of a row under one scale
// byte s, the power of two 2^(s - 127) (255: NaN); an element is 4 bits, sign | exponent (2) |
// mantissa (1), of magnitude 0, 0.5, 1, 1.5, 2, 3, 4, 6. Two elements share a byte, the lower column
// in the lower four bits. With A the block's largest magnitude the scale's exponent is
// e = floor(log2 A) - 2, which brings A into [4, 8); an element is x 2^-e rounded to the nearest
// magnitude, ties to the even code, 6 above that.
#include <hip/hip_runtime.h>

#include <new>
#include <string>

#include "twd_internal.h"
#include "twd_mx.h"

namespace twd {

namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

constexpr uint32_t kMxBlock = 32;
constexpr uint32_t kNanScale = 255;

// fp32 -> bf16 bits, round to nearest even (NaN stays NaN)
__device__ __forceinline__ uint32_t bf16_bits(float v) {
    const uint32_t u = __float_as_uint(v);
    if (v != v) return (u >> 16) | 0x40u;
    return (u + 0x7FFFu + ((u >> 16) & 1u)) >> 16;
}

// 2^(s - 127) of a scale byte as a float: the byte is the float's own exponent field, but for 0
// (2^-127 is a subnormal float) and 255 (NaN).
__device__ __forceinline__ float scale_value(uint32_t s) {
    return s == 0 ? 0x1p-127f : __uint_as_float(s == kNanScale ? 0x7FC00000u : s << 23);
}

// ---- rows to codes and scales, and back -----------------------------------------------------------
//
// Eight consecutive elements per lane, so four lanes hold a block: its largest magnitude is two
// exchanges inside a quad of lanes. The pass is bound by its reads: 151,669 x 3,584 fp32 values in 484 us
// (5.1 TB/s, reads and writes; a copy reaches 4.8), 777 x 2,880 fp16 in 4.3 us, one row in 2.1.

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

// The element nearest y, ties to the even code. From 1 on the codes are a float's exponent and first
// mantissa bit, so the float is rounded to that bit; below 1 they count steps of 0.5.
__device__ __forceinline__ uint32_t encode(float y) {
    const uint32_t u = __float_as_uint(y), m = u & 0x7FFFFFFFu;
    const uint32_t r = ((m + 0x1FFFFFu + ((m >> 22) & 1u)) >> 22) - 252u;
    const uint32_t low = static_cast<uint32_t>(__builtin_rintf(2.0f * __uint_as_float(m)));
    const uint32_t c = m >= 0x3F800000u ? (r < 7u ? r : 7u) : low;
    return c | ((u >> 28) & 8u);
}

struct QuantArgs {
    const void* x;
    uint64_t stride;  // elements between rows
    uint64_t rows;
    uint32_t groups;  // groups of eight columns in a row
    uint8_t* codes;
    uint8_t* scales;
    bool wide;  // rows start at multiples of 16 bytes
};

constexpr uint32_t kQuantThreads = 256;

template <typename T>
__global__ __launch_bounds__(kQuantThreads) void mx_quantize_kernel(QuantArgs a) {
    const uint32_t g = blockIdx.x * kQuantThreads + threadIdx.x;  // a whole block's four lanes lie in or out together
    if (g >= a.groups) return;
    for (uint64_t r = blockIdx.y; r < a.rows; r += gridDim.y) {
        float v[8];
        Eight<T>::load(static_cast<const T*>(a.x) + r * a.stride + 8ull * g, a.wide, v);
        uint32_t top = 0;  // magnitudes order as their bits do, infinity and NaN above all
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t m = __float_as_uint(v[i]) & 0x7FFFFFFFu;
            top = m > top ? m : top;
        }
        uint32_t o = dpp_move<0xB1>(top, top);
        top = o > top ? o : top;
        o = dpp_move<0x4E>(top, top);
        top = o > top ? o : top;
        // floor(log2 A) is the exponent field less 127; a subnormal A gives less than -126, and every
        // exponent below -125 the clamp's -127 alike
        const int e = static_cast<int>(top >> 23) - 129;
        const uint32_t s = top >= 0x7F800000u ? kNanScale : (e < -127 ? 0u : static_cast<uint32_t>(e + 127));
        const float inv = __uint_as_float((254u - s) << 23);  // 2^-e, exact: s is at most 252
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) w |= encode(v[i] * inv) << (4 * i);
        if (s == kNanScale) w = 0;
        reinterpret_cast<uint32_t*>(a.codes)[r * a.groups + g] = w;
        if (g % 4 == 0) a.scales[r * (a.groups / 4) + g / 4] = static_cast<uint8_t>(s);
    }
}

struct DequantArgs {
    const uint8_t* codes;
    const uint8_t* scales;
    uint64_t rows;
    uint32_t pieces;  // of 16 bytes of values in a row
    void* out;
    uint64_t stride;
    bool wide;  // rows start at multiples of 16 bytes
};

// The magnitude bits c as a float's exponent and first mantissa bit are the element's value times
// 2^-126 (a subnormal float for 0.5), so one exact product by 2^126 decodes it.
__device__ __forceinline__ float decode(uint32_t c, float s) {
    return __uint_as_float(((c & 7u) << 22) | ((c & 8u) << 28)) * 0x1p126f * s;
}

// A lane writes 16 bytes, so that a wave's store fills whole lines; the pass is bound by them, and they are not
// read here again: 151,669 x 3,584 fp32 values in 523 us (4.7 TB/s); 32 bytes a lane, two stores half a line apart,
// took 693.
template <typename T>
__global__ __launch_bounds__(kQuantThreads) void mx_dequantize_kernel(DequantArgs a) {
    constexpr uint32_t kEach = 16 / sizeof(T);
    const uint32_t g = blockIdx.x * kQuantThreads + threadIdx.x;
    if (g >= a.pieces) return;
    for (uint64_t r = blockIdx.y; r < a.rows; r += gridDim.y) {
        const uint64_t at = r * a.pieces + g;
        const uint32_t w = kEach == 8 ? reinterpret_cast<const uint32_t*>(a.codes)[at] : reinterpret_cast<const uint16_t*>(a.codes)[at];
        const float s = scale_value(a.scales[at * kEach / kMxBlock]);
        float v[kEach];
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) v[i] = decode(w >> (4 * i), s);
        T* out = static_cast<T*>(a.out) + r * a.stride + kEach * g;
        u32x4_t bits;
        if constexpr (kEach == 8) {
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) bits[i] = f32_to_half<T>(v[2 * i]) | (f32_to_half<T>(v[2 * i + 1]) << 16);
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) bits[i] = __float_as_uint(v[i]);
        }
        if (a.wide) {
            __builtin_nontemporal_store(bits, reinterpret_cast<u32x4_t*>(out));
        } else if constexpr (kEach == 8) {
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) reinterpret_cast<uint16_t*>(out)[i] = static_cast<uint16_t>(bits[i / 2] >> (16 * (i % 2)));
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) reinterpret_cast<uint32_t*>(out)[i] = bits[i];
        }
    }
}

// ---- the head's layout in HBM ---------------------------------------------------------------------
//
// A group is 64 vocabulary rows, four tiles of 16; a chunk is 128 columns, four blocks; a quad is four
// chunks. Both matrix instructions used here (16x16x128 on 4-bit operands, and four 16x16x32 on bf16 ones,
// whose columns may be taken in any order as long as both operands agree) let lane l = 16 kg + r hold row
// r's block kg of a chunk:
//   codes  [group][chunk][tile][lane] 16 bytes, the block's 32 elements
//   scales [group][quad][tile][lane] 4 bytes, byte c the scale of that lane's block in the quad's chunk c
// so a load instruction of a wave moves 1 KB (codes) or 256 B (scales) of contiguous memory, and every
// lane's elements share the lane's own scale. Row r of tile j is the group's vocabulary row
// 16 (r / 4) + 4 j + r % 4: a product's lane then holds, over the four tiles, 16 logits in a row of one
// hidden row. Rows past the vocabulary and columns past d_model are zero codes with scale byte 0 (2^-127).
constexpr uint32_t kMxChunkK = 128;
constexpr uint32_t kMxGroupRows = 64;

__device__ __forceinline__ uint32_t group_row(uint32_t tile, uint32_t r) { return 16 * (r / 4) + 4 * tile + r % 4; }

// Once a head, a block to a group; 262,144 x 5,376 in 380 us.
__global__ __launch_bounds__(256) void mx_repack_kernel(const uint8_t* __restrict__ codes,
                                                       const uint8_t* __restrict__ scales, uint32_t vocab,
                                                       uint32_t d, uint32_t chunks, u32x4_t* __restrict__ out_codes,
                                                       uint32_t* __restrict__ out_scales, uint32_t* bad) {
    const uint32_t lane = threadIdx.x % 64, tile = threadIdx.x / 64, kg = lane / 16, r = lane % 16;
    const uint32_t blocks = d / kMxBlock, quads = (chunks + 3) / 4;
    const uint64_t group = blockIdx.x;
    const uint64_t row = group * kMxGroupRows + group_row(tile, r);
    for (uint32_t q = 0; q < quads; ++q) {
        uint32_t sc = 0;
        for (uint32_t c = 0; c < 4; ++c) {
            const uint32_t chunk = 4 * q + c, b = 4 * chunk + kg;
            if (chunk >= chunks) break;
            u32x4_t w = {0, 0, 0, 0};
            if (row < vocab && b < blocks) {
                w = *reinterpret_cast<const u32x4_t*>(codes + row * (d / 2) + 16ull * b);
                const uint32_t s = scales[row * blocks + b];
                if (s > 227u) *bad = 1;  // above 2^100, NaN among them
                sc |= s << (8 * c);
            }
            out_codes[((group * chunks + chunk) * 4 + tile) * 64 + lane] = w;
        }
        out_scales[((group * quads + q) * 4 + tile) * 64 + lane] = sc;
    }
}

}  // namespace

}  // namespace twd

struct twd_mxhead {
    uint32_t vocab, d, chunks, quads, groups;
    float softcap;
    int device;
    int cus;
    twd::u32x4_t* codes;
    uint32_t* scales;
    uint64_t bytes;
};

namespace twd {

namespace {

// A softcap's reciprocal and its multiples stay normal numbers.
constexpr float kMinSoftCap = 1e-30f, kMaxSoftCap = 1e30f;

struct SoftCap {
    float cap, inv, twice;  // cap (0: none), 1 / cap, 2 log2(e) / cap
};

SoftCap soft_cap(float cap) {
    const double c = cap > 0.0f ? cap : 1.0;
    return SoftCap{cap, static_cast<float>(1.0 / c), static_cast<float>(2.8853900817779268 / c)};
}

struct MxArgs {
    const u32x4_t* codes;
    const uint32_t* scales;
    const void* x;  // bf16 rows, or codes [rows][d / 2]
    const uint8_t* xs;
    uint64_t x_stride;
    void* out;
    uint64_t out_stride;
    uint32_t vocab, d, chunks, quads, groups, rows;
    SoftCap softcap;
};

__device__ __forceinline__ void store_logit(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_logit(uint16_t* p, float v) { *p = static_cast<uint16_t>(bf16_bits(v)); }

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

__device__ __forceinline__ i32x8_t mx_operand(u32x4_t v) {  // 4-bit operands fill half the registers
    const i32x4_t x = __builtin_bit_cast(i32x4_t, v);
    return __builtin_shufflevector(x, x, 0, 1, 2, 3, -1, -1, -1, -1);
}

// One chunk's product of a 16-row weight tile and 16 quantised hidden rows; C: which byte of the weights'
// scale word. The hidden rows' scale is the low byte of xs.
template <int C>
__device__ __forceinline__ f32x4_t mfma_mx(u32x4_t w, uint32_t ws, u32x4_t x, uint32_t xs, f32x4_t acc) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_operand(w), mx_operand(x), acc, 4, 4, C,
                                                            static_cast<int>(ws), 0, static_cast<int>(xs));
}

// Eight elements of a code word times their scale, exact in bf16.
__device__ __forceinline__ bf16x8_t widen(uint32_t w, float s) {
    u32x4_t e;
    e[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0));
    e[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1));
    e[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2));
    e[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3));
    return __builtin_bit_cast(bf16x8_t, e);
}
// The scale of byte c as the conversion reads it, by its exponent field alone: 0 is 2^-127 there.
__device__ __forceinline__ float scale_float(uint32_t word, int c) { return __uint_as_float(((word >> (8 * c)) & 255u) << 23); }

// A barrier that waits for the wave's LDS accesses only: loads on their way into registers stay in flight.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

constexpr int kStreamed = 2;  // non-temporal: read once
__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const void* p, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, static_cast<int>(bytes), 0x00027000);
}

// ---- up to 16 hidden rows: the weights stream past rows held in registers ---------------------------
//
// Bound by the read of the head. The waves of a block split d_model by quads: a wave keeps its quad of the
// hidden rows in registers for the whole launch and streams its quad of one group after another, kRing
// chunks (4 KB each) ahead of the arithmetic. The sums over the quads meet in LDS, two buffers in turn, so
// that one barrier a group is enough and no load waits at it. Where d_model has few quads, several blocks
// share a compute unit (as one block of several groups, 32,003 x 2,048 left a third of the units idle: 10.5 us
// instead of 8.6). One row of 262,144 x 5,376: 115 to 117 us,
// 6.4 to 6.5 TB/s, of the 6.7 that a pure read reaches (a first, simple kernel took 193);
// 7 quantised rows of 151,669 x 3,584: 46 us, 6.3 TB/s; one row of 32,003 x 2,048: 7.7 to 8.3 us, where a wave's first
// bytes and the end of the launch are half of it.
constexpr uint32_t kSmallRows = 16;
constexpr uint32_t kSmallWaves = 12;  // 168 registers each
constexpr uint32_t kRing = 4;

template <bool MX, typename Out>
__global__ __launch_bounds__(kSmallWaves * 64) void mx_small_kernel(MxArgs a) {
    extern __shared__ float part[];  // [2][quad][row][64]
    const uint32_t lane = threadIdx.x % 64, kg = lane / 16, r = lane % 16;
    const uint32_t quad = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t blocks = a.d / kMxBlock;
    const uint32_t here = min(4u, a.chunks - 4 * quad);  // chunks of this wave

    u32x4_t x[MX ? 4 : 16] = {};
    uint32_t xs[MX ? 4 : 1] = {};
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const uint32_t b = 16 * quad + 4 * c + kg;
        if (r < a.rows && b < blocks) {
            if constexpr (MX) {
                x[c] = *reinterpret_cast<const u32x4_t*>(static_cast<const uint8_t*>(a.x) + r * (a.d / 2ull) + 16ull * b);
                xs[c] = a.xs[static_cast<uint64_t>(r) * blocks + b];
            } else {
                const uint16_t* row = static_cast<const uint16_t*>(a.x) + r * a.x_stride + 32ull * b;
#pragma unroll
                for (int t = 0; t < 4; ++t) x[4 * c + t] = *reinterpret_cast<const u32x4_t*>(row + 8 * t);
            }
        }
    }

    // Buffer loads: the base in scalar registers, one lane offset for all. Past the quad's end (the last quad)
    // the last chunk comes again, whose hidden columns are zero.
    // A group past the last has no bytes, so nothing is read of it.
    auto codes_of = [&](uint32_t g) {
        return make_rsrc(a.codes + (static_cast<uint64_t>(g) * a.chunks + 4 * quad) * 256, g < a.groups ? here * 4096 : 0);
    };
    auto scales_of = [&](uint32_t g) {
        return make_rsrc(a.scales + (static_cast<uint64_t>(g) * a.quads + quad) * 256, g < a.groups ? 1024 : 0);
    };
    auto load_codes = [&](const __amdgpu_buffer_rsrc_t& at, uint32_t c, u32x4_t (&to)[4]) {
        const int chunk = static_cast<int>(min(c, here - 1) * 4096);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            to[j] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(at, lane * 16 + 1024 * j, chunk, kStreamed));
    };
    auto load_scales = [&](const __amdgpu_buffer_rsrc_t& at, uint32_t (&to)[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) to[j] = __builtin_amdgcn_raw_buffer_load_b32(at, lane * 4 + 256 * j, 0, kStreamed);
    };
    u32x4_t w[kRing][4];
    uint32_t ws[4];
    {
        const auto codes = codes_of(blockIdx.x), scales = scales_of(blockIdx.x);
#pragma unroll
        for (uint32_t c = 0; c < kRing; ++c) {
            load_codes(codes, c, w[c]);
            if (c == 0) load_scales(scales, ws);
            __builtin_amdgcn_sched_barrier(0);  // the loads in the order of their use, here and in every turn
        }
    }
    uint32_t buf = 0;
    for (uint32_t g = blockIdx.x; g < a.groups; g += gridDim.x) {
        const auto codes = codes_of(g + gridDim.x), scales = scales_of(g + gridDim.x);
        f32x4_t acc[4] = {};
        uint32_t s[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j] = ws[j];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (MX) {
                    if (c == 0) acc[j] = mfma_mx<0>(w[c][j], s[j], x[c], xs[c], acc[j]);
                    if (c == 1) acc[j] = mfma_mx<1>(w[c][j], s[j], x[c], xs[c], acc[j]);
                    if (c == 2) acc[j] = mfma_mx<2>(w[c][j], s[j], x[c], xs[c], acc[j]);
                    if (c == 3) acc[j] = mfma_mx<3>(w[c][j], s[j], x[c], xs[c], acc[j]);
                } else {
                    const float f = scale_float(s[j], c);
#pragma unroll
                    for (int t = 0; t < 4; ++t)
                        acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                            widen(w[c][j][t], f), __builtin_bit_cast(bf16x8_t, x[4 * c + t]), acc[j], 0, 0, 0);
                    __builtin_amdgcn_sched_barrier(0);  // one tile's widened codes at a time
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            load_codes(codes, c, w[c]);
            if (c == 0) load_scales(scales, ws);
            __builtin_amdgcn_sched_barrier(0);
        }
        float* mine = part + (buf * a.quads + quad) * a.rows * 64;
        if (r < a.rows) {
#pragma unroll
            for (int j = 0; j < 4; ++j) *reinterpret_cast<f32x4_t*>(mine + r * 64 + 16 * kg + 4 * j) = acc[j];
        }
        lds_barrier();
        // the waves share the sums: element e is hidden row e / 64, vocabulary row e % 64
        for (uint32_t e = quad * 64 + lane; e < a.rows * 64; e += a.quads * 64) {
            const float* p = part + buf * a.quads * a.rows * 64 + e;
            float y[1] = {p[0]};
            for (uint32_t q = 1; q < a.quads; ++q) y[0] += p[q * a.rows * 64];
            cap_logits(y, a.softcap);
            const uint64_t v = static_cast<uint64_t>(g) * kMxGroupRows + e % 64;
            if (v < a.vocab) store_logit(static_cast<Out*>(a.out) + (e / 64) * a.out_stride + v, y[0]);
        }
        buf ^= 1;
    }
}

// ---- more hidden rows: tiles of 256 vocabulary rows by 16 NT hidden rows -----------------------------
//
// Four waves, a group of weights each, read straight from memory a chunk ahead; the hidden rows' tile goes
// through LDS, loaded there without registers one stage ahead into the other of two buffers. A stage is a
// chunk of bf16 rows (256 bytes a row) or a quad of quantised ones (4 x 64 bytes a row and 16 scales).
//
// Times are medians over hundreds of calls in a row, from card to card. From 128 bf16 rows on bound by the matrix
// instructions, whose clock follows the socket's power: 1,023 rows of 65,537 x 2,880 in 313 to 331 us, 1,165 to 1,233
// TFLOP/s (a large library product: 1,237), with the matrix units busy in 65% of the cycles at 1.6 GHz (1,024 rows of
// 262,144 x 5,376: 1,360 TFLOP/s, 1,577 where all weights are zero). Quantised rows do not keep them busy: 2,048 of 262,144
// x 5,376 take 1,966 to 2,051 us, 2,815 to 2,936 TFLOP/s (3,008), with the matrix units busy in 32% of the cycles, at 2.1
// GHz, vector instructions issued in 41%, 9 TB/s out of the L2s; the two waves of a SIMD wait for loads and barriers in
// 26% of their time and to issue in 43%, and do not cover each other's waits. 64 bf16 rows of 262,144 x 5,376 take 176 to
// 183 us, whatever the data: 112 are the reads of the head; on the card where it took 176, 127 with its codes
// served by an L2 and 156 without the logits' stores. Codes two chunks ahead, stages of two chunks and two blocks to a
// compute unit instead of three did not bring reads and products together (within 3%).
constexpr uint32_t kTileWaves = 4;
constexpr int kVmcnt0 = 0x0F70;  // s_waitcnt vmcnt(0), no other counter

typedef __attribute__((address_space(3))) void lds_void;

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

template <bool MX, int NT, typename Out>
__global__ __launch_bounds__(kTileWaves * 64) __attribute__((amdgpu_waves_per_eu(2))) void mx_tile_kernel(MxArgs a) {
    constexpr uint32_t kRows = 16 * NT;
    constexpr uint32_t kStage = NT * 256;  // 16-byte pieces of a stage
    __shared__ u32x4_t buf0[kStage], buf1[kStage];
    __shared__ uint32_t sc0[MX ? kRows * 4 : 1], sc1[MX ? kRows * 4 : 1];
    const uint32_t lane = threadIdx.x % 64, kg = lane / 16, r = lane % 16;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    // Blocks go to the XCDs in turn. An XCD's blocks take the hidden rows' tiles of one stretch of vocabulary
    // after another, so the weights come to its L2 once; the last stretch, which may be short, goes first.
    const uint32_t row_tiles = (a.rows + kRows - 1) / kRows, stretches = (a.groups + kTileWaves - 1) / kTileWaves;
    const uint32_t xcd = blockIdx.x % 8, turn = blockIdx.x / 8;
    const uint32_t stretch_up = turn / row_tiles * 8 + xcd;
    if (stretch_up >= stretches) return;
    const uint32_t stretch = stretches - 1 - stretch_up;
    const uint32_t m0 = turn % row_tiles * kRows;
    const uint32_t group = stretch * kTileWaves + wave;
    const bool have_group = group < a.groups;
    const uint64_t g = min(group, a.groups - 1);
    const uint32_t blocks = a.d / kMxBlock;

    // The stage's hidden rows, NT pieces of 1 KB a wave: `row` and `byte` say which 16 bytes of a row's stage
    // a lane brings. bf16: [row][16 pieces], the pieces of a row exchanged by the row's number so that a
    // fragment's reads of one piece in 16 rows meet 16 different banks. Quantised: [chunk][tile][lane].
    const uint32_t row_bytes = static_cast<uint32_t>(MX ? a.d / 2 : 2 * a.x_stride);
    const uint32_t width = MX ? a.d / 2 : 2 * a.d, stages = width / 256;  // whole stages; the rest follows
    auto row_of = [&](uint32_t i) {
        const uint32_t p = i * kTileWaves + wave;
        return min(m0 + (MX ? 16 * (p % NT) + r : 4 * p + lane / 16), a.rows - 1) - m0;
    };
    auto byte_of = [&](uint32_t i) {
        const uint32_t p = i * kTileWaves + wave;
        if (MX) return 64 * (p / NT) + 16 * kg;
        const uint32_t q = (lane ^ (4 * p + lane / 16)) % 16;
        return 64 * (0x78u >> (2 * (q / 4)) & 3) + 16 * (q % 4);
    };
    const char* x0 = static_cast<const char*>(a.x) + static_cast<uint64_t>(m0) * row_bytes;
    const uint32_t rows_here = min(a.rows - m0, kRows);
    const auto rsrc = make_rsrc(x0, (rows_here - 1) * row_bytes + width);
    uint32_t off[NT];
#pragma unroll
    for (uint32_t i = 0; i < NT; ++i) off[i] = row_of(i) * row_bytes + byte_of(i);
    auto fetch = [&](uint32_t stage, u32x4_t* to) {
        const int at = __builtin_amdgcn_readfirstlane(static_cast<int>(stage * 256));
#pragma unroll
        for (uint32_t i = 0; i < NT; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void*)(to + (i * kTileWaves + wave) * 64), 16,
                                                     static_cast<int>(off[i]), at, 0, 0);
    };
    // the quantised stage's scales, [row][chunk] with four blocks' bytes each: through registers, so that they
    // too travel beside the arithmetic
    constexpr uint32_t kScales = MX ? (kRows * 4 + kTileWaves * 64 - 1) / (kTileWaves * 64) : 0;
    uint32_t sc_next[MX ? kScales : 1];
    auto fetch_scales = [&](uint32_t stage) {
#pragma unroll
        for (uint32_t i = 0; i < kScales; ++i) {
            const uint32_t e = i * kTileWaves * 64 + threadIdx.x;
            const uint32_t m = min(m0 + e / 4, a.rows - 1), b = 16 * stage + 4 * (e % 4);
            __builtin_memcpy(&sc_next[i], a.xs + static_cast<uint64_t>(m) * blocks + b, 4);
        }
    };
    auto write_scales = [&](uint32_t* to) {
#pragma unroll
        for (uint32_t i = 0; i < kScales; ++i) {
            const uint32_t e = i * kTileWaves * 64 + threadIdx.x;
            if (e < kRows * 4) to[e] = sc_next[i];
        }
    };
    f32x4_t acc[4][NT] = {};
    const auto codes = make_rsrc(a.codes + g * a.chunks * 256, a.chunks * 4096);
    const auto scales = make_rsrc(a.scales + g * a.quads * 256, a.quads * 1024);
    constexpr int kWeights = 0;  // cached: the tiles of other hidden rows read them again from the L2
    // w, ws: the chunk's codes and the quad's scales; wn, wsn: the next ones, on their way
    u32x4_t w[4], wn[4];
    uint32_t ws[4], wsn[4];
    auto load_codes = [&](uint32_t c) {
        const int at = __builtin_amdgcn_readfirstlane(static_cast<int>(min(c, a.chunks - 1) * 4096));
#pragma unroll
        for (int j = 0; j < 4; ++j)
            wn[j] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(codes, lane * 16 + 1024 * j, at, kWeights));
    };
    auto load_scales = [&](uint32_t q) {
        const int at = __builtin_amdgcn_readfirstlane(static_cast<int>(min(q, a.quads - 1) * 1024));
#pragma unroll
        for (int j = 0; j < 4; ++j) wsn[j] = __builtin_amdgcn_raw_buffer_load_b32(scales, lane * 4 + 256 * j, at, kWeights);
    };
    // x(n, t): the hidden fragment of tile n and step t
    auto chunk_bf16 = [&](uint32_t c, auto x) {
        float f[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = __uint_as_float(((ws[j] >> (8 * (c % 4))) & 255u) << 23);
        // Two fragments are read from LDS while the two before them are multiplied, and tiles of 128 rows widen a part
        // of the next step's codes beside them (1,023 rows: 326 to 313 us). Smaller tiles have no registers for it:
        // 64 rows would leave two waves to a SIMD instead of three (of 196,608 x 5,376: 161 instead of 145 us).
        constexpr bool kWidenAhead = NT == 8;
        constexpr int kPairs = NT / 2, kWiden = 4 / kPairs;
        bf16x8_t e[kWidenAhead ? 2 : 1][4], y[2][2];
        auto read = [&](int i) {
#pragma unroll
            for (int k = 0; k < 2; ++k) y[i % 2][k] = __builtin_bit_cast(bf16x8_t, x(2 * (i % kPairs) + k, i / kPairs));
        };
        __builtin_amdgcn_sched_barrier(0);
        read(0);
#pragma unroll
        for (int i = 0; i < 4 * kPairs; ++i) {
            if (i + 1 < 4 * kPairs) read(i + 1);
            __builtin_amdgcn_sched_barrier(0);
            const int t = i / kPairs;
            if (kWidenAhead ? i == 0 : i % kPairs == 0) {
#pragma unroll
                for (int j = 0; j < 4; ++j) e[0][j] = widen(w[j][t], f[j]);
            }
            if (kWidenAhead && t < 3) {
#pragma unroll
                for (int j = i % kPairs * kWiden; j < (i % kPairs + 1) * kWiden; ++j) e[kWidenAhead ? (t + 1) % 2 : 0][j] = widen(w[j][t + 1], f[j]);
            }
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    f32x4_t& sum = acc[j][2 * (i % kPairs) + k];
                    sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(e[kWidenAhead ? t % 2 : 0][j], y[i % 2][k], sum, 0, 0, 0);
                }
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = wn[j], ws[j] = c % 4 == 3 ? wsn[j] : ws[j];
    };
    // x(n, c), xs(n, c): the hidden fragment of tile n and chunk c of the quad, and its scale in the low byte
    auto quad_mx = [&](uint32_t q, uint32_t chunks, auto x, auto xs) {
#pragma unroll
        for (uint32_t c = 0; c < 4; ++c) {
            if (c < chunks) {
                if (c > 0) load_codes(4 * q + c + 1);
                __builtin_amdgcn_sched_barrier(0);  // the loads first, then their chunk of arithmetic
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const u32x4_t y = x(n, c);
                    const uint32_t ys = xs(n, c);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (c == 0) acc[j][n] = mfma_mx<0>(w[j], ws[j], y, ys, acc[j][n]);
                        if (c == 1) acc[j][n] = mfma_mx<1>(w[j], ws[j], y, ys, acc[j][n]);
                        if (c == 2) acc[j][n] = mfma_mx<2>(w[j], ws[j], y, ys, acc[j][n]);
                        if (c == 3) acc[j][n] = mfma_mx<3>(w[j], ws[j], y, ys, acc[j][n]);
                    }
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = wn[j];
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) ws[j] = wsn[j];
    };
    // Loads are waited for in the order of their issue, so the weights' come before the hidden rows'.
    auto ahead = [&](uint32_t s) {
        load_codes(MX ? 4 * s + 1 : s + 1);
        if (MX || s % 4 == 0) load_scales(MX ? s + 1 : s / 4 + 1);
    };
    auto stage = [&](uint32_t s, const u32x4_t* x, const uint32_t* xs, u32x4_t* to, uint32_t* to_xs) {
        __syncthreads();  // stage s has arrived, and nobody reads the other buffer
        ahead(s);
        if (s + 1 < stages) {
            if constexpr (MX) fetch_scales(s + 1);
            fetch(s + 1, to);
        }
        if (have_group) {  // a wave past the vocabulary only helps with the hidden rows
            if constexpr (MX)
                quad_mx(s, 4, [&](int n, uint32_t c) { return x[(c * NT + n) * 64 + lane]; },
                        [&](int n, uint32_t c) { return xs[(16 * n + r) * 4 + c] >> (8 * kg); });
            else
                chunk_bf16(s, [&](int n, int t) { return x[(16 * n + r) * 16 + ((4 * (0x9cu >> (2 * kg) & 3) + t) ^ r)]; });
        }
        if constexpr (MX) {
            if (s + 1 < stages) write_scales(to_xs);
        }
        // the next stage's loads into LDS are done before the barrier that hands it over; where quantised
        // products were made, the next chunk's codes, the last four loads issued, may still be on their way
        __builtin_amdgcn_sched_barrier(0);
        if (MX && have_group) __builtin_amdgcn_s_waitcnt(kVmcnt0 + 4);
        else __builtin_amdgcn_s_waitcnt(kVmcnt0);
        __builtin_amdgcn_sched_barrier(0);
    };
    load_codes(0);
    load_scales(0);
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = wn[j], ws[j] = wsn[j];
    if (stages > 0) {
        fetch(0, buf0);
        if constexpr (MX) fetch_scales(0), write_scales(sc0);
        __builtin_amdgcn_s_waitcnt(kVmcnt0);
    }
    for (uint32_t s = 0; s < stages; s += 2) {
        stage(s, buf0, sc0, buf1, sc1);
        if (s + 1 >= stages) break;
        stage(s + 1, buf1, sc1, buf0, sc0);
    }
    if (have_group && stages * 256 < width) {  // the columns past the last whole stage, straight from memory
        ahead(stages);
        if constexpr (MX) {
            quad_mx(stages, a.chunks - 4 * stages,
                    [&](int n, uint32_t c) {
                        const uint32_t m = min(m0 + 16 * n + r, a.rows - 1), b = 16 * stages + 4 * c + kg;
                        u32x4_t y = {0, 0, 0, 0};
                        if (b < blocks)
                            y = *reinterpret_cast<const u32x4_t*>(static_cast<const uint8_t*>(a.x) + m * (a.d / 2ull) + 16ull * b);
                        return y;
                    },
                    [&](int n, uint32_t c) {
                        const uint32_t m = min(m0 + 16 * n + r, a.rows - 1), b = 16 * stages + 4 * c + kg;
                        return b < blocks ? static_cast<uint32_t>(a.xs[static_cast<uint64_t>(m) * blocks + b]) : 0u;
                    });
        } else {
            chunk_bf16(stages, [&](int n, int t) {
                const uint32_t m = min(m0 + 16 * n + r, a.rows - 1), b = 4 * stages + kg;
                u32x4_t y = {0, 0, 0, 0};
                if (b < blocks)
                    y = *reinterpret_cast<const u32x4_t*>(static_cast<const uint16_t*>(a.x) + m * a.x_stride + 32ull * b + 8 * t);
                return y;
            });
        }
    }
    // A lane's 16 logits of a row are a quarter of the wave's 64: they change places in LDS, so that a store fills
    // whole lines (64 rows of 262,144 x 5,376: 192 us with stores of a lane's own 16, 184 with whole lines, 176 with
    // whole lines past the caches).
    __syncthreads();  // nobody reads the hidden rows any more
    if (!have_group) return;
    constexpr uint32_t kPieces = 4 * sizeof(Out), kOwn = kPieces / 4, kEach = 16 / sizeof(Out);  // of 16 bytes: of a row, of a lane
    u32x4_t* const mine = (wave < 2 ? buf0 : buf1) + wave % 2 * (kStage / 2);
    auto place = [&](uint32_t row, uint32_t piece) {
        const uint32_t p = kPieces == 16 ? 4 * (0x9cu >> (2 * (piece / 4)) & 3) + piece % 4 : piece;
        return row * kPieces + (p ^ row % kPieces);
    };
    const uint64_t v = g * kMxGroupRows + kEach * (lane % kPieces);
    const uint32_t n_v = v < a.vocab ? static_cast<uint32_t>(min<uint64_t>(a.vocab - v, kEach)) : 0u;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        float y[16];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) y[4 * j + i] = acc[j][n][i];
        cap_logits(y, a.softcap);
#pragma unroll
        for (uint32_t k = 0; k < kOwn; ++k) {
            u32x4_t w;
            if constexpr (sizeof(Out) == 4) {
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) w[i] = __float_as_uint(y[4 * k + i]);
            } else {
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) w[i] = bf16_bits(y[8 * k + 2 * i]) | (bf16_bits(y[8 * k + 2 * i + 1]) << 16);
            }
            mine[place(r, kOwn * kg + k)] = w;
        }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (uint32_t k = 0; k < kOwn; ++k) {
            const uint32_t row = k * (64 / kPieces) + lane / kPieces, m = m0 + 16 * n + row;
            const u32x4_t w = mine[place(row, lane % kPieces)];
            if (m < a.rows) store_logits(static_cast<Out*>(a.out) + m * a.out_stride + v, w, n_v);
        }
        __builtin_amdgcn_wave_barrier();
    }
}

bool type_ok(int type) { return type == TWD_F32 || type == TWD_BF16 || type == TWD_F16; }
uint64_t type_size(int type) { return type == TWD_F32 ? 4 : 2; }

bool aligned(const void* p, uint64_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Rows and columns of a matrix in the format; stride 0 stands for no second dimension to check.
int check_matrix(const char* what, uint64_t rows, uint32_t cols) {
    if (rows == 0) return fail(TWD_E_INVALID, std::string(what) + ": no rows");
    if (cols == 0 || cols % kMxBlock != 0)
        return fail(TWD_E_INVALID, std::string(what) + ": columns must be a positive multiple of 32");
    return TWD_OK;
}

template <typename F>
int by_type(int type, F&& f) {
    if (type == TWD_F32) return f(float{});
    if (type == TWD_BF16) return f(Bf16{});
    return f(Fp16{});
}

dim3 matrix_grid(uint32_t groups, uint64_t rows) {
    return dim3((groups + kQuantThreads - 1) / kQuantThreads, static_cast<uint32_t>(rows < 65535 ? rows : 65535));
}

int check_device(const twd_mxhead* h) {
    int dev = 0;
    TWD_HIP(hipGetDevice(&dev));
    if (dev != h->device) return fail(TWD_E_INVALID, "the head lives on another device than the current one");
    return TWD_OK;
}

// The small kernels' sums take more LDS than a launch may ask for by default.
int enable_small() {
    constexpr int kMost = 2 * kSmallWaves * kSmallRows * 64 * sizeof(float);
    for (const void* k : {reinterpret_cast<const void*>(mx_small_kernel<false, float>),
                          reinterpret_cast<const void*>(mx_small_kernel<false, uint16_t>),
                          reinterpret_cast<const void*>(mx_small_kernel<true, float>),
                          reinterpret_cast<const void*>(mx_small_kernel<true, uint16_t>)})
        TWD_HIP(hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, kMost));
    return TWD_OK;
}

template <bool MX, int NT, typename Out>
int launch_tile(const MxArgs& a, hipStream_t s) {
    const uint32_t row_tiles = (a.rows + 16 * NT - 1) / (16 * NT), stretches = (a.groups + kTileWaves - 1) / kTileWaves;
    const uint64_t blocks = static_cast<uint64_t>((stretches + 7) / 8) * 8 * row_tiles;
    if (blocks > 0x7FFFFFFFull) return fail(TWD_E_INVALID, "rows x vocab is too large for one call");
    mx_tile_kernel<MX, NT, Out><<<static_cast<uint32_t>(blocks), kTileWaves * 64, 0, s>>>(a);
    TWD_HIP(hipGetLastError());
    return TWD_OK;
}

template <bool MX, typename Out>
int launch_typed(const twd_mxhead* h, const MxArgs& a, hipStream_t s) {
    // Few rows stream (262,144 x 5,376, 1 row: 116 us; as a tile 134). The more rows there are to the quads whose sums
    // are joined, the more the joining costs, which a tile does not have: 8 bf16 rows of 131,072 x 2,880 take 42 us
    // streamed and 34 as a tile, of 98,304 x 3,584 35 and 32, 16 of 262,144 x 1,024 33 and 29; but 12 of 262,144 x
    // 5,376, whose quads fill a compute unit, 132 and 136, and 8 of 65,536 x 2,048, one tile's block to a unit, 16 and
    // 21. Quantised rows, fewer bytes each, stream as fast or faster (16 of 131,072 x 2,880: 37 and 34). The rule
    // misses the better side where they lie close (8 rows of 131,072 x 2,048: 28 and 30, taken as a tile) and past 8 quads (16
    // rows of 131,072 x 4,608: 64 and 57, of 65,536 x 5,376: 39 and 33, both streamed).
    const bool tiles = !MX && a.rows > a.quads && a.quads <= 8 && a.groups >= 6 * static_cast<uint32_t>(h->cus);
    if (a.rows <= kSmallRows && a.quads <= kSmallWaves && !tiles) {
        const uint32_t blocks = min(a.groups, kSmallWaves / a.quads * static_cast<uint32_t>(h->cus));
        const uint32_t lds = 2 * a.quads * a.rows * 64 * sizeof(float);
        mx_small_kernel<MX, Out><<<blocks, a.quads * 64, lds, s>>>(a);
        TWD_HIP(hipGetLastError());
        return TWD_OK;
    }
    // Rows that a tile lacks are multiplied all the same, and every tile widens the weights anew (64 rows of 262,144 x
    // 5,376: 180 us in one tile of 64, 195 in two of 32; 32 rows: 139 in a tile of 32, 170 in one of 64; 128 rows: 304 in
    // one tile, 303 in two, quantised 179 and 202).
    // A tile's hidden rows are read at 32-bit offsets from its first.
    const uint64_t apart = MX ? a.d / 2 : 2 * a.x_stride;
    if (a.rows <= 32 || apart > 1u << 26) return launch_tile<MX, 2, Out>(a, s);
    if (a.rows <= 64 || apart > 1u << 25) return launch_tile<MX, 4, Out>(a, s);
    return launch_tile<MX, 8, Out>(a, s);
}

template <bool MX>
int launch_logits(const twd_mxhead* h, const MxArgs& a, int out_type, hipStream_t s) {
    return out_type == TWD_F32 ? launch_typed<MX, float>(h, a, s) : launch_typed<MX, uint16_t>(h, a, s);
}

constexpr uint32_t kMxMaxRows = 65536;
constexpr uint64_t kMxMaxStride = 1ull << 26;  // 32 rows within 4 GiB

int check_logits(const twd_mxhead* h, const void* x, uint32_t rows, const void* logits, int out_type,
                 uint64_t out_stride) {
    if (!h) return fail(TWD_E_INVALID, "null head");
    if (!x || !logits) return fail(TWD_E_INVALID, "null argument");
    if (rows == 0 || rows > kMxMaxRows) return fail(TWD_E_INVALID, "rows must be in 1..65536");
    if (out_type != TWD_F32 && out_type != TWD_BF16) return fail(TWD_E_INVALID, "logits must be fp32 or bf16");
    if (out_stride < h->vocab) return fail(TWD_E_INVALID, "the logits' row stride is below vocab");
    if (!aligned(x, 16)) return fail(TWD_E_INVALID, "hidden rows must start at a multiple of 16 bytes");
    if (!aligned(logits, type_size(out_type))) return fail(TWD_E_INVALID, "logits are not aligned to their type");
    return TWD_OK;
}

}  // namespace

}  // namespace twd

using namespace twd;

extern "C" {

TWD_API int twd_mx_quantize(const void* x, int type, uint64_t rows, uint32_t cols, uint64_t row_stride,
                            uint8_t* codes, uint8_t* scales, void* stream) {
    clear_error();
    if (!x || !codes || !scales) return fail(TWD_E_INVALID, "null argument");
    if (!type_ok(type)) return fail(TWD_E_INVALID, "type must be TWD_F32, TWD_BF16 or TWD_F16");
    int rc = check_matrix("twd_mx_quantize", rows, cols);
    if (rc) return rc;
    if (rows > 1 && row_stride < cols) return fail(TWD_E_INVALID, "twd_mx_quantize: the row stride is below cols");
    const uint64_t size = type_size(type);
    if (!aligned(x, size)) return fail(TWD_E_INVALID, "twd_mx_quantize: x is not aligned to its type");
    if (!aligned(codes, 16)) return fail(TWD_E_INVALID, "twd_mx_quantize: codes must start at a multiple of 16 bytes");
    QuantArgs a{x, row_stride, rows, cols / 8, codes, scales,
                aligned(x, 16) && (rows == 1 || row_stride * size % 16 == 0)};
    return by_type(type, [&](auto t) -> int {
        mx_quantize_kernel<decltype(t)>
            <<<matrix_grid(a.groups, rows), kQuantThreads, 0, static_cast<hipStream_t>(stream)>>>(a);
        TWD_HIP(hipGetLastError());
        return TWD_OK;
    });
}

TWD_API int twd_mx_dequantize(const uint8_t* codes, const uint8_t* scales, uint64_t rows, uint32_t cols, void* out,
                              int type, uint64_t row_stride, void* stream) {
    clear_error();
    if (!out || !codes || !scales) return fail(TWD_E_INVALID, "null argument");
    if (!type_ok(type)) return fail(TWD_E_INVALID, "type must be TWD_F32, TWD_BF16 or TWD_F16");
    int rc = check_matrix("twd_mx_dequantize", rows, cols);
    if (rc) return rc;
    if (rows > 1 && row_stride < cols) return fail(TWD_E_INVALID, "twd_mx_dequantize: the row stride is below cols");
    const uint64_t size = type_size(type);
    if (!aligned(out, size)) return fail(TWD_E_INVALID, "twd_mx_dequantize: out is not aligned to its type");
    if (!aligned(codes, 16)) return fail(TWD_E_INVALID, "twd_mx_dequantize: codes must start at a multiple of 16 bytes");
    DequantArgs a{codes, scales, rows, static_cast<uint32_t>(cols * size / 16), out, row_stride,
                  aligned(out, 16) && (rows == 1 || row_stride * size % 16 == 0)};
    return by_type(type, [&](auto t) -> int {
        mx_dequantize_kernel<decltype(t)>
            <<<matrix_grid(a.pieces, rows), kQuantThreads, 0, static_cast<hipStream_t>(stream)>>>(a);
        TWD_HIP(hipGetLastError());
        return TWD_OK;
    });
}

TWD_API int twd_mxhead_create(const uint8_t* codes, const uint8_t* scales, uint32_t vocab, uint32_t d_model,
                              float softcap, void* stream, twd_mxhead** out) {
    clear_error();
    if (!out) return fail(TWD_E_INVALID, "null argument");
    *out = nullptr;
    if (!codes || !scales) return fail(TWD_E_INVALID, "null argument");
    if (vocab == 0 || vocab > (1u << 30)) return fail(TWD_E_INVALID, "vocab must be in 1..2^30");
    if (d_model == 0 || d_model % kMxBlock != 0 || d_model > (1u << 20))
        return fail(TWD_E_INVALID, "d_model must be a positive multiple of 32, at most 2^20");
    if (softcap != 0.0f && !(softcap >= kMinSoftCap && softcap <= kMaxSoftCap))
        return fail(TWD_E_INVALID, "softcap must be 0 (none) or in 1e-30..1e30");
    if (!aligned(codes, 16)) return fail(TWD_E_INVALID, "codes must start at a multiple of 16 bytes");
    const uint32_t chunks = (d_model + kMxChunkK - 1) / kMxChunkK, quads = (chunks + 3) / 4;
    const uint32_t groups = (vocab + kMxGroupRows - 1) / kMxGroupRows;
    const uint64_t code_bytes = static_cast<uint64_t>(groups) * chunks * 4096, scale_bytes = static_cast<uint64_t>(groups) * quads * 1024;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    int dev = 0, cus = 0;
    TWD_HIP(hipGetDevice(&dev));
    if (const int rc = enable_small()) return rc;
    TWD_HIP(hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev));
    void* mem = nullptr;
    TWD_HIP(hipMalloc(&mem, code_bytes + scale_bytes + 16));
    uint8_t* base = static_cast<uint8_t*>(mem);
    uint32_t* bad_dev = reinterpret_cast<uint32_t*>(base + code_bytes + scale_bytes);
    u32x4_t* oc = static_cast<u32x4_t*>(mem);
    uint32_t* os = reinterpret_cast<uint32_t*>(base + code_bytes);
    uint32_t bad = 0;
    hipError_t e = hipMemsetAsync(bad_dev, 0, sizeof(bad), s);
    if (e == hipSuccess) {
        mx_repack_kernel<<<groups, 256, 0, s>>>(codes, scales, vocab, d_model, chunks, oc, os, bad_dev);
        e = hipGetLastError();
    }
    if (e == hipSuccess) e = hipMemcpyAsync(&bad, bad_dev, sizeof(bad), hipMemcpyDeviceToHost, s);
    if (e == hipSuccess) e = hipStreamSynchronize(s);
    if (e != hipSuccess || bad) {
        (void)hipFree(mem);
        if (e != hipSuccess) return hip_fail(e, "repacking the head");
        return fail(TWD_E_UNSUPPORTED, "a block scale exceeds 2^100 or is NaN");
    }
    twd_mxhead* h = new (std::nothrow) twd_mxhead{vocab, d_model, chunks, quads, groups, softcap, dev, cus, oc,
                                                  os, code_bytes + scale_bytes};
    if (!h) {
        (void)hipFree(mem);
        return fail(TWD_E_INVALID, "out of host memory");
    }
    *out = h;
    return TWD_OK;
}

TWD_API void twd_mxhead_destroy(twd_mxhead* head) {
    if (!head) return;
    (void)hipFree(head->codes);
    delete head;
}

TWD_API int twd_mxhead_info(const twd_mxhead* head, uint32_t* vocab, uint32_t* d_model, float* softcap,
                            uint64_t* device_bytes) {
    clear_error();
    if (!head) return fail(TWD_E_INVALID, "null head");
    if (vocab) *vocab = head->vocab;
    if (d_model) *d_model = head->d;
    if (softcap) *softcap = head->softcap;
    if (device_bytes) *device_bytes = head->bytes;
    return TWD_OK;
}

TWD_API int twd_mxhead_logits(const twd_mxhead* head, const uint16_t* hidden_bf16, uint32_t rows,
                              uint64_t hidden_stride, void* logits, int logits_type, uint64_t logits_stride,
                              void* stream) {
    clear_error();
    int rc = check_logits(head, hidden_bf16, rows, logits, logits_type, logits_stride);
    if (rc) return rc;
    if (rows > 1 && (hidden_stride < head->d || hidden_stride % 8 != 0))
        return fail(TWD_E_INVALID, "the hidden rows' stride must be a multiple of 8 and at least d_model");
    if (rows > 1 && hidden_stride > kMxMaxStride)
        return fail(TWD_E_INVALID, "the hidden rows' stride must be at most 2^26 elements");
    if ((rc = check_device(head))) return rc;
    const MxArgs a{head->codes, head->scales, hidden_bf16, nullptr, hidden_stride, logits, logits_stride,
                   head->vocab, head->d, head->chunks, head->quads, head->groups, rows, soft_cap(head->softcap)};
    return launch_logits<false>(head, a, logits_type, static_cast<hipStream_t>(stream));
}

TWD_API int twd_mxhead_logits_mx(const twd_mxhead* head, const uint8_t* codes, const uint8_t* scales, uint32_t rows,
                                 void* logits, int logits_type, uint64_t logits_stride, void* stream) {
    clear_error();
    int rc = check_logits(head, codes, rows, logits, logits_type, logits_stride);
    if (rc) return rc;
    if (!scales) return fail(TWD_E_INVALID, "null argument");
    if ((rc = check_device(head))) return rc;
    const MxArgs a{head->codes, head->scales, codes, scales, head->d, logits, logits_stride,
                   head->vocab, head->d, head->chunks, head->quads, head->groups, rows, soft_cap(head->softcap)};
    return launch_logits<true>(head, a, logits_type, static_cast<hipStream_t>(stream));
}

}  // extern "C"
