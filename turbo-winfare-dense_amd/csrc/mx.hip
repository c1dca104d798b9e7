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
// exchanges inside a quad of lanes. The pass is bound by its reads.

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
    __device__ static void store(float* p, bool wide, const float* v) {
        if (wide) {
            reinterpret_cast<f32x4_t*>(p)[0] = f32x4_t{v[0], v[1], v[2], v[3]};
            reinterpret_cast<f32x4_t*>(p)[1] = f32x4_t{v[4], v[5], v[6], v[7]};
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = v[i];
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
    __device__ static void store(T* p, bool wide, const float* v) {
        if (wide) {
            u32x4_t a;
#pragma unroll
            for (int i = 0; i < 4; ++i) a[i] = f32_to_half<T>(v[2 * i]) | (f32_to_half<T>(v[2 * i + 1]) << 16);
            *reinterpret_cast<u32x4_t*>(p) = a;
        } else {
            uint16_t* q = reinterpret_cast<uint16_t*>(p);
#pragma unroll
            for (int i = 0; i < 8; ++i) q[i] = static_cast<uint16_t>(f32_to_half<T>(v[i]));
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
    uint32_t groups;
    void* out;
    uint64_t stride;
    bool wide;
};

// The magnitude bits c as a float's exponent and first mantissa bit are the element's value times
// 2^-126 (a subnormal float for 0.5), so one exact product by 2^126 decodes it.
template <typename T>
__global__ __launch_bounds__(kQuantThreads) void mx_dequantize_kernel(DequantArgs a) {
    const uint32_t g = blockIdx.x * kQuantThreads + threadIdx.x;
    if (g >= a.groups) return;
    for (uint64_t r = blockIdx.y; r < a.rows; r += gridDim.y) {
        const uint32_t w = reinterpret_cast<const uint32_t*>(a.codes)[r * a.groups + g];
        const float s = scale_value(a.scales[r * (a.groups / 4) + g / 4]);
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t c = w >> (4 * i);
            v[i] = __uint_as_float(((c & 7u) << 22) | ((c & 8u) << 28)) * 0x1p126f * s;
        }
        Eight<T>::store(static_cast<T*>(a.out) + r * a.stride + 8ull * g, a.wide, v);
    }
}

// ---- the head's layout in HBM ---------------------------------------------------------------------
//
// A tile is 16 vocabulary rows; a chunk is 128 columns, four blocks. Both matrix instructions used
// here (16x16x128 on 4-bit operands, and four 16x16x32 on bf16 ones, whose columns may be taken in
// any order as long as both operands agree) let lane l = 16 kg + r hold row r's block kg of a chunk:
//   codes  [tile][chunk][lane] 16 bytes, the block's 32 elements
//   scales [tile][quad of chunks][lane] 4 bytes, byte j the scale of that lane's block in chunk 4q + j
// so a load instruction of a wave moves 1 KB (codes) or 256 B (scales) of contiguous memory, and every
// lane's elements share the lane's own scale. Rows past the vocabulary and columns past d_model are
// zero codes; their scales are 0 (2^-127).
constexpr uint32_t kMxChunkK = 128;
constexpr uint32_t kMxTileRows = 16;

__global__ __launch_bounds__(256) void mx_repack_kernel(const uint8_t* __restrict__ codes,
                                                       const uint8_t* __restrict__ scales, uint32_t vocab,
                                                       uint32_t d, uint32_t chunks, u32x4_t* __restrict__ out_codes,
                                                       uint32_t* __restrict__ out_scales, uint32_t* bad) {
    const uint32_t lane = threadIdx.x % 64, kg = lane / 16, r = lane % 16;
    const uint32_t blocks = d / kMxBlock, quads = (chunks + 3) / 4;
    const uint64_t tile = blockIdx.x;
    const uint64_t row = tile * kMxTileRows + r;
    for (uint32_t q = threadIdx.x / 64; q < quads; q += 4) {
        uint32_t sc = 0;
        for (uint32_t j = 0; j < 4; ++j) {
            const uint32_t chunk = 4 * q + j, b = 4 * chunk + kg;
            if (chunk >= chunks) break;
            u32x4_t c = {0, 0, 0, 0};
            if (row < vocab && b < blocks) {
                c = *reinterpret_cast<const u32x4_t*>(codes + row * (d / 2) + 16ull * b);
                const uint32_t s = scales[row * blocks + b];
                if (s > 227u) *bad = 1;  // above 2^100, NaN among them
                sc |= s << (8 * j);
            }
            out_codes[(tile * chunks + chunk) * 64 + lane] = c;
        }
        out_scales[(tile * quads + q) * 64 + lane] = sc;
    }
}

}  // namespace

}  // namespace twd

struct twd_mxhead {
    uint32_t vocab, d, chunks, quads, tiles;
    float softcap;
    int device;
    twd::u32x4_t* codes;
    uint32_t* scales;
    uint64_t bytes;
};

namespace twd {

namespace {

struct MxArgs {
    const u32x4_t* codes;
    const uint32_t* scales;
    const void* x;  // bf16 rows, or codes [rows][d / 2]
    const uint8_t* xs;
    uint64_t x_stride;
    void* out;
    uint64_t out_stride;
    uint32_t vocab, d, chunks, quads, rows;
    float softcap;
};

__device__ __forceinline__ void store_logit(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_logit(uint16_t* p, float v) { *p = static_cast<uint16_t>(bf16_bits(v)); }

// One wave per tile of 16 vocabulary rows and 16 hidden rows.
template <bool MX, typename Out>
__global__ __launch_bounds__(256) void mx_logits_kernel(MxArgs a) {
    const uint32_t lane = threadIdx.x % 64, kg = lane / 16, r = lane % 16;
    const uint32_t tile = blockIdx.x * 4 + threadIdx.x / 64;
    if (tile * kMxTileRows >= a.vocab) return;
    const uint32_t m = blockIdx.y * 16 + r;
    const bool have = m < a.rows;
    const uint32_t blocks = a.d / kMxBlock;
    f32x4_t acc = {0, 0, 0, 0};
    uint32_t sc = 0;
    for (uint32_t c = 0; c < a.chunks; ++c) {
        const u32x4_t w = a.codes[(static_cast<uint64_t>(tile) * a.chunks + c) * 64 + lane];
        if (c % 4 == 0) sc = a.scales[(static_cast<uint64_t>(tile) * a.quads + c / 4) * 64 + lane];
        const uint32_t s = (sc >> (8 * (c % 4))) & 255u, b = 4 * c + kg;
        if constexpr (MX) {
            u32x4_t x = {0, 0, 0, 0};
            uint32_t xs = 0;
            if (have && b < blocks) {
                x = *reinterpret_cast<const u32x4_t*>(static_cast<const uint8_t*>(a.x) + m * (a.d / 2ull) + 16ull * b);
                xs = a.xs[static_cast<uint64_t>(m) * blocks + b];
            }
            const i32x8_t wa = {static_cast<int>(w[0]), static_cast<int>(w[1]), static_cast<int>(w[2]), static_cast<int>(w[3])};
            const i32x8_t xb = {static_cast<int>(x[0]), static_cast<int>(x[1]), static_cast<int>(x[2]), static_cast<int>(x[3])};
            acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wa, xb, acc, 4, 4, 0, static_cast<int>(s), 0,
                                                                   static_cast<int>(xs));
        } else {
            const float sv = __uint_as_float(s << 23);
            const uint16_t* row = static_cast<const uint16_t*>(a.x) + m * a.x_stride + 32ull * b;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                u32x4_t x = {0, 0, 0, 0};
                if (have && b < blocks) x = *reinterpret_cast<const u32x4_t*>(row + 8 * t);
                u32x4_t e;
                e[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[t], sv, 0));
                e[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[t], sv, 1));
                e[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[t], sv, 2));
                e[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[t], sv, 3));
                acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, e),
                                                              __builtin_bit_cast(bf16x8_t, x), acc, 0, 0, 0);
            }
        }
    }
    if (!have) return;
    Out* out = static_cast<Out*>(a.out) + m * a.out_stride;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t v = tile * kMxTileRows + 4 * kg + i;
        if (v < a.vocab) store_logit(out + v, a.softcap > 0.0f ? a.softcap * tanhf(acc[i] / a.softcap) : acc[i]);
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

template <bool MX>
int launch_logits(const MxArgs& a, int out_type, hipStream_t s) {
    const uint32_t tiles = (a.vocab + kMxTileRows - 1) / kMxTileRows;
    const dim3 grid((tiles + 3) / 4, (a.rows + 15) / 16);
    if (out_type == TWD_F32)
        mx_logits_kernel<MX, float><<<grid, 256, 0, s>>>(a);
    else
        mx_logits_kernel<MX, uint16_t><<<grid, 256, 0, s>>>(a);
    TWD_HIP(hipGetLastError());
    return TWD_OK;
}

constexpr uint32_t kMxMaxRows = 65536;

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
    DequantArgs a{codes, scales, rows, cols / 8, out, row_stride,
                  aligned(out, 16) && (rows == 1 || row_stride * size % 16 == 0)};
    return by_type(type, [&](auto t) -> int {
        mx_dequantize_kernel<decltype(t)>
            <<<matrix_grid(a.groups, rows), kQuantThreads, 0, static_cast<hipStream_t>(stream)>>>(a);
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
    if (!(softcap >= 0.0f) || softcap > 3.0e38f) return fail(TWD_E_INVALID, "softcap must be finite and >= 0 (0: none)");
    if (!aligned(codes, 16)) return fail(TWD_E_INVALID, "codes must start at a multiple of 16 bytes");
    const uint32_t chunks = (d_model + kMxChunkK - 1) / kMxChunkK, quads = (chunks + 3) / 4;
    const uint32_t tiles = (vocab + kMxTileRows - 1) / kMxTileRows;
    const uint64_t code_bytes = static_cast<uint64_t>(tiles) * chunks * 1024, scale_bytes = static_cast<uint64_t>(tiles) * quads * 256;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    int dev = 0;
    TWD_HIP(hipGetDevice(&dev));
    void* mem = nullptr;
    TWD_HIP(hipMalloc(&mem, code_bytes + scale_bytes + 16));
    uint8_t* base = static_cast<uint8_t*>(mem);
    uint32_t* bad_dev = reinterpret_cast<uint32_t*>(base + code_bytes + scale_bytes);
    u32x4_t* oc = static_cast<u32x4_t*>(mem);
    uint32_t* os = reinterpret_cast<uint32_t*>(base + code_bytes);
    uint32_t bad = 0;
    hipError_t e = hipMemcpyAsync(bad_dev, &bad, sizeof(bad), hipMemcpyHostToDevice, s);
    if (e == hipSuccess) {
        mx_repack_kernel<<<tiles, 256, 0, s>>>(codes, scales, vocab, d_model, chunks, oc, os, bad_dev);
        e = hipGetLastError();
    }
    if (e == hipSuccess) e = hipMemcpyAsync(&bad, bad_dev, sizeof(bad), hipMemcpyDeviceToHost, s);
    if (e == hipSuccess) e = hipStreamSynchronize(s);
    if (e != hipSuccess || bad) {
        (void)hipFree(mem);
        if (e != hipSuccess) return hip_fail(e, "repacking the head");
        return fail(TWD_E_UNSUPPORTED, "a block scale exceeds 2^100 or is NaN");
    }
    twd_mxhead* h = new (std::nothrow) twd_mxhead{vocab, d_model, chunks, quads, tiles, softcap, dev, oc, os,
                                                  code_bytes + scale_bytes};
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
    if ((rc = check_device(head))) return rc;
    const MxArgs a{head->codes, head->scales, hidden_bf16, nullptr, hidden_stride, logits, logits_stride,
                   head->vocab, head->d, head->chunks, head->quads, rows, head->softcap};
    return launch_logits<false>(a, logits_type, static_cast<hipStream_t>(stream));
}

TWD_API int twd_mxhead_logits_mx(const twd_mxhead* head, const uint8_t* codes, const uint8_t* scales, uint32_t rows,
                                 void* logits, int logits_type, uint64_t logits_stride, void* stream) {
    clear_error();
    int rc = check_logits(head, codes, rows, logits, logits_type, logits_stride);
    if (rc) return rc;
    if (!scales) return fail(TWD_E_INVALID, "null argument");
    if ((rc = check_device(head))) return rc;
    const MxArgs a{head->codes, head->scales, codes, scales, head->d, logits, logits_stride,
                   head->vocab, head->d, head->chunks, head->quads, rows, head->softcap};
    return launch_logits<true>(a, logits_type, static_cast<hipStream_t>(stream));
}

}  // extern "C"
