// 8-bit floating point with a scale for each block of 128: rows and weights to the format, and the LM head's product with
// weights held in it.
//
//   code(x) = e4m3(x / s), s = max |x| / 448 of the block    y_mv = softcap(sum_b s_mb s_vb sum_{c in b} w_vc h_mc)
//
// An element is an e4m3 code; hidden rows have an fp32 scale for each 128 columns, weights one for each 128 x 128. The product
// of 128 columns runs on matrix instructions, whose sums are then multiplied by the two scales and added up in fp32.
#include <hip/hip_runtime.h>

#include <new>
#include <string>

#include "product.h"
#include "twd_fp8.h"
#include "twd_internal.h"
#include "vocab_core.h"

namespace twd {

namespace {

constexpr uint32_t kBlock = 128;
constexpr float kTop = 448.0f, kLeastScale = 0x1p-126f;
// A weight scale times the largest that hidden rows get, FLT_MAX / 448, is finite: a sum of zero stays zero, and only logits
// past fp32 are infinite. Products of scales below 2^-126 are multiples of 2^-149; a sum of 128 products is below 2^24.7, so
// that takes less than 2^-125 from it.
constexpr float kMostWeightScale = 0x1p8f;

// ---- to the format --------------------------------------------------------------------------------------

// x / s to the nearest float, but where the quotient lies between two floats, to the one with an odd mantissa: rounding
// that to fewer bits is rounding the quotient itself. The remainder's sign says on which side it lies; where it would be
// below the normal numbers, both are brought up first.
__device__ __forceinline__ float quotient(float x, float s) {
    const float up_by = s < 0x1p-64f ? 0x1p64f : 1.0f;
    x *= up_by, s *= up_by;
    const float q = x / s, left = fmaf(-q, s, x);
    const uint32_t u = __float_as_uint(q);
    const bool up = (left > 0.0f) != (x < 0.0f);  // the quotient is larger in magnitude
    const bool move = left != 0.0f && (u & 1u) == 0;
    return __uint_as_float(move ? (up ? u + 1 : u - 1) : u);
}

__device__ __forceinline__ float scale_of(uint32_t top) {  // of the largest magnitude's bits
    const float s = fmaxf(__uint_as_float(top) / kTop, kLeastScale);
    return top >= 0x7F800000u ? __builtin_nanf("") : s;
}

__device__ __forceinline__ u32x2_t codes_of(const float (&v)[8], float s) {
    float q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = quotient(v[i], s);
    u32x2_t w;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        int c = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * i], q[4 * i + 1], 0, false);
        c = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * i + 2], q[4 * i + 3], c, true);
        w[i] = s != s ? 0u : static_cast<uint32_t>(c);
    }
    return w;
}

__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint32_t largest(const float (&v)[8]) {  // magnitudes order as their bits do, NaN above all
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = larger(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    return top;
}
__device__ __forceinline__ uint32_t largest_of_sixteen(uint32_t top) {  // lanes
    top = larger(top, dpp_move<0xB1>(top, top));
    top = larger(top, dpp_move<0x4E>(top, top));
    top = larger(top, dpp_move<0x141>(top, top));
    return larger(top, dpp_move<0x140>(top, top));
}

struct QuantArgs {
    const void* x;
    uint64_t stride;
    uint64_t rows;
    uint32_t blocks;  // of 128 columns
    uint8_t* codes;
    float* scales;
    bool wide;  // rows start at multiples of 16 bytes
};

// Eight columns to a lane, sixteen lanes to a scale. 262,144 x 5,376 fp32 values take 1.39 ms (5.1 TB/s; a copy reaches 4.85),
// bf16 ones 1.10 ms (3.8 TB/s: the exact quotient's dozen instructions a value show); 2,047 rows 13 us, one 4.6, its launch and
// chain.
template <typename T>
__global__ __launch_bounds__(256) void fp8_rows_kernel(QuantArgs a) {
    const uint32_t g = blockIdx.x * 256 + threadIdx.x, b = g / 16;
    if (b >= a.blocks) return;
    for (uint64_t r = blockIdx.y; r < a.rows; r += gridDim.y) {
        float v[8];
        Eight<T>::load(static_cast<const T*>(a.x) + r * a.stride + 8ull * g, a.wide, v);
        const float s = scale_of(largest_of_sixteen(largest(v)));
        reinterpret_cast<u32x2_t*>(a.codes)[(r * a.blocks) * 16 + g] = codes_of(v, s);
        if (g % 16 == 0) a.scales[r * a.blocks + b] = s;
    }
}

// A block to 128 x 128, whose values stay in registers between the scale and the codes. fp32 1.40 ms, bf16 1.04 ms, as above.
template <typename T>
__global__ __launch_bounds__(256) void fp8_weights_kernel(QuantArgs a) {
    __shared__ uint32_t tops[4];
    const uint32_t t = threadIdx.x, b = blockIdx.y, in = t % 16;
    const uint64_t r0 = static_cast<uint64_t>(blockIdx.x) * kBlock;
    float v[8][8] = {};
    uint32_t top = 0;
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
        const uint64_t r = r0 + 16 * i + t / 16;
        if (r < a.rows) Eight<T>::load(static_cast<const T*>(a.x) + r * a.stride + kBlock * b + 8 * in, a.wide, v[i]);
        top = larger(top, largest(v[i]));
    }
    top = wave_reduce(top, 0u, [](uint32_t x, uint32_t y) { return larger(x, y); });
    if (t % 64 == 0) tops[t / 64] = top;
    __syncthreads();
    const float s = scale_of(larger(larger(tops[0], tops[1]), larger(tops[2], tops[3])));
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
        const uint64_t r = r0 + 16 * i + t / 16;
        if (r < a.rows) reinterpret_cast<u32x2_t*>(a.codes)[(r * a.blocks + b) * 16 + in] = codes_of(v[i], s);
    }
    if (t == 0) a.scales[blockIdx.x * static_cast<uint64_t>(a.blocks) + b] = s;
}

// ---- the head's layout in HBM ---------------------------------------------------------------------
//
// A group is 64 vocabulary rows, four tiles of 16; a chunk is 128 columns. Codes are [group][chunk][tile][half][lane] 16 bytes:
// lane 16 kg + r's two halves are row r's columns 32 kg .. 32 kg + 31 of the chunk, as the 16 x 16 x 128 instruction takes
// them; two tiles' lanes of two kg's are an operand of a 32 x 32 x 64 one. A wave's load moves contiguous memory either
// way. Rows past the vocabulary are zero codes. Scales stay [group / 2][chunk]. Once a head: 542 us, 5.2 TB/s, for 262,144 x
// 5,376.
constexpr uint32_t kGroupRows = 64;
constexpr uint32_t kUnit = 512;  // 16-byte pieces of a group's chunk
constexpr uint32_t kRepackBlocks = 65536;  // 2^30 rows are 2^24 groups, a block to each 2^32 threads: more than a launch may have

__global__ __launch_bounds__(256) void fp8_repack_kernel(const uint8_t* __restrict__ codes, uint32_t vocab, uint32_t d,
                                                        u32x4_t* __restrict__ out) {
    const uint32_t lane = threadIdx.x % 64, tile = threadIdx.x / 64, kg = lane / 16, chunks = d / kBlock;
    const uint32_t groups = (vocab + kGroupRows - 1) / kGroupRows;
    for (uint64_t group = blockIdx.x; group < groups; group += gridDim.x) {
        const uint64_t row = group * kGroupRows + 16 * tile + lane % 16;
        for (uint32_t c = 0; c < chunks; ++c)
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h) {
                u32x4_t w = {0, 0, 0, 0};
                if (row < vocab) w = *reinterpret_cast<const u32x4_t*>(codes + row * d + kBlock * c + 32 * kg + 16 * h);
                out[(group * chunks + c) * kUnit + (2 * tile + h) * 64 + lane] = w;
            }
    }
}

__global__ __launch_bounds__(256) void fp8_check_kernel(const float* scales, float* kept, uint64_t n, uint32_t* bad) {
    for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < n; i += gridDim.x * 256ull) {
        const float s = scales[i];
        if (!(s >= 0.0f && s <= kMostWeightScale)) *bad = 1;
        kept[i] = s;
    }
}

struct Fp8Args {
    const u32x4_t* codes;
    const float* scales;
    const uint8_t* x;
    const float* xs;
    void* out;
    uint64_t out_stride;
    uint32_t vocab, d, chunks, groups, rows;
    SoftCap softcap;
};

__device__ __forceinline__ i32x8_t operand(u32x4_t lo, u32x4_t hi) {
    return __builtin_bit_cast(i32x8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// The 8-bit matrix instructions align the products of eight neighbouring columns to the largest of them and cut them at 2^-13
// of it (seen with one product of 2^16 beside others: those below 2^3 are lost in its eight, kept to 2^-10 elsewhere); for
// normal products that is 2e-5 of their magnitudes' sum. bf16 logits of many rows, whose own half step is 2^-8, are computed
// so, at twice the rate. All others widen both operands to bf16, which holds every e4m3 value: exact products, added in fp32.
// Up to 128 rows that costs little, as the read bounds them (64 rows of 262,144 x 5,376 to bf16: 246 us cut, 267 widened).
// Eight elements of two words:
__device__ __forceinline__ bf16x8_t widened(uint32_t lo, uint32_t hi) {
    u32x4_t e;
    e[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false));
    e[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true));
    e[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false));
    e[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true));
    return __builtin_bit_cast(bf16x8_t, e);
}
struct Wide32 {  // a lane's 32 elements
    bf16x8_t e[4];
};
__device__ __forceinline__ Wide32 widened(i32x8_t v) {
    Wide32 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w.e[i] = widened(static_cast<uint32_t>(v[2 * i]), static_cast<uint32_t>(v[2 * i + 1]));
    return w;
}

// ---- up to 16 hidden rows: the weights stream past rows held in registers ---------------------------
//
// Bound by the read of the head. The waves of a block split d_model by quads of chunks; a wave keeps its quad of the hidden
// rows in registers and streams its quad of one group after another, kAhead chunks (8 KB each) ahead of the arithmetic. The
// sums over the quads meet in LDS, two buffers in turn. One row of 262,144 x 5,376: 213 us, 6.6 TB/s, where a pure read reaches
// 6.7; 16 rows 237; seven of 151,669 x 3,584 88 us, 6.2 TB/s. A block has the waves for a d_model of up to 6,144; past it rows go to
// tiles of 32, which read such long rows as fast: of 131,072 rows by 6,144 one takes 120 us and 16 take 130 here, 32 take 129 in a
// tile; by 7,168 1 to 32 rows take 142 there (6.6 TB/s), by 12,288 246.
constexpr uint32_t kSmallRows = 16, kExactRows = 128;
constexpr uint32_t kSmallWaves = 12;
constexpr uint32_t kAhead = 2;

template <typename Out>
__global__ __launch_bounds__(kSmallWaves * 64) void fp8_small_kernel(Fp8Args a) {
    extern __shared__ float part[];  // [2][quad][row][64]
    const uint32_t lane = threadIdx.x % 64, kg = lane / 16, r = lane % 16, quads = (a.chunks + 3) / 4;
    const uint32_t quad = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t here = min(4u, a.chunks - 4 * quad);
    u32x4_t x[4][2];
    float xs[4];
#pragma unroll
    for (uint32_t c = 0; c < 4; ++c) {
        u32x4_t lo = {0, 0, 0, 0}, hi = lo;
        xs[c] = 0.0f;
        if (c < here && r < a.rows) {
            const u32x4_t* p = reinterpret_cast<const u32x4_t*>(a.x + static_cast<uint64_t>(r) * a.d + kBlock * (4 * quad + c) + 32 * kg);
            lo = p[0], hi = p[1];
            xs[c] = a.xs[static_cast<uint64_t>(r) * a.chunks + 4 * quad + c];
        }
        x[c][0] = lo, x[c][1] = hi;
    }
    // a group past the last has no bytes, so nothing is read of it; past the quad's end the last chunk comes again, whose
    // products count for nothing
    auto codes_of_group = [&](uint32_t g) {
        return make_rsrc(a.codes + (static_cast<uint64_t>(g) * a.chunks + 4 * quad) * kUnit, g < a.groups ? here * kUnit * 16 : 0);
    };
    auto scales_of_group = [&](uint32_t g) {
        return make_rsrc(a.scales + static_cast<uint64_t>(g / 2) * a.chunks + 4 * quad, g < a.groups ? here * 4 : 0);
    };
    u32x4_t w[kAhead][8];
    float ws[4];
    auto load_codes = [&](const __amdgpu_buffer_rsrc_t& at, uint32_t c, u32x4_t (&to)[8]) {
        const int chunk = static_cast<int>(min(c, here - 1) * (kUnit * 16));
#pragma unroll
        for (int j = 0; j < 8; ++j)
            to[j] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(at, lane * 16 + 1024 * j, chunk, kStreamed));
    };
    auto load_scales = [&](const __amdgpu_buffer_rsrc_t& at, float (&to)[4]) {
#pragma unroll
        for (int c = 0; c < 4; ++c) to[c] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(at, 0, 4 * c, 0));
    };
    auto codes = codes_of_group(blockIdx.x);
    load_scales(scales_of_group(blockIdx.x), ws);
#pragma unroll
    for (uint32_t c = 0; c < kAhead; ++c) {
        load_codes(codes, c, w[c]);
        __builtin_amdgcn_sched_barrier(0);
    }
    uint32_t buf = 0;
    for (uint32_t g = blockIdx.x; g < a.groups; g += gridDim.x) {
        const auto next = codes_of_group(g + gridDim.x);
        float f[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) f[c] = xs[c] * ws[c];
        f32x4_t acc[4] = {};
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (uint32_t c = 0; c < 4; ++c) {
            f32x4_t sum[4] = {};
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                u32x2_t in = {x[c][t / 2][t % 2 * 2], x[c][t / 2][t % 2 * 2 + 1]};
                asm volatile("; widened anew for every group: held widened, the rows would not fit" : "+v"(in));
                const bf16x8_t y = widened(in[0], in[1]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const u32x4_t& v = w[c % kAhead][2 * j + t / 2];
                    sum[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widened(v[t % 2 * 2], v[t % 2 * 2 + 1]), y, sum[j], 0, 0, 0);
                }
                __builtin_amdgcn_sched_barrier(0);  // a quarter's widened codes at a time
            }
            if (c == 0) load_scales(scales_of_group(g + gridDim.x), ws);
            if (c + kAhead < 4) load_codes(codes, c + kAhead, w[c % kAhead]);
            else load_codes(next, c + kAhead - 4, w[c % kAhead]);
            __builtin_amdgcn_sched_barrier(0);
            if (c < here) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[j][i] = fmaf(sum[j][i], f[c], acc[j][i]);
            }
        }
        codes = next;
        // a lane's sums are of hidden row r and the group's rows 16 j + 4 kg + i
        float* mine = part + (buf * quads + quad) * a.rows * 64;
        if (r < a.rows) {
#pragma unroll
            for (int j = 0; j < 4; ++j) *reinterpret_cast<f32x4_t*>(mine + r * 64 + 16 * j + 4 * kg) = acc[j];
        }
        lds_barrier();
        for (uint32_t e = quad * 64 + lane; e < a.rows * 64; e += quads * 64) {
            const float* p = part + buf * quads * a.rows * 64 + e;
            float y[1] = {p[0]};
            for (uint32_t q = 1; q < quads; ++q) y[0] += p[q * a.rows * 64];
            cap_logits(y, a.softcap);
            const uint64_t v = static_cast<uint64_t>(g) * kGroupRows + e % 64;
            if (v < a.vocab) store_logit(static_cast<Out*>(a.out) + (e / 64) * a.out_stride + v, y[0]);
        }
        buf ^= 1;
    }
}

// ---- more hidden rows: tiles of 256 vocabulary rows by 32 NS hidden rows -----------------------------
//
// Four waves, a group of weights each, read straight from memory a chunk ahead; the hidden rows' chunk goes through LDS,
// loaded there without registers one chunk ahead into the other of two buffers. 64 rows of 262,144 x 5,376 to fp32 take 255 to
// 273 us (5.2 to 5.5 TB/s of codes, and 67 MB stored): the read, with the widening's and the products' 140 us only partly under
// it. 128 rows are two tiles, 428 us; four squares of sums a wave leave the widened operands no registers. fp32 logits of more
// rows stay here, bound by the products: 2,047 rows 5.56 ms, 1,038 TFLOP/s.
constexpr uint32_t kTileWaves = 4;

template <int NS, typename Out, bool STREAMED>
__global__ __launch_bounds__(kTileWaves * 64) __attribute__((amdgpu_waves_per_eu(2))) void fp8_tile_kernel(Fp8Args a) {
    constexpr uint32_t kRows = 32 * NS;
    constexpr uint32_t kStage = kRows * 8;  // 16-byte pieces
    constexpr uint32_t kSpace = kStage > 1024 ? kStage : 1024;  // two waves' logits change places in a buffer
    __shared__ u32x4_t buf0[kSpace], buf1[kSpace];
    const uint32_t lane = threadIdx.x % 64, h = lane / 32, r = lane % 32;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t row_tiles = (a.rows + kRows - 1) / kRows, stretches = (a.groups + kTileWaves - 1) / kTileWaves;
    const uint32_t xcd = blockIdx.x % 8, turn = blockIdx.x / 8;
    const uint32_t stretch_up = turn / row_tiles * 8 + xcd;
    if (stretch_up >= stretches) return;
    const uint32_t stretch = stretches - 1 - stretch_up;
    const uint32_t m0 = turn % row_tiles * kRows;
    const uint32_t group = stretch * kTileWaves + wave;
    const bool have_group = group < a.groups;
    const uint64_t g = min(group, a.groups - 1);
    const uint32_t rows_here = min(a.rows - m0, kRows);

    // eight rows of 128 bytes to a load; a row's pieces change places with its number, so that sixteen rows' reads of one
    // piece meet different banks
    const auto rsrc = make_rsrc(a.x + static_cast<uint64_t>(m0) * a.d, rows_here * a.d);
    auto fetch = [&](uint32_t c, u32x4_t* to) {
        const uint32_t at = c * kBlock;
#pragma unroll
        for (uint32_t i = 0; i < NS; ++i) {
            const uint32_t p = i * kTileWaves + wave, row = 8 * p + lane / 8, piece = (lane % 8) ^ (row / 2 % 8);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void*)(to + p * 64), 16, static_cast<int>(row * a.d + 16 * piece + at), 0, 0, 0);
        }
    };
    const auto codes = make_rsrc(a.codes + g * a.chunks * kUnit, a.chunks * (kUnit * 16));
    const auto scales = make_rsrc(a.scales + g / 2 * a.chunks, a.chunks * 4);
    // square j, step s, half: rows 32 j + r, columns 32 (2 s + h) + 16 half of the chunk
    const uint32_t w_off = 16 * ((r / 16) * 128 + h * 16 + r % 16);
    u32x4_t w[8], wn[8];
    float ws, wsn, xs[NS], xsn[NS];
    auto load_codes = [&](uint32_t c) {
        const int at = __builtin_amdgcn_readfirstlane(static_cast<int>(min(c, a.chunks - 1) * (kUnit * 16)));
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int half = 0; half < 2; ++half)
                    wn[4 * j + 2 * s + half] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(codes, w_off + 4096 * j + 512 * s + 1024 * half, at, STREAMED ? kStreamed : 0));
    };
    const float* xs_at[NS];
#pragma unroll
    for (int n = 0; n < NS; ++n) xs_at[n] = a.xs + static_cast<uint64_t>(min(m0 + 32 * n + r, a.rows - 1)) * a.chunks;
    auto load_scales = [&](uint32_t c) {
        const uint32_t at = min(c, a.chunks - 1);
        wsn = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(scales, 0, static_cast<int>(4 * at), 0));
#pragma unroll
        for (int n = 0; n < NS; ++n) xsn[n] = xs_at[n][at];
    };
    f32x16_t acc[2][NS];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int n = 0; n < NS; ++n) acc[j][n] = f32x16_t{};
    auto turn_over = [&] {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = wn[i];
        ws = wsn;
#pragma unroll
        for (int n = 0; n < NS; ++n) xs[n] = xsn[n];
    };
    auto chunk = [&](uint32_t c, const u32x4_t* x, u32x4_t* to) {
        __syncthreads();  // chunk c has arrived, and nobody reads the other buffer
        load_codes(c + 1);
        load_scales(c + 1);
        if (c + 1 < a.chunks) fetch(c + 1, to);
        __builtin_amdgcn_sched_barrier(0);
        if (have_group) {
            Wide32 e[2][2];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int s = 0; s < 2; ++s) e[j][s] = widened(operand(w[4 * j + 2 * s], w[4 * j + 2 * s + 1]));
#pragma unroll
            for (int n = 0; n < NS; ++n) {
                f32x16_t sum[2] = {};
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const uint32_t row = 32 * n + r, p = 2 * (2 * s + h);
                    const Wide32 z = widened(operand(x[row * 8 + (p ^ (r / 2 % 8))], x[row * 8 + ((p + 1) ^ (r / 2 % 8))]));
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int t = 0; t < 4; ++t) sum[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(e[j][s].e[t], z.e[t], sum[j], 0, 0, 0);
                }
                const float f = xs[n] * ws;
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[j][n][i] = fmaf(sum[j][i], f, acc[j][n][i]);
            }
        }
        turn_over();
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(kVmcnt0);  // the next chunk's loads into LDS are done before the barrier that hands it over
        __builtin_amdgcn_sched_barrier(0);
    };
    load_codes(0);
    load_scales(0);
    fetch(0, buf0);
    turn_over();
    __builtin_amdgcn_s_waitcnt(kVmcnt0);
    for (uint32_t c = 0; c < a.chunks; c += 2) {
        chunk(c, buf0, buf1);
        if (c + 1 >= a.chunks) break;
        chunk(c + 1, buf1, buf0);
    }
    __syncthreads();  // nobody reads the hidden rows any more
    if (!have_group) return;
    constexpr uint32_t kOf = 16 / sizeof(Out);
    each<NS>([&](auto n) {
        store_rows<2, Out>((wave < 2 ? buf0 : buf1) + wave % 2 * 512,
            [&](auto j) {
                float y[16];
                f32x16_t z;
#pragma unroll
                for (int i = 0; i < 16; ++i) y[i] = acc[j][n][i];
                cap_logits(y, a.softcap);
#pragma unroll
                for (int i = 0; i < 16; ++i) z[i] = y[i];
                return z;
            },
            [&](uint32_t row, uint32_t col, u32x4_t v) {
                const uint32_t m = m0 + 32 * n + row;
                const uint64_t at = g * kGroupRows + col;
                if (m < a.rows && at < a.vocab)
                    store_logits(static_cast<Out*>(a.out) + m * a.out_stride + at, v, static_cast<uint32_t>(min<uint64_t>(a.vocab - at, kOf)));
            });
    });
}

// ---- many hidden rows: tiles of 256 x 256 -------------------------------------------------------------
//
// Eight waves, 64 vocabulary rows by 128 hidden rows each, two to a SIMD: one's scaling covers the other's matrix
// instructions. Weights and hidden rows both go through LDS, a chunk of each loaded there without registers one ahead into
// the other of two buffers; the weights' lines are brought to the L2 three chunks ahead. 2,047 rows of 262,144 x 5,376: 2.91 to
// 2.95 ms, 1.97 PFLOP/s. The matrix units are busy in 51% of the cycles, at 1.7 GHz: each square's 16 scalings for its two
// instructions, at one wave's pace, and the barrier of a chunk take the rest. From 129 rows on faster than the tiles above
// (129 rows 419 us, 256 rows 492).
constexpr uint32_t kWideThreads = 512;
constexpr uint32_t kWideStage = 4 * kUnit + 256 * 8;  // 16-byte pieces: four groups' chunk, 256 hidden rows'

template <typename Out>
__global__ __launch_bounds__(kWideThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void fp8_wide_kernel(Fp8Args a) {
    __shared__ u32x4_t buf0[kWideStage], buf1[kWideStage];
    __shared__ float sc0[512], sc1[512];  // hidden row m's scale at 64 (m / 32) + m % 32
    __shared__ uint32_t sink[kWideThreads];
    const TileGrid grid{(a.groups + 3) / 4, (a.rows + 255) / 256, 1};
    const uint32_t id = stretched(grid.tiles());
    if (id >= grid.tiles()) return;
    const TileAt at = tile_at(grid, id);
    const uint32_t lane = threadIdx.x % 64, h = lane / 32, r = lane % 32;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), va = wave % 4, mb = wave / 4;
    const uint32_t m0 = 256 * at.b, rows_here = min(a.rows - m0, 256u), g0 = 4 * at.a, groups_here = min(a.groups - g0, 4u);
    const uint32_t group_bytes = a.chunks * (kUnit * 16);
    // past the last group or row there is nothing: zeros
    const auto codes = make_rsrc(a.codes + static_cast<uint64_t>(g0) * a.chunks * kUnit, groups_here * group_bytes);
    const auto hidden = make_rsrc(a.x + static_cast<uint64_t>(m0) * a.d, rows_here * a.d);
    const auto scales = make_rsrc(a.xs + static_cast<uint64_t>(m0) * a.chunks, rows_here * a.chunks * 4);
    const auto weight_scales = make_rsrc(a.scales + static_cast<uint64_t>((g0 + va) / 2) * a.chunks, va < groups_here ? a.chunks * 4 : 0);
    constexpr uint32_t kLoads = 10;
    uint32_t w_off = 4 * wave / 8 * group_bytes + 4 * wave % 8 * 1024 + lane * 16, x_off[4];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        const uint32_t row = 8 * (4 * wave + i) + lane / 8;
        x_off[i] = row * a.d + 16 * ((lane % 8) ^ (row / 2 % 8));
    }
    const uint32_t s_off = lane < 32 ? (32 * wave + lane) * a.chunks * 4 : 0x80000000u;
    const uint32_t t_off = threadIdx.x < 256 && threadIdx.x % at.share == at.who ? threadIdx.x / 64 * group_bytes + threadIdx.x % 64 * 128 : 0x80000000u;
    // load i of a chunk; past the last chunk none
    auto fetch = [&](uint32_t i, uint32_t c, u32x4_t* to, float* sc) {
        if (i < 4) {
            const uint32_t o = c < a.chunks ? w_off + 1024 * i + c * (kUnit * 16) : 0x80000000u;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(codes, (lds_void*)(to + (4 * wave + i) * 64), 16, static_cast<int>(o), 0, 0, 0);
        } else if (i < 8) {
            const uint32_t o = c < a.chunks ? x_off[i - 4] + c * kBlock : 0x80000000u;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(hidden, (lds_void*)(to + 4 * kUnit + (4 * wave + i - 4) * 64), 16, static_cast<int>(o), 0, 0, 0);
        } else if (i == 8) {
            const uint32_t o = c < a.chunks ? s_off + 4 * c : 0x80000000u;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(scales, (lds_void*)(sc + 64 * wave), 4, static_cast<int>(o), 0, 0, 0);
        } else {
            const uint32_t o = c + 2 < a.chunks ? t_off + (c + 2) * (kUnit * 16) : 0x80000000u;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(codes, (lds_void*)(sink + 64 * wave), 4, static_cast<int>(o), 0, 0, 0);
        }
    };
    f32x16_t acc[2][4];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int n = 0; n < 4; ++n) acc[j][n] = f32x16_t{};
    const uint32_t w_at = va * kUnit + r / 16 * 128 + h * 16 + r % 16, x_at = 4 * kUnit + (128 * mb + r) * 8;
    auto weight_scale = [&](uint32_t c) {
        return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(weight_scales, c < a.chunks ? static_cast<int>(4 * c) : -4, 0, 0));
    };
    float ws_next = weight_scale(0);
    auto chunk = [&](uint32_t c, const u32x4_t* from, const float* sc, u32x4_t* to, float* to_sc) {
        const float ws = ws_next;
        ws_next = weight_scale(c + 1);
        float f[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) f[n] = sc[64 * (4 * mb + n) + r];
        i32x8_t w[2][2], y[2];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int s = 0; s < 2; ++s) w[j][s] = operand(from[w_at + 256 * j + 32 * s], from[w_at + 256 * j + 32 * s + 64]);
        auto read = [&](int n) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const uint32_t p = 2 * (2 * s + h);
                y[s] = operand(from[x_at + 256 * n + (p ^ (r / 2 % 8))], from[x_at + 256 * n + ((p + 1) ^ (r / 2 % 8))]);
            }
        };
        read(0);
        f32x16_t sum[2];
#pragma unroll
        for (int q = 0; q <= 8; ++q) {  // square q's products, and the scaling of the one before
            const int n = q / 2, j = q % 2;
            if (q < 8) {
#pragma unroll
                for (uint32_t i = kLoads * q / 8; i < kLoads * (q + 1) / 8; ++i) fetch(i, c + 1, to, to_sc);
                sum[j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w[j][0], y[0], f32x16_t{}, 0, 0, 0, 0, 0, 0);
                sum[j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w[j][1], y[1], sum[j], 0, 0, 0, 0, 0, 0);
                if (j == 1 && n < 3) read(n + 1);
            }
            __builtin_amdgcn_sched_barrier(0);
            if (q > 0) {
                const int m = (q - 1) / 2, k = (q - 1) % 2;
                if (k == 0) f[m] *= ws;
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[k][m][i] = fmaf(sum[k][i], f[m], acc[k][m][i]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_waitcnt(0x0070 | 1);  // all but the last load, of the lines ahead
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
    };
#pragma unroll
    for (uint32_t i = 0; i < kLoads; ++i) fetch(i, 0, buf0, sc0);
    __builtin_amdgcn_s_waitcnt(kVmcnt0);
    __syncthreads();
    for (uint32_t c = 0; c < a.chunks; c += 2) {
        chunk(c, buf0, sc0, buf1, sc1);
        chunk(c + 1, buf1, sc1, buf0, sc0);  // past the last chunk: zeros
    }
    __builtin_amdgcn_s_waitcnt(kVmcnt0);
    __syncthreads();
    if (va >= groups_here) return;
    constexpr uint32_t kOf = 16 / sizeof(Out);
    each<4>([&](auto n) {
        store_rows<2, Out>((wave < 4 ? buf0 : buf1) + wave % 4 * 512,
            [&](auto j) {
                float y[16];
                f32x16_t z;
#pragma unroll
                for (int i = 0; i < 16; ++i) y[i] = acc[j][n][i];
                cap_logits(y, a.softcap);
#pragma unroll
                for (int i = 0; i < 16; ++i) z[i] = y[i];
                return z;
            },
            [&](uint32_t row, uint32_t col, u32x4_t v) {
                const uint32_t m = m0 + 128 * mb + 32 * n + row;
                const uint64_t at_v = static_cast<uint64_t>(g0 + va) * kGroupRows + col;
                if (m < a.rows && at_v < a.vocab)
                    store_logits(static_cast<Out*>(a.out) + m * a.out_stride + at_v, v, static_cast<uint32_t>(min<uint64_t>(a.vocab - at_v, kOf)));
            });
    });
}

bool fp8_aligned(const void* p, uint64_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

}  // namespace

}  // namespace twd

struct twd_fp8head {
    uint32_t vocab, d, chunks, groups;
    float softcap;
    int device, cus;
    twd::u32x4_t* codes;
    float* scales;
    uint64_t bytes;
};

namespace twd {

namespace {

template <int NS, typename Out, bool STREAMED = false>
int launch_tile(const Fp8Args& a, hipStream_t s) {
    const uint32_t row_tiles = (a.rows + 32 * NS - 1) / (32 * NS), stretches = (a.groups + kTileWaves - 1) / kTileWaves;
    const uint64_t blocks = static_cast<uint64_t>((stretches + 7) / 8) * 8 * row_tiles;
    if (blocks > 0xFFFFFFull) return fail(TWD_E_INVALID, "rows x vocab is too large for one call");
    fp8_tile_kernel<NS, Out, STREAMED><<<static_cast<uint32_t>(blocks), kTileWaves * 64, 0, s>>>(a);
    TWD_HIP(hipGetLastError());
    return TWD_OK;
}

template <typename Out>
int launch_logits(const twd_fp8head* h, const Fp8Args& a, hipStream_t s) {
    const uint32_t quads = (a.chunks + 3) / 4;
    if (a.rows <= kSmallRows && quads <= kSmallWaves) {
        const uint32_t blocks = min(a.groups, kSmallWaves / quads * static_cast<uint32_t>(h->cus));
        fp8_small_kernel<Out><<<blocks, quads * 64, 2 * quads * a.rows * 64 * sizeof(float), s>>>(a);
        TWD_HIP(hipGetLastError());
        return TWD_OK;
    }
    // up to 32 rows the weights past the memory's cache are streamed (24 rows of 151,669 x 3,584: 107 us, otherwise 116; of
    // 32,003 x 2,048, which it holds: 24 and 20); tiles of 64 rows gain nothing (262,144 x 5,376: 290 and 285)
    const bool streamed = static_cast<uint64_t>(a.vocab) * a.d > kMemoryCache;
    if (a.rows <= 32) return streamed ? launch_tile<1, Out, true>(a, s) : launch_tile<1, Out>(a, s);
    if constexpr (sizeof(Out) == 4) {
        return launch_tile<2, Out>(a, s);
    } else {
        if (a.rows <= kExactRows) return launch_tile<2, Out>(a, s);
        const uint64_t tiles = static_cast<uint64_t>((a.groups + 3) / 4) * ((a.rows + 255) / 256);
        if (tiles > 0x7FFFF8ull) return fail(TWD_E_INVALID, "rows x vocab is too large for one call");
        fp8_wide_kernel<Out><<<blocks_for(static_cast<uint32_t>(tiles)), kWideThreads, 0, s>>>(a);
        TWD_HIP(hipGetLastError());
        return TWD_OK;
    }
}

}  // namespace

}  // namespace twd

using namespace twd;

extern "C" {

TWD_API int twd_fp8_quantize(const void* x, int type, uint64_t rows, uint32_t cols, uint64_t row_stride, uint32_t block_rows,
                             uint8_t* codes, float* scales, void* stream) {
    clear_error();
    if (!x || !codes || !scales) return fail(TWD_E_INVALID, "null argument");
    if (type != TWD_F32 && type != TWD_BF16 && type != TWD_F16) return fail(TWD_E_INVALID, "type must be TWD_F32, TWD_BF16 or TWD_F16");
    if (rows == 0) return fail(TWD_E_INVALID, "twd_fp8_quantize: no rows");
    if (cols == 0 || cols % kBlock != 0 || cols > (1u << 20))
        return fail(TWD_E_INVALID, "twd_fp8_quantize: columns must be a positive multiple of 128, at most 2^20");
    if (rows > 1 && row_stride < cols) return fail(TWD_E_INVALID, "twd_fp8_quantize: the row stride is below cols");
    if (block_rows != 1 && block_rows != kBlock) return fail(TWD_E_INVALID, "block_rows must be 1 or 128");
    if (block_rows == kBlock && rows > (1ull << 30)) return fail(TWD_E_INVALID, "twd_fp8_quantize: too many rows");
    const uint64_t size = type == TWD_F32 ? 4 : 2;
    if (!fp8_aligned(x, size) || !fp8_aligned(scales, 4)) return fail(TWD_E_INVALID, "twd_fp8_quantize: x or scales are not aligned to their type");
    if (!fp8_aligned(codes, 16)) return fail(TWD_E_INVALID, "twd_fp8_quantize: codes must start at a multiple of 16 bytes");
    const QuantArgs a{x, row_stride, rows, cols / kBlock, codes, scales, fp8_aligned(x, 16) && (rows == 1 || row_stride * size % 16 == 0)};
    const hipStream_t s = static_cast<hipStream_t>(stream);
    auto go = [&](auto t) {
        using T = decltype(t);
        if (block_rows == 1)
            fp8_rows_kernel<T><<<dim3((a.blocks * 16 + 255) / 256, static_cast<uint32_t>(rows < 65535 ? rows : 65535)), 256, 0, s>>>(a);
        else
            fp8_weights_kernel<T><<<dim3(static_cast<uint32_t>((rows + kBlock - 1) / kBlock), a.blocks), 256, 0, s>>>(a);
    };
    if (type == TWD_F32) go(float{});
    else if (type == TWD_BF16) go(Bf16{});
    else go(Fp16{});
    TWD_HIP(hipGetLastError());
    return TWD_OK;
}

TWD_API int twd_fp8head_create(const uint8_t* codes, const float* scales, uint32_t vocab, uint32_t d_model, float softcap,
                               void* stream, twd_fp8head** out) {
    clear_error();
    if (!out) return fail(TWD_E_INVALID, "null argument");
    *out = nullptr;
    if (!codes || !scales) return fail(TWD_E_INVALID, "null argument");
    if (vocab == 0 || vocab > (1u << 30)) return fail(TWD_E_INVALID, "vocab must be in 1..2^30");
    if (d_model == 0 || d_model % kBlock != 0 || d_model > (1u << 20))
        return fail(TWD_E_INVALID, "d_model must be a positive multiple of 128, at most 2^20");
    if (softcap != 0.0f && !(softcap >= kMinSoftCap && softcap <= kMaxSoftCap))
        return fail(TWD_E_INVALID, "softcap must be 0 (none) or in 1e-30..1e30");
    if (!fp8_aligned(codes, 16) || !fp8_aligned(scales, 4)) return fail(TWD_E_INVALID, "codes must start at a multiple of 16 bytes, scales of 4");
    const uint32_t chunks = d_model / kBlock, groups = (vocab + kGroupRows - 1) / kGroupRows;
    const uint64_t n_scales = static_cast<uint64_t>((vocab + kBlock - 1) / kBlock) * chunks;
    const uint64_t code_bytes = static_cast<uint64_t>(groups) * chunks * kUnit * 16, scale_bytes = (n_scales * 4 + 15) / 16 * 16;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    int dev = 0, cus = 0;
    TWD_HIP(hipGetDevice(&dev));
    TWD_HIP(hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev));
    constexpr int kMost = 2 * kSmallWaves * kSmallRows * 64 * sizeof(float);
    TWD_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(fp8_small_kernel<float>), hipFuncAttributeMaxDynamicSharedMemorySize, kMost));
    TWD_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(fp8_small_kernel<uint16_t>), hipFuncAttributeMaxDynamicSharedMemorySize, kMost));
    void* mem = nullptr;
    TWD_HIP(hipMalloc(&mem, code_bytes + scale_bytes + 16));
    u32x4_t* kept_codes = static_cast<u32x4_t*>(mem);
    float* kept_scales = reinterpret_cast<float*>(static_cast<uint8_t*>(mem) + code_bytes);
    uint32_t* bad_dev = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(mem) + code_bytes + scale_bytes);
    uint32_t bad = 0;
    hipError_t e = hipMemsetAsync(bad_dev, 0, sizeof(bad), s);
    if (e == hipSuccess) {
        fp8_check_kernel<<<256, 256, 0, s>>>(scales, kept_scales, n_scales, bad_dev);
        fp8_repack_kernel<<<min(groups, kRepackBlocks), 256, 0, s>>>(codes, vocab, d_model, kept_codes);
        e = hipGetLastError();
    }
    if (e == hipSuccess) e = hipMemcpyAsync(&bad, bad_dev, sizeof(bad), hipMemcpyDeviceToHost, s);
    if (e == hipSuccess) e = hipStreamSynchronize(s);
    twd_fp8head* h = nullptr;
    if (e == hipSuccess && !bad)
        h = new (std::nothrow) twd_fp8head{vocab, d_model, chunks, groups, softcap, dev, cus, kept_codes, kept_scales, code_bytes + scale_bytes};
    if (!h) {
        (void)hipFree(mem);
        if (e != hipSuccess) return hip_fail(e, "repacking the head");
        if (bad) return fail(TWD_E_UNSUPPORTED, "a block scale is negative, above 2^8 or NaN");
        return fail(TWD_E_INVALID, "out of host memory");
    }
    *out = h;
    return TWD_OK;
}

TWD_API void twd_fp8head_destroy(twd_fp8head* head) {
    if (!head) return;
    (void)hipFree(head->codes);
    delete head;
}

TWD_API int twd_fp8head_info(const twd_fp8head* head, uint32_t* vocab, uint32_t* d_model, float* softcap,
                             uint64_t* device_bytes) {
    clear_error();
    if (!head) return fail(TWD_E_INVALID, "null head");
    if (vocab) *vocab = head->vocab;
    if (d_model) *d_model = head->d;
    if (softcap) *softcap = head->softcap;
    if (device_bytes) *device_bytes = head->bytes;
    return TWD_OK;
}

TWD_API int twd_fp8head_logits(const twd_fp8head* head, const uint8_t* codes, const float* scales, uint32_t rows,
                               void* logits, int logits_type, uint64_t logits_stride, void* stream) {
    clear_error();
    if (!head) return fail(TWD_E_INVALID, "null head");
    if (!codes || !scales || !logits) return fail(TWD_E_INVALID, "null argument");
    if (rows == 0 || rows > 65536u) return fail(TWD_E_INVALID, "rows must be in 1..65536");
    if (logits_type != TWD_F32 && logits_type != TWD_BF16) return fail(TWD_E_INVALID, "logits must be fp32 or bf16");
    if (logits_stride < head->vocab) return fail(TWD_E_INVALID, "the logits' row stride is below vocab");
    if (!fp8_aligned(codes, 16)) return fail(TWD_E_INVALID, "hidden codes must start at a multiple of 16 bytes");
    if (!fp8_aligned(scales, 4) || !fp8_aligned(logits, logits_type == TWD_F32 ? 4 : 2))
        return fail(TWD_E_INVALID, "scales or logits are not aligned to their type");
    int dev = 0;
    TWD_HIP(hipGetDevice(&dev));
    if (dev != head->device) return fail(TWD_E_INVALID, "the head lives on another device than the current one");
    const Fp8Args a{head->codes, head->scales, codes, scales, logits, logits_stride, head->vocab, head->d, head->chunks,
                    head->groups, rows, soft_cap(head->softcap)};
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return logits_type == TWD_F32 ? launch_logits<float>(head, a, s) : launch_logits<uint16_t>(head, a, s);
}

}  // extern "C"
