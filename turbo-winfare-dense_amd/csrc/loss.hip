// Softmax cross entropy of a bf16 head's logits, and its gradients, a piece of the vocabulary at a time.
//
//   z_mv = softcap(h_m . w_v)   lse_m = ln sum_v exp(z_mv)   loss_m = lse_m - z_m,t(m)
//   dz_mv = g_m (exp(z_mv - lse_m) - [v = t(m)]) (1 - (z_mv / cap)^2)   d_hidden = dz W   d_weight = dz^T H
//
// The rows that count are first gathered one behind another, so rows that are left out cost nothing and cannot spoil a
// sum. Forward, each tile of logits is reduced where it was summed to its rows' largest value and their sum of
// exponentials against it; a second kernel joins the tiles. Backward, a piece of the vocabulary after another: the
// logits again, dz of them in bf16 in both orders, then the two products.
#include <hip/hip_runtime.h>

#include <new>
#include <string>

#include "product.h"
#include "twd_internal.h"
#include "twd_loss.h"
#include "vocab_core.h"

namespace twd {

namespace {

constexpr float kLog2e = 1.4426950408889634f;

// The rows that count, one behind another: `count` of them, by rising row.
struct LossRows {
    uint32_t* count;
    uint32_t* at;   // [m] the caller's row
    int32_t* target;
    float* grad;
    float* lse;
    float* hit;     // the target's logit
    uint16_t* h;    // [m][d, zeros up to a multiple of 128]
};

struct GatherArgs {
    LossRows r;
    const uint16_t* hidden;
    uint64_t stride;
    const int32_t* targets;
    const float* grad;    // backward (may be null: all 1)
    const float* lse_in;  // backward
    float* losses;        // forward
    float* lse_out;       // forward
    uint32_t rows, vocab;
    uint32_t pieces, h_pieces;  // of 16 bytes in a row, and in a gathered one, which ends in zeros
};

constexpr uint32_t kGatherRows = 8;

// A block counts the rows before its own that count, then brings its own to their places.
__global__ __launch_bounds__(256) void loss_gather_kernel(GatherArgs a) {
    __shared__ uint32_t wave_sum[4];
    const uint32_t r0 = blockIdx.x * kGatherRows, t = threadIdx.x;
    auto counts = [&](uint32_t r) { return static_cast<uint32_t>(a.targets[r]) < a.vocab; };
    uint32_t before = 0;
    for (uint32_t r = t; r < r0; r += 256) before += counts(r) ? 1u : 0u;
    before = wave_reduce(before, 0u, [](uint32_t x, uint32_t y) { return x + y; });
    if (t % 64 == 0) wave_sum[t / 64] = before;
    __syncthreads();
    uint32_t m = wave_sum[0] + wave_sum[1] + wave_sum[2] + wave_sum[3];
    const uint32_t last = min(r0 + kGatherRows, a.rows);
    for (uint32_t r = r0; r < last; ++r) {
        if (!counts(r)) {
            if (t == 0 && a.losses) a.losses[r] = 0.0f, a.lse_out[r] = 0.0f;
            continue;
        }
        const u32x4_t* from = reinterpret_cast<const u32x4_t*>(a.hidden + r * a.stride);
        u32x4_t* to = reinterpret_cast<u32x4_t*>(a.r.h) + static_cast<uint64_t>(m) * a.h_pieces;
        for (uint32_t i = t; i < a.h_pieces; i += 256) to[i] = i < a.pieces ? from[i] : u32x4_t{0, 0, 0, 0};
        if (t == 0) {
            a.r.at[m] = r;
            a.r.target[m] = a.targets[r];
            if (a.lse_in) a.r.grad[m] = a.grad ? a.grad[r] : 1.0f, a.r.lse[m] = a.lse_in[r];
        }
        ++m;
    }
    if (last == a.rows && t == 0) *a.r.count = m;
}

struct LogitArgs {
    LossRows r;
    Operand weight, hidden;
    uint32_t d, vocab;
    uint32_t v0;          // the piece's first vocabulary row
    SoftCap softcap;
    TileGrid grid;
    float2* part;         // forward: [tile][stride] largest logit and sum of exponentials
    uint16_t* dz;         // backward: [m][dz_stride], from v0 on
    uint16_t* dzt;        // [v - v0][dzt_stride]
    uint32_t part_stride, dz_stride, dzt_stride;
};

template <typename Tile>
constexpr int kWavesPerEu = Tile::kStage * 16 * 4 > 81920 ? 1 : 2;

template <typename Tile, int TA, int TB, int GA, int GB, bool GRAD>
__global__ __launch_bounds__(kProductThreads) __attribute__((amdgpu_waves_per_eu(kWavesPerEu<Tile>, kWavesPerEu<Tile>))) void loss_logits_kernel(LogitArgs a) {
    __shared__ u32x4_t s0[Tile::kStage], s1[Tile::kStage], s2[Tile::kStage], s3[Tile::kStage];
    TileAt at;
    if (!tile_of_block(a.grid, &at)) return;
    const uint32_t count = *a.r.count, m0 = at.b * Tile::kB, v_tile = a.v0 + at.a * Tile::kA;
    if (m0 >= count) return;
    f32x16_t acc[TA][TB];
    Tile::template sums<false>(s0, s1, s2, s3, a.weight, a.hidden, v_tile, m0, a.d, acc);
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64, wa = wave / GB, wb = wave % GB;
    const uint32_t v_lane = v_tile + 32 * TA * wa + 4 * (lane / 32);
    float2* joint = reinterpret_cast<float2*>(s0);  // [wa][kB]
#pragma unroll
    for (int tb = 0; tb < TB; ++tb) {
        const uint32_t in = 32 * (TB * wb + tb) + lane % 32, m = m0 + in;
        const bool live = m < count;
        const int32_t target = live ? a.r.target[m] : -1;
        if constexpr (!GRAD) {
            float top = -INFINITY, sum = 0.0f;
#pragma unroll
            for (int ta = 0; ta < TA; ++ta) {  // sixteen at a time against the largest so far
                float y[16], most = top;
#pragma unroll
                for (int i = 0; i < 16; ++i) y[i] = acc[ta][tb][i];
                cap_logits(y, a.softcap);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const uint32_t v = v_lane + 32 * ta + 8 * (i / 4) + i % 4;
                    if (static_cast<int32_t>(v) == target) a.r.hit[m] = y[i];
                    y[i] = v < a.vocab ? y[i] : -INFINITY;
                    most = fmaxf(most, y[i]);
                }
                const float ref = most > -INFINITY ? most * kLog2e : 0.0f;  // nothing of the vocabulary yet: no infinity less itself
                sum *= __builtin_amdgcn_exp2f(fmaf(top, kLog2e, -ref));
#pragma unroll
                for (int i = 0; i < 16; ++i) sum += __builtin_amdgcn_exp2f(fmaf(y[i], kLog2e, -ref));
                top = most;
            }
            const float other_top = __shfl_xor(top, 32), other_sum = __shfl_xor(sum, 32);
            const float both = fmaxf(top, other_top), ref = both > -INFINITY ? both : 0.0f;
            sum = sum * __builtin_amdgcn_exp2f((top - ref) * kLog2e) + other_sum * __builtin_amdgcn_exp2f((other_top - ref) * kLog2e);
            if (lane < 32) joint[wa * Tile::kB + in] = make_float2(both, sum);
        } else {
            const float lse = live ? a.r.lse[m] : 0.0f, grad = live ? a.r.grad[m] : 0.0f;
#pragma unroll
            for (int ta = 0; ta < TA; ++ta) {
                float y[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) y[i] = acc[ta][tb][i];
                cap_logits(y, a.softcap);
                uint32_t e[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const uint32_t v = v_lane + 32 * ta + 8 * (i / 4) + i % 4;
                    float p = __builtin_amdgcn_exp2f((y[i] - lse) * kLog2e);
                    if (static_cast<int32_t>(v) == target) p -= 1.0f;
                    const float c = y[i] * a.softcap.inv;
                    if (a.softcap.cap > 0.0f) p *= fmaf(-c, c, 1.0f);
                    e[i] = live && v < a.vocab ? bf16_bits(p * grad) : 0u;
                    const uint32_t row = v - a.v0;
                    if (m < a.dzt_stride) a.dzt[static_cast<uint64_t>(row) * a.dzt_stride + m] = static_cast<uint16_t>(e[i]);
                }
                if (m < a.dzt_stride) {
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        const u32x2_t w = {e[i] | e[i + 1] << 16, e[i + 2] | e[i + 3] << 16};
                        *reinterpret_cast<u32x2_t*>(a.dz + static_cast<uint64_t>(m) * a.dz_stride + (v_lane - a.v0) + 32 * ta + 2 * i) = w;
                    }
                }
            }
        }
    }
    if constexpr (!GRAD) {
        __syncthreads();
        for (uint32_t in = threadIdx.x; in < Tile::kB && m0 + in < count; in += kProductThreads) {
            float2 p = joint[in];
#pragma unroll
            for (uint32_t w = 1; w < GA; ++w) {
                const float2 q = joint[w * Tile::kB + in];
                const float top = fmaxf(p.x, q.x), ref = top > -INFINITY ? top : 0.0f;
                p.y = p.y * __builtin_amdgcn_exp2f((p.x - ref) * kLog2e) + q.y * __builtin_amdgcn_exp2f((q.x - ref) * kLog2e);
                p.x = top;
            }
            a.part[static_cast<uint64_t>(at.a) * a.part_stride + m0 + in] = p;
        }
    }
}

struct JoinArgs {
    LossRows r;
    const float2* part;
    uint32_t tiles, part_stride;
    float* losses;
    float* lse;
};

// The tiles' parts of sixteen rows, 64 tiles at a time; the sum of a row's exponentials in 64 bits.
constexpr uint32_t kJoinRows = 16, kJoinThreads = 1024;

__global__ __launch_bounds__(kJoinThreads) void loss_join_kernel(JoinArgs a) {
    __shared__ float tops[kJoinThreads];
    __shared__ double sums[kJoinThreads];
    const uint32_t count = *a.r.count, in = threadIdx.x % kJoinRows, lead = threadIdx.x / kJoinRows;
    constexpr uint32_t kLeads = kJoinThreads / kJoinRows;
    if (blockIdx.x * kJoinRows >= count) return;
    const uint32_t m = min(blockIdx.x * kJoinRows + in, count - 1);
    float top = -INFINITY;
    double sum = 0.0;
    for (uint32_t i = lead; i < a.tiles; i += kLeads) {
        const float2 p = a.part[static_cast<uint64_t>(i) * a.part_stride + m];
        const float both = fmaxf(top, p.x);  // a NaN stays in the sum
        sum = sum * __builtin_amdgcn_exp2f((top - both) * kLog2e) + static_cast<double>(p.y) * __builtin_amdgcn_exp2f((p.x - both) * kLog2e);
        top = both;
    }
    tops[threadIdx.x] = top, sums[threadIdx.x] = sum;
    for (uint32_t half = kLeads / 2; half > 0; half /= 2) {
        __syncthreads();
        if (lead < half) {
            const uint32_t o = threadIdx.x + half * kJoinRows;
            const float other = tops[o], both = fmaxf(top, other), ref = both > -INFINITY ? both : 0.0f;
            sum = sum * __builtin_amdgcn_exp2f((top - ref) * kLog2e) + sums[o] * __builtin_amdgcn_exp2f((other - ref) * kLog2e);
            top = both;
            tops[threadIdx.x] = top, sums[threadIdx.x] = sum;
        }
    }
    if (lead == 0 && blockIdx.x * kJoinRows + in < count) {
        const float extra = static_cast<float>(log(sum));  // the loss without lse's rounding where they are close
        const uint32_t row = a.r.at[m];
        a.lse[row] = static_cast<float>(static_cast<double>(top) + log(sum));
        a.losses[row] = (top - a.r.hit[m]) + extra;
    }
}

// A matrix's columns as rows: out[c][r] = in[r0 + r][c], 64 x 64 at a time; rows from `rows` on read as zero.
struct TurnArgs {
    const uint16_t* in;
    uint64_t stride;
    uint32_t rows, cols;
    const uint32_t* count;  // where given, the rows
    uint16_t* out;
    uint32_t out_stride, out_cols;  // out_cols: a multiple of 8
};

__global__ __launch_bounds__(256) void loss_turn_kernel(TurnArgs a) {
    __shared__ uint16_t tile[64][72];
    const uint32_t rows = a.count ? *a.count : a.rows;
    const uint32_t r0 = blockIdx.x * 64, c0 = blockIdx.y * 64, t = threadIdx.x;
    for (uint32_t i = t; i < 64 * 8; i += 256) {
        const uint32_t r = i / 8, c = i % 8 * 8;
        u32x4_t w = {0, 0, 0, 0};
        if (r0 + r < rows && c0 + c < a.cols) w = *reinterpret_cast<const u32x4_t*>(a.in + (r0 + r) * a.stride + c0 + c);
        *reinterpret_cast<u32x4_t*>(&tile[r][c]) = w;
    }
    __syncthreads();
    for (uint32_t i = t; i < 64 * 8; i += 256) {
        const uint32_t c = i / 8, r = i % 8 * 8;
        if (c0 + c >= a.cols || r0 + r >= a.out_cols) continue;
        u32x4_t w;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = tile[r + 2 * j][c] | static_cast<uint32_t>(tile[r + 2 * j + 1][c]) << 16;
        *reinterpret_cast<u32x4_t*>(a.out + static_cast<uint64_t>(c0 + c) * a.out_stride + r0 + r) = w;
    }
}

struct GradArgs {
    const uint32_t* count;
    Operand a, b;
    uint32_t k, k_part;      // columns, and those of a part of the sum
    uint32_t rows, cols;     // of the result
    bool by_count;           // d_weight: k is the count's; d_hidden: rows are
    TileGrid grid;
    void* out;
    uint64_t stride, part;   // between the result's rows, and its parts
    bool add;
};

__device__ __forceinline__ void put4(float* p, f32x4_t v, bool add) {
    if (add) v += *reinterpret_cast<const f32x4_t*>(p);
    *reinterpret_cast<f32x4_t*>(p) = v;
}
__device__ __forceinline__ void put4(uint16_t* p, f32x4_t v, bool add) {
    if (add) {
        const u32x2_t w = *reinterpret_cast<const u32x2_t*>(p);
        v[0] += bf16_lo(w[0]), v[1] += bf16_hi(w[0]), v[2] += bf16_lo(w[1]), v[3] += bf16_hi(w[1]);
    }
    *reinterpret_cast<u32x2_t*>(p) = u32x2_t{bf16_bits(v[0]) | bf16_bits(v[1]) << 16, bf16_bits(v[2]) | bf16_bits(v[3]) << 16};
}

template <typename Tile, int TA, int TB, int GA, int GB, typename Out>
__global__ __launch_bounds__(kProductThreads) __attribute__((amdgpu_waves_per_eu(kWavesPerEu<Tile>, kWavesPerEu<Tile>))) void loss_grad_kernel(GradArgs a) {
    __shared__ u32x4_t s0[Tile::kStage], s1[Tile::kStage], s2[Tile::kStage], s3[Tile::kStage];
    TileAt at;
    if (!tile_of_block(a.grid, &at)) return;
    const uint32_t count = *a.count, a0 = at.a * Tile::kA, b0 = at.b * Tile::kB;
    if (!a.by_count && a0 >= count) return;
    const uint32_t k_all = a.by_count ? (count + 127) / 128 * 128 : a.k;
    const uint32_t k0 = min(at.part * a.k_part, k_all), k = min(k_all - k0, a.k_part);
    f32x16_t acc[TA][TB];
    if (k > 0) {
        Operand x = a.a, y = a.b;
        x.p += k0, y.p += k0;
        Tile::template sums<true>(s0, s1, s2, s3, x, y, a0, b0, k, acc);
    } else {
#pragma unroll
        for (int i = 0; i < TA; ++i)
#pragma unroll
            for (int j = 0; j < TB; ++j) acc[i][j] = f32x16_t{};
    }
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64, wa = wave / GB, wb = wave % GB;
    Out* const out = static_cast<Out*>(a.out) + at.part * a.part;
#pragma unroll
    for (int ta = 0; ta < TA; ++ta) {
        const uint32_t row = a0 + 32 * (TA * wa + ta) + lane % 32;
        if (row >= a.rows) continue;
#pragma unroll
        for (int tb = 0; tb < TB; ++tb)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const uint32_t col = b0 + 32 * (TB * wb + tb) + 2 * i + 4 * (lane / 32);
                const f32x4_t v = {acc[ta][tb][i], acc[ta][tb][i + 1], acc[ta][tb][i + 2], acc[ta][tb][i + 3]};
                if (col < a.cols) put4(out + row * a.stride + col, v, a.add);
            }
    }
}

struct SpreadArgs {
    LossRows r;
    const int32_t* targets;
    const float* part;   // [part][m][d]
    uint32_t parts, rows, vocab, d;
    uint64_t part_size;
    uint16_t* out;
    uint64_t stride;
};

// d_hidden's parts added up, in the caller's rows; zeros where a row is left out.
__global__ __launch_bounds__(256) void loss_spread_kernel(SpreadArgs a) {
    const uint32_t c = (blockIdx.y * 256 + threadIdx.x) * 8, b = blockIdx.x;
    if (c >= a.d) return;
    // a block writes row `at[b]` from sum b, and row b if it is left out
    if (static_cast<uint32_t>(a.targets[b]) >= a.vocab) *reinterpret_cast<u32x4_t*>(a.out + b * a.stride + c) = u32x4_t{0, 0, 0, 0};
    if (b >= *a.r.count) return;
    f32x4_t lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
    for (uint32_t p = 0; p < a.parts; ++p) {
        const f32x4_t* from = reinterpret_cast<const f32x4_t*>(a.part + p * a.part_size + static_cast<uint64_t>(b) * a.d + c);
        lo += from[0], hi += from[1];
    }
    const u32x4_t w = {bf16_bits(lo[0]) | bf16_bits(lo[1]) << 16, bf16_bits(lo[2]) | bf16_bits(lo[3]) << 16,
                       bf16_bits(hi[0]) | bf16_bits(hi[1]) << 16, bf16_bits(hi[2]) | bf16_bits(hi[3]) << 16};
    *reinterpret_cast<u32x4_t*>(a.out + a.r.at[b] * a.stride + c) = w;
}

uint32_t div_up(uint64_t x, uint32_t y) { return static_cast<uint32_t>((x + y - 1) / y); }
uint32_t round_up(uint32_t x, uint32_t y) { return div_up(x, y) * y; }

constexpr uint32_t kLossMaxRows = 65536, kLossMaxVocab = 1u << 24;
constexpr uint32_t kRowPad = 128;

// How a backward pass over `rows` rows is cut.
struct BackPlan {
    uint32_t m;       // rows, rounded up: dzt's stride
    uint32_t piece;   // vocabulary rows at a time, a multiple of 256
    uint32_t parts;   // of d_hidden's sums
    uint64_t dz, wt, part;  // elements of dz (and of dzt), of the turned weights and of all parts
};

BackPlan back_plan(uint32_t rows, uint32_t vocab, uint32_t d) {
    BackPlan p{};
    p.m = round_up(rows, kRowPad);
    const uint32_t all = round_up(vocab, 256);
    uint32_t most = static_cast<uint32_t>((1ull << 27) / p.m) / 256 * 256;
    most = most < 32768 ? most : 32768;
    most = most > 256 ? most : 256;
    p.piece = round_up(div_up(all, div_up(all, most)), 256);
    const uint32_t tiles = div_up(p.m, 256) * div_up(d, 256);
    const uint32_t want = div_up(512, tiles), can = div_up(p.piece, 1024);
    p.parts = want < can ? want : can;
    p.dz = static_cast<uint64_t>(p.m) * p.piece;
    p.wt = static_cast<uint64_t>(d) * p.piece;
    p.part = static_cast<uint64_t>(p.parts) * p.m * d;
    return p;
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace

}  // namespace twd

struct twd_headloss {
    twd::StreamOrder order;
    twd::LossRows r;
    float2* part;      // forward
    uint16_t* ht;      // backward: [d][m]
    uint16_t* dz;      // [m][piece]
    uint16_t* dzt;     // [piece][m]
    uint16_t* wt;      // [d][piece]
    float* dh;         // [part][m][d]
    void* block;       // the one allocation behind them
    uint64_t bytes;
    uint32_t max_rows, vocab, d, d_pad;  // d_pad: a multiple of 128
    float softcap;
    bool backward;
    int device;
};

namespace twd {

namespace {

template <bool GRAD>
int launch_logits(const twd_headloss* l, LogitArgs a, uint32_t rows, uint32_t vocab_rows, hipStream_t s) {
    auto go = [&](auto tile, auto ta, auto tb, auto ga, auto gb) -> int {
        using Tile = decltype(tile);
        a.grid = TileGrid{div_up(vocab_rows, Tile::kA), div_up(rows, Tile::kB), 1};
        loss_logits_kernel<Tile, ta(), tb(), ga(), gb(), GRAD><<<a.grid.blocks(), kProductThreads, 0, s>>>(a);
        TWD_HIP(hipGetLastError());
        return TWD_OK;
    };
    using std::integral_constant;
    if (!GRAD && rows <= 64)  // dz is written for whole steps of 128 rows
        return go(ProductTile<2, 2, 4, 1>{}, integral_constant<int, 2>{}, integral_constant<int, 2>{}, integral_constant<int, 4>{}, integral_constant<int, 1>{});
    if (rows <= 128)
        return go(ProductTile<4, 2, 2, 2>{}, integral_constant<int, 4>{}, integral_constant<int, 2>{}, integral_constant<int, 2>{}, integral_constant<int, 2>{});
    return go(ProductTile<4, 4, 2, 2>{}, integral_constant<int, 4>{}, integral_constant<int, 4>{}, integral_constant<int, 2>{}, integral_constant<int, 2>{});
}

template <typename Out>
int launch_grad(GradArgs a, hipStream_t s) {
    using Tile = ProductTile<4, 4, 2, 2>;
    a.grid = TileGrid{div_up(a.rows, Tile::kA), div_up(a.cols, Tile::kB), a.grid.parts};
    loss_grad_kernel<Tile, 4, 4, 2, 2, Out><<<a.grid.blocks(), kProductThreads, 0, s>>>(a);
    TWD_HIP(hipGetLastError());
    return TWD_OK;
}

int launch_gather(const twd_headloss* l, GatherArgs a, hipStream_t s) {
    a.r = l->r, a.vocab = l->vocab, a.pieces = l->d / 8, a.h_pieces = l->d_pad / 8;
    loss_gather_kernel<<<div_up(a.rows, kGatherRows), 256, 0, s>>>(a);
    TWD_HIP(hipGetLastError());
    return TWD_OK;
}

int launch_turn(TurnArgs a, hipStream_t s) {
    loss_turn_kernel<<<dim3(div_up(a.out_cols, 64), div_up(a.cols, 64)), 256, 0, s>>>(a);
    TWD_HIP(hipGetLastError());
    return TWD_OK;
}

int forward(const twd_headloss* l, const GatherArgs& g, const Operand& weight, hipStream_t s) {
    if (const int rc = launch_gather(l, g, s)) return rc;
    LogitArgs a{};
    a.r = l->r, a.weight = weight, a.hidden = Operand{l->r.h, l->d_pad, g.rows};
    a.d = l->d, a.vocab = l->vocab, a.softcap = soft_cap(l->softcap), a.part = l->part, a.part_stride = g.rows;
    if (const int rc = launch_logits<false>(l, a, g.rows, l->vocab, s)) return rc;
    loss_join_kernel<<<div_up(g.rows, kJoinRows), kJoinThreads, 0, s>>>(
        JoinArgs{l->r, l->part, div_up(l->vocab, 256), g.rows, g.losses, g.lse_out});
    TWD_HIP(hipGetLastError());
    return TWD_OK;
}

struct BackOut {
    uint16_t* d_hidden;
    uint64_t d_hidden_stride;
    void* d_weight;
    int type;
    uint64_t d_weight_stride;
    bool add;
};

int backward(const twd_headloss* l, const GatherArgs& g, const Operand& weight, const BackOut& o, hipStream_t s) {
    const BackPlan p = back_plan(g.rows, l->vocab, l->d);
    int rc = launch_gather(l, g, s);
    if (rc) return rc;
    if (o.d_weight && (rc = launch_turn(TurnArgs{l->r.h, l->d_pad, 0, l->d, l->r.count, l->ht, p.m, p.m}, s))) return rc;
    for (uint32_t v0 = 0; v0 < l->vocab; v0 += p.piece) {
        const uint32_t here = l->vocab - v0 < p.piece ? l->vocab - v0 : p.piece, k = round_up(here, 128);
        LogitArgs a{};
        a.r = l->r, a.weight = weight, a.hidden = Operand{l->r.h, l->d_pad, g.rows};
        a.d = l->d, a.vocab = l->vocab, a.v0 = v0, a.softcap = soft_cap(l->softcap);
        a.dz = l->dz, a.dzt = l->dzt, a.dz_stride = p.piece, a.dzt_stride = p.m;
        if ((rc = launch_logits<true>(l, a, g.rows, here, s))) return rc;
        if (o.d_weight) {
            GradArgs b{};
            b.count = l->r.count, b.a = Operand{l->dzt, p.m, here}, b.b = Operand{l->ht, p.m, l->d};
            b.k_part = p.m, b.rows = here, b.cols = l->d, b.by_count = true, b.grid.parts = 1;
            b.stride = o.d_weight_stride, b.add = o.add;
            const uint64_t size = o.type == TWD_F32 ? 4 : 2;
            b.out = static_cast<char*>(o.d_weight) + v0 * o.d_weight_stride * size;
            if ((rc = o.type == TWD_F32 ? launch_grad<float>(b, s) : launch_grad<uint16_t>(b, s))) return rc;
        }
        if (o.d_hidden) {
            const TurnArgs t{weight.p + v0 * weight.stride, weight.stride, here, l->d, nullptr, l->wt, p.piece, k};
            if ((rc = launch_turn(t, s))) return rc;
            GradArgs b{};
            b.count = l->r.count, b.a = Operand{l->dz, p.piece, p.m}, b.b = Operand{l->wt, p.piece, l->d};
            b.k = k, b.k_part = round_up(div_up(k, p.parts), 128), b.rows = p.m, b.cols = l->d, b.grid.parts = p.parts;
            b.out = l->dh, b.stride = l->d, b.part = static_cast<uint64_t>(p.m) * l->d, b.add = v0 > 0;
            if ((rc = launch_grad<float>(b, s))) return rc;
        }
    }
    if (!o.d_hidden) return TWD_OK;
    loss_spread_kernel<<<dim3(g.rows, div_up(l->d, 2048)), 256, 0, s>>>(
        SpreadArgs{l->r, g.targets, l->dh, p.parts, g.rows, l->vocab, l->d, static_cast<uint64_t>(p.m) * l->d, o.d_hidden, o.d_hidden_stride});
    TWD_HIP(hipGetLastError());
    return TWD_OK;
}

int check_rows(const char* what, const void* p, uint64_t stride, uint32_t rows, uint32_t d, uint64_t most) {
    if (!aligned16(p)) return fail(TWD_E_INVALID, std::string(what) + " must start at a multiple of 16 bytes");
    if (rows > 1 && (stride < d || stride % 8 != 0))
        return fail(TWD_E_INVALID, std::string(what) + ": the row stride must be a multiple of 8 and at least d_model");
    if (rows > 1 && stride > most) return fail(TWD_E_INVALID, std::string(what) + ": the row stride is too large");
    return TWD_OK;
}

int check_call(const twd_headloss* l, const void* hidden, uint32_t rows, uint64_t hidden_stride, const void* weight,
               uint64_t weight_stride, const void* targets) {
    if (!l) return fail(TWD_E_INVALID, "null head loss");
    if (!hidden || !weight || !targets) return fail(TWD_E_INVALID, "null argument");
    if (rows == 0 || rows > l->max_rows) return fail(TWD_E_INVALID, "rows out of range for this head loss");
    int rc = check_rows("hidden", hidden, hidden_stride, rows, l->d, kMaxProductStride);
    if (rc) return rc;
    if ((rc = check_rows("weight", weight, weight_stride, l->vocab, l->d, kMaxProductStride))) return rc;
    int dev = 0;
    TWD_HIP(hipGetDevice(&dev));
    if (dev != l->device) return fail(TWD_E_INVALID, "the head loss lives on another device than the current one");
    return TWD_OK;
}

}  // namespace

}  // namespace twd

using namespace twd;

extern "C" {

TWD_API int twd_headloss_create(uint32_t max_rows, uint32_t vocab, uint32_t d_model, float softcap, int backward,
                                twd_headloss** out) {
    clear_error();
    if (!out) return fail(TWD_E_INVALID, "null argument");
    *out = nullptr;
    if (max_rows == 0 || max_rows > kLossMaxRows) return fail(TWD_E_INVALID, "max_rows must be in 1..65536");
    if (vocab == 0 || vocab > kLossMaxVocab) return fail(TWD_E_INVALID, "vocab must be in 1..2^24");
    if (d_model == 0 || d_model % 32 != 0 || d_model > (1u << 20))
        return fail(TWD_E_INVALID, "d_model must be a positive multiple of 32, at most 2^20");
    if (softcap != 0.0f && !(softcap >= kMinSoftCap && softcap <= kMaxSoftCap))
        return fail(TWD_E_INVALID, "softcap must be 0 (none) or in 1e-30..1e30");
    int dev = 0;
    TWD_HIP(hipGetDevice(&dev));
    twd_headloss* l = new (std::nothrow) twd_headloss{};
    if (!l) return fail(TWD_E_INVALID, "out of host memory");
    l->max_rows = max_rows, l->vocab = vocab, l->d = d_model, l->d_pad = round_up(d_model, 128), l->softcap = softcap, l->backward = backward != 0, l->device = dev;
    uint64_t dz = 0, wt = 0, part = 0;
    const uint32_t m = round_up(max_rows, kRowPad);
    for (uint32_t rows = kRowPad; l->backward && rows <= m; rows += kRowPad) {  // the most that any number of rows takes
        const BackPlan p = back_plan(rows, vocab, d_model);
        dz = p.dz > dz ? p.dz : dz, wt = p.wt > wt ? p.wt : wt, part = p.part > part ? p.part : part;
    }
    char* at = nullptr;
    uint64_t size = 0;
    auto take = [&](auto*& p, uint64_t n) {
        p = reinterpret_cast<std::remove_reference_t<decltype(p)>>(at + size);
        size += (n * sizeof(*p) + 255) / 256 * 256;
    };
    auto lay_out = [&] {
        size = 0;
        take(l->r.count, 1);
        take(l->r.at, m);
        take(l->r.target, m);
        take(l->r.grad, m);
        take(l->r.lse, m);
        take(l->r.hit, m);
        take(l->r.h, static_cast<uint64_t>(m) * l->d_pad);
        take(l->part, static_cast<uint64_t>(div_up(vocab, 256)) * max_rows);
        if (!l->backward) return;
        take(l->ht, static_cast<uint64_t>(m) * d_model);
        take(l->dz, dz);
        take(l->dzt, dz);
        take(l->wt, wt);
        take(l->dh, part);
    };
    lay_out();
    const hipError_t e = hipMalloc(&l->block, size);
    if (e != hipSuccess) {
        delete l;
        return hip_fail(e, "allocating the head loss's scratch");
    }
    at = static_cast<char*>(l->block);
    lay_out();
    l->bytes = size;
    *out = l;
    return TWD_OK;
}

TWD_API void twd_headloss_destroy(twd_headloss* l) {
    if (!l) return;
    order_release(l->order);
    (void)hipFree(l->block);
    delete l;
}

TWD_API int twd_headloss_info(const twd_headloss* l, uint64_t* device_bytes) {
    clear_error();
    if (!l) return fail(TWD_E_INVALID, "null head loss");
    if (device_bytes) *device_bytes = l->bytes;
    return TWD_OK;
}

TWD_API int twd_headloss_forward(twd_headloss* l, const uint16_t* hidden_bf16, uint32_t rows, uint64_t hidden_stride,
                                 const uint16_t* weight_bf16, uint64_t weight_stride, const int32_t* targets,
                                 float* losses, float* lse, void* stream) {
    clear_error();
    int rc = check_call(l, hidden_bf16, rows, hidden_stride, weight_bf16, weight_stride, targets);
    if (rc) return rc;
    if (!losses || !lse) return fail(TWD_E_INVALID, "null argument");
    const hipStream_t s = static_cast<hipStream_t>(stream);
    GatherArgs g{};
    g.hidden = hidden_bf16, g.stride = hidden_stride, g.targets = targets, g.losses = losses, g.lse_out = lse, g.rows = rows;
    if ((rc = order_before(l->order, s))) return rc;
    if ((rc = forward(l, g, Operand{weight_bf16, weight_stride, l->vocab}, s))) return rc;
    return order_after(l->order, s);
}

TWD_API int twd_headloss_backward(twd_headloss* l, const uint16_t* hidden_bf16, uint32_t rows, uint64_t hidden_stride,
                                  const uint16_t* weight_bf16, uint64_t weight_stride, const int32_t* targets,
                                  const float* lse, const float* grad, uint16_t* d_hidden_bf16, uint64_t d_hidden_stride,
                                  void* d_weight, int d_weight_type, uint64_t d_weight_stride, int accumulate, void* stream) {
    clear_error();
    int rc = check_call(l, hidden_bf16, rows, hidden_stride, weight_bf16, weight_stride, targets);
    if (rc) return rc;
    if (!l->backward) return fail(TWD_E_INVALID, "this head loss was made without its backward pass");
    if (!lse) return fail(TWD_E_INVALID, "null argument");
    if (!d_hidden_bf16 && !d_weight) return fail(TWD_E_INVALID, "neither d_hidden nor d_weight is asked for");
    if (d_hidden_bf16 && (rc = check_rows("d_hidden", d_hidden_bf16, d_hidden_stride, rows, l->d, ~0ull))) return rc;
    if (d_weight) {
        if (d_weight_type != TWD_F32 && d_weight_type != TWD_BF16) return fail(TWD_E_INVALID, "d_weight must be fp32 or bf16");
        if ((rc = check_rows("d_weight", d_weight, d_weight_stride, l->vocab, l->d, ~0ull))) return rc;
    }
    const hipStream_t s = static_cast<hipStream_t>(stream);
    GatherArgs g{};
    g.hidden = hidden_bf16, g.stride = hidden_stride, g.targets = targets, g.grad = grad, g.lse_in = lse, g.rows = rows;
    const BackOut o{d_hidden_bf16, d_hidden_stride, d_weight, d_weight_type, d_weight_stride, accumulate != 0};
    if ((rc = order_before(l->order, s))) return rc;
    if ((rc = backward(l, g, Operand{weight_bf16, weight_stride, l->vocab}, o, s))) return rc;
    return order_after(l->order, s);
}

}  // extern "C"
