// Softmax cross entropy of a bf16 head's logits, and its gradients, a piece of the vocabulary at a time.
//
//   z_mv = softcap(h_m . w_v)   lse_m = ln sum_v exp(z_mv)   loss_m = lse_m - z_m,t(m)
//   dz_mv = g_m (exp(z_mv - lse_m) - [v = t(m)]) (1 - (z_mv / cap)^2)   d_hidden = dz W   d_weight = dz^T H
//
// The rows that count are first gathered one behind another, so rows that are left out cost nothing and cannot spoil a
// sum. Forward, each tile of logits is reduced where it was summed to its rows' largest value and their sum of
// exponentials against it; a second kernel joins the tiles. Backward, a piece of the vocabulary after another: the
// logits again, dz of them in bf16 by rows, then the two products.
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
    uint16_t* h;    // [m][d]
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
    uint32_t rows, vocab, pieces;  // of 16 bytes in a row
    uint32_t each;                 // rows of a block
};

// A block counts the rows before its own that count, then brings its own to their places: one launch instead of a prefix sum
// and a copy. Reads the hidden rows once and writes them once; 2,048 rows of 5,376 take 12 us, 777 of 2,048 6, most of it a
// block's count and the row after it.
__global__ __launch_bounds__(256) void loss_gather_kernel(GatherArgs a) {
    __shared__ uint32_t wave_sum[4];
    const uint32_t r0 = blockIdx.x * a.each, t = threadIdx.x;
    auto counts = [&](uint32_t r) { return static_cast<uint32_t>(a.targets[r]) < a.vocab; };
    uint32_t before = 0;
    for (uint32_t r = t; r < r0; r += 256) before += counts(r) ? 1u : 0u;
    before = wave_reduce(before, 0u, [](uint32_t x, uint32_t y) { return x + y; });
    if (t % 64 == 0) wave_sum[t / 64] = before;
    __syncthreads();
    uint32_t m = wave_sum[0] + wave_sum[1] + wave_sum[2] + wave_sum[3];
    const uint32_t last = min(r0 + a.each, a.rows);
    for (uint32_t r = r0; r < last; ++r) {
        if (!counts(r)) {
            if (t == 0 && a.losses) a.losses[r] = 0.0f, a.lse_out[r] = 0.0f;
            continue;
        }
        const u32x4_t* from = reinterpret_cast<const u32x4_t*>(a.hidden + r * a.stride);
        u32x4_t* to = reinterpret_cast<u32x4_t*>(a.r.h) + static_cast<uint64_t>(m) * a.pieces;
        for (uint32_t i = t; i < a.pieces; i += 256) to[i] = from[i];
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
    uint32_t v0, here;    // the piece's first vocabulary row, and its rows
    SoftCap softcap;
    float2* part;         // forward: [tile][stride] largest logit and sum of exponentials
    uint16_t* dz;         // backward: [m][dz_stride], from v0 on
    uint32_t part_stride, dz_stride;
};

// Logits: both operands by rows. d_hidden: the weights turned. d_weight: dz and the hidden rows turned.
using TileFew = ProductTile<1, 2, 4, 1, 64, 3, false, false, false, true>;
template <bool STREAMED>
using TileFewest = ProductTile<1, 1, 2, 2, 64, 4, false, false, false, STREAMED>;  // 64 vocabulary rows
template <bool STREAMED>
using TileMid = ProductTile<4, 2, 2, 2, 64, 3, false, false, false, STREAMED>;  // 128 hidden rows
using TileMidSmall = ProductTile<2, 2, 2, 2, 64, 4, false, false>;              // and 128 vocabulary rows
using TileWide = ProductTile<4, 4, 2, 2, 64, 2, false, false, true>;
using TileThree = ProductTile<4, 3, 2, 2, 64, 2, false, false, true>;
using TileTwo = ProductTile<4, 2, 2, 2, 64, 2, false, false, true>;
using TileStripe = ProductTile<2, 2, 4, 1, 64, 3, false, false, true>;  // a quarter of a wide one
using TileHidden = ProductTile<4, 4, 2, 2, 32, 4, false, true>;
using TileHiddenFew = ProductTile<4, 2, 1, 4, 32, 3, false, true, false, false, true>;  // up to 128 rows
using TileWeight = ProductTile<4, 2, 2, 2, 32, 3, true, true>;
using TileWeightFew = ProductTile<2, 2, 2, 2, 32, 2, true, true>;

static_assert(TileWide::kA == kVocabTile && TileThree::kA == kVocabTile && TileTwo::kA == kVocabTile && TileStripe::kA == kVocabTile, "one width");
constexpr uint32_t kFewRows = 64, kMidRows = 128;

template <typename Tile>
constexpr int kWavesPerEu = Tile::kBytes > 81920 ? 1 : Tile::kBytes > 40960 ? 2 : 4;  // blocks to a unit

// The tile of vocabulary rows kA va .. and hidden rows m0 ..
template <typename Tile, bool GRAD>
__device__ __forceinline__ void logits_tile(const LogitArgs& a, uint32_t count, uint32_t va, uint32_t m0, uint32_t share, uint32_t who,
                                            u32x4_t* s0, u32x4_t* s1, u32x4_t* s2, u32x4_t* s3, uint32_t* sink) {
    constexpr int TA = Tile::kTA, TB = Tile::kTB, GA = Tile::kGA, GB = Tile::kGB;
    const uint32_t v_tile = a.v0 + va * Tile::kA;
    Operand w = a.weight, h = a.hidden;  // the piece's rows, and those from m0 on
    w.p += a.v0 * w.stride, w.rows = a.here;
    h.rows = count - m0;
    if (m0 > 0) h.p += m0 * h.stride;
    f32x16_t acc[TA][TB];
    Tile::template sums<false>(s0, s1, s2, s3, sink, w, h, TileAt{va, 0, 0, share, who}, a.d, acc);
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64, wa = wave / GB, wb = wave % GB;
    const uint32_t v_lane = v_tile + 32 * TA * wa + 4 * (lane / 32);
    const bool whole = v_tile + Tile::kA <= a.vocab;
    float2* joint = reinterpret_cast<float2*>(s0);  // [wa][kB]
    each<TB>([&](auto tb) {
        const uint32_t in = 32 * (TB * wb + tb) + lane % 32, m = m0 + in;
        const bool live = m < count;
        const uint32_t target = live ? static_cast<uint32_t>(a.r.target[m]) : ~0u;
        // square ta's logits, and which of them is the target's, if one is
        auto logits = [&](auto ta, float (&y)[16]) {
#pragma unroll
            for (int i = 0; i < 16; ++i) y[i] = acc[ta][tb][i];
            cap_logits(y, a.softcap);
        };
        auto in_lane = [](int i) { return 8u * (i / 4) + i % 4; };
        auto at_target = [&](auto ta, auto&& f) {
            const uint32_t off = target - (v_lane + 32 * ta);
            if (__builtin_amdgcn_ballot_w64(off < 32) == 0) return;
#pragma unroll
            for (int i = 0; i < 16; ++i) f(i, off == in_lane(i));
        };
        if constexpr (!GRAD) {
            float top = -INFINITY, sum = 0.0f, hit = 0.0f;
            each<TA>([&](auto ta) {  // sixteen at a time against the largest so far
                float y[16], most = top;
                logits(ta, y);
                at_target(ta, [&](int i, bool is) { hit = is ? y[i] : hit; });
                if (!whole) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) y[i] = v_lane + 32 * ta + in_lane(i) < a.vocab ? y[i] : -INFINITY;
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) most = fmaxf(most, y[i]);
                // the differences first: the logits may be large. Nothing of the vocabulary yet: no infinity less itself
                const float ref = most > -INFINITY ? most : 0.0f;
                sum *= __builtin_amdgcn_exp2f((top - ref) * kLog2e);
#pragma unroll
                for (int i = 0; i < 16; ++i) sum += __builtin_amdgcn_exp2f((y[i] - ref) * kLog2e);
                top = most;
                __builtin_amdgcn_sched_barrier(0);
            });
            const uint32_t off = target - v_lane;
            if (off < 32 * TA && off % 8 < 4) a.r.hit[m] = hit;
            const float other_top = __shfl_xor(top, 32), other_sum = __shfl_xor(sum, 32);
            const float both = fmaxf(top, other_top), ref = both > -INFINITY ? both : 0.0f;
            sum = sum * __builtin_amdgcn_exp2f((top - ref) * kLog2e) + other_sum * __builtin_amdgcn_exp2f((other_top - ref) * kLog2e);
            if (lane < 32) joint[wa * Tile::kB + in] = make_float2(both, sum);
        } else {
            // dz is rounded to bf16, as an operand of the matrix instructions: by at most 2^-8 of each term, of d_weight in fp32
            // too. To bf16 gradients that adds as much as their own rounding (2,048 rows: errors against 64 bits of 0.0024,
            // 0.0017 with dz in fp32); two halves of dz would be two products more beside the step's four, a half of its time.
            const float lse = live ? a.r.lse[m] : 0.0f, grad = live ? a.r.grad[m] : 0.0f;
            store_rows<TA, uint16_t>((wave < 2 ? s0 : s1) + wave % 2 * (TA * 128),
                [&](auto ta) {
                    float y[16];
                    f32x16_t dz;
                    logits(ta, y);
#pragma unroll
                    for (int i = 0; i < 16; ++i) dz[i] = __builtin_amdgcn_exp2f((y[i] - lse) * kLog2e);
                    at_target(ta, [&](int i, bool is) { dz[i] = is ? dz[i] - 1.0f : dz[i]; });
                    if (a.softcap.cap > 0.0f) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const float c = y[i] * a.softcap.inv;
                            dz[i] *= fmaf(-c, c, 1.0f);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) dz[i] *= grad;
                    if (!whole) {  // past the vocabulary the products read zeros
#pragma unroll
                        for (int i = 0; i < 16; ++i) dz[i] = v_lane + 32 * ta + in_lane(i) < a.vocab ? dz[i] : 0.0f;
                    }
                    __builtin_amdgcn_sched_barrier(0);
                    return dz;
                },
                [&](uint32_t row, uint32_t col, u32x4_t w) {
                    const uint32_t m_row = m0 + 32 * (TB * wb + tb) + row;
                    if (m_row < count)
                        *reinterpret_cast<u32x4_t*>(a.dz + static_cast<uint64_t>(m_row) * a.dz_stride + (v_tile - a.v0) + 32 * TA * wa + col) = w;
                });
        }
    });
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
            a.part[static_cast<uint64_t>(va) * a.part_stride + m0 + in] = p;
        }
    }
}

// One block to a unit, whose waves hold 256 sums a lane each: the widest tile reads least through LDS. 2,048 rows of 262,144 x
// 5,376 with a softcap take 4.65 to 4.75 ms, 1,215 to 1,240 TFLOP/s (a plain library product of the same rows 1,333): the matrix units are busy
// in 68% of the cycles, at the clock of some 1.6 GHz that the power leaves, the rest being a tile's first loads and its
// epilogue, which nothing covers: all 256 sums leave the accumulation registers at once there, and 20 registers (with dz 31) go
// through scratch memory, none in the loop of products. Tiles of 256 x 128 with two blocks to a unit, one's epilogue beside the other's products,
// took 6.06 ms where these took 4.90 (32,003 x 2,048 of 777 rows: 145 and 152 us). With dz stored, a piece of 65,536: 1.24 ms.
template <bool GRAD>
__global__ __launch_bounds__(kProductThreads) __attribute__((amdgpu_waves_per_eu(1, 1))) void loss_logits_kernel(LogitArgs a) {
    __shared__ u32x4_t s0[TileWide::kPieces], s1[TileWide::kPieces];
    __shared__ uint32_t sink[TileWide::kSink];
    const uint32_t count = *a.r.count;
    const LogitTiles t = logit_tiles(count, (a.here + kVocabTile - 1) / kVocabTile);
    const uint32_t tiles = t.grid.tiles() - t.cut, id = stretched(tiles);
    if (id >= tiles) return;
    const TileAt at = tile_at(t.grid, id);
    const uint32_t m0 = t.width * at.b;
    if (t.width == 256) logits_tile<TileWide, GRAD>(a, count, at.a, m0, at.share, at.who, s0, s1, nullptr, nullptr, sink);
    else if (t.width == 192) logits_tile<TileThree, GRAD>(a, count, at.a, m0, at.share, at.who, s0, s1, nullptr, nullptr, sink);
    else logits_tile<TileTwo, GRAD>(a, count, at.a, m0, at.share, at.who, s0, s1, nullptr, nullptr, sink);
}

// The last tiles, a stripe of 64 hidden rows to a block. Bound by its own chain of stages: 16 stripes of 2,880 columns 29 us,
// as a round of whole tiles takes 95; where few rows count and no tile is cut, 5 us.
template <bool GRAD>
__global__ __launch_bounds__(kProductThreads) __attribute__((amdgpu_waves_per_eu(1, 1))) void loss_stripes_kernel(LogitArgs a) {
    using Tile = TileStripe;
    __shared__ u32x4_t s0[Tile::kPieces], s1[Tile::kPieces], s2[Tile::kPieces];
    __shared__ uint32_t sink[Tile::kSink];
    const uint32_t count = *a.r.count;
    const LogitTiles t = logit_tiles(count, (a.here + kVocabTile - 1) / kVocabTile);
    const uint32_t each = t.width / 64, id = stretched(each * t.cut);
    if (id >= each * t.cut) return;
    const TileAt at = tile_at(t.grid, t.grid.tiles() - t.cut + id / each);
    const uint32_t m0 = t.width * at.b + 64 * (id % each);
    if (m0 < count) logits_tile<Tile, GRAD>(a, count, at.a, m0, each, id % each, s0, s1, s2, nullptr, sink);
}

// Up to 128 rows: bound by the read of the weights, so a tile has all of the rows. 17 rows of 262,144 x 5,376 take 440 us
// forward (6.4 TB/s; a pure read reaches 6.7), 128 rows 491 (5.7), 17 of 32,003 x 1,024 14 us (4.6 TB/s: the way to a block's
// first products).
template <typename Tile, bool GRAD>
__global__ __launch_bounds__(kProductThreads) __attribute__((amdgpu_waves_per_eu(kWavesPerEu<Tile>, kWavesPerEu<Tile>)))
void loss_few_kernel(LogitArgs a) {
    __shared__ u32x4_t s0[Tile::kPieces], s1[Tile::kPieces], s2[Tile::kPieces2], s3[Tile::kPieces3];
    const uint32_t count = *a.r.count, tiles = (a.here + Tile::kA - 1) / Tile::kA, id = stretched(tiles);
    if (id < tiles && count > 0) logits_tile<Tile, GRAD>(a, count, id, 0, 1, 0, s0, s1, s2, s3, nullptr);
}

// The forward pass of few rows without a gathering before it: a row to a lane.
template <typename Tile>
__global__ __launch_bounds__(kProductThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void loss_few_forward_kernel(LogitArgs a, GatherArgs g) {
    static_assert(kFewRows <= 64, "a row to a lane");
    __shared__ u32x4_t s0[Tile::kPieces], s1[Tile::kPieces], s2[Tile::kPieces], s3[Tile::kPieces3];
    __shared__ uint32_t places[64];
    __shared__ int32_t targets[64];
    const uint32_t r = threadIdx.x % 64;
    const int32_t target = r < g.rows ? g.targets[r] : -1;
    const uint64_t in = __ballot(static_cast<uint32_t>(target) < g.vocab);
    const uint32_t count = static_cast<uint32_t>(__popcll(in)), m = static_cast<uint32_t>(__popcll(in & ((1ull << r) - 1)));
    if (threadIdx.x < 64) {
        const bool counts = (in >> r & 1) != 0;
        if (counts) places[m] = r, targets[m] = target;
        if (blockIdx.x == 0) {
            if (counts) a.r.at[m] = r;
            else if (r < g.rows) g.losses[r] = 0.0f, g.lse_out[r] = 0.0f;
            if (r == 0) *a.r.count = count;
        }
    }
    __syncthreads();
    const uint32_t tiles = (a.here + Tile::kA - 1) / Tile::kA, id = stretched(tiles);
    if (id >= tiles || count == 0) return;
    a.r.target = targets;
    a.hidden.places = places;
    logits_tile<Tile, false>(a, count, id, 0, 1, 0, s0, s1, s2, s3, nullptr);
}

struct JoinArgs {
    LossRows r;
    const float2* part;
    uint32_t tiles, part_stride;
    float* losses;
    float* lse;
};

// The tiles' parts of sixteen rows, 64 tiles at a time; the sum of a row's exponentials in 64 bits. Little to read (2,048 rows
// of 1,024 tiles: 17 MB in 13 us), small calls are a chain of loads, exchanges and two logarithms: 5 us.
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
        // a NaN stays in the sum; a tile whose logits are all minus infinity has none
        const float both = fmaxf(top, p.x), ref = both > -INFINITY ? both : 0.0f;
        sum = sum * __builtin_amdgcn_exp2f((top - ref) * kLog2e) + static_cast<double>(p.y) * __builtin_amdgcn_exp2f((p.x - ref) * kLog2e);
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

// d_hidden has few tiles: its sums are cut into the parts, of at least 1,024 columns, that fill the units best, the fewest
// of those (2,048 rows of 5,376: 168 tiles in 3 parts, two full rounds). A call of few rows has smaller tiles, two to a unit.
__host__ __device__ inline uint32_t hidden_parts(uint32_t rows, uint32_t d, uint32_t piece, bool few) {
    const uint32_t most = few ? 32 : 16, least = few ? 512 : 1024, round = few ? 512 : 256;
    const uint64_t tiles = static_cast<uint64_t>(few ? 1 : (rows + 255) / 256) * ((d + 255) / 256);
    uint32_t best = 1;
    for (uint32_t n = 2; n <= most && n <= (piece + least - 1) / least; ++n)
        if (20 * ((tiles * n + round - 1) / round * best) < 19 * ((tiles * best + round - 1) / round * n)) best = n;
    return best;
}

struct GradArgs {
    const uint32_t* count;
    Operand a, b;
    uint32_t k, piece;     // d_hidden: of this product, and of the first
    uint32_t rows, cols;   // of the result
    void* out;
    uint64_t stride;       // between the result's rows; the parts of d_hidden follow one another
    bool add, few;
};

__device__ __forceinline__ void add4(float* p, f32x4_t v) { *reinterpret_cast<f32x4_t*>(p) += v; }
__device__ __forceinline__ void add4(uint16_t* p, f32x4_t v) {
    const u32x2_t w = *reinterpret_cast<const u32x2_t*>(p);
    *reinterpret_cast<u32x2_t*>(p) = u32x2_t{bf16_pair(v[0] + bf16_lo(w[0]), v[1] + bf16_hi(w[0])), bf16_pair(v[2] + bf16_lo(w[1]), v[3] + bf16_hi(w[1]))};
}

// d_weight = dz^T H (BY_COUNT: k runs over the rows that count) or a piece's part of d_hidden = dz W. For 2,048 rows of 65,536
// x 5,376 1.23 and 1.20 ms: 1,170 and 1,200 TFLOP/s, where the library's products with these operands reach 1,034 and 727.
// d_weight has many tiles with short sums: two blocks to a unit cover each other's first loads and stores, of up to 128 rows
// four, whose tiles are a quarter (128 rows of 32,003 x 1,024: 20 us, 24 in large ones). d_hidden has a long sum and few tiles: one
// large tile to a unit, the sum in parts; of up to 128 rows the read of the weights bounds it, so a tile has just these rows and two
// blocks share a unit (17 rows of 262,144 x 5,376: 432 us, 6.5 TB/s, 583 in large tiles; the small head 25 and 49).
template <typename Tile, typename Out, bool BY_COUNT>
__global__ __launch_bounds__(kProductThreads) __attribute__((amdgpu_waves_per_eu(kWavesPerEu<Tile>, kWavesPerEu<Tile>))) void loss_grad_kernel(GradArgs a) {
    constexpr int TA = Tile::kTA, TB = Tile::kTB, GB = Tile::kGB;
    static_assert(2 * TB * 256 <= Tile::kPieces, "two waves' fp32 sums change places in a buffer");
    __shared__ u32x4_t s0[Tile::kPieces], s1[Tile::kPieces], s2[Tile::kPieces2], s3[Tile::kPieces3];
    __shared__ uint32_t sink[Tile::kSink];
    const uint32_t count = *a.count, rows = BY_COUNT ? a.rows : count;
    const uint32_t parts = BY_COUNT ? 1 : hidden_parts(count, a.cols, a.piece, a.few);
    const TileGrid grid{(rows + Tile::kA - 1) / Tile::kA, (a.cols + Tile::kB - 1) / Tile::kB, parts};
    const uint32_t id = stretched(grid.tiles());
    if (id >= grid.tiles()) return;
    const TileAt at = tile_at(grid, id);
    const uint32_t a0 = at.a * Tile::kA, b0 = at.b * Tile::kB;
    Operand x = a.a, y = a.b;
    uint32_t k;
    if constexpr (BY_COUNT) {
        k = x.rows = y.rows = count;
    } else {
        const uint32_t k_part = ((a.k + parts - 1) / parts + 127) / 128 * 128, k0 = min(at.part * k_part, a.k);
        k = min(a.k - k0, k_part);
        x.rows = count;
        x.p += k0, x.cols = (k + 7) / 8 * 8;  // dz is zero past the vocabulary
        y.p += k0 * y.stride, y.rows = k;
    }
    f32x16_t acc[TA][TB];
    if (k > 0) {
        Tile::template sums<true>(s0, s1, s2, s3, sink, x, y, at, k, acc);
    } else {
#pragma unroll
        for (int i = 0; i < TA; ++i)
#pragma unroll
            for (int j = 0; j < TB; ++j) acc[i][j] = f32x16_t{};
    }
    const uint32_t wave = threadIdx.x / 64, wa = wave / GB, wb = wave % GB;
    Out* const out = static_cast<Out*>(a.out) + at.part * (rows * a.stride);
    auto place = [&](uint32_t ta, uint32_t row, uint32_t col) -> Out* {
        const uint32_t r = a0 + 32 * (TA * wa + ta) + row, c = b0 + 32 * TB * wb + col;
        return r < rows && c < a.cols ? out + r * a.stride + c : nullptr;
    };
    if (a.add) {  // on top of what is there, rounded once
        each<TA>([&](auto ta) {
            store_rows<TB, float>((wave < 2 ? s0 : s1) + wave % 2 * (TB * 256), [&](auto tb) { return acc[ta][tb]; },
                [&](uint32_t row, uint32_t col, u32x4_t w) {
                    Out* const p = place(ta, row, col);
                    if (p) add4(p, __builtin_bit_cast(f32x4_t, w));
                });
        });
    } else {
        each<TA>([&](auto ta) {
            store_rows<TB, Out>((wave < 2 ? s0 : s1) + wave % 2 * (TB * 64 * sizeof(Out)), [&](auto tb) { return acc[ta][tb]; },
                [&](uint32_t row, uint32_t col, u32x4_t w) {
                    Out* const p = place(ta, row, col);
                    if (!p) return;
                    // d_weight is past the caches' size and not read again here
                    if constexpr (BY_COUNT) __builtin_nontemporal_store(w, reinterpret_cast<u32x4_t*>(p));
                    else *reinterpret_cast<u32x4_t*>(p) = w;
                });
        });
    }
}

struct SpreadArgs {
    LossRows r;
    const int32_t* targets;
    const float* part;   // [part][m][d]
    uint32_t piece, vocab, d;
    uint16_t* out;
    uint64_t stride;
    bool few;
};

// d_hidden's parts added up, in the caller's rows; zeros where a row is left out. Bound by the read of the parts: 2,048 rows
// of 5,376 in three parts 30 us, 5.1 TB/s.
__global__ __launch_bounds__(256) void loss_spread_kernel(SpreadArgs a) {
    const uint32_t c = (blockIdx.y * 256 + threadIdx.x) * 8, b = blockIdx.x;
    if (c >= a.d) return;
    // a block writes row `at[b]` from sum b, and row b if it is left out
    if (static_cast<uint32_t>(a.targets[b]) >= a.vocab) *reinterpret_cast<u32x4_t*>(a.out + b * a.stride + c) = u32x4_t{0, 0, 0, 0};
    const uint32_t count = *a.r.count;
    if (b >= count) return;
    const uint32_t parts = hidden_parts(count, a.d, a.piece, a.few);
    f32x4_t lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
#pragma unroll 4
    for (uint32_t p = 0; p < parts; ++p) {
        const f32x4_t* from = reinterpret_cast<const f32x4_t*>(a.part + (static_cast<uint64_t>(p) * count + b) * a.d + c);
        lo += from[0], hi += from[1];
    }
    const u32x4_t w = {bf16_pair(lo[0], lo[1]), bf16_pair(lo[2], lo[3]), bf16_pair(hi[0], hi[1]), bf16_pair(hi[2], hi[3])};
    *reinterpret_cast<u32x4_t*>(a.out + a.r.at[b] * a.stride + c) = w;
}

uint32_t div_up(uint64_t x, uint32_t y) { return static_cast<uint32_t>((x + y - 1) / y); }
uint32_t round_up(uint32_t x, uint32_t y) { return div_up(x, y) * y; }

constexpr uint32_t kLossMaxRows = 65536, kLossMaxVocab = 1u << 24;
constexpr uint64_t kLossMaxLogits = 1ull << 38;  // 2^23 tiles of 128 rows: a launch's threads stay below 2^32

// dz holds a piece of the vocabulary, a multiple of 256 of it: 2^27 values with all rows (256 MB), and rows no further apart
// than a product takes them.
uint32_t most_of_piece(uint32_t rows) {
    const uint32_t most = static_cast<uint32_t>((1ull << 27) / rows) / 256 * 256, apart = kMaxProductStride;
    return most < 256 ? 256 : most < apart ? most : apart;
}
uint32_t piece_of(uint32_t rows, uint32_t vocab) {  // pieces alike
    const uint32_t all = round_up(vocab, 256);
    return round_up(div_up(all, div_up(all, most_of_piece(rows))), 256);
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace

}  // namespace twd

struct twd_headloss {
    twd::StreamOrder order;
    twd::LossRows r;
    float2* part;      // forward
    uint16_t* dz;      // backward: [m][piece]
    float* dh;         // [part][m][d]
    void* block;       // the one allocation behind them
    uint64_t bytes;
    uint32_t max_rows, vocab, d;
    float softcap;
    bool backward;
    int device;
};

namespace twd {

namespace {

// Up to 128 rows have tiles of all of them, so the weights are read once. f(tile): small tiles where large ones would leave
// units idle or not fill them for two rounds (17 rows of 100,000 x 2,048: 92 and 109 us; of 151,669 x 3,584: 209 and 198; 128
// rows of 32,003 x 1,024: 27 and 37; of 50,000 x 4,096: 121 and 109). Weights past the memory's cache are streamed (17 rows of
// 65,537 x 2,880: 84 us, otherwise 91; of 32,003 x 2,048, which it holds: 37 and 30), those of large tiles always, as heads of
// more than 131,072 rows seldom fit (below a d_model of 1,024), those of the smallest heads never.
template <typename F>
auto with_few_tile(uint32_t rows, uint32_t vocab, uint32_t d, F&& f) {
    const bool streamed = 2ull * vocab * d > kMemoryCache;
    if (rows <= kFewRows) {
        if (vocab > 131072) return f(TileFew{});
        return streamed ? f(TileFewest<true>{}) : f(TileFewest<false>{});
    }
    if (vocab <= 40960) return f(TileMidSmall{});
    return streamed ? f(TileMid<true>{}) : f(TileMid<false>{});
}
// Vocabulary rows of a tile of the forward pass.
uint32_t vocab_tile(uint32_t rows, uint32_t vocab, uint32_t d) {
    return rows > kMidRows ? kVocabTile : with_few_tile(rows, vocab, d, [](auto tile) { return decltype(tile)::kA; });
}

// `g`: forward of so few rows that the tiles gather by themselves.
template <bool GRAD>
int launch_few(const LogitArgs& a, uint32_t rows, const GatherArgs* g, hipStream_t s) {
    return with_few_tile(rows, a.vocab, a.d, [&](auto tile) -> int {
        using Tile = decltype(tile);
        const uint32_t blocks = blocks_for(div_up(a.here, Tile::kA));
        if constexpr (!GRAD && Tile::kB <= kFewRows) loss_few_forward_kernel<Tile><<<blocks, kProductThreads, 0, s>>>(a, *g);
        else loss_few_kernel<Tile, GRAD><<<blocks, kProductThreads, 0, s>>>(a);
        TWD_HIP(hipGetLastError());
        return TWD_OK;
    });
}

template <bool GRAD>
int launch_logits(const LogitArgs& a, uint32_t rows, hipStream_t s) {
    uint32_t most = 0, cut = 0;  // blocks, for any number of rows that count
    for (uint32_t n = 64; n < rows + 64; n += 64) {
        const LogitTiles t = logit_tiles(n < rows ? n : rows, div_up(a.here, kVocabTile));
        most = t.grid.tiles() > most ? t.grid.tiles() : most;
        cut = t.cut > cut ? t.cut : cut;
    }
    loss_logits_kernel<GRAD><<<blocks_for(most), kProductThreads, 0, s>>>(a);
    TWD_HIP(hipGetLastError());
    if (cut == 0) return TWD_OK;
    loss_stripes_kernel<GRAD><<<blocks_for(4 * cut), kProductThreads, 0, s>>>(a);
    TWD_HIP(hipGetLastError());
    return TWD_OK;
}

template <typename Tile, typename Out, bool BY_COUNT>
int launch_grad(const GradArgs& a, uint32_t most_tiles, hipStream_t s) {
    const uint64_t nb = div_up(a.cols, Tile::kB), tiles = BY_COUNT ? nb * div_up(a.rows, Tile::kA) : most_tiles;
    loss_grad_kernel<Tile, Out, BY_COUNT><<<blocks_for(static_cast<uint32_t>(tiles)), kProductThreads, 0, s>>>(a);
    TWD_HIP(hipGetLastError());
    return TWD_OK;
}

int launch_gather(const twd_headloss* l, GatherArgs a, hipStream_t s) {
    a.r = l->r, a.vocab = l->vocab, a.pieces = l->d / 8;
    a.each = div_up(a.rows, 4096);  // a block counts all targets before its own: not too many of them
    loss_gather_kernel<<<div_up(a.rows, a.each), 256, 0, s>>>(a);
    TWD_HIP(hipGetLastError());
    return TWD_OK;
}

int forward(const twd_headloss* l, const GatherArgs& g, const Operand& weight, hipStream_t s) {
    LogitArgs a{};
    a.r = l->r, a.weight = weight, a.hidden = Operand{l->r.h, l->d, g.rows, l->d};
    a.d = l->d, a.vocab = a.here = l->vocab, a.softcap = soft_cap(l->softcap), a.part = l->part, a.part_stride = g.rows;
    int rc;
    if (g.rows <= kFewRows) {
        a.hidden = Operand{g.hidden, g.rows > 1 ? g.stride : l->d, g.rows, l->d, nullptr, g.rows};
        GatherArgs own = g;
        own.vocab = l->vocab;
        rc = launch_few<false>(a, g.rows, &own, s);
    } else {
        if ((rc = launch_gather(l, g, s))) return rc;
        rc = g.rows <= kMidRows ? launch_few<false>(a, g.rows, nullptr, s) : launch_logits<false>(a, g.rows, s);
    }
    if (rc) return rc;
    loss_join_kernel<<<div_up(g.rows, kJoinRows), kJoinThreads, 0, s>>>(
        JoinArgs{l->r, l->part, div_up(l->vocab, vocab_tile(g.rows, l->vocab, l->d)), g.rows, g.losses, g.lse_out});
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
    const uint32_t piece = piece_of(g.rows, l->vocab);
    int rc = launch_gather(l, g, s);
    if (rc) return rc;
    const bool few = g.rows <= kMidRows;
    static_assert(TileHiddenFew::kA == kMidRows && TileHiddenFew::kB == 256 && TileHidden::kA == 256 && TileHidden::kB == 256, "as hidden_parts takes them");
    uint32_t most_tiles = 0;  // of d_hidden's product, for any number of rows that count
    for (uint32_t n = 1; n <= div_up(g.rows, 256); ++n) {
        const uint32_t tiles = n * div_up(l->d, 256) * hidden_parts(n * 256, l->d, piece, few);
        most_tiles = tiles > most_tiles ? tiles : most_tiles;
    }
    for (uint32_t v0 = 0; v0 < l->vocab; v0 += piece) {
        const uint32_t here = l->vocab - v0 < piece ? l->vocab - v0 : piece;
        const Operand h{l->r.h, l->d, g.rows, l->d}, w{weight.p + v0 * weight.stride, weight.stride, here, l->d};
        LogitArgs a{};
        a.r = l->r, a.weight = weight, a.hidden = h;
        a.d = l->d, a.vocab = l->vocab, a.v0 = v0, a.here = here, a.softcap = soft_cap(l->softcap), a.dz = l->dz, a.dz_stride = piece;
        if ((rc = few ? launch_few<true>(a, g.rows, nullptr, s) : launch_logits<true>(a, g.rows, s))) return rc;
        if (o.d_weight) {
            GradArgs b{};
            b.count = l->r.count, b.a = Operand{l->dz, piece, g.rows, piece}, b.b = h;
            b.rows = here, b.cols = l->d, b.stride = o.d_weight_stride, b.add = o.add;
            b.out = static_cast<char*>(o.d_weight) + v0 * o.d_weight_stride * (o.type == TWD_F32 ? 4 : 2);
            if (few) rc = o.type == TWD_F32 ? launch_grad<TileWeightFew, float, true>(b, 0, s) : launch_grad<TileWeightFew, uint16_t, true>(b, 0, s);
            else rc = o.type == TWD_F32 ? launch_grad<TileWeight, float, true>(b, 0, s) : launch_grad<TileWeight, uint16_t, true>(b, 0, s);
            if (rc) return rc;
        }
        if (o.d_hidden) {
            GradArgs b{};
            b.count = l->r.count, b.a = Operand{l->dz, piece, g.rows, here}, b.b = w;
            b.k = here, b.piece = piece, b.cols = l->d;
            b.out = l->dh, b.stride = l->d, b.add = v0 > 0, b.few = few;
            rc = few ? launch_grad<TileHiddenFew, float, false>(b, most_tiles, s) : launch_grad<TileHidden, float, false>(b, most_tiles, s);
            if (rc) return rc;
        }
    }
    if (!o.d_hidden) return TWD_OK;
    loss_spread_kernel<<<dim3(g.rows, div_up(l->d, 2048)), 256, 0, s>>>(
        SpreadArgs{l->r, g.targets, l->dh, piece, l->vocab, l->d, o.d_hidden, o.d_hidden_stride, few});
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

Operand weight_of(const twd_headloss* l, const uint16_t* p, uint64_t stride) {  // a single row's stride plays no part
    return Operand{p, l->vocab > 1 ? stride : l->d, l->vocab, l->d};
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
    if (static_cast<uint64_t>(max_rows) * vocab > kLossMaxLogits) return fail(TWD_E_INVALID, "max_rows x vocab must be at most 2^38");
    if (d_model == 0 || d_model % 32 != 0 || d_model > (1u << 20))
        return fail(TWD_E_INVALID, "d_model must be a positive multiple of 32, at most 2^20");
    if (softcap != 0.0f && !(softcap >= kMinSoftCap && softcap <= kMaxSoftCap))
        return fail(TWD_E_INVALID, "softcap must be 0 (none) or in 1e-30..1e30");
    int dev = 0;
    TWD_HIP(hipGetDevice(&dev));
    twd_headloss* l = new (std::nothrow) twd_headloss{};
    if (!l) return fail(TWD_E_INVALID, "out of host memory");
    l->max_rows = max_rows, l->vocab = vocab, l->d = d_model, l->softcap = softcap, l->backward = backward != 0, l->device = dev;
    uint64_t dz = 0, part = 0;  // the most that any number of rows, and of those that count, takes
    for (uint32_t rows = 1; l->backward && rows <= max_rows; ++rows) {
        const uint64_t n = static_cast<uint64_t>(rows) * piece_of(rows, vocab);
        uint32_t parts = hidden_parts(rows, d_model, most_of_piece(rows), false);
        if (rows <= kMidRows) {
            const uint32_t more = hidden_parts(rows, d_model, most_of_piece(rows), true);
            parts = more > parts ? more : parts;
        }
        const uint64_t m = static_cast<uint64_t>(rows) * d_model * parts;
        dz = n > dz ? n : dz, part = m > part ? m : part;
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
        take(l->r.at, max_rows);
        take(l->r.target, max_rows);
        take(l->r.grad, max_rows);
        take(l->r.lse, max_rows);
        take(l->r.hit, max_rows);
        take(l->r.h, static_cast<uint64_t>(max_rows) * d_model);
        uint64_t parts = 0;
        for (const uint32_t rows : {kFewRows, kMidRows, max_rows}) {
            const uint32_t n = rows < max_rows ? rows : max_rows;
            const uint64_t here = static_cast<uint64_t>(div_up(vocab, vocab_tile(n, vocab, d_model))) * n;
            parts = here > parts ? here : parts;
        }
        take(l->part, parts);
        if (!l->backward) return;
        take(l->dz, dz);
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
    rc = forward(l, g, weight_of(l, weight_bf16, weight_stride), s);
    const int rc2 = order_after(l->order, s);
    return rc ? rc : rc2;
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
    rc = backward(l, g, weight_of(l, weight_bf16, weight_stride), o, s);
    const int rc2 = order_after(l->order, s);
    return rc ? rc : rc2;
}

}  // extern "C"
