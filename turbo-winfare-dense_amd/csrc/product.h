// A tile of the product of two bf16 matrices, C[a][b] = sum_k A(a, k) B(b, k), summed in fp32: the core of the head's loss
// and its gradients. The caller brings what happens to the tile's sums.
//
// Four waves share a tile of kA x kB; a wave holds TA x TB squares of 32 x 32. Both operands go through LDS in stages of K of
// k, loaded there without registers, into BUFS buffers in turn; a stage's barrier stands before its last step of 16, so that
// this step's products cover the reads of the next stage's first fragments. What lies outside an operand is read as zero by
// the buffer loads' range check.
//
// An operand lies in memory by rows of k ([a][k]), or turned ([k][a]). By rows, its stage in LDS is [a][K / 8 pieces of 16
// bytes], a row's pieces exchanged by its number, so that sixteen rows' reads of one piece meet different banks (of 64).
// Turned, it is [k][a], a row's pieces of 32 bytes exchanged by k: four rows' reads of two pieces meet different banks, and
// the reads turn 4 (k) x 16 (a) elements over sixteen lanes.
#pragma once

#include "tiles.h"
#include "twd_internal.h"
#include "vocab_core.h"

namespace twd {

namespace {

// Starts at a multiple of 16 bytes; the stride between rows in elements, a multiple of 8 and at most kMaxProductStride (what
// a stage reads lies within 32-bit offsets).
struct Operand {
    const uint16_t* p;
    uint64_t stride;
    uint32_t rows;  // [a][k]: a; [k][a]: k
    uint32_t cols;  // [a][k]: k; [k][a]: a; a multiple of 8, as a load of 16 bytes lies inside the range or out of it
    // [a][k]: where given, row a is row places[a] of `within`, which are at most 64
    const uint32_t* places = nullptr;
    uint32_t within = 0;
};
constexpr uint64_t kMaxProductStride = 1ull << 22;

// Which tile of a grid a block takes: blocks go to the XCDs in turn, and each XCD takes a contiguous stretch of the tiles,
// ordered so that a few rows of tiles along A meet up to eight along B at a time: what an XCD's blocks read at once stays in
// its L2.
struct TileAt {
    uint32_t a, b, part;
    uint32_t share, who;  // the blocks that read the same rows of A at once, and which of them this is
};
__host__ __device__ inline uint32_t blocks_for(uint32_t tiles) { return (tiles + 7) / 8 * 8; }
// This block's number among `tiles`, or one past them.
__device__ __forceinline__ uint32_t stretched(uint32_t tiles) {
    const uint32_t each = (tiles + 7) / 8, in = blockIdx.x / 8;
    return in < each ? blockIdx.x % 8 * each + in : tiles;
}
__device__ __forceinline__ TileAt tile_at(const TileGrid& g, uint32_t id) {
    const uint32_t each = g.na * g.nb, in = id % each;
    const uint32_t group = in / (8 * g.na), left = in - group * 8 * g.na, width = min(8u, g.nb - 8 * group);
    return TileAt{left / width, 8 * group + left % width, id / each, width, left % width};
}

constexpr uint32_t kProductThreads = 256;

typedef short i16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i16x4_t lds_i16x4_t;

// One operand's part of a stage: ROWS of a, K of k, T fragments to a wave.
template <uint32_t ROWS, uint32_t K, int T, bool TURNED, bool STREAMED = false>
struct ProductSide {
    static constexpr uint32_t kLoads = ROWS * K / 2048;                 // of 1 KB, each wave's
    static constexpr uint32_t kLines = 512 / (TURNED ? ROWS : K);       // rows in memory of a load
    static constexpr uint32_t kPerLine = 64 / kLines;                   // lanes, of 16 bytes
    Operand x;
    uint32_t first;   // of a
    uint32_t line;    // bytes between rows in memory
    uint32_t off[kLoads];
    uint32_t column;  // by rows: this lane's byte in a stage, or with bit 6 the other way, in every second load
    __amdgpu_buffer_rsrc_t rsrc;
    uint32_t wave, at;  // at: where this lane's fragments lie in the stage (by rows: pieces; turned: bytes)

    __device__ __forceinline__ ProductSide(const Operand& o, uint32_t a0, uint32_t wave_, uint32_t share) : x(o), first(a0), wave(wave_) {
        const uint32_t lane = threadIdx.x % 64, in = lane / kPerLine, piece = lane % kPerLine;
        line = static_cast<uint32_t>(2 * x.stride);
        if constexpr (TURNED) {
#pragma unroll
            for (uint32_t j = 0; j < kLoads; ++j) {
                const uint32_t row = kLines * (wave * kLoads + j) + in;
                off[j] = row * line + 32 * ((piece / 2) ^ 2 * (row % 4)) + 16 * (piece % 2);
            }
            const uint32_t g = lane / 16, j = lane % 16;
            at = (8 * (g / 2) + j / 4) * (2 * ROWS) + 32 * ((2 * T * share + g % 2) ^ 2 * (j / 4)) + 8 * (j % 4);
        } else {
            // rows four apart (two, of 64 columns) read the same banks: those exchange their pieces
            column = 16 * (piece ^ (K == 64 ? lane / 16 : lane / 16 % 4));
#pragma unroll
            for (uint32_t j = 0; j < kLoads; ++j) off[j] = place_of(kLines * (wave * kLoads + j) + in) + column_of(j);
            const uint32_t here = x.places ? x.within : min(x.rows - first, ROWS);
            rsrc = make_rsrc(x.p + first * x.stride, (here - 1) * line + 2 * x.cols);
            at = (32 * T * share + lane % 32) * (K / 8);
        }
    }
    __device__ __forceinline__ uint32_t place_of(uint32_t row) const {
        static_assert(kMaxProductStride * 2 * 64 <= 1u << 29, "64 rows lie below a place that is out of every range");
        return x.places ? (row < x.rows ? x.places[row] * line : 0x40000000u) : row * line;
    }
    __device__ __forceinline__ uint32_t column_of(uint32_t j) const { return K == 64 && j % 2 ? column ^ 64 : column; }
    // Loads from .. last - 1 of a stage into its buffer.
    __device__ __forceinline__ void load(uint32_t stage, u32x4_t* to, uint32_t from, uint32_t last) {
        if (from >= last) return;
        if constexpr (TURNED) {
            const uint32_t k = stage * K, left = k < x.rows ? min(x.rows - k, K) : 0;
            const auto r = make_rsrc(x.p + k * x.stride + first, left ? (left - 1) * line + 2 * (x.cols - first) : 0);
#pragma unroll
            for (uint32_t j = from; j < last; ++j)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)(to + (wave * kLoads + j) * 64), 16, static_cast<int>(off[j]), 0, 0, STREAMED ? kStreamed : 0);
        } else {
            const uint32_t byte = stage * (2 * K);
#pragma unroll
            for (uint32_t j = from; j < last; ++j) {
                const uint32_t go = byte + column_of(j) < 2 * x.cols ? byte : 0x80000000u;  // beyond any range
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void*)(to + (wave * kLoads + j) * 64), 16,
                                                         static_cast<int>(off[j] + go), 0, 0, STREAMED ? kStreamed : 0);
            }
        }
    }
    // Brings the lines of a stage by rows to the L2, each of `share` blocks that read them its part: one word of a line into
    // LDS, where nobody reads it.
    __device__ __forceinline__ void touch(uint32_t stage, uint32_t* sink, uint32_t share, uint32_t who) {
        static_assert(!TURNED && ROWS == kProductThreads && K == 64, "a line to a thread");
        const uint32_t byte = stage * (2 * K), id = threadIdx.x;
        const uint32_t at_byte = id % share == who && byte < 2 * x.cols ? id * line + byte : 0x80000000u;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void*)(sink + 64 * wave), 4, static_cast<int>(at_byte), 0, 0, 0);
    }
    __device__ __forceinline__ bf16x8_t read(const u32x4_t* from, int step, int t) const {
        if constexpr (TURNED) {
            // fragment t's two pieces of 32 bytes: t's bits change the piece number's alone above the lowest, which g % 2 sets
            const char* p = reinterpret_cast<const char*>(from) + (at ^ (64 * t)) + 16 * step * (2 * ROWS);
            const i16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t*)p);
            const i16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t*)(p + 4 * (2 * ROWS)));
            return __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            const uint32_t lane = threadIdx.x % 64;
            const uint32_t turn = K == 64 ? lane / 2 % 8 : lane / 4 % 4;
            return __builtin_bit_cast(bf16x8_t, from[at + 4 * K * t + ((2 * step + lane / 32) ^ turn)]);
        }
    }
};

// Where several blocks read the same rows of A from memory at once, TOUCH brings its lines to the L2 three stages ahead: the
// loads into LDS, of which one stage is on its way, then seldom wait for memory (2,048 x 65,536 x 5,376: 1,285 TFLOP/s without,
// 1,329 with it; all zeros, where the clock is not held by the power, 1,527 and 1,857; of B's lines too: 1,183). Where a block
// alone reads its part of an operand, STREAMED lets it pass the L2, which keeps the other (17 rows of 262,144 x 5,376: 499 us without, 440).
template <int TA, int TB, int GA, int GB, uint32_t K, uint32_t BUFS, bool TURNED_A, bool TURNED_B, bool TOUCH = false, bool STREAMED_A = false, bool STREAMED_B = false>
struct ProductTile {
    static_assert(GA * GB == 4, "four waves");
    static_assert(BUFS >= 2 && BUFS <= 4, "buffers");
    static_assert(K == 32 || K == 64, "a stage");
    static constexpr int kTA = TA, kTB = TB, kGA = GA, kGB = GB;
    static constexpr uint32_t kA = 32 * TA * GA, kB = 32 * TB * GB;
    static constexpr uint32_t kPieces = (kA + kB) * K / 8, kPiecesA = kA * K / 8;  // of 16 bytes in a buffer
    static constexpr uint32_t kPieces2 = BUFS > 2 ? kPieces : 1, kPieces3 = BUFS > 3 ? kPieces : 1;
    static constexpr uint32_t kBytes = BUFS * kPieces * 16;
    static constexpr uint32_t kSink = TOUCH ? kProductThreads : 1;
    static constexpr uint32_t kLoadsA = kA * K / 2048, kLoads = kPieces / 256;
    static constexpr uint32_t kAhead = (BUFS - 2) * kLoads + (TOUCH ? BUFS - 1 : 0);  // a wave's loads that need not have arrived at a stage's end

    // sum(ta, tb) is the square of A's kA at.a + 32 (TA wa + ta) .. and B's kB at.b + 32 (TB wb + tb) ..; lane l's element i is
    // the one of B's l % 32 and A's 8 (i / 4) + 4 (l / 32) + i % 4, or with SWAP the other way round. s2 and s3 are the third and
    // fourth buffer, if any; sink: kSink words.
    template <bool SWAP>
    static __device__ __forceinline__ void sums(u32x4_t* s0, u32x4_t* s1, u32x4_t* s2, u32x4_t* s3, uint32_t* sink,
                                                const Operand& A, const Operand& B, const TileAt& at, uint32_t k,
                                                f32x16_t (&acc)[TA][TB]) {
        const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
        ProductSide<kA, K, TA, TURNED_A, STREAMED_A> x(A, at.a * kA, wave, wave / GB);
        ProductSide<kB, K, TB, TURNED_B, STREAMED_B> y(B, at.b * kB, wave, wave % GB);
        // whole turns of the buffers; past the operands' ends stages are zero
        const uint32_t turns = (k + BUFS * K - 1) / (BUFS * K);
        auto load = [&](uint32_t stage, u32x4_t* to, uint32_t first, uint32_t last) {
            x.load(stage, to, min(first, kLoadsA), min(last, kLoadsA));
            y.load(stage, to + kPiecesA, max(first, kLoadsA) - kLoadsA, max(last, kLoadsA) - kLoadsA);
        };
        bf16x8_t fa[2][TA], fb[2][TB];
        constexpr int kProducts = TA * TB, kReads = TA + TB;
        // One step's products, with the next step's reads and some loads spread among them.
        auto step = [&](int now, const u32x4_t* from, int next, auto more) {
#pragma unroll
            for (int i = 0; i < kProducts; ++i) {
#pragma unroll
                for (int j = i * kReads / kProducts; j < (i + 1) * kReads / kProducts; ++j) {
                    if (j < TA) fa[next % 2][j] = x.read(from, next, j);
                    else fb[next % 2][j - TA] = y.read(from + kPiecesA, next, j - TA);
                }
                more(i);
                f32x16_t& sum = acc[i / TB][i % TB];
                const bf16x8_t p = fa[now % 2][i / TB], q = fb[now % 2][i % TB];
                sum = SWAP ? __builtin_amdgcn_mfma_f32_32x32x16_bf16(q, p, sum, 0, 0, 0)
                           : __builtin_amdgcn_mfma_f32_32x32x16_bf16(p, q, sum, 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        // A stage's loads are spread over the steps: in one burst they fill the queue to memory, and the wave's products wait
        // behind them (the same product: 1,166 and 1,285 TFLOP/s).
        constexpr uint32_t kSteps = K / 16, kSpread = kSteps > 2 ? kSteps - 1 : kSteps;
        auto part = [&](uint32_t stage, u32x4_t* to, uint32_t p, int n) {
            if (p >= kSpread) return;
            const uint32_t lo = kLoads * p / kSpread, hi = kLoads * (p + 1) / kSpread;
            load(stage, to, lo + (hi - lo) * n / kProducts, lo + (hi - lo) * (n + 1) / kProducts);
        };
        auto stage = [&](uint32_t i, u32x4_t* before, u32x4_t* now, const u32x4_t* next) {
#pragma unroll
            for (uint32_t s = 0; s < kSteps - 1; ++s)
                step(s, now, s + 1, [&](int n) {
                    part(i - 1 + BUFS, before, s + 1, n);
                    if constexpr (TOUCH) {
                        if (s == kSteps - 2 && n == kProducts - 1) x.touch(i + BUFS + 1, sink, at.share, at.who);
                    }
                });
            // this stage has been read, and the next has arrived
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_waitcnt(0x0070 | (kAhead & 15) | (kAhead >> 4) << 14);
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_sched_barrier(0);
            step(kSteps - 1, next, 0, [&](int n) { part(i + BUFS, now, 0, n); });
        };
        u32x4_t* const last = BUFS == 2 ? s1 : BUFS == 3 ? s2 : s3;
        load(0, s0, 0, kLoads);
        if constexpr (BUFS > 2) load(1, s1, 0, kLoads);
        if constexpr (BUFS > 3) load(2, s2, 0, kLoads);
        load(BUFS - 1, last, 0, kLoads / kSpread);
#pragma unroll
        for (int i = 0; i < TA; ++i)
#pragma unroll
            for (int j = 0; j < TB; ++j) acc[i][j] = f32x16_t{};
        // all of them: kAhead counts lines of BUFS - 1 stages before, which the first stages do not have
        __builtin_amdgcn_s_waitcnt(kVmcnt0);
        __syncthreads();
#pragma unroll
        for (int t = 0; t < TA; ++t) fa[0][t] = x.read(s0, 0, t);
#pragma unroll
        for (int t = 0; t < TB; ++t) fb[0][t] = y.read(s0 + kPiecesA, 0, t);
        for (uint32_t i = 0; i < turns * BUFS; i += BUFS) {
            stage(i, last, s0, s1);
            stage(i + 1, s0, s1, BUFS > 2 ? s2 : s0);
            if constexpr (BUFS > 2) stage(i + 2, s1, s2, BUFS > 3 ? s3 : s0);
            if constexpr (BUFS > 3) stage(i + 3, s2, s3, s0);
        }
        __builtin_amdgcn_s_waitcnt(kVmcnt0);  // the buffers may be used for something else
        __syncthreads();
    }
};

// Squares side by side, as a lane holds them (its row l % 32; columns 8 (i / 4) + 4 (l / 32) + i % 4 of each), change places
// in the wave's own part of LDS, so that whole lines are stored: squares(n) gives a lane's sixteen of square n, put(row,
// col, 16 bytes) takes them in rows. `mine`: 32 rows of 32 N columns.
template <int N, typename Out, typename Squares, typename Put>
__device__ __forceinline__ void store_rows(u32x4_t* mine, Squares squares, Put put) {
    constexpr uint32_t kEach = 16 / sizeof(Out), kRow = 32 * N / kEach, kTurn = kRow < 16 ? kRow : 16;
    const uint32_t lane = threadIdx.x % 64, r = lane % 32, h = lane / 32;
    auto place = [&](uint32_t row, uint32_t piece) { return row * kRow + (piece ^ row % kTurn); };
    each<N>([&](auto n) {
        const auto square = squares(n);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x4_t v = {square[4 * i], square[4 * i + 1], square[4 * i + 2], square[4 * i + 3]};
            if constexpr (sizeof(Out) == 4)
                mine[place(r, 8 * n + 2 * i + h)] = __builtin_bit_cast(u32x4_t, v);
            else
                reinterpret_cast<u32x2_t*>(mine + place(r, 4 * n + i))[h] = u32x2_t{bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3])};
        }
    });
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (uint32_t i = 0; i < 32 * kRow / 64; ++i) {
        const uint32_t row = i * (64 / kRow) + lane / kRow, piece = lane % kRow;
        put(row, piece * kEach, mine[place(row, piece)]);
    }
    __builtin_amdgcn_wave_barrier();
}

}  // namespace

}  // namespace twd
