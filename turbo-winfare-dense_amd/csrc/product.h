// A tile of the product of two bf16 matrices along their rows, C[a][b] = sum_k A[a][k] B[b][k], summed in fp32: the
// core of the head's loss and its gradients. The caller brings what happens to the tile's sums.
//
// Four waves share a tile of kA x kB; a wave holds TA x TB squares of 32 x 32. Both operands go through LDS in stages of
// 32 columns, loaded there without registers, three stages ahead into four buffers; a stage's barrier stands between
// its two steps of 16 columns, so that the second step's products cover the reads of the next stage's first
// fragments. In LDS a row's four pieces of 16 bytes change places with its number, so that eight rows' reads of one
// piece meet different banks.
#pragma once

#include "twd_internal.h"
#include "vocab_core.h"

namespace twd {

namespace {

// Operands: rows at a multiple of 16 bytes, strides in elements, multiples of 8 and at most kMaxProductStride (a tile's rows
// lie within 32-bit offsets).
struct Operand {
    const uint16_t* p;
    uint64_t stride;
    uint32_t rows;  // rows past the last read the last
};
constexpr uint64_t kMaxProductStride = 1ull << 22;

constexpr uint32_t kStageK = 32;
constexpr uint32_t kProductThreads = 256;

template <int TA, int TB, int GA, int GB>
struct ProductTile {
    static_assert(GA * GB == 4, "four waves");
    static constexpr uint32_t kA = 32 * TA * GA, kB = 32 * TB * GB;
    static constexpr uint32_t kStage = (kA + kB) * 4;                    // 16-byte pieces
    static constexpr uint32_t kLoadsA = kA / 64, kLoadsB = kB / 64;      // of 16 rows, each wave's
    static constexpr uint32_t kLoads = kLoadsA + kLoadsB;
    static constexpr uint32_t kAhead = 2 * kLoads;                       // a wave's loads of two stages

    static __host__ __device__ constexpr uint32_t padded(uint32_t k) { return (k + 127) / 128 * 128; }

    // sum(ta, tb) is the square of A rows a0 + 32 (TA wa + ta) .. and B rows b0 + 32 (TB wb + tb) ..; lane l's element i is
    // the one of B row l % 32 and A row 8 (i / 4) + 4 (l / 32) + i % 4, or with SWAP the other way round. k: a positive
    // multiple of 32, taken up to a multiple of 128: there B's rows hold zeros, and A's are read from their start again, so
    // that nothing but A's own row meets them.
    template <bool SWAP>
    static __device__ __forceinline__ void sums(u32x4_t* s0, u32x4_t* s1, u32x4_t* s2, u32x4_t* s3, const Operand& A,
                                                const Operand& B, uint32_t a0, uint32_t b0, uint32_t k,
                                                f32x16_t (&acc)[TA][TB]) {
        const uint32_t lane = threadIdx.x % 64;
        const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
        const uint32_t wa = wave / GB, wb = wave % GB;
        const uint32_t rows_a = min(A.rows - a0, kA), rows_b = min(B.rows - b0, kB);
        const uint32_t bytes_a = static_cast<uint32_t>(2 * A.stride), bytes_b = static_cast<uint32_t>(2 * B.stride);
        const auto ra = make_rsrc(A.p + a0 * A.stride, (rows_a - 1) * bytes_a + 2 * k);
        const auto rb = make_rsrc(B.p + b0 * B.stride, (rows_b - 1) * bytes_b + 2 * padded(k));
        // lane l of a load brings the piece that belongs to place l % 4 of row l / 4
        const uint32_t row = lane / 4, piece = (lane % 4) ^ (lane / 8 % 4);
        uint32_t off_a[kLoadsA], off_b[kLoadsB];
#pragma unroll
        for (uint32_t j = 0; j < kLoadsA; ++j) off_a[j] = min(16 * (wave * kLoadsA + j) + row, rows_a - 1) * bytes_a + 16 * piece;
#pragma unroll
        for (uint32_t j = 0; j < kLoadsB; ++j) off_b[j] = min(16 * (wave * kLoadsB + j) + row, rows_b - 1) * bytes_b + 16 * piece;
        const uint32_t stages = padded(k) / kStageK;
        // past the last stage it comes again, into a buffer that is not read any more
        auto load = [&](uint32_t stage, u32x4_t* to, uint32_t first, uint32_t last) {
            const uint32_t at = __builtin_amdgcn_readfirstlane(min(stage, stages - 1) * (2 * kStageK));
            const uint32_t at_a = at + 16 * piece < 2 * k ? at : 0u;
#pragma unroll
            for (uint32_t j = first; j < last; ++j) {
                if (j < kLoadsA)
                    __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lds_void*)(to + (wave * kLoadsA + j) * 64), 16,
                                                             static_cast<int>(off_a[j] + at_a), 0, 0, 0);
                else
                    __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (lds_void*)(to + kA * 4 + (wave * kLoadsB + j - kLoadsA) * 64), 16,
                                                             static_cast<int>(off_b[j - kLoadsA]), static_cast<int>(at), 0, 0);
            }
        };
        const uint32_t r = lane % 32, h = lane / 32, turn = r / 2 % 4;
        const uint32_t at_a = (32 * TA * wa + r) * 4, at_b = kA * 4 + (32 * TB * wb + r) * 4;
        bf16x8_t fa[2][TA], fb[2][TB];
        auto read_a = [&](const u32x4_t* from, int step, int t) {
            fa[step][t] = __builtin_bit_cast(bf16x8_t, from[at_a + 128 * t + ((2 * step + h) ^ turn)]);
        };
        auto read_b = [&](const u32x4_t* from, int step, int t) {
            fb[step][t] = __builtin_bit_cast(bf16x8_t, from[at_b + 128 * t + ((2 * step + h) ^ turn)]);
        };
        auto product = [&](int step, int ta, int tb) {
            acc[ta][tb] = SWAP ? __builtin_amdgcn_mfma_f32_32x32x16_bf16(fb[step][tb], fa[step][ta], acc[ta][tb], 0, 0, 0)
                               : __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[step][ta], fb[step][tb], acc[ta][tb], 0, 0, 0);
        };
        // One step's products, with the next step's reads (from, to_step) spread among them.
        auto step = [&](int now, const u32x4_t* from, int next, auto more) {
            constexpr int kProducts = TA * TB, kReads = TA + TB;
#pragma unroll
            for (int i = 0; i < kProducts; ++i) {
#pragma unroll
                for (int j = i * kReads / kProducts; j < (i + 1) * kReads / kProducts; ++j) {
                    if (j < TA) read_a(from, next, j);
                    else read_b(from, next, j - TA);
                }
                more(i);
                product(now, i / TB, i % TB);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        auto nothing = [](int) {};
        auto stage = [&](uint32_t i, u32x4_t* now, const u32x4_t* next) {
            step(0, now, 1, nothing);
            // this stage is read, and the next has arrived: of the loads only two stages' may still be on their way
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_waitcnt(0x0070 | (kAhead & 15) | (kAhead >> 4) << 14);
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_sched_barrier(0);
            constexpr int kProducts = TA * TB;
            step(1, next, 0, [&](int n) { load(i + 4, now, n * kLoads / kProducts, (n + 1) * kLoads / kProducts); });
        };
        load(0, s0, 0, kLoads);
        load(1, s1, 0, kLoads);
        load(2, s2, 0, kLoads);
        load(3, s3, 0, kLoads);
#pragma unroll
        for (int i = 0; i < TA; ++i)
#pragma unroll
            for (int j = 0; j < TB; ++j) acc[i][j] = f32x16_t{};
        __builtin_amdgcn_s_waitcnt(0x0F70);  // once a tile: everything (the first stage would do)
        __syncthreads();
#pragma unroll
        for (int t = 0; t < TA; ++t) read_a(s0, 0, t);
#pragma unroll
        for (int t = 0; t < TB; ++t) read_b(s0, 0, t);
        for (uint32_t i = 0; i < stages; i += 4) {
            stage(i, s0, s1);
            stage(i + 1, s1, s2);
            stage(i + 2, s2, s3);
            stage(i + 3, s3, s0);
        }
        __builtin_amdgcn_s_waitcnt(kVmcnt0);  // the buffers may be used for something else
        __syncthreads();
    }
};

// Which tile a block takes: blocks go to the XCDs in turn, and each XCD takes a contiguous stretch of the tiles, ordered
// so that a few rows of tiles along A meet up to eight along B at a time: what an XCD's blocks read at once stays in its
// L2.
struct TileGrid {
    uint32_t na, nb, parts;  // tiles along A and B, and parts of the sum
    __host__ __device__ uint32_t tiles() const { return na * nb * parts; }
    __host__ __device__ uint32_t blocks() const { return (tiles() + 7) / 8 * 8; }
};
struct TileAt {
    uint32_t a, b, part;
};
__device__ __forceinline__ bool tile_of_block(const TileGrid& g, TileAt* at) {
    const uint32_t id = blockIdx.x % 8 * (g.blocks() / 8) + blockIdx.x / 8;
    if (id >= g.tiles()) return false;
    const uint32_t each = g.na * g.nb, in = id % each;
    at->part = id / each;
    const uint32_t group = in / (8 * g.na), left = in - group * 8 * g.na, width = min(8u, g.nb - 8 * group);
    at->a = left / width, at->b = 8 * group + left % width;
    return true;
}

}  // namespace

}  // namespace twd
