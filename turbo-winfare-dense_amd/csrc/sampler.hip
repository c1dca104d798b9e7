// Sampling with temperature, top-k, top-p and min-p from given random numbers.
//
// Per row, with l the logits, M their largest and T the temperature: the weights are
// w_i = exp((l_i - M) / T) and the order is by falling logit, equal logits by rising index. Every limit
// keeps a prefix of that order: top-k its first k, top-p the shortest prefix whose weights reach p of the
// top-k's sum, min-p the weights of at least min_p of the largest. The shortest prefix is kept (never less
// than one id), and the draw u takes the first kept id, by index, at which the running sum of kept weights
// exceeds u of their sum.
//
// Arithmetic. Sums decide, so they may not depend on the order in which threads add: weights are
// fixed-point numbers and sums are integers. With z = l log2(e) / T (formed in two doubles), a weight is
// 2^floor(z) times the fraction's power of two, rounded to 37 bits (2^-37 relative). Sums are held in 128
// bits, in units of 2^-77 of the largest weight's octave. Weights from 31 octaves under that one on lose their
// bits below 2^-67 of it, and what lies 67 or more octaves below it weighs nothing (so less than 2^-66 of the largest): 524,288
// such weights are at most 2^-47 of a row's sum, where a draw's own steps are 2^-24. Every decision is then an exact comparison of integers, and
// equal logits have equal weights.
#include <hip/hip_runtime.h>

#include <cmath>
#include <new>
#include <type_traits>

#include "twd_internal.h"
#include "twd_sampler.h"

namespace twd {

namespace {

typedef unsigned __int128 u128;

constexpr int kSumShift = 40;    // sums: the largest octave's weights shifted left by this

struct SampleParams {
    const float* temperature;  // null: 1
    const int32_t* top_k;      // null or <= 0: no limit
    const float* top_p;        // null or >= 1: no limit
    const float* min_p;        // null or <= 0: no limit
    const float* uniform;
};

struct SampleOut {
    uint32_t* tokens;
    float* logprobs;  // may be null
    int32_t* kept;    // may be null
};

// log2(e) / T in two doubles.
struct Scale {
    double hi, lo;
};
__device__ __forceinline__ Scale scale_of(float t) {
    const double kHi = 1.4426950408889634, kLo = 2.0355273740931033e-17;
    const double td = t;
    Scale s;
    s.hi = kHi / td;
    s.lo = t == INFINITY ? 0.0 : (fma(-s.hi, td, kHi) + kLo) / td;  // an infinite T: every weight alike
    return s;
}

// Where a weight lies: floor(8 z), the eighths of its octave counted from 2^0 up. It rises with l.
__device__ __forceinline__ double place_of(float l, const Scale& c) {
    return __builtin_floor(static_cast<double>(l) * (8.0 * c.hi));
}
__device__ __forceinline__ double octave_of(double place) { return __builtin_floor(0.125 * place); }

// 2^(t/8), t in 0..1: the degree-5 polynomial through the Chebyshev nodes (3e-13 relative); and 2^36 times the power
// of two at the lower end of each eighth of an octave, falling, less 2^-30 of it, so that 8,192 weights stay under 2^50.
// A kernel that evaluates them for every logit takes the coefficients as an argument, in scalar registers (as literals
// each would be moved into a register pair before its use), and the eighths in LDS. (One polynomial of degree 9 over the
// octave instead: 35 instead of 28 instructions a logit, 51 instead of 46 us for the slices of 256 rows of 151,669.)
constexpr double kRoot = 0x1p36 * (1.0 - 0x1p-30);
struct WeightTable {
    double c[6], eighth[8];
};
constexpr WeightTable kWeightTable{{0x1.ffffffffff586p-1, 0x1.62e42ff11cbe7p-4, 0x1.ebfbddd2b054ap-9, 0x1.c6b1b1f5de28ap-14,
                                    0x1.3ae471589a702p-19, 0x1.6d07e00a32dbap-25},
                                   {0x1.d5818dcfba487p+0 * kRoot, 0x1.ae89f995ad3adp+0 * kRoot, 0x1.8ace5422aa0dbp+0 * kRoot,
                                    0x1.6a09e667f3bcdp+0 * kRoot, 0x1.4bfdad5362a27p+0 * kRoot, 0x1.306fe0a31b715p+0 * kRoot,
                                    0x1.172b83c7d517bp+0 * kRoot, 0x1.0000000000000p+0 * kRoot}};
// The weight's 37 bits, from its place and its eighth of the octave.
// FAR: |z| may reach 2^45, where neighbouring floats lie more octaves apart than any sum holds and z has no
// fraction left: the weight is its eighth's middle then. A caller that knows better leaves the test out.
template <bool FAR = true>
__device__ __forceinline__ uint64_t weight_of(float l, double place, double eighth, const Scale& c, const WeightTable& k) {
#pragma clang fp contract(off)
    const double ld = l;
    double t = fma(ld, 8.0 * c.lo, fma(ld, 8.0 * c.hi, -place));  // 8 z's fraction
    if (FAR) t = __builtin_fabs(place) < 0x1p48 ? t : 0.5;
    double p = fma(t, k.c[5], k.c[4]);
#pragma unroll
    for (int i = 3; i >= 0; --i) p = fma(t, p, k.c[i]);
    // + 2^52 leaves the nearest integer in the low mantissa bits
    return __builtin_bit_cast(uint64_t, fma(p, eighth, 0x1p52)) & 0xFFFFFFFFFFFFFull;
}

// floor(f s) and ceil(f s) of a float f in [0, 1) and a sum: f is m 2^-k with a 24-bit m.
__device__ __forceinline__ u128 part_of(float f, u128 s, bool up) {
    if (!(f > 0.0f)) return 0;
    const uint32_t u = __float_as_uint(f);
    const uint32_t e = u >> 23;
    const u128 m = e ? (u & 0x7FFFFFu) | 0x800000u : u & 0x7FFFFFu;
    const int k = 150 - static_cast<int>(e ? e : 1u);  // 24 .. 149
    const u128 x = m * s;                               // s < 2^98
    if (k >= 128) return up ? 1 : 0;
    const u128 r = x >> k;
    return r + (up && (r << k) != x ? 1 : 0);
}

__device__ __forceinline__ double to_double(u128 s) {
    return static_cast<double>(static_cast<uint64_t>(s >> 64)) * 0x1p64 + static_cast<double>(static_cast<uint64_t>(s));
}

template <typename T>
__device__ __forceinline__ float load_logit(const void* row, uint32_t i);
template <>
__device__ __forceinline__ float load_logit<float>(const void* row, uint32_t i) {
    return static_cast<const float*>(row)[i];
}
struct Bf16 {
    static constexpr uint32_t kMasked = 0xFF80u;  // -inf
};
struct Fp16 {
    static constexpr uint32_t kMasked = 0xFC00u;
};
template <>
__device__ __forceinline__ float load_logit<Bf16>(const void* row, uint32_t i) {
    return __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(row)[i]) << 16);
}
template <>
__device__ __forceinline__ float load_logit<Fp16>(const void* row, uint32_t i) {
    return static_cast<float>(static_cast<const _Float16*>(row)[i]);
}
template <typename T>
constexpr uint32_t kLogitBytes = 2;
template <>
constexpr uint32_t kLogitBytes<float> = 4;

// ---- the four launches -------------------------------------------------------------------------------
//
//   slices   every slice of 8,192 entries: its largest rank, and its entries' numbers and weights by bin
//   limits   per row: the slices' bins added up, the bins in which the limits cut, and every slice's sum under them
//   collect  every slice: its entries in those bins, onto the row's list
//   finish   per row: the cuts among the listed entries, and the draw
//
// (limits, collect and finish as one block per row measured 78 us where the three, now 38, took 43 us for 64 rows of
// 262,144: one compute unit reads a row at 30 GB/s or so where all of them read it in 8 us.)
// A bin is an eighth of an octave of weight. A slice counts from its own largest octave down (its row's is
// not known yet), 256 bins to a slice, the last one for all that lies deeper; octaves are absolute, so the
// slices' bins line up. A bin's entries share an octave, so its sum of 37-bit weights is one integer; the
// last bin's are brought to its octave (2^-31 of the largest) first.
constexpr uint32_t kSlice = 8192;
constexpr uint32_t kBins = 256;
constexpr uint32_t kTail = kBins - 1;
constexpr uint32_t kTailOct = kTail >> 3;
// From this octave on a weight (37 bits, 36 where it is least) may be nothing in the last bin's unit. It counts as nothing
// everywhere then: in its own sum as in its slice's, whose entries add up before they are shifted and would leave
// a sum that none of them has.
constexpr uint32_t kNothingOct = kTailOct + 36;
// Entries in the deciding bins: up to kNearCap of them are kept in LDS while they are cut, up to kListCap read from the
// list each time, and more (nearly equal logits, or nearly equal weights under a high temperature) from the row, by the
// row's one block: 0.9 to 3.9 ms for 262,144 entries.
constexpr uint32_t kNearCap = 4096, kListCap = 32768;
constexpr uint32_t kMaxSlices = 524288 / kSlice;
// A bin of a slice: its entries' number from bit 50 on, the sum of their weights below.
constexpr int kCountBit = 50;
constexpr uint64_t kMassMask = (1ull << kCountBit) - 1;

struct SliceHead {
    uint64_t best;     // largest rank of the live entries (0: none)
    uint32_t weighed;  // its bins are written
    uint32_t bad;      // a NaN or +inf was seen
};

struct RowState {
    double top;         // the largest weight's octave
    uint64_t best;
    uint64_t rank_m;    // min-p: the least rank kept (0: no limit)
    u128 below_l;       // sum of the weights in bins under lo
    u128 below_k;       // and under bin_k
    u128 all;           // of every live entry
    uint32_t done;      // nothing left to do: greedy or degenerate
    uint32_t live;
    uint32_t lo, hi;    // bins whose entries decide (lo > hi: none, every live entry is kept)
    uint32_t bin_k;     // the bin top-k cuts in, where top-p needs its sum (kBins: none)
    uint32_t k;         // top-k, 0: no limit
    uint32_t use_p;
    uint32_t count_l;   // entries in bins under lo
    uint32_t count_k;   // and under bin_k
    uint32_t in_l, in_k;  // entries in bins lo .. hi, and in bin_k
    uint32_t listed;    // entries in the deciding bins
    uint32_t appended;  // of these, on the list so far
    uint32_t key[4];    // keys of the bins' entries: key[0] .. key[1] - 1 of lo .. hi, key[2] .. key[3] - 1 of bin_k
};

struct SamplerScratch {
    uint64_t* bins;   // [rows][slices][kBins]
    SliceHead* head;  // [rows][slices]
    RowState* state;  // [rows]
    uint64_t* list;   // [rows][list_cap] ranks
    u128* under;      // [rows][slices] a slice's sum of the weights in bins under lo
    uint32_t slices;  // of max_vocab
    uint32_t list_cap;  // kListCap, or all of a smaller vocabulary
};

struct SampleArgs {
    const void* logits;
    uint64_t stride;
    uint32_t vocab, slices;
    SampleParams p;
    SampleOut o;
    SamplerScratch s;
    WeightTable table;
};

// 16 bytes of logits from any address (the hardware splits an unaligned load itself): entries i .. of a row, moved
// down to end with the row where they would pass its end. `first`: the first one's index; those under i are the
// neighbour's. No lane branches and nothing is converted yet, so that the loads of several calls travel together.
// TINY: rows shorter than a load, which are read one by one.
template <typename T>
constexpr uint32_t kVec = 16 / kLogitBytes<T>;
struct Vec {
    uint32_t w[4];
    uint32_t first;
};
template <typename T, bool TINY>
__device__ __forceinline__ Vec load_vec(const void* row, uint32_t i, uint32_t vocab) {
    Vec v;
    if constexpr (TINY) {
        v.first = i;
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            uint32_t bits[2];
#pragma unroll
            for (uint32_t h = 0; h < kVec<T> / 4; ++h) {
                const uint32_t e = i + j * (kVec<T> / 4) + h;
                if constexpr (kLogitBytes<T> == 4) {
                    bits[h] = e < vocab ? static_cast<const uint32_t*>(row)[e] : 0xFF800000u;
                } else {
                    bits[h] = e < vocab ? static_cast<const uint16_t*>(row)[e] : T::kMasked;
                }
            }
            v.w[j] = kLogitBytes<T> == 4 ? bits[0] : bits[0] | bits[kVec<T> / 4 - 1] << 16;
        }
    } else {
        v.first = i < vocab - kVec<T> ? i : vocab - kVec<T>;
        __builtin_memcpy(v.w, static_cast<const char*>(row) + static_cast<uint64_t>(v.first) * kLogitBytes<T>, 16);
    }
    return v;
}

// The bin of a weight counted from octave `top`, and its integer in that bin.
__device__ __forceinline__ uint32_t bin_of(double place, double top) {
    const double down = 8.0 * top + 7.0 - place;
    return down < static_cast<double>(kBins) ? static_cast<uint32_t>(down) : kTail;
}
__device__ __forceinline__ uint64_t mass_of(uint64_t q, double place, uint32_t bin, double top) {
    if (bin != kTail) return q;
    const double deep = top - octave_of(place) - static_cast<double>(kTailOct);
    return deep < static_cast<double>(kNothingOct - kTailOct) ? q >> static_cast<int>(deep) : 0;
}
// The two of one logit; eighths: the table's, in LDS.
__device__ __forceinline__ uint64_t entry_weight(float l, const Scale& c, const WeightTable& k, const double* eighths, double top,
                                          uint32_t* bin) {
    const double place = place_of(l, c);
    const uint32_t e = 7 - static_cast<uint32_t>(place - 8.0 * octave_of(place));
    *bin = bin_of(place, top);
    return mass_of(weight_of(l, place, eighths[e & 7], c, k), place, *bin, top);
}
// A bin's integer in units of the row's sums.
__device__ __forceinline__ u128 unit(uint64_t mass, uint32_t bin) {
    return (static_cast<u128>(mass) << kSumShift) >> (bin >> 3);
}

// Sums travel between lanes in two halves of 39 bits and more, each of which adds up by itself: a step is a
// register move per half, where carrying 128 bits would take four LDS round trips.
constexpr int kHalf = 39;
struct Halves {
    uint64_t lo, hi;
};
__device__ __forceinline__ Halves halve(u128 x) {
    return Halves{static_cast<uint64_t>(x) & ((uint64_t{1} << kHalf) - 1), static_cast<uint64_t>(x >> kHalf)};
}
// halve(unit(q, bin)) of one weight, without 128-bit shifts.
__device__ __forceinline__ Halves unit_halves(uint64_t q, uint32_t bin) {
    static_assert(kSumShift == kHalf + 1 && kTailOct < kHalf, "no bit of a weight is lost");
    return Halves{(q << (kSumShift - (bin >> 3))) & ((uint64_t{1} << kHalf) - 1), (q << 1) >> (bin >> 3)};
}
__device__ __forceinline__ u128 join(const Halves& h) { return (static_cast<u128>(h.hi) << kHalf) + h.lo; }
__device__ __forceinline__ uint64_t wave_incl_scan_u64(uint64_t x) {
    x += dpp_move<0x111>(uint64_t{0}, x);
    x += dpp_move<0x112>(uint64_t{0}, x);
    x += dpp_move<0x114>(uint64_t{0}, x);
    x += dpp_move<0x118>(uint64_t{0}, x);
    x += dpp_move<0x142, 0xA>(uint64_t{0}, x);
    x += dpp_move<0x143, 0xC>(uint64_t{0}, x);
    return x;
}
// The same inside each row of 16 lanes.
__device__ __forceinline__ uint64_t row_incl_scan_u64(uint64_t x) {
    x += dpp_move<0x111>(uint64_t{0}, x);
    x += dpp_move<0x112>(uint64_t{0}, x);
    x += dpp_move<0x114>(uint64_t{0}, x);
    x += dpp_move<0x118>(uint64_t{0}, x);
    return x;
}
// The sum over a row of 16 lanes, in each of them.
__device__ __forceinline__ uint64_t sum_of_16(uint64_t x) {
    x += dpp_move<0xB1>(uint64_t{0}, x);
    x += dpp_move<0x4E>(uint64_t{0}, x);
    x += dpp_move<0x141>(uint64_t{0}, x);
    x += dpp_move<0x140>(uint64_t{0}, x);
    return x;
}

constexpr uint32_t kRowThreads = 512;
constexpr uint32_t kRowWaves = kRowThreads / 64;

__device__ __forceinline__ u128 shfl_xor_u128(u128 v, int d) {
    const uint64_t lo = shfl_xor_u64(static_cast<uint64_t>(v), d), hi = shfl_xor_u64(static_cast<uint64_t>(v >> 64), d);
    return static_cast<u128>(hi) << 64 | lo;
}

// Running sums over the threads of the block's first WAVES waves (each includes its own), and the total, which
// every thread gets. All threads call.
struct ScanMem {
    u128 w[kRowWaves];
    uint32_t n[kRowWaves];
};
template <uint32_t WAVES>
__device__ __forceinline__ void block_scan(uint32_t& n, u128& w, uint32_t* n_all, u128* w_all, ScanMem& mem) {
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    __syncthreads();
    if (wave < WAVES) {
        n = wave_incl_scan_u32(n);
        const Halves h = halve(w);
        w = join(Halves{wave_incl_scan_u64(h.lo), wave_incl_scan_u64(h.hi)});
        if (lane == 63) mem.n[wave] = n, mem.w[wave] = w;
    }
    __syncthreads();
    uint32_t nb = 0, na = 0;
    u128 wb = 0, wa = 0;
#pragma unroll
    for (uint32_t i = 0; i < WAVES; ++i) {
        if (i == wave) nb = na, wb = wa;
        na += mem.n[i], wa += mem.w[i];
    }
    n += nb, w += wb;
    *n_all = na, *w_all = wa;
}

constexpr uint32_t kSliceThreads = 512;
constexpr uint32_t kCopies = 4;  // of a slice's bins, by lane, so that a wave's equal bins meet less often

// Bound by its arithmetic: 28 instructions a logit, 18 of them in doubles, and 10 more for the largest rank; 64 rows of
// 262,144 fp32 logits in 20 to 22 us (3.1 to 3.4 TB/s), 256 of 151,669 in bf16 in 40 to 45, where the vector units are
// busy all the time; one row in 5.5. More copies of the bins, or four and eight entries at once, changed nothing.
template <typename T, bool TINY>
__global__ __launch_bounds__(kSliceThreads) void sample_slices_kernel(SampleArgs a) {
    __shared__ uint64_t bins[kBins][kCopies];
    __shared__ double eighths[8];
    __shared__ uint32_t s_key[kSliceThreads / 64], s_bad[kSliceThreads / 64], s_idx;
    const uint32_t t = threadIdx.x, slice = blockIdx.x, lane = t % 64, wave = t / 64;
    const uint64_t r = blockIdx.y;
    const void* row = static_cast<const char*>(a.logits) + r * a.stride * kLogitBytes<T>;
    constexpr uint32_t kLoads = kSlice / kSliceThreads / kVec<T>, kEach = kLoads * kVec<T>;
    float v[kEach];
    const uint32_t i0 = slice * kSlice + t * kVec<T>;
    Vec raw[kLoads];
#pragma unroll
    for (uint32_t j = 0; j < kLoads; ++j) raw[j] = load_vec<T, TINY>(row, i0 + j * kSliceThreads * kVec<T>, a.vocab);
    const float temp = a.p.temperature ? a.p.temperature[r] : 1.0f;
    for (uint32_t i = t; i < kBins * kCopies; i += kSliceThreads) bins[i / kCopies][i % kCopies] = 0;
    if (t < 8) eighths[t] = a.table.eighth[t];
    if (t == 0) s_idx = ~0u;
    const Scale c = scale_of(temp);
    float best = -INFINITY;
    uint64_t nan = 0;
#pragma unroll
    for (uint32_t j = 0; j < kLoads; ++j) {
#pragma unroll
        for (uint32_t e = 0; e < kVec<T>; ++e) v[j * kVec<T> + e] = load_logit<T>(raw[j].w, e);
        const uint32_t over = i0 + j * kSliceThreads * kVec<T> - raw[j].first;
        if (__ballot(over != 0) != 0) {  // the row's end: the neighbour's entries, or none at all
#pragma unroll
            for (uint32_t e = 0; e < kVec<T>; ++e) v[j * kVec<T> + e] = e < over ? -INFINITY : v[j * kVec<T> + e];
        }
#pragma unroll
        for (uint32_t e = j * kVec<T>; e < (j + 1) * kVec<T>; e += 2) {
            nan |= __ballot(__builtin_isunordered(v[e], v[e + 1]));
            best = fmaxf(best, fmaxf(v[e], v[e + 1]));
        }
    }
    const uint32_t own = float_key(best);
    uint32_t key = wave_reduce(own, 0u, [](uint32_t x, uint32_t y) { return x > y ? x : y; });
    if (lane == 0) s_key[wave] = key, s_bad[wave] = nan != 0 ? 1u : 0u;
    __syncthreads();
    uint32_t bad = 0;
#pragma unroll
    for (uint32_t i = 0; i < kSliceThreads / 64; ++i) key = s_key[i] > key ? s_key[i] : key, bad |= s_bad[i];
    best = key_float(key);
    bad |= best < INFINITY ? 0u : 1u;
    const bool live = best > -INFINITY;
    if (own == key) {
        uint32_t idx = ~0u;
#pragma unroll
        for (uint32_t j = kEach; j-- > 0;)
            if (v[j] == best) idx = raw[j / kVec<T>].first + j % kVec<T>;
        atomicMin(&s_idx, idx);
    }
    const bool weigh = live && bad == 0 && temp > 0.0f;  // a row with a NaN or +inf, and a greedy one, needs no weights
    if (weigh) {
        const double top = octave_of(place_of(best, c));
        if (__builtin_fabs(top) < 0x1p44) {
            // Nothing branches on an entry's value, and only the counting leaves masked ones out. (An entry so far
            // down that its z holds no fraction shifts to nothing.)
#pragma unroll
            for (uint32_t j = 0; j < kEach; ++j) {
                const double place = place_of(v[j], c);
                const uint32_t b = static_cast<uint32_t>(8.0 * top + 7.0 - place);
                const uint64_t q = weight_of<false>(v[j], place, eighths[b & 7], c, a.table);
                const uint32_t d = b >> 3 < kTailOct + 63 ? b >> 3 : kTailOct + 63;
                const uint64_t m = q >> ((d > kTailOct ? d : kTailOct) - kTailOct);
                if (v[j] > -INFINITY)
                    atomicAdd(reinterpret_cast<unsigned long long*>(&bins[b < kTail ? b : kTail][lane % kCopies]),
                              static_cast<unsigned long long>(1ull << kCountBit | m));
            }
        } else {
#pragma unroll 1
            for (uint32_t i = slice * kSlice + t; i < min(a.vocab, (slice + 1) * kSlice); i += kSliceThreads) {
                const float l = load_logit<T>(row, i);
                if (!(l > -INFINITY)) continue;
                uint32_t b;
                const uint64_t m = entry_weight(l, c, a.table, eighths, top, &b);
                atomicAdd(reinterpret_cast<unsigned long long*>(&bins[b][lane % kCopies]),
                          static_cast<unsigned long long>(1ull << kCountBit | m));
            }
        }
    }
    __syncthreads();
    const uint64_t at = r * a.s.slices + slice;
    if (t == 0) a.s.head[at] = SliceHead{live ? static_cast<uint64_t>(key) << 32 | (0xFFFFFFFFu - s_idx) : 0, weigh ? 1u : 0u, bad};
    if (weigh && t < kBins) {
        uint64_t x = 0;
#pragma unroll
        for (uint32_t i = 0; i < kCopies; ++i) x += bins[t][i];
        a.s.bins[at * kBins + t] = x;
    }
}
static_assert(kMaxSlices <= 64, "a lane to a slice");

// The row's bin of a slice's bin, `shift` octaves under the row's largest, and what to shift its sum by.
__device__ __forceinline__ uint32_t row_bin(uint32_t b, uint32_t shift, uint32_t* down) {
    const uint32_t x = b + 8 * shift;
    *down = 0;
    if (x < kTail && b != kTail) return x;
    *down = (b >> 3) + shift - kTailOct;
    return kTail;
}
constexpr uint32_t kNoSlice = 255;  // the shift of a slice whose bins are not written
constexpr uint32_t kFarSlice = 128;  // and of one that lies too deep: its entries count, and every sum is shifted to nothing
static_assert(kFarSlice - kTailOct >= 64, "row_bin's shift");
__device__ __forceinline__ uint32_t slice_shift(const SliceHead& h, double top, const Scale& c) {
    if (h.weighed == 0) return kNoSlice;
    const double d = top - __builtin_floor(static_cast<double>(rank_value(h.best)) * c.hi);
    return d < static_cast<double>(kNothingOct) ? static_cast<uint32_t>(d) : kFarSlice;
}

// The least key at which `yes` holds, by a wave: it holds from there up to `above`, where it is taken to hold.
// First the 64 keys around the guess, then, had that been further off, cuts by 64.
constexpr uint32_t kLeast = 0x007FFFFFu;  // -inf's key: below every entry's
template <typename F>
__device__ __forceinline__ uint32_t least_key(uint32_t guess, uint32_t above, F yes) {
    const uint32_t lane = threadIdx.x % 64;
    uint64_t lo = kLeast + 1, hi = above;  // it lies between, hi included
    uint64_t from = guess > lo + 32 ? (guess < hi ? guess : hi) - 32 : lo;
    uint64_t step = 1;
    for (;;) {
        const uint64_t x = from + lane * step;
        const uint64_t set = __ballot(x >= hi || yes(key_float(static_cast<uint32_t>(x))));
        if (set == 0) {
            lo = from + 63 * step + 1;
        } else {
            const uint32_t first = static_cast<uint32_t>(__builtin_ctzll(set));
            const uint64_t at = from + first * step;
            hi = at < hi ? at : hi;
            if (first != 0) lo = from + (first - 1) * step + 1;
        }
        if (lo >= hi) return static_cast<uint32_t>(hi);
        from = lo, step = (hi - lo + 63) / 64;
    }
}

// The least rank that min-p keeps: (l - M) log2(e) / T >= log2(min_p); the best one where none does.
__device__ uint64_t least_kept(uint64_t best, float min_p, const Scale& c) {
    const float m = rank_value(best);
    const double lim = log2(static_cast<double>(min_p));
    auto keeps = [&](float l) { return (static_cast<double>(l) - static_cast<double>(m)) * c.hi >= lim; };
    if (!keeps(m)) return best;
    if (c.hi == 0.0) return static_cast<uint64_t>(kLeast) << 32;
    // the quotient and the sum are rounded, the float once more: it lies a few floats around their result
    const uint32_t guess = float_key(static_cast<float>(static_cast<double>(m) + lim / c.hi));
    return static_cast<uint64_t>(least_key(guess, static_cast<uint32_t>(best >> 32), keeps)) << 32;
}

// The least key whose entry lies in a bin of at most b (bins fall with rising logits): where z reaches the bin's
// lower end.
__device__ uint32_t bin_key(uint32_t b, uint32_t above, double top, const Scale& c) {
    if (b >= kTail) return kLeast + 1;
    const double z = top + 1.0 - 0.125 * static_cast<double>(b + 1);
    const uint32_t guess = c.hi > 0.0 ? float_key(static_cast<float>(z / c.hi)) : above;
    return least_key(guess, above, [&](float l) { return bin_of(place_of(l, c), top) <= b; });
}

// What every wave of a block learns of its row from the slices' heads.
struct RowHead {
    uint64_t best;
    uint32_t bad;
    SliceHead own;  // of slice `lane`
};
__device__ __forceinline__ RowHead read_heads(const SampleArgs& a, uint64_t r) {
    const uint32_t lane = threadIdx.x % 64;
    RowHead h{0, 0, {0, 0, 0}};
    if (lane < a.slices) h.own = a.s.head[r * a.s.slices + lane];
    h.best = wave_max_u64(h.own.best);
    h.bad = wave_reduce(h.own.bad, 0u, [](uint32_t x, uint32_t y) { return x | y; });
    return h;
}

// A chain of dependent steps in one block to a row (heads, bins, a scan, the cuts, their keys): 9.4 us for one row,
// 10.0 for 256.
__global__ __launch_bounds__(kRowThreads) void sample_limits_kernel(SampleArgs a) {
    __shared__ uint64_t mass[kRowThreads], s_rank_m;
    __shared__ uint32_t count[kRowThreads], counts[kBins], found[3], s_key[4], s_bin_m, s_tail_n;
    __shared__ unsigned long long s_tail;
    __shared__ u128 sums[kBins];
    __shared__ ScanMem scan;
    const uint32_t t = threadIdx.x, lane = t % 64, wave = __builtin_amdgcn_readfirstlane(t / 64);
    const uint64_t r = blockIdx.x;
    const RowHead head = read_heads(a, r);
    const float temp = a.p.temperature ? a.p.temperature[r] : 1.0f, u = a.p.uniform[r];
    const float top_p = a.p.top_p ? a.p.top_p[r] : 1.0f, min_p = a.p.min_p ? a.p.min_p[r] : 0.0f;
    const int32_t top_k = a.p.top_k ? a.p.top_k[r] : 0;
    const uint64_t best = head.best;
    const bool none = head.bad != 0 || best == 0 || temp != temp || u != u || top_p != top_p || min_p != min_p;
    if (none || temp <= 0.0f) {
        if (t == 0) {
            a.s.state[r].done = 1;
            a.s.state[r].listed = 0;
            a.o.tokens[r] = none ? TWD_TOKEN_DEGENERATE : rank_index(best);
            if (a.o.logprobs) a.o.logprobs[r] = none ? __uint_as_float(0x7FC00000u) : 0.0f;
            if (a.o.kept) a.o.kept[r] = none ? 0 : 1;
        }
        return;
    }
    const Scale c = scale_of(temp);
    const double top = octave_of(place_of(rank_value(best), c));
    const uint32_t shift = slice_shift(head.own, top, c);

    // ---- the row's bins. Two threads to a bin, every other slice each: a slice's bin 8 `shift` above it. What lies
    // deeper than the row's last but one bin adds up in that last one.
    const uint64_t* bins = a.s.bins + r * a.s.slices * kBins;
    {
        const uint32_t bin = t % kBins;
        constexpr uint32_t kEvery = kRowThreads / kBins, kTurns = kMaxSlices / kEvery;
        const uint32_t s0 = __builtin_amdgcn_readfirstlane(t / kBins);
        uint64_t m = 0, tail = 0;
        uint32_t n_bin = 0, n_tail = 0;
#pragma unroll 1
        for (uint32_t j = 0; j < kTurns && j * kEvery < a.slices; j += 16) {
            uint64_t x[16], y[16];
#pragma unroll
            for (uint32_t i = 0; i < 16; ++i) {
                const uint32_t slice = s0 + (j + i) * kEvery;
                const uint32_t sh = __builtin_amdgcn_readlane(shift, slice);  // (kNoSlice past the last)
                // (every lane loads, so that the loads travel together; what does not count is dropped after)
                const uint64_t* from = bins + min(slice, a.slices - 1) * kBins;
                x[i] = from[max(bin, 8 * sh) - 8 * sh];
                y[i] = 0;
                if ((bin | 63) + 8 * sh >= kTail) y[i] = from[bin];  // a wave's lanes alike
            }
#pragma unroll
            for (uint32_t i = 0; i < 16; ++i) {
                const uint32_t slice = s0 + (j + i) * kEvery;
                const uint32_t sh = __builtin_amdgcn_readlane(shift, slice);
                if (sh == kNoSlice || bin >= kTail || bin < 8 * sh) x[i] = 0;
                if (sh == kNoSlice || bin + 8 * sh < kTail) y[i] = 0;
            }
#pragma unroll
            for (uint32_t i = 0; i < 16; ++i) {
                const uint32_t slice = s0 + (j + i) * kEvery;
                const uint32_t sh = __builtin_amdgcn_readlane(shift, slice);
                m += x[i] & kMassMask, n_bin += static_cast<uint32_t>(x[i] >> kCountBit);
                const uint32_t down = (bin >> 3) + sh - kTailOct;
                tail += down < 64 ? (y[i] & kMassMask) >> down : 0, n_tail += static_cast<uint32_t>(y[i] >> kCountBit);
            }
        }
        if (t < 3) found[t] = kBins;
        if (t == 0) s_rank_m = 0, s_bin_m = kBins, s_tail = 0, s_tail_n = 0;
        mass[t] = m, count[t] = n_bin;
        __syncthreads();
        if (__ballot(n_tail != 0) != 0) {
            tail = wave_reduce(tail, uint64_t{0}, [](uint64_t p, uint64_t q) { return p + q; });
            n_tail = wave_reduce(n_tail, 0u, [](uint32_t p, uint32_t q) { return p + q; });
            if (lane == 0) atomicAdd(&s_tail, static_cast<unsigned long long>(tail)), atomicAdd(&s_tail_n, n_tail);
        }
        if (wave == kRowThreads / 64 - 1 && min_p > 0.0f) {
            const uint64_t rank = least_kept(best, min_p, c);
            const float l = rank_value(rank);
            const uint32_t b = l > -INFINITY ? bin_of(place_of(l, c), top) : kBins;
            if (lane == 0) s_rank_m = rank, s_bin_m = b;
        }
        __syncthreads();
    }
    uint32_t n = 0, live;
    u128 w = 0, w_all;
    if (t < kBins) {
        uint64_t m = t == kTail ? s_tail : 0;
        n = t == kTail ? s_tail_n : 0;
#pragma unroll
        for (uint32_t i = 0; i < kRowThreads / kBins; ++i) m += mass[i * kBins + t], n += count[i * kBins + t];
        w = unit(m, t);
    }
    block_scan<kBins / 64>(n, w, &live, &w_all, scan);
    if (t < kBins) counts[t] = n, sums[t] = w;
    __syncthreads();

    // ---- the bin each limit cuts in: the first whose running number or sum reaches it
    const uint32_t k = top_k > 0 && static_cast<uint32_t>(top_k) < live ? static_cast<uint32_t>(top_k) : 0;
    const bool use_p = top_p < 1.0f;
    if (k != 0) {
        if (t < kBins && n >= k && (t == 0 || counts[t - 1] < k)) found[0] = t;
        __syncthreads();
    }
    const uint32_t bin_k = found[0];
    if (use_p) {
        if (t < kBins) {
            // the top-k's sum lies between those of the bins under and with its cut
            const u128 low = part_of(top_p, k ? (bin_k ? sums[bin_k - 1] : 0) : w_all, true);
            const u128 high = k ? part_of(top_p, sums[bin_k], true) : low;
            auto reaches = [&](uint32_t b, u128 v) { return counts[b] >= 1 && sums[b] >= v; };
            if (reaches(t, low) && (t == 0 || !reaches(t - 1, low))) found[1] = t;
            if (reaches(t, high) && (t == 0 || !reaches(t - 1, high))) found[2] = t;
        }
        __syncthreads();
    }
    // lo .. hi: the bins whose entries decide (lo = kBins: none, every live entry is kept); need_k: those of bin_k
    // do too, for the top-k's sum
    uint32_t lo = kBins, hi = kBins;
    if (use_p)
        lo = found[1], hi = found[2];
    else if (k)
        lo = hi = bin_k;
    bool need_k = use_p && k;
    const uint32_t bin_m = s_bin_m;
    if (bin_m < lo) lo = hi = bin_m, need_k = false;  // the other limits cut deeper
    if (bin_m < hi) hi = bin_m;
    const bool any = lo < kBins;
    const u128 below_l = any && lo ? sums[lo - 1] : 0, below_k = need_k && bin_k ? sums[bin_k - 1] : 0;
    const uint32_t count_l = any && lo ? counts[lo - 1] : 0, count_k = need_k && bin_k ? counts[bin_k - 1] : 0;
    const uint32_t in_l = any ? counts[hi] - count_l : 0, in_k = need_k ? counts[bin_k] - count_k : 0;
    const uint32_t listed = in_l + (need_k && bin_k > hi ? in_k : 0);

    // ---- the keys that bound those bins, a wave each, and every slice's sum under them: what the draw starts from.
    // key[0] .. key[1] - 1: entries of lo .. hi; key[2] .. key[3] - 1: of bin_k
    if (wave < 4) {
        const uint32_t above = static_cast<uint32_t>(best >> 32) + 1;
        uint32_t key = 0;
        if (wave < 2 ? any : need_k) {
            const uint32_t b0 = wave < 2 ? lo : bin_k, b1 = wave < 2 ? hi : bin_k, b = wave % 2 == 0 ? b1 : b0 - 1;
            key = wave % 2 != 0 && b0 == 0 ? above : bin_key(b, above, top, c);
        }
        if (lane == 0) s_key[wave] = key;
    }
#pragma unroll 1
    for (uint32_t s0 = 0; s0 < a.slices; s0 += kRowThreads / 16) {  // sixteen threads to a slice, sixteen of its bins each
        const uint32_t slice = s0 + t / 16, sh = __shfl(shift, slice % 64);
        uint64_t x[16];
#pragma unroll
        for (uint32_t i = 0; i < 16; ++i) x[i] = bins[min(slice, a.slices - 1) * kBins + t % 16 + 16 * i];
        u128 sum = 0;
#pragma unroll
        for (uint32_t i = 0; i < 16; ++i) {
            uint32_t down;
            const uint32_t b = row_bin(t % 16 + 16 * i, sh, &down);
            if (b < lo && sh != kNoSlice) sum += unit(down < 64 ? (x[i] & kMassMask) >> down : 0, b);
        }
        const Halves h = halve(sum);
        sum = join(Halves{sum_of_16(h.lo), sum_of_16(h.hi)});
        if (t % 16 == 0 && slice < a.slices) a.s.under[r * a.s.slices + slice] = sum;
    }
    __syncthreads();
    if (t == 0) {
        RowState& st = a.s.state[r];
        st.top = top, st.best = best, st.rank_m = s_rank_m, st.all = w_all, st.live = live, st.k = k, st.use_p = use_p;
        st.bin_k = need_k ? bin_k : kBins, st.done = 0, st.appended = 0, st.lo = any ? lo : 1, st.hi = any ? hi : 0;
        st.below_l = below_l, st.count_l = count_l, st.in_l = in_l;
        st.below_k = below_k, st.count_k = count_k, st.in_k = in_k, st.listed = listed;
        for (uint32_t i = 0; i < 4; ++i) st.key[i] = s_key[i];
    }
}

// A second look at the logits, of the slices alone whose largest may decide: 4.2 us for one row, 8.7 for 64 rows of
// 262,144 fp32 logits, 24 for 256 of 151,669 in bf16 (most of the logits, 3.2 TB/s).
template <typename T, bool TINY>
__global__ __launch_bounds__(kSliceThreads) void sample_collect_kernel(SampleArgs a) {
    __shared__ uint32_t s_n, s_base;
    const uint32_t t = threadIdx.x, slice = blockIdx.x, lane = t % 64;
    const uint64_t r = blockIdx.y;
    RowState* st = a.s.state + r;
    const uint32_t listed = st->listed, k0 = st->key[0], k1 = st->key[1], k2 = st->key[2], k3 = st->key[3];
    const uint32_t most = static_cast<uint32_t>(a.s.head[r * a.s.slices + slice].best >> 32);
    if (listed == 0 || listed > a.s.list_cap) return;
    const bool two = k2 < k3 && k2 < k0;  // a bin_k past lo .. hi
    if (most < (two ? k2 : k0)) return;   // all of the slice lies below
    if (t == 0) s_n = 0;
    const void* row = static_cast<const char*>(a.logits) + r * a.stride * kLogitBytes<T>;
    constexpr uint32_t kLoads = kSlice / kSliceThreads / kVec<T>;
    const uint32_t i0 = slice * kSlice + t * kVec<T>;
    Vec v[kLoads];
#pragma unroll
    for (uint32_t j = 0; j < kLoads; ++j) v[j] = load_vec<T, TINY>(row, i0 + j * kSliceThreads * kVec<T>, a.vocab);
    __syncthreads();
    // the lanes whose entry e of load j decides (keys order as their floats do; -inf lies under all)
    const float f0 = key_float(k0), f1 = key_float(k1), f2 = key_float(k2), f3 = key_float(k3);
    uint64_t in[kLoads][kVec<T>];
    uint32_t number = 0;
#pragma unroll
    for (uint32_t j = 0; j < kLoads; ++j) {
#pragma unroll
        for (uint32_t e = 0; e < kVec<T>; ++e) {
            const float l = load_logit<T>(v[j].w, e);
            in[j][e] = __ballot(l >= f0) & __ballot(l < f1);
            if (two) in[j][e] |= __ballot(l >= f2) & __ballot(l < f3);
        }
        const uint32_t over = i0 + j * kSliceThreads * kVec<T> - v[j].first;
        if (__ballot(over != 0) != 0) {  // the row's end: a lane holds its neighbour's entries first
#pragma unroll
            for (uint32_t e = 0; e < kVec<T>; ++e) in[j][e] &= __ballot(e >= over);
        }
#pragma unroll
        for (uint32_t e = 0; e < kVec<T>; ++e) number += static_cast<uint32_t>(__builtin_popcountll(in[j][e]));
    }
    uint32_t at = 0;
    if (lane == 0 && number != 0) at = atomicAdd(&s_n, number);
    __syncthreads();
    if (s_n == 0) return;
    if (t == 0) s_base = atomicAdd(&st->appended, s_n);
    __syncthreads();
    if (number == 0) return;
    at = __builtin_amdgcn_readfirstlane(at) + s_base;
#pragma unroll
    for (uint32_t j = 0; j < kLoads; ++j) {
#pragma unroll
        for (uint32_t e = 0; e < kVec<T>; ++e) {
            if (in[j][e] == 0) continue;
            const uint32_t to = at + __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(in[j][e] >> 32),
                                                              __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(in[j][e]), 0));
            // the bins' own numbers say how many come: the list holds them all
            if ((in[j][e] >> lane & 1) != 0 && to < a.s.list_cap)
                a.s.list[r * a.s.list_cap + to] = rank_key(load_logit<T>(v[j].w, e), v[j].first + e);
            at += static_cast<uint32_t>(__builtin_popcountll(in[j][e]));
        }
    }
}

constexpr uint32_t kFarAhead = 4;         // entries on their way where they come from memory
constexpr uint32_t kSmall = 64;           // entries that are ranked against each other directly
constexpr uint32_t kParts = kRowThreads;  // parts that a range of ranks is cut into
constexpr uint32_t kStageEach = kSlice / kRowThreads, kStageStride = kStageEach + 1;  // a thread's entries, an odd way apart

struct FinishMem {
    union {
        struct {
            uint64_t rank[kNearCap];
            uint64_t weight[kNearCap];  // its bin above bit 48, the weight below
        };
        float stage[kRowThreads * kStageStride];
    };
    uint32_t part_n[kParts];
    unsigned long long part_lo[kParts], part_hi[kParts];
    uint64_t small[kSmall];
    u128 small_w[kSmall];
    unsigned long long slice_lo[kMaxSlices], slice_hi[kMaxSlices];
    ScanMem scan;
    unsigned long long least, most;
    double eighths[8];
    uint64_t cut;
    u128 sum, base_w, want;
    uint32_t n, base_n, pick, id, last;
};

// One block to a row: 9.8 us for one row, the slowest of 64 takes 19 and of 256 bf16 rows (2,000 listed entries of a
// few values each) 29. About half goes to the cuts, a round of adding up by parts after another, a quarter to the
// weights of the one slice that the draw falls in, where all of it is kept (vector units of one compute unit; with sums
// of 128 bits instead of halves there and in the rounds 21 and 31 us). 1,024 threads: 13.7 us for one row, 39 for 256.
template <typename T, bool TINY>
__global__ __launch_bounds__(kRowThreads) void sample_finish_kernel(SampleArgs a) {
    extern __shared__ char finish_mem[];
    FinishMem& sm = *reinterpret_cast<FinishMem*>(finish_mem);
    const uint32_t t = threadIdx.x, lane = t % 64;
    const uint64_t r = blockIdx.x;
    const RowState& st = a.s.state[r];
    const uint32_t done = st.done, listed = st.listed;
    const float temp = a.p.temperature ? a.p.temperature[r] : 1.0f, u = a.p.uniform[r];
    const float top_p = a.p.top_p ? a.p.top_p[r] : 1.0f;
    const u128 under = a.s.under[r * a.s.slices + min(t, a.slices - 1)];
    if (done) return;
    const void* row = static_cast<const char*>(a.logits) + r * a.stride * kLogitBytes<T>;
    const Scale c = scale_of(temp);
    const double top = st.top;
    const uint32_t lo = st.lo, hi = st.hi, k = st.k, bin_k = st.bin_k;
    const bool near = listed <= kNearCap, on_list = listed <= a.s.list_cap, any = lo <= hi, use_p = st.use_p != 0, need_k = bin_k < kBins;
    auto weight = [&](float l, uint32_t* bin) { return entry_weight(l, c, a.table, sm.eighths, top, bin); };
    if (t < kMaxSlices) sm.slice_lo[t] = 0, sm.slice_hi[t] = 0;
    if (t == 0) sm.last = 0, sm.id = ~0u;
    if (t < 8) sm.eighths[t] = a.table.eighth[t];
    __syncthreads();
    const uint64_t* list = a.s.list + r * a.s.list_cap;
    if (near) {
#pragma unroll 1
        for (uint32_t i = t; i < listed; i += kRowThreads) {
            const uint64_t rank = list[i];
            uint32_t b;
            const uint64_t m = weight(rank_value(rank), &b);
            sm.rank[i] = rank, sm.weight[i] = static_cast<uint64_t>(b) << 48 | m;
        }
    }
    // f(rank, bin, weight) of every entry in the row's bins lo .. hi, or, of_k, in bin_k: those whose keys the bins'
    // bound. (A thread meets the same entries in LDS each time.)
    auto members = [&](bool of_k, auto f) {
        const uint32_t key0 = st.key[of_k ? 2 : 0], key1 = st.key[of_k ? 3 : 1];
        auto in = [&](uint64_t rank) {
            const uint32_t key = static_cast<uint32_t>(rank >> 32);
            return key >= key0 && key < key1;
        };
        if (near) {
#pragma unroll 1
            for (uint32_t i = t; i < listed; i += kRowThreads) {
                const uint64_t rank = sm.rank[i], x = sm.weight[i];
                if (in(rank)) f(rank, static_cast<uint32_t>(x >> 48), x & 0xFFFFFFFFFFFFull);
            }
            return;
        }
        const uint32_t end = on_list ? listed : a.vocab;
        auto get = [&](uint32_t i) -> uint64_t {  // (key 0 lies below every entry's)
            if (i >= end) return 0;
            return on_list ? list[i] : rank_key(load_logit<T>(row, i), i);
        };
        uint64_t ahead[kFarAhead];
#pragma unroll
        for (uint32_t j = 0; j < kFarAhead; ++j) ahead[j] = get(t + j * kRowThreads);
#pragma unroll 1
        for (uint32_t i = t; i < end; i += kRowThreads) {
            const uint64_t rank = ahead[0];
#pragma unroll
            for (uint32_t j = 0; j + 1 < kFarAhead; ++j) ahead[j] = ahead[j + 1];
            ahead[kFarAhead - 1] = get(i + kFarAhead * kRowThreads);
            if (in(rank)) {
                uint32_t b;
                const uint64_t m = weight(rank_value(rank), &b);
                f(rank, b, m);
            }
        }
    };
    // Among the entries of bins lo .. hi, or of bin_k, `have` of them, ranks r0 .. r1, with base_n entries of sum base_w before
    // them: the rank of the one that brings the number to n, or the sum to w (by_sum); 0 where none does. *sum:
    // the sum with it. While they are many, the range of their ranks is cut into parts and the part that holds it
    // kept.
    auto select = [&](bool of_k, uint32_t have, uint64_t r0, uint64_t r1, uint32_t base_n, u128 base_w,
                      bool by_sum, uint32_t n, u128 w, u128* sum) {
        for (bool first = true;; first = false) {
            __syncthreads();
            if (t == 0) sm.n = 0, sm.least = ~0ull, sm.most = 0, sm.cut = 0, sm.sum = 0, sm.pick = kParts;
            if (have <= kSmall) {
                __syncthreads();
                members(of_k, [&](uint64_t k, uint32_t b, uint64_t m) {
                    if (k < r0 || k > r1) return;
                    const uint32_t at = atomicAdd(&sm.n, 1u);
                    if (at < kSmall) sm.small[at] = k, sm.small_w[at] = unit(m, b);
                });
                __syncthreads();
                // eight threads to an entry add up those of larger rank
                const uint32_t e = t / 8;
                if (e < have) {
                    const uint64_t mine = sm.small[e];
                    uint32_t more = 0;
                    u128 over = 0;
                    for (uint32_t i = t % 8; i < have; i += 8) {
                        const bool larger = sm.small[i] > mine;
                        more += larger ? 1u : 0u;
                        over += larger ? sm.small_w[i] : 0;
                    }
#pragma unroll
                    for (int d = 1; d < 8; d *= 2) more += __shfl_xor(more, d), over += shfl_xor_u128(over, d);
                    const u128 before = base_w + over, with = before + sm.small_w[e];
                    if (t % 8 == 0 && (by_sum ? before < w && with >= w : base_n + more + 1 == n)) sm.cut = mine, sm.sum = with;
                }
                __syncthreads();
                *sum = sm.sum;
                return sm.cut;
            }
            sm.part_n[t] = 0, sm.part_lo[t] = 0, sm.part_hi[t] = 0;
            __syncthreads();
            if (!first) {  // equal logits: their ranks fill little of the range
                uint64_t least = ~0ull, most = 0;
                members(of_k, [&](uint64_t k, uint32_t, uint64_t) {
                    if (k < r0 || k > r1) return;
                    least = k < least ? k : least, most = k > most ? k : most;
                });
                most = wave_max_u64(most);
                least = ~wave_max_u64(~least);
                if (lane == 0)
                    atomicMax(&sm.most, static_cast<unsigned long long>(most)), atomicMin(&sm.least, static_cast<unsigned long long>(least));
                __syncthreads();
                r0 = sm.least, r1 = sm.most;
            }
            const uint64_t range = r1 - r0;
            const int sft = range < kParts ? 0 : 55 - __builtin_clzll(range);  // range >> sft < 512
            members(of_k, [&](uint64_t k, uint32_t b, uint64_t m) {
                if (k < r0 || k > r1) return;
                const uint32_t d = kParts - 1 - static_cast<uint32_t>((k - r0) >> sft);  // falling
                const Halves x = unit_halves(m, b);
                // Equal logits meet in one part: while a wave's first entry has company, the lanes that hold its part
                // and its weight add up as one.
                bool todo = true;
#pragma unroll 1
                for (uint32_t turn = 0; turn < 16; ++turn) {
                    const uint32_t d0 = __builtin_amdgcn_readfirstlane(d);
                    const uint64_t m0 = static_cast<uint64_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(m >> 32))) << 32 |
                                        __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(m));
                    const bool same = d == d0 && m == m0;
                    const uint64_t mates = __ballot(same);
                    const uint32_t number = static_cast<uint32_t>(__builtin_popcountll(mates));
                    if (number < 4) break;
                    if (same) {
                        if (static_cast<uint32_t>(__builtin_ctzll(mates)) == lane) {
                            atomicAdd(&sm.part_n[d], number);
                            atomicAdd(&sm.part_lo[d], static_cast<unsigned long long>(x.lo * number));
                            atomicAdd(&sm.part_hi[d], static_cast<unsigned long long>(x.hi * number));
                        }
                        todo = false;
                        break;
                    }
                }
                if (!todo) return;
                atomicAdd(&sm.part_n[d], 1u);
                atomicAdd(&sm.part_lo[d], static_cast<unsigned long long>(x.lo));
                atomicAdd(&sm.part_hi[d], static_cast<unsigned long long>(x.hi));
            });
            __syncthreads();
            const uint32_t own_n = sm.part_n[t];
            const u128 own = join(Halves{sm.part_lo[t], sm.part_hi[t]});
            uint32_t x = own_n, x_all;
            u128 y = own, y_all;
            block_scan<kRowWaves>(x, y, &x_all, &y_all, sm.scan);
            if (own_n != 0 && (by_sum ? base_w + y >= w && base_w + y - own < w : base_n + x >= n && base_n + x - own_n < n))
                sm.pick = t, sm.n = own_n, sm.base_n = base_n + x - own_n, sm.base_w = base_w + y - own;
            __syncthreads();
            if (sm.pick == kParts) {
                *sum = base_w + y_all;
                return uint64_t{0};
            }
            base_n = sm.base_n, base_w = sm.base_w, have = sm.n;
            const uint64_t from = r0 + (static_cast<uint64_t>(kParts - 1 - sm.pick) << sft), to = from + ((uint64_t{1} << sft) - 1);
            r1 = to < r1 ? to : r1, r0 = from;
        }
    };

    // ---- top-k's cut by number, then top-p's by its share of the top-k's sum
    uint64_t cut = 0;  // ranks of at least this are kept
    u128 sum = st.all;
#pragma unroll 1
    for (int by_sum = 0; by_sum < 2; ++by_sum) {
        const bool for_k = by_sum == 0 && need_k;
        const u128 want = by_sum ? part_of(top_p, sum, true) : 0;
        if (by_sum ? !use_p : (use_p ? !for_k : k == 0)) continue;
        uint64_t x = st.best;
        if (for_k || by_sum == 0 || want > 0) {
            const uint32_t key0 = st.key[for_k ? 2 : 0], key1 = st.key[for_k ? 3 : 1];
            u128 with;
            x = select(for_k, for_k ? st.in_k : st.in_l, static_cast<uint64_t>(key0) << 32,
                       (static_cast<uint64_t>(key1) << 32) - 1, for_k ? st.count_k : st.count_l, for_k ? st.below_k : st.below_l,
                       by_sum != 0, k, want, &with);
            if (by_sum == 0) sum = with;
        }
        cut = x > cut ? x : cut;
    }
    cut = st.rank_m > cut ? st.rank_m : cut;

    // ---- the draw: kept weights by slice, then through the slice
    __syncthreads();
    if (t == 0) sm.n = 0;
    __syncthreads();
    if (any) {
        members(false, [&](uint64_t k, uint32_t b, uint64_t m) {
            if (k < cut) return;
            const Halves x = unit_halves(m, b);
            const uint32_t slice = rank_index(k) / kSlice;
            atomicAdd(&sm.slice_lo[slice], static_cast<unsigned long long>(x.lo));
            atomicAdd(&sm.slice_hi[slice], static_cast<unsigned long long>(x.hi));
            atomicAdd(&sm.n, 1u);
        });
    }
    __syncthreads();
    uint32_t n = 0, n_all;
    u128 own = 0, kept;
    if (t < a.slices) own = under + join(Halves{sm.slice_lo[t], sm.slice_hi[t]});
    u128 w = own;
    block_scan<kMaxSlices / 64>(n, w, &n_all, &kept, sm.scan);
    const u128 want = u < 1.0f ? part_of(u, kept, false) : kept - 1;  // the first running sum past this is drawn
    // A draw of 0 takes the first kept id, however little it weighs: the first slice whose largest rank is kept, and
    // there the first kept entry. What even a double holds nothing of (exp of less than -745.14, 1,075 octaves) weighs nothing.
    const bool at_zero = !(u > 0.0f);
    const float largest = rank_value(st.best);
    auto positive = [&](float l) { return (static_cast<double>(l) - largest) * c.hi > -1075.0; };
    if (at_zero) {
        static_assert(kMaxSlices == 64, "a wave's lanes are the slices");
        if (t < kMaxSlices) {
            const uint64_t rank = t < a.slices ? a.s.head[r * a.s.slices + t].best : 0;
            const uint64_t in = __ballot(rank != 0 && rank >= cut && positive(rank_value(rank)));
            if (t == 0) sm.pick = static_cast<uint32_t>(__builtin_ctzll(in)), sm.want = 0;  // (the row's largest is one)
        }
    } else if (t < a.slices && w > want && w - own <= want) {
        sm.pick = t, sm.want = want - (w - own);
    }
    __syncthreads();
    const uint32_t first = sm.pick * kSlice;
    const u128 rest = sm.want;
    // the slice through LDS: read in rows, summed by thread
    Vec part[kStageEach / kVec<T>];
#pragma unroll
    for (uint32_t j = 0; j < kStageEach / kVec<T>; ++j) part[j] = load_vec<T, TINY>(row, first + (j * kRowThreads + t) * kVec<T>, a.vocab);
#pragma unroll
    for (uint32_t j = 0; j < kStageEach / kVec<T>; ++j) {
        const uint32_t i = (j * kRowThreads + t) * kVec<T>, over = first + i - part[j].first;
#pragma unroll
        for (uint32_t e = 0; e < kVec<T>; ++e) {
            // a lane at the row's end holds entries from `over` under its own on: it drops them and masks the rest
            const uint32_t to = e >= over ? i + e - over : i + kVec<T> - 1 - e;
            sm.stage[to / kStageEach * kStageStride + to % kStageEach] = e >= over ? load_logit<T>(part[j].w, e) : -INFINITY;
        }
    }
    __syncthreads();
    constexpr uint32_t kWeighs = 1u << 20;  // above every index
    // what entry j of thread `by` counts for in the walk: its weight, or, for a draw of 0, anything at all
    auto counts_for = [&](float l, uint32_t* bin) {
        if (!at_zero) return weight(l, bin);
        *bin = 0;
        return positive(l) ? uint64_t{1} : 0;
    };
    auto kept_at = [&](uint32_t by, uint32_t j, float l) {
        return l > -INFINITY && rank_key(l, first + kStageEach * by + j) >= cut;
    };
    const float floor_l = key_float(static_cast<uint32_t>(cut >> 32));  // (NaN for no cut: nothing lies below it)
    Halves sums{0, 0};
    uint32_t last = 0;
#pragma unroll 1
    for (uint32_t j = 0; j < kStageEach; ++j) {
        const float l = sm.stage[t * kStageStride + j];
        if (__ballot(l > -INFINITY && !(l < floor_l)) == 0) continue;
        const bool in = kept_at(t, j, l);
        uint32_t b;
        const uint64_t m = counts_for(l, &b);
        const Halves x = unit_halves(in ? m : 0, b);
        sums.lo += x.lo, sums.hi += x.hi;
        const uint32_t i = first + kStageEach * t + j;
        if (in) last = m != 0 ? (i + 1) | kWeighs : (last > kWeighs ? last : i + 1);
    }
    const u128 mine = join(sums);
    u128 run = mine;
    last = wave_reduce(last, 0u, [](uint32_t p, uint32_t q) { return p > q ? p : q; });
    if (lane == 0 && last != 0) atomicMax(&sm.last, last);
    u128 ignored;
    block_scan<kRowWaves>(n, run, &n_all, &ignored, sm.scan);
    const u128 start = run - mine;
    if (start <= rest && run > rest) sm.id = t, sm.want = rest - start;
    __syncthreads();
    // One thread's sixteen entries hold it: a lane to each. (The deepest bin's sum may exceed its entries' own by
    // their last bits: the last of them then.)
    static_assert(kStageEach == 16, "a row of lanes");
    if (t >= kStageEach) return;
    const bool found = sm.id != ~0u;
    const uint32_t end = (sm.last & (kWeighs - 1)) - 1, by = found ? sm.id : (end - first) / kStageEach;
    const uint32_t id = first + kStageEach * by + t;
    const float l = sm.stage[by * kStageStride + t];
    uint32_t b;
    const uint64_t m = counts_for(l, &b);
    Halves h = unit_halves(kept_at(by, t, l) ? m : 0, b);
    const u128 e = join(h);
    h.lo = row_incl_scan_u64(h.lo), h.hi = row_incl_scan_u64(h.hi);
    const u128 upto = join(h);
    if (found ? upto > sm.want && upto - e <= sm.want : id == end) {
        a.o.tokens[r] = id;
        if (a.o.logprobs) {
            uint64_t q = weight(l, &b);
            double p = 0.0;
            if (b == kTail) {  // a weight that has lost bits: from the logit, counted from the largest
                p = (static_cast<double>(l) - largest) / temp;
                q = weight(largest, &b);
            }
            p += log(to_double(unit(q, b)) / to_double(kept));
            a.o.logprobs[r] = static_cast<float>(p);
        }
        if (a.o.kept) a.o.kept[r] = static_cast<int32_t>(any ? st.count_l + sm.n : st.live);
    }
}
static_assert(kBins <= kRowThreads && kMaxSlices <= 64, "a thread to a bin, a lane to a slice");

template <typename T>
void launch(const SampleArgs& a, uint32_t rows, hipStream_t s) {
    const auto all = [&](auto tiny) {
        sample_slices_kernel<T, decltype(tiny)::value><<<dim3(a.slices, rows), kSliceThreads, 0, s>>>(a);
        sample_limits_kernel<<<rows, kRowThreads, 0, s>>>(a);
        sample_collect_kernel<T, decltype(tiny)::value><<<dim3(a.slices, rows), kSliceThreads, 0, s>>>(a);
        sample_finish_kernel<T, decltype(tiny)::value><<<rows, kRowThreads, sizeof(FinishMem), s>>>(a);
    };
    if (a.vocab < kVec<T>)
        all(std::true_type{});
    else
        all(std::false_type{});
}

}  // namespace

}  // namespace twd

struct twd_sampler {
    twd::StreamOrder order;
    twd::SamplerScratch scratch;
    void* block;  // the one allocation behind the scratch
    uint32_t max_vocab, max_rows;
    int device;
};

using namespace twd;

extern "C" {

TWD_API int twd_sampler_create(uint32_t max_vocab, uint32_t max_rows, twd_sampler** out) {
    clear_error();
    if (!out) return fail(TWD_E_INVALID, "null argument");
    *out = nullptr;
    if (max_vocab == 0 || max_vocab > 524288u) return fail(TWD_E_INVALID, "max_vocab must be in 1..524288");
    if (max_rows == 0 || max_rows > 4096u) return fail(TWD_E_INVALID, "max_rows must be in 1..4096");
    int dev = 0;
    TWD_HIP(hipGetDevice(&dev));
    twd_sampler* s = new (std::nothrow) twd_sampler{};
    if (!s) return fail(TWD_E_INVALID, "out of host memory");
    s->max_vocab = max_vocab, s->max_rows = max_rows, s->device = dev;
    const uint64_t slices = (max_vocab + kSlice - 1) / kSlice, rows = max_rows;
    const uint32_t cap = static_cast<uint32_t>(slices) * kSlice < kListCap ? static_cast<uint32_t>(slices) * kSlice : kListCap;
    const uint64_t bins = rows * slices * kBins * sizeof(uint64_t), list = rows * cap * sizeof(uint64_t);
    const uint64_t under = rows * slices * sizeof(u128), states = rows * sizeof(RowState);
    const uint64_t heads = rows * slices * sizeof(SliceHead);
    hipError_t e = hipSuccess;
    for (const void* f : {reinterpret_cast<const void*>(sample_finish_kernel<float, false>),
                          reinterpret_cast<const void*>(sample_finish_kernel<Bf16, false>),
                          reinterpret_cast<const void*>(sample_finish_kernel<Fp16, false>),
                          reinterpret_cast<const void*>(sample_finish_kernel<float, true>),
                          reinterpret_cast<const void*>(sample_finish_kernel<Bf16, true>),
                          reinterpret_cast<const void*>(sample_finish_kernel<Fp16, true>)})
        if (e == hipSuccess)
            e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(sizeof(FinishMem)));
    if (e == hipSuccess) e = hipMalloc(&s->block, bins + list + under + states + heads);
    if (e != hipSuccess) {
        delete s;
        return hip_fail(e, "allocating the sampler's scratch");
    }
    char* at = static_cast<char*>(s->block);
    s->scratch.bins = reinterpret_cast<uint64_t*>(at), at += bins;
    s->scratch.list = reinterpret_cast<uint64_t*>(at), at += list;
    s->scratch.under = reinterpret_cast<u128*>(at), at += under;
    s->scratch.state = reinterpret_cast<RowState*>(at), at += states;
    s->scratch.head = reinterpret_cast<SliceHead*>(at);
    s->scratch.slices = static_cast<uint32_t>(slices);
    s->scratch.list_cap = cap;
    *out = s;
    return TWD_OK;
}

TWD_API void twd_sampler_destroy(twd_sampler* s) {
    if (!s) return;
    order_release(s->order);
    (void)hipFree(s->block);
    delete s;
}

TWD_API int twd_sampler_sample(twd_sampler* sampler, const void* logits, int type, uint32_t vocab, uint32_t rows,
                               uint64_t row_stride, const float* temperature, const int32_t* top_k,
                               const float* top_p, const float* min_p, const float* uniform, uint32_t* tokens,
                               float* logprobs, int32_t* kept, void* stream) {
    clear_error();
    if (!sampler) return fail(TWD_E_INVALID, "null sampler");
    if (!logits || !uniform || !tokens) return fail(TWD_E_INVALID, "null logits, uniform or tokens");
    if (type != TWD_F32 && type != TWD_BF16 && type != TWD_F16)
        return fail(TWD_E_INVALID, "type must be TWD_F32, TWD_BF16 or TWD_F16");
    if (vocab == 0 || vocab > sampler->max_vocab) return fail(TWD_E_INVALID, "vocab out of range for this sampler");
    if (rows == 0 || rows > sampler->max_rows) return fail(TWD_E_INVALID, "rows out of range for this sampler");
    if (rows > 1 && row_stride < vocab) return fail(TWD_E_INVALID, "the row stride is below vocab");
    if (reinterpret_cast<uintptr_t>(logits) % (type == TWD_F32 ? 4 : 2) != 0)
        return fail(TWD_E_INVALID, "logits are not aligned to their type");
    int dev = 0;
    TWD_HIP(hipGetDevice(&dev));
    if (dev != sampler->device) return fail(TWD_E_INVALID, "the sampler lives on another device than the current one");
    const hipStream_t s = static_cast<hipStream_t>(stream);
    int rc = order_before(sampler->order, s);
    if (rc) return rc;
    const SampleArgs args{logits, row_stride, vocab, (vocab + kSlice - 1) / kSlice,
                          SampleParams{temperature, top_k, top_p, min_p, uniform}, SampleOut{tokens, logprobs, kept},
                          sampler->scratch, kWeightTable};
    if (type == TWD_F32)
        launch<float>(args, rows, s);
    else if (type == TWD_BF16)
        launch<Bf16>(args, rows, s);
    else
        launch<Fp16>(args, rows, s);
    const hipError_t e = hipGetLastError();
    rc = order_after(sampler->order, s);
    return e != hipSuccess ? hip_fail(e, "launching the sampler") : rc;
}

}  // extern "C"
