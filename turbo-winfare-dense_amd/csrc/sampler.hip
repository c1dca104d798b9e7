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
// 2^floor(z) times the fraction's power of two, rounded to 38 bits (2^-38 relative); sums are held in 128
// bits whose unit is 2^-78 of the largest weight's octave, so nothing above that is dropped. Every decision
// is then an exact comparison of integers, and equal logits have equal weights.
#include <hip/hip_runtime.h>

#include <cmath>
#include <new>

#include "twd_internal.h"
#include "twd_sampler.h"

namespace twd {

namespace {

typedef unsigned __int128 u128;

constexpr int kWeightBits = 38;  // a weight is 2^37 .. 2^38 times its octave
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

// 2^((j + 0.5) / 8 + 37), j = 0..7
__device__ __forceinline__ double eighth(uint32_t j) {
    constexpr double k[8] = {0x1.0b5586cf9890fp+37, 0x1.2387a6e756238p+37, 0x1.3dea64c123422p+37, 0x1.5ab07dd485429p+37,
                             0x1.7a11473eb0187p+37, 0x1.9c49182a3f090p+37, 0x1.c199bdd85529cp+37, 0x1.ea4afa2a490dap+37};
    return k[j];
}

// The weight's octave floor(z) and its eighth of it, both rising with l, and the weight's 38 bits.
struct Weight {
    double oct;
    uint32_t sub;
    uint64_t q;
};
__device__ __forceinline__ Weight weight_of(float l, const Scale& c) {
#pragma clang fp contract(off)
    // (contracted, zh - oct would be formed from the unrounded product, whose excess `rest` adds again)
    const double ld = l;
    const double zh = ld * c.hi;
    const double oct = __builtin_floor(zh);
    const double fr = zh - oct;
    uint32_t sub = static_cast<uint32_t>(fr * 8.0);
    sub = sub < 7u ? sub : 7u;
    // past 2^45 neighbouring floats lie more octaves apart than any sum holds, and z has no fraction left
    const bool far = !(__builtin_fabs(zh) < 0x1p45);
    const double rest = far ? 0.0 : fma(ld, c.hi, -zh) + ld * c.lo;
    // 2^((sub + 0.5) / 8) e^t with |t| <= ln2 / 16, by its degree-6 Taylor polynomial (6e-14 relative)
    const double t = (fr - (static_cast<double>(sub) * 0.125 + 0.0625) + rest) * 0.6931471805599453;
    double p = fma(t, 1.0 / 720.0, 1.0 / 120.0);
    p = fma(t, p, 1.0 / 24.0);
    p = fma(t, p, 1.0 / 6.0);
    p = fma(t, p, 0.5);
    p = fma(t, p, 1.0);
    p = fma(t, p, 1.0);
    Weight w;
    w.oct = oct;
    w.sub = sub;
    // + 2^52 leaves the nearest integer in the low mantissa bits
    w.q = __builtin_bit_cast(uint64_t, eighth(sub) * p + 0x1p52) & 0xFFFFFFFFFFFFFull;
    return w;
}

// The weight in units of the row's sums, `top` being the octave of the largest.
__device__ __forceinline__ u128 in_sum(const Weight& w, double top) {
    const double down = top - w.oct;
    if (!(down < 80.0)) return 0;
    return (static_cast<u128>(w.q) << kSumShift) >> static_cast<int>(down);
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
struct Bf16 {};
struct Fp16 {};
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
//   slices   every slice of 4,096 entries: its largest rank, and its entries' numbers and weights by bin
//   limits   per row: the slices' bins added up, and the bins in which the limits cut
//   collect  every slice: its entries in those bins, onto the row's list
//   finish   per row: the list in order, the cuts, and the draw
//
// A bin is an eighth of an octave of weight. A slice counts from its own largest octave down (its row's is
// not known yet), 256 bins to a slice, the last one for all that lies deeper; octaves are absolute, so the
// slices' bins line up. A bin's entries share an octave, so its sum of 38-bit weights is one integer; the
// last bin's are brought to its octave (2^-31 of the largest) first.
constexpr uint32_t kSlice = 4096;
constexpr uint32_t kBins = 256;
constexpr uint32_t kTail = kBins - 1;
constexpr uint32_t kTailOct = kTail >> 3;
constexpr uint32_t kListCap = 4096;
constexpr uint32_t kMaxSlices = 524288 / kSlice;
// A bin of a slice: entries above bit 51, the sum of their weights (at most 4096 * 2^38 and a little) below.
constexpr int kCountBit = 51;
constexpr uint64_t kMassMask = (1ull << kCountBit) - 1;

struct SliceHead {
    uint64_t best;  // largest rank of the live entries (0: none)
    uint32_t live;
    uint32_t bad;   // a NaN or +inf was seen
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
    uint32_t listed;    // entries in the deciding bins
    uint32_t appended;  // of these, on the list so far
};

struct SamplerScratch {
    uint64_t* bins;   // [rows][slices][kBins]
    SliceHead* head;  // [rows][slices]
    RowState* state;  // [rows]
    uint64_t* list;   // [rows][kListCap] ranks
    u128* sums;       // [rows][kBins] sum of the weights up to a bin
    uint32_t* counts; // [rows][kBins]
    uint32_t slices;  // of max_vocab
};

struct SampleArgs {
    const void* logits;
    uint64_t stride;
    uint32_t vocab, slices;
    SampleParams p;
    SampleOut o;
    SamplerScratch s;
};

// 16 bytes of logits from any address (the hardware splits an unaligned load itself).
template <typename T>
constexpr uint32_t kVec = 16 / kLogitBytes<T>;
template <typename T>
__device__ __forceinline__ void load_vec(const void* row, uint32_t i, uint32_t vocab, float* v) {
    if (i + kVec<T> <= vocab) {
        uint32_t w[4];
        __builtin_memcpy(w, static_cast<const char*>(row) + static_cast<uint64_t>(i) * kLogitBytes<T>, 16);
#pragma unroll
        for (uint32_t j = 0; j < kVec<T>; ++j) v[j] = load_logit<T>(w, j);
    } else {
#pragma unroll
        for (uint32_t j = 0; j < kVec<T>; ++j) v[j] = i + j < vocab ? load_logit<T>(row, i + j) : -INFINITY;
    }
}

// The bin of a weight counted from octave `top`, and its integer in that bin.
__device__ __forceinline__ uint32_t bin_of(const Weight& w, double top) {
    const double down = top - w.oct;
    if (!(down < static_cast<double>(kTailOct + 1))) return kTail;
    return (static_cast<uint32_t>(down) << 3) + 7u - w.sub;
}
__device__ __forceinline__ uint64_t mass_of(const Weight& w, uint32_t bin, double top) {
    if (bin != kTail) return w.q;
    const double deep = top - w.oct - static_cast<double>(kTailOct);
    return deep < 64.0 ? w.q >> static_cast<int>(deep) : 0;
}
// A bin's integer in units of the row's sums.
__device__ __forceinline__ u128 unit(uint64_t mass, uint32_t bin) {
    return (static_cast<u128>(mass) << kSumShift) >> (bin >> 3);
}

__device__ __forceinline__ u128 shfl_up_u128(u128 v, int d) {
    uint64_t lo = static_cast<uint64_t>(v), hi = static_cast<uint64_t>(v >> 64);
    lo = static_cast<uint64_t>(__shfl_up(static_cast<unsigned long long>(lo), d));
    hi = static_cast<uint64_t>(__shfl_up(static_cast<unsigned long long>(hi), d));
    return static_cast<u128>(hi) << 64 | lo;
}

constexpr uint32_t kRowThreads = 1024;
constexpr uint32_t kRowWaves = kRowThreads / 64;

// Running sums over the block's threads (each includes its own), and the total. All threads call.
struct ScanMem {
    u128 w[kRowWaves];
    uint32_t n[kRowWaves];
};
__device__ __forceinline__ void block_scan(uint32_t& n, u128& w, uint32_t* n_all, u128* w_all, ScanMem& mem) {
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    n = wave_incl_scan_u32(n);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const u128 o = shfl_up_u128(w, d);
        if (lane >= static_cast<uint32_t>(d)) w += o;
    }
    __syncthreads();
    if (lane == 63) mem.n[wave] = n, mem.w[wave] = w;
    __syncthreads();
    uint32_t nb = 0, na = 0;
    u128 wb = 0, wa = 0;
    for (uint32_t i = 0; i < kRowWaves; ++i) {
        if (i == wave) nb = na, wb = wa;
        na += mem.n[i], wa += mem.w[i];
    }
    n += nb, w += wb;
    *n_all = na, *w_all = wa;
}

constexpr uint32_t kSliceThreads = 256;

template <typename T>
__global__ __launch_bounds__(kSliceThreads) void sample_slices_kernel(SampleArgs a) {
    __shared__ uint64_t bins[kBins];
    __shared__ uint64_t s_best[kSliceThreads / 64];
    __shared__ uint32_t s_live[kSliceThreads / 64], s_bad[kSliceThreads / 64];
    const uint32_t t = threadIdx.x, slice = blockIdx.x, lane = t % 64, wave = t / 64;
    const uint64_t r = blockIdx.y;
    const void* row = static_cast<const char*>(a.logits) + r * a.stride * kLogitBytes<T>;
    constexpr uint32_t kLoads = kSlice / kSliceThreads / kVec<T>;
    float v[kLoads * kVec<T>];
    const uint32_t i0 = slice * kSlice + t * kVec<T>;
#pragma unroll
    for (uint32_t j = 0; j < kLoads; ++j)
        load_vec<T>(row, i0 + j * kSliceThreads * kVec<T>, a.vocab, v + j * kVec<T>);
    bins[t] = 0;
    uint64_t best = 0;
    uint32_t live = 0, bad = 0;
#pragma unroll
    for (uint32_t j = 0; j < kLoads * kVec<T>; ++j) {
        bad |= v[j] < INFINITY ? 0u : 1u;
        if (v[j] > -INFINITY) {
            ++live;
            const uint64_t k = rank_key(v[j], i0 + (j / kVec<T>) * kSliceThreads * kVec<T> + j % kVec<T>);
            best = k > best ? k : best;
        }
    }
    best = wave_max_u64(best);
    live = wave_reduce(live, 0u, [](uint32_t x, uint32_t y) { return x + y; });
    bad = wave_reduce(bad, 0u, [](uint32_t x, uint32_t y) { return x | y; });
    if (lane == 0) s_best[wave] = best, s_live[wave] = live, s_bad[wave] = bad;
    __syncthreads();
    live = 0;
#pragma unroll
    for (uint32_t i = 0; i < kSliceThreads / 64; ++i) {
        best = s_best[i] > best ? s_best[i] : best;
        live += s_live[i], bad |= s_bad[i];
    }
    const uint64_t at = r * a.s.slices + slice;
    if (t == 0) a.s.head[at] = SliceHead{best, live, bad};
    const float temp = a.p.temperature ? a.p.temperature[r] : 1.0f;
    if (live == 0 || !(temp > 0.0f)) return;
    const Scale c = scale_of(temp);
    const double top = weight_of(rank_value(best), c).oct;
#pragma unroll
    for (uint32_t j = 0; j < kLoads * kVec<T>; ++j) {
        if (v[j] > -INFINITY && v[j] < INFINITY) {
            const Weight w = weight_of(v[j], c);
            const uint32_t b = bin_of(w, top);
            atomicAdd(reinterpret_cast<unsigned long long*>(&bins[b]),
                      static_cast<unsigned long long>(1ull << kCountBit | mass_of(w, b, top)));
        }
    }
    __syncthreads();
    a.s.bins[at * kBins + t] = bins[t];
}
static_assert(kBins == kSliceThreads, "a bin per thread");

// The row's bin of a slice's bin, `shift` octaves under the row's largest, and what to shift its sum by.
__device__ __forceinline__ uint32_t row_bin(uint32_t b, uint32_t shift, uint32_t* down) {
    const uint32_t x = b + 8 * shift;
    *down = 0;
    if (x < kTail && b != kTail) return x;
    *down = (b >> 3) + shift - kTailOct;
    return kTail;
}
__device__ __forceinline__ uint32_t slice_shift(double top, double slice_top) {
    const double d = top - slice_top;
    return d < 128.0 ? static_cast<uint32_t>(d) : 128u;
}

// The next float below and above (the key under 0's is -0's, which float_key takes for 0).
__device__ __forceinline__ float float_below(float l) {
    const uint32_t k = float_key(l);
    return key_float(k == 0x80000000u ? k - 2 : k - 1);
}
__device__ __forceinline__ float float_above(float l) {
    const uint32_t k = float_key(l) + 1;
    return key_float(k == 0x7FFFFFFFu ? k + 1 : k);
}

// The least rank that min-p keeps: (l - M) log2(e) / T >= log2(min_p); the best one where none does.
__device__ uint64_t least_kept(uint64_t best, float min_p, const Scale& c) {
    const float m = rank_value(best);
    const double lim = log2(static_cast<double>(min_p));
    auto keeps = [&](float l) { return (static_cast<double>(l) - static_cast<double>(m)) * c.hi >= lim; };
    if (!keeps(m)) return best;
    if (c.hi == 0.0) return static_cast<uint64_t>(float_key(-INFINITY)) << 32;
    float l = static_cast<float>(static_cast<double>(m) + lim / c.hi);
    l = l < m ? l : m;
    // the quotient and the sum are rounded, the float once more: a few steps at most
    for (int i = 0; i < 8 && l > -INFINITY && keeps(float_below(l)); ++i) l = float_below(l);
    for (int i = 0; i < 8 && l < m && !keeps(l); ++i) l = float_above(l);
    return static_cast<uint64_t>(float_key(l)) << 32;
}

__global__ __launch_bounds__(kRowThreads) void sample_limits_kernel(SampleArgs a) {
    __shared__ unsigned long long mass[kBins];
    __shared__ uint32_t count[kBins];
    __shared__ u128 sums[kBins];
    __shared__ uint32_t counts[kBins];
    __shared__ unsigned long long s_best;
    __shared__ uint32_t s_live, s_bad, found[3];
    __shared__ uint8_t shift[kMaxSlices];
    __shared__ ScanMem scan;
    const uint32_t t = threadIdx.x;
    const uint64_t r = blockIdx.x;
    if (t == 0) s_best = 0, s_live = 0, s_bad = 0;
    if (t < kBins) mass[t] = 0, count[t] = 0;
    if (t < 3) found[t] = kBins;
    __syncthreads();
    const SliceHead* head = a.s.head + r * a.s.slices;
    SliceHead mine{0, 0, 0};
    if (t < a.slices) {
        mine = head[t];
        atomicMax(&s_best, static_cast<unsigned long long>(mine.best));
        atomicAdd(&s_live, mine.live);
        atomicOr(&s_bad, mine.bad);
    }
    __syncthreads();
    const float temp = a.p.temperature ? a.p.temperature[r] : 1.0f, u = a.p.uniform[r];
    const float top_p = a.p.top_p ? a.p.top_p[r] : 1.0f, min_p = a.p.min_p ? a.p.min_p[r] : 0.0f;
    const int32_t top_k = a.p.top_k ? a.p.top_k[r] : 0;
    const uint64_t best = s_best;
    const uint32_t live = s_live;
    const bool none = s_bad != 0 || live == 0 || temp != temp || u != u || top_p != top_p || min_p != min_p;
    if (none || temp <= 0.0f) {
        if (t == 0) {
            a.s.state[r].done = 1;
            a.s.state[r].lo = 1, a.s.state[r].hi = 0, a.s.state[r].bin_k = kBins, a.s.state[r].listed = 0;
            a.o.tokens[r] = none ? TWD_TOKEN_DEGENERATE : rank_index(best);
            if (a.o.logprobs) a.o.logprobs[r] = none ? __uint_as_float(0x7FC00000u) : 0.0f;
            if (a.o.kept) a.o.kept[r] = none ? 0 : 1;
        }
        return;
    }
    const Scale c = scale_of(temp);
    const float m = rank_value(best);
    const double top = weight_of(m, c).oct;
    if (t < a.slices)
        shift[t] = static_cast<uint8_t>(mine.live ? slice_shift(top, weight_of(rank_value(mine.best), c).oct) : 255u);
    __syncthreads();
    const uint64_t* bins = a.s.bins + r * a.s.slices * kBins;
    for (uint32_t i = t; i < a.slices * kBins; i += kRowThreads) {
        const uint32_t sh = shift[i / kBins];
        if (sh == 255u) continue;  // an empty slice writes no bins
        const uint64_t x = bins[i];
        if (x == 0) continue;
        uint32_t down;
        const uint32_t b = row_bin(i % kBins, sh, &down);
        atomicAdd(&mass[b], static_cast<unsigned long long>(down < 64 ? (x & kMassMask) >> down : 0));
        atomicAdd(&count[b], static_cast<uint32_t>(x >> kCountBit));
    }
    __syncthreads();
    uint32_t n = t < kBins ? count[t] : 0, n_all;
    u128 w = t < kBins ? unit(mass[t], t) : 0, w_all;
    block_scan(n, w, &n_all, &w_all, scan);
    if (t < kBins) counts[t] = n, sums[t] = w;
    if (t < kBins) a.s.counts[r * kBins + t] = n, a.s.sums[r * kBins + t] = w;
    __syncthreads();
    // the bin each limit cuts in: the first whose running number or sum reaches it
    const uint32_t k = top_k > 0 && static_cast<uint32_t>(top_k) < live ? static_cast<uint32_t>(top_k) : 0;
    if (t < kBins && k != 0 && counts[t] >= k && (t == 0 || counts[t - 1] < k)) found[0] = t;
    __syncthreads();
    const uint32_t bin_k = found[0];
    const bool use_p = top_p < 1.0f;
    if (use_p && t < kBins) {
        // the top-k's sum lies between those of the bins under and with its cut
        const u128 low = part_of(top_p, k ? (bin_k ? sums[bin_k - 1] : 0) : w_all, true);
        const u128 high = part_of(top_p, k ? sums[bin_k] : w_all, true);
        auto reaches = [&](uint32_t b, u128 x) { return counts[b] >= 1 && sums[b] >= x; };
        if (reaches(t, low) && (t == 0 || !reaches(t - 1, low))) found[1] = t;
        if (reaches(t, high) && (t == 0 || !reaches(t - 1, high))) found[2] = t;
    }
    __syncthreads();
    if (t != 0) return;
    RowState st{};
    uint32_t lo = kBins, hi = kBins;
    if (use_p)
        lo = found[1], hi = found[2];
    else if (k)
        lo = hi = bin_k;
    bool need_k = use_p && k;
    if (min_p > 0.0f) {
        st.rank_m = least_kept(best, min_p, c);
        const float l = rank_value(st.rank_m);
        const uint32_t b = l > -INFINITY ? bin_of(weight_of(l, c), top) : kBins;
        if (b < lo) lo = hi = b, need_k = false;  // the other limits cut deeper
        if (b < hi) hi = b;
    }
    st.top = top, st.best = best, st.all = w_all, st.live = live, st.k = k, st.use_p = use_p;
    st.bin_k = need_k ? bin_k : kBins;
    if (lo < kBins) {
        st.lo = lo, st.hi = hi;
        st.below_l = lo ? sums[lo - 1] : 0, st.count_l = lo ? counts[lo - 1] : 0;
        st.listed = counts[hi] - st.count_l;
    } else {
        st.lo = 1, st.hi = 0;
    }
    if (need_k) {
        st.below_k = bin_k ? sums[bin_k - 1] : 0, st.count_k = bin_k ? counts[bin_k - 1] : 0;
        if (bin_k > hi) st.listed += counts[bin_k] - st.count_k;
    }
    a.s.state[r] = st;
}

template <typename T>
__global__ __launch_bounds__(kSliceThreads) void sample_collect_kernel(SampleArgs a) {
    __shared__ uint32_t s_n, s_base, s_any;
    __shared__ uint64_t s_rank[kSlice];
    const uint32_t t = threadIdx.x, slice = blockIdx.x;
    const uint64_t r = blockIdx.y;
    RowState* st = a.s.state + r;
    const uint32_t lo = st->lo, hi = st->hi, bin_k = st->bin_k;
    if (st->listed == 0 || st->listed > kListCap) return;
    const SliceHead h = a.s.head[r * a.s.slices + slice];
    if (h.live == 0) return;
    const Scale c = scale_of(a.p.temperature ? a.p.temperature[r] : 1.0f);
    const double top = st->top;
    const uint32_t sh = slice_shift(top, weight_of(rank_value(h.best), c).oct);
    if (t == 0) s_n = 0, s_any = 0;
    __syncthreads();
    uint32_t down;
    const uint32_t b = row_bin(t, sh, &down);
    if (((b >= lo && b <= hi) || b == bin_k) && a.s.bins[(r * a.s.slices + slice) * kBins + t] != 0) s_any = 1;
    __syncthreads();
    if (!s_any) return;
    const void* row = static_cast<const char*>(a.logits) + r * a.stride * kLogitBytes<T>;
    constexpr uint32_t kLoads = kSlice / kSliceThreads / kVec<T>;
    const uint32_t i0 = slice * kSlice + t * kVec<T>;
#pragma unroll
    for (uint32_t j = 0; j < kLoads; ++j) {
        float v[kVec<T>];
        const uint32_t i = i0 + j * kSliceThreads * kVec<T>;
        load_vec<T>(row, i, a.vocab, v);
#pragma unroll
        for (uint32_t e = 0; e < kVec<T>; ++e) {
            if (v[e] > -INFINITY) {
                const uint32_t x = bin_of(weight_of(v[e], c), top);
                if ((x >= lo && x <= hi) || x == bin_k) s_rank[atomicAdd(&s_n, 1u)] = rank_key(v[e], i + e);
            }
        }
    }
    __syncthreads();
    if (t == 0) s_base = atomicAdd(&st->appended, s_n);
    __syncthreads();
    // the bins' own numbers say how many come: the list holds them all
    for (uint32_t i = t; i < s_n; i += kSliceThreads)
        if (s_base + i < kListCap) a.s.list[r * kListCap + s_base + i] = s_rank[i];
}

// Ranks in falling order, n <= kListCap, through LDS. A few are placed by counting the larger ones.
__device__ void sort_ranks(uint64_t* x, uint32_t n) {
    const uint32_t t = threadIdx.x;
    if (n <= 256) {
        uint64_t mine = 0;
        uint32_t pos = 0;
        const uint32_t e = t / 4, part = t % 4;
        if (e < n) {
            mine = x[e];
            for (uint32_t i = part; i < n; i += 4) pos += x[i] > mine ? 1u : 0u;
        }
        pos += __shfl_xor(pos, 1);
        pos += __shfl_xor(pos, 2);
        __syncthreads();
        if (e < n && part == 0) x[pos] = mine;
        __syncthreads();
        return;
    }
    uint32_t size = 512;
    while (size < n) size *= 2;
    for (uint32_t i = n + t; i < size; i += kRowThreads) x[i] = 0;
    for (uint32_t len = 2; len <= size; len *= 2) {
        for (uint32_t step = len / 2; step > 0; step /= 2) {
            __syncthreads();
            for (uint32_t i = t; i < size / 2; i += kRowThreads) {
                const uint32_t p = 2 * i - (i & (step - 1)), q = p + step;
                const uint64_t u = x[p], v = x[q];
                if (((p & len) == 0) == (u < v)) x[p] = v, x[q] = u;
            }
        }
    }
    __syncthreads();
}

struct FinishMem {
    uint64_t rank[kListCap];
    ScanMem scan;
    u128 slice[kMaxSlices];
    unsigned long long in_slice[kMaxSlices];
    uint32_t digit_n[kBins];
    unsigned long long digit_w[kBins];
    uint64_t cut, cut2;
    u128 sum, want;
    uint32_t n, pick, id, last;
};

template <typename T>
__global__ __launch_bounds__(kRowThreads) void sample_finish_kernel(SampleArgs a) {
    __shared__ FinishMem sm;
    const uint32_t t = threadIdx.x;
    const uint64_t r = blockIdx.x;
    const RowState& st = a.s.state[r];
    if (st.done) return;
    const void* row = static_cast<const char*>(a.logits) + r * a.stride * kLogitBytes<T>;
    const float temp = a.p.temperature ? a.p.temperature[r] : 1.0f, u = a.p.uniform[r];
    const float top_p = a.p.top_p ? a.p.top_p[r] : 1.0f;
    const Scale c = scale_of(temp);
    const double top = st.top;
    const uint32_t lo = st.lo, hi = st.hi, listed = st.listed;
    const bool on_list = listed <= kListCap;
    auto weight = [&](float l, uint32_t* bin) {
        const Weight w = weight_of(l, c);
        *bin = bin_of(w, top);
        return mass_of(w, *bin, top);
    };
    // f(rank, bin, mass) of every entry in the row's bins b0 .. b1
    auto members = [&](uint32_t b0, uint32_t b1, auto f) {
        if (on_list) {
            for (uint32_t i = t; i < listed; i += kRowThreads) {
                uint32_t b;
                const uint64_t m = weight(rank_value(sm.rank[i]), &b);
                if (b >= b0 && b <= b1) f(sm.rank[i], b, m);
            }
        } else {
            for (uint32_t i = t; i < a.vocab; i += kRowThreads) {
                const float l = load_logit<T>(row, i);
                if (!(l > -INFINITY)) continue;
                uint32_t b;
                const uint64_t m = weight(l, &b);
                if (b >= b0 && b <= b1) f(rank_key(l, i), b, m);
            }
        }
    };
    // In one bin, by digits of the rank from the top: the largest rank such that the entries of at least
    // it number `n` or weigh `w` (whichever `by_sum` says; all of them where they do not reach that).
    // Returns it, and the weight of those entries.
    auto select = [&](uint32_t bin, uint32_t n, u128 w, bool by_sum, u128* sum) {
        uint64_t prefix = 0;
        uint32_t n_done = 0;
        u128 w_done = 0;
        for (int sft = 56; sft >= 0; sft -= 8) {
            __syncthreads();
            if (t < kBins) sm.digit_n[t] = 0, sm.digit_w[t] = 0;
            if (t == 0) sm.pick = 0;
            __syncthreads();
            members(bin, bin, [&](uint64_t k, uint32_t, uint64_t m) {
                if (sft < 56 && (k >> (sft + 8)) != (prefix >> (sft + 8))) return;
                const uint32_t d = 255u - (static_cast<uint32_t>(k >> sft) & 255u);
                atomicAdd(&sm.digit_n[d], 1u);
                atomicAdd(&sm.digit_w[d], static_cast<unsigned long long>(m));
            });
            __syncthreads();
            uint32_t x = t < kBins ? sm.digit_n[t] : 0, x_all;
            const uint32_t own = x;
            u128 y = t < kBins ? unit(sm.digit_w[t], bin) : 0, y_all;
            const u128 own_w = y;
            block_scan(x, y, &x_all, &y_all, sm.scan);
            // the digit at which the running number or sum reaches the target, or the last one there is
            const bool here = own != 0 && (by_sum ? w_done + y >= w && w_done + y - own_w < w
                                                  : n_done + x >= n && n_done + x - own < n);
            const bool end = own != 0 && x == x_all && (by_sum ? w_done + y < w : n_done + x < n);
            const bool first = by_sum && w <= w_done && own != 0 && x == own;
            if (here || end || first) sm.pick = t, sm.n = n_done + x - own, sm.sum = w_done + y - own_w;
            __syncthreads();
            prefix |= static_cast<uint64_t>(255u - sm.pick) << sft;
            n_done = sm.n, w_done = sm.sum;
            if (sft == 0) w_done += unit(sm.digit_w[sm.pick], bin);
        }
        __syncthreads();
        *sum = w_done;
        return prefix;
    };

    uint64_t cut = 0;  // ranks of at least this are kept
    if (on_list && listed != 0) {
        for (uint32_t i = t; i < listed; i += kRowThreads) sm.rank[i] = a.s.list[r * kListCap + i];
        __syncthreads();
        sort_ranks(sm.rank, listed);
        // running sums along the list, four entries to a thread; lo .. hi come first, bin_k after them or
        // among them
        constexpr uint32_t kEach = kListCap / kRowThreads;
        uint32_t bin[kEach], n = 0, n_all;
        u128 w[kEach], run = 0, w_all;
#pragma unroll
        for (uint32_t j = 0; j < kEach; ++j) {
            const uint32_t i = kEach * t + j;
            bin[j] = kBins + 1, w[j] = 0;
            if (i < listed) {
                const uint64_t m = weight(rank_value(sm.rank[i]), &bin[j]);
                w[j] = unit(m, bin[j]);
            }
            run += w[j];
            n += i < listed && bin[j] < st.bin_k ? 1u : 0u;
        }
        const u128 own = run;
        uint32_t n_before = n;
        block_scan(n_before, run, &n_all, &w_all, sm.scan);
        if (t == 0) sm.cut = 0, sm.cut2 = 0, sm.sum = st.all, sm.want = 0;
        __syncthreads();
        u128 before = run - own;
        if (st.use_p) {
            if (st.bin_k < kBins) {
                // the top-k's last entry is number k - count_k of its bin; the sum under that bin is known,
                // and the list's own sum where the bin begins
                const uint32_t at = n_all + (st.k - st.count_k) - 1;
                u128 x = before;
#pragma unroll
                for (uint32_t j = 0; j < kEach; ++j) {
                    const uint32_t i = kEach * t + j;
                    if (i == n_all) sm.want = x;
                    x += w[j];
                    if (i == at) sm.cut = sm.rank[i], sm.sum = x;
                }
                __syncthreads();
                if (t == 0) sm.sum = st.below_k + (sm.sum - sm.want);
                __syncthreads();
            }
            const u128 want = part_of(top_p, sm.sum, true);
            u128 x = st.below_l + before;
#pragma unroll
            for (uint32_t j = 0; j < kEach; ++j) {
                const uint32_t i = kEach * t + j;
                const bool in = i < listed && bin[j] >= lo && bin[j] <= hi;
                const u128 y = x + w[j];
                // the entry that reaches the target; the first one where none is needed
                if (in && ((y >= want && x < want) || (i == 0 && want <= x))) sm.cut2 = sm.rank[i];
                x = y;
            }
            __syncthreads();
            cut = sm.cut > sm.cut2 ? sm.cut : sm.cut2;
        } else if (st.k != 0 && st.count_l < st.k && st.k - st.count_l <= listed) {
            cut = sm.rank[st.k - st.count_l - 1];
        }
    } else if (listed != 0) {
        // more entries than the list holds: equal or nearly equal logits. The row itself is read for each digit.
        u128 sum = st.all;
        const u128* sums = a.s.sums + r * kBins;
        const uint32_t* counts = a.s.counts + r * kBins;
        uint64_t cut_k = 0;
        if (st.use_p && st.bin_k < kBins) {
            cut_k = select(st.bin_k, st.k - st.count_k, 0, false, &sum);
            sum += st.below_k;
        } else if (!st.use_p && st.k != 0 && st.count_l < st.k && counts[hi] >= st.k) {
            cut_k = select(lo, st.k - st.count_l, 0, false, &sum);
        }
        cut = cut_k;
        if (st.use_p) {
            const u128 want = part_of(top_p, sum, true);
            uint32_t b = lo;
            while (b < hi && !(counts[b] >= 1 && sums[b] >= want)) ++b;
            const u128 under = b ? sums[b - 1] : 0;
            // (not reached: min-p cuts before)
            if (counts[b] >= 1 && (sums[b] >= want || b == kTail)) {
                const uint64_t x = select(b, 0, want > under ? want - under : 0, true, &sum);
                cut = x > cut ? x : cut;
            }
        }
    }
    cut = st.rank_m > cut ? st.rank_m : cut;

    // ---- the draw: kept weights by slice, then through the slice
    const bool all = lo > hi;
    // every entry in bins under `full` is kept, and of bin `full` those that reach the cut
    uint32_t full = kBins;
    if (!all) weight(rank_value(cut), &full);
    __syncthreads();
    if (t < kMaxSlices) sm.in_slice[t] = 0, sm.slice[t] = 0;
    if (t == 0) sm.n = 0;
    __syncthreads();
    if (!all) {
        members(full, full, [&](uint64_t k, uint32_t, uint64_t m) {
            if (k < cut) return;
            atomicAdd(&sm.in_slice[rank_index(k) / kSlice], static_cast<unsigned long long>(m));
            atomicAdd(&sm.n, 1u);
        });
    }
    __syncthreads();
    const SliceHead* head = a.s.head + r * a.s.slices;
    const uint64_t* bins = a.s.bins + r * a.s.slices * kBins;
    for (uint32_t s0 = t / 64; s0 < a.slices; s0 += kRowWaves) {  // a wave per slice, four bins a lane
        const SliceHead h = head[s0];
        u128 w = 0;
        if (h.live != 0) {
            const uint32_t sh = slice_shift(top, weight_of(rank_value(h.best), c).oct);
#pragma unroll
            for (uint32_t j = 0; j < kBins / 64; ++j) {
                uint32_t down;
                const uint32_t b = row_bin(64 * j + t % 64, sh, &down);
                if (b < full) {
                    const uint64_t x = bins[s0 * kBins + 64 * j + t % 64];
                    w += unit(down < 64 ? (x & kMassMask) >> down : 0, b);
                }
            }
        }
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const u128 o = shfl_up_u128(w, d);
            if (t % 64 >= static_cast<uint32_t>(d)) w += o;
        }
        if (t % 64 == 63) sm.slice[s0] = w + (all ? 0 : unit(sm.in_slice[s0], full));
    }
    __syncthreads();
    uint32_t n = 0, n_all;
    u128 w = t < a.slices ? sm.slice[t] : 0, kept;
    const u128 own = w;
    block_scan(n, w, &n_all, &kept, sm.scan);
    const u128 want = u < 1.0f ? part_of(u, kept, false) : kept - 1;  // the first running sum past this is drawn
    if (w > want && w - own <= want) sm.pick = t, sm.want = want - (w - own);
    if (t == 0) sm.last = 0, sm.id = ~0u;
    __syncthreads();
    const uint32_t slice = sm.pick;
    const u128 rest = sm.want;
    constexpr uint32_t kEach = kSlice / kRowThreads;
    u128 e[kEach], run = 0, sum;
    const uint32_t i0 = slice * kSlice + kEach * t;
    uint32_t last = 0;
#pragma unroll
    for (uint32_t j = 0; j < kEach; ++j) {
        e[j] = 0;
        if (i0 + j < a.vocab) {
            const float l = load_logit<T>(row, i0 + j);
            if (l > -INFINITY && rank_key(l, i0 + j) >= cut) {
                uint32_t b;
                const uint64_t m = weight(l, &b);
                e[j] = unit(m, b);
                if (e[j] != 0) last = i0 + j + 1;
            }
        }
        run += e[j];
    }
    const u128 mine = run;
    if (last) atomicMax(&sm.last, last);
    block_scan(n, run, &n_all, &sum, sm.scan);
    u128 x = run - mine;
#pragma unroll
    for (uint32_t j = 0; j < kEach; ++j) {
        if (x <= rest && x + e[j] > rest) sm.id = i0 + j;
        x += e[j];
    }
    __syncthreads();
    if (t == 0) {
        // (the deepest bin's sum may exceed its entries' own by their last bits: the last of them then)
        const uint32_t id = sm.id != ~0u ? sm.id : sm.last - 1;
        a.o.tokens[r] = id;
        uint32_t b;
        const uint64_t m = weight(load_logit<T>(row, id), &b);
        if (a.o.logprobs) a.o.logprobs[r] = static_cast<float>(log(to_double(unit(m, b)) / to_double(kept)));
        if (a.o.kept) a.o.kept[r] = static_cast<int32_t>(all ? st.live : (full ? a.s.counts[r * kBins + full - 1] : 0) + sm.n);
    }
}

template <typename T>
void launch(const SampleArgs& a, uint32_t rows, hipStream_t s) {
    const dim3 grid(a.slices, rows);
    sample_slices_kernel<T><<<grid, kSliceThreads, 0, s>>>(a);
    sample_limits_kernel<<<rows, kRowThreads, 0, s>>>(a);
    sample_collect_kernel<T><<<grid, kSliceThreads, 0, s>>>(a);
    sample_finish_kernel<T><<<rows, kRowThreads, 0, s>>>(a);
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
    const uint64_t bins = rows * slices * kBins * sizeof(uint64_t), list = rows * kListCap * sizeof(uint64_t);
    const uint64_t sums = rows * kBins * sizeof(u128), states = (rows * sizeof(RowState) + 255) / 256 * 256;
    const uint64_t heads = rows * slices * sizeof(SliceHead), counts = rows * kBins * sizeof(uint32_t);
    const hipError_t e = hipMalloc(&s->block, bins + list + sums + states + heads + counts);
    if (e != hipSuccess) {
        delete s;
        return hip_fail(e, "allocating the sampler's scratch");
    }
    char* at = static_cast<char*>(s->block);
    s->scratch.bins = reinterpret_cast<uint64_t*>(at), at += bins;
    s->scratch.list = reinterpret_cast<uint64_t*>(at), at += list;
    s->scratch.sums = reinterpret_cast<u128*>(at), at += sums;
    s->scratch.state = reinterpret_cast<RowState*>(at), at += states;
    s->scratch.head = reinterpret_cast<SliceHead*>(at), at += heads;
    s->scratch.counts = reinterpret_cast<uint32_t*>(at);
    s->scratch.slices = static_cast<uint32_t>(slices);
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
                          sampler->scratch};
    if (type == TWD_F32)
        launch<float>(args, rows, s);
    else if (type == TWD_BF16)
        launch<Bf16>(args, rows, s);
    else
        launch<Fp16>(args, rows, s);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return hip_fail(e, "launching the sampler");
    return order_after(sampler->order, s);
}

}  // extern "C"
