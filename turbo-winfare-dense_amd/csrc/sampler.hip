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
    s.lo = t > 3.5e38f ? 0.0 : (fma(-s.hi, td, kHi) + kLo) / td;  // an infinite T: every weight alike
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

constexpr uint32_t kSimpleThreads = 1024;

// Block-wide sum of (count, weight), returned to every thread.
struct Sum {
    uint32_t n;
    u128 w;
};
__device__ Sum block_sum(Sum v, uint32_t* sn, uint64_t* slo, uint64_t* shi) {
    const uint32_t t = threadIdx.x;
    __syncthreads();
    sn[t] = v.n, slo[t] = static_cast<uint64_t>(v.w), shi[t] = static_cast<uint64_t>(v.w >> 64);
    for (uint32_t s = kSimpleThreads / 2; s > 0; s /= 2) {
        __syncthreads();
        if (t < s) {
            const u128 a = (static_cast<u128>(shi[t]) << 64 | slo[t]) + (static_cast<u128>(shi[t + s]) << 64 | slo[t + s]);
            sn[t] += sn[t + s], slo[t] = static_cast<uint64_t>(a), shi[t] = static_cast<uint64_t>(a >> 64);
        }
    }
    __syncthreads();
    return Sum{sn[0], static_cast<u128>(shi[0]) << 64 | slo[0]};
}

// One block per row; each limit by bisection over the 64-bit rank (value, then index).
template <typename T>
__global__ __launch_bounds__(kSimpleThreads) void sample_kernel(const void* logits, uint64_t stride, uint32_t vocab,
                                                                SampleParams p, SampleOut o) {
    __shared__ uint32_t sn[kSimpleThreads];
    __shared__ uint64_t slo[kSimpleThreads], shi[kSimpleThreads];
    __shared__ uint64_t sbest;
    const uint32_t t = threadIdx.x;
    const uint64_t r = blockIdx.x;
    const void* row = static_cast<const char*>(logits) + r * stride * kLogitBytes<T>;
    const float temp = p.temperature ? p.temperature[r] : 1.0f, u = p.uniform[r];
    const float top_p = p.top_p ? p.top_p[r] : 1.0f, min_p = p.min_p ? p.min_p[r] : 0.0f;
    const int32_t top_k = p.top_k ? p.top_k[r] : 0;
    if (t == 0) sbest = 0;
    __syncthreads();
    uint64_t best = 0;
    bool bad = temp != temp || u != u || top_p != top_p || min_p != min_p;
    uint32_t live = 0;
    for (uint32_t i = t; i < vocab; i += kSimpleThreads) {
        const float l = load_logit<T>(row, i);
        bad |= !(l < INFINITY);
        if (l > -INFINITY) {
            ++live;
            const uint64_t k = rank_key(l, i);
            best = k > best ? k : best;
        }
    }
    best = wave_max_u64(best);
    if (t % 64 == 0) atomicMax(reinterpret_cast<unsigned long long*>(&sbest), static_cast<unsigned long long>(best));
    const Sum all = block_sum(Sum{live, bad ? 1u : 0u}, sn, slo, shi);
    best = sbest;
    live = all.n;
    if (all.w != 0 || live == 0) {
        if (t == 0) {
            o.tokens[r] = TWD_TOKEN_DEGENERATE;
            if (o.logprobs) o.logprobs[r] = __uint_as_float(0x7FC00000u);
            if (o.kept) o.kept[r] = 0;
        }
        return;
    }
    if (temp <= 0.0f) {
        if (t == 0) {
            o.tokens[r] = rank_index(best);
            if (o.logprobs) o.logprobs[r] = 0.0f;
            if (o.kept) o.kept[r] = 1;
        }
        return;
    }
    const Scale c = scale_of(temp);
    const float m = rank_value(best);
    const double top = weight_of(m, c).oct;
    // entries of at least rank R
    auto above = [&](uint64_t R) {
        Sum s{0, 0};
        for (uint32_t i = t; i < vocab; i += kSimpleThreads) {
            const float l = load_logit<T>(row, i);
            if (l > -INFINITY && rank_key(l, i) >= R) ++s.n, s.w += in_sum(weight_of(l, c), top);
        }
        return block_sum(s, sn, slo, shi);
    };
    // the largest R whose entries satisfy `enough`, which holds for R = 0
    auto bisect = [&](auto enough) {
        uint64_t R = 0;
        for (int b = 63; b >= 0; --b) {
            const uint64_t x = R | 1ull << b;
            if (enough(above(x))) R = x;
        }
        return R;
    };
    uint64_t cut = 0;
    if (top_k > 0 && static_cast<uint32_t>(top_k) < live)
        cut = bisect([&](const Sum& s) { return s.n >= static_cast<uint32_t>(top_k); });
    if (top_p < 1.0f) {
        const u128 want = part_of(top_p, above(cut).w, true);
        const uint64_t x = bisect([&](const Sum& s) { return s.n >= 1 && s.w >= want; });
        cut = x > cut ? x : cut;
    }
    if (min_p > 0.0f) {
        const double lim = log2(static_cast<double>(min_p));
        Sum s{0, 0};
        uint64_t low = ~0ull;
        for (uint32_t i = t; i < vocab; i += kSimpleThreads) {
            const float l = load_logit<T>(row, i);
            if (l > -INFINITY && (static_cast<double>(l) - static_cast<double>(m)) * c.hi >= lim) {
                const uint64_t k = rank_key(l, i);
                low = k < low ? k : low;
            }
        }
        if (low > best) low = best;
        __syncthreads();
        if (t == 0) sbest = ~0ull;
        __syncthreads();
        atomicMin(reinterpret_cast<unsigned long long*>(&sbest), static_cast<unsigned long long>(low));
        __syncthreads();
        cut = sbest > cut ? sbest : cut;
    }
    cut = cut < best ? cut : best;
    const Sum kept = above(cut);
    const u128 want = u < 1.0f ? part_of(u, kept.w, false) : kept.w - 1;  // the first running sum past u S
    // the smallest index whose running sum exceeds it, by bisection over the index
    uint32_t pos = 0;
    for (int b = 19; b >= 0; --b) {
        const uint32_t x = pos + (1u << b);  // do the kept weights below index x stay at most `want`?
        if (x > vocab) continue;
        Sum s{0, 0};
        for (uint32_t i = t; i < x; i += kSimpleThreads) {
            const float l = load_logit<T>(row, i);
            if (l > -INFINITY && rank_key(l, i) >= cut) s.w += in_sum(weight_of(l, c), top);
        }
        if (block_sum(s, sn, slo, shi).w <= want) pos = x;
    }
    if (t == 0) {
        const u128 w = in_sum(weight_of(load_logit<T>(row, pos), c), top);
        o.tokens[r] = pos;
        if (o.logprobs) o.logprobs[r] = static_cast<float>(log(to_double(w) / to_double(kept.w)));
        if (o.kept) o.kept[r] = static_cast<int32_t>(kept.n);
    }
}

}  // namespace

}  // namespace twd

struct twd_sampler {
    twd::StreamOrder order;
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
    *out = s;
    return TWD_OK;
}

TWD_API void twd_sampler_destroy(twd_sampler* s) {
    if (!s) return;
    order_release(s->order);
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
    const SampleParams p{temperature, top_k, top_p, min_p, uniform};
    const SampleOut o{tokens, logprobs, kept};
    if (type == TWD_F32)
        sample_kernel<float><<<rows, kSimpleThreads, 0, s>>>(logits, row_stride, vocab, p, o);
    else if (type == TWD_BF16)
        sample_kernel<Bf16><<<rows, kSimpleThreads, 0, s>>>(logits, row_stride, vocab, p, o);
    else
        sample_kernel<Fp16><<<rows, kSimpleThreads, 0, s>>>(logits, row_stride, vocab, p, o);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return hip_fail(e, "launching the sampler");
    return order_after(sampler->order, s);
}

}  // extern "C"
