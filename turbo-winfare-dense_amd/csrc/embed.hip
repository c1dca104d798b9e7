// The embedding lookup with scaling, and its gradient by sorted ids.
//
//   out_i = scale table[id_i]        d_table_v = scale sum_{i: id_i = v} d_rows_i
#include <hip/hip_runtime.h>

#include <new>
#include <string>

#include "twd_embed.h"
#include "twd_internal.h"
#include "vocab_core.h"

namespace twd {

namespace {

constexpr uint32_t kEmbedThreads = 256;
constexpr uint32_t kEach = 8;                             // elements of a lane
constexpr uint32_t kSpan = kEmbedThreads * kEach;         // elements of a block's step

// Eight elements of a row to a lane: where rows start at multiples of 16 bytes (wide) they are adjacent, element kEach t + i
// of a step for lane t; otherwise a wave's accesses are, element t + 256 i.
__device__ __forceinline__ uint32_t element(bool wide, uint32_t t, uint32_t i) { return wide ? kEach * t + i : t + kEmbedThreads * i; }

__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(Bf16* p, float v) { p->u = static_cast<uint16_t>(f32_to_half<Bf16>(v)); }
__device__ __forceinline__ void put(Fp16* p, float v) { p->h = static_cast<_Float16>(v); }

// The lane's eight of a row from element `base` on, as they lie in memory; zero past its d.
template <typename T>
struct Raw {
    static constexpr uint32_t kWords = kEach * sizeof(T) / 16;
    u32x4_t w[kWords];

    __device__ __forceinline__ void load(const T* row, bool wide, uint32_t base, uint32_t d) {
        const uint32_t t = threadIdx.x, first = base + kEach * t;
        if (wide && first + kEach <= d) {
#pragma unroll
            for (uint32_t i = 0; i < kWords; ++i) w[i] = reinterpret_cast<const u32x4_t*>(row + first)[i];
            return;
        }
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            const uint32_t e = base + element(wide, t, i);
            if constexpr (sizeof(T) == 4) {
                w[i / 4][i % 4] = e < d ? __float_as_uint(row[e]) : 0u;
            } else {
                const uint32_t bits = e < d ? reinterpret_cast<const uint16_t*>(row)[e] : 0u;
                w[0][i / 2] = i % 2 == 0 ? bits : w[0][i / 2] | bits << 16;
            }
        }
    }
    __device__ __forceinline__ float operator[](uint32_t i) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i / 4][i % 4]);
        else return half_to_f32<T>(i % 2 == 0 ? w[0][i / 2] & 0xFFFFu : w[0][i / 2] >> 16);
    }
};

template <typename T>
__device__ __forceinline__ void store_eight(T* row, bool wide, uint32_t base, uint32_t d, const float (&v)[kEach]) {
    const uint32_t t = threadIdx.x, first = base + kEach * t;
    if (wide && first + kEach <= d) {
        if constexpr (sizeof(T) == 4) {
            f32x4_t* p = reinterpret_cast<f32x4_t*>(row + first);
            p[0] = f32x4_t{v[0], v[1], v[2], v[3]}, p[1] = f32x4_t{v[4], v[5], v[6], v[7]};
        } else {
            u32x4_t w;
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = f32_to_half<T>(v[2 * i]) | f32_to_half<T>(v[2 * i + 1]) << 16;
            *reinterpret_cast<u32x4_t*>(row + first) = w;
        }
        return;
    }
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) {
        const uint32_t e = base + element(wide, t, i);
        if (e < d) put(row + e, v[i]);
    }
}

// ---- lookup ---------------------------------------------------------------------------------------------

struct EmbedArgs {
    const void* table;
    uint64_t table_stride;
    const int32_t* ids;
    void* out;
    uint64_t out_stride;
    uint32_t vocab, d;
    float scale;
    bool wide_in, wide_out;
};

// A block to a row's STEPS steps, all loaded before the first is stored. Bound by the bytes: 8,191 rows of 3,584, fp32 to bf16,
// take 23 us (7.8 TB/s, as the caches hold some of the rows from call to call), one row of 5,376 2.7 us, a launch and the
// chain from its id to its store.
template <typename In, typename Out, int STEPS>
__global__ __launch_bounds__(kEmbedThreads) void embed_kernel(EmbedArgs a) {
    const uint32_t id = static_cast<uint32_t>(a.ids[blockIdx.x]);
    const bool wide = a.wide_in && a.wide_out, live = id < a.vocab;
    const In* row = static_cast<const In*>(a.table) + (live ? id : 0) * a.table_stride;
    Out* out = static_cast<Out*>(a.out) + blockIdx.x * a.out_stride;
    Raw<In> x[STEPS];
    const uint32_t base = blockIdx.y * STEPS * kSpan;
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
        if (live && base + s * kSpan < a.d) x[s].load(row, wide, base + s * kSpan, a.d);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        if (base + s * kSpan >= a.d) break;
        float v[kEach];
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) v[i] = live ? x[s][i] * a.scale : 0.0f;
        store_eight(out, wide, base + s * kSpan, a.d, v);
    }
}

// ---- gradient -------------------------------------------------------------------------------------------
//
// Ids are sorted with their places (equal ids by rising place), lists of kList in LDS first; then each entry's place in
// the whole is its own in its list and, by bisection, the number of smaller ones in every other. Runs of equal ids are
// summed by a block each; of a long run, the stretches of kPiece entries at multiples of kPiece are summed before, so that
// no block adds up more than 2 kPiece - 1 rows and a part for each kPiece, whatever the ids. No atomics: an id's rows are
// added by rising place, so the same ids give the same bits.
//
// What bounds it is the clearing of a table that is mostly zeros: 16,384 ids of 262,144 x 5,376 in bf16 take 592 us, 2.8 GB
// cleared in the first three launches (131 + 170 + 182 us, 5.8 TB/s; a fill reaches 6.8), then the runs, 110 us: their 180 MB of
// rows, and rows of the table that the clearing has left in no cache. 513 ids of 32,003 x 1,024 to fp32: 36 us, 131 MB cleared
// in 24 of them. A run's parts are added by one block, four at a time: 16,384 equal ids of 32,003 x 1,024 in bf16 take 158 us, 72
// drawn as words are; 262,144 of them 2,065 and 522.
constexpr uint32_t kList = 2048, kListThreads = 1024;
constexpr uint32_t kFillEach = 4;  // pieces of 16 bytes that a thread clears
constexpr uint64_t kMostFill = (1ull << 38) - (1u << 20);  // bytes of one launch, which may have fewer than 2^32 threads
constexpr uint32_t kPiece = 32;
constexpr uint32_t kNoId = 0xFFFFFFFFu;  // outside the vocabulary: sorted last

struct SortArgs {
    const int32_t* ids;
    uint32_t n, vocab, lists;
    uint64_t* listed;  // sorted lists of id (high), place (low)
    uint32_t* id;      // sorted
    uint32_t* place;
};

// d_table's bytes to clear, 16 at a time, a share of them by the blocks that follow a launch's own: clearing takes longer
// than everything before the runs, which it hides.
struct Fill {
    u32x4_t* at;
    uint64_t n;
    uint8_t* edge[2];  // bytes before and after, with the first share
    uint32_t edge_bytes[2];
};
__device__ __forceinline__ void clear_share(const Fill& f, uint32_t block) {
    const uint32_t t = threadIdx.x, threads = blockDim.x;
    const uint64_t from = static_cast<uint64_t>(block) * kFillEach * threads + t;
#pragma unroll
    for (uint32_t i = 0; i < kFillEach; ++i)
        if (from + i * threads < f.n) f.at[from + i * threads] = u32x4_t{0, 0, 0, 0};
    if (block == 0)
        for (int e = 0; e < 2; ++e)
            if (t < f.edge_bytes[e]) f.edge[e][t] = 0;
}

__global__ __launch_bounds__(kListThreads) void embed_sort_kernel(SortArgs a, Fill f) {
    __shared__ uint64_t key[kList];
    const uint32_t t = threadIdx.x;
    if (blockIdx.x >= a.lists) {
        clear_share(f, blockIdx.x - a.lists);
        return;
    }
    const uint32_t first = blockIdx.x * kList, here = min(a.n - first, kList);
    for (uint32_t i = t; i < kList; i += kListThreads) {
        const uint32_t id = i < here ? static_cast<uint32_t>(a.ids[first + i]) : kNoId;
        key[i] = static_cast<uint64_t>(i < here && id < a.vocab ? id : kNoId) << 32 | (first + i);
    }
    uint32_t size = 2;  // the list's entries, up to a power of two
    while (size < here) size *= 2;
    for (uint32_t k = 2; k <= size; k *= 2)
        for (uint32_t j = k / 2; j > 0; j /= 2) {
            __syncthreads();
            if (t < size / 2) {
                const uint32_t lo = t / j * 2 * j + t % j, hi = lo + j;
                const uint64_t x = key[lo], y = key[hi];
                if ((x > y) == ((lo & k) == 0)) key[lo] = y, key[hi] = x;
            }
        }
    __syncthreads();
    for (uint32_t i = t; i < here; i += kListThreads) {
        if (a.lists == 1)
            a.id[i] = static_cast<uint32_t>(key[i] >> 32), a.place[i] = static_cast<uint32_t>(key[i]);
        else
            a.listed[first + i] = key[i];
    }
}

__global__ __launch_bounds__(256) void embed_merge_kernel(SortArgs a, Fill f) {
    const uint32_t own_blocks = (a.n + 255) / 256;
    if (blockIdx.x >= own_blocks) {
        clear_share(f, blockIdx.x - own_blocks);
        return;
    }
    const uint32_t at = blockIdx.x * 256 + threadIdx.x;
    if (at >= a.n) return;
    const uint64_t key = a.listed[at];
    const uint32_t own = at / kList;
    uint32_t rank = at % kList;
#pragma unroll 4
    for (uint32_t l = 0; l < a.lists; ++l) {
        const uint64_t* list = a.listed + l * kList;
        uint32_t lo = 0, n = l == own ? 0 : min(a.n - l * kList, kList);  // how many are smaller: in lo .. lo + n
        while (n > 0) {
            const uint32_t half = n / 2;
            if (list[lo + half] < key) lo += half + 1, n -= half + 1;
            else n = half;
        }
        rank += lo;
    }
    a.id[rank] = static_cast<uint32_t>(key >> 32), a.place[rank] = static_cast<uint32_t>(key);
}

struct RunArgs {
    const void* rows;
    uint64_t rows_stride;
    const uint32_t* id;
    const uint32_t* place;
    float* part;  // [piece][d, up to a multiple of 8]: a lane's elements are those of its rows
    void* table;
    uint64_t table_stride;
    uint32_t n, d, vocab;
    float scale;
    bool wide, add;
};

__host__ __device__ inline uint64_t part_stride(uint32_t d) { return (d + 7ull) / 8 * 8; }

// Adds the rows of entries from .. to - 1, several on their way at a time; `places`: lane l's is that of entry from + l.
template <typename In>
__device__ __forceinline__ void add_some(const RunArgs& a, uint32_t n, uint32_t places, uint32_t base, float (&sum)[kEach]) {
    constexpr uint32_t kAtOnce = sizeof(In) == 4 ? 4 : 8;
    for (uint32_t i = 0; i < n; i += kAtOnce) {
        Raw<In> x[kAtOnce];
#pragma unroll
        for (uint32_t j = 0; j < kAtOnce; ++j)
            if (i + j < n) {
                const uint32_t place = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(places), static_cast<int>(i + j)));
                x[j].load(static_cast<const In*>(a.rows) + place * a.rows_stride, a.wide, base, a.d);
            }
#pragma unroll
        for (uint32_t j = 0; j < kAtOnce; ++j)
            if (i + j < n) {
#pragma unroll
                for (uint32_t e = 0; e < kEach; ++e) sum[e] += x[j][e];
            }
    }
}
template <typename In>
__device__ __forceinline__ void add_rows(const RunArgs& a, uint32_t from, uint32_t to, uint32_t base, float (&sum)[kEach]) {
    static_assert(kPiece <= 64, "a lane to each place");
    if (from >= to) return;
    const uint32_t at = from + threadIdx.x % 64;
    add_some<In>(a, to - from, at < to ? a.place[at] : 0u, base, sum);
}

// The parts of long runs: of each stretch of kPiece entries that all have one id.
template <typename In>
__global__ __launch_bounds__(kEmbedThreads) void embed_parts_kernel(RunArgs a, uint32_t steps, Fill f) {
    const uint32_t own = a.n / kPiece * steps;
    if (blockIdx.x >= own) {
        clear_share(f, blockIdx.x - own);
        return;
    }
    const uint32_t piece = blockIdx.x / steps, first = piece * kPiece, base = blockIdx.x % steps * kSpan;
    const uint32_t id = a.id[first];
    if (id == kNoId || a.id[first + kPiece - 1] != id) return;
    float sum[kEach] = {};
    add_rows<In>(a, first, first + kPiece, base, sum);
    store_eight(a.part + piece * part_stride(a.d), a.wide, base, a.d, sum);
}

// A block to each run (that of its first entry) and step of columns. Most runs are short: ids and places of 64 entries come
// at once, and rows after them.
template <typename In, typename Out>
__global__ __launch_bounds__(kEmbedThreads) void embed_runs_kernel(RunArgs a) {
    const uint32_t first = blockIdx.x, base = blockIdx.y * kSpan, lane = threadIdx.x % 64;
    const bool in = first + lane < a.n;
    const uint32_t ids = in ? a.id[first + lane] : kNoId, places = in ? a.place[first + lane] : 0u;
    const uint32_t before = first > 0 ? a.id[first - 1] : kNoId;
    const uint32_t id = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(ids)));
    if (id == kNoId || before == id) return;
    const uint32_t near = static_cast<uint32_t>(__popcll(__ballot(ids == id)));  // sorted: the first ones
    float sum[kEach] = {};
    if (near < 2 * kPiece) {  // (a run of 63 may hold a whole piece: its part is not used)
        add_some<In>(a, near, places, base, sum);
    } else {
        // the end, by a search in 64 places at a time
        uint32_t last = first + near - 1, past = a.n;  // `last` has the id, `past` does not
        while (past - last > 1) {
            const uint32_t step = (past - last + 63) / 64, at = last + (lane + 1) * step;
            last += step * static_cast<uint32_t>(__popcll(__ballot(at < past && a.id[at] == id)));
            past = min(past, last + step);
        }
        const uint32_t end = last + 1, p0 = (first + kPiece - 1) / kPiece, p1 = end / kPiece;  // whole pieces
        add_rows<In>(a, first, p0 * kPiece, base, sum);
        constexpr uint32_t kAtOnce = 4;
        for (uint32_t p = p0; p < p1; p += kAtOnce) {
            Raw<float> x[kAtOnce];
#pragma unroll
            for (uint32_t j = 0; j < kAtOnce; ++j)
                if (p + j < p1) x[j].load(a.part + (p + j) * part_stride(a.d), a.wide, base, a.d);
#pragma unroll
            for (uint32_t j = 0; j < kAtOnce; ++j)
                if (p + j < p1) {
#pragma unroll
                    for (uint32_t e = 0; e < kEach; ++e) sum[e] += x[j][e];
                }
        }
        add_rows<In>(a, p1 * kPiece, end, base, sum);
    }
    Out* row = static_cast<Out*>(a.table) + id * a.table_stride;
#pragma unroll
    for (uint32_t e = 0; e < kEach; ++e) sum[e] *= a.scale;
    if (a.add) {
        Raw<Out> old;
        old.load(row, a.wide, base, a.d);
#pragma unroll
        for (uint32_t e = 0; e < kEach; ++e) sum[e] += old[e];
    }
    store_eight(row, a.wide, base, a.d, sum);
}

// Rows apart from one another, and tables past kMostFill: cleared one by one.
template <typename Out>
__global__ __launch_bounds__(kEmbedThreads) void embed_clear_kernel(Out* table, uint64_t stride, uint32_t vocab, uint32_t d, bool wide) {
    const float zero[kEach] = {};
    for (uint32_t v = blockIdx.x; v < vocab; v += gridDim.x)
        for (uint32_t base = 0; base < d; base += kSpan) store_eight(table + v * stride, wide, base, d, zero);
}

constexpr uint32_t kMaxIds = 1u << 18, kMaxLookups = 1u << 23, kMaxWidth = 1u << 20;

bool known_type(int type) { return type == TWD_F32 || type == TWD_BF16 || type == TWD_F16; }
uint32_t size_of(int type) { return type == TWD_F32 ? 4 : 2; }
bool at_multiple(const void* p, uint64_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
bool wide_rows(const void* p, uint64_t stride, uint64_t rows, int type) {
    return at_multiple(p, 16) && (rows <= 1 || stride * size_of(type) % 16 == 0);
}
uint32_t over(uint64_t x, uint32_t y) { return static_cast<uint32_t>((x + y - 1) / y); }

template <typename F>
int with_type(int type, F&& f) {
    if (type == TWD_F32) return f(float{});
    if (type == TWD_BF16) return f(Bf16{});
    return f(Fp16{});
}

int check_matrix(const char* what, const void* p, int type, uint64_t rows, uint32_t d, uint64_t stride) {
    const std::string name(what);
    if (!known_type(type)) return fail(TWD_E_INVALID, name + ": type must be TWD_F32, TWD_BF16 or TWD_F16");
    if (!at_multiple(p, size_of(type))) return fail(TWD_E_INVALID, name + " is not aligned to its type");
    if (rows > 1 && (stride < d || stride > 1ull << 31)) return fail(TWD_E_INVALID, name + ": the row stride must be at least d_model and at most 2^31");
    return TWD_OK;
}

}  // namespace

}  // namespace twd

struct twd_embedgrad {
    twd::StreamOrder order;
    void* block;  // the one allocation behind the following
    uint64_t* listed;
    uint32_t* id;
    uint32_t* place;
    float* part;
    uint64_t bytes;
    uint32_t max_ids, max_d;
    int device;
};

namespace twd {

namespace {

int run(const twd_embedgrad* g, SortArgs sort, const RunArgs& a, int rows_type, int table_type, bool clear, hipStream_t s) {
    sort.lists = over(sort.n, kList);
    const uint64_t size = size_of(table_type);
    const uint32_t steps = over(a.d, kSpan);
    Fill f{};
    const uint64_t bytes = static_cast<uint64_t>(a.vocab) * a.d * size;
    if (clear && (a.vocab == 1 || a.table_stride == a.d) && bytes <= kMostFill) {
        const uintptr_t from = reinterpret_cast<uintptr_t>(a.table);
        const uint64_t before = (16 - from % 16) % 16 < bytes ? (16 - from % 16) % 16 : bytes;
        f.n = (bytes - before) / 16;
        f.at = reinterpret_cast<u32x4_t*>(from + before);
        f.edge[0] = static_cast<uint8_t*>(a.table), f.edge_bytes[0] = static_cast<uint32_t>(before);
        f.edge[1] = static_cast<uint8_t*>(a.table) + before + 16 * f.n;
        f.edge_bytes[1] = static_cast<uint32_t>(bytes - before - 16 * f.n);
    } else if (clear) {
        const int rc = with_type(table_type, [&](auto t) -> int {
            using Out = decltype(t);
            embed_clear_kernel<<<a.vocab < 65536 ? a.vocab : 65536, kEmbedThreads, 0, s>>>(static_cast<Out*>(a.table), a.table_stride, a.vocab, a.d, a.wide);
            TWD_HIP(hipGetLastError());
            return TWD_OK;
        });
        if (rc) return rc;
    }
    // what is left of the clearing goes with the launches that are left: sorting takes some 6 us, merging 16, the parts 30
    const bool merges = sort.lists > 1, parts = a.n >= kPiece;
    auto share = [&](uint32_t percent, uint32_t threads, uint32_t* blocks) {
        Fill now = f;
        const uint64_t each = static_cast<uint64_t>(kFillEach) * threads;
        const uint64_t want = (f.n * percent / 100 + each - 1) / each;
        now.n = want * each < f.n ? want * each : f.n;
        *blocks = now.n == 0 && now.edge_bytes[0] + now.edge_bytes[1] == 0 ? 0u : static_cast<uint32_t>(want < 1 ? 1 : want);
        f.at += now.n, f.n -= now.n, f.edge_bytes[0] = f.edge_bytes[1] = 0;
        return now;
    };
    uint32_t blocks = 0;
    const Fill first = share(!merges && !parts ? 100 : merges ? 30 : 50, kListThreads, &blocks);
    if (sort.lists + blocks == 0) return TWD_OK;
    embed_sort_kernel<<<sort.lists + blocks, kListThreads, 0, s>>>(sort, first);
    TWD_HIP(hipGetLastError());
    if (a.n == 0) return TWD_OK;
    if (merges) {
        const Fill second = share(parts ? 50 : 100, 256, &blocks);
        embed_merge_kernel<<<over(a.n, 256) + blocks, 256, 0, s>>>(sort, second);
        TWD_HIP(hipGetLastError());
    }
    return with_type(rows_type, [&](auto r) -> int {
        using In = decltype(r);
        if (parts) {
            const Fill third = share(100, kEmbedThreads, &blocks);
            embed_parts_kernel<In><<<a.n / kPiece * steps + blocks, kEmbedThreads, 0, s>>>(a, steps, third);
            TWD_HIP(hipGetLastError());
        }
        return with_type(table_type, [&](auto t) -> int {
            embed_runs_kernel<In, decltype(t)><<<dim3(a.n, steps), kEmbedThreads, 0, s>>>(a);
            TWD_HIP(hipGetLastError());
            return TWD_OK;
        });
    });
}

}  // namespace

}  // namespace twd

using namespace twd;

extern "C" {

TWD_API int twd_embed(const void* table, int table_type, uint32_t vocab, uint32_t d_model, uint64_t table_stride,
                      const int32_t* ids, uint32_t ids_count, float scale, void* out, int out_type, uint64_t out_stride,
                      void* stream) {
    clear_error();
    if (!table || (ids_count > 0 && (!ids || !out))) return fail(TWD_E_INVALID, "null argument");
    if (vocab == 0 || vocab > 0x7FFFFFFFu) return fail(TWD_E_INVALID, "vocab must be in 1..2^31-1");
    if (d_model == 0 || d_model > kMaxWidth) return fail(TWD_E_INVALID, "d_model must be in 1..2^20");
    if (ids_count > kMaxLookups) return fail(TWD_E_INVALID, "ids_count must be at most 2^23");
    int rc = check_matrix("table", table, table_type, vocab, d_model, table_stride);
    if (rc || (rc = check_matrix("out", out, out_type, ids_count, d_model, out_stride))) return rc;
    if (ids_count == 0) return TWD_OK;
    const EmbedArgs a{table, table_stride, ids, out, out_stride, vocab, d_model, scale,
                      wide_rows(table, table_stride, vocab, table_type), wide_rows(out, out_stride, ids_count, out_type)};
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return with_type(table_type, [&](auto in) -> int {
        return with_type(out_type, [&](auto o) -> int {
            // few rows: a block to each step, so that more of them are at work
            if (ids_count < 512)
                embed_kernel<decltype(in), decltype(o), 1><<<dim3(ids_count, over(d_model, kSpan)), kEmbedThreads, 0, s>>>(a);
            else
                embed_kernel<decltype(in), decltype(o), 3><<<dim3(ids_count, over(d_model, 3 * kSpan)), kEmbedThreads, 0, s>>>(a);
            TWD_HIP(hipGetLastError());
            return TWD_OK;
        });
    });
}

TWD_API int twd_embedgrad_create(uint32_t max_ids, uint32_t max_d_model, twd_embedgrad** out) {
    clear_error();
    if (!out) return fail(TWD_E_INVALID, "null argument");
    *out = nullptr;
    if (max_ids == 0 || max_ids > kMaxIds) return fail(TWD_E_INVALID, "max_ids must be in 1..262144");
    if (max_d_model == 0 || max_d_model > kMaxWidth) return fail(TWD_E_INVALID, "max_d_model must be in 1..2^20");
    int dev = 0;
    TWD_HIP(hipGetDevice(&dev));
    twd_embedgrad* g = new (std::nothrow) twd_embedgrad{};
    if (!g) return fail(TWD_E_INVALID, "out of host memory");
    const uint64_t ids = (max_ids + 63ull) / 64 * 64, parts = max_ids / kPiece;
    g->max_ids = max_ids, g->max_d = max_d_model, g->device = dev;
    g->bytes = ids * 16 + parts * part_stride(max_d_model) * sizeof(float);
    const hipError_t e = hipMalloc(&g->block, g->bytes);
    if (e != hipSuccess) {
        delete g;
        return hip_fail(e, "allocating the embedding gradient's scratch");
    }
    g->listed = static_cast<uint64_t*>(g->block);
    g->id = reinterpret_cast<uint32_t*>(g->listed + ids);
    g->place = g->id + ids;
    g->part = reinterpret_cast<float*>(g->place + ids);
    *out = g;
    return TWD_OK;
}

TWD_API void twd_embedgrad_destroy(twd_embedgrad* g) {
    if (!g) return;
    order_release(g->order);
    (void)hipFree(g->block);
    delete g;
}

TWD_API int twd_embedgrad_info(const twd_embedgrad* g, uint64_t* device_bytes) {
    clear_error();
    if (!g) return fail(TWD_E_INVALID, "null embedding gradient");
    if (device_bytes) *device_bytes = g->bytes;
    return TWD_OK;
}

TWD_API int twd_embedgrad_run(twd_embedgrad* g, const void* d_rows, int rows_type, uint32_t ids_count, uint32_t d_model,
                              uint64_t rows_stride, const int32_t* ids, float scale, void* d_table, int table_type,
                              uint32_t vocab, uint64_t table_stride, int accumulate, void* stream) {
    clear_error();
    if (!g) return fail(TWD_E_INVALID, "null embedding gradient");
    if (!d_table || (ids_count > 0 && (!d_rows || !ids))) return fail(TWD_E_INVALID, "null argument");
    if (ids_count > g->max_ids) return fail(TWD_E_INVALID, "ids_count out of range for this embedding gradient");
    if (d_model == 0 || d_model > g->max_d) return fail(TWD_E_INVALID, "d_model out of range for this embedding gradient");
    if (vocab == 0 || vocab > 0x7FFFFFFFu) return fail(TWD_E_INVALID, "vocab must be in 1..2^31-1");
    int rc = check_matrix("d_rows", d_rows, rows_type, ids_count, d_model, rows_stride);
    if (rc || (rc = check_matrix("d_table", d_table, table_type, vocab, d_model, table_stride))) return rc;
    int dev = 0;
    TWD_HIP(hipGetDevice(&dev));
    if (dev != g->device) return fail(TWD_E_INVALID, "the embedding gradient lives on another device than the current one");
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if ((rc = order_before(g->order, s))) return rc;
    SortArgs sort{};
    sort.ids = ids, sort.n = ids_count, sort.vocab = vocab, sort.listed = g->listed, sort.id = g->id, sort.place = g->place;
    const RunArgs a{d_rows, rows_stride, g->id, g->place, g->part, d_table, table_stride, ids_count, d_model, vocab, scale,
                    wide_rows(d_rows, rows_stride, ids_count, rows_type) && wide_rows(d_table, table_stride, vocab, table_type),
                    accumulate != 0};
    rc = run(g, sort, a, rows_type, table_type, accumulate == 0, s);
    const int rc2 = order_after(g->order, s);
    return rc ? rc : rc2;
}

}  // extern "C"
