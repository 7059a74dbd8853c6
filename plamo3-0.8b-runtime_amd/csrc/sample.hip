// Tokens drawn from logits on gfx950: temperature, top-k, top-p and min-p, by given uniform numbers.
//
// A row's tokens are ordered by descending logit, equal ones by ascending id.  With weights
// e_i = exp((x_i - max x) / T): top-k keeps the first k; top-p of those the ones before which less than
// p of the kept weight lies; min-p of those the ones of at least min_p of the largest weight.  All three
// keep a beginning of the order.  The token is the first one up to which more than u of the kept weight
// lies.  Nothing is sorted but the few tokens around a border:
//   1. the largest logit;
//   2. a histogram over bins of the exponent (32 bins for a factor of two): sums of the weights, or, for
//      a top-k of at most 1024, numbers of tokens, for which no exponential is taken;
//   3. prefix sums over the bins give the bin of each border; the tokens of these bins (for a top-k of all
//      bins up to its own) are listed;
//   4. the list is sorted in LDS and searched.  A bin of more tokens than the list holds is divided again
//      by the bits of the logits until it is small enough or one value.
// Each step is a launch over segments of the rows but the last: one CU draws some 45 GB/s from beyond its
// L2, so that a workgroup that read a row of 107,520 BF16 logits alone would take 5 us each time.
// 128 FP32 rows of that length (55 MB) take 10.7, 18.2, 18.0 and 13.2 us: the first reads at 5.1 TB/s (a large read
// reaches 6.3), the second is the weights' FP64 arithmetic and LDS atomics, the third reads again behind 8 us
// of finding its bins, the last is latency.  One BF16 row takes 3.7, 4.6, 9.4 and 6.8 us, all of it latency.
// Weights are whole multiples of 2^-S of the largest (S = 63 - log2 of the vocabulary, at most 46), so
// that all sums are exact whatever their order: the token depends on the row alone, not on how it was
// split, and sums of unsigned 64-bit atomics are the same in every run.  A token of less than 2^-(S+1)
// of the largest weight is never drawn.  exp is evaluated in FP64 to 2^-42: a token is told apart from
// its neighbour by sums over 100,000 of them, where FP32's 2^-24 would move the borders.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstddef>

#include "common.h"
#include "device.h"
#include "paged.h"

namespace plamo {
using namespace dev;

namespace {

constexpr int THREADS = 1024, WAVES = THREADS / 64;  // of the workgroup that ends a row
constexpr int PART_THREADS = 256;    // of a segment's workgroup
constexpr int GROUP_THREADS = 512;   // of one that fills a histogram, or lists tokens
constexpr int STEPS = 256;           // table entries for a factor of two
constexpr int BIN_SHIFT = 3;         // log2 of a bin's table steps
constexpr int BINS = 1536;           // 32 (S + 1) <= 1504 are used
constexpr int LIST = 2048;           // tokens that are sorted at once
// A top-k up to which its tokens' weights are summed in the list, and no others: 64 rows of 107,520 and a top-k of
// 1,000 take 36 us so, 73 the other way.
constexpr int LIST_TOP_K = 1024;
constexpr int BUCKETS = 2048;        // of a list's range of weights
// Tokens of a bucket that are ordered by comparing all; where one has more, the list is sorted by exchanges: 64 BF16
// rows of a top-k of 1,000 take 36 us by buckets, 48 by exchanges, of a top-p of 0.99 41 and 43 (46 with 64 for this).
constexpr int BUCKET_MOST = 128;
constexpr int SUB = 1024;            // parts that a bin is divided into again

typedef unsigned long long u64;

// Row values as they stand: NaN fails every comparison, as minus infinity does, and minus zero equals zero.
template <int TYPE>
struct Element;
template <>
struct Element<TYPE_BF16> {
    typedef uint16_t T;
    static __device__ __forceinline__ float value(uint32_t h) { return bf(h & 0xffffu); }
};
template <>
struct Element<TYPE_F16> {
    typedef uint16_t T;
    static __device__ __forceinline__ float value(uint32_t h) { return float(__builtin_bit_cast(_Float16, uint16_t(h))); }
};
template <>
struct Element<TYPE_F32> {
    typedef uint32_t T;
    static __device__ __forceinline__ float value(uint32_t w) { return __uint_as_float(w); }
};

// f(id, value) for n elements, a thread's in ascending order; 16 bytes a load behind the first
// aligned element, AHEAD loads at once.  ROLLED: one copy of f for each half of a word: these kernels run
// through most of their code once, and its first fetch costs more than the loop.
template <int TYPE, int NT, int AHEAD, bool ROLLED, typename F>
__device__ __forceinline__ void for_row(const void* base, int n, F f) {
    typedef typename Element<TYPE>::T T;
    constexpr int PER = 16 / sizeof(T);
    const T* row = static_cast<const T*>(base);
    const int tid = threadIdx.x;
    const int head = min(n, int(((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / sizeof(T)));
    const int vectors = (n - head) / PER, tail = head + vectors * PER;
    const uint4* body = reinterpret_cast<const uint4*>(row + head);
    auto word = [&](int id, uint32_t w) {
        f(id, Element<TYPE>::value(w));
        if constexpr (PER == 8) f(id + 1, Element<TYPE>::value(w >> 16));
    };
    for (int i = tid; i < vectors; i += NT * AHEAD) {
        uint4 w[AHEAD];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) w[a] = body[min(i + a * NT, vectors - 1)];
        if constexpr (ROLLED) {
#pragma unroll 1
            for (int a = 0; a < AHEAD && i + a * NT < vectors; ++a) {
                int id = head + (i + a * NT) * PER;
#pragma unroll 1
                for (int j = 0; j < 4; ++j, id += PER / 4) {
                    word(id, w[0].x);
                    w[0] = make_uint4(w[0].y, w[0].z, w[0].w, 0);
                }
#pragma unroll
                for (int k = 0; k + 1 < AHEAD; ++k) w[k] = w[k + 1];
            }
        } else {
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                if (i + a * NT >= vectors) break;
                const int id = head + (i + a * NT) * PER;
                word(id, w[a].x);
                word(id + PER / 4, w[a].y);
                word(id + PER / 2, w[a].z);
                word(id + PER / 4 * 3, w[a].w);
            }
        }
    }
    // what lies before the first aligned element and behind the last whole 16 bytes (fewer than a wave's)
    const int rest = head + n - tail;
    if (tid < rest) {
        const int id = tid < head ? tid : tail + tid - head;
        f(id, Element<TYPE>::value(row[id]));
    }
}

// The largest of a workgroup's values and its lowest id, in every thread (id 0xffffffff: minus infinity).
template <int NT>
__device__ __forceinline__ void block_best(float& best, uint32_t& id, float* values, uint32_t* ids) {
    for (int o = 32; o > 0; o >>= 1) {
        const float v = __shfl_xor(best, o, 64);
        const uint32_t i = __shfl_xor(id, o, 64);
        if (v > best || (v == best && i < id)) {
            best = v;
            id = i;
        }
    }
    if ((threadIdx.x & 63) == 0) {
        values[threadIdx.x >> 6] = best;
        ids[threadIdx.x >> 6] = id;
    }
    __syncthreads();
    for (int w = 0; w < NT / 64; ++w)
        if (values[w] > best || (values[w] == best && ids[w] < id)) {
            best = values[w];
            id = ids[w];
        }
}
// The id is looked for where it is asked for: else it is 0, or 0xffffffff for minus infinity.
template <int TYPE, int NT>
__device__ __forceinline__ void find_best(const void* base, int n, bool ids, float& best, uint32_t& id) {
    best = NEG_INF;
    id = 0xffffffffu;
    if (ids) {
        for_row<TYPE, NT, 4, true>(base, n, [&](int i, float v) {
            if (v > best || (v == best && uint32_t(i) < id)) {
                best = v;
                id = v > NEG_INF ? uint32_t(i) : id;
            }
        });
    } else {
        for_row<TYPE, NT, 4, false>(base, n, [&](int, float v) { best = v > best ? v : best; });  // a maximum of a signalling NaN is NaN
        if (best > NEG_INF) id = 0;
    }
}

struct Sum {
    uint32_t count;
    u64 mass;
};

struct Shared {
    double table[STEPS];   // 2^(-j / STEPS)
    u64 bin_mass[BINS];    // then inclusive sums
    uint32_t bin_count[BINS];
    u64 order[LIST];       // descending logit, ascending id
    u64 weight[LIST];      // inclusive sums of the list's weights
    uint32_t bucket[BUCKETS];  // of the list's tokens: how many, then where they end
    Sum waves[WAVES];
    float wave_value[WAVES];
    uint32_t wave_id[WAVES];
    uint32_t low, high, queued, listed, split;
    Sum found;             // a border's count and mass up to and with its token
    uint32_t found_id;
    u64 found_weight;
    int found_bin[2];
    u64 min_mass;          // of the tokens of at least min_p
};

// v of the lane that a DPP control names, 0 where there is none (or the row is not in ROWS).
template <int CONTROL, int ROWS = 0xf>
__device__ __forceinline__ uint32_t shifted(uint32_t v) {
    return uint32_t(__builtin_amdgcn_update_dpp(0, int(v), CONTROL, ROWS, 0xf, false));
}
template <int CONTROL, int ROWS = 0xf>
__device__ __forceinline__ void add_shifted(Sum& v) {
    const uint32_t low = uint32_t(v.mass), high = uint32_t(v.mass >> 32);
    v.count += shifted<CONTROL, ROWS>(v.count);
    v.mass += u64(shifted<CONTROL, ROWS>(high)) << 32 | shifted<CONTROL, ROWS>(low);
}

// Inclusive sums over the workgroup: rows of 16 lanes by shifts of 1, 2, 4 and 8, then the last lane of
// the row, and of the half, before.
template <int NT>
__device__ __forceinline__ Sum block_scan(Sum v, Sum* waves, Sum& total) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    add_shifted<0x111>(v);
    add_shifted<0x112>(v);
    add_shifted<0x114>(v);
    add_shifted<0x118>(v);
    add_shifted<0x142, 0xa>(v);
    add_shifted<0x143, 0xc>(v);
    __syncthreads();  // the sums of a scan before this one have been read
    if (lane == 63) waves[wave] = v;
    __syncthreads();
    // the waves' sums, in a row of 16 lanes
    static_assert(NT <= 1024, "a row");
    Sum sum = {0, 0};
    if ((lane & 15) < NT / 64) sum = waves[lane & 15];
    add_shifted<0x111>(sum);
    add_shifted<0x112>(sum);
    add_shifted<0x114>(sum);
    add_shifted<0x118>(sum);
    auto of = [&](int l) -> Sum {
        return {uint32_t(__builtin_amdgcn_readlane(sum.count, l)),
                u64(uint32_t(__builtin_amdgcn_readlane(uint32_t(sum.mass >> 32), l))) << 32 |
                    uint32_t(__builtin_amdgcn_readlane(uint32_t(sum.mass), l))};
    };
    total = of(15);
    if (wave > 0) {
        const Sum before = of(wave - 1);
        v.count += before.count;
        v.mass += before.mass;
    }
    return v;
}

// Descending logits as ascending 32-bit keys; minus zero's is zero's.  (NaN's is any: no NaN is kept.)
__device__ __forceinline__ uint32_t sort_key(float v) {
    const uint32_t u = __float_as_uint(v + 0.0f);
    return u & 0x80000000u ? u : ~(u | 0x80000000u);
}

__device__ __forceinline__ float key_value(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key : ~key & 0x7fffffffu);
}

// exp(-g log(2) / STEPS) = 1 + g (c1 + g (c2 + g c3)) for |g| <= 1/2: off by (log(2) / 2 STEPS)^4 / 24 < 2^-42.
struct Series {
    static constexpr double C = -0.69314718055994530942 / STEPS;
    double c1 = C, c2 = C * C / 2, c3 = C * C * C / 6;
    // In vector registers, for loops over many: an FP64 product takes one scalar operand, and its constants
    // would be moved into place for every element.
    __device__ __forceinline__ void hold() { asm volatile("" : "+v"(c1), "+v"(c2), "+v"(c3)); }
};

// S: sums of n weights stay below 2^63.
__device__ __forceinline__ int weight_scale(int n) { return min(46, 31 + __clz(n)); }

// A row's weights: 2^S exp((x - top) / T), rounded.
struct Weights {
    static constexpr float MOST = 3.4028234663852886e38f;
    static constexpr double ROUND = 6755399441055744.0;  // sums with it are whole numbers, in their low bits
    float top;        // largest logit
    float cap;        // plus infinity, if that is the largest logit: only such tokens have a weight; else minus infinity
    int scale;        // S
    double rate;      // STEPS log2(e) / T
    double end;       // ROUND and the table steps from which on nothing is weighed

    __device__ __forceinline__ bool infinite() const { return cap == -NEG_INF; }
    __device__ __forceinline__ void set(float best, float temperature, int n) {
        scale = weight_scale(n);
        end = ROUND + (scale + 1) * STEPS;
        // plus infinity's distance from the top is taken as the largest finite value's
        cap = best == -NEG_INF ? best : NEG_INF;
        top = infinite() ? MOST : best;
        rate = infinite() ? double(MOST) : STEPS * 1.44269504088896340736 / double(temperature);
    }
    // The logit's distance from the top in table steps, rounded; false where it weighs nothing, as minus
    // infinity and NaN do (their distance is infinite, or compares with nothing).  FINITE: the row's largest
    // logit is.
    template <bool FINITE = false>
    __device__ __forceinline__ bool step(float v, uint32_t& n, double& below, double& whole) const {
        below = double(top) - double(!FINITE && v == -NEG_INF ? MOST : v);
        const double t = fma(below, rate, ROUND);
        n = uint32_t(__double2loint(t));
        whole = t - ROUND;
        return t < end && (FINITE || !(v < cap));
    }
    template <bool FINITE = false>
    __device__ __forceinline__ bool bin(float v, int& b) const {
        uint32_t n;
        double below, whole;
        const bool any = step<FINITE>(v, n, below, whole);
        b = int(n >> BIN_SHIFT);
        return any;
    }
    // 2^(S - x / STEPS) = table[n % STEPS] 2^-(n / STEPS) exp(-g log(2) / STEPS) for x = n + g.  The powers of two
    // go into the exponent; added to 2^52 a value below 2^47 is rounded to a whole number, which the low bits
    // of the sum hold.
    __device__ __forceinline__ u64 weight(const double* table, const Series& c, uint32_t n, double below, double whole) const {
        const double g = fma(below, rate, -whole);
        const double m = table[n & (STEPS - 1)] * fma(g, fma(g, fma(g, c.c3, c.c2), c.c1), 1.0);
        static_assert(STEPS == 256, "the powers of two are bits 8 and up of n, bits 20 and up of the exponent's word");
        const double w = __hiloint2double(__double2hiint(m) - int((n << 12) & 0xfff00000u), __double2loint(m));
        return u64(__double_as_longlong(w + 4503599627370496.0)) & 0xfffffffffffffull;
    }
    __device__ __forceinline__ u64 weight_of(const double* table, float v) const {
        uint32_t n;
        double below, whole;
        return step(v, n, below, whole) ? weight(table, Series(), n, below, whole) : 0;
    }
};
// 2^(scale - j / STEPS), by the bits of j.
__device__ __forceinline__ double table_entry(int j, int scale) {
    constexpr double ROOT[8] = {0.99729605608547012, 0.99459942348363317, 0.98922801319397555, 0.97857206208770013,
                                0.95760328069857365, 0.91700404320467123, 0.84089641525371454, 0.70710678118654752};
    double v = ldexp(1.0, scale);
#pragma unroll
    for (int k = 0; k < 8; ++k) v *= (j >> k) & 1 ? ROOT[k] : 1.0;
    return v;
}

// A row's controls.
struct Controls {
    float temperature, top_p;
    int top_k;
    u64 least;        // smallest weight that min-p keeps; 0: off
    bool counts, masses;  // which histograms the row needs

    __device__ __forceinline__ Controls(const SampleParams& p, int r) {
        temperature = p.temperature ? p.temperature[r] : 1.0f;
        top_p = p.top_p ? p.top_p[r] : 1.0f;
        top_k = p.top_k ? p.top_k[r] : 0;
        const float min_p = p.min_p ? p.min_p[r] : 0.0f;
        least = min_p > 0.0f ? u64(ceil(ldexp(double(fminf(min_p, 1.0f)), weight_scale(p.n)))) : 0;
        counts = top_k > 0;
        masses = !(top_k > 0 && top_k <= LIST_TOP_K);
    }
    __device__ __forceinline__ bool greedy() const { return !(temperature > 0.0f); }
    __device__ __forceinline__ float share(const SampleParams& p, int r) const {
        const float u = p.uniform[r];
        return u > 0.0f ? fminf(u, 1.0f) : 0.0f;
    }
};

// Histograms of n elements in LDS, and the sum of the weights of at least `least`.
template <int TYPE, int NT, bool FINITE>
__device__ __forceinline__ u64 fill_bins(const void* base, int n, const Weights& w, const double* table, bool counts,
                                         bool masses, u64 least, u64* bin_mass, uint32_t* bin_count) {
    u64 kept = 0;
    Series series;
    series.hold();
    // what weighs nothing is computed along (from any table entry), not branched around
    auto add = [&](float v, bool& any) {
        uint32_t n;
        double below, whole;
        any = w.step<FINITE>(v, n, below, whole);
        const u64 weight = w.weight(table, series, n, below, whole);
        if (any) {
            atomicAdd(&bin_mass[n >> BIN_SHIFT], weight);
            if (!FINITE && counts) atomicAdd(&bin_count[n >> BIN_SHIFT], 1u);
        }
        return weight;
    };
    if (masses && least) {
        for_row<TYPE, NT, 2, true>(base, n, [&](int, float v) {
            bool any;
            const u64 weight = add(v, any);
            kept += any && weight >= least ? weight : 0;
        });
    } else if (masses) {
        for_row<TYPE, NT, 2, true>(base, n, [&](int, float v) {
            bool any;
            add(v, any);
        });
    } else {
        for_row<TYPE, NT, 2, true>(base, n, [&](int, float v) {
            int b;
            if (w.bin<FINITE>(v, b)) atomicAdd(&bin_count[b], 1u);
        });
    }
    return kept;
}

// A border: the first token up to which so many tokens, or so much weight, lie.
struct Goal {
    bool counted;
    u64 value;
    __device__ __forceinline__ bool reached(Sum upto) const { return (counted ? u64(upto.count) : upto.mass) >= value; }
};

// Bitonic steps of strides j, j / 2 .. 1 for place i of runs of k, between lanes.
__device__ __forceinline__ u64 exchange(u64 x, uint32_t i, uint32_t k, uint32_t j) {
#pragma unroll 1
    for (; j > 0; j >>= 1) {
        const u64 y = __shfl_xor(x, int(j), 64);
        // the lower place of an ascending run keeps the smaller one
        const bool smaller = ((i & k) == 0) == ((i & j) == 0);
        x = (y < x) == smaller ? y : x;
    }
    return x;
}

// The list's tokens (s.listed of them) in order, from registers: by buckets, each token in its place and counted by
// how many of its bucket are ahead.  False where a bucket has too many for that.  Buckets are logits and, where there
// are fewer of these, as of 16-bit types with many equal ones, ranges of ids within; else of the weights' logarithms.
__device__ __forceinline__ bool sort_by_buckets(Shared& s, const Weights& w, int n) {
    static_assert(BUCKETS == 2 * THREADS && LIST == 2 * THREADS, "two for each thread");
    const uint32_t tid = threadIdx.x, count = s.listed;
    u64 x[2];
    uint32_t at[2], low = 0xffffffffu, high = 0, differ = 0;
    const uint32_t any = uint32_t(s.order[0] >> 32);
    if (tid == 0) {
        s.low = 0xffffffffu;
        s.high = 0;
        s.queued = 0;
    }
#pragma unroll
    for (uint32_t e = 0; e < 2; ++e) {
        const uint32_t i = tid + e * THREADS;
        x[e] = i < count ? s.order[i] : s.order[0];
        at[e] = uint32_t(x[e] >> 32);
        low = min(low, at[e]);
        high = max(high, at[e]);
        differ |= at[e] ^ any;
        s.bucket[i] = 0;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        low = min(low, uint32_t(__shfl_xor(low, o, 64)));
        high = max(high, uint32_t(__shfl_xor(high, o, 64)));
        differ |= uint32_t(__shfl_xor(differ, o, 64));
    }
    __syncthreads();
    if ((tid & 63) == 0) {
        atomicMin(&s.low, low);
        atomicMax(&s.high, high);
        atomicOr(&s.queued, differ);
    }
    __syncthreads();
    low = s.low;
    high = s.high;
    // the bits below those in which keys differ are the same in all
    const int same = s.queued ? __ffs(int(s.queued)) - 1 : 31;
    const uint32_t span = (high - low) >> same;
    if (span < uint32_t(BUCKETS)) {
        const int id_bits = 32 - __clz(n), more = min(31 - __clz(BUCKETS / int(span + 1)), id_bits);
#pragma unroll
        for (uint32_t e = 0; e < 2; ++e) at[e] = ((at[e] - low) >> same) << more | uint32_t(x[e]) >> (id_bits - more);
    } else {
        auto step = [&](uint32_t key) {
            uint32_t t;
            double below, whole;
            w.step(key_value(key), t, below, whole);
            return t;
        };
        const uint32_t first = step(low), range = step(high) - first;
        int shift = 0;
        while (range >> shift >= uint32_t(BUCKETS)) ++shift;
#pragma unroll
        for (uint32_t e = 0; e < 2; ++e) at[e] = (step(at[e]) - first) >> shift;
    }
#pragma unroll
    for (uint32_t e = 0; e < 2; ++e)
        if (tid + e * THREADS < count) atomicAdd(&s.bucket[at[e]], 1u);
    __syncthreads();
    const uint32_t own[2] = {s.bucket[2 * tid], s.bucket[2 * tid + 1]};
    if (__syncthreads_or(max(own[0], own[1]) > BUCKET_MOST)) return false;
    Sum total;
    const Sum incl = block_scan<THREADS>({own[0] + own[1], 0}, s.waves, total);
    s.bucket[2 * tid] = incl.count - own[0] - own[1];
    s.bucket[2 * tid + 1] = incl.count - own[1];
    __syncthreads();
#pragma unroll
    for (uint32_t e = 0; e < 2; ++e)
        if (tid + e * THREADS < count) s.weight[atomicAdd(&s.bucket[at[e]], 1u)] = x[e];
    __syncthreads();
#pragma unroll 1
    for (uint32_t e = 0; e < 2; ++e) {
        if (tid + e * THREADS < count) {
            const uint32_t begin = at[0] ? s.bucket[at[0] - 1] : 0, end = s.bucket[at[0]];
            uint32_t place = begin;
#pragma unroll 4
            for (uint32_t j = begin; j < end; ++j) place += s.weight[j] < x[0];
            s.order[place] = x[0];
        }
        x[0] = x[1];
        at[0] = at[1];
    }
    return true;
}

// The list's tokens in order: strides of a wave and more through LDS, shorter ones between lanes.
__device__ __forceinline__ void sort_by_exchange(Shared& s) {
    const uint32_t tid = threadIdx.x, count = s.listed;
    uint32_t size = 64;
    while (size < count) size <<= 1;
    for (uint32_t i = count + tid; i < size; i += THREADS) s.order[i] = ~u64(0);
    __syncthreads();
#pragma unroll 1
    for (uint32_t k = 64; k <= size; k <<= 1) {
#pragma unroll 1
        for (uint32_t j = k >> 1; j >= 64; j >>= 1) {
            for (uint32_t t = tid; t < size / 2; t += THREADS) {
                const uint32_t a = (t & ~(j - 1)) * 2 + (t & (j - 1)), b = a + j;
                const u64 x = s.order[a], y = s.order[b];
                if ((x > y) == ((a & k) == 0)) {
                    s.order[a] = y;
                    s.order[b] = x;
                }
            }
            __syncthreads();
        }
#pragma unroll 1
        for (uint32_t i = tid; i < size; i += THREADS) {
            u64 x = s.order[i];
            // the first time, all runs up to 64
#pragma unroll 1
            for (uint32_t run = k == 64 ? 2 : k; run <= k; run <<= 1) x = exchange(x, i, run, min(run >> 1, 32u));
            s.order[i] = x;
        }
        __syncthreads();
    }
}

// The list's tokens in order, and inclusive sums of their weights.
__device__ __forceinline__ void sort_list(Shared& s, const Weights& w, int n) {
    const uint32_t tid = threadIdx.x, count = s.listed;
    constexpr uint32_t FEW = 256;
    if (count <= FEW) {
        // each token's place and sum from those before it, counted by four or more threads: the other ways, a barrier or
        // a lane exchange after the other, take 3 us however few there are (64 rows of a top-p of 0.5 35.4 us, 36.1 with
        // 128 for this; with 512, 0.9 takes 53 for 40)
        u64 *weights = s.weight + FEW, *order = s.weight + 2 * FEW;  // as they were listed
        if (tid < count) {
            const u64 x = s.order[tid];
            weights[tid] = w.weight_of(s.table, key_value(uint32_t(x >> 32)));
            order[tid] = x;
        }
        __syncthreads();
        const uint32_t share = count <= FEW / 4 ? 16 : count <= FEW / 2 ? 8 : 4;
        const uint32_t i = tid / share, part = tid % share;
        if (i < count) {
            const u64 x = order[i];
            Sum before = {0, 0};
#pragma unroll 4
            for (uint32_t j = part; j < count; j += share) {
                const bool ahead = order[j] < x;
                before.count += ahead;
                before.mass += ahead ? weights[j] : 0;
            }
            for (uint32_t o = 1; o < share; o <<= 1) {
                before.count += __shfl_xor(before.count, int(o), 64);
                before.mass += __shfl_xor(before.mass, int(o), 64);
            }
            if (part == 0) {
                s.order[before.count] = x;
                s.weight[before.count] = before.mass + weights[i];
            }
        }
        __syncthreads();
        return;
    }
    if (!sort_by_buckets(s, w, n)) sort_by_exchange(s);
    __syncthreads();
    const uint32_t i = 2 * tid;
    u64 weight[2];
#pragma unroll 1
    for (uint32_t e = 0; e < 2; ++e) {
        weight[1] = i + e < count ? w.weight_of(s.table, key_value(uint32_t(s.order[i + e] >> 32))) : 0;
        if (e == 0) weight[0] = weight[1];
    }
    Sum total;
    const Sum incl = block_scan<THREADS>({0, weight[0] + weight[1]}, s.waves, total);
    if (i < count) {  // i + 1 is a place of the list too
        s.weight[i] = incl.mass - weight[1];
        s.weight[i + 1] = incl.mass;
    }
    __syncthreads();
}

// The border among the sorted list's tokens from `from` to before `to`, `base` before the first of them;
// the result is in s.found, s.found_id and s.found_weight.
__device__ __forceinline__ void search_list(Shared& s, Sum base, Goal goal, uint32_t from, uint32_t to) {
    base.mass -= from ? s.weight[from - 1] : 0;
    for (uint32_t i = from + threadIdx.x; i < to; i += THREADS) {
        const u64 before = i ? s.weight[i - 1] : 0;
        const Sum upto = {base.count + i - from + 1, base.mass + s.weight[i]};
        if (goal.reached(upto) && !goal.reached({upto.count - 1, base.mass + before})) {
            s.found = upto;
            s.found_id = uint32_t(s.order[i]);
            s.found_weight = s.weight[i] - before;
        }
    }
    __syncthreads();
}

// All of the list's tokens; s.min_mass: those of at least `least`.
__device__ __forceinline__ Sum list_sum(Shared& s, u64 least) {
    if (least) {
        for (uint32_t i = threadIdx.x; i < s.listed; i += THREADS) {
            const u64 own = s.weight[i] - (i ? s.weight[i - 1] : 0);
            if (own >= least && (i + 1 == s.listed || s.weight[i + 1] - s.weight[i] < least)) s.min_mass = s.weight[i];
        }
        __syncthreads();
    }
    return {s.listed, s.weight[s.listed - 1]};
}

template <int TYPE>
struct Row {
    const void* base;
    int n;
    Weights w;
};

// The least and largest value of bins first .. last, by a table step more at each end.
struct Window {
    float low, high;
    __device__ __forceinline__ bool has(float v) const { return v >= low && v <= high; }
};
__device__ __forceinline__ Window bin_window(const Weights& w, int first, int last) {
    if (w.infinite()) return {NEG_INF, -NEG_INF};
    return {__double2float_rd(double(w.top) - double(((last + 1) << BIN_SHIFT) + 1) / w.rate),
            __double2float_ru(double(w.top) - double((first << BIN_SHIFT) - 1) / w.rate)};
}

// What is listed: the tokens in either window, and of bins first .. last or `extra` (past `last`; below 0:
// none) where first <= last.
struct Wanted {
    Window one, two;
    int first, last, extra;
    __device__ __forceinline__ void bins(const Weights& w, int from, int to, int other) {
        first = from;
        last = to;
        extra = other;
        one = bin_window(w, from, to);
        two = other < 0 ? one : bin_window(w, other, other);
    }
    __device__ __forceinline__ bool near(float v) const { return one.has(v) || two.has(v); }
    __device__ __forceinline__ bool has(const Weights& w, float v) const {
        int bin = 0;
        return near(v) && (first > last || (w.bin(v, bin) && ((bin >= first && bin <= last) || bin == extra)));
    }
};

// take(id, value) for the wanted ones of n elements.  First the 16 bytes that may hold any are queued, then
// these are taken apart: few are, but in most waves some lane's.  False if the queue (of `room`) overflows.
template <int TYPE, int NT, int AHEAD, typename F>
__device__ __forceinline__ bool gather(const void* base, int n, const Weights& weights, const Wanted& wanted, uint32_t* queued,
                                       uint32_t* queue, uint32_t room, F take) {
    typedef typename Element<TYPE>::T T;
    constexpr int PER = 16 / sizeof(T);
    const T* x = static_cast<const T*>(base);
    const int tid = threadIdx.x;
    const int head = min(n, int(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T)));
    const int vectors = (n - head) / PER, tail = head + vectors * PER, rest = head + n - tail;
    const uint4* body = reinterpret_cast<const uint4*>(x + head);
    __syncthreads();
    if (tid == 0) *queued = 0;
    __syncthreads();
    for (int i = tid; i < vectors; i += NT * AHEAD) {
        uint4 w[AHEAD];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) w[a] = body[min(i + a * NT, vectors - 1)];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            const uint32_t words[4] = {w[a].x, w[a].y, w[a].z, w[a].w};
            bool any = false;
#pragma unroll
            for (int j = 0; j < PER; ++j)
                any |= wanted.near(Element<TYPE>::value(PER == 4 ? words[j % 4] : words[j / 2] >> (j & 1) * 16));
            if (any && i + a * NT < vectors) {
                const uint32_t at = atomicAdd(queued, 1u);
                if (at < room) queue[at] = uint32_t(i + a * NT);
            }
        }
    }
    __syncthreads();
    const uint32_t pieces = *queued;
    if (pieces > room) return false;
    auto look = [&](int id, float v) {
        if (wanted.has(weights, v)) take(id, v);
    };
    for (uint32_t e = tid; e < pieces; e += NT) {
        uint4 w = body[queue[e]];
        int id = head + int(queue[e]) * PER;
#pragma unroll 1
        for (int j = 0; j < 4; ++j) {
            look(id++, Element<TYPE>::value(w.x));
            if constexpr (PER == 8) look(id++, Element<TYPE>::value(w.x >> 16));
            w = make_uint4(w.y, w.z, w.w, 0);
        }
    }
    if (tid < rest) {
        const int id = tid < head ? tid : tail + tid - head;
        look(id, Element<TYPE>::value(x[id]));
    }
    __syncthreads();
    return true;
}

// A row's wanted tokens in the list, sorted if it holds them; else s.listed is more than that.
template <int TYPE>
__device__ __forceinline__ void list_row(Shared& s, const Row<TYPE>& row, const Wanted& wanted) {
    __syncthreads();
    if (threadIdx.x == 0) s.listed = 0;
    const bool all = gather<TYPE, THREADS, 4>(row.base, row.n, row.w, wanted, &s.queued, reinterpret_cast<uint32_t*>(s.weight),
                                              2 * LIST, [&](int id, float v) {
                                                  const uint32_t at = atomicAdd(&s.listed, 1u);
                                                  if (at < LIST) s.order[at] = u64(sort_key(v)) << 32 | uint32_t(id);
                                              });
    if (!all) {  // more 16 bytes than the list has places, each of which holds a token
        if (threadIdx.x == 0) s.listed = LIST + 1;
        __syncthreads();
    }
    if (s.listed <= LIST) sort_list(s, row.w, row.n);
}

// Where the extra bin's tokens begin in the list.
__device__ __forceinline__ void split_list(Shared& s, const Weights& w, int extra) {
    if (threadIdx.x == 0) s.split = s.listed;
    __syncthreads();
    if (extra < 0) return;
    auto bin = [&](uint32_t i) {
        int b;
        w.bin(key_value(uint32_t(s.order[i] >> 32)), b);
        return b;
    };
    for (uint32_t i = threadIdx.x; i < s.listed; i += THREADS)
        if (bin(i) == extra && (i == 0 || bin(i - 1) != extra)) s.split = i;
    __syncthreads();
}

// The token that is the `index`-th, by id, of those of one logit (`key`).
template <int TYPE>
__device__ __forceinline__ void find_equal(Shared& s, const Row<TYPE>& row, uint32_t key, uint32_t index) {
    typedef typename Element<TYPE>::T T;
    const T* x = static_cast<const T*>(row.base);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int each = (row.n + WAVES * 64 - 1) / (WAVES * 64) * 64, begin = wave * each, end = min(row.n, begin + each);
    const float logit = key_value(key);
    auto equal = [&](T w) { return Element<TYPE>::value(w) == logit; };
    uint32_t own = 0;
    for (int i = begin; i < end; i += 64) {
        const bool same = i + lane < end && equal(x[i + lane]);
        own += uint32_t(__popcll(__ballot(same)));
    }
    __syncthreads();
    if (lane == 0) s.wave_id[wave] = own;
    __syncthreads();
    uint32_t before = 0;
    for (int w = 0; w < wave; ++w) before += s.wave_id[w];
    if (index >= before && index < before + own)
        for (int i = begin; i < end; i += 64) {
            const bool same = i + lane < end && equal(x[i + lane]);
            const u64 mask = __ballot(same);
            const uint32_t here = uint32_t(__popcll(mask));
            if (index < before + here) {
                if (same && before + uint32_t(__popcll(mask & ((u64(1) << lane) - 1))) == index) s.found_id = uint32_t(i + lane);
                break;
            }
            before += here;
        }
    __syncthreads();
}

// The border within a bin of more tokens than the list holds: narrows the bin's keys to low .. high, with
// `base` before them, until the list holds them (true), or they are one logit's: then the border is found.
template <int TYPE>
__device__ __forceinline__ bool divide_bin(Shared& s, const Row<TYPE>& row, int bin, Sum& base, Goal goal, uint32_t& low,
                                           uint32_t& high) {
    const int tid = threadIdx.x;
    u64* mass = s.order;  // the list is not in use
    uint32_t* count = reinterpret_cast<uint32_t*>(s.weight);
    __syncthreads();
    if (tid == 0) {
        s.low = 0xffffffffu;
        s.high = 0;
    }
    __syncthreads();
    low = 0xffffffffu;
    high = 0;
    for_row<TYPE, THREADS, 1, true>(row.base, row.n, [&](int, float v) {
        int b;
        if (!row.w.bin(v, b) || b != bin) return;
        low = min(low, sort_key(v));
        high = max(high, sort_key(v));
    });
    atomicMin(&s.low, low);
    atomicMax(&s.high, high);
    __syncthreads();
    low = s.low;
    high = s.high;
    uint32_t held = 0xffffffffu;
    while (held > uint32_t(LIST) && low < high) {
        int shift = 0;
        while ((high - low) >> shift >= SUB) ++shift;
        for (int i = tid; i < SUB; i += THREADS) {
            mass[i] = 0;
            count[i] = 0;
        }
        __syncthreads();
        const float least = key_value(high), most = key_value(low);
        for_row<TYPE, THREADS, 1, true>(row.base, row.n, [&](int, float v) {
            if (!(v >= least && v <= most)) return;
            const uint32_t key = sort_key(v);
            atomicAdd(&count[(key - low) >> shift], 1u);
            atomicAdd(&mass[(key - low) >> shift], row.w.weight_of(s.table, v));
        });
        __syncthreads();
        static_assert(SUB == THREADS, "one part for each thread");
        Sum total;
        const Sum own = {count[tid], mass[tid]}, incl = block_scan<THREADS>(own, s.waves, total);
        const Sum upto = {base.count + incl.count, base.mass + incl.mass};
        const Sum before = {upto.count - own.count, upto.mass - own.mass};
        if (goal.reached(upto) && !goal.reached(before)) {
            s.found_bin[0] = tid;
            s.found = before;
            s.listed = own.count;
        }
        __syncthreads();
        const uint32_t part = uint32_t(s.found_bin[0]);
        base = s.found;
        held = s.listed;
        high = min(high, low + (((part + 1) << shift) - 1));
        low += part << shift;
        __syncthreads();
    }
    if (held <= uint32_t(LIST)) return true;
    // one logit: every token has the same weight
    const u64 w = row.w.weight_of(s.table, key_value(low));
    const u64 index = goal.counted ? goal.value - base.count - 1 : (goal.value - base.mass + w - 1) / w - 1;
    find_equal(s, row, low, uint32_t(index));
    if (tid == 0) {
        s.found = {uint32_t(base.count + index + 1), base.mass + (index + 1) * w};
        s.found_weight = w;
    }
    __syncthreads();
    return false;
}

// A row's histograms in LDS.
struct Bins {
    u64* mass;
    uint32_t* count;
    int* found;

    __device__ __forceinline__ Sum upto(int b) const { return {count[b], mass[b]}; }
    __device__ __forceinline__ Sum before(int b) const { return {b ? count[b - 1] : 0, b ? mass[b - 1] : 0}; }

    // Inclusive sums in place -> all tokens' count and mass.  Where tokens were not counted, twice their number
    // at most is estimated by the power of two below the bin's weights.
    template <int NT>
    __device__ __forceinline__ Sum add_up(Sum* waves, int scale, bool counts) const {
        constexpr int EACH = (BINS + NT - 1) / NT;
        __syncthreads();
        const int first = threadIdx.x * EACH;
        Sum own[EACH], sum = {0, 0}, total;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int b = first + i;
            own[i] = {0, 0};
            if (b < BINS) own[i] = {count[b], mass[b]};
            if (!counts)
                own[i].count = uint32_t(min(own[i].mass >> max(scale - ((b + 1) * (1 << BIN_SHIFT) + STEPS - 1) / STEPS, 0), u64(1) << 20));
            sum = {sum.count + own[i].count, sum.mass + own[i].mass};
        }
        const Sum incl = block_scan<NT>(sum, waves, total);
        Sum run = {incl.count - sum.count, incl.mass - sum.mass};
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            run = {run.count + own[i].count, run.mass + own[i].mass};
            if (first + i < BINS) {
                count[first + i] = run.count;
                mass[first + i] = run.mass;
            }
        }
        __syncthreads();
        return total;
    }

    // The bins of two borders, or of one, in every thread.
    template <int NT>
    __device__ __forceinline__ int2 borders(Goal one, Goal two) const {
        __syncthreads();
        for (int b = threadIdx.x; b < BINS; b += NT) {
            const Sum until = upto(b), ahead = before(b);
            if (one.reached(until) && !one.reached(ahead)) found[0] = b;
            if (two.reached(until) && !two.reached(ahead)) found[1] = b;
        }
        __syncthreads();
        return make_int2(found[0], found[1]);
    }
    template <int NT>
    __device__ __forceinline__ int border(Goal goal) const { return borders<NT>(goal, goal).x; }
};

__device__ __forceinline__ Goal top_p_goal(float top_p, u64 mass) {
    const double part = ceil(double(top_p) * double(mass));
    return {false, part > 1.0 ? u64(part) : u64(1)};
}
// Of a number in [0, 1] of the weight that is kept.
__device__ __forceinline__ Goal draw_goal(float share, u64 mass) {
    return {false, min(u64(double(share) * double(mass)), mass - 1) + 1};
}

// Which bins a border's search lists, given its own.  UPTO: all up to it if they fit, so that further borders
// need no pass; else the bin alone.  For a top-p the drawn token's as well: where it is, is known but for what
// the top-p's bin adds to the weight, which moves it by a bin at most, as a rule.  False where the drawn token's
// may not be among them.
template <int NT, bool UPTO>
__device__ __forceinline__ bool choose_bins(const Bins& bins, int bin, bool top_p, u64 most, float share, int& first, int& last,
                                            int& extra) {
    first = UPTO && bins.count[bin] <= uint32_t(LIST) ? 0 : bin;
    last = bin;
    extra = -1;
    if (!top_p || (UPTO && first == 0)) return true;
    const u64 least = min(bins.before(bin).mass, most), full = min(bins.mass[bin], most);
    const int2 drawn = bins.borders<NT>(draw_goal(share, max(least, u64(1))), draw_goal(share, full));
    const int one = drawn.x, two = drawn.y;
    uint32_t held = bins.count[two] - bins.before(one).count;
    if (two < bin) held += bins.count[bin] - bins.before(bin).count;
    if (held > uint32_t(LIST)) return false;
    first = one;
    last = two;
    extra = two < bin ? bin : -1;
    return true;
}

template <int TYPE>
__device__ __forceinline__ const void* row_base(const SampleParams& p, int r) {
    return static_cast<const typename Element<TYPE>::T*>(p.logits) + r * p.stride;
}

template <int TYPE>
__device__ __forceinline__ const void* segment_base(const SampleParams& p, int r, int begin) {
    return static_cast<const typename Element<TYPE>::T*>(row_base<TYPE>(p, r)) + begin;
}

// A row in the workspace.
struct Best {
    float value;
    uint32_t id;
};
struct Plan {
    bool listed;   // else the row is drawn from by one workgroup
    bool whole;    // all tokens that may be kept are in the list
    int extra;     // the list's bins: its last one, apart from the others (below 0: none is)
    Sum kept;      // before any border
    Sum base, extra_base;  // before the list's bins
};
struct RowState {
    u64 bins[BINS];    // sums of the weights, or numbers of tokens where no weights are summed
    u64 min_mass;
    uint32_t listed;
    Plan plan;
    u64 order[LIST];
};
__device__ __forceinline__ RowState& row_state(const SampleParams& p, int r) { return static_cast<RowState*>(p.workspace)[r]; }
__device__ __forceinline__ Best* row_best(const SampleParams& p, int r, int segments) {
    return reinterpret_cast<Best*>(static_cast<RowState*>(p.workspace) + p.rows) + int64_t(r) * segments;
}

// The largest logit of a segment; the row's sums begin at zero.
template <int TYPE>
__global__ __launch_bounds__(PART_THREADS) void sample_best_kernel(SampleParams p, int each) {
    __shared__ float s_values[PART_THREADS / 64];
    __shared__ uint32_t s_ids[PART_THREADS / 64];
    const int r = blockIdx.x, begin = blockIdx.y * each, n = min(each, p.n - begin);
    RowState& state = row_state(p, r);
    for (int i = blockIdx.y * PART_THREADS + threadIdx.x; i < BINS; i += gridDim.y * PART_THREADS) state.bins[i] = 0;
    if (blockIdx.y == 0 && threadIdx.x == 0) {
        state.min_mass = 0;
        state.listed = 0;
    }
    float best;
    uint32_t id;
    find_best<TYPE, PART_THREADS>(segment_base<TYPE>(p, r, begin), n, Controls(p, r).greedy(), best, id);
    block_best<PART_THREADS>(best, id, s_values, s_ids);
    if (threadIdx.x == 0) row_best(p, r, gridDim.y)[blockIdx.y] = {best, id == 0xffffffffu ? id : id + uint32_t(begin)};
}

// The row's largest logit from its segments', in every thread (a wave's lanes take a segment each).
__device__ __forceinline__ Best segments_best(const Best* segments, int count) {
    Best best = {NEG_INF, 0xffffffffu};
    for (int i = threadIdx.x & 63; i < count; i += 64)
        if (segments[i].value > best.value) best = segments[i];
    for (int o = 32; o > 0; o >>= 1) {
        const float v = __shfl_xor(best.value, o, 64);
        const uint32_t i = __shfl_xor(best.id, o, 64);
        if (v > best.value || (v == best.value && i < best.id)) best = {v, i};
    }
    best.value = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(best.value)));
    best.id = __builtin_amdgcn_readfirstlane(best.id);
    return best;
}

// A segment's histogram, added to the row's.
template <int TYPE>
__global__ __launch_bounds__(GROUP_THREADS) void sample_bins_kernel(SampleParams p, int segments, int each) {
    __shared__ double s_table[STEPS];
    __shared__ u64 s_mass[BINS];
    __shared__ uint32_t s_count[BINS];
    __shared__ u64 s_kept;
    const int r = blockIdx.x, tid = threadIdx.x;
    const Controls c(p, r);
    if (c.greedy()) return;
    for (int i = tid; i < STEPS; i += GROUP_THREADS) s_table[i] = table_entry(i, weight_scale(p.n));
    for (int i = tid; i < BINS; i += GROUP_THREADS) {
        s_mass[i] = 0;
        s_count[i] = 0;
    }
    if (tid == 0) s_kept = 0;
    const Best best = segments_best(row_best(p, r, segments), segments);
    if (best.id == 0xffffffffu || best.value == -NEG_INF) return;  // infinity is the last step's
    Weights w;
    w.set(best.value, c.temperature, p.n);
    __syncthreads();
    const int begin = blockIdx.y * each, n = min(each, p.n - begin);
    const u64 kept = fill_bins<TYPE, GROUP_THREADS, true>(segment_base<TYPE>(p, r, begin), n, w, s_table, false, c.masses, c.least,
                                                   s_mass, s_count);
    if (c.least && kept) atomicAdd(&s_kept, kept);
    __syncthreads();
    RowState& state = row_state(p, r);
    for (int i = tid; i < BINS; i += GROUP_THREADS) {
        const u64 sum = c.masses ? s_mass[i] : s_count[i];
        if (sum) atomicAdd(&state.bins[i], sum);
    }
    if (tid == 0 && s_kept) atomicAdd(&state.min_mass, s_kept);
}

// The bins to list, the same in every workgroup of a row, and a segment's tokens of them.
template <int TYPE>
__global__ __launch_bounds__(GROUP_THREADS) void sample_list_kernel(SampleParams p, int segments, int each) {
    constexpr int STAGE = 512, PIECES = 2 * LIST;
    __shared__ u64 s_mass[BINS];
    __shared__ uint32_t s_count[BINS];
    __shared__ Sum s_waves[GROUP_THREADS / 64];
    __shared__ u64 s_stage[STAGE];
    __shared__ uint32_t s_pieces[PIECES];
    __shared__ uint32_t s_queued, s_listed, s_at;
    __shared__ int s_found[2];
    const int r = blockIdx.x, tid = threadIdx.x;
    const Controls c(p, r);
    if (c.greedy()) return;
    RowState& state = row_state(p, r);
    for (int i = tid; i < BINS; i += GROUP_THREADS) {
        const u64 sum = state.bins[i];
        s_mass[i] = c.masses ? sum : 0;
        s_count[i] = c.masses ? 0 : uint32_t(sum);
    }
    const Best best = segments_best(row_best(p, r, segments), segments);
    if (best.id == 0xffffffffu) return;
    if (best.value == -NEG_INF) {
        if (blockIdx.y == 0 && tid == 0) state.plan.listed = false;
        return;
    }
    Weights w;
    w.set(best.value, c.temperature, p.n);
    const Bins bins = {s_mass, s_count, s_found};
    const u64 most = c.masses && c.least ? state.min_mass : ~u64(0);
    const float share = c.share(p, r);
    Plan plan;
    plan.kept = bins.add_up<GROUP_THREADS>(s_waves, w.scale, !c.masses);
    plan.whole = !c.masses;
    Goal goal;
    bool top_p = false;
    plan.listed = true;
    if (!c.masses) {
        goal = {true, min(u64(c.top_k), u64(plan.kept.count))};
    } else if (c.top_k > 0) {
        plan.listed = false;  // so many that weights and numbers are needed
    } else if (c.top_p < 1.0f) {
        goal = top_p_goal(c.top_p, plan.kept.mass);
        top_p = true;
    } else {
        goal = draw_goal(share, min(plan.kept.mass, most));
    }
    Wanted wanted;
    if (plan.listed) {
        const int bin = bins.border<GROUP_THREADS>(goal);
        int first, last, extra;
        if (plan.whole) {  // all up to the bin
            first = 0;
            last = bin;
            extra = -1;
            plan.listed = bins.count[bin] <= uint32_t(LIST);
        } else {
            plan.listed = choose_bins<GROUP_THREADS, false>(bins, bin, top_p, most, share, first, last, extra);
        }
        plan.extra = extra;
        plan.base = bins.before(first);
        plan.extra_base = bins.before(max(extra, 0));
        wanted.bins(w, first, last, extra);
    }
    if (blockIdx.y == 0 && tid == 0) state.plan = plan;
    if (!plan.listed) return;
    const int begin = blockIdx.y * each, n = min(each, p.n - begin);
    if (tid == 0) s_listed = 0;
    auto append = [&](uint32_t at, u64 entry) {
        if (at < uint32_t(LIST)) state.order[at] = entry;
    };
    const bool all = gather<TYPE, GROUP_THREADS, 4>(
        segment_base<TYPE>(p, r, begin), n, w, wanted, &s_queued, s_pieces, PIECES, [&](int id, float v) {
            const u64 entry = u64(sort_key(v)) << 32 | uint32_t(id + begin);
            const uint32_t at = atomicAdd(&s_listed, 1u);
            if (at < STAGE) s_stage[at] = entry;
            else append(atomicAdd(&state.listed, 1u), entry);
        });
    const uint32_t staged = min(s_listed, uint32_t(STAGE));
    if (tid == 0 && (staged || !all)) s_at = atomicAdd(&state.listed, all ? staged : LIST + 1u);
    __syncthreads();
    if (all)
        for (uint32_t i = tid; i < staged; i += GROUP_THREADS) append(s_at + i, s_stage[i]);
}

// One workgroup's work on a whole row: all four steps.
template <int TYPE>
__device__ __forceinline__ void draw_from_row(Shared& s, const SampleParams& p, const Controls& c, Row<TYPE>& row, float share,
                                              u64& kept_mass) {
    const int tid = threadIdx.x;
    const Bins bins = {s.bin_mass, s.bin_count, s.found_bin};
    // The borders one after the other: of the top-k, of the top-p, the drawn token's.  A small top-k's
    // tokens are listed first of all, with what shares the last one's bin; should too many do, weights are
    // summed after all and all begins again.
    enum Stage { LIST_ALL, TOP_K, TOP_P, DRAW, DONE };
    bool counts = c.counts, masses = c.masses;
    Sum kept;
    int stage;
    do {
        for (int b = tid; b < BINS; b += THREADS) {
            s.bin_mass[b] = 0;
            s.bin_count[b] = 0;
        }
        if (tid == 0) s.min_mass = 0;
        __syncthreads();
        const u64 enough = fill_bins<TYPE, THREADS, false>(row.base, p.n, row.w, s.table, counts, masses, c.least, s.bin_mass, s.bin_count);
        if (c.least && enough) atomicAdd(&s.min_mass, enough);
        kept = bins.add_up<THREADS>(s.waves, row.w.scale, counts);
        // the list holds bins first .. last (none: first > last) and `extra`, or all tokens that may be kept
        int first = 1, last = 0, extra = -1;
        bool whole = false;
        for (stage = masses ? TOP_K : LIST_ALL; stage < DONE; ++stage) {
            Goal goal = {false, 1};
            if (stage == LIST_ALL) {
                goal = {true, min(u64(c.top_k), u64(kept.count))};
            } else if (stage == TOP_K) {
                if (c.top_k <= 0 || uint32_t(c.top_k) >= kept.count) continue;
                goal = {true, u64(c.top_k)};
            } else if (stage == TOP_P) {
                if (!(c.top_p < 1.0f)) continue;
                goal = top_p_goal(c.top_p, kept.mass);
            } else {
                if (c.least) kept.mass = min(kept.mass, s.min_mass);  // both are beginnings of one order
                goal = draw_goal(share, kept.mass);
            }
            // of a list: the border lies from `from` to before `to`, `base` before that
            uint32_t from = 0, to = 0;
            Sum base = {0, 0};
            bool found = false;
            if (!whole) {
                const int bin = bins.border<THREADS>(goal);
                if (bin != extra && (bin < first || bin > last)) {
                    choose_bins<THREADS, true>(bins, bin, stage == TOP_P, c.least ? s.min_mass : ~u64(0), share, first, last, extra);
                    if (stage == LIST_ALL) first = 0;
                    Wanted wanted;
                    wanted.bins(row.w, first, last, extra);
                    while (true) {
                        list_row(s, row, wanted);
                        if (s.listed <= uint32_t(LIST) || stage == LIST_ALL) break;
                        if (first < last || extra >= 0) {
                            // the numbers of tokens were estimates: the bin alone
                            first = last = bin;
                            extra = -1;
                            wanted.bins(row.w, bin, bin, -1);
                            continue;
                        }
                        uint32_t low_key, high_key;
                        base = bins.before(bin);
                        first = wanted.first = 1;  // what is listed now is of no other border's use
                        last = wanted.last = 0;
                        found = !divide_bin(s, row, bin, base, goal, low_key, high_key);
                        if (found) break;
                        wanted.one = wanted.two = {key_value(high_key), key_value(low_key)};
                    }
                    if (stage == LIST_ALL && s.listed > uint32_t(LIST)) break;
                    if (!found) split_list(s, row.w, extra);
                }
                if (first <= last) base = bins.before(bin == extra ? bin : first);
                from = bin == extra ? s.split : 0;
                to = bin == extra ? s.listed : s.split;
            } else {
                __syncthreads();
                to = s.listed;
            }
            if (!found && stage != LIST_ALL) search_list(s, base, goal, from, to);
            if (stage == LIST_ALL) {
                whole = true;
                kept = list_sum(s, c.least);
            } else if (stage != DRAW) {
                kept = s.found;
            }
        }
        if (stage == LIST_ALL) counts = masses = true;
    } while (stage < DONE);
    kept_mass = kept.mass;
}

// The rest of a row.  LISTED: its first three steps are done, in `segments` parts, but where the list could
// not hold what it had to.
template <int TYPE, bool LISTED>
__global__ __launch_bounds__(THREADS) void sample_draw_kernel(SampleParams p, int segments) {
    __shared__ Shared s;
    const int r = blockIdx.x, tid = threadIdx.x;
    Row<TYPE> row;
    row.base = row_base<TYPE>(p, r);
    row.n = p.n;
    const Controls c(p, r);
    Best best;
    if constexpr (LISTED) {
        best = segments_best(row_best(p, r, segments), segments);
    } else {
        find_best<TYPE, THREADS>(row.base, p.n, c.greedy(), best.value, best.id);
        block_best<THREADS>(best.value, best.id, s.wave_value, s.wave_id);
    }
    if (best.id == 0xffffffffu || c.greedy()) {
        if (tid == 0) {
            p.token[r] = int32_t(best.id);  // -1 where nothing can be drawn
            if (p.prob) p.prob[r] = best.id == 0xffffffffu ? 0.0f : 1.0f;
        }
        return;
    }
    row.w.set(best.value, c.temperature, p.n);
    if (tid < STEPS) s.table[tid] = table_entry(tid, row.w.scale);
    const float share = c.share(p, r);
    u64 kept_mass = 0;
    bool done = false;
    if constexpr (LISTED) {
        const RowState& state = row_state(p, r);
        const Plan plan = state.plan;
        const uint32_t listed = state.listed;
        if (plan.listed && listed <= uint32_t(LIST)) {
            for (uint32_t i = tid; i < listed; i += THREADS) s.order[i] = state.order[i];
            if (tid == 0) {
                s.listed = listed;
                s.min_mass = state.min_mass;
            }
            __syncthreads();
            sort_list(s, row.w, p.n);
            split_list(s, row.w, plan.extra);
            Sum kept = plan.whole ? list_sum(s, c.least) : plan.kept;
            // a border in the extra bin has more weight before it than there is before the bin
            auto search = [&](Goal goal) {
                const bool extra = plan.extra >= 0 && !goal.counted && goal.value > plan.extra_base.mass;
                __syncthreads();
                search_list(s, extra ? plan.extra_base : plan.base, goal, extra ? s.split : 0, extra ? s.listed : s.split);
            };
            if (plan.whole && uint32_t(c.top_k) < listed) {
                search({true, u64(c.top_k)});
                kept = s.found;
            }
            if (c.top_p < 1.0f) {
                search(top_p_goal(c.top_p, kept.mass));
                kept = s.found;
            }
            if (c.least) kept.mass = min(kept.mass, s.min_mass);  // both are beginnings of one order
            search(draw_goal(share, kept.mass));
            kept_mass = kept.mass;
            done = true;
        }
    }
    if (!done) draw_from_row(s, p, c, row, share, kept_mass);
    if (tid == 0) {
        p.token[r] = int32_t(s.found_id);
        if (p.prob) p.prob[r] = float(double(s.found_weight) / double(kept_mass));
    }
}

// Whether a workgroup does a whole row by itself: where all rows' run at once, a CU holding one, and the row is
// short.  256 rows of 16,000 BF16 logits take 24 to 33 us so (by what is kept), 36 to 39 in four launches, 64 rows
// of 32,000 26 to 37 and 33 to 38; but 64 of 107,520 38 to 61 against 33 to 46, and 1,024 rows of 4,000 68 to
// 80 against 53 to 59.
bool row_alone(int rows, int n) { return rows <= 256 && n <= 32768; }
// Segments of a row: of 4,096 logits at least, and some 1,024 in all, which fill the CUs.
int row_segments(int rows, int n) { return std::max(1, std::min((n + 4095) / 4096, 1024 / rows)); }
// Workgroups that fill histograms, and that list, over all rows: 128 FP32 rows take 18.7 and 18.0 us so, 24.8
// and 30.3 with 2,048 of 256 threads, each of which adds its histogram to the row's and adds the row's up.
constexpr int GROUPS = 512;

template <int TYPE>
void run_sample(const SampleParams& p, hipStream_t s) {
    if (row_alone(p.rows, p.n)) {
        hipLaunchKernelGGL((sample_draw_kernel<TYPE, false>), dim3(unsigned(p.rows)), dim3(THREADS), 0, s, p, 0);
        return;
    }
    int segments = row_segments(p.rows, p.n);
    const int each = (p.n + segments * 64 - 1) / (segments * 64) * 64;
    segments = (p.n + each - 1) / each;
    hipLaunchKernelGGL((sample_best_kernel<TYPE>), dim3(unsigned(p.rows), unsigned(segments)), dim3(PART_THREADS), 0, s, p, each);
    const int bins = std::max(1, std::min(segments, GROUPS / p.rows)), part = (p.n + bins * 64 - 1) / (bins * 64) * 64;
    hipLaunchKernelGGL((sample_bins_kernel<TYPE>), dim3(unsigned(p.rows), unsigned((p.n + part - 1) / part)), dim3(GROUP_THREADS), 0, s,
                       p, segments, part);
    // each workgroup finds the bins for itself, which takes longer than a few more logits
    const int lists = std::max(1, std::min(segments, GROUPS / p.rows)), share = (p.n + lists * 64 - 1) / (lists * 64) * 64;
    hipLaunchKernelGGL((sample_list_kernel<TYPE>), dim3(unsigned(p.rows), unsigned((p.n + share - 1) / share)), dim3(GROUP_THREADS),
                       0, s, p, segments, share);
    hipLaunchKernelGGL((sample_draw_kernel<TYPE, true>), dim3(unsigned(p.rows)), dim3(THREADS), 0, s, p, segments);
}

}  // namespace

size_t sample_workspace(int rows, int n) {
    return row_alone(rows, n) ? 0 : size_t(rows) * (sizeof(RowState) + size_t(row_segments(rows, n)) * sizeof(Best));
}

void launch_sample(const SampleParams& p, int type, hipStream_t s) {
    if (type == TYPE_BF16) run_sample<TYPE_BF16>(p, s);
    else if (type == TYPE_F16) run_sample<TYPE_F16>(p, s);
    else run_sample<TYPE_F32>(p, s);
}

}  // namespace plamo
