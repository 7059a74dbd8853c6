// Tokens drawn from logits on gfx950: temperature, top-k, top-p and min-p, by given uniform numbers.
//
// A row's tokens are ordered by descending logit, equal ones by ascending id.  With weights
// e_i = exp((x_i - max x) / T): top-k keeps the first k; top-p of those the ones before which less than
// p of the kept weight lies; min-p of those the ones of at least min_p of the largest weight.  All three
// keep a beginning of the order.  The token is the first one up to which more than u of the kept weight
// lies.  Nothing is sorted but the few tokens around a border:
//   1. the largest logit;
//   2. a histogram over bins of the exponent (16 bins for a factor of two) in LDS: sums of the weights,
//      or, for a top-k of at most 1024, numbers of tokens, for which no exponential is taken;
//   3. prefix sums over the bins give the bin of each border; the tokens of that bin (or of all bins
//      up to it) are gathered, sorted in LDS and searched.  A bin of more tokens than the list holds
//      is divided again by the bits of the logits until it is small enough or one value.
// Steps 1 and 2 are spread over segments of a row (a launch each), as one row's 107,520 logits are 40 us
// of one CU's LDS atomics and FP64; the third is one workgroup's.
// Weights are whole multiples of 2^-S of the largest (S = 63 - log2 of the vocabulary, at most 46), so
// that all sums are exact whatever their order: the token depends on the row alone, not on how it was
// split, and sums of unsigned 64-bit atomics are the same in every run.  A token of less than 2^-(S+1)
// of the largest weight is never drawn.  exp is evaluated in FP64 to 2^-50: a token is told apart from
// its neighbour by sums over 100,000 of them, where FP32's 2^-24 would move the borders.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "common.h"
#include "device.h"
#include "paged.h"

namespace plamo {
using namespace dev;

namespace {

constexpr int THREADS = 1024, WAVES = THREADS / 64;  // of the workgroup that ends a row
constexpr int PART_THREADS = 256;    // of a segment's workgroup
constexpr int STEPS = 1024;          // table entries for a factor of two
constexpr int BIN_SHIFT = 6;         // log2 of a bin's table steps
constexpr int BINS = 768;            // 16 (S + 1) <= 752 are used
constexpr int LIST = 2048;           // tokens that are sorted at once
constexpr int LIST_TOP_K = 1024;     // a top-k up to which its tokens' weights are summed in the list
constexpr int SUB = 1024;            // parts that a bin is divided into again

typedef unsigned long long u64;

// Row values: NaN counts as minus infinity; minus zero equals zero.
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
__device__ __forceinline__ float plain(float v) { return v == v ? v + 0.0f : NEG_INF; }

// f(id, value) for n elements, a thread's in ascending order; 16 bytes a load behind the first
// aligned element.
template <int TYPE, int NT, typename F>
__device__ __forceinline__ void for_row(const void* base, int n, F f) {
    typedef typename Element<TYPE>::T T;
    constexpr int PER = 16 / sizeof(T), AHEAD = 4;
    const T* row = static_cast<const T*>(base);
    const int tid = threadIdx.x;
    const int head = min(n, int(((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / sizeof(T)));
    if (tid < head) f(tid, plain(Element<TYPE>::value(row[tid])));
    const int vectors = (n - head) / PER;
    const uint4* body = reinterpret_cast<const uint4*>(row + head);
    for (int i = tid; i < vectors; i += NT * AHEAD) {
        uint4 w[AHEAD];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a)
            if (i + a * NT < vectors) w[a] = body[i + a * NT];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            if (i + a * NT >= vectors) break;
            const int id = head + (i + a * NT) * PER;
            const uint32_t words[4] = {w[a].x, w[a].y, w[a].z, w[a].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (PER == 4) {
                    f(id + j, plain(Element<TYPE>::value(words[j])));
                } else {
                    f(id + 2 * j, plain(Element<TYPE>::value(words[j])));
                    f(id + 2 * j + 1, plain(Element<TYPE>::value(words[j] >> 16)));
                }
            }
        }
    }
    const int tail = head + vectors * PER + tid;
    if (tail < n) f(tail, plain(Element<TYPE>::value(row[tail])));
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
template <int TYPE, int NT>
__device__ __forceinline__ void find_best(const void* base, int n, float& best, uint32_t& id) {
    best = NEG_INF;
    id = 0xffffffffu;
    for_row<TYPE, NT>(base, n, [&](int i, float v) {
        if (v > best) {
            best = v;
            id = uint32_t(i);
        }
    });
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
    Sum waves[WAVES];
    float wave_value[WAVES];
    uint32_t wave_id[WAVES];
    uint32_t low, high, listed;
    Sum found;             // a border's count and mass up to and with its token
    uint32_t found_id;
    u64 found_weight;
    int found_bin;
    u64 min_mass;          // of the tokens of at least min_p
};

// Inclusive sums over the workgroup.
__device__ Sum block_scan(Sum v, Sum* waves, Sum& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t c = __shfl_up(v.count, o, 64);
        const u64 m = __shfl_up(v.mass, o, 64);
        if (lane >= o) {
            v.count += c;
            v.mass += m;
        }
    }
    __syncthreads();  // the sums of a scan before this one have been read
    if (lane == 63) waves[wave] = v;
    __syncthreads();
    total = {0, 0};
    for (int w = 0; w < WAVES; ++w) {
        if (w == wave) {
            v.count += total.count;
            v.mass += total.mass;
        }
        total.count += waves[w].count;
        total.mass += waves[w].mass;
    }
    return v;
}

// Descending logits as ascending 32-bit keys.
__device__ __forceinline__ uint32_t sort_key(float v) {
    const uint32_t u = __float_as_uint(v);
    return u & 0x80000000u ? u : ~(u | 0x80000000u);
}

__device__ __forceinline__ float key_value(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key : ~key & 0x7fffffffu);
}

// A row's weights.
struct Weights {
    float top;        // largest logit
    bool infinite;    // it is plus infinity: only such tokens have a weight
    double rate;      // STEPS log2(e) / T
    double limit;     // exponents from here on weigh nothing
    int scale;        // S

    __device__ __forceinline__ void set(float best, float temperature, int n) {
        scale = min(46, 31 + __clz(n));  // sums of n weights stay below 2^63
        top = best;
        infinite = best == -NEG_INF;
        rate = STEPS * 1.44269504088896340736 / double(temperature);
        limit = double((scale + 1) * STEPS) - 0.5;
    }
    __device__ __forceinline__ bool exponent(float v, double& x) const {
        if (infinite) v = v == top ? 0.0f : NEG_INF;
        x = (double(infinite ? 0.0f : top) - double(v)) * rate;
        return x < limit;  // false for minus infinity
    }
    static __device__ __forceinline__ int steps(double x) { return int(__builtin_rint(x)); }
    __device__ __forceinline__ u64 weight(const double* table, double x, int n) const {
        // 2^(-x / STEPS) = table[n % STEPS] 2^-(n / STEPS) exp(-f), |f| <= log(2) / (2 STEPS): the cubic
        // is off by f^4 / 24 < 2^-50.  Added to 2^52 a value below 2^47 is rounded to a whole number,
        // which the low bits of the sum then hold.
        const double f = (x - double(n)) * (0.69314718055994530942 / STEPS);
        const double e = 1.0 - f * (1.0 - f * (0.5 - f * (1.0 / 6.0)));
        const double w = ldexp(table[n & (STEPS - 1)] * e, scale - n / STEPS);
        return u64(__double_as_longlong(w + 4503599627370496.0)) & 0xfffffffffffffull;
    }
    __device__ __forceinline__ u64 weight_of(const double* table, float v) const {
        double x;
        return exponent(v, x) ? weight(table, x, steps(x)) : 0;
    }
};
__device__ __forceinline__ double table_entry(int j) { return exp2(-double(j) / STEPS); }

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
        least = min_p > 0.0f ? u64(ceil(ldexp(double(fminf(min_p, 1.0f)), min(46, 31 + __clz(p.n))))) : 0;
        counts = top_k > 0;
        masses = !(top_k > 0 && top_k <= LIST_TOP_K);
    }
    __device__ __forceinline__ bool greedy() const { return !(temperature > 0.0f); }
};

// Histograms of n elements in LDS, and the sum of the weights of at least `least`.
template <int TYPE, int NT>
__device__ __forceinline__ u64 fill_bins(const void* base, int n, const Weights& w, const double* table, bool counts,
                                         bool masses, u64 least, u64* bin_mass, uint32_t* bin_count) {
    u64 kept = 0;
    if (masses) {
        for_row<TYPE, NT>(base, n, [&](int, float v) {
            double x;
            if (!w.exponent(v, x)) return;
            const int step = Weights::steps(x);
            const u64 weight = w.weight(table, x, step);
            atomicAdd(&bin_mass[step >> BIN_SHIFT], weight);
            if (counts) atomicAdd(&bin_count[step >> BIN_SHIFT], 1u);
            if (weight >= least) kept += weight;
        });
    } else {
        for_row<TYPE, NT>(base, n, [&](int, float v) {
            double x;
            if (w.exponent(v, x)) atomicAdd(&bin_count[Weights::steps(x) >> BIN_SHIFT], 1u);
        });
    }
    return kept;
}

// A segment's results in the workspace.
struct Segment {
    u64 bin_mass[BINS];
    u64 min_mass;
    uint32_t bin_count[BINS];
    float best;
    uint32_t id;
};

enum Border { BORDER_COUNT, BORDER_MASS, BORDER_DRAW };

// Whether a token with these sums before it is the border, or lies behind it.
template <Border KIND>
__device__ __forceinline__ bool reached(Sum upto, u64 target) {
    return KIND == BORDER_COUNT ? upto.count >= target : KIND == BORDER_MASS ? upto.mass >= target : upto.mass > target;
}

template <int O>
__device__ __forceinline__ void exchange(u64& x, uint32_t i, uint32_t k) {
    const u64 y = u64(xor_lane<O>(uint32_t(x >> 32))) << 32 | xor_lane<O>(uint32_t(x));
    // the lower place of an ascending run keeps the smaller one
    const bool smaller = ((i & k) == 0) == ((i & O) == 0);
    x = (y < x) == smaller ? y : x;
}

// The list's tokens (s.listed of them) in order, bitonic: strides of a wave and more through LDS, shorter
// ones between lanes.  Then inclusive sums of the weights.
__device__ void sort_list(Shared& s, const Weights& w) {
    const uint32_t tid = threadIdx.x, count = s.listed;
    uint32_t size = 64;
    while (size < count) size <<= 1;
    for (uint32_t i = count + tid; i < size; i += THREADS) s.order[i] = ~u64(0);
    __syncthreads();
    for (uint32_t i = tid; i < size; i += THREADS) {
        u64 x = s.order[i];
        exchange<1>(x, i, 2);
        exchange<2>(x, i, 4), exchange<1>(x, i, 4);
        exchange<4>(x, i, 8), exchange<2>(x, i, 8), exchange<1>(x, i, 8);
        exchange<8>(x, i, 16), exchange<4>(x, i, 16), exchange<2>(x, i, 16), exchange<1>(x, i, 16);
        exchange<16>(x, i, 32), exchange<8>(x, i, 32), exchange<4>(x, i, 32), exchange<2>(x, i, 32), exchange<1>(x, i, 32);
        exchange<32>(x, i, 64), exchange<16>(x, i, 64), exchange<8>(x, i, 64), exchange<4>(x, i, 64);
        exchange<2>(x, i, 64), exchange<1>(x, i, 64);
        s.order[i] = x;
    }
    __syncthreads();
    for (uint32_t k = 128; k <= size; k <<= 1) {
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
        for (uint32_t i = tid; i < size; i += THREADS) {
            u64 x = s.order[i];
            exchange<32>(x, i, k), exchange<16>(x, i, k), exchange<8>(x, i, k);
            exchange<4>(x, i, k), exchange<2>(x, i, k), exchange<1>(x, i, k);
            s.order[i] = x;
        }
        __syncthreads();
    }
    const uint32_t i = 2 * tid;
    const u64 w0 = i < count ? w.weight_of(s.table, key_value(uint32_t(s.order[i] >> 32))) : 0;
    const u64 w1 = i + 1 < count ? w.weight_of(s.table, key_value(uint32_t(s.order[i + 1] >> 32))) : 0;
    Sum total;
    const Sum incl = block_scan({0, w0 + w1}, s.waves, total);
    if (i < size) {
        s.weight[i] = incl.mass - w1;
        s.weight[i + 1] = incl.mass;
    }
    __syncthreads();
}

// The border among the sorted list's tokens, `base` before them.
template <Border KIND>
__device__ void search_list(Shared& s, Sum base, u64 target) {
    const uint32_t count = s.listed;
    for (uint32_t i = threadIdx.x; i < count; i += THREADS) {
        const u64 before = i ? s.weight[i - 1] : 0;
        const Sum upto = {base.count + i + 1, base.mass + s.weight[i]};
        if (reached<KIND>(upto, target) && !reached<KIND>({base.count + i, base.mass + before}, target)) {
            s.found = upto;
            s.found_id = uint32_t(s.order[i]);
            s.found_weight = s.weight[i] - before;
        }
    }
    __syncthreads();
}

template <int TYPE>
struct Row {
    const void* base;
    int n;
    Weights w;
};

// The tokens with a value from `low` to `high` for which `inside` says so; sorted if the list holds them.
template <int TYPE, typename P>
__device__ void gather(Shared& s, const Row<TYPE>& row, float low, float high, P inside) {
    __syncthreads();
    if (threadIdx.x == 0) s.listed = 0;
    __syncthreads();
    for_row<TYPE, THREADS>(row.base, row.n, [&](int id, float v) {
        if (v < low || v > high || !inside(v)) return;
        const uint32_t at = atomicAdd(&s.listed, 1u);
        if (at < LIST) s.order[at] = u64(sort_key(v)) << 32 | uint32_t(id);
    });
    __syncthreads();
    if (s.listed <= LIST) sort_list(s, row.w);
}

// The tokens of bins first .. last.
template <int TYPE>
__device__ void gather_bins(Shared& s, const Row<TYPE>& row, int first, int last) {
    // values that may lie there, by a table step more at each end
    float low = NEG_INF, high = -NEG_INF;
    if (!row.w.infinite) {
        low = __double2float_rd(double(row.w.top) - double(((last + 1) << BIN_SHIFT) + 1) / row.w.rate);
        high = __double2float_ru(double(row.w.top) - double((first << BIN_SHIFT) - 1) / row.w.rate);
    }
    const Weights w = row.w;
    gather(s, row, low, high, [=](float v) {
        double x;
        if (!w.exponent(v, x)) return false;
        const int bin = Weights::steps(x) >> BIN_SHIFT;
        return bin >= first && bin <= last;
    });
}

// The token that is the `index`-th, by id, of those of one logit (`key`).
template <int TYPE>
__device__ void find_equal(Shared& s, const Row<TYPE>& row, uint32_t key, uint32_t index) {
    typedef typename Element<TYPE>::T T;
    const T* x = static_cast<const T*>(row.base);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int each = (row.n + WAVES * 64 - 1) / (WAVES * 64) * 64, begin = wave * each, end = min(row.n, begin + each);
    uint32_t own = 0;
    for (int i = begin; i < end; i += 64) {
        const bool same = i + lane < end && sort_key(plain(Element<TYPE>::value(x[i + lane]))) == key;
        own += uint32_t(__popcll(__ballot(same)));
    }
    __syncthreads();
    if (lane == 0) s.wave_id[wave] = own;
    __syncthreads();
    uint32_t before = 0;
    for (int w = 0; w < wave; ++w) before += s.wave_id[w];
    if (index >= before && index < before + own)
        for (int i = begin; i < end; i += 64) {
            const bool same = i + lane < end && sort_key(plain(Element<TYPE>::value(x[i + lane]))) == key;
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

// The border within a bin of more tokens than the list holds.
template <Border KIND, int TYPE>
__device__ void divide_bin(Shared& s, const Row<TYPE>& row, int bin, Sum base, u64 target) {
    const int tid = threadIdx.x;
    u64* mass = s.order;  // the list is not in use
    uint32_t* count = reinterpret_cast<uint32_t*>(s.weight);
    __syncthreads();
    if (tid == 0) {
        s.low = 0xffffffffu;
        s.high = 0;
    }
    __syncthreads();
    uint32_t low = 0xffffffffu, high = 0;
    for_row<TYPE, THREADS>(row.base, row.n, [&](int, float v) {
        double x;
        if (!row.w.exponent(v, x) || Weights::steps(x) >> BIN_SHIFT != bin) return;
        low = min(low, sort_key(v));
        high = max(high, sort_key(v));
    });
    atomicMin(&s.low, low);
    atomicMax(&s.high, high);
    __syncthreads();
    low = s.low;
    high = s.high;
    while (true) {
        if (low == high) {
            // one logit: every token has the same weight
            const u64 w = row.w.weight_of(s.table, key_value(low));
            u64 index;
            if (KIND == BORDER_COUNT) index = target - base.count - 1;
            else if (KIND == BORDER_MASS) index = (target - base.mass + w - 1) / w - 1;
            else index = (target - base.mass) / w;
            if (KIND == BORDER_DRAW) find_equal(s, row, low, uint32_t(index));
            __syncthreads();
            if (tid == 0) {
                s.found = {uint32_t(base.count + index + 1), base.mass + (index + 1) * w};
                s.found_weight = w;
            }
            __syncthreads();
            return;
        }
        int shift = 0;
        while ((high - low) >> shift >= SUB) ++shift;
        for (int i = tid; i < SUB; i += THREADS) {
            mass[i] = 0;
            count[i] = 0;
        }
        __syncthreads();
        for_row<TYPE, THREADS>(row.base, row.n, [&](int, float v) {
            const uint32_t key = sort_key(v);
            if (key < low || key > high) return;
            atomicAdd(&count[(key - low) >> shift], 1u);
            atomicAdd(&mass[(key - low) >> shift], row.w.weight_of(s.table, v));
        });
        __syncthreads();
        static_assert(SUB == THREADS, "one part for each thread");
        Sum total;
        const Sum own = {count[tid], mass[tid]}, incl = block_scan(own, s.waves, total);
        const Sum upto = {base.count + incl.count, base.mass + incl.mass};
        const Sum before = {upto.count - own.count, upto.mass - own.mass};
        if (reached<KIND>(upto, target) && !reached<KIND>(before, target)) {
            s.found_bin = tid;
            s.found = before;
            s.listed = own.count;
        }
        __syncthreads();
        const uint32_t part = uint32_t(s.found_bin);
        base = s.found;
        const uint32_t held = s.listed;
        high = min(high, low + (((part + 1) << shift) - 1));
        low += part << shift;
        __syncthreads();
        if (held <= LIST) {
            gather(s, row, key_value(high), key_value(low), [](float) { return true; });
            search_list<KIND>(s, base, target);
            return;
        }
        if (shift == 0) high = low;
    }
}

// The bins whose tokens are in the list; none: first > last.  `whole`: all tokens that may be kept are.
struct Listed {
    int first, last;
    bool whole;
};

// Finds a border by the bins' sums; the result is in s.found, s.found_id and s.found_weight.
template <Border KIND, int TYPE>
__device__ void find_border(Shared& s, const Row<TYPE>& row, Listed& list, u64 target) {
    __syncthreads();
    if (list.whole) {
        search_list<KIND>(s, {0, 0}, target);
        return;
    }
    for (int b = threadIdx.x; b < BINS; b += THREADS) {
        const Sum upto = {s.bin_count[b], s.bin_mass[b]};
        const Sum before = {b ? s.bin_count[b - 1] : 0, b ? s.bin_mass[b - 1] : 0};
        if (reached<KIND>(upto, target) && !reached<KIND>(before, target)) s.found_bin = b;
    }
    __syncthreads();
    const int bin = s.found_bin;
    __syncthreads();
    auto before = [&](int b) -> Sum { return {b ? s.bin_count[b - 1] : 0, b ? s.bin_mass[b - 1] : 0}; };
    if (bin < list.first || bin > list.last) {
        // all tokens up to the bin if they fit, so that further borders need no pass; else the bin's
        list = {s.bin_count[bin] <= uint32_t(LIST) ? 0 : bin, bin, false};
        gather_bins(s, row, list.first, bin);
        if (s.listed > uint32_t(LIST) && list.first < bin) {  // the numbers of tokens were estimates
            list.first = bin;
            gather_bins(s, row, bin, bin);
        }
        if (s.listed > uint32_t(LIST)) {
            divide_bin<KIND>(s, row, bin, before(bin), target);
            list = {1, 0, false};
            return;
        }
    }
    search_list<KIND>(s, before(list.first), target);
}

// Inclusive sums of the histograms -> all tokens' count and mass.  Where tokens were not counted, their
// number in a bin is estimated by the bin's smallest weight.
__device__ Sum sum_bins(Shared& s, const Weights& w, bool counts, bool masses) {
    __syncthreads();
    const int b = threadIdx.x;
    static_assert(BINS <= THREADS, "one bin for each thread");
    Sum own = {0, 0}, total;
    if (b < BINS) {
        own = {counts ? s.bin_count[b] : 0, masses ? s.bin_mass[b] : 0};
        if (!counts && own.mass) {
            const int step = ((b + 1) << BIN_SHIFT) - 1;
            const u64 least = w.weight(s.table, double(step), step);
            own.count = uint32_t(least ? min(own.mass / least + 1, u64(1) << 21) : u64(1) << 21);
        }
    }
    const Sum incl = block_scan(own, s.waves, total);
    if (b < BINS) {
        s.bin_count[b] = incl.count;
        s.bin_mass[b] = incl.mass;
    }
    __syncthreads();
    return total;
}

template <int TYPE>
__device__ __forceinline__ const void* row_base(const SampleParams& p, int r) {
    return static_cast<const typename Element<TYPE>::T*>(p.logits) + r * p.stride;
}

// The largest logit of a segment.
template <int TYPE>
__global__ __launch_bounds__(PART_THREADS) void sample_best_kernel(SampleParams p, int each) {
    __shared__ float s_values[PART_THREADS / 64];
    __shared__ uint32_t s_ids[PART_THREADS / 64];
    const int begin = blockIdx.x * each, n = min(each, p.n - begin);
    float best;
    uint32_t id;
    find_best<TYPE, PART_THREADS>(static_cast<const typename Element<TYPE>::T*>(row_base<TYPE>(p, blockIdx.y)) + begin, n,
                                  best, id);
    block_best<PART_THREADS>(best, id, s_values, s_ids);
    if (threadIdx.x == 0) {
        Segment& out = static_cast<Segment*>(p.workspace)[int64_t(blockIdx.y) * gridDim.x + blockIdx.x];
        out.best = best;
        out.id = id == 0xffffffffu ? id : id + uint32_t(begin);
    }
}

// The row's largest logit from its segments', in every thread (a wave's lanes take a segment each).
__device__ __forceinline__ void segments_best(const Segment* segments, int count, float& best, uint32_t& id) {
    best = NEG_INF;
    id = 0xffffffffu;
    for (int i = threadIdx.x & 63; i < count; i += 64) {
        if (segments[i].best > best) {
            best = segments[i].best;
            id = segments[i].id;
        }
    }
    for (int o = 32; o > 0; o >>= 1) {
        const float v = __shfl_xor(best, o, 64);
        const uint32_t i = __shfl_xor(id, o, 64);
        if (v > best || (v == best && i < id)) {
            best = v;
            id = i;
        }
    }
}

// A segment's histograms.
template <int TYPE>
__global__ __launch_bounds__(PART_THREADS) void sample_bins_kernel(SampleParams p, int each) {
    __shared__ double s_table[STEPS];
    __shared__ u64 s_mass[BINS];
    __shared__ uint32_t s_count[BINS];
    __shared__ u64 s_kept;
    const int r = blockIdx.y, tid = threadIdx.x;
    Segment* segments = static_cast<Segment*>(p.workspace) + int64_t(r) * gridDim.x;
    const Controls c(p, r);
    if (c.greedy()) return;
    for (int i = tid; i < STEPS; i += PART_THREADS) s_table[i] = table_entry(i);
    for (int i = tid; i < BINS; i += PART_THREADS) {
        s_mass[i] = 0;
        s_count[i] = 0;
    }
    if (tid == 0) s_kept = 0;
    float best;
    uint32_t id;
    segments_best(segments, gridDim.x, best, id);
    if (id == 0xffffffffu) return;
    Weights w;
    w.set(best, c.temperature, p.n);
    __syncthreads();
    const int begin = blockIdx.x * each, n = min(each, p.n - begin);
    const u64 kept = fill_bins<TYPE, PART_THREADS>(
        static_cast<const typename Element<TYPE>::T*>(row_base<TYPE>(p, r)) + begin, n, w, s_table, c.counts, c.masses,
        c.least, s_mass, s_count);
    if (c.least && kept) atomicAdd(&s_kept, kept);
    __syncthreads();
    Segment& out = segments[blockIdx.x];
    for (int i = tid; i < BINS; i += PART_THREADS) {
        if (c.masses) out.bin_mass[i] = s_mass[i];
        if (c.counts) out.bin_count[i] = s_count[i];
    }
    if (tid == 0) out.min_mass = s_kept;
}

// SEGMENTS: the first two steps are done, in `segments` parts; else they are this workgroup's too.
template <int TYPE, bool SEGMENTS>
__global__ __launch_bounds__(THREADS) void sample_pick_kernel(SampleParams p, int segments) {
    __shared__ Shared s;
    const int r = blockIdx.x, tid = threadIdx.x;
    Row<TYPE> row;
    row.base = row_base<TYPE>(p, r);
    row.n = p.n;
    const Controls c(p, r);
    const Segment* parts = static_cast<const Segment*>(p.workspace) + int64_t(r) * segments;
    float best;
    uint32_t id;
    if constexpr (SEGMENTS) {
        segments_best(parts, segments, best, id);
    } else {
        find_best<TYPE, THREADS>(row.base, p.n, best, id);
        block_best<THREADS>(best, id, s.wave_value, s.wave_id);
    }
    if (id == 0xffffffffu || c.greedy()) {
        if (tid == 0) {
            p.token[r] = int32_t(id);  // -1 where nothing can be drawn
            if (p.prob) p.prob[r] = id == 0xffffffffu ? 0.0f : 1.0f;
        }
        return;
    }
    row.w.set(best, c.temperature, p.n);
    static_assert(STEPS == THREADS, "one entry for each thread");
    s.table[tid] = table_entry(tid);
    if (tid == 0) s.min_mass = 0;
    auto fill = [&](bool counts, bool masses) {
        for (int b = tid; b < BINS; b += THREADS) {
            s.bin_mass[b] = 0;
            s.bin_count[b] = 0;
        }
        __syncthreads();
        const u64 kept = fill_bins<TYPE, THREADS>(row.base, p.n, row.w, s.table, counts, masses, c.least, s.bin_mass, s.bin_count);
        if (c.least && kept) atomicAdd(&s.min_mass, kept);
    };
    if constexpr (SEGMENTS) {
        if (tid < BINS) {
            u64 mass = 0;
            uint32_t count = 0;
            if (c.masses) {
#pragma unroll 4
                for (int i = 0; i < segments; ++i) mass += parts[i].bin_mass[tid];
            }
            if (c.counts) {
#pragma unroll 4
                for (int i = 0; i < segments; ++i) count += parts[i].bin_count[tid];
            }
            s.bin_mass[tid] = mass;
            s.bin_count[tid] = count;
        }
        __syncthreads();
        if (c.masses && c.least && tid < segments) atomicAdd(&s.min_mass, parts[tid].min_mass);
    } else {
        fill(c.counts, c.masses);
    }
    Sum kept = sum_bins(s, row.w, c.counts, c.masses);
    Listed list = {1, 0, false};
    if (!c.masses) {
        // the top-k's tokens, and what shares the last one's bin
        int last = BINS - 1;
        if (uint32_t(c.top_k) < kept.count) {
            if (tid < BINS && s.bin_count[tid] >= uint32_t(c.top_k) && (tid == 0 || s.bin_count[tid - 1] < uint32_t(c.top_k)))
                s.found_bin = tid;
            __syncthreads();
            last = s.found_bin;
        }
        gather_bins(s, row, 0, last);
        if (s.listed <= uint32_t(LIST)) {
            list.whole = true;
            kept = {s.listed, s.weight[s.listed - 1]};
        } else {
            // too many share it: weights of all tokens after all
            fill(true, true);
            kept = sum_bins(s, row.w, true, true);
        }
    }
    if (c.top_k > 0 && uint32_t(c.top_k) < kept.count) {
        find_border<BORDER_COUNT>(s, row, list, u64(c.top_k));
        kept = s.found;
    }
    if (c.top_p < 1.0f) {
        const double target = ceil(double(c.top_p) * double(kept.mass));
        find_border<BORDER_MASS>(s, row, list, target > 1.0 ? u64(target) : u64(1));
        kept = s.found;
    }
    if (c.least) {
        if (list.whole) {
            __syncthreads();
            for (uint32_t i = tid; i < s.listed; i += THREADS) {
                const u64 own = s.weight[i] - (i ? s.weight[i - 1] : 0);
                if (own >= c.least && (i + 1 == s.listed || s.weight[i + 1] - s.weight[i] < c.least)) s.min_mass = s.weight[i];
            }
            __syncthreads();
        }
        kept.mass = min(kept.mass, s.min_mass);  // both are beginnings of one order
    }
    const float u = p.uniform[r];
    const u64 at = u > 0.0f ? u64(double(fminf(u, 1.0f)) * double(kept.mass)) : 0;
    find_border<BORDER_DRAW>(s, row, list, at < kept.mass ? at : kept.mass - 1);
    if (tid == 0) {
        p.token[r] = int32_t(s.found_id);
        if (p.prob) p.prob[r] = float(double(s.found_weight) / double(kept.mass));
    }
}

// Segments of a row: of 4,096 logits at least, and some 2,048 in all, which fill the CUs several times;
// 1: a workgroup does the whole row.
int row_segments(int rows, int n) { return std::max(1, std::min((n + 4095) / 4096, 2048 / rows)); }
constexpr int FEWEST_SEGMENTS = 3;

template <int TYPE>
void run_sample(const SampleParams& p, hipStream_t s) {
    int segments = row_segments(p.rows, p.n);
    if (segments < FEWEST_SEGMENTS) {
        hipLaunchKernelGGL((sample_pick_kernel<TYPE, false>), dim3(unsigned(p.rows)), dim3(THREADS), 0, s, p, 0);
        return;
    }
    const int each = (p.n + segments * 64 - 1) / (segments * 64) * 64;
    segments = (p.n + each - 1) / each;
    const dim3 grid(unsigned(segments), unsigned(p.rows));
    hipLaunchKernelGGL((sample_best_kernel<TYPE>), grid, dim3(PART_THREADS), 0, s, p, each);
    hipLaunchKernelGGL((sample_bins_kernel<TYPE>), grid, dim3(PART_THREADS), 0, s, p, each);
    hipLaunchKernelGGL((sample_pick_kernel<TYPE, true>), dim3(unsigned(p.rows)), dim3(THREADS), 0, s, p, segments);
}

}  // namespace

size_t sample_workspace(int rows, int n) {
    const int segments = row_segments(rows, n);
    return segments < FEWEST_SEGMENTS ? 0 : size_t(rows) * size_t(segments) * sizeof(Segment);
}

void launch_sample(const SampleParams& p, int type, hipStream_t s) {
    if (type == TYPE_BF16) run_sample<TYPE_BF16>(p, s);
    else if (type == TYPE_F16) run_sample<TYPE_F16>(p, s);
    else run_sample<TYPE_F32>(p, s);
}

}  // namespace plamo
