// Tokens drawn from logits on gfx950: temperature, top-k, top-p and min-p, by given uniform numbers.
//
// A row's tokens are ordered by descending logit, equal ones by ascending id.  With weights
// e_i = exp((x_i - max x) / T): top-k keeps the first k; top-p of those the ones before which less than
// p of the kept weight lies; min-p of those the ones of at least min_p of the largest weight.  All three
// keep a beginning of the order.  The token is the first one up to which more than u of the kept weight
// lies.  Nothing is sorted but the few tokens around a border:
//   1. the largest logit;
//   2. a histogram of the weights over bins of the exponent (32 bins for a factor of two), counts and
//      sums, from one pass over the row;
//   3. prefix sums over the bins give the bin of each border; the tokens of that bin (or of all bins
//      up to it) are gathered, sorted in LDS and searched.  A bin of more tokens than the list holds
//      is divided again by the bits of the logits until it is small enough or one value.
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

constexpr int THREADS = 1024, WAVES = THREADS / 64;
constexpr int STEPS = 1024;          // table entries for a factor of two
constexpr int BIN_SHIFT = 5;         // table steps of a bin
constexpr int BINS = 1536;           // 32 (S + 1) <= 1504 are used
constexpr int LIST = 2048;           // tokens that are sorted at once
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

// f(id, value) for a row's elements, a thread's in ascending order; 16 bytes a load behind the
// first aligned element.
template <int TYPE, typename F>
__device__ __forceinline__ void for_row(const void* base, int n, F f) {
    typedef typename Element<TYPE>::T T;
    constexpr int PER = 16 / sizeof(T), AHEAD = 4;
    const T* row = static_cast<const T*>(base);
    const int tid = threadIdx.x;
    const int head = min(n, int(((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / sizeof(T)));
    if (tid < head) f(tid, plain(Element<TYPE>::value(row[tid])));
    const int vectors = (n - head) / PER;
    const uint4* body = reinterpret_cast<const uint4*>(row + head);
    for (int i = tid; i < vectors; i += THREADS * AHEAD) {
        uint4 w[AHEAD];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a)
            if (i + a * THREADS < vectors) w[a] = body[i + a * THREADS];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            if (i + a * THREADS >= vectors) break;
            const int id = head + (i + a * THREADS) * PER;
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

struct Sum {
    uint32_t count;
    u64 mass;
};

struct Shared {
    double table[STEPS];   // 2^(-j / STEPS)
    u64 bin_mass[BINS];    // then inclusive sums
    uint32_t bin_count[BINS];
    u64 order[LIST];       // descending logit, ascending id
    u64 weight[LIST];      // then inclusive sums
    Sum waves[WAVES];
    float wave_value[WAVES];
    uint32_t wave_id[WAVES];
    uint32_t low, high, listed;
    Sum found;             // a border's count and mass up to and with its token
    uint32_t found_id;
    u64 found_weight;
    int found_bin;
    uint32_t min_count;    // tokens of at least min_p
    u64 min_mass;
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

// A row's weights.
struct Weights {
    float top;        // largest logit
    bool infinite;    // it is plus infinity: only such tokens have a weight
    double rate;      // STEPS log2(e) / T
    double limit;     // exponents from here on weigh nothing
    int scale;        // S
    const double* table;

    __device__ __forceinline__ bool exponent(float v, double& x) const {
        if (infinite) v = v == top ? 0.0f : NEG_INF;
        x = (double(infinite ? 0.0f : top) - double(v)) * rate;
        return x < limit;  // false for minus infinity
    }
    static __device__ __forceinline__ int steps(double x) { return int(__builtin_rint(x)); }
    __device__ __forceinline__ u64 weight(double x, int n) const {
        // 2^(-x / STEPS) = table[n % STEPS] 2^-(n / STEPS) exp(-f), |f| <= log(2) / (2 STEPS): the cubic
        // is off by f^4 / 24 < 2^-50
        const double f = (x - double(n)) * (0.69314718055994530942 / STEPS);
        const double e = 1.0 - f * (1.0 - f * (0.5 - f * (1.0 / 6.0)));
        return u64(__builtin_rint(ldexp(table[n & (STEPS - 1)] * e, scale - n / STEPS)));
    }
};

enum Border { BORDER_COUNT, BORDER_MASS, BORDER_DRAW };

// Whether a token with these sums before it is the border, or lies behind it.
template <Border KIND>
__device__ __forceinline__ bool reached(Sum upto, u64 target) {
    return KIND == BORDER_COUNT ? upto.count >= target : KIND == BORDER_MASS ? upto.mass >= target : upto.mass > target;
}

// The tokens of the list (s.listed of them, padded to LIST) in order, with inclusive sums of weights.
__device__ void sort_list(Shared& s) {
    const int tid = threadIdx.x;
    const uint32_t count = s.listed;
    uint32_t size = 2;
    while (size < count) size <<= 1;
    for (uint32_t i = count + tid; i < size; i += THREADS) {
        s.order[i] = ~u64(0);
        s.weight[i] = 0;
    }
    __syncthreads();
    for (uint32_t k = 2; k <= size; k <<= 1)
        for (uint32_t j = k >> 1; j > 0; j >>= 1) {
            for (uint32_t t = tid; t < size / 2; t += THREADS) {
                const uint32_t a = (t / j) * 2 * j + t % j, b = a + j;
                const u64 x = s.order[a], y = s.order[b];
                if ((x > y) == ((a & k) == 0)) {
                    s.order[a] = y;
                    s.order[b] = x;
                    const u64 w = s.weight[a];
                    s.weight[a] = s.weight[b];
                    s.weight[b] = w;
                }
            }
            __syncthreads();
        }
    const uint32_t i = 2 * tid;
    const u64 w0 = i < size ? s.weight[i] : 0, w1 = i < size ? s.weight[i + 1] : 0;
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

template <int TYPE, typename P>
__device__ void gather(Shared& s, const Row<TYPE>& row, P inside) {
    __syncthreads();
    if (threadIdx.x == 0) s.listed = 0;
    __syncthreads();
    for_row<TYPE>(row.base, row.n, [&](int id, float v) {
        double x;
        if (!row.w.exponent(v, x)) return;
        const int n = Weights::steps(x);
        if (!inside(n, v)) return;
        const uint32_t at = atomicAdd(&s.listed, 1u);
        if (at < LIST) {
            s.order[at] = u64(sort_key(v)) << 32 | uint32_t(id);
            s.weight[at] = row.w.weight(x, n);
        }
    });
    __syncthreads();
    sort_list(s);
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
    for_row<TYPE>(row.base, row.n, [&](int, float v) {
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
            double x;
            const uint32_t bits = low & 0x80000000u ? low : ~low & 0x7fffffffu;
            row.w.exponent(__uint_as_float(bits), x);
            const u64 w = row.w.weight(x, Weights::steps(x));
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
        for_row<TYPE>(row.base, row.n, [&](int, float v) {
            const uint32_t key = sort_key(v);
            if (key < low || key > high) return;
            double x;
            if (!row.w.exponent(v, x)) return;
            atomicAdd(&count[(key - low) >> shift], 1u);
            atomicAdd(&mass[(key - low) >> shift], row.w.weight(x, Weights::steps(x)));
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
            const uint32_t from = low, to = high;
            gather(s, row, [=](int, float v) { return sort_key(v) >= from && sort_key(v) <= to; });
            search_list<KIND>(s, base, target);
            return;
        }
        if (shift == 0) high = low;
    }
}

// The bins whose tokens are in the list; none: first > last.
struct Listed {
    int first, last;
};

// Finds a border by the bins' sums; the result is in s.found, s.found_id and s.found_weight.
template <Border KIND, int TYPE>
__device__ void find_border(Shared& s, const Row<TYPE>& row, Listed& list, u64 target) {
    __syncthreads();
    for (int b = threadIdx.x; b < BINS; b += THREADS) {
        const Sum upto = {s.bin_count[b], s.bin_mass[b]};
        const Sum before = {b ? s.bin_count[b - 1] : 0, b ? s.bin_mass[b - 1] : 0};
        if (reached<KIND>(upto, target) && !reached<KIND>(before, target)) s.found_bin = b;
    }
    __syncthreads();
    const int bin = s.found_bin;
    __syncthreads();
    if (bin < list.first || bin > list.last) {
        // all tokens up to the bin if they fit, so that further borders need no pass; else the bin's
        const int first = s.bin_count[bin] <= uint32_t(LIST) ? 0 : bin;
        const Sum base = {first ? s.bin_count[first - 1] : 0, first ? s.bin_mass[first - 1] : 0};
        if (s.bin_count[bin] - base.count > uint32_t(LIST)) {
            divide_bin<KIND>(s, row, bin, base, target);
            list = {1, 0};
            return;
        }
        gather(s, row, [=](int n, float) { return n >> BIN_SHIFT >= first && n >> BIN_SHIFT <= bin; });
        list = {first, bin};
    }
    const Sum base = {list.first ? s.bin_count[list.first - 1] : 0, list.first ? s.bin_mass[list.first - 1] : 0};
    search_list<KIND>(s, base, target);
}

template <int TYPE>
__global__ __launch_bounds__(THREADS) void sample_kernel(SampleParams p) {
    __shared__ Shared s;
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    Row<TYPE> row;
    row.base = static_cast<const typename Element<TYPE>::T*>(p.logits) + r * p.stride;
    row.n = p.n;
    // the largest logit and its first token
    float best = NEG_INF;
    uint32_t id = 0xffffffffu;
    for_row<TYPE>(row.base, p.n, [&](int i, float v) {
        if (v > best) {
            best = v;
            id = uint32_t(i);
        }
    });
    for (int o = 32; o > 0; o >>= 1) {
        const float v = __shfl_xor(best, o, 64);
        const uint32_t i = __shfl_xor(id, o, 64);
        if (v > best || (v == best && i < id)) {
            best = v;
            id = i;
        }
    }
    if (lane == 0) {
        s.wave_value[wave] = best;
        s.wave_id[wave] = id;
    }
    for (int b = tid; b < BINS; b += THREADS) {
        s.bin_mass[b] = 0;
        s.bin_count[b] = 0;
    }
    if (tid == 0) {
        s.min_count = 0;
        s.min_mass = 0;
    }
    static_assert(STEPS == THREADS, "one entry for each thread");
    s.table[tid] = exp2(-double(tid) / STEPS);
    __syncthreads();
    for (int w = 0; w < WAVES; ++w)
        if (s.wave_value[w] > best || (s.wave_value[w] == best && s.wave_id[w] < id)) {
            best = s.wave_value[w];
            id = s.wave_id[w];
        }
    const float temperature = p.temperature ? p.temperature[r] : 1.0f;
    if (id == 0xffffffffu || !(temperature > 0.0f)) {
        if (tid == 0) {
            p.token[r] = int32_t(id);  // -1 where nothing can be drawn
            if (p.prob) p.prob[r] = id == 0xffffffffu ? 0.0f : 1.0f;
        }
        return;
    }
    const int scale = min(46, 31 + __clz(p.n));  // sums of n weights stay below 2^63
    row.w.top = best;
    row.w.infinite = best == -NEG_INF;
    row.w.rate = STEPS * 1.44269504088896340736 / double(temperature);
    row.w.limit = double((scale + 1) * STEPS) - 0.5;
    row.w.scale = scale;
    row.w.table = s.table;

    const float min_p = p.min_p ? p.min_p[r] : 0.0f, top_p = p.top_p ? p.top_p[r] : 1.0f;
    const int top_k = p.top_k ? p.top_k[r] : 0;
    const u64 least = min_p > 0.0f ? u64(ceil(ldexp(double(fminf(min_p, 1.0f)), scale))) : 0;
    uint32_t min_count = 0;
    u64 min_mass = 0;
    for_row<TYPE>(row.base, p.n, [&](int, float v) {
        double x;
        if (!row.w.exponent(v, x)) return;
        const int n = Weights::steps(x);
        const u64 w = row.w.weight(x, n);
        atomicAdd(&s.bin_mass[n >> BIN_SHIFT], w);
        atomicAdd(&s.bin_count[n >> BIN_SHIFT], 1u);
        if (w >= least) {
            ++min_count;
            min_mass += w;
        }
    });
    if (least) {
        atomicAdd(&s.min_count, min_count);
        atomicAdd(&s.min_mass, min_mass);
    }
    __syncthreads();
    Sum kept;
    {
        const int b = 2 * tid;
        const bool own = b < BINS;
        const Sum first = {own ? s.bin_count[b] : 0, own ? s.bin_mass[b] : 0};
        const Sum second = {own ? s.bin_count[b + 1] : 0, own ? s.bin_mass[b + 1] : 0};
        const Sum incl = block_scan({first.count + second.count, first.mass + second.mass}, s.waves, kept);
        if (own) {
            s.bin_count[b] = incl.count - second.count;
            s.bin_mass[b] = incl.mass - second.mass;
            s.bin_count[b + 1] = incl.count;
            s.bin_mass[b + 1] = incl.mass;
        }
    }
    Listed list = {1, 0};
    if (top_k > 0 && uint32_t(top_k) < kept.count) {
        find_border<BORDER_COUNT>(s, row, list, u64(top_k));
        kept = s.found;
    }
    if (top_p < 1.0f) {
        const double target = ceil(double(top_p) * double(kept.mass));
        find_border<BORDER_MASS>(s, row, list, target > 1.0 ? u64(target) : u64(1));
        kept = s.found;
    }
    if (least && s.min_count < kept.count) kept = {s.min_count, s.min_mass};
    const float u = p.uniform[r];
    const u64 at = u > 0.0f ? u64(double(fminf(u, 1.0f)) * double(kept.mass)) : 0;
    find_border<BORDER_DRAW>(s, row, list, at < kept.mass ? at : kept.mass - 1);
    if (tid == 0) {
        p.token[r] = int32_t(s.found_id);
        if (p.prob) p.prob[r] = float(double(s.found_weight) / double(kept.mass));
    }
}

}  // namespace

size_t sample_workspace(int, int) { return 0; }

void launch_sample(const SampleParams& p, int type, hipStream_t s) {
    const dim3 grid{unsigned(p.rows)};
    if (type == TYPE_BF16) hipLaunchKernelGGL((sample_kernel<TYPE_BF16>), grid, dim3(THREADS), 0, s, p);
    else if (type == TYPE_F16) hipLaunchKernelGGL((sample_kernel<TYPE_F16>), grid, dim3(THREADS), 0, s, p);
    else hipLaunchKernelGGL((sample_kernel<TYPE_F32>), grid, dim3(THREADS), 0, s, p);
}

}  // namespace plamo
