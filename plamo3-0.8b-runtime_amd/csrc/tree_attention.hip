// Attention of several new tokens a request over its pages on gfx950: drafted trees and chunks of prompts.
//
//   tree_division_kernel   how the keys of very many requests are divided
//   tree_attention_kernel  tiles of the new tokens' query heads over parts of their request's keys
//   tree_join_kernel       parts of a tile joined
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "common.h"
#include "paged_device.h"
#include "speculate.h"

namespace plamo {
using namespace dev;

namespace {

typedef float floatx16 __attribute__((ext_vector_type(16)));

// o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m) over the keys that a token sees, one pass with the running maximum
// and sum.  The rows of a KV head are all new tokens of a request times the query heads that read it, side by side: a
// tile is 32 rows for each of SHARE waves, which share the keys' tiles in LDS; GROUPS such sets of waves take
// every GROUPS-th tile of keys.  A wave's products are
//   S^T = K Q^T     v_mfma_f32_32x32x16 with the keys as rows: lane l has row l % 32 of the queries, so that a row's
//                   softmax is within two lanes and its weights are already the operand of the next product;
//   O^T += V^T P^T  V read from LDS by transposing reads.
// Pages go straight into LDS, each lane from its own address: any page size and any strides.  Where a lane's keys
// of a load are known to lie in one page (EVEN) it looks that page up once.
// What bounds it, with what it took: arithmetic for chunks of prompts (of 999 and 333 tokens, 16 heads of 128, behind 28,000 and
// 30,720 keys: 317 GFLOP in 494 us, 640 TFLOP/s, and half as many again for the weights' second halves; softmax and products of a
// wave take turns, two workgroups a CU fill in);
// memory for a few nodes with a window (48 requests of up to 13 nodes, 32 heads of 64 on 8, 2,048 keys: 171 MB in 54 us); one
// request's 343 keys the latency of its loads (9.5 us, then 3 to join); and many trees each a part (64 of up to 24 nodes behind 33
// to 8,192 keys, 16 heads of 128 on one: 42.5 us for 53 MB) all of these: some 6 to find a part and load its first tile, five
// more tiles of some 4.5, and the parts' results, written and read once more, with a launch of 8.  (With weights rounded once, one
// workgroup of eight waves a CU, of two sets, halved those results and took 46 for 42, and the chunks 537 for 371.)
constexpr int CUS = 256;

template <int D, int SHARE>
struct Shape {
    static constexpr int KEYS = SHARE == 4 ? 64 : 32;  // of a tile
    static constexpr int GROUPS = SHARE == 4 ? 1 : SHARE == 2 || D == 256 ? 2 : 4;
    static constexpr int WAVES = SHARE * GROUPS, THREADS = 64 * WAVES;
    static constexpr int HELD = D == 256 || (D == 128 && SHARE == 1) ? 1 : D == 64 && SHARE == 2 ? 3 : 2;  // workgroups of a CU
    static constexpr int OF_SIMD = HELD * WAVES <= 4 ? 1 : HELD * WAVES > 8 ? HELD * WAVES / 4 : 2;  // waves whose registers fit
    static constexpr int ROW = 2 * D;                 // bytes of a key
    static constexpr int TILE = KEYS * ROW;           // of a tile's keys, or of its values
    static constexpr int LDS = GROUPS * 2 * 2 * TILE; // two stages
    static constexpr int PIECE_KEYS = 512 / D;        // keys of a load: 16 bytes a lane
    static constexpr int PIECES = 16 / PIECE_KEYS;    // loads of 16 keys
    static constexpr int OWN = KEYS / SHARE / 16;     // sixteens that a wave loads
    static constexpr int BLOCKS = KEYS / 32;          // of a product
    static constexpr int STEPS = D / 16, DIMS = D / 32;
    static constexpr int SPLIT = D / 8;               // four dims each of the 64 lanes' rows
};
static_assert(Shape<128, 4>::LDS == 65536 && Shape<128, 2>::LDS == 65536 && Shape<128, 1>::LDS == 131072 && Shape<256, 1>::LDS == 131072 &&
              Shape<256, 2>::LDS == 131072 && Shape<256, 4>::LDS == 131072 && Shape<64, 1>::LDS == 65536 && Shape<64, 2>::LDS == 32768, "of 160 KB");

// Key of row R of sixteen in LDS: a lane's loads are of neighbouring keys.
template <int D>
constexpr int key_of_row(int row) { return 16 / (512 / D) * (row % (512 / D)) + row / (512 / D); }
// The same for the rows of a lane's scores, 8 (i / 4) + 4 (lane / 32) + i % 4: a constant, and what the lane's half adds.
template <int D>
constexpr int score_key(int i) { return 16 * (i / 8) + key_of_row<D>(8 * (i / 4 % 2) + i % 4); }
template <int D>
constexpr int HALF_KEY = key_of_row<D>(4);

// Where 16-byte chunk c of row R lies in its row of keys, 64-byte chunk d in its row of values: operand reads
// then touch all banks.
template <int D>
__device__ __forceinline__ constexpr int key_swizzle(int row) { return D == 64 ? row >> 1 & 7 : row & 15; }
template <int D>
__device__ __forceinline__ constexpr int value_swizzle(int row) { return D == 64 ? row >> 1 & 1 : row & 3; }

// FP16 weights are held times 2^12: their smallest normal value is then 2^-26 of the largest weight's.
template <int TYPE>
constexpr float weight_shift() { return TYPE == TYPE_F16 ? 12.0f : 0.0f; }

template <int TYPE>
__device__ __forceinline__ floatx16 mfma32(uint4 a, uint4 b, floatx16 c) {
    if constexpr (TYPE == TYPE_BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// ------------------------------------------------------------------------------------ division of the work
struct Request {
    int first, count;  // new tokens
    int start, end;    // keys before them, keys in all
    int tiles;
    int low, span;     // the first key that one of them sees, rounded down to 16, and the keys from it on
};
template <int ROWS>  // of a tile
__device__ __forceinline__ Request request(const TreeAttnParams& p, int r) {
    Request q;
    q.first = p.offsets[r];
    const int past = p.offsets[r + 1], length = p.lengths[r];
    const bool fine = q.first >= 0 && past >= q.first && past <= p.tokens;
    q.count = fine ? past - q.first : 0;
    q.first = fine ? q.first : 0;
    const bool held = length >= q.count;  // (the difference of others may wrap)
    q.start = held ? length - q.count : 0;
    q.end = held ? min(length, p.most) : 0;
    q.tiles = (q.count * p.group + ROWS - 1) / ROWS;
    q.low = p.window > 0 ? min(max(q.start - p.window + 1, 0), q.end) & ~15 : 0;
    q.span = q.count > 0 ? q.end - q.low : 0;
    return q;
}
__device__ __forceinline__ int parts_of(int span, int chunk) { return span > 0 ? (span - 1) / chunk + 1 : 1; }

// Keys of a part: all tiles' keys, next to which FP32 is, divided by the parts aimed at, `times` eighths of that.  (A
// little more: tiles of several parts have less than twice as many parts then as are aimed at.)
__device__ __forceinline__ int part_keys(const TreeAttnParams& p, float work, int tiles, int times) {
    const int parts = max(p.target - tiles / 2, (p.target + 1) / 2);  // a tile's last part is half empty
    const float share = work * 1.0001220703125f / float(parts) * (0.125f * float(times));
    if (share <= float(p.least)) return p.least;
    const int each = share < float(p.most) ? int(share) + 1 : p.most;
    return (each + p.least - 1) / p.least * p.least;
}

struct Sums {
    int items, slots, joined;
};
__device__ __forceinline__ Sums row_sums(const Request& q, int chunk) {
    const int parts = parts_of(q.span, chunk);
    return {q.tiles * parts, parts > 1 ? q.tiles * parts : 0, parts > 1 ? q.tiles : 0};
}
__device__ __forceinline__ Sums scan(Sums v) { return {wave_scan(v.items), wave_scan(v.slots), wave_scan(v.joined)}; }
__device__ __forceinline__ Sums at_lane(Sums v, int l) {
    return {__builtin_amdgcn_readlane(v.items, l), __builtin_amdgcn_readlane(v.slots, l), __builtin_amdgcn_readlane(v.joined, l)};
}
// Requests overlap where offsets descend in between, and their tiles, up to 2^23 each, may then be any number of times as many as a
// launch takes: sums of items end at MOST_ITEMS, past all that run, so that none wraps (64 requests' are less than 2^30, as are 64
// sums that end there) and they ascend.  Slots and joined tiles come from the keys' division and stay within its bounds.
constexpr int MOST_ITEMS = 1 << 24;
__device__ __forceinline__ Sums operator+(Sums a, Sums b) { return {min(a.items + b.items, MOST_ITEMS), a.slots + b.slots, a.joined + b.joined}; }
__device__ __forceinline__ Sums operator-(Sums a, Sums b) { return {a.items - b.items, a.slots - b.slots, a.joined - b.joined}; }

// Of an item: its request, the sums of those before, and how many parts its tiles have.
struct Work {
    int row;
    Sums before;
    int parts;
};
struct WorkShared {
    float work[16];
    int number[16];
    Sums waves[16];
    Work found;
};

// Sums over the workgroup's waves, in every wave and in one order.
template <int WAVES>
__device__ __forceinline__ void total(WorkShared& s, float& work, int& number) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    work = wave_sum(work);
    number = __builtin_amdgcn_readlane(wave_scan(number), 63);
    if (WAVES == 1) return;
    __syncthreads();  // the sums before these have been read
    if (lane == 0) {
        s.work[wave] = work;
        s.number[wave] = number;
    }
    __syncthreads();
    work = 0.f;
    number = 0;
    for (int w = 0; w < WAVES; ++w) {
        work += s.work[w];
        number += s.number[w];
    }
}

// A part's keys, from the requests that a thread takes: from row `first` on, every `step`-th.  More of them where
// all parts at once would be a few too many for the CUs, and a second round had to be waited for (64 requests of 33 to 8,192 keys,
// trees of 8 to 24 nodes 47 -> 42.5 us); as many as at first where that does not help.
template <int ROWS, int WAVES>
__device__ __forceinline__ int choose_part(const TreeAttnParams& p, WorkShared& s, int first, int step) {
    constexpr int ENOUGH = 1 << 20;  // more than any target; sums of 1,024 threads' do not wrap
    float work = 0.f, none = 0.f;
    int tiles = 0;
    for (int r = first; r < p.rows; r += step) {
        const Request q = request<ROWS>(p, r);
        work += float(q.tiles) * float(q.span);
        tiles = min(tiles + q.tiles, ENOUGH);
    }
    total<WAVES>(s, work, tiles);
    const int least = __builtin_amdgcn_readfirstlane(part_keys(p, work, tiles, 8));
    if (least == p.least) return least;
    for (int times = 8; times <= 16; ++times) {
        const int chunk = __builtin_amdgcn_readfirstlane(part_keys(p, work, tiles, times));
        int items = 0;
        for (int r = first; r < p.rows; r += step) {
            const Request q = request<ROWS>(p, r);
            items = min(items + q.tiles * parts_of(q.span, chunk), ENOUGH);
        }
        total<WAVES>(s, none, items);
        if (items <= p.target) return chunk;
    }
    return least;
}

// The request of an item, from all requests' lengths and offsets: the same division in all workgroups.  Up to 64
// requests every wave does for itself.  False past the last item; `joined`, for the first: tiles of several parts, none where
// some items are not run.
template <int ROWS, int WAVES>
__device__ __forceinline__ bool find_work(const TreeAttnParams& p, WorkShared& s, int item, Work& work, int& joined) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool few = p.rows <= 64;
    const int step = few ? 64 : 64 * WAVES, own_row = few ? lane : int(threadIdx.x);
    const int chunk = few ? choose_part<ROWS, 1>(p, s, own_row, step) : choose_part<ROWS, WAVES>(p, s, own_row, step);
    Sums run = {0, 0, 0};
    bool found = false;
    for (int base = 0; base < p.rows; base += step) {
        const int r = base + own_row;
        Sums own = {0, 0, 0};
        int parts = 1;
        if (r < p.rows) {
            const Request q = request<ROWS>(p, r);
            own = row_sums(q, chunk);
            parts = parts_of(q.span, chunk);
        }
        const Sums incl = scan(own), all = at_lane(incl, 63);
        Sums before = run;
        if (!few) {
            __syncthreads();  // what the sums of the requests before said has been read
            if (lane == 0) s.waves[wave] = all;
            __syncthreads();
            for (int w = 0; w < WAVES; ++w) {
                if (w < wave) before = before + s.waves[w];
                run = run + s.waves[w];
            }
        } else {
            run = run + all;
        }
        const unsigned long long past = __ballot(before.items + incl.items > item && before.items + incl.items - own.items <= item);
        if (past) {
            const int l = __ffsll(past) - 1;
            work.row = __builtin_amdgcn_readlane(r, l);
            work.parts = __builtin_amdgcn_readlane(parts, l);
            work.before = before + at_lane(incl - own, l);
            if (!few && lane == 0) s.found = work;
        }
        if (!found && item < run.items) {
            found = true;
            if (!few) {
                __syncthreads();
                work = s.found;
            }
            if (item > 0) break;  // the first item's workgroup goes on to say how many tiles have several parts
        }
    }
    joined = run.items <= p.items ? run.joined : 0;
    return found;
}

// The same where tree_division_kernel has been: the last request whose first item is not past `item` and that has any.
__device__ __forceinline__ bool look_up_work(const TreeAttnParams& p, int item, Work& work) {
    const int lane = threadIdx.x & 63;
    int row = 0, span = p.rows;
    while (span > 1) {
        const int step = (span + 63) / 64, at = row + lane * step;
        const bool upto = lane * step < span && at < p.rows && p.row_work[at].x <= item;  // true for the first lanes
        row += (__popcll(__ballot(upto)) - 1) * step;
        span = step;
    }
    row = __builtin_amdgcn_readfirstlane(row);
    const int4 w = p.row_work[row];
    work.row = row;
    work.before = {__builtin_amdgcn_readfirstlane(w.x), __builtin_amdgcn_readfirstlane(w.y), __builtin_amdgcn_readfirstlane(w.z)};
    work.parts = __builtin_amdgcn_readfirstlane(w.w);
    return true;
}

constexpr int DIVIDE_THREADS = 1024;
template <int ROWS>
__global__ __launch_bounds__(DIVIDE_THREADS) void tree_division_kernel(TreeAttnParams p) {
    constexpr int WAVES = DIVIDE_THREADS / 64;
    __shared__ WorkShared s;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int chunk = choose_part<ROWS, WAVES>(p, s, threadIdx.x, DIVIDE_THREADS);
    // a thread's rows are neighbours: sums in order
    const int each = (p.rows + DIVIDE_THREADS - 1) / DIVIDE_THREADS;
    const int begin = min(int(threadIdx.x) * each, p.rows), end = min(begin + each, p.rows);
    Sums own = {0, 0, 0};
    for (int r = begin; r < end; ++r) own = own + row_sums(request<ROWS>(p, r), chunk);
    const Sums incl = scan(own);
    if (lane == 63) s.waves[wave] = incl;
    __syncthreads();
    Sums run = incl - own;
    run.items = min(run.items, MOST_ITEMS);
    for (int w = 0; w < wave; ++w) run = run + s.waves[w];
    for (int r = begin; r < end; ++r) {
        const Request q = request<ROWS>(p, r);
        p.row_work[r] = make_int4(run.items, run.slots, run.joined, parts_of(q.span, chunk));
        run = run + row_sums(q, chunk);
    }
    if (threadIdx.x == DIVIDE_THREADS - 1) *p.joined = run.items <= p.items ? run.joined : 0;
}

// ------------------------------------------------------------------------------------ attention
__device__ const uint4 ZEROS = {0u, 0u, 0u, 0u};

// 16 bytes a lane into LDS, at `lds` (a wave's address) and the lanes side by side.  The compiler does not know of the
// load: what reads its bytes waits first.  No register is written, so nothing in flight can clobber one; M0 is named as
// clobbered, so that the compiler's own writes of it stay in order with these (s_nop: the wait state before its use).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_to_lds(uint32_t lds, uint64_t at) {
    __asm__ volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                     :
                     : "s"(__builtin_amdgcn_readfirstlane(int(lds))), "v"(at)
                     : "m0", "memory");
}
#pragma clang diagnostic pop
__device__ __forceinline__ uint32_t lds_address(const void* p) {
    return uint32_t(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) void*)p));
}

template <int TYPE>
__device__ __forceinline__ bool finite16(uint32_t h) {
    return TYPE == TYPE_BF16 ? (h & 0x7f80u) != 0x7f80u : (h & 0x7c00u) != 0x7c00u;
}
template <int TYPE>
__device__ __forceinline__ uint32_t finite_or_zero(uint32_t w) {
    return (finite16<TYPE>(w) ? w & 0xffffu : 0u) | (finite16<TYPE>(w >> 16) ? w & 0xffff0000u : 0u);
}

// Two weights rounded to the type, and what that leaves of them.
template <int TYPE>
__device__ __forceinline__ void split(float x, float y, uint32_t& high, uint32_t& low) {
    high = pack16<TYPE>(x, y);
    if constexpr (TYPE == TYPE_BF16) {
        // the differences are exact: the pair times (-1, 0) or (0, -1) onto the value (in registers: as literals one of
        // them would be encoded as the inline constant -1, which is no pair)
        uint32_t first = 0x0000bf80u, second = 0xbf800000u;
        __asm__("" : "+s"(first), "+s"(second));
        low = pack16<TYPE>(dot2bf(high, first, x), dot2bf(high, second, y));
    } else {
        low = pack16<TYPE>(x - from16<TYPE>(high), y - from16<TYPE>(high >> 16));
    }
}

// f(std::integral_constant<int, I>) for I = B .. E - 1.
template <int B, int E, class F>
__device__ __forceinline__ void static_for(F&& f) {
    if constexpr (B < E) {
        f(std::integral_constant<int, B>{});
        static_for<B + 1, E>(f);
    }
}

// Bits from .. to - 1 of 64 (any numbers).
__device__ __forceinline__ uint64_t bit_range(int from, int to) {
    const uint64_t below_to = to >= 64 ? ~0ull : to <= 0 ? 0ull : (1ull << to) - 1;
    const uint64_t below_from = from >= 64 ? ~0ull : from <= 0 ? 0ull : (1ull << from) - 1;
    return below_to & ~below_from;
}

template <int TYPE, int D, int SHARE, bool EVEN>
__global__ __launch_bounds__((Shape<D, SHARE>::THREADS), (Shape<D, SHARE>::OF_SIMD)) void tree_attention_kernel(TreeAttnParams p) {
    typedef Shape<D, SHARE> X;
    constexpr int ROWS = 32 * SHARE;
    __shared__ __align__(1024) uint8_t s_ring[X::LDS];
    __shared__ float2 s_ml[X::GROUPS][ROWS];
    __shared__ __align__(8) uint16_t s_there[X::GROUPS][2][4];  // of a stage's tile: bits of sixteen rows each
    __shared__ WorkShared s_work;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int part_wave = wave % SHARE, set = wave / SHARE;
    const int col = lane & 31, half = lane >> 5;
    const int kv = blockIdx.y;
    // workgroups go to the eight XCDs in turn
    const int seq = int(blockIdx.x >> 3);
    const int item = (seq / p.run * 8 + int(blockIdx.x & 7)) * p.run + seq % p.run;
    Work work = {};
    if (p.listed) {
        if (!look_up_work(p, item, work)) return;
    } else {
        int joined = 0;
        const bool any = find_work<ROWS, X::WAVES>(p, s_work, item, work, joined);
        if (item == 0 && kv == 0 && threadIdx.x == 0) *p.joined = joined;
        if (!any) return;  // every wave of the workgroup
    }
    const int row = __builtin_amdgcn_readfirstlane(work.row), parts = __builtin_amdgcn_readfirstlane(work.parts);
    Request rq = request<ROWS>(p, row);
    rq.first = __builtin_amdgcn_readfirstlane(rq.first);
    rq.count = __builtin_amdgcn_readfirstlane(rq.count);
    rq.start = __builtin_amdgcn_readfirstlane(rq.start);
    rq.end = __builtin_amdgcn_readfirstlane(rq.end);
    rq.tiles = __builtin_amdgcn_readfirstlane(rq.tiles);
    const int local = item - __builtin_amdgcn_readfirstlane(work.before.items);
    if (local >= rq.tiles * parts) return;  // past the last item
    const int part = local / rq.tiles, tile = local - part * rq.tiles;
    const int slot = __builtin_amdgcn_readfirstlane(work.before.slots) + local;
    if (parts > 1 && part == 0 && kv == 0 && threadIdx.x == 0) {
        int4* at = p.tile_work + 2 * (__builtin_amdgcn_readfirstlane(work.before.joined) + tile);
        at[0] = make_int4(row, tile, slot, rq.tiles);
        at[1] = make_int4(parts, 0, 0, 0);
    }
    // the lane's row of queries; those past the last are the last again
    const int rows = rq.count * p.group;
    const int own_row = tile * ROWS + part_wave * 32 + col, m = min(own_row, rows - 1);
    const int token = int(divide(uint32_t(m), p.by_group)), head = kv * p.group + (m - token * p.group);
    uint4 q[X::STEPS];
    {
        const uint16_t* from = p.q + int64_t(rq.first + token) * p.q_stride + int64_t(head) * D + 8 * half;
#pragma unroll
        for (int s = 0; s < X::STEPS; ++s) q[s] = *reinterpret_cast<const uint4*>(from + 16 * s);
    }
    // the scale is made positive, so that the largest product is the largest score: of the other sign, or of nothing
    const uint32_t flip = p.scale < 0.f ? 0x80008000u : 0u, kept = p.scale == 0.f ? 0u : ~0u;
    const float scale = p.scale == 0.f ? 1.0f : fabsf(p.scale);
#pragma unroll
    for (int s = 0; s < X::STEPS; ++s)
        q[s] = make_uint4((q[s].x ^ flip) & kept, (q[s].y ^ flip) & kept, (q[s].z ^ flip) & kept, (q[s].w ^ flip) & kept);
    // keys low .. high - 1 before the new tokens (and in a chain up to its own), and by bits
    const uint32_t* bits = nullptr;
    int position = rq.start + token, high = min(position + 1, rq.end);
    if (p.ancestors) {
        bits = p.ancestors + int64_t(rq.first + token) * p.words;
        position = p.positions[rq.first + token];
        high = min(rq.start, rq.end);
    }
    int low = p.window > 0 ? max(max(position, rq.start) - p.window + 1, 0) : 0;
    if (position < 0) {
        low = high = 0;
        bits = nullptr;
    }
    // of the tile: the keys that any of its tokens may see, and those that the wave's all see without a bit
    const int token0 = int(divide(uint32_t(tile * ROWS), p.by_group)), token1 = int(divide(uint32_t(min((tile + 1) * ROWS, rows) - 1), p.by_group));
    int first_key, end;
    if (p.ancestors) {
        first_key = p.window > 0 ? max(rq.start - p.window + 1, 0) : 0;
        end = rq.end;
    } else {
        first_key = p.window > 0 ? max(rq.start + token0 - p.window + 1, 0) : 0;
        end = min(rq.end, rq.start + token1 + 1);
    }
    first_key = min(first_key, end) & ~15;
    int all_low = low, all_high = high;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        all_low = max(all_low, __shfl_xor(all_low, o, 64));
        all_high = min(all_high, __shfl_xor(all_high, o, 64));
    }
    all_low = __builtin_amdgcn_readfirstlane(all_low);
    all_high = __builtin_amdgcn_readfirstlane(all_high);
    constexpr int TURN = X::KEYS * X::GROUPS;
    const int each = __builtin_amdgcn_readfirstlane(((end - first_key + parts - 1) / parts + TURN - 1) / TURN * TURN);
    const int begin = first_key + part * each;
    end = __builtin_amdgcn_readfirstlane(min(end, begin + each));

    // ---- loads: lane's row of a piece and its 16-byte chunk there
    constexpr int LANES = 64 / X::PIECE_KEYS;  // of a row
    const int group = lane / LANES;
    const uint32_t ring = lds_address(s_ring) + uint32_t(set) * (2 * 2 * X::TILE);  // a stage: keys, then values
    const uint64_t keys0 = reinterpret_cast<uint64_t>(p.keys) + kv * p.head_stride;
    const int64_t apart = p.values - p.keys;
    const int32_t* table = p.tables + int64_t(row) * p.width;
    const int first_row = 16 * X::OWN * part_wave;  // of a tile, that the wave loads
    // EVEN: the lane's keys of sixteen, PIECES of them, lie in one page.  (Where sixteen do, the wave could look the page up and find
    // its address: chunks of 999 and 333 tokens 496 -> 492 us, but the loads go out later: 16 requests of 78 rows of 256 59 -> 68, 48
    // of 38 rows of 64 with four waves 144 -> 166.)
    constexpr int LOOK = EVEN ? 1 : X::PIECES;
    const int lane_chunk = lane % LANES;
    const uint32_t lane_key = uint32_t(lane_chunk ^ key_swizzle<D>(group)) * 16;
    const uint32_t lane_value = uint32_t(((lane_chunk >> 2) ^ value_swizzle<D>(group)) * 4 + (lane_chunk & 3)) * 16;
    // pages of a tile's keys, on their way
    int entry[X::OWN][LOOK];
    auto look_up = [&](int pos) __attribute__((always_inline)) {
#pragma unroll
        for (int b = 0; b < X::OWN; ++b)
#pragma unroll
            for (int l = 0; l < LOOK; ++l) {
                const int key = pos + first_row + 16 * b + X::PIECES * group + l;
                entry[b][l] = key < end ? table[divide(uint32_t(key), p.div)] : -1;
            }
    };
    auto request_tile = [&](int pos, int stage) __attribute__((always_inline)) {
#pragma unroll
        for (int b = 0; b < X::OWN; ++b) {
            const int key0 = pos + first_row + 16 * b;  // of the sixteen
            const uint32_t to = ring + uint32_t(stage) * (2 * X::TILE) + uint32_t(first_row + 16 * b) * X::ROW;
            uint32_t there = 0xffffu;
            bool fine = key0 + 16 <= end;
            uint64_t at[LOOK];
#pragma unroll
            for (int l = 0; l < LOOK; ++l) {
                const int key = key0 + X::PIECES * group + l, in_page = key - int(divide(uint32_t(key), p.div)) * p.page_size;
                at[l] = keys0 + uint64_t(int64_t(entry[b][l]) * p.page_stride + int64_t(in_page) * p.slot_stride);
                fine = fine && uint32_t(entry[b][l]) < uint32_t(p.pages);
            }
            if (__all(fine)) {
                static_for<0, X::PIECES>([&](auto n) {
                    constexpr int l = decltype(n)::value;
                    const uint64_t from = at[EVEN ? 0 : l] + (EVEN ? uint64_t(l * p.slot_stride) : 0);
                    load_to_lds(to + uint32_t(l) * 1024, from + (lane_key ^ uint32_t(key_swizzle<D>(X::PIECE_KEYS * l) * 16)));
                    load_to_lds(to + X::TILE + uint32_t(l) * 1024,
                                from + uint64_t(apart) + (lane_value ^ uint32_t(value_swizzle<D>(X::PIECE_KEYS * l) * 64)));
                });
            } else {  // rows past the last key, or of no page, are zeros
                there = 0;
                int own = lane;
                __asm__ volatile("" : "+v"(own));  // (or the compiler would keep all offsets in registers)
                const int chunk = own % LANES, own_group = own / LANES;
#pragma unroll
                for (int l = 0; l < X::PIECES; ++l) {
                    const int key = key0 + X::PIECES * own_group + l, page = entry[b][EVEN ? 0 : l], r = X::PIECE_KEYS * l + own_group;
                    const int in_page = key - int(divide(uint32_t(key), p.div)) * p.page_size;
                    const uint64_t from = keys0 + uint64_t(int64_t(page) * p.page_stride + int64_t(in_page) * p.slot_stride);
                    const bool ok = key < end && uint32_t(page) < uint32_t(p.pages);
                    const uint64_t zeros = reinterpret_cast<uint64_t>(&ZEROS);
                    load_to_lds(to + uint32_t(l) * 1024, ok ? from + uint32_t((chunk ^ key_swizzle<D>(r)) * 16) : zeros);
                    load_to_lds(to + X::TILE + uint32_t(l) * 1024,
                                ok ? from + uint64_t(apart) + uint32_t((((chunk >> 2) ^ value_swizzle<D>(r)) * 4 + (chunk & 3)) * 16) : zeros);
                    const unsigned long long those = __ballot(ok);
#pragma unroll
                    for (int g = 0; g < X::PIECE_KEYS; ++g) there |= uint32_t(those >> (g * LANES) & 1u) << (X::PIECE_KEYS * l + g);
                }
            }
            if (lane == 0) s_there[set][stage][part_wave * X::OWN + b] = uint16_t(there);
        }
    };
    // the bits of the nodes in a tile, as far as they are needed: words from the first node's on
    struct Bits {
        uint32_t w[3];
    };
    Bits node_bits = {};
    auto look_at_bits = [&](int pos) __attribute__((always_inline)) {
        const int from = max(pos - rq.start, 0) >> 5;
        if (p.ancestors && pos + X::KEYS > rq.start) {
#pragma unroll
            for (int i = 0; i <= X::BLOCKS; ++i) node_bits.w[i] = bits && from + i < p.words ? bits[from + i] : 0u;
        }
    };

    // ---- a tile's products
    float most = NEG_INF, sum = 0.f;
    floatx16 o[X::DIMS];
#pragma unroll
    for (int d = 0; d < X::DIMS; ++d) o[d] = floatx16{};
    // Operands by a lane's base in a stage, exclusive-or'ed with the step: the bases are made new for each turn, or the compiler
    // would keep all their variants in registers.
    const uint32_t key_base = uint32_t(set * (2 * 2 * X::TILE) + col * X::ROW + (half ^ key_swizzle<D>(col)) * 16);
    // source lane l of 16 reads 8 bytes of row 4 (lane / 32) + l / 4; lane j gets dim 16 (lane / 16 % 2) + j of the four
    // rows, and of those 8 further (which have the same swizzle)
    const int source_row = 4 * half + (lane >> 2 & 3);
    const uint32_t value_base = uint32_t(set * (2 * 2 * X::TILE) + X::TILE + source_row * X::ROW + value_swizzle<D>(source_row) * 64 +
                                         32 * (lane >> 4 & 1) + 8 * (lane & 3));
    auto base_of = [&](uint32_t base, int stage) __attribute__((always_inline)) {
        uint32_t x = base + uint32_t(stage) * (2 * X::TILE);
        __asm__ volatile("" : "+v"(x));
        return x;
    };
    typedef short short4_t __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) short4_t* tr_ptr_t;
    // dims of d, keys of sixteen s
    auto value_operand = [&](uint32_t base, int s, int d) __attribute__((always_inline)) {
        const uint8_t* at = s_ring + (base ^ uint32_t(d * 64)) + 16 * s * X::ROW;
        const short4_t x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr_t)at);
        const short4_t x1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr_t)(at + 8 * X::ROW));
        uint4 v;
        __builtin_memcpy(&v, &x0, 8);
        __builtin_memcpy(reinterpret_cast<char*>(&v) + 8, &x1, 8);
        return v;
    };
    auto weight = [&](float x, float from) __attribute__((always_inline)) { return __builtin_amdgcn_exp2f(__builtin_fmaf(x, scale, -from)); };
    constexpr int SIXTEENS = X::KEYS / 16;
    // Weights in two halves of the type (2^-16 off for BF16, 2^-22 for FP16), a product for each.  Rounded once they would be half
    // a step off each, as large an error as the output's own rounding (outputs 1.2 to 1.4 times as far from 64 bits), for a third fewer products
    // (chunks of 999 and 333 tokens 380 us for 492, 64 trees of up to 24 nodes 40 for 44).

    bool odd = false;  // a tile that some tokens do not see whole holds values that are not finite
    auto take = [&](int pos, int stage, uint64_t there, const Bits& of_nodes, auto with_care) __attribute__((always_inline)) {
        constexpr int PRODUCTS = X::BLOCKS * X::STEPS, AHEAD = 4;
        const uint32_t k_base = base_of(key_base, stage), v_base = base_of(value_base, stage);
        floatx16 s[X::BLOCKS];
        {
            auto operand = [&](int i) {
                return *reinterpret_cast<const uint4*>(s_ring + (k_base ^ uint32_t(i / X::BLOCKS * 32)) + i % X::BLOCKS * 32 * X::ROW);
            };
            uint4 k[AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) k[i] = operand(i);
            static_for<0, PRODUCTS>([&](auto n) {
                constexpr int i = decltype(n)::value, b = i % X::BLOCKS, t = i / X::BLOCKS;
                s[b] = mfma32<TYPE>(k[i % AHEAD], q[t], t == 0 ? floatx16{} : s[b]);
                if constexpr (i + AHEAD < PRODUCTS) k[i % AHEAD] = operand(i + AHEAD);
                __builtin_amdgcn_sched_barrier(0);
            });
        }
        uint32_t seen[X::BLOCKS];  // bit i: score i is one
#pragma unroll
        for (int b = 0; b < X::BLOCKS; ++b) seen[b] = 0xffffu;
        constexpr uint64_t ALL = X::KEYS == 64 ? ~0ull : 0xffffffffull;
        const bool whole = pos >= all_low && pos + X::KEYS <= all_high && there == ALL;
        if (!whole) {
            // what the lane's token sees of the keys in their order, then of its scores in theirs
            uint64_t see = bit_range(low - pos, high - pos);
            const int node = pos - rq.start;  // of the tile's first key
            if (p.ancestors && node > -X::KEYS) {
                const int shift = max(node, 0) & 31;
                uint64_t of = (uint64_t(of_nodes.w[1]) << 32 | of_nodes.w[0]) >> shift;
                if (X::BLOCKS > 1 && shift) of |= uint64_t(of_nodes.w[2]) << (64 - shift);
                see |= node < 0 ? of << -node : of;
            }
            see >>= HALF_KEY<D> * half;
            const uint64_t rows_there = there >> (4 * half);
#pragma unroll
            for (int b = 0; b < X::BLOCKS; ++b) {
                seen[b] = 0;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const uint32_t yes = uint32_t(see >> (32 * b)) >> score_key<D>(i) & uint32_t(rows_there >> (32 * b)) >> (8 * (i / 4) + i % 4) & 1u;
                    seen[b] |= yes << i;
                    s[b][i] = yes ? s[b][i] : NEG_INF;
                }
            }
            // are all values finite?  An exponent of ones and a one more carry into the sign's bit
            constexpr uint32_t EXPONENT = TYPE == TYPE_BF16 ? 0x7f807f80u : 0x7c007c00u, ONE = TYPE == TYPE_BF16 ? 0x00800080u : 0x04000400u;
            uint32_t carry = 0;
#pragma unroll 4
            for (int c = lane * 16; c < X::TILE; c += 1024) {
                const uint4 w = *reinterpret_cast<const uint4*>(s_ring + (set * 2 + stage) * (2 * X::TILE) + X::TILE + c);
                carry |= ((w.x & EXPONENT) + ONE) | ((w.y & EXPONENT) + ONE) | ((w.z & EXPONENT) + ONE) | ((w.w & EXPONENT) + ONE);
            }
            odd = odd || __any(carry & 0x80008000u);
        }
        float top = s[0][0];
#pragma unroll
        for (int b = 0; b < X::BLOCKS; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, s[b][i]);
        top = fmaxf(top, xor_lane<32>(top));
        const float before = most;
        most = fmaxf(before, top);
        // exponents are taken from the maximum, or any number while that is minus infinity
        const float from = (most == NEG_INF ? 0.f : most * scale) - weight_shift<TYPE>();
        if (__any(most > before)) {
            const float shrink = before == NEG_INF ? 0.f : __builtin_amdgcn_exp2f(before * scale - weight_shift<TYPE>() - from);
            sum *= shrink;
#pragma unroll
            for (int d = 0; d < X::DIMS; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= shrink;
        }
        if constexpr (!decltype(with_care)::value) {
            constexpr int PAIRS = X::DIMS / 2;
            uint32_t high_w[2][4], low_w[2][4];
            uint4 v[2][2];
            v[0][0] = value_operand(v_base, 0, 0);
            v[0][1] = value_operand(v_base, 0, 1);
            // sixteen n / 4: the weights of its eight scores of the lane, two at a time, beside the products of the sixteen
            // before: a wave issues in order, and only so do the matrix units work meanwhile
            static_for<0, 4 * (SIXTEENS + 1)>([&](auto n) {
                constexpr int u = decltype(n)::value / 4, k = decltype(n)::value % 4;
                if constexpr (u > 0) {
                    constexpr int g = (u - 1) & 1;
                    const uint4 ph = make_uint4(high_w[g][0], high_w[g][1], high_w[g][2], high_w[g][3]);
                    const uint4 pl = make_uint4(low_w[g][0], low_w[g][1], low_w[g][2], low_w[g][3]);
                    // products of the pairs of d: high, high, low, low
                    constexpr int OF_PAIR = 4, ALL_OF = PAIRS * OF_PAIR;
                    static_for<k * ALL_OF / 4, (k + 1) * ALL_OF / 4>([&](auto m) {
                        constexpr int pair = decltype(m)::value / OF_PAIR, j = decltype(m)::value % OF_PAIR, turn = ((u - 1) * PAIRS + pair) & 1;
                        if constexpr (j == 0 && (u < SIXTEENS || pair + 1 < PAIRS)) {  // the next pair's operands
                            constexpr int u2 = pair + 1 < PAIRS ? u - 1 : u, p2 = pair + 1 < PAIRS ? pair + 1 : 0;
                            v[turn ^ 1][0] = value_operand(v_base, u2, 2 * p2);
                            v[turn ^ 1][1] = value_operand(v_base, u2, 2 * p2 + 1);
                        }
                        o[2 * pair + (j & 1)] = mfma32<TYPE>(v[turn][j & 1], j < 2 ? ph : pl, o[2 * pair + (j & 1)]);
                    });
                }
                if constexpr (u < SIXTEENS) {
                    constexpr int b = u / 2, i = (u & 1) * 8 + 2 * k;
                    const float x = weight(s[b][i], from), y = weight(s[b][i + 1], from);
                    sum += x;
                    sum += y;
                    split<TYPE>(x, y, high_w[u & 1][k], low_w[u & 1][k]);
                }
                __builtin_amdgcn_sched_barrier(0);
            });
            return;
        }
        // Values that are not finite reach those tokens alone that see their key: they are left out of the products (where a
        // weight of zero would make NaN of them) and added one by one.
#pragma unroll
        for (int b = 0; b < X::BLOCKS; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[b][i] = weight(s[b][i], from);
                sum += s[b][i];
            }
        int half = lane >> 5;
        __asm__ volatile("" : "+v"(half));  // (as the bases)
        const uint8_t* const values = s_ring + (set * 2 + stage) * (2 * X::TILE) + X::TILE;
        for (int r = 0; r < X::KEYS; ++r) {
            bool bad = false;
            for (int c = lane * 4; c < X::ROW; c += 256) {
                const uint32_t w = *reinterpret_cast<const uint32_t*>(values + r * X::ROW + c);
                bad |= !(finite16<TYPE>(w) && finite16<TYPE>(w >> 16));
            }
            if (!__any(bad)) continue;
            const int index = (r & 32) / 2 + (r & 24) / 2 + (r & 3), side = r >> 2 & 1;  // of the lane's scores, and the half
            float w = 0.f;
            uint32_t sees = 0;
#pragma unroll
            for (int b = 0; b < X::BLOCKS; ++b) {
#pragma unroll
                for (int i = 0; i < 16; ++i) w = index == 16 * b + i ? s[b][i] : w;
                sees = index >> 4 == b ? seen[b] >> (index & 15) & 1u : sees;
            }
            const float partner = xor_lane<32>(w);
            const uint32_t partners = xor_lane<32>(sees);
            w = side == half ? w : partner;
            sees = side == half ? sees : partners;
            static_for<0, X::DIMS * 4>([&](auto n) {
                constexpr int d = decltype(n)::value / 4, i = decltype(n)::value % 4 * 4;
                const uint2 h = *reinterpret_cast<const uint2*>(values + r * X::ROW + (d ^ value_swizzle<D>(r)) * 64 + (8 * (i / 4) + 4 * half) * 2);
                const uint32_t of[4] = {h.x & 0xffffu, h.x >> 16, h.y & 0xffffu, h.y >> 16};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float add = w * from16<TYPE>(of[e]);
                    o[d][i + e] += sees && !finite16<TYPE>(of[e]) ? add : 0.f;
                }
                __asm__ volatile("" ::: "memory");  // (a few values at a time: registers)
            });
        }
#pragma unroll
        for (int u = 0; u < SIXTEENS; ++u) {
            uint32_t hw[4], lw[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) split<TYPE>(s[u / 2][(u & 1) * 8 + 2 * i], s[u / 2][(u & 1) * 8 + 2 * i + 1], hw[i], lw[i]);
            const uint4 ph = make_uint4(hw[0], hw[1], hw[2], hw[3]), pl = make_uint4(lw[0], lw[1], lw[2], lw[3]);
#pragma unroll
            for (int d = 0; d < X::DIMS; ++d) {
                uint4 v = value_operand(v_base, u, d);
                v = make_uint4(finite_or_zero<TYPE>(v.x), finite_or_zero<TYPE>(v.y), finite_or_zero<TYPE>(v.z), finite_or_zero<TYPE>(v.w));
                o[d] = mfma32<TYPE>(v, ph, o[d]);
                o[d] = mfma32<TYPE>(v, pl, o[d]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };

    // ---- the part's tiles, the next one's loads on their way
    const int turns = begin < end ? (end - begin + TURN - 1) / TURN : 0;
    // a wave that has no rows only loads (64 trees of up to 24 nodes behind 33 to 8,192 keys 43.2 -> 42.5 us,
    // 64 requests of 73 rows behind 2,000 to 4,000 40 -> 38.5)
    const bool live = tile * ROWS + part_wave * 32 < rows;
    const int taken = live ? end : 0;
    auto run = [&](auto with_care) __attribute__((always_inline)) {
        int pos = begin + set * X::KEYS;
        if (turns > 0) {
            look_up(pos);
            request_tile(pos, 0);
            look_up(pos + TURN);
            look_at_bits(pos);
        }
        for (int turn = 0; turn < turns; ++turn, pos += TURN) {
            __asm__ volatile("" ::: "memory");
            __builtin_amdgcn_s_waitcnt(0x0070);  // the wave's loads, and its LDS operations of the tile before
            if (SHARE > 1) __builtin_amdgcn_s_barrier();
            __asm__ volatile("" ::: "memory");
            const int stage = turn & 1;
            uint64_t there = X::KEYS == 64 ? *reinterpret_cast<const uint64_t*>(s_there[set][stage]) : *reinterpret_cast<const uint32_t*>(s_there[set][stage]);
            there = uint64_t(uint32_t(__builtin_amdgcn_readfirstlane(int(there >> 32)))) << 32 | uint32_t(__builtin_amdgcn_readfirstlane(int(there)));
            const Bits of_nodes = node_bits;
            if (turn + 1 < turns) {
                request_tile(pos + TURN, stage ^ 1);
                look_up(pos + 2 * TURN);
                look_at_bits(pos + TURN);
            }
            if (pos < taken) take(pos, stage, there, of_nodes, with_care);
        }
    };
    run(std::false_type{});
    // once more where values need care: in the same loop their arithmetic cost every tile 64 moves of registers (with weights
    // rounded once, chunks of 999 and 333 tokens 412 us, so 371)
    if (__syncthreads_or(odd)) {
        most = NEG_INF;
        sum = 0.f;
#pragma unroll
        for (int d = 0; d < X::DIMS; ++d) o[d] = floatx16{};
        run(std::true_type{});
        __syncthreads();
    }
    sum += xor_lane<32>(sum);

    // ---- the sets joined, in LDS where the tiles were
    const float exponent = most == NEG_INF ? NEG_INF : most * scale;
    float total = sum, top = exponent;
    constexpr int EACH = X::SPLIT / X::GROUPS;
    float4 mine[EACH];
    if constexpr (X::GROUPS > 1) {
        if (half == 0) s_ml[set][part_wave * 32 + col] = make_float2(exponent, sum);
        __syncthreads();
        top = NEG_INF;
#pragma unroll
        for (int g = 0; g < X::GROUPS; ++g) top = fmaxf(top, s_ml[g][part_wave * 32 + col].x);
        total = 0.f;
#pragma unroll
        for (int g = 0; g < X::GROUPS; ++g) {
            const float2 ml = s_ml[g][part_wave * 32 + col];
            total += ml.y == 0.f ? 0.f : ml.y * __builtin_amdgcn_exp2f(ml.x - top);  // (NaN alone leaves the maximum at minus infinity)
        }
        const float share = exponent == NEG_INF ? 0.f : __builtin_amdgcn_exp2f(exponent - top);
        auto piece = [&](int e) {
            return make_float4(o[e >> 2][4 * (e & 3)] * share, o[e >> 2][4 * (e & 3) + 1] * share, o[e >> 2][4 * (e & 3) + 2] * share,
                               o[e >> 2][4 * (e & 3) + 3] * share);
        };
        // a set gives each other one its EACH pieces of the dims: [to][from][wave of the set][EACH][64]
        float4* all = reinterpret_cast<float4*>(s_ring);
        static_assert((X::GROUPS - 1) * SHARE * X::SPLIT * 1024 <= X::LDS, "where the tiles were");
#pragma unroll
        for (int g = 0; g < X::GROUPS; ++g)
#pragma unroll
            for (int e = 0; e < EACH; ++e) {
                if (g == set) mine[e] = piece(g * EACH + e);
                else all[(((g * (X::GROUPS - 1) + (set < g ? set : set - 1)) * SHARE + part_wave) * EACH + e) * 64 + lane] = piece(g * EACH + e);
            }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < EACH; ++e)
#pragma unroll
            for (int g = 0; g < X::GROUPS - 1; ++g) {
                const float4 v = all[(((set * (X::GROUPS - 1) + g) * SHARE + part_wave) * EACH + e) * 64 + lane];
                mine[e].x += v.x, mine[e].y += v.y, mine[e].z += v.z, mine[e].w += v.w;
            }
    } else {
#pragma unroll
        for (int e = 0; e < EACH; ++e)
            mine[e] = make_float4(o[e >> 2][4 * (e & 3)], o[e >> 2][4 * (e & 3) + 1], o[e >> 2][4 * (e & 3) + 2], o[e >> 2][4 * (e & 3) + 3]);
    }
    if (parts > 1) {
        const int64_t at = (int64_t(slot) * p.kv_heads + kv) * SHARE + part_wave;
        float4* to = reinterpret_cast<float4*>(p.part_o) + (at * X::SPLIT + set * EACH) * 64 + lane;
#pragma unroll
        for (int e = 0; e < EACH; ++e)
            if (live) to[e * 64] = mine[e];
        if (live && set == 0 && half == 0) p.part_ml[at * 32 + col] = make_float2(top, total);
        return;
    }
    if (own_row >= rows) return;
    const float r = total == 0.f ? 0.f : 1.0f / total;  // nothing visible: zeros
    uint16_t* to = p.out + int64_t(rq.first + token) * p.out_stride + int64_t(head) * D + 4 * half;
#pragma unroll
    for (int e = 0; e < EACH; ++e)
        *reinterpret_cast<uint2*>(to + 8 * (set * EACH + e)) =
            make_uint2(pack16<TYPE>(mine[e].x * r, mine[e].y * r), pack16<TYPE>(mine[e].z * r, mine[e].w * r));
    if (p.lse && set == 0 && half == 0)
        p.lse[int64_t(rq.first + token) * (p.kv_heads * p.group) + head] =
            total == 0.f ? NEG_INF : (top - weight_shift<TYPE>() + log2f(total)) * 0.69314718055994531f;
}

// ------------------------------------------------------------------------------------ parts joined
// 32 rows of a tile and a quarter of their dims, in a fixed order: a workgroup's waves take every eighth part, and are
// joined in LDS.  Pieces lie as the attention's lanes held them.  Latency-bound: a part's maximum and results, some of each on
// their way at once, then LDS (509 parts of 128 rows of 128 8 us, 33 MB; one request's three 3 us).
constexpr int JOIN_WAVES = 8;
template <int TYPE, int D, int SHARE>
__global__ __launch_bounds__(64 * JOIN_WAVES) void tree_join_kernel(TreeAttnParams p) {
    constexpr int ROWS = 32 * SHARE, SPLIT = D / 8, EACH = SPLIT / 4, AHEAD = 4;
    __shared__ __align__(16) float4 s_o[JOIN_WAVES][EACH][64];
    __shared__ float2 s_ml[JOIN_WAVES][32];
    if (int(blockIdx.x) >= *p.joined) return;
    const int4 tile = p.tile_work[2 * blockIdx.x];
    const int parts = p.tile_work[2 * blockIdx.x + 1].x;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, half = lane >> 5;
    const int kv = blockIdx.y, part_wave = blockIdx.z / 4, quarter = blockIdx.z & 3;
    const int first_token = p.offsets[tile.x], rows = (p.offsets[tile.x + 1] - first_token) * p.group;
    const int own_row = tile.y * ROWS + part_wave * 32 + col;
    if (tile.y * ROWS + part_wave * 32 >= rows) return;
    float m = NEG_INF, l = 0.f;
    float4 o[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) o[e] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = wave; i < parts; i += JOIN_WAVES * AHEAD) {
        float2 ml[AHEAD];
        float4 v[AHEAD][EACH];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            const int at_part = min(i + a * JOIN_WAVES, parts - 1);
            const int64_t at = ((int64_t(tile.z) + int64_t(at_part) * tile.w) * p.kv_heads + kv) * SHARE + part_wave;
            ml[a] = p.part_ml[at * 32 + col];
#pragma unroll
            for (int e = 0; e < EACH; ++e) v[a][e] = reinterpret_cast<const float4*>(p.part_o)[(at * SPLIT + quarter * EACH + e) * 64 + lane];
        }
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            if (i + a * JOIN_WAVES >= parts) break;
            const float most = fmaxf(m, ml[a].x), from = most == NEG_INF ? 0.f : most;
            const float keep = __builtin_amdgcn_exp2f(m - from), share = __builtin_amdgcn_exp2f(ml[a].x - from);
            m = most;
            l = l * keep + ml[a].y * share;
#pragma unroll
            for (int e = 0; e < EACH; ++e) {
                o[e].x = o[e].x * keep + v[a][e].x * share, o[e].y = o[e].y * keep + v[a][e].y * share;
                o[e].z = o[e].z * keep + v[a][e].z * share, o[e].w = o[e].w * keep + v[a][e].w * share;
            }
        }
    }
#pragma unroll
    for (int e = 0; e < EACH; ++e) s_o[wave][e][lane] = o[e];
    if (half == 0) s_ml[wave][col] = make_float2(m, l);
    __syncthreads();
    if (wave >= EACH || own_row >= rows) return;
    const int live = min(JOIN_WAVES, parts);
    m = NEG_INF;
    for (int w = 0; w < live; ++w) m = fmaxf(m, s_ml[w][col].x);
    const float from = m == NEG_INF ? 0.f : m;
    l = 0.f;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int w = 0; w < live; ++w) {
        const float share = __builtin_amdgcn_exp2f(s_ml[w][col].x - from);
        const float4 v = s_o[w][wave][lane];
        l += s_ml[w][col].y * share;
        sum.x += v.x * share, sum.y += v.y * share, sum.z += v.z * share, sum.w += v.w * share;
    }
    const float r = l == 0.f ? 0.f : 1.0f / l;
    const int token = int(divide(uint32_t(own_row), p.by_group)), head = kv * p.group + (own_row - token * p.group);
    *reinterpret_cast<uint2*>(p.out + int64_t(first_token + token) * p.out_stride + int64_t(head) * D + 8 * (quarter * EACH + wave) + 4 * half) =
        make_uint2(pack16<TYPE>(sum.x * r, sum.y * r), pack16<TYPE>(sum.z * r, sum.w * r));
    if (p.lse && quarter == 0 && wave == 0 && half == 0)
        p.lse[int64_t(first_token + token) * (p.kv_heads * p.group) + head] =
            l == 0.f ? NEG_INF : (m - weight_shift<TYPE>() + log2f(l)) * 0.69314718055994531f;
}

// ------------------------------------------------------------------------------------ launches
// Waves that share a tile, by the rows of queries that a request has on the average: few rows read the keys at the rate of
// memory, and more rows a tile read them fewer times; many are bound by arithmetic.  64 requests of 2,000 to 4,000 keys and 16
// heads of 128 on one, 14 / 22 / 29 / 36 / 58 / 73 / 116 / 153 rows each: 27 / 27 / 30 / 31 / 44 / 49 / 61 / 104 us with one wave,
// 27 / 27 / 29 / 29 / 34 / 36 / 45 / 52 with two, 28 / 28 / 32 / 33 / 36 / 37 / 46 / 50 with four.  16 of 2,000 to 9,000 keys, 8 heads of
// 256 on 2, 18 / 39 / 78 rows: 46 / 60 / 94, 48 / 51 / 65 and 53 / 56 / 59.  (Heads of 64 cross over later between two and
// four: 48 requests, 32 heads on 8, 38 / 117 rows 105 / 252 with two and 144 / 300 with four, 4 requests of 2,000 rows 264 and 170.)
int share_of(int rows, int tokens, int group) {
    const int64_t each = int64_t(tokens) * group / rows;
    return each <= 24 ? 1 : each <= 72 ? 2 : 4;
}
// Workgroups that the CUs hold at once.
int target_of(int share, int kv_heads, int head_dim) {
    return std::max(1, CUS * (head_dim == 256 || (head_dim == 128 && share == 1) ? 1 : head_dim == 64 && share == 2 ? 3 : 2) / kv_heads);
}
int turn_of(int share, int head_dim) {
    return (share == 4 ? 64 : 32) * (share == 4 ? 1 : share == 2 || head_dim == 256 ? 2 : 4);
}
// (2^20 requests and 2^30 rows of queries are less than 2^24 workgroups: a launch holds them)
int64_t tiles_of(const TreeAttnParams& p) { return std::min(p.rows, p.tokens) + int64_t(p.tokens) * p.group / (32 * p.share); }
int64_t items_of(const TreeAttnParams& p) {
    const int64_t items = tiles_of(p) + (p.joins ? p.target : 0), turn = 8 * p.run;
    return (items + turn - 1) / turn * turn;
}
constexpr int FOUND_ROWS = 1024;

template <int TYPE, int D, int SHARE>
void run_shape(const TreeAttnParams& p, hipStream_t s) {
    typedef Shape<D, SHARE> X;
    if (p.listed) hipLaunchKernelGGL((tree_division_kernel<32 * SHARE>), dim3(1), dim3(DIVIDE_THREADS), 0, s, p);
    const dim3 grid(unsigned(p.items), unsigned(p.kv_heads));
    if (p.page_size % X::PIECES == 0) hipLaunchKernelGGL((tree_attention_kernel<TYPE, D, SHARE, true>), grid, dim3(X::THREADS), 0, s, p);
    else hipLaunchKernelGGL((tree_attention_kernel<TYPE, D, SHARE, false>), grid, dim3(X::THREADS), 0, s, p);
    if (p.joins)
        hipLaunchKernelGGL((tree_join_kernel<TYPE, D, SHARE>), dim3(unsigned(std::min<int64_t>(tiles_of(p), p.target)), unsigned(p.kv_heads), 4 * SHARE),
                           dim3(64 * JOIN_WAVES), 0, s, p);
}
template <int TYPE, int D>
void run_dim(const TreeAttnParams& p, hipStream_t s) {
    if (p.share == 1) run_shape<TYPE, D, 1>(p, s);
    else if (p.share == 2) run_shape<TYPE, D, 2>(p, s);
    else run_shape<TYPE, D, 4>(p, s);
}
template <int TYPE>
void run_type(const TreeAttnParams& p, int head_dim, hipStream_t s) {
    if (head_dim == 64) run_dim<TYPE, 64>(p, s);
    else if (head_dim == 128) run_dim<TYPE, 128>(p, s);
    else run_dim<TYPE, 256>(p, s);
}

struct Layout {
    int64_t row_work, tile_work, part_ml, part_o, bytes;
};
Layout layout(int rows, int share, int target, int kv_heads, int head_dim) {
    Layout l;
    const int64_t slots = 2 * int64_t(target) * kv_heads * 32 * share;  // rows of all parts
    l.row_work = 16;
    l.tile_work = l.row_work + int64_t(rows) * int64_t(sizeof(int4));
    l.part_ml = l.tile_work + int64_t(target) * 2 * int64_t(sizeof(int4));
    l.part_o = l.part_ml + slots * int64_t(sizeof(float2));
    l.bytes = l.part_o + slots * head_dim * int64_t(sizeof(float));
    return l;
}

}  // namespace

int64_t tree_attn_workspace(int rows, int tokens, int heads, int kv_heads, int head_dim) {
    // enough for fewer rows and tokens too: the fewer the rows, the more waves a tile, and each number of waves that a call of
    // them can have counts
    int64_t bytes = 0;
    for (int share = 1; share <= share_of(1, tokens, heads / kv_heads); share *= 2)
        bytes = std::max(bytes, layout(rows, share, target_of(share, kv_heads, head_dim), kv_heads, head_dim).bytes);
    return bytes;
}

void tree_attn_bind(TreeAttnParams& p, void* workspace, int head_dim) {
    p.share = share_of(p.rows, p.tokens, p.group);
    p.target = target_of(p.share, p.kv_heads, head_dim);
    p.by_group = divider(uint32_t(p.group));
    p.least = turn_of(p.share, head_dim);
    p.joins = p.most > p.least;
    // Neighbouring workgroups are tiles of the same keys: an XCD takes as many as a request has, as a power of two, so that the
    // workgroups that the XCDs hold at once stay as many on each (chunks of 999 and 333 tokens 507 -> 496 us; 64 requests of two tiles
    // or so 42.5 either way, but 77 MB fetched for 123; by runs of three 64 requests of one tile took 39 us for 27).
    const int64_t tiles = (int64_t(p.tokens) * p.group / p.rows + 32 * p.share - 1) / (32 * p.share);
    p.run = 1;
    while (p.run < tiles && p.run < 16 && p.run * 16 <= p.target) p.run *= 2;
    p.items = int(items_of(p));
    p.listed = p.rows > FOUND_ROWS;
    const Layout l = layout(p.rows, p.share, p.target, p.kv_heads, head_dim);
    char* at = static_cast<char*>(workspace);
    p.joined = reinterpret_cast<int*>(at);
    p.row_work = reinterpret_cast<int4*>(at + l.row_work);
    p.tile_work = reinterpret_cast<int4*>(at + l.tile_work);
    p.part_ml = reinterpret_cast<float2*>(at + l.part_ml);
    p.part_o = reinterpret_cast<float*>(at + l.part_o);
}

void launch_tree_attention(const TreeAttnParams& p, int type, int head_dim, hipStream_t s) {
    if (p.tokens == 0) return;
    if (type == TYPE_BF16) run_type<TYPE_BF16>(p, head_dim, s);
    else run_type<TYPE_F16>(p, head_dim, s);
}

}  // namespace plamo
