// Serving many requests from one pool of KV pages on gfx950.
//
//   paged_tables_kernel     pages taken from and given back to the free list, block tables, offsets
//   paged_slots_kernel      slot and position of each new token
//   paged_qkv_kernel        q and k RMS-normalised and rotated, k and v written to their slots
//   paged_parts_kernel      how the keys of very many rows are divided
//   paged_attention_kernel  attention of one token per request over its pages, split over the keys
//   paged_merge_kernel      parts of a row joined
#include <hip/hip_runtime.h>

#include <algorithm>

#include "common.h"
#include "paged_device.h"

namespace plamo {
using namespace dev;

namespace {

// ------------------------------------------------------------------------------------ tables
// One workgroup: prefix sums over the requests of pages given back, pages taken and tokens, then the
// moves flattened over pages so that a long request's are not one thread's.  Latency-bound: a few KB move
// in the time of some dependent loads (lengths, free pages, tables) and barriers: 64 requests of one new token
// 7.2 us with their slots, 1,000 requests that end, grow and begin 13.2, and 4.1 for 65,536 slots.  Checking that
// what goes back or is filled is a page is 0.9 and 1.6 us of that.  More than one workgroup would have to wait for
// each other between the checks of all requests and the first write.
constexpr int TABLE_THREADS = 1024;

// Places up to which the tables' workgroup fills in the slots too: each costs a search of the offsets, which
// one CU does more slowly than all, but a launch costs 2 us (2,048 places: 8.4 us so, 9.6 in a launch of their
// own; 4,096: 10.1 and 9.7).
constexpr int SLOTS_IN_TABLES = 2048;

// Table entries that requests may give back in a step (their places are 32-bit numbers), and how many are kept in LDS
// between the check and the move, which is then no second reading of the tables.
constexpr int MOST_GIVEN = 1 << 30, KEPT_GIVEN = 8192;

struct Scan3 {
    int back, take, fresh;
};

template <int CONTROL, int ROWS = 0xf>
__device__ __forceinline__ void add_shifted(Scan3& v) {
    v.back += shifted<CONTROL, ROWS>(v.back);
    v.take += shifted<CONTROL, ROWS>(v.take);
    v.fresh += shifted<CONTROL, ROWS>(v.fresh);
}

// Inclusive sums over the workgroup; `total` in every thread.  Rows of 16 lanes by shifts of 1, 2, 4 and 8,
// then the last lane of the row, and of the half, before; the waves' sums as one such row.
__device__ __forceinline__ Scan3 block_scan3(Scan3 v, Scan3* waves, Scan3& total) {
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
    static_assert(TABLE_THREADS / 64 == 16, "a row");
    Scan3 sum = waves[lane & 15];
    add_shifted<0x111>(sum);
    add_shifted<0x112>(sum);
    add_shifted<0x114>(sum);
    add_shifted<0x118>(sum);
    auto of = [&](int l) -> Scan3 {
        return {__builtin_amdgcn_readlane(sum.back, l), __builtin_amdgcn_readlane(sum.take, l), __builtin_amdgcn_readlane(sum.fresh, l)};
    };
    total = of(15);
    if (wave > 0) {
        const Scan3 before = of(wave - 1);
        v = {v.back + before.back, v.take + before.take, v.fresh + before.fresh};
    }
    return v;
}

// What a request of this length and count (both checked) asks for.
__device__ __forceinline__ Scan3 row_moves(const PagedTablesParams& p, int length, int count, int& held) {
    held = int((int64_t(length) + p.page_size - 1) / p.page_size);
    if (count < 0) return {held, 0, 0};
    return {0, int((int64_t(length) + count + p.page_size - 1) / p.page_size) - held, count};
}

// The first of `n` ascending inclusive sums above x.
__device__ __forceinline__ int first_above(const int* sums, int n, int x) {
    int lo = 0;
    while (n > 0) {
        const int half = n >> 1;
        if (sums[lo + half] > x) {
            n = half;
        } else {
            lo += half + 1;
            n -= half + 1;
        }
    }
    return lo;
}

__device__ __forceinline__ bool is_page(const PagedTablesParams& p, int32_t entry) { return uint32_t(entry) < uint32_t(p.pages); }

struct TablesShared {
    Scan3 waves[TABLE_THREADS / 64];
    int sums[TABLE_THREADS], start[TABLE_THREADS], held[TABLE_THREADS];
};

// f(i, entry) for the table entries of all requests that end, in the order of requests and entries: a workgroup's
// threads side by side, those past the last one with no i (INT32_MAX) and -1.
template <typename F>
__device__ __forceinline__ void for_given(const PagedTablesParams& p, TablesShared& s, int own_length, int own_count, F f) {
    const int tid = threadIdx.x;
    int before = 0;
    for (int base = 0; base < p.rows; base += TABLE_THREADS) {
        const int r = base + tid;
        int held = 0, back = 0;
        if (r < p.rows) back = row_moves(p, base ? p.lengths[r] : own_length, base ? p.counts[r] : own_count, held).back;
        Scan3 sum;
        const Scan3 incl = block_scan3({back, 0, 0}, s.waves, sum);
        s.sums[tid] = incl.back;
        s.start[tid] = incl.back - back;
        __syncthreads();
        for (int at = 0; at < sum.back; at += TABLE_THREADS) {
            const int e = at + tid;
            int32_t entry = -1;
            if (e < sum.back) {
                const int q = first_above(s.sums, TABLE_THREADS, e);
                entry = p.tables[int64_t(base + q) * p.width + (e - s.start[q])];
            }
            f(e < sum.back ? before + e : INT32_MAX, entry);
        }
        before += sum.back;
    }
}

// Token j of the step: its request by the ends of all requests' tokens, its position before the request's new
// length, its slot.
__device__ __forceinline__ void token_slot(const PagedTablesParams& p, const int* ends, const int* lengths, int j, int total) {
    int slot = -1, at = -1;
    if (j < total) {
        const int r = first_above(ends, p.rows, j);
        at = lengths[r] - (ends[r] - j);
        const uint32_t page = divide(uint32_t(at), p.div);
        slot = p.tables[int64_t(r) * p.width + page] * p.page_size + (at - int(page) * p.page_size);
    }
    p.slots[j] = slot;
    p.positions[j] = at;
}

template <bool SLOTS>
__global__ __launch_bounds__(TABLE_THREADS) void paged_tables_kernel(PagedTablesParams p) {
    __shared__ TablesShared s;
    __shared__ unsigned long long s_back, s_take, s_fresh;
    __shared__ int s_status, s_given;
    __shared__ int32_t s_entries[KEPT_GIVEN];
    // where the requests' tokens end, and their new lengths (of the last TABLE_THREADS requests)
    __shared__ int s_ends[SLOTS ? TABLE_THREADS : 1], s_lengths[SLOTS ? TABLE_THREADS : 1];
    const int tid = threadIdx.x;
    if (tid == 0) {
        s_back = s_take = s_fresh = 0;
        s_status = s_given = 0;
    }
    const int64_t first = *p.free_count;
    // the stack's top is on its way while the requests are added up
    const int64_t own_top = first - 1 - tid;
    const int32_t own_page = own_top >= 0 && own_top < p.pages ? p.free_pages[own_top] : -1;
    // the first TABLE_THREADS requests' stay in registers
    int own_length = 0, own_count = 0;
    if (tid < p.rows) {
        own_length = p.lengths[tid];
        own_count = p.counts[tid];
    }
    __syncthreads();
    // totals and checks before anything is written
    int bad = 0;
    long long back = 0, take = 0, fresh = 0;
    for (int r = tid; r < p.rows; r += TABLE_THREADS) {
        const int64_t length = r == tid ? own_length : p.lengths[r], count = r == tid ? own_count : p.counts[r];
        if (length < 0 || count < -1) {
            bad |= 8;
            continue;
        }
        const int64_t held = (length + p.page_size - 1) / p.page_size;
        const int64_t after = count < 0 ? 0 : (length + count + p.page_size - 1) / p.page_size;
        if (held > p.width || after > p.width || length + count > INT32_MAX) bad |= 2;
        // a page that new tokens fill up
        else if (count > 0 && held * p.page_size > length && !is_page(p, p.tables[r * int64_t(p.width) + held - 1])) bad |= 8;
        if (count < 0) back += held;
        else take += after - held, fresh += count;
    }
    for (int o = 32; o > 0; o >>= 1) {
        back += __shfl_xor(back, o, 64);
        take += __shfl_xor(take, o, 64);
        fresh += __shfl_xor(fresh, o, 64);
        bad |= __shfl_xor(bad, o, 64);
    }
    if ((tid & 63) == 0) {
        if (bad) atomicOr(&s_status, bad);
        atomicAdd(&s_back, static_cast<unsigned long long>(back));
        atomicAdd(&s_take, static_cast<unsigned long long>(take));
        atomicAdd(&s_fresh, static_cast<unsigned long long>(fresh));
    }
    __syncthreads();
    int status = s_status;
    // entries that go back, and how many of them are pages (behind a window none may be left)
    const int64_t entries = int64_t(s_back);
    if (entries > MOST_GIVEN) status |= 8;
    int64_t given = entries;
    if (entries && !status) {
        int own = 0;
        for_given(p, s, own_length, own_count, [&](int i, int32_t entry) {
            own += is_page(p, entry);
            if (i < KEPT_GIVEN) s_entries[i] = entry;
        });
        for (int o = 32; o > 0; o >>= 1) own += __shfl_xor(own, o, 64);
        if ((tid & 63) == 0) atomicAdd(&s_given, own);
        __syncthreads();
        given = s_given;
    }
    const int64_t full = first + given;
    if (first < 0 || full > p.pages) status |= 8;
    else if (int64_t(s_take) > full) status |= 1;
    if (int64_t(s_fresh) > p.capacity) status |= 4;
    if (!status) {
        // what is taken from the stack as it was
        const int taken = int(max(int64_t(s_take) - given, int64_t(0)));
        int wrong = tid < taken && !is_page(p, own_page);
        for (int i = tid + TABLE_THREADS; i < taken; i += TABLE_THREADS) wrong |= !is_page(p, p.free_pages[first - 1 - i]);
        if (__syncthreads_or(wrong)) status = 8;
    }
    if (tid == 0) {
        *p.status = status;
        p.offsets[0] = 0;
        *p.free_out = status ? int32_t(first) : int32_t(full - int64_t(s_take));
    }
    const int total = status ? 0 : int(s_fresh);
    if (status) {
        for (int r = tid; r < p.rows; r += TABLE_THREADS) {
            p.offsets[r + 1] = 0;
            p.lengths_out[r] = p.lengths[r];
        }
    } else {
        // pages given back, on top of the free ones, in row order
        auto for_kept = [&](auto f) {
            if (entries > KEPT_GIVEN) return for_given(p, s, own_length, own_count, f);
            for (int i = tid; i - tid < entries; i += TABLE_THREADS) f(i < entries ? i : INT32_MAX, i < entries ? s_entries[i] : -1);
        };
        if (given == entries) {
            for_kept([&](int i, int32_t entry) {
                if (i < given) p.free_pages[first + i] = entry;
            });
        } else if (given) {
            int before = 0;
            for_kept([&](int, int32_t entry) {
                const int own = is_page(p, entry);
                Scan3 sum;
                const int at = before + block_scan3({own, 0, 0}, s.waves, sum).back - 1;
                if (own) p.free_pages[first + at] = entry;
                before += sum.back;
            });
        }
        if (given) __syncthreads();  // they are on the stack
        // pages taken, lengths and offsets
        Scan3 run = {0, 0, 0}, sum;
        for (int base = 0; base < p.rows; base += TABLE_THREADS) {
            const int r = base + tid;
            int held = 0, length = own_length, count = own_count;
            if (base > 0 && r < p.rows) {
                length = p.lengths[r];
                count = p.counts[r];
            }
            const Scan3 own = r < p.rows ? row_moves(p, length, count, held) : Scan3{0, 0, 0};
            const Scan3 incl = block_scan3(own, s.waves, sum);
            if (sum.take) {
                s.sums[tid] = incl.take;
                s.start[tid] = incl.take - own.take;
                s.held[tid] = held;
                __syncthreads();
                for (int e = tid; e < sum.take; e += TABLE_THREADS) {
                    const int q = first_above(s.sums, TABLE_THREADS, e);
                    p.tables[int64_t(base + q) * p.width + s.held[q] + (e - s.start[q])] = p.free_pages[full - 1 - (run.take + e)];
                }
            }
            if (r < p.rows) {
                const int end = run.fresh + incl.fresh, now = count < 0 ? 0 : length + count;
                p.offsets[r + 1] = end;
                p.lengths_out[r] = now;
                if constexpr (SLOTS) {
                    s_ends[tid] = end;
                    s_lengths[tid] = now;
                }
            }
            run = {0, run.take + sum.take, run.fresh + sum.fresh};
        }
    }
    if constexpr (SLOTS) {
        __syncthreads();
        if (p.rows <= TABLE_THREADS)
            for (int j = tid; j < p.capacity; j += TABLE_THREADS) token_slot(p, s_ends, s_lengths, j, total);
        else
            for (int j = tid; j < p.capacity; j += TABLE_THREADS) token_slot(p, p.offsets + 1, p.lengths_out, j, total);
    }
}

// The search is in LDS where the offsets fit: its steps wait for each other (1,000 requests, 65,536 places 4.6 us in
// memory, 4.1 so).
constexpr int SLOTS_ENDS = 4096;
__global__ __launch_bounds__(256) void paged_slots_kernel(PagedTablesParams p) {
    __shared__ int s_ends[SLOTS_ENDS];
    const int j = int(blockIdx.x * 256 + threadIdx.x);
    if (p.rows <= SLOTS_ENDS) {
#pragma unroll 4
        for (int r = threadIdx.x; r < p.rows; r += 256) s_ends[r] = p.offsets[r + 1];
        __syncthreads();
        if (j < p.capacity) token_slot(p, s_ends, p.lengths_out, j, s_ends[p.rows - 1]);
    } else if (j < p.capacity) {
        token_slot(p, p.offsets + 1, p.lengths_out, j, p.offsets[p.rows]);
    }
}

// ------------------------------------------------------------------------------------ qkv
template <int SOURCE>
__device__ __forceinline__ void load8(const void* base, int64_t at, float (&v)[8]) {
    if constexpr (SOURCE == TYPE_F32) {
        const float4* from = reinterpret_cast<const float4*>(static_cast<const float*>(base) + at);
        const float4 x = from[0], y = from[1];
        v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
        v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
    } else {
        const uint4 x = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + at);
        v[0] = from16<SOURCE>(x.x), v[1] = from16<SOURCE>(x.x >> 16);
        v[2] = from16<SOURCE>(x.y), v[3] = from16<SOURCE>(x.y >> 16);
        v[4] = from16<SOURCE>(x.z), v[5] = from16<SOURCE>(x.z >> 16);
        v[6] = from16<SOURCE>(x.w), v[7] = from16<SOURCE>(x.w >> 16);
    }
}
template <int TYPE>
__device__ __forceinline__ void store8(uint16_t* to, const float (&v)[8]) {
    *reinterpret_cast<uint4*>(to) =
        make_uint4(pack16<TYPE>(v[0], v[1]), pack16<TYPE>(v[2], v[3]), pack16<TYPE>(v[4], v[5]), pack16<TYPE>(v[6], v[7]));
}

// y = x / sqrt(mean(x^2) + 1e-6) (1 + g), (y_i, y_{i + D/2}) turned by the position's angle, rounded
// once.  D / 16 lanes hold a head, each eight dims of its first half and the same eight of its second, so
// that the rotation stays in a lane and BF16 rows move in 16 bytes.  Bound by memory: each element is read
// and written once, 8,192 BF16 rows of 16 + 2 heads of 128 in 15.2 us back to back, 5.0 TB/s (a large copy: 5.2).
template <int SOURCE, int TYPE, int D>
__global__ __launch_bounds__(256) void paged_qkv_kernel(PagedQkvParams p) {
    constexpr int LANES = D / 16;
    const int wide = p.heads + 2 * p.kv_heads;
    const int64_t item = (int64_t(blockIdx.x) * 256 + threadIdx.x) / LANES;
    if (item >= int64_t(p.tokens) * wide) return;  // whole groups of lanes
    const int t = int(item / wide), h = int(item - int64_t(t) * wide), d = int(threadIdx.x % LANES) * 8;
    const int pos = p.positions ? p.positions[t] : 0;
    if (p.rope ? uint32_t(pos) >= uint32_t(p.rope_rows) : pos < 0) return;  // a padding row
    float a[8], b[8];
    const int64_t at = t * p.stride + int64_t(h) * D + d;
    load8<SOURCE>(p.qkv, at, a);
    load8<SOURCE>(p.qkv, at + D / 2, b);
    const bool query = h < p.heads, value = h >= p.heads + p.kv_heads;
    const uint16_t* gain = value ? nullptr : query ? p.q_norm : p.k_norm;
    if (gain) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss += a[i] * a[i] + b[i] * b[i];
        if constexpr (LANES > 8) ss += xor_lane<8>(ss);
        if constexpr (LANES > 4) ss += xor_lane<4>(ss);
        ss += xor_lane<2>(ss);
        ss += xor_lane<1>(ss);
        const float r = 1.0f / sqrtf(ss / float(D) + 1e-6f);
        float ga[8], gb[8];
        load8<TYPE>(gain, d, ga);
        load8<TYPE>(gain, d + D / 2, gb);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            a[i] = a[i] * r * (1.0f + ga[i]);
            b[i] = b[i] * r * (1.0f + gb[i]);
        }
    }
    if (p.rope && !value) {
        const uint4* w = reinterpret_cast<const uint4*>(p.rope + int64_t(pos) * (D / 2) + d);
        const uint4 u = w[0], v = w[1];
        const uint32_t cs[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float c = lo(cs[i]), s = hi(cs[i]), x = a[i], y = b[i];
            a[i] = x * c - y * s;
            b[i] = y * c + x * s;
        }
    }
    uint16_t* to;
    if (query) {
        to = p.q + t * p.q_stride + int64_t(h) * D;
    } else {
        const int slot = p.slots[t];
        const uint32_t page = divide(uint32_t(slot) & 0x7fffffffu, p.div);
        if (slot < 0 || page >= uint32_t(p.pages)) return;
        to = (value ? p.values : p.keys) + int64_t(page) * p.page_stride +
             int64_t(slot - int(page) * p.page_size) * p.slot_stride +
             int64_t(h - p.heads - (value ? p.kv_heads : 0)) * p.head_stride;
    }
    store8<TYPE>(to + d, a);
    store8<TYPE>(to + d + D / 2, b);
}

// ------------------------------------------------------------------------------------ attention
// o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m) over the visible keys of a row, one pass with the
// running maximum and sum.  A wave holds 16 query heads (one per column) and takes 32 keys at a time:
//   S^T = K Q^T   v_mfma_f32_16x16x32 with the keys as rows: lane l gets head l % 16 and the keys
//                 4 (l / 16) + i of both halves of the tile, so the softmax of a head is within four
//                 lanes and its weights are already the operand of the next product;
//   O^T += V^T P^T  the same four keys of both halves are the depth: lane l reads rows of V (whole
//                 lines: 16 lanes side by side) and transposes its 8 keys x 8 dims in registers.
// Nothing passes through LDS until the four waves of a part are joined.  The bound is the pages'
// bytes: 16 heads on one KV head cost 2 x 16 x 128 products for 512 bytes, a fifth of what the matrix
// units do in that time.  Two rows of 131,072 keys on 4 KV heads (537 MB) take 91.3 us, 5.9 TB/s; 128 rows of 33 to
// 16,384 keys on one (177 MB) 36.0 us, 4.9 TB/s: the start, the search for the work and the last part's end are
// in that.  More than 16 heads of a KV head are tiles of 16, which take the pages from memory once and then from the
// L2 (34 heads on 2 KV heads 80 us, 1.3 times the time of the same bytes on 32).
// The weights are kept in two halves of the type (p = hi + lo, 2^-17 off for BF16, 2^-23 for FP16): one
// rounding of them would be as large an error as the output's own, and the second product is hidden by the loads
// (64 rows of 2,000 to 8,000 keys 36.2 us without, 36.3 with).
constexpr int ATTN_WAVES = 4;
constexpr int ATTN_THREADS = ATTN_WAVES * 64;
constexpr int PART_KEYS = 32 * ATTN_WAVES;  // fewest keys of a part: a tile for each wave
// Rows that can see up to so many keys, by the tables' width or the window, are one part each, which saves the
// search for the work and the launch that joins parts: 64 rows of 200 keys 10.3 -> 8.8 us, 256 rows of them 18.8 ->
// 10.7.  Longer where rows and KV heads fill the CUs by themselves (256 rows of 480 keys 24.5 -> 18.5 us), not where
// they do not (64 rows of 480 keys 12.1 in parts, 15 in one).
constexpr int ONE_PART_KEYS = 256, ONE_PART_KEYS_FULL = 512;
// Parts aimed at over all rows and KV heads: as many workgroups as 256 CUs hold at once of the kernel for even pages
// (registers: six of a head of 64, four of 128, two of 256; of the one for uneven pages five, three and two, which
// get the same parts).  More begin when others end and bring more parts to join, fewer leave loads out: two rows of 131,072 keys 112.8 / 87.3 / 101.1 us with 512 / 1,024 / 1,536, a window
// of 2,048 keys in 48 rows of heads of 64 45.3 / 39.6 / 38.0 with 1,024 / 1,536 / 2,048.
constexpr int CUS = 256;
inline int attn_tiles(int heads, int kv_heads) { return (heads / kv_heads + 15) / 16; }
// Twice as many where the rows alone are as many as the CUs hold: parts of more equal lengths (128 rows of 100 to
// 8,000 keys on 8 KV heads 267 -> 205 us, 1,024 on one 234 -> 188; all of 2,000 keys 185 -> 185 and 179 -> 184).
constexpr int FINER = 2;
inline int attn_target(int rows, int heads, int kv_heads, int head_dim) {
    const int held = head_dim <= 64 ? 6 : head_dim <= 128 ? 4 : 2;
    const int64_t tiles = int64_t(kv_heads) * attn_tiles(heads, kv_heads);
    return std::max(1, int(CUS * held * (rows * tiles >= CUS * held ? FINER : 1) / tiles));
}

// How a workgroup finds its part: it is its row; in all rows' lengths; in the list of a launch before.  The second
// takes a time that grows with the rows, for each of as many workgroups: 1,000 rows of 700 keys take 40.6 us so, 41.8
// with the list, 2,048 of 100 keys 29.8 and 23.0, 65,536 4,760 and 581.
enum { DIVISION_NONE, DIVISION_FOUND, DIVISION_LISTED };
constexpr int FOUND_ROWS = 1024;

struct Row {
    int len;    // keys 0 .. len - 1
    int first;  // the first visible one
    int span;   // keys from `first` rounded down to 16 on
};
__device__ __forceinline__ Row row_keys(const PagedAttnParams& p, int r) {
    Row k;
    k.len = min(max(p.lengths[r], 0), p.most);
    k.first = p.window > 0 ? max(0, k.len - p.window) : 0;
    k.span = k.len - (k.first & ~15);
    return k;
}
__device__ __forceinline__ int row_parts(int span, int chunk) { return (span - 1) / chunk + 1; }  // one of none

// Keys of a part: all rows' keys divided by the parts aimed at, in whole tiles for each wave, and a row's at most.
__host__ __device__ constexpr int part_length(long long keys, int aim, int rows, int least, int reach) {
    // a row's last part is half empty on the average
    const int parts = aim - rows / 2 > (aim + 1) / 2 ? aim - rows / 2 : (aim + 1) / 2;
    const long long share = (keys + parts - 1) / parts, each = share < reach ? share : reach;
    return each <= least ? least : int((each + PART_KEYS - 1) / PART_KEYS * PART_KEYS);
}
// a million rows of 2^30 keys, and a share next to 2^31
static_assert(part_length(1LL << 50, 2048, 1 << 20, PART_KEYS, (1 << 30) + 15) == (1 << 30) + PART_KEYS, "32 bits hold it");
static_assert(part_length((1LL << 42) - 1, 2048, 4096, PART_KEYS, (1 << 30) + 15) == (1 << 30) + PART_KEYS, "32 bits hold it");
static_assert(part_length(2 * 131072, 1024, 2, PART_KEYS, 131072 + 15) == 384, "whole tiles");
__device__ __forceinline__ int part_keys(const PagedAttnParams& p, long long keys) {
    return __builtin_amdgcn_readfirstlane(part_length(keys, p.target, p.rows, p.least, p.reach));
}

// Where the workgroups find their work: the same division in all of them, from all rows' lengths.
struct Work {
    int row, first, parts;  // of the part, the row's first part and number of parts
};
struct WorkShared {
    long long keys[ATTN_WAVES];
    int parts[ATTN_WAVES];
    Work found;
};

// The row of part `item`; false past the last part.  The waves look through 64 rows each at a time (1,000 rows
// 71.6 us, 63.4 since they share the work); up to 64 rows every wave does for itself, without waiting for the others.
__device__ __forceinline__ bool find_work(const PagedAttnParams& p, WorkShared& s, int item, Work& work) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool few = p.rows <= 64;
    long long keys = 0;
    for (int r = few ? lane : int(threadIdx.x); r < p.rows; r += ATTN_THREADS) keys += row_keys(p, r).span;
    for (int o = 32; o > 0; o >>= 1) keys += __shfl_xor(keys, o, 64);
    if (!few) {
        if (lane == 0) s.keys[wave] = keys;
        __syncthreads();
        keys = 0;
        for (int w = 0; w < ATTN_WAVES; ++w) keys += s.keys[w];
    }
    const int chunk = part_keys(p, keys);
    int run = 0;
    for (int base = 0; base < p.rows; base += few ? 64 : ATTN_THREADS) {
        const int r = base + (few ? lane : int(threadIdx.x));
        const int own = r < p.rows ? row_parts(row_keys(p, r).span, chunk) : 0;
        const int incl = wave_scan(own), all = __builtin_amdgcn_readlane(incl, 63);
        int before = run;
        if (!few) {
            __syncthreads();  // what the last rows' sums said has been read
            if (lane == 0) s.parts[wave] = all;
            __syncthreads();
            for (int w = 0; w < ATTN_WAVES; ++w) {
                before += w < wave ? s.parts[w] : 0;
                run += s.parts[w];
            }
        } else {
            run += all;
        }
        if (item < run) {
            const unsigned long long past = __ballot(before + incl > item && before <= item);
            Work here = {0, 0, 0};
            if (past) {
                const int l = __ffsll(past) - 1;
                here = {__builtin_amdgcn_readlane(r, l), 0, __builtin_amdgcn_readlane(own, l)};
                here.first = before + __builtin_amdgcn_readlane(incl, l) - here.parts;
            }
            if (few) {
                work = here;
                return true;
            }
            if (past && lane == 0) s.found = here;
            __syncthreads();
            work = {__builtin_amdgcn_readfirstlane(s.found.row), __builtin_amdgcn_readfirstlane(s.found.first),
                    __builtin_amdgcn_readfirstlane(s.found.parts)};
            return true;
        }
    }
    return false;
}

// The same where paged_parts_kernel has been: the last row whose first part is not past `item`, by looking at
// 64 rows of a range at a time.
__device__ __forceinline__ bool look_up_work(const PagedAttnParams& p, int item, Work& work) {
    const int lane = threadIdx.x & 63;
    int row = 0, span = p.rows;
    while (span > 1) {
        const int step = (span + 63) / 64, at = row + lane * step;
        const bool upto = lane * step < span && at < p.rows && p.row_parts[at].x <= item;  // true for the first lanes
        row += (__popcll(__ballot(upto)) - 1) * step;
        span = step;
    }
    row = __builtin_amdgcn_readfirstlane(row);
    const int2 parts = p.row_parts[row];
    work = {row, __builtin_amdgcn_readfirstlane(parts.x), __builtin_amdgcn_readfirstlane(parts.y)};
    return item < work.first + work.parts;
}

// First part and number of parts of every row, by one workgroup.
constexpr int DIVIDE_THREADS = 1024;
__global__ __launch_bounds__(DIVIDE_THREADS) void paged_parts_kernel(PagedAttnParams p) {
    constexpr int WAVES = DIVIDE_THREADS / 64;
    __shared__ long long s_keys[WAVES];
    __shared__ int s_parts[WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    long long keys = 0;
#pragma unroll 4
    for (int r = threadIdx.x; r < p.rows; r += DIVIDE_THREADS) keys += row_keys(p, r).span;
    for (int o = 32; o > 0; o >>= 1) keys += __shfl_xor(keys, o, 64);
    if (lane == 0) s_keys[wave] = keys;
    __syncthreads();
    keys = 0;
    for (int w = 0; w < WAVES; ++w) keys += s_keys[w];
    const int chunk = part_keys(p, keys);
    // a thread's rows are neighbours: sums in order
    const int each = (p.rows + DIVIDE_THREADS - 1) / DIVIDE_THREADS;
    const int begin = min(int(threadIdx.x) * each, p.rows), end = min(begin + each, p.rows);
    int own = 0;
#pragma unroll 4
    for (int r = begin; r < end; ++r) own += row_parts(row_keys(p, r).span, chunk);
    const int incl = wave_scan(own);
    if (lane == 63) s_parts[wave] = incl;
    __syncthreads();
    int first = incl - own;
    for (int w = 0; w < wave; ++w) first += s_parts[w];
#pragma unroll 4
    for (int r = begin; r < end; ++r) {
        const int parts = row_parts(row_keys(p, r).span, chunk);
        p.row_parts[r] = make_int2(first, parts);
        first += parts;
    }
}

template <int TYPE>
__device__ __forceinline__ floatx4 mfma16(uint4 a, uint4 b, floatx4 c) {
    if constexpr (TYPE == TYPE_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// FP16 weights are held times 2^12: their smallest normal value is then 2^-26 of the largest weight's.
template <int TYPE>
constexpr float weight_shift() { return TYPE == TYPE_F16 ? 12.0f : 0.0f; }

template <int TYPE, int D>
struct Tile {
    static constexpr int STEPS = D / 32;             // products over a head's dims
    static constexpr int CHUNK = D < 128 ? D / 16 : 8;  // dims of V that a lane takes of a key, at once
    static constexpr int SLABS = D < 128 ? 1 : D / 128;
    uint4 k[2][STEPS];
    uint32_t v[8][SLABS][CHUNK / 2];
    uint32_t seen;  // bit i: key 4 (l / 16) + i % 4 of half i / 4 is visible
    bool whole;     // all keys of the tile are
};

// Reads of the pages.  Where a part is one workgroup's they are read once, so not to stay in the caches (nt: two
// rows of 131,072 keys 98.6 -> 88.2 us, 128 ragged rows 41.7 -> 36.8), and issued where they stand (volatile).  Where
// it is several tiles of heads' (SHARED), these are side by side on one XCD and the second finds them in
// its L2: 64 rows of 2,000 to 8,000 keys and 32 heads on one KV head 62.6 -> 49.1 us, 64 heads 109 -> 69.
template <bool SHARED>
__device__ __forceinline__ uint4 read16(__amdgpu_buffer_rsrc_t r, uint32_t off) {
    const u32x4_t v = __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, SHARED ? 0 : int(0x80000002u));
    return make_uint4(v[0], v[1], v[2], v[3]);
}
template <bool SHARED>
__device__ __forceinline__ uint2 read8(__amdgpu_buffer_rsrc_t r, uint32_t off) {
    const u32x2_t v = __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, SHARED ? 0 : int(0x80000002u));
    return make_uint2(v[0], v[1]);
}
template <bool SHARED>
__device__ __forceinline__ uint4 read16(const char* at) {
    const u32x4_t* from = reinterpret_cast<const u32x4_t*>(at);
    const u32x4_t v = SHARED ? *from : __builtin_nontemporal_load(from);
    return make_uint4(v[0], v[1], v[2], v[3]);
}
template <bool SHARED>
__device__ __forceinline__ uint2 read8(const char* at) {
    const u32x2_t* from = reinterpret_cast<const u32x2_t*>(at);
    const u32x2_t v = SHARED ? *from : __builtin_nontemporal_load(from);
    return make_uint2(v[0], v[1]);
}

// EVEN: pages of whole half tiles (a multiple of 16 tokens), so that a half tile is one page's and
// its page and addresses are the wave's, not the lane's.  64 rows of 5,000 keys from memory take 42.1 us so, 43.6 the
// other way, which any page size allows; 48 of a window of 2,048, 32 heads of 64 on 8, 44.7 and 48.8.
template <int TYPE, int D, bool EVEN, bool SHARED>
__device__ __forceinline__ void load_tile(Tile<TYPE, D>& t, const PagedAttnParams& p, const int32_t* table,
                                          int64_t head, int pos, int lo_key, int hi_key) {
    typedef Tile<TYPE, D> X;
    const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
    t.whole = pos >= lo_key && pos + 32 <= hi_key;
    t.seen = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int j = pos + 16 * (i >> 2) + 4 * g + (i & 3);
        t.seen |= uint32_t(j >= lo_key && j < hi_key) << i;
    }
    if constexpr (EVEN) {
        __amdgpu_buffer_rsrc_t kr[2], vr[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            // a half past the last key, or of a page that is none, reads nothing: its view is empty
            const int at = pos + 16 * h;
            int page = -1;
            const uint32_t index = divide(uint32_t(at), p.div);
            if (at < hi_key) page = table[index];
            const bool there = uint32_t(page) < uint32_t(p.pages);
            if (at < hi_key && !there) {
                t.whole = false;
                t.seen &= ~(0xfu << (4 * h));
            }
            const int64_t off = there ? page * p.page_stride + (at - int(index) * p.page_size) * p.slot_stride + head : 0;
            const uint32_t bytes = there ? uint32_t(15 * p.slot_stride + D * 2) : 0u;
            kr[h] = buffer_view(p.keys + off, bytes);
            vr[h] = buffer_view(p.values + off, bytes);
        }
        const uint32_t ks = uint32_t(col * int(p.slot_stride) + g * 16);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int s = 0; s < X::STEPS; ++s) t.k[h][s] = read16<SHARED>(kr[h], ks + s * 64);
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int s = 0; s < X::SLABS; ++s) {
                const uint32_t at = uint32_t((4 * g + (i & 3)) * int(p.slot_stride) + col * X::CHUNK * 2 + s * 256);
                if constexpr (X::CHUNK == 8) {
                    const uint4 w = read16<SHARED>(vr[i >> 2], at);
                    t.v[i][s][0] = w.x, t.v[i][s][1] = w.y, t.v[i][s][2] = w.z, t.v[i][s][3] = w.w;
                } else {
                    const uint2 w = read8<SHARED>(vr[i >> 2], at);
                    t.v[i][s][0] = w.x, t.v[i][s][1] = w.y;
                }
            }
    } else {
        // lane j looks key j of the tile up, for all lanes that read it; -1: not seen
        const int key = pos + (lane & 31);
        int64_t own = -1;
        if (key >= lo_key && key < hi_key) {
            const uint32_t index = divide(uint32_t(key), p.div);
            const int page = table[index];
            if (uint32_t(page) < uint32_t(p.pages))
                own = page * p.page_stride + (key - int(index) * p.page_size) * p.slot_stride + head;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int64_t off = __shfl(own, 16 * h + col, 64);
#pragma unroll
            for (int s = 0; s < X::STEPS; ++s)
                t.k[h][s] = off >= 0 ? read16<SHARED>(p.keys + off + g * 16 + s * 64) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t off = __shfl(own, 16 * (i >> 2) + 4 * g + (i & 3), 64);
            if (off < 0) t.seen &= ~(1u << i);
#pragma unroll
            for (int s = 0; s < X::SLABS; ++s) {
                const char* from = p.values + off + col * X::CHUNK * 2 + s * 256;
                if constexpr (X::CHUNK == 8) {
                    const uint4 x = off >= 0 ? read16<SHARED>(from) : make_uint4(0, 0, 0, 0);
                    t.v[i][s][0] = x.x, t.v[i][s][1] = x.y, t.v[i][s][2] = x.z, t.v[i][s][3] = x.w;
                } else {
                    const uint2 x = off >= 0 ? read8<SHARED>(from) : make_uint2(0, 0);
                    t.v[i][s][0] = x.x, t.v[i][s][1] = x.y;
                }
            }
        }
        t.whole = __all(t.seen == 0xffu);
    }
}

template <int TYPE, int D>
struct Running {
    typedef Tile<TYPE, D> X;
    float m = NEG_INF, l = 0.f;               // of the lane's head; l over the lane's own keys
    floatx4 o[X::SLABS][X::CHUNK];            // dims slab * 128 + (4 (l / 16) + i) CHUNK + j
};

template <int TYPE, int D>
__device__ __forceinline__ void take_tile(Running<TYPE, D>& run, Tile<TYPE, D>& t, const uint4 (&q)[D / 32], float scale) {
    typedef Tile<TYPE, D> X;
    floatx4 s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int c = 0; c < X::STEPS; ++c) {
        s[0] = mfma16<TYPE>(t.k[0][c], q[c], s[0]);
        s[1] = mfma16<TYPE>(t.k[1][c], q[c], s[1]);
    }
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = s[i >> 2][i & 3] * scale;
    if (!t.whole) {
        // what a hidden key's row holds (NaN among it) reaches neither the scores nor the sums
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const bool seen = (t.seen >> i) & 1u;
            x[i] = seen ? x[i] : NEG_INF;
#pragma unroll
            for (int b = 0; b < X::SLABS; ++b)
#pragma unroll
                for (int w = 0; w < X::CHUNK / 2; ++w) t.v[i][b][w] = seen ? t.v[i][b][w] : 0u;
        }
    }
    float most = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) most = fmaxf(most, x[i]);
    most = fmaxf(most, xor_lane<16>(most));
    most = fmaxf(most, xor_lane<32>(most));
    const float before = run.m;
    run.m = fmaxf(before, most);
    // exponents are taken from `from`: the maximum, or any number while that is minus infinity
    const float from = (run.m == NEG_INF ? 0.f : run.m) - weight_shift<TYPE>();
    if (__any(run.m > before)) {
        const float shrink = __builtin_amdgcn_exp2f(before - weight_shift<TYPE>() - from);
        run.l *= shrink;
#pragma unroll
        for (int b = 0; b < X::SLABS; ++b)
#pragma unroll
            for (int j = 0; j < X::CHUNK; ++j) run.o[b][j] *= shrink;
    }
    float e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        e[i] = __builtin_amdgcn_exp2f(x[i] - from);
        run.l += e[i];
    }
    uint32_t high[4], low[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        high[i] = pack16<TYPE>(e[2 * i], e[2 * i + 1]);
        low[i] = pack16<TYPE>(e[2 * i] - from16<TYPE>(high[i]), e[2 * i + 1] - from16<TYPE>(high[i] >> 16));
    }
    const uint4 ph = make_uint4(high[0], high[1], high[2], high[3]), pl = make_uint4(low[0], low[1], low[2], low[3]);
#pragma unroll
    for (int b = 0; b < X::SLABS; ++b)
#pragma unroll
        for (int j = 0; j < X::CHUNK; ++j) {
            // dim j of the lane's eight keys, two keys a word
            const uint32_t pick = j & 1 ? 0x07060302u : 0x05040100u;
            uint32_t a[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) a[i] = __builtin_amdgcn_perm(t.v[2 * i + 1][b][j >> 1], t.v[2 * i][b][j >> 1], pick);
            const uint4 column = make_uint4(a[0], a[1], a[2], a[3]);
            run.o[b][j] = mfma16<TYPE>(column, ph, run.o[b][j]);
            run.o[b][j] = mfma16<TYPE>(column, pl, run.o[b][j]);
        }
}

// Waves of a SIMD whose registers hold them (uneven pages hold 64-bit addresses too).
constexpr int attn_waves(int head_dim, bool even) { return head_dim == 64 ? (even ? 6 : 5) : head_dim == 128 ? (even ? 4 : 3) : 2; }

template <int TYPE, int D, bool EVEN, bool SHARED>
__global__ __launch_bounds__(ATTN_THREADS, attn_waves(D, EVEN)) void paged_attention_kernel(PagedAttnParams p) {
    typedef Tile<TYPE, D> X;
    constexpr int PITCH = D + 4;
    __shared__ __align__(16) float s_o[ATTN_WAVES][16][PITCH];
    __shared__ float s_m[ATTN_WAVES][16], s_l[ATTN_WAVES][16];
    __shared__ WorkShared s_work;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    // workgroups go to the eight XCDs in turn: eight parts' first tiles, their second ones, ...
    const int kv = blockIdx.y;
    int item = blockIdx.x, tile = 0;
    if constexpr (SHARED) {
        const int eight = int(blockIdx.x) / (8 * p.tiles), rest = int(blockIdx.x) - eight * 8 * p.tiles;
        item = eight * 8 + (rest & 7);
        tile = rest >> 3;
    }
    Work work;
    bool any = true;
    if (p.division == DIVISION_NONE) {
        work = {item, item, 1};
        any = !SHARED || item < p.rows;
    } else if (p.division == DIVISION_LISTED) {
        any = look_up_work(p, item, work);
    } else {
        any = find_work(p, s_work, item, work);
    }
    if (!any) return;  // every wave of the workgroup
    const int row = __builtin_amdgcn_readfirstlane(work.row), first_part = __builtin_amdgcn_readfirstlane(work.first),
              parts = __builtin_amdgcn_readfirstlane(work.parts);
    const Row keys = row_keys(p, row);
    const int len = __builtin_amdgcn_readfirstlane(keys.len), first = __builtin_amdgcn_readfirstlane(keys.first);
    const int part = item - first_part;
    const int each = __builtin_amdgcn_readfirstlane(((len - (first & ~15) + parts - 1) / parts + 31) & ~31);
    const int begin = (first & ~15) + part * each, end = min(len, begin + each);
    const int heads = p.kv_heads * p.group, head0 = kv * p.group + tile * 16, live = min(16, p.group - tile * 16);
    if (p.division == DIVISION_FOUND && blockIdx.y == 0 && tile == 0 && threadIdx.x == 0 && part == 0) p.row_parts[row] = make_int2(first_part, parts);

    uint4 q[X::STEPS];
    const uint16_t* qrow = p.q + row * p.q_stride + int64_t(head0 + min(col, live - 1)) * D;
#pragma unroll
    for (int c = 0; c < X::STEPS; ++c) q[c] = *reinterpret_cast<const uint4*>(qrow + c * 32 + g * 8);

    const int32_t* table = p.tables + int64_t(row) * p.width;
    const int64_t head = kv * p.head_stride;
    Running<TYPE, D> run;
#pragma unroll
    for (int b = 0; b < X::SLABS; ++b)
#pragma unroll
        for (int j = 0; j < X::CHUNK; ++j) run.o[b][j] = floatx4{0.f, 0.f, 0.f, 0.f};
    for (int pos = begin + 32 * wave; pos < end; pos += PART_KEYS) {
        Tile<TYPE, D> t;
        load_tile<TYPE, D, EVEN, SHARED>(t, p, table, head, pos, first, end);
        take_tile<TYPE, D>(run, t, q, p.scale);
    }
    run.l += xor_lane<16>(run.l);
    run.l += xor_lane<32>(run.l);

    // the four waves joined
    if (lane < 16) s_m[wave][lane] = run.m;
    __syncthreads();
    float most = s_m[0][col];
#pragma unroll
    for (int w = 1; w < ATTN_WAVES; ++w) most = fmaxf(most, s_m[w][col]);
    const float share = run.m == NEG_INF ? 0.f : __builtin_amdgcn_exp2f(run.m - most);
    if (lane < 16) s_l[wave][lane] = run.l * share;
#pragma unroll
    for (int b = 0; b < X::SLABS; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < X::CHUNK; j += 4) {
                const float4 v = make_float4(run.o[b][j][i] * share, run.o[b][j + 1][i] * share, run.o[b][j + 2][i] * share,
                                             run.o[b][j + 3][i] * share);
                *reinterpret_cast<float4*>(&s_o[wave][col][b * 128 + (4 * g + i) * X::CHUNK + j]) = v;
            }
    __syncthreads();
    for (int e = threadIdx.x; e < live * (D / 4); e += ATTN_THREADS) {
        const int h = e / (D / 4), d = (e - h * (D / 4)) * 4;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        float l = 0.f;
#pragma unroll
        for (int w = 0; w < ATTN_WAVES; ++w) {
            const float4 v = *reinterpret_cast<const float4*>(&s_o[w][h][d]);
            sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
            l += s_l[w][h];
        }
        float m = s_m[0][h];
#pragma unroll
        for (int w = 1; w < ATTN_WAVES; ++w) m = fmaxf(m, s_m[w][h]);
        if (parts == 1) {
            // nothing visible: zeros
            const float r = l == 0.f ? 0.f : 1.0f / l;
            *reinterpret_cast<uint2*>(p.out + row * p.out_stride + int64_t(head0 + h) * D + d) =
                make_uint2(pack16<TYPE>(sum.x * r, sum.y * r), pack16<TYPE>(sum.z * r, sum.w * r));
            if (p.lse && d == 0)
                p.lse[int64_t(row) * heads + head0 + h] =
                    l == 0.f ? NEG_INF : (m - weight_shift<TYPE>() + log2f(l)) * 0.69314718055994531f;
        } else {
            const int64_t at = int64_t(item) * heads + head0 + h;
            *reinterpret_cast<float4*>(p.part_o + at * D + d) = sum;
            if (d == 0) p.part_ml[at] = make_float2(m, l);
        }
    }
}

// HEADS heads of a row from their parts, in a fixed order: D / 4 lanes hold a head's dims, its groups of
// lanes take every GROUPS-th part, eight parts' loads at once, with a running maximum; the groups are joined
// in LDS.  Bound by latency: the row's parts, then the parts themselves (2.4 to 5.8 us).
constexpr int MERGE_THREADS = 512;

template <int TYPE, int D, int HEADS>
__global__ __launch_bounds__(MERGE_THREADS) void paged_merge_kernel(PagedAttnParams p) {
    constexpr int LANES = D / 4, GROUPS = MERGE_THREADS / (LANES * HEADS), AHEAD = 8;
    __shared__ __align__(16) float s_o[HEADS][GROUPS][D];
    __shared__ float s_m[HEADS][GROUPS], s_l[HEADS][GROUPS];
    const int row = blockIdx.x, heads = p.kv_heads * p.group;
    const int2 parts = p.row_parts[row];
    if (parts.y == 1) return;
    const int sub = threadIdx.x / (MERGE_THREADS / HEADS), tid = threadIdx.x - sub * (MERGE_THREADS / HEADS);
    const int group = tid / LANES, d = (tid % LANES) * 4;
    const int h = blockIdx.y * HEADS + sub;
    const bool live_head = h < heads;
    const int64_t first = int64_t(parts.x) * heads + h;
    float m = NEG_INF, l = 0.f;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = live_head ? group : parts.y; i < parts.y; i += GROUPS * AHEAD) {
        float2 ml[AHEAD];
        float4 o[AHEAD];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            const int64_t at = first + int64_t(min(i + a * GROUPS, parts.y - 1)) * heads;
            ml[a] = p.part_ml[at];
            o[a] = *reinterpret_cast<const float4*>(p.part_o + at * D + d);
        }
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            if (i + a * GROUPS >= parts.y) break;
            const float most = fmaxf(m, ml[a].x), from = most == NEG_INF ? 0.f : most;
            const float keep = __builtin_amdgcn_exp2f(m - from), share = __builtin_amdgcn_exp2f(ml[a].x - from);
            m = most;
            l = l * keep + ml[a].y * share;
            sum.x = sum.x * keep + o[a].x * share, sum.y = sum.y * keep + o[a].y * share;
            sum.z = sum.z * keep + o[a].z * share, sum.w = sum.w * keep + o[a].w * share;
        }
    }
    *reinterpret_cast<float4*>(&s_o[sub][group][d]) = sum;
    if (d == 0) {
        s_m[sub][group] = m;
        s_l[sub][group] = l;
    }
    __syncthreads();
    if (tid < LANES && live_head) {
        const int live = min(GROUPS, parts.y);
        for (int k = 0; k < live; ++k) m = fmaxf(m, s_m[sub][k]);
        const float from = m == NEG_INF ? 0.f : m;
        l = 0.f;
        sum = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int k = 0; k < live; ++k) {
            const float share = __builtin_amdgcn_exp2f(s_m[sub][k] - from);
            const float4 v = *reinterpret_cast<const float4*>(&s_o[sub][k][d]);
            l += s_l[sub][k] * share;
            sum.x += v.x * share, sum.y += v.y * share, sum.z += v.z * share, sum.w += v.w * share;
        }
        const float r = l == 0.f ? 0.f : 1.0f / l;
        *reinterpret_cast<uint2*>(p.out + row * p.out_stride + int64_t(h) * D + d) =
            make_uint2(pack16<TYPE>(sum.x * r, sum.y * r), pack16<TYPE>(sum.z * r, sum.w * r));
        if (p.lse && tid == 0)
            p.lse[int64_t(row) * heads + h] = l == 0.f ? NEG_INF : (m - weight_shift<TYPE>() + log2f(l)) * 0.69314718055994531f;
    }
}

// Workgroups of a KV head.
int64_t attn_workgroups(const PagedAttnParams& p) {
    // parts: at most one more than its share of the aimed ones for each row, and none of less than p.least but a
    // row's only one
    const int64_t most = int64_t(p.rows) * std::max<int64_t>(1, (int64_t(p.reach) + p.least - 1) / p.least);
    const int64_t parts = std::min<int64_t>(most, int64_t(p.rows) + p.target);
    return p.tiles > 1 ? (parts + 7) / 8 * 8 * p.tiles : parts;
}

template <int TYPE, int D>
void run_attention(const PagedAttnParams& p, hipStream_t s) {
    const bool shared = p.tiles > 1;
    // parts beside each other, KV heads one after the other: the other way two rows of 131,072 keys on 4 KV heads take
    // 105 us for 91
    const dim3 grid(unsigned(attn_workgroups(p)), unsigned(p.kv_heads));
    if (p.division == DIVISION_LISTED) hipLaunchKernelGGL(paged_parts_kernel, dim3(1), dim3(DIVIDE_THREADS), 0, s, p);
    const bool even = p.page_size % 16 == 0;
    if (even && shared) hipLaunchKernelGGL((paged_attention_kernel<TYPE, D, true, true>), grid, dim3(ATTN_THREADS), 0, s, p);
    else if (even) hipLaunchKernelGGL((paged_attention_kernel<TYPE, D, true, false>), grid, dim3(ATTN_THREADS), 0, s, p);
    else if (shared) hipLaunchKernelGGL((paged_attention_kernel<TYPE, D, false, true>), grid, dim3(ATTN_THREADS), 0, s, p);
    else hipLaunchKernelGGL((paged_attention_kernel<TYPE, D, false, false>), grid, dim3(ATTN_THREADS), 0, s, p);
    if (p.division != DIVISION_NONE) {
        // few rows have many parts each, many rows few: most of their workgroups would find nothing to join (128 rows
        // of 16 heads 5.8 us with a head a workgroup, 6.9 with four; 1,000 rows, attention and all, 81.2 and 71.6)
        const int heads = p.kv_heads * p.group;
        if (int64_t(p.rows) * heads <= 4096)
            hipLaunchKernelGGL((paged_merge_kernel<TYPE, D, 1>), dim3(unsigned(p.rows), unsigned(heads)), dim3(MERGE_THREADS), 0, s, p);
        else
            hipLaunchKernelGGL((paged_merge_kernel<TYPE, D, 4>), dim3(unsigned(p.rows), unsigned((heads + 3) / 4)),
                               dim3(MERGE_THREADS), 0, s, p);
    }
}

template <int SOURCE, int TYPE>
void run_qkv(const PagedQkvParams& p, int head_dim, hipStream_t s) {
    const int64_t threads = int64_t(p.tokens) * (p.heads + 2 * p.kv_heads) * (head_dim / 16);
    const dim3 grid(unsigned((threads + 255) / 256));
    if (head_dim == 64) hipLaunchKernelGGL((paged_qkv_kernel<SOURCE, TYPE, 64>), grid, dim3(256), 0, s, p);
    else if (head_dim == 128) hipLaunchKernelGGL((paged_qkv_kernel<SOURCE, TYPE, 128>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((paged_qkv_kernel<SOURCE, TYPE, 256>), grid, dim3(256), 0, s, p);
}

}  // namespace

void launch_paged_tables(const PagedTablesParams& p, hipStream_t s) {
    if (p.capacity <= SLOTS_IN_TABLES) {
        hipLaunchKernelGGL((paged_tables_kernel<true>), dim3(1), dim3(TABLE_THREADS), 0, s, p);
        return;
    }
    hipLaunchKernelGGL((paged_tables_kernel<false>), dim3(1), dim3(TABLE_THREADS), 0, s, p);
    hipLaunchKernelGGL(paged_slots_kernel, dim3(unsigned((p.capacity + 255) / 256)), dim3(256), 0, s, p);
}

void launch_paged_qkv(const PagedQkvParams& p, int source, int type, int head_dim, hipStream_t s) {
    if (p.tokens == 0) return;
    if (type == TYPE_BF16) {
        if (source == TYPE_F32) run_qkv<TYPE_F32, TYPE_BF16>(p, head_dim, s);
        else run_qkv<TYPE_BF16, TYPE_BF16>(p, head_dim, s);
    } else {
        if (source == TYPE_F32) run_qkv<TYPE_F32, TYPE_F16>(p, head_dim, s);
        else run_qkv<TYPE_F16, TYPE_F16>(p, head_dim, s);
    }
}

size_t paged_attn_workspace(int rows, int heads, int kv_heads, int head_dim) {
    const size_t parts = size_t(rows) + size_t(attn_target(rows, heads, kv_heads, head_dim));
    const size_t lists = (size_t(rows) * sizeof(int2) + 15) / 16 * 16 + (parts * size_t(heads) * sizeof(float2) + 15) / 16 * 16;
    return lists + parts * size_t(heads) * size_t(head_dim) * sizeof(float);
}

void paged_attn_bind(PagedAttnParams& p, void* workspace, int head_dim) {
    const int heads = p.kv_heads * p.group;
    p.tiles = attn_tiles(heads, p.kv_heads);
    p.target = attn_target(p.rows, heads, p.kv_heads, head_dim);
    const int one_part = int64_t(p.rows) * p.kv_heads * p.tiles >= CUS ? ONE_PART_KEYS_FULL : ONE_PART_KEYS;
    p.reach = (p.window > 0 ? std::min(p.window, p.most) : p.most) + 15;
    p.least = p.reach <= one_part ? one_part : PART_KEYS;
    p.division = p.reach <= p.least ? DIVISION_NONE : p.rows <= FOUND_ROWS ? DIVISION_FOUND : DIVISION_LISTED;
    const size_t parts = size_t(p.rows) + size_t(p.target);
    char* at = static_cast<char*>(workspace);
    p.row_parts = reinterpret_cast<int2*>(at);
    at += (size_t(p.rows) * sizeof(int2) + 15) / 16 * 16;
    p.part_ml = reinterpret_cast<float2*>(at);
    at += (parts * size_t(heads) * sizeof(float2) + 15) / 16 * 16;
    p.part_o = reinterpret_cast<float*>(at);
}

bool paged_attn_launches(const PagedAttnParams& p) { return attn_workgroups(p) * ATTN_THREADS <= UINT32_MAX; }

void launch_paged_attention(const PagedAttnParams& p, int type, int head_dim, hipStream_t s) {
    if (type == TYPE_BF16) {
        if (head_dim == 64) run_attention<TYPE_BF16, 64>(p, s);
        else if (head_dim == 128) run_attention<TYPE_BF16, 128>(p, s);
        else run_attention<TYPE_BF16, 256>(p, s);
    } else {
        if (head_dim == 64) run_attention<TYPE_F16, 64>(p, s);
        else if (head_dim == 128) run_attention<TYPE_F16, 128>(p, s);
        else run_attention<TYPE_F16, 256>(p, s);
    }
}

}  // namespace plamo
