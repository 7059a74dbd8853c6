// A speculative step over paged caches on gfx950: what surrounds the attention of drafted tokens.
//
//   tree_wave_kernel, tree_block_kernel   positions and ancestors of the trees' nodes
//   accept_walk_kernel                    the path that the drawn tokens agree with, its moves
//   accept_pages_kernel                   lengths cut, pages given back
//   move_kernel                           keys and values from slot to slot, in all layers
//   controls_kernel                       penalties, n-grams, biases and masks on logits
#include <hip/hip_runtime.h>

#include <algorithm>

#include "common.h"
#include "paged_device.h"
#include "speculate.h"

namespace plamo {
using namespace dev;

namespace {

// A request's new tokens, none where its offsets are no ascending numbers of 0 .. most.
struct Span {
    int first, count;
};
__device__ __forceinline__ Span new_tokens(const int32_t* offsets, int r, int most) {
    const int first = offsets[r], end = offsets[r + 1];
    const bool fine = first >= 0 && end >= first && end <= most;
    return {fine ? first : 0, fine ? end - first : 0};
}

// ------------------------------------------------------------------------------------ trees
// Node i's bits are its parent's and its own.  All nodes at once, by doubling: after step k a node's bits hold the
// 2^k nodes up from it, and its link is the node 2^k up, so that ceil(log2(depth)) steps do.  Parents come before their
// children, so a path's nodes are in the order of their depth, which is the number of bits less one, and a window
// keeps the highest bits.  Latency-bound: some dependent loads, shuffles and barriers (64 requests of 8 nodes 2.6 us).
constexpr int WAVE_THREADS = 256;

// Tokens behind the last request's.
__device__ __forceinline__ void pad_tokens(const TreeParams& p, int block, int blocks, int threads) {
    const int last = max(0, p.offsets[p.rows]);
    for (int64_t t = last + int64_t(block) * threads + threadIdx.x; t < p.tokens; t += int64_t(blocks) * threads) {
        p.positions[t] = -1;
        for (int w = 0; w < p.words; ++w) p.ancestors[t * p.words + w] = 0;
    }
}

// What a request's tokens get that do not fit its bits, or that its length does not hold.
__device__ __forceinline__ void no_tree(const TreeParams& p, Span s, int lane, int lanes) {
    for (int i = lane; i < s.count; i += lanes) {
        p.positions[s.first + i] = -1;
        for (int w = 0; w < p.words; ++w) p.ancestors[int64_t(s.first + i) * p.words + w] = 0;
    }
}

// Among the 64 nodes from `base` on, a node a lane, links followed by shuffles: bits of these nodes alone, and the link is
// the first ancestor before them, or none.
__device__ __forceinline__ void wave_tree(int base, int& up, uint32_t& low, uint32_t& high) {
    const int lane = threadIdx.x & 63;
    low = lane < 32 ? 1u << lane : 0u;
    high = lane < 32 ? 0u : 1u << (lane - 32);
    while (__any(up >= base)) {
        const int at = max(up - base, 0);
        const uint32_t l = __shfl(low, at, 64), h = __shfl(high, at, 64);
        const int next = __shfl(up, at, 64);
        if (up >= base) {
            low |= l;
            high |= h;
            up = next;
        }
    }
}

// Up to 64 nodes: a wave a request.
__global__ __launch_bounds__(WAVE_THREADS) void tree_wave_kernel(TreeParams p) {
    const int lane = threadIdx.x & 63, r = int(blockIdx.x) * (WAVE_THREADS / 64) + int(threadIdx.x >> 6);
    pad_tokens(p, blockIdx.x, gridDim.x, WAVE_THREADS);
    if (r >= p.rows) return;
    const Span s = new_tokens(p.offsets, r, p.tokens);
    const int length = p.lengths[r], start = length - s.count;
    if (s.count > 32 * p.words || length < s.count) return no_tree(p, s, lane, 64);
    int up = lane < s.count ? p.parents[s.first + lane] : -1;
    up = up >= 0 && up < lane ? up : -1;
    uint32_t low, high;
    wave_tree(0, up, low, high);
    if (lane >= s.count) return;
    uint64_t bits = uint64_t(high) << 32 | low;
    const int depth = __popcll(bits) - 1;
    if (p.window > 0)
        for (int drop = depth + 1 - p.window; drop > 0; --drop) bits &= bits - 1;
    const int64_t t = s.first + lane;
    p.positions[t] = start + depth;
    p.ancestors[t * p.words] = uint32_t(bits);
    if (p.words > 1) p.ancestors[t * p.words + 1] = uint32_t(bits >> 32);
}

// More: a workgroup a request.  After each wave's own 64 nodes a link leads to an earlier wave's, so that a path has few of
// them, and rows of words in LDS are doubled that few times (200 requests of 60 nodes, or of a chain of 500, in 16 words: all
// steps on rows in LDS 18.7 us, so 11.3).
template <int W>
__global__ __launch_bounds__(32 * W) void tree_block_kernel(TreeParams p) {
    constexpr int NODES = 32 * W, PITCH = W + 1;  // banks: a row's words in those of its neighbours, one further
    __shared__ uint32_t s_bits[NODES * PITCH];
    __shared__ int s_up[NODES];
    const int i = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    pad_tokens(p, blockIdx.x, gridDim.x, NODES);
    const Span s = new_tokens(p.offsets, blockIdx.x, p.tokens);
    const int length = p.lengths[blockIdx.x], start = length - s.count;
    if (s.count > 32 * p.words || length < s.count) return no_tree(p, s, i, NODES);
    int up = i < s.count ? p.parents[s.first + i] : -1;
    up = up >= 0 && up < i ? up : -1;
    uint32_t bits[W], low, high;
    wave_tree(64 * wave, up, low, high);
#pragma unroll
    for (int w = 0; w < W; ++w) bits[w] = w == 2 * wave ? low : w == 2 * wave + 1 ? high : 0u;
    bool changed = true;
    while (__syncthreads_or(up >= 0)) {  // what the step before read has been read
        s_up[i] = up;
        if (changed) {
#pragma unroll
            for (int w = 0; w < W; ++w)
                if (w < 2 * wave + 2) s_bits[i * PITCH + w] = bits[w];
        }
        __syncthreads();
        changed = __any(up >= 0);
        if (up >= 0) {
#pragma unroll
            for (int w = 0; w < W; ++w)
                if (w < 2 * wave) bits[w] |= w < 2 * (up >> 6) + 2 ? s_bits[up * PITCH + w] : 0u;
            up = s_up[up];
        }
    }
    int depth = -1;
#pragma unroll
    for (int w = 0; w < W; ++w) depth += __popc(bits[w]);
    if (p.window > 0) {
        int drop = depth + 1 - p.window;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const int own = __popc(bits[w]);
            if (drop >= own) {
                bits[w] = 0;
            } else {
                for (int k = drop; k > 0; --k) bits[w] &= bits[w] - 1;
            }
            drop -= own;
        }
    }
#pragma unroll
    for (int w = 0; w < W; ++w)
        if (w < p.words) s_bits[i * PITCH + w] = bits[w];
    if (i < s.count) p.positions[s.first + i] = start + depth;
    __syncthreads();
    uint32_t* to = p.ancestors + int64_t(s.first) * p.words;
    for (int e = i; e < s.count * p.words; e += NODES) {
        const int row = int(divide(uint32_t(e), p.by_words));
        to[e] = s_bits[row * PITCH + e - row * p.words];
    }
}

// ------------------------------------------------------------------------------------ accepted paths
// A wave a request takes 64 nodes at a time: the node that is kept last is known to all lanes, those whose parent it is
// and whose token it drew vote, and the first of them is kept next.  Children come after their parents, so one pass over the
// nodes finds the path.  Both kernels are latency-bound: a few dependent loads.
struct Step {
    Span span;
    int length, given;  // keys with the new tokens; tokens kept whatever was drawn
    bool fine;
};
__device__ __forceinline__ Step accept_step(const AcceptParams& p, int r) {
    Step s;
    s.length = p.lengths[r];
    const int first = p.offsets[r], end = p.offsets[r + 1];
    s.fine = first >= 0 && end >= first && end <= p.capacity && s.length >= end - first;
    s.span = {s.fine ? first : 0, s.fine ? end - first : 0};
    const int given = p.given ? p.given[r] : 1;
    s.given = min(max(given, 1), s.span.count);
    return s;
}

__device__ __forceinline__ int slot_of(const AcceptParams& p, int r, int at) {
    const uint32_t page = divide(uint32_t(at), p.div);
    if (page >= uint32_t(p.width)) return -1;
    const int entry = p.tables[int64_t(r) * p.width + page];
    return uint32_t(entry) < uint32_t(p.pages) ? entry * p.page_size + (at - int(page) * p.page_size) : -1;
}

// The paths of requests r, r + step, ..., EACH of them, by a wave: their loads side by side.  counts (or null): numbers of
// accepted tokens once more, in LDS.
template <int EACH>
__device__ __forceinline__ void accept_walk(const AcceptParams& p, int r0, int step, int* counts) {
    const int lane = threadIdx.x & 63;
    Step steps[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        const int r = r0 + e * step;
        steps[e] = r < p.rows ? accept_step(p, r) : Step{{0, 0}, 0, 0, true};
    }
    int drawn0[EACH], parents[EACH], tokens[EACH], nexts[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        const Step& s = steps[e];
        const int i = s.span.first + s.given + lane;
        const bool there = s.given + lane < s.span.count;
        drawn0[e] = s.span.count > 0 ? p.drawn[s.span.first + s.given - 1] : -1;
        parents[e] = there ? p.parents[i] : -1;
        tokens[e] = there ? p.tokens[i] : -1;
        nexts[e] = there ? p.drawn[i] : -1;
    }
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        const int r = r0 + e * step;
        if (r >= p.rows) return;
        const Step& s = steps[e];
        const int first = s.span.first, count = s.span.count, start = s.length - count;
        int32_t* accepted = p.accepted + int64_t(r) * (p.nodes + 1);
        int32_t *from = p.from + int64_t(r) * p.nodes, *to = p.to + int64_t(r) * p.nodes;
        int current = s.given - 1, kept = 0, drawn = __builtin_amdgcn_readfirstlane(drawn0[e]);
        for (int base = s.given; base < count && drawn >= 0; base += 64) {
            const int i = base + lane;
            int parent = parents[e], token = tokens[e], next = nexts[e];
            if (base > s.given) {
                const bool there = i < count;
                parent = there ? p.parents[first + i] : -1;
                token = there ? p.tokens[first + i] : -1;
                next = there ? p.drawn[first + i] : -1;
            }
            int place = -1;
            while (drawn >= 0) {
                const unsigned long long fits = __ballot(i < count && parent == current && token == drawn && i > current);
                if (!fits) break;
                const int l = __ffsll(fits) - 1;
                if (lane == l) place = kept;
                ++kept;
                current = base + l;
                drawn = __builtin_amdgcn_readlane(next, l);
            }
            if (place >= 0 && place < p.nodes) {
                accepted[place] = token;
                const int at = s.given + place;
                const int source = i != at ? slot_of(p, r, start + i) : -1, target = i != at ? slot_of(p, r, start + at) : -1;
                from[place] = source >= 0 && target >= 0 ? source : -1;
                to[place] = source >= 0 && target >= 0 ? target : -1;
            }
        }
        for (int i = kept + lane; i < p.nodes; i += 64) {
            accepted[i + 1] = -1;
            from[i] = to[i] = -1;
        }
        if (lane == 0) {
            if (kept <= p.nodes) accepted[kept] = drawn;
            p.accepted_counts[r] = count > 0 ? kept + 1 : 0;
            if (counts) counts[r] = count > 0 ? kept + 1 : 0;
            p.last[r] = count > 0 ? first + current : -1;
        }
    }
}

__global__ __launch_bounds__(WAVE_THREADS) void accept_walk_kernel(AcceptParams p) {
    const int r = int(blockIdx.x) * (WAVE_THREADS / 64) + int(threadIdx.x >> 6);
    if (r < p.rows) accept_walk<1>(p, r, 0, nullptr);
}

// One workgroup: a request a thread, sums of the pages given back in the order of requests.  A request gives back few:
// those that its drafts alone were in.
constexpr int PAGES_THREADS = 1024;

// Inclusive sum over the workgroup; `total` in every thread.
__device__ __forceinline__ int block_scan(int v, int* waves, int& total) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    v = wave_scan(v);
    __syncthreads();  // the sums of a scan before this one have been read
    if (lane == 63) waves[wave] = v;
    __syncthreads();
    static_assert(PAGES_THREADS / 64 == 16, "a row");
    const int sum = wave_scan(waves[lane & 15]);  // the lanes of a row hold the waves' sums
    total = __builtin_amdgcn_readlane(sum, 15);
    return wave > 0 ? v + __builtin_amdgcn_readlane(sum, wave - 1) : v;
}

// Requests whose paths this workgroup finds by itself first, a few for each of its waves: a launch less (64 requests of 8
// nodes 11.2 us in two, 8.4 so).
constexpr int WALKED = 4 * PAGES_THREADS / 64;

template <bool WALKS>
__global__ __launch_bounds__(PAGES_THREADS) void accept_pages_kernel(AcceptParams p) {
    __shared__ int s_waves[PAGES_THREADS / 64];
    __shared__ int s_status, s_accepted[WALKS ? WALKED : 1];
    const int tid = threadIdx.x;
    if constexpr (WALKS) {
        accept_walk<WALKED / (PAGES_THREADS / 64)>(p, int(threadIdx.x >> 6), PAGES_THREADS / 64, s_accepted);
    }
    if (tid == 0) s_status = 0;
    const int top = *p.free_count;
    // entries of request r that its length no longer reaches: columns after .. held - 1
    struct Back {
        int length, after, held, bad;
    };
    auto back_of = [&](int r) -> Back {
        const Step s = accept_step(p, r);
        const int accepted = WALKS ? s_accepted[r] : p.accepted_counts[r];
        const int kept = s.span.count > 0 ? s.given + accepted - 1 : 0;
        const int held = int((int64_t(s.length) + p.page_size - 1) / p.page_size);
        Back b;
        b.bad = s.fine ? (held > p.width ? 2 : 0) | (s.span.count - s.given > p.nodes ? 4 : 0) : 8;
        b.length = s.length - s.span.count + kept;
        b.after = int((int64_t(b.length) + p.page_size - 1) / p.page_size);
        b.held = held;
        return b;
    };
    __syncthreads();
    // the first PAGES_THREADS requests' stay in registers
    Back first = {};
    if (tid < p.rows) first = back_of(tid);
    auto pages_of = [&](const Back& b, int r, auto f) {
        for (int c = b.after; c < b.held; ++c) {
            const int entry = p.tables[int64_t(r) * p.width + c];
            if (uint32_t(entry) < uint32_t(p.pages)) f(entry);
        }
    };
    int bad = 0;
    for (int r = tid; r < p.rows; r += PAGES_THREADS) bad |= r == tid ? first.bad : back_of(r).bad;
    if (bad) atomicOr(&s_status, bad);
    __syncthreads();
    int status = s_status;
    if (top < 0 || top > p.pages) status |= 8;
    int64_t total = 0;
    if (!status) {
        for (int base = 0; base < p.rows; base += PAGES_THREADS) {
            const int r = base + tid;
            int own = 0, sum;
            if (r < p.rows) pages_of(base ? back_of(r) : first, r, [&](int) { ++own; });
            block_scan(own, s_waves, sum);
            total += sum;
        }
        if (top + total > p.pages) status |= 8;
    }
    if (!status) {
        int at = top;
        for (int base = 0; base < p.rows; base += PAGES_THREADS) {
            const int r = base + tid;
            int own = 0, sum;
            Back b = {};
            if (r < p.rows) {
                b = base ? back_of(r) : first;
                pages_of(b, r, [&](int) { ++own; });
            }
            int place = at + block_scan(own, s_waves, sum) - own;
            if (r < p.rows) {
                pages_of(b, r, [&](int entry) { p.free_pages[place++] = entry; });
                p.lengths_out[r] = b.length;
            }
            at += sum;
        }
        if (tid == 0) *p.free_out = at;
    } else {
        // nothing is kept, and nothing changes
        for (int r = tid; r < p.rows; r += PAGES_THREADS) {
            p.lengths_out[r] = p.lengths[r];
            p.accepted_counts[r] = 0;
            p.last[r] = -1;
        }
        for (int64_t e = tid; e < int64_t(p.rows) * (p.nodes + 1); e += PAGES_THREADS) p.accepted[e] = -1;
        for (int64_t e = tid; e < int64_t(p.rows) * p.nodes; e += PAGES_THREADS) p.from[e] = p.to[e] = -1;
        if (tid == 0) *p.free_out = top;
    }
    if (tid == 0) *p.status = status;
}

// ------------------------------------------------------------------------------------ moves
// A thread takes a 16-byte piece of a group's tokens, in their order, several loads ahead of the stores: what a move
// of a group writes no later one of it reads.  Bound by memory, which takes rows of 256 bytes from anywhere to anywhere at
// 3.7 TB/s (20,000 tokens of one KV head in 16 layers 88 us; eight copies a thread 112, four layers' keys and values a thread 89),
// or by the latency of three accesses (64 requests of 7 nodes 4.6 us; four moves' keys and values a thread 10).
constexpr int MOVE_AHEAD = 8;

__device__ __forceinline__ int64_t move_at(const MoveParams& p, int slot) {
    const uint32_t page = divide(uint32_t(slot), p.div);
    return page * p.page_stride + int64_t(slot - int(page) * p.page_size) * p.slot_stride;
}

__global__ __launch_bounds__(256) void move_kernel(MoveParams p) {
    const int columns = p.kv_heads * p.chunks;
    const int64_t item = int64_t(blockIdx.x) * 256 + threadIdx.x;
    const int64_t g = item / columns;
    if (g >= p.groups) return;
    const int column = int(item - g * columns), head = column / p.chunks;
    char* base = reinterpret_cast<char*>(blockIdx.z ? p.values[blockIdx.y] : p.keys[blockIdx.y]) + head * p.head_stride +
                 (column - head * p.chunks) * 16;
    const int64_t slots = int64_t(p.pages) * p.page_size;
    for (int i = 0; i < p.group; i += MOVE_AHEAD) {
        uint4 held[MOVE_AHEAD];
        int target[MOVE_AHEAD];
#pragma unroll
        for (int a = 0; a < MOVE_AHEAD; ++a) {
            target[a] = -1;
            if (i + a >= p.group) continue;
            const int64_t at = g * p.group + i + a;
            const int source = p.from[at], to = p.to[at];
            if (source < 0 || to < 0 || source >= slots || to >= slots) continue;
            held[a] = *reinterpret_cast<const uint4*>(base + move_at(p, source));
            target[a] = to;
        }
#pragma unroll
        for (int a = 0; a < MOVE_AHEAD; ++a)
            if (target[a] >= 0) *reinterpret_cast<uint4*>(base + move_at(p, target[a])) = held[a];
    }
}

// ------------------------------------------------------------------------------------ controls
// A workgroup takes a segment of a row's vocabulary: a word of LDS a token counts how often the row's sequence has it,
// and holds whether an n-gram bans it and which bias it has; then one pass over the logits, which were loaded before.  All
// of the sequence is looked through for each segment.  Bound by memory and what a workgroup waits for before it writes
// (145 BF16 rows of 107,520, histories of up to 700 and paths, biases, masks on half of them 17.8 us, 3.5 TB/s read and
// written; segments of 8,192 with 512 threads, and of 16,384 with 1,024, take 17.8 and 18.2).
constexpr int CONTROL_THREADS = 256, CONTROL_SEGMENT = 4096, EACH = 8;
constexpr uint32_t COUNT_BITS = 18, BANNED = 1u << COUNT_BITS, COUNTED = BANNED - 1;
static_assert(CONTROL_MAX_HISTORY + 32 * TREE_MAX_WORDS < int(BANNED) && CONTROL_MAX_BIAS < (1 << (31 - COUNT_BITS)), "a word holds them");

// The sequence of row t, offsets[r] <= t < offsets[r + 1], by looking at 64 of a range at a time; -1 for none.  (Offsets
// that descend may lead to any sequence: it is looked at once more.)
__device__ __forceinline__ int find_sequence(const int32_t* offsets, int sequences, int t) {
    const int lane = threadIdx.x & 63;
    int lo = 0, span = sequences, step;
    do {
        step = (span + 63) / 64;
        const int64_t at = lo + int64_t(lane) * step + step - 1;
        const bool before = at < sequences && offsets[at + 1] <= t;  // true for the first lanes
        lo += __popcll(__ballot(before)) * step;
        span = step;
    } while (step > 1);
    return lo < sequences && offsets[lo] <= t && offsets[lo + 1] > t ? lo : -1;
}

template <int TYPE>
__device__ __forceinline__ float load1(const char* row, int i) {
    if constexpr (TYPE == TYPE_F32) return reinterpret_cast<const float*>(row)[i];
    else return from16<TYPE>(reinterpret_cast<const uint16_t*>(row)[i]);
}
template <int TYPE>
__device__ __forceinline__ void store1(char* row, int i, float v) {
    if constexpr (TYPE == TYPE_F32) reinterpret_cast<float*>(row)[i] = v;
    else reinterpret_cast<uint16_t*>(row)[i] = uint16_t(pack16<TYPE>(v, 0.f));
}
// Eight neighbours, of any alignment.
template <int TYPE>
__device__ __forceinline__ void load8(const char* row, int i, float (&v)[EACH]) {
    if constexpr (TYPE == TYPE_F32) {
        __builtin_memcpy(v, row + int64_t(i) * 4, 32);
    } else {
        uint4 x;
        __builtin_memcpy(&x, row + int64_t(i) * 2, 16);
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int e = 0; e < EACH; ++e) v[e] = from16<TYPE>(w[e >> 1] >> (16 * (e & 1)));
    }
}
template <int TYPE>
__device__ __forceinline__ void store8(char* row, int i, const float (&v)[EACH]) {
    if constexpr (TYPE == TYPE_F32) {
        __builtin_memcpy(row + int64_t(i) * 4, v, 32);
    } else {
        const uint4 x = make_uint4(pack16<TYPE>(v[0], v[1]), pack16<TYPE>(v[2], v[3]), pack16<TYPE>(v[4], v[5]), pack16<TYPE>(v[6], v[7]));
        __builtin_memcpy(row + int64_t(i) * 2, &x, 16);
    }
}

struct Penalties {
    float repetition, presence, frequency;
};
// As the runtime's controls do it (no contraction), then the bias.
__device__ __forceinline__ float controlled(float x, uint32_t word, bool open, const Penalties& c, const float* bias) {
#pragma clang fp contract(off)
    if (word) {
        const uint32_t count = word & COUNTED;
        if (count) {
            if (c.repetition != 1.0f) x = x > 0.0f ? x / c.repetition : x * c.repetition;
            if (c.presence != 0.0f) x = x - c.presence;
            if (c.frequency != 0.0f) {
                const float f = c.frequency * float(count);
                x = x - f;
            }
        }
        const uint32_t entry = word >> (COUNT_BITS + 1);
        if (entry) x = x + bias[entry - 1];
        if (word & BANNED) x = NEG_INF;
    }
    return open ? x : NEG_INF;
}

template <int TYPE, int OUT>
__global__ __launch_bounds__(CONTROL_THREADS) void controls_kernel(ControlParams p, int segments) {
    __shared__ __align__(16) uint32_t s_word[CONTROL_SEGMENT];
    __shared__ int32_t s_path[32 * TREE_MAX_WORDS];
    const int tid = threadIdx.x, lane = tid & 63;
    const int t = int(blockIdx.x) / segments, low = (int(blockIdx.x) - t * segments) * CONTROL_SEGMENT;
    const int r = __builtin_amdgcn_readfirstlane(p.offsets ? find_sequence(p.offsets, p.sequences, t) : t);
    if (r < 0) return;  // a row behind the last sequence's
    const int size = min(CONTROL_SEGMENT, p.n - low);

    // the logits and the mask's bits are on their way while the sequence is looked through
    constexpr int ROUNDS = CONTROL_SEGMENT / (CONTROL_THREADS * EACH);
    const char* in = p.logits + int64_t(t) * p.stride * (TYPE == TYPE_F32 ? 4 : 2);
    const uint8_t* mask = nullptr;
    if (p.masks) {
        const int m = p.mask_rows ? p.mask_rows[t] : t;
        if (uint32_t(m) < uint32_t(p.mask_count)) mask = reinterpret_cast<const uint8_t*>(p.masks + int64_t(m) * p.mask_stride) + low / 8;
    }
    float v[ROUNDS][EACH];
    uint32_t open[ROUNDS];
#pragma unroll
    for (int k = 0; k < ROUNDS; ++k) {
        const int i = (k * CONTROL_THREADS + tid) * EACH;
        open[k] = mask && i < size ? mask[i / 8] : 0xffu;
        if (!p.in_place && i + EACH <= size) load8<TYPE>(in, low + i, v[k]);
    }
#pragma unroll
    for (int i = 0; i < CONTROL_SEGMENT / (4 * CONTROL_THREADS); ++i)
        *reinterpret_cast<uint4*>(&s_word[(i * CONTROL_THREADS + tid) * 4]) = make_uint4(0, 0, 0, 0);
    // the path's tokens, in the order of their bits: the same in every wave
    int path = 0;
    if (p.ancestors) {
        const int first = max(p.offsets[r], 0), count = min(min(p.offsets[r + 1], p.rows) - first, 32 * p.words);
        for (int base = 0; base < count; base += 64) {
            const int node = base + lane;
            const uint32_t bits = node < count ? p.ancestors[int64_t(t) * p.words + node / 32] : 0u;
            const int32_t token = node < count ? p.tokens[first + node] : -1;
            const bool on = bits >> (node & 31) & 1u;
            const unsigned long long all = __ballot(on);
            if (on && tid < 64) s_path[path + __popcll(all & ((1ull << lane) - 1))] = token;
            path += __popcll(all);
        }
    }
    Penalties c = {p.repetition ? p.repetition[r] : 1.0f, p.presence ? p.presence[r] : 0.0f, p.frequency ? p.frequency[r] : 0.0f};
    if (!(c.repetition > 0.0f)) c.repetition = 1.0f;
    if (c.presence != c.presence) c.presence = 0.0f;
    if (c.frequency != c.frequency) c.frequency = 0.0f;
    const int length = p.history ? min(max(p.history_lengths[r], 0), p.history_width) : 0, all = length + path;
    const int32_t* history = p.history + int64_t(r) * p.history_stride;
    // (an n-gram is compared token by token wherever the token before it fits: the longest bounds what a history of one
    // token costs, 4.2 ms for 2^17 of it, 3-grams 0.26)
    const int ngram = p.ngram ? p.ngram[r] : 0, span = ngram > 1 && ngram <= min(all, CONTROL_MAX_NGRAM) ? ngram - 1 : 0;
    const bool looks = span || c.repetition != 1.0f || c.presence != 0.0f || c.frequency != 0.0f;
    // the first tokens and biases are on their way before the counts are cleared, and the tokens before these: few follow
    // the sequence's last one, and all but those need no look at the rest of an n-gram
    constexpr int SOON = 4;
    int32_t soon[SOON], before[SOON];
#pragma unroll
    for (int k = 0; k < SOON; ++k) {
        const int i = k * CONTROL_THREADS + tid;
        soon[k] = looks && i < length ? history[i] : -1;
        before[k] = span && i > 0 && i < length ? history[i - 1] : -1;
    }
    int32_t last = span && path == 0 ? history[length - 1] : -1;
    const int32_t* ids = p.bias_ids + int64_t(r) * p.bias_width;
    const int32_t id = p.bias_ids && tid < p.bias_width ? ids[tid] : -1;
    __syncthreads();
    if (p.bias_ids) {
        for (int i = tid; i < p.bias_width; i += CONTROL_THREADS) {
            const uint32_t at = uint32_t(i == tid ? id : ids[i]) - uint32_t(low);
            if (at < uint32_t(size)) atomicMax(&s_word[at], uint32_t(i + 1) << (COUNT_BITS + 1));
        }
        __syncthreads();
    }
    if (span && path > 0) last = s_path[path - 1];
    if (looks) {
        auto said = [&](int i) { return i < length ? history[i] : s_path[i - length]; };
        auto take = [&](int i, int32_t token, int32_t previous) {
            const uint32_t at = uint32_t(token) - uint32_t(low);
            if (at >= uint32_t(size)) return;
            atomicAdd(&s_word[at], 1u);
            if (span && i >= span && previous == last) {
                bool same = true;
                for (int k = 2; k <= span && same; ++k) same = said(i - k) == said(all - k);
                if (same) atomicOr(&s_word[at], BANNED);
            }
        };
#pragma unroll
        for (int k = 0; k < SOON; ++k)
            if (k * CONTROL_THREADS + tid < length) take(k * CONTROL_THREADS + tid, soon[k], before[k]);
        for (int i = SOON * CONTROL_THREADS + tid; i < length; i += CONTROL_THREADS) take(i, history[i], span ? history[i - 1] : -1);
        for (int i = tid; i < path; i += CONTROL_THREADS)
            take(length + i, s_path[i], i > 0 ? s_path[i - 1] : span && length > 0 ? history[length - 1] : -1);
    }
    __syncthreads();
    char* out = p.out + int64_t(t) * p.out_stride * (OUT == TYPE_F32 ? 4 : 2);
    const float* bias = p.bias + int64_t(r) * p.bias_width;
#pragma unroll
    for (int k = 0; k < ROUNDS; ++k) {
        const int i = (k * CONTROL_THREADS + tid) * EACH;
        if (i >= size) break;
        uint32_t word[EACH], any = 0;
#pragma unroll
        for (int e = 0; e < EACH; ++e) any |= word[e] = s_word[i + e];
        if (p.in_place && !any && open[k] == 0xffu) continue;
        if (i + EACH <= size) {
            if (p.in_place) load8<TYPE>(in, low + i, v[k]);
            if (any || open[k] != 0xffu) {
#pragma unroll
                for (int e = 0; e < EACH; ++e) v[k][e] = controlled(v[k][e], word[e], open[k] >> e & 1u, c, bias);
            }
            store8<OUT>(out, low + i, v[k]);
        } else {
#pragma unroll
            for (int e = 0; e < EACH; ++e)
                if (i + e < size) store1<OUT>(out, low + i + e, controlled(load1<TYPE>(in, low + i + e), word[e], open[k] >> e & 1u, c, bias));
        }
    }
}

}  // namespace

void launch_paged_tree(const TreeParams& p, hipStream_t s) {
    if (p.words <= 2) {
        const int each = WAVE_THREADS / 64;
        hipLaunchKernelGGL(tree_wave_kernel, dim3(unsigned((p.rows + each - 1) / each)), dim3(WAVE_THREADS), 0, s, p);
    } else if (p.words <= 8) {
        hipLaunchKernelGGL(tree_block_kernel<8>, dim3(unsigned(p.rows)), dim3(32 * 8), 0, s, p);
    } else if (p.words <= 16) {
        hipLaunchKernelGGL(tree_block_kernel<16>, dim3(unsigned(p.rows)), dim3(32 * 16), 0, s, p);
    } else {
        hipLaunchKernelGGL(tree_block_kernel<32>, dim3(unsigned(p.rows)), dim3(32 * 32), 0, s, p);
    }
}

void launch_paged_accept(const AcceptParams& p, hipStream_t s) {
    if (p.rows <= WALKED) {
        hipLaunchKernelGGL(accept_pages_kernel<true>, dim3(1), dim3(PAGES_THREADS), 0, s, p);
        return;
    }
    const int each = WAVE_THREADS / 64;
    hipLaunchKernelGGL(accept_walk_kernel, dim3(unsigned((p.rows + each - 1) / each)), dim3(WAVE_THREADS), 0, s, p);
    hipLaunchKernelGGL(accept_pages_kernel<false>, dim3(1), dim3(PAGES_THREADS), 0, s, p);
}

void launch_paged_move(const MoveParams& p, hipStream_t s) {
    const int64_t items = int64_t(p.groups) * p.kv_heads * p.chunks;  // (the caller's check: a launch holds them)
    hipLaunchKernelGGL(move_kernel, dim3(unsigned((items + 255) / 256), unsigned(p.layers), 2), dim3(256), 0, s, p);
}

static int control_segments(int n) { return (n + CONTROL_SEGMENT - 1) / CONTROL_SEGMENT; }
bool controls_launches(int n, int rows) { return int64_t(control_segments(n)) * rows * CONTROL_THREADS <= UINT32_MAX; }

template <int TYPE, int OUT>
static void run_controls(const ControlParams& p, hipStream_t s) {
    const int segments = control_segments(p.n);
    hipLaunchKernelGGL((controls_kernel<TYPE, OUT>), dim3(unsigned(segments) * unsigned(p.rows)), dim3(CONTROL_THREADS), 0, s, p, segments);
}

void launch_logit_controls(const ControlParams& p, int type, int out_type, hipStream_t s) {
    if (type == TYPE_F32) run_controls<TYPE_F32, TYPE_F32>(p, s);
    else if (type == TYPE_BF16 && out_type == TYPE_BF16) run_controls<TYPE_BF16, TYPE_BF16>(p, s);
    else if (type == TYPE_BF16) run_controls<TYPE_BF16, TYPE_F32>(p, s);
    else if (out_type == TYPE_F16) run_controls<TYPE_F16, TYPE_F16>(p, s);
    else run_controls<TYPE_F16, TYPE_F32>(p, s);
}

}  // namespace plamo
