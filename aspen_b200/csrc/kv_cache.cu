// The paged key-value cache: finding, sharing, freeing and moving pages, and writing tokens into them.
//
// The state of the pool (page_table, lengths, refs) lives in device memory and only kernels change it, so a serving loop never waits for the GPU to learn
// a length, and a step of it can be captured.  A page is free when refs is 0; there is no list of free pages that could disagree with that.
//
// extend, fork and compact begin with ONE CTA of 1024 threads that checks everything before it changes anything and picks pages in a fixed order: the state
// is small (4 bytes a page; 65 536 pages are 64 loads a thread) and a grid would need two more launches for its sums.  What moves data is a second kernel over all
// SMs that starts while the first one runs and waits for its end on the device (early_launch.cuh).
// Pages are copied with 16-byte loads, two of each of an SM's 2048 threads in flight (four: compaction of 32 sequences 66 us instead of 62, where 50 are the bytes); bound by memory.
#include "attention.h"
#include "early_launch.cuh"

namespace {

using attn::Pages;
using attn::launch_early;
using attn::let_next_kernel_start;
using attn::wait_for_previous_kernel;

constexpr unsigned BOOK = 1024;                // threads of the CTA that keeps the books
constexpr unsigned MOST_PAGES = 1u << 21;      // for one entry of an extend: sums over the CTA's threads stay below 2^32
constexpr unsigned PLACED = 4;                 // new pages that a thread of extend finds the places of at once
constexpr unsigned COPY = 256, IN_FLIGHT = 2, COPY_CTAS = 8;        // threads of a copying CTA, 16-byte loads in flight of each, CTAs on an SM

struct Pool {
    Pages at;
    int *table, *lengths, *refs;
};

// Workspace, in ints: a header (count, ok), then five arrays.
struct Space {
    int *head;
    int *start;     // [entries + 1] first of an entry's new pages
    int *length;    // [entries]
    int *from;      // [max(entries, pages)]
    int *to;        // [max(entries, pages)] new or free pages
    int *mark;      // [max(sequences, pages)]
};
enum { COUNT = 0, OK = 1, LIVE = 2, HEAD = 4 };

size_t space_ints(const aspen_b200_cache_t &c, unsigned entries) {
    const size_t list = entries > c.pages ? entries : c.pages, mark = c.sequences > c.pages ? c.sequences : c.pages;
    return HEAD + 2 * (size_t)entries + 1 + 2 * list + mark;
}
Space space_of(const aspen_b200_cache_t &c, unsigned entries, void *workspace) {
    const size_t list = entries > c.pages ? entries : c.pages;
    Space w;
    w.head = static_cast<int *>(workspace);
    w.start = w.head + HEAD;
    w.length = w.start + entries + 1;
    w.from = w.length + entries;
    w.to = w.from + list;
    w.mark = w.to + list;
    return w;
}

// Sum over the threads before this one; `all` is that over all of them.  For the whole CTA of BOOK threads.
__device__ __forceinline__ unsigned before_me(unsigned v, unsigned &all, unsigned *sums) {
    const unsigned lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    unsigned s = v;
    #pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const unsigned u = __shfl_up_sync(0xffffffffu, s, o); if (lane >= (unsigned)o) s += u; }
    __syncthreads();                            // the sums of the call before have been read
    if (lane == 31) sums[warp] = s;
    __syncthreads();
    unsigned t = sums[lane];                    // BOOK / 32 = 32 of them
    #pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const unsigned u = __shfl_up_sync(0xffffffffu, t, o); if (lane >= (unsigned)o) t += u; }
    all = __shfl_sync(0xffffffffu, t, 31);
    const unsigned base = __shfl_sync(0xffffffffu, t, warp ? warp - 1 : 0);
    return (warp ? base : 0u) + s - v;
}

constexpr unsigned SCAN = 8;                   // pages a thread looks at in a turn

// The `want` lowest free pages, in order, to `list`; returns how many there are (up to `want`).  A warp looks at 256 pages in a row, 32 a load, and those of the next
// turn are on their way while these are counted.
__device__ unsigned lowest_free(const int *refs, unsigned pages, unsigned want, int *list, unsigned *sums) {
    const unsigned lane = threadIdx.x % 32, mine = threadIdx.x / 32 * (32 * SCAN) + lane;
    unsigned found = 0;
    int v[SCAN];
    auto load = [&](unsigned first) {
        #pragma unroll
        for (unsigned i = 0; i < SCAN; i++) v[i] = first + i * 32 < pages ? refs[first + i * 32] : 1;
    };
    if (want) load(mine);
    for (unsigned p0 = 0; p0 < pages && found < want; p0 += BOOK * SCAN) {
        unsigned free[SCAN], count = 0;
        #pragma unroll
        for (unsigned i = 0; i < SCAN; i++) { free[i] = __ballot_sync(0xffffffffu, v[i] == 0); count += __popc(free[i]); }
        load(p0 + BOOK * SCAN + mine);
        unsigned all, rank = found + before_me(lane == 0 ? count : 0u, all, sums);
        rank = __shfl_sync(0xffffffffu, rank, 0);
        #pragma unroll
        for (unsigned i = 0; i < SCAN; i++) {
            const unsigned at = rank + __popc(free[i] & ((1u << lane) - 1u));
            if (free[i] >> lane & 1u && at < want) list[at] = (int)(p0 + mine + i * 32);
            rank += __popc(free[i]);
        }
        found += all;
    }
    __syncthreads();
    return found < want ? found : want;
}

// The sequences that a refused call would have given tokens to.
__device__ __forceinline__ void refuse(const Pool &pool, const int *slots, unsigned entries) {
    if (!pool.at.refused) return;
    for (unsigned e = threadIdx.x; e < entries; e += BOOK) {
        const int slot = slots ? slots[e] : (int)e;
        if (slot >= 0 && (unsigned)slot < pool.at.sequences) pool.at.refused[slot] = 1;
    }
}

__device__ __forceinline__ unsigned pages_for(unsigned long long tokens, unsigned page) { return (unsigned)((tokens + page - 1) / page); }

__global__ void __launch_bounds__(BOOK) extend_kernel(const Pool pool, const Space w, const int *slots, const int *starts, unsigned entries) {
    __shared__ unsigned sums[32];
    __shared__ int refused;
    const unsigned page = pool.at.page_size;
    wait_for_previous_kernel();
    if (threadIdx.x == 0) refused = 0;
    if (slots)
        for (unsigned i = threadIdx.x; i < pool.at.sequences; i += BOOK) w.mark[i] = 0;
    __syncthreads();
    unsigned total = 0;
    int why = 0;
    for (unsigned e0 = 0; e0 < entries; e0 += BOOK) {
        const unsigned e = e0 + threadIdx.x;
        unsigned need = 0;
        if (e < entries) {
            const int slot = slots ? slots[e] : (int)e;
            const long long more = starts ? (long long)starts[e + 1] - starts[e] : 1;
            if (slot < 0 || (unsigned)slot >= pool.at.sequences || more < 0) why |= ASPEN_B200_CACHE_BAD_INDEX;
            else if (slots && atomicAdd(&w.mark[slot], 1) != 0) why |= ASPEN_B200_CACHE_BAD_INDEX;
            else if (attn::is_refused(pool.at, slot)) why |= ASPEN_B200_CACHE_REFUSED;
            else {
                const unsigned now = attn::sequence_length(pool.at, slot);
                const unsigned long long then = now + (unsigned long long)more;
                if (then > (unsigned long long)pool.at.max_pages * page) why |= ASPEN_B200_CACHE_TOO_LONG;
                else need = pages_for(then, page) - pages_for(now, page);
            }
        }
        if (need > min(pool.at.pages, MOST_PAGES)) { why |= ASPEN_B200_CACHE_NO_PAGES; need = 0; }
        unsigned all;
        const unsigned at = total + before_me(need, all, sums);
        if (e < entries) w.start[e] = (int)at;
        total += all;
        if (total > pool.at.pages) { why |= ASPEN_B200_CACHE_NO_PAGES; total = pool.at.pages + 1; break; }
    }
    if (why) atomicOr(&refused, why);
    __syncthreads();
    if (!refused) {
        if (lowest_free(pool.refs, pool.at.pages, total, w.to, sums) < total && threadIdx.x == 0) refused = ASPEN_B200_CACHE_NO_PAGES;
        __syncthreads();
    }
    if (refused) {
        refuse(pool, slots, entries);
        if (threadIdx.x == 0) atomicOr(pool.at.status, refused | ASPEN_B200_CACHE_REFUSED);
        return;
    }
    unsigned top = 1;                               // the largest power of two that is not above the last entry
    while (top * 2 < entries) top *= 2;
    for (unsigned i0 = threadIdx.x; i0 < total; i0 += BOOK * PLACED) {
        // the last entry that starts at i or before; empty ones start where the next does
        unsigned entry[PLACED];
        #pragma unroll
        for (unsigned u = 0; u < PLACED; u++) entry[u] = 0;
        for (unsigned step = top; step > 0; step /= 2)
            #pragma unroll
            for (unsigned u = 0; u < PLACED; u++) { const unsigned e = entry[u] + step; if (e < entries && (unsigned)w.start[e] <= i0 + u * BOOK) entry[u] = e; }
        #pragma unroll
        for (unsigned u = 0; u < PLACED; u++) {
            const unsigned i = i0 + u * BOOK, e = entry[u];
            if (i >= total) continue;
            const int slot = slots ? slots[e] : (int)e, p = w.to[i];
            pool.table[(size_t)slot * pool.at.max_pages + pages_for(attn::sequence_length(pool.at, slot), page) + (i - (unsigned)w.start[e])] = p;
            pool.refs[p] = 1;
        }
    }
    __syncthreads();
    for (unsigned e = threadIdx.x; e < entries; e += BOOK) {
        const int slot = slots ? slots[e] : (int)e;
        pool.lengths[slot] = (int)(attn::sequence_length(pool.at, slot) + (unsigned)(starts ? starts[e + 1] - starts[e] : 1));
    }
}

enum { TARGET = 1, SOURCE = 2 };               // marks of a sequence
__global__ void __launch_bounds__(BOOK) fork_kernel(const Pool pool, const Space w, const int *from, const int *to, unsigned entries) {
    __shared__ unsigned sums[32];
    __shared__ int refused;
    const unsigned page = pool.at.page_size;
    let_next_kernel_start();
    wait_for_previous_kernel();
    if (threadIdx.x == 0) refused = 0;
    for (unsigned i = threadIdx.x; i < pool.at.sequences; i += BOOK) w.mark[i] = 0;
    __syncthreads();
    unsigned total = 0;
    int why = 0;
    for (unsigned e0 = 0; e0 < entries; e0 += BOOK) {
        const unsigned e = e0 + threadIdx.x;
        unsigned part = 0;
        bool first = false;                         // of the entries with this source
        if (e < entries) {
            const int a = from[e], b = to[e];
            unsigned len = 0;
            if (a < 0 || (unsigned)a >= pool.at.sequences || b < 0 || (unsigned)b >= pool.at.sequences) why |= ASPEN_B200_CACHE_BAD_INDEX;
            else if (atomicOr(&w.mark[b], TARGET) & TARGET || pool.lengths[b] != 0) why |= ASPEN_B200_CACHE_BAD_INDEX;
            else if (attn::is_refused(pool.at, a) || attn::is_refused(pool.at, b)) why |= ASPEN_B200_CACHE_REFUSED;
            else {
                len = attn::sequence_length(pool.at, a);
                first = !(atomicOr(&w.mark[a], SOURCE) & SOURCE);
                part = len % page != 0;
                if (part) {
                    const int last = pool.table[(size_t)a * pool.at.max_pages + len / page];
                    if (last < 0 || (unsigned)last >= pool.at.pages) why |= ASPEN_B200_CACHE_BAD_INDEX;
                    w.from[e] = last;
                }
            }
            w.length[e] = (int)len;
            w.to[e] = first;
        }
        unsigned all;
        const unsigned at = total + before_me(part, all, sums);
        if (e < entries) w.start[e] = (int)at;
        total += all;
        if (total > pool.at.pages) { why |= ASPEN_B200_CACHE_NO_PAGES; break; }
    }
    if (why) atomicOr(&refused, why);
    __syncthreads();
    const bool go_on = !refused;
    __syncthreads();                                // all have read it
    if (go_on) {
        // the sources' full pages, each source's once: 32 pages at a time, the first ones of the source of entry i by warp i
        const unsigned lane = threadIdx.x % 32, warp = threadIdx.x / 32;
        bool bad = false;
        for (unsigned e0 = 0; e0 < entries; e0 += 32) {
            const unsigned e = e0 + lane;
            const bool mine = e < entries && w.to[e];
            const int a = mine ? from[e] : 0;
            const unsigned full = mine ? (unsigned)w.length[e] / page : 0u;
            for (unsigned left = __ballot_sync(0xffffffffu, full > 0); left; left &= left - 1) {
                const unsigned at = __ffs(left) - 1, n = __shfl_sync(0xffffffffu, full, at);
                const int *const row = pool.table + (size_t)__shfl_sync(0xffffffffu, a, at) * pool.at.max_pages;
                for (unsigned i = ((warp - at) % 32) * 32 + lane; i < n; i += BOOK) bad |= (unsigned)row[i] >= pool.at.pages;
            }
        }
        if (bad) atomicOr(&refused, ASPEN_B200_CACHE_BAD_INDEX);
    }
    __syncthreads();
    if (!refused) {
        if (lowest_free(pool.refs, pool.at.pages, total, w.to, sums) < total && threadIdx.x == 0) refused = ASPEN_B200_CACHE_NO_PAGES;
        __syncthreads();
    }
    if (!refused)
        for (unsigned i = threadIdx.x; i < total; i += BOOK) pool.refs[w.to[i]] = 1;
    else refuse(pool, to, entries);
    if (threadIdx.x == 0) {
        if (refused) atomicOr(pool.at.status, refused | (pool.at.refused ? ASPEN_B200_CACHE_REFUSED : 0));
        w.head[OK] = !refused;
    }
}

// One layer's keys or values of a page: `tokens` rows of each head, vectors of 16 bytes.
struct Plane {
    uint4 *base[2];                     // k, v
    size_t layer, page, head, token;    // strides in vectors
    unsigned layers, heads, page_size, row;      // row: vectors of a token of one head
    bool dense;                         // a page of a layer is contiguous
};

// Vectors `first`, first + step, ... (IN_FLIGHT of them, those below `end`) of the first `tokens` tokens of a page, from one page to another.
__device__ __forceinline__ void copy_plane(const Plane &p, const uint4 *src, uint4 *dst, unsigned tokens, unsigned first, unsigned end, unsigned step) {
    const bool dense = p.dense && tokens == p.page_size;
    const unsigned per = tokens * p.row;
    uint4 v[IN_FLIGHT];
    auto at = [&](unsigned i) -> size_t {
        if (dense) return i;
        const unsigned h = i / per, r = i - h * per, t = r / p.row;
        return h * p.head + t * p.token + (r - t * p.row);
    };
    #pragma unroll
    for (unsigned j = 0; j < IN_FLIGHT; j++) if (first + j * step < end) v[j] = __ldcs(src + at(first + j * step));
    #pragma unroll
    for (unsigned j = 0; j < IN_FLIGHT; j++) if (first + j * step < end) __stcs(dst + at(first + j * step), v[j]);
}

// Copies pages of all layers: worker by worker of `workers`, pieces of COPY * IN_FLIGHT vectors.
// Pair: bool operator()(unsigned i, int &from, int &to, unsigned &tokens).
template <typename Pair>
__device__ __forceinline__ void copy_pages(const Plane &p, unsigned count, const Pair &pair, unsigned worker, unsigned workers) {
    constexpr unsigned PIECE = COPY * IN_FLIGHT;
    const unsigned whole = p.heads * p.page_size * p.row, pieces = (whole + PIECE - 1) / PIECE, each = pieces * p.layers * 2;        // of a pair of pages
    const unsigned pairs_on = workers / each, rest_on = workers - pairs_on * each;
    unsigned i = worker / each, rest = worker - i * each;
    for (; i < count; i += pairs_on, rest += rest_on) {
        if (rest >= each) { rest -= each; if (++i >= count) break; }
        const unsigned plane = rest / pieces, piece = rest - plane * pieces, kv = plane & 1u, layer = plane >> 1;
        int a, b;
        unsigned tokens;
        if (!pair(i, a, b, tokens)) continue;
        const unsigned vectors = p.heads * tokens * p.row, first = piece * PIECE, end = min(vectors, first + PIECE);
        if (first >= vectors) continue;
        uint4 *const base = (kv ? p.base[1] : p.base[0]) + layer * p.layer;
        copy_plane(p, base + (size_t)a * p.page, base + (size_t)b * p.page, tokens, first + threadIdx.x, end, COPY);
    }
}

struct ForkPair {
    const Space &w;
    unsigned page;
    __device__ __forceinline__ bool operator()(unsigned e, int &from, int &to, unsigned &tokens) const {
        tokens = (unsigned)w.length[e] % page;
        if (!tokens) return false;
        from = w.from[e];
        to = w.to[w.start[e]];
        return true;
    }
};
__global__ void __launch_bounds__(COPY, COPY_CTAS) fork_copy_kernel(const Pool pool, const Space w, const Plane plane, const int *from, const int *to, unsigned entries) {
    wait_for_previous_kernel();
    if (!w.head[OK]) return;
    const unsigned max_pages = pool.at.max_pages, page = pool.at.page_size, strips = (max_pages + COPY - 1) / COPY, half = gridDim.x / 2;
    // half of the CTAs copy tokens, the others rows of the table
    if (blockIdx.x < half) { copy_pages(plane, entries, ForkPair{w, page}, blockIdx.x, half); return; }
    for (unsigned long long u = blockIdx.x - half; u < (unsigned long long)entries * strips; u += gridDim.x - half) {
        const unsigned e = (unsigned)(u / strips), i = (unsigned)(u % strips) * COPY + threadIdx.x;
        if (i >= max_pages) continue;
        const unsigned len = (unsigned)w.length[e], full = len / page;
        int p = -1;
        if (i < full) {
            p = pool.table[(size_t)from[e] * max_pages + i];
            if ((unsigned)p < pool.at.pages) atomicAdd(&pool.refs[p], 1);
        } else if (i == full && len % page) p = w.to[w.start[e]];
        pool.table[(size_t)to[e] * max_pages + i] = p;
        if (i == 0) pool.lengths[to[e]] = (int)len;
    }
}

__global__ void __launch_bounds__(COPY) free_kernel(const Pool pool, const int *slots) {
    __shared__ unsigned length;
    wait_for_previous_kernel();
    const int slot = slots[blockIdx.x];
    if (slot < 0 || (unsigned)slot >= pool.at.sequences) {
        if (threadIdx.x == 0) atomicOr(pool.at.status, ASPEN_B200_CACHE_BAD_INDEX);
        return;
    }
    const unsigned room = pool.at.max_pages * pool.at.page_size;
    if (threadIdx.x == 0) {
        // the first to take the length frees the pages
        if (pool.at.refused) pool.at.refused[slot] = 0;
        const int n = atomicExch(&pool.lengths[slot], 0);
        length = n <= 0 ? 0u : (unsigned)n < room ? (unsigned)n : room;
    }
    __syncthreads();
    const unsigned held = pages_for(length, pool.at.page_size);
    for (unsigned i = threadIdx.x; i < held; i += COPY) {
        int *const entry = pool.table + (size_t)slot * pool.at.max_pages + i;
        const int p = *entry;
        if (p < 0 || (unsigned)p >= pool.at.pages) atomicOr(pool.at.status, ASPEN_B200_CACHE_BAD_INDEX);
        else if (atomicSub(&pool.refs[p], 1) <= 0) {
            atomicAdd(&pool.refs[p], 1);
            atomicOr(pool.at.status, ASPEN_B200_CACHE_BAD_INDEX);
        }
        *entry = -1;
    }
}

__global__ void __launch_bounds__(BOOK) compact_kernel(const Pool pool, const Space w) {
    __shared__ unsigned sums[32];
    const unsigned pages = pool.at.pages;
    let_next_kernel_start();
    wait_for_previous_kernel();
    unsigned mine = 0, live;
    for (unsigned p0 = threadIdx.x; p0 < pages; p0 += BOOK * SCAN) {
        #pragma unroll
        for (unsigned i = 0; i < SCAN; i++) if (p0 + i * BOOK < pages) mine += pool.refs[p0 + i * BOOK] > 0;
    }
    before_me(mine, live, sums);
    // free pages below `live`, pages in use from there on: as many of the one as of the other
    unsigned holes = 0, movers = 0;
    for (unsigned p0 = 0; p0 < pages; p0 += BOOK * SCAN) {
        const unsigned first = p0 + threadIdx.x * SCAN;
        unsigned hole = 0, mover = 0;
        #pragma unroll
        for (unsigned i = 0; i < SCAN; i++) {
            const unsigned p = first + i;
            if (p >= pages) continue;
            const bool used = pool.refs[p] > 0;
            if (p < live && !used) hole |= 1u << i;
            if (p >= live) { w.mark[p] = (int)p; if (used) mover |= 1u << i; }
        }
        unsigned all, a = holes + before_me(__popc(hole), all, sums);
        holes += all;
        unsigned b = movers + before_me(__popc(mover), all, sums);
        movers += all;
        #pragma unroll
        for (unsigned i = 0; i < SCAN; i++) {
            if (hole >> i & 1u) w.to[a++] = (int)(first + i);
            if (mover >> i & 1u) w.from[b++] = (int)(first + i);
        }
    }
    __syncthreads();
    for (unsigned i = threadIdx.x; i < movers; i += BOOK) {
        const int a = w.from[i], b = w.to[i];
        pool.refs[b] = pool.refs[a];
        pool.refs[a] = 0;
        w.mark[a] = b;
    }
    if (threadIdx.x == 0) { w.head[COUNT] = (int)movers; w.head[LIVE] = (int)live; }
}

struct ListPair {
    const int *from, *to;
    unsigned page, pages;
    __device__ __forceinline__ bool operator()(unsigned i, int &a, int &b, unsigned &tokens) const {
        a = from[i];
        b = to[i];
        tokens = page;
        return a >= 0 && (unsigned)a < pages && b >= 0 && (unsigned)b < pages;
    }
};
__global__ void __launch_bounds__(COPY, COPY_CTAS) compact_copy_kernel(const Pool pool, const Space w, const Plane plane) {
    wait_for_previous_kernel();
    const unsigned live = (unsigned)w.head[LIVE], count = (unsigned)w.head[COUNT];
    if (!count) return;
    copy_pages(plane, count, ListPair{w.from, w.to, pool.at.page_size, pool.at.pages}, blockIdx.x, gridDim.x);
    const unsigned long long n = (unsigned long long)pool.at.sequences * pool.at.max_pages;
    for (unsigned long long i = (unsigned long long)blockIdx.x * COPY + threadIdx.x; i < n; i += (unsigned long long)gridDim.x * COPY) {
        const int p = pool.table[i];
        if (p >= 0 && (unsigned)p >= live && (unsigned)p < pool.at.pages && w.mark[p] != p) pool.table[i] = w.mark[p];
    }
}
__global__ void __launch_bounds__(COPY, COPY_CTAS) copy_kernel(const Pool pool, const Plane plane, const int *from, const int *to, unsigned count) {
    wait_for_previous_kernel();
    const ListPair pair{from, to, pool.at.page_size, pool.at.pages};
    for (unsigned i = blockIdx.x * COPY + threadIdx.x; i < count; i += gridDim.x * COPY) {
        int a, b;
        unsigned tokens;
        if (!pair(i, a, b, tokens)) atomicOr(pool.at.status, ASPEN_B200_CACHE_BAD_INDEX);
    }
    copy_pages(plane, count, pair, blockIdx.x, gridDim.x);
}

// Append: a warp writes the keys and values of one new token.
struct New {
    const uint4 *from[2];
    uint4 *to[2];
    size_t row[2], head[2];         // strides in vectors
    size_t to_head;
    const int *slots, *starts;
    unsigned entries, rows, heads, vectors;         // vectors: of a row of one head
};
__global__ void __launch_bounds__(COPY) append_kernel(const Pages at /* strides in vectors */, const New n) {
    const unsigned lane = threadIdx.x % 32, r = blockIdx.x * (COPY / 32) + threadIdx.x / 32;
    wait_for_previous_kernel();
    // behind an extend that was refused the last places of a sequence are not the new tokens'; without a list of such sequences that goes for all
    if (r >= n.rows || (!at.refused && *reinterpret_cast<volatile int *>(at.status) & ASPEN_B200_CACHE_REFUSED)) return;
    unsigned e = r;
    int begin = (int)r, end = (int)r + 1;
    if (n.starts) {
        // the last entry that starts at r or before: 32 probes a turn
        unsigned lo = 0, hi = n.entries;
        while (hi - lo > 1) {
            const unsigned step = (hi - lo + 31) / 32, i = lo + lane * step;
            const unsigned below = __ballot_sync(0xffffffffu, i < hi && n.starts[i] <= (int)r);
            const unsigned last = below ? 31 - __clz(below) : 0;
            lo += last * step;
            hi = min(hi, lo + step);
        }
        e = lo;
        begin = n.starts[e];
        end = n.starts[e + 1];
    }
    if (begin > (int)r || end <= (int)r) { if (lane == 0) atomicOr(at.status, ASPEN_B200_CACHE_BAD_INDEX); return; }
    const int slot = e >= n.entries ? -1 : n.slots ? n.slots[e] : (int)e;
    if (attn::is_refused(at, slot)) return;
    const long long position = (long long)attn::sequence_length(at, slot) - ((long long)end - r);
    const long long offset = position < 0 ? -1 : attn::token_offset(at, slot, (unsigned)position);
    if (offset < 0) { if (lane == 0) atomicOr(at.status, ASPEN_B200_CACHE_BAD_INDEX); return; }
    const unsigned per = n.heads * n.vectors;
    for (unsigned i = lane; i < per; i += 32) {
        const unsigned h = i / n.vectors, x = i - h * n.vectors;
        #pragma unroll
        for (int kv = 0; kv < 2; kv++) n.to[kv][(size_t)offset + h * n.to_head + x] = __ldg(n.from[kv] + r * n.row[kv] + h * n.head[kv] + x);
    }
}

Pool pool_of(const aspen_b200_cache_t &c) { return {attn::pages_of(c), c.page_table, c.lengths, c.refs}; }

Plane plane_of(const aspen_b200_cache_t &c) {
    const Pages at = attn::pages_of(c);
    const size_t per = 16 / attn::type_size(c.type);
    Plane p;
    p.base[0] = static_cast<uint4 *>(c.k);
    p.base[1] = static_cast<uint4 *>(c.v);
    p.token = at.token_stride / per;
    p.head = at.head_stride / per;
    p.page = at.page_stride / per;
    p.layer = attn::packed(c.layer_stride, at.page_stride * c.pages) / per;
    p.layers = c.layers;
    p.heads = c.kv_heads;
    p.page_size = c.page_size;
    p.row = (unsigned)(c.head_dim / per);
    p.dense = p.token == p.row && p.head == p.token * p.page_size;
    return p;
}

int done(cudaError_t err, const char *what) {
    if (err == cudaSuccess) return 0;
    cudaGetLastError();
    ASPEN_ERR("%s: %s\n", what, cudaGetErrorString(err));
    return -3;
}

int check_space(const aspen_b200_cache_t *c, unsigned entries, const void *workspace, size_t bytes, const char *what) {
    if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 4) { ASPEN_ERR("%s: no workspace, or not on a 4-byte boundary\n", what); return -1; }
    const size_t need = space_ints(*c, entries) * sizeof(int);
    if (bytes < need) { ASPEN_ERR("%s: a workspace of %zu bytes; %zu are needed\n", what, bytes, need); return -1; }
    return 0;
}
int check_entries(unsigned entries, const char *what) {
    if (entries > 0x7fffffffu) { ASPEN_ERR("%s: %u entries\n", what, entries); return -2; }
    return 0;
}

}  // namespace

extern "C" size_t aspen_b200_cache_workspace(const aspen_b200_cache_t *cache, unsigned int entries) {
    const char *what = "aspen_b200_cache_workspace";
    if (attn::check_cache(cache, what, true) || check_entries(entries, what)) return 0;
    return space_ints(*cache, entries) * sizeof(int);
}

extern "C" int aspen_b200_cache_extend(const aspen_b200_cache_t *cache, const int *slots, const int *starts, unsigned int entries, void *workspace,
                                       size_t workspace_bytes, void *cuda_stream) {
    const char *what = "aspen_b200_cache_extend";
    int rc = attn::check_cache(cache, what, true);
    if (!rc) rc = check_entries(entries, what);
    if (!rc) rc = check_space(cache, entries, workspace, workspace_bytes, what);
    if (rc || !entries) return rc;
    const attn::Named ints[] = {{slots, "slots"}, {starts, "starts"}};
    if ((rc = attn::check_ints(ints, 2, what))) return rc;
    const attn::Named all[] = {{cache->page_table, "page_table"}, {cache->lengths, "lengths"}, {cache->refs, "refs"}, {cache->status, "status"},
                               {slots, "slots"}, {starts, "starts"}, {workspace, "workspace"}, {cache->refused, "refused"}};
    if ((rc = attn::check_device(all, 8, what))) return rc;
    return done(launch_early(extend_kernel, 1, BOOK, 0, static_cast<cudaStream_t>(cuda_stream), pool_of(*cache), space_of(*cache, entries, workspace), slots, starts, entries), what);
}

extern "C" int aspen_b200_cache_append(const aspen_b200_cache_t *cache, unsigned int layer, const aspen_b200_append_t *a, void *cuda_stream) {
    const char *what = "aspen_b200_cache_append";
    int rc = attn::check_cache(cache, what, false);
    if (rc) return rc;
    if (!a) { ASPEN_ERR("%s: no rows\n", what); return -1; }
    if (layer >= cache->layers) { ASPEN_ERR("%s: layer %u of %u\n", what, layer, cache->layers); return -1; }
    if ((rc = check_entries(a->entries, what)) || (rc = check_entries(a->rows, what))) return rc;
    if (!a->rows) return 0;
    if (!a->entries || (!a->starts && a->rows != a->entries)) { ASPEN_ERR("%s: %u rows of %u sequences\n", what, a->rows, a->entries); return -1; }
    const size_t row = (size_t)cache->kv_heads * cache->head_dim;
    if ((rc = attn::check_rows(a->k, a->k_row_stride, a->k_head_stride, cache->type, "k", what)) ||
        (rc = attn::check_rows(a->v, a->v_row_stride, a->v_head_stride, cache->type, "v", what))) return rc;
    const attn::Named ints[] = {{a->slots, "slots"}, {a->starts, "starts"}};
    if ((rc = attn::check_ints(ints, 2, what))) return rc;
    const attn::Named all[] = {{cache->k, "the cache's k"}, {cache->v, "the cache's v"}, {cache->page_table, "page_table"}, {cache->lengths, "lengths"}, {cache->status, "status"},
                               {a->k, "k"}, {a->v, "v"}, {a->slots, "slots"}, {a->starts, "starts"}, {cache->refused, "refused"}};
    if ((rc = attn::check_device(all, 10, what))) return rc;
    const Plane p = plane_of(*cache);
    const size_t per = 16 / attn::type_size(cache->type);
    Pages at = attn::pages_of(*cache);
    at.page_stride /= per; at.head_stride /= per; at.token_stride /= per;
    New n;
    n.from[0] = static_cast<const uint4 *>(a->k);
    n.from[1] = static_cast<const uint4 *>(a->v);
    n.to[0] = p.base[0] + layer * p.layer;
    n.to[1] = p.base[1] + layer * p.layer;
    n.row[0] = attn::packed(a->k_row_stride, row) / per;
    n.row[1] = attn::packed(a->v_row_stride, row) / per;
    n.head[0] = attn::packed(a->k_head_stride, cache->head_dim) / per;
    n.head[1] = attn::packed(a->v_head_stride, cache->head_dim) / per;
    n.to_head = p.head;
    n.slots = a->slots;
    n.starts = a->starts;
    n.entries = a->entries;
    n.rows = a->rows;
    n.heads = cache->kv_heads;
    n.vectors = p.row;
    return done(launch_early(append_kernel, (a->rows + COPY / 32 - 1) / (COPY / 32), COPY, 0, static_cast<cudaStream_t>(cuda_stream), at, n), what);
}

extern "C" int aspen_b200_cache_fork(const aspen_b200_cache_t *cache, const int *from, const int *to, unsigned int entries, void *workspace, size_t workspace_bytes,
                                     void *cuda_stream) {
    const char *what = "aspen_b200_cache_fork";
    int rc = attn::check_cache(cache, what, true);
    if (!rc) rc = check_entries(entries, what);
    if (!rc) rc = check_space(cache, entries, workspace, workspace_bytes, what);
    if (rc || !entries) return rc;
    if (!from || !to) { ASPEN_ERR("%s: no list of sequences\n", what); return -1; }
    const attn::Named ints[] = {{from, "from"}, {to, "to"}};
    if ((rc = attn::check_ints(ints, 2, what))) return rc;
    const attn::Named all[] = {{cache->k, "the cache's k"}, {cache->v, "the cache's v"}, {cache->page_table, "page_table"}, {cache->lengths, "lengths"}, {cache->refs, "refs"},
                               {cache->status, "status"}, {from, "from"}, {to, "to"}, {workspace, "workspace"}, {cache->refused, "refused"}};
    if ((rc = attn::check_device(all, 10, what))) return rc;
    const int sms = attn::sm_count(what);
    if (sms < 0) return sms;
    const cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
    const Pool pool = pool_of(*cache);
    const Space w = space_of(*cache, entries, workspace);
    if ((rc = done(launch_early(fork_kernel, 1, BOOK, 0, stream, pool, w, from, to, entries), what))) return rc;
    return done(launch_early(fork_copy_kernel, (unsigned)sms * COPY_CTAS, COPY, 0, stream, pool, w, plane_of(*cache), from, to, entries), what);
}

extern "C" int aspen_b200_cache_free(const aspen_b200_cache_t *cache, const int *slots, unsigned int entries, void *cuda_stream) {
    const char *what = "aspen_b200_cache_free";
    int rc = attn::check_cache(cache, what, true);
    if (!rc) rc = check_entries(entries, what);
    if (rc || !entries) return rc;
    if (!slots) { ASPEN_ERR("%s: no list of sequences\n", what); return -1; }
    const attn::Named ints[] = {{slots, "slots"}};
    if ((rc = attn::check_ints(ints, 1, what))) return rc;
    const attn::Named all[] = {{cache->page_table, "page_table"}, {cache->lengths, "lengths"}, {cache->refs, "refs"}, {cache->status, "status"}, {slots, "slots"}, {cache->refused, "refused"}};
    if ((rc = attn::check_device(all, 6, what))) return rc;
    return done(launch_early(free_kernel, entries, COPY, 0, static_cast<cudaStream_t>(cuda_stream), pool_of(*cache), slots), what);
}

extern "C" int aspen_b200_cache_compact(const aspen_b200_cache_t *cache, void *workspace, size_t workspace_bytes, void *cuda_stream) {
    const char *what = "aspen_b200_cache_compact";
    int rc = attn::check_cache(cache, what, true);
    if (!rc) rc = check_space(cache, 0, workspace, workspace_bytes, what);
    if (rc) return rc;
    const attn::Named all[] = {{cache->k, "the cache's k"}, {cache->v, "the cache's v"}, {cache->page_table, "page_table"}, {cache->refs, "refs"}, {workspace, "workspace"}};
    if ((rc = attn::check_device(all, 5, what))) return rc;
    const int sms = attn::sm_count(what);
    if (sms < 0) return sms;
    const cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
    const Pool pool = pool_of(*cache);
    const Space w = space_of(*cache, 0, workspace);
    if ((rc = done(launch_early(compact_kernel, 1, BOOK, 0, stream, pool, w), what))) return rc;
    return done(launch_early(compact_copy_kernel, (unsigned)sms * COPY_CTAS, COPY, 0, stream, pool, w, plane_of(*cache)), what);
}

extern "C" int aspen_b200_cache_copy(const aspen_b200_cache_t *cache, const int *from, const int *to, unsigned int count, void *cuda_stream) {
    const char *what = "aspen_b200_cache_copy";
    int rc = attn::check_cache(cache, what, false);
    if (!rc) rc = check_entries(count, what);
    if (rc || !count) return rc;
    if (!from || !to) { ASPEN_ERR("%s: no list of pages\n", what); return -1; }
    const attn::Named ints[] = {{from, "from"}, {to, "to"}};
    if ((rc = attn::check_ints(ints, 2, what))) return rc;
    const attn::Named all[] = {{cache->k, "the cache's k"}, {cache->v, "the cache's v"}, {cache->status, "status"}, {from, "from"}, {to, "to"}};
    if ((rc = attn::check_device(all, 5, what))) return rc;
    const int sms = attn::sm_count(what);
    if (sms < 0) return sms;
    return done(launch_early(copy_kernel, (unsigned)sms * COPY_CTAS, COPY, 0, static_cast<cudaStream_t>(cuda_stream), pool_of(*cache), plane_of(*cache), from, to, count), what);
}
