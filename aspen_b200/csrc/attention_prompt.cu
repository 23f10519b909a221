// Attention over whole prompts, packed one behind the other.
//
// One pass over the keys of a block of queries, with the running maximum and sum of the softmax; scores never leave the SM.
//
// prompt_tiles (16 bits, up to 128 features) and prompt_parts (fp32, up to 64): tcgen05, two tiles of 128 rows to a CTA, warps with a role each; attention_tc.cuh has the plan, what
// bounds it and what it measured.
//
// prompt_rows (what is left: wider heads, scales that are not positive, short sequences, few rows over many keys): a warp has 16 queries, its operands and sums in registers as mma.sync takes them (mma_sync.cuh);
// keys and values of a tile go through shared memory for the four warps of a CTA, asked for one tile ahead.  Rows in shared memory are 64 (keys) and 16 bytes (values) longer than a
// power of two, so that the 16-byte pieces that eight lanes read together lie in different banks.  It is bounded by the instructions around mma.sync (fp32: splitting) and, with one block to a
// sequence, by its chain of loads, products and exp2: 12 heads of 64, one prompt of 37 tokens in fp32 9 us with the call, 32 prompts of 100 tokens in bf16 12 us (8 of 512 in fp32 92 us,
// prompt_parts 33; 24 of up to 1024 in bf16 101 us, prompt_tiles 46.5); 8 of 512 with heads of 128 in fp32 194 us.
// Where there are few blocks, the CTAs of a cluster walk the tiles of one in turn and join maxima, sums and values through each other's shared memory, in the order of their ranks: 8 heads of 128,
// one query over 30000 keys in bf16 108 us instead of 392 (prompt_tiles), 4 queries of 12 heads of 64 over 2004 keys in fp32 19 instead of 75 (prompt_parts).
#include "attention_tc.cuh"
#include "early_launch.cuh"
#include "gemm_split.cuh"
#include "index_div.h"
#include "mma_sync.cuh"

namespace {

struct Args {
    const char *q, *k, *v;
    char *out;
    const int *q_starts, *kv_starts;
    unsigned q_row, q_head, k_row, k_head, v_row, v_head, out_row, out_head;    // in elements, below 2^29
    unsigned sequences, q_rows, kv_rows, heads, group, head_dim;
    unsigned part;                      // of 2^16 that is one over the group, rounded up: r / group = r * part >> 16 for r and group up to 128
    unsigned block;                     // 128 / group
    unsigned in_a_row;                  // blocks of a CTA of prompt_rows
    Divisor by_block;
    int masked;
    float scale;                        // with log2(e)
    int *status;                        // or nullptr
};

// A block of queries: rows first ... of the sequence that begins at row q0.
struct Block {
    int q0, queries, k0, keys, first;
};

__device__ __forceinline__ int clamped(const int *starts, unsigned i, unsigned rows) { return min(max(starts[i], 0), (int)rows); }

// Piece `index` of all sequences, `pieces(queries)` of one, counted from the first sequence; a sequence's last one first, because with a mask it has most keys.
// Every warp finds it for itself, 32 sequences a turn.  Returns the piece's number in its sequence, -1: there are not so many.
struct Place { unsigned sequence = 0; unsigned long long before = 0; };       // where a search ended: at 32 sequences, and the pieces before them
template <typename Pieces>
__device__ __forceinline__ int find_piece(const Args &a, unsigned index, Place &from, const Pieces &pieces, int &q_first, int &queries, int &k_first, int &keys) {
    const unsigned lane = threadIdx.x % 32;
    if (index < from.before) from = Place();
    for (; from.sequence < a.sequences; from.sequence += 32) {
        const unsigned s = from.sequence + lane;
        int q0 = 0, q1 = 0;
        if (s < a.sequences) { q0 = clamped(a.q_starts, s, a.q_rows); q1 = max(q0, clamped(a.q_starts, s + 1, a.q_rows)); }
        const unsigned n = pieces((unsigned)(q1 - q0));
        unsigned long long sum = n;
        #pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const unsigned long long u = __shfl_up_sync(0xffffffffu, sum, o); if (lane >= (unsigned)o) sum += u; }
        const unsigned here = __ballot_sync(0xffffffffu, from.before + sum > index);
        if (here) {
            const int at = __ffs(here) - 1;
            const unsigned rank = (unsigned)(from.before + sum - 1 - index);      // of lane `at`: n - 1 for the first index of its sequence, 0 for the last
            q_first = __shfl_sync(0xffffffffu, q0, at);
            queries = __shfl_sync(0xffffffffu, q1, at) - q_first;
            const unsigned mine = from.sequence + at;
            k_first = clamped(a.kv_starts, mine, a.kv_rows);
            keys = max(0, clamped(a.kv_starts, mine + 1, a.kv_rows) - k_first);
            return (int)__shfl_sync(0xffffffffu, rank, at);
        }
        from.before += __shfl_sync(0xffffffffu, sum, 31);
    }
    return -1;
}
__device__ __forceinline__ bool find_block(const Args &a, unsigned index, Place &from, unsigned size, Block &b) {
    const int i = find_piece(a, index, from, [=](unsigned queries) { return (queries + size - 1) / size; }, b.q0, b.queries, b.k0, b.keys);
    b.first = i * (int)size;
    return i >= 0;
}

__device__ __forceinline__ unsigned shared_address(const void *p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(unsigned to, const char *from, bool ok) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT> __device__ __forceinline__ void wait_copies() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

// A cluster's CTAs: how many, a wait for all of them, and a value that one of them has in shared memory where this one has `at`.
__device__ __forceinline__ unsigned cluster_size() { unsigned n; asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(n)); return n; }
__device__ __forceinline__ void cluster_barrier() { asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ float load_of_rank(unsigned at, unsigned rank) {
    float v;
    asm volatile("{\n\t.reg .u32 x;\n\tmapa.shared::cluster.u32 x, %1, %2;\n\tld.shared::cluster.f32 %0, [x];\n\t}" : "=f"(v) : "r"(at), "r"(rank) : "memory");
    return v;
}

template <int TYPE, int DIM>
struct Rows {
    static constexpr int SIZE = TYPE == ASPEN_B200_FP32 ? 4 : 2, VALUES = 16 / SIZE, BYTES = DIM * SIZE;
    static constexpr int QUERIES = 64, THREADS = 128;
    // fp32 rows of 512 bytes: tiles of 32 keys leave room for two CTAs on an SM (8 prompts of 512 tokens, 12 heads of 128: 207 us, 287 with 64); 16-bit ones of 512 take 64 (24 us, 30)
    static constexpr int KEYS = SIZE == 4 && BYTES >= 512 ? 32 : 64;
    static constexpr int KPITCH = BYTES + 64, VPITCH = BYTES + 16, STAGE = KEYS * (KPITCH + VPITCH);
    static constexpr bool HELD = BYTES <= 256;                  // queries stay in registers
    static constexpr int SMEM = 2 * STAGE + (HELD ? 0 : QUERIES * KPITCH);
    static constexpr int PIECES = DIM / (4 * VALUES);           // of a lane and row, product over features
    static constexpr int VPIECES = DIM / (8 * VALUES);
    // Pieces of the product over features in a turn of its loop.  fp32 that reads its queries again takes one: all of them spill registers and are more code than is fetched in time
    // (the 8 prompts 197 us instead of 207, 4 of 300 tokens with 8 heads of 256 106 instead of 129); 16 bits are faster with all (24 us, 26).
    static constexpr int TURN = HELD || SIZE == 2 ? PIECES : 1;
};

// How a CTA has its work: a block of queries; with the CTAs of a cluster, which walk a block's tiles in turn and join what they have; several blocks one after the other.
enum { ALONE, SHARED, IN_A_ROW };
template <int TYPE, int DIM, int WORK>
__global__ void __launch_bounds__(128) prompt_rows(const Args a) {
    typedef Rows<TYPE, DIM> R;
    constexpr int SIZE = R::SIZE, VALUES = R::VALUES, KT = R::KEYS / 8;
    constexpr bool SPLIT = WORK == SHARED;
    extern __shared__ __align__(128) char smem[];
    const unsigned lane = threadIdx.x % 32, warp = threadIdx.x / 32, g = lane >> 2, t = lane & 3, head = blockIdx.y, kv_head = head / a.group;
    attn::wait_for_previous_kernel();
    const unsigned ranks = SPLIT ? cluster_size() : 1u, rank = SPLIT ? blockIdx.x % ranks : 0u;
    Place from;
    #pragma unroll 1
    for (unsigned n = 0; n < (WORK == IN_A_ROW ? a.in_a_row : 1u); n++) {
        Block b;
        if (!find_block(a, WORK == IN_A_ROW ? blockIdx.x * a.in_a_row + n : blockIdx.x / ranks, from, R::QUERIES, b)) return;
        const int behind = b.keys - b.queries;                      // query i sees keys up to i + behind
        const int last = min(b.queries, b.first + R::QUERIES) - 1;
        const int end = a.masked ? min(b.keys, last + behind + 1) : b.keys;
        const int row0 = b.first + (int)warp * 16 + (int)g, row8 = row0 + 8;
        const char *const k = a.k + ((size_t)b.k0 * a.k_row + (size_t)kv_head * a.k_head) * SIZE, *const v = a.v + ((size_t)b.k0 * a.v_row + (size_t)kv_head * a.v_head) * SIZE;
        auto fetch = [&](int tile, int stage) {
            char *const at = smem + stage * R::STAGE;
            constexpr int PER_ROW = R::BYTES / 16;
            #pragma unroll 4
            for (int i = threadIdx.x; i < R::KEYS * PER_ROW; i += R::THREADS) {
                const int r = i / PER_ROW, x = i % PER_ROW, j = tile * R::KEYS + r;
                const bool ok = j < end && x * VALUES < (int)a.head_dim;
                copy16(shared_address(at + r * R::KPITCH + x * 16), k + (ok ? ((size_t)j * a.k_row + x * VALUES) * SIZE : 0), ok);
                copy16(shared_address(at + R::KEYS * R::KPITCH + r * R::VPITCH + x * 16), v + (ok ? ((size_t)j * a.v_row + x * VALUES) * SIZE : 0), ok);
            }
            copies_done();
        };
        const int tiles = end > 0 ? (end + R::KEYS - 1) / R::KEYS : 0;
        if ((int)rank < tiles) fetch((int)rank, 0);
        // queries, rows g and g + 8 of the warp's 16
        const char *const q = a.q + ((size_t)b.q0 * a.q_row + (size_t)head * a.q_head) * SIZE;
        char *const own = smem + 2 * R::STAGE + warp * 16 * R::KPITCH;
        uint4 held[R::HELD ? R::PIECES * 2 : 1];
        #pragma unroll
        for (int i = 0; i < R::PIECES; i++)
            #pragma unroll
            for (int h = 0; h < 2; h++) {
                const int row = h ? row8 : row0;
                const unsigned f = i * 4 * VALUES + t * VALUES;
                uint4 x = make_uint4(0u, 0u, 0u, 0u);
                if (row < b.queries && f < a.head_dim) x = __ldg(reinterpret_cast<const uint4 *>(q + ((size_t)row * a.q_row + f) * SIZE));
                if (R::HELD) held[2 * i + h] = x;
                else *reinterpret_cast<uint4 *>(own + (g + 8 * h) * R::KPITCH + f * SIZE) = x;
            }
        __syncwarp();
        float o[DIM / 8][4], max[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
        #pragma unroll
        for (int i = 0; i < DIM / 8; i++)
            #pragma unroll
            for (int j = 0; j < 4; j++) o[i][j] = 0.f;
        for (int tile = (int)rank, stage = 0; tile < tiles; tile += (int)ranks, stage ^= 1) {
            if (tile + (int)ranks < tiles) { fetch(tile + (int)ranks, stage ^ 1); wait_copies<1>(); } else wait_copies<0>();
            __syncthreads();
            const char *const ks = smem + stage * R::STAGE, *const vs = ks + R::KEYS * R::KPITCH;
            float s[KT][4];
            #pragma unroll
            for (int n = 0; n < KT; n++)
                #pragma unroll
                for (int j = 0; j < 4; j++) s[n][j] = 0.f;
            #pragma unroll R::TURN
            for (int i = 0; i < R::PIECES; i++) {
                const int f = (i * 4 * VALUES + t * VALUES) * SIZE;
                const uint4 x = R::HELD ? held[R::HELD ? 2 * i : 0] : *reinterpret_cast<const uint4 *>(own + g * R::KPITCH + f);
                const uint4 y = R::HELD ? held[R::HELD ? 2 * i + 1 : 0] : *reinterpret_cast<const uint4 *>(own + (g + 8) * R::KPITCH + f);
                #pragma unroll
                for (int n = 0; n < KT; n++) {
                    const uint4 w = *reinterpret_cast<const uint4 *>(ks + (n * 8 + g) * R::KPITCH + f);
                    if constexpr (TYPE == ASPEN_B200_FP32) {
                        // sums of 16 features are added outside: the tensor cores cut off what they add to a sum
                        const unsigned a0[4] = {x.x, y.x, x.y, y.y}, a1[4] = {x.z, y.z, x.w, y.w}, b0[2] = {w.x, w.y}, b1[2] = {w.z, w.w};
                        float part[4] = {0.f, 0.f, 0.f, 0.f};
                        mma::tf32x3(part, a0, b0);
                        mma::tf32x3(part, a1, b1);
                        #pragma unroll
                        for (int j = 0; j < 4; j++) s[n][j] += part[j];
                    } else {
                        mma::Of<TYPE>::step(s[n], x.x, y.x, x.y, y.y, w.x, w.y);
                        mma::Of<TYPE>::step(s[n], x.z, y.z, x.w, y.w, w.z, w.w);
                    }
                }
            }
            // columns 2 t and 2 t + 1 of each eight keys; rows g and g + 8
            const int j0 = tile * R::KEYS + 2 * (int)t;
            const int see0 = a.masked ? min(end, row0 + behind + 1) : end, see8 = a.masked ? min(end, row8 + behind + 1) : end;      // first key that is not seen
            float m[2] = {max[0], max[1]};
            #pragma unroll
            for (int n = 0; n < KT; n++)
                #pragma unroll
                for (int j = 0; j < 4; j++) {
                    s[n][j] = j0 + n * 8 + (j & 1) < (j < 2 ? see0 : see8) ? s[n][j] * a.scale : -INFINITY;
                    m[j / 2] = fmaxf(m[j / 2], s[n][j]);
                }
            float down[2], ref[2];
            #pragma unroll
            for (int h = 0; h < 2; h++) {
                m[h] = fmaxf(m[h], __shfl_xor_sync(0xffffffffu, m[h], 1));
                m[h] = fmaxf(m[h], __shfl_xor_sync(0xffffffffu, m[h], 2));
                ref[h] = m[h] == -INFINITY ? 0.f : m[h];
                down[h] = mma::exp2_fast(max[h] - ref[h]);
                ref[h] -= mma::Of<TYPE>::TOP;
                max[h] = m[h];
                sum[h] *= down[h];
            }
            #pragma unroll
            for (int n = 0; n < KT; n++)
                #pragma unroll
                for (int j = 0; j < 4; j++) { s[n][j] = mma::exp2_fast(s[n][j] - ref[j / 2]); sum[j / 2] += s[n][j]; }
            if (__any_sync(0xffffffffu, down[0] != 1.f || down[1] != 1.f)) {
                #pragma unroll
                for (int i = 0; i < DIM / 8; i++)
                    #pragma unroll
                    for (int j = 0; j < 4; j++) o[i][j] *= down[j / 2];
            }
            if constexpr (TYPE == ASPEN_B200_FP32) {
                #pragma unroll
                for (int i = 0; i < R::VPIECES; i++) {
                    float part[4][4];
                    #pragma unroll
                    for (int j = 0; j < 16; j++) part[j / 4][j % 4] = 0.f;
                    #pragma unroll
                    for (int n = 0; n < KT; n++) {
                        const unsigned p[4] = {__float_as_uint(s[n][0]), __float_as_uint(s[n][2]), __float_as_uint(s[n][1]), __float_as_uint(s[n][3])};
                        const char *const row = vs + (n * 8 + 2 * t) * R::VPITCH + (i * 32 + g * 4) * SIZE;
                        const uint4 x = *reinterpret_cast<const uint4 *>(row), y = *reinterpret_cast<const uint4 *>(row + R::VPITCH);
                        const unsigned w0[4] = {x.x, x.y, x.z, x.w}, w1[4] = {y.x, y.y, y.z, y.w};
                        #pragma unroll
                        for (int j = 0; j < 4; j++) { const unsigned w[2] = {w0[j], w1[j]}; mma::tf32x3(part[j], p, w); }
                    }
                    #pragma unroll
                    for (int j = 0; j < 16; j++) o[i * 4 + j / 4][j % 4] += part[j / 4][j % 4];
                }
            } else {
                typedef mma::Of<TYPE> T;
                #pragma unroll
                for (int n = 0; n < KT; n += 2) {
                    const unsigned p0 = T::pack(s[n][0], s[n][1]), p1 = T::pack(s[n][2], s[n][3]), p2 = T::pack(s[n + 1][0], s[n + 1][1]), p3 = T::pack(s[n + 1][2], s[n + 1][3]);
                    const char *const row = vs + (n * 8 + 2 * t) * R::VPITCH;
                    #pragma unroll
                    for (int i = 0; i < R::VPIECES; i++) {
                        const char *const at = row + (i * 64 + g * 8) * SIZE;
                        const uint4 x0 = *reinterpret_cast<const uint4 *>(at), x1 = *reinterpret_cast<const uint4 *>(at + R::VPITCH);
                        const uint4 x8 = *reinterpret_cast<const uint4 *>(at + 8 * R::VPITCH), x9 = *reinterpret_cast<const uint4 *>(at + 9 * R::VPITCH);
                        const unsigned w0[4] = {x0.x, x0.y, x0.z, x0.w}, w1[4] = {x1.x, x1.y, x1.z, x1.w}, w8[4] = {x8.x, x8.y, x8.z, x8.w}, w9[4] = {x9.x, x9.y, x9.z, x9.w};
                        #pragma unroll
                        for (int j = 0; j < 8; j++)
                            T::step(o[i * 8 + j], p0, p1, p2, p3, mma::pair_of(w0[j / 2], w1[j / 2], j & 1), mma::pair_of(w8[j / 2], w9[j / 2], j & 1));
                    }
                }
            }
            __syncthreads();
        }
        #pragma unroll
        for (int h = 0; h < 2; h++) {
            sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
            sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
        }
        // column n = 2 t + c of tile j holds the value j of piece n
        constexpr int PER = TYPE == ASPEN_B200_FP32 ? 4 : 8;
        auto store = [&](int h, int c, int i, const float *x) {
            const int row = h ? row8 : row0;
            const unsigned f = i * 8 * PER + (2 * t + c) * PER;
            if (row >= b.queries || f >= a.head_dim) return;
            char *const out = a.out + ((size_t)(b.q0 + row) * a.out_row + (size_t)head * a.out_head + f) * SIZE;
            if constexpr (TYPE == ASPEN_B200_FP32) *reinterpret_cast<float4 *>(out) = make_float4(x[0], x[1], x[2], x[3]);
            else {
                typedef mma::Of<TYPE> T;
                *reinterpret_cast<uint4 *>(out) = make_uint4(T::pack(x[0], x[1]), T::pack(x[2], x[3]), T::pack(x[4], x[5]), T::pack(x[6], x[7]));
            }
        };
        if constexpr (!SPLIT) {
            #pragma unroll
            for (int h = 0; h < 2; h++) {
                const float inv = sum[h] == 0.f ? 0.f : 1.f / sum[h];
                #pragma unroll
                for (int i = 0; i < R::VPIECES; i++)
                    #pragma unroll
                    for (int c = 0; c < 2; c++) {
                        float x[PER];
                        #pragma unroll
                        for (int j = 0; j < PER; j++) x[j] = o[i * PER + j][2 * h + c] * inv;
                        store(h, c, i, x);
                    }
            }
        } else {
            // [value of a thread][thread]; a thread joins every `ranks`-th piece of its own place
            float *const mine = reinterpret_cast<float *>(smem) + threadIdx.x;
            constexpr int STATS = DIM / 8 * 4;
            static_assert((STATS + 4) * R::THREADS * 4 <= 2 * R::STAGE, "in place of keys and values");
            #pragma unroll
            for (int i = 0; i < DIM / 8; i++)
                #pragma unroll
                for (int j = 0; j < 4; j++) mine[(i * 4 + j) * R::THREADS] = o[i][j];
            #pragma unroll
            for (int h = 0; h < 2; h++) { mine[(STATS + h) * R::THREADS] = max[h]; mine[(STATS + 2 + h) * R::THREADS] = sum[h]; }
            cluster_barrier();
            const unsigned at = shared_address(mine);
            for (unsigned q = rank; q < 4 * R::VPIECES; q += ranks) {
                const int h = (int)(q & 1u), c = (int)(q >> 1 & 1u), i = (int)(q >> 2);
                float most = -INFINITY, all = 0.f, x[PER];
                #pragma unroll
                for (int j = 0; j < PER; j++) x[j] = 0.f;
                for (unsigned r = 0; r < ranks; r++) most = fmaxf(most, load_of_rank(at + (STATS + h) * R::THREADS * 4, r));
                const float ref = most == -INFINITY ? 0.f : most;
                for (unsigned r = 0; r < ranks; r++) {
                    const float w = mma::exp2_fast(load_of_rank(at + (STATS + h) * R::THREADS * 4, r) - ref);
                    all = fmaf(w, load_of_rank(at + (STATS + 2 + h) * R::THREADS * 4, r), all);
                    #pragma unroll
                    for (int j = 0; j < PER; j++) x[j] = fmaf(w, load_of_rank(at + ((i * PER + j) * 4 + 2 * h + c) * R::THREADS * 4, r), x[j]);
                }
                const float inv = all == 0.f ? 0.f : 1.f / all;
                #pragma unroll
                for (int j = 0; j < PER; j++) x[j] *= inv;
                store(h, c, i, x);
            }
            cluster_barrier();                          // the others have read what is here
        }
    }
}

// CTAs to a block.  Few blocks leave SMs without work; up to 8 CTAs share a block's keys then, 128 or more each, as long as all of them run at once.  An SM has room for two, heads of 256
// features for one.  Wide fp32 heads with a mask take two rounds of CTAs: their last blocks have twice the keys of the mean (one prompt of 549 tokens, 21 heads of 128, 84 us instead of 112; bf16
// heads of 256, two of 400 tokens, take 37 instead of 24).  Keys by the mean of the sequences: a long one among many short ones is walked by one CTA a block, since lengths are on the device.
unsigned blocks_of(const Args &a) { return a.q_rows / 64 + (a.sequences < a.q_rows ? a.sequences : a.q_rows); }
unsigned ranks_of(const Args &a, int type, unsigned sms) {
    const unsigned long long blocks = (unsigned long long)blocks_of(a) * a.heads, rounds = type == ASPEN_B200_FP32 && a.head_dim > 64 && a.masked ? 2 : 1, room = a.head_dim <= 128 ? 2 * sms * rounds : sms;
    const unsigned keys = a.kv_rows / a.sequences;
    unsigned ranks = 1;
    while (ranks < 8 && blocks * ranks * 2 <= room && keys >= ranks * 256) ranks *= 2;
    return ranks;
}
// Blocks in a row of a CTA.  It looks for its first one from the first sequence on, 32 a turn, and goes on from there; with a CTA to a block the search is quadratic in the number of sequences
// (20000 of 5 tokens, 12 fp32 heads of 128, 7.3 ms instead of 103; 4000 of one token, 12 bf16 heads of 64, 0.42 instead of 1.9; 300 of 10 45 us instead of 50).  Eight CTAs to an SM: 16 7.7 ms, 4 7.2
// but 4000 of 30 tokens 2.0 instead of 1.6.
unsigned in_a_row_of(const Args &a, unsigned sms) {
    const unsigned long long ctas = (unsigned long long)blocks_of(a) * a.heads;
    return a.sequences > 128 && ctas > 8 * sms ? (unsigned)(ctas / (8 * sms)) : 1u;
}
template <int TYPE, int DIM>
cudaError_t launch_rows(const Args &a, unsigned ranks, cudaStream_t stream) {
    typedef Rows<TYPE, DIM> R;
    static_assert(R::QUERIES == 64 && R::SMEM <= (DIM <= 128 ? 112 : 226) * 1024, "as blocks_of and ranks_of have it");
    void (*const kernel)(Args) = ranks > 1 ? prompt_rows<TYPE, DIM, SHARED> : a.in_a_row > 1 ? prompt_rows<TYPE, DIM, IN_A_ROW> : prompt_rows<TYPE, DIM, ALONE>;
    cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, R::SMEM);
    if (err != cudaSuccess) return err;
    return attn::launch_early_in_clusters(ranks, kernel, dim3((blocks_of(a) + a.in_a_row - 1) / a.in_a_row * ranks, a.heads), R::THREADS, R::SMEM, stream, a);
}
template <int TYPE>
cudaError_t launch_rows(const Args &a, unsigned ranks, cudaStream_t stream) {
    return a.head_dim <= 64 ? launch_rows<TYPE, 64>(a, ranks, stream) : a.head_dim <= 128 ? launch_rows<TYPE, 128>(a, ranks, stream) : launch_rows<TYPE, 256>(a, ranks, stream);
}

// ---- tcgen05 (attention_tc.cuh) ----

// Finds the jobs of a call: job `index` is two neighbouring tiles of a sequence and a head of keys.  With a mask the keys of a tile go by its number, so pairs of tiles are counted not
// sequence by sequence but from the highest number down: heavy work comes first, whatever sequence it is of, and light work fills the ends (8 prompts of 512 tokens: 7 tiles on the busiest
// SM instead of 10).  For up to 128 sequences, whose numbers of pairs a warp keeps, four a lane.
struct Finder {
    unsigned n[4], most;
    bool levelled;
    Place place;
    static __device__ __forceinline__ unsigned pairs(const Args &a, unsigned queries) { return (div_by(queries + a.block - 1, a.by_block) + 1) / 2; }
    __device__ __forceinline__ Finder(const Args &a) : most(0), levelled(a.masked && a.sequences <= 128) {
        if (!levelled) return;
        #pragma unroll
        for (unsigned k = 0; k < 4; k++) {
            const unsigned s = threadIdx.x % 32 * 4 + k;
            n[k] = s < a.sequences ? pairs(a, (unsigned)max(0, clamped(a.q_starts, s + 1, a.q_rows) - clamped(a.q_starts, s, a.q_rows))) : 0u;
            most = max(most, n[k]);
        }
        most = __reduce_max_sync(0xffffffffu, most);
    }
    // pairs numbered `level` and above
    __device__ __forceinline__ unsigned from(unsigned level) const {
        unsigned x = 0;
        #pragma unroll
        for (unsigned k = 0; k < 4; k++) x += n[k] > level ? n[k] - level : 0u;
        return __reduce_add_sync(0xffffffffu, x);
    }
    // The pair's number in its sequence, -1: there is none.
    __device__ __forceinline__ int by_level(const Args &a, unsigned index, fused::Job &job) const {
        if (index >= from(0)) return -1;
        const unsigned lane = threadIdx.x % 32;
        unsigned lo = 0, hi = most;             // the largest level that `index` is behind: from(lo) > index >= from(hi)
        while (hi - lo > 1) { const unsigned mid = (lo + hi) / 2; if (from(mid) > index) lo = mid; else hi = mid; }
        const unsigned rank = index - from(lo + 1);
        unsigned mine = 0;
        #pragma unroll
        for (unsigned k = 0; k < 4; k++) mine += n[k] > lo;
        unsigned sum = mine;
        #pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const unsigned u = __shfl_up_sync(0xffffffffu, sum, o); if (lane >= (unsigned)o) sum += u; }
        const unsigned behind = __ballot_sync(0xffffffffu, sum > rank);
        if (!behind) return -1;                 // sequences that share rows: more pairs than are counted in 32 bits
        const int at = __ffs(behind) - 1;
        unsigned left = rank - (sum - mine), which = 0;
        #pragma unroll
        for (unsigned k = 0; k < 4; k++) if (n[k] > lo) { if (left == 0) which = k; left--; }
        const unsigned s = at * 4 + __shfl_sync(0xffffffffu, which, at);
        job.q0 = clamped(a.q_starts, s, a.q_rows);
        job.queries = clamped(a.q_starts, s + 1, a.q_rows) - job.q0;
        job.k0 = clamped(a.kv_starts, s, a.kv_rows);
        job.keys = max(0, clamped(a.kv_starts, s + 1, a.kv_rows) - job.k0);
        return (int)lo;
    }
    // turned: the later tile, which has more keys with a mask, is the first one
    __device__ __forceinline__ bool find(const Args &a, unsigned index, unsigned kv_heads, unsigned turned, fused::Job &job) {
        const unsigned number = index / kv_heads;
        const int pair = levelled ? by_level(a, number, job) : find_piece(a, number, place, [&](unsigned queries) { return pairs(a, queries); }, job.q0, job.queries, job.k0, job.keys);
        if (pair < 0) return false;
        job.kv_head = (int)(index - number * kv_heads);
        job.block = (int)a.block;
        #pragma unroll
        for (int w = 0; w < 2; w++) {
            job.first[w] = (pair * 2 + (w ^ (int)turned)) * (int)a.block;
            const bool there = job.first[w] < job.queries;
            job.steps[w] = there ? (job.end(w, a.masked) + (int)fused::TILE - 1) / (int)fused::TILE : 0;
            if (!there) job.first[w] = -1;
        }
        job.live = 1;
        return true;
    }
};
// Where row r of a tile is in a matrix of rows and heads, in elements; -1: nowhere.
__device__ __forceinline__ long long row_at(const Args &a, const fused::Job &job, int first, unsigned r, unsigned row_stride, unsigned head_stride) {
    const unsigned q = r * a.part >> 16, h = r - q * a.group, query = (unsigned)first + q;
    if (q >= a.block || (int)query >= job.queries) return -1;
    return (long long)((unsigned long long)((unsigned)job.q0 + query) * row_stride + (unsigned long long)((unsigned)job.kv_head * a.group + h) * head_stride);
}

// A role's walk through the jobs.
struct Walk {
    fused::Shared *sh;
    unsigned slot = 0, lap = 0;
    __device__ __forceinline__ const fused::Job &job() const { return sh->jobs[slot]; }
    __device__ __forceinline__ bool next(unsigned long long limit = fused::LIMIT_NS) {
        if (!fused::warp_wait(&sh->job_full[slot], lap & 1u, &sh->gave_up, limit)) return false;
        return tc::uniform(job().live) != 0;
    }
    __device__ __forceinline__ void done() {
        __syncwarp();
        if (threadIdx.x % 32 == 0) tc::mbar_arrive(&sh->job_empty[slot]);
        if (++slot == fused::JOBS) { slot = 0; lap++; }
    }
};

// The warp that finds the work: the CTA's own first, then that of others that have not begun.
__device__ __forceinline__ void deal(fused::Shared &sh, const Args &a, unsigned kv_heads) {
    using namespace fused;
    const unsigned lane = threadIdx.x % 32;
    Finder finder(a);
    Job begin;
    bool ok = true, found = finder.find(a, blockIdx.x, kv_heads, 0u, begin);
    unsigned index, slot = 0, lap = 0, asked = 0, wanted = 0;
    while (true) {
        if (found) {
            ok = warp_wait(&sh.job_empty[slot], (lap & 1u) ^ 1u, &sh.gave_up);
            if (ok && lane == 0) { sh.jobs[slot] = begin; tc::mbar_arrive(&sh.job_full[slot]); }
            __syncwarp();
            if (++slot == JOBS) { slot = 0; lap++; }
            if (begin.both() > 0) ok = ok && warp_wait(&sh.wanted, wanted++ & 1u, &sh.gave_up, whole_job(begin.both()));
            if (!ok) break;
        }
        if (lane == 0) ask_for_work(&sh);
        __syncwarp();
        ok = warp_wait(&sh.answered, asked++ & 1u, &sh.gave_up);
        if (!ok) break;
        const bool more = given_work(&sh, index);
        tc::fence_proxy_async_smem();          // the answer has been read before the next one is written
        __syncwarp();
        if (!more) break;
        found = finder.find(a, index, kv_heads, slot, begin);          // slots alternate, and so do the warps that get the longer tile
    }
    if (warp_wait(&sh.job_empty[slot], (lap & 1u) ^ 1u, &sh.gave_up) && lane == 0) { sh.jobs[slot].live = 0; tc::mbar_arrive(&sh.job_full[slot]); }
    __syncwarp();
}

template <int TYPE, int DIM>
__global__ void __launch_bounds__(fused::THREADS, 1) prompt_tiles(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                                                                   const Args a, unsigned kv_heads) {
    using namespace fused;
    typedef Shape<DIM> H;
    extern __shared__ char raw[];
    const unsigned base = (tc::smem_u32(raw) + 1023u) & ~1023u;
    char *const smem = raw + (base - tc::smem_u32(raw));
    const unsigned q_at = base, k_at = base + 2 * H::QUERIES * H::BYTES, v_at = k_at + H::STAGES * H::BYTES;
    __shared__ __align__(16) Shared sh;
    const unsigned warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31u;
    unsigned *const gave_up = &sh.gave_up;
    if (threadIdx.x == 0) {
        sh.gave_up = 0u;
        tc::mbar_init(&sh.answered, 1u); tc::mbar_init(&sh.wanted, 1u);
        for (unsigned i = 0; i < JOBS; i++) { tc::mbar_init(&sh.job_full[i], 1u); tc::mbar_init(&sh.job_empty[i], 13u + H::MMA_WARPS); }
        for (int w = 0; w < 2; w++) {
            for (int b = 0; b < 2; b++) { tc::mbar_init(&sh.q_full[b][w], 1u); tc::mbar_init(&sh.q_empty[b][w], 1u); }
            tc::mbar_init(&sh.s_full[w], 1u); tc::mbar_init(&sh.o_full[w], 1u); tc::mbar_init(&sh.o_done[w], 1u);
            tc::mbar_init(&sh.s_free[w], 4u); tc::mbar_init(&sh.p_full[w][0], 4u); tc::mbar_init(&sh.p_full[w][1], 4u); tc::mbar_init(&sh.o_free[w], 4u); tc::mbar_init(&sh.l_full[w], 4u);
        }
        for (int s = 0; s < 4; s++) { tc::mbar_init(&sh.k_full[s], 1u); tc::mbar_init(&sh.k_empty[s], H::MMA_WARPS); tc::mbar_init(&sh.v_full[s], 1u); tc::mbar_init(&sh.v_empty[s], H::MMA_WARPS); tc::mbar_init(&sh.v_clean[s], 1u); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        tc::fence_proxy_async_smem();
    }
    if (warp == 9) tc::tmem_alloc(&sh.tmem, 512u);
    attn::wait_for_previous_kernel();
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const unsigned tmem = __shfl_sync(0xffffffffu, sh.tmem, 0);
    // Registers: 128 x (2 x 192 + 40 + 88) = 512 x 128, what the launch holds
    if (warp >= 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        const unsigned quarter = warp & 3u, row = quarter * 32u + lane, lanes = tmem + (quarter << 21);
        uint4 *const turn = reinterpret_cast<uint4 *>(smem + (2 * H::QUERIES + 2 * H::STAGES) * H::BYTES + quarter * 2048);
        unsigned done = 0;                             // a bit for each tile: the parity of its jobs
        bool ok = true;
        for (Walk walk{&sh}; walk.next(); walk.done()) {
            const Job &job = walk.job();
            #pragma unroll 1
            for (int w = 0; w < 2; w++) {
                const int first = job.first[w], steps = job.steps[w];
                if (first < 0) continue;
                long long at[4];                       // the rows that the thread stores
                #pragma unroll
                for (unsigned x = 0; x < 4; x++) at[x] = row_at(a, job, first, quarter * 32 + x * 8 + (lane >> 2), a.out_row, a.out_head);
                float factor = 0.f;
                if (steps > 0) {
                    ok = ok && warp_wait(&sh.l_full[w], done >> w & 1u, gave_up, whole_job(steps)) && warp_wait(&sh.o_done[w], done >> w & 1u, gave_up);
                    done ^= 1u << w;
                    tc::tc_fence_after();
                    factor = sh.factor[w][row];
                }
                // 32 features at a time: a thread has its row's, and stores 16 bytes each of eight rows
                #pragma unroll 1
                for (int i = 0; i < DIM; i += 32) {
                    float o[32];
                    if (ok && steps > 0) { ld32(lanes + H::O + w * DIM + i, o); ld_done32(o); }
                    unsigned p[16];
                    #pragma unroll
                    for (int x = 0; x < 16; x++) p[x] = !ok ? 0x7fff7fffu : steps == 0 ? 0u : mma::Of<TYPE>::pack(o[2 * x] * factor, o[2 * x + 1] * factor);
                    if (i + 32 == DIM && steps > 0) {
                        tc::tc_fence_before();
                        __syncwarp();
                        if (lane == 0) tc::mbar_arrive(&sh.o_free[w]);
                    }
                    __syncwarp();
                    #pragma unroll
                    for (unsigned x = 0; x < 4; x++) turn[lane * 4 + (x ^ (lane >> 1 & 3u))] = make_uint4(p[4 * x], p[4 * x + 1], p[4 * x + 2], p[4 * x + 3]);
                    __syncwarp();
                    const unsigned f = i + (lane & 3u) * 8;
                    #pragma unroll
                    for (unsigned x = 0; x < 4; x++) {
                        const unsigned r = x * 8 + (lane >> 2);
                        if (at[x] >= 0 && f < a.head_dim) *reinterpret_cast<uint4 *>(a.out + (at[x] + f) * 2) = turn[r * 4 + ((lane & 3u) ^ (r >> 1 & 3u))];
                    }
                }
            }
        }
        __syncwarp();
        tc::tc_fence_before();
        __syncthreads();
    } else if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        bool ok = true;
        if (warp == 10) {
            deal(sh, a, kv_heads);
        } else if (warp == 8) {
            unsigned stage = 0, lap = 0, q_uses[2] = {0, 0};
            for (Walk walk{&sh}; ok && walk.next(); walk.done()) {
                const Job &job = walk.job();
                const int steps = tc::uniform(job.both()), k0 = tc::uniform(job.k0), kv_head = tc::uniform(job.kv_head);
                for (int j = 0; j < steps; j++) {
                    ok = warp_wait(&sh.k_empty[stage], (lap & 1u) ^ 1u, gave_up);
                    if (!ok) break;
                    if (tc::elect_one()) {
                        tc::mbar_arrive_expect_tx(&sh.k_full[stage], H::BYTES);
                        #pragma unroll
                        for (int c = 0; c < H::CHUNKS; c++) tc::tma_load_3d(k_at + stage * H::BYTES + c * H::CHUNK_BYTES, &k_map, c * 64, kv_head, k0 + j * (int)TILE, &sh.k_full[stage]);
                    }
                    __syncwarp();
                    if (j == 0)
                        #pragma unroll
                        for (int w = 0; w < 2; w++) {
                            if (!ok || tc::uniform(job.steps[w]) == 0) continue;
                            const unsigned b = q_uses[w] % H::QUERIES, use = q_uses[w] / H::QUERIES;
                            ok = warp_wait(&sh.q_empty[b][w], (use & 1u) ^ 1u, gave_up);
                            q_uses[w]++;
                            if (ok && tc::elect_one()) {
                                tc::mbar_arrive_expect_tx(&sh.q_full[b][w], H::CHUNKS * a.group * a.block * 128u);
                                #pragma unroll
                                for (int c = 0; c < H::CHUNKS; c++)
                                    tc::tma_load_3d(q_at + (b * 2 + w) * H::BYTES + c * H::CHUNK_BYTES, &q_map, c * 64, kv_head * (int)a.group, job.q0 + job.first[w], &sh.q_full[b][w]);
                            }
                            __syncwarp();
                        }
                    ok = ok && warp_wait(&sh.v_empty[stage], (lap & 1u) ^ 1u, gave_up);
                    if (!ok) break;
                    if (tc::elect_one()) {
                        tc::mbar_arrive_expect_tx(&sh.v_full[stage], H::BYTES);
                        #pragma unroll
                        for (int c = 0; c < H::CHUNKS; c++) tc::tma_load_3d(v_at + stage * H::BYTES + c * H::CHUNK_BYTES, &v_map, c * 64, kv_head, k0 + j * (int)TILE, &sh.v_full[stage]);
                    }
                    __syncwarp();
                    if (++stage == H::STAGES) { stage = 0; lap++; }
                }
                if (!ok) break;
            }
        } else if (warp == 9 || H::MMA_WARPS == 2) {
            constexpr unsigned FORMAT = TYPE == ASPEN_B200_BF16 ? 1u : 0u;
            constexpr unsigned IDESC = 1u << 4 | FORMAT << 7 | FORMAT << 10 | (128u >> 4) << 24;       // sums fp32, 128 rows
            constexpr unsigned IDESC_S = IDESC | (128u >> 3) << 17, IDESC_O = IDESC | ((unsigned)DIM >> 3) << 17 | 1u << 16;      // the second operand of PV: features contiguous
            constexpr int OWN = 2 / H::MMA_WARPS;     // tiles of this warp, w0 the first
            const unsigned w0 = warp == 11;
            unsigned stage = 0, lap = 0, q_uses[OWN], asked[OWN], done[OWN], outs[OWN], cleaned = 0;      // cleaned: a bit for each stage, the parity of its steps that the keys ended in
            Walk walk{&sh};
            // Steps of the own tiles, and of both, of the job in work and of the next one.  Only the next is looked for while one is in work: the one behind it takes the place of the one in work.
            int steps[OWN], keys, next[OWN], next_all, next_keys = 0;
            #pragma unroll
            for (int i = 0; i < OWN; i++) q_uses[i] = asked[i] = done[i] = outs[i] = 0;
            bool live = true, begun = false;          // begun: the next one's first scores have been asked for
            auto look = [&]() {
                next_all = 0;
                #pragma unroll
                for (int i = 0; i < OWN; i++) next[i] = 0;
                live = walk.next();
                if (!live) return;
                const Job &job = walk.job();
                #pragma unroll
                for (int i = 0; i < OWN; i++) next[i] = tc::uniform(job.steps[w0 + i]);
                next_all = tc::uniform(job.both());
                next_keys = tc::uniform(job.keys);
                walk.done();
            };
            // scores of an own tile over the keys of the stage; the job's first or last ones
            auto scores = [&](int i, bool first, bool last) {
                const unsigned w = w0 + i, use = q_uses[i], b = use % H::QUERIES;
                if (first) ok = ok && warp_wait(&sh.q_full[b][w], use / H::QUERIES & 1u, gave_up);
                // a tile's softmax has read its scores before: it has given their weights, or (weights of their own) said so
                if (H::OWN_P) ok = ok && warp_wait(&sh.s_free[w], (asked[i] & 1u) ^ 1u, gave_up);
                asked[i]++;
                if (last) q_uses[i]++;
                if (!ok) return;
                tc::tc_fence_after();
                const unsigned q = q_at + (b * 2 + w) * H::BYTES;
                if (tc::elect_one()) {
                    #pragma unroll
                    for (int c = 0; c < H::CHUNKS; c++)
                        #pragma unroll
                        for (int k = 0; k < 4; k++)
                            mma_ss(tmem + H::S + w * 128, tc::umma_desc_low(q + c * H::CHUNK_BYTES + k * 32), tc::umma_desc_low(k_at + stage * H::BYTES + c * H::CHUNK_BYTES + k * 32), IDESC_S, c + k);
                    tc::tc_commit(&sh.s_full[w]);
                    if (last) tc::tc_commit(&sh.q_empty[b][w]);
                }
                __syncwarp();
            };
            // keys 16 from ... of the step
            auto values = [&](unsigned w, unsigned st, bool first, bool last, int from, int to) {
                if (tc::elect_one()) {
                    #pragma unroll
                    for (int k = from; k < to; k++)
                        mma_ts(tmem + H::O + w * DIM, tmem + H::P + w * H::P_APART + k * 8, (v_at + st * H::BYTES + k * 2048) >> 4 | (H::CHUNK_BYTES >> 4) << 16, IDESC_O, first ? k : 1);
                    if (to == 8) { tc::tc_commit(&sh.o_full[w]); if (last) tc::tc_commit(&sh.o_done[w]); }
                }
                __syncwarp();
            };
            auto release = [&](unsigned long long *bar) { if (tc::elect_one()) tc::tc_commit(bar); __syncwarp(); };
            for (look(); ok && live;) {
                if (!next_all) { look(); continue; }
                if (!begun) {
                    ok = warp_wait(&sh.k_full[stage], lap & 1u, gave_up);
                    #pragma unroll
                    for (int i = 0; i < OWN; i++) if (next[i]) scores(i, true, next[i] == 1);
                    if (!ok) break;
                    release(&sh.k_empty[stage]);
                }
                #pragma unroll
                for (int i = 0; i < OWN; i++) steps[i] = next[i];
                const int all = next_all;
                keys = next_keys;
                for (int j = 0; j < all; j++) {
                    const unsigned here = stage, at = lap;
                    if (++stage == H::STAGES) { stage = 0; lap++; }
                    // the scores to ask for now: the next step's, or the next job's first ones
                    const bool turn = j + 1 == all;
                    if (w0 == 0 && j == max(0, all - 3) && lane == 0) tc::mbar_arrive(&sh.wanted);
                    if (turn) look();
                    begun = turn && next_all > 0;
                    const bool more = begun || !turn;
                    const int then = turn ? 0 : j + 1;
                    if (more) ok = warp_wait(&sh.k_full[stage], lap & 1u, gave_up);
                    if (!ok) break;
                    if (H::OWN_P && more) {
                        #pragma unroll
                        for (int i = 0; i < OWN; i++) { const int until = turn ? next[i] : steps[i]; if (then < until) scores(i, turn, then + 1 == until); }
                        if (!ok) break;
                        release(&sh.k_empty[stage]);
                    }
                    ok = warp_wait(&sh.v_full[here], at & 1u, gave_up);
                    if (!ok) break;
                    if (keys < (j + 1) * (int)TILE) {
                        if (w0 == 0) {
                            const int from = keys - j * (int)TILE;
                            char *const v = smem + (v_at - base) + here * H::BYTES;
                            for (int i = from * 8 + (int)lane; i < (int)TILE * 8; i += 32)
                                #pragma unroll
                                for (int c = 0; c < H::CHUNKS; c++) *reinterpret_cast<uint4 *>(v + c * H::CHUNK_BYTES + i * 16) = make_uint4(0u, 0u, 0u, 0u);
                            tc::fence_proxy_async_smem();
                            __syncwarp();
                            if (H::MMA_WARPS == 2 && lane == 0) tc::mbar_arrive(&sh.v_clean[here]);
                        } else {
                            ok = warp_wait(&sh.v_clean[here], cleaned >> here & 1u, gave_up);
                            cleaned ^= 1u << here;
                        }
                    }
                    #pragma unroll
                    for (int i = 0; i < OWN; i++) {
                        const unsigned w = w0 + i;
                        const int until = turn ? next[i] : steps[i];
                        if (ok && j < steps[i]) {
                            if (j == 0) { ok = warp_wait(&sh.o_free[w], (outs[i] & 1u) ^ 1u, gave_up); outs[i]++; }        // the job before has been written out
                            ok = ok && warp_wait(&sh.p_full[w][0], done[i] & 1u, gave_up);
                            if (!ok) continue;
                            tc::tc_fence_after();
                            values(w, here, j == 0, false, 0, 6);
                            ok = warp_wait(&sh.p_full[w][1], done[i] & 1u, gave_up);
                            if (!ok) continue;
                            done[i]++;
                            tc::tc_fence_after();
                            values(w, here, false, j + 1 == steps[i], 6, 8);
                        }
                        if (!H::OWN_P && ok && then < until) scores(i, turn, then + 1 == until);
                    }
                    if (!ok) break;
                    release(&sh.v_empty[here]);
                    if (!H::OWN_P && more) release(&sh.k_empty[stage]);
                }
            }
        }
        __syncwarp();
        tc::tc_fence_before();
        __syncthreads();
        if (warp == 9) {
            if (sh.gave_up) {
                if (a.status && lane == 0) atomicOr(a.status, ASPEN_B200_PROMPT_STALLED);
                // copies and MMAs may still be in flight; they take microseconds
                unsigned long long t0, now;
                asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t0));
                do { __nanosleep(1000); asm volatile("mov.u64 %0, %globaltimer;" : "=l"(now)); } while (now - t0 < 2000000ull);
            }
            tc::tc_fence_after();
            tc::tmem_dealloc(tmem, 512u);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
        const int w = (int)(warp >> 2);
        const unsigned row = (warp & 3u) * 32u + lane, lanes = tmem + ((warp & 3u) << 21), s_at = lanes + H::S + w * 128, p_at = lanes + H::P + w * H::P_APART, o_at = lanes + H::O + w * DIM;
        const Pair scale2 = pair(a.scale, a.scale);
        // A row's largest weight is 2^LEVEL, and 2^(LEVEL + LOOSE) until its maximum is followed.  fp16 has its full precision down to 2^-24 of it; following at 4 instead would make that
        // 2^-25 (24 packed prompts 48.1 us instead of 47.2; 46.5 with weights of 1 at most)
        constexpr float LOOSE = TYPE == ASPEN_B200_FP16 ? 5.f : 8.f, LEVEL = mma::Of<TYPE>::TOP > 0.f ? mma::Of<TYPE>::TOP - LOOSE : 0.f;
        unsigned done = 0, outs = 0;
        bool ok = true;
        int both = 0;                                  // steps of the job before: without a tile of their own these warps wait for all of them
        for (Walk walk{&sh}; ok && walk.next(whole_job(both)); walk.done()) {
            const Job &job = walk.job();
            const int first = job.first[w], steps = tc::uniform(job.steps[w]);
            both = job.both();
            if (first < 0 || steps == 0) continue;
            const int query = first + (int)(row * a.part >> 16);
            const int seen = a.masked ? min(job.keys, query + job.behind() + 1) : job.keys;              // first key that the row does not see
            const int least_seen = __shfl_sync(0xffffffffu, seen, 0);            // of the warp's rows
            float max = -INFINITY, sum = 0.f;
            // a NaN stays the maximum, and so it becomes if a score is infinite: then all weights of the row are NaN
            auto grow = [&](float most) { max = max2(max, most); if (max == INFINITY) max = NAN; };
            #pragma unroll 1
            for (int j = 0; j < steps && ok; j++) {
                ok = warp_wait(&sh.s_full[w], done & 1u, gave_up);
                if (!ok) break;
                tc::tc_fence_after();
                float s[128];
                #pragma unroll
                for (int i = 0; i < 4; i++) ld32(s_at + i * 32, s + i * 32);
                #pragma unroll
                for (int i = 0; i < 4; i++) ld_done32(s + i * 32);
                if (H::OWN_P) {
                    tc::tc_fence_before();
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(&sh.s_free[w]);
                }
                const int key0 = j * (int)TILE;
                if (least_seen < key0 + (int)TILE) {
                    #pragma unroll
                    for (int h = 0; h < 4; h++) {
                        if (least_seen >= key0 + 32 * (h + 1)) continue;
                        const int left = seen - key0 - 32 * h;
                        #pragma unroll
                        for (int i = 0; i < 32; i++) s[h * 32 + i] = i < left ? s[h * 32 + i] : -INFINITY;
                    }
                }
                float m0 = max3(s[0], s[1], s[2]), m1 = max3(s[3], s[4], s[5]), m2 = max3(s[6], s[7], s[8]), m3 = max3(s[9], s[10], s[11]);
                #pragma unroll
                for (int i = 12; i < 124; i += 8) { m0 = max3(m0, s[i], s[i + 1]); m1 = max3(m1, s[i + 2], s[i + 3]); m2 = max3(m2, s[i + 4], s[i + 5]); m3 = max3(m3, s[i + 6], s[i + 7]); }
                m0 = max3(m0, s[124], s[125]); m1 = max3(m1, s[126], s[127]);
                const float top = max2(max3(m0, m1, m2), m3);
                if (H::OWN_P && done > 0) { ok = warp_wait(&sh.o_full[w], (done & 1u) ^ 1u, gave_up); tc::tc_fence_after(); }
                if (j == 0) grow(top);
                else if (__any_sync(0xffffffffu, (top - max) * a.scale > LOOSE || (top != top && max == max))) {
                    const float before = max;
                    grow(top);
                    const float down = max == -INFINITY ? 1.f : mma::exp2_fast((before - max) * a.scale);
                    #pragma unroll 1
                    for (int i = 0; i < DIM; i += 16) {
                        float o[16];
                        ld16(o_at + i, o);
                        ld_done16(o);
                        #pragma unroll
                        for (int x = 0; x < 16; x++) o[x] *= down;
                        st16(o_at + i, reinterpret_cast<unsigned *>(o));
                    }
                    sum *= down;
                }
                const float ref = max == -INFINITY ? 0.f : fmaf(-max, a.scale, LEVEL);
                const Pair ref2 = pair(ref, ref);
                Pair part[4] = {0ull, 0ull, 0ull, 0ull};
                #pragma unroll
                for (int h = 0; h < 4; h++) {
                    unsigned p[16];
                    #pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const Pair x = fma2(pair(s[h * 32 + 2 * i], s[h * 32 + 2 * i + 1]), scale2, ref2);
                        float y0, y1;
                        unpair(x, y0, y1);
                        y0 = mma::exp2_fast(y0); y1 = mma::exp2_fast(y1);
                        part[i & 3] = add2(part[i & 3], pair(y0, y1));
                        p[i] = mma::Of<TYPE>::pack(y0, y1);
                    }
                    st16(p_at + h * 16, p);
                    if (h >= 2) {
                        st_done();
                        tc::tc_fence_before();
                        __syncwarp();
                        if (lane == 0) tc::mbar_arrive(&sh.p_full[w][h - 2]);
                    }
                }
                float x0, x1;
                unpair(add2(add2(part[0], part[1]), add2(part[2], part[3])), x0, x1);
                sum += x0 + x1;
                done++;
            }
            // what the outputs are multiplied with, once the job before's have been
            ok = ok && warp_wait(&sh.o_free[w], (outs & 1u) ^ 1u, gave_up);
            outs++;
            if (ok) sh.factor[w][row] = sum == 0.f ? 0.f : 1.f / sum;
            __syncwarp();
            if (lane == 0 && ok) tc::mbar_arrive(&sh.l_full[w]);
        }
        __syncwarp();
        tc::tc_fence_before();
        __syncthreads();
    }
}

// ---- fp32 on tcgen05: operands of three bf16 parts each (attention_tc.cuh) ----
//
// x = x0 + x1 + x2, each part what bf16 holds of what is left: 24 bits.  Of the nine products of parts the six largest are multiplied, those left out are below 2^-22 of the whole; the
// sums of a step are added to those of the steps before in registers, because the tensor cores cut off what they add to a sum (8 x 512 tokens: error of the outputs 2.4e-7, plain
// fp32 4.1e-7).
//
// What bounds it.  A step of a tile takes 3400 cycles of the tensor pipe (24 MMAs of 64 and 48 of 32 cycles at best), two tiles in turn; shared memory holds one buffer each of keys and
// values, so that the splitting of the next ones (four warps, 0.5 us) follows their last use.  Each tile's own warps split its queries, beside the first keys (8 x 512 tokens, 12 heads
// of 64: 35.1 us, split one after another by the same four warps 40.5), and what is split next is asked for while this is being split (33.7).  Beside the 12 us that the products of the
// heaviest CTA take there are 5 us until the first, and the ends of the last tile.  A warp to issue each tile's products, as prompt_tiles has for 64 features, gains nothing here.

// Eight features of a row to the three parts of a tile.
__device__ __forceinline__ void split_piece(const float4 (&v)[2], char *put) {
    constexpr int BYTES = fused::Parts::BYTES;
    split::Pair y[4] = {split::pack(v[0].x, v[0].y), split::pack(v[0].z, v[0].w), split::pack(v[1].x, v[1].y), split::pack(v[1].z, v[1].w)};
    *reinterpret_cast<uint4 *>(put) = make_uint4(split::take_part<0>(y[0]), split::take_part<0>(y[1]), split::take_part<0>(y[2]), split::take_part<0>(y[3]));
    *reinterpret_cast<uint4 *>(put + BYTES) = make_uint4(split::take_part<1>(y[0]), split::take_part<1>(y[1]), split::take_part<1>(y[2]), split::take_part<1>(y[3]));
    *reinterpret_cast<uint4 *>(put + 2 * BYTES) = make_uint4(split::take_part<2>(y[0]), split::take_part<2>(y[1]), split::take_part<2>(y[2]), split::take_part<2>(y[3]));
}
__device__ __forceinline__ void read_piece(float4 (&v)[2], const float *from, bool in) {
    const float4 *const p = reinterpret_cast<const float4 *>(from);
    v[0] = in ? __ldg(p) : make_float4(0.f, 0.f, 0.f, 0.f);
    v[1] = in ? __ldg(p + 1) : make_float4(0.f, 0.f, 0.f, 0.f);
}

__global__ void __launch_bounds__(fused::THREADS, 1) prompt_parts(const Args a, unsigned kv_heads) {
    using namespace fused;
    typedef Parts H;
    extern __shared__ char raw[];
    const unsigned base = (tc::smem_u32(raw) + 1023u) & ~1023u;
    char *const smem = raw + (base - tc::smem_u32(raw));
    const unsigned q_at = base, k_at = base + 6 * H::BYTES, v_at = k_at + 3 * H::BYTES;
    __shared__ __align__(16) Shared sh;
    const unsigned warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31u;
    unsigned *const gave_up = &sh.gave_up;
    if (threadIdx.x == 0) {
        sh.gave_up = 0u;
        tc::mbar_init(&sh.answered, 1u); tc::mbar_init(&sh.wanted, 1u);
        for (unsigned i = 0; i < JOBS; i++) { tc::mbar_init(&sh.job_full[i], 1u); tc::mbar_init(&sh.job_empty[i], 13u); }
        for (int w = 0; w < 2; w++) {
            tc::mbar_init(&sh.q_full[0][w], 128u);
            tc::mbar_init(&sh.s_full[w], 1u); tc::mbar_init(&sh.o_full[w], 1u); tc::mbar_init(&sh.p_full[w][0], 4u);
        }
        tc::mbar_init(&sh.k_full[0], 128u); tc::mbar_init(&sh.k_empty[0], 1u); tc::mbar_init(&sh.v_full[0], 128u); tc::mbar_init(&sh.v_empty[0], 1u);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        tc::fence_proxy_async_smem();
    }
    if (warp == 9) tc::tmem_alloc(&sh.tmem, 512u);
    attn::wait_for_previous_kernel();
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const unsigned tmem = __shfl_sync(0xffffffffu, sh.tmem, 0);
    // Registers: 128 x (2 x 168 + 64 + 112) = 512 x 128, what the launch holds
    if (warp >= 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 112;");
        // Splits keys and values, in turn: a thread eight features of every 16th row.
        const unsigned t = threadIdx.x & 127u, row0 = t >> 3, piece = t & 7u;
        const bool wide = piece * 8 < a.head_dim;
        char *const put = smem + (k_at - base) + row0 * 128 + ((piece ^ (row0 & 7u)) << 4);
        unsigned uses = 0;
        bool ok = true;
        for (Walk walk{&sh}; ok && walk.next(); walk.done()) {
            const Job &job = walk.job();
            const int items = 2 * job.both();
            float4 v[8][2];
            const float *from;
            size_t apart;
            int left;                                  // keys from the thread's first one on
            auto place = [&](int i) {
                const unsigned row = i & 1 ? a.v_row : a.k_row, key = (unsigned)(i / 2) * TILE + row0;
                from = reinterpret_cast<const float *>(i & 1 ? a.v : a.k) + (size_t)(unsigned)job.kv_head * (i & 1 ? a.v_head : a.k_head) + (size_t)((unsigned)job.k0 + key) * row + piece * 8;
                apart = (size_t)16 * row;
                left = wide ? job.keys - (int)key : 0;
            };
            if (items) {
                place(0);
                #pragma unroll
                for (int x = 0; x < 8; x++) read_piece(v[x], from + x * apart, 16 * x < left);
            }
            #pragma unroll 1
            for (int i = 0; i < items; i++) {
                ok = warp_wait(i & 1 ? &sh.v_empty[0] : &sh.k_empty[0], (uses & 1u) ^ 1u, gave_up);
                if (!ok) break;
                uses += i & 1;
                char *const to = put + (i & 1 ? 3 * H::BYTES : 0);
                // each piece of what comes next is asked for as soon as this one's has been taken
                if (i + 1 < items) place(i + 1);
                else left = 0;
                #pragma unroll
                for (int x = 0; x < 8; x++) {
                    split_piece(v[x], to + x * 2048);
                    read_piece(v[x], from + x * apart, 16 * x < left);
                }
                tc::fence_proxy_async_smem();
                tc::mbar_arrive(i & 1 ? &sh.v_full[0] : &sh.k_full[0]);
            }
        }
        __syncwarp();
        tc::tc_fence_before();
        __syncthreads();
    } else if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        bool ok = true;
        if (warp == 10) deal(sh, a, kv_heads);
        else if (warp == 9) {
            constexpr unsigned IDESC = 1u << 4 | 1u << 7 | 1u << 10 | (128u >> 4) << 24;               // sums fp32, operands bf16, 128 rows
            constexpr unsigned IDESC_S = IDESC | (128u >> 3) << 17, IDESC_O = IDESC | (64u >> 3) << 17 | 1u << 16;        // the second operand of PV: features contiguous
            unsigned k_uses = 0, v_uses = 0, q_uses[2] = {0, 0}, done[2] = {0, 0};
            Walk walk{&sh};
            int steps[2], next[2] = {0, 0};
            bool live = true, begun = false;          // begun: the next job's first scores have been asked for
            auto look = [&]() {
                next[0] = next[1] = 0;
                live = walk.next();
                if (!live) return;
                const Job &job = walk.job();
                next[0] = tc::uniform(job.steps[0]);
                next[1] = tc::uniform(job.steps[1]);
                walk.done();
            };
            // Six of the nine products of parts, smallest first: what the sums cut off then is small.  In a loop: the code of all of them is more than is fetched in time.
            auto scores = [&](int w, bool first) {
                if (first) ok = ok && warp_wait(&sh.q_full[0][w], q_uses[w]++ & 1u, gave_up);
                if (!ok) return;
                tc::tc_fence_after();
                const unsigned q = q_at + w * 3 * H::BYTES, d = tmem + w * 256;
                if (tc::elect_one()) {
                    #pragma unroll 1
                    for (int p = 0; p < 6; p++) {
                        const unsigned x = tc::umma_desc_low(q + H::first(p) * H::BYTES), y = tc::umma_desc_low(k_at + H::second(p) * H::BYTES);
                        #pragma unroll
                        for (int k = 0; k < 4; k++) mma_ss(d, x + k * 2, y + k * 2, IDESC_S, p + k);
                    }
                    tc::tc_commit(&sh.s_full[w]);
                }
                __syncwarp();
            };
            auto values = [&](int w) {
                const unsigned d = tmem + w * 256;
                if (tc::elect_one()) {
                    #pragma unroll 1
                    for (int p = 0; p < 6; p++) {
                        const unsigned x = d + (H::first(p) == 2 ? 128 : H::first(p) * 16), apart = H::first(p) == 2 ? 16 : 32, y = (v_at + H::second(p) * H::BYTES) >> 4;
                        #pragma unroll
                        for (int k = 0; k < 8; k++) mma_ts(d + H::O, x + k / 2 * apart + k % 2 * 8, y + k * 128, IDESC_O, p + k);
                    }
                    tc::tc_commit(&sh.o_full[w]);
                }
                __syncwarp();
            };
            auto release = [&](unsigned long long *bar) { if (tc::elect_one()) tc::tc_commit(bar); __syncwarp(); };
            for (look(); ok && live;) {
                if (!next[0] && !next[1]) { look(); continue; }
                if (!begun) {
                    ok = warp_wait(&sh.k_full[0], k_uses++ & 1u, gave_up);
                    #pragma unroll 1
                    for (int w = 0; w < 2; w++) if (next[w]) scores(w, true);
                    if (!ok) break;
                    release(&sh.k_empty[0]);
                }
                steps[0] = next[0]; steps[1] = next[1];
                const int all = max(steps[0], steps[1]);
                #pragma unroll 1
                for (int j = 0; j < all; j++) {
                    // the scores to ask for now: the next step's, or the next job's first ones
                    const bool turn = j + 1 == all;
                    if (j == max(0, all - 3) && lane == 0) tc::mbar_arrive(&sh.wanted);
                    if (turn) look();
                    const int then = turn ? 0 : j + 1, until[2] = {turn ? next[0] : steps[0], turn ? next[1] : steps[1]};
                    const bool more = then < until[0] || then < until[1];
                    begun = turn && more;
                    ok = warp_wait(&sh.v_full[0], v_uses++ & 1u, gave_up);
                    bool keys = false;
                    // the next job's first scores wait for its queries, which are split when these tiles' outputs have been written
                    #pragma unroll 1
                    for (int i = 0; i < 4 && ok; i++) {
                        const int w = turn ? i & 1 : i >> 1;
                        if (i == (turn ? 2 : 3)) release(&sh.v_empty[0]);
                        if (!(turn ? i >> 1 : i & 1)) {
                            if (j >= steps[w]) continue;
                            ok = warp_wait(&sh.p_full[w][0], done[w]++ & 1u, gave_up);
                            if (!ok) break;
                            tc::tc_fence_after();
                            values(w);
                        } else if (then < until[w]) {
                            if (!keys) ok = warp_wait(&sh.k_full[0], k_uses++ & 1u, gave_up);
                            keys = true;
                            scores(w, turn);
                        }
                    }
                    if (!ok) break;
                    if (more) release(&sh.k_empty[0]);
                }
            }
        }
        __syncwarp();
        tc::tc_fence_before();
        __syncthreads();
        if (warp == 9) {
            if (sh.gave_up) {
                if (a.status && lane == 0) atomicOr(a.status, ASPEN_B200_PROMPT_STALLED);
                // MMAs may still be in flight; they take microseconds
                unsigned long long t0, now;
                asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t0));
                do { __nanosleep(1000); asm volatile("mov.u64 %0, %globaltimer;" : "=l"(now)); } while (now - t0 < 2000000ull);
            }
            tc::tc_fence_after();
            tc::tmem_dealloc(tmem, 512u);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
        const int w = (int)(warp >> 2);
        const unsigned row = (warp & 3u) * 32u + lane, s_at = tmem + ((warp & 3u) << 21) + w * 256;
        float4 *const turn = reinterpret_cast<float4 *>(smem + 12 * H::BYTES + warp * 4096);
        const Pair scale2 = pair(a.scale, a.scale);
        unsigned done = 0;
        bool ok = true;
        int both = 0;                                  // steps of the job before: without a tile of their own these warps wait for all of them
        for (Walk walk{&sh}; walk.next(whole_job(both)); walk.done()) {
            const Job &job = walk.job();
            const int first = job.first[w], steps = tc::uniform(job.steps[w]);
            both = job.both();
            if (first < 0) continue;
            if (steps) {
                // the tile's queries; the scores that were multiplied with the last ones have been read
                const unsigned t = threadIdx.x & 127u, row0 = t >> 3, piece = t & 7u;
                char *const put = smem + (q_at - base) + w * 3 * H::BYTES + row0 * 128 + ((piece ^ (row0 & 7u)) << 4);
                float4 v[8][2];
                #pragma unroll
                for (int x = 0; x < 8; x++) {
                    const long long at = row_at(a, job, first, row0 + 16 * x, a.q_row, a.q_head);
                    const bool in = at >= 0 && piece * 8 < a.head_dim;
                    read_piece(v[x], reinterpret_cast<const float *>(a.q) + (in ? at + piece * 8 : 0), in);
                }
                #pragma unroll
                for (int x = 0; x < 8; x++) split_piece(v[x], put + x * 2048);
                tc::fence_proxy_async_smem();
                tc::mbar_arrive(&sh.q_full[0][w]);
            }
            const int query = first + (int)(row * a.part >> 16);
            const int seen = a.masked ? min(job.keys, query + job.behind() + 1) : job.keys;              // first key that the row does not see
            const int least_seen = __shfl_sync(0xffffffffu, seen, 0), most_seen = __shfl_sync(0xffffffffu, seen, 31);       // of the warp's rows
            float max = -INFINITY, sum = 0.f, down = 0.f;
            Pair o[32];
            #pragma unroll
            for (int i = 0; i < 32; i++) o[i] = 0ull;
            // scores of 32 keys; those that are not seen are -inf
            auto load = [&](float *s, int key) {
                ld32(s_at + (key & 127), s);
                ld_done32(s);
                if (least_seen < key + 32) {
                    const int left = seen - key;
                    #pragma unroll
                    for (int i = 0; i < 32; i++) s[i] = i < left ? s[i] : -INFINITY;
                }
            };
            // the last product, relative to the maximum of its step, to the sums
            auto add = [&]() {
                ok = ok && warp_wait(&sh.o_full[w], (done & 1u) ^ 1u, gave_up);
                tc::tc_fence_after();
                const Pair down2 = pair(down, down);
                #pragma unroll
                for (int h = 0; h < 2; h++) {
                    float v[32];
                    ld32(s_at + H::O + h * 32, v);
                    ld_done32(v);
                    #pragma unroll
                    for (int i = 0; i < 16; i++) o[h * 16 + i] = fma2(o[h * 16 + i], down2, pair(v[2 * i], v[2 * i + 1]));
                }
            };
            #pragma unroll 1
            for (int j = 0; j < steps && ok; j++) {
                ok = warp_wait(&sh.s_full[w], done & 1u, gave_up);
                if (!ok) break;
                tc::tc_fence_after();
                const int key0 = j * (int)TILE, key1 = min(key0 + (int)TILE, most_seen);
                float m0 = -INFINITY, m1 = -INFINITY;
                #pragma unroll 1
                for (int key = key0; key < key1; key += 32) {
                    float s[32];
                    load(s, key);
                    #pragma unroll
                    for (int i = 0; i < 32; i += 4) { m0 = max3(m0, s[i], s[i + 1]); m1 = max3(m1, s[i + 2], s[i + 3]); }
                }
                // a NaN stays the maximum, and so it becomes if a score is infinite: then all weights of the row are NaN
                float top = max3(max, m0, m1);
                if (top == INFINITY) top = NAN;
                const float ref = top == -INFINITY ? 0.f : -top * a.scale, next_down = top == -INFINITY ? 1.f : mma::exp2_fast((max - top) * a.scale);
                const Pair ref2 = pair(ref, ref);
                max = top;
                sum *= next_down;
                Pair part[2] = {0ull, 0ull};
                #pragma unroll 1
                for (int key = key0; key < key0 + (int)TILE; key += 32) {
                    unsigned p[3][16];
                    if (most_seen > key) {
                        float s[32];
                        load(s, key);
                        #pragma unroll
                        for (int i = 0; i < 16; i++) {
                            const Pair x = fma2(pair(s[2 * i], s[2 * i + 1]), scale2, ref2);
                            float y0, y1;
                            unpair(x, y0, y1);
                            Pair y = pair(mma::exp2_fast(y0), mma::exp2_fast(y1));
                            part[i & 1] = add2(part[i & 1], y);
                            p[0][i] = split::take_part<0>(y);
                            p[1][i] = split::take_part<1>(y);
                            p[2][i] = split::take_part<2>(y);
                        }
                    } else {
                        #pragma unroll
                        for (int i = 0; i < 16; i++) p[0][i] = p[1][i] = p[2][i] = 0u;
                    }
                    // two parts in the place of their scores
                    st16(s_at + (key & 127), p[0]);
                    st16(s_at + (key & 127) + 16, p[1]);
                    st16(s_at + 128 + (key & 127) / 2, p[2]);
                }
                float x0, x1;
                unpair(add2(part[0], part[1]), x0, x1);
                sum += x0 + x1;
                if (j > 0) add();
                down = next_down;
                st_done();
                tc::tc_fence_before();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&sh.p_full[w][0]);
                done++;
            }
            long long at[8];                           // the rows that the thread stores
            #pragma unroll
            for (unsigned x = 0; x < 8; x++) at[x] = row_at(a, job, first, (warp & 3u) * 32 + x * 4 + (lane >> 3), a.out_row, a.out_head);
            if (steps > 0) add();
            tc::tc_fence_before();
            const float inv = !ok ? NAN : sum == 0.f ? 0.f : 1.f / sum;
            // 32 features at a time: a thread has its row's, and stores 16 bytes each of four rows
            #pragma unroll
            for (int h = 0; h < 2; h++) {
                __syncwarp();
                #pragma unroll
                for (unsigned x = 0; x < 8; x++) {
                    float4 y;
                    unpair(o[h * 16 + 2 * x], y.x, y.y);
                    unpair(o[h * 16 + 2 * x + 1], y.z, y.w);
                    turn[lane * 8 + (x ^ (lane & 7u))] = make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
                }
                __syncwarp();
                const unsigned f = h * 32 + (lane & 7u) * 4;
                #pragma unroll
                for (unsigned x = 0; x < 8; x++) {
                    const unsigned r = x * 4 + (lane >> 3);
                    if (at[x] >= 0 && f < a.head_dim) *reinterpret_cast<float4 *>(a.out + (at[x] + f) * 4) = turn[r * 8 + ((lane & 7u) ^ (r & 7u))];
                }
            }
        }
        __syncwarp();
        tc::tc_fence_before();
        __syncthreads();
    }
}

typedef CUresult (*EncodeFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *, const cuuint32_t *,
                             CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode_fn() {
    static EncodeFn fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess ? (EncodeFn)p : nullptr;
    }();
    return fn;
}
// (feature, head, row) of a 16-bit matrix, boxes of 64 features of some heads of some rows; zeros outside.
bool encode(CUtensorMap *map, int type, const char *p, unsigned dim, unsigned heads, unsigned rows, size_t head, size_t row, unsigned box_heads) {
    const cuuint64_t dims[3] = {dim, heads, rows}, strides[2] = {head * 2, row * 2};
    const cuuint32_t box[3] = {64, box_heads, fused::TILE / box_heads}, one[3] = {1, 1, 1};
    return encode_fn()(map, type == ASPEN_B200_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<char *>(p), dims, strides, box, one,
                       CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Jobs of a call, at most.
unsigned long long jobs_of(const Args &a) {
    const unsigned long long kv_heads = a.heads / a.group, sequences = a.sequences < a.q_rows ? a.sequences : a.q_rows;
    return (a.q_rows / a.block + 2 * sequences) / 2 * kv_heads;
}
cudaError_t launch_parts(const Args &a, cudaStream_t stream) {
    cudaError_t err = cudaFuncSetAttribute(prompt_parts, cudaFuncAttributeMaxDynamicSharedMemorySize, fused::Parts::SMEM);
    if (err != cudaSuccess) return err;
    return attn::launch_early(prompt_parts, (unsigned)jobs_of(a), fused::THREADS, fused::Parts::SMEM, stream, a, a.heads / a.group);
}
template <int TYPE, int DIM>
cudaError_t launch_tiles(const Args &a, const CUtensorMap *maps, cudaStream_t stream) {
    cudaError_t err = cudaFuncSetAttribute(prompt_tiles<TYPE, DIM>, cudaFuncAttributeMaxDynamicSharedMemorySize, fused::Shape<DIM>::SMEM);
    if (err != cudaSuccess) return err;
    return attn::launch_early(prompt_tiles<TYPE, DIM>, (unsigned)jobs_of(a), fused::THREADS, fused::Shape<DIM>::SMEM, stream, maps[0], maps[1], maps[2], a, a.heads / a.group);
}
// False: not a call for these kernels.
bool try_tiles(const Args &a, int type, unsigned ranks, cudaStream_t stream, cudaError_t *err) {
    // a row's largest score is its largest product only for a scale above 0
    if (!a.kv_rows || !(a.scale > 0.f) || a.group > fused::TILE || jobs_of(a) > 0x7fffffffull) return false;
    // A step of 128 keys takes a CTA about half as long as two tiles of 64 take one of prompt_rows, so four of these beside each other are faster, where there is room for them: 12 heads of 64, two
    // sequences of 16 queries over 2016 keys 12.4 us, in tiles 24.4; one prompt of 512 tokens, 8 heads of 64, 9.0 and 11.8 (fp32 17.6 and 27.5).
    if (ranks >= 4) return false;
    // Short sequences, going by the mean: a job of one step takes 4 us (fp32 5), and a block of prompt_rows 1.2 (3), several at once on an SM.  12 heads of 64, bf16 and fp32, 32 prompts of 60
    // tokens 8.6 and 14.3 us (in tiles 14.5 and 21), of 100 tokens 12 and 35 (14.5 and 24.6); 8 heads of 128, fp16, of 96 tokens 14.7 (12.5).  Where one sequence of a few is long and the others
    // short, the blocks take up to three times as long, of 4096 rows at most.
    if (a.group <= 2 && a.q_rows <= 4096 && a.q_rows <= 64ull * a.sequences && a.kv_rows <= 64ull * a.sequences) return false;
    if (type == ASPEN_B200_FP32) {
        if (a.head_dim > 64) return false;
        *err = launch_parts(a, stream);
        return true;
    }
    if (a.head_dim > 128 || !encode_fn()) return false;
    const unsigned kv_heads = a.heads / a.group;
    CUtensorMap maps[3];
    if (!encode(&maps[0], type, a.q, a.head_dim, a.heads, a.q_rows, a.q_head, a.q_row, a.group) || !encode(&maps[1], type, a.k, a.head_dim, kv_heads, a.kv_rows, a.k_head, a.k_row, 1) ||
        !encode(&maps[2], type, a.v, a.head_dim, kv_heads, a.kv_rows, a.v_head, a.v_row, 1)) return false;
    if (a.head_dim <= 64) *err = type == ASPEN_B200_BF16 ? launch_tiles<ASPEN_B200_BF16, 64>(a, maps, stream) : launch_tiles<ASPEN_B200_FP16, 64>(a, maps, stream);
    else *err = type == ASPEN_B200_BF16 ? launch_tiles<ASPEN_B200_BF16, 128>(a, maps, stream) : launch_tiles<ASPEN_B200_FP16, 128>(a, maps, stream);
    return true;
}

}  // namespace

extern "C" int aspen_b200_attention_prompt(const aspen_b200_prompt_t *p, void *cuda_stream) {
    const char *what = "aspen_b200_attention_prompt";
    if (!p) { ASPEN_ERR("%s: no arguments\n", what); return -1; }
    int rc = attn::check_type(p->type, p->head_dim, what);
    if (rc) return rc;
    if (!p->heads || !p->kv_heads || p->heads % p->kv_heads) { ASPEN_ERR("%s: %u heads of queries, %u of keys\n", what, p->heads, p->kv_heads); return -1; }
    if (!(p->scale - p->scale == 0.f)) { ASPEN_ERR("%s: scale is not finite\n", what); return -1; }
    // rows are int on the device; block numbers and 128 rows past the end stay below 2^31; a CTA reads the starts of 2^24 sequences in less time than its roles wait for one another
    if (p->q_rows > 0x3fffffffu || p->kv_rows > 0x3fffffffu || p->sequences > 1u << 24 || p->heads > 0xffffu) { ASPEN_ERR("%s: too many rows, sequences or heads\n", what); return -2; }
    if (!p->sequences || !p->q_rows) return 0;
    if (!p->q_starts || !p->kv_starts) { ASPEN_ERR("%s: q_starts or kv_starts is NULL\n", what); return -1; }
    const attn::Named ints[] = {{p->q_starts, "q_starts"}, {p->kv_starts, "kv_starts"}, {p->status, "status"}};
    if ((rc = attn::check_ints(ints, 3, what))) return rc;
    if ((rc = attn::check_rows(p->q, p->q_row_stride, p->q_head_stride, p->type, "q", what)) || (rc = attn::check_rows(p->out, p->out_row_stride, p->out_head_stride, p->type, "out", what))) return rc;
    if (p->kv_rows && ((rc = attn::check_rows(p->k, p->k_row_stride, p->k_head_stride, p->type, "k", what)) || (rc = attn::check_rows(p->v, p->v_row_stride, p->v_head_stride, p->type, "v", what)))) return rc;
    const int sms = attn::sm_count(what);
    if (sms < 0) return sms;
    const attn::Named all[] = {{p->q, "q"}, {p->out, "out"}, {p->q_starts, "q_starts"}, {p->kv_starts, "kv_starts"}, {p->kv_rows ? p->k : nullptr, "k"}, {p->kv_rows ? p->v : nullptr, "v"}, {p->status, "status"}};
    if ((rc = attn::check_device(all, 7, what))) return rc;
    Args a;
    a.q = static_cast<const char *>(p->q);
    a.k = static_cast<const char *>(p->k);
    a.v = static_cast<const char *>(p->v);
    a.out = static_cast<char *>(p->out);
    a.q_starts = p->q_starts;
    a.kv_starts = p->kv_starts;
    const size_t q_row = (size_t)p->heads * p->head_dim, kv_row = (size_t)p->kv_heads * p->head_dim;
    a.q_row = (unsigned)attn::packed(p->q_row_stride, q_row);
    a.q_head = (unsigned)attn::packed(p->q_head_stride, p->head_dim);
    a.k_row = (unsigned)attn::packed(p->k_row_stride, kv_row);
    a.k_head = (unsigned)attn::packed(p->k_head_stride, p->head_dim);
    a.v_row = (unsigned)attn::packed(p->v_row_stride, kv_row);
    a.v_head = (unsigned)attn::packed(p->v_head_stride, p->head_dim);
    a.out_row = (unsigned)attn::packed(p->out_row_stride, q_row);
    a.out_head = (unsigned)attn::packed(p->out_head_stride, p->head_dim);
    a.sequences = p->sequences;
    a.q_rows = p->q_rows;
    a.kv_rows = p->kv_rows;
    a.heads = p->heads;
    a.group = p->heads / p->kv_heads;
    a.part = (65536 + a.group - 1) / a.group;
    a.block = a.group > fused::TILE ? 0 : fused::TILE / a.group;
    a.by_block = make_divisor(a.block);
    a.head_dim = p->head_dim;
    a.masked = p->masked != 0;
    a.scale = p->scale * 1.4426950408889634f;
    a.status = p->status;
    const cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
    cudaError_t err = cudaSuccess;
    const unsigned ranks = ranks_of(a, p->type, (unsigned)sms);
    a.in_a_row = ranks > 1 ? 1u : in_a_row_of(a, (unsigned)sms);
    if (!try_tiles(a, p->type, ranks, stream, &err))
        err = p->type == ASPEN_B200_FP32 ? launch_rows<ASPEN_B200_FP32>(a, ranks, stream) : p->type == ASPEN_B200_BF16 ? launch_rows<ASPEN_B200_BF16>(a, ranks, stream) : launch_rows<ASPEN_B200_FP16>(a, ranks, stream);
    if (err != cudaSuccess) { cudaGetLastError(); ASPEN_ERR("%s: %s\n", what, cudaGetErrorString(err)); return -3; }
    return 0;
}
