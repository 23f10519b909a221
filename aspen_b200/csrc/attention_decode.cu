// Attention of one new token of each sequence over the pages of its cache.
//
// out = sum_j p_j v_j / sum_j p_j with p_j = exp(scale q k_j - max): one pass over the keys, the maximum and the sum running along (values already summed are scaled by
// exp(old max - new max)).  Parts of a sequence give (max, sum, weighted values) that join the same way.
//
// What bounds it: reading the cache once.  A step of 16 keys is multiplied with all query heads of its key head, so each key and value is read once for 16 heads of its
// group (8 with 256 features, and in fp32 with 128: heads_of_pass); larger groups read it again.
//     S^T [16 keys x 8 heads] = K Q^T, O^T [features x 8 heads] += V^T P^T, by mma.sync with the keys as the 16-row operand: 8 heads fill its columns where tcgen05 would want
// 128 rows of queries, and a warp needs nobody else: keys and values go from memory to registers as 32-byte pieces (mma_sync.cuh), no shared memory, no barrier.  Pieces of the next
// step are asked for before this one is multiplied.  64 sequences of up to 8192 tokens, bf16, 8 heads of keys of 128: 170 us, 6.5 TB/s with start, end and join; one of 100003 70 us, 5.9 TB/s; 32 of
// up to 1024, fp16, 12 heads of 64, 17 us, of which 10 are the first loads and the joins; one of 1000, fp32, 9.3 us on the device; 64 of up to 2000, fp32, 12 heads of 64, 77 us, 5.0 TB/s (the
// splitting of operands takes its share).
//
// Cut: all (sequence, key head) items' steps stand in one line that is dealt to CTAs and then to their warps in equal shares, whatever the lengths (they are known on the
// device only, and a captured call may see others each time).  A warp's whole items are finished in its registers; at most two it shares with its neighbours.  Shares are
// joined in the CTA through shared memory, and those that cross CTAs by a second kernel, started early, in order of the steps: the same call gives the same bits.
#include "early_launch.cuh"
#include "mma_sync.cuh"

namespace {

using attn::Pages;

constexpr int STEP = 16;                        // keys of a step

// Heads of a group that one pass over the keys serves: eight columns of a product, or sixteen where their sums leave room in the registers.
constexpr unsigned heads_of_pass(unsigned group, unsigned dim, int type) { return group <= 8 || dim == 256 || (type == ASPEN_B200_FP32 && dim == 128) ? 8 : 16; }
constexpr unsigned dim_of(unsigned head_dim) { return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256; }
// Threads of a CTA and CTAs on an SM: the warps that the registers are enough for.  16 with 120 registers (16 bits, 64 features), 12 with 168, 8 with 255.
constexpr int ctas_of(int type, unsigned dim) { return type != ASPEN_B200_FP32 && dim == 64 ? 2 : 1; }
constexpr int threads_of(int type, unsigned dim, unsigned heads) { return heads == 8 && dim == (type == ASPEN_B200_FP32 ? 64 : 128) ? 384 : 256; }

struct Args {
    const char *q, *k, *v;
    char *out;
    const int *slots;
    Pages at;
    size_t q_row, q_head, out_row, out_head;    // in elements
    unsigned entries, kv_heads, group, chunks, head_dim;    // chunks: of a group, each up to the kernel's HEADS
    float scale;                                // with log2(e)
    int *record;                                // [CTAs][2]: item that goes on behind the CTA (-1: none), last CTA that has some of it
    float *part;                                // [CTAs][2][HEADS][DIM + 4]: what began before the CTA, and what goes on behind it
};

__device__ __forceinline__ unsigned steps_of(unsigned tokens) { return (tokens + STEP - 1) / STEP; }
__device__ __forceinline__ int slot_of(const Args &a, unsigned e) { return a.slots ? a.slots[e] : (int)e; }

template <int TYPE>
__device__ __forceinline__ void store_value(char *at, float v) {
    if (TYPE == ASPEN_B200_FP32) *reinterpret_cast<float *>(at) = v;
    else if (TYPE == ASPEN_B200_BF16) *reinterpret_cast<__nv_bfloat16 *>(at) = __float2bfloat16_rn(v);
    else *reinterpret_cast<__half *>(at) = __float2half_rn(v);
}

// Steps of all items, and where each thread's entries begin in the line.
template <int THREADS>
struct Line {
    unsigned long long before[THREADS + 1];     // [i]: steps of the entries before thread i's; [THREADS]: all
    unsigned long long sums[THREADS / 32];
    unsigned tokens[THREADS];                   // of each thread's only entry, where there are no more entries than threads
    int slot[THREADS];
    __device__ __forceinline__ void entry(const Args &a, unsigned each, unsigned e, int &s, unsigned &n) const {
        if (each == 1) { s = slot[e]; n = tokens[e]; return; }
        s = slot_of(a, e);
        n = attn::sequence_length(a.at, s);
    }
};

// Also the outputs of sequences without tokens: entry e in CTA e.
template <int TYPE, int THREADS>
__device__ void measure(const Args &a, unsigned each, Line<THREADS> &line) {
    constexpr int SIZE = TYPE == ASPEN_B200_FP32 ? 4 : 2;
    const unsigned lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    unsigned long long mine = 0;
    for (unsigned i = 0; i < each; i++) {
        const unsigned e = threadIdx.x * each + i;
        bool empty = false;
        if (e < a.entries) {
            const int slot = slot_of(a, e);
            const unsigned tokens = attn::sequence_length(a.at, slot);
            mine += steps_of(tokens);
            empty = tokens == 0 && e % gridDim.x == blockIdx.x;
            if (each == 1) { line.tokens[threadIdx.x] = tokens; line.slot[threadIdx.x] = slot; }
            if (empty && (slot < 0 || (unsigned)slot >= a.at.sequences)) atomicOr(a.at.status, ASPEN_B200_CACHE_BAD_INDEX);
        }
        for (unsigned left = __ballot_sync(0xffffffffu, empty); left; left &= left - 1) {
            const size_t row = (size_t)((warp * 32 + __ffs(left) - 1) * each + i) * a.out_row;
            for (unsigned x = lane; x < a.kv_heads * a.group * a.head_dim; x += 32) store_value<TYPE>(a.out + (row + (size_t)(x / a.head_dim) * a.out_head + x % a.head_dim) * SIZE, 0.f);
        }
    }
    mine *= a.kv_heads * a.chunks;
    unsigned long long s = mine;
    #pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const unsigned long long u = __shfl_up_sync(0xffffffffu, s, o); if (lane >= (unsigned)o) s += u; }
    if (lane == 31) line.sums[warp] = s;
    __syncthreads();
    unsigned long long base = 0;
    #pragma unroll
    for (unsigned w = 0; w < THREADS / 32; w++) base += w < warp ? line.sums[w] : 0ull;
    line.before[threadIdx.x] = base + s - mine;
    if (threadIdx.x == THREADS - 1) line.before[THREADS] = base + s;
    __syncthreads();
}

// Running softmax of one item's heads in one warp.  Lane (g, t): heads 2 t and 2 t + 1 of each eight, the features of its pieces.
template <int TYPE, int DIM, int HEADS>
struct Running {
    static constexpr int TILES = HEADS / 8, ROWS = DIM / 16;
    float o[TILES][ROWS][4];                    // [features' 16-row tile]: (feature, head 2 t), (feature, 2 t + 1), (feature + 1, 2 t), (feature + 1, 2 t + 1)
    float max[TILES][2], sum[TILES][2];         // sum: of this lane's keys only
    __device__ __forceinline__ void clear() {
        #pragma unroll
        for (int n = 0; n < TILES; n++) {
            #pragma unroll
            for (int r = 0; r < ROWS; r++)
                #pragma unroll
                for (int i = 0; i < 4; i++) o[n][r][i] = 0.f;
            max[n][0] = max[n][1] = -INFINITY;
            sum[n][0] = sum[n][1] = 0.f;
        }
    }
    __device__ __forceinline__ void add_up() {
        #pragma unroll
        for (int n = 0; n < TILES; n++)
            #pragma unroll
            for (int j = 0; j < 2; j++)
                #pragma unroll
                for (int m = 4; m < 32; m <<= 1) sum[n][j] += __shfl_xor_sync(0xffffffffu, sum[n][j], m);
    }
    // First feature of this lane's piece p, and the values there: PIECE of them for head 2 t + j.
    static constexpr int PIECE = TYPE == ASPEN_B200_FP32 || DIM == 64 ? 8 : 16, PIECES = DIM / (8 * PIECE);
    static __device__ __forceinline__ int feature(int p, unsigned g) { return p * 8 * PIECE + (int)g * PIECE; }
    __device__ __forceinline__ float value(int n, int p, int x, int j) const { return o[n][p * (PIECE / 2) + x / 2][(x & 1) * 2 + j]; }
};

template <int TYPE>
__device__ __forceinline__ void store_piece(char *at, const float *v) {
    if (TYPE == ASPEN_B200_FP32) *reinterpret_cast<float4 *>(at) = make_float4(v[0], v[1], v[2], v[3]);
    else {
        typedef mma::Of<TYPE == ASPEN_B200_FP32 ? ASPEN_B200_BF16 : TYPE> T;
        *reinterpret_cast<uint4 *>(at) = make_uint4(T::pack(v[0], v[1]), T::pack(v[2], v[3]), T::pack(v[4], v[5]), T::pack(v[6], v[7]));
    }
}
__device__ __forceinline__ uint4 load16(const char *p, bool ok) {
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (ok) asm volatile("ld.global.nc.L1::no_allocate.L2::128B.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
// A lane's 32 bytes of a row: one load where every row starts on a 32-byte boundary (WIDE), else two.
struct Piece { unsigned w[8]; };
template <bool WIDE, int BYTES>
__device__ __forceinline__ void load_piece(Piece &v, const char *p, bool ok, int left) {
    if (WIDE && BYTES == 32) {
        #pragma unroll
        for (int i = 0; i < 8; i++) v.w[i] = 0u;
        if (ok && left > 0)
            asm volatile("ld.global.nc.L1::no_allocate.L2::128B.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                         : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3]), "=r"(v.w[4]), "=r"(v.w[5]), "=r"(v.w[6]), "=r"(v.w[7]) : "l"(p));
    } else {
        #pragma unroll
        for (int h = 0; h < BYTES / 16; h++) {
            const uint4 x = load16(p + h * 16, ok && left > h * 16);
            v.w[4 * h] = x.x; v.w[4 * h + 1] = x.y; v.w[4 * h + 2] = x.z; v.w[4 * h + 3] = x.w;
        }
    }
}

// An item and its steps from `begin` to `end`.
struct Share {
    unsigned entry, kv_head, chunk, begin, end, tokens;
    int slot;
};

template <int TYPE, int DIM, int HEADS, bool WIDE>
struct Kernel {
    static constexpr int SIZE = TYPE == ASPEN_B200_FP32 ? 4 : 2, ROW_BYTES = DIM * SIZE;
    // Bytes of a lane's piece of a row: of keys (four lanes to a row), of values (eight).  A buffer is what is on its way together: 128 bytes a lane.
    static constexpr int KEY_PIECE = 32, VALUE_PIECE = ROW_BYTES / 8 < 32 ? ROW_BYTES / 8 : 32;
    static constexpr int CHUNK = ROW_BYTES < 256 ? ROW_BYTES : 256, CHUNKS = ROW_BYTES / CHUNK;       // bytes of a row in a buffer
    static constexpr int KEYS = CHUNK / (4 * KEY_PIECE), VALUES = CHUNK / (8 * VALUE_PIECE);          // pieces of a row
    static constexpr int THREADS = threads_of(TYPE, DIM, HEADS), WARPS = THREADS / 32;
    static constexpr int ROW = DIM + 4;         // floats of a partial result of one head: values, maximum, sum
    static constexpr unsigned SMEM = WARPS * 2 * HEADS * ROW * 4;
    typedef Running<TYPE, DIM, HEADS> Run;
    struct Buffer { Piece p[4]; };

    // Byte offset of the row of key `lane % 32` behind `first`; -1 if there is none.
    static __device__ __forceinline__ long long row_of(const Args &a, const Share &s, unsigned first, unsigned lane) {
        const unsigned key = first + lane;
        if (key >= s.tokens) return -1;
        const long long at = attn::token_offset(a.at, s.slot, key);
        return at < 0 ? -1 : (at + (long long)(s.kv_head * a.at.head_stride)) * SIZE;
    }

    // Keys: rows g and g + 8 of the step.  Values: rows 2 t, 2 t + 1, 2 t + 8, 2 t + 9.
    static __device__ __forceinline__ void load_keys(Buffer &buf, const char *base, long long row0, long long row8, int c, unsigned t, unsigned head_dim) {
        #pragma unroll
        for (int i = 0; i < KEYS; i++) {
            const int at = c * CHUNK + (i * 4 + (int)t) * KEY_PIECE, left = (int)head_dim * SIZE - at;
            load_piece<WIDE, KEY_PIECE>(buf.p[2 * i], base + row0 + at, row0 >= 0, left);
            load_piece<WIDE, KEY_PIECE>(buf.p[2 * i + 1], base + row8 + at, row8 >= 0, left);
        }
    }
    static __device__ __forceinline__ void load_values(Buffer &buf, const char *base, const long long *row, int c, unsigned g, unsigned head_dim) {
        #pragma unroll
        for (int i = 0; i < VALUES; i++) {
            const int at = c * CHUNK + (i * 8 + (int)g) * VALUE_PIECE, left = (int)head_dim * SIZE - at;
            #pragma unroll
            for (int r = 0; r < 4; r++) load_piece<WIDE, VALUE_PIECE>(buf.p[4 * i + r], base + row[r] + at, row[r] >= 0, left);
        }
    }
    static constexpr int TILES = HEADS / 8, QUERY_PIECES = ROW_BYTES / (4 * KEY_PIECE);
    static __device__ __forceinline__ void multiply_keys(float (*s)[4], const Buffer &buf, const Piece (*q)[QUERY_PIECES], int c) {
        #pragma unroll
        for (int i = 0; i < KEYS; i++) {
            const unsigned *x = buf.p[2 * i].w, *y = buf.p[2 * i + 1].w;
            #pragma unroll
            for (int n = 0; n < TILES; n++) {
                const unsigned *b = q[n][c * KEYS + i].w;
                if constexpr (TYPE == ASPEN_B200_FP32) {
                    // sums of eight features are added outside: the tensor cores cut off what they add to a sum
                    float part[4] = {0.f, 0.f, 0.f, 0.f};
                    #pragma unroll
                    for (int k = 0; k < 8; k += 2) { const unsigned u[4] = {x[k], y[k], x[k + 1], y[k + 1]}; mma::tf32x3(part, u, b + k); }
                    #pragma unroll
                    for (int k = 0; k < 4; k++) s[n][k] += part[k];
                } else {
                    #pragma unroll
                    for (int k = 0; k < 8; k += 2) mma::Of<TYPE>::step(s[n], x[k], y[k], x[k + 1], y[k + 1], b[k], b[k + 1]);
                }
            }
        }
    }
    // p: weights as the column operand, 16-bit: one k = 16 step; fp32: two of k = 8
    static __device__ __forceinline__ void multiply_values(Run &run, const Buffer &buf, const unsigned (*p)[4], int c) {
        #pragma unroll
        for (int i = 0; i < VALUES; i++) {
            const unsigned *w0 = buf.p[4 * i].w, *w1 = buf.p[4 * i + 1].w, *w8 = buf.p[4 * i + 2].w, *w9 = buf.p[4 * i + 3].w;
            constexpr int WORDS = VALUE_PIECE / 4;
            if constexpr (TYPE == ASPEN_B200_FP32) {
                #pragma unroll
                for (int j = 0; j < WORDS / 2; j++) {
                    const unsigned lo[4] = {w0[2 * j], w0[2 * j + 1], w1[2 * j], w1[2 * j + 1]}, hi[4] = {w8[2 * j], w8[2 * j + 1], w9[2 * j], w9[2 * j + 1]};
                    #pragma unroll
                    for (int n = 0; n < TILES; n++) {
                        float part[4] = {0.f, 0.f, 0.f, 0.f};
                        mma::tf32x3(part, lo, p[n]);
                        mma::tf32x3(part, hi, p[n] + 2);
                        #pragma unroll
                        for (int k = 0; k < 4; k++) run.o[n][(c * VALUES + i) * (WORDS / 2) + j][k] += part[k];
                    }
                }
            } else {
                #pragma unroll
                for (int j = 0; j < WORDS; j++) {
                    const unsigned a0 = mma::pair_of(w0[j], w1[j], false), a1 = mma::pair_of(w0[j], w1[j], true);
                    const unsigned a2 = mma::pair_of(w8[j], w9[j], false), a3 = mma::pair_of(w8[j], w9[j], true);
                    #pragma unroll
                    for (int n = 0; n < TILES; n++) mma::Of<TYPE>::step(run.o[n][(c * VALUES + i) * WORDS + j], a0, a1, a2, a3, p[n][0], p[n][1]);
                }
            }
        }
    }

    // One step's scores: running maximum and sum, and the weights as an operand.
    static __device__ __forceinline__ void weigh(Run &run, float (*s)[4], bool ok0, bool ok8, float scale, unsigned lane, unsigned (*p)[4]) {
        #pragma unroll
        for (int n = 0; n < TILES; n++) {
            float x[4], w[4];
            #pragma unroll
            for (int i = 0; i < 4; i++) x[i] = (i < 2 ? ok0 : ok8) ? s[n][i] * scale : -INFINITY;
            float down[2];
            #pragma unroll
            for (int j = 0; j < 2; j++) {
                float m = fmaxf(x[j], x[2 + j]);
                #pragma unroll
                for (int o = 4; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                m = fmaxf(m, run.max[n][j]);
                const float ref = m == -INFINITY ? 0.f : m;
                down[j] = mma::exp2_fast(run.max[n][j] - ref);
                run.max[n][j] = m;
                w[j] = mma::exp2_fast(x[j] - (ref - mma::Of<TYPE>::TOP));
                w[2 + j] = mma::exp2_fast(x[2 + j] - (ref - mma::Of<TYPE>::TOP));
                run.sum[n][j] = run.sum[n][j] * down[j] + (w[j] + w[2 + j]);
            }
            if (__any_sync(0xffffffffu, down[0] != 1.f || down[1] != 1.f)) {
                #pragma unroll
                for (int r = 0; r < Run::ROWS; r++)
                    #pragma unroll
                    for (int i = 0; i < 4; i++) run.o[n][r][i] *= down[i & 1];
            }
            if constexpr (TYPE == ASPEN_B200_FP32) {
                // lane (g, t) wants keys 2 t and 2 t + 1 of each eight for head g; lane (key, g / 2) has them
                const unsigned from = 8 * (lane & 3) + (lane >> 3);
                const bool odd = lane >> 2 & 1u;
                #pragma unroll
                for (int h = 0; h < 2; h++)
                    #pragma unroll
                    for (int k = 0; k < 2; k++) {
                        const float u = __shfl_sync(0xffffffffu, w[2 * h], from + 4 * k), v = __shfl_sync(0xffffffffu, w[2 * h + 1], from + 4 * k);
                        p[n][2 * h + k] = __float_as_uint(odd ? v : u);
                    }
            } else {
                p[n][0] = mma::transpose8(mma::Of<TYPE>::pack(w[0], w[1]));
                p[n][1] = mma::transpose8(mma::Of<TYPE>::pack(w[2], w[3]));
            }
        }
    }

    static __device__ __forceinline__ long long from_lane(long long v, unsigned lane) { return __shfl_sync(0xffffffffu, v, lane); }

    // All steps of a share, in one warp.
    static __device__ __forceinline__ void walk(const Args &a, const Share &s, Run &run) {
        const unsigned lane = threadIdx.x % 32, g = lane >> 2, t = lane & 3;
        Piece q[TILES][QUERY_PIECES];
        #pragma unroll
        for (int n = 0; n < TILES; n++) {
            const unsigned in_group = s.chunk * HEADS + n * 8 + g;
            const char *row = a.q + ((size_t)s.entry * a.q_row + (size_t)(s.kv_head * a.group + in_group) * a.q_head) * SIZE;
            #pragma unroll
            for (int i = 0; i < QUERY_PIECES; i++) {
                const int at = (i * 4 + (int)t) * KEY_PIECE;
                load_piece<false, KEY_PIECE>(q[n][i], row + at, in_group < a.group, (int)a.head_dim * SIZE - at);
            }
        }
        run.clear();
        // rows of two steps: lanes 0 ... 15 the first one's keys, 16 ... 31 the second one's
        unsigned step = s.begin;
        long long rows = row_of(a, s, step * STEP, lane);
        Buffer buf[2];
        // buffers in turn: all chunks of a step's keys, then all of its values; each is filled again as soon as it has been multiplied
        long long key0 = from_lane(rows, g), key8 = from_lane(rows, g + 8), value[4];
        bool second = false;
        auto values_of = [&](unsigned at) {
            value[0] = from_lane(rows, at + 2 * t); value[1] = from_lane(rows, at + 2 * t + 1);
            value[2] = from_lane(rows, at + 2 * t + 8); value[3] = from_lane(rows, at + 2 * t + 9);
        };
        values_of(0);
        load_keys(buf[0], a.k, key0, key8, 0, t, a.head_dim);
        if (CHUNKS > 1) load_keys(buf[1], a.k, key0, key8, 1, t, a.head_dim);
        else load_values(buf[1], a.v, value, 0, g, a.head_dim);
        long long later = -1;
        #pragma unroll 1
        for (; step < s.end; step++) {
            const bool ok0 = key0 >= 0, ok8 = key8 >= 0, more = step + 1 < s.end;
            if (!second && step + 2 < s.end) later = row_of(a, s, (step + 2) * STEP, lane);
            float score[TILES][4];
            #pragma unroll
            for (int n = 0; n < TILES; n++)
                #pragma unroll
                for (int i = 0; i < 4; i++) score[n][i] = 0.f;
            #pragma unroll
            for (int c = 0; c < CHUNKS; c++) {
                multiply_keys(score, buf[c % 2], q, c);
                if (c + 2 < CHUNKS) load_keys(buf[c % 2], a.k, key0, key8, c + 2, t, a.head_dim);
                else if (CHUNKS > 1) load_values(buf[c % 2], a.v, value, c + 2 - CHUNKS, g, a.head_dim);
            }
            // the next step's rows
            long long next0 = -1, next8 = -1;
            if (more) {
                const unsigned at = second ? 0u : 16u;
                if (second) rows = later;
                next0 = from_lane(rows, at + g);
                next8 = from_lane(rows, at + g + 8);
            }
            if (CHUNKS == 1 && more) load_keys(buf[0], a.k, next0, next8, 0, t, a.head_dim);
            unsigned p[TILES][4];
            weigh(run, score, ok0, ok8, a.scale, lane, p);
            if (CHUNKS == 1) {
                multiply_values(run, buf[1], p, 0);
                if (more) { values_of(second ? 0u : 16u); load_values(buf[1], a.v, value, 0, g, a.head_dim); }
            } else {
                #pragma unroll
                for (int c = 0; c < CHUNKS; c++) {
                    multiply_values(run, buf[c % 2], p, c);
                    if (c + 2 < CHUNKS) load_values(buf[c % 2], a.v, value, c + 2, g, a.head_dim);
                    else if (more) load_keys(buf[c % 2], a.k, next0, next8, c + 2 - CHUNKS, t, a.head_dim);
                }
                if (more) values_of(second ? 0u : 16u);
            }
            key0 = next0;
            key8 = next8;
            second = !second;
        }
        run.add_up();
    }

    static __device__ __forceinline__ char *out_of(const Args &a, unsigned entry, unsigned kv_head, unsigned in_group) {
        return a.out + ((size_t)entry * a.out_row + (size_t)(kv_head * a.group + in_group) * a.out_head) * SIZE;
    }
    // A whole item's outputs from one warp's registers.
    static __device__ __forceinline__ void finish(const Args &a, const Share &s, const Run &run) {
        const unsigned g = threadIdx.x % 32 >> 2, t = threadIdx.x & 3;
        #pragma unroll
        for (int n = 0; n < TILES; n++)
            #pragma unroll
            for (int j = 0; j < 2; j++) {
                const unsigned in_group = s.chunk * HEADS + n * 8 + 2 * t + j;
                const float inv = run.sum[n][j] == 0.f ? 0.f : 1.f / run.sum[n][j];
                if (in_group >= a.group) continue;
                char *row = out_of(a, s.entry, s.kv_head, in_group);
                constexpr int PER = 16 / SIZE;
                #pragma unroll
                for (int i = 0; i < Run::PIECES; i++)
                    #pragma unroll
                    for (int h = 0; h < Run::PIECE; h += PER) {
                        const unsigned f = Run::feature(i, g) + h;
                        float v[PER];
                        #pragma unroll
                        for (int x = 0; x < PER; x++) v[x] = run.value(n, i, h + x, j) * inv;
                        if (f < a.head_dim) store_piece<TYPE>(row + f * SIZE, v);
                    }
            }
    }
    // A shared item's part to the warp's place in shared memory.
    static __device__ __forceinline__ void keep(float *at, const Run &run, unsigned heads) {
        const unsigned g = threadIdx.x % 32 >> 2, t = threadIdx.x & 3;
        #pragma unroll
        for (int n = 0; n < TILES; n++)
            #pragma unroll
            for (int j = 0; j < 2; j++) {
                if (n * 8 + 2 * t + j >= heads) continue;
                float *row = at + (n * 8 + 2 * t + j) * ROW;
                #pragma unroll
                for (int i = 0; i < Run::PIECES; i++)
                    #pragma unroll
                    for (int x = 0; x < Run::PIECE; x += 4)
                        *reinterpret_cast<float4 *>(row + Run::feature(i, g) + x) = make_float4(run.value(n, i, x, j), run.value(n, i, x + 1, j), run.value(n, i, x + 2, j), run.value(n, i, x + 3, j));
                if (g == 0) *reinterpret_cast<float2 *>(row + DIM) = make_float2(run.max[n][j], run.sum[n][j]);
            }
    }
};

template <int TYPE, int DIM, int HEADS, bool WIDE>
__global__ void __launch_bounds__(threads_of(TYPE, DIM, HEADS), ctas_of(TYPE, DIM)) decode_kernel(const Args a) {
    typedef Kernel<TYPE, DIM, HEADS, WIDE> K;
    typedef typename K::Run Run;
    extern __shared__ __align__(16) float kept[];             // [place][HEADS][ROW]; places: two of each warp, an item that began before its share and one that goes on behind it
    constexpr unsigned PLACES = K::WARPS * 2;
    static_assert(PLACES <= 32, "a lane a place");
    __shared__ Line<K::THREADS> line;
    __shared__ int item_of[PLACES], whole_of[PLACES];         // the item (-1: none); bit 0: the place has its first step, bit 1: its last
    __shared__ unsigned long long last_of[PLACES];            // the item's last step, in the line
    const unsigned lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    attn::let_next_kernel_start();
    attn::wait_for_previous_kernel();
    const unsigned each = (a.entries + K::THREADS - 1) / K::THREADS, items = a.kv_heads * a.chunks;
    if (threadIdx.x < PLACES) item_of[threadIdx.x] = -1;
    if (threadIdx.x == 0) a.record[2 * blockIdx.x] = -1;
    measure<TYPE, K::THREADS>(a, each, line);
    const unsigned long long all = line.before[K::THREADS];
    // CTAs that get a share: a step for each of their warps at least, so that little is joined where little is to do
    const unsigned ctas = (unsigned)min((unsigned long long)gridDim.x, (all + K::WARPS - 1) / K::WARPS);
    if (blockIdx.x >= ctas) return;
    const unsigned long long cta0 = attn::first_step(all, blockIdx.x, ctas), cta1 = attn::first_step(all, blockIdx.x + 1, ctas);
    const unsigned long long steps = cta1 - cta0;
    const unsigned warps = (unsigned)min((unsigned long long)K::WARPS, steps);          // the first ones, if there are fewer steps than warps
    unsigned long long pos = cta0 + attn::first_step(steps, warp, warps);
    const unsigned long long end = cta0 + attn::first_step(steps, warp + 1, warps);
    if (warp < warps) {
        // the last thread whose entries begin at pos or before: of every WARPS-th one, then of the WARPS behind it
        const unsigned block = 31 - __clz(__ballot_sync(0xffffffffu, line.before[lane * K::WARPS] <= pos));
        const unsigned lo = block * K::WARPS + 31 - __clz(__ballot_sync(0xffffffffu, lane < K::WARPS && line.before[block * K::WARPS + lane] <= pos));
        unsigned e = lo * each;
        unsigned long long base = line.before[lo];
        while (pos < end) {
            Share s;
            unsigned n;
            // bounded by the number of entries: `end` does not lie behind the last one's steps
            for (;; e++) {
                line.entry(a, each, e, s.slot, s.tokens);
                n = steps_of(s.tokens);
                if (base + (unsigned long long)n * items > pos || e + 1 >= a.entries) break;
                base += (unsigned long long)n * items;
            }
            const unsigned long long rel = pos - base;
            if (rel >= (unsigned long long)n * items) break;           // lengths that changed under the call
            const unsigned item = rel >> 32 ? (unsigned)(rel / n) : (unsigned)rel / n;
            s.entry = e;
            s.kv_head = item / a.chunks;
            s.chunk = item - s.kv_head * a.chunks;
            s.begin = (unsigned)(rel - (unsigned long long)item * n);
            s.end = (unsigned)min((unsigned long long)n, s.begin + (end - pos));
            Run run;
            K::walk(a, s, run);
            if (s.begin == 0 && s.end == n) K::finish(a, s, run);
            else {
                const unsigned place = warp * 2 + (s.begin != 0 ? 0 : 1);
                K::keep(kept + (size_t)place * HEADS * K::ROW, run, min((unsigned)HEADS, a.group - s.chunk * HEADS));
                if (lane == 0) {
                    item_of[place] = (int)(e * items + item);
                    whole_of[place] = (s.begin == 0 ? 1 : 0) | (s.end == n ? 2 : 0);
                    last_of[place] = base + (unsigned long long)(item + 1) * n - 1;
                }
            }
            pos += s.end - s.begin;
        }
    }
    __syncthreads();
    // Items that warps share.  One's parts are the place where it begins, or the first of a warp that has some of what began before, and the first places of the warps behind.
    // A warp joins one head of one item: a lane weighs a part each, then four features.
    const int place_item = lane < PLACES ? item_of[lane] : -1, place_whole = lane < PLACES ? whole_of[lane] : 0;
    const unsigned same = __match_any_sync(0xffffffffu, place_item), leaders = __ballot_sync(0xffffffffu, place_item >= 0 && (same & ((1u << lane) - 1u)) == 0);
    const unsigned rows = min((unsigned)HEADS, a.group);
    unsigned left = leaders, gone = 0;
    for (unsigned task = warp; task < __popc(leaders) * rows; task += K::WARPS) {
        for (; gone < task / rows; gone++) left &= left - 1;
        const unsigned r = task - gone * rows, first = __ffs(left) - 1, places = __shfl_sync(0xffffffffu, same, first), count = __popc(places);
        const bool begins = __shfl_sync(0xffffffffu, place_whole, first) & 1, ends = __shfl_sync(0xffffffffu, place_whole, 31 - __clz(places)) & 2;
        const unsigned item = (unsigned)__shfl_sync(0xffffffffu, place_item, first), e = item / items, rest = item - e * items, kv_head = rest / a.chunks, chunk = rest - kv_head * a.chunks;
        if (chunk * HEADS + r >= a.group) continue;
        auto row = [&](unsigned i) { return kept + ((i ? (first / 2 + i) * 2 : first) * HEADS + r) * K::ROW; };
        const float2 mine = lane < count ? *reinterpret_cast<const float2 *>(row(lane) + DIM) : make_float2(-INFINITY, 0.f);
        float max = mine.x;
        #pragma unroll
        for (int o = 16; o > 0; o >>= 1) max = fmaxf(max, __shfl_xor_sync(0xffffffffu, max, o));
        const float weight = mma::exp2_fast(mine.x - (max == -INFINITY ? 0.f : max));
        float sum = weight * mine.y;
        #pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        float *const part = a.part + (((size_t)blockIdx.x * 2 + (begins ? 1 : 0)) * HEADS + r) * K::ROW;
        #pragma unroll
        for (unsigned f0 = 0; f0 < DIM; f0 += 128) {
            const unsigned f = f0 + lane * 4;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            #pragma unroll 4
            for (unsigned i = 0; i < count; i++) {
                const float w = __shfl_sync(0xffffffffu, weight, i);
                if (DIM < 128 && f >= DIM) continue;
                const float4 p = *reinterpret_cast<const float4 *>(row(i) + f);
                v.x = fmaf(w, p.x, v.x); v.y = fmaf(w, p.y, v.y); v.z = fmaf(w, p.z, v.z); v.w = fmaf(w, p.w, v.w);
            }
            if (f >= DIM) continue;
            if (!begins || !ends) *reinterpret_cast<float4 *>(part + f) = v;
            else if (f < a.head_dim) {
                char *const out = K::out_of(a, e, kv_head, chunk * HEADS + r) + f * K::SIZE;
                if constexpr (TYPE == ASPEN_B200_FP32) *reinterpret_cast<float4 *>(out) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
                else *reinterpret_cast<uint2 *>(out) = make_uint2(mma::Of<TYPE>::pack(v.x * inv, v.y * inv), mma::Of<TYPE>::pack(v.z * inv, v.w * inv));
            }
        }
        if (lane == 0 && (!begins || !ends)) {
            *reinterpret_cast<float2 *>(part + DIM) = make_float2(max, sum);
            // the joining kernel has to know of one that goes on behind the CTA
            if (begins && r == 0) { a.record[2 * blockIdx.x + 1] = (int)attn::part_of_step(all, last_of[first], ctas); a.record[2 * blockIdx.x] = (int)item; }
        }
    }
}

// Items that several CTAs had a part of: block (b, r) joins head r of the one that began in CTA b and went on.
template <int TYPE, int DIM, int HEADS>
__global__ void __launch_bounds__(DIM) join_kernel(const Args a) {
    typedef Kernel<TYPE, DIM, HEADS, true> K;
    constexpr unsigned AT_ONCE = DIM;
    __shared__ float weight[AT_ONCE], maxima[DIM / 32], sums[DIM / 32];
    attn::wait_for_previous_kernel();
    const int item = a.record[2 * blockIdx.x];
    if (item < 0) return;
    const unsigned parts = (unsigned)a.record[2 * blockIdx.x + 1] - blockIdx.x + 1, items = a.kv_heads * a.chunks;      // of the CTAs from this one on
    const unsigned e = (unsigned)item / items, rest = (unsigned)item % items, kv_head = rest / a.chunks, chunk = rest % a.chunks, f = threadIdx.x;
    const unsigned in_group = chunk * HEADS + blockIdx.y;
    if (in_group >= a.group) return;
    constexpr size_t SLOT = (size_t)HEADS * K::ROW;
    // this CTA's second place, then the first places of the CTAs behind it
    const float *const first = a.part + ((size_t)blockIdx.x * 2 + 1) * SLOT + blockIdx.y * K::ROW;
    auto at = [&](unsigned i) { return first + (i ? (2 * (size_t)i - 1) * SLOT : 0); };
    // few parts: all that a thread needs is asked for at once
    constexpr unsigned FEW = 8;
    if (parts <= FEW) {
        float m[FEW], l[FEW], x[FEW], max = -INFINITY, sum = 0.f, v = 0.f;
        #pragma unroll
        for (unsigned i = 0; i < FEW; i++) {
            m[i] = -INFINITY; l[i] = x[i] = 0.f;
            if (i < parts) { const float *const p = at(i); m[i] = p[DIM]; l[i] = p[DIM + 1]; x[i] = p[f]; }
        }
        #pragma unroll
        for (unsigned i = 0; i < FEW; i++) max = fmaxf(max, m[i]);
        const float ref = max == -INFINITY ? 0.f : max;
        #pragma unroll
        for (unsigned i = 0; i < FEW; i++) { const float w = mma::exp2_fast(m[i] - ref); sum = fmaf(w, l[i], sum); v = fmaf(w, x[i], v); }
        if (f < a.head_dim) store_value<TYPE>(K::out_of(a, e, kv_head, in_group) + f * K::SIZE, sum == 0.f ? 0.f : v / sum);
        return;
    }
    float max = -INFINITY;
    for (unsigned i = f; i < parts; i += DIM) max = fmaxf(max, at(i)[DIM]);
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) max = fmaxf(max, __shfl_xor_sync(0xffffffffu, max, o));
    if (f % 32 == 0) maxima[f / 32] = max;
    __syncthreads();
    #pragma unroll
    for (int i = 0; i < DIM / 32; i++) max = fmaxf(max, maxima[i]);
    const float ref = max == -INFINITY ? 0.f : max;
    float v = 0.f, sum = 0.f;
    for (unsigned i0 = 0; i0 < parts; i0 += AT_ONCE) {
        __syncthreads();
        if (i0 + f < parts) {
            const float *const p = at(i0 + f);
            const float w = mma::exp2_fast(p[DIM] - ref);
            weight[f] = w;
            sum = fmaf(w, p[DIM + 1], sum);
        }
        __syncthreads();
        const unsigned n = min(AT_ONCE, parts - i0);
        #pragma unroll 8
        for (unsigned i = 0; i < n; i++) v = fmaf(weight[i], at(i0 + i)[f], v);
    }
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (f % 32 == 0) sums[f / 32] = sum;
    __syncthreads();
    sum = 0.f;
    #pragma unroll
    for (int i = 0; i < DIM / 32; i++) sum += sums[i];
    if (f < a.head_dim) store_value<TYPE>(K::out_of(a, e, kv_head, in_group) + f * K::SIZE, sum == 0.f ? 0.f : v / sum);
}

size_t workspace_bytes(unsigned sms, unsigned heads, unsigned dim, int type) {
    const size_t ctas = (size_t)sms * ctas_of(type, dim);
    return ctas * 16 + ctas * 2 * heads * (dim + 4) * 4;
}

template <int TYPE, int DIM, int HEADS, bool WIDE>
cudaError_t launch(const Args &a, unsigned sms, cudaStream_t stream) {
    typedef Kernel<TYPE, DIM, HEADS, WIDE> K;
    constexpr unsigned CTAS = ctas_of(TYPE, DIM);
    cudaError_t err = cudaFuncSetAttribute(decode_kernel<TYPE, DIM, HEADS, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, K::SMEM);
    if (err != cudaSuccess) return err;
    err = attn::launch_early(decode_kernel<TYPE, DIM, HEADS, WIDE>, sms * CTAS, K::THREADS, K::SMEM, stream, a);
    if (err != cudaSuccess) return err;
    return attn::launch_early(join_kernel<TYPE, DIM, HEADS>, dim3(sms * CTAS, a.group < HEADS ? a.group : HEADS), DIM, 0, stream, a);
}
template <int TYPE, bool WIDE>
cudaError_t launch(const Args &a, unsigned heads, unsigned dim, unsigned sms, cudaStream_t stream) {
    if (dim == 64) return heads == 8 ? launch<TYPE, 64, 8, WIDE>(a, sms, stream) : launch<TYPE, 64, 16, WIDE>(a, sms, stream);
    if (dim == 256) return launch<TYPE, 256, 8, WIDE>(a, sms, stream);
    if constexpr (TYPE != ASPEN_B200_FP32) if (heads == 16) return launch<TYPE, 128, 16, WIDE>(a, sms, stream);
    return launch<TYPE, 128, 8, WIDE>(a, sms, stream);
}
template <int TYPE>
cudaError_t launch(const Args &a, bool wide, unsigned heads, unsigned dim, unsigned sms, cudaStream_t stream) {
    return wide ? launch<TYPE, true>(a, heads, dim, sms, stream) : launch<TYPE, false>(a, heads, dim, sms, stream);
}

int check_heads(const aspen_b200_cache_t *cache, unsigned entries, unsigned heads, const char *what) {
    const int rc = attn::check_cache(cache, what, false);
    if (rc) return rc;
    if (!heads || heads % cache->kv_heads) { ASPEN_ERR("%s: %u heads of queries, %u of keys\n", what, heads, cache->kv_heads); return -1; }
    if ((unsigned long long)entries * heads > 0x7fffffffull || heads > 0xffffu) { ASPEN_ERR("%s: %u x %u rows of queries\n", what, entries, heads); return -2; }
    return 0;
}

}  // namespace

extern "C" size_t aspen_b200_attention_decode_workspace(const aspen_b200_cache_t *cache, unsigned int entries, unsigned int heads) {
    const char *what = "aspen_b200_attention_decode_workspace";
    if (check_heads(cache, entries, heads, what)) return 0;
    const int sms = attn::sm_count(what);
    if (sms < 0) return 0;
    const unsigned dim = dim_of(cache->head_dim);
    return workspace_bytes((unsigned)sms, heads_of_pass(heads / cache->kv_heads, dim, cache->type), dim, cache->type);
}

extern "C" int aspen_b200_attention_decode(const aspen_b200_cache_t *cache, unsigned int layer, const aspen_b200_decode_t *d, void *cuda_stream) {
    const char *what = "aspen_b200_attention_decode";
    if (!d) { ASPEN_ERR("%s: no arguments\n", what); return -1; }
    int rc = check_heads(cache, d->entries, d->heads, what);
    if (rc) return rc;
    if (layer >= cache->layers) { ASPEN_ERR("%s: layer %u of %u\n", what, layer, cache->layers); return -1; }
    if (!d->entries) return 0;
    if (!(d->scale - d->scale == 0.f)) { ASPEN_ERR("%s: scale is not finite\n", what); return -1; }
    if (!d->slots && d->entries > cache->sequences) { ASPEN_ERR("%s: %u entries, %u sequences\n", what, d->entries, cache->sequences); return -1; }
    if ((rc = attn::check_rows(d->q, d->q_row_stride, d->q_head_stride, cache->type, "q", what)) ||
        (rc = attn::check_rows(d->out, d->out_row_stride, d->out_head_stride, cache->type, "out", what))) return rc;
    const attn::Named ints[] = {{d->slots, "slots"}};
    if ((rc = attn::check_ints(ints, 1, what))) return rc;
    if (!d->workspace || reinterpret_cast<uintptr_t>(d->workspace) % 16) { ASPEN_ERR("%s: no workspace, or not on a 16-byte boundary\n", what); return -1; }
    const int sms = attn::sm_count(what);
    if (sms < 0) return sms;
    const unsigned group = d->heads / cache->kv_heads, dim = dim_of(cache->head_dim), heads = heads_of_pass(group, dim, cache->type);
    const size_t need = workspace_bytes((unsigned)sms, heads, dim, cache->type);
    if (d->workspace_bytes < need) { ASPEN_ERR("%s: a workspace of %zu bytes; %zu are needed\n", what, d->workspace_bytes, need); return -1; }
    const attn::Named all[] = {{cache->k, "the cache's k"}, {cache->v, "the cache's v"}, {cache->page_table, "page_table"}, {cache->lengths, "lengths"}, {cache->status, "status"},
                               {d->q, "q"}, {d->out, "out"}, {d->slots, "slots"}, {d->workspace, "workspace"}};
    if ((rc = attn::check_device(all, 9, what))) return rc;
    Args a;
    a.at = attn::pages_of(*cache);
    const size_t size = attn::type_size(cache->type), skip = layer * attn::packed(cache->layer_stride, a.at.page_stride * cache->pages) * size;
    a.k = static_cast<const char *>(cache->k) + skip;
    a.v = static_cast<const char *>(cache->v) + skip;
    a.q = static_cast<const char *>(d->q);
    a.out = static_cast<char *>(d->out);
    a.slots = d->slots;
    a.q_row = attn::packed(d->q_row_stride, (size_t)d->heads * cache->head_dim);
    a.q_head = attn::packed(d->q_head_stride, cache->head_dim);
    a.out_row = attn::packed(d->out_row_stride, (size_t)d->heads * cache->head_dim);
    a.out_head = attn::packed(d->out_head_stride, cache->head_dim);
    a.entries = d->entries;
    a.kv_heads = cache->kv_heads;
    a.group = group;
    a.chunks = (group + heads - 1) / heads;
    a.head_dim = cache->head_dim;
    a.scale = d->scale * 1.4426950408889634f;
    const size_t ctas = (size_t)sms * ctas_of(cache->type, dim);
    a.record = static_cast<int *>(d->workspace);
    a.part = reinterpret_cast<float *>(static_cast<char *>(d->workspace) + ctas * 16);
    const cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
    // rows of keys and values on 32-byte boundaries, and whole pieces of 32 bytes in them: one load a piece instead of two
    const size_t starts = reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) | (a.at.page_stride | a.at.head_stride | a.at.token_stride | cache->head_dim) * size;
    const bool wide = starts % 32 == 0;
    cudaError_t err;
    switch (cache->type) {
        case ASPEN_B200_FP32: err = launch<ASPEN_B200_FP32>(a, wide, heads, dim, (unsigned)sms, stream); break;
        case ASPEN_B200_BF16: err = launch<ASPEN_B200_BF16>(a, wide, heads, dim, (unsigned)sms, stream); break;
        default: err = launch<ASPEN_B200_FP16>(a, wide, heads, dim, (unsigned)sms, stream); break;
    }
    if (err != cudaSuccess) { cudaGetLastError(); ASPEN_ERR("%s: %s\n", what, cudaGetErrorString(err)); return -3; }
    return 0;
}
