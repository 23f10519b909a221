// Attention over whole prompts, packed one behind the other.
//
// One pass over the keys of a block of queries, with the running maximum and sum of the softmax; scores never leave the SM.
//
// prompt_rows (any type, any head): a warp has 16 queries, its operands and sums in registers as mma.sync takes them (mma_sync.cuh); keys and values of a tile go through
// shared memory for the four warps of a CTA, asked for one tile ahead.  Rows in shared memory are 64 (keys) and 16 bytes (values) longer than a power of two, so that the 16-byte pieces
// that eight lanes read together lie in different banks.
#include "mma_sync.cuh"

#include <cuda_runtime.h>

namespace {

struct Args {
    const char *q, *k, *v;
    char *out;
    const int *q_starts, *kv_starts;
    size_t q_row, q_head, k_row, k_head, v_row, v_head, out_row, out_head;      // in elements
    unsigned sequences, q_rows, kv_rows, heads, group, head_dim;
    int masked;
    float scale;                        // with log2(e)
};

// A block of queries: rows first ... of the sequence that begins at row q0.
struct Block {
    int q0, queries, k0, keys, first;
};

__device__ __forceinline__ int clamped(const int *starts, unsigned i, unsigned rows) { return min(max(starts[i], 0), (int)rows); }

// Block `index` of all sequences' blocks of `size` queries, counted from the first sequence; a sequence's last one first, because with a mask it has most
// keys.  Every warp finds it for itself, 32 sequences a turn.  False: there are not so many.
__device__ __forceinline__ bool find_block(const Args &a, unsigned index, unsigned size, Block &b) {
    const unsigned lane = threadIdx.x % 32;
    unsigned long long before = 0;
    for (unsigned s0 = 0; s0 < a.sequences; s0 += 32) {
        const unsigned s = s0 + lane;
        int q0 = 0, q1 = 0;
        if (s < a.sequences) { q0 = clamped(a.q_starts, s, a.q_rows); q1 = max(q0, clamped(a.q_starts, s + 1, a.q_rows)); }
        const unsigned n = ((unsigned)(q1 - q0) + size - 1) / size;
        unsigned long long sum = n;
        #pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const unsigned long long u = __shfl_up_sync(0xffffffffu, sum, o); if (lane >= (unsigned)o) sum += u; }
        const unsigned here = __ballot_sync(0xffffffffu, before + sum > index);
        if (here) {
            const int at = __ffs(here) - 1;
            const unsigned rank = (unsigned)(before + sum - 1 - index);           // of lane `at`: n - 1 for the first index of its sequence, 0 for the last
            const unsigned back = __shfl_sync(0xffffffffu, rank, at), blocks = __shfl_sync(0xffffffffu, n, at);
            b.q0 = __shfl_sync(0xffffffffu, q0, at);
            b.queries = __shfl_sync(0xffffffffu, q1, at) - b.q0;
            b.first = (int)((back < blocks ? back : 0u) * size);
            const unsigned mine = s0 + at;
            b.k0 = clamped(a.kv_starts, mine, a.kv_rows);
            b.keys = max(0, clamped(a.kv_starts, mine + 1, a.kv_rows) - b.k0);
            return true;
        }
        before += __shfl_sync(0xffffffffu, sum, 31);
    }
    return false;
}

__device__ __forceinline__ unsigned shared_address(const void *p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(unsigned to, const char *from, bool ok) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT> __device__ __forceinline__ void wait_copies() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

template <int TYPE, int DIM>
struct Rows {
    static constexpr int SIZE = TYPE == ASPEN_B200_FP32 ? 4 : 2, VALUES = 16 / SIZE, BYTES = DIM * SIZE;
    static constexpr int QUERIES = 64, KEYS = BYTES > 512 ? 32 : 64, THREADS = 128;
    static constexpr int KPITCH = BYTES + 64, VPITCH = BYTES + 16, STAGE = KEYS * (KPITCH + VPITCH);
    static constexpr bool HELD = BYTES <= 256;                  // queries stay in registers
    static constexpr int SMEM = 2 * STAGE + (HELD ? 0 : QUERIES * KPITCH);
    static constexpr int PIECES = DIM / (4 * VALUES);           // of a lane and row, product over features
    static constexpr int VPIECES = DIM / (8 * VALUES);
};

template <int TYPE, int DIM>
__global__ void __launch_bounds__(128) prompt_rows(const Args a) {
    typedef Rows<TYPE, DIM> R;
    constexpr int SIZE = R::SIZE, VALUES = R::VALUES, KT = R::KEYS / 8;
    extern __shared__ __align__(128) char smem[];
    const unsigned lane = threadIdx.x % 32, warp = threadIdx.x / 32, g = lane >> 2, t = lane & 3, head = blockIdx.y, kv_head = head / a.group;
    Block b;
    if (!find_block(a, blockIdx.x, R::QUERIES, b)) return;
    const int behind = b.keys - b.queries;                      // query i sees keys up to i + behind
    const int last = min(b.queries, b.first + R::QUERIES) - 1;
    const int end = a.masked ? min(b.keys, last + behind + 1) : b.keys;
    const int row0 = b.first + (int)warp * 16 + (int)g, row8 = row0 + 8;
    const char *const k = a.k + ((size_t)b.k0 * a.k_row + kv_head * a.k_head) * SIZE, *const v = a.v + ((size_t)b.k0 * a.v_row + kv_head * a.v_head) * SIZE;
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
    if (tiles > 0) fetch(0, 0);
    // queries, rows g and g + 8 of the warp's 16
    const char *const q = a.q + (size_t)b.q0 * a.q_row * SIZE + head * a.q_head * SIZE;
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
    for (int tile = 0; tile < tiles; tile++) {
        if (tile + 1 < tiles) { fetch(tile + 1, (tile + 1) & 1); wait_copies<1>(); } else wait_copies<0>();
        __syncthreads();
        const char *const ks = smem + (tile & 1) * R::STAGE, *const vs = ks + R::KEYS * R::KPITCH;
        float s[KT][4];
        #pragma unroll
        for (int n = 0; n < KT; n++)
            #pragma unroll
            for (int j = 0; j < 4; j++) s[n][j] = 0.f;
        #pragma unroll
        for (int i = 0; i < R::PIECES; i++) {
            const int f = (i * 4 * VALUES + t * VALUES) * SIZE;
            const uint4 x = R::HELD ? held[R::HELD ? 2 * i : 0] : *reinterpret_cast<const uint4 *>(own + g * R::KPITCH + f);
            const uint4 y = R::HELD ? held[R::HELD ? 2 * i + 1 : 0] : *reinterpret_cast<const uint4 *>(own + (g + 8) * R::KPITCH + f);
            #pragma unroll
            for (int n = 0; n < KT; n++) {
                const uint4 w = *reinterpret_cast<const uint4 *>(ks + (n * 8 + g) * R::KPITCH + f);
                if constexpr (TYPE == ASPEN_B200_FP32) {
                    const unsigned a0[4] = {x.x, y.x, x.y, y.y}, a1[4] = {x.z, y.z, x.w, y.w}, b0[2] = {w.x, w.y}, b1[2] = {w.z, w.w};
                    mma::tf32x3(s[n], a0, b0);
                    mma::tf32x3(s[n], a1, b1);
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
            for (int n = 0; n < KT; n++) {
                const unsigned p[4] = {__float_as_uint(s[n][0]), __float_as_uint(s[n][2]), __float_as_uint(s[n][1]), __float_as_uint(s[n][3])};
                const char *const row = vs + (n * 8 + 2 * t) * R::VPITCH;
                #pragma unroll
                for (int i = 0; i < R::VPIECES; i++) {
                    const uint4 x = *reinterpret_cast<const uint4 *>(row + (i * 32 + g * 4) * SIZE), y = *reinterpret_cast<const uint4 *>(row + R::VPITCH + (i * 32 + g * 4) * SIZE);
                    const unsigned w0[4] = {x.x, x.y, x.z, x.w}, w1[4] = {y.x, y.y, y.z, y.w};
                    #pragma unroll
                    for (int j = 0; j < 4; j++) { const unsigned w[2] = {w0[j], w1[j]}; mma::tf32x3(o[i * 4 + j], p, w); }
                }
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
        const int row = h ? row8 : row0;
        if (row >= b.queries) continue;
        const float inv = sum[h] == 0.f ? 0.f : 1.f / sum[h];
        char *const out = a.out + ((size_t)(b.q0 + row) * a.out_row + head * a.out_head) * SIZE;
        // column n = 2 t + c of tile j holds the value j of piece n
        constexpr int PER = TYPE == ASPEN_B200_FP32 ? 4 : 8;
        #pragma unroll
        for (int i = 0; i < R::VPIECES; i++)
            #pragma unroll
            for (int c = 0; c < 2; c++) {
                const unsigned f = i * 8 * PER + (2 * t + c) * PER;
                float x[PER];
                #pragma unroll
                for (int j = 0; j < PER; j++) x[j] = o[i * PER + j][2 * h + c] * inv;
                if (f >= a.head_dim) continue;
                if constexpr (TYPE == ASPEN_B200_FP32) *reinterpret_cast<float4 *>(out + f * SIZE) = make_float4(x[0], x[1], x[2], x[3]);
                else {
                    typedef mma::Of<TYPE> T;
                    *reinterpret_cast<uint4 *>(out + f * SIZE) = make_uint4(T::pack(x[0], x[1]), T::pack(x[2], x[3]), T::pack(x[4], x[5]), T::pack(x[6], x[7]));
                }
            }
    }
}

template <int TYPE, int DIM>
cudaError_t launch_rows(const Args &a, cudaStream_t stream) {
    typedef Rows<TYPE, DIM> R;
    cudaError_t err = cudaFuncSetAttribute(prompt_rows<TYPE, DIM>, cudaFuncAttributeMaxDynamicSharedMemorySize, R::SMEM);
    if (err != cudaSuccess) return err;
    const unsigned blocks = a.q_rows / R::QUERIES + (a.sequences < a.q_rows ? a.sequences : a.q_rows);
    prompt_rows<TYPE, DIM><<<dim3(blocks, a.heads), R::THREADS, R::SMEM, stream>>>(a);
    return cudaGetLastError();
}
template <int TYPE>
cudaError_t launch_rows(const Args &a, cudaStream_t stream) {
    return a.head_dim <= 64 ? launch_rows<TYPE, 64>(a, stream) : a.head_dim <= 128 ? launch_rows<TYPE, 128>(a, stream) : launch_rows<TYPE, 256>(a, stream);
}

}  // namespace

extern "C" int aspen_b200_attention_prompt(const aspen_b200_prompt_t *p, void *cuda_stream) {
    const char *what = "aspen_b200_attention_prompt";
    if (!p) { ASPEN_ERR("%s: no arguments\n", what); return -1; }
    int rc = attn::check_type(p->type, p->head_dim, what);
    if (rc) return rc;
    if (!p->heads || !p->kv_heads || p->heads % p->kv_heads) { ASPEN_ERR("%s: %u heads of queries, %u of keys\n", what, p->heads, p->kv_heads); return -1; }
    if (!(p->scale - p->scale == 0.f)) { ASPEN_ERR("%s: scale is not finite\n", what); return -1; }
    // rows are int on the device; block numbers and 128 rows past the end stay below 2^31
    if (p->q_rows > 0x3fffffffu || p->kv_rows > 0x3fffffffu || p->sequences > 0x3fffffffu || p->heads > 0xffffu) { ASPEN_ERR("%s: too many rows, sequences or heads\n", what); return -2; }
    if (!p->sequences || !p->q_rows) return 0;
    if (!p->q_starts || !p->kv_starts) { ASPEN_ERR("%s: q_starts or kv_starts is NULL\n", what); return -1; }
    if ((rc = attn::check_rows(p->q, p->q_row_stride, p->q_head_stride, p->type, "q", what)) || (rc = attn::check_rows(p->out, p->out_row_stride, p->out_head_stride, p->type, "out", what))) return rc;
    if (p->kv_rows && ((rc = attn::check_rows(p->k, p->k_row_stride, p->k_head_stride, p->type, "k", what)) || (rc = attn::check_rows(p->v, p->v_row_stride, p->v_head_stride, p->type, "v", what)))) return rc;
    const int sms = attn::sm_count(what);
    if (sms < 0) return sms;
    const attn::Named all[] = {{p->q, "q"}, {p->out, "out"}, {p->q_starts, "q_starts"}, {p->kv_starts, "kv_starts"}, {p->kv_rows ? p->k : nullptr, "k"}, {p->kv_rows ? p->v : nullptr, "v"}};
    if ((rc = attn::check_device(all, 6, what))) return rc;
    Args a;
    a.q = static_cast<const char *>(p->q);
    a.k = static_cast<const char *>(p->k);
    a.v = static_cast<const char *>(p->v);
    a.out = static_cast<char *>(p->out);
    a.q_starts = p->q_starts;
    a.kv_starts = p->kv_starts;
    const size_t q_row = (size_t)p->heads * p->head_dim, kv_row = (size_t)p->kv_heads * p->head_dim;
    a.q_row = attn::packed(p->q_row_stride, q_row);
    a.q_head = attn::packed(p->q_head_stride, p->head_dim);
    a.k_row = attn::packed(p->k_row_stride, kv_row);
    a.k_head = attn::packed(p->k_head_stride, p->head_dim);
    a.v_row = attn::packed(p->v_row_stride, kv_row);
    a.v_head = attn::packed(p->v_head_stride, p->head_dim);
    a.out_row = attn::packed(p->out_row_stride, q_row);
    a.out_head = attn::packed(p->out_head_stride, p->head_dim);
    a.sequences = p->sequences;
    a.q_rows = p->q_rows;
    a.kv_rows = p->kv_rows;
    a.heads = p->heads;
    a.group = p->heads / p->kv_heads;
    a.head_dim = p->head_dim;
    a.masked = p->masked != 0;
    a.scale = p->scale * 1.4426950408889634f;
    const cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
    const cudaError_t err = p->type == ASPEN_B200_FP32 ? launch_rows<ASPEN_B200_FP32>(a, stream) : p->type == ASPEN_B200_BF16 ? launch_rows<ASPEN_B200_BF16>(a, stream) : launch_rows<ASPEN_B200_FP16>(a, stream);
    if (err != cudaSuccess) { cudaGetLastError(); ASPEN_ERR("%s: %s\n", what, cudaGetErrorString(err)); return -3; }
    return 0;
}
