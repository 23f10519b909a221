// Attention over whole prompts on tcgen05, 16-bit types, heads of up to 128 features.
//
// A CTA takes two tiles of 128 rows that see the same head of keys and walks their keys, 128 a step.  A row is a query with one of the heads of the group: 128 / group queries to a
// tile, so that short prompts fill it, too.
//     S [128 rows x 128 keys] = Q K^T     both operands in shared memory, K-major, scores in TMEM
//     P = exp2(S - max)                      a thread a row: its scores from TMEM to registers, weights back to TMEM as 16-bit pairs
//     O [128 rows x features] += P V         P from TMEM, V as it lies in memory (features contiguous: the MN-major operand), sums in TMEM
// The maximum is followed loosely, a known variant of the running softmax: O and the sum are scaled again only when a row's maximum has grown by more than 2^8 (weights up to 256 are as
// exact as weights up to 1), so the sums in TMEM are hardly ever read before the end.  fp16: by more than 2^5, from 2^10, so that weights stay below 2^15 and small ones keep their bits (mma_sync.cuh).
//
// Warps: 0 - 3 and 4 - 7 the softmax of the two tiles, 8 TMA, 9 MMA (with 64 features 9 and 11, a tile each), 10 finds the work, 12 - 15 write outputs; nothing but mbarriers connects them, and while one tile's scores are weighed
// the other's are multiplied.  The first three quarters of a tile's weights are multiplied while the last one is computed.  TMEM, 512 columns: scores 2 x 128, sums 2 x features, and with 64
// features weights 2 x 64 of their own, so that the next scores, the next job's too, are there before the weights of these have been multiplied; with 128 the weights take the place of their
// scores.
//
// A CTA takes job after job: heavy and light ones, whatever the lengths, so the hardware deals them (a running CTA takes over the work of one that has not begun).  The next one is asked
// for three steps before this one ends, and its queries and keys come in under the last steps.  (Asked for at once, CTAs held up to three jobs: of 24 packed prompts one had 8 steps and
// another 25; dealt in turn, 4 prompts of 1231 to 4096 tokens took 152 units of time where 120 are possible.)
//
// What bounds it.  With 128 features a step of two tiles takes 2048 cycles of the tensor pipe at best, and as many of shared memory (Q and K are read from there for each
// product, 128 bytes a cycle; the copies of K and V come on top); with 64 features 1024, and 2048 of the unit for exp2.  4 prompts of 1231 to 4096 tokens, 32 heads over 8 of
// 128: 227 us, 1100 TFLOP/s of visible products, 3600 cycles a step: the chain of a tile (scores from TMEM 100, maximum 270, exponentials and sums 1250, then its products 900)
// is as long as that with the other tile's in between.  24 packed prompts of 12 heads of 64: 46.5 us; the exp2 unit is busy for 45 %
// of it: two tiles in the same phase of a step take 1.7 us for it, in opposite ones 1.35, and starts and ends of jobs of 2.2 steps a tile come on top.
// Tried and slower: two threads a query (16 warps: registers), a quarter of the exponentials by polynomials in packed multiply-adds (FMA and ALU then take what the exp2 unit gives; their
// second copy of the code costs instruction fetches), weights from the maximum of the step before with a second try (the same), 32 keys a turn in a loop (24 packed prompts 72 us), blocks of keys
// that a warp does not see left out by branches (50 us), a late start for the second tile (the same), and for 64 features two CTAs on an SM with steps of 64 keys (49 us; one prompt of 4096 tokens
// 79 instead of 56: a tile alone is slower).
//
// Values behind the end of a sequence are another one's, or nobody's: an MMA warp sets them to zero in shared memory, since 0 x NaN would reach every row.
//
// Every wait is bounded (2 s, or 2 s and 100 us a step) and is for another role of the CTA; if one runs out all roles leave, TMEM is freed, the rows of out that were in work become NaN, those
// not begun stay, and the caller's status word says so.
#pragma once
#include "tiles_tc.cuh"

#include <cuda.h>

namespace fused {

constexpr unsigned THREADS = 512, TILE = 128;
constexpr unsigned long long LIMIT_NS = 2000000000ull;

template <int DIM>
struct Shape {
    static constexpr int CHUNKS = DIM / 64;                         // of 64 features: 128 bytes, the swizzle's width
    static constexpr int CHUNK_BYTES = TILE * 128, BYTES = CHUNKS * CHUNK_BYTES;    // of a tile of queries, keys or values
    static constexpr int STAGES = DIM == 64 ? 4 : 2, QUERIES = DIM == 64 ? 2 : 1;     // buffers: keys and values; queries of both tiles
    static constexpr int OUT_BYTES = 4 * 2048;                      // where a warp turns its outputs round
    static constexpr int SMEM = 2 * QUERIES * BYTES + 2 * STAGES * BYTES + OUT_BYTES + 1024;
    static constexpr bool OWN_P = DIM == 64;
    // With weights of their own the tiles need nothing of each other, and a warp for each lets them: 24 packed prompts 46.9 us, 48.7 with one for both.  Without, one warp keeps the products
    // of one tile behind the other's: 4 long prompts 224.6 us, 229.4 with two.
    static constexpr int MMA_WARPS = OWN_P ? 2 : 1;
    static constexpr unsigned S = 0, O = 256, P = OWN_P ? 384 : 0, P_APART = OWN_P ? 64 : 128;      // TMEM columns
};

// fp32, heads of up to 64 features: every operand as three bf16 parts, six of the nine products.
struct Parts {
    static constexpr int BYTES = TILE * 128;                        // a part of a tile: 128 rows of 64 features
    static constexpr int SMEM = 12 * BYTES + 8 * 4096 + 1024;       // two tiles of queries, keys, values; outputs being turned round
    static constexpr unsigned O = 192;                              // TMEM columns of a tile: scores 128 (then two parts of the weights), the third part 64, a product 64
    // the parts of product p: 2 0, 1 1, 0 2, 1 0, 0 1, 0 0
    static __device__ __forceinline__ unsigned first(int p) { return 0x001012u >> (4 * p) & 15u; }
    static __device__ __forceinline__ unsigned second(int p) { return 0x010210u >> (4 * p) & 15u; }
};

// A CTA's work: two tiles of one sequence and one head of keys.  A tile is `block` queries with all heads of the group: row r is query first + r / group, head r % group.
struct Job {
    int q0, queries, k0, keys;
    int kv_head, block;
    int first[2], steps[2];                        // first query of a tile, -1: no such tile; steps of 128 keys
    int live;                                      // 0: there are no more
    __device__ __forceinline__ int both() const { return max(steps[0], steps[1]); }
    __device__ __forceinline__ int behind() const { return keys - queries; }
    __device__ __forceinline__ int end(int w, int masked) const { return masked ? max(0, min(keys, min(queries, first[w] + block) + behind())) : keys; }
};
constexpr unsigned JOBS = 2;                       // the one in work and the next

struct Shared {
    uint4 answer;                                  // to a request for another CTA's work
    unsigned long long answered, wanted, job_full[JOBS], job_empty[JOBS];
    unsigned long long q_full[2][2], q_empty[2][2], k_full[4], k_empty[4], v_full[4], v_empty[4], v_clean[4];      // q: [buffer][tile]
    unsigned long long s_full[2], s_free[2], p_full[2][2], o_full[2];
    unsigned long long o_done[2], o_free[2], l_full[2];                                                // a job's sums: complete, read; the rows' factors
    Job jobs[JOBS];
    float factor[2][TILE];
    unsigned gave_up, tmem;
};

// The hardware deals the CTAs of the grid; one that runs asks for the next that has not begun, which then never does.
__device__ __forceinline__ void ask_for_work(Shared *sh) {
    tc::mbar_arrive_expect_tx(&sh->answered, 16u);
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(tc::smem_u32(&sh->answer)), "r"(tc::smem_u32(&sh->answered)) : "memory");
}
// The number of the CTA whose work this one has been given; false: none is left.
__device__ __forceinline__ bool given_work(Shared *sh, unsigned &index) {
    unsigned yes;
    asm volatile("{\n\t.reg .b128 h;\n\t.reg .pred p;\n\tld.shared.b128 h, [%2];\n\tclusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\tselp.u32 %0, 1, 0, p;\n\t"
                 "mov.u32 %1, 0;\n\t@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, h;\n\t}" : "=r"(yes), "=r"(index) : "r"(tc::smem_u32(&sh->answer)) : "memory");
    return yes != 0u;
}

__device__ __forceinline__ bool wait(unsigned long long *bar, unsigned parity, unsigned *gave_up, unsigned long long limit) {
    #pragma unroll 1
    for (unsigned spin = 0; spin < 4096u; spin++)
        if (tc::mbar_try_wait(bar, parity)) return true;
    unsigned long long t0, now;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t0));
    #pragma unroll 1
    for (unsigned spin = 1;; spin++) {
        if (tc::mbar_try_wait(bar, parity)) return true;
        if ((spin & 255u) == 0u) {
            asm volatile("mov.u64 %0, %globaltimer;" : "=l"(now));
            if (*(volatile unsigned *)gave_up != 0u) return false;
            if (now - t0 > limit) { atomicExch(gave_up, 1u); return false; }
        }
    }
}
// A warp's lanes wait, and give up, together.
__device__ __forceinline__ bool warp_wait(unsigned long long *bar, unsigned parity, unsigned *gave_up, unsigned long long limit = LIMIT_NS) {
    return __all_sync(0xffffffffu, wait(bar, parity, gave_up, limit));
}
// For something that comes at the end of a job: 100 us a step more.
__device__ __forceinline__ unsigned long long whole_job(int steps) { return LIMIT_NS + 100000ull * (unsigned)steps; }

// Both operands in shared memory, K-major, 128-byte swizzle; or A in TMEM and B with features contiguous (MN-major): 64 features of a row side by side, the next 64
// CHUNK_BYTES on, eight keys 1024 bytes.
__device__ __forceinline__ void mma_ss(unsigned d, unsigned a, unsigned b, unsigned idesc, unsigned accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 x, {%1, %5};\n\tmov.b64 y, {%2, %5};\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(tc::UMMA_DESC_HIGH) : "memory");
}
__device__ __forceinline__ void mma_ts(unsigned d, unsigned a, unsigned b, unsigned idesc, unsigned accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 y;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 y, {%2, %5};\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(tc::UMMA_DESC_HIGH) : "memory");
}

// 32 columns of the warp's lanes, not waited for.
__device__ __forceinline__ void ld32(unsigned at, float *v) {
    unsigned *r = reinterpret_cast<unsigned *>(v);
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                   "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                   "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(at) : "memory");
}
// The loads before are done; what they loaded is used behind this only.
__device__ __forceinline__ void ld_done32(float *v) {
    unsigned *r = reinterpret_cast<unsigned *>(v);
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                   "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]) : : "memory");
    asm volatile("" : "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]) : : "memory");
}
__device__ __forceinline__ void ld16(unsigned at, float *v) {
    unsigned *r = reinterpret_cast<unsigned *>(v);
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ld_done16(float *v) {
    unsigned *r = reinterpret_cast<unsigned *>(v);
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]) : : "memory");
}
__device__ __forceinline__ void st16(unsigned at, const unsigned *r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
                 ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                   "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void st_done() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

typedef unsigned long long Pair;         // two fp32 values
__device__ __forceinline__ Pair pair(float x, float y) { Pair p; asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(x), "f"(y)); return p; }
__device__ __forceinline__ void unpair(Pair p, float &x, float &y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(p)); }
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) { Pair d; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c)); return d; }
__device__ __forceinline__ Pair add2(Pair a, Pair b) { Pair d; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b)); return d; }

__device__ __forceinline__ float max3(float a, float b, float c) { float d; asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c)); return d; }
__device__ __forceinline__ float max2(float a, float b) { float d; asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b)); return d; }

}  // namespace fused
