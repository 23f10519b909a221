// Warp-level matrix products (mma.sync) over operands that lanes hold as 16-byte pieces of rows (32-byte ones are two of them for the same lane), for fp32, bf16 and fp16.
//
// The products run over features or keys in any order, as long as both operands agree, so a lane takes the 16 bytes it has loaded as its part of
// consecutive k steps and nothing is rearranged:
//     features   lane (g, t) = (lane / 4, lane % 4) holds row g, values 8 t ... 8 t + 7 of 32 (16-bit; two steps of k = 16) or 4 t ... 4 t + 3 of 16 (fp32; two
//                steps of k = 8)
//     keys       lane (g, t) holds rows 2 t, 2 t + 1, 2 t + 8, 2 t + 9 of 16 keys, values 8 g ... of 64 (fp32: 4 g ... of 32); two rows are interleaved by byte permutes
//
// fp32: TF32 operands of 11 bits.  x = hi + lo, hi is x rounded to 11 bits and lo the rest, of which TF32 keeps 11 again (2^-22 of x is lost); hi hi + hi lo + lo hi leave
// out lo lo, 2^-22 of a product: 2^-20 in all at most.  Below 2^-104 lo loses bits that TF32 has no exponent for (2^-126 at most), and what hi rounds past the range becomes an infinity.  Sums are fp32.
#pragma once
#include "attention.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace mma {

__device__ __forceinline__ void bf16_16816(float *d, unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void fp16_16816(float *d, unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void tf32_1688(float *d, unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The two TF32 parts of an fp32 value.
__device__ __forceinline__ void parts(unsigned x, unsigned &hi, unsigned &lo) {
    hi = (x + 0x1000u) & 0xffffe000u;          // a NaN may become a zero here; the rest is NaN then
    lo = __float_as_uint(__uint_as_float(x) - __uint_as_float(hi)) & 0xffffe000u;
}
__device__ __forceinline__ void tf32x3(float *d, const unsigned *a, const unsigned *b) {
    unsigned ah[4], al[4], bh[2], bl[2];
    #pragma unroll
    for (int i = 0; i < 4; i++) parts(a[i], ah[i], al[i]);
    #pragma unroll
    for (int i = 0; i < 2; i++) parts(b[i], bh[i], bl[i]);
    tf32_1688(d, al[0], al[1], al[2], al[3], bh[0], bh[1]);
    tf32_1688(d, ah[0], ah[1], ah[2], ah[3], bl[0], bl[1]);
    tf32_1688(d, ah[0], ah[1], ah[2], ah[3], bh[0], bh[1]);
}

__device__ __forceinline__ unsigned transpose8(unsigned x) {
    unsigned y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// 2^x; -inf gives 0.
__device__ __forceinline__ float exp2_fast(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }

// Per type: TOP, the binary logarithm of the largest softmax weight.  fp16 ends at 2^-24, so with 2^15 at the top a weight keeps its 11 bits down to 2^-29 of the largest one; with 1 there, many keys
// of 2^-20 each beside one large one were off by up to 3 %, and those below 2^-25 were lost while the sum below the fraction had them.  The factor cancels in the fraction.
// VALUES of 16 bytes; one loaded piece is two k steps of the product over features (`features`), and a piece of each of four keys' rows is PIECE_TILES
// 16-row tiles of the product over 16 keys.
template <int TYPE> struct Of;

template <> struct Of<ASPEN_B200_BF16> {
    static constexpr int SIZE = 2, VALUES = 8;
    static constexpr float TOP = 0.f;
    static __device__ __forceinline__ void step(float *d, unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) { bf16_16816(d, a0, a1, a2, a3, b0, b1); }
    static __device__ __forceinline__ unsigned pack(float lo, float hi) { unsigned r; asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo)); return r; }
};
template <> struct Of<ASPEN_B200_FP16> {
    static constexpr int SIZE = 2, VALUES = 8;
    static constexpr float TOP = 15.f;
    static __device__ __forceinline__ void step(float *d, unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) { fp16_16816(d, a0, a1, a2, a3, b0, b1); }
    static __device__ __forceinline__ unsigned pack(float lo, float hi) { unsigned r; asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo)); return r; }
};
template <> struct Of<ASPEN_B200_FP32> { static constexpr int SIZE = 4, VALUES = 4; static constexpr float TOP = 0.f; };

// Two rows' pieces (x row 2 t, y row 2 t + 1 of 8 keys): the pairs of keys of value j.
__device__ __forceinline__ unsigned pair_of(unsigned x, unsigned y, bool high) { return __byte_perm(x, y, high ? 0x7632 : 0x5410); }

}  // namespace mma
