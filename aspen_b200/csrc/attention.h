// What the attention operators and the paged cache share: argument checks, the place of a token in the cache, and how the work of single tokens
// is cut.  The parts marked ATTN_FN are host code too (tests/native/attention_index.cpp).
#pragma once
#include "internal.h"

#include <cstdint>

#ifdef __CUDACC__
#define ATTN_FN __host__ __device__ __forceinline__
#else
#define ATTN_FN inline
#endif

namespace attn {

constexpr unsigned MAX_HEAD = 256;

ATTN_FN unsigned type_size(int type) { return type == ASPEN_B200_FP32 ? 4u : 2u; }

// The cache of one layer, strides in elements and never 0.
struct Pages {
    const int *table, *lengths;
    int *status;
    size_t page_stride, head_stride, token_stride;
    unsigned pages, page_size, sequences, max_pages;
    int *refused;                       // or nullptr
};

// Tokens of a sequence: 0 for one that does not exist, never more than its row of the table has room for.
ATTN_FN unsigned sequence_length(const Pages &c, int slot) {
    if (slot < 0 || (unsigned)slot >= c.sequences) return 0u;
    const int n = c.lengths[slot];
    const unsigned room = c.max_pages * c.page_size;         // < 2^31 (checked)
    return n <= 0 ? 0u : (unsigned)n < room ? (unsigned)n : room;
}
// A sequence that a refused call would have given tokens to; also where the cache keeps no list of them: never.
ATTN_FN bool is_refused(const Pages &c, int slot) { return c.refused && slot >= 0 && (unsigned)slot < c.sequences && c.refused[slot] != 0; }
// Offset of a token's first row (of head 0) in elements; -1 if its page does not exist.  The token is below sequence_length.
ATTN_FN long long token_offset(const Pages &c, int slot, unsigned token) {
    const unsigned i = token / c.page_size;
    const int page = c.table[(size_t)slot * c.max_pages + i];
    if (page < 0 || (unsigned)page >= c.pages) return -1;
    return (long long)((size_t)(unsigned)page * c.page_stride + (size_t)(token - i * c.page_size) * c.token_stride);
}

// `steps` pieces of work are dealt to `parts` workers in order: part p has those from first_step(p) = steps * p / parts to before first_step(p + 1).  (In 32 bits where they
// do: a 64-bit division takes a GPU some hundred instructions.)
ATTN_FN unsigned long long first_step(unsigned long long steps, unsigned p, unsigned parts) {
    if (steps >> 32 == 0 && parts < 65536u) {
        const unsigned n = (unsigned)steps, each = n / parts;
        return (unsigned long long)each * p + (n - each * parts) * p / parts;
    }
    return steps / parts * p + steps % parts * p / parts;
}
// The part that has step x: the least p with x < first_step(p + 1), i.e. with (x + 1) * parts <= steps * (p + 1).
ATTN_FN unsigned part_of_step(unsigned long long steps, unsigned long long x, unsigned parts) {
    const unsigned long long all = (x + 1) * parts - 1;
    return (all | steps) >> 32 ? (unsigned)(all / steps) : (unsigned)all / (unsigned)steps;
}

// ---- checks of arguments (attention.cpp) ----
// 0, or the return value after a message; `what` is the entry point.
int check_type(int type, unsigned head_dim, const char *what);
int check_cache(const aspen_b200_cache_t *c, const char *what, bool pool);
Pages pages_of(const aspen_b200_cache_t &c);
int check_rows(const void *p, size_t row, size_t head, int type, const char *name, const char *what);
// All of these are memory of the current device (NULL ones are not looked at).
struct Named { const void *p; const char *name; };
int check_device(const Named *list, unsigned n, const char *what);
// All of these start on a 4-byte boundary (NULL does).
int check_ints(const Named *list, unsigned n, const char *what);
int sm_count(const char *what);            // of the current device, which is an sm_100 one; or a negative return value
size_t packed(size_t stride, size_t dense);

}  // namespace attn
