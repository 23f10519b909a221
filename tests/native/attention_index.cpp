// Index arithmetic of the paged cache and the cut of the work over single tokens (aspen_b200/csrc/attention.h), over their whole range and with tables that
// name pages that do not exist.
#include "../../aspen_b200/csrc/attention.h"

#include <cstdio>

static int fail(const char *what, unsigned long long a, unsigned long long b) { printf("%s: %llu %llu\n", what, a, b); return 1; }

int main() {
    // every step belongs to one part, in order, and part_of_step finds it
    for (unsigned long long steps : {1ull, 2ull, 7ull, 148ull, 295ull, 296ull, 297ull, 5000ull, 123457ull})
        for (unsigned parts : {1u, 2u, 8u, 148u, 296u}) {
            if (attn::first_step(steps, 0, parts) != 0 || attn::first_step(steps, parts, parts) != steps) return fail("ends", steps, parts);
            for (unsigned p = 0; p < parts; p++) {
                const unsigned long long a = attn::first_step(steps, p, parts), b = attn::first_step(steps, p + 1, parts);
                if (b < a || b - a > steps / parts + 1) return fail("share", steps, p);
                for (unsigned long long x = a; x < b; x++) if (attn::part_of_step(steps, x, parts) != p) return fail("part", steps, x);
            }
        }
    const unsigned long long big = 1ull << 45;          // 2^31 tokens in steps of 16, of 2^18 items
    for (unsigned p = 0; p < 296; p++) {
        const unsigned long long a = attn::first_step(big, p, 296), b = attn::first_step(big, p + 1, 296);
        if (attn::part_of_step(big, a, 296) != p || attn::part_of_step(big, b - 1, 296) != p) return fail("big", p, a);
    }
    // three sequences, four pages each of seven tokens; a pool of nine pages whose offsets pass 32 bits
    int table[12] = {3, 8, -1, 9, 0, 0, 2147483647, -2147483647, 8, 5, 1, 2}, lengths[3] = {28, -4, 1000}, status = 0;
    attn::Pages c{table, lengths, &status, 3000000000ull, 8, 16, 9, 7, 3, 4};
    if (attn::sequence_length(c, 0) != 28 || attn::sequence_length(c, 1) != 0 || attn::sequence_length(c, 2) != 28) return fail("length", 0, 0);
    if (attn::sequence_length(c, -1) != 0 || attn::sequence_length(c, 3) != 0) return fail("no sequence", 0, 0);
    for (int s = 0; s < 3; s++)
        for (unsigned t = 0; t < 28; t++) {
            const int page = table[s * 4 + t / 7];
            const long long want = page < 0 || page >= 9 ? -1 : page * 3000000000ll + t % 7 * 16;
            if (attn::token_offset(c, s, t) != want) return fail("offset", s, t);
        }
    return 0;
}
