// Argument checks of the attention operators and the paged cache.
#include "attention.h"

#include <cuda_runtime.h>

namespace attn {

size_t packed(size_t stride, size_t dense) { return stride ? stride : dense; }

int check_type(int type, unsigned head_dim, const char *what) {
    if (type < 0 || type >= ASPEN_B200_NUM_TYPES) { ASPEN_ERR("%s: unknown type %d\n", what, type); return -1; }
    if (head_dim < 8 || head_dim > MAX_HEAD || head_dim % 8) { ASPEN_ERR("%s: heads of %u features; 8, 16 ... %u are possible\n", what, head_dim, MAX_HEAD); return -1; }
    return 0;
}

int check_rows(const void *p, size_t row, size_t head, int type, const char *name, const char *what) {
    const size_t size = type_size(type);
    if (!p) { ASPEN_ERR("%s: %s is NULL\n", what, name); return -1; }
    if (reinterpret_cast<uintptr_t>(p) % 16 || row * size % 16 || head * size % 16) {
        ASPEN_ERR("%s: a row of %s does not start on a 16-byte boundary\n", what, name);
        return -1;
    }
    // offsets are 64-bit sums of up to four products with 32-bit counts
    if (row >= (size_t)1 << 29 || head >= (size_t)1 << 29) { ASPEN_ERR("%s: strides of %s must be below 2^29 elements\n", what, name); return -2; }
    return 0;
}

int check_ints(const Named *list, unsigned n, const char *what) {
    for (unsigned i = 0; i < n; i++)
        if (reinterpret_cast<uintptr_t>(list[i].p) % sizeof(int)) { ASPEN_ERR("%s: %s does not start on a 4-byte boundary\n", what, list[i].name); return -1; }
    return 0;
}

int check_cache(const aspen_b200_cache_t *c, const char *what, bool pool) {
    if (!c) { ASPEN_ERR("%s: no cache\n", what); return -1; }
    if (!c->page_table || !c->lengths || !c->status || (pool && !c->refs)) { ASPEN_ERR("%s: the cache has no page_table, lengths, status or refs\n", what); return -1; }
    const Named ints[] = {{c->page_table, "page_table"}, {c->lengths, "lengths"}, {c->refs, "refs"}, {c->status, "status"}, {c->refused, "refused"}};
    if (check_ints(ints, 5, what)) return -1;
    if (!c->layers || !c->pages || !c->page_size || !c->kv_heads || !c->sequences || !c->max_pages) { ASPEN_ERR("%s: a size of the cache is 0\n", what); return -1; }
    const int bad = check_type(c->type, c->head_dim, what);
    if (bad) return bad;
    if (c->layers > 1024) { ASPEN_ERR("%s: %u layers; 1024 are possible\n", what, c->layers); return -2; }
    if (c->pages > 0x7fffffffu || c->sequences > 0x7fffffffu || (unsigned long long)c->max_pages * c->page_size > 0x7fffffffull) {
        ASPEN_ERR("%s: pages, sequences and the tokens of a sequence must be below 2^31\n", what);
        return -2;
    }
    if ((unsigned long long)c->kv_heads * c->page_size * c->head_dim > 0x7fffffffull || c->kv_heads > 0xffffu) { ASPEN_ERR("%s: a page is too large\n", what); return -2; }
    for (const void *p : {(const void *)c->k, (const void *)c->v}) {
        const int r = check_rows(p, c->token_stride, c->head_stride, c->type, p == c->k ? "the cache's k" : "the cache's v", what);
        if (r) return r;
    }
    const size_t size = type_size(c->type);
    if (c->page_stride * size % 16 || c->layer_stride * size % 16) { ASPEN_ERR("%s: pages and layers of the cache must start on 16-byte boundaries\n", what); return -1; }
    if (c->page_stride >= (size_t)1 << 31 || c->layer_stride >= (size_t)1 << 40) { ASPEN_ERR("%s: strides of the cache are too large\n", what); return -2; }
    return 0;
}

Pages pages_of(const aspen_b200_cache_t &c) {
    Pages p;
    p.table = c.page_table; p.lengths = c.lengths; p.status = c.status;
    p.token_stride = packed(c.token_stride, c.head_dim);
    p.head_stride = packed(c.head_stride, p.token_stride * c.page_size);
    p.page_stride = packed(c.page_stride, p.head_stride * c.kv_heads);
    p.pages = c.pages; p.page_size = c.page_size; p.sequences = c.sequences; p.max_pages = c.max_pages;
    p.refused = c.refused;
    return p;
}

int check_device(const Named *list, unsigned n, const char *what) {
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    for (unsigned i = 0; i < n && err == cudaSuccess; i++) {
        if (!list[i].p) continue;
        cudaPointerAttributes a;
        err = cudaPointerGetAttributes(&a, list[i].p);
        if (err != cudaSuccess) break;
        if (a.type != cudaMemoryTypeDevice) { ASPEN_ERR("%s: %s is not device memory\n", what, list[i].name); return -1; }
        if (a.device != dev) {
            ASPEN_ERR("%s: %s is memory of device %d, the current one is %d\n", what, list[i].name, a.device, dev);
            return -1;
        }
    }
    if (err != cudaSuccess) { cudaGetLastError(); ASPEN_ERR("%s: %s\n", what, cudaGetErrorString(err)); return -3; }
    return 0;
}

int sm_count(const char *what) {
    int dev = 0, sms = 0, major = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err == cudaSuccess) err = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (err == cudaSuccess) err = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev);
    if (err != cudaSuccess || sms <= 0 || major != 10) {
        cudaGetLastError();
        ASPEN_ERR("%s: no sm_100 device (%s)\n", what, cudaGetErrorString(err));
        return -3;
    }
    return sms;
}

}  // namespace attn
