// paged_args.cuh — argument checks that the C entry points of the operators on a
// caller-owned paged cache share, and the descriptions of their rows.
#pragma once

#include "paged.cuh"

#include "kore_cuda.h"

#include <cstdarg>
#include <cstdio>
#include <cstring>

namespace kore {
namespace {

inline int refuse(int code, const char *fmt, ...) {
    char buf[256];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    set_ctxless_error(buf);
    return code;
}

inline int type_bytes(int type) {
    switch (type) {
        case KORE_CUDA_F32: return 4;
        case KORE_CUDA_F16:
        case KORE_CUDA_BF16: return 2;
        case KORE_CUDA_E4M3: return 1;
    }
    return 0;
}

// Makes the device of a buffer current for the call.
struct OnDeviceOf {
    int prev = -1, dev = -1, rc = KORE_CUDA_OK;
    explicit OnDeviceOf(const void *ptr) {
        cudaPointerAttributes a;
        cudaError_t e = cudaPointerGetAttributes(&a, ptr);
        if (e != cudaSuccess) {
            cudaGetLastError();
            rc = refuse(KORE_CUDA_ECUDA, "no CUDA device: %s", cudaGetErrorString(e));
            return;
        }
        if (a.type != cudaMemoryTypeDevice && a.type != cudaMemoryTypeManaged) {
            rc = refuse(KORE_CUDA_EINVAL, "expected device memory");
            return;
        }
        dev = a.device;
        if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
        if (prev != dev && (e = cudaSetDevice(dev)) != cudaSuccess)
            rc = refuse(KORE_CUDA_ECUDA, "cudaSetDevice(%d): %s", dev, cudaGetErrorString(e));
    }
    ~OnDeviceOf() {
        if (prev >= 0 && prev != dev) cudaSetDevice(prev);
    }
};

inline int launched(cudaError_t e, const char *what) {
    if (e == cudaSuccess) return KORE_CUDA_OK;
    cudaGetLastError();
    return refuse(KORE_CUDA_ECUDA, "%s: %s", what, cudaGetErrorString(e));
}

inline bool aligned16(const kore_cuda_rows &r) {
    const long long b = type_bytes(r.type);
    return ((reinterpret_cast<uintptr_t>(r.data) | (uintptr_t)(r.token_stride * b) | (uintptr_t)(r.head_stride * b)) & 15) == 0;
}

inline int check_rows(const kore_cuda_rows *r, const char *name, int head_dim) {
    if (!r || !r->data) return refuse(KORE_CUDA_EINVAL, "%s is null", name);
    const int b = type_bytes(r->type);
    if (b < 2) return refuse(KORE_CUDA_EINVAL, "%s: type %d is none of F32, F16, BF16", name, r->type);
    if (reinterpret_cast<uintptr_t>(r->data) % b) return refuse(KORE_CUDA_EINVAL, "%s is not aligned to its type", name);
    if (r->n_head <= 0 || r->n_head > 65535) return refuse(KORE_CUDA_EINVAL, "%s: n_head %d", name, r->n_head);
    if (r->head_dim != head_dim) return refuse(KORE_CUDA_EINVAL, "%s: head_dim %d, expected %d", name, r->head_dim, head_dim);
    return KORE_CUDA_OK;
}

// Arrays of 32-bit values: a kernel's load or store off their alignment would fault.
template <typename... P>
bool words_aligned(const P *...p) {
    return ((... | reinterpret_cast<uintptr_t>(p)) & 3) == 0;
}

// Rows that are written: several in one place would leave whichever came last.
inline int check_written(const kore_cuda_rows *r, const char *name, int n_tok) {
    if ((n_tok > 1 && r->token_stride == 0) || (r->n_head > 1 && r->head_stride == 0))
        return refuse(KORE_CUDA_EINVAL, "%s: the rows overlap (a stride of 0)", name);
    return KORE_CUDA_OK;
}

inline int check_rope(const kore_cuda_rope_view *r, int head_dim) {
    if (!r->table) return refuse(KORE_CUDA_EINVAL, "the rotation table is null");
    if (reinterpret_cast<uintptr_t>(r->table) & 15)
        return refuse(KORE_CUDA_EINVAL, "the rotation table must be 16-byte aligned");
    if (r->n_pos <= 0) return refuse(KORE_CUDA_EINVAL, "the rotation table holds %d positions", r->n_pos);
    if (r->n_rot < 2 || (r->n_rot & 1) || r->n_rot > head_dim)
        return refuse(KORE_CUDA_EINVAL, "n_rot %d must be even and at most head_dim %d", r->n_rot, head_dim);
    return KORE_CUDA_OK;
}

inline int check_pages(const kore_cuda_pages *c, bool attention) {
    if (!c || !c->k || !c->v) return refuse(KORE_CUDA_EINVAL, "the cache is null");
    const int b = type_bytes(c->type);
    if (b == 0 || (attention && b == 4)) return refuse(KORE_CUDA_EINVAL, "cache type %d is not supported here", c->type);
    if (c->n_pages <= 0) return refuse(KORE_CUDA_EINVAL, "n_pages %d must be positive", c->n_pages);
    if (c->page_tokens <= 0 || c->page_tokens % 16)
        return refuse(KORE_CUDA_EINVAL, "page_tokens %d must be a positive multiple of 16", c->page_tokens);
    if (c->n_head_kv <= 0 || c->n_head_kv > 65535) return refuse(KORE_CUDA_EINVAL, "n_head_kv %d", c->n_head_kv);
    if (c->head_dim <= 0 || c->head_dim % 16 || c->head_dim > 256 ||
        (attention && c->head_dim != 64 && c->head_dim != 128))
        return refuse(KORE_CUDA_EINVAL, "head_dim %d is not supported here", c->head_dim);
    if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15)
        return refuse(KORE_CUDA_EINVAL, "the page pools must be 16-byte aligned");
    const long long page = (long long)c->n_head_kv * c->page_tokens * c->head_dim;
    if (c->page_stride && (c->page_stride < page || c->page_stride * b % 16))
        return refuse(KORE_CUDA_EINVAL, "page_stride %lld must be a multiple of 16 bytes and at least a page (%lld)",
                      c->page_stride, page);
    if (c->type != KORE_CUDA_E4M3 && (c->k_scale || c->v_scale))
        return refuse(KORE_CUDA_EINVAL, "scales belong to an E4M3 cache");
    if (!words_aligned(c->k_scale, c->v_scale)) return refuse(KORE_CUDA_EINVAL, "the scales are not aligned to their type");
    return KORE_CUDA_OK;
}

inline long long page_stride(const kore_cuda_pages *c) {
    return c->page_stride ? c->page_stride : (long long)c->n_head_kv * c->page_tokens * c->head_dim;
}

// Whether some page of the keys and some page of the values (which may lie between one another's) share memory.
inline bool pages_overlap(const kore_cuda_pages *c) {
    const unsigned long long b = type_bytes(c->type), page = (unsigned long long)c->n_head_kv * c->page_tokens * c->head_dim * b;
    const unsigned long long stride = page_stride(c) * b, span = (c->n_pages - 1) * stride + page;
    const uintptr_t k = reinterpret_cast<uintptr_t>(c->k), v = reinterpret_cast<uintptr_t>(c->v);
    const unsigned long long apart = k < v ? v - k : k - v;
    if (apart >= span) return false;   // (most: a commit asks of every layer, and a division takes as long as the rest)
    const unsigned long long rest = apart % stride;
    return rest < page || (stride - rest < page && apart - rest + stride < span);
}

// Keys and values that go into memory that the cache's share: which of them stayed would be chance, unless it is one
// memory and they are the same. changed: the keys are normed or rotated on the way.
inline int check_stored_apart(const kore_cuda_pages *c, const kore_cuda_rows *k, const kore_cuda_rows *v, bool changed) {
    if (!pages_overlap(c)) return KORE_CUDA_OK;
    const bool alike = c->k == c->v && k->data == v->data && k->token_stride == v->token_stride &&
                       k->head_stride == v->head_stride && c->k_scale == c->v_scale && !changed;
    if (alike) return KORE_CUDA_OK;
    return refuse(KORE_CUDA_EINVAL, "the cache's keys and values share memory, and k and v are not the same rows");
}

// tables: the page table is used
inline int check_batch(const kore_cuda_batch *b, int n_tok, bool tables = true) {
    if (!b) return refuse(KORE_CUDA_EINVAL, "the batch is null");
    if (n_tok < 0) return refuse(KORE_CUDA_EINVAL, "n_tok %d", n_tok);
    if (b->n_seq < 0 || b->n_seq > kPagedMaxSeqs)
        return refuse(KORE_CUDA_ERANGE, "n_seq %d outside [0, %d]", b->n_seq, kPagedMaxSeqs);
    if (b->n_seq > 0 && (!b->q_start || !b->kv_len || (tables && !b->page_table)))
        return refuse(KORE_CUDA_EINVAL, "q_start, kv_len or page_table is null");
    if (!words_aligned(b->q_start, b->kv_len, b->page_table))
        return refuse(KORE_CUDA_EINVAL, "q_start, kv_len or page_table is not aligned to its type");
    if (tables && b->n_seq > 0 && b->table_stride <= 0) return refuse(KORE_CUDA_EINVAL, "table_stride %d", b->table_stride);
    if (b->max_q < 0) return refuse(KORE_CUDA_EINVAL, "max_q %d", b->max_q);
    if (b->max_kv < 0) return refuse(KORE_CUDA_EINVAL, "max_kv %d", b->max_kv);
    return KORE_CUDA_OK;
}

// Rows that go into a cache: k and v, and q beside them.
inline int check_appended(const kore_cuda_pages *cache, const kore_cuda_rows *k, const kore_cuda_rows *v,
                          const kore_cuda_rows *q, const kore_cuda_rows *q_out, int n_tok) {
    const int d = cache->head_dim;
    if (int rc = check_rows(k, "k", d)) return rc;
    if (int rc = check_rows(v, "v", d)) return rc;
    if (k->n_head != cache->n_head_kv || v->n_head != cache->n_head_kv)
        return refuse(KORE_CUDA_EINVAL, "k and v must have the cache's %d heads", cache->n_head_kv);
    if (v->type != k->type) return refuse(KORE_CUDA_EINVAL, "k and v have different types");
    if (!q != !q_out) return refuse(KORE_CUDA_EINVAL, "q and q_out come together");
    if (q) {
        if (int rc = check_rows(q, "q", d)) return rc;
        if (int rc = check_rows(q_out, "q_out", d)) return rc;
        if (q->type != k->type || q_out->type != k->type || q_out->n_head != q->n_head)
            return refuse(KORE_CUDA_EINVAL, "q and q_out must have k's type and the same heads");
        if (int rc = check_written(q_out, "q_out", n_tok)) return rc;
    }
    if (cache->type != k->type && cache->type != KORE_CUDA_E4M3 &&
        !(k->type == KORE_CUDA_F32 && (cache->type == KORE_CUDA_F16 || cache->type == KORE_CUDA_BF16)))
        return refuse(KORE_CUDA_EINVAL, "rows of type %d do not go into a cache of type %d", k->type, cache->type);
    return KORE_CUDA_OK;
}

inline int check_words(int words) {
    if (words <= 0 || words > kPagedMaxTree / 32)
        return refuse(KORE_CUDA_EINVAL, "the tree's words %d outside [1, %d]", words, kPagedMaxTree / 32);
    return KORE_CUDA_OK;
}

inline int check_tree(const kore_cuda_tree *t) {
    if (!t->mask) return refuse(KORE_CUDA_EINVAL, "the tree's mask is null");
    if (!words_aligned(t->mask)) return refuse(KORE_CUDA_EINVAL, "the tree's mask is not aligned to its type");
    return check_words(t->words);
}

inline bool rotates_in_vectors(int d, const kore_cuda_rope_view *r) { return d % 16 == 0 && (!r || r->n_rot % 16 == 0); }

inline HeadRows head_rows(const kore_cuda_rows *in, const kore_cuda_rows *out) {
    HeadRows h;
    memset(&h, 0, sizeof h);
    if (!in) return h;
    h.in = in->data;
    h.in_ts = in->token_stride;
    h.in_hs = in->head_stride;
    h.heads = in->n_head;
    if (out) {
        h.out = out->data;
        h.out_ts = out->token_stride;
        h.out_hs = out->head_stride;
    }
    return h;
}

}  // namespace
}  // namespace kore
