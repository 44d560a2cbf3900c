// paged_step_capi.cu — C entry points of a step with drafted tokens over the paged cache
// (include/kore_cuda.h): argument checks, the buffers' device. Nothing is allocated and
// nothing kept between calls.

#include "paged_args.cuh"

#include <cfloat>
#include <cmath>

namespace kore {
namespace {

int check_pool(const kore_cuda_page_pool *p, int n_seq, const int *request, const int *amount, const int *status) {
    if (!p || !p->free_pages || !p->n_free || !p->table || !p->length) return refuse(KORE_CUDA_EINVAL, "the pool is null");
    if (p->n_pages <= 0) return refuse(KORE_CUDA_EINVAL, "n_pages %d must be positive", p->n_pages);
    if (p->page_tokens <= 0 || p->page_tokens % 16)
        return refuse(KORE_CUDA_EINVAL, "page_tokens %d must be a positive multiple of 16", p->page_tokens);
    if (p->n_requests <= 0 || p->n_requests > kPagedMaxRequests)
        return refuse(KORE_CUDA_ERANGE, "n_requests %d outside [1, %d]", p->n_requests, kPagedMaxRequests);
    if (p->table_stride <= 0) return refuse(KORE_CUDA_EINVAL, "table_stride %d", p->table_stride);
    if (n_seq < 0 || n_seq > kPagedMaxSeqs) return refuse(KORE_CUDA_ERANGE, "n_seq %d outside [0, %d]", n_seq, kPagedMaxSeqs);
    if (n_seq > 0 && (!request || !amount)) return refuse(KORE_CUDA_EINVAL, "request, n_new or keep is null");
    if (!words_aligned(p->free_pages, p->n_free, p->table, p->length, request, amount, status))
        return refuse(KORE_CUDA_EINVAL, "an array of the pool, request, n_new, keep or dev_status is not aligned to its type");
    return KORE_CUDA_OK;
}

int check_tokens(int n_tok) {
    if (n_tok < 0) return refuse(KORE_CUDA_EINVAL, "n_tok %d", n_tok);
    if (n_tok > kPagedMaxTokens) return refuse(KORE_CUDA_ERANGE, "n_tok %d is more than %d", n_tok, kPagedMaxTokens);
    return KORE_CUDA_OK;
}

PlanParams plan_params(const kore_cuda_page_pool *pool, int n_seq, const int *request, const int *amount, int *status) {
    PlanParams p;
    memset(&p, 0, sizeof p);
    p.free_pages = pool->free_pages;
    p.n_free = pool->n_free;
    p.table = pool->table;
    p.length = pool->length;
    p.n_pages = pool->n_pages;
    p.n_requests = pool->n_requests;
    p.stride = pool->table_stride;
    p.P = pool->page_tokens;
    p.by_page = FastDiv::of((uint32_t)p.P);
    p.n_seq = n_seq;
    p.request = request;
    p.amount = amount;
    p.status = status;
    return p;
}

TreeParams tree_params(const kore_cuda_batch *batch, int n_tok, const int *parent, int *status) {
    TreeParams p;
    memset(&p, 0, sizeof p);
    p.q_start = batch->q_start;
    p.kv_len = batch->kv_len;
    p.parent = parent;
    p.n_seq = batch->n_seq;
    p.n_tok = n_tok;
    p.cap = 0x7fffffffll;
    p.status = status;
    return p;
}

}  // namespace
}  // namespace kore

using namespace kore;

extern "C" int kore_cuda_paged_plan_dev(const kore_cuda_page_pool *pool, int n_seq, const int *request, const int *n_new,
                                        const kore_cuda_step *step, int *dev_status, void *stream) {
    if (int rc = check_pool(pool, n_seq, request, n_new, dev_status)) return rc;
    if (!step || !step->q_start) return refuse(KORE_CUDA_EINVAL, "the step is null");
    if (int rc = check_tokens(step->n_tok)) return rc;
    if (n_seq > 0 && (!step->kv_len || !step->page_table)) return refuse(KORE_CUDA_EINVAL, "kv_len or page_table is null");
    if (step->n_tok > 0 && (!step->slots || !step->pos)) return refuse(KORE_CUDA_EINVAL, "slots or pos is null");
    if ((reinterpret_cast<uintptr_t>(step->slots) & 7) || !words_aligned(step->q_start, step->kv_len, step->page_table, step->pos))
        return refuse(KORE_CUDA_EINVAL, "an array of the step is not aligned to its type");
    if (step->table_stride < pool->table_stride)
        return refuse(KORE_CUDA_EINVAL, "the step's table_stride %d is less than the pool's %d", step->table_stride, pool->table_stride);
    OnDeviceOf on(pool->table);
    if (on.rc) return on.rc;
    PlanParams p = plan_params(pool, n_seq, request, n_new, dev_status);
    p.n_tok = step->n_tok;
    p.out_stride = step->table_stride;
    p.q_start = step->q_start;
    p.kv_len = step->kv_len;
    p.page_table = step->page_table;
    p.pos = step->pos;
    p.slots = step->slots;
    return launched(launch_plan(p, false, (cudaStream_t)stream), "paged_plan");
}

extern "C" int kore_cuda_paged_trim_dev(const kore_cuda_page_pool *pool, int n_seq, const int *request, const int *keep,
                                        int *dev_status, void *stream) {
    if (int rc = check_pool(pool, n_seq, request, keep, dev_status)) return rc;
    if (n_seq == 0) return KORE_CUDA_OK;
    OnDeviceOf on(pool->table);
    if (on.rc) return on.rc;
    return launched(launch_plan(plan_params(pool, n_seq, request, keep, dev_status), true, (cudaStream_t)stream), "paged_trim");
}

extern "C" int kore_cuda_paged_store_dev(const kore_cuda_pages *cache, int n_tok, const long long *slots, const int *pos,
                                         const kore_cuda_rows *k, const kore_cuda_rows *v, const kore_cuda_rows *q,
                                         const kore_cuda_rows *q_out, const kore_cuda_rope_view *rope,
                                         const kore_cuda_head_norm *norm, int *dev_status, void *stream) {
    if (int rc = check_pages(cache, false)) return rc;
    if (int rc = check_tokens(n_tok)) return rc;
    if (n_tok > 0 && !slots) return refuse(KORE_CUDA_EINVAL, "slots is null");
    if ((reinterpret_cast<uintptr_t>(slots) & 7) || !words_aligned(pos, dev_status))
        return refuse(KORE_CUDA_EINVAL, "slots, pos or dev_status is not aligned to its type");
    const int d = cache->head_dim;
    if (int rc = check_appended(cache, k, v, q, q_out, n_tok)) return rc;
    if (rope) {
        if (int rc = check_rope(rope, d)) return rc;
        if (n_tok > 0 && !pos) return refuse(KORE_CUDA_EINVAL, "a rotation needs positions");
    }
    bool weights16 = true;
    if (norm) {
        const int b = type_bytes(norm->type);
        if (b < 2) return refuse(KORE_CUDA_EINVAL, "norm: type %d is none of F32, F16, BF16", norm->type);
        if (!norm->q_weight && !norm->k_weight) return refuse(KORE_CUDA_EINVAL, "norm: no weights");
        if ((reinterpret_cast<uintptr_t>(norm->q_weight) | reinterpret_cast<uintptr_t>(norm->k_weight)) % b)
            return refuse(KORE_CUDA_EINVAL, "norm: the weights are not aligned to their type");
        if (!(norm->eps >= FLT_MIN) || !std::isfinite(norm->eps))
            return refuse(KORE_CUDA_EINVAL, "norm: eps must be a positive normal number");
        weights16 = ((reinterpret_cast<uintptr_t>(norm->q_weight) | reinterpret_cast<uintptr_t>(norm->k_weight) |
                      (uintptr_t)(norm->q_head_stride * b) | (uintptr_t)(norm->k_head_stride * b)) & 15) == 0;
    }
    if (n_tok == 0) return KORE_CUDA_OK;
    if (int rc = check_stored_apart(cache, k, v, rope || (norm && norm->k_weight))) return rc;
    OnDeviceOf on(cache->k);
    if (on.rc) return on.rc;
    StoreParams p;
    memset(&p, 0, sizeof p);
    p.q = head_rows(q, q_out);
    p.k = head_rows(k, nullptr);
    p.v = head_rows(v, nullptr);
    p.slots = slots;
    p.pos = pos;
    if (rope) {
        p.table = rope->table;
        p.n_pos = rope->n_pos;
        p.rot = rope->n_rot;
        p.interleaved = rope->interleaved != 0;
    }
    p.n_tok = n_tok;
    p.d = d;
    p.P = cache->page_tokens;
    p.G = cache->n_head_kv;
    p.by_page = FastDiv::of((uint32_t)p.P);
    p.n_slots = (long long)cache->n_pages * cache->page_tokens;
    p.page_stride = page_stride(cache);
    p.kc = cache->k;
    p.vc = cache->v;
    p.k_scale = cache->k_scale;
    p.v_scale = cache->v_scale;
    if (norm) {
        p.q_weight = norm->q_weight;
        p.k_weight = norm->k_weight;
        p.weight_type = norm->type;
        p.q_weight_hs = norm->q_head_stride;
        p.k_weight_hs = norm->k_head_stride;
        p.eps = norm->eps;
        p.most = norm->eps < 0x1p100f ? 3.0e38f : 0.f;   // (mean and eps together stay in 32 bits)
    }
    p.status = dev_status;
    const bool vec = (d == 64 || d == 128 || d == 256) && rotates_in_vectors(d, rope) && weights16 &&
                     (!norm || norm->type == KORE_CUDA_F32 || norm->type == k->type) &&
                     aligned16(*k) && aligned16(*v) && (!q || (aligned16(*q) && aligned16(*q_out)));
    int sms = 0;
    if (cudaError_t e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, on.dev))
        return launched(e, "cudaDeviceGetAttribute");
    return launched(launch_store(p, k->type, cache->type, vec, sms, (cudaStream_t)stream), "paged_store");
}

extern "C" int kore_cuda_tree_masks_dev(const kore_cuda_batch *batch, int n_tok, const int *parent, unsigned *mask, int words,
                                        int *pos, int *dev_status, void *stream) {
    if (int rc = check_batch(batch, n_tok, false)) return rc;
    const kore_cuda_tree tree{mask, words};
    if (int rc = check_tree(&tree)) return rc;
    if (!parent || !pos) return refuse(KORE_CUDA_EINVAL, "parent or pos is null");
    if (!words_aligned(parent, pos, dev_status)) return refuse(KORE_CUDA_EINVAL, "parent, pos or dev_status is not aligned to its type");
    if (n_tok == 0 || batch->n_seq == 0) return KORE_CUDA_OK;
    OnDeviceOf on(mask);
    if (on.rc) return on.rc;
    TreeParams p = tree_params(batch, n_tok, parent, dev_status);
    p.most = words * 32;
    p.words = words;
    p.mask = reinterpret_cast<uint32_t *>(mask);
    p.pos = pos;
    return launched(launch_tree_mask(p, (cudaStream_t)stream), "tree_masks");
}

// most: tokens of a chunk at most
static int accept(const kore_cuda_batch *batch, int n_tok, int most, const int *parent, const int *token, const int *choice,
                  const kore_cuda_accepted *out, int *dev_status, void *stream) {
    if (int rc = check_batch(batch, n_tok, false)) return rc;
    if (!parent || !token || !choice) return refuse(KORE_CUDA_EINVAL, "parent, token or choice is null");
    if (!out || !out->path || !out->count || !out->next_token || !out->kept)
        return refuse(KORE_CUDA_EINVAL, "path, count, next_token or kept is null");
    if (!words_aligned(parent, token, choice, out->path, out->count, out->next_token, out->kept, dev_status))
        return refuse(KORE_CUDA_EINVAL, "parent, token, choice, an array of the acceptance or dev_status is not aligned to its type");
    if (out->path_stride <= 0 || out->path_stride > kPagedMaxTree)
        return refuse(KORE_CUDA_EINVAL, "path_stride %d outside [1, %d]", out->path_stride, kPagedMaxTree);
    if (batch->n_seq == 0) return KORE_CUDA_OK;
    OnDeviceOf on(out->path);
    if (on.rc) return on.rc;
    TreeParams p = tree_params(batch, n_tok, parent, dev_status);
    p.token = token;
    p.choice = choice;
    p.most = most;
    p.path = out->path;
    p.path_stride = out->path_stride;
    p.count = out->count;
    p.next = out->next_token;
    p.kept = out->kept;
    return launched(launch_accept(p, (cudaStream_t)stream), "tree_accept");
}

extern "C" int kore_cuda_tree_accept_dev(const kore_cuda_batch *batch, int n_tok, const int *parent, const int *token,
                                         const int *choice, const kore_cuda_accepted *out, int *dev_status, void *stream) {
    return accept(batch, n_tok, kPagedMaxTree, parent, token, choice, out, dev_status, stream);
}

extern "C" int kore_cuda_tree_accept_masked_dev(const kore_cuda_batch *batch, int n_tok, int words, const int *parent,
                                                const int *token, const int *choice, const kore_cuda_accepted *out,
                                                int *dev_status, void *stream) {
    if (int rc = check_words(words)) return rc;
    return accept(batch, n_tok, words * 32, parent, token, choice, out, dev_status, stream);
}

extern "C" int kore_cuda_paged_commit_dev(const kore_cuda_pages *layers, int n_layers, const kore_cuda_batch *batch,
                                          const int *path, int path_stride, const int *count, int *dev_status, void *stream) {
    if (n_layers < 0) return refuse(KORE_CUDA_EINVAL, "n_layers %d", n_layers);
    if (n_layers > 0 && !layers) return refuse(KORE_CUDA_EINVAL, "layers is null");
    // A layer named twice would be moved by two threads at once. Bits of the addresses so far tell most layers
    // apart; only where one's are there already are the earlier ones looked through.
    unsigned long long named[16] = {};
    auto fresh = [&](const void *x) {
        const uint64_t bit = (reinterpret_cast<uintptr_t>(x) >> 4) * 0x9e3779b97f4a7c15ull >> 54;
        const bool was = named[bit >> 6] >> (bit & 63) & 1;
        named[bit >> 6] |= 1ull << (bit & 63);
        return !was;
    };
    for (int l = 0; l < n_layers; ++l) {
        const kore_cuda_pages &c = layers[l];
        if (int rc = check_pages(&c, false)) return rc;
        if (c.type != layers->type || c.n_pages != layers->n_pages || c.page_tokens != layers->page_tokens ||
            c.n_head_kv != layers->n_head_kv || c.head_dim != layers->head_dim || page_stride(&c) != page_stride(layers))
            return refuse(KORE_CUDA_EINVAL, "layer %d has another type or geometry than layer 0", l);
        const bool k_fresh = fresh(c.k), v_fresh = fresh(c.v);
        for (int x = 0; (!k_fresh || !v_fresh) && x < l; ++x)
            if (layers[x].k == c.k || layers[x].v == c.k || layers[x].k == c.v || layers[x].v == c.v)
                return refuse(KORE_CUDA_EINVAL, "layers %d and %d have the same pages", x, l);
    }
    if (int rc = check_batch(batch, 0, true)) return rc;
    if (batch->n_seq > 0 && (!path || !count)) return refuse(KORE_CUDA_EINVAL, "path or count is null");
    if (!words_aligned(path, count, dev_status)) return refuse(KORE_CUDA_EINVAL, "path, count or dev_status is not aligned to its type");
    if (path_stride <= 0 || path_stride > kPagedMaxTree)
        return refuse(KORE_CUDA_EINVAL, "path_stride %d outside [1, %d]", path_stride, kPagedMaxTree);
    if (n_layers == 0 || batch->n_seq == 0) return KORE_CUDA_OK;
    for (int l = 0; l < n_layers; ++l)
        if (layers[l].k != layers[l].v && pages_overlap(&layers[l]))
            return refuse(KORE_CUDA_EINVAL, "layer %d: the keys' pages overlap the values'", l);
    OnDeviceOf on(layers->k);
    if (on.rc) return on.rc;
    CommitParams p;
    memset(&p, 0, sizeof p);
    p.q_start = batch->q_start;
    p.kv_len = batch->kv_len;
    p.page_table = batch->page_table;
    p.path = path;
    p.count = count;
    p.n_seq = batch->n_seq;
    p.table_stride = batch->table_stride;
    p.path_stride = path_stride;
    p.n_pages = layers->n_pages;
    p.P = layers->page_tokens;
    p.G = layers->n_head_kv;
    p.row_pieces = layers->head_dim * type_bytes(layers->type) / 16;
    p.by_page = FastDiv::of((uint32_t)p.P);
    p.page_pieces = page_stride(layers) * type_bytes(layers->type) / 16;
    p.status = dev_status;
    for (int l0 = 0; l0 < n_layers; l0 += kPagedMaxLayers) {
        p.n_layers = n_layers - l0 < kPagedMaxLayers ? n_layers - l0 : kPagedMaxLayers;
        for (int l = 0; l < p.n_layers; ++l) {
            p.k[l] = layers[l0 + l].k;
            p.v[l] = layers[l0 + l].v != p.k[l] ? layers[l0 + l].v : nullptr;   // (one memory's rows move once)
        }
        if (int rc = launched(launch_commit(p, (cudaStream_t)stream), "paged_commit")) return rc;
    }
    return KORE_CUDA_OK;
}
