// paged_capi.cu — C entry points of the operators on a caller-owned paged
// cache (include/kore_cuda.h): argument checks, the buffers' device, kernel
// choice. Nothing is allocated and nothing kept between calls.

#include "paged_args.cuh"

#include <cuda.h>

#include <atomic>
#include <cmath>

namespace kore {
namespace {

std::atomic<unsigned long long> g_wait_ns{kWaitNs};   // of launches from now on
std::atomic<int> g_tree_kernel{KORE_CUDA_TREE_BY_SIZE};

// The pool as a tensor [page][head][token][d], boxes of `box` tokens x 128 bytes
// (or the 64 of a short row), swizzled within rows of that width or (plain) as it is.
bool encode_pages(const void *base, const kore_cuda_pages *c, int box, bool plain, TmaDesc *out) {
    using encode_fn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                   const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const encode_fn fn = []() -> encode_fn {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &r) != cudaSuccess ||
            r != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            return nullptr;
        }
        return reinterpret_cast<encode_fn>(f);
    }();
    if (!fn) return false;
    const cuuint64_t d = c->head_dim, P = c->page_tokens, G = c->n_head_kv;
    const cuuint64_t dims[4] = {d, P, G, (cuuint64_t)c->n_pages};
    const cuuint64_t b = type_bytes(c->type), width = d * b < 128 ? d * b : 128;
    const cuuint64_t strides[3] = {d * b, P * d * b, (cuuint64_t)page_stride(c) * b};
    const cuuint32_t boxes[4] = {(cuuint32_t)(width / b), (cuuint32_t)box, 1, 1}, steps[4] = {1, 1, 1, 1};
    CUtensorMap m;
    static_assert(sizeof m == sizeof *out, "tensor map size");
    if (fn(&m, b == 2 ? CU_TENSOR_MAP_DATA_TYPE_UINT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void *>(base), dims, strides, boxes, steps,
           CU_TENSOR_MAP_INTERLEAVE_NONE, plain ? CU_TENSOR_MAP_SWIZZLE_NONE : width == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return false;
    memcpy(out, &m, sizeof m);
    return true;
}

// Whether a batch of trees goes to the 128-row kernel on the tensor cores, or to the one of 16 rows. What each
// would take, in us, from what they were measured to take on a B200: the row kernel its start, and for each
// unit of 16 rows an SM works on a time of its own and one for every 128 keys; the tile kernel its start, a
// time for every 64 keys (and 8 more of them a unit) of a CTA's share, and a joint for each doubling of the CTAs that
// share a unit. Row against tile kernel, 28/4 heads of 128, 16 bits: 8 tokens on 520 positions 11 / 16; 16
// on 16016 41 / 43; 16 x 8 on 1008 33 / 24; 16 x 24 on 324 42 / 15; 16 x 8 on 8008 161 / 67; 48 x 2 on 1002 30 /
// 36; 64 x 32 on 1532 408 / 89. 8 bits: 16 x 4 on 4004 40 / 47; 64 x 24 on 124 131 / 28. 14/2 heads of 64:
// 64 on 1064 11 / 17; 64 on 30064 58 / 39. Over 144 batches of groups of 7 and 8 query heads the choice takes 0.7 % more than
// the better kernel of each, 35 % at worst (28/4 of 128, 8 bits, 16 x 8 on 1008: 35 for 26). Groups of other sizes were not
// fitted: over 100 batches of 1, 4 and 16 heads 2.5 %, at worst 71 % (8/8 of 128, 8 bits, 16 x 24 on 324: 28 for 16).
bool trees_in_tiles(int d, bool e8, int G, int rep, int n_seq, int n_tok, double kv, int sms) {
    struct Cost {
        double unit, pass, start, tile, joint;
    };
    const Cost c = d == 128 ? e8 ? Cost{5.0, 0.72, 11.0, 1.6, 5.0} : Cost{3.5, 1.05, 9.5, 1.3, 5.0}
                            : e8 ? Cost{3.6, 0.55, 8.5, 1.14, 4.5} : Cost{3.0, 0.5, 7.5, 1.0, 4.5};
    const double packed = (double)n_tok * rep, half = 0.5 * n_seq;
    const double units16 = G * std::fmax(n_seq, packed / 16 + half), units = G * std::fmax(n_seq, packed / 128 + half);
    const double rows = 7 + std::fmax(4, units16 / sms * (c.unit + kv / 128 * c.pass));
    const double tiles = kv / 64, total = units * (tiles + kTreeUnitCost), ctas = 2.0 * sms;
    // (as find_share divides them: short units are not cut)
    const double used = tiles <= 8 || units >= ctas ? std::fmin(units, ctas) : std::fmin(ctas, std::fmax(units, total / 6));
    const double share = used <= units && units <= ctas ? tiles : total / used;
    return c.start + share * c.tile + c.joint * std::log2(std::fmax(1, used / units)) < rows;
}

}  // namespace
}  // namespace kore

using namespace kore;

extern "C" int kore_cuda_rope_freqs(const kore_cuda_rope_spec *spec, float *freq, double *amplitude) {
    if (!spec || !freq || !amplitude) return refuse(KORE_CUDA_EINVAL, "null argument");
    const int r = spec->n_rot;
    if (r < 2 || (r & 1) || r > 256) return refuse(KORE_CUDA_EINVAL, "n_rot %d must be even, 2 to 256", r);
    if (!(spec->base > 0) || !std::isfinite(spec->base)) return refuse(KORE_CUDA_EINVAL, "base must be positive");
    if (spec->scaling < KORE_CUDA_ROPE_NONE || spec->scaling > KORE_CUDA_ROPE_YARN)
        return refuse(KORE_CUDA_EINVAL, "scaling %d", spec->scaling);
    const bool scaled = spec->scaling != KORE_CUDA_ROPE_NONE, yarn = spec->scaling == KORE_CUDA_ROPE_YARN;
    if (scaled && (!(spec->factor > 0) || !std::isfinite(spec->factor)))
        return refuse(KORE_CUDA_EINVAL, "factor must be positive");
    if (!(spec->amplitude >= 0) || !std::isfinite(spec->amplitude))
        return refuse(KORE_CUDA_EINVAL, "amplitude must not be negative");
    double low = 0, high = 0;
    if (yarn) {
        const double fast = spec->beta_fast == 0 ? 32.0 : spec->beta_fast;
        const double slow = spec->beta_slow == 0 ? 1.0 : spec->beta_slow;
        if (!(spec->original_ctx > 0) || !std::isfinite(spec->original_ctx) || !(slow > 0) || !(fast >= slow) ||
            !std::isfinite(fast) || spec->base == 1.0)
            return refuse(KORE_CUDA_EINVAL, "YARN wants original_ctx > 0, beta_fast >= beta_slow > 0 and base != 1");
        // the pair that turns `turns` times over the original context
        auto dim = [&](double turns) {
            return r * std::log(spec->original_ctx / (2 * M_PI * turns)) / (2 * std::log(spec->base));
        };
        low = std::fmax(std::floor(dim(fast)), 0.0);
        high = std::fmin(std::ceil(dim(slow)), r - 1.0);
    }
    for (int i = 0; i < r / 2; ++i) {
        double f = std::pow(spec->base, -2.0 * i / r);
        if (spec->scaling == KORE_CUDA_ROPE_LINEAR) f /= spec->factor;
        if (yarn) {
            const double ramp = std::fmin(std::fmax((i - low) / std::fmax(high - low, 0.001), 0.0), 1.0);
            f = f / spec->factor * ramp + f * (1 - ramp);
        }
        freq[i] = (float)f;
    }
    *amplitude = spec->amplitude != 0 ? spec->amplitude : yarn && spec->factor > 1 ? 0.1 * std::log(spec->factor) + 1.0 : 1.0;
    return KORE_CUDA_OK;
}

extern "C" int kore_cuda_rope_table_dev(const kore_cuda_rope_spec *spec, int n_pos, float *table, void *stream) {
    float freq[128];
    double amp;
    if (int rc = kore_cuda_rope_freqs(spec, freq, &amp)) return rc;
    if (!table || (reinterpret_cast<uintptr_t>(table) & 15))
        return refuse(KORE_CUDA_EINVAL, "table must be 16-byte aligned device memory");
    if (n_pos <= 0) return refuse(KORE_CUDA_EINVAL, "n_pos %d must be positive", n_pos);
    OnDeviceOf on(table);
    if (on.rc) return on.rc;
    return launched(launch_rope_table(freq, spec->n_rot / 2, amp, n_pos, table, (cudaStream_t)stream), "rope_table");
}

extern "C" int kore_cuda_rope_dev(const kore_cuda_rows *x, const kore_cuda_rows *out, int n_tok, const int *pos,
                                  const kore_cuda_rope_view *rope, int *dev_status, void *stream) {
    if (!x || !rope || !pos) return refuse(KORE_CUDA_EINVAL, "null argument");
    if (!words_aligned(pos, dev_status)) return refuse(KORE_CUDA_EINVAL, "pos or dev_status is not aligned to its type");
    const int d = x->head_dim;
    if (d < 2 || (d & 1) || d > 256) return refuse(KORE_CUDA_EINVAL, "head_dim %d must be even, 2 to 256", d);
    if (int rc = check_rows(x, "x", d)) return rc;
    if (int rc = check_rows(out, "out", d)) return rc;
    if (int rc = check_rope(rope, d)) return rc;
    if (out->type != x->type || out->n_head != x->n_head)
        return refuse(KORE_CUDA_EINVAL, "out has another type or number of heads than x");
    if (n_tok < 0) return refuse(KORE_CUDA_EINVAL, "n_tok %d", n_tok);
    if (int rc = check_written(out, "out", n_tok)) return rc;
    if (n_tok == 0) return KORE_CUDA_OK;
    OnDeviceOf on(x->data);
    if (on.rc) return on.rc;
    RotateParams p;
    memset(&p, 0, sizeof p);
    p.q = head_rows(x, out);
    p.table = rope->table;
    p.n_pos = rope->n_pos;
    p.rot = rope->n_rot;
    p.interleaved = rope->interleaved != 0;
    p.pos = pos;
    p.n_tok = n_tok;
    p.d = d;
    p.status = dev_status;
    const bool vec = rotates_in_vectors(d, rope) && aligned16(*x) && aligned16(*out);
    return launched(launch_rotate(p, x->type, -1, vec, (cudaStream_t)stream), "rope");
}

extern "C" int kore_cuda_paged_append_dev(const kore_cuda_pages *cache, const kore_cuda_batch *batch, int n_tok,
                                          const kore_cuda_rows *k, const kore_cuda_rows *v, const kore_cuda_rows *q,
                                          const kore_cuda_rows *q_out, const kore_cuda_rope_view *rope,
                                          int *dev_status, void *stream) {
    if (int rc = check_pages(cache, false)) return rc;
    if (int rc = check_batch(batch, n_tok)) return rc;
    const int d = cache->head_dim;
    if (int rc = check_appended(cache, k, v, q, q_out, n_tok)) return rc;
    if (!words_aligned(dev_status)) return refuse(KORE_CUDA_EINVAL, "dev_status is not aligned to its type");
    if (rope)
        if (int rc = check_rope(rope, d)) return rc;
    if (n_tok == 0 || batch->n_seq == 0) return KORE_CUDA_OK;
    if (int rc = check_stored_apart(cache, k, v, rope != nullptr)) return rc;
    OnDeviceOf on(cache->k);
    if (on.rc) return on.rc;
    RotateParams p;
    memset(&p, 0, sizeof p);
    p.q = head_rows(q, q_out);
    p.k = head_rows(k, nullptr);
    p.v = head_rows(v, nullptr);
    if (rope) {
        p.table = rope->table;
        p.n_pos = rope->n_pos;
        p.rot = rope->n_rot;
        p.interleaved = rope->interleaved != 0;
    }
    p.n_tok = n_tok;
    p.d = d;
    p.n_seq = batch->n_seq;
    p.table_stride = batch->table_stride;
    p.n_pages = cache->n_pages;
    p.P = cache->page_tokens;
    p.G = cache->n_head_kv;
    p.page_stride = page_stride(cache);
    p.q_start = batch->q_start;
    p.kv_len = batch->kv_len;
    p.page_table = batch->page_table;
    p.kc = cache->k;
    p.vc = cache->v;
    p.k_scale = cache->k_scale;
    p.v_scale = cache->v_scale;
    p.status = dev_status;
    const bool vec = rotates_in_vectors(d, rope) && aligned16(*k) && aligned16(*v) &&
                     (!q || (aligned16(*q) && aligned16(*q_out)));
    return launched(launch_rotate(p, k->type, cache->type, vec, (cudaStream_t)stream), "paged_append");
}

extern "C" int kore_cuda_paged_set_wait_limit(unsigned long long nanoseconds) {
    g_wait_ns = nanoseconds ? nanoseconds : kWaitNs;
    return KORE_CUDA_OK;
}

extern "C" int kore_cuda_paged_set_tree_kernel(int kernel) {
    if (kernel < KORE_CUDA_TREE_BY_SIZE || kernel > KORE_CUDA_TREE_TILES) return refuse(KORE_CUDA_EINVAL, "tree kernel %d", kernel);
    g_tree_kernel = kernel;
    return KORE_CUDA_OK;
}

extern "C" long long kore_cuda_paged_attn_workspace(int head_dim) {
    if (head_dim != 64 && head_dim != 128) return refuse(KORE_CUDA_EINVAL, "head_dim %d is not supported here", head_dim);
    return (long long)kPagedZeroed + (long long)kPagedMaxCtas * 2 * kPagedRowsMax * (head_dim + 2) * (long long)sizeof(float);
}

// The attention of chunks (tree null) and of trees.
static int attend(const kore_cuda_pages *cache, const kore_cuda_batch *batch, int n_tok, const kore_cuda_rows *q,
                  const kore_cuda_rows *out, float *lse, const kore_cuda_attn_opts *opts, const kore_cuda_tree *tree,
                  void *workspace, long long workspace_bytes, int *dev_status, void *stream) {
    static_assert(kPagedZeroed == KORE_CUDA_PAGED_WORKSPACE_ZEROED && kPagedMaxCtas * sizeof(int) <= kPagedZeroed,
                  "the counters' place in the workspace");
    if (int rc = check_pages(cache, true)) return rc;
    if (int rc = check_batch(batch, n_tok)) return rc;
    const int d = cache->head_dim;
    if (int rc = check_rows(q, "q", d)) return rc;
    if (int rc = check_rows(out, "out", d)) return rc;
    if (q->type == KORE_CUDA_F32 || out->type != q->type || out->n_head != q->n_head)
        return refuse(KORE_CUDA_EINVAL, "q and out must be F16 or BF16, of one type and number of heads");
    if (int rc = check_written(out, "out", n_tok)) return rc;
    if (out->data == q->data) return refuse(KORE_CUDA_EINVAL, "out must not be q's own rows");
    if (cache->type != q->type && cache->type != KORE_CUDA_E4M3)
        return refuse(KORE_CUDA_EINVAL, "a cache of type %d does not go with queries of type %d", cache->type, q->type);
    const int G = cache->n_head_kv;
    if (q->n_head % G || q->n_head / G > 128)
        return refuse(KORE_CUDA_EINVAL, "unsupported geometry: n_head %d, n_head_kv %d", q->n_head, G);
    if ((long long)n_tok * (q->n_head / G) > 0x7fffffffll - kPagedRowsMax)
        return refuse(KORE_CUDA_ERANGE, "%d tokens are too many for one call", n_tok);
    if (!opts) return refuse(KORE_CUDA_EINVAL, "opts is null");
    if (!words_aligned(lse, dev_status)) return refuse(KORE_CUDA_EINVAL, "lse or dev_status is not aligned to its type");
    if (opts->window < 0) return refuse(KORE_CUDA_EINVAL, "window %d", opts->window);
    if (!std::isfinite(opts->scale)) return refuse(KORE_CUDA_EINVAL, "scale is not finite");
    if (tree) {
        if (int rc = check_tree(tree)) return rc;
        if (!opts->causal || opts->window)
            return refuse(KORE_CUDA_EINVAL, "a tree's tokens see what their masks say: no window, and causal as it is");
    }
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255) ||
        workspace_bytes < kore_cuda_paged_attn_workspace(d))
        return refuse(KORE_CUDA_EINVAL, "the workspace must be 256-byte aligned and hold %lld bytes",
                      kore_cuda_paged_attn_workspace(d));
    if (n_tok == 0 || batch->n_seq == 0) return KORE_CUDA_OK;
    OnDeviceOf on(cache->k);
    if (on.rc) return on.rc;
    int sms = 0;
    if (cudaError_t e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, on.dev))
        return launched(e, "cudaDeviceGetAttribute");
    PagedAttnParams p;
    memset(&p, 0, sizeof p);
    p.k = cache->k;
    p.v = cache->v;
    p.page_stride = page_stride(cache);
    p.q_start = batch->q_start;
    p.kv_len = batch->kv_len;
    p.page_table = batch->page_table;
    p.table_stride = batch->table_stride;
    p.n_seq = batch->n_seq;
    p.n_tok = n_tok;
    p.n_pages = cache->n_pages;
    p.P = cache->page_tokens;
    p.H = q->n_head;
    p.G = G;
    p.rep = q->n_head / G;
    p.by_rep = FastDiv::of((uint32_t)p.rep);
    p.by_page = FastDiv::of((uint32_t)p.P);
    p.q = q->data;
    p.out = out->data;
    p.q_ts = q->token_stride;
    p.q_hs = q->head_stride;
    p.o_ts = out->token_stride;
    p.o_hs = out->head_stride;
    p.lse = lse;
    p.k_scale = cache->k_scale;
    p.v_scale = cache->v_scale;
    p.scale = opts->scale != 0.f ? opts->scale : 1.f / std::sqrt((float)d);
    p.causal = opts->causal != 0;
    p.window = opts->window;
    p.q_vec = aligned16(*q);
    p.o_vec = aligned16(*out);
    p.counters = static_cast<int *>(workspace);
    p.part = reinterpret_cast<float *>(static_cast<char *>(workspace) + kPagedZeroed);
    p.status = dev_status;
    p.wait_ns = g_wait_ns;
    if (tree) {
        p.mask = reinterpret_cast<const uint32_t *>(tree->mask);
        p.words = tree->words;
    }
    const int ctas = sms < kPagedMaxCtas ? sms : kPagedMaxCtas;
    // units are of 16 rows and tiles of 128 keys at least; every sequence may have all rows (a
    // q_start that goes back is reported, and those that fit on their own are still worked on:
    // 16 of 31 sequences with all rows each would bring 16 times what the rows alone allow)
    p.small = p.n_seq * ((double)n_tok * p.rep / 16 + 1) * ((double)p.table_stride * p.P / 128 + 3) < 1e9;
    // The row kernel passes over the keys once for every 16 packed rows, the tile kernel
    // once for every 256 at 2.8 times the cost and some 20 us more for its start, its
    // outputs and the joining of cut units. So the row kernel has what fits one of its
    // units, and chunks up to so many passes over 128 keys in the whole batch (kv counted
    // by max_kv, a unit's own time as three passes). Passes are a rough measure: chunks of few
    // tokens on long contexts favour the rows, many short ones the tiles. Measured, row
    // against tile kernel, us, 28/4 heads of 128, 16 bits: 1179 passes (8 tokens on 8000)
    // 23 / 34; 2465 (128 on 1000) 30 / 26; 3930 (32 on 8000) 39 / 47; 4554 (8 on 32000) 43 /
    // 46; 4768 (8 x 16 on 2000) 43 / 32; 9864 (16 x 8 on 4000) 78 / 50. 8 bits: 2465 34 / 31;
    // 3930 38 / 54; 4554 40 / 52; 4768 44 / 39; 9864 67 / 59; 13376 74 / 86. 14/2 heads of 64, 16
    // bits: 2277 (8 on 32000) 23 / 31; 2595 (8 x 32 on 1000) 23 / 20; 4932 30 / 28. Either
    // kernel is up to 1.6 times the other on the wrong side of the border. A window is not
    // counted: 32 tokens that look back 512 of 30000 positions take the tiles' 19 where the rows take 11.
    const double rows16 = (double)p.G * ((double)n_tok * p.rep / 16 + p.n_seq);
    const double passes = (batch->max_kv > 0 ? batch->max_kv : (double)p.table_stride * p.P) / 128 + 3;
    bool tiles = (long long)batch->max_q * p.rep > 16 &&
                 (tree ? trees_in_tiles(d, cache->type == KORE_CUDA_E4M3, G, p.rep, p.n_seq, n_tok,
                                        batch->max_kv > 0 ? batch->max_kv : (double)p.table_stride * p.P, ctas)
                       : rows16 * passes > (cache->type == KORE_CUDA_E4M3 ? 13500.0 : 6200.0));
    const int wanted = g_tree_kernel;
    if (tree && wanted != KORE_CUDA_TREE_BY_SIZE) tiles = wanted == KORE_CUDA_TREE_TILES;
    const bool plain = tiles && cache->type == KORE_CUDA_E4M3;   // widened before it is read as an operand
    // tokens of a box: the largest power of two that divides the page, up to a tile
    const int most = tiles ? (tree ? 64 : 128) : d * type_bytes(cache->type) == 256 ? 16 : 32;
    p.box = 16;
    while (p.box < most && p.P % (2 * p.box) == 0) p.box *= 2;
    if (!encode_pages(cache->k, cache, p.box, plain, &p.tm_k) || !encode_pages(cache->v, cache, p.box, plain, &p.tm_v))
        return refuse(KORE_CUDA_ECUDA, "the pages' tensor maps could not be encoded");
    if (tiles && tree) return launched(launch_paged_tree_tiles(p, d, q->type, cache->type, ctas, (cudaStream_t)stream), "paged_tree_attn");
    if (tiles) return launched(launch_paged_tiles(p, d, q->type, cache->type, ctas, (cudaStream_t)stream), "paged_attn");
    return launched(launch_paged_rows(p, d, q->type, cache->type, ctas, (cudaStream_t)stream), "paged_attn");
}

extern "C" int kore_cuda_paged_attn_dev(const kore_cuda_pages *cache, const kore_cuda_batch *batch, int n_tok,
                                        const kore_cuda_rows *q, const kore_cuda_rows *out, float *lse,
                                        const kore_cuda_attn_opts *opts, void *workspace, long long workspace_bytes,
                                        int *dev_status, void *stream) {
    return attend(cache, batch, n_tok, q, out, lse, opts, nullptr, workspace, workspace_bytes, dev_status, stream);
}

extern "C" int kore_cuda_paged_tree_attn_dev(const kore_cuda_pages *cache, const kore_cuda_batch *batch, int n_tok,
                                             const kore_cuda_rows *q, const kore_cuda_rows *out, float *lse,
                                             const kore_cuda_attn_opts *opts, const kore_cuda_tree *tree,
                                             void *workspace, long long workspace_bytes, int *dev_status, void *stream) {
    if (!tree) return refuse(KORE_CUDA_EINVAL, "the tree is null");
    return attend(cache, batch, n_tok, q, out, lse, opts, tree, workspace, workspace_bytes, dev_status, stream);
}

extern "C" unsigned long long kore_cuda_capture_id(void *stream) {
    cudaStreamCaptureStatus st;
    unsigned long long id = 0;
    if (cudaStreamGetCaptureInfo((cudaStream_t)stream, &st, &id) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    return st == cudaStreamCaptureStatusActive ? id : 0;
}
