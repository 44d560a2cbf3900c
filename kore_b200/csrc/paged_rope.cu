// paged_rope.cu — rotary positions and the append of a ragged batch into a
// caller-owned paged cache (sm_100a).
//
// rotate: (x0, x1) -> (x0 c - x1 s, x0 s + x1 c) for the first `rot` values of a
// head, pairs (i, i + rot/2) or (2i, 2i + 1); the others are copied. Each
// product is rounded on its own, as kore's rope_neox (kore.cpp:1379-1381), so
// that fp32 rows get kore's bits; 16- and 8-bit results are rounded once.
// append: the same for a batch's new keys (and its queries) with the keys and
// values stored at their sequence's positions in the pages.
//
// Bound by HBM: every value is read once and written once. One CTA per token;
// a thread keeps the (cos, sin) of its 16 values in registers and takes them
// through several heads, so that the table costs one read a token instead of one
// a head. A token's sequence is found by all threads at once (one round of loads); its
// length, page, angles and rows are asked for behind that, one after another, which is what
// a call of few tokens takes. 4096 tokens of 28 heads of 128 in bf16 (61 MB): 13.1 us out of
// HBM, 4.6 TB/s; 9.2 us where the rows are in L2.

#include "paged_values.cuh"

#include "kore_cuda.h"

namespace kore {
namespace {

// Where token t's new key goes: page and slot, or none.
struct Place {
    int pos;         // -1: the token is left out
    int page, slot;
};

// Finds the token's sequence and place with all threads of the CTA.
__device__ __forceinline__ Place place_of(const RotateParams &p, int t, int *found) {
    for (int s = threadIdx.x; s < p.n_seq; s += blockDim.x) {
        const int a = __ldg(p.q_start + s), b = __ldg(p.q_start + s + 1);
        if (a <= t && t < b) *found = s;
        if (t == 0 && (a < 0 || b < a || b > p.n_tok)) raise_error(p.status, DEV_BAD_SEQUENCE);
    }
    __syncthreads();
    const int s = *found;
    Place pl{-1, 0, 0};
    if (s < 0) return pl;   // behind the last sequence
    const int a = __ldg(p.q_start + s), b = __ldg(p.q_start + s + 1), kv = __ldg(p.kv_len + s);
    const int pos = kv - (b - t);
    int code = 0;
    if (a < 0 || b > p.n_tok || kv < b - a || kv > (long long)p.table_stride * p.P) code = DEV_BAD_SEQUENCE;
    else if (p.table && pos >= p.n_pos) code = DEV_BAD_POSITION;
    if (!code) {
        pl.page = __ldg(p.page_table + (long long)s * p.table_stride + pos / p.P);
        pl.slot = pos % p.P;
        if (pl.page < 0 || pl.page >= p.n_pages) code = DEV_BAD_PAGE;
    }
    if (code) {
        if (threadIdx.x == 0) raise_error(p.status, code);
        return pl;
    }
    pl.pos = pos;
    return pl;
}

// T: type of the rows; C: type of the cache; VEC: 8 values at a time (rows
// 16-byte aligned, rot and d multiples of 16) or pairs of single values.
template <typename T, typename C, bool APPEND, bool VEC>
__global__ void __launch_bounds__(256) rotate_kernel(const __grid_constant__ RotateParams p) {
    __shared__ int found;
    const int t = blockIdx.x;
    if (APPEND && threadIdx.x == 0) found = -1;
    grid_dep_wait();
    grid_dep_launch();
    Place pl;
    if constexpr (APPEND) {
        __syncthreads();
        pl = place_of(p, t, &found);
    } else {
        pl.pos = __ldg(p.pos + t);
        if (pl.pos >= p.n_pos) {
            if (threadIdx.x == 0) raise_error(p.status, DEV_BAD_POSITION);
            pl.pos = -1;
        }
    }
    if (pl.pos < 0) return;
    // item j of a head: VEC: two vectors of 8 values that are rotated into each
    // other or (behind rot) copied; else two single values
    constexpr int W = VEC ? 8 : 1;
    const int items = p.d / (2 * W);
    const int lanes = blockDim.x / items;   // heads taken at a time
    const int j = threadIdx.x % items, h0 = threadIdx.x / items;
    if (h0 >= lanes) return;
    const int rot = p.table ? p.rot : 0;
    const bool turn = j < rot / (2 * W);
    const bool inter = p.interleaved || !turn;
    // the pair's two places; items behind rot copy two neighbours
    const int e0 = inter ? 2 * W * j : W * j;
    const int e1 = inter ? e0 + W : e0 + rot / 2;
    float c[W], s[W];
    if (turn) {
        const float *tab = p.table + ((long long)pl.pos * (rot / 2) + W * j) * 2;
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float4 a = __ldg(reinterpret_cast<const float4 *>(tab) + i);
                c[2 * i] = a.x; s[2 * i] = a.y; c[2 * i + 1] = a.z; s[2 * i + 1] = a.w;
            }
        } else {
            c[0] = __ldg(tab);
            s[0] = __ldg(tab + 1);
        }
    }
    const int nq = p.q.heads, nk = APPEND ? nq + p.G : nq, nv = APPEND ? nk + p.G : nq;
#pragma unroll 4
    for (int h = h0; h < nv; h += lanes) {
        const bool is_q = h < nq, is_k = !is_q && h < nk;
        const HeadRows &r = !APPEND || is_q ? p.q : is_k ? p.k : p.v;
        const int hh = is_q ? h : is_k ? h - nq : h - nk;
        const T *src = static_cast<const T *>(r.in) + (long long)t * r.in_ts + (long long)hh * r.in_hs;
        F8 a, b;
        if constexpr (VEC) {
            a = load8(src + e0);
            b = load8(src + e1);
        } else {
            a.v[0] = to_f(src[e0]);
            b.v[0] = to_f(src[e1]);
        }
        if (turn && (!APPEND || is_q || is_k)) {
            if (VEC && p.interleaved) {
#pragma unroll
                for (int i = 0; i < W / 2; ++i) {
                    const float x0 = a.v[2 * i], x1 = a.v[2 * i + 1], y0 = b.v[2 * i], y1 = b.v[2 * i + 1];
                    a.v[2 * i] = rope_lo(x0, x1, c[i], s[i]);
                    a.v[2 * i + 1] = rope_hi(x0, x1, c[i], s[i]);
                    b.v[2 * i] = rope_lo(y0, y1, c[i + W / 2], s[i + W / 2]);
                    b.v[2 * i + 1] = rope_hi(y0, y1, c[i + W / 2], s[i + W / 2]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    const float x0 = a.v[i], x1 = b.v[i];
                    a.v[i] = rope_lo(x0, x1, c[i], s[i]);
                    b.v[i] = rope_hi(x0, x1, c[i], s[i]);
                }
            }
        }
        if (!APPEND || is_q) {
            T *dst = static_cast<T *>(r.out) + (long long)t * r.out_ts + (long long)hh * r.out_hs;
            if constexpr (VEC) {
                store8(dst + e0, a, 1.f);
                store8(dst + e1, b, 1.f);
            } else {
                store1(dst + e0, a.v[0], 1.f);
                store1(dst + e1, b.v[0], 1.f);
            }
        } else {
            const float *scales = is_k ? p.k_scale : p.v_scale;
            float sc = sizeof(C) == 1 && scales ? __ldg(scales + hh) : 1.f;
            if (sizeof(C) == 1 && sc == 0.f) {   // all that the head can hold is 0, and 0 / 0 would not be
                sc = 1.f;
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    a.v[i] *= 0.f;
                    b.v[i] *= 0.f;
                }
            }
            C *dst = static_cast<C *>(is_k ? p.kc : p.vc) + pl.page * p.page_stride +
                     ((long long)hh * p.P + pl.slot) * p.d;
            if constexpr (VEC) {
                store8(dst + e0, a, sc);
                store8(dst + e1, b, sc);
            } else {
                store1(dst + e0, a.v[0], sc);
                store1(dst + e1, b.v[0], sc);
            }
        }
    }
}

// (cos, sin) of position * frequency: the product and the functions in 64 bits
// (fp32 would lose the angle's fraction at far positions), rounded once.
struct Freqs {
    float f[128];
};
__global__ void __launch_bounds__(256) rope_table_kernel(const __grid_constant__ Freqs f, int half, double amp,
                                                         int n_pos, float2 *table) {
    grid_dep_wait();
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= (long long)n_pos * half) return;
    const int pos = (int)(i / half), j = (int)(i % half);
    double s, c;
    sincos((double)pos * (double)f.f[j], &s, &c);
    table[i] = make_float2((float)(c * amp), (float)(s * amp));
}

template <typename T, typename C, bool APPEND>
cudaError_t launch_tc(const RotateParams &p, bool vec, cudaStream_t s) {
    // four heads a thread: the table's values in its registers serve all of them,
    // and a CTA is small enough for many tokens an SM (5303 tokens of 28/4 heads of
    // 128: 19.8 us; two heads 21.9, six 19.9). Two where the CTAs would not fill the SMs
    // (48 tokens: 2.7 us; four heads 2.9)
    const int heads = p.q.heads + (APPEND ? 2 * p.G : 0);
    const int items = p.d / (vec ? 16 : 2);
    const int each = p.n_tok >= 4 * 148 ? 4 : 2;
    int threads = items * ((heads + each - 1) / each);
    threads = threads < items ? items : threads;
    threads = (threads + 31) / 32 * 32;
    if (threads > 256) threads = 256;
    if (vec) return launch(rotate_kernel<T, C, APPEND, true>, p.n_tok, threads, 0, s, p);
    return launch(rotate_kernel<T, C, APPEND, false>, p.n_tok, threads, 0, s, p);
}

}  // namespace

cudaError_t launch_rope_table(const float *freq, int half, double amp, int n_pos, float *table, cudaStream_t s) {
    Freqs f;
    for (int i = 0; i < 128; ++i) f.f[i] = i < half ? freq[i] : 0.f;
    const long long n = (long long)n_pos * half;
    return launch(rope_table_kernel, (int)((n + 255) / 256), 256, 0, s, f, half, amp, n_pos,
                  reinterpret_cast<float2 *>(table));
}

cudaError_t launch_rotate(const RotateParams &p, int in_type, int cache_type, bool vec, cudaStream_t s) {
    using bf16 = __nv_bfloat16;
    using e4m3 = __nv_fp8_e4m3;
    const bool append = p.kc != nullptr;
    if (p.n_tok == 0) return cudaSuccess;
#define KORE_ROTATE(IT, CT, T, C) \
    if (in_type == IT && cache_type == CT) return launch_tc<T, C, true>(p, vec, s)
    if (append) {
        KORE_ROTATE(KORE_CUDA_F32, KORE_CUDA_F32, float, float);
        KORE_ROTATE(KORE_CUDA_F32, KORE_CUDA_F16, float, __half);
        KORE_ROTATE(KORE_CUDA_F32, KORE_CUDA_BF16, float, bf16);
        KORE_ROTATE(KORE_CUDA_F32, KORE_CUDA_E4M3, float, e4m3);
        KORE_ROTATE(KORE_CUDA_F16, KORE_CUDA_F16, __half, __half);
        KORE_ROTATE(KORE_CUDA_F16, KORE_CUDA_E4M3, __half, e4m3);
        KORE_ROTATE(KORE_CUDA_BF16, KORE_CUDA_BF16, bf16, bf16);
        KORE_ROTATE(KORE_CUDA_BF16, KORE_CUDA_E4M3, bf16, e4m3);
    } else {
        if (in_type == KORE_CUDA_F32) return launch_tc<float, float, false>(p, vec, s);
        if (in_type == KORE_CUDA_F16) return launch_tc<__half, __half, false>(p, vec, s);
        if (in_type == KORE_CUDA_BF16) return launch_tc<bf16, bf16, false>(p, vec, s);
    }
#undef KORE_ROTATE
    return cudaErrorInvalidValue;
}

}  // namespace kore
