// paged_store.cu — a step's keys and values stored at given slots of a caller-owned paged
// cache, with norms of queries and keys for each head and the rotation on the way (sm_100a).
//
// y = x / sqrt(mean(x^2) + eps) * w over a head's d values, then the rotation of
// paged_rope.cu at the token's position, then one rounding to the output's type. The
// mean and all else in 32 bits; a head whose squares overflow them is scaled by 2^-96 for its sum.
//
// Bound by HBM: every value is read once and written once, the head's sum is a shuffle
// of the lanes that hold it. A CTA a token; a thread keeps 16 values of a head (two vectors that rotate
// into each other) and takes its angles through up to four heads, whose rows are all asked for
// before the first is worked on; slots and positions come with the token, so that no row waits
// for a search of the batch.

#include "paged_values.cuh"

#include "kore_cuda.h"

namespace kore {
namespace {

constexpr unsigned FULL = 0xffffffffu;

// 8 (1) weights of a head from element e on
__device__ __forceinline__ F8 weights8(const void *w, int type, long long e) {
    if (type == KORE_CUDA_F32) return load8(static_cast<const float *>(w) + e);
    if (type == KORE_CUDA_F16) return load8(static_cast<const __half *>(w) + e);
    return load8(static_cast<const __nv_bfloat16 *>(w) + e);
}
__device__ __forceinline__ float weight1(const void *w, int type, long long e) {
    if (type == KORE_CUDA_F32) return static_cast<const float *>(w)[e];
    if (type == KORE_CUDA_F16) return to_f(static_cast<const __half *>(w)[e]);
    return to_f(static_cast<const __nv_bfloat16 *>(w)[e]);
}

// 1 / sqrt(mean + eps) from the head's sum of squares, to be followed by a factor `post`: 1, or 2^-96
// for heads whose squares pass 32 bits, of which again() gives the sum of (x 2^-96)^2 (eps is
// nothing beside that). The factor stays apart, since their root is below the normal numbers.
template <typename F>
__device__ __forceinline__ float root(float sum, int d, float eps, float &post, F again) {
    post = 1.f;
    if (__any_sync(FULL, sum > 3.0e38f)) {
        const float small = again();
        if (sum > 3.0e38f) {
            post = 0x1p-96f;
            return rsqrtf(__fdiv_rn(small, (float)d));
        }
    }
    return rsqrtf(__fadd_rn(__fdiv_rn(sum, (float)d), eps));
}

// The token's place; false where it is left out.
__device__ __forceinline__ bool place(const StoreParams &p, int t, int &page, int &slot, int &pos) {
    const long long at = __ldg(p.slots + t);
    pos = p.pos ? __ldg(p.pos + t) : 0;
    if (at < 0 || pos < 0) return false;   // padding
    int code = 0;
    if (at >= p.n_slots) code = DEV_BAD_PAGE;
    else if (p.table && pos >= p.n_pos) code = DEV_BAD_POSITION;
    if (code) {
        if (threadIdx.x == 0) raise_error(p.status, code);
        return false;
    }
    page = at <= 0x7fffffffll ? p.by_page.div((int)at) : (int)(at / p.P);
    slot = (int)(at - (long long)page * p.P);
    return true;
}

// T: type of the rows; C: type of the cache; VEC: 8 values at a time, heads of 32, 64, 128 or 256
// (16 a thread: 2 to 16 lanes a head) and 16-byte aligned rows, else a warp a head by pairs.
template <typename T, typename C, bool VEC>
__global__ void __launch_bounds__(256) store_kernel(const __grid_constant__ StoreParams p) {
    constexpr int W = VEC ? 8 : 1;
    constexpr int N = VEC ? 1 : 4;       // pairs a thread of one head
    constexpr int B = VEC ? 4 : 1;       // heads on their way at once
    grid_dep_wait();
    grid_dep_launch();
    const int t = blockIdx.x;
    const int items = p.d / (2 * W);
    const int per = VEC ? items : 32;    // lanes a head
    const int j = threadIdx.x % per, h0 = threadIdx.x / per, lanes = blockDim.x / per;
    const int nq = p.q.heads, nk = nq + p.G, nv = nk + p.G;
    const int rot = p.table ? p.rot : 0;
    int e0[N], e1[N];
    bool turn[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int it = j + i * 32;
        turn[i] = it < rot / (2 * W);
        const bool inter = p.interleaved || !turn[i];
        e0[i] = inter ? 2 * W * it : W * it;
        e1[i] = inter ? e0[i] + W : e0[i] + rot / 2;
    }
    int page, slot, pos;
    if (!place(p, t, page, slot, pos)) return;
    float c[N][W], s[N][W];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (!turn[i]) continue;
        const float *tab = p.table + ((long long)pos * (rot / 2) + W * (j + i * 32)) * 2;
        if constexpr (VEC) {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const float4 a = __ldg(reinterpret_cast<const float4 *>(tab) + x);
                c[i][2 * x] = a.x; s[i][2 * x] = a.y; c[i][2 * x + 1] = a.z; s[i][2 * x + 1] = a.w;
            }
        } else {
            c[i][0] = __ldg(tab);
            s[i][0] = __ldg(tab + 1);
        }
    }
    // (every thread takes every turn: the heads' sums are exchanged by whole warps)
    for (int g0 = 0; g0 < nv; g0 += B * lanes) {
        F8 a[B][N], b[B][N];
#pragma unroll
        for (int k = 0; k < B; ++k) {
            const int h = g0 + k * lanes + h0;
            const bool is_q = h < nq, is_k = !is_q && h < nk;
            const HeadRows &r = is_q ? p.q : is_k ? p.k : p.v;
            const int hh = is_q ? h : is_k ? h - nq : h - nk;
            const T *src = static_cast<const T *>(r.in) + (long long)t * r.in_ts + (long long)hh * r.in_hs;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const bool in = h < nv && (VEC || j + i * 32 < items);
                if constexpr (VEC) {
                    if (in) {
                        a[k][i] = load8(src + e0[i]);
                        b[k][i] = load8(src + e1[i]);
                    } else {
#pragma unroll
                        for (int x = 0; x < 8; ++x) a[k][i].v[x] = b[k][i].v[x] = 0.f;
                    }
                } else {
                    a[k][i].v[0] = in ? to_f(src[e0[i]]) : 0.f;
                    b[k][i].v[0] = in ? to_f(src[e1[i]]) : 0.f;
                }
            }
        }
#pragma unroll
        for (int k = 0; k < B; ++k) {
            const int h = g0 + k * lanes + h0;
            const bool is_q = h < nq, is_k = !is_q && h < nk;
            const HeadRows &r = is_q ? p.q : is_k ? p.k : p.v;
            const int hh = is_q ? h : is_k ? h - nq : h - nk;
            const void *wt = is_q ? p.q_weight : is_k ? p.k_weight : nullptr;
            if (p.q_weight || p.k_weight) {
                auto squares = [&](float f) {
                    float sum = 0.f;
#pragma unroll
                    for (int i = 0; i < N; ++i)
#pragma unroll
                        for (int x = 0; x < W; ++x) {
                            const float y = a[k][i].v[x] * f, z = b[k][i].v[x] * f;
                            sum = fmaf(y, y, fmaf(z, z, sum));
                        }
                    for (int o = 1; o < per; o <<= 1) sum += __shfl_xor_sync(FULL, sum, o);
                    return sum;
                };
                float post;
                const float f = root(squares(1.f), p.d, p.eps, post, [&]() { return squares(0x1p-96f); });
                if (wt && h < nv) {
                    const long long w0 = (long long)hh * (is_q ? p.q_weight_hs : p.k_weight_hs);
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        if (!VEC && j + i * 32 >= items) continue;
                        F8 wa, wb;
                        if constexpr (VEC) {
                            wa = weights8(wt, p.weight_type, w0 + e0[i]);
                            wb = weights8(wt, p.weight_type, w0 + e1[i]);
                        } else {
                            wa.v[0] = weight1(wt, p.weight_type, w0 + e0[i]);
                            wb.v[0] = weight1(wt, p.weight_type, w0 + e1[i]);
                        }
#pragma unroll
                        for (int x = 0; x < W; ++x) {
                            a[k][i].v[x] = a[k][i].v[x] * f * wa.v[x];
                            b[k][i].v[x] = b[k][i].v[x] * f * wb.v[x];
                        }
                        if (post != 1.f) {
#pragma unroll
                            for (int x = 0; x < W; ++x) {
                                a[k][i].v[x] *= post;
                                b[k][i].v[x] *= post;
                            }
                        }
                    }
                }
            }
            if (h >= nv) continue;
            const float *scales = is_k ? p.k_scale : p.v_scale;
            float sc = !is_q && sizeof(C) == 1 && scales ? __ldg(scales + hh) : 1.f;
            const bool none = sc == 0.f;   // all that the head can hold is 0, and 0 / 0 would not be
            if (none) sc = 1.f;
            T *qd = static_cast<T *>(r.out) + (long long)t * r.out_ts + (long long)hh * r.out_hs;
            C *cd = static_cast<C *>(is_k ? p.kc : p.vc) + page * p.page_stride + ((long long)hh * p.P + slot) * p.d;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (!VEC && j + i * 32 >= items) continue;
                F8 &y = a[k][i], &z = b[k][i];
                if (turn[i] && (is_q || is_k)) {
                    if (VEC && p.interleaved) {
#pragma unroll
                        for (int x = 0; x < W / 2; ++x) {
                            const float x0 = y.v[2 * x], x1 = y.v[2 * x + 1], y0 = z.v[2 * x], y1 = z.v[2 * x + 1];
                            y.v[2 * x] = rope_lo(x0, x1, c[i][x], s[i][x]);
                            y.v[2 * x + 1] = rope_hi(x0, x1, c[i][x], s[i][x]);
                            z.v[2 * x] = rope_lo(y0, y1, c[i][x + W / 2], s[i][x + W / 2]);
                            z.v[2 * x + 1] = rope_hi(y0, y1, c[i][x + W / 2], s[i][x + W / 2]);
                        }
                    } else {
#pragma unroll
                        for (int x = 0; x < W; ++x) {
                            const float x0 = y.v[x], x1 = z.v[x];
                            y.v[x] = rope_lo(x0, x1, c[i][x], s[i][x]);
                            z.v[x] = rope_hi(x0, x1, c[i][x], s[i][x]);
                        }
                    }
                }
                if (is_q) {
                    if constexpr (VEC) {
                        store8(qd + e0[i], y, 1.f);
                        store8(qd + e1[i], z, 1.f);
                    } else {
                        store1(qd + e0[i], y.v[0], 1.f);
                        store1(qd + e1[i], z.v[0], 1.f);
                    }
                } else {
                    if (none) {
#pragma unroll
                        for (int x = 0; x < W; ++x) y.v[x] = z.v[x] = 0.f;
                    }
                    if constexpr (VEC) {
                        store8(cd + e0[i], y, sc);
                        store8(cd + e1[i], z, sc);
                    } else {
                        store1(cd + e0[i], y.v[0], sc);
                        store1(cd + e1[i], z.v[0], sc);
                    }
                }
            }
        }
    }
}

template <typename T, typename C>
cudaError_t launch_tc(const StoreParams &p, bool vec, cudaStream_t s) {
    const int heads = p.q.heads + 2 * p.G, per = vec ? p.d / 16 : 32;
    const int each = vec ? 4 : 1;
    int threads = (per * ((heads + each - 1) / each) + 31) / 32 * 32;
    if (threads > 256) threads = 256;
    if (vec) return launch(store_kernel<T, C, true>, p.n_tok, threads, 0, s, p);
    return launch(store_kernel<T, C, false>, p.n_tok, threads, 0, s, p);
}

}  // namespace

cudaError_t launch_store(const StoreParams &p, int in_type, int cache_type, bool vec, cudaStream_t s) {
    using bf16 = __nv_bfloat16;
    using e4m3 = __nv_fp8_e4m3;
#define KORE_STORE(IT, CT, T, C) \
    if (in_type == IT && cache_type == CT) return launch_tc<T, C>(p, vec, s)
    KORE_STORE(KORE_CUDA_F32, KORE_CUDA_F32, float, float);
    KORE_STORE(KORE_CUDA_F32, KORE_CUDA_F16, float, __half);
    KORE_STORE(KORE_CUDA_F32, KORE_CUDA_BF16, float, bf16);
    KORE_STORE(KORE_CUDA_F32, KORE_CUDA_E4M3, float, e4m3);
    KORE_STORE(KORE_CUDA_F16, KORE_CUDA_F16, __half, __half);
    KORE_STORE(KORE_CUDA_F16, KORE_CUDA_E4M3, __half, e4m3);
    KORE_STORE(KORE_CUDA_BF16, KORE_CUDA_BF16, bf16, bf16);
    KORE_STORE(KORE_CUDA_BF16, KORE_CUDA_E4M3, bf16, e4m3);
#undef KORE_STORE
    return cudaErrorInvalidValue;
}

}  // namespace kore
