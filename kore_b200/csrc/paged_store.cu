// paged_store.cu — a step's keys and values stored at given slots of a caller-owned paged
// cache, with norms of queries and keys for each head and the rotation on the way (sm_100a).
//
// y = x / sqrt(mean(x^2) + eps) * w over a head's d values, then the rotation of
// paged_rope.cu at the token's position, then one rounding to the output's type. The
// mean and all else in 32 bits; a head whose squares (or, with an eps of such a size, their mean and eps) overflow them
// is scaled by 2^-96 for its sum, and eps with it.
//
// Bound by HBM in bytes (every value is read once and written once), and nearly as much by
// instructions: some 110 for 16 values of a lane, half of them the rotation's separate products and
// the widening. So what can be known once is: a warp has the same heads of many tokens, their
// weights in registers, and the next token's rows, angles and place on their way while it works on one. A
// head's sum is a shuffle of the lanes that hold it. Slots and positions come with the tokens, so
// that nothing searches the batch. 6689 tokens of 28/4 heads of 128 in f16 (124 MB): 27.2 us, 4.6
// TB/s; a CTA a token with four heads a thread took 56. 48 tokens: 2.3 us. Rows in 32 bits into 32, 16 and 8 bits: 50, 48 and
// 48 us (250, 236 and 230 MB, 4.8 to 5.0 TB/s); without norms 26.6, without the rotation 25.9. By pairs of any place (rows
// off 16 bytes, other head sizes, weights of another 16-bit type than the rows): 98 us, a value a load.

#include "paged_values.cuh"

#include "kore_cuda.h"

#include <type_traits>

namespace kore {
namespace {

constexpr unsigned FULL = 0xffffffffu;

constexpr int kStoreThreads = 128;
// Two query heads a lane and 16 warps an SM: 6689 tokens of 28/4 heads of 128 in f16 take 27 us; three heads
// (their registers spill) 35, one head with 20 warps 28.
constexpr int kStoreHeads = 2;
template <typename T>
constexpr int kStoreCtas = sizeof(T) == 4 ? 3 : 4;   // of an SM, as the registers allow

__device__ __forceinline__ float weight1(const void *w, int type, long long e) {
    if (type == KORE_CUDA_F32) return static_cast<const float *>(w)[e];
    if (type == KORE_CUDA_F16) return to_f(static_cast<const __half *>(w)[e]);
    return to_f(static_cast<const __nv_bfloat16 *>(w)[e]);
}

// of a normal number (eps is one)
__device__ __forceinline__ float rsqrt_normal(float x) {
    float y;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// eps beside a mean of squares of values times 2^-96
__device__ __forceinline__ float eps_scaled(float eps) { return __fmul_rn(__fmul_rn(eps, 0x1p-96f), 0x1p-96f); }

// 1 / sqrt(mean + eps) from the head's sum of squares, to be followed by a factor `post`: 1, or 2^-96
// for heads whose sum passes `most`, of which again() gives the sum of (x 2^-96)^2.
// The factor stays apart, since their root is below the normal numbers.
template <typename F>
__device__ __forceinline__ float root(float sum, int d, float eps, float most, float &post, F again) {
    post = 1.f;
    if (__any_sync(FULL, sum > most)) {
        const float small = again();
        if (sum > most) {
            post = 0x1p-96f;
            return rsqrt_normal(__fadd_rn(__fdiv_rn(small, (float)d), eps_scaled(eps)));
        }
    }
    return rsqrt_normal(__fadd_rn(__fdiv_rn(sum, (float)d), eps));
}

// Where a row goes; none where it is left out.
struct Place {
    int page, slot, pos;   // page -1: none
};
__device__ __forceinline__ Place place_at(const StoreParams &p, long long at, int pos, bool report) {
    Place w{-1, 0, pos};
    if (at < 0 || pos < 0) return w;   // padding
    const int code = at >= p.n_slots ? DEV_BAD_PAGE : p.table && pos >= p.n_pos ? DEV_BAD_POSITION : 0;
    if (code) {
        if (report) raise_error(p.status, code);
        return w;
    }
    w.page = at <= 0x7fffffffll ? p.by_page.div((int)at) : (int)(at / p.P);
    w.slot = (int)(at - (long long)w.page * p.P);
    return w;
}

// ---------------------------------------------------------------- vectors of 8 values

// 16 values of a head as they are in memory (two vectors of 8), and as pairs of fp32.
template <typename T>
struct Raw {
    uint4 v[2 * sizeof(T) / 2];
    __device__ __forceinline__ void load(const T *a, const T *b) {   // (rows may be written in place: no ld.nc)
        constexpr int N = sizeof(T) / 2;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] = reinterpret_cast<const uint4 *>(a)[i];
            v[N + i] = reinterpret_cast<const uint4 *>(b)[i];
        }
    }
};
using Pair = unsigned long long;   // two fp32

template <typename T>
__device__ __forceinline__ void widen(const Raw<T> &r, Pair (&a)[4], Pair (&b)[4]) {
    const T *h = reinterpret_cast<const T *>(r.v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        a[i] = pk2(to_f(h[2 * i]), to_f(h[2 * i + 1]));
        b[i] = pk2(to_f(h[8 + 2 * i]), to_f(h[8 + 2 * i + 1]));
    }
}
__device__ __forceinline__ F8 values(const Pair (&x)[4]) {
    F8 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) upk2(x[i], r.v[2 * i], r.v[2 * i + 1]);
    return r;
}
// Angles as they lie in the table: (cos, sin) of 8 pairs.
struct Angles {
    float4 v[4];
};

// a and b: B heads' 16 values a lane, normed and times their weights; by whole warps, the L lanes of a head
// side by side. weigh(k, wa, wb) gives head k's weights; most: as for root().
template <int D, int B, typename F>
__device__ __forceinline__ void norm_heads(Pair (&a)[B][4], Pair (&b)[B][4], float eps, float most, F weigh) {
    // step by step for all of the heads, so that their chains run side by side
    float f[B], post[B];
    auto squares = [&](float x) {
        const Pair xx = pk2(x, x);
#pragma unroll
        for (int k = 0; k < B; ++k) {
            Pair y = 0ull, z = 0ull;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const Pair u = x == 1.f ? a[k][i] : mul2(a[k][i], xx), v = x == 1.f ? b[k][i] : mul2(b[k][i], xx);
                y = fma2(u, u, y);
                z = fma2(v, v, z);
            }
            float lo, hi;
            upk2(add2(y, z), lo, hi);
            f[k] = lo + hi;
        }
#pragma unroll
        for (int o = 1; o < D / 16; o <<= 1)
#pragma unroll
            for (int k = 0; k < B; ++k) f[k] += __shfl_xor_sync(FULL, f[k], o);
    };
    squares(1.f);
    bool over = false;
#pragma unroll
    for (int k = 0; k < B; ++k) {
        over |= f[k] > most;
        post[k] = 1.f;
    }
    const bool any = __any_sync(FULL, over);
    if (any) {
        float g[B];
#pragma unroll
        for (int k = 0; k < B; ++k) g[k] = f[k];
        squares(0x1p-96f);
#pragma unroll
        for (int k = 0; k < B; ++k) {
            if (g[k] > most) post[k] = 0x1p-96f;
            else f[k] = g[k];
        }
    }
#pragma unroll
    for (int k = 0; k < B; ++k) {
        f[k] = rsqrt_normal(__fadd_rn(f[k] * (1.f / D), post[k] != 1.f ? eps_scaled(eps) : eps));
        Pair wa[4], wb[4];
        weigh(k, wa, wb);
        const Pair ff = pk2(f[k], f[k]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            a[k][i] = mul2(mul2(a[k][i], ff), wa[i]);
            b[k][i] = mul2(mul2(b[k][i], ff), wb[i]);
        }
        if (any) {
            const Pair pp = pk2(post[k], post[k]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                a[k][i] = mul2(a[k][i], pp);
                b[k][i] = mul2(b[k][i], pp);
            }
        }
    }
}

template <bool INTER>
__device__ __forceinline__ void rotate_head(Pair (&a)[4], Pair (&b)[4], const Angles &w) {
    const float *c = reinterpret_cast<const float *>(w.v);   // (cos, sin) by turns
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float x0, x1, y0, y1;
        upk2(a[i], x0, x1);
        upk2(b[i], y0, y1);
        if constexpr (INTER) {   // pairs 8j + i in a and 8j + 4 + i in b
            a[i] = pk2(rope_lo(x0, x1, c[2 * i], c[2 * i + 1]), rope_hi(x0, x1, c[2 * i], c[2 * i + 1]));
            b[i] = pk2(rope_lo(y0, y1, c[2 * i + 8], c[2 * i + 9]), rope_hi(y0, y1, c[2 * i + 8], c[2 * i + 9]));
        } else {   // (one by one: mul.rn.f32x2 and add.rn.f32x2 became one fma, which is not kore's bits)
            a[i] = pk2(rope_lo(x0, y0, c[4 * i], c[4 * i + 1]), rope_lo(x1, y1, c[4 * i + 2], c[4 * i + 3]));
            b[i] = pk2(rope_hi(x0, y0, c[4 * i], c[4 * i + 1]), rope_hi(x1, y1, c[4 * i + 2], c[4 * i + 3]));
        }
    }
}

// One warp's heads of every `stride`-th token from t on: B a lane, HW * B from h0 on, of q (QUERIES), or of k
// or v (is_v). The next token's rows are asked for as soon as this one's are widened, its angles
// behind this one's rotation, the place of the one after with them.
template <typename T, typename C, typename WT, int D, bool INTER, bool QUERIES>
__device__ __forceinline__ void store_heads(const StoreParams &p, int t, int stride, int h0, bool is_v) {
    constexpr int L = D / 16, HW = 32 / L, B = QUERIES ? kStoreHeads : 1;
    const int lane = threadIdx.x & 31, j = lane % L, h = h0 + lane / L, heads = QUERIES ? p.q.heads : p.G;
    const int rot = p.table && !is_v ? p.rot : 0;
    const bool turn = j < rot / 16, inter = INTER || !turn;
    const int e0 = inter ? 16 * j : 8 * j, gap = inter ? 8 : rot / 2;
    const HeadRows &r = QUERIES ? p.q : is_v ? p.v : p.k;
    const T *src = static_cast<const T *>(r.in) + h * r.in_hs + e0;
    const long long ts = r.in_ts, hs = r.in_hs;
    bool live[B];
#pragma unroll
    for (int k = 0; k < B; ++k) live[k] = h + k * HW < heads;
    auto load_rows = [&](Raw<T> (&raw)[B], int x) {
        if (x >= p.n_tok) return;
#pragma unroll
        for (int k = 0; k < B; ++k)
            if (live[k]) raw[k].load(src + x * ts + k * HW * hs, src + x * ts + k * HW * hs + gap);
    };
    auto load_place = [&](int x) -> Place {
        if (x >= p.n_tok) return Place{-1, 0, 0};
        return place_at(p, __ldg(p.slots + x), p.pos ? __ldg(p.pos + x) : 0, is_v && h0 == 0 && lane == 0);
    };
    auto load_angles = [&](Angles &w, const Place &at) {
        if (!turn || at.page < 0) return;
        const float4 *tab = reinterpret_cast<const float4 *>(p.table + ((long long)at.pos * (rot / 2) + 8 * j) * 2);
#pragma unroll
        for (int i = 0; i < 4; ++i) w.v[i] = __ldg(tab + i);
    };
    const WT *wt = static_cast<const WT *>(QUERIES ? p.q_weight : is_v ? nullptr : p.k_weight);
    const long long w_hs = QUERIES ? p.q_weight_hs : p.k_weight_hs;
    auto load_weights = [&](int k, Pair (&wa)[4], Pair (&wb)[4]) {
        const WT *w = wt + (live[k] ? h + k * HW : 0) * w_hs + e0;
        Raw<WT> raw;
        raw.load(w, w + gap);
        widen(raw, wa, wb);
    };
    const float *scales = is_v ? p.v_scale : p.k_scale;
    const float scale = !QUERIES && sizeof(C) == 1 && scales && live[0] ? __ldg(scales + h) : 1.f;
    Raw<T> raw[B];
    Angles ang;
    load_rows(raw, t);
    Place at = load_place(t), next = load_place(t + stride);
    load_angles(ang, at);
    Pair wa[4], wb[4];
    if (wt) load_weights(0, wa, wb);
    for (; t < p.n_tok; t += stride) {
        Pair a[B][4], b[B][4];
#pragma unroll
        for (int k = 0; k < B; ++k) widen(raw[k], a[k], b[k]);
        load_rows(raw, t + stride);
        if (at.page >= 0 && wt)
            norm_heads<D, B>(a, b, p.eps, p.most, [&](int k, Pair (&x)[4], Pair (&y)[4]) {
                if (k > 0 && w_hs) load_weights(k, x, y);
                else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        x[i] = wa[i];
                        y[i] = wb[i];
                    }
                }
            });
        if (turn) {
#pragma unroll
            for (int k = 0; k < B; ++k) rotate_head<INTER>(a[k], b[k], ang);
        }
        const Place w = at;
        at = next;
        load_angles(ang, at);
        next = load_place(t + 2 * stride);
        if (w.page < 0) continue;
        if constexpr (QUERIES) {
            T *dst = static_cast<T *>(p.q.out) + t * p.q.out_ts + h * p.q.out_hs + e0;
#pragma unroll
            for (int k = 0; k < B; ++k) {
                if (!live[k]) continue;
                store8(dst + k * HW * p.q.out_hs, values(a[k]), 1.f);
                store8(dst + k * HW * p.q.out_hs + gap, values(b[k]), 1.f);
            }
        } else if (live[0]) {
            C *dst = static_cast<C *>(is_v ? p.vc : p.kc) + w.page * p.page_stride + ((long long)h * p.P + w.slot) * D + e0;
            if (sizeof(C) == 1 && scale == 0.f) {   // all that the head can hold is 0, and 0 / 0 would not be
#pragma unroll
                for (int i = 0; i < 4; ++i) a[0][i] = b[0][i] = 0ull;
            }
            const float by = sizeof(C) == 1 && scale == 0.f ? 1.f : scale;
            store8(dst, values(a[0]), by);
            store8(dst + gap, values(b[0]), by);
        }
    }
}

// T: type of the rows; C: type of the cache; WT: of the weights; D: head size. Rows and weights 16-byte
// aligned, rot a multiple of 16.
template <typename T, typename C, typename WT, int D, bool INTER>
__global__ void __launch_bounds__(kStoreThreads, kStoreCtas<T>) store_kernel(const __grid_constant__ StoreParams p, int units, int stride) {
    constexpr int HW = 32 / (D / 16), B = kStoreHeads;
    grid_dep_wait();
    grid_dep_launch();
    const int of_q = (p.q.heads + HW * B - 1) / (HW * B);
    const int warp = blockIdx.x * (kStoreThreads / 32) + (threadIdx.x >> 5), t = warp / units, x = warp - t * units;
    if (t >= stride) return;   // (warps left over behind the last whole token)
    if (x < of_q) store_heads<T, C, WT, D, INTER, true>(p, t, stride, x * HW * B, false);
    else store_heads<T, C, WT, D, INTER, false>(p, t, stride, (x - of_q) / 2 * HW, (x - of_q) & 1);
}

// ---------------------------------------------------------------- pairs of any place

// Rows, sizes and weights of any alignment: a CTA a token, a warp a head, its pairs of values (up to
// four a lane) one by one.
template <typename T, typename C>
__global__ void __launch_bounds__(256) store_pairs_kernel(const __grid_constant__ StoreParams p) {
    constexpr int N = 4;
    grid_dep_wait();
    grid_dep_launch();
    const int t = blockIdx.x, lane = threadIdx.x & 31;
    const int nq = p.q.heads, nk = nq + p.G, nv = nk + p.G, pairs = p.d / 2;
    const int rot = p.table ? p.rot : 0;
    const Place w = place_at(p, __ldg(p.slots + t), p.pos ? __ldg(p.pos + t) : 0, threadIdx.x == 0);
    if (w.page < 0) return;
    int e0[N], e1[N];
    float c[N], s[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int x = lane + 32 * i;
        const bool turn = x < rot / 2, inter = p.interleaved || !turn;
        e0[i] = inter ? 2 * x : x;
        e1[i] = inter ? e0[i] + 1 : x + rot / 2;
        c[i] = 1.f;
        s[i] = 0.f;
        if (turn) {
            const float *tab = p.table + ((long long)w.pos * (rot / 2) + x) * 2;
            c[i] = __ldg(tab);
            s[i] = __ldg(tab + 1);
        }
    }
    for (int h = threadIdx.x >> 5; h < nv; h += blockDim.x >> 5) {
        const bool is_q = h < nq, is_k = !is_q && h < nk;
        const HeadRows &r = is_q ? p.q : is_k ? p.k : p.v;
        const int hh = is_q ? h : is_k ? h - nq : h - nk;
        const T *src = static_cast<const T *>(r.in) + (long long)t * r.in_ts + (long long)hh * r.in_hs;
        float a[N], b[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const bool in = lane + 32 * i < pairs;
            a[i] = in ? to_f(src[e0[i]]) : 0.f;
            b[i] = in ? to_f(src[e1[i]]) : 0.f;
        }
        const void *wt = is_q ? p.q_weight : is_k ? p.k_weight : nullptr;
        if (wt) {
            auto squares = [&](float f) {
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < N; ++i) sum = fmaf(a[i] * f, a[i] * f, fmaf(b[i] * f, b[i] * f, sum));
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) sum += __shfl_xor_sync(FULL, sum, o);
                return sum;
            };
            float post;
            const float f = root(squares(1.f), p.d, p.eps, p.most, post, [&]() { return squares(0x1p-96f); });
            const long long w0 = (long long)hh * (is_q ? p.q_weight_hs : p.k_weight_hs);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (lane + 32 * i >= pairs) continue;
                a[i] = a[i] * f * weight1(wt, p.weight_type, w0 + e0[i]) * post;
                b[i] = b[i] * f * weight1(wt, p.weight_type, w0 + e1[i]) * post;
            }
        }
        const float *scales = is_k ? p.k_scale : p.v_scale;
        float sc = !is_q && sizeof(C) == 1 && scales ? __ldg(scales + hh) : 1.f;
        const bool none = sc == 0.f;   // all that the head can hold is 0, and 0 / 0 would not be
        if (none) sc = 1.f;
        T *qd = static_cast<T *>(r.out) + (long long)t * r.out_ts + (long long)hh * r.out_hs;
        C *cd = static_cast<C *>(is_k ? p.kc : p.vc) + w.page * p.page_stride + ((long long)hh * p.P + w.slot) * p.d;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (lane + 32 * i >= pairs) continue;
            float y = a[i], z = b[i];
            if (lane + 32 * i < rot / 2 && (is_q || is_k)) {
                y = rope_lo(a[i], b[i], c[i], s[i]);
                z = rope_hi(a[i], b[i], c[i], s[i]);
            }
            if (is_q) {
                store1(qd + e0[i], y, 1.f);
                store1(qd + e1[i], z, 1.f);
            } else {
                store1(cd + e0[i], none ? 0.f : y, sc);
                store1(cd + e1[i], none ? 0.f : z, sc);
            }
        }
    }
}

template <typename T, typename C>
cudaError_t launch_tc(const StoreParams &p, bool vec, int sms, cudaStream_t s) {
    if (!vec) {
        const int heads = p.q.heads + 2 * p.G, threads = heads < 8 ? 32 * heads : 256;
        return launch(store_pairs_kernel<T, C>, p.n_tok, threads, 0, s, p);
    }
    auto go = [&](auto d, auto inter, auto w) {
        constexpr int D = decltype(d)::value, HW = 32 / (D / 16), B = kStoreHeads;
        using WT = decltype(w);
        constexpr int W = kStoreThreads / 32;
        // units: warps that a token takes; tokens beyond what the SMs hold at once come in turns
        const int units = (p.q.heads + HW * B - 1) / (HW * B) + 2 * ((p.G + HW - 1) / HW);
        const long long want = ((long long)p.n_tok * units + W - 1) / W, hold = (long long)sms * kStoreCtas<T>, least = (units + W - 1) / W;
        const int ctas = (int)(want < hold ? want : hold > least ? hold : least);
        return launch(store_kernel<T, C, WT, D, decltype(inter)::value>, ctas, kStoreThreads, 0, s, p, units, ctas * W / units);
    };
    auto of_size = [&](auto inter, auto w) {
        switch (p.d) {
            case 64: return go(std::integral_constant<int, 64>{}, inter, w);
            case 128: return go(std::integral_constant<int, 128>{}, inter, w);
            default: return go(std::integral_constant<int, 256>{}, inter, w);
        }
    };
    auto of_weights = [&](auto w) { return p.interleaved ? of_size(std::true_type{}, w) : of_size(std::false_type{}, w); };
    return p.weight_type == KORE_CUDA_F32 ? of_weights(0.f) : of_weights(T{});
}

}  // namespace

cudaError_t launch_store(const StoreParams &p, int in_type, int cache_type, bool vec, int sms, cudaStream_t s) {
    using bf16 = __nv_bfloat16;
    using e4m3 = __nv_fp8_e4m3;
#define KORE_STORE(IT, CT, T, C) \
    if (in_type == IT && cache_type == CT) return launch_tc<T, C>(p, vec, sms, s)
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
