// paged_tree_tiles.cu — attention of trees of drafted tokens over a caller-owned paged cache of 16 or 8
// bits on the 5th-generation tensor cores (tcgen05, accumulators in tensor memory), sm_100a.
//
// out = softmax(scale q K^T) V for units of 128 packed rows (tokens x the group's query heads), each of
// which sees its sequence's whole context and, of the chunk behind it, the tokens that its mask names.
// A tree has few rows on a long context: a unit's keys stream by once at 4 d bytes (16 bits) for 4 d
// * rows flops, so HBM and the tensor cores bound it alike at some 100 rows, and what counts is that
// neither waits: two CTAs an SM, each with one tile of rows, so that one streams while the other starts
// a unit, joins its parts or writes its outputs (one CTA an SM with two tiles of rows, as for prompts, left
// 4 to 7 us between a CTA's units in which no key moved). Measured, the GPU's time alone (a call among others takes 3 us more at the first
// two): 32 sequences of 16 tokens on up to 8192, 28/4 heads of 128, bf16: 70.7 us (4.05 TB/s, 440 TFLOP/s; the keys
// stream for 43 of them, a CTA's start takes 5, the joints at the end up to 15); 6 of up to 60 on 32768, 8 bits: 122 us
// (535 TFLOP/s); 48 of up to 33 on 3001, 14/2 heads of 64, f16: 31.4; 8 bits and d = 64: 64 tokens on 30064 42, 48 x 16 on
// 2016 31 (floors 4.2 and 4.2). Every instance spills: at 128 registers a thread (16 bits) 252 bytes of stores and
// 196 of loads at d = 128, 40 and 132 at d = 64; at 80 (8 bits) 584 to 588 and 744 to 780.
//   warps 0-3    softmax, a thread a row. Per step of 64 keys: S from tensor memory, mask (a word of bits for
//                32 keys), online softmax (the reference maximum moves only when a score passes it by 2^8;
//                O in tensor memory is rescaled then), P in 16 bits over S, sums in fp32.
//   warp 4       producer: tiles of 64 keys by TMA straight from the pages, through a ring, in the order of
//                the products: K0 K1 V0 K2 V1 .., so that every place but the one in use is on its way.
//   warp 5       issues the MMAs: for each step j O += P_j V_j, then S_{j+2} = Q K_{j+2}^T into the buffer
//                that P_j leaves.
//   warp 6       watches the ring for the issuer, and clears the rows of V that no row of the unit sees:
//                0 * NaN must not reach an output.
//   warps 8-11   (8-bit caches, in warp 6's place) widen the tiles to f16 (exact) from a ring of their own.
// Events, the joints of units cut between CTAs, precision and failures are those of paged_tiles.cu.

#include "paged_mma.cuh"

#include "kore_cuda.h"

#include <type_traits>

namespace kore {
namespace {

constexpr int kKeys = 64;           // keys of a tile and of a step
constexpr int kCtas = 2;            // of an SM
constexpr float kSlack = 8.0f;      // log2 slack before the reference maximum moves
static_assert(kCtas * kM <= kPagedRowsMax, "workspace slots");
static_assert(kCtas * kPagedMaxCtas * sizeof(int) / 2 <= kPagedZeroed, "two CTAs' counters in a word");

// Ring depths: HBM is as busy with 3 to 5 stages of 16 bits (d = 128: 70.5, 71.0 and 71.9 us for 32 sequences of 16
// tokens on up to 8192), with 3 or 4 of 8 bits (119.8, 122.0 for 6 of up to 60 on 32768); what is more in flight
// only waits longer, and the other loads with it.
template <int D, bool E8>
struct TreeCfg {
    static constexpr int HALVES = D / 64;                    // 128-byte wide column blocks
    static constexpr uint32_t BLOCK = kKeys * 128;           // bytes of one such block of a tile
    static constexpr uint32_t TILE = HALVES * BLOCK;         // K or V tile
    static constexpr int STAGES = E8 ? (D == 128 ? 3 : 6) : D == 128 ? 4 : 6;
    static constexpr int THREADS = E8 ? 384 : 256;           // 80 or 128 registers a thread
    static constexpr uint32_t RAW_TILE = kKeys * D;          // 8-bit K or V tile
    static constexpr int RAW_STAGES = D == 128 ? 3 : 8;
    static constexpr int LOADS = E8 ? RAW_STAGES : STAGES;   // stages that the copies fill
    static constexpr uint32_t RING = HALVES * kM * 128;      // behind q: [HALVES][kM rows][128 B]
    static constexpr uint32_t RAW = RING + STAGES * TILE;
    static constexpr uint32_t BARS = RAW + (E8 ? RAW_STAGES * RAW_TILE : 0);
    static constexpr uint32_t SHIFT = BARS + 512;            // E8: [kM] 1 / (power of two on the q row)
    static constexpr uint32_t BYTES = SHIFT + (E8 ? kM * 4 : 0);
    static constexpr uint32_t T_S = 0, T_O = 128;            // tensor memory: S/P buffer b at 64 b, O at T_O
    static_assert(BYTES <= 115712, "half the shared memory of an SM");
    static_assert(STAGES * TILE >= (kPagedMaxSeqs + 2) * 8, "the sums' place");
};

// CTA c has two slots: slot 0 for the unit it goes on with, slot 1 for the one it begins. A slot:
// O to the row's maximum [D/4][128 rows] float4 (a warp's rows stand side by side), then maxima and sums.
template <int D>
constexpr size_t kSlot = (size_t)kM * (D + 2);

__device__ __forceinline__ int load_acquire_gpu(const int *p) {
    int v;
    asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}

// What some row of the unit sees of the keys from x on (counted as for tree_bits); by a whole warp.
__device__ __forceinline__ uint32_t seen_by_some(const PagedAttnParams &p, const Unit<kM, kKeys, true> &u, int x) {
    const int t0 = p.by_rep.div(u.b * kM), t1 = p.by_rep.div(u.b * kM + u.rows - 1);
    uint32_t bits = 0;
    for (int t = t0 + (threadIdx.x & 31); t <= t1; t += 32)
        bits |= tree_bits(p.mask + (long long)(u.q.q0 + t) * p.words, p.words, x, u.q.n);
    return __reduce_or_sync(FULL, bits);
}

// QBF: queries and outputs in bf16, else f16. E8: 8-bit cache, products in f16.
template <int D, bool QBF, bool E8>
__global__ void __launch_bounds__(TreeCfg<D, E8>::THREADS, kCtas) paged_tree_kernel(const __grid_constant__ PagedAttnParams p) {
    using C = TreeCfg<D, E8>;
    constexpr bool BF = QBF && !E8;   // type of the products
    using U = Unit<kM, kKeys, true>;
    using qt = typename std::conditional<QBF, __nv_bfloat16, __half>::type;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t sbase = smem_u32(smem);
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + C::BARS);
    uint64_t *full = bars;                  // [LOADS] a tile has landed
    uint64_t *empty = bars + 8;             // [STAGES] the MMAs of it are done
    uint64_t *q_full = bars + 16;           // the q rows are in shared memory (4 warps)
    uint64_t *ev = bars + 17;               // [2] events
    uint64_t *drained = bars + 19;
    uint64_t *raw_empty = bars + 20;        // [RAW_STAGES] a tile of 8 bits has been widened (4 warps)
    uint64_t *pv_done = bars + 28;          // the last O += P V is done
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 29);
    int *abort_flag = reinterpret_cast<int *>(bars + 30);
    // counters that the issuer polls: [4] P written (and O rescaled) by each softmax warp; ring tiles that are
    // ready: one by the watcher, or [4] by each widening warp
    uint32_t *p_seq = reinterpret_cast<uint32_t *>(bars + 31);
    uint32_t *landed = reinterpret_cast<uint32_t *>(bars + 33);
    constexpr int kLanded = E8 ? 4 : 1;
    int *join = reinterpret_cast<int *>(bars + 35);   // a joint: whether this CTA is the second
    float *q_shift = reinterpret_cast<float *>(smem + C::SHIFT);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    auto free_tmem = [&](uint32_t at) {   // by warp 5
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(256) : "memory");
    };
    if (threadIdx.x == 128) {
        prefetch_map(&p.tm_k);
        prefetch_map(&p.tm_v);
    }
    __syncwarp();
    grid_dep_wait();
    // The SM's second CTA is let in only when the first has given up the right to allocate tensor memory, so that
    // comes first: behind the share, as late as 3 us, the second one's tiles were the last to come (48 sequences
    // of up to 33 tokens at d = 64: 31.5 us instead of 35; 16 of 8 tokens on 1008, 8 bits, d = 128: 26 instead of 29).
    if (warp == 5) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(256)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    U u;
    long long total, x0, x1;
    int ctas;
    if (!find_share<kM, kKeys, 8, 6, true>(p, reinterpret_cast<long long *>(smem + C::RING), u, total, ctas, x0, x1)) {
        fence_before();
        __syncthreads();
        fence_after();
        if (warp == 5) free_tmem(*tmem_slot);
        return;
    }

    if (threadIdx.x == 0) {
        for (int i = 0; i < C::LOADS; ++i) mbar_init(&full[i], 1);
        for (int i = 0; i < C::STAGES; ++i) mbar_init(&empty[i], 1);
        for (int i = 0; E8 && i < C::RAW_STAGES; ++i) mbar_init(&raw_empty[i], 4);
        mbar_init(q_full, 4);
        mbar_init(&ev[0], 1);
        mbar_init(&ev[1], 1);
        mbar_init(drained, 1);
        mbar_init(pv_done, 1);
        *abort_flag = 0;
        for (int i = 0; i < 4; ++i) p_seq[i] = 0;
        for (int i = 0; i < kLanded; ++i) landed[i] = 0;
        mbar_fence_init();
    }
    fence_proxy_async_smem();   // the sums stood where the ring's copies will land
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_slot;
    // Not before: a following kernel's CTA that holds tensor memory and waits for this one to end must not
    // stand in the way of its allocation (nor this one, which allocates behind its wait, in a preceding one's).
    grid_dep_launch();
    // bounded, by whole warps, with one answer for the warp
    auto wait = [&](uint64_t *bar, uint32_t parity, bool copy = false) -> bool {
        bool got = (!copy || p.wait_ns >= kWaitNs) && mbar_try_wait(bar, parity);
        if (__all_sync(FULL, got)) return true;
        if (!got && !*reinterpret_cast<volatile int *>(abort_flag)) {
            got = late_wait(bar, parity, p.wait_ns);
            if (!got) {
                raise_late(p.status);
                *reinterpret_cast<volatile int *>(abort_flag) = 1;
            }
        }
        return __all_sync(FULL, got);
    };
    // until the counters at word[lane], lane < n, have all reached `want`: bounded, by whole warps
    auto reached = [&](const uint32_t *word, int n, uint32_t want) -> bool {
        uint64_t since = 0;
        for (uint32_t polls = 0;; ++polls) {
            const uint32_t v = lane < n ? ld_acquire(word + lane) : want;
            if (__all_sync(FULL, (int)(v - want) >= 0)) return true;
            if ((polls & 1023) == 1023) {
                const uint64_t now = global_ns();
                if (!since) since = now;
                const bool late = now - since > p.wait_ns;
                if (__any_sync(FULL, late || *reinterpret_cast<volatile int *>(abort_flag))) {
                    if (lane == 0) {
                        raise_late(p.status);
                        *reinterpret_cast<volatile int *>(abort_flag) = 1;
                    }
                    return false;
                }
            }
        }
    };
    auto share_tiles = [&](const U &a, int &t0, int &t1) {   // tiles of unit a in [x0, x1)
        const long long first = a.u0 + U::COST;
        t0 = (int)max(0ll, min((long long)a.nt, x0 - first));
        t1 = (int)max(0ll, min((long long)a.nt, x1 - first));
    };
    auto next_unit = [&](U &a) -> bool { return a.u0 + U::COST + a.nt < x1 && a.next(p); };
    // places in the ring of a share's n tiles of a unit: K0 K1 V0 K2 V1 .. V(n-1)
    auto k_pos = [&](int t) { return max(0, 2 * t - 1); };
    auto v_pos = [&](int t, int n) { return t + 1 < n ? 2 * t + 2 : 2 * n - 1; };

    // E8: 80 registers a thread at launch; the softmax needs more, the others fewer (136 + 48 + 56 = 3 * 80).
    if (warp < 4) {
        if constexpr (E8) asm volatile("setmaxnreg.inc.sync.aligned.u32 136;");
        // ------------------------------------------------------------ softmax
        const int r = threadIdx.x;   // row
        const uint32_t lane_off = (uint32_t)(warp * 32) << 16;
        const uint32_t ts = tmem + C::T_S + lane_off, to = tmem + C::T_O + lane_off;
        uint32_t e = 0, n_p = 0;   // events before this unit, P written so far
        bool ok = true;
        const uint32_t scale_sign = p.scale < 0.f ? 0x80008000u : 0u;   // goes into q, so that maxima stay maxima
        const float qs_all = fabsf(p.scale) * 1.44269504088896340736f;
        // offset of this thread's row of unit a in rows of strides ts, hs (of the unit's
        // first row where it has none): the warp's lanes ask one another for theirs
        auto offset_of = [&](const U &a, long long t_s, long long h_s) -> long long {
            const int pr = a.b * kM + (r < a.rows ? r : 0), tok = p.by_rep.div(pr);
            return (long long)(a.q.q0 + tok) * t_s + (long long)(a.g * p.rep + pr - tok * p.rep) * h_s;
        };
        // the q rows of unit a into shared memory: a warp its 32 rows, half a warp a row at d = 128 (a
        // thread its own row would touch a cache line a lane), many of them on their way at once
        auto load_q = [&](const U &a) {
            uint32_t sign = scale_sign;
            if (E8 && p.k_scale && __ldg(p.k_scale + a.g) < 0.f) sign ^= 0x80008000u;
            constexpr int L = D / 8, N = E8 ? 8 : L;   // lanes a row, loads a lane at a time
            const int c = lane % L;
            const long long off = offset_of(a, p.q_ts, p.q_hs);
            uint8_t *dst = smem + (c >> 3) * (kM * 128);
#pragma unroll
            for (int k0 = 0; k0 < L; k0 += N) {
                uint4 v[N];
                if (p.q_vec) {
#pragma unroll
                    for (int k = 0; k < N; ++k)
                        v[k] = __ldg(reinterpret_cast<const uint4 *>(static_cast<const qt *>(p.q) +
                                                                     __shfl_sync(FULL, off, (k0 + k) * (32 / L) + lane / L) + 8 * c));
                } else {
#pragma unroll
                    for (int k = 0; k < N; ++k) {
                        const unsigned short *h = static_cast<const unsigned short *>(p.q) +
                                                  __shfl_sync(FULL, off, (k0 + k) * (32 / L) + lane / L) + 8 * c;
                        uint32_t w[4];
#pragma unroll
                        for (int x = 0; x < 4; ++x) w[x] = (uint32_t)__ldg(h + 2 * x) | ((uint32_t)__ldg(h + 2 * x + 1) << 16);
                        v[k] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
                if constexpr (E8 && QBF) {
                    // bf16 -> f16: rows whose largest value is between 2^-4 and 2^15 go as they are (what is
                    // below f16's range is then below 2^-21 of the largest): all of these, or each times its
                    // power of two
                    auto largest = [](const uint4 &x) {
                        const __nv_bfloat162 *y = reinterpret_cast<const __nv_bfloat162 *>(&x);
                        return __hmax2(__hmax2(__habs2(y[0]), __habs2(y[1])), __hmax2(__habs2(y[2]), __habs2(y[3])));
                    };
                    constexpr unsigned GROUP = (1u << L) - 1;
                    bool fine = true;
#pragma unroll
                    for (int k = 0; k < N; ++k) {
                        const __nv_bfloat162 t = largest(v[k]);
                        const float m = fmaxf(__low2float(t), __high2float(t));
                        const unsigned some = __ballot_sync(FULL, m >= 0.0625f) >> (lane & ~(L - 1));
                        fine &= (some & GROUP) != 0 && m < 32768.f;
                    }
                    if (!__all_sync(FULL, fine)) {
#pragma unroll 1
                        for (int k = 0; k < N; ++k) {
                            uint4 x = v[0];   // (by turns in v[0]: an index would put v into memory)
#pragma unroll
                            for (int y = 0; y + 1 < N; ++y) v[y] = v[y + 1];
                            __nv_bfloat162 t = largest(x);
#pragma unroll
                            for (int o = 1; o < L; o <<= 1) t = __hmax2(t, __shfl_xor_sync(FULL, t, o));
                            const float f = f16_shift(fmaxf(__low2float(t), __high2float(t)));
                            if (c == 0) q_shift[warp * 32 + (k0 + k) * (32 / L) + lane / L] = 1.f / f;
                            uint32_t *w = reinterpret_cast<uint32_t *>(&x);
#pragma unroll
                            for (int y = 0; y < 4; ++y)
                                w[y] = pack2<false>(__uint_as_float(w[y] << 16) * f, __uint_as_float(w[y] & 0xffff0000u) * f);
                            v[N - 1] = x;
                        }
                    } else {
                        if ((lane * L >> 5) / N * N == k0) q_shift[r] = 1.f;   // (this lane's row is among these)
#pragma unroll
                        for (int k = 0; k < N; ++k) {
                            uint32_t *w = reinterpret_cast<uint32_t *>(&v[k]);
#pragma unroll
                            for (int y = 0; y < 4; ++y)
                                w[y] = pack2<false>(__uint_as_float(w[y] << 16), __uint_as_float(w[y] & 0xffff0000u));
                        }
                    }
                }
#pragma unroll
                for (int k = 0; k < N; ++k) {
                    const int row = warp * 32 + (k0 + k) * (32 / L) + lane / L;
                    v[k].x ^= sign;
                    v[k].y ^= sign;
                    v[k].z ^= sign;
                    v[k].w ^= sign;
                    if (row >= a.rows) v[k] = make_uint4(0, 0, 0, 0);
                    *reinterpret_cast<uint4 *>(dst + sw128(row, c & 7)) = v[k];
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
        };
        // the next unit with a tile in this share, from a on
        auto skip_empty = [&](U &a, int &t0, int &t1) -> bool {
            for (;;) {
                share_tiles(a, t0, t1);
                if (t0 < t1) return true;
                if (!next_unit(a)) return false;
            }
        };
        // O, to the row's maximum, into a slot
        auto put_part = [&](float *slot, float m, float l) {
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
                float o[32];
                ld32(to + c, reinterpret_cast<uint32_t *>(o));
                wait_ld();
#pragma unroll
                for (int k = 0; k < 32; k += 4)
                    *(reinterpret_cast<float4 *>(slot) + ((c + k) / 4) * kM + r) = make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
            }
            slot[kM * D + r] = m;
            slot[kM * (D + 1) + r] = l;
        };
        auto put_out = [&](const U &a, float m, float l) {
            const bool in = r < a.rows;
            const float vs = E8 && p.v_scale ? __ldg(p.v_scale + a.g) : 1.f;
            const float inv = l > 0.f || l != l ? vs / l : 0.f;
            qt *dst = static_cast<qt *>(p.out) + offset_of(a, p.o_ts, p.o_hs);
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
                float o[32];
                ld32(to + c, reinterpret_cast<uint32_t *>(o));
                wait_ld();
                // (a row without keys: O is 0 * V of cleared rows)
                uint32_t w[16];
#pragma unroll
                for (int x = 0; x < 16; ++x) w[x] = pack2<QBF>(o[2 * x] * inv, o[2 * x + 1] * inv);
                if (in && p.o_vec) {
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        reinterpret_cast<uint4 *>(dst + c)[x] = make_uint4(w[4 * x], w[4 * x + 1], w[4 * x + 2], w[4 * x + 3]);
                } else if (in) {
                    unsigned short *y = reinterpret_cast<unsigned short *>(dst + c);
#pragma unroll
                    for (int x = 0; x < 16; ++x) {
                        y[2 * x] = (unsigned short)(w[x] & 0xffffu);
                        y[2 * x + 1] = (unsigned short)(w[x] >> 16);
                    }
                }
                __syncwarp();
            }
            const int pr = a.b * kM + r, tok = p.by_rep.div(pr), h = a.g * p.rep + pr - tok * p.rep;
            if (p.lse && in) p.lse[(long long)(a.q.q0 + tok) * p.H + h] = log_sum<BF>(m, l);
        };
        // A part of a cut unit, O in tensor memory: up the tree of its CTAs as far as this one is the second to
        // finish, and out at its root. CTA c's part is in its slot 1 if the unit begins there, else in its slot 0.
        auto join_parts = [&](const U &a, float m, float l) {
            const int c0 = share_of(a.u0 + U::COST, total, ctas);
            const int parts = share_of(a.u0 + U::COST + a.nt - 1, total, ctas) - c0 + 1;
            auto part_of = [&](int k) { return p.part + (size_t)((c0 + k) * 2 + (k == 0)) * kSlot<D>; };
            const int me = blockIdx.x - c0;
            for (int j = 1; (1 << (j - 1)) < parts; ++j) {
                const int left = me >> j << j, right = left + (1 << (j - 1));   // first parts of the two sides
                if (right >= parts) continue;                                   // no right side
                int *counter = p.counters + ((c0 + right) >> 1);                // two CTAs' in a word
                const int shift = 16 * ((c0 + right) & 1), one = 1 << shift;
                const bool is_left = me < right;
                // the other side may be there already: then nothing of this one has to be put down
                auto agree = [&](int x) -> int {   // of the first thread's x
                    if (r == 0) *join = x;
                    asm volatile("bar.sync 1, 128;" ::: "memory");
                    x = *reinterpret_cast<volatile int *>(join);
                    asm volatile("bar.sync 1, 128;" ::: "memory");
                    return x;
                };
                if (agree(r == 0 ? load_acquire_gpu(counter) >> shift & 0xffff : 0)) {
                    if (r == 0) atomicAdd(counter, -one);   // as the next call wants it
                } else {
                    put_part(part_of(is_left ? left : right), m, l);
                    __threadfence();
                    asm volatile("bar.sync 1, 128;" ::: "memory");
                    if (!agree(r == 0 ? atomicAdd(counter, one) >> shift & 0xffff : 0)) return;   // the other side goes on
                    if (r == 0) atomicAdd(counter, -2 * one);
                }
                __threadfence();
                const float *other = part_of(is_left ? right : left);
                const float m2 = __ldcg(other + kM * D + r), l2 = __ldcg(other + kM * (D + 1) + r);
                const float M = fmaxf(m, m2);
                const float f = m == -INFINITY ? 0.f : fast_exp2(m - M), g = m2 == -INFINITY ? 0.f : fast_exp2(m2 - M);
                m = M;
                l = __fadd_rn(__fmul_rn(f, l), __fmul_rn(g, l2));
#pragma unroll 1
                for (int col = 0; col < D; col += 64) {
                    float4 x[16];   // (all on their way at once: a round trip takes a microsecond)
#pragma unroll
                    for (int k = 0; k < 16; ++k) x[k] = __ldcg(reinterpret_cast<const float4 *>(other) + (col / 4 + k) * kM + r);
#pragma unroll
                    for (int c = 0; c < 64; c += 32) {
                        float o[32];
                        ld32(to + col + c, reinterpret_cast<uint32_t *>(o));
                        wait_ld();
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const float4 y = x[c / 4 + k];
                            o[4 * k] = __fadd_rn(__fmul_rn(f, o[4 * k]), __fmul_rn(g, y.x));
                            o[4 * k + 1] = __fadd_rn(__fmul_rn(f, o[4 * k + 1]), __fmul_rn(g, y.y));
                            o[4 * k + 2] = __fadd_rn(__fmul_rn(f, o[4 * k + 2]), __fmul_rn(g, y.z));
                            o[4 * k + 3] = __fadd_rn(__fmul_rn(f, o[4 * k + 3]), __fmul_rn(g, y.w));
                        }
                        st32(to + col + c, reinterpret_cast<const uint32_t *>(o));
                    }
                }
                wait_st();
            }
            put_out(a, m, l);
        };
        int t0, t1;
        bool more = skip_empty(u, t0, t1);
        if (more) {
            load_q(u);
            if (lane == 0) mbar_arrive(q_full);
        }
        while (more && ok) {
            const bool in = r < u.rows;
            const int pr = u.b * kM + r, first = u.q.kv - u.q.n;   // first: the chunk's first key
            const uint32_t *mask = p.mask + (long long)(u.q.q0 + p.by_rep.div(in ? pr : u.b * kM)) * p.words;
            float qs = qs_all;
            if constexpr (E8 && QBF) qs *= q_shift[r];
            if (E8 && p.k_scale) qs *= fabsf(__ldg(p.k_scale + u.g));
            if constexpr (E8) qs = at_least_normal(qs);
            float m = -INFINITY, l = 0.f;
            const int n = t1 - t0;
            auto event = [&](uint32_t no) { return wait(&ev[no & 1], (no >> 1) & 1); };
            for (int j = 0; j < n; ++j) {
                const uint32_t no = e + j, tb = ts + 64 * (no & 1);
                if (!event(no)) {
                    ok = false;
                    break;
                }
                fence_after();
                float s[64];
                ld32(tb, reinterpret_cast<uint32_t *>(s));
                ld32(tb + 32, reinterpret_cast<uint32_t *>(s) + 32);
                wait_ld();
                const int key0 = (u.tile0 + t0 + j) * kKeys;
                if (key0 + kKeys > first) {
                    const uint32_t see[2] = {in ? tree_bits(mask, p.words, key0 - first, u.q.n) : 0u,
                                             in ? tree_bits(mask, p.words, key0 + 32 - first, u.q.n) : 0u};
#pragma unroll
                    for (int x = 0; x < 64; ++x)
                        if (!(see[x >> 5] >> (x & 31) & 1)) s[x] = -INFINITY;
                }
                float mx[8];
#pragma unroll
                for (int x = 0; x < 8; ++x) mx[x] = s[x];
#pragma unroll
                for (int x = 8; x < 64; x += 2) mx[(x >> 1) & 7] = max3(mx[(x >> 1) & 7], s[x], s[x + 1]);
                const float top = max3(max3(mx[0], mx[1], mx[2]), max3(mx[3], mx[4], mx[5]), fmaxf(mx[6], mx[7])) * qs;
                const bool need = top > m + kSlack;
                if (__any_sync(FULL, need)) {
                    const float a = need ? fast_exp2(m - top) : 1.f;
                    if (need) {
                        m = top;
                        l *= a;
                    }
                    if (j > 0) {   // O holds every step before this one only now
                        if (!event(no + 1)) {
                            ok = false;
                            break;
                        }
                        fence_after();
                        const unsigned long long aa = pk2(a, a);
#pragma unroll 1
                        for (int c = 0; c < D; c += 32) {
                            float o[32];
                            ld32(to + c, reinterpret_cast<uint32_t *>(o));
                            wait_ld();
#pragma unroll
                            for (int x = 0; x < 32; x += 2) upk2(mul2(pk2(o[x], o[x + 1]), aa), o[x], o[x + 1]);
                            st32(to + c, reinterpret_cast<const uint32_t *>(o));
                        }
                    }
                }
                const float z = m == -INFINITY ? 0.f : kBias<BF> - m;
                unsigned long long acc[4] = {0ull, 0ull, 0ull, 0ull};
                const unsigned long long qq = pk2(qs, qs), zz = pk2(z, z);
                auto probs = [&](auto huge) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t w[16];
#pragma unroll
                        for (int x = 0; x < 16; ++x) {
                            float a, b;
                            if constexpr (decltype(huge)::value) {
                                a = __fadd_rn(__fmul_rn(s[32 * h + 2 * x], qs), z);
                                b = __fadd_rn(__fmul_rn(s[32 * h + 2 * x + 1], qs), z);
                            } else {
                                upk2(fma2(pk2(s[32 * h + 2 * x], s[32 * h + 2 * x + 1]), qq, zz), a, b);
                            }
                            a = fast_exp2(a);
                            b = fast_exp2(b);
                            acc[x & 3] = add2(acc[x & 3], pk2(a, b));
                            w[x] = pack2<BF>(a, b);
                        }
                        st16(tb + 16 * h, w);
                    }
                };
                // one fused instruction for the factor and the reference, unless a score is so
                // large that its product's rounding alone (2^-24 of it), which the reference has
                // and a fused one has not, is more than exp2 can take
                if (__any_sync(FULL, fabsf(m) > 4194304.f)) probs(std::true_type{});
                else probs(std::false_type{});
                float x, y;
                upk2(add2(add2(acc[0], acc[1]), add2(acc[2], acc[3])), x, y);
                l += x + y;
                wait_st();
                fence_before();
                __syncwarp();
                ++n_p;
                if (lane == 0) st_release(p_seq + warp, n_p);
            }
            // the next unit's q (this one's products with q are done: the last S has come). The issuer
            // hears of it behind this unit's last event: the next unit's events are on the same barriers.
            const U done = u;
            const int d0 = t0, d1 = t1;
            more = next_unit(u) && skip_empty(u, t0, t1);
            if (ok && more) load_q(u);
            // the last product, before the next unit's events
            if (ok) ok = event(e + n + 1);
            e += n + 2;
            if (ok && more && lane == 0) mbar_arrive(q_full);   // (the next unit's products overlap the epilogue)
            // the four warps go on together or not at all (they meet below)
            int all_ok;
            asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbarrier.cta.red.and.pred q, 1, 128, p;\n\t"
                         "selp.b32 %0, 1, 0, q;\n\t}"
                         : "=r"(all_ok)
                         : "r"((int)ok)
                         : "memory");
            ok = all_ok != 0;
            fence_after();
            if (!ok) break;
            if (d0 == 0 && d1 == done.nt) put_out(done, m, l);
            else join_parts(done, m, l);
            fence_before();
        }
    } else if (warp < 8) {
        if constexpr (E8) asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
        if (warp == 4) {
            // ------------------------------------------------------------ producer
            const int boxes = kKeys / p.box;   // token boxes of a tile; lanes (half of d, box)
            const int b = lane % boxes, h = lane / boxes;
            uint32_t it = 0;
            bool ok = true;
            struct Box {
                int page, tok;   // page -1: it is not needed
            };
            do {
                int t0, t1;
                share_tiles(u, t0, t1);
                if (t0 >= t1) continue;
                const int *pt = p.page_table + (long long)u.s * p.table_stride;
                auto look_up = [&](int t) -> Box {   // this lane's box of tile t
                    const int key = (u.tile0 + t) * kKeys + b * p.box;
                    if (t >= t1 || key >= u.hi || h >= (E8 ? 1 : C::HALVES)) return Box{-1, 0};
                    const int j = p.by_page.div(key);
                    return Box{__ldg(pt + j), p.by_page.mod(key, j) | (int)0x80000000};
                };
                auto load = [&](const Box &x, bool v) -> bool {
                    const bool need = x.tok < 0;
                    int page = x.page;
                    if (need && (page < 0 || page >= p.n_pages)) {
                        raise_error(p.status, DEV_BAD_PAGE);
                        page = p.n_pages;   // outside the pool: zeros
                    }
                    const uint32_t bytes = __popc(__ballot_sync(FULL, need)) * p.box * (E8 ? D : 128);
                    const int st = it % C::LOADS;
                    if (it >= C::LOADS && !wait(E8 ? &raw_empty[st] : &empty[st], (it / C::LOADS - 1) & 1)) return false;
                    if (lane == 0) mbar_arrive_expect_tx(&full[st], bytes);
                    __syncwarp();
                    if (need) {
                        const int tok = x.tok & 0x7fffffff;
                        if constexpr (E8)
                            tma_box(sbase + C::RAW + st * C::RAW_TILE + b * p.box * D, v ? &p.tm_v : &p.tm_k, 0, tok, u.g, page, &full[st]);
                        else
                            tma_box(sbase + C::RING + st * C::TILE + h * C::BLOCK + b * p.box * 128, v ? &p.tm_v : &p.tm_k, h * 64, tok,
                                    u.g, page, &full[st]);
                    }
                    ++it;
                    return true;
                };
                Box now = look_up(t0), next = look_up(t0 + 1);
                ok = load(now, false);
                for (int t = t0; ok && t < t1; ++t) {
                    const Box after = look_up(t + 2);   // (looked up ahead)
                    if (t + 1 < t1) ok = load(next, false);
                    if (ok) ok = load(now, true);
                    now = next;
                    next = after;
                }
            } while (ok && next_unit(u));
            // copies in flight land before the CTA may end, also where this warp issued its last
            // one before another gave up on it (else they have landed, or do while the others work)
            for (uint32_t i = it > (uint32_t)C::LOADS ? it - C::LOADS : 0; i < it; ++i)
                mbar_drain(&full[i % C::LOADS], (i / C::LOADS) & 1);
        } else if (warp == 5) {
            // ------------------------------------------------------------ MMA issuer
            constexpr uint32_t ID_S = idesc(BF, false, kKeys), ID_O = idesc(BF, true, D);
            const uint32_t t_s = uniform(tmem + C::T_S), t_o = uniform(tmem + C::T_O);
            const uint32_t q_lo = uniform(desc_k(sbase));
            uint32_t base = 0;           // ring position of the unit's first tile
            uint32_t n_q = 0, n_p = 0, e = 0, n_pv = 0;   // q and P so far, events, waits for P V
            bool ok = true;
            auto stage_of = [&](uint32_t at) { return sbase + C::RING + (at % C::STAGES) * C::TILE; };
            auto full_wait = [&](uint32_t at) { return reached(landed, kLanded, at + 1); };
            do {
                int t0, t1;
                share_tiles(u, t0, t1);
                if (t0 >= t1) continue;
                const int n = t1 - t0;
                // S of step j into the buffer of its event, its commit
                auto issue_s = [&](int j) {
                    const uint32_t at = base + k_pos(j), turn = uniform((e + j) & 1);
                    const uint32_t kb = uniform(desc_k(stage_of(at)));
                    const uint32_t e_bar = uniform(smem_u32(&ev[turn])), s_bar = uniform(smem_u32(&empty[at % C::STAGES]));
                    if (elect()) {
#pragma unroll
                        for (int c = 0; c < D / 16; ++c) {
                            const uint32_t oq = ((c >> 2) * (kM * 128) + (c & 3) * 32) / 16, ok_ = ((c >> 2) * C::BLOCK + (c & 3) * 32) / 16;
                            if (c == 0) mma_ss<ID_S, false>(t_s + 64 * turn, q_lo + oq, kb + ok_);
                            else mma_ss<ID_S, true>(t_s + 64 * turn, q_lo + oq, kb + ok_);
                        }
                        commit(e_bar);
                        commit(s_bar);
                    }
                    __syncwarp();
                };
                ok = wait(q_full, n_q & 1);
                ++n_q;
                for (int j = 0; ok && j < 2; ++j) {
                    if (j < n) {
                        ok = full_wait(base + k_pos(j));
                        if (!ok) break;
                        fence_after();
                        issue_s(j);
                    } else {   // an event without an S
                        if (elect()) commit(smem_u32(&ev[(e + j) & 1]));
                        __syncwarp();
                    }
                }
                for (int j = 0; ok && j < n; ++j) {
                    const uint32_t vt = base + v_pos(j, n);
                    ok = full_wait(vt);
                    if (!ok) break;
                    ok = reached(p_seq, 4, ++n_p);
                    if (!ok) break;
                    fence_after();
                    const uint32_t b = uniform((e + j) & 1);
                    const uint32_t vb = uniform(desc_mn(stage_of(vt), C::BLOCK));
                    const uint32_t s_bar = uniform(smem_u32(&empty[vt % C::STAGES])), acc = uniform(j > 0);
                    const uint32_t done = uniform(smem_u32(j + 2 < n ? pv_done : &ev[b]));   // (event n or n + 1 behind the last two)
                    if (elect()) {   // O += P V
#pragma unroll
                        for (int c = 0; c < kKeys / 16; ++c)
                            mma_ts<ID_O>(t_o, t_s + 64 * b + 8 * c, vb + c * (16 * 128 / 16), c > 0 ? 1u : acc);
                        commit(done);
                        commit(s_bar);
                    }
                    __syncwarp();
                    if (j + 2 < n) {
                        // S goes over P: only MMAs of one accumulator and shape are sure to run in
                        // the order of their issue
                        ok = wait(pv_done, n_pv & 1);
                        if (!ok) break;
                        ++n_pv;
                        ok = full_wait(base + k_pos(j + 2));
                        if (!ok) break;
                        fence_after();
                        issue_s(j + 2);
                    }
                }
                e += n + 2;
                base += 2 * n;
            } while (ok && next_unit(u));
            // tensor memory is released below only after every MMA issued here is done
            if (elect()) commit(smem_u32(drained));
            __syncwarp();
            if (!mbar_drain(drained, 0)) raise_late(p.status);
        } else if (!E8 && warp == 6) {
            // ------------------------------------------------------------ watcher
            // (the issuer's own look at a barrier after a burst of MMAs waits until the
            // burst has left the queue; a look at a word of shared memory does not)
            uint32_t it = 0;
            bool ok = true;
            do {
                int t0, t1;
                share_tiles(u, t0, t1);
                const int first = u.q.kv - u.q.n;   // the chunk's first key
                auto landed_tile = [&](int t, bool v) -> bool {
                    if (!wait(&full[it % C::STAGES], (it / C::STAGES) & 1, true)) return false;
                    const int key0 = (u.tile0 + t) * kKeys;
                    if (v && key0 + kKeys > first) {   // V's rows that no row of the unit sees
                        uint8_t *y = smem + C::RING + (it % C::STAGES) * C::TILE;
                        const uint32_t lo = seen_by_some(p, u, key0 - first), hi = seen_by_some(p, u, key0 + 32 - first);
                        for (int r = lane >> 3; r < kKeys; r += 4)
                            if (!((r & 32 ? hi : lo) >> (r & 31) & 1))
                                for (int h = 0; h < C::HALVES; ++h)
                                    *reinterpret_cast<uint4 *>(y + h * C::BLOCK + r * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
                        fence_proxy_async_smem();
                    }
                    __syncwarp();
                    ++it;
                    if (lane == 0) st_release(landed, it);
                    return true;
                };
                if (t0 < t1) ok = landed_tile(t0, false);
                for (int t = t0; ok && t < t1; ++t) {
                    if (t + 1 < t1) ok = landed_tile(t + 1, false);
                    if (ok) ok = landed_tile(t, true);
                }
            } while (ok && next_unit(u));
        }
    } else if constexpr (E8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        // ------------------------------------------------------------ widening
        // 16 rows a warp: 8 bytes of a row a lane become one 16-byte piece of f16 (exact) in the
        // layout that the MMA reads (8 lanes write a row's 128 bytes: no bank twice).
        constexpr int L = D / 8, R = 32 / L;   // lanes a row, rows at a time
        const int w = warp - 8, c = lane % L, hi = lane / L;
        uint32_t it = 0;
        bool ok = true;
        do {
            int t0, t1;
            share_tiles(u, t0, t1);
            const int first = u.q.kv - u.q.n;   // the chunk's first key
            auto widen_tile = [&](int t, bool v) -> bool {
                if (!wait(&full[it % C::RAW_STAGES], (it / C::RAW_STAGES) & 1, true)) return false;
                if (it >= C::STAGES && !wait(&empty[it % C::STAGES], (it / C::STAGES - 1) & 1)) return false;
                const int key0 = (u.tile0 + t) * kKeys;
                uint32_t some = ~0u;   // which of this warp's keys any row of the unit sees
                if (v && key0 + kKeys > first) some = seen_by_some(p, u, key0 + 16 * w - first);
                const uint8_t *src = smem + C::RAW + (it % C::RAW_STAGES) * C::RAW_TILE + w * 16 * D + lane * 8;
                uint8_t *dst = smem + C::RING + (it % C::STAGES) * C::TILE + (c >> 3) * C::BLOCK + (w * 16 + hi) * 128;
                uint2 y[16 / R];
#pragma unroll
                for (int x = 0; x < 16 / R; ++x) y[x] = *reinterpret_cast<const uint2 *>(src + x * 256);
                if (some != ~0u) {
#pragma unroll
                    for (int x = 0; x < 16 / R; ++x)
                        if (!(some >> (x * R + hi) & 1)) y[x] = make_uint2(0, 0);
                }
#pragma unroll
                for (int x = 0; x < 16 / R; ++x) {
                    uint4 a;
                    widen4(y[x].x, a.x, a.y);
                    widen4(y[x].y, a.z, a.w);
                    *reinterpret_cast<uint4 *>(dst + x * R * 128 + (((c & 7) ^ ((x * R + hi) & 7)) << 4)) = a;
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    st_release(landed + w, it + 1);
                    mbar_arrive(&raw_empty[it % C::RAW_STAGES]);
                }
                ++it;
                return true;
            };
            if (t0 < t1) ok = widen_tile(t0, false);
            for (int t = t0; ok && t < t1; ++t) {
                if (t + 1 < t1) ok = widen_tile(t + 1, false);
                if (ok) ok = widen_tile(t, true);
            }
        } while (ok && next_unit(u));
    }
    fence_before();
    __syncthreads();
    if (warp == 5) {
        fence_after();
        free_tmem(tmem);
    }
}

template <int D, bool QBF, bool E8>
cudaError_t launch_k(const PagedAttnParams &p, int n_sms, cudaStream_t s) {
    using C = TreeCfg<D, E8>;
    auto kernel = paged_tree_kernel<D, QBF, E8>;
    if (cudaError_t e = ensure_smem_limit(reinterpret_cast<const void *>(kernel), C::BYTES)) return e;
    if constexpr (E8) {
        // the registers that the kernel's warps share out are those it was launched with
        static const int regs = [&]() {
            cudaFuncAttributes a;
            return cudaFuncGetAttributes(&a, reinterpret_cast<const void *>(kernel)) == cudaSuccess ? a.numRegs : 0;
        }();
        if (regs < 80) return cudaErrorLaunchOutOfResources;
    }
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(kCtas * n_sms);
    cfg.blockDim = dim3(C::THREADS);
    cfg.dynamicSmemBytes = C::BYTES;
    cfg.stream = s;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, p);
}

}  // namespace

cudaError_t launch_paged_tree_tiles(const PagedAttnParams &p, int d, int q_type, int cache_type, int n_sms, cudaStream_t s) {
    const bool bf = q_type == KORE_CUDA_BF16, e8 = cache_type == KORE_CUDA_E4M3;
    if (d == 128) {
        if (e8) return bf ? launch_k<128, true, true>(p, n_sms, s) : launch_k<128, false, true>(p, n_sms, s);
        return bf ? launch_k<128, true, false>(p, n_sms, s) : launch_k<128, false, false>(p, n_sms, s);
    }
    if (d == 64) {
        if (e8) return bf ? launch_k<64, true, true>(p, n_sms, s) : launch_k<64, false, true>(p, n_sms, s);
        return bf ? launch_k<64, true, false>(p, n_sms, s) : launch_k<64, false, false>(p, n_sms, s);
    }
    return cudaErrorInvalidValue;
}

}  // namespace kore
