// paged_rows.cu — attention of few query rows a KV head (generation steps,
// short chunks) over a caller-owned paged cache (sm_100a).
//
// out = softmax(scale q K^T) V for up to 16 packed rows (tokens x the group's
// query heads) a work unit: every key and value is read once for the whole
// group. Bound by HBM: 2 d bytes-of-type per key and head against 4 d flops a
// row, far below what the products need on any path, so the products are
// warp-level mma.m16n8k16 (a tcgen05 tile has 128 rows, of which 8 to 16 would
// be used) and everything serves the stream of keys:
//   * one CTA of 8 warps an SM; each warp streams tiles of its own, a fixed
//     8 KB (4 KB for 8 bits and d = 64) of K and V, through a ring of 3 (6)
//     stages that TMA boxes fill straight from the pages (one stage is read while the
//     others land: 128 KB in flight an SM, 160 KB for 8 bits and d = 64;
//     16-byte cp.async by the lanes took as many instructions as the products). No
//     warp waits for another, and the ring runs on over the ends of units.
//   * work in equal shares (paged.cuh): ragged lengths, one long sequence and
//     many short ones all end at the same time. A unit cut between CTAs is
//     joined by the CTA that finishes last, in the CTAs' order, so the sums do not
//     depend on who that is.
//   * a page's rows outside the unit's keys are masked in S and cleared in V, so
//     that whatever the page holds there meets neither product.
//   * the row maximum is moved only when a score passes it by 2^8 (a vote of the
//     warp), so most tiles reduce and rescale nothing; sums and outputs are fp32.
//   * an 8-bit cache is widened to f16 on the way into the fragments (exact: e4m3
//     has fewer exponent and mantissa bits). The order of d in the first
//     product's sum is free, so a thread takes 4 consecutive bytes where the
//     fragment wants (2t, 2t+1, 2t+8, 2t+9), and q the same. bf16 queries over it
//     are scaled by a power of two a row so that they are exact in f16 down
//     to 2^-22 of the row's largest value (smaller ones lose digits: what f16 operands cost).
//   * trees of drafted tokens (TREE): a row sees the context and the tokens of its chunk that its mask
//     names, 32 keys a word; only tiles that reach into the chunk look at the words, and V's rows
//     that none of the unit's rows sees are cleared. 8 tokens on 520 positions, 28/4 heads: 10.8 us.
// Measured: 64 sequences of up to 8192 positions, 16/2 heads of 128, bf16: 55.5 us, 5.46
// TB/s (83 % of the measured copy rate); 12 of up to 32768, 28/4 heads, 8 bits: 49.3 us, 4.77
// TB/s (latency: two warps a scheduler use 36 % of the issue slots, half of them widening);
// one of 513, 28/4 heads: 9.0 us, of which a call on one position takes 5.1. The streaming
// itself runs at HBM's rate; 3.5 us before it (lengths, page table, first copies) and 2
// to 4 us behind it (joining warps and CTAs) are the rest.

#include "paged.cuh"

#include "kore_cuda.h"

#include <type_traits>

namespace kore {
namespace {

constexpr unsigned FULL = 0xffffffffu;
constexpr int kWarps = 8;
constexpr int kRowsU = 16;          // packed rows of a unit
constexpr float kSlack = 8.0f;      // log2 slack before the reference maximum moves

template <int D, int ES>   // ES: bytes of a cached value
struct RowsCfg {
    static constexpr int KT = (D == 128 && ES == 2) ? 16 : 32;   // keys of a warp's tile
    static constexpr int STAGES = (D == 64 && ES == 1) ? 6 : 3;
    static constexpr int ROWB = D * ES;                          // bytes of a key
    static constexpr int HALVES = ROWB == 256 ? 2 : 1;           // boxes are at most 128 bytes wide
    static constexpr int BOXB = ROWB / HALVES;
    static constexpr int HALF = KT * ROWB;                       // K (V) bytes of a stage
    static constexpr int STAGE = 2 * HALF;
    static constexpr int CT = kWarps * KT;                       // keys of a CTA's tile
    static constexpr int CH = ROWB / 16;                         // 16-byte pieces of a key
    static constexpr int RING = kWarps * STAGES * STAGE;
    static constexpr int MERGE = kWarps * 8 * D * 4;             // 8 rows of every warp
    static constexpr int CUM = (kPagedMaxSeqs + 2) * 8;          // shares MERGE's place
    static constexpr int TOP = MERGE > CUM ? MERGE : CUM;
    static constexpr int ML = RING + (TOP + 15) / 16 * 16;
    static constexpr int BARS = ML + 2 * kWarps * kRowsU * 8;
    static constexpr int BYTES = BARS + kWarps * STAGES * 8 + 16;
};

// Byte offset of 16-byte piece c of key r within a stage's half, as the boxes'
// swizzle leaves it (pieces c of 8 consecutive keys lie in distinct banks).
template <int ROWB, int KT>
__device__ __forceinline__ int piece(int r, int c) {
    if constexpr (ROWB == 64) return r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
    else return (c >> 3) * (KT * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a)
                 : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a)
                 : "memory");
}

template <bool BF>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint64_t l2_evict_normal_policy() {
    uint64_t pol;
    asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(pol));
    return pol;
}

// QBF: queries (and output) in bf16, else f16. E4M3: 8-bit cache (products in f16). TREE: the chunks
// are trees of drafted tokens.
template <int D, bool QBF, bool E4M3, bool TREE>
__global__ void __launch_bounds__(kWarps * 32, 1) paged_rows_kernel(const __grid_constant__ PagedAttnParams p) {
    constexpr int ES = E4M3 ? 1 : 2;
    using C = RowsCfg<D, ES>;
    constexpr bool BF = QBF && !E4M3;   // type of the products
    using U = Unit<kRowsU, C::CT, TREE>;
    using qt = typename std::conditional<QBF, __nv_bfloat16, __half>::type;
    extern __shared__ __align__(1024) uint8_t smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int g8 = lane >> 2, t4 = lane & 3;
    float *merge = reinterpret_cast<float *>(smem + C::RING);
    // [warp][row] (max, sum), in two places by turns: a warp may be writing the
    // next unit's while another still reads this one's
    float2 *ml = reinterpret_cast<float2 *>(smem + C::ML);
    int ml_turn = kWarps * kRowsU;
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + C::BARS) + warp * C::STAGES;   // this warp's stages
    int *flag = reinterpret_cast<int *>(smem + C::BARS + kWarps * C::STAGES * 8);
    if (lane < C::STAGES) mbar_init(&full[lane], 1);
    if (lane == 0) {
        prefetch_map(&p.tm_k);
        prefetch_map(&p.tm_v);
    }
    mbar_fence_init();
    __syncwarp();
    grid_dep_wait();
    grid_dep_launch();

    U u;
    long long total, x0, x1;
    int ctas;
    if (!find_share<kRowsU, C::CT, 5, 2, TREE>(p, reinterpret_cast<long long *>(smem + C::RING), u, total, ctas, x0, x1)) return;

    uint8_t *ring = smem + warp * C::STAGES * C::STAGE;

    // q fragments of the unit's rows g8 and g8 + 8, as they are in memory
    uint32_t qf[D / 16][4];
    const uint32_t sign = p.scale < 0.f ? 0x80008000u : 0u;   // goes into q, so that maxima stay maxima
    auto load_q = [&]() {
        const int r0 = u.b * kRowsU + g8, r1 = r0 + 8;
        const bool in0 = g8 < u.rows, in1 = g8 + 8 < u.rows;
        const int i0 = p.by_rep.div(r0), i1 = p.by_rep.div(r1);
        const qt *s0 = static_cast<const qt *>(p.q) + (long long)(u.q.q0 + i0) * p.q_ts +
                       (long long)(u.g * p.rep + r0 - i0 * p.rep) * p.q_hs;
        const qt *s1 = static_cast<const qt *>(p.q) + (long long)(u.q.q0 + i1) * p.q_ts +
                       (long long)(u.g * p.rep + r1 - i1 * p.rep) * p.q_hs;
        auto fill = [&](auto ld) {
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                const int e = E4M3 ? t4 * (D / 4) + 4 * k : 16 * k + 2 * t4;
                const int f = E4M3 ? e + 2 : e + 8;
                qf[k][0] = in0 ? ld(s0 + e) : 0u;
                qf[k][1] = in1 ? ld(s1 + e) : 0u;
                qf[k][2] = in0 ? ld(s0 + f) : 0u;
                qf[k][3] = in1 ? ld(s1 + f) : 0u;
            }
        };
        if (p.q_vec) {
            fill([](const qt *x) { return __ldg(reinterpret_cast<const unsigned int *>(x)); });
        } else {
            fill([](const qt *x) {
                const unsigned short *h = reinterpret_cast<const unsigned short *>(x);
                return (uint32_t)__ldg(h) | ((uint32_t)__ldg(h + 1) << 16);
            });
        }
    };
    load_q();

    // ---- the load side: a unit and a tile that run ahead of the products
    U lu = u;
    bool l_more = true;
    int lt, lt1;   // next tile to load and the end of the share within lu, relative to lu.tile0
    auto share_tiles = [&](const U &a, int &t0, int &t1) {   // tiles of unit a in [x0, x1)
        const long long first = a.u0 + kUnitCost;
        t0 = (int)max(0ll, min((long long)a.nt, x0 - first));
        t1 = (int)max(0ll, min((long long)a.nt, x1 - first));
    };
    auto l_skip = [&]() {   // to the next unit that has a tile left
        while (l_more && lt >= lt1) {
            if (lu.u0 + kUnitCost + lu.nt >= x1 || !lu.next(p)) {
                l_more = false;
                return;
            }
            share_tiles(lu, lt, lt1);
        }
    };
    share_tiles(lu, lt, lt1);
    l_skip();
    // a lane a box: K or V, half of d, group of p.box keys; its page a tile ahead
    const int boxes = 2 * C::HALVES * (C::KT / p.box);
    const int b_half = (lane >> 1) % C::HALVES, b_key = (lane >> 1) / C::HALVES * p.box;
    const TmaDesc *map = (lane & 1) ? &p.tm_v : &p.tm_k;
    const uint32_t b_dst = smem_u32(ring) + (lane & 1) * C::HALF + b_half * (C::KT * 128) + b_key * C::BOXB;
    // a generation step reads every key once; chunks of several units come back to them
    const uint64_t policy = (long long)p.n_tok * p.rep <= (long long)kRowsU * p.n_seq ? l2_evict_first_policy() : l2_evict_normal_policy();
    int b_page, b_tok;   // page -1: the box is not needed
    auto look_up = [&]() {
        b_page = -1;
        if (l_more && lane < boxes) {
            const int key = (lu.tile0 + lt) * C::CT + warp * C::KT + b_key;
            if (key < lu.hi && key + p.box > lu.lo) {
                const int j = p.by_page.div(key);
                b_tok = p.by_page.mod(key, j);
                b_page = __ldg(p.page_table + (long long)lu.s * p.table_stride + j);
                if (b_page < 0 || b_page >= p.n_pages) {
                    raise_error(p.status, DEV_BAD_PAGE);
                    b_page = p.n_pages;   // outside the pool: arrives as zeros
                }
            }
        }
    };
    look_up();
    uint32_t n_loaded = 0, n_taken = 0;   // tiles of this warp
    bool dead = false;                    // a copy did not land in time
    int l_stage = 0;
    auto load_tile = [&]() {
        if (!l_more || dead) return;
        const unsigned need = __ballot_sync(FULL, b_page >= 0);
        if (lane == 0) mbar_arrive_expect_tx(&full[l_stage], __popc(need) * p.box * C::BOXB);
        __syncwarp();
        if (b_page >= 0)
            tma_box(b_dst + l_stage * C::STAGE, map, b_half * (C::BOXB / ES), b_tok, lu.g, b_page, &full[l_stage], policy);
        l_stage = l_stage + 1 == C::STAGES ? 0 : l_stage + 1;
        ++n_loaded;
        ++lt;
        l_skip();
        look_up();
    };
#pragma unroll 1
    for (int i = 0; i < C::STAGES - 1; ++i) load_tile();

    // ---- the products
    int stage = 0;
    for (;;) {
        int t0, t1;
        share_tiles(u, t0, t1);
        if (t0 < t1) {
            const int r0 = u.b * kRowsU + g8, r1 = r0 + 8;   // this thread's packed rows
            const bool in0 = g8 < u.rows, in1 = g8 + 8 < u.rows;
            // keys [lo, hi) of the two rows
            int lo0 = 0, hi0 = 0, lo1 = 0, hi1 = 0;
            // keys that every valid row sees
            int all_lo = 0, all_hi = u.q.kv - u.q.n, t;
            const uint32_t *mask0 = nullptr, *mask1 = nullptr;   // TREE: the two rows'
            if constexpr (TREE) {
                mask0 = p.mask + (long long)(u.q.q0 + p.by_rep.div(in0 ? r0 : u.b * kRowsU)) * p.words;
                mask1 = p.mask + (long long)(u.q.q0 + p.by_rep.div(in1 ? r1 : u.b * kRowsU)) * p.words;
            } else {
                if (in0) key_range<TREE>(p, u.q, r0, r0 + 1, lo0, hi0);
                if (in1) key_range<TREE>(p, u.q, r1, r1 + 1, lo1, hi1);
                key_range<TREE>(p, u.q, u.b * kRowsU, u.b * kRowsU + 1, t, all_hi);
                key_range<TREE>(p, u.q, u.b * kRowsU + u.rows - 1, u.b * kRowsU + u.rows, all_lo, t);
            }

            float qs0 = fabsf(p.scale) * 1.44269504088896340736f, qs1 = qs0;
            {
                if (sign) {
#pragma unroll
                    for (int k = 0; k < D / 16; ++k)
#pragma unroll
                        for (int i = 0; i < 4; ++i) qf[k][i] ^= sign;
                }
                if constexpr (E4M3) {
                    if constexpr (QBF) {
                        // bf16 -> f16 with the row's largest value at 2^7 .. 2^8
                        float m0 = 0.f, m1 = 0.f;
#pragma unroll
                        for (int k = 0; k < D / 16; ++k)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const float a = __uint_as_float(qf[k][i] << 16), b = __uint_as_float(qf[k][i] & 0xffff0000u);
                                const float x = fmaxf(fabsf(a), fabsf(b));
                                if (i & 1) m1 = fmaxf(m1, x);
                                else m0 = fmaxf(m0, x);
                            }
#pragma unroll
                        for (int o = 1; o < 4; o <<= 1) {
                            m0 = fmaxf(m0, __shfl_xor_sync(FULL, m0, o));
                            m1 = fmaxf(m1, __shfl_xor_sync(FULL, m1, o));
                        }
                        const float f0 = f16_shift(m0), f1 = f16_shift(m1);
                        qs0 /= f0;
                        qs1 /= f1;
#pragma unroll
                        for (int k = 0; k < D / 16; ++k)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const float f = (i & 1) ? f1 : f0;
                                const float a = __uint_as_float(qf[k][i] << 16) * f;
                                const float b = __uint_as_float(qf[k][i] & 0xffff0000u) * f;
                                qf[k][i] = pack2<false>(a, b);
                            }
                    }
                    if (p.k_scale) {
                        const float ks = __ldg(p.k_scale + u.g);
                        if (ks < 0.f) {
#pragma unroll
                            for (int k = 0; k < D / 16; ++k)
#pragma unroll
                                for (int i = 0; i < 4; ++i) qf[k][i] ^= 0x80008000u;
                        }
                        qs0 *= fabsf(ks);
                        qs1 *= fabsf(ks);
                    }
                    qs0 = at_least_normal(qs0);
                    qs1 = at_least_normal(qs1);
                }
            }

            float o[D / 8][4];
#pragma unroll
            for (int i = 0; i < D / 8; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) o[i][k] = 0.f;
            float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;   // l: this thread's keys only

            for (int tt = t0; tt < t1; ++tt) {
                if (!dead && !__all_sync(FULL, copy_wait(&full[stage], (n_taken / C::STAGES) & 1, p.wait_ns))) {
                    dead = true;
                    if (lane == 0) raise_late(p.status);
                }
                if (!dead) ++n_taken;
                __syncwarp();   // every lane is done with the tile before this one
                load_tile();    // into its stage
                uint8_t *st = ring + stage * C::STAGE;
                const uint32_t kt = smem_u32(st), vt = kt + C::HALF;
                const int key0 = (u.tile0 + tt) * C::CT + warp * C::KT;
                if (!dead && key0 < u.hi && key0 + C::KT > u.lo) {
                    uint32_t see0 = 0, see1 = 0;   // TREE: the tile's keys that the two rows see
                    uint32_t some = ~0u;           // ... and any row of the unit
                    if (TREE && key0 + C::KT > all_hi) {
                        if (in0) see0 = tree_bits(mask0, p.words, key0 - all_hi, u.q.n);
                        if (in1) see1 = tree_bits(mask1, p.words, key0 - all_hi, u.q.n);
                        some = __reduce_or_sync(FULL, see0 | see1);
                    }
                    if (TREE ? (~some << (32 - C::KT)) != 0 : key0 < u.lo || key0 + C::KT > u.hi) {   // rows outside the unit's keys
                        for (int r = 0; r < C::KT; ++r)
                            if ((TREE ? !(some >> r & 1) : key0 + r < u.lo || key0 + r >= u.hi) && lane < C::CH)
                                *reinterpret_cast<uint4 *>(st + C::HALF + piece<C::ROWB, C::KT>(r, lane)) = make_uint4(0, 0, 0, 0);
                        fence_proxy_async_smem();   // before the stage is filled again
                        __syncwarp();
                    }
                    constexpr int NJ = C::KT / 8;   // groups of 8 keys
                    float s[NJ][4];
#pragma unroll
                    for (int j = 0; j < NJ; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
                    // all of K's fragments, then the products with the groups by turns
                    if constexpr (!E4M3) {
                        uint32_t b[NJ][D / 32][4];
#pragma unroll
                        for (int j = 0; j < NJ; ++j)
#pragma unroll
                            for (int k = 0; k < D / 32; ++k)
                                ldsm4(b[j][k], kt + piece<C::ROWB, C::KT>(8 * j + (lane & 7), 4 * k + (lane >> 3)));
#pragma unroll
                        for (int k = 0; k < D / 32; ++k)
#pragma unroll
                            for (int h = 0; h < 2; ++h)
#pragma unroll
                                for (int j = 0; j < NJ; ++j) mma<BF>(s[j], qf[2 * k + h], b[j][k][2 * h], b[j][k][2 * h + 1]);
                    } else {
                        // thread t4 takes bytes t4*D/4 .. of key g8
                        uint32_t w[NJ][D / 64][4];
#pragma unroll
                        for (int j = 0; j < NJ; ++j)
#pragma unroll
                            for (int h = 0; h < D / 64; ++h)
                                asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                                             : "=r"(w[j][h][0]), "=r"(w[j][h][1]), "=r"(w[j][h][2]), "=r"(w[j][h][3])
                                             : "r"(kt + piece<C::ROWB, C::KT>(8 * j + g8, t4 * (D / 64) + h))
                                             : "memory");
#pragma unroll
                        for (int h = 0; h < D / 64; ++h)
#pragma unroll
                            for (int i = 0; i < 4; ++i)
#pragma unroll
                                for (int j = 0; j < NJ; ++j) {
                                    uint32_t b0, b1;
                                    widen4(w[j][h][i], b0, b1);
                                    mma<false>(s[j], qf[4 * h + i], b0, b1);
                                }
                    }
                    if (key0 < all_lo || key0 + C::KT > all_hi) {
#pragma unroll
                        for (int j = 0; j < NJ; ++j)
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                const int key = key0 + 8 * j + 2 * t4 + i;
                                if (TREE ? !(see0 >> (key - key0) & 1) : key < lo0 || key >= hi0) s[j][i] = -INFINITY;
                                if (TREE ? !(see1 >> (key - key0) & 1) : key < lo1 || key >= hi1) s[j][2 + i] = -INFINITY;
                            }
                    }
                    float x0m = fmaxf(s[0][0], s[0][1]), x1m = fmaxf(s[0][2], s[0][3]);
#pragma unroll
                    for (int j = 1; j < NJ; ++j) {
                        x0m = fmaxf(x0m, fmaxf(s[j][0], s[j][1]));
                        x1m = fmaxf(x1m, fmaxf(s[j][2], s[j][3]));
                    }
                    x0m *= qs0;
                    x1m *= qs1;
                    if (__any_sync(FULL, x0m > m0 + kSlack || x1m > m1 + kSlack)) {
#pragma unroll
                        for (int f = 1; f < 4; f <<= 1) {
                            x0m = fmaxf(x0m, __shfl_xor_sync(FULL, x0m, f));
                            x1m = fmaxf(x1m, __shfl_xor_sync(FULL, x1m, f));
                        }
                        const float n0 = x0m > m0 + kSlack ? x0m : m0, n1 = x1m > m1 + kSlack ? x1m : m1;
                        const float a0 = n0 == m0 ? 1.f : fast_exp2(m0 - n0), a1 = n1 == m1 ? 1.f : fast_exp2(m1 - n1);
                        m0 = n0;
                        m1 = n1;
                        l0 *= a0;
                        l1 *= a1;
#pragma unroll
                        for (int i = 0; i < D / 8; ++i) {
                            o[i][0] *= a0;
                            o[i][1] *= a0;
                            o[i][2] *= a1;
                            o[i][3] *= a1;
                        }
                    }
                    // (the product is rounded as the maximum's was: fused, a score of 2^40 would be
                    // off its own reference by more than exp2 can take)
                    const float z0 = m0 == -INFINITY ? 0.f : kBias<BF> - m0, z1 = m1 == -INFINITY ? 0.f : kBias<BF> - m1;
#pragma unroll
                    for (int j = 0; j < NJ; ++j) {
                        s[j][0] = fast_exp2(__fadd_rn(__fmul_rn(s[j][0], qs0), z0));
                        s[j][1] = fast_exp2(__fadd_rn(__fmul_rn(s[j][1], qs0), z0));
                        s[j][2] = fast_exp2(__fadd_rn(__fmul_rn(s[j][2], qs1), z1));
                        s[j][3] = fast_exp2(__fadd_rn(__fmul_rn(s[j][3], qs1), z1));
                        l0 += s[j][0] + s[j][1];
                        l1 += s[j][2] + s[j][3];
                    }
#pragma unroll
                    for (int jj = 0; jj < C::KT / 16; ++jj) {
                        const uint32_t a[4] = {pack2<BF>(s[2 * jj][0], s[2 * jj][1]), pack2<BF>(s[2 * jj][2], s[2 * jj][3]),
                                               pack2<BF>(s[2 * jj + 1][0], s[2 * jj + 1][1]),
                                               pack2<BF>(s[2 * jj + 1][2], s[2 * jj + 1][3])};
                        // pieces 2c (b0, b1) and 2c + 1 (b2, b3), keys 0-7 and 8-15
                        uint32_t b[C::CH / 2][4];
#pragma unroll
                        for (int c = 0; c < C::CH / 2; ++c)
                            ldsm4t(b[c], vt + piece<C::ROWB, C::KT>(16 * jj + (lane & 15), 2 * c + (lane >> 4)));
#pragma unroll
                        for (int c = 0; c < C::CH / 2; ++c) {
                            if constexpr (!E4M3) {
                                mma<BF>(o[2 * c], a, b[c][0], b[c][1]);
                                mma<BF>(o[2 * c + 1], a, b[c][2], b[c][3]);
                            } else {
                                // b holds, for keys 2t and 2t+1, the bytes d = 2g, 2g+1 of the piece
#pragma unroll
                                for (int h = 0; h < 2; ++h) {
                                    uint32_t w0, w1, y0, y1;
                                    widen4(b[c][2 * h], w0, w1);
                                    widen4(b[c][2 * h + 1], y0, y1);
                                    const int i = 4 * c + 2 * h;
                                    mma<false>(o[i], a, __byte_perm(w0, w1, 0x5410), __byte_perm(y0, y1, 0x5410));
                                    mma<false>(o[i + 1], a, __byte_perm(w0, w1, 0x7632), __byte_perm(y0, y1, 0x7632));
                                }
                            }
                        }
                    }
                }
                stage = stage + 1 == C::STAGES ? 0 : stage + 1;
            }

            // ---- join the warps: rows g8 in one pass, rows g8 + 8 in another
#pragma unroll
            for (int f = 1; f < 4; f <<= 1) {
                l0 += __shfl_xor_sync(FULL, l0, f);
                l1 += __shfl_xor_sync(FULL, l1, f);
            }
            if (t4 == 0) {
                ml[warp * kRowsU + g8] = make_float2(m0, l0);
                ml[warp * kRowsU + g8 + 8] = make_float2(m1, l1);
            }
            const bool whole = t0 == 0 && t1 == u.nt;
            const int c0 = whole ? 0 : share_of(u.u0 + kUnitCost, total, ctas);
            const int c1 = whole ? 0 : share_of(u.u0 + kUnitCost + u.nt - 1, total, ctas);
            // slot: [kRowsU][D] outputs to the row's maximum, then [kRowsU] (max, sum)
            constexpr int SLOT = kRowsU * (D + 2);
            float *slot = p.part + (size_t)(blockIdx.x * 2 + (t0 == 0)) * SLOT;
            constexpr int VW = D / 32;   // values a lane
            const float vs = E4M3 && p.v_scale ? __ldg(p.v_scale + u.g) : 1.f;
            auto write_out = [&](int row, const float (&x)[VW], float M, float L) {   // row of the unit, this lane's values
                const int r = u.b * kRowsU + row, i = p.by_rep.div(r), h = u.g * p.rep + r - i * p.rep;
                const float inv = L > 0.f || L != L ? vs / L : 0.f;
                qt *dst = static_cast<qt *>(p.out) + (long long)(u.q.q0 + i) * p.o_ts + (long long)h * p.o_hs + lane * VW;
                uint32_t w[VW / 2];
#pragma unroll
                for (int k = 0; k < VW / 2; ++k) w[k] = pack2<QBF>(x[2 * k] * inv, x[2 * k + 1] * inv);
                if (p.o_vec) {
                    if constexpr (VW == 4) *reinterpret_cast<uint2 *>(dst) = make_uint2(w[0], w[1]);
                    else *reinterpret_cast<uint32_t *>(dst) = w[0];
                } else {
                    const qt *y = reinterpret_cast<const qt *>(w);
#pragma unroll
                    for (int k = 0; k < VW; ++k) dst[k] = y[k];
                }
                if (p.lse && lane == 0)
                    p.lse[(long long)(u.q.q0 + i) * p.H + h] = log_sum<BF>(M, L);
            };
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                if (half == 1 && u.rows <= 8) break;
                __syncthreads();   // ml is written; merge is free
                const int fr = g8 + 8 * half;
                float M = -INFINITY;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) M = fmaxf(M, ml[w * kRowsU + fr].x);
                const float mine = half ? m1 : m0;
                const float f = mine == -INFINITY ? 0.f : fast_exp2(mine - M);
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    float *dst = merge + (warp * 8 + g8) * D;
                    const int sw = (g8 & 3) * 8;
                    if constexpr (!E4M3) {
                        *reinterpret_cast<float2 *>(dst + ((8 * i + 2 * t4) ^ sw)) =
                            make_float2(o[i][2 * half] * f, o[i][2 * half + 1] * f);
                    } else if ((i & 1) == 0) {   // even and odd d of a piece of 16
                        const int e = 8 * i + 4 * t4;
                        *reinterpret_cast<float4 *>(dst + (e ^ sw)) =
                            make_float4(o[i][2 * half] * f, o[i + 1][2 * half] * f, o[i][2 * half + 1] * f,
                                        o[i + 1][2 * half + 1] * f);
                    }
                }
                __syncthreads();
                // warp w owns row w of these 8
                const int row = warp + 8 * half;
                float Mr = -INFINITY, Lr = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) Mr = fmaxf(Mr, ml[w * kRowsU + row].x);
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    const float2 v = ml[w * kRowsU + row];
                    if (v.x != -INFINITY) Lr = fmaf(v.y, fast_exp2(v.x - Mr), Lr);
                }
                if (row < u.rows) {
                    float x[VW];
#pragma unroll
                    for (int k = 0; k < VW; ++k) x[k] = 0.f;
#pragma unroll
                    for (int w = 0; w < kWarps; ++w) {
                        const float *src = merge + (w * 8 + warp) * D + ((lane * VW) ^ ((warp & 3) * 8));
                        if constexpr (VW == 4) {
                            const float4 v = *reinterpret_cast<const float4 *>(src);
                            x[0] += v.x;
                            x[1] += v.y;
                            x[2] += v.z;
                            x[3] += v.w;
                        } else {
                            const float2 v = *reinterpret_cast<const float2 *>(src);
                            x[0] += v.x;
                            x[1] += v.y;
                        }
                    }
                    if (whole) {
                        write_out(row, x, Mr, Lr);
                    } else {
                        float *dst = slot + row * D + lane * VW;
                        if constexpr (VW == 4) *reinterpret_cast<float4 *>(dst) = make_float4(x[0], x[1], x[2], x[3]);
                        else *reinterpret_cast<float2 *>(dst) = make_float2(x[0], x[1]);
                        if (lane == 0)
                            *reinterpret_cast<float2 *>(slot + kRowsU * D + 2 * row) = make_float2(Mr, Lr);
                    }
                }
            }
            if (!whole) {   // the last of the unit's CTAs joins the parts
                __threadfence();
                __syncthreads();
                if (tid == 0) *flag = atomicAdd(p.counters + c0, 1) == c1 - c0;
                __syncthreads();
                if (*flag) {
                    __threadfence();
                    for (int row = warp; row < u.rows; row += kWarps) {
                        // CTA c0's part is in its second slot, the others' in their first
                        auto part_of = [&](int c) { return p.part + (size_t)(c * 2 + (c == c0)) * SLOT; };
                        float M = -INFINITY;
                        for (int c = c0 + lane; c <= c1; c += 32)
                            M = fmaxf(M, __ldcg(part_of(c) + kRowsU * D + 2 * row));
#pragma unroll
                        for (int f = 16; f; f >>= 1) M = fmaxf(M, __shfl_xor_sync(FULL, M, f));
                        float L = 0.f, x[VW];
#pragma unroll
                        for (int k = 0; k < VW; ++k) x[k] = 0.f;
                        for (int cb = c0; cb <= c1; cb += 32) {
                            float wgt = 0.f, lw = 0.f;   // of CTA cb + lane
                            if (cb + lane <= c1) {
                                const float2 v = __ldcg(reinterpret_cast<const float2 *>(part_of(cb + lane) + kRowsU * D + 2 * row));
                                if (v.x != -INFINITY) {
                                    wgt = fast_exp2(v.x - M);
                                    lw = v.y * wgt;
                                }
                            }
                            const int n = min(32, c1 - cb + 1);
#pragma unroll 8
                            for (int i = 0; i < n; ++i) {
                                const float *src = part_of(cb + i) + row * D + lane * VW;
                                const float w = __shfl_sync(FULL, wgt, i);
                                L += __shfl_sync(FULL, lw, i);
                                if constexpr (VW == 4) {
                                    const float4 v = __ldcg(reinterpret_cast<const float4 *>(src));
                                    x[0] = fmaf(w, v.x, x[0]);
                                    x[1] = fmaf(w, v.y, x[1]);
                                    x[2] = fmaf(w, v.z, x[2]);
                                    x[3] = fmaf(w, v.w, x[3]);
                                } else {
                                    const float2 v = __ldcg(reinterpret_cast<const float2 *>(src));
                                    x[0] = fmaf(w, v.x, x[0]);
                                    x[1] = fmaf(w, v.y, x[1]);
                                }
                            }
                        }
                        write_out(row, x, M, L);
                    }
                    if (tid == 0) p.counters[c0] = 0;   // as the next call wants it
                }
            }
        }
        if (t0 < t1) {
            ml += ml_turn;
            ml_turn = -ml_turn;
        }
        if (u.u0 + kUnitCost + u.nt >= x1 || !u.next(p)) break;
        load_q();
    }
    if (dead)   // copies in flight land before the CTA may end
        for (uint32_t i = n_taken; i < n_loaded; ++i) mbar_drain(&full[i % C::STAGES], (i / C::STAGES) & 1);
}

template <int D, bool QBF, bool E4M3, bool TREE>
cudaError_t launch_t(const PagedAttnParams &p, int n_ctas, cudaStream_t s) {
    using C = RowsCfg<D, E4M3 ? 1 : 2>;
    auto kernel = paged_rows_kernel<D, QBF, E4M3, TREE>;
    static_assert(C::BYTES <= 232448, "shared memory of an SM");
    if (cudaError_t e = ensure_smem_limit(reinterpret_cast<const void *>(kernel), C::BYTES)) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(n_ctas);
    cfg.blockDim = dim3(kWarps * 32);
    cfg.dynamicSmemBytes = C::BYTES;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <int D, bool QBF, bool E4M3>
cudaError_t launch_k(const PagedAttnParams &p, int n_ctas, cudaStream_t s) {
    return p.mask ? launch_t<D, QBF, E4M3, true>(p, n_ctas, s) : launch_t<D, QBF, E4M3, false>(p, n_ctas, s);
}

}  // namespace

cudaError_t launch_paged_rows(const PagedAttnParams &p, int d, int q_type, int cache_type, int n_ctas, cudaStream_t s) {
    const bool bf = q_type == KORE_CUDA_BF16, e = cache_type == KORE_CUDA_E4M3;
    if (d == 128) {
        if (e) return bf ? launch_k<128, true, true>(p, n_ctas, s) : launch_k<128, false, true>(p, n_ctas, s);
        return bf ? launch_k<128, true, false>(p, n_ctas, s) : launch_k<128, false, false>(p, n_ctas, s);
    }
    if (d == 64) {
        if (e) return bf ? launch_k<64, true, true>(p, n_ctas, s) : launch_k<64, false, true>(p, n_ctas, s);
        return bf ? launch_k<64, true, false>(p, n_ctas, s) : launch_k<64, false, false>(p, n_ctas, s);
    }
    return cudaErrorInvalidValue;
}

}  // namespace kore
