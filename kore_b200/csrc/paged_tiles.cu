// paged_tiles.cu — attention of many query rows a KV head (prompt chunks) over a
// caller-owned paged cache of 16 bits, on the 5th-generation tensor cores
// (tcgen05, accumulators in tensor memory), sm_100a.
//
// out = softmax(scale q K^T) V for units of 256 packed rows (tokens x the group's
// query heads), as two tiles of 128 rows that take turns: while the softmax of
// one tile runs, the tensor cores work on the other's products. Bound by the tensor
// cores (4 d flops a pair of row and key) and, close behind, by the exponentials.
//   warps 0-3, 4-7  softmax of tile 0, tile 1: a thread owns a row. S from tensor
//                   memory, mask, online softmax (the reference maximum moves only when
//                   a score passes it by 2^8; O in tensor memory is rescaled then), P in
//                   16 bits over S (the A operand of the second product), sums in fp32.
//                   Prologue: its q row into shared memory, ahead of the last unit's
//                   epilogue, so that the next unit's first products overlap it.
//   warp 8          producer: K and V tiles of 128 keys by TMA straight from the pages
//                   (one box of 16 to 128 tokens a page and half of d, a lane each; a
//                   page outside the pool arrives as zeros), through a ring.
//   warp 9          issues the MMAs: S_i = Q_i K_j^T, O_i += P_i V_j, alternating i. V is
//                   read as it lies in the page (keys x d, the MN-major operand), so
//                   nothing is transposed. In a unit's boundary tiles this warp first clears
//                   the rows of V outside its keys: 0 * NaN must not reach an output.
// Work in equal shares (paged.cuh). The parts of a unit cut between CTAs are joined in
// a binary tree over the CTAs: the second of two neighbours to finish joins both, so that
// no CTA waits and no CTA joins more than log2 of the parts; a joint is symmetric in
// its two sides, so the bits do not depend on who is second.
// Every wait is bounded; tensor memory is always released.

#include "paged.cuh"

#include "kore_cuda.h"

#include <type_traits>

namespace kore {
namespace {

constexpr unsigned FULL = 0xffffffffu;
constexpr int kM = 128;             // rows of a tile
constexpr int kUnitRows = 2 * kM;
constexpr int kKeys = 128;          // keys of a tile
constexpr float kSlack = 8.0f;      // log2 slack before the reference maximum moves
// 12 warps: two warpgroups of softmax and one of the rest. They start with 168
// registers a thread (64512 in all) and move 80 a thread from the last to 40 more for
// each of the first two: a softmax thread holds a row of 128 scores.
constexpr int kThreads = 384;
constexpr int kRegsSoftmax = 208, kRegsRest = 88;
static_assert((2 * kRegsSoftmax + kRegsRest) * 128 <= 168 * kThreads, "registers at launch");
static_assert(kUnitRows == kPagedRowsMax, "workspace slots");

template <int D>
struct TilesCfg {
    static constexpr int HALVES = D / 64;                    // 128-byte wide column blocks
    static constexpr uint32_t BLOCK = kKeys * 128;           // bytes of one such block of a tile
    static constexpr uint32_t TILE = HALVES * BLOCK;         // K or V tile
    static constexpr int STAGES = D == 128 ? 4 : 8;
    static constexpr uint32_t RING = 2 * TILE;               // behind q: [2][HALVES][kM rows][128 B]
    static constexpr uint32_t BARS = RING + STAGES * TILE;
    static constexpr uint32_t BYTES = BARS + 512 + 1024;     // barriers, alignment
    static constexpr uint32_t T_S = 0, T_O = 256;            // tensor memory: S/P of tile i at 128 i, O at T_O + D i
    static_assert(BYTES <= 232448, "shared memory of an SM");
    static_assert(STAGES * TILE >= (kPagedMaxSeqs + 2) * 8, "the sums' place");
};

// ---------------------------------------------------------------- tcgen05

__device__ __forceinline__ uint32_t sw128(int r, int c) {   // 16-byte piece c of 128-byte row r
    return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4));
}
// Shared-memory matrix descriptors (128-byte swizzle, Blackwell version 1).
// K-major: groups of 8 rows 1024 bytes apart. MN-major: blocks of 64 columns
// `lbo` bytes apart, groups of 8 rows (keys) 1024 bytes apart.
__device__ __forceinline__ uint64_t desc_k(uint32_t a) {
    return (uint64_t)((a >> 4) & 0x3FFF) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
           ((uint64_t)2 << 61);
}
__device__ __forceinline__ uint64_t desc_mn(uint32_t a, uint32_t lbo) {
    return (uint64_t)((a >> 4) & 0x3FFF) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// f16 (0) or bf16 (1) operands of one type, fp32 sums; B K-major or MN-major
__host__ __device__ constexpr uint32_t idesc(bool bf, bool b_mn, int N) {
    return (1u << 4) | ((bf ? 1u : 0u) << 7) | ((bf ? 1u : 0u) << 10) | ((b_mn ? 1u : 0u) << 16) |
           ((uint32_t)(N >> 3) << 17) | ((uint32_t)(kM >> 4) << 24);
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(acc)
                 : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(id), "r"(acc)
                 : "memory");
}
__device__ __forceinline__ void commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}
// 32 columns of this thread's row
__device__ __forceinline__ void ld32(uint32_t a, uint32_t *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(a));
}
__device__ __forceinline__ void st32(uint32_t a, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(a),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tma_box(uint32_t dst, const TmaDesc *map, int x, int tok, int g, int page, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
        ::"r"(dst), "l"(map), "r"(x), "r"(tok), "r"(g), "r"(page), "r"(smem_u32(bar))
        : "memory");
}

// two fp32 at once
__device__ __forceinline__ unsigned long long pk2(float a, float b) {
    unsigned long long u;
    asm("mov.b64 %0, {%1, %2};" : "=l"(u) : "f"(a), "f"(b));
    return u;
}
__device__ __forceinline__ void upk2(unsigned long long u, float &a, float &b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(u));
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ unsigned long long mul2(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
template <bool BF>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (BF) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&v);
    } else {
        const __half2 v = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&v);
    }
}

// ---------------------------------------------------------------- parts of a cut unit
//
// CTA c has two slots: slot 0 for the unit it goes on with, slot 1 for the one
// it begins. A slot: O to the row's maximum [D/4][256 rows] float4 (a warp's rows
// stand side by side), then maxima [256] and sums [256].

template <int D>
constexpr size_t kSlot = (size_t)kUnitRows * (D + 2);

template <int D, bool BF>
__global__ void __launch_bounds__(kThreads, 1) paged_tiles_kernel(const __grid_constant__ PagedAttnParams p) {
    using C = TilesCfg<D>;
    using U = Unit<kUnitRows, kKeys>;
    using qt = typename std::conditional<BF, __nv_bfloat16, __half>::type;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t sbase = smem_u32(smem);
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + C::BARS);
    uint64_t *full = bars;                  // [STAGES] a tile has landed
    uint64_t *empty = bars + 8;             // [STAGES] its MMAs are done
    uint64_t *q_full = bars + 16;           // [2] tile i's q rows are in shared memory (4 warps)
    uint64_t *s_full = bars + 18;           // [2] S_i is formed (and every MMA before it done)
    uint64_t *p_full = bars + 20;           // [2] P_i is written, O_i rescaled (4 warps)
    uint64_t *o_full = bars + 22;           // [2] O_i is complete
    uint64_t *drained = bars + 24;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 25);
    int *abort_flag = reinterpret_cast<int *>(bars + 26);
    int *join = reinterpret_cast<int *>(bars + 27);   // [2] a tile's joint: whether it is the second
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 256) {
        prefetch_map(&p.tm_k);
        prefetch_map(&p.tm_v);
    }
    __syncwarp();
    grid_dep_wait();
    grid_dep_launch();
    U u;
    long long total, x0, x1;
    int ctas;
    if (!find_share<kUnitRows, kKeys, 4, 3>(p, reinterpret_cast<long long *>(smem + C::RING), u, total, ctas, x0, x1)) return;

    if (threadIdx.x == 0) {
        for (int i = 0; i < C::STAGES; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&q_full[i], 4);
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);
            mbar_init(&o_full[i], 1);
        }
        mbar_init(drained, 1);
        *abort_flag = 0;
        mbar_fence_init();
    }
    fence_proxy_async_smem();   // the sums stood where the ring's copies will land
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_slot;

    // bounded, by whole warps, with one answer for the warp
    auto wait = [&](uint64_t *bar, uint32_t parity) -> bool {
        bool got = mbar_try_wait(bar, parity);
        if (__all_sync(FULL, got)) return true;
        if (!got && !*reinterpret_cast<volatile int *>(abort_flag)) {
            got = mbar_wait(bar, parity, p.status, DEV_WAIT_FULL_TIMEOUT);
            if (!got) *reinterpret_cast<volatile int *>(abort_flag) = 1;
        }
        return __all_sync(FULL, got);
    };
    auto share_tiles = [&](const U &a, int &t0, int &t1) {   // tiles of unit a in [x0, x1)
        const long long first = a.u0 + kUnitCost;
        t0 = (int)max(0ll, min((long long)a.nt, x0 - first));
        t1 = (int)max(0ll, min((long long)a.nt, x1 - first));
    };
    auto next_unit = [&](U &a) -> bool { return a.u0 + kUnitCost + a.nt < x1 && a.next(p); };

    if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsRest));
    if (warp == 8) {
        // ------------------------------------------------------------ producer
        const int boxes = kKeys / p.box;   // token boxes of a tile; lanes (half of d, box)
        uint32_t it = 0;
        bool ok = true;
        do {
            int t0, t1;
            share_tiles(u, t0, t1);
            const int *pt = p.page_table + (long long)u.s * p.table_stride;
            for (int t = t0; ok && t < t1; ++t) {
                const int key0 = (u.tile0 + t) * kKeys;
                // this lane's box: token box lane % boxes (16 at most)
                const int b = lane % boxes, key = key0 + b * p.box;
                const bool need = key < u.hi && key + p.box > u.lo;
                int page = p.n_pages;   // outside the pool: zeros
                if (need) {
                    page = __ldg(pt + p.by_page.div(key));
                    if (page < 0 || page >= p.n_pages) {
                        raise_error(p.status, DEV_BAD_PAGE);
                        page = p.n_pages;
                    }
                }
                const int tok = p.by_page.mod(key, p.by_page.div(key));
                const unsigned mask = __ballot_sync(FULL, need && lane < boxes);
                const uint32_t bytes = __popc(mask) * p.box * 128 * C::HALVES;
#pragma unroll 1
                for (int kv = 0; kv < 2; ++kv, ++it) {
                    const int st = it % C::STAGES;
                    if (it >= C::STAGES && !wait(&empty[st], (it / C::STAGES - 1) & 1)) {
                        ok = false;
                        break;
                    }
                    if (lane == 0) mbar_arrive_expect_tx(&full[st], bytes);
                    __syncwarp();
                    const uint32_t dst = sbase + C::RING + st * C::TILE;
                    for (int i = lane; i < boxes * C::HALVES; i += 32) {   // boxes <= 8 unless box == 16 ... 32 lanes at most
                        const int h = i / boxes;
                        if (need)
                            tma_box(dst + h * C::BLOCK + b * p.box * 128, kv ? &p.tm_v : &p.tm_k, h * 64, tok, u.g, page,
                                    &full[st]);
                    }
                }
            }
        } while (ok && next_unit(u));
        if (!ok)   // copies in flight land before the CTA may end
            for (uint32_t i = it > (uint32_t)C::STAGES ? it - C::STAGES : 0; i < it; ++i)
                mbar_drain(&full[i % C::STAGES], (i / C::STAGES) & 1);
    } else if (warp == 9) {
        // ------------------------------------------------------------ MMA issuer
        constexpr uint32_t ID_S = idesc(BF, false, kKeys), ID_O = idesc(BF, true, D);
        uint32_t it = 0;             // ring position
        uint32_t n_q[2] = {0, 0}, n_p[2] = {0, 0};   // q and P tiles so far
        bool ok = true;
        auto issue_s = [&](int i, uint32_t at) {   // S_i = Q_i K^T
            if (lane == 0) {
                const uint64_t a = desc_k(sbase + i * C::TILE), b = desc_k(sbase + C::RING + (at % C::STAGES) * C::TILE);
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    const uint32_t o = ((k >> 2) * C::BLOCK + (k & 3) * 32) / 16;
                    mma_ss(tmem + C::T_S + 128 * i, a + o, b + o, ID_S, k > 0);
                }
                commit(&s_full[i]);
            }
            __syncwarp();
        };
        auto issue_pv = [&](int i, uint32_t at, bool first) {   // O_i += P_i V
            if (lane == 0) {
                const uint64_t b = desc_mn(sbase + C::RING + (at % C::STAGES) * C::TILE, C::BLOCK);
#pragma unroll
                for (int k = 0; k < kKeys / 16; ++k)
                    mma_ts(tmem + C::T_O + D * i, tmem + C::T_S + 128 * i + 8 * k, b + k * (16 * 128 / 16), ID_O, !first || k > 0);
            }
            __syncwarp();
        };
        auto release = [&](uint32_t at) {
            if (lane == 0) commit(&empty[at % C::STAGES]);
            __syncwarp();
        };
        auto full_wait = [&](uint32_t at) { return wait(&full[at % C::STAGES], (at / C::STAGES) & 1); };
        // clears the rows of a V tile outside the unit's keys
        auto clear_v = [&](const U &a, int t, uint32_t at) {
            const int key0 = (a.tile0 + t) * kKeys;
            if (key0 >= a.lo && key0 + kKeys <= a.hi) return;
            uint8_t *v = smem + C::RING + (at % C::STAGES) * C::TILE;
            for (int r = lane >> 3; r < kKeys; r += 4)
                if (key0 + r < a.lo || key0 + r >= a.hi)
                    for (int h = 0; h < C::HALVES; ++h)
                        *reinterpret_cast<uint4 *>(v + h * C::BLOCK + r * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
            fence_proxy_async_smem();
            __syncwarp();
        };
        do {
            int t0, t1;
            share_tiles(u, t0, t1);
            if (t0 >= t1) continue;
            const int ni = u.rows > kM ? 2 : 1;
            // first S of both tiles
            for (int i = 0; ok && i < ni; ++i) {
                ok = wait(&q_full[i], n_q[i] & 1) && full_wait(it);
                if (!ok) break;
                ++n_q[i];
                fence_after();
                issue_s(i, it);
            }
            if (ok) release(it);
            for (int t = t0; ok && t < t1; ++t) {
                const uint32_t vt = it + 1, kt = it + 2;
                for (int i = 0; i < ni; ++i) {
                    ok = full_wait(vt);
                    if (!ok) break;
                    if (i == 0) clear_v(u, t, vt);
                    ok = wait(&p_full[i], n_p[i] & 1);
                    if (!ok) break;
                    ++n_p[i];
                    fence_after();
                    issue_pv(i, vt, t == t0);
                    if (t + 1 < t1) {
                        ok = full_wait(kt);
                        if (!ok) break;
                        issue_s(i, kt);
                    } else {
                        if (lane == 0) commit(&o_full[i]);
                        __syncwarp();
                    }
                }
                if (!ok) break;
                release(vt);
                if (t + 1 < t1) release(kt);
                it += 2;
            }
        } while (ok && next_unit(u));
        // tensor memory is released below only after every MMA issued here is done
        if (lane == 0) commit(drained);
        __syncwarp();
        mbar_wait(drained, 0, p.status, DEV_WAIT_FULL_TIMEOUT);
    }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
        // ------------------------------------------------------------ softmax
        const int i = warp >> 2, r = threadIdx.x & 127;   // tile, row
        const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + C::T_S + 128 * i + lane_off, to = tmem + C::T_O + D * i + lane_off;
        uint32_t n_s = 0, n_o = 0;
        bool ok = true;
        const uint32_t sign = p.scale < 0.f ? 0x80008000u : 0u;   // goes into q, so that maxima stay maxima
        const float qs = fabsf(p.scale) * 1.44269504088896340736f;
        // this thread's q row of unit a into shared memory
        auto load_q = [&](const U &a) {
            if (i * kM >= a.rows) return;
            const int pr = a.b * kUnitRows + i * kM + r;   // packed row
            const bool in = i * kM + r < a.rows;
            const int tok = p.by_rep.div(pr);
            const qt *src = static_cast<const qt *>(p.q) + (long long)(a.q.q0 + tok) * p.q_ts +
                            (long long)(a.g * p.rep + pr - tok * p.rep) * p.q_hs;
            uint8_t *dst = smem + i * C::TILE;
            uint4 v[D / 8];   // all of the row on its way at once
            if (p.q_vec) {
#pragma unroll
                for (int c = 0; c < D / 8; ++c)
                    v[c] = in ? __ldg(reinterpret_cast<const uint4 *>(src) + c) : make_uint4(0, 0, 0, 0);
            } else {
#pragma unroll
                for (int c = 0; c < D / 8; ++c) {
                    const unsigned short *h = reinterpret_cast<const unsigned short *>(src) + 8 * c;
                    uint32_t w[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        w[k] = in ? (uint32_t)__ldg(h + 2 * k) | ((uint32_t)__ldg(h + 2 * k + 1) << 16) : 0u;
                    v[c] = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
#pragma unroll
            for (int c = 0; c < D / 8; ++c) {
                v[c].x ^= sign;
                v[c].y ^= sign;
                v[c].z ^= sign;
                v[c].w ^= sign;
                *reinterpret_cast<uint4 *>(dst + (c >> 3) * C::BLOCK + sw128(r, c & 7)) = v[c];
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full[i]);
        };
        // the next unit with a tile in this share, from a on
        auto skip_empty = [&](U &a, int &t0, int &t1) -> bool {
            for (;;) {
                share_tiles(a, t0, t1);
                if (t0 < t1) return true;
                if (!next_unit(a)) return false;
            }
        };
        int t0, t1;
        bool more = skip_empty(u, t0, t1);
        if (more) load_q(u);
        while (more && ok) {
            const bool mine = i * kM < u.rows;            // the tile has rows
            const bool in = i * kM + r < u.rows;
            const int pr = u.b * kUnitRows + i * kM + r;
            int lo = 0, hi = 0, all_lo = 0, all_hi = 0;
            if (mine) {
                if (in) key_range(p, u.q, pr, pr + 1, lo, hi);
                const int b0 = u.b * kUnitRows + i * kM, b1 = u.b * kUnitRows + min(u.rows, (i + 1) * kM);
                int x;
                key_range(p, u.q, b0, b0 + 1, x, all_hi);
                key_range(p, u.q, b1 - 1, b1, all_lo, x);
            }
            float m = -INFINITY, l = 0.f;
            if (mine) {
                for (int t = t0; t < t1; ++t) {
                    if (!wait(&s_full[i], n_s & 1)) {
                        ok = false;
                        break;
                    }
                    ++n_s;
                    fence_after();
                    float s[128];
#pragma unroll
                    for (int c = 0; c < 4; ++c) ld32(ts + 32 * c, reinterpret_cast<uint32_t *>(s) + 32 * c);
                    wait_ld();
                    const int key0 = (u.tile0 + t) * kKeys;
                    if (key0 < all_lo || key0 + kKeys > all_hi) {
#pragma unroll
                        for (int k = 0; k < 128; ++k)
                            if (key0 + k < lo || key0 + k >= hi) s[k] = -INFINITY;
                    }
                    float mx[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) mx[k] = s[k];
#pragma unroll
                    for (int k = 8; k < 128; k += 2) mx[(k >> 1) & 7] = max3(mx[(k >> 1) & 7], s[k], s[k + 1]);
                    const float top = max3(max3(mx[0], mx[1], mx[2]), max3(mx[3], mx[4], mx[5]), fmaxf(mx[6], mx[7])) * qs;
                    const bool need = top > m + kSlack;
                    if (__any_sync(FULL, need)) {
                        const float a = need ? fast_exp2(m - top) : 1.f;
                        if (need) {
                            m = top;
                            l *= a;
                        }
                        if (t > t0) {
                            const unsigned long long aa = pk2(a, a);
#pragma unroll 1
                            for (int c = 0; c < D; c += 32) {
                                float o[32];
                                ld32(to + c, reinterpret_cast<uint32_t *>(o));
                                wait_ld();
#pragma unroll
                                for (int k = 0; k < 32; k += 2) upk2(mul2(pk2(o[k], o[k + 1]), aa), o[k], o[k + 1]);
                                st32(to + c, reinterpret_cast<const uint32_t *>(o));
                            }
                        }
                    }
                    const float z = m == -INFINITY ? 0.f : -m;
                    const unsigned long long qq = pk2(qs, qs), zz = pk2(z, z);
                    unsigned long long acc[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t w[32];
#pragma unroll
                        for (int k = 0; k < 32; ++k) {
                            const int e = 64 * h + 2 * k;
                            float a, b;
                            upk2(fma2(pk2(s[e], s[e + 1]), qq, zz), a, b);
                            a = fast_exp2(a);
                            b = fast_exp2(b);
                            acc[k & 3] = add2(acc[k & 3], pk2(a, b));
                            w[k] = pack2<BF>(a, b);
                        }
                        st32(ts + 32 * h, w);
                    }
                    float x, y;
                    upk2(add2(add2(acc[0], acc[1]), add2(acc[2], acc[3])), x, y);
                    l += x + y;
                    wait_st();
                    fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&p_full[i]);
                }
            }
            // the next unit's q, so that its products may start during the epilogue
            // (every S of this unit is formed, so its q has been read)
            const U done = u;
            const int d0 = t0, d1 = t1;
            if (ok) {
                more = next_unit(u) && skip_empty(u, t0, t1);
                if (more) load_q(u);
            }
            if (!ok || !mine) continue;
            if (!wait(&o_full[i], n_o & 1)) {
                ok = false;
                break;
            }
            ++n_o;
            fence_after();
            // a part of a cut unit: up the tree of its CTAs as far as this one is the
            // second to finish
            bool last = d0 == 0 && d1 == done.nt;
            if (!last) {
                const int c0 = share_of(done.u0 + kUnitCost, total, ctas);
                const int n = share_of(done.u0 + kUnitCost + done.nt - 1, total, ctas) - c0 + 1;   // parts
                const int row = i * kM + r, one = 1 << (16 * i);   // the tiles count apart, in the halves of a counter
                auto slot_of = [&](int k) { return p.part + (size_t)((c0 + k) * 2 + (k == 0)) * kSlot<D>; };
                const int me = blockIdx.x - c0;
                last = true;
                for (int j = 1; (1 << (j - 1)) < n; ++j) {
                    const int left = me >> j << j, right = left + (1 << (j - 1));   // first parts of the two sides
                    if (right >= n) continue;                                      // no right side
                    int *counter = p.counters + c0 + right;
                    const bool is_left = me < right;
                    // has the other side finished? then this one need not be written
                    if (r == 0) join[i] = (atomicAdd(counter, 0) >> (16 * i)) & 0xffff;
                    asm volatile("bar.sync %0, 128;" ::"r"(1 + i) : "memory");
                    int second = *reinterpret_cast<volatile int *>(&join[i]);
                    asm volatile("bar.sync %0, 128;" ::"r"(1 + i) : "memory");
                    if (!second) {
                        float *slot = slot_of(is_left ? left : right);
#pragma unroll 1
                        for (int c = 0; c < D; c += 32) {
                            float o[32];
                            ld32(to + c, reinterpret_cast<uint32_t *>(o));
                            wait_ld();
#pragma unroll
                            for (int k = 0; k < 32; k += 4)
                                *(reinterpret_cast<float4 *>(slot) + ((c + k) / 4) * kUnitRows + row) =
                                    make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
                        }
                        slot[kUnitRows * D + row] = m;
                        slot[kUnitRows * (D + 1) + row] = l;
                        __threadfence();
                        asm volatile("bar.sync %0, 128;" ::"r"(1 + i) : "memory");
                        if (r == 0) join[i] = (atomicAdd(counter, one) >> (16 * i)) & 0xffff;
                        asm volatile("bar.sync %0, 128;" ::"r"(1 + i) : "memory");
                        second = *reinterpret_cast<volatile int *>(&join[i]);
                        asm volatile("bar.sync %0, 128;" ::"r"(1 + i) : "memory");
                        if (!second) {   // the other side goes on
                            last = false;
                            break;
                        }
                        if (r == 0) atomicAdd(counter, -one);   // its own count; below the other's
                    }
                    if (r == 0) atomicAdd(counter, -one);   // as the next call wants it
                    __threadfence();
                    const float *slot = slot_of(is_left ? right : left);
                    const float m2 = __ldcg(slot + kUnitRows * D + row), l2 = __ldcg(slot + kUnitRows * (D + 1) + row);
                    const float M = fmaxf(m, m2);
                    const float a = m == -INFINITY ? 0.f : fast_exp2(m - M), b = m2 == -INFINITY ? 0.f : fast_exp2(m2 - M);
                    m = M;
                    l = __fadd_rn(__fmul_rn(a, l), __fmul_rn(b, l2));
#pragma unroll 1
                    for (int c = 0; c < D; c += 32) {
                        float o[32];
                        float4 x[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            x[k] = __ldcg(reinterpret_cast<const float4 *>(slot) + (c / 4 + k) * kUnitRows + row);
                        ld32(to + c, reinterpret_cast<uint32_t *>(o));
                        wait_ld();
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            o[4 * k] = __fadd_rn(__fmul_rn(a, o[4 * k]), __fmul_rn(b, x[k].x));
                            o[4 * k + 1] = __fadd_rn(__fmul_rn(a, o[4 * k + 1]), __fmul_rn(b, x[k].y));
                            o[4 * k + 2] = __fadd_rn(__fmul_rn(a, o[4 * k + 2]), __fmul_rn(b, x[k].z));
                            o[4 * k + 3] = __fadd_rn(__fmul_rn(a, o[4 * k + 3]), __fmul_rn(b, x[k].w));
                        }
                        st32(to + c, reinterpret_cast<const uint32_t *>(o));
                    }
                    wait_st();
                }
            }
            if (last) {
                const int tok = p.by_rep.div(pr), h = done.g * p.rep + pr - tok * p.rep;
                const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
                qt *dst = static_cast<qt *>(p.out) + (long long)(done.q.q0 + tok) * p.o_ts + (long long)h * p.o_hs;
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                    float o[32];
                    ld32(to + c, reinterpret_cast<uint32_t *>(o));
                    wait_ld();
                    uint32_t w[16];
#pragma unroll
                    for (int k = 0; k < 16; ++k)
                        // (a row without keys: O is 0 * V of cleared rows)
                        w[k] = pack2<BF>(o[2 * k] * inv, o[2 * k + 1] * inv);
                    if (in) {
                        if (p.o_vec) {
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                *(reinterpret_cast<uint4 *>(dst + c) + k) = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
                        } else {
                            unsigned short *y = reinterpret_cast<unsigned short *>(dst + c);
#pragma unroll
                            for (int k = 0; k < 16; ++k) {
                                y[2 * k] = (unsigned short)(w[k] & 0xffffu);
                                y[2 * k + 1] = (unsigned short)(w[k] >> 16);
                            }
                        }
                    }
                }
                if (p.lse && in)
                    p.lse[(long long)(done.q.q0 + tok) * p.H + h] = l > 0.f || l != l ? m * 0.69314718055994530942f + logf(l) : -INFINITY;
            }
            fence_before();
        }
    }
    fence_before();
    __syncthreads();
    if (warp == 9) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

template <int D, bool BF>
cudaError_t launch_k(const PagedAttnParams &p, int n_ctas, cudaStream_t s) {
    using C = TilesCfg<D>;
    if (cudaError_t e = ensure_smem_limit(reinterpret_cast<const void *>(paged_tiles_kernel<D, BF>), C::BYTES)) return e;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(n_ctas);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = C::BYTES;
    cfg.stream = s;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, paged_tiles_kernel<D, BF>, p);
}

}  // namespace

cudaError_t launch_paged_tiles(const PagedAttnParams &p, int d, int type, int n_ctas, cudaStream_t s) {
    const bool bf = type == KORE_CUDA_BF16;
    if (d == 128) return bf ? launch_k<128, true>(p, n_ctas, s) : launch_k<128, false>(p, n_ctas, s);
    if (d == 64) return bf ? launch_k<64, true>(p, n_ctas, s) : launch_k<64, false>(p, n_ctas, s);
    return cudaErrorInvalidValue;
}

}  // namespace kore
