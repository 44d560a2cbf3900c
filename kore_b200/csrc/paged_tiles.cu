// paged_tiles.cu — attention of many query rows a KV head (prompt chunks) over a
// caller-owned paged cache of 16 or 8 bits, on the 5th-generation tensor cores
// (tcgen05, accumulators in tensor memory), sm_100a.
//
// out = softmax(scale q K^T) V for units of 256 packed rows (tokens x the group's
// query heads), as two tiles of 128 rows that share the keys' way through shared
// memory and are otherwise on their own. Bound by the tensor cores (4 d flops a pair
// of row and key) and, close behind, by the exponentials.
//   warps 0-3, 4-7  softmax of tile 0, tile 1: a thread owns a row. Per step of 64 keys:
//                   S from tensor memory, mask, online softmax (the reference maximum
//                   moves only when a score passes it by 2^8; O in tensor memory is
//                   rescaled then), P in 16 bits over S (the A operand of the second
//                   product), sums in fp32. Between units: the next unit's q into shared
//                   memory, then this one's outputs, so that the next products overlap them.
//   warp 8          producer: K and V tiles of 128 keys by TMA straight from the pages
//                   (one box of 16 to 128 tokens a page and half of d, a lane each; a
//                   page outside the pool arrives as zeros), through a ring.
//   warps 9, 10     issue the MMAs of tile 0, tile 1: for each step j O += P_j V_j, then
//                   S_{j+2} = Q K_{j+2}^T into the buffer that P_j leaves, so that the
//                   softmax never waits for the S after its P. V is read as it lies in the
//                   page (keys x d, the MN-major operand), so nothing is transposed.
//   warp 11         watches the ring for the issuers, and clears the rows of V outside the
//                   unit's keys in its boundary tiles: 0 * NaN must not reach an output.
//   warps 12-15     (8-bit caches, in warp 11's place) widen the tiles to f16 (exact) from a
//                   ring of their own into the one that the MMAs read.
// Measured (2048 tokens at the end of 32768, 28/4 heads of 128, bf16): 872 to 902 us, 1030 to 1070 TFLOP/s, 61 to 63 % of
// the measured bf16 peak; a step takes 1.15 us, of which the MMAs themselves are 0.72 (S: 16
// of N = 64, 29 ns each, both operands from shared memory; P V: 8 of N = 128, 31 ns), their
// commits (29 ns each) and the changes of accumulator 0.35. Taken out again: one S buffer of
// 128 keys a tile with P in two halves (844 us here with bursts by turns, but 72 us for a
// mixed batch of 500-token chunks at d = 64 where this form takes 58: its chain softmax, P V,
// S is as long as its step); a quarter of the exponentials by polynomial (10 % slower: the
// exponentials are hidden already).
// Events: tile i's event e is on barrier ev[i][e & 1]: event j of a unit of n steps says
// that S_j is formed and O += P_{j-2} V done; events n and n + 1 that the last two are.
// Work in equal shares (paged.cuh). The parts of a unit cut between CTAs are joined in
// a binary tree over the CTAs: the second of two neighbours to finish joins both, so that
// no CTA waits and no CTA joins more than log2 of the parts; a joint is symmetric in
// its two sides, so the bits do not depend on who is second. (It takes about 4 us; a
// second launch for the joints took 10 to 18.)
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
constexpr int kStep = 64;           // keys of a step
constexpr float kSlack = 8.0f;      // log2 slack before the reference maximum moves
static_assert(kUnitRows == kPagedRowsMax, "workspace slots");

// E8: an 8-bit cache, whose tiles land in a ring of their own (as they are in memory) and
// are widened into the 16-bit ring by four more warps.
template <int D, bool E8>
struct TilesCfg {
    static constexpr int HALVES = D / 64;                    // 128-byte wide column blocks
    static constexpr uint32_t BLOCK = kKeys * 128;           // bytes of one such block of a tile
    static constexpr uint32_t TILE = HALVES * BLOCK;         // K or V tile
    static constexpr int STAGES = E8 ? (D == 128 ? 3 : 6) : D == 128 ? 4 : 8;
    static constexpr int THREADS = E8 ? 512 : 384;           // 168 or 128 registers a thread
    static constexpr uint32_t RAW_TILE = kKeys * D;          // 8-bit K or V tile
    static constexpr int RAW_STAGES = D == 128 ? 2 : 4;
    static constexpr int LOADS = E8 ? RAW_STAGES : STAGES;   // stages that the copies fill
    static constexpr uint32_t RING = 2 * TILE;               // behind q: [2][HALVES][kM rows][128 B]
    static constexpr uint32_t OUT = RING + STAGES * TILE;    // [8 warps][32 rows][128 B] on their way out
    static constexpr uint32_t RAW = OUT + 8 * 4096;
    static constexpr uint32_t BARS = RAW + (E8 ? RAW_STAGES * RAW_TILE : 0);
    static constexpr uint32_t BYTES = BARS + 512 + (E8 ? 2 * kM * 4 : 0) + 1024;   // barriers, alignment
    static constexpr uint32_t T_S = 0, T_O = 256;   // tensor memory: S/P of tile i, buffer b at 128 i + 64 b, O at T_O + D i
    static_assert(BYTES <= 232448, "shared memory of an SM");
    static_assert(STAGES * TILE >= (kPagedMaxSeqs + 2) * 8, "the sums' place");
};

// ---------------------------------------------------------------- tcgen05

__device__ __forceinline__ uint32_t sw128(int r, int c) {   // 16-byte piece c of 128-byte row r
    return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4));
}
// Shared-memory matrix descriptors (128-byte swizzle, Blackwell version 1): the low
// word is the address / 16, the high word and bits 16-29 are the layout's.
// K-major: groups of 8 rows 1024 bytes apart. MN-major: blocks of 64 columns LBO
// bytes apart, groups of 8 rows (keys) 1024 bytes apart.
constexpr uint32_t kDescHi = (1024 >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_k(uint32_t a) { return ((a >> 4) & 0x3FFF) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_mn(uint32_t a, uint32_t lbo) { return ((a >> 4) & 0x3FFF) | ((lbo >> 4) << 16); }
// f16 (0) or bf16 (1) operands of one type, fp32 sums; B K-major or MN-major
__host__ __device__ constexpr uint32_t idesc(bool bf, bool b_mn, int N) {
    return (1u << 4) | ((bf ? 1u : 0u) << 7) | ((bf ? 1u : 0u) << 10) | ((b_mn ? 1u : 0u) << 16) |
           ((uint32_t)(N >> 3) << 17) | ((uint32_t)(kM >> 4) << 24);
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// The issuing thread's time is what counts here: an MMA's operands are uniform
// registers, so the low words come from a warp-wide reduction (whose result is one) and
// all else is constant.
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }
// The lane that issues the products also commits them: a commit follows its own thread's
// operations only, and which lane is elected is not said (for one mask it is always the same).
__device__ __forceinline__ bool elect() {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok));
    return ok != 0;
}
template <uint32_t ID, bool ACC>
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "mov.b64 x, {%1, %5};\n\tmov.b64 y, {%2, %5};\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "n"(ID), "n"(ACC ? 1 : 0),
                 "n"(kDescHi)
                 : "memory");
}
template <uint32_t ID>
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 y;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 y, {%2, %5};\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "n"(ID), "r"(acc),
                 "n"(kDescHi)
                 : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
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
__device__ __forceinline__ void st16(uint32_t a, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(a),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
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
__device__ __forceinline__ uint32_t ld_acquire(const uint32_t *p) {
    uint32_t v;
    asm volatile("ld.acquire.cta.shared.u32 %0, [%1];" : "=r"(v) : "r"(smem_u32(p)) : "memory");
    return v;
}
__device__ __forceinline__ void st_release(uint32_t *p, uint32_t v) {
    asm volatile("st.release.cta.shared.u32 [%0], %1;" ::"r"(smem_u32(p)), "r"(v) : "memory");
}
// ---------------------------------------------------------------- parts of a cut unit
//
// CTA c has two slots: slot 0 for the unit it goes on with, slot 1 for the one
// it begins. A slot: O to the row's maximum [D/4][256 rows] float4 (a warp's rows
// stand side by side), then maxima [256] and sums [256].

template <int D>
constexpr size_t kSlot = (size_t)kUnitRows * (D + 2);

// QBF: queries and outputs in bf16, else f16. E8: 8-bit cache, products in f16.
template <int D, bool QBF, bool E8>
__global__ void __launch_bounds__(TilesCfg<D, E8>::THREADS, 1) paged_tiles_kernel(const __grid_constant__ PagedAttnParams p) {
    using C = TilesCfg<D, E8>;
    constexpr bool BF = QBF && !E8;   // type of the products
    using U = Unit<kUnitRows, kKeys>;
    using qt = typename std::conditional<QBF, __nv_bfloat16, __half>::type;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t sbase = smem_u32(smem);
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + C::BARS);
    uint64_t *full = bars;                  // [LOADS] a tile has landed
    uint64_t *empty = bars + 8;             // [STAGES] both issuers' MMAs of it are done
    uint64_t *q_full = bars + 16;           // [2] tile i's q rows are in shared memory (4 warps)
    uint64_t *ev = bars + 18;               // [2][2] events of tile i (above)
    uint64_t *drained = bars + 22;          // [2]
    uint64_t *raw_empty = bars + 24;        // [RAW_STAGES] a tile of 8 bits has been widened (4 warps)
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 28);
    int *abort_flag = reinterpret_cast<int *>(bars + 29);
    // counters that the issuers poll: [8] P written (and O rescaled) by each softmax
    // warp; ring tiles that are ready (V cleared outside the unit's keys): one by the
    // watcher, or [4] by each widening warp
    uint32_t *p_seq = reinterpret_cast<uint32_t *>(bars + 30);
    uint32_t *landed = reinterpret_cast<uint32_t *>(bars + 34);
    constexpr int kLanded = E8 ? 4 : 1;
    int *join = reinterpret_cast<int *>(bars + 36);   // [2] a tile's joint: whether it is the second
    uint64_t *pv_done = bars + 38;          // [2] tile i's last O += P V is done
    float *q_shift = reinterpret_cast<float *>(bars + 40);   // [2][kM] E8: 1 / (power of two on the q row)
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
        for (int i = 0; i < C::LOADS; ++i) mbar_init(&full[i], 1);
        for (int i = 0; i < C::STAGES; ++i) mbar_init(&empty[i], 2);
        for (int i = 0; E8 && i < C::RAW_STAGES; ++i) mbar_init(&raw_empty[i], 4);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&q_full[i], 4);
            mbar_init(&ev[2 * i], 1);
            mbar_init(&ev[2 * i + 1], 1);
            mbar_init(&drained[i], 1);
            mbar_init(&pv_done[i], 1);
        }
        *abort_flag = 0;
        for (int i = 0; i < 8; ++i) p_seq[i] = 0;
        for (int i = 0; i < kLanded; ++i) landed[i] = 0;
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
    // until the counters at word[lane], lane < n, have all reached `want`: bounded, by
    // whole warps
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
        const long long first = a.u0 + kUnitCost;
        t0 = (int)max(0ll, min((long long)a.nt, x0 - first));
        t1 = (int)max(0ll, min((long long)a.nt, x1 - first));
    };
    auto next_unit = [&](U &a) -> bool { return a.u0 + kUnitCost + a.nt < x1 && a.next(p); };

    // steps [k0, k1) of 64 keys (from key 0 on) of tiles [t0, t1) of unit a; one at
    // least (masked) where it has no keys
    auto steps = [&](const U &a, int t0, int t1, int &k0, int &k1) {
        k0 = max(2 * (a.tile0 + t0), a.lo / kStep);
        k1 = max(k0 + 1, min(2 * (a.tile0 + t1), (a.hi + kStep - 1) / kStep));
    };

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
                const uint32_t bytes = __popc(mask) * p.box * (E8 ? D : 128 * C::HALVES);
#pragma unroll 1
                for (int kv = 0; kv < 2; ++kv, ++it) {
                    const int st = it % C::LOADS;
                    if (it >= C::LOADS && !wait(E8 ? &raw_empty[st] : &empty[st], (it / C::LOADS - 1) & 1)) {
                        ok = false;
                        break;
                    }
                    if (lane == 0) mbar_arrive_expect_tx(&full[st], bytes);
                    __syncwarp();
                    if constexpr (E8) {
                        if (need && lane < boxes)
                            tma_box(sbase + C::RAW + st * C::RAW_TILE + b * p.box * D, kv ? &p.tm_v : &p.tm_k, 0, tok, u.g, page,
                                    &full[st]);
                    } else {
                        const int h = lane / boxes;   // boxes * HALVES <= 16
                        if (need && h < C::HALVES)
                            tma_box(sbase + C::RING + st * C::TILE + h * C::BLOCK + b * p.box * 128, kv ? &p.tm_v : &p.tm_k, h * 64,
                                    tok, u.g, page, &full[st]);
                    }
                }
            }
        } while (ok && next_unit(u));
        // copies in flight land before the CTA may end, also where this warp issued its last
        // one before another gave up on it (else they have landed, or do while the others work)
        for (uint32_t i = it > (uint32_t)C::LOADS ? it - C::LOADS : 0; i < it; ++i)
            mbar_drain(&full[i % C::LOADS], (i / C::LOADS) & 1);
    } else if (warp == 9 || warp == 10) {
        // ------------------------------------------------------------ MMA issuers
        auto issuer = [&](auto tile) {
        constexpr int i = decltype(tile)::value;
        constexpr uint32_t ID_S = idesc(BF, false, kStep), ID_O = idesc(BF, true, D);
        constexpr uint32_t t_s = C::T_S + 128 * i, t_o = C::T_O + D * i;   // (the CTA holds all of tensor memory, from 0 on)
        const uint32_t q_lo = uniform(desc_k(sbase + i * C::TILE));
        uint32_t base = 0;           // ring position of the unit's first tile (K; V follows)
        uint32_t n_q = 0, n_p = 0, e = 0, n_pv = 0;   // q and P so far, events, waits for P V
        const uint32_t pv_bar = uniform(smem_u32(&pv_done[i]));
        bool ok = true;
        auto stage_of = [&](uint32_t at) { return sbase + C::RING + (at % C::STAGES) * C::TILE; };
        auto full_wait = [&](uint32_t at) { return reached(landed, kLanded, at + 1); };
        do {
            int t0, t1, k0, k1;
            share_tiles(u, t0, t1);
            if (t0 >= t1) continue;
            steps(u, t0, t1, k0, k1);
            const int first = u.tile0 + t0;   // the ring's first tile of this unit
            auto k_at = [&](int k) { return base + 2 * ((k >> 1) - first); };
            if (i * kM >= u.rows) {   // the tile has no rows: its share of the ring's releases
                for (int t = 0; ok && t < 2 * (t1 - t0); ++t) {
                    ok = full_wait(base + t);
                    if (ok && lane == 0) mbar_arrive(&empty[(base + t) % C::STAGES]);
                    __syncwarp();
                }
                base += 2 * (t1 - t0);
                continue;
            }
            const int n = k1 - k0;
            // S of step k into the buffer of event `ev_no`, its commit; the K tile is
            // released behind its last step
            auto issue_s = [&](int k, uint32_t ev_no) {
                const uint32_t at = k_at(k), turn = uniform(ev_no & 1);
                const uint32_t kb = uniform(desc_k(stage_of(at) + (k & 1) * (kStep * 128)));
                const uint32_t e_bar = uniform(smem_u32(&ev[2 * i + turn])), s_bar = uniform(smem_u32(&empty[at % C::STAGES]));
                const bool leave = (k & 1) || k + 1 == k1;
                if (elect()) {
#pragma unroll
                    for (int c = 0; c < D / 16; ++c) {
                        const uint32_t o = ((c >> 2) * C::BLOCK + (c & 3) * 32) / 16;
                        if (c == 0) mma_ss<ID_S, false>(t_s + 64 * turn, q_lo + o, kb + o);
                        else mma_ss<ID_S, true>(t_s + 64 * turn, q_lo + o, kb + o);
                    }
                    commit(e_bar);
                    if (leave) commit(s_bar);
                }
                __syncwarp();
            };
            ok = wait(&q_full[i], n_q & 1);
            ++n_q;
            for (int j = 0; ok && j < 2; ++j) {
                if (j < n) {
                    ok = full_wait(k_at(k0 + j));
                    if (!ok) break;
                    fence_after();
                    issue_s(k0 + j, e + j);
                } else {   // an event without an S
                    if (elect()) commit(smem_u32(&ev[2 * i + ((e + j) & 1)]));
                    __syncwarp();
                }
            }
            for (int j = 0; ok && j < n; ++j) {
                const int k = k0 + j;
                const uint32_t vt = k_at(k) + 1;
                if (j == 0 || !(k & 1)) {
                    ok = full_wait(vt);
                    if (!ok) break;
                }
                if (j + 2 < n) {   // (asked before the wait for P, so that the burst below is one)
                    ok = full_wait(k_at(k + 2));
                    if (!ok) break;
                }
                ok = reached(p_seq + 4 * i, 4, ++n_p);
                if (!ok) break;
                fence_after();
                const uint32_t b = uniform((e + j) & 1);
                const uint32_t vb = uniform(desc_mn(stage_of(vt) + (k & 1) * (kStep * 128), C::BLOCK));
                const uint32_t s_bar = uniform(smem_u32(&empty[vt % C::STAGES])), acc = uniform(j > 0);
                const bool leave = (k & 1) || k + 1 == k1;
                if (elect()) {   // O += P V
#pragma unroll
                    for (int c = 0; c < kStep / 16; ++c)
                        mma_ts<ID_O>(t_o, t_s + 64 * b + 8 * c, vb + c * (16 * 128 / 16), c > 0 ? 1u : acc);
                    if (j + 2 < n) commit(pv_bar);
                    else if (leave) commit(s_bar);
                }
                __syncwarp();
                if (j + 2 < n) {
                    // S goes over P: only MMAs of one accumulator and shape are sure to run in
                    // the order of their issue
                    ok = wait(&pv_done[i], n_pv & 1);
                    if (!ok) break;
                    ++n_pv;
                    fence_after();
                    if (leave && lane == 0) mbar_arrive(&empty[vt % C::STAGES]);
                    __syncwarp();
                    issue_s(k + 2, e + j + 2);
                } else {
                    if (elect()) commit(smem_u32(&ev[2 * i + b]));
                    __syncwarp();
                }
            }
            e += n + 2;
            base += 2 * (t1 - t0);
        } while (ok && next_unit(u));
        // tensor memory is released below only after every MMA issued here is done
        if (elect()) commit(smem_u32(&drained[i]));
        __syncwarp();
        if (!mbar_drain(&drained[i], 0)) raise_late(p.status);
        };
        if (warp == 9) issuer(std::integral_constant<int, 0>{});
        else issuer(std::integral_constant<int, 1>{});
    } else if (!E8 && warp == 11) {
        // ------------------------------------------------------------ watcher
        // (an issuer's own look at a barrier after a burst of MMAs waits until the
        // burst has left the queue; a look at a word of shared memory does not)
        uint32_t it = 0;
        bool ok = true;
        do {
            int t0, t1;
            share_tiles(u, t0, t1);
            for (int t = t0; ok && t < t1; ++t) {
                for (int kv = 0; ok && kv < 2; ++kv, ++it) {
                    ok = wait(&full[it % C::STAGES], (it / C::STAGES) & 1, true);
                    const int key0 = (u.tile0 + t) * kKeys;
                    if (ok && kv == 1 && (key0 < u.lo || key0 + kKeys > u.hi)) {   // V's rows outside the unit's keys
                        uint8_t *v = smem + C::RING + (it % C::STAGES) * C::TILE;
                        for (int r = lane >> 3; r < kKeys; r += 4)
                            if (key0 + r < u.lo || key0 + r >= u.hi)
                                for (int h = 0; h < C::HALVES; ++h)
                                    *reinterpret_cast<uint4 *>(v + h * C::BLOCK + r * 128 + (lane & 7) * 16) =
                                        make_uint4(0, 0, 0, 0);
                        fence_proxy_async_smem();
                    }
                    __syncwarp();
                    if (ok && lane == 0) st_release(landed, it + 1);
                }
            }
        } while (ok && next_unit(u));
    } else if (E8 && warp >= 12) {
        // ------------------------------------------------------------ widening
        // 32 rows a warp: 16 bytes of a row a lane become two 16-byte pieces of f16 (exact)
        // in the layout that the MMA reads. The lanes of a row's second half (d = 128) write
        // theirs in the other order, so that a row's 8 writes lie in distinct banks.
        constexpr int L = D / 16;   // lanes a row
        const int w = warp - 12, c = lane % L;
        uint32_t it = 0;
        bool ok = true;
        do {
            int t0, t1;
            share_tiles(u, t0, t1);
            for (int t = t0; ok && t < t1; ++t) {
                const int key0 = (u.tile0 + t) * kKeys;
                for (int kv = 0; ok && kv < 2; ++kv, ++it) {
                    ok = wait(&full[it % C::RAW_STAGES], (it / C::RAW_STAGES) & 1, true);
                    if (ok && it >= C::STAGES) ok = wait(&empty[it % C::STAGES], (it / C::STAGES - 1) & 1);
                    if (!ok) break;
                    const uint8_t *src = smem + C::RAW + (it % C::RAW_STAGES) * C::RAW_TILE + w * 32 * D + lane * 16;
                    uint8_t *dst = smem + C::RING + (it % C::STAGES) * C::TILE + (c >> 2) * C::BLOCK;
#pragma unroll 4
                    for (int x = 0; x < L; ++x) {
                        const int row = w * 32 + x * (32 / L) + lane / L;
                        uint4 v = *reinterpret_cast<const uint4 *>(src + x * 512);
                        if (kv == 1 && (key0 + row < u.lo || key0 + row >= u.hi)) v = make_uint4(0, 0, 0, 0);   // of V
                        uint4 a, b;
                        widen4(v.x, a.x, a.y);
                        widen4(v.y, a.z, a.w);
                        widen4(v.z, b.x, b.y);
                        widen4(v.w, b.z, b.w);
                        const bool swap = (c & 4) != 0;
                        *reinterpret_cast<uint4 *>(dst + sw128(row, 2 * (c & 3) + swap)) = swap ? b : a;
                        *reinterpret_cast<uint4 *>(dst + sw128(row, 2 * (c & 3) + !swap)) = swap ? a : b;
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        st_release(landed + w, it + 1);
                        mbar_arrive(&raw_empty[it % C::RAW_STAGES]);
                    }
                }
            }
        } while (ok && next_unit(u));
    } else if (warp < 8) {
        // ------------------------------------------------------------ softmax
        const int i = warp >> 2, r = threadIdx.x & 127;   // tile, row
        const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + C::T_S + 128 * i + lane_off, to = tmem + C::T_O + D * i + lane_off;
        uint8_t *out_rows = smem + C::OUT + warp * 4096;
        uint32_t e = 0, n_p = 0;   // events before this unit, P written so far
        bool ok = true;
        const uint32_t scale_sign = p.scale < 0.f ? 0x80008000u : 0u;   // goes into q, so that maxima stay maxima
        const float qs_all = fabsf(p.scale) * 1.44269504088896340736f;
        // offset of this thread's row of unit a in rows of strides ts, hs (of the unit's
        // first row where it has none): the warp's lanes ask one another for theirs
        auto offset_of = [&](const U &a, long long t_s, long long h_s) -> long long {
            const int row = i * kM + r;
            const int pr = a.b * kUnitRows + (row < a.rows ? row : 0), tok = p.by_rep.div(pr);
            return (long long)(a.q.q0 + tok) * t_s + (long long)(a.g * p.rep + pr - tok * p.rep) * h_s;
        };
        // the q rows of unit a into shared memory: a warp its 32 rows, half a warp a
        // row at d = 128 (a thread its own row would touch a cache line a lane), all of
        // them on their way at once
        auto load_q = [&](const U &a) {
            if (i * kM >= a.rows) return;
            uint32_t sign = scale_sign;
            if (E8 && p.k_scale && __ldg(p.k_scale + a.g) < 0.f) sign ^= 0x80008000u;
            constexpr int L = D / 8, N = E8 ? 8 : L;   // lanes a row, loads a lane at a time
            const int c = lane % L;
            const long long off = offset_of(a, p.q_ts, p.q_hs);
            uint8_t *dst = smem + i * C::TILE + (c >> 3) * C::BLOCK;
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
                // rows whose largest value is between 2^-4 and 2^15 go to f16 as they are (what
                // is below its range is then below 2^-21 of the largest): all of the warp's, or
                // each row is looked at by itself
                bool as_is = true;
                auto largest = [](const uint4 &x) {
                    const __nv_bfloat162 *y = reinterpret_cast<const __nv_bfloat162 *>(&x);
                    return __hmax2(__hmax2(__habs2(y[0]), __habs2(y[1])), __hmax2(__habs2(y[2]), __habs2(y[3])));
                };
                if constexpr (E8 && QBF) {
                    constexpr unsigned GROUP = L == 32 ? FULL : (1u << (L & 31)) - 1;
                    bool fine = true;
#pragma unroll
                    for (int k = 0; k < N; ++k) {
                        const __nv_bfloat162 t = largest(v[k]);
                        const float m = fmaxf(__low2float(t), __high2float(t));
                        const unsigned some = __ballot_sync(FULL, m >= 0.0625f) >> (lane & ~(L - 1));
                        fine &= (some & GROUP) != 0 && m < 32768.f;
                    }
                    as_is = __all_sync(FULL, fine);
                }
                if constexpr (E8 && QBF) {
                    if (!as_is) {   // each row times its power of two
#pragma unroll 1
                        for (int k = 0; k < N; ++k) {
                            uint4 x = v[0];   // (by turns in v[0]: an index would put v into memory)
#pragma unroll
                            for (int y = 0; y + 1 < N; ++y) v[y] = v[y + 1];
                            __nv_bfloat162 t = largest(x);
#pragma unroll
                            for (int o = 1; o < L; o <<= 1) t = __hmax2(t, __shfl_xor_sync(FULL, t, o));
                            const float f = f16_shift(fmaxf(__low2float(t), __high2float(t)));
                            if (c == 0) q_shift[i * kM + (warp & 3) * 32 + (k0 + k) * (32 / L) + lane / L] = 1.f / f;
                            uint32_t *w = reinterpret_cast<uint32_t *>(&x);
#pragma unroll
                            for (int y = 0; y < 4; ++y)
                                w[y] = pack2<false>(__uint_as_float(w[y] << 16) * f, __uint_as_float(w[y] & 0xffff0000u) * f);
                            v[N - 1] = x;
                        }
                    } else {
                        if ((lane * L >> 5) / N * N == k0) q_shift[i * kM + r] = 1.f;   // (this lane's row is among these)
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
                    const int row = (warp & 3) * 32 + (k0 + k) * (32 / L) + lane / L;
                    v[k].x ^= sign;
                    v[k].y ^= sign;
                    v[k].z ^= sign;
                    v[k].w ^= sign;
                    if (i * kM + row >= a.rows) v[k] = make_uint4(0, 0, 0, 0);
                    *reinterpret_cast<uint4 *>(dst + sw128(row, c & 7)) = v[k];
                }
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
            float qs = qs_all;
            if constexpr (E8 && QBF) qs *= q_shift[i * kM + r];
            if (E8 && p.k_scale) qs *= fabsf(__ldg(p.k_scale + u.g));
            if constexpr (E8) qs = at_least_normal(qs);
            float m = -INFINITY, l = 0.f;
            int k0, k1;
            steps(u, t0, t1, k0, k1);
            int all_ok;
            auto event = [&](uint32_t no) { return wait(&ev[2 * i + (no & 1)], (no >> 1) & 1); };
            if (mine) {
                for (int k = k0; k < k1; ++k) {
                    const uint32_t no = e + (k - k0), tb = ts + 64 * (no & 1);
                    if (!event(no)) {
                        ok = false;
                        break;
                    }
                    fence_after();
                    float s[64];
                    ld32(tb, reinterpret_cast<uint32_t *>(s));
                    ld32(tb + 32, reinterpret_cast<uint32_t *>(s) + 32);
                    wait_ld();
                    const int key0 = k * kStep;
                    if (key0 < all_lo || key0 + kStep > all_hi) {
#pragma unroll
                        for (int x = 0; x < 64; ++x)
                            if (key0 + x < lo || key0 + x >= hi) s[x] = -INFINITY;
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
                        if (k > k0) {   // O holds every step before this one only now
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
                // the last product, before the next unit's events
                if (ok) ok = event(e + (k1 - k0) + 1);
                e += k1 - k0 + 2;
                // the tile's four warps go on together or not at all (they meet below)
                asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbarrier.cta.red.and.pred q, %2, 128, p;\n\t"
                             "selp.b32 %0, 1, 0, q;\n\t}"
                             : "=r"(all_ok)
                             : "r"((int)ok), "r"(1 + i)
                             : "memory");
                ok = all_ok != 0;
            }
            fence_after();
            // the next unit's q, so that its products may start during the epilogue
            const U done = u;
            const int d0 = t0, d1 = t1;
            if (ok) {
                more = next_unit(u) && skip_empty(u, t0, t1);
                if (more) load_q(u);
            }
            if (!ok || !mine) continue;
            // a part of a cut unit: up the tree of its CTAs as far as this one is the
            // second to finish
            bool last = d0 == 0 && d1 == done.nt;
            if (!last) {
                const int c0 = share_of(done.u0 + kUnitCost, total, ctas);
                const int n = share_of(done.u0 + kUnitCost + done.nt - 1, total, ctas) - c0 + 1;   // parts
                constexpr int J = E8 ? 32 : 64;   // columns at a time, as the registers allow
                const int row = i * kM + r, one = 1 << (16 * i);   // the tiles count apart, in the halves of a counter
                auto slot_of = [&](int k) { return p.part + (size_t)((c0 + k) * 2 + (k == 0)) * kSlot<D>; };
                const int me = blockIdx.x - c0;
                last = true;
                for (int j = 1; (1 << (j - 1)) < n; ++j) {
                    const int left = me >> j << j, right = left + (1 << (j - 1));   // first parts of the two sides
                    if (right >= n) continue;                                      // no right side
                    int *counter = p.counters + c0 + right;
                    const bool is_left = me < right;
                    float *slot = slot_of(is_left ? left : right);
#pragma unroll 1
                    for (int c = 0; c < D; c += J) {
                        float o[J];
#pragma unroll
                        for (int x = 0; x < J; x += 32) ld32(to + c + x, reinterpret_cast<uint32_t *>(o) + x);
                        wait_ld();
#pragma unroll
                        for (int k = 0; k < J; k += 4)
                            *(reinterpret_cast<float4 *>(slot) + ((c + k) / 4) * kUnitRows + row) =
                                make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
                    }
                    slot[kUnitRows * D + row] = m;
                    slot[kUnitRows * (D + 1) + row] = l;
                    __threadfence();
                    asm volatile("bar.sync %0, 128;" ::"r"(1 + i) : "memory");
                    if (r == 0) join[i] = (atomicAdd(counter, one) >> (16 * i)) & 0xffff;
                    asm volatile("bar.sync %0, 128;" ::"r"(1 + i) : "memory");
                    const int second = *reinterpret_cast<volatile int *>(&join[i]);
                    asm volatile("bar.sync %0, 128;" ::"r"(1 + i) : "memory");
                    if (!second) {   // the other side goes on
                        last = false;
                        break;
                    }
                    if (r == 0) atomicAdd(counter, -2 * one);   // as the next call wants it
                    __threadfence();
                    const float *other = slot_of(is_left ? right : left);
                    const float m2 = __ldcg(other + kUnitRows * D + row), l2 = __ldcg(other + kUnitRows * (D + 1) + row);
                    const float M = fmaxf(m, m2);
                    const float a = m == -INFINITY ? 0.f : fast_exp2(m - M), b = m2 == -INFINITY ? 0.f : fast_exp2(m2 - M);
                    m = M;
                    l = __fadd_rn(__fmul_rn(a, l), __fmul_rn(b, l2));
#pragma unroll 1
                    for (int c = 0; c < D; c += J) {
                        float4 x[J / 4];
#pragma unroll
                        for (int k = 0; k < J / 4; ++k)
                            x[k] = __ldcg(reinterpret_cast<const float4 *>(other) + (c / 4 + k) * kUnitRows + row);
                        float o[J];
#pragma unroll
                        for (int k = 0; k < J; k += 32) ld32(to + c + k, reinterpret_cast<uint32_t *>(o) + k);
                        wait_ld();
#pragma unroll
                        for (int k = 0; k < J / 4; ++k) {
                            o[4 * k] = __fadd_rn(__fmul_rn(a, o[4 * k]), __fmul_rn(b, x[k].x));
                            o[4 * k + 1] = __fadd_rn(__fmul_rn(a, o[4 * k + 1]), __fmul_rn(b, x[k].y));
                            o[4 * k + 2] = __fadd_rn(__fmul_rn(a, o[4 * k + 2]), __fmul_rn(b, x[k].z));
                            o[4 * k + 3] = __fadd_rn(__fmul_rn(a, o[4 * k + 3]), __fmul_rn(b, x[k].w));
                        }
#pragma unroll
                        for (int k = 0; k < J; k += 32) st32(to + c + k, reinterpret_cast<const uint32_t *>(o) + k);
                    }
                    wait_st();
                }
            }
            if (last) {
                const float vs = E8 && p.v_scale ? __ldg(p.v_scale + done.g) : 1.f;
                const float inv = l > 0.f || l != l ? vs / l : 0.f;
                const long long off = offset_of(done, p.o_ts, p.o_hs);
                // 64 values of the warp's 32 rows at a time through shared memory: 8 lanes
                // write a row's 128 bytes (a thread its own row would touch a line a lane)
#pragma unroll 1
                for (int c = 0; c < D; c += 64) {
                    float o[64];
                    ld32(to + c, reinterpret_cast<uint32_t *>(o));
                    ld32(to + c + 32, reinterpret_cast<uint32_t *>(o) + 32);
                    wait_ld();
                    // (a row without keys: O is 0 * V of cleared rows)
#pragma unroll
                    for (int x = 0; x < 8; ++x)
                        *reinterpret_cast<uint4 *>(out_rows + sw128(lane, x)) =
                            make_uint4(pack2<QBF>(o[8 * x] * inv, o[8 * x + 1] * inv), pack2<QBF>(o[8 * x + 2] * inv, o[8 * x + 3] * inv),
                                       pack2<QBF>(o[8 * x + 4] * inv, o[8 * x + 5] * inv),
                                       pack2<QBF>(o[8 * x + 6] * inv, o[8 * x + 7] * inv));
                    __syncwarp();
                    uint4 v[8];
#pragma unroll
                    for (int x = 0; x < 8; ++x) v[x] = *reinterpret_cast<const uint4 *>(out_rows + sw128(4 * x + (lane >> 3), lane & 7));
#pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        const int lr = 4 * x + (lane >> 3);   // row of the warp
                        qt *dst = static_cast<qt *>(p.out) + __shfl_sync(FULL, off, lr) + c + 8 * (lane & 7);
                        if (i * kM + (warp & 3) * 32 + lr < done.rows) {
                            if (p.o_vec) {
                                *reinterpret_cast<uint4 *>(dst) = v[x];
                            } else {
                                unsigned short *y = reinterpret_cast<unsigned short *>(dst);
                                const uint32_t w[4] = {v[x].x, v[x].y, v[x].z, v[x].w};
#pragma unroll
                                for (int k = 0; k < 4; ++k) {
                                    y[2 * k] = (unsigned short)(w[k] & 0xffffu);
                                    y[2 * k + 1] = (unsigned short)(w[k] >> 16);
                                }
                            }
                        }
                    }
                    __syncwarp();
                }
                const int tok = p.by_rep.div(pr), h = done.g * p.rep + pr - tok * p.rep;
                if (p.lse && in)
                    p.lse[(long long)(done.q.q0 + tok) * p.H + h] = log_sum<BF>(m, l);
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

template <int D, bool QBF, bool E8>
cudaError_t launch_k(const PagedAttnParams &p, int n_ctas, cudaStream_t s) {
    using C = TilesCfg<D, E8>;
    if (cudaError_t e = ensure_smem_limit(reinterpret_cast<const void *>(paged_tiles_kernel<D, QBF, E8>), C::BYTES)) return e;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(n_ctas);
    cfg.blockDim = dim3(C::THREADS);
    cfg.dynamicSmemBytes = C::BYTES;
    cfg.stream = s;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, paged_tiles_kernel<D, QBF, E8>, p);
}

}  // namespace

cudaError_t launch_paged_tiles(const PagedAttnParams &p, int d, int q_type, int cache_type, int n_ctas, cudaStream_t s) {
    const bool bf = q_type == KORE_CUDA_BF16, e8 = cache_type == KORE_CUDA_E4M3;
    if (d == 128) {
        if (e8) return bf ? launch_k<128, true, true>(p, n_ctas, s) : launch_k<128, false, true>(p, n_ctas, s);
        return bf ? launch_k<128, true, false>(p, n_ctas, s) : launch_k<128, false, false>(p, n_ctas, s);
    }
    if (d == 64) {
        if (e8) return bf ? launch_k<64, true, true>(p, n_ctas, s) : launch_k<64, false, true>(p, n_ctas, s);
        return bf ? launch_k<64, true, false>(p, n_ctas, s) : launch_k<64, false, false>(p, n_ctas, s);
    }
    return cudaErrorInvalidValue;
}

}  // namespace kore
