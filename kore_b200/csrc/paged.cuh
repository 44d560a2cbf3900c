// paged.cuh — parameter blocks of the operators on a caller-owned paged cache
// (rotary positions, append, attention) and the attention's division of work.
#pragma once

#include "attn.cuh"
#include "common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

namespace kore {

// Device status codes of these operators, beside common.cuh's (DEV_BAD_PAGE).
constexpr int DEV_BAD_POSITION = 6;   // a position outside the rotation table
constexpr int DEV_BAD_SEQUENCE = 7;   // a sequence's bounds, length or page table do not fit
constexpr int DEV_NO_PAGES = 8;       // the pool has too few free pages

constexpr int kPagedMaxSeqs = 4096;      // sequences of one batch
constexpr int kPagedMaxRequests = 65536; // requests of one pool
constexpr int kPagedMaxTree = 1024;      // tokens of a tree
constexpr int kPagedMaxTokens = 1 << 30; // rows of a plan or a store: steps beyond the last stay in 32 bits
constexpr int kPagedMaxLayers = 128;     // layers of one launch
constexpr int kPagedMaxCtas = 160;       // CTAs (SMs) that an attention launch uses at most
constexpr int kPagedRowsMax = 256;       // query rows of a work unit at most
constexpr size_t kPagedZeroed = 1024;    // leading workspace bytes that are zero between calls

// n / d for 0 <= n < 2^31 by a multiplication and a shift (Granlund and
// Montgomery, 1994): the kernels divide by the group's size and the page's at
// every unit and tile.
struct FastDiv {
    uint32_t mul, shift, d;
    static FastDiv of(uint32_t d) {
        uint32_t s = 0;
        while ((1ull << s) < d) ++s;
        return {(uint32_t)(((1ull << 32) * ((1ull << s) - d)) / d + 1), s, d};
    }
    __device__ __forceinline__ int div(int n) const {
        return (int)((__umulhi((uint32_t)n, mul) + (uint32_t)n) >> shift);
    }
    __device__ __forceinline__ int mod(int n, int q) const { return n - q * (int)d; }
};

// A tensor of rows of heads: element e of head h of row t at t*ts + h*hs + e.
struct HeadRows {
    const void *in;
    void *out;
    long long in_ts, in_hs, out_ts, out_hs;
    int heads;
};

struct RotateParams {
    HeadRows q;                // rotated rows (heads 0: none)
    HeadRows k, v;             // appended rows (append only): out, strides unused
    const float *table;        // [n_pos][rot/2][2]; null: nothing is rotated
    const int *pos;            // rope only: [n_tok]
    int n_tok, n_pos, rot, interleaved, d;
    // append only
    int n_seq, table_stride, n_pages, P, G;
    long long page_stride;
    const int *q_start, *kv_len, *page_table;
    void *kc, *vc;
    const float *k_scale, *v_scale;
    int *status;
};

// A page pool and a step (paged_plan.cu); amount: new tokens (plan) or positions kept (trim).
struct PlanParams {
    int *free_pages, *n_free, *table, *length;
    int n_pages, n_requests, stride, P;
    FastDiv by_page;
    int n_seq, n_tok, out_stride;
    const int *request, *amount;
    int *q_start, *kv_len, *page_table, *pos;
    long long *slots;
    int *status;
};

struct StoreParams {
    HeadRows q, k, v;          // q: heads 0: none; k, v: out, strides unused
    const long long *slots;
    const int *pos;            // null: no row is left out for its position
    const float *table;
    int n_tok, n_pos, rot, interleaved, d, P, G;
    FastDiv by_page;
    long long n_slots, page_stride;
    void *kc, *vc;
    const float *k_scale, *v_scale;
    const void *q_weight, *k_weight;   // null: those heads have no norm
    int weight_type;
    long long q_weight_hs, k_weight_hs;
    float eps, most;                   // most: heads whose squares' sum passes it are scaled
    int *status;
};

struct TreeParams {
    const int *q_start, *kv_len, *parent, *token, *choice;
    int n_seq, n_tok, most, words, path_stride;   // most: tokens of a sequence at most
    long long cap;                                // positions of a sequence at most
    uint32_t *mask;
    int *pos, *path, *count, *next, *kept;
    int *status;
};

struct CommitParams {
    const int *q_start, *kv_len, *page_table, *path, *count;
    int n_seq, table_stride, path_stride, n_pages, n_layers, P, G, row_pieces;   // pieces: of 16 bytes
    FastDiv by_page;
    long long page_pieces;
    int *status;
    void *k[kPagedMaxLayers], *v[kPagedMaxLayers];   // v null: the keys' memory is the values' too
};

struct PagedAttnParams {
    TmaDesc tm_k, tm_v;        // K and V pools as tensor maps (many-row kernel, 16-bit caches)
    const void *k, *v;
    long long page_stride;     // elements
    const int *q_start, *kv_len, *page_table;
    int table_stride, n_seq, n_tok, n_pages, P, H, G, rep;
    FastDiv by_rep, by_page;
    const void *q;
    void *out;
    long long q_ts, q_hs, o_ts, o_hs;
    float *lse;
    const float *k_scale, *v_scale;
    float scale;
    int causal, window;
    int q_vec, o_vec;          // q (out) rows are 16-byte aligned
    int box;                   // rows of a tensor-map box
    int small;                 // no sum of costs comes near 2^31
    int *counters;             // [kPagedMaxCtas] zero between calls
    float *part;               // [kPagedMaxCtas][2] partial results
    int *status;
    unsigned long long wait_ns;   // a wait gives up after so long
    const uint32_t *mask;      // trees: [n_tok][words], bit j: the token sees token j of its chunk
    int words;
};

// four e4m3 values (first in the lowest byte) as two pairs of f16
__device__ __forceinline__ void widen4(uint32_t x, uint32_t &a, uint32_t &b) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(a), "=r"(b)
        : "r"(x));
}

// two values as a pair of bf16 or of f16
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

// A box of a page (tokens from tok on, values from x on) into shared memory; with an L2 policy or
// without.
__device__ __forceinline__ void tma_box(uint32_t dst, const TmaDesc *map, int x, int tok, int g, int page, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
        ::"r"(dst), "l"(map), "r"(x), "r"(tok), "r"(g), "r"(page), "r"(smem_u32(bar))
        : "memory");
}
__device__ __forceinline__ void tma_box(uint32_t dst, const TmaDesc *map, int x, int tok, int g, int page, uint64_t *bar,
                                        uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint "
        "[%0], [%1, {%2, %3, %4, %5}], [%6], %7;" ::"r"(dst),
        "l"(map), "r"(x), "r"(tok), "r"(g), "r"(page), "r"(smem_u32(bar)), "l"(policy)
        : "memory");
}

// The power of two that takes a row's largest value m to 2^7 .. 2^8: bf16 values down
// to 2^-22 of it are then exact in f16. 1 for 0, infinities and NaN; at most 2^100 (a row
// whose largest is below 2^-93 stands lower by as much).
__device__ __forceinline__ float f16_shift(float m) {
    const int e = (__float_as_int(m) >> 23) - 127;
    return m > 0.f && m < INFINITY ? __int_as_float((127 + min(7 - e, 100)) << 23) : 1.f;   // (7 - e >= -120)
}

// The factor on a unit's products with an 8-bit cache (its sign goes into q, so that the largest
// product has the largest score): not 0, since -inf of a masked key times 0 is no mask. A
// product is below 2^40, so that with the least normal value every score is 0 all the same.
__device__ __forceinline__ float at_least_normal(float factor) { return factor < 0x1p-126f ? 0x1p-126f : factor; }

cudaError_t launch_rope_table(const float *freq, int half, double amp, int n_pos, float *table, cudaStream_t s);
cudaError_t launch_rotate(const RotateParams &p, int in_type, int cache_type, bool vec, cudaStream_t s);
cudaError_t launch_plan(const PlanParams &p, bool trim, cudaStream_t s);
cudaError_t launch_store(const StoreParams &p, int in_type, int cache_type, bool vec, int sms, cudaStream_t s);
cudaError_t launch_tree_mask(const TreeParams &p, cudaStream_t s);
cudaError_t launch_accept(const TreeParams &p, cudaStream_t s);
cudaError_t launch_commit(const CommitParams &p, cudaStream_t s);
// n_ctas, n_sms: SMs of the device, at most kPagedMaxCtas. Rows: trees where p.mask is given
cudaError_t launch_paged_rows(const PagedAttnParams &p, int d, int q_type, int cache_type, int n_ctas, cudaStream_t s);
cudaError_t launch_paged_tree_tiles(const PagedAttnParams &p, int d, int q_type, int cache_type, int n_sms, cudaStream_t s);
cudaError_t launch_paged_tiles(const PagedAttnParams &p, int d, int q_type, int cache_type, int n_ctas, cudaStream_t s);

// ---------------------------------------------------------------- division of the attention's work
//
// The work is cut into units: (sequence, KV head, block of ROWS packed query
// rows), where packed row r of a chunk is token r / rep, query head r % rep of
// the group, so that the whole group shares one pass over the keys. A unit's
// key range is cut into tiles. All units' tiles stand in one row (in the order
// sequence, head, block, tile; kUnitCost virtual tiles before each unit's own
// for its start and end), and CTA c of n takes the c-th n-th of the row: equal
// shares however ragged the batch, with nothing planned on the host. At most
// two units of a CTA are shared with other CTAs (its first and its last), so a
// CTA needs two slots for partial results, whatever the batch.

constexpr int kUnitCost = 1;
// Of the trees' 64-key tiles: the change from one unit to the next and the joint of its parts take about as
// long as these (32 sequences of 16 tokens on up to 8192, 28/4 heads of 128: 73.9 us with 1, 71.4 with 8 and 15;
// 48 of up to 33 on 3000, 14/2 heads of 64: 31.3 with 5, 31.6 with 8, 32.3 with 11).
constexpr int kTreeUnitCost = 8;

constexpr uint32_t FULL_WORD = 0xffffffffu;

struct Seq {
    int q0, n, kv;
};

// The sequence's bounds; n = 0 (it is left out) where they do not fit. TREE: its tokens see what
// their masks say of each other, and all that is before them.
template <bool TREE>
__device__ __forceinline__ Seq load_seq(const PagedAttnParams &p, int s, bool report) {
    Seq q;
    q.q0 = __ldg(p.q_start + s);
    q.n = __ldg(p.q_start + s + 1) - q.q0;
    q.kv = __ldg(p.kv_len + s);
    if (q.n != 0 && (q.n < 0 || q.q0 < 0 || q.q0 > p.n_tok - q.n || q.kv < 0 ||
                     q.kv > (long long)p.table_stride * p.P || (TREE && (q.kv < q.n || q.n > p.words * 32)))) {
        if (report) raise_error(p.status, DEV_BAD_SEQUENCE);
        q.n = 0;
    }
    return q;
}

// Probabilities in f16 stand 2^7 higher than exp2(score - reference): f16 ends at
// 2^-24, and many keys of small probability each may weigh as much as one of a large
// one. (With the references' slack of 2^8 they stay below 2^15.) Sums stand as much
// higher, so that outputs need nothing; bf16 has fp32's range.
template <bool BF>
constexpr float kBias = BF ? 0.f : 7.f;

// Natural log of a softmax's sum from its reference (log2) and the sum over it.
template <bool BF>
__device__ __forceinline__ float log_sum(float m, float l) {
    return l > 0.f || l != l ? (m - kBias<BF>)*0.69314718055994530942f + logf(l) : -INFINITY;
}

// Keys [lo, hi) that some token of the packed rows [r0, r1) of the chunk sees (TREE: may see).
template <bool TREE>
__device__ __forceinline__ void key_range(const PagedAttnParams &p, const Seq &q, int r0, int r1, int &lo, int &hi) {
    if constexpr (TREE) {
        lo = 0;
        hi = q.kv;
        return;
    }
    const int first = q.kv - q.n + p.by_rep.div(r0), last = q.kv - q.n + p.by_rep.div(r1 - 1);
    hi = p.causal ? min(q.kv, last + 1) : q.kv;
    lo = p.window > 0 && first >= p.window ? first - p.window + 1 : 0;
    hi = max(hi, 0);
    lo = min(lo, hi);
}

// What a token of a tree sees of the keys from x on (counted from its chunk's first token; x may lie before
// it, in the context), 32 of them; n: tokens of the chunk.
__device__ __forceinline__ uint32_t tree_bits(const uint32_t *mask, int words, int x, int n) {
    auto word = [&](int w) -> uint32_t {
        if (w < 0) return FULL_WORD;
        const int left = n - 32 * w;
        if (left <= 0 || w >= words) return 0u;
        return __ldg(mask + w) & (left < 32 ? (1u << left) - 1 : FULL_WORD);
    };
    const int w = x >> 5;
    return __funnelshift_r(word(w), word(w + 1), x & 31);
}

template <int ROWS, int KEYS, bool TREE = false>
struct Unit {
    static constexpr int COST = TREE && ROWS == 128 ? kTreeUnitCost : kUnitCost;
    int s, g, b;           // sequence, KV head, block of rows
    Seq q;
    int rows;              // valid rows of the block
    int lo, hi;            // keys
    int tile0, nt;         // first tile, tiles (1 for a unit without keys)
    long long u0;          // virtual position of the unit's start

    __device__ __forceinline__ int blocks(const PagedAttnParams &p) const { return (q.n * p.rep + ROWS - 1) / ROWS; }
    __device__ __forceinline__ void range(const PagedAttnParams &p) {
        rows = min(ROWS, q.n * p.rep - b * ROWS);
        key_range<TREE>(p, q, b * ROWS, b * ROWS + rows, lo, hi);
        tile0 = lo / KEYS;
        nt = max(1, (hi + KEYS - 1) / KEYS - tile0);
    }
    // To the next unit; false behind the last one.
    __device__ __forceinline__ bool next(const PagedAttnParams &p) {
        u0 += COST + nt;
        if (++b == blocks(p)) {
            b = 0;
            if (++g == p.G) {
                g = 0;
                do {
                    if (++s >= p.n_seq) return false;
                    q = load_seq<TREE>(p, s, false);
                } while (q.n == 0);
            }
        }
        range(p);
        return true;
    }
};

// Cost (tiles and kUnitCost a unit) of blocks b0 + lane of one head of a
// sequence; 0 behind its last block.
template <int ROWS, int KEYS, bool TREE>
__device__ __forceinline__ int block_cost(const PagedAttnParams &p, const Seq &q, int b, int nb) {
    if (b >= nb) return 0;
    Unit<ROWS, KEYS, TREE> u;
    u.q = q;
    u.b = b;
    u.range(p);
    return u.COST + u.nt;
}

// A wait ran out: in place of any other code, since it is what makes the workspace unusable.
// (The store is enough; without raise_error beside it the compiler's choice of registers made
// the 8-bit chunk kernel 2 to 4 % slower.)
__device__ __forceinline__ void raise_late(int *status) {
    raise_error(status, DEV_WAIT_FULL_TIMEOUT);
    if (status) *reinterpret_cast<volatile int *>(status) = DEV_WAIT_FULL_TIMEOUT;
}

// A wait that did not end at its first look: until the phase is done, or false when
// `limit_ns` (or kWaitPolls looks) are over. (Inline, and without mbar_wait's timing of the
// first look: out of line it cost the chunk kernel 1 %, with that timing 4 %.)
__device__ __forceinline__ bool late_wait(uint64_t *bar, uint32_t parity, uint64_t limit_ns) {
    const uint64_t since = global_ns();
    for (uint32_t looks = 1; looks < kWaitPolls; ++looks) {
        // (a look may itself last until the phase is done: then it counts as well)
        if (mbar_try_wait(bar, parity)) return global_ns() - since <= limit_ns;
        if ((looks & 7) == 0 && global_ns() - since > limit_ns) break;
    }
    return false;
}

// The wait for a tile copy. Under a limit shorter than the default the first look is timed too.
__device__ __forceinline__ bool copy_wait(uint64_t *bar, uint32_t parity, uint64_t limit_ns) {
    if (limit_ns >= kWaitNs && mbar_try_wait(bar, parity)) return true;
    return late_wait(bar, parity, limit_ns);
}

// Asks for a tensor map ahead of its first copy.
__device__ __forceinline__ void prefetch_map(const TmaDesc *m) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory");
}

// Quotient of two non-negative numbers that fit 32 bits in all but absurd cases
// (a 64-bit division takes some hundreds of cycles).
__device__ __forceinline__ long long quick_div(long long a, long long b) {
    if (((a | b) >> 32) == 0) return (unsigned)a / (unsigned)b;
    return a / b;
}

// Sequence s0 + lane; none behind the last.
template <bool TREE>
__device__ __forceinline__ Seq lane_seq(const PagedAttnParams &p, int s0) {
    const int s = s0 + (threadIdx.x & 31);
    return s < p.n_seq ? load_seq<TREE>(p, s, blockIdx.x == 0) : Seq{0, 0, 0};
}

// One head's cost of the lanes' sequences and their blocks: a lane a sequence;
// sequences of several blocks by the whole warp, a lane a block.
template <int ROWS, int KEYS, bool TREE>
__device__ __forceinline__ long long lane_costs(const PagedAttnParams &p, const Seq &q, int &nb) {
    const int lane = threadIdx.x & 31;
    nb = (q.n * p.rep + ROWS - 1) / ROWS;
    long long cost = nb == 1 ? block_cost<ROWS, KEYS, TREE>(p, q, 0, 1) : 0;
    if constexpr (TREE) {   // every block has the whole sequence's keys
        if (nb > 1) cost = (long long)nb * block_cost<ROWS, KEYS, TREE>(p, q, 0, 1);
    }
    for (unsigned many = TREE ? 0u : __ballot_sync(0xffffffffu, nb > 1); many; many &= many - 1) {
        const int from = __ffs(many) - 1;
        const Seq w{__shfl_sync(0xffffffffu, q.q0, from), __shfl_sync(0xffffffffu, q.n, from),
                    __shfl_sync(0xffffffffu, q.kv, from)};
        const int wnb = __shfl_sync(0xffffffffu, nb, from);
        long long c = 0;
        for (int b = 0; b < wnb; b += 32)
            c += __reduce_add_sync(0xffffffffu, (unsigned)block_cost<ROWS, KEYS, TREE>(p, w, b + lane, wnb));
        if (lane == from) cost = c;
    }
    return cost;
}

// inclusive sums over the warp
template <typename T>
__device__ __forceinline__ T warp_scan(T v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T t = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += t;
    }
    return v;
}

// The CTA's share [x0, x1) of the row of tiles and the unit that x0 lies in.
// cum: shared memory for n_seq + 2 sums (batches of more than 64 sequences; up
// to that every warp finds its share by itself, with two sequences a lane, which took 0.6 us less for
// 48 of them); ctas: CTAs that take a share.
// Called by every thread of the CTA; false where there is nothing for it to do.
// Units of no more than WHOLE tiles on average are not cut for the sake of more
// CTAs, since joining the parts takes as long as some tiles; others may be, down to
// MIN tiles a CTA.
template <int ROWS, int KEYS, int WHOLE, int MIN, bool TREE>
__device__ __forceinline__ bool find_share(const PagedAttnParams &p, long long *cum, Unit<ROWS, KEYS, TREE> &u,
                                           long long &total, int &ctas, long long &x0, long long &x1) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const bool few = p.n_seq <= 64 && p.small;
    long long units, cost = 0;
    int sum = 0;                     // few: of the costs up to this lane's sequence and with it
    int cost2 = 0, sum2 = 0;         // of sequence 32 + lane
    Seq q, q2{0, 0, 0};
    if (few) {
        q = lane_seq<TREE>(p, 0);
        if (p.n_seq > 32) q2 = lane_seq<TREE>(p, 32);
        int nb;
        cost = lane_costs<ROWS, KEYS, TREE>(p, q, nb);
        sum = warp_scan((int)cost);
        int all = __shfl_sync(0xffffffffu, sum, 31);
        units = __reduce_add_sync(0xffffffffu, nb);
        if (p.n_seq > 32) {
            cost2 = (int)lane_costs<ROWS, KEYS, TREE>(p, q2, nb);
            sum2 = all + warp_scan(cost2);
            all = __shfl_sync(0xffffffffu, sum2, 31);
            units += __reduce_add_sync(0xffffffffu, nb);
        }
        total = all;
    } else {
        long long &shared_units = cum[p.n_seq + 1];   // of one head of every sequence
        if (threadIdx.x == 0) shared_units = 0;
        __syncthreads();
        for (int s0 = warp * 32; s0 < p.n_seq; s0 += warps * 32) {
            int nb;
            q = lane_seq<TREE>(p, s0);
            const long long c = lane_costs<ROWS, KEYS, TREE>(p, q, nb);
            if (s0 + lane < p.n_seq) cum[s0 + lane + 1] = c;
            const int n = __reduce_add_sync(0xffffffffu, nb);
            if (lane == 0) atomicAdd(reinterpret_cast<unsigned long long *>(&shared_units), (unsigned long long)n);
        }
        __syncthreads();
        if (warp == 0) {   // inclusive sums, 32 sequences at a time
            long long run = 0;
            for (int s = 0; s < p.n_seq; s += 32) {
                const long long v = warp_scan(s + lane < p.n_seq ? cum[s + lane + 1] : 0ll);
                if (s + lane < p.n_seq) cum[s + lane + 1] = run + v;
                run += __shfl_sync(0xffffffffu, v, 31);
            }
            if (lane == 0) cum[0] = 0;
        }
        __syncthreads();
        total = cum[p.n_seq];
        units = shared_units;
    }
    total *= p.G;
    if (total == 0) return false;
    units *= p.G;
    // (never more CTAs than tiles, so that every share holds one)
    ctas = (int)min((long long)gridDim.x, total <= (WHOLE + u.COST) * units ? units : max(units, quick_div(total, MIN)));
    if ((int)blockIdx.x >= ctas) return false;
    x0 = quick_div(total * blockIdx.x, ctas);
    x1 = quick_div(total * (blockIdx.x + 1), ctas);
    long long before;   // one head's cost of the sequences before u.s
    if (few) {
        const unsigned first = __ballot_sync(0xffffffffu, (long long)sum * p.G > x0);
        if (!first) {   // among the sequences from the 33rd on
            q = q2;
            cost = cost2;
            sum = sum2;
        }
        const int a = __ffs(first ? first : __ballot_sync(0xffffffffu, (long long)sum * p.G > x0)) - 1;
        before = __shfl_sync(0xffffffffu, sum - (int)cost, a);
        cost = __shfl_sync(0xffffffffu, (int)cost, a);
        u.s = first ? a : 32 + a;
        u.q = Seq{__shfl_sync(0xffffffffu, q.q0, a), __shfl_sync(0xffffffffu, q.n, a), __shfl_sync(0xffffffffu, q.kv, a)};
    } else {
        int a = 0, b = p.n_seq - 1;   // the sequence with cum[a] * G <= x0 < cum[a + 1] * G
        while (a < b) {
            const int m = (a + b + 1) >> 1;
            if (cum[m] * p.G <= x0) a = m;
            else b = m - 1;
        }
        u.s = a;
        u.q = load_seq<TREE>(p, a, false);
        before = cum[a];
        cost = cum[a + 1] - before;
        __syncthreads();   // cum may be used for something else from here
    }
    const long long rem = x0 - before * p.G;
    u.g = (int)quick_div(rem, cost);
    u.u0 = before * p.G + u.g * cost;
    // the block, a lane each
    u.b = 0;
    const int nb = (u.q.n * p.rep + ROWS - 1) / ROWS;
    if constexpr (TREE) {
        const int c = block_cost<ROWS, KEYS, TREE>(p, u.q, 0, 1);
        u.b = (int)quick_div(x0 - u.u0, c);
        u.u0 += (long long)u.b * c;
    }
    for (int b0 = 0; !TREE && nb > 1; b0 += 32) {
        const int c = block_cost<ROWS, KEYS, TREE>(p, u.q, b0 + lane, nb);
        const int v = warp_scan(c);
        const unsigned in = __ballot_sync(0xffffffffu, u.u0 + v > x0 && c > 0);
        if (in || b0 + 32 >= nb) {
            const int at = in ? __ffs(in) - 1 : 0;
            u.b = b0 + at;
            u.u0 += __shfl_sync(0xffffffffu, v - c, at);
            break;
        }
        u.u0 += __shfl_sync(0xffffffffu, v, 31);
    }
    u.range(p);
    return true;
}

// The CTA whose share position x of `total` lies in.
__device__ __forceinline__ int share_of(long long x, long long total, int ctas) {
    return (int)quick_div((x + 1) * ctas - 1, total);
}

}  // namespace kore
