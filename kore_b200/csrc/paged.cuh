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

constexpr int kPagedMaxSeqs = 4096;      // sequences of one batch
constexpr int kPagedMaxCtas = 160;       // CTAs (SMs) that an attention launch uses at most
constexpr int kPagedRowsMax = 256;       // query rows of a work unit at most
constexpr size_t kPagedZeroed = 1024;    // leading workspace bytes that are zero between calls
constexpr size_t kPagedCutBytes = 32;    // of a cut unit's description

// A tensor of rows of heads: element e of head h of row t at t*ts + h*hs + e.
struct HeadRows {
    const void *in;
    void *out;
    long long in_ts, in_hs, out_ts, out_hs;
    int heads;
    int rotate;
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

struct PagedAttnParams {
    TmaDesc tm_k, tm_v;        // K and V pools as tensor maps (many-row kernel, 16-bit caches)
    const void *k, *v;
    long long page_stride;     // elements
    const int *q_start, *kv_len, *page_table;
    int table_stride, n_seq, n_tok, n_pages, P, H, G, rep;
    const void *q;
    void *out;
    long long q_ts, q_hs, o_ts, o_hs;
    float *lse;
    const float *k_scale, *v_scale;
    float scale;
    int causal, window;
    int q_vec, o_vec;          // q (out) rows are 16-byte aligned
    int box;                   // rows of a tensor-map box
    int *counters;             // [kPagedMaxCtas] zero between calls
    void *cut;                 // [kPagedMaxCtas] units that were cut (many-row kernel)
    float *part;               // [kPagedMaxCtas][2] partial results
    int *status;
};

cudaError_t launch_rope_table(const float *freq, int half, double amp, int n_pos, float *table, cudaStream_t s);
cudaError_t launch_rotate(const RotateParams &p, int in_type, int cache_type, bool vec, cudaStream_t s);
// n_ctas: SMs of the device, at most kPagedMaxCtas
cudaError_t launch_paged_rows(const PagedAttnParams &p, int d, int q_type, int cache_type, int n_ctas, cudaStream_t s);
cudaError_t launch_paged_tiles(const PagedAttnParams &p, int d, int type, int n_ctas, cudaStream_t s);

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

struct Seq {
    int q0, n, kv;
};

// The sequence's bounds; n = 0 (it is left out) where they do not fit.
__device__ __forceinline__ Seq load_seq(const PagedAttnParams &p, int s, bool report) {
    Seq q;
    q.q0 = __ldg(p.q_start + s);
    q.n = __ldg(p.q_start + s + 1) - q.q0;
    q.kv = __ldg(p.kv_len + s);
    if (q.n != 0 && (q.n < 0 || q.q0 < 0 || q.q0 > p.n_tok - q.n || q.kv < 0 ||
                     q.kv > (long long)p.table_stride * p.P)) {
        if (report) raise_error(p.status, DEV_BAD_SEQUENCE);
        q.n = 0;
    }
    return q;
}

// Keys [lo, hi) that some token of the packed rows [r0, r1) of the chunk sees.
__device__ __forceinline__ void key_range(const PagedAttnParams &p, const Seq &q, int r0, int r1, int &lo, int &hi) {
    const int first = q.kv - q.n + r0 / p.rep, last = q.kv - q.n + (r1 - 1) / p.rep;
    hi = p.causal ? min(q.kv, last + 1) : q.kv;
    lo = p.window > 0 ? max(0, first - p.window + 1) : 0;
    hi = max(hi, 0);
    lo = min(lo, hi);
}

template <int ROWS, int KEYS>
struct Unit {
    int s, g, b;           // sequence, KV head, block of rows
    Seq q;
    int rows;              // valid rows of the block
    int lo, hi;            // keys
    int tile0, nt;         // first tile, tiles (1 for a unit without keys)
    long long u0;          // virtual position of the unit's start

    __device__ __forceinline__ int blocks(const PagedAttnParams &p) const { return (q.n * p.rep + ROWS - 1) / ROWS; }
    __device__ __forceinline__ void range(const PagedAttnParams &p) {
        rows = min(ROWS, q.n * p.rep - b * ROWS);
        key_range(p, q, b * ROWS, b * ROWS + rows, lo, hi);
        tile0 = lo / KEYS;
        nt = max(1, (hi + KEYS - 1) / KEYS - tile0);
    }
    // To the next unit; false behind the last one.
    __device__ __forceinline__ bool next(const PagedAttnParams &p) {
        u0 += kUnitCost + nt;
        if (++b == blocks(p)) {
            b = 0;
            if (++g == p.G) {
                g = 0;
                do {
                    if (++s >= p.n_seq) return false;
                    q = load_seq(p, s, false);
                } while (q.n == 0);
            }
        }
        range(p);
        return true;
    }
};

// Cost of one KV head of a sequence, in tiles: summed by one thread.
template <int ROWS, int KEYS>
__device__ __forceinline__ long long seq_cost(const PagedAttnParams &p, const Seq &q) {
    Unit<ROWS, KEYS> u;
    u.q = q;
    long long c = 0;
    const int nb = u.blocks(p);
    for (u.b = 0; u.b < nb; ++u.b) {
        u.range(p);
        c += kUnitCost + u.nt;
    }
    return c;
}

// The CTA's share [x0, x1) of the row of tiles and the unit that x0 lies in.
// cum: shared memory for n_seq + 1 sums; ctas: CTAs that take a share. Called
// by every thread of the CTA; false where there is nothing for it to do.
template <int ROWS, int KEYS>
__device__ __forceinline__ bool find_share(const PagedAttnParams &p, long long *cum, int min_tiles, Unit<ROWS, KEYS> &u,
                                           long long &total, int &ctas, long long &x0, long long &x1) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int s = threadIdx.x; s < p.n_seq; s += blockDim.x) {
        const Seq q = load_seq(p, s, blockIdx.x == 0);
        cum[s + 1] = q.n ? seq_cost<ROWS, KEYS>(p, q) : 0ll;
    }
    __syncthreads();
    if (warp == 0) {   // inclusive sums, 32 sequences at a time
        long long run = 0;
        for (int s = 0; s < p.n_seq; s += 32) {
            long long v = s + lane < p.n_seq ? cum[s + lane + 1] : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long t = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v += t;
            }
            if (s + lane < p.n_seq) cum[s + lane + 1] = run + v;
            run += __shfl_sync(0xffffffffu, v, 31);
        }
        if (lane == 0) cum[0] = 0;
    }
    __syncthreads();
    total = cum[p.n_seq] * p.G;
    if (total == 0) return false;
    // no more CTAs than give each a worthwhile number of tiles; never more than
    // tiles, so that every share holds one
    const long long most = max(1ll, total / min_tiles);
    ctas = (int)min((long long)gridDim.x, most);
    if ((int)blockIdx.x >= ctas) return false;
    x0 = total * blockIdx.x / ctas;
    x1 = total * (blockIdx.x + 1) / ctas;
    int a = 0, b = p.n_seq - 1;   // the sequence with cum[a] * G <= x0 < cum[a + 1] * G
    while (a < b) {
        const int m = (a + b + 1) >> 1;
        if (cum[m] * p.G <= x0) a = m;
        else b = m - 1;
    }
    u.s = a;
    u.q = load_seq(p, a, false);
    const long long cost = cum[a + 1] - cum[a];   // of one head
    const long long rem = x0 - cum[a] * p.G;
    u.g = (int)(rem / cost);
    u.b = 0;
    u.u0 = cum[a] * p.G + u.g * cost;
    u.range(p);
    while (u.u0 + kUnitCost + u.nt <= x0) u.next(p);
    __syncthreads();   // cum may be used for something else from here
    return true;
}

// The CTA whose share position x of `total` lies in.
__device__ __forceinline__ int share_of(long long x, long long total, int ctas) {
    return (int)(((x + 1) * ctas - 1) / total);
}

}  // namespace kore
