// paged_plan.cu — a step's page tables, slots and positions from its requests'
// lengths, and pages given back (sm_100a).
//
// plan: base_s = length[request_s], kv_s = base_s + n_s; sequence s wants
//   need_s = ceil(kv_s / P) - ceil(base_s / P) pages, which it takes in turn from the
//   end of the free list: its j-th is free[n_free - 1 - (need_0 + .. + need_{s-1}) - j].
//   Rows stand one behind the other: q_start is the running sum of n, and token t of
//   sequence s at position p = base_s + t - q_start_s has the slot page(p / P) * P + p % P.
// trim: pages behind ceil(keep_s / P) go back to the list's end, in the order in which
//   taking them again would hand them out.
//
// Two running sums and then writes: no arithmetic to speak of, some tens of KB, so a
// call's time is its chain (requests, lengths, sums, pages). One cluster: every CTA forms the sums
// of the whole batch for itself (4096 sequences are eight a thread), writes its share of tokens
// and tables from the state as it was, and only behind the cluster's barrier does the state change;
// a second launch for the writes, or a pass over counters in memory, would take longer than the sums do.
// A plan and a trim together: 8.4 us for 32 requests of 63 pages, 15.2 for 500 trees of up to 24 tokens with
// their masks, 14.2 for 96 prompts of 100000 tokens (1.2 MB, which HBM would take in 0.2 us: a launch of a
// cluster of sixteen is some 2 us of each, the chain of loads 2 to 3).

#include "paged_values.cuh"

namespace kore {
namespace {

constexpr unsigned FULL = 0xffffffffu;
constexpr int kPlanThreads = 512;   // of a CTA at most
constexpr int kPlanWarps = kPlanThreads / 32;

__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

// Inclusive sums of a and b over the block, on top of what came before (run_a, run_b: updated).
__device__ __forceinline__ void block_scan(long long &a, long long &b, longlong2 (&part)[kPlanWarps + 1], long long &run_a, long long &run_b) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    a = warp_scan(a);
    b = warp_scan(b);
    if (lane == 31) part[warp + 1] = make_longlong2(a, b);
    __syncthreads();
    // (every warp sums up the warps' totals for itself)
    longlong2 w = lane < warps ? part[lane + 1] : make_longlong2(0, 0);
    w.x = warp_scan(w.x);
    w.y = warp_scan(w.y);
    const int from = warp ? warp - 1 : 0;
    const long long xa = __shfl_sync(FULL, w.x, from), xb = __shfl_sync(FULL, w.y, from);
    a += run_a + (warp ? xa : 0);
    b += run_b + (warp ? xb : 0);
    run_a += __shfl_sync(FULL, w.x, 31);
    run_b += __shfl_sync(FULL, w.y, 31);
}

// ceil(n / P) for 0 <= n
__device__ __forceinline__ int pages_of(const PlanParams &p, int n) {
    const int q = p.by_page.div(n);
    return q + (p.by_page.mod(n, q) != 0);
}

template <bool TRIM>
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const __grid_constant__ PlanParams p) {
    extern __shared__ int smem[];
    __shared__ longlong2 part[kPlanWarps + 1];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int words = (p.n_requests + 31) / 32;
    // requests named by the batch, and those named twice
    unsigned *seen = reinterpret_cast<unsigned *>(smem), *twice = seen + words;
    int *end = smem + 2 * words;       // plan: rows up to the sequence's last; trim: pages up to its last
    int *base = end + p.n_seq;         // positions it holds; trim: pages that stay
    int *first = base + p.n_seq;       // plan: its first new page's place in the order, less the pages it has
    int *who = first + p.n_seq;        // its request; -1: it is left out
    for (int i = tid; i < 2 * words; i += blockDim.x) seen[i] = 0;
    __syncthreads();
    grid_dep_wait();
    grid_dep_launch();
    // the first sequences' requests, and what is known of them, are on their way before anything else
    const long long cap = min((long long)p.stride * p.P, 0x7fffffffll);
    auto known = [&](int r) { return r >= 0 && r < p.n_requests; };
    const int listed = *p.n_free;
    int r = tid < p.n_seq ? __ldg(p.request + tid) : -1, a = tid < p.n_seq ? __ldg(p.amount + tid) : 0;
    int len = known(r) ? p.length[r] : 0;
    auto mark = [&](int x) {
        if (known(x) && (atomicOr(seen + (x >> 5), 1u << (x & 31)) >> (x & 31) & 1)) atomicOr(twice + (x >> 5), 1u << (x & 31));
    };
    mark(r);
    for (int s = tid + blockDim.x; s < p.n_seq; s += blockDim.x) mark(__ldg(p.request + s));
    const bool list_ok = listed >= 0 && listed <= p.n_pages;
    const int n_free = list_ok ? listed : 0;
    const bool report = blockIdx.x == 0;
    if (report && tid == 0 && !list_ok) raise_error(p.status, DEV_BAD_SEQUENCE);
    __syncthreads();

    long long rows_run = 0, pages_run = 0;
    for (int s0 = 0; s0 < p.n_seq; s0 += blockDim.x) {
        const int s = s0 + tid;
        if (s0 > 0) {
            r = s < p.n_seq ? __ldg(p.request + s) : -1;
            a = s < p.n_seq ? __ldg(p.amount + s) : 0;
            len = known(r) ? p.length[r] : 0;
            __syncthreads();   // part may be written again
        }
        const bool asked = r >= 0;
        int code = 0;
        if (!asked) a = 0;
        if (asked && (!known(r) || (twice[r >> 5] >> (r & 31) & 1) || len < 0 || len > cap)) code = DEV_BAD_SEQUENCE;
        // (what a trim of a request that holds nothing is asked to keep of it makes no difference)
        if (asked && a < 0 && (!TRIM || len != 0)) code = DEV_BAD_SEQUENCE;
        if (a < 0) a = 0;
        if constexpr (!TRIM) {
            // Sums of rows and of pages at once: the pages of sequences whose rows do not fit count too, but behind the
            // first of these no sequence has rows that do. (One without rows fits wherever it stands.)
            if (asked && !code && (long long)len + a > cap) code = DEV_BAD_SEQUENCE;
            const int have = code ? 0 : pages_of(p, len);
            const long long mine = asked && !code ? pages_of(p, len + a) - have : 0;
            long long rows = a, need = mine;
            block_scan(rows, need, part, rows_run, pages_run);
            if (asked && !code && a > 0 && rows > p.n_tok) code = DEV_BAD_SEQUENCE;
            if (!code && mine > 0 && need > n_free) code = DEV_NO_PAGES;
            if (s < p.n_seq) {
                end[s] = (int)min(rows, 0x7fffffffll);
                base[s] = len;
                first[s] = (int)(need - mine) - have;   // (of a served sequence; its sum fits)
                who[s] = code ? -1 : r;
            }
        } else {
            const bool cut = asked && !code && a < len;
            const int stay = cut ? pages_of(p, a) : 0;
            const long long mine = cut ? pages_of(p, len) - stay : 0;
            long long gone = mine, unused = 0;
            block_scan(gone, unused, part, pages_run, rows_run);
            if (s < p.n_seq) {
                end[s] = (int)min(gone, 0x7fffffffll);
                base[s] = stay;
                first[s] = (int)mine;
                who[s] = cut ? r : -1;
            }
        }
        if (code && report) raise_error(p.status, code);
    }
    __syncthreads();

    const int warps = gridDim.x * (blockDim.x >> 5), w = blockIdx.x * (blockDim.x >> 5) + warp;
    // a warp some of a sequence's pages, four of them a lane on their way at once
    const int split = p.n_seq ? max(1, min(32, warps / p.n_seq)) : 1;
    constexpr int N = 4;
    if constexpr (TRIM) {
        const bool fits = list_ok && pages_run <= p.n_pages - n_free;   // (else a page was given back that none held)
        if (!fits && report && tid == 0) raise_error(p.status, DEV_BAD_SEQUENCE);
        if (fits) {
            const int top = n_free + (int)pages_run - 1;
            for (int x = w; x < p.n_seq * split; x += warps) {
                const int s = x / split;
                if (who[s] < 0) continue;
                int *row = p.table + (long long)who[s] * p.stride + base[s];
                const int n = first[s], at = end[s] - n;
                for (int j = (x - s * split) * 32 + lane; j < n; j += 32 * split * N) {
                    int page[N];
#pragma unroll
                    for (int k = 0; k < N; ++k)
                        if (j + k * 32 * split < n) page[k] = row[j + k * 32 * split];
#pragma unroll
                    for (int k = 0; k < N; ++k) {
                        const int i = j + k * 32 * split;
                        if (i >= n) continue;
                        p.free_pages[top - at - i] = page[k];
                        row[i] = -1;
                    }
                }
            }
        }
        cluster_barrier();   // every CTA has read the state
        if (blockIdx.x != 0 || !fits) return;
        for (int s = tid; s < p.n_seq; s += blockDim.x)
            if (who[s] >= 0) p.length[who[s]] = __ldg(p.amount + s);
        if (tid == 0) *p.n_free = n_free + (int)pages_run;
        return;
    } else {
        auto page_of = [&](int s, int have, int j) -> int {
            return j < have ? p.table[(long long)who[s] * p.stride + j] : p.free_pages[n_free - 1 - (first[s] + j)];
        };
        // tables
        for (int x = w; x < p.n_seq * split; x += warps) {
            const int s = x / split;
            if (who[s] < 0) continue;
            const int have = pages_of(p, base[s]), want = pages_of(p, base[s] + end[s] - (s ? end[s - 1] : 0));
            int *out = p.page_table + (long long)s * p.out_stride, *row = p.table + (long long)who[s] * p.stride;
            for (int j = (x - s * split) * 32 + lane; j < want; j += 32 * split * N) {
                int page[N];
#pragma unroll
                for (int k = 0; k < N; ++k)
                    if (j + k * 32 * split < want) page[k] = page_of(s, have, j + k * 32 * split);
#pragma unroll
                for (int k = 0; k < N; ++k) {
                    const int i = j + k * 32 * split;
                    if (i >= want) continue;
                    out[i] = page[k];
                    if (i >= have) row[i] = page[k];
                }
            }
        }
        // tokens: a warp a run of them
        const int each = ((p.n_tok + warps - 1) / warps + 31) / 32 * 32;
        const long long t0 = (long long)w * each;
        if (t0 < p.n_tok) {
            int s = 0, b = p.n_seq;   // the first sequence that ends behind t0
            while (s < b) {
                const int m = (s + b) >> 1;
                if (end[m] <= t0) s = m + 1;
                else b = m;
            }
            const int t1 = (int)min((long long)p.n_tok, t0 + each);
            for (int t = (int)t0 + lane; t < t1; t += 32 * N) {
                int pos[N], page[N], in[N];   // (in: place in the page)
#pragma unroll
                for (int k = 0; k < N; ++k) {
                    const int x = t + 32 * k;
                    pos[k] = -1;
                    if (x >= t1) continue;
                    while (s < p.n_seq && end[s] <= x) ++s;
                    if (s >= p.n_seq || who[s] < 0) continue;
                    pos[k] = base[s] + x - (s ? end[s - 1] : 0);
                    const int j = p.by_page.div(pos[k]);
                    in[k] = p.by_page.mod(pos[k], j);
                    page[k] = page_of(s, pages_of(p, base[s]), j);
                }
#pragma unroll
                for (int k = 0; k < N; ++k) {
                    const int x = t + 32 * k;
                    if (x >= t1) continue;
                    p.slots[x] = pos[k] < 0 ? -1ll : (long long)page[k] * p.P + in[k];
                    p.pos[x] = pos[k];
                }
            }
        }
        cluster_barrier();   // every CTA has read the state
        if (blockIdx.x != 0) return;
        long long taken = 0;
        for (int s = tid; s < p.n_seq; s += blockDim.x) {
            const int from = s ? end[s - 1] : 0;
            p.q_start[s + 1] = end[s];
            const int kv = base[s] + end[s] - from;
            p.kv_len[s] = who[s] >= 0 ? kv : 0;
            if (who[s] >= 0) {
                p.length[who[s]] = kv;
                const int have = pages_of(p, base[s]), want = pages_of(p, kv);
                if (want > have) taken = max(taken, (long long)first[s] + want);
            }
        }
        // (those that get pages are the first ones of those that want some)
        taken = __reduce_max_sync(FULL, (int)taken);
        if (lane == 0) part[warp].x = taken;
        __syncthreads();
        if (tid == 0) {
            for (int i = 1; i < (int)(blockDim.x >> 5); ++i) taken = max(taken, part[i].x);
            p.q_start[0] = 0;
            if (list_ok) *p.n_free = n_free - (int)taken;
        }
    }
}

template <bool TRIM>
cudaError_t launch_p(const PlanParams &p, int ctas, int threads, cudaStream_t s) {
    const size_t smem = (size_t)((p.n_requests + 31) / 32) * 8 + (size_t)p.n_seq * 16;
    constexpr int most = kPagedMaxRequests / 32 * 8 + kPagedMaxSeqs * 16;
    static_assert(most <= 227 * 1024, "shared memory of an SM");
    if (cudaError_t e = ensure_smem_limit(reinterpret_cast<const void *>(plan_kernel<TRIM>), most)) return e;
    if (ctas > 8)
        if (cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void *>(plan_kernel<TRIM>), cudaFuncAttributeNonPortableClusterSizeAllowed, 1)) return e;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = ctas;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, plan_kernel<TRIM>, p);
}

}  // namespace

cudaError_t launch_plan(const PlanParams &p, bool trim, cudaStream_t s) {
    // A portable cluster of small CTAs, or one of sixteen for many tokens, sequences or table entries. Plan and
    // trim, 8 x 256 against 16 x 512 threads, us: 32 requests of 63 pages 8.5 / 9.1; 500 of up to 251 pages 27.2 / 15.3;
    // 96 with 100000 tokens 28.7 / 14.1. Near the borders: a token for 128, 240, 264 requests of 63, 63, 16 pages 9.5 / 9.3,
    // 11.4 / 9.4, 14.0 / 10.1; 64 requests of 251 pages 10.1 / 9.3; 16 prompts of 120, 136 tokens 7.7 / 7.6, 8.1 / 7.6; one
    // of 2048, 4096 tokens 7.3 / 7.5, 7.6 / 7.4. (So the smaller ones lose up to 2 us just below the borders.)
    const bool large = p.n_tok > 2048 || p.n_seq > 256 || (long long)p.n_seq * p.stride > 16384;
    const int ctas = large ? 16 : 8, threads = large ? kPlanThreads : 256;
    return trim ? launch_p<true>(p, ctas, threads, s) : launch_p<false>(p, ctas, threads, s);
}

}  // namespace kore
