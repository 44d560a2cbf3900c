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
// of the whole batch for itself (4096 sequences are four a thread), writes its share of tokens
// and tables from the state as it was, and only behind the cluster's barrier does the state change;
// a second launch for the writes, or a pass over counters in memory, would take longer than the sums do.

#include "paged_values.cuh"

namespace kore {
namespace {

constexpr unsigned FULL = 0xffffffffu;

__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

// Inclusive sums of a and b over the block, on top of what came before (run_a, run_b: updated).
__device__ __forceinline__ void block_scan(long long &a, long long (&part)[33], long long &run) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    a = warp_scan(a);
    if (lane == 31) part[warp] = a;
    __syncthreads();
    if (warp == 0) {
        const long long w = warp_scan(lane < warps ? part[lane] : 0ll);
        __syncwarp();
        part[lane + 1] = w;
        if (lane == 0) part[0] = 0;
    }
    __syncthreads();
    a += run + part[warp];
    run += part[warps];
    __syncthreads();   // part may be written again
}

// ceil(n / P) for 0 <= n
__device__ __forceinline__ int pages_of(const PlanParams &p, int n) {
    const int q = p.by_page.div(n);
    return q + (p.by_page.mod(n, q) != 0);
}

template <bool TRIM>
__global__ void __launch_bounds__(1024) plan_kernel(const __grid_constant__ PlanParams p) {
    extern __shared__ int smem[];
    __shared__ long long part[33];
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
    for (int s = tid; s < p.n_seq; s += blockDim.x) {
        const int r = __ldg(p.request + s);
        if (r >= 0 && r < p.n_requests && (atomicOr(seen + (r >> 5), 1u << (r & 31)) >> (r & 31) & 1))
            atomicOr(twice + (r >> 5), 1u << (r & 31));
    }
    const int listed = *p.n_free;
    const bool list_ok = listed >= 0 && listed <= p.n_pages;
    const int n_free = list_ok ? listed : 0;
    const long long cap = min((long long)p.stride * p.P, 0x7fffffffll);
    const bool report = blockIdx.x == 0;
    if (report && tid == 0 && !list_ok) raise_error(p.status, DEV_BAD_SEQUENCE);
    __syncthreads();

    long long rows_run = 0, pages_run = 0;
    for (int s0 = 0; s0 < p.n_seq; s0 += blockDim.x) {
        const int s = s0 + tid;
        int r = s < p.n_seq ? __ldg(p.request + s) : -1, code = 0, a = 0, len = 0;
        const bool asked = r >= 0;
        if (asked) {
            a = __ldg(p.amount + s);
            if (r >= p.n_requests || (twice[r >> 5] >> (r & 31) & 1)) code = DEV_BAD_SEQUENCE;
            else if ((len = p.length[r]) < 0 || len > cap) code = DEV_BAD_SEQUENCE;
            if (a < 0) {
                code = DEV_BAD_SEQUENCE;
                a = 0;
            }
        }
        if constexpr (!TRIM) {
            long long rows = a, need = 0;
            block_scan(rows, part, rows_run);
            if (asked && !code && (rows > p.n_tok || (long long)len + a > cap)) code = DEV_BAD_SEQUENCE;
            const int have = code ? 0 : pages_of(p, len);
            if (asked && !code) need = pages_of(p, len + a) - have;
            const bool wants = need > 0;
            const long long mine = need;
            block_scan(need, part, pages_run);
            if (wants && need > n_free) code = DEV_NO_PAGES;
            if (s < p.n_seq) {
                end[s] = (int)min(rows, 0x7fffffffll);
                base[s] = len;
                first[s] = (int)(need - mine) - have;   // (of a served sequence; its sum fits)
                who[s] = code ? -1 : r;
            }
        } else {
            long long gone = 0;
            if (asked && !code && a < len) gone = pages_of(p, len) - pages_of(p, a);
            const long long mine = gone;
            block_scan(gone, part, pages_run);
            if (s < p.n_seq) {
                end[s] = (int)min(gone, 0x7fffffffll);
                base[s] = asked && !code && a < len ? pages_of(p, a) : 0;
                first[s] = (int)mine;
                who[s] = asked && !code && a < len ? r : -1;
            }
        }
        if (code && report) raise_error(p.status, code);
    }
    __syncthreads();

    const int warps = gridDim.x * (blockDim.x >> 5), w = blockIdx.x * (blockDim.x >> 5) + warp;
    if constexpr (TRIM) {
        const bool fits = list_ok && pages_run <= p.n_pages - n_free;   // (else a page was given back that none held)
        if (!fits && report && tid == 0) raise_error(p.status, DEV_BAD_SEQUENCE);
        if (fits) {
            const int top = n_free + (int)pages_run - 1;
            for (int s = w; s < p.n_seq; s += warps) {
                if (who[s] < 0) continue;
                int *row = p.table + (long long)who[s] * p.stride + base[s];
                const int n = first[s], at = end[s] - n;
                for (int j = lane; j < n; j += 32) {
                    p.free_pages[top - at - j] = row[j];
                    row[j] = -1;
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
        // tables: a warp some of a sequence's pages
        const int split = max(1, min(8, warps / max(1, p.n_seq)));
        for (int x = w; x < p.n_seq * split; x += warps) {
            const int s = x / split;
            if (who[s] < 0) continue;
            const int have = pages_of(p, base[s]), want = pages_of(p, base[s] + end[s] - (s ? end[s - 1] : 0));
            int *out = p.page_table + (long long)s * p.out_stride, *row = p.table + (long long)who[s] * p.stride;
            for (int j = (x - s * split) * 32 + lane; j < want; j += 32 * split) {
                const int page = page_of(s, have, j);
                out[j] = page;
                if (j >= have) row[j] = page;
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
            for (int t = (int)t0 + lane; t < t1; t += 32) {
                while (s < p.n_seq && end[s] <= t) ++s;
                long long slot = -1;
                int pos = -1;
                if (s < p.n_seq && who[s] >= 0) {
                    pos = base[s] + t - (s ? end[s - 1] : 0);
                    const int j = p.by_page.div(pos);
                    slot = (long long)page_of(s, pages_of(p, base[s]), j) * p.P + p.by_page.mod(pos, j);
                }
                p.slots[t] = slot;
                p.pos[t] = pos;
            }
        }
        cluster_barrier();   // every CTA has read the state
        if (blockIdx.x != 0) return;
        long long taken = 0;
        for (int s = tid; s < p.n_seq; s += blockDim.x) {
            const int from = s ? end[s - 1] : 0;
            if (s == 0) p.q_start[0] = 0;
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
        if (lane == 0) part[warp] = taken;
        __syncthreads();
        if (tid == 0) {
            for (int i = 1; i < (int)(blockDim.x >> 5); ++i) taken = max(taken, part[i]);
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
    // small batches: one CTA of as many threads as sequences or tokens; else a cluster
    const int n = p.n_tok > p.n_seq ? p.n_tok : p.n_seq;
    int threads = 128;
    while (threads < 1024 && threads < n) threads *= 2;
    const int ctas = n > 1024 ? 8 : 1;
    return trim ? launch_p<true>(p, ctas, threads, s) : launch_p<false>(p, ctas, threads, s);
}

}  // namespace kore
