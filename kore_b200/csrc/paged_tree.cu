// paged_tree.cu — trees of drafted tokens beside the attention: each token's ancestors and
// position, the branch that a model accepts, and its rows moved together in the caches of all
// layers (sm_100a).
//
// A sequence's chunk is a tree (or several): parent[i] < i is a token's parent in the chunk, -1
// a token without one. Token i sees its ancestors and itself: bits of its mask. Its position is
// kv - n + (its depth), its slot that of kv - n + i.
// accept: from token 0 on, the first child whose token is the model's choice behind its parent.
// move: the accepted tokens path[0] < path[1] < ... stand at kv - n + path[j] and go to kv - n + j.
//   path[j] >= j, so a row's old place is written by no token before it in the path: a thread
//   that takes its 16 bytes of every row in the path's order may read all of them first. Nobody else may move
//   the same rows, so keys and values that are one memory are one pool.
//
// Masks and acceptance are chains of dependent looks (some tens of ns each, in shared memory). The move is bound by
// HBM for large batches and by its chain (path, page table, row) for small ones: 16 bytes of a thread at every accepted
// row, eight rows on their way at once. Acceptance and move together: 4.5 us for a sequence, 24 layers of 2 heads of 64
// in f16; 11.1 for 64 sequences of up to 24 tokens, 28 layers of 4 heads of 128 in bf16 (17 MB, 2.6 us of HBM; 8.8 out
// of L2).

#include "paged_values.cuh"

namespace kore {
namespace {

constexpr unsigned FULL = 0xffffffffu;

// The sequence's bounds; n = -1 where they do not fit.
__device__ __forceinline__ Seq tree_seq(const TreeParams &p, int s, bool report) {
    Seq q;
    q.q0 = __ldg(p.q_start + s);
    q.n = __ldg(p.q_start + s + 1) - q.q0;
    q.kv = __ldg(p.kv_len + s);
    if (q.n != 0 && (q.n < 0 || q.q0 < 0 || q.q0 > p.n_tok - q.n || q.kv < q.n || q.kv > p.cap || q.n > p.most)) {
        if (report) raise_error(p.status, DEV_BAD_SEQUENCE);
        q.n = -1;
    }
    return q;
}

// A CTA a sequence, a thread a token: the way up the parents, which stand in shared memory, goes to ever
// lower bits. The tokens of a chunk longer than the masks see nothing and have no position, so that a store leaves
// them out: what stood there may be another step's.
__global__ void __launch_bounds__(128) tree_mask_kernel(const __grid_constant__ TreeParams p) {
    grid_dep_wait();
    grid_dep_launch();
    __shared__ int parent[kPagedMaxTree];
    const Seq q = tree_seq(p, blockIdx.x, threadIdx.x == 0);
    if (q.n < 0) {
        const int n = __ldg(p.q_start + blockIdx.x + 1) - q.q0;
        if (n <= p.most || q.q0 < 0 || q.q0 > p.n_tok - n || q.kv < n) return;   // its rows are no chunk's
        for (int i = threadIdx.x; i < n; i += blockDim.x) {
            for (int y = 0; y < p.words; ++y) p.mask[(long long)(q.q0 + i) * p.words + y] = 0;
            p.pos[q.q0 + i] = -1;
        }
        return;
    }
    for (int i = threadIdx.x; i < q.n; i += blockDim.x) parent[i] = __ldg(p.parent + q.q0 + i);
    __syncthreads();
    for (int i = threadIdx.x; i < q.n; i += blockDim.x) {
        uint32_t *row = p.mask + (long long)(q.q0 + i) * p.words;
        int x = i, depth = 0, w = p.words - 1;
        uint32_t bits = 0;
        for (;;) {
            while (w > x >> 5) {   // words above the next ancestor's
                row[w--] = bits;
                bits = 0;
            }
            bits |= 1u << (x & 31);
            const int up = parent[x];
            if (up == -1) break;
            if (up < -1 || up >= x) {   // no tree: the token is left out
                raise_error(p.status, DEV_BAD_SEQUENCE);
                depth = -1;
                break;
            }
            x = up;
            ++depth;
        }
        while (w >= 0) {
            row[w--] = bits;
            bits = 0;
        }
        if (depth < 0)
            for (int y = 0; y < p.words; ++y) row[y] = 0;
        p.pos[q.q0 + i] = depth < 0 ? -1 : q.kv - q.n + depth;
    }
}

// A warp a sequence; trees of up to kNear tokens are walked in shared memory.
constexpr int kNear = 256;
__global__ void __launch_bounds__(128) accept_kernel(const __grid_constant__ TreeParams p) {
    grid_dep_wait();
    grid_dep_launch();
    const int lane = threadIdx.x & 31, s = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (s >= p.n_seq) return;
    __shared__ int near[4][3][kNear];
    Seq q = tree_seq(p, s, lane == 0);
    int *path = p.path + (long long)s * p.path_stride;
    int count = 0, now = 0, next = -1;
    if (q.n > 0) {
        const int *parent = p.parent + q.q0, *token = p.token + q.q0, *choice = p.choice + q.q0;
        if (q.n <= kNear) {
            int(*to)[kNear] = near[threadIdx.x >> 5];
            for (int i = lane; i < q.n; i += 32) {
                to[0][i] = __ldg(parent + i);
                to[1][i] = __ldg(token + i);
                to[2][i] = __ldg(choice + i);
            }
            __syncwarp();
            parent = to[0];
            token = to[1];
            choice = to[2];
        }
        if (parent[0] != -1) {   // masks and store have left out token 0, and all behind it
            if (lane == 0) raise_error(p.status, DEV_BAD_SEQUENCE);
            q.n = -1;
        }
        while (q.n > 0) {
            if (lane == 0) path[count] = now;
            ++count;
            next = choice[now];
            if (count == p.path_stride) break;
            int child = -1;
            for (int i0 = now + 1; i0 < q.n; i0 += 32) {
                const int i = i0 + lane;
                const unsigned hit = __ballot_sync(FULL, i < q.n && parent[i] == now && token[i] == next);
                if (hit) {
                    child = i0 + __ffs(hit) - 1;
                    break;
                }
            }
            if (child < 0) break;
            now = child;
        }
    }
    for (int j = count + lane; j < p.path_stride; j += 32) path[j] = -1;
    if (lane == 0) {
        p.count[s] = count;
        p.next[s] = next;
        // A sequence without tokens keeps all it has; one of no positions either may be one that a plan left out (it
        // writes 0 then), whose request holds some: 0 would end it.
        p.kept[s] = q.n < 0 || (q.n == 0 && q.kv == 0) ? -1 : q.kv - q.n + count;
    }
}

// A CTA some layers of a sequence. rows: (from, to) offsets of the rows that move, in 16-byte pieces.
__global__ void __launch_bounds__(256) commit_kernel(const __grid_constant__ CommitParams p) {
    extern __shared__ longlong2 rows[];
    __shared__ int bad;
    const int s = blockIdx.y, tid = threadIdx.x;
    if (tid == 0) bad = 0;
    __syncthreads();
    grid_dep_wait();
    grid_dep_launch();
    const int q0 = __ldg(p.q_start + s), n = __ldg(p.q_start + s + 1) - q0, kv = __ldg(p.kv_len + s), m = __ldg(p.count + s);
    if (n == 0 || m <= 0) return;
    const int *path = p.path + (long long)s * p.path_stride;
    bool fits = n > 0 && kv >= n && kv <= (long long)p.table_stride * p.P && m <= n && m <= p.path_stride;
    int code = DEV_BAD_SEQUENCE;
    if (fits) {
        const int *pt = p.page_table + (long long)s * p.table_stride;
        for (int j = tid; j < m; j += blockDim.x) {
            const int x = __ldg(path + j);
            if (x < j || x >= n || (j > 0 && x <= __ldg(path + j - 1))) {
                fits = false;
                break;
            }
            const int a = kv - n + x, b = kv - n + j, pa = p.by_page.div(a), pb = p.by_page.div(b);
            const int from = __ldg(pt + pa), to = __ldg(pt + pb);
            if (from < 0 || from >= p.n_pages || to < 0 || to >= p.n_pages) {
                fits = false;
                code = DEV_BAD_PAGE;
                break;
            }
            rows[j] = longlong2{from * p.page_pieces + (long long)p.by_page.mod(a, pa) * p.row_pieces,
                                to * p.page_pieces + (long long)p.by_page.mod(b, pb) * p.row_pieces};
        }
    }
    if (!fits) {
        bad = 1;
        if (blockIdx.x == 0) raise_error(p.status, code);
    }
    __syncthreads();
    if (bad) return;
    // rows up to the first that moves stay where they are (path[j] == j up to it, and not behind it)
    int j0 = 0;
    while (j0 < m && rows[j0].x == rows[j0].y) ++j0;
    if (j0 == m) return;
    const int head = p.P * p.row_pieces, layer = p.G * p.row_pieces;   // pieces from head to head, of a token
    const int all = p.n_layers * 2 * layer;
    for (int x = blockIdx.x * blockDim.x + tid; x < all; x += gridDim.x * blockDim.x) {
        const int l = x / layer, y = x - l * layer, g = y / p.row_pieces;
        void *pool = (l & 1) ? p.v[l >> 1] : p.k[l >> 1];
        if (!pool) continue;
        uint4 *base = static_cast<uint4 *>(pool) + (long long)g * head + (y - g * p.row_pieces);
        for (int j = j0; j < m; j += 8) {
            uint4 v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (j + k < m) v[k] = base[rows[j + k].x];
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (j + k < m) base[rows[j + k].y] = v[k];
        }
    }
}

}  // namespace

cudaError_t launch_tree_mask(const TreeParams &p, cudaStream_t s) { return launch(tree_mask_kernel, p.n_seq, 128, 0, s, p); }

cudaError_t launch_accept(const TreeParams &p, cudaStream_t s) { return launch(accept_kernel, (p.n_seq + 3) / 4, 128, 0, s, p); }

cudaError_t launch_commit(const CommitParams &p, cudaStream_t s) {
    const int all = p.n_layers * 2 * p.G * p.row_pieces;
    const size_t smem = (size_t)p.path_stride * sizeof(longlong2);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((all + 255) / 256 < 32 ? (all + 255) / 256 : 32, p.n_seq);
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, commit_kernel, p);
}

}  // namespace kore
