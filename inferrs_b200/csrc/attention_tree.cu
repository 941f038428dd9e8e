// Attention of a tree of drafted tokens over the paged cache.
//
// Request r holds context[r] keys; its rows q_start[r] .. q_start[r + 1] - 1 of the step are drafted tokens, and the i-th of them
// has its key and value at place context[r] + i.  A row sees the context from ib_first_visible(position, span) on, and of the
// drafted tokens those whose bit is set in its mask (bit j % 32 of word j / 32): itself and its ancestors, or what else the mask
// says.  o = sum_j p_j v_j with p the softmax over those keys of scale q . k_j; a row that sees none gets zeros.  A key whose
// page is not in the cache is none.
//
// All heads of a key/value head's group and all tokens of the tree share what they read of the cache, so the rows of a tile are
// (token, head of the group) pairs, counted token by token.  The keys are cut into as many parts as the machine has room for:
// the CTAs of a cluster take one each and join their sums through distributed shared memory, in the order of the parts.
#include "tree.cuh"

namespace tree {

// ---- any type and head size: 32-bit arithmetic, 16 rows a CTA, four for each warp ----------------------------------------
constexpr int ROWS = 16, KEYS = 32, WARPS = 4, MINE = ROWS / WARPS;

__host__ __device__ __forceinline__ int padded(int dim) { return (dim + 3) / 4 * 4; }
__host__ __device__ __forceinline__ size_t rows_smem(int dim) {
    return sizeof(float) * (size_t)(ROWS * padded(dim) + KEYS * (padded(dim) + 4) + KEYS * padded(dim) + 2 * ROWS);
}

template <typename T, int PER>       // PER numbers of a head per lane
__global__ void __launch_bounds__(WARPS * 32) tree_rows_kernel(const Args A, int parts) {
    extern __shared__ __align__(16) float smem[];
    const int d = A.dim, dp = padded(d);
    float* sq = smem;                             // [ROWS][dp], later the part's sums
    float* sk = sq + ROWS * dp;                   // [KEYS][dp + 4]
    float* sv = sk + KEYS * (dp + 4);             // [KEYS][dp]
    float* sml = sv + KEYS * dp;                  // [2][ROWS]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int b = blockIdx.x;
    const int part = b % parts;
    b /= parts;
    const int row_tile = b % A.tiles_of_rows;
    b /= A.tiles_of_rows;
    const int head = b % A.n_kv, req = b / A.n_kv;
    const Span S = span_of(A, req);
    const int group = A.n_heads / A.n_kv;
    const int first_row = row_tile * ROWS, rows = S.n_tree * group - first_row;
    if (rows <= 0) return;                        // (the whole cluster leaves)
    const int used = rows < ROWS ? rows : ROWS;

    const T* q = static_cast<const T*>(A.q);
    for (int i = tid; i < ROWS * dp; i += WARPS * 32) {
        const int r = i / dp, e = i - r * dp;
        float x = 0.0f;
        if (r < used && e < d) {
            const int at = first_row + r, token = at / group;
            x = ib_to_float(q[((long)(S.row0 + token) * A.n_heads + head * group + at - token * group) * d + e]) * A.scale_log2;
        }
        sq[i] = x;
    }
    // the warp's rows: their tokens, and the first key that each sees (and any of the tile's)
    int token[MINE], lo[MINE], lo_min = 0x7fffffff;
#pragma unroll
    for (int r = 0; r < MINE; ++r) {
        const int at = first_row + warp * MINE + r;
        token[r] = warp * MINE + r < used ? at / group : -1;
        lo[r] = token[r] >= 0 ? first_key(A, S, token[r]) : 0;
    }
    for (int t = first_row / group; t <= (first_row + used - 1) / group; ++t) lo_min = min(lo_min, first_key(A, S, t));
    lo_min = min(lo_min, S.context);              // (the drafted tokens are looked at in any case)
    const int t0 = lo_min / KEYS, n_tiles = (S.keys + KEYS - 1) / KEYS - t0;
    const int begin = t0 + (int)((long)n_tiles * part / parts), end = t0 + (int)((long)n_tiles * (part + 1) / parts);

    float acc[MINE][PER], m[MINE], l[MINE];
#pragma unroll
    for (int r = 0; r < MINE; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; ++i) acc[r][i] = 0.0f;
    }
    const int* bt = A.table + (long)req * A.max_pages;
    for (int t = begin; t < end; ++t) {
        const int j = t * KEYS + lane;            // every lane's own key
        long at = -1;
        if (j < S.keys) {
            const int page = bt[j / A.page_size];
            if (page >= 0 && page < A.n_pages) at = ((long)page * A.n_kv + head) * A.page_size + j % A.page_size;
        }
        __syncthreads();                          // the tile before has been read
        for (int i = 0; i < KEYS / WARPS; ++i) {
            const int key = warp * (KEYS / WARPS) + i;
            const long from = __shfl_sync(0xffffffffu, at, key);
            for (int e = lane; e < dp; e += 32) {
                const bool some = from >= 0 && e < d;
                sk[key * (dp + 4) + e] = some ? ib_to_float(static_cast<const T*>(A.k)[from * d + e]) : 0.0f;
                sv[key * dp + e] = some ? ib_to_float(static_cast<const T*>(A.v)[from * d + e]) : 0.0f;
            }
        }
        __syncthreads();
        float dot[MINE];
#pragma unroll
        for (int r = 0; r < MINE; ++r) dot[r] = 0.0f;
        for (int e = 0; e < dp; e += 4) {
            const float4 kk = *reinterpret_cast<const float4*>(sk + lane * (dp + 4) + e);
#pragma unroll
            for (int r = 0; r < MINE; ++r) {
                const float4 qq = *reinterpret_cast<const float4*>(sq + (warp * MINE + r) * dp + e);
                dot[r] = fmaf(qq.x, kk.x, fmaf(qq.y, kk.y, fmaf(qq.z, kk.z, fmaf(qq.w, kk.w, dot[r]))));
            }
        }
        float p[MINE];
#pragma unroll
        for (int r = 0; r < MINE; ++r) {
            bool sees = token[r] >= 0 && at >= 0;
            if (sees) {
                if (j < S.context) sees = j >= lo[r];
                else sees = mask_bits(A, S, A.seen + (long)(S.row0 + token[r]) * A.words, j - S.context) & 1u;
            }
            const float x = sees ? dot[r] : -INFINITY;
            const float to = fmaxf(m[r], ib_warp_max(x));
            const float ref = to == -INFINITY ? 0.0f : to;
            p[r] = sees ? exp2f(x - ref) : 0.0f;
            const float c = exp2f(m[r] - ref);    // (of minus infinity: 0)
            l[r] = l[r] * c + ib_warp_sum(p[r]);
#pragma unroll
            for (int i = 0; i < PER; ++i) acc[r][i] *= c;
            m[r] = to;
        }
        for (int key = 0; key < KEYS; ++key) {
            float pk[MINE];
#pragma unroll
            for (int r = 0; r < MINE; ++r) pk[r] = __shfl_sync(0xffffffffu, p[r], key);
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int e = lane + 32 * i;
                if (e >= d) continue;
                const float x = sv[key * dp + e];
#pragma unroll
                for (int r = 0; r < MINE; ++r)
                    if (pk[r] != 0.0f) acc[r][i] = fmaf(pk[r], x, acc[r][i]);      // what a row does not see cannot reach it
            }
        }
    }
    // join the parts: each CTA writes every parts-th row
    __syncthreads();
#pragma unroll
    for (int r = 0; r < MINE; ++r) {
        const int row = warp * MINE + r;
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (lane + 32 * i < d) sq[row * dp + lane + 32 * i] = acc[r][i];
        if (lane == 0) { sml[row] = m[r]; sml[ROWS + row] = l[r]; }
    }
    if (parts > 1) cluster_sync(); else __syncthreads();
    for (int row = part + warp * parts; row < used; row += WARPS * parts) {
        float top = -INFINITY, total = 0.0f;
        for (int c = 0; c < parts; ++c) top = fmaxf(top, remote_f32(&sml[row], c));
        const float ref = top == -INFINITY ? 0.0f : top;
        float o[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) o[i] = 0.0f;
        for (int c = 0; c < parts; ++c) {
            const float lc = remote_f32(&sml[ROWS + row], c);
            if (lc == 0.0f) continue;             // this part of the keys holds none that the row sees
            const float f = exp2f(remote_f32(&sml[row], c) - ref);
            total = fmaf(lc, f, total);
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (lane + 32 * i < d) o[i] = fmaf(remote_f32(&sq[row * dp + lane + 32 * i], c), f, o[i]);
        }
        const int at = first_row + row, tok = at / group;
        T* dst = static_cast<T*>(A.out) + (long)(S.row0 + tok) * A.out_ld + (long)(head * group + at - tok * group) * d;
        const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (lane + 32 * i < d) dst[lane + 32 * i] = ib_from_float<T>(o[i] * inv);
    }
    if (parts > 1) cluster_sync();                // nobody leaves while others read its sums
}

template <typename T, int PER>
static int launch_rows(const Args& A, int max_keys, cudaStream_t stream) {
    static IbDeviceSet done;
    const size_t smem = rows_smem(A.dim);
    if (smem > 48 * 1024) {
        const int code = ib_allow_dynamic_smem(done, tree_rows_kernel<T, PER>, rows_smem(32 * PER));
        if (code != IB_OK) return code;
    }
    const long pairs = (long)A.n_requests * A.n_kv * A.tiles_of_rows;
    int parts = 1;
    while (parts < MAX_CLUSTER && pairs * parts * 2 <= 592 && max_keys >= 2 * KEYS * parts * 2) parts *= 2;
    return launch_cluster(tree_rows_kernel<T, PER>, pairs * parts, parts, WARPS * 32, smem, stream, A, parts);
}

template <typename T>
static int rows_of_type(Args A, int max_tree, int max_keys, cudaStream_t stream) {
    A.tiles_of_rows = (int)(((long)max_tree * (A.n_heads / A.n_kv) + ROWS - 1) / ROWS);
    const int per = (A.dim + 31) / 32;
    if (per <= 1) return launch_rows<T, 1>(A, max_keys, stream);
    if (per <= 2) return launch_rows<T, 2>(A, max_keys, stream);
    if (per <= 3) return launch_rows<T, 3>(A, max_keys, stream);
    if (per <= 4) return launch_rows<T, 4>(A, max_keys, stream);
    if (per <= 6) return launch_rows<T, 6>(A, max_keys, stream);
    if (per <= 8) return launch_rows<T, 8>(A, max_keys, stream);
    return launch_rows<T, 16>(A, max_keys, stream);
}

}  // namespace tree

// A refusal, or IB_OK and the arguments as the kernels take them (n_rows 0: there is nothing to do)
static int tree_args(const IbTreeAttention& c, tree::Args& A, int& max_tree, int& max_keys) {
    if (c.n_rows < 0 || c.n_requests < 0 || c.n_kv <= 0 || c.n_heads <= 0 || c.n_heads % c.n_kv || c.dim <= 0 || c.page_size <= 0 || c.max_tree < 0
        || c.max_pages < 0 || c.n_pages < 0 || c.words < 0)
        return IB_ERR_ARGUMENT;
    if (c.dim > 512 || c.n_rows * c.n_heads > 0x7fffffffL || c.n_requests > 0x7fffffffL || c.max_pages * c.page_size > 0x7fffffffL
        || c.n_pages * c.n_kv * c.page_size > 0x7fffffffL)
        return IB_ERR_UNSUPPORTED;
    A.q = c.q; A.k = c.k; A.v = c.v;
    A.table = c.table; A.q_start = c.q_start; A.context = c.context; A.positions = c.positions; A.seen = c.seen;
    A.out = c.out;
    A.out_ld = c.out_ld;
    A.n_rows = c.n_requests && c.max_tree ? (int)c.n_rows : 0;
    A.n_requests = (int)c.n_requests; A.n_heads = (int)c.n_heads; A.n_kv = (int)c.n_kv; A.dim = (int)c.dim;
    A.max_pages = (int)c.max_pages; A.page_size = (int)c.page_size; A.n_pages = (int)c.n_pages; A.words = (int)c.words; A.span = (int)c.span;
    A.page_shift = (c.page_size & (c.page_size - 1)) == 0 ? __builtin_ctzl(c.page_size) : -1;
    A.scale_log2 = (float)(c.scale * 1.4426950408889634);
    max_tree = (int)(c.max_tree < c.n_rows ? c.max_tree : c.n_rows);
    max_keys = (int)(c.max_keys < 0x3fffffffL ? c.max_keys : 0x3fffffffL);
    return IB_OK;
}

// the bytes of workspace that a call needs (0: none), or a refusal
IB_EXPORT long ib_paged_attention_tree_workspace(const void* call) {
    const IbTreeAttention c = *static_cast<const IbTreeAttention*>(call);
    tree::Args A;
    int max_tree, max_keys;
    if (const int code = tree_args(c, A, max_tree, max_keys)) return code;
    if (A.n_rows == 0 || c.f32) return 0;
    const long bytes = ib_tree_tcgen05(A, max_tree, max_keys, nullptr, true, c.stream);
    return bytes == IB_ERR_UNSUPPORTED ? 0 : bytes;
}

IB_EXPORT int ib_paged_attention_tree(const void* call) {
    const IbTreeAttention c = *static_cast<const IbTreeAttention*>(call);
    tree::Args A;
    int max_tree, max_keys;
    if (const int code = tree_args(c, A, max_tree, max_keys)) return code;
    if (A.n_rows == 0) return IB_OK;
    if (!c.f32) {
        const long code = ib_tree_tcgen05(A, max_tree, max_keys, c.workspace, false, c.stream);
        if (code != IB_ERR_UNSUPPORTED) return (int)code;
    }
    return c.f32 ? tree::rows_of_type<float>(A, max_tree, max_keys, c.stream) : tree::rows_of_type<__nv_bfloat16>(A, max_tree, max_keys, c.stream);
}
