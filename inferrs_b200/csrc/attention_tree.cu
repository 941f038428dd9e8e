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

// ---- any type and head size: 32-bit arithmetic, eight or 16 rows a CTA, two or four for each warp ----------------------------------------
constexpr int KEYS = 32, WARPS = 4;

// Shared memory: the rows' queries (later the part's sums), a tile of keys and values as they lie in the cache, in rows that start 16 bytes
// off a multiple of 128 (a lane a key: eight lanes' 16 bytes meet all banks), references and denominators.
__host__ __device__ __forceinline__ int padded(int dim) { return (dim + 3) / 4 * 4; }
template <typename T> __host__ __device__ __forceinline__ int row_bytes(int dim) { return (dim * (int)sizeof(T) + 15) / 16 * 16 + 16; }
template <typename T> __host__ __device__ __forceinline__ size_t rows_smem(int dim, int rows) {
    return sizeof(float) * (size_t)(rows * padded(dim) + 2 * rows + KEYS * rows) + 2 * (size_t)KEYS * row_bytes<T>(dim);
}

__device__ __forceinline__ float4 four(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 four(const __nv_bfloat16* p) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u));
}

// What bounds it are the warps' own chains of instructions (a tile takes one about 8,000 cycles for some 2,000 instructions), so what counts is
// how many share an SM: one tile of shared memory a CTA, not two (41 requests of 2,000 keys, 32 heads on 8, eight rows, when that was changed:
// 355 us, with two 443), and eight rows a CTA where there are no more or few CTAs (with eight and with sixteen: 41 requests of 2,000 keys 245 and
// 386 us; 2 trees of 13 over up to 777 26.5 and 29; 2 trees of 64 over up to 1,000 with 64 heads 262 and 200).  Four groups of warps with a tile
// each in one CTA, where there are few pairs, were slower below some 4,000 keys (1 request of 300 keys 21.5 us, 14.7 as it is; of 9,000 115 and 142).
// Loops of 16 as they stand below took 3 to 5 % off loops of 8 and 4 (41 requests 238 us, 2 trees of 13 25.8).  PER numbers of a head per lane, four
// neighbours where that is a multiple of four.
template <typename T, int PER, int ROWS>
__global__ void __launch_bounds__(WARPS * 32) tree_rows_kernel(const Args A, int parts, bool wide) {
    constexpr int MINE = ROWS / WARPS, SIDE = PER <= 4 ? 4 : 16 / PER;
    extern __shared__ __align__(16) unsigned char raw[];
    const int d = A.dim, dp = padded(d), rb = row_bytes<T>(d);
    float* sq = reinterpret_cast<float*>(raw);    // [ROWS][dp], later the part's sums
    float* sml = sq + ROWS * dp;                  // [2][ROWS]
    float* sp = sml + 2 * ROWS;                   // [WARPS][KEYS][MINE]: the softmax's numbers
    unsigned char* tile = reinterpret_cast<unsigned char*>(sp + KEYS * ROWS);     // [keys, values][KEYS][rb]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int b = blockIdx.x;
    const int part = b % parts;
    b /= parts;
    const int row_tile = b % A.tiles_of_rows;
    b /= A.tiles_of_rows;
    const int head = b % A.n_kv, req = b / A.n_kv;
    const Span S = span_of(A, req);
    const int group = A.group;
    const int first_row = row_tile * ROWS, rows = S.n_tree * group - first_row;
    if (rows <= 0) return;                        // (the whole cluster leaves)
    const int used = rows < ROWS ? rows : ROWS;

    // the warp's rows: their tokens, and the first key that each sees (and any of the tile's)
    int token[MINE], lo[MINE], lo_min = 0x7fffffff;
#pragma unroll
    for (int r = 0; r < MINE; ++r) {
        const int at = first_row + warp * MINE + r;
        token[r] = warp * MINE + r < used ? at / group : -1;
        lo[r] = token[r] >= 0 ? first_key(A, S, token[r]) : 0;
    }
    if (A.span == 0) lo_min = 0;
    else
#pragma unroll 1
    for (int t = first_row / group; t <= (first_row + used - 1) / group; ++t) lo_min = min(lo_min, first_key(A, S, t));
    lo_min = min(lo_min, S.context);              // (the drafted tokens are looked at in any case)
    const int t0 = lo_min / KEYS, n_tiles = (S.keys + KEYS - 1) / KEYS - t0;
    const int begin = t0 + n_tiles * part / parts, end = t0 + n_tiles * (part + 1) / parts;       // (fewer than 2^26 tiles)
    const int* bt = A.table + (long)req * A.max_pages;
    auto look_up = [&](int t) -> long {           // where this lane's key of a tile lies
        const int j = t * KEYS + lane;
        if (t >= end || j >= S.keys) return -1;
        const int slot = A.page_shift >= 0 ? j >> A.page_shift : j / A.page_size, page = bt[slot];
        return page >= 0 && page < A.n_pages ? ((long)page * A.n_kv + head) * A.page_size + j - slot * A.page_size : -1;
    };
    auto load = [&](long at) {                    // a warp brings every fourth of the tile's keys
#pragma unroll 1
        for (int i = 0; i < KEYS / WARPS; ++i) {
            const int key = i * WARPS + warp;
            const long from = __shfl_sync(0xffffffffu, at, key);
            const T* k = static_cast<const T*>(A.k) + (from < 0 ? 0 : from) * d;
            const T* v = static_cast<const T*>(A.v) + (from < 0 ? 0 : from) * d;
            unsigned char *to_k = tile + key * rb, *to_v = to_k + KEYS * rb;
            if (wide) {
#pragma unroll 1
                for (int c = lane; c < d * (int)sizeof(T) / 16; c += 32) {
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((unsigned)__cvta_generic_to_shared(to_k + c * 16)),
                                 "l"(reinterpret_cast<const uint4*>(k) + c), "r"(from < 0 ? 0 : 16) : "memory");
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((unsigned)__cvta_generic_to_shared(to_v + c * 16)),
                                 "l"(reinterpret_cast<const uint4*>(v) + c), "r"(from < 0 ? 0 : 16) : "memory");
                }
            } else {
#pragma unroll 1
                for (int e = lane; e < dp; e += 32) {
                    const bool some = from >= 0 && e < d;
                    reinterpret_cast<T*>(to_k)[e] = some ? k[e] : ib_from_float<T>(0.0f);
                    reinterpret_cast<T*>(to_v)[e] = some ? v[e] : ib_from_float<T>(0.0f);
                }
            }
        }
    };
    long at = look_up(begin), at_next = look_up(begin + 1);
    load(at);
    const T* q = static_cast<const T*>(A.q);
#pragma unroll 1
    for (int i = warp; i < ROWS; i += WARPS) {
        const int row = first_row + i, tok = row / group;
        const T* from = q + ((long)(S.row0 + tok) * A.n_heads + head * group + row - tok * group) * d;
#pragma unroll 1
        for (int e = lane; e < dp; e += 32) sq[i * dp + e] = i < used && e < d ? ib_to_float(from[e]) * A.scale_log2 : 0.0f;
    }

    float acc[MINE][PER], m[MINE], l[MINE];
#pragma unroll
    for (int r = 0; r < MINE; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; ++i) acc[r][i] = 0.0f;
    }
    // number i of this lane
    auto number = [&](int i) { return PER % 4 == 0 ? (i / 4) * 128 + lane * 4 + i % 4 : lane + 32 * i; };
    for (int t = begin; t < end; ++t) {
        const int j = t * KEYS + lane;            // every lane's own key
        const long next = at_next;
        at_next = look_up(t + 2);
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncthreads();
        const T* sk = reinterpret_cast<const T*>(tile + lane * rb);
        float dot[MINE];
#pragma unroll
        for (int r = 0; r < MINE; ++r) dot[r] = 0.0f;
#pragma unroll 16
        for (int e = 0; e < dp; e += 4) {
            const float4 kk = four(sk + e);
#pragma unroll
            for (int r = 0; r < MINE; ++r) {
                const float4 qq = four(sq + (warp * MINE + r) * dp + e);
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
        float* mine = sp + warp * KEYS * MINE;    // (one look gives a key's numbers of all the warp's rows)
#pragma unroll
        for (int r = 0; r < MINE; ++r) mine[lane * MINE + r] = p[r];
        __syncwarp();
#pragma unroll 16
        for (int key = 0; key < KEYS; ++key) {
            const T* sv = reinterpret_cast<const T*>(tile + (KEYS + key) * rb);
            float pk[MINE];
            if constexpr (MINE == 4) {
                const float4 v = four(mine + key * 4);
                pk[0] = v.x; pk[1] = v.y; pk[2] = v.z; pk[3] = v.w;
            } else {
                const float2 v = *reinterpret_cast<const float2*>(mine + key * 2);
                pk[0] = v.x; pk[1] = v.y;
            }
            float x[PER];
            if constexpr (PER % 4 == 0) {
#pragma unroll
                for (int i = 0; i < PER; i += 4) {
                    const float4 v = number(i) < d ? four(sv + number(i)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w;
                }
            } else {
#pragma unroll
                for (int i = 0; i < PER; ++i) x[i] = number(i) < d ? ib_to_float(sv[number(i)]) : 0.0f;
            }
#pragma unroll
            for (int r = 0; r < MINE; ++r)
                if (pk[r] != 0.0f) {              // (the same for the warp; what a row does not see cannot reach it)
#pragma unroll
                    for (int i = 0; i < PER; ++i) acc[r][i] = fmaf(pk[r], x[i], acc[r][i]);
                }
        }
        at = next;
        __syncthreads();                          // the tile has been read
        if (t + 1 < end) load(next);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    // join the parts: each CTA writes every parts-th row
    __syncthreads();
#pragma unroll
    for (int r = 0; r < MINE; ++r) {
        const int row = warp * MINE + r;
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (number(i) < d) sq[row * dp + number(i)] = acc[r][i];
        if (lane == 0) { sml[row] = m[r]; sml[ROWS + row] = l[r]; }
    }
    if (parts > 1) ib_cluster_sync(); else __syncthreads();
#pragma unroll 1
    for (int row = part + warp * parts; row < used; row += WARPS * parts) {
        // a lane looks at a part's reference and denominator, then all look at some parts' sums at once: a look into another CTA takes 700 cycles
        const float mc = lane < parts ? ib_cluster_f32(&sml[row], lane) : -INFINITY, lc = lane < parts ? ib_cluster_f32(&sml[ROWS + row], lane) : 0.0f;
        const float top = ib_warp_max(mc), ref = top == -INFINITY ? 0.0f : top;
        const float f = lc == 0.0f ? 0.0f : exp2f(mc - ref);           // (0: this part of the keys holds none that the row sees)
        const float total = ib_warp_sum(lc * f);
        float o[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) o[i] = 0.0f;
#pragma unroll 1
        for (int c = 0; c < parts; c += SIDE) {
            float v[SIDE][PER];
#pragma unroll
            for (int k = 0; k < SIDE; ++k)
#pragma unroll
                for (int i = 0; i < PER; ++i) v[k][i] = c + k < parts && number(i) < d ? ib_cluster_f32(&sq[row * dp + number(i)], c + k) : 0.0f;
#pragma unroll
            for (int k = 0; k < SIDE; ++k) {
                const float fc = __shfl_sync(0xffffffffu, f, c + k);
#pragma unroll
                for (int i = 0; i < PER; ++i) o[i] = fmaf(v[k][i], fc, o[i]);
            }
        }
        const int at = first_row + row, tok = at / group;
        T* dst = static_cast<T*>(A.out) + (long)(S.row0 + tok) * A.out_ld + (long)(head * group + at - tok * group) * d;
        const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (number(i) < d) dst[number(i)] = ib_from_float<T>(o[i] * inv);
    }
    if (parts > 1) ib_cluster_sync();                // nobody leaves while others read its sums
}

template <typename T, int PER, int ROWS>
static int launch_rows(Args A, int max_tree, int max_keys, cudaStream_t stream) {
    static IbDeviceSet done;
    if (const int code = ib_allow_dynamic_smem(done, tree_rows_kernel<T, PER, ROWS>, rows_smem<T>(32 * PER, ROWS))) return code;
    A.tiles_of_rows = (int)(((long)max_tree * A.group + ROWS - 1) / ROWS);
    const long pairs = (long)A.n_requests * A.n_kv * A.tiles_of_rows;
    int parts = 1;       // about ten CTAs an SM, two or more that run and as many that follow them
    while (parts < IB_MAX_CLUSTER && pairs * parts * 2 <= 10 * 148 && max_keys >= 2 * KEYS * parts * 2) parts *= 2;
    const bool wide = (reinterpret_cast<uintptr_t>(A.k) | reinterpret_cast<uintptr_t>(A.v) | (uintptr_t)(A.dim * sizeof(T))) % 16 == 0;
    return launch_cluster(tree_rows_kernel<T, PER, ROWS>, pairs * parts, parts, WARPS * 32, rows_smem<T>(A.dim, ROWS), stream, A, parts, wide);
}

template <typename T, int PER>
static int rows_of_heads(const Args& A, int max_tree, int max_keys, cudaStream_t stream) {
    const long rows = (long)max_tree * A.group;
    const bool few = rows <= 8 || (long)A.n_requests * A.n_kv * ((rows + 7) / 8) <= 148;
    return few ? launch_rows<T, PER, 8>(A, max_tree, max_keys, stream) : launch_rows<T, PER, 16>(A, max_tree, max_keys, stream);
}

template <typename T>
static int rows_of_type(const Args& A, int max_tree, int max_keys, cudaStream_t stream) {
    const int per = (A.dim + 31) / 32;
    if (per <= 2) return rows_of_heads<T, 2>(A, max_tree, max_keys, stream);
    if (per <= 4) return rows_of_heads<T, 4>(A, max_tree, max_keys, stream);
    if (per <= 8) return rows_of_heads<T, 8>(A, max_tree, max_keys, stream);
    return rows_of_heads<T, 16>(A, max_tree, max_keys, stream);
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
    A.q = c.q;
    A.k = c.n_pages ? c.k : c.q;      // (a cache without pages: nothing is read, but copies of no bytes want an address)
    A.v = c.n_pages ? c.v : c.q;
    A.table = c.table; A.q_start = c.q_start; A.context = c.context; A.positions = c.positions; A.seen = c.seen;
    A.out = c.out;
    A.out_ld = c.out_ld;
    A.n_rows = c.n_requests && c.max_tree ? (int)c.n_rows : 0;
    A.n_requests = (int)c.n_requests; A.n_heads = (int)c.n_heads; A.n_kv = (int)c.n_kv; A.dim = (int)c.dim;
    A.max_pages = (int)c.max_pages; A.page_size = (int)c.page_size; A.n_pages = (int)c.n_pages; A.words = (int)c.words;
    A.span = (int)(c.span > 0x7fffffffL ? 0x7fffffffL : c.span < -0x7fffffffL ? -0x7fffffffL : c.span);       // (wider than any context)
    A.page_shift = (c.page_size & (c.page_size - 1)) == 0 ? __builtin_ctzl(c.page_size) : -1;
    A.group = A.n_heads / A.n_kv;
    A.group_shift = (A.group & (A.group - 1)) == 0 ? __builtin_ctz((unsigned)A.group) : -1;
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
