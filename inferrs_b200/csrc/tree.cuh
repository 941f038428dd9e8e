// What the kernels for attention of drafted tokens share (attention_tree.cu says what they compute).
#pragma once

#include "clusters.cuh"

namespace tree {

struct Args {
    const void *q, *k, *v;
    const int *table, *q_start, *context, *positions, *seen;
    void* out;
    long out_ld;
    int n_rows, n_requests, n_heads, n_kv, dim, max_pages, page_size, n_pages, words, span, tiles_of_rows;
    int page_shift;            // log2 of the page size, -1: it is no power of two
    int group, group_shift;    // query heads of a key/value head, their log2 or -1
    float scale_log2;          // scale * log2(e)
};

// a request's rows, keys and drafted tokens
struct Span {
    int row0, n_tree, context, keys;
};
__device__ __forceinline__ Span span_of(const Args& A, int req) {
    Span s;
    const int a = A.q_start[req], b = A.q_start[req + 1];
    s.row0 = a < 0 ? 0 : a;
    const int end = b < A.n_rows ? b : A.n_rows;
    s.n_tree = end > s.row0 ? end - s.row0 : 0;
    const int c = A.context[req];
    s.context = c < 0 ? 0 : c;
    const long room = (long)A.max_pages * A.page_size;      // places beyond the block table hold no keys
    if (s.context > room) s.context = (int)room;
    const long all = (long)s.context + s.n_tree;
    s.keys = (int)(all < room ? all : room);
    return s;
}

__device__ __forceinline__ int first_key(const Args& A, const Span& s, int token) {
    return A.span == 0 ? 0 : ib_first_visible(A.positions[s.row0 + token], A.span);
}

// bits j .. j + 31 of a row's mask, where bits below 0 and from n_tree on are not set
__device__ __forceinline__ unsigned mask_bits(const Args& A, const Span& s, const int* row_words, int j) {
    const int at = j >> 5, shift = j & 31;        // (an arithmetic shift: rounds down)
    const unsigned a = at >= 0 && at < A.words ? (unsigned)row_words[at] : 0u;
    const unsigned b = shift && at + 1 >= 0 && at + 1 < A.words ? (unsigned)row_words[at + 1] : 0u;
    unsigned bits = __funnelshift_r(a, b, shift);
    const int left = s.n_tree - j;
    if (left < 32) bits &= left <= 0 ? 0u : (1u << left) - 1u;
    return bits;
}

template <typename... KArgs, typename... Given>
static int launch_cluster(void (*kernel)(KArgs...), long ctas, int cluster, int threads, size_t smem, cudaStream_t stream, Given... args) {
    if (ctas > 0x7fffffffL) return IB_ERR_UNSUPPORTED;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 1 : 0;
    cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
    return ib_launch_status();
}

}  // namespace tree

struct IbTreeAttention {
    const void *q, *k, *v;
    const int *table, *q_start, *context, *positions, *seen;
    void* out;
    void* workspace;           // of ib_paged_attention_tree_workspace bytes
    cudaStream_t stream;
    long f32, out_ld, n_rows, n_requests, n_heads, n_kv, dim, max_pages, page_size, n_pages, words, span, max_tree, max_keys;
    double scale;
};

// Heads of 64 or 128 numbers in bfloat16 (attention_tree_tcgen05.cu): IB_ERR_UNSUPPORTED where it does not take the call; if
// asked, the bytes of workspace that the call needs (nothing is launched), else what the launch says.
long ib_tree_tcgen05(tree::Args A, int max_tree, int max_keys, void* workspace, bool ask, cudaStream_t stream);
