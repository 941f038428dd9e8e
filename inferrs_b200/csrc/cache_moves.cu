// Moving what the paged cache holds, in all layers at once: whole pages (a request is forked), and tokens that are kept while
// others between them go (the path of a tree of drafted tokens, a context that is thinned out).
//
// Both kernels move bytes and know nothing of numbers: a tensor is [outer, pages, page], a page [heads, places, vector].  What
// they cannot do without is each byte read once and written once, and that bounds both where there is much to move: 512 pages of 32 KB
// in 72 planes take 356 us (6.8 TB/s of reads and writes), 1,000 of 2,000 tokens of four requests in 72 planes of 8 heads 207 (5.7 TB/s).
#include "common.cuh"

namespace moves {

struct Pages {
    unsigned char* base;
    long outer, n_pages, page_bytes;     // the tensor [outer][n_pages][page_bytes]
};

// A CTA for 2 units a thread of one page in one plane (512 pages as above, 1 page: with 1 unit 407 and 2.3 us, 2: 356 and 2.2, 4: 361 and 2.2,
// 8: 361 and 2.7).  Source and target pages are different ones, so no CTA reads what another one writes.
template <typename U, int N>
__global__ void __launch_bounds__(256) copy_pages_kernel(Pages P, const int* __restrict__ source, const int* __restrict__ target,
                                                         int n_pairs, int chunks) {
    const long page_units = P.page_bytes / (long)sizeof(U);
    const long at = blockIdx.x / chunks;
    const int chunk = (int)(blockIdx.x - at * chunks);
    const int pair = (int)(at % n_pairs);
    const long outer = at / n_pairs;
    const int from = source[pair], to = target[pair];
    if (from < 0 || to < 0 || from >= P.n_pages || to >= P.n_pages || from == to) return;
    const U* src = reinterpret_cast<const U*>(P.base) + (outer * P.n_pages + from) * page_units;
    U* dst = reinterpret_cast<U*>(P.base) + (outer * P.n_pages + to) * page_units;
    U held[N];
    const long first = (long)chunk * (256 * N) + threadIdx.x;
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (first + i * 256 < page_units) held[i] = src[first + i * 256];
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (first + i * 256 < page_units) dst[first + i * 256] = held[i];
}

// Token kept[r, i] behind context[r] goes to place context[r] + i.  The places are ascending, so a token never moves back and
// never beyond one that follows it: chunk by chunk, with all loads of a chunk ahead of its stores, nothing is overwritten before
// it has been read (a chunk's stores end below the places that the next chunk reads).  One CTA for one or several heads of one
// request in one plane, so chunks of the same vectors never run at once.  Two units a thread and chunk: the 1,000 tokens as above and 5 of 16 of eight
// requests take 205 and 5.9 us with two, 207 and 7.4 with four, 300 and 15.3 with eight (a chunk waits for its own loads).
template <typename U, int N>
__global__ void __launch_bounds__(256) keep_tokens_kernel(Pages P, int heads, int places, int shift, int units, int together,      // log2: of the places or -1, of a CTA's heads
                                                          const int* __restrict__ table, int max_pages,
                                                          const int* __restrict__ context, const int* __restrict__ kept,
                                                          int max_kept, const int* __restrict__ n_kept) {
    const int r = blockIdx.z, head0 = blockIdx.y << together;
    const long outer = blockIdx.x;
    int n = n_kept[r];
    n = n < max_kept ? n : max_kept;
    const long first = context[r];
    const int per = units < (int)blockDim.x ? units : (int)blockDim.x;       // threads that share a vector
    const int step = blockDim.x / per;                                       // vectors that the CTA takes side by side
    const int mine = threadIdx.x / per;
    U* plane = reinterpret_cast<U*>(P.base) + outer * P.n_pages * heads * places * units;
    const int* bt = table + (long)r * max_pages;
    auto vector_at = [&](int head, long place) -> int {                      // a vector's place in the plane, -1: there is no page
        if (place < 0 || place > 0x7fffffffL) return -1;
        const int slot = shift >= 0 ? (int)place >> shift : (int)place / places;
        if (slot >= max_pages) return -1;
        const int page = bt[slot];
        return page >= 0 && page < P.n_pages ? (page * heads + head) * places + ((int)place - slot * places) : -1;
    };
    for (int unit0 = 0; unit0 < units; unit0 += per) {
        const int unit = unit0 + (int)(threadIdx.x - mine * per);
        const bool some = mine < step && unit < units;
        // a chunk's places are looked up while the chunk before it is on its way
        auto look_up = [&](int i0, int (&from)[N], int (&to)[N]) {
#pragma unroll
            for (int k = 0; k < N; ++k) {
                const int q = i0 + k * step + mine, i = q >> together, head = head0 + (q & ((1 << together) - 1));
                from[k] = to[k] = -1;
                if (!some || i >= n) continue;
                const int old = kept[(long)r * max_kept + i];
                if (old == i) continue;
                from[k] = vector_at(head, first + old);
                to[k] = vector_at(head, first + i);
            }
        };
        int from[N], to[N];
        look_up(0, from, to);
        for (int i0 = 0; i0 < n << together; i0 += step * N) {
            U held[N];
#pragma unroll
            for (int k = 0; k < N; ++k)
                if (from[k] >= 0 && to[k] >= 0) held[k] = plane[(long)from[k] * units + unit];
            int from_next[N], to_next[N];
            look_up(i0 + step * N, from_next, to_next);
            __syncthreads();
#pragma unroll
            for (int k = 0; k < N; ++k) {
                if (from[k] >= 0 && to[k] >= 0) plane[(long)to[k] * units + unit] = held[k];
                from[k] = from_next[k];
                to[k] = to_next[k];
            }
        }
        __syncthreads();
    }
}

// the widest unit that both the address and the length are a multiple of
static int unit_of(const void* p, long bytes) {
    const unsigned long long a = (unsigned long long)p | (unsigned long long)bytes;
    for (int u = 16; u > 1; u /= 2)
        if (a % u == 0) return u;
    return 1;
}

}  // namespace moves

using namespace moves;

struct IbCopyPages {
    unsigned char* base;
    const int *source, *target;
    cudaStream_t stream;
    long outer, n_pages, page_bytes, n_pairs;
};

template <typename U>
static int copy_pages_as(const IbCopyPages& a) {
    const Pages P{a.base, a.outer, a.n_pages, a.page_bytes};
    const long units = a.page_bytes / (long)sizeof(U), pages = a.outer * a.n_pairs;
    const long chunks = (units + 256 * 2 - 1) / (256 * 2);
    if (pages * chunks > 0x7fffffffL) return IB_ERR_UNSUPPORTED;
    copy_pages_kernel<U, 2><<<(unsigned)(pages * chunks), 256, 0, a.stream>>>(P, a.source, a.target, (int)a.n_pairs, (int)chunks);
    return ib_launch_status();
}

IB_EXPORT int ib_copy_pages(const void* call) {
    const IbCopyPages a = *static_cast<const IbCopyPages*>(call);
    if (a.outer < 0 || a.n_pages < 0 || a.page_bytes < 0 || a.n_pairs < 0 || a.n_pairs > 0x7fffffffL) return IB_ERR_ARGUMENT;
    if (a.outer == 0 || a.n_pages == 0 || a.page_bytes == 0 || a.n_pairs == 0) return IB_OK;
    switch (unit_of(a.base, a.page_bytes)) {
        case 16: return copy_pages_as<uint4>(a);
        case 8: return copy_pages_as<uint2>(a);
        case 4: return copy_pages_as<unsigned>(a);
        case 2: return copy_pages_as<unsigned short>(a);
        default: return copy_pages_as<unsigned char>(a);
    }
}

struct IbKeepTokens {
    unsigned char* base;
    const int *table, *context, *kept, *n_kept;
    cudaStream_t stream;
    long outer, n_pages, heads, places, vector_bytes, requests, max_pages, max_kept;
};

template <typename U>
static int keep_tokens_as(const IbKeepTokens& a) {
    const int units = (int)(a.vector_bytes / (long)sizeof(U));
    const Pages P{a.base, a.outer, a.n_pages, a.heads * a.places * a.vector_bytes};
    // Heads in one CTA: as many as make up for short lists, while there are two CTAs for every SM.  (72 planes of 8 heads, 1, 2, 4, 8 heads a
    // CTA: 5 tokens of 8 requests 6.0, 6.1, 4.6, 4.0 us; of one request 2.6, 2.5, 2.8, 3.3; 40 tokens of 8 requests 16.1, 13.9, 14.7, 14.5.)
    int together = 0;
    while (a.heads % (2L << together) == 0 && a.max_kept * units << together < 1024 && a.outer * (a.heads >> together) * a.requests >= 2 * 2 * 148) ++together;
    const dim3 grid((unsigned)a.outer, (unsigned)(a.heads >> together), (unsigned)a.requests);
    int threads = 256;
    while (threads > 32 && (long)(threads / 2) >= a.max_kept * units << together) threads /= 2;
    const int shift = (a.places & (a.places - 1)) == 0 ? __builtin_ctzl(a.places) : -1;
    keep_tokens_kernel<U, 2><<<grid, threads, 0, a.stream>>>(P, (int)a.heads, (int)a.places, shift, units, together, a.table, (int)a.max_pages, a.context,
                                                             a.kept, (int)a.max_kept, a.n_kept);
    return ib_launch_status();
}

IB_EXPORT int ib_keep_tokens(const void* call) {
    const IbKeepTokens a = *static_cast<const IbKeepTokens*>(call);
    if (a.outer < 0 || a.n_pages < 0 || a.heads < 0 || a.places <= 0 || a.vector_bytes < 0 || a.requests < 0 || a.max_pages < 0 || a.max_kept < 0)
        return IB_ERR_ARGUMENT;
    if (a.outer == 0 || a.n_pages == 0 || a.heads == 0 || a.vector_bytes == 0 || a.requests == 0 || a.max_pages == 0 || a.max_kept == 0) return IB_OK;
    if (a.max_kept > 0x7fffffffL / 64) return IB_ERR_UNSUPPORTED;
    if (a.outer > 0x7fffffffL || a.heads > 65535 || a.requests > 65535 || a.places > 0x7fffffffL || a.vector_bytes > 0x7fffffffL
        || a.n_pages * a.heads * a.places > 0x7fffffffL) return IB_ERR_UNSUPPORTED;
    switch (unit_of(a.base, a.vector_bytes)) {
        case 16: return keep_tokens_as<uint4>(a);
        case 8: return keep_tokens_as<uint2>(a);
        case 4: return keep_tokens_as<unsigned>(a);
        case 2: return keep_tokens_as<unsigned short>(a);
        default: return keep_tokens_as<unsigned char>(a);
    }
}
