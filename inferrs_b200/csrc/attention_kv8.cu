// Attention over paged keys and values in 8 bits: single tokens, and tiles of a prompt's tokens (bfloat16 queries).
//
// A CTA works for one key/value head of one tile of rows and one part of its keys.  The tile's (token, head) pairs are the
// columns of the products (8 NT of them), keys and the numbers of a head their rows, so eight columns cost what one does.
// Each of four warps takes every fourth slice of 16 keys (which lies in one page) through a ring of its own that it fills
// with cp.async, zeros where the tile sees no key whatever the page holds there: no warp waits for another until the end.  What
// bounds it are the warps' own instruction streams, about five cycles an instruction and warp, so sixteen warps share an SM and
// none does more than it must.  A warp that fills the rings of the others cannot keep up (206 instructions for 32 keys: a thousand
// cycles), with TMA neither (165 cycles a box of 16 keys): 64 requests of 2,048 keys, 32 heads on 8 of 128 numbers, 82 and 75 us;
// this form 50, 5.5 TB/s.
//
//   scores   S = K Q^T: codes become f16 pairs exactly (mma.sync has no e4m3 products of its own on this machine: it converts
//            both operands every time, 867 instead of 830 instructions a stage); a query row is multiplied by the power of two that
//            brings its largest number to 2^13 .. 2^14, so f16 holds all of it that counts (2^-38 of the largest).  A lane
//            takes 16 neighbouring numbers of a key row as its part of four products of 16: any order of the numbers
//            serves, if the queries' is the same.  s = acc * key scale * (softmax scale log2 e / the query's power of two).
//   softmax  with a running reference R per column for s + log2(value scale), so that the weights of values of very different
//            scales, 2^(s + log2(value scale) - R), keep their precision in f16; the sum takes 2^(s - R) in float32, which
//            holds it (value scales below 2^-80 count as that for the reference).  It moves only when a number has
//            outgrown it by 2^8 (a vote of the warp says whether any has).
//   values   O = V^T P^T in f16, which holds the codes exactly: two keys' codes are interleaved byte by byte, P is turned with
//            movmatrix; sums in float32.  P is rounded to f16's 11 bits, three more than a bfloat16 result keeps; below 2^-25 of the
//            reference's weight it is lost (the sum, in float32, counts it).
//   no numbers  a key whose scale is not finite has no score (a negative sum times infinity would count as hidden).  Where some
//            column of a tile does not see some key, a value that is none becomes zeros and its key's scores none.
//
// Warps join through shared memory, the parts of one tile's keys (up to 16 CTAs, a cluster) through distributed shared
// memory in the order of the ranks: nothing is left in global memory, and the same call gives the same bits.
#include "few_bits.cuh"
#include "sm100.cuh"

namespace kv8 {

using namespace sm100;

constexpr int WARPS = 4, THREADS = 32 * WARPS, KEYS = 16;
constexpr float NONE = -1e30f;        // below every score
constexpr float SLACK = 8.0f;         // how far a number may outgrow its reference
constexpr float LEAST = -80.0f;       // log2 of a value scale, for the reference

struct Args {
    const __nv_bfloat16* q;
    const unsigned char *k_pages, *v_pages;
    const float *k_scale, *v_scale;
    const int *block_table, *row_request, *positions;
    const int *tile_req, *tile_row0, *q_start;      // null: a tile is a row
    __nv_bfloat16* out;
    long out_ld;
    int max_pages, page_size, page_shift, n_pages, n_req, n_rows, n_heads, n_kv, chunks, tile_tokens, span, splits, ranked;
    float scale;
};

// sixteen or four bytes, or zeros
__device__ __forceinline__ void copy16(unsigned dst, const void* src, bool in) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(unsigned dst, const void* src, bool in) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(in ? 4 : 0) : "memory");
}
__device__ __forceinline__ void mma_f16(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned turned(unsigned v) {
    unsigned r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ unsigned f16_pair(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const unsigned*>(&h);
}
__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void cluster_barrier() {
    __syncwarp();      // (the threads of a warp arrive as one)
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ unsigned lo8x2(unsigned w) { return few::values8x2((unsigned short)w); }
__device__ __forceinline__ unsigned hi8x2(unsigned w) { return few::values8x2((unsigned short)(w >> 16)); }

// Where chunk c (16 bytes) of a key's row stands, so that eight lanes that read together use all banks.
template <int D> __device__ __forceinline__ int chunk_place(int row, int c) {
    return row * (D / 16) + (D == 64 ? c ^ (row >> 1 & 3) : c ^ (row & 7));
}

template <int D, int NT, int STAGES> struct Plan {
    static constexpr int SLICE = KEYS * D, STAGE = 2 * SLICE + 2 * KEYS * 4, RING = STAGES * STAGE;      // keys, values, their scales
    static constexpr int COLS = 8 * NT, LD = D + 4;                             // of a warp's joined part: floats
    static constexpr int PART = COLS * (LD + 2) * 4;
    static constexpr size_t SMEM = (size_t)WARPS * (RING > PART ? RING : PART);
};

template <int D, int NT, int STAGES>
__global__ void __launch_bounds__(THREADS, D > 128 || NT > 2 ? 2 : NT == 2 ? 3 : 4) attention_kernel(const Args a) {
    using P = Plan<D, NT, STAGES>;
    constexpr int WORDS = D / 16, MT = D / 16;         // words of a key's row that a lane reads; products of 16 numbers of a head
    extern __shared__ __align__(16) unsigned char smem[];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    int tile = a.tile_req != nullptr ? gridDim.y - 1 - blockIdx.y : blockIdx.y;      // a list's longest tile stands last in it
    const int rank = blockIdx.x % a.splits, kv_chunk = blockIdx.x / a.splits;
    if (a.ranked) {      // up to 32 single tokens: the longest request's CTAs come first, so that no long one starts last
        const int mine = lane < a.n_rows ? a.positions[lane] : -2;
        int before = 0;
        for (int j = 0; j < a.n_rows; ++j) {
            const int other = __shfl_sync(0xffffffffu, mine, j);
            before += other > mine || (other == mine && j < lane);
        }
        tile = __ffs(__ballot_sync(0xffffffffu, lane < a.n_rows && before == tile)) - 1;
    }
    const int kvh = kv_chunk / a.chunks, chunk = kv_chunk % a.chunks, group = a.n_heads / a.n_kv;
    // the tile's rows, request and keys: lo .. hi, the first column's end and the last column's start among them
    int row0 = tile, req, n_tok = 1;
    if (a.tile_req != nullptr) {
        req = a.tile_req[tile];
        row0 = a.tile_row0[tile];
        n_tok = req >= 0 && req < a.n_req ? min(a.tile_tokens, a.q_start[req + 1] - row0) : 0;
    } else {
        req = a.row_request[row0];
    }
    // (a row by itself always has work: zeros where its request is none)
    const bool work = n_tok > 0 && row0 >= 0 && row0 + n_tok <= a.n_rows;
    const int pos0 = work ? a.positions[row0] : -1, hi = work ? a.positions[row0 + n_tok - 1] : -1;
    const int lo = ib_first_visible(pos0, a.span), last_lo = ib_first_visible(hi, a.span);
    const bool known = work && req >= 0 && req < a.n_req;
    const int base = lo & ~(KEYS - 1);          // slices start where a page may
    const int slices = known && hi >= lo ? (hi - base) / KEYS + 1 : 0;
    const int s0 = (int)((long)slices * rank / a.splits), s1 = (int)((long)slices * (rank + 1) / a.splits);
    const int col0 = chunk * P::COLS, cols = n_tok * group;
    const int* table = a.block_table + (long)(known ? req : 0) * a.max_pages;
    asm volatile("griddepcontrol.wait;" ::: "memory");

    unsigned char* ring = smem + warp * P::RING;
    constexpr int CHUNKS = D / 16, ROWS = 32 / CHUNKS;          // rows that a copy of the warp covers
    const int row = lane / CHUNKS;
    const unsigned char *kp = a.k_pages + 16 * lane, *vp = a.v_pages + 16 * lane;
    const float* sp = (lane < 16 ? a.k_scale : a.v_scale) + (lane & 15);
    unsigned present = 0;                       // the stages whose slice is in the cache
    // where the first vector of a slice stands, -1 outside the CTA's keys or the cache
    auto look_up = [&](int slice) -> int {
        if (slice >= s1) return -1;
        const int j = base + slice * KEYS;
        const int p = a.page_shift >= 0 ? j >> a.page_shift : j / a.page_size, page = p < a.max_pages ? table[p] : -1;
        return page >= 0 && page < a.n_pages ? (page * a.n_kv + kvh) * a.page_size + (j - p * a.page_size) : -1;
    };
    auto fetch = [&](int place, int slice, int stage) {
        const unsigned at = smem_u32(ring + stage * P::STAGE);
        const int j = base + slice * KEYS, here = place < 0 ? 0 : place;
        const unsigned char *k = kp + (long)here * D, *v = vp + (long)here * D;
        const bool whole = place >= 0 && j >= lo && j + KEYS - 1 <= hi;
        present = (present & ~(1u << stage)) | (unsigned)(place >= 0) << stage;
#pragma unroll
        for (int x = 0; x < KEYS / ROWS; ++x) {
            const int r = x * ROWS + row;
            const bool in = whole || (place >= 0 && j + r >= lo && j + r <= hi);
            const unsigned to = at + 16 * chunk_place<D>(r, lane % CHUNKS);
            copy16(to, k + 512 * x, in);
            copy16(to + P::SLICE, v + 512 * x, in);
        }
        const int r = lane & 15;
        copy4(at + 2 * P::SLICE + 4 * lane, sp + here, whole || (place >= 0 && j + r >= lo && j + r <= hi));
    };
    int next = look_up(s0 + warp);
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) {
        const int place = next;
        next = look_up(s0 + warp + WARPS * (i + 1));
        if (s0 + warp + WARPS * i < s1) fetch(place, s0 + warp + WARPS * i, i);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }

    float o[NT][MT][4], ref[NT][2], l[NT][2];
    auto chunk_of = [&](int i) { return D == 64 ? t : 2 * t + (i & 1) + 8 * (i >> 1); };       // a lane's i-th chunk of a row
    // the queries: column 8 n + g, the numbers that this lane's chunks of a key row meet
    unsigned qf[NT][WORDS][2];
    float factor[NT][2];                   // of columns 8 n + 2t and + 1: what turns a sum of products into log2 of a probability
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int c = col0 + 8 * n + g;
        const bool in = work && c < cols;
        const __nv_bfloat16* src = a.q + ((long)(row0 + (in ? c / group : 0)) * a.n_heads + kvh * group + (in ? c % group : 0)) * D;
        uint2 raw[WORDS];
        unsigned largest = 0;
#pragma unroll
        for (int w = 0; w < WORDS; ++w) {
            raw[w] = in ? *reinterpret_cast<const uint2*>(src + 16 * chunk_of(w >> 2) + 4 * (w & 3)) : make_uint2(0, 0);
            const uint2 v = raw[w];
            largest = max(max(largest, v.x << 16 & 0x7FFFFFFFu), max(v.x & 0x7FFF0000u, max(v.y << 16 & 0x7FFFFFFFu, v.y & 0x7FFF0000u)));
        }
        largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
        largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
        // the power of two that brings the largest to 2^13 .. 2^14 (numbers too small for any: the largest one there is)
        const int e = (int)(largest >> 23), up = largest == 0 ? 0 : 140 - e < 127 ? 140 - e : 127;
        const float by = __uint_as_float((unsigned)(up + 127) << 23);
#pragma unroll
        for (int w = 0; w < WORDS; ++w) {
            qf[n][w][0] = f16_pair(__uint_as_float(raw[w].x << 16) * by, __uint_as_float(raw[w].x & 0xFFFF0000u) * by);
            qf[n][w][1] = f16_pair(__uint_as_float(raw[w].y << 16) * by, __uint_as_float(raw[w].y & 0xFFFF0000u) * by);
        }
        const float f = e == 255 ? __uint_as_float(0x7FC00000u) : a.scale * 1.4426950408889634f / by;     // a query that is none
        factor[n][0] = __shfl_sync(0xffffffffu, f, 8 * t);            // the lane of column 2t
        factor[n][1] = __shfl_sync(0xffffffffu, f, 8 * t + 4);
        ref[n][0] = ref[n][1] = NONE;
        l[n][0] = l[n][1] = 0.0f;
#pragma unroll
        for (int i = 0; i < MT; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.0f;
    }

    int stage = 0;
    for (int s = s0 + warp; s < s1; s += WARPS) {
        {   // the slice STAGES - 1 ahead goes where the slice before this one was
            const int ahead = s + WARPS * (STAGES - 1), place = next;
            next = look_up(ahead + WARPS);
            if (ahead < s1) fetch(place, ahead, stage == 0 ? STAGES - 1 : stage - 1);
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
        __syncwarp();
        unsigned char* at = ring + stage * P::STAGE;
        const float* scales = reinterpret_cast<const float*>(at + 2 * P::SLICE);
        const int j0 = base + s * KEYS;
        const bool there = present >> stage & 1;
        const bool all = there && j0 >= last_lo && j0 + KEYS - 1 <= pos0;      // every column sees every key
        // scores of keys g and g + 8, in two chains
        float sc[NT][2][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int x = 0; x < 4; ++x) sc[n][0][x] = sc[n][1][x] = 0.0f;
#pragma unroll
        for (int c = 0; c < WORDS / 4; ++c) {
            const uint4 x = *reinterpret_cast<const uint4*>(at + 16 * chunk_place<D>(g, chunk_of(c)));
            const uint4 y = *reinterpret_cast<const uint4*>(at + 16 * chunk_place<D>(g + 8, chunk_of(c)));
            const unsigned xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const unsigned a0 = lo8x2(xw[w]), a2 = hi8x2(xw[w]), a1 = lo8x2(yw[w]), a3 = hi8x2(yw[w]);
#pragma unroll
                for (int n = 0; n < NT; ++n) mma_f16(sc[n][w & 1], a0, a1, a2, a3, qf[n][4 * c + w][0], qf[n][4 * c + w][1]);
            }
        }
        const float ks[2] = {few::key_scale(scales[g]), few::key_scale(scales[g + 8])};
        float lv[2] = {lg2(scales[KEYS + g]), lg2(scales[KEYS + g + 8])};
        float least[2] = {fmaxf(lv[0], LEAST), fmaxf(lv[1], LEAST)};
        float p[NT][4];                         // [2 r + c]: key g + 8 r, column 2t + c
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int x = 0; x < 4; ++x) p[n][x] = (sc[n][0][x] + sc[n][1][x]) * (ks[x >> 1] * factor[n][x & 1]);
        if (!all) {
            if (n_tok > 1) {
                // Some column does not see some key, and nothing times no number is none all the same: a value with such a code or scale becomes
                // zeros, and the scores of its key none, for those who see it.  Two lanes look at a key's value.
                uint4* half = reinterpret_cast<uint4*>(at + P::SLICE);
                unsigned found = (__float_as_uint(scales[KEYS + (lane >> 1)]) & 0x7F800000u) == 0x7F800000u ? 0x80u : 0u;
#pragma unroll 1
                for (int c = 0; c < CHUNKS / 2; ++c) {
                    const uint4 w = half[chunk_place<D>(lane >> 1, (lane & 1) * (CHUNKS / 2) + c)];
                    found |= ((w.x & 0x7F7F7F7Fu) + 0x01010101u) | ((w.y & 0x7F7F7F7Fu) + 0x01010101u) |
                             ((w.z & 0x7F7F7F7Fu) + 0x01010101u) | ((w.w & 0x7F7F7F7Fu) + 0x01010101u);
                }
                unsigned none = __ballot_sync(0xffffffffu, (found & 0x80808080u) != 0);
                if (none) {
                    none |= (none >> 1 & 0x55555555u) | (none << 1 & 0xAAAAAAAAu);
#pragma unroll 1
                    for (int c = 0; c < CHUNKS / 2; ++c)
                        if (none >> lane & 1) half[chunk_place<D>(lane >> 1, (lane & 1) * (CHUNKS / 2) + c)] = make_uint4(0, 0, 0, 0);
                    __syncwarp();
#pragma unroll
                    for (int r = 0; r < 2; ++r)
                        if (none >> (2 * g + 16 * r) & 1) {
                            lv[r] = -INFINITY;
                            least[r] = LEAST;
#pragma unroll
                            for (int n = 0; n < NT; ++n) p[n][2 * r] = p[n][2 * r + 1] = __uint_as_float(0x7FC00000u);
                        }
                }
            }
            unsigned hidden = 0;
#pragma unroll 1
            for (int x = 0; x < 4 * NT; ++x) {
                const int c = col0 + 8 * (x >> 2) + 2 * t + (x & 1), j = j0 + g + 4 * (x & 2);
                const int pos = c < cols && there ? (n_tok == 1 ? pos0 : a.positions[row0 + c / group]) : -1;
                hidden |= (unsigned)(j > pos || j < ib_first_visible(pos, a.span)) << x;
            }
#pragma unroll
            for (int x = 0; x < 4 * NT; ++x)
                if (hidden >> x & 1) p[x >> 2][x & 3] = -INFINITY;
        }
        bool outgrown = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int x = 0; x < 4; ++x) outgrown |= p[n][x] + least[x >> 1] > ref[n][x & 1] + SLACK;
        if (__any_sync(0xffffffffu, outgrown)) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float r = fmaxf(ref[n][c], fmaxf(p[n][c] + least[0], p[n][c + 2] + least[1]));
                    r = fmaxf(r, __shfl_xor_sync(0xffffffffu, r, 4));
                    r = fmaxf(r, __shfl_xor_sync(0xffffffffu, r, 8));
                    r = fmaxf(r, __shfl_xor_sync(0xffffffffu, r, 16));
                    const float fade = ex2(ref[n][c] - r);
                    ref[n][c] = r;
                    l[n][c] *= fade;
#pragma unroll
                    for (int x = 0; x < MT; ++x) { o[n][x][c] *= fade; o[n][x][c + 2] *= fade; }
                }
        }
        unsigned pb[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int x = 0; x < 4; ++x) p[n][x] -= ref[n][x & 1];
#pragma unroll
            for (int c = 0; c < 2; ++c) l[n][c] += ex2(p[n][c]) + ex2(p[n][c + 2]);
#pragma unroll
            for (int r = 0; r < 2; ++r) pb[n][r] = turned(f16_pair(ex2(p[n][2 * r] + lv[r]), ex2(p[n][2 * r + 1] + lv[r])));
        }
        // values: rows are the numbers of a head, keys 2t, 2t + 1, 2t + 8, 2t + 9 are this lane's
        const unsigned char* vt = at + P::SLICE;
        constexpr int VWORDS = D / 32;              // words of four numbers that a lane reads of a key
#pragma unroll
        for (int i2 = 0; i2 < (VWORDS + 3) / 4; ++i2) {
            unsigned v[4][VWORDS < 4 ? VWORDS : 4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int key = 2 * t + (r & 1) + 8 * (r >> 1);
                if constexpr (D >= 128) {
                    const uint4 x = *reinterpret_cast<const uint4*>(vt + 16 * chunk_place<D>(key, g + 8 * i2));
                    v[r][0] = x.x; v[r][1] = x.y; v[r][2] = x.z; v[r][3] = x.w;
                } else {
                    const uint2 x = *reinterpret_cast<const uint2*>(vt + 16 * chunk_place<D>(key, g >> 1) + 8 * (g & 1));
                    v[r][0] = x.x; v[r][1] = x.y;
                }
            }
#pragma unroll
            for (int x = 0; x < (VWORDS < 4 ? VWORDS : 4); ++x) {
                const unsigned e0 = __byte_perm(v[0][x], v[1][x], 0x5140), e1 = __byte_perm(v[2][x], v[3][x], 0x5140);
                const unsigned f0 = __byte_perm(v[0][x], v[1][x], 0x7362), f1 = __byte_perm(v[2][x], v[3][x], 0x7362);
                const unsigned ea = lo8x2(e0), eb = hi8x2(e0), ec = lo8x2(e1), ed = hi8x2(e1);
                const unsigned fa = lo8x2(f0), fb = hi8x2(f0), fc = lo8x2(f1), fd = hi8x2(f1);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    mma_f16(o[n][8 * i2 + 2 * x], ea, eb, ec, ed, pb[n][0], pb[n][1]);
                    mma_f16(o[n][8 * i2 + 2 * x + 1], fa, fb, fc, fd, pb[n][0], pb[n][1]);
                }
            }
        }
        __syncwarp();                 // every lane has read the slice before its place is filled again
        stage = stage == STAGES - 1 ? 0 : stage + 1;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");

    // a warp's part: per column the reference, the sum and the weighted values, both relative to 2^reference
    __syncthreads();
    auto part = [&](int w) { return reinterpret_cast<float*>(smem + w * P::PART); };          // [COLS][LD], then [COLS][2]
    {
        float* mine = part(warp);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float sum = l[n][c];
                sum += __shfl_xor_sync(0xffffffffu, sum, 4);
                sum += __shfl_xor_sync(0xffffffffu, sum, 8);
                sum += __shfl_xor_sync(0xffffffffu, sum, 16);
                const int col = 8 * n + 2 * t + c;
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    // row g of product i is number 16 (g + 8 (i / 8)) + 2 (i % 8) of the head, row g + 8 the next one
                    const int d = D >= 128 ? 16 * (g + 8 * (i / 8)) + 2 * (i % 8) : 8 * g + 2 * i;
                    *reinterpret_cast<float2*>(mine + col * P::LD + d) = make_float2(o[n][i][c], o[n][i][c + 2]);
                }
                if (g == 0) *reinterpret_cast<float2*>(mine + P::COLS * P::LD + 2 * col) = make_float2(ref[n][c], sum);
            }
    }
    __syncthreads();
    const int used = min(P::COLS, cols - col0);          // columns of this chunk
    float* own = part(0);
    {   // the warps' parts become the first one's
        float* ml[WARPS];
#pragma unroll
        for (int w = 0; w < WARPS; ++w) ml[w] = part(w) + P::COLS * P::LD;
        for (int i = threadIdx.x; i < used * D / 4; i += THREADS) {
            const int col = i / (D / 4), d = i % (D / 4) * 4;
            float top = NONE;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) top = fmaxf(top, ml[w][2 * col]);
            float4 sum = make_float4(0, 0, 0, 0);
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float by = ex2(ml[w][2 * col] - top);
                const float4 v = *reinterpret_cast<const float4*>(part(w) + col * P::LD + d);
                sum.x += v.x * by; sum.y += v.y * by; sum.z += v.z * by; sum.w += v.w * by;
            }
            *reinterpret_cast<float4*>(own + col * P::LD + d) = sum;      // read by this thread alone before
        }
        __syncthreads();
        for (int col = threadIdx.x; col < used; col += THREADS) {
            float top = NONE, sum = 0.0f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) top = fmaxf(top, ml[w][2 * col]);
#pragma unroll
            for (int w = 0; w < WARPS; ++w) sum += ml[w][2 * col + 1] * ex2(ml[w][2 * col] - top);
            ml[0][2 * col] = top;
            ml[0][2 * col + 1] = sum;
        }
    }
    if (a.splits > 1) {
        cluster_barrier();
    } else {
        __syncthreads();
    }
    auto remote = [&](unsigned r, const float* p) -> unsigned {
        unsigned addr = smem_u32(p);
        if (a.splits > 1) asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(smem_u32(p)), "r"(r));
        return addr;
    };
    // every CTA of the cluster finishes its share of the tile's numbers, four at a time
    const int quads = used * (D / 4);
    const int q0 = (int)((long)quads * rank / a.splits), q1 = (int)((long)quads * (rank + 1) / a.splits);
    for (int i = q0 + (int)threadIdx.x; work && i < q1; i += THREADS) {
        const int col = i / (D / 4), d = i % (D / 4) * 4, c = col0 + col;
        float top = NONE, sum = 0.0f;
        float4 acc = make_float4(0, 0, 0, 0);
        for (int r = 0; r < a.splits; ++r) {
            float pm, pl;
            asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(pm), "=f"(pl) : "r"(remote(r, own + P::COLS * P::LD + 2 * col)) : "memory");
            float4 v;
            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                         : "r"(remote(r, own + col * P::LD + d)) : "memory");
            const float m2 = fmaxf(top, pm), fade = ex2(top - m2), by = ex2(pm - m2);
            top = m2;
            sum = sum * fade + pl * by;
            acc.x = acc.x * fade + v.x * by; acc.y = acc.y * fade + v.y * by; acc.z = acc.z * fade + v.z * by; acc.w = acc.w * fade + v.w * by;
        }
        const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;               // a row that sees no key: zeros
        const uint2 w = make_uint2(sm100::pack_bf16(acc.x * inv, acc.y * inv), sm100::pack_bf16(acc.z * inv, acc.w * inv));
        __nv_bfloat16* dst = a.out + (long)(row0 + c / group) * a.out_ld + (long)(kvh * group + c % group) * D + d;
        if ((reinterpret_cast<uintptr_t>(dst) & 7) == 0) {
            *reinterpret_cast<uint2*>(dst) = w;
        } else {
            const unsigned short* h = reinterpret_cast<const unsigned short*>(&w);
#pragma unroll
            for (int e = 0; e < 4; ++e) reinterpret_cast<unsigned short*>(dst)[e] = h[e];
        }
    }
    // no CTA leaves while another may read its shared memory
    if (a.splits > 1) cluster_barrier();
}

// How many CTAs share a tile's keys: as many as run at once (four an SM), or twice as many for up to 32 single tokens with contexts that may
// reach 8,192 keys: then they come longest first, and lengths that differ even out (us of as many and twice as many, 16 requests of
// 32 heads on 8: all of 2,048 keys 19.1 and 25.7, 100 to 2,048 16.0 and 21.3; all of 8,192 50.8 and 55.6, 100 to 8,192 36.9 and 35.3, to 16,384
// 65.9 and 53.6; 24 requests of 100 to 8,192 61.3 and 42.1).  Clusters of 16 only where one round of them is all there is.
static int splits_for(long pairs, int max_len, bool ranked) {
    int s = 1;
    while (s < 8 && pairs * s * 2 <= (ranked && max_len >= 8192 ? 2 : 1) * 148 * 4 && max_len >= 64 * s) s *= 2;
    return s == 8 && pairs * 16 <= 148 && max_len >= 64 * 16 ? 16 : s;
}

template <int D, int NT, int STAGES>
static int launch(const Args& a, int tiles, cudaStream_t stream) {
    using P = Plan<D, NT, STAGES>;
    auto kernel = attention_kernel<D, NT, STAGES>;
    static IbDeviceSet done, wide;
    if (int r = ib_allow_dynamic_smem(done, kernel, P::SMEM)) return r;
    if (a.splits > 8) {
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return (int)e;
        if (dev >= 64 || !((wide.bits.load(std::memory_order_acquire) >> dev) & 1ull)) {
            if ((e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1)) != cudaSuccess) return (int)e;
            if (dev < 64) wide.bits.fetch_or(1ull << dev, std::memory_order_release);
        }
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.splits * a.n_kv * a.chunks, tiles);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = P::SMEM;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = a.splits;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ib_pdl_enabled ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
    return e == cudaSuccess ? ib_launch_status() : (int)e;
}

}  // namespace kv8

IB_EXPORT int ib_paged_attention_kv8(const IbAttentionKv8* c) {
    using namespace kv8;
    if (c->n > 0x7FFFFFFF || c->n_heads > 65536 || c->max_pages > 0x7FFFFFFF || c->n_pages > 0x7FFFFFFF) return IB_ERR_UNSUPPORTED;
    const void *q = c->q, *k_pages = c->k_pages, *v_pages = c->v_pages;
    const float *k_scale = c->k_scale, *v_scale = c->v_scale;
    const int *block_table = c->block_table, *row_request = c->row_request, *positions = c->positions, *tile_req = c->tile_req,
              *tile_row0 = c->tile_row0, *q_start = c->q_start;
    void* out = c->out;
    const cudaStream_t stream = c->stream;
    const long out_ld = c->out_ld;
    const int max_pages = (int)c->max_pages, page_size = (int)c->page_size, n_pages = (int)c->n_pages, n_req = (int)c->n_req, n = (int)c->n,
              n_tiles = (int)c->n_tiles, n_heads = (int)c->n_heads, n_kv = (int)c->n_kv, d = (int)c->d, span = (int)c->span,
              max_len = (int)(c->max_len < 0x7FFFFFFF ? c->max_len : 0x7FFFFFFF);
    int tile_tokens = (int)c->tile_tokens, splits = (int)c->splits;
    const float scale = (float)c->scale;
    if (n < 0 || n_heads <= 0 || n_kv <= 0 || n_heads % n_kv || page_size <= 0 || splits < 0 || splits > 16 || (splits & (splits - 1))) return IB_ERR_ARGUMENT;
    if (d != 64 && d != 128 && d != 256) return IB_ERR_UNSUPPORTED;
    if ((long)n_pages * n_kv * page_size > 0x7FFFFFFFL || page_size % KEYS) return IB_ERR_UNSUPPORTED;
    if (reinterpret_cast<uintptr_t>(q) % 8 || (reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages)) % 16) return IB_ERR_UNSUPPORTED;
    const int tiles = tile_req ? n_tiles : n, group = n_heads / n_kv;
    if (tiles == 0 || n == 0) return IB_OK;
    if (tile_req == nullptr) tile_tokens = 1;
    const int cols = tile_tokens * group;
    if (tile_tokens < 1) return IB_ERR_ARGUMENT;
    if (tile_tokens > 1 && cols > 32) return ib_kv8_prompt(c);
    const int nt = cols <= 8 ? 1 : cols <= 16 || d == 256 ? 2 : tile_tokens > 1 ? 4 : 2;
    if (tile_tokens > 1 && cols > 8 * nt) return IB_ERR_ARGUMENT;
    const int chunks = (cols + 8 * nt - 1) / (8 * nt);
    const bool ranked = tile_req == nullptr && n > 1 && n <= 32;
    if (splits == 0) splits = splits_for((long)tiles * n_kv * chunks, max_len, ranked);
    Args a = {(const __nv_bfloat16*)q, (const unsigned char*)k_pages, (const unsigned char*)v_pages, k_scale, v_scale, block_table, row_request,
              positions, tile_req, tile_row0, q_start, (__nv_bfloat16*)out, out_ld, max_pages, page_size,
              (page_size & (page_size - 1)) ? -1 : __builtin_ctz(page_size), n_pages, n_req, n, n_heads, n_kv,
              chunks, tile_tokens, span, splits, ranked, scale};
    if (tiles > 65535 || (long)n_kv * chunks * splits > 0x7FFFFFFFL) return IB_ERR_UNSUPPORTED;
    if (d == 64) return nt == 1 ? launch<64, 1, 4>(a, tiles, stream) : nt == 2 ? launch<64, 2, 4>(a, tiles, stream) : launch<64, 4, 4>(a, tiles, stream);
    if (d == 128) return nt == 1 ? launch<128, 1, 3>(a, tiles, stream) : nt == 2 ? launch<128, 2, 4>(a, tiles, stream) : launch<128, 4, 4>(a, tiles, stream);
    return nt == 1 ? launch<256, 1, 3>(a, tiles, stream) : launch<256, 2, 3>(a, tiles, stream);
}
