// Attention over paged keys and values in 8 bits: single tokens, and tiles of a prompt's tokens (bfloat16 queries).
//
// A CTA works for one key/value head of one tile of rows and one part of its keys.  The tile's (token, head) pairs are the
// columns of the products (8 NT of them), keys and the numbers of a head their rows, so eight columns cost what one does.
// Each of four warps takes every fourth slice of 16 keys through a ring of its own (cp.async, a lane looks up a key's place
// one slice ahead of its copies): no warp waits for another until the end.
//
//   scores   S = K Q^T: codes become f16 pairs exactly; a query row is multiplied by the power of two that brings its largest
//            number to 2^13 .. 2^14, so f16 holds all of it that counts (2^-38 of the largest).  A lane takes 16 neighbouring
//            numbers of a key row as its part of four products of 16: any order of the numbers serves, if the queries'
//            is the same.  s = acc * key scale * (softmax scale log2 e / the query's power of two).
//   softmax  with running references: m per lane and column for the sum of 2^(s - m), and R per column for what multiplies
//            the values, 2^(s + log2(value scale) - R), so that values of very different scales keep their precision in f16.
//            A reference moves only when a number has outgrown it by 2^8 (a vote of the warp says whether any has).
//   values   O = V^T P^T: two keys' codes are interleaved byte by byte, P is turned with movmatrix; sums in float32.
//
// Warps join through shared memory, the parts of one tile's keys (up to 16 CTAs, a cluster) through distributed shared
// memory in the order of the ranks: nothing is left in global memory, and the same call gives the same bits.  Places
// outside a tile's keys are filled with zeros on their way, whatever the page holds there.
#include "few_bits.cuh"
#include "sm100.cuh"

namespace kv8 {

using sm100::ex2;
using sm100::smem_u32;

constexpr int WARPS = 4, KEYS = 16;
constexpr float NONE = -1e30f;        // below every score
constexpr float SLACK = 8.0f;         // how far a number may outgrow its reference

struct Args {
    const __nv_bfloat16* q;
    const unsigned char *k_pages, *v_pages;
    const float *k_scale, *v_scale;
    const int *block_table, *row_request, *positions;
    const int *tile_req, *tile_row0, *q_start;      // null: a tile is a row
    __nv_bfloat16* out;
    long out_ld;
    int max_pages, page_size, n_pages, n_req, n_rows, n_heads, n_kv, chunks, tile_tokens, span, splits;
    float scale;
};

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
__device__ __forceinline__ unsigned lo8x2(unsigned w) { return few::values8x2((unsigned short)w); }
__device__ __forceinline__ unsigned hi8x2(unsigned w) { return few::values8x2((unsigned short)(w >> 16)); }

// where chunk c (16 bytes) of a key's row stands in a slice, so that eight lanes that read together use all banks
template <int D> __device__ __forceinline__ int chunk_place(int row, int c) {
    return row * (D / 16) + (D == 64 ? c ^ (row >> 1 & 3) : c ^ (row & 7));
}

template <int D, int NT, int STAGES> struct Plan {
    static constexpr int SLICE = KEYS * D, STAGE = 2 * SLICE + 2 * KEYS * 4, RING = STAGES * STAGE;
    static constexpr int COLS = 8 * NT, LD = D + 4;                        // of a warp's joined part: floats
    static constexpr int PART = COLS * (LD + 2) * 4;
    static constexpr size_t SMEM = (size_t)(WARPS * RING > WARPS * PART ? WARPS * RING : WARPS * PART);
};

template <int D, int NT, int STAGES>
__global__ void __launch_bounds__(32 * WARPS) attention_kernel(const Args a) {
    using P = Plan<D, NT, STAGES>;
    constexpr int CHUNKS = D / 16, PER_LANE = D / 64, KSTEPS = D / 16, MT = D / 16;
    extern __shared__ __align__(16) unsigned char smem[];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int tile = blockIdx.x / a.splits, rank = blockIdx.x % a.splits;
    const int kvh = blockIdx.y / a.chunks, chunk = blockIdx.y % a.chunks, group = a.n_heads / a.n_kv;
    // the tile's rows, request and keys: lo .. hi, the first column's end and the last column's start among them
    int row0 = tile, req, n_tok = 1;
    if (a.tile_req != nullptr) {
        req = a.tile_req[tile];
        row0 = a.tile_row0[tile];
        if (req >= 0) n_tok = min(a.tile_tokens, a.q_start[req + 1] - row0);
    } else {
        req = a.row_request[row0];
    }
    const bool work = req >= 0 && n_tok > 0 && row0 >= 0 && row0 + n_tok <= a.n_rows;
    const int pos0 = work ? a.positions[row0] : -1, hi = work ? a.positions[row0 + n_tok - 1] : -1;
    const int lo = ib_first_visible(pos0, a.span), last_lo = ib_first_visible(hi, a.span);
    const bool known = work && req < a.n_req;
    const int slices = known && hi >= lo ? (hi - lo) / KEYS + 1 : 0;
    const int s0 = (int)((long)slices * rank / a.splits), s1 = (int)((long)slices * (rank + 1) / a.splits);
    const int* table = a.block_table + (long)(known ? req : 0) * a.max_pages;
    asm volatile("griddepcontrol.wait;" ::: "memory");

    unsigned char* ring = smem + warp * P::RING;
    const unsigned ring_at = smem_u32(ring);
    // a lane's key of a slice: where its vector stands, -1 outside the tile's keys or the cache
    auto look_up = [&](int slice) -> int {
        const int j = lo + slice * KEYS + (lane & 15);
        if (slice >= s1 || j > hi) return -1;
        const int p = j / a.page_size, page = p < a.max_pages ? table[p] : -1;
        return page >= 0 && page < a.n_pages ? (page * a.n_kv + kvh) * a.page_size + (j - p * a.page_size) : -1;
    };
    auto fetch = [&](int place, int stage) {
        const unsigned at = ring_at + stage * P::STAGE;
        constexpr int ROWS = 32 / CHUNKS > 0 ? 32 / CHUNKS : 1;           // rows a warp-wide copy covers
#pragma unroll
        for (int i = 0; i < KEYS * CHUNKS / 32; ++i) {
            const int row = i * ROWS + lane / CHUNKS, c = lane % CHUNKS;
            const int pl = __shfl_sync(0xffffffffu, place, row);
            const long off = pl < 0 ? 0 : (long)pl * D + 16 * c;
            const unsigned to = at + 16 * chunk_place<D>(row, c);
            copy16(to, a.k_pages + off, pl >= 0);
            copy16(to + P::SLICE, a.v_pages + off, pl >= 0);
        }
        copy4(at + 2 * P::SLICE + 4 * lane, (lane < 16 ? a.k_scale : a.v_scale) + (place < 0 ? 0 : place), place >= 0);
    };
    int next = look_up(s0 + warp);
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) {
        const int place = next;
        next = look_up(s0 + warp + WARPS * (i + 1));
        if (s0 + warp + WARPS * i < s1) fetch(place, i);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }

    // the queries: column 8 n + g, the numbers that this lane's chunks of a key row meet
    const int col0 = chunk * P::COLS, cols = n_tok * group;
    unsigned qf[NT][KSTEPS][2];
    float factor[NT][2];                   // of columns 8 n + 2t and + 1: what turns a sum of products into log2 of a probability
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int c = col0 + 8 * n + g;
        const bool in = work && c < cols;
        const __nv_bfloat16* src = a.q + ((long)(row0 + (in ? c / group : 0)) * a.n_heads + kvh * group + (in ? c % group : 0)) * D;
        uint2 raw[KSTEPS];
        unsigned largest = 0;
#pragma unroll
        for (int i = 0; i < PER_LANE; ++i) {
            const int ch = D == 64 ? t : 2 * t + (i & 1) + 8 * (i >> 1);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const uint2 v = in ? *reinterpret_cast<const uint2*>(src + 16 * ch + 4 * w) : make_uint2(0, 0);
                raw[4 * i + w] = v;
                largest = max(max(largest, v.x << 16 & 0x7FFFFFFFu), max(v.x & 0x7FFF0000u, max(v.y << 16 & 0x7FFFFFFFu, v.y & 0x7FFF0000u)));
            }
        }
        largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
        largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
        const int e = (int)(largest >> 23) - 127 - 13, up = largest == 0 ? 0 : max(-e, -126) < 127 ? max(-e, -126) : 127;
        const float by = __uint_as_float((unsigned)(up + 127) << 23);
#pragma unroll
        for (int k = 0; k < KSTEPS; ++k) {
            qf[n][k][0] = f16_pair(__uint_as_float(raw[k].x << 16) * by, __uint_as_float(raw[k].x & 0xFFFF0000u) * by);
            qf[n][k][1] = f16_pair(__uint_as_float(raw[k].y << 16) * by, __uint_as_float(raw[k].y & 0xFFFF0000u) * by);
        }
        const float f = a.scale * 1.4426950408889634f / by;
        factor[n][0] = __shfl_sync(0xffffffffu, f, 8 * t);            // the lane of column 2t
        factor[n][1] = __shfl_sync(0xffffffffu, f, 8 * t + 4);
    }

    float o[NT][MT][4], ref[NT][2], m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        ref[n][0] = ref[n][1] = m[n][0] = m[n][1] = NONE;
        l[n][0] = l[n][1] = 0.0f;
#pragma unroll
        for (int i = 0; i < MT; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.0f;
    }

    int stage = 0;
    for (int s = s0 + warp; s < s1; s += WARPS) {
        {   // the slice STAGES - 1 ahead goes where the slice before this one was
            const int ahead = s + WARPS * (STAGES - 1), place = next;
            next = look_up(ahead + WARPS);
            if (ahead < s1) fetch(place, stage == 0 ? STAGES - 1 : stage - 1);
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
        __syncwarp();
        const unsigned char* at = ring + stage * P::STAGE;
        const float* scales = reinterpret_cast<const float*>(at + 2 * P::SLICE);
        // scores of keys g and g + 8
        float sc[NT][2][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) sc[n][h][0] = sc[n][h][1] = sc[n][h][2] = sc[n][h][3] = 0.0f;
#pragma unroll
        for (int i = 0; i < PER_LANE; ++i) {
            const int ch = D == 64 ? t : 2 * t + (i & 1) + 8 * (i >> 1);
            const uint4 x = *reinterpret_cast<const uint4*>(at + 16 * chunk_place<D>(g, ch));
            const uint4 y = *reinterpret_cast<const uint4*>(at + 16 * chunk_place<D>(g + 8, ch));
            const unsigned xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const unsigned a0 = lo8x2(xw[w]), a2 = hi8x2(xw[w]), a1 = lo8x2(yw[w]), a3 = hi8x2(yw[w]);
#pragma unroll
                for (int n = 0; n < NT; ++n) mma_f16(sc[n][w & 1], a0, a1, a2, a3, qf[n][4 * i + w][0], qf[n][4 * i + w][1]);
            }
        }
        const float ks[2] = {scales[g], scales[g + 8]};
        const float lv[2] = {lg2(scales[16 + g]), lg2(scales[24 + g])};
        const int j0 = lo + s * KEYS;
        const bool all = j0 >= last_lo && j0 + KEYS - 1 <= pos0;      // every column sees every key of the slice
        float p[NT][4], w[NT][4];
        bool outgrown = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float v = (sc[n][0][i] + sc[n][1][i]) * (ks[i >> 1] * factor[n][i & 1]);
                p[n][i] = v;
                w[n][i] = v + lv[i >> 1];
                if (!all) {
                    const int c = col0 + 8 * n + 2 * t + (i & 1), j = j0 + g + 8 * (i >> 1);
                    const int pos = c < cols ? (n_tok == 1 ? pos0 : a.positions[row0 + c / group]) : -1;
                    if (j > pos || j < ib_first_visible(pos, a.span)) p[n][i] = w[n][i] = -INFINITY;
                }
                outgrown |= !(p[n][i] <= m[n][i & 1] + SLACK) || !(w[n][i] <= ref[n][i & 1] + SLACK);
            }
        if (__any_sync(0xffffffffu, outgrown)) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const float m2 = fmaxf(m[n][c], fmaxf(p[n][c], p[n][c + 2]));
                    l[n][c] *= ex2(m[n][c] - m2);
                    m[n][c] = m2;
                    float r = fmaxf(ref[n][c], fmaxf(w[n][c], w[n][c + 2]));
                    r = fmaxf(r, __shfl_xor_sync(0xffffffffu, r, 4));
                    r = fmaxf(r, __shfl_xor_sync(0xffffffffu, r, 8));
                    r = fmaxf(r, __shfl_xor_sync(0xffffffffu, r, 16));
                    const float fade = ex2(ref[n][c] - r);
                    ref[n][c] = r;
#pragma unroll
                    for (int i = 0; i < MT; ++i) { o[n][i][c] *= fade; o[n][i][c + 2] *= fade; }
                }
        }
        unsigned pb[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int c = 0; c < 2; ++c) l[n][c] += ex2(p[n][c] - m[n][c]) + ex2(p[n][c + 2] - m[n][c]);
            pb[n][0] = turned(f16_pair(ex2(w[n][0] - ref[n][0]), ex2(w[n][1] - ref[n][1])));
            pb[n][1] = turned(f16_pair(ex2(w[n][2] - ref[n][0]), ex2(w[n][3] - ref[n][1])));
        }
        // values: rows are the numbers of a head, keys 2t, 2t + 1, 2t + 8, 2t + 9 are this lane's
        const unsigned char* vt = at + P::SLICE;
        if constexpr (D >= 128) {
#pragma unroll
            for (int i = 0; i < D / 128; ++i) {
                uint4 v[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = *reinterpret_cast<const uint4*>(vt + 16 * chunk_place<D>(2 * t + (r & 1) + 8 * (r >> 1), g + 8 * i));
                const unsigned* vw[4] = {&v[0].x, &v[1].x, &v[2].x, &v[3].x};
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const unsigned e0 = __byte_perm(vw[0][x], vw[1][x], 0x5140), e1 = __byte_perm(vw[2][x], vw[3][x], 0x5140);
                    const unsigned f0 = __byte_perm(vw[0][x], vw[1][x], 0x7362), f1 = __byte_perm(vw[2][x], vw[3][x], 0x7362);
                    const unsigned ea = lo8x2(e0), eb = hi8x2(e0), ec = lo8x2(e1), ed = hi8x2(e1);
                    const unsigned fa = lo8x2(f0), fb = hi8x2(f0), fc = lo8x2(f1), fd = hi8x2(f1);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        mma_f16(o[n][8 * i + 2 * x], ea, eb, ec, ed, pb[n][0], pb[n][1]);
                        mma_f16(o[n][8 * i + 2 * x + 1], fa, fb, fc, fd, pb[n][0], pb[n][1]);
                    }
                }
            }
        } else {
            uint2 v[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = *reinterpret_cast<const uint2*>(vt + 16 * chunk_place<D>(2 * t + (r & 1) + 8 * (r >> 1), g >> 1) + 8 * (g & 1));
            const unsigned* vw[4] = {&v[0].x, &v[1].x, &v[2].x, &v[3].x};
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const unsigned e0 = __byte_perm(vw[0][x], vw[1][x], 0x5140), e1 = __byte_perm(vw[2][x], vw[3][x], 0x5140);
                const unsigned f0 = __byte_perm(vw[0][x], vw[1][x], 0x7362), f1 = __byte_perm(vw[2][x], vw[3][x], 0x7362);
                const unsigned ea = lo8x2(e0), eb = hi8x2(e0), ec = lo8x2(e1), ed = hi8x2(e1);
                const unsigned fa = lo8x2(f0), fb = hi8x2(f0), fc = lo8x2(f1), fd = hi8x2(f1);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    mma_f16(o[n][2 * x], ea, eb, ec, ed, pb[n][0], pb[n][1]);
                    mma_f16(o[n][2 * x + 1], fa, fb, fc, fd, pb[n][0], pb[n][1]);
                }
            }
        }
        __syncwarp();                 // every lane has read the slice before its place is filled again
        stage = stage == STAGES - 1 ? 0 : stage + 1;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");

    // a warp's part: per column the maximum, the sum and the weighted values, all relative to 2^maximum
    __syncthreads();
    auto part = [&](int w) { return reinterpret_cast<float*>(smem + w * P::PART); };          // [COLS][LD], then [COLS][2]
    {
        float* mine = part(warp);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float top = m[n][c];
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                float sum = l[n][c] * ex2(m[n][c] - top);
                sum += __shfl_xor_sync(0xffffffffu, sum, 4);
                sum += __shfl_xor_sync(0xffffffffu, sum, 8);
                sum += __shfl_xor_sync(0xffffffffu, sum, 16);
                const int col = 8 * n + 2 * t + c;
                const float by = ref[n][c] == NONE ? 0.0f : ex2(ref[n][c] - top);
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    // row g of product i is number 16 (g + 8 (i / 8)) + 2 (i % 8) of the head, row g + 8 the next one
                    const int d = D >= 128 ? 16 * (g + 8 * (i / 8)) + 2 * (i % 8) : 8 * g + 2 * i;
                    *reinterpret_cast<float2*>(mine + col * P::LD + d) = make_float2(o[n][i][c] * by, o[n][i][c + 2] * by);
                }
                if (g == 0) *reinterpret_cast<float2*>(mine + P::COLS * P::LD + 2 * col) = make_float2(top, sum);
            }
    }
    __syncthreads();
    const int used = min(P::COLS, cols - col0);          // columns of this chunk
    float* own = part(0);
    {   // the warps' parts become the first one's
        float* ml[WARPS];
#pragma unroll
        for (int w = 0; w < WARPS; ++w) ml[w] = part(w) + P::COLS * P::LD;
        for (int i = threadIdx.x; i < used * D / 4; i += 32 * WARPS) {
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
        for (int col = threadIdx.x; col < used; col += 32 * WARPS) {
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
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
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
    for (int i = q0 + (int)threadIdx.x; work && i < q1; i += 32 * WARPS) {
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
    __syncwarp();
    // no CTA leaves while another may read its shared memory
    if (a.splits > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// How many CTAs share a tile's keys: up to two rounds of resident CTAs (three an SM), 64 keys at least for each of them.
static int splits_for(long pairs, int max_len) {
    int s = 1;
    while (s < 16 && pairs * s * 2 <= 148 * 3 * 2 && max_len >= 128 * s) s *= 2;
    return s;
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
    cfg.gridDim = dim3((unsigned)tiles * a.splits, a.n_kv * a.chunks);
    cfg.blockDim = dim3(32 * WARPS);
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

// Attention of bfloat16 rows over pages of 8-bit keys and values, heads of 64, 128 or 256 numbers.  tile_req null: every row
// is a tile of its own (row_request says whose); else tile i holds up to tile_tokens rows of request tile_req[i] (-1: none)
// from row tile_row0[i] on, and request r's rows end at q_start[r + 1].  splits: CTAs that share a tile's keys (1, 2, 4, 8, 16; 0: chosen here by max_len, which
// no position is beyond).
IB_EXPORT int ib_paged_attention_kv8(const void* q, const void* k_pages, const void* v_pages, const float* k_scale, const float* v_scale,
                                     const int* block_table, int max_pages, int page_size, int n_pages, int n_req,
                                     const int* row_request, const int* positions, int n, const int* tile_req, const int* tile_row0,
                                     const int* q_start, int n_tiles, int tile_tokens, int n_heads, int n_kv, int d, float scale, int span,
                                     void* out, long out_ld, int splits, int max_len, cudaStream_t stream) {
    using namespace kv8;
    if (n < 0 || n_heads <= 0 || n_kv <= 0 || n_heads % n_kv || page_size <= 0 || splits < 0 || splits > 16 || (splits & (splits - 1))) return IB_ERR_ARGUMENT;
    if (d != 64 && d != 128 && d != 256) return IB_ERR_UNSUPPORTED;
    if ((long)n_pages * n_kv * page_size > 0x7FFFFFFFL || reinterpret_cast<uintptr_t>(q) % 8) return IB_ERR_UNSUPPORTED;
    const int tiles = tile_req ? n_tiles : n, group = n_heads / n_kv;
    if (tiles == 0 || n == 0) return IB_OK;
    if (tile_req == nullptr) tile_tokens = 1;
    const int cols = tile_tokens * group;
    if (tile_tokens < 1 || (tile_tokens > 1 && cols > 32)) return IB_ERR_ARGUMENT;
    const int nt = cols <= 8 ? 1 : cols <= 16 || d == 256 ? 2 : tile_tokens > 1 ? 4 : 2;
    if (tile_tokens > 1 && cols > 8 * nt) return IB_ERR_ARGUMENT;
    const int chunks = (cols + 8 * nt - 1) / (8 * nt);
    if (splits == 0) splits = splits_for((long)tiles * n_kv * chunks, max_len);
    Args a = {(const __nv_bfloat16*)q, (const unsigned char*)k_pages, (const unsigned char*)v_pages, k_scale, v_scale, block_table, row_request,
              positions, tile_req, tile_row0, q_start, (__nv_bfloat16*)out, out_ld, max_pages, page_size, n_pages, n_req, n, n_heads, n_kv,
              chunks, tile_tokens, span, splits, scale};
    if ((long)a.n_kv * a.chunks > 65535 || (long)tiles * splits > 0x7FFFFFFFL) return IB_ERR_UNSUPPORTED;
    if (d == 64) return nt == 1 ? launch<64, 1, 4>(a, tiles, stream) : nt == 2 ? launch<64, 2, 4>(a, tiles, stream) : launch<64, 4, 4>(a, tiles, stream);
    if (d == 128) return nt == 1 ? launch<128, 1, 4>(a, tiles, stream) : nt == 2 ? launch<128, 2, 4>(a, tiles, stream) : launch<128, 4, 4>(a, tiles, stream);
    return nt == 1 ? launch<256, 1, 3>(a, tiles, stream) : launch<256, 2, 3>(a, tiles, stream);
}
