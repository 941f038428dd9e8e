// Keys and values in 8 bits: how a step's join the paged cache, and attention over it for any head size.
// (The layout is in few_bits.cuh.)
#include "few_bits.cuh"

// The first row (plus one) that was left out because its position lay outside the rotation tables; 0: none.
__device__ int ib_kv8_row_fault_word = 0;
IB_EXPORT int ib_kv8_row_fault(int reset) {
    int v = 0;
    cudaError_t e = cudaMemcpyFromSymbol(&v, ib_kv8_row_fault_word, sizeof(int));
    if (e != cudaSuccess) return -(int)e;
    if (reset && v != 0) {
        const int zero = 0;
        cudaMemcpyToSymbol(ib_kv8_row_fault_word, &zero, sizeof(int));
    }
    return v;
}
IB_EXPORT int ib_kv8_row_fault_async(int* out, cudaStream_t stream) {
    return (int)cudaMemcpyFromSymbolAsync(out, ib_kv8_row_fault_word, sizeof(int), 0, cudaMemcpyDeviceToHost, stream);
}

namespace few {

constexpr int STORE_WARPS = 4;

struct StoreArgs {
    long ldx;
    int n_heads, n_kv, d, flags, rot_dim, interleaved, table_rows, max_pages, page_size, n_pages, n_req, wait_first;   // flags: 1 norm q, 2 norm k
    float eps;
};

// a number in float32 that rounds to fewer bits as it does: cut off, with the last bit set where something was
__device__ __forceinline__ float sticky(double v) {
    const float f = __double2float_rz(v);
    return (double)f == v ? f : __uint_as_float(__float_as_uint(f) | 1u);
}

// Heads of 64, 128 or 256 numbers that turn as a whole, element i with i + d / 2, in bfloat16: a lane holds four numbers of the
// first half of a head and the four they turn with, a warp 256 / D heads at a time and STEPS times, whose loads are all on their way
// before the first is used; what belongs to the row (its place, its angles) is fetched once.  2,048 rows of 32 + 8 + 8 heads of 128:
// 47 MB, 51 us with a warp a head through shared memory, 17 us like this.
template <int D, int STEPS, typename WT>
__global__ void __launch_bounds__(32 * STORE_WARPS, 9) kv8_store_whole_kernel(
    const __nv_bfloat16* __restrict__ qkv, const WT* __restrict__ q_weight, const WT* __restrict__ k_weight,
    const float* __restrict__ cos_table, const float* __restrict__ sin_table, const int* __restrict__ positions,
    const int* __restrict__ row_request, const int* __restrict__ block_table, unsigned char* __restrict__ k_pages,
    unsigned char* __restrict__ v_pages, float* __restrict__ k_scale, float* __restrict__ v_scale, __nv_bfloat16* __restrict__ q_out,
    const StoreArgs a) {
    constexpr int LANES = D / 8, HEADS = 32 / LANES;            // of a head; heads a step
    ib_grid_dependency_launch();
    const int row = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, i = 4 * (lane % LANES);
    const int head0 = ((int)blockIdx.y * STORE_WARPS + warp) * HEADS * STEPS + lane / LANES, heads = a.n_heads + 2 * a.n_kv;
    if (a.wait_first) ib_grid_dependency_wait();
    positions = ib_after_wait(positions);
    row_request = ib_after_wait(row_request);
    cos_table = ib_after_wait(cos_table);
    sin_table = ib_after_wait(sin_table);
    const int pos = positions[row], req = row_request[row];
    const bool fault = pos < 0 || pos >= a.table_rows;
    const float4 c = fault ? make_float4(0, 0, 0, 0) : *reinterpret_cast<const float4*>(cos_table + (long)pos * (D / 2) + i);
    const float4 s = fault ? make_float4(0, 0, 0, 0) : *reinterpret_cast<const float4*>(sin_table + (long)pos * (D / 2) + i);
    ib_grid_dependency_wait();
    qkv = ib_after_wait(qkv);
    q_weight = ib_after_wait(q_weight);
    k_weight = ib_after_wait(k_weight);
    block_table = ib_after_wait(block_table);
    if (fault) {
        if (threadIdx.x == 0) atomicCAS(&ib_kv8_row_fault_word, 0, row + 1);
        return;
    }
    uint2 raw[STEPS][2];
#pragma unroll
    for (int t = 0; t < STEPS; ++t) {
        const int head = head0 + t * HEADS;
        const __nv_bfloat16* src = qkv + (long)row * a.ldx + (long)head * D + i;
        raw[t][0] = head < heads ? *reinterpret_cast<const uint2*>(src) : make_uint2(0, 0);
        raw[t][1] = head < heads ? *reinterpret_cast<const uint2*>(src + D / 2) : make_uint2(0, 0);
    }
    const int page = req >= 0 && req < a.n_req && pos / a.page_size < a.max_pages ? block_table[(long)req * a.max_pages + pos / a.page_size] : -1;
    const float cs[4] = {c.x, c.y, c.z, c.w}, sn[4] = {s.x, s.y, s.z, s.w};
    // how far float32 may be off in a key's number times 448 / its largest: 8 last places of 448 (float32 weights: 16)
    constexpr float OFF = sizeof(WT) == 4 ? 448.0f / 1048576.0f : 448.0f / 2097152.0f;
    unsigned near = 0;        // the steps in which a key's number that far up has another code than one that far down
#pragma unroll
    for (int t = 0; t < STEPS; ++t) {
        const int head = head0 + t * HEADS, kind = head < a.n_heads ? 0 : (head < a.n_heads + a.n_kv ? 1 : 2);   // 0 q, 1 k, 2 v
        float x[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            x[h][0] = __uint_as_float(raw[t][h].x << 16);
            x[h][1] = __uint_as_float(raw[t][h].x & 0xFFFF0000u);
            x[h][2] = __uint_as_float(raw[t][h].y << 16);
            x[h][3] = __uint_as_float(raw[t][h].y & 0xFFFF0000u);
        }
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) ss += x[0][e] * x[0][e] + x[1][e] * x[1][e];
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        // the norm's factor comes last: it is one for the whole head, so no code depends on it, and a bfloat16 number times a bfloat16 weight
        // is exact
        float inv = 1.0f;
        if (kind != 2) {
            if (a.flags >> kind & 1) {
                inv = 1.0f / sqrtf(ss / (float)D + a.eps);
                const WT* w = kind == 0 ? q_weight : k_weight;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[0][e] *= w ? ib_to_float(w[i + e]) : 1.0f;
                    x[1][e] *= w ? ib_to_float(w[D / 2 + i + e]) : 1.0f;
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float first = x[0][e], second = x[1][e];
                x[0][e] = fmaf(first, cs[e], -(second * sn[e]));
                x[1][e] = fmaf(second, cs[e], first * sn[e]);
            }
        }
        unsigned m = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) m = max(m, max(__float_as_uint(x[0][e]) & 0x7FFFFFFFu, __float_as_uint(x[1][e]) & 0x7FFFFFFFu));
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (head >= heads) continue;
        if (kind == 0) {
            __nv_bfloat16* dst = q_out + ((long)row * a.n_heads + head) * D + i;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const __nv_bfloat162 lo = __floats2bfloat162_rn(x[h][0] * inv, x[h][1] * inv), hi = __floats2bfloat162_rn(x[h][2] * inv, x[h][3] * inv);
                *reinterpret_cast<uint2*>(dst + h * (D / 2)) = make_uint2(*reinterpret_cast<const unsigned*>(&lo), *reinterpret_cast<const unsigned*>(&hi));
            }
        } else if (page >= 0 && page < a.n_pages) {       // else a request that stands in to fill a batch
            const long place = ((long)page * a.n_kv + (head - a.n_heads) % a.n_kv) * a.page_size + pos % a.page_size;
            unsigned char* dst = (kind == 1 ? k_pages : v_pages) + place * D + i;
            float by, scale;
            vector_scale(__uint_as_float(m) * inv, by, scale);
            if (by != 0.0f) by = 448.0f / __uint_as_float(m);
#pragma unroll
            for (int h = 0; h < 2; ++h)
                *reinterpret_cast<unsigned*>(dst + h * (D / 2)) = by != 0.0f ? codes8x4(x[h][0] * by, x[h][1] * by, x[h][2] * by, x[h][3] * by) : 0u;
            if (kind == 1 && by != 0.0f) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    near |= (unsigned)(codes8x4(fmaf(x[h][0], by, OFF), fmaf(x[h][1], by, OFF), fmaf(x[h][2], by, OFF), fmaf(x[h][3], by, OFF)) !=
                                       codes8x4(fmaf(x[h][0], by, -OFF), fmaf(x[h][1], by, -OFF), fmaf(x[h][2], by, -OFF), fmaf(x[h][3], by, -OFF))) << t;
            }
            if (i == 0) (kind == 1 ? k_scale : v_scale)[place] = scale;
        }
    }
    // A key's codes are the nearest ones to what the float32 tables turn it to: where float32 leaves that open (one of twenty) the head is
    // turned and divided once more in 64 bits.  (At the end, where little else is held: 2,048 rows of 32 + 8 + 8 heads of 128 17.4 us, in its
    // place 18.8, not at all 16.3, all keys in 64 bits 25.)
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) near |= __shfl_xor_sync(0xffffffffu, near, o);
    const unsigned steps = __reduce_or_sync(0xffffffffu, near);
#pragma unroll 1
    for (int t = 0; steps >> t != 0; ++t) {
        if (!(steps >> t & 1)) continue;
        const int head = near >> t & 1 ? head0 + t * HEADS : a.n_heads;
        const __nv_bfloat16* src = qkv + (long)row * a.ldx + (long)head * D + i;
        const WT* w = a.flags >> 1 & 1 ? k_weight : nullptr;
        double y[2][4], top = 0.0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float first = __bfloat162float(src[e]) * (w ? ib_to_float(w[i + e]) : 1.0f);
            const float second = __bfloat162float(src[D / 2 + e]) * (w ? ib_to_float(w[D / 2 + i + e]) : 1.0f);
            y[0][e] = (double)first * cs[e] - (double)second * sn[e];
            y[1][e] = (double)second * cs[e] + (double)first * sn[e];
            top = fmax(top, fmax(fabs(y[0][e]), fabs(y[1][e])));
        }
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
        const double by = 448.0 / top;
        if (!(near >> t & 1)) continue;
        unsigned char* dst = k_pages + (((long)page * a.n_kv + head - a.n_heads) * a.page_size + pos % a.page_size) * D + i;
#pragma unroll
        for (int h = 0; h < 2; ++h)
            *reinterpret_cast<unsigned*>(dst + h * (D / 2)) = codes8x4(sticky(y[h][0] * by), sticky(y[h][1] * by), sticky(y[h][2] * by), sticky(y[h][3] * by));
    }
}

// Everything else, a warp per head of a row: norm, rotation in float32; queries are stored in their type, keys and values as codes
// with a scale per vector.  (A key's codes are the nearest ones to what float32 gives: one may be the neighbour of the kernel's above.)
template <typename T, typename WT>
__global__ void __launch_bounds__(32 * STORE_WARPS) kv8_store_kernel(
    const T* __restrict__ qkv, const WT* __restrict__ q_weight, const WT* __restrict__ k_weight,
    const float* __restrict__ cos_table, const float* __restrict__ sin_table, const int* __restrict__ positions,
    const int* __restrict__ row_request, const int* __restrict__ block_table, unsigned char* __restrict__ k_pages,
    unsigned char* __restrict__ v_pages, float* __restrict__ k_scale, float* __restrict__ v_scale, T* __restrict__ q_out,
    const StoreArgs a) {
    extern __shared__ float smem[];
    ib_grid_dependency_launch();
    const int row = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = a.d;
    const int head = blockIdx.y * STORE_WARPS + warp;
    float* sh = smem + warp * 2 * d;      // the head as it came, and turned
    float* turned = sh + d;
    if (a.wait_first) ib_grid_dependency_wait();
    positions = ib_after_wait(positions);
    const int pos = positions[row];
    const bool fault = pos < 0 || (a.rot_dim > 0 && pos >= a.table_rows);
    ib_grid_dependency_wait();
    qkv = ib_after_wait(qkv);
    q_weight = ib_after_wait(q_weight);
    k_weight = ib_after_wait(k_weight);
    block_table = ib_after_wait(block_table);
    row_request = ib_after_wait(row_request);
    cos_table = ib_after_wait(cos_table);
    sin_table = ib_after_wait(sin_table);
    if (fault) {
        if (threadIdx.x == 0) atomicCAS(&ib_kv8_row_fault_word, 0, row + 1);
        return;
    }
    if (head >= a.n_heads + 2 * a.n_kv) return;
    const int kind = head < a.n_heads ? 0 : (head < a.n_heads + a.n_kv ? 1 : 2);   // 0 q, 1 k, 2 v
    long place = -1;
    if (kind != 0) {
        const int req = row_request[row];
        const int page = req >= 0 && req < a.n_req && pos / a.page_size < a.max_pages ? block_table[(long)req * a.max_pages + pos / a.page_size] : -1;
        if (page < 0 || page >= a.n_pages) return;      // a request that stands in to fill a batch
        place = ((long)page * a.n_kv + (head - a.n_heads) % a.n_kv) * a.page_size + pos % a.page_size;
    }
    const T* src = qkv + (long)row * a.ldx + (long)head * d;
    float ss = 0.0f;
    for (int j = lane; j < d; j += 32) { sh[j] = ib_to_float(src[j]); ss += sh[j] * sh[j]; }
    const float* out = sh;
    if (kind != 2) {
        if (a.flags >> kind & 1) {
            const float inv = 1.0f / sqrtf(ib_warp_sum(ss) / (float)d + a.eps);
            const WT* w = kind == 0 ? q_weight : k_weight;
            for (int j = lane; j < d; j += 32) sh[j] = sh[j] * inv * (w ? ib_to_float(w[j]) : 1.0f);
        }
        __syncwarp();
        const int half = a.rot_dim / 2;
        const float *c = cos_table + (long)pos * half, *s = sin_table + (long)pos * half;
        // element i of the first half turns with element i + rot_dim / 2, or (interleaved) element 2i with 2i + 1.  The
        // products are rounded before they are added up, so that the codes do not depend on how a compiler joins them.
        for (int j = lane; j < d; j += 32) {
            float o = sh[j];
            if (j < a.rot_dim) {
                const int i = a.interleaved ? j >> 1 : (j < half ? j : j - half);
                const bool first = a.interleaved ? !(j & 1) : j < half;
                const float other = a.interleaved ? sh[j ^ 1] : sh[first ? j + half : j - half];
                o = first ? __fsub_rn(__fmul_rn(o, c[i]), __fmul_rn(other, s[i])) : __fadd_rn(__fmul_rn(o, c[i]), __fmul_rn(other, s[i]));
            }
            turned[j] = o;
        }
        out = turned;
    }
    __syncwarp();
    if (kind == 0) {
        T* dst = q_out + ((long)row * a.n_heads + head) * d;
        for (int j = lane; j < d; j += 32) dst[j] = ib_from_float<T>(out[j]);
        return;
    }
    unsigned m = 0;
    for (int j = lane; j < d; j += 32) m = max(m, __float_as_uint(out[j]) & 0x7FFFFFFFu);   // no number counts as the largest
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    float by, scale;
    vector_scale(__uint_as_float(m), by, scale);
    unsigned char* dst = (kind == 1 ? k_pages : v_pages) + place * d;
    for (int j = 4 * lane; j < d; j += 128)
        *reinterpret_cast<unsigned*>(dst + j) = by != 0.0f ? codes8x4(out[j] * by, out[j + 1] * by, out[j + 2] * by, out[j + 3] * by) : 0u;
    if (lane == 0) (kind == 1 ? k_scale : v_scale)[place] = scale;
}

// Attention of every (row, head) by a block of its own: eight warps take every eighth key of the row's, each with a running
// maximum and sum in float32, and join what they have in shared memory.  Any head size up to 512, float32 throughout.
constexpr int SLOW_WARPS = 8, SLOW_PER_LANE = 16;

struct AttendArgs {
    int max_pages, page_size, n_pages, n_req, n_heads, n_kv, d, span;
    float scale;
    long out_ld;
};

template <typename T>
__global__ void __launch_bounds__(32 * SLOW_WARPS) kv8_attention_kernel(
    const T* __restrict__ q, const unsigned char* __restrict__ k_pages, const unsigned char* __restrict__ v_pages,
    const float* __restrict__ k_scale, const float* __restrict__ v_scale, const int* __restrict__ block_table,
    const int* __restrict__ row_request, const int* __restrict__ positions, T* __restrict__ out, const AttendArgs a) {
    __shared__ float part[SLOW_WARPS][512], part_m[SLOW_WARPS], part_l[SLOW_WARPS];
    ib_grid_dependency_sync();
    q = ib_after_wait(q);
    k_pages = ib_after_wait(k_pages);
    v_pages = ib_after_wait(v_pages);
    k_scale = ib_after_wait(k_scale);
    v_scale = ib_after_wait(v_scale);
    block_table = ib_after_wait(block_table);
    row_request = ib_after_wait(row_request);
    positions = ib_after_wait(positions);
    const int row = blockIdx.x, head = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = a.d;
    const int kvh = head / (a.n_heads / a.n_kv), pos = positions[row], req = row_request[row];
    const int lo = ib_first_visible(pos, a.span);
    const bool known = req >= 0 && req < a.n_req;
    float qv[SLOW_PER_LANE], acc[SLOW_PER_LANE], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < SLOW_PER_LANE; ++i) {
        const int j = lane + 32 * i;
        qv[i] = j < d ? ib_to_float(q[((long)row * a.n_heads + head) * d + j]) * a.scale : 0.0f;
        acc[i] = 0.0f;
    }
    for (int t = lo + warp; known && t <= pos; t += SLOW_WARPS) {
        const int page = t / a.page_size < a.max_pages ? block_table[(long)req * a.max_pages + t / a.page_size] : -1;
        if (page < 0 || page >= a.n_pages) continue;
        const long place = ((long)page * a.n_kv + kvh) * a.page_size + t % a.page_size;
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < SLOW_PER_LANE; ++i) {
            const int j = lane + 32 * i;
            if (j < d) s = fmaf(qv[i], value8(k_pages[place * d + j]), s);
        }
        s = ib_warp_sum(s) * key_scale(k_scale[place]);
        const float m2 = fmaxf(m, s), fade = m == -INFINITY ? 0.0f : expf(m - m2), p = expf(s - m2);
        const float pv = p * v_scale[place];
        l = l * fade + p;
        m = m2;
#pragma unroll
        for (int i = 0; i < SLOW_PER_LANE; ++i) {
            const int j = lane + 32 * i;
            if (j < d) acc[i] = acc[i] * fade + pv * value8(v_pages[place * d + j]);
        }
    }
    if (lane == 0) { part_m[warp] = m; part_l[warp] = l; }
#pragma unroll
    for (int i = 0; i < SLOW_PER_LANE; ++i) if (lane + 32 * i < d) part[warp][lane + 32 * i] = acc[i];
    __syncthreads();
    float top = -INFINITY, sum = 0.0f;
    for (int w = 0; w < SLOW_WARPS; ++w) if (part_l[w] != 0.0f) top = fmaxf(top, part_m[w]);
    for (int w = 0; w < SLOW_WARPS; ++w) if (part_l[w] != 0.0f) sum += part_l[w] * expf(part_m[w] - top);
    for (int j = threadIdx.x; j < d; j += 32 * SLOW_WARPS) {
        float o = 0.0f;
        for (int w = 0; w < SLOW_WARPS; ++w) if (part_l[w] != 0.0f) o += part[w][j] * expf(part_m[w] - top);
        out[(long)row * a.out_ld + (long)head * d + j] = ib_from_float<T>(sum != 0.0f ? o / sum : 0.0f);   // a row that sees no key: zeros
    }
}

}  // namespace few

// The step's rows qkv [n, queries | keys | values of n_heads, n_kv, n_kv heads of d numbers] (float32 or bfloat16): per-head
// norm (norm_flags: 1 queries, 2 keys) and rotation, queries to q_out, keys and values as 8-bit codes into their pages.
struct IbStoreKv8 {
    const void *qkv, *q_weight, *k_weight;
    const float *cos_table, *sin_table;
    const int *positions, *row_request, *block_table;
    void *k_pages, *v_pages;
    float *k_scale, *v_scale;
    void* q_out;
    cudaStream_t stream;
    long is_f32, ldx, n, n_heads, n_kv, d, w_is_f32, norm_flags, rot_dim, interleaved, table_rows, max_pages, page_size, n_pages, n_req;
    double eps;
};
IB_EXPORT int ib_qk_norm_rope_store_kv8(const IbStoreKv8* s) {
    using namespace few;
    if (s->n > 0x7FFFFFFF || s->n_heads > 65536 || s->n_kv > 65536 || s->table_rows > 0x7FFFFFFF) return IB_ERR_UNSUPPORTED;
    const void *qkv = s->qkv, *q_weight = s->q_weight, *k_weight = s->k_weight;
    const float *cos_table = s->cos_table, *sin_table = s->sin_table;
    const int *positions = s->positions, *row_request = s->row_request, *block_table = s->block_table;
    void *k_pages = s->k_pages, *v_pages = s->v_pages, *q_out = s->q_out;
    float *k_scale = s->k_scale, *v_scale = s->v_scale;
    const cudaStream_t stream = s->stream;
    const long ldx = s->ldx;
    const int is_f32 = (int)s->is_f32, n = (int)s->n, n_heads = (int)s->n_heads, n_kv = (int)s->n_kv, d = (int)s->d, w_is_f32 = (int)s->w_is_f32,
              norm_flags = (int)s->norm_flags, rot_dim = (int)s->rot_dim, interleaved = (int)s->interleaved, table_rows = (int)s->table_rows,
              max_pages = (int)s->max_pages, page_size = (int)s->page_size, n_pages = (int)s->n_pages, n_req = (int)s->n_req;
    const float eps = (float)s->eps;
    if (n < 0 || n_heads <= 0 || n_kv <= 0 || d <= 0 || d % 4 || d > 1024 || rot_dim < 0 || rot_dim > d || rot_dim % 2 || page_size <= 0) return IB_ERR_ARGUMENT;
    if (n == 0) return IB_OK;
    const StoreArgs a = {ldx, n_heads, n_kv, d, norm_flags, rot_dim, interleaved, table_rows, max_pages, page_size, n_pages, n_req, !ib_pdl_enabled, eps};
    const int heads = n_heads + 2 * n_kv;
    if (!is_f32 && !interleaved && rot_dim == d && (d == 64 || d == 128 || d == 256) &&
        (reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q_out)) % 8 == 0 && ldx % 4 == 0 &&
        (reinterpret_cast<uintptr_t>(cos_table) | reinterpret_cast<uintptr_t>(sin_table)) % 16 == 0) {
        // few rows: every warp a step of its own; many: three, so that what belongs to a row is fetched less often
        const int steps = (long)n * heads * d < 148L * 64 * 256 ? 1 : 3, per_block = STORE_WARPS * (256 / d) * steps;
        const dim3 grid(n, (heads + per_block - 1) / per_block);
#define GO(D, S, WT) ib_launch_early(kv8_store_whole_kernel<D, S, WT>, grid, dim3(32 * STORE_WARPS), 0, stream, (const __nv_bfloat16*)qkv, (const WT*)q_weight, \
    (const WT*)k_weight, cos_table, sin_table, positions, row_request, block_table, (unsigned char*)k_pages, (unsigned char*)v_pages, \
    k_scale, v_scale, (__nv_bfloat16*)q_out, a)
#define GO_D(S, WT) (d == 64 ? GO(64, S, WT) : d == 128 ? GO(128, S, WT) : GO(256, S, WT))
        if (w_is_f32) { if (steps == 1) GO_D(1, float); else GO_D(3, float); }
        else { if (steps == 1) GO_D(1, __nv_bfloat16); else GO_D(3, __nv_bfloat16); }
#undef GO_D
#undef GO
        return ib_launch_status();
    }
    const dim3 grid(n, (n_heads + 2 * n_kv + STORE_WARPS - 1) / STORE_WARPS);
    const size_t smem = (size_t)STORE_WARPS * 2 * d * sizeof(float);
#define GO(T, WT) ib_launch_early(kv8_store_kernel<T, WT>, grid, dim3(32 * STORE_WARPS), smem, stream, (const T*)qkv, (const WT*)q_weight, \
    (const WT*)k_weight, cos_table, sin_table, positions, row_request, block_table, (unsigned char*)k_pages, (unsigned char*)v_pages, \
    k_scale, v_scale, (T*)q_out, a)
    if (is_f32) { if (w_is_f32) GO(float, float); else GO(float, __nv_bfloat16); }
    else { if (w_is_f32) GO(__nv_bfloat16, float); else GO(__nv_bfloat16, __nv_bfloat16); }
#undef GO
    return ib_launch_status();
}

IB_EXPORT int ib_paged_attention_kv8_generic(const void* q, int is_f32, const void* k_pages, const void* v_pages,
                                             const float* k_scale, const float* v_scale, const int* block_table, int max_pages,
                                             int page_size, int n_pages, int n_req, const int* row_request, const int* positions, int n,
                                             int n_heads, int n_kv, int d, float scale, int span, void* out, long out_ld,
                                             cudaStream_t stream) {
    using namespace few;
    if (n < 0 || n_heads <= 0 || n_kv <= 0 || n_heads % n_kv || d <= 0 || page_size <= 0) return IB_ERR_ARGUMENT;
    if (d > 512 || n_heads > 65535) return IB_ERR_UNSUPPORTED;
    if (n == 0) return IB_OK;
    const AttendArgs a = {max_pages, page_size, n_pages, n_req, n_heads, n_kv, d, span, scale, out_ld};
    const dim3 grid(n, n_heads);
#define GO(T) ib_launch_early(kv8_attention_kernel<T>, grid, dim3(32 * SLOW_WARPS), 0, stream, (const T*)q, (const unsigned char*)k_pages, \
    (const unsigned char*)v_pages, k_scale, v_scale, block_table, row_request, positions, (T*)out, a)
    if (is_f32) GO(float); else GO(__nv_bfloat16);
#undef GO
    return ib_launch_status();
}
