// Attention of a prompt's tokens over paged keys and values in 8 bits, on the fifth-generation tensor cores (bfloat16
// queries, heads of 128 numbers).
//
// A CTA owns 256 (token, head) rows of one key/value head as two tiles of 128 that take turns, and walks the keys in tiles
// of 128, as attention_pair_tcgen05.cu does for bfloat16 pages:
//   S  = Q K^T   in tensor memory, one region of 128 x 128 float32 per tile of rows;
//   P  = by one thread a row, 64 keys at a time, written as f16 pairs over columns of S that have been read;
//   O += P V     P from tensor memory, accumulated there over all keys.
// What the codes change:
//   keys and values   come through registers: warps 8 to 11 load a tile's codes while the tile before is in use, turn them into f16
//       and store them in the swizzled form that the products read.  An e4m3 number's bits, moved seven to the left with the sign in its
//       place, are the f16 number 2^-8 times as large, its small ones included: four integer instructions for two numbers, where the
//       conversion instruction would compete with the exponentials (both run at a quarter of the other units' rate or less).
//       A code that is no number would become 480: the largest magnitude is kept beside (one instruction for four codes, 2 to 4 % of the whole), and
//       where it says that there is one, its vector's key scale becomes no number, so that whoever sees the vector gets none.
//   queries           a row is multiplied by the power of two that brings its largest number to 2^13 .. 2^14, as in attention_kv8.cu.
//   scores            s = S * key scale * factor of the row (positive: a negative scale turns the query).
//   value scales      of 32 keys with scales within 2^-11 of one another (or 0) go into the values: V' = code * scale * 2^(7 - e), e the power
//       of two above the largest of them, P = 2^(s + e - R), and the sum takes P 2^-e.  V' is a normal f16 number, rounded
//       to 11 bits like P (with the factor's rounding 3 * 2^-12 of a term in all).  Other keys, and pages that are not in the cache, have P =
//       2^(s + log2(value scale) - R) and a second exponential for the sum: weights of values of very different scales keep
//       their precision.
// What bounds it: a tile of keys takes the tensor pipe 2,048 cycles, the exponentials as many of theirs, and 6,500 in all (about 6,800 with the
// question for codes that are no numbers): a softmax warp's own instruction stream, one warp of either tile of rows on each of the SM's
// four schedulers (without the conversions 6,100, without the key scales and the exponentials too 4,600; more registers for these warps
// change nothing).  With the value scales' logarithms and reciprocals
// from shared memory, which hands out 16 bytes to a whole warp in four cycles, it was 7,500.  A prompt of 2,048 tokens, 32 heads on 8: 80 us, 430
// TFLOP/s (attention_kv8.cu's tiles of 32 rows 272 us; bfloat16 pages 49 us).
// All waits are bounded and report through this file's error word.
#include <type_traits>

#include "few_bits.cuh"
#include "sm100.cuh"

namespace kv8p {

using namespace sm100;

constexpr int D = 128, ROWS = 128, KEYS = 128, SLICE = 16;
constexpr int CONVERT = 4, FIRST_CONVERT = 8, ISSUER = FIRST_CONVERT + CONVERT, THREADS = 32 * (ISSUER + 1);
constexpr int HALF_BYTES = 128 * 128, TILE_BYTES = 2 * HALF_BYTES;      // [128][64] f16 numbers, swizzled; a tile of 128 x 128
constexpr float SLACK = 8.0f, LEAST = -80.0f;                           // see attention_kv8.cu
constexpr int GROUP = 32;                                               // keys that share a power of two, a converting warp's

// what the softmax needs to know of a tile's keys
struct Scales {
    float key[KEYS], value[KEYS];                    // value -1: no such key
    float log_power[KEYS / GROUP], inverse[KEYS / GROUP];        // e and 2^-e of 32 keys
    int apart[KEYS / GROUP];                         // whether their value scales are too far apart for one
};
constexpr int SMEM = 6 * TILE_BYTES + 2 * (int)sizeof(Scales) + 20 * 8 + 1024;
static_assert(CONVERT * GROUP == KEYS && SMEM <= 227 * 1024, "shared memory of an SM");

__device__ int g_error = 0;
__device__ __forceinline__ bool mbar_wait(unsigned bar, unsigned parity, int code) { return mbar_wait_bounded(bar, parity, &g_error, code); }

struct Args {
    const __nv_bfloat16* q;
    const unsigned char *k_pages, *v_pages;
    const float *k_scale, *v_scale;
    const int *block_table, *positions, *tile_req, *tile_row0, *q_start;
    __nv_bfloat16* out;
    long out_ld;
    int max_pages, page_size, n_pages, n_req, n_rows, n_heads, n_kv, tokens, span, wide;
    float scale;
};

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// two float32 operations in one instruction
__device__ __forceinline__ unsigned long long two(float x, float y) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float2 apart(unsigned long long v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ unsigned long long mul2(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("mul.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("add.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
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
__device__ __forceinline__ unsigned mul_f16(unsigned a, unsigned b) {
    const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const unsigned*>(&r);
}
// Codes in the high bytes of two halves to f16 numbers 2^-8 times as large: their magnitudes' bits, and the numbers.  A code that is no number
// becomes 480 * 2^-8, the one magnitude above the largest number's.
__device__ __forceinline__ unsigned magnitudes(unsigned h) { return h >> 1 & 0x3F803F80u; }
__device__ __forceinline__ unsigned widened(unsigned h, unsigned m) { return m | (h & 0x80008000u); }
constexpr unsigned NO_NUMBER = 0x3F80u;
// where chunk c (eight f16 numbers) of a row stands in a tile
__device__ __forceinline__ unsigned place(int row, int c) { return (unsigned)((c >> 3) * HALF_BYTES + row * 128 + ((c & 7) ^ (row & 7)) * 16); }

__global__ void __launch_bounds__(THREADS, 1) prompt_kernel(const Args a) {
    extern __shared__ unsigned char raw_smem[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~(uintptr_t)1023);
    unsigned char *sq = smem, *sk = sq + 2 * TILE_BYTES, *sv = sk + 2 * TILE_BYTES;      // queries; two stages of keys, two of values
    Scales* scales = reinterpret_cast<Scales*>(sv + 2 * TILE_BYTES);                     // of the values' stages
    unsigned long long* bars = reinterpret_cast<unsigned long long*>(scales + 2);
    const unsigned q_full = smem_u32(bars);
    const unsigned k_full0 = smem_u32(bars + 1), k_empty0 = smem_u32(bars + 3), v_full0 = smem_u32(bars + 5), v_empty0 = smem_u32(bars + 7);
    const unsigned s_full0 = smem_u32(bars + 9);      // per tile of rows: S of the next tile of keys is there
    const unsigned p_full0 = smem_u32(bars + 11);     // per tile of rows and half of the keys (2 t + h): its P is there
    const unsigned h_done0 = smem_u32(bars + 15);     // per tile of rows: the first half's products are done
    const unsigned o_full0 = smem_u32(bars + 17);     // per tile of rows: O holds every key
    unsigned* tmem_slot = reinterpret_cast<unsigned*>(bars + 19);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        mbar_init(q_full, 8);
        for (int s = 0; s < 2; ++s) {
            mbar_init(k_full0 + 8 * s, CONVERT); mbar_init(k_empty0 + 8 * s, 1);
            mbar_init(v_full0 + 8 * s, CONVERT); mbar_init(v_empty0 + 8 * s, 1);
            mbar_init(s_full0 + 8 * s, 1); mbar_init(o_full0 + 8 * s, 1); mbar_init(h_done0 + 8 * s, 1);
            mbar_init(p_full0 + 16 * s, 4); mbar_init(p_full0 + 16 * s + 8, 4);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == ISSUER) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    // (not before: a CTA of the next kernel that came first could hold columns that this one waits for, and wait for its end)
    ib_grid_dependency_sync();
    // the last tiles of a prompt see the most keys: they come first, so that the grid's tail is short
    const int tile = (int)(gridDim.x / a.n_kv) - 1 - (int)(blockIdx.x / a.n_kv), kvh = (int)(blockIdx.x % a.n_kv);
    const int req = a.tile_req[tile], row0 = a.tile_row0[tile], group = a.n_heads / a.n_kv;
    const int n_tok = req >= 0 && req < a.n_req ? min(a.tokens, a.q_start[req + 1] - row0) : 0;
    const bool work = n_tok > 0 && row0 >= 0 && row0 + n_tok <= a.n_rows;     // else a place of the list without a tile
    const int tpt = ROWS / group;                                            // tokens of a tile of rows
    const int p0 = work ? a.positions[row0] : -1, pmax = work ? a.positions[row0 + n_tok - 1] : -1;
    const int lo_min = ib_first_visible(p0, a.span), t_begin = lo_min / KEYS;
    const int n_tok_t[2] = {n_tok < tpt ? n_tok : tpt, n_tok > tpt ? n_tok - tpt : 0};
    int n_tiles_t[2];                                                        // tiles of keys that a tile of rows walks (none without a key)
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int last = work && n_tok_t[t] > 0 ? a.positions[row0 + t * tpt + n_tok_t[t] - 1] : -1;
        n_tiles_t[t] = last >= lo_min ? last / KEYS + 1 - t_begin : 0;
    }
    const int n_tiles = max(n_tiles_t[0], n_tiles_t[1]);

    const unsigned tmem = *tmem_slot;      // columns 128 t: S and P of tile t; 256 + 128 t: O of tile t
    bool ok = true;
    // what was stored in shared memory is seen by the products of whoever hears of it through `bar`
    auto handed_over = [&](unsigned bar) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(bar);
    };

    if (!work) {
        // (down to the end, where the tensor memory is given back)
    } else if (warp >= FIRST_CONVERT && warp < ISSUER) {
        // A warp brings 32 keys of every tile, two slices of 16 that lie in one page each: a lane 16 numbers of a row, four rows at a
        // time.  What no row of the tile sees, and what is not in the cache, is zeros.
        const int first = 32 * (warp - FIRST_CONVERT), row = lane >> 2 & 3, c = (lane & 3) | (lane >> 4) << 2;
        const int* table = a.block_table + (long)req * a.max_pages;
        struct Slice { long vector; int begin, end; };      // the first vector of the slice, the places of it that are read
        auto look_up = [&](int i, int half) -> Slice {
            const int j = (t_begin + i) * KEYS + first + SLICE * half, p = j / a.page_size;
            const int page = i < n_tiles && j <= pmax && p < a.max_pages ? table[p] : -1;
            if (page < 0 || page >= a.n_pages) return {0, 0, 0};
            return {((long)page * a.n_kv + kvh) * a.page_size + (j - p * a.page_size), max(lo_min - j, 0), min(pmax - j + 1, SLICE)};
        };
        uint4 k_raw[8], v_raw[8];
        float k_s = 0.0f, v_s = 0.0f;                        // of the lane's key; value -1: its page is not in the cache
        auto load = [&](uint4 (&raw)[8], const unsigned char* pages, const Slice (&at)[2]) {
#pragma unroll
            for (int x = 0; x < 8; ++x) {
                const Slice& s = at[x >> 2];
                const int r = 4 * (x & 3) + row;
                raw[x] = r >= s.begin && r < s.end ? *reinterpret_cast<const uint4*>(pages + (s.vector + r) * D + 16 * c) : make_uint4(0, 0, 0, 0);
            }
        };
        // (VALUES: times the rows' factors, an f16 number in both halves of the lane that has the row's key)
        unsigned largest = 0;                                // magnitude of the tile's codes so far, the even and the odd ones
        auto store = [&](const uint4 (&raw)[8], unsigned char* to, auto values, unsigned factor) {
#pragma unroll
            for (int x = 0; x < 8; ++x) {
                const int r = first + 4 * x + row;
                const unsigned w[4] = {raw[x].x, raw[x].y, raw[x].z, raw[x].w};
                unsigned h[8];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const unsigned a = __byte_perm(w[e], 0, 0x1404), b = __byte_perm(w[e], 0, 0x3424);
                    const unsigned ma = magnitudes(a), mb = magnitudes(b);
                    largest = __vimax3_u16x2(largest, ma, mb);
                    h[2 * e] = widened(a, ma);
                    h[2 * e + 1] = widened(b, mb);
                }
                if constexpr (decltype(values)::value) {
                    const unsigned by = __shfl_sync(0xffffffffu, factor, 4 * x + row);
#pragma unroll
                    for (int e = 0; e < 8; ++e) h[e] = mul_f16(h[e], by);
                }
                *reinterpret_cast<uint4*>(to + place(r, 2 * c)) = make_uint4(h[0], h[1], h[2], h[3]);
                *reinterpret_cast<uint4*>(to + place(r, 2 * c + 1)) = make_uint4(h[4], h[5], h[6], h[7]);
            }
        };
        // Whether the vector whose scale the lane has holds such a code (looked at once more: this is rare).
        auto mine_is_none = [&](const unsigned char* pages, int i) -> bool {
            const Slice at = look_up(i, lane >> 4);
            const int r = lane & 15;
            unsigned found = 0;
            if (r >= at.begin && r < at.end)
#pragma unroll 1
                for (int x = 0; x < D; x += 4) found |= (*reinterpret_cast<const unsigned*>(pages + (at.vector + r) * D + x) & 0x7F7F7F7Fu) + 0x01010101u;
            return (found & 0x80808080u) != 0;
        };
        auto load_scales = [&](const Slice (&at)[2], int i) {
            const int r = lane & 15, j = (t_begin + i) * KEYS + first + lane;
            const bool second = lane >= SLICE;
            const long vector = second ? at[1].vector : at[0].vector;
            const bool here = r >= (second ? at[1].begin : at[0].begin) && r < (second ? at[1].end : at[0].end);
            k_s = here ? a.k_scale[vector + r] : 0.0f;
            v_s = here ? a.v_scale[vector + r] : j >= lo_min && j <= pmax ? -1.0f : 0.0f;
        };
        Slice at[2] = {look_up(0, 0), look_up(0, 1)};
        load(k_raw, a.k_pages, at);
        load(v_raw, a.v_pages, at);
        load_scales(at, 0);
        at[0] = look_up(1, 0);
        at[1] = look_up(1, 1);
        for (int i = 0; i < n_tiles; ++i) {
            const int s = i & 1;
            if (i >= 2) ok = __all_sync(0xffffffffu, mbar_wait(k_empty0 + 8 * s, ((i >> 1) - 1) & 1, 1));
            if (!ok) break;
            largest = 0;
            store(k_raw, sk + s * TILE_BYTES, std::false_type(), 0u);
            handed_over(k_full0 + 8 * s);
            load(k_raw, a.k_pages, at);
            if (i >= 2) ok = __all_sync(0xffffffffu, mbar_wait(v_empty0 + 8 * s, ((i >> 1) - 1) & 1, 1));
            if (!ok) break;
            {
                // the largest scale, the smallest but 0, both as bits (beyond every number's: one that is none, or no key)
                const unsigned bits = __float_as_uint(v_s), most = __reduce_max_sync(0xffffffffu, bits);
                const unsigned least = __reduce_min_sync(0xffffffffu, bits == 0 ? 0x7F800000u : bits);
                const bool wide = most >= 0x7E000000u || (most != 0 && least + (11u << 23) < most) || (most != 0 && most < 0x06000000u);
                const int e = most == 0 || wide ? 0 : (int)(most >> 23) - 126;
                const float by = wide ? 1.0f : v_s * __uint_as_float((unsigned)(127 - e) << 23);
                store(v_raw, sv + s * TILE_BYTES, std::true_type(), f16_pair(32768.0f * by, 32768.0f * by));
                // (a row that sees a value which is none gets none through its score: the values are stored by their scale already)
                if (__any_sync(0xffffffffu, max(largest & 0xFFFFu, largest >> 16) == NO_NUMBER) && (mine_is_none(a.k_pages, i) || mine_is_none(a.v_pages, i)))
                    k_s = __uint_as_float(0x7FC00000u);
                scales[s].key[first + lane] = few::key_scale(k_s);
                scales[s].value[first + lane] = v_s;
                if (lane == 0) {
                    const int g = warp - FIRST_CONVERT;
                    scales[s].log_power[g] = (float)e;
                    scales[s].inverse[g] = __uint_as_float((unsigned)(127 - e) << 23);
                    scales[s].apart[g] = wide;
                }
            }
            handed_over(v_full0 + 8 * s);
            load(v_raw, a.v_pages, at);
            load_scales(at, i + 1);
            at[0] = look_up(i + 2, 0);
            at[1] = look_up(i + 2, 1);
        }
    } else if (warp == ISSUER) {
        // M = 128, N = 128, f16 in, float32 out
        const unsigned idesc_qk = (1u << 4) | ((unsigned)(KEYS >> 3) << 17) | ((unsigned)(ROWS >> 4) << 24), idesc_pv = idesc_qk | (1u << 16);
        if (lane == 0 && n_tiles > 0) {
            auto issue_qk = [&](int t, int i) {
                const int s = i & 1;
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    const unsigned off = (k >> 2) * HALF_BYTES + (k & 3) * 32;
                    umma(tmem + t * 128, desc_k_major(smem_u32(sq + t * TILE_BYTES) + off), desc_k_major(smem_u32(sk + s * TILE_BYTES) + off), idesc_qk, k != 0);
                }
                umma_commit(s_full0 + 8 * t);
            };
            auto issue_pv = [&](int t, int i, int h) {      // 16 keys are eight columns of P and 16 rows of V
                const int s = i & 1;
#pragma unroll
                for (int k = 4 * h; k < 4 * h + 4; ++k)
                    umma_ts(tmem + 256 + t * 128, tmem + t * 128 + k * 8, desc_mn_major(smem_u32(sv + s * TILE_BYTES) + k * 16 * 128, HALF_BYTES), idesc_pv, (i | k) != 0);
            };
            ok = mbar_wait(q_full, 0, 2) && mbar_wait(k_full0, 0, 2);
            if (ok) {
                fence_after();
                for (int t = 0; t < 2; ++t)
                    if (n_tiles_t[t] > 0) issue_qk(t, 0);
                umma_commit(k_empty0);
            }
            for (int i = 0; i < n_tiles && ok; ++i) {
                const int s = i & 1;
                bool have_v = false, have_k = false;
                for (int t = 0; t < 2 && ok; ++t) {
                    if (i < n_tiles_t[t]) {
                        if (!mbar_wait(p_full0 + 16 * t, i & 1, 4)) { ok = false; break; }
                        if (!have_v && !mbar_wait(v_full0 + 8 * s, (i >> 1) & 1, 3)) { ok = false; break; }
                        have_v = true;
                        fence_after();
                        issue_pv(t, i, 0);
                        umma_commit(h_done0 + 8 * t);
                        if (!mbar_wait(p_full0 + 16 * t + 8, i & 1, 4)) { ok = false; break; }
                        fence_after();
                        issue_pv(t, i, 1);
                        if (i == n_tiles_t[t] - 1) umma_commit(o_full0 + 8 * t);
                    }
                    if (i + 1 < n_tiles_t[t]) {
                        if (!have_k && !mbar_wait(k_full0 + 8 * (s ^ 1), ((i + 1) >> 1) & 1, 2)) { ok = false; break; }
                        have_k = true;
                        fence_after();
                        issue_qk(t, i + 1);
                    }
                }
                if (!ok) break;
                umma_commit(v_empty0 + 8 * s);
                if (i + 1 < n_tiles) umma_commit(k_empty0 + 8 * (s ^ 1));
            }
        }
        ok = __all_sync(0xffffffffu, ok);
    } else if (warp < FIRST_CONVERT) {
        const int t = warp >> 2, r = (warp & 3) * 32 + lane, ti = r / group, head = kvh * group + r - ti * group;
        const bool valid = ti < n_tok_t[t];
        const long row = row0 + t * tpt + ti;
        const int pos = valid ? a.positions[row] : -1, lo = valid ? ib_first_visible(pos, a.span) : 0;
        const unsigned lanes = (unsigned)((warp & 3) * 32) << 16, s_addr = tmem + lanes + t * 128, o_addr = s_addr + 256;
        // the row's query
        float factor;
        {
            uint4 raw[16];
            unsigned largest = 0;
            const uint4* src = reinterpret_cast<const uint4*>(a.q + (row * a.n_heads + head) * D);
#pragma unroll
            for (int x = 0; x < 16; ++x) {
                raw[x] = valid ? src[x] : make_uint4(0, 0, 0, 0);
                largest = __vmaxu2(__vmaxu2(largest, raw[x].x & 0x7FFF7FFFu), __vmaxu2(raw[x].y & 0x7FFF7FFFu, __vmaxu2(raw[x].z & 0x7FFF7FFFu, raw[x].w & 0x7FFF7FFFu)));
            }
            largest = max(largest & 0xFFFF0000u, largest << 16);
            const int e = (int)(largest >> 23), up = largest == 0 ? 0 : 140 - e < 127 ? 140 - e : 127;
            const float by = copysignf(__uint_as_float((unsigned)(up + 127) << 23), a.scale);
            factor = e == 255 ? __uint_as_float(0x7FC00000u) : 256.0f * (a.scale * 1.4426950408889634f / by);      // a query that is none
            if (factor == 0.0f) factor = 1.17549435e-38f;      // (a hidden score times it stays one)
            unsigned char* to = sq + t * TILE_BYTES;
#pragma unroll
            for (int x = 0; x < 16; ++x) {
                const unsigned w[4] = {raw[x].x, raw[x].y, raw[x].z, raw[x].w};
                unsigned h[4];
#pragma unroll
                for (int y = 0; y < 4; ++y) h[y] = f16_pair(__uint_as_float(w[y] << 16) * by, __uint_as_float(w[y] & 0xFFFF0000u) * by);
                *reinterpret_cast<uint4*>(to + place(r, x)) = make_uint4(h[0], h[1], h[2], h[3]);
            }
            handed_over(q_full);
        }
        const unsigned long long factor2 = two(factor, factor);
        float ref = -INFINITY, l = 0.0f;      // what P and O are relative to, and the sum
        const int my_tiles = n_tiles_t[t];
        for (int i = 0; i < my_tiles; ++i) {
            const Scales& of = scales[i & 1];
            if (ok && !mbar_wait(v_full0 + 8 * (i & 1), (i >> 1) & 1, 5)) ok = false;
            if (ok && !mbar_wait(s_full0 + 8 * t, i & 1, 5)) ok = false;
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            fence_after();
#pragma unroll 1
            for (int h = 0; h < 2 && ok; ++h) {
                const int in = 64 * h, key0 = (t_begin + i) * KEYS + in;
                unsigned v[2][32];
                tmem_ld32_issue(s_addr + in, v[0]);
                tmem_ld32_issue(s_addr + in + 32, v[1]);
                tmem_ld_wait();
                // t = S * key scale; s + e = t * factor + e is what the reference is one for.  Keys with scales far apart: that at once, each
                // with its own logarithm
                const bool all = key0 >= lo && key0 + 63 <= pos;
                const int2 far = *reinterpret_cast<const int2*>(of.apart + 2 * h);
                const float2 power = *reinterpret_cast<const float2*>(of.log_power + 2 * h);
                float mx = -INFINITY;
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const bool wide = (b == 0 ? far.x : far.y) != 0;
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        unsigned* x = v[b] + j;
                        const float4 ks = *reinterpret_cast<const float4*>(of.key + in + 32 * b + j);
                        const float2 t0 = apart(mul2(two(__uint_as_float(x[0]), __uint_as_float(x[1])), two(ks.x, ks.y)));
                        const float2 t1 = apart(mul2(two(__uint_as_float(x[2]), __uint_as_float(x[3])), two(ks.z, ks.w)));
                        x[0] = __float_as_uint(t0.x); x[1] = __float_as_uint(t0.y); x[2] = __float_as_uint(t1.x); x[3] = __float_as_uint(t1.y);
                    }
                    if (wide) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            const float value = of.value[in + 32 * b + j];
                            const float y = __uint_as_float(v[b][j]) * factor + fmaxf(lg2(value), LEAST) + (value - value);      // (none, if that is none)
                            v[b][j] = __float_as_uint(value < 0.0f ? -INFINITY : y);
                        }
                    }
                    if (!all) {
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (key0 + 32 * b + j < lo || key0 + 32 * b + j > pos) v[b][j] = 0xff800000u;
                    }
                    float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        m0 = max3(m0, __uint_as_float(v[b][j]), __uint_as_float(v[b][j + 1]));
                        m1 = max3(m1, __uint_as_float(v[b][j + 2]), __uint_as_float(v[b][j + 3]));
                    }
                    m0 = fmaxf(m0, m1);
                    mx = fmaxf(mx, wide ? m0 : m0 * factor + (b == 0 ? power.x : power.y));
                }
                const bool move = mx > ref + SLACK || (ref == -INFINITY && mx > -INFINITY);
                if ((i | h) != 0 && __any_sync(0xffffffffu, move)) {
                    // O stands still while its rows are scaled: in the first half, for S of this tile is there and all products
                    // before it are done; in the second the first half's have to be
                    if (h == 1 && !mbar_wait(h_done0 + 8 * t, i & 1, 6)) ok = false;
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    fence_after();
                    const float fade = move ? (ref == -INFINITY ? 0.0f : ex2(ref - mx)) : 1.0f;
#pragma unroll 1
                    for (int x = 0; x < D; x += 16) {
                        float o[16];
                        tmem_ld16(o_addr + x, o);
                        unsigned w[16];
#pragma unroll
                        for (int j = 0; j < 16; ++j) w[j] = __float_as_uint(o[j] * fade);
                        tmem_st16(o_addr + x, w);
                    }
                    l *= fade;
                }
                if (move) ref = mx;
                const float less = ref == -INFINITY ? 0.0f : -ref;
                const float2 inverse = *reinterpret_cast<const float2*>(of.inverse + 2 * h);
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    unsigned w[16];
                    if ((b == 0 ? far.x : far.y) == 0) {
                        const float add = (b == 0 ? power.x : power.y) + less;
                        const unsigned long long add_2 = two(add, add);
                        unsigned long long sum2[2] = {two(0.0f, 0.0f), two(0.0f, 0.0f)};
#pragma unroll
                        for (int j = 0; j < 32; j += 2) {
                            float2 x = apart(fma2(two(__uint_as_float(v[b][j]), __uint_as_float(v[b][j + 1])), factor2, add_2));
                            x.x = ex2(x.x); x.y = ex2(x.y);
                            sum2[j / 2 & 1] = add2(sum2[j / 2 & 1], two(x.x, x.y));
                            w[j / 2] = f16_pair(x.x, x.y);
                        }
                        const float2 sum = apart(add2(sum2[0], sum2[1]));
                        l += (sum.x + sum.y) * (b == 0 ? inverse.x : inverse.y);
                    } else {
#pragma unroll
                        for (int j = 0; j < 32; j += 2) {
                            float p[2];
#pragma unroll
                            for (int x = 0; x < 2; ++x) {
                                const float lv = lg2(of.value[in + 32 * b + j + x]), y = __uint_as_float(v[b][j + x]) + less;
                                const bool hidden = v[b][j + x] == 0xff800000u;
                                const float s = y - fmaxf(lv, LEAST);
                                l += hidden ? 0.0f : ex2(s);
                                p[x] = hidden ? 0.0f : ex2(s + lv);
                            }
                            w[j / 2] = f16_pair(p[0], p[1]);
                        }
                    }
                    tmem_st16(s_addr + 32 * h + 16 * b, w);
                }
                tmem_st_wait();
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full0 + 16 * t + 8 * h);
            }
            if (!ok) break;
        }
        if (ok && my_tiles > 0) ok = __all_sync(0xffffffffu, mbar_wait(o_full0 + 8 * t, 0, 6));
        if (ok) {
            fence_after();
            const float inv = l != 0.0f ? 0.0078125f / l : 0.0f;      // a row that sees no key: zeros
            __nv_bfloat16* dst = a.out + row * a.out_ld + (long)head * D;
#pragma unroll 1
            for (int x = 0; x < D; x += 16) {
                float o[16];
                __syncwarp();      // rows of no token skip the stores
                if (my_tiles > 0) tmem_ld16(o_addr + x, o);
                unsigned w[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j] = inv == 0.0f ? 0u : pack_bf16(o[2 * j] * inv, o[2 * j + 1] * inv);
                if (!valid) continue;
                if (a.wide) {
                    *reinterpret_cast<uint4*>(dst + x) = make_uint4(w[0], w[1], w[2], w[3]);
                    *reinterpret_cast<uint4*>(dst + x + 8) = make_uint4(w[4], w[5], w[6], w[7]);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        reinterpret_cast<unsigned short*>(dst + x)[2 * j] = (unsigned short)w[j];
                        reinterpret_cast<unsigned short*>(dst + x)[2 * j + 1] = (unsigned short)(w[j] >> 16);
                    }
                }
            }
        }
    }
    // after a wait that ran out the products in flight are given time to end before the shared memory is given back
    if (!ok) for (const unsigned long long since = global_ns(); global_ns() - since < 20000000ull;) {}
    fence_before();
    __syncthreads();
    if (warp == ISSUER) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

}  // namespace kv8p

IB_EXPORT int ib_attention_kv8_error(int reset) {
    int v = 0;
    cudaError_t e = cudaMemcpyFromSymbol(&v, kv8p::g_error, sizeof(int));
    if (e != cudaSuccess) return -(int)e;
    if (reset && v != 0) {
        const int zero = 0;
        cudaMemcpyToSymbol(kv8p::g_error, &zero, sizeof(int));
    }
    return v;
}
IB_EXPORT int ib_attention_kv8_error_async(int* out, cudaStream_t stream) {
    return (int)cudaMemcpyFromSymbolAsync(out, kv8p::g_error, sizeof(int), 0, cudaMemcpyDeviceToHost, stream);
}

// Tile i holds up to 2 * (128 / group) rows of request tile_req[i] (-1: none) from row tile_row0[i] on, the request's rows
// end at q_start[r + 1], and their positions grow.
int ib_kv8_prompt(const IbAttentionKv8* c) {
    using namespace kv8p;
    const int group = (int)(c->n_heads / c->n_kv);
    if (c->d != D || group > ROWS || c->tile_tokens > 2 * (ROWS / group) || reinterpret_cast<uintptr_t>(c->q) % 16) return IB_ERR_UNSUPPORTED;
    if (c->n_tiles * c->n_kv > 0x7FFFFFFF) return IB_ERR_UNSUPPORTED;
    static IbDeviceSet done;
    if (int r = ib_allow_dynamic_smem(done, prompt_kernel, SMEM)) return r;
    const Args a = {(const __nv_bfloat16*)c->q, (const unsigned char*)c->k_pages, (const unsigned char*)c->v_pages, c->k_scale, c->v_scale,
                    c->block_table, c->positions, c->tile_req, c->tile_row0, c->q_start, (__nv_bfloat16*)c->out, c->out_ld,
                    (int)c->max_pages, (int)c->page_size, (int)c->n_pages, (int)c->n_req, (int)c->n, (int)c->n_heads, (int)c->n_kv, (int)c->tile_tokens,
                    (int)c->span, reinterpret_cast<uintptr_t>(c->out) % 16 == 0 && c->out_ld % 8 == 0, (float)c->scale};
    ib_launch(prompt_kernel, dim3((unsigned)(c->n_tiles * c->n_kv)), dim3(THREADS), SMEM, c->stream, a);
    return ib_launch_status();
}
